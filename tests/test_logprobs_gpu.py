"""Log-probabilities, entropy, rank and the greatest logits of rows, against 64-bit torch."""
import math

import pytest
import torch

from plain import e4m3_plain as P

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF, F32 = torch.bfloat16, torch.float32


def check(logits, tokens, top):
    """logprob = x_t - m - ln s: s is a sum of positive terms, each off by a factor of 1 + 2^-21 and by
    what rounding x - m (2^-24 of it, twice) does, summed at most V / 256 + 64 deep, so ln s is off by
    at most a = (V / 256 + 64) 2^-24 + 2^-21 + 2^-23 sum p |x - m|; x_t - m by 2^-24 of it.  The entropy
    ln s - t / s adds t's terms, which are off by the same factors."""
    from agave_b200 import kernels
    r = kernels.token_logprobs(logits, tokens, top=top)
    lp, ent, rank, ids, tlp, spread = P.logprobs(logits, tokens, top)
    R, V = logits.shape
    assert torch.equal(r.rank.long(), rank)
    if top == 0:
        assert r.top_ids is None and r.top_logprobs is None
        r.top_ids, r.top_logprobs = ids, tlp
    assert r.top_ids.shape == (R, top) and torch.equal(r.top_ids.long(), ids)
    a = (V / 256 + 64) * 2.0 ** -24 + 2.0 ** -21 + 2.0 ** -23 * spread
    none = torch.isnan(lp)
    assert torch.equal(torch.isnan(r.logprob), none)
    # (a token whose logit is -inf, or so far below the greatest that 32 bits have no number for it)
    shut = torch.isinf(lp.float())
    assert torch.equal(r.logprob[shut], lp.float()[shut])
    assert ((r.logprob.double() - lp).abs() <= a + 2.0 ** -22 * lp.abs())[~none & ~shut].all()
    assert ((r.entropy.double() - ent).abs() <= 3 * a * (1 + spread)).all()
    fine = torch.isfinite(tlp.float())
    assert torch.equal(r.top_logprobs[~fine], tlp.float()[~fine])
    err = (r.top_logprobs.double() - tlp).abs() <= a[:, None] + 2.0 ** -22 * tlp.abs()
    assert err[fine].all()
    return r


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("R,V", [(1, 1), (3, 2), (5, 31), (2, 33), (7, 1000), (1, 4097), (150, 777), (300, 3001),
                                 (1, 262144), (9, 50001), (40, 32768)])
def test_rows_of_many_sizes(dtype, R, V):
    g = torch.Generator().manual_seed(R * 7 + V)
    logits = (torch.randn(R, V, generator=g) * 4).to(dtype).to(DEV)
    tokens = torch.randint(0, V, (R,), generator=g).int().to(DEV)
    tokens[0] = V - 1
    for top in sorted({0, 1, min(V, 5), min(V, 32)}):
        check(logits, tokens, top)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("off", [0, 1, 3, 8])
def test_strided_and_unaligned_rows(dtype, off):
    g = torch.Generator().manual_seed(off)
    for V in (1000, 1003, 20000):
        wide = (torch.randn(6, V + 11, generator=g) * 4).to(dtype).to(DEV)
        tokens = torch.randint(0, V, (6,), generator=g).int().to(DEV)
        check(wide[:, off:off + V], tokens, 20)


@pytest.mark.parametrize("dtype", [F32, BF])
def test_ties_orders_and_masks(dtype):
    """Equal logits go by the index, ascending and descending rows, masked places, zeros of both signs."""
    V = 5000
    g = torch.Generator().manual_seed(1)
    rows = [torch.zeros(V), torch.arange(V).float(), -torch.arange(V).float(),
            torch.randint(0, 3, (V,), generator=g).float(), torch.full((V,), -math.inf),
            torch.randn(V, generator=g), torch.randn(V, generator=g) * 30, torch.randn(V, generator=g)]
    rows[0][1::2] = -0.0
    rows[4][[7, 4000, 4999]] = torch.tensor([1.0, 2.0, 1.0])
    rows[5][:4990] = -math.inf
    rows[7][:] = torch.finfo(F32).min if dtype == F32 else torch.finfo(BF).min
    rows[7][77] = 0.0
    logits = torch.stack(rows).to(dtype).to(DEV)
    for t in (0, 1, 7, 77, 2500, 4999):
        tokens = torch.full((len(rows),), t, dtype=torch.int32, device=DEV)
        for top in (1, 20, 32):
            check(logits, tokens, top)
    # (a small vocabulary of equal halves)
    x = torch.tensor([[1.0, 2.0, 2.0, 1.0, 2.0]], device=DEV).to(dtype)
    r = check(x, torch.tensor([4], dtype=torch.int32, device=DEV), 5)
    assert r.top_ids.tolist() == [[1, 2, 4, 0, 3]] and r.rank.tolist() == [3]


@pytest.mark.parametrize("dtype", [F32, BF])
def test_rows_of_the_lowest_value_and_few_that_are_left(dtype):
    """Rows that a mask has filled with the type's lowest number or -inf, all but a few places."""
    V = 40000
    low = float(torch.finfo(dtype).min)
    rows = [torch.full((V,), low) for _ in range(4)] + [torch.full((V,), -math.inf) for _ in range(3)]
    rows[1][12345] = 3.0
    rows[2][[1, 2, 39999]] = torch.tensor([low / 2, 1.0, -5.0])
    rows[3][::3] = float(torch.finfo(dtype).max)
    rows[4][39999] = low
    rows[5][[0, 7, 20000]] = torch.tensor([0.5, 0.5, -700.0])
    rows[6][20000:20010] = -1.0
    logits = torch.stack(rows).to(dtype).to(DEV)
    for t in (0, 7, 12345, 39999):
        tokens = torch.full((len(rows),), t, dtype=torch.int32, device=DEV)
        for top in (0, 3, 20, 32):
            if t == 7 or top in (0, 20):
                check(logits, tokens, top)


def test_the_greatest_all_in_one_place():
    """Descending and equal runs whose greatest logits are all one thread's or one piece's, and more of
    them than are kept in a list."""
    V = 3_000_000
    x = -torch.rand(1, V, generator=torch.Generator().manual_seed(4)).to(DEV)
    for stride in (1, 2048, 4096, 1 << 16):
        y = x.clone()
        y[0, 1000::stride][:1400] += 5
        check(y, torch.tensor([1000], dtype=torch.int32, device=DEV), 32)
    y = x.clone()
    for q in range(32):                                  # 32 threads' shares
        y[0, q * 4::2048] += 5
    check(y, torch.tensor([5], dtype=torch.int32, device=DEV), 32)


def test_rows_without_a_softmax_and_tokens_outside():
    from agave_b200 import kernels
    V = 3000
    x = torch.randn(5, V, generator=torch.Generator().manual_seed(2)).to(DEV)
    x[1, 17] = math.nan
    x[2, 2999] = math.inf
    x[3] = -math.inf
    t = torch.tensor([-1, 5, 5, 5, V], dtype=torch.int32, device=DEV)
    r = kernels.token_logprobs(x, t, top=3)
    assert r.logprob.isnan().all() and r.rank[[0, 4]].tolist() == [0, 0]
    assert r.entropy.isnan().tolist() == [False, True, True, True, False]
    assert r.top_logprobs[1:4].isnan().all() and torch.isfinite(r.top_logprobs[[0, 4]]).all()
    # the order among what there is
    assert r.top_ids[3].tolist() == [0, 1, 2] and int(r.top_ids[2, 0]) == 2999
    y = x[1].clone()
    y[17] = -math.inf
    assert torch.equal(r.top_ids[1].long(), torch.sort(y, descending=True, stable=True).indices[:3])


def same(a, b):
    return all(torch.equal(getattr(a, n).view(torch.int32), getattr(b, n).view(torch.int32)) for n in a.__slots__)


def test_packed_results():
    from agave_b200 import kernels
    g = torch.Generator().manual_seed(8)
    for R, top in ((1, 0), (5, 3), (40, 32)):
        x = (torch.randn(R, 5000, generator=g) * 3).to(DEV)
        t = torch.randint(0, 5000, (R,), generator=g).int().to(DEV)
        r = kernels.token_logprobs(x, t, top)
        packed = torch.zeros(kernels.token_logprobs_words(R, top) + 5, device=DEV)
        assert kernels.token_logprobs(x, t, top, packed=packed) is None
        assert (packed[-5:] == 0).all()
        for a, b in zip(kernels.unpack_token_logprobs(packed.cpu().numpy(), R, top),
                        (r.logprob, r.entropy, r.rank, r.top_ids, r.top_logprobs)):
            if b is None:
                assert a.size == 0
                continue
            assert a.shape == b.shape and (a == b.cpu().numpy()).all()
        with pytest.raises(kernels.KernelError, match="packed"):
            kernels.token_logprobs(x, t, top, packed=packed[:2])


def test_recorded_and_replayed_and_streams():
    """A recording follows its inputs, and calls on two streams do not share anything."""
    from agave_b200 import kernels
    V = 70001
    g = torch.Generator().manual_seed(3)
    xs = [(torch.randn(4, V, generator=g) * 3).to(DEV) for _ in range(3)]
    ts = [torch.randint(0, V, (4,), generator=g).int().to(DEV) for _ in range(3)]
    x, t = xs[0].clone(), ts[0].clone()
    kernels.token_logprobs(x, t, top=7)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = kernels.token_logprobs(x, t, top=7)
    for a, b in zip(xs, ts):
        x.copy_(a); t.copy_(b)
        graph.replay()
        want = check(a, b, 7)
        assert same(r, want)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for s in range(2):
            with torch.cuda.stream(streams[s]):
                got[s].append(kernels.token_logprobs(xs[s], ts[s], top=7))
    torch.cuda.synchronize()
    for s in range(2):
        want = check(xs[s], ts[s], 7)
        for r in got[s]:
            assert same(r, want)


def test_refusals():
    from agave_b200 import kernels
    E = kernels.KernelError
    x = torch.zeros(2, 100, device=DEV)
    t = torch.zeros(2, dtype=torch.int32, device=DEV)
    for args, word in (((x.cpu(), t), "current CUDA device"), ((x, t.long()), "int32"), ((x, t[:1]), "one token"),
                       ((x, t, 33), "top"), ((x, t, -1), "top"), ((x[:, :3].contiguous(), t, 4), "top"),
                       ((x.half(), t), "no kernels"), ((x.t(), t), "vocabulary"), ((x[0], t), "vocabulary")):
        with pytest.raises(E, match=word):
            kernels.token_logprobs(*args)
    assert kernels.token_logprobs(x[:0], t[:0], 3).top_ids.shape == (0, 3)
