"""The 8-bit cache: the store of keys and values as e4m3 codes with a scale per page and head, and
decode attention over them, against plain 64-bit implementations."""
import math
from types import SimpleNamespace

import pytest
import torch

from plain import e4m3_plain as P

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF, F32 = torch.bfloat16, torch.float32
PAGE = 64


def rnd(*shape, dtype=F32, seed=0, scale=1.0):
    g = torch.Generator(device="cpu").manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).to(DEV)


def make_view(n_slots, cap, nkv, hd, hdv, seed, page=PAGE, spare=2):
    """A cache entry full of other tokens' codes, its pages in a random order."""
    g = torch.Generator(device="cpu").manual_seed(seed)
    pages = n_slots * (cap // page) + spare
    table = torch.randperm(pages, generator=g)[:n_slots * (cap // page)].reshape(n_slots, -1)

    def pool(dim):
        c = (torch.randn(pages, page, nkv, dim, generator=g) * 90).clamp(-448, 448).to(P.F8)
        return c.to(DEV), torch.exp2(torch.randint(-9, -4, (pages, nkv), generator=g).float()).to(DEV)
    k, ks = pool(hd)
    v, vs = pool(hdv)
    return SimpleNamespace(k_pool=k, v_pool=v, k_scale=ks, v_scale=vs, page=page, cap=cap,
                           page_table=table.int().contiguous().to(DEV), window=None)


def make_ctx(counts, lens, slots):
    i = dict(dtype=torch.int32, device=DEV)
    cu = [0]
    for n in counts:
        cu.append(cu[-1] + n)
    return SimpleNamespace(batch=len(counts), cu_seqlens=torch.tensor(cu, **i),
                           slots=torch.tensor(slots, **i), lens=torch.tensor(lens, **i),
                           positions=torch.tensor([n - 1 for n in lens], **i),
                           seq_index=torch.arange(len(lens), **i),
                           max_new=max(counts), max_len=max(lens), mode="decode", cu=cu)


def check_store(view, ctx, k, v, nkv, hd, hdv):
    """Runs the store and compares codes and scales, every one of the pools', with the plain form."""
    from agave_b200 import kernels
    want = []
    for x, pool, scale, dim in ((k, view.k_pool, view.k_scale, hd), (v, view.v_pool, view.v_scale, hdv)):
        codes, scales = pool.float().double().cpu(), scale.double().cpu()
        P.store(x.cpu().reshape(-1, nkv, dim), codes, scales, view.page_table.cpu(), ctx.cu,
                ctx.slots.tolist(), ctx.lens.tolist(), view.page, view.cap)
        want.append((codes, scales))
    kernels.cache_store_e4m3(k, v, view, ctx, nkv, hd, value_dim=hdv)
    for (codes, scales), pool, scale in zip(want, (view.k_pool, view.v_pool), (view.k_scale, view.v_scale)):
        assert torch.equal(scale.double().cpu(), scales)
        got = pool.float().double().cpu()
        assert torch.equal(got.isnan(), codes.isnan())
        assert torch.equal(got.nan_to_num(0.0), codes.nan_to_num(0.0))


HEADS = [(1, 256, 256), (3, 64, 64), (2, 16, 48), (4, 128, 80), (2, 192, 128)]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("nkv,hd,hdv", HEADS)
@pytest.mark.parametrize("counts,lens", [
    ([1], [1]), ([1, 63, 64, 65, 200], [1, 63, 64, 65, 200]),            # prompts
    ([70, 1, 30, 128], [75, 65, 130, 192]),                              # going on inside a page
    ([1, 1, 1, 1, 1], [1, 64, 65, 66, 200])])                            # single tokens
def test_store_codes_and_scales(dtype, nkv, hd, hdv, counts, lens):
    view = make_view(7, 256, nkv, hd, hdv, seed=1)
    T = sum(counts)
    # rows of magnitudes between 2^-6 and 2^6, so that some pages' scales grow and some do not
    mag = torch.exp2(torch.randint(-6, 7, (T, 1), generator=torch.Generator().manual_seed(5)).float())
    kv = (torch.randn(T, nkv * (hd + hdv), generator=torch.Generator().manual_seed(6)) * mag).to(dtype).to(DEV)
    k, v = kv[:, :nkv * hd], kv[:, nkv * hd:]                            # strided rows
    ctx = make_ctx(counts, lens, [3, 0, 6, 2, 1][:len(counts)])
    check_store(view, ctx, k, v, nkv, hd, hdv)
    check_store(view, ctx, k, v, nkv, hd, hdv)                           # once more: nothing moves


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("nkv,hd,hdv,page", [(2, 64, 64, 64), (1, 256, 128, 64), (2, 80, 48, 64), (2, 272, 320, 64),
                                             (2, 64, 128, 128), (3, 128, 64, 16), (1, 16, 16, 1)])
@pytest.mark.parametrize("off", [0, 1, 8])
def test_store_of_rows_anywhere(dtype, nkv, hd, hdv, page, off):
    """Rows that start on no 16-byte boundary, pages of other sizes, heads wider than attention takes."""
    view = make_view(4, 256, nkv, hd, hdv, seed=1, page=page)
    counts, lens = [100, 3, 64, 41], [100, 80, 64, 250]
    wide = rnd(sum(counts), nkv * (hd + hdv) + 11, dtype=dtype, seed=2, scale=3.0)
    k, v = wide[:, off:off + nkv * hd], wide[:, off + nkv * hd:off + nkv * (hd + hdv)]
    check_store(view, make_ctx(counts, lens, [1, 3, 0, 2]), k, v, nkv, hd, hdv)
    # max_new says less than is brought: the rest is stored all the same
    ctx = make_ctx(counts, [n + 5 for n in lens], [1, 3, 0, 2])
    ctx.max_new = 1
    check_store(view, ctx, k, v, nkv, hd, hdv)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("page", [16, 64])
def test_store_in_a_ring(dtype, page):
    """A prompt longer than the ring leaves its last pages; then tokens one by one wrap around."""
    nkv, hd, hdv, cap = 2, 32, 64, 4 * page
    view = make_view(3, cap, nkv, hd, hdv, seed=2, page=page)
    n = [9 * page + 5, 3, 6 * page]
    ctx = make_ctx(n, n, [2, 0, 1])
    check_store(view, ctx, rnd(sum(n), nkv * hd, dtype=dtype, seed=1), rnd(sum(n), nkv * hdv, dtype=dtype, seed=2),
                nkv, hd, hdv)
    for i in range(2 * page + 3):
        ctx = make_ctx([1] * 3, [x + 1 + i for x in n], [2, 0, 1])
        f = 2.0 ** (i % 7 - 3)
        check_store(view, ctx, rnd(3, nkv * hd, dtype=dtype, seed=10 + i, scale=f),
                    rnd(3, nkv * hdv, dtype=dtype, seed=500 + i, scale=1 / f), nkv, hd, hdv)


def test_store_of_unusual_values():
    """Zeros, infinities and NaN, the greatest and the smallest numbers, ties between two codes."""
    nkv, hd = 2, 64
    view = make_view(2, 128, nkv, hd, hd, seed=3)
    big = torch.finfo(F32).max
    rows = [torch.zeros(nkv * hd), torch.full((nkv * hd,), big), torch.full((nkv * hd,), 1e-40),
            torch.full((nkv * hd,), math.inf), torch.full((nkv * hd,), -math.nan),
            torch.arange(nkv * hd).float() / 16, torch.full((nkv * hd,), 448.0), -torch.full((nkv * hd,), 448.001),
            torch.full((nkv * hd,), 2.0 ** -140), torch.linspace(-1, 1, nkv * hd) * 2.0 ** -120]
    rows[5][3] = math.inf
    rows[6][70] = math.nan
    for i, r in enumerate(rows):
        for j, r2 in enumerate(rows):
            x = torch.stack([r, r2]).to(DEV)
            ctx = make_ctx([2], [2], [1])
            check_store(view, ctx, x, x.flip(0).contiguous(), nkv, hd, hd)
            ctx = make_ctx([1], [3], [1])
            check_store(view, ctx, x[:1] * 3, x[1:], nkv, hd, hd)


def test_store_leaves_padding_and_bad_pages_alone():
    """Entries without a slot, slots and pages outside the cache, and entries without tokens store
    nothing; their neighbours do."""
    from agave_b200 import kernels
    nkv, hd = 2, 64
    view = make_view(4, 128, nkv, hd, hd, seed=4)
    view.page_table[1, 0] = -1
    view.page_table[2, 1] = view.k_pool.shape[0]
    counts, lens = [5, 70, 100, 0, 3], [5, 70, 100, 1, 3]
    ctx = make_ctx(counts, lens, [-1, 1, 2, 0, 3])
    x = rnd(sum(counts), 2 * nkv * hd, seed=7)
    check_store(view, ctx, x[:, :nkv * hd], x[:, nkv * hd:], nkv, hd, hd)
    before = view.k_pool.view(torch.uint8).clone()
    ctx = make_ctx([2, 3], [2, 3], [4, 1 << 30])                         # slots behind the table
    kernels.cache_store_e4m3(x[:5, :nkv * hd], x[:5, nkv * hd:], view, ctx, nkv, hd)
    ctx = make_ctx([4], [3], [0])                                        # more tokens than the length
    kernels.cache_store_e4m3(x[:4, :nkv * hd], x[:4, nkv * hd:], view, ctx, nkv, hd)
    assert torch.equal(before, view.k_pool.view(torch.uint8))


# ------------------------------------------------------------------------------ attention
def check_attend(view, q, ctx, nh, nkv, hd, hdv, scale, window=0, out=None, **opt):
    """The kernel against the 64-bit form.  A score is off by at most d = (2^-21 + (hd + 8) 2^-24) *
    scale * max_j sum |q||k| (the query split into two 11-bit halves, products summed in 32 bits) plus
    2^-21 * (1 + |score|) for the exponential's argument; the weights then by a factor of e^(2 d), their sum and that of the
    values by (n + 16) 2^-24; bfloat16 rounds the weights to 11 bits and the result by 2^-8."""
    from agave_b200 import kernels
    if out is None:
        out = torch.full((q.shape[0], nh * hdv), math.nan, dtype=q.dtype, device=DEV)
    kernels.attention_decode_e4m3(q, out, view, ctx, nh, nkv, hd, scale, window, value_dim=hdv, **opt)
    ref, mag, vmax, seen = P.attend(q, view.k_pool.float(), view.k_scale, view.v_pool.float(), view.v_scale,
                                    view.page_table, ctx.slots.tolist(), ctx.positions.tolist(), view.page,
                                    view.cap, nh, scale, window, opt.get("keep_first", 0),
                                    opt.get("sinks"), opt.get("dist_bias"), opt.get("softcap", 0.0))
    got = out.double().reshape(ref.shape)
    n = torch.tensor(seen, device=DEV, dtype=torch.float64)[:, None]
    b = opt.get("dist_bias")
    most = mag + (b.abs().max().double() if b is not None else 0)
    d = (2.0 ** -21 + (hd + 8) * 2.0 ** -24) * mag + 2.0 ** -21 * (1 + most)
    rel = torch.expm1(2 * d) + (n + 16) * 2.0 ** -24 + (2.0 ** -11 if q.dtype == BF else 0)
    tol = rel[:, :, None] * vmax + (2.0 ** -8 if q.dtype == BF else 2.0 ** -24) * ref.abs()
    bad = ~((got - ref).abs() <= tol)
    assert not bad.any(), (int(bad.sum()), float((got - ref).abs().max()), float(tol.max()))
    return out


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("nh,nkv,hd,hdv", [(4, 1, 256, 256), (6, 3, 64, 64), (8, 2, 16, 48), (3, 3, 128, 80),
                                           (16, 2, 128, 128), (20, 2, 80, 192), (17, 1, 64, 256), (2, 2, 192, 16)])
@pytest.mark.parametrize("window", [0, 100, -96])
def test_attention_of_unequal_lengths(dtype, nh, nkv, hd, hdv, window):
    lens = [1, 2, 15, 16, 17, 63, 64, 65, 100, 129, 300, 1, 511]
    view = make_view(14, 512, nkv, hd, hdv, seed=1)
    ctx = make_ctx([1] * len(lens), lens, [5, 0, 13, 2, 1, 7, -1, 9, 3, 11, 4, 6, 8])
    wide = rnd(len(lens), nh * hd + 8, dtype=dtype, seed=2, scale=2.0)
    check_attend(view, wide[:, 8:], ctx, nh, nkv, hd, hdv, 0.5 * hd ** -0.5, window)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("opt", [dict(sinks=True), dict(softcap=5.0), dict(dist_bias=40), dict(dist_bias=1),
                                 dict(sinks=True, softcap=20.0, dist_bias=1000)])
@pytest.mark.parametrize("window,keep_first", [(0, 0), (70, 0), (70, 4), (70, 90), (1, 1), (-64, 0)])
def test_attention_options(dtype, opt, window, keep_first):
    nh, nkv, hd, hdv = 6, 2, 64, 128
    lens = [1, 64, 70, 71, 75, 160, 399]
    view = make_view(8, 448, nkv, hd, hdv, seed=3)
    ctx = make_ctx([1] * len(lens), lens, [5, 0, 2, 1, 7, 3, 4])
    q = rnd(len(lens), nh * hd, dtype=dtype, seed=4, scale=2.0)
    opt = dict(opt)
    if opt.get("sinks"):
        opt["sinks"] = rnd(nh, seed=5, scale=2.0)
    if opt.get("dist_bias"):
        opt["dist_bias"] = rnd(nh, opt["dist_bias"], seed=6)
    check_attend(view, q, ctx, nh, nkv, hd, hdv, hd ** -0.5, window, keep_first=keep_first, **opt)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_attention_in_a_ring(dtype):
    """Sequences much longer than the ring of the window and one page."""
    nh, nkv, hd = 4, 2, 64
    for window, lens in ((128, [5000, 129, 193, 192, 256]), (100, [65537, 64, 101, 191, 200])):
        cap = (window + 63) // 64 * 64 + 64
        view = make_view(6, cap, nkv, hd, hd, seed=5)
        ctx = make_ctx([1] * 5, lens, [2, 0, 5, 1, 4])
        check_attend(view, rnd(5, nh * hd, dtype=dtype, seed=6, scale=2.0), ctx, nh, nkv, hd, hd, hd ** -0.5, window)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("lens,nh,nkv,hd", [([20011], 8, 4, 256), ([9000, 1, 77], 2, 1, 128),
                                            ([4097] * 3, 16, 8, 64), ([3000] + [50, 700] * 70, 6, 3, 128),
                                            ([5000] * 2 + [3], 40, 2, 64), ([2500] * 5, 150, 150, 64)])
def test_attention_of_long_sequences(dtype, lens, nh, nkv, hd):
    cap = (max(lens) + 63) // 64 * 64
    view = make_view(len(lens), cap, nkv, hd, hd, seed=6)
    ctx = make_ctx([1] * len(lens), lens, list(range(len(lens)))[::-1])
    check_attend(view, rnd(len(lens), nh * hd, dtype=dtype, seed=7, scale=2.0), ctx, nh, nkv, hd, hd, hd ** -0.5)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("page", [16, 32, 128])
@pytest.mark.parametrize("window,keep_first", [(0, 0), (150, 0), (150, 20)])
def test_attention_with_pages_of_other_sizes(dtype, page, window, keep_first):
    nh, nkv, hd, lens = 4, 2, 64, [1, 16, 17, 63, 128, 300, 1000, 1024]
    view = make_view(9, 1024, nkv, hd, hd, seed=7, page=page)
    ctx = make_ctx([1] * len(lens), lens, [3, 1, 0, 8, 6, 2, 5, 4])
    q = rnd(len(lens), nh * hd, dtype=dtype, seed=8, scale=2.0)
    check_attend(view, q, ctx, nh, nkv, hd, hd, hd ** -0.5, window, keep_first=keep_first)
    # what max_len says sizes the launch, not what is seen
    for most in (1, 5000, 1 << 20):
        ctx.max_len = most
        check_attend(view, q, ctx, nh, nkv, hd, hd, hd ** -0.5, window, keep_first=keep_first)
    # a sequence without a key: zeros
    ctx.positions[2] = -1
    out = torch.full((len(lens), nh * hd), math.nan, dtype=dtype, device=DEV)
    from agave_b200 import kernels
    kernels.attention_decode_e4m3(q, out, view, ctx, nh, nkv, hd, hd ** -0.5, window)
    assert (out[2] == 0).all() and torch.isfinite(out).all()


@pytest.mark.parametrize("dtype", [BF, F32])
def test_attention_of_many_sequences(dtype):
    nh, nkv, hd = 4, 2, 64
    lens = [1 + (i * 37) % 190 for i in range(300)]
    view = make_view(301, 192, nkv, hd, hd, seed=8)
    slots = [(i * 7) % 301 for i in range(300)]
    slots[17] = slots[299] = -1
    ctx = make_ctx([1] * 300, lens, slots)
    check_attend(view, rnd(300, nh * hd, dtype=dtype, seed=9, scale=2.0), ctx, nh, nkv, hd, hd, hd ** -0.5)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_attention_with_scales_far_apart(dtype):
    """Pages whose scales differ by many powers of two: the small ones matter where the large ones'
    keys get no weight, and queries of any magnitude."""
    nh, nkv, hd = 2, 1, 64
    view = make_view(2, 512, nkv, hd, hd, seed=10)
    page = view.page_table[1].long()
    for shift, at in ((13, 0), (-13, 3), (20, 7)):
        view.v_scale.fill_(2.0 ** -7)
        view.k_scale.fill_(2.0 ** -7)
        view.v_scale[page[at]] *= 2.0 ** shift
        # keys of that page far below the others' scores
        bias = torch.zeros(nh, 512, device=DEV)
        p = 511
        bias[:, p - (at + 1) * 64 + 1:p - at * 64 + 1] = -60.0 if shift > 0 else 0.0
        ctx = make_ctx([1], [512], [1])
        for qs in (2.0, 2.0 ** 60, 2.0 ** -60):
            q = rnd(1, nh * hd, dtype=dtype, seed=11, scale=qs)
            # (the bound takes the values that carry weight: the far page's weights are below 2^-60)
            vs = view.v_scale.clone()
            got = torch.empty(1, nh * hd, dtype=dtype, device=DEV)
            from agave_b200 import kernels
            kernels.attention_decode_e4m3(q, got, view, ctx, nh, nkv, hd, hd ** -0.5 / qs, 0, dist_bias=bias)
            ref, mag, _, _ = P.attend(q, view.k_pool.float(), view.k_scale, view.v_pool.float(), vs,
                                      view.page_table, [1], [p], 64, 512, nh, hd ** -0.5 / qs, bias=bias)
            near = 448 * 2.0 ** -7
            tol = (2.0 ** -11 + 2.0 ** -8 if dtype == BF else 0) + 60 * 2.0 ** -20 + float(mag.max()) * 2.0 ** -18
            assert float((got.double().reshape(ref.shape) - ref).abs().max()) <= tol * near, (shift, qs)


def test_attention_masked_places_hold_anything():
    """NaN codes behind a sequence's end, before its window and in other pages reach no output; a NaN
    among the keys that are seen does."""
    nh, nkv, hd = 4, 2, 64
    lens = [1, 70, 130, 200]
    for dtype in (BF, F32):
        view = make_view(5, 256, nkv, hd, hd, seed=12)
        ctx = make_ctx([1] * 4, lens, [3, 0, 4, 1])
        window = 50
        k8, v8 = view.k_pool.view(torch.uint8), view.v_pool.view(torch.uint8)
        seen = torch.zeros(k8.shape[:2], dtype=torch.bool, device=DEV)
        for s, n in zip([3, 0, 4, 1], lens):
            for j in range(max(0, n - window), n):
                seen[int(view.page_table[s, j // 64]), j % 64] = True
        k8[~seen] = 0x7f
        v8[~seen] = 0xff
        unused = torch.ones(view.k_pool.shape[0], dtype=torch.bool, device=DEV)
        unused[view.page_table.long().flatten()] = False
        view.k_scale[unused] = math.nan
        q = rnd(4, nh * hd, dtype=dtype, seed=13)
        check_attend(view, q, ctx, nh, nkv, hd, hd, hd ** -0.5, window)
        k8[int(view.page_table[0, 1]), 3, 1, 5] = 0x7f                   # position 67 of the second
        got = torch.empty(4, nh * hd, dtype=dtype, device=DEV)
        from agave_b200 import kernels
        kernels.attention_decode_e4m3(q, got, view, ctx, nh, nkv, hd, hd ** -0.5, window)
        nan = got.reshape(4, nh, hd).isnan()
        assert nan[1, 2:].all() and not nan[1, :2].any() and not nan[[0, 2, 3]].any()


def test_attention_with_bad_pages_and_slots():
    """A page number outside the pool counts as keys that are not there; a slot outside the table as
    padding; neither is read."""
    from agave_b200 import kernels
    nh, nkv, hd = 4, 2, 64
    for dtype in (BF, F32):
        view = make_view(4, 256, nkv, hd, hd, seed=14)
        ctx = make_ctx([1] * 3, [200, 64, 90], [1, 9, 2])
        view.page_table[1, 1] = -5
        view.page_table[2, 0] = 1 << 30
        q = rnd(3, nh * hd, dtype=dtype, seed=15)
        got = torch.full((3, nh * hd), math.nan, dtype=dtype, device=DEV)
        kernels.attention_decode_e4m3(q, got, view, ctx, nh, nkv, hd, hd ** -0.5, 0)
        assert torch.isfinite(got).all() and (got[1] == 0).all()
        # the third as if it began at position 64
        two = make_ctx([1], [90], [2])
        check = torch.empty(1, nh * hd, dtype=dtype, device=DEV)
        kernels.attention_decode_e4m3(q[2:], check, view, two, nh, nkv, hd, hd ** -0.5, 26)
        assert float((check[0].double() - got[2].double()).abs().max()) <= 2.0 ** -6


# ------------------------------------------------------------------------- both, as they are used
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("window", [0, 40])
def test_prompts_then_tokens_one_by_one(dtype, window):
    """The store of prompts, then steps of a store and an attention, recorded once as a CUDA graph with
    its inputs in fixed buffers; a second graph of other sizes is replayed in between."""
    from agave_b200 import kernels
    nh, nkv, hd, hdv, cap = 6, 2, 64, 32, 128 if window else 256
    view = make_view(5, cap, nkv, hd, hdv, seed=20)
    slots, n = [4, 0, 2], [90, 1, 64]
    ctx = make_ctx(n, n, slots)
    check_store(view, ctx, rnd(sum(n), nkv * hd, dtype=dtype, seed=1), rnd(sum(n), nkv * hdv, dtype=dtype, seed=2),
                nkv, hd, hdv)
    B, W = 4, nh * hd + nkv * (hd + hdv)

    def record(B):
        i = dict(dtype=torch.int32, device=DEV)
        c = SimpleNamespace(cu_seqlens=torch.arange(B + 1, **i), slots=torch.full((B,), -1, **i),
                            lens=torch.zeros(B, **i), positions=torch.zeros(B, **i), max_new=1,
                            max_len=cap if not window else 4096, mode="decode", cu=list(range(B + 1)))
        row = torch.zeros(B, W, dtype=dtype, device=DEV)
        out = torch.zeros(B, nh * hdv, dtype=dtype, device=DEV)

        def body():
            kernels.cache_store_e4m3(row[:, nh * hd:(nh + nkv) * hd], row[:, (nh + nkv) * hd:], view, c, nkv, hd,
                                     value_dim=hdv)
            kernels.attention_decode_e4m3(row[:, :nh * hd], out, view, c, nh, nkv, hd, hd ** -0.5, window,
                                          value_dim=hdv)
        body()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            body()
        return c, row, out, graph
    c, row, out, graph = record(B)
    other = record(1)
    for step in range(80):
        lens = [x + step + 1 for x in n] + [0]
        row.copy_(rnd(B, W, dtype=dtype, seed=100 + step, scale=2.0 ** (step % 5 - 2)))
        c.lens.copy_(torch.tensor(lens)); c.positions.copy_(torch.tensor([x - 1 for x in lens]).clamp_min(0))
        c.slots.copy_(torch.tensor(slots + [-1]))
        k, v = row[:, nh * hd:(nh + nkv) * hd], row[:, (nh + nkv) * hd:]
        want = []
        for x, pool, scale, dim in ((k, view.k_pool, view.k_scale, hd), (v, view.v_pool, view.v_scale, hdv)):
            codes, scales = pool.float().double().cpu(), scale.double().cpu()
            P.store(x.cpu().reshape(-1, nkv, dim), codes, scales, view.page_table.cpu(), c.cu, slots + [-1], lens,
                    64, cap)
            want.append((codes, scales))
        graph.replay()
        other[3].replay()
        for (codes, scales), pool, scale in zip(want, (view.k_pool, view.v_pool), (view.k_scale, view.v_scale)):
            assert torch.equal(pool.float().double().cpu(), codes) and torch.equal(scale.double().cpu(), scales)
        got = out.clone()
        again = check_attend(view, row[:, :nh * hd], c, nh, nkv, hd, hdv, hd ** -0.5, window)
        assert torch.equal(got, again)


def test_two_streams_at_once():
    """Two calls that overlap on the GPU do not share scratch."""
    from agave_b200 import kernels
    nh, nkv, hd = 8, 2, 128
    views = [make_view(1, 16384, nkv, hd, hd, seed=30 + i) for i in range(2)]
    ctx = make_ctx([1], [16000], [0])
    qs = [rnd(1, nh * hd, dtype=BF, seed=40 + i) for i in range(2)]
    alone = [check_attend(v, q, ctx, nh, nkv, hd, hd, hd ** -0.5) for v, q in zip(views, qs)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[torch.zeros(1, nh * hd, dtype=BF, device=DEV) for _ in range(20)] for _ in range(2)]
    torch.cuda.synchronize()
    for i in range(20):
        for s in range(2):
            with torch.cuda.stream(streams[s]):
                kernels.attention_decode_e4m3(qs[s], outs[s][i], views[s], ctx, nh, nkv, hd, hd ** -0.5, 0)
    torch.cuda.synchronize()
    for s in range(2):
        for o in outs[s]:
            assert torch.equal(o, alone[s])


def test_refusals():
    from agave_b200 import kernels
    nh, nkv, hd = 4, 2, 64
    view = make_view(2, 128, nkv, hd, hd, seed=50)
    ctx = make_ctx([1, 1], [5, 6], [0, 1])
    q = rnd(2, nh * hd)
    k = rnd(2, nkv * hd)
    out = torch.empty_like(q)
    store, attend = kernels.cache_store_e4m3, kernels.attention_decode_e4m3
    E = kernels.KernelError
    with pytest.raises(E, match="current CUDA device"):
        store(k.cpu(), k, view, ctx, nkv, hd)
    with pytest.raises(E, match="do not fit"):
        store(k[:, :-1], k, view, ctx, nkv, hd)
    with pytest.raises(E, match="differ"):
        store(k, k.bfloat16(), view, ctx, nkv, hd)
    with pytest.raises(E, match="no kernels"):
        store(k.half(), k.half(), view, ctx, nkv, hd)
    with pytest.raises(E, match="adjacent"):
        store(k.t().contiguous().t(), k, view, ctx, nkv, hd)
    with pytest.raises(E, match="do not fit"):
        store(k, k, view, make_ctx([1], [1], [0]), nkv, hd, value_dim=32)
    bad = SimpleNamespace(**{**vars(view), "k_pool": view.k_pool.view(torch.uint8)})
    with pytest.raises(E, match="float8_e4m3fn"):
        store(k, k, bad, ctx, nkv, hd)
    with pytest.raises(E, match="scales"):
        store(k, k, SimpleNamespace(**{**vars(view), "k_scale": view.k_scale[:1]}), ctx, nkv, hd)
    with pytest.raises(E, match="not \\[pages"):
        attend(q, out, view, ctx, nh, 1, hd, 1.0, 0)
    with pytest.raises(E, match="multiples of 16"):
        attend(q[:, :nh * 24], out, view, ctx, nh, nkv, 24, 1.0, 0)
    with pytest.raises(E, match="multiples of 16"):
        attend(rnd(2, nh * 512), rnd(2, nh * 512), view, ctx, nh, nkv, 512, 1.0, 0)
    with pytest.raises(E, match="query heads"):
        attend(q[:, :3 * hd], out[:, :3 * hd].contiguous(), view, ctx, 3, nkv, hd, 1.0, 0)
    with pytest.raises(E, match="output"):
        attend(q, out.bfloat16(), view, ctx, nh, nkv, hd, 1.0, 0)
    with pytest.raises(E, match="sink"):
        attend(q, out, view, ctx, nh, nkv, hd, 1.0, 0, sinks=rnd(3))
    with pytest.raises(E, match="int32"):
        c = make_ctx([1, 1], [5, 6], [0, 1])
        c.slots = c.slots.long()
        attend(q, out, view, c, nh, nkv, hd, 1.0, 0)
    with pytest.raises(E, match="geometry"):
        attend(q, out, SimpleNamespace(**{**vars(view), "cap": 256}), ctx, nh, nkv, hd, 1.0, 0)
    # no sequences, no tokens: nothing happens
    none = SimpleNamespace(cu_seqlens=ctx.cu_seqlens[:1], slots=ctx.slots[:0], lens=ctx.lens[:0],
                           positions=ctx.positions[:0], max_new=0, max_len=0, mode="decode")
    store(k[:0], k[:0], view, none, nkv, hd)
    attend(q[:0], out[:0], view, none, nh, nkv, hd, 1.0, 0)
    none.max_len = 1 << 20
    attend(q[:0], out[:0], view, none, nh, nkv, hd, 1.0, 0)
