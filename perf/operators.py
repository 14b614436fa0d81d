"""The work by which three operators of serving are judged: keys and values stored in an 8-bit cache,
attention of single tokens over that cache, and the log-probabilities of given tokens.

The cache holds e4m3 codes (``torch.float8_e4m3fn``) in pages of ``PAGE`` positions, [pages, PAGE, kv
heads, head size], and one 32-bit scale for each page and kv head, [pages, kv heads], for keys and for
values apart; a value is code * scale.  Scales are powers of two, so that scaling rounds nothing and a
value is rounded once, to the nearest code, ties to even.

* ``store``: new tokens' keys and values of a batch of sequences.  The scale of a page and head is the
  smallest 2^e (e >= -126) with 448 * 2^e at or above every finite magnitude stored there; where a page already
  holds tokens of its sequence and a new one needs a greater scale, their codes are rounded to the
  greater scale.  Values that are not finite are held as NaN.  Outputs: the pools and the scales.
* ``attend``: one query per sequence, softmax over the keys it sees (all, the last ``window``, those
  and the first ``keep_first``), a sink logit per head and a soft cap of the scores as options; rows
  of padding entries (slot -1) are zeros.
* ``logprobs``: per row of logits, ln softmax at a given token, the entropy of the row in nats, the
  token's rank (1: none is greater; of equal ones the lower index comes first), and the ``top``
  greatest with their indices.  A token below 0 stands for none: NaN and rank 0.

Sizes are those of the models of the benchmark (262,144 and 262,208 logits, heads of 128 and 256,
1 to 16 kv heads) or generic.
"""
import math
from types import SimpleNamespace

import torch

own = False

PAGE = 64
_DT = {"bf16": torch.bfloat16, "f32": torch.float32}
_F8 = torch.float8_e4m3fn
DEV = "cuda:0"


# ------------------------------------------------------------------------------- the cases
def _store(name, seqs, length, new, kv_heads, head_dim, dtype="bf16", value_dim=0, window=0):
    return {"name": name, "op": "store", "seqs": seqs, "length": length, "new": new,
            "kv_heads": kv_heads, "head_dim": head_dim, "value_dim": value_dim or head_dim,
            "dtype": dtype, "window": window}


def _attend(name, seqs, length, heads, kv_heads, head_dim, dtype="bf16", value_dim=0, window=0,
            keep_first=0, sinks=False, softcap=0.0, padding=0):
    return {"name": name, "op": "attend", "seqs": seqs, "length": length, "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "value_dim": value_dim or head_dim,
            "dtype": dtype, "window": window, "keep_first": keep_first, "sinks": sinks,
            "softcap": softcap, "padding": padding}


def _logprobs(name, rows, vocab, top, dtype="f32", gap=0):
    return {"name": name, "op": "logprobs", "rows": rows, "vocab": vocab, "top": top,
            "dtype": dtype, "gap": gap}


def listed():
    return [
        # one chat, one layer of a decode step: nothing but latency
        _store("store one token", 1, 700, 1, 1, 256),
        # a full decode batch of a middle-sized model
        _store("store a token of 64", 64, 4000, 1, 4, 256),
        # a step of unequal prompts
        _store("store 16 prompts", 16, 2048, 1 << 30, 4, 256),
        # one long document in the 32-bit path, a layer with a window: only its last keys stay
        _store("store long, window, f32", 1, 32768, 1 << 30, 16, 128, "f32", window=16000),
        # one chat, a layer with a window
        _attend("attend one chat", 1, 700, 4, 1, 256, window=512),
        # one very long context
        _attend("attend one of 131072", 1, 131072, 8, 4, 256),
        # a full batch of unequal lengths, a large model
        _attend("attend 64 ragged", 64, 8192, 32, 16, 128),
        # the 32-bit path, with the options that the other architectures have
        _attend("attend 24, options, f32", 24, 3001, 6, 3, 64, "f32", window=1500, keep_first=4,
                sinks=True, softcap=30.0, padding=2),
        # the chosen token of one chat and five alternatives
        _logprobs("logprobs of one", 1, 262144, 5),
        # a full decode batch
        _logprobs("logprobs of 64", 64, 262144, 20),
        # scoring documents: every place of the prompts, no alternatives
        _logprobs("logprobs of 1500", 1500, 262208, 0),
        # 16-bit logits of a small vocabulary in a wider buffer
        _logprobs("logprobs of 777, bf16", 777, 32001, 8, "bf16", gap=31),
    ]


def _log_range(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("store", "attend", "logprobs"))
    if op == "logprobs":
        rows = _log_range(rng, 1, 1500)
        vocab = _log_range(rng, 500, min(262208, 300_000_000 // rows))
        return {k: v for k, v in _logprobs("", rows, vocab, rng.choice((0, 1, 3, 5, 10, 20)),
                                           rng.choice(("f32", "f32", "bf16")),
                                           rng.choice((0, 0, 1, 64))).items() if k != "name"}
    dtype = rng.choice(("bf16", "bf16", "f32"))
    head_dim = rng.choice((64, 64, 128, 128, 256, 256, 80, 192))
    value_dim = rng.choice((head_dim, head_dim, head_dim, 64, 128))
    kv_heads = rng.choice((1, 2, 3, 4, 8, 16))
    if op == "store":
        prompts = rng.random() < 0.5
        seqs = _log_range(rng, 1, 16 if prompts else 200)
        most = 60_000_000 // (seqs * kv_heads * (head_dim + value_dim))
        length = _log_range(rng, 2, max(3, min(32768, most)))
        new = rng.choice((1 << 30, _log_range(rng, 2, length))) if prompts else 1
        window = rng.choice((0, 0, _log_range(rng, 16, 4096)))
        c = _store("", seqs, length, new, kv_heads, head_dim, dtype, value_dim, window)
    else:
        seqs = _log_range(rng, 1, 200)
        most = 500_000_000 // (seqs * kv_heads * (head_dim + value_dim))
        length = _log_range(rng, 1, max(2, min(131072, most)))
        window = rng.choice((0, 0, _log_range(rng, 16, 4096)))
        c = _attend("", seqs, length, kv_heads * rng.choice((1, 2, 2, 4, 5, 8, 16)), kv_heads, head_dim,
                    dtype, value_dim, window, rng.choice((0, 4)) if window else 0,
                    rng.random() < 0.3, rng.choice((0.0, 0.0, 50.0)), rng.choice((0, 0, 1, 3)))
    c.pop("name")
    return c


# ------------------------------------------------------------------------------- the inputs
def _lengths(case):
    """Lengths of the sequences after the step, 1 .. length, spread evenly; the first is the longest."""
    n, most = case["seqs"], case["length"]
    return [most] + [1 + int((most - 1) * ((i * 0.6180339887498949 + 0.37) % 1.0)) for i in range(1, n)]


def _geometry(case):
    """(rows that a sequence may use, pages of the pool, slots): a window's ring has one page more than
    the window takes, so that the page being filled never holds keys that are still seen."""
    up = lambda n: -(-n // PAGE) * PAGE  # noqa: E731
    cap = up(case["length"])
    if case["window"] and not case.get("keep_first"):
        cap = min(cap, up(case["window"]) + PAGE)
    slots = case["seqs"] + 1
    return cap, slots * (cap // PAGE) + 3, slots


def _pool(gen, pages, kv_heads, dim):
    codes = torch.empty((pages, PAGE, kv_heads, dim), dtype=torch.uint8, device=DEV).view(_F8)
    step = max(1, (1 << 28) // (PAGE * kv_heads * dim))
    for a in range(0, pages, step):
        n = min(step, pages - a)
        codes[a:a + n].copy_((torch.randn((n, PAGE, kv_heads, dim), generator=gen, device=DEV) * 100)
                             .clamp_(-448, 448))
    scale = torch.exp2(torch.randint(-8, -4, (pages, kv_heads), generator=gen, device=DEV).float())
    return codes, scale


def _rows(gen, tokens, heads, dim, dtype):
    """Rows of keys or values: magnitudes that differ by head and by token."""
    x = torch.randn((tokens, heads, dim), generator=gen, device=DEV)
    x *= torch.exp2(torch.randint(-3, 3, (1, heads, 1), generator=gen, device=DEV).float())
    x *= torch.exp2(2 * torch.rand((tokens, 1, 1), generator=gen, device=DEV) - 1)
    return x.reshape(tokens, heads * dim).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    dtype = _DT[case["dtype"]]
    s = SimpleNamespace(case=case)
    if case["op"] == "logprobs":
        R, V = case["rows"], case["vocab"]
        wide = torch.randn((R, V + case["gap"]), generator=gen, device=DEV)
        wide *= 2.5
        # some tokens stand out, as in a trained model's rows, and some are shut out
        best = torch.randint(0, V, (R, 12), generator=gen, device=DEV)
        wide.scatter_add_(1, best, 8 + 6 * torch.rand((R, 12), generator=gen, device=DEV))
        wide[1::4, 100:300] = -math.inf
        s.logits = wide.to(dtype)[:, :V]
        s.tokens = torch.randint(0, V, (R,), generator=gen, device=DEV).int()
        s.tokens[::2] = best[::2, 0].int()
        s.tokens[5::64] = -1
        return s
    kv_heads, hd, hdv = case["kv_heads"], case["head_dim"], case["value_dim"]
    lens = _lengths(case)
    B = len(lens)
    cap, pages, slots = _geometry(case)
    k_pool, k_scale = _pool(gen, pages, kv_heads, hd)
    v_pool, v_scale = _pool(gen, pages, kv_heads, hdv)
    table = torch.randperm(pages, generator=gen, device=DEV)[:slots * (cap // PAGE)]
    s.view = SimpleNamespace(k_pool=k_pool, v_pool=v_pool, k_scale=k_scale, v_scale=v_scale,
                             page_table=table.reshape(slots, cap // PAGE).int().contiguous(),
                             page=PAGE, cap=cap, window=case["window"] or None)
    order = torch.randperm(slots, generator=gen, device=DEV)[:B].int()
    i32 = dict(dtype=torch.int32, device=DEV)
    if case["op"] == "store":
        new = [min(case["new"], n) for n in lens]
        cu = [0]
        for n in new:
            cu.append(cu[-1] + n)
        T = cu[-1]
        kv = torch.cat([_rows(gen, T, kv_heads, hd, dtype), _rows(gen, T, kv_heads, hdv, dtype)], 1)
        s.k, s.v = kv[:, :kv_heads * hd], kv[:, kv_heads * hd:]
        counts = torch.tensor(new, device=DEV)
        starts = torch.tensor(lens, device=DEV) - counts
        seq = torch.repeat_interleave(torch.arange(B, device=DEV), counts)
        first = torch.tensor(cu[:-1], device=DEV)
        s.ctx = SimpleNamespace(
            batch=B, cu_seqlens=torch.tensor(cu, **i32), slots=order, lens=torch.tensor(lens, **i32),
            seq_index=seq.int(), positions=(torch.arange(T, device=DEV) - first[seq] + starts[seq]).int(),
            max_len=max(lens), max_new=max(new), mode="decode" if max(new) == 1 else "prefill")
        return s
    pad = min(case["padding"], B - 1)
    if pad:
        order[B - pad:] = -1
        lens[B - pad:] = [1] * pad
    nh = case["heads"]
    s.q = (torch.randn((B, nh * hd), generator=gen, device=DEV) * 3).to(dtype)
    s.out = torch.empty((B, nh * hdv), dtype=dtype, device=DEV)
    s.sinks = torch.randn((nh,), generator=gen, device=DEV) if case["sinks"] else None
    s.scale = 0.5 * hd ** -0.5
    s.ctx = SimpleNamespace(
        batch=B, slots=order, lens=torch.tensor(lens, **i32), max_len=max(lens), max_new=1,
        positions=torch.tensor([n - 1 for n in lens], **i32), seq_index=torch.arange(B, **i32),
        cu_seqlens=torch.arange(B + 1, **i32), mode="decode")
    return s


def work(case):
    if case["op"] == "logprobs":
        R, V = case["rows"], case["vocab"]
        esz = 4 if case["dtype"] == "f32" else 2
        return {"bytes": R * V * esz + R * (4 + 12 + 8 * case["top"]), "flops": 6.0 * R * V}
    nkv, hd, hdv = case["kv_heads"], case["head_dim"], case["value_dim"]
    esz = 4 if case["dtype"] == "f32" else 2
    lens = _lengths(case)
    cap = _geometry(case)[0]
    if case["op"] == "store":
        rows = blocks = 0
        for n in lens:
            first = max(n - min(case["new"], n), ((n - 1) // PAGE - cap // PAGE + 1) * PAGE)
            rows += n - first
            blocks += (n - 1) // PAGE - first // PAGE + 1
        return {"bytes": rows * nkv * (hd + hdv) * (esz + 1) + 8 * blocks * nkv + 4 * blocks,
                "flops": 2.0 * rows * nkv * (hd + hdv)}
    nh, seen, pages = case["heads"], 0, 0
    pad = min(case["padding"], len(lens) - 1)
    for n in lens[:len(lens) - pad]:
        lo = max(0, n - case["window"]) if case["window"] else 0
        vis = n - lo + min(case["keep_first"], lo)
        seen += vis
        pages += -(-vis // PAGE)
    return {"bytes": seen * nkv * (hd + hdv) + 8 * pages * nkv + 4 * pages +
            len(lens) * nh * (hd + hdv) * esz, "flops": 2.0 * seen * nh * (hd + hdv)}


# ------------------------------------------------------------------------------- plain forms
def _plain_store_one(x, pool, scale, view, ctx, keep, page_id, first_page, starts):
    """One of keys and values: x [T, kv heads, dim] in 32 bits."""
    pages, P, nkv, _ = pool.shape
    finite = torch.isfinite(x)
    amax = torch.where(finite, x, 0.0).abs().amax(2)                            # [T, nkv]
    # per page and head; what is not stored goes to a row of its own behind the last page
    where = torch.where(keep, page_id, pages)
    need = torch.zeros((pages + 1, nkv), device=x.device)
    need.scatter_reduce_(0, where[:, None].expand(-1, nkv), amax, "amax")
    touched = torch.zeros(pages + 1, dtype=torch.bool, device=x.device)
    touched[where] = True
    mant, expo = torch.frexp(need[:pages])
    expo = torch.where(mant <= 0.875, expo - 9, expo - 8)                       # 448 = 0.875 * 2^9
    expo = torch.where(need[:pages] > 0, expo, -126).clamp_min(-126)
    fresh = torch.ldexp(torch.ones_like(mant), expo)
    # the sequences' first pages may hold earlier tokens
    r0 = starts % P
    old = scale[first_page]                                                     # [B, nkv]
    go_on = touched[first_page] & (r0 > 0)
    new = torch.where(go_on[:, None], torch.maximum(old, fresh[first_page]), fresh[first_page])
    new = torch.where(touched[first_page][:, None], new, old)
    had = pool.view(torch.uint8)[first_page].view(_F8)                          # [B, P, nkv, dim]
    again = (had.float() * (old / new)[:, None, :, None]).to(_F8)
    change = (go_on[:, None] & (torch.arange(P, device=x.device)[None, :] < r0[:, None]))
    had = torch.where(change[:, :, None, None], again.view(torch.uint8), had.view(torch.uint8))
    pool.view(torch.uint8)[first_page] = had
    scale.copy_(torch.where(touched[:pages, None], fresh, scale))
    scale[first_page] = new
    code = torch.where(finite, x / scale[torch.where(keep, page_id, 0)][:, :, None], math.nan).to(_F8)
    at = (page_id * P + ctx.positions.long() % P)[keep]
    pool.view(torch.uint8).view(pages * P, nkv, -1)[at] = code.view(torch.uint8)[keep]


def _plain_store(s):
    v, c, ctx = s.view, s.case, s.ctx
    nkv, P, cap = c["kv_heads"], v.page, v.cap
    seq, p = ctx.seq_index.long(), ctx.positions.long()
    slots, lens = ctx.slots.long(), ctx.lens.long()
    counts = (ctx.cu_seqlens[1:] - ctx.cu_seqlens[:-1]).long()
    keep = (slots[seq] >= 0) & (p // P > (lens[seq] - 1) // P - cap // P)
    page_id = v.page_table[slots[seq].clamp_min(0), p % cap // P].long()
    starts = lens - counts
    first_page = v.page_table[slots.clamp_min(0), starts % cap // P].long()
    # (a first page that the ring has given to later positions since then holds nothing to keep)
    gone = starts // P <= (lens - 1) // P - cap // P
    starts = torch.where(gone, 0, starts)
    T = s.k.shape[0]
    _plain_store_one(s.k.float().reshape(T, nkv, -1), v.k_pool, v.k_scale, v, ctx, keep, page_id,
                     first_page, starts)
    _plain_store_one(s.v.float().reshape(T, nkv, -1), v.v_pool, v.v_scale, v, ctx, keep, page_id,
                     first_page, starts)
    return {"k": v.k_pool, "v": v.v_pool, "k_scale": v.k_scale, "v_scale": v.v_scale}


def _plain_attend(s):
    v, c, ctx = s.view, s.case, s.ctx
    nh, nkv, hd, hdv = c["heads"], c["kv_heads"], c["head_dim"], c["value_dim"]
    B, G, W, kf = s.q.shape[0], nh // nkv, c["window"], c["keep_first"]
    p, slots = ctx.positions.long(), ctx.slots.long()
    lo = (p - W + 1).clamp_min(0) if W else torch.zeros_like(p)
    base = torch.zeros_like(lo) if kf or not W else lo
    n = min(ctx.max_len, W) if W and not kf else ctx.max_len
    j = base[:, None] + torch.arange(n, device=p.device)[None, :]               # [B, n] positions
    seen = (j <= p[:, None]) & ((j >= lo[:, None]) | (j < kf))
    row = torch.where(seen, j, 0) % v.cap
    page = v.page_table[slots.clamp_min(0)].long().gather(1, row // v.page)
    k = v.k_pool.view(torch.uint8)[page, row % v.page].view(_F8).float() * v.k_scale[page][..., None]
    q = s.q.float().reshape(B, nkv, G, hd)
    x = torch.matmul(q, k.permute(0, 2, 3, 1)) * s.scale                        # [B, nkv, G, n]
    del k
    if c["softcap"]:
        x = c["softcap"] * torch.tanh(x / c["softcap"])
    x = x.masked_fill(~seen[:, None, None, :], -math.inf)
    m = x.amax(-1, keepdim=True)
    sink = 0.0
    if s.sinks is not None:
        m = torch.maximum(m, s.sinks.reshape(1, nkv, G, 1))
        sink = torch.exp(s.sinks.reshape(1, nkv, G, 1) - m)
    e = torch.exp(x - m)
    w = e / (e.sum(-1, keepdim=True) + sink)
    val = v.v_pool.view(torch.uint8)[page, row % v.page].view(_F8).float() * v.v_scale[page][..., None]
    o = torch.matmul(w, val.permute(0, 2, 1, 3)).reshape(B, nh * hdv)
    return torch.where((slots >= 0)[:, None], o, 0.0).to(s.q.dtype)


def _plain_logprobs(s):
    x, top = s.logits.float(), s.case["top"]
    V = x.shape[1]
    t = s.tokens.long()
    has = t >= 0
    m = x.amax(1, keepdim=True)
    d = x - m
    e = torch.exp(d)
    total = e.sum(1, keepdim=True)
    log_total = torch.log(total)
    entropy = (log_total - torch.where(e > 0, e * d, 0.0).sum(1, keepdim=True) / total)[:, 0]
    mine = x.gather(1, t.clamp_min(0)[:, None])
    logprob = torch.where(has, (mine - m - log_total)[:, 0], math.nan)
    index = torch.arange(V, device=x.device)
    ahead = (x > mine) | ((x == mine) & (index[None, :] < t[:, None]))
    rank = torch.where(has, ahead.sum(1) + 1, 0).int()
    out = {"logprob": logprob, "entropy": entropy, "rank": rank}
    if top:
        # whole numbers in the order of (value, lower index first)
        bits = (x + 0.0).view(torch.int32).long()
        key = torch.where(bits < 0, -(bits & 0x7fffffff), bits) * (1 << 32) + (V - 1 - index)[None, :]
        ids = V - 1 - (torch.topk(key, top, dim=1).values & 0xffffffff)
        out["top_ids"] = ids.int()
        out["top_logprobs"] = x.gather(1, ids) - m - log_total
    return out


# ------------------------------------------------------------------------------- one pass
def run(s):
    c = s.case
    if not own:
        return {"store": _plain_store, "attend": _plain_attend, "logprobs": _plain_logprobs}[c["op"]](s)
    from agave_b200 import kernels
    if c["op"] == "store":
        kernels.cache_store_e4m3(s.k, s.v, s.view, s.ctx, c["kv_heads"], c["head_dim"],
                                 value_dim=c["value_dim"])
        return {"k": s.view.k_pool, "v": s.view.v_pool, "k_scale": s.view.k_scale,
                "v_scale": s.view.v_scale}
    if c["op"] == "attend":
        kernels.attention_decode_e4m3(s.q, s.out, s.view, s.ctx, c["heads"], c["kv_heads"],
                                      c["head_dim"], s.scale, c["window"], value_dim=c["value_dim"],
                                      sinks=s.sinks, keep_first=c["keep_first"], softcap=c["softcap"])
        return s.out
    r = kernels.token_logprobs(s.logits, s.tokens, top=c["top"])
    out = {"logprob": r.logprob, "entropy": r.entropy, "rank": r.rank}
    if c["top"]:
        out["top_ids"], out["top_logprobs"] = r.top_ids, r.top_logprobs
    return out


# ------------------------------------------------------------------------------- in 64 bits
def _exact_codes(x, scale):
    """x / scale on the grid of e4m3 (steps of 2^(floor log2 - 3), of 2^-9 below 2^-6), in 64 bits."""
    y = x / scale
    _, e = torch.frexp(y)
    step = torch.ldexp(torch.ones_like(y), (e - 1).clamp_min(-6) - 3)
    return torch.where(torch.isfinite(y), torch.round(y / step) * step, math.nan)


def _exact_store(s):
    v, c, ctx = s.view, s.case, s.ctx
    nkv, P, cap = c["kv_heads"], v.page, v.cap
    cu, lens, slots = ctx.cu_seqlens.tolist(), ctx.lens.tolist(), ctx.slots.tolist()
    table = v.page_table.tolist()
    out = {}
    for name, x, pool, scale in (("k", s.k, v.k_pool, v.k_scale), ("v", s.v, v.v_pool, v.v_scale)):
        codes, scales = pool.double(), scale.double()
        for b, n in enumerate(lens):
            new = cu[b + 1] - cu[b]
            start = n - new
            j_last = (n - 1) // P
            for j in range(max(start // P, j_last - cap // P + 1), j_last + 1):
                a, z = max(start, j * P), min(n, (j + 1) * P)
                rows = x[cu[b] + a - start:cu[b] + z - start].double().reshape(z - a, nkv, -1)
                page = table[slots[b]][j * P % cap // P]
                amax = rows.abs().amax((0, 2))
                need = torch.exp2(torch.ceil(torch.log2(amax / 448)).clamp_min(-126))
                # (the logarithm may land beside a whole number)
                need = torch.where((need * 224 >= amax) & (need > 2.0 ** -126), need / 2, need)
                need = torch.where(need * 448 < amax, need * 2, need)
                if a > j * P:
                    need = torch.maximum(need, scales[page])
                    old = codes[page, :a - j * P]
                    codes[page, :a - j * P] = _exact_codes(old * scales[page][None, :, None],
                                                           need[None, :, None])
                scales[page] = need
                codes[page, a - j * P:z - j * P] = _exact_codes(rows, need[None, :, None])
        out[name], out[name + "_scale"] = codes, scales
    return out


def _exact_attend(s):
    v, c, ctx = s.view, s.case, s.ctx
    nh, nkv, hd, hdv = c["heads"], c["kv_heads"], c["head_dim"], c["value_dim"]
    out = torch.zeros((s.q.shape[0], nh, hdv), dtype=torch.float64, device=DEV)
    for b, (slot, p) in enumerate(zip(ctx.slots.tolist(), ctx.positions.tolist())):
        if slot < 0:
            continue
        lo = max(0, p - c["window"] + 1) if c["window"] else 0
        j = torch.arange(lo, p + 1, device=DEV)
        j = torch.cat([torch.arange(min(c["keep_first"], lo), device=DEV), j])
        page = v.page_table[slot].long()[j % v.cap // v.page]
        for g in range(nkv):
            k, val = (pool.view(torch.uint8)[page, j % v.page, g].view(_F8).double() *
                      scale[page, g].double()[:, None]
                      for pool, scale in ((v.k_pool, v.k_scale), (v.v_pool, v.v_scale)))
            heads = slice(g * (nh // nkv), (g + 1) * (nh // nkv))
            x = s.q[b].double().reshape(nh, hd)[heads] @ k.T * s.scale
            if c["softcap"]:
                x = c["softcap"] * torch.tanh(x / c["softcap"])
            if s.sinks is not None:
                x = torch.cat([x, s.sinks[heads].double()[:, None]], 1)
                val = torch.cat([val, torch.zeros_like(val[:1])])
            out[b, heads] = torch.softmax(x, 1) @ val
    return out.reshape(s.q.shape[0], nh * hdv)


def _exact_logprobs(s):
    R, top = s.logits.shape[0], s.case["top"]
    parts = []
    for a in range(0, R, 256):
        x, t = s.logits[a:a + 256].double(), s.tokens[a:a + 256].long()
        lp = torch.log_softmax(x, 1)
        mine = lp.gather(1, t.clamp_min(0)[:, None])[:, 0]
        parts.append((torch.where(t >= 0, mine, math.nan),
                      -torch.where(lp > -math.inf, lp.exp() * lp, 0.0).sum(1),
                      torch.topk(lp, top, dim=1).values if top else mine[:0]))
    out = {"logprob": torch.cat([p[0] for p in parts]), "entropy": torch.cat([p[1] for p in parts]),
           "rank": None}
    if top:
        out["top_ids"] = None
        out["top_logprobs"] = torch.cat([p[2] for p in parts])
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"store": _exact_store, "attend": _exact_attend, "logprobs": _exact_logprobs}[case["op"]](s)
