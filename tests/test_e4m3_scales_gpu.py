"""Decode attention over 8-bit codes whose pages' scales lie anywhere in the store's range, 2^-126 to
2^120, against the formula in 64 bits: a page's scale counts with the weight that its keys have."""
import math

import pytest
import torch

from plain import e4m3_plain as P
from test_e4m3_cache_gpu import BF, DEV, F32, make_ctx, make_view, rnd

pytestmark = pytest.mark.gpu

N = 512                                 # keys: eight pages


def want(view, q, nh, scale, window=0, bias=None, softcap=0.0, sinks=None):
    """(out [nh, hdv], tolerance) of the query at position N - 1 of slot 1.

    A score is off by d_j = (2^-21 + (hd + 8) 2^-24) scale sum |q||k_j| (the query as two 11-bit halves,
    products summed in 32 bits) + 2^-21 (1 + |s_j| + |m|) (the exponential and its argument); its weight
    and its part of the normaliser by a factor of e^d_j.  Both sums add (n + 16) 2^-24 of their terms,
    bfloat16 queries 2^-11 of a weight.  A weight times its scale is held in half floats against the greatest such
    product G, times 2^14: below 2^-14 it is off by up to 2^-25, that is 2^-39 G, times a code of 448 < 2^9.
    The result is rounded by 2^-8 (bfloat16) or 2^-24.  Numbers below 2^-126 are off by 2^-150 a rounding:
    two for each of four warps (its two factors), two for each of up to 16 parts of a row, one at the end,
    that is 41 * 2^-150 < 2^-144 (their sums round nothing there)."""
    hd = q.shape[1] // nh
    nkv, group = view.k_pool.shape[2], nh // view.k_pool.shape[2]
    j = torch.tensor(P.visible(N - 1, window, 0), device=DEV)
    pg = view.page_table[1].long()[j // view.page]
    k = view.k_pool.float()[pg, j % view.page].double() * view.k_scale[pg].double()[:, :, None]
    code, vs = view.v_pool.float()[pg, j % view.page].double(), view.v_scale[pg].double()
    bf, n = q.dtype == BF, j.numel()
    out, tol = [], []
    for h in range(nh):
        g = h // group
        x = q[0].double().reshape(nh, hd)[h]
        s, mag = k[:, g] @ x * scale, k[:, g].abs() @ x.abs() * abs(scale)
        if softcap:
            s, mag = softcap * torch.tanh(s / softcap), mag + softcap
        if bias is not None:
            s = s + bias[h].double()[(N - 1 - j).clamp_max(bias.shape[1] - 1)]
        m = s.max() if sinks is None else torch.maximum(s.max(), sinks[h].double())
        w = torch.exp(s - m)
        w = w / (w.sum() + (0 if sinks is None else torch.exp(sinks[h].double() - m)))
        d = (2.0 ** -21 + (hd + 8) * 2.0 ** -24) * mag + 2.0 ** -21 * (1 + s.abs() + m.abs())
        e = torch.expm1(d) + (n + 16) * 2.0 ** -24
        v = code[:, g] * vs[:, g, None]
        o = w @ v
        t = (w * (e + (2.0 ** -11 if bf else 0))) @ v.abs() + (w @ v.abs()) * (w @ e)
        t += n * 2.0 ** -30 * (w * vs[:, g]).max() + (2.0 ** -8 if bf else 2.0 ** -24) * o.abs() + 2.0 ** -144
        out.append(o)
        tol.append(t)
    return torch.stack(out), torch.stack(tol)


def check(view, q, nh, nkv, hd, hdv, rows=1, lens=(N, 1 << 20), window=0, **opt):
    """The same query in every row, by the plan for few keys and by that for many."""
    from agave_b200 import kernels
    scale = opt.pop("scale", hd ** -0.5)
    ref, tol = want(view, q, nh, scale, window, opt.get("dist_bias"), opt.get("softcap", 0.0), opt.get("sinks"))
    ctx = make_ctx([1] * rows, [N] * rows, [1] * rows)
    for most in lens:
        ctx.max_len = most
        out = torch.full((rows, nh * hdv), math.nan, dtype=q.dtype, device=DEV)
        kernels.attention_decode_e4m3(q.repeat(rows, 1), out, view, ctx, nh, nkv, hd, scale, window,
                                      value_dim=hdv, **opt)
        got = out.double().reshape(rows, nh, hdv)
        bad = ~((got - ref).abs() <= tol)
        assert not bad.any(), (most, int(bad.sum()), float((got - ref).abs().max()), float(tol.max()))


def far(at, value, nh):
    """A bias by distance of ``value`` for the keys of page ``at`` and 0 for the others."""
    bias = torch.zeros(nh, N, device=DEV)
    bias[:, N - 1 - (at * 64 + 63):N - at * 64] = value
    return bias


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("hd,hdv", [(64, 64), (128, 80), (64, 256)])
@pytest.mark.parametrize("rows", [1, 400])
@pytest.mark.parametrize("shift", [30, 60, 110, -115])
def test_a_page_with_a_scale_far_from_the_others(dtype, hd, hdv, rows, shift):
    """The first, a middle or the last page, with all, hardly any or no weight."""
    nh, nkv = 4, 2
    view = make_view(2, N, nkv, hd, hdv, seed=21)
    q = rnd(1, nh * hd, dtype=dtype, seed=22, scale=2.0)
    for at in (0, 3, 7):
        view.v_scale.fill_(2.0 ** -7)
        view.v_scale[view.page_table[1, at].long()] *= 2.0 ** shift
        for value in (-2000.0, -60.0, -20.0, 60.0):
            check(view, q, nh, nkv, hd, hdv, rows, dist_bias=far(at, value, nh))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("window", [200, -320, 100])
def test_large_rows_before_a_window(dtype, window):
    """The page in which the window begins has its scale from rows that are not seen."""
    nh, nkv, hd = 2, 1, 64
    view = make_view(2, N, nkv, hd, hd, seed=23)
    first = min(P.visible(N - 1, window, 0))
    view.v_scale.fill_(2.0 ** -7)
    page = int(view.page_table[1, first // 64])
    view.v_scale[page] = 2.0 ** 100
    view.v_pool.view(torch.uint8)[page, first % 64:] = 0              # what is seen is too small for its scale
    q = rnd(1, nh * hd, dtype=dtype, seed=24, scale=2.0)
    for rows in (1, 400):
        check(view, q, nh, nkv, hd, hd, rows, window=window)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("exponent", [-126, -100, 100, 117])
def test_scales_at_the_ends_of_the_range(dtype, exponent):
    """All pages alike: the sum of the values of 512 keys would leave 32 bits, their mean does not."""
    nh, nkv, hd = 2, 1, 128
    view = make_view(2, N, nkv, hd, hd, seed=25)
    view.v_scale.fill_(2.0 ** exponent)
    same = view.v_pool.view(torch.uint8)
    same.copy_((torch.full(same.shape, 448.0) * (1 - 2 * (torch.arange(hd) % 2))).to(P.F8).view(torch.uint8))
    q = rnd(1, nh * hd, dtype=dtype, seed=26, scale=2.0)
    for rows in (1, 400):
        check(view, q, nh, nkv, hd, hd, rows)
        check(view, q * 2.0 ** -40, nh, nkv, hd, hd, rows)            # equal weights


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("opt", [dict(), dict(softcap=20.0), dict(sinks=2.0), dict(sinks=300.0), dict(sinks=-300.0)])
def test_every_page_with_a_scale_of_its_own(dtype, opt):
    nh, nkv, hd, hdv = 20, 2, 64, 48
    view = make_view(2, N, nkv, hd, hdv, seed=27)
    g = torch.Generator(device="cpu").manual_seed(28)
    q = rnd(1, nh * hd, dtype=dtype, seed=29, scale=8.0)
    opt = dict(opt)
    if "sinks" in opt:
        opt["sinks"] = torch.full((nh,), opt["sinks"], device=DEV)
    for spread in (10, 40, 110):
        e = torch.randint(-spread, spread + 1, tuple(view.v_scale.shape), generator=g)
        view.v_scale.copy_(torch.exp2(e.float()))
        for rows in (1, 400):
            check(view, q, nh, nkv, hd, hdv, rows, **opt)
