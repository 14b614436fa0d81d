"""Decode attention over 8-bit codes under a bias by distance that masks: the type's lowest value, -inf and
values near the lowest, for some keys and for all of them."""
import math

import pytest
import torch

from test_e4m3_cache_gpu import BF, DEV, F32, make_ctx, make_view, rnd

pytestmark = pytest.mark.gpu

LOWEST = torch.finfo(torch.float32).min


def setup(dtype, rows):
    nh, nkv, hd = 4, 2, 64
    view = make_view(2, 512, nkv, hd, hd, seed=31)
    q = rnd(1, nh * hd, dtype=dtype, seed=32, scale=2.0).repeat(rows, 1)
    return view, q, make_ctx([1] * rows, [400] * rows, [1] * rows), nh, nkv, hd


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows", [1, 400])
@pytest.mark.parametrize("value", [LOWEST, 0.9 * LOWEST, 0.6 * LOWEST])
@pytest.mark.parametrize("most", [400, 1 << 20])
def test_every_key_has_the_lowest_bias(dtype, rows, value, most):
    """The scores vanish in such a bias: all keys weigh the same, as in the formula.  (Sums and weights
    then are exact but for (n + 16) 2^-24 and the result's rounding.)"""
    from agave_b200 import kernels
    view, q, ctx, nh, nkv, hd = setup(dtype, rows)
    ctx.max_len = most
    out = torch.full((rows, nh * hd), math.nan, dtype=dtype, device=DEV)
    bias = torch.full((nh, 1), value, device=DEV)
    kernels.attention_decode_e4m3(q, out, view, ctx, nh, nkv, hd, hd ** -0.5, 0, dist_bias=bias)
    pg = view.page_table[1].long()[torch.arange(400, device=DEV) // 64]
    at = torch.arange(400, device=DEV) % 64
    v = view.v_pool.float()[pg, at].double() * view.v_scale[pg].double()[:, :, None]
    ref = v.mean(0).repeat_interleave(nh // nkv, 0)
    top = v.abs().amax(0).repeat_interleave(nh // nkv, 0)
    tol = 416 * 2.0 ** -24 * top + (2.0 ** -8 if dtype == BF else 2.0 ** -24) * ref.abs()
    assert ((out.double().reshape(rows, nh, hd) - ref).abs() <= tol).all()
    # a sink that is no mask takes all of the weight
    kernels.attention_decode_e4m3(q, out, view, ctx, nh, nkv, hd, hd ** -0.5, 0, dist_bias=bias,
                                  sinks=torch.zeros(nh, device=DEV))
    assert (out == 0).all()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows", [1, 400])
@pytest.mark.parametrize("value", [LOWEST, -math.inf])
@pytest.mark.parametrize("span", [(0, 100), (100, 400), (1, 400), (37, 230)])
def test_some_keys_are_masked_by_their_bias(dtype, rows, value, span):
    """Keys at these distances have no weight, whatever their values are."""
    from agave_b200 import kernels
    view, q, ctx, nh, nkv, hd = setup(dtype, rows)
    bias = rnd(nh, 400, seed=33)
    masked = bias.clone()
    masked[:, span[0]:span[1]] = value
    bias[:, span[0]:span[1]] = -5000.0                        # e^-5000 is 0, too
    a = torch.full((rows, nh * hd), math.nan, dtype=dtype, device=DEV)
    b = a.clone()
    kernels.attention_decode_e4m3(q, a, view, ctx, nh, nkv, hd, hd ** -0.5, 0, dist_bias=masked)
    kernels.attention_decode_e4m3(q, b, view, ctx, nh, nkv, hd, hd ** -0.5, 0, dist_bias=bias)
    assert torch.equal(a, b) and torch.isfinite(a).all()


def test_every_key_masked_by_minus_infinity():
    """No key is seen: zeros."""
    from agave_b200 import kernels
    for dtype in (BF, F32):
        for rows in (1, 400):
            view, q, ctx, nh, nkv, hd = setup(dtype, rows)
            for most in (400, 1 << 20):
                ctx.max_len = most
                out = torch.full((rows, nh * hd), math.nan, dtype=dtype, device=DEV)
                kernels.attention_decode_e4m3(q, out, view, ctx, nh, nkv, hd, hd ** -0.5, 0,
                                              dist_bias=torch.full((nh, 3), -math.inf, device=DEV))
                assert (out == 0).all()


def test_the_same_call_gives_the_same_bits():
    """Rows of one CTA, of clusters and of stretches that a second kernel joins."""
    from agave_b200 import kernels
    for dtype in (BF, F32):
        for lens, nh, nkv, hd in (([700], 4, 1, 256), ([20011], 8, 4, 256), ([1 + 131 * i for i in range(40)], 8, 4, 128),
                                  ([300] * 200, 6, 3, 64)):
            view = make_view(len(lens), (max(lens) + 63) // 64 * 64, nkv, hd, hd, seed=34)
            ctx = make_ctx([1] * len(lens), lens, list(range(len(lens))))
            q = rnd(len(lens), nh * hd, dtype=dtype, seed=35, scale=3.0)
            first = None
            for _ in range(20):
                out = torch.full_like(q, math.nan)
                kernels.attention_decode_e4m3(q, out, view, ctx, nh, nkv, hd, 0.5 * hd ** -0.5, 0)
                first = out if first is None else first
                assert torch.equal(first, out)


def test_a_bias_of_no_distances_is_refused():
    """It has no address: taken as none, it would be left out without a word."""
    from agave_b200 import kernels
    view, q, ctx, nh, nkv, hd = setup(F32, 1)
    for shape in ((nh, 0), (nh + 1, 3), (3,)):
        with pytest.raises(kernels.KernelError, match="bias by distance"):
            kernels.attention_decode_e4m3(q, torch.empty_like(q), view, ctx, nh, nkv, hd, 1.0, 0,
                                          dist_bias=torch.zeros(shape, device=DEV))
