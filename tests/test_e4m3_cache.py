"""What the 8-bit cache decides on the host: groups, rings, refusals of the C functions (which come
before anything touches a device)."""
import ctypes

import pytest
import torch

from plain import e4m3_plain as P


def test_plain_codes_are_the_conversion_torch_has():
    g = torch.Generator().manual_seed(0)
    y = torch.cat([torch.randn(20000, generator=g) * 60, torch.randn(20000, generator=g) * 2.0 ** -7,
                   torch.arange(-448, 449).float() / 2, torch.tensor([0.0, 448.0, -448.0, 2.0 ** -10, 3 * 2.0 ** -10])])
    y = y.clamp(-448, 448)
    assert torch.equal(P.round_codes(y.double()).float(), y.to(P.F8).float())
    a = torch.tensor([0.0, 448.0, 448.1, 449.0, 3.5, 1.75, 1.7500001, 1e-45, 3e38], dtype=torch.float64)
    assert P.scale_of(a).log2().tolist() == [-126, 0, 1, 1, -7, -8, -7, -126, 120]


def test_groups_of_codes():
    from agave_b200.cache import CacheError, plan_groups
    from agave_b200.parts.base import KVRequest
    reqs = [KVRequest(2, 64, eight_bit=True), KVRequest(2, 64, 100, eight_bit=True),
            KVRequest(1, 96, value_dim=64, values_in_keys=True), None, KVRequest(2, 64, 900, eight_bit=True)]
    groups, where = plan_groups(reqs, 4096, 1024, 4, codes=True)
    # a window's ring has a page more than the window takes; one that would not be shorter is none
    assert [(g.window, g.cap, g.codes) for g in groups] == [(None, 1024, True), (100, 192, True), (None, 1024, False)]
    assert where[0] == (0, 0) and where[4] == (0, 1)
    plain, _ = plan_groups(reqs, 4096, 1024, 4)
    assert [(g.window, g.cap, g.codes) for g in plain] == [(None, 1024, False), (100, 128, False),
                                                           (None, 1024, False), (900, 960, False)]
    with pytest.raises(CacheError, match="8 bits"):
        plan_groups([KVRequest(2, 40)], 4096, 1024, 4, codes=True)


def test_cache_on_the_host():
    from agave_b200.cache import Cache, CacheError
    from agave_b200.parts.base import KVRequest
    reqs = [KVRequest(2, 64, 100, value_dim=32, eight_bit=True), KVRequest(1, 96, value_dim=64, values_in_keys=True)]
    c = Cache(reqs, 512, 256, 3, torch.bfloat16, torch.device("cpu"), kv_dtype=P.F8)
    v, latent = c.kv_view(0), c.kv_view(1)
    pages = v.k_pool.shape[0]
    assert v.k_pool.dtype == P.F8 and v.k_pool.shape == (pages, 64, 2, 64) and v.v_pool.shape == (pages, 64, 2, 32)
    assert v.k_scale.shape == v.v_scale.shape == (pages, 2) and v.k_scale.dtype == torch.float32
    assert latent.k_scale is None and latent.k_pool.dtype == torch.bfloat16
    with pytest.raises(CacheError, match="no layer"):
        Cache(reqs[1:], 512, 256, 3, torch.bfloat16, torch.device("cpu"), kv_dtype=P.F8)
    with pytest.raises(CacheError, match="float16"):
        Cache(reqs, 512, 256, 3, torch.bfloat16, torch.device("cpu"), kv_dtype=torch.float16)


@pytest.fixture(scope="module")
def lib():
    from agave_b200 import kernels
    return kernels.library()


def test_store_refuses(lib):
    z = ctypes.c_void_p(0)

    def call(B=1, T=1, nkv=1, hd=64, hdv=64, dtype=0, page=64, cap=128, max_pages=2, n_pages=4, pool=0, n_slots=1):
        ll = ctypes.c_longlong
        rc = lib.agv_cache_store_e4m3(z, ll(64), z, ll(64), dtype, z, z, z, B, T, 1, nkv, hd, hdv,
                                      ctypes.c_void_p(pool), z, z, z, z, n_slots, max_pages, page, cap, n_pages, z)
        return rc, lib.agv_last_error().decode()
    assert call(B=0)[0] == 0 and call(T=0)[0] == 0
    for kw, word in ((dict(hd=24), "multiples of 16"), (dict(hdv=0), "multiples of 16"), (dict(cap=100), "geometry"),
                     (dict(cap=192), "geometry"), (dict(dtype=2), "dtype"), (dict(pool=8), "unaligned"),
                     (dict(B=70000), "grid"), (dict(page=48, cap=96), "geometry"), (dict(nkv=0), "bad sizes"), (dict(n_slots=0), "bad sizes")):
        rc, msg = call(**kw)
        assert rc < 0 and word in msg, (kw, msg)


def test_attention_refuses(lib):
    z = ctypes.c_void_p(0)
    f = ctypes.c_float

    def call(B=1, nh=4, nkv=2, hd=64, hdv=64, dtype=0, page=64, cap=128, max_pages=2, pool=0, keep_first=0, cap_s=0.0,
             bias=0, n_dist=0):
        ll = ctypes.c_longlong
        rc = lib.agv_attention_decode_e4m3(z, ll(256), z, dtype, ctypes.c_void_p(pool), z, z, z, z, 1, max_pages, page,
                                           cap, 4, z, z, B, nh, nkv, hd, hdv, f(1.0), 0, keep_first, z,
                                           ctypes.c_void_p(bias), n_dist, f(cap_s), 1, z, ll(0), z)
        return rc, lib.agv_last_error().decode()
    assert call(B=0)[0] == 0
    # scratch: none for no sequences or few keys, refused for heads that form no groups
    for keys in (1, 1024, 1 << 20):
        assert lib.agv_attention_decode_e4m3_scratch(0, 4, 2, 64, 64, keys) >= 0
    for B, nh, nkv, hd in ((1, 1, 1, 16), (1, 128, 128, 256), (3, 40, 2, 64), (2000, 16, 16, 128)):
        assert lib.agv_attention_decode_e4m3_scratch(B, nh, nkv, hd, hd, 1024) == 0
    for keys in (1 << 20, (1 << 31) - 1):
        assert lib.agv_attention_decode_e4m3_scratch(1, 4, 4, 64, 64, keys) > 0
    for nh, nkv in ((5, 2), (4, 0), (0, 1)):
        assert lib.agv_attention_decode_e4m3_scratch(1, nh, nkv, 64, 64, 4096) < 0
    for kw, word in ((dict(hd=272), "multiples of 16"), (dict(hdv=8), "multiples of 16"), (dict(cap=192), "geometry"),
                     (dict(page=24, cap=48), "geometry"), (dict(dtype=7), "dtype"), (dict(pool=8), "unaligned"),
                     (dict(nh=5), "query heads"), (dict(keep_first=-1), "options"), (dict(cap_s=-1.0), "options"),
                     (dict(bias=16), "options")):
        rc, msg = call(**kw)
        assert rc < 0 and word in msg, (kw, msg)


def test_logprobs_refuses(lib):
    z = ctypes.c_void_p(0)

    def call(R=1, V=100, ld=100, dtype=0, top=0):
        rc = lib.agv_token_logprobs(z, ctypes.c_longlong(ld), dtype, R, V, z, top, z, z, z, z, z, z)
        return rc, lib.agv_last_error().decode()
    assert call(R=0)[0] == 0
    for kw, word in ((dict(V=0), "bad sizes"), (dict(R=2, ld=99), "bad sizes"), (dict(top=33), "top"),
                     (dict(top=4, V=3), "top"), (dict(top=-1), "top"), (dict(dtype=2), "dtype")):
        rc, msg = call(**kw)
        assert rc < 0 and word in msg, (kw, msg)


def test_command_line_options():
    from agave_b200.cli import _holds_codes, _unsupported, build_parser, main
    p = build_parser()
    for argv, codes in (([], False), (["--kv-type", "bf16"], False), (["--kv-type", "e4m3"], True),
                        (["--kv-type", "FP8"], True), (["--kv-type-k", "f8", "--kv-type-v", "e4m3"], True),
                        (["--cache-type-k", "fp8", "--cache-type-v", "fp8"], True),
                        (["--kv-type", "fp8", "--kv-type-k", "fp8"], True)):
        args = p.parse_args(["m"] + argv)
        assert _unsupported(args) is None and _holds_codes(args) is codes, argv
    for argv in (["--kv-type", "e4m3", "--kv-type-v", "bf16"], ["--kv-type-k", "e4m3"], ["--kv-type-v", "e4m3"],
                 ["--kv-type-k", "e4m3", "--kv-type-v", "bf16"], ["--kv-type", "bf16", "--kv-type-k", "fp8"],
                 ["--kv-type", "q4_0"], ["--kv-type", "turbo4"]):
        assert _unsupported(p.parse_args(["m"] + argv)) is not None, argv
    assert main(["/tmp", "--tokens", "1", "--logprobs", "33"]) == 1
