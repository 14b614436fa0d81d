"""The engine with its cache in 8 bits, and its log-probabilities: every store and every decode
attention of a run against the plain 64-bit forms, for every architecture that can hold its cache so;
``generate(logprobs=...)`` and ``score`` against the plain implementation."""
import importlib
import json
import math
import subprocess
import sys
from types import SimpleNamespace

import pytest
import torch

import test_e4m3_cache_gpu as T
from util import ROOT, TINY, TOL, model_folder, plain_logits, random_tokens

pytestmark = pytest.mark.gpu

DTYPES = ["float32", "bfloat16"]
STORE = {"float32": torch.float32, "bfloat16": torch.bfloat16}


def folder_of(family, name, dtype):
    if family == "gemma3":
        return model_folder(name, STORE[dtype]), TINY[name][0]["vocab_size"]
    util = importlib.import_module(f"{family}_util")
    return util.folder_for(name, STORE[dtype]), util.CONFIGS[name]["vocab"]


def engine(folder, dtype, **kw):
    from agave_b200.engine.api import Engine
    return Engine(folder, dtype=dtype, **{"max_tokens": 4096, **kw})


FAMILIES = [("gemma3", "A"), ("gemma3", "B"), ("gemma3", "C"), ("ramilorn", "R1"), ("ramilorn", "R2"),
            ("ramilorn", "R3"), ("zazerax", "Z2"), ("bovozen", "V2"), ("kadavik", "K2"), ("kadavik", "K5"),
            ("savovik", "S2"), ("pubunex", "P2"), ("pubunex", "P5")]
# head sizes that are no multiples of 16
REFUSED = [("ramilorn", "R4"), ("zazerax", "Z1"), ("bovozen", "V1"), ("kadavik", "K4"), ("savovik", "S3"),
           ("pubunex", "P3")]


@pytest.mark.parametrize("family,name", REFUSED)
def test_head_sizes_that_codes_are_not_for(family, name):
    from agave_b200.cache import CacheError
    with pytest.raises(CacheError, match="8 bits"):
        engine(folder_of(family, name, "float32")[0], "float32", cache_dtype="e4m3")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("family,name", FAMILIES)
def test_every_store_and_attention_of_a_run(family, name, dtype, monkeypatch):
    from agave_b200 import kernels
    folder, vocab = folder_of(family, name, dtype)
    eng = engine(folder, dtype, cache_dtype="e4m3", use_graphs=False)
    store, attend = kernels.cache_store_e4m3, kernels.attention_decode_e4m3
    seen = {"store": 0, "attend": 0}

    def checked_store(k, v, view, ctx, nkv, hd, value_dim=0):
        seen["store"] += 1
        with monkeypatch.context() as m:
            m.setattr(kernels, "cache_store_e4m3", store)
            c = SimpleNamespace(**{n: getattr(ctx, n) for n in ("cu_seqlens", "slots", "lens", "max_new")},
                                cu=ctx.cu_seqlens.tolist())
            T.check_store(view, c, k, v, nkv, hd, value_dim or hd)

    def checked_attend(q, out, view, ctx, nh, nkv, hd, scale, window, value_dim=0, op="", **opt):
        seen["attend"] += 1
        with monkeypatch.context() as m:
            m.setattr(kernels, "attention_decode_e4m3", attend)
            T.check_attend(view, q, ctx, nh, nkv, hd, value_dim or hd, scale, window, out=out, **opt)
    monkeypatch.setattr(kernels, "cache_store_e4m3", checked_store)
    monkeypatch.setattr(kernels, "attention_decode_e4m3", checked_attend)
    slots = [eng.acquire() for _ in range(3)]
    prompts = [random_tokens(n, vocab, 7 + n) for n in (70, 1, 29)]
    eng.step([(s, p) for s, p in zip(slots, prompts)], [[len(p) - 1] for p in prompts])
    for i in range(8):
        eng.step([(s, [t]) for s, t in zip(slots, random_tokens(3, vocab, 50 + i))], [[0]] * 3)
    assert seen["store"] >= 9 and seen["attend"] >= 8
    assert eng.runner.cache.bytes_held() > 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name", ["A", "B", "C"])
def test_prompt_logits_and_cache_size(name, dtype):
    """A prompt attends from its own keys and values, so the 8-bit cache leaves its logits alone; the
    pools take half (a quarter) of the bytes, beside the rings' extra page and the scales."""
    folder, vocab = folder_of("gemma3", name, dtype)
    a, b = engine(folder, dtype), engine(folder, dtype, cache_dtype="fp8")
    toks = random_tokens(90, vocab, 3)
    got = []
    for eng in (a, b):
        s = eng.acquire()
        got.append(eng.step([(s, toks)], [list(range(90))]))
        eng.release(s)
    T_ = TOL[dtype]
    assert float((got[0] - got[1]).abs().max()) <= T_ * float(got[0].abs().max())
    full = [sum(p.numel() * p.element_size() for p in e.runner.cache.k_pools) for e in (a, b)]
    rows = [sum(p.numel() for p in e.runner.cache.k_pools) for e in (a, b)]
    assert full[1] * (4 if dtype == "float32" else 2) == full[0] * rows[1] // rows[0]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name", ["A", "C"])
def test_generation_recorded_and_launch_by_launch(name, dtype):
    """The same tokens from recorded steps as launch by launch, whatever runs beside; slots and pages
    are used again by later batches."""
    folder, vocab = folder_of("gemma3", name, dtype)
    outs = []
    for graphs in (True, False):
        eng = engine(folder, dtype, cache_dtype="e4m3", use_graphs=graphs, max_batch=3, max_tokens=768)
        prompts = [random_tokens(n, vocab, n) for n in (5, 64, 130, 1, 63, 65)]
        outs.append(eng.generate(prompts, max_new_tokens=70, stop_token_ids=[]))
        assert [len(o) for o in outs[-1]] == [70] * 6
    assert outs[0] == outs[1]


def test_cache_dtype_names():
    folder, _ = folder_of("gemma3", "A", "float32")
    from agave_b200.engine.api import cache_dtype_of
    assert cache_dtype_of(None, torch.bfloat16) is None and cache_dtype_of("bf16", torch.bfloat16) is None
    with pytest.raises(ValueError, match="cache_dtype"):
        engine(folder, "float32", cache_dtype="bf16")
    with pytest.raises(ValueError, match="cache_dtype"):
        engine(folder, "float32", cache_dtype="int8")


# ------------------------------------------------------------------------- log-probabilities
def ref_logprobs(folder, seq):
    return torch.log_softmax(plain_logits(folder, seq).double(), 1)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("options", [dict(), dict(temperature=0.8, seed=5, top_k=20),
                                     dict(repeat_penalty=1.3), dict(temperature=1.1, seed=3, repeat_penalty=0.8)])
def test_logprobs_of_generated_tokens(dtype, options):
    """One record for each token returned, of the logits before penalty and temperature."""
    folder, vocab = folder_of("gemma3", "B", dtype)
    eng = engine(folder, dtype, max_batch=2)
    prompts = [random_tokens(n, vocab, n) for n in (5, 40, 17)]
    plain = eng.generate(prompts, max_new_tokens=12, **options)
    assert eng.logprobs is None
    outs = eng.generate(prompts, max_new_tokens=12, logprobs=4, **options)
    assert outs == plain                                  # asking changes nothing
    for p, o, scores in zip(prompts, outs, eng.logprobs):
        assert [s.token for s in scores] == o
        ref = ref_logprobs(folder, p + o)
        # (two log-probabilities of logits that are off by TOL of the greatest magnitude each)
        tol = 2 * TOL[dtype] * float(plain_logits(folder, p + o).abs().max())
        for k, s in enumerate(scores):
            row = ref[len(p) - 1 + k]
            assert abs(s.logprob - float(row[s.token])) <= tol
            assert abs(s.entropy - float(-(row.exp() * row).sum())) <= tol * (2 + math.log(vocab))
            assert len(s.top) == 4 and [lp for _, lp in s.top] == sorted((lp for _, lp in s.top), reverse=True)
            assert abs(s.top[0][1] - float(row.max())) <= tol
            if s.rank <= 4:
                assert s.top[s.rank - 1] == (s.token, s.logprob)
            else:
                assert s.logprob <= s.top[-1][1]
            if not options:
                assert s.rank == 1
    eng.generate(prompts[:1], max_new_tokens=3, logprobs=0, **options)
    assert all(s.top == () for s in eng.logprobs[0])
    with pytest.raises(ValueError, match="logprobs"):
        eng.generate(prompts, logprobs=33)


def test_logprobs_stop_with_the_tokens():
    folder, vocab = folder_of("gemma3", "A", "float32")
    eng = engine(folder, "float32")
    prompt = random_tokens(9, vocab, 1)
    free = eng.generate([prompt], max_new_tokens=30, temperature=1.0, seed=9, stop_token_ids=[])[0]
    stop = free[11]
    first = free.index(stop)
    out = eng.generate([prompt], max_new_tokens=30, temperature=1.0, seed=9, stop_token_ids=[stop], logprobs=1)[0]
    assert out == free[:first] and len(eng.logprobs[0]) == first


@pytest.mark.parametrize("cache", [None, "e4m3"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_score(dtype, cache, monkeypatch):
    """Every token after the first, whatever the batches and the rows formed at a time are."""
    from agave_b200.engine import api
    folder, vocab = folder_of("gemma3", "C", dtype)
    seqs = [random_tokens(n, vocab, n) for n in (33, 1, 2, 90, 64)]
    eng = engine(folder, dtype, max_batch=3, cache_dtype=cache)
    whole = eng.score(seqs, top=3)
    assert eng.runner.cache.book.length == {}                # no slot stays held
    monkeypatch.setattr(api, "SCORE_LOGITS", 7 * vocab)
    parts = eng.score(seqs, top=3)
    for seq, a, b in zip(seqs, whole, parts):
        assert [s.token for s in a] == seq[1:] and [s.token for s in b] == seq[1:]
        if len(seq) < 2:
            continue
        ref = ref_logprobs(folder, seq)
        tol = 2 * TOL[dtype] * float(plain_logits(folder, seq).abs().max())
        for k, (s, t) in enumerate(zip(a, b)):
            assert abs(s.logprob - float(ref[k, seq[k + 1]])) <= tol
            assert abs(t.logprob - s.logprob) <= 2 * tol
            assert len(s.top) == 3 and abs(s.top[0][1] - float(ref[k].max())) <= tol
    with pytest.raises(ValueError, match="top"):
        eng.score(seqs, top=-1)
    with pytest.raises(ValueError, match="vocabulary"):
        eng.score([[1, vocab]])
    assert eng.runner.cache.book.length == {}
    assert eng.score([]) == []


def test_command_line():
    folder, _ = folder_of("gemma3", "A", "bfloat16")

    def run(*args):
        r = subprocess.run([sys.executable, "-m", "agave_b200", folder, *args], capture_output=True, text=True,
                           cwd=ROOT, timeout=600)
        assert r.returncode == 0, r.stderr[-2000:]
        return json.loads(r.stdout.strip().splitlines()[-1])
    rec = run("--tokens", "2,17,99,5", "-n", "6", "--json", "--logprobs", "2", "--kv-type", "e4m3")
    assert len(rec["logprobs"]) == rec["tokens"] == len(rec["output_ids"])
    assert all(s["rank"] == 1 and len(s["top"]) == 2 and s["top"][0] == [s["id"], s["logprob"]] for s in rec["logprobs"])
    rec = run("--tokens", "2,17,99,5;2,9", "--json", "--score")
    assert [r["tokens"] for r in rec] == [4, 2] and [len(r["logprobs"]) for r in rec] == [3, 1]
    assert all(abs(r["logprob_sum"] - sum(s["logprob"] for s in r["logprobs"])) < 1e-6 for r in rec)
