"""Cancelling ``Engine.score``: it stops between two portions of logits, and whichever way it ends the next
call does not see the flag."""
import pytest
import torch

from util import TINY, model_folder, random_tokens

pytestmark = pytest.mark.gpu

PORTIONS = 5


@pytest.fixture()
def eng(monkeypatch):
    from agave_b200.engine import api
    e = api.Engine(model_folder("A", torch.float32), dtype="float32", max_tokens=1024)
    monkeypatch.setattr(api, "SCORE_LOGITS", 4 * e.spec.vocab_size)           # four rows a portion
    return e


def at_portion(monkeypatch, n, do):
    """Calls ``do`` behind the n-th portion; the list grows by one for each."""
    from agave_b200 import kernels
    made, real = [], kernels.token_logprobs

    def counted(*args, **kw):
        r = real(*args, **kw)
        made.append(1)
        if len(made) == n:
            do()
        return r
    monkeypatch.setattr(kernels, "token_logprobs", counted)
    return made


def usable(eng):
    out = eng.generate([[2, 5, 9]], max_new_tokens=4, stop_token_ids=[])
    assert len(out[0]) == 4 and eng.finish_reasons == ["length"]
    assert eng.runner.cache.book.length == {}                # no slot stays held


def sequence():
    return random_tokens(4 * PORTIONS + 1, TINY["A"][0]["vocab_size"], 1)


def test_stops_between_two_portions(eng, monkeypatch):
    from agave_b200.engine.batch import Cancelled
    made = at_portion(monkeypatch, 2, eng.cancel)
    with pytest.raises(Cancelled):
        eng.score([sequence()])
    assert len(made) == 2
    usable(eng)
    assert len(eng.score([sequence()])[0]) == 4 * PORTIONS


def test_cancelled_behind_the_last_portion(eng, monkeypatch):
    made = at_portion(monkeypatch, PORTIONS, eng.cancel)
    assert len(eng.score([sequence()])[0]) == 4 * PORTIONS and len(made) == PORTIONS
    usable(eng)


def test_cancelled_and_then_an_error(eng, monkeypatch):
    def fail():
        eng.cancel()
        raise RuntimeError("made to fail")
    at_portion(monkeypatch, 1, fail)
    with pytest.raises(RuntimeError, match="made to fail"):
        eng.score([sequence()])
    usable(eng)


def test_cancelled_before_it_starts(eng):
    from agave_b200.engine.batch import Cancelled
    eng.cancel()
    with pytest.raises(Cancelled):
        eng.score([sequence()])
    usable(eng)
