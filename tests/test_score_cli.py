"""What ``--score`` and ``--logprobs`` print, with an engine that answers by rote."""
import json
import math
from types import SimpleNamespace

import pytest

from agave_b200.sampling import TokenScore


def printed(capsys, logprobs, json_out=True, prompt=None):
    from agave_b200.cli import _score_prompts
    row = [TokenScore(i, lp, 1.0, 1) for i, lp in enumerate(logprobs)]
    engine = SimpleNamespace(score=lambda prompts, top: [row])
    args = SimpleNamespace(logprobs=None, json=json_out, quiet=False)
    assert _score_prompts(engine, [prompt or [1] * (len(row) + 1)], args) == 0
    return capsys.readouterr()


def strict(text):
    def refuse(name):
        raise ValueError(name)
    return json.loads(text, parse_constant=refuse)


@pytest.mark.parametrize("logprobs,total,perplexity", [
    ([], 0, None),                                            # one token: nothing scored
    ([-1.0, -3.0], -4.0, math.exp(2.0)),
    ([0.0], 0.0, 1.0),
    ([-1.0, -math.inf], None, None),                          # an impossible token
    ([math.nan, -1.0], None, None),
    ([-2000.0, -1000.0], -3000.0, None),                      # e^1500 is no float
    ([-700.0], -700.0, math.exp(700.0)),
])
def test_perplexity(capsys, logprobs, total, perplexity):
    rec = strict(printed(capsys, logprobs).out)
    assert rec["logprob_sum"] == total
    assert rec["perplexity"] is None if perplexity is None else abs(rec["perplexity"] / perplexity - 1) < 1e-12
    assert [r["logprob"] for r in rec["logprobs"]] == [lp if math.isfinite(lp) else None for lp in logprobs]
    text = printed(capsys, logprobs, json_out=False)
    assert len(text.out.splitlines()) == len(logprobs)
    assert text.err.strip().endswith("none" if perplexity is None else str(rec["perplexity"]))


@pytest.mark.parametrize("json_out", [True, False])
@pytest.mark.parametrize("score", [True, False])
def test_log_probabilities_are_asked_for_where_they_are_printed(tmp_path, monkeypatch, capsys, json_out, score):
    from agave_b200 import cli
    from agave_b200.engine import api
    from util import TINY
    asked = []

    class Recorder:
        max_seq_len, load_seconds, ignored_tensors = 64, 0.0, ()

        @classmethod
        def from_config(cls, *args, **kw):
            return cls()

        def model_info(self):
            return {"config": {}, "dtype": "bfloat16", "weight_bytes": 0, "cache_bytes": 0}

        def generate(self, prompts, logprobs=None, **kw):
            asked.append(logprobs)
            raise RuntimeError("asked")

        def score(self, prompts, top=0):
            asked.append(top)
            raise RuntimeError("asked")
    monkeypatch.setattr(api, "Engine", Recorder)
    (tmp_path / "config.json").write_text(json.dumps(TINY["A"][0]))
    argv = [str(tmp_path), "--random-weights", "1", "--tokens", "1,2", "--logprobs", "4"]
    assert cli.main(argv + ["--json"] * json_out + ["--score"] * score) == 1
    assert asked == [4 if json_out else 0 if score else None]
