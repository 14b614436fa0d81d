"""Log-probabilities on both sides of every border at which a launch takes other clusters or threads."""
import pytest
import torch

from test_logprobs_gpu import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab", [(36, 16000), (37, 16000), (74, 16001), (148, 15999), (149, 16000), (296, 8200),
                                        (297, 8200), (592, 9001), (593, 9001), (593, 28000), (593, 28001), (297, 65536),
                                        (297, 65537), (1300, 20000)])
def test_borders_of_the_plan(dtype, rows, vocab):
    g = torch.Generator(device="cuda:0").manual_seed(rows + vocab)
    x = (torch.randn(rows, vocab, generator=g, device="cuda:0") * 3).to(dtype)
    tokens = torch.randint(0, vocab, (rows,), generator=g, device="cuda:0").int()
    for top in (0, 32):
        check(x, tokens, top)
