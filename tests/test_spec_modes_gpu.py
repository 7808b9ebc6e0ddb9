"""Draws of sampled requests on the device: steps with and without drafts draw alike."""
from types import SimpleNamespace

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("scale,T", [(3.0, 0.8), (3.0, 1.3), (1.0, 1.0)])
def test_plain_steps_and_tree_steps_draw_the_same_tokens(scale, T):
    """4096 draws among 151936 tokens: one row at a time as a plain step draws them, and along 64 chains of drafts whose tokens are those
    draws, which have to be kept to their ends.  (Sums of the two calls may be cut differently; they are 64-bit, so a draw differs with a
    probability of about 1e-11.)"""
    from coffin_b200.models.qwen35.model import Qwen35Model
    from coffin_b200.ops import tree
    R = C = 64
    V = 151936
    g = torch.Generator(device="cuda").manual_seed(int(10 * scale + 100 * T))
    logits = torch.randn(R, 1, V, generator=g, device="cuda") * scale
    u = torch.rand(R, C, generator=g, device="cuda")
    model = SimpleNamespace(device="cuda")
    draws = torch.stack([Qwen35Model.draw(model, logits[r].expand(C, V), [T] * C, u[r].tolist()) for r in range(R)])
    tokens = torch.zeros(R, C, dtype=torch.int64, device="cuda")
    tokens[:, 1:] = draws[:, :-1]
    anc = torch.tensor([tree.path_words(list(range(-1, C - 1)))] * R, dtype=torch.int64, device="cuda")
    _path, steps, nxt = tree.verify_tree(logits.expand(R, C, V), tokens, anc, torch.full((R,), T, device="cuda"), u)
    assert steps.tolist() == [C] * R
    assert torch.equal(nxt, draws[:, -1])


def test_a_plain_step_draws_hot_and_greedy_rows_together():
    from coffin_b200.models.qwen35.model import Qwen35Model
    g = torch.Generator(device="cuda").manual_seed(2)
    logits = torch.randn(3, 5000, generator=g, device="cuda")
    logits[1, 77] = logits[1, 4000] = 50.0
    model = SimpleNamespace(device="cuda")
    got = Qwen35Model.draw(model, logits, [0.7, 0.0, 1.0], [0.25, 0.9, 0.999])
    for r, (T, u) in enumerate([(0.7, 0.25), (0.0, 0.9), (1.0, 0.999)]):
        if T <= 0:
            want = 77
        else:
            cdf = torch.softmax(logits[r].double() / T, 0).cumsum(0)
            want = int(torch.searchsorted(cdf, torch.tensor(u, dtype=torch.float32, device="cuda").double() * cdf[-1], right=True))
        assert int(got[r]) == want, r
