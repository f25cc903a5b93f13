"""``verify.verify_drafts`` at a position that gives no distribution: its draft is
refused and nothing is drawn in its place."""

import math

import pytest
import torch

from qwenforge_amd import verify

pytestmark = pytest.mark.gpu


def _cu(lens, dev):
    return torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=dev)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("drafter", [False, True])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_a_refused_draft_without_a_distribution_draws_nothing(dev, dtype, drafter, bad):
    """The position's only NaN or infinity is the draft's own logit."""
    v = 5003
    gen = torch.Generator().manual_seed(7)
    x = torch.randn(8, v, generator=gen)
    drafts = [0, 5002, 2048, 77]
    for i, d in enumerate(drafts):
        x[2 * i, d] = bad
    tokens = torch.tensor([t for d in drafts for t in (0, d)], device=dev)
    probs = torch.softmax(torch.randn(8, v, generator=gen), dim=-1).to(dev) if drafter else None
    count, out = verify.verify_drafts(x.to(dtype).to(dev), tokens, _cu([2] * 4, dev), 2,
                                      torch.full((8,), 0.25, device=dev), torch.full((4,), 0.5, device=dev),
                                      draft_probs=probs)
    assert count.tolist() == [0] * 4 and (out == -1).all()
