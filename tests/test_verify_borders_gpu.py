"""``verify.verify_drafts`` where a number stands next to its border.

A draft is accepted while u q < p; here u is one of the two fp32 numbers next to
p / q on either side, at least 2^-30 away from it relative to p.  p in 64 bits is off by less than
2^-36: 2e5 terms of 2^-53 each, summed in either order.
"""

import numpy as np
import pytest
import torch

from qwenforge_amd import verify

pytestmark = pytest.mark.gpu


def _cu(lens, dev):
    return torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=dev)


def _sides(border):
    """The largest fp32 below `border` and the smallest above it, 2^-30 away from it or more."""
    near = np.float32(border)
    low, high = ((np.nextafter(near, np.float32(0)), near) if float(near) > border
                 else (near, np.nextafter(near, np.float32(2))))
    if float(high) - border < border * 2.0 ** -30:
        high = np.nextafter(high, np.float32(2))
    if border - float(low) < border * 2.0 ** -30:
        low = np.nextafter(low, np.float32(0))
    return float(low), float(high)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("drafter", [False, True])
@pytest.mark.parametrize("v,rows,temp", [(7, 40, 1.0), (2049, 40, 0.7), (20011, 700, 1.0), (151936, 24, 1.3),
                                         (300007, 6, 0.3)])
def test_acceptance_next_to_its_border(dev, v, rows, temp, drafter, dtype):
    """Rows of one draft each, u now above and now below; 700 rows leave a position one part."""
    gen = torch.Generator().manual_seed(v + drafter)
    logits = (torch.randn(2 * rows, v, generator=gen) * 2).to(dtype)
    x = logits[::2].double() / temp
    p = torch.softmax(x, dim=-1)
    # Likely and unlikely drafts alike, of probabilities that fp32 holds as normal numbers.
    draft = torch.where(torch.arange(rows) % 3 == 0, p.argmax(dim=-1), torch.multinomial(p, 1, generator=gen)[:, 0])
    p_d = p.gather(1, draft[:, None])[:, 0]
    probs, q_d = None, torch.ones(rows, dtype=torch.float64)
    if drafter:
        probs = torch.softmax(torch.randn(2 * rows, v, generator=gen), dim=-1)
        # As likely as the target's, or u would leave [0, 1).
        probs[torch.arange(0, 2 * rows, 2), draft] = (p_d * (1.2 + torch.rand(rows, generator=gen))).float()
        q_d = probs[torch.arange(0, 2 * rows, 2), draft].double()
    sides = np.array([_sides(b) for b in (p_d / q_d).tolist()])
    assert sides.min() > 0 and sides.max() < 1
    tokens = torch.stack([torch.zeros_like(draft), draft], dim=1).reshape(-1)
    for side in (0, 1):
        u = torch.zeros(2 * rows)
        u[::2] = torch.tensor(sides[:, side], dtype=torch.float32)
        assert ((u[::2].double() * q_d < p_d) == (side == 0)).all()
        _, out = verify.verify_drafts(logits.to(dev), tokens.to(dev), _cu([2] * rows, dev), 2, u.to(dev),
                                      torch.full((rows,), 0.5, device=dev), temperature=temp,
                                      draft_probs=None if probs is None else probs.to(dev), lengths=[2] * rows)
        took = (out[:, 1] >= 0).cpu()
        assert took.all() if side == 0 else not took.any(), (side, took.tolist())


def test_several_borders_in_a_row(dev):
    """Every draft of a row at its border: all kept below it, and none behind the first one above."""
    gen = torch.Generator().manual_seed(5)
    n, v = 40, 3001
    logits = torch.randn(n, v, generator=gen) * 2
    p = torch.softmax(logits.double(), dim=-1)
    tokens = torch.cat([torch.zeros(1, dtype=torch.int64), p.argmax(dim=-1)[:-1]])
    sides = np.array([_sides(p[j, tokens[j + 1]].item()) for j in range(n - 1)])
    for above in (None, 0, 17, n - 2):
        u = torch.zeros(n)
        u[:-1] = torch.tensor(sides[:, 0], dtype=torch.float32)
        if above is not None:
            u[above] = float(sides[above, 1])
            u[above + 1:above + 3] = 0.999              # refused too, behind
        count, out = verify.verify_drafts(logits.to(dev), tokens.to(dev), _cu([n], dev), n, u.to(dev),
                                          torch.full((1,), 0.5, device=dev))
        kept = n - 1 if above is None else above
        assert count.tolist() == [kept + 1]
        assert out[0, :kept].tolist() == tokens[1:kept + 1].tolist()


def test_borders_of_a_few_rows_among_many_positions(dev):
    """So many positions that each is one workgroup's, whose threads add up 75 groups of logits."""
    gen = torch.Generator(dev).manual_seed(9)
    rows, v = 550, 151936
    logits = torch.randn(2 * rows, v, generator=gen, device=dev, dtype=torch.float16) * 2
    tokens = torch.zeros(2 * rows, dtype=torch.int64, device=dev)
    looked = list(range(0, rows, 61)) + [rows - 1]
    p = torch.softmax(logits[[2 * r for r in looked]].cpu().double(), dim=-1)
    draft = p.argmax(dim=-1)
    tokens[[2 * r + 1 for r in looked]] = draft.to(dev)
    sides = np.array([_sides(b) for b in p.gather(1, draft[:, None])[:, 0].tolist()])
    for side in (0, 1):
        u = torch.full((2 * rows,), 0.5, device=dev)
        u[[2 * r for r in looked]] = torch.tensor(sides[:, side], dtype=torch.float32, device=dev)
        _, out = verify.verify_drafts(logits, tokens, _cu([2] * rows, dev), 2, u, torch.full((rows,), 0.5, device=dev))
        took = (out[looked, 1] >= 0).cpu()
        assert took.all() if side == 0 else not took.any(), (side, took.tolist())
