"""A query all of whose visible scores are -infinity has no softmax: NaN, as from
the decode and prefill kernels.  One that sees nothing gets zeros."""

import math

import pytest
import torch

from qwenforge_amd import paged

pytestmark = pytest.mark.gpu
D = 64


def _decode(dev, b, cap_pages, lens, plen, k0):
    """(output, q, pools) of b rows of one group; k0(kp, table) spoils K."""
    gen = torch.Generator().manual_seed(b + cap_pages)
    kp = torch.randn(40, 2, 64, D, generator=gen).half()
    vp = torch.randn(40, 2, 64, D, generator=gen).half().to(dev)
    q = torch.randn(b, 2, 7, D, generator=gen).half()
    q[..., 0] = 1.0                                      # an infinity in dim 0 gives the score its sign
    table = torch.randint(8, 40, (b, cap_pages), generator=gen, dtype=torch.int32)
    whole = plen // 64
    table[:, :whole] = torch.arange(whole, dtype=torch.int32)
    table[:, whole] = torch.arange(7, 7 - b, -1, dtype=torch.int32)
    k0(kp)
    kp, q, table = kp.to(dev), q.to(dev), table.to(dev)
    last = torch.tensor([n - 1 for n in lens], device=dev)
    rows = torch.tensor([0, b], dtype=torch.int32, device=dev)
    got = paged.flash_decode_attention_prefix_paged(q, kp, vp, table, rows,
                                                    torch.tensor([plen], dtype=torch.int32, device=dev), last)
    return got, q, kp, vp, table, last


@pytest.mark.parametrize("cap_pages", [2, 30])
def test_decode_of_infinite_scores(dev, cap_pages):
    from qwenforge_amd import ops

    def spoil(kp):
        kp[0, 0, :, 0] = -math.inf                       # the prefix, of kv head 0 alone
        kp[7, 0, :3, 0] = -math.inf                      # row 0's own slots
        kp[6, 0, :2, 0] = -math.inf                      # two of row 1's three

    got, q, kp, vp, table, last = _decode(dev, 4, cap_pages, [67, 67, 64, 0], 64, spoil)
    flash = ops.make_flash_scratch(3, 2, 7, table.shape[1] * 64, dev)
    alone = paged.flash_decode_attention_paged(q[:3], kp, vp, table[:3].contiguous(), None, flash, kv_last=last[:3])
    assert torch.isnan(got[0, 0]).all() and torch.isnan(alone[0, 0]).all()
    assert torch.isnan(got[2, 0]).all() and torch.isnan(alone[2, 0]).all()
    v = vp[6, 0, 2].float()                              # all of row 1's weight: one slot
    assert torch.equal(got[1, 0].float(), v.expand(7, D))
    assert torch.isfinite(got[:3, 1]).all() and not got[3].any()


@pytest.mark.parametrize("lens", [[3, 5, 2], [40, 70, 9]])
@pytest.mark.parametrize("pages", [1, 20])               # one split, and several
def test_extension_of_infinite_scores(dev, lens, pages):
    gen = torch.Generator().manual_seed(pages)
    total, ctx = sum(lens), [0, 2, -1]
    pages = max(pages, 2)
    kp = torch.randn(3 * pages, 2, 64, D, generator=gen).half()
    vp = torch.randn(3 * pages, 2, 64, D, generator=gen).half().to(dev)
    table = torch.arange(3 * pages, dtype=torch.int32).view(3, pages)
    q = torch.randn(total, 14, D, generator=gen).half()
    k = torch.randn(total, 2, D, generator=gen).half()
    v = torch.randn(total, 2, D, generator=gen).half().to(dev)
    q[..., 0] = 1.0
    k[:2, 0, 0] = -math.inf                              # row 0: the first two tokens
    kp[pages, 1, :2, 0] = -math.inf                      # row 1: the cached slots, and every new one
    k[lens[0]:lens[0] + lens[1], 1, 0] = -math.inf
    starts = [0, lens[0], lens[0] + lens[1], total]
    out = paged.prefill_extend_paged(q.to(dev), k.to(dev), v, torch.tensor(starts, dtype=torch.int32, device=dev),
                                     max(lens), torch.tensor(ctx, device=dev), None, None, kp.to(dev), vp,
                                     table.to(dev), lengths=lens)
    assert torch.isnan(out[:2, :7]).all() and torch.isfinite(out[:2, 7:]).all()
    assert torch.equal(out[2, :7], v[2, 0].expand(7, D))  # its own slot alone
    assert torch.isfinite(out[2:lens[0]]).all()
    mid = slice(starts[1], starts[2])
    assert torch.isnan(out[mid, 7:]).all() and torch.isfinite(out[mid, :7]).all()
    assert not out[starts[2]:].any()                     # parked
