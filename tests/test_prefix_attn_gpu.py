"""Shared-prefix decode and extension (``include/qf_prefix.h``) against the
definition in 64 bits.

Tolerance: with |v| <= V the output is sum_j w_j v_j.  The kernel rounds each
p_j to fp16 (relative 2^-11) and divides by the sum of the rounded ones, so the
weights move by at most 2 * 2^-11 relative and the output by 2 * 2^-11 * V; the
fp16 store adds 2^-11 |out| <= 2^-11 V.  The scores' fp32 sums of 64 products
(|q|, |k| about 1, |score| < 16 after scaling) are off by less than 2^-18, which
moves p by as much.  In all 3.02 * 2^-11 * V, V the largest |v|: TOL * V.
"""

import math

import pytest
import torch

from qwenforge_amd import paged

pytestmark = pytest.mark.gpu
TOL = 3.1 * 2.0 ** -11
D = 64


def _attend(q, k, v, scale=0.125):
    """q (G, 64) over k, v (n, 64), float64; zeros over nothing."""
    if k.shape[0] == 0:
        return torch.zeros_like(q)
    return torch.softmax(q @ k.T * scale, dim=-1) @ v


def _pools(gen, n_pages, kvh, page, dev, dims=D):
    """Pools whose unused memory would show: every value random."""
    return [torch.randn(n_pages, kvh, page, dims, generator=gen).half().to(dev) for _ in range(2)]


def _slots(pool, pages, n):
    """(KVH, n, 64) float64 on the CPU of a row's first n slots."""
    pool, page = pool.cpu().double(), pool.shape[2]
    if n == 0:
        return torch.zeros(pool.shape[1], 0, D, dtype=torch.float64)
    rows = torch.stack([pool[pages[s // page], :, s % page] for s in range(n)])
    return rows.transpose(0, 1)


# --------------------------------------------------------------------------
# shared-prefix decode
# --------------------------------------------------------------------------

def _prefix_case(gen, dev, groups, lens, plens, kvh, page, ppr=None):
    """Rows of `groups` (row counts) sharing plens[g] leading slots, lens[b] slots in all."""
    b = sum(groups)
    ppr = ppr or max(1, -(-max(max(lens), max(plens, default=0)) // page))
    n_pages = sum(p // page + 1 for p in plens) + b * ppr + 3
    kp, vp = _pools(gen, n_pages, kvh, page, dev)
    free = torch.randperm(n_pages, generator=gen).tolist()
    table = torch.full((b, ppr), -1, dtype=torch.int32)
    row = 0
    for n, p in zip(groups, plens):
        whole = p // page
        shared = [free.pop() for _ in range(whole)]
        for r in range(row, row + n):
            mine = [free.pop() for _ in range(ppr - whole)]
            table[r] = torch.tensor(shared + mine, dtype=torch.int32)
            if p % page and r > row:                     # the partly filled page: a copy
                a, c = int(table[row, whole]), int(table[r, whole])
                kp[c, :, :p % page], vp[c, :, :p % page] = kp[a, :, :p % page], vp[a, :, :p % page]
        row += n
    for r in range(row, b):
        table[r] = torch.tensor([free.pop() for _ in range(ppr)], dtype=torch.int32)
    return kp, vp, table


def _prefix_ref(q, kp, vp, table, lens):
    out = torch.zeros(q.shape, dtype=torch.float64)
    q = q.cpu().double()
    for r, n in enumerate(lens):
        k, v = _slots(kp, table[r], n), _slots(vp, table[r], n)
        for h in range(q.shape[1]):
            out[r, h] = _attend(q[r, h], k[h], v[h])
    return out


def _starts(groups, first=0):
    out = [first]
    for n in groups:
        out.append(out[-1] + n)
    return out


CASES = [
    # groups, plens, lens of the rows, kvh, g, page
    ([4], [100], [101, 100, 130, 300], 2, 7, 64),
    ([1], [1], [1], 1, 1, 64),
    ([2], [64], [64, 65], 2, 7, 64),                     # a row that ends with the prefix
    ([3, 1, 2], [257, 64, 0], [300, 259, 900, 64, 1, 77], 2, 7, 64),
    ([5], [700], [0, 701, 33, 700, 1000], 2, 7, 128),    # parked, and shorter than the prefix
    ([20], [515], [516 + 13 * i for i in range(20)], 2, 7, 64),      # several tiles of the larger form
    ([9], [200], [201 + i for i in range(9)], 3, 16, 256),
    ([70], [130], [131 + i for i in range(70)], 1, 8, 64),
    ([1] * 70, [65] * 70, [66 + i for i in range(70)], 1, 4, 64),    # more groups than lanes
]


@pytest.mark.parametrize("case", range(len(CASES)))
def test_prefix_decode_matches_definition(dev, case):
    groups, plens, lens, kvh, g, page = CASES[case]
    gen = torch.Generator().manual_seed(case)
    kp, vp, table = _prefix_case(gen, dev, groups, lens, plens, kvh, page)
    q = torch.randn(len(lens), kvh, g, D, generator=gen).half().to(dev)
    rows = torch.tensor(_starts(groups), dtype=torch.int32, device=dev)
    got = paged.flash_decode_attention_prefix_paged(
        q, kp, vp, table.to(dev), rows, torch.tensor(plens, dtype=torch.int32, device=dev),
        torch.tensor([n - 1 for n in lens], device=dev))
    ref = _prefix_ref(q, kp, vp, table, lens)
    err = (got.cpu().double() - ref).abs().max().item()
    print(f"[prefix] {groups} {plens} err {err:.2e}", flush=True)
    assert err <= TOL * vp.abs().max().item()
    for r, n in enumerate(lens):
        if n == 0:
            assert not got[r].any()


def test_prefix_decode_long_uses_many_splits_and_pages(dev):
    gen = torch.Generator().manual_seed(77)
    lens = [9001, 8500, 8449]
    kp, vp, table = _prefix_case(gen, dev, [3], lens, [8448], 2, 64)
    q = torch.randn(3, 2, 7, D, generator=gen).half().to(dev)
    got = paged.flash_decode_attention_prefix_paged(
        q, kp, vp, table.to(dev), torch.tensor([0, 3], dtype=torch.int32, device=dev),
        torch.tensor([8448], dtype=torch.int32, device=dev), torch.tensor([n - 1 for n in lens], device=dev))
    ref = _prefix_ref(q, kp, vp, table, lens)
    assert (got.cpu().double() - ref).abs().max().item() <= TOL * vp.abs().max().item()


def test_rows_outside_the_groups_and_any_bounds(dev):
    """Rows before, between and behind the groups share nothing; bounds and
    prefix lengths beyond the batch or the table are clamped."""
    gen = torch.Generator().manual_seed(5)
    lens = [90, 200, 130, 70, 260]
    kp, vp, table = _prefix_case(gen, dev, [1] * 5, lens, [0] * 5, 2, 64)
    table[2, 0] = table[1, 0]                            # rows 1 and 2 share 64 slots
    q = torch.randn(5, 2, 7, D, generator=gen).half().to(dev)
    ref = _prefix_ref(q, kp, vp, table, lens)
    last = torch.tensor([n - 1 for n in lens], device=dev)
    tol = TOL * vp.abs().max().item()
    for rows, plen in (([1, 3], [64]), ([1, 3, 3], [64, 9]), ([3, 1, 2], [128, 70]), ([5, 9], [64]),
                       ([-4, 1, 1], [90, 5]), ([4, 2**31 - 1], [2**31 - 1]), ([0, 1], [-7]),
                       ([-2**31, 0], [64])):
        got = paged.flash_decode_attention_prefix_paged(
            q, kp, vp, table.to(dev), torch.tensor(rows, dtype=torch.int32, device=dev),
            torch.tensor(plen, dtype=torch.int32, device=dev), last)
        assert (got.cpu().double() - ref).abs().max().item() <= tol, (rows, plen)


def test_unseen_slots_may_hold_anything(dev):
    """Infinities and NaN behind a row's last slot, in the K and V of pages the
    row maps, and in slots of the prefix that only longer rows see."""
    gen = torch.Generator().manual_seed(6)
    lens = [150, 40, 0, 131]
    kp, vp, table = _prefix_case(gen, dev, [4], lens, [128], 2, 64)
    q = torch.randn(4, 2, 7, D, generator=gen).half().to(dev)
    ref = _prefix_ref(q, kp, vp, table, lens)
    clean = vp.abs().max().item()
    for x in (math.inf, -math.inf, math.nan):
        for r in (0, 3):                                 # behind the last slot of the row's own page
            kp[table[r, 2], :, lens[r] % 64:] = x
            vp[table[r, 2], :, lens[r] % 64:] = x
        got = paged.flash_decode_attention_prefix_paged(
            q, kp, vp, table.to(dev), torch.tensor([0, 4], dtype=torch.int32, device=dev),
            torch.tensor([128], dtype=torch.int32, device=dev), torch.tensor([n - 1 for n in lens], device=dev))
        assert (got.cpu().double() - ref).abs().max().item() <= TOL * clean
    # Row 1 ends at slot 40: what rows 0 and 3 see at slot 50 reaches them alone.
    vp[table[0, 0], 0, 50, 3] = math.inf
    vp[table[0, 0], 1, 51, 9] = math.nan
    got = paged.flash_decode_attention_prefix_paged(
        q, kp, vp, table.to(dev), torch.tensor([0, 4], dtype=torch.int32, device=dev),
        torch.tensor([128], dtype=torch.int32, device=dev), torch.tensor([n - 1 for n in lens], device=dev))
    got = got.cpu().double()
    for r in (1, 2):
        assert (got[r] - ref[r]).abs().max().item() <= TOL * clean
    for r in (0, 3):
        assert torch.isinf(got[r, 0, :, 3]).all() and torch.isnan(got[r, 1, :, 9]).all()
        got[r, 0, :, 3], got[r, 1, :, 9] = ref[r, 0, :, 3], ref[r, 1, :, 9]
        assert (got[r] - ref[r]).abs().max().item() <= TOL * clean


def test_prefix_decode_strides_scale_out_and_another_stream(dev):
    gen = torch.Generator().manual_seed(8)
    lens = [140, 131, 200]
    kp, vp, table = _prefix_case(gen, dev, [3], lens, [128], 2, 64)
    wide = torch.randn(3, 2, 9, 80, generator=gen).half().to(dev)
    q = wide[:, :, 1:8, 8:72]
    # Pools with slots outside heads and a padded row.
    kp2 = torch.empty(kp.shape[0], 64, 2, 72, device=dev, dtype=torch.float16)[..., :64].transpose(1, 2)
    kp2.copy_(kp)
    table_wide = torch.full((3, table.shape[1] + 3), 12345, dtype=torch.int32, device=dev)
    table_wide[:, :table.shape[1]] = table.to(dev)
    last = torch.zeros(3, 2, dtype=torch.int64, device=dev)
    last[:, 0] = torch.tensor([n - 1 for n in lens])
    ref = torch.zeros(q.shape, dtype=torch.float64)
    for r, n in enumerate(lens):
        k, v = _slots(kp, table[r], n), _slots(vp, table[r], n)
        for h in range(2):
            ref[r, h] = _attend(q[r, h].cpu().double(), k[h], v[h], 0.31)
    out = torch.full((3, 2, 7, 128), 5.0, device=dev, dtype=torch.float16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = paged.flash_decode_attention_prefix_paged(
            q, kp2, vp, table_wide[:, :table.shape[1]], torch.tensor([0, 3], dtype=torch.int32, device=dev),
            torch.tensor([128], dtype=torch.int32, device=dev), last[:, 0], scale=0.31, out=out[..., 64:])
    side.synchronize()
    assert got.data_ptr() == out[..., 64:].data_ptr() and (out[..., :64] == 5.0).all()
    assert (got.cpu().double() - ref).abs().max().item() <= TOL * vp.abs().max().item()


def test_captured_prefix_decode_follows_lengths_groups_and_tables(dev):
    gen = torch.Generator().manual_seed(9)
    kp, vp, table = _prefix_case(gen, dev, [6], [500] * 6, [256], 2, 64, ppr=8)
    q = torch.randn(6, 2, 7, D, generator=gen).half().to(dev)
    rows = torch.tensor([0, 3, 6], dtype=torch.int32, device=dev)
    plen = torch.tensor([256, 256], dtype=torch.int32, device=dev)
    last = torch.full((6,), -1, dtype=torch.int64, device=dev)
    t = table.to(dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = paged.flash_decode_attention_prefix_paged(q, kp, vp, t, rows, plen, last)
    for lens, bounds, pl in (([257, 300, 500, 256, 400, 0], [0, 3, 6], [256, 256]),
                             ([400, 1, 129, 260, 300, 512], [0, 6, 6], [192, 1]),
                             ([1, 2, 3, 4, 5, 6], [2, 4, 5], [0, 64])):
        q.normal_()
        last.copy_(torch.tensor([n - 1 for n in lens]))
        rows.copy_(torch.tensor(bounds, dtype=torch.int32))
        plen.copy_(torch.tensor(pl, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        eager = paged.flash_decode_attention_prefix_paged(q, kp, vp, t, rows, plen, last)
        assert torch.equal(got, eager)
        ref = _prefix_ref(q, kp, vp, table, lens)
        assert (got.cpu().double() - ref).abs().max().item() <= TOL * vp.abs().max().item()


def test_prefix_pages_of_their_own_table(dev):
    """Groups whose first rows have nothing mapped: the prefix comes from
    ``prefix_table``; a prefix length past its pages is clamped to them."""
    gen = torch.Generator().manual_seed(12)
    lens = [0, 300, 280, 0, 0, 150]
    kp, vp, table = _prefix_case(gen, dev, [3, 3], lens, [256, 128], 2, 64)
    own = torch.stack([table[1].clone(), table[5].clone()])[:, :4].contiguous()
    own[1, 2:] = -7                                      # group 1's pages end at slot 128
    gone = table.clone()
    gone[0], gone[3] = -1, -1
    q = torch.randn(6, 2, 7, D, generator=gen).half().to(dev)
    ref = _prefix_ref(q, kp, vp, table, lens)
    rows = torch.tensor([0, 3, 6], dtype=torch.int32, device=dev)
    last = torch.tensor([n - 1 for n in lens], device=dev)
    for pages, plen in ((own, [256, 128]), (own[:, :2].contiguous(), [1000, 128])):
        got = paged.flash_decode_attention_prefix_paged(
            q, kp, vp, gone.to(dev), rows, torch.tensor(plen, dtype=torch.int32, device=dev), last,
            prefix_table=pages.to(dev))
        assert (got.cpu().double() - ref).abs().max().item() <= TOL * vp.abs().max().item()
    for bad, kind in ((own[:1], ValueError), (own.long(), TypeError), (own[:, :0], ValueError)):
        with pytest.raises(kind):
            paged.flash_decode_attention_prefix_paged(
                q, kp, vp, gone.to(dev), rows, torch.tensor([256, 128], dtype=torch.int32, device=dev), last,
                prefix_table=bad.to(dev))


def test_a_row_keeps_its_bits_in_any_company(dev):
    gen = torch.Generator().manual_seed(13)
    b = 20
    kp, vp, table = _prefix_case(gen, dev, [b], [1000] * b, [640], 2, 64)
    q = torch.randn(b, 2, 7, D, generator=gen).half().to(dev)
    rows = torch.tensor([0, b], dtype=torch.int32, device=dev)
    plen = torch.tensor([640], dtype=torch.int32, device=dev)
    seen = []
    for others, scale in ((999, 1.0), (-1, 1.0), (641, 30.0)):
        last = torch.full((b,), others, dtype=torch.int64, device=dev)
        last[9] = 800
        qs = q * scale
        qs[9] = q[9]
        seen.append(paged.flash_decode_attention_prefix_paged(qs, kp, vp, table.to(dev), rows, plen, last)[9].clone())
    assert torch.equal(seen[0], seen[1]) and torch.equal(seen[0], seen[2])


def test_prefix_decode_refusals(dev):
    gen = torch.Generator().manual_seed(10)
    kp, vp, table = _prefix_case(gen, dev, [2], [70, 80], [64], 2, 64)
    q = torch.randn(2, 2, 7, D, generator=gen).half().to(dev)
    rows = torch.tensor([0, 2], dtype=torch.int32, device=dev)
    plen = torch.tensor([64], dtype=torch.int32, device=dev)
    last = torch.tensor([69, 79], device=dev)
    ok = dict(grouped=q, k_pool=kp, v_pool=vp, block_table=table.to(dev), prefix_rows=rows,
              prefix_len=plen, kv_last=last)
    paged.flash_decode_attention_prefix_paged(**ok)
    for change, kind in ((dict(prefix_rows=rows[:1]), ValueError), (dict(prefix_rows=rows.long()), TypeError),
                         (dict(prefix_len=plen.cpu()), TypeError), (dict(prefix_len=plen[:0]), ValueError),
                         (dict(kv_last=last[:1]), ValueError), (dict(kv_last=last.int()), TypeError),
                         (dict(kv_last=None), TypeError), (dict(grouped=q.float()), TypeError),
                         (dict(grouped=q[:, :1]), ValueError), (dict(block_table=table.to(dev)[:1]), ValueError),
                         (dict(out=q[:1]), ValueError), (dict(scale=0.0), RuntimeError),
                         (dict(scale=-1.0), RuntimeError), (dict(scale=math.nan), RuntimeError),
                         (dict(grouped=torch.zeros(2, 2, 17, D, device=dev).half()), RuntimeError)):
        with pytest.raises(kind):
            paged.flash_decode_attention_prefix_paged(**{**ok, **change})


# --------------------------------------------------------------------------
# extension
# --------------------------------------------------------------------------

def _extend_ref(q, k, v, cu, ctx, kp, vp, table, cap):
    """Outputs and the pools after the appends, float64 / fp16 on the CPU."""
    kp, vp, page = kp.cpu().clone(), vp.cpu().clone(), kp.shape[2]
    q, k, v = q.cpu(), k.cpu(), v.cpu()
    g = q.shape[1] // k.shape[1]
    for r, c in enumerate(ctx):
        for i in range(cu[r + 1] - cu[r]):
            if 0 <= c and c + i < cap:
                p = int(table[r, (c + i) // page])
                if 0 <= p < kp.shape[0]:
                    kp[p, :, (c + i) % page], vp[p, :, (c + i) % page] = k[cu[r] + i], v[cu[r] + i]
    out = torch.zeros(q.shape, dtype=torch.float64)
    for r, c in enumerate(ctx):
        n = cu[r + 1] - cu[r]
        if c < 0 or n == 0:
            continue
        ks, vs = (_slots(x, table[r], min(c + n, cap)) for x in (kp, vp))
        for i in range(n):
            for h in range(q.shape[1]):
                m = min(c + i + 1, cap)
                out[cu[r] + i, h] = _attend(q[cu[r] + i, h:h + 1].double(), ks[h // g, :m], vs[h // g, :m])[0]
    return out, kp, vp


def _extend_case(gen, dev, lens, ctx, qh, kvh, page, extra=0):
    b = len(lens)
    ppr = max(1, -(-max(max(c, 0) + n for c, n in zip(ctx, lens)) // page)) + extra
    n_pages = b * ppr + 2
    kp, vp = _pools(gen, n_pages, kvh, page, dev)
    table = torch.randperm(n_pages, generator=gen)[:b * ppr].view(b, ppr).to(torch.int32)
    qkv = torch.randn(sum(lens), qh + 2 * kvh, D, generator=gen).half().to(dev)
    return qkv[:, :qh], qkv[:, qh:qh + kvh], qkv[:, qh + kvh:], kp, vp, table


EXTENDS = [
    # lens, contexts, qh, kvh, page
    ([5, 5, 5], [300, 64, 7], 14, 2, 64),
    ([1], [0], 1, 1, 64),
    ([1, 1], [63, 64], 14, 2, 64),
    ([0, 3, 0, 17, 0], [10, 61, 0, 0, 5], 14, 2, 64),    # rows without tokens
    ([130, 9], [70, 513], 14, 2, 128),
    ([33, 2, 64], [0, -1, 100], 8, 2, 64),               # a parked row
    ([150], [1000], 16, 1, 256),
    ([40, 70], [129, 3], 3, 3, 64),                      # one head each
    ([1] * 66, list(range(66)), 4, 2, 64),               # more rows than lanes
]


@pytest.mark.parametrize("case", range(len(EXTENDS)))
def test_extension_matches_definition(dev, case):
    lens, ctx, qh, kvh, page = EXTENDS[case]
    gen = torch.Generator().manual_seed(100 + case)
    q, k, v, kp, vp, table = _extend_case(gen, dev, lens, ctx, qh, kvh, page)
    cu = _starts(lens)
    cap = table.shape[1] * page
    ref, kr, vr = _extend_ref(q, k, v, cu, ctx, kp, vp, table, cap)
    got = paged.prefill_extend_paged(q, k, v, torch.tensor(cu, dtype=torch.int32, device=dev), max(lens),
                                     torch.tensor(ctx, device=dev), None, None, kp, vp, table.to(dev))
    err = (got.cpu().double() - ref).abs().max().item()
    print(f"[extend] {lens} {ctx} err {err:.2e}", flush=True)
    assert torch.equal(kp.cpu(), kr) and torch.equal(vp.cpu(), vr)
    assert err <= TOL * max(vp.abs().max().item(), 1.0)


def test_extension_of_a_long_context(dev):
    gen = torch.Generator().manual_seed(31)
    lens, ctx = [6, 20], [4500, 4200]
    q, k, v, kp, vp, table = _extend_case(gen, dev, lens, ctx, 14, 2, 64)
    cu = _starts(lens)
    ref, _, _ = _extend_ref(q, k, v, cu, ctx, kp, vp, table, table.shape[1] * 64)
    for bound in (None, 4506):
        got = paged.prefill_extend_paged(q, k, v, torch.tensor(cu, dtype=torch.int32, device=dev), 20,
                                         torch.tensor(ctx, device=dev), None, None, kp, vp, table.to(dev),
                                         lengths=lens, max_slots=bound)
        assert (got.cpu().double() - ref).abs().max().item() <= TOL * vp.abs().max().item()


def test_extension_from_nothing_is_the_paged_prefill(dev):
    """Context 0: the same rotated K and raw V in the pages bit for bit, and the
    same attention within both kernels' rounding."""
    from qwenforge_amd.rope import cos_sin, inv_freq

    gen = torch.Generator().manual_seed(32)
    lens = [70, 1, 129]
    q, k, v, kp, vp, table = _extend_case(gen, dev, lens, [0, 0, 0], 14, 2, 64)
    cu = torch.tensor(_starts(lens), dtype=torch.int32, device=dev)
    pos = torch.cat([torch.arange(n) for n in lens]).to(dev)
    cos, sin = cos_sin(pos, inv_freq(64, 1e6, dev))
    kp2, vp2 = kp.clone(), vp.clone()
    want = paged.prefill_varlen_paged(q, k, v, cu, 129, cos, sin, kp2, vp2, table.to(dev))
    got = paged.prefill_extend_paged(q, k, v, cu, 129, torch.zeros(3, dtype=torch.int64, device=dev), cos,
                                     sin, kp, vp, table.to(dev))
    assert torch.equal(kp, kp2) and torch.equal(vp, vp2)
    assert (got.double() - want.double()).abs().max().item() <= 2 * TOL * v.abs().max().item()


def test_extension_in_pieces_is_the_whole(dev):
    """A prompt in chunks writes the same pages as at once, and each chunk's
    outputs are the definition's."""
    gen = torch.Generator().manual_seed(33)
    q, k, v, kp, vp, table = _extend_case(gen, dev, [200], [0], 14, 2, 64)
    ref, kr, vr = _extend_ref(q, k, v, [0, 200], [0], kp, vp, table, table.shape[1] * 64)
    at = 0
    for n in (1, 63, 7, 100, 29):
        part = slice(at, at + n)
        got = paged.prefill_extend_paged(q[part], k[part], v[part],
                                         torch.tensor([0, n], dtype=torch.int32, device=dev), n,
                                         torch.tensor([at], device=dev), None, None, kp, vp, table.to(dev))
        assert (got.cpu().double() - ref[part]).abs().max().item() <= TOL * v.abs().max().item()
        at += n
    assert torch.equal(kp.cpu(), kr) and torch.equal(vp.cpu(), vr)


def test_extension_masked_values_and_bad_pages(dev):
    """A later token's infinite V reaches no earlier token; stale slots may hold
    NaN; a page outside the pool is not written; slots past max_slots neither."""
    gen = torch.Generator().manual_seed(34)
    lens, ctx = [20, 9], [30, 100]
    q, k, v, kp, vp, table = _extend_case(gen, dev, lens, ctx, 14, 2, 64, extra=1)
    q, k, v = q.clone(), k.clone(), v.clone()
    cu = _starts(lens)
    for r in range(2):                                   # stale memory behind the rows
        end = ctx[r] + lens[r]
        kp[table[r, end // 64], :, end % 64:] = math.nan
        vp[table[r, end // 64], :, end % 64:] = math.nan
    cap = table.shape[1] * 64
    ref, kr, vr = _extend_ref(q, k, v, cu, ctx, kp, vp, table, cap)
    args = (torch.tensor(cu, dtype=torch.int32, device=dev), 20, torch.tensor(ctx, device=dev), None, None)
    clean = v.abs().max().item()
    got = paged.prefill_extend_paged(q, k, v, *args, kp, vp, table.to(dev))
    assert (got.cpu().double() - ref).abs().max().item() <= TOL * max(clean, 4.0)
    v[12, 1, 5] = math.inf                               # row 0's token 12
    k[12, 0, 0] = math.nan
    got = paged.prefill_extend_paged(q, k, v, *args, kp, vp, table.to(dev)).cpu().double()
    early = list(range(12)) + list(range(20, 29))
    assert (got[early] - ref[early]).abs().max().item() <= TOL * max(clean, 4.0)
    assert torch.isinf(got[12:20, 7:, 5]).all() and torch.isnan(got[12:20, :7]).all()
    # Bad pages and the bound.
    q, k, v, kp, vp, table = _extend_case(gen, dev, [80], [0], 14, 2, 64)
    bad = table.clone()
    bad[0, 1] = kp.shape[0]
    before = kp.clone(), vp.clone()
    paged.prefill_extend_paged(q, k, v, torch.tensor([0, 80], dtype=torch.int32, device=dev), 80,
                               torch.tensor([0], device=dev), None, None, kp, vp, bad.to(dev))
    touched = [p for p in range(kp.shape[0]) if not torch.equal(kp[p], before[0][p])]
    assert touched == [int(table[0, 0])]
    kp.copy_(before[0]), vp.copy_(before[1])
    paged.prefill_extend_paged(q, k, v, torch.tensor([0, 80], dtype=torch.int32, device=dev), 80,
                               torch.tensor([30], device=dev), None, None, kp, vp, table.to(dev), max_slots=100)
    changed = (kp != before[0]).any(dim=3).any(dim=1).sum().item()
    assert changed == 70                                 # slots 30 .. 99


def test_captured_extension_follows_contexts(dev):
    gen = torch.Generator().manual_seed(35)
    lens = [4, 0, 6]
    q, k, v, kp, vp, table = _extend_case(gen, dev, [4, 1, 6], [250, 250, 250], 14, 2, 64)
    q, k, v = q[:10], k[:10], v[:10]
    cu = torch.tensor(_starts(lens), dtype=torch.int32, device=dev)
    ctx = torch.zeros(3, dtype=torch.int64, device=dev)
    t = table.to(dev)
    kp0, vp0 = kp.clone(), vp.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = paged.prefill_extend_paged(q, k, v, cu, 6, ctx, None, None, kp, vp, t)
    for c in ([0, 0, 0], [250, -1, 63], [-1, 5, 200]):
        ctx.copy_(torch.tensor(c))
        kp.copy_(kp0), vp.copy_(vp0)
        graph.replay()
        torch.cuda.synchronize()
        ref, kr, vr = _extend_ref(q, k, v, _starts(lens), c, kp0, vp0, table, 256)
        assert torch.equal(kp.cpu(), kr) and torch.equal(vp.cpu(), vr)
        assert (got.cpu().double() - ref).abs().max().item() <= TOL * vp.abs().max().item()


@pytest.mark.parametrize("ppr", [1, 5])                  # whole rows, and rows cut into splits
def test_tokens_behind_the_last_row_are_left_alone(dev, ppr):
    """A captured call whose offsets shrink: padding is neither appended nor
    attended, and its outputs stay as they were."""
    gen = torch.Generator().manual_seed(37)
    lens, ctx = [3, 4], [9, 20]
    q, k, v, kp, vp, table = _extend_case(gen, dev, [6, 6], [0, 0], 14, 2, 64, extra=ppr - 1)
    cu = torch.tensor([0, 6, 12], dtype=torch.int32, device=dev)
    context = torch.tensor(ctx, device=dev)
    t = table.to(dev)
    kp0, vp0 = kp.clone(), vp.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = paged.prefill_extend_paged(q, k, v, cu, 6, context, None, None, kp, vp, t)
    for first in (0, 2):
        bounds = _starts(lens, first)
        cu.copy_(torch.tensor(bounds, dtype=torch.int32))
        kp.copy_(kp0), vp.copy_(vp0), got.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        ref, kr, vr = _extend_ref(q, k, v, bounds, ctx, kp0, vp0, table, 64 * ppr)
        assert torch.equal(kp.cpu(), kr) and torch.equal(vp.cpu(), vr)
        rows = slice(bounds[0], bounds[-1])
        assert (got[rows].cpu().double() - ref[rows]).abs().max().item() <= TOL * vp.abs().max().item()
        assert (got[:bounds[0]] == 7).all() and (got[bounds[-1]:] == 7).all()


def test_offsets_past_32_bits(dev):
    """Pages 2^31 elements apart, heads 2^30: attention, appends and copies."""
    gen = torch.Generator().manual_seed(38)
    sp, sh = 2**31 + 1024, 2**30 + 512
    pools = []
    for _ in range(2):
        store = torch.empty(2 * sp + sh + 64 * D, device=dev, dtype=torch.float16)
        pool = store.as_strided((3, 2, 64, D), (sp, sh, D, 1))
        pool.copy_(torch.randn(3, 2, 64, D, generator=gen))
        pools.append(pool)
    kp, vp = pools
    table = torch.tensor([[0, 2], [0, 1]], dtype=torch.int32)
    lens = [110, 70]
    q = torch.randn(2, 2, 7, D, generator=gen).half().to(dev)
    got = paged.flash_decode_attention_prefix_paged(
        q, kp, vp, table.to(dev), torch.tensor([0, 2], dtype=torch.int32, device=dev),
        torch.tensor([64], dtype=torch.int32, device=dev), torch.tensor([n - 1 for n in lens], device=dev))
    tol = TOL * vp.abs().max().item()
    assert (got.cpu().double() - _prefix_ref(q, kp, vp, table, lens)).abs().max().item() <= tol
    qkv = torch.randn(5, 18, D, generator=gen).half().to(dev)
    q, k, v = qkv[:, :14], qkv[:, 14:16], qkv[:, 16:]
    ref, kr, vr = _extend_ref(q, k, v, [0, 3, 5], lens, kp, vp, table, 128)
    got = paged.prefill_extend_paged(q, k, v, torch.tensor([0, 3, 5], dtype=torch.int32, device=dev), 3,
                                     torch.tensor(lens, device=dev), None, None, kp, vp, table.to(dev))
    assert torch.equal(kp.cpu(), kr) and torch.equal(vp.cpu(), vr)
    assert (got.cpu().double() - ref).abs().max().item() <= TOL * max(vp.abs().max().item(), v.abs().max().item())
    paged.copy_pages([kp, vp], [2], [0], slots=[50])
    kr[0, :, :50], vr[0, :, :50] = kr[2, :, :50], vr[2, :, :50]
    assert torch.equal(kp.cpu(), kr) and torch.equal(vp.cpu(), vr)


def test_two_streams_at_once(dev):
    """Calls that overlap take scratch of their own: every result has the bits of
    the same call alone."""
    gen = torch.Generator().manual_seed(39)
    decode, extend = [], []
    for n in (3, 5):
        lens = [2000 + 77 * i for i in range(n)]
        kp, vp, table = _prefix_case(gen, dev, [n], lens, [1900], 2, 64)
        q = torch.randn(n, 2, 7, D, generator=gen).half().to(dev)
        decode.append((q, kp, vp, table.to(dev), torch.tensor([0, n], dtype=torch.int32, device=dev),
                       torch.tensor([1900], dtype=torch.int32, device=dev),
                       torch.tensor([x - 1 for x in lens], device=dev)))
        q, k, v, kp, vp, table = _extend_case(gen, dev, [6] * n, lens, 14, 2, 64)
        extend.append((q, k, v, torch.tensor(_starts([6] * n), dtype=torch.int32, device=dev), 6,
                       torch.tensor(lens, device=dev), None, None, kp, vp, table.to(dev)))
    calls = [(f, args) for f, a in ((paged.flash_decode_attention_prefix_paged, decode),
                                    (paged.prefill_extend_paged, extend)) for args in a]
    want = [f(*args) for f, args in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    got = []
    for _ in range(5):
        for s, (f, args) in zip(streams, calls):
            with torch.cuda.stream(s):
                got.append(f(*args))
    torch.cuda.synchronize()
    for i, w in enumerate(want):
        assert all(torch.equal(g, w) for g in got[i::len(calls)])


def test_extension_refusals(dev):
    gen = torch.Generator().manual_seed(36)
    q, k, v, kp, vp, table = _extend_case(gen, dev, [4, 6], [10, 20], 14, 2, 64)
    cu = torch.tensor([0, 4, 10], dtype=torch.int32, device=dev)
    ok = dict(query=q, key=k, value=v, cu_seqlens=cu, max_seqlen=6, context=torch.tensor([10, 20], device=dev),
              cos=None, sin=None, k_pool=kp, v_pool=vp, block_table=table.to(dev))
    paged.prefill_extend_paged(**ok)
    cs = torch.zeros(10, 64, device=dev, dtype=torch.float16)
    for change, kind in ((dict(query=q.float()), TypeError), (dict(key=k[:5]), ValueError),
                         (dict(query=q[:, :13]), ValueError), (dict(cu_seqlens=cu.long()), TypeError),
                         (dict(cu_seqlens=cu[:2]), ValueError), (dict(max_seqlen=5), ValueError),
                         (dict(max_seqlen=0), ValueError), (dict(context=ok["context"].int()), TypeError),
                         (dict(context=ok["context"][:1]), ValueError), (dict(cos=cs), ValueError),
                         (dict(cos=cs[:5], sin=cs[:5]), ValueError), (dict(max_slots=65), ValueError),
                         (dict(max_slots=3), ValueError), (dict(block_table=table.to(dev)[:1]), ValueError),
                         (dict(lengths=[4, 5]), ValueError), (dict(scale=0.0), RuntimeError),
                         (dict(k_pool=kp[:, :1], v_pool=vp[:, :1]), ValueError)):
        with pytest.raises(kind):
            paged.prefill_extend_paged(**{**ok, **change})
