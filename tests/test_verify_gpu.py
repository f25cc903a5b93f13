"""``verify.verify_drafts`` against its definition in 64 bits: counts and tokens
are whole numbers and have to be equal.

Random cases stay clear of their borders: a case's numbers decide a token only
if every acceptance is 1e-5 away from equality (the kernel's p is off by less
than 2^-20 relative: fp32 exponentials of arguments rounded to 2^-24 of at most
about 40, summed in 64 bits) and every draw 1e-12 away from a running sum (64
bits, 2e5 terms).  The reference says so of each case before the kernel runs.
"""

import math

import numpy as np
import pytest
import torch

from qwenforge_amd import verify

pytestmark = pytest.mark.gpu


def _draw(w, r):
    reach = np.cumsum(w)
    mark = r * reach[-1]
    i = min(int(np.searchsorted(reach, mark, side="right")), int(np.flatnonzero(w)[-1]))
    return i, np.abs(reach[w > 0] - mark).min() / reach[-1]


def _row(x, toks, u, r, temp, q):
    """New tokens of one row (x (n, V) float64, toks (n,)) and how far it stays from a border."""
    n, v = x.shape
    out, clear = [], math.inf
    for j in range(n):
        draft = int(toks[j + 1]) if j + 1 < n else None
        top = x[j].max()
        if temp == 0:
            if not top > -math.inf:
                return out, clear
            best = int(np.argmax(x[j]))
            out.append(best)
            if draft != best:
                return out, clear
            continue
        if not math.isfinite(top):
            return out, clear
        p = np.exp((x[j] - top) / temp)
        p /= p.sum()
        qj = None
        if draft is not None:
            qj = np.zeros(v)
            if 0 <= draft < v:
                qj[draft] = 1.0
            if q is not None:
                qj = q[j]
            if 0 <= draft < v:
                clear = min(clear, abs(u[j] * qj[draft] - p[draft]) / max(p[draft], 1e-30) / 1e-5)
                if u[j] * qj[draft] < p[draft]:
                    out.append(draft)
                    continue
        w = p if qj is None else np.maximum(p - qj, 0)
        if not w.sum() > 0:
            w = p
        i, gap = _draw(w, r)
        clear = min(clear, gap / 1e-12)
        out.append(i)
        return out, clear
    return out, clear


def _expect(logits, tokens, lens, u, r, temp, probs, width):
    x, q = logits.double().cpu().numpy(), None if probs is None else probs.double().cpu().numpy()
    tokens = tokens.cpu().numpy()
    u, r = (None if t is None else t.double().cpu().numpy() for t in (u, r))
    rows, counts, at = [], [], 0
    for b, n in enumerate(lens):
        s = slice(at, at + n)
        new, clear = ([], math.inf) if n == 0 else _row(
            x[s], tokens[s], None if u is None else u[s], None if r is None else r[b], temp,
            None if q is None else q[s])
        assert clear > 1, "the case stands on a border: choose another seed"
        rows.append(new + [-1] * (width - len(new)))
        counts.append(len(new))
        at += n
    return torch.tensor(counts), torch.tensor(rows)


def _case(gen, dev, lens, v, dtype, temp, drafter, sigma=2.0, near=0.3):
    t = sum(lens)
    logits = torch.randn(t, v, generator=gen) * sigma
    like = logits + torch.randn(t, v, generator=gen) * near
    probs = torch.softmax(like / (temp or 1.0), dim=-1)
    picked = torch.multinomial(probs, 1, generator=gen)[:, 0] if drafter else like.argmax(dim=-1)
    tokens = torch.cat([torch.zeros(1, dtype=torch.int64), picked[:-1]])
    u, r = torch.rand(t, generator=gen), torch.rand(len(lens), generator=gen)
    put = lambda x: x.to(dev)  # noqa: E731
    return put(logits.to(dtype)), put(tokens), put(u), put(r), put(probs) if drafter else None


def _cu(lens, dev):
    return torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=dev)


@pytest.mark.parametrize("v", [1, 7, 2041, 2048, 2049, 10007, 151936])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("temp,drafter", [(0.0, False), (1.0, False), (0.7, True), (1.3, True)])
def test_matches_definition(dev, v, dtype, temp, drafter):
    gen = torch.Generator().manual_seed(v + int(10 * temp))
    lens = [5, 1, 3, 2, 8] if v < 100000 else [4, 1, 2]
    logits, tokens, u, r, probs = _case(gen, dev, lens, v, dtype, temp, drafter)
    want = _expect(logits, tokens, lens, u, r, temp, probs, max(lens))
    got = verify.verify_drafts(logits, tokens, _cu(lens, dev), max(lens), u, r, temperature=temp,
                               draft_probs=probs, lengths=lens)
    assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])


@pytest.mark.parametrize("offset", [1, 3, 8])
def test_strided_rows_that_start_anywhere(dev, offset):
    gen = torch.Generator().manual_seed(offset)
    lens = [3, 4, 0, 2]
    for dtype in (torch.float16, torch.float32):
        logits, tokens, u, r, probs = _case(gen, dev, lens, 5003, dtype, 0.9, True)
        wide = torch.full((9, 5003 + 20), math.inf, device=dev, dtype=dtype)
        wide[:, offset:offset + 5003] = logits
        wide_p = torch.full((9, 5003 + 11), math.nan, device=dev)
        wide_p[:, offset:offset + 5003] = probs
        for temp in (0.9, 0.0):
            want = _expect(logits, tokens, lens, u, r, temp, probs, 4)
            got = verify.verify_drafts(wide[:, offset:offset + 5003], tokens, _cu(lens, dev), 4, u, r,
                                       temperature=temp, draft_probs=wide_p[:, offset:offset + 5003])
            assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])


def test_borders_are_strict(dev):
    """Equal logits make p exact: u q = p rejects, a running sum equal to the mark is passed over."""
    x = torch.zeros(8, 4, device=dev)
    tokens = torch.tensor([9, 2, 9, 2, 9, 2, 9, 2], device=dev)
    u = torch.tensor([0.25, 0, 0.25 - 2**-26, 0, 0, 0, 1 - 2**-24, 0], device=dev)
    r = torch.tensor([0.0, 0.25, 0.5, 1 - 2**-24], device=dev)
    count, out = verify.verify_drafts(x, tokens, _cu([2, 2, 2, 2], dev), 2, u, r)
    # Row 0 rejects 2, draws from {0, 1, 3} at 0; row 3 at the end.
    assert out.tolist() == [[0, -1], [2, 1], [2, 2], [3, -1]]
    assert count.tolist() == [1, 2, 2, 1]


def test_ties_go_to_the_lowest_token(dev):
    x = torch.zeros(2, 100003, device=dev, dtype=torch.float16)
    x[0, [70001, 40007, 99999]] = 3.0
    x[1, 65536:] = 1.0
    count, out = verify.verify_drafts(x, torch.tensor([0, 40007], device=dev), _cu([2], dev), 2, None, None,
                                      temperature=0.0)
    assert out.tolist() == [[40007, 65536]] and count.tolist() == [2]


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_masked_and_unusable_logits(dev, dtype):
    v = 3001
    x = torch.full((6, v), -math.inf, device=dev, dtype=dtype)
    x[0, 2999] = -7.0                                   # one token left
    x[2] = 0.5
    x[2, 5] = math.nan
    x[3] = 0.5
    x[3, 7] = math.inf
    x[4] = torch.finfo(dtype).min                       # the type's lowest value everywhere: all alike
    x[5, 17] = torch.finfo(dtype).max
    tokens = torch.zeros(6, dtype=torch.int64, device=dev)
    u, r = torch.full((6,), 0.5, device=dev), torch.full((6,), 0.5, device=dev)
    count, out = verify.verify_drafts(x, tokens, _cu([1] * 6, dev), 1, u, r)
    assert out[:, 0].tolist() == [2999, -1, -1, -1, 1500, 17]
    assert count.tolist() == [1, 0, 0, 0, 1, 1]
    count, out = verify.verify_drafts(x, tokens, _cu([1] * 6, dev), 1, None, None, temperature=0)
    assert out[:, 0].tolist() == [2999, -1, -1, 7, 0, 17] and count.tolist() == [1, 0, 0, 1, 1, 1]
    for at in (0, 1, 2047, 2048, v - 1):                # a NaN anywhere beside an infinity
        x[3, at], x[3, 7] = math.nan, math.inf
        _, out = verify.verify_drafts(x, tokens, _cu([1] * 6, dev), 1, None, None, temperature=0)
        assert out[:, 0].tolist() == [2999, -1, -1, -1, 0, 17]
        x[3, at] = 0.5
    # A draft in front of an unusable position: accepted, then nothing drawn.
    x2 = torch.stack([x[0], x[1]])
    count, out = verify.verify_drafts(x2, torch.tensor([1, 2999], device=dev), _cu([2], dev), 2, u[:2], r[:1])
    assert out.tolist() == [[2999, -1]] and count.tolist() == [1]


def test_drafts_outside_the_vocabulary_and_odd_numbers(dev):
    gen = torch.Generator().manual_seed(3)
    x = torch.randn(12, 50, generator=gen).to(dev)
    tokens = torch.tensor([0, -1, 0, 50, 0, 2**40, 0, -2**40, 0, 3, 0, 4], device=dev)
    u = torch.zeros(12, device=dev)
    u[8], u[10] = math.nan, -1.0
    r = torch.tensor([0.3, 0.3, 0.3, 0.3, 0.3, 2.0], device=dev)
    count, out = verify.verify_drafts(x, tokens, _cu([2] * 6, dev), 2, u, r)
    p = torch.softmax(x.double(), dim=-1).cpu().numpy()
    for b in range(4):
        assert out[b].tolist() == [_draw(p[2 * b], 0.3)[0], -1]
    w = p[8].copy()
    w[3] = 0
    assert out[4].tolist() == [_draw(w, np.float32(0.3).astype(np.float64))[0], -1]
    assert out[5].tolist() == [4, 49]                   # u below zero accepts, r past one ends at the last
    assert count.tolist() == [1, 1, 1, 1, 1, 2]


def test_nothing_left_of_p_draws_from_p(dev):
    gen = torch.Generator().manual_seed(4)
    x = torch.randn(2, 600, generator=gen).to(dev)
    probs = 3 * torch.softmax(x, dim=-1)                # above p everywhere
    tokens = torch.tensor([0, 11], device=dev)
    count, out = verify.verify_drafts(x, tokens, _cu([2], dev), 2, torch.full((2,), 0.9, device=dev),
                                      torch.full((1,), 0.41, device=dev), draft_probs=probs)
    p = torch.softmax(x.double(), dim=-1).cpu().numpy()[0]
    assert out.tolist() == [[_draw(p, float(np.float32(0.41)))[0], -1]] and count.tolist() == [1]


def test_tokens_are_distributed_as_the_target_says(dev):
    """16384 rows of one draft each over six tokens: the first new token follows
    p whatever q is.  Counts within 5 standard deviations (a chance of 1e-5 in
    all with random numbers; these are fixed)."""
    gen = torch.Generator().manual_seed(11)
    rows, v = 16384, 6
    p = torch.tensor([0.4, 0.05, 0.25, 0.1, 0.15, 0.05])
    q = torch.tensor([0.1, 0.3, 0.25, 0.2, 0.05, 0.1])
    for probs in (q.expand(2 * rows, v).contiguous().to(dev), None):
        draft = torch.multinomial(q, rows, replacement=True, generator=gen)
        tokens = torch.stack([torch.zeros_like(draft), draft], dim=1).reshape(-1).to(dev)
        u, r = torch.rand(2 * rows, generator=gen).to(dev), torch.rand(rows, generator=gen).to(dev)
        logits = p.log().expand(2 * rows, v).contiguous().to(dev)
        _, out = verify.verify_drafts(logits, tokens, _cu([2] * rows, dev), 2, u, r, draft_probs=probs)
        seen = torch.bincount(out[:, 0].cpu(), minlength=v).double() / rows
        assert ((seen - p.double()).abs() <= 5 * (p.double() * (1 - p.double()) / rows).sqrt()).all()


def test_captured_verification_follows_its_inputs(dev):
    gen = torch.Generator().manual_seed(21)
    lens = [3, 2, 4]
    logits, tokens, u, r, probs = _case(gen, dev, lens, 9001, torch.float16, 0.8, True)
    cu = _cu(lens, dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = verify.verify_drafts(logits, tokens, cu, 4, u, r, temperature=0.8, draft_probs=probs)
    for _ in range(3):
        for t, x in zip((logits, tokens, u, r, probs), _case(gen, dev, lens, 9001, torch.float16, 0.8, True)):
            t.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        want = _expect(logits, tokens, lens, u, r, 0.8, probs, 4)
        assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])


def test_two_streams_at_once(dev):
    gen = torch.Generator().manual_seed(22)
    lens = [4] * 6
    cases = [_case(gen, dev, lens, 30011, torch.float32, 1.0, True) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for s, (x, t, u, r, q) in zip(streams, cases):
            with torch.cuda.stream(s):
                got.append(verify.verify_drafts(x, t, _cu(lens, dev), 4, u, r, draft_probs=q, lengths=lens))
    torch.cuda.synchronize()
    for i, (x, t, u, r, q) in enumerate(cases):
        want = _expect(x, t, lens, u, r, 1.0, q, 4)
        for count, out in got[i::2]:
            assert torch.equal(count.cpu(), want[0]) and torch.equal(out.cpu(), want[1])


@pytest.mark.parametrize("lens", [[1, 2], [1, 1, 1]])
def test_rows_more_than_32_bits_apart(dev, lens):
    gen = torch.Generator().manual_seed(23)
    v = 2500
    x, tokens, u, r, q = _case(gen, dev, lens, v, torch.float16, 1.0, True)
    step = 2**31 + 8
    far_x = torch.empty(2 * step + v, device=dev, dtype=torch.float16).as_strided((3, v), (step, 1))
    far_q = torch.empty(2 * step + v, device=dev).as_strided((3, v), (step, 1))
    far_x.copy_(x), far_q.copy_(q)
    for probs, temp in ((far_q, 1.0), (None, 1.0), (None, 0.0)):
        count, out = verify.verify_drafts(far_x, tokens, _cu(lens, dev), 3, u, r, temperature=temp,
                                          draft_probs=probs)
        want = _expect(x, tokens, lens, u, r, temp, None if probs is None else q, 3)
        assert torch.equal(count.cpu(), want[0]) and torch.equal(out.cpu(), want[1])


@pytest.mark.parametrize("drafter", [False, True])
def test_more_chunks_than_threads(dev, drafter):
    """A vocabulary of which a thread adds up several chunks."""
    gen = torch.Generator().manual_seed(25)
    lens, v = [2, 1, 3], 1200007
    logits, tokens, u, r, probs = _case(gen, dev, lens, v, torch.float16, 1.0, drafter)
    count, out = verify.verify_drafts(logits, tokens, _cu(lens, dev), 3, u, r, draft_probs=probs)
    want = _expect(logits, tokens, lens, u, r, 1.0, probs, 3)
    assert torch.equal(count.cpu(), want[0]) and torch.equal(out.cpu(), want[1])


def test_more_positions_than_parts_to_go_round(dev):
    """One part to a position, and more rows than a workgroup has lanes."""
    gen = torch.Generator().manual_seed(24)
    lens = [1 + i % 9 for i in range(600)]
    logits, tokens, u, r, probs = _case(gen, dev, lens, 211, torch.float32, 0.9, True)
    count, out = verify.verify_drafts(logits, tokens, _cu(lens, dev), 9, u, r, temperature=0.9,
                                      draft_probs=probs, lengths=lens)
    want = _expect(logits, tokens, lens, u, r, 0.9, probs, 9)
    assert torch.equal(count.cpu(), want[0]) and torch.equal(out.cpu(), want[1])


def test_refusals(dev):
    x = torch.zeros(4, 10, device=dev)
    ok = dict(logits=x, tokens=torch.zeros(4, dtype=torch.int64, device=dev), cu_seqlens=_cu([2, 2], dev),
              max_seqlen=2, accept_u=torch.zeros(4, device=dev), sample_u=torch.zeros(2, device=dev))
    verify.verify_drafts(**ok)
    for change, kind in ((dict(logits=x.cpu()), RuntimeError), (dict(logits=x.double()), TypeError),
                         (dict(logits=x.bfloat16()), TypeError), (dict(logits=x[0]), ValueError),
                         (dict(logits=x.T), ValueError), (dict(logits=x[:, :0]), ValueError),
                         (dict(logits=x[:1].expand(4, 10)), RuntimeError),
                         (dict(tokens=ok["tokens"].int()), TypeError), (dict(tokens=ok["tokens"][:3]), ValueError),
                         (dict(cu_seqlens=_cu([2, 1], dev)), ValueError), (dict(cu_seqlens=_cu([1, 3], dev)), ValueError),
                         (dict(max_seqlen=0), ValueError), (dict(max_seqlen=5), ValueError),
                         (dict(accept_u=None), TypeError), (dict(sample_u=ok["sample_u"].double()), TypeError),
                         (dict(temperature=-1.0), ValueError), (dict(temperature=math.nan), ValueError),
                         (dict(temperature=math.inf), ValueError), (dict(temperature=1e-320), RuntimeError),
                         (dict(temperature=1e39), RuntimeError), (dict(draft_probs=[0.5]), TypeError),
                         (dict(draft_probs=x.half()), TypeError), (dict(draft_probs=x[:, :5]), ValueError)):
        with pytest.raises(kind):
            verify.verify_drafts(**{**ok, **change})
