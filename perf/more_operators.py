"""The operators of a paged cache held in 8 bits, over the range their users put them to.

A page of a kv head holds 64-dim keys slot by slot and values dim by dim in
groups of 64 slots, as int8 or e4m3 codes, and a scale for each 16 slots: a power
of two, at least 2^-24, so that a code's value is exact.  A block's scale is the
least one at which its tokens fit; where later tokens need a larger one, the codes
already there are rounded to it.

The model shape is the Qwen2.5-0.5B one of ``qwenforge_amd.model.Qwen2Config``
(14 query heads over 2 kv heads of 64) unless a case says otherwise.  Kinds of case:

* ``append`` -- one layer's new tokens quantised into their pages.  Returned are the
  pools: int8 codes, or e4m3 values, and their scales.
* ``read`` -- slots of rows back in fp16, packed.
* ``decode`` -- one layer's attention of a batch of single tokens.
* ``extend`` -- one layer's new tokens appended and attended with the slots before them.
"""

import math

import torch

own = False

D = 64
BLOCK = 16
DEV = "cuda"
CODE = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
LARGEST = {"int8": 127.0, "e4m3": 448.0}


# --------------------------------------------------------------------------
# the cases
# --------------------------------------------------------------------------

def listed():
    return [
        # One chat's decoding step.
        dict(name="append_step_b1", kind="append", code="int8", batch=1, kv_heads=2, page=64, lo=1, hi=1,
             clo=777, chi=777),
        # A serving batch's decoding step, every row at a length of its own, two rows free.
        dict(name="append_step_b32", kind="append", code="e4m3", batch=32, kv_heads=2, page=64, lo=1, hi=1,
             clo=33, chi=4001, parked=2),
        # The own prompts of requests behind a system prompt that ends inside a block.
        dict(name="append_b16_ragged", kind="append", code="int8", batch=16, kv_heads=2, page=64, lo=9,
             hi=301, clo=1031, chi=1031),
        # Four long prompts.
        dict(name="append_b4_8192", kind="append", code="e4m3", batch=4, kv_heads=2, page=256, lo=8192,
             hi=8192, clo=0, chi=0),
        # One row taken out, to be kept elsewhere.
        dict(name="read_b1_300", kind="read", code="e4m3", batch=1, kv_heads=2, page=64, lo=300, hi=300,
             clo=0, chi=0),
        # Long rows moved to a cache in fp16.
        dict(name="read_b16_16384", kind="read", code="int8", batch=16, kv_heads=2, page=64, lo=9001,
             hi=16384, clo=0, chi=0),
        # One chat.
        dict(name="decode_b1_1024", kind="decode", code="int8", batch=1, heads=14, kv_heads=2, page=64,
             lo=1024, hi=1024),
        # A serving batch, two rows free.
        dict(name="decode_b24_ragged", kind="decode", code="e4m3", batch=24, heads=14, kv_heads=2, page=64,
             lo=33, hi=4096, parked=2),
        # Many long documents at once, as the memory saved allows.
        dict(name="decode_b64_32768", kind="decode", code="int8", batch=64, heads=14, kv_heads=2, page=256,
             lo=30001, hi=32768),
        # Four chats with four drafted tokens each.
        dict(name="extend_drafts_b4", kind="extend", code="int8", batch=4, heads=14, kv_heads=2, page=64,
             lo=5, hi=5, clo=300, chi=2011),
        # The own prompts of requests behind a system prompt.
        dict(name="extend_b16_ragged", kind="extend", code="e4m3", batch=16, heads=14, kv_heads=2, page=64,
             lo=9, hi=301, clo=2048, chi=2048),
        # A chunk of a long prompt.
        dict(name="extend_chunk_2048", kind="extend", code="int8", batch=1, heads=14, kv_heads=2, page=64,
             lo=2048, hi=2048, clo=16384, chi=16384),
    ]


def _log_int(rng, lo, hi):
    """Whole number spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["append", "read", "decode", "extend"])
    kv_heads = rng.choice([1, 2, 2, 2, 4, 8])
    case = dict(kind=kind, code=rng.choice(["int8", "e4m3"]), kv_heads=kv_heads,
                page=rng.choice([64, 64, 64, 128, 256]))
    if kind in ("append", "read"):
        batch = _log_int(rng, 1, 64)
        hi = _log_int(rng, 1, max(1, min(16384, (60_000 if kind == "append" else 200_000) // (batch * kv_heads))))
        chi = rng.choice([0, _log_int(rng, 1, max(1, min(16384, 400_000 // (batch * kv_heads))))])
        return dict(case, batch=batch, lo=int(hi * rng.uniform(0.0, 1.0)), hi=hi,
                    clo=int(chi * rng.uniform(0.0, 1.0)), chi=chi,
                    parked=rng.choice([0, 0, 1]) if kind == "append" else 0)
    heads = kv_heads * rng.choice([1, 4, 7, 7, 7, 8, 16])
    if kind == "decode":
        batch = _log_int(rng, 1, 96)
        hi = _log_int(rng, 1, min(65536, 3_000_000 // (batch * kv_heads)))
        return dict(case, heads=heads, batch=batch, lo=max(1, int(hi * rng.uniform(0.02, 1.0))), hi=hi,
                    parked=rng.choice([0, 0, 1]))
    batch = _log_int(rng, 1, 32)
    hi = _log_int(rng, 1, min(2048, 8192 // batch, math.isqrt(400_000_000 // (batch * heads))))
    chi = _log_int(rng, 1, max(1, min(32768, 400_000_000 // (batch * hi * heads),
                                      6_000_000 // (batch * kv_heads))))
    return dict(case, heads=heads, batch=batch, lo=int(hi * rng.uniform(0.0, 1.0)), hi=hi,
                clo=int(chi * rng.uniform(0.0, 1.0)), chi=chi)


def _spread(n, lo, hi):
    """n whole numbers evenly over [lo, hi], in an order that is not sorted; ``hi`` is one of them."""
    if n == 1:
        return [hi]
    row = [lo + (hi - lo) * i // (n - 1) for i in range(n)]
    return row[1::2] + row[0::2][::-1]


def _rows(case):
    """(new or read tokens, slots before them) of each row; a free row has -1 before it."""
    b = case["batch"]
    if case["kind"] == "decode":
        new, ctx = [0] * b, _spread(b, case["lo"], case["hi"])
    else:
        new, ctx = _spread(b, case["lo"], case["hi"]), _spread(b, case["clo"], case["chi"])
    for r in range(min(case.get("parked", 0), b - 1)):
        ctx[b - 1 - r] = -1
    return new, ctx


def _ints(values, dtype):
    return torch.tensor(values, dtype=dtype).to(DEV)


# --------------------------------------------------------------------------
# codes and scales
# --------------------------------------------------------------------------

def _scale_for(top, code):
    """The least power of two, 2^-24 or more, at which ``top`` >= 0 (fp32) fits; NaN where it is not finite."""
    m, e = torch.frexp(top)                                    # top = m 2^e, m in [0.5, 1)
    m0, e0 = math.frexp(LARGEST[code])
    e = torch.where(top == 0, torch.full_like(e, -99), e - e0 + (m > m0).int())
    s = torch.ldexp(torch.ones_like(top), e.clamp(min=-24))
    return torch.where(torch.isfinite(top), s, torch.full_like(s, math.nan))


def _encode(x, s, code):
    """Codes, as bytes, of fp32 values x at scales s; no value past what fp16 holds."""
    y = x / s
    if code == "int8":
        top = torch.floor(65504.0 / s).clamp(max=127.0)
        return torch.minimum(torch.maximum(torch.round(y), -top), top).to(torch.int8).view(torch.uint8)
    top = torch.where(s >= 256.0, torch.full_like(s, 240.0), torch.full_like(s, 448.0))
    return torch.minimum(torch.maximum(y, -top), top).to(torch.float8_e4m3fn).view(torch.uint8)


def _decode(c, code):
    """fp32 values of codes given as bytes."""
    return c.contiguous().view(CODE[code]).float()


def _bytes(pool):
    return pool.view(torch.uint8)


# --------------------------------------------------------------------------
# what a user's program has in hand
# --------------------------------------------------------------------------

def _rand(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEV, dtype=torch.float32)


def _channels(gen, kv_heads):
    """Sizes of a head's key channels: some a few times the others, as models have them."""
    return 1.0 + 5.0 * (torch.rand(kv_heads, 1, D, generator=gen, device=DEV) > 0.94)


def _new_pools(gen, code, n_pages, kv_heads, page):
    """Pages full of quantised keys and values: views of one record of bytes for each page."""
    per, blocks = kv_heads * page * D, kv_heads * page // BLOCK
    store = torch.zeros(n_pages, 2 * per + 8 * blocks, dtype=torch.uint8, device=DEV)
    k, v = store[:, :per], store[:, per:2 * per]
    pools = (k.view(CODE[code]).view(n_pages, kv_heads, page, D),
             v.view(CODE[code]).view(n_pages, kv_heads, page // 64, D, 64),
             store[:, 2 * per:2 * per + 4 * blocks].view(torch.float32).view(n_pages, kv_heads, page // BLOCK),
             store[:, 2 * per + 4 * blocks:].view(torch.float32).view(n_pages, kv_heads, page // BLOCK))
    spread = _channels(gen, kv_heads)
    step = max(1, 8_000_000 // per)
    for at in range(0, n_pages, step):
        n = min(step, n_pages - at)
        here = slice(at, at + n)
        for which in (0, 1):
            x = _rand(gen, n, kv_heads, page, D)
            x = (x * spread if which == 0 else x).half().float()
            blocked = x.view(n, kv_heads, page // BLOCK, BLOCK * D)
            s = _scale_for(blocked.abs().amax(dim=-1), code)
            c = _encode(blocked, s[..., None], code)
            pools[2 + which][here] = s
            if which == 0:
                k[here] = c.view(n, per)
            else:
                v[here] = c.view(n, kv_heads, page // 64, 64, D).transpose(3, 4).reshape(n, per)
    return pools, spread


def prepare(case, seed):
    gen = torch.Generator(DEV).manual_seed(seed)
    kvh, page, b = case["kv_heads"], case["page"], case["batch"]
    new, ctx = _rows(case)
    need = [max(1, -(-(n + max(c, 0)) // page)) for n, c in zip(new, ctx)]
    ppr, n_pages, total = max(need), sum(need) + 2, sum(new)
    perm = torch.randperm(n_pages, generator=gen, device=DEV).to(torch.int32)
    at = [sum(need[:r]) for r in range(b)]
    table = torch.full((b, ppr), -1, dtype=torch.int32, device=DEV)
    for r, n in enumerate(need):
        if ctx[r] >= 0:
            table[r, :n] = perm[at[r]:at[r] + n]
    pools, spread = _new_pools(gen, case["code"], n_pages, kvh, page)
    s = dict(case=case, pools=pools, table=table)
    if case["kind"] == "decode":
        q = _rand(gen, b, kvh, case["heads"] // kvh, D).half()
        return dict(s, q=q, last=_ints([c - 1 if c >= 0 else -1 for c in ctx], torch.int64))
    s.update(cu=_ints([sum(new[:r]) for r in range(b + 1)], torch.int32), lens=new, longest=max(new),
             ctx=_ints(ctx, torch.int64), total=total)
    if case["kind"] == "read":
        return s
    qh = case.get("heads", 0)
    # The fused projection's rows: heads of q, then of k, then of v.
    qkv = _rand(gen, total, qh + 2 * kvh, D)
    qkv[:, qh:qh + kvh] *= spread[:, 0]
    qkv = qkv.half()
    return dict(s, q=qkv[:, :qh], k=qkv[:, qh:qh + kvh], v=qkv[:, qh + kvh:],
                most=max(n + c for n, c in zip(new, ctx)))


# --------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------

def run(s):
    if own:
        return _own(s)
    return _plain(s)


def _own(s):
    return {"append": _own_append, "read": _own_read, "decode": _own_decode,
            "extend": _own_extend}[s["case"]["kind"]](s)


def _plain(s):
    return {"append": _plain_append, "read": _plain_read, "decode": _plain_decode,
            "extend": _plain_extend}[s["case"]["kind"]](s)


def _own_append(s):
    from qwenforge_amd import paged8

    paged8.append_paged8(s["k"], s["v"], s["cu"], s["longest"], s["ctx"], None, None, s["pools"], s["table"],
                         lengths=s["lens"])
    return s["pools"]


def _own_read(s):
    from qwenforge_amd import paged8

    return paged8.read_paged8(s["pools"], s["table"], s["cu"], s["longest"], s["ctx"], lengths=s["lens"])


def _own_decode(s):
    from qwenforge_amd import paged8

    return paged8.flash_decode_attention_paged8(s["q"], s["pools"], s["table"], s["last"])


def _own_extend(s):
    from qwenforge_amd import paged8

    out = paged8.prefill_extend_paged8(s["q"], s["k"], s["v"], s["cu"], s["longest"], s["ctx"], None, None,
                                       s["pools"], s["table"], lengths=s["lens"], max_slots=s["most"])
    return (out, *s["pools"])


def _places(s):
    """Of each token: its row, its slot, page and place in the page."""
    cu, page = s["cu"].long(), s["case"]["page"]
    token = torch.arange(s["total"], device=DEV)
    row = torch.searchsorted(cu, token, right=True) - 1
    slot = s["ctx"][row] + token - cu[row]
    return row, slot, s["table"][row, slot.clamp(min=0) // page].long(), slot % page


def _plain_append(s):
    code, page, kvh = s["case"]["code"], s["case"]["page"], s["case"]["kv_heads"]
    row, slot, where, off = _places(s)
    mine = s["ctx"][row] >= 0
    row, slot, where, off = row[mine], slot[mine], where[mine], off[mine]
    per = page // BLOCK
    block = where * per + off // BLOCK                                     # (T,)
    n = s["pools"][0].shape[0] * per
    # The block of each row that holds earlier slots, if it does.
    ctx, counts = s["ctx"], s["cu"][1:] - s["cu"][:-1]
    begun = (ctx > 0) & (ctx % BLOCK != 0) & (counts > 0)
    ctx = ctx[begun]
    first = s["table"][begun].gather(1, (ctx // page)[:, None])[:, 0].long()
    fb = ctx % page // BLOCK
    kept = torch.arange(BLOCK, device=DEV) < (ctx % BLOCK)[:, None]        # (rows, 16)
    slots = fb[:, None] * BLOCK + torch.arange(BLOCK, device=DEV)          # (rows, 16), in the page
    for which, new in ((0, s["k"][mine].float()), (1, s["v"][mine].float())):
        pool, scale = _bytes(s["pools"][which]), s["pools"][2 + which]
        top = torch.zeros(n, kvh, device=DEV).scatter_reduce_(0, block[:, None].expand(-1, kvh),
                                                              new.abs().amax(dim=-1), "amax")
        old = torch.zeros(n, kvh, device=DEV)
        was = scale[first, :, fb]                                          # (rows, kvh)
        old[first * per + fb] = was
        want = torch.maximum(old, _scale_for(top, code))
        # What the first blocks hold, at their new scales.
        if which == 0:
            have = pool[first[:, None], :, slots]                          # (rows, 16, kvh, D)
        else:
            have = pool[first[:, None], :, slots // 64, :, slots % 64]
        now = want[first * per + fb]
        turned = _encode(_decode(have, code) * was[:, None, :, None], now[:, None, :, None], code)
        have = torch.where(kept[:, :, None, None] & (now > was)[:, None, :, None], turned, have)
        codes = _encode(new, want[block][:, :, None], code)
        if which == 0:
            pool[first[:, None], :, slots] = have
            pool[where, :, off] = codes
        else:
            pool[first[:, None], :, slots // 64, :, slots % 64] = have
            pool[where, :, off // 64, :, off % 64] = codes
        scale[where, :, off // BLOCK] = want[block]
    return s["pools"]


def _plain_read(s):
    code = s["case"]["code"]
    _, _, where, off = _places(s)
    k, v, ks, vs = s["pools"]
    block = off // BLOCK
    k = _decode(_bytes(k)[where, :, off], code) * ks[where, :, block][..., None]
    v = _decode(_bytes(v)[where, :, off // 64, :, off % 64], code) * vs[where, :, block][..., None]
    return k.half(), v.half()


def _rows_of(s):
    """K and V (rows, kv heads, slots, 64) fp32 of the rows' pages; pages not mapped read as some page."""
    code, page = s["case"]["code"], s["case"]["page"]
    k, v, ks, vs = s["pools"]
    at = s["table"].clamp(min=0).long()
    b, ppr = at.shape
    got = []
    for which, pool, scale in ((0, k, ks), (1, v, vs)):
        x = _decode(_bytes(pool)[at], code)
        if which == 1:
            x = x.transpose(-1, -2)                                        # groups of 64 slots, dims
        x = x.reshape(b, ppr, -1, page // BLOCK, BLOCK * D) * scale[at][..., None]
        got.append(x.view(b, ppr, -1, page, D).transpose(1, 2).reshape(b, -1, ppr * page, D))
    return got


def _attend(q, k, v, seen):
    """softmax(q k^T / 8) v in fp32 over the ``seen`` slots; zero where there are none.
    q (B, KVH, R, D), k and v (B, KVH, N, D), seen broadcast to (B, KVH, R, N)."""
    scores = torch.matmul(q, k.transpose(2, 3).contiguous()) * D ** -0.5
    scores = scores.masked_fill_(~seen, -math.inf)
    top = scores.amax(dim=-1, keepdim=True)
    p = torch.exp_(scores.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)))
    total = p.sum(dim=-1, keepdim=True)
    return torch.where(total > 0, torch.matmul(p, v) / total, torch.zeros_like(total))


def _plain_decode(s):
    k, v = _rows_of(s)
    seen = torch.arange(k.shape[2], device=DEV) <= s["last"][:, None]
    return _attend(s["q"].float(), k, v, seen[:, None, None, :]).half()


def _plain_extend(s):
    _plain_append(s)
    case, cu, ctx = s["case"], s["cu"].long(), s["ctx"]
    b, longest, kvh = case["batch"], s["longest"], case["kv_heads"]
    g, total = case["heads"] // kvh, s["q"].shape[0]
    token = torch.arange(total, device=DEV)
    row = torch.searchsorted(cu, token, right=True) - 1
    at = token - cu[row]
    k, v = _rows_of(s)
    # Rows side by side, padded to the longest.
    q = torch.zeros(b, longest, case["heads"], D, device=DEV)
    q[row, at] = s["q"].float()
    q = q.view(b, longest, kvh, g, D).permute(0, 2, 3, 1, 4).reshape(b, kvh, g * longest, D)
    last = ctx[:, None] + torch.arange(longest, device=DEV)                # (B, longest)
    seen = torch.arange(k.shape[2], device=DEV) <= last[:, :, None]
    seen = seen[:, None, None].expand(b, 1, g, longest, k.shape[2]).reshape(b, 1, g * longest, -1)
    out = _attend(q, k, v, seen).view(b, kvh, g, longest, D).permute(0, 3, 1, 2, 4)
    return (out.reshape(b, longest, case["heads"], D)[row, at].half(), *s["pools"])


# --------------------------------------------------------------------------
# what a pass cannot do without
# --------------------------------------------------------------------------

def work(case):
    new, ctx = _rows(case)
    kvh, heads = case["kv_heads"], case.get("heads", 0)
    slot = 2.0 * D + 8.0 / BLOCK                    # bytes of a slot's K and V and its share of the scales
    if case["kind"] == "decode":
        live = [c for c in ctx if c > 0]
        return {"bytes": kvh * slot * sum(live) + 4.0 * D * case["batch"] * heads,
                "flops": 4.0 * D * heads * sum(live)}
    live = [(n, c) for n, c in zip(new, ctx) if c >= 0 and n > 0]
    total = sum(n for n, _ in live)
    moved = kvh * total * (4.0 * D + slot)          # fp16 on one side, codes on the other
    if case["kind"] == "read":
        return {"bytes": moved, "flops": 0}
    begun = kvh * slot * sum(c % BLOCK for _, c in live)
    if case["kind"] == "append":
        return {"bytes": moved + begun, "flops": 0}
    return {"bytes": moved + kvh * slot * sum(c for _, c in live) + 4.0 * D * heads * total,
            "flops": 4.0 * D * heads * sum(n * c + n * (n + 1) // 2 for n, c in live)}


# --------------------------------------------------------------------------
# the same from the definition, in 64 bits
# --------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "append":
        return _exact_append(case, s)
    if case["kind"] == "read":
        return _exact_read(case, s)
    if case["kind"] == "decode":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
        for r, last in enumerate(s["last"].tolist()):
            if last >= 0:
                out[r] = _softmax_of(s["q"][r].double(), *_dense(s["pools"], s["table"][r], 0, last + 1), None)
        return out
    return _exact_extend(case, s)


def _dense(pools, pages, lo, hi):
    """K and V (KVH, hi - lo, 64) in 64 bits of slots [lo, hi) of a row's pages."""
    k, v, ks, vs = pools
    slot = torch.arange(lo, hi, device=DEV)
    where, off = pages[slot // k.shape[2]].long(), slot % k.shape[2]
    kk = k.view(torch.uint8)[where, :, off].view(k.dtype).double()
    vv = v.view(torch.uint8)[where, :, off // 64, :, off % 64].view(v.dtype).double()
    kk *= ks[where, :, off // 16].double()[..., None]
    vv *= vs[where, :, off // 16].double()[..., None]
    return kk.transpose(0, 1), vv.transpose(0, 1)


def _softmax_of(q, k, v, seen):
    """q (..., R, D) over k, v (..., N, D), all in 64 bits; seen (R, N) or None."""
    scores = torch.matmul(q, k.transpose(-1, -2).contiguous()) / 8.0
    if seen is not None:
        scores = scores.masked_fill(~seen, -math.inf)
    return torch.matmul(torch.softmax(scores, dim=-1), v.contiguous())


def _nearest(x, s, code):
    """The value of the code nearest to x / s, ties to the even one, that stays within fp16."""
    mag = x.abs() / s
    if code == "int8":
        levels = torch.arange(0, 128, dtype=torch.float64, device=DEV)
    else:
        levels = torch.tensor([(c % 8) * 2.0 ** -9 if c < 8 else (1 + c % 8 / 8) * 2.0 ** (c // 8 - 7)
                               for c in range(127)], dtype=torch.float64, device=DEV)
    i = torch.searchsorted((levels[1:] + levels[:-1]) / 2, mag.contiguous())
    up = torch.clamp(i + 1, max=len(levels) - 1)
    i = torch.where((mag == (levels[i] + levels[up]) / 2) & (i % 2 == 1), up, i)
    most = torch.searchsorted(levels, 65504.0 / s, right=True) - 1
    return torch.copysign(levels[torch.minimum(i, most.expand_as(i))], x)


def _least_scale(top, code):
    """The first of 2^-24, 2^-23 .. that holds ``top`` (fp64)."""
    steps = torch.tensor([2.0 ** e for e in range(-24, 17)], dtype=torch.float64, device=DEV)
    return steps[torch.searchsorted(steps * (127 if code == "int8" else 448), top)]


def _append_row(values, scales, pages, first, new, code, dims_first):
    """One row's new tokens (n, KVH, 64) in 64 bits written at slot ``first``; ``values`` are the pool's codes."""
    page = scales.shape[2] * 16
    lo, hi = first // 16 * 16, first + new.shape[0]
    end = -(-hi // 16) * 16
    slot = torch.arange(lo, end, device=DEV)
    where, off = pages[torch.clamp(slot, max=pages.numel() * page - 1) // page].long(), slot % page
    at = (where, slice(None), off // 64, slice(None), off % 64) if dims_first else (where, slice(None), off)
    have = values[at]                                                       # (slots, KVH, 64)
    old = scales[where, :, off // 16].double().view(-1, 16, *have.shape[1:2])[:, 0]      # (blocks, KVH)
    fresh = torch.zeros_like(have)
    fresh[first - lo:hi - lo] = new
    need = _least_scale(fresh.abs().view(-1, 16, *have.shape[1:]).amax(dim=(1, 3)), code)
    s = need.clone()
    if first > lo:
        s[0] = torch.maximum(s[0], old[0])
    full = s.repeat_interleave(16, dim=0)[..., None]
    was = old.repeat_interleave(16, dim=0)[..., None]
    turned = _nearest(have * was, full, code)
    codes = torch.where((slot < first)[:, None, None], turned, _nearest(fresh, full, code))
    values[at] = torch.where((slot < hi)[:, None, None], codes, have)
    scales[where[::16], :, off[::16] // 16] = s.to(scales.dtype)


def _exact_pools(case, s):
    code = case["code"]
    got = []
    for which, name in ((0, "k"), (1, "v")):
        values = s["pools"][which].view(CODE[code]).double()
        scales = s["pools"][2 + which].double()
        cu = s["cu"].tolist()
        for r, c in enumerate(s["ctx"].tolist()):
            if c >= 0 and cu[r + 1] > cu[r]:
                _append_row(values, scales, s["table"][r], c, s[name][cu[r]:cu[r + 1]].double(), code, which == 1)
        got.append((values, scales))
    return got


def _as_held(case, got):
    (k, ks), (v, vs) = got
    if case["code"] == "int8":
        k, v = k.to(torch.int8), v.to(torch.int8)
    return k, v, ks, vs


def _exact_append(case, s):
    return _as_held(case, _exact_pools(case, s))


def _exact_read(case, s):
    parts = [_dense(s["pools"], s["table"][r], c, c + n)
             for r, (c, n) in enumerate(zip(s["ctx"].tolist(), s["lens"])) if n > 0]
    return tuple(torch.cat([p[i].transpose(0, 1) for p in parts]) for i in (0, 1))


def _exact_extend(case, s):
    got = _exact_pools(case, s)
    kvh, page = case["kv_heads"], case["page"]
    g, out, cu = case["heads"] // kvh, torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV), s["cu"].tolist()
    for r, c in enumerate(s["ctx"].tolist()):
        if cu[r + 1] == cu[r]:
            continue
        slot = torch.arange(c + cu[r + 1] - cu[r], device=DEV)
        where, off = s["table"][r][slot // page].long(), slot % page
        (kc, ks), (vc, vs) = got
        k = (kc[where, :, off] * ks[where, :, off // 16][..., None]).transpose(0, 1)
        v = (vc[where, :, off // 64, :, off % 64] * vs[where, :, off // 16][..., None]).transpose(0, 1)
        for lo in range(cu[r], cu[r + 1], 256):
            hi = min(lo + 256, cu[r + 1])
            first = c + lo - cu[r]
            n = first + hi - lo
            seen = slot[:n] <= first + torch.arange(hi - lo, device=DEV)[:, None]
            for h in range(kvh):
                q = s["q"][lo:hi, h * g:(h + 1) * g].double().transpose(0, 1).contiguous()   # (g, rows, D)
                out[lo:hi, h * g:(h + 1) * g] = _softmax_of(q, k[h, :n], v[h, :n], seen).transpose(0, 1)
    return (out, *_as_held(case, got))
