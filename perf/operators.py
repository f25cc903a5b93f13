"""The operators of serving with shared prefixes and drafted tokens, over the range their users put them to.

The model shape is the Qwen2.5-0.5B one of ``qwenforge_amd.model.Qwen2Config``
(14 query heads over 2 kv heads of 64, 24 layers, vocab 151936) unless a case
says otherwise.  Kinds of case:

* ``copy`` -- pages of every layer's K and V pools copied to other pages: the
  partly filled last page of a forked row, or the moves of a compaction.
* ``prefix`` -- one layer's decode attention of a batch whose rows share long
  prefixes by groups.
* ``extend`` -- one layer's attention of new tokens behind cached ones: the own
  prompts of forked rows, a chunk of a long prompt, drafted tokens.
* ``verify`` -- drafted tokens against the target's logits.
"""

import math

import numpy as np
import torch

own = False

D = 64
DEV = "cuda"


# --------------------------------------------------------------------------
# the cases
# --------------------------------------------------------------------------

def listed():
    return [
        # One request forked: its partly filled last page, in every layer.
        dict(name="copy_fork_1", kind="copy", layers=24, kv_heads=2, page=64, pairs=1, slots=37),
        # A batch of requests forked from one of longer pages, each at its own length.
        dict(name="copy_fork_24", kind="copy", layers=24, kv_heads=2, page=256, pairs=24, slots=-1),
        # A pool compacted after many requests came and went.
        dict(name="copy_compact_700", kind="copy", layers=24, kv_heads=2, page=64, pairs=700, slots=0),
        # Four answers to one question, just begun.
        dict(name="prefix_b4_512", kind="prefix", batch=4, groups=1, parked=0, heads=14, kv_heads=2,
             page=64, plo=512, phi=512, lo=1, hi=40),
        # A serving batch over three system prompts, two rows free.
        dict(name="prefix_b24_groups", kind="prefix", batch=24, groups=3, parked=2, heads=14,
             kv_heads=2, page=64, plo=1024, phi=4096, lo=33, hi=1500),
        # Many questions about one long document.
        dict(name="prefix_b96_32768", kind="prefix", batch=96, groups=1, parked=0, heads=14,
             kv_heads=2, page=64, plo=32768, phi=32768, lo=17, hi=700),
        # Four chats with four drafted tokens each.
        dict(name="extend_drafts_b4", kind="extend", batch=4, heads=14, kv_heads=2, page=64, lo=5, hi=5,
             clo=300, chi=2011),
        # The own prompts of requests forked from a system prompt.
        dict(name="extend_b16_ragged", kind="extend", batch=16, heads=14, kv_heads=2, page=64, lo=9,
             hi=301, clo=2048, chi=2048),
        # A chunk of a long prompt.
        dict(name="extend_chunk_2048", kind="extend", batch=1, heads=14, kv_heads=2, page=64, lo=2048,
             hi=2048, clo=16384, chi=16384),
        # One chat, drafts looked up in its own text, sampled.
        dict(name="verify_b1_k4", kind="verify", batch=1, lo=5, hi=5, vocab=151936, dtype="fp16",
             temperature=0.8, drafter=False),
        # A batch decoded greedily, with as many drafts as each row's text gave.
        dict(name="verify_b8_greedy", kind="verify", batch=8, lo=1, hi=5, vocab=151936, dtype="fp16",
             temperature=0.0, drafter=False),
        # A batch with the probabilities of a draft model.
        dict(name="verify_b32_k7", kind="verify", batch=32, lo=8, hi=8, vocab=151936, dtype="fp16",
             temperature=1.0, drafter=True),
    ]


def _log_int(rng, lo, hi):
    """Whole number spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["copy", "prefix", "extend", "verify"])
    kv_heads = rng.choice([1, 2, 2, 2, 4, 8])
    page = rng.choice([64, 64, 64, 128, 256])
    if kind == "copy":
        layers = rng.randint(2, 24)
        pairs = _log_int(rng, 1, max(1, 90_000_000 // (layers * kv_heads * page * D)))
        return dict(kind=kind, layers=layers, kv_heads=kv_heads, page=page, pairs=pairs,
                    slots=rng.choice([0, 0, -1, rng.randint(1, page)]))
    heads = kv_heads * rng.choice([1, 4, 7, 7, 7, 8, 16])
    if kind == "prefix":
        batch = _log_int(rng, 2, 96)
        phi = _log_int(rng, 64, min(32768, 6_000_000 // (batch * kv_heads)))
        hi = _log_int(rng, 1, max(1, min(4096, 300_000 // (batch * kv_heads))))
        return dict(kind=kind, batch=batch, groups=rng.randint(1, min(batch, 6)),
                    parked=rng.choice([0, 0, 1]), heads=heads, kv_heads=kv_heads, page=page,
                    plo=max(1, int(phi * rng.uniform(0.2, 1.0))), phi=phi,
                    lo=max(1, int(hi * rng.uniform(0.02, 1.0))), hi=hi)
    if kind == "extend":
        batch = _log_int(rng, 1, 32)
        hi = _log_int(rng, 1, min(2048, 8192 // batch, math.isqrt(400_000_000 // (batch * heads))))
        chi = _log_int(rng, 1, max(1, min(32768, 400_000_000 // (batch * hi * heads),
                                          6_000_000 // (batch * kv_heads))))
        return dict(kind=kind, batch=batch, heads=heads, kv_heads=kv_heads, page=page,
                    lo=int(hi * rng.uniform(0.0, 1.0)), hi=hi, clo=int(chi * rng.uniform(0.0, 1.0)),
                    chi=chi)
    batch = _log_int(rng, 1, 32)
    vocab = rng.choice([151936, 151936, rng.randint(1000, 151936)])
    hi = rng.randint(1, 8)
    return dict(kind="verify", batch=batch, lo=rng.randint(1, hi), hi=hi, vocab=vocab,
                dtype=rng.choice(["fp16", "fp16", "fp32"]),
                temperature=rng.choice([0.0, 1.0, round(rng.uniform(0.3, 1.5), 2)]),
                drafter=rng.choice([False, True]))


def _spread(n, lo, hi):
    """n whole numbers evenly over [lo, hi], in an order that is not sorted; ``hi`` is one of them."""
    if n == 1:
        return [hi]
    row = [lo + (hi - lo) * i // (n - 1) for i in range(n)]
    return row[1::2] + row[0::2][::-1]


def _prefix_plan(case):
    """(first row of each group and the end, prefix slots of each group, each row's slots in all)."""
    b, ng = case["batch"], case["groups"]
    starts = [b * g // ng for g in range(ng + 1)]
    plens = _spread(ng, case["plo"], case["phi"])
    own_slots = _spread(b, case["lo"], case["hi"])
    lens = [plens[max(g for g in range(ng) if starts[g] <= r)] + own_slots[r] for r in range(b)]
    for r in range(case["parked"]):          # free rows of the batch, the last ones
        lens[b - 1 - r] = 0
    return starts, plens, lens


def _rand(gen, *shape, dtype=torch.float16):
    return torch.randn(*shape, generator=gen, device=DEV, dtype=torch.float32).to(dtype)


def _ints(values, dtype):
    return torch.tensor(values, dtype=dtype).to(DEV)


# --------------------------------------------------------------------------
# what a user's program has in hand
# --------------------------------------------------------------------------

def prepare(case, seed):
    make = {"copy": _prepare_copy, "prefix": _prepare_prefix, "extend": _prepare_extend,
            "verify": _prepare_verify}[case["kind"]]
    return make(case, torch.Generator(DEV).manual_seed(seed))


def _prepare_copy(case, gen):
    n, page = case["pairs"], case["page"]
    n_pages = 2 * n + 3
    # Layers x (K, V) pools, as the cache allocates them.
    store = _rand(gen, case["layers"], 2, n_pages, case["kv_heads"], page, D)
    perm = torch.randperm(n_pages, generator=gen, device=DEV).to(torch.int32)
    slots = None
    if case["slots"] > 0:
        slots = torch.full((n,), case["slots"], dtype=torch.int32, device=DEV)
    elif case["slots"] < 0:
        slots = torch.randint(1, page, (n,), generator=gen, device=DEV).to(torch.int32)
    return dict(case=case, store=store, src=perm[:n].clone(), dst=perm[n:2 * n].clone(),
                slots=slots)


def _prepare_prefix(case, gen):
    kvh, page, b = case["kv_heads"], case["page"], case["batch"]
    starts, plens, lens = _prefix_plan(case)
    ppr = -(-max(max(lens), 1) // page)
    # Whole pages of a prefix are shared; its last, partly filled page is each row's own copy.
    full = [p // page for p in plens]
    shared = sum(full)
    need = shared + b * (ppr - min(full)) + 2
    perm = torch.randperm(need, generator=gen, device=DEV).to(torch.int32)
    kp, vp = _rand(gen, need, kvh, page, D), _rand(gen, need, kvh, page, D)
    table = torch.full((b, ppr), -1, dtype=torch.int32, device=DEV)
    at = shared
    for g, (p, f) in enumerate(zip(plens, full)):
        rows = slice(starts[g], starts[g + 1])
        table[rows, :f] = perm[sum(full[:g]):sum(full[:g]) + f]
        for r in range(starts[g], starts[g + 1]):
            if lens[r] == 0:
                table[r] = -1
                continue
            more = -(-lens[r] // page) - f
            ids = perm[at:at + more]
            table[r, f:f + more] = ids
            if p % page and r > starts[g]:
                first = int(table[starts[g], f])
                kp[int(ids[0]), :, :p % page] = kp[first, :, :p % page]
                vp[int(ids[0]), :, :p % page] = vp[first, :, :p % page]
            at += more
    q = _rand(gen, b, kvh, case["heads"] // kvh, D)
    return dict(case=case, q=q, kp=kp, vp=vp, table=table, last=_ints([n - 1 for n in lens], torch.int64),
                rows=_ints(starts, torch.int32), plen=_ints(plens, torch.int32))


def _prepare_extend(case, gen):
    kvh, page, b, qh = case["kv_heads"], case["page"], case["batch"], case["heads"]
    lens, ctx = _spread(b, case["lo"], case["hi"]), _spread(b, case["clo"], case["chi"])
    need = [-(-(n + c) // page) for n, c in zip(lens, ctx)]
    ppr, n_pages, total = max(need), sum(need) + 2, sum(lens)
    perm = torch.randperm(n_pages, generator=gen, device=DEV).to(torch.int32)
    table = torch.full((b, ppr), -1, dtype=torch.int32, device=DEV)
    for r, n in enumerate(need):
        table[r, :n] = perm[sum(need[:r]):sum(need[:r]) + n]
    # The fused projection's rows: heads of q, then of k, then of v.
    qkv = _rand(gen, total, qh + 2 * kvh, D)
    return dict(case=case, q=qkv[:, :qh], k=qkv[:, qh:qh + kvh], v=qkv[:, qh + kvh:],
                kp=_rand(gen, n_pages, kvh, page, D), vp=_rand(gen, n_pages, kvh, page, D), table=table,
                cu=_ints([sum(lens[:r]) for r in range(b + 1)], torch.int32), lens=lens,
                ctx=_ints(ctx, torch.int64), longest=max(lens), most=max(n + c for n, c in zip(lens, ctx)))


def _prepare_verify(case, gen):
    b, v, dtype = case["batch"], case["vocab"], {"fp16": torch.float16, "fp32": torch.float32}[case["dtype"]]
    lens = _spread(b, case["lo"], case["hi"])
    total = sum(lens)
    logits = _rand(gen, total, v, dtype=torch.float32) * 3
    # Drafts as a smaller model would make them: drawn from logits near the target's.
    near = logits + _rand(gen, total, v, dtype=torch.float32) * 0.4
    temp = case["temperature"] or 1.0
    race = torch.empty(total, v, device=DEV).exponential_(generator=gen).log_().neg_()
    sharp = 1.0 if case["drafter"] else 3.0          # text found again is what the target likes best
    picked = torch.argmax(near * (sharp / temp) + race, dim=-1)
    probs = torch.softmax(near / temp, dim=-1) if case["drafter"] else None
    cu = [sum(lens[:r]) for r in range(b + 1)]
    # A row is its last token and then the drafts; position j judges the token after it.
    tokens = torch.cat([torch.randint(0, v, (1,), generator=gen, device=DEV), picked[:-1]])
    return dict(case=case, logits=logits.to(dtype), tokens=tokens, cu=_ints(cu, torch.int32), lens=lens,
                longest=max(lens), probs=probs,
                accept_u=torch.rand(total, generator=gen, device=DEV),
                sample_u=torch.rand(b, generator=gen, device=DEV))


# --------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------

def run(s):
    if own:
        return _own(s)
    return _plain(s)


def _own(s):
    return {"copy": _own_copy, "prefix": _own_prefix, "extend": _own_extend,
            "verify": _own_verify}[s["case"]["kind"]](s)


def _plain(s):
    return {"copy": _plain_copy, "prefix": _plain_prefix, "extend": _plain_extend,
            "verify": _plain_verify}[s["case"]["kind"]](s)


def _own_copy(s):
    from qwenforge_amd import paged

    paged.copy_pages(s["store"], s["src"], s["dst"], slots=s["slots"])
    return s["store"]


def _own_prefix(s):
    from qwenforge_amd import paged

    return paged.flash_decode_attention_prefix_paged(s["q"], s["kp"], s["vp"], s["table"], s["rows"],
                                                     s["plen"], s["last"])


def _own_extend(s):
    from qwenforge_amd import paged

    out = paged.prefill_extend_paged(s["q"], s["k"], s["v"], s["cu"], s["longest"], s["ctx"], None, None,
                                     s["kp"], s["vp"], s["table"], lengths=s["lens"], max_slots=s["most"])
    return out, s["kp"], s["vp"]


def _own_verify(s):
    from qwenforge_amd import verify

    return verify.verify_drafts(s["logits"], s["tokens"], s["cu"], s["longest"], s["accept_u"], s["sample_u"],
                                temperature=s["case"]["temperature"], draft_probs=s["probs"], lengths=s["lens"])


def _plain_copy(s):
    store, src, dst = s["store"], s["src"].long(), s["dst"].long()
    taken = store[:, :, src]
    if s["slots"] is not None:
        keep = torch.arange(store.shape[4], device=DEV) < s["slots"][:, None]          # (pairs, page)
        taken = torch.where(keep[:, None, :, None], taken, store[:, :, dst])
    store[:, :, dst] = taken
    return store


def _rows_of(pool, table):
    """(rows, kv heads, slots, 64) fp32 of the rows' pages; pages not mapped read as some page."""
    b, ppr = table.shape
    got = pool[table.clamp(min=0).long()].float()                                       # (B, ppr, KVH, P, D)
    return got.transpose(1, 2).reshape(b, pool.shape[1], ppr * pool.shape[2], D)


def _attend(q, k, v, seen):
    """softmax(q k^T / 8) v in fp32 over the ``seen`` slots; zero where there are none.
    q (B, KVH, R, D), k and v (B, KVH, N, D), seen broadcast to (B, KVH, R, N)."""
    scores = torch.matmul(q, k.transpose(2, 3).contiguous()) * D ** -0.5
    scores = scores.masked_fill_(~seen, -math.inf)
    top = scores.amax(dim=-1, keepdim=True)
    p = torch.exp_(scores.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)))
    total = p.sum(dim=-1, keepdim=True)
    return torch.where(total > 0, torch.matmul(p, v) / total, torch.zeros_like(total))


def _plain_prefix(s):
    k, v = _rows_of(s["kp"], s["table"]), _rows_of(s["vp"], s["table"])
    seen = torch.arange(k.shape[2], device=DEV) <= s["last"][:, None]
    return _attend(s["q"].float(), k, v, seen[:, None, None, :]).half()


def _plain_extend(s):
    case, cu, ctx, table = s["case"], s["cu"].long(), s["ctx"], s["table"]
    b, longest, kvh, page = case["batch"], s["longest"], case["kv_heads"], case["page"]
    g, total = case["heads"] // kvh, s["q"].shape[0]
    token = torch.arange(total, device=DEV)
    row = torch.searchsorted(cu, token, right=True) - 1
    at = token - cu[row]
    slot = ctx[row] + at
    where = table[row, slot // page].long()
    s["kp"][where, :, slot % page] = s["k"]
    s["vp"][where, :, slot % page] = s["v"]
    k, v = _rows_of(s["kp"], table), _rows_of(s["vp"], table)
    # Rows side by side, padded to the longest.
    q = torch.zeros(b, longest, case["heads"], D, device=DEV)
    q[row, at] = s["q"].float()
    q = q.view(b, longest, kvh, g, D).permute(0, 2, 3, 1, 4).reshape(b, kvh, g * longest, D)
    last = ctx[:, None] + torch.arange(longest, device=DEV)                             # (B, longest)
    seen = torch.arange(k.shape[2], device=DEV) <= last[:, :, None]
    seen = seen[:, None, None].expand(b, 1, g, longest, k.shape[2]).reshape(b, 1, g * longest, -1)
    out = _attend(q, k, v, seen).view(b, kvh, g, longest, D).permute(0, 3, 1, 2, 4)
    return out.reshape(b, longest, case["heads"], D)[row, at].half(), s["kp"], s["vp"]


def _plain_verify(s):
    case, cu, tokens = s["case"], s["cu"].long(), s["tokens"]
    b, longest, vocab = case["batch"], s["longest"], case["vocab"]
    n = cu[1:] - cu[:-1]
    step = torch.arange(longest, device=DEV)
    at = torch.minimum(cu[:-1, None] + step, cu[1:, None] - 1)                          # (B, longest)
    nxt = torch.minimum(at + 1, cu[1:, None] - 1)
    judged = step < (n - 1)[:, None]                                                    # positions with a draft
    draft = tokens[nxt]
    x = s["logits"].double()
    if case["temperature"] == 0:
        best = torch.argmax(x, dim=-1)
        good = judged & (draft == best[at])
        count = torch.cumprod(good.long(), dim=1).sum(dim=1)
        final = best[at.gather(1, count[:, None])[:, 0]]
    else:
        x = x / case["temperature"]
        e = torch.exp(x - x.amax(dim=-1, keepdim=True))
        p = e / e.sum(dim=-1, keepdim=True)
        q = None if s["probs"] is None else s["probs"].double()
        p_d = p[at, draft]
        q_d = torch.ones_like(p_d) if q is None else q[at, draft]
        good = judged & (s["accept_u"].double()[at] * q_d < p_d)
        count = torch.cumprod(good.long(), dim=1).sum(dim=1)
        pos = at.gather(1, count[:, None])[:, 0]
        refused = count < n - 1
        w = p[pos]
        if q is None:
            away = torch.zeros_like(w).scatter_(1, draft.gather(1, count[:, None]), 1.0) > 0
            rest = torch.where(away, torch.zeros_like(w), w)
        else:
            rest = (w - q[pos]).clamp(min=0)
        rest = torch.where(rest.sum(dim=1, keepdim=True) > 0, rest, w)
        w = torch.where(refused[:, None], rest, w)
        reach = torch.cumsum(w, dim=1)
        mark = s["sample_u"].double()[:, None] * reach[:, -1:]
        at_least = (reach <= mark).sum(dim=1)
        last = vocab - 1 - (w.flip(1) > 0).long().argmax(dim=1)
        final = torch.minimum(at_least, last)
    out = torch.where(step < count[:, None], draft, torch.full_like(draft, -1))
    out.scatter_(1, count[:, None], final[:, None])
    return count + 1, out


# --------------------------------------------------------------------------
# what a pass cannot do without
# --------------------------------------------------------------------------

def work(case):
    return {"copy": _work_copy, "prefix": _work_prefix, "extend": _work_extend,
            "verify": _work_verify}[case["kind"]](case)


def _work_copy(case):
    n = case["slots"] if case["slots"] > 0 else case["page"] / 2 if case["slots"] < 0 else case["page"]
    return {"bytes": 2.0 * case["layers"] * 2 * case["pairs"] * case["kv_heads"] * n * D * 2, "flops": 0}


def _work_prefix(case):
    starts, plens, lens = _prefix_plan(case)
    alone = sum(n - plens[max(g for g in range(len(plens)) if starts[g] <= r)] for r, n in enumerate(lens) if n)
    slots = alone + sum(plens)
    return {"bytes": 4.0 * D * case["kv_heads"] * slots + 4.0 * D * case["batch"] * case["heads"],
            "flops": 4.0 * D * case["heads"] * sum(lens)}


def _work_extend(case):
    lens, ctx = _spread(case["batch"], case["lo"], case["hi"]), _spread(case["batch"], case["clo"], case["chi"])
    new, seen = sum(lens), sum(n * c + n * (n + 1) // 2 for n, c in zip(lens, ctx))
    cached = sum(c for n, c in zip(lens, ctx) if n)
    return {"bytes": 4.0 * D * (case["kv_heads"] * (cached + 2 * new) + case["heads"] * new),
            "flops": 4.0 * D * case["heads"] * seen}


def _work_verify(case):
    total = sum(_spread(case["batch"], case["lo"], case["hi"]))
    size = 2 if case["dtype"] == "fp16" else 4
    drafter = case["drafter"] and case["temperature"] > 0
    return {"bytes": float(case["vocab"]) * (total * size + (4 * case["batch"] if drafter else 0)),
            "flops": 0 if case["temperature"] == 0 else 4.0 * total * case["vocab"]}


# --------------------------------------------------------------------------
# the same from the definition, in 64 bits
# --------------------------------------------------------------------------

def exact(case, seed):
    find = {"copy": _exact_copy, "prefix": _exact_prefix, "extend": _exact_extend,
            "verify": _exact_verify}[case["kind"]]
    return find(case, prepare(case, seed))


def _exact_copy(case, s):
    store = s["store"].clone()
    slots = [case["page"]] * case["pairs"] if s["slots"] is None else s["slots"].tolist()
    for a, b, n in zip(s["src"].tolist(), s["dst"].tolist(), slots):
        store[:, :, b, :, :n] = s["store"][:, :, a, :, :n]
    return store.double()


def _dense(pool, pages, n):
    """(KVH, n, 64) in 64 bits of the first n slots of a row's pages."""
    slot = torch.arange(n, device=DEV)
    return pool[pages[slot // pool.shape[2]].long(), :, slot % pool.shape[2]].double().transpose(0, 1).contiguous()


def _heads(q, k, v, seen):
    """q (..., R, D) over k, v (..., N, D), all in 64 bits; seen (R, N) or None."""
    scores = torch.matmul(q, k.transpose(-1, -2).contiguous()) / 8.0
    if seen is not None:
        scores = scores.masked_fill(~seen, -math.inf)
    return torch.matmul(torch.softmax(scores, dim=-1), v)


def _exact_prefix(case, s):
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    for r, last in enumerate(s["last"].tolist()):
        if last >= 0:
            out[r] = _heads(s["q"][r].double(), _dense(s["kp"], s["table"][r], last + 1),
                            _dense(s["vp"], s["table"][r], last + 1), None)
    return out


def _exact_extend(case, s):
    kvh, page = case["kv_heads"], case["page"]
    g, out = case["heads"] // kvh, torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    cu = s["cu"].tolist()
    for r, c in enumerate(s["ctx"].tolist()):
        for lo in range(cu[r], cu[r + 1], 256):
            hi = min(lo + 256, cu[r + 1])
            first = c + lo - cu[r]
            n = first + hi - lo
            new = slice(cu[r], hi)
            k = torch.cat([_dense(s["kp"], s["table"][r], c), s["k"][new].double().transpose(0, 1)], dim=1)
            v = torch.cat([_dense(s["vp"], s["table"][r], c), s["v"][new].double().transpose(0, 1)], dim=1)
            slot = torch.arange(n, device=DEV)
            for h in range(kvh):
                q = s["q"][lo:hi, h * g:(h + 1) * g].double().transpose(0, 1).contiguous()   # (g, rows, D)
                seen = slot <= first + torch.arange(hi - lo, device=DEV)[:, None]
                out[lo:hi, h * g:(h + 1) * g] = _heads(q, k[h], v[h], seen).transpose(0, 1)
    return out, None, None


def _exact_verify(case, s):
    x = s["logits"].double().cpu().numpy()
    tokens, u, r = (s[k].cpu().numpy().astype(np.float64 if k != "tokens" else np.int64)
                    for k in ("tokens", "accept_u", "sample_u"))
    counts, out = [], []
    first = 0
    for b, n in enumerate(s["lens"]):
        row, done = [], False
        for j in range(n):
            i = first + j
            draft = int(tokens[i + 1]) if j + 1 < n else None
            if case["temperature"] == 0:
                best = int(np.argmax(x[i]))
                row.append(best)
                done = draft != best
            else:
                y = x[i] / case["temperature"]
                p = np.exp(y - y.max())
                p /= p.sum()
                q = None
                if draft is not None:
                    q = np.zeros_like(p)
                    q[draft] = 1.0
                    if s["probs"] is not None:
                        q = s["probs"][i].double().cpu().numpy()
                if draft is not None and u[i] * q[draft] < p[draft]:
                    row.append(draft)
                else:
                    w = p if q is None else np.maximum(p - q, 0)
                    w = w if w.sum() > 0 else p
                    reach = np.cumsum(w)
                    row.append(min(int(np.searchsorted(reach, r[b] * reach[-1], side="right")),
                                   int(np.flatnonzero(w)[-1])))
                    done = True
            if done:
                break
        first += n
        counts.append(len(row))
        out.append(row + [-1] * (s["longest"] - len(row)))
    return torch.tensor(counts, device=DEV), torch.tensor(out, device=DEV)
