"""Generation over caches held in 8 bits (``paged_engine`` with ``kv_code``).

The reference for a step is the oracle model run over the very keys and values that the
engine's pages hold after it (the new token's among them), so that only the step's own
arithmetic differs; what the pages hold is compared with what the oracle quantises.
"""

import numpy as np
import pytest
import torch

import oracle.model as om
from oracle import kv8
from oracle.attention import eager_attention
from qwenforge_amd.model import Qwen2Config, init_weights, weights_to
from qwenforge_amd.paged_engine import PagedDecodeEngine

pytestmark = pytest.mark.gpu
LOGIT_TOL = 3e-2  # fp16 engine vs fp32 oracle, logits std ~0.6 (as the fp16 engine tests)


def step_over(w, cfg, token, pos, caches):
    """Logits (V,) of one row's token at ``pos`` over caches [(K, V)] (KVH, pos + 1, 64) that hold it already, and
    the keys and values it would write."""
    inv = om.inv_freq32(cfg)
    hidden = om._f(w["embed"])[token].view(1, 1, -1)
    at = torch.tensor([[pos]])
    new = []
    for layer, (kc, vc) in zip(w["layers"], caches):
        q, k, v = om._qkv(om._rms(hidden, om._f(layer["input_norm"]), cfg.rms_eps), layer, cfg)
        q, k = om._rope(q, at, inv), om._rope(k, at, inv)
        new.append((k[0, :, 0], v[0, :, 0]))
        att = eager_attention(q, kc[None].float(), vc[None].float(), causal=False)
        hidden = hidden + att.transpose(1, 2).reshape(1, 1, -1) @ om._f(layer["o_weight"]).T
        hidden = hidden + om._mlp(om._rms(hidden, om._f(layer["post_norm"]), cfg.rms_eps), layer)
    hidden = om._rms(hidden, om._f(w["final_norm"]), cfg.rms_eps)
    return (hidden @ om._f(w["lm_head"]).T)[0, 0], new


def held_within(x, y, big, code):
    """Whether what the pages hold of a token, x, is its fp32 value y up to the engine's fp16 noise (2e-2, as the
    fp16 caches' test has) and the roundings: a block whose largest magnitude is ``big`` has a scale s < 2 big / Q.
    int8 (Q = 127) is off by half a step s, and by less than another half in all for earlier, smaller scales: big /
    63.5.  e4m3 (Q = 448) by 2^-4 of the value, and below its normal range by 2^-10 s for each scale, less than
    2^-9 s in all."""
    noise = 2e-2 * (1 if code == "int8" else 1 + 2.0 ** -4)
    bound = big / 63.5 if code == "int8" else np.abs(y) * 2.0 ** -4 + big / 448 * 2.0 ** -8
    return (np.abs(x - y) <= noise + bound).all()


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("batch,tiles", [(1, True), (3, True), (5, True), (5, False)])
def test_steps_match_the_oracle_over_the_same_pages(dev, batch, tiles, code):
    """The fused step (1 and 3 rows), the wide one and the torch projections, captured, over several replays."""
    cfg = Qwen2Config(layers=2, vocab=4096)
    w_cpu = init_weights(cfg, "cpu", seed=16)
    eng = PagedDecodeEngine(cfg, weights_to(w_cpu, dev), dev, tile_weights=tiles)
    gen = torch.Generator().manual_seed(21)
    lengths = [47, 130, 64, 15, 200][:batch]
    prompts = [torch.randint(0, cfg.vocab, (n,), generator=gen) for n in lengths]
    kv = eng.new_paged_cache(batch, 5 * batch, 64, 5, code)
    for r, n in enumerate(lengths):
        kv.map_row(r, n + 8)
    logits = eng.prefill_paged([p.to(dev) for p in prompts], kv, range(batch)).float().cpu()
    for r, p in enumerate(prompts):
        want, caches = om.prefill(w_cpu, cfg, p.view(1, -1), lengths[r])
        assert (logits[r] - want[0]).abs().max() <= LOGIT_TOL
        for layer in range(cfg.layers):
            for got, ref in zip(kv.gather(layer, r, lengths[r]), caches[layer]):
                got, ref = got.float().cpu().numpy(), ref[0].numpy()
                for s in range(lengths[r]):
                    # The block's values stand together: its largest is the scale's.
                    block = slice(s // 16 * 16, s // 16 * 16 + 16)
                    big = np.abs(ref[:, block]).max()
                    assert held_within(got[:, s], ref[:, s], big + 2e-2, code)
    ctx = eng.make_paged_context(kv, batch, 6)
    eng.capture_paged(ctx)
    ctx["pos"].copy_(torch.tensor(lengths, device=dev))
    ctx["step"].fill_(1)
    token = logits.argmax(-1)
    for t in range(4):
        ctx["token"].copy_(token.to(dev))
        ctx["graph"].replay()
        torch.cuda.synchronize()
        got = ctx["logits"].float().cpu()
        for r in range(batch):
            pos = lengths[r] + t
            caches = [tuple(x.cpu() for x in kv.gather(i, r, pos + 1)) for i in range(cfg.layers)]
            want, new = step_over(w_cpu, cfg, token[r], pos, caches)
            err = (got[r] - want).abs().max().item()
            print(f"[kv8 engine] {code} B={batch} step {t} row {r} max|dlogit| {err:.3e}", flush=True)
            assert err <= LOGIT_TOL
            for pair, ref in zip(caches, new):
                for x, y in zip(pair, ref):
                    block = x[:, pos // 16 * 16:].float().numpy()
                    big = max(np.abs(block).max(), np.abs(y.numpy()).max())
                    assert held_within(x[:, -1].float().numpy(), y.numpy(), big + 2e-2, code)
        token = got.argmax(-1)
    assert ctx["pos"].cpu().tolist() == [n + 4 for n in lengths]


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_extension_matches_the_oracle_over_the_same_pages(dev, code, native, monkeypatch):
    """All layers in one native call, and with torch's projections."""
    cfg = Qwen2Config(layers=2, vocab=4096)
    w_cpu = init_weights(cfg, "cpu", seed=18)
    eng = PagedDecodeEngine(cfg, weights_to(w_cpu, dev), dev)
    if not native:
        monkeypatch.setattr(eng, "_native_extension", lambda *args: False)
    gen = torch.Generator().manual_seed(23)
    prompts = [torch.randint(0, cfg.vocab, (n,), generator=gen) for n in (40, 70)]
    chunks = [torch.randint(0, cfg.vocab, (n,), generator=gen) for n in (5, 3)]
    kv = eng.new_paged_cache(2, 6, 64, 3, code)
    for r in range(2):
        kv.map_row(r, 100)
    eng.prefill_paged([p.to(dev) for p in prompts], kv, range(2))
    got = eng.extend_paged([c.to(dev) for c in chunks], kv, [0, 1], [40, 70], last_only=False).float().cpu()
    first = 0
    for r, (p, c) in enumerate(zip(prompts, chunks)):
        before = [[x.cpu() for x in kv.gather(layer, r, len(p))] for layer in range(cfg.layers)]
        assert all(torch.isfinite(x).all() and x.any() for pair in before for x in pair)
        for i, token in enumerate(c):
            pos = len(p) + i
            caches = [tuple(x.cpu() for x in kv.gather(layer, r, pos + 1)) for layer in range(cfg.layers)]
            want, _ = step_over(w_cpu, cfg, token, pos, caches)
            assert (got[first + i] - want).abs().max() <= LOGIT_TOL, (r, i)
        first += len(c)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("max_batch", [2, 5])
def test_serving_over_eight_bits(dev, max_batch, code):
    """Requests keep their tokens in any company, pages return to the pool; behind a common prefix too."""
    cfg = Qwen2Config(layers=2)
    eng = PagedDecodeEngine(cfg, init_weights(cfg, dev, seed=7), dev)
    gen = torch.Generator().manual_seed(3)
    lengths, news = [40, 100, 7, 64, 130], [6, 3, 8, 1, 5]
    prompts = [torch.randint(0, cfg.vocab, (n,), generator=gen).to(dev) for n in lengths]
    prefix = torch.randint(0, cfg.vocab, (75,), generator=gen).to(dev)
    for common in (None, prefix):
        got = eng.serve(prompts, news, max_batch=max_batch, prefix=common, kv_code=code)
        kv = eng._ctx["kv"]
        assert kv.code == code and kv.free_pages() == kv.n_pages
        for i, (p, n) in enumerate(zip(prompts, news)):
            longest = prompts[4] if i != 4 else prompts[1]
            alone = eng.serve([p, longest], [n, 5 if i != 4 else 1], max_batch=max_batch, prefix=common,
                              n_pages=kv.n_pages, kv_code=code)[0]
            assert got[i].shape == (n,) and torch.equal(got[i].cpu(), alone.cpu()), i


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_generation_and_drafts(dev, code):
    """Shapes, pages and drafts; a cache in 8 bits costs 128.5 bytes a slot and head where fp16 costs 256."""
    cfg = Qwen2Config(layers=2)
    eng = PagedDecodeEngine(cfg, init_weights(cfg, dev, seed=8), dev)
    gen = torch.Generator().manual_seed(4)
    prompts = [torch.randint(0, cfg.vocab, (n,), generator=gen).to(dev) for n in (300, 17, 100)]
    rows = eng.generate_paged(prompts, 12, kv_code=code)
    assert rows.shape == (3, 12)
    kv = eng._ctx["kv"]
    assert kv.store.numel() == cfg.layers * kv.n_pages * cfg.kv_heads * 64 * 257 // 2
    stats = {}
    out = eng.generate_drafted(prompts, 10, drafter=lambda text, n: [int(rows[0, 0])] * n, stats=stats, kv_code=code)
    assert out.shape == (3, 10) and stats["drafted"] > 0
    with pytest.raises(ValueError, match="code must be"):
        eng.generate_paged(prompts, 2, kv_code="int4")


def test_native_extension_s_refusals(dev):
    from qwenforge_amd import prefill_ops

    cfg = Qwen2Config(layers=2, vocab=4096)
    eng = PagedDecodeEngine(cfg, init_weights(cfg, dev, seed=5), dev)
    kv = eng.new_paged_cache(2, 4, 64, 2, "int8")
    kv.map_row(0, 100)
    table = prefill_ops.layer_table(cfg, eng.w["layers"], None, dev, None)
    hidden = torch.zeros(7, cfg.hidden, device=dev, dtype=torch.float16)
    cu = torch.tensor([0, 5, 7], dtype=torch.int32, device=dev)
    ctx = torch.zeros(2, dtype=torch.int64, device=dev)

    def call(pools=kv.pools, hidden=hidden, cu=cu, longest=5, ctx=ctx, most=128, freq=eng.inv_freq, blocks=kv.table):
        prefill_ops.extend_layers_paged8(cfg, table, pools, hidden, cu, longest, ctx, most, freq, blocks)

    for kw in (dict(pools=kv.pools[:1]), dict(pools=[kv.pools[0], kv.all_pools]), dict(hidden=hidden.float()),
               dict(hidden=hidden.t().contiguous().t()), dict(cu=cu.long()), dict(cu=cu[:2]), dict(ctx=ctx.int()),
               dict(freq=eng.inv_freq.half()), dict(blocks=kv.table[:1]), dict(blocks=kv.table.long())):
        with pytest.raises((ValueError, TypeError)):
            call(**kw)
    for kw in (dict(longest=0), dict(longest=8), dict(most=0), dict(most=129)):
        with pytest.raises(RuntimeError):
            call(**kw)
    call()
