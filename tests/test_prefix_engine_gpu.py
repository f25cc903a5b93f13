"""Serving with a shared prefix and with drafted tokens (``paged_engine``): page
forks, extension, shared-prefix decode and draft verification together.

The oracle's logits are fp32; the fp16 engine stays within LOGIT_TOL of them
(the bound of the other engine tests), so a greedy token of the engine has an
oracle logit within 2 * LOGIT_TOL of the row's largest.
"""

import pytest
import torch

import oracle.model as om
from qwenforge_amd.model import Qwen2Config, init_weights, weights_to
from qwenforge_amd.paged_engine import PagedDecodeEngine, lookup_drafts

pytestmark = pytest.mark.gpu
LOGIT_TOL = 3e-2
CFG = Qwen2Config(layers=2, vocab=4096)


@pytest.fixture(scope="module")
def model(dev):
    w = init_weights(CFG, "cpu", seed=8)
    gen = torch.Generator().manual_seed(2)
    for layer in w["layers"]:
        layer["qkv_bias"] = (torch.randn(CFG.qkv_width, generator=gen) * 0.1).half()
    return w, PagedDecodeEngine(CFG, weights_to(w, dev), dev)


def _ids(gen, n):
    return torch.randint(0, CFG.vocab, (n,), generator=gen)


def _oracle_logits(w, ids):
    """fp32 logits after every token of `ids`."""
    caches = om.prefill(w, CFG, ids[:1].view(1, -1), ids.numel())
    logits, caches = [caches[0][0]], caches[1]
    for i in range(1, ids.numel()):
        logits.append(om.decode_step(w, CFG, ids[i:i + 1], torch.tensor([i]), caches, i)[0])
    return torch.stack(logits)


def _assert_greedy(w, prompt, new):
    """Every token of `new` is an argmax of the oracle's logits within both sides' error."""
    logits = _oracle_logits(w, torch.cat([prompt, new[:-1]]))[prompt.numel() - 1:]
    short = logits.max(dim=-1).values - logits.gather(1, new[:, None])[:, 0]
    assert short.max().item() <= 2 * LOGIT_TOL


@pytest.mark.parametrize("native", [True, False])
def test_extension_in_pieces_matches_the_oracle(dev, model, monkeypatch, native):
    w, eng = model
    if native:
        inner = eng._native_extension
        monkeypatch.setattr(eng, "_native_extension", lambda *a: inner(*a) or pytest.fail("not native"))
    else:
        monkeypatch.setattr(eng, "_native_extension", lambda *a: False)
    gen = torch.Generator().manual_seed(3)
    texts = [_ids(gen, n) for n in (150, 70, 9)]
    kv = eng.new_paged_cache(4, 12, 64, 4)
    for r in (2, 0, 3):
        kv.map_row(r, 160)
    at = [0, 0, 0]
    for cut in ((64, 1, 3), (1, 63, 1), (80, 6, 5), (5, 0, 0)):
        go = [i for i in range(3) if cut[i]]
        got = eng.extend_paged([texts[i][at[i]:at[i] + cut[i]] for i in go], kv, [(2, 0, 3)[i] for i in go],
                               [at[i] for i in go], last_only=False).float().cpu()
        row = 0
        for i in go:
            ref = _oracle_logits(w, texts[i][:at[i] + cut[i]])[at[i]:]
            assert (got[row:row + cut[i]] - ref).abs().max().item() <= LOGIT_TOL
            row += cut[i]
            at[i] += cut[i]
    for i, r in enumerate((2, 0, 3)):
        n = texts[i].numel()
        _, caches = om.prefill(w, CFG, texts[i].view(1, -1), n)
        for layer in range(CFG.layers):
            for got, ref in zip(kv.gather(layer, r, n), caches[layer]):
                assert (got.float().cpu() - ref[0, :, :n]).abs().max().item() <= 2e-2


@pytest.mark.parametrize("bounds", [[0, 3, 6], [2, 5, 8], [0, 6, 6]])
def test_layers_of_padded_tokens_append_none_of_them(dev, model, bounds):
    """Tokens before the first row and behind the last reach no page."""
    from qwenforge_amd import prefill_ops

    _, eng = model
    gen = torch.Generator().manual_seed(4)
    kv = eng.new_paged_cache(2, 6, 64, 3)
    for r in range(2):
        kv.map_row(r, 192)
    contexts = [5, 70]
    hidden = (torch.randn(10, CFG.hidden, generator=gen) * 0.1).half().to(dev)
    layers = prefill_ops.layer_table(CFG, eng.w["layers"], kv.pools, hidden.device,
                                     (kv.n_pages, kv.kv_heads, kv.page_size, CFG.head_dim))
    prefill_ops.extend_layers(CFG, layers, hidden, torch.tensor(bounds, dtype=torch.int32, device=dev),
                              torch.tensor(contexts, device=dev), 192, eng.inv_freq, kv.table, kv.n_pages,
                              kv.page_size)
    written = (kv.store != 0).any(dim=-1).cpu()             # (layers, 2, page, head, slot)
    want = torch.zeros_like(written)
    for r, c in enumerate(contexts):
        for slot in range(c, c + bounds[r + 1] - bounds[r]):
            want[:, :, int(kv.table[r, slot // 64]), :, slot % 64] = True
    assert torch.equal(written, want)
    assert hidden[bounds[0]:bounds[-1]].isfinite().all()


def test_forked_rows_extend_and_decode_apart(dev, model):
    """Two rows forked from one go on with texts of their own; the first row's pages stay its own."""
    w, eng = model
    gen = torch.Generator().manual_seed(4)
    base, tails = _ids(gen, 100), [_ids(gen, 30), _ids(gen, 5)]
    kv = eng.new_paged_cache(3, 9, 64, 3)
    kv.map_row(0, 128)
    eng.prefill_paged([base.to(dev)], kv, [0])
    kept = [torch.cat(kv.gather(i, 0, 100)).clone() for i in range(CFG.layers)]
    kv.fork_rows(0, [1, 2], 100)
    for r in (1, 2):
        kv.map_row(r, 140)
    assert kv.shared_pages(1) == 1
    got = eng.extend_paged([t.to(dev) for t in tails], kv, [1, 2], [100, 100]).float().cpu()
    for i, t in enumerate(tails):
        ref = _oracle_logits(w, torch.cat([base, t]))[-1]
        assert (got[i] - ref).abs().max().item() <= LOGIT_TOL
    # Row 0 goes back to slot 60 of the page it shares: it gets a copy first.
    again = _ids(gen, 10)
    got = eng.extend_paged([again.to(dev)], kv, [0], [60]).float().cpu()
    assert (got[0] - _oracle_logits(w, torch.cat([base[:60], again]))[-1]).abs().max().item() <= LOGIT_TOL
    assert kv.shared_pages(0) == 0 and kv.shared_pages(1) == 1
    for i in range(CFG.layers):
        for r in (1, 2):
            assert torch.equal(torch.cat(kv.gather(i, r, 100)), kept[i])
    assert kv.compact() >= 0
    for i in range(CFG.layers):
        assert torch.equal(torch.cat(kv.gather(i, 1, 100)), kept[i])


@pytest.mark.parametrize("once", [True, False])
@pytest.mark.parametrize("max_batch,tiles", [(1, True), (3, True), (6, True), (3, False), (33, True)])
def test_serving_behind_a_prefix(dev, model, monkeypatch, max_batch, tiles, once):
    """Every step form: fused, wide and torch, reading the prefix once or row by
    row; rows are reused, and a request's tokens are those it gets alone in the
    same step shape."""
    w, eng = model
    if not tiles:
        eng = PagedDecodeEngine(CFG, eng.w, dev, fused_step=False)
    monkeypatch.setattr(eng, "reads_prefix_once", lambda batch, slots: once)
    gen = torch.Generator().manual_seed(5)
    prefix = _ids(gen, 150)
    prompts, news = [_ids(gen, n) for n in (9, 40, 1, 17, 30)], [6, 1, 9, 4, 7]
    pages = 2 * max_batch + 6
    got = eng.serve([p.to(dev) for p in prompts], news, max_batch=max_batch, n_pages=pages,
                    prefix=prefix.to(dev))
    kv = eng._ctx["kv"]
    assert kv.free_pages() == kv.n_pages == pages
    for p, n, ids in zip(prompts, news, got):
        assert ids.numel() == n
        _assert_greedy(w, torch.cat([prefix, p]), ids.cpu())
    for i in (0, 2):
        # Padded by a request of the same pages, so that the step keeps its shape.
        alone = eng.serve([prompts[i].to(dev), prompts[1].to(dev)], [news[i], 1], max_batch=max_batch,
                          n_pages=pages, prefix=prefix.to(dev))[0]
        assert torch.equal(alone, got[i])


def test_when_a_prefix_is_read_once(dev, model):
    _, eng = model
    assert not eng.reads_prefix_once(1, 16384) and not eng.reads_prefix_once(4, 1024)
    assert eng.reads_prefix_once(2, 4096) and eng.reads_prefix_once(4, 16384)
    assert not eng.reads_prefix_once(8, 16384) and eng.reads_prefix_once(32, 16384)


def test_prefix_serving_refuses_and_runs_out(dev, model):
    _, eng = model
    gen = torch.Generator().manual_seed(6)
    p = [_ids(gen, 10).to(dev)]
    with pytest.raises(ValueError):
        eng.serve(p, 3, prefix=p[0][:0])
    with pytest.raises(ValueError):
        eng.serve([p[0][:0]], 3, prefix=p[0])
    with pytest.raises(RuntimeError, match="too small"):
        eng.serve(p, 3, max_batch=1, n_pages=2, prefix=_ids(gen, 128).to(dev))
    with pytest.raises(RuntimeError, match="exhausted"):
        eng.serve(p, 3, max_batch=1, n_pages=1, prefix=_ids(gen, 128).to(dev))
    kv = eng.new_paged_cache(2, 2, 64, 1)
    kv.map_row(0, 64)
    for bad in (([p[0]], [0], [60]), ([p[0]], [1], [0]), ([p[0], p[0]], [0, 0], [0, 0]), ([p[0]], [0], [-1]),
                ([p[0][:0]], [0], [0]), ([], [], []), ([p[0]], [0], [])):
        with pytest.raises(ValueError):
            eng.extend_paged(bad[0], kv, bad[1], bad[2])


@pytest.mark.parametrize("draft_len", [0, 3, 8])
def test_drafted_greedy_tokens_are_the_models(dev, model, draft_len):
    w, eng = model
    gen = torch.Generator().manual_seed(7)
    phrase = _ids(gen, 12)
    prompts = [torch.cat([phrase, phrase, phrase[:5]]), _ids(gen, 70), phrase[:1]]
    stats = {}
    got = eng.generate_drafted([p.to(dev) for p in prompts], 11, draft_len=draft_len, stats=stats)
    assert got.shape == (3, 11)
    for p, ids in zip(prompts, got.cpu()):
        _assert_greedy(w, p, ids)
    assert stats["accepted"] <= stats["drafted"]
    if draft_len == 0:
        assert stats == dict(passes=10, drafted=0, accepted=0)


def test_good_drafts_save_passes_and_bad_ones_cost_nothing_but_time(dev, model):
    w, eng = model
    gen = torch.Generator().manual_seed(9)
    prompts = [_ids(gen, 33), _ids(gen, 64)]
    on_dev = [p.to(dev) for p in prompts]
    plain = eng.generate_drafted(on_dev, 12, draft_len=0).cpu().tolist()
    text = {tuple(p.tolist()[:5]): p.tolist() + ids for p, ids in zip(prompts, plain)}

    def knowing(tokens, n):
        return text[tuple(tokens[:5])][len(tokens):len(tokens) + n]

    good, bad = {}, {}
    for drafter, stats in ((knowing, good), (lambda t, n: [7] * n, bad)):
        got = eng.generate_drafted(on_dev, 12, draft_len=4, drafter=drafter, stats=stats).cpu()
        for p, ids in zip(prompts, got):
            _assert_greedy(w, p, ids)
    assert good["accepted"] > 0 and good["passes"] < 11
    with pytest.raises(ValueError, match="vocabulary"):
        eng.generate_drafted(on_dev, 4, drafter=lambda t, n: [CFG.vocab])


def test_sampled_generation_follows_its_seed(dev, model):
    _, eng = model
    gen = torch.Generator().manual_seed(10)
    prompts = [_ids(gen, 20).to(dev), _ids(gen, 41).to(dev)]
    a, b, c = (eng.generate_drafted(prompts, 16, temperature=0.9, seed=s, draft_len=2) for s in (1, 1, 2))
    assert torch.equal(a, b) and not torch.equal(a, c)
    assert ((a >= 0) & (a < CFG.vocab)).all()


def test_lookup_drafts_continue_the_last_occurrence():
    assert lookup_drafts([1, 2, 3, 9, 1, 2, 3, 4, 1, 2, 3], 3) == [4, 1, 2]
    assert lookup_drafts([5, 6, 7], 4) == []
    assert lookup_drafts([4, 4], 2) == [4]
    assert lookup_drafts([], 2) == [] and lookup_drafts([1], 2) == []
