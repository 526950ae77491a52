"""The engine over 4-bit KV pages: prompts in chunks, decode steps, verify blocks, and conversations cut by eviction."""
import dataclasses

import pytest
import torch

from grimoire_b200.config import EngineConfig
from grimoire_b200.engine.engine import Engine, EngineLimits
from grimoire_b200.engine.generation import CopyDrafter, GenerationOptions, generate_tokens
from grimoire_b200.models.config import FULL_ATTN, LINEAR_ATTN, ModelConfig, tiny_dense, tiny_gemma4, tiny_qwen4_exp
from grimoire_b200.models.dense import DenseModel
from grimoire_b200.models.gemma4 import Gemma4Model
from grimoire_b200.models.hybrid import HybridModel, _DictSource
from grimoire_b200.models.mtp import MtpDrafter, MtpHead
from grimoire_b200.models.qwen4_exp import Qwen4ExpModel
from grimoire_b200.models.synthetic import random_gemma4_state_dict, random_qwen4_exp_state_dict, random_state_dict
from grimoire_b200.ops import kv4
from grimoire_b200.ops.kv4 import Kv4Layer
from grimoire_b200.sched.scheduler import Scheduler

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _engine(device, bits=4, seed=0, **lim):
    cfg = tiny_dense()
    model = DenseModel.from_state_dict(cfg, random_state_dict(cfg, seed=seed), device)
    return Engine(model, EngineLimits(**{**dict(max_slots=4, max_ctx=256, prefill_chunk=64, max_decode_rows=16, kv_bits=bits), **lim}))


def _prompt(n, seed=1):
    return torch.randint(0, 4096, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


def _feed(eng, seq, tokens):
    """Logits of teacher-forced decode steps."""
    out = []
    for t in tokens:
        _, lg = eng.decode_rows([t], [seq], [seq.length], use_graph=False, return_logits=True)
        out.append(lg[0].float().cpu().clone())
        eng.commit_rows([seq], [t], [seq.length])
    return out


@pytest.mark.parametrize("device", DEVICES)
def test_four_bit_engine_follows_the_eight_bit_one(device):
    """The same model over both caches: fewer bits move the logits a little, and memory falls to 72 / 136 a token and kv head."""
    a, b = _engine(device), _engine(device, 8)
    assert isinstance(a.kv.layers[0], Kv4Layer) and a.kv.bytes_per_token() * 136 == b.kv.bytes_per_token() * 72
    p, forced = _prompt(100), _prompt(8, 2)
    sa, sb = a.open(), b.open()
    la, lb = [a.prefill(sa, p).float().cpu()], [b.prefill(sb, p).float().cpu()]
    la += _feed(a, sa, forced)
    lb += _feed(b, sb, forced)
    scale = max(float(x.abs().max()) for x in lb)
    for x, y in zip(la, lb):
        assert bool(torch.isfinite(x).all()) and float((x - y).abs().max()) < 0.25 * scale
    a.release(sa)
    assert a.kv.pages_used() == 0


@pytest.mark.gpu
def test_gpu_matches_cpu():
    g, c = _engine("cuda"), _engine("cpu")
    p, forced = _prompt(150), _prompt(10, 3)                 # three chunks: history comes back through the pages
    sg, sc = g.open(), c.open()
    lg, lc = [g.prefill(sg, p).float().cpu()], [c.prefill(sc, p).float().cpu()]
    lg += _feed(g, sg, forced)
    lc += _feed(c, sc, forced)
    scale = max(float(x.abs().max()) for x in lc)
    for x, y in zip(lg, lc):
        assert float((x - y).abs().max()) < 0.05 * max(scale, 1.0)


@pytest.mark.gpu
def test_graph_replay_equals_eager():
    eng = _engine("cuda")
    p = _prompt(61)
    assert eng.generate(p, 24, use_graph=False) == eng.generate(p, 24, use_graph=True)
    assert eng.counters["graph_replays"] > 0


@pytest.mark.gpu
@pytest.mark.parametrize("n", [30, 125, 190])
def test_verify_rows_equal_single_steps_to_the_bit(n):
    """Speculation: rows of a block give the logits that single steps give (the 125-token block crosses a length bound)."""
    eng = _engine("cuda")
    eng.enable_speculation()
    p, forced = _prompt(n), _prompt(5, 4)
    s1, s2 = eng.open(), eng.open()
    eng.prefill(s1, p), eng.prefill(s2, p)
    singles = _feed(eng, s1, forced)
    _, lg = eng.decode_rows(forced, [s2] * 5, list(range(n, n + 5)), use_graph=False, return_logits=True)
    for i in range(5):
        assert torch.equal(lg[i].float().cpu(), singles[i])


@pytest.mark.parametrize("device", DEVICES)
def test_prefix_cache_copies_the_tail_page(device):
    eng = _engine(device)
    eng.enable_prefix_cache()
    p = _prompt(37)
    s = eng.open()
    first = eng.prefill(s, p).float().cpu().clone()
    eng.release(s, cache=True, head_logits=first)
    s = eng.open()
    assert eng.prefix_reuse(s, p + [5, 6]) > 0
    got = eng.prefill(s, (p + [5, 6])[s.length:]).float().cpu()
    t = eng.open()
    want = eng.prefill(t, p + [5, 6]).float().cpu()
    assert float((got - want).abs().max()) < 0.25 * float(want.abs().max())       # the prefix is read through the pages, not as bf16


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("graph", [False, True])
def test_a_cut_conversation_attends_to_what_is_left(device, graph):
    """keep == recent: the tokens that stay are the last ones, so the next rows must equal those of an uncut conversation under a
    sliding window that ends at the same token -- rotation positions, moved pages and tables included."""
    keep, n = 40, 75
    a = _engine(device, kv_keep=keep, kv_recent=keep, kv_sink=0, kv_slack=35)
    b = _engine(device)
    p, forced = _prompt(n), _prompt(3, 5)
    sa, sb = a.open(), b.open()
    a.prefill(sa, p), b.prefill(sb, p)
    assert a.trim(sa) and sa.length == keep and sa.dropped == n - keep and len(sa.pages) == 3
    for i, t in enumerate(forced):
        b.model.geom.window = keep + 1 + i
        _, lb = b.decode_rows([t], [sb], [sb.length], use_graph=False, return_logits=True)
        _, la = a.decode_rows([t], [sa], [sa.length], use_graph=graph, return_logits=True)
        assert float((la[0] - lb[0]).abs().max()) < 0.02 * float(lb[0].abs().max())
        a.commit_rows([sa], [t], [sa.length])
        b.commit_rows([sb], [t], [sb.length])


@pytest.mark.parametrize("device", DEVICES)
def test_eviction_keeps_a_conversation_inside_its_budget(device):
    eng = _engine(device, kv_keep=48, kv_recent=16, kv_slack=16, max_ctx=128)
    p = _prompt(60)
    s = eng.open()
    eng.prefill(s, p)
    lengths = []
    for t in _prompt(40, 6):
        eng.decode_rows([t], [s], [s.length])
        eng.commit_rows([s], [t], [s.length])
        eng.trim(s)
        lengths.append(s.length)
        assert len(s.tokens) == s.length
    assert max(lengths) < 64 and eng.counters["kv_evictions"] == 3 and s.dropped + s.length == 100
    mass = eng.kv.layers[0].mass
    assert bool(torch.isfinite(mass).all()) and float(mass.max()) > 0
    eng.prefill(s, _prompt(20, 7))                            # another turn: rotated behind the dropped tokens, observed on top
    assert s.length == lengths[-1] + 20
    eng.release(s)
    assert eng.kv.pages_used() == 0


@pytest.mark.parametrize("device", DEVICES)
def test_eviction_leaves_what_drew_weight(device):
    """A layer's kept tokens are those of its own mass; pages of other conversations stay untouched."""
    eng = _engine(device, kv_keep=32, kv_recent=8, kv_slack=8)
    a, b = eng.open(), eng.open()
    eng.prefill(a, _prompt(50)), eng.prefill(b, _prompt(50, 9))
    layer = eng.kv.layers[1]
    other = [layer.data[pg].clone() for pg in b.pages]
    t = torch.arange(50)
    mass = layer.mass[torch.tensor(a.pages)[t // 16].to(layer.mass.device), :, (t % 16).to(layer.mass.device)].cpu()          # [50][Hkv]
    assert eng.trim(a) and not eng.kv.evict(b, 60, 4)
    after = layer.mass[torch.tensor(a.pages)[t[:32] // 16].to(layer.mass.device), :, (t[:32] % 16).to(layer.mass.device)].cpu()
    for h in range(mass.shape[1]):
        m = mass[:, h].tolist()
        rest = sorted(range(4, 42), key=lambda i: (-m[i], i))[:20]
        assert after[:, h].tolist() == [m[i] for i in sorted([0, 1, 2, 3] + rest + list(range(42, 50)))]
    for pg, x in zip(b.pages, other):
        assert torch.equal(layer.data[pg], x)


@pytest.mark.gpu
def test_scheduler_serves_conversations_that_outgrow_their_budget():
    eng = _engine("cuda", kv_keep=48, kv_recent=16, kv_slack=16)
    s = Scheduler(eng, width=2, hold_ms=0, hold_long_ms=0)
    try:
        out, why, _ = s.generate(_prompt(40), 70)
        assert len(out) == 70 and why == "length"
        assert eng.counters["kv_evictions"] > 0
    finally:
        s.shutdown()
    assert eng.kv.pages_used() == 0


def test_refusals():
    for lim in (dict(bits=8, kv_keep=32), dict(kv_keep=32, kv_recent=32), dict(kv_keep=32, extra_kv_layers=1), dict(kv_keep=32, kv_slack=0), dict(bits=5)):
        with pytest.raises(ValueError):
            _engine("cpu", **lim)
    with pytest.raises(ValueError):
        _engine("cpu", kv_keep=32).enable_prefix_cache()
    for kw in (dict(kv_bits=3), dict(kv_keep=8), dict(kv_bits=4, kv_keep=-1)):
        with pytest.raises(ValueError):
            EngineConfig(**kw).validate()
    EngineConfig(kv_bits=4, kv_keep=4096).validate()


def _family(name, device):
    if name == "hybrid":
        cfg = ModelConfig(model_type="qwen3_5", hidden_size=512, num_hidden_layers=4, num_attention_heads=4, num_key_value_heads=2, head_dim=128,
                          vocab_size=4096, intermediate_size=1024, partial_rotary_factor=0.5, attn_output_gate=True, qk_norm=True,
                          norm_zero_centered=True, layer_types=[LINEAR_ATTN, LINEAR_ATTN, LINEAR_ATTN, FULL_ATTN], linear_num_key_heads=2,
                          linear_num_value_heads=4, linear_key_head_dim=128, linear_value_head_dim=128, quant="int4")
        return HybridModel.random(cfg, device, seed=2, max_slots=2, gen_device="cpu")
    if name == "gemma4":
        cfg = dataclasses.replace(tiny_gemma4(), hidden_size=512, head_dim=128, intermediate_size=1024, embed_scale=512 ** 0.5)
        return Gemma4Model.from_state_dict(cfg, random_gemma4_state_dict(cfg, seed=2), device)
    cfg = tiny_qwen4_exp(4)
    return Qwen4ExpModel.from_checkpoint(_DictSource(cfg, random_qwen4_exp_state_dict(cfg, 2)), device)


@pytest.mark.parametrize("name,device", [("hybrid", "cpu"), ("gemma4", "cpu"), ("qwen4_exp", "cpu"),
                                         *(pytest.param(n, "cuda", marks=pytest.mark.gpu) for n in ("hybrid", "gemma4"))])
def test_other_families_run_over_four_bit_pages(name, device):
    """Gated, windowed and sparse attention layers: prompts in chunks, decode steps, a replayed step."""
    lim = dict(max_slots=2, max_ctx=128, prefill_chunk=32, max_decode_rows=4)
    got = []
    for bits in (8, 4):
        eng = Engine(_family(name, device), EngineLimits(kv_bits=bits, **lim))
        s, V = eng.open(), eng.model.cfg.vocab_size
        ids = [t % V for t in _prompt(56, 3)]
        logits = [eng.prefill(s, ids[:50]).float().cpu()] + _feed(eng, s, ids[50:54])
        if device == "cuda":
            for t in ids[54:]:
                _, lg = eng.decode_rows([t], [s], [s.length], use_graph=True, return_logits=True)
                logits.append(lg[0].float().cpu().clone())
                eng.commit_rows([s], [t], [s.length])
        got.append(torch.stack(logits))
        eng.release(s)
    assert bool(torch.isfinite(got[1]).all()) and not torch.equal(got[0], got[1])
    assert float((got[0] - got[1]).abs().max()) < 0.25 * float(got[0].abs().max())


@pytest.mark.parametrize("device", DEVICES)
def test_draft_head_over_four_bit_pages_reproduces_greedy(device, monkeypatch):
    """Speculative output equals plain output, and every call is planned for the lengths that it has."""
    cfg = dataclasses.replace(tiny_dense(), tie_word_embeddings=False)
    lim = EngineLimits(max_slots=2, max_ctx=160, prefill_chunk=16, max_decode_rows=8, extra_kv_layers=1, kv_bits=4)
    p = _prompt(37, 3)
    plain = Engine(DenseModel.random(cfg, device, seed=1, gen_device="cpu"), lim)
    plain.enable_speculation()
    want = plain.generate(p, 24, use_graph=False)
    model = DenseModel.random(cfg, device, seed=1, gen_device="cpu")
    eng = Engine(model, lim)
    drafter = MtpDrafter(eng, MtpHead.random_from_target(model, seed=1, noise=0.01, gen_device="cpu"))
    real, calls = kv4.kv4_attn, []

    def watched(q, row_seq, row_pos, table, kv, geom, out, max_len, *a, **k):
        calls.append((int(row_pos.max()) + 1, max_len))
        return real(q, row_seq, row_pos, table, kv, geom, out, max_len, *a, **k)

    monkeypatch.setattr(kv4, "kv4_attn", watched)
    opts = GenerationOptions(max_new=24, draft_depth=3, drafter=drafter, use_graph=False)
    toks, _ = generate_tokens(eng, p, opts)
    assert toks == want and opts.stats.rounds > 0
    assert calls and all(n <= bound for n, bound in calls)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("drafts", [False, True])
def test_single_requests_stay_inside_the_budget(device, drafts):
    """The path of a single request (with and without drafts from the conversation) cuts the cache as the scheduler does."""
    eng = _engine(device, kv_keep=48, kv_recent=16, kv_slack=16, max_ctx=96)
    opts = GenerationOptions(max_new=60, draft_depth=3 if drafts else 0, drafter=CopyDrafter() if drafts else None, use_graph=False)
    s = eng.open()
    toks, _ = generate_tokens(eng, _prompt(10, 5) * 5, opts, seq=s)
    assert len(toks) == 60 and eng.counters["kv_evictions"] >= 2 and s.length + s.dropped >= 50 + 59 and s.length < 64 + 4
