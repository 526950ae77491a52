"""Conversations cut by attention weight: what the weight counts, when a cut happens, and what must not depend on it."""
import threading

import pytest
import torch

from grimoire_b200.engine.generation import CopyDrafter, GenerationOptions, generate_tokens
from grimoire_b200.engine.sampling import SamplingOptions
from grimoire_b200.sched.scheduler import Scheduler

from .test_kv4_engine import DEVICES, _engine, _prompt

CUT = dict(kv_keep=48, kv_recent=16, kv_slack=16)


def _mass(eng, seq):
    """Weight of the cached tokens: [layers][tokens][kv heads]."""
    t = torch.arange(seq.length)
    page = torch.tensor(seq.pages)[t // 16]
    return torch.stack([layer.mass.cpu()[page, :, t % 16] for layer in eng.kv.layers])


@pytest.mark.parametrize("device", DEVICES)
def test_drafts_leave_no_weight_behind(device):
    """A drafter changes neither the tokens nor the weight that a later cut goes by, to the bit: nothing is drafted."""
    p, got = _prompt(10, 5) * 5, []
    for drafter in (None, CopyDrafter()):
        eng = _engine(device, **CUT)
        opts = GenerationOptions(max_new=40, draft_depth=3 if drafter else 0, drafter=drafter, use_graph=False)
        s = eng.open()
        toks, _ = generate_tokens(eng, p, opts, seq=s)
        assert opts.stats.rounds == 0 and eng.counters["kv_evictions"] > 0
        got.append((toks, s.length, s.dropped, _mass(eng, s)))
    assert got[0][:3] == got[1][:3] and torch.equal(got[0][3], got[1][3])


def test_a_step_over_a_cut_cache_takes_one_row_of_a_conversation():
    eng = _engine("cpu", **CUT)
    a, b = eng.open(), eng.open()
    eng.prefill(a, _prompt(20)), eng.prefill(b, _prompt(21))
    eng.decode_rows([1, 2], [a, b], [20, 21])
    before = [layer.mass.clone() for layer in eng.kv.layers]
    with pytest.raises(NotImplementedError):
        eng.decode_rows([1, 2], [a, a], [20, 21])
    assert all(torch.equal(x, layer.mass) for x, layer in zip(before, eng.kv.layers))


def test_scheduler_drafts_nothing_over_a_cut_cache():
    p = _prompt(10, 5) * 4
    outs = []
    for drafts in (False, True):
        s = Scheduler(_engine("cpu", **CUT), width=2, hold_ms=0, hold_long_ms=0, copy_drafts=drafts, depths=(3,))
        try:
            outs.append(s.generate(p, 30)[:2])
            assert s.metrics["spec_rounds"] == 0 and s.metrics["errors"] == 0
        finally:
            s.shutdown()
    assert outs[0] == outs[1] and len(outs[0][0]) == 30


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("n", [20, 100, 131])
def test_a_prompt_is_observed_once_however_it_is_read(device, n):
    """Whole, in chunks whose last one would be short, in slices: the last 32 rows (all, of a shorter prompt) and nothing else."""
    p, got = _prompt(n), []
    for chunk, step in ((256, n), (33, n), (64, n), (256, 25), (64, 40), (128, 7)):
        eng = _engine(device, kv_keep=48, kv_recent=16, prefill_chunk=chunk, kv_slack=200)
        s = eng.open()
        lo = 0
        while lo < n:
            hi = min(n, lo + step)
            hi = n if eng.ends_prompt(n - hi) else hi
            eng.prefill(s, p[lo:hi], last=hi == n)
            lo = hi
        m = _mass(eng, s)
        rows = min(n, 32) * (eng.model.geom.Hq // eng.model.geom.Hkv)
        # every row and query head gives a weight of one in all, summed in fp32 from weights that are off by 2^-9 at most
        assert float((m.sum(1) - rows).abs().max()) < 2 ** -9 * rows
        got.append(m[0])
    # the first layer's rows and keys are the same up to the rounding of a projection (q is bf16): a few percent of a weight
    for m in got[1:]:
        assert float((m - got[0]).abs().sum(0).max()) < 0.05 * rows


def test_scheduler_observes_a_sliced_prompt_once():
    """A long prompt beside a conversation that decodes is read in slices; one observation of its last rows is made of it."""
    eng = _engine("cpu", kv_keep=200, kv_recent=16, kv_slack=40, max_ctx=256)
    seen, real = [], eng.model.forward

    def forward(rb, *a):
        if rb.mode == "prefill":
            seen.append((rb.tokens.shape[0], rb.observe_rows, rb.observe))
        return real(rb, *a)

    eng.model.forward = forward
    s = Scheduler(eng, width=2, hold_ms=0, hold_long_ms=0, interleave_chunk=24)
    try:
        started = threading.Event()
        t = threading.Thread(target=lambda: s.generate(_prompt(8), 120, on_token=lambda _: started.set() or True))
        t.start()
        assert started.wait(60)
        s.generate(_prompt(100, 2), 2)
        t.join()
    finally:
        s.shutdown()
    slices = seen[1:]
    assert seen[0] == (8, 8, "set") and len(slices) > 1 and sum(x[0] for x in slices) == 100
    assert [x[1] for x in slices] == [0] * (len(slices) - 1) + [32]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("slots,pages", [(1, 0), (1, 4), (2, 8)])
def test_a_full_pool_can_still_be_cut(device, slots, pages):
    """A pool that conversations fill to the last page: every one is cut in its turn, and never grows past keep + slack tokens."""
    eng = _engine(device, **CUT, max_slots=slots, max_ctx=64, kv_pages=pages)
    seqs = [eng.open() for _ in range(slots)]
    for i, s in enumerate(seqs):
        eng.prefill(s, _prompt(60, i))
    for i, t in enumerate(_prompt(60, 6)):
        eng.decode_rows([t] * slots, seqs, [s.length for s in seqs])
        eng.commit_rows(seqs, [t] * slots, [s.length for s in seqs])
        for s in seqs:
            assert eng.trim(s) == ((60 + i + 1 - 64) % 16 == 0 and i >= 3)
    assert eng.counters["kv_evictions"] == 4 * slots and "kv_evictions_failed" not in eng.counters
    assert eng.kv.pages_free() == eng.kv.num_pages - sum(len(s.pages) for s in seqs)
    for s in seqs:
        eng.release(s)
    assert eng.kv.pages_used() == 0 and eng.kv.pages_free() == eng.kv.num_pages


def test_one_request_in_a_pool_of_its_own_size_is_bounded():
    """The path of a single request with one slot, whose pool holds one context: cut instead of growing to the end of it."""
    eng = _engine("cpu", **CUT, max_slots=1, max_ctx=96)
    toks = eng.generate(_prompt(40), 56, use_graph=False)
    assert len(toks) == 56 and eng.counters["kv_evictions"] == 2


def test_limits_that_would_never_cut_are_refused():
    for lim in (dict(kv_keep=48, kv_slack=16, max_ctx=63), dict(kv_keep=48, kv_slack=16, max_ctx=96, kv_pages=3)):
        with pytest.raises(ValueError):
            _engine("cpu", **lim)
    _engine("cpu", kv_keep=48, kv_slack=16, max_ctx=64, kv_pages=4)


def test_a_cut_that_finds_no_pages_is_counted():
    """Sequences that share pages keep them from the reserve: the cut is refused, counted, and tried again later."""
    eng = _engine("cpu", **CUT, max_slots=3, max_ctx=64, kv_pages=8)
    a, b, c = eng.open(), eng.open(), eng.open()
    eng.prefill(a, _prompt(64))
    eng.kv.share_prefix(a, b, 64)
    eng.prefill(c, _prompt(64, 2))
    assert eng.trim(a) and eng.kv.pages_free() == 0                  # b holds what a left
    assert not eng.trim(c) and c.length == 64 and eng.counters["kv_evictions_failed"] == 1
    eng.release(b)
    assert eng.trim(c) and c.length == 48


@pytest.mark.parametrize("device", DEVICES)
def test_sampled_tokens_are_drawn_at_positions_that_never_come_back(device):
    """A draw is a function of (seed, position): over several cuts the positions are those of the conversation."""
    eng = _engine(device, **CUT)
    drawn, real = [], eng.sample_rows

    def sample_rows(logits, opts, positions):
        drawn.extend(positions)
        return real(logits, opts, positions)

    eng.sample_rows = sample_rows
    s = Scheduler(eng, width=2, hold_ms=0, hold_long_ms=0)
    try:
        out, _, _ = s.generate(_prompt(40), 80, sampling=SamplingOptions(temperature=0.8, top_k=20, seed=3))
    finally:
        s.shutdown()
    assert eng.counters["kv_evictions"] >= 3 and len(out) == 80
    assert drawn == list(range(40, 120))


def test_a_failed_capture_does_not_stop_the_weight():
    """The run before a capture counts no rows; where it fails, the steps after it count theirs."""
    eng = _engine("cpu", **CUT)
    s = eng.open()
    eng.prefill(s, _prompt(40))
    real = eng.model.forward
    eng.model.forward = lambda *a: (_ for _ in ()).throw(RuntimeError("out of memory"))
    eng._stage_rows([1], [s.slot], [40], [s])
    with pytest.raises(RuntimeError):
        eng._capture(1, 64)
    eng.model.forward = real
    before = float(_mass(eng, s).sum())
    eng.decode_rows([1], [s], [40], use_graph=False)
    eng.commit_rows([s], [1], [40])
    rows = len(eng.kv.layers) * eng.model.geom.Hq                    # a row gives a weight of one a layer and query head
    assert abs(float(_mass(eng, s).sum()) - before - rows) < 2 ** -9 * rows


@pytest.mark.gpu
def test_replayed_steps_count_their_rows_once():
    """The run before a capture and the capture itself add nothing; every replay adds its row."""
    eng = _engine("cuda", kv_keep=200, kv_recent=16, kv_slack=40)
    s = eng.open()
    eng.prefill(s, _prompt(40))
    rows = len(eng.kv.layers) * eng.model.geom.Hq
    for i in range(4):
        before = float(_mass(eng, s).sum())
        eng.decode_rows([1], [s], [40 + i], use_graph=True)
        eng.commit_rows([s], [1], [40 + i])
        assert abs(float(_mass(eng, s).sum()) - before - rows) < 2 ** -9 * rows


def test_a_loaded_model_whose_cache_is_cut_drafts_nothing():
    """The loader's defaults (copy drafts on) with a cut cache: single requests and the scheduler work and draft nothing; limits that
    cannot hold the cut are refused at load."""
    from grimoire_b200.api import Grimoire
    from grimoire_b200.config import EngineConfig
    from grimoire_b200.engine.generation import SpecStats

    ec = dict(model="synthetic:tiny_dense", seq_slots=2, prefill_chunk=64, kv_bits=4, kv_keep=32)
    g = Grimoire.load(EngineConfig(ctx=320, **ec), device="cpu")
    assert "speculation: off" in g.banner()
    st, p = SpecStats(), _prompt(10, 5) * 3
    toks, _ = g.generate(p, 20, draft_depth=3, stats=st)
    out = g.generate_batch([p, p[:17]], 20)
    assert len(toks) == 20 and st.rounds == 0 and out[0][0] == toks and len(out[1][0]) == 20
    assert g.scheduler().metrics["spec_rounds"] == 0
    g.close()
    with pytest.raises(ValueError):
        Grimoire.load(EngineConfig(ctx=256, **ec), device="cpu")
