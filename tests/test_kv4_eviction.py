"""Conversations cut by attention weight: what the weight counts, when a cut happens, and what must not depend on it."""
import pytest
import torch

from grimoire_b200.engine.generation import CopyDrafter, GenerationOptions, generate_tokens
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
