"""The measured cases of the sparse layer's operators (perf/operators.py), on
the CPU: the calls they make of the framework."""
import types

import pytest
import torch

import perf.operators as cases
from neuralscript_amd import runtime

CASES = [{"kind": "experts", "T": 3, "K": 2, "D": 8, "H": 12, "E": 4, "act": 6},
         {"kind": "train", "T": 3, "K": 2, "D": 8, "H": 12, "E": 4, "act": 6},
         {"kind": "ns", "n": 2, "r": 8, "c": 12}, {"kind": "muon", "n": 2, "r": 8, "c": 12}]
# where the calls have their workspace among their arguments
ROOM = {"moe_experts": 13, "moe_experts_grad": 16, "newton_schulz": 6, "muon_ns_step": 10}


@pytest.mark.parametrize("first", CASES, ids=lambda c: c["kind"])
@pytest.mark.parametrize("second", CASES, ids=lambda c: c["kind"])
def test_calls_that_overlap_share_no_workspace(first, second, monkeypatch):
    """A second pass begins before the first has run, as on two streams: each of
    its calls has a workspace apart from those still in use."""
    monkeypatch.setattr(cases, "DEV", "cpu")
    monkeypatch.setattr(torch.cuda, "current_stream", lambda: types.SimpleNamespace(cuda_stream=0))
    lib = runtime.lib()
    states = [cases.prepare(c, i) for i, c in enumerate((first, second))]
    outer, inner = [], []

    def size(name, case):
        if name in ("newton_schulz", "muon_ns_step"):
            return lib.nsh_op_newton_schulz_workspace(case["n"], case["r"], case["c"])
        return lib.nsh_op_moe_experts_workspace(*(case[k] for k in ("T", "K", "D", "H", "E")), int(case["kind"] == "train"))

    def op(name, *args):
        if inner is seen[0]:
            inner.append((args[ROOM[name]], size(name, second)))
            return
        outer.append((args[ROOM[name]], size(name, first)))
        seen[0] = inner
        cases._own(states[1])
        seen[0] = outer

    seen = [outer]
    monkeypatch.setattr(runtime, "op", op)
    cases._own(states[0])
    assert outer and inner
    for a, n in outer:
        for b, k in inner:
            assert a + n <= b or b + k <= a
