"""Barriers that every thread of a workgroup reaches, read from the sources (CPU
only): a barrier behind a return of some waves or lanes leans on the hardware
counting the rest, which HIP does not promise."""
import glob
import os
import re

import pytest

from neuralscript_amd import build

SOURCES = sorted(glob.glob(os.path.join(build.CSRC, "*.hip")))
# names that the kernels give what differs between a workgroup's threads
OWN = re.compile(r"\b(threadIdx|t|tid|lane|wave|w|wv|l16|l32|kh|kq|row|col|r|c|tok|pos|slot|i)\b")


def kernels(text):
    """(name, body) of every __global__ function."""
    text = re.sub(r"//[^\n]*", "", text)
    for m in re.finditer(r"__global__", text):
        at = text.index("{", m.end())
        depth, end = 0, at
        while True:
            depth += {"{": 1, "}": -1}.get(text[end], 0)
            end += 1
            if depth == 0:
                break
        yield re.search(r"(\w+)\s*\([^()]*\)\s*$", text[m.end():at]).group(1), text[at:end]


def early_returns(body):
    """Conditions on a thread's own values under which it returns before a later barrier."""
    last = body.rfind("__syncthreads")
    return [m.group(1) for m in re.finditer(r"if\s*\(([^;{}]*)\)\s*return;", body)
            if m.end() < last and OWN.search(re.sub(r"blockIdx\.\w", "", m.group(1)))]


@pytest.mark.parametrize("source", SOURCES, ids=os.path.basename)
def test_no_barrier_behind_a_return_of_some_threads(source):
    with open(source) as f:
        found = {name: early_returns(body) for name, body in kernels(f.read())}
    print({k: v for k, v in found.items() if v})
    assert not any(found.values()), {k: v for k, v in found.items() if v}
