"""CPU: kernels launched as programmatic dependents wait for the kernel before
them. Such a kernel may start while its predecessor runs; what that one (and all
before it) wrote is visible only after griddepcontrol.wait, so every thread has
to execute it, ahead of its first access to global memory."""
import glob
import os
import re

import pytest

from conftest import ROOT

CSRC = os.path.join(ROOT, "dreamcompiler_b200", "csrc")
WAIT = re.compile(r'asm volatile\("griddepcontrol\.wait;" ::: "memory"\);|wait_for_predecessor\(\);')


def dependents():
    """(file, kernel, body) of every kernel in the files that launch theirs through launch.h."""
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu"))):
        text = open(path).read()
        if '#include "launch.h"' not in text:
            continue
        text = re.sub(r"//[^\n]*", "", text)
        for m in re.finditer(r"__global__ void (?:__launch_bounds__\([^{;]*?\)\s*)?(\w+)\(", text):
            start = text.index("{", m.end())
            depth, i = 0, start
            while True:
                depth += {"{": 1, "}": -1}.get(text[i], 0)
                i += 1
                if not depth:
                    break
            yield os.path.basename(path), m.group(1), text[start:i]


KERNELS = list(dependents())


def test_the_kernels_are_found():
    names = {k for _, k, _ in KERNELS}
    assert {"embed_fwd_kernel", "embed_sort_kernel", "embed_sum_kernel", "embed_few_kernel", "head_logits_kernel",
            "head_grads_kernel", "head_small_kernel", "head_lists_kernel", "head_finish_kernel", "head_mean_kernel",
            "head_sums_kernel"} <= names


@pytest.mark.parametrize("file,kernel,body", KERNELS, ids=[k for _, k, _ in KERNELS])
def test_every_thread_waits(file, kernel, body):
    waits = [m for m in WAIT.finditer(body)]
    assert len(waits) == 1, "one wait"
    before = body[:waits[0].start()]
    line = before[before.rindex("\n") + 1:]
    assert not line.strip(), f"the wait is conditional: {line}"
    assert before.count("{") - before.count("}") == 1, "the wait is inside a branch or a loop"
    assert "return" not in before
