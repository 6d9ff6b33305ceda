"""plan_step where its shared memory reaches the size that a launch may have without asking for more.

What one launch has asked for holds for the later ones of the process, so the batches are planned
smallest first in a process of their own."""

from __future__ import annotations

import pathlib
import random
import subprocess
import sys

import pytest

import test_plan_gpu as plans

pytestmark = pytest.mark.gpu

# 16 bytes a request and one entry more: with what the kernel has besides, 48 KB is passed from 3063 requests on
BATCHES = (3000, 3062, 3063, 3064, 3070, 3071, 4000, 8192)


def plan_smallest_first(most_new: int) -> None:
    for batch in BATCHES:
        rng = random.Random(batch)
        table, ctx, new, free, num_free = plans.draw(rng, batch, 16, 40, most_new)
        plans.run_both(table, ctx, new, free, num_free, 16, sum(new))


@pytest.mark.parametrize("most_new", [1, 9], ids=["few tokens", "many tokens"])
def test_batches_about_the_default_limit_of_shared_memory(most_new):
    here = pathlib.Path(__file__).resolve().parent
    code = (f"import sys; sys.path[:0] = [{str(here)!r}, {str(here.parent)!r}]\n"
            f"import test_plan_sizes_gpu as t; t.plan_smallest_first({most_new})")
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]
