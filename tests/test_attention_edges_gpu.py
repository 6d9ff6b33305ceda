"""Attention over the paged cache where its rows, keys and workers are laid out at an edge: against
the definitions in 64 bits, with the bounds derived in operators_ref."""

from __future__ import annotations

import pytest
import torch

import operators_ref as ref

pytestmark = pytest.mark.gpu


def check_rows(got, c, r, rows, what=""):
    """The first ``rows`` rows of ``got`` against the same rows of ``r``, all of which have to be finite."""
    out, bound = (x[:rows] for x in r)
    assert rows > 0 and out.isfinite().all() and bound.isfinite().all()
    off = (got[:rows].double() - out).abs()
    assert (off <= bound).all(), f"{what}: off by {float(off.nan_to_num(float('inf')).max()):.3e}"


@pytest.mark.parametrize("kernel", ["simple", "stream"])
@pytest.mark.parametrize("maps", [1, 2])
@pytest.mark.parametrize("kv", ["fp16", "bf16", "int8"])
@pytest.mark.parametrize("lens,new,rows", [([35], [30], 11), ([300, 520], [300, 520], 401), ([9000, 8000], [40, 30], 45)])
def test_rows_are_cut_off_where_the_starts_name_more(kernel, maps, kv, lens, new, rows):
    """q holds fewer rows than query_start_loc names: those it holds see the keys they would see in the whole."""
    c = ref.make(lens, new, heads=4, kv_heads=2, dim=64, kv=kv, maps=maps, lam="heads", seed=3)
    r = ref.reference(c)
    c.q = c.q[:rows].contiguous()
    check_rows(c.call(kernel=kernel), c, r, rows, kernel)
