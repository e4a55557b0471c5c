"""Calls on the paged cache and draft verification that their documentation allows and that lie at its edges: packed tokens that no row
owns, rope tables of any angles and too short ones, what is kept of weights and rotated keys, signed zeros, caches in the
reference mode, refusals. Bounds are the ones at the head of `test_paged.py`, named there term by term."""

import math

import numpy as np
import pytest
import torch

from gdn_hybrid_architecture_ideas_b200 import ops
from gdn_hybrid_architecture_ideas_b200.ops import paged as pg
from tests.test_paged import E4M3, _batch, _check_attention, _dense_attention, _random_cache, _status_clean, _tables, _values


def _poison(shape, value=7.0):
    """Free blocks of the allocator that hold `value`: what an output that nobody writes would show."""
    held = [torch.full(shape, value, dtype=torch.bfloat16, device="cuda") for _ in range(64)]
    torch.cuda.synchronize()
    del held


# ------------------------------------------------------------------------------------------------------------ tokens that no row owns

@pytest.mark.gpu
@pytest.mark.parametrize("fmt,hd", [("fp4", 64), ("bf16", 64), ("bf16", 256)])
@pytest.mark.parametrize("lead,tail", [(2, 0), (0, 3), (5, 40), (300, 0)])
def test_tokens_before_the_first_row_are_zeros(fmt, hd, lead, tail):
    """A group of rows beside the whole packed q (as of q_start[lo:hi + 1]): the tokens before and behind the group are zeros as in the statement, the
    group's are what a call that writes into `out` gives, and there the others stay."""
    rows, page = [(20, 1, 0), (33, 3, 4), (0, 0, 0), (9, 1, 0)], 16
    pages, q_start, lens, start, n, n_pages = _batch(rows, page)
    cache, cpu = _random_cache(n_pages, page, 2, hd, fmt)
    q_start, total = q_start + lead, lead + n + tail
    q = torch.randn(total, 8, hd).bfloat16()
    args = [t.cuda() for t in (pages, q_start, lens)]
    _poison((total, 8, hd))
    got = ops.paged_attention(q.cuda(), cache, *args, start=start.cuda())
    out = torch.full((total, 8, hd), 3.0, dtype=torch.bfloat16, device="cuda")
    ops.paged_attention(q.cuda(), cache, *args, start=start.cuda(), out=out)
    mine = slice(lead, lead + n)
    assert torch.equal(got[mine], out[mine]) and bool((out[:lead] == 3).all()) and bool((out[lead + n:] == 3).all())
    assert not got[:lead].any() and not got[lead + n:].any()
    want = ops.paged_attention(q, cpu, pages, q_start, lens, start=start)
    assert not want[:lead].any() and not want[lead + n:].any()
    _check_attention(q, cache, cpu, rows, pages, q_start, lens, start, None, None, page=page, got=got)


@pytest.mark.gpu
@pytest.mark.parametrize("q_start,owned", [([0, 1, 3, 9], [0, 1, 2]), ([2, 4, 0, 1], [0, 2, 3]), ([-3, 1, 3, 4], [1, 2, 3]), ([0, 9, 3, 4], [3]), ([5, 6, 8, 9], [])])
def test_tokens_of_refused_rows_are_zeros(q_start, owned):
    """Ranges out of order, negative or behind the packed tokens: status 301, zeros for every token that no accepted row owns, the others as
    with an `out`, in which the rest stays."""
    from gdn_hybrid_architecture_ideas_b200.ops import native

    rows, page, n = [(20, 1, 0), (33, 2, 0), (9, 1, 0)], 16, 5
    pages, _, lens, _, _, n_pages = _batch(rows, page)
    cache, _ = _random_cache(n_pages, page, 2, 64, "fp4")
    q = torch.randn(n, 8, 64, device="cuda").bfloat16()
    args = pages.cuda(), torch.tensor(q_start, dtype=torch.int32, device="cuda"), lens.cuda()
    _poison((n, 8, 64))
    got = ops.paged_attention(q, cache, *args)
    with pytest.raises(RuntimeError, match="status 301"):
        native.check_status()
    out = torch.full((n, 8, 64), 3.0, dtype=torch.bfloat16, device="cuda")
    ops.paged_attention(q, cache, *args, out=out)
    with pytest.raises(RuntimeError, match="status 301"):
        native.check_status()
    rest = [j for j in range(n) if j not in owned]
    assert torch.equal(got[owned], out[owned]) and not got[rest].any() and bool((out[rest] == 3).all())
    assert all(bool(got[j].any()) for j in owned)
