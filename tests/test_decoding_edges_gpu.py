"""GPU: calls of the decoding operators at the edges of what their documents allow."""
import math
from fractions import Fraction

import numpy as np
import pytest
import torch

from tests import _paged as ref
from tests.test_paged_gpu import check_tables, close, freqs, gen, i32

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------- block tables
def blocks_disjoint(lens, table, free, count, bs):
    """No block is free twice, held twice, or free and held."""
    held = [b for n, row in zip(lens, table) for b in row[:-(-int(n) // bs)]]
    return len(set(held) | set(free[:count])) == len(held) + count


@pytest.mark.parametrize("lens,new,mb,bs,spare,mt", [
    ([0, 16], [5, -1], 2, 16, 1, 3),                             # one release behind the overflow
    ([0, 16, 3], [5, -1, -1], 2, 16, 1, 3),
    ([0, 40, 16, 0], [2000000000, -1, -1, 7], 4, 16, 4, 8),      # a count of no sense in front
    ([8, 0, 24, 5, 9], [1, 30, -1, 0, -1], 4, 8, 6, 4),          # a grant, the overflow, releases
    ([0] + [17] * 1100, [9] + [-1, 1] * 550, 3, 16, 3, 2),       # eight CTAs
])
def test_block_table_releases_behind_an_overflow(rb, lens, new, mb, bs, spare, mt):
    """A release has no tokens, so none of its own pass max_tokens: it is done, whatever the
    requests before it asked for, and its blocks are free and no longer held."""
    got, want = check_tables(rb, lens, new, mb, bs, spare, mt)
    for r, n in enumerate(new):
        if n == -1:
            assert int(got.status[r]) == 0 and int(got.lens[r]) == 0
    assert blocks_disjoint(got.lens.tolist(), want["table"], want["free"], int(got.free_count), bs)
