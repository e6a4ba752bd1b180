"""CPU: refusals and host-side rules of the decoding operators at the edges of what their
documents allow."""
import ctypes

import pytest

import remora_b200 as rb
from tests.test_paged_cpu import A, L, append, attention, rope, tables  # noqa: F401


@pytest.mark.parametrize("bad", [2.0 ** 64, -2.0 ** 64, 1e300])
def test_rope_refuses_frequencies_it_cannot_hold(L, bad):  # noqa: F811
    freq = (ctypes.c_double * 64)(*[0.5] * 63, bad)
    for call in (rope, append):
        assert call(L, freq=ctypes.addressof(freq)) == rb.ERR_INVALID and "freq[63]" in rb.last_error()
