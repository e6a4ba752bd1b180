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


@pytest.mark.parametrize("config,tile,grid", [
    ("64x32x8x4096", 1, 64),     # fewer tokens than SMs
    ("4000x4x4x100", 2, 2000),   # 12 heads of 8 units: 32 of them fill a block's units
    ("4096x4x1x16", 5, 820),     # 6 heads
    ("8192x32x8x100", 1, 2368),  # 48 heads: one token, 16 blocks to each of 148 SMs
])
def test_decode_plan_cuts_the_append_as_the_launch_does(L, config, tile, grid):  # noqa: F811
    line = next(x for x in rb.launch_plan("decode", config).splitlines() if "k_rope" in x)
    assert f"grid {grid} x block 128" in line and f"tiles of {tile} tokens" in line


@pytest.mark.parametrize("bad", [dict(scale=3e38), dict(scale=-3e38),
                                 dict(cdt=rb.E4M3, scale=1e10, ks=1e30),
                                 dict(cdt=rb.E4M3, scale=3e9, ks=1e29, R=0)])
def test_attention_refuses_scales_whose_product_is_infinite(L, bad):  # noqa: F811
    assert attention(L, **bad) == rb.ERR_INVALID and "k_scale" in rb.last_error()


_SCARCE = """
import ctypes, resource, sys
import remora_b200 as rb
L, big = rb.lib(), b"x" * (64 << 20)
buf = ctypes.create_string_buffer(64)
held = int(next(x for x in open("/proc/self/status") if x.startswith("VmSize")).split()[1]) * 1024
resource.setrlimit(resource.RLIMIT_AS, (held + (16 << 20), resource.RLIM_INFINITY))
print(L.remora_b200_recognise(big), L.remora_b200_launch_plan(b"decode", big, buf, 64))
print(L.remora_b200_last_error().decode())
print(L.remora_b200_launch_plan(big, None, buf, 64), L.remora_b200_recognise(b"decode"))
"""


def test_no_exception_leaves_the_c_entry_points(L):  # noqa: F811
    """Host memory that cannot be had is a status, not the end of the process."""
    import subprocess
    import sys

    r = subprocess.run([sys.executable, "-c", _SCARCE], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr
    first, text, last = r.stdout.splitlines()
    assert first == f"0 {rb.ERR_INVALID}" and "launch_plan" in text and last == f"{rb.ERR_INVALID} 1"


@pytest.mark.parametrize("off", [1, 2, 3])
@pytest.mark.parametrize("call,fields", [
    (tables, "lens new table free count lo co cu slots pos req status"), (rope, "pos"),
    (append, "pos slots"), (attention, "table lens lse")])
def test_arrays_between_elements_are_refused(L, call, fields, off):  # noqa: F811
    """A 32-bit array at an address that no 32-bit load can take."""
    for name in fields.split():
        assert call(L, **{name: A + off}) == rb.ERR_INVALID and "aligned" in rb.last_error(), name


@pytest.mark.parametrize("call,bad", [
    (rope, dict(oh=0)), (rope, dict(os=0)), (rope, dict(os=127)), (rope, dict(oh=-64)),
    (rope, dict(B=2, ob=0, ld=8)), (rope, dict(x=2 * A, os=-127)),
    (append, dict(ot=0)), (append, dict(oh=64)), (append, dict(ot=-1)),
    (append, dict(kb=0)), (append, dict(ktok=0)), (append, dict(khd=120)), (append, dict(vb=0)),
    (append, dict(vtok=-8)), (append, dict(vhd=0)),
    (attention, dict(ot=0)), (attention, dict(oh=0)), (attention, dict(oh=-120))])
def test_outputs_whose_rows_overlap_are_refused(L, call, bad):  # noqa: F811
    """Rows that share elements (an expanded tensor, say) would hold whichever came last; in
    place, values turned once or twice."""
    assert call(L, **bad) == rb.ERR_INVALID and "overlap" in rb.last_error()


_RENAMED = """
import types
import torch
for name in ("_cuda_getDevice", "_cuda_getCurrentRawStream"):
    if hasattr(torch._C, name):
        delattr(torch._C, name)
import remora_b200 as rb
torch.cuda.current_device = rb._current_device = lambda: 0
torch.cuda.current_stream = lambda index: types.SimpleNamespace(cuda_stream=70 + index)
seen = []
rb._launch(lambda args, stream: seen.append((args, stream)) or rb.OK, b"x", 0)
print(seen)
"""


def test_calls_without_torchs_private_functions():
    """A torch that has renamed them: streams and devices come from its public interface."""
    import subprocess
    import sys

    r = subprocess.run([sys.executable, "-c", _RENAMED], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr
    assert r.stdout.strip() == "[(b'x', 70)]"
