"""CPU tests: the decoding entry points reject bad arguments on the host, before
any CUDA call, and their Python mirrors reject bad tensors."""
import ctypes

import numpy as np
import pytest
import torch

import remora_b200 as rb
from tests import _paged as ref

A = 1 << 20  # never read: every refusal comes before the first access
ODD = A + 8


def call(fn, packer, fields):
    """The entry point on a packed argument struct (None = a null pointer)."""
    return fn(packer.pack(*(0 if v is None else v for v in fields.values())), None)


@pytest.fixture(scope="module")
def L():
    from remora_b200 import build

    build.build()
    return rb.lib()


def tables(L, **c):
    d = dict(lens=A, new=A, table=A, free=A, count=A, lo=A, co=A, cu=A, slots=A, pos=A, req=A,
             status=A, R=4, ld=8, mb=8, nb=32, bs=16, mt=4)
    d.update(c)
    return call(L.remora_b200_kv_block_table, rb._BLOCK_TABLE_ARGS, d)


@pytest.mark.parametrize("bad", [
    dict(R=-1), dict(R=8193), dict(mt=-1), dict(mt=2 ** 31 - 1), dict(bs=0), dict(nb=0),
    dict(nb=2 ** 27, bs=16), dict(mb=0), dict(mb=2 ** 27, ld=2 ** 27), dict(ld=7), dict(lens=None),
    dict(new=None), dict(table=None), dict(free=None), dict(count=None), dict(lo=None),
    dict(co=None), dict(cu=None), dict(slots=None), dict(pos=None), dict(req=None),
    dict(status=None)])
def test_block_table_refuses(L, bad):
    assert tables(L, **bad) == rb.ERR_INVALID and "kv_block_table" in rb.last_error()


_FREQ = (ctypes.c_double * 64)(*[0.5] * 64)
_NAN = (ctypes.c_double * 64)(*[0.5] * 63, float("nan"))
_INF = (ctypes.c_double * 64)(*[float("inf")] * 64)
_AXES = (ctypes.c_int32 * 64)(*[0] * 63, 1)
FREQ, NAN, INF, AXES = (ctypes.addressof(x) for x in (_FREQ, _NAN, _INF, _AXES))


def rope(L, **c):
    d = dict(x=A, out=A, pos=A, freq=FREQ, ax=None, B=1, S=4, H=2, D=128, rot=128, xb=0, xs=256,
             xh=128, ob=0, os=256, oh=128, ld=4, dt=rb.BF16, axes=1, inter=0, inv=0)
    d.update(c)
    return call(L.remora_b200_rope, rb._ROPE_ARGS, d)


@pytest.mark.parametrize("bad", [
    dict(x=None), dict(out=None), dict(dt=rb.E4M3), dict(dt=9), dict(B=-1), dict(S=-1), dict(H=-1),
    dict(D=0), dict(D=2048), dict(pos=None), dict(ld=3, axes=2), dict(axes=0), dict(axes=9),
    dict(freq=None), dict(ax=AXES), dict(rot=3), dict(rot=130), dict(rot=258, D=512),
    dict(x=A + 1), dict(freq=NAN), dict(freq=INF), dict(xs=2 ** 31),
    dict(oh=-2 ** 31), dict(D=300, xs=601), dict(D=512, rot=2), dict(S=2 ** 30 + 1, ld=2 ** 31), dict(B=2 ** 20, S=2 ** 20, ld=2 ** 41)])
def test_rope_refuses(L, bad):
    assert rope(L, **bad) == rb.ERR_INVALID and "rope" in rb.last_error()


def test_rope_without_rows_is_done(L):
    assert rope(L, S=0, ld=0, pos=None, x=None, out=None) == rb.OK
    assert rope(L, H=0, x=None, out=None) == rb.OK


def append(L, **c):
    d = dict(q=A, k=A, v=A, qo=A, kc=A, vc=A, pos=A, slots=A, freq=FREQ, ax=None, T=4, Hq=4, Hkv=2,
             D=128, rot=128, qt=512, qh=128, kt=256, kh=128, vt=256, vh=128, ot=512, oh=128, ld=4,
             nb=4, bs=16, kb=4096, ktok=256, khd=128, vb=4096, vtok=256, vhd=128, ks=1.0, vs=1.0,
             dt=rb.BF16, cdt=rb.BF16, axes=1, inter=0)
    d.update(c)
    return call(L.remora_b200_rope_kv_append, rb._APPEND_ARGS, d)


@pytest.mark.parametrize("bad", [
    dict(q=None), dict(k=None), dict(v=None), dict(qo=None), dict(slots=None), dict(kc=None),
    dict(vc=None), dict(pos=None), dict(dt=rb.F32), dict(cdt=rb.F16), dict(T=-1), dict(Hkv=0),
    dict(nb=0), dict(bs=0), dict(nb=2 ** 28), dict(ks=0.0), dict(vs=-1.0), dict(ks=2.0),
    dict(cdt=rb.E4M3, ks=float("nan")), dict(cdt=rb.E4M3, vs=float("inf")), dict(rot=200),
    dict(cdt=rb.E4M3, ks=1e-31), dict(cdt=rb.E4M3, vs=1e31), dict(qt=2 ** 31), dict(T=2 ** 31),
    dict(kc=A + 1)])
def test_append_refuses(L, bad):
    assert append(L, **bad) == rb.ERR_INVALID and "rope_kv_append" in rb.last_error()


def attention(L, **c):
    d = dict(q=A, kc=A, vc=A, table=A, lens=A, out=2 * A, lse=None, ws=A, wsb=1 << 40, R=2, Hq=8, Hkv=2,
             D=128, qt=1024, qh=128, ot=1024, oh=128, nb=8, bs=16, kb=4096, kt=256, kh=128, vb=4096,
             vt=256, vh=128, ld=8, mb=8, window=0, scale=1.0, ks=1.0, vs=1.0, dt=rb.BF16,
             cdt=rb.BF16)
    d.update(c)
    return call(L.remora_b200_paged_attention, rb._ATTENTION_ARGS, d)


@pytest.mark.parametrize("bad", [
    dict(q=None), dict(kc=None), dict(vc=None), dict(table=None), dict(lens=None), dict(out=None),
    dict(out=A), dict(q=ODD), dict(kc=ODD), dict(vc=ODD), dict(out=ODD), dict(ws=ODD), dict(ws=None),
    dict(wsb=0), dict(dt=rb.F32), dict(cdt=rb.F16), dict(R=-1), dict(R=8193), dict(Hq=7),
    dict(Hkv=0), dict(Hq=0), dict(D=96), dict(nb=0), dict(bs=0), dict(nb=2 ** 28), dict(mb=0),
    dict(ld=7), dict(mb=2 ** 28, ld=2 ** 28), dict(scale=float("nan")), dict(scale=float("inf")),
    dict(window=-1), dict(ks=0.5), dict(vs=2.0), dict(cdt=rb.E4M3, ks=0.0), dict(cdt=rb.E4M3, vs=1e31),
    dict(cdt=rb.E4M3, kt=264), dict(qt=1020), dict(oh=4), dict(kt=12), dict(vb=4)])
def test_attention_refuses(L, bad):
    assert attention(L, **bad) == rb.ERR_INVALID and "paged_attention" in rb.last_error()


def test_null_argument_structs_are_refused(L):
    for fn in (L.remora_b200_kv_block_table, L.remora_b200_rope, L.remora_b200_rope_kv_append,
               L.remora_b200_paged_attention):
        assert fn(None, None) == rb.ERR_INVALID and "null" in rb.last_error()


def test_packed_structs_have_the_headers_layout(tmp_path):
    """The packers' sizes, and their last fields' places, as a C compiler lays the structs out."""
    import os
    import subprocess

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    names = {"kv_block_table": ("max_tokens", rb._BLOCK_TABLE_ARGS),
             "rope": ("inverse", rb._ROPE_ARGS),
             "rope_kv_append": ("interleaved", rb._APPEND_ARGS),
             "paged_attention": ("cache_dtype", rb._ATTENTION_ARGS)}
    src = '#include <stdio.h>\n#include <stddef.h>\n#include "remora_b200.h"\nint main(void) {\n'
    for n, (last, _) in names.items():
        src += f'printf("%zu %zu\\n", sizeof(remora_b200_{n}_args), ' \
               f'offsetof(remora_b200_{n}_args, {last}));\n'
    (tmp_path / "s.c").write_text(src + "return 0; }\n")
    exe = str(tmp_path / "s")
    subprocess.run(["gcc", "-I", os.path.join(root, "include"), str(tmp_path / "s.c"), "-o", exe],
                   check=True)
    lines = subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split("\n")
    for line, (n, (last, packer)) in zip(lines, names.items()):
        size, at = map(int, line.split())
        pad = 4 if n == "paged_attention" else 0
        width = 8 if n == "kv_block_table" else 4
        assert size == packer.size and at == packer.size - pad - width, n


def test_attention_without_requests_is_done_and_workspace_sizes(L):
    assert attention(L, R=0, q=None, ws=None, wsb=0) == rb.OK
    assert L.remora_b200_paged_attention_workspace_bytes(8, 32, 8, 128) > 0
    for bad in ((-1, 8, 2, 128), (8, 7, 2, 128), (8, 8, 0, 128), (8, 8, 2, 80), (9000, 8, 2, 128)):
        assert L.remora_b200_paged_attention_workspace_bytes(*bad) == 0


def test_decode_program_is_recognised_and_planned(L):
    assert rb.recognise("decode")
    plan = rb.launch_plan("decode")
    for word in ("remora_b200_kv_block_table", "k_block_table", "remora_b200_rope_kv_append",
                 "k_rope", "remora_b200_paged_attention", "k_paged_split", "k_paged_join", "grid"):
        assert word in plan
    assert "k_paged_join" not in rb.launch_plan("decode", "1x1x1x1")  # one CTA: nothing to join
    for bad in ("64", "0x8x2x16", "4x7x2x16", "9000x8x2x16", "4x8x2x0", "8192x8x2x1048576"):
        with pytest.raises(rb.RemoraError, match="decode config"):
            rb.launch_plan("decode", bad)


def test_python_mirrors_refuse_host_tensors_and_bad_shapes():
    i = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    b = lambda *s: torch.zeros(s, dtype=torch.bfloat16)  # noqa: E731
    f = torch.zeros(32, dtype=torch.float64)
    with pytest.raises(ValueError, match="CUDA"):
        rb.kv_block_table(i(2), i(2), i(2, 4), i(8), i(1), 16, 4)
    with pytest.raises(ValueError, match="new_tokens"):
        rb.kv_block_table(i(2), i(3), i(2, 4), i(8), i(1), 16, 4)
    with pytest.raises(ValueError, match="block_table"):
        rb.kv_block_table(i(2), i(2), i(3, 4), i(8), i(1), 16, 4)
    with pytest.raises(ValueError, match="CUDA"):
        rb.rope(b(4, 2, 64), i(4), f)
    with pytest.raises(ValueError, match="positions"):
        rb.rope(b(4, 2, 64), i(5), f)
    with pytest.raises(ValueError, match="axis_of"):
        rb.rope(b(4, 2, 64), i(3, 4), f)
    with pytest.raises(TypeError):
        rb.rope(torch.zeros(4, 2, 64, dtype=torch.float64), i(4), f)
    with pytest.raises(ValueError, match="host float64"):
        rb.rope(b(4, 2, 64), i(4), f.float())
    with pytest.raises(ValueError, match="CUDA"):
        rb.rope_kv_append(b(4, 2, 64), b(4, 1, 64), b(4, 1, 64), i(4), i(4), f, b(2, 8, 1, 64),
                          b(2, 8, 1, 64))
    with pytest.raises(TypeError):
        rb.rope_kv_append(b(4, 2, 64), b(4, 1, 64), b(4, 1, 64), i(4), i(4), f,
                          b(2, 8, 1, 64).half(), b(2, 8, 1, 64).half())
    with pytest.raises(ValueError, match="caches"):
        rb.rope_kv_append(b(4, 2, 64), b(4, 1, 64), b(4, 1, 64), i(4), i(4), f, b(2, 8, 2, 64),
                          b(2, 8, 2, 64))
    with pytest.raises(ValueError, match="CUDA"):
        rb.paged_attention(b(2, 4, 64), b(4, 8, 2, 64), b(4, 8, 2, 64), i(2, 3), i(2))
    with pytest.raises(ValueError, match="block_table"):
        rb.paged_attention(b(2, 4, 64), b(4, 8, 2, 64), b(4, 8, 2, 64), i(3, 3), i(2))


def test_the_plain_models_agree_with_themselves():
    """The block-table model: a step's slots are distinct and inside the cache, and releasing
    everything gives every block back."""
    rng = np.random.default_rng(0)
    R, bs, mb, nb = 9, 4, 12, 60
    table, free = np.full((R, mb), -1), rng.permutation(nb)
    lens, count = np.zeros(R, np.int64), nb
    for new in (rng.integers(0, 12, R), rng.integers(0, 12, R), np.full(R, -1)):
        w = ref.block_table(lens, new, table, free, count, bs, 200)
        lens, table, free, count = w["lens"], w["table"], w["free"], int(w["free_count"][0])
        live = w["slots"][w["slots"] >= 0]
        assert len(set(live)) == len(live) and (live < nb * bs).all()
    assert count == nb and sorted(free) == list(range(nb)) and not lens.any()
