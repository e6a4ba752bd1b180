"""CPU tests: the decoding entry points reject bad arguments on the host, before
any CUDA call, and their Python mirrors reject bad tensors."""
import ctypes

import numpy as np
import pytest
import torch

import remora_b200 as rb
from tests import _paged as ref

A = ctypes.c_void_p(1 << 20)
ODD = ctypes.c_void_p((1 << 20) + 8)


@pytest.fixture(scope="module")
def L():
    from remora_b200 import build

    build.build()
    return rb.lib()


def tables(L, **c):
    d = dict(lens=A, new=A, R=4, table=A, ld=8, mb=8, free=A, count=A, nb=32, bs=16, lo=A, co=A,
             cu=A, slots=A, pos=A, req=A, mt=4, status=A)
    d.update(c)
    return L.remora_b200_kv_block_table(*d.values(), None)


@pytest.mark.parametrize("bad", [
    dict(R=-1), dict(R=8193), dict(mt=-1), dict(mt=2 ** 31 - 1), dict(bs=0), dict(nb=0),
    dict(nb=2 ** 27, bs=16), dict(mb=0), dict(mb=2 ** 27, ld=2 ** 27), dict(ld=7), dict(lens=None),
    dict(new=None), dict(table=None), dict(free=None), dict(count=None), dict(lo=None),
    dict(co=None), dict(cu=None), dict(slots=None), dict(pos=None), dict(req=None),
    dict(status=None)])
def test_block_table_refuses(L, bad):
    assert tables(L, **bad) == rb.ERR_INVALID and "kv_block_table" in rb.last_error()


FREQ = (ctypes.c_double * 64)(*[0.5] * 64)
AXES = (ctypes.c_int32 * 64)(*[0] * 63, 1)


def rope(L, **c):
    d = dict(x=A, out=A, dt=rb.BF16, B=1, S=4, H=2, D=128, xb=0, xs=256, xh=128, ob=0, os=256,
             oh=128, pos=A, ld=4, axes=1, freq=FREQ, ax=None, rot=128, inter=0, inv=0)
    d.update(c)
    return L.remora_b200_rope(*d.values(), None)


@pytest.mark.parametrize("bad", [
    dict(x=None), dict(out=None), dict(dt=rb.E4M3), dict(dt=9), dict(B=-1), dict(S=-1), dict(H=-1),
    dict(D=0), dict(D=2048), dict(pos=None), dict(ld=3, axes=2), dict(axes=0), dict(axes=9),
    dict(freq=None), dict(ax=AXES), dict(rot=3), dict(rot=130), dict(rot=258, D=512),
    dict(x=ctypes.c_void_p((1 << 20) + 1)), dict(freq=(ctypes.c_double * 64)(*[float("nan")] * 64)),
    dict(freq=(ctypes.c_double * 64)(*[float("inf")] * 64))])
def test_rope_refuses(L, bad):
    assert rope(L, **bad) == rb.ERR_INVALID and "rope" in rb.last_error()


def test_rope_without_rows_is_done(L):
    assert rope(L, S=0, ld=0, pos=None, x=None, out=None) == rb.OK
    assert rope(L, H=0, x=None, out=None) == rb.OK


def append(L, **c):
    d = dict(q=A, k=A, v=A, qo=A, dt=rb.BF16, T=4, Hq=4, Hkv=2, D=128, qt=512, qh=128, kt=256,
             kh=128, vt=256, vh=128, ot=512, oh=128, pos=A, ld=4, axes=1, freq=FREQ, ax=None,
             rot=128, inter=0, slots=A, kc=A, vc=A, cdt=rb.BF16, nb=4, bs=16, kb=4096, ktok=256,
             khd=128, vb=4096, vtok=256, vhd=128, ks=1.0, vs=1.0)
    d.update(c)
    return L.remora_b200_rope_kv_append(*d.values(), None)


@pytest.mark.parametrize("bad", [
    dict(q=None), dict(k=None), dict(v=None), dict(qo=None), dict(slots=None), dict(kc=None),
    dict(vc=None), dict(pos=None), dict(dt=rb.F32), dict(cdt=rb.F16), dict(T=-1), dict(Hkv=0),
    dict(nb=0), dict(bs=0), dict(nb=2 ** 28), dict(ks=0.0), dict(vs=-1.0), dict(ks=2.0),
    dict(cdt=rb.E4M3, ks=float("nan")), dict(cdt=rb.E4M3, vs=float("inf")), dict(rot=200),
    dict(kc=ctypes.c_void_p((1 << 20) + 1))])
def test_append_refuses(L, bad):
    assert append(L, **bad) == rb.ERR_INVALID and "rope_kv_append" in rb.last_error()


def attention(L, **c):
    d = dict(q=A, kc=A, vc=A, table=A, lens=A, out=A, lse=None, dt=rb.BF16, cdt=rb.BF16, R=2, Hq=8,
             Hkv=2, D=128, qt=1024, qh=128, ot=1024, oh=128, nb=8, bs=16, kb=4096, kt=256, kh=128,
             vb=4096, vt=256, vh=128, ld=8, mb=8, scale=1.0, window=0, ks=1.0, vs=1.0, ws=A,
             wsb=1 << 40)
    d.update(c)
    return L.remora_b200_paged_attention(*d.values(), None)


@pytest.mark.parametrize("bad", [
    dict(q=None), dict(kc=None), dict(vc=None), dict(table=None), dict(lens=None), dict(out=None),
    dict(q=ODD), dict(kc=ODD), dict(vc=ODD), dict(out=ODD), dict(ws=ODD), dict(ws=None),
    dict(wsb=0), dict(dt=rb.F32), dict(cdt=rb.F16), dict(R=-1), dict(R=8193), dict(Hq=7),
    dict(Hkv=0), dict(Hq=0), dict(D=96), dict(nb=0), dict(bs=0), dict(nb=2 ** 28), dict(mb=0),
    dict(ld=7), dict(mb=2 ** 28, ld=2 ** 28), dict(scale=float("nan")), dict(scale=float("inf")),
    dict(window=-1), dict(ks=0.5), dict(vs=2.0), dict(cdt=rb.E4M3, ks=0.0),
    dict(cdt=rb.E4M3, kt=264), dict(qt=1020), dict(oh=4), dict(kt=12), dict(vb=4)])
def test_attention_refuses(L, bad):
    assert attention(L, **bad) == rb.ERR_INVALID and "paged_attention" in rb.last_error()


def test_attention_without_requests_is_done_and_workspace_sizes(L):
    assert attention(L, R=0, q=None, ws=None, wsb=0) == rb.OK
    assert L.remora_b200_paged_attention_workspace_bytes(8, 32, 8, 128) > 0
    for bad in ((-1, 8, 2, 128), (8, 7, 2, 128), (8, 8, 0, 128), (8, 8, 2, 80), (9000, 8, 2, 128)):
        assert L.remora_b200_paged_attention_workspace_bytes(*bad) == 0


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
