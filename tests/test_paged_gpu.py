"""GPU parity: block tables, rotary positions, the cache append and single-token
attention over a paged cache, against plain 64-bit models."""
import math

import numpy as np
import pytest
import torch

from tests import _paged as ref

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32,
      "e4m3": torch.float8_e4m3fn}


def gen(seed=0):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


# ------------------------------------------------------------- block tables
def make_tables(lens, max_blocks, bs, spare, seed=0):
    """Tables whose blocks are a random permutation, and the stack of the rest."""
    rng = np.random.default_rng(seed)
    held = [-(-max(0, n) // bs) if n <= max_blocks * bs else 0 for n in lens]
    total = sum(held) + spare
    ids = rng.permutation(total)
    table = np.full((len(lens), max_blocks), -1, np.int64)
    at = 0
    for r, h in enumerate(held):
        table[r, :h] = ids[at:at + h]
        at += h
    free = np.full(max(total, 1), -7, np.int64)
    free[:spare] = ids[at:]
    return table, free, spare


def check_tables(rb, lens, new, max_blocks, bs, spare, max_tokens, seed=0, pad=0):
    table, free, count = make_tables(lens, max_blocks, bs, spare, seed)
    want = ref.block_table(lens, new, table, free, count, bs, max_tokens)
    t = torch.full((len(lens), max_blocks + pad), -9, dtype=torch.int32, device="cuda")
    t[:, :max_blocks] = i32(table)
    f = i32(free)
    args = (i32(lens), i32(new), t[:, :max_blocks], f, i32([count]))
    for _ in range(2):  # the same step twice: the same results
        got = rb.kv_block_table(*args, block_size=bs, max_tokens=max_tokens)
        for name in rb.KvStep._fields:
            np.testing.assert_array_equal(getattr(got, name).cpu().numpy(), want[name], name)
        np.testing.assert_array_equal(t[:, :max_blocks].cpu().numpy(), want["table"])
        np.testing.assert_array_equal(f.cpu().numpy(), want["free"])
        assert bool((t[:, max_blocks:] == -9).all())
    rb.synchronize_and_check()
    return got, want


@pytest.mark.parametrize("bs", [1, 7, 16, 64])
@pytest.mark.parametrize("R,seed", [(1, 0), (5, 1), (33, 2), (300, 3), (1025, 4)])
def test_block_table_random_steps(rb, bs, R, seed):
    rng = np.random.default_rng(seed)
    lens = rng.integers(0, 200, R)
    new = rng.choice([-1, 0, 1, 1, 1, 5, 40], R)
    mb = -(-260 // bs)
    tokens = int(np.maximum(new, 0).sum())
    need = sum(-(-(a + max(b, 0)) // bs) - -(-a // bs) for a, b in zip(lens, new))
    check_tables(rb, lens, new, mb, bs, spare=need, max_tokens=tokens + 13, seed=seed, pad=seed)
    # too few free blocks: some are refused
    check_tables(rb, lens, new, mb, bs, spare=max(0, need // 3), max_tokens=tokens, seed=seed)


@pytest.mark.parametrize("lens,new,mb,bs,spare,mt", [
    ([0], [0], 1, 16, 0, 0),                                # nothing at all
    ([0], [1], 1, 16, 1, 1),
    ([16], [1], 1, 16, 5, 1),                               # the table row is full
    ([15, 16, 17], [1, 1, 1], 2, 16, 1, 3),                 # only one opens a block
    ([0, 0, 0], [16, 17, 1], 2, 16, 3, 34),                 # the last is refused: stack empty
    ([0, 5, 0], [40, 1, 16], 3, 16, 2, 57),                 # dry first, the second needs none
    ([32, 32], [-1, 48], 3, 16, 0, 48),                     # takes the blocks just released
    ([0, 3, 0], [4, 4, 4], 2, 4, 6, 9),                     # the third passes max_tokens
    ([-3, 5, 99], [1, -2, 1], 4, 8, 4, 3),                  # bad length, bad count, bad length
    ([-3, 5, 99], [-1, -1, -1], 4, 8, 4, 0),                # releases of bad lengths
    ([0, 0], [2000000000, 2000000000], 4, 8, 4, 5),         # sums pass 32 bits
    ([3, 0, 7], [-1, -1, -1], 2, 4, 0, 8),                  # all released, padding only
])
def test_block_table_edges(rb, lens, new, mb, bs, spare, mt):
    check_tables(rb, lens, new, mb, bs, spare, mt)


def test_block_table_largest(rb):
    rng = np.random.default_rng(5)
    R = 8192
    lens = rng.integers(0, 64, R)
    new = rng.choice([-1, 1, 1, 9], R)
    check_tables(rb, lens, new, 10, 8, 8192, int(np.maximum(new, 0).sum()) + 1)
    check_tables(rb, [3], [70000], 4400, 16, 4400, 70007)


def test_block_table_in_place_and_many_steps(rb):
    """lens and free_count updated in place over steps, replayed from a graph."""
    R, bs, mb = 6, 4, 8
    table, free, count = make_tables([0] * R, mb, bs, R * mb)
    t, f, c = i32(table), i32(free), i32([count])
    lens, new = i32([0] * R), i32([3, 1, 4, 1, 5, 9])
    N = 30
    out = rb.KvStep(lens, c, *(torch.empty(n, dtype=torch.int32, device="cuda")
                               for n in (R + 1, N, N, N, R)))
    args = (lens, new, t, f, c)
    rb.kv_block_table(*args, block_size=bs, max_tokens=N, out=out)
    l, tt, ff, cc = np.zeros(R), table, free, count
    w = ref.block_table(l, new.cpu(), tt, ff, cc, bs, N)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        rb.kv_block_table(*args, block_size=bs, max_tokens=N, out=out)
    for step in ([1] * 6, [2, 0, -1, 1, 1, 1], [1, 1, 16, 1, 1, 9], [-1, -1, -1, 1, -1, -1]):
        for name in rb.KvStep._fields:
            np.testing.assert_array_equal(getattr(out, name).cpu().numpy(), w[name], name)
        new.copy_(i32(step))
        g.replay()
        torch.cuda.synchronize()
        w = ref.block_table(w["lens"], step, w["table"], w["free"], int(w["free_count"][0]), bs, N)
    for name in rb.KvStep._fields:
        np.testing.assert_array_equal(getattr(out, name).cpu().numpy(), w[name], name)
    np.testing.assert_array_equal(t.cpu().numpy(), w["table"])
    rb.synchronize_and_check()


def test_block_table_reports_bad_ids_and_counts(rb):
    lens, new = i32([4]), i32([2])
    t, f = i32([[77, -1]]), i32([3, 5, 1, 0])  # 77 is not a block
    got = rb.kv_block_table(lens, new, t, f, i32([4]), block_size=8, max_tokens=2)
    torch.cuda.synchronize()
    assert got.slots.tolist() == [-1, -1]
    with pytest.raises(rb.RemoraError, match="block id"):
        rb.synchronize_and_check()
    t = i32([[2, -1]])
    got = rb.kv_block_table(lens, i32([8]), t, f, i32([9]), block_size=8, max_tokens=8)
    assert got.slots.tolist() == [20, 21, 22, 23, 0, 1, 2, 3]  # the count is taken as 4
    with pytest.raises(rb.RemoraError, match="block id"):
        rb.synchronize_and_check()
    rb.synchronize_and_check()


# ------------------------------------------------------------------- rotary
def freqs(rot, base=10000.0):
    return base ** (-2.0 * torch.arange(rot // 2, dtype=torch.float64) / max(rot, 1))


def close(got, want, bound, what=""):
    d = (got.double().cpu() - want).abs()
    bad = ~(d <= bound)
    assert not bool(bad.any()), \
        f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((d / bound)[bad].max()):.3g}x"


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("B,S,H,D,rot,axes", [
    (1, 1, 1, 64, 64, 1), (2, 37, 3, 128, 128, 3), (1, 130, 5, 80, 80, 2), (3, 11, 2, 72, 72, 2),
    (2, 9, 4, 96, 32, 1), (1, 5, 2, 40, 6, 3), (2, 3, 1, 7, 2, 1), (1, 4, 2, 256, 256, 4), (1, 5, 3, 512, 256, 2), (2, 4, 2, 255, 100, 2),
    (1, 3, 2, 64, 0, 1), (1, 300, 48, 128, 64, 1)])
def test_rope_against_64_bits(rb, dtype, inter, B, S, H, D, rot, axes):
    g = gen(B * S + H)
    x = torch.randn(B, S, H, D, generator=g).to(DT[dtype])
    pos = torch.randint(0, 40000, (axes, B, S), generator=g, dtype=torch.int32)
    f = freqs(rot)
    ax = (torch.arange(rot // 2) % axes).to(torch.int32)
    for inverse in (False, True):
        got = rb.rope(x.cuda(), pos.cuda(), f, axis_of=ax, interleaved=inter, inverse=inverse)
        want = ref.rope(x, pos, f, ax, inter, inverse)
        close(got, want, ref.rope_bound(x, want, f, pos, DT[dtype], inter))
    # heads before positions, into a slice of a larger tensor, and in place
    xt = x.transpose(1, 2).contiguous().cuda().transpose(1, 2)
    room = torch.zeros(B, S, H + 1, D + 8, dtype=DT[dtype], device="cuda")
    got = rb.rope(xt, pos.cuda(), f, axis_of=ax, interleaved=inter, inverse=True,
                  out=room[:, :, :H, :D])
    close(got, want, ref.rope_bound(x, want, f, pos, DT[dtype], inter))
    assert not bool(room[:, :, H].any()) and not bool(room[..., D:].any())
    assert rb.rope(xt, pos.cuda(), f, axis_of=ax, interleaved=inter, inverse=True,
                   out=xt) is xt
    assert torch.equal(xt, got)


def test_rope_far_positions(rb):
    """Angles keep their precision at the ends of 32 bits and below zero."""
    pos = torch.tensor([[0, 1, -1, 2 ** 24 + 1, 2 ** 31 - 1, -2 ** 31, 123456789]],
                       dtype=torch.int32)
    x = torch.randn(7, 2, 128, generator=gen(1))
    for f in (freqs(128), freqs(128, 5e5), torch.tensor([-1.0, 0.0, 7.5, 1e-9] * 16,
                                                        dtype=torch.float64)):
        want = ref.rope(x, pos, f, None, False)
        got = rb.rope(x.cuda(), pos.cuda(), f)
        close(got, want, ref.rope_bound(x, want, f, pos, torch.float32, False))


def test_rope_gradient(rb):
    """inverse=True is the gradient: against autograd of the formula, and against differences."""
    B, S, H, D = 2, 5, 3, 64
    g = gen(2)
    x = torch.randn(B, S, H, D, generator=g, dtype=torch.float64)
    dy = torch.randn(B, S, H, D, generator=g)
    pos = torch.randint(0, 5000, (2, B, S), generator=g, dtype=torch.int32)
    f, ax = freqs(D), (torch.arange(32) % 2).to(torch.int32)
    leaf = x.clone().requires_grad_(True)
    half = D // 2
    ang = pos.double()[ax.long()].movedim(0, -1) * f
    c, s = ang.cos().unsqueeze(-2), ang.sin().unsqueeze(-2)
    a, b = leaf[..., :half], leaf[..., half:]
    y = torch.cat([a * c - b * s, a * s + b * c], -1)
    (y * dy.double()).sum().backward()
    got = rb.rope(dy.cuda(), pos.cuda(), f, axis_of=ax, inverse=True)
    close(got, leaf.grad, ref.rope_bound(dy, leaf.grad, f, pos, torch.float32, False))
    # differences of the forward kernel itself: linear, so a step of 1 is exact but for rounding
    x32 = x.float()
    e = torch.zeros_like(x32)
    e[1, 2, 1, 7] = 1.0
    up, dn = (rb.rope((x32 + k * e).cuda(), pos.cuda(), f, axis_of=ax).double().cpu()
              for k in (1, -1))
    diff = float(((up - dn) / 2 * dy.double()).sum())
    assert abs(diff - float(leaf.grad[1, 2, 1, 7])) <= 64 * 2.0 ** -21 * float(dy.abs().max()) * 4


def test_rope_empty(rb):
    x = torch.empty(0, 4, 64, device="cuda")
    assert rb.rope(x, torch.empty(0, dtype=torch.int32, device="cuda"), freqs(64)).shape == x.shape


# ------------------------------------------------------------------- append
def make_cache(nb, bs, Hkv, D, dt, layout, fill=None, seed=9):
    shape = (nb, Hkv, bs, D) if layout == "heads" else (nb, bs, Hkv, D)
    if fill is None:
        c = torch.randn(shape, generator=gen(seed)).clamp(-400, 400).to(dt)
    else:
        c = torch.full(shape, fill).to(dt)
    c = c.cuda()
    return c.transpose(1, 2) if layout == "heads" else c


@pytest.mark.parametrize("dtype,cache", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "e4m3"),
                                         ("f16", "e4m3")])
@pytest.mark.parametrize("T,Hq,Hkv,D,rot,bs,inter,layout", [
    (1, 8, 2, 64, 64, 16, False, "tokens"), (70, 4, 4, 128, 128, 16, True, "heads"),
    (33, 7, 1, 80, 80, 5, False, "tokens"), (9, 3, 3, 72, 18, 1, True, "heads"),
    (200, 32, 8, 128, 64, 64, False, "heads"), (5, 0, 2, 64, 32, 8, False, "tokens")])
def test_append(rb, dtype, cache, T, Hq, Hkv, D, rot, bs, inter, layout):
    g = gen(T)
    qkv = torch.randn(T, (Hq + 2 * Hkv) * D, generator=g).to(DT[dtype])
    nb = -(-T // bs) + 3
    slots = torch.randperm(nb * bs, generator=g)[:T].to(torch.int32)
    slots[::5] = -1
    pos = torch.randint(0, 9000, (1, T), generator=g, dtype=torch.int32)
    f = freqs(rot)
    scales = (0.031, 0.27) if cache == "e4m3" else (1.0, 1.0)
    kc, vc = (make_cache(nb, bs, Hkv, D, DT[cache], layout, seed=s) for s in (3, 4))
    kc0, vc0 = kc.float().cpu().double(), vc.float().cpu().double()
    dev = qkv.cuda()
    split = [a.view(T, h, D) for a, h in zip(dev.split([Hq * D, Hkv * D, Hkv * D], 1),
                                             (Hq, Hkv, Hkv))]
    q, k, v = (a.view(T, h, D) for a, h in zip(qkv.split([Hq * D, Hkv * D, Hkv * D], 1),
                                               (Hq, Hkv, Hkv)))
    got = rb.rope_kv_append(*split, pos.cuda(), slots.cuda(), f, kc, vc, interleaved=inter,
                            k_scale=scales[0], v_scale=scales[1])
    want = ref.rope(q, pos, f, None, inter)
    close(got, want, ref.rope_bound(q, want, f, pos, DT[dtype], inter), "q")
    assert torch.equal(dev.cpu(), qkv)
    kr = ref.rope(k, pos, f, None, inter)
    kb = ref.rope_bound(k, kr, f, pos, torch.float32, inter)
    live = (slots >= 0).nonzero()[:, 0]
    page, off = slots[live].long() // bs, slots[live].long() % bs
    for name, c, c0, row, b, sc in (("k", kc, kc0, kr, kb, scales[0]),
                                    ("v", vc, vc0, v.double(), torch.zeros_like(kb), scales[1])):
        w, tol = c0.clone(), torch.zeros_like(c0)
        r = row[live] / sc
        # stored: (f32 value, off by b) / scale (2^-24), then the cache type's half step and,
        # below its normal range, half its smallest subnormal
        e = b[live] / sc + r.abs() * 2.0 ** -23
        fi = torch.finfo(DT[cache])
        w[page, off] = r.clamp(-448, 448) if cache == "e4m3" else r
        tol[page, off] = e + fi.eps / 2 * (r.abs() + e) + fi.smallest_normal * fi.eps / 2
        close(c.float(), w, tol, name)
    rb.synchronize_and_check()


def test_append_e4m3_saturates_and_keeps_nan(rb):
    k = torch.tensor([1e4, -1e4, math.inf, -math.inf, math.nan, 448.0, 463.9, 0.0] * 8,
                     dtype=torch.bfloat16).view(1, 1, 64).cuda()
    kc = torch.zeros(1, 1, 1, 64, dtype=torch.float8_e4m3fn, device="cuda")
    vc = kc.clone()
    rb.rope_kv_append(k, k, k, i32([0]), i32([0]), freqs(0), kc, vc)
    want = [448.0, -448.0, 448.0, -448.0, math.nan, 448.0, 448.0, 0.0] * 8
    np.testing.assert_array_equal(vc.float().cpu().view(-1).numpy(), np.array(want, np.float32))


@pytest.mark.parametrize("scale", [0.031, 1.7e-30, 9.1e29, 3.0, 448.0])
def test_append_e4m3_rounds_as_the_division(rb, scale):
    """Values over the whole of bf16 (every exponent and mantissa, both signs): the stored byte
    is that of the exact quotient x / scale, rounded once."""
    bits = torch.arange(0, 1 << 16, 1, dtype=torch.int32)
    x = bits.to(torch.int16).view(torch.bfloat16)
    x = x[x.isfinite()][:65024].view(-1, 1, 64)
    T = x.shape[0]
    kc = torch.zeros(T, 1, 1, 64, dtype=torch.float8_e4m3fn, device="cuda")
    vc = kc.clone()
    rb.rope_kv_append(x.cuda(), x.cuda(), x.cuda(), i32(np.zeros(T)), i32(np.arange(T)), freqs(0),
                      kc, vc, k_scale=scale, v_scale=scale)
    # the quotient in 64 bits, rounded to 32 as the division is, then to 8
    s32 = float(np.float32(scale))
    want = (x.double() / s32).float().clamp(-448, 448).to(torch.float8_e4m3fn)
    for c in (kc, vc):
        assert torch.equal(c.view(T, 1, 64).cpu().float(), want.float())


def test_append_reports_bad_slots(rb):
    x = torch.ones(3, 1, 64, dtype=torch.bfloat16, device="cuda")
    kc = torch.zeros(2, 4, 1, 64, dtype=torch.bfloat16, device="cuda")
    vc = kc.clone()
    rb.rope_kv_append(x, x, x, i32([0, 0, 0]), i32([8, -2, 7]), freqs(64), kc, vc)
    torch.cuda.synchronize()
    assert bool((kc.view(8, 64)[:7] == 0).all()) and bool((vc.view(8, 64)[7] == 1).all())
    with pytest.raises(rb.RemoraError, match="slot"):
        rb.synchronize_and_check()
    rb.synchronize_and_check()


# ---------------------------------------------------------------- attention
def make_pages(lens, bs, max_blocks, seed):
    rng = np.random.default_rng(seed)
    held = [-(-n // bs) for n in lens]
    ids = rng.permutation(sum(held) + 2)
    table = np.full((len(lens), max_blocks), -1, np.int64)
    at = 0
    for r, h in enumerate(held):
        table[r, :h] = ids[at:at + h]
        at += h
    return table, sum(held) + 2


def check_attention(rb, lens, Hq, Hkv, D, bs, dtype, cache, layout="tokens", window=0, scale=None,
                    poison=True, qscale=2.0, seed=0, q=None, pad=0, want_lse=True):
    g = gen(seed)
    R = len(lens)
    mb = max(1, max(-(-n // bs) for n in lens)) + pad
    table, nb = make_pages(lens, bs, mb, seed)
    sc = (0.07, 0.11) if cache == "e4m3" else (1.0, 1.0)
    kc, vc = (make_cache(nb, bs, Hkv, D, DT[cache], layout, seed=seed + s) for s in (1, 2))
    if cache == "e4m3":
        kc, vc = ((c.float() * 14).clamp(-448, 448).to(DT[cache]) for c in (kc, vc))
    kf, vf = kc.float().cpu(), vc.float().cpu()
    if poison:  # rows of no request hold NaN and infinities
        used = torch.zeros(nb, bs, dtype=torch.bool)
        for r, n in enumerate(lens):
            for j in range(n):
                used[table[r, j // bs], j % bs] = True
        for c in (kc, vc):
            c.view(torch.uint8).masked_fill_(~used.cuda()[:, :, None, None], 0x7f)
    if q is None:
        q = (torch.randn(R, Hq, D, generator=g) * qscale).to(DT[dtype])
    s = D ** -0.5 if scale is None else scale
    lse = torch.full((R, Hq), 5.0, device="cuda") if want_lse else None
    args = (q.cuda(), kc, vc, i32(table), i32(lens))
    kw = dict(scale=scale, window=window, k_scale=sc[0], v_scale=sc[1])
    out = rb.paged_attention(*args, lse=lse, **kw)
    rb.synchronize_and_check()
    for r, n in enumerate(lens):
        first = max(0, n - window) if window else 0
        j = np.arange(first, n)
        page = torch.from_numpy(table[r, j // bs]).long()
        k, v = (c[page, torch.from_numpy(j % bs)] * w for c, w in
                ((kf.double(), sc[0]), (vf.double(), sc[1])))
        o, l, mag, size = ref.attention(q[r], k, v, s)
        vmax = float(v.abs().max()) if len(j) else 0.0
        b, bl = ref.attention_bound(o, l, mag, size, len(j), D, DT[dtype], vmax, DT[cache])
        if len(j) == 0:
            assert not bool(out[r].any())
            assert not want_lse or bool((lse[r] == -math.inf).all())
            continue
        close(out[r], o, b, f"request {r} of {n} keys")
        if want_lse:
            close(lse[r], l, bl, f"lse of request {r}")
    again = rb.paged_attention(*args, **kw)
    assert torch.equal(out.view(torch.int16), again.view(torch.int16))
    return out, args, kw


TYPES = [("bf16", "bf16"), ("f16", "f16"), ("bf16", "e4m3"), ("f16", "e4m3")]


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("Hq,Hkv,D", [(8, 2, 64), (32, 8, 128), (7, 1, 128), (12, 1, 128),
                                      (16, 1, 64), (5, 5, 64), (6, 2, 256), (16, 1, 256),
                                      (40, 1, 128)])
@pytest.mark.parametrize("lens,bs,layout", [
    ([1], 16, "tokens"), ([17, 0, 33, 1, 500], 16, "heads"), ([130, 64, 65, 63, 0], 5, "tokens")])
def test_attention_shapes(rb, dtype, cache, Hq, Hkv, D, lens, bs, layout):
    check_attention(rb, lens, Hq, Hkv, D, bs, dtype, cache, layout)


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("lens", [[5000], [3001, 2, 1, 0, 0, 900], list(range(70))])
@pytest.mark.parametrize("window", [0, 1, 100, 1000])
def test_attention_lengths_and_windows(rb, dtype, cache, lens, window):
    check_attention(rb, lens, 8, 2, 128, 16, dtype, cache, window=window, pad=3)


@pytest.mark.parametrize("bs", [1, 3, 16, 24, 128, 4096])
def test_attention_block_sizes(rb, bs):
    check_attention(rb, [4000, 31, 129], 4, 2, 64, bs, "bf16", "bf16", "heads")


@pytest.mark.parametrize("dtype,cache", TYPES)
def test_attention_many_requests(rb, dtype, cache):
    """More requests than workers, each short: whole requests per worker."""
    lens = [int(n) for n in np.random.default_rng(3).integers(0, 60, 700)]
    check_attention(rb, lens, 8, 4, 64, 8, dtype, cache, poison=False)


def test_attention_one_long_request(rb):
    """One request over every worker: the join of many pieces."""
    check_attention(rb, [40001], 4, 1, 64, 16, "bf16", "bf16", poison=False)
    check_attention(rb, [40001], 2, 2, 128, 16, "f16", "e4m3", poison=False)


def test_attention_zero_and_negative_scale(rb):
    check_attention(rb, [100, 3], 4, 2, 64, 16, "bf16", "bf16", scale=0.0)
    check_attention(rb, [100, 3], 4, 2, 64, 16, "f16", "f16", scale=-0.3)


@pytest.mark.parametrize("dtype,cache", TYPES)
def test_attention_sharp_scores(rb, dtype, cache):
    """Scores tens apart: nearly all weight on one key, maxima that keep rising."""
    check_attention(rb, [900, 64], 8, 1, 128, 16, dtype, cache, qscale=30.0)


@pytest.mark.parametrize("qscale", [1e-30, 1e30])
def test_attention_extreme_queries_over_8_bit_keys(rb, qscale):
    """bf16 queries beyond f16's range, over e4m3 keys."""
    q = (torch.randn(2, 4, 64, generator=gen(1)) * qscale).to(torch.bfloat16)
    check_attention(rb, [300, 40], 4, 2, 64, 16, "bf16", "e4m3", scale=1.0 / qscale / 8, q=q)


def test_attention_infinite_and_nan_keys(rb):
    """A NaN in a used row makes that head's output NaN; scores that are all -inf leave an
    empty row; one key at +inf is NaN as the formula says (inf - inf)."""
    R, D, bs = 4, 64, 16
    kc = torch.zeros(8, bs, 1, D, dtype=torch.bfloat16, device="cuda")
    vc = torch.ones_like(kc)
    q = torch.ones(R, 1, D, dtype=torch.bfloat16, device="cuda")
    kc[0, 3, 0, 5] = math.nan
    kc[1, :, 0, 0] = -math.inf
    kc[2, 2, 0, 0] = math.inf
    kc[3, 2, 0, 0] = -math.inf
    lse = torch.empty(R, 1, device="cuda")
    out = rb.paged_attention(q, kc, vc, i32([[0], [1], [2], [3]]), i32([16, 16, 16, 16]), lse=lse)
    assert bool(out[0].isnan().all()) and bool(lse[0].isnan().all())
    assert not bool(out[1].any()) and float(lse[1]) == -math.inf
    assert bool(out[2].isnan().all())
    assert bool((out[3] == 1).all()) and abs(float(lse[3]) - math.log(15)) < 1e-5
    rb.synchronize_and_check()


def test_attention_reports_bad_pages_and_lengths(rb):
    """A page outside the cache is skipped and reported; so is a length past the table."""
    D, bs = 64, 16
    kc = torch.randn(4, bs, 1, D, generator=gen(4)).to(torch.bfloat16).cuda()
    vc = torch.randn(4, bs, 1, D, generator=gen(5)).to(torch.bfloat16).cuda()
    q = torch.randn(1, 2, D, generator=gen(6)).to(torch.bfloat16).cuda()
    want = rb.paged_attention(q, kc, vc, i32([[1, 3]]), i32([32]))
    rb.synchronize_and_check()
    got = rb.paged_attention(q, kc, vc, i32([[1, 9, 3]]), i32([48]))
    torch.cuda.synchronize()
    assert float((got.float() - want.float()).abs().max()) <= 2 ** -6
    with pytest.raises(rb.RemoraError, match="block id"):
        rb.synchronize_and_check()
    for bad, same in ((99, 32), (-5, 0)):
        got = rb.paged_attention(q, kc, vc, i32([[1, 3]]), i32([bad]))
        with pytest.raises(rb.RemoraError, match="length"):
            rb.synchronize_and_check()
        assert torch.equal(got, rb.paged_attention(q, kc, vc, i32([[1, 3]]), i32([same])))
    rb.synchronize_and_check()


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("size", [3e2, 3e4])
def test_attention_huge_scores(rb, dtype, cache, size):
    """Scores of 1e5 to 1e10, where their own rounding exceeds a factor of two of a weight: the
    result stays a mean of the values, and where one key leads by far it is that key's value."""
    D, n = 128, 70
    g = gen(3)
    k = torch.randn(n, 1, D, generator=g).sign() * (size if cache != "e4m3" else 448.0)
    v = torch.randn(n, 1, D, generator=g)
    q = torch.randn(1, 2, D, generator=g).sign() * size
    q[0, 1] = k[17, 0] / k[17, 0].abs() * size  # head 1 is key 17's own direction
    kc, vc = torch.zeros(5, 16, 1, D).to(DT[cache]), torch.zeros(5, 16, 1, D).to(DT[cache])
    kc.view(80, 1, D)[:n], vc.view(80, 1, D)[:n] = k.to(DT[cache]), v.to(DT[cache])
    out = rb.paged_attention(q.to(DT[dtype]).cuda(), kc.cuda(), vc.cuda(), i32([[0, 1, 2, 3, 4]]),
                             i32([n]), scale=1.0)
    vs = vc.view(80, D)[:n].float()
    assert bool(out.isfinite().all()) and float(out.float().abs().max()) <= float(vs.abs().max())
    assert torch.equal(out[0, 1].float().cpu(), vs[17].to(DT[dtype]).float())


def test_attention_most_requests(rb):
    """8192 requests, every other one empty, lengths of 0 to 3."""
    R, D, bs = 8192, 64, 4
    g = gen(2)
    lens = torch.arange(R) % 4
    kc = torch.randn(R, bs, 2, D, generator=g).to(torch.bfloat16).cuda()
    vc = torch.randn(R, bs, 2, D, generator=g).to(torch.bfloat16).cuda()
    q = torch.randn(R, 4, D, generator=g).to(torch.bfloat16).cuda()
    out = rb.paged_attention(q, kc, vc, i32(np.arange(R))[:, None], i32(lens))
    j = torch.arange(bs, device="cuda")
    s = torch.einsum("rgd,rjgd->rgj", q.double().view(R, 2, 2, D).flatten(1, 2),
                     kc.double().repeat_interleave(2, 2)) / 8
    s = s.masked_fill(j >= lens.cuda()[:, None, None], -math.inf)
    want = torch.einsum("rgj,rjgd->rgd", torch.softmax(s, -1).nan_to_num(0.0),
                        vc.double().repeat_interleave(2, 2))
    # half a step of bf16, and below it what four weights' roundings leave (2^-17 each) with room
    assert bool(((out.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -12).all())
    assert not bool(out[::4].any())
    rb.synchronize_and_check()


def test_attention_window_over_freed_pages(rb):
    """Table entries wholly in front of the window may be anything."""
    out, args, kw = check_attention(rb, [100, 33, 64], 4, 2, 64, 16, "bf16", "bf16", window=20)
    table = args[3].clone()
    table[0, :5] = -1       # keys 80 on count
    table[2, :2] = 1 << 30  # keys 44 on
    got = rb.paged_attention(*args[:3], table, args[4], **kw)
    assert torch.equal(got, out)
    rb.synchronize_and_check()


def test_attention_table_and_cache_strides(rb):
    """A table that is a slice of a wider one; keys heads first, values tokens first."""
    out, args, kw = check_attention(rb, [70, 300, 5], 8, 2, 128, 16, "f16", "f16")
    q, kc, vc, table, lens = args
    wide = torch.full((3, table.shape[1] + 5), -3, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    kh = kc.transpose(1, 2).contiguous().transpose(1, 2)
    assert kh.stride() != vc.stride()
    assert torch.equal(rb.paged_attention(q, kh, vc, wide[:, :table.shape[1]], lens, **kw), out)
    rb.synchronize_and_check()


def test_attention_in_a_graph_behind_copies(rb):
    """Captured right behind a copy of its lengths and a fill of its output, each replay sees the
    new lengths (the launch may be set up before the copy is done, but must wait for it)."""
    out, args, kw = check_attention(rb, [900, 20, 7], 8, 2, 128, 16, "bf16", "bf16")
    q, kc, vc, table, lens = args
    room, src = torch.empty_like(out), lens.clone()
    now = torch.zeros_like(lens)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        room.fill_(9)
        now.copy_(src)
        rb.paged_attention(q, kc, vc, table, now, out=room, **kw)
        again = room.clone()
    for new in ([900, 20, 7], [0, 20, 3], [899, 1, 0], [900, 20, 7]):
        src.copy_(i32(new))
        want = rb.paged_attention(q, kc, vc, table, src, **kw)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(again, want) and torch.equal(room, want)


def test_calls_refuse_mixed_devices_and_bad_buffers(rb):
    """Each refusal comes before any launch; the next good call is not disturbed."""
    out, (q, kc, vc, table, lens), kw = check_attention(rb, [40, 3], 4, 2, 64, 16, "bf16", "bf16")
    need = rb.paged_attention_workspace_bytes(2, 4, 2, 64)
    small = torch.empty(need - 1, dtype=torch.uint8, device="cuda")
    odd = torch.empty(need + 8, dtype=torch.uint8, device="cuda")[8:]
    for bad in (dict(out=q), dict(workspace=small), dict(workspace=odd), dict(window=-1),
                dict(k_scale=0.5), dict(scale=math.nan)):
        with pytest.raises(rb.RemoraError):
            rb.paged_attention(q, kc, vc, table, lens, **{**kw, **bad})
    for args in ((q.cpu(), kc, vc, table, lens), (q, kc, vc, table.cpu(), lens),
                 (q, kc, vc, table, lens.long()), (q[:1], kc, vc, table, lens),
                 (q, kc, vc[:-1], table, lens), (q, kc, vc, table.t(), lens)):
        with pytest.raises((ValueError, TypeError)):
            rb.paged_attention(*args, **kw)
    x, pos = torch.ones(3, 2, 64, device="cuda"), i32([0, 1, 2])
    for args in ((x.cpu(), pos, freqs(64)), (x, pos.cpu(), freqs(64)), (x, pos, freqs(64).cuda()),
                 (x, pos[:2], freqs(64)), (x.transpose(1, 2), pos, freqs(4))):
        with pytest.raises((ValueError, TypeError)):
            rb.rope(*args)
    t, f, c = i32([[0, 1]]), i32([2, 3]), i32([2])
    for args in ((i32([1]).cpu(), i32([1]), t, f, c), (i32([1]), i32([1]), t, f, c.long()),
                 (i32([1]), i32([1, 1]), t, f, c), (i32([1]), i32([1]), t.t(), f, c)):
        with pytest.raises((ValueError, TypeError)):
            rb.kv_block_table(*args, block_size=4, max_tokens=1)
    assert torch.equal(rb.paged_attention(q, kc, vc, table, lens, **kw), out)
    rb.synchronize_and_check()


def test_attention_strided_q_and_out(rb):
    D = 128
    out, args, kw = check_attention(rb, [70, 0, 5], 8, 2, D, 16, "bf16", "bf16")
    q = torch.zeros(3, 20, D, dtype=torch.bfloat16, device="cuda")
    q[:, 4:20:2] = args[0]
    room = torch.full((4, 8, D + 8), 7.0, dtype=torch.bfloat16, device="cuda")
    got = rb.paged_attention(q[:, 4:20:2], *args[1:], out=room[:3, :, :D], **kw)
    assert torch.equal(got, out)
    assert bool((room[3] == 7).all()) and bool((room[..., D:] == 7).all())  # rows behind are left


def test_attention_streams_and_graphs(rb):
    """Two streams at once and two captured graphs give what one call gives."""
    cases = [check_attention(rb, [3000, 20, 7], 8, 2, 128, 16, "bf16", "bf16", seed=s)
             for s in (0, 5)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(5):
        got = []
        for (_, args, kw), st in zip(cases, streams):
            with torch.cuda.stream(st):
                got.append(rb.paged_attention(*args, **kw))
        torch.cuda.synchronize()
        for (want, _, _), o in zip(cases, got):
            assert torch.equal(o, want)
    graphs = []
    for _, args, kw in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o = rb.paged_attention(*args, **kw)
        graphs.append((g, o))
    for _ in range(3):
        for (g, o), st in zip(graphs, streams):
            o.zero_()
        torch.cuda.synchronize()
        for (g, o), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for (want, _, _), (g, o) in zip(cases, graphs):
            assert torch.equal(o, want)


def test_attention_past_32_bit_offsets(rb):
    """A cache of more than 2^32 elements: pages at its far end."""
    bs, Hkv, D = 64, 8, 128
    nb = (1 << 32) // (bs * Hkv * D) + 40
    kc = torch.zeros(nb, bs, Hkv, D, dtype=torch.bfloat16, device="cuda")
    vc = torch.zeros_like(kc)
    ids = [nb - 1, 3, nb - 17, nb - 2]
    g = gen(8)
    for i in ids:
        kc[i] = torch.randn(bs, Hkv, D, generator=g).to(torch.bfloat16)
        vc[i] = torch.randn(bs, Hkv, D, generator=g).to(torch.bfloat16)
    n, Hq = 4 * bs - 5, 16
    q = torch.randn(1, Hq, D, generator=g).to(torch.bfloat16)
    out = rb.paged_attention(q.cuda(), kc, vc, i32([ids]), i32([n]))
    k = torch.cat([kc[i].cpu() for i in ids])[:n]
    v = torch.cat([vc[i].cpu() for i in ids])[:n]
    o, l, mag, size = ref.attention(q[0], k, v, D ** -0.5)
    close(out[0], o, ref.attention_bound(o, l, mag, size, n, D, torch.bfloat16, 5.0)[0])
    # and the append there
    x = torch.randn(1, Hkv, D, generator=g).to(torch.bfloat16).cuda()
    rb.rope_kv_append(x, x, x, i32([0]), i32([(nb - 1) * bs + 7]), freqs(128), kc, vc)
    assert torch.equal(kc[nb - 1, 7], x[0]) and torch.equal(vc[nb - 1, 7], x[0])
    rb.synchronize_and_check()


# ------------------------------------------------------------- the step together
@pytest.mark.parametrize("config", [None, "3x8x2x100", "1x16x1x5000", "40x4x4x33"])
def test_run_test_decode(rb, config):
    rep = rb.run_test("decode", iters=2, warmup=1, config=config)
    assert rep["passed"] and rep["checked"] == 32 * 128 and rep["max_rel_err"] <= 2e-2


def test_cli_decode(rb, tmp_path):
    import os
    import subprocess

    from remora_b200 import build

    prog = tmp_path / "prog.mlir"
    prog.write_text("func.func public @main()\n")
    r = subprocess.run([build.CLI, str(prog), "--run-gpu", "--test=decode",
                        "--config=2x8x4x300"], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "Validation: PASS" in r.stdout and "decode step" in r.stdout
    assert os.path.exists(build.CLI)


@pytest.mark.parametrize("dtype,cache", TYPES)
def test_serving_steps(rb, dtype, cache):
    """Prompts, then decoding steps, a release and a newcomer: tables, append and attention in
    turn, against attention over each request's own history in 64 bits."""
    R, Hq, Hkv, D, bs, mb = 3, 8, 2, 64, 8, 12
    nb = 20
    g = gen(11)
    dt, scales = DT[dtype], ((0.02, 0.03) if cache == "e4m3" else (1.0, 1.0))
    kc, vc = (make_cache(nb, bs, Hkv, D, DT[cache], "tokens", fill=math.nan) for _ in range(2))
    table, free = torch.full((R, mb), -1, dtype=torch.int32, device="cuda"), i32(np.arange(nb))
    lens, count = i32([0] * R), i32([nb])
    f = freqs(D)
    hist = [[], [], []]
    for new in ([30, 1, 9], [1, 1, 1], [1, -1, 1], [1, 20, 1], [1, 1, 1]):
        T = sum(max(n, 0) for n in new)
        st = rb.kv_block_table(lens, i32(new), table, free, count, block_size=bs, max_tokens=T + 2)
        lens, count = st.lens, st.free_count
        assert st.status.tolist() == [0] * R
        q, k, v = (torch.randn(T + 2, h, D, generator=g).to(dt).cuda() for h in (Hq, Hkv, Hkv))
        qr = rb.rope_kv_append(q, k, v, st.positions, st.slots, f, kc, vc, k_scale=scales[0],
                               v_scale=scales[1])
        rows = st.slots.tolist()
        kk, vv = (c.float().cpu().double().view(nb * bs, Hkv, D) * s for c, s in
                  zip((kc, vc), scales))
        at = 0
        last = []
        for r, n in enumerate(new):
            hist[r] = [] if n < 0 else hist[r] + rows[at:at + n]
            at += max(n, 0)
            last.append(max(at - 1, 0))
        qd = qr[torch.tensor(last, device="cuda")]
        out = rb.paged_attention(qd, kc, vc, table, lens, k_scale=scales[0], v_scale=scales[1])
        rb.synchronize_and_check()
        assert len({s for h in hist for s in h}) == sum(len(h) for h in hist)
        for r in range(R):
            h = torch.tensor(hist[r], dtype=torch.long)
            if len(h) == 0:
                assert not bool(out[r].any())
                continue
            # the newest key is in the cache as it was rotated at its own position
            kw = ref.rope(k[last[r]].cpu()[None], st.positions[last[r]].cpu().view(1, 1), f, None,
                          False)[0]
            fi = torch.finfo(DT[cache])
            assert bool(((kk[h[-1]] - kw).abs() <= fi.eps / 2 * 1.01 * kw.abs() +
                         scales[0] * fi.smallest_normal * fi.eps + 2e-6).all())
            o, l, mag, size = ref.attention(qd[r].cpu(), kk[h], vv[h], D ** -0.5)
            b = ref.attention_bound(o, l, mag, size, len(h), D, dt, float(vv[h].abs().max()),
                                    DT[cache])[0]
            close(out[r], o, b, f"request {r}")
