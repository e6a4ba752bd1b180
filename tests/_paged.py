"""Plain 64-bit models of the decoding operators, and the tolerances that follow
from how the kernels compute (see each function)."""
import math

import numpy as np
import torch


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


# ------------------------------------------------------------- block tables
def block_table(lens, new, table, free, count, bs, max_tokens):
    """The step of kv_block_table, request by request."""
    lens, new, table, free = (np.array(np.asarray(x), dtype=np.int64) for x in (lens, new, table, free))
    R, max_blocks = table.shape
    room = max_blocks * bs
    need_blocks = lambda n: -(-n // bs)  # noqa: E731
    out_lens, status = lens.copy(), np.zeros(R, np.int64)
    cu = np.zeros(R + 1, np.int64)
    top = count
    for r in range(R):  # released blocks first
        if new[r] == -1 and 0 <= lens[r] <= room:
            for p in range(need_blocks(lens[r])):
                free[top] = table[r, p]
                top += 1
            out_lens[r] = 0
    left, dry = top, False
    wanted = 0
    slots = np.full(max_tokens, -1)
    pos = np.zeros(max_tokens, np.int64)
    req = np.full(max_tokens, -1)
    for r in range(R):
        n = max(new[r], 0)
        cu[r + 1] = cu[r] + n
        req[cu[r]:min(cu[r + 1], max_tokens)] = r
        held_ok = 0 <= lens[r] <= room
        if new[r] < 0:
            status[r] = 0 if new[r] == -1 and held_ok else 2
            continue
        if not held_ok or lens[r] + n > room or cu[r + 1] > max_tokens:
            status[r] = 2
            continue
        own, need = need_blocks(lens[r]), need_blocks(lens[r] + n) - need_blocks(lens[r])
        wanted += need
        if need and wanted > top:
            dry = True
            status[r] = 1
            continue
        assert not (dry and need)
        for p in range(own, own + need):
            left -= 1
            table[r, p] = free[left]
        for j in range(n):
            p = lens[r] + j
            slots[cu[r] + j] = table[r, p // bs] * bs + p % bs
            pos[cu[r] + j] = p
        out_lens[r] = lens[r] + n
    return dict(lens=out_lens, free_count=np.array([left]), cu_tokens=np.minimum(cu, 2 ** 31 - 1), slots=slots,
                positions=pos, requests=req, status=status, table=table, free=free)


# ------------------------------------------------------------------- rotary
def rope(x, pos, freq, axis_of, interleaved, inverse=False):
    """x [..., H, D] in 64 bits; pos [axes, ...]."""
    x = x.double().cpu()
    half = freq.numel()
    ax = torch.zeros(half, dtype=torch.long) if axis_of is None else axis_of.long()
    ang = pos.cpu().double()[ax].movedim(0, -1) * freq
    c, s = ang.cos().unsqueeze(-2), ang.sin().unsqueeze(-2)
    s = -s if inverse else s
    lo = torch.arange(half) * 2 if interleaved else torch.arange(half)
    hi = lo + 1 if interleaved else lo + half
    y = x.clone()
    y[..., lo] = x[..., lo] * c - x[..., hi] * s
    y[..., hi] = x[..., lo] * s + x[..., hi] * c
    return y


def rope_bound(x, ref, freq, pos, dtype, interleaved):
    """How far a rotated element may be from its 64-bit value.

    Output rounding: half a step of the value.  Before it, in f32: the angle's
    rest is rounded by 2^-25 of at most pi/4, sincospif by at most 2 ulp
    (2^-23 of at most 1), then two products and a sum (at most 2^-24 each of
    the pair's magnitude): below 2^-21 (|a| + |b|) together.  The reference's
    own angle is a rounded product, off by 2^-53 of itself."""
    half = freq.numel()
    x = x.double().cpu().abs()
    lo = torch.arange(half) * 2 if interleaved else torch.arange(half)
    hi = lo + 1 if interleaved else lo + half
    far = float(pos.abs().max()) * float(freq.abs().max() if half else 0) * 2.0 ** -52
    b = torch.zeros_like(x)
    b[..., lo] = b[..., hi] = (x[..., lo] + x[..., hi]) * (2.0 ** -21 + far)
    # a value within b of a rounding border may go either way: half a step of it and of b
    return half_step(dtype) * (ref.abs() + b) + b + torch.finfo(dtype).smallest_normal * \
        torch.finfo(dtype).eps / 2 * (1 if dtype != torch.float32 else 0)


# ---------------------------------------------------------------- attention
def attention(q, k, v, scale):
    """One request: q [Hq, D], k and v [n, Hkv, D] in 64 bits -> out, lse, and the
    weighted magnitude sum_j p_j |v_j| and the scores' error that bounds need."""
    q, k, v = q.double(), k.double(), v.double()
    Hq, D = q.shape
    n, Hkv, _ = k.shape
    if n == 0:
        z = torch.zeros(Hq, D, dtype=torch.float64)
        return z, torch.full((Hq,), -math.inf, dtype=torch.float64), z, torch.zeros(Hq)
    g = Hq // Hkv
    kk = k.repeat_interleave(g, 1).permute(1, 0, 2)
    vv = v.repeat_interleave(g, 1).permute(1, 0, 2)
    s = torch.einsum("hd,hnd->hn", q, kk) * scale
    size = torch.einsum("hd,hnd->hn", q.abs(), kk.abs()) * abs(scale)
    lse = torch.logsumexp(s, -1)
    p = torch.exp(s - lse[:, None])
    out = torch.einsum("hn,hnd->hd", p, vv)
    mag = torch.einsum("hn,hnd->hd", p, vv.abs())
    return out, lse, mag, size.amax(-1)


def attention_bound(ref, lse, mag, size, n, D, dtype, vmax, cache=None):
    """(bound of out, bound of lse).

    Scores: D exact products summed in f32, off by at most D 2^-23 of the sum of
    their magnitudes (the tensor core may cut instead of rounding: a whole ulp
    per step), then scaled (2^-23).  The exponential: 2 ulp and its argument's
    rounding, 2^-24 of a score's distance to the maximum (at most 2 size).
    Weights enter the second product as two pieces of the 16-bit type: 2^-17
    left over (bf16), or 2^-25 of the largest (f16, a subnormal weight).  With
    a bf16 output over an 8-bit cache they are one f16 piece, rounded to at
    most half a step: eps / 2 = 2^-11 of each weight.  Sums
    of n weights and values in f32: n 2^-23.  Each is relative to
    sum_j p_j |v_j|; the result is divided and rounded once."""
    ds = (D + 4) * 2.0 ** -23 * size
    piece = 2.0 ** -11 if dtype == torch.bfloat16 and cache == torch.float8_e4m3fn else 2.0 ** -17
    rel = torch.as_tensor(2 * ds + 2.0 ** -21 + piece + n * 2.0 ** -23)
    b = rel[:, None] * mag + n * 2.0 ** -25 * vmax / max(1, n) + \
        torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    return half_step(dtype) * (ref.abs() + b) + b, \
        rel - piece + lse.abs() * 2.0 ** -22
