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


def test_block_table_ids_out_of_range_enter_neither_table_nor_stack(rb):
    """A bad id on the stack: the table takes -1 for it and its tokens have no slot.  A bad id in
    a released row: the stack takes -1, and so does the next request.  Each step reports."""
    free = i32([3, 77, 1, 2])
    table = torch.full((2, 3), -9, dtype=torch.int32, device="cuda")
    st = rb.kv_block_table(i32([0, 0]), i32([8, 11]), table, free, i32([4]), block_size=8,
                           max_tokens=19)
    assert table.tolist() == [[2, -9, -9], [1, -1, -9]]
    assert st.slots.tolist() == [*range(16, 24), *range(8, 16), -1, -1, -1]
    assert st.positions.tolist() == [*range(8), *range(11)]
    assert st.lens.tolist() == [8, 11] and st.status.tolist() == [0, 0]
    assert st.free_count.tolist() == [1] and free.tolist() == [3, 77, 1, 2]
    with pytest.raises(rb.RemoraError, match="block id"):
        rb.synchronize_and_check()
    for bad in (-1, 4, -5, 2 ** 31 - 1, -2 ** 31):
        table, free, count = i32([[2, bad], [-9, -9]]), i32([0, 1, -7, -7]), i32([2])
        st = rb.kv_block_table(i32([16, 0]), i32([-1, 0]), table, free, count, block_size=8,
                               max_tokens=4)
        assert free.tolist() == [0, 1, 2, -1] and st.free_count.tolist() == [4]
        assert st.lens.tolist() == [0, 0] and st.status.tolist() == [0, 0]
        with pytest.raises(rb.RemoraError, match="block id"):
            rb.synchronize_and_check()
        st = rb.kv_block_table(st.lens, i32([0, 12]), table, free, st.free_count, block_size=8,
                               max_tokens=12)
        assert table[1].tolist() == [-1, 2] and st.free_count.tolist() == [2]
        assert st.slots.tolist() == [-1] * 8 + [16, 17, 18, 19]
        with pytest.raises(rb.RemoraError, match="block id"):
            rb.synchronize_and_check()
    rb.synchronize_and_check()


def test_attention_over_a_block_that_was_missing(rb):
    """The keys of a block that a step could not give are left out, and reported."""
    D, bs = 64, 8
    kc = torch.randn(4, bs, 1, D, generator=gen(1)).to(torch.bfloat16).cuda()
    vc = torch.randn(4, bs, 1, D, generator=gen(2)).to(torch.bfloat16).cuda()
    q = torch.randn(1, 2, D, generator=gen(3)).to(torch.bfloat16).cuda()
    table = i32([[-9, -9]])
    st = rb.kv_block_table(i32([0]), i32([12]), table, i32([4, 3, -7, -7]), i32([2]),
                           block_size=bs, max_tokens=12)
    assert table.tolist() == [[3, -1]]
    got = rb.paged_attention(q, kc, vc, table, st.lens)
    with pytest.raises(rb.RemoraError, match="block id"):
        rb.synchronize_and_check()
    o, l, mag, size = ref.attention(q[0].cpu(), kc[3].cpu(), vc[3].cpu(), D ** -0.5)
    close(got[0], o, ref.attention_bound(o, l, mag, size, bs, D, torch.bfloat16,
                                         float(vc.abs().max()))[0])


# ------------------------------------------------------------------- rotary
def two_pi(bits):
    """floor(2 pi * 2^bits), by arctan(1/5) and arctan(1/239)."""
    def arctan_inverse(n):
        term = (1 << bits + 32) // n
        total, k, sign = term, 1, -1
        while term:
            term //= n * n
            k += 2
            total += sign * (term // k)
            sign = -sign
        return total >> 32
    return 8 * (4 * arctan_inverse(5) - arctan_inverse(239))


def angle_of(position, freq, turn=two_pi(400)):
    """position * freq modulo 2 pi, exactly and then rounded."""
    f = Fraction(float(freq)) * position * 2 ** 400
    return float(Fraction(f.numerator % (turn * f.denominator), f.denominator * 2 ** 400))


@pytest.mark.parametrize("inverse", [False, True])
def test_rope_frequencies_of_many_turns(rb, inverse):
    """The angle keeps its precision whatever the frequency: here to just below 2^64."""
    below = math.nextafter(2.0 ** 64, 0)
    f = [1.0, 6.28, 2 * math.pi, math.nextafter(2 * math.pi, 7), 7.5, 1e3, 1e4, 31415.9, 1e6, 1e9,
         1e12 + 0.5, 2.0 ** 53 - 1, 1e18, below, 2.0 ** 63, 1e-9]
    f = torch.tensor(f + [-x for x in f], dtype=torch.float64)
    pos = [0, 1, -1, 5, 2 ** 24 + 1, 2 ** 31 - 1, -2 ** 31, 123456789]
    x = torch.randn(len(pos), 2, 64, generator=gen(4))
    got = rb.rope(x.cuda(), i32(pos), f, inverse=inverse)
    a = torch.tensor([[angle_of(p, v) for v in f.tolist()] for p in pos], dtype=torch.float64)
    c, s = a.cos()[:, None], a.sin()[:, None] * (-1 if inverse else 1)
    lo, hi = x[..., :32].double(), x[..., 32:].double()
    want = torch.cat([lo * c - hi * s, lo * s + hi * c], -1)
    # the errors that rope_bound counts, without its reference's own rounded angle
    b = ((lo.abs() + hi.abs()) * 2.0 ** -21).repeat(1, 1, 2)
    close(got, want, ref.half_step(torch.float32) * (want.abs() + b) + b)


# ---------------------------------------------------------------- attention
@pytest.mark.parametrize("below", [14, 20, 27, 30])
def test_attention_small_queries_beside_large_ones(rb, below):
    """bf16 queries over 8-bit keys: one element is 2^below times the others and meets zeros, so
    the others decide.  All of a bf16's bits of theirs count."""
    D, n, bs = 128, 100, 16
    g = gen(below)
    k = torch.randint(-448, 449, (7 * bs, 1, D), generator=g).float().to(torch.float8_e4m3fn)
    k.view(torch.uint8)[..., 5] = 0
    v = torch.randn(7 * bs, 1, D, generator=g).to(torch.float8_e4m3fn)
    q = torch.randn(1, 2, D, generator=g).sign() * (1 + torch.randint(0, 128, (1, 2, D), generator=g) / 128)
    q[..., 5] = 2.0 ** below
    scale = 1.0 / 2000
    lse = torch.empty(1, 2, device="cuda")
    out = rb.paged_attention(q.to(torch.bfloat16).cuda(), k.view(7, bs, 1, D).cuda(),
                             v.view(7, bs, 1, D).cuda(), i32([range(7)]), i32([n]), scale=scale,
                             lse=lse)
    o, l, mag, size = ref.attention(q[0], k[:n].float(), v[:n].float(), scale)
    b, bl = ref.attention_bound(o, l, mag, size, n, D, torch.bfloat16, float(v.float().abs().max()),
                                torch.float8_e4m3fn)
    close(out[0], o, b)
    close(lse[0], l, bl)


@pytest.mark.parametrize("dtype,cache,q,key,scale,k_scale", [
    ("bf16", "e4m3", 1e38, 0.0, 0.125, 1e6),      # a factor past 32 bits, of products of zero
    ("bf16", "e4m3", 1e38, 0.0, -1e7, 1.0),
    ("bf16", "bf16", 1e18, 1e18, 1e-40, 1.0),     # a scale below the normal range
    ("f16", "e4m3", 3e4, 448.0, 1e-30, 1e-12),
    ("bf16", "e4m3", 1e-38, 448.0, 1e-8, 1e-30),  # a factor that is zero in 32 bits
])
def test_attention_factors_out_of_range(rb, dtype, cache, q, key, scale, k_scale):
    """Scores that are ordinary numbers (here equal, so the output is the mean of the values and
    lse = score + log n), though the factor of their products is none."""
    from tests.test_paged_gpu import DT
    D, n = 64, 20
    kc = torch.full((2, 16, 1, D), key).to(DT[cache]).cuda()
    vc = torch.randn(2, 16, 1, D, generator=gen(2)).to(DT[cache]).cuda()
    lse = torch.empty(1, 2, device="cuda")
    x = torch.full((1, 2, D), q).to(DT[dtype])
    out = rb.paged_attention(x.cuda(), kc, vc, i32([[0, 1]]), i32([n]), scale=scale, k_scale=k_scale,
                             lse=lse)
    v = vc.float().cpu().view(32, D)[:n].double()
    score = float(x[0, 0, 0].double() * kc[0, 0, 0, 0].cpu().double()) * D * scale * k_scale
    mean, mag = v.mean(0), v.abs().mean(0)
    # the mean's sums and weights (2^-11 of one f16 piece), then the output's rounding
    b = mag * (2.0 ** -11 + (n + 8) * 2.0 ** -23) + 2.0 ** -24
    assert bool(((out[0].double().cpu() - mean).abs() <= b + ref.half_step(DT[dtype]) *
                 (mean.abs() + b)).all())
    # 1e-40 holds 17 bits: 2^-17 of the score, and the logarithm's sum 2^-20
    want = score + math.log(n)
    assert bool(((lse.cpu().double() - want).abs() <= 2.0 ** -16 * abs(score) + 2.0 ** -20).all())
    rb.synchronize_and_check()


# ---------------------------------------------------------------- gradients
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("inter,inverse", [(False, False), (True, False), (False, True)])
def test_rope_records_its_gradient(rb, dtype, inter, inverse):
    """backward() through rope: against the formula's transpose in 64 bits, of strided inputs and
    of gradients of several layouts, added to what else the leaf is used for."""
    B, S, H, D, rot = 2, 7, 3, 40, 24
    g = gen(5)
    pos = torch.randint(0, 4000, (2, B, S), generator=g, dtype=torch.int32)
    f, ax = freqs(rot), (torch.arange(rot // 2) % 2).to(torch.int32)
    x = torch.randn(B, H, S, D, generator=g).to(dtype)
    leaf = x.cuda().requires_grad_(True)
    y = rb.rope(leaf.transpose(1, 2), pos.cuda(), f, axis_of=ax, interleaved=inter, inverse=inverse)
    with torch.no_grad():
        plain = rb.rope(leaf.transpose(1, 2), pos.cuda(), f, axis_of=ax, interleaved=inter,
                        inverse=inverse)
    assert plain.grad_fn is None and torch.equal(plain, y) and y.stride() == plain.stride()
    dy = torch.randn(B, S, H, D, generator=g).to(dtype)
    for grad in (dy, dy.transpose(0, 2).contiguous().transpose(0, 2), dy[:, :, :, :1].expand_as(dy)):
        got, = torch.autograd.grad(y, leaf, grad.cuda(), retain_graph=True)
        want = ref.rope(grad, pos, f, ax, inter, not inverse)
        bound = ref.rope_bound(grad, want, f, pos, dtype, inter)
        close(got.transpose(1, 2), want, bound)
    (y.float().sum() + leaf.float().sum()).backward()
    want = ref.rope(torch.ones_like(dy), pos, f, ax, inter, not inverse)
    bound = ref.rope_bound(torch.ones_like(dy), want, f, pos, dtype, inter)
    # the sum's two gradients are added in dtype: a rounding more
    close(leaf.grad.transpose(1, 2), want + 1, bound + ref.half_step(dtype) * ((want + 1).abs() + bound))


def test_rope_gradient_against_differences_and_its_own(rb):
    """Differences of a loss (linear in x but for its square, so a step of 1/8 is exact enough),
    and the gradient of the gradient."""
    g = gen(6)
    x = torch.randn(4, 2, 16, generator=g)
    pos, f = i32([0, 3, 50, 900]), freqs(16)
    w = torch.randn(4, 2, 16, generator=g).cuda()

    def loss(t):
        y = rb.rope(t, pos, f)
        return (w * y + y * y * 0.25).double().sum()

    leaf = x.cuda().requires_grad_(True)
    grad, = torch.autograd.grad(loss(leaf), leaf, create_graph=True)
    h = 0.125
    for at in ((0, 0, 0), (1, 1, 3), (2, 0, 9), (3, 1, 15)):
        e = torch.zeros_like(x)
        e[at] = h
        with torch.no_grad():
            diff = (loss((x + e).cuda()) - loss((x - e).cuda())) / (2 * h)
        # 128 elements of at most 16, each rounded a few times in 32 bits, over the step
        assert abs(float(diff - grad[at].detach())) <= 128 * 16 * 2.0 ** -21 / h
    # the loss is w y + y^2 / 4 and |y| = |x|: grad = rope back of w, + x / 2
    second, = torch.autograd.grad(grad.sum(), leaf)
    assert float((second - 0.5).abs().max()) <= 2.0 ** -20


def test_rope_gradient_keeps_to_its_positions(rb):
    """Positions changed between the two passes are an error, not another angle; a call with out
    records nothing; nor do the serving calls."""
    x, pos, f = torch.ones(3, 1, 8, device="cuda", requires_grad=True), i32([1, 2, 3]), freqs(8)
    y = rb.rope(x, pos, f)
    pos.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    y = rb.rope(x, pos, f, out=torch.empty(3, 1, 8, device="cuda"))
    assert y.grad_fn is None
    kc = torch.zeros(1, 4, 1, 8, device="cuda", dtype=torch.bfloat16)
    q = torch.ones(3, 1, 8, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    assert rb.rope_kv_append(q, q, q, pos, i32([0, 1, 2]), f, kc, kc.clone()).grad_fn is None


def test_rope_gradient_in_a_graph(rb):
    """Forward and backward captured together: each replay takes the inputs of its time."""
    g = gen(7)
    f, pos = freqs(64), torch.arange(12, dtype=torch.int32, device="cuda")
    x, dy = (torch.randn(12, 2, 64, generator=g).cuda() for _ in range(2))
    leaf = x.clone().requires_grad_(True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(rb.rope(leaf, pos, f), leaf, dy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = rb.rope(leaf, pos, f)
        grad, = torch.autograd.grad(y, leaf, dy)
    for _ in range(2):
        with torch.no_grad():
            leaf.copy_(torch.randn(12, 2, 64, generator=g))
        dy.copy_(torch.randn(12, 2, 64, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, rb.rope(leaf.detach(), pos, f))
        assert torch.equal(grad, rb.rope(dy, pos, f, inverse=True))


# ------------------------------------------------- attention whose values cancel
@pytest.mark.parametrize("dtype,cache", [("bf16", "e4m3"), ("f16", "e4m3"), ("bf16", "bf16")])
@pytest.mark.parametrize("Hq,D", [(4, 64), (8, 128), (12, 128), (4, 256)])
def test_attention_values_that_cancel(rb, dtype, cache, Hq, D):
    """Pairs of keys of nearly the same score hold opposite values, so that the output is small
    beside what it is summed from, and the weights' own rounding shows: 2^-17 whatever the types."""
    from tests.test_paged_gpu import DT
    n, bs = 32, 16
    g = gen(D + Hq)
    k = torch.randn(n // 2, 1, D, generator=g).repeat_interleave(2, 0)
    k[1::2, 0, :2] += 0.25
    v = torch.randn(n // 2, 1, D, generator=g).sign() * 240
    v = torch.stack([v, -v], 1).flatten(0, 1)
    q = torch.randn(1, Hq, D, generator=g).to(DT[dtype])
    kc, vc = k.to(DT[cache]), v.to(DT[cache])
    scale = 2.0 ** -5 / D  # small scores: their own rounding does not hide the weights'
    out = rb.paged_attention(q.cuda(), kc.view(2, bs, 1, D).cuda(), vc.view(2, bs, 1, D).cuda(),
                             i32([[0, 1]]), i32([n]), scale=scale)
    o, l, mag, size = ref.attention(q[0], kc.float(), vc.float(), scale)
    assert float(o.abs().max()) < 2.0 ** -6 * float(mag.min())
    close(out[0], o, ref.attention_bound(o, l, mag, size, n, D, DT[dtype], 240.0)[0])


def test_rope_frequencies_near_nothing(rb):
    """Frequencies whose turns vanish beside one, of either sign: no angle at all, or next to."""
    f = torch.tensor([0.0, -0.0, 1e-30, -1e-30, 5e-324, -5e-324, -1e-19, -2.0 ** -60] * 4,
                     dtype=torch.float64)
    pos = [0, 1, -7, 2 ** 31 - 1, -2 ** 31]
    x = torch.randn(len(pos), 2, 64, generator=gen(8))
    for inverse in (False, True):
        # 2^31 times 2^-60, and one unit of the phase, 2^-32 of a turn; then the output's rounding
        b = 2.0 ** -28 * (x[..., :32].abs() + x[..., 32:].abs()).double().repeat(1, 1, 2)
        close(rb.rope(x.cuda(), i32(pos), f, inverse=inverse), x.double(),
              ref.half_step(torch.float32) * (x.double().abs() + b) + b)
