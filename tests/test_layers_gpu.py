"""The layer operators (head norm with rotation, low-rank adapters,
distillation loss) against plain implementations in 64 bits, at the sizes,
strides and masks where they can go wrong, and their gradients against the
formulas' and against differences.

Tolerances are elementwise: one rounding to the output's type (unit u: 2^-8
bf16, 2^-11 fp16, 2^-24 fp32, half the smallest subnormal in fp16) plus the
fp32 arithmetic's error, bounded by a power of two times the sum of the
magnitudes that enter the element.
"""
import math

import pytest
import torch

from sdc_b200.layers import (AdapterBatch, distillation_loss, distillation_loss_and_grad, head_norm_rotary,
                             low_rank_adapters, low_rank_adapters_, rotary_table)

pytestmark = pytest.mark.gpu
DEV = "cuda"
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
FLOOR = {torch.bfloat16: 1e-38, torch.float16: 2.0 ** -25, torch.float32: 1e-38}
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def rng(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def normal(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, device=DEV, generator=g) * scale).to(dtype)


def close(got, exact, magnitude, arithmetic):
    """One rounding of ``exact`` and ``arithmetic`` times ``magnitude``."""
    assert got.shape == exact.shape
    tolerance = UNIT[got.dtype] * exact.abs() * (1 + 2.0 ** -10) + FLOOR[got.dtype] + arithmetic * magnitude
    off = (got.double() - exact).abs()
    bad = ~(off <= tolerance)
    assert not bad.any(), (off[bad].max().item(), tolerance[bad].min().item(), int(bad.sum()), bad.nonzero()[:3])


# ------------------------------------------------- head norm and rotation ----

def rotate64(x, cos, sin, rotary, interleaved):
    x, y = x.clone(), x.clone()
    first = slice(0, rotary, 2) if interleaved else slice(0, rotary // 2)
    second = slice(1, rotary, 2) if interleaved else slice(rotary // 2, rotary)
    y[..., first] = x[..., first] * cos - x[..., second] * sin
    y[..., second] = x[..., second] * cos + x[..., first] * sin
    return y


def rotary64(x, table, positions, weight, eps, interleaved):
    """(output, magnitude of what enters each element) of [B, S, H, D] heads."""
    rotary = table.shape[1]
    angles = table.double()[positions][:, :, None]
    cos, sin = angles[..., :rotary // 2], angles[..., rotary // 2:]
    x = x.double()
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * weight.double()
    return (rotate64(x, cos, sin, rotary, interleaved),
            rotate64(x.abs(), cos.abs(), -sin.abs(), rotary, interleaved).abs() + x.abs())


ROTARY_CASES = [
    # batch, sequence, heads, kv heads, dim, rotary, interleaved, norm, fp32 weights
    (1, 1, 28, 4, 128, 128, False, True, False),
    (2, 17, 14, 2, 64, 64, False, True, True),
    (3, 5, 7, 1, 80, 40, True, True, False),
    (1, 33, 3, 3, 96, 32, False, True, False),
    (1, 9, 5, 2, 256, 256, True, True, False),
    (2, 3, 2, 1, 512, 512, False, True, True),
    (1, 7, 3, 1, 6, 4, False, True, False),     # no vector form
    (1, 11, 2, 1, 34, 10, True, True, False),
    (2, 4, 1, 1, 2, 2, False, True, False),
    (1, 1031, 4, 1, 128, 64, False, False, False),
    (1, 3, 9, 5, 48, 24, False, False, False),  # whole heads, rotary part not in runs of 16
]


def _rotary_inputs(case, dtype, seed=0):
    batch, sequence, heads, kv, dim, rotary, interleaved, norm, f32 = case
    g = rng(seed)
    qkv = normal(g, batch, sequence, (heads + 2 * kv) * dim, dtype=dtype, scale=1.5)
    q = qkv[..., :heads * dim].unflatten(-1, (heads, dim))
    k = qkv[..., heads * dim:(heads + kv) * dim].unflatten(-1, (kv, dim))
    table = rotary_table(3000, rotary, 1e4)
    positions = torch.randint(0, 3000, (batch, sequence), device=DEV, generator=g)
    weights = (None, None)
    if norm:
        weights = tuple((1 + normal(g, dim, scale=0.3)).to(torch.float32 if f32 else dtype) for _ in range(2))
    return q, k, table, positions, weights, interleaved


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", ROTARY_CASES)
def test_head_norm_rotary_forward_and_backward(case, dtype):
    q, k, table, positions, weights, interleaved = _rotary_inputs(case, dtype)
    g = rng(1)
    leaves = [t.detach().requires_grad_() for t in (q, k, *weights) if t is not None]
    q_weight, k_weight = leaves[2:] or (None, None)
    out = head_norm_rotary(leaves[0], leaves[1], table, positions, q_weight, k_weight, 1e-6, interleaved)
    assert all(o.is_contiguous() for o in out)
    # Without autograd the same bits.
    for o, again in zip(out, head_norm_rotary(q, k, table, positions, *weights, 1e-6, interleaved)):
        assert torch.equal(o, again)
    upstream = [normal(g, *o.shape, dtype=dtype) for o in out]
    grads = torch.autograd.grad(out, leaves, upstream)
    exact = [t.detach().double().requires_grad_() for t in leaves]
    for i in range(2):
        weight = exact[2 + i] if weights[0] is not None else None
        reference, magnitude = rotary64(exact[i], table, positions, weight, 1e-6, interleaved)
        close(out[i], reference.detach(), magnitude.detach(), 2.0 ** -19)
        targets = [exact[i]] + ([weight] if weight is not None else [])
        expected = torch.autograd.grad(reference, targets, upstream[i].double())
        # r (|g w| + |u| mean |g w u|) and sum |g u|, with |g| the turned upstream's magnitude.
        angles = table.double()[positions][:, :, None]
        half = table.shape[1] // 2
        turned = rotate64(upstream[i].double().abs(), angles[..., :half].abs(), -angles[..., half:].abs(),
                          table.shape[1], interleaved).abs() + upstream[i].double().abs()
        if weight is None:
            close(grads[i], expected[0], turned, 2.0 ** -19)
            continue
        x = exact[i].detach()
        r = torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)
        gw, u = turned * weight.detach().abs(), (x * r).abs()
        close(grads[i], expected[0], r * (gw + u * (gw * u).mean(-1, keepdim=True)), 2.0 ** -18)
        close(grads[2 + i], expected[1], (turned * u).sum((0, 1, 2)), 2.0 ** -18)


def test_head_norm_rotary_takes_any_strides_and_alignment():
    table = rotary_table(64, 64)
    g = rng(3)
    positions = torch.arange(5, device=DEV, dtype=torch.int32)
    for dtype in TYPES:
        # [batch, heads, sequence, dim] turned to [batch, sequence, heads, dim]; positions broadcast over the batch.
        q = normal(g, 2, 6, 5, 64, dtype=dtype).transpose(1, 2)
        k = normal(g, 2, 2, 5, 64, dtype=dtype).transpose(1, 2)
        want = head_norm_rotary(q.contiguous(), k.contiguous(), table, positions)
        for a, b in zip(head_norm_rotary(q, k, table, positions), want):
            assert torch.equal(a, b)
        # A view that starts off a 16-byte boundary, and odd row strides.
        wide = torch.zeros(2, 5, 6 * 64 + 3, device=DEV, dtype=dtype)
        odd = wide[..., 1:6 * 64 + 1].unflatten(-1, (6, 64))
        odd.copy_(q)
        for a, b in zip(head_norm_rotary(odd, k, table, positions), want):
            assert torch.equal(a, b)
        # Heads whose elements are apart.
        apart = q.transpose(2, 3).contiguous().transpose(2, 3)
        for a, b in zip(head_norm_rotary(apart, k, table, positions), want):
            assert torch.equal(a, b)
        # A broadcast gradient (zero strides), and an output that is not used.
        leaf = q.contiguous().requires_grad_()
        out = head_norm_rotary(leaf, k, table, positions)
        (broadcast,) = torch.autograd.grad(out[0].sum(), leaf, retain_graph=True)
        (full,) = torch.autograd.grad(out[0], leaf, torch.ones_like(out[0]))
        assert torch.equal(broadcast, full)


def test_head_norm_rotary_positions_outside_the_table_are_nan():
    table = rotary_table(8, 32)
    q, k = normal(rng(4), 3, 2, 64, dtype=torch.bfloat16), normal(rng(5), 3, 1, 64, dtype=torch.bfloat16)
    out, _ = head_norm_rotary(q, k, table, torch.tensor([7, 8, -1], device=DEV))
    assert out[0].isfinite().all()
    assert out[1:, :, :32].isnan().all() and torch.equal(out[1:, :, 32:], q[1:, :, 32:])


def test_head_norm_rotary_without_tokens():
    table = rotary_table(8, 64)
    q = torch.empty(0, 4, 64, device=DEV, requires_grad=True)
    k = torch.empty(0, 2, 64, device=DEV)
    w = torch.ones(64, device=DEV, requires_grad=True)
    out = head_norm_rotary(q, k, table, torch.empty(0, device=DEV, dtype=torch.int64), w, w.detach())
    assert out[0].shape == (0, 4, 64) and out[1].shape == (0, 2, 64)
    dq, dw = torch.autograd.grad(out[0].sum(), (q, w))
    assert dq.shape == q.shape and torch.equal(dw, torch.zeros_like(w))


def test_head_norm_rotary_zero_heads_and_not_finite_values_stay_in_their_head():
    table = rotary_table(8, 64)
    q = normal(rng(6), 2, 3, 64)
    q[0, 1] = 0
    q[1, 2, 5] = math.inf
    w = torch.ones(64, device=DEV)
    out, _ = head_norm_rotary(q, q, table, torch.arange(2, device=DEV), w, w)
    assert torch.equal(out[0, 1], torch.zeros_like(out[0, 1]))
    rest = torch.ones(2, 3, dtype=torch.bool, device=DEV)
    rest[1, 2] = False
    assert out[rest].isfinite().all() and out[1, 2].isnan().any()


def test_head_norm_rotary_gradient_against_differences():
    q, k, table, positions, weights, _ = _rotary_inputs(ROTARY_CASES[1], torch.float32)
    inputs = [t.detach().contiguous().requires_grad_() for t in (q, k, *weights)]
    out = head_norm_rotary(inputs[0], inputs[1], table, positions, inputs[2], inputs[3])
    g = rng(8)
    upstream = [normal(g, *o.shape) for o in out]
    grads = torch.autograd.grad(out, inputs, upstream)
    h = 2.0 ** -7

    def value(step, i, direction):
        moved = [t.detach() + (step * direction if j == i else 0) for j, t in enumerate(inputs)]
        return sum((o.double() * u.double()).sum()
                   for o, u in zip(head_norm_rotary(moved[0], moved[1], table, positions, moved[2], moved[3]), upstream))

    for i, grad in enumerate(grads):
        direction = torch.sign(grad)  # the slope is the sum of |grad|: nothing cancels
        slope = (value(h, i, direction) - value(-h, i, direction)) / (2 * h)
        # Third-order term: h^2 / 6 times third derivatives of order 1 per element; rounding 2^-24 / h.
        assert abs(slope - grad.double().abs().sum()) <= 2.0 ** -8 * grad.double().abs().sum()


# ------------------------------------------------------ low-rank adapters ----

ADAPTER_CASES = [
    # lengths, adapters, count, rank, in, out
    ([1], [0], 1, 16, 896, 896),
    ([1, 1, 1, 1, 1], [2, 0, -1, 2, 1], 4, 8, 256, 384),
    ([3, 0, 70, 1, 40, 0], [1, 0, 0, -1, 1, 2], 3, 24, 320, 264),
    ([200], [0], 1, 64, 128, 72),
    ([65, 64, 63], [0, 1, 0], 2, 5, 104, 1000),
    ([33, 2], [1, 1], 2, 1, 37, 53),              # widths without a vector form
    ([17, 48], [0, 1], 2, 100, 200, 136),         # more than one block of ranks
    ([130], [0], 1, 256, 264, 136),
    ([12], [-1], 2, 16, 64, 64),                  # nothing adapted
    ([1000, 500], [0, 1], 2, 32, 896, 520),
    # Tiles of 128 rows: ranks of each kind, odd widths, unused adapters, tokens without one between.
    ([1000, 37, 700, 0], [0, -1, 1, 1], 3, 16, 320, 264),
    ([2000], [0], 1, 64, 136, 72),
    ([901, 800, 13], [1, 0, 1], 2, 5, 104, 1000),
    ([1700], [0], 1, 24, 37, 53),
    ([1024, 640], [0, 1], 2, 100, 200, 136),
    ([1600], [0], 1, 256, 264, 136),
    ([2] * 40, list(range(40)), 40, 16, 1032, 904),
]


def _adapter_inputs(case, dtype, seed=0):
    lengths, adapters, count, rank, k, n = case
    g = rng(seed)
    tokens = sum(lengths)
    x, base = normal(g, tokens, k, dtype=dtype), normal(g, tokens, n, dtype=dtype)
    a, b = normal(g, count, rank, k, dtype=dtype, scale=k ** -0.5), normal(g, count, n, rank, dtype=dtype, scale=rank ** -0.5)
    scale = torch.rand(count, device=DEV, generator=g) + 0.5
    return x, base, a, b, scale, AdapterBatch(lengths, adapters, count)


def adapters64(lengths, adapters, x, base, a, b, scale, grad=None):
    """Outputs and gradients, each with the magnitude of what enters its elements."""
    x, base, a, b, scale = (t.double() for t in (x, base, a, b, scale))
    out, out_size = base.clone(), base.abs()
    parts = None
    if grad is not None:
        grad = grad.double()
        parts = [torch.zeros_like(t) for t in (x, x, a, a, b, b)]
    start = 0
    for length, g in zip(lengths, adapters):
        rows = slice(start, start + length)
        start += length
        if g < 0:
            continue
        low, low_size = x[rows] @ a[g].T * scale[g], x[rows].abs() @ a[g].abs().T * scale[g]
        out[rows] += low @ b[g].T
        out_size[rows] += low_size @ b[g].abs().T
        if grad is None:
            continue
        down, down_size = grad[rows] @ b[g] * scale[g], grad[rows].abs() @ b[g].abs() * scale[g]
        parts[0][rows] += down @ a[g]
        parts[1][rows] += down_size @ a[g].abs()
        parts[2][g] += down.T @ x[rows]
        parts[3][g] += down_size.T @ x[rows].abs()
        parts[4][g] += grad[rows].T @ low
        parts[5][g] += grad[rows].abs().T @ low_size
    return out, out_size, parts


# The low-rank rows' two terms keep 2^-16 (bf16); fp32 sums of n products err by at most n 2^-23 of their magnitude.
def adapter_arithmetic(*lengths):
    return 2.0 ** -15 + sum(lengths) * 2.0 ** -23


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", ADAPTER_CASES)
def test_low_rank_adapters_forward_and_backward(case, dtype):
    lengths, adapters, count, rank, k, n = case
    x, base, a, b, scale, batch = _adapter_inputs(case, dtype)
    grad = normal(rng(1), *base.shape, dtype=dtype)
    leaves = [t.detach().requires_grad_() for t in (base, x, a, b)]
    out = low_rank_adapters(*leaves[:2], *leaves[2:], batch, scale)
    exact, size, parts = adapters64(lengths, adapters, x, base, a, b, scale, grad)
    close(out.detach(), exact, size, adapter_arithmetic(k, rank))
    in_place = base.clone()
    assert low_rank_adapters_(in_place, x, a, b, batch, scale) is in_place
    assert torch.equal(in_place, out)
    d_base, dx, da, db = torch.autograd.grad(out, leaves, grad)
    assert torch.equal(d_base, grad)
    close(dx, parts[0], parts[1], adapter_arithmetic(n, rank))
    close(da, parts[2], parts[3], adapter_arithmetic(n, len(grad)))
    close(db, parts[4], parts[5], adapter_arithmetic(k, len(grad)))
    # Nothing depends on the order in which blocks run.
    again = low_rank_adapters(*leaves[:2], *leaves[2:], batch, scale)
    assert torch.equal(out, again)
    for first, second in zip((dx, da, db), torch.autograd.grad(again, leaves[1:], grad)):
        assert torch.equal(first, second)


# Token sums long enough for clusters of 9 to 16 blocks: few column blocks, both forms of a row, blocks of ranks, empty adapters.
@pytest.mark.parametrize("case", [([2100], [0], 1, 16, 37, 53), ([5000, 3], [0, 2], 3, 64, 136, 520),
                                  ([2500, 0, 2400], [0, 2, 1], 3, 100, 200, 136), ([4096], [0], 1, 32, 896, 2056),
                                  ([3001], [0], 1, 5, 1032, 264)])
def test_low_rank_adapters_sum_long_batches(case):
    test_low_rank_adapters_forward_and_backward(case, torch.bfloat16)


@pytest.mark.parametrize("requests", [1, 5, 60])
def test_low_rank_adapters_tiles_do_not_change_a_token(requests):
    """A token's output has the same exact value whatever shares its batch."""
    dtype = torch.bfloat16
    case = ([7] * requests, [i % 3 for i in range(requests)], 3, 16, 512, 640)
    x, base, a, b, scale, batch = _adapter_inputs(case, dtype)
    out = low_rank_adapters(base, x, a, b, batch, scale)
    exact, size, _ = adapters64(*case[:2], x, base, a, b, scale)
    close(out, exact, size, adapter_arithmetic(512, 16))


def test_low_rank_adapters_take_strided_rows_and_no_scale():
    case = ([40, 9], [1, 0], 2, 16, 128, 192)
    for dtype in (torch.bfloat16, torch.float16):
        x, base, a, b, _, batch = _adapter_inputs(case, dtype)
        want = low_rank_adapters(base, x, a, b, batch)
        exact, size, _ = adapters64(*case[:2], x, base, a, b, torch.ones(2, device=DEV))
        close(want, exact, size, adapter_arithmetic(128, 16))
        for pad, shift in ((8, 0), (8, 8), (3, 1)):
            wide_x = torch.zeros(49, 128 + pad + shift, device=DEV, dtype=dtype)
            wide_base = torch.zeros(49, 192 + pad + shift, device=DEV, dtype=dtype)
            vx, vb = wide_x[:, shift:shift + 128], wide_base[:, shift:shift + 192]
            vx.copy_(x), vb.copy_(base)
            assert torch.equal(low_rank_adapters(vb, vx, a, b, batch), want)
            low_rank_adapters_(vb, vx, a, b, batch)
            assert torch.equal(vb, want)
            rest = torch.ones(192 + pad + shift, dtype=torch.bool, device=DEV)
            rest[shift:shift + 192] = False
            assert not wide_base[:, rest].any()


def test_low_rank_adapters_take_column_major_operands():
    """The FP8 projections' outputs are column-major, and so is what is computed from them."""
    case = ([40, 9], [1, 0], 2, 16, 128, 192)
    x, base, a, b, scale, batch = _adapter_inputs(case, torch.bfloat16)
    grad = normal(rng(2), 49, 192, dtype=torch.bfloat16)

    def results(x, base, grad):
        leaves = [t.detach().requires_grad_() for t in (x, a, b)]
        out = low_rank_adapters(base, *leaves, batch, scale)
        return (out, *torch.autograd.grad(out, leaves, grad))

    columns = [t.t().contiguous().t() for t in (x, base, grad)]
    for got, want in zip(results(*columns), results(x, base, grad)):
        assert torch.equal(got, want)
    in_place = columns[1].clone(memory_format=torch.preserve_format)
    assert in_place.stride() == columns[1].stride()
    low_rank_adapters_(in_place, columns[0], a, b, batch, scale)
    assert torch.equal(in_place, low_rank_adapters(base, x, a, b, batch, scale))


def test_low_rank_adapters_keep_foreign_values_out():
    """Not-finite rows reach neither other tokens nor adapters without them; infinite sums stay infinite."""
    case = ([20, 5, 20], [0, -1, 1], 3, 16, 64, 128)
    x, base, a, b, scale, batch = _adapter_inputs(case, torch.bfloat16)
    x[22], base[23] = math.nan, math.inf
    x[3] = math.nan
    a[2], b[2] = math.nan, math.nan
    leaves = [t.detach().requires_grad_() for t in (x, a, b)]
    out = low_rank_adapters(base, *leaves, batch, scale)
    fine = torch.ones(45, dtype=torch.bool, device=DEV)
    fine[[3, 23]] = False
    assert out[fine].isfinite().all() and out[3].isnan().all() and out[23].isinf().all()
    grad = torch.ones_like(out)
    grad[21] = math.nan
    dx, da, db = torch.autograd.grad(out, leaves, grad)
    assert dx.isfinite().all() and not dx[20:25].any()
    assert not da[2].any() and not db[2].any()
    assert da[1].isfinite().all() and db[1].isfinite().all()
    assert da[0].isnan().any() and db[0].isnan().any()
    high = torch.full((1, 64), 3e4, device=DEV, dtype=torch.float16)
    ones = torch.ones(1, 1, 64, device=DEV, dtype=torch.float16)
    batch = AdapterBatch([1], [0], 1)
    assert (low_rank_adapters(high, high, ones, ones.view(1, 64, 1), batch) == math.inf).all()


def test_low_rank_adapters_without_tokens():
    batch = AdapterBatch([], [], 2)
    x = torch.empty(0, 64, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    a = torch.ones(2, 8, 64, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    b = torch.ones(2, 48, 8, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    out = low_rank_adapters(torch.empty(0, 48, device=DEV, dtype=torch.bfloat16), x, a, b, batch)
    assert out.shape == (0, 48)
    dx, da, db = torch.autograd.grad(out.sum(), (x, a, b))
    assert dx.shape == (0, 64) and not da.any() and not db.any()


def test_low_rank_adapters_gradient_against_differences():
    """The output is linear in x, a and b each: central differences are exact up to rounding."""
    case = ([40, 9], [1, 0], 2, 8, 128, 64)
    x, base, a, b, scale, batch = _adapter_inputs(case, torch.float16)
    base.zero_()
    leaves = [t.detach().requires_grad_() for t in (x, a, b)]
    out = low_rank_adapters(base, *leaves, batch, scale)
    upstream = normal(rng(5), *out.shape, dtype=torch.float16)
    grads = torch.autograd.grad(out, leaves, upstream)
    for i, grad in enumerate(grads):
        step = 2.0 ** -4 * torch.sign(grad)
        values = []
        for sign in (1, -1):
            moved = [t.detach() + (sign * step if j == i else 0) for j, t in enumerate(leaves)]
            values.append((low_rank_adapters(base, *moved, batch, scale).double() * upstream.double()).sum())
        slope = (values[0] - values[1]) / 2 ** -3
        total = grad.double().abs().sum()
        # Each of the 49 x 64 outputs and moved inputs is rounded at 2^-11; the errors' signs are unrelated.
        assert abs(slope - total) <= 2.0 ** -6 * total


# ----------------------------------------------------------- distillation ----

def distill64(logits, indices, teacher, temperature):
    """Per row: loss, its magnitude, gradient, q, p scattered over the vocabulary."""
    s, t = logits.double() / temperature, teacher.double() / temperature
    kept = (indices >= 0) & (t != -math.inf)
    some = kept.any(1)
    log_q = torch.where(some[:, None], torch.log_softmax(torch.where(some[:, None], s, 0.0), 1), 0.0)
    log_p = torch.log_softmax(torch.where(some[:, None], torch.where(kept, t, -math.inf), 0.0), 1)
    p = torch.where(kept, log_p.exp(), 0.0)
    at = indices.clamp_min(0)
    chosen = log_q.gather(1, at)
    loss = torch.where(p > 0, p * (log_p - chosen), 0.0).sum(1) * temperature ** 2
    size = torch.where(p > 0, p * (log_p.abs() + chosen.abs() + 1), 0.0).sum(1) * temperature ** 2
    spread = torch.zeros_like(s).scatter_add_(1, at, p)
    q = torch.where(some[:, None], log_q.exp(), 0.0)
    return loss, size, temperature * (q - spread), q, spread


def _distill_inputs(rows, vocab, top, dtype, seed=0, repeat=False):
    g = rng(seed)
    logits = normal(g, rows, vocab, dtype=dtype, scale=3.0)
    if repeat:
        indices = torch.randint(0, vocab, (rows, top), device=DEV, generator=g)
    else:
        indices = torch.rand(rows, vocab, device=DEV, generator=g).topk(top, 1).indices
    teacher = normal(g, rows, top, scale=3.0)
    return logits, indices, teacher


DISTILL_CASES = [
    # rows, vocabulary, top, temperature, repeated indices
    (1, 1, 1, 1.0, False), (3, 3, 2, 1.0, False), (5, 7, 7, 0.5, False), (4, 9, 4, 2.0, True),
    (2, 1000, 33, 1.0, False), (7, 4099, 64, 3.0, False), (3, 50021, 100, 1.5, False), (2, 151936, 64, 2.0, False),
    (300, 513, 20, 1.0, False), (5, 3001, 1024, 1.0, True), (1, 200003, 256, 1.0, True),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", DISTILL_CASES)
def test_distillation_loss_and_gradient(case, dtype):
    rows, vocab, top, temperature, repeat = case
    logits, indices, teacher = _distill_inputs(rows, vocab, top, dtype, repeat=repeat)
    drop = torch.rand(rows, top, device=DEV, generator=rng(2)) < 0.2
    indices[drop] = -1
    if rows > 2:
        indices[1] = -1
        teacher[2] = -math.inf
    loss64, size, grad64, q, p = distill64(logits, indices, teacher, temperature)
    # Exponents of up to 40 in units of 2^-24, sums in fp32: 2^-17 of a probability, 2^-17 of a logarithm's terms.
    upstream = normal(rng(3), rows)

    def check_grad(got, row):
        row = row.double()[:, None]
        close(got, grad64 * row, temperature * row.abs() * (q + p), 2.0 ** -17)

    loss, grad = distillation_loss_and_grad(logits, indices, teacher, temperature, upstream)
    close(loss, loss64, size, 2.0 ** -17)
    check_grad(grad, upstream)
    # 32-bit indices, the mean through autograd, and the plain losses.
    leaf = logits.detach().requires_grad_()
    losses = distillation_loss(leaf, indices.int(), teacher, temperature, "none")
    close(losses.detach(), loss64, size, 2.0 ** -17)
    (got,) = torch.autograd.grad(losses, leaf, upstream)
    check_grad(got, upstream)
    valid = max(1, int(((indices >= 0) & (teacher > -math.inf)).any(1).sum()))
    mean = distillation_loss(leaf, indices, teacher, temperature)
    close(mean.detach(), loss64.sum() / valid, size.sum() / valid, 2.0 ** -16)
    (got,) = torch.autograd.grad(mean * 3, leaf)
    check_grad(got, torch.full((rows,), 3 / valid, device=DEV))
    total = distillation_loss(logits, indices, teacher, temperature, "sum")
    close(total, loss64.sum(), size.sum(), 2.0 ** -16)
    # In place, with one upstream value, and again: the same bits.
    one = torch.full((), 0.5, device=DEV)
    fresh = distillation_loss_and_grad(logits, indices, teacher, temperature, one)
    check_grad(fresh[1], one.expand(rows))
    replaced = logits.clone()
    loss, grad = distillation_loss_and_grad(replaced, indices, teacher, temperature, one, in_place=True)
    assert grad.data_ptr() == replaced.data_ptr() and torch.equal(grad, fresh[1]) and torch.equal(loss, fresh[0])


@pytest.mark.parametrize("dtype", TYPES)
def test_distillation_of_a_row_beyond_a_clusters_shared_memory(dtype):
    vocab = 1_000_003 if dtype != torch.float32 else 500_009
    logits, indices, teacher = _distill_inputs(2, vocab, 50, dtype, repeat=True)
    indices[0, 3] = vocab - 1
    loss64, size, grad64, q, p = distill64(logits, indices, teacher, 1.0)
    for in_place in (False, True):
        loss, grad = distillation_loss_and_grad(logits, indices, teacher, in_place=in_place)
        close(loss, loss64, size, 2.0 ** -17)
        close(grad, grad64, q + p, 2.0 ** -17)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shift", [0, 1, 5, 8])
def test_distillation_takes_strided_rows(dtype, shift):
    logits, indices, teacher = _distill_inputs(6, 2051, 16, dtype)
    wide = torch.full((6, 2051 + shift + 3), 1e4, device=DEV, dtype=dtype)
    view = wide[:, shift:shift + 2051]
    view.copy_(logits)
    want = distillation_loss_and_grad(logits, indices, teacher)
    got = distillation_loss_and_grad(view, indices, teacher)
    # The words a thread takes, hence the order of a row's sum, go by its alignment.
    torch.testing.assert_close(got[0], want[0], rtol=2.0 ** -17, atol=2.0 ** -17)
    _, _, grad64, q, p = distill64(logits, indices, teacher, 1.0)
    close(got[1], grad64, q + p, 2.0 ** -17)
    leaf = view.detach().requires_grad_()
    (grad,) = torch.autograd.grad(distillation_loss(leaf, indices, teacher, reduction="sum"), leaf)
    close(grad, grad64, q + p, 2.0 ** -17)
    distillation_loss_and_grad(view, indices, teacher, in_place=True)
    close(view, grad64, q + p, 2.0 ** -17)
    rest = torch.ones(2051 + shift + 3, dtype=torch.bool, device=DEV)
    rest[shift:shift + 2051] = False
    assert (wide[:, rest] == torch.tensor(1e4).to(dtype)).all()


def test_distillation_masks_and_values_that_are_not_finite():
    vocab, top = 3000, 4
    logits, indices, teacher = _distill_inputs(9, vocab, top, torch.float32)
    indices[0] = -1                      # nothing to learn, and nothing of the row is looked at
    logits[0] = math.nan
    teacher[1] = -math.inf               # neither here
    logits[1, 7] = math.inf
    teacher[2, 1:] = -math.inf           # one entry left
    keep = torch.zeros(vocab, dtype=torch.bool, device=DEV)
    keep[indices[3]] = True
    logits[3, ~keep] = -math.inf         # all of the vocabulary that the list does not name is masked
    logits[4, indices[4, 0]] = torch.finfo(torch.float32).min  # the lowest value as a mask
    logits[5, indices[5, 2]] = -math.inf  # the teacher's token is masked: the loss is infinite
    logits[6] = -math.inf                # all masked
    logits[7, 11] = math.nan
    indices[8, 1] = vocab                # beyond the vocabulary
    loss, grad = distillation_loss_and_grad(logits, indices, teacher)
    assert loss[0] == 0 and loss[1] == 0 and not grad[:2].any()
    loss64, size, grad64, q, p = distill64(logits[2:5], indices[2:5], teacher[2:5], 1.0)
    close(loss[2:5], loss64, size, 2.0 ** -17)
    close(grad[2:5], grad64, q + p, 2.0 ** -17)
    assert loss[5] == math.inf and grad[5].isfinite().all()
    assert loss[6].isnan() and loss[7].isnan() and loss[8].isnan() and grad[6:].isnan().all()
    leaf = logits.clone().requires_grad_()
    losses = distillation_loss(leaf, indices, teacher, reduction="none")
    torch.testing.assert_close(losses.detach(), loss, equal_nan=True)
    (again,) = torch.autograd.grad(losses, leaf, torch.ones_like(losses))
    torch.testing.assert_close(again, grad, equal_nan=True)
    # The mean counts the rows that have entries; none gives 0.
    two = distillation_loss(logits[:3], indices[:3], teacher[:3])
    torch.testing.assert_close(two, loss[2])
    empty = logits[:2].clone().requires_grad_()
    nothing = distillation_loss(empty, indices[:2], teacher[:2])
    assert nothing == 0 and not torch.autograd.grad(nothing, empty)[0].any()


@pytest.mark.parametrize("dtype", TYPES)
def test_distillation_finds_one_value_that_is_not_finite_anywhere(dtype):
    """Wherever in a 16-byte word it is: NaN and inf make the row NaN, -inf and the lowest value are left out."""
    vocab = 1003
    logits, indices, teacher = _distill_inputs(64, vocab, 4, dtype)
    indices[:] = torch.tensor([100, 200, 300, 400], device=DEV)
    for i in range(16):
        logits[i, 500 + i] = math.nan
        logits[16 + i, 500 + i] = math.inf
        logits[32 + i, 500 + i] = -math.inf
        logits[48 + i, 500 + i] = torch.finfo(dtype).min
    loss, grad = distillation_loss_and_grad(logits, indices, teacher)
    leaf = logits.detach().requires_grad_()
    losses = distillation_loss(leaf, indices, teacher, reduction="none")
    (again,) = torch.autograd.grad(losses, leaf, torch.ones_like(losses))
    loss64, size, grad64, q, p = distill64(logits[32:], indices[32:], teacher[32:], 1.0)
    for one, slope in ((loss, grad), (losses.detach(), again)):
        assert one[:32].isnan().all() and slope[:32].isnan().all()
        close(one[32:], loss64, size, 2.0 ** -17)
        close(slope[32:], grad64, q + p, 2.0 ** -17)
    for i in range(32):
        assert grad[32 + i, 500 + i % 16] == 0 and again[32 + i, 500 + i % 16] == 0


@pytest.mark.parametrize("dtype", TYPES)
def test_distillation_of_rows_masked_throughout(dtype):
    """All of the vocabulary at the type's lowest value is a uniform distribution."""
    vocab = 5001
    logits, indices, teacher = _distill_inputs(3, vocab, 4, dtype)
    logits[0] = torch.finfo(dtype).min
    logits[1] = torch.finfo(dtype).max
    logits[2, ::2] = torch.finfo(dtype).min
    loss64, size, grad64, q, p = distill64(logits, indices, teacher, 1.0)
    loss, grad = distillation_loss_and_grad(logits, indices, teacher)
    close(loss, loss64, size, 2.0 ** -17)
    close(grad, grad64, q + p, 2.0 ** -17)
    losses = distillation_loss(logits, indices, teacher, reduction="none")
    close(losses, loss64, size, 2.0 ** -17)


def test_distillation_shapes_types_and_no_rows():
    logits, indices, teacher = _distill_inputs(6, 500, 8, torch.bfloat16)
    flat = distillation_loss_and_grad(logits, indices, teacher)
    columns = [t.t().contiguous().t() for t in (logits, indices, teacher)]
    for got, want in zip(distillation_loss_and_grad(*columns), flat):
        assert torch.equal(got, want)
    leaf = columns[0].requires_grad_()
    (grad,) = torch.autograd.grad(distillation_loss(leaf, *columns[1:], reduction="sum"), leaf)
    _, _, grad64, q, p = distill64(logits, indices, teacher, 1.0)
    close(grad, grad64, q + p, 2.0 ** -17)
    loss, grad = distillation_loss_and_grad(logits.view(2, 3, 500), indices.view(2, 3, 8), teacher.view(2, 3, 8),
                                            grad_loss=torch.ones(2, 3, device=DEV))
    assert torch.equal(loss.view(-1), flat[0]) and torch.equal(grad.view(6, 500), flat[1])
    assert distillation_loss(logits.view(2, 3, 500), indices.view(2, 3, 8), teacher.view(2, 3, 8),
                             reduction="none").shape == (2, 3)
    for dtype in (torch.bfloat16, torch.float16):
        rounded = teacher.to(dtype)
        assert torch.equal(distillation_loss(logits, indices, rounded, reduction="none"),
                           distillation_loss(logits, indices, rounded.float(), reduction="none"))
    none = logits[:0].clone().requires_grad_()
    loss = distillation_loss(none, indices[:0], teacher[:0])
    assert loss == 0 and torch.autograd.grad(loss, none)[0].shape == (0, 500)
    assert distillation_loss_and_grad(logits[:0], indices[:0], teacher[:0])[0].shape == (0,)


def test_distillation_gradient_against_differences():
    logits, indices, teacher = _distill_inputs(4, 50, 6, torch.float32)
    loss, grad = distillation_loss_and_grad(logits, indices, teacher, 2.0)
    direction = torch.sign(grad)
    h = 2.0 ** -6
    up = distillation_loss(logits + h * direction, indices, teacher, 2.0, "none")
    down = distillation_loss(logits - h * direction, indices, teacher, 2.0, "none")
    slope = (up.double() - down.double()) / (2 * h)
    total = grad.double().abs().sum(1)
    # h^2 / 6 of third derivatives of order 1 / tau, and 2^-23 of a loss of order 10 over h.
    assert ((slope - total).abs() <= 2.0 ** -10 * total + 2.0 ** -12).all()


# -------------------------------------------------------------- all three ----

def _everything(seed):
    g = rng(seed)
    q, k = normal(g, 40, 14, 64, dtype=torch.bfloat16), normal(g, 40, 2, 64, dtype=torch.bfloat16)
    table, positions = rotary_table(64, 64), torch.arange(40, device=DEV)
    x, base, a, b, scale, batch = _adapter_inputs(ADAPTER_CASES[2], torch.bfloat16, seed)
    logits, indices, teacher = _distill_inputs(5, 9001, 16, torch.bfloat16, seed)

    def call():
        return (*head_norm_rotary(q, k, table, positions), low_rank_adapters(base, x, a, b, batch, scale),
                *distillation_loss_and_grad(logits, indices, teacher),
                distillation_loss(logits, indices, teacher))

    return call, (q, base, logits)


def test_on_another_stream_and_in_a_graph():
    call, inputs = _everything(0)
    want = call()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = call()
    side.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = call()
    for t in inputs:
        t.copy_(torch.roll(t, 1, 0))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(captured, call()))


def test_second_derivatives_are_refused():
    call, _ = _everything(1)
    logits, indices, teacher = _distill_inputs(5, 900, 16, torch.float32)
    leaf = logits.requires_grad_()
    (grad,) = torch.autograd.grad(distillation_loss(leaf, indices, teacher), leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiate twice"):
        grad.square().sum().backward()


def test_in_place_forms_are_seen_by_autograd():
    x, base, a, b, scale, batch = _adapter_inputs(ADAPTER_CASES[1], torch.bfloat16)
    factor = base.clone().requires_grad_()
    product = factor * base  # saves base
    low_rank_adapters_(base, x, a, b, batch, scale)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        product.sum().backward()
    # In place on a projection's output with gradients: as out of place.
    leaves = [t.detach().clone().requires_grad_() for t in (base, x, a, b)]
    want = torch.autograd.grad(low_rank_adapters(leaves[0] * 2, *leaves[1:], batch, scale).float().square().sum(), leaves)
    out = low_rank_adapters_(leaves[0] * 2, *leaves[1:], batch, scale)
    for g, w in zip(torch.autograd.grad(out.float().square().sum(), leaves), want):
        assert torch.equal(g, w)
    logits, indices, teacher = _distill_inputs(3, 100, 4, torch.float32)
    factor = torch.ones_like(logits, requires_grad=True)
    product = factor * logits
    distillation_loss_and_grad(logits, indices, teacher, in_place=True)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        product.sum().backward()
    with torch.inference_mode():
        low_rank_adapters_(base.clone(), x, a, b, batch, scale)
        distillation_loss_and_grad(logits.clone(), indices, teacher, in_place=True)


def test_refusals():
    q, k = torch.zeros(4, 2, 64, device=DEV), torch.zeros(4, 1, 64, device=DEV)
    table, positions = rotary_table(8, 64), torch.arange(4, device=DEV)
    w = torch.ones(64, device=DEV)
    with pytest.raises(RuntimeError, match="same dtype"):
        head_norm_rotary(q, k.half(), table, positions)
    with pytest.raises(RuntimeError, match="positions must be"):
        head_norm_rotary(q, k, table, positions[:3])
    with pytest.raises(RuntimeError, match="positions must be int"):
        head_norm_rotary(q, k, table, positions.float())
    with pytest.raises(RuntimeError, match="agree in tokens"):
        head_norm_rotary(q, k[:3], table, positions)
    with pytest.raises(RuntimeError, match="both q and k"):
        head_norm_rotary(q, k, table, positions, w)
    with pytest.raises(RuntimeError, match=r"\[dim\]"):
        head_norm_rotary(q, k, table, positions, w[:32], w[:32])
    with pytest.raises(RuntimeError, match="rotary dimension"):
        head_norm_rotary(q, k, rotary_table(8, 66), positions)
    with pytest.raises(RuntimeError, match="head dimension"):
        head_norm_rotary(q[..., :63], k[..., :63], rotary_table(8, 2), positions)
    with pytest.raises(RuntimeError, match="eps"):
        head_norm_rotary(q, k, table, positions, w, w, -1.0)

    x, base, a, b, scale, batch = _adapter_inputs(ADAPTER_CASES[1], torch.bfloat16)
    with pytest.raises(RuntimeError, match="BF16 or FP16"):
        low_rank_adapters(base.float(), x.float(), a.float(), b.float(), batch, scale)
    with pytest.raises(RuntimeError, match="another number of tokens"):
        low_rank_adapters(base[:4], x[:4], a, b, batch, scale)
    with pytest.raises(RuntimeError, match="another number of tokens or adapters"):
        low_rank_adapters(base, x, a[:3], b[:3], batch, scale[:3])
    with pytest.raises(RuntimeError, match="contiguous"):
        low_rank_adapters(base, x, a.transpose(1, 2).contiguous().transpose(1, 2), b, batch, scale)
    with pytest.raises(RuntimeError, match="rank"):
        low_rank_adapters(base, x, a[:, :4].contiguous(), b, batch, scale)
    with pytest.raises(RuntimeError, match="scales"):
        low_rank_adapters(base, x, a, b, batch, scale.half())
    with pytest.raises(RuntimeError, match="projection's output"):
        low_rank_adapters(base[:, 1:], x, a, b, batch, scale)
    with pytest.raises(RuntimeError, match="overlap|single memory location"):
        low_rank_adapters_(base[:1].expand(5, -1), x, a, b, batch, scale)
    with pytest.raises(ValueError, match="AdapterBatch"):
        low_rank_adapters(base, x, a, b, None, scale)
    with pytest.raises(RuntimeError, match="not differentiable"):
        low_rank_adapters(base, x, a, b, batch, scale.requires_grad_())

    logits, indices, teacher = _distill_inputs(3, 100, 4, torch.float32)
    with pytest.raises(ValueError, match="temperature"):
        distillation_loss(logits, indices, teacher, 0.0)
    with pytest.raises(ValueError, match="reduction"):
        distillation_loss(logits, indices, teacher, reduction="batchmean")
    with pytest.raises(ValueError, match="teacher indices"):
        distillation_loss(logits, indices[:2], teacher[:2])
    with pytest.raises(RuntimeError, match="1 to 1024"):
        distillation_loss(logits, indices.repeat(1, 300), teacher.repeat(1, 300))
    with pytest.raises(RuntimeError, match="int32 or int64"):
        distillation_loss(logits, indices.float(), teacher)
    with pytest.raises(RuntimeError, match="FP32, BF16 or FP16"):
        distillation_loss(logits.double(), indices, teacher)
    with pytest.raises(RuntimeError, match="contiguous"):
        distillation_loss_and_grad(logits.t().contiguous().t(), indices, teacher, in_place=True)
    with pytest.raises(RuntimeError, match="overlap"):
        distillation_loss_and_grad(logits[:1].expand(3, -1), indices, teacher, in_place=True)
    with pytest.raises(RuntimeError, match="loss gradient"):
        distillation_loss_and_grad(logits, indices, teacher, grad_loss=torch.ones(2, device=DEV))
