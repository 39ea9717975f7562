"""Uses of the layer operators that are easily lost beside the ordinary ones:
several host threads, values that are not finite beside finite ones, the ends
of a type's range, derivatives that do not exist, views under autograd, waits
that run out, and walks of many rows, tiles and tokens by one block.

Tolerances as in the operators' other tests: one rounding to the output's type
plus a power of two times the sum of the magnitudes that enter an element.
"""
import ctypes
import threading

import pytest
import torch
from torch.autograd import forward_ad

import test_layers_gpu as layers
from sdc_b200 import capi
from sdc_b200.layers import (AdapterBatch, distillation_loss, distillation_loss_and_grad, head_norm_rotary,
                             low_rank_adapters, low_rank_adapters_, rotary_table)

pytestmark = pytest.mark.gpu
DEV = "cuda"


def rng(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def normal(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, device=DEV, generator=g) * scale).to(dtype)


# ------------------------------------------------------------------ threads ----

@pytest.mark.parametrize("lengths,ranks", [([1600], (64, 32)), ([700], (256, 160))])
def test_threads_do_not_take_each_others_shared_memory(lengths, ranks):
    """The kernels' shared memory grows with the rank (tiles of 128 rows and of 16). A second thread's first, smaller
    call comes between two larger ones of the first thread."""
    inputs = {}
    for rank in ranks:
        g = rng(rank)
        tokens, dtype = sum(lengths), torch.bfloat16
        inputs[rank] = (normal(g, tokens, 264, dtype=dtype), normal(g, tokens, 136, dtype=dtype),
                        normal(g, 1, rank, 136, dtype=dtype), normal(g, 1, 264, rank, dtype=dtype),
                        AdapterBatch(lengths, [0], 1))
    large, small = ranks
    between, done = threading.Event(), threading.Event()
    results, errors = [], []

    def call(rank):
        try:
            results.append(low_rank_adapters(*inputs[rank]))
        except Exception as error:  # reported by the test, in its own thread
            errors.append(error)

    def first():
        call(large)
        between.set()
        done.wait(60)
        call(large)

    def second():
        between.wait(60)
        call(small)
        done.set()

    threads = [threading.Thread(target=f) for f in (first, second)]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    assert not errors
    assert torch.equal(results[0], results[2])


# ----------------------------------------------------------------- rotation ----

# dim, rotary, interleaved: half-split and interleaved heads in whole runs, and heads without a vector form.
PASSING = [(128, 64, False), (96, 32, False), (80, 40, True), (64, 10, True), (34, 10, True), (48, 24, False), (6, 4, False)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("case", PASSING)
def test_passing_elements_of_a_head_stay_apart(case, dtype):
    """Elements beyond the rotary part pass each by itself: one that is not finite leaves all others as they were."""
    dim, rotary, interleaved = case
    heads = 2 * (dim - rotary)  # one head for every passing element and value
    clean = normal(rng(0), 3, heads, dim, dtype=dtype)
    q = clean.clone()
    expected_bad = torch.zeros_like(q, dtype=torch.bool)
    for i in range(dim - rotary):
        q[:, i, rotary + i] = float("inf")
        q[:, dim - rotary + i, rotary + i] = float("nan")
        expected_bad[:, [i, dim - rotary + i], rotary + i] = True
    table, positions = rotary_table(8, rotary), torch.tensor([0, 3, 7], device=DEV)
    k = clean[:, :1]
    want = head_norm_rotary(clean, k, table, positions, interleaved=interleaved)[0]
    got = head_norm_rotary(q, k, table, positions, interleaved=interleaved)[0]
    assert torch.equal(got[~expected_bad], want[~expected_bad])
    assert torch.equal(torch.nan_to_num(got[expected_bad], 1., 2.), torch.nan_to_num(q[expected_bad], 1., 2.))
    # The gradient is the opposite rotation.
    grads = []
    for upstream in (clean, q):
        leaf = clean.detach().requires_grad_()
        out = head_norm_rotary(leaf, k, table, positions, interleaved=interleaved)[0]
        grads.append(torch.autograd.grad(out, leaf, upstream)[0])
    assert torch.equal(grads[1][~expected_bad], grads[0][~expected_bad])
    assert not grads[1][expected_bad].isfinite().any()
    # With the norm an infinite head is zeros beside its infinity over infinity.
    ones = torch.ones(dim, device=DEV, dtype=dtype)
    normed = head_norm_rotary(q, k, table, positions, ones, ones, interleaved=interleaved)[0][:, :dim - rotary]
    bad = expected_bad[:, :dim - rotary]
    assert normed[bad].isnan().all() and not normed[~bad].any()


# -------------------------------------------------------------- derivatives ----

def _small():
    g = rng(7)
    q, table, positions, w = normal(g, 3, 2, 64), rotary_table(8, 64), torch.arange(3, device=DEV), normal(g, 64)
    base, x = normal(g, 8, 48, dtype=torch.bfloat16), normal(g, 8, 64, dtype=torch.bfloat16)
    a, b = normal(g, 2, 8, 64, dtype=torch.bfloat16), normal(g, 2, 48, 8, dtype=torch.bfloat16)
    logits, teacher = normal(g, 3, 50), normal(g, 3, 4)
    return q, table, positions, w, base, x, a, b, torch.ones(2, device=DEV), AdapterBatch([5, 3], [0, 1], 2), logits, teacher


def test_forward_mode_derivatives_are_refused():
    """A dual tensor that asks for no gradient must not lose its tangent."""
    q, table, positions, w, base, x, a, b, scale, batch, logits, teacher = _small()
    indices = torch.tensor([[0, 7, 49, -1]] * 3, device=DEV)
    calls = [
        (q, lambda t: head_norm_rotary(t, q, table, positions)), (q, lambda t: head_norm_rotary(q, t, table, positions)),
        (table, lambda t: head_norm_rotary(q, q, t, positions)), (w, lambda t: head_norm_rotary(q, q, table, positions, t, w)),
        (w, lambda t: head_norm_rotary(q, q, table, positions, w, t)),
        (base, lambda t: low_rank_adapters(t, x, a, b, batch)), (x, lambda t: low_rank_adapters(base, t, a, b, batch)),
        (a, lambda t: low_rank_adapters(base, x, t, b, batch)), (b, lambda t: low_rank_adapters(base, x, a, t, batch)),
        (scale, lambda t: low_rank_adapters(base, x, a, b, batch, t)),
        (base, lambda t: low_rank_adapters_(t, x, a, b, batch)), (x, lambda t: low_rank_adapters_(base, t, a, b, batch)),
        (logits, lambda t: distillation_loss(t, indices, teacher)), (teacher, lambda t: distillation_loss(logits, indices, t)),
        (logits, lambda t: distillation_loss_and_grad(t, indices, teacher)),
        (logits, lambda t: distillation_loss_and_grad(t, indices, teacher, in_place=True)),
    ]
    for primal, call in calls:
        before = primal.clone()
        for requires_grad in (False, True):
            with forward_ad.dual_level():
                dual = forward_ad.make_dual(primal.clone().requires_grad_(requires_grad), torch.ones_like(primal))
                with pytest.raises(RuntimeError, match="forward-mode|not differentiable|leaf"):
                    call(dual)
        assert torch.equal(primal, before)


def test_gradients_that_do_not_exist_are_refused():
    """Of the rotation table and of the teacher's logits, unless nothing is recorded."""
    q, table, positions, _, _, _, _, _, _, _, logits, teacher = _small()
    indices = torch.tensor([[0, 7, 49, -1]] * 3, device=DEV)
    with pytest.raises(RuntimeError, match="table is not differentiable"):
        head_norm_rotary(q, q, table.clone().requires_grad_(), positions)
    tracked = teacher.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="teacher"):
        distillation_loss(logits, indices, tracked)
    want = distillation_loss(logits, indices, teacher)
    assert torch.equal(distillation_loss(logits, indices, tracked.detach()), want)
    with torch.no_grad():
        assert torch.equal(distillation_loss(logits, indices, tracked), want)
        head_norm_rotary(q, q, table.clone().requires_grad_(), positions)
    distillation_loss_and_grad(logits, indices, tracked)  # records nothing


def test_adapters_into_views_under_autograd():
    """A projection's output is often a view: of other dimensions, or of a wider tensor whose rest is used as well."""
    _, _, _, _, base, x, a, b, scale, batch, _, _ = _small()

    def gradients(call, record_base):
        leaves = [t.clone().requires_grad_() for t in (base, x, a, b)]
        first = leaves[0] * 2 if record_base else leaves[0].detach() * 2
        out = call(first, *leaves[1:])
        return (out, *torch.autograd.grad(out.float().square().sum(), leaves, allow_unused=True))

    def reshaped(first, *rest):
        low_rank_adapters_(first.view(2, 4, 48).view(8, 48), *rest, batch, scale)
        return first

    def part(first, *rest):
        side = first.detach()  # one gradient a column: autograd's own bf16 additions have no fixed order
        wide = torch.cat((side, first, side), 1)
        low_rank_adapters_(wide[:, 48:96], *rest, batch, scale)
        return wide

    for record_base in (True, False):
        want = gradients(lambda first, *rest: low_rank_adapters(first, *rest, batch, scale), record_base)
        for got, expected in zip(gradients(reshaped, record_base), want):
            assert got is expected is None or torch.equal(got, expected)
        want = gradients(lambda first, *rest: torch.cat((first.detach(), low_rank_adapters(first, *rest, batch, scale),
                                                         first.detach()), 1), record_base)
        for got, expected in zip(gradients(part, record_base), want):
            assert got is expected is None or torch.equal(got, expected)


def test_adapters_refuse_a_leaf_before_they_change_it():
    _, _, _, _, base, x, a, b, scale, batch, _, _ = _small()
    for refused in (base.clone().requires_grad_(), base.clone().requires_grad_().view(8, 48)):
        with pytest.raises(RuntimeError, match="leaf Variable that requires grad"):
            low_rank_adapters_(refused, x, a, b, batch, scale)
        assert torch.equal(refused, base)
        with torch.no_grad():
            assert torch.equal(low_rank_adapters_(refused, x, a, b, batch, scale),
                               low_rank_adapters(base, x, a, b, batch, scale))


# ----------------------------------------------------------- adapters' values ----

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens", [9, 1600])
@pytest.mark.parametrize("rank", [1, 5, 16, 24])
def test_adapters_of_any_rank_keep_infinities(rank, tokens, dtype):
    """An infinite input with weights of one sign is an infinite output: the columns that pad a rank add nothing."""
    g = rng(rank)
    batch = AdapterBatch([tokens], [0], 1)
    x, base = normal(g, tokens, 72, dtype=dtype), normal(g, tokens, 136, dtype=dtype)
    x[3, 5], x[4, 6] = float("inf"), float("-inf")
    a, b = normal(g, 1, rank, 72, dtype=dtype).abs() + 0.1, normal(g, 1, 136, rank, dtype=dtype).abs() + 0.1
    leaf = x.clone().requires_grad_()
    out = low_rank_adapters(base, leaf, a, b, batch)
    assert (out[3] == float("inf")).all() and (out[4] == float("-inf")).all()
    rest = torch.ones(tokens, dtype=torch.bool, device=DEV)
    rest[3:5] = False
    assert out[rest].isfinite().all()
    grad = torch.ones_like(out)
    grad[7, 9] = float("inf")
    (dx,) = torch.autograd.grad(out, leaf, grad)
    assert (dx[7] == float("inf")).all()
    dx[7] = 0
    assert dx.isfinite().all()


def close(got, exact, magnitude, arithmetic):
    """One rounding of ``exact`` to fp16 and ``arithmetic`` times ``magnitude``."""
    tolerance = 2.0 ** -11 * exact.abs() * (1 + 2.0 ** -10) + 2.0 ** -25 + arithmetic * magnitude
    off = (got.double() - exact).abs()
    bad = ~(off <= tolerance)
    assert not bad.any(), (off[bad].max().item(), tolerance[bad].min().item(), int(bad.sum()))


# Two terms of the low-rank rows lose 2^-21, and the floor of their scaling (2^-39 of the largest) less than that among
# normal rows; fp32 sums of n products lose at most n 2^-23 of their magnitude.
def fp16_arithmetic(*lengths):
    return 2.0 ** -20 + sum(lengths) * 2.0 ** -23


def adapters64(x, base, a, b, grad):
    """One adapter's outputs and gradients, each with the magnitude of what enters its elements."""
    def run(x, base, a, b, grad):
        low, down = x @ a.T, grad @ b
        return base + low @ b.T, down @ a, down.T @ x, grad.T @ low
    x, base, a, b, grad = (t.double() for t in (x, base, a, b, grad))
    return list(zip(run(x, base, a, b, grad), run(x.abs(), base.abs(), a.abs(), b.abs(), grad.abs())))


# Scales of x, a, b and the gradient. The gradients of a mean loss beside a weight that starts near zero: low-rank rows
# of 1e-7 (fp16 ends at 6e-8). Large inputs: rows beyond 65504 that the second weight brings back.
FP16_RANGES = {"small": (1.0, 0.05, 1e-3, 1e-5), "smaller": (1e-2, 1e-3, 10.0, 1e-6), "large": (100.0, 10.0, 1e-4, 1e-4)}


@pytest.mark.parametrize("ranges", list(FP16_RANGES))
@pytest.mark.parametrize("tokens,rank,k,n", [(1, 16, 200, 136), (60, 5, 104, 520), (300, 256, 264, 136), (1600, 24, 200, 136),
                                             (1600, 64, 37, 53), (2100, 100, 200, 136), (1600, 256, 264, 136)])
def test_fp16_adapters_over_the_range_of_their_low_rows(tokens, rank, k, n, ranges):
    g = rng(tokens + rank)
    sx, sa, sb, sg = FP16_RANGES[ranges]
    dtype = torch.float16
    x, base, grad = (normal(g, tokens, k, dtype=dtype, scale=sx), normal(g, tokens, n, dtype=dtype),
                     normal(g, tokens, n, dtype=dtype, scale=sg))
    a, b = normal(g, 1, rank, k, dtype=dtype, scale=sa), normal(g, 1, n, rank, dtype=dtype, scale=sb)
    leaves = [t.clone().requires_grad_() for t in (x, a, b)]
    out = low_rank_adapters(base, *leaves, AdapterBatch([tokens], [0], 1))
    dx, da, db = torch.autograd.grad(out, leaves, grad)
    exact = adapters64(x, base, a[0], b[0], grad)
    for got, (value, size), lengths in zip((out.detach(), dx, da[0], db[0]), exact,
                                           ((k, rank), (n, rank), (n, tokens), (k, tokens))):
        close(got, value, size, fp16_arithmetic(*lengths))


@pytest.mark.parametrize("tokens", [40, 1700])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_adapters_of_a_token_do_not_depend_on_the_other_tokens_values(tokens, dtype):
    g = rng(tokens)
    x, base = normal(g, tokens, 128, dtype=dtype), normal(g, tokens, 264, dtype=dtype)
    a, b = normal(g, 1, 24, 128, dtype=dtype, scale=0.1), normal(g, 1, 264, 24, dtype=dtype, scale=0.1)
    grad, batch = normal(g, tokens, 264, dtype=dtype), AdapterBatch([tokens], [0], 1)

    def results(x, grad):
        leaf = x.clone().requires_grad_()
        out = low_rank_adapters(base, leaf, a, b, batch)
        return out, torch.autograd.grad(out, leaf, grad)[0]

    want = results(x, grad)
    changed = torch.arange(0, tokens, 3, device=DEV)
    factors = torch.tensor([2.0 ** -14, 1e3, 0.0, float("inf")], device=DEV)[torch.arange(len(changed), device=DEV) % 4, None]
    x2, grad2 = x.clone(), grad.clone()
    x2[changed] = (x2[changed].float() * factors).to(dtype)
    grad2[changed] = (grad2[changed].float() * factors).to(dtype)
    rest = torch.ones(tokens, dtype=torch.bool, device=DEV)
    rest[changed] = False
    for got, expected in zip(results(x2, grad2), want):
        assert torch.equal(got[rest], expected[rest])


def test_fp16_adapters_add_tokens_of_unlike_sizes():
    """The weights' gradients of tokens between 2^-14 and 2^7 of one another, in long and short runs."""
    dtype = torch.float16
    for tokens in (50, 1600, 5000):
        g = rng(tokens)
        size = 2.0 ** torch.randint(-14, 8, (tokens, 1), device=DEV, generator=g)
        x, grad = (normal(g, tokens, 136) * size).to(dtype), (normal(g, tokens, 264) * size.flip(0) * 2.0 ** -8).to(dtype)
        base = normal(g, tokens, 264, dtype=dtype)
        a, b = normal(g, 1, 40, 136, dtype=dtype, scale=0.1), normal(g, 1, 264, 40, dtype=dtype, scale=0.1)
        leaves = [t.clone().requires_grad_() for t in (x, a, b)]
        out = low_rank_adapters(base, *leaves, AdapterBatch([tokens], [0], 1))
        dx, da, db = torch.autograd.grad(out, leaves, grad)
        for got, (value, magnitude), lengths in zip((out.detach(), dx, da[0], db[0]), adapters64(x, base, a[0], b[0], grad),
                                                    ((136, 40), (264, 40), (264, tokens), (136, tokens))):
            close(got, value, magnitude, fp16_arithmetic(*lengths))


# ------------------------------------------------------------- expired waits ----

WAIT_ADAPTERS, WAIT_DISTILL = 9, 10  # codes of the device watchdog


def _watchdog():
    code = ctypes.c_int32(-1)
    capi.check(capi.lib().sdc_read_device_error(torch.cuda.current_stream().cuda_stream, ctypes.byref(code)))
    return code.value


def _expired(call):
    """The call's result where a wait runs out after a millisecond (one for a barrier that nothing arrives at)."""
    try:
        capi.check(capi.lib().sdc_test_set_watchdog(1_000_000, 1))
        result = call()
        torch.cuda.synchronize()
    finally:
        capi.check(capi.lib().sdc_test_set_watchdog(0, 0))
    return result


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_adapters_report_an_expired_wait_in_their_results(dtype):
    g = rng(9)
    lengths, adapters = [1300, 40, 700], [0, -1, 1]
    tokens, batch = sum(lengths), AdapterBatch(lengths, adapters, 3)
    x, base, grad = (normal(g, tokens, w, dtype=dtype) for w in (264, 520, 520))
    a, b = normal(g, 3, 24, 264, dtype=dtype), normal(g, 3, 520, 24, dtype=dtype)
    adapted = torch.ones(tokens, dtype=torch.bool, device=DEV)
    adapted[1300:1340] = False

    def call():
        leaves = [t.clone().requires_grad_() for t in (x, a, b)]
        out = low_rank_adapters(base, *leaves, batch)
        return (out, *torch.autograd.grad(out, leaves, grad))

    assert _watchdog() == 0
    want = call()
    out, dx, da, db = _expired(call)
    assert out[adapted].isnan().all() and dx[adapted].isnan().all()
    assert da[:2].isnan().all() and db[:2].isnan().all() and not da[2].any() and not db[2].any()
    assert _watchdog() == WAIT_ADAPTERS
    assert low_rank_adapters_(base.clone(), x, a, b, batch).isfinite().all()
    in_place = _expired(lambda: low_rank_adapters_(base.clone(), x, a, b, batch))
    assert in_place[adapted].isnan().all()
    assert torch.equal(in_place[~adapted], base[~adapted])
    assert _watchdog() == WAIT_ADAPTERS

    # Each kernel by itself, on whole operands.
    rows, groups, tiles, slots, active, tile_rows = batch.arguments(24)
    assert tile_rows == 128
    low = torch.ops.sdc_cutlass.low_rank_adapters(base, x, a, b, None, *batch.arguments(24))[1]
    code, stream = {torch.bfloat16: 1, torch.float16: 2}[dtype], torch.cuda.current_stream().cuda_stream
    expanded, outer = torch.zeros_like(base), torch.zeros_like(b)

    def expand():
        capi.check(capi.lib().sdc_adapter_expand(code, base.data_ptr(), 520, tokens, rows.data_ptr(), tiles.data_ptr(), active,
                                                 128, b.data_ptr(), 3, 24, 520, 1, low.data_ptr(), slots, 0,
                                                 expanded.data_ptr(), 520, stream))
        return expanded

    def products():
        capi.check(capi.lib().sdc_adapter_outer(code, grad.data_ptr(), 520, tokens, rows.data_ptr(), groups.data_ptr(), 3,
                                                low.data_ptr(), slots, 24, 520, 1, outer.data_ptr(), stream))
        return outer

    assert _expired(expand)[adapted].isnan().all() and not expanded[~adapted].any()
    assert _expired(products)[:2].isnan().all() and not outer[2].any()
    assert _watchdog() == WAIT_ADAPTERS
    assert torch.equal(expand()[adapted], want[0][adapted]) and torch.equal(products(), want[3])
    for got, expected in zip(call(), want):
        assert torch.equal(got, expected)
    assert _watchdog() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_distillation_reports_an_expired_wait_in_its_results(dtype):
    g = rng(10)
    for rows, vocab in ((5, 3001), (700, 513)):  # clusters of several blocks, and several rows a cluster
        logits, teacher = normal(g, rows, vocab, dtype=dtype), normal(g, rows, 8)
        indices = torch.randint(0, vocab, (rows, 8), device=DEV, generator=g)
        indices[1] = -1
        want = distillation_loss_and_grad(logits, indices, teacher)
        assert _watchdog() == 0
        for in_place in (False, True):
            loss, grad = _expired(lambda: distillation_loss_and_grad(logits.clone(), indices, teacher, in_place=in_place))
            assert loss.isnan().all() and grad.isnan().all()
            assert _watchdog() == WAIT_DISTILL
        for got, expected in zip(distillation_loss_and_grad(logits, indices, teacher), want):
            assert torch.equal(got, expected)
        assert _watchdog() == 0


# -------------------------------------------------------------------- walks ----
# Blocks that stay for the whole launch walk over tokens, tiles or rows. Here each of them has several.

def _sms():
    return torch.cuda.get_device_properties(0).multi_processor_count


@pytest.mark.parametrize("rows,vocab,top,dtype", [(2000, 513, 16, torch.bfloat16), (1999, 514, 16, torch.float32),
                                                  (700, 50021, 33, torch.float32), (300, 151937, 64, torch.bfloat16),
                                                  (2100, 4099, 200, torch.float16)])
def test_distillation_walks_many_rows(rows, vocab, top, dtype):
    """Odd vocabularies (rows start elsewhere in their words), rows without entries and with stray ones between others."""
    g = rng(rows)
    logits, teacher = normal(g, rows, vocab, dtype=dtype, scale=3.0), normal(g, rows, top, scale=3.0)
    indices = torch.randint(0, vocab, (rows, top), device=DEV, generator=g)
    indices[torch.rand(rows, top, device=DEV, generator=g) < 0.2] = -1
    kind = torch.rand(rows, device=DEV, generator=g)
    empty, stray = kind < 0.2, kind > 0.95
    indices[empty] = -1
    logits[empty] = float("nan")  # of which nothing is looked at
    indices[stray, 0] = vocab
    # At most three blocks stay on an SM; a row's words fill as many blocks of 74 KB as it takes.
    assert rows > 3 * _sms() / max(1, vocab * logits.element_size() // (74 * 1024)) * 2
    upstream = normal(g, rows)
    loss, grad = distillation_loss_and_grad(logits, indices, teacher, 1.5, upstream)
    replaced = logits.clone()
    again = distillation_loss_and_grad(replaced, indices, teacher, 1.5, upstream, in_place=True)
    good = ~stray
    for first, second in ((loss, again[0]), (grad, replaced)):
        assert torch.equal(first[good], second[good])
        assert first[stray].isnan().all() and second[stray].isnan().all()
        assert not first[empty].any()
    kept = indices >= 0
    for start in range(0, rows, 200):
        part = slice(start, start + 200)
        some = good[part] & ~empty[part]
        s, t, at = logits[part][some].double() / 1.5, teacher[part][some].double() / 1.5, indices[part][some]
        log_q = torch.log_softmax(s, 1)
        log_p = torch.log_softmax(t.masked_fill(at < 0, -float("inf")), 1)
        p = log_p.exp()
        chosen = log_q.gather(1, at.clamp_min(0))
        exact = torch.where(at >= 0, p * (log_p - chosen), 0.0).sum(1) * 2.25
        size = torch.where(at >= 0, p * (log_p.abs() + chosen.abs() + 1), 0.0).sum(1) * 2.25
        assert ((loss[part][some].double() - exact).abs() <= 2.0 ** -24 * exact.abs() + 2.0 ** -17 * size).all()
        spread = torch.zeros_like(s).scatter_add_(1, at.clamp_min(0), torch.where(at >= 0, p, 0.0))
        row = upstream[part][some].double()[:, None] * 1.5
        q = log_q.exp()
        exact, size = (q - spread) * row, (q + spread) * row.abs()
        unit = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}[dtype]
        tolerance = unit * exact.abs() * (1 + 2.0 ** -10) + (2.0 ** -25 if dtype == torch.float16 else 1e-38) + 2.0 ** -17 * size
        assert ((grad[part][some].double() - exact).abs() <= tolerance).all()
    assert kept[good & ~empty].any(1).all()


@pytest.mark.parametrize("lengths,ids,count,rank,k,n", [
    ([700, 300, 37, 900, 128, 1100], [0, 1, -1, 2, 0, 1], 4, 16, 136, 18944),   # two weights
    ([700, 300, 37, 900, 128, 1100], [0, 1, -1, 2, 0, 1], 4, 48, 18944, 136),
    ([2000, 30, 1500], [0, -1, 2], 3, 64, 136, 18944),                          # one
    ([130, 140, 1900, 150, 800], [3, 0, 1, 2, -1], 4, 128, 18941, 37),          # no vector form
    ([130, 140, 1900, 150, 800], [3, 0, 1, 2, -1], 4, 24, 37, 18941),
])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_adapters_walk_many_tiles(lengths, ids, count, rank, k, n, dtype):
    g = rng(rank)
    tokens, batch = sum(lengths), AdapterBatch(lengths, ids, count)
    x, base, grad = (normal(g, tokens, w, dtype=dtype) for w in (k, n, n))
    a, b = normal(g, count, rank, k, dtype=dtype, scale=k ** -0.5), normal(g, count, n, rank, dtype=dtype, scale=rank ** -0.5)
    scale = torch.rand(count, device=DEV, generator=g) + 0.5
    tiles, tile_rows = batch.arguments(rank)[2], batch.arguments(rank)[5]
    # Blocks of 256 columns, at most two on an SM.
    assert tile_rows == 128 and len(tiles) > 2 * (2 * _sms() // -(-max(k, n) // 256))
    leaves = [t.clone().requires_grad_() for t in (x, a, b)]
    out = low_rank_adapters(base, *leaves, batch, scale)
    dx, da, db = torch.autograd.grad(out, leaves, grad)
    in_place = low_rank_adapters_(base.clone(), x, a, b, batch, scale)
    assert torch.equal(in_place, out)
    exact, size, parts = layers.adapters64(lengths, ids, x, base, a, b, scale, grad)
    layers.close(out.detach(), exact, size, layers.adapter_arithmetic(k, rank))
    layers.close(dx, parts[0], parts[1], layers.adapter_arithmetic(n, rank))
    layers.close(da, parts[2], parts[3], layers.adapter_arithmetic(n, tokens))
    layers.close(db, parts[4], parts[5], layers.adapter_arithmetic(k, tokens))


# batch, sequence, heads, kv heads, dim, rotary, interleaved, norm, fp32 weights: groups of lanes walk several tokens in
# whole runs (a few pieces or many of a token on their way), and without the vector form.
@pytest.mark.parametrize("case,dtype", [
    ((2, 8192, 14, 2, 64, 64, False, True, False), torch.bfloat16), ((1, 16385, 28, 4, 64, 32, False, True, True), torch.float16),
    ((1, 9001, 14, 2, 80, 40, True, True, False), torch.float32), ((1, 16000, 14, 3, 34, 10, False, True, True), torch.bfloat16),
    ((3, 3001, 28, 4, 128, 128, True, True, False), torch.bfloat16), ((1, 9001, 14, 2, 128, 128, False, False, False), torch.float32)])
def test_head_norm_rotary_walks_many_tokens(case, dtype):
    batch, sequence, heads, kv, dim = case[:5]
    lanes = 1
    while 16 * lanes < dim:
        lanes *= 2
    # Two blocks of 256 threads on an SM; a group takes four heads at most.
    assert batch * sequence * (-(-heads // 4) + -(-kv // 4)) > 2 * (2 * _sms() * 256 // lanes)
    q, k, table, positions, weights, interleaved = layers._rotary_inputs(case, dtype)
    leaves = [t.detach().requires_grad_() for t in (q, k, *weights) if t is not None]
    q_weight, k_weight = leaves[2:] or (None, None)
    out = head_norm_rotary(leaves[0], leaves[1], table, positions, q_weight, k_weight, 1e-6, interleaved)
    g = rng(1)
    upstream = [normal(g, *o.shape, dtype=dtype) for o in out]
    grads = torch.autograd.grad(out, leaves, upstream)
    angles = table.double()[positions][:, :, None]
    half = table.shape[1] // 2
    for i in range(2):
        exact = [t.detach().double().requires_grad_() for t in ([leaves[i]] + ([leaves[2 + i]] if len(leaves) > 2 else []))]
        weight = exact[1] if len(exact) > 1 else None
        reference, magnitude = layers.rotary64(exact[0], table, positions, weight, 1e-6, interleaved)
        layers.close(out[i].detach(), reference.detach(), magnitude.detach(), 2.0 ** -19)
        expected = torch.autograd.grad(reference, exact, upstream[i].double())
        size = upstream[i].double().abs()
        turned = layers.rotate64(size, angles[..., :half].abs(), -angles[..., half:].abs(), table.shape[1], interleaved).abs() + size
        if weight is None:
            layers.close(grads[i], expected[0], turned, 2.0 ** -19)
            continue
        x = exact[0].detach()
        r = torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)
        gw, u = turned * weight.detach().abs(), (x * r).abs()
        layers.close(grads[i], expected[0], r * (gw + u * (gw * u).mean(-1, keepdim=True)), 2.0 ** -18)
        # A weight's gradient is a sum of fp32 chains: a thread's tokens and heads, a block's groups, a strand's blocks, 32
        # strands: less than 256 additions deep.
        layers.close(grads[2 + i], expected[1], (turned * u).sum((0, 1, 2)), 2.0 ** -16)
