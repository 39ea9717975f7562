"""Uses of the layer operators that are easily lost beside the ordinary ones:
several host threads, values that are not finite beside finite ones, the ends
of a type's range, derivatives that do not exist, views under autograd, waits
that run out, and walks of many rows, tiles and tokens by one block.

Tolerances as in the operators' other tests: one rounding to the output's type
plus a power of two times the sum of the magnitudes that enter an element.
"""
import threading

import pytest
import torch

from sdc_b200.layers import AdapterBatch, head_norm_rotary, low_rank_adapters, rotary_table

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
