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

from sdc_b200.layers import AdapterBatch, low_rank_adapters

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
