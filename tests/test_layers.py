"""Host side of the layer operators, without a GPU: the adapter batch's
layout and refusals, the C ABI's argument checks, the operators' schemas."""
import ctypes

import numpy as np
import pytest
import torch

import sdc_b200
from sdc_b200 import capi
from sdc_b200.layers import (AdapterBatch, distillation_loss, head_norm_rotary, low_rank_adapters, rotary_table)


@pytest.mark.parametrize("lengths,adapters,count", [
    ([], [], 1), ([0, 0], [0, -1], 2), ([1], [0], 1), ([5], [-1], 3), ([1] * 30, [i % 7 - 1 for i in range(30)], 8),
    ([100, 3, 0, 250, 64], [1, 0, 1, 1, -1], 2), ([1000, 3, 0, 2500, 64], [1, 0, 1, 1, -1], 2), ([63, 64, 65, 128], [0, 1, 2, 3], 4)])
def test_adapter_batch_lists_every_token_once_under_its_adapter(lengths, adapters, count):
    batch = AdapterBatch(lengths, adapters, count, device="cpu")
    of_token = np.repeat(np.asarray(adapters, dtype=np.int64), lengths)
    for rank in (1, 128, 129, 256):
        rows, groups, tiles, slots, active, tile_rows = batch.arguments(rank)
        rows, groups, tiles = (t.numpy() for t in (rows, groups, tiles))
        assert tile_rows == 16 or (tile_rows == 128 and rank <= 128)
        assert sorted(rows.tolist()) == list(range(len(of_token)))
        assert slots == int((of_token >= 0).sum()) == groups[-1]
        for g in range(count):
            assert rows[groups[g]:groups[g + 1]].tolist() == np.flatnonzero(of_token == g).tolist()
        seen = np.zeros(len(of_token), dtype=int)
        for i, (first, length, adapter) in enumerate(tiles):
            assert 1 <= length <= tile_rows
            assert (adapter >= 0) == (i < active)
            assert (of_token[rows[first:first + length]] == adapter).all()
            seen[first:first + length] += 1
        assert (seen == 1).all()


def test_adapter_batch_refusals():
    for args, text in ((([1, 2], [0], 1), "one adapter a request"), (([1], [1], 1), "below count"),
                       (([1], [-2], 1), "below count"), (([-1], [0], 1), "negative"), (([1], [0], 0), "65535"),
                       (([1], [0], 70000), "65535"), (([2 ** 31], [0], 1), "fewer than")):
        with pytest.raises(ValueError, match=text):
            AdapterBatch(*args, device="cpu")


def test_rotary_table_holds_cosines_then_sines():
    table = rotary_table(50, 8, 100.0, device="cpu")
    angle = np.arange(50)[:, None] * 100.0 ** (-np.arange(0, 8, 2) / 8)
    np.testing.assert_array_equal(table.numpy(), np.concatenate((np.cos(angle), np.sin(angle)), 1).astype(np.float32))
    for args in ((0, 8), (4, 7), (4, 0)):
        with pytest.raises(ValueError, match="rotary"):
            rotary_table(*args, device="cpu")


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 4, 8)
    with pytest.raises(ValueError, match="CUDA"):
        head_norm_rotary(x, x, rotary_table(4, 8, device="cpu"), torch.arange(2))
    with pytest.raises(ValueError, match="CUDA"):
        low_rank_adapters(x[0], x[0], x, x, AdapterBatch([4], [0], 2, device="cpu"))
    with pytest.raises(ValueError, match="CUDA"):
        distillation_loss(x[0], torch.zeros(4, 1, dtype=torch.int64), torch.zeros(4, 1))


def test_argument_contracts_are_checked_before_launch():
    lib = capi.lib()
    fake = 1 << 20  # never dereferenced: validation fails first
    strides = (ctypes.c_int64 * 3)(0, 64, 64)
    s = ctypes.cast(strides, ctypes.c_void_p)

    def rotary(dtype=1, batch=1, sequence=2, heads=2, dim=64, rotary=64, q_weight=None, k_weight=None, eps=1e-6,
               q=fake):
        return lib.sdc_head_norm_rotary(dtype, q, s, fake, s, batch, sequence, heads, 1, dim, fake, 8, rotary, 0, fake,
                                        1, s, q_weight, k_weight, 0, eps, fake, fake, None)

    for kwargs, text in ((dict(dtype=3), "FP16"), (dict(dim=63), "even"), (dict(dim=514), "512"),
                         (dict(rotary=66), "within the head"), (dict(rotary=0), "rotary"), (dict(q_weight=fake), "both"),
                         (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(heads=0), "needs a head"),
                         (dict(batch=2 ** 20, sequence=2 ** 20), "tokens"), (dict(q=None), "null")):
        assert rotary(**kwargs) == capi.SDC_ERR_INVALID and text in capi.last_error(), kwargs
    assert rotary(sequence=0) == capi.SDC_OK
    assert lib.sdc_head_norm_rotary_workspace_bytes(1, 0, 2, 1, 64) == 0
    assert lib.sdc_head_norm_rotary_workspace_bytes(1, 2, 2, 1, 64) > 0

    def shrink(dtype=1, tile_rows=16, rank=8, adapters=2, width=64, low=fake, tiles=1):
        return lib.sdc_adapter_shrink(dtype, fake, 64, 4, fake, fake, tiles, tile_rows, fake, adapters, rank, width, 0,
                                      None, low, 4, None)

    for kwargs, text in ((dict(dtype=0), "BF16"), (dict(tile_rows=32), "16 rows"), (dict(rank=257), "256"), (dict(rank=129, tile_rows=128), "up to 128"),
                         (dict(adapters=0), "adapters"), (dict(width=0), "positive"), (dict(low=None), "null"),
                         (dict(low=fake + 8), "aligned")):
        assert shrink(**kwargs) == capi.SDC_ERR_INVALID and text in capi.last_error(), kwargs
    assert shrink(tiles=0) == capi.SDC_OK
    assert lib.sdc_adapter_expand(1, fake, 64, 4, fake, fake, 1, 16, fake, 2, 8, 64, 1, None, 4, 0, fake, 64,
                                  None) == capi.SDC_ERR_INVALID
    assert lib.sdc_adapter_outer(1, fake, 64, 4, fake, None, 2, fake, 4, 8, 64, 0, fake, None) == capi.SDC_ERR_INVALID
    assert lib.sdc_adapter_low_bytes(10, 17) == 2 * 10 * 32 * 2 and lib.sdc_adapter_low_bytes(0, 17) == 0

    def distill(dtype=1, rows=2, vocab=100, top=4, temperature=1.0, loss=fake, stats=fake, teacher=0):
        return lib.sdc_distill_loss(dtype, fake, rows, vocab, vocab, fake, 0, top, fake, teacher, top, top, temperature,
                                    loss, stats, None)

    for kwargs, text in ((dict(dtype=5), "FP16"), (dict(teacher=5), "teacher"), (dict(vocab=0), "vocabulary"),
                         (dict(top=0), "1024"), (dict(top=1025), "1024"), (dict(temperature=0.0), "temperature"),
                         (dict(temperature=float("inf")), "temperature"), (dict(loss=None), "null"),
                         (dict(stats=fake + 4), "aligned")):
        assert distill(**kwargs) == capi.SDC_ERR_INVALID and text in capi.last_error(), kwargs
    assert distill(rows=0) == capi.SDC_OK
    rc = lib.sdc_distill_loss_and_grad(1, fake, 2, 100, 100, fake, 0, 4, fake, 0, 4, 4, 1.0, None, 0, fake, fake, fake,
                                       99, None)
    assert rc == capi.SDC_ERR_INVALID and "overlap" in capi.last_error()
    rc = lib.sdc_distill_backward(1, fake, 2, 100, 100, fake, 0, 4, fake, 0, 4, 4, 1.0, fake, fake, 2, None, fake, 100,
                                  None)
    assert rc == capi.SDC_ERR_INVALID and "upstream" in capi.last_error()
    assert lib.sdc_distill_reduce(None, None, 3, 1, fake, None) == capi.SDC_ERR_INVALID


def test_operators_are_registered():
    sdc_b200.load()
    for name in ("head_norm_rotary", "head_norm_rotary_backward", "low_rank_adapters", "low_rank_adapters_",
                 "low_rank_adapters_backward", "distillation_loss", "distill_loss", "distill_reduce", "distill_backward",
                 "distill_loss_and_grad", "distill_loss_and_grad_"):
        assert str(getattr(torch.ops.sdc_cutlass, name).default._schema).startswith(f"sdc_cutlass::{name}(")
