"""Low-rank adapters of many requests beside a shared projection."""
from __future__ import annotations

import numpy as np
import torch

from .. import ops

_OP, _OP_IN_PLACE = ops.low_rank_adapters.default, ops.low_rank_adapters_.default

# Rows of a tile: 16 (warp-level products, a short start) or 128 (tensor
# memory, one read of the adapter's weights for all rows). Measured forward
# passes, narrow against wide: 4 adapters of 128 tokens each at 3584 -> 3584
# rank 16 15.4 against 19.4 us, of 256 21.5 against 19.4; 32 of 64 27.6 against
# 27.6, of 128 42.0 against 33.8, of 256 74.8 against 50.2; at 896 -> 4864 rank
# 64 4 of 256 23.6 against 29.7, 32 of 64 40.0 against 46.1, of 128 74.8
# against 56.3. Ranks beyond _WIDE_RANK leave no room for wide tiles beside
# the weight.
_WIDE_TILE, _NARROW_TILE, _WIDE_FROM, _WIDE_SLOTS, _WIDE_RANK = 128, 16, 96, 1536, 128


def _tiles(offsets, tokens, rows):
    """``[n, 3]`` runs {first slot, slots, adapter} of at most ``rows`` slots, the adapters' first, then those of
    the tokens without one (adapter -1), and how many have an adapter."""
    starts = np.append(offsets[:-1], offsets[-1])
    counts = np.append(np.diff(offsets), tokens - offsets[-1])
    per = -(-counts // rows)
    group = np.repeat(np.arange(len(counts)), per)
    within = np.arange(per.sum()) - np.repeat(np.cumsum(per) - per, per)
    first = starts[group] + within * rows
    slots = np.minimum(rows, starts[group] + counts[group] - first)
    adapter = np.where(group == len(counts) - 1, -1, group)
    return np.stack((first, slots, adapter), 1).astype(np.int32), int(per[:-1].sum())


class AdapterBatch:
    """Which adapter each token of a batch takes, laid out for the kernels.

    ``lengths``: tokens of each request, in the order of the batch's rows;
    ``adapters``: each request's adapter, or -1 for none (host sequences);
    ``count``: number of adapters whose weights the calls will pass. Requests
    that share an adapter share its tiles wherever they are in the batch.
    Built once for a batch on the host (one copy to ``device``, which it waits
    for; 80 us for one token, 95 for 192 requests, 200 for 16384 tokens) and
    used for every projection of every layer, forward and backward. A scheduler
    builds another when the batch's lengths or adapters change, and a captured
    graph replays the batch that it was captured with. It must stay alive until
    the work that uses it is done."""

    def __init__(self, lengths, adapters, count, device="cuda"):
        lengths = np.asarray(lengths, dtype=np.int64).reshape(-1)
        adapters = np.asarray(adapters, dtype=np.int64).reshape(-1)
        if lengths.shape != adapters.shape:
            raise ValueError("AdapterBatch needs one adapter a request")
        if count < 1 or count > 65535:
            raise ValueError("AdapterBatch takes 1 to 65535 adapters")
        if lengths.size and (lengths.min() < 0 or adapters.min() < -1 or adapters.max() >= count):
            raise ValueError("AdapterBatch lengths must not be negative and adapters must be -1 or below count")
        tokens = int(lengths.sum())
        if tokens >= 2 ** 31 - 1024:
            raise ValueError("AdapterBatch takes fewer than 2^31 - 1024 tokens")
        of_token = np.repeat(np.where(adapters < 0, count, adapters), lengths)
        offsets = np.concatenate(([0], np.cumsum(np.bincount(of_token, minlength=count + 1))))[:count + 1]
        slots = int(offsets[-1])
        used = int((np.diff(offsets) > 0).sum())
        self.tokens, self.count, self.slots = tokens, int(count), slots
        rows = np.argsort(of_token, kind="stable").astype(np.int32)
        narrow, narrow_active = _tiles(offsets, tokens, _NARROW_TILE)
        wide, wide_active = narrow[:0], 0
        if slots >= max(_WIDE_SLOTS, _WIDE_FROM * used):
            wide, wide_active = _tiles(offsets, tokens, _WIDE_TILE)
        packed = torch.from_numpy(np.concatenate((rows, offsets.astype(np.int32), narrow.reshape(-1),
                                                  wide.reshape(-1)))).to(device)
        self.rows, self.groups, narrow, wide = packed.split((tokens, count + 1, narrow.size, wide.size))
        self._narrow = (self.rows, self.groups, narrow.view(-1, 3), slots, narrow_active, _NARROW_TILE)
        self._wide = (self.rows, self.groups, wide.view(-1, 3), slots, wide_active, _WIDE_TILE)

    def arguments(self, rank):
        """The kernels' view of the batch for adapters of a rank."""
        return self._wide if self._wide[4] and rank <= _WIDE_RANK else self._narrow


def _check(x, batch):
    if not x.is_cuda:
        raise ValueError("low_rank_adapters requires CUDA tensors")
    if not isinstance(batch, AdapterBatch):
        raise ValueError("low_rank_adapters needs an AdapterBatch")


def low_rank_adapters(base, x, a, b, batch, scale=None):
    """``base + scale[g] * (x a[g]^T) b[g]^T`` with each token's adapter ``g``.

    ``base`` ``[tokens, out]``: the shared projection's output; ``x``
    ``[tokens, in]``: its input (bf16 or fp16, any row stride; a column-major
    tensor, like the FP8 projections' outputs, is copied to rows first); ``a``
    ``[count, rank, in]`` and ``b`` ``[count, out, rank]``: contiguous weights
    of the same dtype, rank up to 256 (adapters of lower rank are padded with
    zeros); ``scale`` fp32 ``[count]``, 1 when None; ``batch``: an
    ``AdapterBatch`` of the same tokens and count. Tokens without an adapter
    keep ``base``. Returns a new tensor; differentiable in ``base``, ``x``,
    ``a`` and ``b``. Adapters without tokens get zero gradients. The low-rank
    rows (and their gradients) are sums in 32 bits; the second product takes
    them as two 16-bit terms, which lose 2^-17 of a value in bf16. In fp16 they
    are scaled by a power of two first, so that the range is that of fp32, and
    lose 2^-21 of a value and 2^-39 of the largest: of the token's own row, or
    in the weights' gradients of the tokens added up."""
    _check(x, batch)
    return _OP(base, x, a, b, scale, *batch.arguments(a.shape[1]))[0]


def low_rank_adapters_(base, x, a, b, batch, scale=None):
    """``low_rank_adapters`` into ``base``: rows without an adapter are not touched."""
    _check(x, batch)
    _OP_IN_PLACE(base, x, a, b, scale, *batch.arguments(a.shape[1]))
    return base
