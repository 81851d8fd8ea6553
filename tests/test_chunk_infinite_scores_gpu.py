"""GPU tests of the chunk attention over keys whose scores are minus infinity: they count for nothing, wherever they lie."""

import numpy as np
import pytest
import torch

from chunk_cases import ChunkBatch
from helpers import to_np

pytestmark = pytest.mark.gpu


def plain(batch, first, scale=128 ** -0.5):
    """64-bit outputs of the one row without its first keys, and bounds (those of ChunkBatch.plain over the other keys)."""
    _, t, n = batch.rows[0]
    slot = int(batch.ids_host[0])
    k, v = (np.concatenate([to_np(tail[slot, :t]), to_np(new[:n])]).astype(np.float64)
            for tail, new in ((batch.tail_key, batch.key), (batch.tail_value, batch.value)))
    q = to_np(batch.query).astype(np.float64)
    k, v = k[first:], v[first:]
    seen = np.arange(len(k))[None, :] + first <= (t + np.arange(n))[:, None]
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    for h in range(batch.heads_q):
        kv = h // (batch.heads_q // batch.heads_kv)
        s = np.where(seen, scale * (q[:, h] @ k[:, kv].T), -np.inf)
        with np.errstate(invalid="ignore"):
            p = np.exp(s - s.max(1, keepdims=True))
            p /= p.sum(1, keepdims=True)
        out[:, h] = p @ v[:, kv]
        size = np.where(seen, scale * (np.abs(q[:, h]) @ np.abs(k[:, kv]).T) * 130 * 2.0 ** -24, 0.0).max(1, keepdims=True)
        bound[:, h] = 2.0 ** -8 * np.abs(out[:, h]) + (2.0 ** -8 + 2 * size + 2.0 ** -20) * (p @ np.abs(v[:, kv]))
        bound[:, h] += 2.0 ** -32 * (seen @ np.abs(v[:, kv]))
    return out, bound


@pytest.mark.parametrize("heads", [(2, 2), (8, 2)])
@pytest.mark.parametrize("row,splits", [((0, 0, 300), 1), ((0, 0, 300), 3), ((0, 128, 129), 3), ((0, 128, 9), 2), ((0, 128, 9), 1)])
def test_a_range_that_opens_with_them(cuda_device, heads, row, splits):
    """The first 64, or 128, keys of the row score -inf: half a tile, or a whole one, of nothing at the start of a chunk, or
    of a range of keys that is the tail alone.  Tokens that see a later key are the softmax over those."""
    for first in (64, 128):
        batch = ChunkBatch([row], *heads, cuda_device, seed=50 + first)
        batch.query[:, :, 0] = 1.0
        if row[1]:
            batch.tail_key[int(batch.ids_host[0]), :first, :, 0] = float("-inf")
        else:
            batch.key[:first, :, 0] = float("-inf")
        want, bound = plain(batch, first)
        sees = np.arange(row[2]) + row[1] >= first
        got = to_np(batch.attend(num_splits=splits)).astype(np.float64)
        assert (np.abs(got - want)[sees] <= bound[sees]).all()
