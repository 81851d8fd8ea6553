"""GPU tests of the chunk attention where one strong key stands before a long flat history: the many small
probabilities keep their share, also in channels where the strong key's value is zero."""

import numpy as np
import pytest
import torch

from chunk_cases import PAGE, blocks_of
from helpers import to_np

pytestmark = pytest.mark.gpu

GROUP = 4


def flat_history(device, pages, gap, chunk):
    """Row 0: a page of strong keys, then `pages` times one page of zero keys, then the chunk's zero keys; the strong keys'
    scores are `gap` (log2) above the others.  Returns the call's arguments, and outputs and bounds in 64 bits."""
    from nvfp4_attn_kernel_b200.nvfp4_decode_kernel import _quantize, dequantize_pages

    cache, views = blocks_of(3, 1, 0, device)
    key = torch.zeros(2, PAGE, 1, 128, dtype=torch.bfloat16, device=device)
    key[0] = 1.0
    value = torch.ones_like(key)
    value[0, ..., :64] = 0.0
    ids = torch.tensor([2, 0], device=device)
    for view, new in zip(views, (*_quantize.quantize_key_pages(key), *_quantize.quantize_value_pages(value))):
        view.view(torch.uint8)[ids] = new.view(torch.uint8)
    k, v = (to_np(x).astype(np.float64)[:, 0, 0] for x in dequantize_pages(*views, ids.int()))
    assert (k[1] == 0).all() and (k[0] == k[0, 0]).all() and (v[0, :64] == 0).all() and (v[1] == v[1, 0]).all()
    scale = float(np.float32(gap * np.log(2) / (128 * k[0, 0])))
    table = torch.zeros(1, pages + 1, dtype=torch.int32, device=device)
    table[0, 0] = 2
    int32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)   # noqa: E731
    bf16 = lambda h, x: torch.full((chunk, h, 128), x, dtype=torch.bfloat16, device=device)   # noqa: E731
    call = dict(query=bf16(GROUP, 1.0), key=bf16(1, 0.0), value=bf16(1, 1.0), key_pages_fp4=views[0], key_scales=views[1],
                value_pages_fp4=views[2], value_scales=views[3], fp4_page_table=table,
                seqused_fp4=int32([(pages + 1) * PAGE]), chunk_start_loc=int32([0, chunk]), max_chunk_len=chunk,
                softmax_scale=scale)
    score = scale * 128 * k[0, 0]
    small = np.exp(-score)                                   # of one flat key, relative to a strong one
    fresh = np.arange(1, chunk + 1)[:, None]
    far = pages * PAGE
    total = PAGE + (far + fresh) * small
    out = (PAGE * v[0] + far * small * v[1] + fresh * small) / total
    # Roundings: the result to BF16 (2^-8); the chunk's probabilities to BF16 (2^-8 of each), the history's to FP16 (2^-11 of
    # each, or half a step of 2^-24 where 1 stands for 2^-7 of the row's largest: 2^-32); a score's 128 products and its
    # scaling (130 * 2^-24 of its magnitude), which move a probability and the sum; exp2 and a tile's sums, 2^-20 with room.
    # A row's sum takes in 64 keys at a time, 2 (pages + 2) fp32 additions one after the other: each rounds by up to 2^-24 of
    # the sum so far, which is at most the final one, so 2 (pages + 2) 2^-24 of it in all.  (8192 pages: 9.8e-4.  Of the
    # flat keys 64 at a time are 64 * 2^-25.1 beside 128 strong ones, under half a step of the sum: lost to it, 2.3e-4.)
    adds = 2 * (pages + 2) * 2.0 ** -24
    both = 2 * 130 * 2.0 ** -24 * score + 2.0 ** -20 + adds
    bound = 2.0 ** -8 * np.abs(out) + (2.0 ** -11 + both) * (PAGE * v[0] + far * small * v[1]) / total
    bound += (2.0 ** -8 + both) * fresh * small / total + 2.0 ** -32 * (PAGE * v[0] + far * v[1]) / total
    # The product's accumulator takes in 16 keys at a time, 8 (pages + 2) additions, and what is added is cut off at its last
    # bit, not rounded: each is off by up to 2^-23 of the sum so far, which is the strong keys' part from the start and the
    # flat keys' share of it on the way, half on average.  (8192 pages: 7.8e-3 and 3.9e-3 of them at most.)
    bound += 8 * (pages + 2) * 2.0 ** -23 * (PAGE * v[0] + far * small * v[1] / 2) / total
    lse = score + np.log(total)
    return call, out, bound, lse, 130 * 2.0 ** -24 * score + 2.0 ** -20 * (1 + np.abs(lse)) + adds


@pytest.mark.parametrize("splits", [1, 3])
@pytest.mark.parametrize("chunk", [1, 40])
@pytest.mark.parametrize("pages,gap", [(1024, 25.1), (1024, 24.5), (1024, 12.3), (8192, 25.1), (8192, 21.7), (8192, 27.0)])
def test_small_probabilities_keep_their_share(cuda_device, pages, gap, chunk, splits):
    from nvfp4_attn_kernel_b200.nvfp4_decode_kernel import fp4_chunk_attention

    call, want, bound, lse_want, lse_bound = flat_history(cuda_device, pages, gap, chunk)
    lse = torch.empty(chunk, GROUP, device=cuda_device)
    got = to_np(fp4_chunk_attention(**call, num_splits=splits, lse=lse)).astype(np.float64)
    error = np.abs(got - want[:, None])
    assert (error <= bound[:, None]).all(), f"{(error / bound[:, None]).max():.2f} times the bound"
    assert (np.abs(to_np(lse) - lse_want) <= lse_bound).all()
