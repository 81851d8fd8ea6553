"""Seeded batches for the chunk operators, and their plain form in 64 bits."""

from __future__ import annotations

import numpy as np
import torch

import nvfp4_oracle as O
from helpers import interleave_vllm, scale_bytes, to_np

PAGE = 128


def blocks_of(pages: int, heads: int, fill: int, device):
    """An empty cache in the vLLM block layout, every byte ``fill``: the array and its four views."""
    from nvfp4_attn_kernel_b200.nvfp4_vllm import layout

    cache = torch.full((pages, layout.page_bytes(heads)), fill, dtype=torch.uint8, device=device)
    return cache, layout.carve(cache, heads, 128)


class ChunkBatch:
    """rows: list of (full pages, tail tokens, chunk tokens)."""

    def __init__(self, rows, heads_q, heads_kv, device, seed=0, shift=False, pad=0, query_gain=1.5, poison=True,
                 spread=False):
        from nvfp4_attn_kernel_b200.nvfp4_decode_kernel import _quantize

        g = torch.Generator().manual_seed(seed)
        self.rows, self.heads_q, self.heads_kv, self.device = rows, heads_q, heads_kv, device

        def normal(*shape):
            return torch.randn(*shape, generator=g).to(torch.bfloat16).to(device)

        full = [r[0] for r in rows]
        sealed = [(t + n) // PAGE for _, t, n in rows]
        count = sum(full) + sum(sealed)
        pages = count + 2
        order = torch.randperm(pages, generator=g).int()
        self.columns = max([1] + [f + s for f, s in zip(full, sealed)])
        # a table with a row stride of its own; entries that must not be used are out of range
        store = torch.full((len(rows), self.columns + 3), 1 << 28, dtype=torch.int32)
        at = 0
        for r, (f, s) in enumerate(zip(full, sealed)):
            store[r, :f + s] = order[at:at + f + s]
            at += f + s
        self.table_host = store[:, :self.columns].clone()
        self.table = store.to(device)[:, :self.columns]
        k_pages, v_pages = normal(pages, PAGE, heads_kv, 128), normal(pages, PAGE, heads_kv, 128)
        k_fp4, k_sf = _quantize.quantize_key_pages(k_pages)
        v_fp4, v_sf = _quantize.quantize_value_pages(v_pages)
        self.cache, *self.views = interleave_vllm(k_fp4, k_sf, v_fp4, v_sf)
        used = {int(p) for r, f in enumerate(full) for p in self.table_host[r, :f]}
        if poison:       # every other page holds NaN scales
            for p in set(range(pages)) - used:
                self.cache[p] = 255
        self.slots = len(rows) + 1
        self.tail_key, self.tail_value = normal(self.slots, PAGE, heads_kv, 128), normal(self.slots, PAGE, heads_kv, 128)
        self.ids_host = torch.randperm(self.slots, generator=g).int()[:len(rows)]
        if poison:       # nothing past a row's tail may be read
            keep = torch.zeros(self.slots, PAGE, dtype=torch.bool)
            for r, (_, t, _) in enumerate(rows):
                keep[self.ids_host[r], :t] = True
            for tail, bad in ((self.tail_key, float("inf")), (self.tail_value, float("nan"))):
                tail[~keep.to(device)] = bad
        self.ids = self.ids_host.to(device)
        n = [r[2] for r in rows]
        self.starts_host = np.concatenate([[0], np.cumsum(n)]).astype(np.int32)
        self.tokens = int(self.starts_host[-1]) + pad
        self.starts = torch.from_numpy(self.starts_host).to(device)
        self.max_chunk = max(n)
        self.seqused_fp4 = torch.tensor([f * PAGE for f in full], dtype=torch.int32, device=device)
        self.seqused_tail = torch.tensor([r[1] for r in rows], dtype=torch.int32, device=device)
        self.shift = (2 * torch.randn(heads_kv, 128, generator=g)).to(torch.bfloat16).to(device) if shift else None
        width = (heads_q + 2 * heads_kv) * 128
        if spread:       # query, key and value as slices of one projection, heads of the query apart
            fused = normal(self.tokens, width + 64)
            self.query = fused[:, :heads_q * 128].unflatten(1, (heads_q, 128))
            self.key = fused[:, heads_q * 128:(heads_q + heads_kv) * 128].unflatten(1, (heads_kv, 128))
            self.value = fused[:, (heads_q + heads_kv) * 128:width].unflatten(1, (heads_kv, 128))
        else:
            self.query = normal(self.tokens, heads_q, 128)
            self.key, self.value = normal(self.tokens, heads_kv, 128), normal(self.tokens, heads_kv, 128)
        self.query.mul_(query_gain)
        if shift:
            self.key += self.shift
        if pad and poison:
            self.query[-pad:], self.key[-pad:], self.value[-pad:] = float("nan"), float("inf"), float("nan")

    def arguments(self):
        return dict(max_chunk_len=self.max_chunk, residual_key_pages_bf16=self.tail_key,
                    residual_value_pages_bf16=self.tail_value, residual_page_ids=self.ids,
                    seqused_residual=self.seqused_tail, key_shift=self.shift)

    def attend(self, **kw):
        from nvfp4_attn_kernel_b200.nvfp4_decode_kernel import fp4_chunk_attention

        return fp4_chunk_attention(self.query, self.key, self.value, *self.views, self.table, self.seqused_fp4,
                                   self.starts, **{**self.arguments(), **kw})

    def append(self, **kw):
        from nvfp4_attn_kernel_b200.nvfp4_decode_kernel import append_kv_chunk

        return append_kv_chunk(self.key, self.value, *self.views, self.table, self.seqused_fp4, self.starts,
                               **{**self.arguments(), **kw})

    # -- 64-bit plain form -------------------------------------------------------------------

    def page_values(self):
        k_fp4, k_sf, v_fp4, v_sf = self.views
        with np.errstate(invalid="ignore"):
            k = O.dequantize_key_pages(to_np(k_fp4), scale_bytes(k_sf))
            v = O.dequantize_value_pages(to_np(v_fp4), scale_bytes(v_sf))
        return k.astype(np.float64), v.astype(np.float64)

    def history(self, row, k_pages, v_pages):
        """K and V [tokens, heads, 128] of a row's cache."""
        f, t, _ = self.rows[row]
        ids = self.table_host[row, :f].tolist()
        slot = int(self.ids_host[row])
        return (np.concatenate([k_pages[ids].reshape(-1, self.heads_kv, 128), to_np(self.tail_key[slot, :t]).astype(np.float64)]),
                np.concatenate([v_pages[ids].reshape(-1, self.heads_kv, 128), to_np(self.tail_value[slot, :t]).astype(np.float64)]))

    def plain(self, scale=128 ** -0.5):
        """Outputs, LSEs and the bounds of their errors, per row: [(o, lse, o's bound, lse's bound)].

        The bound counts the kernel's roundings to first order: the result to BF16 (2^-8 of its value); every
        probability to BF16 at worst (2^-8, so 2^-8 * sum p|v|); each score's fp32 products and sums (128 additions
        and a scaling, 130 * 2^-24 of the sum of magnitudes, the shift's product likewise), which move a
        probability and the sum it is divided by, hence twice; exp2 and the sums of a row, 2^-20 with room.
        Tiny probabilities have an absolute error too: relative to the row's largest (which is 1 before the division
        by their sum), fp16 holds numbers below 2^-14 in steps of 2^-24 and fp32's exp2 gives zero below 2^-126, so
        every probability may be off by half such a step, 2^-25, beside its relative rounding: together
        2^-25 * sum |v| / sum exp(s - max).  (Without this term a channel whose only near keys hold zeros has a
        bound far below what any fp32 softmax can give.)
        An LSE moves by the scores' error and by the rounding of its own fp32 logarithm and product."""
        k_pages, v_pages = self.page_values()
        group = self.heads_q // self.heads_kv
        q_all, k_all, v_all = (to_np(x).astype(np.float64) for x in (self.query, self.key, self.value))
        shift = 0.0 if self.shift is None else to_np(self.shift).astype(np.float64)
        results = []
        for r, (f, t, n) in enumerate(self.rows):
            a = self.starts_host[r]
            hk, hv = self.history(r, k_pages, v_pages)
            k = np.concatenate([hk, k_all[a:a + n] - shift])
            k_size = np.concatenate([np.abs(hk), np.abs(k_all[a:a + n]) + np.abs(shift)])
            v = np.concatenate([hv, v_all[a:a + n]])
            o = np.zeros((n, self.heads_q, 128))
            lse, bound, lse_bound = np.zeros((n, self.heads_q)), np.zeros_like(o), np.zeros((n, self.heads_q))
            seen = np.arange(len(k))[None, :] <= (f * PAGE + t + np.arange(n))[:, None]
            for h in range(self.heads_q):
                q, kh, vh = q_all[a:a + n, h], k[:, h // group], v[:, h // group]
                s = np.where(seen, scale * (q @ kh.T), -np.inf)
                top = s.max(1, keepdims=True)
                p = np.exp(s - top)
                total = p.sum(1, keepdims=True)
                p /= total
                o[:, h] = p @ vh
                lse[:, h] = (top + np.log(total))[:, 0]
                size = scale * (np.abs(q) @ k_size[:, h // group].T) * 130 * 2.0 ** -24
                wobble = np.where(seen, size, 0.0).max(1, keepdims=True)
                spread = p @ np.abs(vh)
                lse_bound[:, h] = wobble[:, 0] + 2.0 ** -20 * (1 + np.abs(lse[:, h]))
                bound[:, h] = 2.0 ** -8 * np.abs(o[:, h]) + (2.0 ** -8 + 2 * wobble + 2.0 ** -20) * spread
                bound[:, h] += 2.0 ** -25 * (seen @ np.abs(vh)) / total
            results.append((o, lse, bound, lse_bound))
        return results
