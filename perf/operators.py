"""Cases of the operators that continue sequences over the paged NVFP4 cache: attention of a chunk of new tokens,
the chunk's write into pages and tails, reading pages back, and the page pool (fork, release, compact).

A row's cache is ``f`` tokens in sealed NVFP4 pages (a multiple of 128), ``t`` tokens in its BF16 tail; a chunk
brings ``n`` more.  Head dimension and page size are 128.
"""

import math
import random

import torch

own = False

PAGE = 128
DIM = 128
GROUP = 16
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)

# ---------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------


def listed():
    return [
        # a step that verifies four drafted tokens for a few running sequences: latency counts
        {"name": "attend verify 4x4", "op": "attend", "rows": 4, "chunk": 4, "history": 2048, "heads_q": 32,
         "heads_kv": 8, "ragged": True, "shift": True, "pad": 0},
        # one long prompt continued by a chunk after the pages of its earlier chunks
        {"name": "attend 1x512 after 16k", "op": "attend", "rows": 1, "chunk": 512, "history": 16384, "heads_q": 32,
         "heads_kv": 8, "ragged": False, "shift": False, "pad": 0},
        # a mixed batch: fresh prompts, continued ones and an empty row; five heads to a KV head; padded tokens
        {"name": "attend ragged 7x777", "op": "attend", "rows": 7, "chunk": 777, "history": 5000, "heads_q": 40,
         "heads_kv": 8, "ragged": True, "shift": True, "pad": 5},
        # the largest: two sequences, chunks of 2048 tokens at 32k of context
        {"name": "attend 2x2048 after 32k", "op": "attend", "rows": 2, "chunk": 2048, "history": 32768, "heads_q": 32,
         "heads_kv": 8, "ragged": False, "shift": False, "pad": 0},
        # the verification step's accepted tokens enter the cache
        {"name": "append 4x5", "op": "append", "rows": 4, "chunk": 5, "history": 700, "heads_kv": 8, "ragged": True,
         "shift": True},
        # chunks of a prefill step enter the cache, most of them as sealed pages
        {"name": "append 8x2048", "op": "append", "rows": 8, "chunk": 2048, "history": 1000, "heads_kv": 8,
         "ragged": True, "shift": True},
        # a short prefix read back for a caller that keeps BF16
        {"name": "dequantize 6 pages", "op": "dequantize", "pages": 6, "heads_kv": 2},
        # a 32k prefix read back
        {"name": "dequantize 256 pages", "op": "dequantize", "pages": 256, "heads_kv": 8},
        # one sequence forked into three continuations on a GPU's KV-head shard
        {"name": "fork 3 of 1 kv head", "op": "fork", "layers": 4, "slots": 8, "forks": 3, "columns": 32,
         "heads_kv": 1},
        # a step of a wide search: finished continuations released, better ones forked in their place
        {"name": "fork 40 x 32 layers", "op": "fork", "layers": 32, "slots": 64, "forks": 40, "columns": 256,
         "heads_kv": 8},
        # a small pool after some releases
        {"name": "compact 300 pages", "op": "compact", "layers": 1, "pages": 300, "rows": 9, "heads_kv": 1,
         "live": 0.6},
        # a pool of several layers, a third of it free, packed together
        {"name": "compact 1500 x 8 layers", "op": "compact", "layers": 8, "pages": 1500, "rows": 24, "heads_kv": 8,
         "live": 0.66},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "append", "dequantize", "fork", "compact"])
    if op == "attend":
        heads_kv = rng.choice([1, 2, 4, 8])
        heads_q = heads_kv * rng.choice([1, 2, 3, 4, 4, 5, 6, 7, 8, 16])
        case = {"op": op, "rows": _log(rng, 1, 24), "chunk": _log(rng, 1, 2048), "history": _log(rng, 1, 32768) - 1,
                "heads_q": heads_q, "heads_kv": heads_kv, "ragged": rng.random() < 0.7, "shift": rng.random() < 0.5,
                "pad": rng.choice([0, 0, 1, 9])}
        largest = 2 * 32 * 2048 * (32768 + 2048)
        while case["rows"] * case["heads_q"] * case["chunk"] * (case["history"] + case["chunk"] + 256) > largest:
            if case["rows"] > 1:
                case["rows"] -= (case["rows"] + 3) // 4
            else:
                case["chunk"] = max(1, case["chunk"] // 2)
        return case
    if op == "append":
        return {"op": op, "rows": _log(rng, 1, 16), "chunk": _log(rng, 1, 2048), "history": _log(rng, 1, 8192) - 1,
                "heads_kv": rng.choice([1, 2, 4, 8]), "ragged": rng.random() < 0.7, "shift": rng.random() < 0.5}
    if op == "dequantize":
        return {"op": op, "pages": _log(rng, 1, 256), "heads_kv": rng.choice([1, 2, 4, 8])}
    if op == "fork":
        slots = rng.randint(4, 64)
        return {"op": op, "layers": rng.randint(1, 32), "slots": slots, "forks": rng.randint(1, slots * 5 // 8),
                "columns": _log(rng, 2, 256), "heads_kv": rng.choice([1, 2, 4, 8])}
    return {"op": op, "layers": rng.randint(1, 8), "pages": _log(rng, 40, 1500), "rows": _log(rng, 2, 24),
            "heads_kv": rng.choice([1, 2, 4, 8]), "live": round(rng.uniform(0.2, 0.95), 2)}


def _lengths(case):
    """History and chunk length of every row, from the case alone."""
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    history, chunk = [], []
    for r in range(case["rows"]):
        if not case["ragged"]:
            history.append(case["history"])
            chunk.append(case["chunk"])
            continue
        history.append(rng.choice([0, case["history"], rng.randint(0, case["history"]), rng.randint(0, case["history"])]))
        chunk.append(rng.choice([case["chunk"], rng.randint(1, case["chunk"]), rng.randint(1, case["chunk"])]))
    if case["ragged"]:
        history[0], chunk[0] = case["history"], case["chunk"]
        if case["rows"] > 4:
            chunk[3] = 0
    return history, chunk


def _tail_of(tokens, r):
    """Tail length of a history: its last partial page, or now and then a full page not yet sealed."""
    t = tokens % PAGE
    return PAGE if t == 0 and tokens > 0 and r % 2 else t


def work(case):
    if case["op"] == "attend":
        history, chunk = _lengths(case)
        hq, hkv = case["heads_q"], case["heads_kv"]
        nbytes = flops = 0
        for r, (h, n) in enumerate(zip(history, chunk)):
            t = _tail_of(h, r)
            if n:
                nbytes += (h - t) * hkv * 144 + t * hkv * 512 + n * hkv * 512 + 2 * n * hq * 256
                flops += 4 * DIM * hq * (n * h + n * (n + 1) // 2)
        return {"bytes": nbytes, "flops": flops}
    if case["op"] == "append":
        history, chunk = _lengths(case)
        hkv, nbytes = case["heads_kv"], 0
        for r, (h, n) in enumerate(zip(history, chunk)):
            t = _tail_of(h, r)
            sealed, rest = (t + n) // PAGE, (t + n) % PAGE
            # the chunk, the tail that joins its first page, sealed pages out and back in, the tail out, the pages' values
            nbytes += n * hkv * 512
            if sealed:
                nbytes += t * hkv * 512 + sealed * PAGE * hkv * (2 * 144 + 512) + rest * hkv * 512
            else:
                nbytes += n * hkv * 512
        return {"bytes": nbytes, "flops": 0}
    if case["op"] == "dequantize":
        return {"bytes": case["pages"] * PAGE * case["heads_kv"] * (144 + 512), "flops": 0}
    if case["op"] == "fork":
        pairs, lengths, held = _fork_plan(case)
        copied = sum(lengths[s] % PAGE for s, _ in pairs)
        shared = sum(lengths[s] // PAGE for s, _ in pairs)
        # tails of K and V in every layer, read and written; table entries read and written, counts up and down
        return {"bytes": copied * case["layers"] * case["heads_kv"] * 2 * 2 * 256 + shared * (8 + 16), "flops": 0}
    live, moves = _compact_plan(case)
    block = 2 * PAGE * case["heads_kv"] * 72
    return {"bytes": 2 * moves * block * case["layers"] + 8 * case["pages"] + 8 * live, "flops": 0}


# ---------------------------------------------------------------------------------------------
# the cache's format, in elementary operations
# ---------------------------------------------------------------------------------------------


def _scale_places(device):
    """Byte of (row, 16-element group) inside a 1024-byte scale block: [128, 8]."""
    row = torch.arange(PAGE, device=device)[:, None]
    g = torch.arange(8, device=device)[None, :]
    return (g // 4) * 512 + (row % 32) * 16 + (row // 32) * 4 + g % 4


def _quantize(x):
    """x [..., 128 rows, 128 elements] in fp32 -> packed bytes [..., 128, 64], scale bytes [..., 128, 8]."""
    blocks = x.unflatten(-1, (8, GROUP))
    scale = (blocks.abs().amax(-1) * torch.tensor(1.0 / 6.0, dtype=torch.float32, device=x.device)).clamp(max=448.0)
    scale = scale.to(torch.float8_e4m3fn)
    inverse = 1.0 / (scale.float() + 1e-30)
    y = blocks * inverse[..., None]
    mag = y.abs()
    mids = ((0.25, False), (0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False))
    code = sum((mag >= m if up else mag > m).to(torch.uint8) for m, up in mids)      # a tie goes to the even code
    code = code + (y < 0).to(torch.uint8) * 8
    code = code.flatten(-2)
    return code[..., 0::2] + code[..., 1::2] * 16, scale.view(torch.uint8)


def _scatter_scales(scales):
    """[..., 128, 8] scale bytes -> [..., 1024] in the block's order."""
    out = torch.empty(*scales.shape[:-2], 1024, dtype=torch.uint8, device=scales.device)
    out[..., _scale_places(scales.device).flatten()] = scales.flatten(-2)
    return out


def _values(packed, scale_block):
    """Packed bytes [..., 128, 64] and scale blocks [..., 1024] -> fp32 [..., 128, 128]."""
    levels = torch.tensor(LEVELS + tuple(-v for v in LEVELS), dtype=torch.float32, device=packed.device)
    codes = torch.stack((packed & 15, packed >> 4), -1).flatten(-2)
    scales = scale_block[..., _scale_places(packed.device).flatten()].view(torch.float8_e4m3fn).float()
    scales = scales.unflatten(-1, (PAGE, 8))
    return (levels[codes.int()].unflatten(-1, (8, GROUP)) * scales[..., None]).flatten(-2)


def _regions(blocks, heads):
    """One layer's block array [pages, bytes] as K packed [p, 128, h, 64], K scales [p, h, 1024], V packed
    [p, h, 128, 64], V scales [p, h, 1024]."""
    a, b = PAGE * heads * 64, heads * 1024
    return (blocks[:, :a].unflatten(1, (PAGE, heads, 64)), blocks[:, a:a + b].unflatten(1, (heads, 1024)),
            blocks[:, a + b:2 * a + b].unflatten(1, (heads, PAGE, 64)),
            blocks[:, 2 * a + b:].unflatten(1, (heads, 1024)))


def _page_values(blocks, heads, ids):
    """K and V of the pages ``ids`` in fp32: [n, 128 tokens, heads, 128] each."""
    kp, ks, vp, vs = (x[ids] for x in _regions(blocks, heads))
    return (_values(kp.transpose(1, 2), ks).transpose(1, 2), _values(vp, vs).permute(0, 3, 1, 2))


def _store_pages(blocks, heads, ids, key, value):
    """Quantise fp32 pages [n, 128, heads, 128] into the blocks ``ids``."""
    kp, ks, vp, vs = _regions(blocks, heads)
    packed, scales = _quantize(key.transpose(1, 2))
    kp[ids], ks[ids] = packed.transpose(1, 2), _scatter_scales(scales)
    packed, scales = _quantize(value.permute(0, 2, 3, 1))
    vp[ids], vs[ids] = packed, _scatter_scales(scales)


def _views(blocks, heads):
    """The same regions in the shapes the framework's operators take."""
    pages, pitch = blocks.shape
    flat, a, b = blocks.view(-1), PAGE * heads * 64, heads * 1024

    def scales(offset):
        return flat.as_strided((pages, 32, 4, 1, 4, 2, heads), (pitch, 16, 4, 1024, 1, 512, 1024),
                               offset).view(torch.float8_e4m3fn)

    return (flat.as_strided((pages, PAGE, heads, 64), (pitch, heads * 64, 64, 1), 0), scales(a),
            flat.as_strided((pages, heads, DIM, 64), (pitch, DIM * 64, 64, 1), a + b), scales(2 * a + b))


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(shape, gen, mean=None):
    x = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)
    return (x if mean is None else x + mean).to(torch.bfloat16)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _fill_pages(blocks, heads, ids, gen, key_mean):
    for part in ids.split(64):
        _store_pages(blocks, heads, part,
                     torch.randn(len(part), PAGE, heads, DIM, generator=gen, device="cuda") + key_mean,
                     torch.randn(len(part), PAGE, heads, DIM, generator=gen, device="cuda"))


def _prepare_rows(case, seed):
    """Cache, tails and chunk of a batch (attend, append)."""
    gen = _generator(seed)
    heads = case["heads_kv"]
    history, chunk = _lengths(case)
    tails = [_tail_of(h, r) for r, h in enumerate(history)]
    full = [(h - t) // PAGE for h, t in zip(history, tails)]
    spare = [(t + n) // PAGE for t, n in zip(tails, chunk)]
    columns = max(1, max(f + s for f, s in zip(full, spare)))
    pages = sum(full) + sum(spare) + 3
    order = torch.randperm(pages, generator=gen, device="cuda").int()
    table = torch.full((case["rows"], columns), -1, dtype=torch.int32, device="cuda")
    at = 0
    for r in range(case["rows"]):
        count = full[r] + spare[r]
        table[r, :count] = order[at:at + count]
        at += count
    blocks = torch.full((pages, 2 * PAGE * heads * 72), 255, dtype=torch.uint8, device="cuda")
    used = torch.cat([table[r, :full[r]] for r in range(case["rows"])]).long()
    _fill_pages(blocks, heads, used, gen, 0.0)
    slots = case["rows"] + 1
    mean = 2.0 * torch.randn(heads, DIM, generator=gen, device="cuda")
    shift = mean.to(torch.bfloat16) if case["shift"] else None
    tokens = sum(chunk) + case.get("pad", 0)
    ids = torch.randperm(slots, generator=gen, device="cuda")[:case["rows"]].int()
    state = {"op": case["op"], "heads": heads, "blocks": blocks, "views": _views(blocks, heads), "table": table,
             "seqused_fp4": _ints([f * PAGE for f in full]), "seqused_tail": _ints(tails), "tail_ids": ids,
             "tail_key": _normal((slots, PAGE, heads, DIM), gen), "tail_value": _normal((slots, PAGE, heads, DIM), gen),
             "starts": _ints([sum(chunk[:r]) for r in range(case["rows"] + 1)]), "max_chunk": case["chunk"],
             "key": _normal((tokens, heads, DIM), gen, mean if case["shift"] else None),
             "value": _normal((tokens, heads, DIM), gen), "shift": shift, "tokens": sum(chunk),
             "columns": columns, "first_new": [f for f in full], "sealed": spare}
    if case["op"] == "attend":
        # queries that prefer some keys to others, as a trained model's do
        state["query"] = (1.5 * torch.randn(tokens, case["heads_q"], DIM, generator=gen, device="cuda")).to(torch.bfloat16)
        state["out"] = torch.full((tokens, case["heads_q"], DIM), 0.0625, dtype=torch.bfloat16, device="cuda")
    else:
        written = [table[r, full[r]:full[r] + spare[r]] for r in range(case["rows"])]
        state["written"] = torch.cat(written)
    return state


def _fork_plan(case):
    """Pairs (source row, destination row), cached length of every row, page-table entries held."""
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    rows = list(range(case["slots"]))
    rng.shuffle(rows)
    targets, sources = rows[:case["forks"]], rows[case["forks"]:]
    pairs = [(rng.choice(sources), d) for d in targets]
    lengths = [rng.randint(1, case["columns"] * PAGE - 1) for _ in rows]
    return pairs, lengths, [n // PAGE for n in lengths]


def _prepare_fork(case, seed):
    gen = _generator(seed)
    pairs, lengths, held = _fork_plan(case)
    order = torch.randperm(len(pairs), generator=gen, device="cuda").tolist()
    pairs = [pairs[i] for i in order]
    pages = sum(held) + 1
    ids = torch.randperm(pages, generator=gen, device="cuda").int()
    table = torch.full((case["slots"], case["columns"]), -1, dtype=torch.int32, device="cuda")
    refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    at = 0
    for r, n in enumerate(held):
        table[r, :n] = ids[at:at + n]
        refs[ids[at:at + n].long()] = 1
        at += n
    shape = (case["layers"], case["slots"], PAGE, case["heads_kv"], DIM)
    # forking shares pages and touches none of their bytes: one layer's block array stands for all
    blocks = [torch.zeros(pages, 2 * PAGE * case["heads_kv"] * 72, dtype=torch.uint8, device="cuda")]
    state = {"op": "fork", "table": table, "held": _ints(held), "refs": refs, "seqused_fp4": _ints([n * PAGE for n in held]),
             "seqused_tail": _ints([n % PAGE for n in lengths]),
             "slots": torch.randperm(case["slots"], generator=gen, device="cuda").int(),
             "tail_key": _normal(shape, gen), "tail_value": _normal(shape, gen),
             "source": _ints([s for s, _ in pairs]), "target": _ints([d for _, d in pairs]), "pool": None}
    if own:
        from nvfp4_attn_kernel_b200.nvfp4_vllm.pages import PagePool

        state["pool"] = PagePool(blocks, refs=refs, tail_key=state["tail_key"], tail_value=state["tail_value"])
    return state


def _compact_plan(case):
    """Live pages, and how many of them lie at or above their count (the ones that move)."""
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    live = max(1, int(case["pages"] * case["live"]))
    chosen = rng.sample(range(case["pages"]), live)
    return live, sum(p >= live for p in chosen)


def _prepare_compact(case, seed):
    gen = _generator(seed)
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    live = max(1, int(case["pages"] * case["live"]))
    chosen = rng.sample(range(case["pages"]), live)
    chosen = [chosen[i] for i in torch.randperm(live, generator=gen, device="cuda").tolist()]
    rows = min(case["rows"], live)
    cuts = [live * r // rows for r in range(rows + 1)]
    held = [cuts[r + 1] - cuts[r] for r in range(rows)]
    shared = min(held[0], 3) if rows > 1 else 0       # every other row starts with a few pages of the first
    columns = max(held) + shared
    table = torch.full((rows, columns), -1, dtype=torch.int32, device="cuda")
    refs = torch.zeros(case["pages"], dtype=torch.int32, device="cuda")
    for r in range(rows):
        mine = chosen[cuts[r]:cuts[r + 1]]
        if r % 2:
            mine = chosen[:shared] + mine
            held[r] += shared
        table[r, :len(mine)] = _ints(mine)
        refs[_ints(mine).long()] += 1
    block = 2 * PAGE * case["heads_kv"] * 72
    blocks = [torch.randint(0, 256, (case["pages"], block), generator=gen, device="cuda", dtype=torch.uint8)
              for _ in range(case["layers"])]
    state = {"op": "compact", "table": table, "held": _ints(held), "refs": refs, "blocks": blocks, "live": live,
             "pool": None}
    if own:
        from nvfp4_attn_kernel_b200.nvfp4_vllm.pages import PagePool

        state["pool"] = PagePool(blocks, refs=refs.clone())
    return state


def prepare(case, seed):
    if case["op"] in ("attend", "append"):
        return _prepare_rows(case, seed)
    if case["op"] == "dequantize":
        gen = _generator(seed)
        heads, pages = case["heads_kv"], case["pages"] + case["pages"] // 8 + 1
        blocks = torch.full((pages, 2 * PAGE * heads * 72), 255, dtype=torch.uint8, device="cuda")
        ids = torch.randperm(pages, generator=gen, device="cuda")[:case["pages"]]
        _fill_pages(blocks, heads, ids, gen, 0.0)
        return {"op": "dequantize", "heads": heads, "blocks": blocks, "views": _views(blocks, heads), "ids": ids.int()}
    return _prepare_fork(case, seed) if case["op"] == "fork" else _prepare_compact(case, seed)


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------


def _attend_plain(s):
    heads, device = s["heads"], "cuda"
    rows, columns = s["table"].shape
    group = s["query"].shape[1] // heads
    longest = s["max_chunk"]
    place = torch.arange(longest, device=device)
    length = s["starts"][1:] - s["starts"][:-1]
    token = (s["starts"][:-1, None] + place).clamp(max=max(0, len(s["key"]) - 1)).long()
    fresh = place < length[:, None]
    ids = s["table"].clamp(min=0).long()
    inside = torch.arange(columns, device=device) < (s["seqused_fp4"] // PAGE)[:, None]
    key, value = (x.reshape(rows, columns * PAGE, heads, DIM) for x in _page_values(s["blocks"], heads, ids.flatten()))
    inside = inside.repeat_interleave(PAGE, 1)
    tail = s["tail_ids"].long()
    in_tail = torch.arange(PAGE, device=device) < s["seqused_tail"][:, None]
    new_key = s["key"].float() - (s["shift"].float() if s["shift"] is not None else 0.0)
    keys = torch.cat((key, s["tail_key"][tail].float(), new_key[token]), 1)
    values = torch.cat((value, s["tail_value"][tail].float(), s["value"].float()[token]), 1)
    # [rows, 1, positions] of the past and [rows, chunk, chunk] of the chunk itself
    past = torch.cat((inside, in_tail), 1)[:, None, :].expand(-1, longest, -1)
    now = fresh[:, None, :] & (place[None, None, :] <= place[None, :, None])
    seen = torch.cat((past, now), 2)
    values = torch.where(seen.any(1)[:, :, None, None], values, 0.0)     # unwritten pages may hold anything
    keys = torch.where(seen.any(1)[:, :, None, None], keys, 0.0)
    q = s["query"].float()[token].view(rows, longest, heads, group, DIM).permute(0, 2, 3, 1, 4)
    scores = q.reshape(rows, heads, group * longest, DIM) @ keys.permute(0, 2, 3, 1)
    scores = scores.view(rows, heads, group, longest, -1).mul_(DIM ** -0.5)
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=-1e30)
    scores.sub_(top).exp_()
    total = scores.sum(-1, keepdim=True).clamp(min=1e-30)
    result = scores.view(rows, heads, group * longest, -1) @ values.permute(0, 2, 1, 3)
    result = result.view(rows, heads, group, longest, DIM) / total
    result = result.permute(0, 3, 1, 2, 4).reshape(rows, longest, heads * group, DIM).to(torch.bfloat16)
    s["out"][token[fresh]] = result[fresh]
    return s["out"]


def _append_plain(s):
    heads = s["heads"]
    key, value = s["key"].float(), s["value"].float()
    if s["shift"] is not None:
        key = (key - s["shift"].float()).to(torch.bfloat16).float()
    rows, columns = s["table"].shape
    width = (s["max_chunk"] + 2 * PAGE) // PAGE
    length = s["starts"][1:] - s["starts"][:-1]
    tail, slot = s["seqused_tail"], s["tail_ids"].long()
    place = torch.arange(width * PAGE, device="cuda")
    token = (s["starts"][:-1, None] + place - tail[:, None]).clamp(0, len(key) - 1).long()
    old = place < tail[:, None]
    beside = place.clamp(max=PAGE - 1)
    stream_key = torch.where(old[:, :, None, None], s["tail_key"][slot][:, beside].float(), key[token])
    stream_value = torch.where(old[:, :, None, None], s["tail_value"][slot][:, beside].float(), value[token])
    total = tail + length
    sealed, rest = total // PAGE, total % PAGE
    column = torch.arange(width, device="cuda")
    take = column < sealed[:, None]
    target = ((s["seqused_fp4"] // PAGE)[:, None] + column).clamp(max=columns - 1).long()
    pages = torch.gather(s["table"], 1, target)[take].long()
    _store_pages(s["blocks"], heads, pages, stream_key.view(rows, width, PAGE, heads, DIM)[take],
                 stream_value.view(rows, width, PAGE, heads, DIM)[take])
    left = (sealed[:, None] * PAGE + torch.arange(PAGE, device="cuda")).clamp(max=width * PAGE - 1)
    keep = torch.arange(PAGE, device="cuda") < rest[:, None]
    row = torch.arange(rows, device="cuda")[:, None].expand(-1, PAGE)
    where = (slot[:, None].expand(-1, PAGE)[keep], torch.arange(PAGE, device="cuda").expand(rows, -1)[keep])
    s["tail_key"][where] = stream_key[row[keep], left[keep]].to(torch.bfloat16)
    s["tail_value"][where] = stream_value[row[keep], left[keep]].to(torch.bfloat16)
    return (s["seqused_fp4"] + sealed * PAGE).int(), rest.int()


def _fork_plain(s):
    """Release the destination rows, then make each a fork of its source."""
    table, refs = s["table"], s["refs"]
    column = torch.arange(table.shape[1], device="cuda")
    target, source = s["target"].long(), s["source"].long()
    gone = table[target][column < s["held"][target][:, None]].long()
    refs.scatter_add_(0, gone, torch.full_like(gone, -1, dtype=torch.int32))
    full = s["seqused_fp4"][source] // PAGE
    shared = column < full[:, None]
    table[target] = torch.where(shared, table[source], table[target])
    taken = table[source][shared].long()
    refs.scatter_add_(0, taken, torch.ones_like(taken, dtype=torch.int32))
    s["held"][target] = full
    s["seqused_fp4"][target] = s["seqused_fp4"][source]
    length = s["seqused_tail"][source]
    s["seqused_tail"][target] = length
    pair, place = (torch.arange(PAGE, device="cuda") < length[:, None]).nonzero(as_tuple=True)
    to, of = s["slots"][target[pair]].long(), s["slots"][source[pair]].long()
    s["tail_key"][:, to, place] = s["tail_key"][:, of, place]
    s["tail_value"][:, to, place] = s["tail_value"][:, of, place]


def _compact_plain(s, table, refs):
    live = refs > 0
    count = live.sum()
    index = torch.arange(len(refs), device="cuda")
    holes = (~live & (index < count)).nonzero()[:, 0]
    movers = (live & (index >= count)).nonzero()[:, 0]
    new = index.clone()
    new[movers] = holes
    for blocks in s["blocks"]:
        blocks[holes] = blocks[movers]
    refs[holes] = refs[movers]
    refs[movers] = 0
    used = torch.arange(table.shape[1], device="cuda") < s["held"][:, None]
    table[used] = new[table[used].long()].int()
    return count.int()


def run(s):
    if s["op"] == "attend":
        if not own:
            return {"out": _attend_plain(s)}
        from nvfp4_attn_kernel_b200.nvfp4_decode_kernel import fp4_chunk_attention

        return {"out": fp4_chunk_attention(
            s["query"], s["key"], s["value"], *s["views"], s["table"], s["seqused_fp4"], s["starts"],
            max_chunk_len=s["max_chunk"], residual_key_pages_bf16=s["tail_key"],
            residual_value_pages_bf16=s["tail_value"], residual_page_ids=s["tail_ids"],
            seqused_residual=s["seqused_tail"], key_shift=s["shift"], out=s["out"], trusted_metadata=True)}
    if s["op"] == "append":
        if own:
            from nvfp4_attn_kernel_b200.nvfp4_decode_kernel import append_kv_chunk, dequantize_pages

            full, rest = append_kv_chunk(
                s["key"], s["value"], *s["views"], s["table"], s["seqused_fp4"], s["starts"],
                max_chunk_len=s["max_chunk"], residual_key_pages_bf16=s["tail_key"],
                residual_value_pages_bf16=s["tail_value"], residual_page_ids=s["tail_ids"],
                seqused_residual=s["seqused_tail"], key_shift=s["shift"], trusted_metadata=True)
            key, value = dequantize_pages(*s["views"], s["written"])
        else:
            full, rest = _append_plain(s)
            key, value = (x.to(torch.bfloat16) for x in _page_values(s["blocks"], s["heads"], s["written"].long()))
        return {"key": key, "value": value, "tail_key": s["tail_key"], "tail_value": s["tail_value"], "seqused_fp4": full,
                "seqused_tail": rest}
    if s["op"] == "dequantize":
        if own:
            from nvfp4_attn_kernel_b200.nvfp4_decode_kernel import dequantize_pages

            key, value = dequantize_pages(*s["views"], s["ids"])
        else:
            key, value = (x.to(torch.bfloat16).contiguous()
                          for x in _page_values(s["blocks"], s["heads"], s["ids"].long()))
        return {"key": key, "value": value}
    if s["op"] == "fork":
        if own:
            s["pool"].release(s["target"], s["table"], s["held"])
            s["pool"].fork(s["source"], s["target"], s["table"], s["held"], s["seqused_fp4"], s["seqused_tail"],
                           s["slots"])
        else:
            _fork_plain(s)
        return {k: s[k] for k in ("table", "held", "refs", "seqused_fp4", "seqused_tail", "tail_key", "tail_value")}
    table = s["table"].clone()
    if own:
        s["pool"].refs.copy_(s["refs"])
        count = s["pool"].compact(table, s["held"])
        refs = s["pool"].refs
    else:
        refs = s["refs"].clone()
        count = _compact_plain(s, table, refs)
    return {"table": table, "refs": refs, "blocks": s["blocks"], "count": count.reshape(())}


# ---------------------------------------------------------------------------------------------
# from the definitions, in 64 bits
# ---------------------------------------------------------------------------------------------


def _exact_page(blocks, heads, page):
    """K and V [128 tokens, heads, 128] of one page, value = e2m1 * e4m3, byte by byte of the format."""
    raw = blocks[page]
    table = torch.tensor(LEVELS, dtype=torch.float64, device=raw.device)

    def number(code):
        return torch.where(code >= 8, -table[(code & 7).long()], table[(code & 7).long()])

    def scale(byte):
        exponent, fraction = (byte >> 3) & 15, byte & 7
        return torch.where(exponent == 0, fraction.double() * 2.0 ** -9,
                           (8 + fraction).double() * torch.exp2(exponent.double() - 10))

    bytes_k, bytes_s = PAGE * heads * 64, heads * 1024
    row, group = torch.arange(128, device=raw.device)[:, None], torch.arange(8, device=raw.device)[None, :]
    atom = (group // 4) * 512 + (row % 32) * 16 + (row // 32) * 4 + group % 4
    key, value = [], []
    for h in range(heads):
        k = raw[:bytes_k].view(PAGE, heads, 64)[:, h].int()
        s = raw[bytes_k + h * 1024 + atom].int()
        x = torch.stack((number(k & 15), number(k >> 4)), 2).view(128, 8, 16) * scale(s)[:, :, None]
        key.append(x.view(128, 128))
        v = raw[bytes_k + bytes_s:][h * 8192:(h + 1) * 8192].view(128, 64).int()
        s = raw[2 * bytes_k + bytes_s + h * 1024 + atom].int()
        x = torch.stack((number(v & 15), number(v >> 4)), 2).view(128, 8, 16) * scale(s)[:, :, None]
        value.append(x.view(128, 128).T)
    return torch.stack(key, 1), torch.stack(value, 1)


def _exact_attend(s):
    heads, out = s["heads"], s["out"].double()
    starts, full, tails = s["starts"].tolist(), s["seqused_fp4"].tolist(), s["seqused_tail"].tolist()
    group = s["query"].shape[1] // heads
    for r in range(len(full)):
        first, n = starts[r], starts[r + 1] - starts[r]
        if not n:
            continue
        pages = [_exact_page(s["blocks"], heads, int(p)) for p in s["table"][r, :full[r] // PAGE].tolist()]
        slot = int(s["tail_ids"][r])
        new = s["key"][first:first + n].double()
        if s["shift"] is not None:
            new = new - s["shift"].double()
        keys = torch.cat([k for k, _ in pages] + [s["tail_key"][slot, :tails[r]].double(), new])
        values = torch.cat([v for _, v in pages] + [s["tail_value"][slot, :tails[r]].double(),
                                                    s["value"][first:first + n].double()])
        position = torch.arange(len(keys), device="cuda")
        limit = full[r] + tails[r] + torch.arange(n, device="cuda")
        for h in range(heads):
            for q in range(h * group, (h + 1) * group):
                score = s["query"][first:first + n, q].double() @ keys[:, h].T / math.sqrt(DIM)
                score[position[None, :] > limit[:, None]] = -math.inf
                out[first:first + n, q] = torch.softmax(score, 1) @ values[:, h]
    return {"out": out}


def _exact_quantized(x):
    """What x [rows, 128] (groups of 16 along the last axis) becomes in the cache.  The scale is the largest magnitude
    over six in E4M3; the format fixes that elements are multiplied by the scale's reciprocal rounded to fp32."""
    g = x.view(-1, 8, 16)
    scale = (g.abs().amax(-1, keepdim=True) / 6).clamp(max=448).float().to(torch.float8_e4m3fn).double()
    reciprocal = (1 / (scale + 1e-30)).float().double()
    y = (g * reciprocal).float().double()
    grid = torch.tensor(LEVELS, dtype=torch.float64, device=x.device)
    distance = (y.abs()[..., None] - grid).abs()
    near = distance.amin(-1, keepdim=True)
    even = torch.tensor([0.0, 1.0] * 4, dtype=torch.float64, device=x.device)
    pick = torch.where(distance == near, even, 9.0).argmin(-1)           # of two equally near ones the even code
    return (grid[pick] * y.sign() * scale).view(-1, 128)


def _exact_append(s):
    heads = s["heads"]
    starts, full, tails = s["starts"].tolist(), s["seqused_fp4"].tolist(), s["seqused_tail"].tolist()
    tail_key, tail_value = s["tail_key"].double(), s["tail_value"].double()
    pages_key, pages_value, after_full, after_tail = [], [], [], []
    for r in range(len(full)):
        slot, first, last = int(s["tail_ids"][r]), starts[r], starts[r + 1]
        key, value = s["key"][first:last].double(), s["value"][first:last].double()
        if s["shift"] is not None:
            key = (key - s["shift"].double()).to(torch.bfloat16).double()
        key = torch.cat((tail_key[slot, :tails[r]], key))
        value = torch.cat((tail_value[slot, :tails[r]], value))
        sealed = len(key) // PAGE
        for p in range(sealed):
            k = key[p * PAGE:(p + 1) * PAGE].reshape(-1, DIM)
            pages_key.append(_exact_quantized(k).view(PAGE, heads, DIM))
            v = value[p * PAGE:(p + 1) * PAGE].permute(1, 2, 0).reshape(-1, PAGE)
            pages_value.append(_exact_quantized(v).view(heads, DIM, PAGE).permute(2, 0, 1))
        rest = len(key) - sealed * PAGE
        tail_key[slot, :rest], tail_value[slot, :rest] = key[sealed * PAGE:], value[sealed * PAGE:]
        after_full.append(full[r] + sealed * PAGE)
        after_tail.append(rest)
    empty = torch.zeros(0, PAGE, heads, DIM, dtype=torch.float64, device="cuda")
    return {"key": torch.stack(pages_key) if pages_key else empty,
            "value": torch.stack(pages_value) if pages_value else empty, "tail_key": tail_key, "tail_value": tail_value,
            "seqused_fp4": _ints(after_full), "seqused_tail": _ints(after_tail)}


def _exact_fork(s):
    refs, table, held = s["refs"].tolist(), s["table"].tolist(), s["held"].tolist()
    full, tails, slots = s["seqused_fp4"].tolist(), s["seqused_tail"].tolist(), s["slots"].tolist()
    for d in s["target"].tolist():
        for p in table[d][:held[d]]:
            refs[p] -= 1
        held[d] = 0
    for src, d in zip(s["source"].tolist(), s["target"].tolist()):
        count = full[src] // PAGE
        for c in range(count):
            table[d][c] = table[src][c]
            refs[table[src][c]] += 1
        held[d], full[d], tails[d] = count, full[src], tails[src]
        s["tail_key"][:, slots[d], :tails[src]] = s["tail_key"][:, slots[src], :tails[src]]
        s["tail_value"][:, slots[d], :tails[src]] = s["tail_value"][:, slots[src], :tails[src]]
    return {"table": _ints(table), "held": _ints(held), "refs": _ints(refs), "seqused_fp4": _ints(full),
            "seqused_tail": _ints(tails), "tail_key": s["tail_key"], "tail_value": s["tail_value"]}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attend":
        return _exact_attend(s)
    if case["op"] == "append":
        return _exact_append(s)
    if case["op"] == "dequantize":
        pages = [_exact_page(s["blocks"], s["heads"], int(p)) for p in s["ids"].tolist()]
        return {"key": torch.stack([k for k, _ in pages]), "value": torch.stack([v for _, v in pages])}
    if case["op"] == "fork":
        return _exact_fork(s)
    return None         # whole pages are moved: every output is a whole number
