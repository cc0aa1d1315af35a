"""Workloads of the serving-step operators over the paged, quantised KV cache: page tables built on the GPU from request
lengths, the search for shared prefixes, decode attention over a shared prefix, and attention with a score shape (tanh cap,
distance bias, sliding window with sink tokens) for single tokens, verify windows and prefill chunks.

`run` computes each in plain torch operations, or, with `own` set, through the framework's own calls.
"""
import math

import numpy as np
import torch

own = False

PAGE = 32                      # tokens of a page
HEADS, GROUP, DIM = 4, 6, 256  # KV heads, query heads per KV head, head dimension
EXTENT = 256                   # pages of an extent
FORMATS = {"int8": 1, "bf16": 2, "int4": 3, "fp8": 4}
DATA = {"int4": PAGE * HEADS * DIM // 2, "int8": PAGE * HEADS * DIM, "fp8": PAGE * HEADS * DIM, "bf16": PAGE * HEADS * DIM * 2}
SCALES = {"int4": PAGE * HEADS * 4, "int8": PAGE * HEADS * 4, "fp8": PAGE * HEADS * 4, "bf16": 0}
POOL_BASE = 0x7F0000000000     # where the table workloads' pool would lie: entries are computed, never followed
STRIDE = 32                    # staging rows of a lane


def listed():
    return [
        # one decode step of eight long requests: one page entry at most is new per request, latency is all
        {"name": "tables 8 requests one token each", "op": "tables", "lanes": 8, "pages": 1024, "known": True, "rows": 1},
        # every table of a full batch built anew, verify windows of up to 16 rows
        {"name": "tables 1024 requests anew", "op": "tables", "lanes": 1024, "pages": 4096, "known": False, "rows": 16},
        # 32 requests forked from one 8K-token prefix (the prefix-sharing configuration of the benchmark)
        {"name": "groups 32 forks of 8K", "op": "groups", "lanes": 32, "prompts": 1, "pages": 273},
        # a large batch over 24 system prompts of different lengths
        {"name": "groups 1024 requests of 24 prompts", "op": "groups", "lanes": 1024, "prompts": 24, "pages": 1000},
        # best-of-four sampling of one 2K-token prompt
        {"name": "shared int8 4 x 2K", "op": "shared", "format": "int8", "lanes": 4, "groups": 1, "prefix": 2048, "suffix": 100,
         "loose": 0, "softcap": 0.0, "slopes": False},
        # 32 requests over one 8K-token prefix, each up to 512 tokens into its own text
        {"name": "shared int4 32 x 8K", "op": "shared", "format": "int4", "lanes": 32, "groups": 1, "prefix": 8192, "suffix": 512,
         "loose": 0, "softcap": 0.0, "slopes": False},
        # a large batch over one 32K-token document
        {"name": "shared int4 256 x 32K", "op": "shared", "format": "int4", "lanes": 256, "groups": 1, "prefix": 32768, "suffix": 1024,
         "loose": 0, "softcap": 0.0, "slopes": False},
        # one short request of a bf16 pool
        {"name": "decode bf16 1 x 100 capped", "op": "decode", "format": "bf16", "lanes": 1, "context": 100, "ragged": False,
         "softcap": 30.0, "window": 0, "sinks": 0, "slopes": False},
        # a full-attention layer with capped scores, 32 x 16K (the format sweep's size)
        {"name": "decode int4 32 x 16K capped", "op": "decode", "format": "int4", "lanes": 32, "context": 16384, "ragged": False,
         "softcap": 50.0, "window": 0, "sinks": 0, "slopes": False},
        # a sliding-window layer with sink tokens and a distance bias, ragged requests of up to 16K tokens
        {"name": "decode fp8 64 x 16K window 4096", "op": "decode", "format": "fp8", "lanes": 64, "context": 16384, "ragged": True,
         "softcap": 0.0, "window": 4096, "sinks": 4, "slopes": True},
        # a 16-row verify window over long capped layers
        {"name": "verify int4 4 x 32K capped", "op": "verify", "format": "int4", "lanes": 4, "context": 32768, "rows": 16, "capacity": 16,
         "softcap": 50.0, "window": 0, "sinks": 0, "slopes": False},
        # a whole prefill chunk of a sliding-window layer
        {"name": "prefill int8 2048 rows over 6K window 4096", "op": "prefill", "format": "int8", "context": 6144, "rows": 2048,
         "softcap": 0.0, "window": 4096, "sinks": 4, "slopes": True},
    ]


def _spread(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["tables", "groups", "shared", "shared", "decode", "decode", "verify", "prefill"])
    fmt = rng.choice(["int4", "int8", "fp8", "bf16"])
    wide = {"int4": 1, "int8": 2, "fp8": 2, "bf16": 4}[fmt]
    shape = {"softcap": rng.choice([0.0, 20.0, 50.0]), "window": rng.choice([0, _spread(rng, 1, 8192)]), "slopes": rng.random() < 0.5}
    shape["sinks"] = rng.choice([0, 4, 70]) if shape["window"] else 0
    if op == "tables":
        return {"op": op, "lanes": _spread(rng, 1, 1024), "pages": _spread(rng, 2, 4096), "known": rng.random() < 0.5, "rows": rng.choice([1, 8, 16])}
    if op == "groups":
        return {"op": op, "lanes": _spread(rng, 2, 1024), "prompts": _spread(rng, 1, 64), "pages": _spread(rng, 2, 1000)}
    if op == "shared":
        lanes = _spread(rng, 2, 256)
        return {"op": op, "format": fmt, "lanes": lanes, "groups": _spread(rng, 1, max(1, min(8, lanes // 2))),
                "prefix": PAGE * _spread(rng, 1, 1024 // wide), "suffix": _spread(rng, 1, 1024 // wide), "loose": rng.choice([0, 0, lanes // 4]),
                "softcap": shape["softcap"], "slopes": shape["slopes"]}
    if op == "decode":
        lanes = _spread(rng, 1, 128)
        return {"op": op, "format": fmt, "lanes": lanes, "context": _spread(rng, 1, min(32768, 524288 // wide // lanes)), "ragged": rng.random() < 0.7, **shape}
    if op == "verify":
        lanes, capacity = _spread(rng, 1, 16), rng.choice([8, 16])
        return {"op": op, "format": fmt, "lanes": lanes, "context": _spread(rng, 1, min(32768, 131072 // wide // lanes)),
                "rows": rng.randint(1, capacity), "capacity": capacity, **shape}
    return {"op": op, "format": fmt, "context": _spread(rng, 1, 6144), "rows": _spread(rng, 1, 2048), **shape}


# ---- inputs ------------------------------------------------------------------------------------------------------

def _device(array):
    return torch.from_numpy(np.ascontiguousarray(array)).cuda()


def _random_slopes(case):
    """The usual geometric slopes of a distance bias, one per query head."""
    if not case.get("slopes"):
        return None
    heads = HEADS * GROUP
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / heads) for h in range(heads)], dtype=torch.float32, device="cuda")


def _pool(fmt, pages, generator):
    """A pool's bytes: extents of [keys x pages][key scales][values][value scales], filled with quantised rows whose
    values are N(0, 1) with four outlier channels per head."""
    extents = -(-pages // EXTENT)
    extent_bytes = EXTENT * 2 * (DATA[fmt] + SCALES[fmt])
    raw = torch.zeros(extents * extent_bytes + 16384, dtype=torch.uint8, device="cuda")
    skip = -raw.data_ptr() % 16384
    pool = raw[skip:skip + extents * extent_bytes].view(extents, extent_bytes)
    parts = _parts(fmt, pool)
    channels = torch.randint(0, DIM, (2, HEADS, 4), device="cuda", generator=generator)
    gain = torch.ones(2, HEADS, DIM, device="cuda").scatter_(2, channels, 20.0)
    gain[1] = gain[1].clamp(max=4.0)
    step = 8
    for first in range(0, extents, step):
        n = min(step, extents - first)
        for which in range(2):
            x = torch.randn(n, EXTENT, HEADS, PAGE, DIM, device="cuda", generator=generator) * gain[which][:, None, :]
            x = x.bfloat16()
            codes, scales = parts[2 * which], parts[2 * which + 1]
            if fmt == "bf16":
                data = x if which == 0 else x.transpose(-1, -2)
                codes[first:first + n] = data.contiguous().view(torch.uint8).reshape(n, EXTENT, -1)
                continue
            x = x.float()
            amax = x.abs().amax(-1, keepdim=True)
            top = {"int4": 7.0, "int8": 127.0, "fp8": 448.0}[fmt]
            scales[first:first + n] = (amax / top).reshape(n, EXTENT, -1)
            y = x * top / amax
            if fmt == "int4":
                c = y.round().clamp(-7, 7).to(torch.int8).view(torch.uint8) & 15
                data = c[..., 0::2] | (c[..., 1::2] << 4)
            else:
                c = y.round().clamp(-127, 127).to(torch.int8).view(torch.uint8) if fmt == "int8" else y.to(torch.float8_e4m3fn).view(torch.uint8)
                data = c if which == 0 else c.transpose(-1, -2)
            codes[first:first + n] = data.reshape(n, EXTENT, -1)
    return raw, pool, extent_bytes


def _parts(fmt, pool):
    """Views of a pool: key codes, key scales, value codes, value scales, each [extent][page][...]."""
    data, scale = EXTENT * DATA[fmt], EXTENT * SCALES[fmt]
    cuts = [0, data, data + scale, 2 * data + scale, 2 * (data + scale)]
    views = [pool[:, a:b] for a, b in zip(cuts, cuts[1:])]
    return [v if not v.shape[1] else v.unflatten(1, (EXTENT, -1)) if i % 2 == 0 else v.unflatten(1, (EXTENT, -1)).view(torch.float32)
            for i, v in enumerate(views)]


def _attention_state(case, seed, contexts, page_lists, query_rows):
    """Pool, page tables and parameter blocks of a batch. `contexts`: committed tokens per lane."""
    generator = torch.Generator("cuda").manual_seed(seed)
    fmt, lanes = case["format"], len(contexts)
    total = 1 + max(int(p.max()) for p in page_lists)
    raw, pool, extent_bytes = _pool(fmt, total, generator)
    width = max(len(p) for p in page_lists)
    pages = np.zeros((lanes, width), np.int64)
    for l, p in enumerate(page_lists):
        pages[l, :len(p)] = p
    pages = _device(pages)
    entries = pool.data_ptr() + (pages // EXTENT) * extent_bytes + pages % EXTENT
    state = {"case": case, "raw": raw, "pool": pool, "pages": pages, "entries": entries,
             "pointers": entries.data_ptr() + 8 * width * torch.arange(lanes, device="cuda"),
             "committed": _device(np.asarray(contexts, np.int64)), "counts": [len(p) for p in page_lists], "slopes": _random_slopes(case),
             "layer": (EXTENT, 0), "window": (pool.data_ptr(), pool.numel())}
    state["queries"] = torch.randn(*query_rows, GROUP, DIM, device="cuda", generator=generator).bfloat16()
    state["output"] = torch.zeros_like(state["queries"])
    return state


def _verify_params(contexts, counts, rows, capacity, splits):
    """The lanes' 36-byte verify parameter blocks as 32-bit words."""
    block = np.zeros((len(contexts), 9), np.uint32)
    block[:, 0], block[:, 1], block[:, 2] = contexts, counts, EXTENT
    block[:, 4], block[:, 5], block[:, 6], block[:, 7] = splits, splits, rows, capacity
    return _device(block.view(np.int32))


def _shuffled(rng, lengths):
    """Page ids of lanes that need `lengths` pages each, from a shuffled pool."""
    ids = rng.permutation(int(sum(lengths))).astype(np.int64)
    return np.split(ids, np.cumsum(lengths)[:-1])


def _contexts(case, rng):
    top = case["context"]
    return [int(rng.randint(max(1, top // 4), top + 1)) if case.get("ragged") else top for _ in range(case.get("lanes", 1))]


def _prepare_tables(case, seed):
    rng = np.random.RandomState(seed)
    lanes, rows = case["lanes"], case["rows"]
    live = rng.randint(1, rows + 1, lanes).astype(np.int32)
    counts = rng.randint(max(1, case["pages"] // 4), case["pages"] + 1, lanes)
    committed = np.maximum(0, np.minimum(counts * PAGE, 262144) - live - rng.randint(0, PAGE, lanes)).astype(np.int32)
    total = int(counts.sum())
    ids = rng.permutation(total).astype(np.int32)
    known = committed // PAGE
    state = {"case": case, "page_ids": _device(ids), "offsets": _device(np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)),
             "committed": _device(committed), "rows": _device(live), "known": _device(known.astype(np.int32)) if case["known"] else None,
             "total": total}
    extent_bytes = EXTENT * 2 * (DATA["int4"] + SCALES["int4"])
    state["extent_bytes"] = extent_bytes
    if own:
        from richengine_b200 import ops
        state["tables"] = ops.StepTables(lanes, case["pages"], (POOL_BASE, -(-total // EXTENT) * extent_bytes), extent_bytes, EXTENT,
                                         total, row_capacity=rows)
    else:
        state["entries"] = torch.zeros(lanes, case["pages"], dtype=torch.int64, device="cuda")
        state["slots"] = torch.zeros(lanes * rows, dtype=torch.int64, device="cuda")
    return state


def _prepare_groups(case, seed):
    rng = np.random.RandomState(seed)
    lanes, width = case["lanes"], case["pages"]
    prompts = [rng.randint(max(1, width // 8), max(2, width * 15 // 16)) for _ in range(case["prompts"])]
    free = rng.permutation(sum(prompts) + lanes * width).astype(np.int64)
    firsts = np.split(free[:sum(prompts)], np.cumsum(prompts)[:-1])
    entries, committed, counts, at = np.zeros((lanes, width), np.int64), np.zeros(lanes, np.int64), np.zeros(lanes, np.int64), sum(prompts)
    extent_bytes = EXTENT * 2 * (DATA["int4"] + SCALES["int4"])
    for l in range(lanes):
        prompt = firsts[rng.randint(case["prompts"])]
        shared = len(prompt) if rng.random_sample() < 0.8 else rng.randint(1, len(prompt) + 1)
        n = rng.randint(shared, width) + 1
        ids = np.concatenate([prompt[:shared], free[at:at + n - shared]])
        at += n - shared
        entries[l, :n] = POOL_BASE + ids // EXTENT * extent_bytes + ids % EXTENT
        counts[l], committed[l] = n, min(n * PAGE - 1 - rng.randint(0, PAGE), 262143)
    state = {"case": case, "entries": _device(entries), "committed": _device(committed),
             "params": _verify_params(committed, counts, 1, 1, 1)}
    state["pointers"] = state["entries"].data_ptr() + 8 * width * torch.arange(lanes, device="cuda")
    state["lane_groups"] = torch.zeros(lanes, dtype=torch.int32, device="cuda")
    state["group_pages"] = torch.zeros(lanes, dtype=torch.int32, device="cuda")
    return state


def _prepare_shared(case, seed):
    rng = np.random.RandomState(seed)
    lanes, groups = case["lanes"], case["groups"]
    top = case["prefix"] // PAGE
    prefix_pages = [top] + [int(rng.randint(max(1, top // 4), top + 1)) for _ in range(groups - 1)]
    member = np.concatenate([np.arange(lanes - case["loose"]) % groups, np.full(case["loose"], -1)])
    rng.shuffle(member)
    suffix = rng.randint(1, case["suffix"] + 1, lanes)  # tokens past the prefix, this step's own token among them
    own_pages = [-(-int(s) // PAGE) for s in suffix]
    lists = _shuffled(rng, prefix_pages + own_pages)
    pages = [np.concatenate([lists[g], lists[groups + l]]) if g >= 0 else lists[groups + l] for l, g in enumerate(member)]
    contexts = [int((prefix_pages[g] if g >= 0 else 0) * PAGE + suffix[l] - 1) for l, g in enumerate(member)]
    state = _attention_state(case, seed, contexts, pages, (lanes, HEADS, STRIDE))
    state["params"] = _verify_params(contexts, state["counts"], 1, 1, 1)
    # a group is named by its first lane, as the search for shared prefixes names it
    leader = [int(np.nonzero(member == g)[0][0]) if (member == g).any() else 0 for g in range(groups)]
    lane_groups = np.array([leader[g] if g >= 0 else -1 for g in member], np.int32)
    group_pages = np.zeros(lanes, np.int32)
    for g in range(groups):
        if (member == g).any():
            group_pages[leader[g]] = prefix_pages[g]
    state["lane_groups"], state["group_pages"] = _device(lane_groups), _device(group_pages)
    state["host"] = {"contexts": contexts, "member": member, "prefix_pages": prefix_pages}
    # members of each group side by side, for the plain form
    most = max(1, max(int((member == g).sum()) for g in range(groups)))
    seats, seat_of = np.zeros((groups, most), np.int64), np.zeros(lanes, np.int64)
    for g in range(groups):
        who = np.nonzero(member == g)[0]
        seats[g, :len(who)] = who
        seat_of[who] = g * most + np.arange(len(who))
    state["seats"], state["seat_of"] = _device(seats), _device(seat_of)
    widest = max(prefix_pages)
    prefix_ids = np.zeros((groups, widest), np.int64)
    for g in range(groups):
        prefix_ids[g, :prefix_pages[g]] = lists[g]
    suffix_ids = np.zeros((lanes, max(own_pages)), np.int64)
    for l in range(lanes):
        suffix_ids[l, :own_pages[l]] = lists[groups + l]
    state["prefix_ids"], state["suffix_ids"] = _device(prefix_ids), _device(suffix_ids)
    state["prefix_tokens"] = _device(np.array(prefix_pages, np.int64) * PAGE)
    state["lane_prefix"] = _device(np.array([prefix_pages[g] * PAGE if g >= 0 else 0 for g in member], np.int64))
    state["grouped"] = _device(member >= 0)
    if own:
        from richengine_b200 import ops
        state["attention"] = ops.SharedPrefixDecode(_layout(case), HEADS * GROUP, lanes, state["window"])
        state["shape"] = _shape(state)
    return state


def _prepare_decode(case, seed):
    rng = np.random.RandomState(seed)
    contexts = [c - 1 for c in _contexts(case, rng)]  # the step's own token is in its page already
    pages = _shuffled(rng, [(c + PAGE) // PAGE for c in contexts])
    state = _attention_state(case, seed, contexts, pages, (len(contexts), HEADS, STRIDE))
    state["params"] = _verify_params(contexts, state["counts"], 1, 1, 1)
    state["host"] = {"contexts": contexts}
    if own:
        from richengine_b200 import ops
        state["attention"] = ops.DecodeAttention(_layout(case), HEADS * GROUP, len(contexts), state["window"])
        state["shape"] = _shape(state)
    return state


def _prepare_verify(case, seed):
    rng = np.random.RandomState(seed)
    contexts, rows, capacity = _contexts(case, rng), case["rows"], case["capacity"]
    lanes = len(contexts)
    pages = _shuffled(rng, [-(-(c + rows) // PAGE) for c in contexts])
    state = _attention_state(case, seed, contexts, pages, (lanes, HEADS, STRIDE))
    most = max(state["counts"])
    splits = max(1, min(148 // (4 * lanes), 128, (most + 1) // 2))  # a CTA per (KV head, split, lane), whole 64-token groups
    state["splits"] = splits
    state["params"] = _verify_params(contexts, state["counts"], rows, capacity, splits)
    slots = lanes * HEADS * splits * capacity * GROUP
    state["partials"] = torch.empty(slots * DIM, device="cuda")
    state["statistics"] = torch.empty(slots * 2, device="cuda")
    state["host"] = {"contexts": contexts}
    if own:
        from richengine_b200 import ops
        state["attention"] = ops.VerifyWindowAttention(_layout(case), HEADS * GROUP, state["window"])
        state["shape"] = _shape(state)
    return state


def _prepare_prefill(case, seed):
    rng = np.random.RandomState(seed)
    contexts, rows = _contexts(case, rng), case["rows"]
    pages = _shuffled(rng, [-(-(c + rows) // PAGE) for c in contexts])
    stride = -(-rows // PAGE) * PAGE
    state = _attention_state(case, seed, contexts, pages, (HEADS, stride))
    tiles = -(-rows // 8)
    splits = max(1, min(32, 32 // tiles))
    state["splits"] = splits
    slots = tiles * HEADS * splits * 8 * GROUP
    state["partials"] = torch.empty(slots * DIM, device="cuda")
    state["statistics"] = torch.empty(slots * 2, device="cuda")
    state["host"] = {"contexts": contexts}
    if own:
        from richengine_b200 import lib, ops
        state["attention"] = ops.VerifyWindowAttention(_layout(case), HEADS * GROUP, state["window"])
        state["params"] = lib.PrefillParams(contexts[0], rows, stride, state["counts"][0], lib.KvLayer(EXTENT, 0), splits, 0.0)
        state["shape"] = _shape(state)
    return state


def prepare(case, seed):
    return {"tables": _prepare_tables, "groups": _prepare_groups, "shared": _prepare_shared, "decode": _prepare_decode,
            "verify": _prepare_verify, "prefill": _prepare_prefill}[case["op"]](case, seed)


# ---- the framework's calls ---------------------------------------------------------------------------------------

def _layout(case):
    from richengine_b200.abi import Layout
    return Layout(1, HEADS, DIM, FORMATS[case["format"]])


def _shape(state):
    from richengine_b200 import ops
    case = state["case"]
    return ops.ScoreShape(softcap=case["softcap"], window=case.get("window", 0), sink_tokens=case.get("sinks", 0), slopes=state["slopes"])


def _words(tensor):
    return tensor.view(torch.uint8).reshape(-1).view(torch.int32)


def _run_own(state):
    from richengine_b200 import lib, ops
    case = state["case"]
    if case["op"] == "tables":
        t = state["tables"]
        t.build(state["page_ids"], state["offsets"], state["committed"], state["rows"], known_pages=state["known"])
        return {"entries": t.entries, "chunk": _words(t.chunk_params).view(-1, 6), "verify": _words(t.verify_params).view(-1, 9),
                "row_offsets": t.row_offsets, "row_slots": t.row_slots}
    if case["op"] == "groups":
        ops.prefix_groups(case["lanes"], state["pointers"], state["params"], state["lane_groups"], state["group_pages"])
        return {"lane_groups": state["lane_groups"], "group_pages": state["group_pages"]}
    layer = lib.KvLayer(*state["layer"])
    if case["op"] == "shared":
        state["attention"].run(state["queries"], state["output"], state["pointers"], state["params"], layer, state["lane_groups"],
                               state["group_pages"], shape=state["shape"])
        return state["output"][:, :, :1]
    if case["op"] == "decode":
        state["attention"].run(state["queries"], state["output"], state["pointers"], state["params"], layer, shape=state["shape"])
        return state["output"][:, :, :1]
    if case["op"] == "verify":
        layout = _layout(case)
        state["attention"].split(case["lanes"], case["capacity"], state["splits"], state["queries"], state["partials"], state["statistics"],
                                 state["pointers"], None, state["params"], layer, shape=state["shape"])
        ops.attention_verify_reduce(layout, HEADS * GROUP, case["lanes"], case["capacity"], state["partials"], state["statistics"],
                                    state["output"], state["params"])
        return state["output"][:, :, :case["rows"]]
    layout = _layout(case)
    state["attention"].prefill_split(state["queries"], state["partials"], state["statistics"], state["entries"], state["params"],
                                     shape=state["shape"])
    ops.attention_prefill_reduce(layout, HEADS * GROUP, state["partials"], state["statistics"], state["output"], state["params"])
    return state["output"][:, :case["rows"]]


# ---- the plain forms ---------------------------------------------------------------------------------------------

def _plain_tables(state):
    case, committed, rows = state["case"], state["committed"].long(), state["rows"].long()
    lanes, width = case["lanes"], case["pages"]
    offsets = state["offsets"].long()
    lane = torch.repeat_interleave(torch.arange(lanes, device="cuda"), offsets[1:] - offsets[:-1], output_size=state["total"])
    column = torch.arange(state["total"], device="cuda") - offsets[lane]
    need = (committed + rows + PAGE - 1) // PAGE
    from_page = state["known"].long() if state["known"] is not None else torch.zeros_like(committed)
    ids = state["page_ids"].long()
    values = POOL_BASE + ids // EXTENT * state["extent_bytes"] + ids % EXTENT
    write = (column < need[lane]) & (column >= from_page[lane])
    entries = torch.where(write, values, state["entries"].view(-1)[lane * width + column])
    state["entries"].view(-1)[lane * width + column] = entries
    zero, one = torch.zeros_like(committed), torch.ones_like(committed)
    counts = offsets[1:] - offsets[:-1]
    chunk = torch.stack([committed, rows, one * STRIDE, counts, zero, zero], 1).int()
    verify = torch.stack([committed, counts, zero, zero, one, one, rows, one * case["rows"], zero], 1).int()
    row_offsets = torch.cat([zero[:1], rows.cumsum(0)])
    within = torch.arange(case["rows"], device="cuda")
    position = committed[:, None] + within
    live = within < rows[:, None]
    page = ids[torch.where(live, offsets[:-1, None] + position // PAGE, 0)]
    target = torch.where(live, row_offsets[:-1, None] + within, lanes * case["rows"])
    slots = torch.cat([state["slots"], zero[:1]])
    slots[target.view(-1)] = (page * PAGE + position % PAGE).view(-1)
    state["slots"] = slots[:-1]
    return {"entries": state["entries"], "chunk": chunk, "verify": verify, "row_offsets": row_offsets.int(), "row_slots": state["slots"]}


def _plain_groups(state):
    entries, full = state["entries"], state["committed"] // PAGE
    lanes, width = entries.shape
    index = torch.arange(lanes, device="cuda")
    fit = full > 0
    same_first = (entries[:, None, 0] == entries[None, :, 0]) & fit[:, None] & fit[None, :]
    leader = torch.where(same_first, index[None, :], lanes).amin(1)
    head = leader.clamp(max=lanes - 1)
    reach = torch.minimum(full, full[head])
    equal = (entries == entries[head]) & (torch.arange(width, device="cuda") < reach[:, None])
    common = torch.where(fit, equal.to(torch.uint8).cumprod(1).sum(1), 0)
    together = same_first & (leader[:, None] == leader[None, :])
    number = (together & (common[None, :] >= common[:, None])).sum(1)
    key = torch.where(fit & (number >= 2) & (common >= 1), (number - 1) * common * 65536 + common, 0)
    best = torch.where(together, key[None, :], 0).amax(1) % 65536
    joins = fit & (best > 0) & (common >= best)
    lane_groups = torch.where(joins, leader, -1).int()
    group_pages = torch.where(joins & (leader == index), best, 0).int()
    return {"lane_groups": lane_groups, "group_pages": group_pages}


def _rows_of(state, ids):
    """Keys and values of pages `ids` (any shape) as fp32 [..., KV head, token, dim]."""
    fmt = state["case"]["format"]
    keys, key_scales, values, value_scales = _parts(fmt, state["pool"])
    e, i = ids // EXTENT, ids % EXTENT
    shape = (*ids.shape, HEADS, PAGE, DIM)
    if fmt == "bf16":
        k, v = keys[e, i].view(torch.bfloat16).float(), values[e, i].view(torch.bfloat16).float()
        return k.view(shape), v.view(*ids.shape, HEADS, DIM, PAGE).transpose(-1, -2)
    ks, vs = key_scales[e, i].view(*ids.shape, HEADS, PAGE, 1), value_scales[e, i].view(*ids.shape, HEADS, PAGE, 1)
    if fmt == "int4":
        def expand(b):
            return torch.stack([((b & 15) ^ 8).to(torch.int8) - 8, ((b >> 4) ^ 8).to(torch.int8) - 8], -1).view(shape).float()
        return expand(keys[e, i]) * ks, expand(values[e, i]) * vs
    kind = torch.int8 if fmt == "int8" else torch.float8_e4m3fn
    k, v = keys[e, i].view(kind).float().view(shape), values[e, i].view(kind).float().view(*ids.shape, HEADS, DIM, PAGE).transpose(-1, -2)
    return k * ks, v * vs


def _part(state, q, ids, base, position, last):
    """One part of an attention: rows q [batch, KV head, row, group, dim] at `position` [batch, row] over pages `ids`
    [batch, page] whose first token is `base` [batch]; tokens past `last` [batch] do not exist. Maximum, sum and sum of values."""
    case = state["case"]
    batch, rows = q.shape[0], q.shape[2]
    k, v = _rows_of(state, ids)                                                       # [batch, page, head, token, dim]
    flat = q.float().reshape(batch, 1, HEADS, rows * GROUP, DIM)
    x = torch.matmul(flat, k.transpose(-1, -2)) / 16.0                                # [batch, page, head, row x group, token]
    x = x.view(batch, -1, HEADS, rows, GROUP, PAGE)
    if case["softcap"]:
        x = case["softcap"] * torch.tanh(x / case["softcap"])
    token = base[:, None, None] + torch.arange(ids.shape[1] * PAGE, device="cuda").view(-1, PAGE)  # [batch, page, token]
    token = token[:, :, None, None, None, :]
    at = position[:, None, None, :, None, None]
    if state["slopes"] is not None:
        x = x - state["slopes"].view(HEADS, 1, GROUP, 1) * (at - token).float()
    seen = (token <= at) & (token <= last[:, None, None, None, None, None])
    if case.get("window"):
        seen = seen & ((at - token < case["window"]) | (token < case["sinks"]))
    x = torch.where(seen, x, -math.inf)
    top = x.amax((1, 5), keepdim=True)
    p = torch.exp(x - torch.where(top > -math.inf, top, 0.0))
    total = p.sum((1, 5))
    o = torch.matmul(p.reshape(batch, -1, HEADS, rows * GROUP, PAGE), v).sum(1)
    return top[:, 0, ..., 0], total, o.view(batch, HEADS, rows, GROUP, DIM)


def _plain_shared(state):
    q = state["queries"][:, :, :1]
    committed = state["committed"]
    seats, groups = state["seats"], state["seats"].shape[0]
    zeros = torch.zeros(groups, dtype=torch.int64, device="cuda")
    first = _part(state, q[seats, :, 0].transpose(1, 2), state["prefix_ids"], zeros, committed[seats], state["prefix_tokens"] - 1)
    # back to one row per lane: [group, head, seat, ...] -> [lane, head, 1, ...]
    m1, l1, o1 = (t.transpose(1, 2).flatten(0, 1)[state["seat_of"]].unsqueeze(2) for t in first)
    m2, l2, o2 = _part(state, q, state["suffix_ids"], state["lane_prefix"], committed[:, None], committed)
    m1 = torch.where(state["grouped"].view(-1, 1, 1, 1), m1, -math.inf)
    m = torch.maximum(m1, m2)
    w1, w2 = torch.exp(m1 - m), torch.exp(m2 - m)
    return ((w1[..., None] * o1 + w2[..., None] * o2) / (w1 * l1 + w2 * l2)[..., None]).bfloat16()


def _plain_rows(state):
    case = state["case"]
    prefill = case["op"] == "prefill"
    rows = case.get("rows", 1)
    q = state["queries"][None, :, :rows] if prefill else state["queries"][:, :, :rows]
    committed = state["committed"]
    position = committed[:, None] + torch.arange(rows, device="cuda")
    _, total, o = _part(state, q, state["pages"], torch.zeros_like(committed), position, committed + rows - 1)
    out = (o / total[..., None]).bfloat16()
    return out[0] if prefill else out


def run(state):
    if own:
        return _run_own(state)
    return {"tables": _plain_tables, "groups": _plain_groups, "shared": _plain_shared, "decode": _plain_rows, "verify": _plain_rows,
            "prefill": _plain_rows}[state["case"]["op"]](state)


# ---- what a pass cannot do without -------------------------------------------------------------------------------

def _seen_tokens(case, position, first_position=None):
    """Tokens that a row at `position` (or rows from first_position on) sees."""
    window = case.get("window", 0)
    low = position if first_position is None else first_position
    if not window or low + 1 <= window:
        return position + 1
    return position - low + window + min(case["sinks"], low + 1 - window)


def work(case):
    op = case["op"]
    if op == "tables":
        lanes, pages = case["lanes"], case["lanes"] * case["pages"] * 5 // 8
        if case["known"]:
            pages = lanes * 2
        return {"bytes": pages * 12 + lanes * (4 + 8 + 24 + 36 + 4) + lanes * (1 + case["rows"]) // 2 * 8, "flops": pages * 4}
    if op == "groups":
        return {"bytes": case["lanes"] * case["pages"] // 2 * 8 + case["lanes"] * (36 + 8), "flops": case["lanes"] * case["pages"] // 2}
    token = 2 * (DATA[case["format"]] + SCALES[case["format"]]) // PAGE
    row = 2 * HEADS * GROUP * DIM * 2
    per_score = 4 * DIM * HEADS * GROUP
    if op == "shared":
        lanes, grouped = case["lanes"], case["lanes"] - case["loose"]
        mean = case["prefix"] * (1 + (case["groups"] - 1) * 5 / 8) / case["groups"]
        own_tokens = lanes * (case["suffix"] + 1) / 2
        return {"bytes": (mean * case["groups"] + own_tokens) * token + lanes * row, "flops": (grouped * mean + own_tokens) * per_score}
    mean = case["context"] * 5 // 8 if case.get("ragged") else case["context"]
    if op == "decode":
        seen = _seen_tokens(case, max(0, mean - 1)) * case["lanes"]
        return {"bytes": seen * token + case["lanes"] * row, "flops": seen * per_score}
    lanes, rows = case.get("lanes", 1), case["rows"]
    seen = _seen_tokens(case, mean + rows - 1, mean)
    scores = sum(_seen_tokens(case, mean + r) for r in range(rows))
    return {"bytes": lanes * (seen * token + rows * row), "flops": lanes * scores * per_score}


# ---- the definition in 64 bits -----------------------------------------------------------------------------------

def _page64(fmt, state, page):
    """One lane's pages, straight from the pool's bytes: keys and values [head, tokens, dim] in 64 bits."""
    flat, size = state["pool"].view(-1), DATA[fmt]
    extent_bytes = state["pool"].shape[1]
    start = (page // EXTENT) * extent_bytes
    inside = page % EXTENT

    def bytes_at(tensor, length):
        before = EXTENT * ((tensor + 1) // 2 * size + tensor // 2 * SCALES[fmt])
        where = (start + before + inside * length)[:, None] + torch.arange(length, device="cuda")
        return flat[where]

    result = []
    for tensor in (0, 2):
        raw = bytes_at(tensor, size)
        if fmt == "int4":
            nibble = torch.tensor([n - 16 if n > 7 else n for n in range(16)], dtype=torch.float64, device="cuda")
            table = torch.stack([nibble.repeat(16), nibble.repeat_interleave(16)], 1)  # byte -> (low, high)
            x = table[raw.long()].reshape(-1, HEADS, PAGE, DIM)
        else:
            kind = {"int8": torch.int8, "fp8": torch.float8_e4m3fn, "bf16": torch.bfloat16}[fmt]
            x = raw.view(kind).double()
            x = x.reshape(-1, HEADS, PAGE, DIM) if tensor == 0 else x.reshape(-1, HEADS, DIM, PAGE).permute(0, 1, 3, 2)
        if fmt != "bf16":
            x = x * bytes_at(tensor + 1, SCALES[fmt]).view(torch.float32).double().reshape(-1, HEADS, PAGE, 1)
        result.append(x.permute(1, 0, 2, 3).reshape(HEADS, -1, DIM))
    return result


def exact(case, seed):
    if case["op"] in ("tables", "groups"):
        return None
    state = prepare(case, seed)
    rows, prefill = case.get("rows", 1), case["op"] == "prefill"
    if case["op"] == "shared":
        rows = 1
    outputs = []
    for lane, committed in enumerate(state["host"]["contexts"]):
        tokens = committed + rows
        page = state["pages"][lane, :-(-tokens // PAGE)]
        keys, values = (x[:, :tokens] for x in _page64(case["format"], state, page))
        q = (state["queries"] if prefill else state["queries"][lane])[:, :rows].double()
        t = torch.arange(tokens, device="cuda")
        blocks = []
        for first in range(0, rows, 256):
            part = q[:, first:first + 256]
            n = part.shape[1]
            score = torch.einsum("hrgd,htd->hrgt", part, keys) * 0.0625
            if case["softcap"]:
                score = torch.tanh(score / case["softcap"]) * case["softcap"]
            distance = committed + first + torch.arange(n, device="cuda")[:, None] - t
            if state["slopes"] is not None:
                score -= state["slopes"].double().view(HEADS, 1, GROUP, 1) * distance.double()[None, :, None, :]
            hidden = distance < 0
            if case.get("window"):
                hidden |= (distance >= case["window"]) & (t >= case["sinks"])
            score.masked_fill_(hidden[None, :, None, :], -math.inf)
            blocks.append(torch.einsum("hrgt,htd->hrgd", score.softmax(-1), values))
        outputs.append(torch.cat(blocks, 1))
    return outputs[0] if prefill else torch.stack(outputs)
