"""A small serving step on the GPU: tables from request lengths, groups from the tables, decode over the shared prefix, and a verify
window with a score shape; the rows against 64-bit attention from the pages' bytes."""
import numpy as np
import torch

from gpuhelp import dev
from richengine_b200 import ops
from servingcase import DIM, GROUP, HEADS, Batch, check_rows, host16, make_queries


def run(fmt):
    rng = np.random.default_rng(1)
    ids = [[4, 7, 1, 9], [4, 7, 1, 2], [4, 7, 1, 5], [0, 3]]
    committed = [100, 127, 96, 40]
    batch = Batch(fmt, ids, 1)
    lanes = len(ids)
    q = make_queries(rng, lanes, HEADS, 32, GROUP, DIM)
    queries = dev(q)
    out, out32 = torch.zeros(q.shape, dtype=torch.bfloat16, device="cuda"), torch.zeros(q.shape, dtype=torch.float32, device="cuda")
    tables = ops.StepTables.for_storage(batch.storage, lanes, 4)
    tables.build(dev(np.concatenate(ids).astype(np.int32)), dev(np.cumsum([0] + [len(p) for p in ids]).astype(np.int32)),
                 dev(np.array(committed, np.int32)), torch.ones(lanes, dtype=torch.int32, device="cuda"))
    lane_groups, group_pages = (torch.zeros(lanes, dtype=torch.int32, device="cuda") for _ in range(2))
    ops.prefix_groups(lanes, tables.table_pointers, tables.verify_params, lane_groups, group_pages)
    shared = ops.SharedPrefixDecode(batch.layout, HEADS * GROUP, lanes, batch.storage.window())
    shape = ops.ScoreShape(softcap=20.0, window=60, sink_tokens=4)
    shared.run(queries, out, tables.table_pointers, tables.verify_params, batch.layer, lane_groups, group_pages, output_f32=out32, shape=shape)
    shared.status()
    tables.check()
    assert lane_groups.tolist() == [0, 0, 0, -1] and group_pages.tolist() == [3, 0, 0, 0]
    for lane in range(lanes):
        want, bound = batch.attend(lane, committed[lane], q[lane, :, 0], (20.0, 60, 4, None))
        # two partials meet in the merge: a few roundings of 2^-23 more
        check_rows(out32[lane, :, 0].cpu().numpy(), host16(out)[lane, :, 0], want, bound + 2.0 ** -20 * np.abs(want).max(), f"shared decode, lane {lane}")
    shared.close()
    # the last eight tokens of each lane as a verify window
    first = [c - 7 for c in committed]
    params = batch.params(first, 8, 8, 1)
    slots = lanes * HEADS * 8 * GROUP
    partials, statistics = torch.empty(slots * DIM, device="cuda"), torch.empty(slots * 2, device="cuda")
    window = ops.VerifyWindowAttention(batch.layout, HEADS * GROUP, batch.storage.window())
    window.split(lanes, 8, 1, queries, partials, statistics, batch.pointers, None, params, batch.layer, shape=shape)
    ops.attention_verify_reduce(batch.layout, HEADS * GROUP, lanes, 8, partials, statistics, out, params, output_f32=out32)
    window.check()
    for lane in range(lanes):
        for r in (0, 7):
            want, bound = batch.attend(lane, first[lane] + r, q[lane, :, r], (20.0, 60, 4, None))
            check_rows(out32[lane, :, r].cpu().numpy(), host16(out)[lane, :, r], want, bound, f"verify window, lane {lane}, row {r}")
    window.close()
    batch.close()
