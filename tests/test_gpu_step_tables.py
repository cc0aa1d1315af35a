"""GPU: page tables, parameter blocks and row slots built from request lengths; groups of lanes with a shared prefix."""
import numpy as np
import pytest
import torch

from richengine_b200 import lib, ops
from richengine_b200.abi import CHUNK_PARAMS, VERIFY_PARAMS

pytestmark = pytest.mark.gpu

BASE, EXTENT_PAGES, EXTENT_STRIDE = 0x7F0000000000, 200, 1 << 24


def entry(page):
    return BASE + page // EXTENT_PAGES * EXTENT_STRIDE | page % EXTENT_PAGES


def i32(values):
    return torch.tensor(np.asarray(values, np.int64).astype(np.uint32).view(np.int32), device="cuda")


def expected(before, width, capacity, page_count, ids, committed, rows, known, splits=1, scale=0.0):
    """The definition, lane by lane."""
    lanes = len(ids)
    entries = before.copy()
    chunk, verify = np.zeros(lanes, CHUNK_PARAMS), np.zeros(lanes, VERIFY_PARAMS)
    offsets, slots, refused = [0], [], False
    for l in range(lanes):
        need = -(-(committed[l] + rows[l]) // 32)
        good = 0 < rows[l] <= capacity and committed[l] + rows[l] <= 262159 and need <= min(len(ids[l]), width)
        first = min(known[l] if known is not None else 0, need)
        taken = [j for j in range(first, need)] if good else []
        for j in taken:
            if ids[l][j] < page_count:
                entries[l, j] = entry(ids[l][j])
        lines = [(ids[l][(committed[l] + r) // 32], (committed[l] + r) % 32) for r in range(rows[l])] if good else []
        good = good and all(ids[l][j] < page_count for j in taken) and all(p < page_count for p, _ in lines)
        refused |= rows[l] > 0 and not good
        mine = min(rows[l], capacity)
        slots += [p * 32 + t for p, t in lines] if good else [-1] * mine
        offsets.append(offsets[-1] + mine)
        live = rows[l] if good else 0
        chunk[l] = (committed[l], live, 32, len(ids[l]), (0, 0))
        verify[l] = (committed[l], len(ids[l]), (0, 0), splits, splits, live, capacity, scale)
    return entries, chunk, verify, offsets, slots, refused


def build(ids, committed, rows, width, capacity, page_count, known=None, splits=1, scale=0.0):
    tables = ops.StepTables(len(ids), width, (BASE, 1 << 34), EXTENT_STRIDE, EXTENT_PAGES, page_count, capacity, splits, scale)
    before = np.random.default_rng(1).integers(1, 2 ** 40, (len(ids), width))
    tables.entries.copy_(torch.from_numpy(before))
    tables.row_slots.fill_(-7)
    offsets = np.concatenate([[0], np.cumsum([len(p) for p in ids])])
    flat = np.concatenate([np.asarray(p, np.int64) for p in ids] + [np.zeros(1, np.int64)])
    tables.build(i32(flat), i32(offsets), i32(committed), i32(rows), i32(known) if known is not None else None)
    return tables, before


def compare(tables, before, *args, **kwargs):
    entries, chunk, verify, offsets, slots, refused = expected(before, *args, **kwargs)
    assert np.array_equal(tables.entries.cpu().numpy(), entries)
    assert tables.chunk_params.cpu().numpy().tobytes() == chunk.tobytes()
    assert tables.verify_params.cpu().numpy().tobytes() == verify.tobytes()
    assert tables.row_offsets.cpu().tolist() == offsets
    assert tables.row_slots.cpu().tolist() == slots + [-7] * (tables.row_slots.numel() - len(slots))
    if refused:
        with pytest.raises(lib.RichKvError, match="rk_step_tables"):
            tables.check()
    tables.check()


@pytest.mark.parametrize("lanes,width,capacity", [(1, 1, 1), (1, 8193, 16), (7, 5, 1), (33, 601, 8), (1024, 37, 16)])
@pytest.mark.parametrize("known", [False, True])
def test_tables_match_the_definition(lanes, width, capacity, known):
    rng = np.random.default_rng(lanes + width)
    counts = [int(rng.integers(1, width + 1)) for _ in range(lanes)]
    counts[0] = width
    rows = [int(rng.integers(0, capacity + 1)) for _ in range(lanes)]
    committed = [max(0, min(n * 32, 262159) - r - int(rng.integers(0, 40))) for n, r in zip(counts, rows)]
    ids = [rng.integers(0, 10 ** 6, n) for n in counts]
    from_page = [int(rng.integers(0, n + 2)) for n in counts] if known else None
    tables, before = build(ids, committed, rows, width, capacity, 10 ** 6, from_page, splits=5, scale=0.25)
    compare(tables, before, width, capacity, 10 ** 6, ids, committed, rows, from_page, 5, 0.25)


def test_refused_lanes_become_idle_and_leave_the_others_alone():
    good = [3, 4, 5]
    cases = [  # (pages, committed, rows)
        (good, 40, 2),
        (good, 95, 2),              # past its pages
        (good, 10, 9),              # past the row capacity
        ([], 0, 1),                 # no page at all
        ([1] * 9, 200, 1),          # more pages than the table holds
        ([3, 100, 5], 70, 1),       # a page past the pool
        ([3, 4, 2 ** 32 - 1], 64, 1),
        (good, 2 ** 32 - 1, 8),     # far past any sequence
        (good, 0, 0),               # idle, not refused
        (good, 64, 8),
    ]
    ids, committed, rows = ([c[i] for c in cases] for i in range(3))
    tables, before = build(ids, committed, rows, 6, 8, 100)
    compare(tables, before, 6, 8, 100, ids, committed, rows, None)
    live = np.frombuffer(tables.verify_params.cpu().numpy().tobytes(), VERIFY_PARAMS)["active_rows"]
    assert live.tolist() == [2, 0, 0, 0, 0, 0, 0, 0, 0, 8]


def test_the_page_of_a_new_row_is_looked_at_among_the_known_ones_too():
    ids, committed, rows, known = [[1, 500]], [40], [1], [2]
    tables, before = build(ids, committed, rows, 4, 1, 100, known)
    compare(tables, before, 4, 1, 100, ids, committed, rows, known)
    assert tables.row_slots.cpu().tolist() == [-1]


def test_offsets_past_the_page_ids_are_refused():
    """page_ids is the middle of a longer vector of good ids: a lane whose offsets leave it, on either side, is idle and writes no
    entry; its neighbours are what they are alone."""
    around = i32([7] * 40)
    page_ids = around[16:22]
    page_ids.copy_(i32([3, 4, 5, 6, 8, 9]))
    offsets = [(0, 2), (2, 7), (7, 8), (-4, 2), (2 ** 32 - 2, 2 ** 32 - 1), (5, 4), (4, 6)]
    for begin, end in offsets:
        tables = ops.StepTables(2, 4, (BASE, 1 << 30), EXTENT_STRIDE, EXTENT_PAGES, 100)
        # lane 1 has what the pair says; lane 0 whatever ends where that begins
        tables.build(page_ids, i32([min(begin % 2 ** 32, 1), begin % 2 ** 32, end % 2 ** 32]), i32([0, 0]), i32([0, 1]))
        live = np.frombuffer(tables.verify_params.cpu().numpy().tobytes(), VERIFY_PARAMS)
        good = 0 <= begin <= end <= 6
        assert live["active_rows"].tolist() == [0, int(good)] and live["page_table_entries"][1] == (end - begin if good else 0)
        assert tables.entries[1].tolist() == ([entry(int(page_ids[begin])), 0, 0, 0] if good else [0] * 4)
        if not good:
            with pytest.raises(lib.RichKvError, match="rk_step_tables"):
                tables.check()
        tables.check()


@pytest.mark.parametrize("fmt", [1, 2, 3, 4])
def test_entries_equal_the_storage_s_own(fmt):
    """Against rk_storage_entry for pages of every extent (an extent's address range is rounded up to the mapping's grain)."""
    from richengine_b200.abi import Layout
    from richengine_b200.storage import PageStorage
    layout = Layout(1, 4, 256, fmt)
    extent_pages = layout.extent_alignment_pages()
    storage = PageStorage(layout, 5 * extent_pages, extent_pages)
    for extent in range(5):
        assert storage.allocate_extent(extent)
    ids = np.random.default_rng(fmt).permutation(5 * extent_pages)[:40]
    tables = ops.StepTables.for_storage(storage, 1, 40)
    tables.build(i32(ids), i32([0, len(ids)]), i32([len(ids) * 32 - 1]), i32([1]))
    assert tables.entries[0, :len(ids)].tolist() == [storage.entry(int(p)) for p in ids]
    tables.check()
    storage.close()


def test_argument_checks():
    tables = ops.StepTables(2, 4, (BASE, 1 << 30), EXTENT_STRIDE, EXTENT_PAGES, 100)
    two, three = i32([0, 0]), i32([0, 0, 0])
    with pytest.raises(ValueError, match="committed"):
        tables.build(two, three, three, two)
    with pytest.raises(ValueError, match="rows"):
        tables.build(two, three, two, two.long())
    with pytest.raises(ValueError, match="page_ids"):
        tables.build(torch.zeros(4, 2, dtype=torch.int32, device="cuda")[:, 0], three, two, two)
    with pytest.raises(lib.RichKvError, match="16 KiB"):
        ops.StepTables(2, 4, (BASE + 4096, 1 << 30), EXTENT_STRIDE, EXTENT_PAGES, 100).build(two, three, two, two)


# ---- groups ---------------------------------------------------------------------------------------------------------

def groups(tables, committed, active, minimum_lanes=2, minimum_pages=1):
    lanes = len(tables)
    width = max(len(t) for t in tables)
    entries = torch.zeros(lanes, width, dtype=torch.int64)
    params = np.zeros(lanes, VERIFY_PARAMS)
    for l, t in enumerate(tables):
        entries[l, :len(t)] = torch.tensor([entry(p) for p in t])
        params[l] = (committed[l], len(t), (0, 0), 1, 1, active[l], 1, 0.0)
    entries = entries.cuda()
    pointers = entries.data_ptr() + 8 * width * torch.arange(lanes, device="cuda")
    lane_groups, group_pages = (torch.full((lanes,), 77, dtype=torch.int32, device="cuda") for _ in range(2))
    ops.prefix_groups(lanes, pointers, torch.from_numpy(params.view(np.uint8)).cuda(), lane_groups, group_pages, minimum_lanes, minimum_pages)
    return lane_groups.cpu().tolist(), group_pages.cpu().tolist()


def expected_groups(tables, committed, active, minimum_lanes=2, minimum_pages=1):
    lanes = len(tables)
    full = [min(c // 32, len(t)) if a == 1 and -(-(c + 1) // 32) <= len(t) else 0 for t, c, a in zip(tables, committed, active)]
    lane_groups, group_pages = [-1] * lanes, [0] * lanes
    for leader in range(lanes):
        if not full[leader] or any(full[l] and tables[l][0] == tables[leader][0] for l in range(leader)):
            continue
        common = {}
        for l in range(leader, lanes):
            if full[l] and tables[l][0] == tables[leader][0]:
                n = 0
                while n < min(full[l], full[leader]) and tables[l][n] == tables[leader][n]:
                    n += 1
                common[l] = n
        best = (0, 0)
        for p in set(common.values()):
            members = sum(c >= p for c in common.values())
            if members >= minimum_lanes and p >= minimum_pages:
                best = max(best, ((members - 1) * p, p))
        if best[0]:
            group_pages[leader] = best[1]
            for l, c in common.items():
                if c >= best[1]:
                    lane_groups[l] = leader
    return lane_groups, group_pages


@pytest.mark.parametrize("lanes,prompts,longest", [(2, 1, 1), (5, 2, 40), (32, 1, 300), (33, 5, 9), (700, 24, 50), (1024, 3, 700), (1, 1, 5)])
@pytest.mark.parametrize("minimum", [(2, 1), (3, 4)])
def test_groups_match_the_definition(lanes, prompts, longest, minimum):
    rng = np.random.default_rng(lanes * prompts)
    firsts = [list(rng.integers(0, 1000, longest) + 1000 * k) for k in range(prompts)]
    tables, committed, active = [], [], []
    for l in range(lanes):
        prompt = firsts[rng.integers(prompts)]
        shared = int(rng.choice([0, 1, len(prompt) // 2, len(prompt)]))
        tail = [10 ** 5 + 50 * l + k for k in range(int(rng.integers(1, 9)))]
        tables.append(prompt[:shared] + tail)
        committed.append(int(rng.integers(0, len(tables[-1]) * 32)))
        active.append(int(rng.random() < 0.9))
    args = (tables, committed, active, *minimum)
    assert groups(*args) == expected_groups(*args)


def test_group_boundaries():
    same = [1, 2, 3, 4]
    # the page being written is not shared, however equal the entries are
    assert groups([same, same], [95, 127], [1, 1]) == ([0, 0], [2, 0])
    assert groups([same, same], [31, 31], [1, 1]) == ([-1, -1], [0, 0])
    # equal pages behind an unequal first one are no prefix
    assert groups([[9, 2, 3], [1, 2, 3]], [64, 64], [1, 1]) == ([-1, -1], [0, 0])
    # more lanes over fewer pages against fewer lanes over more: (4 - 1) * 2 < (2 - 1) * 7
    long, short = list(range(50, 58)), [50, 51]
    tables = [long + [100 + i] for i in range(2)] + [short + list(range(200 + 9 * i, 209 + 9 * i)) for i in range(2)]
    assert groups(tables, [32 * 7 + 5] * 4, [1] * 4) == ([0, 0, -1, -1], [7, 0, 0, 0])
    # a tie goes to the larger p: (3 - 1) * 2 = (2 - 1) * 4
    tables = [[1, 2, 3, 4, 5], [1, 2, 3, 4, 6], [1, 2, 7, 8, 9]]
    assert groups(tables, [130] * 3, [1] * 3) == ([0, 0, -1], [4, 0, 0])


def test_group_refusals():
    lanes = i32([0, 0])
    for arguments, text in (((2, lanes, lanes, lanes, i32([0, 0]), 1, 1), "two lanes"), ((2, lanes, lanes, lanes, i32([0, 0]), 2, 0), "two lanes"),
                            ((2, lanes, lanes, lanes, lanes, 2, 1), "invalid")):
        with pytest.raises(lib.RichKvError, match=text):
            ops.prefix_groups(*arguments)
    with pytest.raises(ValueError, match="lane_groups"):
        ops.prefix_groups(3, lanes, lanes, lanes, lanes)


def test_the_first_call_may_take_another_stream():
    """Made under a busy stream and built on an idle one at once: the object's own fills are over."""
    busy, idle = torch.cuda.Stream(), torch.cuda.Stream()
    inputs = [i32(v) for v in ([3, 1], [0, 1, 2], [5, 9], [1, 1])]
    torch.cuda.synchronize()
    with torch.cuda.stream(busy):
        torch.cuda._sleep(50_000_000)
        tables = ops.StepTables(2, 4, (1 << 40, 1 << 20), 1 << 16, 2, 8)
    tables.build(*inputs, stream=idle)
    with torch.cuda.stream(idle):
        pointers, slots = tables.table_pointers.clone(), tables.row_slots.clone()
    idle.synchronize()
    assert pointers.tolist() == [tables.entries.data_ptr(), tables.entries.data_ptr() + 32] and slots.tolist() == [101, 41]
    torch.cuda.synchronize()
    assert tables.row_slots.tolist() == [101, 41]


def test_check_waits_for_the_stream_of_the_build():
    """A refusal still on its way on another stream is not missed, and the word is clear before a build anywhere follows."""
    tables = ops.StepTables(1, 4, (BASE, 1 << 30), EXTENT_STRIDE, EXTENT_PAGES, 100)
    bad, good = ([i32(v) for v in ([3, 4], [0, 2], [c], [1])] for c in (70, 5))
    other = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(other):
        torch.cuda._sleep(200_000_000)
    tables.build(*bad, stream=other)
    with pytest.raises(lib.RichKvError, match="rk_step_tables"):
        tables.check()
    with torch.cuda.stream(other):
        torch.cuda._sleep(50_000_000)
    tables.build(*good, stream=other)
    tables.check()
    assert tables.row_slots.tolist() == [3 * 32 + 5]


def test_a_batch_without_pages():
    """Every lane idle and no page named: an empty vector of ids will do; a lane that asks for a row all the same is refused."""
    for rows in ([0, 0], [0, 1]):
        tables = ops.StepTables(2, 4, (BASE, 1 << 30), EXTENT_STRIDE, EXTENT_PAGES, 100)
        for offsets in ([0, 0, 0], [0, 0, 1]):
            tables.build(i32([]), i32(offsets), i32([0, 0]), i32(rows))
            live = np.frombuffer(tables.verify_params.cpu().numpy().tobytes(), VERIFY_PARAMS)
            assert live["active_rows"].tolist() == [0, 0] and tables.row_offsets.tolist() == [0, 0, rows[1]] and not tables.entries.any()
            if rows[1]:
                with pytest.raises(lib.RichKvError, match="rk_step_tables"):
                    tables.check()
            tables.check()
