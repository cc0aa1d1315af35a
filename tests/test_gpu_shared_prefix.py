"""GPU: decode attention over shared prefixes against attention in 64 bits from the pages' bytes, and the whole step:
tables from request lengths, groups from the tables, append, attention, as eager calls and as a replayed graph."""
import numpy as np
import pytest
import torch

from gpuhelp import dev
from richengine_b200 import lib, ops
from richengine_b200.abi import BF16, FP8E4M3, INT4, INT8
from servingcase import DIM, FORMATS, GROUP, HEADS, PAGE, SLOPES, Batch, check_rows, host16, make_queries, shape_of

pytestmark = pytest.mark.gpu


class Shared:
    """`groups`: (prefix pages, members) each; `loose` lanes share nothing. Lanes of all groups are mixed."""

    def __init__(self, fmt, groups, loose=0, suffix=70, seed=4, members_first=False):
        rng = np.random.default_rng(seed)
        member = [g for g, (_, n) in enumerate(groups) for _ in range(n)] + [-1] * loose
        if not members_first:
            rng.shuffle(member)
        lanes = len(member)
        tokens = rng.integers(1, suffix + 1, lanes)  # past the prefix, this step's own among them
        own = [-(-int(t) // PAGE) for t in tokens]
        ids = iter(rng.permutation(sum(p for p, _ in groups) + sum(own)))
        prefixes = [[next(ids) for _ in range(p)] for p, _ in groups]
        pages = [(prefixes[g] if g >= 0 else []) + [next(ids) for _ in range(own[l])] for l, g in enumerate(member)]
        self.committed = [(len(prefixes[g]) * PAGE if g >= 0 else 0) + int(tokens[l]) - 1 for l, g in enumerate(member)]
        self.member, self.lanes = member, lanes
        self.batch = Batch(fmt, pages, seed)
        self.queries = make_queries(rng, lanes, HEADS, 32, GROUP, DIM)
        names = list(rng.permutation(lanes)[:len(groups)])  # any number below `lanes` names a group
        self.lane_groups = dev(np.array([names[g] if g >= 0 else -1 for g in member], np.int32))
        group_pages = np.zeros(lanes, np.int32)
        for g, (p, _) in enumerate(groups):
            group_pages[names[g]] = p
        self.group_pages = dev(group_pages)

    def run(self, shape=None, ctas=0, params=None, runner=None, lane_groups=None):
        b = self.batch
        own = runner is None
        if own:
            runner = ops.SharedPrefixDecode(b.layout, 24, self.lanes, b.storage.window(), ctas)
            for scratch in (runner.partials, runner.statistics, runner.prefix_partials, runner.prefix_statistics):
                scratch.fill_(float("nan"))
            runner.prefix_descriptors.fill_(0x7f7f7f7f)
        q = dev(self.queries)
        out = torch.zeros(q.shape, dtype=torch.bfloat16, device="cuda")
        out32 = torch.zeros(q.shape, dtype=torch.float32, device="cuda")
        runner.run(q, out, b.pointers, params if params is not None else b.params(self.committed), b.layer,
                   lane_groups if lane_groups is not None else self.lane_groups, self.group_pages, output_f32=out32,
                   shape=shape_of(shape) if shape else None)
        runner.status()
        if own:
            runner.close()
        return host16(out), out32.cpu().numpy()

    def check(self, got16, got32, shape=None, lanes=None, scale=1.0 / 16.0):
        for lane in lanes if lanes is not None else range(self.lanes):
            want, bound = self.batch.attend(lane, self.committed[lane], self.queries[lane, :, 0], shape, scale)
            # two partials meet in the merge: their weights' exponentials and the sum add a few roundings of 2^-23
            check_rows(got32[lane, :, 0], got16[lane, :, 0], want, bound + 2.0 ** -20 * np.abs(want).max(), f"lane {lane}")
        assert not got16[:, :, 1:].any()


GROUPS = {
    "one page, two lanes": ([(1, 2)], 0),
    "one lane alone": ([(3, 1)], 2),
    "a tile and its neighbours": ([(2, 21), (3, 22), (1, 43)], 0),
    "odd pages": ([(7, 5), (1, 3), (10, 4)], 3),
    "a long prefix": ([(40, 6)], 1),
    "nobody shares": ([], 4),
}


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("name", GROUPS)
def test_against_64_bits(fmt, name):
    groups, loose = GROUPS[name]
    s = Shared(fmt, groups, loose)
    pick = sorted(set(range(0, s.lanes, max(1, s.lanes // 8))) | {s.lanes - 1})
    for ctas in (0, 5):  # five CTAs: more tiles than CTAs, each CTA takes several
        s.check(*s.run(ctas=ctas), lanes=pick)
    s.batch.close()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("ctas", [1, 2])
def test_many_items_per_block(fmt, ctas):
    """24 tiles and heads on one or two CTAs: each takes more of them than it plans at a time."""
    groups, loose = GROUPS["a tile and its neighbours"]
    s = Shared(fmt, groups, loose, suffix=40)
    s.check(*s.run(ctas=ctas), lanes=range(0, s.lanes, 9))
    s.batch.close()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("shape", [(4.0, 0, 0, None), (0.0, 0, 0, SLOPES), (0.0, 60, 3, None), (6.0, 150, 40, SLOPES), (0.0, 1, 0, None)])
def test_with_a_score_shape(fmt, shape):
    s = Shared(fmt, [(5, 6), (3, 2)], 2)
    s.check(*s.run(shape), shape)
    s.batch.close()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("shape", [(0.0, 200, 40, None), (0.0, 90, 0, SLOPES), (0.0, 10, 33, None), (7.0, 1000, 1, None)])
@pytest.mark.parametrize("ctas", [0, 3])
def test_prefix_pages_outside_every_window_are_not_read(fmt, shape, ctas):
    """Prefixes longer than the window: pages that no member sees are 0xFF throughout, NaN where the format or its scales
    have one. Some members see the prefix's end, some only its sinks, some nothing of it."""
    _, window, sinks, _ = shape
    s = Shared(fmt, [(40, 6), (9, 30), (3, 2)], 2, suffix=150)
    seen = {page for lane, pages in enumerate(s.batch.pages) for j, page in enumerate(pages)
            if j * PAGE < sinks or (j + 1) * PAGE + window > s.committed[lane] + 1}
    poisoned = {page for pages in s.batch.pages for page in pages} - seen
    assert window == 1000 or poisoned
    for page in poisoned:
        for tensor in range(4):
            view = s.batch.host.tensor_view(page, 0, tensor)
            view.view(np.uint8)[:] = 0xff
    s.batch.upload()
    s.check(*s.run(shape, ctas=ctas), shape, lanes=range(0, s.lanes, 5))
    s.batch.close()


@pytest.mark.parametrize("fmt", [INT4, BF16])
def test_equals_the_plain_decode(fmt):
    """The same batch without its groups is rk_attention_decode's business: same rows up to the bound, and bit for bit
    when no lane belongs to a group."""
    s = Shared(fmt, [(9, 30)], 5)
    b = s.batch
    alone = dev(np.full(s.lanes, -1, np.int32))
    none16, none32 = s.run(lane_groups=alone)
    shared16, shared32 = s.run()
    s.check(none16, none32, lanes=range(0, s.lanes, 5))
    s.check(shared16, shared32, lanes=range(0, s.lanes, 5))
    plain = ops.DecodeAttention(b.layout, 24, s.lanes, b.storage.window())
    q = dev(s.queries)
    out32 = torch.zeros(q.shape, dtype=torch.float32, device="cuda")
    plain.run(q, torch.zeros(q.shape, dtype=torch.bfloat16, device="cuda"), b.pointers, b.params(s.committed), b.layer, output_f32=out32)
    # the merges divide differently (a reciprocal against a division) and group their slots differently: 2^-20 of a row's largest
    difference = np.abs(out32.cpu().numpy() - none32)
    assert difference.max() <= 2.0 ** -20 * np.abs(none32).max()
    plain.close()
    b.close()


def test_repeats_bit_for_bit_and_scratch_is_reused():
    s = Shared(INT4, [(12, 25), (4, 3)], 2)
    b = s.batch
    runner = ops.SharedPrefixDecode(b.layout, 24, s.lanes, b.storage.window())
    first = s.run(runner=runner)
    other = s.run((3.0, 0, 0, None), runner=runner)
    again = s.run(runner=runner)
    assert np.array_equal(first[0], again[0]) and np.array_equal(first[1], again[1]) and not np.array_equal(first[1], other[1])
    runner.close()
    b.close()


@pytest.mark.parametrize("fmt", [INT8, FP8E4M3])
def test_idle_lanes(fmt):
    """Idle members and idle leaders: the others of their group go on, the idle ones' rows stay as they are."""
    s = Shared(fmt, [(3, 6), (2, 2)], 2)
    rows = [1] * s.lanes
    for g in (0, 1):
        rows[s.member.index(g)] = 0  # the lowest member of each
    got16, got32 = s.run(params=s.batch.params(s.committed, rows=rows))
    idle = [l for l in range(s.lanes) if not rows[l]]
    assert not got16[idle].any() and not got32[idle].any()
    s.check(got16, got32, lanes=[l for l in range(s.lanes) if rows[l]])
    s.batch.close()


@pytest.mark.parametrize("fmt", [INT4, BF16])
def test_a_prefix_that_covers_everything(fmt):
    """Every committed page shared and the step's own token alone behind it; and a batch whose lanes lie inside the prefix
    (no lane has anything to stream)."""
    s = Shared(fmt, [(4, 9)], 0, suffix=1)
    s.check(*s.run())
    s.committed = [127 - l for l in range(s.lanes)]  # rows of the prefix itself
    s.check(*s.run(ctas=3))
    s.batch.close()


@pytest.mark.parametrize("fmt", FORMATS)
def test_many_lanes(fmt):
    s = Shared(fmt, [(6, 300), (3, 40)], 60, suffix=40)
    s.check(*s.run(), lanes=range(0, s.lanes, 37))
    s.batch.close()


@pytest.mark.parametrize("fmt", [INT4, FP8E4M3])
def test_large_queries_and_peaked_rows(fmt):
    s = Shared(fmt, [(10, 8)], 1)
    s.queries = (s.queries.astype(np.int32) + (3 << 7)).astype(np.uint16)  # x 8 (three more in the exponent)
    got16, got32 = s.run()
    s.check(got16, got32)
    s.queries = (s.queries.astype(np.int32) + (12 << 7)).astype(np.uint16)  # past fp16's range: a power of two keeps it
    params = s.batch.params(s.committed, score_scale=2.0 ** -16)
    got16, got32 = s.run(params=params)
    s.check(got16, got32, scale=2.0 ** -16)
    s.batch.close()


def test_refusals():
    s = Shared(INT4, [(1, 2)], 0)
    b = s.batch
    with pytest.raises(lib.RichKvError, match="lanes out of range"):
        ops.SharedPrefixDecode(b.layout, 24, 1025, b.storage.window())
    with pytest.raises(lib.RichKvError, match="4 KV heads"):
        ops.SharedPrefixDecode(b.layout, 32, 4, b.storage.window())
    runner = ops.SharedPrefixDecode(b.layout, 24, 2, b.storage.window())
    with pytest.raises(ValueError, match="lane_groups"):
        s.run(runner=runner, lane_groups=dev(np.zeros(3, np.int32)))
    runner.close()
    b.close()


# ---- the step as it is used -------------------------------------------------------------------------------------------

@pytest.mark.parametrize("fmt", FORMATS)
def test_a_whole_step_eager_and_replayed(fmt):
    """Lengths in, attention out: tables, groups, append and shared attention, for a batch that grows by a token a step;
    the steps run eagerly and once more as one captured graph with the lengths changed between replays."""
    rng = np.random.default_rng(12)
    prefix, lanes, steps = 5, 9, 3
    start = [prefix * PAGE + int(rng.integers(0, 60)) for _ in range(lanes - 1)] + [40]
    counts = [-(-(c + steps) // PAGE) for c in start]
    free = iter(rng.permutation(300))  # pages of several extents
    shared = [next(free) for _ in range(prefix)]
    ids = [(shared if l < lanes - 1 else []) + [next(free) for _ in range(n - prefix if l < lanes - 1 else n)] for l, n in enumerate(counts)]
    batch = Batch(fmt, ids, 12)
    layout, storage = batch.layout, batch.storage
    tables = ops.StepTables.for_storage(storage, lanes, max(counts))
    runner = ops.SharedPrefixDecode(layout, 24, lanes, storage.window())
    lane_groups, group_pages = (torch.zeros(lanes, dtype=torch.int32, device="cuda") for _ in range(2))
    flat, offsets = dev(np.concatenate(ids).astype(np.int32)), dev(np.concatenate([[0], np.cumsum(counts)]).astype(np.int32))
    committed, rows = dev(np.array(start, np.int32)), torch.ones(lanes, dtype=torch.int32, device="cuda")
    keys = dev(make_queries(rng, steps, lanes, HEADS, 32, DIM))
    values = dev(make_queries(rng, steps, lanes, HEADS, DIM, 32))
    queries = dev(make_queries(rng, steps, lanes, HEADS, 32, GROUP, DIM))
    k, v, q = keys[0].clone(), values[0].clone(), queries[0].clone()
    out = torch.zeros(q.shape, dtype=torch.bfloat16, device="cuda")
    out32 = torch.zeros(q.shape, dtype=torch.float32, device="cuda")

    def step(stream=None):
        tables.build(flat, offsets, committed, rows, stream=stream)
        ops.prefix_groups(lanes, tables.table_pointers, tables.verify_params, lane_groups, group_pages, stream=stream)
        ops.store_verify(layout, k, v, tables.table_pointers, tables.chunk_params, batch.layer, lanes, 1, stream)
        runner.run(q, out, tables.table_pointers, tables.verify_params, batch.layer, lane_groups, group_pages, output_f32=out32, stream=stream)

    def feed(s):
        committed.copy_(torch.tensor(start, dtype=torch.int32) + s)
        k.copy_(keys[s]), v.copy_(values[s]), q.copy_(queries[s])

    eager = []
    for s in range(steps):
        feed(s)
        step()
        tables.check()
        runner.status()
        assert lane_groups.cpu().tolist() == [0] * (lanes - 1) + [-1] and group_pages.cpu().tolist() == [prefix] + [0] * (lanes - 1)
        eager.append((host16(out), out32.cpu().numpy()))
    for extent in range(batch.host.extents):  # the pages as the device has them now
        batch.host.bytes[extent][:] = storage.read_extent(extent)
    host_queries = queries.cpu().view(torch.int16).numpy().view(np.uint16)
    for s in range(steps):
        for lane in range(lanes):
            want, bound = batch.attend(lane, start[lane] + s, host_queries[s, lane, :, 0])
            check_rows(eager[s][1][lane, :, 0], eager[s][0][lane, :, 0], want, bound + 2.0 ** -20 * np.abs(want).max(), f"step {s}, lane {lane}")

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    feed(0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step(stream)
    for s in (0, 2, 1, 2):
        feed(s)
        out.zero_(), out32.zero_()
        graph.replay()
        assert np.array_equal(host16(out), eager[s][0]) and np.array_equal(out32.cpu().numpy(), eager[s][1])
    runner.status()
    del graph
    runner.close()
    batch.close()


@pytest.mark.parametrize("fmt", [INT4, BF16])
def test_a_session_that_shares_prefixes(fmt):
    """DecodeSession: tables from lengths, append and attention of each step through step_device, with the prefix shared and
    without, with a layer's score shape and without."""
    from richengine_b200.session import DecodeSession
    s = Shared(fmt, [(6, 7)], 2, suffix=40)
    b, shape = s.batch, (9.0, 0, 0, SLOPES)
    session = DecodeSession(b.storage, 24, s.lanes)
    tables = session.step_tables(max(map(len, b.pages)))
    ids, counts = np.concatenate(b.pages).astype(np.int32), [len(p) for p in b.pages]
    tables.build(dev(ids), dev(np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)), dev(np.array(s.committed, np.int32)),
                 torch.ones(s.lanes, dtype=torch.int32, device="cuda"))
    rng = np.random.default_rng(3)
    session.chunk_keys.copy_(dev(make_queries(rng, s.lanes, HEADS, 32, DIM)).view(torch.bfloat16))
    session.chunk_values.copy_(dev(make_queries(rng, s.lanes, HEADS, DIM, 32)).view(torch.bfloat16))
    session.queries.copy_(dev(s.queries).view(torch.bfloat16))
    steps = []
    for sharing, with_shape in ((False, False), (True, False), (True, True), (False, True)):
        if sharing:
            session.share_prefixes(tables.table_pointers, tables.verify_params, minimum_pages=1)
            assert int(session._group_pages.max()) == 6 and int((session._lane_groups >= 0).sum()) == 7
        else:
            session.forget_prefixes()
        session.output.zero_()
        session.step_device(0, tables.table_pointers, tables.chunk_params, tables.verify_params, shape=shape_of(shape) if with_shape else None)
        steps.append((with_shape, host16(session.output)))
    session.status()
    tables.check()
    # by default two lanes over a few pages are not worth a kernel of their own
    session.share_prefixes(tables.table_pointers, tables.verify_params)
    assert int(session._group_pages.max()) == 0
    for extent in range(b.host.extents):
        b.host.bytes[extent][:] = b.storage.read_extent(extent)
    for with_shape, got16 in steps:
        for lane in range(s.lanes):
            want, bound = b.attend(lane, s.committed[lane], s.queries[lane, :, 0], shape if with_shape else None)
            got = (got16[lane, :, 0].astype(np.uint32) << 16).view(np.float32)
            assert (np.abs(got - want) <= bound + 2.0 ** -20 * np.abs(want).max() + np.abs(want) * 2.0 ** -8 + bound * 2.0 ** -8).all()
    session.close()
    b.close()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("shape", [None, (20.0, 0, 0, None), (300.0, 0, 0, SLOPES)])
def test_a_query_row_that_is_no_number_comes_out_as_zeros(fmt, shape):
    s = Shared(fmt, [(5, 6)], 2)
    clean = s.queries.copy()
    grouped, loose = s.member.index(0), s.member.index(-1)
    for lane in (grouped, loose):
        s.queries[lane, 1, 0, 3, 100] = 0x7fc0
    got16, got32 = s.run(shape)
    s.queries = clean
    for lane in (grouped, loose):
        assert not got16[lane, 1, 0, 3].any() and not got32[lane, 1, 0, 3].any()
        want, bound = s.batch.attend(lane, s.committed[lane], clean[lane, :, 0], shape)
        got32[lane, 1, 0, 3] = want[1, 3]
        check_rows(got32[lane, :, 0], None, want, bound + 2.0 ** -20 * np.abs(want).max(), f"lane {lane}")
    s.check(got16, got32, shape, lanes=[l for l in range(s.lanes) if l not in (grouped, loose)])
    s.batch.close()


def session_of(s):
    """A session over a Shared batch, its queries in place; and a step's rows and launches."""
    from richengine_b200.session import DecodeSession
    session = DecodeSession(s.batch.storage, 24, s.lanes)
    session.queries.copy_(dev(s.queries).view(torch.bfloat16))
    params = s.batch.params(s.committed)

    def attend(shape=None):
        before = session.kernel_launches
        session.output.zero_()
        session.attend_device(0, s.batch.pointers, params, shape=shape_of(shape) if shape else None)
        return host16(session.output), session.kernel_launches - before

    return session, params, attend


def check16(s, got16, lanes, shape=None):
    for lane in lanes:
        want, bound = s.batch.attend(lane, s.committed[lane], s.queries[lane, :, 0], shape)
        got = (got16[lane, :, 0].astype(np.uint32) << 16).view(np.float32)
        assert (np.abs(got - want) <= bound + 2.0 ** -20 * np.abs(want).max() + np.abs(want) * 2.0 ** -8 + bound * 2.0 ** -8).all(), lane


@pytest.mark.parametrize("fmt", [INT4, BF16])
def test_a_session_shares_only_what_is_worth_it(fmt):
    """By default: a pair in a large batch is not read apart, however the pair would look if all lanes shared its pages; nor is a batch
    without a group, whichever way it is asked; the step is then the plain one. A group that saves enough is, but not in a layer
    whose window leaves little of it."""
    pair = Shared(fmt, [(110, 2)], 62, suffix=20)
    session, params, attend = session_of(pair)
    session.share_prefixes(pair.batch.pointers, params)
    got16, launches = attend()
    assert launches == 2 and int(session._group_pages.max()) == 0 and int(session._lane_groups.max()) == -1
    check16(pair, got16, sorted({pair.member.index(0), 0, 63}))
    session.share_prefixes(pair.batch.pointers, params, minimum_pages=100)  # a caller's own threshold holds
    shared16, launches = attend()
    assert launches == 3 and int(session._group_pages.max()) == 110
    check16(pair, shared16, sorted({pair.member.index(0), 0, 63}))
    session.share_prefixes(pair.batch.pointers, params, minimum_pages=111)
    again16, launches = attend()
    assert launches == 2 and np.array_equal(again16, got16)
    session.close()
    pair.batch.close()

    many = Shared(fmt, [(40, 24)], 3, suffix=20)
    session, params, attend = session_of(many)
    session.kWorthLaneBytes, session.kWorthBytes = 0, 40 * many.batch.layout.bytes_per_layer_page()  # a threshold that small pools reach
    session.share_prefixes(many.batch.pointers, params)
    for shape, expected in ((None, 3), ((9.0, 0, 0, None), 3), ((0.0, 32 * 39, 0, None), 3), ((0.0, 20, 0, None), 2), ((0.0, 20, 32 * 39, None), 3)):
        got16, launches = attend(shape)
        assert launches == expected, shape
        check16(many, got16, (0, 13, 26), shape)
    session.forget_prefixes()
    assert attend()[1] == 2
    session.close()
    many.batch.close()


def test_a_captured_search_decides_on_the_gpu():
    """share_prefixes inside a capture cannot wait for its result: the groups of each replay are used as they are found."""
    s = Shared(INT4, [(6, 9)], 2, suffix=20)
    session, params, attend = session_of(s)
    session.kWorthLaneBytes, session.kWorthBytes = 0, 6 * s.batch.layout.bytes_per_layer_page()
    session.share_prefixes(s.batch.pointers, params)
    eager16, launches = attend()
    assert launches == 3
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        session.share_prefixes(s.batch.pointers, params, stream=stream)
        session.attend_device(0, s.batch.pointers, params, stream=stream)
    session.output.zero_()
    session._group_pages.zero_()
    graph.replay()
    assert np.array_equal(host16(session.output), eager16) and int(session._group_pages.max()) == 6
    del graph
    session.close()
    s.batch.close()


def test_a_search_on_any_kind_of_stream():
    """share_prefixes takes a stream as the other calls do: none, an object or a handle, the default stream's among them."""
    s = Shared(INT4, [(6, 9)], 2, suffix=20)
    session, params, attend = session_of(s)
    side = torch.cuda.Stream()
    for stream in (None, side, side.cuda_stream, torch.cuda.default_stream().cuda_stream):
        torch.cuda.synchronize()
        session.forget_prefixes()
        session.share_prefixes(s.batch.pointers, params, minimum_pages=2, stream=stream)
        torch.cuda.synchronize()
        assert int(session._group_pages.max()) == 6 and int((session._lane_groups >= 0).sum()) == 9
        got16, launches = attend()
        assert launches == 3
        check16(s, got16, (0, 10))
    session.close()
    s.batch.close()
