"""GPU: score shapes (tanh cap, sliding window with sinks, distance bias) on the streaming decode kernels, the verify
windows and the prefill tiles, against attention in 64 bits from the pages' bytes."""
import numpy as np
import pytest
import torch

from gpuhelp import dev
from richengine_b200 import lib, ops
from richengine_b200.abi import BF16, FP8E4M3, INT4, INT8
from servingcase import (DIM, FORMATS, GROUP, HEADS, PAGE, SLOPES, Batch, check_rows, host16, make_queries, shape_of, shuffled_pages)

pytestmark = pytest.mark.gpu

SHAPES = {
    "cap": (3.0, 0, 0, None),
    "wide cap": (1.0e5, 0, 0, None),
    "window 1": (0.0, 1, 0, None),
    "window 32": (0.0, 32, 0, None),
    "window 33, sinks": (0.0, 33, 5, None),
    "window 200, sinks over pages": (0.0, 200, 70, None),
    "window past everything": (0.0, 2 ** 32 - 1, 2 ** 32 - 1, None),
    "bias": (0.0, 0, 0, SLOPES),
    "all": (5.0, 100, 33, SLOPES),
}
CONTEXTS = [0, 31, 32, 700, 64, 1055]


def decode(batch, committed, queries, shape, ctas=0, fill=float("nan"), params=None):
    runner = ops.DecodeAttention(batch.layout, 24, batch.lanes, batch.storage.window(), ctas)
    runner.partials.fill_(fill)
    runner.statistics.fill_(fill)
    q = dev(queries)
    out = torch.zeros(q.shape, dtype=torch.bfloat16, device="cuda")
    out32 = torch.zeros(q.shape, dtype=torch.float32, device="cuda")
    runner.run(q, out, batch.pointers, params if params is not None else batch.params(committed), batch.layer, output_f32=out32, shape=shape)
    runner.status()
    runner.close()
    return host16(out), out32.cpu().numpy()


def prepared(fmt, contexts, rows=1, seed=5):
    rng = np.random.default_rng(seed)
    batch = Batch(fmt, shuffled_pages(rng, [-(-(c + rows) // PAGE) for c in contexts]), seed)
    return batch, make_queries(rng, len(contexts), HEADS, 32, GROUP, DIM)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("name", SHAPES)
def test_decode(fmt, name):
    batch, q = prepared(fmt, CONTEXTS)
    shape = SHAPES[name]
    for ctas in (0, 3):
        got16, got32 = decode(batch, CONTEXTS, q, shape_of(shape), ctas)
        for lane, context in enumerate(CONTEXTS):
            want, bound = batch.attend(lane, context, q[lane, :, 0], shape)
            check_rows(got32[lane, :, 0], got16[lane, :, 0], want, bound, f"{name}, lane {lane}, ctas {ctas}")
        assert not got16[:, :, 1:].any()
    batch.close()


@pytest.mark.parametrize("fmt", FORMATS)
def test_an_empty_shape_changes_nothing(fmt):
    batch, q = prepared(fmt, CONTEXTS)
    plain16, plain32 = decode(batch, CONTEXTS, q, None)
    got16, got32 = decode(batch, CONTEXTS, q, ops.ScoreShape())
    assert np.array_equal(plain16, got16) and np.array_equal(plain32, got32)
    batch.close()


@pytest.mark.parametrize("fmt", FORMATS)
def test_unseen_tokens_may_hold_anything(fmt):
    """Everything outside the window and the sinks, on seen pages too, and everything behind the last token is 0xFF:
    NaN where the format has one, NaN scales elsewhere."""
    context, window, sinks = 500, 77, 37
    batch, q = prepared(fmt, [context])
    seen = [t for t in range(len(batch.pages[0]) * PAGE) if t <= context and (t > context - window or t < sinks)]
    kept = {}
    keys_shape = {INT4: (HEADS, PAGE, DIM // 2), BF16: (HEADS, PAGE, DIM * 2)}.get(fmt, (HEADS, PAGE, DIM))
    for t in range(len(batch.pages[0]) * PAGE):
        if t in seen:
            continue
        page, at = batch.pages[0][t // PAGE], t % PAGE
        keys, key_scales, values, value_scales = (batch.host.tensor_view(page, 0, i) for i in range(4))
        keys.reshape(keys_shape)[:, at] = 0xff
        if fmt == INT4:
            values.reshape(keys_shape)[:, at] = 0xff
        else:
            values.reshape(HEADS, DIM, PAGE, -1)[:, :, at] = 0xff
        if fmt != BF16:
            key_scales.view(np.uint32).reshape(HEADS, PAGE)[:, at] = 0xffffffff
            value_scales.view(np.uint32).reshape(HEADS, PAGE)[:, at] = 0xffffffff
    batch.upload()
    shape = (20.0, window, sinks, SLOPES)
    want, bound = batch.attend(0, context, q[0, :, 0], shape)
    got16, got32 = decode(batch, [context], q, shape_of(shape))
    check_rows(got32[0, :, 0], got16[0, :, 0], want, bound, "decode")
    # the same row as the only live one of a verify window and of a prefill chunk
    got16, got32 = verify(batch, [context], 1, 8, q, shape_of(shape), splits=3)
    check_rows(got32[0, :, 0], got16[0, :, 0], want, bound, "verify")
    got16, got32 = prefill(batch, context, 1, q[0], shape_of(shape), splits=2)
    check_rows(got32[:, 0], got16[:, 0], want, bound, "prefill")
    batch.close()


@pytest.mark.parametrize("fmt", FORMATS)
def test_the_last_position_of_the_longest_context(fmt):
    """A table of 8 192 entries over a few pages: offsets past 32 bits of scores and of distance, windows at the far end."""
    rng = np.random.default_rng(2)
    committed = 262143
    batch = Batch(fmt, [list(rng.integers(0, 60, 8192))], 2)
    q = make_queries(rng, 1, HEADS, 32, GROUP, DIM)
    for shape in ((0.0, 129, 3, SLOPES), (7.0, 4001, 0, None)):
        want, bound = batch.attend(0, committed, q[0, :, 0], shape)
        got16, got32 = decode(batch, [committed], q, shape_of(shape))
        check_rows(got32[0, :, 0], got16[0, :, 0], want, bound, "decode")
    batch.close()


@pytest.mark.parametrize("fmt", [INT4, BF16])
def test_idle_and_refused_lanes_are_left_as_they_are(fmt):
    batch, q = prepared(fmt, [100, 200, 300])
    params = batch.params([100, 200, 300], rows=[1, 0, 1])
    runner_shape = shape_of((0.0, 50, 4, None))
    got16, got32 = decode(batch, [100, 200, 300], q, runner_shape, params=params)
    assert not got16[1].any() and not got32[1].any()
    for lane, context in ((0, 100), (2, 300)):
        want, bound = batch.attend(lane, context, q[lane, :, 0], (0.0, 50, 4, None))
        check_rows(got32[lane, :, 0], got16[lane, :, 0], want, bound, f"lane {lane}")
    batch.close()


@pytest.mark.parametrize("fmt", [INT4, FP8E4M3])
def test_many_lanes_and_large_scores(fmt):
    """More lanes than CTAs; scores far past the cap (the tanh saturates) and a scale of the caller's own."""
    rng = np.random.default_rng(9)
    contexts = [int(c) for c in rng.integers(0, 90, 200)]
    batch, q = prepared(fmt, contexts, seed=9)
    runner = batch.params(contexts, score_scale=0.5)
    shape = (15.0, 40, 2, SLOPES)
    got16, got32 = decode(batch, contexts, q, shape_of(shape), params=runner)
    for lane in range(0, 200, 7):
        want, bound = batch.attend(lane, contexts[lane], q[lane, :, 0], shape, scale=0.5)
        check_rows(got32[lane, :, 0], got16[lane, :, 0], want, bound, f"lane {lane}")
    batch.close()


# ---- verify windows -------------------------------------------------------------------------------------------------

def verify(batch, committed, rows, capacity, queries, shape, splits):
    params = batch.params(committed, rows, capacity, splits)
    slots = batch.lanes * HEADS * splits * capacity * GROUP
    partials = torch.full((slots * DIM,), float("nan"), device="cuda")
    statistics = torch.full((slots * 2,), float("nan"), device="cuda")
    q = dev(queries)
    out, out32 = torch.zeros(q.shape, dtype=torch.bfloat16, device="cuda"), torch.zeros(q.shape, dtype=torch.float32, device="cuda")
    runner = ops.VerifyWindowAttention(batch.layout, 24, batch.storage.window())
    runner.split(batch.lanes, capacity, splits, q, partials, statistics, batch.pointers, None, params, batch.layer, shape=shape)
    ops.attention_verify_reduce(batch.layout, 24, batch.lanes, capacity, partials, statistics, out, params, output_f32=out32)
    runner.check()
    runner.close()
    return host16(out), out32.cpu().numpy()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("name", SHAPES)
@pytest.mark.parametrize("rows,capacity,splits", [(8, 8, 1), (11, 16, 3), (16, 16, 9), (1, 8, 4)])
def test_verify(fmt, name, rows, capacity, splits):
    contexts = [0, 31, 300, 64]
    batch, q = prepared(fmt, contexts, rows)
    shape = SHAPES[name]
    got16, got32 = verify(batch, contexts, rows, capacity, q, shape_of(shape), splits)
    for lane, context in enumerate(contexts):
        for r in sorted({0, rows // 2, rows - 1}):
            want, bound = batch.attend(lane, context + r, q[lane, :, r], shape)
            check_rows(got32[lane, :, r], got16[lane, :, r], want, bound, f"{name}, lane {lane}, row {r}")
    assert not got16[:, :, rows:].any()
    batch.close()


@pytest.mark.parametrize("fmt", [INT4, BF16])
def test_verify_of_many_lanes(fmt):
    """1 920 tiles, heads and splits: more per SM than it plans at a time, lanes without rows and splits without pages
    among them."""
    rng = np.random.default_rng(12)
    contexts = [int(c) for c in rng.integers(0, 150, 160)]
    rows = [int(r) for r in rng.integers(0, 9, 160)]
    batch, q = prepared(fmt, contexts, 8, seed=12)
    shape = (9.0, 60, 3, SLOPES)
    got16, got32 = verify(batch, contexts, rows, 8, q, shape_of(shape), 3)
    for lane in range(0, 160, 9):
        for r in sorted({0, rows[lane] - 1} & set(range(8))):
            if r < rows[lane]:
                want, bound = batch.attend(lane, contexts[lane] + r, q[lane, :, r], shape)
                check_rows(got32[lane, :, r], got16[lane, :, r], want, bound, f"lane {lane}, row {r}")
    for lane in range(160):
        assert not got16[lane, :, rows[lane]:].any()
    batch.close()


# ---- prefill tiles --------------------------------------------------------------------------------------------------

def prefill(batch, committed, rows, queries, shape, splits):
    """queries [head][stride][group][dim] bf16 bits."""
    stride = queries.shape[1]
    params = lib.PrefillParams(committed, rows, stride, len(batch.pages[0]), batch.layer, splits, 0.0)
    tiles = -(-rows // 8)
    slots = tiles * HEADS * splits * 8 * GROUP
    partials = torch.full((slots * DIM,), float("nan"), device="cuda")
    statistics = torch.full((slots * 2,), float("nan"), device="cuda")
    q = dev(queries)
    out, out32 = torch.zeros(q.shape, dtype=torch.bfloat16, device="cuda"), torch.zeros(q.shape, dtype=torch.float32, device="cuda")
    runner = ops.VerifyWindowAttention(batch.layout, 24, batch.storage.window())
    runner.prefill_split(q, partials, statistics, batch.tables[0], params, shape=shape)
    ops.attention_prefill_reduce(batch.layout, 24, partials, statistics, out, params, output_f32=out32)
    runner.check()
    runner.close()
    return host16(out), out32.cpu().numpy()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("name", SHAPES)
@pytest.mark.parametrize("committed,rows,splits", [(0, 1, 4), (0, 33, 1), (170, 21, 3), (300, 100, 1), (77, 8, 5)])
def test_prefill(fmt, name, committed, rows, splits):
    batch, _ = prepared(fmt, [committed], rows)
    q = make_queries(np.random.default_rng(rows), HEADS, -(-rows // 32) * 32, GROUP, DIM)
    shape = SHAPES[name]
    got16, got32 = prefill(batch, committed, rows, q, shape_of(shape), splits)
    for r in sorted({0, 7, 8, rows // 2, rows - 1} & set(range(rows))):
        want, bound = batch.attend(0, committed + r, q[:, r], shape)
        check_rows(got32[:, r], got16[:, r], want, bound, f"{name}, row {r}")
    batch.close()


@pytest.mark.parametrize("fmt", [INT8, FP8E4M3])
def test_prefill_of_many_tiles(fmt):
    """1 280 tiles, heads and splits: more per SM than it plans at a time."""
    committed, rows, shape = 90, 320, (0.0, 70, 2, SLOPES)
    batch, _ = prepared(fmt, [committed], rows)
    q = make_queries(np.random.default_rng(3), HEADS, rows, GROUP, DIM)
    got16, got32 = prefill(batch, committed, rows, q, shape_of(shape), splits=8)
    for r in range(0, rows, 29):
        want, bound = batch.attend(0, committed + r, q[:, r], shape)
        check_rows(got32[:, r], got16[:, r], want, bound, f"row {r}")
    batch.close()


@pytest.mark.parametrize("shift16,shift32", [(1, 0), (0, 1), (3, 2)])
def test_merges_into_rows_at_any_address(shift16, shift32):
    """Outputs that start between the words the merge would like to write: the same bits."""
    contexts, rows, splits = [0, 100, 333], 5, 4
    batch, _ = prepared(INT4, contexts, rows)
    params = batch.params(contexts, rows, 8, splits)
    prefill_params = lib.PrefillParams(100, 21, 32, 8, batch.layer, splits, 0.0)
    generator = torch.Generator("cuda").manual_seed(1)
    partials = torch.randn(3 * HEADS * splits * 8 * GROUP * DIM, device="cuda", generator=generator)
    statistics = torch.rand(3 * HEADS * splits * 8 * GROUP * 2, device="cuda", generator=generator)
    for shape, merge in (((3, HEADS, 32, GROUP, DIM), lambda o, f: ops.attention_verify_reduce(batch.layout, 24, 3, 8, partials, statistics, o, params, output_f32=f)),
                         ((HEADS, 32, GROUP, DIM), lambda o, f: ops.attention_prefill_reduce(batch.layout, 24, partials, statistics, o, prefill_params, output_f32=f))):
        size, results = int(np.prod(shape)), []
        for a, b in ((0, 0), (shift16, shift32)):
            out, out32 = torch.zeros(size + 8, dtype=torch.bfloat16, device="cuda"), torch.zeros(size + 8, device="cuda")
            merge(out[a:a + size].view(shape), out32[b:b + size].view(shape))
            assert not out[:a].any() and not out[a + size:].any() and not out32[:b].any() and not out32[b + size:].any()
            results.append((out[a:a + size].clone(), out32[b:b + size].clone()))
        assert torch.equal(results[0][0], results[1][0]) and torch.equal(results[0][1], results[1][1]) and results[0][1].any()
    batch.close()


def test_refusals():
    batch, q = prepared(INT4, [40], 8)
    shape = ops.ScoreShape(softcap=10.0)
    runner = ops.VerifyWindowAttention(batch.layout, 24, batch.storage.window())
    scratch, masks = torch.zeros(8, device="cuda"), torch.zeros(16, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="chain windows"):
        runner.split(1, 8, 1, scratch, scratch, scratch, batch.pointers, masks, scratch, batch.layer, shape=shape)
    with pytest.raises(lib.RichKvError, match="rk_attention_decode_shaped"):
        runner.split(1, 1, 1, scratch, scratch, scratch, batch.pointers, None, scratch, batch.layer, shape=shape)
    with pytest.raises(ValueError, match="24 query heads"):
        decode(batch, [40], q, ops.ScoreShape(slopes=torch.ones(23, device="cuda")))
    for slopes in (torch.ones(24), torch.ones(24, dtype=torch.float64, device="cuda"), torch.ones(24, 2, device="cuda")[:, 0]):
        with pytest.raises(ValueError, match="slopes"):
            ops.ScoreShape(slopes=slopes)
    runner.close()
    batch.close()


# ---- queries that are no numbers ------------------------------------------------------------------------------------

@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("shape", [None, (0.0, 0, 0, None), (20.0, 0, 0, None), (256.0, 50, 3, SLOPES), (1.0e4, 0, 0, None)])
def test_a_query_row_that_is_no_number_comes_out_as_zeros(fmt, shape):
    """One element of one query head is NaN: that row is zeros, with a shape and without, and its neighbours (the other head of its
    pair, the other rows of its tile) are what they are without it."""
    contexts, head, sibling = [40, 700, 333], 2, 5
    batch, q = prepared(fmt, contexts, 8)
    block = None if shape is None else shape_of(shape)
    clean = q.copy()
    q[1, head, 0, sibling, 7] = 0x7fc0
    got16, got32 = decode(batch, contexts, q, block)
    for lane, context in enumerate(contexts):
        want, bound = batch.attend(lane, context, clean[lane, :, 0], shape)
        if lane == 1:
            assert not got16[lane, head, 0, sibling].any() and not got32[lane, head, 0, sibling].any()
            got16[lane, head, 0, sibling], got32[lane, head, 0, sibling] = 0, want[head, sibling]
            assert np.isfinite(got32).all()
            check_rows(got32[lane, :, 0], None, want, bound, f"lane {lane}")
        else:
            check_rows(got32[lane, :, 0], got16[lane, :, 0], want, bound, f"lane {lane}")
    if shape is None:
        batch.close()
        return
    # row 3 of an eight-row window, and of a prefill chunk
    q = clean.copy()
    q[1, head, 3, sibling, 200] = 0xffc0
    got16, got32 = verify(batch, contexts, 8, 8, q, block, splits=3)
    chunk16, chunk32 = prefill(Lane(batch, 1), contexts[1], 8, q[1], block, splits=1)
    for r in range(8):
        want, bound = batch.attend(1, contexts[1] + r, clean[1, :, r], shape)
        for row32, row16, what in ((got32[1, :, r], got16[1, :, r], "verify"), (chunk32[:, r], chunk16[:, r], "prefill")):
            if r == 3:
                assert not row16[head, sibling].any() and not row32[head, sibling].any(), what
                row32[head, sibling] = want[head, sibling]
            check_rows(row32, None, want, bound, f"{what}, row {r}")
    batch.close()


class Lane:
    """One lane of a batch as a batch of its own, for `prefill`."""

    def __init__(self, batch, lane):
        self.layout, self.layer, self.storage = batch.layout, batch.layer, batch.storage
        self.pages, self.tables = [batch.pages[lane]], [batch.tables[lane]]


@pytest.mark.parametrize("fmt", [INT4, BF16])
@pytest.mark.parametrize("cap", [1.0, 63.0, 64.0, 65.0, 255.0, 256.0, 257.0])
@pytest.mark.parametrize("reach", [0.05, 3.0])
def test_caps_on_both_sides_of_the_switch(fmt, cap, reach):
    """Scores far below the cap and past it, of both signs, at caps around the one where the form of the tanh changes. The form for the
    smaller caps is off by at most cap * 2^-19.7 on a score, which moves a weight by that and the row by twice that of its largest
    value; the other by 10^-6 of the score, which the bound of every row allows."""
    contexts = [300, 64]
    batch, q = prepared(fmt, contexts, 8)
    scale = 2.0 ** round(np.log2(reach * cap / 48))  # the largest of a row's scores q.k is near 48
    shape = (cap, 0, 0, None)
    for lane, context in enumerate(contexts):
        largest = max(np.abs(v).max() for v in [batch.rows(lane, range(context + 1))[1]])
        slack = 2 * cap * 2.0 ** -19.7 * largest if cap <= 64 else 0.0
        params = batch.params(contexts, score_scale=scale)
        got16, got32 = decode(batch, contexts, q, shape_of(shape), params=params)
        want, bound = batch.attend(lane, context, q[lane, :, 0], shape, scale)
        check_rows(got32[lane, :, 0], got16[lane, :, 0], want, bound + slack, f"decode, lane {lane}")
        plain_params = batch.params
        batch.params = lambda *arguments: plain_params(*arguments, score_scale=scale)
        got16, got32 = verify(batch, contexts, 8, 8, q, shape_of(shape), 2)
        batch.params = plain_params
        for r in (0, 7):
            want, bound = batch.attend(lane, context + r, q[lane, :, r], shape, scale)
            check_rows(got32[lane, :, r], got16[lane, :, r], want, bound + slack, f"verify, lane {lane}, row {r}")
    batch.close()


@pytest.mark.parametrize("fmt", FORMATS)
def test_negative_slopes(fmt):
    """Slopes of either sign, the far tokens favoured by half of the heads."""
    slopes = [(-1.0) ** h * 2.0 ** (-4 - h / 8) for h in range(24)]
    contexts = [500, 31, 1055]
    batch, q = prepared(fmt, contexts, 8)
    for shape in ((0.0, 0, 0, slopes), (20.0, 300, 40, slopes)):
        block = shape_of(shape)
        got16, got32 = decode(batch, contexts, q, block)
        window16, window32 = verify(batch, contexts, 8, 8, q, block, 3)
        chunk16, chunk32 = prefill(Lane(batch, 0), contexts[0], 8, q[0], block, 1)
        for lane, context in enumerate(contexts):
            want, bound = batch.attend(lane, context, q[lane, :, 0], shape)
            check_rows(got32[lane, :, 0], got16[lane, :, 0], want, bound, f"decode, lane {lane}")
            for r in (0, 7):
                want, bound = batch.attend(lane, context + r, q[lane, :, r], shape)
                check_rows(window32[lane, :, r], window16[lane, :, r], want, bound, f"verify, lane {lane}, row {r}")
                if lane == 0:
                    check_rows(chunk32[:, r], chunk16[:, r], want, bound, f"prefill, row {r}")
    batch.close()
