"""What the serving-step entry points refuse before anything is launched: argument checks on the host, no GPU needed."""
import ctypes as C

import pytest
import torch

from richengine_b200 import abi, lib, ops

POOL = lib.StepPool(1 << 30, 1 << 20, 128, 1000)


def step_tables(pool=POOL, lanes=4, table_pages=8, capacity=1, splits=1, missing=None):
    arrays = [16 * (i + 1) for i in range(11)]  # never followed
    if missing is not None:
        arrays[missing] = None
    layout = lib.StepLayout(pool, lanes, table_pages, capacity, splits, 0.0, 0) if pool else None
    return lib.load().rk_step_tables(layout, *arrays[:5], lib.StepOutputs(*arrays[5:]), None)


@pytest.mark.parametrize("change", [dict(lanes=0), dict(lanes=1025), dict(table_pages=0), dict(capacity=0), dict(capacity=17), dict(splits=0),
                                    dict(splits=129), dict(pool=None), dict(pool=lib.StepPool(0, 1 << 20, 128, 10)),
                                    dict(pool=lib.StepPool(1 << 30, 12345, 128, 10)), dict(pool=lib.StepPool((1 << 30) + 1, 1 << 20, 128, 10)),
                                    dict(pool=lib.StepPool(1 << 30, 1 << 20, 16385, 10)), dict(pool=lib.StepPool(1 << 30, 1 << 20, 0, 10)),
                                    dict(pool=lib.StepPool(1 << 30, 1 << 20, 128, 0))] + [dict(missing=i) for i in range(11) if i != 4])
def test_step_tables(change):
    assert step_tables(**change) == lib.INVALID
    assert b"rk_step_tables" in lib.load().rk_last_error()


@pytest.mark.parametrize("arguments", [(0, 16, 32, 2, 1, 48, 64), (1025, 16, 32, 2, 1, 48, 64), (4, 16, 32, 1, 1, 48, 64), (4, 16, 32, 2, 0, 48, 64),
                                       (4, None, 32, 2, 1, 48, 64), (4, 16, None, 2, 1, 48, 64), (4, 16, 32, 2, 1, None, 64),
                                       (4, 16, 32, 2, 1, 48, None), (4, 16, 32, 2, 1, 48, 48)])
def test_prefix_groups(arguments):
    assert lib.load().rk_prefix_groups(*arguments, None) == lib.INVALID
    assert b"rk_prefix_groups" in lib.load().rk_last_error()


BAD_SHAPES = [lib.ScoreShape(-1.0, 0, 0, 0, None), lib.ScoreShape(float("nan"), 0, 0, 0, None), lib.ScoreShape(float("inf"), 0, 0, 0, None),
              lib.ScoreShape(1.0e-35, 0, 0, 0, None)]


@pytest.mark.parametrize("shape", BAD_SHAPES + [None])
def test_shapes(shape):
    library, layer = lib.load(), lib.KvLayer(128, 0)
    block = C.byref(shape) if shape is not None else None
    plan, prefill = lib.DecodePlan(4, 148, 152), lib.PrefillParams(0, 8, 32, 1, layer, 1, 0.0)
    assert library.rk_attention_decode_shaped(16, C.byref(plan), abi.INT4, 16, 16, None, 16, 16, 16, 16, 16, layer, block, None) == lib.INVALID
    assert library.rk_attention_verify_split_shaped(16, abi.INT4, 4, 24, 256, 1, 8, 1, 16, 16, 16, 16, 16, layer, block, 16, None) == lib.INVALID
    assert library.rk_attention_prefill_split_shaped(16, abi.INT4, 4, 24, 256, 16, 16, 16, 16, C.byref(prefill), block, 16, None) == lib.INVALID
    if shape is not None:
        shared, buffers = lib.SharedPlan(plan, 148), lib.SharedBuffers(16, 16, 16, 16, 16, 16)
        assert library.rk_attention_decode_shared(16, C.byref(shared), abi.INT4, 16, 16, None, C.byref(buffers), 16, 16, layer, 16, 16, block,
                                                  None) == lib.INVALID


def test_one_row_is_the_streaming_kernels_business():
    shape = lib.ScoreShape(1.0, 0, 0, 0, None)
    assert lib.load().rk_attention_verify_split_shaped(16, abi.INT4, 4, 24, 256, 1, 1, 1, 16, 16, 16, 16, 16, lib.KvLayer(128, 0), C.byref(shape), 16,
                                                       None) == lib.UNSUPPORTED


def test_shared_plan_and_missing_arguments():
    library, plan = lib.load(), lib.SharedPlan()
    assert library.rk_shared_plan_make(abi.INT4, 4, 24, 256, 64, 148, C.byref(plan)) == lib.OK
    assert plan.decode.lanes == 64 and plan.prefix_ctas == 148 and plan.prefix_partials_bytes == 148 * 128 * 1024
    assert library.rk_shared_plan_make(abi.INT4, 4, 24, 256, 1024, 4, C.byref(plan)) == lib.OK
    assert plan.prefix_partials_bytes == 1024 * 24 * 1024 and plan.prefix_descriptor_bytes == 1024 * 16
    assert library.rk_shared_plan_make(abi.INT4, 4, 24, 256, 1025, 4, C.byref(plan)) == lib.INVALID
    assert library.rk_shared_plan_make(abi.INT4, 8, 24, 256, 8, 4, C.byref(plan)) == lib.UNSUPPORTED
    assert library.rk_shared_plan_make(abi.INT4, 4, 24, 256, 8, 4, None) == lib.INVALID
    assert library.rk_shared_plan_make(abi.INT4, 4, 24, 256, 8, 4, C.byref(plan)) == lib.OK
    good = [16, C.byref(plan), abi.INT4, 16, 16, None, C.byref(lib.SharedBuffers(16, 16, 16, 16, 16, 16)), 16, 16, lib.KvLayer(128, 0), 16, 16, None, None]
    for at, bad in [(0, None), (1, None), (2, 9), (3, None), (4, None), (6, None), (7, None), (8, None), (9, lib.KvLayer(0, 0)), (10, None), (11, None)] + \
            [(6, C.byref(lib.SharedBuffers(*(None if i == j else 16 for i in range(6))))) for j in range(6)]:
        arguments = list(good)
        arguments[at] = bad
        assert library.rk_attention_decode_shared(*arguments) == lib.INVALID, at
        assert b"rk_attention_decode_shared" in library.rk_last_error()


# What each entry moves 16 (8) bytes at a time, by the position of its argument; a window of zeros that nothing looks at.
WINDOW = C.create_string_buffer(8192)


def attention_calls():
    library, layer, shape = lib.load(), lib.KvLayer(128, 0), lib.ScoreShape(0.0, 9, 0, 0, None)
    plan, prefill = lib.DecodePlan(4, 148, 152), lib.PrefillParams(0, 8, 32, 1, layer, 1, 0.0)
    shared = lib.SharedPlan(plan, 148)
    return {
        "rk_attention_decode": (library.rk_attention_decode, [WINDOW, C.byref(plan), abi.INT4, 32, 32, 32, 32, 32, 32, 32, 32, layer, None],
                                (3, 5, 6), (4, 7, 8, 9)),
        "rk_attention_decode_shaped": (library.rk_attention_decode_shaped, [WINDOW, C.byref(plan), abi.INT4, 32, 32, 32, 32, 32, 32, 32, 32, layer,
                                                                            C.byref(shape), None], (3, 5, 6), (4, 7, 8, 9)),
        "rk_attention_verify_split_shaped": (library.rk_attention_verify_split_shaped, [WINDOW, abi.INT4, 4, 24, 256, 1, 8, 1, 32, 32, 32, 32, 32, layer,
                                                                                        C.byref(shape), 32, None], (8, 9), (10, 11)),
        "rk_attention_prefill_split_shaped": (library.rk_attention_prefill_split_shaped, [WINDOW, abi.INT4, 4, 24, 256, 32, 32, 32, 32, C.byref(prefill),
                                                                                          C.byref(shape), 32, None], (5, 6), (7, 8)),
        "rk_attention_decode_shared": (library.rk_attention_decode_shared, [WINDOW, C.byref(shared), abi.INT4, 32, 32, 32, [32] * 6, 32, 32, layer, 32, 32,
                                                                            None, None], (3, 5, (6, 0), (6, 3), (6, 5)), (4, (6, 1), (6, 2), (6, 4), 7)),
    }


@pytest.mark.parametrize("name", ["rk_attention_decode", "rk_attention_decode_shaped", "rk_attention_verify_split_shaped",
                                  "rk_attention_prefill_split_shaped", "rk_attention_decode_shared"])
def test_addresses_between_words_are_refused(name):
    """A tensor that starts between the words its kernel moves would be a fault on the device: refused on the host, whichever it is."""
    call, arguments, sixteens, eights = attention_calls()[name]
    for positions, offsets in ((sixteens, (2, 4, 8)), (eights, (2, 4))):
        for at in positions:
            for offset in offsets:
                changed = [list(a) if isinstance(a, list) else a for a in arguments]
                if isinstance(at, tuple):
                    changed[at[0]][at[1]] += offset
                else:
                    changed[at] += offset
                changed = [C.byref(lib.SharedBuffers(*a)) if isinstance(a, list) else a for a in changed]
                assert call(*changed) == lib.INVALID, (at, offset)
                text = lib.load().rk_last_error()
                assert text.startswith(name.encode() + b":") and b"boundaries" in text


def test_block_sizes():
    assert C.sizeof(lib.ScoreShape) == 24 and lib.ScoreShape.slopes.offset == 16
    assert C.sizeof(lib.StepPool) == 24 and C.sizeof(lib.SharedPlan) == C.sizeof(lib.DecodePlan) + 32


def test_python_shapes():
    for bad in (dict(softcap=-1.0), dict(softcap=float("inf")), dict(softcap=float("nan")), dict(window=-1), dict(window=2 ** 32), dict(sink_tokens=-1)):
        with pytest.raises(ValueError, match="ScoreShape"):
            ops.ScoreShape(**bad)
    with pytest.raises(ValueError, match="slopes"):
        ops.ScoreShape(slopes=torch.ones(24))
