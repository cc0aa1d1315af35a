"""Kernel entry points over torch device tensors (thin: pointers and sizes only).

Buffer layouts are the reference kernels' (runtime/metal/kernels/decode/
paged_attention_store.metal:32-35, decode/paged_attention.metal:39-47):
  chunk_keys   bf16 [lane][kv_head][stride][D]
  chunk_values bf16 [lane][kv_head][D][stride]          (dimension-major)
  queries/out  bf16 [lane][kv_head][stride][group][D]
  tables       one device array of uint64 entries per lane; `table_pointers`
               is a device array of their addresses
  params       device array of the 24/36-byte parameter blocks, one per lane
torch is used for device memory and streams only.
"""
from __future__ import annotations

import ctypes as C

import numpy as np
import torch

from . import lib
from .abi import CHUNK_PARAMS, TREE_NODES, VERIFY_PARAMS, Layout


def _stream(stream) -> int:
    if stream is None:  # the current stream's handle without a Stream object around it: 0.3 us of a call instead of 3.2
        return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device())
    return stream.cuda_stream if hasattr(stream, "cuda_stream") else int(stream)


def params_to_device(array: np.ndarray, device="cuda") -> torch.Tensor:
    """Uploads a numpy structured array of parameter blocks as raw bytes."""
    raw = np.ascontiguousarray(array).view(np.uint8).reshape(-1)
    return torch.from_numpy(raw.copy()).to(device)


def table_pointer_array(tables, device="cuda") -> torch.Tensor:
    return torch.tensor([t.data_ptr() for t in tables], dtype=torch.int64, device=device)


def store_verify(layout: Layout, chunk_keys, chunk_values, table_pointers, params, layer: lib.KvLayer,
                 lanes: int, max_rows: int, stream=None) -> None:
    status = lib.load().rk_store_verify(layout.format, layout.kv_heads, layout.head_dimension, lanes, max_rows,
                                        chunk_keys.data_ptr(), chunk_values.data_ptr(), table_pointers.data_ptr(),
                                        params.data_ptr(), layer, _stream(stream))
    lib.check(status, "rk_store_verify")


def store_chunk(layout: Layout, chunk_keys, chunk_values, table, params: lib.ChunkParams, stream=None) -> None:
    status = lib.load().rk_store_chunk(layout.format, layout.kv_heads, layout.head_dimension, chunk_keys.data_ptr(),
                                       chunk_values.data_ptr(), table.data_ptr(), C.byref(params), _stream(stream))
    lib.check(status, "rk_store_chunk")


def attention_verify_split(layout: Layout, query_heads: int, lanes: int, row_capacity: int, grid_splits: int,
                           queries, partials, statistics, table_pointers, row_masks, params, layer: lib.KvLayer,
                           stream=None) -> None:
    status = lib.load().rk_attention_verify_split(
        layout.format, layout.kv_heads, query_heads, layout.head_dimension, lanes, row_capacity, grid_splits,
        queries.data_ptr(), partials.data_ptr(), statistics.data_ptr(), table_pointers.data_ptr(),
        row_masks.data_ptr() if row_masks is not None else None, params.data_ptr(), layer, _stream(stream))
    lib.check(status, "rk_attention_verify_split")


class ScoreShape:
    """What a score goes through before the softmax (rk_score_shape): `softcap` * tanh(score / softcap), minus slope *
    distance per query head, seen only inside a sliding `window` (the first `sink_tokens` stay visible beside it)."""

    def __init__(self, softcap: float = 0.0, window: int = 0, sink_tokens: int = 0, slopes=None):
        if not 0.0 <= softcap < float("inf"):
            raise ValueError("ScoreShape: softcap must be finite and not negative")
        if not 0 <= window < 2 ** 32 or not 0 <= sink_tokens < 2 ** 32:
            raise ValueError("ScoreShape: window and sink_tokens are counts of tokens")
        if slopes is not None and (slopes.dtype != torch.float32 or not slopes.is_cuda or not slopes.is_contiguous() or slopes.dim() != 1):
            raise ValueError("ScoreShape: slopes is a contiguous fp32 device vector, one per query head")
        self.softcap, self.window, self.sink_tokens, self.slopes = softcap, window, sink_tokens, slopes

        self._block = lib.ScoreShape(softcap, window, sink_tokens, 0, slopes.data_ptr() if slopes is not None else None)

    def block(self, query_heads: int) -> lib.ScoreShape:
        """The C block; `slopes` stays alive with this object."""
        if self.slopes is not None and self.slopes.numel() != query_heads:
            raise ValueError(f"ScoreShape: {self.slopes.numel()} slopes for {query_heads} query heads")
        return self._block


class VerifyWindowAttention:
    """8/16-row int4 verify windows on the tcgen05 split kernel (rk_attention_verify_split_tc).

    Holds the pool window's tensor maps and the status word; partials and statistics stay the
    caller's, in the layout of attention_verify_split, and attention_verify_reduce merges them."""

    def __init__(self, layout: Layout, query_heads: int, window: tuple[int, int]):
        self._lib = lib.load()
        self.layout, self.query_heads = layout, query_heads
        self._window = self._lib.rk_window_create(window[0], window[1])
        if not self._window:
            raise lib.RichKvError(lib.INVALID, "rk_window_create")
        self.status_word = torch.zeros(1, dtype=torch.int32, device="cuda")

    def close(self) -> None:
        if self._window:
            self._lib.rk_window_destroy(self._window)
            self._window = None

    def __del__(self):
        self.close()

    def split(self, lanes: int, row_capacity: int, grid_splits: int, queries, partials, statistics, table_pointers,
              row_masks, params, layer: lib.KvLayer, stream=None, shape: ScoreShape | None = None) -> None:
        if shape is not None:  # chain windows of 8 or 16 rows
            if row_masks is not None:
                raise ValueError("a score shape goes with chain windows, not with tree masks")
            status = self._lib.rk_attention_verify_split_shaped(
                self._window, self.layout.format, self.layout.kv_heads, self.query_heads, self.layout.head_dimension,
                lanes, row_capacity, grid_splits, queries.data_ptr(), partials.data_ptr(), statistics.data_ptr(),
                table_pointers.data_ptr(), params.data_ptr(), layer, shape.block(self.query_heads),
                self.status_word.data_ptr(), _stream(stream))
            lib.check(status, "rk_attention_verify_split_shaped")
            return
        status = self._lib.rk_attention_verify_split_tc(
            self._window, self.layout.format, self.layout.kv_heads, self.query_heads, self.layout.head_dimension,
            lanes, row_capacity, grid_splits, queries.data_ptr(), partials.data_ptr(), statistics.data_ptr(),
            table_pointers.data_ptr(), row_masks.data_ptr() if row_masks is not None else None, params.data_ptr(),
            layer, self.status_word.data_ptr(), _stream(stream))
        lib.check(status, "rk_attention_verify_split_tc")

    def prefill_split(self, queries, partials, statistics, table, params: lib.PrefillParams, stream=None,
                      shape: ScoreShape | None = None) -> None:
        """The 8-row tiles of a prefill chunk (rk_attention_prefill_split_tc); merge with attention_prefill_reduce."""
        if shape is not None:
            status = self._lib.rk_attention_prefill_split_shaped(
                self._window, self.layout.format, self.layout.kv_heads, self.query_heads, self.layout.head_dimension,
                queries.data_ptr(), partials.data_ptr(), statistics.data_ptr(), table.data_ptr(), C.byref(params),
                shape.block(self.query_heads), self.status_word.data_ptr(), _stream(stream))
            lib.check(status, "rk_attention_prefill_split_shaped")
            return
        status = self._lib.rk_attention_prefill_split_tc(
            self._window, self.layout.format, self.layout.kv_heads, self.query_heads, self.layout.head_dimension,
            queries.data_ptr(), partials.data_ptr(), statistics.data_ptr(), table.data_ptr(), C.byref(params),
            self.status_word.data_ptr(), _stream(stream))
        lib.check(status, "rk_attention_prefill_split_tc")

    def check(self) -> None:
        """Synchronises and raises if a bounded wait ran out in a launched step."""
        if int(self.status_word.item()) != 0:
            raise lib.RichKvError(lib.TIMEOUT, "rk_attention_verify_split_tc: a bounded wait ran out")


class WindowDecodeAttention:
    """One-query decode on the tcgen05 window kernel (row capacity 1) + the split merge: the decode path of the
    int8, fp8 and bf16 pools (int4 has the streaming kernel, DecodeAttention). Same call shape as DecodeAttention;
    the lanes' parameters carry split_count = slot_splits = `splits`."""

    def __init__(self, layout: Layout, query_heads: int, lanes: int, window: tuple[int, int], splits: int = 1):
        self.layout, self.query_heads, self.lanes, self.splits = layout, query_heads, lanes, splits
        self.inner = VerifyWindowAttention(layout, query_heads, window)
        group = query_heads // layout.kv_heads
        slots = lanes * layout.kv_heads * splits * group
        self.partials = torch.empty(slots * layout.head_dimension, dtype=torch.float32, device="cuda")
        self.statistics = torch.empty(slots * 2, dtype=torch.float32, device="cuda")

    def close(self) -> None:
        self.inner.close()

    def run(self, queries, output, table_pointers, params, layer: lib.KvLayer, output_f32=None, stream=None) -> None:
        self.inner.split(self.lanes, 1, self.splits, queries, self.partials, self.statistics, table_pointers, None, params,
                         layer, stream)
        attention_verify_reduce(self.layout, self.query_heads, self.lanes, 1, self.partials, self.statistics, output,
                                params, output_f32, stream)

    def status(self) -> None:
        self.inner.check()


def attention_verify_reduce(layout: Layout, query_heads: int, lanes: int, row_capacity: int, partials, statistics,
                            output, params, output_f32=None, stream=None) -> None:
    status = lib.load().rk_attention_verify_reduce(
        layout.kv_heads, query_heads, layout.head_dimension, lanes, row_capacity, partials.data_ptr(),
        statistics.data_ptr(), output.data_ptr(), output_f32.data_ptr() if output_f32 is not None else None,
        params.data_ptr(), _stream(stream))
    lib.check(status, "rk_attention_verify_reduce")


def attention_prefill(layout: Layout, query_heads: int, queries, output, partials, statistics, table,
                      params: lib.PrefillParams, output_f32=None, stream=None) -> None:
    library = lib.load()
    lib.check(library.rk_attention_prefill_split(layout.format, layout.kv_heads, query_heads, layout.head_dimension,
                                                 queries.data_ptr(), partials.data_ptr(), statistics.data_ptr(),
                                                 table.data_ptr(), C.byref(params), _stream(stream)),
              "rk_attention_prefill_split")
    lib.check(library.rk_attention_prefill_reduce(layout.kv_heads, query_heads, layout.head_dimension,
                                                  partials.data_ptr(), statistics.data_ptr(), output.data_ptr(),
                                                  output_f32.data_ptr() if output_f32 is not None else None,
                                                  C.byref(params), _stream(stream)),
              "rk_attention_prefill_reduce")


def qkv_prepare(layout: Layout, query_heads: int, lanes: int, rows: int, packed_qkv, q_norm, k_norm, rope_cos, rope_sin,
                queries, chunk_keys, chunk_values, eps: float = 1e-6, stream=None) -> None:
    """Packed projection rows -> the stagings of the store and the attention (rk_qkv_prepare)."""
    status = lib.load().rk_qkv_prepare(layout.kv_heads, query_heads, layout.head_dimension, lanes, rows,
                                       packed_qkv.data_ptr(), q_norm.data_ptr(), k_norm.data_ptr(),
                                       int(q_norm.dtype == torch.float32), rope_cos.data_ptr(), rope_sin.data_ptr(), eps,
                                       queries.data_ptr(), chunk_keys.data_ptr(), chunk_values.data_ptr(), _stream(stream))
    lib.check(status, "rk_qkv_prepare")


def qkv_prepare_store(layout: Layout, query_heads: int, lanes: int, rows: int, packed_qkv, q_norm, k_norm, rope_cos,
                      rope_sin, queries, table_pointers, params, layer: lib.KvLayer, eps: float = 1e-6, stream=None) -> None:
    """The same with the page store merged in: K/V rows go straight into their page slots (rk_qkv_prepare_store)."""
    status = lib.load().rk_qkv_prepare_store(layout.format, layout.kv_heads, query_heads, layout.head_dimension, lanes, rows,
                                             packed_qkv.data_ptr(), q_norm.data_ptr(), k_norm.data_ptr(),
                                             int(q_norm.dtype == torch.float32), rope_cos.data_ptr(), rope_sin.data_ptr(),
                                             eps, queries.data_ptr(), table_pointers.data_ptr(), params.data_ptr(), layer,
                                             _stream(stream))
    lib.check(status, "rk_qkv_prepare_store")


def attention_verify_reduce_gate(layout: Layout, query_heads: int, lanes: int, row_capacity: int, partials, statistics,
                                 output, packed_qkv, hidden, params, stream=None) -> None:
    """Merge + out-projection input: hidden [lane][row][query head][D] = merged row x sigmoid(gate of packed_qkv), or
    the merged row itself when packed_qkv is None (rk_attention_verify_reduce_gate)."""
    status = lib.load().rk_attention_verify_reduce_gate(
        layout.kv_heads, query_heads, layout.head_dimension, lanes, row_capacity, partials.data_ptr(),
        statistics.data_ptr(), output.data_ptr() if output is not None else None,
        packed_qkv.data_ptr() if packed_qkv is not None else None, hidden.data_ptr(), params.data_ptr(), _stream(stream))
    lib.check(status, "rk_attention_verify_reduce_gate")


def attention_prefill_reduce(layout: Layout, query_heads: int, partials, statistics, output, params: lib.PrefillParams,
                             output_f32=None, stream=None) -> None:
    lib.check(lib.load().rk_attention_prefill_reduce(layout.kv_heads, query_heads, layout.head_dimension,
                                                     partials.data_ptr(), statistics.data_ptr(), output.data_ptr(),
                                                     output_f32.data_ptr() if output_f32 is not None else None,
                                                     C.byref(params), _stream(stream)),
              "rk_attention_prefill_reduce")


def tree_compact(layout: Layout, lanes: int, table_pointers, params, layer: lib.KvLayer, retained_path,
                 retained_count, stream=None) -> None:
    status = lib.load().rk_tree_compact(layout.format, layout.kv_heads, layout.head_dimension, lanes,
                                        table_pointers.data_ptr(), params.data_ptr(), layer,
                                        retained_path.data_ptr(), retained_count.data_ptr(), _stream(stream))
    lib.check(status, "rk_tree_compact")


def chunk_params_array(lanes: int) -> np.ndarray:
    return np.zeros(lanes, dtype=CHUNK_PARAMS)


def verify_params_array(lanes: int) -> np.ndarray:
    return np.zeros(lanes, dtype=VERIFY_PARAMS)


class DecodeAttention:
    """Streaming decode attention over one pool's address window (rk_attention_decode).

    Holds the window's tensor map and the step's scratch, sized by the plan:
    one query row per lane, row capacity 1; the lane parameter blocks and the
    page tables live on the device.
    """

    def __init__(self, layout: Layout, query_heads: int, lanes: int, window: tuple[int, int], ctas: int = 0):
        self._lib = lib.load()
        self.layout, self.query_heads, self.lanes = layout, query_heads, lanes
        self.plan = lib.DecodePlan()
        lib.check(self._lib.rk_decode_plan_make(layout.format, layout.kv_heads, query_heads, layout.head_dimension,
                                                lanes, ctas, C.byref(self.plan)), "rk_decode_plan_make")
        self._window = self._lib.rk_window_create(window[0], window[1])
        if not self._window:
            raise lib.RichKvError(lib.INVALID, "rk_window_create")
        self.partials = torch.empty(self.plan.partials_bytes // 4, dtype=torch.float32, device="cuda")
        self.statistics = torch.empty(self.plan.statistics_bytes // 4, dtype=torch.float32, device="cuda")
        self.descriptors = torch.zeros(self.plan.descriptor_bytes // 4, dtype=torch.int32, device="cuda")

    def close(self):
        if self._window:
            self._lib.rk_window_destroy(self._window)
            self._window = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def run(self, queries, output, table_pointers, params, layer: lib.KvLayer, output_f32=None, stream=None,
            shape: ScoreShape | None = None):
        if shape is not None:
            status = self._lib.rk_attention_decode_shaped(
                self._window, C.byref(self.plan), self.layout.format, queries.data_ptr(), output.data_ptr(),
                output_f32.data_ptr() if output_f32 is not None else None, self.partials.data_ptr(),
                self.statistics.data_ptr(), self.descriptors.data_ptr(), table_pointers.data_ptr(), params.data_ptr(),
                layer, shape.block(self.query_heads), _stream(stream))
            lib.check(status, "rk_attention_decode_shaped")
            return
        status = self._lib.rk_attention_decode(
            self._window, C.byref(self.plan), self.layout.format, queries.data_ptr(), output.data_ptr(),
            output_f32.data_ptr() if output_f32 is not None else None, self.partials.data_ptr(),
            self.statistics.data_ptr(), self.descriptors.data_ptr(), table_pointers.data_ptr(), params.data_ptr(),
            layer, _stream(stream))
        lib.check(status, "rk_attention_decode")

    def status(self, stream=None) -> None:
        """Raises if a bounded device wait ran out during the steps launched so far."""
        lib.check(self._lib.rk_attention_decode_status(C.byref(self.plan), self.descriptors.data_ptr(), _stream(stream)),
                  "rk_attention_decode_status")


def _int32_vector(name: str, vector, size: int | None, device) -> None:
    if vector.dtype is not torch.int32 or vector.device != device or not vector.is_contiguous() or (size is not None and vector.numel() != size):
        raise ValueError(f"{name} is a contiguous int32 vector on {device}" + (f" of {size}" if size is not None else ""))


class StepTables:
    """A step's page tables, parameter blocks and row slots, built on the GPU from request lengths (rk_step_tables).

    `window` (its base), `extent_stride`, `extent_pages` and `page_count` say where page ids lie (for_storage takes them from a
    PageStorage; others answer for the whole pool lying in the window that attention is given); build() fills `entries`, `chunk_params`, `verify_params`, `row_offsets` and `row_slots` in stream order, and the
    stores and attention kernels take `table_pointers` and the parameter blocks as they are."""

    def __init__(self, lanes: int, table_pages: int, window: tuple[int, int], extent_stride: int, extent_pages: int,
                 page_count: int, row_capacity: int = 1, split_count: int = 1, score_scale: float = 0.0):
        if lanes < 1 or table_pages < 1 or not 1 <= row_capacity <= TREE_NODES:
            raise ValueError("StepTables: lanes, table pages and a row capacity of at most 16")
        self._lib = lib.load()
        self.lanes, self.table_pages, self.row_capacity = lanes, table_pages, row_capacity
        self.split_count, self.score_scale = split_count, score_scale
        self.entries = torch.zeros((lanes, table_pages), dtype=torch.int64, device="cuda")
        self.table_pointers = self.entries.data_ptr() + 8 * table_pages * torch.arange(lanes, dtype=torch.int64, device="cuda")
        self.chunk_params = torch.zeros((lanes, CHUNK_PARAMS.itemsize), dtype=torch.uint8, device="cuda")
        self.verify_params = torch.zeros((lanes, VERIFY_PARAMS.itemsize), dtype=torch.uint8, device="cuda")
        self.row_offsets = torch.zeros(lanes + 1, dtype=torch.int32, device="cuda")
        self.row_slots = torch.zeros(lanes * row_capacity, dtype=torch.int64, device="cuda")
        self.status_word = torch.zeros(1, dtype=torch.int32, device="cuda")
        self._no_ids = torch.full((1,), -1, dtype=torch.int32, device="cuda")  # what an empty page_ids stands for: past every pool
        self._device = self.entries.device
        self._call = self._lib.rk_step_tables
        self._layout = lib.StepLayout(lib.StepPool(window[0], extent_stride, extent_pages, page_count), lanes, table_pages, row_capacity,
                                      split_count, score_scale, 0)
        self._outputs = lib.StepOutputs(*(t.data_ptr() for t in (self.entries, self.chunk_params, self.verify_params, self.row_offsets,
                                                                 self.row_slots, self.status_word)))
        torch.cuda.current_stream().synchronize()  # the fills above are done, whichever stream the first call takes

    @classmethod
    def for_storage(cls, storage, lanes: int, table_pages: int, row_capacity: int = 1, split_count: int = 1,
                    score_scale: float = 0.0) -> "StepTables":
        pool = storage.step_pool()
        return cls(lanes, table_pages, storage.window(), pool.extent_stride, pool.extent_pages, pool.page_count, row_capacity, split_count,
                   score_scale)

    def build(self, page_ids, page_offsets, committed, rows, known_pages=None, stream=None) -> None:
        """Per lane l: page ids page_ids[page_offsets[l] : page_offsets[l + 1]], committed tokens, new rows (0: idle);
        entries before known_pages[l] stay as they are, and all of an idle lane's. All int32 device vectors. A lane whose offsets
        reach past page_ids is refused like one that asks for too much."""
        lanes, device = self.lanes, self._device
        _int32_vector("page_ids", page_ids, None, device)
        _int32_vector("page_offsets", page_offsets, lanes + 1, device)
        _int32_vector("committed", committed, lanes, device)
        _int32_vector("rows", rows, lanes, device)
        if known_pages is not None:
            _int32_vector("known_pages", known_pages, lanes, device)
        if not page_ids.numel():
            page_ids = self._no_ids
        self._layout.id_count = page_ids.numel()
        status = self._call(self._layout, page_ids.data_ptr(), page_offsets.data_ptr(), committed.data_ptr(), rows.data_ptr(),
                            known_pages.data_ptr() if known_pages is not None else None, self._outputs, _stream(stream))
        lib.check(status, "rk_step_tables")

    def check(self) -> None:
        """Waits for the device (whichever streams the builds took, eagerly or in a replayed graph), raises if a lane was refused
        since the last check, and clears the word."""
        torch.cuda.synchronize(self._device)
        if int(self.status_word.item()):
            self.status_word.zero_()
            torch.cuda.current_stream(self._device).synchronize()  # a build on another stream may follow at once
            raise lib.RichKvError(lib.INVALID, "rk_step_tables: a lane asks for rows, tokens or pages it cannot have")


def prefix_groups(lanes: int, table_pointers, params, lane_groups, group_pages, minimum_lanes: int = 2, minimum_pages: int = 1,
                  stream=None) -> None:
    """Which lanes share how long a prefix, from their page tables (rk_prefix_groups): lane_groups[l] = the lowest lane
    of l's group or -1, group_pages[that lane] = the pages they share. Both int32 device vectors of `lanes`."""
    _int32_vector("lane_groups", lane_groups, lanes, table_pointers.device)
    _int32_vector("group_pages", group_pages, lanes, table_pointers.device)
    status = lib.load().rk_prefix_groups(lanes, table_pointers.data_ptr(), params.data_ptr(), minimum_lanes, minimum_pages,
                                         lane_groups.data_ptr(), group_pages.data_ptr(), _stream(stream))
    lib.check(status, "rk_prefix_groups")


class SharedPrefixDecode:
    """Decode attention for a batch in which groups of lanes share the first pages of their tables
    (rk_attention_decode_shared): a group's prefix is read once for all of its lanes. Holds the window's tensor maps and
    the step's scratch; lane_groups and group_pages are prefix_groups' output (or a caller's own in that form)."""

    def __init__(self, layout: Layout, query_heads: int, lanes: int, window: tuple[int, int], ctas: int = 0):
        self._lib = lib.load()
        self.layout, self.query_heads, self.lanes = layout, query_heads, lanes
        self.plan = lib.SharedPlan()
        self._window = None
        lib.check(self._lib.rk_shared_plan_make(layout.format, layout.kv_heads, query_heads, layout.head_dimension, lanes, ctas,
                                                C.byref(self.plan)), "rk_shared_plan_make")
        self._window = self._lib.rk_window_create(window[0], window[1])
        if not self._window:
            raise lib.RichKvError(lib.INVALID, "rk_window_create")
        decode = self.plan.decode
        self.partials = torch.empty(decode.partials_bytes // 4, dtype=torch.float32, device="cuda")
        self.statistics = torch.empty(decode.statistics_bytes // 4, dtype=torch.float32, device="cuda")
        self.descriptors = torch.zeros(decode.descriptor_bytes // 4, dtype=torch.int32, device="cuda")
        self.prefix_partials = torch.empty(self.plan.prefix_partials_bytes // 4, dtype=torch.float32, device="cuda")
        self.prefix_statistics = torch.empty(self.plan.prefix_statistics_bytes // 4, dtype=torch.float32, device="cuda")
        self.prefix_descriptors = torch.zeros(self.plan.prefix_descriptor_bytes // 4, dtype=torch.int32, device="cuda")
        self._device = self.partials.device
        self._buffers = lib.SharedBuffers(*(t.data_ptr() for t in (self.partials, self.statistics, self.descriptors, self.prefix_partials,
                                                                   self.prefix_statistics, self.prefix_descriptors)))
        torch.cuda.current_stream().synchronize()  # the fills above are done, whichever stream the first call takes

    def close(self):
        if self._window:
            self._lib.rk_window_destroy(self._window)
            self._window = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def run(self, queries, output, table_pointers, params, layer: lib.KvLayer, lane_groups, group_pages, output_f32=None,
            stream=None, shape: ScoreShape | None = None):
        _int32_vector("lane_groups", lane_groups, self.lanes, self._device)
        _int32_vector("group_pages", group_pages, self.lanes, self._device)
        block = shape.block(self.query_heads) if shape is not None else None
        status = self._lib.rk_attention_decode_shared(
            self._window, self.plan, self.layout.format, queries.data_ptr(), output.data_ptr(),
            output_f32.data_ptr() if output_f32 is not None else None, self._buffers, table_pointers.data_ptr(),
            params.data_ptr(), layer, lane_groups.data_ptr(), group_pages.data_ptr(), block, _stream(stream))
        lib.check(status, "rk_attention_decode_shared")

    def status(self, stream=None) -> None:
        """Raises if a bounded device wait ran out during the steps launched so far."""
        lib.check(self._lib.rk_attention_decode_status(C.byref(self.plan.decode), self.descriptors.data_ptr(), _stream(stream)),
                  "rk_attention_decode_shared")
