"""One decode step's worth of buffers and launches: append each lane's new K/V row and
attend its one query row over the paged history, layer by layer.

This is the step the reference encodes per attention layer as store -> split ->
reduce (runtime/ops/PagedAttention.cpp:467-545, called from
runtime/model/QwenTarget.cpp:799-812), with the lanes generalised from the
reference's four to any batch width. Two entry points:
  step_device(...)  inputs already staged on the device (what a model runtime calls);
                    (a score shape, and after share_prefixes() each shared prefix read once);
  step_host(...)    compact host rows in pinned memory in, compact host rows out
                    (copies, staging scatter and output gather inside the call).
step_host is one call into the library (rk_session_step_host, include/richkv.h): calls pipeline there — the upload
of a call's rows runs on a copy stream while the previous call's kernels run, and a call's result goes back on a
second copy stream while the next call computes. finish_host() makes the compute stream wait for the copies still
in flight.
"""
from __future__ import annotations

import ctypes as C
from collections import Counter

import torch

from . import lib, ops
from .abi import BF16, FP8E4M3, INT4, INT8, VERIFY_CHUNK_STRIDE, Layout, pages_for
from .storage import PageStorage


def _stream_handle(stream) -> int:
    return ops._stream(stream)


# What a tile of a shared prefix costs, in lanes that stream the same pages: 128 rows x 64 tokens take a CTA the same time however
# many of the rows are real (21 lanes fill them), and lanes that read the same pages by themselves find part of them in L2.
# Measured on a B200 without a score shape: int4 loses with four lanes a group (32 groups of 8K: 176 us against 148) and wins with
# six (20 groups of 8K: 124 against 146); int8 wins with four (215 against 234) and loses with three (211 against 184); fp8 loses
# with four (251 against 234) and is even with five; bf16 wins with three (301 against 337) and loses with two.
TILE_PRICE = {INT4: 4.6, INT8: 3.9, FP8E4M3: 4.2, BF16: 2.7}


def prefix_saving(layout, groups) -> float:
    """Bytes of pages a layer that reading shared prefixes once is worth; `groups`: (lanes, pages shared) of each."""
    price = TILE_PRICE[layout.format]
    tiles = (-(-lanes * 6 // 128) for lanes, _ in groups)  # six query heads a KV head
    return sum((lanes - price * t) * pages for (lanes, pages), t in zip(groups, tiles)) * layout.bytes_per_layer_page()


class DecodeSession:
    # What shared prefixes have to save a layer. The third kernel costs 7 us and the wider merge up to 13 more, growing with the lanes
    # while those are few (with many, a tile has fewer splits to merge): 8 lanes of int8 over 16K, 140 MB, win (48 us to 40), 16 of
    # bf16 over 2K, 112 MB, and 32 of int8 over 2K, 103 MB, lose (29 to 34, 32 to 40), 32 of int4 over 8K, 197 MB, win (60 to 49).
    kWorthBytes, kWorthLaneBytes = 72 << 20, 3 << 20
    _sharing = False
    _groups = None    # (lanes, pages shared) of each group; None: not known, or the caller has decided

    def __init__(self, storage: PageStorage, query_heads: int, lanes: int, ctas: int = 0):
        layout = storage.layout
        self.storage, self.layout, self.query_heads, self.lanes = storage, layout, query_heads, lanes
        self._lib = lib.load()
        H, D, G = layout.kv_heads, layout.head_dimension, query_heads // layout.kv_heads
        stride = VERIFY_CHUNK_STRIDE
        device = "cuda"
        self.queries = torch.zeros((lanes, H, stride, G, D), dtype=torch.bfloat16, device=device)
        self.output = torch.zeros_like(self.queries)
        self.chunk_keys = torch.zeros((lanes, H, stride, D), dtype=torch.bfloat16, device=device)
        self.chunk_values = torch.zeros((lanes, H, D, stride), dtype=torch.bfloat16, device=device)
        self._c_session, self._ctas = None, ctas  # the host-rows pipeline lives in the library (rk_session_*)
        # every format decodes on its streaming kernel
        self.attention = ops.DecodeAttention(layout, query_heads, lanes, storage.window(), ctas)
        self.layers = storage.layers()
        self.kernel_launches = 0
        self._shared = self._lane_groups = self._group_pages = None

    def close(self):
        if self._c_session:
            self._lib.rk_session_destroy(self._c_session)
            self._c_session = None
        self.attention.close()
        if self._shared is not None:
            self._shared.close()

    def step_tables(self, table_pages: int, score_scale: float = 0.0) -> ops.StepTables:
        """Tables and parameter blocks of this session's lanes, built on the GPU from request lengths each step: its
        table_pointers, chunk_params and verify_params are what step_device takes."""
        return ops.StepTables.for_storage(self.storage, self.lanes, table_pages, score_scale=score_scale)

    def share_prefixes(self, table_pointers, verify_params, minimum_pages: int | None = None, stream=None) -> None:
        """Finds which lanes share how long a prefix; until the next call (or forget_prefixes) the device steps read every
        shared prefix once. To be called when the batch changes: a group's pages must stay full and shared. By default groups
        are formed where a tile costs less than its lanes (TILE_PRICE) and used where together they save worth_bytes() of pages a
        layer, which is counted anew for a layer with a sliding window; with `minimum_pages`, two lanes over that many pages are a
        group and every layer uses it. Without a group the steps stay as they are. The call waits for the search on the GPU;
        captured into a graph it cannot, so the default then uses whatever groups could save that much if all lanes were one."""
        default = minimum_pages is None
        if self._shared is None:
            self._shared = ops.SharedPrefixDecode(self.layout, self.query_heads, self.lanes, self.storage.window(), self._ctas)
            self._lane_groups, self._group_pages = (torch.empty(self.lanes, dtype=torch.int32, device="cuda") for _ in range(2))
        self._sharing, self._groups, self._worth = False, None, {}
        if stream is not None and not isinstance(stream, torch.cuda.Stream):
            stream = torch.cuda.ExternalStream(_stream_handle(stream))
        with torch.cuda.stream(stream):
            captured = torch.cuda.is_current_stream_capturing()
            if default:
                # no group of fewer pages is worth it, the largest being the whole batch
                most = max(prefix_saving(self.layout, [(self.lanes, 1)]), 1)
                minimum_pages = max(1, int(-(-self.worth_bytes() // most))) if captured else 1
            ops.prefix_groups(self.lanes, table_pointers, verify_params, self._lane_groups, self._group_pages,
                              minimum_lanes=int(TILE_PRICE[self.layout.format]) + 1 if default else 2, minimum_pages=minimum_pages)
            if captured:
                self._sharing = True
                return
            members, pages = Counter(self._lane_groups.tolist()), self._group_pages.tolist()
            groups = [(lanes, pages[g]) for g, lanes in members.items() if g >= 0]
            if groups and (not default or prefix_saving(self.layout, groups) >= self.worth_bytes()):
                self._sharing, self._groups = True, groups if default else None
            else:
                self._lane_groups.fill_(-1)
                self._group_pages.zero_()

    def worth_bytes(self) -> int:
        return self.kWorthBytes + min(self.lanes, 32) * self.kWorthLaneBytes

    def _shares(self, shape) -> bool:
        """Whether a layer's step reads the shared prefixes apart."""
        if not self._sharing or self._groups is None or shape is None or not shape.window:
            return self._sharing
        seen = pages_for(shape.window) + pages_for(shape.sink_tokens)  # pages that a row looks at, give or take one
        if seen not in self._worth:
            self._worth[seen] = prefix_saving(self.layout, [(lanes, min(pages, seen)) for lanes, pages in self._groups]) >= self.worth_bytes()
        return self._worth[seen]

    def forget_prefixes(self) -> None:
        """The device steps go back to one stream of pages per lane."""
        self._sharing = False

    def status(self, stream=None) -> None:
        """Raises when a bounded wait ran out in any device step since the last call (sticky; cleared by this read)."""
        self.attention.status(stream)
        if self._shared is not None:
            self._shared.status(stream)

    def _attend(self, layer: int, table_pointers, verify_params, stream, shape) -> None:
        if self._shares(shape):
            self._shared.run(self.queries, self.output, table_pointers, verify_params, self.layers[layer], self._lane_groups,
                             self._group_pages, stream=stream, shape=shape)
            self.kernel_launches += 3
        else:
            self.attention.run(self.queries, self.output, table_pointers, verify_params, self.layers[layer], stream=stream, shape=shape)
            self.kernel_launches += 2

    def step_device(self, layer: int, table_pointers, chunk_params, verify_params, stream=None, shape=None) -> None:
        """Store row 0 of the stagings at each lane's committed position, then attend (3 kernels, 4 while prefixes are shared).
        `shape`: the layer's ops.ScoreShape."""
        place = self.layers[layer]
        ops.store_verify(self.layout, self.chunk_keys, self.chunk_values, table_pointers, chunk_params, place,
                         self.lanes, 1, stream)
        self.kernel_launches += 1
        self._attend(layer, table_pointers, verify_params, stream, shape)

    def attend_device(self, layer: int, table_pointers, verify_params, stream=None, shape=None) -> None:
        self._attend(layer, table_pointers, verify_params, stream, shape)

    def step_host(self, layer: int, q_host, k_host, v_host, out_host, table_pointers, chunk_params, verify_params,
                  stream=None) -> None:
        """The step lane by lane, also while prefixes are shared. q_host [lanes][query_heads][D], k_host / v_host
        [lanes][kv_heads][D], out_host like q_host: pinned bf16 host tensors. One C call (rk_session_step_host: uploads, append, attention, download, all
        asynchronous); out_host is valid after finish_host() and a synchronise of the stream. The host tensors must
        stay unchanged until then."""
        lib.check(self._lib.rk_session_step_host(self._host_session(), layer, q_host.data_ptr(), k_host.data_ptr(),
                                                 v_host.data_ptr(), out_host.data_ptr(), table_pointers.data_ptr(),
                                                 chunk_params.data_ptr(), verify_params.data_ptr(), _stream_handle(stream)),
                  "rk_session_step_host")
        self.kernel_launches += 5

    def finish_host(self, stream=None) -> None:
        """Orders `stream` after every result copy step_host has started: synchronising it then makes out_host valid."""
        lib.check(self._lib.rk_session_finish_host(self._host_session(), _stream_handle(stream)), "rk_session_finish_host")

    def host_status(self, stream=None) -> None:
        """Raises when a bounded wait ran out in any host step since the last call (sticky; cleared by this read)."""
        lib.check(self._lib.rk_session_status(self._host_session(), _stream_handle(stream)), "rk_session_status")

    def _host_session(self):
        if self._c_session is None:
            layers = (lib.KvLayer * len(self.layers))(*self.layers)
            layout = self.layout
            self._c_session = self._lib.rk_session_create(layout.format, layout.kv_heads, self.query_heads,
                                                          layout.head_dimension, self.lanes, self.attention._window,
                                                          layers, len(self.layers), self._ctas)
            if not self._c_session:
                raise lib.RichKvError(lib.INVALID, "rk_session_create")
        return self._c_session

    def host_bytes_per_layer(self) -> tuple[int, int]:
        """(host->device, device->host) bytes one step_host call moves."""
        D, H = self.layout.head_dimension, self.layout.kv_heads
        return self.lanes * (self.query_heads + 2 * H) * D * 2, self.lanes * self.query_heads * D * 2
