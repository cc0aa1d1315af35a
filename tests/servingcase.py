"""Paged batches with random page bytes, and the attention of their rows in 64 bits straight from those bytes."""
import math

import numpy as np
import torch

from gpuhelp import dev
from kvcase import HostPool, bf16_to_f32, f32_to_bf16
from richengine_b200 import abi, lib, ops
from richengine_b200.abi import BF16, FP8E4M3, INT4, INT8, Layout
from richengine_b200.storage import PageStorage

HEADS, GROUP, DIM, PAGE = 4, 6, 256, 32
FORMATS = [INT4, INT8, FP8E4M3, BF16]


def e4m3_values():
    """The value of every e4m3 byte, from the format's definition."""
    byte = np.arange(256)
    sign, exponent, mantissa = byte >> 7, (byte >> 3) & 15, byte & 7
    value = np.where(exponent > 0, (1 + mantissa / 8) * 2.0 ** (exponent - 7.0), mantissa / 8 * 2.0 ** -6)
    value = np.where((exponent == 15) & (mantissa == 7), np.nan, value)
    return np.where(sign == 1, -value, value)


class Batch:
    """`page_lists`: each lane's pages. Every page of the pool holds random finite rows."""

    def __init__(self, fmt, page_lists, seed=3, pool_pages=None):
        self.layout = Layout(1, HEADS, DIM, fmt)
        self.fmt, self.pages, self.lanes = fmt, [list(map(int, p)) for p in page_lists], len(page_lists)
        extent_pages = self.layout.extent_alignment_pages()
        need = max([pool_pages or 1] + [max(p) + 1 for p in self.pages if p])
        self.host = HostPool(self.layout, extent_pages, -(-need // extent_pages))
        rng = np.random.default_rng(seed)
        for page in range(need):
            keys, key_scales, values, value_scales = (self.host.tensor_view(page, 0, t) for t in range(4))
            if fmt == BF16:
                keys.view(np.uint16)[:] = f32_to_bf16(rng.standard_normal(keys.size // 2, dtype=np.float32))
                values.view(np.uint16)[:] = f32_to_bf16(rng.standard_normal(values.size // 2, dtype=np.float32))
                continue
            for data, scales, size in ((keys, key_scales, 1.0), (values, value_scales, 1.0)):
                data[:] = rng.integers(0, 256, data.size, dtype=np.uint8)
                if fmt == FP8E4M3:
                    data[(data & 0x7f) >= 0x60] &= 0x9f  # finite, below 16
                top = {INT4: 4.0, INT8: 64.0, FP8E4M3: 2.0}[fmt]
                scales.view(np.float32)[:] = size / top * rng.uniform(0.5, 1.5, scales.size // 4)
        self.storage = PageStorage(self.layout, self.host.page_count, extent_pages)
        for extent in range(self.host.extents):
            assert self.storage.allocate_extent(extent)
        self.upload()
        self.layer = self.storage.layers()[0]
        self.tables = []
        for pages in self.pages:
            table = torch.zeros(max(len(pages), 1), dtype=torch.int64, device="cuda")
            if pages:
                self.storage.write_entries(pages, 0, table)
            self.tables.append(table)
        self.pointers = ops.table_pointer_array(self.tables)

    def upload(self):
        for extent in range(self.host.extents):
            self.storage.write_extent(extent, self.host.bytes[extent])

    def close(self):
        self.storage.close()

    def params(self, committed, rows=1, capacity=1, splits=1, score_scale=0.0):
        rows = rows if isinstance(rows, (list, tuple)) else [rows] * self.lanes
        array = (lib.VerifyParams * self.lanes)()
        for i in range(self.lanes):
            array[i] = lib.VerifyParams(committed[i], len(self.pages[i]), lib.KvLayer(0, 0), splits, splits, rows[i], capacity, score_scale)
        return torch.from_numpy(np.frombuffer(bytes(array), np.uint8).copy()).cuda()

    def row(self, page, token):
        """Keys and values [head][dim] of one token in 64 bits."""
        keys, key_scales, values, value_scales = (self.host.tensor_view(page, 0, t) for t in range(4))
        at = token % PAGE
        if self.fmt == BF16:
            return (bf16_to_f32(keys.view(np.uint16)).reshape(HEADS, PAGE, DIM)[:, at].astype(np.float64),
                    bf16_to_f32(values.view(np.uint16)).reshape(HEADS, DIM, PAGE)[:, :, at].astype(np.float64))
        ks = key_scales.view(np.float32).reshape(HEADS, PAGE)[:, at, None].astype(np.float64)
        vs = value_scales.view(np.float32).reshape(HEADS, PAGE)[:, at, None].astype(np.float64)
        if self.fmt == INT4:
            def nibbles(raw):
                b = raw.reshape(HEADS, PAGE, DIM // 2)[:, at]
                low, high = (b & 15).astype(int), (b >> 4).astype(int)
                both = np.stack([low, high], -1).reshape(HEADS, DIM)
                return np.where(both > 7, both - 16, both).astype(np.float64)
            return nibbles(keys) * ks, nibbles(values) * vs
        table = e4m3_values() if self.fmt == FP8E4M3 else np.arange(256, dtype=np.uint8).view(np.int8).astype(np.float64)
        return table[keys.reshape(HEADS, PAGE, DIM)[:, at]] * ks, table[values.reshape(HEADS, DIM, PAGE)[:, :, at]] * vs

    def rows(self, lane, tokens):
        """Keys and values [head][token][dim] of a lane's `tokens`."""
        pairs = [self.row(self.pages[lane][t // PAGE], t) for t in tokens]
        return np.stack([k for k, _ in pairs], 1), np.stack([v for _, v in pairs], 1)

    def attend(self, lane, position, query, shape=None, scale=1.0 / 16.0):
        """One row's attention [head][group][dim] and the bound on a kernel's error.

        The bound: a weight is rounded once to 11 bits (2^-11 of itself; the bf16 pools keep 16), and a score is off by
        the fp32 accumulation of 256 products (256 * 2^-24 of the sum of their magnitudes) and a few roundings of its own
        value (the fold of the scales, the cap, the bias: 2^-19 of it), which moves a weight by twice that at most (the
        normalisation follows); the exponentials and the folded value scale add under 2^-17. A weight's change moves the
        output by at most itself times the largest value."""
        softcap, window, sinks, slopes = shape or (0.0, 0, 0, None)
        low = max(0, position + 1 - window) if window else 0
        tokens = sorted(set(range(low, position + 1)) | set(range(min(sinks, position + 1)) if window else []))
        k, v = self.rows(lane, tokens)
        q = bf16_to_f32(query).astype(np.float64)  # [head][group][dim]
        x = np.einsum("hgd,htd->hgt", q, k) * scale
        magnitude = np.einsum("hgd,htd->hgt", np.abs(q), np.abs(k)).max() * abs(scale)
        top = np.abs(x).max()
        if softcap:
            x = softcap * np.tanh(x / softcap)
        if slopes is not None:
            distance = position - np.array(tokens)
            x = x - np.asarray(slopes, np.float64).reshape(HEADS, GROUP, 1) * distance
            # far tokens carry a large bias and no weight: only the scores within 30 of the row's best count
            near = x > x.max(-1, keepdims=True) - 30
            top = max(top, np.abs(np.where(near, x, 0.0)).max())
        p = np.exp(x - x.max(-1, keepdims=True))
        p /= p.sum(-1, keepdims=True)
        out = np.einsum("hgt,htd->hgd", p, v)
        bound = (2.0 ** -11 + 2 * (256 * 2.0 ** -24 * magnitude + 2.0 ** -19 * top) + 2.0 ** -17) * np.abs(v).max()
        return out, bound


def make_queries(rng, *shape):
    return f32_to_bf16(rng.standard_normal(shape, dtype=np.float32))


def check_rows(got32, got16, want, bound, what):
    """fp32 rows within the bound; the bf16 rows half a step of theirs further."""
    assert np.isfinite(got32).all(), f"{what}: non-finite"
    error = np.abs(got32 - want)
    assert error.max() <= bound, f"{what}: off by {error.max():.3e}, bound {bound:.3e}"
    if got16 is not None:
        assert (np.abs(bf16_to_f32(got16) - want) <= bound + np.abs(got32) * 2.0 ** -8).all(), f"{what}: bf16 row"


def shape_of(shape):
    """(softcap, window, sinks, slopes) -> ops.ScoreShape."""
    softcap, window, sinks, slopes = shape
    return ops.ScoreShape(softcap, window, sinks, None if slopes is None else torch.tensor(slopes, dtype=torch.float32, device="cuda"))


SLOPES = [2.0 ** (-8.0 * (h + 1) / 24) for h in range(24)]


def shuffled_pages(rng, counts):
    ids = rng.permutation(int(sum(counts)))
    return [list(p) for p in np.split(ids, np.cumsum(counts)[:-1])]


def host16(t):
    return t.cpu().view(torch.int16).numpy().view(np.uint16)
