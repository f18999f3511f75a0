"""Kernel programs: ordered launch lists for one quantized linear and for one MoE expert layer.

The engine runs a *program* -- an ordered list of kernel records whose buffers it owns
(crates/orinfer-engine/src/backend/cuda/executor.rs:1095-1124).  These classes are that list for
the paths of this library, with every buffer allocated once up front (torch is used only for
device memory and the stream), so `run()` only enqueues and can be captured in a graph.
Program order of the expert layer follows python/orinfer_build/models/flash_next (router top-k,
histogram, offsets, tiles, A8, dispatch, grouped gate_up, SwiGLU->A8, grouped down, combine).
"""
import math

import numpy as np
import torch

from . import byte_tiles, codebook, int8, mxfp4
from .lib import ORX_ERR_BAD_VARIANT, Kernel, OrxError, current_stream


def _dev(array):
    a = np.ascontiguousarray(array)
    view = {np.dtype(np.uint16): np.int16, np.dtype(np.uint32): np.int32}.get(a.dtype)
    return torch.from_numpy(a.view(view) if view else a).cuda()


PANEL_ROWS = 1024


def panels_pay(rows, n, k, cus):
    """Whether quantiser and projection of two-stage codes are faster over token panels than row-major (time of the pair over panels / row-major, 256 CUs,
    by blocks of 16 channels to a CU).
    65-128 rows: 4 to 5 blocks 0.65-0.84; more than 6 0.82-0.98 from 97 rows on, below 0.85-1.04; up to 2 blocks 0.77-0.96 above 112 rows, 0.81-0.98 above 96 up to
    K = 5120, 0.83-0.98 at K = 1024, otherwise to 1.3; 2 to 4 blocks 0.76-0.87 at K = 1024, 0.79-0.96 at K = 2048 above 80 rows, otherwise to 1.27; 5 to 6 1.0-1.1.
    Where the channel runs fill one round (up to 240 rows of up to 2 blocks, 257-384 of up to 1.3): up to one block 0.90-0.95 at K = 1024, 0.96-1.3 beyond;
    1.2 to 1.5 0.87-0.97 up to K = 2048, 0.96-1.12 beyond; 1.75 and 2 0.81-0.98; 257-384 rows 1.05-1.3.
    Elsewhere up to 512 rows: up to one block 1.1-2.2, wider 0.36-0.98 (5120 x 12288 1.01).  513-1024 rows: up to one block 0.44-1.02 up to K = 4096, 0.75-1.5
    beyond; wider 0.64-0.99 (5120 x 8192 and x 12288 at 640-768 rows 1.0-1.12, K below 2048 at 1024 rows 0.66-1.13).  Beyond 1024 rows decoding once is mostly faster
    (1280 rows 0.72-1.5)."""
    if not 64 < rows <= PANEL_ROWS:
        return False
    blocks = -(-n // 16)
    if rows <= 128:
        if blocks <= 2 * cus:
            return rows > 112 or k <= (5120 if rows > 96 else 1024)
        if blocks <= 4 * cus:
            return k <= (2048 if rows > 80 else 1024)
        return blocks <= 5 * cus or (blocks > 6 * cus and rows > 96)
    if rows > 512:
        if blocks <= cus:
            return k <= 4096
        return (rows <= 768 or k >= 2048) and (4 * blocks > 5 * cus or k <= 5120)
    row_tiles = -(-rows // 128)
    if blocks <= 2 * cus and row_tiles * -(-blocks // 4) <= cus and not (240 < rows <= 256 and blocks > cus):  # the channel runs in one round
        if rows > 256:
            return False
        return k <= 1024 or (blocks > cus and k <= 2048) or 2 * blocks > 3 * cus
    return blocks > cus


def int8_panels_pay(rows, n, k, cus):
    """The same for int8 weights (figures as above).
    65-128 rows: more than 5 blocks to a CU 0.55-0.94; 3 to 5 0.48-1.0 from 81 rows on, 1.0-1.3 below; 2 to 3 0.43-0.84 above 112 rows up to K = 8192, else 0.85-1.4; up to
    two 0.78-0.96 above 112 rows (up to one K to 8192, up to two K to 2048), otherwise 0.9-1.5.
    129-512 rows: where the channel runs fill one round 0.92-2.5 (K = 1024 of more than one block 0.39-0.5); elsewhere half to one block 0.46-0.99 up to K = 4096, 0.88-1.65
    beyond; to 1.5 blocks 0.4-0.96 up to K = 5120, 0.92-1.5 beyond; to two 0.39-1.01 up to K = 8192, 0.53-1.2 beyond; more 0.43-1.02 (17408 x 5120 at 130 / 512 rows 0.67 /
    0.82), but up to 256 rows of 2 to 3 blocks and K above 8192 0.83-1.1 and more than 5 blocks at 448-512 rows 0.7-1.2.
    513-768 rows: up to 1.5 blocks 0.44-0.87 up to K = 2048, 0.77-1.8 beyond; 1.75 to 3 0.62-1.0; more 0.73-1.25.  Above: half a block 0.53-0.73 up to K = 2048, others 0.71-2.1."""
    if not 64 < rows <= PANEL_ROWS:
        return False
    blocks = -(-n // 16)
    if rows <= 128:
        if blocks <= 3 * cus:
            return rows > 112 and k <= (2048 if cus < blocks <= 2 * cus else 8192)
        return blocks > 5 * cus or rows > 80
    if rows > 512:
        if 2 * blocks <= 3 * cus:
            return k <= 2048 and (rows <= 768 or 2 * blocks <= cus)
        return rows <= 768 and blocks <= 3 * cus
    row_tiles = -(-rows // 128)
    tile_rows = -(-rows // row_tiles)
    most = 5 if tile_rows <= 80 else 3 if tile_rows <= 112 else 2  # blocks of the widest run
    if row_tiles * -(-blocks // most) <= cus or 2 * blocks <= cus:
        return k <= 1024 and blocks > cus
    if blocks > 5 * cus:
        return rows <= 384
    if blocks > 2 * cus:
        return k <= 8192 or rows > 256 or blocks >= 3 * cus
    return k <= (4096 if blocks <= cus else 5120 if 2 * blocks <= 3 * cus else 8192)


def tiles_pay(codec, rows, n, k, cus):
    """Whether row-major rows over 128 x 128 tiles are faster than panels where these were the faster ones before the tiles (time of the pair over panels / row-major, 256 CUs,
    by blocks of 16 channels to a CU; 2600 shapes with weights in cache, both layouts of codes; median behind the range).
    Codes, 513-1024 rows: half to 1.5 blocks 0.94-1.60, 1.22, where the tiles are there (split_pays); to two blocks 0.90-1.33, 1.14 above 768 rows, 0.77-1.29, 1.02 below; wider 0.77-1.23, 0.97;
    up to half a block 0.96-1.11, 1.03 above 896 rows from K = 2048 on, 0.70-1.04, 0.86 otherwise.  Up to 512 rows panels (where they were) 0.56-0.98.
    int8, 129-256 rows: two to three blocks 1.01-1.12, 1.06 above 208 rows, up to 208 0.85-1.14, 0.99.  257-512 rows: up to two blocks 0.97-1.41, 1.15, wider 0.89-1.18, 1.05 up to K = 1024,
    0.84-1.26, 1.02 above.  513 rows and more: above half a block 1.07-1.67, 1.31; a third to half 0.97-1.26, 1.10 above 640 rows, 0.90-1.08, 0.98 below; up to a third 0.98-1.17, 1.06 above
    704, 0.88-1.05, 0.95 below."""
    if rows <= 128 or -(-rows // 128) * -(-n // 128) > 2 * cus:
        return False
    blocks = -(-n // 16)
    if codec == "q4":
        if rows <= 512:
            return False
        if 2 * blocks <= cus:
            return rows > 896 and k >= 2048
        return 2 * blocks <= 3 * cus or (rows > 768 and blocks <= 2 * cus)
    if rows <= 256:
        return rows > 208 and 2 * cus < blocks <= 3 * cus
    if rows <= 512:
        return blocks <= 2 * cus or k <= 1024
    return 2 * blocks > cus or rows > (640 if 3 * blocks > cus else 704)


def split_pays(rows, n, cus):
    """The same for codes without the 128 x 128 int8 tiles: these are decoded for them once, into a Workspace that is never larger than the launch's without them, and
    the older split tiles hold 64 MiB (513 to 896 rows of 5121 to 6144 channels and K from 11008 on).  Time over panels / split tiles: rows that fill 15/16 of their row tiles of up to
    22 channels to a CU 0.98-1.10, rows that fill less 0.90-1.06 there, wider 0.87-1.02."""
    return 16 * rows >= 15 * 128 * -(-rows // 128) and n <= 22 * cus


FEW_ROWS = 8  # rows that a projection of two-stage codes quantises itself


class QuantizedLinear:
    """A8 quantiser + one projection (E8P-Q4 or W8A8) with a dynamic row count up to `capacity`."""

    def __init__(self, codec, weight, scales, capacity, *, packed_k=0, algorithm="auto", block_m=0, book=None):
        if codec not in ("q4", "w8"):
            raise ValueError("codec must be q4 or w8")
        self.codec, self.capacity = codec, capacity
        scales = np.asarray(scales)
        self.n = scales.shape[0]
        weight = np.asarray(weight)
        if codec == "q4":
            self.k = weight.shape[1] * 8
            stored = codebook.q4_to_k_major(weight, 128) if packed_k == 128 else weight
        else:
            self.k = weight.shape[1]
            stored = weight
        self.weight = _dev(stored)
        self.scales = _dev(scales)
        self.book = _dev(codebook.book() if book is None else book)
        # rows over panels: the quantiser leaves the int8 rows a second time, in the order of the matrix operands
        top = min(capacity, PANEL_ROWS)
        self.over_panels = [False] * (top + 1)
        cus = self.cus = torch.cuda.get_device_properties(self.weight.device).multi_processor_count
        if algorithm == "auto" and not block_m and self.k % 128 == 0 and 256 <= self.k <= 32768 and self.n * self.k < 2**31:
            pays = panels_pay if codec == "q4" else int8_panels_pay
            self.over_panels = [pays(rows, self.n, self.k, cus) for rows in range(top + 1)]
        self.over_tiles = {}  # of row counts that have come: whether row-major is faster after all
        # (both copies in one allocation: a second one, new from the driver, took 2 ms of a construction)
        padded = (top + 15) // 16 * 16 if any(self.over_panels) else 0
        codes = torch.empty((capacity + padded, self.k), dtype=torch.int8, device="cuda")
        self.a_q, self.panels = codes[:capacity], codes[capacity:]
        self.a_s = torch.empty((capacity, 1), dtype=torch.float16, device="cuda")
        self.out = torch.empty((capacity, self.n), dtype=torch.float16, device="cuda")
        self.quantizer = Kernel("activation_quantization", K=self.k)
        if padded:
            self.sums = torch.empty(top, dtype=torch.int32, device="cuda")
            self.panel_quantizer = Kernel("activation_quantization", K=self.k, panels=True)
            variant = dict(M=top, N=self.n, K=self.k, dynamic_rows=True, panels=True)
            self.panel_projection = Kernel("e8p_q4_projection", packed_k=packed_k, **variant) if codec == "q4" else Kernel("int8_projection", **variant)
        # workspace=True: the projection takes a `Workspace` buffer (allocated below, once, at the size
        # orx_workspace_bytes reports) for split tiles and decode-once launches
        variant = dict(M=capacity, N=self.n, K=self.k, dynamic_rows=True, algorithm=algorithm, workspace=True)
        if block_m:
            variant["block_m"] = block_m
        if codec == "q4":
            if packed_k:
                variant["packed_k"] = packed_k
            self.projection = Kernel("e8p_q4_projection", **variant)
        else:
            self.projection = Kernel("int8_projection", **variant)
        # one row of two-stage codes, where the GEMV serves the shape: it quantises the fp16 row itself, one launch instead of two
        # (9728 x 2560: 8.7 -> 6.4 us)
        # (K-major codes of K = 512 i + 256 and at most 16 channels to a CU are as fast in two from K = 3072 on: 1392 x 3328 / 4352 / 5888 / 7424 7.8 / 8.9 / 11.0 / 12.4 us
        # in one, 7.3 / 7.8 / 8.4 / 9.2 in two)
        self.single = None
        two_are_faster = algorithm == "auto" and packed_k and self.k % 512 == 256 and self.k >= 3072 and self.n <= 16 * cus
        if codec == "q4" and algorithm in ("auto", "gemv") and not block_m and not two_are_faster:
            try:
                self.single = Kernel("e8p_q4_projection", M=1, N=self.n, K=self.k, algorithm=algorithm, packed_k=packed_k,
                                     input_dtype="float16", codes=True)
            except OrxError as error:
                if error.code != ORX_ERR_BAD_VARIANT:
                    raise
        # two to eight rows, where the loader-wave kernel serves the shape: it quantises the fp16 rows itself.  Time against quantiser and projection, 600 shapes of 1000 to 34816
        # channels, weights out of cache: 2 and 4 rows 0.65 (K = 512) to 0.93, 5 and 8 rows 0.68 to 0.98 (17408 x 5120 at 8 rows 17.1 -> 16.3 us, at 4 16.6 -> 14.5;
        # 9728 x 2560 9.4 -> 7.7)
        self.few = None
        if codec == "q4" and algorithm == "auto" and not block_m and capacity > 1:
            try:
                self.few = Kernel("e8p_q4_projection", M=min(capacity, FEW_ROWS), N=self.n, K=self.k, packed_k=packed_k, dynamic_rows=True, quantize=True)
            except OrxError as error:
                if error.code != ORX_ERR_BAD_VARIANT:
                    raise
        self.workspace = self.projection.workspace()

    def quantize(self, x16, stream=None):
        rows = x16.shape[0]
        self.quantizer(stream=stream, Mask=None, Q=self.a_q, S=self.a_s, X=x16, rows=rows)
        return rows

    def project(self, rows, stream=None):
        if self.codec == "q4":
            self.projection(stream=stream, A=self.a_q, AS=self.a_s, Book=self.book, Out=self.out, S=self.scales,
                            W=self.weight, Workspace=self.workspace, m=rows)
        else:
            self.projection(stream=stream, A=self.a_q, Output=self.out, TokenScale=self.a_s, Weight=self.weight,
                            WeightScale=self.scales, Workspace=self.workspace, m=rows)
        return self._rows(rows)

    def _rows(self, rows):
        """A tensor of the caller's own over the first rows of `out`: what it does to its shape stays with it.  (One view, 1.0 us of
        host time beside the launch, slicing 1.4; a kept slice and detach() take 0.5, but 12 more on a first call.)"""
        return self.out.as_strided((rows, self.n), (self.n, 1))

    def _row_major(self, rows):
        """Whether row-major rows are faster than panels, asked when such rows first come (0.2 us, of codes 1.5; for every row count at construction it was 3 ms)."""
        known = self.over_tiles.get(rows)
        if known is None:
            known = tiles_pay(self.codec, rows, self.n, self.k, self.cus)
            if known and self.codec == "q4" and self.projection.workspace_bytes(rows) < self.n * self.k:
                known = split_pays(rows, self.n, self.cus)
            self.over_tiles[rows] = known
        return known

    def run(self, x16, stream=None):
        if stream is None:
            stream = current_stream()
        if self.single is not None and x16.shape[0] == 1 and x16.data_ptr() % 16 == 0:  # (the quantiser takes any fp16 address)
            self.single(stream=stream, A=x16, AS=self.a_s, Book=self.book, Out=self.out, Q=self.a_q, S=self.scales, W=self.weight)
            return self._rows(1)
        rows = x16.shape[0]
        if 1 < rows <= FEW_ROWS and self.few is not None and x16.data_ptr() % 16 == 0:
            self.few(stream=stream, A=x16, AS=self.a_s, Book=self.book, Out=self.out, Q=self.a_q, S=self.scales, W=self.weight, m=rows)
            return self._rows(rows)
        if rows < len(self.over_panels) and self.over_panels[rows] and not self._row_major(rows):
            self.panel_quantizer(stream=stream, Mask=None, Panels=self.panels, Q=self.a_q, S=self.a_s, Sums=self.sums, X=x16, rows=rows)
            if self.codec == "q4":
                self.panel_projection(stream=stream, A=self.panels, AS=self.a_s, Book=self.book, Out=self.out, S=self.scales, Sums=self.sums,
                                      W=self.weight, m=rows)
            else:
                self.panel_projection(stream=stream, A=self.panels, Output=self.out, TokenScale=self.a_s, Weight=self.weight,
                                      WeightScale=self.scales, m=rows)
            return self._rows(rows)
        return self.project(self.quantize(x16, stream), stream)


BULK_ROWS = 128  # tile height of the routed projections of many rows
# Routed rows per expert from which they beat the seven-launch order over tiles of 32 rows whatever the shape (us, seven launches against six):
# 64 experts x top-6, H 3072, I 256: 73 / 76 at 24 rows, 87 / 85 at 48, 136 / 99 at 96; 16 x top-2, H 4096, I 1536: 85 / 88 at 32,
# 121 / 93 at 64, 325 / 171 at 256.
BULK_ROWS_PER_EXPERT = 48


def small_tile_work(routed, experts, hidden, intermediate):
    """Units of 32 rows (half a tile per expert more than the rows fill) x 512 channels that the projections of a layer come to, those of the second by the length of its rows."""
    return (routed / 32 + experts / 2) * (-(-2 * intermediate // 512) + -(-hidden // 512) * intermediate / hidden)


def routes_pay(routed, experts, hidden, intermediate, cus):
    """Whether the four launches over 32-row tiles whose first projection works out its tiles by itself are faster than the order over 128-row tiles where that was the faster one (time of the
    layer, the latter over the former; 75 layers of up to 4096 routes, popularity like 1 / rank^1.1, 256 CUs, by the small tiles' work to a CU).  Up to 1.5 units 0.96-1.36, median 1.08 (two of 58
    below 0.98); above 0.87-1.19, median 0.96."""
    return 2 * small_tile_work(routed, experts, hidden, intermediate) <= 3 * cus


def bulk_pays(routed, experts, hidden, intermediate, cus):
    """Whether the order over 128-row tiles is faster than the one over tiles of 32 rows, five launches of either kind (time of the layer, the latter over the former; 600 shapes
    with 6 to 48 routed rows per expert, popularity like 1 / rank^1.1, 256 CUs).  What counts is the small tiles' work: units of 32 rows (half a tile per expert more than the rows
    fill) x 512 channels to a CU, those of the second projection by the length of its rows.  From 24 rows per expert and half a unit on 0.95-1.64 (median 1.2), of up to 64 experts from 16 rows
    (32 experts: 12) and 0.7 on 0.97-1.35, of up to 32 experts with 896 and more channels between, where the small tiles of the second projection hold the fewest rows, from 7 rows and 0.4 on
    0.96-1.33; otherwise 0.64-1.1 (of 128 experts with fewer rows 0.75-1.29 without a line between)."""
    work = small_tile_work(routed, experts, hidden, intermediate)
    rows = routed / experts
    return (rows >= 24 and work >= 0.5 * cus or experts <= 64 and rows >= (12 if experts <= 32 else 16) and work >= 0.7 * cus
            or experts <= 32 and intermediate >= 896 and rows >= 7 and work >= 0.4 * cus)


def one_launch_routes(tokens, top_k, experts):
    """Whether router and metadata of few tokens are faster in one launch, whose workgroup has sixteen waves: a token to a wave at a time, top_k ranks one after another
    (time of the layer, one launch over two: up to 18 ranks a wave 0.79-0.99, 24 and 32 1.01-1.11)."""
    return tokens <= 64 and tokens * top_k <= 1024 and experts <= 512 and -(-tokens // 16) * top_k <= 18


def few_pays(tokens, top_k, experts, hidden, intermediate, cus):
    """Whether five launches over tiles of 32 rows (few_rows) are faster than the seven, where the resident kernel is not there (time of the layer, seven over five, 3700 shapes, popularity
    like 1 / rank^0.9, 256 CUs, the median behind the range; weights in cache, and in brackets out of it).  Every workgroup of their second projection quantises its tile's rows again,
    which few or short rows pay for.  Rows of all tiles together (routed x intermediate) up to 80000 0.85-1.80, 1.30 (0.98-1.72, 1.31); above, up to 640 channels between 0.87-1.55, 1.12
    (0.92-1.35, 1.11); up to 1152 where gate | up has at most seven workgroups of 64 channels to a CU 0.85-1.26, 1.02 (0.90-1.27, 1.05), beyond 0.77-1.31, 0.94 (0.82-1.25, 1.01); longer ones
    0.66-1.11, 0.89 (0.72-1.16, 0.97)."""
    routed = tokens * top_k
    if intermediate <= 640 or routed * intermediate <= 80000:
        return True
    tiles = max(experts * (1 - math.exp(-routed / experts)), routed / 32)  # of uniform popularity
    return intermediate <= 1152 and tiles * -(-intermediate // 32) <= 7 * cus


class MoeLayer:
    """Q2A8 expert layer: token-sort, grouped gate_up, SwiGLU->A8, grouped down, weighted combine."""

    def __init__(self, tokens, experts, top_k, hidden, intermediate, gate_up, gate_up_scales, down, down_scales,
                 block_m=32, packed_k=128, fused_metadata=None, fused_dispatch=True, signs=None, fused_stages=None,
                 keep_intermediates=False, grouped_algorithm="auto"):
        self.tokens, self.experts, self.top_k = tokens, experts, top_k
        self.hidden, self.inter, self.block_m = hidden, intermediate, block_m
        assignments = tokens * top_k
        self.assignments = assignments
        # capacity bound of the tile list (kernels/cuda/model/moe.py:263-264)
        self.tile_capacity = (assignments + block_m - 1) // block_m + min(experts, assignments)
        gate_up, down = np.asarray(gate_up), np.asarray(down)
        if packed_k == 128:
            gate_up, down = codebook.q2_to_k_major(gate_up), codebook.q2_to_k_major(down)
        self.w1, self.w2 = _dev(gate_up), _dev(down)
        self.s1, self.s2 = _dev(gate_up_scales), _dev(down_scales)
        self.book = _dev(codebook.book())
        i32 = dict(dtype=torch.int32, device="cuda")
        f16 = dict(dtype=torch.float16, device="cuda")
        i8 = dict(dtype=torch.int8, device="cuda")
        self.ids = torch.empty((tokens, top_k), **i32)
        self.prob = torch.empty((tokens, top_k), dtype=torch.float32, device="cuda")
        self.counts = torch.empty(experts, **i32)
        self.relative = torch.empty((tokens, top_k), **i32)
        self.row_offsets = torch.empty(experts, **i32)
        self.tile_offsets = torch.empty(experts, **i32)
        self.tile_count = torch.empty(1, **i32)
        self.tile_expert = torch.empty(self.tile_capacity, **i32)
        self.tile_row = torch.empty(self.tile_capacity, **i32)
        self.slot_map = torch.empty((tokens, top_k), **i32)
        self.a_q = torch.empty((tokens, hidden), **i8)
        self.a_s = torch.empty((tokens, 1), **f16)
        self.h_q = torch.empty((assignments, intermediate), **i8)
        self.h_s = torch.empty((assignments, 1), **f16)
        self.down_out = torch.empty((assignments, hidden), **f16)
        self.out = torch.empty((tokens, hidden), **f16)
        common = dict(M=tokens, E=experts, top_k=top_k)
        # one launch for all routing metadata where the fused kernel applies (kernels/cuda/model/moe.py:713-764),
        # the three-kernel form otherwise
        one_launch_refused = fused_metadata is False
        fused_metadata_asked = fused_metadata
        if fused_metadata is None:
            fused_metadata = experts <= 1024 and (16 * experts + 32 + 2 * tokens * top_k) * 4 <= 160 * 1024
        self.k_metadata = Kernel("route_metadata", block_m=block_m, **common) if fused_metadata else None
        self.k_router = Kernel("router_topk", renormalize=True, **common)
        self.k_histogram = Kernel("expert_histogram", **common)
        self.k_offsets = Kernel("expert_offsets", E=experts, block_m=block_m)
        self.k_tiles = Kernel("expert_tiles", block_m=block_m, **common)
        # the dispatch quantises the fp16 rows on its way (one launch instead of quantiser + copy) where
        # the row layout allows it
        self.fused_dispatch = fused_dispatch and hidden % 8 == 0
        self.k_a8 = Kernel("activation_quantization", K=hidden)
        self.k_dispatch = Kernel("expert_dispatch", H=hidden, scale_group=hidden, **common,
                                 **({"input_dtype": "float16"} if self.fused_dispatch else {}))
        # signs: the layer's input is rotated first (block-128 signed Hadamard); rotation, A8 and the
        # scatter to the expert-sorted slots are one launch (kernels/cuda/model/rotation_a8.py:558-604)
        self.signs = None if signs is None else _dev(np.asarray(signs, np.int8))
        self.k_rotate_dispatch = None
        if signs is not None:
            self.k_rotate_dispatch = Kernel("rotate_expert_a8", M=tokens, K=hidden, routing="scatter", top_k=top_k,
                                            experts=experts, hand_over="int8")
        grouped = dict(rows=assignments, E=experts, tiles=self.tile_capacity, block_m=block_m, packed_k=packed_k,
                       algorithm=grouped_algorithm)
        self.k_gate_up = Kernel("e8p_decode_grouped", N=2 * intermediate, K=hidden, **grouped)
        self.k_swiglu_a8 = Kernel("activation_quantization", K=intermediate, fused=True)
        self.k_down = Kernel("e8p_decode_grouped", N=hidden, K=intermediate, **grouped)
        # Five launches instead of seven where the resident expert kernel takes the shapes:
        #   router top-k that also quantises every token's row (once per token, not once per route),
        #   metadata that also writes SlotMap, its inverse and zeroed per-slot maxima,
        #   gate_up that gathers the int8 token rows by slot while it stages a tile (no dispatch copy) and
        #     whose epilogue writes fp16(silu(gate) * up) and raises every slot's largest magnitude,
        #   down that quantises those fp16 rows while it stages a tile (no SwiGLU->A8 launch),
        #   combine.
        # The library refuses the variants it does not serve that way, and the seven-launch program stays.
        # Four where gate_up also works out its tiles from the ids (up to 4096 routes): no launch for the metadata, which it leaves for down and combine; the router then
        # clears the maxima.
        self.fused_stages = self.routes_inside = False
        self.keep_intermediates = keep_intermediates
        if fused_stages is not False and fused_metadata and signs is None and hidden % 8 == 0:
            try:
                if fused_metadata_asked is None:
                    try:
                        self.k_gate_up_routes = Kernel("e8p_decode_grouped", N=2 * intermediate, K=hidden, gather=True, epilogue="swiglu", routes=True,
                                                       top_k=top_k, **grouped)
                        self.k_router_clear = Kernel("router_topk", renormalize=True, quantize_hidden=hidden, row_max=True, **common)
                        self.routes_inside = True
                    except OrxError as error:
                        if error.code != ORX_ERR_BAD_VARIANT:
                            raise
                if not self.routes_inside:
                    self.k_router_a8 = Kernel("router_topk", renormalize=True, quantize_hidden=hidden, **common)
                    self.k_metadata_slots = Kernel("route_metadata", block_m=block_m, slot_maps=True, **common)
                    self.k_gate_up_fused = Kernel("e8p_decode_grouped", N=2 * intermediate, K=hidden, gather=True,
                                                  epilogue="swiglu", **grouped)
                self.k_down_fused = Kernel("e8p_decode_grouped", N=hidden, K=intermediate, input_dtype="float16",
                                           tile_units=self.routes_inside, **grouped)
                self.fused_stages = True
            except OrxError as error:
                self.routes_inside = False
                if fused_stages or error.code != ORX_ERR_BAD_VARIANT:
                    raise
        # Many rows: six launches over tiles of 128 rows (`block_m` is the tile height of the orders above).
        #   router top-k + A8 of every token's row, metadata in segments (two launches above 16384 routes, of few experts above 8192 or 12288),
        #   gate_up that gathers the token rows and writes fp16(silu(gate) * up), A8, down, combine.
        # A caller who asked for the quantiser and the dispatch, or the metadata, as launches of their own gets them; `fused_stages` stays
        # true where the five launches are served too.
        self.bulk, bulk_tiles, bulk_kernels = False, 0, {}
        if (fused_stages is None and not keep_intermediates and signs is None and self.fused_dispatch
                and not one_launch_refused and packed_k == 128 and experts <= 1024 and grouped_algorithm == "auto"
                and (not self.fused_stages and assignments >= BULK_ROWS_PER_EXPERT * experts
                     or bulk_pays(assignments, experts, hidden, intermediate, torch.cuda.get_device_properties(self.w1.device).multi_processor_count))):
            try:
                bulk_tiles = (assignments + BULK_ROWS - 1) // BULK_ROWS + min(experts, assignments)
                bulk = dict(rows=assignments, E=experts, tiles=bulk_tiles, block_m=BULK_ROWS, tile_units=True)
                # (all of them before the first is kept: the five launches have kernels of the same names)
                bulk_kernels = dict(
                    k_router_a8=Kernel("router_topk", renormalize=True, quantize_hidden=hidden, **common),
                    k_metadata_slots=Kernel("route_metadata", block_m=BULK_ROWS, slot_maps=True, workspace=True, tile_units=True, **common),
                    k_gate_up_bulk=Kernel("e8p_decode_grouped", N=2 * intermediate, K=hidden, gather=True, epilogue="swiglu", **bulk),
                    k_act_a8=Kernel("activation_quantization", K=intermediate),
                    k_down_bulk=Kernel("e8p_decode_grouped", N=hidden, K=intermediate, **bulk))
                self.bulk = True
            except OrxError as error:
                if error.code != ORX_ERR_BAD_VARIANT:
                    raise
        # Few rows: where neither order applies, five launches over tiles of 32 rows, any hidden and intermediate width, where they are the faster ones.
        #   router top-k + A8 of every token's row, metadata with the tiles as units,
        #   gate_up that gathers the token rows, writes fp16(silu(gate) * up) and raises every slot's largest magnitude,
        #   down that quantises those rows on their way, combine.
        # A caller who asked for launches of their own, for the values in between (`keep_intermediates`) or for an algorithm gets them.
        self.few = False
        if (fused_stages is None and not self.bulk and not self.fused_stages and not keep_intermediates and signs is None and self.fused_dispatch
                and not one_launch_refused and packed_k == 128 and block_m == 32 and experts <= 1024 and grouped_algorithm == "auto"
                and few_pays(tokens, top_k, experts, hidden, intermediate, torch.cuda.get_device_properties(self.w1.device).multi_processor_count)):
            try:
                few = dict(rows=assignments, E=experts, tiles=self.tile_capacity, block_m=block_m, few_rows=True)
                # four where router and metadata are one
                self.k_routes = None
                if one_launch_routes(tokens, top_k, experts):
                    self.k_routes = Kernel("router_topk", renormalize=True, quantize_hidden=hidden, metadata=True, block_m=block_m, **common)
                self.k_router_a8 = Kernel("router_topk", renormalize=True, quantize_hidden=hidden, **common)
                self.k_metadata_slots = Kernel("route_metadata", block_m=block_m, slot_maps=True, workspace=True, tile_units=True, **common)
                self.k_gate_up_few = Kernel("e8p_decode_grouped", N=2 * intermediate, K=hidden, gather=True, epilogue="swiglu", **few)
                self.k_down_few = Kernel("e8p_decode_grouped", N=hidden, K=intermediate, input_dtype="float16", **few)
                self.few = True
            except OrxError as error:
                if error.code != ORX_ERR_BAD_VARIANT:
                    raise
        # The four launches also where nothing but the seven is left (1.06-1.28 times as fast, 11 layers), and over the order for many rows where they are the faster ones.  `bulk` says that that
        # one is served and would run; `routes_first` that these run before either.
        self.routes_first = False
        if (fused_stages is None and not self.few and not keep_intermediates and signs is None and self.fused_dispatch and fused_metadata and fused_metadata_asked is None
                and packed_k == 128 and block_m == 32 and grouped_algorithm == "auto"
                and (routes_pay(assignments, experts, hidden, intermediate, torch.cuda.get_device_properties(self.w1.device).multi_processor_count) if self.bulk
                     else not self.fused_stages)):
            if not self.routes_inside:
                try:
                    resident = dict(grouped, algorithm="resident")
                    served = dict(
                        k_gate_up_routes=Kernel("e8p_decode_grouped", N=2 * intermediate, K=hidden, gather=True, epilogue="swiglu", routes=True, top_k=top_k, **resident),
                        k_router_clear=Kernel("router_topk", renormalize=True, quantize_hidden=hidden, row_max=True, **common),
                        k_down_fused=Kernel("e8p_decode_grouped", N=hidden, K=intermediate, input_dtype="float16", tile_units=True, **resident))
                    vars(self).update(served)
                    self.routes_inside = True
                except OrxError as error:
                    if error.code != ORX_ERR_BAD_VARIANT:
                        raise
            self.routes_first = self.routes_inside
        # What the order that `run` takes needs between its launches, behind all decisions: orders that are served and not taken leave no buffer and no length of a list.
        takes_bulk = self.bulk and not self.routes_first
        if takes_bulk:
            vars(self).update(bulk_kernels)
        if takes_bulk or self.few or self.fused_stages or self.routes_first:
            tiles = bulk_tiles if takes_bulk else self.tile_capacity
            if tiles > self.tile_capacity:
                self.tile_expert, self.tile_row = torch.empty(tiles, **i32), torch.empty(tiles, **i32)
            if takes_bulk or self.few or self.routes_inside:
                self.tile_units = torch.empty((tiles, 4), **i32)
            if not takes_bulk:
                self.row_max = torch.empty(assignments, **i32)
            self.slot_token = torch.empty(assignments, **i32)
            self.act = torch.empty((assignments, intermediate), **f16)
        if takes_bulk or self.few:
            self.segments = self.k_metadata_slots.workspace()
        # the dispatched rows and the gate | up outputs, which the orders for long prompts and for few rows do without
        self.d = self.ds = self.gate_up_out = None
        if not self.bulk and not self.few and not self.routes_first:
            self.d = torch.empty((assignments, hidden), **i8)
            self.ds = torch.empty((assignments, 1), **f16)
            self.gate_up_out = torch.empty((assignments, 2 * intermediate), **f16)
        self.k_combine = Kernel("moe_combine", H=hidden, slots=assignments, **common)

    def run(self, x16, logits, stream=None):
        s = current_stream() if stream is None else stream
        if self.routes_first:
            return self._run_routes_inside(x16, logits, s)
        if self.bulk:
            return self._run_bulk(x16, logits, s)
        if self.fused_stages:
            return self._run_fused(x16, logits, s)
        if self.few:
            return self._run_few(x16, logits, s)
        self.k_router(stream=s, IDs=self.ids, Logits=logits, Prob=self.prob)
        if self.k_metadata is not None:
            self.k_metadata(stream=s, Counts=self.counts, IDs=self.ids, RelativeSlot=self.relative,
                            RowOffsets=self.row_offsets, TileCount=self.tile_count, TileExpert=self.tile_expert,
                            TileOffsets=self.tile_offsets, TileRow=self.tile_row)
        else:
            self.k_histogram(stream=s, Counts=self.counts, IDs=self.ids, RelativeSlot=self.relative)
            self.k_offsets(stream=s, Counts=self.counts, RowOffsets=self.row_offsets, TileCount=self.tile_count,
                           TileOffsets=self.tile_offsets)
            self.k_tiles(stream=s, Counts=self.counts, TileExpert=self.tile_expert, TileOffsets=self.tile_offsets,
                         TileRow=self.tile_row)
        if self.k_rotate_dispatch is not None:
            self.k_rotate_dispatch(stream=s, D=self.d, DS=self.ds, IDs=self.ids, Q=None, RelativeSlot=self.relative,
                                   RowOffsets=self.row_offsets, S=self.a_s, Signs=self.signs, SlotMap=self.slot_map,
                                   Sum=None, X=x16)
        elif self.fused_dispatch:
            self.k_dispatch(stream=s, A=x16, D=self.d, DS=self.ds, IDs=self.ids, RelativeSlot=self.relative,
                            RowOffsets=self.row_offsets, Scale=None, SlotMap=self.slot_map)
        else:
            self.k_a8(stream=s, Mask=None, Q=self.a_q, S=self.a_s, X=x16, rows=self.tokens)
            self.k_dispatch(stream=s, A=self.a_q, D=self.d, DS=self.ds, IDs=self.ids, RelativeSlot=self.relative,
                            RowOffsets=self.row_offsets, Scale=self.a_s, SlotMap=self.slot_map)
        routed = dict(Book=self.book, Counts=self.counts, Offsets=self.row_offsets, TileCount=self.tile_count,
                      TileExpert=self.tile_expert, TileRow=self.tile_row)
        self.k_gate_up(stream=s, A=self.d, AS=self.ds, C=self.gate_up_out, P=self.w1, WS=self.s1, **routed)
        self.k_swiglu_a8(stream=s, Mask=None, Q=self.h_q, S=self.h_s, X=self.gate_up_out, rows=self.assignments)
        self.k_down(stream=s, A=self.h_q, AS=self.h_s, C=self.down_out, P=self.w2, WS=self.s2, **routed)
        self.k_combine(stream=s, Expert=self.down_out, Output=self.out, Prob=self.prob, Shared=None, SharedGate=None,
                       SlotMap=self.slot_map)
        return self.out

    def _run_bulk(self, x16, logits, s):
        self.k_router_a8(stream=s, IDs=self.ids, Logits=logits, Prob=self.prob, Q=self.a_q, S=self.a_s, X=x16)
        self.k_metadata_slots(stream=s, Counts=self.counts, IDs=self.ids, RelativeSlot=self.relative, RowMax=None,
                              RowOffsets=self.row_offsets, SlotMap=self.slot_map, SlotToken=self.slot_token,
                              TileCount=self.tile_count, TileExpert=self.tile_expert, TileOffsets=self.tile_offsets,
                              TileRow=self.tile_row, TileUnits=self.tile_units, Workspace=self.segments)
        routed = dict(Book=self.book, Counts=self.counts, Offsets=self.row_offsets, TileCount=self.tile_count,
                      TileExpert=self.tile_expert, TileRow=self.tile_row, TileUnits=self.tile_units)
        self.k_gate_up_bulk(stream=s, A=self.a_q, AS=self.a_s, Act=self.act, C=None, P=self.w1, RowMax=None,
                            SlotToken=self.slot_token, WS=self.s1, **routed)
        self.k_act_a8(stream=s, Mask=None, Q=self.h_q, S=self.h_s, X=self.act, rows=self.assignments)
        self.k_down_bulk(stream=s, A=self.h_q, AS=self.h_s, C=self.down_out, P=self.w2, WS=self.s2, **routed)
        self.k_combine(stream=s, Expert=self.down_out, Output=self.out, Prob=self.prob, Shared=None, SharedGate=None,
                       SlotMap=self.slot_map)
        return self.out

    def _run_few(self, x16, logits, s):
        metadata = dict(Counts=self.counts, IDs=self.ids, RelativeSlot=self.relative, RowMax=self.row_max, RowOffsets=self.row_offsets,
                        SlotMap=self.slot_map, SlotToken=self.slot_token, TileCount=self.tile_count, TileExpert=self.tile_expert,
                        TileOffsets=self.tile_offsets, TileRow=self.tile_row, TileUnits=self.tile_units)
        if self.k_routes is not None:
            self.k_routes(stream=s, Logits=logits, Prob=self.prob, Q=self.a_q, S=self.a_s, X=x16, **metadata)
        else:
            self.k_router_a8(stream=s, IDs=self.ids, Logits=logits, Prob=self.prob, Q=self.a_q, S=self.a_s, X=x16)
            self.k_metadata_slots(stream=s, Workspace=self.segments, **metadata)
        routed = dict(Book=self.book, RowMax=self.row_max, TileCount=self.tile_count, TileUnits=self.tile_units)
        self.k_gate_up_few(stream=s, A=self.a_q, AS=self.a_s, Act=self.act, P=self.w1, SlotToken=self.slot_token, WS=self.s1, **routed)
        self.k_down_few(stream=s, A=self.act, C=self.down_out, P=self.w2, WS=self.s2, **routed)
        self.k_combine(stream=s, Expert=self.down_out, Output=self.out, Prob=self.prob, Shared=None, SharedGate=None,
                       SlotMap=self.slot_map)
        return self.out

    def _run_fused(self, x16, logits, s):
        keep = self.keep_intermediates
        if self.routes_inside:
            return self._run_routes_inside(x16, logits, s)
        self.k_router_a8(stream=s, IDs=self.ids, Logits=logits, Prob=self.prob, Q=self.a_q, S=self.a_s, X=x16)
        self.k_metadata_slots(stream=s, Counts=self.counts, IDs=self.ids, RelativeSlot=self.relative, RowMax=self.row_max,
                              RowOffsets=self.row_offsets, SlotMap=self.slot_map, SlotToken=self.slot_token,
                              TileCount=self.tile_count, TileExpert=self.tile_expert, TileOffsets=self.tile_offsets,
                              TileRow=self.tile_row)
        routed = dict(Book=self.book, Counts=self.counts, Offsets=self.row_offsets, TileCount=self.tile_count,
                      TileExpert=self.tile_expert, TileRow=self.tile_row)
        self.k_gate_up_fused(stream=s, A=self.a_q, AS=self.a_s, Act=self.act, C=self.gate_up_out if keep else None,
                             P=self.w1, RowMax=self.row_max, SlotToken=self.slot_token, WS=self.s1, **routed)
        self.k_down_fused(stream=s, A=self.act, AS=self.h_s if keep else None, C=self.down_out, P=self.w2,
                          Q=self.h_q if keep else None, RowMax=self.row_max, WS=self.s2, **routed)
        self.k_combine(stream=s, Expert=self.down_out, Output=self.out, Prob=self.prob, Shared=None, SharedGate=None,
                       SlotMap=self.slot_map)
        return self.out

    def _run_routes_inside(self, x16, logits, s):
        keep = self.keep_intermediates
        self.k_router_clear(stream=s, IDs=self.ids, Logits=logits, Prob=self.prob, Q=self.a_q, RowMax=self.row_max, S=self.a_s, X=x16)
        routed = dict(Book=self.book, Counts=self.counts, Offsets=self.row_offsets, RowMax=self.row_max, TileCount=self.tile_count,
                      TileExpert=self.tile_expert, TileRow=self.tile_row, TileUnits=self.tile_units)
        self.k_gate_up_routes(stream=s, A=self.a_q, AS=self.a_s, Act=self.act, C=self.gate_up_out if keep else None, IDs=self.ids, P=self.w1,
                              RelativeSlot=self.relative, SlotMap=self.slot_map, SlotToken=self.slot_token, TileOffsets=self.tile_offsets, WS=self.s1, **routed)
        self.k_down_fused(stream=s, A=self.act, AS=self.h_s if keep else None, C=self.down_out, P=self.w2, Q=self.h_q if keep else None, WS=self.s2, **routed)
        self.k_combine(stream=s, Expert=self.down_out, Output=self.out, Prob=self.prob, Shared=None, SharedGate=None,
                       SlotMap=self.slot_map)
        return self.out


def combine_pays(routes, hidden, intermediate, cus):
    """Whether the second projection of one token with the SwiGLU in front and the sum over its routes behind is faster than projection and sum in two launches (time of the layer, one over
    two; 256 CUs; without the SwiGLU it also is where `MoeTokenLayer` says).  Every workgroup of 8 channels makes the codes of all routes itself, in turns of 512 values, and one route's are a wave's.
    Up to 512 values 0.78-0.97, with three workgroups to a CU 1.06-1.09 up to two routes and 0.79-0.96 above.  Up to 1024: one workgroup to a CU 0.92-0.98 up to four routes
    and 0.92-0.96 above (up to half of the CUs 1.0-1.03); two and three to a CU 0.98-1.22 up to four routes, 0.89-0.99 above.  Beyond mostly 1.0-1.33 (0.97 at best, 8 routes of
    4096 x 1536)."""
    per_cu = -(-hidden // (8 * cus))
    if intermediate <= 512:
        return per_cu <= 2 or routes > 2
    if intermediate <= 1024:
        return (routes <= 4 or hidden > 4 * cus) if per_cu == 1 else routes > 4
    return False


class MoeTokenLayer:
    """The same expert layer for ONE token: its routes index the expert banks directly
    (kernels/cuda/model/integer_vq.py:380-444), so there is no sorting, no tile list and no dispatch copy:
    router top-k, gate/up of every route from the shared row (quantised on the way), SwiGLU->A8 per route,
    down per route, weighted combine."""

    def __init__(self, experts, top_k, hidden, intermediate, gate_up, gate_up_scales, down, down_scales, fused=None):
        self.experts, self.top_k, self.hidden, self.inter = experts, top_k, hidden, intermediate
        self.w1 = _dev(codebook.q2_to_k_major(np.asarray(gate_up)))
        self.w2 = _dev(codebook.q2_to_k_major(np.asarray(down)))
        self.s1, self.s2 = _dev(gate_up_scales), _dev(down_scales)
        self.book = _dev(codebook.raw_book())
        f16 = dict(dtype=torch.float16, device="cuda")
        i8 = dict(dtype=torch.int8, device="cuda")
        self.ids = torch.empty((1, top_k), dtype=torch.int32, device="cuda")
        self.prob = torch.empty((1, top_k), dtype=torch.float32, device="cuda")
        self.a_s = torch.empty((1, 1), **f16)
        self.gate_up_out = torch.empty((top_k, 2 * intermediate), **f16)
        self.h_q = torch.empty((top_k, intermediate), **i8)
        self.h_s = torch.empty((top_k, 1), **f16)
        self.down_out = torch.empty((top_k, hidden), **f16)
        self.slot_map = torch.arange(top_k, dtype=torch.int32, device="cuda").view(1, top_k)  # route r is slot r
        self.out = torch.empty((1, hidden), **f16)
        common = dict(M=1, E=experts, top_k=top_k)
        self.k_router = Kernel("router_topk", renormalize=True, **common)
        # gate/up quantises the shared fp16 row itself (no launch for the A8 of one row)
        self.k_gate_up = Kernel("integer_e8p_gemv", E=experts, routes=top_k, N=2 * intermediate, K=hidden,
                                shared_input=True, input_dtype="float16")
        self.k_swiglu_a8 = Kernel("activation_quantization", K=intermediate, fused=True)
        self.k_down = Kernel("integer_e8p_gemv", E=experts, routes=top_k, N=hidden, K=intermediate, shared_input=False)
        self.k_combine = Kernel("moe_combine", H=hidden, slots=top_k, **common)
        # Fewer than five launches where the library has the forms (up to 512 experts): gate/up selects the token's
        # routes itself while it builds its tables (no router launch), down turns the fp16 gate|up rows into
        # SwiGLU -> A8 codes on their way into LDS (no launch in between).  These are three; two below.
        self.fused = False
        if fused is not False:
            try:
                routes = dict(E=experts, routes=top_k)
                self.k_gate_up_routing = Kernel("integer_e8p_gemv", N=2 * intermediate, K=hidden, shared_input=True,
                                                input_dtype="float16", route_logits=True, renormalize=True, **routes)
                self.k_down_swiglu = Kernel("integer_e8p_gemv", N=hidden, K=intermediate, shared_input=False,
                                            input_dtype="float16", fused_swiglu=True, **routes)
                self.fused = True
            except OrxError as error:
                if fused or error.code != ORX_ERR_BAD_VARIANT:
                    raise
        # Two launches where the sum over the routes joins the second projection: 13.8 -> 11.6 us for 8 of 128 experts, 2048 x 512, and 10.9 since the first one leaves
        # fp16(silu(gate) * up), which every workgroup of the second made again, beside gate | up.  Three launches over two (140 shapes of up to 2048 channels between): up to two workgroups to a CU
        # 0.99-1.37, median 1.13.  `k_down_combine` names it where it also paid with the SwiGLU in front.
        self.k_down_combine = self.k_down_act = None
        cus = torch.cuda.get_device_properties(self.w2.device).multi_processor_count
        pays = combine_pays(top_k, hidden, intermediate, cus)
        if self.fused and (pays or hidden <= 16 * cus):
            try:
                served = dict(
                    k_gate_up_act=Kernel("integer_e8p_gemv", N=2 * intermediate, K=hidden, shared_input=True, input_dtype="float16", route_logits=True,
                                         renormalize=True, epilogue="swiglu", **routes),
                    k_down_act=Kernel("integer_e8p_gemv", N=hidden, K=intermediate, shared_input=False, input_dtype="float16", combine=True, **routes))
                vars(self).update(served)
                self.act = torch.empty((top_k, intermediate), **f16)
                self.k_down_combine = self.k_down_act if pays else None
            except OrxError as error:
                if error.code != ORX_ERR_BAD_VARIANT:
                    raise

    def run(self, x16, logits, stream=None):
        s = current_stream() if stream is None else stream
        if self.k_down_act is not None:
            self.k_gate_up_act(stream=s, A=x16, AS=self.a_s, Act=self.act, Book=self.book, C=self.gate_up_out, IDs=self.ids,
                               Logits=logits, P=self.w1, Prob=self.prob, WS=self.s1)
            self.k_down_act(stream=s, A=self.act, AS=self.h_s, Book=self.book, C=self.down_out, IDs=self.ids,
                                Output=self.out, P=self.w2, Prob=self.prob, WS=self.s2)
            return self.out
        if self.fused:
            self.k_gate_up_routing(stream=s, A=x16, AS=self.a_s, Book=self.book, C=self.gate_up_out, IDs=self.ids,
                                   Logits=logits, P=self.w1, Prob=self.prob, WS=self.s1)
            self.k_down_swiglu(stream=s, A=self.gate_up_out, AS=self.h_s, Book=self.book, C=self.down_out, IDs=self.ids,
                               P=self.w2, WS=self.s2)
            self.k_combine(stream=s, Expert=self.down_out, Output=self.out, Prob=self.prob, Shared=None, SharedGate=None,
                           SlotMap=self.slot_map)
            return self.out
        self.k_router(stream=s, IDs=self.ids, Logits=logits, Prob=self.prob)
        self.k_gate_up(stream=s, A=x16, AS=self.a_s, Book=self.book, C=self.gate_up_out, IDs=self.ids, P=self.w1,
                       WS=self.s1)
        self.k_swiglu_a8(stream=s, Mask=None, Q=self.h_q, S=self.h_s, X=self.gate_up_out, rows=self.top_k)
        self.k_down(stream=s, A=self.h_q, AS=self.h_s, Book=self.book, C=self.down_out, IDs=self.ids, P=self.w2,
                    WS=self.s2)
        self.k_combine(stream=s, Expert=self.down_out, Output=self.out, Prob=self.prob, Shared=None, SharedGate=None,
                       SlotMap=self.slot_map)
        return self.out


def _check_rows(x, rows, columns, dtype, device, what):
    if x.dim() != 2 or x.shape[1] != columns or x.dtype != dtype or x.device != device or not x.is_contiguous():
        raise ValueError(f"{what} must be a contiguous {dtype} tensor (rows, {columns}) on {device}, not {tuple(x.shape)} {x.dtype} on {x.device}")
    if isinstance(rows, int) and x.shape[0] != rows:
        raise ValueError(f"{what} has {x.shape[0]} rows, not {rows}")


def _apart(a, b):
    """Two contiguous tensors share no memory."""
    return a.data_ptr() + a.nbytes <= b.data_ptr() or b.data_ptr() + b.nbytes <= a.data_ptr()


class _OnDevice:
    """Launches on the GPU of the weights, whichever is current (weights on the host go to the current one); its current stream unless the caller names one."""

    @staticmethod
    def _device_of(*tensors):
        """The GPU that the weights are on, or the current one.  (`.cuda()` would copy a tensor of another GPU to the current one.)"""
        devices = {t.device for t in tensors if t.is_cuda}
        if len(devices) > 1:
            raise ValueError(f"the weights are on several GPUs: {sorted(map(str, devices))}")
        return devices.pop() if devices else torch.device("cuda", torch.cuda.current_device())

    def _call(self, body, *args, stream=None):
        if torch._C._cuda_getDevice() == self.device.index:
            return body(*args, stream=current_stream() if stream is None else stream)
        with torch.cuda.device(self.device):
            return body(*args, stream=current_stream() if stream is None else stream)


def _where_it_fits(symbol, **keys):
    """The kernel, or None where its codes do not fit LDS."""
    try:
        return Kernel(symbol, **keys)
    except OrxError as error:
        if error.code != ORX_ERR_BAD_VARIANT:
            raise
        return None


class Mxfp4Linear(_OnDevice):
    """Rows of 16-bit values, quantised to MXFP4, times MXFP4 weights: codes (N, K / 2) and exponents (N, K / 32), both uint8 (the format: mxfp4.py), up to `capacity`
    rows at a time.  epilogue="swiglu": the upper half of the channels are the up channels of the gate channels in the lower half, and silu(gate) * up comes out.
    `run` returns the object's own output buffer, or a view of its first rows, which the next call overwrites; one object serves one stream at a time."""

    def __init__(self, codes, exponents, capacity, *, dtype=torch.float16, epilogue="none"):
        if dtype not in (torch.float16, torch.bfloat16):
            raise ValueError("dtype must be torch.float16 or torch.bfloat16")
        if codes.ndim != 2:
            raise ValueError("codes must be (N, K / 2)")
        if not 0 < capacity <= 1 << 24:
            raise ValueError("capacity must be 1 to 2^24 rows")
        self.capacity, self.dtype = capacity, dtype
        channels, self.k = codes.shape[0], 2 * codes.shape[1]
        codes, exponents = torch.as_tensor(codes), torch.as_tensor(exponents)
        self.device = self._device_of(codes, exponents)
        self.weight, self.powers = (t.to(self.device) for t in mxfp4.tiles(codes, exponents, paired=epilogue == "swiglu"))
        name = mxfp4.dtype_name(dtype)
        shape = dict(N=channels, K=self.k, dynamic_rows=True, epilogue=epilogue, output_dtype=name)
        with torch.cuda.device(self.device):
            self.projection = Kernel("mxfp4_projection", M=capacity, **shape)
            self.quantizer = Kernel("mxfp4_quantization", M=capacity, K=self.k, input_dtype=name, layout="tiles")
            # Few rows: the projection quantises them itself, every workgroup all of them, one launch instead of two (weights out of cache, us of the two launches / of the one:
            # 17408 x 5120, 1 row 15.1 / 12.3, 4 rows 15.0 / 15.0, 6 rows 15.2 / 16.7; 9728 x 2560, 1 row 8.3 / 5.8, 6 rows 8.2 / 7.8, 8 rows 8.2 / 8.5; 4096 x 4096 6.3 / 4.4, 6.4 / 6.2, 6.3 / 6.9).
            # Not where their codes do not fit LDS.
            self.few_rows = min(capacity, 6 if channels <= 10240 else 4)
            self.few = _where_it_fits("mxfp4_projection", M=self.few_rows, input_dtype=name, **shape)
        self.n = channels // 2 if epilogue == "swiglu" else channels
        # the quantised rows, by tiles of 16
        tiles = -(-capacity // 16) * -(-self.k // mxfp4.STEP)
        self.a_q = torch.empty((tiles, 2048), dtype=torch.uint8, device=self.device)
        self.a_s = torch.empty((tiles, 128), dtype=torch.uint8, device=self.device)
        self.out = torch.empty((capacity, self.n), dtype=dtype, device=self.device)

    def run(self, x, stream=None):
        _check_rows(x, None, self.k, self.dtype, self.device, "x")
        rows = x.shape[0]
        if rows > self.capacity:
            raise ValueError(f"{rows} rows are more than the capacity of {self.capacity}")
        if rows:
            self._call(self._run, x, rows, stream=stream)
        return self.out if rows == self.capacity else self.out.as_strided((rows, self.n), (self.n, 1))

    def _run(self, x, rows, stream):
        # (not rows in the object's own output, a call's result given to the next one: workgroups that have ended write over what others have yet to read)
        if rows <= self.few_rows and self.few is not None and _apart(x, self.out):
            self.few(stream=stream, A=x, Out=self.out, W=self.weight, WS=self.powers, m=rows)
            return
        self.quantizer(stream=stream, Q=self.a_q, S=self.a_s, X=x, rows=rows)
        self.projection(stream=stream, A=self.a_q, AS=self.a_s, Out=self.out, W=self.weight, WS=self.powers, m=rows)


class _ExpertLayer(_OnDevice):
    """What layers of routed experts have in common: the router, the places of the routes, the weighted sum, and the buffers of all of these."""

    def _set_up(self, tokens, experts, top_k, hidden, intermediate, dtype, block_m, *, scoring, bias, groups, top_groups, group_best, renormalize, scale):
        """Kernels and buffers, with the layer's GPU in `device`."""
        self.dtype = dtype
        self.tokens, self.experts, self.top_k, self.hidden, self.inter = tokens, experts, top_k, hidden, intermediate
        self.bias = None
        if bias is not None:
            self.bias = torch.as_tensor(bias, dtype=torch.float32).to(self.device).contiguous()
            if self.bias.shape != (experts,):
                raise ValueError(f"bias must have {experts} values")
        routes = self.assignments = tokens * top_k
        self.block_m = block_m
        capacity = -(-routes // block_m) + min(experts, routes)
        common = dict(M=tokens, E=experts, top_k=top_k)
        scores = dict(scoring=scoring, bias=bias is not None, groups=groups, top_groups=groups if top_groups is None else top_groups, group_best=group_best, scale=scale)
        plain = scoring == "softmax" and bias is None and groups == 1 and top_groups in (None, 1) and group_best in (1, 2) and scale == 1.0
        with torch.cuda.device(self.device):
            self.k_router = Kernel("router_topk", renormalize=renormalize, **common, **({} if plain else scores))
            self.k_metadata = Kernel("route_metadata", block_m=block_m, slot_maps=True, workspace=True, tile_units=True, **common)
            self.k_combine = Kernel("moe_combine", H=hidden, slots=routes, expert_dtype="float32", output_dtype=mxfp4.dtype_name(dtype), **common)
            self.segments = self.k_metadata.workspace()
        i32, values = dict(dtype=torch.int32, device=self.device), dict(dtype=dtype, device=self.device)
        self.ids = torch.empty((tokens, top_k), **i32)
        self.prob = torch.empty((tokens, top_k), dtype=torch.float32, device=self.device)
        self.counts, self.row_offsets, self.tile_offsets = (torch.empty(experts, **i32) for _ in range(3))
        self.relative, self.slot_map = torch.empty((tokens, top_k), **i32), torch.empty((tokens, top_k), **i32)
        self.slot_token = torch.empty(routes, **i32)
        # (no units until a launch has listed them, not even for work that has passed `place` by and not waited for it)
        self.tile_count = torch.zeros(1, **i32)
        self.slot_map.fill_(-1)
        self.placed = False
        self.tile_expert, self.tile_row, self.tile_units = torch.empty(capacity, **i32), torch.empty(capacity, **i32), torch.empty((capacity, 4), **i32)
        self.act = torch.empty((routes, intermediate), **values)
        # (The second products stay fp32 until they are weighted and summed: as fp16, one beyond 65504 made its token's sum infinite or NaN however small its weight, and each was
        # a rounding more.  Its price with MXFP4, 128 experts x 8 of 2048 x 512, us of place and down with fp16 / fp32: 256 tokens 25.7 / 29.2, 4096 tokens 105.6 / 158.8.)
        self.down_out = torch.empty((routes, hidden), dtype=torch.float32, device=self.device)
        self.out = torch.empty((tokens, hidden), **values)
        # what the grouped kernels are made for
        self.grouped = dict(rows=routes, E=experts, tiles=capacity, block_m=block_m)

    def route(self, logits, stream=None):
        """fp32 logits (tokens, experts) -> the routes' experts (tokens, top_k) int32 and weights fp32."""
        _check_rows(logits, self.tokens, self.experts, torch.float32, self.device, "logits")
        self._call(self._route, logits, stream=stream)
        return self.ids, self.prob

    def _route(self, logits, stream):
        bias = {} if self.bias is None else {"Bias": self.bias}
        self.k_router(stream=stream, IDs=self.ids, Logits=logits, Prob=self.prob, **bias)

    def place(self, ids, stream=None):
        """Experts of every token's routes, int32 in [0, experts) -> the order of the slots: by expert, then by token (`slot_map`, `slot_token`)."""
        _check_rows(ids, self.tokens, self.top_k, torch.int32, self.device, "ids")
        self._call(self._place, ids, stream=stream)
        self.placed = True
        return self.slot_map

    def _check_placed(self):
        if not self.placed:
            raise RuntimeError("the routes have no places yet: `place` comes before `up` and `down`")

    def _place(self, ids, stream):
        self.k_metadata(stream=stream, Counts=self.counts, IDs=ids, RelativeSlot=self.relative, RowMax=None, RowOffsets=self.row_offsets, SlotMap=self.slot_map,
                        SlotToken=self.slot_token, TileCount=self.tile_count, TileExpert=self.tile_expert, TileOffsets=self.tile_offsets, TileRow=self.tile_row,
                        TileUnits=self.tile_units, Workspace=self.segments)

    def up(self, x, stream=None):
        """Rows (tokens, hidden) -> silu(gate) * up of every route, (tokens * top_k, intermediate) in the order of the slots, of the layer's dtype both."""
        _check_rows(x, self.tokens, self.hidden, self.dtype, self.device, "x")
        self._check_placed()
        self._call(self._up, x, stream=stream)
        return self.act

    def down(self, act, prob, shared=None, shared_gate=None, stream=None):
        """Rows in the order of the slots and fp32 weights (tokens, top_k) -> (tokens, hidden): the weighted sum, in fp32, of the routes' second products (those of weight 0 count nothing) and, where they are given,
        of sigmoid(shared_gate) (tokens) times shared (tokens, hidden); rows, result and these two of the layer's dtype."""
        _check_rows(act, self.assignments, self.inter, self.dtype, self.device, "act")
        _check_rows(prob, self.tokens, self.top_k, torch.float32, self.device, "prob")
        if (shared is None) != (shared_gate is None):
            raise ValueError("shared and shared_gate go together")
        if shared is not None:
            _check_rows(shared, self.tokens, self.hidden, self.dtype, self.device, "shared")
            _check_rows(shared_gate.view(-1, 1), self.tokens, 1, self.dtype, self.device, "shared_gate")
        self._check_placed()
        self._call(self._down, act, prob, shared, shared_gate, stream=stream)
        return self.out

    def _down(self, act, prob, shared, shared_gate, stream):
        self._second_products(act, stream)
        self.k_combine(stream=stream, Expert=self.down_out, Output=self.out, Prob=prob, Shared=shared, SharedGate=shared_gate, SlotMap=self.slot_map)

    def run(self, x, logits, shared=None, shared_gate=None, stream=None):
        self.route(logits, stream=stream)
        self.place(self.ids, stream=stream)
        return self.down(self.up(x, stream=stream), self.prob, shared, shared_gate, stream=stream)


class Mxfp4MoeLayer(_ExpertLayer):
    """Routed experts with MXFP4 weights for `tokens` rows: router, places of the routes, gate | up with SwiGLU, down, weighted sum.

    gate_up (E, 2 I, H / 2) and gate_up_exponents (E, 2 I, H / 32): gate channels, then up channels; down (E, H, I / 2), down_exponents (E, H, I / 32); uint8.
    scoring, bias (E fp32 values added for the choice only), groups, top_groups, group_best, renormalize and scale: the router's (k_router_scores.hip); as they stand here, the softmax router.
    dtype: of the rows, the shared expert's values, the activations between the two products and the result, torch.float16 or torch.bfloat16.  An activation beyond fp16's 65504 becomes
    infinite there, its block of 32 NaN and so its token's result: bfloat16 is for layers whose activations leave fp16's range.
    `run` does all of it; `route`, `place`, `up` and `down` are its parts, for a caller with routes of its own (`place` before `up` and `down`).  They work on the object's buffers: one stream at a time."""

    def __init__(self, tokens, experts, top_k, hidden, intermediate, gate_up, gate_up_exponents, down, down_exponents, *, scoring="softmax", bias=None, groups=1,
                 top_groups=None, group_best=2, renormalize=True, scale=1.0, block_m=None, dtype=torch.float16):
        if dtype not in (torch.float16, torch.bfloat16):
            raise ValueError("dtype must be torch.float16 or torch.bfloat16")
        if tuple(gate_up.shape) != (experts, 2 * intermediate, hidden // 2) or tuple(down.shape) != (experts, hidden, intermediate // 2):
            raise ValueError(f"gate_up must be ({experts}, {2 * intermediate}, {hidden // 2}) and down ({experts}, {hidden}, {intermediate // 2}), "
                             f"not {tuple(gate_up.shape)} and {tuple(down.shape)}")
        weights = tuple(map(torch.as_tensor, (gate_up, gate_up_exponents, down, down_exponents)))
        self.device = self._device_of(*weights)
        self.w1, self.p1 = (t.to(self.device) for t in mxfp4.tiles(*weights[:2], paired=True))
        self.w2, self.p2 = (t.to(self.device) for t in mxfp4.tiles(*weights[2:]))
        routes = tokens * top_k
        if block_m is None:
            block_m = 16 if routes <= 10 * experts else 64 if routes < 192 * experts else 128 if routes < 512 * experts else 256
        self._set_up(tokens, experts, top_k, hidden, intermediate, dtype, block_m, scoring=scoring, bias=bias, groups=groups, top_groups=top_groups, group_best=group_best,
                     renormalize=renormalize, scale=scale)
        name = mxfp4.dtype_name(dtype)
        with torch.cuda.device(self.device):
            self.k_quantise_tokens = Kernel("mxfp4_quantization", M=tokens, K=hidden, input_dtype=name, pad=mxfp4.STEP)
            up = dict(N=2 * intermediate, K=hidden, gather=True, epilogue="swiglu", output_dtype=name, **self.grouped)
            self.k_up = Kernel("mxfp4_grouped", **up)
            self.k_quantise_act = Kernel("mxfp4_quantization", M=routes, K=intermediate, input_dtype=name, pad=mxfp4.STEP)
            down = dict(N=hidden, K=intermediate, output_dtype="float32", **self.grouped)
            self.k_down = Kernel("mxfp4_grouped", **down)
            # A route to an expert or less: the products quantise their rows themselves where these are fp16, one launch instead of two (us without / with it: 128 experts x 8 of 2048 x 512, 3 tokens, up
            # 7.6 / 6.0 and down 5.1 / 4.4, 8 tokens 9.7 / 8.5 and 7.4 / 7.3, 16 tokens 10.7 / 10.7 and 8.9 / 10.3; 16 x 2 of 4096 x 1536, 8 tokens, 10.7 / 9.9 and 7.9 / 6.6).
            few = block_m == 16 and dtype == torch.float16
            self.few_up = _where_it_fits("mxfp4_grouped", input_dtype="float16", **up) if few and routes <= experts else None
            self.few_down = _where_it_fits("mxfp4_grouped", input_dtype="float16", **down) if few and 4 * routes <= 3 * experts else None
        u8 = dict(dtype=torch.uint8, device=self.device)
        wide, inner = mxfp4.padded(hidden), mxfp4.padded(intermediate)
        self.a_q, self.a_s = torch.empty((tokens, wide // 2), **u8), torch.empty((tokens, wide // 32), **u8)
        self.h_q, self.h_s = torch.empty((routes, inner // 2), **u8), torch.empty((routes, inner // 32), **u8)

    def _up(self, x, stream):
        if self.few_up is not None and _apart(x, self.act):  # (as Mxfp4Linear's)
            self.few_up(stream=stream, A=x, Out=self.act, SlotToken=self.slot_token, W=self.w1, WS=self.p1, TileCount=self.tile_count, TileUnits=self.tile_units)
            return
        self.k_quantise_tokens(stream=stream, Q=self.a_q, S=self.a_s, X=x, rows=self.tokens)
        self.k_up(stream=stream, A=self.a_q, AS=self.a_s, Out=self.act, SlotToken=self.slot_token, W=self.w1, WS=self.p1, TileCount=self.tile_count, TileUnits=self.tile_units)

    def _second_products(self, act, stream):
        if self.few_down is not None:
            self.few_down(stream=stream, A=act, Out=self.down_out, W=self.w2, WS=self.p2, TileCount=self.tile_count, TileUnits=self.tile_units)
            return
        self.k_quantise_act(stream=stream, Q=self.h_q, S=self.h_s, X=act, rows=self.assignments)
        self.k_down(stream=stream, A=self.h_q, AS=self.h_s, Out=self.down_out, W=self.w2, WS=self.p2, TileCount=self.tile_count, TileUnits=self.tile_units)


class Int8Linear(_OnDevice):
    """Rows of 16-bit values, quantised to 8-bit integers with a scale (zero_points: and a zero point) for each, times weights (N, K) of int8 with fp32 scales (N), plus a bias (N) if one is given,
    up to `capacity` rows at a time (the rules: int8.py).  K is up to 65536.  epilogue="swiglu": the upper half of the channels are the up channels of the gate channels in the lower half, and
    silu(gate) * up comes out.  `run` returns the object's own output buffer, or a view of its first rows, which the next call overwrites; one object serves one stream at a time."""

    def __init__(self, weight, scale, capacity, *, bias=None, zero_points=False, dtype=torch.float16, epilogue="none"):
        if dtype not in (torch.float16, torch.bfloat16):
            raise ValueError("dtype must be torch.float16 or torch.bfloat16")
        weight, scale = torch.as_tensor(weight), torch.as_tensor(scale)
        if weight.ndim != 2 or weight.dtype != torch.int8:
            raise ValueError("weight must be int8 (N, K)")
        if not 0 < capacity <= 1 << 24:
            raise ValueError("capacity must be 1 to 2^24 rows")
        self.capacity, self.dtype, self.zero_points = capacity, dtype, bool(zero_points)
        channels, self.k = weight.shape
        bias = None if bias is None else torch.as_tensor(bias)
        if scale.shape != (channels,) or (bias is not None and bias.shape != (channels,)):
            raise ValueError(f"scale and bias must have {channels} values")
        self.device = self._device_of(weight, scale, *([] if bias is None else [bias]))
        paired = epilogue == "swiglu"
        self.weight = byte_tiles.tiles(weight, paired).to(self.device)
        self.channel = dict(WS=byte_tiles.channels(scale.float(), paired).to(self.device))
        if bias is not None:
            self.channel["Bias"] = byte_tiles.channels(bias.float(), paired).to(self.device)
        if self.zero_points:
            self.channel["WSum"] = byte_tiles.channels(weight.sum(1, dtype=torch.int32), paired).to(self.device)
        name = int8.dtype_name(dtype)
        shape = dict(N=channels, K=self.k, dynamic_rows=True, zero_points=self.zero_points, bias=bias is not None, epilogue=epilogue, output_dtype=name)
        with torch.cuda.device(self.device):
            self.projection = Kernel("int8_token_projection", M=capacity, **shape)
            self.quantizer = Kernel("int8_token_quantization", M=capacity, K=self.k, input_dtype=name, zero_points=self.zero_points, layout="tiles")
            # Few rows: the projection quantises them itself, every workgroup all of them, one launch instead of two.  us, two and one:
            #   no zero points, no SwiGLU: 4096 x 4096, 1 row 9.0 and 8.0, 8 9.1 and 9.2; 17408 x 5120, 1 22.9 and 20.4, 4 23.4 and 22.0; 9728 x 2560, 8 12.0 and 10.6; 24576 x 1536, 8 13.7 and 12.3;
            #   zero points: 9728 x 2560, 4 12.6 and 10.7, 8 12.7 and 12.3; 8192 x 4096, 4 level, 8 11.8 and 13.9; 17408 x 5120, 4 23.4 and 22.4;
            #   SwiGLU: 9728 x 2560, 8 12.1 and 11.1; 8192 x 4096, 4 11.3 and 10.5, 8 11.6 and 12.2; 17408 x 5120, 2 level, 4 23.4 and 25.9; 8192 x 8192, 2 17.4 and 15.6, 4 17.7 and 18.4;
            #   both: 9728 x 2560, 8 level; 8192 x 4096, 4 11.0 and 10.2, 8 12.0 and 13.7; 17408 x 5120, 2 22.8 and 23.5, 4 23.6 and 26.8.
            # Not where their codes do not fit LDS, or a row its threads.
            most = 2 if paired and self.k > 4096 else 4 if (paired or self.zero_points) and self.k > 2560 else 8
            self.few, self.few_rows = None, 0
            for rows in (8, 4, 2, 1):
                if self.few is None and rows <= most:
                    self.few_rows = min(rows, capacity)
                    self.few = _where_it_fits("int8_token_projection", M=self.few_rows, input_dtype=name, **shape)
        self.n = channels // 2 if paired else channels
        # the quantised rows, by tiles of 16
        self.a_q = torch.empty((-(-capacity // 16), int8.steps(self.k), 2048), dtype=torch.int8, device=self.device)
        self.a_s = torch.empty(capacity, dtype=torch.float32, device=self.device)
        self.a_z = torch.empty(capacity, dtype=torch.int32, device=self.device) if self.zero_points else None
        self.out = torch.empty((capacity, self.n), dtype=dtype, device=self.device)

    def run(self, x, stream=None):
        _check_rows(x, None, self.k, self.dtype, self.device, "x")
        rows = x.shape[0]
        if rows > self.capacity:
            raise ValueError(f"{rows} rows are more than the capacity of {self.capacity}")
        if rows:
            self._call(self._run, x, rows, stream=stream)
        return self.out if rows == self.capacity else self.out.as_strided((rows, self.n), (self.n, 1))

    def _run(self, x, rows, stream):
        if rows <= self.few_rows and self.few is not None and _apart(x, self.out):  # (as Mxfp4Linear's)
            self.few(stream=stream, A=x, Out=self.out, W=self.weight, m=rows, **self.channel)
            return
        zero = ({"Z": self.a_z}, {"AZ": self.a_z}) if self.zero_points else ({}, {})
        self.quantizer(stream=stream, Q=self.a_q, S=self.a_s, X=x, rows=rows, **zero[0])
        self.projection(stream=stream, A=self.a_q, AS=self.a_s, Out=self.out, W=self.weight, m=rows, **zero[1], **self.channel)


def _unit_rows(routes, experts, hidden, intermediate, expert_bytes):
    """Rows to a unit of the experts' products, by the routes that an expert has in the mean and by the tiles of 64 x 128 that both products have at one unit to an expert: where these are few, short
    units spread the work over the GPU.  Measured at 892 banks (4 to 256 experts of 256 to 4096 and 128 to 1536, int8 and bf16, 5 to 400 routes to an expert, popularity like 1 / rank^1.1 or even):
    this rule's units take 1.01 times the best of the three in the geometric mean, 1.09 at the 95th and 1.19 at the 99th percentile; bounds of 8 and 30 routes whatever the bank 1.20, 1.98, 2.64.
    Times with units of 64 over those with 16, and of 128 over 64 (int8, popularity skewed and even; bf16 is within 0.2 of these):
        3072 tiles, 128 experts of 2048 and 512: 8 routes to an expert 0.97 and 1.05, 12 0.95 and 1.01, 16 0.89 and 0.84; 36 1.01 and 1.02, 56 0.98 and 0.93;
        1200, 60 of 1024 and 768: 8 1.10 and 1.12, 12 1.02 and 1.11, 16 0.98 and 0.98; 44 1.11 and 1.06, 64 1.02 and 0.88;
        896, 16 of 4096 and 1536: 8 1.01 and 1.06, 14 0.95 and 0.92; 44 1.07 and 1.00, 64 0.98 and 0.81;
        192, 8 of 1024 and 1024: 20 1.70 and 1.59, 48 1.40 and 1.41, 96 1.03 and 1.03; 256 1.12 and 1.14, 512 1.06 and 1.07;
        32, 8 of 256 and 128: 64 1.61 and 1.65, 256 1.18 and 1.18; 512 1.42 and 1.42.
    Kernels of 64 and 128 rows count the bytes of an expert's matrix in 32 bits."""
    tiles = experts * (-(-2 * intermediate // 128) + -(-hidden // 128))
    short, long = max(8, 12288 // tiles), max(48, 81920 // tiles)
    return 16 if routes < short * experts or expert_bytes >= 1 << 32 else 64 if routes < long * experts else 128


def _check_experts(gate_up, down, experts, hidden, intermediate, dtypes):
    if experts < 1:
        raise ValueError("there must be at least one expert")
    if tuple(gate_up.shape) != (experts, 2 * intermediate, hidden) or tuple(down.shape) != (experts, hidden, intermediate):
        raise ValueError(f"gate_up must be ({experts}, {2 * intermediate}, {hidden}) and down ({experts}, {hidden}, {intermediate}), not {tuple(gate_up.shape)} and {tuple(down.shape)}")
    if gate_up.dtype not in dtypes or down.dtype != gate_up.dtype:
        raise ValueError(f"gate_up and down must both be {' or '.join(map(str, dtypes))}, not {gate_up.dtype} and {down.dtype}")


class Int8MoeLayer(_ExpertLayer):
    """Routed experts with weights of 8-bit integers and fp32 scales for each channel, for `tokens` rows that are quantised with a scale for each (int8.py): router, places of the routes,
    gate | up with SwiGLU, down, weighted sum.

    gate_up (E, 2 I, H) int8 with gate_up_scale (E, 2 I): gate channels, then up channels; down (E, H, I) int8 with down_scale (E, H).
    scoring, bias (E fp32 values added for the choice only), groups, top_groups, group_best, renormalize and scale: the router's (k_router_scores.hip); as they stand here, the softmax router.
    dtype: of the rows, the shared expert's values, the activations between the two products and the result, torch.float16 or torch.bfloat16.  An activation beyond fp16's 65504 becomes
    infinite there and its token's result NaN: bfloat16 is for layers whose activations leave fp16's range.
    `run` does all of it; `route`, `place`, `up` and `down` are its parts, for a caller with routes of its own (`place` before `up` and `down`).  They work on the object's buffers: one stream at a time."""

    def __init__(self, tokens, experts, top_k, hidden, intermediate, gate_up, gate_up_scale, down, down_scale, *, scoring="softmax", bias=None, groups=1,
                 top_groups=None, group_best=2, renormalize=True, scale=1.0, block_m=None, dtype=torch.float16):
        if dtype not in (torch.float16, torch.bfloat16):
            raise ValueError("dtype must be torch.float16 or torch.bfloat16")
        gate_up, gate_up_scale, down, down_scale = map(torch.as_tensor, (gate_up, gate_up_scale, down, down_scale))
        _check_experts(gate_up, down, experts, hidden, intermediate, (torch.int8,))
        if tuple(gate_up_scale.shape) != (experts, 2 * intermediate) or tuple(down_scale.shape) != (experts, hidden):
            raise ValueError(f"gate_up_scale must be ({experts}, {2 * intermediate}) and down_scale ({experts}, {hidden}), not {tuple(gate_up_scale.shape)} and {tuple(down_scale.shape)}")
        self.device = self._device_of(gate_up, gate_up_scale, down, down_scale)
        self.w1, self.s1 = byte_tiles.tiles(gate_up, paired=True).to(self.device), byte_tiles.channels(gate_up_scale.float(), paired=True).to(self.device)
        self.w2, self.s2 = byte_tiles.tiles(down).to(self.device), byte_tiles.channels(down_scale.float()).to(self.device)
        routes = tokens * top_k
        if block_m is None:
            block_m = _unit_rows(tokens * top_k, experts, hidden, intermediate, max(self.w1.nbytes, self.w2.nbytes) // experts)
        self._set_up(tokens, experts, top_k, hidden, intermediate, dtype, block_m, scoring=scoring, bias=bias, groups=groups, top_groups=top_groups, group_best=group_best,
                     renormalize=renormalize, scale=scale)
        name = int8.dtype_name(dtype)
        with torch.cuda.device(self.device):
            self.k_quantise_tokens = Kernel("int8_token_quantization", M=tokens, K=hidden, input_dtype=name)
            self.k_quantise_act = Kernel("int8_token_quantization", M=routes, K=intermediate, input_dtype=name)
            up = dict(N=2 * intermediate, K=hidden, gather=True, epilogue="swiglu", output_dtype=name, **self.grouped)
            down = dict(N=hidden, K=intermediate, output_dtype="float32", **self.grouped)
            self.k_up, self.k_down = Kernel("int8_token_grouped", **up), Kernel("int8_token_grouped", **down)
            # Few routes: the products quantise their rows themselves, one launch instead of two, but every workgroup again (32 gate | up channels or 16 down channels to one): values that
            # are quantised up to 2^21.  (us, two launches and one: 128 experts of 2048 and 512, up 16 routes, 2^20: 11.2 and 9.5, 64, 2^22: 25.0 and 25.6; down 16, 2^20: 9.3 and 7.4, 64,
            # 2^22: 14.4 and 17.6; 16 experts of 4096 and 1536, up 2, 0.8 10^6: 10.6 and 8.4, 8, 3.1 10^6: 23.3 and 26.7; down 2: 8.6 and 6.3, 8: 13.6 and 17.6.)
            few_up, few_down = block_m == 16 and routes * -(-intermediate // 16) * hidden < 1 << 21, block_m == 16 and routes * -(-hidden // 16) * intermediate < 1 << 21
            self.few_up = _where_it_fits("int8_token_grouped", input_dtype=name, **up) if few_up else None
            self.few_down = _where_it_fits("int8_token_grouped", input_dtype=name, **down) if few_down else None
        i8, f32 = dict(dtype=torch.int8, device=self.device), dict(dtype=torch.float32, device=self.device)
        self.a_q, self.a_s = torch.empty((tokens, int8.padded(hidden)), **i8), torch.empty(tokens, **f32)
        self.h_q, self.h_s = torch.empty((routes, int8.padded(intermediate)), **i8), torch.empty(routes, **f32)

    def _up(self, x, stream):
        if self.few_up is not None and _apart(x, self.act):  # (as Mxfp4Linear's)
            self.few_up(stream=stream, A=x, Out=self.act, SlotToken=self.slot_token, W=self.w1, WS=self.s1, TileCount=self.tile_count, TileUnits=self.tile_units)
            return
        self.k_quantise_tokens(stream=stream, Q=self.a_q, S=self.a_s, X=x, rows=self.tokens)
        self.k_up(stream=stream, A=self.a_q, AS=self.a_s, Out=self.act, SlotToken=self.slot_token, W=self.w1, WS=self.s1, TileCount=self.tile_count, TileUnits=self.tile_units)

    def _second_products(self, act, stream):
        if self.few_down is not None:
            self.few_down(stream=stream, A=act, Out=self.down_out, W=self.w2, WS=self.s2, TileCount=self.tile_count, TileUnits=self.tile_units)
            return
        self.k_quantise_act(stream=stream, Q=self.h_q, S=self.h_s, X=act, rows=self.assignments)
        self.k_down(stream=stream, A=self.h_q, AS=self.h_s, Out=self.down_out, W=self.w2, WS=self.s2, TileCount=self.tile_count, TileUnits=self.tile_units)


class HalfMoeLayer(_ExpertLayer):
    """Routed experts with weights of fp16 or bf16 for `tokens` rows of that type: router, places of the routes, gate | up with SwiGLU, down, weighted sum; products and sums in fp32.

    gate_up (E, 2 I, H): gate channels, then up channels; down (E, H, I); H and I are multiples of 8, and the rows given to `up` and `down` start at addresses that are multiples of 16.
    The router's arguments: as Int8MoeLayer's.  An activation beyond fp16's 65504 becomes infinite there: bf16 is for layers whose activations leave fp16's range.
    `run` does all of it; `route`, `place`, `up` and `down` are its parts, for a caller with routes of its own (`place` before `up` and `down`).  They work on the object's buffers: one stream at a time."""

    def __init__(self, tokens, experts, top_k, hidden, intermediate, gate_up, down, *, scoring="softmax", bias=None, groups=1, top_groups=None, group_best=2, renormalize=True, scale=1.0,
                 block_m=None):
        gate_up, down = torch.as_tensor(gate_up), torch.as_tensor(down)
        _check_experts(gate_up, down, experts, hidden, intermediate, (torch.float16, torch.bfloat16))
        self.device = self._device_of(gate_up, down)
        self.w1, self.w2 = byte_tiles.tiles(gate_up, paired=True).to(self.device), byte_tiles.tiles(down).to(self.device)
        if block_m is None:
            block_m = _unit_rows(tokens * top_k, experts, hidden, intermediate, max(self.w1.nbytes, self.w2.nbytes) // experts)
        self._set_up(tokens, experts, top_k, hidden, intermediate, gate_up.dtype, block_m, scoring=scoring, bias=bias, groups=groups, top_groups=top_groups, group_best=group_best,
                     renormalize=renormalize, scale=scale)
        name = int8.dtype_name(gate_up.dtype)
        with torch.cuda.device(self.device):
            self.k_up = Kernel("half_grouped", N=2 * intermediate, K=hidden, gather=True, dtype=name, epilogue="swiglu", output_dtype=name, **self.grouped)
            self.k_down = Kernel("half_grouped", N=hidden, K=intermediate, dtype=name, output_dtype="float32", **self.grouped)

    def _up(self, x, stream):
        if not _apart(x, self.act):  # (workgroups that have ended would write over what others have yet to read)
            with torch.cuda.stream(torch.cuda.ExternalStream(stream, device=self.device)):
                x = x.clone()
        self.k_up(stream=stream, A=x, Out=self.act, SlotToken=self.slot_token, W=self.w1, TileCount=self.tile_count, TileUnits=self.tile_units)

    def _second_products(self, act, stream):
        self.k_down(stream=stream, A=act, Out=self.down_out, W=self.w2, TileCount=self.tile_count, TileUnits=self.tile_units)
