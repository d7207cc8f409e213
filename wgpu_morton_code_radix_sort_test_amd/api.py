"""Host-side mirror of the C ABI: contexts and sort plans over torch device tensors.

torch is used for device memory and streams only; every computation is a call
into libmrs.so.  Buffer roles follow the reference's `Buffers` struct
(src/types.rs:68-77): `morton_codes`/`morton_codes_2` are keys A/B and
`indices`/`indices_2` are payload A/B of `SortPlan.sort_pairs`.
"""
import ctypes
from dataclasses import dataclass, field
from typing import Optional

import torch

from . import _lib

ALGO_THREE_KERNEL = 0
ALGO_ONESWEEP = 1
ALGO_HYBRID = 2

GATE_SOFTMAX = 0
GATE_SIGMOID = 1

MORTON_UNIFORMS_BYTES = 51248
VERTEX_STRIDE = 48
TRIANGLE_STRIDE = 16


def _ptr(t):
    if t is None:
        return None
    if not t.is_cuda:
        raise ValueError("expected a device tensor")
    if not t.is_contiguous():
        raise ValueError("expected a contiguous tensor")
    return ctypes.c_void_p(t.data_ptr())


def _nbytes(t):
    return t.numel() * t.element_size()


def _stream(stream):
    if stream is None:
        stream = torch.cuda.current_stream()
    return ctypes.c_void_p(stream.cuda_stream)


@dataclass
class PlanInfo:
    num_passes: int
    radix: int
    tile_items: int
    threads: int
    max_tiles: int
    histogram_len: int
    temp_bytes: int


class Context:
    """`mrs_context`: one per GPU (replaces device acquisition, src/main.rs:692-707)."""

    def __init__(self, device=0):
        self.lib = _lib.load_library()
        self.device = torch.device("cuda", device if isinstance(device, int) else device.index)
        torch.cuda.set_device(self.device)
        handle = ctypes.c_void_p()
        _lib.check(self.lib.mrs_context_create(self.device.index, ctypes.byref(handle)))
        self._h = handle

    ATTR_COMPUTE_UNITS = 0
    ATTR_RANK_MODE = 1
    ATTR_DIE_AWARE_TICKETS = 2
    ATTR_NOALLOC_TIMEOUT = 3
    ATTR_ROCTX_RANGES = 4
    # aids for tests and A/B runs: a plan copies them from its context when it is created
    ATTR_TEST_HYBRID_MIN_N = 5
    ATTR_TEST_HYBRID_LEADING_BITS = 6
    ATTR_TEST_HYBRID_FORCE_FALLBACK = 7
    ATTR_TEST_NO_SMALL_SORT = 8
    ATTR_TEST_NO_PASS_SKIP = 9
    ATTR_TEST_WIDE_STATUS = 10
    ATTR_TEST_HYBRID_FORCE_ADAPTIVE = 11
    ATTR_TEST_HYBRID_NO_ADAPTIVE = 12
    ATTR_TEST_HYBRID_CAPACITY = 13
    ATTR_TEST_HYBRID_BIG_LOCAL = 14
    NOALLOC_MAX_N = 1 << 26

    def attribute(self, which):
        """`mrs_context_get_attribute`: what the context found on its device."""
        value = ctypes.c_int64()
        _lib.check(self.lib.mrs_context_get_attribute(self._h, int(which), ctypes.byref(value)))
        return int(value.value)

    def set_attribute(self, which, value):
        """`mrs_context_set_attribute`."""
        _lib.check(self.lib.mrs_context_set_attribute(self._h, int(which), int(value)))

    @property
    def rank_mode(self):
        """"atomic" (returning LDS atomics) or "match" (ballot matching)."""
        return "atomic" if self.attribute(self.ATTR_RANK_MODE) == 1 else "match"

    def close(self):
        if self._h:
            self.lib.mrs_context_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    # ---- Morton encoders -------------------------------------------------
    def morton_encode30(self, xyz, mn, mx, keys_out=None, idx_out=None, stream=None, keys_only=False):
        """30-bit Morton keys + index payload of an [n, 3] f32 point tensor.  `keys_only`: no index
        array is written (for SortPlan.sort_pairs_indexed); the second value returned is None."""
        n = xyz.numel() // 3
        if xyz.dtype != torch.float32:
            raise ValueError("xyz must be float32")
        if keys_out is None:
            keys_out = torch.empty(n, dtype=torch.int32, device=self.device)
        if idx_out is None and not keys_only:
            idx_out = torch.empty(n, dtype=torch.int32, device=self.device)
        if keys_out.numel() < n or (idx_out is not None and idx_out.numel() < n):
            raise ValueError("output tensors are too small")
        c3 = ctypes.c_float * 3
        _lib.check(
            self.lib.mrs_morton_encode30(
                self._h, _ptr(xyz), n, c3(*[float(v) for v in mn]), c3(*[float(v) for v in mx]),
                _ptr(keys_out), _ptr(idx_out) if idx_out is not None else None, _stream(stream),
            )
        )
        return keys_out, idx_out

    def morton_encode_lut(self, uniforms, vertices, triangles, codes_out=None, stream=None):
        """Extended Morton codes from the reference's buffer layouts (bytes tensors)."""
        if _nbytes(uniforms) != MORTON_UNIFORMS_BYTES:
            raise ValueError(f"uniforms must be {MORTON_UNIFORMS_BYTES} bytes")
        if _nbytes(vertices) % VERTEX_STRIDE or _nbytes(triangles) % TRIANGLE_STRIDE:
            raise ValueError("vertices must have stride 48 and triangles stride 16")
        n = _nbytes(triangles) // TRIANGLE_STRIDE
        nv = _nbytes(vertices) // VERTEX_STRIDE
        if codes_out is None:
            codes_out = torch.empty(2 * n, dtype=torch.int32, device=self.device)
        if _nbytes(codes_out) < 8 * n:
            raise ValueError("codes_out is too small")
        _lib.check(
            self.lib.mrs_morton_encode_lut(
                self._h, _ptr(uniforms), _ptr(vertices), nv, _ptr(triangles), n, _ptr(codes_out), _stream(stream)
            )
        )
        return codes_out

    # ---- the sort without a plan and without allocations ---------------------------
    def sort_pairs_noalloc(self, keys_a, vals_a, keys_b, vals_b, n, begin_bit=0, end_bit=32, stream=None):
        """`mrs_sort_pairs_noalloc`: (u32 key, u32 payload) pairs, temporary memory in the library's
        static scratch array (n <= NOALLOC_MAX_N).  Returns True when the result is in the B tensors."""
        for t in (keys_a, vals_a, keys_b, vals_b):
            if t is None or _nbytes(t) < 4 * n:
                raise ValueError("tensor is missing or too small")
        in_b = ctypes.c_int(0)
        _lib.check(
            self.lib.mrs_sort_pairs_noalloc(self._h, n, _ptr(keys_a), _ptr(vals_a), _ptr(keys_b), _ptr(vals_b),
                                            begin_bit, end_bit, _stream(stream), ctypes.byref(in_b))
        )
        return bool(in_b.value)

    # ---- generators ----------------------------------------------------------
    def generate_points(self, seed, n, stream=None):
        xyz = torch.empty((n, 3), dtype=torch.float32, device=self.device)
        _lib.check(self.lib.mrs_generate_points(self._h, seed, n, _ptr(xyz), _stream(stream)))
        return xyz

    def generate_u32(self, seed, stream_id, n, stream=None):
        out = torch.empty(n, dtype=torch.int32, device=self.device)
        _lib.check(self.lib.mrs_generate_u32(self._h, seed, stream_id, n, _ptr(out), _stream(stream)))
        return out

    # ---- multi-GPU building block ----------------------------------------------
    def bucket_histogram(self, keys, n, key_words, shift, bits, stream=None):
        counts = torch.empty(1 << bits, dtype=torch.int64, device=self.device)
        _lib.check(
            self.lib.mrs_bucket_histogram(self._h, _ptr(keys), n, key_words, shift, bits, _ptr(counts), _stream(stream))
        )
        return counts


class SortPlan:
    """`mrs_plan`: owns the temporaries of one sort shape (src/main.rs:31-85, 236-253)."""

    def __init__(self, ctx, n, key_words=1, payload_bytes=4, digit_bits=8, begin_bit=0, end_bit=None,
                 algo=ALGO_ONESWEEP, tile_items=0):
        self.ctx = ctx
        self.lib = ctx.lib
        if end_bit is None:
            end_bit = 32 * key_words
        self.desc = _lib.PlanDesc(n, key_words, payload_bytes, digit_bits, begin_bit, end_bit, algo, tile_items)
        handle = ctypes.c_void_p()
        _lib.check(self.lib.mrs_plan_create(ctx._h, ctypes.byref(self.desc), ctypes.byref(handle)))
        self._h = handle
        raw = _lib.PlanInfoStruct()
        _lib.check(self.lib.mrs_plan_get_info(self._h, ctypes.byref(raw)))
        self.info = PlanInfo(raw.num_passes, raw.radix, raw.tile_items, raw.threads, raw.max_tiles,
                             raw.histogram_len, raw.temp_bytes)
        self.n = n
        self.key_words = key_words
        self.payload_bytes = payload_bytes

    def close(self):
        if self._h:
            self.lib.mrs_plan_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _check_sizes(self, n, keys, vals):
        for k in keys:
            if k is not None and _nbytes(k) < 4 * self.key_words * n:
                raise ValueError("key tensor is too small")
        if self.payload_bytes:
            for v in vals:
                if v is None or _nbytes(v) < self.payload_bytes * n:
                    raise ValueError("payload tensor is missing or too small")

    def num_tiles(self, n):
        return (n + self.info.tile_items - 1) // self.info.tile_items

    def sort_pairs(self, keys_a, vals_a, keys_b, vals_b, n=None, stream=None):
        """Sorts; returns True when the result is in the B tensors (odd pass count)."""
        n = self.n if n is None else n
        self._check_sizes(n, (keys_a, keys_b), (vals_a, vals_b))
        in_b = ctypes.c_int(0)
        _lib.check(
            self.lib.mrs_sort_pairs(self._h, n, _ptr(keys_a), _ptr(vals_a), _ptr(keys_b), _ptr(vals_b),
                                    _stream(stream), ctypes.byref(in_b))
        )
        return bool(in_b.value)

    def sort_pairs_primed(self, keys_a, vals_a, keys_b, vals_b, n=None, stream=None):
        """`mrs_sort_pairs_primed`: sort_pairs that uses the histograms morton_encode30_for_sort left
        in this plan for exactly these keys (raises MrsError if the plan does not hold them)."""
        n = self.n if n is None else n
        self._check_sizes(n, (keys_a, keys_b), (vals_a, vals_b))
        in_b = ctypes.c_int(0)
        _lib.check(
            self.lib.mrs_sort_pairs_primed(self._h, n, _ptr(keys_a), _ptr(vals_a), _ptr(keys_b), _ptr(vals_b),
                                           _stream(stream), ctypes.byref(in_b))
        )
        return bool(in_b.value)

    def sort_pairs_indexed(self, keys_a, vals_a, keys_b, vals_b, n=None, stream=None):
        """`mrs_sort_pairs_indexed`: sort_pairs whose input payload is the element index; vals_a is
        ping-pong space and need not hold anything.  Returns True when the result is in the B tensors."""
        n = self.n if n is None else n
        self._check_sizes(n, (keys_a, keys_b), (vals_a, vals_b))
        in_b = ctypes.c_int(0)
        _lib.check(
            self.lib.mrs_sort_pairs_indexed(self._h, n, _ptr(keys_a), _ptr(vals_a), _ptr(keys_b), _ptr(vals_b),
                                            _stream(stream), ctypes.byref(in_b))
        )
        return bool(in_b.value)

    def morton_encode30_for_sort(self, xyz, mn, mx, keys_out=None, idx_out=None, stream=None):
        """`mrs_morton_encode30_for_sort`: the encoder that also leaves the digit histograms of the
        keys in this plan; pass the returned key tensor to sort_pairs_primed as keys_a, unchanged."""
        n = xyz.numel() // 3
        if xyz.dtype != torch.float32:
            raise ValueError("xyz must be float32")
        if keys_out is None:
            keys_out = torch.empty(n, dtype=torch.int32, device=self.ctx.device)
        if idx_out is None:
            idx_out = torch.empty(n, dtype=torch.int32, device=self.ctx.device)
        if keys_out.numel() < n or idx_out.numel() < n:
            raise ValueError("output tensors are too small")
        c3 = ctypes.c_float * 3
        _lib.check(
            self.lib.mrs_morton_encode30_for_sort(
                self._h, _ptr(xyz), n, c3(*[float(v) for v in mn]), c3(*[float(v) for v in mx]),
                _ptr(keys_out), _ptr(idx_out), _stream(stream),
            )
        )
        return keys_out, idx_out

    def sort_gather(self, keys_a, keys_b, records_in, records_out, record_bytes, n=None, index_a=None, index_b=None,
                    stream=None):
        """`mrs_sort_gather`: sorts (key, source index) pairs and moves each record of
        `record_bytes` once.  Returns (result_in_b, sorted source indices)."""
        n = self.n if n is None else n
        if self.payload_bytes != 4:
            raise ValueError("sort_gather needs a plan with payload_bytes=4")
        if index_a is None:
            index_a = torch.empty(max(1, n), dtype=torch.int32, device=self.ctx.device)
        if index_b is None:
            index_b = torch.empty(max(1, n), dtype=torch.int32, device=self.ctx.device)
        self._check_sizes(n, (keys_a, keys_b), (index_a, index_b))
        if _nbytes(records_in) < n * record_bytes or _nbytes(records_out) < n * record_bytes:
            raise ValueError("record buffers are too small")
        in_b = ctypes.c_int(0)
        _lib.check(
            self.lib.mrs_sort_gather(self._h, n, _ptr(keys_a), _ptr(keys_b), _ptr(index_a), _ptr(index_b),
                                     _ptr(records_in), _ptr(records_out), record_bytes, _stream(stream),
                                     ctypes.byref(in_b))
        )
        return bool(in_b.value), (index_b if in_b.value else index_a)

    def histogram(self, keys, pass_number, n=None, hist_out=None, stream=None):
        n = self.n if n is None else n
        self._check_sizes(n, (keys,), ())
        length = self.info.radix * self.num_tiles(n)
        if hist_out is None:
            hist_out = torch.empty(length, dtype=torch.int32, device=self.ctx.device)
        if hist_out.numel() < length:
            raise ValueError("hist_out is too small")
        _lib.check(self.lib.mrs_histogram(self._h, n, _ptr(keys), pass_number, _ptr(hist_out), _stream(stream)))
        return hist_out

    def scan(self, hist, n=None, stream=None):
        n = self.n if n is None else n
        if hist.numel() < self.info.radix * self.num_tiles(n):
            raise ValueError("hist is too small")
        _lib.check(self.lib.mrs_scan(self._h, n, _ptr(hist), _stream(stream)))
        return hist

    def scatter(self, keys_in, vals_in, keys_out, vals_out, scanned, pass_number, n=None, stream=None):
        n = self.n if n is None else n
        self._check_sizes(n, (keys_in, keys_out), (vals_in, vals_out))
        if scanned.numel() < self.info.radix * self.num_tiles(n):
            raise ValueError("scanned histogram is too small")
        _lib.check(
            self.lib.mrs_scatter(self._h, n, _ptr(keys_in), _ptr(vals_in), _ptr(keys_out), _ptr(vals_out),
                                 _ptr(scanned), pass_number, _stream(stream))
        )

    def partition(self, keys_in, vals_in, keys_out, vals_out, shift, bits, bucket_map, num_parts, n=None,
                  stream=None):
        """Stable partition by bucket_map[(key >> shift) & mask]; returns u32[16] part sizes (device)."""
        n = self.n if n is None else n
        self._check_sizes(n, (keys_in, keys_out), (vals_in, vals_out))
        if bucket_map.dtype != torch.uint8 or bucket_map.numel() < (1 << bits):
            raise ValueError("bucket_map must be a uint8 tensor with 1 << bits entries")
        counts = torch.empty(16, dtype=torch.int32, device=self.ctx.device)
        _lib.check(
            self.lib.mrs_partition(self._h, n, _ptr(keys_in), _ptr(vals_in), _ptr(keys_out), _ptr(vals_out),
                                   shift, bits, _ptr(bucket_map), num_parts, _ptr(counts), _stream(stream))
        )
        return counts

    def set_timing(self, enable=True):
        _lib.check(self.lib.mrs_plan_set_timing(self._h, 1 if enable else 0))

    def timings(self):
        """[(label, milliseconds)] for every launch of the last sort_pairs call (timing must be on)."""
        cap = 96
        ms = (ctypes.c_float * cap)()
        labels = ctypes.create_string_buffer(32 * cap)
        count = ctypes.c_int(0)
        _lib.check(self.lib.mrs_plan_get_timings(self._h, cap, ms, labels, ctypes.byref(count)))
        out = []
        for i in range(count.value):
            raw = labels.raw[32 * i: 32 * i + 32]
            out.append((raw.split(b"\0", 1)[0].decode(), float(ms[i])))
        return out

    def check(self, stream=None):
        """Synchronises and raises MrsError if a look-back timed out on the device."""
        _lib.check(self.lib.mrs_plan_check(self._h, _stream(stream)))

    def passes_left_out(self, stream=None):
        """Synchronises; bit p is set if pass p of the last sort_pairs did not run on the device
        (64-bit keys whose digit p is the same for every key)."""
        mask = ctypes.c_uint32(0)
        _lib.check(self.lib.mrs_plan_get_passes_left_out(self._h, _stream(stream), ctypes.byref(mask)))
        return mask.value

    SCHEDULE_PASSES = 0
    SCHEDULE_MSD = 1
    SCHEDULE_MSD_REFUSED = 2
    SCHEDULE_MSD_ADAPTIVE = 3

    def schedule(self, stream=None):
        """`mrs_plan_get_schedule`: synchronises; (schedule the last sort ran, largest sub-bucket the
        device counted).  Only ALGO_HYBRID plans ever report anything but SCHEDULE_PASSES."""
        which, largest = ctypes.c_int32(0), ctypes.c_uint32(0)
        _lib.check(self.lib.mrs_plan_get_schedule(self._h, _stream(stream), ctypes.byref(which), ctypes.byref(largest)))
        return which.value, largest.value

    def oversized(self, stream=None):
        """`mrs_plan_get_oversized`: synchronises; (sub-buckets the last three-move sort found too large
        for a workgroup and sorted with its two extra passes, pairs they held, pairs a workgroup held)."""
        subs, pairs, cap = ctypes.c_uint32(0), ctypes.c_uint64(0), ctypes.c_uint32(0)
        _lib.check(self.lib.mrs_plan_get_oversized(self._h, _stream(stream), ctypes.byref(subs), ctypes.byref(pairs),
                                                   ctypes.byref(cap)))
        return subs.value, pairs.value, cap.value

    def adaptive(self, stream=None):
        """`mrs_plan_get_adaptive`: synchronises; (buckets, groups) the last sort was cut into if it
        ran SCHEDULE_MSD_ADAPTIVE, else zeros."""
        buckets, groups = ctypes.c_uint32(0), ctypes.c_uint32(0)
        _lib.check(self.lib.mrs_plan_get_adaptive(self._h, _stream(stream), ctypes.byref(buckets), ctypes.byref(groups)))
        return buckets.value, groups.value


# MRS_TYPE_* of the element types rows can have
_ROW_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_TYPE_8BIT = 3
# The current stream's handle without the Stream object around it, which takes 3 us to make.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", lambda index: torch.cuda.current_stream(index).cuda_stream)
_capturing = torch.cuda.is_current_stream_capturing


@dataclass(frozen=True)
class RouteMap:
    """`mrs_route_map`: int32 device tensors that say where every slot's row is.  `row_of_slot` [tokens,
    topk] holds a row or -1, `slot_of_row` [rows] a slot (token * topk + j) or -1, `counts` [experts] the rows an
    expert has, `offsets` [experts + 1] where its segment starts and, last, where all of them end.  `tokens` is how many the last
    `order` into this map had: entries of row_of_slot behind them say nothing.  None: no `order` was, all entries count."""

    row_of_slot: torch.Tensor
    slot_of_row: torch.Tensor
    counts: torch.Tensor
    offsets: torch.Tensor
    tokens: Optional[int] = field(default=None, compare=False)
    # a graph's replays write the map without a word here: once an ordering into it was captured, a second
    # number of tokens makes `tokens` -1, not known, for good
    _in_graph: bool = field(default=False, compare=False, repr=False)

    def _ordered(self, tokens, capturing):
        if (capturing or self._in_graph) and self.tokens is not None and self.tokens != tokens:
            tokens = -1
        object.__setattr__(self, "tokens", tokens)
        if capturing:
            object.__setattr__(self, "_in_graph", True)


class RoutePlan:
    """`mrs_route`: tokens routed to experts.  Every one of at most `tokens` tokens has `topk` slots; `select`
    picks their experts, `order` sorts the slots by expert, `dispatch` moves the tokens' rows into that
    order, `combine` brings them back weighted; the `*_backward` calls are the gradients.  An expert's rows start
    at a multiple of `align`; beyond `capacity` rows (0 = no limit) its later slots are dropped.  `gate`,
    `normalize` and `scale` say how scores become weights (include/mrs.h).  One handle runs one `order` at a time.
    Nothing is recorded for autograd: a training step makes the backward calls itself.

    Calls run on `stream` (the current one by default), and outputs they make belong to it.  As everywhere in torch, what a caller
    hands over from another stream is the caller's to keep in order: `stream` has to wait for what writes an input, and the input's memory
    must not be given back before the call has run (`Tensor.record_stream`, or a wait of the stream it was made on)."""

    def __init__(self, ctx, tokens, experts, topk, align=1, capacity=0, gate=GATE_SOFTMAX, normalize=True, scale=1.0):
        self._h = None
        self.ctx = ctx
        self.lib = ctx.lib
        self.device = ctx.device
        # a ctypes field keeps the low bits of a number that does not fit
        for name, v in (("tokens", tokens), ("capacity", capacity)):
            if v < 0:
                raise ValueError(f"{name} must not be negative")
            if v >= 1 << 64:
                raise ValueError(f"{name} = {v} does not fit 64 bits")
        for name, v in (("experts", experts), ("topk", topk), ("align", align), ("gate", gate)):
            if not -(1 << 31) <= v < 1 << 31:
                raise ValueError(f"{name} = {v} does not fit 32 bits")
        self.desc = _lib.RouteDesc(tokens, experts, topk, align, gate, capacity, 1 if normalize else 0, scale)
        rows = ctypes.c_uint64()
        _lib.check(self.lib.mrs_route_max_rows(ctypes.byref(self.desc), ctypes.byref(rows)))
        handle = ctypes.c_void_p()
        _lib.check(self.lib.mrs_route_create(ctx._h, ctypes.byref(self.desc), ctypes.byref(handle)))
        self._h = handle
        self.tokens, self.experts, self.topk = tokens, experts, topk
        self.max_rows = rows.value

    def close(self):
        if self._h:
            self.lib.mrs_route_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    # ---- checks: a call takes a few microseconds of host time, most of them here -----------------
    def _on_device(self, t, name):
        if t.device != self.device:
            raise ValueError(f"{name} is on {t.device}, the plan on {self.device}")

    def _rows(self, t, name, rows, hidden, dtype):
        """Pointer and row stride of a matrix whose rows are contiguous."""
        if t.device != self.device:
            self._on_device(t, name)
        if t.shape != (rows, hidden):
            raise ValueError(f"{name} must have shape [{rows}, {hidden}], not {list(t.shape)}")
        if t.dtype != dtype:
            raise ValueError(f"{name} must be {dtype}, not {t.dtype}")
        ld, step = t.stride()
        if step != 1 and hidden > 1:
            raise ValueError(f"the rows of {name} must be contiguous")
        if rows <= 1 and ld < hidden:
            ld = hidden
        return t.data_ptr(), ld

    def _per_slot(self, t, name, tokens, dtype):
        if t.device != self.device:
            self._on_device(t, name)
        if t.dtype != dtype or t.shape != (tokens, self.topk) or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape [{tokens}, {self.topk}]")
        return t.data_ptr()

    def _slots(self, t, name):
        if t.dim() != 2:
            raise ValueError(f"{name} must have two dimensions, not {t.dim()}")
        return t.size(0)

    def _map(self, route, tokens):
        """The map's structure for the library, and its number of rows."""
        device, int32 = self.device, torch.int32
        to_row, to_slot, counts, offsets = route.row_of_slot, route.slot_of_row, route.counts, route.offsets
        if not (to_row.device == to_slot.device == counts.device == offsets.device == device):
            raise ValueError(f"a tensor of the map is on another device than the plan, which is on {device}")
        if not (to_row.dtype is int32 and to_slot.dtype is int32 and counts.dtype is int32 and offsets.dtype is int32
                and to_row.is_contiguous() and to_slot.is_contiguous() and counts.is_contiguous() and offsets.is_contiguous()):
            raise ValueError("the tensors of the map must be contiguous and int32")
        if to_row.numel() < tokens * self.topk or counts.numel() < self.experts or offsets.numel() <= self.experts:
            raise ValueError(f"the map is too small for {tokens} tokens, {self.topk} slots each, and {self.experts} experts")
        rows = to_slot.numel()
        return _lib.RouteMapStruct(to_row.data_ptr(), to_slot.data_ptr(), counts.data_ptr(), offsets.data_ptr(), rows), rows

    def _new(self, stream, shape, dtype):
        """A tensor whose memory belongs to the stream the call writes it on: memory of another stream's may still be
        written there by work of its previous owner."""
        if stream is None:
            return torch.empty(*shape, dtype=dtype, device=self.device)  # 0.3 us sooner than with the tuple itself
        with torch.cuda.stream(stream):
            return torch.empty(*shape, dtype=dtype, device=self.device)

    def _slots_out(self, t, name, tokens, dtype, stream):
        """A caller's output for every slot, checked, or a new one; and its pointer."""
        if t is not None:
            return t, self._per_slot(t, name, tokens, dtype)
        t = self._new(stream, (tokens, self.topk), dtype)
        return t, t.data_ptr()

    def _rows_out(self, t, name, rows, hidden, dtype, stream):
        """A caller's output matrix, checked, or a new one; its pointer and row stride."""
        if t is not None:
            return (t, *self._rows(t, name, rows, hidden, dtype))
        t = self._new(stream, (rows, hidden), dtype)
        return t, t.data_ptr(), hidden

    def _on_stream(self, stream):
        return _raw_stream(self.device.index) if stream is None else stream.cuda_stream

    def _row_type(self, t, name, eight_bits=False):
        if t.dim() != 2:
            raise ValueError(f"{name} must have two dimensions, not {t.dim()}")
        kind = _ROW_TYPES.get(t.dtype)
        if kind is None and eight_bits and t.element_size() == 1:
            kind = _TYPE_8BIT
        if kind is None:
            raise ValueError(f"{name} has the unsupported type {t.dtype}")
        return kind

    def _bias(self, bias):
        if bias is None:
            return None
        self._on_device(bias, "bias")
        if bias.dtype != torch.float32 or bias.numel() != self.experts or not bias.is_contiguous():
            raise ValueError(f"bias must be a contiguous float32 tensor of {self.experts} elements")
        return bias.data_ptr()

    def _scores(self, scores):
        kind = self._row_type(scores, "scores")
        tokens = scores.size(0)
        ptr, ld = self._rows(scores, "scores", tokens, self.experts, scores.dtype)
        return tokens, kind, ptr, ld

    # ---- calls -----------------------------------------------------------------------
    def new_map(self, tokens=None, stream=None):
        """An unwritten RouteMap for `order` calls of up to `tokens` tokens (the plan's, by default)."""
        tokens = self.tokens if tokens is None else tokens
        shapes = ((tokens, self.topk), (self.max_rows,), (self.experts,), (self.experts + 1,))
        return RouteMap(*(self._new(stream, shape, torch.int32) for shape in shapes))

    def select(self, scores, bias=None, ids_out=None, weights_out=None, stream=None):
        """`mrs_route_select`: the topk experts of every token and their weights, (ids int32, weights float32), both
        [tokens, topk], from scores [tokens, experts] (float32, float16 or bfloat16)."""
        tokens, kind, ptr, ld = self._scores(scores)
        ids_out, ids_ptr = self._slots_out(ids_out, "ids_out", tokens, torch.int32, stream)
        weights_out, weights_ptr = self._slots_out(weights_out, "weights_out", tokens, torch.float32, stream)
        _lib.check(
            self.lib.mrs_route_select(self._h, tokens, ptr, ld, kind, self._bias(bias), ids_ptr, weights_ptr,
                                      self._on_stream(stream))
        )
        return ids_out, weights_out

    def select_backward(self, scores, ids, weights_grad, bias=None, scores_grad_out=None, stream=None):
        """`mrs_route_select_backward`: the gradient of `scores`, of their type, from that of the weights."""
        tokens, kind, ptr, ld = self._scores(scores)
        out, grad_ptr, grad_ld = self._rows_out(scores_grad_out, "scores_grad_out", tokens, self.experts, scores.dtype, stream)
        _lib.check(
            self.lib.mrs_route_select_backward(self._h, tokens, ptr, ld, kind, self._bias(bias),
                                               self._per_slot(ids, "ids", tokens, torch.int32),
                                               self._per_slot(weights_grad, "weights_grad", tokens, torch.float32),
                                               grad_ptr, grad_ld, self._on_stream(stream))
        )
        return out

    def order(self, ids, map_out=None, stream=None):
        """`mrs_route_order`: a RouteMap of the slots sorted by ids [tokens, topk] (int32; ids outside [0, experts)
        get no row).  Every tensor of `map_out` is written, row_of_slot as far as the tokens go: what it holds behind them stays
        and means nothing."""
        tokens = self._slots(ids, "ids")
        ids_ptr = self._per_slot(ids, "ids", tokens, torch.int32)
        if map_out is None:
            map_out = self.new_map(tokens, stream)
        raw, _ = self._map(map_out, tokens)
        on = self._on_stream(stream)
        _lib.check(self.lib.mrs_route_order(self._h, tokens, ids_ptr, raw, on))
        # nothing is captured from the null stream; asking about others takes 0.3 us
        capturing = on != 0 and _capturing()
        if capturing or map_out.tokens != tokens:
            map_out._ordered(tokens, capturing)
        return map_out

    def dispatch(self, x, route, rows_out=None, stream=None):
        """`mrs_route_dispatch`: x [tokens, hidden] in expert order, [rows, hidden].  Rows behind the last segment are
        left as they are: in an own `rows_out` that is what was there, in a new tensor anything."""
        kind = self._row_type(x, "x", eight_bits=True)
        tokens, hidden = x.shape
        raw, rows = self._map(route, tokens)
        x_ptr, ld_x = self._rows(x, "x", tokens, hidden, x.dtype)
        rows_out, out_ptr, ld_out = self._rows_out(rows_out, "rows_out", rows, hidden, x.dtype, stream)
        _lib.check(self.lib.mrs_route_dispatch(self._h, tokens, raw, kind, hidden, x_ptr, ld_x, out_ptr, ld_out,
                                               self._on_stream(stream)))
        return rows_out

    def dispatch_backward(self, rows_grad, route, x_grad_out=None, tokens=None, stream=None):
        """`mrs_route_dispatch_backward`: the gradient of x [tokens, hidden].  `tokens` is by default that of the last `order` into
        this map, and has to be given where orderings of different sizes share a map and one of them was captured into a graph."""
        kind = self._row_type(rows_grad, "rows_grad")
        hidden = rows_grad.size(1)
        if tokens is None:
            tokens = route.tokens
            if tokens is None:
                tokens = route.row_of_slot.numel() // self.topk
            elif tokens < 0:
                raise ValueError("orderings of different sizes into this map, some of them in a graph: tokens has to be given")
        raw, rows = self._map(route, tokens)
        in_ptr, ld_in = self._rows(rows_grad, "rows_grad", rows, hidden, rows_grad.dtype)
        x_grad_out, out_ptr, ld_out = self._rows_out(x_grad_out, "x_grad_out", tokens, hidden, rows_grad.dtype, stream)
        _lib.check(
            self.lib.mrs_route_dispatch_backward(self._h, tokens, raw, kind, hidden, in_ptr, ld_in, out_ptr, ld_out,
                                                 self._on_stream(stream))
        )
        return x_grad_out

    def combine(self, rows, route, weights, out=None, stream=None):
        """`mrs_route_combine`: out[t] = sum over j of weights[t, j] * rows[row_of_slot[t, j]], of the rows' type."""
        kind = self._row_type(rows, "rows")
        tokens, hidden = self._slots(weights, "weights"), rows.size(1)
        raw, count = self._map(route, tokens)
        in_ptr, ld_in = self._rows(rows, "rows", count, hidden, rows.dtype)
        out, out_ptr, ld_out = self._rows_out(out, "out", tokens, hidden, rows.dtype, stream)
        _lib.check(
            self.lib.mrs_route_combine(self._h, tokens, raw, kind, hidden, in_ptr, ld_in,
                                       self._per_slot(weights, "weights", tokens, torch.float32), out_ptr, ld_out,
                                       self._on_stream(stream))
        )
        return out

    def combine_backward(self, out_grad, rows, route, weights, drows_out=None, dweights_out=None, stream=None):
        """`mrs_route_combine_backward`: (gradient of rows, gradient of weights float32).  Rows behind the last segment
        are left as they are, as in `dispatch`."""
        kind = self._row_type(rows, "rows")
        tokens, hidden = self._slots(weights, "weights"), rows.size(1)
        raw, count = self._map(route, tokens)
        grad_ptr, ld_grad = self._rows(out_grad, "out_grad", tokens, hidden, rows.dtype)
        in_ptr, ld_in = self._rows(rows, "rows", count, hidden, rows.dtype)
        weights_ptr = self._per_slot(weights, "weights", tokens, torch.float32)
        drows_out, out_ptr, ld_out = self._rows_out(drows_out, "drows_out", count, hidden, rows.dtype, stream)
        dweights_out, sums_ptr = self._slots_out(dweights_out, "dweights_out", tokens, torch.float32, stream)
        _lib.check(
            self.lib.mrs_route_combine_backward(self._h, tokens, raw, kind, hidden, grad_ptr, ld_grad, in_ptr, ld_in,
                                                weights_ptr, out_ptr, ld_out, sums_ptr, self._on_stream(stream))
        )
        return drows_out, dweights_out
