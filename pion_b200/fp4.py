"""Microscaled 4-bit floating-point rows: a store quantised as it is written, read back,
multiplied with query batches and searched (the pion_v_b200_fp4_* entry points).

* ``FP4Rows`` — the store: device buffers of codes, block scales and row scales; ``write``
  quantises rows into slots, ``read`` returns slots as rows;
* ``quantize_rows_fp4`` — a new store holding the given rows;
* ``fp4_scores`` — every query's inner product with every row;
* ``FlatFP4Index.search`` — the k best rows per query, ids exact.

Formats: ``"mx"`` (blocks of 32, power-of-two scales) and ``"nv"`` (blocks of 16, e4m3 scales,
one float32 scale per row).  Rows and queries are numpy arrays (float32 or float16, host
memory) or torch tensors (float32, bfloat16 or float16; CUDA tensors are used in place on
torch's current stream of their device, and calls on them can be captured into CUDA graphs).
"""
from __future__ import annotations

import ctypes
import functools
import operator

import numpy as np

from . import _lib
from ._lib import MEM_DEVICE, MEM_HOST, PionError
from .search import Context, torch

FORMATS = {"mx": _lib.FP4_MX, "nv": _lib.FP4_NV}
TYPES = {} if torch is None else {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16,
                                  torch.float16: _lib.F16}


def _device_of(ctx: Context) -> int:
    """Index of the CUDA device a context runs on."""
    at = getattr(ctx, "_device_index", None)
    if at is None:
        at = ctx._device_index = int(ctx.lib.pion_v_b200_ctx_device(ctx.h))
    return at


# torch's current stream of a device as a handle; without the Stream object around it where torch
# has that (1.2 us less a call).
_raw_stream = getattr(getattr(torch, "_C", None), "_cuda_getCurrentRawStream", None) or \
    (lambda device: torch.cuda.current_stream(device).cuda_stream)


def _stream(ctx: Context) -> int:
    """torch's current stream of the context's device as a cudaStream_t (handle 0, torch's
    legacy default stream, is cudaStreamLegacy to the library)."""
    return _raw_stream(_device_of(ctx)) or 1


def _call(ctx: Context, fn, *args, mem: int = MEM_DEVICE):
    """fn(ctx, *args, mem, stream), leaving torch's current device as it is.  A store is torch's
    memory whatever memory the call's arrays are in, so host-memory calls are ordered with
    torch's current stream too."""
    before = torch.cuda.current_device()
    try:
        if mem == MEM_DEVICE:
            rc = fn(ctx.h, *args, mem, _stream(ctx))
            if rc != 0:
                ctx.check(rc)
        else:
            lib = ctx.lib
            ctx.check(lib.pion_v_b200_set_stream(ctx.h, _stream(ctx)))
            try:
                ctx.check(fn(ctx.h, *args, mem, None))
            finally:
                lib.pion_v_b200_set_stream(ctx.h, ctx._stream)
    finally:
        if before != _device_of(ctx):
            torch.cuda.set_device(before)


def _int64(x, what: str) -> int:
    """x as an int of 64 bits (ctypes would wrap a larger one)."""
    x = operator.index(x)
    if not -2 ** 63 <= x < 2 ** 63:
        raise ValueError(f"{what} {x} is past 64 bits")
    return x


def _matrix(ctx: Context, x, what: str, dim: int):
    """(pointer, type, row stride, rows, mem, the tensor) of a [n, dim] array whose elements are
    contiguous in a row."""
    if not isinstance(x, torch.Tensor):
        x = np.asarray(x)
        if x.dtype not in (np.float32, np.float16):
            x = x.astype(np.float32)
        if any(s < 0 for s in x.strides) or not x.flags.writeable:
            x = x.copy()
        x = torch.from_numpy(x)
    if x.dim() != 2 or x.shape[1] != dim:
        raise ValueError(f"{what} must be [n, {dim}], got {tuple(x.shape)}")
    typ = TYPES.get(x.dtype)
    if typ is None:
        raise TypeError(f"{what} must be float32, bfloat16 or float16, got {x.dtype}")
    n = x.shape[0]
    s0, s1 = x.stride()
    if n > 0 and ((s1 != 1 and dim > 1) or (s0 < dim and n > 1)):
        x = x.contiguous()
        s0 = dim
    mem = MEM_HOST
    if x.is_cuda:
        mem = MEM_DEVICE
        if x.get_device() != _device_of(ctx):
            raise ValueError(f"{what} is on {x.device}, the context on device {_device_of(ctx)}")
    return x.data_ptr(), typ, (s0 if n > 1 else dim), n, mem, x


def _slots(ctx: Context, slots, mem: int):
    """The slots as an int64 tensor in the call's memory."""
    if not isinstance(slots, torch.Tensor):
        slots = np.asarray(slots)
        if slots.size and slots.dtype.kind not in "iu":
            raise TypeError("slots must be a list of integers")
        if slots.dtype.kind == "u" and slots.size and int(slots.max()) > np.iinfo(np.int64).max:
            raise ValueError("a slot is past 64 bits")
        slots = torch.from_numpy(slots.astype(np.int64))
    if slots.dim() != 1 or slots.dtype not in (torch.int64, torch.int32):
        raise TypeError("slots must be a list of integers")
    want = torch.device("cuda", _device_of(ctx)) if mem == MEM_DEVICE else torch.device("cpu")
    if slots.device != want or slots.dtype != torch.int64 or not slots.is_contiguous():
        slots = slots.to(device=want, dtype=torch.int64).contiguous()
    return slots


def _output(out, shape, dtype, device, make=None):
    """(tensor, type, row stride) of an output of rows: `out`, checked, or a new tensor."""
    if out is None:
        out = (make or torch.empty)(shape, dtype=dtype or torch.float32, device=device)
    elif tuple(out.shape) != tuple(shape) or out.device != device or \
            (dtype is not None and dtype != out.dtype) or \
            (out.numel() > 0 and ((shape[1] > 1 and out.stride(1) != 1) or
                                  (shape[0] > 1 and out.stride(0) < shape[1]))):
        raise ValueError(f"out must be {tuple(shape)} {dtype or ''} rows on {device}")
    typ = TYPES.get(out.dtype)
    if typ is None:
        raise TypeError(f"dtype must be float32, bfloat16 or float16, got {out.dtype}")
    return out, typ, (out.stride(0) if shape[0] > 1 else shape[1])


@functools.lru_cache(maxsize=256)
def _sizes(format: str, n_rows: int, dim: int):
    """Bytes of a store's codes and scales."""
    if format not in FORMATS:
        raise ValueError(f"format must be one of {sorted(FORMATS)}, got {format!r}")
    n_rows, dim = _int64(n_rows, "n_rows"), _int64(dim, "dim")
    cb, sb = ctypes.c_int64(), ctypes.c_int64()
    rc = _lib.load().pion_v_b200_fp4_sizes(FORMATS[format], n_rows, dim, ctypes.byref(cb),
                                           ctypes.byref(sb))
    if rc != 0:
        raise PionError(rc, f"unsupported store: {n_rows} rows of {dim} elements")
    return cb.value, sb.value


class FP4Rows:
    """A store of ``n_rows`` slots of ``dim`` elements in 4 bits (every slot empty at first).

    ``codes`` uint8 [n_rows, dp / 2], ``scales`` uint8, ``row_scale`` float32 [n_rows],
    ``norm_max`` float32 [1] and ``claim`` int32 [n_rows] (zeros) may be given: the store then
    is those tensors, as the C struct ``pion_b200_fp4_rows`` lays them out.
    """

    def __init__(self, n_rows: int, dim: int, format: str = "nv", device=None, *, codes=None,
                 scales=None, row_scale=None, norm_max=None, claim=None):
        cb, sb = _sizes(format, n_rows, dim)
        if codes is None and scales is None and row_scale is None and norm_max is None:
            if claim is not None:
                raise ValueError("claim is given with codes, scales, row_scale and norm_max only")
            device = torch.device("cuda" if device is None else device)
            codes = torch.zeros((n_rows, cb // max(n_rows, 1)), dtype=torch.uint8, device=device)
            scales = torch.zeros(sb, dtype=torch.uint8, device=device)
            row_scale = torch.full((n_rows,), float("nan"), dtype=torch.float32, device=device)
            norm_max = torch.zeros(1, dtype=torch.float32, device=device)
            claim = torch.zeros(n_rows, dtype=torch.int32, device=device)
        elif codes is None or scales is None or row_scale is None or norm_max is None:
            raise ValueError("a store of given tensors needs codes, scales, row_scale and norm_max")
        else:
            at = codes.get_device()
            for name, t, dtype, size in (("codes", codes, torch.uint8, cb),
                                         ("scales", scales, torch.uint8, sb),
                                         ("row_scale", row_scale, torch.float32, n_rows),
                                         ("norm_max", norm_max, torch.float32, 1),
                                         ("claim", claim, torch.int32, n_rows)):
                if t is None and name == "claim":
                    continue
                if t.dtype is not dtype or t.numel() != size or not t.is_contiguous():
                    raise ValueError(f"{name} must be {size} contiguous {dtype} values")
                if at < 0 or t.get_device() != at:
                    raise ValueError(f"{name} must be on the store's CUDA device")
        self._n_rows, self._dim, self._format = n_rows, dim, format
        self._codes, self._scales, self._row_scale = codes, scales, row_scale
        self._norm_max, self._claim = norm_max, claim
        self._c = _lib.FP4RowsDesc(
            FORMATS[format], 0, n_rows, dim, codes.data_ptr(), scales.data_ptr(),
            row_scale.data_ptr(), norm_max.data_ptr(),
            claim.data_ptr() if claim is not None else None)

    # What _c holds the addresses and sizes of stays as it is.
    n_rows = property(operator.attrgetter("_n_rows"))
    dim = property(operator.attrgetter("_dim"))
    format = property(operator.attrgetter("_format"))
    codes = property(operator.attrgetter("_codes"))
    scales = property(operator.attrgetter("_scales"))
    row_scale = property(operator.attrgetter("_row_scale"))
    norm_max = property(operator.attrgetter("_norm_max"))
    claim = property(operator.attrgetter("_claim"))

    @property
    def device(self):
        return self._codes.device

    def _ref(self, ctx: Context):
        if self._codes.get_device() != _device_of(ctx):
            raise ValueError(f"the store is on {self.device}, the context on device "
                             f"{_device_of(ctx)}")
        return ctypes.byref(self._c)

    def clear(self, ctx: Context):
        """Empties every slot."""
        _call(ctx, lambda h, ref, mem, st: ctx.lib.pion_v_b200_fp4_clear(h, ref, st),
              self._ref(ctx))

    def write(self, ctx: Context, src, slots=None, start: int = 0):
        """Quantises the rows of ``src`` [n, dim] into slots ``slots[i]``, or ``start + i``.
        A negative slot skips its row; of several rows for one slot the last is kept."""
        p, typ, stride, n, mem, keep = _matrix(ctx, src, "src", self._dim)
        ps = None
        if slots is not None:
            slots = _slots(ctx, slots, mem)
            if len(slots) != n:
                raise ValueError(f"{len(slots)} slots for {n} rows")
            ps = slots.data_ptr()
        _call(ctx, ctx.lib.pion_v_b200_fp4_write, self._ref(ctx), p, typ, stride, n, ps,
              start and _int64(start, "start"), mem=mem)

    def read(self, ctx: Context, slots=None, start: int = 0, count: int | None = None,
             dtype=None, out=None):
        """Slots ``slots``, or ``count`` slots from ``start`` (default: all), as rows [n, dim] of
        ``dtype`` (default float32) on the store's device, or into ``out``.  An empty slot
        reads as NaN; a negative one leaves its row of ``out`` as it was (undefined without)."""
        ps, start = None, start and _int64(start, "start")
        if slots is not None:
            slots = _slots(ctx, slots, MEM_DEVICE)
            n, ps = len(slots), slots.data_ptr()
        else:
            n = self.n_rows - start if count is None else _int64(count, "count")
        out, typ, stride = _output(out, (max(n, 0), self._dim), dtype, self.device)
        _call(ctx, ctx.lib.pion_v_b200_fp4_read, self._ref(ctx), ps, start, n, out.data_ptr(), typ,
              stride)
        return out


def quantize_rows_fp4(ctx: Context, src, format: str = "nv") -> FP4Rows:
    """A new store holding the rows of ``src`` [n, dim], row i in slot i."""
    src = src if isinstance(src, torch.Tensor) else np.asarray(src)
    if src.ndim != 2:
        raise ValueError(f"src must be [n, dim], got {tuple(src.shape)}")
    rows = FP4Rows(src.shape[0], src.shape[1], format, torch.device("cuda", _device_of(ctx)))
    rows.write(ctx, src)
    return rows


def _workspace(ctx: Context, rows: FP4Rows, n_rows: int, nq: int, k: int, mem: int):
    """(tensor, pointer, bytes) of a device-memory call's scratch."""
    need = ctx.lib.pion_v_b200_fp4_workspace(rows._ref(ctx), n_rows, nq, k) \
        if mem == MEM_DEVICE else 0
    if need <= 0:
        return None, None, 0  # host memory, nothing to hold, or sizes that the call refuses
    ws = rows._codes.new_empty(need)
    return ws, ws.data_ptr(), need


def fp4_scores(ctx: Context, rows: FP4Rows, q, n_rows: int | None = None, dtype=None, out=None):
    """Scores [nq, n_rows] of the queries ``q`` [nq, dim] (quantised in the store's format) with
    the rows of slots [0, n_rows), accumulated in float32; -inf for an empty slot.  Into ``out``
    (rows may be strided) or a new tensor of ``dtype`` (default float32), in q's memory."""
    n = rows.n_rows if n_rows is None else _int64(n_rows, "n_rows")
    p, typ, stride, nq, mem, keep = _matrix(ctx, q, "q", rows.dim)
    out, otyp, ostride = _output(out, (nq, max(n, 0)), dtype,
                                 rows.device if mem == MEM_DEVICE else torch.device("cpu"))
    ws, pws, nws = _workspace(ctx, rows, n, nq, 0, mem)
    _call(ctx, ctx.lib.pion_v_b200_fp4_scores, rows._ref(ctx), n, p, typ, stride, nq,
          out.data_ptr(), otyp, ostride, pws, nws, mem=mem)
    return out if isinstance(q, torch.Tensor) else out.numpy()


class FlatFP4Index:
    """Exact search of a store's rows by their 4-bit inner products.

    ``rows``: an ``FP4Rows`` (searched as it is at the time of each call), or an array of rows to
    quantise.  Result ids are ``id_base + slot``."""

    def __init__(self, ctx: Context, rows, id_base: int = 0, format: str = "nv"):
        self.ctx = ctx
        self.rows = rows if isinstance(rows, FP4Rows) else quantize_rows_fp4(ctx, rows, format)
        self.id_base = id_base and _int64(id_base, "id_base")
        self.dim = self.rows.dim

    @property
    def n_rows(self) -> int:
        return self.rows.n_rows

    def search(self, q, k: int, n_rows: int | None = None):
        """Top-k of slots [0, n_rows) by (score desc, id asc) per query -> (ids int32 [nq, k],
        scores float32 [nq, k]), in q's memory; -1 / -inf past the rows that are not empty."""
        ctx, rows = self.ctx, self.rows
        n, k = rows.n_rows if n_rows is None else _int64(n_rows, "n_rows"), operator.index(k)
        p, typ, stride, nq, mem, keep = _matrix(ctx, q, "q", rows.dim)
        device = rows.device if mem == MEM_DEVICE else torch.device("cpu")
        ids = torch.empty((nq, max(k, 0)), dtype=torch.int32, device=device)
        scores = torch.empty((nq, max(k, 0)), dtype=torch.float32, device=device)
        ws, pws, nws = _workspace(ctx, rows, n, nq, k, mem)
        _call(ctx, ctx.lib.pion_v_b200_flat_fp4_knn, rows._ref(ctx), n, self.id_base, p, typ,
              stride, nq, k, ids.data_ptr(), scores.data_ptr(), pws, nws, mem=mem)
        return (ids, scores) if isinstance(q, torch.Tensor) else (ids.numpy(), scores.numpy())
