"""KV cache in pages: ctypes binding of include/jfb/jfb_paged.h.

The calls of one layer's step, in order:

    rope_append(q, k, v, pos, rope, cache, batch, q_out)   rotate, append to the pages
    attention(q_out, cache, batch, out, workspace, lse=lse)  new tokens over their pages
    attention_mass(q_out, lse, cache, batch, mass)           weight each key received (optional)
    evict(mass, cache, batch, keep, kv_len, recent=...)      cut long sequences (now and then)

Arguments are torch CUDA tensors; PyTorch only provides device memory and
streams. A call runs on `stream` or the current stream of the tensors' device
(which need not be the current device). Nothing is synchronised: what only the
device knows (page ids, lengths) is reported through `error_flag`, an int32
tensor of one element that the caller clears and reads. Wrong arguments raise
InvalidArgument.
"""
from __future__ import annotations

import ctypes as C

from .engine import InvalidArgument, Status, check, lib

_VP, _U32, _U64 = C.c_void_p, C.c_uint32, C.c_uint64

ERROR_RANGE, ERROR_TIMEOUT = 1, 2
MAX_SEQUENCES = 4096
SCALINGS = {"none": 0, "linear": 1, "ntk": 2, "yarn": 3, "bands": 4}


class CacheC(C.Structure):
    _fields_ = [("k", _VP), ("v", _VP), ("page_stride", _U64), ("token_stride", _U64), ("head_stride", _U64),
                ("dtype", _U32), ("pages", _U32), ("page_size", _U32), ("kv_heads", _U32), ("head_dim", _U32),
                ("reserved", _U32)]


class BatchC(C.Structure):
    _fields_ = [("q_start", _VP), ("kv_len", _VP), ("page_table", _VP), ("table_stride", _U64), ("sequences", _U32),
                ("table_width", _U32)]


class RopeC(C.Structure):
    _fields_ = [("freq", _VP), ("rope_dims", _U32), ("interleaved", _U32), ("factor", C.c_float), ("reserved", _U32)]


_bound = None
torch = None
_DTYPES: dict = {}  # torch dtype -> jfb_dtype
_raw_stream = None


def _bind():
    """The library with its signatures; binds torch on first use like the other modules."""
    global _bound, torch, _raw_stream
    if _bound is None:
        import torch as t
        L = lib()
        cache, batch = C.POINTER(CacheC), C.POINTER(BatchC)
        sig = {
            "jfb_rope_frequencies_host": ([_VP, _VP, _U32, C.c_double, _U32, C.c_double, C.c_double, C.c_double,
                                           C.c_double], Status),
            "jfb_rope_paged_append": ([_VP, _VP, _VP, _U32, _U64, _U64, _U64, _U32, _U32, _VP, C.POINTER(RopeC), cache,
                                       batch, _VP, _U64, _VP, _VP], Status),
            "jfb_paged_attention_workspace_bytes": ([], _U64),
            "jfb_paged_attention": ([_VP, _U64, _U32, _U32, C.c_float, _U32, cache, batch, _VP, _U64, _VP, _VP, _U64,
                                     _VP, _VP], Status),
            "jfb_paged_attention_mass": ([_VP, _U64, _U32, _U32, C.c_float, _U32, _VP, cache, batch, _VP, _VP, _U64,
                                          _VP, _VP], Status),
            "jfb_paged_evict": ([_VP, _U64, cache, batch, _U32, _U32, _VP, _VP, _VP, _U64, _VP, _U64, _U32, _VP, _VP],
                                Status),
        }
        for name, (args, res) in sig.items():
            fn = getattr(L, name)
            fn.argtypes = args
            fn.restype = res
        torch = t
        _DTYPES.update({t.float32: 0, t.float16: 1, t.bfloat16: 2})
        # the current stream's address without building a Stream object, where torch offers it
        _raw_stream = getattr(t._C, "_cuda_getCurrentRawStream", None) or (lambda i: t.cuda.current_stream(i).cuda_stream)
        _bound = L
    return _bound


def _require(ok: bool, message: str) -> None:
    if not ok:
        raise InvalidArgument(message)


class PagedCache:
    """One layer's K and V pools, [pages, page_size, kv_heads, head_dim] of
    float16 or bfloat16. Any strides that are multiples of 8 elements with
    contiguous heads will do: a pool stored [pages, kv_heads, page_size,
    head_dim] is passed as pool.transpose(1, 2)."""

    def __init__(self, k, v):
        _bind()
        _require(k.dim() == 4 and k.shape == v.shape, "paged pools are [pages, page_size, kv_heads, head_dim]")
        _require(k.is_cuda and v.device == k.device, "paged pools must be on one CUDA device")
        _require(k.dtype in (torch.float16, torch.bfloat16) and v.dtype == k.dtype, "paged pools are float16 or bfloat16")
        _require(all(n > 0 for n in k.shape), "paged pools must not be empty")
        _require(k.shape[3] == 1 or (k.stride(3) == 1 and v.stride(3) == 1), "paged heads must be contiguous")
        strides = []
        for dim in range(3):
            if k.shape[dim] == 1:
                strides.append((k.shape[3] + 7) // 8 * 8)  # never stepped over
            else:
                _require(k.stride(dim) == v.stride(dim), "paged pools must share their strides")
                strides.append(k.stride(dim))
        self.k, self.v, self.device = k, v, k.device
        self.dtype = k.dtype
        self.scale = k.shape[3] ** -0.5
        self.pages, self.page_size, self.kv_heads, self.head_dim = k.shape
        self.desc = CacheC(k.data_ptr(), v.data_ptr(), *strides, _DTYPES[k.dtype], *k.shape, 0)
        self.ref = C.byref(self.desc)


def _int32(t, dim: int, device, what: str) -> None:
    if t.dtype != torch.int32 or t.dim() != dim or t.device != device:
        raise InvalidArgument(f"{what} must be int32 with {dim} dimensions on the cache's device")


class PagedBatch:
    """The sequences of a step: q_start [sequences + 1] first new row of each,
    kv_len [sequences] keys with the new ones, page_table [sequences, width];
    int32 CUDA tensors that the calls read on the device, so their contents may
    change between calls."""

    def __init__(self, q_start, kv_len, page_table):
        _bind()
        dev = q_start.device
        _require(q_start.is_cuda, "paged batch arrays must be on a CUDA device")
        _int32(q_start, 1, dev, "q_start")
        _int32(kv_len, 1, dev, "kv_len")
        _int32(page_table, 2, dev, "page_table")
        n = kv_len.shape[0]
        _require(q_start.shape[0] == n + 1 and page_table.shape[0] == n, "paged batch arrays disagree about the sequences")
        _require(q_start.is_contiguous() and kv_len.is_contiguous(), "q_start and kv_len must be contiguous")
        _require(page_table.shape[1] > 0 and (page_table.shape[1] == 1 or page_table.stride(1) == 1),
                 "page_table rows must be contiguous")
        self.q_start, self.kv_len, self.page_table, self.device, self.sequences = q_start, kv_len, page_table, dev, n
        self.desc = BatchC(q_start.data_ptr(), kv_len.data_ptr(), page_table.data_ptr(), _row_stride(page_table), n,
                           page_table.shape[1])
        self.ref = C.byref(self.desc)


def _row_stride(table) -> int:
    # a single row is never stepped over
    return table.stride(0) if table.shape[0] > 1 else max(table.stride(0), table.shape[1])


def rope_frequencies(rope_dims: int, base: float, scaling: str = "none", factor: float = 1.0, trained: float = 0.0,
                     low: float | None = None, high: float | None = None):
    """(numpy float64 [rope_dims / 2] radians per position, factor on cos and sin)
    under `scaling`: none, linear, ntk, yarn or bands (jfb_rope_frequencies_host)."""
    import numpy as np
    _require(scaling in SCALINGS, f"unknown rope scaling {scaling!r}")
    _require(0 < rope_dims < 1 << 20, "rope frequencies need an even rope_dims and a positive base")
    low = 1.0 if low is None else low
    high = (32.0 if scaling == "yarn" else 4.0) if high is None else high
    freq = np.empty((rope_dims + 1) // 2, dtype=np.float64)
    out = C.c_double()
    check(_bind().jfb_rope_frequencies_host(freq.ctypes.data, C.addressof(out), rope_dims, base, SCALINGS[scaling], factor,
                                            trained, low, high))
    return freq, out.value


class Rope:
    """Rotation of the first 2 * len(freq) elements of each head; freq is a
    float64 CUDA tensor of radians per position, `factor` multiplies cos and sin."""

    def __init__(self, freq, interleaved: bool = False, factor: float = 1.0):
        _bind()
        _require(freq.is_cuda and freq.dtype == torch.float64 and freq.dim() == 1 and freq.is_contiguous() and freq.numel() > 0,
                 "rope frequencies are a contiguous float64 CUDA vector")
        self.freq, self.device = freq, freq.device
        self.desc = RopeC(freq.data_ptr(), 2 * freq.numel(), int(interleaved), factor, 0)
        self.ref = C.byref(self.desc)

    @classmethod
    def scaled(cls, rope_dims: int, base: float, scaling: str = "none", interleaved: bool = False, device="cuda", **kw):
        freq, factor = rope_frequencies(rope_dims, base, scaling, **kw)
        return cls(torch.from_numpy(freq).to(device), interleaved, factor)


def _rows(x, cache: PagedCache, what: str):
    """(address, row stride, rows, heads) of [rows, heads, head_dim] or [rows, heads * head_dim]."""
    if x.device != cache.device:
        raise InvalidArgument(f"{what} must be on the cache's device")
    hd = cache.head_dim
    shape, strides = x.shape, x.stride()
    rows = shape[0] if shape else 0
    if len(shape) == 3:
        heads = shape[1]
        ok = shape[2] == hd and strides[2] == 1 and (strides[1] == hd or heads == 1)
    else:
        ok = len(shape) == 2 and shape[1] % hd == 0 and strides[1] == 1
        heads = shape[1] // hd if ok else 0
    if not ok or heads == 0:
        raise InvalidArgument(f"{what} must be rows of contiguous heads of {hd}")
    stride = strides[0] if rows > 1 else heads * hd  # a single row is never stepped over
    if stride < heads * hd:
        raise InvalidArgument(f"{what} rows overlap")
    return x.data_ptr(), stride, rows, heads


def _cache_rows(x, cache: PagedCache, what: str):
    if x.dtype != cache.dtype:
        raise InvalidArgument(f"{what} must have the cache's dtype, {cache.dtype}")
    return _rows(x, cache, what)


def _flag(error_flag, device):
    if error_flag is None:
        return None
    _require(error_flag.dtype == torch.int32 and error_flag.device == device and error_flag.numel() == 1,
             "error_flag must be one int32 on the cache's device")
    return error_flag.data_ptr()


def _call(fn, device, stream, *args) -> None:
    """The C call on the device of its tensors, on `stream` or that device's current one."""
    index = device.index
    if stream is None:
        address = _raw_stream(index)
    else:
        _require(stream.device == device, "the stream must be on the cache's device")
        address = stream.cuda_stream
    if index == torch.cuda.current_device():
        status = fn(*args, address)
    else:
        with torch.cuda.device(device):
            status = fn(*args, address)
    if status.code:
        check(status)


def _on(batch: PagedBatch, cache: PagedCache) -> None:
    if batch.device != cache.device:
        raise InvalidArgument("cache and batch must be on one device")


def rope_append(q, k, v, pos, rope: Rope, cache: PagedCache, batch: PagedBatch, q_out, error_flag=None, stream=None) -> None:
    """q_out = rotated q; the rotated k and the v of the new tokens go to their
    slots in the pages (jfb_rope_paged_append). q, k and v share one dtype
    (float32, float16 or bfloat16), q_out has the cache's; pos int32 [rows]."""
    _on(batch, cache)
    _require(rope.device == cache.device, "rope and cache must be on one device")
    dtype = _DTYPES.get(q.dtype)
    _require(dtype is not None and k.dtype == q.dtype and v.dtype == q.dtype, "q, k and v must share a float dtype")
    qp, qs, rows, heads = _rows(q, cache, "q")
    kp, ks, k_rows, k_heads = _rows(k, cache, "k")
    vp, vs, v_rows, v_heads = _rows(v, cache, "v")
    op, os, o_rows, o_heads = _cache_rows(q_out, cache, "q_out")
    _require(k_rows == v_rows == o_rows == rows, "q, k, v and q_out must have the same rows")
    _require(k_heads == v_heads == cache.kv_heads and o_heads == heads, "the heads of q, k, v and q_out do not fit the cache")
    _int32(pos, 1, cache.device, "pos")
    _require(pos.shape[0] == rows and pos.is_contiguous(), "pos must hold one position per row")
    _call(_bound.jfb_rope_paged_append, cache.device, stream, qp, kp, vp, dtype, qs, ks, vs, rows, heads, pos.data_ptr(), rope.ref,
          cache.ref, batch.ref, op, os, _flag(error_flag, cache.device))


def attention_workspace(device=None):
    """A zero-filled workspace for attention() on `device`: one per stream that
    runs attention calls, or captured graph that may overlap others."""
    L = _bind()
    dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    with torch.cuda.device(dev):
        return torch.zeros(int(L.jfb_paged_attention_workspace_bytes()), dtype=torch.uint8, device=dev)


def attention(q, cache: PagedCache, batch: PagedBatch, out, workspace, scale: float | None = None, window: int = 0, lse=None,
              error_flag=None, stream=None) -> None:
    """out = attention of the new tokens' q over their sequences' pages, causal,
    with `window` > 0 only over the last `window` slots (jfb_paged_attention);
    lse, if given, float32 [rows, heads]. scale defaults to head_dim ** -0.5."""
    _on(batch, cache)
    qp, qs, rows, heads = _cache_rows(q, cache, "q")
    op, os, o_rows, o_heads = _cache_rows(out, cache, "out")
    _require(o_rows == rows and o_heads == heads, "q and out must have the same rows and heads")
    _lse(lse, rows, heads, cache, optional=True)
    _require(workspace.device == cache.device and workspace.is_contiguous(), "workspace must be on the cache's device")
    _window(window)
    _call(_bound.jfb_paged_attention, cache.device, stream, qp, qs, rows, heads, cache.scale if scale is None else scale,
          window, cache.ref, batch.ref, op, os, None if lse is None else lse.data_ptr(), workspace.data_ptr(),
          workspace.numel() * workspace.element_size(), _flag(error_flag, cache.device))


def _window(window: int) -> None:
    _require(0 <= window < 1 << 31, "window must be from 0 (none) to 2^31 - 1")


def _lse(lse, rows, heads, cache, optional=False) -> None:
    if lse is None and optional:
        return
    _require(lse.dtype == torch.float32 and lse.device == cache.device and lse.shape == (rows, heads) and lse.is_contiguous(),
             "lse must be contiguous float32 [rows, heads]")


def _masses(x, batch: PagedBatch, cache: PagedCache, what: str) -> int:
    _require(x.dtype == torch.float32 and x.device == cache.device and x.dim() == 3 and x.is_contiguous() and
             x.shape[0] == batch.sequences and x.shape[1] == cache.kv_heads and x.shape[2] > 0,
             f"{what} must be contiguous float32 [sequences, kv_heads, slots]")
    return x.shape[2]


def attention_mass(q, lse, cache: PagedCache, batch: PagedBatch, mass_out, mass_in=None, scale: float | None = None,
                   window: int = 0, error_flag=None, stream=None) -> None:
    """mass_out [sequences, kv_heads, slots] = mass_in (0 for new tokens' slots,
    and everywhere without mass_in) plus the attention weight every key received
    from the rows of q (jfb_paged_attention_mass); mass_in may be mass_out."""
    _on(batch, cache)
    qp, qs, rows, heads = _cache_rows(q, cache, "q")
    _lse(lse, rows, heads, cache)
    slots = _masses(mass_out, batch, cache, "mass_out")
    if mass_in is not None:
        _require(_masses(mass_in, batch, cache, "mass_in") == slots, "mass_in and mass_out must hold the same slots")
    _window(window)
    _call(_bound.jfb_paged_attention_mass, cache.device, stream, qp, qs, rows, heads,
          cache.scale if scale is None else scale, window, lse.data_ptr(), cache.ref, batch.ref,
          None if mass_in is None else mass_in.data_ptr(), mass_out.data_ptr(), slots, _flag(error_flag, cache.device))


def evict(mass, cache: PagedCache, batch: PagedBatch, keep, kv_len_out, recent: int, mass_out=None, page_table_out=None,
          error_flag=None, stream=None) -> None:
    """Cuts every sequence to keep.shape[2] keys per kv head: the last `recent`
    and the heaviest others, ties to the lowest slot (jfb_paged_evict). keep int32
    [sequences, kv_heads, budget] receives the kept slots, kv_len_out [sequences]
    the new lengths. Without mass_out the masses move in place, without
    page_table_out the cache does; no page may then belong to two sequences.
    page_table_out is the batch's own tensor (in place) or shares no page with
    it: a copy of the batch's table would have rows overwrite others that are
    still to be moved, so nothing is moved then and the error flag is set."""
    _on(batch, cache)
    slots = _masses(mass, batch, cache, "mass")
    mass_out = mass if mass_out is None else mass_out
    out_slots = _masses(mass_out, batch, cache, "mass_out")
    table = batch.page_table if page_table_out is None else page_table_out
    _int32(table, 2, cache.device, "page_table_out")
    _int32(keep, 3, cache.device, "keep")
    _int32(kv_len_out, 1, cache.device, "kv_len_out")
    _require(table.shape[0] == batch.sequences and table.shape[1] > 0 and (table.shape[1] == 1 or table.stride(1) == 1),
             "page_table_out must be [sequences, pages] with contiguous rows")
    _require(keep.is_contiguous() and keep.shape[0] == batch.sequences and keep.shape[1] == cache.kv_heads and keep.shape[2] > 0,
             "keep must be contiguous [sequences, kv_heads, budget]")
    _require(kv_len_out.is_contiguous() and kv_len_out.shape[0] == batch.sequences, "kv_len_out must be [sequences]")
    _require(0 <= recent <= keep.shape[2], "recent must be from 0 to the budget")
    _call(_bound.jfb_paged_evict, cache.device, stream, mass.data_ptr(), slots, cache.ref, batch.ref, keep.shape[2], recent,
          keep.data_ptr(), kv_len_out.data_ptr(), mass_out.data_ptr(), out_slots, table.data_ptr(), _row_stride(table),
          table.shape[1], _flag(error_flag, cache.device))
