"""pygpann.blocks — ctypes binding of the block operators of libgpann_hip.so (include/gpann_blocks.h): routing of query rows to the blocks of a
key/value cache, attention over the probed blocks and its gradients, attention weights of the cache rows, and eviction.

Tensors are raw device pointers (ints, e.g. `tensor.data_ptr()`), streams are raw hipStream_t handles.  Calls only enqueue work."""
import ctypes as C
import operator

from . import GpannError, _check, lib as _base_lib   # noqa: F401  (GpannError: what the calls raise)

BF16, FP16 = 0, 1
CAUSAL = 1
CALLS = {"route": 1, "attend": 2, "backward": 4, "weigh": 8, "evict": 16}
MAX_PROBE, MAX_BLOCKS = 64, 16384
_DTYPES = {"bf16": BF16, "fp16": FP16, BF16: BF16, FP16: FP16}

EXPORTS = ["gpann_blocks_workspace_bytes", "gpann_blocks_summarize", "gpann_blocks_route", "gpann_blocks_attend", "gpann_blocks_attend_backward",
           "gpann_blocks_weigh", "gpann_blocks_evict"]


class _Layout(C.Structure):
    _fields_ = [("struct_bytes", C.c_uint32), ("device", C.c_int32), ("dtype", C.c_int32), ("flags", C.c_uint32), ("batch", C.c_uint32), ("q_rows", C.c_uint32),
                ("kv_rows", C.c_uint32), ("q_heads", C.c_uint32), ("kv_heads", C.c_uint32), ("head_dim", C.c_uint32), ("block_rows", C.c_uint32),
                ("scale", C.c_float), ("q_len", C.c_void_p), ("kv_len", C.c_void_p), ("page_table", C.c_void_p), ("page_stride", C.c_uint32),
                ("n_pages", C.c_uint32), ("q_stride", C.c_int64 * 3), ("k_stride", C.c_int64 * 3), ("v_stride", C.c_int64 * 3), ("out_stride", C.c_int64 * 3)]


_lib = None


def lib():
    """the library with the argument types of the block operators"""
    global _lib
    if _lib is None:
        L = _base_lib()
        p, u, z, lay = C.c_void_p, C.c_uint32, C.c_size_t, C.POINTER(_Layout)
        L.gpann_blocks_workspace_bytes.argtypes = [lay, u, u, C.POINTER(C.c_size_t)]
        L.gpann_blocks_summarize.argtypes = [lay, p, u, p, p]
        L.gpann_blocks_route.argtypes = [lay, p, p, u, u, u, p, p, z, p]
        L.gpann_blocks_attend.argtypes = [lay, p, p, p, p, u, p, p, p, z, p]
        L.gpann_blocks_attend_backward.argtypes = [lay, p, p, p, p, u, p, p, p, p, p, p, p, z, p]
        L.gpann_blocks_weigh.argtypes = [lay, p, p, p, u, p, p, p, p, z, p]
        L.gpann_blocks_evict.argtypes = [lay, p, p, p, u, u, u, p, p, p, p, C.POINTER(C.c_int64 * 3), p, p, z, p]
        _lib = L
    return _lib


def _whole(name, x, least, most, what):
    x = operator.index(x)
    if not least <= x <= most:
        raise GpannError(1, f"invalid argument: {name} = {x} is not {what}")
    return x


# A C integer takes any Python int modulo its size: what would wrap is refused.  (A call has a dozen of them, so a plain int in range goes no further.)
def _u32(name, x):
    return x if x.__class__ is int and 0 <= x <= 0xFFFFFFFF else _whole(name, x, 0, 0xFFFFFFFF, "an unsigned 32-bit number")


def _i32(name, x):
    return _whole(name, x, -0x80000000, 0x7FFFFFFF, "a signed 32-bit number")


def _size(name, x):
    return x if x.__class__ is int and 0 <= x <= 0xFFFFFFFFFFFFFFFF else _whole(name, x, 0, 0xFFFFFFFFFFFFFFFF, "an unsigned 64-bit number")


def _p(x):
    """a device pointer or None, which 0 counts as"""
    if x.__class__ is int and 0 < x <= 0xFFFFFFFFFFFFFFFF:
        return x
    return (_whole("a tensor's or stream's address", x, 1, 0xFFFFFFFFFFFFFFFF, "a pointer")) if x else None


def _strides(name, s):
    s = tuple(operator.index(x) for x in s)
    if len(s) != 3 or not all(-1 << 63 <= x < 1 << 63 for x in s):
        raise GpannError(1, f"invalid argument: {name} = {s} is not three signed 64-bit numbers")
    return (C.c_int64 * 3)(*s)


class Layout:
    """The shapes of a call's tensors (gpann_blocks_layout).  Strides {batch or page, row, head} default to those of contiguous tensors; a page table's
    rows default to the blocks of a sequence."""

    def __init__(self, batch, q_rows, kv_rows, q_heads, kv_heads, head_dim, block_rows, dtype="bf16", causal=True, scale=None, device=0, q_len=None, kv_len=None,
                 page_table=None, page_stride=None, n_pages=0, q_stride=None, k_stride=None, v_stride=None, out_stride=None):
        if dtype not in _DTYPES:
            raise GpannError(1, f"invalid argument: dtype {dtype!r} is not one of {sorted(map(str, _DTYPES))}")
        blocks = -(-kv_rows // block_rows) if block_rows else 0
        q = (q_rows * q_heads * head_dim, q_heads * head_dim, head_dim)
        kv = ((block_rows if page_table else kv_rows) * kv_heads * head_dim, kv_heads * head_dim, head_dim)
        c = self.c = _Layout()
        c.struct_bytes, c.device, c.dtype, c.flags = C.sizeof(_Layout), _i32("device", device), _DTYPES[dtype], CAUSAL if causal else 0
        for name, x in (("batch", batch), ("q_rows", q_rows), ("kv_rows", kv_rows), ("q_heads", q_heads), ("kv_heads", kv_heads), ("head_dim", head_dim),
                        ("block_rows", block_rows), ("page_stride", blocks if page_stride is None else page_stride), ("n_pages", n_pages)):
            setattr(c, name, _u32(name, x))
        c.scale = scale if scale is not None else head_dim ** -0.5 if head_dim > 0 else 1.0
        c.q_len, c.kv_len, c.page_table = _p(q_len), _p(kv_len), _p(page_table)
        for name, s in (("q_stride", q_stride or q), ("k_stride", k_stride or kv), ("v_stride", v_stride or kv), ("out_stride", out_stride or q)):
            setattr(c, name, _strides(name, s))
        self.blocks = blocks


def workspace_bytes(layout, nprobe, calls):
    """bytes that any of the named calls ("route", "attend", "backward", "weigh", "evict") needs (gpann_blocks_workspace_bytes)"""
    mask = 0
    for c in calls:
        if c not in CALLS:
            raise GpannError(1, f"invalid argument: {c!r} is none of {sorted(CALLS)}")
        mask |= CALLS[c]
    need = C.c_size_t(0)
    _check(lib().gpann_blocks_workspace_bytes(C.byref(layout.c), _u32("nprobe", nprobe), mask, C.byref(need)))
    return need.value


def summarize(layout, k, summary, new_rows=0, stream=None):
    """centroids of the blocks that hold one of the last new_rows rows of a sequence (0: of all blocks)"""
    _check(lib().gpann_blocks_summarize(C.byref(layout.c), _p(k), _u32("new_rows", new_rows), _p(summary), _p(stream)))


def route(layout, q, summary, nprobe, probes, first=1, last=2, workspace=None, workspace_bytes=0, stream=None):
    """probes of every query row: the first and last visible blocks and the best-scored others, in block order, -1 behind them"""
    _check(lib().gpann_blocks_route(C.byref(layout.c), _p(q), _p(summary), _u32("nprobe", nprobe), _u32("first", first), _u32("last", last), _p(probes),
                                    _p(workspace), _size("workspace_bytes", workspace_bytes), _p(stream)))


def attend(layout, q, k, v, probes, nprobe, out, lse=None, workspace=None, workspace_bytes=0, stream=None):
    """attention over the probed blocks"""
    _check(lib().gpann_blocks_attend(C.byref(layout.c), _p(q), _p(k), _p(v), _p(probes), _u32("nprobe", nprobe), _p(out), _p(lse), _p(workspace),
                                     _size("workspace_bytes", workspace_bytes), _p(stream)))


def attend_backward(layout, q, k, v, probes, nprobe, out, lse, dout, dq, dk, dv, workspace=None, workspace_bytes=0, stream=None):
    """gradients of attend"""
    _check(lib().gpann_blocks_attend_backward(C.byref(layout.c), _p(q), _p(k), _p(v), _p(probes), _u32("nprobe", nprobe), _p(out), _p(lse), _p(dout), _p(dq),
                                              _p(dk), _p(dv), _p(workspace), _size("workspace_bytes", workspace_bytes), _p(stream)))


def weigh(layout, q, k, probes, nprobe, lse, mass_in, mass_out, workspace=None, workspace_bytes=0, stream=None):
    """mass_out = mass_in + the attention weights of this call's query rows"""
    _check(lib().gpann_blocks_weigh(C.byref(layout.c), _p(q), _p(k), _p(probes), _u32("nprobe", nprobe), _p(lse), _p(mass_in), _p(mass_out), _p(workspace),
                                    _size("workspace_bytes", workspace_bytes), _p(stream)))


def evict(layout, k, v, mass, keep, rows, count, k_out=None, v_out=None, mass_out=None, first=0, last=0, out_kv_stride=None, workspace=None, workspace_bytes=0,
          stream=None):
    """keeps the first, last and heaviest rows of every sequence and head; out_kv_stride defaults to contiguous [batch][keep][kv_heads][head_dim]"""
    c = layout.c
    keep = _u32("keep", keep)
    strides = _strides("out_kv_stride", out_kv_stride or (keep * c.kv_heads * c.head_dim, c.kv_heads * c.head_dim, c.head_dim))
    _check(lib().gpann_blocks_evict(C.byref(c), _p(k), _p(v), _p(mass), keep, _u32("first", first), _u32("last", last), _p(rows), _p(count),
                                    _p(k_out), _p(v_out), C.byref(strides), _p(mass_out), _p(workspace), _size("workspace_bytes", workspace_bytes), _p(stream)))
