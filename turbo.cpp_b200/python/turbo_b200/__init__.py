"""Python binding of libturbo_b200.so, the C ABI in include/turbo_b200.h.

Used by the tests and bench.py to drive the CUDA kernels through exactly the
entry points a C/C++ caller uses.  Device memory comes from PyTorch tensors
(plumbing only); every computation is a kernel of the library.  There is no
fallback: if the library is missing or the device is not an sm_100 part, the
calls raise.
"""
import ctypes
import os

_HERE = os.path.dirname(os.path.abspath(__file__))
PKG_ROOT = os.path.dirname(os.path.dirname(_HERE))  # turbo.cpp_b200/
LIB_PATH = os.path.join(PKG_ROOT, "libturbo_b200.so")
HEADER = os.path.join(os.path.dirname(PKG_ROOT), "include", "turbo_b200.h")

MAX_RANK = 8
F32, F16, Q8_0, Q4_0, I32, BF16 = 0, 1, 2, 3, 4, 5
OK, EINVAL, ERANGE, ERUNTIME, ECUDA, ETIMEOUT, ENOMEM = range(7)


class TbError(RuntimeError):
    def __init__(self, status, msg):
        super().__init__("%s: %s" % (STATUS_NAMES.get(status, status), msg))
        self.status = status


STATUS_NAMES = {0: "TB_OK", 1: "TB_EINVAL", 2: "TB_ERANGE", 3: "TB_ERUNTIME", 4: "TB_ECUDA",
                5: "TB_ETIMEOUT", 6: "TB_ENOMEM"}


class View(ctypes.Structure):
    """tb_view: data, dtype, rank, offset, shape[8], strides[8] (elements)."""
    _fields_ = [("data", ctypes.c_void_p), ("dtype", ctypes.c_int32), ("rank", ctypes.c_int32),
                ("offset", ctypes.c_int64), ("shape", ctypes.c_int64 * MAX_RANK),
                ("strides", ctypes.c_int64 * MAX_RANK)]


class PagedCache(ctypes.Structure):
    """tb_paged_cache: the pools, their type, extents and strides (elements)."""
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("dtype", ctypes.c_int32),
                ("page_size", ctypes.c_int32), ("n_pages", ctypes.c_int64), ("kv_heads", ctypes.c_int64),
                ("head_dim", ctypes.c_int64), ("page_stride", ctypes.c_int64), ("token_stride", ctypes.c_int64),
                ("head_stride", ctypes.c_int64)]


class PagedBatch(ctypes.Structure):
    """tb_paged_batch: lengths and page table of a batch of sequences."""
    _fields_ = [("batch", ctypes.c_int64), ("lens", ctypes.c_void_p), ("table", ctypes.c_void_p),
                ("max_pages", ctypes.c_int64), ("table_stride", ctypes.c_int64)]


_P = ctypes.c_void_p
_I = ctypes.c_int
_I64 = ctypes.c_int64
_F = ctypes.c_float
_SZ = ctypes.c_size_t
_VP = ctypes.POINTER(View)
_PC = ctypes.POINTER(PagedCache)
_PB = ctypes.POINTER(PagedBatch)

SIGNATURES = {
    "tb_init": [_I],
    "tb_last_error": None,
    "tb_status_name": [_I],
    "tb_version": [],
    "tb_alloc": [ctypes.POINTER(_P), _SZ],
    "tb_free": [_P],
    "tb_upload": [_P, _P, _SZ, _P],
    "tb_download": [_P, _P, _SZ, _P],
    "tb_memset": [_P, _I, _SZ, _P],
    "tb_sync": [_P],
    "tb_take_device_errors": [ctypes.POINTER(ctypes.c_uint32)],
    "tb_set_wait_limit_ns": [ctypes.c_uint64],
    "tb_binary": [_I, _VP, _VP, _VP, _P],
    "tb_scale": [_VP, _F, _VP, _P],
    "tb_copy": [_VP, _VP, _P],
    "tb_rmsnorm": [_I, _P, _P, _P, _I64, _I64, _F, _P],
    "tb_swiglu": [_I, _P, _P, _P, _I64, _P],
    "tb_softmax": [_P, _P, _I64, _I64, _P],
    "tb_argmax": [_P, _I64, _I64, _P, _P],
    "tb_sample_top_p": [_P, _I64, _F, _F, ctypes.c_double, _P, _P],
    "tb_sample_top_p_at": [_P, _I64, _F, _F, _P, _P, _I64, _P, _P],
    "tb_rope": [_VP, _P, _P, _I64, _I64, _I64, _P],
    "tb_fill_upper": [_P, _I64, _I64, _I64, _I64, _F, _P],
    "tb_dequant": [_I, _P, _I64, _P, _P],
    "tb_quantize_q8_0": [_P, _I64, _I64, _P, _P],
    "tb_embedding": [_I, _P, _I64, _I64, _P, _I64, _P, _P],
    "tb_matmul_quant": [_I, _P, _I64, _I64, _P, _I64, _P, _P],
    "tb_matmul_quant_exact": [_I, _P, _I64, _I64, _P, _I64, _P, _P],
    "tb_matmul_q4_0_static_scratch": [_P, _I64, _I64, _P, _I64, _P, _P],
    "tb_packed_quant_weights_bytes": [_I, _I64, _I64, _P],
    "tb_pack_quant_weights": [_I, _P, _I64, _I64, _P, _SZ, _P],
    "tb_matmul_quant_packed": [_I, _P, _I64, _I64, _P, _I64, _P, _P],
    "tb_matmul_f32": [_VP, _VP, _VP, _P],
    "tb_softmax_shard_stats": [_P, _I64, _I64, _I64, _P, _P, _P],
    "tb_softmax_shard_rescale": [_P, _P, _P, _I64, _P],
    "tb_softmax_shard_finish": [_P, _I64, _I64, _I64, _P, _P, _P, _I64, _P],
    "tb_argmax_shard_keys": [_P, _I64, _I64, _I64, _I64, _P, _P],
    "tb_argmax_key_index": [_P, _I64, _P, _P],
    "tb_shard_group_unique_id": [_P],
    "tb_shard_group_create": [_I, _I, _P, _I64, ctypes.c_double, ctypes.POINTER(_P)],
    "tb_shard_group_wait": [_P, _P, ctypes.c_double],
    "tb_shard_group_abort": [_P],
    "tb_shard_group_destroy": [_P],
    "tb_softmax_vocab_sharded": [_P, _P, _I64, _I64, _I64, _P, _I64, _P],
    "tb_argmax_vocab_sharded": [_P, _P, _I64, _I64, _I64, _I64, _P, _P],
    "tb_shard_group_enable_peer": [_P, _I64],
    "tb_gemv_q8_0_row_sharded": [_P, _P, _I64, _P, _I64, _P, _P],
    "tb_decode_workspace_bytes": [_P, ctypes.POINTER(_SZ)],
    "tb_attention_prefill": [_P, _I64, _P, _P, _I64, _I64, _I64, _I64, _I64, _F, _P, _I64, _P],
    "tb_rope_paged_append": [_PC, _PB, _I, _P, _I64, _P, _I64, _P, _I64, _I64, _I64, _P, _P, _P, _I64, _P, _I64, _P],
    "tb_paged_attention_workspace_bytes": [_I64, _I64, _I64, _I64, ctypes.POINTER(_SZ)],
    "tb_paged_attention_decode": [_PC, _PB, _I, _P, _I64, _I64, _F, _P, _I64, _P, _SZ, _P],
    "tb_paged_attention_shared": [_PC, _PB, _P, _I64, _I, _P, _I64, _I64, _F, _P, _I64, _P, _SZ, _P],
    "tb_decode_step_persistent": [_P, _P],
    "tb_rope_at": [_VP, _P, _P, _I64, _I64, _P, _P],
    "tb_kv_append": [_P, _P, _P, _P, _I64, _I64, _P, _P],
    "tb_attention_decode": [_P, _P, _P, _I64, _I64, _I64, _I64, _F, _P, _P, _P],
    "tb_decode_margin": [_P, _I64, _P, _P, _I64, _P, _P],
    "tb_decode_advance": [_P, _P, _P, _P, _I64, _P],
    "tb_stream_create": [ctypes.POINTER(_P)],
    "tb_stream_destroy": [_P],
    "tb_capture_begin": [_P],
    "tb_capture_end": [_P, ctypes.POINTER(_P)],
    "tb_graph_launch": [_P, _P],
    "tb_graph_destroy": [_P],
    "tb_gemv_q8_0_multi": [_P, _I64, _P, _F, _P, _I, _P],
    "tb_gemv_q8_0_swiglu": [_P, _I64, _P, _F, _P, _P, _I64, _P, _P],
    "tb_rope_kv_append": [_P, _P, _P, _I64, _I64, _I64, _P, _P, _I64, _P, _P, _I64, _P, _P],
    "tb_prefetch_l2": [_P, _P, _I, _P],
    "tb_rope_attention_decode": [_P, _P, _P, _I64, _I64, _I64, _P, _P, _I64, _P, _P, _I64, _F, _P, _P, _P],
}


class GemvSegment(ctypes.Structure):
    """tb_gemv_segment: w, n, y, residual."""
    _fields_ = [("w", ctypes.c_void_p), ("n", ctypes.c_int64), ("y", ctypes.c_void_p), ("residual", ctypes.c_void_p)]

_lib = None


def load():
    """Loads the library (raises if it is not built)."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise ImportError("libturbo_b200.so is not built: run __graft_entry__.build() or "
                              "python turbo.cpp_b200/build.py")
        L = ctypes.CDLL(LIB_PATH)
        for name, args in SIGNATURES.items():
            fn = getattr(L, name)
            if name in ("tb_last_error", "tb_status_name", "tb_version"):
                fn.restype = ctypes.c_char_p
                fn.argtypes = [] if args is None else args
            else:
                fn.restype = ctypes.c_int
                fn.argtypes = args
        _lib = L
    return _lib


def lib():
    return load()


def check(status, what=""):
    if status != OK:
        msg = load().tb_last_error().decode(errors="replace")
        raise TbError(status, (what + ": " if what else "") + msg)


_FN = {}


def call(name, *args):
    fn = _FN.get(name)
    if fn is None:
        fn = _FN[name] = getattr(load(), name)
    status = fn(*args)
    if status != OK:
        check(status, name)


# ---- torch helpers -----------------------------------------------------------

_raw_stream = None


def stream_handle(stream=None):
    """The cudaStream_t of a torch stream, or of the current one."""
    global _raw_stream
    if stream is not None:
        return ctypes.c_void_p(stream.cuda_stream)
    if _raw_stream is None:
        import torch
        try:  # the handle alone: torch.cuda.current_stream() builds a Stream object around it (3 us)
            get, device = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice
            torch.cuda.current_stream()  # initialises CUDA
            get(device())
            _raw_stream = lambda: get(device())
        except AttributeError:
            _raw_stream = lambda: torch.cuda.current_stream().cuda_stream
    return ctypes.c_void_p(_raw_stream())


def ptr(t):
    return ctypes.c_void_p(t.data_ptr())


_DTYPES = {}


def dtype_code(t):
    if not _DTYPES:
        import torch
        _DTYPES.update({torch.float32: F32, torch.float16: F16, torch.int32: I32, torch.bfloat16: BF16})
    return _DTYPES[t.dtype]


def view(base, offset=None, shape=None, strides=None, dtype=None):
    """A tb_view over a torch tensor.  With explicit offset/shape/strides the
    view addresses `base`'s storage from its first element (the reference's
    Tensor{storage, offset, shape, strides}); otherwise it describes `base`."""
    v = View()
    if offset is None:
        v.data = base.data_ptr()
        v.offset = 0
        shape = list(base.shape)
        strides = list(base.stride())
    else:
        v.data = base.data_ptr()
        v.offset = int(offset)
    v.dtype = dtype if dtype is not None else dtype_code(base)
    v.rank = len(shape)
    for i, (s, st) in enumerate(zip(shape, strides)):
        v.shape[i] = int(s)
        v.strides[i] = int(st)
    return v


def paged_cache(k, v):
    """A tb_paged_cache over two pools given as torch tensors [pages,
    page_size, kv_heads, head_dim] (permuted views of head-major pools
    included).  The caller keeps the tensors."""
    if k.shape != v.shape or k.stride() != v.stride() or k.dtype != v.dtype or k.dim() != 4:
        raise ValueError("paged_cache: k and v need the same 4-d shape, strides and type")
    if k.shape[3] > 1 and k.stride(3) != 1:
        raise ValueError("paged_cache: the elements of a head must be contiguous")
    if not k.is_cuda or k.device != v.device:
        raise ValueError("paged_cache: k and v are in one GPU's memory")
    c = PagedCache()
    c.k, c.v, c.dtype = k.data_ptr(), v.data_ptr(), dtype_code(k)
    c.n_pages, c.page_size, c.kv_heads, c.head_dim = k.shape
    c.page_stride, c.token_stride, c.head_stride = k.stride()[:3]
    return c


def paged_batch(lens, table):
    """A tb_paged_batch over int32 tensors lens [batch] and table [batch,
    max_pages], whose rows may be those of a wider table but not overlap (as
    those of an expanded one).  The caller keeps the tensors."""
    import torch
    if lens.dtype != torch.int32 or table.dtype != torch.int32:
        raise ValueError("paged_batch: lens and table are int32")
    if lens.dim() != 1 or not lens.is_contiguous() or table.dim() != 2 or table.shape[0] != lens.shape[0] or (
            table.shape[1] > 1 and table.stride(1) != 1):
        raise ValueError("paged_batch: lens [batch], table [batch, max_pages] with contiguous rows")
    if table.shape[0] > 1 and table.stride(0) < table.shape[1]:
        raise ValueError("paged_batch: the table's rows overlap (an expanded table needs .contiguous())")
    if not lens.is_cuda or lens.device != table.device:
        raise ValueError("paged_batch: lens and table are in one GPU's memory")
    b = PagedBatch()
    b.batch, b.lens, b.table = lens.shape[0], lens.data_ptr(), table.data_ptr()
    b.max_pages, b.table_stride = table.shape[1], max(table.stride(0), table.shape[1])
    return b


def byref(v):
    return ctypes.byref(v)


def take_device_errors():
    flags = ctypes.c_uint32(0)
    call("tb_take_device_errors", ctypes.byref(flags))
    return flags.value
