"""tie_amd -- MI355X (gfx950) Qwen3-MoE FFN block for TIE.

The product is the C-ABI library ``libtie_hip.so`` (include/tie_hip.h),
built from tie_amd/csrc by tie_amd/Makefile.  This module is a thin ctypes
binding used by the tests and bench.py; it mirrors the C entry points one to
one and adds no computation of its own.  Importing it never falls back to a
CPU path: if the library is missing, every call raises.
"""
import ctypes
import os

import numpy as np

HERE = os.path.dirname(os.path.abspath(__file__))
# TIE_AMD_LIB selects another build of the same library (e.g. a tuning variant)
LIB_PATH = os.environ.get("TIE_AMD_LIB") or os.path.join(HERE, "libtie_hip.so")

F32, Q4_K, Q6_K, BF16 = 0, 12, 14, 30
F16, I8 = 1, 24  # cache types
PAGE_ROWS = 64
OK, EINVAL, EHIP, ENOMEM, ENOINIT = 0, -1, -2, -3, -4
PATH_AUTO, PATH_EXACT, PATH_MFMA = 0, 1, 2
ROUTE_SOFTMAX, ROUTE_SIGMOID = 0, 1
DEFAULT_STREAM = 1  # TIE_HIP_STREAM_DEFAULT: HIP's default stream
SILU_TABLE_SIZE = 8192

# every symbol include/tie_hip.h declares
EXPORTS = (
    "tie_hip_init", "tie_hip_shutdown", "tie_hip_last_error", "tie_hip_moe_ffn", "tie_hip_moe_ffn_lfm2",
    "tie_hip_qwen3_ffn", "tie_hip_moe_forward_residual", "tie_hip_matrix_create", "tie_hip_matrix_destroy",
    "tie_hip_mat_mat", "tie_hip_gguf_inspect", "tie_hip_gguf_tensor_info", "tie_hip_gguf_load", "tie_hip_model_info_get", "tie_hip_model_layer",
    "tie_hip_model_ffn_norm", "tie_hip_model_close", "tie_hip_set_silu_table",
    "tie_hip_silu_table_host", "tie_hip_layer_create", "tie_hip_layer_destroy", "tie_hip_layer_bytes",
    "tie_hip_moe_forward", "tie_hip_exact_max_tokens", "tie_hip_set_exact_max_tokens",
    "tie_hip_debug_fail_alloc", "tie_hip_host_expf", "tie_hip_profile_enable", "tie_hip_profile_read",
    "tie_hip_moe_forward_noalloc", "tie_hip_stream_status", "tie_hip_debug_decode_give_up", "tie_hip_debug_decode_form",
    "tie_hip_stream_release", "tie_hip_debug_layer_shifts",
    "tie_hip_kv_append", "tie_hip_kv_read", "tie_hip_kv_keep", "tie_hip_tree_attention",
    "tie_hip_tree_attention_work_bytes", "tie_hip_verify_tree", "tie_hip_verify_tree_work_bytes",
)


class TieError(RuntimeError):
    def __init__(self, code, msg):
        super().__init__("tie_hip error %d: %s" % (code, msg))
        self.code = code


class LayerDesc(ctypes.Structure):
    _fields_ = [
        ("d", ctypes.c_int), ("F", ctypes.c_int), ("E", ctypes.c_int),
        ("router_w", ctypes.c_void_p), ("router_type", ctypes.c_int),
        ("gate_exps", ctypes.c_void_p), ("gate_type", ctypes.c_int),
        ("up_exps", ctypes.c_void_p), ("up_type", ctypes.c_int),
        ("down_exps", ctypes.c_void_p), ("down_type", ctypes.c_int),
        ("router_bias", ctypes.c_void_p),
        ("src_on_device", ctypes.c_int),
        ("literal_bf16_stride", ctypes.c_int),
        ("routing", ctypes.c_int),
        ("probs_bias", ctypes.c_void_p),
    ]


class ModelInfo(ctypes.Structure):
    _fields_ = [
        ("architecture", ctypes.c_char * 32),
        ("d", ctypes.c_int), ("F", ctypes.c_int), ("E", ctypes.c_int), ("k", ctypes.c_int),
        ("n_layers", ctypes.c_int), ("first_moe_layer", ctypes.c_int),
        ("norm_eps", ctypes.c_float), ("routing", ctypes.c_int),
    ]


class KVCacheDesc(ctypes.Structure):
    _fields_ = [
        ("type", ctypes.c_int), ("n_layers", ctypes.c_int), ("n_pages", ctypes.c_int), ("kv_heads", ctypes.c_int),
        ("head_dim", ctypes.c_int), ("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("k_scale", ctypes.c_void_p),
        ("v_scale", ctypes.c_void_p),
    ]


class KVSeqsDesc(ctypes.Structure):
    _fields_ = [
        ("n_seqs", ctypes.c_int), ("max_pages", ctypes.c_int), ("n_tokens", ctypes.c_int),
        ("pages", ctypes.c_void_p), ("len", ctypes.c_void_p), ("first", ctypes.c_void_p),
    ]


_lib = None


def lib():
    """The loaded C-ABI library (raises if it has not been built)."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError("libtie_hip.so is not built: run `make -C tie_amd` or __graft_entry__.build()")
        L = ctypes.CDLL(LIB_PATH)
        P, I = ctypes.c_void_p, ctypes.c_int
        L.tie_hip_init.argtypes = [I]
        L.tie_hip_init.restype = I
        L.tie_hip_shutdown.restype = None
        L.tie_hip_last_error.restype = ctypes.c_char_p
        L.tie_hip_moe_ffn.argtypes = [P, I, I, I, I, I, P, I, P, I, P, I, P, I, P, P, P]
        L.tie_hip_moe_ffn.restype = I
        L.tie_hip_moe_ffn_lfm2.argtypes = [P, I, I, I, I, I, P, I, P, P, I, P, I, P, I, P, P, P]
        L.tie_hip_moe_ffn_lfm2.restype = I
        L.tie_hip_qwen3_ffn.argtypes = [P, I, I, I, I, I, P, ctypes.c_float, P, I, P, I, P, I, P, I, P, P]
        L.tie_hip_qwen3_ffn.restype = I
        L.tie_hip_moe_forward_residual.argtypes = [P, P, P, ctypes.c_float, I, I, P, P, P, I, P]
        L.tie_hip_moe_forward_residual.restype = I
        L.tie_hip_matrix_create.argtypes = [P, I, I, I, I, ctypes.POINTER(ctypes.c_void_p)]
        L.tie_hip_matrix_create.restype = I
        L.tie_hip_matrix_destroy.argtypes = [P]
        L.tie_hip_matrix_destroy.restype = None
        L.tie_hip_mat_mat.argtypes = [P, P, I, P, I, P]
        L.tie_hip_mat_mat.restype = I
        L.tie_hip_gguf_inspect.argtypes = [ctypes.c_char_p, ctypes.POINTER(ModelInfo)]
        L.tie_hip_gguf_inspect.restype = I
        L.tie_hip_gguf_tensor_info.argtypes = [ctypes.c_char_p, ctypes.c_char_p, P, P, P, P]
        L.tie_hip_gguf_tensor_info.restype = I
        L.tie_hip_gguf_load.argtypes = [ctypes.c_char_p, ctypes.POINTER(ctypes.c_void_p)]
        L.tie_hip_gguf_load.restype = I
        L.tie_hip_model_info_get.argtypes = [P, ctypes.POINTER(ModelInfo)]
        L.tie_hip_model_info_get.restype = None
        L.tie_hip_model_layer.argtypes = [P, I]
        L.tie_hip_model_layer.restype = P
        L.tie_hip_model_ffn_norm.argtypes = [P, I]
        L.tie_hip_model_ffn_norm.restype = P
        L.tie_hip_model_close.argtypes = [P]
        L.tie_hip_model_close.restype = None
        L.tie_hip_set_silu_table.argtypes = [P, I]
        L.tie_hip_set_silu_table.restype = I
        L.tie_hip_silu_table_host.argtypes = [P, I]
        L.tie_hip_silu_table_host.restype = I
        L.tie_hip_layer_create.argtypes = [ctypes.POINTER(LayerDesc), ctypes.POINTER(ctypes.c_void_p)]
        L.tie_hip_layer_create.restype = I
        L.tie_hip_layer_destroy.argtypes = [P]
        L.tie_hip_layer_destroy.restype = None
        L.tie_hip_layer_bytes.argtypes = [P]
        L.tie_hip_layer_bytes.restype = ctypes.c_size_t
        L.tie_hip_moe_forward.argtypes = [P, P, I, I, P, P, P, I, P]
        L.tie_hip_moe_forward.restype = I
        L.tie_hip_moe_forward_noalloc.argtypes = [P, P, I, I, P, P, P, I, P]
        L.tie_hip_moe_forward_noalloc.restype = I
        L.tie_hip_exact_max_tokens.restype = I
        L.tie_hip_set_exact_max_tokens.argtypes = [I]
        L.tie_hip_set_exact_max_tokens.restype = None
        L.tie_hip_debug_fail_alloc.argtypes = [I]
        L.tie_hip_debug_fail_alloc.restype = None
        L.tie_hip_host_expf.argtypes = [P, P, ctypes.c_size_t]
        L.tie_hip_host_expf.restype = None
        L.tie_hip_debug_layer_shifts.argtypes = [P, P, P]
        L.tie_hip_debug_layer_shifts.restype = I
        L.tie_hip_stream_release.argtypes = [P]
        L.tie_hip_stream_release.restype = I
        L.tie_hip_stream_status.argtypes = [P]
        L.tie_hip_stream_status.restype = I
        L.tie_hip_debug_decode_give_up.argtypes = [I]
        L.tie_hip_debug_decode_give_up.restype = None
        L.tie_hip_debug_decode_form.argtypes = [I]
        L.tie_hip_debug_decode_form.restype = None
        L.tie_hip_profile_enable.argtypes = [I]
        L.tie_hip_profile_enable.restype = I
        L.tie_hip_profile_read.argtypes = [ctypes.c_char_p, ctypes.c_size_t, P, P, I]
        L.tie_hip_profile_read.restype = I
        Z, F = ctypes.c_size_t, ctypes.c_float
        L.tie_hip_kv_append.argtypes = [P, I, P, P, Z, P, Z, P, Z, I, P, P, F, F, P, P, Z, P]
        L.tie_hip_kv_append.restype = I
        L.tie_hip_kv_read.argtypes = [P, I, I, P, P, P, P]
        L.tie_hip_kv_read.restype = I
        L.tie_hip_kv_keep.argtypes = [P, P, P, I, P, P, P]
        L.tie_hip_kv_keep.restype = I
        L.tie_hip_tree_attention.argtypes = [P, I, P, P, Z, I, F, P, I, P, Z, P, Z, P]
        L.tie_hip_tree_attention.restype = I
        L.tie_hip_tree_attention_work_bytes.argtypes = [P, P, I]
        L.tie_hip_tree_attention_work_bytes.restype = Z
        L.tie_hip_verify_tree.argtypes = [P, Z, P, Z, I, I, I, P, P, P, P, P, F, I, I, P, P, P, P, Z, P]
        L.tie_hip_verify_tree.restype = I
        L.tie_hip_verify_tree_work_bytes.argtypes = [I, I, I, I]
        L.tie_hip_verify_tree_work_bytes.restype = Z
        _lib = L
    return _lib


def last_error():
    return lib().tie_hip_last_error().decode()


def check(rc):
    if rc != OK:
        raise TieError(rc, last_error())
    return rc


def _p(a):
    if a is None:
        return None
    if isinstance(a, int):
        return a
    if hasattr(a, "data_ptr"):
        return a.data_ptr()
    return a.ctypes.data


def _s(stream):
    """A stream's handle for the library.  None is the library's own stream;
    torch's handle of the default stream, 0, would be that one too."""
    return DEFAULT_STREAM if stream == 0 else stream


_device = None  # the library's GPU


def init(device=0):
    global _device
    check(lib().tie_hip_init(device))
    _device = device


def shutdown():
    global _device
    lib().tie_hip_shutdown()
    _device = None


def silu_table_host():
    t = np.empty(SILU_TABLE_SIZE, np.float32)
    check(lib().tie_hip_silu_table_host(_p(t), SILU_TABLE_SIZE))
    return t


def set_silu_table(table):
    table = np.ascontiguousarray(table, np.float32)
    check(lib().tie_hip_set_silu_table(_p(table), table.size))


def host_expf(x):
    x = np.ascontiguousarray(x, np.float32)
    out = np.empty_like(x)
    lib().tie_hip_host_expf(_p(x), _p(out), x.size)
    return out


def stream_status(stream=None):
    """tie_hip_stream_status: raises TieError when a one-token forward on
    the stream had a wait between workgroups give up since the last check."""
    check(lib().tie_hip_stream_status(_s(stream)))


def stream_release(stream=None):
    """tie_hip_stream_release: free the workspace kept for the stream."""
    check(lib().tie_hip_stream_release(_s(stream)))


def debug_decode_give_up(n):
    lib().tie_hip_debug_decode_give_up(int(n))


def debug_decode_form(form):
    """Force the one-token kernel's form (0 a lane per dot, 1 lane pairs;
    -1 by the shape)."""
    lib().tie_hip_debug_decode_form(int(form))


def profile_enable(on=True):
    check(lib().tie_hip_profile_enable(int(on)))


def profile_read(max_kernels=32):
    """{kernel name: (total ms, launches)} since profile_enable(True)."""
    names = ctypes.create_string_buffer(4096)
    tot = np.zeros(max_kernels, np.float64)
    cnt = np.zeros(max_kernels, np.int32)
    n = lib().tie_hip_profile_read(names, 4096, _p(tot), _p(cnt), max_kernels)
    if n < 0:
        check(n)
    keys = names.value.decode().split(",") if n else []
    return {k: (float(tot[i]), int(cnt[i])) for i, k in enumerate(keys)}


def moe_ffn(x, layer, k, with_topk=True):
    """tie_hip_moe_ffn on host arrays (the drop-in for model_qwen3.c:404-471),
    or tie_hip_moe_ffn_lfm2 (model_lfm2.c:414-497) for a layer with sigmoid
    routing.  `layer` is a tie_amd.synth.MoELayer (GGUF-layout host arrays)."""
    x = np.ascontiguousarray(x, np.float32)
    T, d = x.shape
    out = np.empty((T, d), np.float32)
    idx = np.empty((T, k), np.int32) if with_topk else None
    w = np.empty((T, k), np.float32) if with_topk else None
    if layer.bias is not None:
        raise ValueError("the host drop-ins take no logit bias (TIE has none); use Layer for biased routing")
    if getattr(layer, "routing", ROUTE_SOFTMAX) == ROUTE_SIGMOID:
        # tie_hip_moe_ffn_lfm2: the drop-in for model_lfm2.c:414-497
        check(lib().tie_hip_moe_ffn_lfm2(_p(x), T, d, layer.F, layer.E, k, _p(layer.router), F32,
                                         _p(layer.probs_bias), _p(layer.gate), layer.gate_type, _p(layer.up),
                                         layer.up_type, _p(layer.down), layer.down_type, _p(out), _p(idx),
                                         _p(w)))
    else:
        check(lib().tie_hip_moe_ffn(_p(x), T, d, layer.F, layer.E, k, _p(layer.router), F32, _p(layer.gate),
                                    layer.gate_type, _p(layer.up), layer.up_type, _p(layer.down),
                                    layer.down_type, _p(out), _p(idx), _p(w)))
    return out, idx, w


def qwen3_ffn(hidden, layer, k, ffn_norm, eps, with_topk=True):
    """tie_hip_qwen3_ffn on host arrays: the FFN half of transformer_layer_qwen3
    (RMSNorm, MoE block, residual add; model_qwen3.c:392-491).  Returns the
    new hidden state (the input array is not changed) and the selection."""
    h = np.array(hidden, np.float32, copy=True, order="C")
    T, d = h.shape
    idx = np.empty((T, k), np.int32) if with_topk else None
    w = np.empty((T, k), np.float32) if with_topk else None
    norm = np.ascontiguousarray(ffn_norm, np.float32)
    check(lib().tie_hip_qwen3_ffn(_p(h), T, d, layer.F, layer.E, k, _p(norm), eps, _p(layer.router), F32,
                                  _p(layer.gate), layer.gate_type, _p(layer.up), layer.up_type, _p(layer.down),
                                  layer.down_type, _p(idx), _p(w)))
    return h, idx, w


def gguf_tensor_info(path, name):
    """tie_hip_gguf_tensor_info: (type, ne[4], file offset, bytes) of one
    tensor as the library's reader maps it (no GPU needed)."""
    t = ctypes.c_int(0)
    ne = np.zeros(4, np.uint64)
    off = ctypes.c_uint64(0)
    nb = ctypes.c_uint64(0)
    rc = lib().tie_hip_gguf_tensor_info(os.fsencode(path), name.encode(), ctypes.byref(t), _p(ne),
                                        ctypes.byref(off), ctypes.byref(nb))
    check(min(rc, 0))  # >= 0: the tensor count
    return t.value, tuple(int(v) for v in ne), off.value, nb.value


def gguf_tensor_count(path):
    n = lib().tie_hip_gguf_tensor_info(os.fsencode(path), None, None, None, None, None)
    check(min(n, 0))
    return n


def gguf_inspect(path):
    """tie_hip_gguf_inspect: the MoE shape of a GGUF file (no GPU needed)."""
    info = ModelInfo()
    check(lib().tie_hip_gguf_inspect(os.fsencode(path), ctypes.byref(info)))
    return info


class _LayerRef:
    """A layer owned by a Model (forward/forward_residual of Layer, no close)."""

    def __init__(self, handle):
        self.handle = handle

    forward = lambda self, *a, **kw: Layer.forward(self, *a, **kw)  # noqa: E731
    forward_residual = lambda self, *a, **kw: Layer.forward_residual(self, *a, **kw)  # noqa: E731


class Model:
    """tie_hip_gguf_load: every MoE layer of a GGUF file on the device."""

    def __init__(self, path):
        h = ctypes.c_void_p()
        check(lib().tie_hip_gguf_load(os.fsencode(path), ctypes.byref(h)))
        self.handle = h
        self.info = ModelInfo()
        lib().tie_hip_model_info_get(h, ctypes.byref(self.info))

    def layer(self, n):
        h = lib().tie_hip_model_layer(self.handle, n)
        return _LayerRef(ctypes.c_void_p(h)) if h else None

    def ffn_norm(self, n):
        """Device pointer (int) of layer n's ffn_norm, or None."""
        return lib().tie_hip_model_ffn_norm(self.handle, n)

    def close(self):
        if self.handle:
            lib().tie_hip_model_close(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class Matrix:
    """A device-resident dense weight matrix (tie_hip_matrix_create):
    GGUF layout [rows][in_dim] of type F32, Q4_K, Q6_K or BF16."""

    def __init__(self, w, wtype, rows, in_dim, on_device=False):
        self.rows, self.in_dim = rows, in_dim
        h = ctypes.c_void_p()
        check(lib().tie_hip_matrix_create(_p(w), wtype, rows, in_dim, int(on_device), ctypes.byref(h)))
        self.handle = h

    def mat_mat(self, x_dev, T, out_dev, flags=PATH_AUTO, stream=None):
        """out[t][r] = W[r] . x[t] on device pointers (dispatch_mat_mat);
        PATH_AUTO takes the matrix cores above the exact threshold where the
        matrix allows them, PATH_EXACT always TIE's row kernels."""
        check(lib().tie_hip_mat_mat(self.handle, _p(x_dev), T, _p(out_dev), flags, _s(stream)))

    def close(self):
        if self.handle:
            lib().tie_hip_matrix_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class Layer:
    """A device-resident layer (tie_hip_layer_create).  Weight sources are
    host numpy arrays or device tensors (anything with data_ptr())."""

    def __init__(self, d, F, E, router, gate, up, down, gate_type, up_type, down_type, bias=None,
                 on_device=False, literal_bf16_stride=False, routing=ROUTE_SOFTMAX, probs_bias=None):
        self.d, self.F, self.E = d, F, E
        desc = LayerDesc(d, F, E, _p(router), F32, _p(gate), gate_type, _p(up), up_type, _p(down), down_type,
                         _p(bias), int(on_device), int(literal_bf16_stride), int(routing), _p(probs_bias))
        h = ctypes.c_void_p()
        check(lib().tie_hip_layer_create(ctypes.byref(desc), ctypes.byref(h)))
        self.handle = h

    @classmethod
    def from_synth(cls, s, literal_bf16_stride=False):
        return cls(s.d, s.F, s.E, s.router, s.gate, s.up, s.down, s.gate_type, s.up_type, s.down_type,
                   bias=s.bias, literal_bf16_stride=literal_bf16_stride,
                   routing=getattr(s, "routing", ROUTE_SOFTMAX), probs_bias=getattr(s, "probs_bias", None))

    def nbytes(self):
        return lib().tie_hip_layer_bytes(self.handle)

    def shifts(self):
        """(h_shift, y_shift): the matrix-core path's f16 scales of h and y."""
        h, y = ctypes.c_int(0), ctypes.c_int(0)
        check(lib().tie_hip_debug_layer_shifts(self.handle, ctypes.byref(h), ctypes.byref(y)))
        return h.value, y.value

    def forward(self, x_dev, T, k, out_dev, topk_idx_dev=None, topk_w_dev=None, flags=PATH_AUTO, stream=None):
        """Enqueue the block on device pointers (torch tensors or ints)."""
        check(lib().tie_hip_moe_forward(self.handle, _p(x_dev), T, k, _p(out_dev), _p(topk_idx_dev),
                                        _p(topk_w_dev), flags, _s(stream)))

    def forward_noalloc(self, x_dev, T, k, out_dev, topk_idx_dev=None, topk_w_dev=None, flags=PATH_AUTO,
                        stream=None):
        """tie_hip_moe_forward_noalloc: forward with the library's static
        scratch array (no allocation; small T only)."""
        check(lib().tie_hip_moe_forward_noalloc(self.handle, _p(x_dev), T, k, _p(out_dev), _p(topk_idx_dev),
                                                _p(topk_w_dev), flags, _s(stream)))

    def forward_residual(self, hidden_dev, ffn_norm_dev, eps, T, k, out_dev=None, topk_idx_dev=None,
                         topk_w_dev=None, flags=PATH_AUTO, stream=None):
        """out = hidden + block(rms_norm(hidden)) on device pointers (out
        defaults to hidden: the in-place update)."""
        check(lib().tie_hip_moe_forward_residual(self.handle, _p(hidden_dev), _p(ffn_norm_dev), eps, T, k,
                                                 _p(hidden_dev if out_dev is None else out_dev), _p(topk_idx_dev),
                                                 _p(topk_w_dev), flags, _s(stream)))

    def close(self):
        if self.handle:
            lib().tie_hip_layer_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def _dtype(name):
    """torch's type of this name (torch is the caller's: the library needs none)."""
    t = _dtypes.get(name)
    if t is None:
        import torch
        t = _dtypes[name] = getattr(torch, name)
    return t


_dtypes = {}


def _on_device(device, other, what):
    """Tensors of another GPU than the library's, or of the CPU, would be read as addresses of it."""
    if other != device or (_device is not None and device != _device):
        raise ValueError("%s on device %s: device %s is wanted" % (what, other, device if _device is None else _device))


def _rows(a, what, device, width=None, n_rows=0):
    """(pointer, row stride, values of a row) of n_rows or more F32 rows: a 2-D
    tensor, or one of [rows][heads][head_dim] whose rows are contiguous."""
    st, sh = a.stride(), a.shape
    if len(st) == 2:
        n, inner = sh[1], st[1] == 1 or sh[1] == 1
    elif len(st) == 3:
        n = sh[1] * sh[2]
        inner = (st[2] == 1 or sh[2] == 1) and (st[1] == sh[2] or sh[1] == 1)
    else:
        n, inner = -1, False
    if a.dtype is not (_dtypes.get("float32") or _dtype("float32")) or not inner or (width is not None and n != width) or sh[0] < n_rows or \
            (st[0] < n and sh[0] > 1):
        raise ValueError("%s: %d rows of %s contiguous float32 values are wanted (got %s, shape %s, strides %s)"
                         % (what, n_rows, width or "", a.dtype, tuple(sh), st))
    if a.get_device() != device:
        _on_device(device, a.get_device(), what)
    return a.data_ptr(), (st[0] if st[0] > n else n), n


def _array(a, dtype, shape, what, device):
    """The pointer of a contiguous array on `device` of this type and shape (None for None)."""
    if a is None:
        return None
    if a.dtype is not (_dtypes.get(dtype) or _dtype(dtype)) or a.shape != shape or not a.is_contiguous():
        raise ValueError("%s: a contiguous %s array of shape %s is wanted (got %s, %s)" % (what, dtype, tuple(shape), a.dtype,
                                                                                           tuple(a.shape)))
    if a.get_device() != device:
        _on_device(device, a.get_device(), what)
    return a.data_ptr()


_raw_stream = None


def _current(stream, device):
    """The handle of `stream`; None: the stream that torch works on now, on which the tensors are made and used."""
    if stream is None:
        if device < 0:
            return None  # (tensors of the CPU: the call is refused)
        global _raw_stream
        if _raw_stream is None:
            from torch._C import _cuda_getCurrentRawStream
            _raw_stream = _cuda_getCurrentRawStream  # (torch.cuda.current_stream makes an object for each call)
        stream = _raw_stream(device)
    return stream or DEFAULT_STREAM


def _work(work, device):
    """Pointer and bytes of a call's scratch memory (None: the stream's own)."""
    if work is None:
        return None, 0
    if not work.is_contiguous() or work.get_device() != device:
        _on_device(device, work.get_device(), "work")
        raise ValueError("work: contiguous memory is wanted")
    return work.data_ptr(), work.numel() * work.element_size()


class KVSeqs:
    """The sequences of a call (tie_hip_kv_seqs): device int32 tensors `pages`
    [n_seqs][max_pages], `lens` [n_seqs] and `first` [n_seqs + 1] (None: one
    token each), read when the kernels run; n_tokens rows of activations."""

    def __init__(self, pages, lens, first=None, n_tokens=None):
        n_seqs, max_pages = pages.shape
        if n_tokens is None:
            n_tokens = n_seqs if first is None else int(first[-1])
        dev = pages.get_device()
        self.n_seqs, self.n_tokens, self.device, self.keep = n_seqs, n_tokens, dev, (pages, lens, first)
        self.desc = KVSeqsDesc(n_seqs, max_pages, n_tokens, _array(pages, "int32", pages.shape, "pages", dev),
                               _array(lens, "int32", (n_seqs,), "lens", dev),
                               _array(first, "int32", (n_seqs + 1,), "first", dev))
        self.ref = ctypes.byref(self.desc)


class KVCache:
    """A paged cache in the caller's tensors (tie_hip_kv_cache): k [n_layers]
    [n_pages][kv_heads][64][head_dim] and v [n_layers][n_pages][kv_heads]
    [head_dim][64], float16, or int8 with float32 scales [n_layers][n_pages]
    [kv_heads][64].

    The calls go to `stream`, or, where that is None, to the stream that torch
    works on when they are made, in order with the tensors' other uses.  (None
    is the library's own stream for Layer and Matrix, whose buffers need not be
    torch's: calls of both kinds in one program get one stream.)"""

    def __init__(self, k, v, k_scale=None, v_scale=None):
        kind = {"torch.float16": F16, "torch.int8": I8}.get(str(k.dtype))
        if kind is None or len(k.shape) != 5 or k.shape[3] != PAGE_ROWS:
            raise ValueError("k: [layers][pages][kv heads][%d][head_dim] of float16 or int8 is wanted (got %s, %s)"
                             % (PAGE_ROWS, k.dtype, tuple(k.shape)))
        nl, npg, kvh, _, hd = k.shape
        name = str(k.dtype)[6:]
        if kind == I8 and (k_scale is None or v_scale is None):
            raise ValueError("an int8 cache needs k_scale and v_scale")
        self.kv_heads, self.head_dim, self.n_layers, self.keep_alive = kvh, hd, nl, (k, v, k_scale, v_scale)
        self.width, self.head_shape, self.device = kvh * hd, (hd,), k.get_device()
        dev = self.device
        self.desc = KVCacheDesc(kind, nl, npg, kvh, hd, _array(k, name, k.shape, "k", dev),
                                _array(v, name, (nl, npg, kvh, hd, PAGE_ROWS), "v", dev),
                                _array(k_scale, "float32", k.shape[:4], "k_scale", dev),
                                _array(v_scale, "float32", k.shape[:4], "v_scale", dev))
        self.ref = ctypes.byref(self.desc)

    def _heads(self, width, what):
        if width % self.head_dim:
            raise ValueError("%s: rows of %d values are no whole heads of %d" % (what, width, self.head_dim))
        return width // self.head_dim

    def _seqs(self, seqs):
        if seqs.device != self.device or self.device != _device:
            _on_device(self.device, seqs.device, "seqs")

    def _q(self, q, out, seqs, what):
        self._seqs(seqs)
        pq, sq, w = _rows(q, "q", self.device, None, seqs.n_tokens)
        if out is q:
            po, so = pq, sq
        else:
            po, so, _ = _rows(out, what, self.device, w, seqs.n_tokens)
        return pq, sq, po, so, self._heads(w, "q")

    def append(self, layer, seqs, q, k, v, q_out, pos=None, q_norm=None, k_norm=None, eps=1e-6, theta=1e6, stream=None):
        """tie_hip_kv_append: norm and rotation of q and k, cache write of k and v."""
        n, dev = seqs.n_tokens, self.device
        pq, sq, po, so, heads = self._q(q, q_out, seqs, "q_out")
        pk, sk, _ = _rows(k, "k", dev, self.width, n)
        pv, sv, _ = _rows(v, "v", dev, self.width, n)
        check(lib().tie_hip_kv_append(self.ref, layer, seqs.ref, pq, sq, pk, sk, pv, sv, heads,
                                      _array(q_norm, "float32", self.head_shape, "q_norm", dev),
                                      _array(k_norm, "float32", self.head_shape, "k_norm", dev), eps, theta,
                                      _array(pos, "int32", (n,), "pos", dev), po, so, _current(stream, dev)))

    def read(self, seqs, k_out, v_out, layer=0, n_layers=1, stream=None):
        """tie_hip_kv_read: rows of the cache as float32 [n_layers][n_tokens][kv_heads][head_dim]."""
        self._seqs(seqs)
        shape, dev = (n_layers, seqs.n_tokens, self.kv_heads, self.head_dim), self.device
        check(lib().tie_hip_kv_read(self.ref, layer, n_layers, seqs.ref, _array(k_out, "float32", shape, "k_out", dev),
                                    _array(v_out, "float32", shape, "v_out", dev), _current(stream, dev)))

    def attention(self, layer, seqs, q, out, scale, mask=None, work=None, stream=None):
        """tie_hip_tree_attention; mask: int64 [n_tokens][words] (bit patterns), None: causal; work: a uint8 tensor."""
        pq, sq, po, so, heads = self._q(q, out, seqs, "out")
        words, (pw, nw) = 0 if mask is None else mask.shape[1], _work(work, self.device)
        check(lib().tie_hip_tree_attention(self.ref, layer, seqs.ref, pq, sq, heads, scale,
                                           _array(mask, "int64", (seqs.n_tokens, words), "mask", self.device), words, po, so, pw,
                                           nw, _current(stream, self.device)))

    def attention_work_bytes(self, seqs, n_heads):
        return lib().tie_hip_tree_attention_work_bytes(self.ref, seqs.ref, n_heads)

    def keep(self, seqs, path, n_keep, len_out=None, stream=None):
        """tie_hip_kv_keep: the accepted paths' rows moved down in every layer."""
        self._seqs(seqs)
        dev = self.device
        check(lib().tie_hip_kv_keep(self.ref, seqs.ref, _array(path, "int32", (seqs.n_seqs, path.shape[1]), "path", dev),
                                    path.shape[1], _array(n_keep, "int32", (seqs.n_seqs,), "n_keep", dev),
                                    _array(len_out, "int32", (seqs.n_seqs,), "len_out", dev), _current(stream, dev)))


def verify_tree_work_bytes(vocab, n_tokens, max_children, with_draft):
    return lib().tie_hip_verify_tree_work_bytes(vocab, n_tokens, max_children, int(with_draft))


def verify_tree(logits, first, tokens, parent, u_accept, u_sample, path, n_keep, next_token, temperature=1.0, draft=None,
                max_children=1, work=None, stream=None):
    """tie_hip_verify_tree: the accepted path [n_seqs][max_path], its length and the next token of each sequence; stream
    as for KVCache."""
    n, n_seqs, dev = tokens.shape[0], n_keep.shape[0], logits.get_device()
    if dev != _device:
        _on_device(dev, dev, "logits")
    pl, sl, vocab = _rows(logits, "logits", dev, None, n)
    pd, sd, _ = (None, 0, 0) if draft is None else _rows(draft, "draft", dev, vocab, n)
    pw, nw = _work(work, dev)
    check(lib().tie_hip_verify_tree(pl, sl, pd, sd, vocab, n_seqs, n, _array(first, "int32", (n_seqs + 1,), "first", dev),
                                    _array(tokens, "int32", (n,), "tokens", dev), _array(parent, "int32", (n,), "parent", dev),
                                    _array(u_accept, "float32", (n,), "u_accept", dev),
                                    _array(u_sample, "float32", (n,), "u_sample", dev), temperature, max_children, path.shape[1],
                                    _array(path, "int32", (n_seqs, path.shape[1]), "path", dev),
                                    _array(n_keep, "int32", (n_seqs,), "n_keep", dev),
                                    _array(next_token, "int32", (n_seqs,), "next_token", dev), pw, nw,
                                    _current(stream, dev)))
