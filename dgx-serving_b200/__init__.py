"""Host-side Python binding of libw4a8_b200.so, the B200 (sm_100a) W4A8 quantized-matmul library.

The product is the C-ABI shared library (include/w4a8_b200.h) plus the C++ shim launchers in
kernels/*.cuh that carry the reference's launcher names.  This module is the thin ctypes layer the
tests and the benchmark use to call that ABI with torch tensors as device memory; torch is plumbing
(allocation, streams, torch.distributed), never a compute path.  There is no CPU or torch fallback:
if the library is missing or the device is not sm_100 every call raises.

Function names and argument order mirror the reference launchers
(kernels/quantize_x.cuh:41, kernels/gemv_w4a8.cuh:155,168, kernels/gemm_batch.cuh:228,
kernels/gemm_mmq.cuh:230, kernels/gemm_mmq_raster.cuh:115).
"""
import ctypes
import importlib.machinery
import importlib.util
import os

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.environ.get("W4A8_LIB") or os.path.join(_HERE, "libw4a8_b200.so")   # W4A8_LIB: another build, for A/B timing
QBLK = 32

OK, ERR_ARG, ERR_ALIGN, ERR_CUDA, ERR_IO, ERR_DEVICE, ERR_UNSUPPORTED, ERR_WORKSPACE = range(8)

_lib = None


class W4A8Error(RuntimeError):
    def __init__(self, code, text):
        super().__init__("w4a8 error %d: %s" % (code, text))
        self.code = code


class QMat(ctypes.Structure):
    """Mirror of w4a8_qmat (the N-sharded form of the reference's QMat, runtime/weights_qwen.h:8)."""
    _fields_ = [("wq", ctypes.c_void_p), ("sc", ctypes.c_void_p), ("row0", ctypes.c_int64),
                ("rows", ctypes.c_int64), ("N", ctypes.c_int64), ("K", ctypes.c_int64),
                ("scale_dtype", ctypes.c_int)]


class MoeLayout(ctypes.Structure):
    """Mirror of w4a8_moe_layout: byte offsets of the routed-expert block's intermediates in the caller's workspace."""
    _fields_ = [(n, ctypes.c_size_t) for n in ("perm", "pos", "offsets", "items", "num_items", "xq", "xs", "xq_g", "xs_g", "gu",
                                               "xq_h", "xs_h", "sout", "bytes")]


class KVCache(ctypes.Structure):
    """Mirror of w4a8_kv_cache: codes k, v [num_blocks][heads][block][dim] int8, scales [num_blocks][heads] fp32."""
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("k_scale", ctypes.c_void_p), ("v_scale", ctypes.c_void_p),
                ("num_blocks", ctypes.c_int), ("heads", ctypes.c_int), ("block", ctypes.c_int), ("dim", ctypes.c_int)]

    @classmethod
    def of(cls, k, v, k_scale, v_scale):
        """The cache in four tensors, which the object keeps alive."""
        for t in (k, v, k_scale, v_scale):
            if not t.is_contiguous():
                raise ValueError("a KV cache's tensors are contiguous")
        if k.dim() != 4 or k.shape != v.shape or k_scale.shape != k.shape[:2] or v_scale.shape != k.shape[:2]:
            raise ValueError("k, v: [num_blocks][heads][block][dim]; k_scale, v_scale: [num_blocks][heads]")
        if [str(t.dtype) for t in (k, v, k_scale, v_scale)] != ["torch.int8", "torch.int8", "torch.float32", "torch.float32"]:
            raise ValueError("a KV cache holds int8 codes and fp32 scales")
        if len({t.device for t in (k, v, k_scale, v_scale)}) != 1:
            raise ValueError("a KV cache's tensors are on one device")
        c = cls(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), *k.shape)
        c._tensors = (k, v, k_scale, v_scale)
        c._host = not k.is_cuda
        return c


def _fp32_vector(t, n, name):
    """A contiguous fp32 tensor of n elements on a GPU, or None."""
    if t is not None and (str(t.dtype) != "torch.float32" or t.numel() != n or not t.is_contiguous() or not t.is_cuda):
        raise ValueError("%s: %d contiguous fp32 numbers on a GPU" % (name, n))
    return t


def _gpu_of(tensors, name):
    """The GPU that all tensors of a struct lie on (-1: host memory), None without any."""
    at = {t.get_device() for t in tensors if t is not None}
    if len(at) > 1:
        raise ValueError("%s: tensors that are not on one GPU" % name)
    return at.pop() if at else None


def struct_on(struct, device, name):
    """Refuses a Norm, Rope or Router whose tensors are not on `device`."""
    if struct._gpu is not None and struct._gpu != (device.index if device.type == "cuda" else -1):
        raise ValueError("%s: tensors that are not on %s" % (name, device))


class Norm(ctypes.Structure):
    """Mirror of w4a8_norm: the weights and constants of one residual add with its norms."""
    _fields_ = [("weight", ctypes.c_void_p), ("post_weight", ctypes.c_void_p), ("gate", ctypes.c_void_p), ("gate_ld", ctypes.c_int64), ("eps", ctypes.c_double),
                ("alpha", ctypes.c_float), ("K", ctypes.c_int), ("variant", ctypes.c_int), ("post_variant", ctypes.c_int), ("dtype", ctypes.c_int), ("y_dtype", ctypes.c_int)]

    _gate_rows = 1 << 63
    _gpu = None

    @classmethod
    def of(cls, K, weight=None, variant=0, eps=1e-6, post_weight=None, post_variant=-1, gate=None, alpha=1.0, dtype="fp32", y_dtype=None):
        """weight, post_weight: fp32 [K] tensors, which the object keeps alive.  gate: fp32 [K], or [S][K] with a row for each token.  variant -1: no norm,
        0: * weight, 1: * (1 + weight), 2: no weight.  y_dtype None: dtype."""
        _fp32_vector(weight, K, "weight")
        _fp32_vector(post_weight, K, "post_weight")
        gate_ld = 0
        if gate is not None and gate.dim() == 2 and gate.shape[0] == 1:
            gate = gate[0]
        if gate is not None:
            if str(gate.dtype) != "torch.float32" or not gate.is_cuda or gate.dim() not in (1, 2) or gate.shape[-1] != K or (K > 1 and gate.stride(-1) != 1):
                raise ValueError("gate: fp32 [%d] or [rows][%d] on a GPU" % (K, K))
            gate_ld = gate.stride(0) if gate.dim() == 2 else 0
            if gate.dim() == 2 and gate_ld < K:
                raise ValueError("gate: rows that overlap")
        n = cls(_ptr(weight), _ptr(post_weight), _ptr(gate), gate_ld, float(eps), float(alpha), K, variant, post_variant, DTYPES[dtype], DTYPES[dtype if y_dtype is None else y_dtype])
        n._tensors = (weight, post_weight, gate)
        n._gpu = _gpu_of(n._tensors, "Norm")
        if gate_ld:
            n._gate_rows = gate.shape[0]
        return n


ROPE_SCALINGS = {"none": 0, "linear": 1, "ntk": 2, "yarn": 3, "bands": 4, "divisors": 5}


def rope_table(rotary, base=10000.0, scaling="none", factor=1.0, original=0.0, low=0.0, high=0.0, divisors=None):
    """The frequencies of rotary / 2 pairs in units of 2^-64 turn a token (a list of whole numbers), and what cosine and sine are multiplied by
    (w4a8_rope_table)."""
    n = max(0, rotary) // 2
    if divisors is not None and len(divisors) != n:
        raise ValueError("divisors: one for each of the %d pairs" % n)
    turns, magnitude = (ctypes.c_uint64 * max(1, n))(), ctypes.c_float(0.0)
    _check(lib().w4a8_rope_table(rotary, float(base), ROPE_SCALINGS[scaling], float(factor), float(original), float(low), float(high),
                                 None if divisors is None else (ctypes.c_double * max(1, n))(*[float(d) for d in divisors]), turns, ctypes.byref(magnitude)))
    return list(turns[:n]), magnitude.value


class Rope(ctypes.Structure):
    """Mirror of w4a8_rope: frequencies of rotary positions on the GPU, and the norms of queries and keys."""
    _fields_ = [("turns", ctypes.c_void_p), ("q_weight", ctypes.c_void_p), ("k_weight", ctypes.c_void_p), ("eps", ctypes.c_double), ("magnitude", ctypes.c_float),
                ("dim", ctypes.c_int), ("rotary", ctypes.c_int), ("interleaved", ctypes.c_int), ("variant", ctypes.c_int)]

    _host = False
    _gpu = None

    @classmethod
    def of(cls, dim, rotary, base=10000.0, scaling="none", interleaved=False, q_weight=None, k_weight=None, variant=-1, eps=1e-6, device="cuda", magnitude=None, **parameters):
        """Heads of `dim` elements, the first `rotary` of them turned.  scaling and parameters: rope_table's; magnitude: instead of the scaling's own.
        q_weight, k_weight: fp32 [dim], kept alive as the table is."""
        import torch
        _fp32_vector(q_weight, dim, "q_weight")
        _fp32_vector(k_weight, dim, "k_weight")
        turns, m = rope_table(rotary, base, scaling, **parameters)
        table = torch.tensor([t - (1 << 64) if t >> 63 else t for t in turns], dtype=torch.int64, device=device)
        r = cls(_ptr(table) if turns else None, _ptr(q_weight), _ptr(k_weight), float(eps), float(m if magnitude is None else magnitude), dim, rotary, int(bool(interleaved)), variant)
        r._tensors = (table, q_weight, k_weight)
        r._host = bool(turns) and not table.is_cuda
        r._gpu = _gpu_of((table if turns else None, q_weight, k_weight), "Rope")
        return r


class Router(ctypes.Structure):
    """Mirror of w4a8_router: how experts are chosen."""
    _fields_ = [("bias", ctypes.c_void_p), ("experts", ctypes.c_int), ("topk", ctypes.c_int), ("scoring", ctypes.c_int), ("groups", ctypes.c_int), ("topk_groups", ctypes.c_int),
                ("group_score", ctypes.c_int), ("renormalise", ctypes.c_int), ("scale", ctypes.c_float)]

    _gpu = None

    @classmethod
    def of(cls, experts, topk, scoring="softmax", bias=None, groups=1, topk_groups=1, group_score="max", renormalise=True, scale=1.0):
        """scoring: "softmax" or "sigmoid"; group_score: "max" or "sum2"; bias: fp32 [experts], kept alive."""
        _fp32_vector(bias, experts, "bias")
        r = cls(_ptr(bias), experts, topk, {"softmax": 0, "sigmoid": 1}[scoring], groups, topk_groups, {"max": 0, "sum2": 1}[group_score], int(bool(renormalise)), float(scale))
        r._tensors = (bias,)
        r._gpu = _gpu_of(r._tensors, "Router")
        return r


def _on_gpu(cache):
    """The cache, unless KVCache.of made it of tensors in host memory: a launch would follow their pointers."""
    if getattr(cache, "_host", False):
        raise ValueError("the KV cache's tensors are not on a GPU")
    return cache


DTYPES = {"fp32": 0, "fp16": 1, "bf16": 2}          # W4A8_F32, W4A8_F16, W4A8_BF16: rows of the attention operators

_P, _I, _Z, _L = ctypes.c_void_p, ctypes.c_int, ctypes.c_size_t, ctypes.c_int64
_SIGNATURES = {
    "w4a8_version": (_I, []),
    "w4a8_last_error": (ctypes.c_char_p, []),
    "w4a8_device_status": (_I, [ctypes.POINTER(ctypes.c_uint32)]),
    "w4a8_config": (_I, [ctypes.c_char_p, _I]),
    "w4a8_quantize_x_q8": (_I, [_P, _P, _P, _P, _I, _I, _P]),
    "w4a8_rmsnorm_quantize_x_q8": (_I, [_P, _P, ctypes.c_float, _I, _P, _P, _P, _P, _I, _I, _P]),
    "w4a8_glu_quantize_x_q8": (_I, [_P, _P, _I, _P, _P, _P, _P, _I, _I, _P]),
    "w4a8_gemv": (_I, [_P, _P, _P, _P, _P, _I, _I, _I, _I, _P]),
    "w4a8_gemv_multi": (_I, [_P, _P, _I, _P, _P, _P, _P, _I, _I, _I, _P]),
    "w4a8_gemm": (_I, [_P, _P, _P, _P, _P, _I, _I, _I, _I, _P]),
    "w4a8_gemm_splitk_workspace_bytes": (_Z, [_I, _I, _I, _I]),
    "w4a8_gemm_splitk": (_I, [_P, _P, _P, _P, _P, _I, _I, _I, _I, _I, _P, _Z, _P]),
    "w4a8_gemm_splitk_static": (_I, [_P, _P, _P, _P, _P, _I, _I, _I, _I, _I, _P]),
    "w4a8_group_dots": (_I, [_P, _P, _P, _I, _I, _I, _I, _P]),
    "w4a8_linear": (_I, [_P, _P, _P, _P, _P, _P, _P, _I, _I, _I, _I, _I, _P]),
    "w4a8_linear_host": (_I, [_P, _P, _P, _P, _P, _P, _P, _P, _P, _I, _I, _I, _I, _P]),
    "w4a8_moe_gemv": (_I, [_P, _P, _P, _P, _P, _P, _I, _I, _I, _I, _I, _I, _I, _P]),
    "w4a8_moe_layout_for": (_I, [_I, _I, _I, _I, _I, ctypes.POINTER(MoeLayout)]),
    "w4a8_moe_block": (_I, [_P, _P, _P, _P, _P, _P, _P, _P, _I, _I, _I, _I, _I, _I, _I, _P, _Z, _P]),
    "w4a8_moe_block_shard": (_I, [_P, _P, _P, _P, _P, _P, _P, _P, _I, _I, _I, _I, _I, _I, _I, _I, _P, _Z, _P, _Z, ctypes.c_uint32, _I, _I, _P]),
    "w4a8_kv_plan": (_I, [_P, _P, _I, _I, _P, _I, _P, _I, _P, _P, _P, _P, _P, _I, _P, _P]),
    "w4a8_kv_append_q8": (_I, [_P, _P, _L, _P, _I, ctypes.POINTER(KVCache), _I, _P]),
    "w4a8_kv_read_q8": (_I, [ctypes.POINTER(KVCache), _P, _I, _P, _P, _I, _I, _P, _P, _L, _I, _P]),
    "w4a8_attention_q8_workspace_bytes": (_Z, [ctypes.POINTER(KVCache), _I, _I, _I]),
    "w4a8_attention_q8": (_I, [_P, _L, ctypes.POINTER(KVCache), _P, _I, _P, _P, _I, _I, _I, _P, _L, _P, ctypes.c_float, _I, _I, ctypes.c_float, _I, _I,
                               _P, _Z, _P]),
    "w4a8_add_norm": (_I, [ctypes.POINTER(Norm), _P, _L, _P, _L, _P, _L, _P, _L, _P, _P, _P, _I, _I, _P]),
    "w4a8_rope_table": (_I, [_I, ctypes.c_double, _I, ctypes.c_double, ctypes.c_double, ctypes.c_double, ctypes.c_double, _P, _P, ctypes.POINTER(ctypes.c_float)]),
    "w4a8_rope_qk": (_I, [ctypes.POINTER(Rope), _P, _L, _I, _P, _L, _I, _P, _I, _P, _L, _P, _L, _I, _P]),
    "w4a8_moe_route": (_I, [ctypes.POINTER(Router), _P, _L, _I, _I, _P, _P, _P]),
    "w4a8_quantize_rows_q8": (_I, [_P, _L, _I, _I, _I, _P, _P, _P]),
    "w4a8_gemm_w8a8": (_I, [_P, _P, _P, _P, _P, _P, _L, _I, _I, _I, _I, _P]),
    "w4a8_linear_w8a8": (_I, [_P, _L, _P, _P, _P, _P, _P, _P, _L, _I, _I, _I, _I, _I, _I, _P]),
    "w4a8_shard_rows": (_I, [_L, _I, _I, ctypes.POINTER(_L), ctypes.POINTER(_L)]),
    "w4a8_load_qmat_shard": (_I, [ctypes.c_char_p, ctypes.c_char_p, _L, _L, _I, _I, _I, ctypes.POINTER(QMat)]),
    "w4a8_upload_qmat_shard": (_I, [_P, _P, _L, _L, _I, _I, _I, ctypes.POINTER(QMat)]),
    "w4a8_free_qmat": (_I, [ctypes.POINTER(QMat)]),
    "w4a8_arena_create": (_I, [_Z, _I, _I, ctypes.POINTER(_P)]),
    "w4a8_arena_base": (_P, [_P]),
    "w4a8_arena_connect": (_I, [_P, ctypes.POINTER(_P)]),
    "w4a8_arena_destroy": (_I, [_P]),
    "w4a8_ipc_export": (_I, [_P, ctypes.c_char_p]),
    "w4a8_ipc_open": (_I, [ctypes.c_char_p, ctypes.POINTER(_P)]),
    "w4a8_ipc_close": (_I, [_P]),
    "w4a8_gemv_allgather": (_I, [_P, _P, _P, _P, _P, _Z, _I, _I, _I, _I, _I, _I, ctypes.c_uint32, _P]),
    "w4a8_gemm_allgather": (_I, [_P, _P, _P, _P, _P, _Z, _I, _I, _I, _I, _I, _I, ctypes.c_uint32, _P]),
    "w4a8_allgather_wait": (_I, [_P, ctypes.c_uint32, _I, _P]),
    "w4a8_gemv_allgather_sync": (_I, [_P, _P, _P, _P, _P, _Z, _I, _I, _I, _I, _I, _I, ctypes.c_uint32, _I, _P]),
    "w4a8_gemm_allgather_sync": (_I, [_P, _P, _P, _P, _P, _Z, _I, _I, _I, _I, _I, _I, ctypes.c_uint32, _I, _P]),
    "w4a8_arena_advance_epoch": (_I, [_P, ctypes.c_uint32, _P]),
}
EXPORTS = tuple(_SIGNATURES)


def lib():
    """Loads the C-ABI library (once).  Raises if it has not been built: there is no fallback."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError("%s not built; run python dgx-serving_b200/build.py (needs nvcc). "
                               "This library has no CPU or PyTorch fallback." % LIB_PATH)
        l = ctypes.CDLL(LIB_PATH)
        for name, (res, args) in _SIGNATURES.items():
            fn = getattr(l, name)
            fn.restype, fn.argtypes = res, args
        _lib = l
    return _lib


_native = None
_NATIVE_ENTRIES = ("add_norm", "rope_qk", "moe_route", "quantize_rows_q8", "gemm_w8a8", "linear_w8a8")


def _binding():
    """csrc/binding.c: the layer operators' entries without ctypes, whose conversions take longer than their smallest kernels."""
    global _native
    if _native is None:
        path = os.path.join(_HERE, "_binding.so")
        if not os.path.exists(path):
            raise RuntimeError("%s not built; run python dgx-serving_b200/build.py" % path)
        loader = importlib.machinery.ExtensionFileLoader("_binding", path)
        module = importlib.util.module_from_spec(importlib.util.spec_from_loader("_binding", loader))
        loader.exec_module(module)
        module.bind(*[ctypes.cast(getattr(lib(), "w4a8_" + n), ctypes.c_void_p).value for n in _NATIVE_ENTRIES])
        import torch
        device, raw = getattr(torch._C, "_cuda_getDevice", None), getattr(torch._C, "_cuda_getCurrentRawStream", None)
        if device is None or raw is None:
            device, raw = torch.cuda.current_device, lambda d: torch.cuda.current_stream(d).cuda_stream
        there = torch.cuda.is_available()
        if there:
            torch.cuda.init()                                         # the two functions above expect it
        module.streams(device, raw, torch.cuda.device_count() if there else 0, torch.Tensor)
        _native = module
    return _native


def _check(rc):
    if rc != OK:
        raise W4A8Error(rc, lib().w4a8_last_error().decode())


def _ptr(t):
    if t is None or isinstance(t, int):
        return t
    return t.data_ptr()


_raw_stream = None


def _stream(stream):
    if stream is None:
        # the handle of torch's current stream of the current device.  torch.cuda.current_stream() builds a Stream object
        # around it on every call, a good part of what a one-row launch costs on the host.
        global _raw_stream
        if _raw_stream is None:
            import torch
            handle = torch.cuda.current_stream().cuda_stream          # initialises CUDA
            device, raw = getattr(torch._C, "_cuda_getDevice", None), getattr(torch._C, "_cuda_getCurrentRawStream", None)
            if device is None or raw is None:
                _raw_stream = lambda: torch.cuda.current_stream().cuda_stream
            else:
                _raw_stream = lambda: raw(device())
            return handle
        return _raw_stream()
    if isinstance(stream, int):
        return stream
    return stream.cuda_stream


def config(key, value):
    """Run-time policy switch, e.g. config("gemv_kernel", 2): tensor-path GEMV for every S (see include/w4a8_b200.h)."""
    _check(lib().w4a8_config(key.encode(), int(value)))


def device_status():
    """Synchronises and raises if a kernel recorded a device-side error (a bounded wait ran out)."""
    d = ctypes.c_uint32(0)
    _check(lib().w4a8_device_status(ctypes.byref(d)))


def launch_quantize_x_q8(X, xq, xs, xsum, IN, S, stream=None):
    _check(lib().w4a8_quantize_x_q8(_ptr(X), _ptr(xq), _ptr(xs), _ptr(xsum), IN, S, _stream(stream)))


def launch_rmsnorm_quantize_x_q8(X, W, eps, variant, Y, xq, xs, xsum, IN, S, stream=None):
    """RMSNorm (variant 0: * W, 1: * (1 + W), 2: no scale) and quantize_x in one kernel; Y (may be None) also gets the
    fp32 intermediate.  Same bits as the reference's launch_rmsnorm* followed by launch_quantize_x_q8."""
    _check(lib().w4a8_rmsnorm_quantize_x_q8(_ptr(X), _ptr(W), float(eps), variant, _ptr(Y), _ptr(xq), _ptr(xs), _ptr(xsum), IN, S,
                                            _stream(stream)))


def launch_glu_quantize_x_q8(G, U, act, Y, xq, xs, xsum, IN, S, stream=None):
    """SwiGLU (act 0) or GeGLU (act 1) of (G, U) and quantize_x in one kernel; Y (may be None) also gets the fp32 product."""
    _check(lib().w4a8_glu_quantize_x_q8(_ptr(G), _ptr(U), act, _ptr(Y), _ptr(xq), _ptr(xs), _ptr(xsum), IN, S, _stream(stream)))


def gemv_multi(xq, xs, Wqs, sws, Ys, OUTs, IN, S, scale_dtype=0, stream=None):
    """Several matrices (at most 4) against the same activation rows in one call; one launch for a single row on the
    bulk-copy kernel and for 2 to 16 rows on the tensor-path kernel.  Each Ys[i] equals launch_gemv_w4a8 of matrix i."""
    n = len(Wqs)
    arr = lambda xs_: (ctypes.c_void_p * n)(*[_ptr(t) for t in xs_])
    outs = (ctypes.c_int * n)(*[int(o) for o in OUTs])
    _check(lib().w4a8_gemv_multi(_ptr(xq), _ptr(xs), n, arr(Wqs), arr(sws), arr(Ys), outs, IN, S, scale_dtype, _stream(stream)))


def launch_gemv_w4a8(xq, xs, xsum, Wq, sw, Y, IN, OUT, S, scale_dtype=0, stream=None):
    """xsum is accepted and ignored, as in the reference (kernels/gemv_w4a8.cuh:23-25)."""
    _check(lib().w4a8_gemv(_ptr(xq), _ptr(xs), _ptr(Wq), _ptr(sw), _ptr(Y), IN, OUT, S, scale_dtype, _stream(stream)))


def launch_gemv_w4a8_sb(xq, xs, Wq, sw, Y, IN, OUT, S, scale_dtype=0, stream=None):
    _check(lib().w4a8_gemv(_ptr(xq), _ptr(xs), _ptr(Wq), _ptr(sw), _ptr(Y), IN, OUT, S, scale_dtype, _stream(stream)))


launch_gemv_w4a8_mlp = launch_gemv_w4a8_mlp_auto = launch_gemv_w4a8_g4 = launch_gemv_w4a8
launch_gemv_w4a8_sb_g4 = launch_gemv_w4a8_sb


def launch_gemm_batch_w4a8(xq, xs, Wq, sw, Y, IN, OUT, B, scale_dtype=0, stream=None):
    _check(lib().w4a8_gemv(_ptr(xq), _ptr(xs), _ptr(Wq), _ptr(sw), _ptr(Y), IN, OUT, B, scale_dtype, _stream(stream)))


def launch_gemm_mmq_w4a8(X, xs, Wq, sw, Y, M, N, K, scale_dtype=0, stream=None):
    _check(lib().w4a8_gemm(_ptr(X), _ptr(xs), _ptr(Wq), _ptr(sw), _ptr(Y), M, N, K, scale_dtype, _stream(stream)))


launch_gemm_mmq_w4a8_auto = launch_gemm_mma_w4a8 = launch_gemm_mmq_w4a8


def launch_gemm_mmq_raster_w4a8(X, xs, Wq, sw, Y, M, N, K, scale_dtype, raster, group, stream=None):
    """raster/group only re-order tiles in the reference (kernels/gemm_mmq_raster.cuh:16-27); results are equal."""
    launch_gemm_mmq_w4a8(X, xs, Wq, sw, Y, M, N, K, scale_dtype, stream)


def gemm_splitk_workspace_bytes(M, N, K, splitk=0):
    return int(lib().w4a8_gemm_splitk_workspace_bytes(M, N, K, splitk))


def launch_gemm_bm16_splitk(X, xs, Wq, sw, Y, M, N, K, scale_dtype=0, splitk=0, workspace=None, stream=None):
    nbytes = 0 if workspace is None else workspace.numel() * workspace.element_size()
    _check(lib().w4a8_gemm_splitk(_ptr(X), _ptr(xs), _ptr(Wq), _ptr(sw), _ptr(Y), M, N, K, scale_dtype, splitk,
                                  _ptr(workspace), nbytes, _stream(stream)))


SPLITK_STATIC_BYTES = 16 * 1024 * 1024


def launch_gemm_splitk_static(X, xs, Wq, sw, Y, M, N, K, scale_dtype=0, splitk=0, stream=None):
    """Split-K GEMM whose partial sums live in a buffer built into the library: no workspace, no allocation.
    For callers that cannot allocate at the point of the call; at most SPLITK_STATIC_BYTES of partial sums."""
    _check(lib().w4a8_gemm_splitk_static(_ptr(X), _ptr(xs), _ptr(Wq), _ptr(sw), _ptr(Y), M, N, K, scale_dtype, splitk,
                                         _stream(stream)))


def group_dots(xq, Wq, D, M, N, K, path=0, stream=None):
    _check(lib().w4a8_group_dots(_ptr(xq), _ptr(Wq), _ptr(D), M, N, K, path, _stream(stream)))


def linear(X, xq, xs, xsum, Wq, sw, Y, S, N, K, scale_dtype=0, skip_quantize=0, stream=None):
    """The mm() dispatcher of the model graphs (models/qwen35_decode.cu:51-62)."""
    _check(lib().w4a8_linear(_ptr(X), _ptr(xq), _ptr(xs), _ptr(xsum), _ptr(Wq), _ptr(sw), _ptr(Y), S, N, K,
                             scale_dtype, skip_quantize, _stream(stream)))


def linear_host(X_host, Y_host, X_dev, xq, xs, xsum, Y_dev, Wq, sw, S, N, K, scale_dtype=0, stream=None):
    """mm() with host activations in and host results out (pinned torch tensors or raw host pointers); synchronous."""
    _check(lib().w4a8_linear_host(_ptr(X_host), _ptr(Y_host), _ptr(X_dev), _ptr(xq), _ptr(xs), _ptr(xsum), _ptr(Y_dev), _ptr(Wq),
                                  _ptr(sw), S, N, K, scale_dtype, _stream(stream)))


def moe_gemv(xq, xs, Wq, sw, idx, Y, nslots, topk, x_per_slot, N, K, num_experts, scale_dtype=0, stream=None):
    _check(lib().w4a8_moe_gemv(_ptr(xq), _ptr(xs), _ptr(Wq), _ptr(sw), _ptr(idx), _ptr(Y), nslots, topk, x_per_slot,
                               N, K, num_experts, scale_dtype, _stream(stream)))


def moe_layout_for(S, topk, H, MI, experts):
    l = MoeLayout()
    _check(lib().w4a8_moe_layout_for(S, topk, H, MI, experts, ctypes.byref(l)))
    return l


def moe_block(n2, gu_wq, gu_sc, dn_wq, dn_sc, idx, dw, out, S, topk, H, MI, num_experts, workspace, scale_dtype=0, act=0, stream=None):
    """The routed-expert block of models/moe_block.cuh:45-52 in W4A8 (w4a8_moe_block); workspace = a uint8 device tensor
    of moe_layout_for(...).bytes bytes."""
    _check(lib().w4a8_moe_block(_ptr(n2), _ptr(gu_wq), _ptr(gu_sc), _ptr(dn_wq), _ptr(dn_sc), _ptr(idx), _ptr(dw), _ptr(out), S, topk, H, MI,
                                num_experts, scale_dtype, act, _ptr(workspace), workspace.numel() * workspace.element_size(), _stream(stream)))


def moe_block_shard(n2, gu_wq, gu_sc, dn_wq, dn_sc, idx, dw, out, S, topk, H, MI, expert_base, experts_local, workspace, arena, sout_offset,
                    epoch, scale_dtype=0, act=0, timeout_us=1000000, phase=0, stream=None):
    """Expert-sharded routed-expert block (w4a8_moe_block_shard): this rank's experts only, down outputs exchanged through the arenas."""
    _check(lib().w4a8_moe_block_shard(_ptr(n2), _ptr(gu_wq), _ptr(gu_sc), _ptr(dn_wq), _ptr(dn_sc), _ptr(idx), _ptr(dw), _ptr(out), S, topk, H, MI,
                                      expert_base, experts_local, scale_dtype, act, _ptr(workspace),
                                      workspace.numel() * workspace.element_size(), arena.handle, sout_offset, epoch, timeout_us, phase, _stream(stream)))


def kv_plan(kv_len, new_len, R, block, block_table, table_width, free_blocks, num_free, first_free, seq_len, cu_new, slot, position, T, status, stream=None):
    """Block tables and slot maps of a step from the requests' lengths, on the GPU (w4a8_kv_plan); position may be None."""
    _check(lib().w4a8_kv_plan(_ptr(kv_len), _ptr(new_len), R, block, _ptr(block_table), table_width, _ptr(free_blocks), num_free, _ptr(first_free),
                              _ptr(seq_len), _ptr(cu_new), _ptr(slot), _ptr(position), T, _ptr(status), _stream(stream)))


def launch_kv_append_q8(K, V, ld, slot, T, cache, dtype="fp32", stream=None):
    """Rows K, V [T][heads * dim] (pitch ld elements) into their slots of the 8-bit cache (w4a8_kv_append_q8)."""
    _check(lib().w4a8_kv_append_q8(_ptr(K), _ptr(V), ld, _ptr(slot), T, _on_gpu(cache), DTYPES.get(dtype, dtype), _stream(stream)))


def launch_kv_read_q8(cache, block_table, table_width, begin, cu, R, T, K, V, ld, dtype="fp32", stream=None):
    """The numbers that the cache holds for tokens begin[r] + i of each request, to rows cu[r] + i of K and V (w4a8_kv_read_q8)."""
    _check(lib().w4a8_kv_read_q8(_on_gpu(cache), _ptr(block_table), table_width, _ptr(begin), _ptr(cu), R, T, _ptr(K), _ptr(V), ld, DTYPES.get(dtype, dtype),
                                 _stream(stream)))


def attention_q8_workspace_bytes(heads_q, cache, T=0, max_q=0):
    return int(lib().w4a8_attention_q8_workspace_bytes(cache, heads_q, T, max_q))


def launch_attention_q8(Q, ldq, cache, block_table, table_width, cu_q, seq_len, R, T, heads_q, O, ldo, scale, dtype, workspace, causal=1, window=0,
                        softcap=0.0, max_q=0, lse=None, stream=None):
    """Attention of the rows Q[T][heads_q * dim], the last tokens of R requests, over the 8-bit cache (w4a8_attention_q8).  workspace: a device
    tensor of attention_q8_workspace_bytes(...) bytes, zeroed once."""
    _check(lib().w4a8_attention_q8(_ptr(Q), ldq, _on_gpu(cache), _ptr(block_table), table_width, _ptr(cu_q), _ptr(seq_len), R, T, heads_q, _ptr(O), ldo, _ptr(lse),
                                   scale, causal, window, softcap, max_q, DTYPES.get(dtype, dtype), _ptr(workspace),
                                   workspace.numel() * workspace.element_size(), _stream(stream)))


# What the launches refuse of their parameters alone: calls without rows, which launch nothing and follow no pointer.
def check_norm(norm):
    _check(lib().w4a8_add_norm(norm, None, 0, None, 0, None, 0, None, 0, None, None, None, 32, 0, None))


def check_rope(rope, heads_q, heads_k):
    _check(lib().w4a8_rope_qk(rope, None, 0, heads_q, None, 0, heads_k, None, 0, None, 0, None, 0, 0, None))


def check_router(router):
    _check(lib().w4a8_moe_route(router, None, router.experts, 0, 0, None, None, None))


def check_moe(topk, H, MI, num_experts, scale_dtype, act):
    _check(lib().w4a8_moe_block(None, None, None, None, None, None, None, None, 0, topk, H, MI, num_experts, scale_dtype, act, None, 0, None))


def check_attention(cache, heads_q, scale, window, softcap):
    _check(lib().w4a8_attention_q8(None, 0, cache, None, 0, None, None, 0, 0, heads_q, None, 0, None, scale, 1, window, softcap, 0, 0, None, 0, None))


def launch_add_norm(norm, H, Y, S, H_out=None, N=None, xq=None, xs=None, xsum=None, group=32, ldh=0, ldy=0, ldo=0, ldn=0, stream=None):
    """h' = h + norm(y) * gate * alpha of S rows, to H_out, and its norm n, to N and / or quantized to xq, xs, xsum (w4a8_add_norm).  Y None: h' = h.
    group 32: blocks of 32 elements, 0: one scale for a row.  Pitches of 0: K."""
    K = norm.K
    if S > norm._gate_rows:
        raise ValueError("%d rows, a gate of %d" % (S, norm._gate_rows))
    rc = (_native or _binding()).add_norm(norm, H, ldh or K, Y, ldy or K, H_out, ldo or K, N, ldn or K, xq, xs, xsum, group, S, stream)
    if rc:
        _check(rc)


def launch_rope_qk(rope, Q, ldq, heads_q, K, ldk, heads_k, position, T, Q_out=None, ldqo=0, K_out=None, ldko=0, dtype="fp32", stream=None):
    """Norms and rotary positions of queries Q[T][heads_q * dim] and keys K[T][heads_k * dim] (w4a8_rope_qk); outputs None: in place."""
    if rope._host:
        raise ValueError("the rope's table is not on a GPU")
    if Q_out is None:
        Q_out, ldqo = Q, ldq
    if K_out is None:
        K_out, ldko = K, ldk
    rc = (_native or _binding()).rope_qk(rope, Q, ldq, heads_q, K, ldk, heads_k, position, T, Q_out, ldqo, K_out, ldko, DTYPES.get(dtype, dtype), stream)
    if rc:
        _check(rc)


def launch_moe_route(router, logits, ld, S, idx, weight, dtype="fp32", stream=None):
    """The experts idx[S][topk] of S tokens and their weights, from logits[S][experts] (w4a8_moe_route): what moe_block takes."""
    rc = (_native or _binding()).moe_route(router, logits, ld, S, DTYPES.get(dtype, dtype), idx, weight, stream)
    if rc:
        _check(rc)


def launch_quantize_rows_q8(X, ldx, S, K, xq, xs, dtype="fp32", stream=None):
    """Rows to int8 with one scale each (w4a8_quantize_rows_q8): activations of the 8-bit products, or their weights, a channel per row."""
    rc = (_native or _binding()).quantize_rows_q8(X, ldx, S, K, DTYPES.get(dtype, dtype), xq, xs, stream)
    if rc:
        _check(rc)


def launch_gemm_w8a8(xq, xs, wq, ws, Y, ldy, M, N, K, dtype="fp32", bias=None, stream=None):
    """Y[M][N] = xq wq^T * xs[m] * ws[n] + bias[n], the sums exact (w4a8_gemm_w8a8)."""
    rc = (_native or _binding()).gemm_w8a8(xq, xs, wq, ws, bias, Y, ldy, M, N, K, DTYPES.get(dtype, dtype), stream)
    if rc:
        _check(rc)


def linear_w8a8(X, ldx, xq, xs, wq, ws, Y, ldy, S, N, K, x_dtype="fp32", y_dtype="fp32", bias=None, skip_quantize=0, stream=None):
    """linear() for 8-bit weights with a scale for each output channel (w4a8_linear_w8a8)."""
    rc = (_native or _binding()).linear_w8a8(X, ldx, xq, xs, wq, ws, bias, Y, ldy, S, N, K, DTYPES.get(x_dtype, x_dtype), DTYPES.get(y_dtype, y_dtype), skip_quantize, stream)
    if rc:
        _check(rc)


def shard_rows(N, rank, world):
    r0, rows = _L(0), _L(0)
    _check(lib().w4a8_shard_rows(N, rank, world, ctypes.byref(r0), ctypes.byref(rows)))
    return r0.value, rows.value


def load_qmat_shard(q4_path, scale_path, N, K, scale_dtype, rank, world):
    m = QMat()
    _check(lib().w4a8_load_qmat_shard(os.fsencode(q4_path), os.fsencode(scale_path), N, K, scale_dtype, rank, world,
                                      ctypes.byref(m)))
    return m


def upload_qmat_shard(host_wq, host_sc, N, K, scale_dtype, rank, world):
    """host_wq / host_sc: numpy arrays (or anything with .ctypes) holding the full [N] tensors."""
    m = QMat()
    _check(lib().w4a8_upload_qmat_shard(host_wq.ctypes.data, host_sc.ctypes.data, N, K, scale_dtype, rank, world,
                                        ctypes.byref(m)))
    return m


def free_qmat(m):
    _check(lib().w4a8_free_qmat(ctypes.byref(m)))


class Arena:
    """Peer-visible device memory for the fused GEMV + all-gather (w4a8_arena in include/w4a8_b200.h)."""

    def __init__(self, nbytes, rank, world):
        h = _P()
        _check(lib().w4a8_arena_create(nbytes, rank, world, ctypes.byref(h)))
        self.handle, self.rank, self.world, self.nbytes = h, rank, world, nbytes
        self.base = lib().w4a8_arena_base(h)
        self._opened = []

    def export_handle(self):
        buf = ctypes.create_string_buffer(64)
        _check(lib().w4a8_ipc_export(self.base, buf))
        return buf.raw

    def connect_handles(self, handles):
        """handles[r] = 64-byte CUDA IPC handle of rank r's arena (this rank's own entry is ignored)."""
        bases = (_P * self.world)()
        for r, hd in enumerate(handles):
            if r == self.rank:
                bases[r] = self.base
            else:
                p = _P()
                _check(lib().w4a8_ipc_open(hd, ctypes.byref(p)))
                self._opened.append(p)
                bases[r] = p.value
        _check(lib().w4a8_arena_connect(self.handle, bases))

    def connect_pointers(self, pointers):
        """pointers[r] = arena base of rank r already mapped into this process (same-process emulation, or another
        peer-mapping mechanism)."""
        bases = (_P * self.world)(*[int(p) for p in pointers])
        _check(lib().w4a8_arena_connect(self.handle, bases))

    def tensor(self, offset, shape, dtype=None):
        """A torch view of the local arena (no copy)."""
        import torch
        dtype = dtype or torch.float32
        return _as_tensor(self.base + offset, shape, dtype)

    def gemv_allgather(self, xq, xs, Wq, sw, y_offset, IN, rows, row0, ldY, S, scale_dtype, epoch, stream=None):
        _check(lib().w4a8_gemv_allgather(_ptr(xq), _ptr(xs), _ptr(Wq), _ptr(sw), self.handle, y_offset, IN, rows, row0, ldY, S,
                                         scale_dtype, epoch, _stream(stream)))

    def gemm_allgather(self, X, xs, Wq, sw, y_offset, M, rows, row0, ldY, K, scale_dtype, epoch, stream=None):
        _check(lib().w4a8_gemm_allgather(_ptr(X), _ptr(xs), _ptr(Wq), _ptr(sw), self.handle, y_offset, M, rows, row0, ldY, K,
                                         scale_dtype, epoch, _stream(stream)))

    def gemv_allgather_sync(self, xq, xs, Wq, sw, y_offset, IN, rows, row0, ldY, S, scale_dtype, epoch, timeout_us=1000000, stream=None):
        """gemv_allgather with the wait folded into its last kernel: when that kernel completes, Y is complete here."""
        _check(lib().w4a8_gemv_allgather_sync(_ptr(xq), _ptr(xs), _ptr(Wq), _ptr(sw), self.handle, y_offset, IN, rows, row0, ldY, S,
                                              scale_dtype, epoch, timeout_us, _stream(stream)))

    def gemm_allgather_sync(self, X, xs, Wq, sw, y_offset, M, rows, row0, ldY, K, scale_dtype, epoch, timeout_us=1000000, stream=None):
        _check(lib().w4a8_gemm_allgather_sync(_ptr(X), _ptr(xs), _ptr(Wq), _ptr(sw), self.handle, y_offset, M, rows, row0, ldY, K,
                                              scale_dtype, epoch, timeout_us, _stream(stream)))

    def wait(self, epoch, timeout_us=1000000, stream=None):
        _check(lib().w4a8_allgather_wait(self.handle, epoch, timeout_us, _stream(stream)))

    def advance_epoch(self, delta, stream=None):
        _check(lib().w4a8_arena_advance_epoch(self.handle, delta, _stream(stream)))

    def close(self):
        for p in self._opened:
            lib().w4a8_ipc_close(p)
        self._opened = []
        if self.handle:
            lib().w4a8_arena_destroy(self.handle)
            self.handle = None


def _as_tensor(ptr, shape, dtype):
    """Wraps raw device memory as a torch tensor through the CUDA array interface (no copy, no ownership)."""
    import torch
    typestr = {torch.float32: "<f4", torch.int32: "<i4", torch.uint8: "|u1", torch.int8: "|i1"}[dtype]

    class _Holder:
        pass
    h = _Holder()
    h.__cuda_array_interface__ = {"shape": tuple(shape), "typestr": typestr, "data": (int(ptr), False), "version": 3, "strides": None}
    return torch.as_tensor(h, device="cuda")
