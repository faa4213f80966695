"""ctypes binding of liboxinfer_hip.so and `HipBackend`, the mirror of `trait Backend`
(src/gpu.rs:151-294 of the reference): name / wants / upload / matmul / stats with the reference's
conventions (False / None = declined, nothing written), plus the device-pointer entry points.

Device buffers are torch tensors (torch is plumbing for memory and streams only).
"""
import ctypes as C
import math
import os

import numpy as np

_HERE = os.path.dirname(os.path.abspath(__file__))
_SO = os.path.join(_HERE, "liboxinfer_hip.so")

W_BF16, W_Q8, W_Q4, W_GGUF, W_MLX_Q4 = 0, 1, 2, 3, 4
GGML_Q4_0, GGML_Q8_0, GGML_Q4_K, GGML_Q5_K, GGML_Q6_K, GGML_MXFP4, GGML_NVFP4, GGML_F8E4M3 = 2, 8, 12, 13, 14, 39, 40, 0x1000
GGML_BLOCK = {GGML_Q4_0: (32, 18), GGML_Q8_0: (32, 34), GGML_Q4_K: (256, 144), GGML_Q5_K: (256, 176), GGML_Q6_K: (256, 210), GGML_MXFP4: (32, 17), GGML_NVFP4: (64, 36)}


class WeightDesc(C.Structure):
    _fields_ = [("kind", C.c_uint32), ("ggml_type", C.c_uint32), ("n_out", C.c_size_t), ("n_in", C.c_size_t),
                ("data", C.c_void_p), ("scales", C.c_void_p), ("offsets", C.c_void_p), ("group", C.c_uint32),
                ("block_scales", C.c_void_p), ("bs_rows", C.c_uint32), ("bs_cols", C.c_uint32)]


class Job(C.Structure):
    _fields_ = [("w", C.c_void_p), ("n_out", C.c_size_t), ("y", C.c_void_p)]


class DecodeJob(C.Structure):
    _fields_ = [("w", C.c_void_p), ("xa", C.c_void_p), ("x", C.c_void_p), ("t", C.c_size_t), ("y", C.c_void_p),
                ("ev_start", C.c_void_p), ("ev_stop", C.c_void_p)]


class GpuInfo(C.Structure):
    _fields_ = [("index", C.c_int), ("name", C.c_char * 256), ("arch", C.c_char * 64), ("memory_bytes", C.c_uint64),
                ("driver", C.c_char * 64), ("usable", C.c_int)]


class QuantJob(C.Structure):
    _fields_ = [("x", C.c_void_p), ("t", C.c_size_t), ("n_in", C.c_size_t), ("out", C.c_void_p)]


class RowsJob(C.Structure):
    _fields_ = [("w", C.c_void_p), ("up", C.c_void_p), ("n_out", C.c_size_t), ("y", C.c_void_p)]


class QActC(C.Structure):
    _fields_ = [("q", C.c_void_p), ("scales", C.c_void_p), ("sums", C.c_void_p), ("fsums", C.c_void_p),
                ("hsums", C.c_void_p), ("sums16", C.c_void_p), ("t", C.c_size_t), ("n_in", C.c_size_t)]


class KvCacheC(C.Structure):
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("k_scale", C.c_void_p), ("v_scale", C.c_void_p), ("n_pages", C.c_size_t),
                ("page_tokens", C.c_size_t), ("n_kv", C.c_size_t), ("d", C.c_size_t)]


class KvBatchC(C.Structure):
    _fields_ = [("n_seqs", C.c_size_t), ("rows", C.c_size_t), ("row_start", C.c_void_p), ("kv_len", C.c_void_p), ("pages", C.c_void_p),
                ("max_pages", C.c_size_t)]


class RopeC(C.Structure):
    _fields_ = [("table", C.c_void_p), ("n_pos", C.c_size_t), ("n_rot", C.c_size_t), ("interleaved", C.c_int)]


class AttendRulesC(C.Structure):
    _fields_ = [("cap", C.c_float), ("slopes", C.c_void_p), ("window", C.c_size_t), ("prefix", C.c_void_p), ("first", C.c_void_p)]


class LogitRulesC(C.Structure):
    _fields_ = [("history", C.c_void_p), ("history_stride", C.c_size_t), ("history_len", C.c_void_p), ("prompt_len", C.c_void_p),
                ("repetition", C.c_void_p), ("presence", C.c_void_p), ("frequency", C.c_void_p), ("bias_start", C.c_void_p),
                ("bias_id", C.c_void_p), ("bias", C.c_void_p), ("n_bias", C.c_size_t), ("allowed", C.c_void_p), ("n_allowed", C.c_size_t),
                ("allowed_stride", C.c_size_t), ("allowed_row", C.c_void_p)]


_lib = None
_torch = None


def library_path():
    return _SO


def load_library():
    """Loads liboxinfer_hip.so (built in-tree by `python -m oxinfer_amd.build`). Raises if it is missing."""
    global _lib, _torch
    if _lib is not None:
        return _lib
    if not os.path.exists(_SO):
        raise RuntimeError(f"{_SO} is not built: run `python -m oxinfer_amd.build` (hipcc, gfx950). "
                           "There is no CPU fallback in this package.")
    try:
        import torch as _torch  # (its bundled HIP runtime must be the one this process uses)
    except ImportError:
        pass
    lib = C.CDLL(_SO)
    vp, sz = C.c_void_p, C.c_size_t
    sig = {
        "oxhip_probe": (C.c_int, [C.POINTER(GpuInfo), C.c_int]),
        "oxhip_open": (C.c_int, [C.c_int, C.POINTER(vp)]),
        "oxhip_close": (None, [vp]),
        "oxhip_name": (C.c_char_p, [vp]),
        "oxhip_last_error": (C.c_char_p, []),
        "oxhip_stats": (sz, [vp, C.c_char_p, sz]),
        "oxhip_wants": (C.c_int, [vp, sz, sz, sz]),
        "oxhip_upload": (vp, [vp, C.POINTER(WeightDesc)]),
        "oxhip_free_weight": (None, [vp, vp]),
        "oxhip_weight_bytes": (sz, [vp]),
        "oxhip_matmul": (C.c_int, [vp, vp, sz, sz, C.POINTER(Job), sz]),
        "oxhip_dev_quantize_act": (C.c_int, [vp, vp, sz, sz, C.POINTER(QActC), vp]),
        "oxhip_dev_quantize_act_batch": (C.c_int, [vp, C.POINTER(QuantJob), sz, vp]),
        "oxhip_dev_dequantize": (C.c_int, [vp, vp, sz, sz, vp, vp]),
        "oxhip_dev_decode": (C.c_int, [vp, vp, C.POINTER(QActC), vp, sz, vp, vp]),
        "oxhip_dev_decode_noalloc": (C.c_int, [vp, vp, C.POINTER(QActC), sz, vp, vp]),
        "oxhip_dev_isums": (C.c_int, [vp, vp, C.POINTER(QActC), vp, vp]),
        "oxhip_dev_decode_batch": (C.c_int, [vp, C.POINTER(DecodeJob), sz, vp]),
        "oxhip_dev_gemm": (C.c_int, [vp, vp, vp, C.c_int, sz, vp, C.c_int, C.c_int, vp]),
        "oxhip_dev_gemm_timed": (C.c_int, [vp, vp, vp, C.c_int, sz, vp, C.c_int, C.c_int, vp, vp, vp]),
        "oxhip_dev_gemm_isums": (C.c_int, [vp, vp, vp, C.c_int, sz, vp, vp]),
        "oxhip_matvec_rows": (C.c_int, [vp, vp, sz, sz, C.POINTER(RowsJob), sz]),
        "oxhip_upload_moe": (vp, [vp, C.POINTER(WeightDesc), C.POINTER(WeightDesc), C.POINTER(WeightDesc), sz, sz, sz, C.c_uint32, C.c_float]),
        "oxhip_free_moe": (None, [vp, vp]),
        "oxhip_moe_set_mode": (C.c_int, [vp, C.c_uint32]),
        "oxhip_moe_forward": (C.c_int, [vp, vp, sz, sz, sz, vp, vp, sz, vp, vp]),
        "oxhip_dev_route_top_k": (C.c_int, [vp, vp, sz, sz, sz, vp, vp, vp]),
        "oxhip_dev_moe": (C.c_int, [vp, vp, vp, sz, vp, vp, sz, vp, vp]),
        "oxhip_buf_alloc": (vp, [vp, sz]),
        "oxhip_buf_free": (None, [vp, vp]),
        "oxhip_buf_write": (C.c_int, [vp, vp, vp, sz, vp]),
        "oxhip_buf_read": (C.c_int, [vp, vp, vp, sz, vp]),
        "oxhip_dev_rmsnorm_quantize": (C.c_int, [vp, vp, vp, vp, C.c_float, sz, sz, vp, C.POINTER(QActC), vp]),
        "oxhip_dev_norm": (C.c_int, [vp, vp, vp, vp, vp, C.c_float, sz, sz, sz, sz, C.c_float, C.c_int, C.POINTER(QActC), vp]),
        "oxhip_stream_release": (C.c_int, [vp, vp]),
        "oxhip_dev_linear": (C.c_int, [vp, vp, vp, C.POINTER(QActC), vp, sz, vp, C.c_uint32, vp, vp]),
        "oxhip_dev_glu": (C.c_int, [vp, vp, vp, sz, C.c_int, vp, vp]),
        "oxhip_dev_route": (C.c_int, [vp, vp, vp, vp, sz, sz, sz, sz, vp, vp, vp, vp]),
        "oxhip_dev_experts": (C.c_int, [vp, vp, vp, sz, vp, sz, vp, C.c_int, vp]),
        "oxhip_dev_moe_routed": (C.c_int, [vp, vp, vp, sz, vp, sz, sz, vp, vp, vp, C.c_int, vp]),
        "oxhip_dev_kv_append": (C.c_int, [vp, C.POINTER(KvCacheC), C.POINTER(KvBatchC), vp, sz, vp, sz, vp, sz, vp, sz, sz, C.c_int, C.POINTER(RopeC), vp]),
        "oxhip_dev_kv_read": (C.c_int, [vp, C.POINTER(KvCacheC), C.POINTER(KvBatchC), sz, vp, vp, C.c_int, vp]),
        "oxhip_dev_attend": (C.c_int, [vp, C.POINTER(KvCacheC), C.POINTER(KvBatchC), vp, sz, sz, C.c_int, C.c_float, C.POINTER(AttendRulesC), vp, sz, vp]),
        "oxhip_dev_logits": (C.c_int, [vp, vp, sz, vp, sz, sz, sz, C.c_int, C.POINTER(LogitRulesC), vp, vp]),
        "oxhip_plan_begin": (vp, [vp, vp]),
        "oxhip_plan_end": (C.c_int, [vp]),
        "oxhip_plan_launches": (sz, [vp]),
        "oxhip_plan_one_by_one": (C.c_int, [vp]),
        "oxhip_plan_replay": (C.c_int, [vp, vp]),
        "oxhip_plan_free": (None, [vp]),
        "oxhip_event_create": (vp, []),
        "oxhip_event_destroy": (None, [vp]),
        "oxhip_event_elapsed_ms": (C.c_float, [vp, vp]),
    }
    for name, (res, args) in sig.items():
        fn = getattr(lib, name)
        fn.restype, fn.argtypes = res, args
    _lib = lib
    return lib


def _np_ptr(a):
    return None if a is None else a.ctypes.data_as(C.c_void_p)


def probe():
    """platform::gpu::cuda::probe for HIP devices (src/platform.rs:446-482): a list of dicts like `GpuInfo`."""
    lib = load_library()
    arr = (GpuInfo * 16)()
    n = lib.oxhip_probe(arr, 16)
    return [dict(kind="hip", index=g.index, name=g.name.decode(), arch=g.arch.decode(), memory_bytes=int(g.memory_bytes),
                 driver=g.driver.decode(), usable=bool(g.usable)) for g in arr[:min(n, 16)]]


class DeviceWeight:
    """`gpu::DeviceWeight` of one matrix (src/gpu.rs:57): freed when dropped."""

    def __init__(self, be, handle, n_out, n_in):
        self.be, self.handle, self.n_out, self.n_in = be, handle, n_out, n_in

    @property
    def bytes(self):
        return load_library().oxhip_weight_bytes(self.handle)

    def __del__(self):
        if getattr(self, "handle", None) and self.be.ctx:
            load_library().oxhip_free_weight(self.be.ctx, self.handle)
            self.handle = None


class DeviceMoe:
    """`DeviceWeight` of the routed experts of one MoE layer (Backend::upload_moe, src/gpu.rs:206-216)."""

    def __init__(self, be, handle, n_exp, h, inter):
        self.be, self.handle, self.n_exp, self.h, self.inter = be, handle, n_exp, h, inter

    def set_mode(self, mode):
        """MOE_AUTO: the reference's split by pass size; MOE_INT8: the integer kernels at every size."""
        if not load_library().oxhip_moe_set_mode(self.handle, mode):
            raise RuntimeError(self.be.last_error())

    def __del__(self):
        if getattr(self, "handle", None) and self.be.ctx:
            load_library().oxhip_free_moe(self.be.ctx, self.handle)
            self.handle = None


class Plan:
    """A recorded chain of device-pointer ops (oxhip_plan_*): the matmul side of `DecodePlan` (src/gpu_decode.rs:572-587)."""

    def __init__(self, be, handle):
        self.be, self.handle = be, handle

    @property
    def launches(self):
        return load_library().oxhip_plan_launches(self.handle)

    @property
    def one_by_one(self):
        """Whether replays go out launch by launch (short plans of the library's own kernels), not as one submission."""
        return bool(load_library().oxhip_plan_one_by_one(self.handle))

    def replay(self, stream=None):
        if not load_library().oxhip_plan_replay(self.handle, C.c_void_p(stream) if stream else None):
            raise RuntimeError(self.be.last_error())

    def __del__(self):
        if getattr(self, "handle", None):
            load_library().oxhip_plan_free(self.handle)
            self.handle = None


ACT_SILU, ACT_GELU_TANH, ACT_SILU_CLAMP = 0, 1, 2
MOE_AUTO, MOE_INT8 = 0, 1
LIN_STORE, LIN_ADD, LIN_SILU_PAIR, LIN_GELU_PAIR, LIN_ADD_GATED = 0, 1, 2, 3, 4


class QAct:
    """`quant::QAct` (src/quant.rs:222-238) in device memory (torch tensors)."""

    def __init__(self, t, n_in, device):
        import torch
        self.t, self.n_in = t, n_in
        self.q = torch.empty((t, n_in), dtype=torch.int8, device=device)
        self.scales = torch.empty((t, n_in // 32), dtype=torch.float32, device=device)
        self.sums = torch.empty((t, n_in // 32), dtype=torch.int32, device=device)
        self.fsums = torch.empty((t, n_in // 32), dtype=torch.float32, device=device)
        self.hsums = torch.empty((t, n_in // 16), dtype=torch.float32, device=device)
        self.sums16 = torch.empty((t, n_in // 16), dtype=torch.int32, device=device)
        self.c = QActC(self.q.data_ptr(), self.scales.data_ptr(), self.sums.data_ptr(), self.fsums.data_ptr(),
                       self.hsums.data_ptr(), self.sums16.data_ptr(), t, n_in)


# Checks of the tensors that the library gets by their pointers. They are most of what a call costs the host, so each asks a tensor for little: the
# wrong ones are told apart where they are found wrong.
def _array(name, t, dtype, device=None, count=None):
    """A dense device tensor of `dtype` (with `count` values, if given): its pointer, or None for None."""
    if t is None:
        return None
    on = t.get_device()
    if t.dtype is not dtype or not t.is_contiguous() or on < 0 or (on != device and device is not None) or (count is not None and t.numel() != count):
        raise ValueError(f"{name}: {t.dtype} {tuple(t.shape)} on {t.device}{'' if t.is_contiguous() else ', not contiguous'}; wanted {dtype}"
                         f"{'' if count is None else f' of {count} values'} on cuda:{'*' if device is None else device}")
    return t.data_ptr()


def _rows(name, t, width, rows, device):
    """Rows [rows, ...] of `width` dense values each, f32 or bf16, which may lie further apart: (pointer, stride in values, bf16)."""
    bf16 = t.dtype is _torch.bfloat16
    if not bf16 and t.dtype is not _torch.float32:
        raise ValueError(f"{name}: {t.dtype}, wanted torch.float32 or torch.bfloat16")
    if t.get_device() != device:
        raise ValueError(f"{name}: on {t.device}, wanted cuda:{device}")
    shape, strides = t.shape, t.stride()
    if len(shape) == 2 and shape[1] == width and strides[1] == 1 and shape[0] >= rows and strides[0] >= width:
        return t.data_ptr(), strides[0], int(bf16)
    if len(shape) < 2 or shape[0] < rows or math.prod(shape[1:]) != width:
        raise ValueError(f"{name}: shape {tuple(shape)}, wanted at least {rows} rows of {width} values")
    dense = 1
    for i in range(len(shape) - 1, 0, -1):
        if strides[i] != dense and shape[i] != 1:
            raise ValueError(f"{name}: a row's values are not dense")
        dense *= shape[i]
    stride = strides[0] if shape[0] > 1 else width
    if stride < width:
        raise ValueError(f"{name}: rows overlap")
    return t.data_ptr(), stride, int(bf16)


class KvCache:
    """`oxhip_kv_cache`: an 8-bit key / value cache in torch tensors, codes uint8 [n_pages, n_kv, page_tokens / 32, 32 d] and f32 scales
    [n_pages, n_kv, page_tokens / 32] each. `HipBackend.kv_cache` makes a new one."""

    def __init__(self, k, v, k_scale, v_scale, page_tokens, d):
        import torch
        if k.dim() != 4 or page_tokens < 32 or k.shape[2] != page_tokens // 32 or k.shape[3] != 32 * d:
            raise ValueError(f"k: shape {tuple(k.shape)}, wanted [n_pages, n_kv, {page_tokens // 32}, {32 * d}]")
        n_pages, n_kv = k.shape[:2]
        dev, blocks = k.get_device() if k.is_cuda else None, n_pages * n_kv * (page_tokens // 32)
        p = [_array(n, t, torch.uint8, dev, blocks * 32 * d) for n, t in (("k", k), ("v", v))]
        p += [_array(n, t, torch.float32, dev, blocks) for n, t in (("k_scale", k_scale), ("v_scale", v_scale))]
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.page_tokens, self.n_kv, self.d, self.device = page_tokens, n_kv, d, dev
        self.c = KvCacheC(*p, n_pages, page_tokens, n_kv, d)
        self.ref = C.byref(self.c)


class KvBatch:
    """`oxhip_kv_batch`: kv_len int32 [n_seqs], pages int32 [n_seqs, max_pages], row_start int32 [n_seqs + 1] or None (one row each). Their
    contents may change between calls (and between a recorded plan's replays)."""

    def __init__(self, kv_len, pages, rows=None, row_start=None):
        import torch
        n, dev = kv_len.numel(), kv_len.get_device() if kv_len.is_cuda else None
        if pages.dim() != 2:
            raise ValueError(f"pages: shape {tuple(pages.shape)}, wanted [{n}, max_pages]")
        p = _array("kv_len", kv_len, torch.int32, dev), _array("pages", pages, torch.int32, dev, n * pages.shape[1])
        start = _array("row_start", row_start, torch.int32, dev, n + 1)
        if rows is None and row_start is not None:
            raise ValueError("rows: how many the batch has in all is the host's to know")
        self.kv_len, self.pages, self.row_start = kv_len, pages, row_start
        self.rows, self.n_seqs, self.device = n if rows is None else rows, n, dev
        self.c = KvBatchC(n, self.rows, start, *p, pages.shape[1])
        self.ref = C.byref(self.c)


class Rope:
    """`oxhip_rope`: a table of angles f32 [n_pos, n_rot / 2, 2] of (cos, sin)."""

    def __init__(self, table, interleaved=False):
        import torch
        if table.dim() != 3 or table.shape[2] != 2:
            raise ValueError(f"table: shape {tuple(table.shape)}, wanted [n_pos, n_rot / 2, 2]")
        self.table = table
        self.c = RopeC(_array("table", table, torch.float32), table.shape[0], 2 * table.shape[1], int(interleaved))
        self.ref, self.device = C.byref(self.c), table.get_device()


class HipBackend:
    """Mirror of `impl Backend for CudaBackend` (src/cuda.rs) over the HIP library."""

    def __init__(self, device=0):
        self.lib = load_library()
        ctx = C.c_void_p()
        if not self.lib.oxhip_open(device, C.byref(ctx)):
            raise RuntimeError("device hip: " + self.last_error())
        self.ctx = ctx
        self.device = device

    def close(self):
        if self.ctx:
            self.lib.oxhip_close(self.ctx)
            self.ctx = None

    def last_error(self):
        return (self.lib.oxhip_last_error() or b"").decode()

    # ---- Backend surface -------------------------------------------------------------------
    def name(self):
        return self.lib.oxhip_name(self.ctx).decode()

    def wants(self, n_out, n_in, t):
        return bool(self.lib.oxhip_wants(self.ctx, n_out, n_in, t))

    def stats(self):
        buf = C.create_string_buffer(256)
        self.lib.oxhip_stats(self.ctx, buf, 256)
        return buf.value.decode()

    def _upload(self, desc, keep):
        h = self.lib.oxhip_upload(self.ctx, C.byref(desc))
        del keep
        return DeviceWeight(self, h, desc.n_out, desc.n_in) if h else None

    @staticmethod
    def desc_gguf(ggml_type, data, n_out, n_in):
        data = np.ascontiguousarray(data, np.uint8)
        return WeightDesc(kind=W_GGUF, ggml_type=ggml_type, n_out=n_out, n_in=n_in, data=_np_ptr(data)), (data,)

    @staticmethod
    def desc_mlx_q4(w, scales, biases, group, n_out, n_in):
        w = np.ascontiguousarray(w, np.uint32)
        scales, biases = np.ascontiguousarray(scales, np.uint16), np.ascontiguousarray(biases, np.uint16)
        return (WeightDesc(kind=W_MLX_Q4, n_out=n_out, n_in=n_in, data=_np_ptr(w), scales=_np_ptr(scales), offsets=_np_ptr(biases),
                           group=group), (w, scales, biases))

    def upload_moe(self, gate_up, down, h, inter, up=None, act=ACT_SILU, act_param=0.0):
        """Backend::upload_moe: gate_up / down (/ up) are lists of (WeightDesc, keepalive) per expert."""
        n = len(gate_up)

        def arr(ds):
            a = (WeightDesc * n)()
            for i, (d, _) in enumerate(ds):
                a[i] = d
            return a
        hnd = self.lib.oxhip_upload_moe(self.ctx, arr(gate_up), arr(up) if up else None, arr(down), n, h, inter, act, act_param)
        return DeviceMoe(self, hnd, n, h, inter) if hnd else None

    def moe(self, x, t, h, inter, route_idx, route_w, k, dev, y):
        """Backend::moe: adds the routed experts' output into y ([t, h] f32, host). False = declined, y untouched."""
        x = np.ascontiguousarray(x, np.float32)
        ri, rw = np.ascontiguousarray(route_idx, np.uint32), np.ascontiguousarray(route_w, np.float32)
        assert y.dtype == np.float32 and y.flags.c_contiguous
        return bool(self.lib.oxhip_moe_forward(self.ctx, _np_ptr(x), t, h, inter, _np_ptr(ri), _np_ptr(rw), k, dev.handle, _np_ptr(y)))

    def dev_moe(self, dev, x, route_idx, route_w, y):
        """The same on device tensors: x [t, h] f32, route_idx [t, k] int32 (values as u32), route_w [t, k] f32, y += ."""
        t, k = route_idx.shape
        if not self.lib.oxhip_dev_moe(self.ctx, dev.handle, x.data_ptr(), t, route_idx.data_ptr(), route_w.data_ptr(), k,
                                      y.data_ptr(), self._stream()):
            raise RuntimeError(self.last_error())
        return y

    def route_top_k(self, logits, k):
        """moe::route_top_k on device logits [t, n_experts] -> (idx int32 [t, k], w f32 [t, k])."""
        import torch
        t, n = logits.shape
        idx = torch.empty((t, k), dtype=torch.int32, device=logits.device)
        w = torch.empty((t, k), dtype=torch.float32, device=logits.device)
        if not self.lib.oxhip_dev_route_top_k(self.ctx, logits.data_ptr(), t, n, k, idx.data_ptr(), w.data_ptr(), self._stream()):
            raise RuntimeError(self.last_error())
        return idx, w

    def matvec_rows(self, x, t, n_in, jobs):
        """Backend::matvec_rows: jobs = [(w, up or None, y ndarray [t, n_out])], 1 <= t <= 4."""
        x = np.ascontiguousarray(x, np.float32)
        arr = (RowsJob * len(jobs))()
        for i, (w, up, y) in enumerate(jobs):
            arr[i] = RowsJob(w.handle, up.handle if up is not None else None, w.n_out, y.ctypes.data)
        return bool(self.lib.oxhip_matvec_rows(self.ctx, _np_ptr(x), t, n_in, arr, len(jobs)))

    def upload_gguf(self, ggml_type, data, n_out, n_in):
        """WeightRef::Gguf: raw blocks, rows of `row_bytes` (src/ggml.rs:240-248)."""
        data = np.ascontiguousarray(data, np.uint8)
        bs, ts = GGML_BLOCK.get(ggml_type, (1, 0))
        if ts and data.size != n_out * (n_in // bs) * ts:
            raise ValueError("GGUF byte count does not match the shape")
        d = WeightDesc(kind=W_GGUF, ggml_type=ggml_type, n_out=n_out, n_in=n_in, data=_np_ptr(data))
        return self._upload(d, data)

    def upload_fp8(self, data, block_scales, n_out, n_in, block=(128, 128)):
        """GgufMatrix::fp8 (src/ggml.rs:325-341)."""
        data = np.ascontiguousarray(data, np.uint8)
        bs = np.ascontiguousarray(block_scales, np.float32)
        d = WeightDesc(kind=W_GGUF, ggml_type=GGML_F8E4M3, n_out=n_out, n_in=n_in, data=_np_ptr(data),
                       block_scales=_np_ptr(bs), bs_rows=block[0], bs_cols=block[1])
        return self._upload(d, (data, bs))

    def upload_nvfp4(self, data, n_out, n_in, scales=None, block=None):
        """GgufMatrix of NVFP4 blocks (src/ggml.rs:79-83) with, optionally, the matrix's scales on top (`block` = rows x
        columns per scale; default one scale for the matrix, as model::nvfp4_blocks builds it)."""
        data = np.ascontiguousarray(data, np.uint8)
        if data.size != n_out * (n_in // 64) * 36:
            raise ValueError("NVFP4 byte count does not match the shape")
        bs = None if scales is None else np.ascontiguousarray(np.atleast_1d(scales), np.float32)
        br, bc = block or (n_out, n_in)
        d = WeightDesc(kind=W_GGUF, ggml_type=GGML_NVFP4, n_out=n_out, n_in=n_in, data=_np_ptr(data), block_scales=_np_ptr(bs),
                       bs_rows=br if bs is not None else 0, bs_cols=bc if bs is not None else 0)
        return self._upload(d, (data, bs))

    def upload_q8(self, q, scales, n_out, n_in):
        """WeightRef::Q8 (QMatrix, src/quant.rs:128-133): int8 codes, one f32 scale per block of 32."""
        q, scales = np.ascontiguousarray(q, np.int8), np.ascontiguousarray(scales, np.float32)
        d = WeightDesc(kind=W_Q8, n_out=n_out, n_in=n_in, data=_np_ptr(q), scales=_np_ptr(scales))
        return self._upload(d, (q, scales))

    def upload_q4(self, q, scales, offsets, group, n_out, n_in):
        """WeightRef::Q4 (src/quant.rs:427-440): nibbles, f16 scales per 32, optional bf16 offsets."""
        q, scales = np.ascontiguousarray(q, np.uint8), np.ascontiguousarray(scales, np.uint16)
        offsets = None if offsets is None else np.ascontiguousarray(offsets, np.uint16)
        d = WeightDesc(kind=W_Q4, n_out=n_out, n_in=n_in, data=_np_ptr(q), scales=_np_ptr(scales),
                       offsets=_np_ptr(offsets), group=group if offsets is not None else 0)
        return self._upload(d, (q, scales, offsets))

    def upload_mlx_q4(self, w, scales, biases, group, n_out, n_in):
        """The MLX triplet; the device does what from_mlx_q4 does (src/quant.rs:518-563)."""
        w = np.ascontiguousarray(w, np.uint32)
        scales, biases = np.ascontiguousarray(scales, np.uint16), np.ascontiguousarray(biases, np.uint16)
        d = WeightDesc(kind=W_MLX_Q4, n_out=n_out, n_in=n_in, data=_np_ptr(w), scales=_np_ptr(scales),
                       offsets=_np_ptr(biases), group=group)
        return self._upload(d, (w, scales, biases))

    def upload_bf16(self, w, n_out, n_in):
        w = np.ascontiguousarray(w, np.uint16)
        d = WeightDesc(kind=W_BF16, n_out=n_out, n_in=n_in, data=_np_ptr(w))
        return self._upload(d, w)

    def matmul(self, x, t, n_in, jobs):
        """Backend::matmul: jobs = [(DeviceWeight, y ndarray [t, n_out] f32)]; True if every y was written."""
        x = np.ascontiguousarray(x, np.float32)
        arr = (Job * len(jobs))()
        for i, (w, y) in enumerate(jobs):
            assert y.dtype == np.float32 and y.flags.c_contiguous
            arr[i] = Job(w.handle, w.n_out, y.ctypes.data)
        return bool(self.lib.oxhip_matmul(self.ctx, _np_ptr(x), t, n_in, arr, len(jobs)))

    # ---- device-pointer entry points -------------------------------------------------------
    @staticmethod
    def _stream():
        """The current torch stream of the current device, as the handle that the library takes. By torch's accessor of the handle
        itself where it has one: building a torch Stream object for its handle took 3 us of the 6.5 us that a call of one launch
        takes, this 0.2 us (a 4096 x 4096 product of one token, two calls: 14.5 -> 9.3 us). (`_cuda_getDevice` initialises the device
        as torch's own calls do, or raises as they do.)"""
        torch = _torch
        if torch is None:
            import torch
        try:
            return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())
        except AttributeError:
            return torch.cuda.current_stream().cuda_stream

    def quantize_act(self, x, out=None):
        """x: torch f32 [t, n_in] on the device -> QAct (device)."""
        t, n_in = x.shape
        out = out or QAct(t, n_in, x.device)
        if not self.lib.oxhip_dev_quantize_act(self.ctx, x.data_ptr(), t, n_in, C.byref(out.c), self._stream()):
            raise RuntimeError(self.last_error())
        return out

    def quantize_jobs(self, pairs):
        """A reusable job array for quantize_act_batch: pairs = [(x f32 [t, n_in] on the device, QAct)]."""
        arr = (QuantJob * len(pairs))()
        for i, (x, out) in enumerate(pairs):
            arr[i] = QuantJob(x.data_ptr(), x.shape[0], x.shape[1], C.addressof(out.c))
        return arr

    def quantize_act_batch(self, arr):
        if not self.lib.oxhip_dev_quantize_act_batch(self.ctx, arr, len(arr), self._stream()):
            raise RuntimeError(self.last_error())

    def dequantize(self, w, r0=0, r1=None):
        import torch
        r1 = w.n_out if r1 is None else r1
        out = torch.empty((r1 - r0, w.n_in), dtype=torch.float32, device=f"cuda:{self.device}")
        if not self.lib.oxhip_dev_dequantize(self.ctx, w.handle, r0, r1, out.data_ptr(), self._stream()):
            raise RuntimeError(self.last_error())
        return out

    def decode(self, w, xa=None, x=None, t=None, y=None):
        """The decode kernels on device buffers: xa (QAct) for quantized weights, x (f32) for float-stored ones."""
        import torch
        t = t or (xa.t if xa is not None else x.shape[0])
        if y is None:
            y = torch.empty((t, w.n_out), dtype=torch.float32, device=f"cuda:{self.device}")
        ok = self.lib.oxhip_dev_decode(self.ctx, w.handle, C.byref(xa.c) if xa is not None else None,
                                       x.data_ptr() if x is not None else None, t, y.data_ptr(), self._stream())
        if not ok:
            raise RuntimeError(self.last_error())
        return y

    def decode_noalloc(self, w, xa, t=None, y=None):
        """oxhip_dev_decode_noalloc: the decode kernels over the library's static scratch. False = declined."""
        import torch
        t = t or xa.t
        if y is None:
            y = torch.empty((t, w.n_out), dtype=torch.float32, device=f"cuda:{self.device}")
        ok = self.lib.oxhip_dev_decode_noalloc(self.ctx, w.handle, C.byref(xa.c), t, y.data_ptr(), self._stream())
        return y if ok else None

    # ---- decode-graph ops (device tensors; Op::Norm / Linear / Route / Experts of src/gpu_decode.rs) -----------
    def rmsnorm_quantize(self, x, w=None, eps=1e-6, want_out=True, want_q=True):
        """x [t, n] f32 -> (normed [t, n] f32 or None, QAct or None); w: f32 or bf16 device tensor [n], or None."""
        import torch
        t, n = x.shape
        out = torch.empty_like(x) if want_out else None
        q = QAct(t, n, x.device) if want_q else None
        wf = w.data_ptr() if w is not None and w.dtype == torch.float32 else None
        wb = w.data_ptr() if w is not None and w.dtype == torch.bfloat16 else None
        ok = self.lib.oxhip_dev_rmsnorm_quantize(self.ctx, x.data_ptr(), wf, wb, eps, t, n, out.data_ptr() if want_out else None,
                                                 C.byref(q.c) if want_q else None, self._stream())
        if not ok:
            raise RuntimeError(self.last_error())
        return out, q

    def norm(self, x, n, rows, out=None, w=None, pre=1.0, x_stride=0, out_stride=0, eps=1e-6, add=False, want_q=False):
        """Op::Norm with all its fields on device tensors (x, out: f32, any float offset into a larger buffer)."""
        import torch
        q = QAct(rows, n, x.device) if want_q else None
        wf = w.data_ptr() if w is not None and w.dtype == torch.float32 else None
        wb = w.data_ptr() if w is not None and w.dtype == torch.bfloat16 else None
        ok = self.lib.oxhip_dev_norm(self.ctx, x.data_ptr(), out.data_ptr() if out is not None else None, wf, wb, pre, n, rows, x_stride,
                                     out_stride, eps, int(add), C.byref(q.c) if want_q else None, self._stream())
        return (bool(ok), q)

    def stream_release(self, stream):
        return bool(self.lib.oxhip_stream_release(self.ctx, C.c_void_p(stream)))

    def linear(self, w, y, xa=None, x=None, t=None, mode=LIN_STORE, w2=None, gate=None):
        """Op::Linear on device tensors; y [t, n_out] f32 is written or added to according to `mode`. False = declined."""
        t = t or (xa.t if xa is not None else x.shape[0])
        return bool(self.lib.oxhip_dev_linear(self.ctx, w.handle, w2.handle if w2 is not None else None,
                                              C.byref(xa.c) if xa is not None else None, x.data_ptr() if x is not None else None, t,
                                              y.data_ptr(), mode, gate.data_ptr() if gate is not None else None, self._stream()))

    def glu(self, g, u, gelu=False):
        import torch
        y = torch.empty_like(g)
        if not self.lib.oxhip_dev_glu(self.ctx, g.data_ptr(), u.data_ptr(), g.numel(), int(gelu), y.data_ptr(), self._stream()):
            raise RuntimeError(self.last_error())
        return y

    def route(self, x, router, k, gate=None, expert_scale=None):
        """Op::Route: x [t, h], router [n_exp, h] f32 -> (logits [t, n_exp (+1)], sel int32 [2, t, k]: ids, then weight bits)."""
        import torch
        t, h = x.shape
        n_exp = router.shape[0]
        logits = torch.empty((t, n_exp + (1 if gate is not None else 0)), dtype=torch.float32, device=x.device)
        sel = torch.empty((2, t, k), dtype=torch.int32, device=x.device)
        ok = self.lib.oxhip_dev_route(self.ctx, x.data_ptr(), router.data_ptr(), gate.data_ptr() if gate is not None else None, t, n_exp, h, k,
                                      logits.data_ptr(), sel.data_ptr(), expert_scale.data_ptr() if expert_scale is not None else None, self._stream())
        if not ok:
            raise RuntimeError(self.last_error())
        return logits, sel

    def experts(self, dev, x, sel, y, add=True):
        """Op::Experts: the experts chosen in `sel` (as route() returns it) over x [t, h]; y += or y =."""
        _, t, k = sel.shape
        return bool(self.lib.oxhip_dev_experts(self.ctx, dev.handle, x.data_ptr(), t, sel.data_ptr(), k, y.data_ptr(), int(add), self._stream()))

    def moe_routed(self, dev, x, logits, k, y, sel=None, add=True, expert_scale=None):
        """Top-k of `logits` [t, n_exp (+...)] and the routed experts over x [t, h] in one call; returns sel [2, t, k]."""
        import torch
        t = x.shape[0]
        if sel is None:
            sel = torch.empty((2, t, k), dtype=torch.int32, device=x.device)
        ok = self.lib.oxhip_dev_moe_routed(self.ctx, dev.handle, x.data_ptr(), t, logits.data_ptr(), logits.shape[1], k,
                                           expert_scale.data_ptr() if expert_scale is not None else None, sel.data_ptr(), y.data_ptr(),
                                           int(add), self._stream())
        if not ok:
            raise RuntimeError(self.last_error())
        return sel

    # ---- attention over an 8-bit cache, the logits' rules ---------------------------------------------------------
    def _stream_here(self):
        """The current torch stream of this backend's device, which need not be the current device."""
        if _torch._C._cuda_getDevice() == self.device:
            return self._stream()
        return _torch.cuda.current_stream(self.device).cuda_stream

    def _held(self, cache, batch):
        if cache.device != self.device or batch.device != self.device:
            raise ValueError(f"the cache and the batch are wanted on cuda:{self.device}")

    def kv_cache(self, n_pages, n_kv, d, page_tokens=64):
        """A new 8-bit cache of n_pages pages of page_tokens tokens (a power of two, 32 at least), d a multiple of 32 up to 256."""
        import torch
        dev, per = f"cuda:{self.device}", page_tokens // 32
        codes = [torch.full((n_pages, n_kv, per, 32 * d), 128, dtype=torch.uint8, device=dev) for _ in range(2)]
        scales = [torch.zeros((n_pages, n_kv, per), dtype=torch.float32, device=dev) for _ in range(2)]
        return KvCache(*codes, *scales, page_tokens, d)

    def kv_append(self, cache, batch, k, v, q=None, rope=None, q_out=None):
        """The rows' keys and values [rows, n_kv * d] (f32 or bf16; any row stride) into the cache; the keys, and the queries [rows, n_q * d],
        rotated by `rope`. Returns the rotated queries (`q_out`, which may be q) or None. Rows behind the last sequence, and rows before a
        sequence's first token, are left as `q_out` has them: in a new one they may hold anything."""
        self._held(cache, batch)
        dev, rows, width = self.device, batch.rows, cache.n_kv * cache.d
        kp, ks, kd = _rows("k", k, width, rows, dev)
        vp, vs, vd = _rows("v", v, width, rows, dev)
        qp = op = None
        qs = os_ = n_q = 0
        qd = od = kd
        if q is not None:
            q_width = math.prod(q.shape[1:])
            n_q = q_width // cache.d
            qp, qs, qd = _rows("q", q, n_q * cache.d, rows, dev)
            if q_out is None:
                q_out = q.new_empty(q.shape)
                op, os_ = q_out.data_ptr(), q_width
            else:
                op, os_, od = _rows("q_out", q_out, n_q * cache.d, rows, dev)
        elif q_out is not None:
            raise ValueError("q_out without q")
        if not kd == vd == qd == od:
            raise ValueError("q, q_out, k and v have one type")
        if rope is not None and rope.device != dev:
            raise ValueError(f"rope: wanted on cuda:{dev}")
        if rows and not self.lib.oxhip_dev_kv_append(self.ctx, cache.ref, batch.ref, kp, ks, vp, vs, qp, qs, op, os_, n_q, kd, rope.ref if rope is not None else None,
                                                     self._stream_here()):
            raise RuntimeError(self.last_error())
        return q_out

    def kv_read(self, cache, batch, count, dtype=None):
        """The values that the last `count` tokens of every sequence stand for: (k, v), each [n_seqs, count, n_kv, d] f32 (or bf16)."""
        self._held(cache, batch)
        dtype = dtype or _torch.float32
        if dtype not in (_torch.float32, _torch.bfloat16):
            raise ValueError(f"dtype: {dtype}")
        both = cache.k_scale.new_empty((2, batch.n_seqs, count, cache.n_kv, cache.d), dtype=dtype)
        at = both.data_ptr()
        if count and not self.lib.oxhip_dev_kv_read(self.ctx, cache.ref, batch.ref, count, at, at + both.nbytes // 2, int(dtype is _torch.bfloat16), self._stream_here()):
            raise RuntimeError(self.last_error())
        return both.unbind(0)

    def attend(self, cache, batch, q, scale=None, cap=0.0, slopes=None, window=0, prefix=None, first=None, out=None):
        """Attention of q [rows, n_q * d] (f32 or bf16; any row stride) over the cache; scale: 1 / sqrt(d) by default. The rules are those of
        `oxhip_attend_rules`. Returns out, of q's shape and type; rows behind the last sequence are left as `out` has them: in a new one they
        may hold anything."""
        self._held(cache, batch)
        dev, width = self.device, math.prod(q.shape[1:])
        n_q = width // cache.d
        qp, qs, qd = _rows("q", q, n_q * cache.d, batch.rows, dev)
        if out is None:
            out = q.new_empty(q.shape)
            op, os_ = out.data_ptr(), width
        else:
            op, os_, od = _rows("out", out, n_q * cache.d, batch.rows, dev)
            if qd != od:
                raise ValueError("q and out have one type")
        rules = None
        if cap or window or slopes is not None or prefix is not None or first is not None:
            if window < 0:
                raise ValueError("window: at least 0")
            if first is not None and first.numel() < batch.rows:
                raise ValueError("first: one for each row")
            rules = C.byref(AttendRulesC(cap, _array("slopes", slopes, _torch.float32, dev, n_q), window, _array("prefix", prefix, _torch.int32, dev, batch.n_seqs),
                                         _array("first", first, _torch.int32, dev)))
        if batch.rows and not self.lib.oxhip_dev_attend(self.ctx, cache.ref, batch.ref, qp, qs, n_q, qd, cache.d**-0.5 if scale is None else scale, rules, op, os_,
                                                        self._stream_here()):
            raise RuntimeError(self.last_error())
        return out

    def adjust_logits(self, logits, out=None, want_out=True, want_next=True, history=None, history_len=None, prompt_len=None, repetition=None,
                      presence=None, frequency=None, bias_start=None, bias_id=None, bias=None, allowed=None, allowed_row=None):
        """The rules of `oxhip_logit_rules` on rows of logits [rows, vocab] (f32 or bf16; any row stride): (out, next), the adjusted logits (`out`
        may be `logits`) and the best token of each row, int32. history int32 [rows, most], allowed int32 words [masks, (vocab + 31) / 32]."""
        t, vocab = logits.shape
        dev, i32, f32 = self.device, _torch.int32, _torch.float32
        lp, ls, ld = _rows("logits", logits, vocab, t, dev)
        op, os_, best = None, 0, None
        if out is not None:
            op, os_, od = _rows("out", out, vocab, t, dev)
            if od != ld:
                raise ValueError("logits and out have one type")
        elif want_out:
            out = logits.new_empty((t, vocab))
            op, os_ = out.data_ptr(), vocab
        if want_next:
            best = logits.new_empty(t, dtype=i32)
        elif op is None:
            raise ValueError("neither the adjusted logits nor the best tokens are wanted")
        rules = None
        if history is not None or bias_start is not None or allowed is not None:
            r = LogitRulesC()
            empty = False
            if history is not None:
                if history.dim() != 2 or history.shape[0] != t or history_len is None:
                    raise ValueError(f"history: shape {tuple(history.shape)}{', without history_len' if history_len is None else ''}, wanted [{t}, most] and a length for each row")
                empty = not history.shape[1]  # (no token at all: the tensor has no address, and no logit a penalty)
                at, lens = _array("history", history, i32, dev), _array("history_len", history_len, i32, dev, t)
                if not empty:
                    r.history, r.history_stride, r.history_len = at, history.shape[1], lens
            for name, value, kind in (("prompt_len", prompt_len, i32), ("repetition", repetition, f32), ("presence", presence, f32), ("frequency", frequency, f32)):
                if value is not None:
                    at = _array(name, value, kind, dev, t)
                    if not empty:
                        setattr(r, name, at)
            if bias_start is not None or bias_id is not None or bias is not None:
                n = bias_id.numel() if bias_id is not None else 0
                r.bias_start, r.bias_id, r.bias, r.n_bias = _array("bias_start", bias_start, i32, dev, t + 1), _array("bias_id", bias_id, i32, dev), _array("bias", bias, f32, dev, n), n
                if bias_id is not None and bias_start is not None and bias is not None and not n:  # (no biases at all: their tensors have no address)
                    r.bias_start = r.bias_id = r.bias = None
            if allowed is not None:
                if allowed.dim() != 2:
                    raise ValueError(f"allowed: shape {tuple(allowed.shape)}, wanted [masks, words]")
                r.allowed, r.n_allowed, r.allowed_stride = _array("allowed", allowed, i32, dev), allowed.shape[0], allowed.shape[1]
            r.allowed_row = _array("allowed_row", allowed_row, i32, dev, t)
            rules = C.byref(r)
        elif any(v is not None for v in (history_len, prompt_len, repetition, presence, frequency, bias_id, bias, allowed_row)):
            raise ValueError("penalties need a history, biases bias_start, allowed_row masks")
        if t and not self.lib.oxhip_dev_logits(self.ctx, lp, ls, op, os_, t, vocab, ld, rules, best.data_ptr() if want_next else None, self._stream_here()):
            raise RuntimeError(self.last_error())
        return out, best

    def plan_record(self, chain):
        """Records chain() (device-pointer calls on the current torch stream, which must not be the null stream) and
        returns a Plan; raises when the recording fails. Run chain() once on that stream beforehand."""
        h = self.lib.oxhip_plan_begin(self.ctx, self._stream())
        if not h:
            raise RuntimeError(self.last_error())
        try:
            chain()
        except BaseException:
            self.lib.oxhip_plan_free(h)
            raise
        if not self.lib.oxhip_plan_end(h):
            msg = self.last_error()
            self.lib.oxhip_plan_free(h)
            raise RuntimeError(msg)
        return Plan(self, h)

    def decode_jobs(self, jobs):
        """Builds a reusable job array for decode_batch: jobs = [(DeviceWeight, QAct | None, x | None, t, y, ev0, ev1)]."""
        arr = (DecodeJob * len(jobs))()
        for i, (w, xa, x, t, y, e0, e1) in enumerate(jobs):
            arr[i] = DecodeJob(w.handle, C.addressof(xa.c) if xa is not None else None,
                               x.data_ptr() if x is not None else None, t, y.data_ptr(), e0, e1)
        return arr

    def decode_batch(self, arr):
        if not self.lib.oxhip_dev_decode_batch(self.ctx, arr, len(arr), self._stream()):
            raise RuntimeError(self.last_error())

    def event(self):
        e = self.lib.oxhip_event_create()
        if not e:
            raise RuntimeError(self.last_error())
        return e

    def elapsed_ms(self, a, b):
        return self.lib.oxhip_event_elapsed_ms(a, b)

    def gemm(self, w, x, variant=0, out_bf16=False, events=None):
        """Prefill GEMM on device tensors: x [t, n_in] f32 or bf16 -> y [t, n_out] f32 (or bf16). `events`: a pair from
        event() that the library records right before and after the variant's matrix kernel."""
        import torch
        t = x.shape[0]
        y = torch.empty((t, w.n_out), dtype=torch.bfloat16 if out_bf16 else torch.float32, device=x.device)
        xd = 1 if x.dtype == torch.bfloat16 else 0
        assert x.dtype in (torch.bfloat16, torch.float32) and x.is_contiguous()
        if events is None:
            ok = self.lib.oxhip_dev_gemm(self.ctx, w.handle, x.data_ptr(), xd, t, y.data_ptr(), int(out_bf16), variant, self._stream())
        else:
            ok = self.lib.oxhip_dev_gemm_timed(self.ctx, w.handle, x.data_ptr(), xd, t, y.data_ptr(), int(out_bf16), variant, self._stream(),
                                               events[0], events[1])
        if not ok:
            raise RuntimeError(self.last_error())
        return y

    def gemm_isums(self, w, x):
        """The int8 GEMM's exact block sums [t, n_out, n_in/32] (int32)."""
        import torch
        t = x.shape[0]
        out = torch.zeros((t, w.n_out, w.n_in // 32), dtype=torch.int32, device=x.device)
        xd = 1 if x.dtype == torch.bfloat16 else 0
        assert x.dtype in (torch.bfloat16, torch.float32) and x.is_contiguous()
        if not self.lib.oxhip_dev_gemm_isums(self.ctx, w.handle, x.data_ptr(), xd, t, out.data_ptr(), self._stream()):
            raise RuntimeError(self.last_error())
        return out

    def isums(self, w, xa, per):
        import torch
        out = torch.empty((xa.t, w.n_out, w.n_in // per), dtype=torch.int32, device=f"cuda:{self.device}")
        if not self.lib.oxhip_dev_isums(self.ctx, w.handle, C.byref(xa.c), out.data_ptr(), self._stream()):
            raise RuntimeError(self.last_error())
        return out
