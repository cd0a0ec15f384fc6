"""ctypes binding of libehip.so, the C ABI declared in include/ehip.h.

The library takes raw device pointers; this module accepts torch tensors that
live on the GPU (torch is only the allocator and stream provider here) and
turns every nonzero status into a RuntimeError carrying ehip_last_error().
Loading fails loudly if the library is not built: there is no fallback.
"""
import ctypes as C
import os

ROOT = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(ROOT, "lib", "libehip.so")
HEADER = os.path.join(os.path.dirname(ROOT), "include", "ehip.h")

_vp, _i, _i64, _f, _sz = C.c_void_p, C.c_int, C.c_int64, C.c_float, C.c_size_t

ADD, SUB, MUL, DIV = 0, 1, 2, 3


class Window(C.Structure):
    _fields_ = [(n, C.c_int64) for n in (
        "batch", "channels", "height", "width", "kernel_h", "kernel_w", "stride", "padding",
        "out_h", "out_w")]


def window(n, c, h, w, kh, kw, stride, pad):
    return Window(n, c, h, w, kh, kw, stride, pad, (h + 2 * pad - kh) // stride + 1,
                  (w + 2 * pad - kw) // stride + 1)


class AdamTensor(C.Structure):
    _fields_ = [("p", C.c_void_p), ("g", C.c_void_p), ("m", C.c_void_p), ("v", C.c_void_p),
                ("n", C.c_int64)]


class KernelOccupancy(C.Structure):
    _fields_ = [("name", C.c_char * 96), ("block_threads", C.c_int), ("registers", C.c_int),
                ("lds_bytes", C.c_int64), ("blocks_per_cu", C.c_int), ("occupancy", C.c_double),
                ("limiter", C.c_char * 16)]


class DeviceInfo(C.Structure):
    _fields_ = [("name", C.c_char * 256), ("arch", C.c_char * 64), ("compute_units", C.c_int),
                ("clock_khz", C.c_int), ("memory_clock_khz", C.c_int),
                ("memory_bus_width_bits", C.c_int), ("total_memory", C.c_size_t),
                ("lds_per_block", C.c_size_t), ("l2_bytes", C.c_int),
                ("peak_fp32_mfma_gflops", C.c_double), ("peak_hbm_gbs", C.c_double)]


class ArenaStats(C.Structure):
    _fields_ = [(n, C.c_uint64) for n in ("bytes_in_use", "bytes_cached", "bytes_reserved",
                                         "allocations", "driver_allocations",
                                         "bytes_graph_held")]


class TransferStats(C.Structure):
    _fields_ = [(n, C.c_uint64) for n in (
        "to_device_bytes", "to_host_bytes", "device_to_device_bytes", "to_device_count",
        "to_host_count", "device_to_device_count")] + [
        ("to_device_seconds", C.c_double), ("to_host_seconds", C.c_double)]


class ConvReduce(C.Structure):
    """ehip_conv_reduce_t: one layer's weight partials and where their sums go."""
    _fields_ = [("partials", C.c_void_p), ("chunks", C.c_int64), ("out_channels", C.c_int64),
                ("k", C.c_int64), ("dweight", C.c_void_p), ("dbias", C.c_void_p)]


class GemmEx(C.Structure):
    """ehip_gemm_ex_t: two-level batch strides and the alpha / addend / beta / residual
    epilogue."""
    _fields_ = [("trans_a", C.c_int), ("trans_b", C.c_int), ("batch", C.c_int64),
                ("inner", C.c_int64), ("m", C.c_int64), ("n", C.c_int64), ("k", C.c_int64),
                ("a", C.c_void_p), ("lda", C.c_int64), ("stride_a", C.c_int64),
                ("stride_a_inner", C.c_int64), ("b", C.c_void_p), ("ldb", C.c_int64),
                ("stride_b", C.c_int64), ("stride_b_inner", C.c_int64), ("c", C.c_void_p),
                ("ldc", C.c_int64), ("stride_c", C.c_int64), ("stride_c_inner", C.c_int64),
                ("alpha", C.c_float), ("addend", C.c_void_p), ("ld_addend", C.c_int64),
                ("stride_addend", C.c_int64), ("addend_period", C.c_int64), ("beta", C.c_float),
                ("relu", C.c_int), ("colsum_b", C.c_void_p), ("causal", C.c_int),
                ("residual", C.c_void_p), ("ld_residual", C.c_int64)]


class AttentionPacked(C.Structure):
    """ehip_attention_packed_t: packed sequences, grouped heads, and where the result goes."""
    _fields_ = [("q", C.c_void_p), ("k", C.c_void_p), ("v", C.c_void_p), ("ld_q", C.c_int64),
                ("ld_k", C.c_int64), ("ld_v", C.c_int64), ("cu_q", C.c_void_p),
                ("cu_k", C.c_void_p), ("sequences", C.c_int64), ("total_q", C.c_int64),
                ("total_k", C.c_int64), ("heads", C.c_int64), ("kv_heads", C.c_int64),
                ("head_dim", C.c_int64), ("scale", C.c_float), ("causal", C.c_int),
                ("out", C.c_void_p), ("ld_out", C.c_int64), ("lse", C.c_void_p),
                ("longest_q", C.c_int64), ("longest_k", C.c_int64)]


class Cache(C.Structure):
    """ehip_cache_t: the pools of a paged key-value cache and the sequences' page table."""
    _fields_ = [("k_pages", C.c_void_p), ("v_pages", C.c_void_p), ("type", C.c_int),
                ("pages", C.c_int64), ("page_size", C.c_int64), ("kv_heads", C.c_int64),
                ("head_dim", C.c_int64), ("table", C.c_void_p), ("ld_table", C.c_int64),
                ("table_width", C.c_int64), ("sequences", C.c_int64)]


# name -> argtypes (all return int unless listed in _RESTYPES)
_SIGS = {
    "ehip_init": [], "ehip_available": [], "ehip_enabled": [], "ehip_set_enabled": [_i],
    "ehip_device_info": [C.POINTER(DeviceInfo)], "ehip_synchronize": [],
    "ehip_version_info": [C.POINTER(C.c_int)] * 3,
    "ehip_kernel_occupancy": [C.POINTER(KernelOccupancy), C.c_int, C.POINTER(C.c_int)],
    "ehip_stream_synchronize": [_vp], "ehip_kernels_launched": [], "ehip_kernels_failed": [],
    "ehip_reset_counters": [], "ehip_fail_launch_after": [_i64], "ehip_transfer_stats": [C.POINTER(TransferStats)],
    "ehip_reset_transfer_stats": [], "ehip_arena_alloc": [_sz, C.POINTER(_vp)],
    "ehip_arena_free": [_vp], "ehip_arena_trim": [], "ehip_arena_stats": [C.POINTER(ArenaStats)],
    "ehip_memcpy_h2d": [_vp, _vp, _sz, _vp], "ehip_memcpy_d2h": [_vp, _vp, _sz, _vp],
    "ehip_memcpy_d2d": [_vp, _vp, _sz, _vp],
    "ehip_gemm_f32": [_i, _i, _i64, _i64, _i64, _i64, _vp, _i64, _i64, _vp, _i64, _i64, _f, _vp,
                      _i64, _i64, _vp],
    "ehip_matmul_backward_f32": [_i64, _i64, _i64, _vp, _i64, _vp, _i64, _vp, _i64, _vp, _i64, _f,
                                 _vp, _i64, _f, _vp],
    "ehip_gemm_f32_noalloc": [_i, _i, _i64, _i64, _i64, _i64, _vp, _i64, _i64, _vp, _i64, _i64,
                              _f, _vp, _i64, _i64, _vp],
    "ehip_gemm_ex_f32": [C.POINTER(GemmEx), _vp],
    "ehip_gemm_groupable": [C.POINTER(GemmEx)],
    "ehip_gemm_batch_f32": [C.POINTER(GemmEx), _i, _vp],
    "ehip_linear_backward_plan": [_i64, _i64, _i64],
    "ehip_gemm_probe_arm": [_i, _i, C.POINTER(C.c_int64), _i, _i],
    "ehip_gemm_probe_read": [C.POINTER(C.c_double), C.POINTER(C.c_int64), C.POINTER(C.c_double)],
    "ehip_linear_backward_f32": [_vp] * 6 + [_i64, _i64, _i64, _vp],
    "ehip_binary_f32": [_i, _vp, _vp, _vp, _i64, _i64, _vp],
    "ehip_scalar_f32": [_vp, _vp, _i64, _f, _f, _vp],
    "ehip_relu_f32": [_vp, _vp, _i64, _vp],
    "ehip_relu_backward_f32": [_vp, _vp, _vp, _i64, _vp],
    "ehip_accumulate_grad_f32": [_vp, _vp, _i64, _i, _vp],
    "ehip_add_backward_f32": [_vp, _vp, _vp, _i64, _i, _i, _vp],
    "ehip_mul_backward_f32": [_vp, _vp, _vp, _vp, _vp, _i64, _i, _i, _vp],
    "ehip_fill_f32": [_vp, _i64, _f, _vp],
    "ehip_store_f32": [_vp, _vp, _i, _vp],
    "ehip_activation_f32": [_i, _vp, _vp, _i64, _vp],
    "ehip_activation_backward_f32": [_i, _vp, _vp, _vp, _vp, _i64, _vp],
    "ehip_copy_rows_f32": [_vp, _i64, _vp, _i64, _i64, _i64, _vp],
    "ehip_max_axis_f32": [_vp, _vp, _vp, _i64, _i64, _i64, _vp],
    "ehip_max_axis_backward_f32": [_vp, _vp, _vp, _i64, _i64, _i64, _vp],
    "ehip_scale_f32": [_vp, _i64, _f, _vp],
    "ehip_sgd_f32": [_vp, _vp, _vp, _i64, _f, _f, _f, _vp],
    "ehip_adam_f32": [_vp, _vp, _vp, _vp, _i64] + [_f] * 7 + [_vp],
    "ehip_adam_multi_f32": [C.POINTER(AdamTensor), _i] + [_f] * 7 + [_vp],
    "ehip_adam_multi_reduce_f32": [C.POINTER(AdamTensor), _i, C.POINTER(ConvReduce), _i] +
                                  [_f] * 7 + [_vp],
    "ehip_adam_multi_dev_f32": [C.POINTER(AdamTensor), _i, _vp] + [_f] * 4 + [_vp],
    "ehip_adam_multi_reduce_dev_f32": [C.POINTER(AdamTensor), _i, C.POINTER(ConvReduce), _i,
                                       _vp] + [_f] * 4 + [_vp],
    "ehip_graph_begin": [], "ehip_graph_end": [C.POINTER(_vp)], "ehip_graph_abort": [],
    "ehip_capturing": [], "ehip_graph_launch": [_vp, _vp], "ehip_graph_destroy": [_vp],
    "ehip_permute_f32": [_vp, _vp, _i, C.POINTER(_i64), C.POINTER(_i64), _vp],
    "ehip_transpose_f32": [_vp, _vp, _i64, _i64, _i64, _vp],
    "ehip_im2col_f32": [_vp, _vp, C.POINTER(Window), _vp],
    "ehip_col2im_f32": [_vp, _vp, C.POINTER(Window), _vp],
    "ehip_maxpool_f32": [_vp, _vp, _vp, C.POINTER(Window), _vp],
    "ehip_maxpool_backward_f32": [_vp, _vp, _vp, C.POINTER(Window), _vp],
    "ehip_maxpool_fidx_f32": [_vp, _vp, _vp, C.POINTER(Window), _vp],
    "ehip_maxpool_backward_fidx_f32": [_vp, _vp, _vp, C.POINTER(Window), _vp],
    "ehip_dropout_f32": [_vp, _vp, _vp, _i64, _f, C.c_uint64, C.c_uint64, _vp],
    "ehip_conv2d_direct_supported": [C.POINTER(Window), _i64],
    "ehip_conv2d_forward_f32": [_vp, _vp, _vp, _vp, C.POINTER(Window), _i64, _vp],
    "ehip_conv2d_backward_input_f32": [_vp, _vp, _vp, C.POINTER(Window), _i64, _vp],
    "ehip_conv2d_backward_weight_f32": [_vp, _vp, _vp, _vp, C.POINTER(Window), _i64, _vp],
    "ehip_attention_short_supported": [_i64, _i64],
    "ehip_attention_short_f32": [_vp] * 5 + [_i64] * 5 + [_f, _i, _vp],
    "ehip_attention_short_backward_f32": [_vp] * 8 + [_i64] * 5 + [_f, _i, _vp],
    "ehip_conv2d_igemm_supported": [C.POINTER(Window), _i64],
    "ehip_conv2d_igemm_f32": [_vp, _vp, _vp, _vp, C.POINTER(Window), _i64, _vp],
    "ehip_conv2d_igemm_backward_f32": [_vp] * 6 + [C.POINTER(Window), _i64, _vp],
    "ehip_conv2d_relu_maxpool_supported": [C.POINTER(Window), _i64, C.POINTER(Window)],
    "ehip_conv2d_relu_maxpool_f32": [_vp, _vp, _vp, _vp, _vp, C.POINTER(Window), _i64,
                                     C.POINTER(Window), _vp],
    "ehip_conv2d_relu_maxpool_backward_f32": [_vp] * 8 + [C.POINTER(Window), _i64,
                                                          C.POINTER(Window), _vp],
    "ehip_conv2d_relu_maxpool_partials": [C.POINTER(Window), _i64, C.POINTER(Window), _i,
                                          C.POINTER(_i64)],
    "ehip_conv2d_relu_maxpool_backward_partials_f32": [_vp] * 7 + [_i64, C.POINTER(Window),
                                                                   _i64, C.POINTER(Window), _vp],
    "ehip_conv_weight_reduce_f32": [C.POINTER(ConvReduce), _i, _vp],
    "ehip_select_rows_f32": [_vp, _vp, _vp, _i64, _i64, _i64, _vp],
    "ehip_scatter_add_rows_f32": [_vp, _vp, _vp, _vp, _i64, _i64, _i64, _i, _vp],
    "ehip_sum_axis_f32": [_vp, _vp, _i64, _i64, _i64, _vp],
    "ehip_reduce_sum_f32": [_vp, _i64, _i, _vp, _vp, _vp],
    "ehip_softmax_f32": [_vp, _vp, _i64, _i64, _vp],
    "ehip_softmax_backward_f32": [_vp, _vp, _vp, _i64, _i64, _vp],
    "ehip_softmax_backward_scaled_f32": [_vp, _vp, _vp, _i64, _i64, _f, _vp],
    "ehip_softmax_causal_f32": [_vp, _vp, _i64, _i64, _vp],
    "ehip_softmax_backward_scaled_causal_f32": [_vp, _vp, _vp, _i64, _i64, _f, _vp],
    "ehip_layernorm_f32": [_vp] * 6 + [_i64, _i64, _f, _vp],
    "ehip_layernorm_backward_f32": [_vp] * 7 + [_i64, _i64, _vp],
    "ehip_layernorm_backward_partials": [_i64, _i64, C.POINTER(_i64)],
    "ehip_linear_bias_from_dw": [_i],
    "ehip_layernorm_backward_partials_f32": [_vp] * 6 + [_i64, _i64, _i64, _i, _vp],
    "ehip_cross_entropy_f32": [_vp, _vp, _vp, _vp, _i64, _i64, _vp],
    "ehip_cross_entropy_backward_f32": [_vp, _vp, _vp, _i64, _i64, _vp, _vp],
    "ehip_cross_entropy_fused_supported": [_i64, _i64],
    "ehip_cross_entropy_fused_f32": [_vp] * 5 + [_i64, _i64, _vp],
    "ehip_softmax_xent_backward_f32": [_vp, _vp, _vp, _i64, _i64, _vp, _vp],
    "ehip_attention_packed_workspace": [C.POINTER(AttentionPacked)],
    "ehip_attention_packed_f32": [C.POINTER(AttentionPacked), _vp, _sz, _vp],
    "ehip_attention_packed_backward_workspace": [C.POINTER(AttentionPacked)],
    "ehip_attention_packed_backward_f32": [C.POINTER(AttentionPacked)] + [_vp, _i64] * 4 +
                                          [_vp, _sz, _vp],
    "ehip_cache_append_f32": [C.POINTER(Cache), _vp, _i64, _vp, _i64, _vp, _vp, _i64, _vp],
    "ehip_attention_paged_workspace": [C.POINTER(Cache), _i64, _i64],
    "ehip_attention_paged_f32": [C.POINTER(Cache), _vp, _i64, _i64, _vp, _i64, _f, _vp, _i64,
                                 _vp, _vp, _sz, _vp],
    "ehip_token_logprobs_workspace": [_i64, _i64, _i64],
    "ehip_token_logprobs_f32": [_vp, _i64, _vp, _i64, _i64, _vp, _vp, _vp, _i64, _vp, _vp, _vp,
                                _sz, _vp],
    "ehip_token_logprobs_backward_f32": [_vp, _i64] + [_vp] * 6 + [_i64, _i64, _i64, _vp],
    "ehip_last_error": [],
}
_RESTYPES = {"ehip_last_error": C.c_char_p,
             "ehip_attention_packed_workspace": C.c_int64,
             "ehip_attention_packed_backward_workspace": C.c_int64,
             "ehip_attention_paged_workspace": C.c_int64,
             "ehip_token_logprobs_workspace": C.c_int64, "ehip_kernels_launched": C.c_uint64,
             "ehip_conv2d_relu_maxpool_partials": C.c_int64,
             "ehip_layernorm_backward_partials": C.c_int64,
             "ehip_kernels_failed": C.c_uint64, "ehip_reset_counters": None,
             "ehip_fail_launch_after": None,
             "ehip_set_enabled": None, "ehip_transfer_stats": None,
             "ehip_reset_transfer_stats": None, "ehip_arena_free": None,
             "ehip_arena_stats": None}


def load_library(path=LIB_PATH):
    """Loads libehip.so and declares every entry point; no GPU needed."""
    if not os.path.exists(path):
        raise FileNotFoundError(f"{path} is not built: run __graft_entry__.build() or "
                                f"make -C cpp-ai-engine_amd")
    lib = C.CDLL(path)
    for name, args in _SIGS.items():
        fn = getattr(lib, name)
        fn.argtypes = args
        fn.restype = _RESTYPES.get(name, C.c_int)
    return lib


def header_symbols(path=HEADER):
    """Names of every function include/ehip.h declares."""
    import re
    text = open(path).read()
    return sorted(set(re.findall(r"^\s*(?:const char\*|int|void|uint64_t|int64_t)\s+(ehip_\w+)\(", text,
                                 re.M)))


class Backend:
    """The device ops over torch CUDA tensors. Raises if no gfx950 device."""

    def __init__(self, path=LIB_PATH):
        import torch
        self.torch = torch
        self.lib = load_library(path)
        rc = self.lib.ehip_init()
        if rc != 0:
            raise RuntimeError(f"ehip_init failed ({rc}): {self.error()}")

    # ---------------------------------------------------------- plumbing
    def error(self):
        return self.lib.ehip_last_error().decode()

    def ok(self, rc, what):
        if rc != 0:
            raise RuntimeError(f"{what} failed ({rc}): {self.error()}")

    def stream(self):
        cuda = self.torch.cuda  # the handle alone: making a Stream object of it takes 2.7 us
        return _vp(self.torch._C._cuda_getCurrentRawStream(cuda.current_device()))

    @staticmethod
    def p(t):
        if t is None:
            return None
        assert t.is_cuda and t.is_contiguous(), "device tensors must be contiguous on the GPU"
        return _vp(t.data_ptr())

    def f32(self, shape):
        return self.torch.empty(shape, dtype=self.torch.float32, device="cuda")

    def device_info(self):
        info = DeviceInfo()
        self.ok(self.lib.ehip_device_info(C.byref(info)), "device_info")
        return info

    def attention_short(self, q, k, v, heads, scale, causal):
        """q, k, v: (batch, seq, width) device tensors; returns (weights, out)."""
        b, s_, w = q.shape
        hd = w // heads
        weights, out = self.f32((b, heads, s_, s_)), self.f32((b, s_, w))
        self.ok(self.lib.ehip_attention_short_f32(self.p(q), self.p(k), self.p(v), self.p(weights),
                                                  self.p(out), b, s_, w, heads, hd, scale,
                                                  int(causal), self.stream()), "attention_short")
        return weights, out

    def attention_short_backward(self, q, k, v, weights, g, heads, scale, causal,
                                 want=(True, True, True)):
        b, s_, w = q.shape
        hd = w // heads
        outs = [self.f32((b, s_, w)) if x else None for x in want]
        self.ok(self.lib.ehip_attention_short_backward_f32(
            self.p(q), self.p(k), self.p(v), self.p(weights), self.p(g), self.p(outs[0]),
            self.p(outs[1]), self.p(outs[2]), b, s_, w, heads, hd, scale, int(causal),
            self.stream()), "attention_short_backward")
        return outs

    def gemm_probe_arm(self, trans_a, trans_b, shapes, max_products):
        """Arms the timing probe for batch-1 products with these transposes and (m, n, k)
        in `shapes`."""
        flat = (C.c_int64 * (3 * len(shapes)))(*[int(v) for s_ in shapes for v in s_])
        self.ok(self.lib.ehip_gemm_probe_arm(int(bool(trans_a)), int(bool(trans_b)), flat,
                                             len(shapes), int(max_products)), "gemm_probe_arm")

    def gemm_probe_read(self):
        """(ms, products, flop) of the probed products since arming; disarms."""
        ms, n, fl = C.c_double(0), C.c_int64(0), C.c_double(0)
        self.ok(self.lib.ehip_gemm_probe_read(C.byref(ms), C.byref(n), C.byref(fl)),
                "gemm_probe_read")
        return ms.value, n.value, fl.value

    def versions(self):
        v = [C.c_int(0) for _ in range(3)]
        self.ok(self.lib.ehip_version_info(*[C.byref(x) for x in v]), "version_info")
        return tuple(x.value for x in v)

    def kernel_occupancy(self):
        count = C.c_int(0)
        self.ok(self.lib.ehip_kernel_occupancy(None, 0, C.byref(count)), "kernel_occupancy")
        arr = (KernelOccupancy * max(count.value, 1))()
        self.ok(self.lib.ehip_kernel_occupancy(arr, count.value, C.byref(count)),
                "kernel_occupancy")
        return [arr[i] for i in range(count.value)]

    def launched(self):
        return self.lib.ehip_kernels_launched()

    def arena_stats(self):
        s = ArenaStats()
        self.lib.ehip_arena_stats(C.byref(s))
        return s

    # ---------------------------------------------------------- dense
    def gemm_ex(self, desc):
        """Runs an ehip_gemm_ex_t (a GemmEx whose pointers are device addresses)."""
        self.ok(self.lib.ehip_gemm_ex_f32(C.byref(desc), self.stream()), "gemm_ex")

    def linear_backward(self, x, w, dy, want=("dx", "dw", "db")):
        """(dx, dw, db) of y = x w + b through ehip_linear_backward_f32; parts not
        in `want` are None."""
        rows, inp = x.shape
        out = w.shape[1]
        dx = self.f32((rows, inp)) if "dx" in want else None
        dw = self.f32((inp, out)) if "dw" in want else None
        db = self.f32((out,)) if "db" in want else None
        self.ok(self.lib.ehip_linear_backward_f32(self.p(x), self.p(w), self.p(dy), self.p(dx),
                                                  self.p(dw), self.p(db), rows, inp, out,
                                                  self.stream()), "linear_backward")
        return dx, dw, db

    def gemm(self, a, b, c=None, trans_a=False, trans_b=False, beta=0.0):
        """c = op(a) op(b) + beta c; a, b 2-D or 3-D (batched), 2-D operands shared."""
        ab, bb = a.dim() == 3, b.dim() == 3
        batch = a.shape[0] if ab else (b.shape[0] if bb else 1)
        am, ak = a.shape[-2:]
        m, k = (ak, am) if trans_a else (am, ak)
        bk, bn = b.shape[-2:]
        kb, n = (bn, bk) if trans_b else (bk, bn)
        assert k == kb, (a.shape, b.shape, trans_a, trans_b)
        if c is None:
            c = self.f32((batch, m, n) if (ab or bb) else (m, n))
        self.ok(self.lib.ehip_gemm_f32(int(trans_a), int(trans_b), batch, m, n, k, self.p(a),
                                       a.shape[-1], am * ak if ab else 0, self.p(b), b.shape[-1],
                                       bk * bn if bb else 0, beta, self.p(c), n,
                                       m * n if (ab or bb) else 0, self.stream()), "gemm")
        return c

    # ---------------------------------------------------------- element-wise
    def binary(self, op, a, b, out=None):
        out = self.f32(a.shape) if out is None else out
        inner = b.numel()
        self.ok(self.lib.ehip_binary_f32(op, self.p(a), self.p(b), self.p(out), inner,
                                         a.numel() // inner, self.stream()), "binary")
        return out

    def scalar(self, x, mul, add):
        out = self.f32(x.shape)
        self.ok(self.lib.ehip_scalar_f32(self.p(x), self.p(out), x.numel(), mul, add,
                                         self.stream()), "scalar")
        return out

    def relu(self, x):
        y = self.f32(x.shape)
        self.ok(self.lib.ehip_relu_f32(self.p(x), self.p(y), x.numel(), self.stream()), "relu")
        return y

    def relu_backward(self, x, g, dx=None):
        dx = self.f32(x.shape) if dx is None else dx
        self.ok(self.lib.ehip_relu_backward_f32(self.p(x), self.p(g), self.p(dx), x.numel(),
                                                self.stream()), "relu_backward")
        return dx

    def accumulate_grad(self, grad, g, initialize):
        self.ok(self.lib.ehip_accumulate_grad_f32(self.p(grad), self.p(g), g.numel(),
                                                  int(initialize), self.stream()),
                "accumulate_grad")
        return grad

    def mul_backward(self, g, a, b, da=None, db=None, acc_a=False, acc_b=False):
        """da (+)= g * b, db (+)= g * a in one launch; None skips that gradient."""
        self.ok(self.lib.ehip_mul_backward_f32(self.p(g), self.p(a), self.p(b), self.p(da),
                                               self.p(db), g.numel(), int(acc_a), int(acc_b),
                                               self.stream()), "mul_backward")
        return da, db

    def add_backward(self, g, da, db, acc_a, acc_b):
        self.ok(self.lib.ehip_add_backward_f32(self.p(g), self.p(da), self.p(db), g.numel(),
                                               int(acc_a), int(acc_b), self.stream()),
                "add_backward")

    def fill(self, x, value):
        self.ok(self.lib.ehip_fill_f32(self.p(x), x.numel(), value, self.stream()), "fill")
        return x

    def scale(self, x, factor):
        self.ok(self.lib.ehip_scale_f32(self.p(x), x.numel(), factor, self.stream()), "scale")
        return x

    def sgd(self, p, g, vel, lr, momentum, wd):
        self.ok(self.lib.ehip_sgd_f32(self.p(p), self.p(g), self.p(vel), p.numel(), lr, momentum,
                                      wd, self.stream()), "sgd")

    def adam(self, p, g, m, v, lr, b1, b2, eps, wd, c1, c2):
        self.ok(self.lib.ehip_adam_f32(self.p(p), self.p(g), self.p(m), self.p(v), p.numel(), lr,
                                       b1, b2, eps, wd, c1, c2, self.stream()), "adam")

    def adam_multi(self, groups, lr, b1, b2, eps, wd, c1, c2):
        """groups: list of (p, g, m, v) device tensors."""
        arr = (AdamTensor * len(groups))(*[
            AdamTensor(p.data_ptr(), g.data_ptr(), m.data_ptr(), v.data_ptr(), p.numel())
            for p, g, m, v in groups])
        self.ok(self.lib.ehip_adam_multi_f32(arr, len(groups), lr, b1, b2, eps, wd, c1, c2,
                                             self.stream()), "adam_multi")

    def adam_multi_reduce(self, groups, jobs, lr, b1, b2, eps, wd, c1, c2):
        """groups: (p, g, m, v) device tensors; jobs: (partials, chunks, dweight, dbias) with
        dweight shaped (co, ...) -- the sums land in dweight / dbias first."""
        arr = (AdamTensor * len(groups))(*[
            AdamTensor(p.data_ptr(), g.data_ptr(), m.data_ptr(), v.data_ptr(), p.numel())
            for p, g, m, v in groups])
        jarr = (ConvReduce * len(jobs))()
        for i, (part, chunks, dw, db) in enumerate(jobs):
            jarr[i] = ConvReduce(self.p(part), chunks, dw.shape[0], dw.numel() // dw.shape[0],
                                 self.p(dw), self.p(db) if db is not None else None)
        self.ok(self.lib.ehip_adam_multi_reduce_f32(arr, len(groups), jarr, len(jobs), lr, b1, b2,
                                                    eps, wd, c1, c2, self.stream()),
                "adam_multi_reduce")

    # ---------------------------------------------------------- layout
    def permute(self, x, order):
        shape = list(x.shape)
        in_stride = [1] * len(shape)
        for d in range(len(shape) - 2, -1, -1):
            in_stride[d] = in_stride[d + 1] * shape[d + 1]
        out_shape = [shape[o] for o in order]
        src = [in_stride[o] for o in order]
        out = self.f32(out_shape)
        arr = C.c_int64 * len(shape)
        self.ok(self.lib.ehip_permute_f32(self.p(x), self.p(out), len(shape), arr(*out_shape),
                                          arr(*src), self.stream()), "permute")
        return out

    def transpose(self, x):
        rows, cols = x.shape[-2:]
        batch = x.numel() // max(1, rows * cols)
        out = self.f32(tuple(x.shape[:-2]) + (cols, rows))
        self.ok(self.lib.ehip_transpose_f32(self.p(x), self.p(out), batch, rows, cols,
                                            self.stream()), "transpose")
        return out

    def im2col(self, x, kh, kw, stride, pad):
        w = window(*x.shape, kh, kw, stride, pad)
        cols = self.f32((w.batch * w.out_h * w.out_w, w.channels * kh * kw))
        self.ok(self.lib.ehip_im2col_f32(self.p(x), self.p(cols), C.byref(w), self.stream()),
                "im2col")
        return cols

    def col2im(self, cols, shape, kh, kw, stride, pad):
        w = window(*shape, kh, kw, stride, pad)
        x = self.f32(shape)
        self.ok(self.lib.ehip_col2im_f32(self.p(cols), self.p(x), C.byref(w), self.stream()),
                "col2im")
        return x

    def maxpool(self, x, k, stride, pad=0, float_index=False, out=None):
        """float_index selects the float argmax layout of the reference's device path;
        out = (y, argmax) reuses preallocated outputs."""
        w = window(*x.shape, k, k, stride, pad)
        if out is not None:
            y, am = out
        else:
            y = self.f32((w.batch, w.channels, w.out_h, w.out_w))
            am = (self.f32(y.shape) if float_index else
                  self.torch.empty(y.shape, dtype=self.torch.int32, device="cuda"))
        if float_index:
            rc = self.lib.ehip_maxpool_fidx_f32(self.p(x), self.p(y), self.p(am), C.byref(w),
                                                self.stream())
        else:
            rc = self.lib.ehip_maxpool_f32(self.p(x), self.p(y), self.p(am), C.byref(w),
                                           self.stream())
        self.ok(rc, "maxpool")
        return y, am

    def maxpool_backward(self, argmax, g, in_shape, k, stride, pad=0, dx=None):
        """argmax as returned by maxpool: int32, or float32 for the float layout."""
        w = window(*in_shape, k, k, stride, pad)
        dx = self.f32(in_shape) if dx is None else dx
        f = (self.lib.ehip_maxpool_backward_fidx_f32 if argmax.dtype == self.torch.float32
             else self.lib.ehip_maxpool_backward_f32)
        self.ok(f(self.p(argmax), self.p(g), self.p(dx), C.byref(w), self.stream()),
                "maxpool_backward")
        return dx

    def conv2d(self, x, weight, bias, stride, pad):
        """Direct convolution, NCHW in and out; bias may be None."""
        co, ci, kh, kw = weight.shape
        w = window(*x.shape, kh, kw, stride, pad)
        out = self.f32((w.batch, co, w.out_h, w.out_w))
        self.ok(self.lib.ehip_conv2d_forward_f32(self.p(x), self.p(weight),
                                                 self.p(bias) if bias is not None else None,
                                                 self.p(out), C.byref(w), co, self.stream()),
                "conv2d_forward")
        return out

    def conv2d_backward_input(self, g, weight, in_shape, stride, pad):
        co, ci, kh, kw = weight.shape
        w = window(*in_shape, kh, kw, stride, pad)
        dx = self.f32(in_shape)
        self.ok(self.lib.ehip_conv2d_backward_input_f32(self.p(g), self.p(weight), self.p(dx),
                                                        C.byref(w), co, self.stream()),
                "conv2d_backward_input")
        return dx

    def conv2d_backward_weight(self, x, g, weight_shape, stride, pad, bias=True):
        co, ci, kh, kw = weight_shape
        w = window(*x.shape, kh, kw, stride, pad)
        dw = self.f32(weight_shape)
        db = self.f32((co,)) if bias else None
        self.ok(self.lib.ehip_conv2d_backward_weight_f32(
            self.p(x), self.p(g), self.p(dw), self.p(db) if bias else None, C.byref(w), co,
            self.stream()), "conv2d_backward_weight")
        return dw, db

    def conv2d_igemm(self, x, weight, bias, stride, pad):
        co, ci, kh, kw = weight.shape
        w = window(*x.shape, kh, kw, stride, pad)
        out = self.f32((w.batch, co, w.out_h, w.out_w))
        self.ok(self.lib.ehip_conv2d_igemm_f32(
            self.p(x), self.p(weight), self.p(bias) if bias is not None else None, self.p(out),
            C.byref(w), co, self.stream()), "conv2d_igemm")
        return out

    def conv2d_igemm_backward(self, x, weight, g, stride, pad, want=(True, True, True)):
        """(dx, dweight, dbias); the parts not in `want` are skipped and returned as None."""
        co, ci, kh, kw = weight.shape
        w = window(*x.shape, kh, kw, stride, pad)
        dx = self.f32(tuple(x.shape)) if want[0] else None
        dw = self.f32(tuple(weight.shape)) if want[1] else None
        db = self.f32((co,)) if want[2] else None
        self.ok(self.lib.ehip_conv2d_igemm_backward_f32(
            self.p(x), self.p(weight), self.p(g), self.p(dx) if want[0] else None,
            self.p(dw) if want[1] else None, self.p(db) if want[2] else None, C.byref(w), co,
            self.stream()), "conv2d_igemm_backward")
        return dx, dw, db

    def conv_relu_pool_windows(self, x_shape, weight_shape, stride, pad, pk):
        co, ci, kh, kw = weight_shape
        cw = window(*x_shape, kh, kw, stride, pad)
        pw = window(cw.batch, co, cw.out_h, cw.out_w, pk, pk, pk, 0)
        return cw, pw

    def conv2d_relu_maxpool(self, x, weight, bias, stride, pad, pk):
        """Fused Conv2d -> ReLU -> MaxPool2d(pk, pk); returns (pooled, argmax int32)."""
        cw, pw = self.conv_relu_pool_windows(x.shape, weight.shape, stride, pad, pk)
        co = weight.shape[0]
        out = self.f32((pw.batch, co, pw.out_h, pw.out_w))
        am = self.torch.empty(out.shape, dtype=self.torch.int32, device="cuda")
        self.ok(self.lib.ehip_conv2d_relu_maxpool_f32(
            self.p(x), self.p(weight), self.p(bias) if bias is not None else None, self.p(out),
            self.p(am), C.byref(cw), co, C.byref(pw), self.stream()), "conv2d_relu_maxpool")
        return out, am

    def conv2d_relu_maxpool_backward(self, x, weight, g, out, am, stride, pad, pk, need_dx=True,
                                     bias=True, need_dw=True):
        cw, pw = self.conv_relu_pool_windows(x.shape, weight.shape, stride, pad, pk)
        co = weight.shape[0]
        dx = self.f32(x.shape) if need_dx else None
        dw = self.f32(weight.shape) if need_dw else None
        db = self.f32((co,)) if bias and need_dw else None
        self.ok(self.lib.ehip_conv2d_relu_maxpool_backward_f32(
            self.p(x), self.p(weight), self.p(g), self.p(out), self.p(am),
            self.p(dx) if need_dx else None, self.p(dw) if need_dw else None,
            self.p(db) if db is not None else None,
            C.byref(cw), co, C.byref(pw), self.stream()), "conv2d_relu_maxpool_backward")
        return dx, dw, db

    def conv2d_relu_maxpool_partials(self, x, weight, g, out, am, stride, pad, pk,
                                     need_dx=True):
        """The tile kernel alone: returns (dx, partials, chunks), or None when the layer has
        no tile path."""
        cw, pw = self.conv_relu_pool_windows(x.shape, weight.shape, stride, pad, pk)
        co = weight.shape[0]
        chunks = C.c_int64(0)
        n = self.lib.ehip_conv2d_relu_maxpool_partials(C.byref(cw), co, C.byref(pw),
                                                       int(need_dx), C.byref(chunks))
        if n == 0:
            return None
        dx = self.f32(x.shape) if need_dx else None
        part = self.f32((n,))
        self.ok(self.lib.ehip_conv2d_relu_maxpool_backward_partials_f32(
            self.p(x), self.p(weight), self.p(g), self.p(out), self.p(am),
            self.p(dx) if need_dx else None, self.p(part), chunks.value, C.byref(cw), co,
            C.byref(pw), self.stream()), "conv2d_relu_maxpool_backward_partials")
        return dx, part, chunks.value

    def conv_weight_reduce(self, jobs):
        """jobs: (partials, chunks, weight_shape, with_bias) per layer; one launch. Returns
        [(dw, db)]."""
        arr = (ConvReduce * len(jobs))()
        outs = []
        for i, (part, chunks, wshape, with_bias) in enumerate(jobs):
            dw = self.f32(wshape)
            db = self.f32((wshape[0],)) if with_bias else None
            k = 1
            for d in wshape[1:]:
                k *= int(d)
            arr[i] = ConvReduce(self.p(part), chunks, wshape[0], k, self.p(dw),
                                self.p(db) if with_bias else None)
            outs.append((dw, db))
        self.ok(self.lib.ehip_conv_weight_reduce_f32(arr, len(jobs), self.stream()),
                "conv_weight_reduce")
        return outs

    def dropout(self, x, p, seed, offset=0, want_mask=True):
        y = self.f32(x.shape)
        m = self.f32(x.shape) if want_mask else None
        self.ok(self.lib.ehip_dropout_f32(self.p(x), self.p(y), self.p(m) if want_mask else None,
                                          x.numel(), p, seed, offset, self.stream()), "dropout")
        return y, m

    def select_rows(self, x, idx):
        rs = x.numel() // x.shape[0]
        out = self.f32((idx.numel(),) + tuple(x.shape[1:]))
        self.ok(self.lib.ehip_select_rows_f32(self.p(x), self.p(idx), self.p(out), idx.numel(),
                                              rs, x.shape[0], self.stream()), "select_rows")
        return out

    def scatter_add_rows(self, g, row_ptr, pos, dx, accumulate=False):
        rs = dx.numel() // dx.shape[0]
        self.ok(self.lib.ehip_scatter_add_rows_f32(self.p(g), self.p(row_ptr), self.p(pos),
                                                   self.p(dx), dx.shape[0], rs, g.shape[0],
                                                   int(accumulate), self.stream()),
                "scatter_add_rows")
        return dx

    # ---------------------------------------------------------- reductions
    def sum_axis(self, x, outer, axis_len, inner):
        out = self.f32((outer * inner,))
        self.ok(self.lib.ehip_sum_axis_f32(self.p(x), self.p(out), outer, axis_len, inner,
                                           self.stream()), "sum_axis")
        return out

    def reduce_sum(self, x, squares=False):
        d = self.torch.empty(1, dtype=self.torch.float64, device="cuda")
        f = self.f32((1,))
        self.ok(self.lib.ehip_reduce_sum_f32(self.p(x), x.numel(), int(squares), self.p(d),
                                             self.p(f), self.stream()), "reduce_sum")
        return d, f

    # ---------------------------------------------------------- rows
    def softmax(self, x):
        cols = x.shape[-1]
        y = self.f32(x.shape)
        self.ok(self.lib.ehip_softmax_f32(self.p(x), self.p(y), x.numel() // cols, cols,
                                          self.stream()), "softmax")
        return y

    def softmax_backward(self, y, g, scale=None, out=None):
        """dx = y (g - sum(g y)), times `scale` when given (the scaled entry point);
        `out` may be g itself."""
        cols = y.shape[-1]
        dx = self.f32(y.shape) if out is None else out
        if scale is None:
            rc = self.lib.ehip_softmax_backward_f32(self.p(y), self.p(g), self.p(dx),
                                                    y.numel() // cols, cols, self.stream())
        else:
            rc = self.lib.ehip_softmax_backward_scaled_f32(self.p(y), self.p(g), self.p(dx),
                                                           y.numel() // cols, cols, scale,
                                                           self.stream())
        self.ok(rc, "softmax_backward")
        return dx

    def layernorm(self, x, gamma, beta, eps=1e-5):
        d = x.shape[-1]
        rows = x.numel() // d
        out, xhat, inv = self.f32(x.shape), self.f32(x.shape), self.f32((rows,))
        self.ok(self.lib.ehip_layernorm_f32(self.p(x), self.p(gamma), self.p(beta), self.p(out),
                                            self.p(xhat), self.p(inv), rows, d, eps,
                                            self.stream()), "layernorm")
        return out, xhat, inv

    def layernorm_backward(self, dy, xhat, gamma, inv):
        d = dy.shape[-1]
        dx, dg, db = self.f32(dy.shape), self.f32((d,)), self.f32((d,))
        self.ok(self.lib.ehip_layernorm_backward_f32(self.p(dy), self.p(xhat), self.p(gamma),
                                                     self.p(inv), self.p(dx), self.p(dg),
                                                     self.p(db), dy.numel() // d, d,
                                                     self.stream()), "layernorm_backward")
        return dx, dg, db

    def layernorm_backward_partials(self, dy, xhat, gamma, inv, groups=None, dx=None):
        """dx and the per-group dgamma / dbeta partials ([groups][d][2]) of the deferred
        LayerNorm backward; returns (dx, partials, groups), or None when the shape is summed
        in one call only. `groups` overrides the count (to test the refusal); a given `dx`
        receives dx + the input gradient (accumulate)."""
        d = dy.shape[-1]
        rows = dy.numel() // d
        g = _i64(0)
        n = self.lib.ehip_layernorm_backward_partials(rows, d, C.byref(g))
        if n == 0 and groups is None:
            return None
        acc = dx is not None
        dx = dx if acc else self.f32(dy.shape)
        part = self.f32((max(n, 1),))
        use = g.value if groups is None else groups
        self.ok(self.lib.ehip_layernorm_backward_partials_f32(
            self.p(dy), self.p(xhat), self.p(gamma), self.p(inv), self.p(dx), self.p(part), use,
            rows, d, int(acc), self.stream()), "layernorm_backward_partials")
        return dx, part, g.value

    def cross_entropy(self, logits, targets):
        rows, cols = logits.shape
        probs, loss = self.f32(logits.shape), self.f32((1,))
        self.ok(self.lib.ehip_cross_entropy_f32(self.p(logits), self.p(targets), self.p(probs),
                                                self.p(loss), rows, cols, self.stream()),
                "cross_entropy")
        return loss, probs

    def cross_entropy_fused(self, logits, targets):
        """Forward plus the logits' gradient for an upstream gradient of 1 in one launch;
        returns (loss, probs, dlogits)."""
        rows, cols = logits.shape
        probs, loss, dl = self.f32(logits.shape), self.f32((1,)), self.f32(logits.shape)
        self.ok(self.lib.ehip_cross_entropy_fused_f32(self.p(logits), self.p(targets),
                                                      self.p(probs), self.p(loss), self.p(dl),
                                                      rows, cols, self.stream()),
                "cross_entropy_fused")
        return loss, probs, dl

    def cross_entropy_backward(self, probs, targets, grad):
        rows, cols = probs.shape
        dx = self.f32(probs.shape)
        self.ok(self.lib.ehip_cross_entropy_backward_f32(self.p(probs), self.p(targets),
                                                         self.p(dx), rows, cols, self.p(grad),
                                                         self.stream()), "cross_entropy_backward")
        return dx

    def softmax_xent_backward(self, logits, targets, grad, dx=None):
        rows, cols = logits.shape
        dx = self.f32(logits.shape) if dx is None else dx
        self.ok(self.lib.ehip_softmax_xent_backward_f32(self.p(logits), self.p(targets),
                                                        self.p(dx), rows, cols, self.p(grad),
                                                        self.stream()), "softmax_xent_backward")
        return dx

    # ------------------------------ packed sequences, a cache, token scores
    def _here(self, *tensors):
        """Refuses tensors that are not all on the current device (whose stream is used)."""
        index = self.torch.cuda.current_device()
        for t in tensors:
            if t is not None and not (t.is_cuda and t.device.index == index):
                raise ValueError(f"tensor on {t.device}, the current device is cuda:{index}")

    def _rows(self, t, what, shape, dtype=None):
        """The row pitch of a float32 tensor of this shape whose rows are dense (a column
        range of a wider matrix may be passed), checked."""
        if t.dtype != (dtype or self.torch.float32) or t.shape != shape:
            raise ValueError(f"{what}: {t.dtype} {tuple(t.shape)}, expected "
                             f"{dtype or self.torch.float32} {tuple(shape)}")
        if t.is_contiguous() and t.shape[0] > 1:
            return t.stride(0)
        row = 1
        for n, stride in zip(reversed(t.shape[1:]), reversed(t.stride()[1:])):
            if n != 1 and stride != row:
                raise ValueError(f"{what}: rows must be dense, strides are {t.stride()}")
            row *= n
        if t.shape[0] <= 1 or t.numel() == 0:
            return row
        if t.stride(0) < row:
            raise ValueError(f"{what}: rows overlap, strides are {t.stride()}")
        return t.stride(0)

    def _index(self, t, what, *shape):
        if t.dtype != self.torch.int32 or t.shape != shape or not t.is_contiguous():
            raise ValueError(f"{what}: {t.dtype} {tuple(t.shape)}, expected contiguous int32 "
                             f"{shape}")
        return _vp(t.data_ptr())

    def _workspace(self, n, what):
        """(tensor, pointer, bytes) of a call's own workspace of n bytes."""
        if n < 0:
            raise RuntimeError(f"{what} failed: {self.error()}")
        if n == 0:
            return None, None, 0
        w = self.torch.empty(n, dtype=self.torch.uint8, device="cuda")
        return w, _vp(w.data_ptr()), n

    def _packed(self, q, k, v, cu_q, cu_k, scale, causal, out, lse, longest_q=None,
                longest_k=None):
        if q.dim() != 3 or k.dim() != 3:
            raise ValueError("q and k: expected (tokens, heads, head_dim)")
        self._here(q, k, v, cu_q, cu_k, out, lse)
        (tq, h, d), (tk, kv) = q.shape, k.shape[:2]
        if cu_k is None:
            cu_k, longest_k = cu_q, longest_k or longest_q
        sequences = cu_q.numel() - 1
        if sequences < 0:
            raise ValueError("cu_q: expected one offset more than sequences")
        return AttentionPacked(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), self._rows(q, "q", (tq, h, d)),
            self._rows(k, "k", (tk, kv, d)), self._rows(v, "v", (tk, kv, d)),
            self._index(cu_q, "cu_q", sequences + 1), self._index(cu_k, "cu_k", sequences + 1),
            sequences, tq, tk, h, kv, d, d ** -0.5 if scale is None else scale, int(causal),
            out.data_ptr(), self._rows(out, "out", (tq, h, d)), self._dense(lse, "lse", (tq, h)),
            longest_q or 0, longest_k or 0)

    def _dense(self, t, what, shape):
        if t.dtype != self.torch.float32 or t.shape != shape or not t.is_contiguous():
            raise ValueError(f"{what}: {t.dtype} {tuple(t.shape)}, expected contiguous float32 "
                             f"{tuple(shape)}")
        return t.data_ptr()

    def attention_packed(self, q, k, v, cu_q, cu_k=None, scale=None, causal=True, out=None,
                         lse=None, longest_q=None, longest_k=None):
        """Attention over packed sequences (ehip_attention_packed_f32): q (total_q, heads,
        head_dim), k and v (total_k, kv_heads, head_dim), column ranges of a fused projection
        allowed; cu_q, cu_k int32 offsets of the sequences on the device (cu_k: cu_q). scale:
        head_dim ** -0.5. longest_q, longest_k: rows of the longest sequence, where known, for
        batches of one long and many short or empty ones. Returns (out, lse (total_q, heads)),
        written into `out` and `lse` where given."""
        out = self.f32(q.shape) if out is None else out
        lse = self.f32(q.shape[:2]) if lse is None else lse
        desc = self._packed(q, k, v, cu_q, cu_k, scale, causal, out, lse, longest_q, longest_k)
        need = self.lib.ehip_attention_packed_workspace(C.byref(desc))
        space, at, n = self._workspace(need, "attention_packed")
        self.ok(self.lib.ehip_attention_packed_f32(C.byref(desc), at, n, self.stream()),
                "attention_packed")
        return out, lse

    def attention_packed_backward(self, g, q, k, v, out, lse, cu_q, cu_k=None, scale=None,
                                  causal=True, want=(True, True, True), grads=None,
                                  longest_q=None, longest_k=None):
        """(dq, dk, dv) of attention_packed from its out and lse; None where `want` says so.
        `grads`: tensors to write them into (rows may be column ranges)."""
        desc = self._packed(q, k, v, cu_q, cu_k, scale, causal, out, lse, longest_q, longest_k)
        if grads is None:
            grads = [self.f32(t.shape) if w else None for t, w in zip((q, k, v), want)]
        self._here(g, *grads)
        args = []
        for t, like, what in zip(grads, (q, k, v), ("dq", "dk", "dv")):
            args += [None, 0] if t is None else [_vp(t.data_ptr()),
                                                 self._rows(t, what, like.shape)]
        need = self.lib.ehip_attention_packed_backward_workspace(C.byref(desc))
        space, at, n = self._workspace(need, "attention_packed_backward")
        self.ok(self.lib.ehip_attention_packed_backward_f32(
            C.byref(desc), _vp(g.data_ptr()), self._rows(g, "g", q.shape), *args, at, n,
            self.stream()), "attention_packed_backward")
        return grads

    def _cache(self, k_pages, v_pages, table):
        self._here(k_pages, v_pages, table)
        if k_pages.dim() != 4 or k_pages.dtype not in (self.torch.float32, self.torch.bfloat16):
            raise ValueError("k_pages: expected float32 or bfloat16 (pages, page_size, kv_heads, "
                             "head_dim)")
        if (v_pages.shape != k_pages.shape or v_pages.dtype != k_pages.dtype
                or not k_pages.is_contiguous() or not v_pages.is_contiguous()):
            raise ValueError("k_pages, v_pages: expected contiguous pools of one shape and type")
        if table.dim() != 2:
            raise ValueError("table: expected (sequences, pages of the longest)")
        pages, size, kv, d = k_pages.shape
        return Cache(k_pages.data_ptr(), v_pages.data_ptr(),
                     int(k_pages.dtype == self.torch.bfloat16), pages, size, kv, d,
                     table.data_ptr(), self._rows(table, "table", table.shape, self.torch.int32),
                     table.shape[1], table.shape[0])

    def cache_append(self, k, v, k_pages, v_pages, table, starts, cu=None):
        """Writes tokens' keys and values (tokens, kv_heads, head_dim) into the pools
        (pages, page_size, kv_heads, head_dim; float32 or bfloat16) at positions starts[s],
        starts[s] + 1, ... of each sequence (ehip_cache_append_f32). cu: int32 offsets of the
        sequences' tokens, None for one token each."""
        cache = self._cache(k_pages, v_pages, table)
        self._here(k, v, starts, cu)
        tokens = k.shape[0]
        if cu is None and tokens != cache.sequences:
            raise ValueError(f"k: {tokens} tokens for {cache.sequences} sequences without cu")
        shape = (tokens,) + tuple(k_pages.shape[2:])
        self.ok(self.lib.ehip_cache_append_f32(
            C.byref(cache), _vp(k.data_ptr()), self._rows(k, "k", shape), _vp(v.data_ptr()),
            self._rows(v, "v", shape), self._index(starts, "starts", cache.sequences),
            None if cu is None else self._index(cu, "cu", cache.sequences + 1), tokens,
            self.stream()), "cache_append")

    def attention_paged(self, q, k_pages, v_pages, table, lengths, longest=None, scale=None,
                        out=None, lse=None):
        """Attention of one new token per sequence over a paged cache
        (ehip_attention_paged_f32): q (sequences, heads, head_dim); table int32 (sequences,
        pages); lengths int32, at most `longest` (None: what the table holds). Returns
        (out, lse (sequences, heads)), written into `out` and `lse` where given."""
        if q.dim() != 3:
            raise ValueError("q: expected (sequences, heads, head_dim)")
        cache = self._cache(k_pages, v_pages, table)
        out = self.f32(q.shape) if out is None else out
        lse = self.f32(q.shape[:2]) if lse is None else lse
        self._here(q, lengths, out, lse)
        n, h, d = cache.sequences, q.shape[1], cache.head_dim
        if longest is None:
            longest = cache.table_width * cache.page_size
        need = self.lib.ehip_attention_paged_workspace(C.byref(cache), h, longest)
        space, at, size = self._workspace(need, "attention_paged")
        self.ok(self.lib.ehip_attention_paged_f32(
            C.byref(cache), _vp(q.data_ptr()), self._rows(q, "q", (n, h, d)), h,
            self._index(lengths, "lengths", n), longest, d ** -0.5 if scale is None else scale,
            _vp(out.data_ptr()), self._rows(out, "out", (n, h, d)),
            _vp(self._dense(lse, "lse", (n, h))), at, size, self.stream()), "attention_paged")
        return out, lse

    def token_logprobs(self, logits, targets=None, top=0, want_entropy=True):
        """Per row of logits (rows, vocab): (logprob of the int32 target, entropy, lse, the
        `top` largest log probabilities, their int32 indices) (ehip_token_logprobs_f32); None
        for what was not asked for."""
        torch = self.torch
        if logits.dim() != 2:
            raise ValueError("logits: expected (rows, vocab)")
        self._here(logits, targets)
        rows, vocab = logits.shape
        ld = self._rows(logits, "logits", (rows, vocab))
        lse = self.f32((rows,))
        logprob = None if targets is None else self.f32((rows,))
        entropy = self.f32((rows,)) if want_entropy else None
        best = self.f32((rows, top)) if top else None
        index = torch.empty((rows, top), dtype=torch.int32, device="cuda") if top else None
        need = self.lib.ehip_token_logprobs_workspace(rows, vocab, top)
        space, at, size = self._workspace(need, "token_logprobs")
        self.ok(self.lib.ehip_token_logprobs_f32(
            _vp(logits.data_ptr()), ld,
            None if targets is None else self._index(targets, "targets", rows), rows, vocab,
            self.p(logprob), self.p(entropy), self.p(lse), top, self.p(best), self.p(index), at,
            size, self.stream()), "token_logprobs")
        return logprob, entropy, lse, best, index

    def token_logprobs_backward(self, logits, targets, lse, entropy, g_logprob, g_entropy=None,
                                dlogits=None):
        """The logits' gradient from those of logprob and entropy and token_logprobs' lse and
        entropy; `dlogits` may be `logits` itself."""
        if logits.dim() != 2:
            raise ValueError("logits: expected (rows, vocab)")
        dlogits = self.f32(logits.shape) if dlogits is None else dlogits
        entropy = None if g_entropy is None else entropy
        self._here(logits, targets, lse, entropy, g_logprob, g_entropy, dlogits)
        rows, vocab = logits.shape
        part = lambda t, what: None if t is None else _vp(self._dense(t, what, (rows,)))
        self.ok(self.lib.ehip_token_logprobs_backward_f32(
            _vp(logits.data_ptr()), self._rows(logits, "logits", (rows, vocab)),
            self._index(targets, "targets", rows), part(lse, "lse"), part(entropy, "entropy"),
            part(g_logprob, "g_logprob"), part(g_entropy, "g_entropy"), _vp(dlogits.data_ptr()),
            self._rows(dlogits, "dlogits", (rows, vocab)), rows, vocab, self.stream()),
            "token_logprobs_backward")
        return dlogits
