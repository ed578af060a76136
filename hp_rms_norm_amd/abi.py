"""ctypes binding of the C ABI of ``libhprms.so`` (include/hp_rms_norm_amd.h).

This is the binding a caller without the torch extension would use; the
tests use it to drive the kernels through the C ABI directly.  ``BENCH`` binds
the same ABI in the bench library ``libhprms_bench.so``, which bench.py and
the tuning tests load for the kernel shapes no table row selects.  Device
pointers and streams are plain integers (e.g. ``tensor.data_ptr()`` and
``torch.cuda.current_stream().cuda_stream``).
"""
import ctypes
import os

_HERE = os.path.dirname(os.path.abspath(__file__))
KERNEL_LIB = os.path.join(_HERE, "libhprms.so")
BENCH_LIB = os.path.join(_HERE, "libhprms_bench.so")  # bench and tests only, never the product path

HPRMS_OK = 0
HPRMS_E_INVALID = -22
HPRMS_E_LAUNCH = -5
HPRMS_E_RANGE = -34
DTYPE_BF16, DTYPE_FP16, DTYPE_FP32 = 0, 1, 2  # FP32: gradients and logits only
STREAM_COPY, STREAM_RELU = 0, 1
MAX_PARTS = 8
# the `mode` numbering of hprms_select_config / hprms_kernel_configs
MODE_FUSED, MODE_PLAIN, MODE_FP8, MODE_OUT, MODE_REDUCE, MODE_MXFP8, MODE_MXFP4, MODE_FP8_GROUP = 0, 1, 2, 3, 4, 5, 6, 7
MX_FP8_E4M3, MX_FP4_E2M1 = 0, 1

# every symbol the header declares
SYMBOLS = (
    "hprms_fused_add_rmsnorm",
    "hprms_fused_add_rmsnorm_fp8",
    "hprms_fused_add_rmsnorm_fp8_static",
    "hprms_fused_add_rmsnorm_fp8_group",
    "hprms_fused_add_rmsnorm_fp8_ub",
    "hprms_fused_add_rmsnorm_out",
    "hprms_reduce_add_rmsnorm",
    "hprms_fused_add_rmsnorm_mx",
    "hprms_streamer",
    "hprms_rmsnorm",
    "hprms_rmsnorm_backward_workspace",
    "hprms_rmsnorm_backward",
    "hprms_linear_cross_entropy_workspace",
    "hprms_linear_cross_entropy",
    "hprms_linear_cross_entropy_backward_workspace",
    "hprms_linear_cross_entropy_backward",
    "hprms_grad_norm_workspace",
    "hprms_grad_norm",
    "hprms_clip_grad_norm",
    "hprms_norm_add_rmsnorm",
    "hprms_norm_add_rmsnorm_int8",
    "hprms_norm_add_rmsnorm_backward_workspace",
    "hprms_norm_add_rmsnorm_backward",
    "hprms_int8_linear_workspace",
    "hprms_int8_linear",
    "hprms_token_log_probs_workspace",
    "hprms_token_log_probs",
    "hprms_token_log_probs_backward",
    "hprms_fused_add_rmsnorm_config",
    "hprms_select_config",
    "hprms_select_config_cu",
    "hprms_device_cu_count",
    "hprms_set_batch_invariant",
    "hprms_batch_invariant",
    "hprms_kernel_configs",
    "hprms_last_error",
    "hprms_abi_version",
)


class Config(ctypes.Structure):
    _fields_ = [("tier", ctypes.c_int32), ("lanes_per_row", ctypes.c_int32),
                ("vec_per_lane", ctypes.c_int32), ("lds_vec_per_lane", ctypes.c_int32),
                ("block_threads", ctypes.c_int32), ("grid_blocks", ctypes.c_int32),
                ("flags", ctypes.c_int32)]

    def as_tuple(self):
        return tuple(getattr(self, f) for f, _ in self._fields_)


class HprmsError(RuntimeError):
    def __init__(self, code, msg):
        super().__init__(f"{msg} (status {code})")
        self.code = code


def _bind(L, bench):
    vp, i64, ci, cd = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_double
    L.hprms_fused_add_rmsnorm.argtypes = [vp, vp, vp, i64, i64, i64, i64, ci, cd, vp]
    L.hprms_fused_add_rmsnorm_config.argtypes = [vp, vp, vp, i64, i64, i64, i64, ci, cd,
                                                 ctypes.POINTER(Config), vp]
    L.hprms_rmsnorm.argtypes = [vp, vp, vp, i64, i64, i64, i64, ci, cd, vp]
    L.hprms_fused_add_rmsnorm_fp8.argtypes = [vp, vp, vp, vp, vp, i64, i64, i64, i64, i64, ci, cd, vp]
    L.hprms_fused_add_rmsnorm_fp8_static.argtypes = [vp, vp, vp, vp, vp, i64, i64, i64, i64, i64, ci, cd, vp]
    L.hprms_fused_add_rmsnorm_fp8_ub.argtypes = [vp, vp, vp, vp, vp, vp, i64, i64, i64, i64, i64, ci, cd, vp]
    L.hprms_fused_add_rmsnorm_fp8_group.argtypes = [vp, vp, vp, vp, vp, i64, i64, i64, i64, i64, i64, i64, ci, cd,
                                                    vp]
    L.hprms_fused_add_rmsnorm_out.argtypes = [vp, vp, vp, vp, vp, i64, i64, i64, i64, i64, i64, ci, cd, vp]
    L.hprms_reduce_add_rmsnorm.argtypes = [vp, ctypes.POINTER(vp), ci, vp, vp, i64, i64, i64, i64, i64, ci,
                                           cd, vp]
    L.hprms_fused_add_rmsnorm_mx.argtypes = [vp, vp, vp, vp, vp, i64, i64, i64, i64, i64, i64, ci, ci, cd, vp]
    pvp, pi64, pci = ctypes.POINTER(vp), ctypes.POINTER(i64), ctypes.POINTER(ci)
    L.hprms_rmsnorm_backward_workspace.argtypes = [i64, i64]
    L.hprms_rmsnorm_backward.argtypes = [vp] * 7 + [i64] * 7 + [ci, ci, cd, vp]
    L.hprms_linear_cross_entropy_workspace.argtypes = [i64, i64, i64, vp, i64]
    L.hprms_linear_cross_entropy.argtypes = [vp] * 6 + [i64] * 7 + [ci, vp]
    L.hprms_linear_cross_entropy_backward_workspace.argtypes = [i64, i64, i64, vp, i64]
    L.hprms_linear_cross_entropy_backward.argtypes = [vp] * 8 + [i64] * 9 + [ci, vp]
    L.hprms_grad_norm_workspace.argtypes = [pi64, ci]
    L.hprms_grad_norm.argtypes = [vp, pvp, pci, pi64, ci, vp, i64, vp]
    L.hprms_clip_grad_norm.argtypes = [vp, pvp, pci, pvp, pci, pi64, ci, cd, vp, i64, vp]
    L.hprms_norm_add_rmsnorm.argtypes = [vp] * 7 + [i64] * 8 + [ci, cd, cd, vp]
    L.hprms_norm_add_rmsnorm_int8.argtypes = [vp] * 8 + [i64] * 8 + [ci, cd, cd, vp]
    L.hprms_norm_add_rmsnorm_backward_workspace.argtypes = [i64] * 3
    L.hprms_norm_add_rmsnorm_backward.argtypes = [vp] * 13 + [i64] * 12 + [ci] * 3 + [cd, cd, vp]
    L.hprms_int8_linear_workspace.argtypes = [i64] * 3 + [vp, i64, vp, i64]
    L.hprms_int8_linear.argtypes = [vp] * 7 + [i64] * 7 + [ci, vp]
    L.hprms_token_log_probs_workspace.argtypes = [i64] * 3 + [ci]
    L.hprms_token_log_probs.argtypes = [vp] * 8 + [i64] * 6 + [ci, vp]
    L.hprms_token_log_probs_backward.argtypes = [vp] * 7 + [i64] * 5 + [ci, vp]
    for name in ("hprms_rmsnorm_backward_workspace", "hprms_linear_cross_entropy_workspace",
                 "hprms_linear_cross_entropy_backward_workspace", "hprms_grad_norm_workspace",
                 "hprms_norm_add_rmsnorm_backward_workspace", "hprms_int8_linear_workspace",
                 "hprms_token_log_probs_workspace"):
        getattr(L, name).restype = i64
    L.hprms_streamer.argtypes = [vp, vp, i64, i64, i64, i64, ci, ci, vp]
    L.hprms_select_config.argtypes = [i64, i64, ci, ci, ctypes.POINTER(Config)]
    L.hprms_select_config_cu.argtypes = [i64, i64, ci, ci, ci, ctypes.POINTER(Config)]
    L.hprms_device_cu_count.argtypes = [ci]
    L.hprms_set_batch_invariant.argtypes = [ci]
    L.hprms_batch_invariant.argtypes = []
    L.hprms_kernel_configs.argtypes = [ci, ci, ctypes.POINTER(Config), ci]
    L.hprms_last_error.restype = ctypes.c_char_p
    L.hprms_last_error.argtypes = []
    L.hprms_abi_version.restype = ci
    names = ["hprms_fused_add_rmsnorm", "hprms_fused_add_rmsnorm_config", "hprms_rmsnorm",
             "hprms_fused_add_rmsnorm_fp8", "hprms_fused_add_rmsnorm_fp8_static", "hprms_fused_add_rmsnorm_fp8_group",
             "hprms_fused_add_rmsnorm_fp8_ub",
             "hprms_fused_add_rmsnorm_out",
             "hprms_reduce_add_rmsnorm",
             "hprms_fused_add_rmsnorm_mx", "hprms_rmsnorm_backward", "hprms_linear_cross_entropy",
             "hprms_linear_cross_entropy_backward", "hprms_grad_norm", "hprms_clip_grad_norm",
             "hprms_norm_add_rmsnorm", "hprms_norm_add_rmsnorm_int8", "hprms_norm_add_rmsnorm_backward",
             "hprms_int8_linear", "hprms_token_log_probs", "hprms_token_log_probs_backward", "hprms_streamer", "hprms_select_config", "hprms_select_config_cu",
             "hprms_device_cu_count", "hprms_kernel_configs", "hprms_set_batch_invariant", "hprms_batch_invariant"]
    if bench:
        L.hprms_bench_fused_timeline.argtypes = [vp, vp, vp, i64, i64, ci, cd, ctypes.POINTER(Config), vp, vp]
        L.hprms_ceil_empty.argtypes = [i64, ci, vp]
        L.hprms_ceil_read.argtypes = [vp, vp, i64, vp, vp]
        L.hprms_ceil_write.argtypes = [vp, vp, i64, vp]
        L.hprms_ceil_copy.argtypes = [vp, vp, i64, vp]
        L.hprms_ceil_skeleton.argtypes = [vp, vp, i64, i64, ci, ci, ci, ci, vp]
        L.hprms_ceil_streams.argtypes = [ci, vp, vp, vp, vp, i64, vp]
        L.hprms_ceil_flat.argtypes = [ci, ci, ci, ci, vp, vp, i64, vp]
        L.hprms_bench_form_config.argtypes = [ci, vp, vp, i64, i64, vp, vp, vp, i64, i64, ci, cd,
                                              ctypes.POINTER(Config), vp]
        names += ["hprms_bench_fused_timeline", "hprms_bench_form_config", "hprms_ceil_empty", "hprms_ceil_read", "hprms_ceil_write",
                  "hprms_ceil_copy", "hprms_ceil_skeleton", "hprms_ceil_streams", "hprms_ceil_flat"]
    for name in names:
        getattr(L, name).restype = ci


class Library:
    """One build of the C ABI: the product ``libhprms.so`` or the bench
    library ``libhprms_bench.so`` (the same entry points, the tuning-only
    kernel shapes, and the ceiling and timeline entry points)."""

    def __init__(self, path, bench=False):
        self.path = path
        self.bench = bench
        self._L = None

    def lib(self):
        """Load the library.  When torch is importable it is imported first,
        so that the library binds to the HIP runtime torch already loaded."""
        if self._L is None:
            try:
                import torch  # noqa: F401
            except ImportError:
                pass
            if not os.path.exists(self.path):
                raise ImportError(f"{self.path} not built: run `python hp_rms_norm_amd/build.py`")
            L = ctypes.CDLL(self.path)
            _bind(L, self.bench)
            self._L = L
        return self._L

    def last_error(self):
        return self.lib().hprms_last_error().decode()

    def _check(self, rc):
        if rc != HPRMS_OK:
            raise HprmsError(rc, self.last_error())
        return rc

    def fused_add_rmsnorm(self, input_ptr, weight_ptr, residual_ptr, rows, hidden, input_stride, residual_stride,
                          dtype, eps, stream=0, config=None):
        L = self.lib()
        if config is None:
            return self._check(L.hprms_fused_add_rmsnorm(input_ptr, weight_ptr, residual_ptr, rows, hidden,
                                                         input_stride, residual_stride, dtype, eps, stream))
        return self._check(L.hprms_fused_add_rmsnorm_config(input_ptr, weight_ptr, residual_ptr, rows, hidden,
                                                            input_stride, residual_stride, dtype, eps,
                                                            ctypes.byref(config), stream))

    def fused_add_rmsnorm_fp8(self, out_ptr, scale_ptr, input_ptr, weight_ptr, residual_ptr, rows, hidden,
                              out_stride, input_stride, residual_stride, dtype, eps, stream=0):
        return self._check(self.lib().hprms_fused_add_rmsnorm_fp8(out_ptr, scale_ptr, input_ptr, weight_ptr,
                                                                  residual_ptr, rows, hidden, out_stride,
                                                                  input_stride, residual_stride, dtype, eps, stream))

    def fused_add_rmsnorm_fp8_static(self, out_ptr, scale_ptr, input_ptr, weight_ptr, residual_ptr, rows, hidden,
                                     out_stride, input_stride, residual_stride, dtype, eps, stream=0):
        return self._check(self.lib().hprms_fused_add_rmsnorm_fp8_static(
            out_ptr, scale_ptr, input_ptr, weight_ptr, residual_ptr, rows, hidden, out_stride, input_stride,
            residual_stride, dtype, eps, stream))

    def fused_add_rmsnorm_fp8_ub(self, out_ptr, scale_ptr, scale_ub_ptr, input_ptr, weight_ptr, residual_ptr, rows,
                                 hidden, out_stride, input_stride, residual_stride, dtype, eps, stream=0):
        return self._check(self.lib().hprms_fused_add_rmsnorm_fp8_ub(
            out_ptr, scale_ptr, scale_ub_ptr, input_ptr, weight_ptr, residual_ptr, rows, hidden, out_stride,
            input_stride, residual_stride, dtype, eps, stream))

    def fused_add_rmsnorm_fp8_group(self, out_ptr, scales_ptr, input_ptr, weight_ptr, residual_ptr, rows, hidden,
                                    out_stride, scale_stride, scale_group_stride, input_stride, residual_stride,
                                    dtype, eps, stream=0):
        return self._check(self.lib().hprms_fused_add_rmsnorm_fp8_group(
            out_ptr, scales_ptr, input_ptr, weight_ptr, residual_ptr, rows, hidden, out_stride, scale_stride,
            scale_group_stride, input_stride, residual_stride, dtype, eps, stream))

    def fused_add_rmsnorm_out(self, out_ptr, residual_out_ptr, input_ptr, residual_ptr, weight_ptr, rows, hidden,
                              out_stride, residual_out_stride, input_stride, residual_stride, dtype, eps, stream=0):
        return self._check(self.lib().hprms_fused_add_rmsnorm_out(out_ptr, residual_out_ptr, input_ptr,
                                                                  residual_ptr, weight_ptr, rows, hidden, out_stride,
                                                                  residual_out_stride, input_stride, residual_stride,
                                                                  dtype, eps, stream))

    def reduce_add_rmsnorm(self, out_ptr, part_ptrs, weight_ptr, residual_ptr, rows, hidden, out_stride,
                           part_stride, residual_stride, dtype, eps, stream=0):
        """``part_ptrs``: a sequence of device pointers (1 ... MAX_PARTS); a
        ``None`` sequence passes a null array."""
        arr = None if part_ptrs is None else (ctypes.c_void_p * max(1, len(part_ptrs)))(*part_ptrs)
        n = 0 if part_ptrs is None else len(part_ptrs)
        return self._check(self.lib().hprms_reduce_add_rmsnorm(out_ptr, arr, n, weight_ptr, residual_ptr, rows,
                                                               hidden, out_stride, part_stride, residual_stride,
                                                               dtype, eps, stream))

    def fused_add_rmsnorm_mx(self, out_ptr, scales_ptr, input_ptr, weight_ptr, residual_ptr, rows, hidden,
                             out_stride, scale_stride, input_stride, residual_stride, fmt, dtype, eps, stream=0):
        return self._check(self.lib().hprms_fused_add_rmsnorm_mx(out_ptr, scales_ptr, input_ptr, weight_ptr,
                                                                 residual_ptr, rows, hidden, out_stride,
                                                                 scale_stride, input_stride, residual_stride, fmt,
                                                                 dtype, eps, stream))

    def rmsnorm(self, out_ptr, in_ptr, weight_ptr, rows, hidden, out_stride, in_stride, dtype, eps, stream=0):
        return self._check(self.lib().hprms_rmsnorm(out_ptr, in_ptr, weight_ptr, rows, hidden, out_stride,
                                                    in_stride, dtype, eps, stream))

    def _bytes(self, n):
        if n < 0:
            raise HprmsError(n, self.last_error())
        return n

    def rmsnorm_backward_workspace(self, rows, hidden):
        return self._bytes(self.lib().hprms_rmsnorm_backward_workspace(rows, hidden))

    def rmsnorm_backward(self, dinput_ptr, dweight_ptr, dout_ptr, input_ptr, weight_ptr, dresidual_ptr, workspace_ptr,
                         workspace_size, rows, hidden, dinput_stride, dout_stride, input_stride, dresidual_stride,
                         dtype, dweight_dtype, eps, stream=0):
        return self._check(self.lib().hprms_rmsnorm_backward(
            dinput_ptr, dweight_ptr, dout_ptr, input_ptr, weight_ptr, dresidual_ptr, workspace_ptr, workspace_size,
            rows, hidden, dinput_stride, dout_stride, input_stride, dresidual_stride, dtype, dweight_dtype, eps,
            stream))

    def linear_cross_entropy_workspace(self, rows, hidden, vocab, weight_ptr=0, weight_stride=None):
        """For a weight at ``weight_ptr`` (default: any aligned address) with
        ``weight_stride`` elements between rows (default: ``hidden``)."""
        return self._bytes(self.lib().hprms_linear_cross_entropy_workspace(
            rows, hidden, vocab, weight_ptr, hidden if weight_stride is None else weight_stride))

    def linear_cross_entropy(self, loss_ptr, lse_ptr, hidden_ptr, weight_ptr, target_ptr, workspace_ptr,
                             workspace_size, rows, hidden, vocab, hidden_stride, weight_stride, ignore_index, dtype,
                             stream=0):
        return self._check(self.lib().hprms_linear_cross_entropy(
            loss_ptr, lse_ptr, hidden_ptr, weight_ptr, target_ptr, workspace_ptr, workspace_size, rows, hidden, vocab,
            hidden_stride, weight_stride, ignore_index, dtype, stream))

    def linear_cross_entropy_backward_workspace(self, rows, hidden, vocab, weight_ptr=0, weight_stride=None):
        """For a weight at ``weight_ptr`` (default: any aligned address) with
        ``weight_stride`` elements between rows (default: ``hidden``)."""
        return self._bytes(self.lib().hprms_linear_cross_entropy_backward_workspace(
            rows, hidden, vocab, weight_ptr, hidden if weight_stride is None else weight_stride))

    def linear_cross_entropy_backward(self, dhidden_ptr, dweight_ptr, dloss_ptr, hidden_ptr, weight_ptr, target_ptr,
                                      lse_ptr, workspace_ptr, workspace_size, rows, hidden, vocab, dhidden_stride,
                                      dweight_stride, hidden_stride, weight_stride, ignore_index, dtype, stream=0):
        return self._check(self.lib().hprms_linear_cross_entropy_backward(
            dhidden_ptr, dweight_ptr, dloss_ptr, hidden_ptr, weight_ptr, target_ptr, lse_ptr, workspace_ptr,
            workspace_size, rows, hidden, vocab, dhidden_stride, dweight_stride, hidden_stride, weight_stride,
            ignore_index, dtype, stream))

    @staticmethod
    def _arrays(ptrs, dtypes, counts):
        n = len(counts)
        return ((ctypes.c_void_p * max(1, n))(*ptrs), (ctypes.c_int * max(1, n))(*dtypes),
                (ctypes.c_int64 * max(1, n))(*counts), n)

    def grad_norm_workspace(self, counts):
        arr = (ctypes.c_int64 * max(1, len(counts)))(*counts)
        return self._bytes(self.lib().hprms_grad_norm_workspace(arr, len(counts)))

    def grad_norm(self, norm_ptr, grad_ptrs, dtypes, counts, workspace_ptr, workspace_size, stream=0):
        """``grad_ptrs``, ``dtypes`` and ``counts``: sequences of one length."""
        g, d, c, n = self._arrays(grad_ptrs, dtypes, counts)
        return self._check(self.lib().hprms_grad_norm(norm_ptr, g, d, c, n, workspace_ptr, workspace_size, stream))

    def clip_grad_norm(self, norm_ptr, out_ptrs, out_dtypes, grad_ptrs, dtypes, counts, max_norm, workspace_ptr,
                       workspace_size, stream=0):
        g, d, c, n = self._arrays(grad_ptrs, dtypes, counts)
        o, od, _, _ = self._arrays(out_ptrs, out_dtypes, counts)
        return self._check(self.lib().hprms_clip_grad_norm(norm_ptr, o, od, g, d, c, n, max_norm, workspace_ptr,
                                                           workspace_size, stream))

    def norm_add_rmsnorm(self, out_ptr, residual_out_ptr, input_ptr, post_weight_ptr, weight_ptr, residual_ptr,
                         gate_ptr, rows, hidden, rows_per_gate, out_stride, residual_out_stride, input_stride,
                         residual_stride, gate_stride, dtype, residual_scale, eps, stream=0):
        return self._check(self.lib().hprms_norm_add_rmsnorm(
            out_ptr, residual_out_ptr, input_ptr, post_weight_ptr, weight_ptr, residual_ptr, gate_ptr, rows, hidden,
            rows_per_gate, out_stride, residual_out_stride, input_stride, residual_stride, gate_stride, dtype,
            residual_scale, eps, stream))

    def norm_add_rmsnorm_int8(self, out_ptr, scale_ptr, residual_out_ptr, input_ptr, post_weight_ptr, weight_ptr,
                              residual_ptr, gate_ptr, rows, hidden, rows_per_gate, out_stride, residual_out_stride,
                              input_stride, residual_stride, gate_stride, dtype, residual_scale, eps, stream=0):
        return self._check(self.lib().hprms_norm_add_rmsnorm_int8(
            out_ptr, scale_ptr, residual_out_ptr, input_ptr, post_weight_ptr, weight_ptr, residual_ptr, gate_ptr, rows,
            hidden, rows_per_gate, out_stride, residual_out_stride, input_stride, residual_stride, gate_stride, dtype,
            residual_scale, eps, stream))

    def norm_add_rmsnorm_backward_workspace(self, rows, hidden, gate_rows):
        return self._bytes(self.lib().hprms_norm_add_rmsnorm_backward_workspace(rows, hidden, gate_rows))

    def norm_add_rmsnorm_backward(self, dinput_ptr, dresidual_in_ptr, dpost_weight_ptr, dweight_ptr, dgate_ptr,
                                  dout_ptr, dresidual_ptr, input_ptr, residual_ptr, post_weight_ptr, weight_ptr,
                                  gate_ptr, workspace_ptr, workspace_size, rows, hidden, gate_rows, dinput_stride,
                                  dresidual_in_stride, dgate_stride, dout_stride, dresidual_stride, input_stride,
                                  residual_stride, gate_stride, dtype, dpost_weight_dtype, dweight_dtype,
                                  residual_scale, eps, stream=0):
        return self._check(self.lib().hprms_norm_add_rmsnorm_backward(
            dinput_ptr, dresidual_in_ptr, dpost_weight_ptr, dweight_ptr, dgate_ptr, dout_ptr, dresidual_ptr, input_ptr,
            residual_ptr, post_weight_ptr, weight_ptr, gate_ptr, workspace_ptr, workspace_size, rows, hidden,
            gate_rows, dinput_stride, dresidual_in_stride, dgate_stride, dout_stride, dresidual_stride, input_stride,
            residual_stride, gate_stride, dtype, dpost_weight_dtype, dweight_dtype, residual_scale, eps, stream))

    def int8_linear_workspace(self, rows, inner, outer, input_ptr=0, input_stride=None, weight_ptr=0,
                              weight_stride=None):
        """For operands at these addresses (default: any aligned ones) with
        these strides between rows (default: ``inner``)."""
        return self._bytes(self.lib().hprms_int8_linear_workspace(
            rows, inner, outer, input_ptr, inner if input_stride is None else input_stride, weight_ptr,
            inner if weight_stride is None else weight_stride))

    def int8_linear(self, out_ptr, input_ptr, scale_ptr, weight_ptr, weight_scale_ptr, bias_ptr, workspace_ptr,
                    workspace_size, rows, inner, outer, out_stride, input_stride, weight_stride, dtype, stream=0):
        return self._check(self.lib().hprms_int8_linear(
            out_ptr, input_ptr, scale_ptr, weight_ptr, weight_scale_ptr, bias_ptr, workspace_ptr, workspace_size,
            rows, inner, outer, out_stride, input_stride, weight_stride, dtype, stream))

    def token_log_probs_workspace(self, rows, vocab, top, dtype):
        return self._bytes(self.lib().hprms_token_log_probs_workspace(rows, vocab, top, dtype))

    def token_log_probs(self, log_prob_ptr, entropy_ptr, lse_ptr, top_log_prob_ptr, top_index_ptr, logits_ptr,
                        tokens_ptr, workspace_ptr, workspace_size, rows, vocab, top, logits_stride, ignore_index,
                        dtype, stream=0):
        return self._check(self.lib().hprms_token_log_probs(
            log_prob_ptr, entropy_ptr, lse_ptr, top_log_prob_ptr, top_index_ptr, logits_ptr, tokens_ptr, workspace_ptr,
            workspace_size, rows, vocab, top, logits_stride, ignore_index, dtype, stream))

    def token_log_probs_backward(self, dlogits_ptr, dlog_prob_ptr, dentropy_ptr, logits_ptr, tokens_ptr, lse_ptr,
                                 entropy_ptr, rows, vocab, dlogits_stride, logits_stride, ignore_index, dtype,
                                 stream=0):
        return self._check(self.lib().hprms_token_log_probs_backward(
            dlogits_ptr, dlog_prob_ptr, dentropy_ptr, logits_ptr, tokens_ptr, lse_ptr, entropy_ptr, rows, vocab,
            dlogits_stride, logits_stride, ignore_index, dtype, stream))

    def streamer(self, out_ptr, in_ptr, rows, hidden, out_stride, in_stride, dtype, op, stream=0):
        return self._check(self.lib().hprms_streamer(out_ptr, in_ptr, rows, hidden, out_stride, in_stride, dtype,
                                                     op, stream))

    def select_config(self, rows, hidden, dtype, mode=0, cus=None):
        """The table's configuration for a MODE_* entry point, on a device of
        `cus` compute units (None: 256, a whole MI355X)."""
        c = Config()
        L = self.lib()
        if cus is None:
            self._check(L.hprms_select_config(rows, hidden, dtype, mode, ctypes.byref(c)))
        else:
            self._check(L.hprms_select_config_cu(rows, hidden, dtype, mode, cus, ctypes.byref(c)))
        return c

    def set_batch_invariant(self, enable):
        """hprms_set_batch_invariant: returns the previous setting."""
        rc = self.lib().hprms_set_batch_invariant(1 if enable else 0)
        if rc < 0:
            raise HprmsError(rc, self.last_error())
        return bool(rc)

    def batch_invariant(self):
        return bool(self.lib().hprms_batch_invariant())

    def device_cu_count(self, device=-1):
        """Compute units of a HIP device (-1: the current one) as the entry
        points use them."""
        n = self.lib().hprms_device_cu_count(device)
        if n < 0:
            raise HprmsError(n, self.last_error())
        return n

    def bench_fused_timeline(self, input_ptr, weight_ptr, residual_ptr, rows, hidden, dtype, eps, config,
                             timeline_ptr, stream=0):
        """Bench library only: the in-place op on contiguous rows with a forced
        configuration carrying flags bit 9 and its timeline buffer."""
        return self._check(self.lib().hprms_bench_fused_timeline(input_ptr, weight_ptr, residual_ptr, rows, hidden,
                                                                 dtype, eps, ctypes.byref(config), timeline_ptr,
                                                                 stream))

    def bench_form_config(self, mode, out_ptr, aux_ptr, aux_stride, aux_group_stride, input_ptr, weight_ptr,
                          residual_ptr, rows, hidden, dtype, eps, config, stream=0):
        """Bench library only: a form of the op (mode 1, 2, 3, 5, 6 or 7) on
        contiguous rows with a forced configuration; `aux` is the residual
        output (mode 3) or the scales."""
        return self._check(self.lib().hprms_bench_form_config(mode, out_ptr, aux_ptr, aux_stride, aux_group_stride,
                                                              input_ptr, weight_ptr, residual_ptr, rows, hidden,
                                                              dtype, eps, ctypes.byref(config), stream))

    def kernel_configs(self, dtype, mode=0):
        """Every vector-tier configuration built for (dtype, mode)."""
        L = self.lib()
        n = L.hprms_kernel_configs(dtype, mode, None, 0)
        if n < 0:
            raise HprmsError(n, self.last_error())
        arr = (Config * n)()
        self._check(0 if L.hprms_kernel_configs(dtype, mode, arr, n) == n else HPRMS_E_INVALID)
        return list(arr)


PRODUCT = Library(KERNEL_LIB)
BENCH = Library(BENCH_LIB, bench=True)


def lib():
    return PRODUCT.lib()


def last_error():
    return PRODUCT.last_error()


fused_add_rmsnorm = PRODUCT.fused_add_rmsnorm
fused_add_rmsnorm_fp8 = PRODUCT.fused_add_rmsnorm_fp8
fused_add_rmsnorm_fp8_static = PRODUCT.fused_add_rmsnorm_fp8_static
fused_add_rmsnorm_fp8_group = PRODUCT.fused_add_rmsnorm_fp8_group
fused_add_rmsnorm_fp8_ub = PRODUCT.fused_add_rmsnorm_fp8_ub
fused_add_rmsnorm_out = PRODUCT.fused_add_rmsnorm_out
reduce_add_rmsnorm = PRODUCT.reduce_add_rmsnorm
fused_add_rmsnorm_mx = PRODUCT.fused_add_rmsnorm_mx
rmsnorm = PRODUCT.rmsnorm
rmsnorm_backward_workspace = PRODUCT.rmsnorm_backward_workspace
rmsnorm_backward = PRODUCT.rmsnorm_backward
linear_cross_entropy_workspace = PRODUCT.linear_cross_entropy_workspace
linear_cross_entropy = PRODUCT.linear_cross_entropy
linear_cross_entropy_backward_workspace = PRODUCT.linear_cross_entropy_backward_workspace
linear_cross_entropy_backward = PRODUCT.linear_cross_entropy_backward
grad_norm_workspace = PRODUCT.grad_norm_workspace
grad_norm = PRODUCT.grad_norm
clip_grad_norm = PRODUCT.clip_grad_norm
norm_add_rmsnorm = PRODUCT.norm_add_rmsnorm
norm_add_rmsnorm_int8 = PRODUCT.norm_add_rmsnorm_int8
norm_add_rmsnorm_backward_workspace = PRODUCT.norm_add_rmsnorm_backward_workspace
norm_add_rmsnorm_backward = PRODUCT.norm_add_rmsnorm_backward
int8_linear_workspace = PRODUCT.int8_linear_workspace
int8_linear = PRODUCT.int8_linear
token_log_probs_workspace = PRODUCT.token_log_probs_workspace
token_log_probs = PRODUCT.token_log_probs
token_log_probs_backward = PRODUCT.token_log_probs_backward
streamer = PRODUCT.streamer
select_config = PRODUCT.select_config
device_cu_count = PRODUCT.device_cu_count
set_batch_invariant = PRODUCT.set_batch_invariant
batch_invariant = PRODUCT.batch_invariant
kernel_configs = PRODUCT.kernel_configs
