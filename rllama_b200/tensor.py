"""Device tensors: the Python mirror of rllama's ``OpenCLTensor`` surface
(``src/tensor_opencl_support.rs:171-412``) over the C ABI, used by the op-level parity tests
the way ``src/tensor.rs``'s ``#[cfg(feature = "opencl")]`` tests use the OpenCL backend.
"""
import ctypes
import sys

import numpy as np

from . import _ffi
from ._ffi import F16, F32, check


def capacity_cols(cols, dtype):
    """Row stride rllama's Tensor uses: cols rounded up to 8 (f32) or 16 (f16)
    (``src/tensor.rs:192-222``)."""
    m = 16 if dtype == F16 else 8
    return (int(cols) + m - 1) // m * m


_MOST = 2 ** 31 - 1


def _i32(args):
    """The library takes 32-bit numbers, and ctypes would cut off the rest. ``args``: the bits of all of them, or-ed (of numbers that fit the sign is all
    that lies beyond 31 bits, and a negative one among others is refused by the library)."""
    if args >> 31 not in (0, -1):
        raise OverflowError("an argument does not fit in 32 bits")


def _given(tensor):
    """The handle of an optional argument."""
    if tensor is None:
        return None
    if not tensor._h:
        raise ValueError("the tensor has been freed")
    return tensor._h


class Cuda:
    """Counterpart of ``OpenCL`` (``OpenCL::new(verbose, nth_device)``). ``stream``: a CUDA stream handle (an integer, e.g.
    ``torch.cuda.current_stream().cuda_stream``; 0 is the legacy default stream, the per-thread one is refused) that the ops are queued
    on, in order with the caller's own work there; the stream must outlive the context. Without it the context has a stream of its own."""

    def __init__(self, verbose=False, nth_device=0, stream=None):
        self._h = ctypes.c_void_p()
        if stream is None:
            check(_ffi.lib().rlb_ctx_create(int(verbose), int(nth_device), ctypes.byref(self._h)))
        else:
            check(_ffi.lib().rlb_ctx_create_on_stream(int(verbose), int(nth_device), ctypes.c_void_p(int(stream)), ctypes.byref(self._h)))

    def flush(self):
        check(_ffi.lib().rlb_ctx_flush(self._h))

    def kernel_launches(self):
        n = ctypes.c_uint64()
        check(_ffi.lib().rlb_ctx_kernel_launches(self._h, ctypes.byref(n)))
        return n.value

    def close(self):
        if self._h:
            _ffi.lib().rlb_ctx_destroy(self._h)
            self._h = ctypes.c_void_p()

    # -- tensors ------------------------------------------------------------------------
    def upload(self, array):
        """``OpenCL::data_u16_to_gpu``: pads rows to the capacity rule and uploads."""
        a = np.asarray(array)
        if a.ndim == 1:
            a = a.reshape(1, -1)
        dt = F16 if a.dtype == np.float16 else F32
        a = a.astype(np.float16 if dt == F16 else np.float32, copy=False)
        cap = capacity_cols(a.shape[1], dt)
        padded = np.zeros((a.shape[0], cap), dtype=a.dtype)
        padded[:, : a.shape[1]] = a
        t = CudaTensor(self, a.shape[0], a.shape[1], cap, dt)
        t._keep = padded  # must outlive the asynchronous copy
        check(_ffi.lib().rlb_tensor_upload(self._h, padded.ctypes.data_as(ctypes.c_void_p), a.shape[0], a.shape[1], cap, dt,
                                           ctypes.byref(t._h)))
        return t

    def zeros(self, rows, cols, dtype):
        cap = capacity_cols(cols, dtype)
        t = CudaTensor(self, rows, cols, cap, dtype)
        check(_ffi.lib().rlb_tensor_zeros(self._h, rows, cols, cap, dtype, ctypes.byref(t._h)))
        return t

    def wrap(self, tensor):
        """A view of a torch CUDA tensor (f16 or f32, two-dimensional, contiguous columns, rows a multiple of 16 bytes apart):
        no copy. The view keeps the torch tensor alive. Without a shared ``stream`` the caller orders the two streams."""
        if tensor.dim() != 2 or (tensor.shape[1] > 1 and tensor.stride(1) != 1):
            raise ValueError("wrap takes a two-dimensional tensor with contiguous columns")
        dt = {"torch.float16": F16, "torch.float32": F32}.get(str(tensor.dtype))
        if dt is None or not tensor.is_cuda:
            raise ValueError("wrap takes an f16 or f32 CUDA tensor, not %s on %s" % (tensor.dtype, tensor.device))
        rows, cols = tensor.shape
        cap = tensor.stride(0) if rows > 1 else capacity_cols(cols, dt)
        if cap < cols:
            raise ValueError("wrap takes rows that do not overlap")
        t = CudaTensor(self, rows, cols, cap, dt)
        check(_ffi.lib().rlb_tensor_wrap(self._h, ctypes.c_void_p(tensor.data_ptr()), rows, cols, cap, dt, ctypes.byref(t._h)))
        t._keep_view = tensor
        return t

    def rope_table(self, max_seq_len, head_dim):
        """The rotation's (cos, sin) pairs, one row a position (``compute_freqs_cis``)."""
        _i32(int(max_seq_len) | int(head_dim))
        t = CudaTensor(self, max_seq_len, head_dim, head_dim, F32)
        check(_ffi.lib().rlb_rope_table(self._h, int(max_seq_len), int(head_dim), ctypes.byref(t._h)))
        return t


class CudaTensor:
    def __init__(self, cl, rows, cols, cap, dtype):
        self.cl, self.rows, self.cols, self.cap, self.dtype = cl, int(rows), int(cols), int(cap), dtype
        self._h = ctypes.c_void_p()
        self._keep = None

    def wait_until_ready(self):
        check(_ffi.lib().rlb_tensor_wait(self._h))
        self._keep = None

    def to_numpy(self):
        """``data_u16_from_gpu`` + ``OpenCLEvent::wait``; returns the unpadded values."""
        out = np.empty((self.rows, self.cap), dtype=np.float16 if self.dtype == F16 else np.float32)
        ev = ctypes.c_void_p()
        check(_ffi.lib().rlb_tensor_download(self._h, out.ctypes.data_as(ctypes.c_void_p), ctypes.byref(ev)))
        check(_ffi.lib().rlb_event_wait(ev))
        return out[:, : self.cols].copy()

    def copy_inplace(self, other):
        check(_ffi.lib().rlb_copy_inplace(self._h, other._h))

    def transpose_from(self, other):
        check(_ffi.lib().rlb_transpose_from(self._h, other._h))

    def hadamard_product_inplace(self, other):
        check(_ffi.lib().rlb_hadamard_product_inplace(self._h, other._h))

    def silu_inplace(self):
        check(_ffi.lib().rlb_silu_inplace(self._h))

    def matrix_mul_inplace_transposed(self, src, other):
        check(_ffi.lib().rlb_matrix_mul_inplace_transposed(self._h, src._h, other._h))

    def attention_decode(self, q, kcache, vcache, heads, max_seq_len, pos, n_split=1):
        """self <- single-query attention of q over positions 0..pos of the caches."""
        check(_ffi.lib().rlb_attention_decode(self._h, q._h, kcache._h, vcache._h, heads, max_seq_len, pos, n_split))

    def attention_prefill(self, q, kcache, vcache, heads, max_seq_len, start_pos=0, tensor_cores=True):
        """self <- causal attention of the rows of q (row i attends to positions 0..start_pos+i)."""
        check(_ffi.lib().rlb_attention_prefill(self._h, q._h, kcache._h, vcache._h, heads, max_seq_len, start_pos, int(bool(tensor_cores))))

    def attention_decode_static(self, q, kcache, vcache, heads, max_seq_len, pos, n_split=1):
        """Same as ``attention_decode`` but allocation-free: the kernel's scratch is a fixed
        array inside the library (for hosts that cannot allocate on the token path). Fails
        beyond 256 heads or 262144 scratch floats; calls on one device must not overlap."""
        check(_ffi.lib().rlb_attention_decode_static(self._h, q._h, kcache._h, vcache._h, heads, max_seq_len, pos, n_split))

    def norm_rope_append(self, kcache, vcache, q, k, v, rope, heads, kv_heads, max_seq_len, start_pos, q_gain=None, k_gain=None, eps=1e-6):
        """self <- the rows of q, their heads normalised (with a gain) and rotated; k likewise and v as it is go to positions
        start_pos, start_pos + 1, ... of the caches."""
        _i32(heads | kv_heads | max_seq_len | start_pos)
        check(_ffi.lib().rlb_norm_rope_append(self._h, kcache._h, vcache._h, q._h, k._h, v._h, _given(q_gain), _given(k_gain), eps, rope._h,
                                              heads, kv_heads, max_seq_len, start_pos))

    def attention_window(self, q, kcache, vcache, heads, kv_heads, max_seq_len, start_pos, window, sinks=0):
        """self <- attention of the rows of q (row i at position p = start_pos + i) over the positions t <= p with
        t > p - window or t < sinks; heads / kv_heads query heads share a K/V head."""
        window, sinks = min(window, _MOST), min(sinks, _MOST)
        _i32(heads | kv_heads | max_seq_len | start_pos | window | sinks)
        check(_ffi.lib().rlb_attention_window(self._h, q._h, kcache._h, vcache._h, heads, kv_heads, max_seq_len, start_pos, window, sinks))

    def free(self):
        if self._h:
            _ffi.lib().rlb_tensor_free(self._h)
            self._h = ctypes.c_void_p()

    def __del__(self):
        # at interpreter shutdown the CUDA runtime may already be gone: leave the memory to process exit
        try:
            if sys is not None and not sys.is_finalizing():
                self.free()
        except Exception:
            pass


class Cache4:
    """A KV cache held in 4 bits: groups of 32 values share an f16 scale, a value is scale * (-7 .. 7) and always an f16 number
    (the storage is described in ``include/rllama_b200.h``)."""

    def __init__(self, cl, kv_heads, max_seq_len, head_dim, _arrays=None):
        self.cl, self.kv_heads, self.max_seq_len, self.head_dim = cl, int(kv_heads), int(max_seq_len), int(head_dim)
        self._h = ctypes.c_void_p()
        _i32(self.kv_heads | self.max_seq_len | self.head_dim)
        self._keep = _arrays
        if _arrays is None:
            check(_ffi.lib().rlb_cache4_create(cl._h, self.kv_heads, self.max_seq_len, self.head_dim, ctypes.byref(self._h)))
        else:
            check(_ffi.lib().rlb_cache4_wrap(cl._h, *(ctypes.c_void_p(t.data_ptr()) for t in _arrays), self.kv_heads, self.max_seq_len,
                                             self.head_dim, ctypes.byref(self._h)))

    @classmethod
    def wrap(cls, cl, k_codes, k_scales, v_codes, v_scales, kv_heads, max_seq_len, head_dim):
        """Over torch CUDA tensors: uint8 codes and f16 scales of kv_heads * max_seq_len contiguous rows each. No copy."""
        for t, dtype, width in ((k_codes, "torch.uint8", head_dim // 2), (k_scales, "torch.float16", head_dim // 32),
                                (v_codes, "torch.uint8", head_dim // 2), (v_scales, "torch.float16", head_dim // 32)):
            if str(t.dtype) != dtype or not t.is_cuda or not t.is_contiguous() or t.numel() != kv_heads * max_seq_len * width:
                raise ValueError("Cache4.wrap takes contiguous CUDA tensors: uint8 codes, kv_heads*max_seq_len x head_dim/2, and f16 scales, x head_dim/32")
        return cls(cl, kv_heads, max_seq_len, head_dim, (k_codes, k_scales, v_codes, v_scales))

    def append(self, k, v, start_pos):
        """Rows of rotated k and v (both f32 or both f16) to positions start_pos, start_pos + 1, ..."""
        _i32(start_pos)
        check(_ffi.lib().rlb_cache4_append(self._h, k._h, v._h, start_pos))

    def norm_rope_append(self, q_out, q, k, v, rope, heads, start_pos, q_gain=None, k_gain=None, eps=1e-6):
        """``CudaTensor.norm_rope_append`` into this cache: q_out <- the rows of q, k and v to positions start_pos, start_pos + 1, ..."""
        _i32(heads | start_pos)
        check(_ffi.lib().rlb_cache4_norm_rope_append(self._h, q_out._h, q._h, k._h, v._h, _given(q_gain), _given(k_gain), eps, rope._h, heads, start_pos))

    def read(self, k_out, v_out, start_pos):
        """The values held, into f16 or f32 rows; either may be None."""
        _i32(start_pos)
        check(_ffi.lib().rlb_cache4_read(self._h, _given(k_out), _given(v_out), start_pos))

    def attention(self, out, q, heads, start_pos, window=None, sinks=0):
        """out (f16) <- ``attention_window`` of the rows of q over the values held; no window by default."""
        window, sinks = _MOST if window is None else min(window, _MOST), min(sinks, _MOST)
        _i32(heads | start_pos | window | sinks)
        check(_ffi.lib().rlb_cache4_attention(self._h, out._h, q._h, heads, start_pos, window, sinks))

    def free(self):
        if self._h:
            _ffi.lib().rlb_cache4_free(self._h)
            self._h = ctypes.c_void_p()
            self._keep = None

    def __del__(self):
        # at interpreter shutdown the CUDA runtime may already be gone: leave the memory to process exit
        try:
            if sys is not None and not sys.is_finalizing():
                self.free()
        except Exception:
            pass
