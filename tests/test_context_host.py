"""The host side of contexts and tensors (``rllama_b200/csrc/context.cu``) against a small CUDA runtime of the test's own, built with g++: two
devices, a current device, and a log of what is queued where. As in CUDA, the NULL stream is that of the current device and an event
only records on a stream of its own device. No GPU needed."""
import ctypes
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CUDA = os.path.dirname(os.path.dirname(os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")))

RUNTIME = r"""
#include <cuda_runtime.h>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <map>
#include <string>
#include "internal.h"

static int g_device = 0;
static std::map<const void*, int> g_memory, g_events, g_streams;   // their device
static bool g_capturing = false;
static std::string g_log;
static int on(cudaStream_t s) { return s == nullptr || s == cudaStreamLegacy ? g_device : g_streams.count(s) ? g_streams[s] : -1; }
static cudaError_t queue(const char* what, cudaStream_t s) {
    char line[64];
    snprintf(line, sizeof(line), "%s %d\n", what, on(s));
    g_log += line;
    return cudaSuccess;
}

extern "C" {
const char* fake_log(void) { return g_log.c_str(); }
void fake_reset(int device) { g_log.clear(); g_device = device; g_capturing = false; }
int fake_device(void) { return g_device; }
void fake_capture(int yes) { g_capturing = yes != 0; }
void* fake_stream(int device) { void* s = malloc(16); g_streams[s] = device; return s; }

cudaError_t cudaGetDevice(int* d) { *d = g_device; return cudaSuccess; }
cudaError_t cudaSetDevice(int d) { g_device = d; return cudaSuccess; }
cudaError_t cudaGetDeviceCount(int* n) { *n = 2; return cudaSuccess; }
cudaError_t cudaGetDeviceProperties(cudaDeviceProp* p, int) { memset(p, 0, sizeof(*p)); p->major = 10; p->multiProcessorCount = 4; return cudaSuccess; }
const char* cudaGetErrorString(cudaError_t) { return "an error of the test's runtime"; }
cudaError_t cudaGetLastError(void) { return cudaSuccess; }
cudaError_t cudaMalloc(void** p, size_t n) { *p = calloc(1, n); g_memory[*p] = g_device; return cudaSuccess; }
cudaError_t cudaFree(void* p) { g_memory.erase(p); free(p); g_log += "free\n"; return cudaSuccess; }
cudaError_t cudaMallocAsync(void** p, size_t n, cudaStream_t s) { queue("malloc", s); return cudaMalloc(p, n); }
cudaError_t cudaFreeAsync(void* p, cudaStream_t s) { queue("free", s); g_memory.erase(p); free(p); return cudaSuccess; }
cudaError_t cudaHostAlloc(void** p, size_t n, unsigned) { *p = calloc(1, n); return cudaSuccess; }
cudaError_t cudaHostGetDevicePointer(void** d, void* h, unsigned) { *d = h; return cudaSuccess; }
cudaError_t cudaFreeHost(void* p) { free(p); return cudaSuccess; }
cudaError_t cudaMemcpyAsync(void* d, const void* s, size_t n, cudaMemcpyKind, cudaStream_t st) { memcpy(d, s, n); return queue("copy", st); }
cudaError_t cudaMemcpy2DAsync(void*, size_t, const void*, size_t, size_t, size_t, cudaMemcpyKind, cudaStream_t st) { return queue("copy", st); }
cudaError_t cudaMemsetAsync(void* d, int v, size_t n, cudaStream_t st) { memset(d, v, n); return queue("set", st); }
cudaError_t cudaStreamCreateWithFlags(cudaStream_t* s, unsigned) { *s = (cudaStream_t)fake_stream(g_device); return cudaSuccess; }
cudaError_t cudaStreamDestroy(cudaStream_t s) { g_streams.erase(s); free(s); return cudaSuccess; }
cudaError_t cudaStreamSynchronize(cudaStream_t s) { return g_capturing ? cudaErrorStreamCaptureUnsupported : queue("wait", s); }
cudaError_t cudaStreamGetDevice(cudaStream_t s, int* d) { *d = on(s); return *d < 0 ? cudaErrorInvalidResourceHandle : cudaSuccess; }
cudaError_t cudaStreamIsCapturing(cudaStream_t, cudaStreamCaptureStatus* st) { *st = g_capturing ? cudaStreamCaptureStatusActive : cudaStreamCaptureStatusNone; return cudaSuccess; }
cudaError_t cudaThreadExchangeStreamCaptureMode(cudaStreamCaptureMode*) { return cudaSuccess; }
cudaError_t cudaEventCreateWithFlags(cudaEvent_t* e, unsigned) { *e = (cudaEvent_t)malloc(16); g_events[*e] = g_device; return cudaSuccess; }
cudaError_t cudaEventDestroy(cudaEvent_t e) { g_events.erase(e); free(e); return cudaSuccess; }
cudaError_t cudaEventRecord(cudaEvent_t e, cudaStream_t s) { return g_events[e] != on(s) ? cudaErrorInvalidResourceHandle : queue("event", s); }
cudaError_t cudaEventSynchronize(cudaEvent_t) { g_log += "event wait\n"; return cudaSuccess; }
cudaError_t cudaPointerGetAttributes(cudaPointerAttributes* a, const void* p) {
    auto it = g_memory.upper_bound(p);
    memset(a, 0, sizeof(*a));
    if (it != g_memory.begin()) { a->type = cudaMemoryTypeDevice; a->device = (--it)->second; }
    return cudaSuccess;
}
}

int launch_gemv(rlb_ctx* c, rlb_dtype, int, int, const GemvArgs&) { queue("kernel", c->stream); return RLB_OK; }
int launch_silu(rlb_ctx* c, void*, rlb_dtype, int64_t, int64_t, int64_t) { queue("kernel", c->stream); return RLB_OK; }
int launch_hadamard(rlb_ctx* c, void*, const void*, rlb_dtype, int64_t, int64_t, int64_t, int64_t) { queue("kernel", c->stream); return RLB_OK; }
int launch_transpose(rlb_ctx* c, void*, const void*, rlb_dtype, int64_t, int64_t, int64_t, int64_t) { queue("kernel", c->stream); return RLB_OK; }
int launch_attn_decode(rlb_ctx* c, rlb_dtype, const AttnDecodeArgs&, int) { queue("kernel", c->stream); return RLB_OK; }
int launch_attn_prefill(rlb_ctx* c, rlb_dtype, const AttnPrefillArgs&) { queue("kernel", c->stream); return RLB_OK; }
int launch_gemm_nt_typed(rlb_ctx* c, rlb_dtype, const void*, int64_t, const void*, int64_t, void*, int64_t, int, int, int) { queue("kernel", c->stream); return RLB_OK; }
size_t attn_decode_scratch_floats(int, int, int) { return 64; }
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    at = tmp_path_factory.mktemp("context_host")
    (at / "runtime.cpp").write_text(RUNTIME)
    so, csrc = str(at / "context_host.so"), os.path.join(ROOT, "rllama_b200", "csrc")
    subprocess.run([os.environ.get("CXX", "g++"), "-std=c++17", "-O1", "-shared", "-fPIC", "-Wl,-Bsymbolic", "-I" + csrc, "-I" + os.path.join(CUDA, "include"),
                    "-x", "c++", os.path.join(csrc, "context.cu"), str(at / "runtime.cpp"), "-o", so], check=True)
    lib = ctypes.CDLL(so)
    lib.fake_log.restype = lib.rlb_last_error.restype = ctypes.c_char_p
    lib.fake_stream.restype = ctypes.c_void_p
    for name in ("rlb_tensor_upload", "rlb_tensor_zeros"):
        getattr(lib, name).argtypes = [ctypes.c_void_p] * (2 if name.endswith("upload") else 1) + [ctypes.c_int64] * 3 + [ctypes.c_int, ctypes.POINTER(ctypes.c_void_p)]
    return lib


def context(lib, device, stream):
    h = ctypes.c_void_p()
    assert lib.rlb_ctx_create_on_stream(0, device, ctypes.c_void_p(stream), ctypes.byref(h)) == 0
    return h


LEGACY, PER_THREAD = 1, 2   # cudaStreamLegacy, cudaStreamPerThread


def test_the_per_thread_stream_is_refused(lib):
    """It is another stream in every host thread, and a context's calls share scratch on the ground that they follow one another."""
    lib.fake_reset(0)
    h = ctypes.c_void_p(7)
    assert lib.rlb_ctx_create_on_stream(0, 0, ctypes.c_void_p(PER_THREAD), ctypes.byref(h)) == 1 and not h.value
    assert b"per-thread" in lib.rlb_last_error()
    for stream in (None, LEGACY, lib.fake_stream(0)):
        lib.rlb_ctx_destroy(context(lib, 0, stream))
    assert lib.rlb_ctx_create_on_stream(0, 1, ctypes.c_void_p(lib.fake_stream(0)), ctypes.byref(h)) == 1 and not h.value   # another device's


@pytest.mark.parametrize("stream", [None, LEGACY])
def test_the_default_stream_is_that_of_the_context_s_device(lib, stream):
    """A context on device 1's default stream while device 0 is current: everything is queued on, and waited for, device 1."""
    lib.fake_reset(0)
    ctx, t, host, ev = context(lib, 1, stream), ctypes.c_void_p(), (ctypes.c_float * 32)(*range(32)), ctypes.c_void_p()
    for make in (lambda: lib.rlb_tensor_zeros(ctx, 4, 8, 8, 0, ctypes.byref(t)), lambda: lib.rlb_tensor_upload(ctx, host, 4, 8, 8, 0, ctypes.byref(t))):
        lib.fake_reset(0)
        assert make() == 0, lib.rlb_last_error()
        assert lib.rlb_tensor_wait(t) == 0 and lib.rlb_ctx_flush(ctx) == 0
        assert lib.rlb_silu_inplace(t) == 0 and lib.rlb_copy_inplace(t, t) == 0
        assert lib.rlb_tensor_download(t, host, ctypes.byref(ev)) == 0 and lib.rlb_event_wait(ev) == 0
        log = [line.split() for line in lib.fake_log().decode().splitlines() if line != "event wait"]
        assert len(log) >= 8 and all(line[1] == "1" for line in log), log
        assert lib.fake_device() == 0
        assert lib.rlb_tensor_free(t) == 0
    assert lib.rlb_ctx_destroy(ctx) == 0 and lib.fake_device() == 0


def test_calls_that_cannot_be_captured_are_refused_before_they_reach_the_runtime(lib):
    """Allocations and waits would break the capture of the caller's stream and report something else."""
    lib.fake_reset(0)
    ctx, t, u, host, ev = context(lib, 0, lib.fake_stream(0)), ctypes.c_void_p(), ctypes.c_void_p(), (ctypes.c_float * 32)(), ctypes.c_void_p()
    assert lib.rlb_tensor_zeros(ctx, 4, 8, 8, 0, ctypes.byref(t)) == 0
    lib.fake_reset(0)
    lib.fake_capture(1)
    for call in (lambda: lib.rlb_tensor_zeros(ctx, 4, 8, 8, 0, ctypes.byref(u)), lambda: lib.rlb_tensor_upload(ctx, host, 4, 8, 8, 0, ctypes.byref(u)),
                 lambda: lib.rlb_tensor_wait(t), lambda: lib.rlb_ctx_flush(ctx), lambda: lib.rlb_tensor_download(t, host, ctypes.byref(ev))):
        assert call() == 5 and lib.fake_log() == b"" and not u.value and not ev.value
    assert lib.rlb_silu_inplace(t) == 0   # (an op that may be captured)
    lib.fake_capture(0)
    assert lib.rlb_tensor_wait(t) == 0 and lib.rlb_tensor_free(t) == 0 and lib.rlb_ctx_destroy(ctx) == 0
