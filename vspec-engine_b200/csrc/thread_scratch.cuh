// thread_scratch.cuh -- library-managed device scratch: one grow-only buffer per
// device and host thread, given back when the thread ends.
#pragma once

#include "common.cuh"

namespace vb200 {

// What may block or free on the device, with no regard to captures of other threads (they see none of it).
class RelaxedCapture {
public:
    RelaxedCapture() { cudaThreadExchangeStreamCaptureMode(&mode_); }
    ~RelaxedCapture() { cudaThreadExchangeStreamCaptureMode(&mode_); }

private:
    cudaStreamCaptureMode mode_ = cudaStreamCaptureModeRelaxed;
};

// To be thread_local.
class ThreadScratch {
public:
    ~ThreadScratch() {
        RelaxedCapture relaxed;
        for (Buffer& b : buffers_)
            if (b.ptr && !b.captured) (void)cudaFree(b.ptr);
    }

    // Sets *out to at least `bytes` on the current device, the first `zeros` of them 0 when they are new; else an
    // error code with its message.  A buffer that a captured call uses stays for good: replays have its address.
    int get(size_t bytes, size_t zeros, cudaStream_t st, void** out) {
        int dev = 0;
        VB_CHECK_CUDA(cudaGetDevice(&dev));
        if (dev < 0 || dev >= kDevices) { set_error("device %d is out of range for the library's scratch", dev); return VSPEC_B200_ERR_UNSUPPORTED; }
        Buffer& b = buffers_[dev];
        cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
        VB_CHECK_CUDA(cudaStreamIsCapturing(st, &capture));
        const bool capturing = capture != cudaStreamCaptureStatusNone;
        if (b.cap < bytes) {
            if (capturing) {
                set_error("the library's scratch cannot grow to %zu bytes during a capture: pass d_workspace, or make the call once before", bytes);
                return VSPEC_B200_ERR_ARG;
            }
            RelaxedCapture relaxed;
            if (b.ptr && !b.captured) (void)cudaFree(b.ptr);
            b = Buffer();
            void* p = nullptr;
            if (cudaMalloc(&p, bytes) != cudaSuccess) {
                (void)cudaGetLastError();
                set_error("cannot allocate %zu bytes of scratch", bytes);
                return VSPEC_B200_ERR_NOMEM;
            }
            if (zeros) {
                const cudaError_t e = cudaMemsetAsync(p, 0, zeros, st);
                if (e != cudaSuccess) { (void)cudaFree(p); return cuda_status(e, "scratch memset"); }
            }
            b.ptr = p;
            b.cap = bytes;
        }
        b.captured |= capturing;
        *out = b.ptr;
        return VSPEC_B200_OK;
    }

private:
    static constexpr int kDevices = 64;
    struct Buffer {
        void* ptr = nullptr;
        size_t cap = 0;
        bool captured = false;
    };
    Buffer buffers_[kDevices];
};

}  // namespace vb200
