// Host-side internals shared by the files that implement the C ABI: error reporting, the device guard and the
// layer handle.
#pragma once
#include <atomic>
#include <cstdarg>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <initializer_list>
#include <string>
#include <vector>

#include "pmoe_common.cuh"

namespace pmoe {

int fail(int code, const char *fmt, ...);
int fail_cuda(cudaError_t e, const char *what);

#define CU(call)                                                  \
    do {                                                          \
        cudaError_t _e = (call);                                  \
        if (_e != cudaSuccess) return fail_cuda(_e, #call);       \
    } while (0)

// Makes `device` current for the calling thread and restores the previous one on exit.
struct DeviceGuard {
    int prev = -1;
    bool ok = false;
    explicit DeviceGuard(int device)
    {
        if (cudaGetDevice(&prev) != cudaSuccess) prev = -1;
        ok = prev == device || cudaSetDevice(device) == cudaSuccess;
        if (prev == device) prev = -1;   // nothing to restore
    }
    ~DeviceGuard()
    {
        if (prev >= 0) cudaSetDevice(prev);
    }
};

// Lets `kern` have up to `most` bytes of dynamic shared memory on the current device, once a device (`asked`, one for each kernel,
// has a bit for each).  The limit belongs to the kernel, not to a launch: it must be the same in every call, or a thread
// that lowers it makes another thread's launch fail.
inline cudaError_t allow_smem(const void *kern, size_t most, std::atomic<uint64_t> &asked)
{
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return e;
    if (device > 63 || !(asked.load(std::memory_order_relaxed) >> device & 1)) {
        e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most);
        if (e != cudaSuccess) return e;
        if (device <= 63) asked.fetch_or(1ull << device, std::memory_order_relaxed);
    }
    return cudaSuccess;
}

// Memory that a call reads or writes
struct Span {
    const void *at;
    size_t bytes;
    bool over(const Span &o) const
    {
        return at && o.at && (uintptr_t)at < (uintptr_t)o.at + o.bytes && (uintptr_t)o.at < (uintptr_t)at + bytes;
    }
};
// Whether an output lies over one of the inputs or over another output.  Kernels read some inputs more than once and in several
// CTAs, which must see the same each time.
inline bool overlap(std::initializer_list<Span> outputs, std::initializer_list<Span> inputs)
{
    for (auto o = outputs.begin(); o != outputs.end(); o++) {
        for (auto &i : inputs)
            if (o->over(i)) return true;
        for (auto p = o + 1; p != outputs.end(); p++)
            if (o->over(*p)) return true;
    }
    return false;
}

}  // namespace pmoe

struct pmoe_ep_state;   // buffers of the expert-parallel forward (pmoe_ep.cu)

struct pmoe_layer {
    pmoe_layer_desc desc;
    pmoe::LayerDev dev;
    pmoe::Workspace ws;
    int device;
    std::vector<void *> owned;  // device allocations freed at destroy
    // device staging for the host-buffer entry point
    void *st_x = nullptr, *st_out = nullptr;
    float *st_logits = nullptr;
    uint32_t *st_idx = nullptr;
    float *st_w = nullptr;
    // per-phase CUDA events of the last traced call (pmoe_layer_trace)
    // pmoe_forward_host replays the kernel chain of its last shape as a CUDA graph (the chain works on
    // the handle's own staging buffers, so its arguments do not change from call to call)
    cudaStream_t cap_stream = nullptr;
    cudaGraphExec_t hg_exec = nullptr;
    int hg_n = -1, hg_x_dtype = 0, hg_out_dtype = 0, hg_flags = 0, hg_launches = 0;
    int hg_seen_n = -1, hg_seen_x = 0, hg_seen_out = 0, hg_seen_flags = 0;
    void *hg_out = nullptr, *hg_seen_out_ptr = nullptr;   // where the chain writes the block output
    bool hg_off = false;
    // rows the shared expert serves in the next run_experts call; count < 0 = every row
    int req_sh_begin = 0, req_sh_count = -1;
    // block-scale multipliers (training mode): the tensors as created, and the scaled copies the kernels read
    // while multipliers are installed (index: 0 gate_exps, 1 up_exps, 2 down_exps, 3 sh_gate, 4 sh_up, 5 sh_down)
    const uint8_t *orig[6] = {};
    void *scaled[6] = {};
    pmoe_ep_state *ep = nullptr;   // created by the first pmoe_ep_forward
    bool trace = false;
    cudaEvent_t ev0[PMOE_TRACE_PHASES] = {}, ev1[PMOE_TRACE_PHASES] = {};
    bool ev_used[PMOE_TRACE_PHASES] = {};
};

namespace pmoe {

// experts (+ shared expert) given routing already in device memory; `ws` is the layer's workspace or a copy of it
// with some arrays redirected
int run_experts(pmoe_layer *L, Workspace &ws, const void *x, int x_dtype, const uint32_t *idx, const float *w, int n, int top_k,
                bool routed, bool shared, bool prep_done, void *out, int out_dtype, cudaStream_t s);
int check_call(pmoe_layer *L, const void *x, int x_dtype, int n, const void *out, int out_dtype);
void ep_state_destroy(pmoe_ep_state *st);

}  // namespace pmoe
