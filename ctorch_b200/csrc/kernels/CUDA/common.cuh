// Shared host/device helpers of the sm_100a kernel library.
#pragma once
#include <cuda_runtime.h>
#include <nvtx3/nvToolsExt.h>
#include <stdint.h>
#include <atomic>
#include <string>

#include "ctorch_b200.h"

namespace ctk {

// Thread-local message of the last failure; returns `code` so launchers can `return fail(...)`.
ctk_status fail(ctk_status code, const std::string& msg);
extern std::atomic<uint64_t> g_launches;
inline void count_launch(int n = 1) { g_launches.fetch_add(static_cast<uint64_t>(n), std::memory_order_relaxed); }

// Number of SMs of the current device (cached per device ordinal).
int sm_count();
// Library-owned per-device scratch, grown on demand (never shrinks).  slot 0: reductions,
// slot 1: matmul workspace.
ctk_status device_scratch(int slot, size_t bytes, void** out);

// Scratch for one call: allocated from the device's pool and given back in the order of `stream`, so calls on
// different streams never share it, and a call that is being captured records its own allocation in the graph.
ctk_status stream_alloc(size_t bytes, void* stream, void** out);
struct StreamScratch {
    void* p = nullptr;
    void* stream = nullptr;
    ctk_status get(size_t bytes, void* st) { stream = st; return stream_alloc(bytes, st, &p); }
    StreamScratch() = default;
    ~StreamScratch() { if (p && cudaFreeAsync(p, reinterpret_cast<cudaStream_t>(stream)) != cudaSuccess) (void)cudaGetLastError(); }
    StreamScratch(const StreamScratch&) = delete;
    StreamScratch& operator=(const StreamScratch&) = delete;
};

inline bool aligned_to(const void* p, uintptr_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
// Whether two [rows, cols] fp32 arrays of row pitch lda / ldb overlap: share a byte between their first and last element, unless
// both are columns of one buffer (the same pitch) that lie side by side.
inline bool spans_overlap(const void* a, int64_t rows_a, int64_t cols_a, int64_t lda, const void* b, int64_t rows_b, int64_t cols_b, int64_t ldb) {
    if (rows_a <= 0 || cols_a <= 0 || rows_b <= 0 || cols_b <= 0) return false;
    const uintptr_t a0 = reinterpret_cast<uintptr_t>(a), b0 = reinterpret_cast<uintptr_t>(b);
    const uintptr_t a1 = a0 + 4 * static_cast<uintptr_t>((rows_a - 1) * lda + cols_a), b1 = b0 + 4 * static_cast<uintptr_t>((rows_b - 1) * ldb + cols_b);
    if (a0 >= b1 || b0 >= a1) return false;
    if (lda != ldb || (a0 - b0) % 4) return true;
    // side by side in the rows of one buffer
    const int64_t shift = static_cast<int64_t>(b0 > a0 ? (b0 - a0) / 4 : (a0 - b0) / 4) % lda, first = b0 > a0 ? cols_a : cols_b, second = b0 > a0 ? cols_b : cols_a;
    return shift < first || shift + second > lda;
}

// Whether the [rows, cols] fp32 array at a, row pitch ld, shares a byte with the `bytes` bytes at b.
inline bool touches(const void* a, int64_t rows, int64_t cols, int64_t ld, const void* b, size_t bytes) {
    if (!b || rows <= 0 || cols <= 0 || bytes == 0) return false;
    const uintptr_t a0 = reinterpret_cast<uintptr_t>(a), b0 = reinterpret_cast<uintptr_t>(b), b1 = b0 + bytes;
    const uintptr_t pitch = 4 * static_cast<uintptr_t>(ld), row = 4 * static_cast<uintptr_t>(cols);
    if (a0 >= b1 || b0 >= a0 + (static_cast<uintptr_t>(rows) - 1) * pitch + row) return false;
    if (b0 <= a0) return true;
    const uintptr_t r = (b0 - a0) / pitch;  // b starts in this row or in the gap behind it
    return (b0 - a0) % pitch < row || (r + 1 < static_cast<uintptr_t>(rows) && b1 > a0 + (r + 1) * pitch);
}

inline cudaStream_t as_stream(void* s) { return reinterpret_cast<cudaStream_t>(s); }

// NVTX range around the host side of an entry point (header-only NVTX: a no-op costing a few
// nanoseconds unless a profiler has injected itself), so a timeline shows which C-ABI call issued
// which kernels.
struct Range {
    explicit Range(const char* name) { nvtxRangePushA(name); }
    ~Range() { nvtxRangePop(); }
    Range(const Range&) = delete;
    Range& operator=(const Range&) = delete;
};

// One-time set-up that belongs to a (kernel, device) pair -- cudaFuncSetAttribute, occupancy queries --
// is guarded by one of these per kernel instantiation: first() is true once per device ordinal, for
// the device that is current at the call (a process may drive several GPUs through ctk_set_device).
struct PerDeviceOnce {
    bool done[64] = {false};
    bool first() {
        int dev = 0;
        if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return true;  // unknown device: redo the set-up, it is idempotent
        if (done[dev]) return false;
        done[dev] = true;
        return true;
    }
};

// The same where threads may make their first calls at once: every thread that finds the set-up missing does it (it is
// idempotent) before it launches, and only a set-up that succeeded is marked.
struct PerDeviceReady {
    std::atomic<bool> done[64];
    template <typename F>
    ctk_status ensure(F&& set_up) {
        int dev = 0;
        const bool known = cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < 64;
        if (known && done[dev].load(std::memory_order_acquire)) return CTK_OK;
        const ctk_status st = set_up();
        if (!st && known) done[dev].store(true, std::memory_order_release);
        return st;
    }
};

}  // namespace ctk

// (A failed call also leaves its code as the thread's "last error"; it is taken back here, or the
// next kernel launch check -- which reads that state -- would report this failure as its own.)
#define CTK_CUDA(call)                                                                          \
    do {                                                                                        \
        cudaError_t _e = (call);                                                                \
        if (_e != cudaSuccess) {                                                                \
            (void)cudaGetLastError();                                                           \
            return ctk::fail(CTK_ERR_CUDA, std::string(#call) + ": " + cudaGetErrorString(_e)); \
        }                                                                                       \
    } while (0)

#define CTK_LAUNCH_CHECK(name)                                                                    \
    do {                                                                                          \
        cudaError_t _e = cudaGetLastError();                                                      \
        if (_e != cudaSuccess)                                                                    \
            return ctk::fail(CTK_ERR_CUDA, std::string(name) + " launch: " + cudaGetErrorString(_e)); \
        ctk::count_launch();                                                                      \
    } while (0)

#define CTK_RANGE(name) ctk::Range _ctk_nvtx_range(name)

#define CTK_REQUIRE(cond, msg)                                    \
    do {                                                          \
        if (!(cond)) return ctk::fail(CTK_ERR_INVALID, (msg));    \
    } while (0)

// Grid size for a grid-stride streaming kernel: a whole number of waves of the SM count.
static inline int ctk_stream_grid(int64_t work_items, int threads, int ctas_per_sm) {
    int64_t need = (work_items + threads - 1) / threads;
    int64_t cap = static_cast<int64_t>(ctk::sm_count()) * ctas_per_sm;
    if (need < 1) need = 1;
    return static_cast<int>(need < cap ? need : cap);
}
