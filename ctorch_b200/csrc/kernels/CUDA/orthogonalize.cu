// Orthogonalised updates: NS(G) by Newton-Schulz steps, and the weight update built on it.
//
//   X0 = G / (|G|_F + eps);  X <- a X + (b A + c A A) X,  A = X X^T (the short side's Gram matrix)
#include <math.h>

#include "common.cuh"

namespace {
using namespace ctk;

constexpr float kA = 3.4445f, kB = -4.7750f, kC = 2.0315f;
constexpr int PREP_THREADS = 256;

struct Source {
    const float* g;
    int64_t ldg;
    float* momentum;  // nullptr: U = G
    int64_t ldm;
    float mu;
    int nesterov;
    int64_t rows, cols;
};

// ---- pass 1: momentum update and the Frobenius norm ------------------------------------------------------
// |U|_F^2 as a double per CTA (one double multiply-add per element neither overflows nor loses small
// elements); the partial sums are added in CTA order by whoever needs the norm.
__global__ void __launch_bounds__(PREP_THREADS) prep_norm_kernel(Source S, double* __restrict__ partial) {
    const int64_t total = S.rows * S.cols;
    double acc = 0.0;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * PREP_THREADS + threadIdx.x; i < total; i += static_cast<int64_t>(gridDim.x) * PREP_THREADS) {
        const int64_t r = i / S.cols, c = i - r * S.cols;
        float u = S.g[r * S.ldg + c];
        if (S.momentum) {
            float* mp = S.momentum + r * S.ldm + c;
            const float m = fmaf(S.mu, *mp, u);
            *mp = m;
            u = S.nesterov ? fmaf(S.mu, m, u) : m;
        }
        acc = fma(static_cast<double>(u), static_cast<double>(u), acc);
    }
    __shared__ double sums[PREP_THREADS / 32];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
    if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = acc;
    __syncthreads();
    if (threadIdx.x == 0) {
        double t = 0.0;
        for (int w = 0; w < PREP_THREADS / 32; ++w) t += sums[w];
        partial[blockIdx.x] = t;
    }
}

// ---- pass 2: Y = U / (|U|_F + eps) -----------------------------------------------------------------------
__global__ void __launch_bounds__(PREP_THREADS) prep_scale_kernel(Source S, const double* __restrict__ partial, int parts, float eps, float* __restrict__ y) {
    __shared__ float inv_s;
    if (threadIdx.x == 0) {
        double t = 0.0;
        for (int i = 0; i < parts; ++i) t += partial[i];
        inv_s = isfinite(t) ? static_cast<float>(1.0 / (sqrt(t) + static_cast<double>(eps))) : __int_as_float(0x7fc00000);
    }
    __syncthreads();
    const float inv = inv_s;
    const int64_t total = S.rows * S.cols;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * PREP_THREADS + threadIdx.x; i < total; i += static_cast<int64_t>(gridDim.x) * PREP_THREADS) {
        const int64_t r = i / S.cols, c = i - r * S.cols;
        float u = S.g[r * S.ldg + c];
        if (S.momentum) {
            const float m = S.momentum[r * S.ldm + c];
            u = S.nesterov ? fmaf(S.mu, m, u) : m;
        }
        y[i] = u * inv;
    }
}

__global__ void __launch_bounds__(PREP_THREADS) poly_kernel(float* __restrict__ a, const float* __restrict__ a2, int64_t n) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * PREP_THREADS + threadIdx.x;
    if (i < n) a[i] = fmaf(kB, a[i], kC * a2[i]);
}
__global__ void __launch_bounds__(PREP_THREADS) combine_kernel(float* __restrict__ x, const float* __restrict__ bx, int64_t n) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * PREP_THREADS + threadIdx.x;
    if (i < n) x[i] = fmaf(kA, x[i], bx[i]);
}

// ---- where the result goes -------------------------------------------------------------------------------
struct Sink {
    float* out;  // NS(U), or the weights of an update
    int64_t ldo;
    int update;  // 0: out = o;  1: out = keep * out - step * o
    float keep, step;
};
__global__ void __launch_bounds__(PREP_THREADS) sink_kernel(Sink K, const float* __restrict__ x, int64_t rows, int64_t cols) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * PREP_THREADS + threadIdx.x;
    if (i >= rows * cols) return;
    float* o = K.out + (i / cols) * K.ldo + i % cols;
    *o = K.update ? fmaf(-K.step, x[i], K.keep * *o) : x[i];
}

struct Layout {
    size_t partial, x, x2, a, a2, total;
};
Layout layout_for(int64_t rows, int64_t cols) {
    const size_t d = static_cast<size_t>(rows < cols ? rows : cols), n = static_cast<size_t>(rows) * static_cast<size_t>(cols);
    auto up = [](size_t b) { return (b + 255) & ~size_t(255); };
    Layout L;
    size_t at = 0;
    auto take = [&](size_t b) { const size_t p = at; at += up(b); return p; };
    L.partial = take(4096 * sizeof(double));
    L.x = take(n * 4);
    L.x2 = take(n * 4);
    L.a = take(d * d * 4);
    L.a2 = take(d * d * 4);
    L.total = at;
    return L;
}

ctk_status newton_schulz(const Source& S, const Sink& K, int steps, float eps, void* workspace, void* stream) {
    const Layout L = layout_for(S.rows, S.cols);
    StreamScratch scratch;
    if (!workspace) {
        ctk_status st = scratch.get(L.total, stream);
        if (st) return st;
        workspace = scratch.p;
    }
    char* ws = static_cast<char*>(workspace);
    double* partial = reinterpret_cast<double*>(ws + L.partial);
    float *x = reinterpret_cast<float*>(ws + L.x), *x2 = reinterpret_cast<float*>(ws + L.x2);
    float *a = reinterpret_cast<float*>(ws + L.a), *a2 = reinterpret_cast<float*>(ws + L.a2);
    cudaStream_t st = as_stream(stream);
    const int64_t rows = S.rows, cols = S.cols, n = rows * cols;
    const bool tall = rows > cols;
    const int64_t d = tall ? cols : rows;
    const int grid = ctk_stream_grid(n, PREP_THREADS, 4);
    prep_norm_kernel<<<grid, PREP_THREADS, 0, st>>>(S, partial);
    CTK_LAUNCH_CHECK("orthogonalize: norm");
    prep_scale_kernel<<<grid, PREP_THREADS, 0, st>>>(S, partial, grid, eps, x);
    CTK_LAUNCH_CHECK("orthogonalize: scale");
    auto blocks = [](int64_t c) { return static_cast<unsigned>((c + PREP_THREADS - 1) / PREP_THREADS); };
    for (int s = 0; s < steps; ++s) {
        ctk_status rc = tall ? ctk_matmul_f32(x, x, a, d, d, rows, 1, cols, cols, 1, CTK_MATMUL_FP32_SIMT, nullptr, stream)
                             : ctk_matmul_f32(x, x, a, d, d, cols, cols, 1, 1, cols, CTK_MATMUL_FP32_SIMT, nullptr, stream);
        if (!rc) rc = ctk_matmul_f32(a, a, a2, d, d, d, d, 1, d, 1, CTK_MATMUL_FP32_SIMT, nullptr, stream);
        if (rc) return rc;
        poly_kernel<<<blocks(d * d), PREP_THREADS, 0, st>>>(a, a2, d * d);
        CTK_LAUNCH_CHECK("orthogonalize: polynomial");
        rc = tall ? ctk_matmul_f32(x, a, x2, rows, cols, cols, cols, 1, cols, 1, CTK_MATMUL_FP32_SIMT, nullptr, stream)
                  : ctk_matmul_f32(a, x, x2, rows, cols, rows, rows, 1, cols, 1, CTK_MATMUL_FP32_SIMT, nullptr, stream);
        if (rc) return rc;
        combine_kernel<<<blocks(n), PREP_THREADS, 0, st>>>(x, x2, n);
        CTK_LAUNCH_CHECK("orthogonalize: combine");
    }
    sink_kernel<<<blocks(n), PREP_THREADS, 0, st>>>(K, x, rows, cols);
    CTK_LAUNCH_CHECK("orthogonalize: result");
    return CTK_OK;
}

ctk_status check_common(const char* who, int64_t rows, int64_t cols, int steps, float eps, const void* workspace) {
    const std::string w(who);
    CTK_REQUIRE(rows >= 0 && cols >= 0, w + ": negative size");
    CTK_REQUIRE(steps >= 1 && steps <= 64, w + ": steps must be in [1, 64]");
    CTK_REQUIRE(eps > 0.0f && isfinite(eps), w + ": eps must be positive and finite");
    CTK_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 255u) == 0, w + ": workspace must be 256-byte aligned");
    if (rows > (int64_t(1) << 30) || cols > (int64_t(1) << 30) || (rows && cols > (int64_t(1) << 30) / rows))
        return fail(CTK_ERR_LIMIT, w + ": more than 2^30 elements");
    return CTK_OK;
}

}  // namespace

extern "C" {

size_t ctk_orthogonalize_workspace_bytes(int64_t rows, int64_t cols) {
    if (rows <= 0 || cols <= 0 || rows > (int64_t(1) << 30) || cols > (int64_t(1) << 30) / rows) return 0;
    return layout_for(rows, cols).total;
}

ctk_status ctk_orthogonalize_f32(const float* g, int64_t ldg, float* out, int64_t ldo, int64_t rows, int64_t cols, int steps, float eps, void* workspace,
                                 void* stream) {
    CTK_RANGE("ctk_orthogonalize_f32");
    ctk_status rc = check_common("ctk_orthogonalize_f32", rows, cols, steps, eps, workspace);
    if (rc) return rc;
    CTK_REQUIRE(ldg >= cols && ldo >= cols, "ctk_orthogonalize_f32: row pitch below cols");
    if (rows == 0 || cols == 0) return CTK_OK;
    CTK_REQUIRE(g && out, "ctk_orthogonalize_f32: null pointer");
    CTK_REQUIRE(aligned_to(g, 4) && aligned_to(out, 4), "ctk_orthogonalize_f32: misaligned pointer");
    CTK_REQUIRE((g == out && ldg == ldo) || !spans_overlap(g, rows, cols, ldg, out, rows, cols, ldo), "ctk_orthogonalize_f32: out overlaps g (only in place is allowed)");
    const Source S{g, ldg, nullptr, 0, 0.0f, 0, rows, cols};
    const Sink K{out, ldo, 0, 0.0f, 0.0f};
    return newton_schulz(S, K, steps, eps, workspace, stream);
}

ctk_status ctk_muon_update_f32(float* p, int64_t ldp, const float* g, int64_t ldg, float* momentum, int64_t ldm, int64_t rows, int64_t cols, float lr, float mu,
                               int nesterov, float weight_decay, float scale, int steps, float eps, void* workspace, void* stream) {
    CTK_RANGE("ctk_muon_update_f32");
    ctk_status rc = check_common("ctk_muon_update_f32", rows, cols, steps, eps, workspace);
    if (rc) return rc;
    CTK_REQUIRE(ldp >= cols && ldg >= cols && ldm >= cols, "ctk_muon_update_f32: row pitch below cols");
    if (rows == 0 || cols == 0) return CTK_OK;
    CTK_REQUIRE(p && g && momentum, "ctk_muon_update_f32: null pointer");
    CTK_REQUIRE(aligned_to(p, 4) && aligned_to(g, 4) && aligned_to(momentum, 4), "ctk_muon_update_f32: misaligned pointer");
    CTK_REQUIRE(!spans_overlap(p, rows, cols, ldp, g, rows, cols, ldg) && !spans_overlap(p, rows, cols, ldp, momentum, rows, cols, ldm) &&
                    !spans_overlap(g, rows, cols, ldg, momentum, rows, cols, ldm),
                "ctk_muon_update_f32: p, g and momentum must not overlap");
    const Source S{g, ldg, momentum, ldm, mu, nesterov, rows, cols};
    const Sink K{p, ldp, 1, 1.0f - lr * weight_decay, lr * scale};
    return newton_schulz(S, K, steps, eps, workspace, stream);
}

ctk_status ctk_orthogonalize_status(int* status) {
    CTK_REQUIRE(status, "ctk_orthogonalize_status: null pointer");
    CTK_CUDA(cudaDeviceSynchronize());
    *status = 0;
    return CTK_OK;
}

}  // extern "C"
