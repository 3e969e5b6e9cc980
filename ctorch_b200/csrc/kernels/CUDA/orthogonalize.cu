// Orthogonalised updates: NS(G) by Newton-Schulz steps, and the weight update built on it.
//
//   X0 = G / (|G|_F + eps);  X <- a X + (b A + c A A) X,  A = X X^T (the short side's Gram matrix)
//
// Two passes over U (momentum update + norm, then scaling) and three products a step:
//   GRAM   A = X X^T       symmetric: one triangle of tiles, each written to its mirror place too
//   POLY   B = b A + c A A symmetric, the polynomial in the epilogue
//   APPLY  X = a X + B X   (X B where rows > cols); the last one writes the result, or the weights of an update
// The products run on the tensor cores at fp32 accuracy: every matrix is held as hi + lo, two fp16 numbers
// (22 bits), and hi hi + hi lo + lo hi are three kind::f16 products into one accumulator -- 1.5 units of TF32-rate
// work per fp32 product where a TF32 split costs 2 or 3, for the same 4 bytes per element.  fp16's range is no
// obstacle here: the singular values of X never pass 1.21 (the step's polynomial maps [0, 1.21] into itself), so
// |X| <= 1.21, |A| <= 1.46 and |B| <= 2.81 element by element, and a fixed power of two puts them high in fp16's range
// (2^15, 2^15, 2^14); elements 2^-24 below the largest keep 11 bits or more between hi and lo.
// The tensor core truncates as it adds into its fp32 accumulator, so an accumulator holds 64 or 256 terms
// at a time; the epilogue warps add those up in registers with rounding.
#include <math.h>

#include "tcgen05.cuh"

namespace {
using namespace ctk;

__device__ int g_ns_status = 0;  // first bounded wait that ran out: (role << 8) | barrier, else 0

constexpr float kA = 3.4445f, kB = -4.7750f, kC = 2.0315f;
// Powers of two by which X, A (= X X^T) and B (= b A + c A A) are held.
constexpr float kScaleX = 32768.0f;
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
// elements); the partial sums are added in a fixed order by whoever needs the norm.  V elements per access (4 where
// every pitch and pointer allows it).  Bound by the bytes of G and M.
template <int V>
struct Vec;
template <>
struct Vec<1> { float v[1]; };
template <>
struct __align__(16) Vec<4> { float v[4]; };

template <int V>
__device__ __forceinline__ Vec<V> load_vec(const float* p) { return *reinterpret_cast<const Vec<V>*>(p); }

__device__ __forceinline__ double block_sum(double acc) {
    __shared__ double sums[PREP_THREADS / 32];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
    if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = acc;
    __syncthreads();
    double t = 0.0;
#pragma unroll
    for (int w = 0; w < PREP_THREADS / 32; ++w) t += sums[w];
    return t;
}

template <int V, bool MOMENTUM>
__global__ void __launch_bounds__(PREP_THREADS) prep_norm_kernel(Source S, double* __restrict__ partial) {
    const uint32_t per_row = static_cast<uint32_t>(S.cols / V), total = static_cast<uint32_t>(S.rows) * per_row;
    double acc = 0.0;
    for (uint32_t i = blockIdx.x * PREP_THREADS + threadIdx.x; i < total; i += gridDim.x * PREP_THREADS) {
        const uint32_t r = i / per_row, c = (i - r * per_row) * V;
        Vec<V> u = load_vec<V>(S.g + r * S.ldg + c);
        if (MOMENTUM) {
            float* mp = S.momentum + r * S.ldm + c;
            Vec<V> m = load_vec<V>(mp);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                m.v[e] = fmaf(S.mu, m.v[e], u.v[e]);
                u.v[e] = S.nesterov ? fmaf(S.mu, m.v[e], u.v[e]) : m.v[e];
            }
            *reinterpret_cast<Vec<V>*>(mp) = m;
        }
#pragma unroll
        for (int e = 0; e < V; ++e) acc = fma(static_cast<double>(u.v[e]), static_cast<double>(u.v[e]), acc);
    }
    const double t = block_sum(acc);
    if (threadIdx.x == 0) partial[blockIdx.x] = t;
}

// ---- pass 2: X0 as hi + lo, and the steps' coefficients --------------------------------------------------
// With n = |U|_F and T = n + eps, X0 = U / T.  Where eps is not small beside n, X0 is small as a whole and
// would sink in fp16's range; it is held as Y = X0 2^e instead, e >= 0 such that |Y|_F lies in (1/4, 1].  A step on Y is
// Y <- f (a Y + (b 4^-e A_Y + c 16^-e A_Y A_Y) Y) with f = 1/4 and e <- e - 2 as long as e > 0 (the step multiplies by
// less than 4), all exact powers of two.  coef[4 s ..] = {b 4^-e, c 16^-e, f, -} of step s; the last step's f undoes 2^e.
struct Normaliser {
    float p2, rest;  // Y = (U * p2) * rest * kScaleX
    int e;
};
__device__ __forceinline__ Normaliser normaliser(double sumsq, float eps) {
    Normaliser N;
    if (!(sumsq < 1.7e308)) return Normaliser{__int_as_float(0x7fc00000), 1.0f, 0};  // a non-finite element: NaN everywhere
    const double n = sqrt(sumsq), t = n + static_cast<double>(eps);
    int en = 0, et = 0;
    (void)frexp(n, &en);
    const double mt = frexp(t, &et);
    if (n == 0.0 || en < -126) en = n == 0.0 ? et : -126;  // (2^-en stays a normal number)
    const int gap = et - en;
    N.e = gap > 1 ? gap - 1 : 0;
    N.p2 = static_cast<float>(ldexp(1.0, -en));
    N.rest = static_cast<float>(gap >= 1 ? 0.5 / mt : 1.0 / mt);
    return N;
}

__device__ __forceinline__ void split_half(float x, __half& hi, __half& lo) {
    hi = __float2half_rn(x);
    lo = __float2half_rn(x - __half2float(hi));
}

// Two elements at a time: {hi0, hi1} and {lo0, lo1} as the conversion instruction packs them.
__device__ __forceinline__ void split2(float x0, float x1, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(x0, x1);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(x0 - f.x, x1 - f.y);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&l);
}

// One matrix as hi and lo arrays: [outer, pitch] each, lo behind hi.
struct Pair {
    __half* hi;
    int64_t pitch;
    int64_t lo;  // elements from hi to lo
};

template <int V, bool MOMENTUM>
__global__ void __launch_bounds__(PREP_THREADS) prep_split_kernel(Source S, const double* __restrict__ partial, int parts, float eps, int steps,
                                                                  Pair X, float* __restrict__ coef) {
    double acc = 0.0;
    for (int i = threadIdx.x; i < parts; i += PREP_THREADS) acc += partial[i];
    const Normaliser N = normaliser(block_sum(acc), eps);
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        int e = N.e;
        for (int s = 0; s < steps; ++s) {
            const int drop = e < 2 ? e : 2;
            coef[4 * s] = ldexpf(kB, -2 * e);
            coef[4 * s + 1] = ldexpf(kC, -4 * e);
            coef[4 * s + 2] = s + 1 == steps ? ldexpf(1.0f, -e) : ldexpf(1.0f, -drop);
            coef[4 * s + 3] = 0.0f;
            e -= drop;
        }
    }
    const uint32_t per_row = static_cast<uint32_t>(S.cols / V), total = static_cast<uint32_t>(S.rows) * per_row;
    for (uint32_t i = blockIdx.x * PREP_THREADS + threadIdx.x; i < total; i += gridDim.x * PREP_THREADS) {
        const uint32_t r = i / per_row, c = (i - r * per_row) * V;
        Vec<V> u = load_vec<V>(S.g + r * S.ldg + c);
        if (MOMENTUM) {
            const Vec<V> m = load_vec<V>(S.momentum + r * S.ldm + c);
#pragma unroll
            for (int e = 0; e < V; ++e) u.v[e] = S.nesterov ? fmaf(S.mu, m.v[e], u.v[e]) : m.v[e];
        }
        __half hi[V], lo[V];
#pragma unroll
        for (int e = 0; e < V; ++e) split_half((u.v[e] * N.p2) * (N.rest * kScaleX), hi[e], lo[e]);
        __half* dst = X.hi + r * X.pitch + c;
        if (V == 4) {
            *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(hi);
            *reinterpret_cast<uint2*>(dst + X.lo) = *reinterpret_cast<const uint2*>(lo);
        } else {
            dst[0] = hi[0];
            dst[X.lo] = lo[0];
        }
    }
}

// ---- where the result goes -------------------------------------------------------------------------------
struct Sink {
    float* out;  // NS(U), or the weights of an update
    int64_t ldo;
    int update;  // 0: out = o;  1: out = keep * out - step * o
    float keep, step;
    int vec;     // 16-byte accesses are possible
};
__device__ __forceinline__ float sink_value(const Sink& K, float o, float old) { return K.update ? fmaf(-K.step, o, K.keep * old) : o; }

// ---- the products ----------------------------------------------------------------------------------------
enum { GRAM = 0, POLY = 1, APPLY = 2 };
constexpr int BM = 128, BK = 64;
constexpr int THREADS = 320;      // warp 0 loads, warp 1 multiplies, warps 2-9 take the accumulators
constexpr int EPI_WARPS = 8;
constexpr int STAGE_BYTES = 4 * BM * BK * 2;  // [A hi | lo][B hi | lo], 128 rows of each per CTA
constexpr int STAGES = 3;
// k-blocks of 64 terms summed in TMEM before they move to registers.  Relative error of NS(G) against 64 bits at 784 x 128
// with 1 / 2 / 4 / 8 blocks: 1.8 / 3.1 / 3.4 / 4.0e-6, at 4096 x 4096 0.7 / 0.9 / 1.6 / 3.0e-6 (fp32 library products: 1.4 and
// 3.8e-6).  A drain of the 128 x 256 accumulator costs the tensor pipe about 0.6 us (4096 x 4096 APPLY: 350 / 335 / 315 us
// with 2 / 4 / 8 blocks, 293 without drains), so the pairs' product takes 4 and the kernels of smaller matrices, which are not
// bound by the pipe, 1.
constexpr int CHUNK_KB = 4;
constexpr int OUT_PITCH = 33;
constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + EPI_WARPS * 32 * OUT_PITCH * 4 + 1024;

struct Params {
    int m, n;                 // extents of the product's result
    int tiles_m, tiles_n, units, num_kb;
    int split;                // medium matrices: CTAs that share a tile's k-blocks
    int slabs;                // GRAM of a long, thin matrix: clusters that share a tile, each with its part of k
    float* slab_sums;         // [slab][tile][row][column] of them, taken up by ns_join_kernel
    Pair src;                 // POLY: A; APPLY: X before the step
    Pair dst;                 // GRAM: A; POLY: B; APPLY: X after the step (unless last)
    const float* coef;        // this step's {b, c, f}
    int last;                 // APPLY: the result goes to the sink
    Sink sink;
};

// Tile u of the launch.  Symmetric products count the upper triangle column by column.
template <int MODE>
__device__ __forceinline__ void unit_tile(int u, const Params& P, int& tm, int& tn) {
    if (MODE != APPLY) {
        int j = static_cast<int>((sqrtf(8.0f * static_cast<float>(u) + 1.0f) - 1.0f) * 0.5f);
        while (j * (j + 1) / 2 > u) --j;
        while ((j + 1) * (j + 2) / 2 <= u) ++j;
        tn = j;
        tm = u - j * (j + 1) / 2;
        return;
    }
    // bands of 8 tile columns, row after row inside a band: the tiles in flight share rows of A and columns of B in L2
    constexpr int BAND = 8;
    const int band = u / (BAND * P.tiles_m), first = band * BAND;
    const int width = P.tiles_n - first < BAND ? P.tiles_n - first : BAND;
    const int r = u - band * (BAND * P.tiles_m);
    tm = r / width;
    tn = first + r % width;
}

// A 32 x 32 block of the result, lane = row (the layout tcgen05.ld delivers), on its way to memory.  It goes through
// `stage`, so that 8 lanes share a row's 32 elements and every load and store is 64 contiguous bytes or more; the other
// triangle of a symmetric product is read back transposed, two rows to a lane, hi in the lower 16 lanes and lo in the
// upper.  (POLY with its A read and its mirror written element by element from the accumulator's own layout: 275 us at
// 4096 x 4096, this way 176 us.)
template <int MODE>
__device__ __forceinline__ void emit_block(const Params& P, bool mirror, int row_base, int lane, int col0, const float (&v)[32], uint32_t* stage,
                                           const float (&cf)[3]) {
    if (col0 >= P.n || row_base >= P.m) return;  // the whole warp
    const int sub = lane >> 3, c4 = (lane & 7) * 4;
    const int64_t col = col0 + c4;
#pragma unroll
    for (int i = 0; i < 32; ++i) stage[lane * OUT_PITCH + i] = __float_as_uint(v[i]);
    __syncwarp();
    constexpr int HALF = 4;  // rows of a lane at a time (2500 x 2500 with 8: 1130 us, 4: 1097, 2: the same)
#pragma unroll 1
    for (int r0 = 0; r0 < 32; r0 += 4 * HALF) {
        uint2 h4[HALF], l4[HALF];
        if (MODE != GRAM) {  // all of these reads in flight before anything waits
            const __half* xp = P.src.hi + (row_base + r0 + sub) * P.src.pitch + col;  // (pitches are multiples of 8: four elements never leave the row)
#pragma unroll
            for (int i = 0; i < HALF; ++i) {
                h4[i] = l4[i] = make_uint2(0u, 0u);
                if (row_base + r0 + i * 4 + sub < P.m && col < P.n) {
                    h4[i] = __ldcg(reinterpret_cast<const uint2*>(xp + i * 4 * P.src.pitch));
                    l4[i] = __ldcg(reinterpret_cast<const uint2*>(xp + i * 4 * P.src.pitch + P.src.lo));
                }
            }
        }
#pragma unroll
        for (int i = 0; i < HALF; ++i) {
            const int r = r0 + i * 4 + sub;
            uint32_t* s = stage + r * OUT_PITCH + c4;
            const __half2 h0 = *reinterpret_cast<const __half2*>(&h4[i].x), h1 = *reinterpret_cast<const __half2*>(&h4[i].y);
            const __half2 l0 = *reinterpret_cast<const __half2*>(&l4[i].x), l1 = *reinterpret_cast<const __half2*>(&l4[i].y);
            const float src[4] = {__low2float(h0) + __low2float(l0), __high2float(h0) + __high2float(l0), __low2float(h1) + __low2float(l1),
                                  __high2float(h1) + __high2float(l1)};
            float o[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float d = __uint_as_float(s[e]);
                if (MODE == GRAM) o[e] = d * (1.0f / 32768.0f);
                if (MODE == POLY) o[e] = fmaf(cf[0] * 0.5f, src[e], cf[1] * (1.0f / 65536.0f) * d);
                if (MODE == APPLY) o[e] = cf[2] * fmaf(kA, src[e], d * (1.0f / 16384.0f));
            }
            const bool inside = row_base + r < P.m && col < P.n;
            if (MODE == APPLY && P.last) {
                if (!inside) continue;
                float* out = P.sink.out + (row_base + r) * P.sink.ldo + col;
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] *= 1.0f / kScaleX;
                if (P.sink.vec && col + 4 <= P.n) {
                    float4 old = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (P.sink.update) old = *reinterpret_cast<const float4*>(out);
                    *reinterpret_cast<float4*>(out) = make_float4(sink_value(P.sink, o[0], old.x), sink_value(P.sink, o[1], old.y), sink_value(P.sink, o[2], old.z),
                                                                  sink_value(P.sink, o[3], old.w));
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (col + e < P.n) out[e] = sink_value(P.sink, o[e], P.sink.update ? out[e] : 0.0f);
                }
                continue;
            }
            uint2 hi, lo;
            split2(o[0], o[1], hi.x, lo.x);
            split2(o[2], o[3], hi.y, lo.y);
            if (inside) {
                __half* d = P.dst.hi + (row_base + r) * P.dst.pitch + col;
                *reinterpret_cast<uint2*>(d) = hi;
                *reinterpret_cast<uint2*>(d + P.dst.lo) = lo;
            }
            if (MODE != APPLY && mirror) {  // {hi, lo} of one element in one word
                s[0] = __byte_perm(hi.x, lo.x, 0x5410);
                s[1] = __byte_perm(hi.x, lo.x, 0x7632);
                s[2] = __byte_perm(hi.y, lo.y, 0x5410);
                s[3] = __byte_perm(hi.y, lo.y, 0x7632);
            }
        }
    }
    __syncwarp();
    if (MODE != APPLY && mirror) {
        const int pair = (lane & 15) * 2;
        __half* d = P.dst.hi + row_base + pair + (lane < 16 ? 0 : P.dst.lo);
        if (row_base + pair < P.m) {
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                const uint32_t w = __byte_perm(stage[pair * OUT_PITCH + i], stage[(pair + 1) * OUT_PITCH + i], lane < 16 ? 0x5410 : 0x7632);
                if (col0 + i < P.n) *reinterpret_cast<uint32_t*>(d + (col0 + i) * P.dst.pitch) = w;
            }
        }
        __syncwarp();
    }
}

// D = A B^T over k, persistent.  A pair of CTAs per 256 x 256 tile, each with 128 rows of A and 128 columns of B.
// A stage is one box of hi and lo per operand (K-major), or two, one per 64 columns (MN-major).  Two accumulators: the next
// chunk is multiplied while the epilogue warps add the last one.
template <int MODE, bool A_MN, bool B_MN>
__global__ void __launch_bounds__(THREADS, 1) ns_product_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const Params P) {
    using namespace t5;
    constexpr int BN = 256;
    constexpr int TMEM_COLS = 2 * BN;
    constexpr int BLOCKS = BN / 64;  // 32-column blocks per epilogue warp: two warps share a row quarter
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t bars[2 * STAGES + 4];
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int abort_flag;
    const uint32_t rank = cluster_ctarank();
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint32_t* out_stage = reinterpret_cast<uint32_t*>(smem_raw + (smem_base - smem_u32(smem_raw)) + STAGES * STAGE_BYTES);
    const uint32_t bar0 = smem_u32(bars);
    auto full_bar = [&](int s) { return bar0 + 8u * s; };
    auto empty_bar = [&](int s) { return bar0 + 8u * (STAGES + s); };
    auto tfull_bar = [&](int a) { return bar0 + 8u * (2 * STAGES + a); };
    auto tempty_bar = [&](int a) { return bar0 + 8u * (2 * STAGES + 2 + a); };
    const uint32_t peer_abort = map_to_cta(smem_u32(const_cast<int*>(&abort_flag)), rank ^ 1u);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        abort_flag = 0;
        for (int s = 0; s < STAGES; ++s) { mbar_init(full_bar(s), 1); mbar_init(empty_bar(s), 1); }
        for (int a = 0; a < 2; ++a) { mbar_init(tfull_bar(a), 1); mbar_init(tempty_bar(a), EPI_WARPS * 2); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        prefetch_tmap(&map_a);
        prefetch_tmap(&map_b);
    }
    if (warp == 1) tmem_alloc<2>(smem_u32(&tmem_slot), TMEM_COLS);
    fence_before();
    __syncthreads();
    cluster_sync_all();  // the peer's barriers exist before anything is signalled across
    fence_after();
    const uint32_t tmem_base = tmem_slot;
    asm volatile("griddepcontrol.wait;" ::: "memory");  // what the kernel before wrote is there
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int first_unit = blockIdx.x / 2, unit_step = gridDim.x / 2;

    if (warp == 0) {
        if (lane == 0) {
            int stage = 0;
            uint32_t phase = 0, issued = 0;
            bool ok = true;
            for (int u = first_unit; u < P.units && ok; u += unit_step) {
                int tm, tn;
                unit_tile<MODE>(u, P, tm, tn);
                const int m0 = (tm * 2 + static_cast<int>(rank)) * BM, n0 = tn * BN + static_cast<int>(rank) * BM;
                for (int kb = 0; kb < P.num_kb; ++kb) {
                    if (!mbar_wait(empty_bar(stage), phase ^ 1u, &abort_flag, &g_ns_status, 0x100 | stage)) { ok = false; break; }
                    if (rank == 0) mbar_expect_tx(full_bar(stage), 2 * STAGE_BYTES);
                    const uint32_t fb = map_to_cta(full_bar(stage), 0);
                    const uint32_t base = smem_base + stage * STAGE_BYTES;
                    const int k0 = kb * BK;
                    if (A_MN) {
                        tma_load_3d<2>(base, &map_a, fb, m0, k0, 0);
                        tma_load_3d<2>(base + STAGE_BYTES / 4, &map_a, fb, m0 + 64, k0, 0);
                    } else {
                        tma_load_3d<2>(base, &map_a, fb, k0, m0, 0);
                    }
                    if (B_MN) {
                        tma_load_3d<2>(base + STAGE_BYTES / 2, &map_b, fb, n0, k0, 0);
                        tma_load_3d<2>(base + 3 * (STAGE_BYTES / 4), &map_b, fb, n0 + 64, k0, 0);
                    } else {
                        tma_load_3d<2>(base + STAGE_BYTES / 2, &map_b, fb, k0, n0, 0);
                    }
                    ++issued;
                    if (++stage == STAGES) { stage = 0; phase ^= 1u; }
                }
            }
            // Every stage that was filled has been released: no copy and no arrival is in flight any more.  After a wait
            // that ran out this is bounded too, and the copies in flight get a couple of milliseconds to land.
            const uint32_t pending = issued < static_cast<uint32_t>(STAGES) ? issued : STAGES;
            if (issued < static_cast<uint32_t>(STAGES)) { stage = 0; phase = 1u; }  // (the ring never came round: from its start)
            for (uint32_t i = 0; i < pending && ok; ++i) {
                if (!mbar_wait(empty_bar(stage), phase ^ 1u, &abort_flag, &g_ns_status, 0x180 | stage)) ok = false;
                if (++stage == STAGES) { stage = 0; phase ^= 1u; }
            }
            if (!ok) {
                st_cluster_u32(peer_abort, 1u);
                settle();
            }
        }
    } else if (warp == 1) {
        if (rank == 0) {
            constexpr uint32_t idesc = make_idesc(BM * 2, BN, A_MN, B_MN);
            // hi and lo of a K-major tile lie half an operand apart; of an MN-major one a quarter, inside each column group
            // (descriptors hold addresses in units of 16 bytes: every step is an addition of a constant)
            constexpr uint64_t a_lo = (A_MN ? STAGE_BYTES / 8 : STAGE_BYTES / 4) >> 4, b_lo = (B_MN ? STAGE_BYTES / 8 : STAGE_BYTES / 4) >> 4;
            constexpr uint64_t a_step = (A_MN ? 2048u : 32u) >> 4, b_step = (B_MN ? 2048u : 32u) >> 4;
            constexpr uint32_t a_lbo = A_MN ? STAGE_BYTES / 4 : 0u, b_lbo = B_MN ? STAGE_BYTES / 4 : 0u;
            int stage = 0, acc = 0;
            uint32_t phase = 0, acc_phase = 0;
            bool ok = true;
            for (int u = first_unit; u < P.units && ok; u += unit_step) {
                for (int c0 = 0; c0 < P.num_kb && ok; c0 += CHUNK_KB) {
                    const int c1 = c0 + CHUNK_KB < P.num_kb ? c0 + CHUNK_KB : P.num_kb;
                    if (!mbar_wait(tempty_bar(acc), acc_phase ^ 1u, &abort_flag, &g_ns_status, 0x200 | acc)) { ok = false; break; }
                    const uint32_t d = tmem_base + static_cast<uint32_t>(acc * BN);
                    for (int kb = c0; kb < c1; ++kb) {
                        if (!mbar_wait(full_bar(stage), phase, &abort_flag, &g_ns_status, 0x210 | stage)) { ok = false; break; }
                        fence_after();
                        const uint64_t a = make_desc(smem_base + stage * STAGE_BYTES, a_lbo), b = make_desc(smem_base + stage * STAGE_BYTES + STAGE_BYTES / 2, b_lbo);
                        __syncwarp();
                        if (elect_one()) {
#pragma unroll
                            for (int ks = 0; ks < BK / 16; ++ks) {  // the small terms first, while the accumulator is small
                                mma_f16<2>(d, a + a_lo + ks * a_step, b + ks * b_step, idesc, kb > c0 || ks > 0);
                                mma_f16<2>(d, a + ks * a_step, b + b_lo + ks * b_step, idesc, 1u);
                            }
#pragma unroll
                            for (int ks = 0; ks < BK / 16; ++ks) mma_f16<2>(d, a + ks * a_step, b + ks * b_step, idesc, 1u);
                            commit<2>(empty_bar(stage));
                            if (kb + 1 == c1) commit<2>(tfull_bar(acc));
                        }
                        if (++stage == STAGES) { stage = 0; phase ^= 1u; }
                    }
                    if (++acc == 2) { acc = 0; acc_phase ^= 1u; }
                }
            }
            if (!ok && lane == 0) st_cluster_u32(peer_abort, 1u);
        }
    } else {
        const int quarter = warp & 3, side = (warp - 2) >> 2;  // rows 32 quarter.., columns BN/2 side..
        const uint32_t te0 = map_to_cta(tempty_bar(0), 0), te1 = map_to_cta(tempty_bar(1), 0);
        const float cf[3] = {__ldg(P.coef), __ldg(P.coef + 1), __ldg(P.coef + 2)};
        uint32_t* stage = out_stage + (warp - 2) * 32 * OUT_PITCH;
        int acc = 0;
        uint32_t acc_phase = 0;
        bool ok = true;
        for (int u = first_unit; u < P.units && ok; u += unit_step) {
            int tm, tn;
            unit_tile<MODE>(u, P, tm, tn);
            float sum[BLOCKS][32];
#pragma unroll
            for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
                for (int i = 0; i < 32; ++i) sum[b][i] = 0.0f;
            for (int c0 = 0; c0 < P.num_kb; c0 += CHUNK_KB) {
                if (!mbar_wait(tfull_bar(acc), acc_phase, &abort_flag, &g_ns_status, 0x300 | acc)) { ok = false; break; }
                fence_after();
                const uint32_t t = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + static_cast<uint32_t>(acc * BN + side * (BN / 2));
#pragma unroll
                for (int b = 0; b < BLOCKS; ++b) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {  // 16 columns at a time: with 32 the sums spill (2500 x 2500: 1087 us, this way 1069)
                        uint32_t r[16];
                        tmem_ld_cols(t + b * 32 + h * 16, r);
                        tmem_ld_wait();
                        if (b == BLOCKS - 1 && h == 1) {  // read completely: the next but one chunk may go there
                            fence_before();
                            __syncwarp();
                            if (lane == 0) mbar_arrive_cluster(acc ? te1 : te0);
                        }
#pragma unroll
                        for (int i = 0; i < 16; ++i) sum[b][h * 16 + i] += __uint_as_float(r[i]);
                    }
                }
                if (++acc == 2) { acc = 0; acc_phase ^= 1u; }
            }
            if (!ok) break;
            const int row_base = (tm * 2 + static_cast<int>(rank)) * BM + quarter * 32;
            // one copy of the code, the blocks moved through its registers: unrolled four times, instruction fetch was most of an
            // epilogue's time (2500 x 2500: 1247 us unrolled, 1137 this way)
#pragma unroll 1
            for (int b = 0; b < BLOCKS; ++b) {
                emit_block<MODE>(P, MODE != APPLY && tm != tn, row_base, lane, tn * BN + side * (BN / 2) + b * 32, sum[0], stage, cf);
#pragma unroll
                for (int c = 0; c + 1 < BLOCKS; ++c)
#pragma unroll
                    for (int i = 0; i < 32; ++i) sum[c][i] = sum[c + 1][i];
            }
        }
        if (!ok && lane == 0) st_cluster_u32(peer_abort, 1u);
    }

    fence_before();
    __syncthreads();
    cluster_sync_all();  // neither CTA leaves (or frees TMEM) while the other may still signal it
    if (warp == 1) {
        fence_after();
        tmem_dealloc<2>(tmem_base, TMEM_COLS);
    }
}

__device__ __forceinline__ void split8(const float (&x)[8], uint4& hi, uint4& lo) {
    split2(x[0], x[1], hi.x, lo.x);
    split2(x[2], x[3], hi.y, lo.y);
    split2(x[4], x[5], hi.z, lo.z);
    split2(x[6], x[7], hi.w, lo.w);
}
__device__ __forceinline__ void join8(const uint4& hi, const uint4& lo, float (&x)[8]) {
    const uint32_t h[4] = {hi.x, hi.y, hi.z, hi.w}, l[4] = {lo.x, lo.y, lo.z, lo.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&h[e])), b = __half22float2(*reinterpret_cast<const __half2*>(&l[e]));
        x[2 * e] = a.x + b.x;
        x[2 * e + 1] = a.y + b.y;
    }
}

// ---- products of medium matrices -------------------------------------------------------------------------
// A 128 x 128 tile per cluster of `split` CTAs, each with its share of the k-blocks: with d up to 2048 there are few tiles,
// and a CTA alone takes its operands from L2 at one SM's rate (64 KB a k-block, about 0.9 us).  The CTAs' sums meet in L2
// (fp32, [column quad][row], so that a warp's store is one run); after a cluster barrier each CTA adds 128 / split
// columns over all of them, in rank order, and takes these through the epilogue from shared memory -- compact loops,
// because at these sizes straight-line code spends its time on instruction fetches.  What bounds it up to d of about 600 is
// latency, 6.7 - 8.5 us a launch: 1.4 us from one launch to the next, 1.4 to the first accumulator, 3 for the sums to meet, 1 for
// the epilogue.
constexpr int MID_THREADS = 576;  // warp 0 loads, warp 1 multiplies, warps 2-17: 4 per quarter of the rows, 32 columns each
constexpr int MID_MAX_CTAS = 160, MAX_SLABS = 16;
constexpr int MID_SMEM = STAGES * STAGE_BYTES + 1024;
constexpr int MID_PITCH = 129;

template <int MODE, bool A_MN, bool B_MN>
__global__ void __launch_bounds__(MID_THREADS, 1) ns_tile_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const Params P,
                                                                 float4* __restrict__ partial) {
    using namespace t5;
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t bars[2 * STAGES + 4];
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int abort_flag;
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    float* const E = reinterpret_cast<float*>(smem_raw + (smem_base - smem_u32(smem_raw)));  // after the main loop: the tile, [row][column]
    const uint32_t bar0 = smem_u32(bars);
    auto full_bar = [&](int s) { return bar0 + 8u * s; };
    auto empty_bar = [&](int s) { return bar0 + 8u * (STAGES + s); };
    auto tfull_bar = [&](int a) { return bar0 + 8u * (2 * STAGES + a); };
    auto tempty_bar = [&](int a) { return bar0 + 8u * (2 * STAGES + 2 + a); };
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int split = P.split, rank = static_cast<int>(cluster_ctarank()), cluster = blockIdx.x / split, slab = cluster / P.units, unit = cluster % P.units;
    const int share = slab * split + rank, shares = P.slabs * split;
    const int kb0 = static_cast<int>(static_cast<int64_t>(P.num_kb) * share / shares), kb1 = static_cast<int>(static_cast<int64_t>(P.num_kb) * (share + 1) / shares);
    int tm, tn;
    unit_tile<MODE>(unit, P, tm, tn);

    if (tid == 0) {
        abort_flag = 0;
        for (int s = 0; s < STAGES; ++s) { mbar_init(full_bar(s), 1); mbar_init(empty_bar(s), 1); }
        for (int a = 0; a < 2; ++a) { mbar_init(tfull_bar(a), 1); mbar_init(tempty_bar(a), 16); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        prefetch_tmap(&map_a);
        prefetch_tmap(&map_b);
    }
    if (warp == 1) tmem_alloc<1>(smem_u32(&tmem_slot), 256);
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = tmem_slot;
    asm volatile("griddepcontrol.wait;" ::: "memory");  // what the kernel before wrote is there

    float v[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = 0.0f;
    const int quarter = warp & 3, c0 = ((warp - 2) >> 2) * 32;  // epilogue warps: rows 32 quarter.., columns c0..
    if (warp == 0) {
        if (lane == 0) {
            bool ok = true;
            const int m0 = tm * BM, n0 = tn * BM;
            int issued = 0;
            for (int kb = kb0; kb < kb1; ++kb, ++issued) {
                const int st = issued % STAGES;
                if (!mbar_wait(empty_bar(st), ((issued / STAGES) & 1) ^ 1u, &abort_flag, &g_ns_status, 0x500 | st)) { ok = false; break; }
                mbar_expect_tx(full_bar(st), STAGE_BYTES);
                const uint32_t fb = full_bar(st), base = smem_base + st * STAGE_BYTES;
                const int k0 = kb * BK;
                if (A_MN) {
                    tma_load_3d<1>(base, &map_a, fb, m0, k0, 0);
                    tma_load_3d<1>(base + STAGE_BYTES / 4, &map_a, fb, m0 + 64, k0, 0);
                } else {
                    tma_load_3d<1>(base, &map_a, fb, k0, m0, 0);
                }
                if (B_MN) {
                    tma_load_3d<1>(base + STAGE_BYTES / 2, &map_b, fb, n0, k0, 0);
                    tma_load_3d<1>(base + 3 * (STAGE_BYTES / 4), &map_b, fb, n0 + 64, k0, 0);
                } else {
                    tma_load_3d<1>(base + STAGE_BYTES / 2, &map_b, fb, k0, n0, 0);
                }
            }
            // (every copy issued has been waited for by the multiplying warp unless a wait ran out: then give the copies in flight
            // a couple of milliseconds to land)
            if (!ok) settle();
        }
    } else if (warp == 1) {
        {
            constexpr uint32_t idesc = make_idesc(BM, BM, A_MN, B_MN);
            constexpr uint64_t a_lo = (A_MN ? STAGE_BYTES / 8 : STAGE_BYTES / 4) >> 4, b_lo = (B_MN ? STAGE_BYTES / 8 : STAGE_BYTES / 4) >> 4;
            constexpr uint64_t a_step = (A_MN ? 2048u : 32u) >> 4, b_step = (B_MN ? 2048u : 32u) >> 4;
            constexpr uint32_t a_lbo = A_MN ? STAGE_BYTES / 4 : 0u, b_lbo = B_MN ? STAGE_BYTES / 4 : 0u;
            for (int i = 0; i < kb1 - kb0; ++i) {
                const int st = i % STAGES, acc = i & 1;
                if (!mbar_wait(tempty_bar(acc), ((i >> 1) & 1) ^ 1u, &abort_flag, &g_ns_status, 0x600 | acc) ||
                    !mbar_wait(full_bar(st), (i / STAGES) & 1, &abort_flag, &g_ns_status, 0x610 | st)) {
                    settle();  // (the loading warp may have issued its last copies and be gone)
                    break;
                }
                fence_after();
                const uint32_t d = tmem + acc * 128;
                const uint64_t a = make_desc(smem_base + st * STAGE_BYTES, a_lbo), b = make_desc(smem_base + st * STAGE_BYTES + STAGE_BYTES / 2, b_lbo);
                __syncwarp();
                if (!elect_one()) continue;
#pragma unroll
                for (int ks = 0; ks < BK / 16; ++ks) {  // the small terms first, while the accumulator is small
                    mma_f16<1>(d, a + a_lo + ks * a_step, b + ks * b_step, idesc, ks > 0);
                    mma_f16<1>(d, a + ks * a_step, b + b_lo + ks * b_step, idesc, 1u);
                }
#pragma unroll
                for (int ks = 0; ks < BK / 16; ++ks) mma_f16<1>(d, a + ks * a_step, b + ks * b_step, idesc, 1u);
                commit<1>(empty_bar(st));
                commit<1>(tfull_bar(acc));
            }
        }
    } else {
        const uint32_t t_row = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + c0;
        for (int i = 0; i < kb1 - kb0; ++i) {
            const int acc = i & 1;
            if (!mbar_wait(tfull_bar(acc), (i >> 1) & 1, &abort_flag, &g_ns_status, 0x700 | acc)) {
                settle();
                break;
            }
            fence_after();
            uint32_t r[32];
            tmem_ld32(t_row + acc * 128, r);
            tmem_ld_wait();
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(tempty_bar(acc));
#pragma unroll
            for (int q = 0; q < 32; ++q) v[q] += __uint_as_float(r[q]);
        }
    }
    // ---- the CTAs' sums meet; this CTA's columns of the tile into E ----
    const int row = quarter * 32 + lane, cols = BM / split;  // (epilogue warps; columns this CTA finishes)
    if (split > 1) {
        if (warp >= 2) {
            float4* out = partial + (static_cast<int64_t>(blockIdx.x) * 32 + (c0 >> 2)) * BM + row;
#pragma unroll
            for (int q = 0; q < 8; ++q) __stcg(out + q * BM, make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]));
        }
        fence_before();
        cluster_sync_all();
        for (int t = tid; t < (cols / 4) * BM; t += MID_THREADS) {
            const int c = t / BM, i = t % BM;
            const float4* in = partial + (static_cast<int64_t>(cluster) * split * 32 + rank * (cols / 4) + c) * BM + i;
            float4 sum = make_float4(0.f, 0.f, 0.f, 0.f), p[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                p[k] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (k < split) p[k] = __ldcg(in + static_cast<int64_t>(k) * 32 * BM);
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) { sum.x += p[k].x; sum.y += p[k].y; sum.z += p[k].z; sum.w += p[k].w; }
            float* e = E + i * MID_PITCH + c * 4;
            e[0] = sum.x; e[1] = sum.y; e[2] = sum.z; e[3] = sum.w;
        }
    } else {
        fence_before();
        if (warp >= 2) {
#pragma unroll
            for (int q = 0; q < 32; ++q) E[row * MID_PITCH + c0 + q] = v[q];
        }
    }
    __syncthreads();
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (warp == 1) {
        fence_after();
        tmem_dealloc<1>(tmem, 256);
    }

    if (MODE == GRAM && P.slabs > 1) {  // a part of the sum: the join kernel has the epilogue
        float* to = P.slab_sums + (static_cast<int64_t>(slab) * P.units + unit) * BM * BM + rank * cols;
        for (int t = tid; t < cols * BM; t += MID_THREADS) to[t / cols * BM + t % cols] = E[t / cols * MID_PITCH + t % cols];
        return;
    }

    // ---- the epilogue, 8 columns of a row at a time ----
    const float cf0 = __ldg(P.coef), cf1 = __ldg(P.coef + 1), cf2 = __ldg(P.coef + 2);
    const int chunks = cols / 8, col_base = tn * BM + rank * cols, row_base = tm * BM;
    for (int t = tid; t < chunks * BM; t += MID_THREADS) {
        const int i = t / chunks, c = (t - i * chunks) * 8;
        const int64_t r = row_base + i, col = col_base + c;
        if (r >= P.m || col >= P.n) continue;
        float* e = E + i * MID_PITCH + c;
        float x[8];
        if (MODE != GRAM) {  // (pitches are multiples of 8: eight elements never leave the row)
            const __half* sp = P.src.hi + r * P.src.pitch + col;
            join8(__ldcg(reinterpret_cast<const uint4*>(sp)), __ldcg(reinterpret_cast<const uint4*>(sp + P.src.lo)), x);
        }
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            if (MODE == GRAM) x[q] = e[q] * (1.0f / 32768.0f);
            if (MODE == POLY) x[q] = fmaf(cf0 * 0.5f, x[q], cf1 * (1.0f / 65536.0f) * e[q]);
            if (MODE == APPLY) x[q] = cf2 * fmaf(kA, x[q], e[q] * (1.0f / 16384.0f));
        }
        if (MODE == APPLY && P.last) {
            float* out = P.sink.out + r * P.sink.ldo + col;
            for (int q = 0; q < 8; ++q)
                if (col + q < P.n) out[q] = sink_value(P.sink, x[q] * (1.0f / kScaleX), P.sink.update ? out[q] : 0.0f);
            continue;
        }
        uint4 hi, lo;
        split8(x, hi, lo);
        __half* d = P.dst.hi + r * P.dst.pitch + col;
        *reinterpret_cast<uint4*>(d) = hi;
        *reinterpret_cast<uint4*>(d + P.dst.lo) = lo;
        if (MODE != APPLY && tm != tn) {
#pragma unroll
            for (int q = 0; q < 8; ++q) e[q] = x[q];
        }
    }
    if (MODE != APPLY && tm != tn) {  // the mirror place: 8 rows of a column at a time
        __syncthreads();
        for (int t = tid; t < cols * (BM / 8); t += MID_THREADS) {
            const int c = t / (BM / 8), i = (t % (BM / 8)) * 8;
            if (col_base + c >= P.n || row_base + i >= P.m) continue;
            float x[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) x[q] = E[(i + q) * MID_PITCH + c];
            uint4 hi, lo;
            split8(x, hi, lo);
            __half* d = P.dst.hi + static_cast<int64_t>(col_base + c) * P.dst.pitch + row_base + i;
            *reinterpret_cast<uint4*>(d) = hi;
            *reinterpret_cast<uint4*>(d + P.dst.lo) = lo;
        }
    }
}

// A = X X^T from the slabs' sums, added in slab order: a thread per 8 columns of a row and, for the mirror place, 8 rows of a
// column of its tile (the other triangle is read transposed: long, thin matrices have one to a few tiles).
__global__ void __launch_bounds__(256) ns_join_kernel(const Params P) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int unit = blockIdx.x;
    int tm, tn;
    unit_tile<GRAM>(unit, P, tm, tn);
    const float* in = P.slab_sums + static_cast<int64_t>(unit) * BM * BM;
    const int64_t next = static_cast<int64_t>(P.units) * BM * BM;
    const int sides = tm == tn ? 1 : 2;
    for (int t = blockIdx.y * 256 + threadIdx.x; t < sides * BM * (BM / 8); t += gridDim.y * 256) {
        const bool mirror = t >= BM * (BM / 8);
        const int i = (t / (BM / 8)) % BM, c = t % (BM / 8) * 8;  // of the place written to: row, first of 8 columns
        const int64_t row = (mirror ? tn : tm) * BM + i, col = (mirror ? tm : tn) * BM + c;
        if (row >= P.m || col >= P.n) continue;
        float x[8] = {};
        for (int s = 0; s < P.slabs; ++s)
#pragma unroll
            for (int q = 0; q < 8; ++q) x[q] += __ldcg(in + s * next + (mirror ? (c + q) * BM + i : i * BM + c + q));
#pragma unroll
        for (int q = 0; q < 8; ++q) x[q] *= 1.0f / 32768.0f;
        uint4 hi, lo;
        split8(x, hi, lo);
        __half* d = P.dst.hi + row * P.dst.pitch + col;
        *reinterpret_cast<uint4*>(d) = hi;
        *reinterpret_cast<uint4*>(d + P.dst.lo) = lo;
    }
}

// ---- small matrices: every step in one launch ------------------------------------------------------------
// d <= 128 and L <= 2048: a cluster of C CTAs, C = 1, 2, 4, 8 or 16, holds X in shared memory, each CTA a slab of at most 128
// of the L side, from the first read of G to the last write.  A slab row is one index of the short side, 128 bytes of 64
// neighbours along L, 16-byte chunks XORed with row % 8 -- read along L it is the K-major operand of X X^T, read down the
// rows the MN-major operand of B X, so one copy serves both (a tall G is transposed on its way in and out).  A step:
//   X X^T of the slab -> global, fp32 | cluster barrier | each CTA adds d / C columns over all CTAs, in rank order, and
//   writes A's hi and lo as shared memory has them -> global | cluster barrier | one bulk copy per array brings A back |
//   A A, B and B X in each CTA for itself.
// Everything a product reads is there before it starts, so the small terms go first; an accumulator takes half of K.
// What bounds it is latency: at 784 x 128 a step is 10 us, half of it hand-overs between the CTAs, and what comes before and
// after the steps 11.  (The exchange through the other CTAs' shared memory instead of L2 took 18000 of 37000 clocks a step there:
// 64 KB in and out of every CTA at 7 bytes a clock.)
constexpr int CL_THREADS = 512;                    // 4 warps per quarter of the accumulator's rows, 32 columns each
constexpr int CL_SIDE = 128;                       // largest d, widest slab
constexpr int CL_GROUP = CL_SIDE * 128;            // bytes of a 64-wide column group of a matrix of 128 rows
constexpr int CL_MATRIX = 4 * CL_GROUP;            // hi: 2 groups, lo: 2 groups
constexpr int CL_PITCH = 132, CL_PITCH_TALL = 129;  // floats per row of the fp32 buffer, which a tall G enters and leaves down its
                                                    // columns (784 x 128 with 132: 65.4 us, with 129: 60.5)
constexpr int CL_MAX = 16;                         // CTAs of a cluster
constexpr int CL_SMEM = 2 * CL_MATRIX + CL_SIDE * CL_PITCH * 4 + 1024;
constexpr int CL_PARTIAL = CL_SIDE * CL_SIDE * 4;  // bytes of one CTA's X X^T
constexpr size_t cl_workspace(int ctas) { return ctas > 1 ? static_cast<size_t>(ctas) * CL_PARTIAL + CL_MATRIX : 0; }

// Byte offset of the 16-byte chunk with elements [8 c, 8 c + 8) of row r.
__device__ __forceinline__ uint32_t cl_chunk(int r, int c) { return static_cast<uint32_t>((c >> 3) * CL_GROUP + r * 128 + (((c & 7) ^ (r & 7)) << 4)); }

struct ClusterArgs {
    Source S;
    Sink K;
    int d, length, slab;  // short side, long side, columns of the long side per CTA (a multiple of 16)
    int steps;
    float eps;
    float4* partial;      // [C][32 column quads][128 rows]
    uint8_t* image;       // A as it lies in shared memory
};

// V elements of the long (wide G) or the short side (tall G), whichever is contiguous, at a time.
template <int V, bool MOMENTUM, bool TALL>
__global__ void __launch_bounds__(CL_THREADS, 1) ns_cluster_kernel(const ClusterArgs P) {
    using namespace t5;
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t done_bar, copy_bar;
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int abort_flag;
    __shared__ double norms[CL_MAX], sums[CL_THREADS / 32];
    uint8_t* const smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint8_t* const X = smem;                        // hi, lo of this CTA's slab: [d][slab]
    uint8_t* const A = smem + CL_MATRIX;            // hi, lo of A, then of B: [d][d]
    float* const E = reinterpret_cast<float*>(smem + 2 * CL_MATRIX);
    const uint32_t x_addr = smem_u32(X), a_addr = smem_u32(A), bar = smem_u32(&done_bar), cbar = smem_u32(&copy_bar);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = static_cast<int>(cluster_ctarank()), ctas = static_cast<int>(gridDim.x);
    const int d = P.d, d16 = (d + 15) & ~15, w16 = P.slab, n0 = rank * P.slab;
    const int width = P.length - n0 < P.slab ? (P.length - n0 > 0 ? P.length - n0 : 0) : P.slab;  // this CTA's part that exists

    constexpr int pitch = TALL ? CL_PITCH_TALL : CL_PITCH;
    if (tid == 0) {
        abort_flag = 0;
        mbar_init(bar, 1);
        mbar_init(cbar, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) tmem_alloc<1>(smem_u32(&tmem_slot), 256);
    // every operand byte a product may touch is defined: rows and columns past d and the slab are zero
    for (int i = tid; i < 2 * CL_MATRIX / 16; i += CL_THREADS) *reinterpret_cast<uint4*>(smem + i * 16) = make_uint4(0u, 0u, 0u, 0u);
    if (width < w16)
        for (int t = tid; t < d * (w16 - width); t += CL_THREADS) E[(t % d) * pitch + width + t / d] = 0.0f;

    // ---- U into E, the momentum update, the norm ----
    const Source& S = P.S;
    const int fast = (TALL ? d : width) / V, total = (TALL ? width : d) * fast;  // accesses of V elements
    constexpr int U = 4;                                                           // of them in flight per thread
    double acc = 0.0;
    for (int t0 = tid; t0 < total; t0 += U * CL_THREADS) {
        Vec<V> u[U], m[U];
        int sl[U], fa[U];
#pragma unroll
        for (int k = 0; k < U; ++k) {
            const int t = t0 + k * CL_THREADS;
            sl[k] = t / fast;
            fa[k] = (t - sl[k] * fast) * V;
            if (t >= total) continue;
            const int64_t r = TALL ? n0 + sl[k] : sl[k], c = TALL ? fa[k] : n0 + fa[k];
            u[k] = load_vec<V>(S.g + r * S.ldg + c);
            if (MOMENTUM) m[k] = load_vec<V>(S.momentum + r * S.ldm + c);
        }
#pragma unroll
        for (int k = 0; k < U; ++k) {
            if (t0 + k * CL_THREADS >= total) continue;
            if (MOMENTUM) {
#pragma unroll
                for (int q = 0; q < V; ++q) {
                    m[k].v[q] = fmaf(S.mu, m[k].v[q], u[k].v[q]);
                    u[k].v[q] = S.nesterov ? fmaf(S.mu, m[k].v[q], u[k].v[q]) : m[k].v[q];
                }
                *reinterpret_cast<Vec<V>*>(S.momentum + (TALL ? n0 + sl[k] : sl[k]) * S.ldm + (TALL ? fa[k] : n0 + fa[k])) = m[k];
            }
#pragma unroll
            for (int q = 0; q < V; ++q) {
                acc = fma(static_cast<double>(u[k].v[q]), static_cast<double>(u[k].v[q]), acc);
                E[(TALL ? fa[k] + q : sl[k]) * pitch + (TALL ? sl[k] : fa[k] + q)] = u[k].v[q];
            }
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
    if (lane == 0) sums[warp] = acc;
    cluster_sync_all();  // every CTA runs (its shared memory may be written), and this one's sums are there
    if (tid < ctas) {
        double part = 0.0;
        for (int w = 0; w < CL_THREADS / 32; ++w) part += sums[w];
        const uint32_t to = map_to_cta(smem_u32(&norms[rank]), static_cast<uint32_t>(tid));
        asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(to), "d"(part) : "memory");
    }
    cluster_sync_all();
    double sumsq = 0.0;
    for (int i = 0; i < ctas; ++i) sumsq += norms[i];
    const Normaliser N = normaliser(sumsq, P.eps);
    int e = N.e;
    for (int t = tid; t < d * (w16 / 8); t += CL_THREADS) {
        const int i = t / (w16 / 8), c = t % (w16 / 8);
        float x[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) x[q] = (E[i * pitch + c * 8 + q] * N.p2) * (N.rest * kScaleX);
        uint4 hi, lo;
        split8(x, hi, lo);
        *reinterpret_cast<uint4*>(X + cl_chunk(i, c)) = hi;
        *reinterpret_cast<uint4*>(X + 2 * CL_GROUP + cl_chunk(i, c)) = lo;
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = tmem_slot;
    uint32_t phase = 0, copy_phase = 0;
    const int row = (warp & 3) * 32 + lane, c0 = (warp >> 2) * 32;  // accumulator row and first of 32 columns of this thread
    const uint32_t t_row = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16) + c0;
    const bool live = row < d;

    // operand a (K-major) times operand b over `kk` terms, the first half of them into columns 0.., the second into 128..;
    // in each the small terms go first.
    auto product = [&](uint32_t a, uint32_t b, bool b_mn, int n, int kk) {
        if (warp != 0) return;
        __syncwarp();
        fence_after();
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        if (!elect_one()) return;
        const uint32_t idesc = make_idesc(128, 0, false, b_mn) | (static_cast<uint32_t>(n >> 3) << 17);
        // (descriptors hold addresses in units of 16 bytes: every step is an addition of a constant)
        constexpr uint64_t LO = (2 * CL_GROUP) >> 4, GROUP = CL_GROUP >> 4, K16 = 32 >> 4, K16_MN = 2048 >> 4;
        const uint64_t da = make_desc(a, 0), db = make_desc(b, b_mn ? CL_GROUP : 0);
        const uint64_t b_step = b_mn ? K16_MN : K16, b_half = b_mn ? 4 * K16_MN : GROUP;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t acc_at = tmem + h * 128;
            const uint64_t ah = da + h * GROUP, bh = db + h * b_half;
            const int n16 = kk / 16 - h * 4;
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) {
                if (ks >= n16) break;
                mma_f16<1>(acc_at, ah + LO + ks * K16, bh + ks * b_step, idesc, ks > 0);
                mma_f16<1>(acc_at, ah + ks * K16, bh + LO + ks * b_step, idesc, 1u);
            }
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) {
                if (ks >= n16) break;
                mma_f16<1>(acc_at, ah + ks * K16, bh + ks * b_step, idesc, 1u);
            }
        }
        commit<1>(bar);
    };
    // This thread's 32 columns of the last product.  (A wait that runs out is recorded; the kernel carries on to its end,
    // so that no CTA is left at a cluster barrier.)
    auto result = [&](int n, bool two, float (&v)[32]) {
        mbar_wait(bar, phase, &abort_flag, &g_ns_status, 0x400);
        phase ^= 1u;
        fence_after();
        if (c0 >= n) return false;  // (the same for the whole warp)
        uint32_t r[32];
        tmem_ld32(t_row, r);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
        if (two) {
            tmem_ld32(t_row + 128, r);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] += __uint_as_float(r[i]);
        }
        return live;
    };
    // The 16-byte chunk q of this thread's 32 columns, of hi or (lo != 0) lo.
    auto chunk_of = [&](uint8_t* m, int q, int lo) { return reinterpret_cast<uint4*>(m + lo * 2 * CL_GROUP + cl_chunk(row, (c0 >> 3) + q)); };

    for (int s = 0; s < P.steps; ++s) {
        const int drop = e < 2 ? e : 2;
        const float cb = ldexpf(kB, -2 * e) * 0.5f, cc = ldexpf(kC, -4 * e) * (1.0f / 65536.0f);
        const bool last = s + 1 == P.steps;
        const float f = ldexpf(1.0f, last ? -e : -drop);
        e -= drop;
        float v[32];

        // ---- A = X X^T ----
        product(x_addr, x_addr, false, d16, w16);
        if (result(d16, w16 > 64, v)) {
            if (ctas == 1) {
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    if (c0 + q * 8 >= d16) break;
                    float x[8];
#pragma unroll
                    for (int k = 0; k < 8; ++k) x[k] = v[q * 8 + k] * (1.0f / 32768.0f);
                    uint4 hi, lo;
                    split8(x, hi, lo);
                    *chunk_of(A, q, 0) = hi;
                    *chunk_of(A, q, 1) = lo;
                }
            } else {
                float4* out = P.partial + (rank * 32 + (c0 >> 2)) * CL_SIDE + row;
#pragma unroll
                for (int q = 0; q < 8; ++q)
                    if (c0 + q * 4 < d16) __stcg(out + q * CL_SIDE, make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]));
            }
        }
        if (ctas == 1) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            fence_before();
            __syncthreads();
        } else {
            fence_before();
            cluster_sync_all();
            const int quads = d16 / 4;
            for (int t = tid; t < ((quads - rank + ctas - 1) / ctas) * CL_SIDE; t += CL_THREADS) {
                const int c = rank + (t / CL_SIDE) * ctas, i = t % CL_SIDE;  // columns 4c.., row i
                if (c >= quads || i >= d) continue;
                float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
                for (int k0 = 0; k0 < ctas; k0 += 8) {
                    float4 p[8];
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        p[k] = make_float4(0.f, 0.f, 0.f, 0.f);
                        if (k0 + k < ctas) p[k] = __ldcg(P.partial + ((k0 + k) * 32 + c) * CL_SIDE + i);
                    }
#pragma unroll
                    for (int k = 0; k < 8; ++k) { sum.x += p[k].x; sum.y += p[k].y; sum.z += p[k].z; sum.w += p[k].w; }
                }
                constexpr float S2 = 1.0f / 32768.0f;
                uint2 hi, lo;
                split2(sum.x * S2, sum.y * S2, hi.x, lo.x);
                split2(sum.z * S2, sum.w * S2, hi.y, lo.y);
                uint8_t* to = P.image + cl_chunk(i, c >> 1) + (c & 1) * 8;
                __stcg(reinterpret_cast<uint2*>(to), hi);
                __stcg(reinterpret_cast<uint2*>(to + 2 * CL_GROUP), lo);
            }
            asm volatile("fence.proxy.async;" ::: "memory");  // the copies below read what these stores wrote
            cluster_sync_all();
            const int groups = d16 > 64 ? 2 : 1;
            if (tid == 0) {
                asm volatile("fence.proxy.async;" ::: "memory");
                mbar_expect_tx(cbar, static_cast<uint32_t>(2 * groups * d * 128));
                for (int g = 0; g < 2 * groups; ++g) {
                    const uint32_t at = ((g & 1) * 2 + (g >> 1)) * CL_GROUP;  // hi and lo of group 0, then of group 1
                    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                                 ::"r"(a_addr + at), "l"(P.image + at), "r"(static_cast<uint32_t>(d * 128)), "r"(cbar) : "memory");
                }
            }
            mbar_wait(cbar, copy_phase, &abort_flag, &g_ns_status, 0x410);
            copy_phase ^= 1u;
        }

        // ---- B = b A + c A A, in A's place ----
        product(a_addr, a_addr, false, d16, d16);
        if (result(d16, d16 > 64, v)) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                if (c0 + q * 8 >= d16) break;
                float x[8];
                uint4 hi = *chunk_of(A, q, 0), lo = *chunk_of(A, q, 1);
                join8(hi, lo, x);
#pragma unroll
                for (int k = 0; k < 8; ++k) x[k] = fmaf(cb, x[k], cc * v[q * 8 + k]);
                split8(x, hi, lo);
                *chunk_of(A, q, 0) = hi;
                *chunk_of(A, q, 1) = lo;
            }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        fence_before();
        __syncthreads();

        // ---- X = f (a X + B X) ----
        product(a_addr, x_addr, true, w16, d16);
        if (result(w16, d16 > 64, v)) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                if (c0 + q * 8 >= w16) break;
                float x[8];
                uint4 hi = *chunk_of(X, q, 0), lo = *chunk_of(X, q, 1);
                join8(hi, lo, x);
#pragma unroll
                for (int k = 0; k < 8; ++k) x[k] = f * fmaf(kA, x[k], v[q * 8 + k] * (1.0f / 16384.0f));
                if (last) {
                    float* out = E + row * pitch + c0 + q * 8;
                    if constexpr (TALL) {
#pragma unroll
                        for (int k = 0; k < 8; ++k) out[k] = x[k];
                    } else {
                        reinterpret_cast<float4*>(out)[0] = make_float4(x[0], x[1], x[2], x[3]);
                        reinterpret_cast<float4*>(out)[1] = make_float4(x[4], x[5], x[6], x[7]);
                    }
                } else {
                    split8(x, hi, lo);
                    *chunk_of(X, q, 0) = hi;
                    *chunk_of(X, q, 1) = lo;
                }
            }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        fence_before();
        __syncthreads();
    }

    // ---- the result ----
    for (int t0 = tid; t0 < total; t0 += U * CL_THREADS) {
        Vec<V> old[U];
        float* at[U];
#pragma unroll
        for (int k = 0; k < U; ++k) {
            const int t = t0 + k * CL_THREADS, sl = t / fast, fa = (t - sl * fast) * V;
            at[k] = P.K.out + (TALL ? n0 + sl : sl) * P.K.ldo + (TALL ? fa : n0 + fa);
            if (P.K.update && t < total) old[k] = load_vec<V>(at[k]);
        }
#pragma unroll
        for (int k = 0; k < U; ++k) {
            const int t = t0 + k * CL_THREADS, sl = t / fast, fa = (t - sl * fast) * V;
            if (t >= total) continue;
            Vec<V> o;
#pragma unroll
            for (int q = 0; q < V; ++q)
                o.v[q] = sink_value(P.K, E[(TALL ? fa + q : sl) * pitch + (TALL ? sl : fa + q)] * (1.0f / kScaleX), P.K.update ? old[k].v[q] : 0.0f);
            *reinterpret_cast<Vec<V>*>(at[k]) = o;
        }
    }
    if (abort_flag) settle();
    if (ctas > 1) cluster_sync_all();  // no CTA leaves while another may still signal it
    else __syncthreads();
    if (warp == 0) {
        fence_after();
        tmem_dealloc<1>(tmem, 256);
    }
}

// ---- host side -------------------------------------------------------------------------------------------
// {inner, outer, hi | lo} with box {64, box_outer, 2}: one copy brings hi and lo.  Elements past an extent read as zero.
ctk_status make_map(CUtensorMap* map, const Pair& p, int64_t inner, int64_t outer, int box_outer) {
    t5::EncodeTiledFn enc;
    ctk_status st = t5::get_encoder(&enc);
    if (st) return st;
    const cuuint64_t dims[3] = {static_cast<cuuint64_t>(inner), static_cast<cuuint64_t>(outer), 2u};
    const cuuint64_t strides[2] = {static_cast<cuuint64_t>(p.pitch) * 2, static_cast<cuuint64_t>(p.lo) * 2};
    const cuuint32_t box[3] = {64u, static_cast<cuuint32_t>(box_outer), 2u}, estr[3] = {1u, 1u, 1u};
    const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, p.hi, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                           CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(CTK_ERR_CUDA, "cuTensorMapEncodeTiled failed with code " + std::to_string(static_cast<int>(r)));
    return CTK_OK;
}

template <int MODE, bool A_MN, bool B_MN>
ctk_status launch_product(const CUtensorMap& a, const CUtensorMap& b, Params P, cudaStream_t st) {
    auto kernel = ns_product_kernel<MODE, A_MN, B_MN>;
    static std::atomic<int> resident[64];  // tiles in flight on a device
    int dev = 0;
    CTK_CUDA(cudaGetDevice(&dev));
    CTK_REQUIRE(dev >= 0 && dev < 64, "device ordinal out of range");
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = SMEM_BYTES;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int at_once = resident[dev];
    if (!at_once) {
        CTK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES));
        cfg.gridDim = dim3(static_cast<unsigned>(2 * ctk::sm_count()));
        CTK_CUDA(cudaOccupancyMaxActiveClusters(&at_once, kernel, &cfg));
        CTK_REQUIRE(at_once > 0, "the device cannot hold the orthogonalisation kernel");
        resident[dev] = at_once;
    }
    constexpr int T = BM * 2;
    P.tiles_m = (P.m + T - 1) / T;
    P.tiles_n = (P.n + T - 1) / T;
    P.units = MODE == APPLY ? P.tiles_m * P.tiles_n : P.tiles_n * (P.tiles_n + 1) / 2;
    cfg.gridDim = dim3(static_cast<unsigned>(2 * (P.units < at_once ? P.units : at_once)));
    cfg.numAttrs = 2;
    CTK_CUDA(cudaLaunchKernelEx(&cfg, kernel, a, b, P));
    CTK_LAUNCH_CHECK("ns_product_kernel");
    return CTK_OK;
}

// PDL: the launch may start before the kernel in front of it has ended, up to its griddepcontrol.wait.
template <int MODE, bool A_MN, bool B_MN>
ctk_status launch_tile(const CUtensorMap& a, const CUtensorMap& b, Params P, float4* partial, cudaStream_t st) {
    auto kernel = ns_tile_kernel<MODE, A_MN, B_MN>;
    static ctk::PerDeviceReady ready;
    const ctk_status rc = ready.ensure([&]() -> ctk_status {
        CTK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, MID_SMEM));
        return CTK_OK;
    });
    if (rc) return rc;
    P.tiles_m = (P.m + BM - 1) / BM;
    P.tiles_n = (P.n + BM - 1) / BM;
    P.units = MODE == APPLY ? P.tiles_m * P.tiles_n : P.tiles_n * (P.tiles_n + 1) / 2;
    // as many CTAs to a tile as the SMs hold at once, each with a k-block at least, where four k-blocks or more pay for the
    // hand-over (130 x 140, three of them: 116 us in one CTA, 136 in two; 256 x 256, four: 144 and 116 us in four)
    P.split = 1;
    while (P.split < 8 && P.num_kb >= 4 && P.units * P.split * 2 <= MID_MAX_CTAS && P.units * P.split * 2 <= ctk::sm_count() && P.split * 2 <= P.num_kb) P.split *= 2;
    // a long, thin matrix has few tiles and very many k-blocks: several clusters to a tile (128 x 50000: 336 us in all)
    P.slabs = 1;
    if (MODE == GRAM && P.split == 8)
        while (P.slabs < MAX_SLABS && P.units * 8 * P.slabs * 2 <= MID_MAX_CTAS && P.units * 8 * P.slabs * 2 <= ctk::sm_count() && P.num_kb >= 8 * P.slabs * 8) P.slabs *= 2;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(P.split);
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3(static_cast<unsigned>(P.units * P.slabs * P.split));
    cfg.blockDim = dim3(MID_THREADS);
    cfg.dynamicSmemBytes = MID_SMEM;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    CTK_CUDA(cudaLaunchKernelEx(&cfg, kernel, a, b, P, partial));
    CTK_LAUNCH_CHECK("ns_tile_kernel");
    if (P.slabs > 1) {
        cfg.gridDim = dim3(static_cast<unsigned>(P.units), 8u);
        cfg.blockDim = dim3(256);
        cfg.dynamicSmemBytes = 0;
        cfg.attrs = attr + 1;
        cfg.numAttrs = 1;
        CTK_CUDA(cudaLaunchKernelEx(&cfg, ns_join_kernel, P));
        CTK_LAUNCH_CHECK("ns_join_kernel");
    }
    return CTK_OK;
}

struct Layout {
    size_t partial, coef, x[2], a, b, sums, slabs, total;
    int64_t pitch_x, pitch_d;
};
constexpr int MAX_PARTS = 1024, MAX_STEPS = 64;
// Short sides up to this take the medium kernels (with / without: 1300 x 1300 302 / 533 us, 2048 x 2048 544 / 729, 2048 x 4096
// 863 / 1084, 2500 x 2500 1454 / 1253 before the pairs' epilogue was made shorter).
constexpr int64_t MID_SIDE = 2048;
Layout layout_for(int64_t rows, int64_t cols) {
    Layout L;
    const int64_t d = rows < cols ? rows : cols;
    L.pitch_x = (cols + 7) / 8 * 8;
    L.pitch_d = (d + 7) / 8 * 8;
    size_t at = 0;
    auto take = [&](size_t b) { const size_t p = at; at += (b + 255) & ~size_t(255); return p; };
    L.partial = take(MAX_PARTS * sizeof(double));
    L.coef = take(MAX_STEPS * 4 * sizeof(float));
    L.x[0] = take(static_cast<size_t>(rows) * L.pitch_x * 4);
    L.x[1] = take(static_cast<size_t>(rows) * L.pitch_x * 4);
    L.a = take(static_cast<size_t>(d) * L.pitch_d * 4);
    L.b = take(static_cast<size_t>(d) * L.pitch_d * 4);
    L.sums = take(d > MID_SIDE ? 0 : static_cast<size_t>(MID_MAX_CTAS) * BM * BM * 4);
    L.slabs = take(d > MID_SIDE ? 0 : static_cast<size_t>(MID_MAX_CTAS / 8) * BM * BM * 4);  // (slabs x tiles <= MID_MAX_CTAS / 8)
    L.total = at;
    return L;
}

ctk_status run_steps(const Layout& L, char* ws, int64_t rows, int64_t cols, Sink K, int steps, cudaStream_t st) {
    const bool tall = rows > cols;
    const int64_t d = tall ? cols : rows;
    Pair X[2], A, B;
    for (int i = 0; i < 2; ++i) X[i] = Pair{reinterpret_cast<__half*>(ws + L.x[i]), L.pitch_x, rows * L.pitch_x};
    A = Pair{reinterpret_cast<__half*>(ws + L.a), L.pitch_d, d * L.pitch_d};
    B = Pair{reinterpret_cast<__half*>(ws + L.b), L.pitch_d, d * L.pitch_d};
    CUtensorMap mx_k[2], mx_mn[2], ma, mb;
    ctk_status rc = CTK_OK;
    for (int i = 0; i < 2 && !rc; ++i) {
        rc = make_map(&mx_k[i], X[i], cols, rows, 128);
        if (!rc) rc = make_map(&mx_mn[i], X[i], cols, rows, 64);
    }
    if (!rc) rc = make_map(&ma, A, d, d, 128);
    if (!rc) rc = make_map(&mb, B, d, d, 128);
    const float* coef = reinterpret_cast<const float*>(ws + L.coef);
    const bool medium = d <= MID_SIDE;
    // B X of a medium matrix that has more 128 x 128 tiles than SMs: the pairs' 256 x 256 tiles take half the operand traffic and
    // no second round (with / without: 784 x 4096 283 / 300 us, 2048 x 2048 533 / 593, 2048 x 4096 843 / 988) -- unless too much
    // of them lies past the edges (300 x 20000 389 / 370, 50000 x 128 384 / 336, 20 x 100000 558 / 387)
    const int64_t apply_tiles = ((rows + BM - 1) / BM) * ((cols + BM - 1) / BM), pair_tiles = ((rows + 2 * BM - 1) / (2 * BM)) * ((cols + 2 * BM - 1) / (2 * BM));
    const bool apply_pairs = !medium || (apply_tiles > ctk::sm_count() && 16 * pair_tiles <= 5 * apply_tiles);
    float4* sums = reinterpret_cast<float4*>(ws + L.sums);
    auto blocks = [](int64_t k) { return static_cast<int>((k + BK - 1) / BK); };
    for (int s = 0; s < steps && !rc; ++s) {
        const int at = s & 1;
        Params P = {};
        P.coef = coef + 4 * s;
        P.sink = K;
        P.m = P.n = static_cast<int>(d);
        P.num_kb = blocks(tall ? rows : cols);
        P.dst = A;
        P.slab_sums = reinterpret_cast<float*>(ws + L.slabs);
        if (medium) rc = tall ? launch_tile<GRAM, true, true>(mx_mn[at], mx_mn[at], P, sums, st) : launch_tile<GRAM, false, false>(mx_k[at], mx_k[at], P, sums, st);
        else rc = tall ? launch_product<GRAM, true, true>(mx_mn[at], mx_mn[at], P, st) : launch_product<GRAM, false, false>(mx_k[at], mx_k[at], P, st);
        if (rc) return rc;
        P.num_kb = blocks(d);
        P.src = A;
        P.dst = B;
        rc = medium ? launch_tile<POLY, false, false>(ma, ma, P, sums, st) : launch_product<POLY, false, false>(ma, ma, P, st);
        if (rc) return rc;
        P.m = static_cast<int>(rows);
        P.n = static_cast<int>(cols);
        P.src = X[at];
        P.dst = X[at ^ 1];
        P.last = s + 1 == steps;
        if (!apply_pairs) rc = tall ? launch_tile<APPLY, false, false>(mx_k[at], mb, P, sums, st) : launch_tile<APPLY, false, true>(mb, mx_mn[at], P, sums, st);
        else rc = tall ? launch_product<APPLY, false, false>(mx_k[at], mb, P, st) : launch_product<APPLY, false, true>(mb, mx_mn[at], P, st);
    }
    return rc;
}

template <int V, bool MOMENTUM, bool TALL>
ctk_status launch_cluster(const ClusterArgs& P, int ctas, cudaStream_t st) {
    auto kernel = ns_cluster_kernel<V, MOMENTUM, TALL>;
    static ctk::PerDeviceReady ready;
    const ctk_status rc = ready.ensure([&]() -> ctk_status {
        CTK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, CL_SMEM));
        CTK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        return CTK_OK;
    });
    if (rc) return rc;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(ctas);
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3(static_cast<unsigned>(ctas));
    cfg.blockDim = dim3(CL_THREADS);
    cfg.dynamicSmemBytes = CL_SMEM;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    CTK_CUDA(cudaLaunchKernelEx(&cfg, kernel, P));
    CTK_LAUNCH_CHECK("ns_cluster_kernel");
    return CTK_OK;
}

// How many CTAs take a matrix in one launch, 0 if it is too large for that.
int cluster_ctas(int64_t d, int64_t length) {
    if (d > CL_SIDE || length > CL_MAX * CL_SIDE) return 0;
    int ctas = 1;
    while (ctas * CL_SIDE < length) ctas *= 2;
    return ctas;
}
size_t workspace_for(int64_t rows, int64_t cols) {
    const int ctas = cluster_ctas(rows < cols ? rows : cols, rows < cols ? cols : rows);
    return ctas ? (cl_workspace(ctas) ? cl_workspace(ctas) : 256) : layout_for(rows, cols).total;
}

ctk_status newton_schulz(const Source& S, Sink K, int steps, float eps, void* workspace, void* stream) {
    const int64_t d = S.rows < S.cols ? S.rows : S.cols, length = S.rows < S.cols ? S.cols : S.rows;
    const bool vec = S.cols % 4 == 0 && S.ldg % 4 == 0 && aligned_to(S.g, 16) && (!S.momentum || (S.ldm % 4 == 0 && aligned_to(S.momentum, 16)));
    K.vec = K.ldo % 4 == 0 && aligned_to(K.out, 16);
    StreamScratch scratch;
    const int ctas = cluster_ctas(d, length);
    if (!workspace && ctas != 1) {
        ctk_status st = scratch.get(workspace_for(S.rows, S.cols), stream);
        if (st) return st;
        workspace = scratch.p;
    }
    if (ctas) {
        ClusterArgs P = {};
        P.S = S;
        P.K = K;
        P.d = static_cast<int>(d);
        P.length = static_cast<int>(length);
        P.slab = static_cast<int>((length + ctas - 1) / ctas + 15) / 16 * 16;
        P.steps = steps;
        P.eps = eps;
        P.partial = static_cast<float4*>(workspace);
        P.image = static_cast<uint8_t*>(workspace) + static_cast<size_t>(ctas) * CL_PARTIAL;
        const bool v4 = vec && K.vec;
        cudaStream_t st = as_stream(stream);
        if (S.rows > S.cols) {
            if (S.momentum) return v4 ? launch_cluster<4, true, true>(P, ctas, st) : launch_cluster<1, true, true>(P, ctas, st);
            return v4 ? launch_cluster<4, false, true>(P, ctas, st) : launch_cluster<1, false, true>(P, ctas, st);
        }
        if (S.momentum) return v4 ? launch_cluster<4, true, false>(P, ctas, st) : launch_cluster<1, true, false>(P, ctas, st);
        return v4 ? launch_cluster<4, false, false>(P, ctas, st) : launch_cluster<1, false, false>(P, ctas, st);
    }
    const Layout L = layout_for(S.rows, S.cols);
    char* ws = static_cast<char*>(workspace);
    double* partial = reinterpret_cast<double*>(ws + L.partial);
    float* coef = reinterpret_cast<float*>(ws + L.coef);
    cudaStream_t st = as_stream(stream);
    int grid = ctk_stream_grid(S.rows * S.cols / (vec ? 4 : 1), PREP_THREADS, 6);
    if (grid > MAX_PARTS) grid = MAX_PARTS;
    const Pair X0{reinterpret_cast<__half*>(ws + L.x[0]), L.pitch_x, S.rows * L.pitch_x};
    auto prep = [&](auto norm, auto split) -> ctk_status {
        norm<<<grid, PREP_THREADS, 0, st>>>(S, partial);
        CTK_LAUNCH_CHECK("orthogonalize: norm");
        split<<<grid, PREP_THREADS, 0, st>>>(S, partial, grid, eps, steps, X0, coef);
        CTK_LAUNCH_CHECK("orthogonalize: split");
        return CTK_OK;
    };
    ctk_status rc = S.momentum ? (vec ? prep(prep_norm_kernel<4, true>, prep_split_kernel<4, true>) : prep(prep_norm_kernel<1, true>, prep_split_kernel<1, true>))
                               : (vec ? prep(prep_norm_kernel<4, false>, prep_split_kernel<4, false>) : prep(prep_norm_kernel<1, false>, prep_split_kernel<1, false>));
    if (rc) return rc;
    return run_steps(L, ws, S.rows, S.cols, K, steps, st);
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
    return workspace_for(rows, cols);
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
    const Sink K{out, ldo, 0, 0.0f, 0.0f, 0};
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
    const Sink K{p, ldp, 1, 1.0f - lr * weight_decay, lr * scale, 0};
    return newton_schulz(S, K, steps, eps, workspace, stream);
}

ctk_status ctk_orthogonalize_status(int* status) {
    CTK_REQUIRE(status, "ctk_orthogonalize_status: null pointer");
    CTK_CUDA(cudaDeviceSynchronize());
    CTK_CUDA(cudaMemcpyFromSymbol(status, g_ns_status, sizeof(int)));
    return CTK_OK;
}

}  // extern "C"
