// 4-bit weights with group scales: quantising, the values they stand for, and y = [relu](x W + bias).
// The layout is described in ctorch_b200.h.
#include <cuda_bf16.h>

#include "common.cuh"

namespace {
using namespace ctk;

constexpr int W4_THREADS = 256;

// Bit position of code i of a word: the pairs (2p, 2p+1) sit 16 bits apart, so one mask takes both as the
// two halves of a register.
__host__ __device__ constexpr int nibble_shift(int i) { return 4 * (i >> 1) + 16 * (i & 1); }

// ---- quantise ------------------------------------------------------------------------------------------
// A thread owns one group of one column: lanes are neighbouring columns (coalesced rows of w), the group's
// GROUP values stay in registers between the maximum and the rounding, so w is read once, with up to GROUP
// loads in flight per thread.  Bound by w's bytes.
//
// round(w / s) exactly: with q = round(w * (1/s)) at most one step off, the remainder d = w - q s is exact in one
// fma (|d| <= s (1/2 + tiny), a multiple of the smaller of both ulps), so comparing 2|d| with s decides the
// rounding and its ties without a division.
__device__ __forceinline__ float round_quotient(float w, float s, float inv) {
    float q = rintf(w * inv);
    const float d = fmaf(-q, s, w), e = 2.0f * fabsf(d);
    if (e > s || (e == s && (static_cast<int>(q) & 1))) q += d > 0.0f ? 1.0f : -1.0f;
    return q;
}

template <int GROUP, bool SYM>
__global__ void __launch_bounds__(W4_THREADS) w4_quantize_kernel(const float* __restrict__ w, int64_t ldw, int64_t k, int64_t n, int64_t groups,
                                                                 uint32_t* __restrict__ packed, float* __restrict__ scales, uint8_t* __restrict__ zeros) {
    const int64_t j = static_cast<int64_t>(blockIdx.x) * 32 + (threadIdx.x & 31);
    const int64_t grp = static_cast<int64_t>(blockIdx.y) * (W4_THREADS / 32) + (threadIdx.x >> 5);
    if (j >= n || grp >= groups) return;
    const int64_t k0 = grp * GROUP;
    const int len = static_cast<int>(k - k0 < GROUP ? k - k0 : GROUP);
    const float* src = w + k0 * ldw + j;
    float v[GROUP];
#pragma unroll
    for (int i = 0; i < GROUP; ++i) v[i] = i < len ? __ldcs(src + i * ldw) : 0.0f;
    float top = 0.0f, bottom = 0.0f, poison = 0.0f;
#pragma unroll
    for (int i = 0; i < GROUP; ++i) {
        top = fmaxf(top, SYM ? fabsf(v[i]) : v[i]);
        if (!SYM) bottom = fminf(bottom, v[i]);
        poison = fmaf(v[i], 0.0f, poison);  // NaN once a value is not finite
    }
    // the one division of the group, in 64 bits so that the scale is the nearest fp32 number
    const float s = poison == 0.0f ? static_cast<float>(SYM ? static_cast<double>(top) / 7.0 : (static_cast<double>(top) - static_cast<double>(bottom)) / 15.0)
                                   : __int_as_float(0x7fc00000);
    const bool live = s > 0.0f;  // false for a group of zeros and for NaN
    float zero = 8.0f;
    if (!SYM) zero = live ? static_cast<float>(rint(-static_cast<double>(bottom) / static_cast<double>(s))) : 0.0f;
    if (!SYM && zero > 15.0f) zero = 15.0f;  // (subnormal scales only: the range is no longer 15 steps wide)
    const float inv = 1.0f / s;
    const bool plain = live && inv <= 3.0e38f;  // else s is subnormal and 1/s overflows: divide in 64 bits
    uint32_t* dst = packed + j * (groups * (GROUP / 8)) + grp * (GROUP / 8);
#pragma unroll
    for (int q4 = 0; q4 < GROUP / 32; ++q4) {
        uint4 out;
        uint32_t* o = &out.x;
#pragma unroll
        for (int wd = 0; wd < 4; ++wd) {
            uint32_t word = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float x = v[q4 * 32 + wd * 8 + i];
                float c = zero;
                if (plain) c += round_quotient(x, s, inv);
                else if (live) c += static_cast<float>(rint(static_cast<double>(x) / static_cast<double>(s)));
                c = fminf(fmaxf(c, SYM ? 1.0f : 0.0f), 15.0f);
                word |= static_cast<uint32_t>(c) << nibble_shift(i);
            }
            o[wd] = word;
        }
        *reinterpret_cast<uint4*>(dst + q4 * 4) = out;
    }
    scales[j * groups + grp] = s;
    if (!SYM) zeros[j * groups + grp] = static_cast<uint8_t>(zero);
}

// ---- dequantise ----------------------------------------------------------------------------------------
// A thread takes 32 k of one column: one 16-byte load of codes, 32 coalesced stores (lanes are columns).
__global__ void __launch_bounds__(W4_THREADS) w4_dequantize_kernel(const uint32_t* __restrict__ packed, const float* __restrict__ scales,
                                                                   const uint8_t* __restrict__ zeros, int64_t k, int64_t n, int group, int64_t groups,
                                                                   float* __restrict__ w, int64_t ldw) {
    const int64_t j = static_cast<int64_t>(blockIdx.x) * 32 + (threadIdx.x & 31);
    const int64_t k0 = (static_cast<int64_t>(blockIdx.y) * (W4_THREADS / 32) + (threadIdx.x >> 5)) * 32;
    if (j >= n || k0 >= k) return;
    const int64_t grp = k0 / group;
    const uint4 c = __ldg(reinterpret_cast<const uint4*>(packed + j * (groups * (group / 8)) + k0 / 8));
    const float s = scales[j * groups + grp];
    const float zero = zeros ? static_cast<float>(zeros[j * groups + grp]) : 8.0f;
    const uint32_t word[4] = {c.x, c.y, c.z, c.w};
    float* dst = w + k0 * ldw + j;
    const int len = static_cast<int>(k - k0 < 32 ? k - k0 : 32);
#pragma unroll
    for (int i = 0; i < 32; ++i)
        if (i < len) __stcs(dst + i * ldw, (static_cast<float>((word[i >> 3] >> nibble_shift(i & 7)) & 15u) - zero) * s);
}

// ---- y = [relu](x W + bias) ------------------------------------------------------------------------------
// mma.sync on exact factors.  A code minus its zero point is an integer of at most 4 bits and a sign, exact in bf16; x is cut
// into three bf16 parts of 8 bits that add up to it exactly (by truncation: no part overflows); the products are
// exact and meet in fp32.  Within a group the tensor core adds (8 instructions at most), the group's sum is scaled and
// added to the result with one rounded fma: fp32 accuracy with no conversion of the weight but the mask that puts two codes
// beside each other under bf16's exponent (0x4300 | code = 128 + code) and one packed subtraction.
//
// The weight is the instruction's A (16 output columns by 16 k), the parts of x its B: eight columns, (row, part) pairs, so one
// instruction serves two rows and NT of them 8 NT / 3.  k may be taken in any order as long as A and B agree: thread t of a
// quad holds GROUP / 32 whole words of a group, as they lie in memory.  For few rows the weight's bytes are the bound
// (per 128 k of 16 columns: 1 KB, 72 instructions to unpack, 8 NT products), from NT = 3 on the products.
//
// A CTA: 8 warps of 16 columns each; a cluster of `split` CTAs shares the k of its columns.  x's parts lie in shared memory (XC k at a time), 16-byte pieces ordered so that a quad's four pieces are neighbours.
constexpr int MM_THREADS = 256, MM_COLS = 128, R_PITCH = 132;
template <int NT>
struct MmCfg {
    static constexpr int XC = NT == 1 ? 2048 : NT <= 3 ? 1024 : 512;  // k of x held at a time
    static constexpr int PITCH = XC * 2 + 64;                         // bytes per (row, part): 4 pieces past a multiple of 8, no bank conflicts
    static constexpr int X_BYTES = 8 * NT * PITCH;
    static constexpr int R_BYTES = 8 * NT * R_PITCH * 4;                  // a CTA's sums, [(row, part)][column], in the same place afterwards
    static constexpr int SMEM = X_BYTES > R_BYTES ? X_BYTES : R_BYTES;
    static constexpr int ROWS = 8 * NT / 3;
};

struct MmArgs {
    const float* x;
    int64_t ldx;
    const uint32_t* packed;
    const float* scales;
    const uint8_t* zeros;
    const float* bias;
    float* y;
    int64_t ldy;
    int64_t m, k, n, groups;
    int relu, split;
    int vec_x;  // x can be read 16 bytes at a time
};

__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// codes (2p, 2p+1) of a word, minus the zero point: two bf16 integers
__device__ __forceinline__ uint32_t pair_of(uint32_t word, int p, uint32_t zero2) {
    const uint32_t biased = ((word >> (4 * p)) & 0x000F000Fu) | 0x43004300u;
    const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&biased), *reinterpret_cast<const __nv_bfloat162*>(&zero2));
    return *reinterpret_cast<const uint32_t*>(&d);
}
// x = p0 + p1 + p2 in bits 16-31 of the three: 8 leading bits each, truncated, so the sum is exact
__device__ __forceinline__ void cut3(float x, uint32_t (&p)[3]) {
    const uint32_t u = __float_as_uint(x);
    if ((u & 0x7F800000u) == 0x7F800000u) {  // infinities stay, NaN stays NaN
        p[0] = (u & 0x007FFFFFu) ? 0x7FC00000u : u;
        p[1] = p[2] = 0u;
        return;
    }
    p[0] = u & 0xFFFF0000u;
    const float r = x - __uint_as_float(p[0]);
    p[1] = __float_as_uint(r) & 0xFFFF0000u;
    p[2] = __float_as_uint(r - __uint_as_float(p[1]));
}

template <int GROUP>
struct Words;
template <>
struct Words<32> { uint32_t w[1]; };
template <>
struct __align__(8) Words<64> { uint32_t w[2]; };
template <>
struct __align__(16) Words<128> { uint32_t w[4]; };

template <int GROUP>
__device__ __forceinline__ Words<GROUP> load_words(const uint32_t* p) {
    Words<GROUP> r;
    if (GROUP == 32) {
        r.w[0] = __ldg(p);
    } else if (GROUP == 64) {
        *reinterpret_cast<uint2*>(&r) = __ldg(reinterpret_cast<const uint2*>(p));
    } else {
        *reinterpret_cast<uint4*>(&r) = __ldg(reinterpret_cast<const uint4*>(p));
    }
    return r;
}

template <int GROUP, int NT>
__global__ void __launch_bounds__(MM_THREADS, 2) w4_matmul_kernel(const MmArgs P) {
    using C = MmCfg<NT>;
    constexpr int W = GROUP / 32;             // words of a group per thread of a quad
    constexpr int AHEAD = GROUP == 32 ? 8 : 4;  // groups whose words are in flight
    extern __shared__ __align__(16) uint8_t smem[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gr = lane >> 2, qt = lane & 3;
    const int split = P.split, rank = blockIdx.x % split;
    const int64_t col_base = static_cast<int64_t>(blockIdx.x / split) * MM_COLS, row_base = static_cast<int64_t>(blockIdx.y) * C::ROWS;
    const int rows = static_cast<int>(P.m - row_base < C::ROWS ? P.m - row_base : C::ROWS);
    // this CTA's groups, taken XC / GROUP at a time
    const int g_begin = static_cast<int>(P.groups * rank / split), g_end = static_cast<int>(P.groups * (rank + 1) / split);
    constexpr int PIECE = C::XC / GROUP;
    static_assert(PIECE % AHEAD == 0, "a piece starts at held[0]");
    const bool idle = col_base + warp * 16 >= P.n;  // this warp has no columns: it only helps with x

    const int64_t j0 = col_base + warp * 16 + gr, j1 = j0 + 8;  // this thread's two output columns
    const int64_t c0 = j0 < P.n ? j0 : P.n - 1, c1 = j1 < P.n ? j1 : P.n - 1;  // (past the end: any column that exists)
    const uint32_t* w0 = P.packed + c0 * (P.groups * (GROUP / 8)) + qt * W;
    const uint32_t* w1 = P.packed + c1 * (P.groups * (GROUP / 8)) + qt * W;
    const float *s0 = P.scales + c0 * P.groups, *s1 = P.scales + c1 * P.groups;
    const uint8_t *z0 = P.zeros ? P.zeros + c0 * P.groups : nullptr, *z1 = P.zeros ? P.zeros + c1 * P.groups : nullptr;

    float total[NT][4];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) total[t][i] = 0.0f;

    struct Held {
        Words<GROUP> a, b;
        float sa, sb;
        uint32_t za, zb;
    } held[AHEAD];
    auto fetch = [&](Held& h, int g) {
        if (g >= g_end || idle) return;
        h.a = load_words<GROUP>(w0 + static_cast<int64_t>(g) * (GROUP / 8));
        h.b = load_words<GROUP>(w1 + static_cast<int64_t>(g) * (GROUP / 8));
        h.sa = __ldg(s0 + g);
        h.sb = __ldg(s1 + g);
        h.za = z0 ? __ldg(z0 + g) : 8u;
        h.zb = z1 ? __ldg(z1 + g) : 8u;
    };
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) fetch(held[i], g_begin + i);

    for (int p0 = g_begin; p0 < g_end; p0 += PIECE) {
        const int p1 = p0 + PIECE < g_end ? p0 + PIECE : g_end;
        if (p0 != g_begin) __syncthreads();  // the piece before has been read
        // ---- x's parts: eight k of one row a thread, into the three columns of that row ----
        const int pieces = (p1 - p0) * (GROUP / 8);
        for (int t = tid; t < rows * pieces; t += MM_THREADS) {
            const int r = t / pieces, q = t - r * pieces;
            const int64_t k0 = static_cast<int64_t>(p0) * GROUP + q * 8;
            const float* src = P.x + (row_base + r) * P.ldx + k0;
            float v[8];
            if (P.vec_x && k0 + 8 <= P.k) {
                *reinterpret_cast<float4*>(v) = __ldg(reinterpret_cast<const float4*>(src));
                *reinterpret_cast<float4*>(v + 4) = __ldg(reinterpret_cast<const float4*>(src) + 1);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = k0 + e < P.k ? __ldg(src + e) : 0.0f;
            }
            uint4 out[3];
            uint32_t* o[3] = {&out[0].x, &out[1].x, &out[2].x};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                uint32_t a[3], b[3];
                cut3(v[2 * e], a);
                cut3(v[2 * e + 1], b);
#pragma unroll
                for (int part = 0; part < 3; ++part) o[part][e] = __byte_perm(a[part], b[part], 0x7632);
            }
            const int in = q % (GROUP / 8), at = (q - in) + (in % W) * 4 + in / W;  // piece (thread in / W, word in % W) of its group
#pragma unroll
            for (int part = 0; part < 3; ++part) *reinterpret_cast<uint4*>(smem + (r * 3 + part) * C::PITCH + at * 16) = out[part];
        }
        __syncthreads();
        // ---- the piece's groups ----
        for (int g0 = p0; g0 < p1 && !idle; g0 += AHEAD) {
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                const int g = g0 + i;
                if (g >= p1) break;
                const Held h = held[i];
                fetch(held[i], g + AHEAD);
                const uint32_t za = 0x43004300u | h.za | (h.za << 16), zb = 0x43004300u | h.zb | (h.zb << 16);
                float sum[NT][4];
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e) sum[t][e] = 0.0f;
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    uint32_t a[4], b[4];
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        a[q] = pair_of(h.a.w[w], q, za);
                        b[q] = pair_of(h.b.w[w], q, zb);
                    }
                    const uint8_t* xs = smem + gr * C::PITCH + ((g - p0) * (GROUP / 8) + w * 4 + qt) * 16;
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        const uint4 xv = *reinterpret_cast<const uint4*>(xs + t * 8 * C::PITCH);
                        mma_bf16(sum[t], a[0], b[0], a[1], b[1], xv.x, xv.y);
                        mma_bf16(sum[t], a[2], b[2], a[3], b[3], xv.z, xv.w);
                    }
                }
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    total[t][0] = fmaf(h.sa, sum[t][0], total[t][0]);
                    total[t][1] = fmaf(h.sa, sum[t][1], total[t][1]);
                    total[t][2] = fmaf(h.sb, sum[t][2], total[t][2]);
                    total[t][3] = fmaf(h.sb, sum[t][3], total[t][3]);
                }
            }
        }
    }

    // ---- the sums of the cluster's CTAs and of the three parts ----
    float* const R = reinterpret_cast<float*>(smem);
    __syncthreads();  // x has been read
    if (!idle) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) R[(t * 8 + qt * 2 + (i & 1)) * R_PITCH + warp * 16 + gr + (i >> 1) * 8] = total[t][i];
    }
    if (split > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    else __syncthreads();
    const int outs = rows * MM_COLS;
    for (int t = rank * MM_THREADS + tid; t < outs; t += split * MM_THREADS) {
        const int r = t / MM_COLS, c = t % MM_COLS;
        if (col_base + c >= P.n) continue;
        float v = 0.0f;
        const uint32_t at = static_cast<uint32_t>(__cvta_generic_to_shared(R + r * 3 * R_PITCH + c));
        for (int q = 0; q < split; ++q) {
            float p[3];
#pragma unroll
            for (int part = 0; part < 3; ++part) {
                if (split > 1) {
                    uint32_t from;
                    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(from) : "r"(at + part * R_PITCH * 4), "r"(q));
                    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(p[part]) : "r"(from) : "memory");
                } else {
                    p[part] = R[(r * 3 + part) * R_PITCH + c];
                }
            }
            v += p[0] + (p[1] + p[2]);
        }
        if (P.bias) v += __ldg(P.bias + col_base + c);
        if (P.relu) v = v > 0.0f ? v : 0.0f;
        P.y[(row_base + r) * P.ldy + col_base + c] = v;
    }
    if (split > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");  // the peers have read this CTA's sums
}

template <int GROUP, int NT>
ctk_status launch_matmul(MmArgs P, cudaStream_t st) {
    using C = MmCfg<NT>;
    auto kernel = w4_matmul_kernel<GROUP, NT>;
    static ctk::PerDeviceOnce attr_set;
    if (attr_set.first()) CTK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
    const int64_t blocks = (P.n + MM_COLS - 1) / MM_COLS, row_blocks = (P.m + C::ROWS - 1) / C::ROWS;
    // split k over a cluster while that fills idle SMs and leaves a CTA two groups
    P.split = 1;
    while (P.split < 8 && blocks * row_blocks * P.split * 2 <= 3 * ctk::sm_count() && P.groups >= P.split * 4) P.split *= 2;
    if (blocks * P.split > 0x7FFFFFFF || row_blocks > 65535) return fail(CTK_ERR_LIMIT, "ctk_w4_matmul_f32: too many rows or columns");
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(P.split);
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3(static_cast<unsigned>(blocks * P.split), static_cast<unsigned>(row_blocks));
    cfg.blockDim = dim3(MM_THREADS);
    cfg.dynamicSmemBytes = C::SMEM;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    CTK_CUDA(cudaLaunchKernelEx(&cfg, kernel, P));
    CTK_LAUNCH_CHECK("w4_matmul");
    return CTK_OK;
}
template <int GROUP>
ctk_status matmul_rows(const MmArgs& P, cudaStream_t st) {
    if (P.m <= MmCfg<1>::ROWS) return launch_matmul<GROUP, 1>(P, st);
    if (P.m <= MmCfg<2>::ROWS) return launch_matmul<GROUP, 2>(P, st);
    if (P.m <= MmCfg<3>::ROWS) return launch_matmul<GROUP, 3>(P, st);
    return launch_matmul<GROUP, 6>(P, st);
}

bool group_ok(int group) { return group == 32 || group == 64 || group == 128; }
constexpr int64_t kMaxExtent = int64_t(1) << 30;

}  // namespace

extern "C" {

size_t ctk_w4_packed_bytes(int64_t k, int64_t n, int group) {
    if (k < 0 || n < 0 || !group_ok(group)) return 0;
    return static_cast<size_t>((k + group - 1) / group) * static_cast<size_t>(group / 2) * static_cast<size_t>(n);
}

ctk_status ctk_w4_quantize_f32(const float* w, int64_t ldw, int64_t k, int64_t n, int group, uint32_t* packed, float* scales, uint8_t* zeros, void* stream) {
    CTK_RANGE("ctk_w4_quantize_f32");
    CTK_REQUIRE(k >= 0 && n >= 0, "ctk_w4_quantize_f32: negative size");
    CTK_REQUIRE(group_ok(group), "ctk_w4_quantize_f32: group must be 32, 64 or 128");
    CTK_REQUIRE(ldw >= n, "ctk_w4_quantize_f32: row pitch below n");
    if (k > kMaxExtent || n > kMaxExtent) return fail(CTK_ERR_LIMIT, "ctk_w4_quantize_f32: an extent above 2^30");
    if (k == 0 || n == 0) return CTK_OK;
    CTK_REQUIRE(w && packed && scales, "ctk_w4_quantize_f32: null pointer");
    CTK_REQUIRE((reinterpret_cast<uintptr_t>(packed) & 15u) == 0, "ctk_w4_quantize_f32: packed must be 16-byte aligned");
    CTK_REQUIRE(aligned_to(w, 4) && aligned_to(scales, 4), "ctk_w4_quantize_f32: misaligned pointer");
    const int64_t groups = (k + group - 1) / group, gy = (groups + W4_THREADS / 32 - 1) / (W4_THREADS / 32);
    if (gy > 65535) return fail(CTK_ERR_LIMIT, "ctk_w4_quantize_f32: k too large");
    const dim3 grid(static_cast<unsigned>((n + 31) / 32), static_cast<unsigned>(gy));
    auto go = [&](auto kernel) { kernel<<<grid, W4_THREADS, 0, as_stream(stream)>>>(w, ldw, k, n, groups, packed, scales, zeros); };
    if (zeros) group == 32 ? go(w4_quantize_kernel<32, false>) : group == 64 ? go(w4_quantize_kernel<64, false>) : go(w4_quantize_kernel<128, false>);
    else group == 32 ? go(w4_quantize_kernel<32, true>) : group == 64 ? go(w4_quantize_kernel<64, true>) : go(w4_quantize_kernel<128, true>);
    CTK_LAUNCH_CHECK("w4_quantize");
    return CTK_OK;
}

ctk_status ctk_w4_dequantize_f32(const uint32_t* packed, const float* scales, const uint8_t* zeros, int64_t k, int64_t n, int group, float* w, int64_t ldw,
                                 void* stream) {
    CTK_RANGE("ctk_w4_dequantize_f32");
    CTK_REQUIRE(k >= 0 && n >= 0, "ctk_w4_dequantize_f32: negative size");
    CTK_REQUIRE(group_ok(group), "ctk_w4_dequantize_f32: group must be 32, 64 or 128");
    CTK_REQUIRE(ldw >= n, "ctk_w4_dequantize_f32: row pitch below n");
    if (k > kMaxExtent || n > kMaxExtent) return fail(CTK_ERR_LIMIT, "ctk_w4_dequantize_f32: an extent above 2^30");
    if (k == 0 || n == 0) return CTK_OK;
    CTK_REQUIRE(w && packed && scales, "ctk_w4_dequantize_f32: null pointer");
    CTK_REQUIRE((reinterpret_cast<uintptr_t>(packed) & 15u) == 0, "ctk_w4_dequantize_f32: packed must be 16-byte aligned");
    CTK_REQUIRE(aligned_to(w, 4) && aligned_to(scales, 4), "ctk_w4_dequantize_f32: misaligned pointer");
    const int64_t groups = (k + group - 1) / group, gy = (k + 32 * (W4_THREADS / 32) - 1) / (32 * (W4_THREADS / 32));
    if (gy > 65535) return fail(CTK_ERR_LIMIT, "ctk_w4_dequantize_f32: k too large");
    const dim3 grid(static_cast<unsigned>((n + 31) / 32), static_cast<unsigned>(gy));
    w4_dequantize_kernel<<<grid, W4_THREADS, 0, as_stream(stream)>>>(packed, scales, zeros, k, n, group, groups, w, ldw);
    CTK_LAUNCH_CHECK("w4_dequantize");
    return CTK_OK;
}

ctk_status ctk_w4_matmul_f32(const float* x, int64_t ldx, const uint32_t* packed, const float* scales, const uint8_t* zeros, const float* bias, int relu,
                             float* y, int64_t ldy, int64_t m, int64_t k, int64_t n, int group, void* stream) {
    CTK_RANGE("ctk_w4_matmul_f32");
    CTK_REQUIRE(m >= 0 && k >= 0 && n >= 0, "ctk_w4_matmul_f32: negative size");
    CTK_REQUIRE(group_ok(group), "ctk_w4_matmul_f32: group must be 32, 64 or 128");
    CTK_REQUIRE(ldx >= k && ldy >= n, "ctk_w4_matmul_f32: row pitch below the row's length");
    if (m > kMaxExtent || k > kMaxExtent || n > kMaxExtent) return fail(CTK_ERR_LIMIT, "ctk_w4_matmul_f32: an extent above 2^30");
    if (m == 0 || n == 0) return CTK_OK;
    CTK_REQUIRE(y && (k == 0 || (x && packed && scales)), "ctk_w4_matmul_f32: null pointer");
    CTK_REQUIRE((reinterpret_cast<uintptr_t>(packed) & 15u) == 0, "ctk_w4_matmul_f32: packed must be 16-byte aligned");
    CTK_REQUIRE(aligned_to(x, 4) && aligned_to(scales, 4) && aligned_to(bias, 4) && aligned_to(y, 4), "ctk_w4_matmul_f32: misaligned pointer");
    CTK_REQUIRE(!spans_overlap(x, m, k, ldx, y, m, n, ldy), "ctk_w4_matmul_f32: x and y overlap");
    MmArgs P = {};
    P.x = x;
    P.ldx = ldx;
    P.packed = packed;
    P.scales = scales;
    P.zeros = zeros;
    P.bias = bias;
    P.y = y;
    P.ldy = ldy;
    P.m = m;
    P.k = k;
    P.n = n;
    P.groups = (k + group - 1) / group;
    P.relu = relu;
    P.vec_x = ldx % 4 == 0 && aligned_to(x, 16);
    cudaStream_t st = as_stream(stream);
    return group == 32 ? matmul_rows<32>(P, st) : group == 64 ? matmul_rows<64>(P, st) : matmul_rows<128>(P, st);
}

}  // extern "C"
