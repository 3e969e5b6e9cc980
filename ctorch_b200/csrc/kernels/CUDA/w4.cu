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
// The plain form: a warp per output column and block of ROWS rows; lanes stride over the column's words.
constexpr int MV_ROWS = 4;
__global__ void __launch_bounds__(W4_THREADS) w4_matmul_simple_kernel(const float* __restrict__ x, int64_t ldx, const uint32_t* __restrict__ packed,
                                                                      const float* __restrict__ scales, const uint8_t* __restrict__ zeros,
                                                                      const float* __restrict__ bias, int relu, float* __restrict__ y, int64_t ldy,
                                                                      int64_t m, int64_t k, int64_t n, int group, int64_t groups) {
    const int lane = threadIdx.x & 31;
    const int64_t j = static_cast<int64_t>(blockIdx.x) * (W4_THREADS / 32) + (threadIdx.x >> 5);
    const int64_t r0 = static_cast<int64_t>(blockIdx.y) * MV_ROWS;
    if (j >= n) return;
    const int64_t kw = groups * (group / 8);
    float acc[MV_ROWS] = {};
    for (int64_t wd = lane; wd < kw; wd += 32) {
        const int64_t k0 = wd * 8, grp = k0 / group;
        if (k0 >= k) break;
        const uint32_t c = packed[j * kw + wd];
        const float s = scales[j * groups + grp], zero = zeros ? static_cast<float>(zeros[j * groups + grp]) : 8.0f;
        float part[MV_ROWS] = {};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (k0 + i >= k) break;
            const float q = static_cast<float>((c >> nibble_shift(i)) & 15u) - zero;
#pragma unroll
            for (int r = 0; r < MV_ROWS; ++r)
                if (r0 + r < m) part[r] = fmaf(x[(r0 + r) * ldx + k0 + i], q, part[r]);
        }
#pragma unroll
        for (int r = 0; r < MV_ROWS; ++r) acc[r] = fmaf(part[r], s, acc[r]);
    }
#pragma unroll
    for (int r = 0; r < MV_ROWS; ++r) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) acc[r] += __shfl_xor_sync(0xffffffffu, acc[r], o);
        if (lane == 0 && r0 + r < m) {
            float v = acc[r] + (bias ? bias[j] : 0.0f);
            if (relu) v = v > 0.0f ? v : 0.0f;
            y[(r0 + r) * ldy + j] = v;
        }
    }
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
    const int64_t groups = (k + group - 1) / group, gy = (m + MV_ROWS - 1) / MV_ROWS;
    if (gy > 65535) return fail(CTK_ERR_LIMIT, "ctk_w4_matmul_f32: too many rows");
    const dim3 grid(static_cast<unsigned>((n + W4_THREADS / 32 - 1) / (W4_THREADS / 32)), static_cast<unsigned>(gy));
    w4_matmul_simple_kernel<<<grid, W4_THREADS, 0, as_stream(stream)>>>(x, ldx, packed, scales, zeros, bias, relu, y, ldy, m, k, n, group, groups);
    CTK_LAUNCH_CHECK("w4_matmul");
    return CTK_OK;
}

}  // extern "C"
