// 4-bit weights with group scales: quantising, the values they stand for, and y = [relu](x W + bias).
// The layout is described in ctorch_b200.h.
#include <algorithm>

#include "tcgen05.cuh"

namespace {
using namespace ctk;

constexpr int W4_THREADS = 128;  // neighbouring columns: 512 contiguous bytes of a row of w per access (with 32 columns to a CTA quantising
                                 // 4096 x 4096 took 59 us)

// Bit position of code i of a word: the pairs (2p, 2p+1) sit 16 bits apart, so one mask takes both as the
// two halves of a register.
__host__ __device__ constexpr int nibble_shift(int i) { return 4 * (i >> 1) + 16 * (i & 1); }

// the larger one, a NaN if either is one
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// ---- quantise ------------------------------------------------------------------------------------------
// A thread owns 32 or 64 k of one column: lanes are neighbouring columns (coalesced rows of w), the values stay in registers
// between the maximum and the rounding, so w is read once with that many loads in flight; the two halves of a group of 128
// exchange their extremes through shared memory.  Bound by instruction issue until the rounding became what it is:
//
// round(w / s) exactly, ties to even: t = fma(w, 1/s, 1.5 * 2^23 + zero) has the code in its low bits and is at most one step
// off; the remainder d = w - q s is exact in one fma (|d| <= s (1/2 + tiny), a multiple of the smaller of both ulps), so only
// where |d| >= s / 2 is there anything to decide, which the word's eight codes ask about together.
// (With a rounding, a conversion to int and three comparisons per value: 36 instructions and 50 us at 4096 x 4096,
// this way 20 us.  The codes are added up shifted, with the bits above them, and those taken off once a word: 256 against 234 us
// for 16384 x 16384 g128.)
__device__ __forceinline__ uint32_t exact_code(float w, float s, float t, float q) {
    const float d = fmaf(-q, s, w), e = 2.0f * fabsf(d);
    if (e > s || (e == s && ((__float_as_uint(q + 12582912.0f)) & 1u))) t += d > 0.0f ? 1.0f : -1.0f;
    return __float_as_uint(fminf(fmaxf(t, 12582912.0f), 12582927.0f)) & 15u;
}

// Threads that share a column of a CTA: 4 groups of 32, one of 64 (two of them: 262 us for 16384 x 16384 with zero points, 232
// alone), or the halves of one of 128.
__host__ __device__ constexpr int quantize_parts(int group) { return group == 32 ? 4 : group == 64 ? 1 : 2; }
template <int GROUP, bool SYM>
__global__ void __launch_bounds__(W4_THREADS * quantize_parts(GROUP)) w4_quantize_kernel(const float* __restrict__ w, int64_t ldw, int64_t k, int64_t n, int64_t groups,
                                                                                           uint32_t* __restrict__ packed, float* __restrict__ scales,
                                                                                           uint8_t* __restrict__ zeros, bool wide) {
    constexpr int LEN = GROUP == 128 ? 64 : GROUP, PARTS = quantize_parts(GROUP), GROUPS = PARTS * LEN / GROUP;  // k of a thread; threads and groups of a column
    const uint32_t col_blocks = static_cast<uint32_t>((n + W4_THREADS - 1) / W4_THREADS);
    const int lane_col = threadIdx.x % W4_THREADS, part = threadIdx.x / W4_THREADS;
    const int64_t j = static_cast<int64_t>(blockIdx.x % col_blocks) * W4_THREADS + lane_col, first = blockIdx.x / col_blocks * GROUPS;
    const int64_t k0 = first * GROUP + part * LEN;
    const bool there = j < n && k0 < groups * GROUP;
    const int len = !there || k0 >= k ? 0 : static_cast<int>(k - k0 < LEN ? k - k0 : LEN);
    const float* src = w + k0 * ldw + j;
    float v[LEN];
    if (len == LEN) {
#pragma unroll
        for (int i = 0; i < LEN; ++i) v[i] = __ldcs(src + i * ldw);
    } else {
#pragma unroll
        for (int i = 0; i < LEN; ++i) v[i] = i < len ? __ldcs(src + i * ldw) : 0.0f;
    }
    float top = 0.0f, bottom = 0.0f;  // (a NaN stays in top, an infinity in either)
#pragma unroll
    for (int i = 0; i < LEN; ++i) {
        top = max_nan(top, SYM ? fabsf(v[i]) : v[i]);
        if (!SYM) bottom = fminf(bottom, v[i]);
    }
    if constexpr (GROUP == 128) {
        __shared__ float ends[2][2][W4_THREADS];
        ends[0][part][lane_col] = top;
        ends[1][part][lane_col] = bottom;
        __syncthreads();
        top = max_nan(ends[0][0][lane_col], ends[0][1][lane_col]);
        bottom = fminf(ends[1][0][lane_col], ends[1][1][lane_col]);
    }
    // the one division of the group, in 64 bits so that the scale is the nearest fp32 number
    const bool finite = top < __int_as_float(0x7f800000) && bottom > __int_as_float(0xff800000);
    const float s = finite ? static_cast<float>(SYM ? static_cast<double>(top) / 7.0 : (static_cast<double>(top) - static_cast<double>(bottom)) / 15.0)
                           : __int_as_float(0x7fc00000);
    const bool live = s > 0.0f;  // false for a group of zeros and for NaN
    float zero = 8.0f;
    if (!SYM) zero = live ? static_cast<float>(rint(-static_cast<double>(bottom) / static_cast<double>(s))) : 0.0f;
    if (!SYM && zero > 15.0f) zero = 15.0f;  // (subnormal scales only: the range is no longer 15 steps wide)
    const float inv = live ? 1.0f / s : 0.0f;
    uint32_t* dst = packed + j * (groups * (GROUP / 8)) + k0 / 8;
    if (!there) {
    } else if (!(inv <= 3.0e38f)) {  // a subnormal scale, 1/s overflows: divide in 64 bits, one by one (rare: no code of it in the loop below)
#pragma unroll 1
        for (int wd = 0; wd < LEN / 8; ++wd) {
            uint32_t word = 0;
#pragma unroll 1
            for (int i = 0; i < 8; ++i) {
                const float x = wd * 8 + i < len ? __ldg(src + (wd * 8 + i) * ldw) : 0.0f;
                const float c = fminf(fmaxf(zero + static_cast<float>(rint(static_cast<double>(x) / static_cast<double>(s))), SYM ? 1.0f : 0.0f), 15.0f);
                word |= static_cast<uint32_t>(c) << nibble_shift(i);
            }
            dst[wd] = word;
        }
    } else if (!live) {  // zeros, or a value that is not finite: every code the zero point
#pragma unroll
        for (int wd = 0; wd < LEN / 8; ++wd) dst[wd] = SYM ? 0x88888888u : 0u;
    } else {
        const float base = 12582912.0f + zero, half = 0.5f * s;
#pragma unroll
        for (int q4 = 0; q4 < LEN / 32; ++q4) {
            uint32_t out[4];
#pragma unroll
            for (int wd = 0; wd < 4; ++wd) {
                uint32_t word = 0;  // t's bits are 0x4B400000 + code: added up shifted, the constants taken off once
                bool close = false;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float x = v[q4 * 32 + wd * 8 + i];
                    float t = fmaf(x, inv, base);
                    close |= fabsf(fmaf(base - t, s, x)) >= half;
                    if (!SYM) t = fminf(t, 12582927.0f);  // (symmetric: 1 .. 15 by construction; the lower end as well)
                    word += __float_as_uint(t) << nibble_shift(i);
                }
                word -= 0x4B400000u * 0x11111111u;
                if (close) {
                    word = 0;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float x = v[q4 * 32 + wd * 8 + i], t = fmaf(x, inv, base);
                        word |= exact_code(x, s, t, t - base) << nibble_shift(i);
                    }
                }
                out[wd] = word;
            }
            *reinterpret_cast<uint4*>(dst + q4 * 4) = make_uint4(out[0], out[1], out[2], out[3]);
        }
    }
    if constexpr (GROUPS == 1) {
        if (part == 0 && there) {
            scales[j * groups + first] = s;
            if (!SYM) zeros[j * groups + first] = static_cast<uint8_t>(zero);
        }
    } else {  // a column's four groups together: one by one, each store is a sector of its own (16384 x 16384 308 us, this way 263)
        __shared__ float group_scales[GROUPS][W4_THREADS];
        __shared__ uint8_t group_zeros[GROUPS][W4_THREADS];
        group_scales[part][lane_col] = s;
        group_zeros[part][lane_col] = static_cast<uint8_t>(zero);
        __syncthreads();
        if (part != 0 || j >= n) return;
        const int64_t at = j * groups + first;
        if (wide && groups % 4 == 0) {
            *reinterpret_cast<float4*>(scales + at) = make_float4(group_scales[0][lane_col], group_scales[1][lane_col], group_scales[2][lane_col], group_scales[3][lane_col]);
            if (!SYM)
                *reinterpret_cast<uchar4*>(zeros + at) = make_uchar4(group_zeros[0][lane_col], group_zeros[1][lane_col], group_zeros[2][lane_col], group_zeros[3][lane_col]);
            return;
        }
        for (int g = 0; g < GROUPS && first + g < groups; ++g) {
            scales[at + g] = group_scales[g][lane_col];
            if (!SYM) zeros[at + g] = group_zeros[g][lane_col];
        }
    }
}

// ---- dequantise ----------------------------------------------------------------------------------------
// A thread takes 32 k of one column: one 16-byte load of codes, 32 coalesced stores (lanes are columns).  16384 x 16384 g64 206 us,
// 5.6 TB/s (with a shift and a conversion to float per value 233).
__global__ void __launch_bounds__(W4_THREADS) w4_dequantize_kernel(const uint32_t* __restrict__ packed, const float* __restrict__ scales,
                                                                   const uint8_t* __restrict__ zeros, int64_t k, int64_t n, int group, int64_t groups,
                                                                   float* __restrict__ w, int64_t ldw) {
    const uint32_t col_blocks = static_cast<uint32_t>((n + W4_THREADS - 1) / W4_THREADS);
    const int64_t j = static_cast<int64_t>(blockIdx.x % col_blocks) * W4_THREADS + threadIdx.x, k0 = static_cast<int64_t>(blockIdx.x / col_blocks) * 32;
    if (j >= n) return;
    const int64_t grp = k0 / group;
    const uint4 c = __ldg(reinterpret_cast<const uint4*>(packed + j * (groups * (group / 8)) + k0 / 8));
    const float s = scales[j * groups + grp];
    const float zero = zeros ? static_cast<float>(zeros[j * groups + grp]) : 8.0f;
    const uint32_t word[4] = {c.x, c.y, c.z, c.w};
    float* dst = w + k0 * ldw + j;
    // the nibble at bit 4p under an exponent of 23 - 4p is the number 2^(23 - 4p) + code: no conversion, no shift
    float base[4];
#pragma unroll
    for (int p = 0; p < 4; ++p) base[p] = static_cast<float>(1 << (23 - 4 * p)) + zero;
    auto value = [&](int i) {
        const int p = (i & 7) >> 1;
        const uint32_t half = i & 1 ? word[i >> 3] >> 16 : word[i >> 3];
        return (__uint_as_float((half & (15u << (4 * p))) | (static_cast<uint32_t>(150 - 4 * p) << 23)) - base[p]) * s;
    };
    if (k - k0 >= 32) {
#pragma unroll
        for (int i = 0; i < 32; ++i) __stcs(dst + i * ldw, value(i));
    } else {
        const int len = static_cast<int>(k - k0);
#pragma unroll
        for (int i = 0; i < 32; ++i)
            if (i < len) __stcs(dst + i * ldw, value(i));
    }
}

// ---- y = [relu](x W + bias) ------------------------------------------------------------------------------
// tcgen05 on whole numbers.  A code of 0..15 in a byte IS an e4m3 number: 0..7 are its subnormals, 8..15 its first
// normals, and both count in steps of 2^-9, so the weight's operand is made by two masks and a shift per eight codes.  x is
// taken in fixed point: 38 bits below the largest |x| of its row's 128 neighbours, as eight signed digits base 32, and
// a digit of -16..16, doubled, in sign and magnitude is an e4m3 number of four significant bits.  So each (row, digit) is a column of the
// instruction's B, every product and every sum of a group is a whole number below 2^24 times 2^-17 -- exact in the fp32
// accumulator whatever it does -- and so is the zero point's share, zero * (sum of the digits).  What rounds: x to its 38 bits,
// eight digits joined in fp32, one fma per group with the scale.
//
// A first, small kernel writes x's digits (w4_digits_kernel: a warp per row and 128 k) piece by piece as the main kernel's
// shared memory wants them; where x is small, every CTA makes its own.  A CTA of the main kernel takes 128 columns of W and, in
// blocks of 256 k, its share of k (a cluster of `split` CTAs shares the whole):
//   2 warps     loads: the block's codes (one TMA copy, 128 columns x 128 bytes, RAW blocks in flight, the first of them before
//               x's digits are there) and x's digits, their sums and x's steps (one bulk copy);
//   4 warps     a thread per column: its 128 bytes of codes, masked, into the operand's place in tensor memory;
//   1 warp      the products: one instruction per 32 k, an accumulator [128 columns][(row, digit)] per group, BATCH groups to a
//               hand-over;
//   4 or 8      a thread per column: digits joined, zero point, scale, added to the column's results.
// A hand-over between warps (an mbarrier's arrival and wait) takes some 200 clocks, the bytes of 128 columns x 128 k take 180 at
// HBM's rate: hence the large blocks.  Before this: mma.sync with x cut into three bf16 parts (about 32 clocks an instruction on
// this machine) 95 us for 4 x 16384 x 16384 and 46 us for 64 x 4096 x 4096; the operand in shared memory, its codes through
// registers, 96 and 35 us (the load and store unit was the bound); blocks of 128 k, 69 and 37 us; this one 54 and 22 us.  (fp16 in place of e4m3
// with x in three digits base 2048 reads back three columns per row instead of eight, but a piece of the operand in tensor
// memory then holds half as many k, and the hand-overs cost more than that gains: 64 and 36 us.)
constexpr int MM_COLS = 128, MM_PIECE = 128, MM_BLOCK = 256;  // columns of a CTA; k of one piece of x and of a block
constexpr int MM_RAW_BYTES = MM_COLS * MM_BLOCK / 2;          // codes of a block
constexpr int MM_A_COLS = MM_BLOCK / 4;                       // tensor memory columns of a block's operand
constexpr int R_PITCH = 132;

template <int GROUP, int ROWS>
struct MmCfg {
    static constexpr int N = 8 * ROWS;               // columns of one accumulator
    static constexpr int GPP = MM_PIECE / GROUP, GPB = MM_BLOCK / GROUP;  // groups of a piece, of a block
    static constexpr int STAGES = 2;                 // blocks of operands in tensor memory
    static constexpr int BATCH = N >= 64 ? 1 : 64 / N < GPB ? 64 / N : GPB;  // groups whose accumulators are handed over together
    static constexpr int USED_COLS = 2 * BATCH * N + STAGES * MM_A_COLS;     // two such batches in turn
    static constexpr int TMEM_COLS = USED_COLS <= 256 ? 256 : 512;
    static constexpr int PER_SM = 512 / TMEM_COLS;
    static constexpr int RAW = ROWS == 8 ? 3 : 4, XS = ROWS <= 4 ? 4 : 3;    // blocks of codes and of x in flight or in use
    static constexpr int B_BYTES = N * MM_PIECE;
    static constexpr int T_BYTES = (GPP * ROWS * 4 + ROWS) * 4;              // joined sums of digits per (group, row), x's step per row
    static constexpr int X_BYTES = (B_BYTES + T_BYTES + 1023) / 1024 * 1024; // a piece of x as the first kernel leaves it
    static constexpr int RING = RAW * MM_RAW_BYTES + XS * 2 * X_BYTES, R_BYTES = ROWS * R_PITCH * 4;
    static constexpr int SMEM = (RING > R_BYTES ? RING : R_BYTES) + 1024;
    static constexpr int DRAIN = ROWS <= 8 ? 4 : 8;  // warps that take the accumulators: 4, or 8 with half of the rows each
    static constexpr int MINE = ROWS * 4 / DRAIN;    // rows of such a warp
    static constexpr int RC = ROWS <= 8 ? 2 : 4;     // rows joined at a time
    static constexpr int U = GPB < 4 ? GPB : 4;      // groups whose scales are read together
    static constexpr int THREADS = (DRAIN + 4 + 3) * 32;
    static constexpr int QUAD = GPP >= 4 ? 1 : 4 / GPP;  // pieces of four groups
    static __host__ __device__ int64_t share_begin(int64_t pieces, int rank, int split) { return rank == split ? pieces : pieces * rank / split / QUAD * QUAD; }
    static_assert(USED_COLS <= 512 && SMEM * PER_SM <= 225 * 1024 && MINE % 2 == 0 && GPB % BATCH == 0 && BATCH <= 4, "");
};

__device__ int g_w4_status = 0;  // first bounded wait that ran out, else 0

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
    int quads;             // scales and zero points can be read four at a time
    const uint8_t* image;  // x's digits, [row block][piece][X_BYTES]; nullptr: each CTA makes its own
};

// x's digits.  A warp takes one row's 128 k of a piece, lane l the k 4l .. 4l+3 (load_x; rows past m give zeros), and writes
// row r of the piece at `out` (global memory, or a stage of the main kernel).
__device__ __forceinline__ float4 load_x(const float* __restrict__ x, int64_t ldx, int64_t m, int64_t k, int64_t row, int64_t k0) {
    const float* p = x + row * ldx + k0;
    const bool here = row < m;
    return make_float4(here && k0 < k ? __ldg(p) : 0.0f, here && k0 + 1 < k ? __ldg(p + 1) : 0.0f, here && k0 + 2 < k ? __ldg(p + 2) : 0.0f,
                       here && k0 + 3 < k ? __ldg(p + 3) : 0.0f);
}
template <int GROUP, int ROWS>
__device__ __forceinline__ void write_digits(float4 x, int r, int lane, uint8_t* out) {
    using C = MmCfg<GROUP, ROWS>;
    float* const sums = reinterpret_cast<float*>(out + C::B_BYTES);
    const float v[4] = {x.x, x.y, x.z, x.w};
    // the largest exponent (as bits, so that an infinity or a NaN wins)
    uint32_t top = max(max(__float_as_uint(v[0]) & 0x7FFFFFFFu, __float_as_uint(v[1]) & 0x7FFFFFFFu), max(__float_as_uint(v[2]) & 0x7FFFFFFFu, __float_as_uint(v[3]) & 0x7FFFFFFFu));
    top = __reduce_max_sync(0xffffffffu, top);
    int ex = static_cast<int>(top >> 23);  // |v| < 2^(ex - 126)
    const bool bad = ex == 255;
    // |v| 2^(164 - ex) < 2^38.  The smallest unit is 2^-149, of which every fp32 number is a multiple.
    ex = max(ex, 15);
    const int up = 127 + 164 - ex, up0 = min(up, 254);  // in two exact factors: one would overflow for the smallest x
    const float up_by = __uint_as_float(static_cast<uint32_t>(up0) << 23), up_rest = __uint_as_float(static_cast<uint32_t>(127 + up - up0) << 23);
    uint32_t digits[2][4];                 // four digits of five bits each, 16 too large: the lower ones, the upper ones
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float t = bad ? 0.0f : v[e] * up_by * up_rest, upper = rintf(t * (1.0f / 1048576.0f));
        const uint32_t low = static_cast<uint32_t>(__float2int_rn(fmaf(upper, -1048576.0f, t)) + 0x84210);  // 16 in each of four digits
        digits[0][e] = low;
        digits[1][e] = static_cast<uint32_t>(static_cast<int>(upper) + 0x84210) + (low >> 20);  // (the rest may be too large for its digits by one)
    }
    // four bytes of digit d: sign and twice the magnitude; this lane's four k are codes 0..3 (even lanes) or 4..7 of a word
    int pair = 0;  // sums over the group of digit 2p and 32 times digit 2p + 1
#pragma unroll
    for (int d = 0; d < 8; ++d) {
        uint32_t four = 0;
        int sum = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int g = static_cast<int>((digits[d / 4][e] >> (5 * (d % 4))) & 31u) - 16;
            sum += g;
            const int mag = abs(g);
            four |= static_cast<uint32_t>((mag + min(mag, 8)) | ((g >> 24) & 0x80)) << (8 * e);  // (2 mag: up to 16 as it stands, then in steps of 2)
        }
        const uint32_t other = __shfl_xor_sync(0xffffffffu, four, 1);
        const uint32_t first = lane & 1 ? other : four, second = lane & 1 ? four : other;
        const uint32_t bytes = lane & 1 ? __byte_perm(first, second, 0x7362) : __byte_perm(first, second, 0x5140);
        const int col = r * 8 + d;
        *reinterpret_cast<uint32_t*>(out + col * 128 + (((lane >> 2) ^ (col & 7)) << 4) + (lane & 3) * 4) = bytes;
#pragma unroll
        for (int s = 1; s < GROUP / 4; s <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);  // of the group's lanes
        pair = d & 1 ? pair + 32 * sum : sum;
        if ((d & 1) && lane % (GROUP / 4) == 0) sums[((lane / (GROUP / 4)) * ROWS + r) * 4 + d / 2] = static_cast<float>(pair) * (1.0f / 131072.0f);
    }
    // x's step: what a unit of the joined digits stands for, 2^(ex - 164) of digit 0 by 2^17 (the accumulator's units) and 2^20 (those
    // of the upper digits): 2^(ex - 127), no more than the largest |v| and more than half of it
    if (lane == 0) sums[C::GPP * ROWS * 4 + r] = __uint_as_float(bad ? 0x7FC00000u : static_cast<uint32_t>(ex) << 23);
}
template <int GROUP, int ROWS>
__global__ void __launch_bounds__(128) w4_digits_kernel(const float* __restrict__ x, int64_t ldx, int64_t m, int64_t k, int64_t pieces, uint8_t* __restrict__ image) {
    const int lane = threadIdx.x & 31;
    const int64_t piece = static_cast<int64_t>(blockIdx.y) * 4 + (threadIdx.x >> 5);
    const int64_t row = blockIdx.x, row_block = row / ROWS;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // (the main kernel starts with what does not depend on this one)
    if (piece >= pieces) return;
    write_digits<GROUP, ROWS>(load_x(x, ldx, m, k, row, piece * MM_PIECE + lane * 4), static_cast<int>(row - row_block * ROWS), lane,
                              image + (row_block * pieces + piece) * MmCfg<GROUP, ROWS>::X_BYTES);
}

template <int GROUP, int ROWS>
__global__ void __launch_bounds__((MmCfg<GROUP, ROWS>::THREADS), (MmCfg<GROUP, ROWS>::PER_SM))
w4_matmul_kernel(const __grid_constant__ CUtensorMap codes, const MmArgs P) {
    using namespace t5;
    using C = MmCfg<GROUP, ROWS>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t bars[2 * C::RAW + 2 * C::XS + 2 * C::STAGES + 4];
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int abort_flag;
    uint8_t* const smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);  // [blocks of x][blocks of codes]
    const uint32_t bar0 = smem_u32(bars), base = smem_u32(smem);
    auto raw_full = [&](int i) { return bar0 + 8u * i; };
    auto raw_empty = [&](int i) { return bar0 + 8u * (C::RAW + i); };
    auto x_full = [&](int i) { return bar0 + 8u * (2 * C::RAW + i); };
    auto x_empty = [&](int i) { return bar0 + 8u * (2 * C::RAW + C::XS + i); };
    auto op_full = [&](int s) { return bar0 + 8u * (2 * C::RAW + 2 * C::XS + s); };
    auto op_empty = [&](int s) { return bar0 + 8u * (2 * C::RAW + 2 * C::XS + C::STAGES + s); };
    auto acc_full = [&](int a) { return bar0 + 8u * (2 * C::RAW + 2 * C::XS + 2 * C::STAGES + a); };
    auto acc_empty = [&](int a) { return bar0 + 8u * (2 * C::RAW + 2 * C::XS + 2 * C::STAGES + 2 + a); };
    constexpr uint32_t RAW_AT = C::XS * 2 * C::X_BYTES;
    constexpr int W_OP = C::DRAIN, W_MMA = W_OP + 4, W_CODES = W_MMA + 1, W_X = W_CODES + 1;  // warps by role (W_OP a multiple of 4)
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int split = P.split, rank = blockIdx.x % split;
    const int64_t col_base = static_cast<int64_t>(blockIdx.x / split) * MM_COLS, row_base = static_cast<int64_t>(blockIdx.y) * ROWS;
    const int rows = static_cast<int>(P.m - row_base < ROWS ? P.m - row_base : ROWS);
    // this CTA's share: pieces of 128 k, groups, blocks
    // (a share starts at a multiple of four groups, so that their scales can be read together)
    const int64_t all_pieces = (P.groups + C::GPP - 1) / C::GPP, p_begin = C::share_begin(all_pieces, rank, split), p_end = C::share_begin(all_pieces, rank + 1, split);
    const int pieces = static_cast<int>(p_end - p_begin), blocks = (pieces + 1) / 2;
    const int groups = static_cast<int>((p_end * C::GPP < P.groups ? p_end * C::GPP : P.groups) - p_begin * C::GPP);

    if (tid == 0) {
        abort_flag = 0;
        for (int i = 0; i < C::RAW; ++i) { mbar_init(raw_full(i), 1); mbar_init(raw_empty(i), 4); }
        for (int i = 0; i < C::XS; ++i) { mbar_init(x_full(i), 1); mbar_init(x_empty(i), 1 + C::DRAIN); }
        for (int s = 0; s < C::STAGES; ++s) { mbar_init(op_full(s), 4); mbar_init(op_empty(s), 1); }
        for (int a = 0; a < 2; ++a) { mbar_init(acc_full(a), 1); mbar_init(acc_empty(a), C::DRAIN); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        if (!P.image) {  // the first codes set off before x's digits are made
            for (int b = 0; b < blocks && b < C::RAW; ++b) {
                mbar_expect_tx(raw_full(b), MM_RAW_BYTES);
                tma_load_2d(base + RAW_AT + b * MM_RAW_BYTES, &codes, raw_full(b), static_cast<int>(p_begin * (MM_PIECE / 8)) + b * (MM_BLOCK / 8), static_cast<int>(col_base));
            }
        }
    }
    if (!P.image) {  // all of this CTA's x fits its ring: every warp makes a share of the digits, here and once
        for (int t = warp; t < pieces * ROWS; t += C::THREADS / 32) {
            const int p = t / ROWS, r = t - p * ROWS;
            write_digits<GROUP, ROWS>(load_x(P.x, P.ldx, P.m, P.k, row_base + r, (p_begin + p) * MM_PIECE + lane * 4), r, lane, smem + p * C::X_BYTES);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == W_MMA) tmem_alloc<1>(smem_u32(&tmem_slot), C::TMEM_COLS);
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = tmem_slot, op_tmem = tmem + 2 * C::BATCH * C::N;
    if (!P.image && tid == 0)
        for (int b = 0; b < blocks; ++b) mbar_arrive(x_full(b));

    float result[C::MINE];
#pragma unroll
    for (int r = 0; r < C::MINE; ++r) result[r] = 0.0f;

    if (warp == W_CODES) {
        // ------------------------------ codes: global -> shared ------------------------------
        if (lane == 0) {
            for (int b = P.image ? 0 : C::RAW; b < blocks; ++b) {
                const int i = b % C::RAW;
                if (!mbar_wait(raw_empty(i), ((b / C::RAW) & 1) ^ 1u, &abort_flag, &g_w4_status, 0x100 | i)) break;
                mbar_expect_tx(raw_full(i), MM_RAW_BYTES);
                tma_load_2d(base + RAW_AT + i * MM_RAW_BYTES, &codes, raw_full(i), static_cast<int>(p_begin * (MM_PIECE / 8)) + b * (MM_BLOCK / 8), static_cast<int>(col_base));
            }
        }
    } else if (warp == W_X) {
        // ------------------------------ x: global -> shared ------------------------------
        if (lane == 0 && P.image) {
            asm volatile("griddepcontrol.wait;" ::: "memory");  // x's digits are there
            const uint8_t* from = P.image + (blockIdx.y * all_pieces + p_begin) * C::X_BYTES;
            for (int b = 0; b < blocks; ++b) {
                const int i = b % C::XS;
                const uint32_t bytes = (2 * b + 1 < pieces ? 2 : 1) * C::X_BYTES;
                if (!mbar_wait(x_empty(i), ((b / C::XS) & 1) ^ 1u, &abort_flag, &g_w4_status, 0x180 | i)) break;
                mbar_expect_tx(x_full(i), bytes);
                bulk_load(base + i * 2 * C::X_BYTES, from + static_cast<int64_t>(b) * 2 * C::X_BYTES, bytes, x_full(i));
            }
        }
    } else if (warp >= W_OP && warp < W_MMA) {
        // ------------------------------ codes: shared -> operand ------------------------------
        const int row = (warp & 3) * 32 + lane;  // this thread's column of W
        for (int b = 0; b < blocks; ++b) {
            const int i = b % C::RAW, st = b % C::STAGES;
            if (!mbar_wait(raw_full(i), (b / C::RAW) & 1, &abort_flag, &g_w4_status, 0x400 | i)) break;
            const uint8_t* raw = smem + RAW_AT + i * MM_RAW_BYTES + row * 128;
            uint4 w[8];
#pragma unroll
            for (int c = 0; c < 8; ++c) w[c] = *reinterpret_cast<const uint4*>(raw + ((c ^ (row & 7)) << 4));  // (the copy's 128-byte swizzle)
            if (!mbar_wait(op_empty(st), ((b / C::STAGES) & 1) ^ 1u, &abort_flag, &g_w4_status, 0x410 | st)) break;
            fence_after();
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t o[32];
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const uint4 v = w[h * 4 + c];
                    constexpr uint32_t M = 0x0F0F0F0Fu;
                    o[c * 8] = v.x & M; o[c * 8 + 1] = (v.x >> 4) & M;
                    o[c * 8 + 2] = v.y & M; o[c * 8 + 3] = (v.y >> 4) & M;
                    o[c * 8 + 4] = v.z & M; o[c * 8 + 5] = (v.z >> 4) & M;
                    o[c * 8 + 6] = v.w & M; o[c * 8 + 7] = (v.w >> 4) & M;
                }
                tmem_st32(op_tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16) + st * MM_A_COLS + h * 32, o);
            }
            tmem_st_wait();
            fence_before();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(op_full(st));
                mbar_arrive(raw_empty(i));
            }
        }
    } else if (warp == W_MMA) {
        // ------------------------------ products ------------------------------
        constexpr uint32_t idesc = make_idesc(MM_COLS, C::N, false, false);
        int acc = 0;
        uint32_t acc_phase = 0;
        bool ok = true;
        for (int b = 0; b < blocks && ok; ++b) {
            const int st = b % C::STAGES, xi = b % C::XS;
            const int here = groups - b * C::GPB < C::GPB ? groups - b * C::GPB : C::GPB;
            if (!mbar_wait(x_full(xi), (b / C::XS) & 1, &abort_flag, &g_w4_status, 0x200 | xi)) break;
            if (!mbar_wait(op_full(st), (b / C::STAGES) & 1, &abort_flag, &g_w4_status, 0x208 | st)) break;
            const uint64_t x = make_desc(base + xi * 2 * C::X_BYTES, 0);
#pragma unroll
            for (int g0 = 0; g0 < C::GPB; g0 += C::BATCH) {
                if (g0 >= here) break;
                if (!mbar_wait(acc_empty(acc), acc_phase ^ 1u, &abort_flag, &g_w4_status, 0x210 | acc)) { ok = false; break; }
                fence_after();
                __syncwarp();
                if (elect_one()) {
#pragma unroll
                    for (int i = 0; i < C::BATCH; ++i) {
                        const int g = g0 + i;
                        if (g >= here) break;
#pragma unroll
                        for (int ks = 0; ks < GROUP / 32; ++ks) {
                            const int k32 = g * (GROUP / 32) + ks;  // of the block; four of them are a piece of x
                            mma_f8_ts(tmem + (acc * C::BATCH + i) * C::N, op_tmem + st * MM_A_COLS + k32 * 8, x + (k32 / 4) * (C::X_BYTES / 16) + (k32 % 4) * 2, idesc, ks > 0);
                        }
                    }
                    commit<1>(acc_full(acc));
                    if (g0 + C::BATCH >= here) {
                        commit<1>(op_empty(st));
                        commit<1>(x_empty(xi));
                    }
                }
                acc ^= 1;
                acc_phase ^= static_cast<uint32_t>(acc == 0);
            }
        }
    } else {
        // ------------------------------ results ------------------------------
        const int quarter = warp & 3, r_first = (warp >> 2) * C::MINE;  // columns of the tile, rows of x
        const int64_t col = col_base + quarter * 32 + lane, at = (col < P.n ? col : P.n - 1) * P.groups + p_begin * C::GPP;
        const uint32_t t_row = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + r_first * 8;
        // Scales and zero points, each lane its own row of them: U groups at a time, two such units ahead (a load's latency is
        // several groups long).  Read together where rows of them are aligned for it: one by one, each brings its sector of
        // 32 bytes from L2 again.
        constexpr int U = C::U;
        float scale[U], scale1[U], scale2[U];
        uint32_t zero = 0, zero1 = 0, zero2 = 0;
        auto fetch = [&](float (&s)[U], uint32_t& z, int g) {
            z = 0x08080808u;
            if (g >= groups) return;
            const float* ps = P.scales + at + g;
            const uint8_t* pz = P.zeros + at + g;
            if (P.quads) {
                if constexpr (U == 4) {
                    *reinterpret_cast<float4*>(s) = __ldg(reinterpret_cast<const float4*>(ps));
                    if (P.zeros) z = __ldg(reinterpret_cast<const uint32_t*>(pz));
                } else {
                    *reinterpret_cast<float2*>(s) = __ldg(reinterpret_cast<const float2*>(ps));
                    if (P.zeros) z = __ldg(reinterpret_cast<const uint16_t*>(pz));
                }
                return;
            }
            uint32_t w = 0;
#pragma unroll
            for (int e = 0; e < U; ++e) {
                s[e] = g + e < groups ? __ldg(ps + e) : 0.0f;
                if (P.zeros && g + e < groups) w |= static_cast<uint32_t>(__ldg(pz + e)) << (8 * e);
            }
            if (P.zeros) z = w;
        };
        fetch(scale1, zero1, 0);
        fetch(scale2, zero2, U);
        int acc = 0, xi = 0;
        uint32_t acc_phase = 0, x_phase = 0;
        bool ok = true;
        // A unit of U groups: code for each of them, so that what depends on the group's place costs nothing, but no more of it
        // -- unrolled further it does not fit the instruction caches beside the other warps' and took up to twice the time.
#pragma unroll 1
        for (int g0 = 0; g0 < groups && ok; g0 += U) {
#pragma unroll
            for (int e = 0; e < U; ++e) { scale[e] = scale1[e]; scale1[e] = scale2[e]; }
            zero = zero1;
            zero1 = zero2;
            fetch(scale2, zero2, g0 + 2 * U);
            const int in_block = C::GPB == U ? 0 : g0 % C::GPB;  // groups of the block before this unit
            if (in_block == 0 && !mbar_wait(x_full(xi), x_phase, &abort_flag, &g_w4_status, 0x300 | xi)) break;
            const uint8_t* x_block = smem + xi * 2 * C::X_BYTES + C::B_BYTES;
#pragma unroll
            for (int b0 = 0; b0 < U; b0 += C::BATCH) {
                if (g0 + b0 >= groups) break;
                if (!mbar_wait(acc_full(acc), acc_phase, &abort_flag, &g_w4_status, 0x310 | acc)) { ok = false; break; }
                fence_after();
                // RC rows of a group at a time, the next on their way while these are joined
                constexpr int RC = C::RC, PER_GROUP = C::MINE / RC, CHUNKS = C::BATCH * PER_GROUP;
                const uint32_t t_acc = t_row + acc * C::BATCH * C::N;
                uint32_t d[2][RC * 8];
                tmem_ld_cols(t_acc, d[0]);
#pragma unroll
                for (int c = 0; c < CHUNKS; ++c) {
                    const int g = b0 + c / PER_GROUP, r0 = c % PER_GROUP * RC;  // group of the unit, first row
                    const int gb = in_block + g;                               // ... of the block
                    const float* tables = reinterpret_cast<const float*>(x_block + gb / C::GPP * C::X_BYTES);
                    const float* sums = tables + ((gb % C::GPP) * ROWS + r_first + r0) * 4;
                    const float* step = tables + C::GPP * ROWS * 4 + r_first + r0;
                    const float z = -static_cast<float>((zero >> (8 * g)) & 255u);
                    float4 ds[RC];
                    float up[RC];
#pragma unroll
                    for (int r = 0; r < RC; ++r) {
                        ds[r] = *reinterpret_cast<const float4*>(sums + r * 4);
                        up[r] = step[r] * scale[g];
                    }
                    tmem_ld_wait();
                    if (c + 1 < CHUNKS) {
                        tmem_ld_cols(t_acc + (c + 1) / PER_GROUP * C::N + (c + 1) % PER_GROUP * RC * 8, d[(c + 1) & 1]);
                    } else {  // read completely
                        fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(acc_empty(acc));
                    }
                    if (g0 + g >= groups) continue;  // (a batch cut short: nothing was multiplied into this accumulator)
#pragma unroll
                    for (int r = 0; r < RC; ++r) {
                        const uint32_t* q = &d[c & 1][r * 8];
                        auto pair = [&](int e) { return fmaf(__uint_as_float(q[2 * e + 1]), 32.0f, __uint_as_float(q[2 * e])); };  // exact: below 2^20 units
                        const float w0 = fmaf(z, ds[r].x, pair(0)), w1 = fmaf(z, ds[r].y, pair(1)), w2 = fmaf(z, ds[r].z, pair(2)), w3 = fmaf(z, ds[r].w, pair(3));
                        // (Joined in units of the upper digits, so that up is the size of the group's largest product: it leaves fp32's
                        // range where that does.  In units of digit 0 it was subnormal below products of 1e-32.  A factor of its own for
                        // the step costs 2 to 7 %.)
                        result[r0 + r] = fmaf(fmaf(fmaf(w1, 1024.0f, w0), 1.0f / 1048576.0f, fmaf(w3, 1024.0f, w2)), up[r], result[r0 + r]);
                    }
                }
                acc ^= 1;
                acc_phase ^= static_cast<uint32_t>(acc == 0);
            }
            if (in_block + U == C::GPB || g0 + U >= groups) {
                __syncwarp();
                if (lane == 0) mbar_arrive(x_empty(xi));
                if (++xi == C::XS) { xi = 0; x_phase ^= 1u; }
            }
        }
    }

    // ---- the sums of the cluster's CTAs ----
    fence_before();
    __syncthreads();  // no operand is read any more
    if (abort_flag) {  // a wait has run out: no plausible numbers
        settle();
#pragma unroll
        for (int r = 0; r < C::MINE; ++r) result[r] = __int_as_float(0x7fc00000);
    }
    fence_after();
    if (warp == W_MMA) tmem_dealloc<1>(tmem, C::TMEM_COLS);
    float* const R = reinterpret_cast<float*>(smem);
    if (warp < C::DRAIN) {
#pragma unroll
        for (int r = 0; r < C::MINE; ++r) R[((warp >> 2) * C::MINE + r) * R_PITCH + (warp & 3) * 32 + lane] = result[r];
    }
    if (split > 1) cluster_sync_all();
    else __syncthreads();
    const int outs = rows * MM_COLS;
    for (int t = rank * C::THREADS + tid; t < outs; t += split * C::THREADS) {
        const int r = t / MM_COLS, c = t % MM_COLS;
        if (col_base + c >= P.n) continue;
        float v = 0.0f;
        if (split > 1) {
            const uint32_t from = smem_u32(R + r * R_PITCH + c);
            float p[8];
#pragma unroll
            for (int s = 0; s < 8; ++s)
                if (s < split) asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(p[s]) : "r"(map_to_cta(from, static_cast<uint32_t>(s))) : "memory");
#pragma unroll
            for (int s = 0; s < 8; ++s)
                if (s < split) v += p[s];
        } else {
            v = R[r * R_PITCH + c];
        }
        if (P.bias) v += __ldg(P.bias + col_base + c);
        if (P.relu) v = v <= 0.0f ? 0.0f : v;  // (a NaN stays one)
        P.y[(row_base + r) * P.ldy + col_base + c] = v;
    }
    if (split > 1) cluster_sync_all();  // the peers have read this CTA's sums
}

template <int GROUP, int ROWS>
ctk_status launch_matmul(MmArgs P, int split, cudaStream_t st) {
    using C = MmCfg<GROUP, ROWS>;
    auto kernel = w4_matmul_kernel<GROUP, ROWS>;
    static ctk::PerDeviceReady ready;
    ctk_status set = ready.ensure([&]() -> ctk_status {
        CTK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
        return CTK_OK;
    });
    if (set) return set;
    const int64_t col_blocks = (P.n + MM_COLS - 1) / MM_COLS, row_blocks = (P.m + ROWS - 1) / ROWS, pieces = (P.groups + C::GPP - 1) / C::GPP;
    P.split = split;
    if (col_blocks * P.split > 0x7FFFFFFF || row_blocks > 65535 || (pieces + 3) / 4 > 65535) return fail(CTK_ERR_LIMIT, "ctk_w4_matmul_f32: k or n too large");
    // Where a CTA's share of x is small it makes the digits itself, the same ones in every CTA of the row of column blocks: no
    // first kernel, no scratch.  3 x 1001 x 517 g32: 8.2 us a call against 10.1, 5.7 against 6.1 in a graph; 8 x 1024 x 4096 g64:
    // 19 us from the call to its end against 21, but 7.8 against 7.4 in a graph.  With shares of 8 pieces the first kernel wins
    // there by more (1 x 4096 x 4096 g128: 6.9 us against 7.6).
    StreamScratch scratch;
    int64_t share = 0;  // the longest one, in pieces
    for (int r = 0; r < split; ++r) share = std::max(share, C::share_begin(pieces, r + 1, split) - C::share_begin(pieces, r, split));
    const bool alone = share <= 4 && share * ROWS <= 16;
    static_assert(2 * C::XS >= 4, "a share fits the ring");
    if (pieces && !alone) {
        ctk_status rc = scratch.get(static_cast<size_t>(row_blocks * pieces) * C::X_BYTES, st);
        if (rc) return rc;
        uint8_t* image = static_cast<uint8_t*>(scratch.p);
        P.image = image;
        w4_digits_kernel<GROUP, ROWS><<<dim3(static_cast<unsigned>(row_blocks * ROWS), static_cast<unsigned>((pieces + 3) / 4)), 128, 0, st>>>(P.x, P.ldx, P.m, P.k, pieces, image);
        CTK_LAUNCH_CHECK("w4_digits");
    }
    // the codes as a matrix of 32-bit words, 128 columns x 32 words a copy; what lies past its extents reads as zero
    CUtensorMap codes = {};
    if (pieces) {
        t5::EncodeTiledFn enc;
        ctk_status rc = t5::get_encoder(&enc);
        if (rc) return rc;
        const cuuint64_t words = static_cast<cuuint64_t>(P.groups) * (GROUP / 8);
        const cuuint64_t dims[2] = {words, static_cast<cuuint64_t>(P.n)}, strides[1] = {words * 4};
        const cuuint32_t box[2] = {MM_BLOCK / 8, MM_COLS}, estr[2] = {1u, 1u};
        const CUresult r = enc(&codes, CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, const_cast<uint32_t*>(P.packed), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
        if (r != CUDA_SUCCESS) return fail(CTK_ERR_CUDA, "cuTensorMapEncodeTiled failed with code " + std::to_string(static_cast<int>(r)));
    }
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(P.split);
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // may start before the digits are written, up to its griddepcontrol.wait
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3(static_cast<unsigned>(col_blocks * P.split), static_cast<unsigned>(row_blocks));
    cfg.blockDim = dim3(C::THREADS);
    cfg.dynamicSmemBytes = C::SMEM;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = P.image ? 2 : 1;  // (without the first kernel there is nothing to wait for in the kernel)
    CTK_CUDA(cudaLaunchKernelEx(&cfg, kernel, codes, P));
    CTK_LAUNCH_CHECK("w4_matmul");
    return CTK_OK;
}
// How many rows a CTA takes and how many CTAs share a column's k: the pair with the least estimated time.  A CTA's start and end
// cost START clocks (barriers, first loads, the cluster's sums), a block of 256 k in an SM that is full (two CTAs up to 8 rows,
// one above) PER_BLOCK; alone on its SM a CTA of few rows is 1.4 times slower per block.  From 16384 x 16384 g128: 31.6 / 36 /
// 45 / 68 us with 2 / 4 / 8 / 16 rows, 253 us for 64 rows in three passes of 24.  So 64 x 4096 x 4096 takes 16 rows and whole
// columns (128 CTAs: 21.6 us; 24 rows and a split of 4: 31.8 us; 8 rows: 23.2 us) and 1 x 4096 x 4096 2 rows and a split of 4.
struct Shape {
    int rows, split;
};
Shape pick_shape(int64_t m, int64_t n, int64_t groups, int group) {
    constexpr int ROWS[5] = {2, 4, 8, 16, 24}, PER_SM[5] = {2, 2, 2, 1, 1};
    constexpr double PER_BLOCK[5] = {1060, 1200, 1490, 2330, 2900}, START = 5000;
    const int64_t sms = ctk::sm_count(), cols = (n + MM_COLS - 1) / MM_COLS, blocks = (groups * group + MM_BLOCK - 1) / MM_BLOCK;
    Shape best = {24, 1};
    double least = 1e300;
    for (int i = 0; i < 5; ++i) {
        if (i && ROWS[i - 1] >= m) break;  // fewer rows hold them all
        const int64_t row_blocks = (m + ROWS[i] - 1) / ROWS[i];
        for (int split = 1; split <= 8 && (split == 1 || groups >= 8 * split); split *= 2) {
            const int64_t ctas = cols * row_blocks * split, waves = (ctas + sms * PER_SM[i] - 1) / (sms * PER_SM[i]);
            const bool alone = PER_SM[i] == 2 && ctas <= sms;
            const double per_cta = static_cast<double>((blocks + split - 1) / split);
            const double t = static_cast<double>(waves) * (START + per_cta * PER_BLOCK[i] * (alone ? 1.4 : PER_SM[i]));
            if (t < least) {
                least = t;
                best = {ROWS[i], split};
            }
        }
    }
    return best;
}
template <int GROUP>
ctk_status matmul_rows(const MmArgs& P, cudaStream_t st) {
    const Shape s = pick_shape(P.m, P.n, P.groups, GROUP);
    switch (s.rows) {
        case 2: return launch_matmul<GROUP, 2>(P, s.split, st);
        case 4: return launch_matmul<GROUP, 4>(P, s.split, st);
        case 8: return launch_matmul<GROUP, 8>(P, s.split, st);
        case 16: return launch_matmul<GROUP, 16>(P, s.split, st);
        default: return launch_matmul<GROUP, 24>(P, s.split, st);
    }
}

// Whether an fp32 matrix shares memory with a part of the 4-bit weight.
bool touches_weight(const float* a, int64_t rows, int64_t cols, int64_t ld, const uint32_t* packed, const float* scales, const uint8_t* zeros, int64_t k, int64_t n, int group) {
    const size_t groups = static_cast<size_t>((k + group - 1) / group) * static_cast<size_t>(n);
    return touches(a, rows, cols, ld, packed, groups * static_cast<size_t>(group / 2)) || touches(a, rows, cols, ld, scales, groups * 4) || touches(a, rows, cols, ld, zeros, groups);
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
    CTK_REQUIRE(!touches_weight(w, k, n, ldw, packed, scales, zeros, k, n, group), "ctk_w4_quantize_f32: w overlaps packed, scales or zeros");
    const int64_t groups = (k + group - 1) / group, per_cta = group == 32 ? quantize_parts(32) : 1;
    const int64_t grid = (groups + per_cta - 1) / per_cta * ((n + W4_THREADS - 1) / W4_THREADS);
    if (grid > 0x7FFFFFFF) return fail(CTK_ERR_LIMIT, "ctk_w4_quantize_f32: too many groups");
    const bool wide = aligned_to(scales, 16) && aligned_to(zeros, 4);
    auto go = [&](auto kernel) { kernel<<<static_cast<unsigned>(grid), W4_THREADS * quantize_parts(group), 0, as_stream(stream)>>>(w, ldw, k, n, groups, packed, scales, zeros, wide); };
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
    CTK_REQUIRE(!touches_weight(w, k, n, ldw, packed, scales, zeros, k, n, group), "ctk_w4_dequantize_f32: w overlaps packed, scales or zeros");
    const int64_t groups = (k + group - 1) / group, grid = (k + 31) / 32 * ((n + W4_THREADS - 1) / W4_THREADS);
    if (grid > 0x7FFFFFFF) return fail(CTK_ERR_LIMIT, "ctk_w4_dequantize_f32: too large");
    w4_dequantize_kernel<<<static_cast<unsigned>(grid), W4_THREADS, 0, as_stream(stream)>>>(packed, scales, zeros, k, n, group, groups, w, ldw);
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
    CTK_REQUIRE(!touches_weight(y, m, n, ldy, packed, scales, zeros, k, n, group), "ctk_w4_matmul_f32: y overlaps packed, scales or zeros");
    // (one row added to what y holds: each element is read before it is written, and by the same thread)
    CTK_REQUIRE((m == 1 && bias == y) || !touches(y, m, n, ldy, bias, static_cast<size_t>(n) * 4), "ctk_w4_matmul_f32: y overlaps bias");
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
    P.quads = P.groups % 4 == 0 && aligned_to(scales, 16) && aligned_to(zeros, 4);
    cudaStream_t st = as_stream(stream);
    // x's digits take 8.3 to 12 bytes per element of x (X_BYTES / (128 ROWS)): many rows go in slabs of at most 512 MB of them (a
    // multiple of every kernel's rows)
    const int64_t per_row = P.groups * group * 12 + 1, slab = std::min<int64_t>(65520, std::max<int64_t>(48, (int64_t(512) << 20) / per_row / 48 * 48));
    for (int64_t r = 0; r < m; r += slab) {
        MmArgs Q = P;
        Q.m = m - r < slab ? m - r : slab;
        Q.x = x + r * ldx;
        Q.y = y + r * ldy;
        const ctk_status rc = group == 32 ? matmul_rows<32>(Q, st) : group == 64 ? matmul_rows<64>(Q, st) : matmul_rows<128>(Q, st);
        if (rc) return rc;
    }
    return CTK_OK;
}

ctk_status ctk_w4_status(int* status) {
    CTK_REQUIRE(status, "ctk_w4_status: null pointer");
    CTK_CUDA(cudaDeviceSynchronize());
    CTK_CUDA(cudaMemcpyFromSymbol(status, g_w4_status, sizeof(int)));
    return CTK_OK;
}

}  // extern "C"
