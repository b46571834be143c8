// Matrices held in 4 bits: packing, reading back, and the product with few rows of x (packed.cuh says how they lie in memory).
#define CHIBI_UNIT packed_weights
#define CHIBI_UNIT_ID 19
#include "packed.cuh"
#include "sm100.cuh"

#include <cuda_fp16.h>
#include <string.h>

#include <type_traits>

namespace chibi {
namespace {

// ------------------------------------------------------------------ packing
// 128 threads make one record: thread (r, b) the four words of row r's columns 32 b ... 32 b + 31 (with one word a thread, what is
// done once a thread was most of the work: 64 us instead of 37 for 12,288 x 4,096 bfloat16 numbers, 3.4 TB/s).  The threads of a group (1, 2 or 4
// neighbouring lanes) find its largest element together.
//   s = bf16(m / -8), m the element of largest magnitude, the first of equals; q = w / s rounded to nearest, ties to even,
//   within -8 ... 7.  A group with what is not a finite number has the scale NaN.
// The quotient is w times 1 / s and one correction from what is left of w (exact), which makes it the 32-bit number nearest to
// w / s.  For bfloat16 w that decides: w / s has 8 bits over 8 bits, so it is a half or far from one.  A 32-bit w / s can be so close
// to a half that the nearest 32-bit number is the half itself; a thread that meets one decides again with w - q s, which is exact
// (q s has 12 bits, and the difference no more than w has).
struct PackSource {
    const void* w[2];          // a matrix, or gate and up
    long long stride[2];
    int rows, cols;            // of each
    int pair;
};

// q + 8 for an element next to a half, by w - q s against s / 2.
__device__ __noinline__ uint32_t code_next_to_a_half(float w, float s)
{
    float q = fminf(fmaxf(rintf(w / s), -9.f), 8.f);
    const float rest = fmaf(-q, s, w), half = 0.5f * fabsf(s);
    const float away = (rest > 0.f) == (s > 0.f) ? 1.f : -1.f;
    if (fabsf(rest) > half || (fabsf(rest) == half && ((int)q & 1)))
        q += away;
    return (uint32_t)((int)fminf(fmaxf(q, -8.f), 7.f) + 8);
}

template <typename T> __device__ __forceinline__ uint32_t code_word(const T (&w)[8], float s, float by)
{
    // (1.5 2^23 + 8: the sum's last bits are the whole number plus 8)
    constexpr float SHIFT = 12582920.f;
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
        v[i] = to_f32(w[i]);
    uint32_t word = 0;
    float far = 0.f;                             // the largest distance from a whole number
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float t = v[i] * by;
        // (|w / s| is 8.04 at most, the smallest s aside: -8.04 goes to -8, 8 has to go to 7)
        const float q = fminf(fmaf(fmaf(-t, s, v[i]), by, t), 7.25f);
        const float sum = q + SHIFT;
        if (sizeof(T) == 4)
            far = fmaxf(far, fabsf(q - (sum - SHIFT)));
        word |= (__float_as_uint(sum) & 15u) << (4 * (i / 2) + 16 * (i & 1));
    }
    // (the smallest s: 1 / s is infinite, or s has lost so many bits that w / s is beyond -8)
    if (far < 0.5f && fabsf(s) >= 0x1p-125f)
        return word;
    word = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
        word |= code_next_to_a_half(v[i], s) << (4 * (i / 2) + 16 * (i & 1));
    return word;
}

// 8 neighbouring numbers of a row from column `col` on, zeros beyond its k columns.
template <typename T> __device__ __forceinline__ void read_eight(const T* row, int col, int k, T (&v)[8])
{
    const T* src = row + col;
    if (col + 8 <= k && (reinterpret_cast<uintptr_t>(src) & 15) == 0) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i)
            reinterpret_cast<uint4*>(v)[i] = reinterpret_cast<const uint4*>(src)[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            v[i] = col + i < k ? src[i] : from_f32<T>(0.f);
    }
}

// Products fetch their matrix before the kernel ahead of them has ended.  So the kernels that write one, in 4 bits or as values read
// back, let nothing start early (no pdl_trigger; and no mark in a timeline), and every thread's stores are performed, for tile copies
// too, before it ends.
__device__ __forceinline__ void packed_done()
{
    __threadfence();
    asm volatile("fence.proxy.async;" ::: "memory");
}

// A block's records, gridDim.x apart.
struct RecordWalk {
    int rb, cb, rows_step, cols_step, col_blocks;
    __device__ __forceinline__ explicit RecordWalk(int col_blocks_)
        : rb(blockIdx.x / col_blocks_), cb(blockIdx.x % col_blocks_), rows_step(gridDim.x / col_blocks_),
          cols_step(gridDim.x % col_blocks_), col_blocks(col_blocks_)
    {
    }
    __device__ __forceinline__ void next()
    {
        rb += rows_step;
        cb += cols_step;
        if (cb >= col_blocks) {
            cb -= col_blocks;
            ++rb;
        }
    }
};

template <typename T>
__global__ void __launch_bounds__(128, 8) pack_kernel(PackSource p, int row_blocks, int col_blocks, int group, uint8_t* out)
{
    pdl_wait_now();                                  // (see packed_done)
    const int r = threadIdx.x >> 2, b = threadIdx.x & 3;
    const int lanes = group / 32;
    const int side = packed_side(p.pair, r);
    const T* base = static_cast<const T*>(side ? p.w[1] : p.w[0]);
    const long long stride = side ? p.stride[1] : p.stride[0];
    for (RecordWalk at(col_blocks); at.rb < row_blocks; at.next()) {
        const int row = packed_source_row(p.pair, at.rb, r), col = at.cb * PACKED_COLS + b * 32;
        // (a row beyond the matrix is read as one without columns)
        const T* src = base + (row < p.rows ? (long long)row * stride : 0);
        const int cols = row < p.rows ? p.cols : 0;
        __align__(16) T raw[4][8];
#pragma unroll
        for (int c = 0; c < 4; ++c)
            read_eight(src, col + c * 8, cols, raw[c]);
        // The largest positive and the largest negative element, by their bits as whole numbers with and without a sign (what
        // is not finite is beyond all that is); bfloat16 two at a time.
        int most_bits = (int)0x80000000;
        uint32_t least_bits = 0;
        if constexpr (sizeof(T) == 2) {
            const uint32_t* two = reinterpret_cast<const uint32_t*>(raw);
            uint32_t most_two = __vmaxs2(two[0], two[15]), least_two = __vmaxu2(two[0], two[15]);
#pragma unroll
            for (int i = 1; i < 15; i += 2) {
                most_two = __vimax3_s16x2(most_two, two[i], two[i + 1]);
                least_two = __vimax3_u16x2(least_two, two[i], two[i + 1]);
            }
            most_bits = max((int)(most_two << 16), (int)(most_two & 0xffff0000u));
            least_bits = max(least_two << 16, least_two & 0xffff0000u);
        } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                most_bits = max(most_bits, __float_as_int(to_f32(raw[i / 8][i % 8])));
                least_bits = max(least_bits, __float_as_uint(to_f32(raw[i / 8][i % 8])));
            }
        }
        for (int o = 1; o < lanes; o <<= 1) {
            most_bits = max(most_bits, __shfl_xor_sync(0xffffffffu, most_bits, o));
            least_bits = max(least_bits, __shfl_xor_sync(0xffffffffu, least_bits, o));
        }
        const uint32_t above = most_bits > 0 ? (uint32_t)most_bits : 0u, below = least_bits > 0x80000000u ? least_bits & 0x7fffffffu : 0u;
        const bool finite = max(above, below) < 0x7f800000u;
        bool up = above > below;
        if (__any_sync(0xffffffffu, above == below && above != 0)) {
            // both signs: the first of equals (a group's lanes are neighbours, a lane's elements in order)
            int first = 0;                           // 1 positive, -1 negative
#pragma unroll
            for (int i = 31; i >= 0; --i) {
                const float v = to_f32(raw[i / 8][i % 8]);
                first = (__float_as_uint(v) & 0x7fffffffu) == above ? (__float_as_int(v) >= 0 ? 1 : -1) : first;
            }
            const uint32_t group_lanes = ((1u << lanes) - 1u) << (threadIdx.x & 31 & ~(lanes - 1));
            const uint32_t have = __ballot_sync(0xffffffffu, first != 0) & group_lanes;
            const int sign = __shfl_sync(0xffffffffu, first, have ? __ffs(have) - 1 : 0);
            up = above == below ? sign > 0 : up;
        }
        const float best = __uint_as_float(up ? above : below | 0x80000000u);
        __nv_bfloat16 s16 = __float2bfloat16_rn(finite ? best * -0.125f : __int_as_float(0x7fc00000));
        const float s = __bfloat162float(s16);
        if (s == 0.f)
            s16 = __float2bfloat16_rn(0.f);      // (no minus zeros)
        const bool any = finite && s != 0.f;
        const float by = 1.f / s;
        uint8_t* dst = out + ((long long)at.rb * col_blocks + at.cb) * packed_record_bytes(group);
#pragma unroll
        for (int c = 0; c < 4; ++c)
            *reinterpret_cast<uint32_t*>(dst + packed_word_at(r, b * 4 + c)) = any ? code_word<T>(raw[c], s, by) : 0x88888888u;
        if (b % lanes == 0)
            *reinterpret_cast<__nv_bfloat16*>(dst + packed_scale_at(r, b / lanes)) = s16;
    }
    packed_done();
}

// Whole numbers and scales that somebody else has made, into records.
struct CodeSource {
    const int8_t* codes[2];
    const __nv_bfloat16* scales[2];
    long long stride[2], scale_stride[2];
    int rows, cols, pair;
};

__global__ void __launch_bounds__(512, 4) pack_codes_kernel(CodeSource p, int row_blocks, int col_blocks, int group, uint8_t* out)
{
    pdl_wait_now();
    const int r = threadIdx.x >> 4, seg = threadIdx.x & 15;
    const int lanes = group / 8;
    for (RecordWalk at(col_blocks); at.rb < row_blocks; at.next()) {
        const int rb = at.rb, cb = at.cb;
        const int side = packed_side(p.pair, r), row = packed_source_row(p.pair, rb, r);
        const int col = cb * PACKED_COLS + seg * 8;
        uint32_t word = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int q = row < p.rows && col + i < p.cols ? p.codes[side][(long long)row * p.stride[side] + col + i] : 0;
            word |= (uint32_t)((q + 8) & 15) << (4 * (i / 2) + 16 * (i & 1));
        }
        uint8_t* dst = out + ((long long)rb * col_blocks + cb) * packed_record_bytes(group);
        *reinterpret_cast<uint32_t*>(dst + packed_word_at(r, seg)) = word;
        if (seg % lanes == 0)
            *reinterpret_cast<__nv_bfloat16*>(dst + packed_scale_at(r, seg / lanes))
                = row < p.rows && col < p.cols ? p.scales[side][(long long)row * p.scale_stride[side] + col / group] : __float2bfloat16_rn(0.f);
    }
    packed_done();
}

// The values, rows of a pair's first matrix before those of its second.  A thread makes 16 neighbouring bytes of the output, so a
// warp writes whole lines; the next record's codes are on their way meanwhile.
template <typename T>
__global__ void __launch_bounds__(512, 4) unpack_kernel(const uint8_t* __restrict__ data, int row_blocks, int col_blocks, int group, int rows,
                                                     int cols, int pair, T* __restrict__ out, long long stride)
{
    pdl_wait_now();                                  // (see packed_done)
    constexpr int EACH = 16 / sizeof(T), ROW_THREADS = PACKED_COLS / EACH, TURNS = PACKED_ROWS * ROW_THREADS / 512;
    uint32_t next_word[TURNS];
    __nv_bfloat16 next_scale[TURNS];
    auto fetch = [&](const RecordWalk& at) {
        const uint8_t* src = data + ((long long)at.rb * col_blocks + at.cb) * packed_record_bytes(group);
#pragma unroll
        for (int turn = 0; turn < TURNS; ++turn) {
            const int i = threadIdx.x + turn * 512, r = i / ROW_THREADS, col = i % ROW_THREADS * EACH;
            next_word[turn] = *reinterpret_cast<const uint32_t*>(src + packed_word_at(r, col >> 3));
            next_scale[turn] = *reinterpret_cast<const __nv_bfloat16*>(src + packed_scale_at(r, col / group));
        }
    };
    RecordWalk at(col_blocks), ahead = at;
    if (ahead.rb < row_blocks)
        fetch(ahead);
    for (; at.rb < row_blocks; at.next()) {
        uint32_t words[TURNS];
        float scales[TURNS];
#pragma unroll
        for (int turn = 0; turn < TURNS; ++turn) {
            words[turn] = next_word[turn];
            scales[turn] = to_f32(next_scale[turn]);
        }
        ahead.next();
        if (ahead.rb < row_blocks)
            fetch(ahead);
#pragma unroll
        for (int turn = 0; turn < TURNS; ++turn) {
            const int i = threadIdx.x + turn * 512, r = i / ROW_THREADS, first = i % ROW_THREADS * EACH;
            const int row = packed_source_row(pair, at.rb, r), col = at.cb * PACKED_COLS + first;
            if (row >= rows || col >= cols)
                continue;
            T* dst = out + (long long)(row + packed_side(pair, r) * rows) * stride + col;
            __align__(16) T v[EACH];
#pragma unroll
            for (int j = 0; j < EACH; ++j) {
                const int e = (first & 7) + j;
                // (2^23 + code has its code in the last bits)
                v[j] = from_f32<T>((__uint_as_float(0x4b000000u | ((words[turn] >> (4 * (e / 2) + 16 * (e & 1))) & 15u)) - 8388616.f) * scales[turn]);
            }
            if (col + EACH <= cols && (reinterpret_cast<uintptr_t>(dst) & 15) == 0)
                *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(v);
            else
                for (int j = 0; j < EACH && col + j < cols; ++j)
                    dst[j] = v[j];
        }
    }
    packed_done();
}

// ------------------------------------------------------------------ few rows of x
// out[m][n] = sum over groups of s[n][g] * (sum over the group of q[n][k] x[m][k]).
//
// What bounds it is the bytes of the matrix.  A CTA of 8 or 16 warps stays on its SM; every warp streams records of its own
// (tile copies into a ring of its own, no barrier between warps), makes float16 fragments of the codes and multiplies
// them with x by `mma.m16n8k16`: 16 rows of a record are the instruction's rows, 8 tokens its columns.  x lies in shared
// memory as the fragments want it, 16 bytes to a lane for four instructions.  Each group's sums start at zero and are
// multiplied by the scales in 32 bits.  (The codes are held times 2^-14, so that this does not pass 2^128 where a row of x has been
// multiplied: 2^-100 times 64 sevens of scale 2^106 came out infinite.)
//
// x becomes float16 too (two nibbles of a word are float16 numbers without a shift, which bfloat16's seven bits of mantissa
// do not allow; the conversion of the codes is most of the kernel's instructions).  A row's numbers, as far as the CTA's columns go, are
// multiplied by a power of two and its sums by the inverse: 2^6 where that keeps every bit of a bfloat16 row (its numbers within
// 2^-20 ... 2^9, as a norm's output has them, or zero), else the one that brings the largest to 2^14 ... 2^15.  So bfloat16 numbers from
// 2^-28 of the largest on keep all of their bits.  32-bit numbers are two float16 numbers, the nearest and the nearest to what is left:
// off by 2^-23 of themselves, or by 2^-25, half of float16's last step, which is 2^-39 of the row's largest at most and 2^-16 of
// numbers from 2^-9 on.  What is smaller (bfloat16: 2^-14, 32-bit: 2^-9, as multiplied) and lost bits is added to the warps' sums in
// 32 bits after the stream, so nothing vanishes beside a large number whose weights are zeros (add_what_was_lost; a row of 4,096 normal
// numbers has one with a chance of 1e-5, a 32-bit one of 1e-3; one such number makes the product with 4,096 x 4,096 take 7.4 us
// instead of 4.8, a row of nothing else 31).
//
// How the work is shared out (CudaKernels.packed_plan chooses): `splits` CTAs of a cluster share the columns, `along_k`
// warps of a CTA share the CTA's columns of one block of 32 rows, the CTA's warps / along_k blocks of rows are a unit, and clusters
// take units in turn.  The sums of up to `batch` units stay in shared memory; then the cluster adds them up in one order
// (each CTA its warps, then CTA by CTA), each CTA a share of the outputs, so the same plan gives the same bits.
//
// Measured (replayed in a graph, matrices out of L2): one row of 2,048 x 1,024 3.0 us, of 4,096 x 4,096 4.8, of 4,096 x 12,288 9.0, of a gated
// pair of 2 x 12,288 x 4,096 13.2 (4.1 TB/s); four rows of 151,936 x 4,096 64.6 (5.1 TB/s), 284 instructions a record at 2.55 a
// cycle and SM; 12 32-bit rows of a pair of 2 x 2,730 x 1,024 6.3.  Before and after the stream of one row go by 2.5 us: a kernel's start, x from
// L2, a barrier, the warps' sums.
constexpr int FEW_THREADS = 512;             // at most

struct FewRows {
    int row_blocks, chunks;        // blocks of 32 rows, of 128 columns
    int n, k, pair;
    const void* x;
    long long x_stride;
    int m;
    void* out;
    int out_type;
    long long out_stride;
    const float* residual;
    long long residual_stride;
    int act;                       // pairs: 1 gelu with tanh, 2 silu
    int warps, split_shift, along_shift, batch, depth, run, tokens;  // run: records of a stage; tokens: rows of x of a CTA
    int clusters, units;
    int* error;
    const uint8_t* data;           // the records, for what goes around the tile copies
};

// FIRST: d is what comes out, else it is added to.
template <bool FIRST> __device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    if constexpr (FIRST) {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
        return;
    }
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float peer_shared_f32(uint32_t own_smem_addr, uint32_t rank)
{
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(sm100::peer_smem_addr(own_smem_addr, rank)) : "memory");
    return v;
}

// The exponents of the powers of two by which rows are multiplied: the first, with the range that it suits (as bits of an exponent),
// and what a row's largest finite magnitude asks for.  (As far as a 32-bit number goes: rows below 2^-112 come out smaller.)
constexpr int ROW_EXPONENT = 6;
constexpr uint32_t ROW_LEAST = 127 - 14 - ROW_EXPONENT, ROW_MOST = 127 + 15 - ROW_EXPONENT;
__device__ __forceinline__ int row_exponent(uint32_t largest_bits)
{
    return largest_bits == 0 ? 0 : min(14 + 127 - (int)(largest_bits >> 23), 126);
}
struct RowNotes {
    uint32_t largest[16];          // their largest finite magnitudes, as bits (where a row's factor is its own)
    int exponent[16];              // of their factors
    uint32_t lossy, odd;           // a bit for each that lost bits; for each that the first factor does not suit
};
__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((e + 127) << 23); }

// Two numbers as float16, and what is left of them (nothing of an infinity or NaN).
__device__ __forceinline__ uint32_t take_half_pair(float (&v)[2])
{
    const __half2 h = __floats2half2_rn(v[0], v[1]);
    v[0] = isfinite(v[0]) ? v[0] - __low2float(h) : 0.f;
    v[1] = isfinite(v[1]) ? v[1] - __high2float(h) : 0.f;
    return *reinterpret_cast<const uint32_t*>(&h);
}

// Numbers below this, as multiplied, may have lost bits that count.
template <bool X32> __device__ __forceinline__ float least_kept() { return X32 ? 0x1p-9f : 0x1p-14f; }
// What float16 has lost of such a number, exactly: v and the multiple of 2^(-24 - e) next to it differ by what 24 bits hold.
template <bool X32> __device__ __forceinline__ float lost_of(float v, int e)
{
    const float up = v * power_of_two(e);
    float held = __half2float(__float2half_rn(up));
    if (X32)
        held += __half2float(__float2half_rn(up - held));
    return fabsf(up) < least_kept<X32>() ? fmaf(-held, power_of_two(-e), v) : 0.f;
}

// Adds what the rows of x in `rows` (a bit each) lost to a warp's sums of a block of 32 rows of the matrix, columns w0 ... w1: a
// lane a row of the matrix.  A number that lost nothing costs its test alone, 32 columns at a time.
template <bool X32, int NT>
__device__ __noinline__ void add_what_was_lost(const FewRows& p, uint32_t rows, int token0, int block, int w0, int w1, int group,
                                               const RowNotes& notes, float* sums)
{
    using T = typename std::conditional<X32, float, __nv_bfloat16>::type;
    const int lane = threadIdx.x & 31;
    for (; rows != 0; rows &= rows - 1) {
        const int token = __ffs(rows) - 1;
        const T* x = static_cast<const T*>(p.x) + (token0 + token) * p.x_stride;
        const int e = notes.exponent[token];
        float sum = 0.f;
#pragma unroll 1
        for (int chunk = w0; chunk < w1; ++chunk) {
            float lost[4];
#pragma unroll
            for (int b = 0; b < 4; ++b) {                    // blocks of 32 columns
                const int col = chunk * PACKED_COLS + b * 32 + lane;
                lost[b] = col < p.k ? to_f32(x[col]) : 0.f;
            }
            bool any = false;
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                lost[b] = lost_of<X32>(lost[b], e);
                any = any || lost[b] != 0.f;
            }
            if (!__any_sync(0xffffffffu, any))
                continue;
            const uint8_t* rec = p.data + ((long long)block * p.chunks + chunk) * packed_record_bytes(group);
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                float part = 0.f;
#pragma unroll 1
                for (uint32_t todo = __ballot_sync(0xffffffffu, lost[b] != 0.f); todo != 0; todo &= todo - 1) {
                    const int j = __ffs(todo) - 1;
                    const uint32_t word = *reinterpret_cast<const uint32_t*>(rec + packed_word_at(lane, b * 4 + (j >> 3)));
                    const int q = (int)((word >> (4 * ((j & 7) / 2) + 16 * (j & 1))) & 15u) - 8;
                    part = fmaf((float)q, __shfl_sync(0xffffffffu, lost[b], j), part);
                }
                sum = fmaf(to_f32(*reinterpret_cast<const __nv_bfloat16*>(rec + packed_scale_at(lane, b * 32 / group))), part, sum);
            }
        }
        // (the fragment's place of the row and the token)
        sums[(((lane >> 4) * NT + (token >> 3)) * 4 + ((lane >> 3) & 1) * 2 + (token & 1)) * 32 + (lane & 7) * 4 + (token & 7) / 2] += sum;
    }
}

// 8 neighbouring numbers of a row as float16, for a lane of four instructions; 32-bit ones in two parts, `plane` bytes apart.
template <typename T> __device__ __forceinline__ void put_piece(uint8_t* to, uint32_t plane, const T (&raw)[8], float up_by)
{
    float pairs[4][2];
#pragma unroll
    for (int j = 0; j < 8; ++j)
        pairs[j / 2][j % 2] = to_f32(raw[j]) * up_by;
#pragma unroll
    for (int part = 0; part < (int)sizeof(T) / 2; ++part)
        *reinterpret_cast<uint4*>(to + part * plane)
            = make_uint4(take_half_pair(pairs[0]), take_half_pair(pairs[1]), take_half_pair(pairs[2]), take_half_pair(pairs[3]));
}

// bfloat16 rows that the first factor does not suit, once more, by all warps: `pieces` of 8 columns from block c0 on.  Begins and ends
// with the CTA together.
__device__ __noinline__ void put_rows_again(const FewRows& p, uint8_t* xs, RowNotes& notes, int token0, int c0, int pieces)
{
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t odd = notes.odd;
    const int rows = __popc(odd), turn = warp / rows, each = p.warps / rows;
    uint32_t from = odd;
    for (int skip = warp - turn * rows; skip > 0; --skip)
        from &= from - 1;
    const int of = __ffs(from) - 1, first = turn < each ? turn * 32 + lane : pieces;
    const __nv_bfloat16* row = static_cast<const __nv_bfloat16*>(p.x) + (token0 + of) * p.x_stride;
    float most = 0.f, least = INFINITY;
#pragma unroll 1
    for (int i = first; i < pieces; i += each * 32) {
        __align__(16) __nv_bfloat16 raw[8];
        read_eight(row, (c0 * 16 + i) * 8, p.k, raw);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float v = fabsf(to_f32(raw[j]));
            most = v < INFINITY ? fmaxf(most, v) : most;
            least = v > 0.f ? fminf(least, v) : least;
        }
    }
    const uint32_t warps_most = __reduce_max_sync(0xffffffffu, __float_as_uint(most));
    if (lane == 0)
        atomicMax(&notes.largest[of], warps_most);
    __syncthreads();
    const int e = row_exponent(notes.largest[of]);
    if (least < least_kept<false>() * power_of_two(-e))
        atomicOr(&notes.lossy, 1u << of);
    if (lane == 0)
        notes.exponent[of] = e;
#pragma unroll 1
    for (int i = first; i < pieces; i += each * 32) {
        __align__(16) __nv_bfloat16 raw[8];
        read_eight(row, (c0 * 16 + i) * 8, p.k, raw);
        put_piece(xs + of * 64 + (i >> 2) * p.tokens * 64 + (i & 3) * 16, 0, raw, power_of_two(e));
    }
    __syncthreads();
}

template <int NT, bool X32, int GROUP_BLOCKS>
__global__ void __launch_bounds__(FEW_THREADS, 1) packed_few_rows_kernel(const __grid_constant__ CUtensorMap map, const __grid_constant__ FewRows p)
{
    using namespace sm100;
    using T = typename std::conditional<X32, float, __nv_bfloat16>::type;
    constexpr int PARTS = X32 ? 2 : 1;
    constexpr int GROUPS = 4 / GROUP_BLOCKS;
    constexpr int RECORD = PACKED_CODE_BYTES + GROUPS * 64;
    constexpr int SUMS = 256 * NT;               // 32-bit sums of a warp
    extern __shared__ __align__(1024) uint8_t smem[];
    pdl_trigger();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int splits = 1 << p.split_shift, along_k = 1 << p.along_shift;
    if (threadIdx.x == 0)
        tma_prefetch_descriptor(&map);
    const int rank = splits > 1 ? (int)cluster_cta_rank() : 0;
    const int cluster = blockIdx.x >> p.split_shift;
    const int token0 = blockIdx.y * p.tokens;
    const int tokens = min(p.tokens, p.m - token0);
    const int c0 = (p.chunks * rank) >> p.split_shift, c1 = (p.chunks * (rank + 1)) >> p.split_shift;
    const int most = (p.chunks + splits - 1) >> p.split_shift;
    const int unit_shift = (p.warps == 16 ? 4 : 3) - p.along_shift, blocks_per_unit = 1 << unit_shift;

    // shared memory: rings | x | sums | notes about the rows of x (RowNotes) | barriers
    const uint32_t x_plane = (uint32_t)most * 4 * p.tokens * 64;
    const int stage = (p.run * RECORD + 127) / 128 * 128;        // (a tile copy's place starts on 128 bytes)
    uint8_t* ring = smem + warp * p.depth * stage;
    uint8_t* xs = smem + p.warps * p.depth * stage;
    float* sums = reinterpret_cast<float*>(xs + (size_t)PARTS * x_plane);
    RowNotes& notes = *reinterpret_cast<RowNotes*>(sums + p.batch * p.warps * SUMS);
    uint64_t* full = reinterpret_cast<uint64_t*>(&notes + 1) + warp * p.depth;

    // the warp's records: of its block of rows in every unit, columns w0 ... w1
    const int wk = warp & (along_k - 1), wr = warp >> p.along_shift;
    const int w0 = c0 + (((c1 - c0) * wk) >> p.along_shift), w1 = c0 + (((c1 - c0) * (wk + 1)) >> p.along_shift);
    const int my_rounds = cluster < p.units ? (p.units - 1 - cluster) / p.clusters + 1 : 0;
    const int last_unit = cluster + (my_rounds - 1) * p.clusters;
    const int warp_rounds = my_rounds > 0 && last_unit * blocks_per_unit + wr >= p.row_blocks ? my_rounds - 1 : my_rounds;
    int rounds_to_ask = w1 > w0 ? warp_rounds : 0, next_chunk = w0, next_block = cluster * blocks_per_unit + wr;
    // asks for the next `run` records of the warp's block of rows (the last of them may be another warp's, or beyond the matrix)
    auto issue = [&](int slot) {
        if (lane == 0) {
            mbar_arrive_expect_tx(&full[slot], p.run * RECORD);
            tma_load_4d(ring + slot * stage, &map, &full[slot], 0, 0, next_chunk, next_block);
        }
        next_chunk += p.run;
        if (next_chunk >= w1) {
            next_chunk = w0;
            next_block += p.clusters * blocks_per_unit;
            --rounds_to_ask;
        }
    };
    if (lane == 0)
        for (int i = 0; i < p.depth; ++i)
            mbar_init(&full[i], 1);
    if (threadIdx.x < 16) {
        notes.largest[threadIdx.x] = 0;
        notes.exponent[threadIdx.x] = ROW_EXPONENT;
    }
    if (threadIdx.x == 0)
        notes.lossy = notes.odd = 0;
    fence_barrier_init();
    fence_proxy_async();
    __syncthreads();
    int open = 0;                                // stages that were asked for and not waited for
    for (; open < p.depth && rounds_to_ask > 0; ++open)
        issue(open);

    // ---- x as fragments: [block of 32 columns][token][lane % 4], 8 neighbouring columns each
    pdl_wait();
    // (warps / tokens warps to a token)
    const int token_pieces = (c1 - c0) * 16, token_warps = p.warps / tokens;
    const int token_turn = warp / tokens, token = warp - token_turn * tokens;
    const int first_piece = token_turn < token_warps ? token_turn * 32 + lane : token_pieces, step = token_warps * 32;
    const T* x_row = static_cast<const T*>(p.x) + (token0 + token) * p.x_stride;
    constexpr float AT_FIRST = float(1 << ROW_EXPONENT);
    auto put = [&](int i, const T (&raw)[8], float up_by) { put_piece(xs + token * 64 + (i >> 2) * p.tokens * 64 + (i & 3) * 16, x_plane, raw, up_by); };
    // A row's factor wants its largest number before any is converted.  32-bit rows are fetched twice, unless a thread's pieces fit its
    // registers and wait there.  bfloat16 rows are multiplied by 2^6 at once, and only those with a number that this does not suit (two at
    // a time, their bits as whole numbers; less 1, so that a zero is the largest of all) once more (put_rows_again):
    // one row of 4,096 x 4,096 4.8 us, such a one 6.2; 8 rows through a gated pair of 2 x 12,288 x 4,096 16.8, with one such 18.3.
    const bool whole = ((reinterpret_cast<uintptr_t>(p.x) | (uintptr_t)p.x_stride * sizeof(T)) & 15) == 0 && (p.k & 7) == 0;  // on 16 bytes
    const int there = min(token_pieces, (p.k - c0 * PACKED_COLS) >> 3);
    const T* src = x_row + c0 * PACKED_COLS;
    // calls f for this thread's pieces: AT_ONCE on their way, one copy of f's code (what a kernel runs once it waits for)
    auto each_piece = [&](auto f) {
        constexpr int AT_ONCE = X32 ? 2 : 4;
        if (whole) {
#pragma unroll 1
            for (int i0 = first_piece; i0 < token_pieces; i0 += AT_ONCE * step) {
                __align__(16) T raw[AT_ONCE][8];
#pragma unroll
                for (int a = 0; a < AT_ONCE; ++a)
#pragma unroll
                    for (int h = 0; h < (int)sizeof(T) / 2; ++h)
                        reinterpret_cast<uint4*>(raw[a])[h]
                            = i0 + a * step < there ? reinterpret_cast<const uint4*>(src + (i0 + a * step) * 8)[h] : make_uint4(0, 0, 0, 0);
#pragma unroll 1
                for (int i = i0; i < min(i0 + AT_ONCE * step, token_pieces); i += step) {
                    f(i, raw[0]);
#pragma unroll
                    for (int a = 0; a + 1 < AT_ONCE; ++a)
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            raw[a][j] = raw[a + 1][j];
                }
            }
        } else {
#pragma unroll 1
            for (int i = first_piece; i < token_pieces; i += step) {
                __align__(16) T raw[8];
                read_eight(x_row, (c0 * 16 + i) * 8, p.k, raw);
                f(i, raw);
            }
        }
    };
    if constexpr (X32) {
        // the largest finite magnitude among this warp's pieces (`most`: the largest of all) into its row's
        auto note_most = [&](float of_all) {
            uint32_t most = __reduce_max_sync(0xffffffffu, __float_as_uint(of_all));
            if (most == 0x7f800000u) {           // (an infinity aside)
                float finite = 0.f;
#pragma unroll 1
                for (int i = first_piece; i < token_pieces; i += step) {
                    __align__(16) T raw[8];
                    read_eight(x_row, (c0 * 16 + i) * 8, p.k, raw);
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        finite = fabsf(raw[j]) < INFINITY ? fmaxf(finite, fabsf(raw[j])) : finite;
                }
                most = __reduce_max_sync(0xffffffffu, __float_as_uint(finite));
            }
            if (lane == 0)
                atomicMax(&notes.largest[token], most);
        };
        uint32_t smallest = 0xffffffffu;         // but zero, its bits less 1
        auto note_row = [&](int e) {
            if (smallest < __float_as_uint(least_kept<X32>() * power_of_two(-e)) - 1)
                atomicOr(&notes.lossy, 1u << token);
            if (lane == 0)
                notes.exponent[token] = e;
        };
        auto put_and_note = [&](int i, const T (&raw)[8], int e) {
            put(i, raw, power_of_two(e));
#pragma unroll
            for (int j = 0; j < 8; ++j)
                smallest = __viaddmin_u32(__float_as_uint(raw[j]) & 0x7fffffffu, 0xffffffffu, smallest);
        };
        float most = 0.f;                        // (fmaxf passes NaN over)
        auto look = [&](const T (&raw)[8]) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                most = fmaxf(most, fabsf(raw[j]));
        };
        constexpr int KEPT = 4;
        if (whole && token_pieces <= KEPT * step) {
            __align__(16) T raw[KEPT][8];
#pragma unroll
            for (int a = 0; a < KEPT; ++a)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    reinterpret_cast<uint4*>(raw[a])[h] = first_piece + a * step < there
                        ? reinterpret_cast<const uint4*>(src + (first_piece + a * step) * 8)[h] : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int a = 0; a < KEPT; ++a)
                look(raw[a]);
            note_most(most);
            __syncthreads();
            const int e = row_exponent(notes.largest[token]);
#pragma unroll 1
            for (int i = first_piece; i < token_pieces; i += step) {
                put_and_note(i, raw[0], e);
#pragma unroll
                for (int a = 0; a + 1 < KEPT; ++a)
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        raw[a][j] = raw[a + 1][j];
            }
            note_row(e);
        } else {
            each_piece([&](int, const T (&raw)[8]) { look(raw); });
            note_most(most);
            __syncthreads();
            const int e = row_exponent(notes.largest[token]);
#pragma unroll 1
            for (int i = first_piece; i < token_pieces; i += step) {
                __align__(16) T raw[8];
                read_eight(x_row, (c0 * 16 + i) * 8, p.k, raw);
                put_and_note(i, raw, e);
            }
            note_row(e);
        }
        __syncthreads();
    } else {
        uint32_t most_two = 0, least_two = 0xffffffffu;
        each_piece([&](int i, const T (&raw)[8]) {
            put(i, raw, AT_FIRST);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t two = reinterpret_cast<const uint32_t*>(raw)[j] & 0x7fff7fffu;
                most_two = __vmaxu2(most_two, two);
                least_two = __viaddmin_u16x2(two, 0xffffffffu, least_two);
            }
        });
        const bool odd = max(most_two >> 16, most_two & 0xffffu) >= ROW_MOST << 7 || min(least_two >> 16, least_two & 0xffffu) < (ROW_LEAST << 7) - 1;
        if (odd)
            atomicOr(&notes.odd, 1u << token);
        if (__builtin_expect(__syncthreads_or(odd), false))
            put_rows_again(p, xs, notes, token0, c0, token_pieces);
    }

    // ---- the stream
    const int r = lane >> 2, c = lane & 3;
    const uint32_t code_at = (uint32_t)packed_word_at(r, c);
    uint32_t x_lane[NT];
    float down[NT][2];                           // undo the rows' factors and the codes'
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        x_lane[t] = (uint32_t)min(t * 8 + r, tokens - 1) * 64 + c * 16;
#pragma unroll
        for (int j = 0; j < 2; ++j)
            down[t][j] = power_of_two(PACKED_HALF_EXPONENT - notes.exponent[min(t * 8 + 2 * c + j, tokens - 1)]);
    }
    const uint32_t lossy = notes.lossy;
    const uint32_t x_block = (uint32_t)p.tokens * 64;
    bool dead = false;                           // a wait ran out: nothing more is asked for
    int slot = 0;
    uint32_t phase = 0;

    for (int first = 0; first < my_rounds; first += p.batch) {
        const int now = min(p.batch, my_rounds - first);
        for (int u = 0; u < now; ++u) {
            float acc[2][NT][4];
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int t = 0; t < NT; ++t)
                    acc[h][t][0] = acc[h][t][1] = acc[h][t][2] = acc[h][t][3] = 0.f;
            int todo = first + u < warp_rounds ? w1 - w0 : 0;
            const uint8_t* x_at = xs + (w0 - c0) * 4 * x_block;
            while (todo > 0) {
                if (open > 0) {
                    dead = !mbar_wait_warp(&full[slot], phase, p.error, 41) || dead;
                    --open;
                }
                const uint8_t* rec = ring + slot * stage + code_at;
                const uint8_t* rec_scales = ring + slot * stage + PACKED_CODE_BYTES + r * 8;
                const int here = min(todo, p.run);
                todo -= here;
                for (int j = 0; j < here; ++j, rec += RECORD, rec_scales += RECORD, x_at += 4 * x_block) {
                    __align__(16) uint32_t w[4][4];          // rows r, r + 8, r + 16, r + 24
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        *reinterpret_cast<uint4*>(w[i]) = *reinterpret_cast<const uint4*>(rec + i * 512);
#pragma unroll
                    for (int g = 0; g < GROUPS; ++g) {
                        const uint2 s = *reinterpret_cast<const uint2*>(rec_scales + g * 64);
                        float d[2][NT][4];
#pragma unroll
                        for (int i = 0; i < GROUP_BLOCKS; ++i) {
                            const int b = g * GROUP_BLOCKS + i;
                            uint4 f[PARTS][NT];
#pragma unroll
                            for (int part = 0; part < PARTS; ++part)
#pragma unroll
                                for (int t = 0; t < NT; ++t)
                                    f[part][t] = *reinterpret_cast<const uint4*>(x_at + x_lane[t] + b * x_block + part * x_plane);
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                uint32_t q0[4], q1[4];
                                packed_half_pairs(w[2 * h][b], q0);
                                packed_half_pairs(w[2 * h + 1][b], q1);
                                const uint32_t a0[4] = { q0[0], q1[0], q0[1], q1[1] }, a1[4] = { q0[2], q1[2], q0[3], q1[3] };
#pragma unroll
                                for (int part = 0; part < PARTS; ++part)
#pragma unroll
                                    for (int t = 0; t < NT; ++t) {
                                        if (i == 0 && part == 0)
                                            mma_16816<true>(d[h][t], a0, f[part][t].x, f[part][t].y);
                                        else
                                            mma_16816<false>(d[h][t], a0, f[part][t].x, f[part][t].y);
                                        mma_16816<false>(d[h][t], a1, f[part][t].z, f[part][t].w);
                                    }
                            }
                        }
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const uint32_t two = h ? s.y : s.x;
                            const float s0 = __uint_as_float(two << 16), s1 = __uint_as_float(two & 0xffff0000u);
#pragma unroll
                            for (int t = 0; t < NT; ++t) {
                                acc[h][t][0] = fmaf(s0, d[h][t][0], acc[h][t][0]);
                                acc[h][t][1] = fmaf(s0, d[h][t][1], acc[h][t][1]);
                                acc[h][t][2] = fmaf(s1, d[h][t][2], acc[h][t][2]);
                                acc[h][t][3] = fmaf(s1, d[h][t][3], acc[h][t][3]);
                            }
                        }
                    }
                }
                __syncwarp();                    // all lanes have read the stage
                if (!dead && rounds_to_ask > 0) {
                    issue(slot);
                    ++open;
                }
                if (++slot == p.depth) {
                    slot = 0;
                    phase ^= 1;
                }
            }
            float* mine = sums + (u * p.warps + warp) * SUMS + lane;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        mine[((h * NT + t) * 4 + e) * 32] = acc[h][t][e] * down[t][e & 1];
        }
        if (__builtin_expect(lossy != 0, false)) {
            __syncwarp();
            for (int u = 0; u < min(now, warp_rounds - first); ++u)
                add_what_was_lost<X32, NT>(p, lossy, token0, (cluster + (first + u) * p.clusters) * blocks_per_unit + wr, w0, w1,
                                           GROUP_BLOCKS * 32, notes, sums + (u * p.warps + warp) * SUMS);
        }

        // ---- the cluster adds up what its warps have
        __syncthreads();
        if (splits > 1) {
            // a CTA's warps first, in place: another CTA's shared memory is far
            for (int i = threadIdx.x; i < now * blocks_per_unit * SUMS && along_k > 1; i += blockDim.x) {
                float* to = sums + (i / SUMS) * along_k * SUMS + i % SUMS;
                float v = to[0];
#pragma unroll 4
                for (int w = 1; w < along_k; ++w)
                    v += to[w * SUMS];
                to[0] = v;
            }
            __syncwarp();
            cluster_sync();
        }
        const int rows_out = p.pair ? PACKED_ROWS / 2 : PACKED_ROWS;
        const int outputs = now * blocks_per_unit * rows_out * tokens;
        for (int e = rank * blockDim.x + threadIdx.x; e < outputs; e += splits * blockDim.x) {
            const int row = e & (rows_out - 1), rest = e >> (p.pair ? 4 : 5);
            const int block = rest / tokens, token = rest - block * tokens;          // block: of the batch, unit by unit
            const int u = block >> unit_shift, b = block & (blocks_per_unit - 1);
            const int at = ((cluster + (first + u) * p.clusters) * blocks_per_unit + b) * rows_out + row;
            if (at >= p.n)
                continue;
            // the fragment's place of (row of the record, token); a pair's up lies two registers behind its gate
            const int in_record = p.pair ? (row >> 3) * 16 + (row & 7) : row;
            const int reg = ((in_record >> 4) * NT + (token >> 3)) * 4 + ((in_record >> 3) & 1) * 2 + (token & 1);
            const float* place = sums + (u * p.warps + b * along_k) * SUMS + reg * 32 + (in_record & 7) * 4 + (token & 7) / 2;
            float v = 0.f, up = 0.f;
            if (splits > 1) {
                const uint32_t from = smem_addr(place);
                for (int s = 0; s < splits; ++s) {
                    v += peer_shared_f32(from, s);
                    if (p.pair)
                        up += peer_shared_f32(from + 256, s);
                }
            } else {
#pragma unroll 4
                for (int w = 0; w < along_k; ++w) {
                    v += place[w * SUMS];
                    if (p.pair)
                        up += place[w * SUMS + 64];
                }
            }
            if (p.pair)
                v = (p.out_type == CHIBI_F32 ? packed_activate<false>(v, p.act) : packed_activate<true>(v, p.act)) * up;
            const long long m = token0 + token;
            if (p.residual)
                v += p.residual[m * p.residual_stride + at];
            if (p.out_type == CHIBI_F32)
                static_cast<float*>(p.out)[m * p.out_stride + at] = v;
            else
                static_cast<__nv_bfloat16*>(p.out)[m * p.out_stride + at] = from_f32<__nv_bfloat16>(v);
        }
        __syncwarp();
        if (splits > 1)
            cluster_sync();                      // nobody leaves, or writes new sums, while another reads
        else if (first + p.batch < my_rounds)
            __syncthreads();
    }
}

template <int NT, bool X32>
void (*few_rows_kernel_of(int group))(const CUtensorMap, const FewRows)
{
    return group == 32 ? packed_few_rows_kernel<NT, X32, 1>
                       : (group == 64 ? packed_few_rows_kernel<NT, X32, 2> : packed_few_rows_kernel<NT, X32, 4>);
}

constexpr size_t FEW_SMEM_LIMIT = 226 * 1024;        // (a timeline build has a word of its own)

size_t few_rows_smem(bool x32, int group, int chunks, int warps, int splits, int batch, int depth, int run, int tokens)
{
    const size_t x_plane = (size_t)((chunks + splits - 1) / splits) * 4 * tokens * 64;
    return (size_t)warps * depth * ((run * packed_record_bytes(group) + 127) / 128 * 128) + (x32 ? 2 : 1) * x_plane
        + (size_t)batch * warps * 256 * (tokens <= 8 ? 1 : 2) * 4 + sizeof(RowNotes) + warps * depth * 8;
}

void (*few_rows_kernel(bool x32, int tokens, int group))(const CUtensorMap, const FewRows)
{
    return x32 ? (tokens <= 8 ? few_rows_kernel_of<1, true>(group) : few_rows_kernel_of<2, true>(group))
               : (tokens <= 8 ? few_rows_kernel_of<1, false>(group) : few_rows_kernel_of<2, false>(group));
}

// As many blocks as run at once, which go over the records together.
dim3 pack_grid(long long records, int on_an_sm)
{
    const long long most = (long long)on_an_sm * device_sm_count();
    return dim3((unsigned)(records < most ? records : most));
}

} // namespace
} // namespace chibi

using namespace chibi;

// w (and up, with the same shape): a matrix of 32-bit or bfloat16 numbers; out: room for all records.
CHIBI_API int chibi_pack_weights(const void* w, const void* up, int type, int rows, int cols, long long stride, long long up_stride,
                                 int group, void* out, void* stream)
{
    if (!w || !out || rows < 1 || cols < 1 || !packed_group_ok(group))
        return CHIBI_ERR_ARGUMENT;
    const PackSource src { { w, up }, { stride, up_stride }, rows, cols, up ? 1 : 0 };
    const int each = up ? PACKED_ROWS / 2 : PACKED_ROWS;
    const int row_blocks = (rows + each - 1) / each, col_blocks = (cols + PACKED_COLS - 1) / PACKED_COLS;
    const long long records = (long long)row_blocks * col_blocks;
    if (records > 0x3fffffff)
        return CHIBI_ERR_UNSUPPORTED;
    CHIBI_DISPATCH_TYPE(type, T, launch(pack_kernel<T>, pack_grid(records, 8), dim3(128), 0,
                                        (cudaStream_t)stream, src, row_blocks, col_blocks, group, (uint8_t*)out));
    return launch_status();
}

CHIBI_API int chibi_pack_codes(const void* codes, const void* scales, const void* up_codes, const void* up_scales, int rows, int cols,
                               long long stride, long long scale_stride, long long up_stride, long long up_scale_stride, int group,
                               void* out, void* stream)
{
    if (!codes || !scales || !out || rows < 1 || cols < 1 || !packed_group_ok(group) || !up_codes != !up_scales)
        return CHIBI_ERR_ARGUMENT;
    const CodeSource src { { (const int8_t*)codes, (const int8_t*)up_codes },
                           { (const __nv_bfloat16*)scales, (const __nv_bfloat16*)up_scales },
                           { stride, up_stride }, { scale_stride, up_scale_stride }, rows, cols, up_codes ? 1 : 0 };
    const int each = up_codes ? PACKED_ROWS / 2 : PACKED_ROWS;
    const int row_blocks = (rows + each - 1) / each, col_blocks = (cols + PACKED_COLS - 1) / PACKED_COLS;
    const long long records = (long long)row_blocks * col_blocks;
    if (records > 0x3fffffff)
        return CHIBI_ERR_UNSUPPORTED;
    launch(pack_codes_kernel, pack_grid(records, 4), dim3(512), 0, (cudaStream_t)stream, src, row_blocks,
           col_blocks, group, (uint8_t*)out);
    return launch_status();
}

CHIBI_API int chibi_unpack_weights(const void* data, int rows, int cols, int pair, int group, void* out, int out_type, long long stride,
                                   void* stream)
{
    if (!data || !out || rows < 1 || cols < 1 || !packed_group_ok(group))
        return CHIBI_ERR_ARGUMENT;
    const int each = pair ? PACKED_ROWS / 2 : PACKED_ROWS;
    const int row_blocks = (rows + each - 1) / each, col_blocks = (cols + PACKED_COLS - 1) / PACKED_COLS;
    const long long records = (long long)row_blocks * col_blocks;
    if (records > 0x3fffffff)
        return CHIBI_ERR_UNSUPPORTED;
    CHIBI_DISPATCH_TYPE(out_type, T, launch(unpack_kernel<T>, pack_grid(records, 4), dim3(512), 0,
                                            (cudaStream_t)stream, (const uint8_t*)data, row_blocks, col_blocks, group, rows, cols, pair,
                                            (T*)out, stride));
    return launch_status();
}

// Shared memory of the kernel for few rows under a plan, in KB (rounded up); CudaKernels.packed_plan asks.
CHIBI_API int chibi_packed_few_rows_kb(int x32, int group, int cols, int tokens, int warps, int splits, int batch, int depth, int run)
{
    return (int)((few_rows_smem(x32 != 0, group, (cols + PACKED_COLS - 1) / PACKED_COLS, warps, splits, batch, depth, run, tokens) + 1023)
                 / 1024);
}

// How many clusters of `splits` CTAs with that much shared memory run at once (0: none, or an error).
CHIBI_API int chibi_packed_few_rows_clusters(int x32, int group, int tokens, int warps, int splits, int kb)
{
    if (!packed_group_ok(group) || splits < 1 || splits > 8 || tokens < 1 || tokens > 16 || kb < 1 || kb > 226 || warps < 1 || warps > 16)
        return 0;
    void (*kernel)(const CUtensorMap, const FewRows) = few_rows_kernel(x32 != 0, tokens, group);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)splits);
    cfg.blockDim = dim3((unsigned)warps * 32);
    cfg.dynamicSmemBytes = (size_t)kb * 1024;
    cudaLaunchAttribute attr = {};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)splits;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    int clusters = 0;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)FEW_SMEM_LIMIT) != cudaSuccess
        || cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg) != cudaSuccess) {
        cudaGetLastError();
        return 0;
    }
    return clusters;
}

// Fills in what a call keeps beside its sizes: the tensor map over the records.  `many`: for chibi_packed_many_rows.
CHIBI_API int chibi_packed_prepare(ChibiPackedCall* c, int many)
{
    if (!c || !c->data || c->n < 1 || c->k < 1 || !packed_group_ok(c->group) || (!many && (c->run < 1 || c->run > 256)))
        return CHIBI_ERR_ARGUMENT;
    const int each = c->pair ? PACKED_ROWS / 2 : PACKED_ROWS;
    CUtensorMap map;
    if (!packed_map(c->data, c->group, (c->n + each - 1) / each, (c->k + PACKED_COLS - 1) / PACKED_COLS, many ? 1 : c->run,
                    many ? 128 / PACKED_ROWS : 1, &map))
        return CHIBI_ERR_UNSUPPORTED;
    static_assert(sizeof(map) == sizeof(c->map), "");
    memcpy(c->map, &map, sizeof(map));
    return CHIBI_OK;
}

// out[m, n] = x[m, k] times the matrix (+ residual); pair: act(x gate) * (x up), n features.  The plan: see FewRows.
CHIBI_API int chibi_packed_few_rows(const ChibiPackedCall* c, const void* x, long long x_stride, void* out, long long out_stride,
                                    const void* residual, long long residual_stride, void* stream)
{
    if (!c || !c->data || !x || !out || c->n < 1 || c->k < 1 || c->m < 1 || !packed_group_ok(c->group)
        || (c->x_type != CHIBI_F32 && c->x_type != CHIBI_BF16) || (c->out_type != CHIBI_F32 && c->out_type != CHIBI_BF16)
        || (c->pair && (residual || (c->act != 1 && c->act != 2))))
        return CHIBI_ERR_ARGUMENT;
    const int chunks = (c->k + PACKED_COLS - 1) / PACKED_COLS;
    if ((c->warps != 8 && c->warps != 16) || c->splits < 1 || c->splits > 8 || (c->splits & (c->splits - 1)) || c->splits > chunks
        || c->along_k < 1 || c->along_k > c->warps || (c->along_k & (c->along_k - 1)) || c->batch < 1 || c->depth < 1 || c->run < 1
        || c->run > 256 || chunks > (1 << 27) || c->tokens < 1 || c->tokens > c->warps || c->clusters < 1)
        return CHIBI_ERR_ARGUMENT;
    const bool x32 = c->x_type == CHIBI_F32;
    const size_t smem = few_rows_smem(x32, c->group, chunks, c->warps, c->splits, c->batch, c->depth, c->run, c->tokens);
    const int each = c->pair ? PACKED_ROWS / 2 : PACKED_ROWS, row_blocks = (c->n + each - 1) / each;
    if (smem > FEW_SMEM_LIMIT)
        return CHIBI_ERR_UNSUPPORTED;
    CUtensorMap map;
    memcpy(&map, c->map, sizeof(map));
    int split_shift = 0, along_shift = 0;
    while ((1 << split_shift) < c->splits)
        ++split_shift;
    while ((1 << along_shift) < c->along_k)
        ++along_shift;
    const int per_unit = c->warps >> along_shift;
    FewRows p { row_blocks, chunks, c->n, c->k, c->pair, x, x_stride, c->m, out, c->out_type, out_stride, (const float*)residual,
                residual_stride, c->act, c->warps, split_shift, along_shift, c->batch, c->depth, c->run, c->tokens, c->clusters,
                (row_blocks + per_unit - 1) / per_unit, (int*)c->error,
                static_cast<const uint8_t*>(c->data) };
    void (*kernel)(const CUtensorMap, const FewRows) = few_rows_kernel(x32, c->tokens, c->group);
    static std::atomic<unsigned long long> allowed[2][2][3];
    const cudaError_t e = packed_allow_shared(kernel, allowed[x32][c->tokens <= 8][c->group / 64], FEW_SMEM_LIMIT);
    if (e != cudaSuccess)
        return (int)e;
    const dim3 block((unsigned)c->warps * 32);
    // (a grid's second axis has 65,535 places: rows of x beyond that many blocks of them are launches of their own)
    const long long at_once = 65535ll * c->tokens;
    for (long long first = 0; first < c->m; first += at_once) {
        p.m = (int)(c->m - first < at_once ? c->m - first : at_once);
        p.x = static_cast<const char*>(x) + first * x_stride * (x32 ? 4 : 2);
        p.out = static_cast<char*>(out) + first * out_stride * (c->out_type == CHIBI_F32 ? 4 : 2);
        p.residual = residual ? static_cast<const float*>(residual) + first * residual_stride : nullptr;
        const dim3 grid((unsigned)(c->clusters * c->splits), (unsigned)((p.m + c->tokens - 1) / c->tokens));
        if (c->splits > 1)
            launch_cluster_x(kernel, grid, block, smem, (cudaStream_t)stream, c->splits, map, p);
        else
            launch(kernel, grid, block, smem, (cudaStream_t)stream, map, p);
    }
    return launch_status();
}
