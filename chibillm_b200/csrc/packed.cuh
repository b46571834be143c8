// Matrices held in 4 bits: how they lie in memory.
//
// A value is q * s: q a whole number of -8 ... 7, s a bfloat16 that the `group` neighbouring columns of a row share
// (32, 64 or 128; the last group of a row may be shorter).  q has at most 4 significant bits, so it is a bfloat16 or
// float16 without rounding: the tensor cores make exact products q * x, and a group's 32-bit sum is multiplied by s once.
//
// The matrix is cut into records of 32 rows x 128 columns, [block of rows][block of columns][record], rows and columns
// beyond the matrix filled with zeros.  A record is one run of bytes, so that a bulk copy brings codes and scales at once:
//   2,048 bytes of codes, first those of rows 0 ... 15, then of rows 16 ... 31: a row has 64 bytes, four pieces of 16, piece c
//     at place c ^ (row / 2 % 4).  Piece c holds four words, word b the columns 32 b + 8 c + 0 ... 7: what the lanes with
//     lane % 4 == c need for the two 16-column steps of `mma.m16n8k16` over columns 32 b ... 32 b + 31 (which column of A
//     meets which row of B is free, as long as both agree).  In a word, nibbles j and j + 4 hold q + 8 of columns 2 j and
//     2 j + 1, so that (word >> 4 j) & 0x000f000f has them in the two halves.  The places' order lets eight lanes that read
//     pieces of two rows, and eight that read the same piece of eight rows, meet all 32 banks once.
//   64 bytes of scales for each group: those of rows r, r + 8, r + 16 and r + 24 side by side.
// A pair of matrices (gate and up, features x columns each) is one matrix of which each 16 rows are 8 rows of gate and the
// same 8 of up: a lane's two rows of `mma.m16n8k16` are then a feature's gate and its up.
#pragma once
#include "common.cuh"
#include "tensor_map.cuh"

#include <atomic>

// What stays the same from call to call of a product with such a matrix: made once for a number of rows and the types
// (library.py has the same fields).
struct ChibiPackedCall {
    const void* data;
    void* error;
    int group, n, k, pair;           // n: rows of the matrix, of a pair its features
    int m, x_type, out_type, act;    // act (pairs): 1 gelu with tanh, 2 silu
    int splits, clusters, tokens;    // both kernels
    int warps, along_k, batch, depth, run;         // few rows
    int rounds;                      // many rows
    unsigned long long map[16];      // the tensor map over the records (chibi_packed_prepare)
};

namespace chibi {

constexpr int PACKED_ROWS = 32, PACKED_COLS = 128, PACKED_CODE_BYTES = PACKED_ROWS * PACKED_COLS / 2;

__host__ __device__ constexpr int packed_record_bytes(int group) { return PACKED_CODE_BYTES + PACKED_COLS / group * PACKED_ROWS * 2; }
__host__ __device__ constexpr bool packed_group_ok(int group) { return group == 32 || group == 64 || group == 128; }

// Where in a record the word of row r for columns 8 seg ... 8 seg + 7 lies, in bytes.
__host__ __device__ constexpr int packed_word_at(int r, int seg)
{
    return r * 64 + (((seg & 3) ^ ((r >> 1) & 3)) << 4) + (seg >> 2) * 4;
}
// Where the scale of row r in group g of a record lies.
__host__ __device__ constexpr int packed_scale_at(int r, int g) { return PACKED_CODE_BYTES + g * 64 + (r & 7) * 8 + (r >> 3) * 2; }

// Which matrix of a pair, and which of its rows, row r of block rb is (of a single matrix: the first, and its row).
__host__ __device__ constexpr int packed_side(int pair, int r) { return pair ? (r >> 3) & 1 : 0; }
__host__ __device__ constexpr int packed_source_row(int pair, int rb, int r)
{
    return pair ? rb * (PACKED_ROWS / 2) + (r >> 4) * 8 + (r & 7) : rb * PACKED_ROWS + r;
}

// Lets `kernel` have so much shared memory; asked of each device once.
template <typename K> inline cudaError_t packed_allow_shared(K kernel, std::atomic<unsigned long long>& allowed, size_t bytes)
{
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess)
        return e;
    const unsigned long long bit = 1ull << (device & 63);
    if (device < 64 && (allowed.load(std::memory_order_relaxed) & bit))
        return cudaSuccess;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e == cudaSuccess)
        allowed.fetch_or(bit, std::memory_order_relaxed);
    else
        cudaGetLastError();
    return e;
}

// A tensor map over the records: a box is `box_cols` neighbouring records of each of `box_rows` blocks of rows, and lands record
// by record.  (An untiled bulk copy of a record or two is simpler and slower: 17 bytes a cycle and SM.)  A record is two runs of
// 8-byte elements, since a box has at most 256 in a row.
inline bool packed_map(const void* data, int group, int row_blocks, int col_blocks, int box_cols, int box_rows, CUtensorMap* out)
{
    EncodeTiledFn fn = encode_tiled();
    if (!fn)
        return false;
    const cuuint64_t record = (cuuint64_t)packed_record_bytes(group);
    const cuuint64_t dims[4] = { record / 16, 2, (cuuint64_t)col_blocks, (cuuint64_t)row_blocks };
    const cuuint64_t strides[3] = { record / 2, record, record * (cuuint64_t)col_blocks };
    const cuuint32_t box[4] = { (cuuint32_t)(record / 16), 2, (cuuint32_t)box_cols, (cuuint32_t)box_rows };
    const cuuint32_t elem[4] = { 1, 1, 1, 1 };
    return fn(out, CU_TENSOR_MAP_DATA_TYPE_FLOAT64, 4, const_cast<void*>(data), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// The whole numbers of a word as float16, columns 2 j and 2 j + 1 in pair j (exact: 1,024 + code and 1,024 + 16 code have
// the code in float16's ten bits of mantissa, and what is taken off leaves a small whole number).
__device__ __forceinline__ void packed_half_pairs(uint32_t word, uint32_t (&pair)[4])
{
    const uint32_t next = word >> 8;
    asm("lop3.b32 %0, %1, 0x000f000f, 0x64006400, 0xea;" : "=r"(pair[0]) : "r"(word));
    asm("lop3.b32 %0, %1, 0x00f000f0, 0x64006400, 0xea;" : "=r"(pair[1]) : "r"(word));
    asm("lop3.b32 %0, %1, 0x000f000f, 0x64006400, 0xea;" : "=r"(pair[2]) : "r"(next));
    asm("lop3.b32 %0, %1, 0x00f000f0, 0x64006400, 0xea;" : "=r"(pair[3]) : "r"(next));
    asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(pair[0]) : "r"(0x64086408u));                       // - 1,032
    asm("fma.rn.f16x2 %0, %0, %1, %2;" : "+r"(pair[1]) : "r"(0x2c002c00u), "r"(0xd480d480u)); // / 16 - 72
    asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(pair[2]) : "r"(0x64086408u));
    asm("fma.rn.f16x2 %0, %0, %1, %2;" : "+r"(pair[3]) : "r"(0x2c002c00u), "r"(0xd480d480u));
}

// The same as bfloat16, times 2^-10 (2^-3 + 2^-10 code has its code in the lowest of bfloat16's seven bits of mantissa).  A group's
// sum over 128 finite bfloat16 numbers is below 2^138, times 2^-10 within 32 bits; PACKED_BF16_UNDO brings it back.  (Sums of x below
// 2^-120 come into the range where 32-bit numbers have fewer bits.)
constexpr float PACKED_BF16_UNDO = 1024.f;
template <int J> __device__ __forceinline__ uint32_t packed_bf16_pair(uint32_t word)
{
    uint32_t r;
    asm("lop3.b32 %0, %1, 0x000f000f, 0x3e003e00, 0xea;" : "=r"(r) : "r"(word >> (4 * J)));
    asm("sub.rn.bf16x2 %0, %0, %1;" : "+r"(r) : "r"(0x3e083e08u));                           // - 136 * 2^-10
    return r;
}

// The gate's activation, silu (2) or gelu with tanh (1): both are z / (1 + exp(-y)), y = z or 2 sqrt(2 / pi) (z + 0.044715 z^3),
// since (1 + tanh(u)) / 2 = 1 / (1 + exp(-2 u)); no difference of near numbers where tanh is close to -1.  (Short: a kernel that
// applies it to every accumulator column has it dozens of times, and with tanhf and erff beside it ran out of instruction cache,
// 285 us instead of 133 for 2,048 rows of a 2 x 6,144 x 2,048 pair.)
template <bool ROUNDED> __device__ __forceinline__ float packed_activate(float z, int act)
{
    const float y = act == 2 ? z : 1.5957691216057308f * fmaf(0.044715f * z * z, z, z);
    return ROUNDED ? __fdividef(z, 1.f + __expf(-y)) : z / (1.f + expf(-y));
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

// Products of rows of the matrix with rows of x, by a warp each and in 64 bits: for sums that came out as no number although every
// number of x is one (a group's sum, or its product with a scale, can pass 2^128 where the whole does not: weights from 10^32 on,
// x from 10^35 on).  Terms are exact (4, 8 and 24 bits).  The whole warp calls; a lane that asks has the block of rows, the row in
// its records and the row of x, and gets the sum instead of v.  Slow, 6 us for 4,096 columns (less where a NaN ends it).
template <typename T>
__device__ __forceinline__ float packed_sums_in_64_bits(const uint8_t* data, int group, int chunks, int k, bool asks, int block, int r,
                                                        const T* x, float v)
{
    const int lane = threadIdx.x & 31;
#pragma unroll 1
    for (uint32_t todo = __ballot_sync(0xffffffffu, asks); todo != 0; todo &= todo - 1) {
        const int who = __ffs(todo) - 1;
        const int row = __shfl_sync(0xffffffffu, r, who);
        const uint8_t* rec = data + (long long)__shfl_sync(0xffffffffu, block, who) * chunks * packed_record_bytes(group);
        const T* from = reinterpret_cast<const T*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(x), who));
        double sum = 0.;
#pragma unroll 1
        for (int col = lane * 8; __any_sync(0xffffffffu, col < k); col += 256) {
            if (col < k) {
                __align__(16) T eight[8];
                read_eight(from, col, k, eight);
                const uint8_t* at = rec + (long long)(col / PACKED_COLS) * packed_record_bytes(group);
                const uint32_t word = *reinterpret_cast<const uint32_t*>(at + packed_word_at(row, col % PACKED_COLS >> 3));
                double part = 0.;
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    part = fma((double)((int)((word >> (4 * (i / 2) + 16 * (i & 1))) & 15u) - 8), (double)to_f32(eight[i]), part);
                sum = fma((double)to_f32(*reinterpret_cast<const __nv_bfloat16*>(at + packed_scale_at(row, col % PACKED_COLS / group))), part, sum);
            }
            if (__any_sync(0xffffffffu, sum != sum))
                break;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
            sum += __shfl_xor_sync(0xffffffffu, sum, o);
        v = lane == who ? (float)sum : v;
    }
    return v;
}

} // namespace chibi
