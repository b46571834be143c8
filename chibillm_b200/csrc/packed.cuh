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

// The whole numbers of a word as float16, columns 2 j and 2 j + 1 in pair j, times 2^-14 (exact: 2^-4 + 2^-14 code and 2^-4 + 2^-10 code
// have the code in float16's ten bits of mantissa, a way that open 4-bit kernels share; what is taken off leaves a small number).
// x is held at 2^15 at most, so a group's sum is below 2^11 and its product with a scale finite for scales below 2^117, weights of
// 10^36; for weights below 10^-35 it comes into the range where 32-bit numbers have fewer bits.  PACKED_HALF_EXPONENT undoes it.
constexpr int PACKED_HALF_EXPONENT = 14;
__device__ __forceinline__ void packed_half_pairs(uint32_t word, uint32_t (&pair)[4])
{
    const uint32_t next = word >> 8;
    asm("lop3.b32 %0, %1, 0x000f000f, 0x2c002c00, 0xea;" : "=r"(pair[0]) : "r"(word));
    asm("lop3.b32 %0, %1, 0x00f000f0, 0x2c002c00, 0xea;" : "=r"(pair[1]) : "r"(word));
    asm("lop3.b32 %0, %1, 0x000f000f, 0x2c002c00, 0xea;" : "=r"(pair[2]) : "r"(next));
    asm("lop3.b32 %0, %1, 0x00f000f0, 0x2c002c00, 0xea;" : "=r"(pair[3]) : "r"(next));
    asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(pair[0]) : "r"(0x2c082c08u));                       // - 1,032 * 2^-14
    asm("fma.rn.f16x2 %0, %0, %1, %2;" : "+r"(pair[1]) : "r"(0x2c002c00u), "r"(0x9c809c80u)); // / 16 - 72 * 2^-14
    asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(pair[2]) : "r"(0x2c082c08u));
    asm("fma.rn.f16x2 %0, %0, %1, %2;" : "+r"(pair[3]) : "r"(0x2c002c00u), "r"(0x9c809c80u));
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

} // namespace chibi
