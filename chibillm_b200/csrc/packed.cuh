// Matrices held in 4 bits: how they lie in memory.
//
// A value is q * s: q a whole number of -8 ... 7, s a bfloat16 that the `group` neighbouring columns of a row share
// (32, 64 or 128; the last group of a row may be shorter).  q has at most 4 significant bits, so it is a bfloat16
// without rounding: the tensor cores make exact products q * x, and a group's 32-bit sum is multiplied by s once.
//
// The matrix is cut into records of 16 rows x 128 columns, [block of rows][block of columns][record], rows and columns
// beyond the matrix filled with zeros.  A record is one run of bytes, so that a bulk copy brings codes and scales at once:
//   1,024 bytes of codes: row r has 64 bytes, four pieces of 16, piece c at place c ^ (r / 2 % 4).  Piece c holds four
//     words, word b the columns 32 b + 8 c + 0 ... 7: what the lanes with lane % 4 == c need for the two 16-column steps
//     of `mma.m16n8k16` over columns 32 b ... 32 b + 31 (which column of A meets which row of B is free, as long as both
//     agree).  In a word, nibbles j and j + 4 hold q + 8 of columns 2 j and 2 j + 1, so that (word >> 4 j) & 0x000f000f has
//     them in the two halves.  The places' order lets eight lanes that read pieces of two rows, and eight that read the
//     same piece of eight rows, meet all 32 banks once.
//   32 bytes of scales for each group: those of rows r and r + 8 side by side.
// A pair of matrices (gate and up, features x columns each) is one matrix whose blocks of 16 rows are 8 rows of gate and
// the same 8 of up: a lane's two rows of `mma.m16n8k16` are then a feature's gate and its up.
#pragma once
#include "common.cuh"

namespace chibi {

constexpr int PACKED_ROWS = 16, PACKED_COLS = 128, PACKED_CODE_BYTES = PACKED_ROWS * PACKED_COLS / 2;

__host__ __device__ constexpr int packed_record_bytes(int group) { return PACKED_CODE_BYTES + PACKED_COLS / group * 32; }
__host__ __device__ constexpr bool packed_group_ok(int group) { return group == 32 || group == 64 || group == 128; }

// Where in a record the word of row r for columns 8 seg ... 8 seg + 7 lies, in bytes.
__host__ __device__ constexpr int packed_word_at(int r, int seg)
{
    return r * 64 + (((seg & 3) ^ ((r >> 1) & 3)) << 4) + (seg >> 2) * 4;
}
// Where the scale of row r in group g of a record lies.
__host__ __device__ constexpr int packed_scale_at(int r, int g) { return PACKED_CODE_BYTES + g * 32 + ((r & 7) * 2 + (r >> 3)) * 2; }

// The whole numbers of columns 2 j and 2 j + 1 of a word as two bfloat16 (exact: 128 + code has its codes in the lowest
// bits of bfloat16, and the difference to 136 is exact).
template <int J> __device__ __forceinline__ uint32_t packed_pair(uint32_t word)
{
    uint32_t r;
    asm("lop3.b32 %0, %1, 0x000f000f, 0x43004300, 0xea;" : "=r"(r) : "r"(word >> (4 * J)));
    asm("sub.rn.bf16x2 %0, %0, %1;" : "+r"(r) : "r"(0x43084308u));
    return r;
}

} // namespace chibi
