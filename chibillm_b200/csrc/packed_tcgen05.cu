// The product of many bfloat16 rows of x with a matrix held in 4 bits (packed.cuh), on tcgen05.
//
//   out[m][n] = sum over groups of s[n][g] * (sum over the group of q[n][k] x[m][k])
//
// The matrix's 128 rows of a tile are the instruction's rows, TOKENS rows of x its columns.  Warps that do nothing else turn
// codes into bfloat16 whole numbers (exact) and write them to TMEM, where they are the A operand: shared memory carries only
// the rows of x and the codes themselves.  Each group's sum is an accumulator of its own in TMEM; three warpgroups read it, each
// a third of the columns, and add it times the row's scale to sums in registers.  So nothing is rounded but 32-bit sums, and a
// lane's row has one scale for all of its columns.  (The whole numbers are held times 2^-10, so that the sums of finite x are
// finite; a CTA's sums are multiplied by 2^10 in the end.  They are infinite where they pass 2^128, or a group's part of them
// 2^138.)  A thread's sums are an output column of 32 lanes: stores are whole
// lines without a detour.
//
// What bounds it: an instruction of 128 x TOKENS x 16 with its A operand in TMEM takes 118 cycles at 64 as at 128 columns, so tiles
// are 192 tokens wide, the most that leaves room in TMEM for two accumulators and two operands (two of 192 columns, two of 64).
// A group costs some 200 cycles beside its instructions, and as much again while the adding warps multiply and add.  Measured (replayed in a
// graph): 1,999 rows of 6,144 x 4,096 in groups of 128 87 us (1,150 TFLOP/s), 64 113, 32 191; 2,048 of a gated pair of 2 x 6,144 x 2,048,
// groups of 64, 131, of which 25 go by while the sums are activated and written; 64 rows of a pair of 2 x 12,288 x 4,096 31.
//
// A CTA stays on its SM and takes tiles in turn.  What is left after whole rounds of tiles (all of them, if they are few) is shared
// out: `splits` CTAs of a cluster share a tile's columns; their sums go to shared memory and each CTA adds up a share of them,
// CTA by CTA in one order.
#define CHIBI_UNIT packed_tcgen05
#define CHIBI_UNIT_ID 20
#include "packed.cuh"
#include "sm100.cuh"
#include "split_f32.cuh"
#include "tensor_map.cuh"

#include <string.h>

namespace chibi {
namespace {

constexpr int PT_ADDERS = 12;                    // warps
constexpr int PT_THREADS = (4 + 4 + PT_ADDERS) * 32;             // codes' loader, issuer, x's loader, an idle warp | converting | adding
constexpr int PT_ROWS = 128;
constexpr int PT_SCALE_SLOTS = 8;                // blocks of columns whose scales are kept

template <int TOKENS, int GROUP_BLOCKS> struct PackedTile {
    static constexpr int GROUPS = 4 / GROUP_BLOCKS;
    static constexpr int RECORD = PACKED_CODE_BYTES + GROUPS * 64;
    static constexpr int X_BYTES = TOKENS * PACKED_COLS * 2, X_STAGES = TOKENS > 96 ? 3 : TOKENS > 48 ? 4 : 6;
    static constexpr int CODE_BYTES = PT_ROWS / PACKED_ROWS * RECORD, CODE_STAGES = TOKENS > 96 ? 4 : 6;
    static_assert(CODE_BYTES % 128 == 0 && X_BYTES % 2048 == 0, "a tile copy's place");
    static constexpr int SCALES = PT_SCALE_SLOTS * GROUPS * PT_ROWS * 4;
    // accumulators (one for each group on its way) and operand blocks in TMEM's 512 columns
    static constexpr int SUMS = TOKENS > 96 ? 2 : TOKENS > 48 ? 3 : 4, OPERANDS = SUMS;
    static_assert(SUMS * TOKENS + OPERANDS * 64 <= 512, "");
    // Block i's scales go where block i - 8's were.  Its operand's place is free when the products of block i - OPERANDS are
    // done, which began when all groups but the last SUMS up to there had been added up: those of block i - 8 among them.
    static_assert(SUMS <= (PT_SCALE_SLOTS - OPERANDS) * GROUPS, "");
    static constexpr size_t SMEM = 1024 + X_STAGES * X_BYTES + CODE_STAGES * CODE_BYTES + SCALES
        + 2 * (X_STAGES + CODE_STAGES + OPERANDS + SUMS) * 8 + 16;
    static_assert(X_STAGES * X_BYTES >= TOKENS * PT_ROWS * 4, "a tile's sums fit where x was");
    static_assert(SMEM <= 226 * 1024, "");
};

struct PackedProduct {
    int chunks;                                  // blocks of 128 columns
    int n, pair;
    int m;
    void* out;
    int out_type;
    long long out_stride;
    const float* residual;
    long long residual_stride;
    int act;                                     // pairs: 1 gelu with tanh, 2 silu
    int rounds, splits, tiles, token_tiles;      // see piece()
    int* error;
};

__device__ __forceinline__ void peer_shared_f32x4(uint32_t own_smem_addr, uint32_t rank, float (&v)[4])
{
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3])
                 : "r"(sm100::peer_smem_addr(own_smem_addr, rank))
                 : "memory");
}

// An adding warp's columns of a tile: lane l has row l of a record, two neighbouring tokens to a pair.
template <int COLS, typename OUT>
__device__ __forceinline__ void write_columns(const PackedProduct& p, const uint64_t (&acc)[COLS / 2], int token0, int left, int n_tile,
                                              int quarter, int lane)
{
    OUT* out = static_cast<OUT*>(p.out) + (long long)token0 * p.out_stride;
    const long long step = p.out_stride;
    if (p.pair) {
        // lanes l and l ^ 8 hold a feature's gate and up: one makes the even tokens, the other the odd ones
        const bool is_up = lane & 8;
        const int at = n_tile * (PT_ROWS / 2) + quarter * 16 + (lane >> 4) * 8 + (lane & 7);
        out += at + (is_up ? step : 0);
        left = at < p.n ? left - (is_up ? 1 : 0) : 0;
#pragma unroll
        for (int j = 0; j < COLS / 2; ++j) {
            const float2 v = halves_of(acc[j]);
            const float other = __shfl_xor_sync(0xffffffffu, is_up ? v.x : v.y, 8);
            const float gate = is_up ? other : v.x, up = is_up ? v.y : other;
            if (2 * j < left)
                *out = from_f32<OUT>(packed_activate<sizeof(OUT) == 2>(gate, p.act) * up);
            out += 2 * step;
        }
        return;
    }
    const int at = n_tile * PT_ROWS + quarter * 32 + lane;
    if (at >= p.n)
        return;
    out += at;
    const float* residual = p.residual ? p.residual + (long long)token0 * p.residual_stride + at : nullptr;
#pragma unroll
    for (int j0 = 0; j0 < COLS; j0 += 8) {
        float r[8] = {};
        if (residual) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (j0 + j < left)
                    r[j] = residual[(long long)(j0 + j) * p.residual_stride];
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float2 v = halves_of(acc[(j0 + j) / 2]);
            if (j0 + j < left)
                *out = from_f32<OUT>((j & 1 ? v.y : v.x) + r[j]);
            out += step;
        }
    }
}

template <int TOKENS, int GROUP_BLOCKS>
__global__ void __launch_bounds__(PT_THREADS, 1) packed_many_rows_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const PackedProduct p)
{
    using namespace sm100;
    using T = PackedTile<TOKENS, GROUP_BLOCKS>;
    constexpr int GROUPS = T::GROUPS, RECORD = T::RECORD, X_STAGES = T::X_STAGES, CODE_STAGES = T::CODE_STAGES;
    constexpr int OPERANDS = T::OPERANDS, SUMS = T::SUMS;
    constexpr int COLS = TOKENS / (PT_ADDERS / 4);           // of an adding warpgroup
    pdl_trigger();
    extern __shared__ uint8_t smem_raw[];
    uint8_t* xs = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* codes = xs + X_STAGES * T::X_BYTES;
    float* scales = reinterpret_cast<float*>(codes + CODE_STAGES * T::CODE_BYTES);        // [slot][group][row]
    uint64_t* x_full = reinterpret_cast<uint64_t*>(scales + T::SCALES / 4);
    uint64_t* x_empty = x_full + X_STAGES;
    uint64_t* codes_full = x_empty + X_STAGES;
    uint64_t* codes_empty = codes_full + CODE_STAGES;
    uint64_t* operand_full = codes_empty + CODE_STAGES;
    uint64_t* operand_empty = operand_full + OPERANDS;
    uint64_t* sums_full = operand_empty + OPERANDS;
    uint64_t* sums_empty = sums_full + SUMS;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sums_empty + SUMS);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = p.splits > 1 ? (int)cluster_cta_rank() : 0;
    // A CTA's r-th piece of work, blocks c0 ... c1 of a tile: `rounds` whole tiles, then, in clusters, its share of one more.
    struct Piece {
        int tile, c0, c1;
    };
    auto piece = [&](int r, Piece& out) -> bool {
        out = { (int)(blockIdx.x + r * gridDim.x), 0, p.chunks };
        if (r == p.rounds)
            out = { (int)(p.rounds * gridDim.x + blockIdx.x / p.splits), p.chunks * rank / p.splits, p.chunks * (rank + 1) / p.splits };
        return out.tile < p.tiles && (r < p.rounds || (r == p.rounds && p.splits > 1));
    };

    if (threadIdx.x == 0) {
        for (int s = 0; s < X_STAGES; ++s) {
            mbar_init(&x_full[s], 1);
            mbar_init(&x_empty[s], 1);
        }
        for (int s = 0; s < CODE_STAGES; ++s) {
            mbar_init(&codes_full[s], 1);
            mbar_init(&codes_empty[s], 4);
        }
        for (int s = 0; s < OPERANDS; ++s) {
            mbar_init(&operand_full[s], 4);
            mbar_init(&operand_empty[s], 1);
        }
        for (int s = 0; s < SUMS; ++s) {
            mbar_init(&sums_full[s], 1);
            mbar_init(&sums_empty[s], PT_ADDERS);
        }
        fence_barrier_init();
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const uint32_t tmem_sums = *tmem_slot, tmem_operands = tmem_sums + SUMS * TOKENS;

    // registers where they are needed: 96 a thread at launch, 5 x 96 = 480 >= 40 + 88 + 3 x 112 a lane of the five warpgroups
    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
        if (warp == 0 && elect_one()) {
            // ---- codes: constant, so they are asked for before the kernel ahead has ended
            tma_prefetch_descriptor(&map_w);
            uint32_t i = 0, s = 0;
            bool ok = true;
            Piece at;
            for (int r = 0; ok && piece(r, at); ++r) {
                const int rb = at.tile / p.token_tiles * (PT_ROWS / PACKED_ROWS);
                for (int chunk = at.c0; chunk < at.c1; ++chunk, ++i) {
                    if (i >= CODE_STAGES && !mbar_wait(&codes_empty[s], (i / CODE_STAGES - 1) & 1, p.error, 42)) {
                        ok = false;
                        break;
                    }
                    mbar_arrive_expect_tx(&codes_full[s], T::CODE_BYTES);
                    tma_load_4d(codes + s * T::CODE_BYTES, &map_w, &codes_full[s], 0, 0, chunk, rb);
                    s = s + 1 == CODE_STAGES ? 0 : s + 1;
                }
            }
            // every copy has landed before this CTA's shared memory is anybody else's
            for (uint32_t j = i > CODE_STAGES ? i - CODE_STAGES : 0; j < i; ++j)
                mbar_wait(&codes_full[j % CODE_STAGES], (j / CODE_STAGES) & 1, p.error, 42);
        } else if (warp == 2 && elect_one()) {
            // ---- rows of x
            tma_prefetch_descriptor(&map_x);
            pdl_wait();
            uint32_t i = 0, s = 0;
            bool ok = true;
            Piece at;
            for (int r = 0; ok && piece(r, at); ++r) {
                const int token0 = at.tile % p.token_tiles * TOKENS;
                for (int chunk = at.c0; chunk < at.c1; ++chunk, ++i) {
                    if (i >= X_STAGES && !mbar_wait(&x_empty[s], (i / X_STAGES - 1) & 1, p.error, 42)) {
                        ok = false;
                        break;
                    }
                    uint8_t* dst = xs + s * T::X_BYTES;
                    mbar_arrive_expect_tx(&x_full[s], T::X_BYTES);
                    tma_load_2d(dst, &map_x, &x_full[s], chunk * PACKED_COLS, token0);
                    tma_load_2d(dst + T::X_BYTES / 2, &map_x, &x_full[s], chunk * PACKED_COLS + 64, token0);
                    s = s + 1 == X_STAGES ? 0 : s + 1;
                }
            }
            for (uint32_t j = i > X_STAGES ? i - X_STAGES : 0; j < i; ++j)
                mbar_wait(&x_full[j % X_STAGES], (j / X_STAGES) & 1, p.error, 42);
        } else if (warp == 1 && elect_one()) {
            constexpr uint32_t idesc = make_idesc_bf16_f32(PT_ROWS, TOKENS);
            constexpr int STEPS = GROUP_BLOCKS * 2;          // 16-column steps of a group
            uint32_t i = 0, a = 0;
            bool ok = true;
            Piece at;
            for (int r = 0; ok && piece(r, at); ++r)
                for (int chunk = at.c0; ok && chunk < at.c1; ++chunk, ++i) {
                    const uint32_t s = i % X_STAGES, o = i % OPERANDS;
                    if (!mbar_wait(&x_full[s], (i / X_STAGES) & 1, p.error, 43) || !mbar_wait(&operand_full[o], (i / OPERANDS) & 1, p.error, 43)) {
                        ok = false;
                        break;
                    }
                    const uint64_t x_desc = make_kmajor_sw128_desc(smem_addr(xs + s * T::X_BYTES));
#pragma unroll
                    for (int g = 0; g < GROUPS; ++g, ++a) {
                        const uint32_t d = a % SUMS;
                        if (a >= SUMS && !mbar_wait(&sums_empty[d], (a / SUMS - 1) & 1, p.error, 44)) {
                            ok = false;
                            break;
                        }
                        tcgen05_fence_after();
#pragma unroll
                        for (int k = 0; k < STEPS; ++k) {
                            const int step = g * STEPS + k;
                            // (the address field counts 16 bytes)
                            tcgen05_mma_bf16_a_tmem(tmem_sums + d * TOKENS, tmem_operands + o * 64 + step * 8,
                                                    x_desc + ((step >> 2) * (T::X_BYTES / 2) + (step & 3) * 32) / 16, idesc, k > 0 ? 1u : 0u);
                        }
                        tcgen05_commit(&sums_full[d]);
                    }
                    tcgen05_commit(&operand_empty[o]);
                    tcgen05_commit(&x_empty[s]);
                }
        }
    } else if (warp < 8) {
        // ---- codes to bfloat16 in TMEM: a thread its row's 128 columns
        asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
        const int quarter = warp & 3;
        const uint32_t to = tmem_operands + (static_cast<uint32_t>(quarter * 32) << 16);
        uint32_t i = 0;
        bool ok = true;
        Piece at;
        for (int r = 0; ok && piece(r, at); ++r)
            for (int chunk = at.c0; chunk < at.c1; ++chunk, ++i) {
                const uint32_t s = i % CODE_STAGES, o = i % OPERANDS;
                if (!mbar_wait_warp(&codes_full[s], (i / CODE_STAGES) & 1, p.error, 45)) {
                    ok = false;
                    break;
                }
                const uint8_t* rec = codes + s * T::CODE_BYTES + quarter * RECORD;
                __align__(16) uint32_t w[4][4];  // [piece][word]
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    *reinterpret_cast<uint4*>(w[c]) = *reinterpret_cast<const uint4*>(rec + packed_word_at(lane, c));
                float sc[GROUPS];
#pragma unroll
                for (int g = 0; g < GROUPS; ++g)
                    sc[g] = to_f32(*reinterpret_cast<const __nv_bfloat16*>(rec + packed_scale_at(lane, g)));
                __syncwarp();
                if (lane == 0)
                    mbar_arrive(&codes_empty[s]);
                uint32_t v[32];
                auto convert = [&](int half) {
#pragma unroll
                    for (int b = 0; b < 2; ++b)
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            const uint32_t word = w[c][2 * half + b];
                            v[b * 16 + c * 4 + 0] = packed_bf16_pair<0>(word);
                            v[b * 16 + c * 4 + 1] = packed_bf16_pair<1>(word);
                            v[b * 16 + c * 4 + 2] = packed_bf16_pair<2>(word);
                            v[b * 16 + c * 4 + 3] = packed_bf16_pair<3>(word);
                        }
                };
                // (the first half while the products before still read the operand's place)
                convert(0);
                if (i >= OPERANDS && !mbar_wait_warp(&operand_empty[o], (i / OPERANDS - 1) & 1, p.error, 46)) {
                    ok = false;
                    break;
                }
                tcgen05_fence_after();
                tmem_store_32x32(to + o * 64, v);
#pragma unroll
                for (int g = 0; g < GROUPS; ++g)
                    scales[((i % PT_SCALE_SLOTS) * GROUPS + g) * PT_ROWS + quarter * 32 + lane] = sc[g];
                convert(1);
                tmem_store_32x32(to + o * 64 + 32, v);
                tmem_store_wait();
                tcgen05_fence_before();
                __syncwarp();
                if (lane == 0)
                    mbar_arrive(&operand_full[o]);
            }
    } else {
        // ---- group sums times scales
        asm volatile("setmaxnreg.inc.sync.aligned.u32 112;");
        pdl_wait();
        const int quarter = warp & 3, part = (warp - 8) >> 2;
        const uint32_t from = tmem_sums + (static_cast<uint32_t>(quarter * 32) << 16) + part * COLS;
        constexpr int LOAD = COLS < 32 ? COLS : 32;
        uint32_t i = 0, a = 0;
        bool ok = true;
        Piece at;
        for (int r = 0; ok && piece(r, at); ++r) {
            uint64_t acc[COLS / 2];
#pragma unroll
            for (int j = 0; j < COLS / 2; ++j)
                acc[j] = 0;
            for (int chunk = at.c0; ok && chunk < at.c1; ++chunk, ++i)
#pragma unroll 1
                for (int g = 0; g < GROUPS; ++g, ++a) {
                    const uint32_t d = a % SUMS;
                    if (!mbar_wait_warp(&sums_full[d], (a / SUMS) & 1, p.error, 47)) {
                        ok = false;
                        break;
                    }
                    tcgen05_fence_after();
                    const float s = scales[((i % PT_SCALE_SLOTS) * GROUPS + g) * PT_ROWS + quarter * 32 + lane];
                    const uint64_t s2 = pair_of(s, s);
#pragma unroll
                    for (int col = 0; col < COLS; col += LOAD) {
                        uint32_t v[LOAD];
                        if constexpr (LOAD == 32)
                            tmem_load_32x32(from + d * TOKENS + col, v);
                        else
                            tmem_load_32x16(from + d * TOKENS + col, v);
                        tmem_load_wait();
                        if (col + LOAD == COLS) {
                            tcgen05_fence_before();
                            __syncwarp();
                            if (lane == 0)
                                mbar_arrive(&sums_empty[d]);
                        }
#pragma unroll
                        for (int j = 0; j < LOAD / 2; ++j)
                            acc[col / 2 + j] = pair_fma(s2, pair_of(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1])), acc[col / 2 + j]);
                    }
                }
            if (!ok)
                break;
#pragma unroll
            for (int j = 0; j < COLS / 2; ++j)
                acc[j] = pair_mul(acc[j], pair_of(PACKED_BF16_UNDO, PACKED_BF16_UNDO));
            if (r == p.rounds) {
                // [column][row], where x was: all of this CTA's copies and products are done
                float* mine = reinterpret_cast<float*>(xs) + part * COLS * PT_ROWS + quarter * 32 + lane;
#pragma unroll
                for (int j = 0; j < COLS / 2; ++j) {
                    const float2 v = halves_of(acc[j]);
                    mine[2 * j * PT_ROWS] = v.x;
                    mine[(2 * j + 1) * PT_ROWS] = v.y;
                }
                continue;
            }
            const int token0 = at.tile % p.token_tiles * TOKENS + part * COLS, n_tile = at.tile / p.token_tiles;
            const int left = p.m - token0;
            if (p.out_type == CHIBI_F32)
                write_columns<COLS, float>(p, acc, token0, left, n_tile, quarter, lane);
            else
                write_columns<COLS, __nv_bfloat16>(p, acc, token0, left, n_tile, quarter, lane);
        }
    }

    __syncwarp();
    if (p.splits > 1) {
        pdl_wait();
        __syncthreads();
        cluster_sync();
        // every CTA of the cluster adds up a share of the tile's columns, four rows a thread
        Piece at;
        const bool any = piece(p.rounds, at);
        const int token0 = at.tile % p.token_tiles * TOKENS, n_tile = at.tile / p.token_tiles;
        const int tokens = any ? min(TOKENS, p.m - token0) : 0;
        const int t0 = tokens * rank / p.splits, t1 = tokens * (rank + 1) / p.splits;
        const uint32_t base = smem_addr(xs);
        for (int e = threadIdx.x; e < (t1 - t0) * (PT_ROWS / 4); e += PT_THREADS) {
            const int token = t0 + e / (PT_ROWS / 4), row = e % (PT_ROWS / 4) * 4;
            const bool up_rows = p.pair && (row & 8);
            if (up_rows)
                continue;
            float v[4] = {}, up[4] = {};
            for (int s = 0; s < p.splits; ++s) {
                float part[4], up_part[4] = {};
                peer_shared_f32x4(base + (token * PT_ROWS + row) * 4, s, part);
                if (p.pair)
                    peer_shared_f32x4(base + (token * PT_ROWS + row + 8) * 4, s, up_part);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    v[j] += part[j];
                    up[j] += up_part[j];
                }
            }
            const long long m = token0 + token;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int at = p.pair ? n_tile * (PT_ROWS / 2) + (row >> 4) * 8 + (row & 7) + j : n_tile * PT_ROWS + row + j;
                if (at >= p.n)
                    continue;
                if (p.pair)
                    v[j] = (p.out_type == CHIBI_F32 ? packed_activate<false>(v[j], p.act) : packed_activate<true>(v[j], p.act)) * up[j];
                else if (p.residual)
                    v[j] += p.residual[m * p.residual_stride + at];
                if (p.out_type == CHIBI_F32)
                    static_cast<float*>(p.out)[m * p.out_stride + at] = v[j];
                else
                    static_cast<__nv_bfloat16*>(p.out)[m * p.out_stride + at] = from_f32<__nv_bfloat16>(v[j]);
            }
        }
        __syncwarp();
        cluster_sync();                          // nobody leaves while another reads
    }
    tcgen05_fence_before();
    __syncthreads();
    if (warp == 1) {
        tcgen05_fence_after();
        tmem_dealloc(tmem_sums, 512);
    }
}

template <int TOKENS, int GROUP_BLOCKS>
int launch_many_rows(const CUtensorMap& map_w, const CUtensorMap& map, const PackedProduct& p, int ctas, cudaStream_t stream)
{
    constexpr size_t SMEM = PackedTile<TOKENS, GROUP_BLOCKS>::SMEM;
    static std::atomic<unsigned long long> allowed;
    const cudaError_t e = packed_allow_shared(packed_many_rows_kernel<TOKENS, GROUP_BLOCKS>, allowed, SMEM);
    if (e != cudaSuccess)
        return (int)e;
    const dim3 grid((unsigned)ctas), block(PT_THREADS);
    if (p.splits > 1)
        launch_cluster_x(packed_many_rows_kernel<TOKENS, GROUP_BLOCKS>, grid, block, SMEM, stream, p.splits, map_w, map, p);
    else
        launch(packed_many_rows_kernel<TOKENS, GROUP_BLOCKS>, grid, block, SMEM, stream, map_w, map, p);
    return launch_status();
}

template <int TOKENS> int launch_many_rows_of(int group, const CUtensorMap& map_w, const CUtensorMap& map, const PackedProduct& p, int ctas,
                                              cudaStream_t stream)
{
    return group == 32 ? launch_many_rows<TOKENS, 1>(map_w, map, p, ctas, stream)
                       : (group == 64 ? launch_many_rows<TOKENS, 2>(map_w, map, p, ctas, stream) : launch_many_rows<TOKENS, 4>(map_w, map, p, ctas, stream));
}

} // namespace
} // namespace chibi

using namespace chibi;

// How many clusters of `splits` CTAs run at once (0: an error); CudaKernels.packed_cut asks.
CHIBI_API int chibi_packed_many_rows_clusters(int splits)
{
    using T = PackedTile<192, 1>;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)splits);
    cfg.blockDim = dim3(PT_THREADS);
    cfg.dynamicSmemBytes = T::SMEM;
    cudaLaunchAttribute attr = {};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)splits;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    int clusters = 0;
    if (splits < 1 || splits > 8
        || cudaFuncSetAttribute(packed_many_rows_kernel<192, 1>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)T::SMEM) != cudaSuccess
        || cudaOccupancyMaxActiveClusters(&clusters, packed_many_rows_kernel<192, 1>, &cfg) != cudaSuccess) {
        cudaGetLastError();
        return 0;
    }
    return clusters;
}

// out[m, n] = x[m, k] times the matrix (+ residual); pair: act(x gate) * (x up), n features.  `tokens`: rows of x of a tile;
// every CTA takes `rounds` whole tiles, what is left is shared by clusters of `splits` CTAs, `clusters` of them (splits 1: CTAs).
// CHIBI_ERR_UNSUPPORTED where x's rows do not start on 16 bytes, or overlap (a tensor map's strides are at least its rows).
CHIBI_API int chibi_packed_many_rows(const ChibiPackedCall* c, const void* x, long long x_stride, void* out, long long out_stride,
                                     const void* residual, long long residual_stride, void* stream)
{
    if (!c || !c->data || !x || !out || c->n < 1 || c->k < 1 || c->m < 1 || !packed_group_ok(c->group) || c->x_type != CHIBI_BF16
        || (c->out_type != CHIBI_F32 && c->out_type != CHIBI_BF16) || (c->pair && (residual || (c->act != 1 && c->act != 2))))
        return CHIBI_ERR_ARGUMENT;
    const int chunks = (c->k + PACKED_COLS - 1) / PACKED_COLS, tokens = c->tokens, splits = c->splits;
    if ((tokens != 48 && tokens != 96 && tokens != 192) || splits < 1 || splits > 8 || splits > chunks || c->rounds < 0 || c->clusters < 1)
        return CHIBI_ERR_ARGUMENT;
    if ((reinterpret_cast<uintptr_t>(x) & 15) || x_stride % 8 || x_stride < c->k)
        return CHIBI_ERR_UNSUPPORTED;
    const int tile_rows = c->pair ? PT_ROWS / 2 : PT_ROWS;
    const long long token_tiles = (c->m + (long long)tokens - 1) / tokens, tiles = (c->n + (long long)tile_rows - 1) / tile_rows * token_tiles;
    if (tiles > 0x3fffffff)
        return CHIBI_ERR_UNSUPPORTED;
    const long long whole = (long long)c->rounds * c->clusters * splits;
    if (splits > 1 ? tiles < whole || tiles - whole > c->clusters : tiles > whole)
        return CHIBI_ERR_ARGUMENT;             // the pieces are not all tiles, each once
    CUtensorMap map_w, map;
    if (!tensor_map_2d(x, c->m, c->k, x_stride, tokens, &map))
        return CHIBI_ERR_UNSUPPORTED;
    memcpy(&map_w, c->map, sizeof(map_w));
    const PackedProduct p { chunks, c->n, c->pair, c->m, out, c->out_type, out_stride, (const float*)residual, residual_stride, c->act,
                            c->rounds, splits, (int)tiles, (int)token_tiles, (int*)c->error };
    const int ctas = c->clusters * splits;
    const cudaStream_t s = (cudaStream_t)stream;
    return tokens == 48 ? launch_many_rows_of<48>(c->group, map_w, map, p, ctas, s)
                        : (tokens == 96 ? launch_many_rows_of<96>(c->group, map_w, map, p, ctas, s)
                                        : launch_many_rows_of<192>(c->group, map_w, map, p, ctas, s));
}
