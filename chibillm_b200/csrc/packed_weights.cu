// Matrices held in 4 bits: packing, reading back, and the product with few rows of x (packed.cuh says how they lie in memory).
#define CHIBI_UNIT packed_weights
#define CHIBI_UNIT_ID 19
#include "packed.cuh"
#include "sm100.cuh"

namespace chibi {
namespace {

// ------------------------------------------------------------------ packing
// A block makes one record: thread (r, seg) the word of row r's columns 8 seg ... 8 seg + 7.  The threads of a group (4, 8 or
// 16 neighbouring lanes) find its largest element together.
//   s = bf16(m / -8), m the element of largest magnitude, the first of equals; q = w / s rounded to nearest, ties to even,
//   within -8 ... 7.  A group with what is not a finite number has the scale NaN.
// w / s is rounded to 32 bits before it is rounded to a whole number, which may go wrong next to a half; w - q s is exact
// (q s has 12 bits, and the difference no more than w has), so it is compared with s / 2.
struct PackSource {
    const void* w[2];          // a matrix, or gate and up
    long long stride[2];
    int rows, cols;            // of each
    int pair;
};

__device__ __forceinline__ int nearest_code(float w, float s)
{
    float q = fminf(fmaxf(rintf(w / s), -9.f), 8.f);
    const float rest = fmaf(-q, s, w), half = 0.5f * fabsf(s);
    const float away = (rest > 0.f) == (s > 0.f) ? 1.f : -1.f;
    if (fabsf(rest) > half || (fabsf(rest) == half && ((int)q & 1)))
        q += away;
    return (int)fminf(fmaxf(q, -8.f), 7.f);
}

template <typename T>
__global__ void __launch_bounds__(256) pack_kernel(PackSource p, int row_blocks, int col_blocks, int group, uint8_t* out)
{
    // (No pdl_trigger: products read their matrix before the kernel ahead of them has ended, so nothing may start before
    // this kernel has.)
    pdl_wait();
    const int r = threadIdx.x >> 4, seg = threadIdx.x & 15;
    const int lanes = group / 8;
    for (long long record = blockIdx.x; record < (long long)row_blocks * col_blocks; record += gridDim.x) {
        const int rb = (int)(record / col_blocks), cb = (int)(record % col_blocks);
        const int side = p.pair ? r >> 3 : 0;
        const int row = p.pair ? rb * 8 + (r & 7) : rb * PACKED_ROWS + r;
        const int col = cb * PACKED_COLS + seg * 8;
        float v[8];
        const T* src = static_cast<const T*>(p.w[side]) + (long long)row * p.stride[side] + col;
        if (row < p.rows && col + 8 <= p.cols && (reinterpret_cast<uintptr_t>(src) & 15) == 0) {
            T raw[8];
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; ++i)
                reinterpret_cast<uint4*>(raw)[i] = reinterpret_cast<const uint4*>(src)[i];
#pragma unroll
            for (int i = 0; i < 8; ++i)
                v[i] = to_f32(raw[i]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                v[i] = row < p.rows && col + i < p.cols ? to_f32(src[i]) : 0.f;
        }
        // the first element of largest magnitude; what is not finite counts as larger than everything
        float best = v[0];
        bool finite = isfinite(v[0]);
#pragma unroll
        for (int i = 1; i < 8; ++i) {
            best = fabsf(v[i]) > fabsf(best) ? v[i] : best;
            finite = finite && isfinite(v[i]);
        }
        for (int o = 1; o < lanes; o <<= 1) {
            const float other = __shfl_xor_sync(0xffffffffu, best, o);
            const bool other_first = (threadIdx.x & o) != 0;
            const bool take = other_first ? fabsf(other) >= fabsf(best) : fabsf(other) > fabsf(best);
            best = take ? other : best;
            finite = __shfl_xor_sync(0xffffffffu, (int)finite, o) && finite;
        }
        __nv_bfloat16 s16 = __float2bfloat16_rn(finite ? best * -0.125f : __int_as_float(0x7fc00000));
        const float s = __bfloat162float(s16);
        if (s == 0.f)
            s16 = __float2bfloat16_rn(0.f);      // (no minus zeros)
        uint32_t word = 0x88888888u;
        if (finite && s != 0.f) {
            word = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                word |= (uint32_t)(nearest_code(v[i], s) + 8) << (4 * (i / 2) + 16 * (i & 1));
        }
        uint8_t* dst = out + record * packed_record_bytes(group);
        *reinterpret_cast<uint32_t*>(dst + packed_word_at(r, seg)) = word;
        if (seg % lanes == 0)
            *reinterpret_cast<__nv_bfloat16*>(dst + packed_scale_at(r, seg / lanes)) = s16;
    }
}

// Whole numbers and scales that somebody else has made, into records.
struct CodeSource {
    const int8_t* codes[2];
    const __nv_bfloat16* scales[2];
    long long stride[2], scale_stride[2];
    int rows, cols, pair;
};

__global__ void __launch_bounds__(256) pack_codes_kernel(CodeSource p, int row_blocks, int col_blocks, int group, uint8_t* out)
{
    pdl_wait();
    const int r = threadIdx.x >> 4, seg = threadIdx.x & 15;
    const int lanes = group / 8;
    for (long long record = blockIdx.x; record < (long long)row_blocks * col_blocks; record += gridDim.x) {
        const int rb = (int)(record / col_blocks), cb = (int)(record % col_blocks);
        const int side = p.pair ? r >> 3 : 0;
        const int row = p.pair ? rb * 8 + (r & 7) : rb * PACKED_ROWS + r;
        const int col = cb * PACKED_COLS + seg * 8;
        uint32_t word = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int q = row < p.rows && col + i < p.cols ? p.codes[side][(long long)row * p.stride[side] + col + i] : 0;
            word |= (uint32_t)((q + 8) & 15) << (4 * (i / 2) + 16 * (i & 1));
        }
        uint8_t* dst = out + record * packed_record_bytes(group);
        *reinterpret_cast<uint32_t*>(dst + packed_word_at(r, seg)) = word;
        if (seg % lanes == 0)
            *reinterpret_cast<__nv_bfloat16*>(dst + packed_scale_at(r, seg / lanes))
                = row < p.rows && col < p.cols ? p.scales[side][(long long)row * p.scale_stride[side] + col / group] : __float2bfloat16_rn(0.f);
    }
}

// The values, rows of a pair's first matrix before those of its second.
template <typename T>
__global__ void __launch_bounds__(256) unpack_kernel(const uint8_t* data, int row_blocks, int col_blocks, int group, int rows, int cols,
                                                     int pair, T* out, long long stride)
{
    pdl_enter();
    const int r = threadIdx.x >> 4, seg = threadIdx.x & 15;
    for (long long record = blockIdx.x; record < (long long)row_blocks * col_blocks; record += gridDim.x) {
        const int rb = (int)(record / col_blocks), cb = (int)(record % col_blocks);
        const int row = pair ? rb * 8 + (r & 7) : rb * PACKED_ROWS + r;
        const int col = cb * PACKED_COLS + seg * 8;
        if (row >= rows || col >= cols)
            continue;
        const uint8_t* src = data + record * packed_record_bytes(group);
        const uint32_t word = *reinterpret_cast<const uint32_t*>(src + packed_word_at(r, seg));
        const float s = to_f32(*reinterpret_cast<const __nv_bfloat16*>(src + packed_scale_at(r, seg * 8 / group)));
        T* dst = out + (long long)(row + (pair ? (r >> 3) * rows : 0)) * stride + col;
        T v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
            v[i] = from_f32<T>((float)((int)((word >> (4 * (i / 2) + 16 * (i & 1))) & 15) - 8) * s);
        if (col + 8 <= cols && (reinterpret_cast<uintptr_t>(dst) & 15) == 0) {
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; ++i)
                reinterpret_cast<uint4*>(dst)[i] = reinterpret_cast<const uint4*>(v)[i];
        } else {
            for (int i = 0; i < 8 && col + i < cols; ++i)
                dst[i] = v[i];
        }
    }
}

// ------------------------------------------------------------------ few rows of x
// out[m][n] = sum over groups of s[n][g] * (sum over the group of q[n][k] x[m][k]).
//
// What bounds it is the bytes of the matrix.  A CTA of 16 warps stays on its SM; every warp streams records of its own
// (bulk copies into a ring of its own, no barrier between warps), makes bfloat16 fragments of the codes and multiplies
// them with x by `mma.m16n8k16`: the 16 rows of a record are the instruction's rows, 8 tokens its columns.  x lies in shared
// memory as the fragments want it, 16 bytes to a lane for two instructions.  Each group's sums start at zero and are
// multiplied by the scales in 32 bits.
//
// 32-bit x is the sum of three bfloat16 numbers (its leading 8 bits, the next 8 and the last 8, cut off, not rounded, so that
// the first does not overflow), three instructions for one.  Rows whose numbers in a CTA's columns are all small or some
// very large are scaled by a power of two before and after, so that last parts are not lost below bfloat16's range and
// sums over q x do not leave 32 bits where sums over s q x would not.
//
// How the work is shared out (CudaKernels.packed_plan chooses): `splits` CTAs of a cluster share the columns, `along_k`
// warps of a CTA share the CTA's columns of one block of 16 rows, 16 / along_k blocks of rows are a unit, and clusters
// take units in turn.  The sums of up to `batch` units stay in shared memory; then the cluster adds them up in one order
// (CTA by CTA, warp by warp), each CTA a share of the outputs, so the same plan gives the same bits.
constexpr int FEW_WARPS = 16, FEW_THREADS = FEW_WARPS * 32;

struct FewRows {
    const uint8_t* data;
    int row_blocks, chunks;        // blocks of 16 rows, of 128 columns
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
    int splits, along_k, batch, depth, tokens;     // tokens: rows of x of a CTA
    int clusters;
    int* error;
};

__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float peer_shared_f32(uint32_t own_smem_addr, uint32_t rank)
{
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(sm100::peer_smem_addr(own_smem_addr, rank)) : "memory");
    return v;
}

// The three parts of two 32-bit numbers, cut off: 8 + 8 + 8 bits, nothing lost above bfloat16's smallest number.  An infinity
// or NaN is its first part alone.
__device__ __forceinline__ void cut_parts(float a, float b, uint32_t (&parts)[3])
{
    float r[2] = { a, b };
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        uint32_t top[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const uint32_t bits = __float_as_uint(r[j]);
            // (a NaN whose upper half has no mantissa bit would turn into an infinity)
            top[j] = i == 0 && isnan(r[j]) ? 0x7fc00000u : bits & 0xffff0000u;
            r[j] = i == 0 && !isfinite(r[j]) ? 0.f : r[j] - __uint_as_float(top[j]);
        }
        parts[i] = (top[0] >> 16) | top[1];
    }
}

// The power of two by which a row of 32-bit numbers is multiplied, from the largest magnitude among its finite ones.
__device__ __forceinline__ float row_factor(uint32_t largest_bits)
{
    const float v = __uint_as_float(largest_bits);
    return v > 0x1p80f ? 0x1p-80f : (v < 0x1p-40f ? 0x1p80f : 1.f);
}

template <int NT, bool X32, int GROUP_BLOCKS>
__global__ void __launch_bounds__(FEW_THREADS, 1) packed_few_rows_kernel(FewRows p)
{
    using namespace sm100;
    constexpr int PARTS = X32 ? 3 : 1;
    constexpr int GROUPS = 4 / GROUP_BLOCKS;
    constexpr int RECORD = PACKED_CODE_BYTES + GROUPS * 32;
    constexpr int SUMS = 128 * NT;               // 32-bit sums of a warp
    extern __shared__ __align__(1024) uint8_t smem[];
    pdl_trigger();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = p.splits > 1 ? (int)cluster_cta_rank() : 0;
    const int cluster = blockIdx.x / p.splits;
    const int token0 = blockIdx.y * p.tokens;
    const int tokens = min(p.tokens, p.m - token0);
    const int c0 = (int)((long long)p.chunks * rank / p.splits), c1 = (int)((long long)p.chunks * (rank + 1) / p.splits);
    const int most = (p.chunks + p.splits - 1) / p.splits;
    const int blocks_per_unit = FEW_WARPS / p.along_k;
    const int units = (p.row_blocks + blocks_per_unit - 1) / blocks_per_unit;

    // shared memory: rings | x | sums | row factors | barriers
    const uint32_t x_plane = (uint32_t)most * 4 * p.tokens * 64;
    uint8_t* ring = smem + (size_t)warp * p.depth * RECORD;
    uint8_t* xs = smem + (size_t)FEW_WARPS * p.depth * RECORD;
    float* sums = reinterpret_cast<float*>(xs + (size_t)PARTS * x_plane);
    uint32_t* largest = reinterpret_cast<uint32_t*>(sums + (size_t)p.batch * FEW_WARPS * SUMS);
    uint64_t* full = reinterpret_cast<uint64_t*>(largest + 16 * NT) + warp * p.depth;

    // the warp's records: of its block of rows in every unit, columns w0 ... w1
    const int wk = warp % p.along_k, wr = warp / p.along_k;
    const int w0 = c0 + (int)((long long)(c1 - c0) * wk / p.along_k), w1 = c0 + (int)((long long)(c1 - c0) * (wk + 1) / p.along_k);
    const int my_rounds = cluster < units ? (units - 1 - cluster) / p.clusters + 1 : 0;
    const int last_unit = cluster + (my_rounds - 1) * p.clusters;
    const int warp_rounds = my_rounds > 0 && last_unit * blocks_per_unit + wr >= p.row_blocks ? my_rounds - 1 : my_rounds;
    const long long total = (long long)warp_rounds * (w1 - w0);
    const long long round_step = (long long)p.clusters * blocks_per_unit * p.chunks * RECORD;
    const uint8_t* next_src = p.data + ((long long)(cluster * blocks_per_unit + wr) * p.chunks + w0) * RECORD;
    long long issued = 0;
    int next_chunk = w0;
    // (one lane)
    auto issue = [&](int slot) {
        mbar_arrive_expect_tx(&full[slot], RECORD);
        bulk_load(ring + (size_t)slot * RECORD, next_src, RECORD, &full[slot]);
    };
    auto advance = [&]() {
        ++issued;
        next_src += RECORD;
        if (++next_chunk == w1) {
            next_chunk = w0;
            next_src += round_step - (long long)(w1 - w0) * RECORD;
        }
    };
    if (lane == 0)
        for (int i = 0; i < p.depth; ++i)
            mbar_init(&full[i], 1);
    if (X32 && threadIdx.x < 16 * NT)
        largest[threadIdx.x] = 0;
    fence_barrier_init();
    fence_proxy_async();
    __syncwarp();
    for (int i = 0; i < p.depth && issued < total; ++i) {
        if (lane == 0)
            issue(i);
        advance();
    }

    // ---- x as fragments: [block of 32 columns][token][lane % 4], 8 neighbouring columns each
    pdl_wait();
    const int pieces = (c1 - c0) * 16 * tokens;
    auto read_piece = [&](int i, float (&v)[8]) -> uint32_t {
        // neighbouring threads take neighbouring pieces of a token; returns where the piece goes
        const int token = i / ((c1 - c0) * 16), seg = i % ((c1 - c0) * 16);
        const int col = c0 * PACKED_COLS + seg * 8;
        if constexpr (X32) {
            const float* src = static_cast<const float*>(p.x) + (long long)(token0 + token) * p.x_stride + col;
            if (col + 8 <= p.k && (reinterpret_cast<uintptr_t>(src) & 15) == 0) {
                *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(src);
                *reinterpret_cast<float4*>(v + 4) = *reinterpret_cast<const float4*>(src + 4);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    v[j] = col + j < p.k ? src[j] : 0.f;
            }
        }
        return (uint32_t)(((seg >> 2) * p.tokens + token) * 64 + (seg & 3) * 16);
    };
    if constexpr (X32) {
        __syncthreads();
        for (int i = threadIdx.x; i < pieces; i += FEW_THREADS) {
            float v[8];
            read_piece(i, v);
            float most_of = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                most_of = isfinite(v[j]) ? fmaxf(most_of, fabsf(v[j])) : most_of;
            atomicMax(&largest[i / ((c1 - c0) * 16)], __float_as_uint(most_of));
        }
        __syncthreads();
    }
    for (int i = threadIdx.x; i < pieces; i += FEW_THREADS) {
        float v[8];
        const uint32_t at = read_piece(i, v);
        if constexpr (X32) {
            const float f = row_factor(largest[i / ((c1 - c0) * 16)]);
            uint32_t parts[4][3];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                cut_parts(v[2 * j] * f, v[2 * j + 1] * f, parts[j]);
#pragma unroll
            for (int part = 0; part < 3; ++part)
                *reinterpret_cast<uint4*>(xs + part * x_plane + at) = make_uint4(parts[0][part], parts[1][part], parts[2][part], parts[3][part]);
        } else {
            const int token = i / ((c1 - c0) * 16), seg = i % ((c1 - c0) * 16);
            const int col = c0 * PACKED_COLS + seg * 8;
            const __nv_bfloat16* src = static_cast<const __nv_bfloat16*>(p.x) + (long long)(token0 + token) * p.x_stride + col;
            uint4 w;
            if (col + 8 <= p.k && (reinterpret_cast<uintptr_t>(src) & 15) == 0) {
                w = *reinterpret_cast<const uint4*>(src);
            } else {
                uint32_t h[8];
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    h[j] = col + j < p.k ? (uint32_t)__bfloat16_as_ushort(src[j]) : 0u;
                w = make_uint4(h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16);
            }
            *reinterpret_cast<uint4*>(xs + at) = w;
        }
    }
    __syncthreads();

    // ---- the stream
    const int r = lane >> 2, c = lane & 3;
    const uint32_t code_at = (uint32_t)packed_word_at(r, c);
    uint32_t x_lane[NT];
    float down[NT][2];                           // undo the rows' factors
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        x_lane[t] = smem_addr(xs) + (uint32_t)min(t * 8 + r, tokens - 1) * 64 + c * 16;
#pragma unroll
        for (int j = 0; j < 2; ++j)
            down[t][j] = X32 ? 1.f / row_factor(largest[min(t * 8 + 2 * c + j, tokens - 1)]) : 1.f;
    }
    const uint32_t x_block = (uint32_t)p.tokens * 64;
    bool dead = false;                           // a wait ran out: nothing more is asked for or computed
    int slot = 0;
    uint32_t phase = 0;
    long long taken = 0;

    for (int first = 0; first < my_rounds; first += p.batch) {
        const int now = min(p.batch, my_rounds - first);
        for (int u = 0; u < now; ++u) {
            float acc[NT][4];
#pragma unroll
            for (int t = 0; t < NT; ++t)
                acc[t][0] = acc[t][1] = acc[t][2] = acc[t][3] = 0.f;
            const int todo = first + u < warp_rounds ? w1 - w0 : 0;
            for (int j = 0; j < todo; ++j) {
                if (!dead || taken < issued)
                    dead = !mbar_wait_warp(&full[slot], phase, p.error, 41) || dead;
                ++taken;
                const uint8_t* rec = ring + (size_t)slot * RECORD;
                const uint4 lo = *reinterpret_cast<const uint4*>(rec + code_at);
                const uint4 hi = *reinterpret_cast<const uint4*>(rec + code_at + 512);
                uint32_t scale[GROUPS];
#pragma unroll
                for (int g = 0; g < GROUPS; ++g)
                    scale[g] = *reinterpret_cast<const uint32_t*>(rec + PACKED_CODE_BYTES + g * 32 + r * 4);
                __syncwarp();
                if (!dead && issued < total) {
                    if (lane == 0)
                        issue(slot);
                    advance();
                }
                if (++slot == p.depth) {
                    slot = 0;
                    phase ^= 1;
                }
                const uint32_t words[2][4] = { { lo.x, lo.y, lo.z, lo.w }, { hi.x, hi.y, hi.z, hi.w } };
                const uint32_t x_at = (uint32_t)(w0 - c0 + j) * 4 * x_block;
#pragma unroll
                for (int g = 0; g < GROUPS; ++g) {
                    float d[NT][4];
#pragma unroll
                    for (int t = 0; t < NT; ++t)
                        d[t][0] = d[t][1] = d[t][2] = d[t][3] = 0.f;
#pragma unroll
                    for (int i = 0; i < GROUP_BLOCKS; ++i) {
                        const int b = g * GROUP_BLOCKS + i;
                        const uint32_t a0[4] = { packed_pair<0>(words[0][b]), packed_pair<0>(words[1][b]),
                                                 packed_pair<1>(words[0][b]), packed_pair<1>(words[1][b]) };
                        const uint32_t a1[4] = { packed_pair<2>(words[0][b]), packed_pair<2>(words[1][b]),
                                                 packed_pair<3>(words[0][b]), packed_pair<3>(words[1][b]) };
#pragma unroll
                        for (int part = 0; part < PARTS; ++part) {
#pragma unroll
                            for (int t = 0; t < NT; ++t) {
                                uint4 f;
                                asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                                             : "=r"(f.x), "=r"(f.y), "=r"(f.z), "=r"(f.w)
                                             : "r"(x_lane[t] + x_at + b * x_block + part * x_plane));
                                mma_16816(d[t], a0, f.x, f.y);
                                mma_16816(d[t], a1, f.z, f.w);
                            }
                        }
                    }
                    const float s0 = __uint_as_float(scale[g] << 16), s1 = __uint_as_float(scale[g] & 0xffff0000u);
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        acc[t][0] = fmaf(s0, d[t][0], acc[t][0]);
                        acc[t][1] = fmaf(s0, d[t][1], acc[t][1]);
                        acc[t][2] = fmaf(s1, d[t][2], acc[t][2]);
                        acc[t][3] = fmaf(s1, d[t][3], acc[t][3]);
                    }
                }
            }
            float* mine = sums + ((size_t)u * FEW_WARPS + warp) * SUMS + lane;
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    mine[(t * 4 + e) * 32] = acc[t][e] * down[t][e & 1];
        }

        // ---- the cluster adds up what its warps have
        __syncwarp();
        if (p.splits > 1)
            cluster_sync();
        else
            __syncthreads();
        const int rows_out = p.pair ? 8 : 16;
        const int outputs = now * blocks_per_unit * rows_out * tokens;
        for (int e = rank * FEW_THREADS + threadIdx.x; e < outputs; e += p.splits * FEW_THREADS) {
            const int row = e % rows_out;
            const int token = e / rows_out % tokens;
            const int block = e / (rows_out * tokens);                   // of the batch: unit by unit
            const int u = block / blocks_per_unit, b = block % blocks_per_unit;
            const int rb = (cluster + (first + u) * p.clusters) * blocks_per_unit + b;
            const int at = rb * rows_out + row;
            if (at >= p.n)
                continue;
            // the fragment's place of (row, token)
            const int reg = (token >> 3) * 4 + (row >> 3) * 2 + (token & 1);
            const uint32_t place = smem_addr(sums + ((size_t)u * FEW_WARPS + b * p.along_k) * SUMS + reg * 32 + (row & 7) * 4 + (token & 7) / 2);
            float v = 0.f, up = 0.f;
            for (int s = 0; s < p.splits; ++s)
                for (int w = 0; w < p.along_k; ++w) {
                    const uint32_t from = place + (uint32_t)w * SUMS * 4;
                    v += p.splits > 1 ? peer_shared_f32(from, s) : *reinterpret_cast<const float*>(__cvta_shared_to_generic(from));
                    if (p.pair)
                        up += p.splits > 1 ? peer_shared_f32(from + 256, s) : *reinterpret_cast<const float*>(__cvta_shared_to_generic(from + 256));
                }
            if (p.pair)
                v = activate(v, p.act) * up;
            const long long m = token0 + token;
            if (p.residual)
                v += p.residual[m * p.residual_stride + at];
            if (p.out_type == CHIBI_F32)
                static_cast<float*>(p.out)[m * p.out_stride + at] = v;
            else
                static_cast<__nv_bfloat16*>(p.out)[m * p.out_stride + at] = from_f32<__nv_bfloat16>(v);
        }
        __syncwarp();
        if (p.splits > 1)
            cluster_sync();                      // nobody leaves, or writes new sums, while another reads
        else if (first + p.batch < my_rounds)
            __syncthreads();
    }
}

template <int NT, bool X32>
void (*few_rows_kernel_of(int group))(FewRows)
{
    return group == 32 ? packed_few_rows_kernel<NT, X32, 1>
                       : (group == 64 ? packed_few_rows_kernel<NT, X32, 2> : packed_few_rows_kernel<NT, X32, 4>);
}

constexpr size_t FEW_SMEM_LIMIT = 227 * 1024;

size_t few_rows_smem(int nt, bool x32, int group, int chunks, int splits, int batch, int depth, int tokens)
{
    const size_t x_plane = (size_t)((chunks + splits - 1) / splits) * 4 * tokens * 64;
    return (size_t)FEW_WARPS * depth * packed_record_bytes(group) + (x32 ? 3 : 1) * x_plane
        + (size_t)batch * FEW_WARPS * 128 * nt * 4 + 16 * nt * 4 + FEW_WARPS * depth * 8;
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
    const int each = up ? 8 : PACKED_ROWS;
    const int row_blocks = (rows + each - 1) / each, col_blocks = (cols + PACKED_COLS - 1) / PACKED_COLS;
    const long long records = (long long)row_blocks * col_blocks;
    CHIBI_DISPATCH_TYPE(type, T, launch(pack_kernel<T>, dim3((unsigned)(records < 65536 ? records : 65536)), dim3(256), 0,
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
    const int each = up_codes ? 8 : PACKED_ROWS;
    const int row_blocks = (rows + each - 1) / each, col_blocks = (cols + PACKED_COLS - 1) / PACKED_COLS;
    const long long records = (long long)row_blocks * col_blocks;
    launch(pack_codes_kernel, dim3((unsigned)(records < 65536 ? records : 65536)), dim3(256), 0, (cudaStream_t)stream, src, row_blocks,
           col_blocks, group, (uint8_t*)out);
    return launch_status();
}

CHIBI_API int chibi_unpack_weights(const void* data, int rows, int cols, int pair, int group, void* out, int out_type, long long stride,
                                   void* stream)
{
    if (!data || !out || rows < 1 || cols < 1 || !packed_group_ok(group))
        return CHIBI_ERR_ARGUMENT;
    const int each = pair ? 8 : PACKED_ROWS;
    const int row_blocks = (rows + each - 1) / each, col_blocks = (cols + PACKED_COLS - 1) / PACKED_COLS;
    const long long records = (long long)row_blocks * col_blocks;
    CHIBI_DISPATCH_TYPE(out_type, T, launch(unpack_kernel<T>, dim3((unsigned)(records < 65536 ? records : 65536)), dim3(256), 0,
                                            (cudaStream_t)stream, (const uint8_t*)data, row_blocks, col_blocks, group, rows, cols, pair,
                                            (T*)out, stride));
    return launch_status();
}

// Shared memory of the kernel for few rows under a plan, in KB (rounded up); CudaKernels.packed_plan asks.
CHIBI_API int chibi_packed_few_rows_kb(int x32, int group, int cols, int tokens, int splits, int batch, int depth)
{
    const int nt = tokens <= 8 ? 1 : 2;
    return (int)((few_rows_smem(nt, x32 != 0, group, (cols + PACKED_COLS - 1) / PACKED_COLS, splits, batch, depth, tokens) + 1023) / 1024);
}

// How many clusters of `splits` CTAs with that much shared memory run at once (0: none, or an error).
CHIBI_API int chibi_packed_few_rows_clusters(int x32, int group, int tokens, int splits, int kb)
{
    if (!packed_group_ok(group) || splits < 1 || splits > 8 || tokens < 1 || tokens > 16 || kb < 1 || kb > 227)
        return 0;
    const int nt = tokens <= 8 ? 1 : 2;
    void (*kernel)(FewRows) = x32 ? (nt == 1 ? few_rows_kernel_of<1, true>(group) : few_rows_kernel_of<2, true>(group))
                                  : (nt == 1 ? few_rows_kernel_of<1, false>(group) : few_rows_kernel_of<2, false>(group));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)splits);
    cfg.blockDim = dim3(FEW_THREADS);
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

// out[m, n] = x[m, k] times the matrix (+ residual); pair: act(x gate) * (x up), n features.  The plan: see FewRows.
CHIBI_API int chibi_packed_few_rows(const void* data, int group, int n, int k, int pair, const void* x, int x_type, long long x_stride,
                                    int m, void* out, int out_type, long long out_stride, const void* residual,
                                    long long residual_stride, int act, int splits, int along_k, int batch, int depth, int tokens,
                                    int clusters, void* error, void* stream)
{
    if (!data || !x || !out || n < 1 || k < 1 || m < 1 || !packed_group_ok(group) || (x_type != CHIBI_F32 && x_type != CHIBI_BF16)
        || (out_type != CHIBI_F32 && out_type != CHIBI_BF16) || (pair && (residual || (act != 1 && act != 2))))
        return CHIBI_ERR_ARGUMENT;
    const int chunks = (k + PACKED_COLS - 1) / PACKED_COLS;
    if (splits < 1 || splits > 8 || (splits & (splits - 1)) || splits > chunks || along_k < 1 || along_k > FEW_WARPS
        || (along_k & (along_k - 1)) || batch < 1 || depth < 1 || tokens < 1 || tokens > 16 || clusters < 1)
        return CHIBI_ERR_ARGUMENT;
    const int nt = tokens <= 8 ? 1 : 2;
    const bool x32 = x_type == CHIBI_F32;
    const size_t smem = few_rows_smem(nt, x32, group, chunks, splits, batch, depth, tokens);
    const long long token_blocks = ((long long)m + tokens - 1) / tokens;
    if (smem > FEW_SMEM_LIMIT || token_blocks > 65535)
        return CHIBI_ERR_UNSUPPORTED;
    const int each = pair ? 8 : PACKED_ROWS;
    const FewRows p { (const uint8_t*)data, (n + each - 1) / each, chunks, n, k, pair, x, x_stride, m, out, out_type, out_stride,
                      (const float*)residual, residual_stride, act, splits, along_k, batch, depth, tokens, clusters, (int*)error };
    void (*kernel)(FewRows) = x32 ? (nt == 1 ? few_rows_kernel_of<1, true>(group) : few_rows_kernel_of<2, true>(group))
                                  : (nt == 1 ? few_rows_kernel_of<1, false>(group) : few_rows_kernel_of<2, false>(group));
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)FEW_SMEM_LIMIT);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return (int)e;
    }
    launch_cluster_x(kernel, dim3((unsigned)(clusters * splits), (unsigned)token_blocks), dim3(FEW_THREADS), smem, (cudaStream_t)stream,
                     splits, p);
    return launch_status();
}
