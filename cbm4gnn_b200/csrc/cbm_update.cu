// Orthogonalised updates by Newton-Schulz products on the 5th-generation tensor cores (sm_100a), fp32-accurate.
//
// X = U / (|U| + eps), turned so that it is no taller than wide; then, `steps` times,
//   A = X X^T,  B = b A + c A A,  X <- a X + B X
// with the quintic (a, b, c) that the Muon optimiser publishes: every singular value is led to between 0.68 and 1.21.
//
// Precision: no entry of X, A or B exceeds 2.9, since none of their singular values does (X stays below 1.21).  So each is kept as
// two fp16 terms of 2^12 times its value, h = fp16(v), l = fp16(v - h): 22 bits, down to 2^-37 of the largest, where fp16 ends.  A
// product takes three fp16 MMAs, h h + h l + l h; l l is below 2^-22 of it.  (The dense maps, whose operands may have any
// exponent, need three bf16 terms and six products, twice the time and a half more shared memory than there is for small matrices.)
// Against float64: 500 x 777 0.6 to 0.8e-6 of the result, where torch's fp32 products give 2.4e-6.  That is of the whole: a row or
// column far below the others meets the floor of 2^-37 sooner (see LOW), and a matrix that has one goes another way, plain_products.
// As in cbm_map.cuh, an accumulator holds 64 columns of a contraction, the small products first, and is added to sums in registers,
// because the tensor cores cut off towards zero at every step.
//
// Work: m (m + 1) n + m^2 (m + 1) + 2 m^2 n a step, as A and A A are symmetric: only tiles that reach the upper triangle are computed,
// and the other half is written with them.
//
// One kernel for larger matrices (small ones have their own, below) and all their products, three kinds of them, in one cooperative launch.
// A block holds a tile of 128 x 64, or a pair of blocks on two SMs one of 256 x 128, of which each fetches half of both operands: one warp
// fetches the operands' terms by TMA (boxes of both terms, 64 columns by 64 or 128 rows, 128-byte swizzled), one issues the MMAs, eight add
// up and write the result, split again, with the term that is added to it.
// X is the second operand of X X^T with the contraction along its rows, and of B X with the contraction across them: the same boxes of
// memory, described to the tensor cores as K-major or MN-major, so that no turned copy exists.
#include "cbm_common.h"
#include "cbm_launch.cuh"
#include "cbm_map.cuh"

#include <cuda.h>
#include <cuda_fp16.h>

#include <cmath>
#include <string>

namespace {

using namespace cbm_map;

constexpr float QUINTIC_A = 3.4445f, QUINTIC_B = -4.7750f, QUINTIC_C = 2.0315f;
constexpr float SCALE = 4096.f, UNSCALE = 1.f / 4096.f;
constexpr int THREADS = 256, PARTS = 64;  // of the norm

constexpr int MAX_JOBS = 8;
constexpr int PRODUCER = 8, ISSUER = 9, TILE_THREADS = 320;  // warps 0 - 7 add up and write
constexpr int BOX_BYTES = 64 * 64 * 2;
constexpr int SLICE = 128 * 128;                 // bytes: 128 rows of 64 columns of one term
constexpr int SMALL_ARRAY = 4 * SLICE;           // [64 columns][term][row]

struct Matrix {
    const float* g;  // update, or gradient
    float *m, *w;    // momentum and weights, or NULL
    float* out;      // result, where there are no weights
    int64_t ldg, ldm, ldw, ldout, next_g, next_out;
    float lr, keep;

    // Up to eight values of a row of the result, 2^12 times what they are.
    __device__ __forceinline__ void write(int64_t matrix, int row, int col, int count, const float (&v)[8]) const {
        float* to = w ? w + row * ldw + col : out + matrix * next_out + row * ldout + col;
        if (count == 8 && (reinterpret_cast<u64>(to) & 15) == 0) {
#pragma unroll
            for (int i = 0; i < 8; i += 4) {
                float4 r = make_float4(v[i] * UNSCALE, v[i + 1] * UNSCALE, v[i + 2] * UNSCALE, v[i + 3] * UNSCALE);
                float4* at = reinterpret_cast<float4*>(to + i);
                if (w) {
                    const float4 was = *at;
                    r = make_float4(keep * was.x - lr * r.x, keep * was.y - lr * r.y, keep * was.z - lr * r.z, keep * was.w - lr * r.w);
                }
                *at = r;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < count) to[i] = w ? keep * to[i] - lr * (v[i] * UNSCALE) : v[i] * UNSCALE;
        }
    }
};

// Matrices of one shape: a stack, or one weight of a list.
struct Shape {
    __half *px[2], *pa, *pb;
    double* parts;             // [batch][PARTS]
    int* low;                  // [batch]: whether it has stretches of rows or columns that two fp16 terms do not hold
    Matrix of;
    int m, n, ldx, lda, turned, batch;
    int tiles_sym, tiles_all;  // of one matrix: that reach the upper triangle of A, of X
};
// [batch][2 terms][rows][columns]; boxes of both terms of 64 columns and 128 rows, for the first operand, or 64, for the second.
struct Maps {
    CUtensorMap first_x[2], first_a, first_b, second_x[2], second_a;
};

struct Jobs {
    Maps map[MAX_JOBS];
    Shape job[MAX_JOBS];
    int count;
    float momentum, eps;
    int nesterov;
    int* timeout;
    u32* arrived;              // of the products' blocks, zeroed by the first kernel
    int* any_low;              // whether a matrix of the call has `low` set
};

enum Kind { GRAM, SQUARE, APPLY };

// ---- start ----------------------------------------------------------------------------------------
__device__ __forceinline__ float update_at(const Jobs& p, const Shape& q, int64_t b, int i, int j) {
    const float g = q.of.g[b * q.of.next_g + i * q.of.ldg + j];
    if (!q.of.m) return g;
    const float m = __ldcg(&q.of.m[i * q.of.ldm + j]);  // already this step's
    return p.nesterov ? g + p.momentum * m : m;
}

// This step's momentum, and parts of the squared norm of the update in 64 bits.  Block x: a part, y: a matrix.
__global__ void __launch_bounds__(THREADS) norm_kernel(const __grid_constant__ Jobs p) {
    cbm::wait_before();
    int j = 0, b = blockIdx.y;
    while (b >= p.job[j].batch) b -= p.job[j++].batch;
    const Shape& q = p.job[j];
    const int rows = q.turned ? q.n : q.m, cols = q.turned ? q.m : q.n;
    double s = 0.0;
    for (int i = blockIdx.x; i < rows; i += PARTS)
        for (int c = threadIdx.x; c < cols; c += THREADS) {
            if (q.of.m) {
                float* m = &q.of.m[i * q.of.ldm + c];
                *m = p.momentum * *m + q.of.g[i * q.of.ldg + c];
            }
            const double u = update_at(p, q, b, i, c);
            s += u * u;
        }
    __shared__ double part[THREADS / 32];
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < THREADS / 32; ++i) s += part[i];
        q.parts[b * PARTS + blockIdx.x] = s;
        if (blockIdx.x == 0) q.low[b] = 0;
        if (blockIdx.x == 0 && blockIdx.y == 0) *p.arrived = 0, *p.any_low = 0;
    }
}

// A matrix is low where a stretch of a row or column (32 values of larger matrices, up to 128 of small ones) with FEWEST or more that are not 0
// has none of LOW of the norm.  (One value or two may be that small by chance.)  In two fp16 terms rows of 128 x 512 whose largest value is 2^-16 of the norm come out with an error of 9e-7, at 2^-23 of 9e-5,
// at 2^-30 of 9e-3, and below 2^-37 not at all; in fp32 all with 2e-7 (1 600 x 1 500: 5e-4 at 2^-26, 4e-7 in fp32).  The time of
// fp32 is why it is not taken sooner: 2 048 x 4 096 13.1 ms, in two terms 1.12 (by a library's products 8.0); 64 x 500 369 us, 56 (439).
constexpr float LOW = 1.f / (1 << 24);
constexpr int FEWEST = 4;
__device__ __forceinline__ u32 magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }  // (in the order of the values; NaN above all)
__device__ __forceinline__ bool is_low(u32 most, float scale) { return most && most < __float_as_uint(LOW * scale); }

__device__ __forceinline__ double norm_of(const Shape& q, int b) {  // (by a warp)
    double s = 0.0;
    for (int i = 0; i < PARTS; i += 32) s += __ldcg(&q.parts[b * PARTS + i + (threadIdx.x & 31)]);
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    return sqrt(s);
}

__device__ __forceinline__ void split(float v, __half& h, __half& l) {
    h = __float2half_rn(v);
    l = __float2half_rn(v - __half2float(h));
}

// X, split: 32 x 32 values to a block, through shared memory where it is turned.  Block x: a tile (of the largest job), y: a matrix.
__global__ void __launch_bounds__(THREADS) start_kernel(const __grid_constant__ Jobs p) {
    constexpr int EACH = 32 * 32 / THREADS;
    __shared__ float turn[32][33];
    __shared__ u32 s_column[32], s_values[32];
    cbm::wait_before();
    int j = 0, b = blockIdx.y;
    while (b >= p.job[j].batch) b -= p.job[j++].batch;
    const Shape& q = p.job[j];
    const int across = (q.n + 31) / 32, tiles = across * ((q.m + 31) / 32), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const double scale = (double)SCALE / (norm_of(q, b) + (double)p.eps);
    bool low = false;
    const int64_t plane = (int64_t)q.m * q.ldx;
    __half* x = q.px[0] + 2 * b * plane;
    for (int t = blockIdx.x; t < tiles; t += gridDim.x) {
        const int r0 = t / across * 32, c0 = t % across * 32;
        if (q.turned) {  // (the barrier at the end is behind the last tile's reads)
            for (int i = warp; i < 32; i += THREADS / 32)
                if (c0 + i < q.n && r0 + lane < q.m) turn[i][lane] = update_at(p, q, b, c0 + i, r0 + lane);
            __syncthreads();
        }
        float v[EACH];
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
            const int i = warp + e * (THREADS / 32);
            v[e] = r0 + i < q.m && c0 + lane < q.n ? (q.turned ? turn[lane][i] : update_at(p, q, b, r0 + i, c0 + lane)) : 0.f;
        }
        u32 column = 0;
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
            const int i = warp + e * (THREADS / 32);
            v[e] = (float)((double)v[e] * scale);
            column = max(column, magnitude(v[e]));
            if (is_low(__reduce_max_sync(0xffffffffu, magnitude(v[e])), SCALE)) low |= __popc(__ballot_sync(0xffffffffu, magnitude(v[e]))) >= FEWEST;
            if (r0 + i < q.m && c0 + lane < q.n) {
                __half h, l;
                split(v[e], h, l);
                const int64_t at = (int64_t)(r0 + i) * q.ldx + c0 + lane;
                x[at] = h;
                x[at + plane] = l;
            }
        }
        // a column is low where all that warps have of it is
        if (__syncthreads_or(is_low(column, SCALE))) {
            if (warp == 0) s_column[lane] = s_values[lane] = 0;
            __syncthreads();
            u32 values = 0;
#pragma unroll
            for (int e = 0; e < EACH; ++e) values += magnitude(v[e]) != 0;
            atomicMax(&s_column[lane], column);
            atomicAdd(&s_values[lane], values);
            __syncthreads();
            if (warp == 0) low |= s_values[lane] >= FEWEST && is_low(s_column[lane], SCALE);
        }
    }
    if (low) q.low[b] = 1, *p.any_low = 1;
}

// ---- products -------------------------------------------------------------------------------------
// SINGLE: a block to a tile.  PAIR: two blocks on neighbouring SMs to a tile, whose MMAs the first one issues for both.
enum Mode { SINGLE, PAIR };

template <Mode MODE>
struct Sizes {
    static constexpr int BN = MODE == PAIR ? 128 : 64;        // columns of a tile
    static constexpr int ROWS = MODE == PAIR ? 256 : 128;     // rows of a tile
    static constexpr int STAGES = 4;
    static constexpr int A_BYTES = 4 * BOX_BYTES;             // 2 terms of 128 x 64, of this block
    static constexpr int B_TERM = BOX_BYTES;                  // 64 x 64
    static constexpr int STAGE = A_BYTES + 2 * B_TERM;
    static constexpr int TURN = 32 * 32 * 4;                  // a warp's block of 32 x 32 on its way out
    static constexpr int SMEM = STAGES * STAGE + 8 * TURN + 1024;
    static constexpr int ACC_COLS = 2 * BN;                   // of an accumulator, see mma_chunk
    static constexpr int ACCS = TMEM_COLS / ACC_COLS;
};

// A chunk of 64 of the contraction: with the second operand's terms h and l behind one another as one operand of twice the columns,
// A_h [B_h | B_l] is one MMA a step, and A_l B_h the other, added to the columns from 64 on.  (So A_h is read once for two products: an
// MMA's operands come out of shared memory at about 64 bytes a cycle, and a tile is too narrow to hide that: 256 x 128 3 x 96 cycles a step,
// 128 + 96 so.  That bound, not L2, is also why single blocks have tiles of 64 columns.)  A block's half of the columns has its own 128:
// h h, then h l and l h; in the second block of a pair l h comes to h h instead, which makes no difference to the sum of both.
// Issued as one, by one elected thread: one by one, with an election and descriptors for each, twelve MMAs took 1 440 cycles.
template <bool TWO>
__device__ __forceinline__ void mma_chunk(u32 d, u64 ah, u64 al, u64 b, u64 next_b, u32 both, u32 one) {
#define CBM_MMA(D, A, B, I, ADD) "@e tcgen05.mma.cta_group::" CBM_GROUP ".kind::f16 [" D "], " A ", " B ", " I ", " ADD ";\n\t"
#define CBM_CHUNK                                                                                                              \
    "{\n\t.reg .pred e, no, yes;\n\t.reg .b64 ah1, ah2, ah3, al1, al2, al3, b1, b2, b3;\n\t.reg .b32 d1;\n\t"                       \
    "elect.sync _|e, 0xffffffff;\n\tsetp.ne.u32 no, 0, 0;\n\tsetp.eq.u32 yes, 0, 0;\n\tadd.u32 d1, %0, 64;\n\t"                    \
    "add.s64 ah1, %1, 2;\n\tadd.s64 ah2, %1, 4;\n\tadd.s64 ah3, %1, 6;\n\t"                                                      \
    "add.s64 al1, %2, 2;\n\tadd.s64 al2, %2, 4;\n\tadd.s64 al3, %2, 6;\n\t"                                                      \
    "add.s64 b1, %3, %4;\n\tadd.s64 b2, b1, %4;\n\tadd.s64 b3, b2, %4;\n\t"                                                      \
    CBM_MMA("%0", "%1", "%3", "%5", "no") CBM_MMA("d1", "%2", "%3", "%6", "yes") CBM_MMA("d1", "al1", "b1", "%6", "yes")       \
    CBM_MMA("d1", "al2", "b2", "%6", "yes") CBM_MMA("d1", "al3", "b3", "%6", "yes") CBM_MMA("%0", "ah1", "b1", "%5", "yes")    \
    CBM_MMA("%0", "ah2", "b2", "%5", "yes") CBM_MMA("%0", "ah3", "b3", "%5", "yes") "}"
    if constexpr (TWO) {
#define CBM_GROUP "2"
        asm volatile(CBM_CHUNK ::"r"(d), "l"(ah), "l"(al), "l"(b), "l"(next_b), "r"(both), "r"(one) : "memory");
#undef CBM_GROUP
    } else {
#define CBM_GROUP "1"
        asm volatile(CBM_CHUNK ::"r"(d), "l"(ah), "l"(al), "l"(b), "l"(next_b), "r"(both), "r"(one) : "memory");
#undef CBM_GROUP
    }
#undef CBM_CHUNK
#undef CBM_MMA
}
// fp32 accumulator, fp16 operands; bit 16: the second operand is MN-major.
__host__ __device__ constexpr u32 idesc_half(u32 m, u32 n, bool mn_major) { return (1u << 4) | ((u32)mn_major << 16) | ((n >> 3) << 17) | ((m >> 4) << 24); }
// MN-major operand of 64-wide, 128-byte swizzled blocks: 8 steps of the contraction are 1024 bytes, the next 64 columns a box further on.
__device__ __forceinline__ u64 desc_mn(u32 addr) {
    return (u64)((addr & 0x3ffff) >> 4) | ((u64)(BOX_BYTES >> 4) << 16) | ((u64)(1024 >> 4) << 32) | ((u64)1 << 46) | ((u64)2 << 61);
}

__device__ __forceinline__ void ld32(float (&r)[32], u32 at) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, "
        "%21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]), "=f"(r[9]), "=f"(r[10]),
          "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]), "=f"(r[16]), "=f"(r[17]), "=f"(r[18]), "=f"(r[19]), "=f"(r[20]),
          "=f"(r[21]), "=f"(r[22]), "=f"(r[23]), "=f"(r[24]), "=f"(r[25]), "=f"(r[26]), "=f"(r[27]), "=f"(r[28]), "=f"(r[29]), "=f"(r[30]),
          "=f"(r[31])
        : "r"(at));
}

// `bar` may be the other block's of a pair.  (By an elected thread of a warp that stays together, see mma; and one fetch for both terms
// of all rows: issued one by one from a branch for lane 0, the 64 x 64 boxes took 190 cycles each, more than the MMAs waiting for them.)
template <bool TWO>
__device__ __forceinline__ void box_in(u32 to, const CUtensorMap* map, int col, int row, int matrix, u32 bar) {
    if constexpr (TWO)
        asm volatile(
            "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
            "@e cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3, 0, %4}], [%5];\n\t}" ::"r"(to),
            "l"(map), "r"(col), "r"(row), "r"(matrix), "r"(bar)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
            "@e cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, 0, %4}], [%5];\n\t}" ::"r"(to),
            "l"(map), "r"(col), "r"(row), "r"(matrix), "r"(bar)
            : "memory");
}
__device__ __forceinline__ void expect(u32 bar, u32 bytes) {
    asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t@e mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n\t}" ::"r"(bar), "r"(bytes)
                 : "memory");
}

// ---- a pair of blocks -----------------------------------------------------------------------------
__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}
// The first block's address of what lies at `local` in this one.
__device__ __forceinline__ u32 in_first(u32 local) {
    u32 r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(local));
    return r;
}
__device__ __forceinline__ void arrive_in_first(u32 mapped) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(mapped) : "memory");
}
// In both blocks, once the MMAs issued so far are done.
__device__ __forceinline__ void commit_both(u32 bar) {
    asm volatile(
        "{\n\t.reg .pred e;\n\t.reg .b16 both;\n\tmov.b16 both, 3;\n\telect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], both;\n\t}" ::"r"(bar)
        : "memory");
}
__device__ __forceinline__ void pair_alloc(u32 where) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(where), "n"(TMEM_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
}
__device__ __forceinline__ void pair_free(u32 base) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(base), "n"(TMEM_COLS));
}
struct Where {
    int job, matrix, row, col;  // tile: rows from ROWS row, columns from BN col
};
// Tile t of a matrix.
template <int ROWS, int BN>
__device__ __forceinline__ void place(const Shape& q, Kind kind, int t, Where& w) {
    if (kind == APPLY) {
        // down the columns first: neighbouring blocks share X's columns, and B is small
        const int down = (q.m + ROWS - 1) / ROWS;
        if (down == 1) w.col = t, w.row = 0;  // (a division costs a small product a tenth of its time)
        else if (down == 2) w.col = t >> 1, w.row = t & 1;
        else w.col = t / down, w.row = t - w.col * down;
        return;
    }
    const int across = (q.m + BN - 1) / BN;
    w.row = 0;
    for (int left = across; t >= left; left = across - w.row * (ROWS / BN)) t -= left, ++w.row;
    w.col = w.row * (ROWS / BN) + t;
}
// The tile with running number t of a kind of product, over all matrices.
template <int ROWS, int BN>
__device__ __forceinline__ Where tile_of(const Shape* jobs, Kind kind, int t) {
    Where w{0, 0, 0, 0};
    for (;; ++w.job) {
        const Shape& q = jobs[w.job];
        const int each = kind == APPLY ? q.tiles_all : q.tiles_sym, all = each * q.batch;
        if (t >= all) {
            t -= all;
            continue;
        }
        w.matrix = t / each;
        place<ROWS, BN>(q, kind, t - w.matrix * each, w);
        return w;
    }
}

// Two fp16 terms of eight values.
struct Terms {
    uint4 h, l;
    __device__ __forceinline__ void load(const __half* p, int64_t plane) {
        h = __ldcg(reinterpret_cast<const uint4*>(p));
        l = __ldcg(reinterpret_cast<const uint4*>(p + plane));
    }
    __device__ __forceinline__ void store(__half* p, int64_t plane) const {
        *reinterpret_cast<uint4*>(p) = h;
        *reinterpret_cast<uint4*>(p + plane) = l;
    }
    __device__ __forceinline__ void set(int i, u32 a, u32 b) {
        (i == 0 ? h.x : i == 1 ? h.y : i == 2 ? h.z : h.w) = a;
        (i == 0 ? l.x : i == 1 ? l.y : i == 2 ? l.z : l.w) = b;
    }
    // Both terms of value j in one word, the first below; and back.
    __device__ __forceinline__ u32 word(int j) const {
        const u32 a = j < 2 ? h.x : j < 4 ? h.y : j < 6 ? h.z : h.w, b = j < 2 ? l.x : j < 4 ? l.y : j < 6 ? l.z : l.w;
        return __byte_perm(a, b, j & 1 ? 0x7632 : 0x5410);
    }
    __device__ __forceinline__ void pair(int i, u32 first, u32 second) {
        set(i, __byte_perm(first, second, 0x5410), __byte_perm(first, second, 0x7632));
    }
    // v += f * these
    __device__ __forceinline__ void add_to(float (&v)[8], float f) const {
        const u32 x[4] = {h.x, h.y, h.z, h.w}, y[4] = {l.x, l.y, l.z, l.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 s = __half22float2(reinterpret_cast<const __half2&>(x[i])), t = __half22float2(reinterpret_cast<const __half2&>(y[i]));
            v[2 * i] += f * s.x + f * t.x;
            v[2 * i + 1] += f * s.y + f * t.y;
        }
    }
};
// The two terms of eight values.  (Two values a conversion: one by one they are converted at a quarter of the rate.)
__device__ __forceinline__ Terms terms_of(const float (&v)[8]) {
    Terms t;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
        const float2 f = __half22float2(h);
        const __half2 l = __floats2half2_rn(v[2 * i] - f.x, v[2 * i + 1] - f.y);
        t.set(i, reinterpret_cast<const u32&>(h), reinterpret_cast<const u32&>(l));
    }
    return t;
}

// Between two products: what any block wrote before is seen by all behind it, their TMA fetches included.  All blocks are resident (the
// launch is a cooperative one), so each comes here; a block that has given up goes on without waiting.
// (The warps of a block come here from different places.)
__device__ __forceinline__ void block_barrier() { asm volatile("barrier.sync 1, %0;" ::"n"(TILE_THREADS) : "memory"); }
__device__ __forceinline__ void all_blocks(u32* arrived, u32 due, volatile int* gave_up, int* timeout, bool wrote, bool fetches) {
    if (wrote) asm volatile("fence.proxy.async;" ::: "memory");
    block_barrier();
    if (threadIdx.x == 0 && gridDim.x > 1) {
        __threadfence();
        asm volatile("red.release.gpu.global.add.u32 [%0], 1;" ::"l"(arrived) : "memory");
        u64 t0 = 0;
        for (u32 spins = 0; !*gave_up; ++spins) {
            u32 n;
            asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(n) : "l"(arrived) : "memory");
            if ((int)(n - due) >= 0) break;
            if ((spins & 31u) == 31u) {
                const u64 t = now_ns();
                if (t0 == 0) t0 = t;
                if (t - t0 > WAIT_NS || spins > (1u << 26)) {
                    *gave_up = 1;
                    *(volatile int*)timeout = 1;
                }
            }
        }
        __threadfence();
    }
    block_barrier();
    if (fetches) asm volatile("fence.proxy.async;" ::: "memory");
}

// ---- matrices with rows or columns far below the others ----------------------------------------------
// The steps in fp32 without tensor cores, by `blocks` blocks that meet in `sync` between products, what they wrote then seen by all.  256
// threads to a tile, of 128 x 128 beside pairs of blocks, else 64 x 64: 64 products to 16 values out of shared memory, or 16 to 8; the next piece of the contraction is on its way meanwhile.  X, A and B lie where their two terms would.  Of A and
// B half the tiles are computed: the other half comes out the same, as its products commute.
constexpr int PLAIN_VALUES = 2048, PLAIN_SMEM = 4 * 32 * (64 + 4) * 4;  // of an operand's piece; bytes for two pieces of both
static_assert(PLAIN_SMEM >= 4 * 16 * (128 + 4) * 4 && PLAIN_SMEM <= SMALL_ARRAY && PLAIN_SMEM <= Sizes<SINGLE>::STAGES * Sizes<SINGLE>::STAGE,
              "operands lie where the tensor cores' would");

// sum = rows from i0 on of `first` times rows (or, ACROSS, columns) from j0 on of `second`, whose rows start at multiples of 16 bytes.
template <int TILE, bool ACROSS>
__device__ __forceinline__ void plain_tile(const float* first, int ld1, int rows1, int i0, const float* second, int ld2, int width, int j0, int deep,
                                           float* smem, float (&sum)[TILE / 16][TILE / 16]) {
    constexpr int DEEP = PLAIN_VALUES / TILE, PITCH = TILE + 4, PIECE = DEEP * PITCH, EACH = TILE / 16;
    const int at = threadIdx.x, ty = at >> 4, tx = at & 15;
    const bool works = at < 256;
    float4 a[2], b[2];
    auto row_of = [&](const float* from, int ld, int rows, int r, int k) {
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        if (r < rows && k < deep) {
            v = __ldcg(reinterpret_cast<const float4*>(from + (int64_t)r * ld + k));
            if (k + 1 >= deep) v.y = 0.f;
            if (k + 2 >= deep) v.z = 0.f;
            if (k + 3 >= deep) v.w = 0.f;
        }
        return v;
    };
    auto fetch = [&](int k0) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int i = at + 256 * e, r = i / (DEEP / 4), k = k0 + 4 * (i % (DEEP / 4));
            a[e] = row_of(first, ld1, rows1, i0 + r, k);
            if constexpr (ACROSS) {  // (columns past the last make results past the last)
                const int d = k0 + i / (TILE / 4), j = j0 + 4 * (i % (TILE / 4));
                b[e] = d < deep && j < width ? __ldcg(reinterpret_cast<const float4*>(second + (int64_t)d * ld2 + j)) : make_float4(0.f, 0.f, 0.f, 0.f);
            } else {
                b[e] = row_of(second, ld2, width, j0 + r, k);
            }
        }
    };
    auto put = [&](float* to) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int i = at + 256 * e, r = i / (DEEP / 4), k = 4 * (i % (DEEP / 4));
            to[k * PITCH + r] = a[e].x, to[(k + 1) * PITCH + r] = a[e].y, to[(k + 2) * PITCH + r] = a[e].z, to[(k + 3) * PITCH + r] = a[e].w;
            float* const next = to + PIECE;
            if constexpr (ACROSS) *reinterpret_cast<float4*>(next + i / (TILE / 4) * PITCH + 4 * (i % (TILE / 4))) = b[e];
            else next[k * PITCH + r] = b[e].x, next[(k + 1) * PITCH + r] = b[e].y, next[(k + 2) * PITCH + r] = b[e].z, next[(k + 3) * PITCH + r] = b[e].w;
        }
    };
#pragma unroll
    for (int i = 0; i < EACH; ++i)
#pragma unroll
        for (int j = 0; j < EACH; ++j) sum[i][j] = 0.f;
    __syncthreads();  // (the last tile's reads)
    if (works) fetch(0), put(smem);
    int turn = 0;
    for (int k0 = 0; k0 < deep; k0 += DEEP, turn ^= 1) {
        __syncthreads();
        if (!works) continue;
        const bool more = k0 + DEEP < deep;
        if (more) fetch(k0 + DEEP);
        const float* const from = smem + turn * 2 * PIECE;
#pragma unroll 4
        for (int k = 0; k < DEEP; ++k) {
            float u[EACH], v[EACH];
#pragma unroll
            for (int i = 0; i < EACH; i += 4) {
                *reinterpret_cast<float4*>(&u[i]) = *reinterpret_cast<const float4*>(from + k * PITCH + 16 * i + 4 * ty);
                *reinterpret_cast<float4*>(&v[i]) = *reinterpret_cast<const float4*>(from + PIECE + k * PITCH + 16 * i + 4 * tx);
            }
#pragma unroll
            for (int i = 0; i < EACH; ++i)
#pragma unroll
                for (int j = 0; j < EACH; ++j) sum[i][j] += u[i] * v[j];
        }
        if (more) put(smem + (turn ^ 1) * 2 * PIECE);
    }
}

struct Plain {
    float *x[2], *gram, *poly;
    __device__ __forceinline__ Plain(const Shape& q, int b) {
        x[0] = reinterpret_cast<float*>(q.px[0]) + (int64_t)b * q.m * q.ldx, x[1] = reinterpret_cast<float*>(q.px[1]) + (int64_t)b * q.m * q.ldx;
        gram = reinterpret_cast<float*>(q.pa) + (int64_t)b * q.m * q.lda, poly = reinterpret_cast<float*>(q.pb) + (int64_t)b * q.m * q.lda;
    }
};
// Tiles first, first + blocks, ... of a product of a matrix, of `tiles`, `across` in a row.
template <int TILE, bool ACROSS>
__device__ __forceinline__ void plain_product(const Shape& q, int b, Kind kind, int from, bool last, int first, int blocks, float* smem) {
    const Plain is(q, b);
    const int m = q.m, width = kind == APPLY ? q.n : m, across = (width + TILE - 1) / TILE, down = (m + TILE - 1) / TILE;
    const int tiles = kind == APPLY ? across * down : across * (across + 1) / 2;
    for (int t = first; t < tiles; t += blocks) {
        int i0 = t / across, j0 = t % across;
        if (kind != APPLY) {
            i0 = 0, j0 = t;
            for (int left = across; j0 >= left; left = across - i0) j0 -= left, ++i0;
            j0 += i0;
        }
        i0 *= TILE, j0 *= TILE;
        float sum[TILE / 16][TILE / 16];
        if (kind == GRAM) plain_tile<TILE, ACROSS>(is.x[from], q.ldx, m, i0, is.x[from], q.ldx, m, j0, q.n, smem, sum);
        else plain_tile<TILE, ACROSS>(kind == SQUARE ? is.gram : is.poly, q.lda, m, i0, ACROSS ? is.x[from] : is.gram, ACROSS ? q.ldx : q.lda, width, j0, m, smem, sum);
        if (threadIdx.x >= 256) continue;
#pragma unroll
        for (int i = 0; i < TILE / 16; ++i)
#pragma unroll
            for (int j = 0; j < TILE / 16; ++j) {
                const int r = i0 + i / 4 * 64 + 4 * (threadIdx.x >> 4) + i % 4, c = j0 + j / 4 * 64 + 4 * (threadIdx.x & 15) + j % 4;
                if (r >= m || c >= width) continue;
                float v = sum[i][j];
                if constexpr (!ACROSS) {
                    if (kind == SQUARE) v = QUINTIC_C * v + QUINTIC_B * __ldcg(is.gram + (int64_t)r * q.lda + c);
                    float* const to = kind == GRAM ? is.gram : is.poly;
                    to[(int64_t)r * q.lda + c] = v;
                    if (j0 != i0) to[(int64_t)c * q.lda + r] = v;
                } else {
                    v += QUINTIC_A * __ldcg(is.x[from] + (int64_t)r * q.ldx + c);
                    const float o[8] = {SCALE * v};
                    if (!last) is.x[from ^ 1][(int64_t)r * q.ldx + c] = v;
                    else if (q.turned) q.of.write(b, c, r, 1, o);
                    else q.of.write(b, r, c, 1, o);
                }
            }
    }
}

// Matrix `only` of the first job, whose norm is given, or all that have `low` set.
template <int TILE, class Sync>
__device__ __noinline__ void plain_products(const Jobs& p, const Shape* jobs, int only, double norm, int steps, int rank, int blocks, float* smem, Sync sync) {
    auto each = [&](auto&& f) {
        if (only >= 0) return f(jobs[0], only);
        for (int j = 0; j < p.count; ++j)
            for (int b0 = 0; b0 < jobs[j].batch; b0 += 32) {
                const int b = b0 + (threadIdx.x & 31);
                for (u32 set = __ballot_sync(0xffffffffu, b < jobs[j].batch && __ldcg(&jobs[j].low[b])); set; set &= set - 1) f(jobs[j], b0 + __ffs(set) - 1);
            }
    };
    each([&](const Shape& q, int b) {
        float* const x = Plain(q, b).x[0];
        const double scale = 1.0 / ((only >= 0 ? norm : norm_of(q, b)) + (double)p.eps);
        for (int i = rank; i < q.m; i += blocks)
            for (int j = threadIdx.x; j < q.n; j += blockDim.x)
                x[(int64_t)i * q.ldx + j] = (float)((double)(q.turned ? update_at(p, q, b, j, i) : update_at(p, q, b, i, j)) * scale);
    });
    sync();
    for (int k = 0; k < steps; ++k)
        for (int kind = GRAM; kind <= APPLY; ++kind) {
            int at = rank;  // this block's next tile, from where a matrix' tiles begin
            each([&](const Shape& q, int b) {
                const int width = kind == APPLY ? q.n : q.m;
                const int across = (width + TILE - 1) / TILE, tiles = kind == APPLY ? across * ((q.m + TILE - 1) / TILE) : across * (across + 1) / 2;
                if (kind == APPLY) plain_product<TILE, true>(q, b, APPLY, k & 1, k + 1 == steps, at, blocks, smem);
                else plain_product<TILE, false>(q, b, (Kind)kind, k & 1, false, at, blocks, smem);
                at = ((at - tiles) % blocks + blocks) % blocks;
            });
            sync();
        }
}

// All products of all matrices, one kind after the other: as launches of their own each of the fifteen took 5 to 8 us before its first MMA.
// (320 threads may have 168 registers each; pairs, whose warps add up 64 columns, spill some 204 bytes of them a thread, single blocks none.)
template <Mode MODE>
__global__ void __launch_bounds__(TILE_THREADS, 1) product_kernel(const __grid_constant__ Jobs p, const int sym_tiles, const int all_tiles,
                                                                  const int steps) {
    using S = Sizes<MODE>;
    constexpr int BN = S::BN;
    constexpr bool TWO = MODE == PAIR;
    extern __shared__ unsigned char smem_raw[];
    __shared__ u64 s_bar[2 * S::STAGES + 2 * S::ACCS + 1];
    __shared__ u32 s_tmem;
    __shared__ int s_gave_up, s_any_low;
    // (at an index that is not known beforehand, parameters are read from the constant bank at hundreds of cycles a time)
    __shared__ Shape s_jobs[MAX_JOBS];
    const u32 smem = (smem_u32(smem_raw) + 1023) & ~1023u;
    const int lane = threadIdx.x & 31, warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
    const u32 full = smem_u32(s_bar), empty = full + 8 * S::STAGES, acc_full = empty + 8 * S::STAGES, acc_empty = acc_full + 8 * S::ACCS,
              drained = acc_empty + 8 * S::ACCS;
    if (warp == ISSUER) {
        if constexpr (TWO) pair_alloc(smem_u32(&s_tmem));
        else tmem_alloc(smem_u32(&s_tmem));
    }
    for (int i = threadIdx.x; i < p.count * (int)(sizeof(Shape) / 4); i += TILE_THREADS)
        reinterpret_cast<u32*>(s_jobs)[i] = reinterpret_cast<const u32*>(p.job)[i];
    if (threadIdx.x == 0) {
        for (int s = 0; s < S::STAGES; ++s) bar_init(full + 8 * s, 1), bar_init(empty + 8 * s, 1);
        for (int s = 0; s < S::ACCS; ++s) bar_init(acc_full + 8 * s, 1), bar_init(acc_empty + 8 * s, TWO ? 16 : 8);
        bar_init(drained, 1);
        s_gave_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    if constexpr (TWO) cluster_barrier();  // the other block's barriers and tensor memory are there
    fence_after();
    const u32 tmem = __shfl_sync(0xffffffffu, s_tmem, 0);
    volatile int* gave_up = &s_gave_up;
    cbm::wait_before();
    int rank = blockIdx.x, stride = gridDim.x, side = 0;  // (side: which block of a pair)
    if constexpr (TWO) {
        asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(side));
        rank >>= 1, stride >>= 1;
    }
    auto wait = [&](u32 bar, u32 parity) { return warp_wait(bar, parity, gave_up, p.timeout); };
    // f(kind, the buffer X is in, whether it is the last product)
    auto each_product = [&](auto&& f) {
        u32 due = 0;
        for (int k = 0; k < steps; ++k)
            for (int kind = GRAM; kind <= APPLY; ++kind) {
                f((Kind)kind, k & 1, k + 1 == steps);
                due += gridDim.x;
                if (kind != APPLY || k + 1 < steps) all_blocks(p.arrived, due, gave_up, p.timeout, warp < PRODUCER, warp == PRODUCER);
            }
    };
    auto tiles_of = [&](Kind kind) { return kind == APPLY ? all_tiles : sym_tiles; };

    if (warp == PRODUCER) {
        const u32 first_full = TWO ? in_first(full) : full;
        u32 it = 0;
        bool ok = true;
        each_product([&](Kind kind, int from, bool) {
          for (int t = rank; t < tiles_of(kind) && ok; t += stride) {
            const Where w = tile_of<S::ROWS, BN>(s_jobs, kind, t);
            const Shape& q = s_jobs[w.job];
            const int depth = kind == GRAM ? q.n : q.m;
            const Maps& maps = p.map[w.job];
            const CUtensorMap* ma = kind == GRAM ? &maps.first_x[from] : kind == SQUARE ? &maps.first_a : &maps.first_b;
            const CUtensorMap* mb = kind == SQUARE ? &maps.second_a : &maps.second_x[from];
            const int row0 = S::ROWS * w.row + 128 * side, col0 = BN * w.col + 64 * side;
            for (int k = 0; k < depth; k += 64, ++it) {
                const u32 slot = it % S::STAGES, use = it / S::STAGES, at = smem + slot * S::STAGE;
                if (use > 0 && !(ok = wait(empty + 8 * slot, (use + 1) & 1))) break;
                // (what lies past the matrix comes as zeros; the first block of a pair answers for both)
                if (side == 0) expect(full + 8 * slot, TWO ? 2 * S::STAGE : S::STAGE);
                box_in<TWO>(at, ma, k, row0, w.matrix, first_full + 8 * slot);
                if (kind == APPLY) box_in<TWO>(at + S::A_BYTES, mb, col0, k, w.matrix, first_full + 8 * slot);
                else box_in<TWO>(at + S::A_BYTES, mb, k, col0, w.matrix, first_full + 8 * slot);
                __syncwarp();
            }
          }
        });
        // What was fetched has arrived before the block leaves, also where others have given up.
        // (The second block of a pair is told by the first, with the barrier at the end.)
        for (u32 back = 1; side == 0 && back <= (u32)S::STAGES && back <= it; ++back) {
            const u32 i = it - back;
            for (u32 spins = 0; spins < (1u << 22) && !bar_poll(full + 8 * (i % S::STAGES), (i / S::STAGES) & 1); ++spins) {
            }
        }
        __syncwarp();
    } else if (warp == ISSUER) {
        u32 it = 0;
        bool ok = true;
        each_product([&](Kind kind, int, bool) {
          const u32 both = idesc_half(S::ROWS, 2 * BN, kind == APPLY), one_term = idesc_half(S::ROWS, BN, kind == APPLY);
          for (int t = rank; t < tiles_of(kind) && ok && side == 0; t += stride) {
            const Where w = tile_of<S::ROWS, BN>(s_jobs, kind, t);
            const Shape& q = s_jobs[w.job];
            const int depth = kind == GRAM ? q.n : q.m;
            for (int k = 0; k < depth; k += 64, ++it) {
                const u32 slot = it % S::STAGES, use = it / S::STAGES, at = smem + slot * S::STAGE;
                const u32 as = it % S::ACCS, acc_use = it / S::ACCS, d = tmem + as * S::ACC_COLS;
                if (acc_use > 0 && !(ok = wait(acc_empty + 8 * as, (acc_use + 1) & 1))) break;
                if (!(ok = wait(full + 8 * slot, use & 1))) break;
                const u64 ah = desc_of(at), al = desc_of(at + 2 * BOX_BYTES);
                // (what lies past the last column of the contraction has been fetched as zeros)
                if (kind == APPLY) mma_chunk<TWO>(d, ah, al, desc_mn(at + S::A_BYTES), 2048 >> 4, both, one_term);
                else mma_chunk<TWO>(d, ah, al, desc_of(at + S::A_BYTES), 32 >> 4, both, one_term);
                if constexpr (TWO) {
                    commit_both(empty + 8 * slot);
                    commit_both(acc_full + 8 * as);
                } else {
                    commit(empty + 8 * slot);
                    commit(acc_full + 8 * as);
                }
            }
          }
        });
        if (!ok) {  // the MMAs under way end before the block frees its tensor memory
            if constexpr (TWO) commit_both(drained);
            else commit(drained);
            for (u32 spins = 0; spins < (1u << 20) && !bar_poll(drained, 0); ++spins) {
            }
            __syncwarp();
        }
    } else {
        const int quarter = warp & 3, half = warp >> 2;
        constexpr int EACH = BN / 2;  // columns of this warp
        float4* turn = reinterpret_cast<float4*>(smem_raw + (smem - smem_u32(smem_raw)) + S::STAGES * S::STAGE) + warp * (S::TURN / 16);
        u32 it = 0;
        bool ok = true;
        const bool any_low = __any_sync(0xffffffffu, __ldcg(p.any_low) != 0);
        if (threadIdx.x == 0) s_any_low = any_low;
        each_product([&](Kind kind, int from, bool last) {
          for (int t = rank; t < tiles_of(kind) && ok; t += stride) {
            const Where w = tile_of<S::ROWS, BN>(s_jobs, kind, t);
            const Shape& q = s_jobs[w.job];
            const int depth = kind == GRAM ? q.n : q.m, width = kind == APPLY ? q.n : q.m, ld = kind == APPLY ? q.ldx : q.lda;
            float sum[EACH];
#pragma unroll
            for (int i = 0; i < EACH; ++i) sum[i] = 0.f;
            for (int k = 0; k < depth; k += 64, ++it) {
                const u32 as = it % S::ACCS, use = it / S::ACCS;
                if (!(ok = wait(acc_full + 8 * as, use & 1))) break;
                const u32 at = tmem + as * S::ACC_COLS + half * (TWO ? 128 : EACH) + ((u32)(quarter * 32) << 16);
#pragma unroll
                for (int c = 0; c < EACH; c += 32) {
                    float r[2][32];
                    ld32(r[0], at + c);
                    ld32(r[1], at + 64 + c);
                    wait_ld();
#pragma unroll
                    for (int i = 0; i < 32; ++i) asm volatile("" : "+f"(r[0][i]), "+f"(r[1][i]));  // not before the wait
                    if (c + 32 == EACH) {
                        fence_before();
                        __syncwarp();
                        if (lane == 0) {
                            if constexpr (TWO) arrive_in_first(in_first(acc_empty + 8 * as));
                            else bar_arrive(acc_empty + 8 * as);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 32; i += 2) {
                        add2(r[0][i], r[0][i + 1], r[1][i], r[1][i + 1]);
                        add2(sum[c + i], sum[c + i + 1], r[0][i], r[0][i + 1]);
                    }
                }
            }
            if (!ok) break;
            const int m = q.m;
            const int64_t plane = (int64_t)m * ld, matrix = 2 * w.matrix * plane;
            __half* to = (kind == GRAM ? q.pa : kind == SQUARE ? q.pb : q.px[from ^ 1]) + matrix;
            const __half* more = (kind == SQUARE ? q.pa : q.px[from]) + matrix;
            const float factor = kind == SQUARE ? QUINTIC_C * UNSCALE : UNSCALE, more_factor = kind == SQUARE ? QUINTIC_B : QUINTIC_A;
            const bool result = kind == APPLY && last;
            const Matrix of = q.of;
            // 32 x 32 values at a time: as they were summed up a lane has a row; then it has eight neighbours of a row, four times.
            const int row0 = S::ROWS * w.row + 128 * side + 32 * quarter, row = row0 + (lane >> 2), eighth = 8 * (lane & 3);
            Terms add[EACH / 32][4];
            if (kind != GRAM) {  // (without a question about single ones, which would come one after the other; what lies outside is not used)
#pragma unroll
                for (int block = 0; block < EACH / 32; ++block) {
                    const __half* at = more + min(BN * w.col + half * EACH + 32 * block + eighth, ld - 8);
#pragma unroll
                    for (int i = 0; i < 4; ++i) add[block][i].load(at + (int64_t)min(row + 8 * i, m - 1) * ld, plane);
                }
            }
            // Four columns of a row lie together in shared memory, those of row r at (column / 4) ^ (r & 7) ^ 2 (r / 8): no two lanes meet in
            // a bank, by rows or by columns.
            const int by_row = (lane >> 2) * 8, swirl = lane >> 2;
#pragma unroll
            for (int block = 0; block < EACH / 32; ++block) {
                const int col0 = BN * w.col + half * EACH + 32 * block, col = col0 + eighth;
                if (row0 >= m || col0 >= width || (kind != APPLY && col0 < row0)) continue;  // (below the diagonal: written across)
#pragma unroll
                for (int c = 0; c < 8; ++c)
                    turn[lane * 8 + (c ^ (lane & 7) ^ (lane >> 3 << 1))] =
                        make_float4(sum[32 * block + 4 * c], sum[32 * block + 4 * c + 1], sum[32 * block + 4 * c + 2], sum[32 * block + 4 * c + 3]);
                __syncwarp();
                auto values = [&](int i, float(&v)[8]) {
                    const float4 x = turn[64 * i + by_row + ((eighth >> 2) ^ swirl ^ (2 * i))], y = turn[64 * i + by_row + (((eighth >> 2) + 1) ^ swirl ^ (2 * i))];
                    v[0] = factor * x.x, v[1] = factor * x.y, v[2] = factor * x.z, v[3] = factor * x.w;
                    v[4] = factor * y.x, v[5] = factor * y.y, v[6] = factor * y.z, v[7] = factor * y.w;
                    if (kind != GRAM) add[block][i].add_to(v, more_factor);
                };
                auto put = [&](int i, uint4 x, uint4 y) {
                    reinterpret_cast<uint4&>(turn[64 * i + by_row + ((eighth >> 2) ^ swirl ^ (2 * i))]) = x;
                    reinterpret_cast<uint4&>(turn[64 * i + by_row + (((eighth >> 2) + 1) ^ swirl ^ (2 * i))]) = y;
                };
                // the same, turned: eight neighbours of a column, of the rows from 8 (lane % 4) on
                auto turned_words = [&](int i, u32(&words)[8]) {
                    const int column = 8 * i + (lane >> 2);
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        words[j] = reinterpret_cast<const u32*>(turn)[(eighth + j) * 32 + (((column >> 2) ^ j ^ (2 * (lane & 3))) << 2) + (column & 3)];
                };
                const int r = row0 + eighth, c = col0 + (lane >> 2);
                if (!result) {
                    const bool across = kind != APPLY && col0 > row0;
                    __half* out = to + (int64_t)row * ld + col;
#pragma unroll
                    for (int i = 0; i < 4; ++i, out += 8 * ld) {
                        float v[8];
                        values(i, v);
                        const Terms t = terms_of(v);
                        if (row + 8 * i < m && col < width) t.store(out, plane);  // (the row's padding may be written over)
                        if (across) put(i, make_uint4(t.word(0), t.word(1), t.word(2), t.word(3)), make_uint4(t.word(4), t.word(5), t.word(6), t.word(7)));
                    }
                    if (across) {
                        __syncwarp();
                        out = to + (int64_t)c * ld + r;
#pragma unroll
                        for (int i = 0; i < 4; ++i, out += 8 * ld) {
                            u32 words[8];
                            turned_words(i, words);
                            Terms t;
#pragma unroll
                            for (int j = 0; j < 4; ++j) t.pair(j, words[2 * j], words[2 * j + 1]);
                            if (r < m && c + 8 * i < width) t.store(out, plane);
                        }
                    }
                } else if (!any_low || !__any_sync(0xffffffffu, __ldcg(&q.low[w.matrix]))) {  // (of the others the result comes at the end)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float v[8];
                        values(i, v);
                        if (q.turned) put(i, make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])), make_uint4(__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7])));
                        else if (row + 8 * i < m && col < width) of.write(w.matrix, row + 8 * i, col, min(8, width - col), v);
                    }
                    if (q.turned) {
                        __syncwarp();
#pragma unroll 1
                        for (int i = 0; i < 4; ++i) {
                            u32 words[8];
                            float v[8];
                            turned_words(i, words);
#pragma unroll
                            for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(words[j]);
                            if (r < m && c + 8 * i < width) of.write(w.matrix, c + 8 * i, r, min(8, m - r), v);
                        }
                    }
                }
                __syncwarp();
            }
          }
        });
    }
    fence_before();
    __syncthreads();
    if constexpr (TWO) cluster_barrier();  // nothing of the other block is under way here any more
    fence_after();
    if (warp == ISSUER) {
        if constexpr (TWO) pair_free(tmem);
        else tmem_free(tmem);
    }
    // Matrices that have to go another way, once nobody reads what lies in their place.  (Here, and not ahead of the others: a question about each
    // tile in the loops above costs all matrices 4 %.)
    if (!s_any_low) return;
    u32 due = (3 * steps - 1) * gridDim.x;
    const auto sync = [&] { all_blocks(p.arrived, due += gridDim.x, gave_up, p.timeout, false, false); };
    sync();
    plain_products<TWO ? 128 : 64>(p, s_jobs, -1, 0.0, steps, blockIdx.x, gridDim.x, reinterpret_cast<float*>(smem_raw + (smem - smem_u32(smem_raw))), sync);
}

// ---- small matrices -------------------------------------------------------------------------------
// Up to 128 x 1024: everything by a cluster of blocks that hold the matrix in shared memory, 128 columns each, as a product between
// global memory and back takes 4 us however small it is (64 x 500 57 us, as tiles of the other kernel 158; eight of 128 x 1 000 82 and
// 211).  A block adds up its columns' part of X X^T; the parts are exchanged through the
// cluster's shared memory, each block joining some rows for all; A A is computed by every block for itself, and B X is a matter of its
// own columns.  X serves both products as it lies: its rows are the contraction of one and the columns of the other.
constexpr int SMALL_THREADS = 512, SMALL_COLS = 128, SMALL_BLOCKS = 8;
constexpr int SMALL_SMEM = 3 * SMALL_ARRAY + 1024;

__device__ __forceinline__ void cluster_barrier_async() {
    asm volatile("fence.proxy.async;" ::: "memory");
    cluster_barrier();
    asm volatile("fence.proxy.async;" ::: "memory");
}
__device__ __forceinline__ u32 in_block(u32 local, int rank) {
    u32 r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(local), "r"(rank));
    return r;
}
// A factor that may lie outside fp32 where its products do not: a number between 1 and 2, rounded once, and two powers of two.
struct Scale {
    float rest, first, second;
    __device__ __forceinline__ Scale(double f) {
        int e = 0;
        rest = (float)(2.0 * frexp(f, &e));
        e = min(max(e - 1, -250), 250);
        first = exp2f((float)(e / 2)), second = exp2f((float)(e - e / 2));
        if (!(f > 0.0 && f < INFINITY)) rest = (float)f, first = second = 1.f;
    }
    __device__ __forceinline__ float of(float u) const { return u * first * rest * second; }
};
// D (+)= A B^T of one step, by one elected thread.
__device__ __forceinline__ void mma_one(u32 d, u64 a, u64 b, u32 idesc, bool add) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\tsetp.ne.u32 p, %4, 0;\n\telect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"((u32)add)
        : "memory");
}
// MN-major operand whose blocks of 64 columns lie `next` bytes apart.
__device__ __forceinline__ u64 desc_mn_of(u32 addr, u32 next) {
    return (u64)((addr & 0x3ffff) >> 4) | ((u64)(next >> 4) << 16) | ((u64)(1024 >> 4) << 32) | ((u64)1 << 46) | ((u64)2 << 61);
}

__global__ void __launch_bounds__(SMALL_THREADS, 1) small_kernel(const __grid_constant__ Jobs p, const int steps) {
    extern __shared__ unsigned char smem_raw[];
    __shared__ u64 s_bar;
    __shared__ u32 s_tmem;
    __shared__ int s_gave_up;
    __shared__ double s_part[SMALL_THREADS / 32], s_norm[SMALL_BLOCKS];
    __shared__ double s_low;  // the norm of a matrix that has low rows or columns, -1: it has none
    // largest across rows of the update, and how many are not 0; least of the largest of those with enough
    __shared__ u32 s_across[128], s_values[128], s_least, s_lows[SMALL_BLOCKS];
    const u32 smem = (smem_u32(smem_raw) + 1023) & ~1023u;
    unsigned char* const base = smem_raw + (smem - smem_u32(smem_raw));
    unsigned char *const xs = base, *const as = base + SMALL_ARRAY, *const bs = base + 2 * SMALL_ARRAY;
    float* const sums = reinterpret_cast<float*>(bs);  // [128][128] where B is not needed; four columns c of row r at (c / 4) ^ (r % 32)
    const u32 x0 = smem, a0 = smem + SMALL_ARRAY, b0 = smem + 2 * SMALL_ARRAY;
    const int lane = threadIdx.x & 31, warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
    const u32 bar = smem_u32(&s_bar);
    if (warp == 0) tmem_alloc(smem_u32(&s_tmem));
    if (threadIdx.x == 0) {
        bar_init(bar, 1);
        s_gave_up = 0;
        s_least = 0xffffffffu;
        s_low = -1.0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (threadIdx.x < 128) s_across[threadIdx.x] = s_values[threadIdx.x] = 0;
    fence_before();
    cluster_barrier();
    fence_after();
    const u32 tmem = __shfl_sync(0xffffffffu, s_tmem, 0);
    volatile int* gave_up = &s_gave_up;
    int rank, blocks;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(blocks));
    int job = 0, b = blockIdx.x / blocks;
    while (b >= p.job[job].batch) b -= p.job[job++].batch;
    const Shape& q = p.job[job];
    const Matrix of = q.of;
    const int m = q.m, n = q.n, active = (n + SMALL_COLS - 1) / SMALL_COLS, c0 = rank * SMALL_COLS, cols = min(max(n - c0, 0), SMALL_COLS);
    const bool turned = q.turned;
    cbm::wait_before();

    int by_terms = steps;
    // ---- momentum, norm, X
    auto at_sum = [&](int r, int c) -> float& { return sums[r * 128 + (((c >> 2) ^ (r & 31)) << 2) + (c & 3)]; };
    {
        double s = 0.0;
        const int slow = turned ? cols : m, fast = turned ? m : cols;  // (along the rows of the update as it lies)
        const float* const g = of.g + b * of.next_g + (turned ? c0 * of.ldg : c0);
        float* const mom = of.m ? of.m + (turned ? c0 * of.ldm : c0) : nullptr;
        constexpr int AT_ONCE = 2;  // rows, of four values a lane each, which are fetched together
        u32 least = 0xffffffffu, across[4] = {0, 0, 0, 0}, values[4] = {0, 0, 0, 0};
#pragma unroll 1
        for (int i0 = warp; i0 < slow; i0 += AT_ONCE * (SMALL_THREADS / 32)) {
            float u[AT_ONCE][4], mm[AT_ONCE][4];
#pragma unroll
            for (int h = 0; h < AT_ONCE; ++h)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int i = i0 + h * (SMALL_THREADS / 32), j = lane + 32 * e;
                    const bool on = i < slow && j < fast;
                    u[h][e] = fetch1(g + (on ? i * of.ldg + j : 0), on);
                    mm[h][e] = fetch1(mom + (on ? i * of.ldm + j : 0), on && mom);
                }
#pragma unroll
            for (int h = 0; h < AT_ONCE; ++h) {
                u32 most = 0, found = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int i = i0 + h * (SMALL_THREADS / 32), j = lane + 32 * e;
                    if (i >= slow || j >= fast) continue;
                    if (mom) {
                        const float next = p.momentum * mm[h][e] + u[h][e];
                        mom[i * of.ldm + j] = next;
                        u[h][e] = p.nesterov ? u[h][e] + p.momentum * next : next;
                    }
                    at_sum(turned ? j : i, turned ? i : j) = u[h][e];
                    s += (double)u[h][e] * u[h][e];
                    const u32 size = magnitude(u[h][e]), is = size != 0;
                    most = max(most, size), across[e] = max(across[e], size);
                    found += is, values[e] += is;
                }
                most = __reduce_max_sync(0xffffffffu, most);
                if (__reduce_add_sync(0xffffffffu, found) >= FEWEST) least = min(least, most);
            }
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (lane == 0) s_part[warp] = s, atomicMin(&s_least, least);
#pragma unroll
        for (int e = 0; e < 4; ++e) atomicMax(&s_across[lane + 32 * e], across[e]), atomicAdd(&s_values[lane + 32 * e], values[e]);
        __syncthreads();
        if (warp == 0) {
            least = s_least;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (s_values[lane + 32 * e] >= FEWEST) least = min(least, s_across[lane + 32 * e]);
            least = __reduce_min_sync(0xffffffffu, least);
        }
        if (threadIdx.x < blocks) {
            s = 0.0;
            for (int i = 0; i < SMALL_THREADS / 32; ++i) s += s_part[i];
            asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(in_block(smem_u32(&s_norm[rank]), threadIdx.x)), "d"(s) : "memory");
            asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(in_block(smem_u32(&s_lows[rank]), threadIdx.x)), "r"(least) : "memory");
        }
        cluster_barrier();
        s = 0.0;
        least = 0xffffffffu;
        for (int i = 0; i < blocks; ++i) s += s_norm[i], least = min(least, s_lows[i]);
        if (least < __float_as_uint(INFINITY) && (double)__uint_as_float(least) < (double)LOW * (sqrt(s) + (double)p.eps)) {
            if (threadIdx.x == 0) s_low = sqrt(s);
            by_terms = 0;  // (see the end)
        }
        const Scale scale((double)SCALE / (sqrt(s) + (double)p.eps));
#pragma unroll 1
        for (int i = threadIdx.x; i < 128 * 16; i += SMALL_THREADS) {  // eight values: row i / 16, columns from 8 (i % 16) on
            const int r = i >> 4, c = 8 * (i & 15);
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; j += 4) {
                const float4 u = *reinterpret_cast<const float4*>(&at_sum(r, c + j));  // (what lies outside is not used)
                v[j] = scale.of(u.x), v[j + 1] = scale.of(u.y), v[j + 2] = scale.of(u.z), v[j + 3] = scale.of(u.w);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = r < m && c + j < cols ? v[j] : 0.f;
            const Terms t = terms_of(v);
            unsigned char* to = xs + (c >> 6) * 2 * SLICE + swizzled(r, (c & 63) >> 3);
            *reinterpret_cast<uint4*>(to) = t.h;
            *reinterpret_cast<uint4*>(to + SLICE) = t.l;
        }
        // (rows of A past the last come to no block of several: they are, and stay, zero)
        for (int i = threadIdx.x; i < SMALL_ARRAY / 16; i += SMALL_THREADS) reinterpret_cast<uint4*>(as)[i] = make_uint4(0, 0, 0, 0);
        fence_async();
        __syncthreads();
    }

    // this thread's row, and its 32 columns: from `from` on of slice `half`
    const int quarter = warp & 3, half = warp >> 3, from = 32 * (warp >> 2 & 1), row = 32 * quarter + lane;
    const u32 mine = tmem + ((u32)(32 * quarter) << 16);
    u32 phase = 0;
    // all MMAs issued so far are done
    auto done = [&] {
        if (warp == 0) commit(bar);
        (void)warp_wait(bar, phase, gave_up, p.timeout);
        phase ^= 1;
    };
    // what accumulator columns `first` and `second` on hold of this warp's rows, added
    auto add_columns = [&](float(&sum)[32], u32 first, u32 second) {
        float r[32];
        ld32(sum, mine + first);
        ld32(r, mine + second);
        wait_ld();
#pragma unroll
        for (int i = 0; i < 32; ++i) asm volatile("" : "+f"(sum[i]), "+f"(r[i]));
#pragma unroll
        for (int i = 0; i < 32; i += 2) add2(sum[i], sum[i + 1], r[i], r[i + 1]);
    };
    // eight values of this thread's row, from column 8 k8 of the 64 columns of slice pair `of`
    auto load_terms = [&](const unsigned char* array, int k8) {
        Terms t;
        const unsigned char* at = array + half * 2 * SLICE + swizzled(row, k8);
        t.h = *reinterpret_cast<const uint4*>(at);
        t.l = *reinterpret_cast<const uint4*>(at + SLICE);
        return t;
    };
    auto store_terms = [&](unsigned char* array, int k8, const Terms& t) {
        unsigned char* at = array + half * 2 * SLICE + swizzled(row, k8);
        *reinterpret_cast<uint4*>(at) = t.h;
        *reinterpret_cast<uint4*>(at + SLICE) = t.l;
    };
    const u32 both = idesc_half(128, 256, false), one = idesc_half(128, 128, false);
    const int deep = (m + 63) / 64, wide = (cols + 63) / 64;  // slices of 64 of a contraction over rows, of this block's columns
#pragma unroll 1
    for (int k = 0; k < by_terms; ++k) {
        // ---- A = X X^T
        if (active > rank) {
            if (warp == 0)
                for (int i = 0; i < wide; ++i)
                    for (int s = 0; s < 4; ++s) {
                        const u32 at = x0 + i * 2 * SLICE + 32 * s;
                        mma_one(tmem, desc_of(at), desc_of(at), both, i + s > 0);
                        mma_one(tmem + 128, desc_of(at + SLICE), desc_of(at), one, true);
                    }
            done();
            {
                const int c = from;
                float sum[32];
                add_columns(sum, 64 * half + c, 128 + 64 * half + c);
#pragma unroll
                for (int i = 0; i < 32; i += 8) {
                    if (active == 1) {
                        float v[8];
#pragma unroll
                        for (int j = 0; j < 8; ++j) v[j] = UNSCALE * sum[i + j];
                        store_terms(as, (c + i) >> 3, terms_of(v));
                    } else {
#pragma unroll
                        for (int j = 0; j < 8; j += 4)
                            *reinterpret_cast<float4*>(&at_sum(row, 64 * half + c + i + j)) = make_float4(sum[i + j], sum[i + j + 1], sum[i + j + 2], sum[i + j + 3]);
                    }
                }
            }
            fence_before();
        }
        if (active > 1) {
            cluster_barrier();
            // This block's rows of the sum, for all, a warp to a row: what its lanes read and write in another block is contiguous (eight
            // values to a lane, whose two fetches leave gaps, took 5 600 cycles, one for each 16 bytes).
            const int rows = (m + active - 1) / active, c = 4 * lane, last = rank < active ? min(rows * rank + rows, m) : 0;
            for (int r = rows * rank + warp; r < last; r += SMALL_THREADS / 32) {
                // (all parts on their way together; in place of one that there is none of, this block's own, which is not added)
                const u32 at = smem_u32(&at_sum(r, c));
                float4 x[SMALL_BLOCKS];
#pragma unroll
                for (int i = 0; i < SMALL_BLOCKS; ++i)
                    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                                 : "=f"(x[i].x), "=f"(x[i].y), "=f"(x[i].z), "=f"(x[i].w)
                                 : "r"(in_block(at, i < active ? i : rank)));
                float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = 0; i < SMALL_BLOCKS; ++i)
                    if (i < active) v[0] += x[i].x, v[1] += x[i].y, v[2] += x[i].z, v[3] += x[i].w;
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] *= UNSCALE;
                const Terms t = terms_of(v);
                const u32 to = a0 + (c >> 6) * 2 * SLICE + swizzled(r, (c & 63) >> 3) + 2 * (c & 4);
                for (int i = 0; i < active; ++i) {
                    asm volatile("st.shared::cluster.v2.u32 [%0], {%1, %2};" ::"r"(in_block(to, i)), "r"(t.h.x), "r"(t.h.y) : "memory");
                    asm volatile("st.shared::cluster.v2.u32 [%0], {%1, %2};" ::"r"(in_block(to + SLICE, i)), "r"(t.l.x), "r"(t.l.y) : "memory");
                }
            }
            cluster_barrier_async();
        }
        if (active <= rank) continue;
        fence_async();
        __syncthreads();
        fence_after();
        // ---- B = b A + c A A
        if (warp == 0)
            for (int i = 0; i < deep; ++i)
                for (int s = 0; s < 4; ++s) {
                    const u32 at = a0 + i * 2 * SLICE + 32 * s;
                    mma_one(tmem, desc_of(at), desc_of(at), both, i + s > 0);
                    mma_one(tmem + 128, desc_of(at + SLICE), desc_of(at), one, true);
                }
        done();
        {
            const int c = from;
            float sum[32];
            add_columns(sum, 64 * half + c, 128 + 64 * half + c);
#pragma unroll
            for (int i = 0; i < 32; i += 8) {
                float v[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = QUINTIC_C * UNSCALE * sum[i + j];
                load_terms(as, (c + i) >> 3).add_to(v, QUINTIC_B);
                store_terms(bs, (c + i) >> 3, terms_of(v));
            }
        }
        fence_before();
        fence_async();
        __syncthreads();
        fence_after();
        // ---- X <- a X + B X: with [X_h | X_l] of each 64 columns behind one another, then B_l X_h into accumulators of its own
        if (warp == 0)
            for (int i = 0; i < deep; ++i)
                for (int s = 0; s < 4; ++s) {
                    const u32 a = b0 + i * 2 * SLICE + 32 * s, x = x0 + i * 64 * 128 + s * 16 * 128;
                    mma_one(tmem, desc_of(a), desc_mn_of(x, SLICE), idesc_half(128, 128 * wide, true), i + s > 0);
                    mma_one(tmem + 256, desc_of(a + SLICE), desc_mn_of(x, 2 * SLICE), idesc_half(128, 64 * wide, true), i + s > 0);
                }
        done();
        if (half < wide) {
            {
                const int c = from;
                float sum[32];
                add_columns(sum, 128 * half + c, 128 * half + 64 + c);
                {
                    float r[32];
                    ld32(r, mine + 256 + 64 * half + c);
                    wait_ld();
#pragma unroll
                    for (int i = 0; i < 32; ++i) asm volatile("" : "+f"(r[i]));
#pragma unroll
                    for (int i = 0; i < 32; i += 2) add2(sum[i], sum[i + 1], r[i], r[i + 1]);
                }
#pragma unroll
                for (int i = 0; i < 32; i += 8) {
                    float v[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[j] = UNSCALE * sum[i + j];
                    load_terms(xs, (c + i) >> 3).add_to(v, QUINTIC_A);
                    if (k + 1 < steps) {
                        store_terms(xs, (c + i) >> 3, terms_of(v));
                        continue;
                    }
                    const int col = c0 + 64 * half + c + i;
                    if (row >= m || col >= n) continue;
                    if (!turned) {
                        of.write(b, row, col, min(8, n - col), v);
                    } else {
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const float o[8] = {v[j]};
                            if (col + j < n) of.write(b, col + j, row, 1, o);
                        }
                    }
                }
            }
        }
        fence_before();
        fence_async();
        __syncthreads();
        fence_after();
    }
    if (s_gave_up && warp == 0)  // the MMAs under way end before the block frees its tensor memory
        for (u32 spins = 0; spins < (1u << 20) && !bar_poll(bar, phase ^ 1); ++spins) {
        }
    fence_before();
    __syncthreads();
    fence_after();
    if (warp == 0) tmem_free(tmem);
    if (s_low >= 0.0)
        plain_products<64>(p, &q, b, s_low, steps, rank, blocks, reinterpret_cast<float*>(xs), [] { cluster_barrier(); });
}

// ---- host -----------------------------------------------------------------------------------------
using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                            const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

Encode encoder() {
    static const Encode encode = [] {
        void* fn = nullptr;
        cudaDriverEntryPointQueryResult got;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &got) != cudaSuccess || got != cudaDriverEntryPointSuccess) {
            cudaGetLastError();
            fn = nullptr;
        }
        return reinterpret_cast<Encode>(fn);
    }();
    return encode;
}

bool describe(CUtensorMap* map, const __half* p, int rows, int cols, int ld, int batch, int box_rows) {
    const Encode encode = encoder();
    if (!encode) return false;
    const cuuint64_t size[4] = {(cuuint64_t)cols, (cuuint64_t)rows, 2, (cuuint64_t)batch};
    const cuuint64_t pitch[3] = {(cuuint64_t)ld * 2, (cuuint64_t)ld * 2 * rows, (cuuint64_t)ld * 4 * rows};
    const cuuint32_t box[4] = {64, (cuuint32_t)box_rows, 2, 1}, step[4] = {1, 1, 1, 1};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<__half*>(p), size, pitch, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int64_t pad(int64_t bytes) { return (bytes + 255) / 256 * 256; }

// Workspace of a job, and where its arrays lie in it.
int64_t lay_out(Shape* q, int rows, int cols, int batch, unsigned char* at) {
    const int m = rows < cols ? rows : cols, n = rows < cols ? cols : rows;
    const int ldx = (n + 7) / 8 * 8, lda = (m + 7) / 8 * 8;
    const int64_t x = pad((int64_t)4 * batch * m * ldx), a = pad((int64_t)4 * batch * m * lda), parts = pad((int64_t)8 * batch * PARTS),
                  low = pad((int64_t)4 * batch);
    if (q) {
        q->m = m, q->n = n, q->ldx = ldx, q->lda = lda, q->turned = rows > cols, q->batch = batch;
        q->px[0] = reinterpret_cast<__half*>(at), q->px[1] = reinterpret_cast<__half*>(at + x);
        q->pa = reinterpret_cast<__half*>(at + 2 * x), q->pb = reinterpret_cast<__half*>(at + 2 * x + a);
        q->parts = reinterpret_cast<double*>(at + 2 * x + 2 * a);
        q->low = reinterpret_cast<int*>(at + 2 * x + 2 * a + parts);
    }
    return 2 * x + 2 * a + parts + low;
}

template <Mode MODE>
int tiles_sym(int m) {
    using S = Sizes<MODE>;
    int t = 0;
    for (int r = 0; r * S::ROWS < m; ++r) t += (m + S::BN - 1) / S::BN - r * (S::ROWS / S::BN);
    return t;
}
template <Mode MODE>
int tiles_all(int m, int n) {
    using S = Sizes<MODE>;
    return (m + S::ROWS - 1) / S::ROWS * ((n + S::BN - 1) / S::BN);
}

template <Mode MODE>
int products(const char* who, Jobs& p, int steps, const cbm::Stream& on) {
    constexpr auto kernel = product_kernel<MODE>;
    if (!allow_smem<kernel>(Sizes<MODE>::SMEM)) return cbm::fail(CBM_B200_ERR_CUDA, std::string(who) + ": no room in shared memory");
    int sym = 0, all = 0, matrices = 0, blocks = 1;
    for (int i = 0; i < p.count; ++i) {
        Shape& q = p.job[i];
        q.tiles_sym = tiles_sym<MODE>(q.m), q.tiles_all = tiles_all<MODE>(q.m, q.n);
        sym += q.tiles_sym * q.batch, all += q.tiles_all * q.batch, matrices += q.batch;
        const int64_t tiles = (int64_t)((q.m + 31) / 32) * ((q.n + 31) / 32);
        if (tiles > blocks) blocks = (int)(tiles < 2048 ? tiles : 2048);
    }
    cbm::launch_next(norm_kernel, dim3(PARTS, matrices), THREADS, 0, on, p);
    cbm::launch_next(start_kernel, dim3(blocks, matrices), THREADS, 0, on, p);
    const int cluster = MODE == PAIR ? 2 : 1, most = sm_count() / cluster, wanted = sym > all ? sym : all;
    cudaLaunchAttribute attrs[2] = {};
    attrs[0].id = cudaLaunchAttributeCooperative;
    attrs[0].val.cooperative = 1;
    attrs[1].id = cudaLaunchAttributeClusterDimension;
    attrs[1].val.clusterDim.x = cluster;
    attrs[1].val.clusterDim.y = attrs[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3((wanted < most ? wanted : most) * cluster);
    config.blockDim = dim3(TILE_THREADS);
    config.dynamicSmemBytes = Sizes<MODE>::SMEM;
    config.stream = on.s;
    config.attrs = attrs;
    config.numAttrs = MODE == PAIR ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&config, kernel, p, sym, all, steps);
    if (e != cudaSuccess) (void)cudaGetLastError();
    return e == cudaSuccess ? CBM_B200_OK : cbm::fail(CBM_B200_ERR_CUDA, std::string(who) + ": " + cudaGetErrorString(e));
}

bool is_small(int m, int n) { return m <= 128 && n <= SMALL_COLS * SMALL_BLOCKS; }

int small_ones(const char* who, Jobs& p, int steps, const cbm::Stream& on) {
    if (!allow_smem<small_kernel>(SMALL_SMEM)) return cbm::fail(CBM_B200_ERR_CUDA, std::string(who) + ": no room in shared memory");
    int matrices = 0, blocks = 1;
    for (int i = 0; i < p.count; ++i) {
        matrices += p.job[i].batch;
        while (blocks * SMALL_COLS < p.job[i].n) blocks *= 2;
    }
    cudaLaunchAttribute attrs[2] = {};
    attrs[0].id = cudaLaunchAttributeClusterDimension;
    attrs[0].val.clusterDim.x = blocks;
    attrs[0].val.clusterDim.y = attrs[0].val.clusterDim.z = 1;
    attrs[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[1].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(matrices * blocks);
    config.blockDim = dim3(SMALL_THREADS);
    config.dynamicSmemBytes = SMALL_SMEM;
    config.stream = on.s;
    config.attrs = attrs;
    config.numAttrs = on.captured ? 1 : 2;
    const cudaError_t e = cudaLaunchKernelEx(&config, small_kernel, p, steps);
    if (e != cudaSuccess) (void)cudaGetLastError();
    return e == cudaSuccess ? CBM_B200_OK : cbm::fail(CBM_B200_ERR_CUDA, std::string(who) + ": " + cudaGetErrorString(e));
}

int run(const char* who, Jobs& p, bool small, int steps, void* stream) {
    if (int rc = check_timeout(who)) return rc;
    p.timeout = timeout_word();
    const cbm::Stream on(static_cast<cudaStream_t>(stream));
    if (small) return small_ones(who, p, steps, on);
    int64_t pairs = 0;
    for (int i = 0; i < p.count; ++i) {
        Shape& q = p.job[i];
        Maps& map = p.map[i];
        bool done = describe(&map.first_a, q.pa, q.m, q.m, q.lda, q.batch, 128) && describe(&map.second_a, q.pa, q.m, q.m, q.lda, q.batch, 64) &&
                    describe(&map.first_b, q.pb, q.m, q.m, q.lda, q.batch, 128);
        for (int k = 0; k < 2; ++k)
            done = done && describe(&map.first_x[k], q.px[k], q.m, q.n, q.ldx, q.batch, 128) && describe(&map.second_x[k], q.px[k], q.m, q.n, q.ldx, q.batch, 64);
        if (!done)
            return cbm::fail(CBM_B200_ERR_CUDA, std::string(who) + ": no tensor map for its operands");
        pairs += (int64_t)q.batch * tiles_sym<PAIR>(q.m);
    }
    // Pairs of blocks where there are tiles of 256 x 128 for half of them at least, else single ones (square: 900 single 260 us, pairs 322;
    // 1 100 336 and 334; 1 500 551 and 418; 2 048 x 4 096 1 458 and 1 135).
    const int rc = pairs * 4 >= sm_count() ? products<PAIR>(who, p, steps, on) : products<SINGLE>(who, p, steps, on);
    if (rc) return rc;
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? CBM_B200_OK : cbm::fail(CBM_B200_ERR_CUDA, std::string(who) + ": " + cudaGetErrorString(e));
}

constexpr int HEAD = 256;  // of a workspace: the count of blocks, and whether a matrix has low rows or columns
constexpr int MAX_SIDE = 1 << 16, MAX_BATCH = 32768;  // (tiles are counted in 31 bits, matrices in a grid's second dimension)

}  // namespace

extern "C" int64_t cbm_b200_orthogonalise_workspace(int32_t batch, int32_t rows, int32_t cols) {
    return batch > 0 && rows > 0 && cols > 0 ? HEAD + lay_out(nullptr, rows, cols, batch, nullptr) : 0;
}

extern "C" int cbm_b200_orthogonalise(const float* u, int64_t ldu, int64_t next_u, float* out, int64_t ldout, int64_t next_out, int32_t batch,
                                      int32_t rows, int32_t cols, int32_t steps, float eps, void* workspace, int64_t workspace_bytes,
                                      void* stream) {
    if (batch < 0 || rows < 0 || cols < 0 || rows > MAX_SIDE || cols > MAX_SIDE || batch > MAX_BATCH || steps < 1 || steps > CBM_B200_MAX_STEPS ||
        ldu < cols || ldout < cols || !(eps >= 0.f))
        return cbm::fail(CBM_B200_ERR_ARG, "orthogonalise: bad sizes");
    if (batch == 0 || rows == 0 || cols == 0) return CBM_B200_OK;
    if (!u || !out || !workspace || reinterpret_cast<uintptr_t>(workspace) % 256) return cbm::fail(CBM_B200_ERR_ARG, "orthogonalise: NULL argument, or workspace not at 256 bytes");
    if (workspace_bytes < cbm_b200_orthogonalise_workspace(batch, rows, cols)) return cbm::fail(CBM_B200_ERR_ARG, "orthogonalise: workspace too small");
    Jobs p{};
    p.count = 1, p.eps = eps;
    p.arrived = static_cast<u32*>(workspace), p.any_low = static_cast<int*>(workspace) + 1;
    lay_out(&p.job[0], rows, cols, batch, static_cast<unsigned char*>(workspace) + HEAD);
    p.job[0].of = Matrix{u, nullptr, nullptr, out, ldu, 0, 0, ldout, next_u, next_out, 0.f, 0.f};
    return run("orthogonalise", p, is_small(p.job[0].m, p.job[0].n), steps, stream);
}

extern "C" int64_t cbm_b200_orthogonal_step_workspace(const cbm_b200_update_of* of, int32_t count) {
    int64_t all = 0;
    for (int i = 0; of && i < count; ++i)
        if (of[i].rows > 0 && of[i].cols > 0) all += lay_out(nullptr, of[i].rows, of[i].cols, 1, nullptr);
    return all ? HEAD + all : 0;
}

extern "C" int cbm_b200_orthogonal_step(const cbm_b200_update_of* of, int32_t count, float lr, float momentum, int32_t nesterov,
                                        float weight_decay, int32_t steps, float eps, void* workspace, int64_t workspace_bytes, void* stream) {
    if (count < 0 || (count && !of) || steps < 1 || steps > CBM_B200_MAX_STEPS || !(eps >= 0.f))
        return cbm::fail(CBM_B200_ERR_ARG, "orthogonal_step: bad arguments");
    for (int i = 0; i < count; ++i) {
        const cbm_b200_update_of& u = of[i];
        if (u.rows < 0 || u.cols < 0 || u.rows > MAX_SIDE || u.cols > MAX_SIDE || u.ldw < u.cols || u.ldg < u.cols || u.ldm < u.cols)
            return cbm::fail(CBM_B200_ERR_ARG, "orthogonal_step: bad sizes");
        if (u.rows && u.cols && (!u.w || !u.g || !u.m)) return cbm::fail(CBM_B200_ERR_ARG, "orthogonal_step: NULL argument");
    }
    const int64_t need = cbm_b200_orthogonal_step_workspace(of, count);
    if (need && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 256 || workspace_bytes < need))
        return cbm::fail(CBM_B200_ERR_ARG, "orthogonal_step: workspace too small, or not at 256 bytes");
    unsigned char* at = static_cast<unsigned char*>(workspace) + HEAD;
    // All matrices side by side: by clusters where all are small, else small ones among the others, whose products take longer anyway (one
    // after the other, 256 x 100, 256 x 256 and 47 x 256 took 213 us, side by side 147).
    bool small = true;
    for (int i = 0; i < count; ++i)
        small = small && (of[i].rows < of[i].cols ? is_small(of[i].rows, of[i].cols) : is_small(of[i].cols, of[i].rows));
    for (int i = 0; i < count;) {
        Jobs p{};
        p.eps = eps, p.momentum = momentum, p.nesterov = nesterov, p.arrived = static_cast<u32*>(workspace);
        p.any_low = static_cast<int*>(workspace) + 1;
        for (; i < count && p.count < MAX_JOBS; ++i) {
            const cbm_b200_update_of& u = of[i];
            if (u.rows == 0 || u.cols == 0) continue;
            Shape& q = p.job[p.count++];
            at += lay_out(&q, u.rows, u.cols, 1, at);
            const double tall = u.rows > u.cols ? std::sqrt((double)u.rows / u.cols) : 1.0;
            q.of = Matrix{u.g, u.m, u.w, nullptr, u.ldg, u.ldm, u.ldw, 0, 0, 0, (float)(lr * tall), (float)(1.0 - (double)lr * weight_decay)};
        }
        if (p.count)
            if (int rc = run("orthogonal_step", p, small, steps, stream)) return rc;
    }
    return CBM_B200_OK;
}
