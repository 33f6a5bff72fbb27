// Orthogonalised updates by Newton-Schulz products on the 5th-generation tensor cores (sm_100a), fp32-accurate.
//
// X = U / (|U| + eps), turned so that it is no taller than wide; then, `steps` times,
//   A = X X^T,  B = b A + c A A,  X <- a X + B X
// with the quintic (a, b, c) that the Muon optimiser publishes: every singular value is led to between 0.68 and 1.21.
//
// Precision: no entry of X, A or B exceeds 2.9, since none of their singular values does (X stays below 1.21).  So each is kept as
// two fp16 terms of 2^12 times its value, h = fp16(v), l = fp16(v - h): 22 bits, down to 2^-37 of the largest, where fp16 ends.  A
// product takes three fp16 MMAs, h h + h l + l h; l l is below 2^-22 of it.  (The dense maps, whose operands may have any
// exponent, need three bf16 terms and six products.)  Against float64: 500 x 777 0.6 to 0.8e-6 of the result, where torch's fp32 products
// give 2.4e-6.  As in cbm_map.cuh, an accumulator holds 64 columns of a contraction, the small products first, and is added to sums in
// registers, because the tensor cores cut off towards zero at every step.
//
// Work: m (m + 1) n + m^2 (m + 1) + 2 m^2 n a step, as A and A A are symmetric: only tiles that reach the upper triangle are computed,
// and the other half is written with them.
//
// One kernel, three kinds of products.  A block holds a tile of 128 x BN: one warp fetches both operands' terms by TMA (64 x 64
// boxes, 128-byte swizzled), one issues the MMAs, eight add up and write the result, split again, with the term that is added to it.
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

struct Matrix {
    const float* g;  // update, or gradient
    float *m, *w;    // momentum and weights, or NULL
    float* out;      // result, where there are no weights
    int64_t ldg, ldm, ldw, ldout, next_g, next_out;
    float lr, keep;
};

// Matrices of one shape: a stack, or one weight of a list.
struct Job {
    CUtensorMap x[2], a, b;    // [batch][2 terms][rows][columns], boxes of 64 x 64
    __half *px[2], *pa, *pb;
    double* parts;             // [batch][PARTS]
    Matrix of;
    int m, n, ldx, lda, turned, batch;
    int tiles_sym, tiles_all;  // of one matrix: that reach the upper triangle of A, of X
};

struct Jobs {
    Job job[MAX_JOBS];
    int count;
    float momentum, eps;
    int nesterov;
    int* timeout;
};

enum Kind { GRAM, SQUARE, APPLY };

// ---- start ----------------------------------------------------------------------------------------
__device__ __forceinline__ float update_at(const Jobs& p, const Job& q, int64_t b, int i, int j) {
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
    const Job& q = p.job[j];
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
    }
}

__device__ __forceinline__ void split(float v, __half& h, __half& l) {
    h = __float2half_rn(v);
    l = __float2half_rn(v - __half2float(h));
}

// X, split: 32 x 32 values to a block, through shared memory where it is turned.  Block x: a tile (of the largest job), y: a matrix.
__global__ void __launch_bounds__(THREADS) start_kernel(const __grid_constant__ Jobs p) {
    __shared__ float turn[32][33];
    cbm::wait_before();
    int j = 0, b = blockIdx.y;
    while (b >= p.job[j].batch) b -= p.job[j++].batch;
    const Job& q = p.job[j];
    const int across = (q.n + 31) / 32, tiles = across * ((q.m + 31) / 32), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    double s = 0.0;
    for (int i = 0; i < PARTS; i += 32) s += q.parts[b * PARTS + i + lane];
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    const double scale = (double)SCALE / (sqrt(s) + (double)p.eps);
    const int64_t plane = (int64_t)q.m * q.ldx;
    __half* x = q.px[0] + 2 * b * plane;
    for (int t = blockIdx.x; t < tiles; t += gridDim.x) {
        const int r0 = t / across * 32, c0 = t % across * 32;
        if (q.turned) {
            __syncthreads();
            for (int i = warp; i < 32; i += THREADS / 32)
                if (c0 + i < q.n && r0 + lane < q.m) turn[i][lane] = update_at(p, q, b, c0 + i, r0 + lane);
            __syncthreads();
        }
        for (int i = warp; i < 32; i += THREADS / 32)
            if (r0 + i < q.m && c0 + lane < q.n) {
                const float u = q.turned ? turn[lane][i] : update_at(p, q, b, r0 + i, c0 + lane);
                __half h, l;
                split((float)((double)u * scale), h, l);
                const int64_t at = (int64_t)(r0 + i) * q.ldx + c0 + lane;
                x[at] = h;
                x[at + plane] = l;
            }
    }
}

// ---- products -------------------------------------------------------------------------------------
template <int BN>
struct Shape {
    static constexpr int STAGES = BN == 64 ? 4 : 3;
    static constexpr int A_BYTES = 4 * BOX_BYTES;             // 2 terms of 128 x 64
    static constexpr int B_TERM = BN / 64 * BOX_BYTES;
    static constexpr int STAGE = A_BYTES + 2 * B_TERM;
    static constexpr int SMEM = STAGES * STAGE + 1024;
    static constexpr int ACCS = 4;                             // accumulators of BN columns
};

// D[128, N] (+)= A[128, 16] B[16, N], both in shared memory.
__device__ __forceinline__ void mma_ss(u32 d, u64 a, u64 b, u32 idesc, bool add) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\tsetp.ne.u32 p, %4, 0;\n\telect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"((u32)add)
        : "memory");
}
// fp32 accumulator, fp16 operands, M = 128; bit 16: the second operand is MN-major.
__host__ __device__ constexpr u32 idesc_half(u32 n, bool mn_major) { return (1u << 4) | ((u32)mn_major << 16) | ((n >> 3) << 17) | ((128u >> 4) << 24); }
// MN-major operand of 64-wide, 128-byte swizzled blocks: 8 steps of the contraction are 1024 bytes, the next 64 columns a box further on.
__device__ __forceinline__ u64 desc_mn(u32 addr) {
    return (u64)((addr & 0x3ffff) >> 4) | ((u64)(BOX_BYTES >> 4) << 16) | ((u64)(1024 >> 4) << 32) | ((u64)1 << 46) | ((u64)2 << 61);
}

__device__ __forceinline__ void box_in(u32 to, const CUtensorMap* map, int col, int row, int term, int matrix, u32 bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(to),
                 "l"(map), "r"(col), "r"(row), "r"(term), "r"(matrix), "r"(bar)
                 : "memory");
}

struct Where {
    int job, matrix, row, col;  // tile: rows from 128 row, columns from BN col
};
// The tile with running number t of a kind of product.
template <int BN>
__device__ __forceinline__ Where tile_of(const Jobs& p, Kind kind, int t) {
    Where w{0, 0, 0, 0};
    for (;; ++w.job) {
        const Job& q = p.job[w.job];
        const int each = kind == APPLY ? q.tiles_all : q.tiles_sym, all = each * q.batch;
        if (t >= all) {
            t -= all;
            continue;
        }
        w.matrix = t / each;
        t -= w.matrix * each;
        const int across = ((kind == APPLY ? q.n : q.m) + BN - 1) / BN;
        if (kind == APPLY) {
            // down the columns first: neighbouring blocks share X's columns, and B is small
            const int down = (q.m + 127) / 128;
            w.col = t / down, w.row = t % down;
        } else {
            for (int left = across; t >= left; left = across - w.row * (128 / BN)) t -= left, ++w.row;
            w.col = w.row * (128 / BN) + t;
        }
        return w;
    }
}

__device__ __forceinline__ void halves8(const __half* p, float (&v)[8], float f) {
    const uint4 w = __ldcg(reinterpret_cast<const uint4*>(p));
    const u32 q[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&q[i]));
        v[2 * i] += f * t.x, v[2 * i + 1] += f * t.y;
    }
}

template <int BN>
__global__ void __launch_bounds__(TILE_THREADS, 1) product_kernel(const __grid_constant__ Jobs p, const Kind kind, const int from, const int tiles,
                                                                  const bool last) {
    using S = Shape<BN>;
    extern __shared__ unsigned char smem_raw[];
    __shared__ u64 s_bar[2 * S::STAGES + 2 * S::ACCS + 1];
    __shared__ u32 s_tmem;
    __shared__ int s_gave_up;
    const u32 smem = (smem_u32(smem_raw) + 1023) & ~1023u;
    const int lane = threadIdx.x & 31, warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
    const u32 full = smem_u32(s_bar), empty = full + 8 * S::STAGES, acc_full = empty + 8 * S::STAGES, acc_empty = acc_full + 8 * S::ACCS,
              drained = acc_empty + 8 * S::ACCS;
    if (warp == ISSUER) tmem_alloc(smem_u32(&s_tmem));
    if (threadIdx.x == 0) {
        for (int s = 0; s < S::STAGES; ++s) bar_init(full + 8 * s, 1), bar_init(empty + 8 * s, 1);
        for (int s = 0; s < S::ACCS; ++s) bar_init(acc_full + 8 * s, 1), bar_init(acc_empty + 8 * s, 8);
        bar_init(drained, 1);
        s_gave_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const u32 tmem = __shfl_sync(0xffffffffu, s_tmem, 0);
    volatile int* gave_up = &s_gave_up;
    cbm::wait_before();

    if (warp == PRODUCER) {
        u32 it = 0;
        bool ok = true;
        for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
            const Where w = tile_of<BN>(p, kind, t);
            const Job& q = p.job[w.job];
            const int depth = kind == GRAM ? q.n : q.m, width = kind == APPLY ? q.n : q.m;
            const CUtensorMap *ma = kind == GRAM ? &q.x[from] : kind == SQUARE ? &q.a : &q.b, *mb = kind == SQUARE ? &q.a : &q.x[from];
            // boxes that lie past the matrix are left out: their rows and columns of the tile are not written
            const int boxes_a = q.m - 128 * w.row > 64 ? 2 : 1, boxes_b = min((width - BN * w.col + 63) / 64, BN / 64);
            for (int k = 0; k < depth; k += 64, ++it) {
                const u32 slot = it % S::STAGES, use = it / S::STAGES, bar = full + 8 * slot, at = smem + slot * S::STAGE;
                if (use > 0 && !(ok = warp_wait(empty + 8 * slot, (use + 1) & 1, gave_up, p.timeout))) break;
                if (lane == 0) {
                    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(2 * (boxes_a + boxes_b) * BOX_BYTES) : "memory");
                    for (int term = 0; term < 2; ++term) {
                        for (int i = 0; i < boxes_a; ++i) box_in(at + (2 * term + i) * BOX_BYTES, ma, k, 128 * w.row + 64 * i, term, w.matrix, bar);
                        for (int i = 0; i < boxes_b; ++i) {
                            const u32 to = at + S::A_BYTES + term * S::B_TERM + i * BOX_BYTES;
                            if (kind == APPLY) box_in(to, mb, BN * w.col + 64 * i, k, term, w.matrix, bar);
                            else box_in(to, mb, k, BN * w.col + 64 * i, term, w.matrix, bar);
                        }
                    }
                }
                __syncwarp();
            }
        }
        // What was fetched has arrived before the block leaves, also where others have given up.
        for (u32 back = 1; back <= (u32)S::STAGES && back <= it; ++back) {
            const u32 i = it - back;
            for (u32 spins = 0; spins < (1u << 22) && !bar_poll(full + 8 * (i % S::STAGES), (i / S::STAGES) & 1); ++spins) {
            }
        }
        __syncwarp();
    } else if (warp == ISSUER) {
        const u32 idesc = idesc_half(BN, kind == APPLY);
        u32 it = 0;
        bool ok = true;
        for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
            const Where w = tile_of<BN>(p, kind, t);
            const Job& q = p.job[w.job];
            const int depth = kind == GRAM ? q.n : q.m;
            for (int k = 0; k < depth; k += 64, ++it) {
                const u32 slot = it % S::STAGES, use = it / S::STAGES, at = smem + slot * S::STAGE;
                const u32 as = it % S::ACCS, acc_use = it / S::ACCS, d = tmem + as * BN;
                if (acc_use > 0 && !(ok = warp_wait(acc_empty + 8 * as, (acc_use + 1) & 1, gave_up, p.timeout))) break;
                if (!(ok = warp_wait(full + 8 * slot, use & 1, gave_up, p.timeout))) break;
                const int steps = min(4, (depth - k + 15) / 16);
                bool add = false;
#pragma unroll
                for (int pass = 0; pass < 3; ++pass) {  // l h, h l, h h
                    const u32 a = at + (pass == 0 ? 2 * BOX_BYTES : 0), b = at + S::A_BYTES + (pass == 1 ? S::B_TERM : 0);
                    for (int s = 0; s < steps; ++s) {
                        mma_ss(d, desc_of(a + 32 * s), kind == APPLY ? desc_mn(b + 2048 * s) : desc_of(b + 32 * s), idesc, add);
                        add = true;
                    }
                }
                commit(empty + 8 * slot);
                commit(acc_full + 8 * as);
            }
        }
        if (!ok) {  // the MMAs under way end before the block frees its tensor memory
            commit(drained);
            for (u32 spins = 0; spins < (1u << 20) && !bar_poll(drained, 0); ++spins) {
            }
            __syncwarp();
        }
    } else {
        const int quarter = warp & 3, half = warp >> 2;
        constexpr int EACH = BN / 2;  // columns of this warp
        u32 it = 0;
        for (int t = blockIdx.x; t < tiles; t += gridDim.x) {
            const Where w = tile_of<BN>(p, kind, t);
            const Job& q = p.job[w.job];
            const int depth = kind == GRAM ? q.n : q.m, width = kind == APPLY ? q.n : q.m, ld = kind == APPLY ? q.ldx : q.lda;
            float sum[EACH];
#pragma unroll
            for (int i = 0; i < EACH; ++i) sum[i] = 0.f;
            bool ok = true;
            for (int k = 0; k < depth; k += 64, ++it) {
                const u32 as = it % S::ACCS, use = it / S::ACCS;
                if (!(ok = warp_wait(acc_full + 8 * as, use & 1, gave_up, p.timeout))) break;
                const u32 at = tmem + as * BN + half * EACH + ((u32)(quarter * 32) << 16);
#pragma unroll
                for (int c = 0; c < EACH; c += 16) {
                    float r[16];
                    asm volatile(
                        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                        : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]), "=f"(r[9]),
                          "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15])
                        : "r"(at + c));
                    wait_ld();
#pragma unroll
                    for (int i = 0; i < 16; ++i) asm volatile("" : "+f"(r[i]));  // not before the wait
#pragma unroll
                    for (int i = 0; i < 16; i += 2) add2(sum[c + i], sum[c + i + 1], r[i], r[i + 1]);
                }
                fence_before();
                __syncwarp();
                if (lane == 0) bar_arrive(acc_empty + 8 * as);
            }
            if (!ok) break;
            const int row = 128 * w.row + 32 * quarter + lane, col0 = BN * w.col + half * EACH;
            const int64_t plane = (int64_t)q.m * ld, matrix = 2 * w.matrix * plane;
            __half* to = (kind == GRAM ? q.pa : kind == SQUARE ? q.pb : q.px[from ^ 1]) + matrix + (int64_t)row * ld;
            const __half* more = (kind == SQUARE ? q.pa : q.px[from]) + matrix + (int64_t)row * ld;
#pragma unroll
            for (int c = 0; c < EACH; c += 8) {
                const int col = col0 + c;
                if (row >= q.m || col >= width) break;
                if (kind != APPLY && col + 8 <= row) continue;  // below the diagonal: written by the tile above it
                float v[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = sum[c + i] * (kind == SQUARE ? QUINTIC_C * UNSCALE : UNSCALE);
                if (kind != GRAM) {
                    const float f = kind == SQUARE ? QUINTIC_B : QUINTIC_A;
                    halves8(more + col, v, f);
                    halves8(more + plane + col, v, f);
                }
                if (kind == APPLY && last) {
                    const Matrix& o = q.of;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        if (col + i >= q.n) break;
                        const int64_t r = q.turned ? col + i : row, s = q.turned ? row : col + i;
                        if (o.w) o.w[r * o.ldw + s] = o.keep * o.w[r * o.ldw + s] - o.lr * (v[i] * UNSCALE);
                        else o.out[w.matrix * o.next_out + r * o.ldout + s] = v[i] * UNSCALE;
                    }
                    continue;
                }
                __half h[8], l[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) split(v[i], h[i], l[i]);
                if (kind == APPLY || col >= row) {  // (the row's padding may be written over)
                    *reinterpret_cast<uint4*>(to + col) = *reinterpret_cast<const uint4*>(h);
                    *reinterpret_cast<uint4*>(to + plane + col) = *reinterpret_cast<const uint4*>(l);
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (col + i >= row) to[col + i] = h[i], to[plane + col + i] = l[i];
                }
                if (kind != APPLY) {
                    __half* across = (kind == GRAM ? q.pa : q.pb) + matrix + row;
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (col + i > row && col + i < q.m) across[(int64_t)(col + i) * ld] = h[i], across[plane + (int64_t)(col + i) * ld] = l[i];
                }
            }
            __syncwarp();
        }
    }
    fence_before();
    __syncthreads();
    fence_after();
    if (warp == ISSUER) tmem_free(tmem);
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

bool describe(CUtensorMap* map, const __half* p, int rows, int cols, int ld, int batch) {
    const Encode encode = encoder();
    if (!encode) return false;
    const cuuint64_t size[4] = {(cuuint64_t)cols, (cuuint64_t)rows, 2, (cuuint64_t)batch};
    const cuuint64_t pitch[3] = {(cuuint64_t)ld * 2, (cuuint64_t)ld * 2 * rows, (cuuint64_t)ld * 4 * rows};
    const cuuint32_t box[4] = {64, 64, 1, 1}, step[4] = {1, 1, 1, 1};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<__half*>(p), size, pitch, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int64_t pad(int64_t bytes) { return (bytes + 255) / 256 * 256; }

// Workspace of a job, and where its arrays lie in it.
int64_t lay_out(Job* q, int rows, int cols, int batch, unsigned char* at) {
    const int m = rows < cols ? rows : cols, n = rows < cols ? cols : rows;
    const int ldx = (n + 7) / 8 * 8, lda = (m + 7) / 8 * 8;
    const int64_t x = pad((int64_t)4 * batch * m * ldx), a = pad((int64_t)4 * batch * m * lda), parts = pad((int64_t)8 * batch * PARTS);
    if (q) {
        q->m = m, q->n = n, q->ldx = ldx, q->lda = lda, q->turned = rows > cols, q->batch = batch;
        q->px[0] = reinterpret_cast<__half*>(at), q->px[1] = reinterpret_cast<__half*>(at + x);
        q->pa = reinterpret_cast<__half*>(at + 2 * x), q->pb = reinterpret_cast<__half*>(at + 2 * x + a);
        q->parts = reinterpret_cast<double*>(at + 2 * x + 2 * a);
    }
    return 2 * x + 2 * a + parts;
}

int tiles_sym(int m, int bn) {
    int t = 0;
    for (int r = 0; r * 128 < m; ++r) t += (m + bn - 1) / bn - r * (128 / bn);
    return t;
}
int tiles_all(int m, int n, int bn) { return (m + 127) / 128 * ((n + bn - 1) / bn); }

template <int BN>
int products(const char* who, Jobs& p, int steps, const cbm::Stream& on) {
    using S = Shape<BN>;
    if (!allow_smem<product_kernel<BN>>(S::SMEM)) return cbm::fail(CBM_B200_ERR_CUDA, std::string(who) + ": no room in shared memory");
    int sym = 0, all = 0;
    for (int i = 0; i < p.count; ++i) {
        Job& q = p.job[i];
        q.tiles_sym = tiles_sym(q.m, BN), q.tiles_all = tiles_all(q.m, q.n, BN);
        sym += q.tiles_sym * q.batch, all += q.tiles_all * q.batch;
    }
    const int sms = sm_count();
    for (int k = 0; k < steps; ++k) {
        cbm::launch_next(product_kernel<BN>, dim3(sym < sms ? sym : sms), TILE_THREADS, S::SMEM, on, p, GRAM, k & 1, sym, false);
        cbm::launch_next(product_kernel<BN>, dim3(sym < sms ? sym : sms), TILE_THREADS, S::SMEM, on, p, SQUARE, k & 1, sym, false);
        cbm::launch_next(product_kernel<BN>, dim3(all < sms ? all : sms), TILE_THREADS, S::SMEM, on, p, APPLY, k & 1, all, k + 1 == steps);
    }
    return CBM_B200_OK;
}

int run(const char* who, Jobs& p, int steps, void* stream) {
    if (int rc = check_timeout(who)) return rc;
    p.timeout = timeout_word();
    const cbm::Stream on(static_cast<cudaStream_t>(stream));
    int matrices = 0, blocks = 1;
    int64_t wide = 0;
    for (int i = 0; i < p.count; ++i) {
        Job& q = p.job[i];
        if (!describe(&q.x[0], q.px[0], q.m, q.n, q.ldx, q.batch) || !describe(&q.x[1], q.px[1], q.m, q.n, q.ldx, q.batch) ||
            !describe(&q.a, q.pa, q.m, q.m, q.lda, q.batch) || !describe(&q.b, q.pb, q.m, q.m, q.lda, q.batch))
            return cbm::fail(CBM_B200_ERR_CUDA, std::string(who) + ": no tensor map for its operands");
        matrices += q.batch;
        const int64_t tiles = (int64_t)((q.m + 31) / 32) * ((q.n + 31) / 32);
        if (tiles > blocks) blocks = (int)(tiles < 2048 ? tiles : 2048);
        wide += (int64_t)q.batch * tiles_sym(q.m, 128);
    }
    cbm::launch_next(norm_kernel, dim3(PARTS, matrices), THREADS, 0, on, p);
    cbm::launch_next(start_kernel, dim3(blocks, matrices), THREADS, 0, on, p);
    // Tiles of 128 columns where there are enough of them for most SMs, else of 64.
    if (int rc = wide * 4 >= sm_count() * 3 ? products<128>(who, p, steps, on) : products<64>(who, p, steps, on)) return rc;
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? CBM_B200_OK : cbm::fail(CBM_B200_ERR_CUDA, std::string(who) + ": " + cudaGetErrorString(e));
}

constexpr int MAX_SIDE = 1 << 16, MAX_BATCH = 32768;  // (tiles are counted in 31 bits, matrices in a grid's second dimension)

}  // namespace

extern "C" int64_t cbm_b200_orthogonalise_workspace(int32_t batch, int32_t rows, int32_t cols) {
    return batch > 0 && rows > 0 && cols > 0 ? lay_out(nullptr, rows, cols, batch, nullptr) : 0;
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
    lay_out(&p.job[0], rows, cols, batch, static_cast<unsigned char*>(workspace));
    p.job[0].of = Matrix{u, nullptr, nullptr, out, ldu, 0, 0, ldout, next_u, next_out, 0.f, 0.f};
    return run("orthogonalise", p, steps, stream);
}

extern "C" int64_t cbm_b200_orthogonal_step_workspace(const cbm_b200_update_of* of, int32_t count) {
    int64_t all = 0;
    for (int i = 0; of && i < count; ++i)
        if (of[i].rows > 0 && of[i].cols > 0) all += lay_out(nullptr, of[i].rows, of[i].cols, 1, nullptr);
    return all;
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
    unsigned char* at = static_cast<unsigned char*>(workspace);
    for (int i = 0; i < count;) {
        Jobs p{};
        p.eps = eps, p.momentum = momentum, p.nesterov = nesterov;
        for (; i < count && p.count < MAX_JOBS; ++i) {
            const cbm_b200_update_of& u = of[i];
            if (u.rows == 0 || u.cols == 0) continue;
            Job& q = p.job[p.count++];
            at += lay_out(&q, u.rows, u.cols, 1, at);
            const double tall = u.rows > u.cols ? std::sqrt((double)u.rows / u.cols) : 1.0;
            q.of = Matrix{u.g, u.m, u.w, nullptr, u.ldg, u.ldm, u.ldw, 0, 0, 0, (float)(lr * tall), (float)(1.0 - (double)lr * weight_decay)};
        }
        if (p.count)
            if (int rc = run("orthogonal_step", p, steps, stream)) return rc;
    }
    return CBM_B200_OK;
}
