// Class log probabilities of rows of logits, with entropy and the most probable classes, and the gradient (sm_100a).
//
// With m the largest of a row, s the sum of exp(x - m) over the others and t = sum exp(x - m) (m - x):
//   log p_j = (x_j - m) - log1p(s),   entropy = log1p(s) + t / (1 + s).
// Nothing in these is subtracted that is nearly equal, so a decided row keeps the digits of a log probability near 0.
// What bounds it is memory: logits are read once, forwards and backwards, and the gradient is written once.  Narrow rows go through shared
// memory, where lanes of a row lie a bank apart; long ones are gone over once by a block or a cluster, which keeps m, s and t as it goes
// (2 449 029 x 47 fp32 102 us, 4.9 TB/s, with the gradient 244 us, of 220 at the rate of a copy).
// Gradient: dx_j = g_log ([j = label] - p_j) - g_ent p_j (log p_j + entropy) + sum_i g_top_i ([j = c_i] - p_j).
// What a class is given itself is multiplied by 1 - p_j = -expm1(log p_j), so that a decided row keeps its digits here, too.
#include "cbm_common.h"
#include "cbm_launch.cuh"
#include "cbm_values.cuh"

#include <cmath>
#include <string>
#include <type_traits>

namespace {

using u32 = uint32_t;
using u64 = unsigned long long;

constexpr u32 FULL = 0xffffffffu;
constexpr float LOWEST = -200.f;  // exp of it is 0: differences are cut off there, so that 0 times infinity does not come up

// Whole numbers in the order of the values: NaN above all, the two zeros equal.  (NaN is not the largest number there is: the key of class 0
// would then be 2^64 - 1, where the search for the first place starts, and never be behind it.)
constexpr u32 NAN_KEY = 0xfffffffeu;
__device__ __forceinline__ u32 ordered(float x) {
    if (x != x) return NAN_KEY;
    const u32 b = __float_as_uint(x + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(u32 key) {
    return key == NAN_KEY ? NAN : __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}
// In the order in which classes are listed: by value, then the lower class first.
__device__ __forceinline__ u64 key_of(u32 value, u32 j) { return (u64)value << 32 | (u32)~j; }

// max that passes NaN on.
__device__ __forceinline__ float max_nan(float x, float y) {
    float z;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(z) : "f"(x), "f"(y));
    return z;
}
// exp of d <= 0, by the fast form: its argument is rounded once, |d| U of the result, and in a sum the terms of large |d| are small.
// (A tile kernel with the exact form: 2.4 M x 47 fp32 115 us, with this one 102.)
__device__ __forceinline__ float exp_of(float d) { return __expf(d); }

struct ForwardParams {
    const void* x;
    const void* labels;
    int64_t ld, n;
    int c, top, wide_labels, lanes, shift;  // lanes = 1 << shift
    float *log_prob, *entropy, *stats, *top_log_prob;
    int64_t* top_class;
};

__device__ __forceinline__ int64_t label_of(const void* labels, int wide, int64_t row) {
    return wide ? static_cast<const int64_t*>(labels)[row] : (int64_t) static_cast<const int32_t*>(labels)[row];
}

// What a row leaves behind: m, the sums s (others) and t over it.
template <class T>
__device__ __forceinline__ void store_row(const ForwardParams& p, int64_t row, const T* x, float m, float ls, float entropy) {
    const int64_t label = label_of(p.labels, p.wide_labels, row);
    p.log_prob[row] = label < 0 ? 0.f : label >= p.c ? NAN : m == -INFINITY ? -INFINITY : (cbm::widen(x[label]) - m) - ls;
    p.entropy[row] = entropy;
    if (p.stats) *reinterpret_cast<float2*>(p.stats + 2 * row) = float2{m, ls};
}

// Rows of up to 32 VALUES classes that are wide, or lie at odd places: `lanes` neighbouring lanes to a row (a power of two), which hold
// it in registers, class j in lane j mod lanes.  As few lanes as VALUES allow, since what they exchange comes on top of it.
template <class T, int VALUES>
__global__ void __launch_bounds__(256) rows_kernel(const ForwardParams p) {
    cbm::wait_before();
    const int lanes = p.lanes, lane = threadIdx.x & (lanes - 1);
    const int64_t row = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> p.shift;
    const bool on = row < p.n;  // (the lanes of a warp stay together)
    const T* x = static_cast<const T*>(p.x) + (on ? row : 0) * p.ld;
    float v[VALUES];
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < VALUES; ++i) {
        const int j = lane + i * lanes;
        v[i] = on && j < p.c ? cbm::widen(x[j]) : -INFINITY;
    }
#pragma unroll
    for (int i = 0; i < VALUES; ++i) m = max_nan(m, v[i]);
    for (int o = lanes >> 1; o; o >>= 1) m = max_nan(m, __shfl_xor_sync(FULL, m, o));
    const bool closed = m == -INFINITY, undefined = !(m < INFINITY);
    const float from = closed ? 0.f : m;
    float s = 0.f, t = 0.f, equal = 0.f;
#pragma unroll
    for (int i = 0; i < VALUES; ++i) {
        const float d = fmaxf(v[i] - from, LOWEST), e = exp_of(d);
        if (d < 0.f) s += e;
        else equal += 1.f;
        t -= e * d;
    }
    for (int o = lanes >> 1; o; o >>= 1) {
        s += __shfl_xor_sync(FULL, s, o);
        t += __shfl_xor_sync(FULL, t, o);
        equal += __shfl_xor_sync(FULL, equal, o);
    }
    s += equal - 1.f;
    const float ls = undefined ? NAN : closed ? 0.f : log1pf(s);
    if (on && lane == 0) store_row(p, row, x, m, ls, closed ? 0.f : ls + t / (1.f + s));
    if (p.top == 0) return;
    // The most probable classes, one after the other: each lane's best that is behind the last one taken.
    u64 last = ~0ull;
    for (int i = 0; i < p.top; ++i) {
        u64 best = 0;
#pragma unroll
        for (int k = 0; k < VALUES; ++k) {
            const int j = lane + k * lanes;
            const u64 key = j < p.c ? key_of(ordered(v[k]), j) : 0;
            best = key < last && key > best ? key : best;
        }
        for (int o = lanes >> 1; o; o >>= 1) {
            const u64 other = __shfl_xor_sync(FULL, best, o);
            best = other > best ? other : best;
        }
        last = best;
        if (on && lane == 0) {
            p.top_class[row * p.top + i] = (u32) ~(u32)best;
            p.top_log_prob[row * p.top + i] = closed ? -INFINITY : (value_of((u32)(best >> 32)) - m) - ls;
        }
    }
}

// ---- narrow rows ------------------------------------------------------------------------------------
// A block takes a tile of rows through shared memory, 16 bytes at a time on the way in (and, for the gradient, out), and a
// thread, or a few, work on a row there: what a row costs beside its values (the logarithm, label, results) is then paid for by one or
// four lanes and not by eight to thirty-two, and rows of any width are fetched in whole lines.
// Rows are read in vectors of E values.  Where rows are 16-byte aligned they are put at a pitch that is an odd multiple of 16 bytes;
// otherwise the tile is one stretch of memory and E is the largest power of two that divides the row: the pitch is
// an odd number of vectors either way, so that the lanes' vectors fall into different banks.
constexpr int TILE_THREADS = 128;

struct Tile {
    int rows, pitch;   // of a tile; in bytes
    int chunks;        // 16-byte pieces of a row, 0: the tile is one stretch
    u32 per_chunk;     // 2^20 / chunks, rounded up: pieces are counted up to 2^11, so i * per_chunk >> 20 is i / chunks
    int bytes;         // of shared memory
};

template <class T, int E>
union Values {
    T v[E];
    std::conditional_t<sizeof(T) * E == 16, uint4, std::conditional_t<sizeof(T) * E == 8, uint2, std::conditional_t<sizeof(T) * E == 4, u32, uint16_t>>> bits;
    __device__ Values() {}
};

__device__ __forceinline__ void copy_in(void* to, const void* from, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((u32)__cvta_generic_to_shared(to)), "l"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ void tile_in(unsigned char* smem, const unsigned char* x, int64_t ld_bytes, int64_t first, int rows, int row_bytes, const Tile& t) {
    if (t.chunks) {
        for (int i = threadIdx.x; i < rows * t.chunks; i += TILE_THREADS) {
            const int r = (int)((u32)i * t.per_chunk >> 20), q = i - r * t.chunks;
            copy_in(smem + r * t.pitch + 16 * q, x + (first + r) * ld_bytes + 16 * q, min(16, row_bytes - 16 * q));
        }
    } else {
        const int bytes = rows * row_bytes;
        for (int i = 16 * threadIdx.x; i < bytes; i += 16 * TILE_THREADS) copy_in(smem + i, x + first * ld_bytes + i, min(16, bytes - i));
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
}

template <class T, int E>
__global__ void __launch_bounds__(TILE_THREADS) tile_kernel(const ForwardParams p, const Tile t) {
    extern __shared__ __align__(16) unsigned char smem[];
    cbm::wait_before();
    const int lane = threadIdx.x & (p.lanes - 1), mine = threadIdx.x >> p.shift;
    const int64_t first = (int64_t)blockIdx.x * t.rows, row = first + mine;
    const int rows = (int)min((int64_t)t.rows, p.n - first);
    tile_in(smem, static_cast<const unsigned char*>(p.x), p.ld * sizeof(T), first, rows, p.c * (int)sizeof(T), t);
    const bool on = mine < rows;
    const T* x = reinterpret_cast<const T*>(smem + (on ? mine : 0) * t.pitch);
    // f(j, value) for the values of this lane's vectors
    auto each = [&](auto&& f) {
        int j0 = lane * E;
        for (; j0 + E <= p.c; j0 += p.lanes * E) {
            Values<T, E> w;
            w.bits = *reinterpret_cast<const decltype(w.bits)*>(x + j0);
#pragma unroll
            for (int i = 0; i < E; ++i) f(j0 + i, cbm::widen(w.v[i]));
        }
        if constexpr (E > 1)
            for (int j = j0; j < p.c && j < j0 + E; ++j) f(j, cbm::widen(x[j]));
    };
    float m = -INFINITY;
    each([&](int, float v) { m = max_nan(m, v); });
    for (int o = p.lanes >> 1; o; o >>= 1) m = max_nan(m, __shfl_xor_sync(FULL, m, o));
    const bool closed = m == -INFINITY, undefined = !(m < INFINITY);
    const float from = closed ? 0.f : m;
    float s = 0.f, u = 0.f, equal = 0.f;
    each([&](int, float v) {
        const float d = fmaxf(v - from, LOWEST), e = exp_of(d);
        if (d < 0.f) s += e;
        else equal += 1.f;
        u -= e * d;
    });
    for (int o = p.lanes >> 1; o; o >>= 1) {
        s += __shfl_xor_sync(FULL, s, o);
        u += __shfl_xor_sync(FULL, u, o);
        equal += __shfl_xor_sync(FULL, equal, o);
    }
    s += equal - 1.f;
    const float ls = undefined ? NAN : closed ? 0.f : log1pf(s);
    if (on && lane == 0) store_row(p, row, x, m, ls, closed ? 0.f : ls + u / (1.f + s));
    // The most probable classes, one after the other: each lane's best that is behind the last one taken.  Values are compared as they
    // are; only a row with NaN goes by whole numbers.
    const bool by_value = __all_sync(FULL, !undefined);
    float taken = INFINITY;
    int at = -1;
    for (int i = 0; i < p.top; ++i) {
        float best = -INFINITY;
        int where = -1;
        if (by_value) {
            each([&](int j, float v) {
                const bool behind = v < taken || (v == taken && j > at);
                if (behind && (v > best || where < 0)) best = v, where = j;
            });
            for (int o = p.lanes >> 1; o; o >>= 1) {
                const float v = __shfl_xor_sync(FULL, best, o);
                const int j = __shfl_xor_sync(FULL, where, o);
                if (j >= 0 && (where < 0 || v > best || (v == best && j < where))) best = v, where = j;
            }
        } else {
            const u64 last = i ? key_of(ordered(taken), at) : ~0ull;
            u64 next = 0;
            each([&](int j, float v) {
                const u64 key = key_of(ordered(v), j);
                next = key < last && key > next ? key : next;
            });
            for (int o = p.lanes >> 1; o; o >>= 1) {
                const u64 other = __shfl_xor_sync(FULL, next, o);
                next = other > next ? other : next;
            }
            best = value_of((u32)(next >> 32)), where = (int)~(u32)next;
        }
        taken = best, at = where;
        if (on && lane == 0) {
            p.top_class[row * p.top + i] = where;
            p.top_log_prob[row * p.top + i] = closed ? -INFINITY : (best - m) - ls;
        }
    }
}

// ---- long rows ------------------------------------------------------------------------------------
constexpr int CLUSTER = 8;
constexpr int LISTED = 512;  // candidates for the list that a block keeps

// A part of a row: its largest value m and s = sum exp(x - m), t = sum exp(x - m) (m - x) over all of it.
struct alignas(16) Part {  // (handed over in one 16-byte store)
    float m, s, t, unused;
};
// The sums around a larger value.
__device__ __forceinline__ void move_to(float m, Part& a) {
    if (a.m < m && a.m > -INFINITY) {
        const float d = fmaxf(a.m - m, LOWEST), f = exp_of(d);
        a.t = f * (a.t - d * a.s);
        a.s *= f;
    }
    a.m = m;
}

__device__ __forceinline__ u32 cluster_rank() {
    u32 r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ u32 cluster_size() {
    u32 r;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
// The address in the first block of the cluster of what lies at `p` in this one's shared memory.
__device__ __forceinline__ u32 in_first(const void* p) {
    u32 r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"((u32)__cvta_generic_to_shared(p)));
    return r;
}

template <class T>
union Vector {
    static constexpr int N = 16 / sizeof(T);
    uint4 bits;
    T v[N];
    __device__ Vector() {}
};

// Calls f(first, value) for single values and g(first, values) for batches of up to BATCH vectors, BATCH vectors N values, of [a, b)
// of x that fall to this thread.
template <class T, int THREADS>
struct Stretch {
    static constexpr int N = Vector<T>::N, BATCH = 4;
    const T* x;
    int a, b, head, vectors, done;
    __device__ __forceinline__ Stretch(const T* row, int from, int to) : x(row), a(from), b(to) {
        const int off = (int)(((16 - (reinterpret_cast<u64>(x + a) & 15)) & 15) / sizeof(T));
        head = min(off, b - a), vectors = (b - a - head) / N, done = a + head + vectors * N;
    }
    template <class F, class G>
    __device__ __forceinline__ void run(F&& f, G&& g) const {
        const uint4* at = reinterpret_cast<const uint4*>(x + a + head);
        if ((int)threadIdx.x < head + b - done) {
            const int j = (int)threadIdx.x < head ? a + (int)threadIdx.x : done + (int)threadIdx.x - head;
            f(j, cbm::widen(x[j]));
        }
        int i = threadIdx.x;
        for (; i + (BATCH - 1) * THREADS < vectors; i += BATCH * THREADS) {
            Vector<T> w[BATCH];
#pragma unroll
            for (int k = 0; k < BATCH; ++k) w[k].bits = at[i + k * THREADS];
            g(w, std::integral_constant<int, BATCH>(), i);
        }
        for (; i < vectors; i += THREADS) {
            Vector<T> w[1];
            w[0].bits = at[i];
            g(w, std::integral_constant<int, 1>(), i);
        }
    }
    __device__ __forceinline__ int index(int vector, int i) const { return a + head + vector * N + i; }
};

// Pairs of fp32 operations in one instruction.
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 r;
    asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 r;
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\tfma.rn.f32x2 x, x, y, z;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return r;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(FULL, v, o);
    return v;
}

// A cluster of blocks to a row, each with its part of it, in one pass: every thread keeps its largest value so far and the sums around
// it, which move when a larger one comes.  In a decided row (s close to 1) the sum over the others is taken in a second pass, without the
// largest value, so that its digits are not lost beside it.
// For the list, the top-th largest of the largest values of 32 groups of threads bounds the last place from below: the values that
// reach it, not many more than the list is long, are collected in a second pass (out of L2) and ranked by comparing each with all.
// Where equal values make them too many, the list is found by one pass for each place.
// THREADS: 256, or 128 for rows of less than 32 KB, of which more are then under way (30 000 rows of 2 000 fp32, 3 best: 256 -> 209 us).
template <class T, int THREADS>
__global__ void __launch_bounds__(THREADS) long_kernel(const ForwardParams p) {
    constexpr int WARPS = THREADS / 32, GROUP = THREADS / 32;  // (32 groups of so many threads)
    __shared__ __align__(16) float s_max[WARPS];
    __shared__ float2 s_sum[WARPS];
    __shared__ float s_group[32], s_others[WARPS];
    __shared__ u64 s_list[LISTED];
    __shared__ u64 s_reduce[WARPS];
    __shared__ float s_bound;
    __shared__ u32 s_count;
    __shared__ Part s_parts[CLUSTER];                       // what the blocks of the cluster found ...
    __shared__ u64 s_lists[CLUSTER * CBM_B200_MAX_TOP];     // ... in the first block
    cluster_arrive();  // the others' shared memory is there once all have started
    cbm::wait_before();
    const int rank = (int)cluster_rank(), blocks = (int)cluster_size(), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int each = ((p.c + blocks - 1) / blocks + 63) / 64 * 64;
    const int a = min(rank * each, p.c), b = min(a + each, p.c);
    const int64_t row = blockIdx.x / blocks;
    const T* x = static_cast<const T*>(p.x) + row * p.ld;
    const Stretch<T, THREADS> part(x, a, b);

    Part mine{-INFINITY, 0.f, 0.f, 0.f};
    part.run(
        [&](int, float v) {  // (a thread's first value)
            mine.m = v;
            mine.s = v > -INFINITY ? 1.f : 0.f;
        },
        [&](const auto& w, auto batch, int) {
            constexpr int N = Vector<T>::N, B = decltype(batch)::value;
            constexpr float L = 1.4426950408889634f;
            float v[B * N], high = -INFINITY;
#pragma unroll
            for (int i = 0; i < B * N; ++i) v[i] = cbm::widen(w[i / N].v[i % N]);
#pragma unroll
            for (int i = 0; i < B * N; ++i) high = max_nan(high, v[i]);
            if (high > mine.m || high != high) move_to(high, mine);  // (NaN stays, once it is the largest)
            const float from = mine.m == -INFINITY ? 0.f : mine.m;
            float2 s{0.f, 0.f}, t{0.f, 0.f};
#pragma unroll
            for (int i = 0; i < B * N; i += 2) {
                float2 d = add2(float2{v[i], v[i + 1]}, float2{-from, -from});
                d.x = fmaxf(d.x, LOWEST), d.y = fmaxf(d.y, LOWEST);
                const float2 y = fma2(d, float2{L, L}, float2{0.f, 0.f});
                float2 e;
                asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(y.x));
                asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(y.y));
                s = add2(s, e);
                t = fma2(e, d, t);
            }
            mine.s += s.x + s.y;
            mine.t -= t.x + t.y;
        });
    // the block's largest value; on the way there, those of groups of threads
    float m = mine.m;
#pragma unroll
    for (int o = 1; o < GROUP; o <<= 1) m = max_nan(m, __shfl_xor_sync(FULL, m, o));
    if (lane % GROUP == 0) s_group[(int)threadIdx.x / GROUP] = m;
#pragma unroll
    for (int o = GROUP; o < 32; o <<= 1) m = max_nan(m, __shfl_xor_sync(FULL, m, o));
    if (lane == 0) s_max[warp] = m;
    if (threadIdx.x == 0) s_count = 0;
    __syncthreads();
    m = s_max[0];
#pragma unroll
    for (int i = 1; i < WARPS; ++i) m = max_nan(m, s_max[i]);
    move_to(m, mine);
    const float2 sums{warp_sum(mine.s), warp_sum(mine.t)};
    if (lane == 0) s_sum[warp] = sums;
    if (p.top && warp == 0) {  // the top-th largest of the groups' (of equal ones, the lower group's counts as larger)
        const u32 key = ordered(s_group[lane]);
        int above = 0;
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            const u32 other = __shfl_sync(FULL, key, i);
            above += other > key || (other == key && i < lane);
        }
        if (above == p.top - 1) s_bound = s_group[lane];
    }
    __syncthreads();
    Part all{m, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < WARPS; ++i) all.s += s_sum[i].x, all.t += s_sum[i].y;
    cluster_wait();
    if (threadIdx.x == 0) {
        const u32 to = in_first(&s_parts[rank]);
        asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(to), "f"(all.m), "f"(all.s), "f"(all.t), "f"(0.f) : "memory");
    }
    if (p.top) {
        const float bound = s_bound;
        auto collect = [&](int j, float v) {
            if (v < bound) return;  // (NaN is collected)
            const u32 at = atomicAdd(&s_count, 1u);
            if (at < LISTED) s_list[at] = key_of(ordered(v), (u32)j);
        };
        part.run(collect, [&](const auto& w, auto batch, int first) {
            constexpr int N = Vector<T>::N, B = decltype(batch)::value;
#pragma unroll
            for (int k = 0; k < B; ++k) {
                float high = -INFINITY;
#pragma unroll
                for (int i = 0; i < N; ++i) high = max_nan(high, cbm::widen(w[k].v[i]));
                if (!(high < bound)) {
#pragma unroll
                    for (int i = 0; i < N; ++i) collect(part.index(first + k * THREADS, i), cbm::widen(w[k].v[i]));
                }
            }
        });
        __syncthreads();
        const int found = (int)s_count;
        const u32 to = in_first(&s_lists[rank * CBM_B200_MAX_TOP]);
        auto put = [&](int place, u64 k) { asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(to + 8 * place), "l"(k) : "memory"); };
        if (found <= LISTED) {
            for (int i = threadIdx.x; i < found; i += THREADS) {
                const u64 k = s_list[i];
                int above = 0;
                for (int q = 0; q < found; ++q) above += s_list[q] > k;
                if (above < p.top) put(above, k);
            }
            for (int i = found + threadIdx.x; i < p.top; i += THREADS) put(i, 0);  // (a part shorter than the list)
        } else {
            u64 last = ~0ull;
            for (int place = 0; place < p.top; ++place) {
                u64 best = 0;
                auto behind = [&](int j, float v) {
                    const u64 k = key_of(ordered(v), (u32)j);
                    best = k < last && k > best ? k : best;
                };
                part.run(behind, [&](const auto& w, auto batch, int first) {
                    constexpr int N = Vector<T>::N, B = decltype(batch)::value;
#pragma unroll
                    for (int k = 0; k < B; ++k)
#pragma unroll
                        for (int i = 0; i < N; ++i) behind(part.index(first + k * THREADS, i), cbm::widen(w[k].v[i]));
                });
#pragma unroll
                for (int o = 16; o; o >>= 1) {
                    const u64 other = __shfl_xor_sync(FULL, best, o);
                    best = other > best ? other : best;
                }
                __syncthreads();
                if (lane == 0) s_reduce[warp] = best;
                __syncthreads();
                best = s_reduce[0];
#pragma unroll
                for (int q = 1; q < WARPS; ++q) best = s_reduce[q] > best ? s_reduce[q] : best;
                last = best;
                if (threadIdx.x == 0) put(place, best);
            }
        }
    }
    cluster_arrive();
    cluster_wait();
    if (rank != 0) return;
    m = s_parts[0].m;
    for (int i = 1; i < blocks; ++i) m = max_nan(m, s_parts[i].m);
    all = Part{m, 0.f, 0.f, 0.f};
    for (int i = 0; i < blocks; ++i) {
        Part one = s_parts[i];
        move_to(m, one);
        all.s += one.s;
        all.t += one.t;
    }
    const bool closed = m == -INFINITY, undefined = !(m < INFINITY);
    float others = all.s - 1.f;
    if (!closed && !undefined && others < 0.0078125f) {  // (below 2^-7, s has lost 7 digits of 24 of what is added to 1)
        float sum = 0.f, equal = 0.f;
        auto add = [&](int, float v) {
            if (v < m) sum += exp_of(fmaxf(v - m, LOWEST));
            else equal += 1.f;
        };
        const Stretch<T, THREADS> whole(x, 0, p.c);
        whole.run(add, [&](const auto& w, auto batch, int) {
#pragma unroll
            for (int k = 0; k < decltype(batch)::value; ++k)
#pragma unroll
                for (int i = 0; i < Vector<T>::N; ++i) add(0, cbm::widen(w[k].v[i]));
        });
        sum = warp_sum(sum), equal = warp_sum(equal);
        if (lane == 0) s_others[warp] = sum, s_max[warp] = equal;
        __syncthreads();
        others = 0.f, equal = 0.f;
#pragma unroll
        for (int i = 0; i < WARPS; ++i) others += s_others[i], equal += s_max[i];
        others += equal - 1.f;
    }
    const float ls = undefined ? NAN : closed ? 0.f : log1pf(others);
    if (threadIdx.x == 0) store_row(p, row, x, m, ls, closed ? 0.f : ls + all.t / (1.f + others));
    const int found = blocks * CBM_B200_MAX_TOP;
    for (int i = threadIdx.x; p.top && i < found; i += THREADS) {
        if (i % CBM_B200_MAX_TOP >= p.top) continue;
        const u64 k = s_lists[i];
        int above = 0;
        for (int q = 0; q < blocks; ++q)
            for (int e = 0; e < p.top; ++e) above += s_lists[q * CBM_B200_MAX_TOP + e] > k;
        if (above < p.top && k) {
            p.top_class[row * p.top + above] = (u32) ~(u32)k;
            p.top_log_prob[row * p.top + above] = closed ? -INFINITY : (value_of((u32)(k >> 32)) - m) - ls;
        }
    }
}

// ---- gradient -------------------------------------------------------------------------------------
struct BackwardParams {
    const void* x;
    const void* labels;
    int64_t ld, ld_out, n;
    int c, top, wide_labels, lanes, shift;
    const float *stats, *entropy, *g_log, *g_entropy, *g_top;
    const int64_t* top_class;
    void* dx;
};

// dx_j = base(x_j), and for the label and the listed classes something more.
template <class T>
struct RowGradient {
    float m, ls, gl, ge, rest, all;  // rest: what every class is given but for its own, gl left out
    int label;  // -1: none
    bool closed;
    __device__ __forceinline__ RowGradient(const BackwardParams& p, int64_t row) {
        const int64_t given = label_of(p.labels, p.wide_labels, row);
        label = given >= 0 && given < p.c ? (int)given : -1;
        m = p.stats[2 * row], ls = p.stats[2 * row + 1];
        closed = m == -INFINITY;
        if (closed) m = 0.f;
        gl = !p.g_log || given < 0 || closed ? 0.f : given >= p.c ? NAN : p.g_log[row];
        ge = p.g_entropy && !closed ? p.g_entropy[row] : 0.f;
        rest = ge * p.entropy[row];
        if (p.g_top && !closed)
            for (int i = 0; i < p.top; ++i) rest += p.g_top[row * p.top + i];
        all = gl + rest;
    }
    __device__ __forceinline__ float base(float x) const {
        const float lp = fmaxf((x - m) - ls, LOWEST);
        return -exp_of(lp) * (all + ge * lp);
    }
    // Of a class that is given `own` itself, `others` by the other classes.
    __device__ __forceinline__ float of_given(float x, float own, float others) const {
        const float lp = fmaxf((x - m) - ls, LOWEST);
        return own * -expm1f(lp) - exp_of(lp) * (others + ge * lp);
    }
    __device__ __forceinline__ float at_label(float x) const { return of_given(x, gl, rest); }
    // Of the i-th class of the list, j.
    __device__ __forceinline__ float at_listed(const BackwardParams& p, int64_t row, int i, int64_t j, float x) const {
        const float* given = p.g_top + row * p.top;
        float others = ge * p.entropy[row];
        for (int q = 0; q < p.top; ++q) others += q == i ? 0.f : given[q];
        return j == label ? of_given(x, given[i] + gl, others) : of_given(x, given[i], others + gl);
    }
};

// Narrow rows: in place in a tile of shared memory.
template <class T, int E>
__global__ void __launch_bounds__(TILE_THREADS) tile_grad_kernel(const BackwardParams p, const Tile t) {
    extern __shared__ __align__(16) unsigned char smem[];
    cbm::wait_before();
    const int lane = threadIdx.x & (p.lanes - 1), mine = threadIdx.x >> p.shift;
    const int64_t first = (int64_t)blockIdx.x * t.rows, row = first + mine;
    const int rows = (int)min((int64_t)t.rows, p.n - first), row_bytes = p.c * (int)sizeof(T);
    const bool on = mine < rows;
    const RowGradient<T> g(p, on ? row : first);
    tile_in(smem, static_cast<const unsigned char*>(p.x), p.ld * sizeof(T), first, rows, row_bytes, t);
    T* x = reinterpret_cast<T*>(smem + (on ? mine : 0) * t.pitch);
    float at_label = 0.f;
    const int owner = on && g.label >= 0 ? g.label / E & (p.lanes - 1) : -1;  // the lane whose vector holds the label
    if (lane == owner) at_label = cbm::widen(x[g.label]);
    if (on) {
        int j0 = lane * E;
        for (; j0 + E <= p.c; j0 += p.lanes * E) {
            Values<T, E> w;
            w.bits = *reinterpret_cast<const decltype(w.bits)*>(x + j0);
#pragma unroll
            for (int i = 0; i < E; ++i) w.v[i] = cbm::narrow<T>(g.base(cbm::widen(w.v[i])));
            *reinterpret_cast<decltype(w.bits)*>(x + j0) = w.bits;
        }
        if constexpr (E > 1)
            for (int j = j0; j < p.c && j < j0 + E; ++j) x[j] = cbm::narrow<T>(g.base(cbm::widen(x[j])));
        if (lane == owner) x[g.label] = cbm::narrow<T>(g.at_label(at_label));
    }
    __syncthreads();
    unsigned char* to = static_cast<unsigned char*>(p.dx) + first * p.ld_out * (int64_t)sizeof(T);
    // the last 16 bytes of a row, or of the stretch, value by value where not all are the row's
    auto out = [&](unsigned char* d, const unsigned char* from, int bytes) {
        if (bytes >= 16) *reinterpret_cast<uint4*>(d) = *reinterpret_cast<const uint4*>(from);
        else
            for (int b = 0; b < bytes; b += (int)sizeof(T)) *reinterpret_cast<T*>(d + b) = *reinterpret_cast<const T*>(from + b);
    };
    if (t.chunks) {
        for (int i = threadIdx.x; i < rows * t.chunks; i += TILE_THREADS) {
            const int r = (int)((u32)i * t.per_chunk >> 20), q = 16 * (i - r * t.chunks);
            out(to + r * p.ld_out * (int64_t)sizeof(T) + q, smem + r * t.pitch + q, row_bytes - q);
        }
    } else {
        for (int i = 16 * threadIdx.x; i < rows * row_bytes; i += 16 * TILE_THREADS) out(to + i, smem + i, rows * row_bytes - i);
    }
    if (!p.g_top || p.top == 0) return;
    __syncthreads();
    if (on && !g.closed)
        for (int i = lane; i < p.top; i += p.lanes) {
            const int64_t j = p.top_class[row * p.top + i];
            if (j < 0 || j >= p.c) continue;  // (no class)
            static_cast<T*>(p.dx)[row * p.ld_out + j] = cbm::narrow<T>(g.at_listed(p, row, i, j, cbm::widen(static_cast<const T*>(p.x)[row * p.ld + j])));
        }
}

// Rows of up to a few hundred classes: `lanes` lanes to a row.
template <class T>
__global__ void __launch_bounds__(256) rows_grad_kernel(const BackwardParams p) {
    cbm::wait_before();
    const int lanes = p.lanes, lane = threadIdx.x & (lanes - 1);
    const int64_t row = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> p.shift;
    const bool on = row < p.n;
    const T* x = static_cast<const T*>(p.x) + (on ? row : 0) * p.ld;
    T* dx = static_cast<T*>(p.dx) + (on ? row : 0) * p.ld_out;
    const RowGradient<T> g(p, on ? row : 0);
    if (on) {
#pragma unroll 4
        for (int j = lane; j < p.c; j += lanes) {
            const float v = cbm::widen(x[j]);
            dx[j] = cbm::narrow<T>(j == g.label ? g.at_label(v) : g.base(v));
        }
    }
    if (!p.g_top || p.top == 0) return;
    __syncwarp();
    if (on && !g.closed)
        for (int i = lane; i < p.top; i += lanes) {
            const int64_t j = p.top_class[row * p.top + i];
            if (j < 0 || j >= p.c) continue;  // (no class)
            dx[j] = cbm::narrow<T>(g.at_listed(p, row, i, j, cbm::widen(x[j])));
        }
}

// Long rows: a block to a stretch of a row, four vectors a thread, which are on their way before anything else is asked for.
constexpr int THREADS = 256;
constexpr int stretch_of(int size) { return 4 * THREADS * 16 / size; }

template <class T>
__global__ void __launch_bounds__(THREADS) long_grad_kernel(const BackwardParams p, const int stretches) {
    constexpr int N = Vector<T>::N, EACH = 4, STRETCH = EACH * THREADS * N;
    cbm::wait_before();
    const int64_t row = blockIdx.x / stretches;
    const int a = (int)(blockIdx.x % stretches) * STRETCH, b = min(a + STRETCH, p.c);
    const T* x = static_cast<const T*>(p.x) + row * p.ld;
    T* dx = static_cast<T*>(p.dx) + row * p.ld_out;
    const bool alike = ((reinterpret_cast<u64>(x) ^ reinterpret_cast<u64>(dx)) & 15) == 0;
    const int off = (int)(((16 - (reinterpret_cast<u64>(x + a) & 15)) & 15) / sizeof(T));
    const int head = min(off, b - a), vectors = (b - a - head) / N, done = a + head + vectors * N;
    Vector<T> w[EACH];
    if (alike) {
#pragma unroll
        for (int k = 0; k < EACH; ++k)
            if ((int)threadIdx.x + k * THREADS < vectors) w[k].bits = reinterpret_cast<const uint4*>(x + a + head)[threadIdx.x + k * THREADS];
    }
    const RowGradient<T> g(p, row);
    auto one = [&](int j) {
        const float v = cbm::widen(x[j]);
        dx[j] = cbm::narrow<T>(j == g.label ? g.at_label(v) : g.base(v));
    };
    if (alike) {
        if ((int)threadIdx.x < head) one(a + threadIdx.x);
        if ((int)threadIdx.x < b - done) one(done + threadIdx.x);
#pragma unroll
        for (int k = 0; k < EACH; ++k)
            if ((int)threadIdx.x + k * THREADS < vectors) {
#pragma unroll
                for (int i = 0; i < N; ++i) w[k].v[i] = cbm::narrow<T>(g.base(cbm::widen(w[k].v[i])));
                reinterpret_cast<uint4*>(dx + a + head)[threadIdx.x + k * THREADS] = w[k].bits;
            }
        if (g.label >= a + head && g.label < done) {  // (one of the vectors': put right behind them)
            __syncthreads();
            if (threadIdx.x == 0) dx[g.label] = cbm::narrow<T>(g.at_label(cbm::widen(x[g.label])));
        }
    } else {
        for (int j = a + threadIdx.x; j < b; j += THREADS) one(j);
    }
    if (!p.g_top || p.top == 0) return;
    __syncthreads();
    if (!g.closed && (int)threadIdx.x < p.top) {
        const int64_t j = p.top_class[row * p.top + threadIdx.x];
        if (j >= a && j < b) dx[j] = cbm::narrow<T>(g.at_listed(p, row, (int)threadIdx.x, j, cbm::widen(x[j])));
    }
}

constexpr int ROW_MAX = 1024;  // classes that 32 lanes hold in registers, 32 each

constexpr int MOST_CLASSES = 1 << 30;  // (sums of an index and a stretch's classes are held in 31 bits)

int check(const char* who, int64_t n, int64_t ld, int32_t c, int32_t top, int32_t type) {
    if (n < 0 || c < 1 || c > MOST_CLASSES || ld < c || top < 0 || top > CBM_B200_MAX_TOP || top > c || type < 0 || type > CBM_B200_FP16)
        return cbm::fail(CBM_B200_ERR_ARG, std::string(who) + ": bad sizes or type");
    // (a grid has at most 2^31 - 1 blocks: a row to 32 lanes, or to a block for every stretch of 4 096 classes)
    if (n > ((int64_t)1 << 31) - 1 || (c > ROW_MAX && n * ((c + 4095) / 4096) > ((int64_t)1 << 31) - 1))
        return cbm::fail(CBM_B200_ERR_ARG, std::string(who) + ": more rows than a launch has blocks for");
    return CBM_B200_OK;
}

unsigned blocks_of(int64_t n, int each) { return (unsigned)((n + each - 1) / each); }

int launched(const char* who) {
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? CBM_B200_OK : cbm::fail(CBM_B200_ERR_CUDA, std::string(who) + ": " + cudaGetErrorString(e));
}

// Lanes to a row that is held in registers.
int lanes_for(int c, int values) {
    int shift = 0;
    while (shift < 5 && values << shift < c) ++shift;
    return shift;
}

// Bytes of a row that goes through shared memory.  (With the gradient, fp32: 300 000 x 172 115 us, in registers 315; 100 000 x 1 000 221 us,
// by a block each 420.)
constexpr int TILE_ROW = 4096;

// Values of a vector and the tile's layout for rows of `c` values at a pitch of `ld`; 0 where rows do not go that way.
int tile_for(const void* x, int64_t ld, int c, int size, int* shift, Tile* t) {
    const int row = c * size;
    if (reinterpret_cast<uintptr_t>(x) % 16 || row > TILE_ROW) return 0;
    *shift = row <= 256 ? 0 : row <= 1024 ? 2 : row <= 2048 ? 3 : 4;
    t->rows = TILE_THREADS >> *shift;
    if (ld * size % 16 == 0) {
        t->chunks = (row + 15) / 16;
        t->per_chunk = (1u << 20) / t->chunks + 1;
        t->pitch = (t->chunks | 1) * 16;
        t->bytes = t->rows * t->pitch;
        return 16 / size;
    }
    if (ld != c) return 0;
    t->chunks = 0, t->per_chunk = 0;
    t->pitch = row;
    t->bytes = t->rows * row + 16;  // (the last piece is filled up)
    return (row & -row) / size;
}

// Calls f with the number of values of a vector as a constant.
template <class T, class F>
void with_vector(int e, F&& f) {
    switch (e) {
        case 1: f(std::integral_constant<int, 1>()); break;
        case 2: f(std::integral_constant<int, 2>()); break;
        case 4: f(std::integral_constant<int, 4>()); break;
        default:
            if constexpr (sizeof(T) == 2) f(std::integral_constant<int, 8>());
    }
}

// Blocks to a row: while the rows alone leave SMs without one (two of them to each), and a part keeps 8 vectors a thread.  (16 rows of
// 128 256 bf16, 20 best: 8 blocks 20.5 us, one 33; 32 rows of 30 000: 16.4, one 20.5.)
int blocks_to_row(int64_t n, int c, int32_t type) {
    int k = 1;
    while (k < CLUSTER && n * k * 2 <= 2 * 148 && (int64_t)c * cbm::size_of_type(type) / (k * 2) >= THREADS * 16 * 8) k *= 2;
    return k;
}

template <class P>
void launch_clusters(void (*kernel)(P), int64_t blocks, int cluster, int threads, const cbm::Stream& on, const P& p) {
    cudaLaunchAttribute attrs[2] = {};
    attrs[0].id = cudaLaunchAttributeClusterDimension;
    attrs[0].val.clusterDim.x = cluster;
    attrs[0].val.clusterDim.y = attrs[0].val.clusterDim.z = 1;
    attrs[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[1].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3((unsigned)blocks);
    config.blockDim = dim3(threads);
    config.stream = on.s;
    config.attrs = attrs;
    config.numAttrs = on.captured ? 1 : 2;
    (void)cudaLaunchKernelEx(&config, kernel, p);
}

}  // namespace

extern "C" int cbm_b200_class_log_probs(const void* logits, int64_t ld, int32_t type, const void* labels, int32_t wide_labels,
                                        int64_t n_rows, int32_t n_classes, int32_t top, float* log_prob, float* entropy, float* stats,
                                        float* top_log_prob, int64_t* top_class, void* stream) {
    if (int rc = check("class_log_probs", n_rows, ld, n_classes, top, type)) return rc;
    if (n_rows == 0) return CBM_B200_OK;
    if (!logits || !labels || !log_prob || !entropy || (top && (!top_log_prob || !top_class)))
        return cbm::fail(CBM_B200_ERR_ARG, "class_log_probs: NULL argument");
    if (reinterpret_cast<uintptr_t>(stats) % 8) return cbm::fail(CBM_B200_ERR_ARG, "class_log_probs: statistics not at 8 bytes");
    ForwardParams p{logits, labels, ld, n_rows, n_classes, top, wide_labels, 1, 0, log_prob, entropy, stats, top_log_prob, top_class};
    const cbm::Stream on(static_cast<cudaStream_t>(stream));
    cbm::with_type(type, [&](auto t) {
        using T = decltype(t);
        Tile tile;
        if (const int e = tile_for(logits, ld, n_classes, sizeof(T), &p.shift, &tile)) {
            p.lanes = 1 << p.shift;
            with_vector<T>(e, [&](auto v) {
                const auto kernel = tile_kernel<T, decltype(v)::value>;
                cbm::launch_next(kernel, dim3(blocks_of(n_rows, tile.rows)), TILE_THREADS, tile.bytes, on, p, tile);
            });
            return;
        }
        if (n_classes > ROW_MAX) {
            const int k = blocks_to_row(n_rows, n_classes, type);
            if (k == 1 && n_classes * (int64_t)sizeof(T) < 32 * 1024) launch_clusters(long_kernel<T, 128>, n_rows, 1, 128, on, p);
            else launch_clusters(long_kernel<T, 256>, n_rows * k, k, 256, on, p);
            return;
        }
        const int values = n_classes <= 256 ? 8 : 32;
        p.shift = lanes_for(n_classes, values);
        p.lanes = 1 << p.shift;
        const dim3 grid(blocks_of(n_rows, 256 >> p.shift));
        if (values == 8) cbm::launch_next(rows_kernel<T, 8>, grid, 256, 0, on, p);
        else cbm::launch_next(rows_kernel<T, 32>, grid, 256, 0, on, p);
    });
    return launched("class_log_probs");
}

extern "C" int cbm_b200_class_log_probs_grad(const void* logits, int64_t ld, int32_t type, const void* labels, int32_t wide_labels,
                                             int64_t n_rows, int32_t n_classes, int32_t top, const float* stats, const float* entropy,
                                             const int64_t* top_class, const float* g_log_prob, const float* g_entropy,
                                             const float* g_top, void* dx, int64_t lddx, void* stream) {
    if (int rc = check("class_log_probs_grad", n_rows, ld, n_classes, top, type)) return rc;
    if (lddx < n_classes) return cbm::fail(CBM_B200_ERR_ARG, "class_log_probs_grad: rows of the gradient overlap");
    if (n_rows == 0) return CBM_B200_OK;
    if (!logits || !labels || !stats || !entropy || !dx || (g_top && top && !top_class))
        return cbm::fail(CBM_B200_ERR_ARG, "class_log_probs_grad: NULL argument");
    if (reinterpret_cast<uintptr_t>(stats) % 8) return cbm::fail(CBM_B200_ERR_ARG, "class_log_probs_grad: statistics not at 8 bytes");
    BackwardParams p{logits, labels, ld, lddx, n_rows, n_classes, top, wide_labels, 1, 0, stats, entropy, g_log_prob, g_entropy, g_top, top_class, dx};
    const cbm::Stream on(static_cast<cudaStream_t>(stream));
    cbm::with_type(type, [&](auto t) {
        using T = decltype(t);
        Tile tile, out;
        int shift;
        const int e = tile_for(logits, ld, n_classes, sizeof(T), &p.shift, &tile);
        if (e && tile_for(dx, lddx, n_classes, sizeof(T), &shift, &out) && !tile.chunks == !out.chunks) {
            p.lanes = 1 << p.shift;
            with_vector<T>(e, [&](auto v) {
                const auto kernel = tile_grad_kernel<T, decltype(v)::value>;
                cbm::launch_next(kernel, dim3(blocks_of(n_rows, tile.rows)), TILE_THREADS, tile.bytes, on, p, tile);
            });
        } else if (n_classes > ROW_MAX) {
            const int stretch = stretch_of(sizeof(T)), stretches = (n_classes + stretch - 1) / stretch;
            cbm::launch_next(long_grad_kernel<T>, dim3((unsigned)(n_rows * stretches)), THREADS, 0, on, p, stretches);
        } else {
            p.shift = lanes_for(n_classes, 8);
            p.lanes = 1 << p.shift;
            cbm::launch_next(rows_grad_kernel<T>, dim3(blocks_of(n_rows, 256 >> p.shift)), 256, 0, on, p);
        }
    });
    return launched("class_log_probs_grad");
}
