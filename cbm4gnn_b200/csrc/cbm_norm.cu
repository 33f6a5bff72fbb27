// Group norm with an activation over channels-last rows, and its gradients (sm_100a).
//
// A sample is a range of rows (a graph), a group a range of channels.  With mean and r = 1 / sqrt(var + eps) over the values of
// a sample's group:  xh = (x - mean) r,  z = w xh + b,  y = act(z).
// Gradients, with g = gy act'(z) and u = w g:  gb = sum g,  gw = sum g xh,  gx = r (u - mean(u) - xh mean(u xh)).
//
// What bounds all of it is memory: x is read and y written once, x and gy are read and gx written once.  The ways:
//   * Samples of one row: lanes hold their part of a group in registers; nothing is read twice, and the gradient computes the
//     statistics anew instead of reading them.
//   * Samples of up to a tile's rows: a team of threads reads a sample, joins its sums in registers or shared memory and reads it again,
//     out of L1 or L2, to write the results.  Tiles end where samples do, so that each of these is one team's.
//   * Longer samples: every tile leaves a partial result, a warp or a block to a sample joins them in a fixed order, and a third kernel
//     goes over the rows again, from their ends, of which L2 still holds some (of 307 MB 41, in the gradient 47 of 614).
//   * A few samples of some hundred rows: a cluster of blocks to each, which join through one another's shared memory: one launch.
//   * Groups wider than a block's threads hold: a block to each, value by value, with sums in 64 bits.
// Elsewhere means and squares around them are kept for every few rows and joined (mean and sum of squares around it of two parts give those
// of both), so that a mean far from 0 costs no digits; no sum depends on the order in which blocks run.
#include "cbm_common.h"
#include "cbm_launch.cuh"
#include "cbm_values.cuh"

#include <string>
#include <type_traits>

namespace {

using u32 = uint32_t;
using u64 = unsigned long long;

constexpr int THREADS = 256, SMS = 148;
constexpr u32 FULL = 0xffffffffu;

struct Params {
    const void *x, *gy;
    const void *w, *b;
    int64_t ldx, ldgy, ldy, n_rows, n_samples, rows_each;
    const int64_t* ptr;  // or NULL: samples of `rows_each` rows
    int c, groups, width, act, wide_params;
    float eps;
    void* y;  // or gx
    float *mean, *r;
    float *gw, *gb;
    // tiles
    int64_t tile, tiles;        // rows to a tile; tiles
    int team, slab_groups, lanes;    // threads of a team; groups of a column slab; threads of a group
    float2 *pieces, *joined;    // [2][groups][tiles], [tiles][groups]
    int64_t* longer;            // [2][tiles]: the samples that pieces are of, -1: none
    float2* channels;           // [tiles][c]: sums of g xh and g
    int64_t parts;              // of `channels`
};

template <class T>
__device__ __forceinline__ float param(const void* w, int wide, int c, float none) {
    return !w ? none : wide ? static_cast<const float*>(w)[c] : cbm::widen(static_cast<const T*>(w)[c]);
}

// By the fast forms: exp's argument and the quotient's are rounded once more, |z| U and 2 U of the result, where z itself comes with a
// rounding of |z| U.  (With expf and a division 1 000 000 x 64 bf16 in samples of 2 300 rows 143 us instead of 127, with the gradient 352
// instead of 270; 262 147 x 100 bf16 in samples of 30 84 and 67, 256 and 172.)
__device__ __forceinline__ float sigmoid(float z) { return __fdividef(1.f, 1.f + __expf(-z)); }
template <int ACT>
__device__ __forceinline__ float activated(float z) {
    if constexpr (ACT == CBM_B200_ACT_RELU) return z <= 0.f ? 0.f : z;  // NaN passes
    return ACT == CBM_B200_ACT_SILU ? z * sigmoid(z) : z;
}
template <int ACT>
__device__ __forceinline__ float slope(float z) {
    if constexpr (ACT == CBM_B200_ACT_RELU) return z <= 0.f ? 0.f : 1.f;
    if constexpr (ACT != CBM_B200_ACT_SILU) return 1.f;
    const float s = sigmoid(z);
    return s * (1.f + z * (1.f - s));
}
// Calls f with the activation as a constant: asked for value by value it costs as much as the rest.
template <class F>
__device__ __forceinline__ void with_activation(int act, F&& f) {
    if (act == CBM_B200_ACT_SILU) f(std::integral_constant<int, CBM_B200_ACT_SILU>());
    else if (act == CBM_B200_ACT_RELU) f(std::integral_constant<int, CBM_B200_ACT_RELU>());
    else f(std::integral_constant<int, CBM_B200_ACT_NONE>());
}

// The E values of a group that fall to a thread in each row.  Where rows and groups allow it they are one vector of up to 16 bytes; else
// (STRIDED) they lie `lanes` values apart, so that neighbouring threads read neighbouring values, and the last may be missing.
template <class T, int E, bool STRIDED>
struct Values {
    union {
        T v[E];
        std::conditional_t<sizeof(T) * E == 16, uint4, std::conditional_t<sizeof(T) * E == 8, uint2, std::conditional_t<sizeof(T) * E == 4, u32, uint16_t>>> bits;
    };
    __device__ Values() {}
    __device__ __forceinline__ void load(const T* p, int lanes, int there) {
        if constexpr (STRIDED) {
            // (the first again in place of a missing one, which is not used: a branch for each would make them wait for one another)
#pragma unroll
            for (int i = 0; i < E; ++i) v[i] = p[i < there ? i * lanes : 0];
        } else {
            bits = *reinterpret_cast<const decltype(bits)*>(p);
        }
    }
    __device__ __forceinline__ void store(T* p, int lanes, int there) const {
        if constexpr (STRIDED) {
#pragma unroll
            for (int i = 0; i < E; ++i)
                if (i < there) p[i * lanes] = v[i];
        } else {
            *reinterpret_cast<decltype(bits)*>(p) = bits;
        }
    }
};
// Whether a thread has an i-th value.
template <bool STRIDED>
__device__ __forceinline__ bool has(int i, int there) {
    return !STRIDED || i < there;
}
template <int E, bool STRIDED>
__device__ __forceinline__ int values_of(int lane, int lanes, int width) {
    return STRIDED ? (width - lane + lanes - 1) / lanes : E;
}

// Sum over `lanes` neighbouring lanes, a power of two.
__device__ __forceinline__ float lanes_sum(float v, int lanes) {
    for (int o = lanes >> 1; o; o >>= 1) v += __shfl_xor_sync(FULL, v, o);
    return v;
}

// ---- samples of one row ---------------------------------------------------------------------------
// The threads of a group (of up to 32: padded to a power of two; of more: to whole warps) hold its values in registers.  A thread's
// channels stay the same from row to row, so that its weights are fetched once.
struct RowShape {
    int shift;           // threads of a group, with padding: 1 << shift, or 32 times `warps`
    int warps;           // 0: up to 32 threads
    int slots, at_once;  // threads of a slab's row, rows of a block
    __host__ __device__ int padded() const { return warps ? 32 * warps : 1 << shift; }
};

// Sums of two values over a group's threads.
// (`s_warp` is another place from one sum to the next, so that a barrier for each does.)
__device__ __forceinline__ float2 group_sum(float2 v, const RowShape& h, float2 (*s_warp)[32], int& turn) {
    if (!h.warps) return float2{lanes_sum(v.x, 1 << h.shift), lanes_sum(v.y, 1 << h.shift)};
    v = float2{lanes_sum(v.x, 32), lanes_sum(v.y, 32)};
    const int warp = threadIdx.x >> 5, first = warp / h.warps * h.warps;
    float2* const here = s_warp[turn ^= 1];
    if ((threadIdx.x & 31) == 0) here[warp] = v;
    __syncthreads();
    v = here[first];
    for (int i = 1; i < h.warps; ++i) v.x += here[first + i].x, v.y += here[first + i].y;
    return v;
}

// (Bounded to the 64 registers that 1 024 threads may have, as the widest groups need; the gradient of eight values spills 316 to 420 bytes a
// thread for that, also where groups have 256 threads.)
template <class T, int E, bool STRIDED, bool GRAD>
__global__ void __launch_bounds__(1024) rows_kernel(const Params p, const RowShape h) {
    __shared__ float2 s_warp[2][32];
    int turn = 0;
    cbm::wait_before();
    const int row_in = threadIdx.x / h.slots, slot = threadIdx.x % h.slots, lane = slot % h.padded();
    const int group = blockIdx.y * p.slab_groups + slot / h.padded();
    const bool used = row_in < h.at_once && lane < p.lanes && group < p.groups;
    const int there = used ? values_of<E, STRIDED>(lane, p.lanes, p.width) : 0;
    const int at = group * p.width + (STRIDED ? lane : lane * E), stride = STRIDED ? p.lanes : 1;
    float w[E], b[E], gw[E], gb[E];
#pragma unroll
    for (int i = 0; i < E; ++i) {
        w[i] = i < there ? param<T>(p.w, p.wide_params, at + i * stride, 1.f) : 0.f;
        b[i] = i < there ? param<T>(p.b, p.wide_params, at + i * stride, 0.f) : 0.f;
        gw[i] = gb[i] = 0.f;
    }
    const float share = 1.f / (float)p.width;
    const int64_t step = (int64_t)gridDim.x * h.at_once;
    using V = Values<T, E, STRIDED>;
    V xv, gv;
    auto fetch = [&](int64_t row) {
        if (used && row < p.n_rows) {
            xv.load(static_cast<const T*>(p.x) + row * p.ldx + at, p.lanes, there);
            if (GRAD) gv.load(static_cast<const T*>(p.gy) + row * p.ldgy + at, p.lanes, there);
        }
    };
    int64_t row = (int64_t)blockIdx.x * h.at_once + row_in;
    fetch(row);
    // (all threads of a block take the same number of turns)
    for (int64_t first = (int64_t)blockIdx.x * h.at_once; first < p.n_rows; first += step, row += step) {
        const int now = row < p.n_rows ? there : 0;
        float x[E], u[E];
        float2 s{0.f, 0.f};
#pragma unroll
        for (int i = 0; i < E; ++i) {
            x[i] = i < now ? cbm::widen(xv.v[i]) : 0.f;
            if (GRAD) u[i] = i < now ? cbm::widen(gv.v[i]) : 0.f;
            s.x += x[i];
        }
        fetch(row + step);  // on its way meanwhile
        const float mean = group_sum(s, h, s_warp, turn).x * share;
        s.x = 0.f;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            x[i] = i < now ? x[i] - mean : 0.f;
            s.x += x[i] * x[i];
        }
        const float r = rsqrtf(group_sum(s, h, s_warp, turn).x * share + p.eps);
        V out;
        if constexpr (!GRAD) {
            with_activation(p.act, [&](auto act) {
#pragma unroll
                for (int i = 0; i < E; ++i) out.v[i] = cbm::narrow<T>(activated<decltype(act)::value>(x[i] * (r * w[i]) + b[i]));
            });
        } else {
            s.x = 0.f;
            with_activation(p.act, [&](auto act) {
#pragma unroll
                for (int i = 0; i < E; ++i) {
                    x[i] *= r;
                    const float g = u[i] * slope<decltype(act)::value>(x[i] * w[i] + b[i]);
                    gw[i] += g * x[i];
                    gb[i] += g;
                    u[i] = g * w[i];
                    s.x += u[i];
                    s.y += u[i] * x[i];
                }
            });
            s = group_sum(s, h, s_warp, turn);
#pragma unroll
            for (int i = 0; i < E; ++i) out.v[i] = cbm::narrow<T>(r * (u[i] - s.x * share - x[i] * (s.y * share)));
        }
        if (now) out.store(static_cast<T*>(p.y) + row * p.ldy + at, p.lanes, there);
    }
    if constexpr (GRAD) {
        if (!p.channels) return;
        // the block's rows, one after the other
        extern __shared__ float2 s_sum[];
#pragma unroll
        for (int i = 0; i < E; ++i) {
            __syncthreads();
            s_sum[threadIdx.x] = float2{gw[i], gb[i]};
            __syncthreads();
            if (row_in == 0 && i < there) {
                float2 all = s_sum[slot];
                for (int q = 1; q < h.at_once; ++q) {
                    const float2 one = s_sum[q * h.slots + slot];
                    all.x += one.x, all.y += one.y;
                }
                p.channels[(int64_t)blockIdx.x * p.c + at + i * stride] = all;
            }
        }
    }
}

// ---- samples of several rows ----------------------------------------------------------------------
// Row at which sample s starts; what a pointer array says is kept inside the rows there are.
__device__ __forceinline__ int64_t start_of(const Params& p, int64_t s) {
    return p.ptr ? min(max(p.ptr[s], (int64_t)0), p.n_rows) : s * p.rows_each;
}
// The last samples that start at `row` and at `other` or before them, -1: none.  Half a warp's lanes each try 16 places at a time.
__device__ __forceinline__ void samples_at(const Params& p, int64_t row, int64_t other, int64_t& s, int64_t& t) {
    if (!p.ptr) {
        s = p.rows_each ? min(row / p.rows_each, p.n_samples - 1) : p.n_samples - 1;
        t = p.rows_each ? min(other / p.rows_each, p.n_samples - 1) : p.n_samples - 1;
        return;
    }
    const int lane = threadIdx.x & 15, upper = threadIdx.x & 16;
    if (upper) row = other;
    int64_t lo = 0, hi = p.n_samples + 1;  // entries before lo are <= row, those from hi on are larger
    while (__any_sync(FULL, lo < hi)) {
        const int64_t each = (hi - lo + 15) / 16, probe = lo + each * lane + each - 1;
        const bool below = lo < hi && probe < hi && p.ptr[probe] <= row;
        const int n = __popc(__ballot_sync(FULL, below) >> upper & 0xffffu);
        const int64_t from = lo;
        lo = min(from + each * n, hi);
        hi = max(lo, min(hi, from + each * (n + 1) - 1));
    }
    s = __shfl_sync(FULL, lo, 0) - 1;
    t = __shfl_sync(FULL, lo, 16) - 1;
}
// Where the tile that should start at `row`, where sample s lies, does: samples that are no longer than a tile are not cut.
__device__ __forceinline__ int64_t tile_start(const Params& p, int64_t row, int64_t s) {
    if (row >= p.n_rows) return p.n_rows;
    if (s < 0 || s >= p.n_samples) return row;
    const int64_t a = start_of(p, s), e = start_of(p, s + 1);
    return row < e && e - a <= p.tile ? a : row;
}

struct Team {
    int id, thread, size;              // of the block's; of the team's
    int groups, vectors, at_once;      // of the slab; threads of its rows, rows at once
    int group0, row_in, group, lane;   // this thread's; row_in >= at_once: none
    int channel, there;                // first of its values, and how many
    bool flat;                         // a warp whose groups' threads are told apart by bits of their numbers
    __device__ __forceinline__ Team(const Params& p, int E, bool strided) {
        size = p.team;
        id = threadIdx.x / size, thread = threadIdx.x % size;
        group0 = blockIdx.y * p.slab_groups;
        groups = min(p.slab_groups, p.groups - group0);
        vectors = groups * p.lanes;
        at_once = size / vectors;
        row_in = thread / vectors;
        group = group0 + thread % vectors / p.lanes, lane = thread % p.lanes;
        if (row_in >= at_once) group = group0, lane = 0;
        else lane = thread % vectors % p.lanes;
        channel = group * p.width + (strided ? lane : lane * E);
        there = strided ? (p.width - lane + p.lanes - 1) / p.lanes : E;
        flat = size == 32 && !(p.lanes & (p.lanes - 1)) && !(vectors & (vectors - 1));
    }
    // Rows, of `rows`, of row r of those at work at once: one division for all of them.
    __device__ __forceinline__ int turns(int rows, int r) const {
        const u32 each = (u32)rows / (u32)at_once;
        return (int)each + (r < rows - (int)each * at_once);
    }
    // Sum over a group's threads, flat teams only: all of them get it.
    __device__ __forceinline__ float flat_sum(float v, int lanes) const {
        for (int o = 1; o < lanes; o <<= 1) v += __shfl_xor_sync(FULL, v, o);
        for (int o = vectors; o < 32; o <<= 1) v += __shfl_xor_sync(FULL, v, o);
        return v;
    }
    __device__ __forceinline__ bool on() const { return row_in < at_once; }
    __device__ __forceinline__ void sync() const {
        if (size == 32) __syncwarp();
        else asm volatile("barrier.sync %0, %1;" ::"r"(id + 1), "r"(size) : "memory");
    }
};

// What two parts of a group come to: the mean of all values and the squares around it, or (not MEANS) sums of two values.  `part` holds
// what each thread of a team found in `rows` rows: the mean over its values of all its rows and the squares around it, or its sums.
template <bool MEANS, int E, bool STRIDED>
struct Join {
    const Params& p;
    const Team& t;
    const float2* part;  // of the group
    int rows;
    // By one thread: f(what a thread left, how many values it is of).
    template <class F>
    __device__ __forceinline__ void alone(F&& f) const {
        const int most = min(t.at_once, rows);
        const float2* at = part;
        for (int r = 0; r < most; ++r, at += t.vectors) {
            const int n = t.turns(rows, r);
            const float full = (float)(n * E);
            for (int l = 0; l < p.lanes; ++l) f(at[l], STRIDED ? (float)(n * values_of<E, STRIDED>(l, p.lanes, p.width)) : full);
        }
    }
    // By a warp.
    template <class F>
    __device__ __forceinline__ void together(F&& f) const {
        const int entries = min(t.at_once, rows) * p.lanes;
        for (int i = threadIdx.x & 31; i < entries; i += 32) {
            const int r = i / p.lanes, l = i - r * p.lanes;
            f(part[r * t.vectors + l], (float)(t.turns(rows, r) * values_of<E, STRIDED>(l, p.lanes, p.width)));
        }
    }
    template <bool WARP>
    __device__ __forceinline__ float2 run() const {
        float2 s{0.f, 0.f};
        if (rows == 0) return s;
        auto each = [&](auto&& f) {
            if constexpr (WARP) together(f);
            else alone(f);
        };
        auto sum = [&](float v) { return WARP ? lanes_sum(v, 32) : v; };
        if constexpr (MEANS) {
            const float ref = part[0].x;
            each([&](float2 one, float n) { s.x += n * (one.x - ref); });
            s.x = ref + sum(s.x) / ((float)rows * (float)p.width);
            each([&](float2 one, float n) { s.y += one.y + n * (one.x - s.x) * (one.x - s.x); });
            s.y = sum(s.y);
        } else {
            each([&](float2 one, float) { s.x += one.x, s.y += one.y; });
            s = float2{sum(s.x), sum(s.y)};
        }
        return s;
    }
};
// The same out of registers, by a flat team.
template <bool MEANS>
__device__ __forceinline__ float2 joined_flat(const Params& p, const Team& t, float2 mine, int rows) {
    if constexpr (!MEANS) return float2{t.flat_sum(mine.x, p.lanes), t.flat_sum(mine.y, p.lanes)};
    const float ref = __shfl_sync(FULL, mine.x, (t.group - t.group0) * p.lanes), n = (float)(t.turns(rows, t.row_in) * t.there);
    const float mean = ref + t.flat_sum(n * (mine.x - ref), p.lanes) / ((float)rows * (float)p.width);
    return float2{mean, t.flat_sum(mine.y + n * (mine.x - mean) * (mine.x - mean), p.lanes)};
}
// A group of few threads is joined by each of them for itself, which saves the way through shared memory and a barrier.
constexpr int FEW = 32;

// A number of rows that is known beforehand.
template <int N>
struct All {
    __device__ __forceinline__ constexpr operator int() const { return N; }
};
// The gradient's vectors of 16 bytes come through shared memory, where each thread has DEPTH places of its own: rows ahead take no registers,
// the code of a turn is that of one row, and the rows of a short sample are still there when they are asked for again.  (1 000 000 x 64 bf16 in
// samples of 2 300 rows, with the gradient 465 -> 364 us; 235 868 x 256 fp32 350 -> 342.  Narrower vectors lose: 262 147 x 100 bf16 by pairs
// 262 -> 290; so does the forward pass, whose turns are short: 102 -> 143.)
template <class T, int E, bool STRIDED, bool GRAD>
struct Ring {
    static constexpr int VECTOR = E * sizeof(T), DEPTH = 4;
    static constexpr bool ON = GRAD && !STRIDED && VECTOR == 16;
    static constexpr int ROWS = ON ? DEPTH * 2 * VECTOR : 0, CHANNELS = GRAD ? 8 * E : 0;
    static constexpr int EACH = ROWS > CHANNELS ? ROWS : CHANNELS;  // bytes to a thread; behind its rows, a team's channels' sums use them
    static constexpr int BYTES = EACH ? EACH * THREADS : 16;
    unsigned char *team, *at;  // this team's places, this thread's first
    int apart;
    __device__ __forceinline__ Ring(unsigned char* smem, const Team& t)
        : team(smem + t.id * t.size * EACH), at(team + t.thread * VECTOR), apart(t.size * VECTOR) {}
    __device__ __forceinline__ unsigned char* place(int row, int which) const { return at + ((row & (DEPTH - 1)) * 2 + which) * apart; }
    __device__ __forceinline__ void copy(const T* from, int row, int which) const {
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"((u32)__cvta_generic_to_shared(place(row, which))), "l"(from), "n"(VECTOR) : "memory");
    }
    // Whether `count` rows that were gone over are all there.
    __device__ __forceinline__ bool keeps(int count) const { return ON && count <= DEPTH; }
};
// Rows that a thread takes at a time: out of its places one, else as many as it fetches.
template <class T, int E, bool STRIDED, bool GRAD>
__host__ __device__ constexpr int batch_of() {
    return Ring<T, E, STRIDED, GRAD>::ON ? 1 : STRIDED ? (E == 1 ? 8 : E == 4 || !GRAD ? 4 : 2) : E * sizeof(T) >= 8 ? 4 : 8;
}
// Calls f(values, values of the gradient, how many rows) for the `count` rows from x on, `dx` apart, a batch at a time; where `kept`, they are
// in their places already.  The last rows of a fetch are fetched without a question about each, the last one again in place of those that are
// not there: as branches the fetches would come one after the other.
template <class T, int E, bool STRIDED, bool GRAD, class F>
__device__ __forceinline__ void for_rows(const Ring<T, E, STRIDED, GRAD>& ring, bool kept, const T* x, const T* gy, int64_t dx, int64_t dg, int count,
                                         int lanes, int there, F&& f) {
    constexpr int BATCH = batch_of<T, E, STRIDED, GRAD>();
    Values<T, E, STRIDED> v[BATCH], g[GRAD ? BATCH : 1];
    if constexpr (Ring<T, E, STRIDED, GRAD>::ON) {
        constexpr int AHEAD = Ring<T, E, STRIDED, GRAD>::DEPTH - 1;
        int asked = 0;
        auto ask = [&] {  // (a group of copies for each row, where there are no more an empty one)
            if (asked < count) {
                ring.copy(x, asked, 0), x += dx;
                ring.copy(gy, asked, 1), gy += dg;
            }
            ++asked;
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        if (!kept)
#pragma unroll 1
            while (asked < AHEAD) ask();
#pragma unroll 1
        for (int i = 0; i < count; ++i) {
            if (!kept) {
                ask();  // into the place of the row before this one, which is done with
                asm volatile("cp.async.wait_group %0;" ::"n"(AHEAD) : "memory");
            }
            v[0].bits = *reinterpret_cast<const uint4*>(ring.place(i, 0));
            g[0].bits = *reinterpret_cast<const uint4*>(ring.place(i, 1));
            f(v, g, All<1>());
        }
    } else {
        for (; count >= BATCH; count -= BATCH) {
#pragma unroll
            for (int k = 0; k < BATCH; ++k) {
                v[k].load(x, lanes, there), x += dx;
                if constexpr (GRAD) g[k].load(gy, lanes, there), gy += dg;
            }
            f(v, g, All<BATCH>());
        }
        if (count > 0) {
            const int have = count;
#pragma unroll
            for (int k = 0; k < BATCH; ++k) {
                v[k].load(x, lanes, there);
                if constexpr (GRAD) g[k].load(gy, lanes, there);
                if (k + 1 < have) x += dx, gy += dg;
            }
            f(v, g, have);
        }
    }
}

// y, or gx, from the statistics (mean, r) and, for the gradient, the means of u and u xh.
template <class T, int E, bool STRIDED, bool GRAD, int ACT>
__device__ __forceinline__ Values<T, E, STRIDED> finished(const Values<T, E, STRIDED>& x, const Values<T, E, STRIDED>& gy, const float (&w)[E],
                                                          const float (&b)[E], float2 stat, float2 sums) {
    Values<T, E, STRIDED> to;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const float d = cbm::widen(x.v[i]) - stat.x, z = d * (stat.y * w[i]) + b[i];
        if constexpr (GRAD) {
            const float u = cbm::widen(gy.v[i]) * slope<ACT>(z) * w[i];
            to.v[i] = cbm::narrow<T>(stat.y * (u - sums.x - d * stat.y * sums.y));
        } else {
            to.v[i] = cbm::narrow<T>(activated<ACT>(z));
        }
    }
    return to;
}

// Rows [lo, hi) of a sample, from the last row to the first where BACK.
template <class T, int E, bool STRIDED, bool GRAD, bool BACK>
__device__ __forceinline__ void write_rows(const Params& p, const Team& t, const Ring<T, E, STRIDED, GRAD>& ring, bool kept, int64_t lo, int64_t hi, const float (&w)[E], const float (&b)[E],
                                           float2 stat, float2 sums) {
    const int64_t first = lo + t.row_in;
    if (!t.on() || first >= hi) return;
    const int count = t.turns((int)(hi - lo), t.row_in);  // (at most two tiles, or a block's part of a short sample: they fit 31 bits)
    const int64_t begin = BACK ? first + (int64_t)(count - 1) * t.at_once : first, step = BACK ? -t.at_once : t.at_once;
    T* y = static_cast<T*>(p.y) + t.channel + begin * p.ldy;
    const int64_t dy = step * p.ldy;
    with_activation(p.act, [&](auto act) {
        constexpr int BATCH = batch_of<T, E, STRIDED, GRAD>();
        for_rows<T, E, STRIDED, GRAD>(ring, kept && ring.keeps(count), static_cast<const T*>(p.x) + t.channel + begin * p.ldx, static_cast<const T*>(p.gy) + t.channel + begin * p.ldgy,
                                      step * p.ldx, step * p.ldgy, count, p.lanes, t.there, [&](const auto& v, const auto& g, auto have) {
#pragma unroll
            for (int k = 0; k < BATCH; ++k) {
                const auto out = finished<T, E, STRIDED, GRAD, decltype(act)::value>(v[k], g[GRAD ? k : 0], w, b, stat, sums);
                if (k < have) out.store(y, p.lanes, t.there), y += dy;
            }
        });
    });
}

template <class T, int E, bool STRIDED>
__device__ __forceinline__ void fetch_params(const Params& p, const Team& t, float (&w)[E], float (&b)[E]) {
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const bool on = t.on() && has<STRIDED>(i, t.there);
        w[i] = on ? param<T>(p.w, p.wide_params, t.channel + i * (STRIDED ? p.lanes : 1), 1.f) : 0.f;
        b[i] = on ? param<T>(p.b, p.wide_params, t.channel + i * (STRIDED ? p.lanes : 1), 0.f) : 0.f;
    }
}

// Blocks of an SM: with one fewer too little is on its way.  Some forms spill registers at that, by -Xptxas -v: tiles of single values up to
// 460 bytes a thread, of pairs in the gradient 224, of four fp32 144, of eight 16-bit ones 144; clusters of single values up to 916.  With
// one block more all of them do.
constexpr int blocks_resident(int e, bool grad) { return e == 8 ? (grad ? 2 : 3) : e == 4 && grad ? 3 : 4; }

// What a thread finds in `rows` rows of a sample from row lo on: the mean over its values and the squares around it; or, for the gradient,
// its sums of u and u xh, and by channel those of g xh and g, added to gw and gb.
template <class T, int E, bool STRIDED, bool GRAD>
__device__ __forceinline__ float2 gathered(const Params& p, const Team& t, const Ring<T, E, STRIDED, GRAD>& ring, int64_t lo, int rows, const float (&w)[E], const float (&b)[E], float2 at,
                                           float (&gw)[E], float (&gb)[E]) {
    constexpr int BATCH = batch_of<T, E, STRIDED, GRAD>();
    const T *x = static_cast<const T*>(p.x) + t.channel, *gy = static_cast<const T*>(p.gy) + t.channel;
    float2 mine{0.f, 0.f};
    if (!t.on()) return mine;
    float mean[E], m2[E];  // of each channel (also of missing ones, which are left out in the end); for the gradient the sums of g xh and g
    int n = 0;
#pragma unroll
    for (int i = 0; i < E; ++i) mean[i] = m2[i] = 0.f;
    auto rows_of = [&](auto&& f) {
        for_rows<T, E, STRIDED, GRAD>(ring, false, x + (lo + t.row_in) * p.ldx, gy + (lo + t.row_in) * p.ldgy, t.at_once * p.ldx, t.at_once * p.ldgy,
                                      t.turns(rows, t.row_in), p.lanes, t.there, f);
    };
    if constexpr (GRAD) {
        with_activation(p.act, [&](auto act) {
            rows_of([&](const auto& v, const auto& gv, auto have) {
#pragma unroll
                for (int k = 0; k < BATCH; ++k)
#pragma unroll
                    for (int i = 0; i < E; ++i) {
                        const float xh = (cbm::widen(v[k].v[i]) - at.x) * at.y;
                        const float g = k < have ? cbm::widen(gv[k].v[i]) * slope<decltype(act)::value>(xh * w[i] + b[i]) : 0.f;
                        mean[i] += g * xh;
                        m2[i] += g;
                    }
            });
        });
    } else {
        rows_of([&](const auto& v, const auto&, auto have) {
            const float share = 1.f / (float)have, to_mean = (float)have / (float)(n + have), to_squares = (float)n * to_mean;
#pragma unroll
            for (int i = 0; i < E; ++i) {
                float sum = 0.f, squares = 0.f;
#pragma unroll
                for (int k = 0; k < BATCH; ++k) sum += k < have ? cbm::widen(v[k].v[i]) : 0.f;
                const float here = sum * share;
#pragma unroll
                for (int k = 0; k < BATCH; ++k) {
                    const float d = k < have ? cbm::widen(v[k].v[i]) - here : 0.f;
                    squares += d * d;
                }
                const float d = here - mean[i];
                mean[i] += d * to_mean;
                m2[i] += squares + d * d * to_squares;
            }
            n += have;
        });
    }
    if constexpr (GRAD) {
#pragma unroll
        for (int i = 0; i < E; ++i) {
            mine.x += m2[i] * w[i];    // u
            mine.y += mean[i] * w[i];  // u xh
            gw[i] += mean[i];
            gb[i] += m2[i];
        }
    } else {
        float shift = 0.f;
#pragma unroll
        for (int i = 1; i < E; ++i) shift += has<STRIDED>(i, t.there) ? mean[i] - mean[0] : 0.f;
        mine.x = mean[0] + shift / (float)t.there;
#pragma unroll
        for (int i = 0; i < E; ++i)
            if (has<STRIDED>(i, t.there)) mine.y += m2[i] + (float)n * (mean[i] - mine.x) * (mean[i] - mine.x);
    }
    return mine;
}

// A team's sums of g xh and g, as part `to`.
template <class T, int E, bool STRIDED>
__device__ __forceinline__ void store_channels(const Params& p, const Team& t, const float (&gw)[E], const float (&gb)[E], float2* s_channel, int64_t to) {
    t.sync();  // (where the rows' places were)
#pragma unroll
    for (int i = 0; i < E; ++i) s_channel[i * t.size + t.thread] = float2{gw[i], gb[i]};
    t.sync();
    if (t.row_in) return;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        if (!has<STRIDED>(i, t.there)) break;
        float2 all = s_channel[i * t.size + t.thread];
        for (int q = 1; q < t.at_once; ++q) {
            const float2 one = s_channel[i * t.size + t.thread + q * t.vectors];
            all.x += one.x, all.y += one.y;
        }
        p.channels[to * p.c + t.channel + i * (STRIDED ? p.lanes : 1)] = all;
    }
}

// A team to a tile: samples that lie in it are done with, of longer ones their part is left in `pieces`.
template <class T, int E, bool STRIDED, bool GRAD>
__global__ void __launch_bounds__(THREADS, blocks_resident(E, GRAD)) tiles_kernel(const Params p) {
    __shared__ float2 s_part[2][THREADS], s_stat[THREADS];  // (parts: of this sample and of the one before, which may still be read)
    __shared__ __align__(16) unsigned char s_rows[Ring<T, E, STRIDED, GRAD>::BYTES];
    cbm::wait_before();
    const Team t(p, E, STRIDED);
    const Ring<T, E, STRIDED, GRAD> ring(s_rows, t);
    const int64_t tile = (int64_t)blockIdx.x * (THREADS / p.team) + t.id;
    if (tile >= p.tiles) return;
    float2 *part = s_part[0] + t.id * t.size, *stat = s_stat + t.id * t.size;
    float w[E], b[E], gw[E], gb[E];
    fetch_params<T, E, STRIDED>(p, t, w, b);
#pragma unroll
    for (int i = 0; i < E; ++i) gw[i] = gb[i] = 0.f;
    int64_t s, after;
    samples_at(p, tile * p.tile, (tile + 1) * p.tile, s, after);
    const int64_t tb = tile_start(p, tile * p.tile, s), te = tile_start(p, (tile + 1) * p.tile, after);
    if (p.longer && t.thread < 2 && blockIdx.y == 0) p.longer[t.thread * p.tiles + tile] = -1;
    t.sync();
    if (p.ptr && tb < te) {  // rows of no sample
        const int64_t head = p.n_samples ? start_of(p, 0) : p.n_rows, tail = p.n_samples ? start_of(p, p.n_samples) : p.n_rows;
        Values<T, E, STRIDED> none;
#pragma unroll
        for (int i = 0; i < E; ++i) none.v[i] = cbm::narrow<T>(0.f);
        T* y = static_cast<T*>(p.y) + t.channel;
        for (int64_t row = tb + t.row_in; t.on() && row < min(te, head); row += t.at_once) none.store(y + row * p.ldy, p.lanes, t.there);
        for (int64_t row = max(tb, tail) + t.row_in; t.on() && row < te; row += t.at_once) none.store(y + row * p.ldy, p.lanes, t.there);
    }
    // (the sample at the tile's nominal start is the one at its start, too; where several start there, those before the last are empty)
    s = tb < te ? max(s, (int64_t)0) : p.n_samples;
    int64_t a = s < p.n_samples ? start_of(p, s) : te, next = s < p.n_samples ? start_of(p, s + 1) : te, e;
    for (; s < p.n_samples && a < te; ++s, a = e) {
        e = next;
        if (s + 1 < p.n_samples) next = start_of(p, s + 2);  // on its way meanwhile
        const int64_t lo = max(a, tb), hi = min(e, te);
        if (lo >= hi) continue;
        const int rows = (int)(hi - lo);  // (at most two tiles, which fit 31 bits)
        float2 at{0.f, 0.f};
        if constexpr (GRAD) at = float2{p.mean[s * p.groups + t.group], p.r[s * p.groups + t.group]};
        const float2 mine = gathered<T, E, STRIDED, GRAD>(p, t, ring, lo, rows, w, b, at, gw, gb);
        if (!t.flat) {
            part[t.thread] = mine;
            t.sync();
        }
        const float share = 1.f / ((float)rows * (float)p.width);
        const bool whole = e - a <= p.tile;
        // for a group: what was found, from its threads' joined parts
        auto finish = [&](int group, float2 all, bool writes) {
            if (!whole) {
                const int64_t slot = a > tile * p.tile ? 1 : 0;  // a longer sample that starts inside the tile is its second one
                if (writes) p.pieces[(slot * p.groups + group) * p.tiles + tile] = all;
                return all;
            }
            if constexpr (GRAD) return float2{all.x * share, all.y * share};
            const float2 found{all.x, rsqrtf(all.y * share + p.eps)};
            if (writes && p.mean) {
                p.mean[s * p.groups + group] = found.x;
                p.r[s * p.groups + group] = found.y;
            }
            return found;
        };
        float2 found{0.f, 0.f};
        if (t.flat) {
            found = finish(t.group, joined_flat<!GRAD>(p, t, mine, rows), t.row_in == 0 && t.lane == 0);
        } else if (p.lanes * t.at_once <= FEW) {
            const Join<!GRAD, E, STRIDED> join{p, t, part + (t.group - t.group0) * p.lanes, rows};
            found = finish(t.group, join.template run<false>(), t.row_in == 0 && t.lane == 0);
            part = part == s_part[0] + t.id * t.size ? s_part[1] + t.id * t.size : s_part[0] + t.id * t.size;
        } else {
            for (int g = t.thread >> 5; g < t.groups; g += t.size >> 5) {
                const Join<!GRAD, E, STRIDED> join{p, t, part + g * p.lanes, rows};
                const float2 one = finish(t.group0 + g, join.template run<true>(), (t.thread & 31) == 0);
                if ((t.thread & 31) == 0) stat[g] = one;
            }
            t.sync();
            found = stat[t.group - t.group0];
        }
        if (!whole) {
            if (t.thread == 0 && blockIdx.y == 0) p.longer[(a > tile * p.tile ? p.tiles : 0) + tile] = s;
            continue;
        }
        write_rows<T, E, STRIDED, GRAD, false>(p, t, ring, true, lo, hi, w, b, GRAD ? at : found, found);
    }
    if constexpr (GRAD) {
        if (p.channels) store_channels<T, E, STRIDED>(p, t, gw, gb, reinterpret_cast<float2*>(ring.team), tile);
    }
}

// The pieces of each sample that is longer than a tile: by a warp, or where they are many by a block.  Block x: JOINED tiles, for the samples
// that start in them, or where samples are equal, JOINED samples; y: the groups y, y + gridDim.y, ...  The blocks behind add up the channels'
// sums, CHANNELS each.
constexpr int JOINERS = 256, JOINED = JOINERS / 32, MANY = 128, CHANNELS = 4;

__device__ __forceinline__ float joiners_sum(float v, float* s_sum) {
    v = lanes_sum(v, 32);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s_sum[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int i = 0; i < JOINERS / 32; ++i) v += s_sum[i];
    return v;
}

// Sample s, which starts in `tile`, [a, e), by the threads `at` of `size`, whose values `sum` adds up.
template <bool GRAD, class Sum>
__device__ __forceinline__ void join_sample(const Params& p, int64_t s, int64_t a, int64_t e, int at, int size, Sum&& sum) {
    const int64_t tile = a / p.tile, last = (e - 1) / p.tile;
    const float count = (float)(e - a) * (float)p.width;
    for (int g = blockIdx.y; g < p.groups; g += gridDim.y) {
        const float2* found = p.pieces + (int64_t)g * p.tiles;
        // of the first tile it is the second piece unless the sample starts with the tile
        auto piece = [&](int64_t q) { return found[(q == tile && a > tile * p.tile ? p.groups * p.tiles : 0) + q]; };
        if constexpr (GRAD) {
            float2 all{0.f, 0.f};
#pragma unroll 4
            for (int64_t q = tile + at; q <= last; q += size) {
                const float2 one = piece(q);
                all.x += one.x, all.y += one.y;
            }
            all = float2{sum(all.x), sum(all.y)};
            if (at == 0) p.joined[tile * p.groups + g] = float2{all.x / count, all.y / count};
        } else {
            auto rows = [&](int64_t q) { return (float)(min(e, (q + 1) * p.tile) - max(a, q * p.tile)); };
            const float ref = piece(tile).x;
            float m = 0.f, squares = 0.f;
#pragma unroll 4
            for (int64_t q = tile + at; q <= last; q += size) m += rows(q) * (piece(q).x - ref);
            const float mean = ref + sum(m) / (float)(e - a);
#pragma unroll 4
            for (int64_t q = tile + at; q <= last; q += size) {
                const float2 one = piece(q);
                squares += one.y + rows(q) * (float)p.width * (one.x - mean) * (one.x - mean);
            }
            const float r = rsqrtf(sum(squares) / count + p.eps);
            if (at == 0) {
                p.joined[tile * p.groups + g] = float2{mean, r};
                if (p.mean) {
                    p.mean[s * p.groups + g] = mean;
                    p.r[s * p.groups + g] = r;
                }
            }
        }
    }
}

template <class T, bool GRAD>
__global__ void __launch_bounds__(JOINERS) join_kernel(const Params p, const int64_t starts) {
    __shared__ float s_sum[JOINERS / 32];
    __shared__ int64_t s_long[JOINED];
    cbm::wait_before();
    const int64_t blocks = (starts + JOINED - 1) / JOINED;
    const int warp = threadIdx.x >> 5;
    if (blockIdx.x < blocks) {
        const int64_t mine = (int64_t)blockIdx.x * JOINED + warp;
        int64_t s = mine < starts ? mine : -1, a = 0, e = 0;
        if (p.ptr && s >= 0) {
            // (a sample that starts with the tile fills it)
            s = p.longer[p.tiles + mine];
            if (s < 0) s = p.longer[mine];
        }
        if (s >= 0) {
            a = start_of(p, s), e = start_of(p, s + 1);
            if (p.ptr && a < mine * p.tile) s = -1;
        }
        const bool many = s >= 0 && e - a > MANY * p.tile;
        if (s >= 0 && !many) join_sample<GRAD>(p, s, a, e, threadIdx.x & 31, 32, [](float v) { return lanes_sum(v, 32); });
        if ((threadIdx.x & 31) == 0) s_long[warp] = many ? s : -1;
        if (!__syncthreads_or(many)) return;
        for (int i = 0; i < JOINED; ++i) {
            s = s_long[i];
            if (s >= 0) join_sample<GRAD>(p, s, start_of(p, s), start_of(p, s + 1), threadIdx.x, JOINERS, [&](float v) { return joiners_sum(v, s_sum); });
        }
    } else if constexpr (GRAD) {
        if (blockIdx.y) return;
        __shared__ float2 s_part[JOINED][CHANNELS];
        const int column = threadIdx.x % CHANNELS, c = (int)(blockIdx.x - blocks) * CHANNELS + column;
        float2 all{0.f, 0.f};
        if (c < p.c)
#pragma unroll 8
            for (int64_t q = threadIdx.x / CHANNELS; q < p.parts; q += JOINERS / CHANNELS) {
                const float2 one = p.channels[q * p.c + c];
                all.x += one.x, all.y += one.y;
            }
#pragma unroll
        for (int o = CHANNELS; o < 32; o <<= 1) all.x += __shfl_xor_sync(FULL, all.x, o), all.y += __shfl_xor_sync(FULL, all.y, o);
        if ((threadIdx.x & 31) < CHANNELS) s_part[warp][column] = all;
        __syncthreads();
        if (threadIdx.x < CHANNELS && c < p.c) {
            for (int i = 1; i < JOINED; ++i) all.x += s_part[i][column].x, all.y += s_part[i][column].y;
            if (p.gw) p.gw[c] = all.x;
            if (p.gb) p.gb[c] = all.y;
        }
    }
}

// The rows of samples that are longer than a tile: at most two of them meet in one.
template <class T, int E, bool STRIDED, bool GRAD>
__global__ void __launch_bounds__(THREADS, blocks_resident(E, GRAD)) long_kernel(const Params p) {
    __shared__ __align__(16) unsigned char s_rows[Ring<T, E, STRIDED, GRAD>::BYTES];
    cbm::wait_before();
    const Team t(p, E, STRIDED);
    const Ring<T, E, STRIDED, GRAD> ring(s_rows, t);
    const int64_t tile = (int64_t)blockIdx.x * (THREADS / p.team) + t.id;
    if (tile >= p.tiles) return;
    float w[E], b[E];
    fetch_params<T, E, STRIDED>(p, t, w, b);
    const int64_t begin = tile * p.tile, end = min(begin + p.tile, p.n_rows);
    for (int k = 1; k >= 0; --k) {
        const int64_t s = p.longer[k * p.tiles + tile];
        if (s < 0) continue;
        const int64_t a = start_of(p, s), e = start_of(p, s + 1);
        const int64_t lo = max(a, begin), hi = min(e, end);
        const float2 found = p.joined[(a / p.tile) * p.groups + t.group];
        float2 at = found;
        if constexpr (GRAD) at = float2{p.mean[s * p.groups + t.group], p.r[s * p.groups + t.group]};
        if (lo < hi) write_rows<T, E, STRIDED, GRAD, true>(p, t, ring, false, lo, hi, w, b, at, found);
    }
}

// ---- a few samples that are not long: a cluster of blocks to each ----------------------------------
constexpr int CLUSTER = 8, GROUPS = 128;  // blocks to a sample; groups of a slab at most

// Every block has a stretch of the sample's rows; what it finds goes to all blocks of the cluster, which read their rows again, out of L1 or
// L2: one launch, where tiles, joins and rows take three.  y: a slab of groups.
template <class T, int E, bool STRIDED, bool GRAD>
__global__ void __launch_bounds__(THREADS, blocks_resident(E, GRAD)) cluster_kernel(const Params p) {
    __shared__ float2 s_part[THREADS], s_stat[THREADS], s_all[CLUSTER][GROUPS];
    __shared__ __align__(16) unsigned char s_rows[Ring<T, E, STRIDED, GRAD>::BYTES];
    u32 rank;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");  // the others' shared memory is there once all have started
    cbm::wait_before();
    const Team t(p, E, STRIDED);
    const Ring<T, E, STRIDED, GRAD> ring(s_rows, t);
    const int64_t s = blockIdx.x / CLUSTER, each = (p.rows_each + CLUSTER - 1) / CLUSTER;
    auto rows_of = [&](int64_t k) { return (int)max(min(p.rows_each - k * each, each), (int64_t)0); };
    const int64_t lo = s * p.rows_each + min(rank * each, p.rows_each);
    const int rows = rows_of(rank);
    float w[E], b[E], gw[E], gb[E];
    fetch_params<T, E, STRIDED>(p, t, w, b);
#pragma unroll
    for (int i = 0; i < E; ++i) gw[i] = gb[i] = 0.f;
    float2 at{0.f, 0.f};
    if constexpr (GRAD) at = float2{p.mean[s * p.groups + t.group], p.r[s * p.groups + t.group]};
    s_part[t.thread] = gathered<T, E, STRIDED, GRAD>(p, t, ring, lo, rows, w, b, at, gw, gb);
    __syncthreads();
    for (int g = t.thread >> 5; g < t.groups; g += THREADS / 32) {
        const Join<!GRAD, E, STRIDED> join{p, t, s_part + g * p.lanes, rows};
        const float2 one = join.template run<true>();
        if ((t.thread & 31) == 0) s_stat[g] = one;
    }
    __syncthreads();
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
    for (int i = t.thread; i < t.groups * CLUSTER; i += THREADS) {
        const int to = i / t.groups, g = i - to * t.groups;
        u32 place;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(place) : "r"((u32)__cvta_generic_to_shared(&s_all[rank][g])), "r"(to));
        asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(place), "f"(s_stat[g].x), "f"(s_stat[g].y) : "memory");
    }
    asm volatile("barrier.cluster.arrive.release;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
    const int mine = t.group - t.group0;
    const float share = 1.f / ((float)p.rows_each * (float)p.width);
    float2 found{0.f, 0.f};
    if constexpr (GRAD) {
        for (int k = 0; k < CLUSTER; ++k) found.x += s_all[k][mine].x, found.y += s_all[k][mine].y;
        found = float2{found.x * share, found.y * share};
    } else {
        const float ref = s_all[0][mine].x;
        float m = 0.f, squares = 0.f;
        for (int k = 0; k < CLUSTER; ++k) m += (float)rows_of(k) * (s_all[k][mine].x - ref);
        const float mean = ref + m / (float)p.rows_each;
        for (int k = 0; k < CLUSTER; ++k) {
            const float2 one = s_all[k][mine];
            squares += one.y + (float)rows_of(k) * (float)p.width * (one.x - mean) * (one.x - mean);
        }
        found = float2{mean, rsqrtf(squares * share + p.eps)};
        if (rank == 0 && p.mean && t.row_in == 0 && t.lane == 0) {
            p.mean[s * p.groups + t.group] = found.x;
            p.r[s * p.groups + t.group] = found.y;
        }
    }
    write_rows<T, E, STRIDED, GRAD, false>(p, t, ring, true, lo, lo + rows, w, b, GRAD ? at : found, found);
    if constexpr (GRAD) {
        if (p.channels) store_channels<T, E, STRIDED>(p, t, gw, gb, reinterpret_cast<float2*>(ring.team), blockIdx.x);
    }
}

// ---- groups that are wider than a block -----------------------------------------------------------
__device__ __forceinline__ double block_sum(double v) {
    __shared__ double part[THREADS / 32];
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(FULL, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    double s = 0.0;
#pragma unroll
    for (int i = 0; i < THREADS / 32; ++i) s += part[i];
    return s;
}

__device__ __forceinline__ float slope_by(float z, int act) {
    float s;
    with_activation(act, [&](auto a) { s = slope<decltype(a)::value>(z); });
    return s;
}

// A block to a sample's group, value by value.  A thread adds up to rows x width / 256 values: eight or 32 at a time and those in 64 bits, as in 32
// the sum of a long sample far from 0 is off by more than its spread (50 000 x 4 096 around 1 000: the mean by five spreads, the variance
// 27 times).
// SINGLE: samples of one row, of which many blocks are under way: in one plain loop (20 000 x 8 192 fp32 with SiLU 313 us, by rows of eight
// values abreast 443); longer samples eight abreast (one of 2 000 x 2 304 5.0 ms, in one loop over each row 6.9).
constexpr int ABREAST = 8;
template <class T, bool GRAD, bool SINGLE>
__global__ void __launch_bounds__(THREADS) wide_kernel(const Params p) {
    cbm::wait_before();
    for (int64_t unit = blockIdx.x; unit < p.n_samples * p.groups; unit += gridDim.x) {
        const int64_t s = unit / p.groups, first = start_of(p, s), last = max(start_of(p, s + 1), first), count = (last - first) * p.width;
        const int c0 = (int)(unit % p.groups) * p.width;
        const T *x = static_cast<const T*>(p.x), *gy = static_cast<const T*>(p.gy);
        const double share = 1.0 / (double)max(count, (int64_t)1);
        // f(row, channel, value, and where asked for the gradient's value, weight and bias) for all values, and what it gives added up
        auto each = [&](auto with_params, auto with_gy, auto&& f) {
            constexpr bool PARAMS = decltype(with_params)::value, PAIRS = decltype(with_gy)::value;
            double2 all{0.0, 0.0};
            if constexpr (SINGLE) {
                for (int c = threadIdx.x; c < p.width; c += 32 * THREADS) {
                    const int to = min(p.width, c + 32 * THREADS);
                    float2 some{0.f, 0.f};
#pragma unroll 8
                    for (int k = c; k < to; k += THREADS) {
                        const int channel = c0 + k;
                        const float2 one = f(first, channel, cbm::widen(x[first * p.ldx + channel]), PAIRS ? cbm::widen(gy[first * p.ldgy + channel]) : 0.f,
                                             PARAMS ? param<T>(p.w, p.wide_params, channel, 1.f) : 1.f, PARAMS ? param<T>(p.b, p.wide_params, channel, 0.f) : 0.f);
                        some.x += one.x, some.y += one.y;
                    }
                    all.x += some.x, all.y += some.y;
                }
            } else {
                for (int64_t row = first; row < last; ++row)
                    for (int c = threadIdx.x; c < p.width; c += ABREAST * THREADS) {
                        T v[ABREAST], g[PAIRS ? ABREAST : 1];
                        float w[PARAMS ? ABREAST : 1], b[PARAMS ? ABREAST : 1];
#pragma unroll
                        for (int k = 0; k < ABREAST; ++k) {  // (the last again in place of those that are not there: branches would wait for one another)
                            const int channel = c0 + min(c + k * THREADS, p.width - 1);
                            v[k] = x[row * p.ldx + channel];
                            if constexpr (PAIRS) g[k] = gy[row * p.ldgy + channel];
                            if constexpr (PARAMS) w[k] = param<T>(p.w, p.wide_params, channel, 1.f), b[k] = param<T>(p.b, p.wide_params, channel, 0.f);
                        }
                        float2 some{0.f, 0.f};
#pragma unroll
                        for (int k = 0; k < ABREAST; ++k)
                            if (c + k * THREADS < p.width) {
                                const float2 one = f(row, c0 + c + k * THREADS, cbm::widen(v[k]), PAIRS ? cbm::widen(g[PAIRS ? k : 0]) : 0.f, w[PARAMS ? k : 0], b[PARAMS ? k : 0]);
                                some.x += one.x, some.y += one.y;
                            }
                        all.x += some.x, all.y += some.y;
                    }
            }
            return all;
        };
        const auto yes = std::true_type();
        const auto no = std::false_type();
        const float mean = (float)(block_sum(each(no, no, [&](int64_t, int, float v, float, float, float) { return float2{v, 0.f}; }).x) * share);
        const double sum = each(no, no, [&](int64_t, int, float v, float, float, float) { return float2{(v - mean) * (v - mean), 0.f}; }).x;
        const float r = rsqrtf((float)(block_sum(sum) * share) + p.eps);
        if constexpr (!GRAD) {
            with_activation(p.act, [&](auto act) {
                each(yes, no, [&](int64_t row, int c, float v, float, float w, float b) {
                    static_cast<T*>(p.y)[row * p.ldy + c] = cbm::narrow<T>(activated<decltype(act)::value>((v - mean) * (r * w) + b));
                    return float2{0.f, 0.f};
                });
            });
            if (threadIdx.x == 0 && p.mean) p.mean[unit] = mean, p.r[unit] = r;
        } else {
            with_activation(p.act, [&](auto act) {
                auto u_of = [](float xh, float g, float w, float b) { return g * slope<decltype(act)::value>(xh * w + b) * w; };
                const double2 sums = each(yes, yes, [&](int64_t, int, float v, float g, float w, float b) {
                    const float xh = (v - mean) * r, u = u_of(xh, g, w, b);
                    return float2{u, u * xh};
                });
                const float su = (float)(block_sum(sums.x) * share), sux = (float)(block_sum(sums.y) * share);
                each(yes, yes, [&](int64_t row, int c, float v, float g, float w, float b) {
                    const float xh = (v - mean) * r;
                    static_cast<T*>(p.y)[row * p.ldy + c] = cbm::narrow<T>(r * (u_of(xh, g, w, b) - su - xh * sux));
                    return float2{0.f, 0.f};
                });
            });
            if (threadIdx.x == 0) p.joined[unit] = float2{mean, r};
        }
    }
}

// Sums over ranges of samples of g xh and g, a thread to a channel, in 64 bits like those above; behind wide_kernel, with its statistics.
template <class T>
__global__ void __launch_bounds__(THREADS) wide_params_kernel(const Params p) {
    cbm::wait_before();
    const int c = blockIdx.y * THREADS + threadIdx.x;
    if (c >= p.c) return;
    const float w = param<T>(p.w, p.wide_params, c, 1.f), b = param<T>(p.b, p.wide_params, c, 0.f);
    double all_x = 0.0, all = 0.0;
    const int64_t each = (p.n_samples + p.parts - 1) / p.parts, to = min((blockIdx.x + 1) * each, p.n_samples);
    for (int64_t s = blockIdx.x * each; s < to; ++s) {
        const float2 at = p.joined[s * p.groups + c / p.width];
        const int64_t last = start_of(p, s + 1);
        for (int64_t row = start_of(p, s); row < last; ++row) {
            const float xh = (cbm::widen(static_cast<const T*>(p.x)[row * p.ldx + c]) - at.x) * at.y;
            const float g = cbm::widen(static_cast<const T*>(p.gy)[row * p.ldgy + c]) * slope_by(xh * w + b, p.act);
            all_x += g * xh, all += g;
        }
    }
    p.channels[(int64_t)blockIdx.x * p.c + c] = float2{(float)all_x, (float)all};
}

// Rows of no sample: 0.
template <class T>
__global__ void __launch_bounds__(THREADS) outside_kernel(const Params p) {
    cbm::wait_before();
    const int64_t head = p.n_samples ? start_of(p, 0) : p.n_rows, tail = p.n_samples ? max(start_of(p, p.n_samples), head) : p.n_rows;
    const int64_t outside = head + p.n_rows - tail;
    for (int64_t i = blockIdx.x; i < outside; i += gridDim.x) {
        T* to = static_cast<T*>(p.y) + (i < head ? i : i - head + tail) * p.ldy;
        for (int c = threadIdx.x; c < p.c; c += THREADS) to[c] = cbm::narrow<T>(0.f);
    }
}

// ---- host -----------------------------------------------------------------------------------------
int launched(const char* who) {
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? CBM_B200_OK : cbm::fail(CBM_B200_ERR_CUDA, std::string(who) + ": " + cudaGetErrorString(e));
}

constexpr int MOST_CHANNELS = 1 << 22;  // (slabs of 128 groups, or of 256 threads, are counted in a grid's second dimension)

int check(const char* who, const Params& p, int32_t type) {
    const bool fits = p.n_rows >= 0 && p.n_rows < ((int64_t)1 << 40) && p.n_samples >= 0 && p.c >= 1 && p.c <= MOST_CHANNELS && p.groups >= 1 && p.c % p.groups == 0 &&
                      p.ldx >= p.c && p.ldy >= p.c && p.act >= 0 && p.act <= CBM_B200_ACT_SILU && type >= 0 && type <= CBM_B200_FP16 && p.eps >= 0.f &&
                      (p.ptr || (p.rows_each >= 0 && (p.n_samples == 0 ? p.n_rows == 0 : p.n_rows % p.n_samples == 0 && p.n_rows / p.n_samples == p.rows_each)));
    return fits ? CBM_B200_OK : cbm::fail(CBM_B200_ERR_ARG, std::string(who) + ": bad sizes, type or activation");
}

enum Way { ROWS, TILES, CLUSTERS, WIDE };

// The values of a row that fall to a thread: E of them, as one vector or (strided) as many threads of a group apart.
struct Form {
    int e;
    bool strided;
    int lanes(int width) const { return (width + e - 1) / e; }
};

// How a norm is computed, from its sizes and the form.
struct Plan {
    Way way;
    Form form;
    RowShape rows;
    int64_t blocks;    // with ROWS
    int lanes, team, slab_groups;
    int64_t tile, tiles, parts;
    bool joins;        // whether samples may be longer than a tile

    Plan(int64_t n_rows, int64_t n_samples, bool ptr, int64_t rows_each, int c, int groups, Form f, bool grad) : form(f) {
        const int width = c / groups;
        joins = false;
        tile = tiles = 0;
        if (!ptr && rows_each == 1 && form.lanes(width) <= 1024) {
            way = ROWS;
            lanes = form.lanes(width);
            rows.warps = lanes > 32 ? (lanes + 31) / 32 : 0;
            for (rows.shift = 0; rows.shift < 5 && 1 << rows.shift < lanes;) ++rows.shift;
            slab_groups = THREADS / rows.padded() < 1 ? 1 : THREADS / rows.padded() < groups ? THREADS / rows.padded() : groups;
            rows.slots = slab_groups * rows.padded();
            rows.at_once = rows.slots >= THREADS ? 1 : THREADS / rows.slots;
            const int64_t turns = (n_rows + rows.at_once - 1) / rows.at_once;
            const int64_t most = (int64_t)SMS * (2048 / threads()) / 2;  // (half of what an SM holds: their registers)
            blocks = turns < most ? turns : most;
            parts = blocks;
            return;
        }
        if (form.lanes(width) > THREADS) form = Form{8, true};
        lanes = form.lanes(width);
        if (lanes > THREADS) {
            way = WIDE;
            parts = n_samples < SMS ? (n_samples > 0 ? n_samples : 1) : SMS;
            return;
        }
        way = TILES;
        slab_groups = THREADS / lanes < GROUPS ? THREADS / lanes : GROUPS;
        if (groups < slab_groups) slab_groups = groups;
        // A few samples whose rows a cluster goes over in some dozen turns, with tiles, joins and rows by themselves above (x 64 fp32, turns of
        // 128 rows, out of DRAM): one of 1 000 rows 10 us, by tiles 16, with the gradient 21 and 29; one of 3 000 14 and 18, 33 both; 16 of 6 000 26
        // and 41, 62 and 72, but one of 6 000 20 and 18, 49 and 33; past the limit 16 of 12 000 47 and 51, 117 and 102, one 33 and 23, 82 and 39.
        const int64_t slabs = (groups + slab_groups - 1) / slab_groups, turn = (int64_t)CLUSTER * (THREADS / (slab_groups * lanes));
        if (!ptr && rows_each > 1 && n_samples * CLUSTER * slabs <= 2 * SMS && rows_each <= 48 * turn) {
            way = CLUSTERS;
            team = THREADS;
            parts = n_samples * CLUSTER;
            return;
        }
        // Four rows at once, or where samples are short one, so that more of them are under way (262 147 x 100 bf16 with SiLU, samples of 30 rows:
        // one at once 66 us, four 129; of 60 61 and 94; of 100 71 and 78, with the gradient 197 and 180; of 200 78 and 62, 184 and 150).
        const int wanted = (n_samples && n_rows / n_samples > 64 ? 4 : 1) * slab_groups * lanes;
        for (team = 32; team < THREADS && team < wanted;) team *= 2;
        const int at_once = team / (slab_groups * lanes);
        int64_t teams = (int64_t)SMS * blocks_resident(form.e, grad) * (THREADS / team) / slabs;  // resident at the same time
        if (teams < 1) teams = 1;
        tile = (n_rows + teams - 1) / teams;
        // At least two turns, or where samples are shorter than a turn as much as two of them (54 718 x 5 fp32, samples of 9 rows, with the
        // gradient: eight turns 209 us, eight samples 158, two 111; 4 000 x 32 in samples of 23: 61 -> 52).
        const int64_t mean = n_samples ? n_rows / n_samples + 1 : n_rows + 1, least = 2 * (mean < at_once ? mean : at_once);
        if (tile < least) tile = least;
        tiles = (n_rows + tile - 1) / tile;
        parts = tiles;
        joins = ptr || rows_each > tile;
    }
    int threads() const { return (rows.slots * rows.at_once + 31) / 32 * 32; }
    int64_t piece_bytes(int groups) const { return way == TILES && joins ? 8 * (3 * tiles * groups + 2 * tiles) : 0; }
    int64_t bytes(int64_t n_samples, int c, int groups, bool grad) const {
        return (grad ? 8 * parts * c : 0) + piece_bytes(groups) + (way == WIDE && grad ? 8 * n_samples * groups : 0);
    }
};

// Vectors of the largest power of two of values, up to 16 bytes, that divides a group's channels and at which all rows are aligned;
// where that is one value, four strided ones (narrow groups: one).
Form form_of(const Params& p, int size) {
    int e = 16 / size;
    auto aligned = [&](const void* q, int64_t ld) { return reinterpret_cast<uintptr_t>(q) % (e * size) == 0 && ld % e == 0; };
    while (e > 1 && (p.width % e || !aligned(p.x, p.ldx) || !aligned(p.y, p.ldy) || (p.gy && !aligned(p.gy, p.ldgy)))) e /= 2;
    return e > 1 ? Form{e, false} : Form{p.width > 2 ? 4 : 1, true};
}

// Calls f with the number of values and whether they are strided as constants.
template <class T, class F>
void with_form(Form form, F&& f) {
    using Y = std::true_type;
    using N = std::false_type;
    if (form.strided) {
        if (form.e == 1) f(std::integral_constant<int, 1>(), Y());
        else if (form.e == 4) f(std::integral_constant<int, 4>(), Y());
        else f(std::integral_constant<int, 8>(), Y());
    } else {
        if (form.e == 2) f(std::integral_constant<int, 2>(), N());
        else if (form.e == 4) f(std::integral_constant<int, 4>(), N());
        else if constexpr (sizeof(T) == 2) f(std::integral_constant<int, 8>(), N());
    }
}

dim3 blocks_for(int64_t units) { return dim3((unsigned)(units < SMS * 32 ? (units > 0 ? units : 1) : SMS * 32)); }

template <class T, bool GRAD>
void launch(Params& p, const Plan& plan, unsigned char* workspace, const cbm::Stream& on) {
    const bool sums = GRAD && (p.gw || p.gb);
    p.parts = p.n_rows ? plan.parts : 0;
    if (sums) p.channels = reinterpret_cast<float2*>(workspace);
    workspace += GRAD ? 8 * plan.parts * p.c : 0;
    p.lanes = plan.lanes, p.slab_groups = plan.slab_groups, p.team = plan.team, p.tile = plan.tile, p.tiles = plan.tiles;
    int64_t joins = 0;
    if (p.n_rows == 0) {
        // nothing but the sums of nothing
    } else if (plan.way == ROWS) {
        with_form<T>(plan.form, [&](auto e, auto strided) {
            const unsigned threads = plan.threads();
            const dim3 grid((unsigned)plan.blocks, (p.groups + p.slab_groups - 1) / p.slab_groups);
            cbm::launch_next(rows_kernel<T, decltype(e)::value, decltype(strided)::value, GRAD>, grid, threads, sums ? 8 * threads : 0, on, p, plan.rows);
        });
    } else if (plan.way == CLUSTERS) {
        with_form<T>(plan.form, [&](auto e, auto strided) {
            cudaLaunchAttribute attrs[2] = {};
            attrs[0].id = cudaLaunchAttributeClusterDimension;
            attrs[0].val.clusterDim.x = CLUSTER;
            attrs[0].val.clusterDim.y = attrs[0].val.clusterDim.z = 1;
            attrs[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
            attrs[1].val.programmaticStreamSerializationAllowed = 1;
            cudaLaunchConfig_t config = {};
            config.gridDim = dim3((unsigned)plan.parts, (p.groups + p.slab_groups - 1) / p.slab_groups);
            config.blockDim = dim3(THREADS);
            config.stream = on.s;
            config.attrs = attrs;
            config.numAttrs = on.captured ? 1 : 2;
            (void)cudaLaunchKernelEx(&config, cluster_kernel<T, decltype(e)::value, decltype(strided)::value, GRAD>, static_cast<Params>(p));
        });
    } else if (plan.way == TILES) {
        p.pieces = reinterpret_cast<float2*>(workspace);
        p.joined = p.pieces + 2 * p.tiles * p.groups;
        if (plan.joins) p.longer = reinterpret_cast<int64_t*>(p.joined + p.tiles * p.groups);
        const int per_block = THREADS / p.team;
        const dim3 grid((unsigned)((p.tiles + per_block - 1) / per_block), (p.groups + p.slab_groups - 1) / p.slab_groups);
        with_form<T>(plan.form, [&](auto e, auto strided) {
            constexpr int E = decltype(e)::value;
            constexpr bool STRIDED = decltype(strided)::value;
            cbm::launch_next(tiles_kernel<T, E, STRIDED, GRAD>, grid, THREADS, 0, on, p);
            if (!plan.joins) return;
            joins = p.ptr ? p.tiles : p.n_samples;
            const int most = p.ptr ? 4 : 65535, across = p.groups < most ? p.groups : most;  // (most blocks of tiles find nothing to do)
            cbm::launch_next(join_kernel<T, GRAD>, dim3((unsigned)((joins + JOINED - 1) / JOINED + (sums ? (p.c + CHANNELS - 1) / CHANNELS : 0)), across), JOINERS, 0, on, p, joins);
            cbm::launch_next(long_kernel<T, E, STRIDED, GRAD>, grid, THREADS, 0, on, p);
        });
    } else {
        p.joined = reinterpret_cast<float2*>(workspace);
        if (p.n_samples) cbm::launch_next(!p.ptr && p.rows_each == 1 ? wide_kernel<T, GRAD, true> : wide_kernel<T, GRAD, false>, blocks_for(p.n_samples * p.groups), THREADS, 0, on, p);
        if (p.ptr) cbm::launch_next(outside_kernel<T>, blocks_for(p.n_rows), THREADS, 0, on, p);
        if (sums) cbm::launch_next(wide_params_kernel<T>, dim3((unsigned)p.parts, (p.c + THREADS - 1) / THREADS), THREADS, 0, on, p);
    }
    if (sums && !joins) cbm::launch_next(join_kernel<T, true>, dim3((p.c + CHANNELS - 1) / CHANNELS), JOINERS, 0, on, p, joins);
}

// Workspace of a call, whatever the type and the alignment of its rows.
int64_t workspace_of(int64_t n_rows, int64_t n_samples, bool ptr, int64_t rows_each, int c, int groups, bool grad) {
    static const Form forms[] = {{1, true}, {4, true}, {2, false}, {4, false}, {8, false}};
    int64_t most = 0;
    for (const Form f : forms) {
        if (!f.strided && c / groups % f.e) continue;
        const int64_t bytes = Plan(n_rows, n_samples, ptr, rows_each, c, groups, f, grad).bytes(n_samples, c, groups, grad);
        most = bytes > most ? bytes : most;
    }
    return most;
}

}  // namespace

extern "C" int64_t cbm_b200_group_norm_workspace(int64_t n_rows, int64_t n_samples, int32_t channels, int32_t groups, int32_t gradient) {
    const bool ptr = n_samples >= 0;
    const int64_t samples = ptr ? n_samples : -n_samples;
    if (n_rows < 0 || channels < 1 || groups < 1 || channels % groups) return 0;
    return workspace_of(n_rows, samples, ptr, ptr || samples == 0 ? 0 : n_rows / samples, channels, groups, gradient != 0);
}

extern "C" int cbm_b200_group_norm(const void* x, int64_t ldx, int32_t type, int64_t n_rows, int32_t channels, int32_t groups,
                                   const int64_t* ptr, int64_t n_samples, int64_t rows_each, const void* weight, const void* bias,
                                   int32_t wide_params, float eps, int32_t activation, void* y, int64_t ldy, float* mean, float* rstd,
                                   void* workspace, int64_t workspace_bytes, void* stream) {
    Params p{};
    p.x = x, p.w = weight, p.b = bias, p.ldx = ldx, p.ldy = ldy, p.n_rows = n_rows, p.n_samples = n_samples, p.rows_each = rows_each;
    p.ptr = ptr, p.c = channels, p.groups = groups, p.width = groups > 0 ? channels / groups : 0, p.act = activation;
    p.wide_params = wide_params, p.eps = eps, p.y = y, p.mean = mean, p.r = rstd;
    if (int rc = check("group_norm", p, type)) return rc;
    if (n_rows == 0) return CBM_B200_OK;
    if (!x || !y || !mean != !rstd) return cbm::fail(CBM_B200_ERR_ARG, "group_norm: NULL argument");
    const Plan plan(n_rows, n_samples, ptr != nullptr, rows_each, channels, groups, form_of(p, cbm::size_of_type(type)), false);
    const int64_t need = plan.bytes(n_samples, channels, groups, false);
    if (need && (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 8))
        return cbm::fail(CBM_B200_ERR_ARG, "group_norm: workspace too small, or not at 8 bytes");
    const cbm::Stream on(static_cast<cudaStream_t>(stream));
    cbm::with_type(type, [&](auto t) { launch<decltype(t), false>(p, plan, static_cast<unsigned char*>(workspace), on); });
    return launched("group_norm");
}

extern "C" int cbm_b200_group_norm_grad(const void* x, int64_t ldx, const void* gy, int64_t ldgy, int32_t type, int64_t n_rows,
                                        int32_t channels, int32_t groups, const int64_t* ptr, int64_t n_samples, int64_t rows_each,
                                        const void* weight, const void* bias, int32_t wide_params, float eps, int32_t activation,
                                        float* mean, float* rstd, void* gx, int64_t ldgx, float* gw, float* gb, void* workspace,
                                        int64_t workspace_bytes, void* stream) {
    Params p{};
    p.x = x, p.gy = gy, p.w = weight, p.b = bias, p.ldx = ldx, p.ldgy = ldgy, p.ldy = ldgx, p.n_rows = n_rows, p.n_samples = n_samples;
    p.rows_each = rows_each, p.ptr = ptr, p.c = channels, p.groups = groups, p.width = groups > 0 ? channels / groups : 0, p.act = activation;
    p.wide_params = wide_params, p.eps = eps, p.y = gx, p.mean = mean, p.r = rstd, p.gw = gw, p.gb = gb;
    if (int rc = check("group_norm_grad", p, type)) return rc;
    if (ldgy < channels) return cbm::fail(CBM_B200_ERR_ARG, "group_norm_grad: rows of the gradient overlap");
    if (n_rows && (!x || !gy || !gx)) return cbm::fail(CBM_B200_ERR_ARG, "group_norm_grad: NULL argument");
    const Plan plan(n_rows, n_samples, ptr != nullptr, rows_each, channels, groups, form_of(p, cbm::size_of_type(type)), true);
    if (n_rows && n_samples && (plan.way == TILES || plan.way == CLUSTERS) && (!mean || !rstd)) return cbm::fail(CBM_B200_ERR_ARG, "group_norm_grad: NULL argument");
    const int64_t need = plan.bytes(n_samples, channels, groups, true);
    if (need && (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 8))
        return cbm::fail(CBM_B200_ERR_ARG, "group_norm_grad: workspace too small, or not at 8 bytes");
    const cbm::Stream on(static_cast<cudaStream_t>(stream));
    cbm::with_type(type, [&](auto t) { launch<decltype(t), true>(p, plan, static_cast<unsigned char*>(workspace), on); });
    return launched("group_norm_grad");
}
