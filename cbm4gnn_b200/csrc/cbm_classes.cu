// Class log probabilities of rows of logits, with entropy and the most probable classes, and the gradient (sm_100a).
//
// With m the largest of a row, s the sum of exp(x - m) over the others and t = sum exp(x - m) (m - x):
//   log p_j = (x_j - m) - log1p(s),   entropy = log1p(s) + t / (1 + s).
// Nothing in these is subtracted that is nearly equal, so a decided row keeps the digits of a log probability near 0.
// Gradient: dx_j = g_log ([j = label] - p_j) - g_ent p_j (log p_j + entropy) + sum_i g_top_i ([j = c_i] - p_j).
#include "cbm_common.h"
#include "cbm_launch.cuh"
#include "cbm_values.cuh"

#include <cmath>
#include <string>

namespace {

using u32 = uint32_t;
using u64 = unsigned long long;

constexpr int WARPS = 8;
constexpr u32 FULL = 0xffffffffu;

// Whole numbers in the order of the values: NaN above all, the two zeros equal.
__device__ __forceinline__ u32 ordered(float x) {
    if (x != x) return 0xffffffffu;
    const u32 b = __float_as_uint(x + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ u64 key_of(float x, u32 j) { return (u64)ordered(x) << 32 | (u32)~j; }

__device__ __forceinline__ u64 warp_max(u64 v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        const u64 w = __shfl_xor_sync(FULL, v, o);
        v = w > v ? w : v;
    }
    return v;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(FULL, v, o);
    return v;
}

struct ForwardParams {
    const void* x;
    const void* labels;
    int64_t ld, n;
    int c, top, wide_labels;
    float *log_prob, *entropy, *stats, *top_log_prob;
    int64_t* top_class;
};

__device__ __forceinline__ int64_t label_of(const void* labels, int wide, int64_t row) {
    return wide ? static_cast<const int64_t*>(labels)[row] : (int64_t) static_cast<const int32_t*>(labels)[row];
}

template <class T>
__global__ void __launch_bounds__(WARPS * 32) classes_kernel(const ForwardParams p) {
    cbm::wait_before();
    const int lane = threadIdx.x & 31;
    for (int64_t row = (int64_t)blockIdx.x * WARPS + (threadIdx.x >> 5); row < p.n; row += (int64_t)gridDim.x * WARPS) {
        const T* x = static_cast<const T*>(p.x) + row * p.ld;
        u64 best = 0;
        for (int j = lane; j < p.c; j += 32) {
            const u64 k = key_of(cbm::widen(x[j]), j);
            best = k > best ? k : best;
        }
        best = warp_max(best);
        const u32 first = ~(u32)best;
        const float m = cbm::widen(x[first]);
        const bool closed = m == -INFINITY;  // no class is open
        float s = 0.f, t = 0.f;
        for (int j = lane; j < p.c; j += 32) {
            const float d = cbm::widen(x[j]) - m, e = expf(d);
            if (j != first && !closed) {
                s += e;
                t -= e > 0.f ? e * d : 0.f;
            } else if (!closed) {
                s += d;  // 0, or NaN for an infinite or undefined row
            }
        }
        s = warp_sum(s), t = warp_sum(t);
        const float ls = closed ? 0.f : log1pf(s);
        if (lane == 0) {
            const int64_t label = label_of(p.labels, p.wide_labels, row);
            p.log_prob[row] = label < 0 ? 0.f : label >= p.c ? NAN : closed ? -INFINITY : (cbm::widen(x[label]) - m) - ls;
            p.entropy[row] = ls + t / (1.f + s);
            p.stats[2 * row] = m;
            p.stats[2 * row + 1] = ls;
        }
        u64 last = best;
        for (int i = 0; i < p.top; ++i) {
            if (i) {
                u64 next = 0;
                for (int j = lane; j < p.c; j += 32) {
                    const u64 k = key_of(cbm::widen(x[j]), j);
                    next = k < last && k > next ? k : next;
                }
                last = warp_max(next);
            }
            if (lane == 0) {
                const u32 j = ~(u32)last;
                p.top_class[row * p.top + i] = j;
                p.top_log_prob[row * p.top + i] = closed ? -INFINITY : (cbm::widen(x[j]) - m) - ls;
            }
        }
    }
}

struct BackwardParams {
    const void* x;
    const void* labels;
    int64_t ld, ld_out, n;
    int c, top, wide_labels;
    const float *stats, *entropy, *g_log, *g_entropy, *g_top;
    const int64_t* top_class;
    void* dx;
};

template <class T>
__global__ void __launch_bounds__(WARPS * 32) classes_grad_kernel(const BackwardParams p) {
    cbm::wait_before();
    const int lane = threadIdx.x & 31;
    for (int64_t row = (int64_t)blockIdx.x * WARPS + (threadIdx.x >> 5); row < p.n; row += (int64_t)gridDim.x * WARPS) {
        const T* x = static_cast<const T*>(p.x) + row * p.ld;
        T* dx = static_cast<T*>(p.dx) + row * p.ld_out;
        const int64_t label = label_of(p.labels, p.wide_labels, row);
        const float m = p.stats[2 * row], ls = p.stats[2 * row + 1];
        const bool closed = m == -INFINITY;
        const float gl = !p.g_log || label < 0 ? 0.f : label >= p.c ? NAN : p.g_log[row];
        const float ge = p.g_entropy ? p.g_entropy[row] : 0.f;
        const float gt = p.g_top && lane < p.top ? p.g_top[row * p.top + lane] : 0.f;
        const float all = gl + warp_sum(gt) + ge * p.entropy[row];
        auto base = [&](int j) {
            const float lp = (cbm::widen(x[j]) - m) - ls, q = expf(lp);
            return closed ? 0.f : -q * (all + (q > 0.f ? ge * lp : 0.f));
        };
        for (int j = lane; j < p.c; j += 32) dx[j] = cbm::narrow<T>(base(j));
        __syncwarp();
        // what falls to single classes: the label's and those of the list, of which one may be the label
        const int64_t mine = p.g_top && lane < p.top ? p.top_class[row * p.top + lane] : -1;
        const bool listed = __any_sync(FULL, mine >= 0 && mine == label);
        if (mine >= 0) dx[mine] = cbm::narrow<T>(closed ? 0.f : base((int)mine) + gt + (mine == label ? gl : 0.f));
        if (lane == 0 && !listed && label >= 0 && label < p.c) dx[label] = cbm::narrow<T>(closed ? 0.f : base((int)label) + gl);
        __syncwarp();
    }
}

int check(const char* who, int64_t n, int64_t ld, int32_t c, int32_t top, int32_t type) {
    if (n < 0 || c < 1 || ld < c || top < 0 || top > CBM_B200_MAX_TOP || top > c || type < 0 || type > CBM_B200_FP16)
        return cbm::fail(CBM_B200_ERR_ARG, std::string(who) + ": bad sizes or type");
    return CBM_B200_OK;
}

int launched(const char* who) {
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? CBM_B200_OK : cbm::fail(CBM_B200_ERR_CUDA, std::string(who) + ": " + cudaGetErrorString(e));
}

unsigned blocks_for(int64_t n) {
    const int64_t b = (n + WARPS - 1) / WARPS;
    return (unsigned)(b < 148 * 64 ? b : 148 * 64);
}

}  // namespace

extern "C" int cbm_b200_class_log_probs(const void* logits, int64_t ld, int32_t type, const void* labels, int32_t wide_labels,
                                        int64_t n_rows, int32_t n_classes, int32_t top, float* log_prob, float* entropy, float* stats,
                                        float* top_log_prob, int64_t* top_class, void* stream) {
    if (int rc = check("class_log_probs", n_rows, ld, n_classes, top, type)) return rc;
    if (n_rows == 0) return CBM_B200_OK;
    if (!logits || !labels || !log_prob || !entropy || !stats || (top && (!top_log_prob || !top_class)))
        return cbm::fail(CBM_B200_ERR_ARG, "class_log_probs: NULL argument");
    const ForwardParams p{logits, labels, ld, n_rows, n_classes, top, wide_labels, log_prob, entropy, stats, top_log_prob, top_class};
    const cbm::Stream on(static_cast<cudaStream_t>(stream));
    cbm::with_type(type, [&](auto t) { cbm::launch_next(classes_kernel<decltype(t)>, dim3(blocks_for(n_rows)), WARPS * 32, 0, on, p); });
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
    const BackwardParams p{logits, labels, ld, lddx, n_rows, n_classes, top, wide_labels, stats, entropy, g_log_prob, g_entropy, g_top, top_class, dx};
    const cbm::Stream on(static_cast<cudaStream_t>(stream));
    cbm::with_type(type, [&](auto t) { cbm::launch_next(classes_grad_kernel<decltype(t)>, dim3(blocks_for(n_rows)), WARPS * 32, 0, on, p); });
    return launched("class_log_probs_grad");
}
