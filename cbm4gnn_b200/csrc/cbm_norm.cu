// Group norm with an activation over channels-last rows, and its gradients (sm_100a).
//
// A sample is a range of rows (a graph), a group a range of channels.  With mean and r = 1 / sqrt(var + eps) over the values of
// a sample's group:  xh = (x - mean) r,  z = w xh + b,  y = act(z).
// Gradients, with g = gy act'(z) and u = w g:  gb = sum g,  gw = sum g xh,  gx = r (u - mean(u) - xh mean(u xh)).
#include "cbm_common.h"
#include "cbm_launch.cuh"
#include "cbm_values.cuh"

#include <string>

namespace {

using u32 = uint32_t;

constexpr int THREADS = 256;

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
};

// Rows [first, last) of a sample; what a pointer array says is kept inside the rows there are.
__device__ __forceinline__ void rows_of(const Params& p, int64_t s, int64_t& first, int64_t& last) {
    if (p.ptr) {
        first = min(max(p.ptr[s], (int64_t)0), p.n_rows);
        last = min(max(p.ptr[s + 1], first), p.n_rows);
    } else {
        first = s * p.rows_each;
        last = first + p.rows_each;
    }
}

template <class T>
__device__ __forceinline__ float param(const void* w, int wide, int c, float none) {
    return !w ? none : wide ? static_cast<const float*>(w)[c] : cbm::widen(static_cast<const T*>(w)[c]);
}

__device__ __forceinline__ float sigmoid(float z) { return 1.f / (1.f + expf(-z)); }
__device__ __forceinline__ float activated(float z, int act) {
    if (act == CBM_B200_ACT_RELU) return z <= 0.f ? 0.f : z;  // NaN passes
    return act == CBM_B200_ACT_SILU ? z * sigmoid(z) : z;
}
__device__ __forceinline__ float slope(float z, int act) {
    if (act == CBM_B200_ACT_RELU) return z <= 0.f ? 0.f : 1.f;
    if (act != CBM_B200_ACT_SILU) return 1.f;
    const float s = sigmoid(z);
    return s * (1.f + z * (1.f - s));
}

__device__ __forceinline__ float block_sum(float v) {
    __shared__ float part[THREADS / 32];
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < THREADS / 32; ++i) s += part[i];
    return s;
}

// A block to a sample's group.
template <class T>
__global__ void __launch_bounds__(THREADS) norm_kernel(const Params p) {
    cbm::wait_before();
    for (int64_t unit = blockIdx.x; unit < p.n_samples * p.groups; unit += gridDim.x) {
        int64_t first, last;
        rows_of(p, unit / p.groups, first, last);
        const int c0 = (int)(unit % p.groups) * p.width;
        const int64_t count = (last - first) * p.width;
        const T* x = static_cast<const T*>(p.x);
        float s = 0.f;
        for (int64_t i = threadIdx.x; i < count; i += THREADS) s += cbm::widen(x[(first + i / p.width) * p.ldx + c0 + i % p.width]);
        const float mean = block_sum(s) / (float)max(count, (int64_t)1);
        s = 0.f;
        for (int64_t i = threadIdx.x; i < count; i += THREADS) {
            const float d = cbm::widen(x[(first + i / p.width) * p.ldx + c0 + i % p.width]) - mean;
            s += d * d;
        }
        const float r = rsqrtf(block_sum(s) / (float)max(count, (int64_t)1) + p.eps);
        for (int64_t i = threadIdx.x; i < count; i += THREADS) {
            const int64_t row = first + i / p.width;
            const int c = c0 + (int)(i % p.width);
            const float z = (cbm::widen(x[row * p.ldx + c]) - mean) * r * param<T>(p.w, p.wide_params, c, 1.f) + param<T>(p.b, p.wide_params, c, 0.f);
            static_cast<T*>(p.y)[row * p.ldy + c] = cbm::narrow<T>(activated(z, p.act));
        }
        if (threadIdx.x == 0 && p.mean) {
            p.mean[unit] = mean;
            p.r[unit] = r;
        }
    }
}

template <class T>
__global__ void __launch_bounds__(THREADS) norm_grad_kernel(const Params p) {
    cbm::wait_before();
    for (int64_t unit = blockIdx.x; unit < p.n_samples * p.groups; unit += gridDim.x) {
        int64_t first, last;
        rows_of(p, unit / p.groups, first, last);
        const int c0 = (int)(unit % p.groups) * p.width;
        const int64_t count = (last - first) * p.width;
        const float mean = p.mean[unit], r = p.r[unit];
        const T *x = static_cast<const T*>(p.x), *gy = static_cast<const T*>(p.gy);
        float su = 0.f, sux = 0.f;
        for (int step = 0; step < 2; ++step) {
            for (int64_t i = threadIdx.x; i < count; i += THREADS) {
                const int64_t row = first + i / p.width;
                const int c = c0 + (int)(i % p.width);
                const float w = param<T>(p.w, p.wide_params, c, 1.f), xh = (cbm::widen(x[row * p.ldx + c]) - mean) * r;
                const float u = cbm::widen(gy[row * p.ldgy + c]) * slope(xh * w + param<T>(p.b, p.wide_params, c, 0.f), p.act) * w;
                if (step == 0) su += u, sux += u * xh;
                else static_cast<T*>(p.y)[row * p.ldy + c] = cbm::narrow<T>(r * (u - su - xh * sux));
            }
            if (step == 0) {
                su = block_sum(su) / (float)max(count, (int64_t)1);
                sux = block_sum(sux) / (float)max(count, (int64_t)1);
            }
        }
    }
}

// A block to a channel: the gradients of its weight and bias, over all samples.
template <class T>
__global__ void __launch_bounds__(THREADS) norm_params_kernel(const Params p) {
    cbm::wait_before();
    const int c = blockIdx.x, group = c / p.width;
    const float w = param<T>(p.w, p.wide_params, c, 1.f), b = param<T>(p.b, p.wide_params, c, 0.f);
    float gw = 0.f, gb = 0.f;
    for (int64_t s = 0; s < p.n_samples; ++s) {
        int64_t first, last;
        rows_of(p, s, first, last);
        const float mean = p.mean[s * p.groups + group], r = p.r[s * p.groups + group];
        for (int64_t row = first + threadIdx.x; row < last; row += THREADS) {
            const float xh = (cbm::widen(static_cast<const T*>(p.x)[row * p.ldx + c]) - mean) * r;
            const float g = cbm::widen(static_cast<const T*>(p.gy)[row * p.ldgy + c]) * slope(xh * w + b, p.act);
            gw += g * xh;
            gb += g;
        }
    }
    gw = block_sum(gw);
    gb = block_sum(gb);
    if (threadIdx.x == 0) {
        if (p.gw) p.gw[c] = gw;
        if (p.gb) p.gb[c] = gb;
    }
}

// Rows of no sample: 0.
template <class T>
__global__ void __launch_bounds__(THREADS) norm_outside_kernel(const Params p) {
    cbm::wait_before();
    const int64_t head = p.n_samples ? min(max(p.ptr[0], (int64_t)0), p.n_rows) : p.n_rows;
    const int64_t tail = p.n_samples ? min(max(p.ptr[p.n_samples], head), p.n_rows) : p.n_rows;
    const int64_t outside = head + p.n_rows - tail;
    for (int64_t i = blockIdx.x; i < outside; i += gridDim.x) {
        T* to = static_cast<T*>(p.y) + (i < head ? i : i - head + tail) * p.ldy;
        for (int c = threadIdx.x; c < p.c; c += THREADS) to[c] = cbm::narrow<T>(0.f);
    }
}

int check(const char* who, const Params& p, int32_t type) {
    const bool fits = p.n_rows >= 0 && p.n_samples >= 0 && p.c >= 1 && p.groups >= 1 && p.c % p.groups == 0 && p.ldx >= p.c && p.ldy >= p.c &&
                      p.act >= 0 && p.act <= CBM_B200_ACT_SILU && type >= 0 && type <= CBM_B200_FP16 && p.eps >= 0.f &&
                      (p.ptr || (p.rows_each >= 0 && (p.n_samples == 0 ? p.n_rows == 0 : p.n_rows % p.n_samples == 0 && p.n_rows / p.n_samples == p.rows_each)));
    return fits ? CBM_B200_OK : cbm::fail(CBM_B200_ERR_ARG, std::string(who) + ": bad sizes, type or activation");
}

int launched(const char* who) {
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? CBM_B200_OK : cbm::fail(CBM_B200_ERR_CUDA, std::string(who) + ": " + cudaGetErrorString(e));
}

dim3 blocks_for(int64_t units) { return dim3((unsigned)(units < 148 * 32 ? units : 148 * 32)); }

}  // namespace

extern "C" int64_t cbm_b200_group_norm_workspace(int64_t, int64_t, int32_t, int32_t, int32_t) { return 0; }

extern "C" int cbm_b200_group_norm(const void* x, int64_t ldx, int32_t type, int64_t n_rows, int32_t channels, int32_t groups,
                                   const int64_t* ptr, int64_t n_samples, int64_t rows_each, const void* weight, const void* bias,
                                   int32_t wide_params, float eps, int32_t activation, void* y, int64_t ldy, float* mean, float* rstd,
                                   void*, int64_t, void* stream) {
    Params p{x, nullptr, weight, bias, ldx, 0, ldy, n_rows, n_samples, rows_each, ptr, channels, groups, groups > 0 ? channels / groups : 0,
             activation, wide_params, eps, y, mean, rstd, nullptr, nullptr};
    if (int rc = check("group_norm", p, type)) return rc;
    if (n_rows == 0) return CBM_B200_OK;
    if (!x || !y || !mean != !rstd) return cbm::fail(CBM_B200_ERR_ARG, "group_norm: NULL argument");
    const cbm::Stream on(static_cast<cudaStream_t>(stream));
    cbm::with_type(type, [&](auto t) {
        using T = decltype(t);
        if (n_samples) cbm::launch_next(norm_kernel<T>, blocks_for(n_samples * groups), THREADS, 0, on, p);
        if (ptr) cbm::launch_next(norm_outside_kernel<T>, blocks_for(n_rows), THREADS, 0, on, p);
    });
    return launched("group_norm");
}

extern "C" int cbm_b200_group_norm_grad(const void* x, int64_t ldx, const void* gy, int64_t ldgy, int32_t type, int64_t n_rows,
                                        int32_t channels, int32_t groups, const int64_t* ptr, int64_t n_samples, int64_t rows_each,
                                        const void* weight, const void* bias, int32_t wide_params, int32_t activation, float* mean,
                                        float* rstd, void* gx, int64_t ldgx, float* gw, float* gb, void*, int64_t, void* stream) {
    Params p{x, gy, weight, bias, ldx, ldgy, ldgx, n_rows, n_samples, rows_each, ptr, channels, groups, groups > 0 ? channels / groups : 0,
             activation, wide_params, 0.f, gx, mean, rstd, gw, gb};
    if (int rc = check("group_norm_grad", p, type)) return rc;
    if (ldgy < channels) return cbm::fail(CBM_B200_ERR_ARG, "group_norm_grad: rows of the gradient overlap");
    if ((n_samples && (!mean || !rstd)) || (n_rows && (!x || !gy || !gx))) return cbm::fail(CBM_B200_ERR_ARG, "group_norm_grad: NULL argument");
    const cbm::Stream on(static_cast<cudaStream_t>(stream));
    cbm::with_type(type, [&](auto t) {
        using T = decltype(t);
        if (n_samples && n_rows) cbm::launch_next(norm_grad_kernel<T>, blocks_for(n_samples * groups), THREADS, 0, on, p);
        if (ptr && n_rows) cbm::launch_next(norm_outside_kernel<T>, blocks_for(n_rows), THREADS, 0, on, p);
        if (gw || gb) cbm::launch_next(norm_params_kernel<T>, dim3(channels), THREADS, 0, on, p);
    });
    return launched("group_norm_grad");
}
