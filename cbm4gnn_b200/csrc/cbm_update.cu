// Orthogonalised updates by Newton-Schulz products (sm_100a).
//
// X = U / (|U| + eps), turned so that it is no taller than wide; then, `steps` times,
//   A = X X^T,  B = b A + c A A,  X <- a X + B X
// with the quintic (a, b, c) that the Muon optimiser publishes: every singular value is led to between 0.68 and 1.21.
#include "cbm_common.h"
#include "cbm_launch.cuh"

#include "cbm_b200.h"

#include <cmath>
#include <string>

namespace {

constexpr float QUINTIC_A = 3.4445f, QUINTIC_B = -4.7750f, QUINTIC_C = 2.0315f;
constexpr int THREADS = 256;

struct Matrix {
    const float* g;  // update, or gradient
    float *m, *w;    // momentum and weights, or NULL
    float* out;      // result, where there are no weights
    int64_t ldg, ldm, ldw, ldout;
    int rows, cols;
    float lr, momentum, nesterov, keep;
};

__device__ __forceinline__ float update_at(const Matrix& p, int64_t i, int64_t j) {
    const float g = p.g[i * p.ldg + j];
    if (!p.m) return g;
    const float m = p.m[i * p.ldm + j];  // already this step's
    return p.nesterov != 0.f ? g + p.momentum * m : m;
}

// This step's momentum, and the norm of the update in 64 bits.
__global__ void __launch_bounds__(1024) norm_of_update(const Matrix p, float eps, float* scale) {
    cbm::wait_before();
    double s = 0.0;
    const int64_t count = (int64_t)p.rows * p.cols;
    for (int64_t e = threadIdx.x; e < count; e += blockDim.x) {
        const int64_t i = e / p.cols, j = e % p.cols;
        if (p.m) p.m[i * p.ldm + j] = p.momentum * p.m[i * p.ldm + j] + p.g[i * p.ldg + j];
        const double u = update_at(p, i, j);
        s += u * u;
    }
    __shared__ double part[32];
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        s = 0.0;
        for (int i = 0; i < 32; ++i) s += part[i];
        *scale = (float)(1.0 / (sqrt(s) + (double)eps));
    }
}

__global__ void __launch_bounds__(THREADS) start(const Matrix p, const float* scale, float* x, int turned, int n) {
    cbm::wait_before();
    const int64_t count = (int64_t)p.rows * p.cols;
    for (int64_t e = (int64_t)blockIdx.x * THREADS + threadIdx.x; e < count; e += (int64_t)gridDim.x * THREADS) {
        const int64_t i = e / n, j = e % n;
        x[e] = *scale * (turned ? update_at(p, j, i) : update_at(p, i, j));
    }
}

// y = f x + h y
__global__ void __launch_bounds__(THREADS) combine(float* y, const float* x, float f, float h, int64_t count) {
    cbm::wait_before();
    for (int64_t e = (int64_t)blockIdx.x * THREADS + threadIdx.x; e < count; e += (int64_t)gridDim.x * THREADS) y[e] = f * x[e] + h * y[e];
}

__global__ void __launch_bounds__(THREADS) finish(const Matrix p, const float* x, int turned, int n) {
    cbm::wait_before();
    const int64_t count = (int64_t)p.rows * p.cols;
    for (int64_t e = (int64_t)blockIdx.x * THREADS + threadIdx.x; e < count; e += (int64_t)gridDim.x * THREADS) {
        const int64_t i = e / p.cols, j = e % p.cols;
        const float o = turned ? x[j * n + i] : x[i * n + j];
        if (p.w) p.w[i * p.ldw + j] = p.keep * p.w[i * p.ldw + j] - p.lr * o;
        else p.out[i * p.ldout + j] = o;
    }
}

unsigned blocks_for(int64_t count) {
    const int64_t b = (count + THREADS - 1) / THREADS;
    return (unsigned)(b < 148 * 8 ? b : 148 * 8);
}

int64_t pad(int64_t floats) { return (floats + 63) / 64 * 64; }

int64_t space_of(int64_t rows, int64_t cols) {
    const int64_t m = rows < cols ? rows : cols;
    return 4 * (2 * pad(rows * cols) + 2 * pad(m * m) + 64);
}

int orthogonal(const Matrix& p, float eps, int steps, void* workspace, void* stream) {
    const cbm::Stream on(static_cast<cudaStream_t>(stream));
    const int turned = p.rows > p.cols, m = turned ? p.cols : p.rows, n = turned ? p.rows : p.cols;
    const int64_t count = (int64_t)m * n;
    float* x = static_cast<float*>(workspace);
    float *y = x + pad(count), *a = y + pad(count), *b = a + pad((int64_t)m * m), *scale = b + pad((int64_t)m * m);
    cbm::launch_next(norm_of_update, dim3(1), 1024, 0, on, p, eps, scale);
    cbm::launch_next(start, dim3(blocks_for(count)), THREADS, 0, on, p, scale, x, turned, n);
    for (int k = 0; k < steps; ++k) {
        if (int rc = cbm_b200_dense_forward(x, n, x, n, a, m, m, n, m, stream)) return rc;
        if (int rc = cbm_b200_dense_forward(a, m, a, m, b, m, m, m, m, stream)) return rc;
        cbm::launch_next(combine, dim3(blocks_for((int64_t)m * m)), THREADS, 0, on, b, a, QUINTIC_B, QUINTIC_C, (int64_t)m * m);
        if (int rc = cbm_b200_dense_grad_input(b, m, x, n, y, n, m, n, m, stream)) return rc;
        cbm::launch_next(combine, dim3(blocks_for(count)), THREADS, 0, on, y, x, QUINTIC_A, 1.f, count);
        float* t = x;
        x = y, y = t;
    }
    cbm::launch_next(finish, dim3(blocks_for(count)), THREADS, 0, on, p, x, turned, n);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? CBM_B200_OK : cbm::fail(CBM_B200_ERR_CUDA, std::string("orthogonal update: ") + cudaGetErrorString(e));
}

}  // namespace

extern "C" int64_t cbm_b200_orthogonalise_workspace(int32_t batch, int32_t rows, int32_t cols) {
    return batch > 0 && rows > 0 && cols > 0 ? space_of(rows, cols) : 0;
}

extern "C" int cbm_b200_orthogonalise(const float* u, int64_t ldu, int64_t next_u, float* out, int64_t ldout, int64_t next_out, int32_t batch,
                                      int32_t rows, int32_t cols, int32_t steps, float eps, void* workspace, int64_t workspace_bytes,
                                      void* stream) {
    if (batch < 0 || rows < 0 || cols < 0 || steps < 1 || steps > CBM_B200_MAX_STEPS || ldu < cols || ldout < cols || !(eps >= 0.f))
        return cbm::fail(CBM_B200_ERR_ARG, "orthogonalise: bad sizes");
    if (batch == 0 || rows == 0 || cols == 0) return CBM_B200_OK;
    if (!u || !out || !workspace) return cbm::fail(CBM_B200_ERR_ARG, "orthogonalise: NULL argument");
    if (workspace_bytes < cbm_b200_orthogonalise_workspace(batch, rows, cols)) return cbm::fail(CBM_B200_ERR_ARG, "orthogonalise: workspace too small");
    for (int i = 0; i < batch; ++i) {
        const Matrix p{u + i * next_u, nullptr, nullptr, out + i * next_out, ldu, 0, 0, ldout, rows, cols, 0.f, 0.f, 0.f, 0.f};
        if (int rc = orthogonal(p, eps, steps, workspace, stream)) return rc;
    }
    return CBM_B200_OK;
}

extern "C" int64_t cbm_b200_orthogonal_step_workspace(const cbm_b200_update_of* of, int32_t count) {
    int64_t most = 0;
    for (int i = 0; of && i < count; ++i)
        if (of[i].rows > 0 && of[i].cols > 0) {
            const int64_t s = space_of(of[i].rows, of[i].cols);
            most = s > most ? s : most;
        }
    return most;
}

extern "C" int cbm_b200_orthogonal_step(const cbm_b200_update_of* of, int32_t count, float lr, float momentum, int32_t nesterov,
                                        float weight_decay, int32_t steps, float eps, void* workspace, int64_t workspace_bytes, void* stream) {
    if (count < 0 || (count && !of) || steps < 1 || steps > CBM_B200_MAX_STEPS || !(eps >= 0.f))
        return cbm::fail(CBM_B200_ERR_ARG, "orthogonal_step: bad arguments");
    for (int i = 0; i < count; ++i) {
        const cbm_b200_update_of& u = of[i];
        if (u.rows < 0 || u.cols < 0 || u.ldw < u.cols || u.ldg < u.cols || u.ldm < u.cols) return cbm::fail(CBM_B200_ERR_ARG, "orthogonal_step: bad sizes");
        if (u.rows && u.cols && (!u.w || !u.g || !u.m)) return cbm::fail(CBM_B200_ERR_ARG, "orthogonal_step: NULL argument");
    }
    const int64_t need = cbm_b200_orthogonal_step_workspace(of, count);
    if (need && (!workspace || workspace_bytes < need)) return cbm::fail(CBM_B200_ERR_ARG, "orthogonal_step: workspace too small");
    for (int i = 0; i < count; ++i) {
        const cbm_b200_update_of& u = of[i];
        if (u.rows == 0 || u.cols == 0) continue;
        const double tall = u.rows > u.cols ? std::sqrt((double)u.rows / u.cols) : 1.0;
        const Matrix p{u.g, u.m, u.w, nullptr, u.ldg, u.ldm, u.ldw, 0, u.rows, u.cols, (float)(lr * tall), momentum, nesterov ? 1.f : 0.f, (float)(1.0 - (double)lr * weight_decay)};
        if (int rc = orthogonal(p, eps, steps, workspace, stream)) return rc;
    }
    return CBM_B200_OK;
}
