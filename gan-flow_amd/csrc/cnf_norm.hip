// cnf_norm.hip -- layer normalisation of the rows of a (rows x cols) matrix and its backward pass.
//
//   y = (x - mean) rstd w + b,   mean = sum x / n,   rstd = (sum (x - mean)^2 / n + eps)^(-1/2)      (per row, n = cols)
//   h = dy w,  xh = (x - mean) rstd:
//   dx = rstd (h - mean(h) - xh mean(h xh)),   dw = sum over rows of dy xh,   db = sum over rows of dy
//
// All statistics and sums are fp32 (the variance from centred values, never as a difference of moments).  The column sums
// go through partial sums per block of rows that a second kernel adds in a fixed order: no atomics, the same bits every run.
#include "cnf_ops.h"

namespace cnf {
namespace {

constexpr int kThreads = 256;
constexpr long kMaxChunks = 256;

__device__ __forceinline__ float block_sum(float v, float* red) {
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return red[0] + red[1] + red[2] + red[3];
}

template <typename T, typename W>
__global__ __launch_bounds__(kThreads) void norm_fwd_kernel(NormArgs a) {
    __shared__ float red[kThreads / 64];
    const T* x = (const T*)a.x;
    const W *w = (const W*)a.weight, *b = (const W*)a.bias;
    T* y = (T*)a.y;
    const float inv_n = 1.0f / (float)a.cols;
    for (long r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T* xr = x + r * a.x_stride;
        float s = 0.f, q = 0.f;
        for (long c = threadIdx.x; c < a.cols; c += kThreads) s += to_f32(xr[c]);
        const float mean = block_sum(s, red) * inv_n;
        for (long c = threadIdx.x; c < a.cols; c += kThreads) {
            const float d = to_f32(xr[c]) - mean;
            q = fmaf(d, d, q);
        }
        const float rstd = 1.0f / sqrtf(block_sum(q, red) * inv_n + a.eps);
        for (long c = threadIdx.x; c < a.cols; c += kThreads) {
            float v = (to_f32(xr[c]) - mean) * rstd;
            if (w) v *= to_f32(w[c]);
            if (b) v += to_f32(b[c]);
            y[r * a.cols + c] = from_f32<T>(v);
        }
        if (threadIdx.x == 0) {
            if (a.mean) a.mean[r] = mean;
            if (a.rstd) a.rstd[r] = rstd;
        }
    }
}

template <typename T, typename W>
__global__ __launch_bounds__(kThreads) void norm_dx_kernel(NormArgs a) {
    __shared__ float red[kThreads / 64];
    const T *x = (const T*)a.x, *dy = (const T*)a.dy;
    const W* w = (const W*)a.weight;
    T* dx = (T*)a.dx;
    const float inv_n = 1.0f / (float)a.cols;
    for (long r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T *xr = x + r * a.x_stride, *gr = dy + r * a.dy_stride;
        const float mean = a.mean[r], rstd = a.rstd[r];
        float s = 0.f, q = 0.f;
        for (long c = threadIdx.x; c < a.cols; c += kThreads) {
            const float h = w ? to_f32(gr[c]) * to_f32(w[c]) : to_f32(gr[c]);
            s += h;
            q = fmaf(h, (to_f32(xr[c]) - mean) * rstd, q);
        }
        const float mh = block_sum(s, red) * inv_n, mx = block_sum(q, red) * inv_n;
        for (long c = threadIdx.x; c < a.cols; c += kThreads) {
            const float h = w ? to_f32(gr[c]) * to_f32(w[c]) : to_f32(gr[c]);
            dx[r * a.cols + c] = from_f32<T>(rstd * (h - mh - (to_f32(xr[c]) - mean) * rstd * mx));
        }
    }
}

// partial column sums of one chunk of rows: part[0][chunk][col] = sum dy xh, part[1][chunk][col] = sum dy
template <typename T>
__global__ __launch_bounds__(kThreads) void norm_part_kernel(NormArgs a, long chunks) {
    __shared__ float red[2][kThreads];
    const T *x = (const T*)a.x, *dy = (const T*)a.dy;
    const long c = (long)blockIdx.x * 64 + (threadIdx.x & 63), per = (a.rows + chunks - 1) / chunks;
    const long r0 = blockIdx.y * per, r1 = r0 + per < a.rows ? r0 + per : a.rows;
    float sw = 0.f, sb = 0.f;
    if (c < a.cols)
        for (long r = r0 + (threadIdx.x >> 6); r < r1; r += kThreads / 64) {
            const float g = to_f32(dy[r * a.dy_stride + c]);
            sw = fmaf(g, (to_f32(x[r * a.x_stride + c]) - a.mean[r]) * a.rstd[r], sw);
            sb += g;
        }
    red[0][threadIdx.x] = sw;
    red[1][threadIdx.x] = sb;
    __syncthreads();
    if (threadIdx.x < 64 && c < a.cols)
        for (int k = 0; k < 2; ++k)
            a.part[(k * chunks + blockIdx.y) * a.cols + c] =
                (red[k][threadIdx.x] + red[k][threadIdx.x + 64]) + (red[k][threadIdx.x + 128] + red[k][threadIdx.x + 192]);
}

template <typename W>
__global__ __launch_bounds__(kThreads) void norm_cols_kernel(NormArgs a, long chunks) {
    const long c = (long)blockIdx.x * kThreads + threadIdx.x;
    W* out = (W*)(blockIdx.y ? a.dbias : a.dweight);
    if (c >= a.cols || !out) return;
    const float* p = a.part + (long)blockIdx.y * chunks * a.cols + c;
    float s = 0.f;
    for (long k = 0; k < chunks; ++k) s += p[k * a.cols];
    out[c] = from_f32<W>(s);
}

long chunks_of(long rows) {
    const long c = (rows + 63) / 64;
    return c < kMaxChunks ? c : kMaxChunks;
}

template <typename T, typename W>
hipError_t fwd(const NormArgs& a, hipStream_t s) {
    const long grid = a.rows < 65536 ? a.rows : 65536;
    norm_fwd_kernel<T, W><<<dim3((unsigned)grid), dim3(kThreads), 0, s>>>(a);
    return hipGetLastError();
}

template <typename T, typename W>
hipError_t bwd(const NormArgs& a, hipStream_t s) {
    const long chunks = chunks_of(a.rows);
    if (a.dx && a.rows > 0) {
        const long grid = a.rows < 65536 ? a.rows : 65536;
        norm_dx_kernel<T, W><<<dim3((unsigned)grid), dim3(kThreads), 0, s>>>(a);
    }
    if (a.dweight || a.dbias) {
        if (chunks > 0) norm_part_kernel<T><<<dim3((unsigned)((a.cols + 63) / 64), (unsigned)chunks), dim3(kThreads), 0, s>>>(a, chunks);
        norm_cols_kernel<W><<<dim3((unsigned)((a.cols + kThreads - 1) / kThreads), 2), dim3(kThreads), 0, s>>>(a, chunks);
    }
    return hipGetLastError();
}

}  // namespace

size_t layer_norm_workspace_bytes(long rows, long cols) { return (size_t)2 * chunks_of(rows) * cols * sizeof(float); }

#define CNF_NORM_DISPATCH(fn)                                                          \
    if (dtype == CNF_F32 && wdtype == CNF_F32) return fn<float, float>(a, s);           \
    if (dtype == CNF_F16 && wdtype == CNF_F32) return fn<f16, float>(a, s);             \
    if (dtype == CNF_F16 && wdtype == CNF_F16) return fn<f16, f16>(a, s);               \
    if (dtype == CNF_BF16 && wdtype == CNF_F32) return fn<bf16, float>(a, s);           \
    if (dtype == CNF_BF16 && wdtype == CNF_BF16) return fn<bf16, bf16>(a, s);           \
    return hipErrorInvalidValue;

hipError_t launch_layer_norm_fwd(int dtype, int wdtype, const NormArgs& a, hipStream_t s) { CNF_NORM_DISPATCH(fwd) }
hipError_t launch_layer_norm_bwd(int dtype, int wdtype, const NormArgs& a, hipStream_t s) { CNF_NORM_DISPATCH(bwd) }

}  // namespace cnf
