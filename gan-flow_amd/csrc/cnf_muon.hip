// cnf_muon.hip -- Newton-Schulz orthogonalisation of matrices, and the Muon update built on it.
//
//   X0 = G / (|G|_F + eps);   A = X X^T;   X <- a X + (b A + c A^2) X     for each step's (a, b, c)
// on the side that is shorter (m <= n after a transposition), for `count` matrices of one shape at a time.  The Muon update:
//   M <- mu M + g;   G = g + mu M (Nesterov) or M;   W <- (1 - lr wd) W - lr scale X.
// The Frobenius norm is summed in double from per-block partial sums added in a fixed order; everything else is fp32.
#include "cnf_ops.h"

namespace cnf {
namespace {

constexpr int kThreads = 256;
constexpr int kNormBlocks = 128;

struct Ptrs {
    const void* g[CNF_MAX_MATRICES];
    void* out[CNF_MAX_MATRICES];
    float* m[CNF_MAX_MATRICES];
};

struct Dims {
    long rows, cols, ldg, ldo, ldm;
    long m, n;      // the shorter and the longer side
    int tall;       // rows > cols: the iteration runs on the transposed matrix
};

// the matrix the iteration starts from, before normalisation: X (m x n) and the partial sums of its squares
template <typename T, bool kMuon>
__global__ __launch_bounds__(kThreads) void begin_kernel(Ptrs p, Dims d, float* x, double* part, float mu, int nesterov,
                                                         const CnfStats* guard) {
    __shared__ double red[kThreads / 64];
    const int mat = blockIdx.y;
    const bool skip = guard && guard->status != 0;
    const T* g = (const T*)p.g[mat];
    float* xm = x + (long)mat * d.m * d.n;
    double s = 0.;
    for (long i = (long)blockIdx.x * kThreads + threadIdx.x; i < d.rows * d.cols; i += (long)gridDim.x * kThreads) {
        const long r = i / d.cols, c = i % d.cols;
        float v = to_f32(g[r * d.ldg + c]);
        if (kMuon) {
            float* pm = p.m[mat] + r * d.ldm + c;
            const float mv = fmaf(mu, *pm, v);
            if (!skip) *pm = mv;
            v = nesterov ? fmaf(mu, mv, v) : mv;
        }
        xm[d.tall ? c * d.n + r : i] = v;
        s += (double)v * (double)v;
    }
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) part[mat * kNormBlocks + blockIdx.x] = (red[0] + red[1]) + (red[2] + red[3]);
}

__global__ __launch_bounds__(kThreads) void normalize_kernel(Dims d, float* x, const double* part, double eps) {
    __shared__ float inv;
    const int mat = blockIdx.y;
    if (threadIdx.x == 0) {
        double s = 0.;
        for (int k = 0; k < kNormBlocks; ++k) s += part[mat * kNormBlocks + k];
        inv = (float)(1.0 / (sqrt(s) + eps));
    }
    __syncthreads();
    for (long i = (long)blockIdx.x * kThreads + threadIdx.x; i < d.m * d.n; i += (long)gridDim.x * kThreads) x[(long)mat * d.m * d.n + i] *= inv;
}

// C (M x N) = alpha op(P, Q) + beta D;  kNT: sum_k P[i,k] Q[j,k], else sum_k P[i,k] Q[k,j].  64 x 64 tile, 4 x 4 per thread.
template <bool kNT>
__global__ __launch_bounds__(kThreads) void gemm_kernel(const float* p, const float* q, const float* dd, float* cc, long M, long N, long K,
                                                        long bp, long bq, long bd, long bc, float alpha, float beta) {
    __shared__ float ps[16][65], qs[16][65];
    const int mat = blockIdx.z;
    p += mat * bp, q += mat * bq, cc += mat * bc;
    const long i0 = (long)blockIdx.y * 64, j0 = (long)blockIdx.x * 64;
    const int ti = threadIdx.x >> 4, tj = threadIdx.x & 15;
    float acc[4][4] = {};
    for (long k0 = 0; k0 < K; k0 += 16) {
        for (int e = threadIdx.x; e < 1024; e += kThreads) {
            const int row = e >> 4, k = e & 15;
            ps[k][row] = (i0 + row < M && k0 + k < K) ? p[(i0 + row) * K + k0 + k] : 0.f;
            if (kNT) {
                qs[k][row] = (j0 + row < N && k0 + k < K) ? q[(j0 + row) * K + k0 + k] : 0.f;
            } else {
                const int kk = e >> 6, col = e & 63;
                qs[kk][col] = (j0 + col < N && k0 + kk < K) ? q[(k0 + kk) * N + j0 + col] : 0.f;
            }
        }
        __syncthreads();
        for (int k = 0; k < 16; ++k)
            for (int u = 0; u < 4; ++u)
                for (int v = 0; v < 4; ++v) acc[u][v] = fmaf(ps[k][ti + 16 * u], qs[k][tj + 16 * v], acc[u][v]);
        __syncthreads();
    }
    for (int u = 0; u < 4; ++u)
        for (int v = 0; v < 4; ++v) {
            const long i = i0 + ti + 16 * u, j = j0 + tj + 16 * v;
            if (i < M && j < N) cc[i * N + j] = alpha * acc[u][v] + (dd ? beta * dd[mat * bd + i * N + j] : 0.f);
        }
}

template <typename T, bool kMuon>
__global__ __launch_bounds__(kThreads) void end_kernel(Ptrs p, Dims d, const float* x, float decay, float step, const CnfStats* guard) {
    if (guard && guard->status != 0) return;
    const int mat = blockIdx.y;
    T* out = (T*)p.out[mat];
    const float* xm = x + (long)mat * d.m * d.n;
    for (long i = (long)blockIdx.x * kThreads + threadIdx.x; i < d.rows * d.cols; i += (long)gridDim.x * kThreads) {
        const long r = i / d.cols, c = i % d.cols;
        const float v = xm[d.tall ? c * d.n + r : i];
        T* o = out + r * d.ldo + c;
        *o = from_f32<T>(kMuon ? fmaf(-step, v, decay * to_f32(*o)) : v);
    }
}

template <typename T, bool kMuon>
hipError_t run(const MuonArgs& a, hipStream_t s) {
    Ptrs p{};
    for (int i = 0; i < a.count; ++i) {
        p.g[i] = a.g[i];
        p.out[i] = a.out[i];
        p.m[i] = kMuon ? a.momenta[i] : nullptr;
    }
    Dims d{a.rows, a.cols, a.ldg, a.ldo, a.ldm, a.rows < a.cols ? a.rows : a.cols, a.rows < a.cols ? a.cols : a.rows, a.rows > a.cols};
    const long mn = d.m * d.n, mm = d.m * d.m;
    double* part = (double*)a.ws;
    float *x = (float*)(part + (size_t)a.count * kNormBlocks), *x2 = x + a.count * mn, *A = x2 + a.count * mn, *B = A + a.count * mm;
    const float mu = kMuon ? (float)a.opts->momentum : 0.f;
    const dim3 elem(kNormBlocks, a.count);
    begin_kernel<T, kMuon><<<elem, kThreads, 0, s>>>(p, d, x, part, mu, kMuon ? a.opts->nesterov : 0, a.guard);
    normalize_kernel<<<elem, kThreads, 0, s>>>(d, x, part, a.ns->eps);
    const unsigned tm = (unsigned)((d.m + 63) / 64), tn = (unsigned)((d.n + 63) / 64);
    for (int k = 0; k < a.ns->steps; ++k) {
        gemm_kernel<true><<<dim3(tm, tm, a.count), kThreads, 0, s>>>(x, x, nullptr, A, d.m, d.m, d.n, mn, mn, 0, mm, 1.f, 0.f);
        gemm_kernel<true><<<dim3(tm, tm, a.count), kThreads, 0, s>>>(A, A, A, B, d.m, d.m, d.m, mm, mm, mm, mm, (float)a.ns->c[k], (float)a.ns->b[k]);
        gemm_kernel<false><<<dim3(tn, tm, a.count), kThreads, 0, s>>>(B, x, x, x2, d.m, d.n, d.m, mm, mn, mn, mn, 1.f, (float)a.ns->a[k]);
        float* t = x;
        x = x2;
        x2 = t;
    }
    const float decay = kMuon ? (float)(1.0 - a.opts->lr * a.opts->weight_decay) : 1.f;
    const float step = kMuon ? (float)(a.opts->lr * a.opts->scale) : 1.f;
    end_kernel<T, kMuon><<<elem, kThreads, 0, s>>>(p, d, x, decay, step, a.guard);
    return hipGetLastError();
}

template <typename T>
hipError_t run_op(const MuonArgs& a, hipStream_t s) {
    return a.opts ? run<T, true>(a, s) : run<T, false>(a, s);
}

}  // namespace

size_t muon_workspace_bytes(long count, long rows, long cols) {
    const size_t m = rows < cols ? rows : cols, n = rows < cols ? cols : rows;
    return (size_t)count * (kNormBlocks * sizeof(double) + (2 * m * n + 2 * m * m) * sizeof(float));
}

hipError_t launch_muon(int dtype, const MuonArgs& a, hipStream_t s) {
    if (dtype == CNF_F32) return run_op<float>(a, s);
    if (dtype == CNF_F16) return run_op<f16>(a, s);
    if (dtype == CNF_BF16) return run_op<bf16>(a, s);
    return hipErrorInvalidValue;
}

}  // namespace cnf
