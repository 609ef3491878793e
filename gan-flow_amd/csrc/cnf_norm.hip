// cnf_norm.hip -- layer normalisation of the rows of a (rows x cols) matrix and its backward pass.
//
//   y = (x - mean) rstd w + b,   mean = sum x / n,   rstd = (sum (x - mean)^2 / n + eps)^(-1/2)      (per row, n = cols)
//   h = dy w,  xh = (x - mean) rstd:
//   dx = rstd (h - mean(h) - xh mean(h xh)),   dw = sum over rows of dy xh,   db = sum over rows of dy
//
// All statistics and sums are fp32 (the variance from centred values, never as a difference of moments).  Bound by memory: every element
// is read once and written once, so a row stays in registers between its statistics and its result -- 16 bytes of it at a time per
// thread, loaded at whatever alignment the rows have.  A row belongs to a power of two of a wave's lanes while it fits two chunks a
// lane, to a workgroup of 256 threads beyond that (up to 8192 columns), and is read again for each pass in the kernels at the
// end of this file beyond that.  The weights stay in registers while a workgroup goes through its rows.
// The column sums of the backward pass are kept per thread over a workgroup's rows, written as one partial sum per workgroup, and added by a second
// kernel in a fixed order: no atomics, the same bits every run.
#include "cnf_ops.h"

namespace cnf {
namespace {

constexpr int kThreads = 256;
constexpr long kMaxBlocks = 2048;     // forward: eight workgroups per CU
constexpr long kInRegisters = 8192;   // columns

template <typename T>
constexpr int kVec = 16 / sizeof(T);

// one chunk of a row: kVec<T> elements, the ones past the end 0
template <typename T, typename E = T>
struct Chunk {
    static constexpr int V = kVec<T>;
    E e[V];

    __device__ __forceinline__ void load(const E* p, long at, long n) {
        if (at + V <= n) {
            __builtin_memcpy(e, (const char*)(p + at), sizeof e);
        } else {
            for (int k = 0; k < V; ++k) e[k] = at + k < n ? p[at + k] : from_f32<E>(0.f);
        }
    }
    __device__ __forceinline__ void store(E* p, long at, long n) const {
        if (at + V <= n) {
            __builtin_memcpy((char*)(p + at), e, sizeof e);
        } else {
            for (int k = 0; k < V; ++k)
                if (at + k < n) p[at + k] = e[k];
        }
    }
    __device__ __forceinline__ float operator[](int k) const { return to_f32(e[k]); }
};

// sums over the threads of a row: `group`, a power of two of a wave's lanes, or (TB > 0) the workgroup's TB; red: this sum's own LDS words
template <int TB, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], int group, float (*red)[TB > 0 ? TB / 64 : 1]) {
    for (int o = (TB > 0 ? 64 : group) / 2; o > 0; o >>= 1)
        for (int k = 0; k < N; ++k) v[k] += __shfl_xor(v[k], o);
    if constexpr (TB > 0) {
        if ((threadIdx.x & 63) == 0)
            for (int k = 0; k < N; ++k) red[k][threadIdx.x >> 6] = v[k];
        __syncthreads();
        for (int k = 0; k < N; ++k) {
            v[k] = 0.f;
            for (int u = 0; u < TB / 64; u += 4) v[k] += (red[k][u] + red[k][u + 1]) + (red[k][u + 2] + red[k][u + 3]);
        }
    }
}

template <typename T, typename W, int NC, bool kBlock>
__global__ __launch_bounds__(kThreads) void norm_fwd_kernel(NormArgs a, int group) {
    constexpr int V = kVec<T>;
    constexpr int TB = kBlock ? kThreads : 0;
    __shared__ float red[2][1][kBlock ? kThreads / 64 : 1];
    const int lane = kBlock ? threadIdx.x : threadIdx.x & (group - 1), sub = kBlock ? 0 : threadIdx.x / group;
    const int across = kBlock ? kThreads : group, high = kThreads / across;
    const T* x = (const T*)a.x;
    const W *w = (const W*)a.weight, *b = (const W*)a.bias;
    T* y = (T*)a.y;
    const float inv_n = 1.0f / (float)a.cols;
    Chunk<T, W> wc[NC], bc[NC];
    for (int j = 0; j < NC; ++j) {
        const long c = (long)(j * across + lane) * V;
        if (w) wc[j].load(w, c, a.cols);
        if (b) bc[j].load(b, c, a.cols);
    }
    // (a group past the last row has no work, but goes round with its workgroup: uniform barriers)
    for (long r0 = (long)blockIdx.x * high; r0 < a.rows; r0 += (long)gridDim.x * high) {
        const long r = r0 + sub;
        const bool on = kBlock || r < a.rows;
        const T* xr = x + (on ? r : r0) * a.x_stride;
        Chunk<T> xc[NC];
        for (int j = 0; j < NC; ++j) xc[j].load(xr, (long)(j * across + lane) * V, a.cols);
        float s[1] = {0.f};
        for (int j = 0; j < NC; ++j)
            for (int k = 0; k < V; ++k) s[0] += xc[j][k];
        row_sum<TB>(s, group, red[0]);
        const float mean = s[0] * inv_n;
        float q[1] = {0.f};
        for (int j = 0; j < NC; ++j)
            for (int k = 0; k < V; ++k) {
                const float d = xc[j][k] - mean;
                q[0] = (long)(j * across + lane) * V + k < a.cols ? fmaf(d, d, q[0]) : q[0];
            }
        row_sum<TB>(q, group, red[1]);
        const float rstd = 1.0f / sqrtf(q[0] * inv_n + a.eps);
        if (!on) continue;
        for (int j = 0; j < NC; ++j) {
            const long c = (long)(j * across + lane) * V;
            if (c >= a.cols) continue;
            Chunk<T> out;
            for (int k = 0; k < V; ++k) {
                float v = (xc[j][k] - mean) * rstd;
                if (w) v *= wc[j][k];
                if (b) v += bc[j][k];
                out.e[k] = from_f32<T>(v);
            }
            out.store(y + r * a.cols, c, a.cols);
        }
        if (lane == 0) {
            if (a.mean) a.mean[r] = mean;
            if (a.rstd) a.rstd[r] = rstd;
        }
    }
}

// dx of a workgroup's rows, and their partial column sums to part[block][0 | 1][col] (dy xh | dy)
// TB: threads that share a row, or 0: a wave's lanes by `group`, 256 threads
template <typename T, typename W, int NC, int TB>
__global__ __launch_bounds__(TB > 0 ? TB : kThreads) void norm_bwd_kernel(NormArgs a, int group) {
    constexpr int V = kVec<T>;
    constexpr bool kBlock = TB > 0;
    __shared__ float red[2][2][kBlock ? TB / 64 : 1];
    __shared__ float sums[kBlock ? 1 : kThreads / 64][kBlock ? 1 : 64 * NC * V];
    const int lane = kBlock ? threadIdx.x : threadIdx.x & (group - 1), sub = kBlock ? 0 : threadIdx.x / group;
    const int across = kBlock ? TB : group, high = kBlock ? 1 : kThreads / group;
    const T *x = (const T*)a.x, *dy = (const T*)a.dy;
    const W* w = (const W*)a.weight;
    T* dx = (T*)a.dx;
    const float inv_n = 1.0f / (float)a.cols;
    Chunk<T, W> wc[NC];
    if (w)
        for (int j = 0; j < NC; ++j) wc[j].load(w, (long)(j * across + lane) * V, a.cols);
    float dw[NC][V] = {}, db[NC][V] = {};
    Chunk<T> xn[NC], gn[NC];                                 // the next row, on its way while this one is worked on
    float mean_n = 0.f, rstd_n = 0.f;
    auto fetch = [&](long r0) {
        const long rr = kBlock || r0 + sub < a.rows ? r0 + sub : r0;
        for (int j = 0; j < NC; ++j) {
            const long c = (long)(j * across + lane) * V;
            xn[j].load(x + rr * a.x_stride, c, a.cols);
            gn[j].load(dy + rr * a.dy_stride, c, a.cols);
        }
        mean_n = a.mean[rr], rstd_n = a.rstd[rr];
    };
    int turn = 0;
    const long step = (long)gridDim.x * high;
    if ((long)blockIdx.x * high < a.rows) fetch((long)blockIdx.x * high);
    for (long r0 = (long)blockIdx.x * high; r0 < a.rows; r0 += step) {
        const long r = r0 + sub;
        const bool on = kBlock || r < a.rows;
        Chunk<T> xc[NC], gc[NC];
        for (int j = 0; j < NC; ++j) xc[j] = xn[j], gc[j] = gn[j];
        const float mean = mean_n, rstd = rstd_n;
        if (r0 + step < a.rows) fetch(r0 + step);
        // (past the end of the row dy and w are 0: nothing to leave out)
        float s[2] = {0.f, 0.f};
        for (int j = 0; j < NC; ++j)
            for (int k = 0; k < V; ++k) {
                const float g = gc[j][k], xm = xc[j][k] - mean, h = w ? g * wc[j][k] : g;
                s[0] += h;
                s[1] = fmaf(h, xm, s[1]);
                const float gr = on ? g * rstd : 0.f;
                dw[j][k] = fmaf(gr, xm, dw[j][k]);
                db[j][k] += on ? g : 0.f;
            }
        if (!dx) continue;                                   // (a kernel argument: the same way round for every thread)
        row_sum<TB>(s, group, red[turn]);
        turn ^= 1;
        if (!on) continue;
        // dx = rstd h - (x - mean) rstd^2 mean(h xh) - rstd mean(h)
        const float c0 = -rstd * (s[0] * inv_n), c1 = -(rstd * rstd) * ((s[1] * rstd) * inv_n);
        for (int j = 0; j < NC; ++j) {
            const long c = (long)(j * across + lane) * V;
            if (c >= a.cols) continue;
            Chunk<T> out;
            for (int k = 0; k < V; ++k) {
                const float h = w ? gc[j][k] * wc[j][k] : gc[j][k];
                out.e[k] = from_f32<T>(fmaf(h, rstd, fmaf(xc[j][k] - mean, c1, c0)));
            }
            out.store(dx + r * a.cols, c, a.cols);
        }
    }
    if (!a.dweight && !a.dbias) return;
    float* part = a.part + (long)blockIdx.x * 2 * a.cols;
    if (kBlock) {
        for (int j = 0; j < NC; ++j)
            for (int k = 0; k < V; ++k) {
                const long c = (long)(j * across + lane) * V + k;
                if (c < a.cols) part[c] = dw[j][k], part[a.cols + c] = db[j][k];
            }
        return;
    }
    // the rows of a wave side by side, then the waves
    for (int which = 0; which < 2; ++which) {
        for (int j = 0; j < NC; ++j)
            for (int k = 0; k < V; ++k) {
                float v = which ? db[j][k] : dw[j][k];
                for (int o = group; o < 64; o <<= 1) v += __shfl_xor(v, o);
                if ((threadIdx.x & 63) < group) sums[threadIdx.x >> 6][(j * group + lane) * V + k] = v;
            }
        __syncthreads();
        for (long c = threadIdx.x; c < a.cols; c += kThreads) part[which * a.cols + c] = (sums[0][c] + sums[1][c]) + (sums[2][c] + sums[3][c]);
        __syncthreads();
    }
}

// dweight and dbias: the sum of `parts` partial sums; 32 columns per workgroup, 32 threads over the partial sums of each
constexpr int kSumThreads = 1024;

template <typename W>
__global__ __launch_bounds__(kSumThreads) void norm_cols_kernel(NormArgs a, long parts) {
    __shared__ float red[32][33];
    const int which = blockIdx.y, col = threadIdx.x & 31, split = threadIdx.x >> 5;
    W* out = (W*)(which ? a.dbias : a.dweight);
    if (!out) return;
    const long c = (long)blockIdx.x * 32 + col;
    float s[4] = {};
    if (c < a.cols) {
        const float* p = a.part + which * a.cols + c;
        const long step = 2 * a.cols;
        long k = split;
        for (; k + 224 < parts; k += 256) {                  // (eight loads at a time: the latency of one)
            float v[8];
            for (int u = 0; u < 8; ++u) v[u] = p[(k + u * 32) * step];
            for (int u = 0; u < 8; ++u) s[u & 3] += v[u];
        }
        for (; k < parts; k += 32) s[0] += p[k * step];
    }
    red[split][col] = (s[0] + s[1]) + (s[2] + s[3]);
    __syncthreads();
    for (int half = 16; half > 0; half >>= 1) {
        if (split < half) red[split][col] += red[split + half][col];
        __syncthreads();
    }
    if (split == 0 && c < a.cols) out[c] = from_f32<W>(red[0][col]);
}

// ---- rows too long for registers: a workgroup per row, which reads it again for each pass ------------------------------------------

__device__ __forceinline__ float block_sum(float v, float* red) {
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return (red[0] + red[1]) + (red[2] + red[3]);
}

template <typename T, typename W>
__global__ __launch_bounds__(kThreads) void long_fwd_kernel(NormArgs a) {
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
__global__ __launch_bounds__(kThreads) void long_dx_kernel(NormArgs a) {
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

// partial column sums of chunk blockIdx.y of the rows, 64 columns per workgroup
template <typename T>
__global__ __launch_bounds__(kThreads) void long_part_kernel(NormArgs a, long parts) {
    __shared__ float red[2][kThreads];
    const T *x = (const T*)a.x, *dy = (const T*)a.dy;
    const long c = (long)blockIdx.x * 64 + (threadIdx.x & 63), per = (a.rows + parts - 1) / parts;
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
            a.part[((long)blockIdx.y * 2 + k) * a.cols + c] =
                (red[k][threadIdx.x] + red[k][threadIdx.x + 64]) + (red[k][threadIdx.x + 128] + red[k][threadIdx.x + 192]);
}

// ---- launches --------------------------------------------------------------------------------------------------------------------

// threads per row and chunks per thread: a wave's lanes while kWaveChunks chunks each hold the row, else the workgroup
constexpr int kWaveChunks = 2;
constexpr long kBwdThreads = 1024 * 256;   // resident in the backward kernel, about
struct Shape {
    int group, chunks;
    bool block;
};

Shape shape_of(long cols, int vec) {
    const long n = (cols + vec - 1) / vec;
    Shape s{1, 1, false};
    while (s.group < 64 && s.group < n) s.group *= 2;
    if (n > 64 * kWaveChunks) s.block = true, s.group = kThreads;
    while ((long)s.group * s.chunks < n) s.chunks *= 2;
    return s;
}

// backward: past a wave one chunk per thread and as many threads as the row needs -- a thread holds 2 kVec column sums per chunk, and what
// bounds the kernel is how many loads are in flight.  `most`: workgroups, each with a partial sum to write: as many as are resident.
// us for 16-bit rows, x, dy and dx 402 MB: 2048 columns 105, 4096 columns 106 (two chunks on 256 threads: 112 .. 150), 8192 columns
// 118 (four chunks on 256: 220 .. 250); 1024 columns, two chunks a lane, 98 with 768 workgroups and 133 with 1024.
Shape bwd_shape(long cols, int vec, long& most) {
    Shape s = shape_of(cols, vec);
    most = s.chunks == 2 && vec == 8 ? 768 : 1024;
    if (s.block) {
        const long n = (cols + vec - 1) / vec;
        s.group = n <= 256 ? 256 : n <= 512 ? 512 : 1024;
        s.chunks = n <= 1024 ? 1 : 2;
        most = kBwdThreads / s.group;
    }
    return s;
}

long parts_of(long rows, long cols, int vec) {
    if (cols > kInRegisters) {
        const long c = (rows + 63) / 64;
        return c < 256 ? c : 256;
    }
    long most;
    const Shape s = bwd_shape(cols, vec, most);
    const long high = s.block ? 1 : kThreads / s.group, c = (rows + high - 1) / high;
    return c < most ? c : most;
}

template <typename T, typename W>
hipError_t fwd(const NormArgs& a, hipStream_t s) {
    if (a.cols > kInRegisters) {
        long_fwd_kernel<T, W><<<dim3((unsigned)(a.rows < 65536 ? a.rows : 65536)), kThreads, 0, s>>>(a);
        return hipGetLastError();
    }
    const Shape p = shape_of(a.cols, kVec<T>);
    const long high = kThreads / p.group, blocks = (a.rows + high - 1) / high;
    const dim3 grid((unsigned)(blocks < kMaxBlocks ? blocks : kMaxBlocks));
    if (!p.block && p.chunks == 1) norm_fwd_kernel<T, W, 1, false><<<grid, kThreads, 0, s>>>(a, p.group);
    else if (!p.block) norm_fwd_kernel<T, W, 2, false><<<grid, kThreads, 0, s>>>(a, p.group);
    else if (p.chunks == 1) norm_fwd_kernel<T, W, 1, true><<<grid, kThreads, 0, s>>>(a, p.group);
    else if (p.chunks == 2) norm_fwd_kernel<T, W, 2, true><<<grid, kThreads, 0, s>>>(a, p.group);
    else if (p.chunks == 4) norm_fwd_kernel<T, W, 4, true><<<grid, kThreads, 0, s>>>(a, p.group);
    else if constexpr (kVec<T> == 4) norm_fwd_kernel<T, W, 8, true><<<grid, kThreads, 0, s>>>(a, p.group);
    return hipGetLastError();
}

template <typename T, typename W>
hipError_t bwd(const NormArgs& a, hipStream_t s) {
    const long parts = parts_of(a.rows, a.cols, kVec<T>);
    const bool sums = a.dweight || a.dbias;
    if (a.cols > kInRegisters) {
        if (a.dx && a.rows > 0) long_dx_kernel<T, W><<<dim3((unsigned)(a.rows < 65536 ? a.rows : 65536)), kThreads, 0, s>>>(a);
        if (sums && parts > 0) long_part_kernel<T><<<dim3((unsigned)((a.cols + 63) / 64), (unsigned)parts), kThreads, 0, s>>>(a, parts);
    } else if (a.rows > 0) {
        long most;
        const Shape p = bwd_shape(a.cols, kVec<T>, most);
        const dim3 grid((unsigned)parts);
        if (!p.block && p.chunks == 1) norm_bwd_kernel<T, W, 1, 0><<<grid, kThreads, 0, s>>>(a, p.group);
        else if (!p.block) norm_bwd_kernel<T, W, 2, 0><<<grid, kThreads, 0, s>>>(a, p.group);
        else if (p.group == 256) norm_bwd_kernel<T, W, 1, 256><<<grid, 256, 0, s>>>(a, p.group);
        else if (p.group == 512) norm_bwd_kernel<T, W, 1, 512><<<grid, 512, 0, s>>>(a, p.group);
        else if (p.chunks == 1) norm_bwd_kernel<T, W, 1, 1024><<<grid, 1024, 0, s>>>(a, p.group);
        else if constexpr (kVec<T> == 4) norm_bwd_kernel<T, W, 2, 1024><<<grid, 1024, 0, s>>>(a, p.group);
    }
    if (sums) norm_cols_kernel<W><<<dim3((unsigned)((a.cols + 31) / 32), 2), kSumThreads, 0, s>>>(a, parts);
    return hipGetLastError();
}

}  // namespace

size_t layer_norm_workspace_bytes(long rows, long cols) {
    const long p = parts_of(rows, cols, 4), q = parts_of(rows, cols, 8);
    return (size_t)2 * (p > q ? p : q) * cols * sizeof(float);
}

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
