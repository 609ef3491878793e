// cnf_muon.hip -- Newton-Schulz orthogonalisation of matrices, and the Muon update built on it.
//
//   X0 = G / (|G|_F + eps);   A = X X^T;   X <- a X + (b A + c A^2) X     for each step's (a, b, c)
// on the side that is shorter (m <= n after a transposition), for `count` matrices of one shape at a time.  The Muon update:
//   M <- mu M + g;   G = g + mu M (Nesterov) or M;   W <- (1 - lr wd) W - lr scale X.
//
// ARITHMETIC.  The steps amplify small singular values (3.4445-fold each with the usual coefficients, 485-fold over five), and
// a rounding of the operands with them: products of bf16 or fp16 operands leave 2e-2 / 2e-3 of the result wrong, which is not
// the rounding of any output type here.  An operand is therefore kept as TWO fp16 pieces of its value times 2^10: hi = fp16(v),
// lo = fp16(v - hi), together 23 bits (|v| < 64, which cnf_api.hip's check of the coefficients guarantees; what lies below
// 2^-34 is lost, against a norm of at most 1.3).  A product is hi hi + hi lo + lo hi on the fp16 matrix pipe with fp32 sums -- the
// lo lo term is 2^-22 of it -- at a third of the pipe's 2.5 PFLOP/s instead of the 0.157 of fp32 MFMAs.  The Frobenius norm
// is summed in double from per-block partial sums added in a fixed order.
//
// A gradient far below eps makes X0 = G / eps tiny, below what pieces hold.  X is therefore s Y with a factor s per matrix and
// step: s = 1 unless |X0|_F < 1/2, then s = |X0|_F, Y = G / |G|_F, and every step takes s to min(1, s max|a + b t + c t^2|), which never lets Y grow
// before s has reached 1:   A = s^2 Y Y^T,   Y' = (s / s') (a I + b A + c A^2) Y.
//
// LAYOUT ("piece matrix").  R x K, padded with zeros to multiples of 64 and stored in blocks of 64 rows x 32 columns, 8 KB
// each, block (r / 64, k / 32) after block along k.  A row of a block is one 128-byte line: four 16-byte slots of hi, four of lo, slot s
// at s ^ (row / 2 & 7): a block copied to LDS as it lies is read as MFMA operands (a 16-byte slot of 16 rows per cycle, two rows
// to a line of the 64 banks) without bank conflicts.
// Every product is of the form C[r][c] = sum_k P[r][k] Q[c][k] with both operands contiguous along k: A = X X^T, A A (A is
// symmetric) and X' = (a I + b A + c A^2) X with Q = X^T, which the step that makes X writes beside it.  A and A^2 are symmetric: only
// tiles on and below the diagonal are computed, and written twice.
#include <cmath>
#include <type_traits>

#include "cnf_ops.h"

namespace cnf {
namespace {

constexpr int kThreads = 256;
constexpr int kNormBlocks = 512;   // at most, per matrix
constexpr float kScale = 1024.f, kInvScale = 1.f / 1024.f;
constexpr long kBlockBytes = 64 * 128;

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef float float16v __attribute__((ext_vector_type(16)));

struct Ptrs {
    const void* g[CNF_MAX_MATRICES];
    void* out[CNF_MAX_MATRICES];
    float* m[CNF_MAX_MATRICES];
};

struct Dims {
    long rows, cols, ldg, ldo, ldm;
    long m, n;      // the shorter and the longer side
    long mp, np;    // padded
    int tall;       // rows > cols: the iteration runs on the transposed matrix
};

// byte offset of element (r, c)'s hi piece in a piece matrix of kc blocks per row panel; its lo piece is at this ^ 64
__device__ __forceinline__ long piece_at(long r, long c, long kc) {
    return ((r >> 6) * kc + (c >> 5)) * kBlockBytes + ((r & 63) << 7) + ((((c >> 3) & 3) ^ ((r >> 1) & 7)) << 4) + ((c & 7) << 1);
}

__device__ __forceinline__ void split(float v, f16& hi, f16& lo) {
    hi = (f16)v;
    lo = (f16)(v - (float)hi);
}

// four neighbouring elements of a row, or the last ones of it
template <typename T, bool kVec>
__device__ __forceinline__ void load4(const T* p, long left, float (&v)[4]) {
    if (kVec) {
        struct alignas(4 * sizeof(T)) Four { T e[4]; } four = *(const Four*)p;
        for (int k = 0; k < 4; ++k) v[k] = to_f32(four.e[k]);
    } else {
        for (int k = 0; k < 4; ++k) v[k] = k < left ? to_f32(p[k]) : 0.f;
    }
}

// The matrix the iteration starts from, before normalisation: the new momentum, and the partial sums of the matrix's squares.  A
// workgroup takes every gridDim.x-th band of 1024 / cols rows (kVec: cols, strides and pointers allow four elements at a time).
template <typename T, bool kMuon, bool kVec>
__global__ __launch_bounds__(kThreads) void begin_kernel(Ptrs p, Dims d, double* part, float mu, int nesterov, const CnfStats* guard) {
    __shared__ double red[kThreads / 64];
    const int mat = blockIdx.y;
    const bool skip = guard && guard->status != 0;
    const T* g = (const T*)p.g[mat];
    const int quads = (int)((d.cols + 3) / 4);               // groups of four per row
    const int wide = quads < kThreads ? quads : kThreads;    // threads along a row
    const int band = kThreads / wide;                        // rows at a time
    const int tr = threadIdx.x / wide, tc = threadIdx.x % wide;
    double s = 0.;
    for (long r = (long)blockIdx.x * band + tr; tr < band && r < d.rows; r += (long)gridDim.x * band)
        for (int q = tc; q < quads; q += wide) {
            const long c = (long)q * 4, left = d.cols - c;
            float v[4];
            load4<T, kVec>(g + r * d.ldg + c, left, v);
            if (kMuon) {
                float* pm = p.m[mat] + r * d.ldm + c;
                float m[4];
                load4<float, kVec>(pm, left, m);
                for (int k = 0; k < 4; ++k) {
                    m[k] = fmaf(mu, m[k], v[k]);
                    v[k] = nesterov ? fmaf(mu, m[k], v[k]) : m[k];
                }
                if (!skip) {
                    if (kVec) {
                        *(float4*)pm = make_float4(m[0], m[1], m[2], m[3]);
                    } else {
                        for (int k = 0; k < 4; ++k)
                            if (k < left) pm[k] = m[k];
                    }
                }
            }
            for (int k = 0; k < 4; ++k) s = fma((double)v[k], (double)v[k], s);
        }
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) part[mat * kNormBlocks + blockIdx.x] = (red[0] + red[1]) + (red[2] + red[3]);
}

struct Steps {
    int n;
    float a[CNF_NS_MAX_STEPS], b[CNF_NS_MAX_STEPS], c[CNF_NS_MAX_STEPS];
    float grow[CNF_NS_MAX_STEPS];   // what s is multiplied by, at most to 1
};

// what the matrix is multiplied by to become Y times 2^10, and the first factor s
__device__ __forceinline__ double start_scale(double norm, double eps, float& f) {
    const bool small = norm < eps;                           // |X0| = norm / (norm + eps) < 1/2
    f = small && norm > 0. ? fmaxf((float)(norm / (norm + eps)), 1e-37f) : 1.f;   // (never 0: it divides)
    return (double)kScale * (small ? (norm > 0. ? 1. / norm : 0.) : 1. / (norm + eps));
}

// X0 = G / (|G| + eps) as the piece matrices X (m x n) and X^T (n x m); one 64 x 64 tile of G per workgroup, through LDS
template <typename T, bool kMuon>
__global__ __launch_bounds__(kThreads) void pieces_kernel(Ptrs p, Dims d, char* x, char* xt, const double* part, int parts, double eps, float mu,
                                                          int nesterov, Steps st, float* factors) {
    __shared__ float tile[64][65];
    __shared__ double scale;     // (double: the largest and smallest fp32 gradients have a scale outside fp32)
    const int mat = blockIdx.z;
    if (threadIdx.x < 64) {
        double s = 0.;
        for (int k = threadIdx.x; k < parts; k += 64) s += part[mat * kNormBlocks + k];
        for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
        if (threadIdx.x == 0) {
            float f;
            scale = start_scale(sqrt(s), eps, f);
            if (blockIdx.x == 0 && blockIdx.y == 0) {
                for (int k = 0; k < CNF_NS_MAX_STEPS; ++k) {
                    factors[mat * CNF_NS_MAX_STEPS + k] = f;
                    f = fminf(1.f, f * st.grow[k]);
                }
            }
        }
    }
    const T* g = (const T*)p.g[mat];
    const long r0 = (long)blockIdx.y * 64, c0 = (long)blockIdx.x * 64;
    __syncthreads();
    for (int e = threadIdx.x; e < 4096; e += kThreads) {
        const int i = e >> 6, j = e & 63;
        const long r = r0 + i, c = c0 + j;
        float v = 0.f;
        if (r < d.rows && c < d.cols) {
            v = to_f32(g[r * d.ldg + c]);
            if (kMuon) {
                const float mv = p.m[mat][r * d.ldm + c];     // the new momentum
                v = nesterov ? fmaf(mu, mv, v) : mv;
            }
            v = (float)((double)v * scale);
        }
        tile[i][j] = v;
    }
    __syncthreads();
    // (rows, cols) as they are, then transposed; X gets the one whose rows are the shorter side
    char* straight = (d.tall ? xt : x) + mat * d.mp * d.np * 4;
    char* flipped = (d.tall ? x : xt) + mat * d.mp * d.np * 4;
    const long kc_s = (d.tall ? d.mp : d.np) >> 5, kc_f = (d.tall ? d.np : d.mp) >> 5;
    for (int e = threadIdx.x; e < 1024; e += kThreads) {
        const int i = (e & 511) >> 3, q = (e & 7) * 8;
        half8 hi, lo;
        for (int k = 0; k < 8; ++k) {
            f16 h, l;
            split(e < 512 ? tile[i][q + k] : tile[q + k][i], h, l);
            hi[k] = h;
            lo[k] = l;
        }
        char* base = e < 512 ? straight : flipped;
        const long at = e < 512 ? piece_at(r0 + i, c0 + q, kc_s) : piece_at(c0 + i, r0 + q, kc_f);
        *(half8*)(base + at) = hi;
        *(half8*)(base + (at ^ 64)) = lo;
    }
}

constexpr int kGram = 0, kPoly = 1, kApply = 2, kFinal = 3;

struct GemmArgs {
    const char *p, *q;          // piece matrices; C[r][c] = sum_k P[r][k] Q[c][k]
    long bp, bq;                // bytes between matrices of the batch
    int kc;                     // blocks of 32 along k
    int tiles_r, tiles_c;       // tiles of C (kGram, kPoly: tiles_r x tiles_r symmetric)
    // kGram, kPoly: C to `c0` (symmetric); kApply: C to c0 and its transpose to c1
    char *c0, *c1;
    long b0, b1;
    int kc0, kc1;
    float ca, cb, cc;           // kPoly: a I + b P + c C
    long m;                     // kPoly: rows of the identity
    const float* factors;       // of this step; the next one's follow
};

struct FinalArgs : GemmArgs {   // kFinal: the iteration's result to the output matrices, or into the parameters
    Ptrs ptrs;
    long rows, cols, ldo;
    float decay, step;
    int vec;                    // out's rows can be accessed four elements at a time
    const CnfStats* guard;
};

template <int kMode>
using ArgsOf = std::conditional_t<kMode == kFinal, FinalArgs, GemmArgs>;

// four neighbouring elements of a row of the result to the output matrix, or into the parameters
template <typename O, bool kMuon>
__device__ __forceinline__ void put4(const FinalArgs& a, int mat, long r, long c, const float (&x)[4]) {
    O* o = (O*)a.ptrs.out[mat] + r * a.ldo + c;
    if (a.vec && c + 4 <= a.cols) {
        struct alignas(4 * sizeof(O)) Four { O e[4]; } four;
        if (kMuon) four = *(const Four*)o;
        for (int e = 0; e < 4; ++e) four.e[e] = from_f32<O>(kMuon ? fmaf(-a.step, x[e], a.decay * to_f32(four.e[e])) : x[e]);
        *(Four*)o = four;
    } else {
        for (int e = 0; e < 4; ++e)
            if (c + e < a.cols) o[e] = from_f32<O>(kMuon ? fmaf(-a.step, x[e], a.decay * to_f32(o[e])) : x[e]);
    }
}

using gptr = const __attribute__((address_space(1))) void*;
using lptr = __attribute__((address_space(3))) void*;

// One T x T tile of C per workgroup of four waves (2 x 2), each a (T/2) x (T/2) square of 32 x 32 MFMA tiles.  A stage is one block column (32 k) of
// both operands, copied to LDS by global_load_lds kStages - 1 stages ahead of the products.
template <int T, int kStages, int kMode, typename O = float, bool kMuon = false>
__global__ __launch_bounds__(kThreads) void gemm_kernel(ArgsOf<kMode> a) {
    constexpr int kStage = 2 * T * 128, kN = T / 64;         // bytes of a stage; 32 x 32 tiles per wave and direction
    constexpr int kLoads = kStage / 1024 / 4;                // 1 KB copies per wave and stage
    __shared__ __align__(16) char lds[kStages][kStage];
    const int mat = blockIdx.y, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    int ti, tj;
    if (kMode == kGram || kMode == kPoly) {                  // tile (ti, tj), tj <= ti, of the lower triangle
        const int id = blockIdx.x;
        ti = (int)((sqrtf(8.f * (float)id + 1.f) - 1.f) * 0.5f);
        while ((ti + 1) * (ti + 2) / 2 <= id) ++ti;
        while (ti * (ti + 1) / 2 > id) --ti;
        tj = id - ti * (ti + 1) / 2;
    } else {
        ti = blockIdx.x % a.tiles_r;
        tj = blockIdx.x / a.tiles_r;
    }
    const char* src[kLoads];
    for (int i = 0; i < kLoads; ++i) {
        const int kb = wave * kLoads + i;                    // which KB of the stage: T / 8 of them are P's
        const int row = (kb % (T / 8)) * 8;                  // first of its eight rows
        const bool is_p = kb < T / 8;
        const long panel = (long)(is_p ? ti : tj) * (T / 64) + (row >> 6);
        src[i] = (is_p ? a.p + mat * a.bp : a.q + mat * a.bq) + panel * a.kc * kBlockBytes + (row & 63) * 128 + lane * 16;
    }
    auto load = [&](int stage, int k) {
        for (int i = 0; i < kLoads; ++i)
            __builtin_amdgcn_global_load_lds((gptr)(src[i] + k * kBlockBytes), (lptr)(&lds[stage][(wave * kLoads + i) * 1024]), 16, 0, 0);
    };
    const int wr = (wave >> 1) * (T / 2), wc = (wave & 1) * (T / 2);
    const int slot = ((lane >> 5) ^ ((lane >> 1) & 7)) << 4, line = (lane & 31) << 7;
    float16v acc[kN][kN] = {};
    for (int k = 0; k < kStages - 1 && k < a.kc; ++k) load(k, k);
    for (int k = 0; k < a.kc; ++k) {
        // this stage has landed (the kStages - 2 after it may be on their way), and every wave's reads of the one before are done
        if (k + kStages - 1 <= a.kc)
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((kStages - 2) * kLoads) : "memory");
        else
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (k + kStages - 1 < a.kc) load((k + kStages - 1) % kStages, k + kStages - 1);
        const char* st = lds[k % kStages] + line;
#pragma unroll
        for (int kh = 0; kh < 2; ++kh) {
            half8 ph[kN], pl[kN], qh[kN], ql[kN];
            for (int u = 0; u < kN; ++u) {
                const char* pr = st + (wr + u * 32) * 128;
                const char* qr = st + (T + wc + u * 32) * 128;
                ph[u] = *(const half8*)(pr + (slot ^ (kh << 5)));
                pl[u] = *(const half8*)(pr + (slot ^ (kh << 5) ^ 64));
                qh[u] = *(const half8*)(qr + (slot ^ (kh << 5)));
                ql[u] = *(const half8*)(qr + (slot ^ (kh << 5) ^ 64));
            }
            for (int u = 0; u < kN; ++u)
                for (int v = 0; v < kN; ++v) {               // operands exchanged: a lane holds four neighbouring columns of a row of C
                    acc[u][v] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ql[v], ph[u], acc[u][v], 0, 0, 0);
                    acc[u][v] = __builtin_amdgcn_mfma_f32_32x32x16_f16(qh[v], pl[u], acc[u][v], 0, 0, 0);
                    acc[u][v] = __builtin_amdgcn_mfma_f32_32x32x16_f16(qh[v], ph[u], acc[u][v], 0, 0, 0);
                }
        }
    }
    if constexpr (kMode == kFinal) {
        if (a.guard && a.guard->status != 0) return;
    }
    float scale = kInvScale;                                 // from the accumulator to C times 2^10
    if (kMode != kPoly) {
        const float f = a.factors[mat * CNF_NS_MAX_STEPS];
        scale *= kMode == kGram ? f * f : kMode == kApply ? f / a.factors[mat * CNF_NS_MAX_STEPS + 1] : f * kInvScale;
    }
    for (int u = 0; u < kN; ++u)
        for (int v = 0; v < kN; ++v)
            for (int g = 0; g < 4; ++g) {
                const long r = (long)ti * T + wr + u * 32 + (lane & 31), c = (long)tj * T + wc + v * 32 + g * 8 + (lane >> 5) * 4;
                float val[4];
                for (int e = 0; e < 4; ++e) val[e] = acc[u][v][g * 4 + e] * scale;
                if constexpr (kMode == kFinal) {
                    if (r < a.rows) put4<O, kMuon>(a, mat, r, c, val);
                } else {
                const long at = piece_at(r, c, a.kc0);
                if (kMode == kPoly) {
                    const char* pm = a.p + mat * a.bp;
                    const half4 h = *(const half4*)(pm + at), l = *(const half4*)(pm + (at ^ 64));
                    for (int e = 0; e < 4; ++e) {
                        val[e] = fmaf(a.cc, val[e], a.cb * ((float)h[e] + (float)l[e]));
                        if (r == c + e && r < a.m) val[e] += a.ca * kScale;
                    }
                }
                half4 hi, lo;
                for (int e = 0; e < 4; ++e) {
                    f16 h, l;
                    split(val[e], h, l);
                    hi[e] = h;
                    lo[e] = l;
                }
                char* c0 = a.c0 + mat * a.b0;
                *(half4*)(c0 + at) = hi;
                *(half4*)(c0 + (at ^ 64)) = lo;
                if (kMode == kApply || ti != tj) {
                    char* ct = kMode == kApply ? a.c1 + mat * a.b1 : c0;
                    for (int e = 0; e < 4; ++e) {
                        const long t = piece_at(c + e, r, kMode == kApply ? a.kc1 : a.kc0);
                        *(f16*)(ct + t) = hi[e];
                        *(f16*)(ct + (t ^ 64)) = lo[e];
                    }
                }
                }
            }
}

// Matrices of at most 64 x 64: one workgroup per matrix does the whole update, with X, X^T, A and a I + b A + c A^2 as piece matrices in LDS
// (two blocks of 8 KB each).  A wave computes one 32 x 32 quadrant of every product.  What bounds it is the chain: 3 products per
// step, each a barrier, its operands' LDS reads, 12 dependent MFMAs and the split of its result.
template <typename O, bool kMuon>
__global__ __launch_bounds__(kThreads) void small_kernel(FinalArgs a, Dims d, Steps st, double eps, float mu, int nesterov) {
    __shared__ __align__(16) char xs[2 * kBlockBytes], xts[2 * kBlockBytes], as[2 * kBlockBytes], bs[2 * kBlockBytes];
    __shared__ double red[kThreads / 64];
    const int mat = blockIdx.x, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const bool skip = a.guard && a.guard->status != 0;
    const O* g = (const O*)a.ptrs.g[mat];
    // the matrix: thread (tr, tc) holds four rows of four columns (what lies outside is read at the last element and not used)
    const int tr = threadIdx.x >> 4, tc = (threadIdx.x & 15) * 4;
    float v[4][4], old[4][4];
    for (int i = 0; i < 4; ++i)
        for (int k = 0; k < 4; ++k) {
            const int r = min(tr * 4 + i, (int)a.rows - 1), c = min(tc + k, (int)a.cols - 1);
            v[i][k] = to_f32(g[r * d.ldg + c]);
            if (kMuon) old[i][k] = a.ptrs.m[mat][r * d.ldm + c];
        }
    double s = 0.;
    for (int i = 0; i < 4; ++i)
        for (int k = 0; k < 4; ++k) {
            const int r = tr * 4 + i, c = tc + k;
            const bool in = r < a.rows && c < a.cols;
            if (kMuon) {
                const float mv = fmaf(mu, old[i][k], v[i][k]);
                if (in && !skip) a.ptrs.m[mat][r * d.ldm + c] = mv;
                v[i][k] = nesterov ? fmaf(mu, mv, v[i][k]) : mv;
            }
            if (!in) v[i][k] = 0.f;
            s = fma((double)v[i][k], (double)v[i][k], s);
        }
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
    if (lane == 0) red[wave] = s;
    __syncthreads();
    float f;
    const double scale = start_scale(sqrt((red[0] + red[1]) + (red[2] + red[3])), eps, f);
    char *straight = d.tall ? xts : xs, *flipped = d.tall ? xs : xts;
    for (int i = 0; i < 4; ++i)
        for (int k = 0; k < 4; ++k) v[i][k] = (float)((double)v[i][k] * scale);
    for (int i = 0; i < 4; ++i) {
        half4 h, l, ht, lt;
        for (int k = 0; k < 4; ++k) {
            f16 hi, lo;
            split(v[i][k], hi, lo);
            h[k] = hi, l[k] = lo;
            split(v[k][i], hi, lo);
            ht[k] = hi, lt[k] = lo;
        }
        const long at = piece_at(tr * 4 + i, tc, 2), att = piece_at(tc + i, tr * 4, 2);
        *(half4*)(straight + at) = h;
        *(half4*)(straight + (at ^ 64)) = l;
        *(half4*)(flipped + att) = ht;
        *(half4*)(flipped + (att ^ 64)) = lt;
    }
    const int wr = (wave >> 1) * 32, wc = (wave & 1) * 32;
    const int slot = ((lane >> 5) ^ ((lane >> 1) & 7)) << 4, line = (lane & 31) << 7;
    // quadrant (pr, qr) of sum_k P[r][k] Q[c][k]: a lane holds columns 8 g + 4 (lane / 32) + e of row lane % 32
    auto multiply = [&](const char* p, int pr, const char* q, int qr) {
        float16v acc = {};
#pragma unroll
        for (int kb = 0; kb < 4; ++kb) {
            const char *pp = p + (kb >> 1) * kBlockBytes + pr * 128 + line, *qq = q + (kb >> 1) * kBlockBytes + qr * 128 + line;
            const int so = slot ^ ((kb & 1) << 5);
            const half8 ph = *(const half8*)(pp + so), pl = *(const half8*)(pp + (so ^ 64));
            const half8 qh = *(const half8*)(qq + so), ql = *(const half8*)(qq + (so ^ 64));
            acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(ql, ph, acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(qh, pl, acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(qh, ph, acc, 0, 0, 0);
        }
        return acc;
    };
    const int row = wr + (lane & 31), col = wc + (lane >> 5) * 4;
    auto store = [&](char* to, char* flip, const float16v& x) {      // pieces of the quadrant, and of its transpose where flip is given
        for (int q = 0; q < 4; ++q) {
            half4 h, l;
            for (int e = 0; e < 4; ++e) {
                f16 hi, lo;
                split(x[q * 4 + e], hi, lo);
                h[e] = hi, l[e] = lo;
            }
            const long at = piece_at(row, col + q * 8, 2);
            *(half4*)(to + at) = h;
            *(half4*)(to + (at ^ 64)) = l;
            if (flip)
                for (int e = 0; e < 4; ++e) {
                    const long t = piece_at(col + q * 8 + e, row, 2);
                    *(f16*)(flip + t) = h[e];
                    *(f16*)(flip + (t ^ 64)) = l[e];
                }
        }
    };
    for (int k = 0; k < st.n; ++k) {
        __syncthreads();
        float16v A = multiply(xs, wr, xs, wc);
        for (int i = 0; i < 16; ++i) A[i] *= kInvScale * f * f;
        store(as, nullptr, A);
        __syncthreads();
        float16v B = multiply(as, wr, as, wc);
        const float diag = row < d.m ? st.a[k] * kScale : 0.f;
        for (int i = 0; i < 16; ++i) {
            B[i] = fmaf(st.c[k] * kInvScale, B[i], st.b[k] * A[i]);
            B[i] += row == col + (i >> 2) * 8 + (i & 3) ? diag : 0.f;
        }
        store(bs, nullptr, B);
        __syncthreads();
        if (k + 1 < st.n) {
            float16v X = multiply(bs, wr, xts, wc);
            const float f1 = fminf(1.f, f * st.grow[k]);
            for (int i = 0; i < 16; ++i) X[i] *= kInvScale * (f / f1);
            f = f1;
            __syncthreads();                                 // everybody has read X^T
            store(xs, xts, X);
        }
    }
    if (skip) return;
    const float16v X = d.tall ? multiply(xts, wr, bs, wc) : multiply(bs, wr, xts, wc);
    if (row >= a.rows) return;
    for (int q = 0; q < 4; ++q) {
        float val[4];
        for (int e = 0; e < 4; ++e) val[e] = X[q * 4 + e] * (kInvScale * kInvScale * f);
        if (col + q * 8 < a.cols) put4<O, kMuon>(a, mat, row, col + q * 8, val);
    }
}

long pad_to(long v, long t) { return (v + t - 1) / t * t; }

// The tile of a product of `tiles` 128 x 128 tiles: 128 reads its operands half as often, 64 has four times the workgroups.
bool wide_tiles(long tiles) { return tiles >= 128; }

struct Plan {
    long m, n, mp, np;
    bool wide_sym, wide_full;
    bool small;     // one workgroup per matrix does everything in LDS
};

Plan plan_of(long count, long rows, long cols) {
    Plan p{};
    p.m = rows < cols ? rows : cols;
    p.n = rows < cols ? cols : rows;
    p.small = p.n <= 64;
    const long t = pad_to(p.m, 128) / 128, u = pad_to(p.n, 128) / 128;
    p.wide_sym = wide_tiles(t * (t + 1) / 2 * count);
    p.wide_full = wide_tiles(t * u * count);
    const long to = p.wide_sym || p.wide_full ? 128 : 64;
    p.mp = pad_to(p.m, to);
    p.np = pad_to(p.n, to);
    return p;
}

template <int kMode, typename O = float, bool kMuon = false>
void product(bool wide, const FinalArgs& args, const Plan& p, bool transposed, int count, hipStream_t s) {
    FinalArgs g = args;
    const int t = wide ? 128 : 64, tm = (int)(p.mp / t), tn = (int)(p.np / t);
    const bool sym = kMode == kGram || kMode == kPoly;
    g.tiles_r = transposed ? tn : tm;
    g.tiles_c = sym ? tm : transposed ? tm : tn;
    const dim3 grid(sym ? tm * (tm + 1) / 2 : tm * tn, count);
    // at most one workgroup per CU: 128 KB of stages in flight each, else 64 KB and two workgroups
    const bool deep = (long)grid.x * grid.y <= 256;
    if (wide && deep)
        gemm_kernel<128, 4, kMode, O, kMuon><<<grid, kThreads, 0, s>>>(g);
    else if (wide)
        gemm_kernel<128, 2, kMode, O, kMuon><<<grid, kThreads, 0, s>>>(g);
    else if (deep)
        gemm_kernel<64, 8, kMode, O, kMuon><<<grid, kThreads, 0, s>>>(g);
    else
        gemm_kernel<64, 4, kMode, O, kMuon><<<grid, kThreads, 0, s>>>(g);
}

template <typename O, bool kMuon>
hipError_t run(const MuonArgs& a, hipStream_t s) {
    double grow[CNF_NS_MAX_STEPS];
    if (ns_bounds(*a.ns, grow)) return hipErrorInvalidValue;
    Steps st{};
    st.n = a.ns->steps;
    for (int k = 0; k < st.n; ++k) {
        st.a[k] = (float)a.ns->a[k];
        st.b[k] = (float)a.ns->b[k];
        st.c[k] = (float)a.ns->c[k];
        st.grow[k] = (float)fmax(1., grow[k]);
    }
    const Plan pl = plan_of(a.count, a.rows, a.cols);
    Ptrs p{};
    bool vec_in = a.cols % 4 == 0 && a.ldg % 4 == 0 && (!kMuon || a.ldm % 4 == 0), vec_out = a.ldo % 4 == 0;
    for (int i = 0; i < a.count; ++i) {
        p.g[i] = a.g[i];
        p.out[i] = a.out[i];
        p.m[i] = kMuon ? a.momenta[i] : nullptr;
        vec_in = vec_in && (uintptr_t)p.g[i] % (4 * sizeof(O)) == 0 && (uintptr_t)p.m[i] % 16 == 0;
        vec_out = vec_out && (uintptr_t)p.out[i] % (4 * sizeof(O)) == 0;
    }
    Dims d{};
    d.rows = a.rows, d.cols = a.cols, d.ldg = a.ldg, d.ldo = a.ldo, d.ldm = a.ldm;
    d.tall = a.rows > a.cols;
    d.m = pl.m, d.n = pl.n, d.mp = pl.mp, d.np = pl.np;
    const float mu = kMuon ? (float)a.opts->momentum : 0.f;
    const int nesterov = kMuon ? a.opts->nesterov : 0;
    FinalArgs g{};
    g.ptrs = p, g.rows = d.rows, g.cols = d.cols, g.ldo = d.ldo, g.guard = a.guard;
    g.decay = kMuon ? (float)(1.0 - a.opts->lr * a.opts->weight_decay) : 1.f;
    g.step = kMuon ? (float)(a.opts->lr * a.opts->scale) : 1.f;
    g.vec = vec_out;
    if (pl.small) {
        small_kernel<O, kMuon><<<dim3(a.count), kThreads, 0, s>>>(g, d, st, a.ns->eps, mu, nesterov);
        return hipGetLastError();
    }
    const long xb = d.mp * d.np * 4, ab = d.mp * d.mp * 4;
    double* part = (double*)a.ws;
    char *x = (char*)(part + (size_t)a.count * kNormBlocks), *xt = x + a.count * xb, *xt2 = xt + a.count * xb, *A = xt2 + a.count * xb,
         *B = A + a.count * ab;
    float* factors = (float*)(B + a.count * ab);
    // partial sums: enough workgroups for the device, at least 2 K elements each
    long parts = (d.rows * d.cols + 2047) / 2048, most = (2048 + a.count - 1) / a.count;
    most = most < kNormBlocks ? most : kNormBlocks;
    parts = parts < most ? parts : most;
    const dim3 grid_in((unsigned)parts, a.count);
    if (vec_in)
        begin_kernel<O, kMuon, true><<<grid_in, kThreads, 0, s>>>(p, d, part, mu, nesterov, a.guard);
    else
        begin_kernel<O, kMuon, false><<<grid_in, kThreads, 0, s>>>(p, d, part, mu, nesterov, a.guard);
    const long rp = d.tall ? d.np : d.mp, cp = d.tall ? d.mp : d.np;
    pieces_kernel<O, kMuon><<<dim3((unsigned)(cp / 64), (unsigned)(rp / 64), a.count), kThreads, 0, s>>>(p, d, x, xt, part, (int)parts, a.ns->eps,
                                                                                                         mu, nesterov, st, factors);
    const int km = (int)(d.mp / 32), kn = (int)(d.np / 32);
    for (int k = 0; k < st.n; ++k) {
        g.factors = factors + k;
        g.p = g.q = x, g.bp = g.bq = xb, g.kc = kn;
        g.c0 = A, g.b0 = ab, g.kc0 = km;
        product<kGram>(pl.wide_sym, g, pl, false, a.count, s);
        g.p = g.q = A, g.bp = g.bq = ab, g.kc = km;
        g.c0 = B;
        g.ca = st.a[k], g.cb = st.b[k], g.cc = st.c[k], g.m = d.m;
        product<kPoly>(pl.wide_sym, g, pl, false, a.count, s);
        g.p = B, g.bp = ab, g.q = xt, g.bq = xb;
        if (k + 1 < st.n) {
            g.c0 = x, g.b0 = xb, g.kc0 = kn;
            g.c1 = xt2, g.b1 = xb, g.kc1 = km;
            product<kApply>(pl.wide_full, g, pl, false, a.count, s);
            char* t = xt;
            xt = xt2;
            xt2 = t;
            continue;
        }
        if (d.tall) g.p = xt, g.bp = xb, g.q = B, g.bq = ab;   // the output's rows are X^T's
        product<kFinal, O, kMuon>(pl.wide_full, g, pl, d.tall, a.count, s);
    }
    return hipGetLastError();
}

template <typename O>
hipError_t run_op(const MuonArgs& a, hipStream_t s) {
    return a.opts ? run<O, true>(a, s) : run<O, false>(a, s);
}

}  // namespace

// The largest |f| on [0, s] of f(u) = a u + b u^3 + c u^5: at the ends or where f' = a + 3 b u^2 + 5 c u^4 vanishes.
static double quintic_max(double a, double b, double c, double s) {
    auto f = [&](double u) { return std::fabs(u * (a + u * u * (b + u * u * c))); };
    double best = f(s);
    double roots[2] = {-1., -1.};
    const double A = 5. * c, B = 3. * b, D = B * B - 4. * A * a;
    if (A != 0. && D >= 0.) {
        roots[0] = (-B + std::sqrt(D)) / (2. * A);
        roots[1] = (-B - std::sqrt(D)) / (2. * A);
    } else if (A == 0. && B != 0.) {
        roots[0] = -a / B;
    }
    for (double r : roots)
        if (r > 0. && std::sqrt(r) < s) best = std::fmax(best, f(std::sqrt(r)));
    return best;
}

int ns_bounds(const CnfNewtonSchulz& ns, double (&grow)[CNF_NS_MAX_STEPS]) {
    double s = 1.;   // bound of |X|; A = X X^T (<= s^2) and a I + b A + c A^2 have to stay within the pieces' 64
    for (int k = 0; k < ns.steps; ++k) {
        const double a = ns.a[k], b = ns.b[k], c = ns.c[k], t = s * s;
        double h = std::fmax(std::fabs(a), std::fabs(a + b * t + c * t * t));
        if (c != 0. && -b / (2. * c) > 0. && -b / (2. * c) < t) h = std::fmax(h, std::fabs(a - b * b / (4. * c)));
        grow[k] = h;
        s = quintic_max(a, b, c, s);
        if (!(h < 60.) || !(s <= 7.5)) return k + 1;
        s = std::fmax(s * 1.0001, 1e-3);
    }
    return 0;
}

size_t muon_workspace_bytes(long count, long rows, long cols) {
    const Plan p = plan_of(count, rows, cols);
    const size_t m = p.mp, n = p.np;
    if (p.small) return 256;   // (uses none; 0 stands for a call that is not supported)
    return (size_t)count * (kNormBlocks * sizeof(double) + (3 * m * n + 2 * m * m) * 4 + CNF_NS_MAX_STEPS * sizeof(float));
}

hipError_t launch_muon(int dtype, const MuonArgs& a, hipStream_t s) {
    if (dtype == CNF_F32) return run_op<float>(a, s);
    if (dtype == CNF_F16) return run_op<f16>(a, s);
    if (dtype == CNF_BF16) return run_op<bf16>(a, s);
    return hipErrorInvalidValue;
}

}  // namespace cnf
