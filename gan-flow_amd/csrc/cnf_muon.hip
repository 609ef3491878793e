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
// before s has reached 1:   A = s^2 Y Y^T,   Y' = (s / s') (a I + b A + c A^2) Y.  (A 16-bit matrix starts with s in [1/2, 1]: power_of_two.)
//
// LAYOUT ("piece matrix").  R x K, padded with zeros to multiples of 64 and stored in blocks of 64 rows x 32 columns, 8 KB
// each, block (r / 64, k / 32) after block along k.  A block is eight fragments of 1 KB -- by 16 columns, 32 rows, piece (hi, lo) -- and a
// fragment is one operand of a 32 x 32 x 16 MFMA as its 64 lanes take it: row l % 32, columns 8 (l / 32) .. + 7 at 16 l.  So an operand is one
// access of a whole kilobyte, from memory, into LDS and out of it without bank conflicts.
// Every product is of the form C[r][c] = sum_k P[r][k] Q[c][k] with both operands contiguous along k: A = X X^T, A A (A is
// symmetric) and X' = (a I + b A + c A^2) X with Q = X^T, which the step that makes X writes beside it.  A and A^2 are symmetric: only
// tiles on and below the diagonal are computed, and written twice.
#include <cmath>
#include <type_traits>
#include <utility>

#include "cnf_ops.h"

namespace cnf {
namespace {

constexpr int kThreads = 256;
constexpr long kCus = 256;
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

// byte offset of element (r, c)'s hi piece in a piece matrix of kc blocks per row panel; its lo piece is kLo behind
constexpr int kLo = 1024;
__device__ __forceinline__ long piece_at(long r, long c, long kc) {
    return ((r >> 6) * kc + (c >> 5)) * kBlockBytes + ((c >> 4 & 1) << 12) + ((r >> 5 & 1) << 11) + ((c >> 3 & 1) << 9) + ((r & 31) << 4) + ((c & 7) << 1);
}

// The pieces of two values.  The values are settled before they are split: the compiler otherwise folds the operation that makes one into one
// of its conversions (fp32 arithmetic with an fp16 result, rounded once), and a hi from the unrounded value beside a lo from the
// rounded one is a whole fp16 step off where the two round differently.
typedef float float2v __attribute__((ext_vector_type(2)));
typedef _Float16 half2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ void split2(float v0, float v1, half2& hi, half2& lo) {
    asm("" : "+v"(v0), "+v"(v1));
    hi = __builtin_convertvector((float2v){v0, v1}, half2);
    // v - hi is exact; as a multiply-add it reads hi's halves without converting them first
    lo = __builtin_convertvector((float2v){__builtin_fmaf(-1.f, (float)hi[0], v0), __builtin_fmaf(-1.f, (float)hi[1], v1)}, half2);
}

__device__ __forceinline__ void split4(const float (&v)[4], half4& hi, half4& lo) {
    half2 h0, l0, h1, l1;
    split2(v[0], v[1], h0, l0);
    split2(v[2], v[3], h1, l1);
    hi = __builtin_shufflevector(h0, h1, 0, 1, 2, 3);
    lo = __builtin_shufflevector(l0, l1, 0, 1, 2, 3);
}

__device__ __forceinline__ void split8(const float (&v)[8], half8& hi, half8& lo) {
    half4 h0, l0, h1, l1;
    split4({v[0], v[1], v[2], v[3]}, h0, l0);
    split4({v[4], v[5], v[6], v[7]}, h1, l1);
    hi = __builtin_shufflevector(h0, h1, 0, 1, 2, 3, 4, 5, 6, 7);
    lo = __builtin_shufflevector(l0, l1, 0, 1, 2, 3, 4, 5, 6, 7);
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

// A 16-bit matrix scaled by a power of two has no low pieces (but for what lies below 2^-34), and its first products are fewer by as
// much: the rest of the scale, at least 1/2, goes to s (4096 x 4096: 3360 us against 3525).  Not in Muon, where what is iterated is made of
// the fp32 momentum.
template <typename T, bool kMuon>
constexpr bool kHighPieces = !kMuon && sizeof(T) == 2;

__device__ __forceinline__ double power_of_two(double scale, float& f) {
    if (scale == 0.) return scale;
    int e;
    const double rest = frexp(scale, &e);                    // 1/2 <= rest < 1
    f = fmaxf((float)(f * rest), 1e-37f);
    return ldexp(1., e);
}

// s before every step
__device__ __forceinline__ void put_factors(float* to, float f, const Steps& st) {
    for (int k = 0; k <= CNF_NS_MAX_STEPS; ++k) {
        to[k] = f;
        if (k < st.n) f = fminf(1.f, f * st.grow[k]);
    }
}

// four neighbouring elements of X0 times 2^10: zeros outside G (what is outside is read at its last row and not used)
template <typename T, bool kMuon, bool kVec>
__device__ __forceinline__ void start_values(const Ptrs& p, const Dims& d, int mat, long row, long c, float mu, int nesterov, double scale, float (&v)[4]) {
    const long r = min(row, d.rows - 1), left = d.cols - c;  // columns from here on
    float m[4] = {};
    for (int k = 0; k < 4; ++k) v[k] = 0.f;
    if (left > 0) {
        load4<T, kVec>((const T*)p.g[mat] + r * d.ldg + c, left, v);
        if (kMuon) load4<float, kVec>(p.m[mat] + r * d.ldm + c, left, m);        // the new momentum
    }
    for (int k = 0; k < 4; ++k) {
        const float u = kMuon ? (nesterov ? fmaf(mu, m[k], v[k]) : m[k]) : v[k];
        v[k] = row < d.rows ? (float)((double)u * scale) : 0.f;
    }
}

// X0 = G / (|G| + eps) as the piece matrices X (m x n) and X^T (n x m); one 64 x 64 tile of G per workgroup, through LDS.  Thread (tr, tc)
// loads columns 4 tc .. of rows tr, tr + 16, ..; what is outside G is read at its last row and not used.
template <typename T, bool kMuon, bool kVec>
__global__ __launch_bounds__(kThreads) void pieces_kernel(Ptrs p, Dims d, char* x, char* xt, const double* part, int parts, double eps, float mu,
                                                          int nesterov, Steps st, float* factors) {
    __shared__ float tile[64][68];
    __shared__ double red[kThreads / 64];
    const int mat = blockIdx.z, tr = threadIdx.x >> 4, tc = (threadIdx.x & 15) * 4;
    const T* g = (const T*)p.g[mat];
    const long r0 = (long)blockIdx.y * 64, c0 = (long)blockIdx.x * 64, c = c0 + tc;
    const long left = d.cols - c;                            // columns from here on
    float v[4][4], m[4][4];
    for (int i = 0; i < 4; ++i) {
        const long r = min(r0 + tr + i * 16, d.rows - 1);
        for (int k = 0; k < 4; ++k) v[i][k] = m[i][k] = 0.f;
        if (left > 0) {
            load4<T, kVec>(g + r * d.ldg + c, left, v[i]);
            if (kMuon) load4<float, kVec>(p.m[mat] + r * d.ldm + c, left, m[i]);      // the new momentum
        }
    }
    double s = 0.;
    for (int k = threadIdx.x; k < parts; k += kThreads) s += part[mat * kNormBlocks + k];
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    float f;
    // (double: the largest and smallest fp32 gradients have a scale outside fp32)
    double scale = start_scale(sqrt((red[0] + red[1]) + (red[2] + red[3])), eps, f);
    if (kHighPieces<T, kMuon>) scale = power_of_two(scale, f);
    if (threadIdx.x == 0 && blockIdx.x == 0 && blockIdx.y == 0)
        put_factors(factors + mat * (CNF_NS_MAX_STEPS + 1), f, st);
    for (int i = 0; i < 4; ++i) {
        const bool in = r0 + tr + i * 16 < d.rows;
        for (int k = 0; k < 4; ++k) {
            const float u = kMuon ? (nesterov ? fmaf(mu, m[i][k], v[i][k]) : m[i][k]) : v[i][k];
            v[i][k] = in ? (float)((double)u * scale) : 0.f;
        }
        *(float4*)&tile[tr + i * 16][tc] = make_float4(v[i][0], v[i][1], v[i][2], v[i][3]);
    }
    __syncthreads();
    // (rows, cols) as they are, then transposed; X gets the one whose rows are the shorter side
    char* straight = (d.tall ? xt : x) + mat * d.mp * d.np * 4;
    char* flipped = (d.tall ? x : xt) + mat * d.mp * d.np * 4;
    const long kc_s = (d.tall ? d.mp : d.np) >> 5, kc_f = (d.tall ? d.np : d.mp) >> 5;
    for (int e = threadIdx.x; e < 1024; e += kThreads) {
        const int i = e & 63, q = (e >> 6 & 7) * 8;
        float w[8];
        for (int k = 0; k < 8; ++k) w[k] = e < 512 ? tile[i][q + k] : tile[q + k][i];
        half8 h, l;
        split8(w, h, l);
        char* base = e < 512 ? straight : flipped;
        const long at = e < 512 ? piece_at(r0 + i, c0 + q, kc_s) : piece_at(c0 + i, r0 + q, kc_f);
        *(half8*)(base + at) = h;
        *(half8*)(base + at + kLo) = l;
    }
}

constexpr int kGram = 0, kPoly = 1, kSym = 2, kApply = 3, kFinal = 4;

struct GemmArgs {
    const char *p, *q;          // piece matrices; C[r][c] = sum_k P[r][k] Q[c][k]
    long bp, bq;                // bytes between matrices of the batch
    int kc;                     // blocks of 32 along k (even)
    int panels_p, panels_q;     // panels of 64 rows of P and Q
    // kGram, kPoly, kSym: C to `c0` (symmetric); kApply: C to c0 and its transpose to c1
    char *c0, *c1;
    long b0, b1;
    float ca, cb, cc;           // kPoly: a I + b P + c C
    long m;                     // kPoly: rows of the identity
    const float* factors;       // kGram, kApply, kFinal: s at this step; `ahead` further on: after the steps the product stands for
    int ahead;
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
template <int kMode>
constexpr bool kSymmetric = kMode == kGram || kMode == kPoly || kMode == kSym;

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

constexpr int kSchedMfma = 0x8, kSchedVmem = 0x10, kSchedLdsRead = 0x100;   // classes of __builtin_amdgcn_sched_group_barrier

using gptr = const __attribute__((address_space(1))) void*;
using lptr = __attribute__((address_space(3))) void*;

// Which tile a workgroup computes.  Consecutive workgroups go to the eight XCDs in turn, each with an L2 of its own: an XCD gets
// a contiguous run of the tiles -- matrix after matrix, each in bands of eight tile rows, a band column after column -- so that the
// workgroups that share an L2 share operand panels.  With tiles dealt out in turn instead every L2 streams nearly all of X, and the fabric
// behind the L2s bounds the products (Muon 8 x (1024 x 512): 26 against 19 us a Gram product); so it does where the lower triangle is
// taken row after row (4096 x 4096: 345 against 235 us).
__device__ __forceinline__ int triangle_row(int id) {        // the row of element `id` of a lower triangle stored row after row
    int r = (int)((sqrtf(8.f * (float)id + 1.f) - 1.f) * 0.5f);
    while ((r + 1) * (r + 2) / 2 <= id) ++r;
    while (r * (r + 1) / 2 > id) --r;
    return r;
}

__device__ __forceinline__ void my_tile(int tiles_r, int tiles_c, bool sym, int& mat, int& ti, int& tj) {
    constexpr int kBand = 8;
    const int total = gridDim.x, q = total >> 3, rem = total & 7, xcd = blockIdx.x & 7, nth = blockIdx.x >> 3;
    int id = xcd * q + (xcd < rem ? xcd : rem) + nth;
    const int per = sym ? tiles_r * (tiles_r + 1) / 2 : tiles_r * tiles_c;
    mat = id / per;
    id -= mat * per;
    if (sym) {                                               // tj <= ti: a band's columns before its diagonal, then the triangle on it
        const int first = triangle_row(id) / kBand * kBand, high = min(kBand, tiles_r - first);
        id -= first * (first + 1) / 2;
        if (id < first * high) {
            ti = first + id % high;
            tj = id / high;
        } else {
            id -= first * high;
            ti = triangle_row(id);
            tj = first + id - ti * (ti + 1) / 2;
            ti += first;
        }
    } else {
        const int band = id / (kBand * tiles_c), first = band * kBand, high = min(kBand, tiles_r - first);
        id -= first * tiles_c;
        ti = first + id % high;
        tj = id / high;
    }
}

// Operands of the products of 16 k: kNu x kNv tiles of 32 x 32.  kTerms: 3 products of pieces, or 2 where Q has no low pieces, or 1 where P has none either
template <int kNu, int kNv, int kTerms>
struct Frag {
    static constexpr int kReads = (kTerms > 1 ? 2 : 1) * kNu + (kTerms > 2 ? 2 : 1) * kNv;
    half8 ph[kNu], pl[kNu], qh[kNv], ql[kNv];
    // p, q: the first of the wave's fragments of either operand, in LDS or in memory
    __device__ __forceinline__ void read(const char* p, const char* q, int lane) {
        for (int v = 0; v < kNv; ++v) {
            if (kTerms > 2) ql[v] = *(const half8*)(q + v * 2048 + kLo + lane * 16);
            qh[v] = *(const half8*)(q + v * 2048 + lane * 16);
        }
        for (int u = 0; u < kNu; ++u) {
            ph[u] = *(const half8*)(p + u * 2048 + lane * 16);
            if (kTerms > 1) pl[u] = *(const half8*)(p + u * 2048 + kLo + lane * 16);
        }
    }
    // operands exchanged: a lane gets four neighbouring columns of a row of C
    __device__ __forceinline__ void multiply(float16v (&acc)[kNu][kNv]) const {
        for (int j = 3 - kTerms; j < 3; ++j)                          // lo hi, hi lo, hi hi: the three on one tile as far apart as they can be
            for (int u = 0; u < kNu; ++u)
                for (int v = 0; v < kNv; ++v)
                    acc[u][v] = __builtin_amdgcn_mfma_f32_32x32x16_f16(j == 0 ? ql[v] : qh[v], j == 1 ? pl[u] : ph[u], acc[u][v], 0, 0, 0);
    }
};

// What happens to a 32 x 32 tile of C whose first element is (r0, c0): lane l holds columns 8 g + 4 (l / 32) + e (register 4 g + e) of
// row l % 32.  It goes through LDS (4.6 KB a wave, hi and lo of an element in a word), and its fragments and those of its transpose
// are stored a whole kilobyte at a time; stored from where the products leave it, it would go out in pieces of 8 bytes
// (a 256 x 256 tile of X and X^T in pieces of 16: 14 us).
constexpr int kFlipBytes = 32 * 36 * 4;

template <int kMode, typename O, bool kMuon>
__device__ __forceinline__ void finish(const ArgsOf<kMode>& a, int mat, float scale, const float16v& acc, long r0, long c0, bool flip, int lane,
                                       char* lds) {
    if (r0 >= (long)a.panels_p * 64 || c0 >= (long)a.panels_q * 64) return;     // (a tile larger than 64 can reach past the end)
    const int row = lane & 31, half = lane >> 5;
    // (a wave's LDS operations are executed in order: reads see the writes before them, and writes come after the reads before them)
    if constexpr (kMode == kFinal) {
        float* t = (float*)lds;
        for (int g = 0; g < 4; ++g)
            *(float4*)(t + row * 36 + g * 8 + half * 4) = make_float4(acc[g * 4] * scale, acc[g * 4 + 1] * scale, acc[g * 4 + 2] * scale, acc[g * 4 + 3] * scale);
        for (int i = 0; i < 4; ++i) {                        // stored eight rows of 32 columns at a time
            const long r = r0 + i * 8 + (lane >> 3), c = c0 + (lane & 7) * 4;
            const float4 x = *(const float4*)(t + (i * 8 + (lane >> 3)) * 36 + (lane & 7) * 4);
            const float val[4] = {x.x, x.y, x.z, x.w};
            if (r < a.rows && c < a.cols) put4<O, kMuon>(a, mat, r, c, val);
        }
    } else {
        const long kc0 = a.panels_q * 2, kc1 = a.panels_p * 2, at = piece_at(r0, c0, kc0);
        half4 old_h[4], old_l[4];
        if (kMode == kPoly) {                                // the same elements of P
            const char* pm = a.p + mat * a.bp + at + row * 16 + half * 8;
            for (int g = 0; g < 4; ++g) {
                old_h[g] = *(const half4*)(pm + (g >> 1) * 4096 + (g & 1) * 512);
                old_l[g] = *(const half4*)(pm + (g >> 1) * 4096 + (g & 1) * 512 + kLo);
            }
        }
        unsigned* t = (unsigned*)lds;                        // (hi, lo) of element (r, c) at r * 36 + c
        for (int g = 0; g < 4; ++g) {
            float val[4];
            for (int e = 0; e < 4; ++e) {
                val[e] = acc[g * 4 + e] * scale;
                if (kMode == kPoly) {
                    val[e] = fmaf(a.cc, val[e], a.cb * ((float)old_h[g][e] + (float)old_l[g][e]));
                    val[e] += r0 + row == c0 + g * 8 + half * 4 + e && r0 + row < a.m ? a.ca * kScale : 0.f;
                }
            }
            half4 h, l;
            split4(val, h, l);
            union { half4 v; unsigned w[2]; } hi = {h}, lo = {l};
            *(uint4*)(t + row * 36 + g * 8 + half * 4) =
                make_uint4(__builtin_amdgcn_perm(lo.w[0], hi.w[0], 0x05040100u), __builtin_amdgcn_perm(lo.w[0], hi.w[0], 0x07060302u),
                           __builtin_amdgcn_perm(lo.w[1], hi.w[1], 0x05040100u), __builtin_amdgcn_perm(lo.w[1], hi.w[1], 0x07060302u));
        }
        auto pack = [&](const unsigned (&w)[8], unsigned part) {
            return make_uint4(__builtin_amdgcn_perm(w[1], w[0], part), __builtin_amdgcn_perm(w[3], w[2], part),
                              __builtin_amdgcn_perm(w[5], w[4], part), __builtin_amdgcn_perm(w[7], w[6], part));
        };
        auto put = [&](char* to, const unsigned (&w)[8]) {
            *(uint4*)(to + lane * 16) = pack(w, 0x05040100u);
            *(uint4*)(to + lane * 16 + kLo) = pack(w, 0x07060302u);
        };
        for (int k = 0; k < 2; ++k) {
            const unsigned* from = t + row * 36 + k * 16 + half * 8;
            const uint4 x = *(const uint4*)from, y = *(const uint4*)(from + 4);
            put(a.c0 + mat * a.b0 + at + k * 4096, {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w});
        }
        if (flip) {
            char* tc = (kMode == kApply ? a.c1 + mat * a.b1 : a.c0 + mat * a.b0) + piece_at(c0, r0, kMode == kApply ? kc1 : kc0);
            for (int k = 0; k < 2; ++k) {
                unsigned w[8];
                for (int e = 0; e < 8; ++e) w[e] = t[(k * 16 + half * 8 + e) * 36 + row];
                put(tc + k * 4096, w);
            }
        }
    }
}

// from the accumulator to C times 2^10 (kFinal: to C)
template <int kMode>
__device__ __forceinline__ float scale_of(const ArgsOf<kMode>& a, int mat) {
    if (kMode == kPoly || kMode == kSym) return kInvScale;
    const float* f = a.factors + mat * (CNF_NS_MAX_STEPS + 1);
    return kInvScale * (kMode == kGram ? f[0] * f[0] : kMode == kApply ? f[0] / f[a.ahead] : f[0] * kInvScale);
}

// 64 x 64 tiles: each of four waves computes the whole tile over every fourth 16 columns of k, on operands that it loads from memory into
// registers kAhead steps before it needs them, and the partial sums are added at the end, in a fixed order.  The waves share no operands,
// so LDS would only add its own traffic: four matrices' 1024 x 1024 x 1024 symmetric products take 24 us, and 27 with operands copied to LDS
// (by one, two or four waves, which then wait for LDS).  What bounds it is the operands' way from L2, 16 TB/s.
template <int kMode, int kTerms, typename O = float, bool kMuon = false>
__global__ __launch_bounds__(256) void tile64_kernel(ArgsOf<kMode> a) {
    constexpr int kW = 4, kAhead = 4;
    __shared__ __align__(16) char lds[49152];                // partial sums: [quadrant][other wave][register][lane]; then finish()'s
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    int mat, ti, tj;
    my_tile(a.panels_p, a.panels_q, kSymmetric<kMode>, mat, ti, tj);
    const char* ps = a.p + mat * a.bp + (long)ti * a.kc * kBlockBytes + wave * 4096;
    const char* qs = a.q + mat * a.bq + (long)tj * a.kc * kBlockBytes + wave * 4096;
    const int steps = 2 * a.kc / kW;                         // (kc is even)
    float16v acc[2][2] = {};
    Frag<2, 2, kTerms> f[kAhead];
    auto load = [&](int d, int s) { f[d].read(ps + (long)s * (kW * 4096), qs + (long)s * (kW * 4096), lane); };
#pragma unroll
    for (int d = 0; d < kAhead; ++d)
        if (d < steps) load(d, d);
    int s = 0;
    for (; s + 2 * kAhead <= steps; s += kAhead) {
#pragma unroll
        for (int d = 0; d < kAhead; ++d) {
            f[d].multiply(acc);
            load(d, s + d + kAhead);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    // up to 2 kAhead - 1 are left, kAhead of them loaded
#pragma unroll
    for (int d = 0; d < kAhead; ++d)
        if (s + d < steps) {
            f[d].multiply(acc);
            if (s + d + kAhead < steps) load(d, s + d + kAhead);
        }
#pragma unroll
    for (int d = 0; d < kAhead; ++d)
        if (s + kAhead + d < steps) f[d].multiply(acc);
    if constexpr (kMode == kFinal) {
        if (a.guard && a.guard->status != 0) return;
    }
    const float scale = scale_of<kMode>(a, mat);
    const bool flip = kMode == kApply || (kSymmetric<kMode> && ti != tj);
    float* sums = (float*)lds;
#pragma unroll
    for (int t = 0; t < 4; ++t)
        if (t != wave)
            for (int i = 0; i < 16; ++i) sums[((t * 3 + (wave - (wave > t))) * 16 + i) * 64 + lane] = acc[t >> 1][t & 1][i];
    __syncthreads();
    float16v mine = wave == 0 ? acc[0][0] : wave == 1 ? acc[0][1] : wave == 2 ? acc[1][0] : acc[1][1];
    for (int w = 0; w < 3; ++w)
        for (int i = 0; i < 16; ++i) mine[i] += sums[((wave * 3 + w) * 16 + i) * 64 + lane];
    // (settled before the barrier: the compiler moves a read whose value only one side of a branch needs past it)
    for (int i = 0; i < 16; ++i) asm volatile("" ::"v"(mine[i]));
    __syncthreads();                                     // everybody has read the sums
    finish<kMode, O, kMuon>(a, mat, scale, mine, ti * 64l + (wave >> 1) * 32, tj * 64l + (wave & 1) * 32, flip, lane, lds + wave * kFlipBytes);
}

// T x T tiles for larger products: waves of kNu x kNv MFMA tiles share kStages stages of one block column each.  The operands of each 16 k are
// read while the products of the 16 before are computed, and the stage's one barrier falls between the two halves, with products on
// either side; the loop holds no branch, so that the compiler (T = 256) or the group barriers (kDealt) can place the reads and copies
// between the products.  4096 x 4096 x 4096 with T = 256, the loop timed by itself: 300 us (1.38 PFLOP/s of piece products; a large library product of
// fp16 matrices: 1.35), against 374 with reads and products in turn and 335 with the copies under a condition; the products alone, on operands that
// stay in registers, take 252 us: the device's power limit (177 with zeros for operands).  The kernel among the others of a call, its results stored: 347
// us (1.19 PFLOP/s).
template <int T, int kNu, int kNv, int kStages, int kMode, int kTerms, typename O = float, bool kMuon = false>
__global__ __launch_bounds__((T / 32 / kNu) * (T / 32 / kNv) * 64) void tile_kernel(ArgsOf<kMode> a) {
    constexpr int kAcross = T / 32 / kNv, kW = T / 32 / kNu * kAcross, kStage = 2 * T * 128, kLoads = kStage / 1024 / kW;
    constexpr bool kDealt = T < 256;
    static_assert(kW * kFlipBytes <= kStage && kLoads * kW * 1024 == kStage, "");
    __shared__ __align__(16) char lds[kStages][kStage];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    int mat, ti, tj;
    my_tile((a.panels_p + T / 64 - 1) / (T / 64), (a.panels_q + T / 64 - 1) / (T / 64), kSymmetric<kMode>, mat, ti, tj);
    const char* src[kLoads];
    for (int i = 0; i < kLoads; ++i) {
        // a stage in LDS: by 16 k (half a stage), operand, 32 rows, piece, a kilobyte each
        const int kb = wave * kLoads + i, half = kb / (T / 8), row32 = kb / 2 % (T / 32);
        const bool is_p = kb / (T / 16) % 2 == 0;
        const int panel = min((is_p ? ti : tj) * (T / 64) + row32 / 2, (is_p ? a.panels_p : a.panels_q) - 1);   // (past the end: the last one again)
        src[i] = (is_p ? a.p + mat * a.bp : a.q + mat * a.bq) + (long)panel * a.kc * kBlockBytes + half * 4096 + row32 % 2 * 2048 + kb % 2 * kLo;
    }
    auto load = [&](int k) {
        for (int i = 0; i < kLoads; ++i)
            __builtin_amdgcn_global_load_lds((gptr)(src[i] + k * kBlockBytes + lane * 16), (lptr)(&lds[k % kStages][(wave * kLoads + i) * 1024]), 16, 0, 0);
    };
    const int wr = (wave / kAcross) * kNu * 32, wc = (wave % kAcross) * kNv * 32;
    float16v acc[kNu][kNv] = {};
    Frag<kNu, kNv, kTerms> f0, f1;
    for (int k = 0; k < kStages && k < a.kc; ++k) load(k);
    if (kStages <= a.kc)
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"((kStages - 1) * kLoads) : "memory");
    else
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    f0.read(lds[0] + wr * 64, lds[0] + (T + wc) * 64, lane);
    constexpr int kReads = f0.kReads, kMul = kTerms * kNu * kNv;
    int k = 0;
    for (; k < a.kc - kStages; ++k) {
        f1.read(lds[k % kStages] + (2 * T + wr) * 64, lds[k % kStages] + (3 * T + wc) * 64, lane);
        f0.multiply(acc);
        if (kDealt) {
            for (int i = 0; i < kReads; ++i) {
                __builtin_amdgcn_sched_group_barrier(kSchedLdsRead, 1, 0);
                __builtin_amdgcn_sched_group_barrier(kSchedMfma, 1, 0);
            }
            __builtin_amdgcn_sched_group_barrier(kSchedMfma, kMul, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
        // the next stage has landed (the kStages - 2 after it may be on their way), and every wave has read this one
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((kStages - 2) * kLoads) : "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        const char* next = lds[(k + 1) % kStages];
        f0.read(next + wr * 64, next + (T + wc) * 64, lane);
        load(k + kStages);
        f1.multiply(acc);
        if (kDealt) {
            for (int i = 0; i < (kReads + 1) / 2; ++i) {
                __builtin_amdgcn_sched_group_barrier(kSchedLdsRead, 2, 0);
                __builtin_amdgcn_sched_group_barrier(kSchedMfma, 1, 0);
            }
            for (int i = 0; i < kLoads; ++i) {
                __builtin_amdgcn_sched_group_barrier(kSchedVmem, 1, 0);
                __builtin_amdgcn_sched_group_barrier(kSchedMfma, 1, 0);
            }
            __builtin_amdgcn_sched_group_barrier(kSchedMfma, kMul, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
    }
    for (; k < a.kc; ++k) {                                  // the last stages: nothing left to copy
        f1.read(lds[k % kStages] + (2 * T + wr) * 64, lds[k % kStages] + (3 * T + wc) * 64, lane);
        f0.multiply(acc);
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        const char* next = lds[(k + 1) % kStages];
        if (k + 1 < a.kc) f0.read(next + wr * 64, next + (T + wc) * 64, lane);
        f1.multiply(acc);
        __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (kMode == kFinal) {
        if (a.guard && a.guard->status != 0) return;
    }
    const float scale = scale_of<kMode>(a, mat);
    const bool flip = kMode == kApply || (kSymmetric<kMode> && ti != tj);
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kNu; ++u)
#pragma unroll
        for (int v = 0; v < kNv; ++v)
            finish<kMode, O, kMuon>(a, mat, scale, acc[u][v], (long)ti * T + wr + u * 32, (long)tj * T + wc + v * 32, flip, lane,
                                    lds[0] + wave * kFlipBytes);
}

// Matrices of at most 64 x 64: one workgroup per matrix does the whole update, with X, X^T, A and a I + b A + c A^2 as piece matrices in LDS
// (two blocks of 8 KB each), where the rows of every 8 columns are in another order: threads write what is 8 columns apart, which would
// lie in the same banks.  Each of eight waves computes 16 rows x 32 columns of every product.  What bounds it is the chain: 3 products per
// step, each a barrier, its operands' LDS reads, MFMAs, the split of its result; two waves on a SIMD fill each other's waits (64 x 64, five
// steps: 14 us; one wave a SIMD with 32 x 32 quadrants, 17).
constexpr int kSmall = 512;
typedef float float4v __attribute__((ext_vector_type(4)));

__device__ __forceinline__ int small_at(int r, int c) {
    return ((c >> 4) << 12) + ((r >> 5) << 11) + ((c >> 3 & 1) << 9) + (((r & 31) ^ (c >> 3)) << 4) + ((c & 7) << 1);
}

// rows pr .. + 15 and columns qr .. + 31 of sum_k P[r][k] Q[c][k], k = 0 .. 63: a lane holds columns 16 t + 4 (lane / 16) + e of row lane % 16
struct Part { float4v t[2]; };

__device__ __forceinline__ void multiply64(Part& acc, const char* p, int pr, const char* q, int qr, int lane) {
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
        const int c = kb * 32 + (lane >> 4) * 8, pat = small_at(pr + (lane & 15), c);
        const half8 ph = *(const half8*)(p + pat), pl = *(const half8*)(p + pat + kLo);
        half8 qh[2], ql[2];
        for (int t = 0; t < 2; ++t) {
            const int qat = small_at(qr + t * 16 + (lane & 15), c);
            qh[t] = *(const half8*)(q + qat);
            ql[t] = *(const half8*)(q + qat + kLo);
        }
        for (int t = 0; t < 2; ++t) acc.t[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ql[t], ph, acc.t[t], 0, 0, 0);
        for (int t = 0; t < 2; ++t) acc.t[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(qh[t], pl, acc.t[t], 0, 0, 0);
        for (int t = 0; t < 2; ++t) acc.t[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(qh[t], ph, acc.t[t], 0, 0, 0);
    }
}

// pieces of a wave's part, whose lane has columns col + 16 t .. + 3 of `row`: in LDS, or (kMemory) in a piece matrix 64 columns wide
template <bool kMemory = false>
__device__ __forceinline__ void store64(char* to, const Part& x, int row, int col) {
    for (int t = 0; t < 2; ++t) {
        half4 h, l;
        split4({x.t[t][0], x.t[t][1], x.t[t][2], x.t[t][3]}, h, l);
        const long at = kMemory ? piece_at(row, col + t * 16, 2) : small_at(row, col + t * 16);
        *(half4*)(to + at) = h;
        *(half4*)(to + at + kLo) = l;
    }
}

// a I + b A + c A^2 from A and, in B's place, the accumulator of A A
__device__ __forceinline__ void poly64(Part& B, const Part& A, float a, float b, float c, int row, int col, long m) {
    const float diag = row < m ? a * kScale : 0.f;
    for (int t = 0; t < 2; ++t)
        for (int e = 0; e < 4; ++e) {
            B.t[t][e] = fmaf(c * kInvScale, B.t[t][e], b * A.t[t][e]);
            B.t[t][e] += row == col + t * 16 + e ? diag : 0.f;
        }
}

template <typename O, bool kMuon>
__global__ __launch_bounds__(kSmall) void small_kernel(FinalArgs a, Dims d, Steps st, double eps, float mu, int nesterov) {
    __shared__ __align__(16) char xs[2 * kBlockBytes], xts[2 * kBlockBytes], as[2 * kBlockBytes], bs[2 * kBlockBytes];
    __shared__ double red[kSmall / 64];
    const int mat = blockIdx.x, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const bool skip = a.guard && a.guard->status != 0;
    const O* g = (const O*)a.ptrs.g[mat];
    // the matrix: thread (tr, tc) holds two rows of four columns (what lies outside is read at the last element and not used)
    const int tr = (threadIdx.x >> 4) * 2, tc = (threadIdx.x & 15) * 4;
    float v[2][4], old[2][4];
    for (int i = 0; i < 2; ++i)
        for (int k = 0; k < 4; ++k) {
            const int r = min(tr + i, (int)a.rows - 1), c = min(tc + k, (int)a.cols - 1);
            v[i][k] = to_f32(g[r * d.ldg + c]);
            if (kMuon) old[i][k] = a.ptrs.m[mat][r * d.ldm + c];
        }
    double s = 0.;
    for (int i = 0; i < 2; ++i)
        for (int k = 0; k < 4; ++k) {
            const int r = tr + i, c = tc + k;
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
    const double scale = start_scale(sqrt(((red[0] + red[1]) + (red[2] + red[3])) + ((red[4] + red[5]) + (red[6] + red[7]))), eps, f);
    char *straight = d.tall ? xts : xs, *flipped = d.tall ? xs : xts;
    for (int i = 0; i < 2; ++i)
        for (int k = 0; k < 4; ++k) v[i][k] = (float)((double)v[i][k] * scale);
    half4 h[2], l[2];
    for (int i = 0; i < 2; ++i) {
        split4(v[i], h[i], l[i]);
        const int at = small_at(tr + i, tc);
        *(half4*)(straight + at) = h[i];
        *(half4*)(straight + at + kLo) = l[i];
    }
    for (int k = 0; k < 4; ++k) {
        const int at = small_at(tc + k, tr);
        *(half2*)(flipped + at) = (half2){h[0][k], h[1][k]};
        *(half2*)(flipped + at + kLo) = (half2){l[0][k], l[1][k]};
    }
    const int wr = (wave >> 1) * 16, wc = (wave & 1) * 32;
    auto multiply = [&](const char* p, int pr, const char* q, int qr) {
        Part acc = {};
        multiply64(acc, p, pr, q, qr, lane);
        return acc;
    };
    const int row = wr + (lane & 15), col = wc + (lane >> 4) * 4;
    auto flip = [&](char* to, const Part& x) {               // pieces of the transpose of the wave's part
        for (int t = 0; t < 2; ++t) {
            half4 h, l;
            split4({x.t[t][0], x.t[t][1], x.t[t][2], x.t[t][3]}, h, l);
            for (int e = 0; e < 4; ++e) {
                const int at = small_at(col + t * 16 + e, row);
                *(f16*)(to + at) = h[e];
                *(f16*)(to + at + kLo) = l[e];
            }
        }
    };
    for (int k = 0; k < st.n; ++k) {
        __syncthreads();
        Part A = multiply(xs, wr, xs, wc);
        for (int t = 0; t < 2; ++t) A.t[t] *= kInvScale * f * f;
        store64(as, A, row, col);
        __syncthreads();
        Part B = multiply(as, wr, as, wc);
        poly64(B, A, st.a[k], st.b[k], st.c[k], row, col, d.m);
        store64(bs, B, row, col);
        __syncthreads();
        if (k + 1 < st.n) {
            Part X = multiply(bs, wr, xts, wc);
            const float f1 = fminf(1.f, f * st.grow[k]);
            for (int t = 0; t < 2; ++t) X.t[t] *= kInvScale * (f / f1);
            f = f1;
            __syncthreads();                                 // everybody has read X^T
            store64(xs, X, row, col);
            flip(xts, X);
        }
    }
    if (skip) return;
    const Part X = d.tall ? multiply(xts, wr, bs, wc) : multiply(bs, wr, xts, wc);
    if (row >= a.rows) return;
    for (int t = 0; t < 2; ++t) {
        float val[4];
        for (int e = 0; e < 4; ++e) val[e] = X.t[t][e] * (kInvScale * kInvScale * f);
        if (col + t * 16 < a.cols) put4<O, kMuon>(a, mat, row, col + t * 16, val);
    }
}

// Matrices whose shorter side is at most 64 and whose longer one is not.  A 64 x 64 tile of X is a whole block of columns, so the workgroup that
// makes it adds its part of X X^T at once, and X itself is never stored (the next product reads X^T).  Five steps are seven launches instead of
// twenty (64 x 1000: 42 us against 86).  `gram`: per matrix and workgroup the partial sums of X X^T as the waves hold them.  (Three steps at a time as
// in run() would save two more launches, 33 us, but a step costs little here and the grouping two thirds of the accuracy:
// 2.7e-6 against 0.9e-6 for 64 x 66, where plain fp32 is 1.2e-6 off.)

// How many workgroups share the tiles of a matrix: more make shorter loops and longer sums.  A step of 64 x 1000 takes 5.9 us with 16 workgroups
// and 6.8 with 8; 64 x 4096 14.8 with 8, 9.7 with 23, 13.1 with 64; 64 x 65536 94 with 16, 35 with 91.  Of many matrices no more than
// one to a CU, or two where there are tiles for long loops: 64 matrices 64 x 1000 88 us a call with 256 in all, 110 with 512, 159 without
// a limit; 64 x (64 x 20000) 1185 with 256, 966 with 512.
int skinny_parts(long count, long tiles) {
    const long most = (count * tiles > 4096 ? 2 : 1) * kCus / count;
    long n = (long)std::fmax(16., std::ceil(std::sqrt(8. * (double)tiles)));
    n = n < most ? n : most;
    return (int)(n < tiles ? n : tiles);
}

__device__ __forceinline__ void put_gram(float* gram, const Part& x, int wave, int lane) {
    float4v* to = (float4v*)(gram + ((long)blockIdx.y * gridDim.x + blockIdx.x) * 4096 + wave * 512) + lane * 2;
    to[0] = x.t[0], to[1] = x.t[1];
}

// 16 KB of a piece matrix 64 columns wide to LDS, in small_at's order
__device__ __forceinline__ void fetch64(char* to, const char* from) {
    for (int i = 0; i < 2; ++i) {
        const int at = (i * kSmall + threadIdx.x) * 16, c8 = (at >> 12) * 2 + (at >> 9 & 1);
        *(uint4*)(to + (at ^ c8 << 4)) = *(const uint4*)(from + at);
    }
}

template <typename T, bool kMuon, bool kVec>
__global__ __launch_bounds__(kSmall) void skinny_start_kernel(Ptrs p, Dims d, char* xt, const double* part, int parts, double eps, float mu,
                                                              int nesterov, Steps st, float* factors, float* gram) {
    __shared__ float tile[64][68];
    __shared__ __align__(16) char xs[2 * kBlockBytes];
    __shared__ double red[kSmall / 64];
    const int mat = blockIdx.y, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int tr = threadIdx.x >> 4, tc = (threadIdx.x & 15) * 4, wr = (wave >> 1) * 16, wc = (wave & 1) * 32;
    double s = 0.;
    for (int k = threadIdx.x; k < parts; k += kSmall) s += part[mat * kNormBlocks + k];
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
    if (lane == 0) red[wave] = s;
    __syncthreads();
    float f;
    const double scale = start_scale(sqrt(((red[0] + red[1]) + (red[2] + red[3])) + ((red[4] + red[5]) + (red[6] + red[7]))), eps, f);
    if (threadIdx.x == 0 && blockIdx.x == 0) put_factors(factors + mat * (CNF_NS_MAX_STEPS + 1), f, st);
    xt += mat * d.np * (64 * 4);
    Part acc = {};
    for (long t = blockIdx.x; t * 64 < d.np; t += gridDim.x) {
        const long r0 = d.tall ? t * 64 : 0, c = (d.tall ? 0 : t * 64) + tc;
        for (int i = 0; i < 2; ++i) {
            float v[4];
            start_values<T, kMuon, kVec>(p, d, mat, r0 + tr + i * 32, c, mu, nesterov, scale, v);
            *(float4*)&tile[tr + i * 32][tc] = make_float4(v[0], v[1], v[2], v[3]);
        }
        __syncthreads();
        const int i = threadIdx.x & 63, q = wave * 8;
        for (int out = 0; out < 2; ++out) {                     // X to LDS, X^T to memory
            float w[8];
            for (int k = 0; k < 8; ++k) w[k] = (out == 0) != (d.tall != 0) ? tile[i][q + k] : tile[q + k][i];
            half8 h, l;
            split8(w, h, l);
            char* to = out == 0 ? xs + small_at(i, q) : xt + t * (2 * kBlockBytes) + piece_at(i, q, 2);
            *(half8*)to = h;
            *(half8*)(to + kLo) = l;
        }
        __syncthreads();
        multiply64(acc, xs, wr, xs, wc, lane);
    }
    put_gram(gram, acc, wave, lane);
}

// One step: every workgroup adds the partial sums of X X^T and makes Q = a I + b A + c A^2 of them; X <- Q X for its tiles: X^T to xt2 and
// the partial sums of the new X X^T to gram2, or (kLast) X to the output.
template <bool kLast, typename O, bool kMuon>
__global__ __launch_bounds__(kSmall) void skinny_step_kernel(FinalArgs a, Dims d, Steps st, int k, const float* factors, const char* xt, char* xt2,
                                                             const float* gram, float* gram2) {
    __shared__ __align__(16) char as[2 * kBlockBytes], qs[2 * kBlockBytes], xts[2 * kBlockBytes];
    char* const xs = as;                                     // (A is not needed once Q is there)
    const int mat = blockIdx.y, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int wr = (wave >> 1) * 16, wc = (wave & 1) * 32, row = wr + (lane & 15), col = wc + (lane >> 4) * 4;
    const float f = factors[mat * (CNF_NS_MAX_STEPS + 1) + k];
    const float scale = kInvScale * (kLast ? f * kInvScale : f / factors[mat * (CNF_NS_MAX_STEPS + 1) + k + 1]);
    const bool skip = kLast && a.guard && a.guard->status != 0;
    xt += mat * d.np * (64 * 4);
    xt2 += mat * d.np * (64 * 4);
    long t = blockIdx.x;
    fetch64(xts, xt + t * (2 * kBlockBytes));
    Part A = {};
    const float4v* from = (const float4v*)(gram + (long)mat * gridDim.x * 4096 + wave * 512) + lane * 2;
    const int sums = gridDim.x;
    for (int w = 0; w < sums; w += 8) {                      // eight at a time on their way (past the last one: the last one again)
        Part x[8];
        for (int i = 0; i < 8; ++i)
            for (int u = 0; u < 2; ++u) x[i].t[u] = from[min(w + i, sums - 1) * 1024 + u];
        for (int i = 0; i < 8; ++i)
            for (int u = 0; u < 2; ++u)
                if (w + i < sums) A.t[u] += x[i].t[u];
    }
    for (int u = 0; u < 2; ++u) A.t[u] *= kInvScale * f * f;
    store64(as, A, row, col);
    __syncthreads();
    Part Q = {}, acc = {};
    multiply64(Q, as, wr, as, wc, lane);
    poly64(Q, A, st.a[k], st.b[k], st.c[k], row, col, d.m);
    store64(qs, Q, row, col);
    __syncthreads();
    while (true) {
        const long next = t + gridDim.x;
        Part X = {};
        if (kLast) {
            if (d.tall)                                      // the output's rows are X^T's
                multiply64(X, xts, wr, qs, wc, lane);
            else
                multiply64(X, qs, wr, xts, wc, lane);
            const long r = row + (d.tall ? t * 64 : 0);
            for (int u = 0; u < 2; ++u) {
                const long c = col + u * 16 + (d.tall ? 0 : t * 64);
                float val[4];
                for (int e = 0; e < 4; ++e) val[e] = X.t[u][e] * scale;
                if (!skip && r < a.rows && c < a.cols) put4<O, kMuon>(a, mat, r, c, val);
            }
        } else {
            Part Xt = {};
            multiply64(X, qs, wr, xts, wc, lane);
            multiply64(Xt, xts, wr, qs, wc, lane);
            for (int u = 0; u < 2; ++u) X.t[u] *= scale, Xt.t[u] *= scale;
            store64(xs, X, row, col);
            store64<true>(xt2 + t * (2 * kBlockBytes), Xt, row, col);
        }
        if (kLast && next * 64 >= d.np) return;
        __syncthreads();                                     // X^T is read, X is there
        if (next * 64 < d.np) fetch64(xts, xt + next * (2 * kBlockBytes));
        if (!kLast) multiply64(acc, xs, wr, xs, wc, lane);
        if (next * 64 >= d.np) break;
        t = next;
        __syncthreads();
    }
    if (!kLast) put_gram(gram2, acc, wave, lane);
}

// Which kernel computes a product: the one whose estimated time is least.  A round is as many workgroups as run at once; it takes `few` us per
// 4096 of k with few of them and `full` us when full, and `fixed` us whatever k is (its first operands, its results).  Where two run on a
// CU, a round takes `full` as soon as one CU has two; where one does, what lies behind the CUs slows down from half full on.  Fitted
// to products of 1 .. 1024 tiles and k = 256 .. 4096 (within a tenth for most, a quarter at worst); of those no choice was 5 % behind the best.
int choose(long count, int panels_p, int panels_q, bool sym, int kc) {
    struct Entry {
        int tile;
        long at_once;
        double few, full, fixed;
    };
    static constexpr Entry entries[] = {{64, 512, 22, 50, 4}, {128, 512, 84, 178, 7}, {192, 256, 135, 183, 14}, {256, 256, 196, 298, 20}};
    int best = 0;
    double least = 1e300;
    for (const Entry& e : entries) {
        const int t = e.tile / 64;
        const long r = (panels_p + t - 1) / t, c = (panels_q + t - 1) / t, tiles = count * (sym ? r * (r + 1) / 2 : r * c);
        const long whole = tiles / e.at_once, rest = tiles % e.at_once;
        double last = 0.;
        if (rest) last = e.at_once > kCus ? (rest > kCus ? e.full : e.few) : e.few + (e.full - e.few) * std::fmax(0., 2. * rest / kCus - 1.);
        const double time = (whole * e.full + last) * kc / 128. + (whole + (rest > 0)) * e.fixed;
        if (time < least) least = time, best = e.tile;
    }
    return best;
}

struct Plan {
    long m, n;      // the shorter and the longer side
    int pm, pn;     // in panels of 64
    bool small;     // one workgroup per matrix does everything in LDS
    bool skinny;    // the shorter side fits a tile: skinny_start_kernel and its like
    bool together;  // several steps at a time on the m x m side
};

// Several steps at a time need fewer operations where n is larger than m, and round the matrix of squared singular values, whose small ones the
// steps lift most.  Error of fp32 results against plain fp32's (normal matrices, gradient-like ones, and singular values over one, two and four
// decades): at most 1.45 times for m > 192 and n >= 2 m, where step by step it is 0.3 .. 1.1 times (1.5 at n >= 4096), but 3.5 times for 80 x 5000 and 2.2 for
// 100 x 4000, whose plain sums are no longer while their operands weigh more: those go step by step.  Time, step by step and together:
// 200 x 800 114 and 118 us, 200 x 1600 137 and 128, 400 x 800 138 and 148, 400 x 1600 166 and 158, 512 x 1024 147 and 151 (eight of them 256 and 242),
// 1024 x 4096 363 and 291 (four of them in a Muon update 1097 and 777).  A rule on the shape alone: what a matrix's neighbours are does not change its error.
Plan plan_of(long rows, long cols) {
    Plan p{};
    p.m = rows < cols ? rows : cols;
    p.n = rows < cols ? cols : rows;
    p.small = p.n <= 64;
    p.pm = (int)((p.m + 63) / 64);
    p.pn = (int)((p.n + 63) / 64);
    p.skinny = !p.small && p.pm == 1;
    p.together = p.m > 192 && p.n >= (p.m < 512 ? 4 : 2) * p.m;
    return p;
}

// how many of the steps from k on to take together: the matrix A <- B A B loses what its small eigenvalues' growth leaves of fp32 (their growth
// twice, up to 256), and the polynomials' product Q has to stay within the pieces' 64
int steps_together(const Plan& p, int steps, const double (&grow)[CNF_NS_MAX_STEPS], int k) {
    int n = 1;
    double up = std::fmax(1., grow[k]);
    while (p.together && n < 3 && k + n < steps && up * up <= 256. && up * std::fmax(1., grow[k + n]) <= 48.) up *= std::fmax(1., grow[k + n++]);
    return n;
}

template <int kMode, int kTerms = 3, typename O = float, bool kMuon = false>
void product(const FinalArgs& g, int count, hipStream_t s) {
    const int tile = choose(count, g.panels_p, g.panels_q, kSymmetric<kMode>, g.kc);
    const int t = tile / 64;
    const long r = (g.panels_p + t - 1) / t, c = (g.panels_q + t - 1) / t;
    const dim3 grid((unsigned)(count * (kSymmetric<kMode> ? r * (r + 1) / 2 : r * c)));
    if (tile == 256)
        tile_kernel<256, 4, 2, 2, kMode, kTerms, O, kMuon><<<grid, 512, 0, s>>>(g);
    else if (tile == 192)
        tile_kernel<192, 3, 3, 3, kMode, kTerms, O, kMuon><<<grid, 256, 0, s>>>(g);
    else if (tile == 128)
        tile_kernel<128, 2, 2, 2, kMode, kTerms, O, kMuon><<<grid, 256, 0, s>>>(g);
    else
        tile64_kernel<kMode, kTerms, O, kMuon><<<grid, 256, 0, s>>>(g);
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
    const Plan pl = plan_of(a.rows, a.cols);
    constexpr bool kHigh = kHighPieces<O, kMuon>;
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
    d.m = pl.m, d.n = pl.n, d.mp = pl.pm * 64l, d.np = pl.pn * 64l;
    const float mu = kMuon ? (float)a.opts->momentum : 0.f;
    const int nesterov = kMuon ? a.opts->nesterov : 0;
    FinalArgs g{};
    g.ptrs = p, g.rows = d.rows, g.cols = d.cols, g.ldo = d.ldo, g.guard = a.guard;
    g.decay = kMuon ? (float)(1.0 - a.opts->lr * a.opts->weight_decay) : 1.f;
    g.step = kMuon ? (float)(a.opts->lr * a.opts->scale) : 1.f;
    g.vec = vec_out;
    if (pl.small) {
        small_kernel<O, kMuon><<<dim3(a.count), kSmall, 0, s>>>(g, d, st, a.ns->eps, mu, nesterov);
        return hipGetLastError();
    }
    const long xb = d.mp * d.np * 4, ab = d.mp * d.mp * 4;
    double* part = (double*)a.ws;
    // partial sums: enough workgroups for the device, at least 2 K elements each
    long parts = (d.rows * d.cols + 2047) / 2048, most = (2048 + a.count - 1) / a.count;
    most = most < kNormBlocks ? most : kNormBlocks;
    parts = parts < most ? parts : most;
    const dim3 grid_in((unsigned)parts, a.count);
    if (vec_in)
        begin_kernel<O, kMuon, true><<<grid_in, kThreads, 0, s>>>(p, d, part, mu, nesterov, a.guard);
    else
        begin_kernel<O, kMuon, false><<<grid_in, kThreads, 0, s>>>(p, d, part, mu, nesterov, a.guard);
    char* const data = (char*)(part + (size_t)a.count * kNormBlocks);
    if (pl.skinny) {
        const int n_parts = skinny_parts(a.count, pl.pn);
        char *xt = data, *xt2 = xt + a.count * xb;
        float *gram = (float*)(xt2 + a.count * xb), *gram2 = gram + (long)a.count * n_parts * 4096, *factors = gram2 + (long)a.count * n_parts * 4096;
        const dim3 grid((unsigned)n_parts, a.count);
        if (vec_in)
            skinny_start_kernel<O, kMuon, true><<<grid, kSmall, 0, s>>>(p, d, xt, part, (int)parts, a.ns->eps, mu, nesterov, st, factors, gram);
        else
            skinny_start_kernel<O, kMuon, false><<<grid, kSmall, 0, s>>>(p, d, xt, part, (int)parts, a.ns->eps, mu, nesterov, st, factors, gram);
        for (int k = 0; k + 1 < st.n; ++k) {
            skinny_step_kernel<false, float, false><<<grid, kSmall, 0, s>>>(g, d, st, k, factors, xt, xt2, gram, gram2);
            std::swap(xt, xt2);
            std::swap(gram, gram2);
        }
        skinny_step_kernel<true, O, kMuon><<<grid, kSmall, 0, s>>>(g, d, st, st.n - 1, factors, xt, xt2, gram, gram2);
        return hipGetLastError();
    }
    char *x = data, *xt = x + a.count * xb, *xt2 = xt + a.count * xb, *sym[5];
    for (int i = 0; i < 5; ++i) sym[i] = xt2 + a.count * (xb + i * ab);
    float* factors = (float*)(sym[pl.together ? 4 : 1] + a.count * ab);
    const long rp = d.tall ? d.np : d.mp, cp = d.tall ? d.mp : d.np;
    const dim3 tiles((unsigned)(cp / 64), (unsigned)(rp / 64), a.count);
    if (vec_in)
        pieces_kernel<O, kMuon, true><<<tiles, kThreads, 0, s>>>(p, d, x, xt, part, (int)parts, a.ns->eps, mu, nesterov, st, factors);
    else
        pieces_kernel<O, kMuon, false><<<tiles, kThreads, 0, s>>>(p, d, x, xt, part, (int)parts, a.ns->eps, mu, nesterov, st, factors);
    const int km = pl.pm * 2, kn = pl.pn * 2;
    // `Q` times X: the steps k .. k + n - 1, to X and X^T, or to the output
    auto apply = [&](char* Q, int k, int n) {
        g.factors = factors + k, g.ahead = n;
        g.kc = km;
        g.p = Q, g.bp = ab, g.panels_p = pl.pm;
        g.q = xt, g.bq = xb, g.panels_q = pl.pn;
        if (k + n < st.n) {
            g.c0 = x, g.b0 = xb;
            g.c1 = xt2, g.b1 = xb;
            if (kHigh && k == 0)
                product<kApply, 2>(g, a.count, s);
            else
                product<kApply>(g, a.count, s);
            std::swap(xt, xt2);
            return;
        }
        if (d.tall) {                                        // the output's rows are X^T's
            std::swap(g.p, g.q);
            std::swap(g.bp, g.bq);
            std::swap(g.panels_p, g.panels_q);
        }
        product<kFinal, 3, O, kMuon>(g, a.count, s);
    };
    auto symmetric = [&](auto mode, auto terms, const char* p, const char* q, long bytes, int kc, char* to) {
        g.p = p, g.q = q, g.bp = g.bq = bytes, g.kc = kc;
        g.panels_p = g.panels_q = pl.pm;
        g.c0 = to, g.b0 = ab;
        product<decltype(mode)::value, decltype(terms)::value>(g, a.count, s);
    };
    constexpr std::integral_constant<int, 3> three{};
    auto gram = [&](int k, char* to) {
        g.factors = factors + k;
        if (kHigh && k == 0)
            symmetric(std::integral_constant<int, kGram>{}, std::integral_constant<int, 1>{}, x, x, xb, kn, to);
        else
            symmetric(std::integral_constant<int, kGram>{}, three, x, x, xb, kn, to);
    };
    auto poly = [&](int k, const char* A, char* to) {
        g.ca = st.a[k], g.cb = st.b[k], g.cc = st.c[k], g.m = d.m;
        symmetric(std::integral_constant<int, kPoly>{}, three, A, A, ab, km, to);
    };
    auto times = [&](const char* p, const char* q, char* to) { symmetric(std::integral_constant<int, kSym>{}, three, p, q, ab, km, to); };
    for (int k = 0; k < st.n;) {
        const int n = steps_together(pl, st.n, grow, k);
        char *A = sym[0], *B = sym[1], *Q = B;
        gram(k, A);
        poly(k, A, B);
        char *A2 = sym[2], *T = sym[3], *Q2 = sym[4];
        for (int i = 1; i < n; ++i) {
            // A <- B A B, the next polynomial to the place of T, Q <- B Q
            times(A, B, T);
            times(T, B, A2);
            std::swap(A, A2);
            if (i == 1) {                                    // Q is B itself: the next B gets another place
                poly(k + i, A, T);
                B = T;
                times(B, Q, Q2);
                T = A2;                                      // (the old A)
                A2 = Q;                                      // (the old B, after this product)
                Q = Q2;
            } else {
                poly(k + i, A, T);
                times(T, Q, A2);
                Q = A2;
            }
        }
        apply(Q, k, n);
        k += n;
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
    // the roots in u^2, from the sum of two numbers of one sign: a difference loses the smaller root where c is small
    const double A = 5. * c, B = 3. * b, D = B * B - 4. * A * a;
    if (!(D >= 0.)) return best;
    const double q = -0.5 * (B + std::copysign(std::sqrt(D), B));
    const double roots[2] = {q / A, a / q};                  // (infinite or NaN where there is none)
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

void muon_plan(long count, long rows, long cols, int32_t (&plan)[5]) {
    const Plan p = plan_of(rows, cols);
    plan[0] = p.small ? 0 : p.skinny ? 1 : 2;
    plan[1] = plan[0] == 2 && p.together;
    plan[2] = plan[3] = plan[4] = 64;
    if (plan[0] != 2) return;
    plan[2] = choose(count, p.pm, p.pm, true, 2 * p.pn);
    plan[3] = choose(count, p.pm, p.pm, true, 2 * p.pm);
    plan[4] = choose(count, p.pm, p.pn, false, 2 * p.pm);
}

size_t muon_workspace_bytes(long count, long rows, long cols) {
    const Plan p = plan_of(rows, cols);
    if (p.small) return 256;   // (uses none; 0 stands for a call that is not supported)
    const size_t m = p.pm * 64, n = p.pn * 64;
    if (p.skinny)
        return (size_t)count *
               (kNormBlocks * sizeof(double) + 2 * m * n * 4 + (size_t)skinny_parts(count, p.pn) * (2 * 16384) + (CNF_NS_MAX_STEPS + 1) * sizeof(float));
    return (size_t)count * (kNormBlocks * sizeof(double) + (3 * m * n + (p.together ? 5 : 2) * m * m) * 4 + (CNF_NS_MAX_STEPS + 1) * sizeof(float));
}

hipError_t launch_muon(int dtype, const MuonArgs& a, hipStream_t s) {
    if (dtype == CNF_F32) return run_op<float>(a, s);
    if (dtype == CNF_F16) return run_op<f16>(a, s);
    if (dtype == CNF_BF16) return run_op<bf16>(a, s);
    return hipErrorInvalidValue;
}

}  // namespace cnf
