// cnf_ops.h -- what the operators of a training step outside the solves share (cnf_norm.hip, cnf_muon.hip): element types,
// loads and stores that convert to fp32, and the launcher prototypes cnf_api.hip calls.
#pragma once
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include "../../include/cnf_hip.h"

namespace cnf {

using f16 = _Float16;
using bf16 = __hip_bfloat16;

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(f16 v) { return (float)v; }
__device__ __forceinline__ float to_f32(bf16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ f16 from_f32<f16>(float v) { return (f16)v; }
template <>
__device__ __forceinline__ bf16 from_f32<bf16>(float v) { return __float2bfloat16(v); }   // to nearest, ties to even

// ---- layer normalisation (cnf_norm.hip) -----------------------------------------------------------------------------
struct NormArgs {
    const void *x, *dy, *weight, *bias;
    long x_stride, dy_stride;   // elements between rows
    long rows, cols;
    float eps;
    void* y;
    float *mean, *rstd;         // forward: nullable outputs; backward: inputs
    void *dx, *dweight, *dbias; // backward, each nullable
    float* part;                // backward: partial column sums
};
size_t layer_norm_workspace_bytes(long rows, long cols);
hipError_t launch_layer_norm_fwd(int dtype, int wdtype, const NormArgs& a, hipStream_t s);
hipError_t launch_layer_norm_bwd(int dtype, int wdtype, const NormArgs& a, hipStream_t s);

// ---- Newton-Schulz orthogonalisation and the Muon update (cnf_muon.hip) ----------------------------------------------
struct MuonArgs {
    const void* const* g;       // host arrays of `count` device pointers
    void* const* out;           // the orthogonalised matrices, or the parameters a Muon update changes
    float* const* momenta;      // Muon update only
    long ldg, ldo, ldm;
    int count;
    long rows, cols;
    const CnfNewtonSchulz* ns;
    const CnfMuonOpts* opts;    // null: orthogonalise only
    const CnfStats* guard;
    void* ws;
};
// bounds the iteration over singular values in [0, 1]: 0, or the number of the first step that lets them leave the range the
// kernels hold; grow[k]: the largest |a + b t + c t^2| of step k
int ns_bounds(const CnfNewtonSchulz& ns, double (&grow)[CNF_NS_MAX_STEPS]);
void muon_plan(long count, long rows, long cols, int32_t (&plan)[5]);   // cnf_debug_matrix_plan
size_t muon_workspace_bytes(long count, long rows, long cols);
hipError_t launch_muon(int dtype, const MuonArgs& a, hipStream_t s);

}  // namespace cnf
