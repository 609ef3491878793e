#!/bin/bash
# `make -C gan-flow_amd/csrc debug`: the four kernel libraries with -DCNF_DEBUG_BOUNDS (csrc/cnf_launch.h, dbg_ws) into
# gan-flow_amd/debug/ (git-ignored).  Run a program on them with CNF_HIP_LIBDIR=$PWD/gan-flow_amd/debug: a workspace range
# outside what cnf_workspace_bytes() names is printed, the solve's status becomes CNF_ERR_DEBUG_BOUNDS (5) and the access is
# redirected -- no GPU fault.  Compiler flags per file as in the release build, except where noted below.
set -e
cd "$(dirname "$0")/../gan-flow_amd/csrc"
OUT=../debug
mkdir -p $OUT
FLAGS="-O3 -std=c++17 -fPIC --offload-arch=gfx950 -Wall -Wno-unused-function -ffp-contract=off -DCNF_DEBUG_BOUNDS"
NOPK="-Xclang -target-feature -Xclang -packed-fp32-ops"
SRCS="cnf_fwd cnf_bwd cnf_split cnf_split_fwd cnf_split16 cnf_wide cnf_wide_bwd cnf_train cnf_data cnf_norm cnf_muon cnf_api"
build_lib() {   # $1: suffix, $2: -DCNF_ACT=..., $3: library name
  objs=""
  for f in $SRCS; do
    extra=""
    # cnf_split / cnf_split_fwd: the release build passes their assembly through pk_hazard_pass.py (packed fp32 beside bf16 MFMA
    # streams); here they are simply compiled without packed fp32 -- same arithmetic, no such instruction
    case $f in cnf_fwd|cnf_wide_bwd|cnf_split|cnf_norm|cnf_muon) extra="$NOPK";; cnf_split_fwd) extra="$NOPK -mllvm -amdgpu-sched-strategy=max-ilp";; esac
    /opt/rocm/bin/hipcc $FLAGS $extra $2 -c $f.hip -o $OUT/$f$1.o 2> >(grep -v "not a recognized feature" >&2)
    objs="$objs $OUT/$f$1.o"
  done
  /opt/rocm/bin/hipcc --offload-arch=gfx950 -shared -fPIC -o $OUT/$3 $objs
  rm -f $objs
  echo built $OUT/$3
}
build_lib "" "" libcnf_hip.so &
build_lib .softplus -DCNF_ACT=1 libcnf_hip_softplus.so &
build_lib .elu -DCNF_ACT=2 libcnf_hip_elu.so &
build_lib .relu -DCNF_ACT=3 libcnf_hip_relu.so &
wait
