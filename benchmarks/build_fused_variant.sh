#!/bin/bash
# build_fused_variant.sh NAME [extra hipcc flags...]: like build_variant.sh, but only nf_fused.hip is recompiled with the
# extra flags; the other objects are the in-tree ones (run `make -C normalizing-flows_amd/csrc` first).
set -e
name=$1; shift
root=$(cd "$(dirname "$0")/.." && pwd)
src=$root/normalizing-flows_amd/csrc
mkdir -p /tmp/nf_fv_$name $root/normalizing-flows_amd/variants
/opt/rocm/bin/hipcc -O3 --offload-arch=gfx950 -fPIC -std=c++17 -Xclang -target-feature -Xclang -packed-fp32-ops -Wno-unused-function -Wno-pass-failed -I$src -ffp-contract=off -fno-slp-vectorize "$@" \
    -c $src/nf_fused.hip -o /tmp/nf_fv_$name/nf_fused.o
/opt/rocm/bin/hipcc --offload-arch=gfx950 -shared -fPIC -o $root/normalizing-flows_amd/variants/libnf_hip_$name.so \
    /tmp/nf_fv_$name/nf_fused.o $src/nf_api.o $src/nf_spline.o $src/nf_gemm.o $src/nf_maf.o $src/nf_resnet.o $src/nf_inverse.o $src/nf_hidden.o $src/nf_coupling.o $src/nf_norm.o $src/nf_orth.o
echo built $name
