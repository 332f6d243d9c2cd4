#!/bin/bash
# Builds libdragon_hip.so for gfx950, in-tree: HIP kernels + C ABI + runtime bridge
# (hipcc) and the host-side engine mirror (g++, plain C++ above the C ABI).
set -uo pipefail
cd "$(dirname "$0")"
HIPCC=${HIPCC:-/opt/rocm/bin/hipcc}
HIPFLAGS="--offload-arch=gfx950 -O3 -std=c++17 -fPIC -Wall -Wno-unused-function \
  -Xclang -target-feature -Xclang -packed-fp32-ops"
mkdir -p build
OBJS=""
PIDS=""
for s in gemm_mfma.hip gemm_mfma_biased.hip gemm_mfma_dma.hip gemm_mfma_streamk.hip gemm_mfma_band.hip gemm_mfma_shortk.hip gemm_skinny.hip gemm_mfma_conv.hip skbuf_summary.hip bias_row.hip c_abi_gemm.hip c_abi_conv.hip runtime.hip transfer.hip transpose.hip softmax.hip attention.hip attention_window.hip attention_window_grad.hip linear_attention.hip; do
  o=build/${s%.hip}.o
  # the host pass does not know the packed-fp32 target feature and says so: harmless
  if [ "$s" = gemm_mfma_streamk.hip ]; then
    # the balanced kernel's register and scratch use per instantiation, as the compiler reports it, kept beside the
    # object for tests/test_kernel_resources.py
    ( $HIPCC $HIPFLAGS -Rpass-analysis=kernel-resource-usage -c "$s" -o "$o" > build/gemm_mfma_streamk.resources.txt 2>&1; rc=$?
      if [ $rc -ne 0 ]; then grep -v "packed-fp32-ops" build/gemm_mfma_streamk.resources.txt | grep -B2 -A6 "error" >&2; fi
      exit $rc ) &
    PIDS="$PIDS $!"
    OBJS="$OBJS $o"
    continue
  fi
  # accumulators of matrix instructions stay in the vector registers that the vector instructions reach: with the
  # compiler's own choice window_grad_kv moved all 128 of them out and in again in every step
  EXTRA=""
  [ "$s" = attention_window_grad.hip ] && EXTRA="-mllvm -amdgpu-mfma-vgpr-form=true"
  ( $HIPCC $HIPFLAGS $EXTRA -c "$s" -o "$o" 2>&1 | grep -v "packed-fp32-ops" >&2; exit ${PIPESTATUS[0]} ) &
  PIDS="$PIDS $!"
  OBJS="$OBJS $o"
done
for s in ../engine/dragon_engine.cpp ../engine/engine_c_api.cpp; do
  o=build/$(basename "${s%.cpp}").o
  g++ -O2 -std=c++17 -fPIC -Wall -c "$s" -o "$o" &
  PIDS="$PIDS $!"
  OBJS="$OBJS $o"
done
for p in $PIDS; do
  wait "$p" || { echo "build.sh: a compile step failed" >&2; exit 1; }
done
$HIPCC --offload-arch=gfx950 -shared -fPIC -o ../libdragon_hip.so $OBJS || exit 1
echo "built $(cd .. && pwd)/libdragon_hip.so"
