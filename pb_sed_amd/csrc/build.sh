#!/bin/bash
# Build libpbsed_mi355.so for gfx950 (cross-compiles without a GPU).  Usage: build.sh [-j]
set -e
cd "$(dirname "$0")"
HIPCC=${HIPCC:-/opt/rocm/bin/hipcc}
# -packed-fp32-ops: no v_pk_{add,mul,fma}_f32 from ordinary float code (the host pass warns that it does not know the feature: harmless)
FLAGS="--offload-arch=gfx950 -O3 -std=c++17 -fPIC -Wno-unused-result -Wno-unused-value -Xclang -target-feature -Xclang -packed-fp32-ops"
mkdir -p build
pids=()
for f in api conv conv_bf16 conv_wino conv_winox3 conv_s16 conv1d_pc conv_wgrad gru gru_stack gru_wgrad tm_gemm causal_conv selective_scan layer_norm dropout misc logmel postproc collective; do
  if [ ! -f build/$f.o ] || [ -n "$(find $f.hip build.sh *.h *.inc -newer build/$f.o)" ]; then
    # logmel: products and sums contract within a statement only; the transform's fused multiply-adds are written out (fft512.h)
    EXTRA=""; [ $f = logmel ] && EXTRA="-ffp-contract=on"
    $HIPCC $FLAGS $EXTRA -c $f.hip -o build/$f.o &
    pids+=($!)
  fi
done
for p in "${pids[@]}"; do wait $p; done
$HIPCC --offload-arch=gfx950 -shared -fPIC build/*.o -L/opt/rocm/lib -lrccl -Wl,-rpath,/opt/rocm/lib -o ../libpbsed_mi355.so
echo "built $(cd .. && pwd)/libpbsed_mi355.so"
