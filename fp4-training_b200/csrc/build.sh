#!/usr/bin/env bash
# Builds the C-ABI library for sm_100a into ../lib/libfp4t.so (in-tree, git-ignored).
# The translation units are compiled side by side.
set -euo pipefail
here="$(cd "$(dirname "${BASH_SOURCE[0]}")" && pwd)"
out="$here/../lib"
mkdir -p "$out"
NVCC="${NVCC:-/usr/local/cuda/bin/nvcc}"
ARCH=(-gencode arch=compute_100a,code=sm_100a)
tmp="$(mktemp -d)"
trap 'rm -rf "$tmp"' EXIT
pids=()
for unit in quantize gemm misc linear allreduce norm rotary xent; do
  "$NVCC" "${ARCH[@]}" -O3 -lineinfo -std=c++17 -Xcompiler -fPIC -Xcompiler -fvisibility=hidden ${FP4T_NVCC_EXTRA:-} \
    -c -o "$tmp/$unit.o" "$here/fp4t_$unit.cu" &
  pids+=($!)
done
for pid in "${pids[@]}"; do wait "$pid"; done
"$NVCC" "${ARCH[@]}" -shared -o "$out/libfp4t.so" "$tmp"/*.o
echo "built $out/libfp4t.so"
