#!/usr/bin/env bash
# Builds the C-ABI library for sm_100a into ../lib/libfp4t.so and the torch-side module that calls it into
# ../lib/fp4t_torch.so (both in-tree, git-ignored).  The translation units are compiled side by side.
set -euo pipefail
here="$(cd "$(dirname "${BASH_SOURCE[0]}")" && pwd)"
out="$here/../lib"
mkdir -p "$out"
NVCC="${NVCC:-/usr/local/cuda/bin/nvcc}"
PYTHON="${PYTHON:-python3}"
CXX_HOST="${CXX:-g++}"
ARCH=(-gencode arch=compute_100a,code=sm_100a)
tmp="$(mktemp -d)"
trap 'rm -rf "$tmp"' EXIT
pids=()
for unit in quantize gemm misc linear allreduce norm rotary xent; do
  "$NVCC" "${ARCH[@]}" -O3 -lineinfo -std=c++17 -Xcompiler -fPIC -Xcompiler -fvisibility=hidden ${FP4T_NVCC_EXTRA:-} \
    -c -o "$tmp/$unit.o" "$here/fp4t_$unit.cu" &
  pids+=($!)
done
# torch's own headers and libraries, of the interpreter that will load the module
torch_flags="$("$PYTHON" - <<'PY'
import os
import sysconfig

import torch

root = os.path.dirname(torch.__file__)
print(" ".join(f"-isystem {root}/include{d}" for d in ("", "/torch/csrc/api/include")), f"-isystem {sysconfig.get_paths()['include']}",
      f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", f"-L{root}/lib")
PY
)"
"$CXX_HOST" -O2 -std=c++17 -fPIC -fvisibility=hidden -DTORCH_EXTENSION_NAME=fp4t_torch -DTORCH_API_INCLUDE_EXTENSION_H $torch_flags \
  -isystem "$(dirname "$NVCC")/../include" -c -o "$tmp/fp4t_torch.o" "$here/fp4t_torch.cpp" &
pids+=($!)
for pid in "${pids[@]}"; do wait "$pid"; done
units=()
for unit in quantize gemm misc linear allreduce norm rotary xent; do units+=("$tmp/$unit.o"); done
"$NVCC" "${ARCH[@]}" -shared -o "$out/libfp4t.so" "${units[@]}"
# (the C++ runtime is named: a second, static copy of it, which some compiler installations link, ends the
# process at the first formatted error message)
"$CXX_HOST" -shared -o "$out/fp4t_torch.so" "$tmp/fp4t_torch.o" -l:libstdc++.so.6 $torch_flags -L"$out" -lfp4t -lc10 -lc10_cuda -ltorch_cpu -ltorch -ltorch_python \
  -Wl,-rpath,'$ORIGIN'
echo "built $out/libfp4t.so $out/fp4t_torch.so"
