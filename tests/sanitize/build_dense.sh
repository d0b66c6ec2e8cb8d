#!/bin/bash
# Sanitizer build of the dense products', the adapters' and the plan's host code
# (every source compiled with its host side instrumented) linked with
# dense_probe.cpp. Usage: build_dense.sh OUTDIR
set -euo pipefail
HERE=$(cd "$(dirname "$0")" && pwd)
ROOT=$(cd "$HERE/../.." && pwd)
OUT=$1
mkdir -p "$OUT"
HIPCC=${HIPCC:-/opt/rocm/bin/hipcc}
SAN="-Xarch_host -fsanitize=address -Xarch_host -fsanitize=undefined -Xarch_host -fno-sanitize-recover=all"
pids=()
objs=()
for src in abi.cpp plan.hip combine.hip dense.hip dense_gemm.hip lora.hip plan_blocks.hip; do
  obj="$OUT/${src%.*}.dense.o"
  objs+=("$obj")
  $HIPCC -x hip -O1 -g -fPIC -std=c++17 --offload-arch=gfx950 $SAN -Xclang -target-feature -Xclang -packed-fp32-ops \
    -Wno-unused-command-line-argument \
    -c "$ROOT/keep_amd/csrc/$src" -o "$obj" &
  pids+=($!)
done
for p in "${pids[@]}"; do wait "$p"; done
$HIPCC -O1 -g -std=c++17 --offload-host-only $SAN -I "$ROOT/include" -c "$HERE/dense_probe.cpp" -o "$OUT/dense_probe.o"
$HIPCC --offload-arch=gfx950 $SAN "$OUT/dense_probe.o" "${objs[@]}" -o "$OUT/dense_probe"
