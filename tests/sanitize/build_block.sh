#!/bin/bash
# Sanitizer build of the host code of the norms, the choice of experts and the
# dense projections (every source compiled with its host side instrumented)
# linked with block_probe.cpp. Usage: build_block.sh OUTDIR
set -euo pipefail
HERE=$(cd "$(dirname "$0")" && pwd)
ROOT=$(cd "$HERE/../.." && pwd)
OUT=$1
mkdir -p "$OUT"
HIPCC=${HIPCC:-/opt/rocm/bin/hipcc}
SAN="-Xarch_host -fsanitize=address -Xarch_host -fsanitize=undefined -Xarch_host -fno-sanitize-recover=all"
pids=()
objs=()
for src in abi.cpp norm.hip norm_grad.hip route_experts.hip linear.hip; do
  obj="$OUT/${src%.*}.block.o"
  objs+=("$obj")
  $HIPCC -x hip -O1 -g -fPIC -std=c++17 --offload-arch=gfx950 $SAN -Xclang -target-feature -Xclang -packed-fp32-ops \
    -Wno-unused-command-line-argument \
    -c "$ROOT/keep_amd/csrc/$src" -o "$obj" &
  pids+=($!)
done
for p in "${pids[@]}"; do wait "$p"; done
$HIPCC -x hip -O1 -g -std=c++17 --offload-host-only $SAN -I "$ROOT/include" -c "$HERE/block_probe.cpp" -o "$OUT/block_probe.o"
$HIPCC --offload-arch=gfx950 $SAN "$OUT/block_probe.o" "${objs[@]}" -o "$OUT/block_probe"
