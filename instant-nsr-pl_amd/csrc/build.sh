#!/bin/bash
# Build libnsr_hip.so for gfx950 (cross-compiles without a GPU).  Usage: build.sh [outdir]
set -e
HERE="$(cd "$(dirname "$0")" && pwd)"
OUT="${1:-$HERE/../nsr_hip}"
. "$HERE/flags.sh"
mkdir -p "$HERE/obj"
pids=()
for f in $NSR_UNITS; do
  ( hipcc $NSR_FLAGS ${NSR_EXTRA_FLAGS} -c "$HERE/$f.hip" -o "$HERE/obj/$f.o" ) &
  pids+=($!)
done
for p in "${pids[@]}"; do wait $p; done
hipcc --offload-arch=gfx950 -shared -fPIC -o "$OUT/libnsr_hip.so" $(nsr_objects "$HERE/obj")
echo "built $OUT/libnsr_hip.so"
