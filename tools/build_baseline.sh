#!/bin/bash
# Baseline build for A/B runs on the GPU box: csrc/hashgrid.hip (+ its includes) as of a given commit, linked with the
# CURRENT objects of every other translation unit into build/variants/libnsr_hip_<tag>.so (pick it with NSR_HIP_LIB=<path>).
# Entry points the old source does not have are stubbed so that the ctypes binding table still resolves.
#   tools/build_baseline.sh <commit> <tag>
set -e
COMMIT="${1:?commit}"; TAG="${2:?tag}"
HERE="$(cd "$(dirname "$0")/.." && pwd)"
CS="$HERE/instant-nsr-pl_amd/csrc"
. "$CS/flags.sh"
SRC="$(mktemp -d)/repo"; mkdir -p "$SRC" "$HERE/build/variants"
git -C "$HERE" archive "$COMMIT" instant-nsr-pl_amd/csrc include | tar x -C "$SRC"
cat > "$SRC/stubs.cpp" <<'EOS'
#include <stdint.h>
extern "C" __attribute__((weak)) float nsr_hashgrid_owner_tune(int, float) { return -1.f; }
extern "C" __attribute__((weak)) int nsr_hashgrid_owner_debug_map(const void *, int, uint32_t, uint32_t, int, uint32_t *) { return -1; }
EOS
OUT="$HERE/build/variants"
hipcc $NSR_FLAGS -c "$SRC/instant-nsr-pl_amd/csrc/hashgrid.hip" -o "$OUT/hashgrid_$TAG.o"
g++ -O2 -fPIC -c "$SRC/stubs.cpp" -o "$OUT/stubs_$TAG.o"
hipcc --offload-arch=gfx950 -shared -fPIC -o "$OUT/libnsr_hip_$TAG.so" "$OUT/hashgrid_$TAG.o" "$OUT/stubs_$TAG.o" \
  $(nsr_objects "$CS/obj" hashgrid)
echo "built $OUT/libnsr_hip_$TAG.so (hashgrid.hip @ $COMMIT)"
