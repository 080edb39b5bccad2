# What every build of the library is made of (sourced by build.sh, tools/build_variants.sh, tools/build_baseline.sh): the
# translation units, and the compiler's flags.  Without packed fp32 instructions: some of their forms are not reliable here.
NSR_UNITS="util hashgrid gridmlp mlp vmlp neus march render fused occupancy step optim norm"
NSR_FLAGS="--offload-arch=gfx950 -O3 -std=c++17 -fPIC -ffp-contract=off -munsafe-fp-atomics -Wall -Wno-unused-function -Xclang -target-feature -Xclang -packed-fp32-ops"
# objects of all units but the named one: nsr_objects <folder> [unit]
nsr_objects() {
  local u
  for u in $NSR_UNITS; do [ "$u" = "$2" ] || echo "$1/$u.o"; done
}
