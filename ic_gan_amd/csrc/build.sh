#!/bin/bash
# Build libicgan_hip.so for gfx950 (MI355X).  hipcc cross-compiles without a GPU.
set -euo pipefail
HERE="$(cd "$(dirname "${BASH_SOURCE[0]}")" && pwd)"
OUT="$HERE/../lib"
mkdir -p "$OUT" "$HERE/obj"
HIPCC="${HIPCC:-/opt/rocm/bin/hipcc}"
# -packed-fp32-ops: no v_pk_{add,mul,fma}_f32 (the compiler forms them from ordinary float code by itself)
FLAGS="--offload-arch=gfx950 -O3 -std=c++17 -fPIC -Xclang -target-feature -Xclang -packed-fp32-ops -Wno-unused-value -Wno-sometimes-uninitialized -Wno-uninitialized"
pids=()
for src in "$HERE"/*.hip; do
  obj="$HERE/obj/$(basename "${src%.hip}").o"
  if [ ! -f "$obj" ] || [ "$src" -nt "$obj" ] || [ -n "$(find "$HERE" \( -name '*.h' -o -name build.sh \) -newer "$obj")" ] || [ "$HERE/../../include/icgan_hip.h" -nt "$obj" ]; then
    ( $HIPCC $FLAGS -c "$src" -o "$obj" ) &
    pids+=($!)
  fi
done
for p in "${pids[@]:-}"; do [ -n "$p" ] && wait "$p"; done
$HIPCC --offload-arch=gfx950 -shared -fPIC "$HERE"/obj/*.o -o "$OUT/libicgan_hip.so"
echo "built $OUT/libicgan_hip.so"
