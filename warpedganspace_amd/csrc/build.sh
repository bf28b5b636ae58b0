#!/usr/bin/env bash
# Build libwgs_hip.so for gfx950 (MI355X) in-tree.  No torch headers, no pybind: a plain C-ABI library.
set -euo pipefail
cd "$(dirname "$0")"
HIPCC=${HIPCC:-/opt/rocm/bin/hipcc}
# No packed fp32 instructions (v_pk_add_f32 and the like), from the compiler or by hand: some of their forms have given wrong results now and then on
# gfx950, without an error.  (hipcc's host pass warns that it does not know the feature.)
FLAGS="--offload-arch=gfx950 -O3 -std=c++17 -fPIC -munsafe-fp-atomics -Wall -Wno-unused-function -Xclang -target-feature -Xclang -packed-fp32-ops"
OBJS=() PIDS=()
for src in *.hip; do
  obj="build/${src%.hip}.o"
  mkdir -p build
  if [ ! -f "$obj" ] || [ "$src" -nt "$obj" ] || [ wgs_common.h -nt "$obj" ] || [ conv_args.h -nt "$obj" ] || [ fir4.h -nt "$obj" ] || [ conv_epilogue.h -nt "$obj" ] || [ conv_scheme.h -nt "$obj" ] || [ conv_nt_kernel.inc -nt "$obj" ] || [ conv_nt_launch.inc -nt "$obj" ] || [ ../../include/wgs.h -nt "$obj" ] || [ build.sh -nt "$obj" ] \
     || { [ -f "${src%.hip}.inc" ] && [ "${src%.hip}.inc" -nt "$obj" ]; }; then
    echo "[hipcc] $src"
    rm -f "$obj"                # (a failed compilation leaves no object of older sources)
    $HIPCC $FLAGS -c "$src" -o "$obj" &
    PIDS+=($!)
  fi
  OBJS+=("$obj")
done
for pid in ${PIDS[@]+"${PIDS[@]}"}; do wait "$pid"; done       # (a plain wait forgets a job's failure)
$HIPCC --offload-arch=gfx950 -shared -fPIC -o ../libwgs_hip.so "${OBJS[@]}"
# fingerprint of the sources and flags this library was built from (checked by __graft_entry__.build() and warpedganspace_amd._lib: a prebuilt
# .so that travels with a snapshot must match the sources beside it)
LC_ALL=C; export LC_ALL; cat *.hip *.h *.inc ../../include/wgs.h build.sh | sha256sum | cut -d' ' -f1 > ../libwgs_hip.so.sources.sha256
echo "built $(cd .. && pwd)/libwgs_hip.so"
