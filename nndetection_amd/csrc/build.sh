#!/bin/bash
# Build libnndet_amd.so for gfx950 (cross-compiles without a GPU). Usage: csrc/build.sh; REBUILD=1 compiles every source again
set -e
cd "$(dirname "$0")"
HIPCC=${HIPCC:-/opt/rocm/bin/hipcc}
# -packed-fp32-ops: hipcc -O3 makes v_pk_{add,mul,fma}_f32 out of ordinary float code, and some of their forms have given wrong results
# on this part without any error; scalar fp32 instructions only. (The host pass warns that it does not know the feature: harmless.)
COMMON="--offload-arch=gfx950 -O3 -std=c++17 -fPIC -munsafe-fp-atomics -Wno-unused-result -Xclang -target-feature -Xclang -packed-fp32-ops"
mkdir -p _obj
pids=()
# build.sh --asm DIR : emit the gfx950 ISA of every source (same flags) into DIR/*.s instead of building the library
# (tests/test_isa_hazards.py scans it with tools/scan_store_hazard.py)
ASM_DIR=""
if [ "$1" = "--asm" ]; then ASM_DIR=$2; mkdir -p "$ASM_DIR"; fi
build() { # src extra-flags
  local src=$1; shift
  if [ -n "$ASM_DIR" ]; then
    $HIPCC $COMMON "$@" --cuda-device-only -S "$src" -o "$ASM_DIR/${src%.hip}.s" 2>/dev/null &
    pids+=($!)
    return
  fi
  local obj=_obj/${src%.hip}.o
  if [ -n "$REBUILD" ] || [ ! -f "$obj" ] || [ build.sh -nt "$obj" ] || [ "$src" -nt "$obj" ] || [ common.h -nt "$obj" ] || [ conv_common.h -nt "$obj" ] || [ radix_select.h -nt "$obj" ] || [ ../../include/nndet_amd.h -nt "$obj" ]; then
    $HIPCC $COMMON "$@" -c "$src" -o "$obj" &
    pids+=($!)
  fi
}
# bit-exact box kernels: no FMA contraction (IEEE division / sqrt are hipcc defaults)
build nms3d.hip -ffp-contract=off
build boxes.hip -ffp-contract=off
build atss3d.hip -ffp-contract=off
build postproc.hip -ffp-contract=off
build targets.hip
build sampler.hip
build wbc3d.hip -ffp-contract=off
# k_ig3r is one fully unrolled 432-MFMA tile body: beyond the default size limit of '#pragma unroll'
build conv_igemm.hip -mllvm -pragma-unroll-threshold=1000000
build conv_wgrad.hip
build conv_pw.hip
build conv_dgs.hip
build conv_ig3s.hip
build conv_stem.hip
build norm.hip
build segloss.hip
build headio.hip
build sparse_out.hip
build segbranch.hip
build optim.hip -ffp-contract=off
build api.hip
# the host side of the optimiser's tensor lists (torch's C++ headers; a Python module, no GPU code). It has the layout of torch's tensors built in:
# another torch or Python than it was built for compiles it again here, and _lib.host_lists() refuses it.
if [ -z "$ASM_DIR" ]; then
  HOST=$(${PYTHON:-python3} -c "import sysconfig, os, torch; print(sysconfig.get_paths()['include'], os.path.dirname(torch.__file__), int(torch._C._GLIBCXX_USE_CXX11_ABI), torch.__version__, sysconfig.get_config_var('SOABI'))")
  read -r PYINC TORCH ABI VERSION SOABI <<< "$HOST"
  if [ -n "$REBUILD" ] || [ ! -f nndet_host.so ] || [ "$(cat _obj/host_for 2>/dev/null)" != "$HOST" ] || [ build.sh -nt nndet_host.so ] || [ host_lists.cpp -nt nndet_host.so ] || [ ../../include/nndet_amd.h -nt nndet_host.so ]; then
    rm -f _obj/host_for
    g++ -O2 -std=c++17 -fPIC -shared -D_GLIBCXX_USE_CXX11_ABI=$ABI -DNNDET_BUILT_FOR="\"$VERSION $SOABI\"" -I"$PYINC" -isystem "$TORCH/include" -isystem "$TORCH/include/torch/csrc/api/include" \
      host_lists.cpp -o nndet_host.so -L"$TORCH/lib" -ltorch_python -ltorch_cpu -lc10 -Wl,-rpath,"$TORCH/lib" && echo "$HOST" > _obj/host_for &
    pids+=($!)
  fi
fi
rc=0
for p in "${pids[@]}"; do wait $p || rc=1; done
[ $rc -eq 0 ] || { echo "compile failed"; exit 1; }
[ -z "$ASM_DIR" ] || { echo "ISA in $ASM_DIR"; exit 0; }
$HIPCC --offload-arch=gfx950 -shared -fPIC -Wl,--no-undefined -o libnndet_amd.so _obj/*.o
echo "built $(pwd)/libnndet_amd.so"
