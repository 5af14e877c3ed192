#!/bin/bash
# Build libhorizonnet_hip.so in-tree for gfx950 (cross-compiles without a GPU).
set -e
cd "$(dirname "$0")"
OUT=${HN_BUILD_OUT:-../libhorizonnet_hip.so}      # HN_BUILD_OUT / HN_BUILD_FLAGS / HN_BUILD_OBJ: throw-away measurement builds (tools/ab_lib.sh)
OBJDIR=${HN_BUILD_OBJ:-../../build/obj}
# no packed float32 instructions (v_pk_add/mul/fma_f32): hipcc makes them from ordinary float code, and some of their forms have given wrong
# results on this hardware now and then (the host pass says that it does not know the feature: harmless)
NOPK="-Xclang -target-feature -Xclang -packed-fp32-ops"
SRCS="engine.hip engine_bf16.hip train.hip conv_igemm_f32.hip conv_wgrad_f32.hip conv_wgrad_bf16.hip bn_fold.hip conv_igemm_bf16.hip conv_igemm_bf16_pp.hip conv3x3_dwr_bf16.hip conv3x3_dwr64_bf16.hip stem_pool_bf16.hip stem_pool_f32.hip elementwise.hip train_ops.hip lstm.hip lstm_wide_f32.hip lstm_bf16.hip panostretch.hip augment.hip labels.hip peaks.hip multi_job.hip layout_fit.hip probe.hip gated_recurrence.hip gated_linear.hip gated_linear_pp.hip dropout.hip"
mkdir -p $OBJDIR
compile() {      # source, object
  local f=$1 o=$2
  case $f in
    conv_igemm_bf16_pp.hip|conv3x3_dwr_bf16.hip|conv3x3_dwr64_bf16.hip|gated_linear_pp.hip)
      # these kernels count their LDS-DMA queue by hand (s_waitcnt vmcnt(n), conv_bf16_pp.h): a scratch spill is a VMEM operation the
      # count does not know about, so a build whose hand-counted kernels spill is refused, not shipped
      /opt/rocm/bin/hipcc --offload-arch=gfx950 -O3 -std=c++17 -fPIC -Wall -Wno-unused-function -Wno-pass-failed $NOPK ${HN_BUILD_FLAGS:-} -Rpass-analysis=kernel-resource-usage -c "$f" -o "$o" 2> "$o.usage" || { cat "$o.usage"; exit 1; }
      grep -v 'kernel-resource-usage' "$o.usage" >&2 || true
      python3 - "$o.usage" <<'PY' || { rm -f "$o"; exit 1; }
import re, sys
name, bad = None, []
for line in open(sys.argv[1]):
    m = re.search(r"Function Name: (\S+)", line)
    if m: name = m.group(1)
    m = re.search(r"ScratchSize \[bytes/lane\]: (\d+)", line)
    if m and int(m.group(1)) and name and ("_kernel" in name):
        bad.append((name, int(m.group(1))))
for n, b in bad: print("build.sh: %s spills %d bytes/lane of scratch (hand-counted vmcnt kernels must not)" % (n, b))
sys.exit(1 if bad else 0)
PY
      ;;
    *)
      /opt/rocm/bin/hipcc --offload-arch=gfx950 -O3 -std=c++17 -fPIC -Wall -Wno-unused-function -Wno-pass-failed $NOPK ${HN_BUILD_FLAGS:-} -c "$f" -o "$o"
      ;;
  esac
}
# an object is rebuilt where its source, a header or this script, which holds its flags, is newer
HEADERS="*.h ../../include/horizonnet_hip.h"
stale() {      # source, object
  local d
  [ -f "$2" ] || return 0
  for d in "$1" $HEADERS build.sh; do [ "$d" -nt "$2" ] && return 0; done
  return 1
}
if [ -n "${HN_BUILD_LIST:-}" ]; then      # say what would be compiled, and stop
  for f in $SRCS; do if stale "$f" "$OBJDIR/${f%.hip}.o"; then echo "$f"; fi; done
  exit 0
fi
PIDS=""
OBJS=""
for f in $SRCS; do
  o=$OBJDIR/${f%.hip}.o
  if stale "$f" "$o"; then
    compile "$f" "$o" &
    PIDS="$PIDS $!"
    if [ $(jobs -rp | wc -l) -ge ${HN_BUILD_JOBS:-8} ]; then wait -n || exit 1; fi
  fi
  OBJS="$OBJS $o"
done
for q in $PIDS; do wait $q || exit 1; done
/opt/rocm/bin/hipcc --offload-arch=gfx950 -shared -fPIC -o $OUT $OBJS
echo "built $(readlink -f $OUT)"
# an unresolved kernel stub only shows up at dlopen time: fail the build, not the first GPU call
python3 -c "import ctypes,sys; ctypes.CDLL('$(readlink -f $OUT)')" || { echo "libhorizonnet_hip.so does not load"; exit 1; }
# the sequence operators' torch side (argument checks, autograd nodes): host code over the library just built
if [ "$OUT" = ../libhorizonnet_hip.so ]; then
  EXT=../_sequence_torch.so
  if [ ! -f $EXT ] || [ sequence_torch.cpp -nt $EXT ] || [ ../../include/horizonnet_hip.h -nt $EXT ] || [ build.sh -nt $EXT ]; then
    TORCH=$(python3 -c "import os, torch; print(os.path.dirname(torch.__file__))")
    PYINC=$(python3 -c "import sysconfig; print(sysconfig.get_paths()['include'])")
    g++ -O2 -std=c++17 -fPIC -shared -Wall -Wno-unused-function -D__HIP_PLATFORM_AMD__=1 -DUSE_ROCM=1 -DTORCH_EXTENSION_NAME=_sequence_torch -DTORCH_API_INCLUDE_EXTENSION_H \
      -isystem $TORCH/include -isystem $TORCH/include/torch/csrc/api/include -isystem $PYINC -isystem /opt/rocm/include sequence_torch.cpp -o $EXT \
      -L.. -lhorizonnet_hip -L$TORCH/lib -ltorch_python -ltorch -ltorch_cpu -ltorch_hip -lc10 -lc10_hip -Wl,-rpath,'$ORIGIN'
  fi
  (cd ../.. && python3 -c "import torch; from horizonnet_amd import _sequence_torch") || { echo "_sequence_torch.so does not load"; exit 1; }
fi
