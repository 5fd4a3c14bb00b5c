#!/bin/sh
# Builds libazgomoku.so for gfx950 (MI355X).
#  -ffp-contract=off keeps the PUCT and running-mean arithmetic in the reference's operation
#   order (no fused multiply-add).
#  -fno-slp-vectorize keeps float32 arithmetic on single-lane VALU instructions.  Left on, -O3 packs
#   adjacent multiply-adds into v_pk_fma_f32; in the kernel whose tree waves share their SIMDs with
#   matrix-dense waves such an operation, fed its x from the high dword of a register pair
#   (op_sel:[0,1,0]), came out one term short in lanes 48-55 (50-70 of 256 identical searches wrong;
#   the note at AZG_EXP_PKFC in azg_dual.hpp has the measurements).  The build FAILS when a kernel of either
#   translation unit holds any two-wide float32 instruction (check_asm.sh), whatever flag or compiler
#   version produced it.
#  -no-hip-rt leaves the HIP runtime symbols undefined: the process must hold exactly ONE HIP
#   runtime, and PyTorch ships its own libamdhip64.so.  The loader (alphazero_gomoku_amd/_lib.py)
#   loads the runtime PyTorch will use (or /opt/rocm's when PyTorch is absent) with RTLD_GLOBAL
#   before this library; a C/C++ host simply links -lamdhip64 itself.
set -e
here="$(cd "$(dirname "$0")" && pwd)"
out="$here/../libazgomoku.so"
log="$(mktemp)"
tmp="$(mktemp -d)"
trap 'rm -rf "$tmp"' EXIT
# (the device assembly is kept as a by-product of the one compilation: -save-temps, in a scratch directory)
# No translation unit may form two-wide float32 instructions at all (-packed-fp32-ops).  azg_ops.hip (the training heads'
# operators) is one of its own, compiled beside the other.
nopk="-Xclang -target-feature -Xclang -packed-fp32-ops"
( cd "$tmp" && hipcc --offload-arch=gfx950 -O3 -fno-slp-vectorize -fPIC -std=c++17 -Wall $nopk -save-temps=cwd -c "$here/azg_ops.hip" -o "$tmp/azg_ops.o" > "$tmp/ops.log" 2>&1; echo $? > "$tmp/ops.rc" ) &
ops=$!
( cd "$tmp" && hipcc --offload-arch=gfx950 -O3 -ffp-contract=off -fno-slp-vectorize -fPIC -c -std=c++17 -Wall $nopk \
    -Rpass-analysis=kernel-resource-usage -save-temps=cwd \
    "$here/azgomoku.hip" -o "$tmp/azgomoku.o" "$@" ) 2> "$log" || { cat "$log" >&2; rm -f "$log"; exit 1; }
wait $ops
# (the host pass does not know the device feature and says so: harmless)
grep -v "packed-fp32-ops" "$tmp/ops.log" >&2 || true
[ "$(cat "$tmp/ops.rc")" = 0 ] || { rm -f "$out" "$log"; exit 1; }
grep -v "packed-fp32-ops" "$log" > "$tmp/log" || true
cp "$tmp/log" "$log"
sh "$here/check_asm.sh" "$tmp"/azgomoku*gfx950.s "$tmp"/azg_ops*gfx950.s || { rm -f "$out" "$log"; exit 1; }
hipcc --offload-arch=gfx950 -fPIC -shared -no-hip-rt "$tmp/azgomoku.o" "$tmp/azg_ops.o" -o "$out" -lpthread
# compiler warnings, without the resource-usage remarks and their source excerpts
if grep -q "warning:" "$log"; then
    awk '/kernel-resource-usage/ { skip = 2; next } skip > 0 { skip--; next } { print }' "$log" >&2
fi
# The split-f16 search kernels for boards up to 8x8 run two workgroups per CU and are capped at 240
# VGPRs (azg_kernels.hpp, AZG_CAPPED_SEARCH_KERNEL), so that copy kernels can run beside them;
# this check reports a build in which the cap did not hold.
awk '/Function Name: _ZN3azg21search_kernel_f16_[678]x[678]ENS_8DevStateE/ { k = $0; sub(/.*Function Name: /, "", k); sub(/ .*/, "", k) }
     k != "" && / VGPRs: / { v = $0; sub(/.* VGPRs: /, "", v); sub(/ .*/, "", v);
         if (v + 0 > 240) printf("WARNING: %s uses %d VGPRs (> 240): copy kernels cannot run beside it\n", k, v);
         k = "" }' "$log" >&2
rm -f "$log"
echo "built $out"
