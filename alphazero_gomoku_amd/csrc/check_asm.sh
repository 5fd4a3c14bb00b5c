#!/bin/sh
# check_asm.sh FILE...: fails when a device assembly file is missing, empty of kernels, or holds a two-wide float32
# instruction (v_pk_fma_f32 / v_pk_mul_f32 / v_pk_add_f32); names the kernel and the instruction.
[ $# -gt 0 ] || { echo "check_asm.sh: no device assembly to check" >&2; exit 1; }
for asm in "$@"; do
    grep -q "^[ 	]*\.amdhsa_kernel" "$asm" 2>/dev/null || { echo "check_asm.sh: no kernels in $asm" >&2; exit 1; }
    bad="$(awk '/^_Z[^ ]*:/ { fn = $1 } /v_pk_(fma|mul|add)_f32/ { print fn " " $0 }' "$asm" | head -5)"
    [ -z "$bad" ] || { echo "$bad" >&2; echo "check_asm.sh: two-wide float32 instructions in $asm (see above)" >&2; exit 1; }
done
