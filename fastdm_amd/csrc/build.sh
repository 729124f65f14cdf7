#!/bin/bash
# Build libfastdm_amd.so for gfx950 (cross-compiles without a GPU).
#   build.sh                                   the product library -> fastdm_amd/_lib/   (NO extra flags accepted there)
#   FDM_OUT=tools/micro/_ab/<name> build.sh -DX  an A/B variant with extra hipcc flags -> its own directory, never _lib/
# The library carries its own provenance: fdm_source_digest() (content digest of everything it is built from, the manifest
# rule of _native.current_source_digest) and fdm_build_flags() (the extra flags, "" for the product).  No stamp file.
# env: FDM_SKIP_AUDIT=1 builds without the register audits; FDM_BUILD_UNITS="capi elementwise" builds a partial library
# (tests of this script only; recorded in the flags string, so it can never pass for the product).
set -e
HERE="$(cd "$(dirname "$0")" && pwd)"
PRODUCT_OUT="$(cd "$HERE/.." && pwd)/_lib"
OUT="${FDM_OUT:-$PRODUCT_OUT}"
mkdir -p "$OUT"
OUT="$(cd "$OUT" && pwd)"
HIPCC="${HIPCC:-/opt/rocm/bin/hipcc}"
EXTRA="$*"
UNITS="${FDM_BUILD_UNITS:-elementwise gemm attention attention_window decoder capi}"
[ -n "$FDM_BUILD_UNITS" ] && EXTRA="$EXTRA [units: $FDM_BUILD_UNITS]"
[ -n "$FDM_SKIP_AUDIT" ] && EXTRA="$EXTRA [no audit]"
EXTRA="${EXTRA# }"
if [ "$OUT" = "$PRODUCT_OUT" ] && [ -n "$EXTRA" ]; then
  echo "build.sh: extra flags / partial builds ('$EXTRA') never go into $PRODUCT_OUT: set FDM_OUT=tools/micro/_ab/<name>" >&2
  exit 2
fi
FLAGS="--offload-arch=gfx950 -O3 -std=c++17 -fPIC -ffp-contract=off -Wno-unused-result $*"

# gemm_p4_kernel's body is generated assembly.  The committed gemm_p4_body_*.inc are what gets compiled; when python3 is there
# the generator must reproduce them byte for byte (a stale body under a fresh generator fails the build instead of shipping).
if command -v python3 > /dev/null 2>&1; then
  python3 "$HERE/gen_gemm_p4.py" --check || { echo "build.sh: committed gemm_p4_body_*.inc differ from gen_gemm_p4.py's output (run: python3 $HERE/gen_gemm_p4.py)" >&2; exit 1; }
fi

# source digest: sha256 over the manifest "<sha256 of file>  <basename>\n" of csrc/*.{hip,h,sh,inc,py} + include/fastdm_amd.h,
# basenames in C order (fastdm_amd/_native.py:current_source_digest computes the same thing)
digest_manifest() {
  for f in "$HERE"/*.hip "$HERE"/*.h "$HERE"/*.sh "$HERE"/*.inc "$HERE"/*.py "$HERE/../../include/fastdm_amd.h"; do
    [ -f "$f" ] && printf '%s %s\n' "$(basename "$f")" "$f"
  done | LC_ALL=C sort | while read -r base path; do
    printf '%s  %s\n' "$(sha256sum < "$path" | cut -d' ' -f1)" "$base"
  done
}
DIGEST="$(digest_manifest | sha256sum | cut -d' ' -f1)"
cat > "$OUT/build_info.h" <<EOF
// generated by build.sh
#define FDM_SOURCE_DIGEST "$DIGEST"
#define FDM_BUILD_FLAGS "$(printf '%s' "$EXTRA" | sed 's/\\/\\\\/g; s/"/\\"/g')"
EOF

pids=()
# attention.hip: the hand-placed MFMA gaps of attn_fwd64_kernel must not be re-packed by the SLP vectoriser (it merges the
# two q-blocks' row-sum chains into v_pk_add_f32 and sinks them below the tile)
# gemm.hip / attention.hip: keep the device assembly of exactly this build beside the objects (-save-temps=obj costs nothing extra);
# tools/micro/audit_{gemm,attn}_asm.sh check it for compiler-made AGPR / scratch / call instructions inside the hand-scheduled kernels
for f in $UNITS; do
  extra=""
  [ "$f" = attention ] && extra="-fno-slp-vectorize -save-temps=obj"
  [ "$f" = gemm ] && extra="-save-temps=obj -Werror=inline-asm"     # (an asm clobber list naming a reserved register is an error)
  # the decoder-side units: no packed-fp32 instructions (hipcc makes them of ordinary float code; some of their forms have given wrong results on these cards).
  # The flag also reaches the host pass, which warns that it does not know the feature: harmless
  [ "$f" = decoder ] || [ "$f" = attention_window ] && extra="-Xclang -target-feature -Xclang -packed-fp32-ops"
  # attention_window: MFMA results in vector registers also where one wave per SIMD could have accumulation registers too (a softmax reads every one of
  # them: one token, window 4096, 32/8 heads x 128: 11.0 -> 10.0 us)
  [ "$f" = attention_window ] && extra="$extra -mllvm -amdgpu-mfma-vgpr-form=1"
  [ "$f" = capi ] && extra="-I$OUT -DFDM_HAVE_BUILD_INFO"
  "$HIPCC" $FLAGS $extra -c "$HERE/$f.hip" -o "$OUT/$f.o" &
  pids+=($!)
done
for p in "${pids[@]}"; do wait "$p"; done
objs=()
for f in $UNITS; do objs+=("$OUT/$f.o"); done
for f in gemm attention; do   # (best effort: the audit falls back to compiling if the file is not there)
  [ -f "$OUT/$f-hip-amdgcn-amd-amdhsa-gfx950.s" ] && mv -f "$OUT/$f-hip-amdgcn-amd-amdhsa-gfx950.s" "$OUT/$f.gfx950.s" || rm -f "$OUT/$f.gfx950.s"
  rm -f "$OUT/$f"-hip-amdgcn-amd-amdhsa-gfx950.* "$OUT/$f"-host-x86_64-unknown-linux-gnu.* "$OUT/$f".hip-hip-amdgcn-amd-amdhsa.hipfb
done
# the hand-scheduled kernels' register audits run on exactly this build's assembly; a failing audit fails the build.
# A vendored fastdm_amd/ without tools/ (or a box without python3) builds with a warning instead.
AUDIT_DIR="$HERE/../../tools/micro"
if [ -n "$FDM_SKIP_AUDIT" ] || [ -n "$FDM_BUILD_UNITS" ]; then
  :
elif [ ! -f "$AUDIT_DIR/audit_gemm_asm.sh" ] || ! command -v python3 > /dev/null 2>&1; then
  echo "build.sh: WARNING: tools/micro/audit_*.sh or python3 not found - the register audits were NOT run on this build" >&2
else
  FDM_AUDIT_ASM="$OUT/gemm.gfx950.s" bash "$AUDIT_DIR/audit_gemm_asm.sh" > "$OUT/audit_gemm.log" 2>&1 || { cat "$OUT/audit_gemm.log"; echo "audit_gemm_asm.sh FAILED (FDM_SKIP_AUDIT=1 builds an A/B variant anyway)"; exit 1; }
  FDM_AUDIT_ASM="$OUT/attention.gfx950.s" bash "$AUDIT_DIR/audit_attn_asm.sh" > "$OUT/audit_attn.log" 2>&1 || { cat "$OUT/audit_attn.log"; echo "audit_attn_asm.sh FAILED (FDM_SKIP_AUDIT=1 builds an A/B variant anyway)"; exit 1; }
  MASKED=1 FDM_AUDIT_ASM="$OUT/attention.gfx950.s" bash "$AUDIT_DIR/audit_attn_asm.sh" > "$OUT/audit_attn_masked.log" 2>&1 || { cat "$OUT/audit_attn_masked.log"; echo "audit_attn_asm.sh (MASKED) FAILED (FDM_SKIP_AUDIT=1 builds an A/B variant anyway)"; exit 1; }
  PV8=1 FDM_AUDIT_ASM="$OUT/attention.gfx950.s" bash "$AUDIT_DIR/audit_attn_asm.sh" > "$OUT/audit_attn_pv8.log" 2>&1 || { cat "$OUT/audit_attn_pv8.log"; echo "audit_attn_asm.sh (PV8) FAILED (FDM_SKIP_AUDIT=1 builds an A/B variant anyway)"; exit 1; }
  QK8=1 FDM_AUDIT_ASM="$OUT/attention.gfx950.s" bash "$AUDIT_DIR/audit_attn_asm.sh" > "$OUT/audit_attn_qk8.log" 2>&1 || { cat "$OUT/audit_attn_qk8.log"; echo "audit_attn_asm.sh (QK8) FAILED (FDM_SKIP_AUDIT=1 builds an A/B variant anyway)"; exit 1; }
  for v in "PV8=1 MASKED=1" "QK8=1 MASKED=1"; do
    env $v FDM_AUDIT_ASM="$OUT/attention.gfx950.s" bash "$AUDIT_DIR/audit_attn_asm.sh" > "$OUT/audit_attn_quant_masked.log" 2>&1 || { cat "$OUT/audit_attn_quant_masked.log"; echo "audit_attn_asm.sh ($v) FAILED (FDM_SKIP_AUDIT=1 builds an A/B variant anyway)"; exit 1; }
  done
fi
# link under a temporary name and rename: a process that has the old library mapped (another rank, another job) keeps its inode
# instead of seeing a truncated file
TMP_SO="$OUT/.libfastdm_amd.so.$$"
"$HIPCC" --offload-arch=gfx950 -shared -fPIC -o "$TMP_SO" "${objs[@]}"
mv -f "$TMP_SO" "$OUT/libfastdm_amd.so"
echo "built $OUT/libfastdm_amd.so (source digest ${DIGEST:0:12}, flags '${EXTRA}')"
