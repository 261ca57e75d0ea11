#!/bin/bash
# Ablation builds of the two VALU-heavy front-end kernels (measurement only, never shipped): a patched COPY of
# csrc/gs_frontend.hip (tools/ubench/frontend_ablation.patch) compiled with -DGS_ABLATE_KEYS=1|2|3 (gs_make_keys: stop after
# the scans / after the record loads and box arithmetic / walk without stores) and -DGS_ABLATE_PRE=1|2|3 (gs_preprocess: no
# colour / no bin walk / neither), linked with the tree's other objects into variants/libgsplat_hip_abl_<tag>.so.
# Time them with tools/ablate_probe.py (GS_LIB_PATH=...).  The tree's sources (and their profile hash) stay untouched.
set -e
ROOT=$(cd "$(dirname "$0")/.." && pwd)
SRC=$ROOT/taichi_3d_gaussian_splatting_amd/csrc
OUT=${GS_VARIANTS_DIR:-$ROOT/variants}
TMP=$(mktemp -d)
mkdir -p $TMP/pkg $OUT
cp -rp $SRC $TMP/pkg/csrc && cp -rp $ROOT/include $TMP/include     # (with their times: what is built there stays built here)
patch -s $TMP/pkg/csrc/gs_frontend.hip $ROOT/tools/ubench/frontend_ablation.patch
cd $TMP/pkg/csrc
for spec in "k1:-DGS_ABLATE_KEYS=1" "k2:-DGS_ABLATE_KEYS=2" "k3:-DGS_ABLATE_KEYS=3" "p1:-DGS_ABLATE_PRE=1" "p2:-DGS_ABLATE_PRE=2" "p3:-DGS_ABLATE_PRE=3"; do
    tag=${spec%%:*}; flags=${spec#*:}
    rm -f gs_frontend.o
    make -s -j8 EXTRA="$flags" ../libgsplat_hip.so
    cp ../libgsplat_hip.so $OUT/libgsplat_hip_abl_$tag.so
    echo "built $tag ($flags)"
done
rm -rf $TMP
