#!/bin/bash
# measurement aid (build container): build a variant of the library next to the shipped one, never over it.
#   tools/mkvariant.sh <name> [extra hipcc flags ...]     -> fair_marl_amd/csrc/variants/libfmarl_<name>.so  (working tree)
#   REV=<git rev> tools/mkvariant.sh <name> [flags ...]    -> the same from a revision's sources (must have today's C-ABI)
# Variants are git-ignored (*.so) but travel to the GPU box; select one with FMARL_LIB=<path> (fair_marl_amd/_lib.py).
set -e
R=$(cd "$(dirname "$0")/.." && pwd)
NAME=$1; shift
SRC=$R
if [ -n "$REV" ]; then
  SRC=/tmp/variant_src_$NAME; rm -rf $SRC; mkdir -p $SRC
  (cd $R && git archive $REV fair_marl_amd/csrc include | tar -x -C $SRC)
fi
mkdir -p $R/fair_marl_amd/csrc/variants
cd $SRC/fair_marl_amd/csrc
OBJS=
for U in libfmarl fmarl_memory fmarl_block fmarl_actions; do   # (a revision from before the policy operators has the first only)
  [ -f $U.hip ] || continue
  FLAGS=; [ $U = libfmarl ] && FLAGS="-ffp-contract=off -mllvm -disable-machine-licm"
  /opt/rocm/bin/hipcc --offload-arch=gfx950 -O3 -std=c++17 -Xclang -target-feature -Xclang -packed-fp32-ops $FLAGS -fPIC "$@" -c -o /tmp/variant_${NAME}_$U.o $U.hip
  OBJS="$OBJS /tmp/variant_${NAME}_$U.o"
done
/opt/rocm/bin/hipcc --offload-arch=gfx950 -shared -fPIC -o $R/fair_marl_amd/csrc/variants/libfmarl_$NAME.so $OBJS
echo "built fair_marl_amd/csrc/variants/libfmarl_$NAME.so from ${REV:-the working tree} $*"
