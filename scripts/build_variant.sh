#!/bin/bash
# Builds a variant of libtrag.so with extra compiler flags for some of its files:
#   scripts/build_variant.sh <name> [-f "<file.hip> ..."] [-DQS_FLUSH_MIN=8 ...]  ->  trueno-rag_amd/lib_var/<name>/libtrag.so
# (run a bench against it with TRAG_LIB=<that path>). Default files: the two prefilter files; the other
# objects come from trueno-rag_amd/lib.
set -e
ROOT=$(cd "$(dirname "$0")/.." && pwd)
N="$1"; shift
FILES="trag_qstat.hip trag_bf16.hip"
if [ "$1" = "-f" ]; then FILES="$2"; shift 2; fi
OUT=$ROOT/trueno-rag_amd/lib_var/$N
mkdir -p $OUT
cd $ROOT/trueno-rag_amd/csrc
# flags and objects are the library's own, as its Makefile has them
FLAGS=$(make -s print-HIPFLAGS)
LIST=$(make -s print-OBJS)
for F in $FILES; do rm -f $OUT/${F%.hip}.o; /opt/rocm/bin/hipcc $FLAGS "$@" -c $F -o $OUT/${F%.hip}.o & done
wait
for F in $FILES; do [ -f $OUT/${F%.hip}.o ] || { echo "compile of $F failed: no variant built"; rm -f $OUT/libtrag.so; exit 1; }; done
OBJS=""
for O in $LIST; do
  B=$(basename $O)
  if [ -f $OUT/$B ]; then OBJS="$OBJS $OUT/$B"; else OBJS="$OBJS $O"; fi
done
/opt/rocm/bin/hipcc --offload-arch=gfx950 -shared -o $OUT/libtrag.so $OBJS -ldl
echo built $OUT/libtrag.so
