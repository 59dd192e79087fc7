#!/bin/sh
# Build libgoib2d.so for sm_100a (the engine and the policy operators), and beside it libgoib2d_rotcheck.so (the
# rot_of self-check the GPU tests run). __graft_entry__.build() runs this script. The engine's floats follow the
# reference operation by operation (no contraction); the policy operators are compared within tolerances and keep
# fused multiply-adds. The translation units compile side by side.
set -e
cd "$(dirname "$0")"
OUT=${1:-../goib2d/libgoib2d.so}
BASE="-gencode arch=compute_100a,code=sm_100a -O3 -lineinfo -std=c++17 -Xcompiler -fPIC"
FLAGS="$BASE -fmad=false -prec-div=true -prec-sqrt=true -ftz=false"
nvcc $FLAGS -c step.cu -o step.o & PIDS=$!
nvcc $FLAGS -c api.cu -o api.o & PIDS="$PIDS $!"
for f in delta_step delta_forward delta_backward clip; do
  nvcc $BASE -c $f.cu -o $f.o & PIDS="$PIDS $!"
done
nvcc $FLAGS -shared -o "$(dirname "$OUT")/libgoib2d_rotcheck.so" rot_check.cu & PIDS="$PIDS $!"
for p in $PIDS; do wait $p; done
nvcc -gencode arch=compute_100a,code=sm_100a -shared -o "$OUT" step.o api.o delta_step.o delta_forward.o delta_backward.o clip.o
rm -f step.o api.o delta_step.o delta_forward.o delta_backward.o clip.o
