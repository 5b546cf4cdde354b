#!/bin/bash
# Build an experiment variant of libdoko_amd.so: tools/build_variant.sh <name> [-DFLAG=...]
# -> master_doko_reinforcement_learning_amd/libdoko_amd_<name>.so (A/B with tools/ab_inproc.py)
set -eu
P=master_doko_reinforcement_learning_amd
name=$1; shift
O=$(mktemp -d)
trap 'rm -r "$O"' EXIT
FLAGS="--offload-arch=gfx950 -O3 -std=c++17 -fPIC -Xclang -target-feature -Xclang -packed-fp32-ops"   # no packed f32 instructions
/opt/rocm/bin/hipcc $FLAGS -c -o "$O/net_train.o" $P/csrc/net_train.hip
/opt/rocm/bin/hipcc $FLAGS -ffp-contract=off -shared "$@" -o $P/libdoko_amd_$name.so $P/csrc/doko_amd.hip "$O/net_train.o"
