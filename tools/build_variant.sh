#!/bin/bash
# Study build of the library with extra compile flags, for same-box A/B runs (WF_BITNET_LIB=...):
#   bash tools/build_variant.sh NAME -DFLAG=VALUE ...  ->  wrinklefree-inference-engine_amd/lib/libwfbitnet_NAME.so
# The Makefile's flags and sources with these defines on top. Never the product library (lib/libwfbitnet.so is built by
# the Makefile / __graft_entry__.build()).
set -eu
cd "$(dirname "$0")/../wrinklefree-inference-engine_amd"
NAME=$1; shift
make -B -j8 BUILD="build/var_$NAME" LIB="lib/libwfbitnet_$NAME.so" DEFS="$*"
echo "built lib/libwfbitnet_$NAME.so"
