#!/bin/bash
# Build the library of a git revision as a study variant for same-box A/B runs:
#   bash tools/build_rev.sh REV NAME  ->  wrinklefree-inference-engine_amd/lib/libwfbitnet_NAME.so
# The revision's sources with the working tree's flags.
set -eu
cd "$(dirname "$0")/.."
REV=$1; NAME=$2
T=$(mktemp -d)
trap 'rm -rf "$T"' EXIT
git archive "$REV" wrinklefree-inference-engine_amd/csrc include | tar -x -C "$T"
make -B -j8 -C wrinklefree-inference-engine_amd CSRC="$T/wrinklefree-inference-engine_amd/csrc" INCLUDE="$T/include" \
  BUILD="$T/build" LIB="lib/libwfbitnet_$NAME.so"
echo "built lib/libwfbitnet_$NAME.so from $REV"
