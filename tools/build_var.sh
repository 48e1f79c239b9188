#!/bin/bash
# Build the working tree's library with extra study defines for same-box A/B runs:
#   bash tools/build_var.sh NAME "-DWF_X -DWF_Y"  ->  wrinklefree-inference-engine_amd/lib/libwfbitnet_NAME.so
set -eu
exec bash "$(dirname "$0")/build_variant.sh" "$1" ${2:-}
