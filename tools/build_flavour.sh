#!/bin/bash
# A diagnostic / experimental build of the whole library:
#   tools/build_flavour.sh <name> [extra hipcc flags...]  ->  pcl-augmentation_amd/libreal3daug_hip_<name>.so
# Every source is compiled afresh into a temporary directory (nothing is taken from the normal build's objects), every
# compile job is waited for by its own PID (a failed job fails the script, it does not surface as a link error), and
# r3d_level1 gets the same R3D_SRC_HASH csrc/Makefile passes, so that r3d_build_info() of the flavour names the sources it
# was built from (__graft_entry__.build() compares it with the tree when the flavour is loaded through R3D_LIB).
# Sources, headers and flags are the Makefile's; `tools/build_flavour.sh --sources` lists the sources.
set -e
cd "$(dirname "$0")/../pcl-augmentation_amd/csrc"
SRCS=$(make -s print-SRCS)
if [ "$1" = --sources ]; then echo $SRCS; exit 0; fi
name=$1; shift
HASH=$(make -s print-SRC_HASH)
HIPFLAGS=$(make -s print-HIPFLAGS)
INSERT_FLAGS=$(make -s print-INSERT_FLAGS)
T=$(mktemp -d)
trap 'rm -rf "$T"' EXIT
pids=()
for f in $SRCS; do
  extra=()
  [ $f = r3d_insert.hip ] && extra=($INSERT_FLAGS)
  [ $f = r3d_level1.hip ] && extra=("-DR3D_SRC_HASH=\"$HASH\"")
  case $f in
    *.cpp) hipcc $(make -s print-FLAGS) -c $f -o $T/${f%.*}.o & ;;
    *) hipcc $HIPFLAGS "$@" "${extra[@]}" -c $f -o $T/${f%.*}.o & ;;
  esac
  pids+=($!)
done
for p in "${pids[@]}"; do
  wait $p || { echo "build_flavour: a compile job failed" >&2; exit 1; }
done
hipcc --offload-arch=gfx950 -shared -fPIC $T/*.o -lpthread -o ../libreal3daug_hip_$name.so
ls -la ../libreal3daug_hip_$name.so
