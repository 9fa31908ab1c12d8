#!/bin/bash
# diagnostics build of libmbhip (intra-kernel marks): mockingbird_amd/libmbhip_diag.so.  Sources and flags are the library's own, plus the marks.
set -e
cd "$(dirname "$0")/../mockingbird_amd/csrc"
HIPCC=${HIPCC:-/opt/rocm/bin/hipcc}
FLAGS=$(python3 -c 'import sys; sys.path.insert(0, ".."); import build; print(*build.FLAGS)')
SOURCES=$(python3 -c 'import sys; sys.path.insert(0, ".."); import build; print(*build.SOURCES)')
tmp=$(mktemp -d)
trap 'rm -rf "$tmp"' EXIT
objs=""
pids=""
for f in $SOURCES; do
  $HIPCC $FLAGS -DMB_TRACE_MARKS -c $f -o $tmp/${f%.hip}.o &
  pids="$pids $!"
  objs="$objs $tmp/${f%.hip}.o"
done
for p in $pids; do wait $p; done
$HIPCC -shared -fPIC --offload-arch=gfx950 -o ../libmbhip_diag.so $objs
echo built ../libmbhip_diag.so
