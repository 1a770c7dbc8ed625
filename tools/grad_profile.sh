#!/bin/bash
# rocprofv3 passes over the cases of perf/operators.py (tools/grad_profile.py), from the repo root.
# Each set of counters in a run of its own.
#   bash tools/grad_profile.sh DIR
out=$(realpath -m "${1:?where the results go}")
prog=$PWD/tools/grad_profile.py
mkdir -p "$out"
cd /tmp && export TMPDIR=/tmp
timeout -s KILL 120 rocprofv3 --kernel-trace --stats -f csv -d "$out" -o kt -- python3 "$prog" passes 60 && \
timeout -s KILL 60 rocprofv3 --pmc FETCH_SIZE -f csv -d "$out" -o fetch -- python3 "$prog" passes 6 && \
timeout -s KILL 60 rocprofv3 --pmc WRITE_SIZE -f csv -d "$out" -o write -- python3 "$prog" passes 6 && \
timeout -s KILL 60 rocprofv3 --pmc SQ_ACTIVE_INST_VALU SQ_WAVE_CYCLES -f csv -d "$out" -o sq -- python3 "$prog" passes 6
