#!/bin/bash
cd $GRAFT_REPO_ROOT
set -o pipefail
timeout -k 10 400 python -u -m pytest -q -x --timeout 200 --timeout-method thread tests/test_fused_dense.py > gpurun_out/r04ac_tests.log 2>&1 || { tail -20 gpurun_out/r04ac_tests.log; exit 1; }
tail -1 gpurun_out/r04ac_tests.log
