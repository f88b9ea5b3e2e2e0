#!/bin/bash
# 128-column default: 1x1 + node tests, bench, timeline
set -o pipefail
cd $GRAFT_REPO_ROOT
O=gpurun_out/r06v; mkdir -p $O
timeout -k 10 600 python -u -m pytest -x -q --timeout 200 --timeout-method thread tests/test_conv1x1_bn.py tests/test_bottleneck_block.py -m gpu > $O/tests.log 2>&1 || { echo "tests rc=$?"; tail -15 $O/tests.log; exit 1; }
tail -1 $O/tests.log
timeout -k 10 300 python bench.py > $O/bench.log 2>&1 || { tail -5 $O/bench.log; exit 1; }
tail -1 $O/bench.log | cut -c1-200
bash tools/gpu_r06e.sh r06v_tl > /dev/null || exit 1
