#!/bin/bash
# NIRRT* 2D, 4096 trees: sweep of the iterations per launch.  usage: scripts/nirrt_groups_sweep.sh 512 1024 2048 ...
for W in "$@"; do
NIRRT_BATCH_WINDOW=$W python bench.py --algo nirrt --trees 4096 --steps 1 --warmup 0 --no-cpu-baseline --no-ttfs --no-secondary > gpurun_out/nx_$W.json 2> gpurun_out/nx_$W.err
python - <<PY
import json
d=json.load(open("gpurun_out/nx_$W.json"))
c=d["config"]
print("window $W:", round(d["value"]/1e6,2), "M it/s step", round(d["ms_per_step"]/1e3,2), "s kernel", round(d["roofline"]["kernel_ms"]/1e3,2), "launches", c.get("launches_per_step"), c.get("host_seconds_last_step"))
PY
done
