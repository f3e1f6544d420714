# The records of the layer operators, from the repository's root on a machine with the GPU: results under OUT (default /tmp/layers_prof).
set -e
OUT=${OUT:-/tmp/layers_prof}
mkdir -p "$OUT"
{
echo "Kernel times of the layer operators: rocprofv3 --kernel-trace --stats, one section per case (scan = gated linear recurrence)."
for c in "scan step" "scan forward 128" "scan train 256" "scan train gauge" "scan forward long" "norm forward basin" "norm forward 256" "norm train 128" "norm train wide" "norm train odd" "dropout train" "dropout residual"; do
    d="$OUT/$(echo $c | tr ' ' '_')"
    timeout -k 10 60 rocprofv3 --kernel-trace --stats --output-format csv -d "$d" -- python3 profiles/layers_prof.py run "$c" 20 > "$OUT/run.log" 2>&1
    echo "== $c"
    python3 profiles/layers_prof.py stats "$d"
done
} > "$OUT/layers_kernel_stats.txt"
for k in FETCH_SIZE WRITE_SIZE; do
    timeout -s KILL 100 rocprofv3 --pmc $k --output-format csv -d "$OUT/$k" -- python3 profiles/layers_prof.py run "scan forward 128,scan train 256,norm forward 256,norm train 128,dropout train" 4 > "$OUT/run.log" 2>&1
done
python3 profiles/layers_prof.py traffic "$OUT/FETCH_SIZE" "$OUT/WRITE_SIZE" > "$OUT/layers_kernel_traffic.csv"
timeout -k 10 240 python3 -u profiles/layers_prof.py head > "$OUT/layers_head_step.txt"
