#!/bin/bash
# kernel trace and counters of the large cases of tools/operators_times.py:
#   bash tools/prof_operators.sh <folder for the results, new>
set -e
root=$(pwd)
mkdir "$1"
out=$(cd "$1" && pwd)
cd /tmp
export TMPDIR=/tmp
run="python3 $root/tools/operators_times.py --calls"
cases=("norm forward 16384 x 4096 bf16" "norm backward 16384 x 4096 bf16" "norm forward 4096 x 16384 bf16" "norm backward 4096 x 16384 bf16"
       "distill forward 4096 x 32768 bf16, 64 listed, with the rest" "distill backward 4096 x 32768 bf16" "quantise 12288 x 4096 bf16"
       "linear 16 x 12288 x 4096 bf16" "linear 1024 x 4096 x 4096 bf16" "gradient 1024 x 4096 x 4096 bf16" "bias gradient 1024 x 4096 bf16"
       "product 8192 x 8192 x 8192 bf16")
timeout -k 10 120 rocprofv3 --kernel-trace --stats -d "$out" -o ops --output-format csv -- $run 20 "${cases[@]}" > "$out/out.txt" 2> "$out/err.txt"
pass() {
    timeout -s KILL 60 rocprofv3 --pmc "${@:2}" -d "$out/$1" -o c --output-format csv -- $run 4 "${cases[@]}" >> "$out/out.txt" 2>> "$out/err.txt"
    echo "pass $1 done"
}
pass c1 FETCH_SIZE
pass c2 WRITE_SIZE
pass c3 SQ_BUSY_CYCLES SQ_WAVE_CYCLES SQ_INSTS_VALU SQ_VALU_MFMA_BUSY_CYCLES SQ_INSTS_LDS SQ_LDS_BANK_CONFLICT SQ_WAIT_INST_LDS SQ_ACTIVE_INST_VALU
pass c4 SQ_WAIT_ANY SQ_WAIT_INST_ANY SQ_ACTIVE_INST_LDS SQ_ACTIVE_INST_ANY SQ_LDS_IDX_ACTIVE GRBM_GUI_ACTIVE
python3 "$root/tools/operators_profile.py" "$out" > "$out/trace.txt"
cat "$out/trace.txt"
