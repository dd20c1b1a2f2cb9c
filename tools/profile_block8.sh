#!/bin/bash
# Kernel times of every case of perf/operators.py, and counters of the three products of the training batch: rocprofv3 passes around
# tools/block8_profile.py.
#   tools/profile_block8.sh DIR    -> DIR/block8_kernel_times.txt, DIR/block8_counters.txt
# Each pass holds at most 8 SQ, 4 TCC, 4 TCP and 2 GRBM counters and runs under its own time limit; the script stops at the first failure.
set -e
root=$(cd "$(dirname "$0")/.." && pwd)
mkdir -p "$1"
out=$(cd "$1" && pwd)
cd /tmp && export TMPDIR=/tmp
tool=$root/tools/block8_profile.py
timeout -s KILL 150 rocprofv3 --kernel-trace --stats -M -f csv -d "$out/block8_trace" -o p -- python3 "$tool" run > "$out/block8_trace.log" 2>&1
python3 "$tool" times "$out/block8_trace/p_kernel_trace.csv" > "$out/block8_kernel_times.txt"
pass() {
    name=$1; shift
    timeout -s KILL 100 rocprofv3 --pmc "$@" --kernel-include-regex "(product|transposed|gradient)_kernel" -M -f csv -d "$out/block8_$name" -o p -- \
        python3 "$tool" run product_batch,transposed_batch,gradient_batch > "$out/block8_$name.log" 2>&1
}
pass waits SQ_BUSY_CYCLES SQ_WAVE_CYCLES SQ_VALU_MFMA_BUSY_CYCLES SQ_LDS_BANK_CONFLICT SQ_INSTS_LDS SQ_LDS_IDX_ACTIVE SQ_WAIT_INST_LDS SQ_WAIT_ANY
pass issue SQ_INSTS_VALU SQ_ACTIVE_INST_VALU SQ_INSTS_VMEM_RD SQ_ACTIVE_INST_LDS SQ_WAIT_INST_ANY GRBM_GUI_ACTIVE TCC_HIT_sum TCC_MISS_sum
pass cache TCP_TCC_READ_REQ_sum TCP_TOTAL_CACHE_ACCESSES_sum TCP_PENDING_STALL_CYCLES_sum TCP_TCR_TCP_STALL_CYCLES_sum FETCH_SIZE
python3 "$tool" counters "$out"/block8_waits/p_counter_collection.csv "$out"/block8_issue/p_counter_collection.csv "$out"/block8_cache/p_counter_collection.csv \
    > "$out/block8_counters.txt"
echo "8-bit block profile done"
