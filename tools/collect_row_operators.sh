#!/bin/bash
# profiles/row_operators_kernel_stats.txt: kernel times of the row operators at the sizes of perf/operators.py, counters of those that take longest
# (one run each: a run holds few counters), and the card's rates.  From the repository's root, with a GPU: tools/collect_row_operators.sh FOLDER, which
# takes the runs' raw output; the result is on stdout.
set -e
O=${1:?a folder for the runs}
mkdir -p $O
export TMPDIR=/tmp
run() {   # case, kind, profiler's arguments (the profiler may end with 139 when all is done and written: the calls' last line counts then)
  local n=$1 kind=$2 rc=0
  shift 2
  timeout -s KILL 90 rocprofv3 "$@" --mangled-kernels -d $O/$n.$kind -o t --output-format csv -- python3 tools/row_operators_profile.py calls $n > $O/$n.$kind.log 2>&1 || rc=$?
  if [ $rc != 0 ] && ! { [ $rc = 139 ] && grep -q "^done" $O/$n.$kind.log; }; then
    tail -3 $O/$n.$kind.log >&2
    exit $rc
  fi
  echo "$n $kind" >&2
}
for n in norm_rows_small norm_rows_block norm_map_serve norm_map_train rows_append rows_token rows_table rows_heads linear_vertex linear_tokens linear_block linear_prompt; do
  run $n trace --kernel-trace
done
for n in norm_rows_block norm_map_serve norm_map_train rows_table rows_heads linear_tokens linear_block linear_prompt; do
  run $n a --kernel-trace --pmc SQ_INSTS_VALU SQ_INSTS_VMEM_RD SQ_INSTS_VMEM_WR SQ_INSTS_LDS SQ_WAVES SQ_WAVE_CYCLES SQ_WAIT_ANY SQ_LDS_BANK_CONFLICT GRBM_GUI_ACTIVE
  run $n b --kernel-trace --pmc FETCH_SIZE
  run $n c --kernel-trace --pmc WRITE_SIZE
done
for n in linear_tokens linear_block linear_prompt; do
  run $n d --kernel-trace --pmc SQ_VALU_MFMA_BUSY_CYCLES SQ_INSTS_MFMA SQ_LDS_IDX_ACTIVE GRBM_GUI_ACTIVE
done
echo "Kernels of the row operators on one MI355X: rocprofv3 --kernel-trace, 12 calls over three sets of operands; us, median and minimum.  Below them counters (rocprofv3"
echo "--pmc, median of 12 launches): FETCH_SIZE (which counts half of the bytes here) and WRITE_SIZE in KB, SQ_VALU_MFMA_BUSY_CYCLES summed over 1024 SIMDs, GRBM_GUI_ACTIVE over 8 XCDs."
echo
python3 tools/row_operators_profile.py table $O
echo
echo "The card's rates in the same call:"
tools/micro/stream_copy | grep -e hipMemcpy -e "one float4"
tools/micro/mfma_i8_rate
