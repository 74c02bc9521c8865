# The counter passes behind `roofline.traffic` of the bench line, on the tree's kernel sources: FETCH_SIZE and WRITE_SIZE of a few
# training steps, each in a run of its own.  Leaves traffic.json and pmc_hbm.md in the folder that it is given; traffic.json goes to
# profiles/.  To be run again after any change to a kernel source: bench.py withholds figures taken on others.
#   bash tools/run_gpu_traffic.sh FOLDER
export TMPDIR=/tmp ADVOC_WGRAD_STREAM=0
OUT=${1:?folder}; mkdir -p $OUT
CMD="python3 bench.py --steps 3 --warmup 1 --no-cpu-baseline --train-only --prof-steps 0"
timeout -s KILL 170 rocprofv3 --kernel-trace --pmc FETCH_SIZE --output-format csv -d $OUT/fetch -- $CMD > $OUT/fetch.log 2>&1 &&
timeout -s KILL 170 rocprofv3 --kernel-trace --pmc WRITE_SIZE --output-format csv -d $OUT/write -- $CMD > $OUT/write.log 2>&1 &&
python3 tools/pmc_summary.py $(ls $OUT/fetch/*/*counter_collection.csv | head -1) $(ls $OUT/write/*/*counter_collection.csv | head -1) \
  --json $OUT/traffic.json > $OUT/pmc_hbm.md
rc=$?; tail -qn 2 $OUT/fetch.log $OUT/write.log | cut -c1-200; exit $rc
