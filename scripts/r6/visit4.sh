#!/bin/bash
# round 6, visit 4: the shard sizes with the planner's grouped defaults, the whole GPU suite, a default bench run
O=gpurun_out/r6
mkdir -p $O
timeout 300 python scripts/r6/shard_time.py planner_defaults 640 1250 2500 5000 10000 20000 > $O/v4_shard_defaults.jsonl 2> $O/v4_shard_defaults.err
HIPADJ_FUSED_GROUP=0 timeout 300 python scripts/r6/shard_time.py plain_form 640 1250 2500 5000 10000 >> $O/v4_shard_defaults.jsonl 2>> $O/v4_shard_defaults.err
cut -c1-150 $O/v4_shard_defaults.jsonl
( time timeout 1100 python -m pytest tests -x -q -m gpu -p no:cacheprovider ) > $O/v4_gpu_suite.log 2>&1
tail -n 6 $O/v4_gpu_suite.log
timeout 600 python bench.py --steps 20 --warmup 5 > $O/v4_bench.json 2> $O/v4_bench.err; cp bench_extras.json $O/v4_bench_extras.json
cat $O/v4_bench.json | cut -c1-1200
