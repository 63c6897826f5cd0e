#!/bin/bash
# round 6, visit 6: the issue-priority A/B of the two waves of a SIMD, the
# shard sizes with the tuned top-segment weight
O=gpurun_out/r6
mkdir -p $O
: > $O/v6_prio.jsonl
for rep in 1 2; do
  timeout 200 python scripts/r6/shard_time.py default_$rep 10000 5000 >> $O/v6_prio.jsonl 2>> $O/v6_prio.err
  HIPADJ_LIBRARY=$PWD/scripts/r6/libhipadj_prio0.so timeout 200 python scripts/r6/shard_time.py prio_toggle_every_block_$rep 10000 5000 >> $O/v6_prio.jsonl 2>> $O/v6_prio.err
  HIPADJ_LIBRARY=$PWD/scripts/r6/libhipadj_prio2.so timeout 200 python scripts/r6/shard_time.py prio_toggle_every_4_blocks_$rep 10000 5000 >> $O/v6_prio.jsonl 2>> $O/v6_prio.err
done
cut -c1-150 $O/v6_prio.jsonl
timeout 200 python scripts/r6/shard_time.py tuned_wtop 640 1250 2500 5000 10000 > $O/v6_shard_defaults.jsonl 2> $O/v6_shard.err
cut -c1-150 $O/v6_shard_defaults.jsonl
