#!/bin/bash
# Kernel times and counters of the operators' cases: writes operators_kernel_times.txt and operators_counters.txt into $1
# (tools/operators_tables.py makes them from rocprofv3's files).  Run with a GPU, from the repository's root, on a built tree.
set -e
out=${1:?usage: operators_profile.sh DIRECTORY}
here=$PWD
raw=$(mktemp -d)
mkdir -p "$out"
out=$(cd "$out" && pwd)
export TMPDIR=/tmp
cd /tmp
times="lm_score_8_pairs lm_train_32_tuples 1088,32128,768,f32 lm_train_odd_vocab lm_contrast_512 lm_train_8k_tokens 64,32128,768 ckpt_300_tokens ckpt_139k_tokens
       dw_1001_tokens dw_139k_tokens ln_one_token ln_train_odd_f32 ln_train_139k_tokens"
for c in $times; do
    timeout -s KILL 100 rocprofv3 --kernel-trace -d "$raw/times/$c" -o p --output-format csv -- python3 "$here/tools/operators_pass.py" "$c" 120 > "$raw/log" 2>&1 \
        || { tail -5 "$raw/log"; exit 1; }
    echo "traced $c"
done
for c in lm_train_32_tuples lm_train_8k_tokens dw_139k_tokens ln_train_139k_tokens ckpt_139k_tokens; do
    for set in "SQ_WAVES SQ_BUSY_CYCLES SQ_INSTS_VALU_MFMA_MOPS_BF16 SQ_LDS_BANK_CONFLICT SQ_LDS_IDX_ACTIVE SQ_ACTIVE_INST_VALU SQ_ACTIVE_INST_LDS GRBM_GUI_ACTIVE" FETCH_SIZE WRITE_SIZE; do
        timeout -s KILL 60 rocprofv3 --pmc $set -d "$raw/pmc/$c/${set%% *}" -o p --output-format csv -- python3 "$here/tools/operators_pass.py" "$c" 6 > "$raw/log" 2>&1 \
            || { tail -5 "$raw/log"; exit 1; }
    done
    echo "counted $c"
done
cd "$here"
python3 tools/operators_tables.py "$raw" "$out"
