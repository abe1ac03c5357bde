"""operators_kernel_times.txt and operators_counters.txt from the files that tools/operators_profile.sh leaves.

usage: operators_tables.py RAW_DIRECTORY OUTPUT_DIRECTORY"""
import collections
import csv
import glob
import os
import re
import sys

TITLES = {
    "lm_score_8_pairs": "loss forward, 16 rows x 32128 entries x 768",
    "lm_train_32_tuples": "loss and gradients, 1088 x 32128 x 768, dw bf16",
    "1088,32128,768,f32": "loss and gradients, 1088 x 32128 x 768, dw fp32 added to",
    "lm_train_odd_vocab": "loss and gradients, 777 x 6401 x 512, dw bf16",
    "lm_contrast_512": "loss and gradients, 512 queries x 8704 documents x 768, scale 20, dw bf16",
    "lm_train_8k_tokens": "loss and gradients, 8192 x 50001 x 1024, dw bf16",
    "64,32128,768": "loss and gradients, 64 x 32128 x 768, dw bf16",
    "ckpt_300_tokens": "checkpoint written and read, 300 x 512",
    "ckpt_139k_tokens": "checkpoint written and read, 139264 x 768",
    "dw_1001_tokens": "weight gradient from a checkpoint, 512 x 2048 from 1001 tokens",
    "dw_139k_tokens": "weight gradient from a checkpoint, 2304 x 768 from 139264 tokens",
    "ln_one_token": "layer norm forward, 1 x 768 bf16, residual",
    "ln_train_odd_f32": "layer norm forward and backward, 5001 x 1023 fp32",
    "ln_train_139k_tokens": "layer norm forward and backward, 139264 x 768 bf16, residual",
}
EPILOGUES = {"0": "bf16", "9": "loss statistics", "10": "loss gradient", "11": "fp32 slabs"}
PASSES, WARM = 120, 80


def short(name):
    """A kernel's name without its argument list, template arguments in words."""
    mangled = re.match(r"_ZN12_GLOBAL__N_113ln_(fwd|bwd)_kernelI(DF16b|f)Li(\d+)ELi(\d+)ELNS_3EndE(\d)E", name)
    if mangled:                                    # (the trace leaves bf16 templates as they are)
        kind, t, team, per, end = mangled.groups()
        return f"ln_{kind}_kernel<{'bf16' if t == 'DF16b' else 'float'}, {team}, {per}, {('fits', 'laps', 'short')[int(end)]}>"
    name = name.replace("(anonymous namespace)::", "").replace("(End)0", "fits").replace("(End)1", "laps").replace("(End)2", "short")
    name = re.sub(r"^void ", "", name)
    name = re.sub(r"ln_(fwd|bwd)_kernel<bool _Accum, int, ELi(\d+)ELNS_3EndE(\d)E>.*",
                  lambda m: f"ln_{m[1]}_kernel<bf16, 16, {m[2]}, {('fits', 'laps', 'short')[int(m[3])]}>", name)
    name = name.split("(")[0]
    return re.sub(r"<(Cfg\w+, )?(false|true), (false|true), (\d+)", lambda m: f"<{m[1] or ''}{m[2]}, {m[3]}, {EPILOGUES.get(m[4], m[4])}", name)


def ours(name):
    return not any(s in name for s in ("at::native", "rocprim", "Cijk", "copyBuffer", "fillBuffer"))


def rows(path, pattern):
    for f in glob.glob(os.path.join(path, "**", pattern), recursive=True):
        with open(f) as fh:
            yield from csv.DictReader(fh)


def times(raw):
    out = [f"Kernel times of one pass of each operator case (rocprofv3 --kernel-trace, {PASSES - WARM} passes after {WARM} to warm up; us a pass, launches a pass, "
           "least and most us of a launch).", "Template names: gemm_*<A transposed, B transposed, epilogue>.", ""]
    for case, title in TITLES.items():
        t = collections.defaultdict(list)
        for r in sorted(rows(os.path.join(raw, "times", case), "*kernel_trace.csv"), key=lambda r: int(r["Start_Timestamp"])):
            if ours(r["Kernel_Name"]):
                t[short(r["Kernel_Name"])].append((int(r["End_Timestamp"]) - int(r["Start_Timestamp"])) / 1e3)
        out.append(title)
        for k, v in sorted(t.items(), key=lambda kv: -sum(kv[1])):
            v, per = v[len(v) * WARM // PASSES:], len(v) / PASSES
            out.append(f"  {sum(v) / len(v) * per:8.1f} us {per:4.1f} x  ({min(v):.1f} - {max(v):.1f})  {k}")
        out.append("")
    return out


def counters(raw):
    out = ["Counters of one launch (mean; rocprofv3 --pmc, three passes: SQ and GRBM, FETCH_SIZE, WRITE_SIZE).  MFMA work = SQ_INSTS_VALU_MFMA_MOPS_BF16 x 512;",
           "fetched = FETCH_SIZE x 2 (128-byte requests are counted as 64), written = WRITE_SIZE; LDS conflicts = SQ_LDS_BANK_CONFLICT / SQ_LDS_IDX_ACTIVE.", ""]
    for case, title in TITLES.items():
        if not os.path.isdir(os.path.join(raw, "pmc", case)):
            continue
        t = collections.defaultdict(lambda: collections.defaultdict(list))
        for r in rows(os.path.join(raw, "pmc", case), "*counter_collection.csv"):
            if ours(r["Kernel_Name"]):
                t[short(r["Kernel_Name"])][r["Counter_Name"]].append(float(r["Counter_Value"]))
        out += [title, "  %-62s %12s %12s %12s %10s %10s" % ("kernel", "MFMA GFLOP", "fetched MB", "written MB", "waves", "conflicts")]
        for k in sorted(t):
            c = {n: sum(v[len(v) // 3:]) / len(v[len(v) // 3:]) for n, v in t[k].items()}
            conflicts = "%.2f" % (c["SQ_LDS_BANK_CONFLICT"] / c["SQ_LDS_IDX_ACTIVE"]) if c.get("SQ_LDS_IDX_ACTIVE") else "-"
            out.append("  %-62s %12.1f %12.1f %12.1f %10d %10s" % (k, c.get("SQ_INSTS_VALU_MFMA_MOPS_BF16", 0) * 512 / 1e9, c.get("FETCH_SIZE", 0) * 2 * 1024 / 1e6,
                                                                    c.get("WRITE_SIZE", 0) * 1024 / 1e6, c.get("SQ_WAVES", 0), conflicts))
        out.append("")
    return out


def main(raw, target):
    for name, lines in (("operators_kernel_times.txt", times(raw)), ("operators_counters.txt", counters(raw))):
        with open(os.path.join(target, name), "w") as f:
            f.write("\n".join(lines).rstrip() + "\n")


if __name__ == "__main__":
    main(*sys.argv[1:3])
