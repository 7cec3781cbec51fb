"""Kernel times and counters of the sequence operators' cases (perf/operators.py).

    rocprofv3 --kernel-trace --stats -d DIR --output-format csv -- python3 tools/sequence_ops_profile.py run 12 train_long
    rocprofv3 --pmc GRBM_GUI_ACTIVE SQ_WAVE_CYCLES SQ_WAIT_ANY SQ_WAIT_INST_ANY SQ_ACTIVE_INST_VALU SQ_VALU_MFMA_BUSY_CYCLES \\
        --kernel-trace -d DIR --output-format csv -- python3 tools/sequence_ops_profile.py run 8 train_long
    python3 tools/sequence_ops_profile.py times DIR
    python3 tools/sequence_ops_profile.py counters DIR

`run` calls the framework's operators REPS times for each named case; `times` prints the median time of each kernel, `counters` what
each launch's counters say per SIMD (256 compute units of four, eight dies that each count GRBM_GUI_ACTIVE).
"""
import collections
import csv
import glob
import importlib.util
import os
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
# the longer names first: some profilers print the 16-bit kernels' names mangled
OURS = ("fwd_rows_join_kernel", "fwd_rows_kernel", "fwd_split_kernel", "fwd_join_kernel", "dq_join_kernel", "dq_kernel", "dkv_join_kernel", "dkv_kernel",
        "dtable_kernel", "pack_kernel", "fwd_wide_kernel", "bwd_wide_kernel", "fwd_kernel", "bwd_kernel", "join_kernel")


def run(reps, names):
    import torch
    spec = importlib.util.spec_from_file_location("operators", os.path.join(ROOT, "perf", "operators.py"))
    cases = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(cases)
    cases.own = True
    for name in names:
        state = cases.prepare(next(c for c in cases.listed() if c["name"] == name), 1)
        for _ in range(reps):
            cases.run(state)
        torch.cuda.synchronize()
        print(name, flush=True)


def rows(folder, kind):
    for path in sorted(glob.glob(os.path.join(folder, "**", f"*{kind}.csv"), recursive=True)):
        with open(path) as f:
            for r in csv.DictReader(f):
                name = next((k for k in OURS if k in r["Kernel_Name"]), None)
                if name:
                    yield name, r


def micros(r):
    return (int(r["End_Timestamp"]) - int(r["Start_Timestamp"])) / 1e3


def median(values):
    return sorted(values)[len(values) // 2]


def times(folder):
    found = collections.OrderedDict()
    for name, r in rows(folder, "kernel_trace"):
        found.setdefault(name, []).append(micros(r))
    for name, t in found.items():
        print(f"{name:22s} {median(t):9.2f} us")


def shares(v):
    cycles = v["GRBM_GUI_ACTIVE"] / 8
    out = {"us": v["us"], "GHz": cycles / v["us"] / 1e3}
    for key, label, per in (("SQ_VALU_MFMA_BUSY_CYCLES", "matrix cores", cycles * 1024), ("SQ_ACTIVE_INST_VALU", "vector", cycles * 256),
                            ("SQ_WAVE_CYCLES", "waves a SIMD", cycles * 256), ("SQ_LDS_IDX_ACTIVE", "LDS busy", cycles * 256),
                            ("SQ_LDS_BANK_CONFLICT", "LDS conflicts", cycles * 256), ("SQ_WAIT_ANY", "waiting", v["SQ_WAVE_CYCLES"]),
                            ("SQ_WAIT_INST_ANY", "for a turn", v["SQ_WAVE_CYCLES"])):
        if key in v:
            out[label] = v[key] / per
    return out


def counters(folder):
    found, kernels = collections.OrderedDict(), collections.OrderedDict()
    for name, r in rows(folder, "counter_collection"):
        v = found.setdefault((name, r["Dispatch_Id"]), {"us": micros(r)})
        v[r["Counter_Name"]] = v.get(r["Counter_Name"], 0.0) + float(r["Counter_Value"])
    for (name, _), v in found.items():
        kernels.setdefault(name, []).append(shares(v))
    for name, launches in kernels.items():                   # a clock out of the chip's range: that counter missed the launch's borders
        good = [v for v in launches if 1.0 < v["GHz"] < 2.6]
        if good:
            print(f"{name:22s}", "  ".join(f"{label} {median([v[label] for v in good]):.2f}" for label in good[0]), f" ({len(good)} of {len(launches)} launches)")


if __name__ == "__main__":
    if sys.argv[1] == "run":
        run(int(sys.argv[2]), sys.argv[3:])
    else:
        {"times": times, "counters": counters}[sys.argv[1]](sys.argv[2])
