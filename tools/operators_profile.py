"""One table per kernel from the trace and the counter passes of tools/prof_operators.sh: python tools/operators_profile.py <folder>"""
import collections
import csv
import re
import sys

folder = sys.argv[1]


def name_of(raw):
    """k_name<template arguments>, from a mangled or a demangled kernel name; None for other libraries' kernels."""
    m = re.match(r"_ZN3drm(\d+)(.*)", raw)
    if not m:
        m = re.match(r"(?:void )?drm::(k_\w+(?:<[^(]*>)?)", raw)
        # (the profiler shows the type code DF16bLi1E of one kernel as "bool _Accum, int, E")
        return m[1].replace("bool _Accum, int, E", "bf16, 1").replace("std::bfloat16_t", "bf16").replace("__bf16", "bf16").replace("_Float16", "fp16").replace("float", "fp32") if m else None
    name, rest = m[2][:int(m[1])], m[2][int(m[1]):]
    if not name.startswith("k_") or rest[:1] != "I":
        return name if name.startswith("k_") else None
    args, at = [], 1
    while rest[at] != "E":
        for pattern, show in ((r"DF16b", lambda x: "bf16"), (r"DF16_", lambda x: "fp16"), (r"f", lambda x: "fp32"), (r"Li(\d+)E", lambda x: x[1]),
                              (r"Lb(\d)E", lambda x: "yes" if x[1] == "1" else "no")):
            x = re.match(pattern, rest[at:])
            if x:
                args.append(show(x))
                at += x.end()
                break
        else:
            return raw
    return f"{name}<{', '.join(args)}>"


trace = {}
for row in csv.DictReader(open(f"{folder}/ops_kernel_stats.csv")):
    name = name_of(row["Name"])
    if name:
        trace[name] = (int(row["Calls"]), float(row["AverageNs"]) / 1e3, float(row["MinNs"]) / 1e3)
order = sorted(trace, key=lambda n: -trace[n][1])
counters = collections.defaultdict(dict)
for run in ("c1", "c2", "c3", "c4"):
    seen = collections.defaultdict(list)
    for row in csv.DictReader(open(f"{folder}/{run}/c_counter_collection.csv")):
        name = name_of(row["Kernel_Name"])
        if name:
            seen[name, row["Counter_Name"]].append(float(row["Counter_Value"]))
    for (name, counter), values in seen.items():
        counters[name][counter] = sum(values) / len(values)
print("Calls from Python, one after the other (tools/prof_operators.sh); the cases:")
for line in list(dict.fromkeys(open(f"{folder}/out.txt").read().splitlines())):
    if " x " in line:
        print("  " + line)
print("\nkernel trace, times in microseconds from the start of a kernel to its end, by itself\n")
print(f"{'kernel':58s} {'calls':>6s} {'mean':>9s} {'least':>9s}")
for n in order:
    print(f"{n:58s} {trace[n][0]:6d} {trace[n][1]:9.2f} {trace[n][2]:9.2f}")
print("""
counters per call: MiB read and written beyond the caches of the XCDs (FETCH_SIZE, WRITE_SIZE; FETCH_SIZE counts 64 bytes a request,
half of what the wide loads of these kernels ask for); share of the time that the matrix pipes are busy; share of the waves' time
spent waiting; LDS bank conflicts per LDS-active cycle
""")
print(f"{'kernel':58s} {'read':>9s} {'written':>9s} {'matrix':>7s} {'waiting':>8s} {'conflict':>9s}")
for n in order:
    v = counters.get(n)
    if not v:
        continue
    matrix = v.get("SQ_VALU_MFMA_BUSY_CYCLES", 0) / max(1, v.get("GRBM_GUI_ACTIVE", 0) / 8 * 256 * 4)
    waiting = v.get("SQ_WAIT_ANY", 0) / max(1, v.get("SQ_WAVE_CYCLES", 1))
    conflict = v.get("SQ_LDS_BANK_CONFLICT", 0) / max(1, v.get("SQ_LDS_IDX_ACTIVE", 1))
    print(f"{n:58s} {v.get('FETCH_SIZE', 0) / 1024:9.1f} {v.get('WRITE_SIZE', 0) / 1024:9.1f} {matrix:7.2f} {waiting:8.2f} {conflict:9.2f}")
