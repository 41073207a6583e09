"""Profiles of the row operators at the sizes of perf/operators.py (``tools/collect_row_operators.sh`` runs both steps):
``calls NAME`` makes twelve calls of one case over three sets of operands, for a profiler to watch; ``table DIR`` prints what its runs left under DIR/NAME.*."""
import collections
import csv
import glob
import os
import re
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))


def calls(name):
    import torch
    from perf import operators
    operators.own = True
    case, = (c for c in operators.listed() if c["name"] == name)
    states = [operators.prepare(case, seed) for seed in range(3)]
    torch.cuda.synchronize()
    for i in range(12):
        operators.run(states[i % 3])
    torch.cuda.synchronize()
    print("done", flush=True)


def short(kernel):
    """``k_gn_stats<bfloat16, 8, false>`` of a mangled name (demanglers do not know its 16-bit types); None: not one of the row operators' kernels."""
    m = re.match(r"_Z\d+(k_(?:gn|quant|dequant|i8)_[a-z_]*)(?:I(DF16b|DF16_|f)((?:L[ib]\d+E)*))?", kernel)
    if not m:
        return None
    if not m.group(2):
        return m.group(1)
    args = [v if k == "i" else ("false", "true")[int(v)] for k, v in re.findall(r"L([ib])(\d+)E", m.group(3))]
    return "%s<%s>" % (m.group(1), ", ".join([{"DF16b": "bfloat16", "DF16_": "float16", "f": "float"}[m.group(2)]] + args))


def table(root):
    from perf import operators
    for case in operators.listed():
        times, counters = collections.defaultdict(list), collections.defaultdict(lambda: collections.defaultdict(list))
        for f in glob.glob("%s/%s.*/**/*.csv" % (root, case["name"]), recursive=True):
            for r in csv.DictReader(open(f)):
                k = short(r.get("Kernel_Name", ""))
                if k and f.endswith("counter_collection.csv"):
                    counters[k][r["Counter_Name"]].append(float(r["Counter_Value"]))
                elif k and f.endswith("kernel_trace.csv") and "/%s.trace/" % case["name"] in f:
                    times[k].append((int(r["End_Timestamp"]) - int(r["Start_Timestamp"])) / 1e3)
        print("%s  (%s)" % (case["name"], ", ".join("%s %s" % kv for kv in case.items() if kv[0] not in ("name", "op"))))
        for k, v in sorted(times.items(), key=lambda t: -sum(t[1])):
            v.sort()
            print("  %9.2f %9.2f   %s" % (v[len(v) // 2], v[0], k))
        for k, of in counters.items():
            print("    %s" % k)
            for c, v in sorted(of.items()):
                v.sort()
                print("      %-26s %.4g" % (c, v[len(v) // 2]))


if __name__ == "__main__":
    {"calls": calls, "table": table}[sys.argv[1]](sys.argv[2])
