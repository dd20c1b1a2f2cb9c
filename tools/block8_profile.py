#!/usr/bin/env python3
"""Kernel times and counters of the 8-bit block products (tools/profile_block8.sh runs both under rocprofv3).

    python tools/block8_profile.py run [CASE,CASE]            20 passes of the cases of perf/operators.py (all without a list)
    python tools/block8_profile.py times TRACE.csv             least and median time of every kernel, in the order of the cases
    python tools/block8_profile.py counters COUNTERS.csv ...   mean of every counter, a kernel at a time
"""
import collections
import csv
import os
import re
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
os.chdir(ROOT)

KERNELS = r"(quantize8|restore8|set_values|few_vectors|product|split|transposed|gradient|join)_kernel"
TYPES = {"DF16b": "bf16", "DF16_": "fp16", "f": "float", "h": "8 bits"}


def short(name):
    """kernel<arguments> of a mangled or a plain name; None for kernels that are not of block8.hip"""
    m = re.match(r"_ZN4spmv\d+" + KERNELS + r"I(.*?)EEv", name)
    if m:
        args = re.findall(r"DF16b|DF16_|L[bi]\d+E|f|h", m.group(2) + "E")
        args = [TYPES.get(a) or (a[2:-1] if a[1] == "i" else "true" if a[2] == "1" else "false") for a in args]
        return f"{m.group(1)}_kernel<{', '.join(args)}>"
    m = re.match(r"(?:void )?spmv::" + KERNELS + r"(<.*?>)?\(", name)
    return f"{m.group(1)}_kernel{m.group(2) or ''}" if m else None


def run(names):
    import torch
    from perf import operators
    operators.own = True
    for case in operators.listed():
        if names and case["name"] not in names:
            continue
        state = operators.prepare(case, 1)
        torch.cuda.synchronize()
        print(case["name"], flush=True)
        for _ in range(20):
            operators.run(state)
        torch.cuda.synchronize()
        del state
    print("done", flush=True)


def times(path):
    d = collections.OrderedDict()
    for r in csv.DictReader(open(path)):
        name = short(r["Kernel_Name"])
        if name:
            key = name, int(r["Grid_Size_X"]) // int(r["Workgroup_Size_X"]), r["Grid_Size_Y"], r["Workgroup_Size_X"], r["LDS_Block_Size"]
            d.setdefault(key, []).append((int(r["End_Timestamp"]) - int(r["Start_Timestamp"])) / 1e3)
    print("Kernels of the cases in the table of 8-bit blocks, 20 calls each, in the order of the cases (tools/profile_block8.sh), us.\n"
          "workgroups: x (times y: slices of a cut sum); threads of one; bytes of LDS; least and median time.\n")
    for k, t in d.items():
        t.sort()
        print(f"{k[0]:46s} {k[1]:6d} x {k[2]:2s} threads {k[3]:4s} lds {k[4]:7s} least {t[0]:8.2f}  median {t[len(t) // 2]:8.2f}")


def counters(paths):
    d = collections.defaultdict(lambda: collections.defaultdict(list))
    for path in paths:
        for r in csv.DictReader(open(path)):
            name = short(r["Kernel_Name"])
            if name:
                d[name][r["Counter_Name"]].append(float(r["Counter_Value"]))
    print("Counters of the three products of 8192 bf16 vectors with a full 8192 x 8192 (tools/profile_block8.sh, a run a set, mean over 20 calls;\n"
          "sums over the device: GRBM_GUI_ACTIVE over 8 XCDs, SQ_VALU_MFMA_BUSY_CYCLES over 1024 SIMDs, FETCH_SIZE in KiB with 128-byte requests\n"
          "counted as 64).")
    for name, v in d.items():
        mean = {c: sum(x) / len(x) for c, x in sorted(v.items())}
        print("\n" + name)
        for c, x in mean.items():
            print(f"  {c:32s} {x:.4g}")
        print(f"  matrix pipes busy                {mean['SQ_VALU_MFMA_BUSY_CYCLES'] / 1024 / (mean['GRBM_GUI_ACTIVE'] / 8):.2f} of the cycles")


if __name__ == "__main__":
    what, rest = sys.argv[1], sys.argv[2:]
    if what == "run":
        run(rest[0].split(",") if rest else None)
    elif what == "times":
        times(rest[0])
    elif what == "counters":
        counters(rest)
    else:
        sys.exit(__doc__)
