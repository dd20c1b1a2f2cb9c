"""The pipelined kernels of 8-bit blocks as they are built: at every step's barrier, have the loads into LDS that the step reads
arrived?

A step waits until at most N of its wave's loads are outstanding, N being counted in the source.  Whether that covers the
right loads depends on the order and number of loads that the compiler leaves: a load whose result nothing uses is dropped,
and one moved across another changes which are the last N.  So the built code is walked, along every path through its
branches: loads enter a queue, a wait for N drops all but the last N from it (they return in order), and at the wait of step
k no load into LDS of a stage up to k may be left.
"""
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.abspath(os.path.join(os.path.dirname(__file__), ".."))
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
STEPS = 14                       # steps to walk: several rounds of up to 4 stages, and what is left after them

pytestmark = pytest.mark.skipif(not os.path.exists(HIPCC), reason="needs hipcc")


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    """name -> lines of assembly of the pipelined kernels"""
    out = tmp_path_factory.mktemp("block8") / "block8.s"
    flags = re.search(r"^CXXFLAGS\s*=\s*(.*?[^\\])$", open(os.path.join(ROOT, "spmv_amd/csrc/Makefile")).read(), re.S | re.M).group(1)
    flags = flags.replace("\\\n", " ").replace("$(ARCH)", "gfx950").replace("$(ROOT)", ROOT).replace("$(HERE)", os.path.join(ROOT, "spmv_amd/csrc")).split()
    assert not any("$" in f for f in flags), flags
    subprocess.run([HIPCC, *[f for f in flags if f != "-fPIC"], "-w", "-S", "--offload-device-only", os.path.join(ROOT, "spmv_amd/csrc/block8.hip"), "-o", str(out)],
                   check=True, stderr=subprocess.DEVNULL)
    text = out.read_text()
    found = {m.group(1): m.group(2).split("\n") for m in
             re.finditer(r"^(_ZN4spmv\d+(?:product|transposed|gradient)_kernel\S*):(.*?)\n\s+\.section", text, re.S | re.M)}
    assert len(found) > 30
    return found


def _loads_per_stage(name):
    kind, args = re.match(r"_ZN4spmv\d+(\w+?)_kernelI(.*?)EEv", name).groups()
    a = [int(v) for v in re.findall(r"L[ib](\d+)E", args)]
    return {"product": lambda: a[1], "transposed": lambda: 2 + a[0] * a[1], "gradient": lambda: 2 * a[0]}[kind]()


def _blocks(lines):
    """label -> its loads ('L' into LDS, 'g' others), waits ('step', N) / ('wait', N), jumps; labels in their order"""
    blocks, order, cur = {"entry": []}, ["entry"], "entry"
    for t in (line.strip() for line in lines):
        label = re.match(r"(\.LBB\w+):", t)
        if label:
            cur = label.group(1)
            blocks[cur] = []
            order.append(cur)
        elif t.startswith("buffer_load") and " lds" in t:
            blocks[cur].append("L")
        elif t.startswith(("global_load", "buffer_load", "flat_load", "scratch_", "global_store", "flat_store")):
            blocks[cur].append("g")
        elif t.startswith("s_waitcnt") and "vmcnt" in t:
            n = int(re.search(r"vmcnt\((\d+)\)", t).group(1))
            blocks[cur].append(("step" if re.fullmatch(r"s_waitcnt vmcnt\(\d+\) lgkmcnt\(0\)", t) else "wait", n))
        elif t.startswith(("s_cbranch", "s_branch")):
            blocks[cur].append(("may" if t.startswith("s_cbranch") else "must", t.split()[-1]))
        elif t.startswith("s_endpgm"):
            blocks[cur].append(("end", 0))
    return blocks, order


def _uncovered(lines, per_stage):
    """(steps seen, {(label, N, step)} where a stage's loads may still be on their way)"""
    blocks, order = _blocks(lines)
    after = dict(zip(order, order[1:]))
    to = {b: [o[1] for o in ops if o[0] in ("may", "must")] + ([after[b]] if b in after and not any(o[0] in ("must", "end") for o in ops) else [])
          for b, ops in blocks.items()}
    ahead = {b for b, ops in blocks.items() if any(o[0] == "step" for o in ops)}      # a step's wait is still to come
    while True:
        more = {b for b in blocks if b not in ahead and any(t in ahead for t in to[b])}
        if not more:
            break
        ahead |= more
    bad, seen, most = set(), set(), 0
    stack = [("entry", 0, (), 0)]
    while stack:
        state = stack.pop()
        if state in seen or state[0] not in ahead:
            continue
        seen.add(state)
        assert len(seen) < 1000000
        b, step, queue, loads = state
        for o in blocks[b]:
            if o == "L":
                queue, loads = queue + (loads // per_stage,), loads + 1
            elif o == "g":
                queue += (-1,)
            elif o[0] in ("step", "wait"):
                queue = queue[-o[1]:] if o[1] else ()
                if o[0] == "step":
                    if any(0 <= stage <= step for stage in queue):
                        bad.add((b, o[1], step))
                    step += 1
                    most = max(most, step)
                    if step > STEPS:
                        break
            elif o[0] == "may":
                stack.append((o[1], step, queue, loads))
            elif o[0] == "must":
                stack.append((o[1], step, queue, loads))
                break
            else:
                break
        else:
            if b in after:
                stack.append((after[b], step, queue, loads))
    return most, bad


def test_the_walk_sees_a_missing_wait():
    """two stages of one load in flight; the last step's next load is there, or was dropped"""
    lines = """
        buffer_load_dwordx4 v0, s[0:3], 0 offen lds
        global_load_dwordx4 v[0:3], v4, s[0:1]
        global_load_dwordx4 v[0:3], v4, s[0:1]
        buffer_load_dwordx4 v0, s[0:3], 0 offen lds
        s_waitcnt vmcnt({n}) lgkmcnt(0)
        s_cbranch_scc1 .LBB0_2
        global_load_dwordx4 v[0:3], v4, s[0:1]
        .LBB0_2:
        s_waitcnt vmcnt({m}) lgkmcnt(0)
        s_endpgm
    """
    walk = lambda n, m: _uncovered(lines.format(n=n, m=m).split("\n"), 1)
    assert walk(3, 0) == (2, set()) and walk(1, 0) == (2, set())
    assert walk(4, 0) == (2, {("entry", 4, 0)})
    assert walk(3, 1) == (2, {(".LBB0_2", 1, 1)})            # covered only where the branch is not taken


def test_no_step_reads_what_may_still_be_on_its_way(kernels):
    for name, lines in kernels.items():
        steps, bad = _uncovered(lines, _loads_per_stage(name))
        assert steps > STEPS and not bad, (name, sorted(bad)[:5])
