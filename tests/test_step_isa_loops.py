"""Static checks on the loops of the optimizer step's kernels in the gfx950 assembly (no GPU)."""
import itertools
import os
import re
import subprocess

import pytest

from test_step_isa import CSRC, FLAGS


@pytest.fixture(scope="module")
def loops(tmp_path_factory):
    """name -> the innermost loops of every kernel, each a list of instructions."""
    dst = str(tmp_path_factory.mktemp("isa") / "step.s")
    subprocess.run(["hipcc"] + FLAGS + [os.path.join(CSRC, "step_kernels.hip"), "-o", dst], check=True,
                   stdout=subprocess.DEVNULL, stderr=subprocess.DEVNULL)
    out = {}
    for m in re.finditer(r"^(_ZN9xccl_rocm\w+):.*?\n(.*?)\.amdhsa_kernel", open(dst).read(), flags=re.S | re.M):
        found, label, body = [], None, []
        for line in m.group(2).splitlines():
            text = line.split(";")[0].strip()
            if re.match(r"\.LBB\w+:", text):
                label, body = text[:-1], []
            elif text and not text.startswith("."):
                body.append(text)
                if label and re.match(r"s_(cbranch_\w+|branch) %s$" % re.escape(label), text):
                    found.append(body)
        out[m.group(1)] = found
    return out


def test_both_halves_of_the_norms_loop_request_before_they_sum(loops):
    """A round is two halves, each of which requests 4 KiB and then sums the 4 KiB that the half before requested.  The sums wait
    for loads in the order of their requests, so a half's first wait leaves all of its own loads outstanding, and so do the rest."""
    kernels = {n: x for n, x in loops.items() if "grad_norm_kernel" in n}
    assert len(kernels) == 3
    for name, found in kernels.items():
        main = [x for x in found if sum("buffer_load_dwordx4" in ln for ln in x) == 8]
        assert len(main) == 1, (name, [len(x) for x in found])
        events = []                                          # ("load" | "sum" | "wait", outstanding loads it leaves)
        for ln in main[0]:
            wait = re.search(r"vmcnt\((\d+)\)", ln)
            if ln.startswith("buffer_load"):
                events.append(("load", 0))
            elif re.match(r"v_fmac?_f64", ln):
                events.append(("sum", 0))
            elif wait:
                events.append(("wait", int(wait.group(1))))
        turns = [k for k, _ in itertools.groupby(k for k, _ in events if k != "wait")]
        assert turns == ["load", "sum", "load", "sum"], (name, turns)
        per_half = sum(k == "load" for k, _ in events) // 2
        waits = [n for k, n in events if k == "wait"]
        assert waits and min(waits) >= per_half, (name, per_half, waits)
