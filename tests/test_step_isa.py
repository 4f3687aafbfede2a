"""Static checks on the gfx950 assembly of the optimizer step's kernels (no GPU): what the design relies on and a compiler
upgrade or an edit could silently undo."""
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "xccl_amd", "csrc")
FLAGS = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-ffp-contract=off", "-Xclang", "-target-feature", "-Xclang",
         "-packed-fp32-ops", "-Wno-unused-command-line-argument", "-I", os.path.join(ROOT, "include"), "-S",
         "--cuda-device-only"]


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    """name -> (instructions, descriptor) of every kernel."""
    dst = str(tmp_path_factory.mktemp("isa") / "step.s")
    subprocess.run(["hipcc"] + FLAGS + [os.path.join(CSRC, "step_kernels.hip"), "-o", dst], check=True,
                   stdout=subprocess.DEVNULL, stderr=subprocess.DEVNULL)
    out = {}
    for m in re.finditer(r"^(_ZN9xccl_rocm\w+):.*?\n(.*?)\.amdhsa_kernel(.*?)\.end_amdhsa_kernel", open(dst).read(),
                         flags=re.S | re.M):
        lines = [ln.strip() for ln in m.group(2).splitlines() if ln.startswith("\t")]
        out[m.group(1)] = ([ln for ln in lines if ln and not ln.startswith((".", ";"))], m.group(3))
    return out


def test_every_variant_is_there(kernels):
    names = list(kernels)
    assert sum("adamw_kernel" in n for n in names) == 3 * 3 * 2 * 2      # parameter, gradient, states, peers
    assert sum("grad_norm_kernel" in n for n in names) == 3 and sum("fold_norm_kernel" in n for n in names) == 3
    assert sum("step_clock_kernel" in n for n in names) == 1 and len(names) == 43


def test_nothing_leaves_the_registers(kernels):
    """No scratch memory, no flat access (a pointer whose address space was lost), no packed 32-bit arithmetic."""
    for name, (code, desc) in kernels.items():
        assert re.search(r"\.amdhsa_private_segment_fixed_size 0\b", desc), name
        bad = [ln for ln in code if ln.startswith(("scratch_", "flat_", "v_pk_add_f32", "v_pk_mul_f32", "v_pk_fma_f32"))]
        assert not bad, (name, bad[:3])


def test_registers_leave_room_for_the_waves(kernels):
    """The step runs with up to 32 waves on a compute unit (64 registers each), the norm with 8 waves (two to a SIMD)."""
    for name, (_, desc) in kernels.items():
        vgprs = int(re.search(r"\.amdhsa_next_free_vgpr (\d+)", desc).group(1))
        assert vgprs <= (64 if "adamw_kernel" in name else 128), (name, vgprs)


def test_partial_results_are_in_memory_before_the_arrival(kernels):
    """The workgroup that counts itself in has waited for its own partial result: a full wait lies between the stores, which
    are written through, and the first arrival."""
    for name, (code, _) in kernels.items():
        if "norm_kernel" not in name:
            continue
        arrivals = [i for i, ln in enumerate(code) if ln.startswith("global_atomic_inc")]
        assert len(arrivals) == 2, name
        before = code[:arrivals[0]]
        wait = max(i for i, ln in enumerate(before) if ln == "s_waitcnt vmcnt(0)")
        stores = [i for i, ln in enumerate(before) if ln.startswith("global_store_dwordx2")]
        assert len(stores) >= 2 and max(stores) < wait, name
        assert all("sc0 sc1" in before[i] for i in stores), name


def test_the_norm_requests_before_it_sums(kernels):
    """In the loop a round's 16-byte loads go out in front of the sums of the round before: no wait for all loads in between."""
    for name, (code, _) in kernels.items():
        if "grad_norm_kernel" not in name:
            continue
        loads = [i for i, ln in enumerate(code) if ln.startswith("buffer_load_dwordx4")]
        first_sum = next(i for i, ln in enumerate(code) if ln.startswith("v_fma_f64") or ln.startswith("v_fmac_f64"))
        assert sum(i < first_sum for i in loads) == 8, name     # two rounds of 4 KiB
        assert "s_waitcnt vmcnt(0)" not in code[loads[0]:first_sum], name
