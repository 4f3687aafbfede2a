"""The optimizer step's sources in the in-tree build (-DXCCL_MC_ROCM_IN_TREE), where types, vtable and dispatcher come from the
tree's own headers: over the patched reference where its files are there, and over stand-ins that declare what those declare."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "xccl_amd", "csrc")
INC = os.path.join(ROOT, "include")
REFERENCE = "/root/reference"
FLAGS = ["-DXCCL_MC_ROCM_IN_TREE", "-I", INC]
STRICT = ["-Werror=implicit-function-declaration", "-Werror=incompatible-pointer-types", "-Werror=int-conversion",
          "-Werror=implicit-int", "-Werror=return-type"]


def _outside_the_tree(header):
    """What one of our headers declares where there is no tree around it."""
    text = open(os.path.join(INC, header)).read()
    return text[text.index('#ifdef __cplusplus\nextern "C" {'):text.index("#endif /* XCCL_MC_ROCM_IN_TREE */")]


def _stand_in(d):
    files = {"api/xccl.h": "#include <stddef.h>\n#include <stdint.h>\n" + _outside_the_tree("xccl_rocm_types.h"),
             "ucs/memory/memory_type.h": "",
             "utils/mem_component.h": "#include <api/xccl.h>\n" + _outside_the_tree("xccl_rocm_mem_component.h")}
    for name, text in files.items():
        (d / name).parent.mkdir(parents=True, exist_ok=True)
        (d / name).write_text("#pragma once\n" + text)
    return ["-I", str(d)]


def _patched_reference(d):
    if not os.path.exists(os.path.join(REFERENCE, "src", "utils", "mem_component.h")):
        pytest.skip("reference files not present")
    shutil.copytree(os.path.join(REFERENCE, "src"), d / "src")
    subprocess.run(["patch", "-s", "-p1", "--fuzz=0", "-i", os.path.join(ROOT, "integration", "xccl-rocm.patch")], cwd=d, check=True)
    return ["-I", os.path.join(ROOT, "tests", "stubs")] + [x for s in ("src", "src/core", "src/utils") for x in ("-I", str(d / s))]


@pytest.fixture(scope="module", params=[_stand_in, _patched_reference], ids=["stand_in", "patched_reference"])
def includes(request, tmp_path_factory):
    return request.param(tmp_path_factory.mktemp("tree"))


def _run(args):
    return subprocess.run(args, capture_output=True, text=True)


def test_host_side(includes):
    out = _run(["gcc", "-std=gnu11", "-O1", "-c", "-o", os.devnull, "-D__HIP_PLATFORM_AMD__", "-I", "/opt/rocm/include"] + STRICT +
               FLAGS + includes + [os.path.join(CSRC, "mc_step.c")])
    assert out.returncode == 0, out.stderr


def test_kernels_and_their_launches(includes):
    out = _run(["hipcc", "--offload-arch=gfx950", "-std=c++17", "-fsyntax-only", "-Wno-unused-command-line-argument"] + FLAGS +
               includes + [os.path.join(CSRC, "step_kernels.hip")])
    assert out.returncode == 0, out.stderr


def test_the_trees_headers_are_the_ones_that_count(includes, tmp_path):
    """A vtable in the tree that differs from what the component was written for stops the build."""
    wrong = tmp_path / "utils"
    wrong.mkdir()
    (wrong / "mem_component.h").write_text("#pragma once\n#include <api/xccl.h>\ntypedef struct xccl_mem_component { int open; } xccl_mem_component_t;\n")
    out = _run(["gcc", "-std=gnu11", "-fsyntax-only", "-D__HIP_PLATFORM_AMD__", "-I", "/opt/rocm/include", "-I", str(tmp_path)] + STRICT +
               FLAGS + includes + [os.path.join(CSRC, "mc_step.c")])
    assert out.returncode != 0
