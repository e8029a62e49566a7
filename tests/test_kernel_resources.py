"""Registers and scratch of every compiled kernel form, from the compiler's resource report of the build:
no form that a launch can select spills, and the register bound leaves a CU the workgroups that its LDS
holds.  (The 64-bit addressing form of the 256 x 256 work tile spills; launches route such problems to
the 128 x 128 work tile of the same macro-tile.)"""
import json
import re
import subprocess
from pathlib import Path

import pytest

from grouped_gemm_gpu_kernel_amd import build

LARGE = (0, 1, 2)  # GGK_VARIANT_64x64x16, 128x64x32, 64x128x32: 256 x 256 work tiles on the MFMA path
MFMA, FMA = 1, 0


def _forms():
    path = build.BUILD / build.FORMS_NAME
    if not path.exists():
        pytest.skip("no regular build in the tree (build first)")
    return json.loads(path.read_text())


def _key(f):
    return f["kind"], f["variant"], f["path"], f["traced"], f["wide"]


def test_report_covers_every_form():
    # grouped: 6 variants x 2 paths x traced x wide; single: 6 x 2 x wide
    forms = _forms()
    assert len(forms) == 6 * 2 * 4 + 6 * 2 * 2
    assert len({_key(f) for f in forms}) == len(forms)


def test_no_selectable_form_spills():
    spills = {}
    for f in _forms():
        if f["path"] == MFMA and f["wide"] and f["variant"] in LARGE:
            continue  # not launched
        if f["scratch"]:
            spills[_key(f)] = f["scratch"]
    assert not spills, f"(kind, variant, path, traced, wide): bytes of scratch a lane {spills}"


def test_fma_registers_allow_the_workgroups_that_lds_holds():
    """160 KB of LDS hold four 64 x 64 tiles or three larger ones; a workgroup is one wave per SIMD."""
    for f in _forms():
        if f["path"] == FMA and not f["wide"]:
            assert f["waves"] >= (4 if f["variant"] in (0, 5) else 3), f


# ---------------------------------------------------------------- routing and 4-bit products

def _scratch(name, tmp_path):
    """Bytes of scratch a lane of every kernel of a device source, by the notes of the built object."""
    built = build.BUILD / name
    if not built.exists():
        pytest.skip("no regular build in the tree (build first)")
    llvm = Path("/opt/rocm/llvm/bin")
    subprocess.run([str(llvm / "llvm-objcopy"), f"--dump-section=.hip_fatbin={tmp_path / 'fat'}", str(built),
                    str(tmp_path / "copy.o")], check=True)
    subprocess.run([str(llvm / "clang-offload-bundler"), "--unbundle", "--type=o",
                    "--targets=hipv4-amdgcn-amd-amdhsa--gfx950", f"--input={tmp_path / 'fat'}",
                    f"--output={tmp_path / 'gfx950.o'}"], check=True)
    notes = subprocess.run([str(llvm / "llvm-readelf"), "--notes", str(tmp_path / "gfx950.o")], check=True,
                           capture_output=True, text=True).stdout
    kernels = [(re.search(r"\.name:\s+(\S+)", k), re.search(r"\.private_segment_fixed_size:\s+(\d+)", k))
               for k in notes.split(".agpr_count:")[1:]]
    assert kernels and all(name and size for name, size in kernels)
    return {name[1]: int(size[1]) for name, size in kernels}


def test_routing_spills_nothing(tmp_path):
    assert not {k: v for k, v in _scratch("gg_route.o", tmp_path).items() if v}


def test_4_bit_products_spill_in_three_forms_of_the_experts_kernel(tmp_path):
    """Groups that are not whole steps of 128, one wave along K: items of 32 rows, and of 16 with zero points (template
    arguments: waves, rows, waves along K, experts, such groups, zero points)."""
    spills = {}
    for kernel, size in _scratch("gg_w4.o", tmp_path).items():
        if size:
            spills[tuple(int(x) for x in re.findall(r"L[ib](\d+)E", kernel))] = size
    most = {(8, 32, 1, 1, 1, 1): 64, (8, 32, 1, 1, 1, 0): 32, (8, 16, 1, 1, 1, 1): 32}
    assert set(spills) <= set(most) and all(size <= most[form] for form, size in spills.items()), spills
