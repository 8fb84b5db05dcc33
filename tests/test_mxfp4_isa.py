"""CPU: the ISA check of the MXFP4 tile kernel (tools/check_isa.py, part of the build) on the assembly of the linked object, and on the same
assembly with one violation planted at a time: each is reported."""
import importlib.util
import os
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ASM = os.path.join(ROOT, "flux-2-swift-mlx_amd", "csrc", "build", "mxfp4_gemm-hip-amdgcn-amd-amdhsa-gfx950.s")


@pytest.fixture(scope="module")
def isa():
    spec = importlib.util.spec_from_file_location("check_isa", os.path.join(ROOT, "tools", "check_isa.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.fixture(scope="module")
def kernel(flux2mi):
    """The text of one 256 x 256 tile kernel with its metadata."""
    if not os.path.exists(ASM):
        pytest.skip("no device assembly next to the objects (library built elsewhere)")
    text = open(ASM).read()
    name = re.search(r"^(_Z\S*\d+mxfp4_gemm_tile_kernelILi256ELi256ELb1ELb1ELi0E\S+):", text, re.M).group(1)
    body = re.search(r"^" + re.escape(name) + r":\s*;.*?^\.Lfunc_end\d+:", text, re.S | re.M).group(0)
    meta = re.search(r"^    \.name:\s+" + re.escape(name) + r"\n(?:    \s*\..*\n)+", text, re.M).group(0)
    return body + "\n" + meta


def reported(isa, text):
    errors = []
    isa.check_m0("mxfp4_gemm", text, errors)
    isa.check_mxfp4_tile(text, errors)
    return " ".join(str(e) for e in errors)


def test_every_tile_kernel_of_the_linked_object(isa, flux2mi):
    if not os.path.exists(ASM):
        pytest.skip("no device assembly next to the objects (library built elsewhere)")
    assert reported(isa, open(ASM).read()) == ""


def test_build_runs_the_check():
    makefile = open(os.path.join(ROOT, "flux-2-swift-mlx_amd", "csrc", "Makefile")).read()
    assert "mxfp4_gemm" in re.search(r"^ISA_SRC :=(.*)$", makefile, re.M).group(1).split()


def behind_mfma(text, n, *lines):
    """`lines` behind the n-th MFMA"""
    at = [m.end() for m in re.finditer(r"^\tv_mfma.*$", text, re.M)][n]
    return text[:at] + "".join("\n\t" + line for line in lines) + text[at:]


def sources(text, n):
    line = re.findall(r"^\tv_mfma.*$", text, re.M)[n]
    return [o.strip() for o in line.split(None, 1)[1].split(" op_sel")[0].split(",")]


@pytest.mark.parametrize("what,plant", [
    ("v_accvgpr_read_b32", lambda t: behind_mfma(t, 40, "v_accvgpr_read_b32 v255, a3")),
    ("copy", lambda t: behind_mfma(t, 100, "v_mov_b32_e32 v250, v251")),
    ("scratch_store_dword", lambda t: behind_mfma(t, 7, "scratch_store_dword off, v1, off")),
    ("global_load_dword ", lambda t: behind_mfma(t, 7, "global_load_dword v250, v1, s[2:3]")),
    ("M0", lambda t: behind_mfma(t, 60, "s_mov_b32 m0, 0")),
    ("M0 is not this piece's", lambda t: re.sub(r"(\n\tglobal_load_lds_dwordx4 \S+ \S+ offset:1024|\n\tglobal_load_lds_dwordx4 \S+ \S+ offset:0x400)", r"\n\ts_mov_b32 m0, s4\n\ts_nop 0\1", t, count=1)),
    ("vmcnt", lambda t: behind_mfma(t, 90, "s_waitcnt vmcnt(0)")),
    ("wait states", lambda t: behind_mfma(t, 99, f"v_add_u32_e32 {sources(t, 101)[4]}, 1, v250")),
    ("wait states", lambda t: behind_mfma(t, 98, f"v_lshlrev_b32_e32 v{re.search('[0-9]+', sources(t, 100)[1]).group(0)}, 1, v250")),
    ("behind the copies", lambda t: t.replace("s_nop 7", "s_nop 0")),
    ("accumulator moves", lambda t: t.replace(re.findall(r"^\tv_mfma.*$", t, re.M)[9], "\tv_mfma_scale_f32_16x16x128_f8f6f4 a[0:3], v[2:5], v[6:9], a[4:7], v10, v11 op_sel_hi:[0,0,0] cbsz:4 blgp:4", 1)),
    ("ds_read_b128", lambda t: behind_mfma(t, 30, "ds_read_b128 v[250:253], v249")),
    ("drained", lambda t: t.replace("s_nop 15", "s_nop 0")),
    ("spills", lambda t: re.sub(r"(\.vgpr_spill_count:\s+)0", r"\g<1>3", t)),
    ("not found", lambda t: behind_mfma(t, 3, re.findall(r"^\t(v_mfma.*)$", t, re.M)[3])),
])
def test_planted_violations_are_reported(isa, kernel, what, plant):
    assert reported(isa, kernel) == ""
    text = plant(kernel)
    assert text != kernel
    assert what in reported(isa, text)
