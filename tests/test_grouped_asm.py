"""CPU: properties of the grouped products' compiled gfx950 code that their source
relies on, checked on the AMD assembly of this build (device side only; no GPU).

* M0 belongs to the direct-to-LDS loads, which write it in their own asm block.
* No kernel spills: a spill's loads count as vector memory, which the rings' waits
  count themselves.
* The tall tiles keep their registers within two waves a SIMD.
"""
from __future__ import annotations

import re
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
CSRC = ROOT / "td_benchmark_amd" / "csrc"
HIPCC = "/opt/rocm/bin/hipcc"


@pytest.fixture(scope="module")
def asm(tmp_path_factory) -> str:
    if not Path(HIPCC).exists() or shutil.which("make") is None:
        pytest.skip("hipcc not available")
    out = tmp_path_factory.mktemp("asm") / "grouped_mm.s"
    # the device flags of csrc/Makefile
    cmd = [HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++20", "-Xclang", "-target-feature", "-Xclang",
           "-packed-fp32-ops", "-mllvm", "-amdgpu-mfma-vgpr-form=1", f"-I{ROOT / 'include'}",
           "--cuda-device-only", "-S", "-o", str(out), str(CSRC / "grouped_mm.hip")]
    subprocess.run(cmd, check=True, capture_output=True)
    return out.read_text()


def code_lines(asm: str) -> list[str]:
    lines = [ln.strip() for ln in asm.splitlines()]
    return [ln for ln in lines if ln and not ln.startswith((";", ".", "//")) and not ln.endswith(":")]


def test_m0_is_written_only_by_the_direct_to_lds_loads(asm):
    code = code_lines(asm)
    uses = [i for i, ln in enumerate(code) if re.search(r"\bm0\b", ln)]
    assert uses, "no M0 reference found: the direct-to-LDS loads are missing"
    bad = []
    for i in uses:
        ok = (re.fullmatch(r"s_mov_b32 m0, (s\d+|vcc_lo|vcc_hi)", code[i]) is not None
              and i + 2 < len(code) and code[i + 1] == "s_nop 0"
              and re.match(r"global_load_lds_dword(x4)? v\[\d+:\d+\], off$", code[i + 2]) is not None)
        if not ok:
            bad.append(" | ".join(code[i:i + 3]))
    assert not bad, f"{len(bad)} M0 references outside the asm load blocks, e.g. {bad[:3]}"


def test_no_spills_and_no_packed_fp32(asm):
    kernels = re.findall(r"\.amdhsa_kernel (\S+)(.*?)\.end_amdhsa_kernel", asm, flags=re.S)
    assert len(kernels) >= 30
    for name, body in kernels:
        assert re.search(r"private_segment_fixed_size (\d+)", body).group(1) == "0", name
    assert not re.search(r"\bv_pk_(add|mul|fma)_f32\b", asm)


def test_tall_tiles_run_two_waves_a_simd(asm):
    tall = [(n, b) for n, b in re.findall(r"\.amdhsa_kernel (\S+)(.*?)\.end_amdhsa_kernel", asm, flags=re.S)
            if "tile_mm_kernel" in n and "ILi256ELi256E" in n]
    assert len(tall) >= 8
    for name, body in tall:
        assert int(re.search(r"next_free_vgpr (\d+)", body).group(1)) <= 256, name


def test_two_workgroups_of_the_weights_gradient_share_a_cu(asm):
    found = [(n, b) for n, b in re.findall(r"\.amdhsa_kernel (\S+)(.*?)\.end_amdhsa_kernel", asm, flags=re.S)
             if "tile_mm_kernel" in n and "ILi128ELi256ELi4E" in n]
    assert len(found) == 2
    for name, body in found:
        assert int(re.search(r"next_free_vgpr (\d+)", body).group(1)) <= 256, name
