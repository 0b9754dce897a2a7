"""CPU: properties of the compiled gfx950 code of the feed-forward block and of the
block-scaled FP8 product that their source relies on, checked on the device code of
this build's own objects (no GPU).

* M0 belongs to the direct-to-LDS loads, which write it in their own asm block.
* No kernel spills: a spill's loads count as vector memory, which the rings' waits
  count themselves.
* The tall tiles keep their registers within two waves a SIMD.
"""
from __future__ import annotations

import re
import subprocess
from pathlib import Path

import pytest

BUILD = Path(__file__).resolve().parents[1] / "td_benchmark_amd" / "csrc" / "build"
LLVM = Path("/opt/rocm/llvm/bin")


@pytest.fixture(scope="module", params=["gated", "fp8_mm"])
def device_code(request, tmp_path_factory) -> Path:
    obj = BUILD / f"{request.param}.o"
    if not obj.exists() or not (LLVM / "llvm-objcopy").exists():
        pytest.skip("native library not built here")
    tmp = tmp_path_factory.mktemp("code")
    fat, out = tmp / "fat", tmp / "device.o"
    subprocess.run([LLVM / "llvm-objcopy", "--dump-section", f".hip_fatbin={fat}", obj, tmp / "copy.o"], check=True)
    subprocess.run([LLVM / "clang-offload-bundler", "--unbundle", "--type=o", "--targets=hipv4-amdgcn-amd-amdhsa--gfx950",
                    f"--input={fat}", f"--output={out}"], check=True)
    return out


def run(tool, *args) -> str:
    return subprocess.run([LLVM / tool, *args], check=True, capture_output=True, text=True).stdout


def test_registers_and_no_spills(device_code):
    notes = run("llvm-readelf", "--notes", device_code)
    found = re.findall(r"\.name: +(_Z\S+)\n.*?\.private_segment_fixed_size: (\d+).*?\.vgpr_count: +(\d+)\n +\.vgpr_spill_count: (\d+)",
                       notes, flags=re.S)
    assert len(found) >= 20
    for name, scratch, vgprs, spills in found:
        assert scratch == spills == "0", name
        if "ILi256ELi256E" in name:
            assert int(vgprs) <= 256, name
    assert sum("ILi256ELi256E" in f[0] for f in found) >= 2


def test_m0_is_written_only_by_the_direct_to_lds_loads(device_code):
    code = [ln.split("//")[0].strip() for ln in run("llvm-objdump", "-d", "--no-show-raw-insn", device_code).splitlines()]
    code = [ln for ln in code if ln and not ln.endswith(":")]
    uses = [i for i, ln in enumerate(code) if re.search(r"\bm0\b", ln)]
    assert uses, "no M0 reference found: the direct-to-LDS loads are missing"
    for i in uses:
        assert re.fullmatch(r"s_mov_b32 m0, (s\d+|vcc_lo|vcc_hi)", code[i]) and code[i + 1] == "s_nop 0", code[i:i + 3]
        assert re.match(r"global_load_lds_dword(x4)? v(\d+, s)?\[\d+:\d+\](, off)?$", code[i + 2]), code[i:i + 3]
    assert not any(re.match(r"v_pk_(add|mul|fma)_f32\b", ln) for ln in code)
