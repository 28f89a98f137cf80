"""The tile kernel's compiled code (``csrc/w8a8_tile.hip``): its matrix products are inline asm,
whose latency the compiler does not know, and the waits for its LDS DMA count by hand the loads
issued since. Reads the code that this tree built; no GPU needed."""

from __future__ import annotations

import re
import shutil
import subprocess
from pathlib import Path

import pytest

OBJDUMP = Path("/opt/rocm/llvm/bin/llvm-objdump")
# cycles after which a VALU may read what a 32x32x32 product (at most sixteen passes) wrote, and
# before which one may not write what a product reads
AFTER, BEFORE = 19, 2


@pytest.fixture(scope="module")
def kernels(tmp_path_factory) -> dict[str, list[str]]:
    """The instructions of every tile kernel, by its name."""
    from slipstream_amd import build

    if not OBJDUMP.exists():
        pytest.skip("no llvm-objdump")
    tmp = tmp_path_factory.mktemp("code")
    lib = tmp / "lib.so"
    shutil.copy(build.OUT_DIR / build.LIB_NAME, lib)
    subprocess.run([OBJDUMP, "--offloading", str(lib)], check=True, capture_output=True, cwd=tmp)
    for code in tmp.glob("lib.so.*gfx950"):
        if b"w8a8_tile_kernel" not in code.read_bytes():
            continue
        text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", str(code)], check=True, capture_output=True,
                              text=True).stdout
        found = {}
        for part in re.split(r"^[0-9a-f]+ <", text, flags=re.M)[1:]:
            name, body = part.split(">:", 1)
            if "w8a8_tile_kernel" in name:
                found[name] = [line.split("//")[0].strip() for line in body.splitlines() if line.startswith("\t")]
        assert len(found) == 70  # ten tiles: three output types, weights kept or not, and the sums of a split
        return found
    raise AssertionError("no tile kernel in the library")


def _cycles(code: list[str]) -> int:
    return sum(int(line.split()[1]) + 1 if line.startswith("s_nop") else 1 for line in code)


def test_accumulators_keep_clear_of_the_products(kernels):
    """Between the first and the last product only products touch the accumulators; the last
    write before the first and the first read after the last are far enough away, at one cycle
    an instruction and n + 1 for an s_nop n."""
    for name, code in kernels.items():
        products = [i for i, line in enumerate(code) if line.startswith("v_mfma")]
        first, last = products[0], products[-1]
        touch = [i for i, line in enumerate(code) if re.search(r"\ba\[?\d", line) and not line.startswith("v_mfma")]
        assert not [i for i in touch if first < i < last], name
        before, after = [i for i in touch if i < first], [i for i in touch if i > last]
        assert before and after, name
        assert _cycles(code[before[-1] + 1 : first]) >= BEFORE, name
        assert _cycles(code[last + 1 : after[0]]) >= AFTER, (name, code[last + 1 : after[0] + 1])


def test_dma_waits_leave_what_was_issued_since(kernels):
    """In the loop the wait for the next stage leaves the loads issued after that stage's: those of
    one stage's window at most less than are on their way, and every loop has as many loads as
    a stage has pieces for a wave."""
    for name, code in kernels.items():
        products = [i for i, line in enumerate(code) if line.startswith("v_mfma")]
        tile = [int(v) for v in re.search(r"Li(\d+)ELi(\d+)ELi(\d+)ELi(\d+)E", name).groups()]
        mt, nt, wm, _ = tile
        bm, bn = 32 * mt * wm, 32 * nt * (4 // wm)
        loop = code[products[0] - 1 : products[-1] + 1]
        loads = [i for i, line in enumerate(loop) if line.startswith("buffer_load") and line.endswith("lds")]  # the DMAs
        assert len(loads) == (bm + bn) // 32, name
        lds = 160 * 1024 // (2 if bm + bn <= 256 else 1)
        dw = max(d for d in range(2, 7) if d * (bm + bn) * 128 <= lds)
        dx = dw + 1 if dw < 6 and ((dw + 1) * bm + dw * bn) * 128 <= lds else dw
        waits = [(i, int(re.search(r"vmcnt\((\d+)\)", line)[1])) for i, line in enumerate(loop) if "vmcnt" in line]
        assert len(waits) == 1, (name, waits)
        at, left = waits[0]
        issued = sum(i < at for i in loads)  # of this stage's window, the channels' first
        each = len(loads)
        # newer than the next stage's channels: the tokens of that window, the windows between and
        # this one's; newer than its tokens: the windows between and this one's
        assert left == min((dw - 2) * each + bm // 32 + issued, (dx - 2) * each + issued), (name, left, issued)
