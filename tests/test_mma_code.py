"""Compiled code of the kernels whose matrix products are inline asm (``csrc/fp8_tile.hip``,
``csrc/latent_tile.hip``, ``csrc/latent_expanded.hip``): the compiler does not know the products'
latency, so their results have to be read late enough by construction. Reads the code that this
tree built; no GPU needed."""

from __future__ import annotations

import re
import shutil
import subprocess
from pathlib import Path

import pytest

OBJDUMP = Path("/opt/rocm/llvm/bin/llvm-objdump")
KERNELS = {"fp8_tile_kernel": 26, "latent_tile_kernel": 16, "latent_mixed_kernel": 8, "latent_expanded_kernel": 6}
# passes of the matrix cores (a wait state each) by a product's shape, and the states past the last of them
# after which another instruction may touch its result
PASSES = {"16x16x16": 4, "16x16x32": 4, "16x16x128": 8, "32x32x16": 8}
PAST = 4
# wait states between a vector instruction and a product that reads what it wrote
BEFORE = 2


@pytest.fixture(scope="module")
def kernels(tmp_path_factory) -> dict[str, list[str]]:
    from slipstream_amd import build

    if not OBJDUMP.exists():
        pytest.skip("no llvm-objdump")
    tmp = tmp_path_factory.mktemp("code")
    lib = tmp / "lib.so"
    shutil.copy(build.OUT_DIR / build.LIB_NAME, lib)
    subprocess.run([OBJDUMP, "--offloading", str(lib)], check=True, capture_output=True, cwd=tmp)
    found: dict[str, list[str]] = {}
    for code in tmp.glob("lib.so.*gfx950"):
        raw = code.read_bytes()
        if not any(name.encode() in raw for name in KERNELS):
            continue
        text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", str(code)], check=True, capture_output=True,
                              text=True).stdout
        for part in re.split(r"^[0-9a-f]+ <", text, flags=re.M)[1:]:
            name, body = part.split(">:", 1)
            if any(k in name for k in KERNELS):
                found[name] = [line for line in body.splitlines() if line.startswith("\t")]
    return found


def _registers(text: str) -> set[str]:
    regs = set()
    for kind, lo, hi in re.findall(r"\b([va])\[(\d+):(\d+)\]", text):
        regs.update(f"{kind}{i}" for i in range(int(lo), int(hi) + 1))
    regs.update(a + b for a, b in re.findall(r"\b([va])(\d+)\b", text))
    return regs


def too_early(lines: list[str]) -> list[str]:
    """Instructions that may touch a product's result before it is there, and products that may read a register before
    a vector instruction has written it: every instruction takes a wait state, an s_nop n + 1, and a product waits
    until the matrix cores are done with the one before it. Straight through, and once more from the target of each
    backward branch."""
    code, at = [], {}
    for line in lines:
        text, _, note = line.partition("//")
        address = re.search(r"([0-9A-Fa-f]{8,}):", note)
        if address is None:  # filling behind the end
            continue
        at[int(address[1], 16)] = len(code)
        code.append(text.strip())
    addresses = sorted(at)
    faults: list[str] = []

    def run(i, now, free, ready, wrote, left, jump):
        while i < len(code) and left:
            text = code[i]
            op, _, args = text.partition(" ")
            if op.startswith("v_mfma"):
                passes = next(v for k, v in PASSES.items() if k + "_" in op)
                dst, a, b = re.findall(r"[va]\[\d+:\d+\]", args)[:3]  # (asm products add to their own result or to 0)
                for r in _registers(a) | _registers(b):
                    if ready.get(r, 0) > now or wrote.get(r, -9) + BEFORE >= now:
                        faults.append(text)
                        break
                now = max(now, free)
                free = now + passes
                now += 1
                for r in _registers(dst):
                    ready[r] = free + PAST
            else:
                if any(ready.get(r, 0) > now for r in _registers(args)):
                    faults.append(text)
                if op.startswith("v_"):
                    written = args if "swap" in op else args.split(",")[0]
                    for r in _registers(written):
                        wrote[r] = now
                now += int(args.split()[0]) + 1 if op == "s_nop" else 1
                if jump and (op.startswith("s_cbranch") or op == "s_branch"):
                    word = int(args.split()[0])
                    target = addresses[i] + 4 + 4 * (word - 65536 if word >= 32768 else word)
                    if target in at and target <= addresses[i]:
                        run(at[target], now, free, dict(ready), dict(wrote), 200, False)
            i += 1
            left -= 1

    run(0, 0, 0, {}, {}, len(code), True)
    return faults


def test_every_kernel_is_there(kernels):
    for name, count in KERNELS.items():
        assert sum(name in k for k in kernels) == count, (name, sum(name in k for k in kernels))


def test_results_are_read_when_they_are_there(kernels):
    wrong = {name: too_early(lines)[:4] for name, lines in kernels.items()}
    wrong = {name: lines for name, lines in wrong.items() if lines}
    assert not wrong


def test_an_early_read_is_found():
    def listing(*code):
        return [f"\t{text} // {0x1000 + 4 * i:012X}:" for i, text in enumerate(code)]

    product = "v_mfma_f32_16x16x128_f8f6f4 v[{}:{}], v[20:27], v[30:37], 0"
    first, second, third = (product.format(i, i + 3) for i in (0, 4, 8))
    read = "v_fmac_f32_e32 v60, v1, v70"
    assert too_early(listing(first, read)) == [read]
    assert too_early(listing(first, second, read)) == [read]
    assert not too_early(listing(first, second, third, read))
    assert too_early(listing(first, "s_nop 9", read)) == [read]
    assert not too_early(listing(first, "s_nop 11", read))
    made = "v_mov_b32_e32 v25, 0"
    assert too_early(listing(made, "s_nop 0", first)) == [first]
    assert not too_early(listing(made, "s_nop 1", first))
