"""Wait states behind the matrix products of the built library, along every path.

The matrix cores write their results some wait states after the instruction, and the hardware does not hold
back an ordinary instruction that reads or overwrites them: the compiler fills in s_nop.  It does so within a block; where a
branch follows the product (on something that a lane does only rarely, or around the next product) it has been seen to leave
one wait state of eight, and the first of four values was then wrong now and then.  Here the library's own code is walked from each
product to the first use of its result, along all branches."""
import re
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"
# wait states until a result may be used, as the compiler leaves them within a block
WAITS = {"v_mfma_f32_16x16x32_bf16": 8, "v_mfma_f32_16x16x4_f32": 10, "v_mfma_i32_32x32x16_i8": 12}
# (a load's own result comes from memory, later than any of these waits)
LOAD, LOADED = re.compile(r"(global|buffer|flat|scratch)_load_(?!lds)|ds_read"), re.compile(r"^[^,]*,")
LINE = re.compile(r"^\t(\S+)\s*(.*?)\s*// ([0-9A-F]{12}): ([0-9A-F]{8})")


def registers(text):
    out = set()
    for first, last, one in re.findall(r"\bv\[(\d+):(\d+)\]|\bv(\d+)\b", text):
        out |= {int(one)} if one else set(range(int(first), int(last) + 1))
    return out


def kernels(text):
    """{name: [(opcode, operands, address, the branch's target or None)]}"""
    out, now = {}, None
    for line in text.splitlines():
        head = re.match(r"^[0-9a-f]+ <(\w+)>:", line)
        if head:
            now = out.setdefault(head.group(1), [])
        m = LINE.match(line)
        if m and now is not None:
            op, operands, at = m.group(1), m.group(2), int(m.group(3), 16)
            to = None
            if op.startswith(("s_branch", "s_cbranch")):
                n = int(m.group(4), 16) & 0xFFFF
                to = at + 4 + 4 * (n - 0x10000 if n & 0x8000 else n)
            now.append((op, operands, at, to))
    return out


def shortest(code, index, start):
    """Wait states from product `start` to the nearest use of its result on any path -> (waits, instruction)."""
    most = WAITS[code[start][0]]
    result = registers(code[start][1].split(",")[0])
    best, seen, paths = (most, None), {}, [(start + 1, 0)]
    while paths:
        i, waits = paths.pop()
        while i < len(code) and waits < best[0] and seen.get(i, most) > waits:
            seen[i] = waits
            op, operands, at, to = code[i]
            if op == "s_nop":
                waits += int(operands) + 1
                i += 1
                continue
            if op == "s_endpgm":
                break
            if op.startswith("v_mfma"):
                parts = re.findall(r"[av]\[\d+:\d+\]|[^,\s]+", operands)
                if (registers(parts[1]) | registers(parts[2])) & result:
                    best = (waits, code[i])
                    break
                if registers(parts[0]) & result:  # (the next product of the sum: it has its own way)
                    break
            elif op[0] != "s" and registers(LOADED.sub("", operands) if LOAD.match(op) else operands) & result:
                best = (waits, code[i])
                break
            waits += 1
            if op.startswith("s_branch"):
                i = index[to]
                continue
            if to is not None:
                paths.append((index[to], waits))
            i += 1
    return best


def test_walk_finds_a_branch_that_follows_a_product():
    """The walk itself, on a product whose result is used behind a branch, and behind enough waits."""
    def code(between):
        lines = ["\tv_mfma_f32_16x16x32_bf16 v[2:5], v[6:9], v[10:13], v[2:5] // 000000000000: 00000000", *between,
                 "\ts_cbranch_vccnz 2 // 000000000010: BF870002", "\ts_nop 7 // 000000000014: BF800007",
                 "\ts_nop 0 // 000000000018: BF800000", "\tv_mul_f32_e32 v2, s0, v2 // 00000000001C: 00000000",
                 "\ts_endpgm // 000000000020: BF810000"]
        return kernels("0000 <k>:\n" + "\n".join(lines))["k"]

    for between, waits in (([], 1), (["\ts_nop 5 // 000000000008: BF800005"], 7), (["\ts_nop 6 // 000000000008: BF800006"], 8)):
        c = code(between)
        assert shortest(c, {x[2]: i for i, x in enumerate(c)}, 0)[0] == waits


@pytest.mark.skipif(not Path(OBJDUMP).exists(), reason="no llvm-objdump")
def test_results_are_not_used_too_early(tmp_path):
    shutil.copy(ROOT / "qwen35-ax7020-edge-llm_amd" / "libqwen_kernels.so", tmp_path / "lib.so")
    subprocess.run([OBJDUMP, "--offloading", "lib.so"], cwd=tmp_path, check=True, capture_output=True)
    early, products = [], 0
    for part in sorted(tmp_path.glob("*gfx950*")):
        text = subprocess.run([OBJDUMP, "-d", part.name], cwd=tmp_path, check=True, capture_output=True, text=True).stdout
        for name, code in kernels(text).items():
            index = {x[2]: i for i, x in enumerate(code)}
            for i, x in enumerate(code):
                if not x[0].startswith("v_mfma"):
                    continue
                products += 1
                assert x[0] in WAITS, f"{x[0]}: its wait states are not in the table"
                assert x[1].startswith("v["), f"{name}: a result in accumulator registers, which the walk does not follow"
                waits, use = shortest(code, index, i)
                if waits < WAITS[x[0]]:
                    early.append((name, x[0], hex(x[2]), waits, use))
    assert products > 1000 and not early, early[:5]
