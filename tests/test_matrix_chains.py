"""The built kernels' matrix instructions: a sum that goes from one to the next goes through instructions of one shape. (Where a
16 x 16 x 16 product's result was the addend of a 16 x 16 x 32 product two instructions behind it, rows of the sum were lost on
gfx950, without a wait from the compiler.) Runs without a GPU."""
import re
import subprocess

import pytest

from tests.test_wait_states import code_object

MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"

NEAR = 16          # instructions that a result is followed for
REG = re.compile(r"\b([av])(?:(\d+)\b|\[(\d+):(\d+)\])")


def _regs(text):
    return {f"{kind}{i}" for kind, one, lo, hi in REG.findall(text) for i in (range(int(lo), int(hi) + 1) if lo else (int(one),))}


def mixed(lines):
    found, kernel, made, now = [], "", {}, 0       # made: register -> (instruction, when) of the matrix instruction that wrote it
    for line in lines:
        if line.endswith(">:"):
            kernel, made = line, {}
            continue
        op, _, rest = line.split("//")[0].strip().partition(" ")
        if not op:
            continue
        now += 1
        args = re.split(r",\s*(?![^\[]*\])", rest)
        if op.startswith("v_mfma"):
            for r in _regs(args[3]):
                if r in made and made[r][0] != op and now - made[r][1] <= NEAR:
                    found.append((kernel, made[r][0], op, r))
                    break
            made |= {r: (op, now) for r in _regs(args[0])}
        elif op.startswith("v_"):
            for r in _regs(args[0]):
                made.pop(r, None)
    return found


def listing(tmp_path):
    """The disassembly of all of the library's code objects, one for each source file."""
    co, tool = code_object(tmp_path)
    fat, lines = (tmp_path / "fat.bin").read_bytes(), []
    for k, bundle in enumerate(fat.split(MAGIC)[1:]):
        (tmp_path / f"bundle{k}").write_bytes(MAGIC + bundle)
        subprocess.run([tool("clang-offload-bundler"), "--type=o", "--unbundle", f"--input={tmp_path}/bundle{k}", "--targets=hipv4-amdgcn-amd-amdhsa--gfx950",
                        f"--output={co}"], check=True)
        lines += subprocess.run([tool("llvm-objdump"), "-d", "--no-show-raw-insn", co], check=True, capture_output=True, text=True).stdout.splitlines()
    return lines


def test_one_shape_a_sum(tmp_path):
    lines = listing(tmp_path)
    assert any("v_mfma_f32_16x16x16" in x for x in lines) and any("v_mfma_f32_16x16x32" in x for x in lines)
    assert not mixed(lines)


@pytest.mark.parametrize("code,n", [
    ("v_mfma_f32_16x16x16_bf16 v[18:21], v[122:123], v[110:111], 0\nv_mfma_f32_16x16x32_bf16 v[86:89], v[86:89], v[82:85], v[18:21]", 1),
    ("v_mfma_f32_16x16x16_bf16 a[0:3], v[122:123], v[110:111], 0\nv_mfma_f32_16x16x32_bf16 v[86:89], v[86:89], v[82:85], a[0:3]", 1),
    ("v_mfma_f32_16x16x16_bf16 v[18:21], v[122:123], v[110:111], 0\nv_mfma_f32_16x16x16_bf16 v[86:89], v[86:87], v[82:83], v[18:21]", 0),
    ("v_mfma_f32_16x16x16_bf16 v[18:21], v[122:123], v[110:111], 0\nv_mfma_f32_16x16x32_bf16 v[86:89], v[86:89], v[82:85], v[22:25]", 0),
    ("v_mfma_f32_16x16x16_bf16 v[18:19], v[122:123], v[110:111], 0\nv_mov_b32_e32 v18, v2\nv_mov_b32_e32 v19, v2\nv_mfma_f32_16x16x32_bf16 v[86:89], v[86:89], v[82:85], v[18:19]", 0)])
def test_the_check_finds(code, n):
    assert len(mixed(code.splitlines())) == n
