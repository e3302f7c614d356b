"""Wait states of the loads that write LDS directly, in the code of the built library.

Such a load takes its LDS address from m0, and one wait state must lie between a
scalar write of m0 and the load; five must lie between a vector instruction that
writes a scalar register and a memory instruction that reads it.  The compiler
keeps both distances for its own instructions, but does not look into inline asm,
where these loads are.  Read from the disassembly; no GPU needed."""
import re
import shutil
import struct
import subprocess
from pathlib import Path

import pytest

from tilebench_amd import runtime as rt

LLVM = Path("/opt/rocm/llvm/bin")
MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"


def code_objects(lib, tmp):
    """The gfx950 code objects of a library, as files."""
    fat = tmp / "fat"
    subprocess.run([LLVM / "llvm-objcopy", "--dump-section", f".hip_fatbin={fat}", lib, tmp / "rest"], check=True)
    raw = fat.read_bytes()
    for n, start in enumerate(m.start() for m in re.finditer(MAGIC, raw)):
        at = start + len(MAGIC) + 8
        for _ in range(struct.unpack_from("<Q", raw, at - 8)[0]):
            offset, size, length = struct.unpack_from("<QQQ", raw, at)
            name = raw[at + 24:at + 24 + length].decode()
            at += 24 + length
            if "gfx950" in name:
                path = tmp / f"{n}.o"
                path.write_bytes(raw[start + offset:start + offset + size])
                yield path


def registers(operand):
    m = re.fullmatch(r"s\[(\d+):(\d+)\]", operand)
    if m:
        return {f"s{i}" for i in range(int(m[1]), int(m[2]) + 1)}
    return {operand} if re.fullmatch(r"s\d+|m0", operand) else {"vcc"} if operand.startswith("vcc") else set()


def offences(lines):
    """(loads to LDS, [what is too close]) of a kernel's instructions in their order."""
    loads, bad, before = 0, [], []  # before: (wait states, registers written by vector / scalar instructions)
    for line in lines:
        text = line.split("//")[0].strip()
        op, _, rest = text.partition(" ")
        operands = [x.split()[0] for x in re.split(r",(?![^\[]*\])", rest) if x.strip()]
        if re.match(r"(buffer|global|flat|scratch)_", op):
            to_lds = "_lds_" in op or text.endswith(" lds")
            loads += to_lds
            if to_lds and before and "m0" in before[-1][2]:
                bad.append(f"m0 written right before: {text}")
            need, waited = set().union(*map(registers, operands)), 0
            for states, vector, scalar in reversed(before):
                if waited >= 5 or not need:
                    break
                if vector & need:
                    bad.append(f"{sorted(vector & need)} written {waited} wait states before: {text}")
                    break
                need, waited = need - scalar, waited + states
        written = registers(operands[0]) if operands else set()
        if len(operands) > 1 and re.search(r"_co_|div_scale|mad_[ui]64", op):
            written |= registers(operands[1])
        vector = written if op.startswith("v_") else set()
        scalar = written if op.startswith("s_") and not op.startswith(("s_cmp", "s_bitcmp", "s_nop")) else set()
        before = before[-5:] + [(int(operands[0]) + 1 if op == "s_nop" else 1, vector, scalar)]
    return loads, bad


def test_the_reader_sees_both_kinds():
    close = ["s_mov_b32 m0, s4", "global_load_lds_dwordx4 v1, s[2:3]"]
    assert offences(close)[0] == 1 and "m0" in offences(close)[1][0]
    assert not offences([close[0], "s_nop 0", close[1]])[1]
    fresh = ["v_readlane_b32 s3, v9, 1", "s_nop 2", "buffer_load_dwordx4 v1, s[0:3], s9 offen lds"]
    assert "3 wait states" in offences(fresh)[1][0]
    assert not offences([fresh[0], "s_nop 4", fresh[2]])[1]
    assert not offences([fresh[0], "s_add_u32 s3, s3, s5", fresh[2]])[1]


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    """{kernel: (loads to LDS, [what is too close])} of the built library."""
    if not rt.LIB_PATH.exists() or not all(shutil.which(LLVM / t) for t in ("llvm-objcopy", "llvm-objdump")):
        pytest.skip("no built library or no LLVM tools")
    out = {}
    for path in code_objects(rt.LIB_PATH, tmp_path_factory.mktemp("code")):
        text = subprocess.run([LLVM / "llvm-objdump", "-d", "--no-show-raw-insn", path], check=True, capture_output=True,
                              text=True).stdout
        for name, body in re.findall(r"^[0-9a-f]+ <(\S+)>:\n(.*?)(?=\n\n|\Z)", text, re.M | re.S):
            if "_lds_" in body or " lds" in body:
                out[name] = offences(body.splitlines())
    return out


@pytest.mark.parametrize("part", ["prefix", "fp8", "w4a16", "ntg"])
def test_loads_to_lds_keep_their_distances(part, kernels):
    some = {name: x for name, x in kernels.items() if part in name}
    assert sum(loads for loads, _ in some.values()) > 0
    bad = [f"{name}: {x}" for name, (_, b) in some.items() for x in b]
    assert not bad, (len(bad), bad[:5])


def test_every_kernel_with_such_loads_is_looked_at(kernels):
    assert not [k for k, (loads, _) in kernels.items()
                if loads and not any(part in k for part in ("prefix", "fp8", "w4a16", "ntg"))]
