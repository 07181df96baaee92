"""The built gfx950 code's loads to LDS: what an asm copy has to keep by itself, since the compiler's hazard pass does not
look inside one. Read from the library's own code objects; no GPU needed."""

from __future__ import annotations

import re
import shutil
import struct
import subprocess

import pytest

OBJDUMP = shutil.which("llvm-objdump", path="/opt/rocm/llvm/bin") or shutil.which("llvm-objdump")
BUNDLE = b"__CLANG_OFFLOAD_BUNDLE__"


def _code_objects(lib: bytes):
    at = lib.find(BUNDLE)
    while at >= 0:
        count, entry = struct.unpack_from("<Q", lib, at + len(BUNDLE))[0], at + len(BUNDLE) + 8
        for _ in range(count if count < 16 else 0):
            offset, size, n = struct.unpack_from("<QQQ", lib, entry)
            if b"gfx950" in lib[entry + 24:entry + 24 + n]:
                yield lib[at + offset:at + offset + size]
            entry += 24 + n
        at = lib.find(BUNDLE, at + len(BUNDLE))


def _scalars(text: str) -> set[int]:
    regs = {int(x) for x in re.findall(r"\bs(\d+)\b", text)}
    for a, b in re.findall(r"\bs\[(\d+):(\d+)\]", text):
        regs |= set(range(int(a), int(b) + 1))
    return regs


@pytest.mark.skipif(OBJDUMP is None, reason="no llvm-objdump")
def test_loads_to_lds_keep_their_wait_states(tmp_path):
    """A load to LDS takes its place from M0: one wait state after M0's write at the earliest. A scalar register that a
    vector instruction wrote (its address, its descriptor) is read by a vector memory instruction five wait states
    later at the earliest."""
    from gen_worker_amd import build

    loads, m0, scalar = 0, [], []
    for i, code in enumerate(_code_objects(build.LIB_PATH.read_bytes())):
        path = tmp_path / f"{i}.co"
        path.write_bytes(code)
        text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", str(path)], capture_output=True, text=True,
                              check=True).stdout
        before: list[str] = []
        for line in text.splitlines():
            if line.endswith(">:"):
                kernel, before = line, []
                continue
            ins = line.split("//")[0].strip()
            if re.match(r"(global_load_lds|(buffer|global)_load\S* .*\blds\b)", ins):
                loads += 1
                if re.match(r"s_\w+ m0\b", before[-1]):
                    m0.append((kernel, before[-1], ins))
                states, reads = 0, _scalars(ins)
                for p in reversed(before[-6:]):
                    if states >= 5:
                        break
                    if re.match(r"v_(readfirstlane|readlane|cmp)", p) and _scalars(p.split(",")[0]) & reads:
                        scalar.append((kernel, p, ins))
                    states += 1 + (int(p.split()[1], 0) if p.startswith("s_nop") else 0)
            if ins:
                before = before[-7:] + [ins]
    assert loads > 0
    assert not m0, (len(m0), m0[0])
    assert not scalar, (len(scalar), scalar[0])
