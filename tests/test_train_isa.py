"""What the compiler made of libfedtrain.so (built here; on the CPU, nothing runs).

* No packed float32 arithmetic: some of its forms have given wrong results on
  this hardware now and then.
* A load that goes to LDS directly reads a buffer descriptor in scalar registers.
  A vector instruction that writes such a register (v_readlane, v_readfirstlane, a
  compare) has to lie at least 5 wait states before the load; the source holds one
  s_nop for it where the descriptor is made, and the compiler does not see into
  the loads, so nothing else keeps a later change from breaking it.
* The large tiles keep their sums in registers: no kernel uses scratch memory.
"""
import glob
import os
import re
import shutil
import subprocess

import pytest

from test_isa_guard import FUNC, INSN, OBJDUMP

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = os.path.join(REPO, "fedsim_amd", "libfedtrain.so")
NM = os.path.join(os.path.dirname(OBJDUMP), "llvm-readelf")


@pytest.fixture(scope="module")
def objects(tmp_path_factory):
    d = str(tmp_path_factory.mktemp("isa"))
    shutil.copy(LIB, os.path.join(d, "lib.so"))
    subprocess.run([OBJDUMP, "--offloading", os.path.join(d, "lib.so")], cwd=d, check=True,
                   capture_output=True)
    found = glob.glob(os.path.join(d, "*gfx950"))
    assert len(found) == 2, found  # one a source
    return found


def _instructions(co):
    """(function, mnemonic, operands) in order."""
    out = subprocess.Popen([OBJDUMP, "-d", "--no-show-raw-insn", co], stdout=subprocess.PIPE,
                           text=True)
    name = None
    for line in out.stdout:
        m = FUNC.match(line)
        if m:
            name = m.group(2)
            continue
        m = INSN.match(line)
        if m and name:
            yield name, m.group(1), m.group(2).strip()
    assert out.wait() == 0


def _scalars(text):
    """The scalar registers an operand list names first (a destination)."""
    m = re.match(r"s\[(\d+):(\d+)\]|s(\d+)\b", text)
    if not m:
        return set()
    if m.group(3):
        return {int(m.group(3))}
    return set(range(int(m.group(1)), int(m.group(2)) + 1))


def _wait(mnemonic, operands):
    return int(operands, 0) + 1 if mnemonic == "s_nop" else 1


def test_no_packed_float32_and_descriptors_settle(objects):
    packed, early, direct, kernels = [], [], 0, set()
    for co in objects:
        name, recent = None, []  # (scalars a vector instruction wrote, wait states)
        for fn, op, args in _instructions(co):
            if fn != name:
                name, recent = fn, []
                kernels.add(fn)
            if re.match(r"v_pk_(add|mul|fma)_f32", op):
                packed.append((fn, op))
            if op.startswith("buffer_load") and " lds" in args:
                direct += 1
                m = re.search(r"s\[(\d+):(\d+)\]", args)
                need = set(range(int(m.group(1)), int(m.group(2)) + 1))
                states = 0
                for wrote, n in reversed(recent):
                    if states >= 5:
                        break
                    if wrote & need:
                        early.append((fn, args))
                    states += n
            wrote = _scalars(args) if op.startswith("v_") else set()
            if op.startswith("v_cmp") and args.startswith("vcc"):
                wrote = set()
            recent.append((wrote, _wait(op, args)))
            del recent[:-8]
    assert len(kernels) > 100 and direct > 1000  # the listing was read
    assert not packed, packed[:3]
    assert not early, early[:3]


def test_no_kernel_uses_scratch(objects):
    seen = 0
    for co in objects:
        notes = subprocess.check_output([NM, "--notes", co], text=True)
        for key in (".private_segment_fixed_size", ".vgpr_spill_count", ".sgpr_spill_count"):
            sizes = [int(n) for n in re.findall(re.escape(key) + r":\s+(\d+)", notes)]
            assert sizes and (key != ".private_segment_fixed_size" or not any(sizes)), key
            seen += len(sizes)
    assert seen > 100
