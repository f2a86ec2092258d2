#!/usr/bin/env python
"""Build guard: the scalar memory instructions of libgrk's GPU code objects read,
and do nothing else.  A write through the scalar data cache is not expected of the
compiler for this code; the build looks at the disassembly instead of trusting
that.  What is not in the list below fails, so it names no instruction that may
not be there.

    python scripts/check_scalar_writes.py build/obj/grk_*.o
"""
import os
import re
import sys

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from check_mfma_overlap import disassemble  # noqa: E402

SMEM = 0b110000   # bits 31..26 of a scalar memory instruction's first word (gfx9)
READS = re.compile(r'(s_load|s_buffer_load|s_scratch_load)_dword(x\d+)?|s_memtime|s_memrealtime')
LINE = re.compile(r'^\s+(\w+)[^\n]*//\s*[0-9A-F]+:\s*([0-9A-F]{8})', re.M)


def scalar_memory(disasm_text):
    """Mnemonics of the scalar memory instructions, told by their encoding."""
    return [m.group(1) for m in LINE.finditer(disasm_text) if int(m.group(2), 16) >> 26 == SMEM]


def scalar_writes(obj):
    """[(mnemonic, count)] of the scalar memory instructions of one object's GPU code
    that are not plain reads."""
    seen = scalar_memory(disassemble(obj))
    if not seen:   # every kernel reads its arguments this way
        raise ValueError(f'{obj}: no scalar memory instruction found (another disassembly format?)')
    return sorted((n, seen.count(n)) for n in set(seen) if not READS.fullmatch(n))


def main(paths):
    bad = 0
    for p in paths:
        w = scalar_writes(p)
        if w:
            bad += 1
            print(f'{p}: {w}')
    print(f'check_scalar_writes: {"FAIL" if bad else "ok"} ({len(paths)} object(s))')
    return 1 if bad else 0


if __name__ == '__main__':
    sys.exit(main(sys.argv[1:]))
