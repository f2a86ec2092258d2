"""The guard on scalar memory instructions tells them by their encoding and lets only
reads pass (CPU: disassembly text)."""
import os
import sys

import pytest

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'scripts'))

TEXT = ('0000000000001000 <k>:\n'
        '\ts_load_dwordx4 s[4:7], s[0:1], 0x8                         // 000000001000: C00A0100 00000008\n'
        '\ts_mul_i32 s0, s3, s10                                      // 000000001008: 92000A03\n'
        '\ts_memtime s[2:3]                                           // 00000000100C: C0900080 00000000\n'
        '\tglobal_store_dword v0, v1, s[4:5]                          // 000000001014: DC708000 00040100\n')


def test_reads_pass_and_anything_else_does_not(monkeypatch):
    import check_scalar_writes as c
    assert c.scalar_memory(TEXT) == ['s_load_dwordx4', 's_memtime']
    monkeypatch.setattr(c, 'disassemble', lambda obj: TEXT)
    assert c.scalar_writes('k.o') == []
    other = TEXT + '\ts_poke_dword s2, s[0:1], 0x0                               // 000000001018: C0400080 00000000\n' * 2
    monkeypatch.setattr(c, 'disassemble', lambda obj: other)
    assert c.scalar_writes('k.o') == [('s_poke_dword', 2)] and c.main(['k.o']) == 1


def test_a_disassembly_that_it_cannot_read_is_refused(monkeypatch):
    import check_scalar_writes as c
    monkeypatch.setattr(c, 'disassemble', lambda obj: TEXT.replace('//', ';'))
    with pytest.raises(ValueError):
        c.scalar_writes('k.o')
