"""Attention over caches of 4 bits keeps tiles and sums in registers: no form of it that the library holds uses scratch memory."""
import os
import re
import subprocess

import pytest

from test_kernel_registers import LIB, READELF, device_code


def test_no_form_uses_scratch_memory(tmp_path):
    if not (os.path.exists(READELF) and os.path.exists(LIB)):
        pytest.skip("needs the built library and llvm-readelf")
    forms = {}
    for code in device_code(open(LIB, "rb").read()):
        if b"attn_kv4_" not in code and b"append_paged_kernel" not in code:
            continue
        (tmp_path / "code").write_bytes(code)
        notes = subprocess.check_output([READELF, "--notes", str(tmp_path / "code")], text=True)
        for name, scratch in re.findall(r"\.name:\s+(\S*(?:attn_kv4_|append_paged_kernel)\S*)\n(?:(?!\.name:).)*?\.private_segment_fixed_size:\s+(\d+)", notes, re.S):
            forms[name] = int(scratch)
    # (two types: five shapes with 3 ways to put rows side by side but one, all but 16 rows by four waves or one, their joins; three tiles and the joins of their ranges; the append's
    # kinds, aligned or not)
    assert len(forms) >= 2 * (23 + 10 + 15 + 2 + 18)
    assert not {k: v for k, v in forms.items() if v}
