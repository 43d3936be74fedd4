"""How many waves a SIMD holds of the kernels that count on it, by the registers
that the built library says they take (no GPU)."""
import os
import re

import pytest

import ana_amd

msgpack = pytest.importorskip("msgpack")

# a wave's registers come in eights of a SIMD's 512
WAVES = {("f", 32): 6, ("f", 64): 4, ("f", 128): 3, ("DF16b", 32): 5, ("DF16b", 64): 4, ("DF16b", 128): 3,
         ("DF16_", 32): 7, ("DF16_", 64): 5, ("DF16_", 128): 4}


@pytest.fixture(scope="module")
def kernels():
    """Every kernel's own notes, by its name."""
    if not os.path.exists(ana_amd.LIB_PATH):
        from ana_amd import build
        build.build()
    with open(ana_amd.LIB_PATH, "rb") as f:
        data = f.read()
    out = {}
    for m in re.finditer(rb"\x07\0\0\0(....)\x20\0\0\0AMDGPU\0\0", data, re.DOTALL):
        note = msgpack.unpackb(data[m.end():m.end() + int.from_bytes(m[1], "little")])
        out.update({k[".name"]: k for k in note["amdhsa.kernels"]})
    return out


@pytest.mark.parametrize("typ,hd", list(WAVES))
def test_attention_over_own_positions(kernels, typ, hd):
    """What ana_kv4_attend launches for many rows is no wider for the forms
    that also take prefixes in."""
    found = [k for n, k in kernels.items() if f"k_kv4_manyI{typ}Li{hd}ELNS0_4SeenE0E" in n]
    assert len(found) == 1
    regs = -(-found[0][".vgpr_count"] // 8) * 8
    assert 512 // regs >= WAVES[typ, hd]
    assert found[0][".private_segment_fixed_size"] == 0
