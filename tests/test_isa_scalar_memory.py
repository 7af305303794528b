"""tools/isa_review.py tells scalar memory instructions by their encoding and allows loads alone."""
import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "tools"))
import isa_review  # noqa: E402


@pytest.mark.parametrize("line,bad", [
    ("s_load_dword s54, s[0:1], 0x108    // 0000000DE804: C0020D80 00000108", False),
    ("s_load_dwordx16 s[8:23], s[0:1], 0x0    // 0000000DE2B8: C0120200 00000000", False),
    ("s_buffer_load_dwordx2 s[4:5], s[8:11], 0x0    // 000000001000: C0260104 00000000", False),
    ("s_something s5, s[0:1], 0x0    // 000000001000: C0420140 00000000", True),  # of scalar memory, and no load
    ("s_load_other s5, s[0:1], 0x0    // 000000001000: C0420140 00000000", True),
    ("s_add_u32 s0, s0, s1    // 000000001000: 80000100", False),
    ("v_add_f32_e32 v0, v0, v1    // 000000001000: 02000300", False),
])
def test_scalar_memory_is_loads(line, bad):
    assert isa_review.scalar_write(line) == bad


def test_every_instruction_carries_its_encoding():
    """Without it the review would see no scalar memory at all."""
    if not os.path.exists(os.path.join(isa_review.LLVM, "clang-offload-bundler")):
        pytest.skip("ROCm LLVM tools not found")
    import tempfile
    with tempfile.TemporaryDirectory() as d:
        dis = isa_review.disassembly(isa_review.code_object(os.path.join(isa_review.PKG, "build", "gncde_norm.o"), d))
    lines = [x for ins in dis.values() for x in ins if x.startswith(("s_", "v_", "global_", "ds_", "buffer_"))]
    assert len(lines) > 1000 and all(isa_review.ENCODED.search(x) for x in lines)
    assert any(x.startswith("s_load_dword") for x in lines)
