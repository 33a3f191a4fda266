"""The hazard check's rule for scalar registers that vector instructions write
ahead of an LDS-direct load, and the text operators' code object under it."""
import os

import pytest

from conftest import ROOT
from test_hazard_check import hc, kinds

LOAD = "buffer_load_dwordx4 v1, s[4:7], s9 offen lds"


@pytest.mark.parametrize("body, want", [
    (["v_readfirstlane_b32 s6, v7", LOAD], [("vsgpr->lds", 0, 5)]),
    (["v_readlane_b32 s9, v7, 3", "s_mov_b32 m0, s1", "s_nop 0", LOAD], [("vsgpr->lds", 2, 5)]),
    (["v_readlane_b32 s9, v7, 3", "s_mov_b32 m0, s1", "s_nop 3", LOAD], []),
    (["v_readlane_b32 s8, v7, 3", "s_mov_b32 m0, s1", "s_nop 0", LOAD], []),  # not read
    (["v_cmp_eq_u32_e64 s[4:5], v1, v2", "s_mov_b32 m0, s1", "s_nop 0", LOAD],
     [("vsgpr->lds", 2, 5)]),
    (["s_add_u32 s4, s2, s3", "s_mov_b32 m0, s1", "s_nop 0", LOAD], []),  # scalar writes wait
])
def test_scalar_written_by_a_vector_instruction(body, want):
    assert kinds(body) == want


def test_text_code_object_is_clean():
    hsaco = os.path.join(ROOT, "qwen-metal_amd", "lib", "qwen_text_kernels.hsaco")
    if not os.path.exists(os.path.join(hc.LLVM, "llvm-objdump")):
        pytest.skip("llvm-objdump absent")
    funcs = hc.functions(hc.disassemble(hsaco))
    assert any(any(x.lds_dma for x in v) for v in funcs.values())
    bad = [b for b in hc.check(funcs) if b[1].endswith("->lds")]
    assert not bad, [(b[0], b[1], b[2], b[3], b[4].text, b[5].text) for b in bad[:5]]
