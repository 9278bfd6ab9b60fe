"""The bf16 matrix products are asm, whose results the compiler takes for ready at once: no copy or spill of one may come too early
(tools/check_mfma_overlap.py, which tests/test_host_cpu.py runs over every source; here on planted texts)."""
import importlib.util
import os

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _tool():
    spec = importlib.util.spec_from_file_location("check_mfma_overlap", os.path.join(ROOT, "tools", "check_mfma_overlap.py"))
    tool = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(tool)
    return tool


P = "\tv_mfma_f32_16x16x32_bf16 v[0:3], v[8:11], v[12:15], v[0:3]\n"
Q = "\tv_mfma_f32_16x16x32_bf16 v[4:7], v[8:11], v[12:15], v[4:7]\n"
WAIT = "\ts_nop 7\n\ts_nop 7\n"


@pytest.mark.parametrize("text,found", [
    (P + WAIT + "\tv_add_f32_e32 v0, v0, v9\n", 0),
    (P + Q + P + Q + WAIT + "\tv_add_f32_e32 v20, v0, v4\n", 0),                       # a chain of products waits for itself
    (P + "\tv_mov_b32_e32 v20, v3\n" + WAIT, 1),                                        # a copy
    (P + "\tscratch_store_dwordx4 off, v[0:3], off offset:16\n" + WAIT, 1),             # a spill
    (P + "\ts_nop 7\n\tv_add_f32_e32 v20, v1, v9\n", 1),                               # not long enough
    (P + "\ts_nop 7\n\ts_nop 1\n\ts_nop 0\n\tv_add_f32_e32 v20, v1, v9\n", 0),
    (P + "\tds_read_b128 v[0:3], v30\n" + WAIT, 1),                                     # overwritten while it is on its way
    (P + "\tv_mfma_f32_16x16x32_bf16 v[4:7], v[0:3], v[12:15], v[4:7]\n" + WAIT, 1),   # an operand of another product
    (P + "\ts_cbranch_scc1 .LBB0_2\n" + WAIT + "\ts_branch .LBB0_3\n.LBB0_2:\n\tv_mov_b32_e32 v20, v1\n.LBB0_3:\n\tv_mov_b32_e32 v21, v1\n", 2),   # both, by the branch
    (".LBB0_1:\n\tv_mov_b32_e32 v20, v1\n" + P + "\ts_cbranch_scc1 .LBB0_1\n" + WAIT, 1),   # round a loop
])
def test_early_accesses_are_found(tmp_path, text, found):
    asm = tmp_path / "x.s"
    asm.write_text("_Z6kernelv:\n" + text + "\ts_endpgm\n.Lfunc_end0:\n")
    assert len(_tool().scan_unfinished(str(asm))) == found
