"""Wait states of the row matching kernels' inline asm (loads to LDS whose address is in scalar registers), on the code
that the compiler emits for them."""
import os
import shutil
import subprocess
import sys

import pytest

from custereomatching_amd import build

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "custereomatching_amd"))
import hazard_check as hc  # noqa: E402
import vmcnt_check as vc  # noqa: E402

ASM = ";;#ASMSTART\n{}\n;;#ASMEND\n"


def _hits(body, tool):
    lines = ("_Zk:\n" + body + "\ts_endpgm\n.Lfunc_end0:\n").split("\n")
    return [h for _, (a, b) in tool.kernels(lines, []).items() for h in tool.check_kernel(lines, a, b)]


@pytest.mark.parametrize("nop,flagged", [(0, True), (2, True), (3, False)])
@pytest.mark.parametrize("writer", ["v_readfirstlane_b32 s4, v9", "v_readlane_b32 s4, v9, 3"])
def test_scalar_address_written_just_before(writer, nop, flagged):
    body = f"\t{writer}\n" + ASM.format(f"\ts_mov_b32 m0, s1\n\ts_nop {nop}\n\tglobal_load_lds_dwordx4 v2, s[4:5]")
    assert [h[0] for h in _hits(body, hc)] == (["R1"] if flagged else [])


def test_load_to_lds_has_no_register_in_flight():
    body = ASM.format("\tglobal_load_lds_dwordx4 v2, s[4:5]") + "\tv_add_u32_e32 v2, v1, v3\n"
    assert not _hits(body, vc)
    body = ASM.format("\tglobal_load_dwordx4 v[4:7], v2, s[4:5]") + "\tv_add_u32_e32 v4, v1, v3\n"
    assert _hits(body, vc)


def test_build_checks_every_unit_with_such_loads():
    for src in build.SOURCES:
        with open(os.path.join(build.CSRC, src)) as f:
            if any(w in f.read() for w in ("Filler<", "fill_tile<", "fill_rows<", "load_lds")):
                assert src in build.WAIT_CHECKED + build.HAZARD_CHECKED, src


@pytest.mark.skipif(shutil.which(build.HIPCC) is None, reason="no hipcc")
@pytest.mark.parametrize("name", ["match_bwd_c32", "match_fwd_c32", "match_wide"])
def test_listings_are_clean(name, tmp_path):
    unit = next(u for u in build.UNITS if u[0] == name)
    out = tmp_path / "k.s"
    r = subprocess.run([build.HIPCC, *build._flags(unit), "--cuda-device-only", "-S", os.path.join(build.CSRC, unit[1]), "-o",
                        str(out)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    assert "global_load_lds_dword" in out.read_text()
    assert hc.main(["hazard_check.py", str(out)]) == 0
