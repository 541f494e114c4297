"""The build entry point (no GPU): what it compiles, and when."""
import re
import subprocess

import __graft_entry__ as entry
import gfx_ocean_amd as g


def test_build_compiles_also_where_a_library_is_there(monkeypatch):
    """A stale check by file times misses a change of the compile flags: build() runs hipcc every time it is called."""
    g.build_library()                                          # a library is there
    calls = []
    monkeypatch.setattr(subprocess, "check_call", lambda cmd, *a, **k: calls.append([str(c) for c in cmd]) or 0)
    entry.build()
    assert [c for c in calls if any("hipcc" in w for w in c[:1]) and "--offload-arch=gfx950" in c], calls


def test_the_library_holds_no_packed_fp32_arithmetic_and_no_spills(tmp_path):
    """Some forms of gfx950's packed fp32 instructions have given wrong values with no error: the compiler makes none.
    And no kernel spills a register: the flag that does it changed the 16-bit intermediate's pass 2 from 0 to 11."""
    cmd = g._lib.hipcc_command(out=str(tmp_path / "ocean.s"), extra=("--cuda-device-only", "-S"))
    i = cmd.index("-packed-fp32-ops")
    assert cmd[i - 3:i] == ["-Xclang", "-target-feature", "-Xclang"]
    subprocess.check_call(cmd)
    with open(tmp_path / "ocean.s") as f:
        text = f.read()
    assert text.count("v_fma_f32") > 1000                      # this is the library's assembly
    assert not re.findall(r"v_pk_(?:add|mul|fma)_f32", text)
    spills = [int(v) for v in re.findall(r"\.vgpr_spill_count:\s*(\d+)", text)]
    assert len(spills) > 50 and max(spills) == 0
