"""The build entry point (no GPU): what it compiles, and when."""
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
