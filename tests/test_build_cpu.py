"""What __graft_entry__.build() compiles."""
import glob
import os

import pytest


@pytest.mark.parametrize("force", [None, False])
def test_every_source_is_compiled_every_time(force, tmp_path, monkeypatch):
    """also where everything is built and newer than its sources; force=False compiles what is older than its sources"""
    import __graft_entry__ as g
    from lgd_amd import hip
    if not os.path.exists(hip.lib_path()):
        g.build()
    monkeypatch.setattr(g.sys, "path", list(g.sys.path))
    monkeypatch.setattr(g, "ROOT", str(tmp_path))
    monkeypatch.setattr(g, "LIB", str(tmp_path / "lgd_amd" / "_lib" / "liblgd_hip.so"))
    ran = []

    def compiler(cmd, cwd):
        ran.append(cmd)
        open(cmd[cmd.index("-o") + 1], "w").close()
    monkeypatch.setattr(g.subprocess, "check_call", compiler)
    header = tmp_path / "include"
    header.mkdir()
    (header / "lgd_hip.h").write_text("")
    g.build()
    everything = len(glob.glob(os.path.join(g.CSRC, "*.hip"))) + 2   # objects, the library, the host extension
    assert len(ran) == everything and not glob.glob(str(tmp_path / "**" / "*.new"), recursive=True)
    g.build() if force is None else g.build(force=force)
    assert len(ran) == (2 * everything if force is None else everything)
