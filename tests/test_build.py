"""What a build compiles again."""
import os

from wavernn_amd import build as B


def test_changed_flags_compile_everything_again(tmp_path, monkeypatch):
    """The compilers' flags stand in build.py: a change there makes every object stale (some flags decide whether kernels are right)."""
    here = tmp_path / "build.py"
    here.write_text("")
    ran = []

    def run(cmd, check):
        ran.append(cmd)
        open(cmd[cmd.index("-o") + 1], "w").close()

    monkeypatch.setattr(B, "LIB_DIR", str(tmp_path))
    monkeypatch.setattr(B, "OBJ_DIR", str(tmp_path / "obj"))
    monkeypatch.setattr(B, "LIB_PATH", str(tmp_path / "lib.so"))
    monkeypatch.setattr(B, "__file__", str(here))
    monkeypatch.setattr(B.subprocess, "run", run)
    assert B.needs_build()
    B.build(verbose=False)
    assert len(ran) == len(B.SOURCES) + 1
    assert not B.needs_build()
    B.build(verbose=False)
    assert len(ran) == len(B.SOURCES) + 1
    t = os.path.getmtime(B.LIB_PATH) + 10
    os.utime(here, (t, t))
    assert B.needs_build()
    B.build(verbose=False)
    assert len(ran) == 2 * (len(B.SOURCES) + 1)
