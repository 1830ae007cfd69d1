"""What build_native compiles, with the compilers replaced by a stand-in that writes empty outputs."""
import glob
import os

import pytest

import build_native


@pytest.fixture
def compiled(tmp_path, monkeypatch):
    calls = []

    def run(cmd):
        out = cmd[cmd.index("-o") + 1]
        open(out, "w").close()
        calls.append(os.path.basename(cmd[cmd.index("-c") + 1]) if "-c" in cmd else os.path.basename(out))
        return 0, " ".join(cmd), ""
    monkeypatch.setattr(build_native, "_run", run)
    monkeypatch.setattr(build_native, "OUT_DIR", str(tmp_path / "lib"))
    monkeypatch.setattr(build_native, "BUILD_DIR", str(tmp_path / "obj"))
    return calls


def test_everything_once_then_nothing_then_everything_by_force(compiled):
    sources = {os.path.basename(f) for p in ("*.hip", "runtime/*.cpp") for f in glob.glob(os.path.join(build_native.CSRC, p))}
    links = {"libtdl_kernels.so.tmp", "libtdl_runtime.so.tmp"}
    build_native.build()
    assert set(compiled) == sources | links
    compiled.clear()
    build_native.build()
    assert not compiled
    build_native.build(force=True)
    assert set(compiled) == sources | links
