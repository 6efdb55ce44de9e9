"""Builds that run at once (ranks of one node on a fresh checkout) do not write into each other's output."""

from __future__ import annotations

import os
import subprocess
import threading

import pytest

from turbo_roformer_b200 import _build


@pytest.mark.parametrize("build,path", [("build", "LIB_PATH"), ("build_binding", "BINDING_PATH")])
def test_builds_at_once(monkeypatch, tmp_path, build, path):
    """Three compilers write their outputs half, wait for each other and finish: every build ends with a whole library."""
    target = tmp_path / "lib.so"
    monkeypatch.setattr(_build, path, str(target))
    meet, outputs = threading.Barrier(3, timeout=60), []

    def compiler(cmd, **kw):
        out = cmd[cmd.index("-o") + 1]
        outputs.append(out)
        with open(out, "w") as f:
            f.write("first half ")
            f.flush()
            meet.wait()
            f.write("second half")
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(_build.subprocess, "run", compiler)
    results = []
    threads = [threading.Thread(target=lambda: results.append(getattr(_build, build)(force=True))) for _ in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert results == [str(target)] * 3
    assert len(set(outputs)) == 3
    assert target.read_text() == "first half second half"
    assert sorted(os.listdir(tmp_path)) == ["lib.so", "lib.so.hash"]


@pytest.mark.parametrize("build,path", [("build", "LIB_PATH"), ("build_binding", "BINDING_PATH")])
def test_failed_build_leaves_nothing(monkeypatch, tmp_path, build, path):
    monkeypatch.setattr(_build, path, str(tmp_path / "lib.so"))

    def compiler(cmd, **kw):
        open(cmd[cmd.index("-o") + 1], "w").close()
        return subprocess.CompletedProcess(cmd, 1, "", "no such thing")

    monkeypatch.setattr(_build.subprocess, "run", compiler)
    with pytest.raises(RuntimeError, match="no such thing"):
        getattr(_build, build)(force=True)
    assert os.listdir(tmp_path) == []


def test_binding_follows_the_header(monkeypatch, tmp_path):
    """The binding takes the C ABI's signatures and limits from the header: a changed header means a new binding."""
    include = tmp_path / "include"
    include.mkdir()
    with open(os.path.join(_build.INCLUDE, "trcuda.h")) as f:
        text = f.read()
    (include / "trcuda.h").write_text(text)
    monkeypatch.setattr(_build, "BINDING_PATH", str(tmp_path / "lib.so"))
    monkeypatch.setattr(_build, "INCLUDE", str(include))
    compiled = []

    def compiler(cmd, **kw):
        compiled.append(cmd)
        open(cmd[cmd.index("-o") + 1], "w").close()
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(_build.subprocess, "run", compiler)
    for expected in (1, 1):
        _build.build_binding()
        assert len(compiled) == expected
    (include / "trcuda.h").write_text(text.replace("TRC_CACHE_MAX_WHOLE 512", "TRC_CACHE_MAX_WHOLE 256"))
    _build.build_binding()
    assert len(compiled) == 2
    with open(_build.BINDING_SOURCE) as f:
        source = f.read()
    assert "512" not in source and "TRC_CACHE_MAX_WHOLE" in source
