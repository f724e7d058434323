"""The C library builds where PyTorch, Python's headers or a host compiler are missing: only
the Python binding of the serving operators needs them.  (No compiler runs here.)"""
import importlib.util
import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture
def build(tmp_path, monkeypatch):
    spec = importlib.util.spec_from_file_location("coalibi_build_test", os.path.join(ROOT, "co-alibi_b200", "build.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    for name in ("OUT", "BINDING"):
        monkeypatch.setattr(mod, name, str(tmp_path / os.path.basename(getattr(mod, name))))
    ran = []

    def run(cmd, verbose, what):
        ran.append(what)
        open(cmd[cmd.index("-o") + 1], "w").close()
        return type("Done", (), {"stderr": ""})

    monkeypatch.setattr(mod, "_run", run)
    mod.ran = ran
    return mod


def test_all_there(build):
    build.build()
    assert build.ran == ["nvcc", "g++"] and os.path.exists(build.BINDING)


@pytest.mark.parametrize("missing", ["torch", "headers", "compiler"])
def test_one_is_missing(build, missing, monkeypatch, tmp_path, capsys):
    if missing == "torch":
        monkeypatch.setitem(sys.modules, "torch", None)
    elif missing == "headers":
        paths = build.sysconfig.get_paths()
        monkeypatch.setattr(build.sysconfig, "get_paths", lambda: {**paths, "include": str(tmp_path)})
    else:
        monkeypatch.setenv("CXX", str(tmp_path / "no-such-compiler"))
    assert build.build() == build.OUT and os.path.exists(build.OUT)
    assert build.ran == ["nvcc"] and not os.path.exists(build.BINDING)
    assert "binding" in capsys.readouterr().err
    with pytest.raises(RuntimeError, match="binding"):
        build.build(binding=True)
