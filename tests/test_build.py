"""The build where torch or a part of what its binding needs is absent: the library needs none of them."""
import importlib.util
import os
import shutil
import sysconfig

import pytest

from dtts import LIB_PATH


@pytest.fixture
def build(monkeypatch, tmp_path):
    spec = importlib.util.spec_from_file_location("dtts_build", os.path.join(os.path.dirname(LIB_PATH), "build.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    monkeypatch.setattr(module, "BINDING", str(tmp_path / "_serving.so"))
    return module


@pytest.mark.parametrize("missing", ["torch", "a ROCm torch's headers", "Python.h", "g++"])
def test_no_binding_without_what_it_needs(build, monkeypatch, tmp_path, capsys, missing):
    if missing == "torch":
        monkeypatch.setattr(importlib.util, "find_spec", lambda name: None)
    elif missing == "g++":
        monkeypatch.setattr(shutil, "which", lambda name: None)
    elif missing == "Python.h":
        monkeypatch.setattr(sysconfig, "get_paths", lambda: {"include": str(tmp_path)})
    else:
        found = importlib.util.spec_from_loader("torch", None)
        found.submodule_search_locations = [str(tmp_path)]
        monkeypatch.setattr(importlib.util, "find_spec", lambda name: found)
    with open(build.BINDING, "w") as f:
        f.write("of another torch")
    assert build.build_binding() is None
    assert missing in capsys.readouterr().err and not os.path.exists(build.BINDING)


def test_headers_beside_the_compiler_in_use(build, monkeypatch, tmp_path):
    (tmp_path / "bin").mkdir()
    (tmp_path / "bin" / "hipcc").touch(mode=0o755)
    monkeypatch.setattr(build, "HIPCC", str(tmp_path / "bin" / "hipcc"))
    assert build._rocm_include() == str(tmp_path / "include")
