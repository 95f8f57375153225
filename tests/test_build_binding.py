"""CPU tests of the quantised ops' binding as a part that the library does without: its build, its
stamp, and the ops where it is missing."""
import os

import pytest
import torch

from gpu_offloading_amd import _lib, build
from gpu_offloading_amd import quantized as qz


@pytest.fixture
def tools(tmp_path, monkeypatch):
    """A build into tmp_path whose compilers are stand-ins: ``bad`` names what fails."""
    lib = tmp_path / "lib"
    for name, file in (("LIB_DIR", ""), ("LIB_PATH", "libkvc.so"),
                       ("STAMP_PATH", "libkvc.so.srchash"), ("BIND_PATH", "kvc_bind.so"),
                       ("BIND_STAMP_PATH", "kvc_bind.so.srchash")):
        monkeypatch.setattr(build, name, str(lib / file), raising=False)
    bad = set()

    def run(cmd):
        made = cmd[cmd.index("-o") + 1]
        if any(b in part for b in bad for part in cmd):
            return 1, ["no such header"]
        with open(made, "w") as f:
            f.write(" ".join(cmd))
        return 0, []

    monkeypatch.setattr(build, "_run", run)
    monkeypatch.setattr(build, "hipcc", lambda: "hipcc")
    return lib, bad


def files(lib):
    return sorted(f for f in os.listdir(lib) if f != "obj")


BOTH = ["kvc_bind.so", "kvc_bind.so.srchash", "libkvc.so", "libkvc.so.srchash"]


def test_the_library_is_built_without_its_binding(tools, capfd):
    lib, bad = tools
    assert build.build_library() == str(lib / "libkvc.so") and files(lib) == BOTH
    bad.add("bind.cpp")
    assert build.build_library() == str(lib / "libkvc.so")
    assert files(lib) == ["libkvc.so", "libkvc.so.srchash"]    # (nor is an older binding left)
    assert "no such header" in capfd.readouterr().err
    assert open(build.STAMP_PATH).read().strip() == build.source_hash()
    bad.clear()
    build.build_library()
    assert files(lib) == BOTH


def test_the_library_is_built_without_torch_or_a_host_compiler(tools, monkeypatch, capfd):
    import importlib.util

    lib, _ = tools
    find = importlib.util.find_spec
    with monkeypatch.context() as p:
        p.setattr(importlib.util, "find_spec", lambda name, *a: None if name == "torch" else find(name, *a))
        build.build_library()
        assert files(lib) == ["libkvc.so", "libkvc.so.srchash"]
        assert "torch" in capfd.readouterr().err
    run = build._run

    def no_gcc(cmd):
        if cmd[0] == "g++":
            raise FileNotFoundError("g++")
        return run(cmd)

    monkeypatch.setattr(build, "_run", no_gcc)
    build.build_library()
    assert files(lib) == ["libkvc.so", "libkvc.so.srchash"]
    assert "g++" in capfd.readouterr().err


def test_a_source_that_does_not_compile_still_fails_the_build(tools):
    lib, bad = tools
    bad.add("quant_decode.hip")
    with pytest.raises(RuntimeError, match="no such header"):
        build.build_library()
    assert files(lib) == []


def refused(m):
    """The ops find nothing in ``m`` and go on in Python, which refuses what is not on a GPU."""
    for f in (m.write, m.read, m.decode):
        assert f() is None and f(1, 2, 3) is None
    c = qz.quantized_cache(4, 2, 64, torch.int8, "cpu")[:3]
    k = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        qz.reshape_and_cache_quantized(k, k, *c, torch.arange(3))


def test_ops_do_without_the_binding(tmp_path, monkeypatch):
    monkeypatch.setattr(build, "BIND_PATH", str(tmp_path / "kvc_bind.so"))
    monkeypatch.setattr(_lib, "_bind", None)
    with pytest.warns(RuntimeWarning, match="not built"):
        m = _lib.binding()
    assert _lib.binding() is m          # (said once)
    refused(m)


def test_a_binding_that_does_not_load_is_done_without(tmp_path, monkeypatch):
    path = tmp_path / "kvc_bind.so"
    path.write_bytes(b"not a library")
    monkeypatch.setattr(build, "BIND_PATH", str(path))
    monkeypatch.setattr(_lib, "_bind", None)
    with pytest.warns(RuntimeWarning, match="kvc_bind"):
        refused(_lib.binding())


def test_a_binding_of_another_torch_is_not_loaded(monkeypatch):
    """Its C++ calls are those of the torch that it was built against."""
    _lib.load()
    with monkeypatch.context() as p:
        p.setattr(torch, "__version__", "0.0.1")
        p.setattr(_lib, "_bind", None)
        with pytest.warns(RuntimeWarning, match="another torch"):
            refused(_lib.binding())
        assert open(build.STAMP_PATH).read().strip() == build.source_hash()    # (the library's stays)
    monkeypatch.setattr(_lib, "_bind", None)
    assert type(_lib.binding()).__name__ == "module"
