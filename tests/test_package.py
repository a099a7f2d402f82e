"""CPU: the package and its build where parts of the world are missing."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_everything_that_needs_no_torch_comes_without_it():
    code = ("import sys; sys.modules['torch'] = None\nfrom deep_contact_estimator_amd import *\nassert contact_cnn and load_checkpoint and synth.make_state_dict(1)\n"
            "import deep_contact_estimator_amd as d\n"
            "try: d.ops\nexcept ImportError: print('fine')")
    r = subprocess.run([sys.executable, "-c", code], env=dict(os.environ, PYTHONPATH=ROOT), capture_output=True, text=True, timeout=120, cwd=ROOT)
    assert r.returncode == 0 and "fine" in r.stdout, r.stderr[-800:]


def test_the_extension_module_belongs_to_one_torch_and_one_interpreter(monkeypatch):
    """another of either: another hash (so that it is compiled again), and what is there is not taken"""
    torch = pytest.importorskip("torch")
    import sysconfig

    from deep_contact_estimator_amd import _lib, build, ops
    if not os.path.exists(build.LIB):
        build.build()
    here = build.entries_hash()
    assert build.built_hash(build.ENTRIES) == here and ops._entries.__wrapped__().ABI == build.entries_abi()
    var = sysconfig.get_config_var
    with monkeypatch.context() as m:
        m.setattr(sysconfig, "get_config_var", lambda k: "cpython-399-x86_64-linux-gnu" if k == "SOABI" else var(k))
        assert build.entries_hash() != here
        with pytest.raises(RuntimeError, match="cpython-399"):
            ops._entries.__wrapped__()
    with monkeypatch.context() as m:
        m.setattr(torch, "__version__", "9.9")
        assert build.entries_hash() != here
        with pytest.raises(RuntimeError, match="this is torch 9.9"):
            ops._entries.__wrapped__()
    with monkeypatch.context() as m:
        m.setattr(torch._C, "_GLIBCXX_USE_CXX11_ABI", not torch._C._GLIBCXX_USE_CXX11_ABI)
        assert build.entries_hash() != here
    assert build.entries_hash() == here


@pytest.mark.parametrize("compiler", ["/nonexistent/g++", "false"])
def test_the_library_is_built_where_the_extension_module_is_not(monkeypatch, tmp_path, compiler):
    pytest.importorskip("torch")
    from deep_contact_estimator_amd import build
    made = []
    monkeypatch.setattr(build, "_build_lib", lambda force, verbose: made.append(force) or "libdce.so")
    monkeypatch.setattr(build, "ENTRIES", str(tmp_path / "_entries.so"))
    command = build._entries_command()
    monkeypatch.setattr(build, "_entries_command", lambda: [compiler, *command[1:]])
    with pytest.warns(UserWarning, match="_entries.so was not built"):
        assert build.build() == "libdce.so"
    assert made == [False]
    (tmp_path / "_entries.so").write_bytes(b"of other sources")
    with pytest.warns(UserWarning, match="_entries.so was not built"):
        build.build()
    assert not (tmp_path / "_entries.so").exists()
    with pytest.raises(RuntimeError):
        build.build_entries()
