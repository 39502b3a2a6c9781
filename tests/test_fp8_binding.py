"""The host binding of the 8-bit operators on the CPU: what its built file is named after."""
import os
import sysconfig

from logssms_b200.ops import build


def test_another_interpreter_gets_a_build_of_its_own(monkeypatch):
    """A module compiled against one Python's headers is not loaded by another, nor removed when the other builds its own."""
    (name,) = build.package_bindings()
    here, kernel = build.library_path(name), build.library_path("fp8_rows")
    ask = sysconfig.get_config_var
    monkeypatch.setattr(sysconfig, "get_config_var", lambda key: "cpython-399-other" if key == "SOABI" else ask(key))
    there = build.library_path(name)
    assert there != here and os.path.basename(there).rsplit("-", 1)[0] != os.path.basename(here).rsplit("-", 1)[0]
    assert build.library_path("fp8_rows") == kernel        # the kernels' libraries know nothing of Python


def test_another_compiler_gets_a_build_of_its_own(monkeypatch):
    (name,) = build.package_bindings()
    monkeypatch.delenv("CXX", raising=False)
    here = build.library_path(name)
    monkeypatch.setenv("CXX", "/opt/other/bin/c++")
    assert build.library_path(name) != here
    monkeypatch.delenv("CXX")
    monkeypatch.setattr(build.shutil, "which", lambda tool: None)        # a machine that has none takes what was built elsewhere
    assert build.library_path(name) == here
