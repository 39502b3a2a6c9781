"""The binding of the serving operators (`csrc/host_calls.cpp`): an operator's library is loaded for its own calls alone."""
import pytest

from logssms_b200.ops import build
from logssms_b200.ops import kernels as K

LIBRARIES = {"attention": "attention_shared", "adapters": "adapters", "rules": "logit_rules"}


@pytest.fixture
def loaded(monkeypatch):
    monkeypatch.setattr(K, "_serving_binding", None)
    monkeypatch.setattr(K, "_serving_known", set(), raising=False)
    names, load = [], build.load
    monkeypatch.setattr(build, "load", lambda name: (names.append(name), load(name))[1])
    return names


@pytest.mark.parametrize("operator", list(LIBRARIES))
def test_an_operator_loads_its_own_library(loaded, operator):
    K._serving_calls(operator)
    assert set(loaded) == {LIBRARIES[operator]}
    K._serving_calls(operator)
    assert len(loaded) == 1                              # asked for once


def test_one_behind_the_other(loaded):
    for operator in LIBRARIES:
        K._serving_calls(operator)
    assert loaded == list(LIBRARIES.values())


def test_what_does_not_build_takes_no_other_with_it(loaded, monkeypatch):
    load = build.load

    def broken(name):
        if name == "attention_shared":
            raise build.KernelBuildError("does not build")
        return load(name)

    monkeypatch.setattr(build, "load", broken)
    K._serving_calls("rules")
    with pytest.raises(build.KernelBuildError):
        K._serving_calls("attention")
    K._serving_calls("adapters")
