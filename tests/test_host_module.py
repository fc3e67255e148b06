"""The module of the small calls' host side: compiled against one torch and one Python, and found by no other."""
import os
import sysconfig

import pytest
import torch

from nemicli_terminal_b200 import _lib, build


def other_torch(m):
    m.setattr(torch, "__version__", "9.9.9")


def other_commit(m):
    m.setattr(torch.version, "git_version", "0" * 40)


def other_abi(m):
    m.setattr(torch._C, "_GLIBCXX_USE_CXX11_ABI", not torch._C._GLIBCXX_USE_CXX11_ABI)


def other_python(m):
    real = sysconfig.get_config_var
    m.setattr(sysconfig, "get_config_var", lambda name: "cpython-399-x" if name == "SOABI" else real(name))


def test_is_there():
    assert os.path.exists(build.host_path())
    assert _lib.host().__file__ == build.host_path()


@pytest.mark.parametrize("change", [other_torch, other_commit, other_abi, other_python])
def test_of_another_environment_is_not_taken(monkeypatch, change):
    """It has torch's inline accessors compiled in: against another layout it would read wrong pointers."""
    change(monkeypatch)
    assert build._host_stale() and not os.path.exists(build.host_path())
    monkeypatch.setattr(_lib, "_host", None)
    with pytest.raises(RuntimeError, match="module missing"):
        _lib.host()
