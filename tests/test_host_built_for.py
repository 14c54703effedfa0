"""CPU: the helper that reads torch's objects by their layout is refused under another torch or Python than it was built for."""
import sys

import pytest
import torch

from neat_amd import lib


def test_it_says_what_it_was_built_for():
    lib.step_list()
    assert lib._host_lib().neat_host_for().decode() == "torch %s, Python %d.%d" % (torch.__version__, *sys.version_info[:2])


def test_another_torch_is_refused(monkeypatch):
    monkeypatch.setattr(lib, "_host", None)
    monkeypatch.setattr(torch, "__version__", "9.9.9")
    with pytest.raises(RuntimeError, match="built for torch .*this is torch 9.9.9.*make -C neat_amd/csrc host"):
        lib.step_list()
    assert lib._host is None                         # and stays refused
    with pytest.raises(RuntimeError, match="build it anew"):
        lib.written()


def test_a_helper_that_does_not_say_is_refused(monkeypatch, tmp_path):
    (tmp_path / "libneat_host.so").write_bytes(b"no library")
    monkeypatch.setattr(lib, "_host", None)
    monkeypatch.setattr(lib, "_HERE", str(tmp_path))
    with pytest.raises(RuntimeError, match="build it anew"):
        lib.step_list()
