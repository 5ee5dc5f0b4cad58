"""The two compiled files and when they are built."""

import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_the_optimizers_do_not_need_the_module_built_for_torch():
    """Importing the package loads the kernel library only; the activations' C++ host side comes with their first call."""
    code = (
        "import torch, optimi_b200, optimi_b200._lib as lib\n"
        "optimi_b200.AdamW([torch.zeros(3, requires_grad=True)], lr=1e-3)\n"
        "assert 'HOST' not in vars(lib)\n"
        "try: optimi_b200.activations.compress(torch.zeros(3))\n"
        "except RuntimeError as e: assert 'CUDA tensors only' in str(e)\n"
        "assert 'HOST' in vars(lib) and lib.HOST is lib.HOST\n"
        "try: lib.OTHER\n"
        "except AttributeError: print('fine')\n"
    )
    res = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=ROOT)
    assert res.returncode == 0 and "fine" in res.stdout, res.stdout + res.stderr


def test_another_torch_makes_only_the_host_module_stale(tmp_path, monkeypatch):
    from optimi_b200 import build

    build.build()
    assert build.up_to_date() and build.host_up_to_date()
    (tmp_path / "version.py").write_text("__version__ = 'another'\n")
    monkeypatch.setattr(build, "torch_dir", lambda: str(tmp_path))
    assert build.up_to_date() and not build.host_up_to_date()
    monkeypatch.setattr(build, "HOST_LIB", str(tmp_path / "missing.so"))
    assert build.up_to_date() and not build.host_up_to_date()
    compiled = []
    monkeypatch.setattr(build, "find_nvcc", lambda: pytest.fail("nvcc is not needed"))
    assert build.build(host=False) == build.LIB
    monkeypatch.setattr(build, "host_compile", lambda obj: compiled.append(obj) or ["true"])
    monkeypatch.setattr(build, "host_link", lambda obj, lib, out: ["touch", out])
    monkeypatch.setattr(build, "HOST_STAMP", str(tmp_path / "missing.so.srchash"))
    build.build()
    assert len(compiled) == 1 and build.host_up_to_date()
