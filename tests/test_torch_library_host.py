"""The library of torch operators: what runs without it, and that one built for another torch is neither loaded nor kept."""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from fp8_b200 import build

PACKAGE = Path(build.__file__).resolve().parent


@pytest.fixture()
def copy(tmp_path):
    """The package, with its library of kernels and without the one of torch operators."""
    to = tmp_path / "fp8_b200"
    shutil.copytree(PACKAGE, to, ignore=shutil.ignore_patterns("_build", "__pycache__", "libfp8torch.so"))
    return to


def _python(copy, code):
    env = {**os.environ, "PYTHONPATH": str(copy.parent)}
    return subprocess.run([sys.executable, "-c", code], env=env, capture_output=True, text=True)


FP8_ALONE = """
import torch, fp8_b200
from fp8_b200.unet import UNet, UNetConfig
UNet(UNetConfig())
assert not hasattr(torch.ops.fp8_b200, "cross_attention")
"""


def test_the_fp8_operators_run_without_it(copy):
    done = _python(copy, FP8_ALONE)
    assert done.returncode == 0, done.stderr
    done = _python(copy, "import fp8_b200.cross_attention")
    assert done.returncode != 0 and "libfp8torch.so is missing" in done.stderr
    done = _python(copy, "from fp8_b200.unet import UNet, UNetConfig; UNet(UNetConfig(prompt_vocab=9))")
    assert done.returncode != 0 and "libfp8torch.so is missing" in done.stderr


def test_one_of_another_torch_is_not_loaded(copy):
    library = (PACKAGE / "libfp8torch.so").read_bytes()
    mark = (build.TORCH_MARK + torch.__version__).encode()
    assert library.count(mark) == 1
    (copy / "libfp8torch.so").write_bytes(library.replace(mark, mark[:-1] + b"?"))
    done = _python(copy, FP8_ALONE)
    assert done.returncode == 0, done.stderr
    done = _python(copy, "import fp8_b200.embedding")
    assert done.returncode != 0 and "another torch" in done.stderr


def test_one_of_another_torch_is_built_again(monkeypatch):
    assert build.torch_library_fits(torch.__version__)
    assert not build.torch_library_fits(torch.__version__[:-1])
    assert not build.torch_library_fits(torch.__version__, PACKAGE / "missing.so")
    monkeypatch.setattr(build, "sources", lambda: [])
    assert not build.needs_rebuild()
    monkeypatch.setattr(torch, "__version__", "0.0.1")
    assert build.needs_rebuild()
