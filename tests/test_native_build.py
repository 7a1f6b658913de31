"""CPU: the compiled Python module belongs to the torch and the Python it was built against."""
import os
import subprocess

import pytest
import torch

from qlinear import decoder

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mlx-gen_b200", "csrc")


def script(path, text):
    path.write_text("#!/bin/sh\n" + text)
    path.chmod(0o755)
    return str(path)


def test_another_torch_rebuilds_the_module(tmp_path):
    """With a compiler that only notes that it ran, and a Python whose answer stands for its torch."""
    (tmp_path / "torch").write_text("one")
    cxx = script(tmp_path / "cxx", f"echo built >> {tmp_path}/log\ntouch {tmp_path}/module.so\n")
    python = script(tmp_path / "python", f"cat {tmp_path}/torch\n")
    call = ["make", "-s", "-C", CSRC, f"{tmp_path}/module.so", f"NATIVE={tmp_path}/module.so", f"STAMP={tmp_path}/stamp",
            f"PYTHON={python}", f"HOSTCXX={cxx}"]
    built = lambda: (tmp_path / "log").read_text().count("built")  # noqa: E731
    for torch_is, times in (("one", 1), ("one", 1), ("two", 2), ("two", 2)):
        (tmp_path / "torch").write_text(torch_is)
        subprocess.run(call, check=True, capture_output=True)
        assert built() == times


def test_a_module_of_another_torch_is_refused(monkeypatch):
    assert decoder._Native().norm_residual
    monkeypatch.setattr(torch, "__version__", "1.0.0")
    with pytest.raises(ImportError, match="built for torch"):
        decoder._Native().norm_residual
