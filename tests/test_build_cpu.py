"""When the Python binding is built again (no compiler runs: g++ is faked)."""

import os
import subprocess
import sysconfig

import torch

from qextract_infer_b200 import build


def test_the_binding_follows_torch_and_python(monkeypatch, tmp_path):
    runs = []

    def compiler(cmd, **kw):
        runs.append(cmd)
        with open(cmd[cmd.index("-o") + 1], "w") as f:
            f.write("binding")
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(build, "BINDING", str(tmp_path / "_binding.so"))
    monkeypatch.setattr(build, "BUILD", str(tmp_path / "_build"))
    monkeypatch.setattr(build.subprocess, "run", compiler)

    def built(**kw):
        n = len(runs)
        assert build.build_binding(**kw) == build.BINDING and os.path.exists(build.BINDING)
        return len(runs) - n

    assert built() == 1 and built() == 0 and built(force=True) == 1 and built() == 0
    monkeypatch.setattr(torch, "__version__", "0.0.1")
    assert built() == 1 and built() == 0
    monkeypatch.setattr(torch._C, "_GLIBCXX_USE_CXX11_ABI", not torch._C._GLIBCXX_USE_CXX11_ABI)
    assert built() == 1 and built() == 0
    soabi = sysconfig.get_config_var
    monkeypatch.setattr(sysconfig, "get_config_var", lambda n: "cpython-0" if n == "SOABI" else soabi(n))
    assert built() == 1 and built() == 0
    old = os.path.getmtime(os.path.join(build.CSRC, "binding.cpp")) - 10
    os.utime(build.BINDING, (old, old))
    assert built() == 1 and built() == 0
