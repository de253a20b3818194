"""CPU checks of the host side around the window attention and 8-bit cache
calls: helpers of the package, split counts, the build of the binding."""
import ctypes
import math
import os
import subprocess
import sysconfig

import pytest
import torch

from grout_b200 import attn, build


def test_default_scale():
    """The softmax scale that the attention calls use where none is given."""
    assert attn.default_scale() == 1.0 / math.sqrt(128)
    assert attn.default_scale(64) == 0.125


def _no_binding(monkeypatch):
    monkeypatch.setattr(attn, "_bind", None)
    with pytest.raises(attn.GroutError, match="python -m grout_b200.build"):
        attn._load_bind()


def test_binding_belongs_to_one_pytorch(monkeypatch):
    """After a change of PyTorch or Python the binding that was built for the
    other one is neither up to date nor loaded."""
    build.build()
    assert build.up_to_date()
    attn._load_bind()
    with monkeypatch.context() as m:
        m.setattr(torch, "__version__", "0.1.0")
        assert not build.up_to_date()
        _no_binding(m)
    with monkeypatch.context() as m:
        m.setattr(sysconfig, "get_config_var", lambda name: ".cpython-39-x86_64-linux-gnu.so")
        assert not build.up_to_date()
        _no_binding(m)
    assert build.up_to_date()


@pytest.fixture
def scratch(monkeypatch, tmp_path):
    """A library of one small source, built elsewhere."""
    src = tmp_path / "one.cu"
    src.write_text('extern "C" int one() { return 1; }\n')
    monkeypatch.setattr(build, "HERE", str(tmp_path))
    monkeypatch.setattr(build, "LIB", str(tmp_path / "libone.so"))
    monkeypatch.setattr(build, "BUILD_DIR", str(tmp_path / "_build"))
    monkeypatch.setattr(build, "_sources", lambda: [str(src)])
    return tmp_path


def test_library_builds_without_the_binding(monkeypatch, scratch):
    """A binding that does not compile, or PyTorch missing, leaves the C library built."""
    def without_torch(out):
        raise ImportError("no torch")

    monkeypatch.setattr(build, "_bind_command", lambda out: ["false"])
    with pytest.raises(RuntimeError, match="compilation failed: false"):
        build.build()
    assert ctypes.CDLL(build.LIB).one() == 1
    os.remove(build.LIB)
    monkeypatch.setattr(build, "_bind_command", without_torch)
    assert build.build() == build.LIB
    assert ctypes.CDLL(build.LIB).one() == 1


def test_a_failed_build_leaves_no_compiler_running(monkeypatch, scratch):
    with open(scratch / "one.cu", "w") as f:
        f.write("this is no code\n")
    started = []
    popen = subprocess.Popen
    monkeypatch.setattr(build.subprocess, "Popen", lambda cmd: started.append(popen(cmd)) or started[-1])
    monkeypatch.setattr(build, "_sources", lambda: [str(scratch / "one.cu"), str(scratch / "none.cu")])
    with pytest.raises(RuntimeError, match="compilation failed"):
        build.build()
    assert len(started) == 2 and all(p.returncode not in (None, 0) for p in started)
    assert not os.path.exists(build.LIB)


@pytest.mark.parametrize("fp8", [False, True])
def test_split_count_of_large_batches(fp8):
    """Long contexts: two splits up to three units (sequence and KV head) per SM,
    one for batches of more, however many."""
    count = lambda units, keys: attn.decode_window_splits(units, keys, keys, 0, 4, 1, 1 << 20, fp8=fp8)  # noqa: E731
    sms = 148  # of a B200, and what is assumed where there is no device
    for units in (160, 300, 3 * sms):
        assert count(units, 16384) == 2
        assert count(units, 1 << 19) == 2
        assert count(units, 16320) == 1  # 255 tiles
    for units in (3 * sms + 1, 512, 2048, 65535):
        assert count(units, 16384) == count(units, 1 << 19) == 1
