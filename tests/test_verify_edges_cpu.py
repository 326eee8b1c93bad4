"""Edges of the verification operators' host-side parts (no GPU)."""

import math
import subprocess

import pytest
import torch

import torch_spyre_b200 as tsb
from tests.test_verify_cpu import store
from torch_spyre_b200 import _eager, _lib, build


# ------------------------------------------------------------------ tables --
@pytest.mark.parametrize("rotary_dim,base,original,factor", [
    (128, 1e4, 131072, 4.0),  # the slow end of the ramp lies past the last pair
    (128, 1e4, 65536, 8.0),
    (16, 1e4, 32768, 4.0),
    (4, 1e4, 4096, 4.0),
    (64, 1e5, 2048, 8.0),  # and here before it
    (128, 5e5, 8192, 32.0),
])
def test_yarn_ramp(rotary_dim, base, original, factor):
    """Pair i's frequency against the definition, pair by pair: the ramp is linear in the index between the
    (real) indices that turn beta_fast = 32 times and once over the original context, rounded outwards."""
    t = tsb.rotary_table(2, rotary_dim, base=base, scaling="yarn", factor=factor, original_max_pos=original)
    got = torch.atan2(t[1, :, 1].double(), t[1, :, 0].double())

    def index_of(turns):  # base^(-2 i / rotary_dim) * original = 2 pi turns
        return rotary_dim / 2 * math.log(original / (2 * math.pi * turns)) / math.log(base)

    lo, hi = max(math.floor(index_of(32.0)), 0), min(math.ceil(index_of(1.0)), rotary_dim - 1)
    for i in range(rotary_dim // 2):
        inv = base ** (-2.0 * i / rotary_dim)
        part = min(max((i - lo) / (hi - lo), 0.0), 1.0)  # of the interpolated frequency
        want = inv * (1 - part) + inv / factor * part
        assert math.isclose(float(got[i]), want, rel_tol=1e-6), i
        turns = original * inv / (2 * math.pi)
        if turns > 1.0:  # a pair that turns is not interpolated whole
            assert float(got[i]) > inv / factor * (1 + 1e-6)
        assert math.isclose(float(t[1, i].double().norm()), 0.1 * math.log(factor) + 1, rel_tol=1e-6)


# ------------------------------------------------------------------- build --
class Tools:
    """In place of subprocess.run: writes what the compilers would."""

    def __init__(self, monkeypatch, tmp_path, gxx):
        self.ran, self.gxx = [], gxx
        for name in ("LIB_DIR", "LIB_PATH", "FAST_PATH"):
            monkeypatch.setattr(build, name, tmp_path / "lib" / getattr(build, name).name if name != "LIB_DIR"
                                else tmp_path / "lib")
        monkeypatch.setattr(build.subprocess, "run", self.run)
        monkeypatch.setattr(build, "nvcc_path", lambda: "/somewhere/bin/nvcc")

    def run(self, cmd, **kw):
        tool = cmd[0].split("/")[-1]
        self.ran.append(tool)
        if tool == "g++" and self.gxx != "works":
            if self.gxx == "absent":
                raise FileNotFoundError("g++")
            return subprocess.CompletedProcess(cmd, 1, "", "Python.h: No such file or directory")
        with open(cmd[cmd.index("-o") + 1], "w") as f:
            f.write(tool)
        return subprocess.CompletedProcess(cmd, 0, "", "")


@pytest.mark.parametrize("gxx", ["absent", "fails", "works"])
def test_the_library_is_built_without_a_host_compiler_of_torch_extensions(monkeypatch, tmp_path, gxx):
    tools = Tools(monkeypatch, tmp_path, gxx)
    if gxx == "works":
        build.build()
    else:
        with pytest.warns(RuntimeWarning, match="through Python"):
            build.build()
    assert build.LIB_PATH.read_text() == "nvcc" and build.FAST_PATH.exists() == (gxx == "works")
    assert tools.ran == ["nvcc", "g++"]


def test_calls_without_the_module_take_the_python_way(monkeypatch, tmp_path):
    monkeypatch.setattr(_eager, "__file__", str(tmp_path / "_eager.py"))
    monkeypatch.setattr(_eager, "fast", _eager._Unbound())
    with pytest.warns(RuntimeWarning, match="is missing"):
        assert _eager.fast.rotary(1, 2, 3) is None
    assert _eager.fast.tree_mask() is None and _eager.fast.set_workspace(None) is None


def test_a_module_built_for_another_torch_is_not_loaded(monkeypatch, tmp_path):
    monkeypatch.setattr(torch, "__version__", torch.__version__ + ".other")
    other = build.fast_name()
    monkeypatch.undo()
    assert other != build.fast_name() and build.FAST_PATH.name == build.fast_name()
    tools = Tools(monkeypatch, tmp_path, "works")
    build.build()
    build.FAST_PATH.rename(build.FAST_PATH.with_name(other))  # left from before: is built anew, newer source or not
    build.build()
    assert tools.ran == ["nvcc", "g++", "g++"] and build.FAST_PATH.exists()
    build.FAST_PATH.unlink()
    monkeypatch.setattr(_eager, "__file__", str(tmp_path / "_eager.py"))
    monkeypatch.setattr(_eager, "fast", _eager._Unbound())
    with pytest.warns(RuntimeWarning, match="is missing"):
        assert _eager.fast.kv_load() is None


# ---------------------------------------------------------------- refusals --
def test_token_counts_that_the_product_with_the_heads_would_wrap():
    for n in (1 << 31, 1 << 58, (1 << 63) - 1):
        assert store(N=n) == 1 and "num_tokens" in _lib.last_error()
