"""Edges of the verification operators' host-side parts (no GPU)."""

import math

import pytest
import torch

import torch_spyre_b200 as tsb


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
