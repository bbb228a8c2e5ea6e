"""Frequencies of the rotary positions against their formulas, and what the C entry refuses (no GPU)."""
import ctypes
import math

import pytest
import torch

import alto_amd.mxfp4 as m


def test_plain_linear_and_ntk():
    f, factor = m.rotary_frequencies(64)
    assert f.dtype == torch.float64 and f.shape == (32,) and factor == 1.0
    for i in range(32):
        assert abs(float(f[i]) - 10000.0 ** (-2 * i / 64)) < 1e-15
    g, factor = m.rotary_frequencies(64, scaling=dict(type="linear", factor=4))
    assert torch.equal(g, f / 4) and factor == 1.0
    g, factor = m.rotary_frequencies(64, scaling=dict(type="ntk", factor=8))
    assert float(g[0]) == 1.0 and abs(float(g[31] / f[31]) - 1 / 8) < 1e-13 and factor == 1.0
    assert bool((g <= f).all())


@pytest.mark.parametrize("kind", ["yarn", "wavelength"])
def test_blended_frequencies(kind):
    length, by = 4096, 16.0
    f, _ = m.rotary_frequencies(128, base=500000.0)
    g, factor = m.rotary_frequencies(128, base=500000.0, scaling=dict(type=kind, factor=by, original_length=length))
    low, high = (1.0, 32.0) if kind == "yarn" else (1.0, 4.0)
    assert abs(factor - (0.1 * math.log(by) + 1 if kind == "yarn" else 1.0)) < 1e-15
    seen = set()
    for x, y in zip(f.tolist(), g.tolist()):
        turns = length * x / (2 * math.pi)
        share = min(1.0, max(0.0, (turns - low) / (high - low)))
        assert abs(y - ((1 - share) * x / by + share * x)) < 1e-15
        seen.add(0 if share == 0 else 2 if share == 1 else 1)
    assert seen == {0, 1, 2}


def test_refused_frequencies():
    for bad in (dict(rotary_dim=0), dict(rotary_dim=7), dict(rotary_dim=8, base=0.0), dict(rotary_dim=2, scaling=dict(type="ntk", factor=2)),
                dict(rotary_dim=8, scaling=dict(type="linear", factor=0)), dict(rotary_dim=8, scaling=dict(type="cubic")),
                dict(rotary_dim=8, scaling=dict(type="yarn", factor=2, original_length=64, beta_fast=1, beta_slow=1))):
        with pytest.raises(ValueError):
            m.rotary_frequencies(**bad)


def test_a_cpu_tensor_is_refused():
    with pytest.raises(RuntimeError):
        m.apply_rotary(torch.zeros(1, 1, 2, 4), None, m.rotary_frequencies(4)[0])


def test_the_c_entry_checks_its_arguments():
    from alto_amd import _lib
    from alto_amd.mxfp4.rotary import _Args
    lib = _lib.load()
    assert lib.alto_mxfp4_rotary(None, None) == -1
    good = dict(q=4096, q_out=8192, inv_freq=4096, B=1, S=1, Hq=1, Hk=0, D=8, R=8, dtype=0)
    for name, value in (("q", 0), ("q_out", 0), ("inv_freq", 0), ("inv_freq", 4100), ("q", 4097), ("Hq", 0), ("Hk", -1), ("Hk", 1), ("R", 7), ("R", 0), ("R", 10), ("D", 0),
                        ("B", -1), ("S", 2 ** 31), ("dtype", 2), ("q_sb", -1), ("qo_ss", 2 ** 41), ("pos_ss", -8), ("positions", 4)):
        a = _Args(**{**good, name: value})
        assert lib.alto_mxfp4_rotary(ctypes.byref(a), None) == -1 and lib.alto_mxfp4_last_error(), (name, value)
    empty = _Args(**{**good, "S": 0})
    assert lib.alto_mxfp4_rotary(ctypes.byref(empty), None) == 0
