"""Rotary frequencies and their scaling for long contexts, on the host."""

import math

import pytest
import torch

from logkv_amd import rotary_frequencies, rotary_tables


def test_plain_and_linear():
    f, a = rotary_frequencies(8, 10000.0, device="cpu")
    assert f.dtype == torch.float64 and a == 1.0
    assert torch.allclose(f, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-15)
    g, _ = rotary_frequencies(8, 10000.0, scaling=dict(kind="linear", factor=4), device="cpu")
    assert torch.equal(g, f / 4)


def test_wavelength():
    n, factor, low, high = 8192.0, 8.0, 1.0, 4.0
    f, _ = rotary_frequencies(128, 500000.0, device="cpu")
    g, a = rotary_frequencies(128, 500000.0, device="cpu", scaling=dict(
        kind="wavelength", factor=factor, original_max_seq_len=n, low_freq_factor=low, high_freq_factor=high))
    assert a == 1.0
    seen = set()
    for x, y in zip(f.tolist(), g.tolist()):
        wave = 2 * math.pi / x
        if wave < n / high:
            want, at = x, "kept"
        elif wave > n / low:
            want, at = x / factor, "divided"
        else:
            s = (n / wave - low) / (high - low)
            want, at = (1 - s) * x / factor + s * x, "between"
        seen.add(at)
        assert math.isclose(y, want, rel_tol=1e-12)
    assert seen == {"kept", "between", "divided"}


def test_yarn():
    dim, base, n, factor = 64, 10000.0, 4096, 16.0
    f, _ = rotary_frequencies(dim, base, device="cpu")
    g, a = rotary_frequencies(dim, base, device="cpu", scaling=dict(kind="yarn", factor=factor, original_max_seq_len=n))
    assert math.isclose(a, 0.1 * math.log(factor) + 1)
    turns = [n * x / (2 * math.pi) for x in f.tolist()]
    lo = math.floor(dim * math.log(n / (32 * 2 * math.pi)) / (2 * math.log(base)))
    hi = math.ceil(dim * math.log(n / (1 * 2 * math.pi)) / (2 * math.log(base)))
    for i, (x, y, t) in enumerate(zip(f.tolist(), g.tolist(), turns)):
        if i <= lo:
            assert y == x and t > 30
        elif i >= hi:
            assert math.isclose(y, x / factor, rel_tol=1e-12) and t < 1.3
        else:
            s = (i - lo) / (hi - lo)
            assert math.isclose(y, x * (1 - s) + x / factor * s, rel_tol=1e-12)
    assert rotary_frequencies(dim, base, device="cpu", scaling=dict(
        kind="yarn", factor=0.5, original_max_seq_len=n))[1] == 1.0
    assert rotary_frequencies(dim, base, device="cpu", scaling=dict(
        kind="yarn", factor=2.0, original_max_seq_len=n, attention_factor=1.5))[1] == 1.5


def test_tables():
    f, _ = rotary_frequencies(16, device="cpu")
    cos, sin = rotary_tables(f, 50, amplitude=2.0, dtype=torch.bfloat16)
    for p in (0, 1, 49):
        for i in range(16):
            assert cos[p, i] == torch.tensor(2.0 * math.cos(p * float(f[i % 8]))).to(torch.bfloat16)
            assert sin[p, i] == torch.tensor(2.0 * math.sin(p * float(f[i % 8]))).to(torch.bfloat16)


@pytest.mark.parametrize("args,scaling", [
    ((7,), None), ((0,), None), ((514,), None), ((8, 1.0), None), ((8, float("inf")), None),
    ((8,), {}), ((8,), dict(kind="linear")), ((8,), dict(kind="linear", factor=0)), ((8,), dict(kind="other", factor=2)),
    ((8,), dict(kind="linear", factor=2, beta_fast=3)), ((8,), dict(kind="wavelength", factor=2, low_freq_factor=1)),
    ((8,), dict(kind="wavelength", factor=2, low_freq_factor=4, high_freq_factor=1, original_max_seq_len=10)),
    ((8,), dict(kind="yarn", factor=2)), ((8,), dict(kind="yarn", factor=2, original_max_seq_len=0)),
    ((8,), dict(kind="yarn", factor=2, original_max_seq_len=10, beta_fast=1, beta_slow=2)),
    ((8,), dict(kind="yarn", factor=2, original_max_seq_len=10, attention_factor=float("nan")))])
def test_refusals(args, scaling):
    with pytest.raises(ValueError):
        rotary_frequencies(*args, scaling=scaling, device="cpu")
