"""How far gd_kv_attn_scored's caps are off: kv_attn.h's two ways to a capped score, with the coefficients
that stand there, formed operation by operation in 32 bits, the hardware's reciprocal and
exponential a step off either way, within what gadeon_hip.h states."""
import re
from pathlib import Path

import numpy as np
import pytest

ROOT = Path(__file__).resolve().parents[1]
CODE = (ROOT / "gadeon_amd/csrc/kv_attn.h").read_text()
F, D, L = np.float32, np.float64, np.longdouble
LOG2E = F(1.4426950408889634)


def stated(of):
    """The bound that the header gives, a power of 2."""
    text = re.sub(r"[\s*]+", " ", (ROOT / "include/gadeon_hip.h").read_text())
    (bound,) = re.findall(r"2\^-(\d+(?:\.\d+)?) of " + of, text)
    return 2.0 ** -float(bound)


def coefficients(name):
    """Of a polynomial in u, the highest power first."""
    (line,) = re.findall(r"const float %s = (fmaf.*?);" % name, CODE)
    return [F(c) for c in re.findall(r"(?<![\w.])\d+\.\d*(?:e-\d+)?", line)]


def fma(a, b, c):
    return (a.astype(D) * D(b) + D(c)).astype(F) if np.isscalar(b) else (a.astype(D) * b.astype(D) + D(c)).astype(F)


def off(x, steps):
    return np.nextafter(x, F(np.inf * steps)) if steps else x


END = float(re.search(r"TANH_END = ([\d.]+)f", CODE)[1])
X = np.concatenate([np.linspace(1e-3, END + 1, 250001), np.geomspace(1e-20, 40, 50001)]).astype(F)
X = np.concatenate([-X[::-1], X])
TANH = np.tanh(X.astype(L))


def test_coefficients():
    p, q = coefficients("p"), coefficients("q")
    assert len(p) == len(q) == 5 and min(p + q) > 0 and q[-1] == 1
    at = np.linspace(1e-3, END, 200001).astype(L)
    of = lambda c: sum(L(k) * at ** (2 * (4 - i)) for i, k in enumerate(c))  # noqa: E731
    (bound,) = re.findall(r"off by 2\^-([\d.]+) of itself in exact arithmetic", re.sub(r"[\s/]+", " ", CODE))
    assert np.abs(at * of(p) / of(q) / np.tanh(at) - 1).max() <= 2.0 ** -float(bound)


@pytest.mark.parametrize("cap", [1e-3, 5.0, 64.0, 1e4])
@pytest.mark.parametrize("step", [-1, 0, 1])
def test_by_a_quotient(cap, step):
    cap = F(cap) * LOG2E
    x = np.clip(X, F(-END), F(END))
    u, p, q = x * x, *(np.full_like(x, coefficients(c)[0]) for c in "pq")
    for a, b in zip(coefficients("p")[1:], coefficients("q")[1:]):
        p, q = fma(p, u, a), fma(q, u, b)
    y = (cap * x) * (p * off((1 / q.astype(D)).astype(F), step))
    assert np.abs(y / (L(cap) * TANH) - 1).max() <= stated("itself")


@pytest.mark.parametrize("cap", [1e-3, 5.0, 64.0, 1024.0])
@pytest.mark.parametrize("steps", [(i, j) for i in (-1, 0, 1) for j in (-1, 0, 1)], ids=str)
def test_by_an_exponential(cap, steps):
    cap = F(cap) * LOG2E
    with np.errstate(over="ignore"):
        e = off(np.exp2((X * (F(2) * LOG2E)).astype(D)).astype(F), steps[0])
        r = off((1 / (F(1) + e).astype(D)).astype(F), steps[1])
    y = fma(r, float(-2 * cap), cap)
    assert np.abs(y - L(cap) * TANH).max() <= stated("the cap") * L(cap)
