"""The polynomials of the paged attention's capped scores, by the coefficients that the source holds."""
import re

import numpy as np
import pytest

from conftest import PKG, ROOT

SOURCE = (ROOT / PKG / "csrc" / "paged_attend.h").read_text()


def coefficients(name):
    """As the compiler holds them, in the type that they are declared with."""
    kind, numbers = re.search(r"constexpr (float|double) " + name + r"\[\d\] = \{([^}]*)\}", SOURCE).groups()
    values = [float(x.strip().rstrip("f")) for x in numbers.split(",")]
    return [float(np.float32(x)) for x in values] if kind == "float" else values


def most(name):
    return float(re.search(name + r"Most = ([0-9.]+)f", SOURCE).group(1))


def off(c, d, value):
    return float(np.abs(np.polyval(c[::-1], d * d) * d / value - 1).max())


@pytest.mark.parametrize("name", ["kCapLeast", "kCapNear", "kCapFar"])
def test_fit(name):
    """tanh(t) within 3e-8 of its value, as the comment beside them says."""
    t = np.linspace(1e-4, most(name), 200001)
    assert off(coefficients(name), t, np.tanh(t)) <= 3e-8


@pytest.mark.parametrize("name", ["kCapLeast", "kCapNear", "kCapFar"])
@pytest.mark.parametrize("scale,cap", [(128 ** -0.5, 50.0), (128 ** -0.5, 30.0), (0.1, 1.0), (0.037, 7.3), (1.7, 1000.0), (0.3, 0.11)])
def test_scaled_coefficients(name, scale, cap):
    """cap log2(e) tanh(d scale / cap), its coefficients rounded to fp32 once: 3e-8 of the value, and half a step of each
    coefficient, whose terms' magnitudes add up to 1.5 of the value at most."""
    scale, cap = float(np.float32(scale)), float(np.float32(cap))
    by = [scale * np.log2(np.e) * (scale / cap) ** (2 * i) for i in range(6)]
    c = [float(np.float32(x * y)) for x, y in zip(coefficients(name), by)]
    d = np.linspace(1e-4, most(name), 20001) * cap / scale
    assert off(c, d, cap * np.log2(np.e) * np.tanh(d * scale / cap)) <= 3e-8 + 1.5 * 2.0 ** -24


def test_fp32_coefficients():
    """Those of any score, used in fp32."""
    t = np.linspace(1e-4, most("kCapFar"), 200001)
    assert off([float(np.float32(x)) for x in coefficients("kCapFar")], t, np.tanh(t)) <= 7e-8
