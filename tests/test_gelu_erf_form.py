"""CPU: the erf GELU of the linear and group norm epilogues.

gelu_erf (seedvr2_ncnn_b200/csrc/activation.cuh) is max(x, 0) - a q with a = |x| and
q = erfc(a / sqrt 2) / 2 = r P(6 r - 1) exp(-a^2 / 2), r = 1 / (a + 3).  This replays its float32 steps in numpy
(coefficients read from the kernel source, so the two cannot drift apart), with the reciprocal one ulp and the
exponential two ulp off in either direction, as the device's may be, and holds q to the stated
(20 + 2 x^2) 2^-24 of itself."""
import os
import re

import numpy as np
import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SRC = os.path.join(ROOT, "seedvr2_ncnn_b200", "csrc", "activation.cuh")
f32 = np.float32


def _coefficients():
    m = re.search(r"constexpr float c\[9\] = \{([^}]*)\};", open(SRC).read())
    assert m, "coefficients not found in the kernel source"
    c = [f32(float(v.strip().rstrip("f"))) for v in m.group(1).split(",")]
    assert len(c) == 9
    return c


def _fma(x, y, z):  # rounded once
    return (x.astype(np.float64) * np.float64(y) + np.float64(z)).astype(f32)


def q_of(a, rcp=0.0, ex2=0.0):
    c = _coefficients()
    a = a.astype(f32)
    r = ((1 + rcp) / (a + f32(3)).astype(np.float64)).astype(f32)
    s = _fma(r, 6.0, -1.0)
    p = np.full_like(s, c[8])
    for ci in c[7::-1]:
        p = (p.astype(np.float64) * s.astype(np.float64) + np.float64(ci)).astype(f32)
    z = (a * f32(-0.5 * 1.4426950408889634)) * a
    e = (np.exp2(z.astype(np.float64)) * (1 + ex2)).astype(f32)
    return (p * r) * e


@pytest.mark.parametrize("rcp", [-2.0**-23, 0.0, 2.0**-23])
@pytest.mark.parametrize("ex2", [-2.0**-22, 0.0, 2.0**-22])
def test_q_keeps_its_digits(rcp, ex2):
    a = np.concatenate([np.linspace(0, 13, 400_001), np.logspace(-30, 0, 2001)]).astype(f32)
    want = torch.special.erfc(torch.from_numpy(a.astype(np.float64)) / np.sqrt(2)).numpy() / 2
    over = np.abs(q_of(a, rcp, ex2) / want - 1) / ((20 + 2 * a.astype(np.float64) ** 2) * 2.0**-24)
    assert over.max() < 1, (over.max(), a[over.argmax()])


def test_q_ends_at_zero():
    q = q_of(np.linspace(13, 30, 10_001))
    assert np.all(q >= 0) and np.all(q < 1e-36)
