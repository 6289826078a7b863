"""The polynomial behind the fused layer's GELU (fast_gelu.cuh) against the complementary error function, evaluated in float32 as the kernel
does: both errors that its comment claims."""
import math
import os
import re

import numpy as np

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "orion_b200", "csrc", "kernels", "fast_gelu.cuh")


def test_tail_of_the_normal_distribution():
    text = open(HEADER).read()
    body = text[text.index("uint64_t gauss_tail_pair("):]
    c = [np.float32(v) for v in re.findall(r"-?\d\.\d+(?:e-\d+)?(?=f)", body[body.index("{", body.index("constexpr float c[")):body.index(";")])]
    clamp = float(re.search(r"fmaxf\(-fabsf\(a0\), -(\d+\.\d+)f\)", text).group(1))
    x = np.linspace(0, 12, 60001).astype(np.float32)
    nx = -np.minimum(x, np.float32(clamp))
    p = np.full(x.shape, c[-1])
    for k in c[-2::-1]:   # a fused multiply-add: one rounding
        p = np.float32(p.astype(np.float64) * nx + np.float64(k))
    e = np.exp(-0.5 * x.astype(np.float64) ** 2)
    got = p.astype(np.float64) * e
    want = np.array([0.5 * math.erfc(v / math.sqrt(2)) for v in x.astype(np.float64)])
    assert np.abs(got - want).max() <= 1.1e-7
    inside = x <= clamp
    assert (np.abs(got - want) / want)[inside].max() <= 1.6e-3
    # a * Phi(a) at a = -x, whose factor is clamped as well
    gelu, exact = nx * got, -x.astype(np.float64) * want
    assert (np.abs(gelu - exact)[1:] / -exact[1:]).max() <= 0.025
