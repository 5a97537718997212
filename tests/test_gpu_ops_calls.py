"""Calls of the operators on packed blocks at the edges of what they allow, on the GPU."""

from fractions import Fraction
from math import floor

import numpy as np
import pytest
import torch

import ops_reference as ref
from kernels import ops
from test_gpu_ops import check_product, cuda, experts_want

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("qtype", ref.TYPES)
@pytest.mark.parametrize("tokens", [2, 40, 300])
@pytest.mark.parametrize("padded", [False, True])
def test_experts_of_one_row(qtype, tokens, padded):
    """One weight row per expert, of any number of bytes, next to each other or apart."""
    rng = np.random.default_rng(tokens)
    e, k = 3, ref.qk(qtype)
    w = ref.random_blocks(qtype, (e, 1), k, rng)
    x = ref.random_blocks("q8_0", (tokens,), k, rng)
    ids = rng.integers(-1, e, (tokens, 2)).astype(np.int32)
    wc = cuda(w)
    if padded:
        wide = torch.full((e, 2, w.shape[2] + 16), 255, dtype=torch.uint8, device="cuda")
        wide[:, :1, :w.shape[2]] = wc
        wc = wide[:, :1, :w.shape[2]]
    if wc.stride(0) % {"q4_k": 16, "q5_k": 16, "q5_1": 8, "iq4_xs": 8, "q4_1": 4, "q2_k": 4}.get(qtype, 2):
        pytest.skip("this stride is refused for this format")
    got = ops.matmul_experts(wc, int(ref.GTYPE[qtype]), cuda(x), ops.expert_plan(cuda(ids), e))
    check_product(got, *experts_want(x, w, qtype, ids, None, False))


def near_border(rng, count):
    """(t, w, level): rows of 32 float32 values and weights whose second value lies within 2^-47 of the border
    between two levels, on a known side: h t0 w0 - 254 t w is a small integer (levels are 127 t w / (t0 w0))."""
    out = []
    while len(out) < count:
        h = 2 * int(rng.integers(64, 127)) + 1  # 127 x / m next to h / 2
        t0, t = int(rng.integers(1 << 23, 1 << 24)) | 1, int(rng.integers(1 << 23, 1 << 24)) | 1
        # w / w0 next to h t0 / (254 t): convergents of the continued fraction
        a, b = h * t0, 254 * t
        p0, q0, p1, q1 = 0, 1, 1, 0
        while b:
            c, (a, b) = a // b, (b, a % b)
            p0, q0, p1, q1 = p1, q1, c * p1 + p0, c * q1 + q0
            if max(p1, q1) >= 1 << 24:
                break
            if q1 < 1 << 20 or p1 >= q1 * 2:
                continue
            w, w0 = p1, q1
            over = 254 * t * w - h * t0 * w0
            if t * w >= t0 * w0 or abs(Fraction(over, 2 * t0 * w0)) > Fraction(1, 1 << 47):
                continue
            out.append((t0, w0, t, w, floor(Fraction(127 * t * w, t0 * w0) + Fraction(1, 2))))
    return out


@pytest.mark.parametrize("scale", [2.0 ** -130, 2.0 ** -60, 2.0 ** 80])
def test_norm_next_to_borders(scale):
    """Levels as in exact arithmetic: products within 2^-47 of a border, small, ordinary and large."""
    cases = near_border(np.random.default_rng(3), 64)
    for t0, w0, t, w, level in cases:
        x, wt = np.zeros((1, 32)), np.ones(32)
        x[0, 0], wt[0], x[0, 1], wt[1] = t0, w0, t, -w
        x, wt = (x * scale).astype(np.float32), wt.astype(np.float32)
        _, q = ref.split_q8(ops.rms_norm_q8(cuda(x), cuda(wt), 1e-6).cpu().numpy())
        assert q[0, 0, 0] == 127 and q[0, 0, 1] == -level, (t0, w0, t, w)
