"""Accuracy of the products as documented, over whole results (GPU).

The element bounds of test_gpu_ops.py hold for any order and sign of the roundings; they grow with the
sum of the terms' magnitudes and are wide for long rows. Here the 2-norm of a result's error is compared
with what the roundings amount to, for activations of both signs and of one sign, whose level and
minimum terms nearly cancel.
"""

import numpy as np
import pytest
import torch

import ops_reference as ref
from kernels import ops

pytestmark = pytest.mark.gpu

K, N = 4096, 131


def halves(v):
    return v.astype(np.float16)[..., None].view(np.uint8)


def centred(qtype, n, k, rng):
    """Packed rows whose minima lie at the middle of the levels, so that weights of both signs come out."""
    b = ref.random_blocks(qtype, (n,), k, rng).reshape(n, k // ref.qk(qtype), -1)
    if qtype not in ref.LEVELS:
        return b.reshape(n, -1)
    d = (0.01 * (0.5 + rng.random(b.shape[:2]))).astype(np.float16).astype(np.float64)
    if qtype in ("q4_1", "q5_1"):
        b[..., :2], b[..., 2:4] = halves(d), halves(d * (-7.5 if qtype == "q4_1" else -15.5))
    elif qtype == "q2_k":
        s = rng.integers(4, 16, (*b.shape[:2], 16)).astype(np.uint8)
        b[..., :16] = s | (s << 4)
        b[..., 80:82], b[..., 82:84] = halves(d), halves(1.5 * d)
    else:
        s = rng.integers(16, 64, (*b.shape[:2], 8)).astype(np.uint8)
        lo, hi = s[..., :4], s[..., 4:]
        b[..., 4:8] = b[..., 8:12] = lo | ((hi >> 4) << 6)
        b[..., 12:16] = (hi & 15) | ((hi & 15) << 4)
        b[..., :2], b[..., 2:4] = halves(d), halves(d * (7.5 if qtype == "q4_k" else 15.5))
    return b.reshape(n, -1)


def activations(kind, rows, k, rng):
    """Q8_0 blocks of rows of values."""
    x = rng.standard_normal((rows, k))
    if kind == "relu2":
        x = np.maximum(x, 0) ** 2
    elif kind == "one sign":
        x = np.abs(x)
    elif kind == "mean 1":
        x = 1 + 0.1 * x
    b = x.reshape(rows, -1, 32)
    d = (np.abs(b).max(-1, keepdims=True) / 127).astype(np.float16)
    q = np.rint(b / d.astype(np.float64)).clip(-127, 127).astype(np.int8)
    return np.concatenate([d.view(np.uint8), q.view(np.uint8)], -1).reshape(rows, -1)


def rounded_activations(xq):
    """The activations at 11 bits: float16 after a power of two per row that takes its largest scale to 2^7 .. 2^8."""
    x, d = ref.decode64(xq, "q8_0"), ref.split_q8(xq)[0].astype(np.float64)
    up = 2.0 ** (8 - np.frexp(np.abs(d).max(1, keepdims=True))[1])
    return (x * up).astype(np.float16).astype(np.float64) / up


def rounded_weights(wq, qtype):
    """Q6_K: level times sub-scale at 11 bits; the other formats' are exact there."""
    w = ref.decode64(wq, qtype)
    if qtype != "q6_k":
        return w
    b = wq.reshape(wq.shape[0], -1, 210)
    one = b.copy()
    one[..., 208:] = halves(np.ones(b.shape[:2]))
    ints = ref.decode64(one.reshape(wq.shape), qtype).astype(np.float16).astype(np.float64)
    d = b[..., 208:].copy().view(np.float16).astype(np.float64)
    return (ints.reshape(*b.shape[:2], 256) * d).reshape(wq.shape[0], -1)


def terms(x, wq, qtype):
    """sum |x| (|dl l| + |ml|) of every result."""
    mag = np.abs(ref.decode64(wq, qtype))
    if qtype in ref.LEVELS:
        _, bb = ref.GGML_QUANT_SIZES[ref.GTYPE[qtype]]
        z = wq.reshape(wq.shape[0], -1, bb).copy()
        z[..., slice(*ref.LEVELS[qtype])] = 0
        mag = mag + 2 * np.abs(ref.decode64(z.reshape(wq.shape), qtype))
    return np.abs(x) @ mag.T


def bf16(y):
    return torch.from_numpy(y).to(torch.bfloat16).double().numpy()


def matmul(wq, qtype, xq, dtype):
    got = ops.matmul(torch.from_numpy(wq).cuda(), int(ref.GTYPE[qtype]), torch.from_numpy(xq).cuda(), out_dtype=dtype)
    return got.double().cpu().numpy()


KINDS = ["normal", "relu2", "one sign", "mean 1"]


@pytest.mark.parametrize("qtype", ref.TYPES)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows", [100, 130])
def test_bfloat16_results_of_many_rows(qtype, kind, rows):
    """The result's own rounding and that of the activations to 11 bits (Q6_K: of weight factors too), no other.

    Element by element, against the products of the rounded operands in 64 bits: half a step of the result,
    and the sums' error. That is at most 2^-18 of the terms: 256 values are summed in 16 steps of 16,
    each truncated (2^-23 of the sum: 2^-19 in all), then 16 superblocks and their minima in float32.

    In the 2-norm, against the exact products: an activation's rounding lies evenly within 2^-11 of it, so the
    products' is 2^-11 / sqrt(3) = 2.8e-4 of the result at most where the weights' signs are random; a bfloat16's is
    1.66e-3. Together sqrt(1.66^2 + 0.28^2) / 1.66 = 1.014 of the latter; 1.03 leaves the inner part 4.1e-4.
    """
    rng = np.random.default_rng(rows)
    wq, xq = centred(qtype, N, K, rng), activations(kind, rows, K, rng)
    got = matmul(wq, qtype, xq, torch.bfloat16)
    x = ref.decode64(xq, "q8_0")
    y, yr = x @ ref.decode64(wq, qtype).T, rounded_activations(xq) @ rounded_weights(wq, qtype).T
    half_step = 2.0 ** (np.frexp(np.abs(yr))[1] - 9)  # of 8 bits
    slack = 2.0 ** -18 * terms(x, wq, qtype)
    over = np.abs(got - yr) / (half_step + slack)
    assert over.max() <= 1, f"worst {over.max():.3g}"
    assert np.linalg.norm(got - y) <= 1.03 * np.linalg.norm(bf16(y) - y), \
        f"{np.linalg.norm(got - y) / np.linalg.norm(y):.3g}, the rounding alone {np.linalg.norm(bf16(y) - y) / np.linalg.norm(y):.3g}"


@pytest.mark.parametrize("qtype", ref.TYPES)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows", [1, 3, 9, 60, 100])
def test_float32_results(qtype, kind, rows):
    """At most 2^-20 of the result for activations of both signs, of the terms for others.

    Four float32 roundings (2^-24 of the running sum, at most) for each of the 128 units of a row, of random
    sign: sqrt(512) 2^-24 / sqrt(3) = 2^-20.3 of a sum that reaches its final size at once, about 2/3 of that for
    one that grows with the root of its length. By tcgen05 the sums of 128 values are truncated: 2^-23 in each of
    8 steps, one half on average, is 2^-21 of a sum that starts at its final size, half of it for one that grows.
    """
    rng = np.random.default_rng(rows)
    wq, xq = centred(qtype, N, K, rng), activations(kind, rows, K, rng)
    got = matmul(wq, qtype, xq, torch.float32)
    x = ref.decode64(xq, "q8_0")
    y = x @ ref.decode64(wq, qtype).T
    size = y if kind == "normal" else terms(x, wq, qtype)
    err = np.linalg.norm(got - y) / np.linalg.norm(size)
    assert err <= 2.0 ** -20, f"{err:.3g}"


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("ratio", [10, 16, 22])
@pytest.mark.parametrize("rows", [9, 100, 130])
def test_one_large_block_that_no_weight_meets(dtype, ratio, rows):
    """Values 2^-ratio of their row's largest, which alone make the result: held to 2^-39 of 128 times the row's
    largest scale (a level of 1 lies at 2^-7 of its block's largest)."""
    rng = np.random.default_rng(ratio)
    wq, xq = centred("q8_0", N, 1024, rng), activations("normal", rows, 1024, rng)
    x = xq.reshape(rows, -1, 34)
    x[:, 5, :2], d = halves(np.full(rows, 16.0)), x[..., :2].copy().view(np.float16)[..., 0]
    d = d.astype(np.float64) / d.astype(np.float64).max() * 16 * 2.0 ** -ratio
    keep = np.arange(32) != 5
    x[:, keep, :2] = halves(d[:, keep])
    wq.reshape(N, -1, 34)[:, 5, :2] = 0
    got = matmul(wq, "q8_0", xq, getattr(torch, dtype))
    y, bound = ref.product(xq, wq, "q8_0", dtype)
    bound = bound + 2.0 ** -39 * 128 * 16 * np.abs(ref.decode64(wq, "q8_0")).sum(1)
    assert (np.abs(got - y) <= bound + ref.rounding(np.abs(y) + bound, dtype)).all()


@pytest.mark.parametrize("qtype", ref.TYPES)
@pytest.mark.parametrize("rows", [1, 9, 100])
def test_float16_results(qtype, rows):
    """float16's own rounding: its half steps lie 8 times closer than bfloat16's, 2.1e-4 in the 2-norm. 2^-20 of
    float32 sums (test_float32_results) beside it are sqrt(2.1e-4^2 + 9.5e-7^2), 1.00001 of it."""
    rng = np.random.default_rng(rows)
    wq, xq = centred(qtype, N, K, rng), activations("normal", rows, K, rng)
    y = ref.decode64(xq, "q8_0") @ ref.decode64(wq, qtype).T
    got = matmul(wq, qtype, xq, torch.float16)
    # values below 2^-14 round to steps of 2^-24
    alone = np.linalg.norm(y.astype(np.float16).astype(np.float64) - y)
    assert np.linalg.norm(got - y) <= 1.01 * alone


@pytest.mark.parametrize("qtype", ["q4_k", "q2_k", "q5_1", "q6_k", "q4_0"])
@pytest.mark.parametrize("kind", ["normal", "one sign"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("tokens", [2, 60, 400])
def test_experts(qtype, kind, dtype, tokens):
    """The same for the products of experts, for all three kernels (averages of 1, 30 and 200 slots)."""
    rng = np.random.default_rng(tokens)
    e, n, k = 4, 67, 2048
    wq = np.stack([centred(qtype, n, k, rng) for _ in range(e)])
    xq = activations(kind, tokens, k, rng)
    ids = rng.integers(0, e, (tokens, 2)).astype(np.int32)
    plan = ops.expert_plan(torch.from_numpy(ids).cuda(), e)
    got = ops.matmul_experts(torch.from_numpy(wq).cuda(), int(ref.GTYPE[qtype]), torch.from_numpy(xq).cuda(), plan,
                             out_dtype=getattr(torch, dtype)).double().cpu().numpy()
    x = ref.decode64(xq, "q8_0")
    y, size = np.zeros(got.shape), np.zeros(got.shape)
    for i in range(e):
        t, j = np.nonzero(ids == i)
        y[t, j] = x[t] @ ref.decode64(wq[i], qtype).T
        size[t, j] = np.abs(y[t, j]) if kind == "normal" else terms(x[t], wq[i], qtype)
    err = np.linalg.norm(got - y)
    if dtype == "float32":
        assert err <= 2.0 ** -20 * np.linalg.norm(size)
    else:
        assert err <= 1.03 * np.linalg.norm(bf16(y) - y)
