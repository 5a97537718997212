"""Calls of the operators on packed blocks at the edges of what they allow, on the GPU."""

import subprocess
import sys
from fractions import Fraction
from math import floor
from pathlib import Path

import numpy as np
import pytest
import torch

import ops_reference as ref
from kernels import _native, ops
from test_gpu_ops import check_norm, check_product, check_route, cuda, experts_want

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
    p = ops.expert_plan(cuda(ids), e)
    if wc.stride(0) % {"q4_k": 16, "q5_k": 16, "q5_1": 8, "iq4_xs": 8, "q4_1": 4, "q2_k": 4}.get(qtype, 2):
        with pytest.raises(_native.QsError):
            ops.matmul_experts(wc, int(ref.GTYPE[qtype]), cuda(x), p)
        return
    got = ops.matmul_experts(wc, int(ref.GTYPE[qtype]), cuda(x), p)
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


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("scale", [3e35, 2e36, 1e37])
def test_norm_of_rows_whose_factor_is_subnormal(dtype, scale):
    """1 / (127 rms) below float32's normal range, with products inside it."""
    g = torch.Generator(device="cuda").manual_seed(5)
    x = (torch.randn((64, 1024), device="cuda", generator=g) * scale).to(getattr(torch, dtype))
    w = 0.01 + 0.1 * torch.rand(1024, device="cuda", generator=g)
    assert torch.isfinite(x).all()
    check_norm(x, w, 1e-6, None, ops.rms_norm_q8(x, w, 1e-6))


@pytest.mark.parametrize("k", [32, 512, 8224, 20480])
@pytest.mark.parametrize("off,gap", [(0, 0), (1, 0), (2, 6), (16, 48), (3, 5)])
def test_norm_into_any_address(k, off, gap):
    """Blocks at any address and row distance; bytes before, between and behind the rows stay."""
    n, row = 5, k // 32 * 34
    g = torch.Generator(device="cuda").manual_seed(k)
    x, w = torch.randn((n, k), device="cuda", generator=g), torch.rand(k, device="cuda", generator=g) + 0.5
    want = ops.rms_norm_q8(x, w)
    buf = torch.full((off + n * (row + gap) + 64,), 171, dtype=torch.uint8, device="cuda")
    _native.check(_native.lib().qs_rms_norm_q8(x.data_ptr(), 0, k, None, 0, None, 0, w.data_ptr(), 1e-6, n, k, buf.data_ptr() + off, row + gap,
                                               torch.cuda.current_stream().cuda_stream))
    rows = buf[off:off + n * (row + gap)].reshape(n, row + gap)
    assert torch.equal(rows[:, :row], want)
    assert (rows[:, row:] == 171).all() and (buf[:off] == 171).all() and (buf[off + n * (row + gap):] == 171).all()


CAPTURED = """
import sys
sys.path[:0] = [sys.argv[1], sys.argv[2]]
import torch
import test_gpu_ops as t
from kernels import _native, ops
_native.check(_native.lib().qs_init(0))
a = t.layer_inputs(int(sys.argv[3]), 1) if sys.argv[4] == "layer" else None
g = torch.cuda.CUDAGraph()
if a is not None:
    with torch.cuda.graph(g):
        got = t.layer(*a)
    want = lambda: t.layer(*a)
else:
    rows = int(sys.argv[3])
    gen = torch.Generator(device="cuda").manual_seed(5)
    def blocks(n, nb):
        b = torch.randint(0, 256, (n, 4, nb), device="cuda", generator=gen, dtype=torch.uint8)
        b[..., 1] = 0x1C
        b[..., -1] = 0x1C
        return b.reshape(n, 4 * nb)
    w, x = blocks(300, 66), torch.randint(0, 256, (rows, 32, 34), device="cuda", generator=gen, dtype=torch.uint8)
    x[..., 1] = 0x1C
    x = x.reshape(rows, -1)
    with torch.cuda.graph(g):
        got = ops.matmul(w, 16, x, out_dtype=torch.bfloat16),
    want = lambda: (ops.matmul(w, 16, x, out_dtype=torch.bfloat16),)
g.replay()
torch.cuda.synchronize()
got = [v.clone() for v in got]
assert all(torch.equal(p, q) and torch.isfinite(p.float()).all() for p, q in zip(got, want()))
"""


@pytest.mark.parametrize("rows,what", [(1, "layer"), (40, "layer"), (3, "matmul"), (20, "matmul"), (100, "matmul"), (300, "matmul")])
def test_first_call_of_a_kernel_is_captured(rows, what):
    """qs_init is all that a capture needs: no kernel of the calls has run in the process."""
    here = Path(__file__).resolve().parent
    r = subprocess.run([sys.executable, "-c", CAPTURED, str(here), str(here.parent / "quant-studio_b200"), str(rows), what], capture_output=True,
                       text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


@pytest.mark.parametrize("sign", [1, -1])
def test_route_biases_whose_sums_leave_float32(sign):
    """Sums of two biases beyond float32's range still order the groups."""
    rng = np.random.default_rng(9)
    z = rng.standard_normal((40, 8)).astype(np.float32)
    bias = np.array([2.0e38, 2.1e38, 3.0e38, 3.3e38, 1.8e38, 1.9e38, 2.5e38, 2.6e38], np.float32) * sign
    for score in ("softmax", "sigmoid"):
        for kept in (1, 2):
            check_route(cuda(z), top_k=2, score=score, bias=bias, n_groups=4, groups_kept=kept, group_score="top2")
            check_route(cuda(z), top_k=2, score=score, bias=bias, n_groups=4, groups_kept=kept)


def sampled(got, xq, wq, qtype, rows, cols, out="float32"):
    """Check of some rows and columns of a large product (blocks on the GPU)."""
    r, c = torch.tensor(rows, device="cuda"), torch.tensor(cols, device="cuda")
    check_product(got[r][:, c], *ref.product(xq[r].cpu().numpy(), wq[c].cpu().numpy(), qtype, out))


def q8_rows(n, k, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    b = torch.randint(0, 256, (n, k // 32, 34), device="cuda", generator=g, dtype=torch.uint8)
    b[..., 1] = 0x1C  # scales of 2^-8 .. 2^-7
    return b.reshape(n, -1)


def test_results_beyond_32_bits():
    """More than 2^31 results."""
    rows, n, k = 140_000, 16_400, 256
    x, w = q8_rows(rows, k, 1), q8_rows(n, k, 2)
    got = ops.matmul(w, 8, x, out_dtype=torch.bfloat16)
    assert got.numel() > 1 << 31
    sampled(got, x, w, "q8_0", [0, 1, 65_535, 130_943, 130_944, 139_998, 139_999], [0, 127, 128, 8191, 16_383, 16_384, 16_399], "bfloat16")


@pytest.mark.parametrize("rows", [1, 4, 40, 100])
def test_weights_beyond_32_bits(rows):
    """More than 2^32 bytes of weights."""
    n, k = 500_001, 8192
    x, w = q8_rows(rows, k, 3), q8_rows(n, k, 4)
    assert w.numel() > 1 << 32
    sampled(ops.matmul(w, 8, x), x, w, "q8_0", [0, rows - 1], [0, 1, 246_723, 246_724, 493_447, 493_448, 499_999, 500_000])


def test_norm_and_route_beyond_32_bits():
    n, k = 270_000, 8192
    x = torch.randn((n, 64), device="cuda", dtype=torch.bfloat16).repeat(1, k // 64)
    w = torch.rand(k, device="cuda") + 0.5
    got = ops.rms_norm_q8(x, w)
    at = torch.tensor([0, 1, 131_071, 262_143, 262_144, 262_145, n - 1], device="cuda")
    assert torch.equal(got[at], ops.rms_norm_q8(x[at], w))
    z = x.reshape(n * 64, 128)
    at = torch.tensor([0, 1, (1 << 24) - 1, 1 << 24, (1 << 24) + 1, n * 64 - 1], device="cuda")
    ids, ws = ops.route(z, 8)
    one, wone = ops.route(z[at], 8)
    assert torch.equal(ids[at], one) and torch.equal(ws[at], wone)


@pytest.mark.parametrize("qtype", ["q4_k", "q8_0", "q2_k"])
@pytest.mark.parametrize("rows", [1, 3, 40, 100])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_very_long_rows(qtype, rows, dtype):
    rng = np.random.default_rng(rows)
    n, k = 131, 131_072
    w, x = ref.random_blocks(qtype, (n,), k, rng), ref.random_blocks("q8_0", (rows,), k, rng)
    got = ops.matmul(cuda(w), int(ref.GTYPE[qtype]), cuda(x), out_dtype=getattr(torch, dtype))
    check_product(got, *ref.product(x, w, qtype, dtype))
