"""Operators on packed blocks on the GPU against their 64-bit definitions."""

import numpy as np
import pytest
import torch

import ops_reference as ref
from kernels import _native, ops

pytestmark = pytest.mark.gpu

DT = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


def cuda(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


# --- norm -----------------------------------------------------------------------------------

def check_norm(x, w, eps, residual=None, blocks=None, total=None):
    t = x.float() if residual is None else (x.float() + residual.float()).to(x.dtype)
    if residual is not None:
        assert torch.equal(t.view(torch.uint8), total.contiguous().view(torch.uint8))
    d, q = ref.norm_q8(t.float().cpu().numpy(), w.cpu().numpy(), eps)
    gd, gq = ref.split_q8(blocks.cpu().numpy())
    assert np.array_equal(gd.view(np.uint16), d.view(np.uint16))
    assert np.array_equal(gq, q)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("n,k", [(1, 32), (1, 4096), (3, 96), (5, 8192), (2, 8224), (700, 544), (601, 2048), (2, 16384), (3, 20000 // 32 * 32), (1, 40960)])
@pytest.mark.parametrize("with_residual", [False, True])
def test_norm(dtype, n, k, with_residual):
    g = torch.Generator(device="cuda").manual_seed(n * k)
    x = (torch.randn((n, k), device="cuda", generator=g) * 3).to(DT[dtype])
    r = torch.randn((n, k), device="cuda", generator=g).to(DT[dtype]) if with_residual else None
    w = 1 + 0.3 * torch.randn(k, device="cuda", generator=g)
    got = ops.rms_norm_q8(x, w, 1e-5, residual=r)
    check_norm(x, w, 1e-5, r, *(got if with_residual else (got,)))


@pytest.mark.parametrize("scale", [1e-30, 1e-18, 1e-6, 1e15, 1e30])
def test_norm_magnitudes(scale):
    """Squares that leave float32's range, and weights of one (levels on exact borders)."""
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn((4, 256), device="cuda", generator=g) * scale
    x[1] = x[1].to(torch.bfloat16).float()
    x[2] = scale * torch.tensor([1.0, 0.5, -0.5, 0.25] * 64, device="cuda")
    x[3] = 0
    w = torch.ones(256, device="cuda")
    check_norm(x, w, 1e-12, None, ops.rms_norm_q8(x, w, 1e-12))


def test_norm_not_finite_rows_stay_apart():
    x = torch.randn((4, 128), device="cuda")
    w = torch.ones(128, device="cuda")
    want = ops.rms_norm_q8(x, w)
    bad = x.clone()
    bad[1, 5] = float("inf")
    bad[2, 77] = float("nan")
    got = ops.rms_norm_q8(bad, w)
    assert torch.equal(got[[0, 3]], want[[0, 3]])
    assert torch.isnan(_native.dequantize(got, 8)[1:3]).all()


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("k", [512, 20480])
def test_norm_in_place_and_strided(dtype, k):
    g = torch.Generator(device="cuda").manual_seed(k)
    x = torch.randn((9, k + 64), device="cuda", generator=g).to(DT[dtype])[:, :k]
    r = torch.randn((9, 2 * k), device="cuda", generator=g).to(DT[dtype])[:, k:]
    w = torch.rand(k, device="cuda", generator=g) - 0.5
    want = ops.rms_norm_q8(x, w, residual=r)
    check_norm(x, w, 1e-6, r, *want)
    x2, r2 = x.clone(), r.clone()
    b, t = ops.rms_norm_q8(x2, w, residual=r2, total=r2)
    assert t is r2 and torch.equal(b, want[0]) and torch.equal(r2, want[1]) and torch.equal(x2, x)
    r2 = r.clone()
    b, t = ops.rms_norm_q8(x2, w, residual=r2, total=x2)
    assert torch.equal(b, want[0]) and torch.equal(x2, want[1]) and torch.equal(r2, r)
    # rows that do not start on 16 bytes are copied first
    odd = torch.randn((3, k + 1), device="cuda", generator=g).to(DT[dtype])[:, 1:]
    check_norm(odd, w, 1e-6, None, ops.rms_norm_q8(odd, w))


# --- routing --------------------------------------------------------------------------------

def check_route(z, **kw):
    bias = kw.pop("bias", None)
    ids, w = ops.route(z, bias=None if bias is None else cuda(bias), **kw)
    wi, ww = ref.route(z.float().cpu().numpy(), bias=bias, **kw)
    assert np.array_equal(ids.cpu().numpy(), wi)
    # a float64 value rounded once to float32; float64 functions are good to a few 2^-53
    np.testing.assert_allclose(w.cpu().numpy(), ww, rtol=2.0 ** -23, atol=1e-40)


@pytest.mark.parametrize("e,k", [(1, 1), (2, 2), (33, 5), (64, 6), (100, 32), (128, 8), (256, 8), (300, 4), (1024, 9)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
def test_route(e, k, score, biased):
    rng = np.random.default_rng(e + k)
    z = cuda((rng.standard_normal((37, e)) * 3).astype(np.float32))
    bias = (rng.standard_normal(e) * 0.2).astype(np.float32) if biased else None
    check_route(z, top_k=k, score=score, bias=bias)
    check_route(z[:1], top_k=k, score=score, bias=bias, renormalize=False, scale=2.5)


@pytest.mark.parametrize("e,groups,kept,k", [(64, 8, 4, 8), (256, 8, 4, 8), (96, 3, 2, 6), (60, 60, 7, 7), (64, 64, 3, 3), (160, 8, 3, 6), (1024, 32, 5, 16)])
@pytest.mark.parametrize("group_score", ["max", "top2"])
@pytest.mark.parametrize("score,biased", [("softmax", False), ("sigmoid", True), ("sigmoid", False)])
def test_route_groups(e, groups, kept, k, group_score, score, biased):
    if e // groups == 1 and group_score == "top2":
        pytest.skip("groups of one expert have no second")
    rng = np.random.default_rng(e)
    z = cuda((rng.standard_normal((29, e)) * 2).astype(np.float32))
    bias = (rng.standard_normal(e) * 0.2).astype(np.float32) if biased else None
    check_route(z, top_k=k, score=score, bias=bias, n_groups=groups, groups_kept=kept, group_score=group_score)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_route_ties_and_strides(dtype):
    """Few distinct logits: the lowest expert of equal ones first."""
    rng = np.random.default_rng(3)
    z = cuda(rng.integers(-2, 3, (64, 200)).astype(np.float32)).to(DT[dtype])[:, 7:107]
    check_route(z, top_k=16)
    check_route(z, top_k=8, n_groups=10, groups_kept=3)
    check_route(z, top_k=5, score="sigmoid", bias=np.zeros(100, np.float32))
    check_route(torch.zeros((3, 64), device="cuda", dtype=DT[dtype]), top_k=4, n_groups=8, groups_kept=2)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups", [1, 4])
def test_route_masked(score, groups):
    """-inf, NaN and the type's lowest value in logits, rows without any expert, +inf."""
    rng = np.random.default_rng(5)
    z = rng.standard_normal((8, 64)).astype(np.float32)
    z[0] = -np.inf
    z[1] = np.nan
    z[2, 3:] = -np.inf
    z[3, ::2] = np.nan
    z[4] = np.finfo(np.float32).min
    z[4, 9] = 0
    z[5, 17] = np.inf
    z[6, [5, 6]] = np.inf
    z[7, 16:] = -np.inf
    kw = dict(top_k=4, score=score, n_groups=groups, groups_kept=min(groups, 2))
    check_route(cuda(z), **kw)
    bias = rng.standard_normal(64).astype(np.float32) * 0.1
    bias[[1, 2]] = -np.inf, np.nan
    check_route(cuda(z[:4]), bias=bias, **kw)


def test_route_near_ties():
    """Scores that differ by less than a float32 step are ordered as in 64 bits."""
    rng = np.random.default_rng(7)
    z = (rng.standard_normal((512, 64)) * 1e-6).astype(np.float32)
    bias = (rng.integers(0, 3, 64) * 1e-7).astype(np.float32)
    for score in ("softmax", "sigmoid"):
        check_route(cuda(z), top_k=8, score=score, bias=bias)
        check_route(cuda(z), top_k=8, score=score, bias=bias, n_groups=8, groups_kept=4, group_score="top2")


@pytest.mark.parametrize("tokens,top,e", [(1, 1, 1), (1, 8, 64), (7, 3, 5), (1000, 4, 100), (2049, 8, 256), (5, 2, 1024)])
def test_plan(tokens, top, e):
    rng = np.random.default_rng(tokens)
    ids = rng.integers(-2, e + 2, (tokens, top)).astype(np.int32)
    p = ops.expert_plan(cuda(ids), e)
    order, offsets = ref.plan(ids, e)
    assert np.array_equal(p.order.cpu().numpy(), order) and np.array_equal(p.offsets.cpu().numpy(), offsets)


# --- products -------------------------------------------------------------------------------

def check_product(got, y, bound):
    dtype = str(got.dtype).split(".")[1]
    err = np.abs(got.float().cpu().numpy().astype(np.float64) - y)
    lim = bound + ref.rounding(np.abs(y) + bound, dtype)
    assert (err <= lim).all(), f"worst {np.nanmax(err / np.maximum(lim, 1e-300)):.3g} of the bound"


@pytest.mark.parametrize("qtype", ref.TYPES)
@pytest.mark.parametrize("rows", [1, 2, 4, 5, 8, 9, 33, 70, 200])
def test_matmul(qtype, rows):
    rng = np.random.default_rng(rows)
    k = 7 * 32 if ref.qk(qtype) == 32 else 768
    w = ref.random_blocks(qtype, (131,), k, rng)
    x = ref.random_blocks("q8_0", (rows,), k, rng)
    check_product(ops.matmul(cuda(w), int(ref.GTYPE[qtype]), cuda(x)), *ref.product(x, w, qtype))


@pytest.mark.parametrize("qtype", ["q4_0", "q2_k", "q4_k", "q6_k", "iq2_xs"])
@pytest.mark.parametrize("rows,n,k", [(1, 1, 256), (1, 4096, 256), (3, 33, 16384), (8, 16, 5120), (12, 5, 14336), (61, 128, 8192), (129, 384, 1024), (300, 260, 512)])
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_matmul_sizes(qtype, rows, n, k, dtype):
    rng = np.random.default_rng(n + k)
    w = ref.random_blocks(qtype, (n,), k, rng)
    x = ref.random_blocks("q8_0", (rows,), k, rng)
    got = ops.matmul(cuda(w), int(ref.GTYPE[qtype]), cuda(x), out_dtype=DT[dtype])
    check_product(got, *ref.product(x, w, qtype, dtype))


@pytest.mark.parametrize("qtype", ref.TYPES)
@pytest.mark.parametrize("rows", [130, 257])
def test_matmul_wide_tiles(qtype, rows):
    """Tiles of 256 slots that fill the GPU without splitting rows, an odd number of them, a ragged last one."""
    rng = np.random.default_rng(rows)
    k, n = (5 * 32 if ref.qk(qtype) == 32 else 512), 149 * 128 - 27 if rows < 256 else 75 * 128 - 27
    w = ref.random_blocks(qtype, (n,), k, rng)
    x = ref.random_blocks("q8_0", (rows,), k, rng)
    got = ops.matmul(cuda(w), int(ref.GTYPE[qtype]), cuda(x), out_dtype=torch.bfloat16)
    check_product(got, *ref.product(x, w, qtype, "bfloat16"))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("qtype,n,k", [("q6_k", 131, 768), ("q2_k", 131, 768), ("q4_k", 131, 768), ("q4_k", 2048, 16384)])
@pytest.mark.parametrize("rows", [32, 33, 64, 65])
def test_matmul_between_kernels(qtype, n, k, rows, dtype):
    """Row counts at which another kernel takes over, for formats and sizes on both sides of the rule."""
    rng = np.random.default_rng(rows)
    w = ref.random_blocks(qtype, (n,), k, rng)
    x = ref.random_blocks("q8_0", (rows,), k, rng)
    got = ops.matmul(cuda(w), int(ref.GTYPE[qtype]), cuda(x), out_dtype=DT[dtype])
    check_product(got, *ref.product(x, w, qtype, dtype))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("qtype", ["q4_0", "q4_k", "q6_k"])
@pytest.mark.parametrize("tokens", [32, 33, 56, 57])
def test_experts_between_kernels(qtype, tokens, dtype):
    """Averages at which another kernel takes over; one expert has no slot, one three times the average."""
    rng = np.random.default_rng(tokens)
    e, n, k = 4, 131, 512
    w = ref.random_blocks(qtype, (e, n), k, rng)
    x = ref.random_blocks("q8_0", (tokens * e,), k, rng)
    ids = np.full((tokens * e, 1), 1, dtype=np.int32)
    ids[:tokens] = 3
    got = ops.matmul_experts(cuda(w), int(ref.GTYPE[qtype]), cuda(x), ops.expert_plan(cuda(ids), e), out_dtype=DT[dtype])
    check_product(got, *experts_want(x, w, qtype, ids, None, True, dtype))


@pytest.mark.parametrize("qtype", ["q4_k", "q5_0"])
@pytest.mark.parametrize("weighted", [False, True])
def test_experts_wide_tiles(qtype, weighted):
    rng = np.random.default_rng(41)
    e, tokens, n, k = 8, 1300, 19 * 128, 256
    w = ref.random_blocks(qtype, (e, n), k, rng)
    x = ref.random_blocks("q8_0", (tokens,), k, rng)
    ids = rng.integers(-1, e, (tokens, 1)).astype(np.int32)
    ids[:700] = 5
    wt = rng.random((tokens, 1)).astype(np.float32) if weighted else None
    got = ops.matmul_experts(cuda(w), int(ref.GTYPE[qtype]), cuda(x), ops.expert_plan(cuda(ids), e), weights=None if wt is None else cuda(wt), out_dtype=torch.bfloat16)
    check_product(got, *experts_want(x, w, qtype, ids, wt, True, "bfloat16"))


@pytest.mark.parametrize("qtype", ["q8_0", "q4_k", "q6_k"])
@pytest.mark.parametrize("rows", [2, 40])
def test_matmul_strides(qtype, rows):
    """Row strides beyond the rows, activations at odd addresses, rows that follow stay untouched."""
    rng = np.random.default_rng(11)
    k, n = 512, 130
    w = ref.random_blocks(qtype, (n,), k, rng)
    x = ref.random_blocks("q8_0", (rows,), k, rng)
    wide = torch.full((n, w.shape[1] + 48), 255, dtype=torch.uint8, device="cuda")
    wide[:, 16:16 + w.shape[1]] = cuda(w)
    xs = torch.full((rows, x.shape[1] + 3), 255, dtype=torch.uint8, device="cuda")
    xs[:, 3:] = cuda(x)
    want = ops.matmul(cuda(w), int(ref.GTYPE[qtype]), cuda(x))
    got = ops.matmul(wide[:, 16:16 + w.shape[1]], int(ref.GTYPE[qtype]), xs[:, 3:])
    assert torch.equal(got, want)
    # rows behind the last, and columns behind the n-th
    L = _native.lib()
    import ctypes
    size = ctypes.c_int64()
    _native.check(L.qs_matmul_workspace(int(ref.GTYPE[qtype]), n, k, rows, 0, ctypes.byref(size)))
    ws = torch.empty(max(size.value, 1), dtype=torch.uint8, device="cuda")
    out = torch.full((rows + 1, n + 5), 7.0, device="cuda")
    wc, xc = cuda(w), cuda(x)
    _native.check(L.qs_matmul(int(ref.GTYPE[qtype]), wc.data_ptr(), w.shape[1], n, k, xc.data_ptr(), x.shape[1], rows, out.data_ptr(), 0,
                              n + 5, ws.data_ptr(), size.value, torch.cuda.current_stream().cuda_stream))
    assert torch.equal(out[:rows, :n], want) and (out[rows] == 7).all() and (out[:, n:] == 7).all()


@pytest.mark.parametrize("rows", [1, 6, 30, 150])
def test_matmul_extremes(rows):
    """Levels of -128 throughout (the largest sums), zero, infinite and NaN scales."""
    rng = np.random.default_rng(13)
    n, k = 140, 1024
    w = ref.random_blocks("q8_0", (n,), k, rng).reshape(n, -1, 34)
    x = ref.random_blocks("q8_0", (rows,), k, rng).reshape(rows, -1, 34)
    w[..., 2:], x[..., 2:] = 128, 128
    w[5, :, :2] = 0
    got = ops.matmul(cuda(w.reshape(n, -1)), 8, cuda(x.reshape(rows, -1)))
    check_product(got, *ref.product(x.reshape(rows, -1), w.reshape(n, -1), "q8_0"))
    clean = got.clone()
    w[3, 7, :2] = np.array([np.inf], np.float16).view(np.uint8)
    w[130, 0, :2] = np.array([np.nan], np.float16).view(np.uint8)
    got = ops.matmul(cuda(w.reshape(n, -1)), 8, cuda(x.reshape(rows, -1)))
    keep = [i for i in range(n) if i not in (3, 130)]
    assert not torch.isfinite(got[:, [3, 130]]).any() and torch.equal(got[:, keep], clean[:, keep])


def experts_want(x, w, qtype, ids, weights, per_slot, out="float32"):
    t, k = ids.shape
    n = w.shape[1]
    y, b = np.zeros((t, k, n)), np.zeros((t, k, n))
    for e in range(w.shape[0]):
        i, j = np.nonzero(ids == e)
        if len(i):
            y[i, j], b[i, j] = ref.product(x[i * k + j if per_slot else i], w[e], qtype, out)
    if weights is None:
        return y, b
    wt = weights[..., None].astype(np.float64)
    s = np.abs(wt) * (np.abs(y) + b)
    # a rounded product and a rounded addition per slot
    return np.nansum(np.where(y == 0, 0, y * wt), 1), (np.abs(wt) * b).sum(1) + k * 2.0 ** -23 * s.sum(1)


@pytest.mark.parametrize("qtype", ["q4_k", "q6_k", "q8_0", "iq3_xxs", "q2_k"])
@pytest.mark.parametrize("tokens,top,e", [(1, 1, 1), (1, 3, 8), (2, 2, 3), (9, 2, 4), (40, 4, 6), (3, 6, 40), (200, 1, 2)])
@pytest.mark.parametrize("per_slot", [False, True])
@pytest.mark.parametrize("weighted", [False, True])
def test_experts(qtype, tokens, top, e, per_slot, weighted):
    rng = np.random.default_rng(tokens + e)
    n, k = 70, 256
    w = ref.random_blocks(qtype, (e, n), k, rng)
    x = ref.random_blocks("q8_0", (tokens * top if per_slot else tokens,), k, rng)
    ids = rng.integers(0, e, (tokens, top)).astype(np.int32)  # the same expert twice among them
    if tokens > 2:
        ids[1], ids[2, 0], ids[-1, -1] = -1, e, -5
    wt = rng.random((tokens, top)).astype(np.float32) if weighted else None
    p = ops.expert_plan(cuda(ids), e)
    got = ops.matmul_experts(cuda(w), int(ref.GTYPE[qtype]), cuda(x), p, weights=None if wt is None else cuda(wt))
    check_product(got, *experts_want(x, w, qtype, ids, wt, per_slot or top == 1))


@pytest.mark.parametrize("tokens,top,e", [(3000, 4, 300), (800, 4, 20), (700, 2, 9), (2100, 1, 1000)])
@pytest.mark.parametrize("dtype,weighted", [("float32", False), ("bfloat16", True)])
def test_experts_many(tokens, top, e, dtype, weighted):
    """Many experts of very different popularity, ids that name none, several tiles per expert."""
    rng = np.random.default_rng(e)
    n, k = 70, 512
    w = ref.random_blocks("q5_k", (e, n), k, rng)
    x = ref.random_blocks("q8_0", (tokens,), k, rng)
    ids = np.minimum((e * rng.random((tokens, top)) ** 2).astype(np.int32), e - 1)
    ids[rng.random((tokens, top)) < 0.05] = -1
    wt = rng.random((tokens, top)).astype(np.float32) if weighted else None
    got = ops.matmul_experts(cuda(w), 13, cuda(x), ops.expert_plan(cuda(ids), e), weights=None if wt is None else cuda(wt), out_dtype=DT[dtype])
    check_product(got, *experts_want(x, w, "q5_k", ids, wt, False, dtype))


def test_products_on_two_streams():
    """Products of every kernel under way at the same time give the bits that they give alone."""
    rng = np.random.default_rng(31)
    w = cuda(ref.random_blocks("q4_k", (1024,), 2048, rng))
    xs = [cuda(ref.random_blocks("q8_0", (r,), 2048, rng)) for r in (1, 4, 7, 60, 100, 600)]
    want = [ops.matmul(w, 12, x, out_dtype=d) for x in xs for d in (torch.float32, torch.bfloat16)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for _ in range(4):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                order = xs[i:] + xs[:i]
                got.append([ops.matmul(w, 12, x, out_dtype=d) for x in order for d in (torch.float32, torch.bfloat16)])
    torch.cuda.synchronize()
    for n, g in enumerate(got):
        i = 2 * (n % 3)
        assert all(torch.equal(p, q) for p, q in zip(g, want[i:] + want[:i]))


def test_experts_all_empty_and_one_crowded():
    rng = np.random.default_rng(17)
    w = ref.random_blocks("q4_k", (5, 64), 256, rng)
    x = ref.random_blocks("q8_0", (300,), 256, rng)
    ids = np.full((300, 2), -1, np.int32)
    got = ops.matmul_experts(cuda(w), 12, cuda(x), ops.expert_plan(cuda(ids), 5), out_dtype=torch.bfloat16)
    assert (got == 0).all()
    got = ops.matmul_experts(cuda(w), 12, cuda(x), ops.expert_plan(cuda(ids), 5), weights=torch.full((300, 2), float("nan"), device="cuda"))
    assert (got == 0).all()
    ids[:] = 3
    got = ops.matmul_experts(cuda(w), 12, cuda(x), ops.expert_plan(cuda(ids), 5))
    check_product(got, *experts_want(x, w, "q4_k", ids, None, False))


# --- together -------------------------------------------------------------------------------

def layer(x, residual, norm_w, router, w_up, w_down, top):
    """A layer of experts on packed weights: norm, choice, up product, squares, down product."""
    h, total = ops.rms_norm_q8(x, norm_w, 1e-6, residual=residual)
    ids, wts = ops.route(ops.matmul(router, 8, h), top, score="sigmoid", scale=1.5)
    plan = ops.expert_plan(ids, w_up.shape[0])
    up = ops.matmul_experts(w_up, 12, h, plan)
    act = _native.quantize(8, torch.relu(up).square().reshape(-1, up.shape[-1]), None)
    return total, ids, ops.matmul_experts(w_down, 14, act, plan, weights=wts, out_dtype=x.dtype)


def layer_inputs(tokens, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    e, hid, mid = 6, 512, 256
    rnd = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
    pack = lambda t, *s: _native.quantize(t, rnd(int(np.prod(s[:-1])), s[-1]) * 0.05, None).reshape(*s[:-1], -1)  # noqa: E731
    return [rnd(tokens, hid).to(torch.bfloat16), rnd(tokens, hid).to(torch.bfloat16), 1 + 0.1 * rnd(hid), pack(8, e, hid), pack(12, e, mid, hid),
            pack(14, e, hid, mid), 2]


@pytest.mark.parametrize("tokens", [1, 5, 77])
def test_layer(tokens):
    """The operators one after the other against the same layer in 64 bits from the packed values.
    The choices and the intermediate 8-bit levels are taken as computed (each is tested above)."""
    a = layer_inputs(tokens, tokens)
    x, residual, nw, router, wu, wd, top = a
    total, ids, out = layer(*a)
    h, t2 = ops.rms_norm_q8(x, nw, 1e-6, residual=residual)
    check_norm(x, nw, 1e-6, residual, h, total)
    hn, idn = h.cpu().numpy(), ids.cpu().numpy()
    z, zb = ref.product(hn, router.cpu().numpy(), "q8_0")
    s = 1 / (1 + np.exp(-z))
    pick = np.take_along_axis(s, idn.astype(np.int64), 1)
    # the chosen scores are the largest but for the logits' own error (a sigmoid's slope is <= 1/4)
    assert (np.sort(s, 1)[:, ::-1][:, :top] - pick <= zb.max() / 2).all()
    up, ub = experts_want(hn, wu.cpu().numpy(), "q4_k", idn, None, False)
    got_up = ops.matmul_experts(wu, 12, h, ops.expert_plan(ids, 6))
    check_product(got_up, up, ub)
    act = _native.quantize(8, torch.relu(got_up).square().reshape(-1, 256), None).cpu().numpy()
    wts = (1.5 * pick / pick.sum(1, keepdims=True)).astype(np.float32)
    y, b = experts_want(act, wd.cpu().numpy(), "q6_k", idn, wts, True, "bfloat16")
    # weights: the logits' error in the scores, twice (score and sum), and their rounding
    slack = (4 * zb.max() + 2.0 ** -22) * np.abs(experts_want(act, wd.cpu().numpy(), "q6_k", idn, None, True)[0]).sum(1) * 1.5
    check_product(out, y, b + slack)


@pytest.mark.parametrize("tokens", [1, 40])
def test_layer_captured_and_on_another_stream(tokens):
    """Two captured graphs and a second stream give the eager results, with new inputs too."""
    a, b = layer_inputs(tokens, 1), layer_inputs(tokens, 2)
    want = [layer(*a), layer(*b)]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = layer(*a)
    side.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want[0]))
    graphs = []
    for src in (a, b):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = layer(*src)
        graphs.append((g, outs))
    for _ in range(3):
        for g, _ in graphs:
            g.replay()
    torch.cuda.synchronize()
    for (_, outs), w in zip(graphs, want):
        assert all(torch.equal(p, q) for p, q in zip(outs, w))
    for t, u in zip(a[:6], b[:6]):  # the first graph on the second layer's data
        t.copy_(u)
    graphs[0][0].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(graphs[0][1], want[1]))


def test_same_bits_every_time():
    rng = np.random.default_rng(23)
    w, x = cuda(ref.random_blocks("q4_k", (4, 512), 4096, rng)), cuda(ref.random_blocks("q8_0", (100,), 4096, rng))
    ids = cuda(rng.integers(0, 4, (100, 2)).astype(np.int32))
    wt = torch.rand((100, 2), device="cuda")
    first = None
    for _ in range(5):
        got = (ops.matmul(w[0], 12, x), ops.matmul(w[0], 12, x[:3]), ops.matmul_experts(w, 12, x, ops.expert_plan(ids, 4), weights=wt))
        first = first or got
        assert all(torch.equal(p, q) for p, q in zip(got, first))


def test_empty_calls():
    x = torch.empty((0, 256), device="cuda")
    assert ops.rms_norm_q8(x, torch.ones(256, device="cuda")).shape == (0, 272)
    assert ops.route(torch.empty((0, 8), device="cuda"), 2)[0].shape == (0, 2)
    w = torch.zeros((3, 4, 144), dtype=torch.uint8, device="cuda")
    none = torch.empty((0, 272), dtype=torch.uint8, device="cuda")
    assert ops.matmul(w[0], 12, none).shape == (0, 4)
    p = ops.expert_plan(torch.empty((0, 2), dtype=torch.int32, device="cuda"), 3)
    assert p.offsets.tolist() == [0, 0, 0, 0]
    assert ops.matmul_experts(w, 12, none, p).shape == (0, 2, 4)


def test_refusals_on_the_gpu():
    w = torch.zeros((4, 144), dtype=torch.uint8, device="cuda")
    x = torch.zeros((2, 272), dtype=torch.uint8, device="cuda")
    for call in (lambda: ops.matmul(w, 12, x[:, :34]), lambda: ops.matmul(w[:, :100], 12, x), lambda: ops.matmul(w, 12, x.cpu()),
                 lambda: ops.matmul(w, 12, x, out_dtype=torch.float64), lambda: ops.matmul(w.int(), 12, x),
                 lambda: ops.rms_norm_q8(torch.zeros((2, 40), device="cuda"), torch.ones(40, device="cuda")),
                 lambda: ops.rms_norm_q8(torch.zeros((2, 64), device="cuda"), torch.ones(32, device="cuda")),
                 lambda: ops.rms_norm_q8(torch.zeros((2, 64), device="cuda"), torch.ones(64, device="cuda"), 0.0),
                 lambda: ops.route(torch.zeros((2, 8), device="cuda"), 9), lambda: ops.route(torch.zeros((2, 8), device="cuda"), 0),
                 lambda: ops.route(torch.zeros((2, 8), device="cuda"), 2, score="relu"),
                 lambda: ops.expert_plan(torch.zeros((2, 2), dtype=torch.int64, device="cuda"), 4),
                 lambda: ops.matmul_experts(w[None], 12, x, ops.expert_plan(torch.zeros((2, 2), dtype=torch.int32, device="cuda"), 4)),
                 lambda: ops.matmul_experts(w[None], 12, x[:1], ops.expert_plan(torch.zeros((2, 2), dtype=torch.int32, device="cuda"), 1))):
        with pytest.raises(_native.QsError):
            call()
