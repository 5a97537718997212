"""Plain 64-bit forms of the operators on packed blocks, and random packed blocks."""

import numpy as np
from gguf import GGML_QUANT_SIZES
from gguf import GGMLQuantizationType as GT
from gguf.quants import dequantize

TYPES = ["q4_0", "q4_1", "q5_0", "q5_1", "q8_0", "q2_k", "q3_k", "q4_k", "q5_k", "q6_k", "iq2_xxs", "iq2_xs", "iq2_s",
         "iq3_xxs", "iq3_s", "iq4_xs"]
GTYPE = {t: getattr(GT, t.upper()) for t in TYPES}
# places of the float16 scales (kept small and finite), and of the level bytes of formats with minima
F16 = {"q4_0": (0,), "q4_1": (0, 2), "q5_0": (0,), "q5_1": (0, 2), "q8_0": (0,), "q2_k": (80, 82), "q3_k": (108,),
       "q4_k": (0, 2), "q5_k": (0, 2), "q6_k": (208,), "iq2_xxs": (0,), "iq2_xs": (0,), "iq2_s": (0,), "iq3_xxs": (0,),
       "iq3_s": (0,), "iq4_xs": (0,)}
LEVELS = {"q4_1": (4, 20), "q5_1": (4, 24), "q2_k": (16, 80), "q4_k": (16, 144), "q5_k": (16, 176)}


def qk(qtype):
    return GGML_QUANT_SIZES[GTYPE[qtype]][0]


def random_blocks(qtype, shape, k, rng):
    q, bb = GGML_QUANT_SIZES[GTYPE[qtype]]
    b = rng.integers(0, 256, size=(*shape, k // q, bb), dtype=np.uint8)
    for off in F16[qtype]:
        d = (rng.standard_normal((*shape, k // q)) * 0.01).astype(np.float16)
        b[..., off:off + 2] = d.view(np.uint8).reshape(*shape, k // q, 2)
    return b.reshape(*shape, -1)


def decode64(blocks, qtype):
    flat = blocks.reshape(-1, blocks.shape[-1])
    return dequantize(flat, GTYPE[qtype]).astype(np.float64).reshape(*blocks.shape[:-1], -1)


def product(xq, w, qtype, out="float32"):
    """(y, bound): the 64-bit product and how far a float32 evaluation may be from it.

    Per unit of 32 values the integer sums are exact; a unit adds up to 4 terms (two halves, two
    minima), each with a rounded scale product and a rounded addition, and the terms of a row
    are added in any order: at most (8 units + 8) roundings, each of at most half a step of
    the sum of the terms' magnitudes. Minima are separate terms: |dl l| <= |w| + |ml|. gguf-py's
    decode rounds each weight once more. For bfloat16 results the activations may be rounded to
    float16 (half a step: 2^-11 of a value).
    """
    x, ww = decode64(xq, "q8_0"), decode64(w, qtype)
    mag = np.abs(ww)
    if qtype in LEVELS:
        z = w.reshape(*w.shape[:-1], -1, GGML_QUANT_SIZES[GTYPE[qtype]][1]).copy()
        lo, hi = LEVELS[qtype]
        z[..., lo:hi] = 0
        mag = mag + 2 * np.abs(decode64(z.reshape(w.shape), qtype))
    y = x @ np.swapaxes(ww, -1, -2)
    steps = (8 * (x.shape[-1] // 32) + 8) * 2.0 ** -24 + (2.0 ** -11 if out == "bfloat16" else 0.0)
    return y, steps * (np.abs(x) @ np.swapaxes(mag, -1, -2))


def rounding(y, dtype):
    """Half a step of the output type, at most (plus its smallest step near zero)."""
    return {"float32": 0.0, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}[dtype] * np.abs(y) + (2.0 ** -25 if dtype == "float16" else 0.0)


def norm_q8(t, weight, eps):
    """Q8_0 (scales float16, levels) of the norm of rows t, as defined: in float64, where products
    of float32 values are exact."""
    t, w = t.astype(np.float64), weight.astype(np.float64)
    r = 1.0 / np.sqrt((t * t).mean(-1, keepdims=True) + eps)
    p = (t * w).reshape(t.shape[0], -1, 32)
    m = np.abs(p).max(-1, keepdims=True)
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        q = np.where(m > 0, np.floor(127 * (np.abs(p) / m) + 0.5) * np.sign(p), 0)
        d = (m * (r[..., None] / 127)).astype(np.float32).astype(np.float16)
    return d[..., 0], q.astype(np.int8)


def split_q8(blocks):
    b = np.ascontiguousarray(blocks.reshape(blocks.shape[0], -1, 34))
    return b[..., :2].copy().view(np.float16)[..., 0], b[..., 2:].view(np.int8)


def route(z, top_k, score="softmax", bias=None, n_groups=1, groups_kept=1, group_score="max", renormalize=True, scale=1.0):
    z = z.astype(np.float64)
    n, e = z.shape
    ids, ws = np.full((n, top_k), -1, np.int32), np.zeros((n, top_k))
    for i in range(n):
        ok = z[i] > -np.inf
        s = np.zeros(e)
        if ok.any():
            if score == "softmax":
                m = z[i][ok].max()
                s[ok] = [1.0 if v == m else np.exp(v - m) for v in z[i][ok]]
                s /= s.sum()
            else:
                s[ok] = 1 / (1 + np.exp(-z[i][ok]))
        v = s + (0 if bias is None else bias.astype(np.float64))
        # scores are monotone in the logits, which order exactly
        by_logit = bias is None and not (n_groups > 1 and group_score == "top2")
        v = np.where(ok & ~np.isnan(v), z[i] if by_logit else v, -np.inf)
        if n_groups > 1:
            g = v.reshape(n_groups, -1)
            gs = g.max(1) if group_score == "max" else np.sort(g, 1)[:, -2:].sum(1) if g.shape[1] > 1 else np.full(n_groups, -np.inf)
            kept = np.argsort(-gs, kind="stable")[:groups_kept]
            mask = np.zeros(n_groups, bool)
            mask[kept] = True
            v = np.where(np.repeat(mask, e // n_groups), v, -np.inf)
        o = np.argsort(-v, kind="stable")[:top_k]
        o = o[v[o] > -np.inf]
        ids[i, :len(o)] = o
        w = s[o]
        if renormalize:
            w = w / w.sum() if len(o) and w.sum() > 0 else w * 0
        ws[i, :len(o)] = w * scale
    return ids, ws


def plan(ids, n_experts):
    flat = ids.reshape(-1)
    c = np.where((flat >= 0) & (flat < n_experts), flat, n_experts)
    order = np.argsort(c, kind="stable").astype(np.int32)
    return order, np.searchsorted(c[order], np.arange(n_experts + 1)).astype(np.int32)
