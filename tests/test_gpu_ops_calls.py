"""Calls of the operators on packed blocks at the edges of what they allow, on the GPU."""

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
