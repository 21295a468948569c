"""Attention of drafted tokens with scores of any size."""
import math

import pytest
import torch

import tree_util as tu

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


@pytest.mark.parametrize("dtype,plain", [("fp16", False), ("bf16", False), ("fp16", True), ("bf16", True), ("fp32", False)])
@pytest.mark.parametrize("power", [0, 10, 18, 20, 21, 22, 23, 24, 25, 26, 27, 28, 30, 32, 34, 40, 100])
@pytest.mark.parametrize("sign", [1, -1])
def test_scores_of_any_size(cuda, dtype, plain, power, sign):
    """From some size on the largest score has all the weight; its neighbours in fp32 are then further apart than all that has weight."""
    n, C, D = 7, 900, 64
    s = tu.batch([n, 3], [C, 70], "tree", dtype=DT[dtype], dim=D, n_kv=2, qpk=2, seed=53)
    s.scale = sign * 2.0 ** power
    pool, cut = s.cache.pool, s.heads * D
    pool[:, 0, ..., 1:] = 0                            # (scores are exact in fp32)
    s.qkv[:, :cut + s.n_kv * D].view(-1, s.heads + s.n_kv, D)[:, :, 1:] = 0
    s.qkv[:, :cut].view(-1, s.heads, D)[:, :, 0] = 1
    before = pool.clone()
    out = tu.run(s, plain=plain).double()
    assert torch.isfinite(out).all() and s.flag.item() == 0
    half = torch.finfo(s.dtype).eps / 2
    for i, (n, C) in enumerate(zip(s.counts, s.starts)):
        K, V = tu._pages(s, s.cache.pool, i, C + n)
        seen = torch.zeros((n, C + n), dtype=torch.bool, device=cuda)
        seen[:, :C] = True
        for r, up in enumerate(tu.lines(s.parents[i])):
            seen[r, [C + b for b in up]] = True
        z = (K[:, :, 0] * s.scale)[:, None].expand(-1, n, -1).masked_fill(~seen, -math.inf)
        # fp32 keeps a score, and its product with log2(e), to 2^-23 of itself: what lies nearer to the largest than 2^-21 of it may be weighed otherwise
        top = z.amax(-1, keepdim=True)
        second = torch.where(z == top, torch.full_like(z, -math.inf), z).amax(-1, keepdim=True)
        assert power < 10 or bool(((top - second) > top.abs() * 2.0 ** -21 + 60).all())
        w = torch.softmax(z, -1)
        exp = (w @ V)[:, :, None].expand(-1, n, 2, D).permute(1, 0, 2, 3).reshape(n, -1)
        slack = (half + 2.0 ** -14 + (C + n) * 2.0 ** -23) * (w @ V.abs())[:, :, None].expand(-1, n, 2, D).permute(1, 0, 2, 3).reshape(n, -1)
        assert ((out[s.cu[i]:s.cu[i] + n] - exp).abs() <= slack + 2.0 ** -25).all(), i
