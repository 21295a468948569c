"""Attention of drafted tokens where one key has by far the highest score and all of the output is the others': they count as exactly as 16-bit weights allow."""
import math

import pytest
import torch

import tree_util as tu

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# few sequences, whose keys many blocks share, and many, where a block has a sequence's keys to itself
@pytest.mark.parametrize("n_seq", [1, 60, 200])
@pytest.mark.parametrize("dtype,plain", [("fp16", False), ("bf16", False), ("fp16", True), ("fp32", False)])
@pytest.mark.parametrize("below", [8.0, 12.0, 14.5, 17.5, 19.0])
@pytest.mark.parametrize("where", [3, 1500])
def test_flat_tail_behind_a_spike(cuda, n_seq, dtype, plain, below, where):
    """A weight and the output are rounded to 16 bits at most once (bf16: the weights in two parts, 2^-15), the fp32 sums lose 2^-23 a key."""
    n, C, D = 4, 2000, 64
    s = tu.batch([n] * n_seq, [C] * n_seq, "tree", dtype=DT[dtype], dim=D, n_kv=2, qpk=2, seed=51)
    s.scale = 1.0
    g = torch.Generator(device=cuda).manual_seed(52)
    pool, cut = s.cache.pool, s.heads * D
    # scores are exact: q is a unit vector, and the keys' first channel is the score
    pool[:, 0] = 0
    pool[:, 0, ..., 0] = -below
    pool[:, 1] = (torch.rand(pool[:, 1].shape, generator=g, device=cuda) * 250 + 250).to(s.dtype)
    for i in range(n_seq):
        page = s.table[s.slot[i]][where // s.page]
        pool[page, 0, :, where % s.page, 0] = 0
        pool[page, 1, :, where % s.page] = 0               # all of the output is the tail's
    s.qkv[:] = 0
    s.qkv[:, :cut].view(-1, s.heads, D)[:, :, 0] = 1
    s.qkv[:, cut:cut + s.n_kv * D].view(-1, s.n_kv, D)[:, :, 0] = -below
    s.qkv[:, cut + s.n_kv * D:] = 300
    out = tu.run(s, plain=plain).double()
    half = torch.finfo(s.dtype).eps / 2
    w = math.exp(-below)
    for i in range(n_seq):
        _, V = tu._pages(s, s.cache.pool, i, C)
        up = torch.tensor([len(a) for a in tu.lines(s.parents[i])], dtype=torch.float64, device=cuda)
        tail = V.sum(1)[None] + 300 * up[:, None, None]    # [n, n_kv, D]
        exp = (w * tail / (1 + (C - 1 + up[:, None, None]) * w))[:, :, None].expand(n, 2, 2, D).reshape(n, s.heads * D)
        bound = exp * (half + max(2.0 ** -11 if s.dtype == torch.float16 else 0.0, 2.0 ** -15) + (C + n) * 2.0 ** -23)
        worst = float(((out[s.cu[i]:s.cu[i] + n] - exp).abs() / bound).max())
        assert worst <= 1.0, f"sequence {i}: off by {worst:.2f} of the tolerance"


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


@pytest.mark.parametrize("dtype,plain", [("fp16", False), ("bf16", False), ("bf16", True), ("fp32", False)])
@pytest.mark.parametrize("power", [9, 14, 20, 24, 30, 40, 60])
@pytest.mark.parametrize("times", [0.01, 0.3, 1.0])
def test_capped_scores_of_any_size(cuda, dtype, plain, power, times):
    """Caps that the scores come near: the largest has all the weight, or shares it with those that fp32 cannot tell from it."""
    n, C, D = 7, 900, 64
    s = tu.batch([n, 3], [C, 70], "tree", dtype=DT[dtype], dim=D, n_kv=2, qpk=2, seed=53)
    cap = 2.0 ** power
    s.scale = times * cap
    pool, cut = s.cache.pool, s.heads * D
    pool[:, 0, ..., 1:] = 0
    s.qkv[:, :cut + s.n_kv * D].view(-1, s.heads + s.n_kv, D)[:, :, 1:] = 0
    s.qkv[:, :cut].view(-1, s.heads, D)[:, :, 0] = 1
    out = tu.run(s, softcap=cap, plain=plain).double()
    assert torch.isfinite(out).all() and s.flag.item() == 0
    for i, (n, C) in enumerate(zip(s.counts, s.starts)):
        K, V = tu._pages(s, s.cache.pool, i, C + n)
        seen = torch.zeros((n, C + n), dtype=torch.bool, device=cuda)
        seen[:, :C] = True
        for r, up in enumerate(tu.lines(s.parents[i])):
            seen[r, [C + b for b in up]] = True
        z = (cap * torch.tanh(K[:, :, 0] * s.scale / cap))[:, None].expand(-1, n, -1).masked_fill(~seen, -math.inf)
        # capped scores are right to 2^-19 of themselves: the output lies between the smallest and the largest value of those that may have weight
        top = z.amax(-1, keepdim=True)
        may = z >= top - top.abs() * 2.0 ** -18 - 40
        big = V[:, None].masked_fill(~may[..., None], -math.inf).amax(2)[:, :, None].expand(-1, n, 2, D).permute(1, 0, 2, 3).reshape(n, -1)
        small = V[:, None].masked_fill(~may[..., None], math.inf).amin(2)[:, :, None].expand(-1, n, 2, D).permute(1, 0, 2, 3).reshape(n, -1)
        got, slack = out[s.cu[i]:s.cu[i] + n], torch.finfo(s.dtype).eps * torch.maximum(big.abs(), small.abs()) + 2.0 ** -12 * V.abs().max()
        assert ((got <= big + slack) & (got >= small - slack)).all(), i
