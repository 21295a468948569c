"""Prompts over caches of eight bits, by the kernels that read unpacked pages: fp32 pages for rows of any type, fp16 pages for chunks of 256 tokens."""
from types import SimpleNamespace

import pytest
import torch

import kv8_util as ku

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["fp16", "fp32", "bf16"])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("window", [0, 40])
def test_a_prompt_by_pages_of_32_bits(cuda, dtype, fmt, window):
    """Nothing but the output is rounded to the rows' type.  Against the bytes in 64 bits; kv8_util.reference's tolerance of fp32 rows has the scores (unpacked keys are off by 2^-24 each, its dim + 8 count
    them) and the exponentials.  The kernel adds up to n weighted values one by one, and as many weights: 2 n 2^-24 of the largest value more."""
    from poptransformer_b200 import ops
    s = ku.batch([70, 1, 130], [0, 200, 63], ku.DT[dtype], ku.DT[fmt], n_kv=2, qpk=3, dim=64, rot=32, seed=1, slots=5)
    q = torch.empty((s.n_tok, s.q_cols), dtype=s.dtype, device=cuda)
    ops.kv8_append(s.view, s.qkv, s.ld, s.cache, s.heads, rope=s.rope, q_out=q, q_out_ld=s.q_cols, error_flag=s.flag)
    wide = ops.PagedKVCache(5, s.n_kv, s.dim, s.max_len, 64, cuda, dtype=torch.float32)
    ops.kv8_unpack(s.view, s.cache, wide, error_flag=s.flag)
    out = torch.empty((s.n_tok, s.q_cols), dtype=torch.float32, device=cuda)
    ops.window_attn(s.view, q.float(), s.q_cols, wide, out, s.q_cols, s.heads, s.scale, window=window, append=False, max_tokens_per_seq=130, error_flag=s.flag)
    want, tol = ku.reference(SimpleNamespace(**{**vars(s), "dtype": torch.float32}), q, window)
    n = max(a + b for a, b in zip(s.counts, s.starts))
    most = max(float(ku.history(s, i, s.starts[i] + s.counts[i], 1).abs().max()) for i in range(3))
    tol = tol + 2 * n * 2.0 ** -24 * most
    assert ((out.double().view(s.n_tok, s.heads, -1) - want).abs() <= tol).all() and s.flag.item() == 0
    rounded = out.to(s.dtype).double().view(s.n_tok, s.heads, -1)
    assert ((rounded - want).abs() <= tol + torch.finfo(s.dtype).eps / 2 * (want.abs() + tol) + 2.0 ** -25).all()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dim,page", [(128, 64), (80, 16)])
def test_a_chunk_of_fp16_behind_a_cached_beginning(cuda, fmt, dim, page):
    """The beginning is unpacked to fp16, tree_attn reads it and appends the chunk's keys and values in 16 bits; kv8_append keeps the same rows in eight for later."""
    from poptransformer_b200 import ops
    s = ku.batch([70, 1, 256], [0, 200, 63], torch.float16, ku.DT[fmt], n_kv=2, qpk=3, dim=dim, page=page, seed=2, slots=5)
    wide = ops.PagedKVCache(5, s.n_kv, dim, s.max_len, page, cuda, dtype=torch.float16)
    before = ops.batch_view(3, 0, ku.ints([0, 0, 0, 0]), s.start, s.slot, ku.ints([]))       # (no new token yet: what is cached)
    ops.kv8_unpack(before, s.cache, wide, error_flag=s.flag)
    out = torch.empty((s.n_tok, s.q_cols), dtype=torch.float16, device=cuda)
    ws = ops.tree_attn_workspace(3, 256, s.heads, s.n_kv, dim)
    ops.tree_attn(s.view, s.qkv, s.ld, wide, out, s.q_cols, s.heads, s.scale, max_tokens_per_seq=256, workspace=ws, error_flag=s.flag)
    pool, scales, _ = ku.appended(s)
    ops.kv8_append(s.view, s.qkv, s.ld, s.cache, s.heads, error_flag=s.flag)
    assert torch.equal(s.pool.view(torch.uint8).cpu(), pool) and s.flag.item() == 0
    rows, half = s.qkv.double(), 2.0 ** -11
    for i, (n, C) in enumerate(zip(s.counts, s.starts)):
        x = rows[s.cu_host[i]:s.cu_host[i] + n]
        new = [x[:, s.q_cols + w * s.n_kv * dim:s.q_cols + (w + 1) * s.n_kv * dim].view(n, s.n_kv, dim).transpose(0, 1) for w in (0, 1)]
        K, V = (torch.cat([ku.history(s, i, C, w).float().half().double(), new[w]], 1) if C else new[w] for w in (0, 1))
        q = x[:, :s.q_cols].view(n, s.n_kv, 3, dim).permute(1, 2, 0, 3)
        seen = torch.arange(C + n, device=cuda) <= C + torch.arange(n, device=cuda)[:, None]
        z = q @ K[:, None].transpose(-1, -2) * s.scale
        size = (q.abs() @ K[:, None].abs().transpose(-1, -2) * s.scale).masked_fill(~seen, 0.0).amax(-1, keepdim=True)
        p = torch.softmax(z.masked_fill(~seen, -torch.inf), -1)
        want, mean = p @ V[:, None], p @ V[:, None].abs()
        # as tests of tree_attn have it: products and sums of dim terms 2^-23 each, a score's error twice in a weight, weights 2^-15, sums 2^-24 a position; the output half a step
        tol = (2 * dim * 2.0 ** -23 * size + 2.0 ** -15 + (C + n) * 2.0 ** -24) * mean + half * want.abs() + 2.0 ** -24
        got = out[s.cu_host[i]:s.cu_host[i] + n].double().view(n, s.n_kv, 3, dim).permute(1, 2, 0, 3)
        assert ((got - want).abs() <= tol).all()
