"""Caches of eight bits: outputs of 16 bits are the exact ones, rounded once, but for what sums in 32 bits lose; pages of bytes without scales."""
from types import SimpleNamespace

import pytest
import torch

import kv8_util as ku

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dim,qpk", [(64, 8), (128, 4), (256, 2), (80, 3)])
def test_rows_of_bf16_have_weights_of_more_bits_than_their_output(cuda, fmt, dim, qpk):
    """Values are positive and scores small, so that the tolerance of rows of 32 bits (kv8_util.reference) is about 2^-16 of an output: a weight that keeps eleven bits is off by eight times that and moves
    what lies near the middle of two numbers of bf16.  The output itself is off by half a step of bf16."""
    s = ku.cached(ku.batch([1] * 6, [2, 5, 11, 40, 90, 300], torch.bfloat16, ku.DT[fmt], dim=dim, n_kv=2, qpk=qpk, seed=dim))
    raw = s.pool.view(torch.uint8)
    raw.copy_(s.pool.view(torch.int8).abs().view(torch.uint8) if fmt == "int8" else raw & 0x7f)
    s.qkv *= 0.02
    out = ku.attend(s, s.qkv).double().view(s.n_tok, s.heads, s.vdim)
    want, tol = ku.reference(SimpleNamespace(**{**vars(s), "dtype": torch.float32}), s.qkv)
    assert (tol <= 2.0 ** -15 * want).all()          # (the inputs are what the text says)
    off = (out - want).abs()
    bad = off > tol + torch.finfo(torch.bfloat16).eps / 2 * want
    assert not bad.any(), (int(bad.sum()), bad.numel(), (off / want).max().item())


@pytest.mark.parametrize("dim,vdim", [(64, 64), (576, 0), (300, 17)])
def test_pages_of_bytes_are_copied(cuda, dim, vdim):
    from poptransformer_b200 import ops
    kv = ops.PagedKVCache(2, 3, dim, 128, 64, cuda, v_dim=vdim, dtype=torch.uint8)
    kv.pool.random_(0, 256)
    want = kv.pool.clone()
    want[3] = want[0]
    ops.PagePools([kv]).copy_pages(ku.ints([0]), ku.ints([3]))
    assert torch.equal(kv.pool, want)


@pytest.mark.parametrize("rot", [32, 64])
def test_appending_turns_what_the_table_turns(cuda, rot):
    from poptransformer_b200 import ops
    s = ku.batch([5, 2], [10, 70], torch.float16, torch.int8, rot=rot, seed=rot)
    pool, scales, q = ku.appended(s)
    out = torch.empty((s.n_tok, s.q_cols), dtype=s.dtype, device=cuda)
    ops.kv8_append(s.view, s.qkv, s.ld, s.cache, s.heads, rope=s.rope, q_out=out, q_out_ld=s.q_cols, error_flag=s.flag)
    assert torch.equal(s.pool.view(torch.uint8).cpu(), pool) and torch.equal(s.scales.cpu().nan_to_num(-1), scales.nan_to_num(-1)) and torch.equal(out.cpu(), q.to(s.dtype)) and s.flag.item() == 0
