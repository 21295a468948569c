"""Attention for trees of drafted tokens where values are infinite or NaN, and scores pass through caps of any size (tolerances: tree_util.reference)."""
import math

import pytest
import torch

import tree_util as tu

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


@pytest.mark.parametrize("dtype,plain", [("bf16", False), ("fp16", False), ("bf16", True)])
@pytest.mark.parametrize("window", [0, 70])
def test_many_short_sequences_whose_second_halves_are_bad(cuda, dtype, plain, window):
    """Every sequence is one tile of keys that no row sees whole, and most values in its second half are NaN: one of the two warps that bring tiles in has all the
    work, tile after tile.  Rows that see none of those values keep their bits."""
    n, n_seq = 60, 600
    s = tu.batch([n] * n_seq, [64] * n_seq, "star", dtype=DT[dtype], dim=64, n_kv=1, qpk=1, page=128, seed=21)
    before = s.cache.pool.clone()
    want = tu.run(s, window=window, plain=plain).clone()
    some = tu.batch([n] * 4, [64] * 4, "star", dtype=DT[dtype], dim=64, n_kv=1, qpk=1, page=128, seed=22)
    held = some.cache.pool.clone()
    tu.check(some, held, tu.run(some, window=window, plain=plain), window=window)
    s.cache.pool.copy_(before)
    bad = (torch.arange(s.n_tok, device=cuda) % n) % 8 != 0      # (the root, which all see, is good)
    s.qkv[bad, 2 * 64:] = float("nan")
    for _ in range(5):
        s.cache.pool.copy_(before)
        got = tu.run(s, window=window, plain=plain)
        assert s.flag.item() == 0
        assert torch.equal(got[~bad], want[~bad]) and got[bad].isnan().all()


def _capped(s, pool, softcap):
    """(out, tolerance) as tree_util.reference has them without a rotation, but for the cap, which is not allowed to be off by a part of itself.

    x = score / cap comes with three roundings, 2^-22 of it.  tanh by its series is right to 2^-21.  1 - 2 / (e^2x + 1) from x = 0.55 on: the exponential is off by 2^-22 of
    itself and by 2^-23 of its exponent, the quotient by 2^-22: 1.3 2^-22 in all, of a tanh of 0.5 and more 2^-20.  So a score is off by 2^-19 of itself, tanh's slope being
    at most tanh(x) / x.  Up to a cap of 256 it may be off by 2^-21 of the cap instead, with 16 bits."""
    half, out, tol = torch.finfo(s.dtype).eps / 2, [], []
    for i, (n, C) in enumerate(zip(s.counts, s.starts)):
        x = s.qkv[s.cu[i]:s.cu[i] + n].double()
        H, G, D, V = s.heads, s.n_kv, s.dim, s.vdim
        q, k, v = x[:, :H * D].view(n, H, D), x[:, H * D:(H + G) * D].view(n, G, D), x[:, (H + G) * D:].view(n, G, V)
        K, W = tu._pages(s, pool, i, C + n)
        K[:, C:], W[:, C:] = k.transpose(0, 1), v.transpose(0, 1)
        seen = torch.ones((n, C + n), dtype=torch.bool, device=s.device)
        seen[:, C:] = False
        for r, up in enumerate(tu.lines(s.parents[i])):
            seen[r, [C + b for b in up]] = True
        rows, slack_rows = [], []
        for h in range(H):
            g = h // s.qpk
            z = softcap * torch.tanh(q[:, h] @ K[g].T * s.scale / softcap)
            off = q[:, h].abs() @ K[g].abs().T * s.scale * D * 2.0 ** -23 + z.abs() * 2.0 ** -19
            if s.dtype != torch.float32 and softcap <= 256:
                off = off + softcap * 2.0 ** -21
            off = off.masked_fill(~seen, 0.0).amax(1, keepdim=True)
            w = torch.softmax(z.masked_fill(~seen, -math.inf), -1)
            rows.append(w @ W[g])
            slack_rows.append((torch.expm1(2 * off) + 2.0 ** -14 + (C + n) * 2.0 ** -23) * (w @ W[g].abs()))
        o, slack = torch.cat(rows, 1), torch.cat(slack_rows, 1)
        out.append(o)
        tol.append(half * o.abs() + (1 + half) * slack + torch.finfo(s.dtype).tiny)
    return torch.cat(out), torch.cat(tol)


@pytest.mark.parametrize("dtype,plain", [("bf16", False), ("fp16", False), ("bf16", True), ("fp32", False)])
@pytest.mark.parametrize("softcap", [0.5, 30.0, 256.0, 257.0, 1e4, 1e6, 1e8, 1e12, 1e20])
@pytest.mark.parametrize("scale", [0.3, -0.3])
def test_caps_of_any_size(cuda, dtype, plain, softcap, scale):
    """A cap that no score comes near changes next to nothing."""
    s = tu.batch([20, 7], [150, 700], dtype=DT[dtype], dim=128, seed=23)
    s.scale = scale                                    # scores up to 15 or so
    before = s.cache.pool.clone()
    out = tu.run(s, softcap=softcap, plain=plain)
    s.scale = abs(scale)
    if scale < 0:
        s.qkv[:, :s.heads * s.dim] *= -1
    ref, tol = _capped(s, before, softcap)
    worst = float(((out.double() - ref).abs() / tol).max())
    assert worst <= 1.0, f"off by {worst:.2f} of the tolerance"
