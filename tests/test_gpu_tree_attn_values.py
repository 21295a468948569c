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


def _expected(s, pool, window=0):
    """(out, tolerance, what is infinite or NaN): columns with such values that a row sees are their sum, the others as if those were 0."""
    keep = s.qkv
    clean = torch.where(torch.isfinite(pool), pool, torch.zeros_like(pool))
    s.qkv = torch.where(torch.isfinite(keep), keep, torch.zeros_like(keep))
    out, tol, _ = tu.reference(s, clean, window=window)
    s.qkv = keep
    odd = torch.zeros_like(out)
    for i, (n, C) in enumerate(zip(s.counts, s.starts)):
        _, W = tu._pages(s, pool, i, C + n)
        W[:, C:] = s.qkv[s.cu[i]:s.cu[i] + n, (s.heads + s.n_kv) * s.dim:].double().view(n, s.n_kv, s.vdim).transpose(0, 1)
        up = tu.lines(s.parents[i])
        depth = torch.tensor([len(a) - 1 for a in up], device=s.device)
        seen = torch.ones((n, C + n), dtype=torch.bool, device=s.device)
        seen[:, C:] = False
        for r, a in enumerate(up):
            seen[r, [C + b for b in a]] = True
        if window:
            seen &= (C + depth)[:, None] - torch.cat([torch.arange(C, device=s.device), C + depth]) < window
        for g in range(s.n_kv):
            has = [(seen.double() @ m.double()) > 0 for m in (W[g].isnan(), W[g] == math.inf, W[g] == -math.inf)]
            x = torch.zeros((n, s.vdim), dtype=torch.float64, device=s.device)
            x[has[1]], x[has[2]] = math.inf, -math.inf
            x[has[0] | has[1] & has[2]] = math.nan
            for h in range(g * s.qpk, (g + 1) * s.qpk):
                odd[s.cu[i]:s.cu[i] + n, h * s.vdim:(h + 1) * s.vdim] = x
    return out, tol, odd


def _values(s, got, want):
    out, tol, odd = want
    got = got.double()
    fine = odd == 0
    assert torch.isfinite(got[fine]).all()
    worst = float(((got - out).abs() / tol)[fine].max())
    assert worst <= 1.0, f"off by {worst:.2f} of the tolerance"
    assert torch.equal(got[~fine].nan_to_num(7.0, 8.0, 9.0), odd[~fine].nan_to_num(7.0, 8.0, 9.0))
    return int((~fine).sum())


KERNELS = [("bf16", False), ("fp16", False), ("bf16", True), ("fp16", True), ("fp32", False)]


@pytest.mark.parametrize("dtype,plain", KERNELS)
@pytest.mark.parametrize("kind", ["tree", "star", "chain"])
def test_infinite_values_of_drafted_tokens_reach_their_columns(cuda, dtype, plain, kind):
    """One column of a token's values, of one head: that column of the rows that see it, and no other."""
    s = tu.batch([30, 9, 60], [200, 70, 0], kind, dtype=DT[dtype], dim=64, n_kv=2, qpk=3, seed=24)
    value = lambda tok, g, c, x: s.qkv[tok, (s.heads + s.n_kv) * 64 + g * 64 + c].fill_(x)
    value(4, 0, 3, math.inf), value(7, 1, 63, math.nan), value(9, 1, 0, -math.inf), value(11, 1, 0, math.inf), value(12, 1, 0, -math.inf)
    value(30, 0, 17, -math.inf), value(39 + 59, 1, 40, math.nan), value(39 + 33, 0, 8, math.inf), value(39 + 33, 0, 9, math.nan)
    before = s.cache.pool.clone()
    want = _expected(s, before)
    assert _values(s, tu.run(s, plain=plain), want) > 0 and s.flag.item() == 0


@pytest.mark.parametrize("dtype,plain", KERNELS)
@pytest.mark.parametrize("window,start", [(100, 300), (70, 64), (129, 256), (5, 40), (300, 128)])
def test_infinite_values_at_the_edge_of_a_window(cuda, dtype, plain, window, start):
    """Cached positions that tokens of small depth still see and deeper ones do not, and keys there that are NaN for nobody."""
    n = 24
    s = tu.batch([n, 3], [start, 20], "tree", dtype=DT[dtype], dim=64, n_kv=2, qpk=2, seed=25)
    edge = start - window + 1
    pool = s.cache.pool
    for at, x in ((edge, math.nan), (edge + 1, math.inf), (edge + 2, -math.inf), (edge + 5, math.inf), (edge + 9, math.nan), (edge - 1, math.nan), (edge - 2, math.inf)):
        if 0 <= at < start:
            page = s.table[s.slot[0]][at // s.page]
            pool[page, 1, 0, at % s.page, (5 * at) % 64] = x
            pool[page, 1, 1, at % s.page, 8 + at % 8] = -x
            if at < edge:
                pool[page, 0, :, at % s.page] = x      # (a key that no row sees)
    before = pool.clone()
    want = _expected(s, before, window)
    assert (_values(s, tu.run(s, window=window, plain=plain), want) > 0) == (edge + 9 >= 0) and s.flag.item() == 0      # (a window over all has no edge)


@pytest.mark.parametrize("dtype,plain", KERNELS)
def test_infinite_values_that_all_rows_see(cuda, dtype, plain):
    """In whole tiles of a short and of a long cache, which several blocks share."""
    s = tu.batch([20, 40], [300, 9000], "tree", dtype=DT[dtype], dim=128, n_kv=2, qpk=4, seed=26)
    s.scale = 0.02                                     # (every weight is a number that fp32 holds)
    for i, at, g, c, x in ((0, 10, 0, 5, math.inf), (0, 100, 0, 5, math.inf), (0, 130, 1, 90, -math.inf), (0, 140, 1, 127, math.nan), (1, 0, 0, 0, math.inf), (1, 8000, 0, 0, -math.inf),
                           (1, 4000, 0, 64, math.inf), (1, 4001, 1, 65, math.nan), (1, 77, 1, 66, -math.inf), (1, 8999, 1, 100, math.inf)):
        s.cache.pool[s.table[s.slot[i]][at // s.page], 1, g, at % s.page, c] = x
    before = s.cache.pool.clone()
    want = _expected(s, before)
    assert _values(s, tu.run(s, plain=plain), want) == 4 * (20 * 3 + 40 * 5) and s.flag.item() == 0


@pytest.mark.parametrize("dtype,plain", KERNELS)
def test_a_bad_query_is_its_own(cuda, dtype, plain):
    """A row whose scores are NaN is NaN everywhere; others keep their bits, infinite values included."""
    s = tu.batch([20, 7], [300, 40], "star", dtype=DT[dtype], dim=64, n_kv=2, qpk=2, seed=27)
    s.qkv[3, (s.heads + s.n_kv) * 64 + 2] = math.inf
    want = tu.run(s, plain=plain).clone()
    s.qkv[5, :s.heads * 64] = math.nan
    got = tu.run(s, plain=plain)
    rows = [r for r in range(27) if r != 5]
    assert torch.equal(got[rows], want[rows]) and got[5].isnan().all()


@pytest.mark.parametrize("dtype,plain", KERNELS)
@pytest.mark.parametrize("window,start", [(0, 120), (300, 120), (300, 400), (600, 400), (40, 1000), (5000, 3000)])
def test_infinite_values_in_cached_and_drafted_positions_meet(cuda, dtype, plain, window, start):
    """The same columns of cached positions that all rows see, in tiles that they see whole and in tiles with drafted tokens, and of drafted tokens."""
    s = tu.batch([24, 5], [start, 9], "tree", dtype=DT[dtype], dim=64, n_kv=1, qpk=2, seed=28)
    s.scale = 0.02
    for back, c, x in ((1, 3, math.inf), (20, 4, -math.inf), (20, 5, math.nan), (60, 6, math.inf), (119, 7, math.inf), (250, 8, math.inf), (399, 9, -math.inf)):
        if back <= start:
            s.cache.pool[s.table[s.slot[0]][(start - back) // s.page], 1, 0, (start - back) % s.page, c] = x
    for tok, c, x in ((2, 3, -math.inf), (5, 4, -math.inf), (9, 6, math.inf), (4, 8, -math.inf), (7, 9, math.inf), (11, 40, math.nan)):
        s.qkv[tok, (s.heads + 1) * 64 + c] = x
    before = s.cache.pool.clone()
    want = _expected(s, before, window)
    assert _values(s, tu.run(s, window=window, plain=plain), want) > 0 and s.flag.item() == 0


def test_a_long_cache_of_infinite_values_ends_in_time(cuda):
    """Every column of every row looks at every key again: no wait runs out meanwhile."""
    s = tu.batch([40], [200000], "chain", dtype=torch.bfloat16, dim=128, n_kv=8, qpk=4, seed=29)
    s.cache.pool[:, 1, :, 5] = math.inf
    out = tu.run(s)
    assert s.flag.item() == 0 and (out == math.inf).all()
