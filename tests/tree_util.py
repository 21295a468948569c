"""Trees of drafted tokens over a paged cache, and their attention in 64 bits with what a kernel may be off by."""
import math
import random
from types import SimpleNamespace

import torch


def tree(n, kind, rng):
    if n == 0:
        return []
    if kind == "chain":
        return [-1] + list(range(n - 1))
    if kind == "star":
        return [-1] + [0] * (n - 1)
    if kind == "roots":
        return [-1] * n
    return [-1] + [rng.randint(max(-1, i - 5), i - 1) for i in range(1, n)]


def lines(parent):
    out = []
    for i, p in enumerate(parent):
        out.append((out[p] if p >= 0 else []) + [i])
    return out


def batch(counts, starts, kind="tree", n_kv=2, qpk=2, dim=64, vdim=None, dtype=torch.bfloat16, page=64, seed=0, rot=0, spare_rows=0, device="cuda", slots=None, max_len=None):
    """Inputs of tree_attn with pages in any order; the new rows' pages hold something else before."""
    from poptransformer_b200 import ops
    rng, g = random.Random(seed), torch.Generator(device="cpu").manual_seed(seed)
    vdim = dim if vdim is None else vdim
    s = SimpleNamespace(counts=counts, starts=starts, n_kv=n_kv, qpk=qpk, dim=dim, vdim=vdim, dtype=dtype, page=page, rot=rot, device=device, heads=n_kv * qpk)
    s.parents = [tree(n, kind, rng) for n in counts]
    s.cu = [sum(counts[:i]) for i in range(len(counts) + 1)]
    s.max_len = max_len or max([a + n for a, n in zip(starts, counts)] + [1])
    max_pages = -(-s.max_len // page)
    need = [-(-(a + n) // page) for a, n in zip(starts, counts)]
    pages = list(range(sum(need) + 1))
    rng.shuffle(pages)
    n_slots = len(counts) if slots is None else slots
    s.slot = rng.sample(range(n_slots), len(counts))
    table = [[0] * max_pages for _ in range(n_slots)]
    for i, k in enumerate(need):
        table[s.slot[i]][:k] = pages[sum(need[:i]):sum(need[:i]) + k]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=device)
    s.n_tok = s.cu[-1]
    s.table = table
    s.ld = s.heads * dim + n_kv * (dim + vdim)
    rand = lambda *shape: torch.randn(shape, generator=g).to(dtype)
    s.qkv = rand(s.n_tok + spare_rows, s.ld).to(device)
    page_table = i32(table)
    pool = rand(len(pages), n_kv * page * (dim + vdim)).to(device)
    if vdim == dim:
        pool = pool.view(len(pages), 2, n_kv, page, dim)
    s.cache = ops.PagedKVCache(n_slots, n_kv, dim, s.max_len, page, device, page_table, v_dim=vdim, dtype=dtype, pool=pool)
    s.rope = None
    if rot:
        a = torch.arange(s.max_len, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(rot // 2, dtype=torch.float64) * 2 / rot)
        s.rope = torch.stack([a.cos(), a.sin()], -1).float().to(device)
    s.parent = i32([p for q in s.parents for p in q] + [0] * spare_rows)
    s.cu_d, s.start_d, s.slot_d = i32(s.cu), i32(starts), i32(s.slot)
    s.tok_seq = i32([i for i, n in enumerate(counts) for _ in range(n)] + [0] * spare_rows)
    s.view = ops.batch_view(len(counts), s.n_tok + spare_rows, s.cu_d, s.start_d, s.slot_d, s.tok_seq)
    s.scale = dim ** -0.5
    s.flag = torch.zeros(1, dtype=torch.int32, device=device)
    return s


def run(s, out=None, out_ld=None, parent="tree", workspace=None, most=None, **kw):
    from poptransformer_b200 import ops
    if out is None:
        out_ld = s.heads * s.vdim
        out = torch.full((s.qkv.shape[0], out_ld), 7.0, dtype=s.dtype, device=s.device)
    most = max(s.counts) if most is None else most
    if workspace is None:
        workspace = ops.tree_attn_workspace(len(s.counts), most, s.heads, s.n_kv, s.vdim, s.device)
    ops.tree_attn(s.view, s.qkv, s.ld, s.cache, out, out_ld, s.heads, s.scale, s.parent if parent == "tree" else parent, rope=s.rope, rope_dims=s.rot, max_tokens_per_seq=most,
                  workspace=workspace, error_flag=s.flag, **kw)
    return out


def _pages(s, pool, i, upto):
    """K and V [n_kv, positions, ..] of a sequence from a pool, in 64 bits."""
    flat = pool.reshape(pool.shape[0], -1)
    rows = flat[s.table[s.slot[i]][:-(-upto // s.page)]].double()
    cut = s.n_kv * s.page * s.dim
    k = rows[:, :cut].view(-1, s.n_kv, s.page, s.dim).transpose(0, 1).flatten(1, 2)[:, :upto]
    v = rows[:, cut:].view(-1, s.n_kv, s.page, s.vdim).transpose(0, 1).flatten(1, 2)[:, :upto]
    return k.clone(), v.clone()


def turned(s, x, pos):
    h = s.rot // 2
    if not h:
        return x
    a = s.rope[pos].double()[:, None]
    u, v = x[..., :h], x[..., h:2 * h]
    return torch.cat([u * a[..., 0] - v * a[..., 1], v * a[..., 0] + u * a[..., 1], x[..., 2 * h:]], -1)


def reference(s, pool, window=0, softcap=0.0, chain=False):
    """(out, tolerance), and the new rows' keys and values per sequence.  pool: before the call.

    With t = eps / 2 of the type, a kernel rounds the output (t), rotated keys (t: where its fp32 rotation lies on the other side of a border, a
    whole step 2 t) and may round rotated queries (t); all else is fp32 or better: products and sums of dim terms are off by dim 2^-23 of the sum of
    their sizes, and rotation by 2^-22.  A score that is off by e changes a weight by a factor within exp(+-2 e); a weight itself may lose 2^-15 (its
    exponential and two 8-bit parts), sums over T positions T 2^-24."""
    n_out = s.heads * s.vdim
    half = torch.finfo(s.dtype).eps / 2
    out = torch.full((s.n_tok, n_out), math.nan, dtype=torch.float64, device=s.device)
    tol = torch.zeros_like(out)
    new = []
    for i, (n, C) in enumerate(zip(s.counts, s.starts)):
        if n == 0:
            new.append(None)
            continue
        parent = [r - 1 for r in range(n)] if chain else s.parents[i]
        up = lines(parent)
        depth = torch.tensor([len(a) - 1 for a in up], device=s.device)
        x = s.qkv[s.cu[i]:s.cu[i] + n].double()
        H, G, D, V = s.heads, s.n_kv, s.dim, s.vdim
        q = turned(s, x[:, :H * D].view(n, H, D), C + depth)
        k = turned(s, x[:, H * D:(H + G) * D].view(n, G, D), C + depth)
        v = x[:, (H + G) * D:].view(n, G, V)
        K, W = _pages(s, pool, i, C + n)
        K[:, C:], W[:, C:] = k.to(s.dtype).double().transpose(0, 1), v.transpose(0, 1)
        new.append((k, v))
        seen = torch.zeros((n, C + n), dtype=torch.bool, device=s.device)
        where = torch.cat([torch.arange(C, device=s.device), C + depth])
        seen[:, :C] = True
        for r, a in enumerate(up):
            seen[r, [C + b for b in a]] = True
        if window:
            seen &= (C + depth)[:, None] - where < window
        rel = D * 2.0 ** -23 + (3 * half + 2.0 ** -21 if s.rot else 0.0)
        for g in range(G):
            Wg = torch.where(seen.any(0)[:, None], W[g], 0.0)      # (never seen: whatever it is)
            for h in range(g * s.qpk, (g + 1) * s.qpk):
                z = q[:, h] @ K[g].T * s.scale
                off = (q[:, h].abs() @ K[g].abs().T * s.scale).masked_fill(~seen, 0.0).nan_to_num(0.0).amax(1, keepdim=True) * rel
                if softcap:
                    z = softcap * torch.tanh(z / softcap)
                    off = off + softcap * 2.0 ** -21
                w = torch.softmax(z.masked_fill(~seen, -math.inf), -1)
                o = w @ Wg
                out[s.cu[i]:s.cu[i] + n, h * V:(h + 1) * V] = o
                slack = torch.expm1(2 * off) + 2.0 ** -14 + (C + n) * 2.0 ** -23
                tol[s.cu[i]:s.cu[i] + n, h * V:(h + 1) * V] = half * o.abs() + (1 + half) * slack * (w @ Wg.abs()) + torch.finfo(s.dtype).tiny
    return out, tol, new


def check(s, pool, out, window=0, softcap=0.0, chain=False):
    ref, tol, new = reference(s, pool, window, softcap, chain)
    got = out[:s.n_tok, :s.heads * s.vdim].double()
    assert torch.isfinite(got).all()
    worst = ((got - ref).abs() / tol).max()
    assert worst <= 1.0, f"off by {worst:.2f} of the tolerance"
    half = torch.finfo(s.dtype).eps / 2
    for i, x in enumerate(new):
        if x is None:
            continue
        K, V = _pages(s, s.cache.pool, i, s.starts[i] + s.counts[i])
        k, v = x[0].transpose(0, 1), x[1].transpose(0, 1)
        assert torch.equal(V[:, s.starts[i]:], v)
        # (rotated in fp32: 2^-22 of both terms, then rounded)
        size = (k.abs().amax(-1, keepdim=True) * 2.0 ** -20) if s.rot else 0.0
        assert ((K[:, s.starts[i]:] - k).abs() <= half * (k.abs() + size) + size).all()
        before_k, before_v = _pages(s, pool, i, s.starts[i] + s.counts[i])
        assert torch.equal(K[:, :s.starts[i]].nan_to_num(9.0), before_k[:, :s.starts[i]].nan_to_num(9.0)) and torch.equal(V[:, :s.starts[i]].nan_to_num(9.0), before_v[:, :s.starts[i]].nan_to_num(9.0))
