"""Caches of eight bits: batches, and the operators' formulas in 64 bits."""
import math
from types import SimpleNamespace

import torch

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "int8": torch.int8, "e4m3": torch.float8_e4m3fn}
TOP = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def ints(v, device="cuda"):
    return torch.tensor(v, dtype=torch.int32, device=device)


def batch(counts, starts, dtype=torch.bfloat16, fmt=torch.int8, n_kv=2, qpk=4, dim=64, vdim=None, page=64, rot=0, seed=0, spare_rows=0, slots=None, max_len=None, base_page=0, extra=3,
          device="cuda", pad=0):
    """Rows [q | k | v] of the new tokens, a cache whose pages hold bytes and scales of earlier ones and, everywhere else, scales that are NaN."""
    from poptransformer_b200 import ops
    gen = torch.Generator().manual_seed(seed)
    s = SimpleNamespace(counts=counts, starts=starts, dtype=dtype, fmt=fmt, n_kv=n_kv, heads=n_kv * qpk, dim=dim, vdim=dim if vdim is None else vdim, page=page, rot=rot, device=device)
    n_seq = len(counts)
    s.max_len = max_len or max(1, max(a + n for a, n in zip(starts, counts)))
    need = [-(-min(a + n, s.max_len) // page) for a, n in zip(starts, counts)]
    max_pages = -(-s.max_len // page)
    n_pages = base_page + sum(need) + extra
    order = (torch.randperm(sum(need) + extra, generator=gen) + base_page).tolist()
    slots = n_seq if slots is None else slots
    slot = torch.randperm(slots, generator=gen)[:n_seq].tolist()
    table, at = [[0] * max_pages for _ in range(slots)], 0
    for i, n in enumerate(need):
        table[slot[i]][:n] = order[at:at + n]
        at += n
    s.cu_host = [sum(counts[:i]) for i in range(n_seq + 1)]
    s.n_tok = s.cu_host[-1]
    s.table_host, s.slot_host = table, slot
    s.cu, s.start, s.slot, s.page_table = ints(s.cu_host, device), ints(starts, device), ints(slot, device), ints(table, device)
    s.tok_seq = ints([i for i, n in enumerate(counts) for _ in range(n)] + [0] * spare_rows, device)
    s.view = ops.batch_view(n_seq, s.n_tok + spare_rows, s.cu, s.start, s.slot, s.tok_seq) if device == "cuda" else None
    s.flag = ints([0], device)
    s.q_cols, s.width = s.heads * dim, s.heads * dim + n_kv * (dim + s.vdim)
    s.ld = s.width + pad
    s.qkv = torch.randn((s.n_tok + spare_rows, s.ld), generator=gen)
    s.qkv[:, s.q_cols + 1::19] *= 5.0
    s.qkv = s.qkv.to(dtype).to(device)
    s.scale = dim ** -0.5
    s.rope = ops.rope_table(s.max_len, rot, device=device) if rot else None
    # bytes that read as numbers everywhere; scales that do at the positions that are cached
    elements = n_kv * page * (dim + s.vdim)
    if n_pages * elements < 1 << 26:
        raw = (torch.randn((n_pages, elements), generator=gen) * (TOP[fmt] / 3)).clamp(-TOP[fmt], TOP[fmt])
        s.pool = (raw.round() if fmt == torch.int8 else raw).to(fmt).to(device)
        s.scales = torch.full((n_pages, 2, n_kv, page), math.nan, device=device)
    else:
        s.pool = torch.zeros((n_pages, elements), dtype=torch.int8, device=device).random_(-120, 120).view(fmt)
        s.scales = torch.full((n_pages, 2, n_kv, page), math.nan, device=device)
    for i in range(n_seq):
        for p in range(-(-min(starts[i], s.max_len) // page)):
            rows = min(page, starts[i] - p * page)
            s.scales[table[slot[i]][p], :, :, :rows] = (torch.exp(0.5 * torch.randn((2, n_kv, rows), generator=gen)) * 3.0 / TOP[fmt]).to(device)
    s.cache = ops.PagedKVCache(slots, n_kv, dim, s.max_len, page, device, s.page_table, v_dim=s.vdim, dtype=fmt, pool=s.pool, scales=s.scales)
    return s


def rotate(x, rope, pos, rot, interleaved, inverse=False):
    """x [rows, heads, dim] with the type of x: three roundings, as written."""
    if not rot:
        return x
    cs = rope[pos.long()].to(x.dtype)[:, None]
    c, n = cs[..., 0], -cs[..., 1] if inverse else cs[..., 1]
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    y = x.clone()
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * n, x[..., b] * c + x[..., a] * n
    return y


def to_bytes(x, fmt):
    """fp32 rows -> (bytes, scales), rounded as appending rounds."""
    m = x.abs().amax(-1)
    fine = m <= 2.0 ** 64
    m = torch.where(fine, m, 1.0).clamp(min=2.0 ** -64)
    top = torch.full_like(m, TOP[fmt])
    y = torch.where(fine[..., None], x, 0.0) * torch.div(top, m)[..., None]
    y = y.round().clamp(-127, 127) if fmt == torch.int8 else y
    return y.to(fmt), torch.where(fine, torch.div(m, top), math.nan)


def part(s, pool, page, which):
    """K (0) or V (1) of pages, as [.., n_kv, page, width] of the pool's type."""
    k = s.n_kv * s.page * s.dim
    flat = pool[page]
    return flat[..., :k].unflatten(-1, (s.n_kv, s.page, s.dim)) if which == 0 else flat[..., k:].unflatten(-1, (s.n_kv, s.page, s.vdim))


def appended(s, interleaved=False):
    """What appending leaves (pool, scales) and the rotated queries in 32 bits, computed on the CPU."""
    pool, scales = s.pool.cpu().view(torch.uint8).clone(), s.scales.cpu().clone()
    qkv, rope = s.qkv.cpu().float(), None if s.rope is None else s.rope.cpu()
    q_out = torch.zeros((s.qkv.shape[0], s.q_cols))
    for i, n in enumerate(s.counts):
        if not n or s.starts[i] + n > s.max_len:
            continue
        x = qkv[s.cu_host[i]:s.cu_host[i] + n]
        pos = torch.arange(s.starts[i], s.starts[i] + n)
        q_out[s.cu_host[i]:s.cu_host[i] + n] = rotate(x[:, :s.q_cols].reshape(n, -1, s.dim), rope, pos, s.rot, interleaved).flatten(1)
        k = rotate(x[:, s.q_cols:s.q_cols + s.n_kv * s.dim].reshape(n, -1, s.dim), rope, pos, s.rot, interleaved)
        v = x[:, s.q_cols + s.n_kv * s.dim:s.width].reshape(n, -1, s.vdim)
        for which, y in ((0, k), (1, v)):
            by, sc = to_bytes(y, s.fmt)
            for r in range(n):
                page, place = s.table_host[s.slot_host[i]][int(pos[r]) // s.page], int(pos[r]) % s.page
                part(s, pool, page, which)[:, place] = by[r].view(torch.uint8)
                scales[page, which, :, place] = sc[r]
    return pool, scales, q_out


def history(s, i, n, which):
    """The first n positions of sequence i in 64 bits: [n_kv, n, width]."""
    pages = ints(s.table_host[s.slot_host[i]], s.device).long()[:-(-n // s.page)]
    x = part(s, s.pool, pages, which)
    x = x.to(torch.float32).double() * s.scales[pages, which][..., None].double()
    return x.transpose(0, 1).flatten(1, 2)[:, :n]


def reference(s, q, window=0, softcap=0.0):
    """(outputs, how far a kernel's may be off) in 64 bits, [n_tok, heads, vdim].

    A score is a sum of dim products in 32 bits, each exact but for the query (kept to 2^-22 of its row's largest element, or exactly), times two factors: off by at most
    e = (dim + 8) 2^-24 sum |q_i k_i| scale, and with a softcap a few units of its result more.  exp and its argument in powers of two add 2^-20 at scores below 2^10 (their own
    rounding is in e).  A weight is rounded once, to fp16 (half a step: 2^-11) for rows of bf16 and to two fp16 parts (2^-21) for others, and below 2^-29 of the largest it is off by 2^-40 of
    that.  The sums of the weighted values are sums in 32 bits of n terms in runs, 2^-22 of the sum of magnitudes.  So an output is off by at most
    (2 e + 2^-20 + weight) sum p |v| + n 2^-40 max |v|, and half a step of its type."""
    H, G = s.heads, s.n_kv
    out = torch.zeros((s.n_tok, H, s.vdim), dtype=torch.float64, device=s.device)
    tol = torch.zeros_like(out)
    weight = 2.0 ** -11 if s.dtype == torch.bfloat16 else 2.0 ** -21
    half = torch.finfo(s.dtype).eps / 2
    for i, n in enumerate(s.counts):
        if not n:
            continue
        K, V = history(s, i, s.starts[i] + n, 0), history(s, i, s.starts[i] + n, 1)
        for r in range(n):
            pos = s.starts[i] + r
            first = max(0, pos - window + 1) if window else 0
            x = q[s.cu_host[i] + r, :H * s.dim].double().view(G, H // G, s.dim)
            k, v = K[:, first:pos + 1], V[:, first:pos + 1]
            z = x @ k.transpose(1, 2) * s.scale
            most = (x.abs() @ k.abs().transpose(1, 2) * abs(s.scale)).amax(-1, keepdim=True)
            e = (s.dim + 8) * 2.0 ** -24 * most
            if softcap:
                z = softcap * torch.tanh(z / softcap)
                e = e + softcap * 2.0 ** -21
            p = torch.softmax(z, -1)
            o = p @ v
            t = (2 * e + 2.0 ** -20 + weight) * (p @ v.abs()) + (pos + 1 - first) * 2.0 ** -40 * v.abs().amax(1, keepdim=True) + half * o.abs()
            if s.dtype == torch.float16:
                t = t + 2.0 ** -25          # half a step of the smallest fp16 numbers
            out[s.cu_host[i] + r], tol[s.cu_host[i] + r] = o.reshape(H, -1), t.reshape(H, -1)
    return out, tol


def attend(s, q, window=0, softcap=0.0, out=None, plain=False, workspace=None):
    from poptransformer_b200 import ops
    n = s.view.n_tok
    out = torch.empty((n, s.heads * s.vdim), dtype=s.dtype, device=s.device) if out is None else out
    if workspace is None and not plain:
        workspace = ops.kv8_attn_workspace(n, s.heads, s.n_kv, max(s.dim, s.vdim), s.device)
    return ops.kv8_attn(s.view, q, q.shape[1], s.cache, out, out.shape[1], s.heads, s.scale, window=window, softcap=softcap, workspace=workspace, error_flag=s.flag, plain=plain)


def check(s, q, out, window=0, softcap=0.0):
    want, tol = reference(s, q, window, softcap)
    got = out[:s.n_tok, :s.heads * s.vdim].double().view(s.n_tok, s.heads, s.vdim)
    off = (got - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:5].tolist(), off[bad][:5].tolist(), tol[bad][:5].tolist(), got[bad][:5].tolist(), want[bad][:5].tolist())


def cached(s):
    """A batch whose new tokens are in the cache already (their scales numbers): what attention finds."""
    for i, n in enumerate(s.counts):
        for p in range(s.starts[i], s.starts[i] + n):
            page = s.table_host[s.slot_host[i]][p // s.page]
            s.scales[page, :, :, p % s.page] = 3.0 / TOP[s.fmt]
    return s
