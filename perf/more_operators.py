"""Operators of decoding over caches of eight bits, as cases that can be timed and compared.

Keys and values are kept as bytes, int8 or E4M3, with one scale for every position and head: half of what 16 bits take of the memory, and of
the time that a decode step reads its history in.  Four operators go with them: the rotation of queries and keys by their positions (both layouts of the pairs, part of a
head), appending keys and values on the way through rotation and rounding, attention of one new token a sequence over what is cached, and
pages turned back into the rows' type for whatever reads those.

`run` computes each of them in elementary torch operations, or (own) through the framework.  `exact` computes the same in 64 bits, one
sequence after the other."""
import math
import random
from types import SimpleNamespace

import torch

own = False

PAGE = 64            # positions of a cache page, as the decoders have it by default
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "int8": torch.int8, "e4m3": torch.float8_e4m3fn}
TOP = {"int8": 127.0, "e4m3": 448.0}              # the largest byte of a row
SMALL, LARGE = 2.0 ** -64, 2.0 ** 64              # a row's scale goes by its largest magnitude, this at least; a row beyond the other reads back as NaN


def listed():
    return [
        # ---- rotation
        # One user's new token: queries and keys of a multi-head model, latency.
        dict(name="rotate one token", op="rotary", type="fp16", rows=1, heads=64, dim=128, rot=128, interleaved=False, inverse=False, table=2048),
        # A prompt through a model that rotates neighbouring pairs in half of a head; two of its heads are keys.
        dict(name="rotate prompt", op="rotary", type="bf16", rows=4000, heads=34, dim=128, rot=64, interleaved=True, inverse=False, table=32768),
        # ---- appending
        # One user's new token, multi-head attention with 32 heads.
        dict(name="append one token", op="append", type="fp16", cache="int8", seqs=1, rows=1, heads=32, kv_heads=32, dim=128, rot=128, interleaved=False, context=700),
        # A step of a served batch.
        dict(name="append 48 tokens", op="append", type="bf16", cache="e4m3", seqs=48, rows=1, heads=32, kv_heads=8, dim=128, rot=128, interleaved=False, context=4000),
        # Prompts of unequal lengths behind a cached beginning.
        dict(name="append prompts", op="append", type="bf16", cache="int8", seqs=5, rows=3001, heads=32, kv_heads=8, dim=128, rot=128, interleaved=False, context=500),
        # ---- attention of new tokens
        # One user, a short chat: latency.
        dict(name="attn one sequence", op="attn", type="fp16", cache="int8", seqs=1, heads=32, kv_heads=8, dim=128, context=700, window=0, cap=0.0),
        # Two key/value heads for 32 query heads, a small batch.
        dict(name="attn two kv heads", op="attn", type="fp16", cache="int8", seqs=8, heads=32, kv_heads=2, dim=128, context=1151, window=0, cap=0.0),
        # True 32-bit model, sliding window and softcap, an odd head width, a ragged batch.
        dict(name="attn fp32 window", op="attn", type="fp32", cache="e4m3", seqs=7, heads=12, kv_heads=4, dim=80, context=2500, window=1500, cap=30.0),
        # A large served batch of unequal lengths: the ordinary case of a busy server.
        dict(name="attn 48 sequences", op="attn", type="bf16", cache="int8", seqs=48, heads=32, kv_heads=8, dim=128, context=8000, window=0, cap=0.0),
        # Two long documents.
        dict(name="attn long context", op="attn", type="bf16", cache="e4m3", seqs=2, heads=32, kv_heads=8, dim=128, context=100000, window=0, cap=0.0),
        # ---- pages back into the rows' type, for a prompt's attention
        # The cached beginning of one sequence.
        dict(name="unpack one sequence", op="unpack", type="bf16", cache="int8", seqs=1, rows=200, kv_heads=8, dim=128, context=700),
        # Long beginnings of a batch.
        dict(name="unpack long", op="unpack", type="fp16", cache="e4m3", seqs=4, rows=500, kv_heads=8, dim=128, context=16000),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["attn", "attn", "attn", "append", "append", "rotary", "unpack"])
    kind, cache, dim = rng.choice(["bf16", "bf16", "fp16", "fp32"]), rng.choice(["int8", "int8", "e4m3"]), rng.choice([64, 128, 128, 128, 80, 96, 256])
    kv = rng.choice([1, 2, 4, 8, 12])
    heads = kv * rng.choice([f for f in (1, 2, 3, 4, 8, 16) if kv * f <= 48])
    rot = rng.choice([dim, dim, dim // 2, dim // 4, 0])
    if op == "rotary":
        rows = log(1, 8000)
        while rows * heads * dim > 30000000:
            rows = max(1, rows // 2)
        return dict(op="rotary", type=kind, rows=rows, heads=heads, dim=dim, rot=rot or dim, interleaved=rng.random() < 0.4, inverse=rng.random() < 0.3, table=log(100, 100000))
    if op == "append":
        c = dict(op="append", type=kind, cache=cache, seqs=log(1, 64), rows=log(1, 4000) if rng.random() < 0.6 else 1, heads=heads, kv_heads=kv, dim=dim, rot=rot,
                 interleaved=rng.random() < 0.4, context=log(1, 4000))
        while c["seqs"] * c["rows"] * (heads + 2 * kv) * dim > 60000000:
            c["seqs"], c["rows"] = max(1, c["seqs"] // 2), max(1, c["rows"] * 3 // 4)
        return c
    if op == "unpack":
        c = dict(op="unpack", type=kind, cache=cache, seqs=log(1, 24), rows=log(1, 1000), kv_heads=kv, dim=dim, context=log(1, 20000))
        while c["seqs"] * (c["context"] + c["rows"]) * kv * dim > 50000000:
            c["seqs"], c["context"], c["rows"] = max(1, c["seqs"] // 2), c["context"] * 3 // 4, max(1, c["rows"] * 3 // 4)
        return c
    c = dict(op="attn", type=kind, cache=cache, seqs=log(1, 64), heads=heads, kv_heads=kv, dim=dim, context=log(1, 40000), window=0, cap=0.0)
    if rng.random() < 0.25:
        c["window"] = log(8, 4000)
    if rng.random() < 0.2:
        c["cap"] = float(rng.randint(10, 50))
    while c["seqs"] * c["context"] * max(kv * dim, heads * 4) > 200000000:
        c["seqs"], c["context"] = max(1, c["seqs"] // 2), c["context"] * 3 // 4
    return c


# ------------------------------------------------------------------------------------------ sizes that follow from a case alone
def lengths(case):
    """Cached positions of every sequence: the longest has all of the context."""
    rng = random.Random(7 * case["context"] + case["seqs"])
    return [case["context"]] + [max(0, int(case["context"] * rng.uniform(0.3, 1.0))) for _ in range(case["seqs"] - 1)]


def row_counts(case):
    """New rows of every sequence: the first has all of them."""
    most = case.get("rows", 1)
    rng = random.Random(11 * most + case["seqs"])
    return [most] + [max(1, int(most * rng.uniform(0.4, 1.0))) for _ in range(case["seqs"] - 1)]


def work(case):
    es, D = TYPES[case["type"]].itemsize, case["dim"]
    if case["op"] == "rotary":
        n = case["rows"] * case["heads"]
        return dict(bytes=2 * es * n * D + 4 * case["rows"] * (case["rot"] + 1), flops=3 * n * case["rot"])
    G, row = case["kv_heads"], 2 * case["kv_heads"] * (D + 4)                # the bytes of a cached position with its scales
    if case["op"] == "append":
        n = sum(row_counts(case))
        return dict(bytes=n * (2 * (case["heads"] + G) * D * es + row + 4 * case["rot"]), flops=n * D * (3 * case["heads"] + 7 * G))
    if case["op"] == "attn":
        seen = [min(a + 1, case["window"] or a + 1) for a in lengths(case)]
        return dict(bytes=sum(seen) * row + 2 * case["seqs"] * case["heads"] * D * es, flops=4 * sum(seen) * case["heads"] * D)
    n = sum(a + b for a, b in zip(lengths(case), row_counts(case)))
    return dict(bytes=n * (row + 2 * G * D * es), flops=2 * n * G * D)


# ------------------------------------------------------------------------------------------ inputs
def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return globals()["prepare_" + case["op"]](SimpleNamespace(**case), case, gen, random.Random(seed))


def angles(positions, rot):
    """(cos, sin) of every position and pair, from angles in 64 bits."""
    a = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(rot // 2, device="cuda", dtype=torch.float64) * 2 / max(1, rot))
    return torch.stack([a.cos(), a.sin()], -1).float().contiguous()


def normal(gen, dt, *shape):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32 if dt == torch.float32 else torch.bfloat16).to(dt)


def paged(s, case, rng):
    """The batch, and pages of every sequence in any order with a table that has a row per slot; sequences sit in slots of their own."""
    s.counts, s.start_host = row_counts(case), lengths(case)
    s.n_tok, s.most = sum(s.counts), max(s.counts)
    s.cu_host = [sum(s.counts[:i]) for i in range(s.seqs + 1)]
    s.max_len = max(a + n for a, n in zip(s.start_host, s.counts))
    s.max_pages = -(-s.max_len // PAGE)
    need = [-(-(a + n) // PAGE) for a, n in zip(s.start_host, s.counts)]
    s.n_pages = sum(need) + 2
    order = list(range(s.n_pages))
    rng.shuffle(order)
    s.slot_host = list(range(s.seqs))
    rng.shuffle(s.slot_host)
    table, at = [[0] * s.max_pages for _ in range(s.seqs)], 0
    for i, n in enumerate(need):
        table[s.slot_host[i]][:n] = order[at:at + n]
        at += n
    s.cu, s.start, s.slot, s.page_table = ints(s.cu_host), ints(s.start_host), ints(s.slot_host), ints(table)
    s.tok_seq = ints([i for i, n in enumerate(s.counts) for _ in range(n)])
    s.row_of = torch.arange(s.n_tok, device="cuda") - s.cu[s.tok_seq.long()]
    if own:
        from poptransformer_b200 import ops
        s.view, s.flag = ops.batch_view(s.seqs, s.n_tok, s.cu, s.start, s.slot, s.tok_seq), ints([0])


def filled(s, gen):
    """A pool as appending leaves it: bytes whose largest of a row is near the top, scales that differ from position to position."""
    shape = (s.n_pages, 2, s.kv_heads, PAGE, s.dim)
    x = torch.randn(shape, generator=gen, device="cuda", dtype=torch.bfloat16) * (TOP[s.cache] / 3.5)
    s.pool = x.clamp_(-TOP[s.cache], TOP[s.cache]).to(TYPES[s.cache])
    s.scales = torch.exp(0.4 * torch.randn(shape[:4], generator=gen, device="cuda")) * (3.5 / TOP[s.cache])


def cache_of(s):
    from poptransformer_b200 import ops
    return ops.PagedKVCache(s.seqs, s.kv_heads, s.dim, s.max_len, PAGE, "cuda", s.page_table, dtype=s.pool.dtype, pool=s.pool, scales=s.scales)


def prepare_rotary(s, case, gen, rng):
    s.x = normal(gen, TYPES[s.type], s.rows, s.heads * s.dim)
    first = rng.randint(0, max(0, s.table - s.rows))
    s.positions = ((first + torch.arange(s.rows, device="cuda")) % s.table).int()
    s.rope = angles(s.table, s.rot)
    s.out = torch.empty_like(s.x)
    return s


def prepare_append(s, case, gen, rng):
    paged(s, case, rng)
    G, H, D = s.kv_heads, s.heads, s.dim
    s.ld = (H + 2 * G) * D
    s.qkv = normal(gen, TYPES[s.type], s.n_tok, s.ld)
    s.qkv[:, H * D + 3::37] *= 6.0                                     # keys and values have columns that are always large
    s.rope = angles(s.max_len, s.rot) if s.rot else None
    s.q_out = torch.empty((s.n_tok, H * D), dtype=s.qkv.dtype, device="cuda")
    filled(s, gen)
    if own:
        s.kv = cache_of(s)
    return s


def prepare_attn(s, case, gen, rng):
    paged(s, case, rng)
    s.scale = s.dim ** -0.5
    s.q = normal(gen, TYPES[s.type], s.seqs, s.heads * s.dim) * 1.5
    filled(s, gen)
    s.out = torch.empty_like(s.q)
    if own:
        from poptransformer_b200 import ops
        s.kv = cache_of(s)
        s.workspace = ops.kv8_attn_workspace(s.n_tok, s.heads, s.kv_heads, s.dim, "cuda")
    return s


def prepare_unpack(s, case, gen, rng):
    paged(s, case, rng)
    filled(s, gen)
    s.into = torch.zeros(s.pool.shape, dtype=TYPES[s.type], device="cuda")
    if own:
        from poptransformer_b200 import ops
        s.kv = cache_of(s)
        s.plain_kv = ops.PagedKVCache(s.seqs, s.kv_heads, s.dim, s.max_len, PAGE, "cuda", s.page_table, dtype=s.into.dtype, pool=s.into)
    return s


# ------------------------------------------------------------------------------------------ one pass
def run(state):
    if own:
        return globals()["own_" + state.op](state)
    return globals()["plain_" + state.op](state)


def own_rotary(s):
    from poptransformer_b200 import ops
    return ops.rotary(s.x, s.heads, s.dim, s.rope, s.positions, out=s.out, rope_dims=s.rot, interleaved=s.interleaved, inverse=s.inverse)


def own_append(s):
    from poptransformer_b200 import ops
    ops.kv8_append(s.view, s.qkv, s.ld, s.kv, s.heads, rope=s.rope, rope_dims=s.rot, interleaved=s.interleaved, q_out=s.q_out, q_out_ld=s.heads * s.dim, error_flag=s.flag)
    return s.q_out, s.pool, s.scales


def own_attn(s):
    from poptransformer_b200 import ops
    return ops.kv8_attn(s.view, s.q, s.q.shape[1], s.kv, s.out, s.out.shape[1], s.heads, s.scale, window=s.window, softcap=s.cap, workspace=s.workspace, error_flag=s.flag)


def own_unpack(s):
    from poptransformer_b200 import ops
    ops.kv8_unpack(s.view, s.kv, s.plain_kv, error_flag=s.flag)
    return s.into


def rotate(x, rope, position, rot, interleaved, inverse=False):
    """x [.., heads, dim], position [..]: of the first `rot` dimensions the pairs (i, i + rot / 2), or (2 i, 2 i + 1), turn."""
    if not rot:
        return x
    c, n = rope[position.long()][..., None, :, 0], rope[position.long()][..., None, :, 1]
    if inverse:
        n = -n
    if interleaved:
        u, v = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack([u * c - v * n, v * c + u * n], -1).flatten(-2)
    else:
        u, v = x[..., :rot // 2], x[..., rot // 2:rot]
        turned = torch.cat([u * c - v * n, v * c + u * n], -1)
    return torch.cat([turned, x[..., rot:]], -1)


def plain_rotary(s):
    x = s.x.float().unflatten(-1, (s.heads, s.dim))
    s.out.copy_(rotate(x, s.rope, s.positions, s.rot, s.interleaved, s.inverse).flatten(1))
    return s.out


def to_bytes(x, kind):
    """Rows as bytes and the scale of each: the largest magnitude becomes the largest byte."""
    most = x.abs().amax(-1)
    fine = most <= LARGE
    most = torch.where(fine, most, 1.0).clamp(min=SMALL)
    top = torch.full_like(most, TOP[kind])
    y = torch.where(fine[..., None], x, 0.0) * torch.div(top, most)[..., None]
    if kind == "int8":
        y = y.round().clamp(-127, 127)
    return y.to(TYPES[kind]), torch.where(fine, torch.div(most, top), math.nan)


def plain_append(s):
    G, H, D = s.kv_heads, s.heads, s.dim
    x = s.qkv.float().unflatten(-1, (H + 2 * G, D))
    position = s.start[s.tok_seq.long()].long() + s.row_of
    qk = rotate(x[:, :H + G], s.rope, position, s.rot, s.interleaved)
    s.q_out.copy_(qk[:, :H].flatten(1))
    page, place = s.page_table[s.slot[s.tok_seq.long()].long(), position // PAGE].long(), position % PAGE
    pool = s.pool.view(torch.uint8)
    k, ks = to_bytes(qk[:, H:], s.cache)
    v, vs = to_bytes(x[:, H + G:], s.cache)
    pool[page, 0, :, place], s.scales[page, 0, :, place] = k.view(torch.uint8), ks
    pool[page, 1, :, place], s.scales[page, 1, :, place] = v.view(torch.uint8), vs
    return s.q_out, s.pool, s.scales


def plain_attn(s):
    G, H, D = s.kv_heads, s.heads, s.dim
    j = torch.arange(s.max_len, device="cuda")
    page = s.page_table[s.slot.long()].long()[:, j // PAGE]
    seen = j <= s.start[:, None]
    if s.window:
        seen = seen & (j > s.start[:, None] - s.window)
    place = j % PAGE
    q = s.q.float().view(s.seqs, G, H // G, D)
    k = s.pool[page, 0, :, place].float().mul_(s.scales[page, 0, :, place][..., None]).transpose(1, 2)     # [sequence, kv head, position, dim]
    score = (q @ k.transpose(-1, -2)).mul_(s.scale)
    del k
    if s.cap:
        score = torch.tanh(score / s.cap) * s.cap
    score = score.masked_fill_(~seen[:, None, None], -math.inf)
    w = torch.exp(score - score.amax(-1, keepdim=True))
    v = s.pool[page, 1, :, place].float().mul_(s.scales[page, 1, :, place][..., None]).masked_fill_(~seen[..., None, None], 0.0).transpose(1, 2)
    s.out.copy_(((w @ v) / w.sum(-1, keepdim=True)).flatten(1))
    return s.out


def plain_unpack(s):
    last = s.start.long() + s.cu[1:] - s.cu[:-1] - 1
    j = torch.minimum(torch.arange(s.max_len, device="cuda"), last[:, None])          # (behind a sequence's end its last row once more)
    page, place = s.page_table[s.slot.long()].long().gather(1, j // PAGE), j % PAGE
    s.into[page, :, :, place] = (s.pool[page, :, :, place].float() * s.scales[page, :, :, place][..., None]).to(s.into.dtype)
    return s.into


# ------------------------------------------------------------------------------------------ the definitions, in 64 bits
def exact(case, seed):
    return globals()["exact_" + case["op"]](prepare(case, seed))


def turned(x, rope, position, rot, interleaved, inverse=False):
    """The rotation as a product of complex numbers."""
    if not rot:
        return x
    by = torch.view_as_complex(rope[position.long()].double().contiguous())[:, None]
    by = by.conj() if inverse else by
    y = x.clone()
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    z = torch.complex(x[..., a], x[..., b]) * by
    y[..., a], y[..., b] = z.real, z.imag
    return y


def exact_rotary(s):
    x = s.x.double().view(s.rows, s.heads, s.dim)
    return turned(x, s.rope, s.positions, s.rot, s.interleaved, s.inverse).view(s.rows, -1)


def exact_append(s):
    G, H, D = s.kv_heads, s.heads, s.dim
    q_out, scales = torch.empty((s.n_tok, H * D), dtype=torch.float64, device="cuda"), s.scales.double()
    for i in range(s.seqs):
        r0, n, C = s.cu_host[i], s.counts[i], s.start_host[i]
        x = s.qkv[r0:r0 + n].double().view(n, H + 2 * G, D)
        at = torch.arange(C, C + n, device="cuda")
        q_out[r0:r0 + n] = turned(x[:, :H], s.rope, at, s.rot, s.interleaved).reshape(n, -1)
        pages = s.page_table[s.slot_host[i]].long()[at // PAGE]
        for part, y in ((0, turned(x[:, H:H + G], s.rope, at, s.rot, s.interleaved)), (1, x[:, H + G:])):
            scales[pages, part, :, at % PAGE] = y.abs().max(-1).values / TOP[s.cache]
    return q_out, None, scales                   # (bytes are rounded, and have no value in between)


def exact_attn(s):
    G, H, D = s.kv_heads, s.heads, s.dim
    out = torch.empty((s.seqs, H, D), dtype=torch.float64, device="cuda")
    for i in range(s.seqs):
        n = s.start_host[i] + 1
        first = max(0, n - s.window) if s.window else 0
        pages = s.page_table[s.slot_host[i], :-(-n // PAGE)].long()
        for g in range(G):
            k, v = (s.pool[pages, p, g].to(torch.float64) * s.scales[pages, p, g, :, None].double() for p in (0, 1))
            k, v = k.flatten(0, 1)[first:n], v.flatten(0, 1)[first:n]
            heads = slice(g * (H // G), (g + 1) * (H // G))
            z = s.q[i].double().view(H, D)[heads] @ k.T * s.scale
            z = s.cap * torch.tanh(z / s.cap) if s.cap else z
            out[i, heads] = torch.softmax(z, -1) @ v
    return out.view(s.seqs, -1)


def exact_unpack(s):
    into = s.into.double()
    for i in range(s.seqs):
        n = s.start_host[i] + s.counts[i]
        for b in range(-(-n // PAGE)):
            page, rows = int(s.page_table[s.slot_host[i], b]), min(PAGE, n - b * PAGE)
            into[page, :, :, :rows] = s.pool[page, :, :, :rows].double() * s.scales[page, :, :, :rows, None].double()
    return into
