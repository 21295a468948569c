"""Operators of a step of speculative decoding over paged caches, as cases that can be timed and compared.

A step drafts a tree of tokens behind every sequence, runs them through the model at once (attention for the tree over the sequence's
cached pages), lets the target's probabilities decide which of them stand, and puts the cache right: the rows of the accepted path move
together, and sequences are forked or compacted by copying pages.

`run` computes each of them in elementary torch operations, or (own) through the framework.  `exact` computes the same in 64 bits, one
sequence after the other."""
import math
import random
from types import SimpleNamespace

import torch

own = False

PAGE = 64            # positions of a cache page, as the decoders have it by default
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # ---- attention for drafted tokens (rows: drafted tokens of a sequence, its last known token first)
        # One user, a chain of four drafts behind a short chat: latency.
        dict(name="attn chain of 5", op="attn", type="bf16", seqs=1, rows=5, tree="chain", heads=32, kv_heads=8, dim=128, context=700, window=0, cap=0.0, rot=128),
        # Multi-head attention with narrow heads, a small batch.
        dict(name="attn 8 rows 64 wide", op="attn", type="fp16", seqs=4, rows=8, tree="tree", heads=12, kv_heads=12, dim=64, context=500, window=0, cap=0.0, rot=0),
        # Two key/value heads for 32 query heads: many query rows share what is read.
        dict(name="attn two kv heads", op="attn", type="fp16", seqs=8, rows=26, tree="tree", heads=32, kv_heads=2, dim=128, context=1151, window=0, cap=0.0, rot=64),
        # A served batch of unequal lengths: the ordinary case.
        dict(name="attn 16 sequences", op="attn", type="bf16", seqs=16, rows=16, tree="tree", heads=32, kv_heads=8, dim=128, context=4000, window=0, cap=0.0, rot=128),
        # One long document and a wide tree.
        dict(name="attn long context", op="attn", type="bf16", seqs=2, rows=63, tree="tree", heads=32, kv_heads=8, dim=128, context=60000, window=0, cap=0.0, rot=128),
        # True 32-bit model, sliding window and softcap, an odd head width.
        dict(name="attn fp32 window", op="attn", type="fp32", seqs=3, rows=11, tree="tree", heads=16, kv_heads=4, dim=80, context=900, window=512, cap=30.0, rot=80),
        # ---- verification
        # Greedy check of one user's four drafts.
        dict(name="verify greedy", op="verify", type="fp32", seqs=1, rows=5, tree="chain", vocab=32000, draft="none", temperature=0.0),
        # A served batch, drafts sampled from a smaller model whose probabilities are known.
        dict(name="verify sampled chains", op="verify", type="fp32", seqs=32, rows=6, tree="chain", vocab=50257, draft="probs", temperature=0.8),
        # Trees of the draft model's likeliest tokens.
        dict(name="verify trees", op="verify", type="fp16", seqs=16, rows=32, tree="tree", vocab=65024, draft="none", temperature=1.0),
        # ---- pages
        # Sixteen sequences fork: the page that each is filling is copied in every layer.
        dict(name="pages fork", op="pages", type="bf16", layers=32, kv_heads=8, dim=128, pages=96, copies=16),
        # The pool is compacted: many pages move, of a model with few heads.
        dict(name="pages compact", op="pages", type="fp16", layers=28, kv_heads=2, dim=128, pages=1000, copies=450),
        # After verification the accepted rows of every sequence move together.
        dict(name="rows accepted", op="rows", type="bf16", layers=32, kv_heads=8, dim=128, seqs=24, rows=24, path=6, context=1000),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["attn", "attn", "attn", "verify", "verify", "pages", "rows"])
    if op == "attn":
        kv = rng.choice([1, 2, 4, 8])
        c = dict(op="attn", type=rng.choice(["bf16", "bf16", "fp16", "fp32"]), seqs=log(1, 32), rows=log(1, 64), tree=rng.choice(["chain", "tree", "tree"]),
                 heads=kv * rng.choice([f for f in (1, 2, 3, 4, 8) if kv * f <= 32]), kv_heads=kv, dim=rng.choice([64, 128, 128, 128, 96, 72]), context=log(1, 20000), window=0, cap=0.0, rot=0)
        if c["type"] == "fp32":
            c["context"] = min(c["context"], 2000)
        if rng.random() < 0.3:
            c["window"] = log(8, 2000)
        if rng.random() < 0.2:
            c["cap"] = float(rng.randint(10, 50))
        if rng.random() < 0.7:
            c["rot"] = c["dim"] if rng.random() < 0.7 else c["dim"] // 2
        while c["seqs"] * c["context"] * kv > 800000:
            c["seqs"] = max(1, c["seqs"] // 2)
            c["context"] = c["context"] * 3 // 4
        return c
    if op == "verify":
        c = dict(op="verify", type=rng.choice(["fp32", "fp32", "fp16", "bf16"]), seqs=log(1, 48), rows=log(1, 32), tree=rng.choice(["chain", "tree"]), vocab=log(1000, 130000),
                 draft=rng.choice(["none", "probs"]), temperature=rng.choice([0.0, 0.6, 1.0, 1.3]))
        while c["seqs"] * c["rows"] * c["vocab"] > 20000000:
            c["seqs"] = max(1, c["seqs"] // 2)
            c["vocab"] = c["vocab"] * 3 // 4
        return c
    if op == "pages":
        c = dict(op="pages", type=rng.choice(["bf16", "fp16", "fp32"]), layers=log(1, 48), kv_heads=rng.choice([1, 2, 4, 8]), dim=rng.choice([64, 80, 128]), pages=0, copies=log(1, 600))
        while c["layers"] * c["kv_heads"] * c["copies"] > 40000:
            c["copies"] = max(1, c["copies"] // 2)
        c["pages"] = 2 * c["copies"] + rng.randint(3, 90)
        return c
    rows = log(2, 64)
    return dict(op="rows", type=rng.choice(["bf16", "fp16", "fp32"]), layers=log(1, 48), kv_heads=rng.choice([1, 2, 4, 8]), dim=rng.choice([64, 80, 128]), seqs=log(1, 32), rows=rows,
                path=rng.randint(1, min(rows, 8)), context=log(1, 1500))


# ------------------------------------------------------------------------------------------ sizes that follow from a case alone
def lengths(case):
    """Cached positions of every sequence: the longest has all of the context."""
    rng = random.Random(7 * case["context"] + case["seqs"])
    return [case["context"]] + [max(0, int(case["context"] * rng.uniform(0.3, 1.0))) for _ in range(case["seqs"] - 1)]


def row_counts(case):
    """New rows of every sequence: the first has all of them."""
    rng = random.Random(11 * case["rows"] + case["seqs"])
    return [case["rows"]] + [max(1, int(case["rows"] * rng.uniform(0.6, 1.0))) for _ in range(case["seqs"] - 1)]


def parents(case, counts, rng):
    """The row of every row's parent, sequence after sequence: the root's is -1, a chain's the row before."""
    out = []
    for n in counts:
        out += [-1] + [i - 1 if case["tree"] == "chain" else rng.randint(max(0, (i - 1) // 3 - 1), max(0, (i - 1) // 2)) for i in range(1, n)]
    return out


def depths(counts, parent):
    out, at = [], 0
    for n in counts:
        for i in range(n):
            out.append(0 if parent[at + i] < 0 else out[at + parent[at + i]] + 1)
        at += n
    return out


def work(case):
    es = TYPES[case["type"]].itemsize
    if case["op"] == "attn":
        c, n = lengths(case), row_counts(case)
        G, H, D, W = case["kv_heads"], case["heads"], case["dim"], case["window"]
        seen = [min(a, W) if W else a for a in c]
        moved = sum(seen) * 2 * G * D + sum(n) * (2 * H + 4 * G) * D     # cached keys and values; q, k, v in, output and appended rows out
        return dict(bytes=moved * es, flops=sum(4 * D * H * k * (a + k / 2) for a, k in zip(seen, n)))
    if case["op"] == "verify":
        # a sequence's path: about half of its levels are reached, and what is not accepted is drawn from one more row's rest
        levels = 1.0 if case["rows"] == 1 else case["rows"] / 2 if case["tree"] == "chain" else math.log2(case["rows"] + 1) / 1.5
        visited = case["seqs"] * min(levels, case["rows"])
        return dict(bytes=visited * case["vocab"] * (es + (4 if case["draft"] == "probs" and case["temperature"] > 0 else 0)), flops=visited * case["vocab"] * 4)
    if case["op"] == "pages":
        return dict(bytes=2 * es * case["copies"] * case["layers"] * 2 * case["kv_heads"] * PAGE * case["dim"], flops=0)
    return dict(bytes=2 * es * case["seqs"] * case["path"] * 0.75 * case["layers"] * 2 * case["kv_heads"] * case["dim"], flops=0)


# ------------------------------------------------------------------------------------------ inputs
def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return globals()["prepare_" + case["op"]](SimpleNamespace(**case), case, gen, random.Random(seed))


def packed(s, case, rng):
    """Where the new rows of every sequence lie, and the tree that they form."""
    s.counts = row_counts(case)
    s.n_tok, s.most = sum(s.counts), max(s.counts)
    s.host_parent = parents(case, s.counts, rng)
    s.cu_host = [sum(s.counts[:i]) for i in range(s.seqs + 1)]
    s.cu, s.parent = ints(s.cu_host), ints(s.host_parent)
    s.tok_seq = ints([i for i, n in enumerate(s.counts) for _ in range(n)])
    s.row_of = torch.arange(s.n_tok, device="cuda") - s.cu[s.tok_seq.long()]


def paged(s, case, rng):
    """Pages of every sequence, in any order, and a table with a row per slot; sequences sit in slots of their own."""
    s.start_host = lengths(case)
    s.max_len = max(a + n for a, n in zip(s.start_host, s.counts))
    s.max_pages = -(-s.max_len // PAGE)
    need = [-(-(a + n) // PAGE) for a, n in zip(s.start_host, s.counts)]
    s.n_pages = sum(need) + 2
    order = list(range(s.n_pages))
    rng.shuffle(order)
    s.slot_host = list(range(s.seqs))
    rng.shuffle(s.slot_host)
    table = [[0] * s.max_pages for _ in range(s.seqs)]
    for i, n in enumerate(need):
        at = sum(need[:i])
        table[s.slot_host[i]][:n] = order[at:at + n]
    s.start, s.slot, s.page_table = ints(s.start_host), ints(s.slot_host), ints(table)


def cache_of(s, pool):
    from poptransformer_b200 import ops
    return ops.PagedKVCache(s.seqs, s.kv_heads, s.dim, s.max_len, PAGE, "cuda", s.page_table, dtype=pool.dtype, pool=pool)


def prepare_attn(s, case, gen, rng):
    dt = TYPES[s.type]
    packed(s, case, rng)
    paged(s, case, rng)
    D, G, H = s.dim, s.kv_heads, s.heads
    s.ld = (H + 2 * G) * D
    rand = lambda *shape: torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32 if dt == torch.float32 else torch.bfloat16)
    s.pool = rand(s.n_pages, 2, G, PAGE, D).to(dt)
    s.qkv = rand(s.n_tok, s.ld)
    s.qkv[:, :H * D] *= 1.5
    s.qkv = s.qkv.to(dt)
    s.scale = D ** -0.5
    s.rope = None
    if s.rot:
        angle = torch.arange(s.max_len, device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(s.rot // 2, device="cuda", dtype=torch.float64) * 2 / s.rot)
        s.rope = torch.stack([angle.cos(), angle.sin()], -1).float().contiguous()
    s.out = torch.empty((s.n_tok, H * D), dtype=dt, device="cuda")
    s.where = padded_rows(s)
    if own:
        from poptransformer_b200 import ops
        s.cache, s.view = cache_of(s, s.pool), ops.batch_view(s.seqs, s.n_tok, s.cu, s.start, s.slot, s.tok_seq)
        s.flag = ints([0])
        s.workspace = ops.tree_attn_workspace(s.seqs, s.most, H, G, D, "cuda")
    return s


def padded_rows(s):
    """[sequence, row] -> packed row, and which of them there are."""
    row = torch.arange(s.most, device="cuda")
    at = s.cu[:-1, None].long() + row
    there = at < s.cu[1:, None]
    return torch.where(there, at, 0), there


def prepare_verify(s, case, gen, rng):
    dt = TYPES[s.type]
    packed(s, case, rng)
    n, V = s.n_tok, s.vocab
    # logits as a language model has them: a few tokens carry the weight; the draft model's are near
    s.logits = torch.randn((n, V), generator=gen, device="cuda") * 2.0
    s.logits += 9.0 * torch.rand((n, V), generator=gen, device="cuda") ** 40
    draft = s.logits + 0.5 * torch.randn((n, V), generator=gen, device="cuda")
    s.logits = s.logits.to(dt)
    s.up = torch.tensor([max(0, p) + s.cu_host[i] for i, p in zip(s.tok_seq.tolist(), s.host_parent)], device="cuda")   # packed row of the parent
    seen, rank = {}, []
    for r, u in enumerate(s.up.tolist()):
        root = s.host_parent[r] < 0
        rank.append(0 if root else seen.get(u, 0))
        if not root:
            seen[u] = seen.get(u, 0) + 1
    s.width = max(seen.values(), default=0)
    s.rank = torch.tensor(rank, device="cuda")
    s.depth = max(depths(s.counts, s.host_parent)) + 1
    q = torch.softmax(draft / (s.temperature or 1.0), -1)
    if s.draft == "probs":
        s.token = torch.multinomial(q[s.up], 1, generator=gen)[:, 0].int()
        s.probs = q
    else:
        likely = torch.topk(draft, max(1, s.width), dim=-1).indices
        s.token = likely[s.up, s.rank].int()
        s.probs = None
    s.uniform = torch.rand(n, generator=gen, device="cuda")
    s.uniform_next = torch.rand(s.seqs, generator=gen, device="cuda")
    s.temp = torch.full((s.seqs,), s.temperature, device="cuda") if s.temperature > 0 else None
    s.root = torch.tensor([p < 0 for p in s.host_parent], device="cuda")
    return s


def prepare_pages(s, case, gen, rng):
    dt = TYPES[s.type]
    s.seqs, s.max_len = 1, PAGE
    shape = (s.layers, s.pages, 2, s.kv_heads, PAGE, s.dim)
    s.pool = torch.randn(shape, generator=gen, device="cuda", dtype=dt)
    order = list(range(s.pages))
    rng.shuffle(order)
    s.src, s.dst = ints(order[:s.copies]), ints(order[s.copies:2 * s.copies])
    s.page_table = ints([[0]])
    if own:
        from poptransformer_b200 import ops
        s.pools = ops.PagePools([cache_of(s, p) for p in s.pool])
    return s


def prepare_rows(s, case, gen, rng):
    dt = TYPES[s.type]
    packed(s, dict(case, tree="chain"), rng)
    paged(s, case, rng)
    s.pool = torch.randn((s.layers, s.n_pages, 2, s.kv_heads, PAGE, s.dim), generator=gen, device="cuda", dtype=dt)
    # the root is always kept; how many of its descendants stand differs from sequence to sequence
    s.kept = [[0] + sorted(rng.sample(range(1, n), min(n - 1, rng.randint(s.path // 2, s.path) - 1))) if s.path > 1 and n > 1 else [0] for n in s.counts]
    s.count = ints([len(k) for k in s.kept])
    s.path_rows = ints([k + [-1] * (s.path - len(k)) for k in s.kept])
    if own:
        from poptransformer_b200 import ops
        s.pools = ops.PagePools([cache_of(s, p) for p in s.pool])
        s.view = ops.batch_view(s.seqs, s.n_tok, s.cu, s.start, s.slot, s.tok_seq)
        s.flag = ints([0])
    return s


# ------------------------------------------------------------------------------------------ one pass
def run(state):
    if own:
        return globals()["own_" + state.op](state)
    return globals()["plain_" + state.op](state)


def own_attn(s):
    from poptransformer_b200 import ops
    ops.tree_attn(s.view, s.qkv, s.ld, s.cache, s.out, s.out.shape[1], s.heads, s.scale, None if s.tree == "chain" else s.parent, window=s.window, softcap=s.cap, rope=s.rope,
                  rope_dims=s.rot, max_tokens_per_seq=s.most, workspace=s.workspace, error_flag=s.flag)
    return s.out, s.pool


def own_verify(s):
    from poptransformer_b200 import ops
    return ops.verify_drafts(s.logits, s.cu, s.token, None if s.tree == "chain" else s.parent, max_path=s.depth, draft=s.probs, temperature=s.temp, uniform=s.uniform,
                             uniform_next=s.uniform_next)


def own_pages(s):
    s.pools.copy_pages(s.src, s.dst)
    return s.pool


def own_rows(s):
    s.pools.move_rows(s.view, s.path_rows, s.count, error_flag=s.flag)
    return s.pool


def ancestors(s):
    """[sequence, row, row]: whether a row is another's ancestor or itself."""
    at, there = s.where
    up = torch.where(there, s.parent.long()[at], -1)
    a = torch.eye(s.most, device="cuda").expand(s.seqs, -1, -1)
    a = a + (torch.arange(s.most, device="cuda") == up[:, :, None])
    for _ in range(max(1, s.most - 1).bit_length()):      # twice as many generations a time
        a = (a @ a).clamp(max=1.0)
    return a > 0


def rotate(s, x, position):
    """x [.., heads, dim], position [..]: the first `rot` dimensions turn in pairs (i, i + rot / 2)."""
    h = s.rot // 2
    if not h:
        return x
    c, n = s.rope[position][..., None, :, 0], s.rope[position][..., None, :, 1]
    u, v = x[..., :h], x[..., h:2 * h]
    return torch.cat([u * c - v * n, v * c + u * n, x[..., 2 * h:]], -1)


def plain_attn(s):
    G, H, D, dt = s.kv_heads, s.heads, s.dim, s.qkv.dtype
    at, there = s.where
    up = ancestors(s)
    depth = up.sum(-1) - 1                                                    # [sequence, row]
    x = s.qkv.float()[at]                                                     # [sequence, row, ..]
    position = s.start[:, None].long() + depth
    q = rotate(s, x[..., :H * D].unflatten(-1, (H, D)), position)
    k = rotate(s, x[..., H * D:(H + G) * D].unflatten(-1, (G, D)), position).to(dt)
    v = x[..., (H + G) * D:].unflatten(-1, (G, D)).to(dt)
    row = s.start[:, None].long() + torch.arange(s.most, device="cuda")
    last = s.start[:, None].long() + (s.cu[1:] - s.cu[:-1])[:, None].long() - 1
    keep = there[..., None, None]
    table = s.page_table[s.slot.long()].long()
    page, place = table.gather(1, torch.minimum(row, last) // PAGE), torch.minimum(row, last) % PAGE
    # (rows that are not there write the last row's values once more)
    own_last = (last - s.start[:, None].long())[..., None, None].expand(-1, s.most, G, D)
    s.pool[page, 0, :, place] = torch.where(keep, k, k.gather(1, own_last))
    s.pool[page, 1, :, place] = torch.where(keep, v, v.gather(1, own_last))
    j = torch.arange(s.max_len, device="cuda")
    page = table[:, j // PAGE]
    K, V = (s.pool[page, i, :, j % PAGE].float().transpose(1, 2) for i in (0, 1))      # [sequence, kv head, position, dim]
    q = q.unflatten(2, (G, H // G)).permute(0, 2, 1, 3, 4).flatten(2, 3)               # [sequence, kv head, row x head, dim]
    score = (q @ K.transpose(-1, -2)).mul_(s.scale)
    if s.cap:
        score = torch.tanh(score / s.cap) * s.cap
    drafted = j - s.start[:, None].long()                                              # [sequence, position]: the row that a position holds
    inside = drafted.clamp(0, s.most - 1)
    of = inside[:, None, :].expand(-1, s.most, -1)
    seen = torch.where(drafted[:, None] < 0, True, up.gather(2, of) & (drafted <= last - s.start[:, None])[:, None])
    if s.window:
        behind = torch.where(drafted < 0, j, s.start[:, None].long() + depth.gather(1, inside))
        seen = seen & (position[:, :, None] - behind[:, None] < s.window)
    seen = seen[:, None, :, None].expand(-1, 1, -1, H // G, -1).flatten(2, 3)
    score = score.masked_fill_(~seen, -math.inf)
    w = torch.exp(score - score.amax(-1, keepdim=True))
    out = (w @ V) / w.sum(-1, keepdim=True)
    out = out.unflatten(2, (s.most, H // G)).permute(0, 2, 1, 3, 4).flatten(2)         # [sequence, row, ..]
    s.out.copy_(out[s.tok_seq.long(), s.row_of])
    return s.out, s.pool


def plain_verify(s):
    n, V = s.n_tok, s.vocab
    x = s.logits.double()
    token, u = s.token.long(), s.uniform.double()
    none = torch.full((n,), n, device="cuda")
    logp = x / (s.temperature or 1.0)
    logp = logp - logp.amax(-1, keepdim=True)
    p = torch.exp(logp)
    total = p.sum(-1, keepdim=True)
    p, logp = p / total, logp - torch.log(total)
    if s.temperature == 0:
        best = x.argmax(-1)
        accepted = best[s.up] == token
        rest = None
    else:
        accepted = torch.zeros(n, dtype=torch.bool, device="cuda")
        taken = torch.zeros(n, dtype=torch.float64, device="cuda")             # with draft probabilities: how many times q has left p
        rest = p.clone()
        for j in range(s.width):                                               # the j-th child of every row
            mine = (s.rank == j) & ~s.root
            mass = rest.sum(-1)
            q = s.probs[s.up, token].double() if s.probs is not None else 1.0
            accepted |= mine & (u * q * mass[s.up] < rest[s.up, token])
            child = torch.zeros(n, dtype=torch.bool, device="cuda").index_put((s.up,), mine, accumulate=True)
            if s.probs is not None:
                taken = taken + torch.where(child, mass, 0.0)
                rest = torch.where(child[:, None], (p - taken[:, None] * s.probs).clamp(min=0), rest)
            else:
                gone = torch.zeros((n, V), dtype=torch.bool, device="cuda").index_put((s.up, token), mine, accumulate=True)
                rest = rest.masked_fill(gone, 0.0)
        rest = torch.where(rest.sum(-1, keepdim=True) > 0, rest, p)
    # down the tree: the first accepted child of every row
    order = torch.arange(n, device="cuda")
    first = none.scatter_reduce(0, s.up, torch.where(accepted & ~s.root, order, n), "amin")
    node = s.cu[:-1].long()
    path = [node]
    for _ in range(s.depth - 1):
        child = torch.where(path[-1] < n, first[path[-1].clamp(max=n - 1)], n)
        path.append(child)
    path = torch.stack(path, 1)                                                # [sequence, level], n behind the end
    on = path < n
    count = on.sum(1)
    end = path.gather(1, count[:, None] - 1)[:, 0]
    if rest is None:
        drawn = best[end]
    else:
        r = rest[end]
        cdf = r.cumsum(-1)
        hit = (cdf > s.uniform_next.double()[:, None] * cdf[:, -1:]) & (r > 0)
        last = V - 1 - (r > 0).flip(-1).int().argmax(-1)
        drawn = torch.where(hit.any(-1), hit.int().argmax(-1), last)
    level = torch.arange(s.depth, device="cuda")
    following = torch.cat([path[:, 1:], torch.full_like(path[:, :1], n)], 1).clamp(max=n - 1)
    out = torch.where(level == count[:, None] - 1, drawn[:, None], token[following])
    out = torch.where(on, out, -1)
    lp = logp[path.clamp(max=n - 1), out.clamp(min=0)]
    rows = torch.where(on, path - s.cu[:-1, None], -1)
    return rows.int(), count.int(), out.int(), torch.where(on, lp, 0.0).float()


def plain_pages(s):
    s.pool.index_copy_(1, s.dst.long(), s.pool.index_select(1, s.src.long()))
    return s.pool


def plain_rows(s):
    i = torch.arange(s.path, device="cuda")
    src = s.start[:, None].long() + torch.where(i < s.count[:, None], s.path_rows, i)
    dst = s.start[:, None].long() + i
    most = s.start[:, None].long() + (s.cu[1:] - s.cu[:-1])[:, None].long() - 1          # (rows that a sequence does not have stay where they are)
    src, dst = torch.minimum(src, most), torch.minimum(dst, most)
    table = s.page_table[s.slot.long()].long()
    s.pool[:, table.gather(1, dst // PAGE), :, :, dst % PAGE] = s.pool[:, table.gather(1, src // PAGE), :, :, src % PAGE]
    return s.pool


# ------------------------------------------------------------------------------------------ the definitions, in 64 bits
def exact(case, seed):
    return globals()["exact_" + case["op"]](prepare(case, seed))


def line(parent, r):
    """Row r's ancestors and itself, root first."""
    up = []
    while r >= 0:
        up.append(r)
        r = parent[r]
    return up[::-1]


def exact_attn(s):
    G, H, D, dt = s.kv_heads, s.heads, s.dim, s.qkv.dtype
    out = torch.empty((s.n_tok, H * D), dtype=torch.float64, device="cuda")
    pool = s.pool.double()
    for i in range(s.seqs):
        r0, n, C = s.cu_host[i], s.counts[i], s.start_host[i]
        parent = s.host_parent[r0:r0 + n]
        lines = [line(parent, r) for r in range(n)]
        x = s.qkv[r0:r0 + n].double()
        at = torch.tensor([C + len(a) - 1 for a in lines], device="cuda")

        def turned(y):
            h = s.rot // 2
            if not h:
                return y
            z = torch.complex(y[..., :h], y[..., h:2 * h]) * torch.view_as_complex(s.rope[at].double())[:, None]
            return torch.cat([z.real, z.imag, y[..., 2 * h:]], -1)

        q, k, v = turned(x[:, :H * D].view(n, H, D)), turned(x[:, H * D:(H + G) * D].view(n, G, D)), x[:, (H + G) * D:].view(n, G, D)
        pages = s.page_table[s.slot_host[i], :-(-(C + n) // PAGE)].long()
        place = torch.arange(C, C + n, device="cuda")
        pool[pages[place // PAGE], 0, :, place % PAGE], pool[pages[place // PAGE], 1, :, place % PAGE] = k, v
        # (a row that was appended is read as it is kept: in the cache's type)
        K, V = (pool[pages, j].transpose(0, 1).flatten(1, 2)[:, :C + n].clone() for j in (0, 1))
        K[:, C:] = K[:, C:].to(dt).double()
        seen = torch.zeros((n, C + n), dtype=torch.bool, device="cuda")
        seen[:, :C] = True
        where = torch.cat([torch.arange(C, device="cuda"), at])
        for r, a in enumerate(lines):
            seen[r, [C + b for b in a]] = True
        if s.window:
            seen &= at[:, None] - where < s.window
        for g in range(G):
            for h in range(g * (H // G), (g + 1) * (H // G)):
                z = q[:, h] @ K[g].T * s.scale
                z = s.cap * torch.tanh(z / s.cap) if s.cap else z
                out[r0:r0 + n, h * D:(h + 1) * D] = torch.softmax(z.masked_fill(~seen, -math.inf), -1) @ V[g]
    return out, pool


def exact_verify(s):
    rows, counts, tokens, logs = [], [], [], []
    token, u, last = s.token.tolist(), s.uniform.double().tolist(), s.uniform_next.double().tolist()
    for i in range(s.seqs):
        r0, parent = s.cu_host[i], s.host_parent[s.cu_host[i]:s.cu_host[i + 1]]
        path, said, lp, at = [0], [], [], 0
        while True:
            z = s.logits[r0 + at].double()
            logp = torch.log_softmax(z / (s.temperature or 1.0), -1)
            p = logp.exp()
            rest, taken, go = p, 0.0, None
            for c in [c for c in range(len(parent)) if parent[c] == at]:
                x = token[r0 + c]
                if s.temperature == 0:
                    ok = int(z.argmax()) == x
                elif s.probs is not None:
                    mass = float(rest.sum())
                    ok = u[r0 + c] * float(s.probs[r0 + at, x]) * mass < float(rest[x])
                    taken += mass
                    following = (p - taken * s.probs[r0 + at].double()).clamp(min=0)
                else:
                    ok = u[r0 + c] * float(rest.sum()) < float(rest[x])
                    following = rest.clone()
                    following[x] = 0
                if ok:
                    go = c
                    break
                if s.temperature > 0:
                    rest = following
            if go is None:
                if s.temperature == 0:
                    x = int(z.argmax())
                else:
                    rest = rest if float(rest.sum()) > 0 else p
                    cdf = rest.cumsum(-1)
                    x = int(torch.searchsorted(cdf, last[i] * cdf[-1], right=True).clamp(max=s.vocab - 1))
                said.append(x)
                lp.append(float(logp[x]))
                break
            said.append(token[r0 + go])
            lp.append(float(logp[token[r0 + go]]))
            path.append(go)
            at = go
        pad = s.depth - len(path)
        rows.append(path + [-1] * pad)
        counts.append(len(path))
        tokens.append(said + [-1] * pad)
        logs.append(lp + [0.0] * pad)
    return ints(rows), ints(counts), ints(tokens), torch.tensor(logs, dtype=torch.float64, device="cuda")


def exact_pages(s):
    pool = s.pool.clone()
    for a, b in zip(s.src.tolist(), s.dst.tolist()):
        pool[:, b] = s.pool[:, a]
    return pool


def exact_rows(s):
    pool = s.pool.clone()
    for i, kept in enumerate(s.kept):
        pages = s.page_table[s.slot_host[i]].tolist()
        for to, r in enumerate(kept):
            a, b = s.start_host[i] + r, s.start_host[i] + to
            pool[:, pages[b // PAGE], :, :, b % PAGE] = s.pool[:, pages[a // PAGE], :, :, a % PAGE]
    return pool
