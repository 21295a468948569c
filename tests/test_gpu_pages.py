"""Copies of pages and moves of rows in the caches of several layers, bit by bit."""
import random
from types import SimpleNamespace

import pytest
import torch

import tree_util as tu

pytestmark = pytest.mark.gpu


def _caches(cuda, shapes, rows, max_len, page, n_pages, seed):
    """Layers of different shapes and types over one page table in a random order."""
    from poptransformer_b200 import ops
    g, rng = torch.Generator(device="cpu").manual_seed(seed), random.Random(seed)
    per = -(-max_len // page)
    table = torch.tensor(rng.sample(range(n_pages), rows * per), dtype=torch.int32).view(rows, per).to(cuda)
    out = []
    for n_kv, dim, vdim, dt in shapes:
        c = ops.PagedKVCache(rows, n_kv, dim, max_len, page, cuda, table, v_dim=vdim, dtype=dt, n_pages=n_pages)
        raw = c.pool.view(n_pages, -1).view(torch.uint8)
        raw.copy_(torch.randint(0, 256, raw.shape, generator=g, dtype=torch.uint8))
        out.append(c)
    return out, table


def _bytes(c):
    return c.pool.view(c.pool.shape[0], -1).view(torch.uint8)


SHAPES = {"one": [(2, 128, 128, torch.bfloat16)], "mixed": [(2, 128, 128, torch.bfloat16), (1, 64, 32, torch.float16), (3, 7, 5, torch.bfloat16), (1, 36, 0, torch.float32)],
          "odd": [(1, 3, 1, torch.float16)], "many": [(1, 8, 8, torch.bfloat16)] * 70}


@pytest.mark.parametrize("shapes", list(SHAPES))
@pytest.mark.parametrize("page,n", [(64, 5), (16, 33), (5, 1), (64, 0)])
def test_copies(cuda, shapes, page, n):
    from poptransformer_b200 import ops
    caches, _ = _caches(cuda, SHAPES[shapes], 1, page, page, 80, n)
    pools = ops.PagePools(caches)
    order = random.Random(n).sample(range(80), 2 * n)
    before = [_bytes(c).clone() for c in caches]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda)
    pools.copy_pages(i32(order[:n]), i32(order[n:]))
    for c, b in zip(caches, before):
        want = b.clone()
        want[order[n:]] = b[order[:n]]
        assert torch.equal(_bytes(c), want)


def test_copies_left_out(cuda):
    """Negative pages, a page onto itself, and pages that the pool does not have (which set the flag)."""
    from poptransformer_b200 import ops
    caches, _ = _caches(cuda, SHAPES["mixed"], 1, 64, 64, 10, 1)
    pools, flag = ops.PagePools(caches), torch.zeros(1, dtype=torch.int32, device=cuda)
    before = [_bytes(c).clone() for c in caches]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda)
    pools.copy_pages(i32([-1, 3, 4, 5]), i32([2, -1, 4, 6]), error_flag=flag)
    assert flag.item() == 0
    pools.copy_pages(i32([10, 0]), i32([7, 1 << 30]), error_flag=flag)
    assert flag.item() == 12
    for c, b in zip(caches, before):
        b[6] = b[5].clone()
        assert torch.equal(_bytes(c), b)


@pytest.mark.parametrize("shapes", list(SHAPES))
@pytest.mark.parametrize("page", [64, 16, 5])
def test_moves(cuda, shapes, page):
    from poptransformer_b200 import ops
    rng = random.Random(page)
    counts, starts = [20, 1, 0, 256, 9, 30], [60, 0, 3, 11, 63, 128]
    kept = [[0, 3, 4, 10, 19], [0], [], sorted(rng.sample(range(256), 200)), [0, 1, 2, 3, 4, 5, 6, 7, 8], [2, 29]]
    rows, max_len = 8, 280
    caches, table = _caches(cuda, SHAPES[shapes], rows, max_len, page, rows * -(-max_len // page) + 3, page)
    slot = rng.sample(range(rows), len(counts))
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda)
    cu = [sum(counts[:i]) for i in range(len(counts) + 1)]
    view = ops.batch_view(len(counts), cu[-1], i32(cu), i32(starts), i32(slot), i32([0] * cu[-1]))
    path = i32([k + [-1] * (200 - len(k)) for k in kept])
    before, flag = [_bytes(c).clone() for c in caches], torch.zeros(1, dtype=torch.int32, device=cuda)
    ops.PagePools(caches).move_rows(view, path, i32([len(k) for k in kept]), error_flag=flag)
    host = table.tolist()
    for c, b in zip(caches, before):
        es, cut = c.pool.element_size(), c.n_kv * page * c.head_dim * c.pool.element_size()
        K, V = b[:, :cut].reshape(len(b), c.n_kv, page, c.head_dim * es), b[:, cut:].reshape(len(b), c.n_kv, page, c.v_dim * es)
        want_k, want_v = K.clone(), V.clone()
        for s, k in enumerate(kept):
            for to, r in enumerate(k):
                (pa, ia), (pb, ib) = (divmod(starts[s] + x, page) for x in (r, to))
                want_k[host[slot[s]][pb], :, ib] = K[host[slot[s]][pa], :, ia]
                want_v[host[slot[s]][pb], :, ib] = V[host[slot[s]][pa], :, ia]
        assert torch.equal(_bytes(c), torch.cat([want_k.flatten(1), want_v.flatten(1)], 1))
    assert flag.item() == 0


def test_moves_refused_on_the_device(cuda):
    """Paths that do not increase or leave the new tokens, counts beyond them, positions outside the table: nothing of the sequence moves."""
    from poptransformer_b200 import ops
    caches, table = _caches(cuda, SHAPES["one"], 6, 128, 64, 12, 3)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda)
    before, flag = _bytes(caches[0]).clone(), torch.zeros(1, dtype=torch.int32, device=cuda)
    pools = ops.PagePools(caches)

    def move(path, count, start=50, n=8):
        flag.zero_()
        pools.move_rows(ops.batch_view(1, n, i32([0, n]), i32([start]), i32([2]), i32([0] * n)), i32([path]), i32([count]), error_flag=flag)
        assert torch.equal(_bytes(caches[0]), before)
        return flag.item()

    assert move([0, 2, 2, 5], 4) == 14 and move([0, 3, 1, 5], 4) == 14 and move([-1, 2, 3, 4], 4) == 14 and move([0, 2, 3, 8], 4) == 14
    assert move([0, 2, 3, 4], 5) == 14 and move([0, 1, 2, 3], 4, n=3) == 14
    assert move([0, 2, 3, 4], 4, start=-1) == 12 and move([0, 2, 3, 4], 4, start=121) == 12
    assert move([1, 2, 3, 4], 0) == 0 and move([1, 2, 3, 4], -3) == 0 and move([0, 1, 2, 3], 4) == 0
    table[2, 0] = -1
    assert move([0, 2, 3, 4], 4) == 12


def _model(cuda, V, W, layers, heads, n_kv, dim, seed):
    g = torch.Generator(device="cpu").manual_seed(seed)
    r = lambda *s: (torch.randn(s, generator=g) / s[-1] ** 0.5).to(cuda)
    return SimpleNamespace(emb=r(V, W) * W ** 0.5, qkv=[r((heads + 2 * n_kv) * dim, W) for _ in range(layers)], o=[r(W, heads * dim) for _ in range(layers)], head=r(V, W) * 3)


def test_a_speculative_generation_is_the_plain_one(cuda):
    """A small fp32 model generates greedily token by token (window_attn), and in steps of drafted trees: tree_attn, verify_drafts, move_rows, truncate.  Half
    way the sequences fork, and the pool is compacted.  The drafts are the plain run's tokens with mistakes."""
    from poptransformer_b200 import ops
    from poptransformer_b200.cache import SequenceSlots
    V, W, L, H, G, D, B, new, page = 97, 64, 3, 4, 2, 32, 3, 40, 8
    m = _model(cuda, V, W, L, H, G, D, 1)
    rope = torch.stack([f(torch.arange(128, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(D // 2, dtype=torch.float64) / (D // 2))) for f in (torch.cos, torch.sin)],
                       -1).float().to(cuda)
    prompts = [[5, 17, 3, 80, 41], [9], [60, 2, 2, 33, 1, 0, 8, 77, 19, 20, 21]]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda)

    def caches(slots):
        return [ops.PagedKVCache(8, G, D, 128, page, cuda, slots.page_table, dtype=torch.float32, n_pages=slots.n_pages) for _ in range(L)]

    def forward(cs, entries, attend):
        """entries: (slot, start, tokens, parents); logits of all rows."""
        counts = [len(e[2]) for e in entries]
        cu = [sum(counts[:i]) for i in range(len(counts) + 1)]
        view = ops.batch_view(len(entries), cu[-1], i32(cu), i32([e[1] for e in entries]), i32([e[0] for e in entries]), i32([i for i, n in enumerate(counts) for _ in range(n)]))
        x = m.emb[[t for e in entries for t in e[2]]]
        parent = i32([p for e in entries for p in e[3]])
        for c, wq, wo in zip(cs, m.qkv, m.o):
            rows = (torch.nn.functional.layer_norm(x, (W,)) @ wq.T).contiguous()
            out = torch.empty((cu[-1], H * D), device=cuda)
            attend(view, rows, c, out, parent, max(counts))
            x = x + out @ wo.T
        return view, torch.nn.functional.layer_norm(x, (W,)) @ m.head.T

    ws = ops.tree_attn_workspace(8, 16, H, G, D)

    def by_tree(view, rows, c, out, parent, most):
        ops.tree_attn(view, rows, rows.shape[1], c, out, H * D, H, D ** -0.5, parent, rope=rope, rope_dims=D, max_tokens_per_seq=most, workspace=ws)

    def by_window(view, rows, c, out, parent, most):
        ops.window_attn(view, rows, rows.shape[1], c, out, H * D, H, D ** -0.5, rope=rope, rope_dims=D, max_tokens_per_seq=most)

    # ---- token by token
    slots = SequenceSlots(8, 128, page, 60, cuda)
    cs = caches(slots)
    plain = []
    for prompt in prompts:
        s, ids, todo = slots.open(), list(prompt), list(prompt)
        while len(ids) < len(prompt) + new + 12:
            start = slots.extend(s, len(todo))
            _, logits = forward(cs, [(s, start, todo, list(range(-1, len(todo) - 1)))], by_window)
            todo = [int(logits[-1].argmax())]
            ids += todo
        plain.append(ids)
        slots.close(s)
    # ---- in steps of trees
    rng = random.Random(3)
    slots = SequenceSlots(8, 128, page, 60, cuda)
    cs = caches(slots)
    pools = ops.PagePools(cs)
    state = []
    for k, prompt in enumerate(prompts):
        s = slots.open()
        if len(prompt) > 1:
            forward(cs, [(s, slots.extend(s, len(prompt) - 1), prompt[:-1], list(range(-1, len(prompt) - 2)))], by_tree)
        state.append(SimpleNamespace(slot=s, ids=list(prompt), of=k, steps=0))
    forked = False
    while any(len(x.ids) < len(prompts[x.of]) + new for x in state):
        live = [x for x in state if len(x.ids) < len(prompts[x.of]) + new]
        entries = []
        for x in live:
            n = rng.randint(1, 10)
            tokens, parents = [x.ids[-1]], [-1]
            for i in range(1, n):                      # a node's right token, or a wrong one
                p = rng.randint(max(0, i - 4), i - 1)
                depth, q = 0, p
                while q > 0:
                    q, depth = parents[q], depth + 1
                right = plain[x.of][len(x.ids) + depth]
                tokens.append(right if rng.random() < 0.7 else rng.randint(0, V - 1))
                parents.append(p)
            entries.append((x.slot, slots.extend(x.slot, n), tokens, parents))
        view, logits = forward(cs, entries, by_tree)
        counts = [len(e[2]) for e in entries]
        path, count, said, _ = ops.verify_drafts(logits.contiguous(), i32([sum(counts[:i]) for i in range(len(counts) + 1)]), i32([t for e in entries for t in e[2]]),
                                                 i32([p for e in entries for p in e[3]]), max_path=10)
        pools.move_rows(view, path, count)
        for x, e, k, t in zip(live, entries, count.tolist(), said.tolist()):
            x.ids += t[:k]
            x.steps += 1
            pools.copy(slots.truncate(x.slot, e[1] + k))
            assert slots.length[x.slot] == len(x.ids) - 1
        if not forked and all(len(x.ids) > len(prompts[x.of]) + new // 3 for x in state):
            forked = True
            for x in list(state):
                back = len(x.ids) - 1 - rng.randint(0, 5)
                s, copies = slots.fork(x.slot, back)
                pools.copy(copies)
                state.append(SimpleNamespace(slot=s, ids=x.ids[:back + 1], of=x.of, steps=0))
            slots.close(state.pop(1).slot)
            pools.copy(slots.compact())
            assert sorted(slots._free_pages) == list(range(slots.n_pages - slots.free_pages, slots.n_pages))
    assert forked and len(state) == 5
    for x in state:
        n = min(len(x.ids), len(plain[x.of]))
        assert x.ids[:n] == plain[x.of][:n]
    assert any(x.steps < 0.6 * new for x in state)     # (several tokens a step)
