"""Verification of drafted tokens against the rules in 64 bits.  Whole numbers are compared exactly: both sides hold their sums in 64 bits, so that a
draw differs only where a random number lies within 1e-12 of a border."""
import math
import random

import pytest
import torch

import tree_util as tu

pytestmark = pytest.mark.gpu
DT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def walk(logits, parent, token, q, t, u, u_next, max_path):
    """One sequence: (path, tokens, log p)."""
    V = logits.shape[1]
    path, said, logs, at = [], [], [], 0
    while True:
        path.append(at)
        z = logits[at].double()
        z = torch.where(z.isnan(), -math.inf, z)
        top = z.max()
        if top == -math.inf:
            return path, said + [-1], logs + [0.0]
        d = torch.where(z == top, 0.0, (z - top) / (t or 1.0))
        p = d.exp() / d.exp().sum()
        logp = d - d.exp().sum().log()
        rest, S, go = p, 0.0, None
        kids = [c for c in range(at + 1, len(parent)) if parent[c] == at] if len(path) < max_path else []
        for c in kids:
            x = token[c]
            if t == 0:
                ok = x == int(z.argmax())
            elif not 0 <= x < V:
                ok = False
            elif q is not None:
                ok = float(u[c]) * float(q[at, x]) * float(rest.sum()) < float(rest[x])
            else:
                ok = float(u[c]) * float(rest.sum()) < float(rest[x])
            if ok:
                go = c
                break
            if t and q is not None:
                S += float(rest.sum())
                rest = (p - S * q[at].double()).clamp(min=0)
            elif t and 0 <= x < V:
                rest = rest.clone()
                rest[x] = 0
        if go is None:
            if t == 0:
                x = int(z.argmax())
            else:
                rest = rest if float(rest.sum()) > 0 else p
                cdf = rest.cumsum(-1)
                hit = ((cdf > float(u_next) * cdf[-1]) & (rest > 0)).nonzero()
                x = int(hit[0]) if len(hit) else int((rest > 0).nonzero()[-1])
            return path, said + [x], logs + [float(logp[x])]
        said.append(token[go])
        logs.append(float(logp[token[go]]))
        at = go


def compare(logits, counts, parents, token, draft, temps, u, u_next, max_path, chain=False, **kw):
    from poptransformer_b200 import ops
    dev = logits.device
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)
    cu = [sum(counts[:i]) for i in range(len(counts) + 1)]
    temperature = None if temps is None else torch.tensor(temps, dtype=torch.float32, device=dev)
    path, count, said, logprob = ops.verify_drafts(logits, i32(cu), token, None if chain else i32([p for q in parents for p in q]), max_path=max_path, draft=draft,
                                                   temperature=temperature, uniform=u, uniform_next=u_next, **kw)
    for i, n in enumerate(counts):
        r = slice(cu[i], cu[i + 1])
        t = 0.0 if temps is None else float(temperature[i])
        want = ([], [], []) if n == 0 else walk(logits[r], parents[i], token[r].tolist(), None if draft is None else draft[r], t, None if u is None else u[r].double(),
                                                None if u_next is None else u_next[i].double(), max_path)
        k = len(want[0])
        assert int(count[i]) == k and path[i].tolist() == want[0] + [-1] * (max_path - k) and said[i].tolist() == want[1] + [-1] * (max_path - k), i
        for a, b in zip(logprob[i].tolist(), want[2] + [0.0] * (max_path - k)):
            assert abs(a - b) <= 2.0 ** -23 * abs(b) + 2.0 ** -30
    return path, count, said


def inputs(dev, counts, kind, vocab, dtype, seed, close=0.5, sharp=9.0):
    g, rng = torch.Generator(device=dev).manual_seed(seed), random.Random(seed)
    n = sum(counts)
    logits = torch.randn((n, vocab), generator=g, device=dev) * 2 + sharp * torch.rand((n, vocab), generator=g, device=dev) ** 40
    q = torch.softmax(logits + close * torch.randn((n, vocab), generator=g, device=dev), -1)
    parents = [tu.tree(k, kind, rng) for k in counts]
    for p in parents:
        p[1:] = [max(0, x) for x in p[1:]]
    base = [sum(counts[:i]) for i in range(len(counts))]
    up = [b + max(0, x) for b, p in zip(base, parents) for x in p]
    token = torch.multinomial(q[up], 1, generator=g)[:, 0].int() if n else torch.zeros(0, dtype=torch.int32, device=dev)
    u, u_next = torch.rand(max(1, n), generator=g, device=dev), torch.rand(len(counts), generator=g, device=dev)
    return logits.to(dtype), parents, token, q, u, u_next


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("kind", ["chain", "tree", "star"])
@pytest.mark.parametrize("vocab", [2, 31, 513, 5003, 50257])
@pytest.mark.parametrize("mode", ["greedy", "drawn", "chosen"])
def test_rules(cuda, dtype, kind, vocab, mode):
    counts = [6, 1, 0, 12, 25]
    logits, parents, token, q, u, u_next = inputs(cuda, counts, kind, vocab, DT[dtype], vocab + len(mode))
    if mode == "greedy":                               # some drafts are right
        cu = [sum(counts[:i]) for i in range(len(counts) + 1)]
        for i, p in enumerate(parents):
            for r in range(1, len(p)):
                if (r + i) % 3:
                    token[cu[i] + r] = int(logits[cu[i] + p[r]].argmax())
        compare(logits, counts, parents, token, None, None, None, None, 25)
        compare(logits, counts, parents, token, None, [0.0] * 5, u, u_next, 25)
    else:
        compare(logits, counts, parents, token, q if mode == "drawn" else None, [1.0, 0.7, 1.0, 1.4, 0.0], u, u_next, 25)


def test_chains_without_parents_and_short_paths(cuda):
    counts = [7, 3]
    logits, parents, token, q, u, u_next = inputs(cuda, counts, "chain", 1000, torch.float32, 5, close=0.01)
    for most in (1, 2, 3, 7, 40):
        compare(logits, counts, parents, token, q, [1.0, 1.0], u * 0.2, u_next, most, chain=True)


@pytest.mark.parametrize("mode", ["drawn", "chosen"])
def test_a_draft_that_is_the_target_stands(cuda, mode):
    """q = p: every first child is accepted (as far as fp32 holds q), and what is left of p where nothing is left is p."""
    logits, parents, token, _, u, u_next = inputs(cuda, [5, 9], "chain", 4096, torch.float32, 6, close=0.0)
    q = torch.softmax(logits.double(), -1).float()
    compare(logits, [5, 9], parents, token, q if mode == "drawn" else None, [1.0, 1.0], u * (1 - 1e-6), u_next, 9)
    one = torch.full((2, 16), -math.inf, device=cuda)
    one[:, 3] = 1.0
    q = torch.zeros((2, 16), device=cuda)
    q[:, 3] = 2.0                                      # a draft that covers p more than once: r is zero everywhere
    tok = torch.tensor([0, 3], dtype=torch.int32, device=cuda)
    _, count, said = compare(one, [2], [[-1, 0]], tok, q, [1.0], torch.full((2,), 0.9, device=cuda), torch.full((1,), 0.5, device=cuda), 2)
    assert count.tolist() == [1] and said[0, 0] == 3


def test_infinite_and_missing_logits(cuda):
    """-inf is a masked token, NaN too, infinities share the weight, and a row of nothing ends the path."""
    for dtype in DT.values():
        logits, parents, token, q, u, u_next = inputs(cuda, [4, 4, 4, 3], "chain", 300, dtype, 7)
        logits[:, ::2] = -math.inf
        logits[1, 5:50] = math.nan
        logits[4] = -math.inf
        logits[8, [7, 9, 200]] = math.inf
        logits[12] = math.nan
        for draft, temps in ((q, [1.0, 1.0, 0.8, 1.0]), (None, [1.0, 1.0, 0.8, 1.0]), (None, None)):
            _, count, said = compare(logits, [4, 4, 4, 3], parents, token, draft, temps, u, u_next, 4)
            assert int(count[1]) == 1 and said[1].tolist() == [-1] * 4 and said[3].tolist() == [-1] * 4
            assert (said[0][said[0] >= 0] % 2 == 1).all()


def test_equal_logits_take_the_lowest(cuda):
    logits = torch.zeros((3, 70000), device=cuda)
    logits[1, [69999, 40000, 40001]] = 2.0
    token = torch.tensor([9, 0, 40000], dtype=torch.int32, device=cuda)
    _, count, said = compare(logits, [3], [[-1, 0, 1]], token, None, None, None, None, 3)
    assert count.tolist() == [3] and said[0].tolist() == [0, 40000, 0]


def test_ends_of_the_random_numbers(cuda):
    """u = 0 accepts whatever has weight, the last float below one draws the last tokens; tokens outside the vocabulary and parents that are none never stand."""
    counts = [6, 6]
    logits, parents, token, q, u, u_next = inputs(cuda, counts, "tree", 999, torch.float32, 8)
    last = torch.nextafter(torch.ones(1), torch.zeros(1)).item()
    for a in (0.0, last):
        for b in (0.0, last):
            for draft in (q, None):
                compare(logits, counts, parents, token, draft, [1.0, 1.0], torch.full_like(u, a), torch.full_like(u_next, b), 6)
    token[2], token[8] = -5, 999
    parents[0][3], parents[1][4] = 70, -7
    for draft, temps in ((q, [1.0, 1.0]), (None, [1.0, 1.0]), (None, None)):
        compare(logits, counts, parents, token, draft, temps, u, u_next, 6)


@pytest.mark.parametrize("mode", ["drawn", "chosen"])
def test_tokens_follow_the_target(cuda, mode):
    """Whatever the draft, the first token has the target's distribution: frequencies over many sequences within five standard deviations."""
    from poptransformer_b200 import ops
    N, V, kids = 40000, 6, 3
    g = torch.Generator(device=cuda).manual_seed(11)
    p = torch.tensor([0.05, 0.4, 0.1, 0.25, 0.15, 0.05], device=cuda)
    q = torch.tensor([0.3, 0.1, 0.3, 0.1, 0.1, 0.1], device=cuda)
    rows = N * (1 + kids)
    logits = p.log().expand(rows, V).contiguous()
    drafts = torch.multinomial(q.expand(N, V), kids, replacement=mode == "drawn", generator=g).int()
    token = torch.cat([torch.zeros((N, 1), dtype=torch.int32, device=cuda), drafts], 1).reshape(-1).contiguous()
    parent = torch.tensor([-1] + [0] * kids, dtype=torch.int32, device=cuda).repeat(N)
    cu = torch.arange(0, rows + 1, 1 + kids, dtype=torch.int32, device=cuda)
    _, _, said, _ = ops.verify_drafts(logits, cu, token, parent, max_path=2, draft=q.expand(rows, V).contiguous() if mode == "drawn" else None, temperature=torch.ones(N, device=cuda),
                                      uniform=torch.rand(rows, generator=g, device=cuda), uniform_next=torch.rand(N, generator=g, device=cuda))
    freq = torch.bincount(said[:, 0].long(), minlength=V).double() / N
    assert ((freq - p.double()).abs() <= 5 * (p.double() * (1 - p.double()) / N).sqrt()).all(), freq


def test_captured_and_given_outputs(cuda):
    from poptransformer_b200 import ops
    counts = [5, 8, 2]
    sets = [inputs(cuda, counts, "tree", 3001, torch.float32, s) for s in (20, 21)]
    cu = torch.tensor([0, 5, 13, 15], dtype=torch.int32, device=cuda)
    temp = torch.ones(3, device=cuda)
    buf = [t.clone() for t in (sets[0][0], sets[0][2], sets[0][3], sets[0][4], sets[0][5])]
    parent = torch.tensor([p for q in sets[0][1] for p in q], dtype=torch.int32, device=cuda)
    out = ops.verify_drafts(buf[0], cu, buf[1], parent, max_path=8, draft=buf[2], temperature=temp, uniform=buf[3], uniform_next=buf[4])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        assert ops.verify_drafts(buf[0], cu, buf[1], parent, draft=buf[2], temperature=temp, uniform=buf[3], uniform_next=buf[4], out=out) is out
    for x in sets:
        for b, t in zip(buf, (x[0], x[2], x[3], x[4], x[5])):
            b.copy_(t)
        parent.copy_(torch.tensor([p for q in x[1] for p in q], dtype=torch.int32))
        graph.replay()
        got = [t.clone() for t in out]
        want = compare(x[0], counts, x[1], x[2], x[3], [1.0] * 3, x[4], x[5], 8)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("seqs", [1, 3, 20, 200])
@pytest.mark.parametrize("vocab,mode", [(1025, "drawn"), (16384, "chosen"), (130001, "drawn")])
def test_batches_share_the_gpu_in_any_way(cuda, seqs, vocab, mode):
    """The vocabulary is cut by how many sequences there are."""
    seqs = min(seqs, 2000000 // vocab)
    counts = [1 + i % 4 for i in range(seqs)]
    logits, parents, token, q, u, u_next = inputs(cuda, counts, "tree", vocab, torch.float32, seqs)
    compare(logits, counts, parents, token, q if mode == "drawn" else None, [0.9] * seqs, u, u_next, 4)


def test_a_vocabulary_whose_weights_are_not_kept(cuda):
    """More tokens than a cluster's shared memory has room for: weights are computed again where they are needed."""
    for dtype in DT.values():
        for mode in ("drawn", "chosen"):
            logits, parents, token, q, u, u_next = inputs(cuda, [4, 3], "star", 450001, dtype, 9)
            compare(logits, [4, 3], parents, token, q if mode == "drawn" else None, [1.0, 0.7], u, u_next, 4)


def test_rows_behind_the_first_512(cuda):
    logits, parents, token, q, u, u_next = inputs(cuda, [600], "star", 40, torch.float32, 10)
    best = int(logits[0].argmax())
    token[1:] = (best + 1) % 40
    token[511] = token[512] = best
    _, count, said = compare(logits, [600], parents, token, None, None, None, None, 2)
    assert count.tolist() == [2] and said[0, 0] == best
    from poptransformer_b200 import ops
    token[511] = (best + 1) % 40                        # now only the row behind them has the right token
    path, count, said, _ = ops.verify_drafts(logits, torch.tensor([0, 600], dtype=torch.int32, device=cuda), token, torch.tensor(parents[0], dtype=torch.int32, device=cuda), max_path=2)
    assert count.tolist() == [1] and said[0].tolist() == [best, -1]


def test_strided_and_unaligned_rows(cuda):
    from poptransformer_b200 import _lib, ops
    import ctypes
    logits, parents, token, q, u, u_next = inputs(cuda, [5], "chain", 777, torch.float16, 12)
    wide = torch.full((5, 801), 50.0, dtype=torch.float16, device=cuda)
    qw = torch.ones((5, 790), device=cuda)
    wide[:, 3:780], qw[:, :777] = logits, q
    temp = torch.ones(1, device=cuda)
    want = compare(logits, [5], parents, token, q, [1.0], u, u_next, 5)
    out = [torch.empty_like(t) for t in want]
    cu = torch.tensor([0, 5], dtype=torch.int32, device=cuda)
    a = _lib.VerifyArgs(1, 5, cu.data_ptr(), ops.DT_F16, 777, 801, wide.data_ptr() + 6, token.data_ptr(), None, qw.data_ptr(), 790, temp.data_ptr(), u.data_ptr(), u_next.data_ptr(), 5,
                        out[0].data_ptr(), out[1].data_ptr(), out[2].data_ptr(), None)
    _lib.check(_lib.lib().pt_verify_drafts(ctypes.byref(a), ops._stream()), "pt_verify_drafts")
    assert all(torch.equal(x, y) for x, y in zip(out, want))


@pytest.mark.parametrize("t", [1e-30, 1e-12, 1e-5, 1e-3, 50.0, 1e20])
@pytest.mark.parametrize("mode", ["drawn", "chosen"])
def test_temperatures_of_any_size(cuda, t, mode):
    """Next to 0 the largest logit has all the weight (equal ones share it), far above all tokens weigh the same."""
    for kind in ("chain", "star"):
        logits, parents, token, q, u, u_next = inputs(cuda, [5, 4], kind, 2000, torch.float32, 13)
        logits[0, [7, 1500]] = logits[0].max() + 1.0
        compare(logits, [5, 4], parents, token, q if mode == "drawn" else None, [t, t], u, u_next, 5, chain=kind == "chain")


@pytest.mark.parametrize("n", [2, 3, 5, 9, 16, 17, 40])
@pytest.mark.parametrize("vocab", [40, 2001, 40000])
def test_chains_of_any_length(cuda, n, vocab):
    """Chains whose parents are not given take a way of their own; drafts near the target, so that many stand, and greedy ones that all stand."""
    logits, parents, token, q, u, u_next = inputs(cuda, [n, 1, n // 2], "chain", vocab, torch.bfloat16, n, close=0.02)
    logits = logits[:, :vocab]
    for draft in (q, None):
        for temps in ([1.0, 0.8, 0.0], [0.0, 0.5, 2.0]):
            compare(logits, [n, 1, n // 2], parents, token, draft, temps, u * 0.3, u_next, n, chain=True)
    for i in range(1, n):
        token[i] = int(logits[i - 1].argmax())
    _, count, _ = compare(logits, [n, 1, n // 2], parents, token, None, None, None, None, n, chain=True)
    assert int(count[0]) == n
    token[n // 2] = (int(token[n // 2]) + 1) % vocab
    logits[n // 3] = -math.inf
    compare(logits, [n, 1, n // 2], parents, token, None, None, None, None, n, chain=True)
    compare(logits, [n, 1, n // 2], parents, token, q, [1.0] * 3, u * 0.1, u_next, max(1, n // 2), chain=True)
