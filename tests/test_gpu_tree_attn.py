"""Attention for trees of drafted tokens against the formula in 64 bits (tolerances: tree_util.reference)."""
import pytest
import torch

import tree_util as tu

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("kind", ["chain", "tree", "star", "roots"])
@pytest.mark.parametrize("plain", [False, True])
def test_trees(cuda, dtype, kind, plain):
    s = tu.batch([5, 1, 17, 33], [300, 0, 63, 129], kind, dtype=DT[dtype], dim=128, n_kv=2, qpk=4, rot=128, seed=1)
    before = s.cache.pool.clone()
    tu.check(s, before, tu.run(s, plain=plain))
    assert s.flag.item() == 0


# one token, tile borders, no context, contexts of one, one key tile and its neighbours, and a run over several blocks
@pytest.mark.parametrize("n,start", [(1, 0), (1, 1), (2, 0), (3, 62), (1, 63), (1, 127), (1, 128), (64, 64), (65, 31), (128, 1), (256, 0), (256, 77), (8, 1023), (40, 5000)])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_lengths(cuda, n, start, dtype):
    s = tu.batch([n], [start], dtype=DT[dtype], dim=64, n_kv=1, qpk=2, seed=n + start)
    before = s.cache.pool.clone()
    tu.check(s, before, tu.run(s))


@pytest.mark.parametrize("n_kv,qpk,dim,vdim,page,dtype", [(1, 1, 64, 64, 64, "bf16"), (2, 16, 128, 128, 64, "fp16"), (8, 4, 128, 128, 16, "bf16"), (3, 5, 72, 72, 64, "bf16"), (2, 3, 96, 64, 64, "bf16"),
                                                          (2, 2, 128, 48, 32, "fp16"), (1, 7, 20, 33, 7, "bf16"), (2, 2, 80, 80, 100, "fp16"), (1, 4, 256, 256, 64, "bf16"),
                                                          (2, 1, 256, 130, 64, "fp32"), (5, 3, 17, 5, 3, "fp32"), (1, 32, 64, 64, 128, "bf16"), (4, 8, 8, 8, 64, "fp16")])
def test_heads_and_pages(cuda, n_kv, qpk, dim, vdim, page, dtype):
    s = tu.batch([9, 26], [200, 515], n_kv=n_kv, qpk=qpk, dim=dim, vdim=vdim, page=page, dtype=DT[dtype], seed=dim + page, rot=dim // 2 // 2 * 2)
    before = s.cache.pool.clone()
    tu.check(s, before, tu.run(s))


@pytest.mark.parametrize("window", [1, 2, 5, 64, 65, 200, 100000])
@pytest.mark.parametrize("dtype,plain", [("bf16", False), ("bf16", True), ("fp16", False), ("fp32", False)])
def test_windows(cuda, window, dtype, plain):
    s = tu.batch([12, 30, 3], [300, 2, 64], dtype=DT[dtype], dim=64, seed=window)
    before = s.cache.pool.clone()
    tu.check(s, before, tu.run(s, window=window, plain=plain), window=window)
    s = tu.batch([100], [90], "chain", dtype=DT[dtype], dim=64, seed=window)
    before = s.cache.pool.clone()
    tu.check(s, before, tu.run(s, parent=None, window=window, plain=plain), window=window, chain=True)


@pytest.mark.parametrize("dtype,plain", [("bf16", False), ("fp16", False), ("fp16", True), ("fp32", False)])
def test_softcap_and_scale(cuda, dtype, plain):
    s = tu.batch([20, 7], [150, 700], dtype=DT[dtype], dim=128, seed=3)
    s.scale = 0.7                                     # scores far beyond the cap
    before = s.cache.pool.clone()
    tu.check(s, before, tu.run(s, softcap=5.0, plain=plain), softcap=5.0)
    s.scale = -0.05
    before = s.cache.pool.clone()
    tu.check(s, before, tu.run(s, plain=plain))


@pytest.mark.parametrize("dtype,plain", [("bf16", False), ("bf16", True), ("fp16", False), ("fp32", False)])
def test_unequal_batches_and_empty_sequences(cuda, dtype, plain):
    """Sequences without new tokens, slots in any order, rows behind the last sequence, padding columns of the output."""
    s = tu.batch([0, 6, 0, 0, 31, 2, 0], [100, 1000, 5, 0, 10, 0, 64], dtype=DT[dtype], dim=64, n_kv=2, qpk=3, seed=5, spare_rows=4, slots=11)
    before = s.cache.pool.clone()
    width = s.heads * s.vdim
    out = torch.full((s.n_tok + 4, width + 10), 7.0, dtype=s.dtype, device=s.device)
    tu.run(s, out=out, out_ld=width + 10, out_cols=width + 6, plain=plain)
    tu.check(s, before, out)
    assert (out[:s.n_tok, width:width + 6] == 0).all() and (out[:s.n_tok, width + 6:] == 7).all() and (out[s.n_tok:] == 7).all()
    assert s.flag.item() == 0


@pytest.mark.parametrize("n_seq", [1, 33, 1024])
def test_many_sequences(cuda, n_seq):
    counts, starts = [1 + i % 4 for i in range(n_seq)], [(i * 37) % 300 for i in range(n_seq)]
    s = tu.batch(counts, starts, dtype=torch.bfloat16, dim=64, n_kv=1, qpk=2, seed=6)
    before = s.cache.pool.clone()
    tu.check(s, before, tu.run(s))


def test_strided_rows(cuda):
    """Row strides beyond the heads, in units that are no multiples of 16 bytes too."""
    for dtype, extra in ((torch.bfloat16, 8), (torch.bfloat16, 3), (torch.float32, 1), (torch.float16, 2)):
        s = tu.batch([7, 20], [130, 64], dtype=dtype, dim=64, seed=7)
        wide = torch.full((s.n_tok, s.ld + extra), 3.0, dtype=dtype, device=s.device)
        wide[:, :s.ld] = s.qkv
        before = s.cache.pool.clone()
        rows, s.qkv, ld = s.qkv, wide, s.ld
        s.ld = ld + extra
        out = tu.run(s)
        s.qkv, s.ld = rows, ld
        tu.check(s, before, out)


@pytest.mark.parametrize("dtype,plain", [("bf16", False), ("bf16", True), ("fp16", False), ("fp32", False)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_what_nobody_sees_does_not_matter(cuda, dtype, plain, bad):
    """Positions behind a sequence's last, other pages and (with a window) positions behind it hold infinities and NaN; so does a sibling."""
    s = tu.batch([6, 9], [200, 70], "star", dtype=DT[dtype], dim=64, seed=8)
    flat = s.cache.pool
    live = torch.zeros(flat.shape[0], s.page, dtype=torch.bool, device=s.device)
    for i in range(2):
        for j in range(s.starts[i]):
            if j > s.starts[i] - 100:
                live[s.table[s.slot[i]][j // s.page], j % s.page] = True
    flat.masked_fill_(~live[:, None, None, :, None], bad)
    before = flat.clone()
    out = tu.run(s, window=100, plain=plain)
    tu.check(s, before, out, window=100)
    # the second token of the first sequence is a leaf: its key and value reach its own row alone
    s2 = tu.batch([6, 9], [200, 70], "star", dtype=DT[dtype], dim=64, seed=8)
    want = tu.run(s2, plain=plain)
    s2.qkv[1, s2.heads * 64:] = bad
    got = tu.run(s2, plain=plain)
    rows = [r for r in range(15) if r != 1]
    assert torch.equal(got[rows], want[rows])
    assert not torch.isfinite(got[1]).any()


def test_same_bits_on_every_run_and_workspace_contents_do_not_matter(cuda):
    from poptransformer_b200 import ops
    s = tu.batch([30, 5], [3000, 900], dtype=torch.bfloat16, dim=128, n_kv=4, qpk=4, seed=9, rot=128)
    ws = ops.tree_attn_workspace(2, 30, s.heads, s.n_kv, s.vdim)
    first = tu.run(s, workspace=ws.fill_(0)).clone()
    for fill in (255, 127):
        assert torch.equal(tu.run(s, workspace=ws.fill_(fill)), first)


def test_captured_with_lengths_that_grow(cuda):
    """A captured call reads lengths, pages and trees on the device: replayed after they changed, on a stream of its own."""
    from poptransformer_b200 import ops
    s = tu.batch([6, 11], [120, 700], dtype=torch.bfloat16, dim=128, n_kv=2, qpk=4, seed=10, rot=64)
    t = tu.batch([11, 6], [640, 33], dtype=torch.bfloat16, dim=128, n_kv=2, qpk=4, seed=11, rot=64, max_len=s.max_len)
    ws = ops.tree_attn_workspace(2, 11, s.heads, s.n_kv, s.vdim)
    out = torch.zeros((17, s.heads * s.vdim), dtype=s.dtype, device=cuda)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    pool = torch.zeros((max(s.cache.pool.shape[0], t.cache.pool.shape[0]),) + tuple(s.cache.pool.shape[1:]), dtype=s.dtype, device=cuda)
    own = s.cache.pool
    pool[:own.shape[0]] = own
    s.cache.pool = pool
    with torch.cuda.stream(side):
        tu.run(s, out=out, out_ld=out.shape[1], workspace=ws, most=11)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            tu.run(s, out=out, out_ld=out.shape[1], workspace=ws, most=11)
        for x in (s, t):
            s.qkv.copy_(x.qkv); s.parent.copy_(x.parent); s.cu_d.copy_(x.cu_d); s.start_d.copy_(x.start_d); s.slot_d.copy_(x.slot_d); s.cache.page_table.copy_(x.cache.page_table)
            source = own if x is s else x.cache.pool
            pool[:source.shape[0]] = source
            before = pool.clone()
            graph.replay()
            x.cache.pool = pool
            tu.check(x, before, out)
    side.synchronize()


def test_flags(cuda):
    """What the host cannot see: too many tokens, positions without pages, parents that are none."""
    s = tu.batch([5, 9, 3], [100, 20, 64], dtype=torch.bfloat16, dim=64, seed=12)
    before = s.cache.pool.clone()
    out = tu.run(s, most=6)                            # the second sequence has 9
    assert s.flag.item() == 14 and (out[5:14] == 7).all()
    assert torch.equal(tu._pages(s, s.cache.pool, 1, 29)[0], tu._pages(s, before, 1, 29)[0])
    keep = [0, 1, 2, 3, 4, 14, 15, 16]
    ref, tol, _ = tu.reference(s, before)
    assert ((out.double() - ref).abs()[keep] <= tol[keep]).all()
    s.flag.zero_()
    s.start_d[0] = s.max_len - 4                       # five tokens do not fit
    out = tu.run(s)
    assert s.flag.item() == 12 and (out[:5] == 7).all()
    s.start_d[0] = -1
    s.flag.zero_()
    out = tu.run(s)
    assert s.flag.item() == 12 and (out[:5] == 7).all()
    s.start_d[0] = 100
    s.flag.zero_()
    for wrong in (3, 4, -2, 1 << 30):                  # token 3: itself, a later one, below -1, far outside; it then follows the context
        s.parent[3] = wrong
        s.parents[0][3] = -1
        before = s.cache.pool.clone()
        out = tu.run(s)
        assert s.flag.item() == 14
        tu.check(s, before, out)


@pytest.mark.parametrize("dtype,plain", [("bf16", False), ("fp16", False), ("fp16", True), ("fp32", False)])
def test_a_scale_of_zero_weighs_all_that_is_seen_alike(cuda, dtype, plain):
    s = tu.batch([20, 7], [150, 700], dtype=DT[dtype], dim=64, seed=13)
    s.scale = 0.0
    before = s.cache.pool.clone()
    tu.check(s, before, tu.run(s, plain=plain))
    before = s.cache.pool.clone()
    tu.check(s, before, tu.run(s, softcap=5.0, window=50, plain=plain), softcap=5.0, window=50)


def test_two_captured_calls_at_once(cuda):
    """Graphs on two streams, each with a workspace of its own, many times over: the same bits as one after the other."""
    from poptransformer_b200 import ops
    sets = [tu.batch([9, 20], [900, 77], dtype=torch.bfloat16, dim=128, n_kv=2, qpk=4, seed=14, rot=128), tu.batch([31], [2000], dtype=torch.float16, dim=64, n_kv=4, qpk=2, seed=15),
            tu.batch([12, 3], [300, 40], dtype=torch.float32, dim=80, n_kv=2, qpk=2, seed=16)]
    want = [tu.run(s).clone() for s in sets]
    runs = []
    for s in sets:
        stream, out = torch.cuda.Stream(), torch.zeros((s.n_tok, s.heads * s.vdim), dtype=s.dtype, device=cuda)
        ws = ops.tree_attn_workspace(len(s.counts), max(s.counts), s.heads, s.n_kv, s.vdim)
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            tu.run(s, out=out, out_ld=out.shape[1], workspace=ws)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                for _ in range(5):
                    tu.run(s, out=out, out_ld=out.shape[1], workspace=ws)
        runs.append((stream, graph, out, ws))
    torch.cuda.synchronize()
    for _ in range(4):
        for stream, graph, out, _ in runs:
            out.zero_()
        torch.cuda.synchronize()
        for stream, graph, out, _ in runs:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for (stream, graph, out, _), w, s in zip(runs, want, sets):
            assert torch.equal(out, w) and s.flag.item() == 0


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("counts,starts", [([63, 40], [40000, 20001]), ([33, 64, 5], [25000, 31000, 70])])
def test_several_row_tiles_over_the_same_long_cache(cuda, dtype, counts, starts):
    """Items of several blocks each, two row tiles of tensor cores or eight of fp32 to a kv head."""
    s = tu.batch(counts, starts, dtype=DT[dtype], dim=64, n_kv=4, qpk=4, rot=64, seed=17)
    before = s.cache.pool.clone()
    tu.check(s, before, tu.run(s))


@pytest.mark.parametrize("dtype,plain", [("bf16", False), ("fp32", True)])
def test_rows_that_the_batch_has_not(cuda, dtype, plain):
    """A sequence that ends behind the batch's rows is left alone, and said."""
    s = tu.batch([5, 9], [100, 20], dtype=DT[dtype], dim=64, seed=18)
    before = s.cache.pool.clone()
    s.cu_d[2] = s.n_tok + 3
    out = tu.run(s, most=12, plain=plain)
    assert s.flag.item() == 14 and (out[5:] == 7).all()
    assert torch.equal(tu._pages(s, s.cache.pool, 1, 29)[0], tu._pages(s, before, 1, 29)[0])
    ref, tol, _ = tu.reference(s, before)
    assert ((out.double() - ref).abs()[:5] <= tol[:5]).all()
