"""Caches of eight bits: batches of thousands of rows, rows that lie anywhere, bytes of any kind behind a sequence's end, launches that share a workspace (formulas and tolerances: kv8_util)."""
import math

import pytest
import torch

import kv8_util as ku

pytestmark = pytest.mark.gpu
DT = ku.DT


def append(s, interleaved=False, q=True):
    from poptransformer_b200 import ops
    q_out = torch.full((s.qkv.shape[0], s.q_cols), 7.0, dtype=s.dtype, device=s.device) if q else None
    ops.kv8_append(s.view, s.qkv, s.ld, s.cache, s.heads, rope=s.rope, rope_dims=s.rot, interleaved=interleaved, q_out=q_out, q_out_ld=s.q_cols, error_flag=s.flag)
    return q_out


def expected(s, interleaved):
    """As kv8_util.appended, for many tokens at once."""
    qkv, rope = s.qkv[:s.n_tok].float(), s.rope
    seq = s.tok_seq[:s.n_tok].long()
    pos = s.start[seq].long() + torch.arange(s.n_tok, device=s.device) - s.cu[seq].long()
    q = ku.rotate(qkv[:, :s.q_cols].reshape(s.n_tok, -1, s.dim), rope, pos, s.rot, interleaved).flatten(1)
    k = ku.rotate(qkv[:, s.q_cols:s.q_cols + s.n_kv * s.dim].reshape(s.n_tok, -1, s.dim), rope, pos, s.rot, interleaved)
    v = qkv[:, s.q_cols + s.n_kv * s.dim:s.width].reshape(s.n_tok, -1, s.vdim)
    page, place = s.page_table[s.slot[seq].long(), pos // s.page].long(), pos % s.page
    pool, scales = s.pool.view(torch.uint8).clone(), s.scales.clone()
    split = s.n_kv * s.page * s.dim
    flat = pool.flatten(1)
    for which, y, block, width in ((0, k, slice(0, split), s.dim), (1, v, slice(split, None), s.vdim)):
        by, sc = ku.to_bytes(y, s.fmt)
        part = flat[:, block].unflatten(1, (s.n_kv, s.page, width)).clone()
        part[page, :, place] = by.view(torch.uint8)
        flat[:, block] = part.flatten(1)
        scales[page, which, :, place] = sc
    return q.to(s.dtype), pool, scales


@pytest.mark.parametrize("n_kv,qpk,dim,vdim,rot,interleaved", [(8, 4, 128, 128, 128, False), (1, 3, 128, 128, 64, True), (3, 1, 64, 64, 32, False), (5, 2, 256, 256, 256, True), (2, 7, 80, 80, 16, False),
                                                             (1, 1, 96, 160, 96, False), (4, 2, 48, 32, 0, False)])
@pytest.mark.parametrize("dtype,fmt", [("bf16", "int8"), ("fp16", "e4m3"), ("fp32", "int8"), ("fp32", "e4m3")])
def test_thousands_of_tokens_are_appended(cuda, n_kv, qpk, dim, vdim, rot, interleaved, dtype, fmt):
    s = ku.batch([2500, 1, 0, 1777], [3, 900, 5, 64], DT[dtype], DT[fmt], n_kv=n_kv, qpk=qpk, dim=dim, vdim=vdim, rot=rot, seed=dim, spare_rows=2)
    q, pool, scales = expected(s, interleaved)
    got = append(s, interleaved)
    assert torch.equal(got[:s.n_tok], q) and (got[s.n_tok:] == 7).all()
    assert torch.equal(s.pool.view(torch.uint8), pool) and torch.equal(s.scales.nan_to_num(-1.0), scales.nan_to_num(-1.0)) and s.flag.item() == 0
    s.scales.fill_(math.nan)
    scales2 = s.scales.clone()
    assert append(s, interleaved, q=False) is None           # (keys and values alone: other rows are a lane's neighbours)
    seen = ~s.scales.isnan()
    assert torch.equal(s.scales[seen], scales[seen]) and seen.sum() == 2 * n_kv * s.n_tok and torch.equal(s.pool.view(torch.uint8), pool) and scales2.isnan().all()


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("interleaved,inverse", [(False, False), (True, True)])
def test_thousands_of_rows_are_rotated(cuda, dtype, interleaved, inverse):
    from poptransformer_b200 import ops
    for heads, dim, rot in ((34, 128, 64), (5, 80, 80), (3, 256, 192)):
        x = torch.randn((3001, heads * dim), device=cuda).to(DT[dtype])
        rope, pos = ops.rope_table(5000, rot, device=cuda), (torch.arange(3001, device=cuda) * 7 % 5000).int()
        want = ku.rotate(x.float().view(3001, heads, dim), rope, pos, rot, interleaved, inverse).flatten(1).to(DT[dtype])
        assert torch.equal(ops.rotary(x, heads, dim, rope, pos, out=torch.empty_like(x), interleaved=interleaved, inverse=inverse), want)


@pytest.mark.parametrize("n_tok", [1025, 2300])
def test_more_tokens_than_a_launch_plans(cuda, n_tok):
    s = ku.cached(ku.batch([1] * n_tok, [(i * 13) % 90 for i in range(n_tok)], torch.bfloat16, torch.int8, dim=64, n_kv=2, qpk=2, seed=1))
    ku.check(s, s.qkv, ku.attend(s, s.qkv))


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_rows_on_any_address(cuda, dtype):
    """Queries and outputs with odd strides and beginnings, against the same call on whole rows."""
    from poptransformer_b200 import ops
    s = ku.cached(ku.batch([1, 1, 1], [700, 33, 2000], DT[dtype], torch.int8, dim=128, n_kv=2, qpk=3, seed=2))
    want = ku.attend(s, s.qkv)
    ku.check(s, s.qkv, want)
    ld = s.qkv.shape[1] + 3
    room = torch.empty(3 * ld + 1, dtype=s.dtype, device=cuda)
    q = room[1:]
    for r in range(3):
        q[r * ld:r * ld + s.qkv.shape[1]] = s.qkv[r]
    out = torch.full((3 * 1001 + 1,), 7.0, dtype=s.dtype, device=cuda)
    ops.kv8_attn(s.view, q, ld, s.cache, out[1:], 1001, s.heads, s.scale, workspace=ops.kv8_attn_workspace(3, s.heads, s.n_kv, 128))
    got = out[1:].view(3, 1001)
    assert torch.equal(got[:, :768], want) and (got[:, 768:] == 7).all() and out[0] == 7


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("plain", [False, True])
@pytest.mark.parametrize("dim,page", [(128, 64), (64, 16), (256, 48)])
def test_bytes_behind_the_end_are_not_seen(cuda, fmt, dtype, plain, dim, page):
    """Bytes that are NaN in E4M3 (and the largest in int8) and NaN scales behind every sequence's own position and in front of its window."""
    s = ku.cached(ku.batch([1, 1, 1, 1], [100, 0, 31, 700], DT[dtype], DT[fmt], dim=dim, page=page, n_kv=2, qpk=2, seed=3))
    want = ku.attend(s, s.qkv, plain=plain).clone(), ku.attend(s, s.qkv, window=40, plain=plain).clone()
    for window, y in ((0, want[0]), (40, want[1])):
        for i in range(4):
            n = s.starts[i] + 1
            first = max(0, n - window) if window else 0
            for p, page_id in enumerate(s.table_host[s.slot_host[i]][:-(-n // page)]):
                rows = [r for r in range(page) if not first <= p * page + r < n]
                s.scales[page_id][:, :, rows] = math.nan
                flat = s.pool.view(torch.uint8)[page_id].view(2, s.n_kv, page, dim)
                flat[:, :, rows] = 0x7f
        assert torch.equal(ku.attend(s, s.qkv, window=window, plain=plain), y) and not y.isnan().any()


def test_e4m3_bytes_that_are_nan_read_as_nan(cuda):
    for plain in (False, True):
        s = ku.cached(ku.batch([1, 1], [100, 90], torch.bfloat16, torch.float8_e4m3fn, dim=64, n_kv=2, qpk=2, seed=4))
        page = s.table_host[s.slot_host[0]][0]
        ku.part(s, s.pool.view(torch.uint8), page, 1)[1, 7, 3] = 0x7f
        out = ku.attend(s, s.qkv, plain=plain).view(2, 4, 64)
        assert out[0, 2:, 3].isnan().all() and out.isnan().sum() == 2


def test_graphs_and_batches_of_other_sizes_share_a_workspace(cuda):
    from poptransformer_b200 import ops
    batches = [ku.cached(ku.batch([1] * n, [length] * n, torch.bfloat16, fmt, dim=dim, n_kv=2, qpk=qpk, seed=n))
               for n, length, fmt, dim, qpk in ((1, 9000, torch.int8, 128, 4), (40, 700, torch.float8_e4m3fn, 128, 12), (3, 5000, torch.int8, 64, 2), (2, 3000, torch.int8, 256, 1))]
    ws = ops.kv8_attn_workspace(40, 24, 2, 256)
    outs = [torch.empty((s.n_tok, s.heads * s.vdim), dtype=s.dtype, device=cuda) for s in batches]
    want = [ku.attend(s, s.qkv).clone() for s in batches]
    graphs = []
    for s, o in zip(batches, outs):
        ku.attend(s, s.qkv, out=o, workspace=ws)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ku.attend(s, s.qkv, out=o, workspace=ws)
        graphs.append(g)
    for order in ((0, 1, 2, 3), (3, 1, 0, 2, 1, 1, 0)):
        for o in outs:
            o.fill_(7.0)
        for i in order:
            graphs[i].replay()
        for o, y in zip(outs, want):
            assert torch.equal(o, y)
    for s, o, y in zip(batches, outs, want):
        ku.check(s, s.qkv, o)


def test_long_contexts(cuda):
    """Parts of many blocks come together, whatever else the launch holds."""
    for dtype, fmt, dim in (("bf16", "int8", 128), ("fp32", "e4m3", 64), ("fp16", "int8", 256)):
        s = ku.cached(ku.batch([1, 1, 1], [40000, 17, 9001], DT[dtype], DT[fmt], dim=dim, n_kv=1, qpk=3, seed=5))
        ku.check(s, s.qkv, ku.attend(s, s.qkv))


@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_queries_that_are_no_numbers(cuda, value, fmt):
    """Such a head's output is NaN, the others' are not."""
    for plain in (False, True):
        s = ku.cached(ku.batch([1, 1], [100, 700], torch.float32, DT[fmt], dim=64, n_kv=2, qpk=2, seed=6))
        want = ku.attend(s, s.qkv, plain=plain).clone().view(2, 4, 64)
        s.qkv[0, 64 + 5] = value
        out = ku.attend(s, s.qkv, plain=plain).view(2, 4, 64)
        assert out[0, 1].isnan().all()
        want[0, 1] = out[0, 1] = 0
        assert torch.equal(out, want)


@pytest.mark.parametrize("plain", [False, True])
def test_outputs_in_the_place_of_queries(cuda, plain):
    from poptransformer_b200 import ops
    for qpk, lengths in ((4, [5000, 3, 700]), (12, [100, 9000])):
        s = ku.cached(ku.batch([1] * len(lengths), lengths, torch.bfloat16, torch.int8, dim=128, n_kv=2, qpk=qpk, seed=7))
        want = ku.attend(s, s.qkv, plain=plain).clone()
        rows = s.qkv.clone()
        ws = ops.kv8_attn_workspace(len(lengths), s.heads, 2, 128)
        ops.kv8_attn(s.view, rows, s.ld, s.cache, rows, s.ld, s.heads, s.scale, workspace=ws, plain=plain)
        assert torch.equal(rows[:, :s.q_cols], want) and torch.equal(rows[:, s.q_cols:], s.qkv[:, s.q_cols:])


def test_rotation_into_other_columns_of_the_same_rows(cuda):
    from poptransformer_b200 import ops
    wide = torch.randn((70, 600), device=cuda)
    before, rope, pos = wide.clone(), ops.rope_table(70, 64, device=cuda), torch.arange(70, dtype=torch.int32, device=cuda)
    ops.rotary(wide[:, 16:272], 4, 64, rope, pos, out=wide[:, 300:556])
    want = ku.rotate(before[:, 16:272].cpu().reshape(70, 4, 64), rope.cpu(), pos.cpu(), 64, False).flatten(1)
    assert torch.equal(wide[:, 300:556].cpu(), want) and torch.equal(wide[:, :300], before[:, :300]) and torch.equal(wide[:, 556:], before[:, 556:])


def test_a_batch_without_tokens(cuda):
    """Nothing is appended or attended to; what is cached can be unpacked."""
    from poptransformer_b200 import ops
    s = ku.batch([0, 0], [70, 0], torch.bfloat16, torch.int8, dim=64, seed=8)
    pool, scales = s.pool.clone(), s.scales.clone()
    assert append(s).shape[0] == 0 and ku.attend(s, s.qkv).shape[0] == 0
    into = ops.PagedKVCache(2, s.n_kv, 64, 128, 64, cuda, dtype=torch.bfloat16)
    ops.kv8_unpack(s.view, s.cache, into, error_flag=s.flag)
    x = ku.history(s, 0, 70, 0).float().bfloat16()
    pages = into.page_table[s.slot_host[0]].long()
    assert torch.equal(into.pool[pages, 0].transpose(0, 1).flatten(1, 2)[:, :70], x) and (into.pool[pages, 0].transpose(0, 1).flatten(1, 2)[:, 70:] == 0).all()
    assert torch.equal(s.pool, pool) and torch.equal(s.scales.nan_to_num(-1), scales.nan_to_num(-1)) and s.flag.item() == 0


@pytest.mark.parametrize("plain", [False, True])
@pytest.mark.parametrize("fmt", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 16), (128, 32), (256, 16), (96, 48)])
def test_pages_in_front_of_the_window_may_be_gone(cuda, dim, page, fmt, plain):
    """Pages whose positions all lie in front of every token's window are negative: the same outputs, and no error; with one page more gone there is one."""
    counts, starts, window = [1, 1, 3, 1], [300, 60, 777, 1023], 50
    s = ku.cached(ku.batch(counts, starts, torch.bfloat16, fmt, dim=dim, page=page, seed=dim + page))
    want = ku.attend(s, s.qkv, window=window, plain=plain).clone()
    gone = [max(0, n - window + 1) // page for n in starts]
    for i, n in enumerate(gone):
        s.page_table[s.slot_host[i], :n] = -1
    assert torch.equal(ku.attend(s, s.qkv, window=window, plain=plain), want) and s.flag.item() == 0
    s.page_table[s.slot_host[2], gone[2]] = -1
    ku.attend(s, s.qkv, window=window, plain=plain)
    assert s.flag.item() == 12
