"""Rotation, caches of eight bits and the attention that reads them, against the formulas (tolerances: kv8_util.reference; rows that are rounded: equal bits)."""
import math

import pytest
import torch

import kv8_util as ku

pytestmark = pytest.mark.gpu
DT = ku.DT


# ------------------------------------------------------------------------------------------ rotation
# (heads, dim, rot): whole and odd heads, a part of the head, pairs that no vector holds
SIZES = [(4, 128, 128), (3, 64, 32), (1, 80, 80), (5, 80, 20), (2, 256, 64), (7, 33, 6), (2, 96, 96), (1, 2, 2), (34, 128, 64), (3, 48, 16)]


@pytest.mark.parametrize("heads,dim,rot", SIZES)
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("inverse", [False, True])
def test_rotary(cuda, heads, dim, rot, dtype, interleaved, inverse):
    from poptransformer_b200 import ops
    gen = torch.Generator().manual_seed(dim + rot)
    for rows in (1, 37):
        x = torch.randn((rows, heads * dim), generator=gen).to(DT[dtype]).to(cuda)
        rope = ops.rope_table(500, rot, device=cuda)
        pos = torch.randint(0, 500, (rows,), generator=gen, dtype=torch.int32).to(cuda)
        want = ku.rotate(x.cpu().float().view(rows, heads, dim), rope.cpu(), pos.cpu(), rot, interleaved, inverse).flatten(1).to(DT[dtype])
        out = ops.rotary(x, heads, dim, rope, pos, out=torch.empty_like(x), interleaved=interleaved, inverse=inverse)
        assert torch.equal(out.cpu(), want)
        assert ops.rotary(x, heads, dim, rope, pos, interleaved=interleaved, inverse=inverse) is x and torch.equal(x.cpu(), want)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("first,pad", [(0, 8), (3, 5), (16, 0)])
def test_rotary_of_a_part_of_wider_rows(cuda, dtype, first, pad):
    from poptransformer_b200 import ops
    wide = torch.randn((50, first + 4 * 64 + pad), device=cuda).to(DT[dtype])
    before = wide.clone()
    rope, pos = ops.rope_table(60, 64, device=cuda), torch.arange(50, dtype=torch.int32, device=cuda)
    ops.rotary(wide[:, first:first + 256], 4, 64, rope, pos)
    want = before.clone()
    want[:, first:first + 256] = ku.rotate(before[:, first:first + 256].cpu().float().reshape(50, 4, 64), rope.cpu(), pos.cpu(), 64, False).flatten(1).to(DT[dtype]).to(cuda)
    assert torch.equal(wide, want)


def test_rotary_positions_outside_the_table(cuda):
    from poptransformer_b200 import ops
    x, flag = torch.randn((4, 64), device=cuda), ku.ints([0])
    before, rope = x.clone(), ops.rope_table(10, 64, device=cuda)
    ops.rotary(x, 1, 64, rope, ku.ints([-1, 3, 10, 9]), error_flag=flag)
    assert flag.item() == 12 and torch.equal(x[[0, 2]], before[[0, 2]]) and not torch.equal(x[[1, 3]], before[[1, 3]])
    assert ops.rotary(x[:0], 1, 64, rope, ku.ints([])).shape == (0, 64)


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_gradient(cuda, interleaved):
    """The gradient of a sum over outputs is the rotation by negative angles: against the transpose in 64 bits, and against differences (the rotation is linear, so they are exact up to rounding)."""
    from poptransformer_b200 import ops
    rows, heads, dim, rot = 5, 3, 48, 32
    x, g = torch.randn((rows, heads * dim), device=cuda), torch.randn((rows, heads * dim), device=cuda)
    rope, pos = ops.rope_table(4000, rot, scaling=dict(kind="ramp", factor=4.0, original=1000), device=cuda), ku.ints([0, 1, 77, 999, 3999])
    got = ops.rotary(g, heads, dim, rope, pos, out=torch.empty_like(g), interleaved=interleaved, inverse=True)
    xd = x.double().requires_grad_()
    y = ku.rotate(xd.view(rows, heads, dim) * 1.0, rope, pos, rot, interleaved).flatten(1)
    want, = torch.autograd.grad((y * g.double()).sum(), xd)
    # two products and a sum of them in 32 bits, of factors below 1.14 in magnitude
    tol = 4 * 2.0 ** -24 * 1.14 * (g.abs().amax() * 2).double()
    assert ((got.double() - want).abs() <= tol).all()
    for col in (0, 7, 16, 31, 40, 100):
        step = torch.zeros_like(x)
        step[:, col] = 1.0
        up, down = (ops.rotary(x + d, heads, dim, rope, pos, out=torch.empty_like(x), interleaved=interleaved).double() for d in (step, -step))
        slope = ((up - down) / 2 * g.double()).sum(-1)
        # each of the two outputs that move is off by 3 roundings of values below 1.14 (|x| + 1) sqrt 2
        assert ((slope - got[:, col].double()).abs() <= 2 * 4 * 2.0 ** -24 * 1.62 * (x.abs().amax() + 1).double() * g.abs().amax().double() + 2.0 ** -20).all()


# ------------------------------------------------------------------------------------------ appending
def check_append(s, interleaved=False, n_head=None, q_in_place=False):
    from poptransformer_b200 import ops
    pool, scales, q = ku.appended(s, interleaved)
    rows = s.qkv.clone()
    q_out = rows if q_in_place else torch.full((rows.shape[0], s.q_cols + 3), 7.0, dtype=s.dtype, device=s.device)
    ops.kv8_append(s.view, rows, s.ld, s.cache, s.heads, rope=s.rope, rope_dims=s.rot, interleaved=interleaved, q_out=q_out, q_out_ld=q_out.shape[1], error_flag=s.flag)
    assert torch.equal(s.pool.view(torch.uint8).cpu(), pool)
    assert torch.equal(s.scales.cpu().nan_to_num(-1.0), scales.nan_to_num(-1.0))
    for i, n in enumerate(s.counts):
        r = slice(s.cu_host[i], s.cu_host[i] + n)
        if s.starts[i] + n <= s.max_len:
            assert torch.equal(q_out[r, :s.q_cols].cpu(), q[r].to(s.dtype))
        else:
            assert torch.equal(q_out[r], s.qkv[r] if q_in_place else torch.full_like(q_out[r], 7.0))
    if q_in_place:
        assert torch.equal(rows[:, s.q_cols:], s.qkv[:, s.q_cols:]) and torch.equal(rows[s.n_tok:], s.qkv[s.n_tok:])
    else:
        assert (q_out[:, s.q_cols:] == 7).all() and (q_out[s.n_tok:] == 7).all() and torch.equal(rows.nan_to_num(), s.qkv.nan_to_num())
    return s


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("interleaved", [False, True])
def test_append(cuda, fmt, dtype, interleaved):
    s = check_append(ku.batch([5, 0, 1, 70, 1], [300, 12, 63, 0, 5], DT[dtype], DT[fmt], dim=128, rot=128, seed=1, spare_rows=3, slots=9), interleaved)
    assert s.flag.item() == 0
    check_append(ku.batch([3, 9], [0, 100], DT[dtype], DT[fmt], dim=128, rot=64, seed=2, pad=8), interleaved, q_in_place=True)


@pytest.mark.parametrize("n_kv,qpk,dim,vdim,page,rot,pad", [(1, 1, 64, 64, 16, 64, 0), (3, 5, 80, 80, 64, 20, 0), (2, 3, 96, 64, 7, 96, 8), (1, 2, 33, 5, 3, 6, 1), (5, 1, 256, 256, 64, 128, 0),
                                                            (2, 8, 80, 128, 1, 80, 3), (12, 1, 64, 64, 128, 0, 0), (1, 1, 1, 1, 5, 0, 0), (2, 2, 16, 48, 64, 16, 16)])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_append_heads_and_pages(cuda, n_kv, qpk, dim, vdim, page, rot, pad, fmt):
    for dtype in (torch.bfloat16, torch.float32):
        check_append(ku.batch([4, 13, 1], [50, 7, 0], dtype, DT[fmt], n_kv=n_kv, qpk=qpk, dim=dim, vdim=vdim, page=page, rot=rot, pad=pad, seed=dim), interleaved=dim % 3 == 0)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_append_rows_that_no_byte_holds(cuda, fmt):
    """Zeros, the smallest and largest numbers, infinities and NaN: the row alone reads as NaN; tiny rows are kept relative to 2^-64."""
    s = ku.batch([10], [3], torch.float32, DT[fmt], n_kv=1, qpk=1, dim=64, seed=3)
    k = s.qkv[:, 64:128]
    k[0] = 0.0
    k[1, 5] = math.inf
    k[2, 63] = math.nan
    k[3] *= 1e-30
    k[4] = 1e-45
    k[5, 1] = 2.0 ** 64
    k[6, 2] = -3e38
    k[7] = -0.0
    k[8, 9] = 2.0 ** -64
    s.qkv[9, 128:] = -math.inf
    check_append(s)
    page = s.table_host[0][0]
    nan = s.scales[page, 0, 0, 3:13].isnan().tolist()
    assert nan == [False, True, True, False, False, False, True, False, False, False] and s.scales[page, 1, 0, 12].isnan()


def test_append_beyond_the_table(cuda):
    """A sequence that does not fit, or has a page that is none, is left alone and said."""
    s = check_append(ku.batch([5, 3, 4], [60, 62, 10], torch.bfloat16, torch.int8, rot=64, seed=4, max_len=64))
    assert s.flag.item() == 12
    s = ku.batch([2, 2], [0, 0], torch.bfloat16, torch.int8, seed=4)
    s.page_table[s.slot_host[1], 0] = -1
    s.counts, before = [2, 0], s.pool.clone()
    pool, scales, _ = ku.appended(s)
    from poptransformer_b200 import ops
    ops.kv8_append(s.view, s.qkv, s.ld, s.cache, s.heads, error_flag=s.flag)
    assert s.flag.item() == 12 and torch.equal(s.pool.view(torch.uint8).cpu(), pool) and not torch.equal(s.pool.view(torch.uint8), before.view(torch.uint8))
    s.start[0] = -1
    s.flag.zero_()
    ops.kv8_append(s.view, s.qkv, s.ld, s.cache, s.heads, error_flag=s.flag)
    assert s.flag.item() == 12 and torch.equal(s.pool.view(torch.uint8).cpu(), pool)


def test_append_without_queries(cuda):
    from poptransformer_b200 import ops
    s = ku.batch([6, 2], [10, 70], torch.float16, torch.int8, rot=32, seed=5)
    pool, scales, _ = ku.appended(s)
    kv = s.qkv[:, s.q_cols:].contiguous()
    ops.kv8_append(s.view, kv, kv.shape[1], s.cache, rope=s.rope, rope_dims=32)
    assert torch.equal(s.pool.view(torch.uint8).cpu(), pool) and torch.equal(s.scales.cpu().nan_to_num(-1), scales.nan_to_num(-1))


# ------------------------------------------------------------------------------------------ attention
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("plain", [False, True])
def test_attention(cuda, fmt, dtype, plain):
    s = ku.cached(ku.batch([1, 1, 1, 1, 1], [300, 0, 63, 1299, 64], DT[dtype], DT[fmt], dim=128, n_kv=2, qpk=4, seed=1))
    ku.check(s, s.qkv, ku.attend(s, s.qkv, plain=plain))
    assert s.flag.item() == 0


# the own token alone, tile and page borders, a history over many tiles
@pytest.mark.parametrize("start", [0, 1, 14, 15, 16, 30, 31, 32, 33, 62, 63, 64, 127, 128, 1023, 5000])
@pytest.mark.parametrize("dtype,fmt", [("bf16", "int8"), ("fp32", "e4m3"), ("fp16", "e4m3")])
def test_lengths(cuda, start, dtype, fmt):
    s = ku.cached(ku.batch([1], [start], DT[dtype], DT[fmt], dim=64, n_kv=1, qpk=2, seed=start))
    ku.check(s, s.qkv, ku.attend(s, s.qkv))


@pytest.mark.parametrize("n_kv,qpk,dim,vdim,page", [(1, 1, 64, 64, 64), (2, 16, 128, 128, 64), (8, 4, 128, 128, 16), (3, 5, 72, 72, 64), (2, 3, 96, 64, 64), (2, 2, 128, 48, 32), (1, 7, 20, 33, 7),
                                                    (2, 2, 80, 80, 100), (1, 4, 256, 256, 64), (2, 1, 256, 130, 64), (5, 3, 17, 5, 3), (1, 32, 64, 64, 128), (4, 8, 16, 16, 64), (12, 1, 64, 64, 64),
                                                    (1, 48, 256, 256, 16), (2, 9, 112, 240, 48), (32, 1, 128, 128, 64), (1, 8, 32, 256, 64), (1, 8, 256, 32, 16)])
@pytest.mark.parametrize("dtype,fmt", [("bf16", "int8"), ("fp32", "int8"), ("fp16", "e4m3")])
def test_heads_and_pages(cuda, n_kv, qpk, dim, vdim, page, dtype, fmt):
    s = ku.cached(ku.batch([1, 1, 1], [200, 515, 3], DT[dtype], DT[fmt], n_kv=n_kv, qpk=qpk, dim=dim, vdim=vdim, page=page, seed=dim + page))
    ku.check(s, s.qkv, ku.attend(s, s.qkv))
    assert s.flag.item() == 0


@pytest.mark.parametrize("window", [1, 2, 5, 31, 32, 33, 64, 65, 200, 100000])
@pytest.mark.parametrize("dtype,plain", [("bf16", False), ("bf16", True), ("fp16", False), ("fp32", False)])
def test_windows(cuda, window, dtype, plain):
    s = ku.cached(ku.batch([1, 1, 1, 1], [300, 2, 64, 901], DT[dtype], torch.int8, dim=64, seed=window))
    ku.check(s, s.qkv, ku.attend(s, s.qkv, window=window, plain=plain), window=window)


@pytest.mark.parametrize("dtype,plain", [("bf16", False), ("fp16", True), ("fp32", False)])
def test_softcap_and_scale(cuda, dtype, plain):
    s = ku.cached(ku.batch([1, 1], [150, 700], DT[dtype], torch.int8, dim=128, seed=3))
    s.scale = 0.7                                     # scores far beyond the cap
    ku.check(s, s.qkv, ku.attend(s, s.qkv, softcap=5.0, plain=plain), softcap=5.0)
    s.scale = -0.05
    ku.check(s, s.qkv, ku.attend(s, s.qkv, plain=plain))
    s.scale = 0.0
    ku.check(s, s.qkv, ku.attend(s, s.qkv, plain=plain))


@pytest.mark.parametrize("dtype,plain", [("bf16", False), ("bf16", True), ("fp32", False)])
def test_several_tokens_empty_sequences_and_rows_behind(cuda, dtype, plain):
    s = ku.cached(ku.batch([0, 6, 0, 1, 31, 2, 0], [100, 1000, 5, 0, 10, 0, 64], DT[dtype], torch.int8, dim=64, n_kv=2, qpk=3, seed=5, spare_rows=4, slots=11))
    width = s.heads * s.vdim
    out = torch.full((s.n_tok + 4, width + 10), 7.0, dtype=s.dtype, device=s.device)
    ku.attend(s, s.qkv, out=out, plain=plain)
    ku.check(s, s.qkv, out)
    assert (out[:, width:] == 7).all() and (out[s.n_tok:] == 7).all() and s.flag.item() == 0


@pytest.mark.parametrize("n_seq", [1, 33, 700])
def test_many_sequences(cuda, n_seq):
    s = ku.cached(ku.batch([1] * n_seq, [(i * 37) % 300 for i in range(n_seq)], torch.bfloat16, torch.int8, dim=64, n_kv=1, qpk=2, seed=6))
    ku.check(s, s.qkv, ku.attend(s, s.qkv))


@pytest.mark.parametrize("plain", [False, True])
def test_attention_beyond_the_table(cuda, plain):
    s = ku.cached(ku.batch([1, 2, 1], [60, 70, 10], torch.bfloat16, torch.int8, seed=4, max_len=71))
    s.start[1] = 70                                   # positions 70 and 71 of 71
    s.counts = [1, 0, 1]
    out = torch.full((4, s.heads * s.vdim), 7.0, dtype=s.dtype, device=s.device)
    ku.attend(s, s.qkv, out=out, plain=plain)
    assert s.flag.item() == 12 and (out[1:3] == 7).all()
    want, tol = ku.reference(s, s.qkv)
    for r in (0, 3):
        s.cu_host = [0, 1, 1, 3]
        assert ((out[r].double().view(s.heads, -1) - want[r]).abs() <= tol[r]).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("plain", [False, True])
def test_scores_and_values_of_any_size(cuda, dtype, plain):
    """One high score before 20,000 small ones whose weights matter together, values whose scales lie far apart, and scores up to the thousands."""
    n = 20000
    s = ku.cached(ku.batch([1], [n], DT[dtype], torch.int8, dim=64, n_kv=1, qpk=4, seed=8))
    s.qkv[:] = 0
    s.qkv[:, 0:256:64] = 1.0
    s.scale = 1.0
    pages = ku.ints(s.table_host[s.slot_host[0]]).long()
    key = ku.part(s, s.pool, pages, 0)                # (a copy)
    key[..., 0] = 100
    k = s.n_kv * s.page * s.dim
    s.pool[pages, :k] = key.flatten(1)
    s.scales[pages, 0] = 0.0
    s.scales[pages[0], 0, 0, 7] = 0.1                 # score 10, the others 0: weights of e^-10 each
    s.scales[pages, 1] = 1.0
    s.scales[pages[0], 1, 0, 7] = 1e-4
    ku.check(s, s.qkv, ku.attend(s, s.qkv, plain=plain))
    s.scales[pages[5], 1, 0, 3] = 1e9                 # a value that is large enough to count behind the others
    ku.check(s, s.qkv, ku.attend(s, s.qkv, plain=plain))
    s.scales[pages[9], 0, 0, 1] = 40.0                # a score of 4000: it has all of the weight
    s.scales[pages[9], 1, 0, 1] = 1e-12
    ku.check(s, s.qkv, ku.attend(s, s.qkv, plain=plain))


@pytest.mark.parametrize("plain", [False, True])
def test_rows_that_read_as_nan(cuda, plain):
    """A NaN key makes every output of its kv head NaN for whoever sees it, a NaN value too; nobody else notices."""
    s = ku.cached(ku.batch([1, 1, 1], [100, 80, 90], torch.bfloat16, torch.int8, dim=64, n_kv=2, qpk=2, seed=9))
    s.scales[s.table_host[s.slot_host[0]][0], 0, 1, 5] = math.nan
    s.scales[s.table_host[s.slot_host[1]][1], 1, 0, 5] = math.nan
    out = ku.attend(s, s.qkv, plain=plain).view(3, 4, 64)
    assert out[0, 2:].isnan().all() and out[1, :2].isnan().all() and not out[0, :2].isnan().any() and not out[1, 2:].isnan().any() and not out[2].isnan().any()
    out = ku.attend(s, s.qkv, window=20, plain=plain).view(3, 4, 64)
    assert not out[0].isnan().any() and out[1, :2].isnan().all() and not out[2].isnan().any()


def test_the_same_call_gives_the_same_bits(cuda):
    from poptransformer_b200 import ops
    s = ku.cached(ku.batch([1] * 6, [7000, 3, 900, 2500, 64, 11000], torch.float32, torch.int8, dim=128, n_kv=2, qpk=4, seed=10))
    ws = ops.kv8_attn_workspace(6, s.heads, s.n_kv, s.vdim)
    first = ku.attend(s, s.qkv, workspace=ws).clone()
    for _ in range(5):
        assert torch.equal(ku.attend(s, s.qkv, workspace=ws), first)


def test_pages_behind_the_first_four_gigabytes(cuda):
    """Offsets of pages, scales and positions pass 32 bits."""
    s = ku.batch([2, 1], [130, 64], torch.bfloat16, torch.int8, n_kv=8, qpk=1, dim=128, page=64, base_page=40000, seed=11)     # pages of 128 KB
    from poptransformer_b200 import ops
    ops.kv8_append(s.view, s.qkv, s.ld, s.cache, s.heads, error_flag=s.flag)
    x = s.qkv.float()
    for tok, (i, pos) in enumerate([(0, 130), (0, 131), (1, 64)]):
        page = s.table_host[s.slot_host[i]][pos // 64]
        for which, first in ((0, s.q_cols), (1, s.q_cols + 8 * 128)):
            by, sc = ku.to_bytes(x[tok, first:first + 1024].view(8, 128), torch.int8)
            assert torch.equal(ku.part(s, s.pool, page, which)[:, pos % 64], by) and torch.equal(s.scales[page, which, :, pos % 64], sc)
    ku.check(s, s.qkv, ku.attend(s, s.qkv))
    ku.check(s, s.qkv, ku.attend(s, s.qkv, plain=True))
    assert s.flag.item() == 0


# ------------------------------------------------------------------------------------------ pages in a wider type
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("dim,vdim,page,into_page", [(128, 128, 64, 64), (64, 32, 16, 64), (33, 5, 7, 3), (80, 80, 64, 16)])
def test_unpack(cuda, fmt, dtype, dim, vdim, page, into_page):
    from poptransformer_b200 import ops
    s = ku.cached(ku.batch([3, 0, 1, 9], [120, 70, 0, 64], DT[dtype], DT[fmt], dim=dim, vdim=vdim, page=page, seed=dim, slots=6))
    into = ops.PagedKVCache(6, s.n_kv, dim, s.max_len, into_page, cuda, v_dim=vdim, dtype=DT[dtype])
    into.pool.fill_(7.0)
    ops.kv8_unpack(s.view, s.cache, into, error_flag=s.flag)
    flat = into.pool.flatten(1)
    want = torch.full_like(flat, 7.0)
    k = s.n_kv * into_page * dim
    for i, n in enumerate(s.counts):
        for which, width in ((0, dim), (1, vdim)):
            x = ku.history(s, i, s.starts[i] + n, which).float()       # (a byte times a scale, rounded to 32 bits as the kernel does, then to the type)
            for pos in range(s.starts[i] + n):
                p = int(into.page_table[s.slot_host[i], pos // into_page])
                at = want[p, :k].view(s.n_kv, into_page, dim) if which == 0 else want[p, k:].view(s.n_kv, into_page, vdim)
                at[:, pos % into_page] = x[:, pos].to(DT[dtype])
    assert torch.equal(flat, want) and s.flag.item() == 0


def test_unpack_beyond_the_tables(cuda):
    from poptransformer_b200 import ops
    s = ku.cached(ku.batch([1, 1], [40, 70], torch.bfloat16, torch.int8, seed=12))
    into = ops.PagedKVCache(2, s.n_kv, s.dim, 64, 64, cuda, dtype=torch.bfloat16)
    into.pool.fill_(7.0)
    ops.kv8_unpack(s.view, s.cache, into, error_flag=s.flag)
    other = into.pool[int(into.page_table[s.slot_host[1], 0])]
    assert s.flag.item() == 12 and (other == 7).all() and (into.pool[int(into.page_table[s.slot_host[0], 0]), :, :, :41] != 7).any()


# ------------------------------------------------------------------------------------------ together, as they are used
@pytest.mark.parametrize("fmt,interleaved", [("int8", False), ("e4m3", True)])
def test_a_prompt_and_decode_steps(cuda, fmt, interleaved):
    """Prompts go to the cache, their attention runs on the pages in 16 bits, steps of one token follow; everything from one graph that is replayed."""
    from poptransformer_b200 import cache, ops
    G, H, D, steps = 2, 8, 64, 4
    slots = cache.SequenceSlots(4, 256, 64)
    kv = ops.PagedKVCache(4, G, D, 256, 64, "cuda", slots.page_table, dtype=DT[fmt], n_pages=slots.n_pages)
    wide = ops.PagedKVCache(4, G, D, 256, 64, "cuda", slots.page_table, dtype=torch.bfloat16, n_pages=slots.n_pages)
    rope = ops.rope_table(256, D, scaling=dict(kind="linear", factor=2.0))
    prompts = [100, 1, 60]
    seqs = [slots.open() for _ in prompts]
    gen = torch.Generator().manual_seed(0)
    all_rows = [torch.randn((n + steps, (H + 2 * G) * D), generator=gen).bfloat16().cuda() for n in prompts]
    flag = ku.ints([0])

    def view_of(counts, starts):
        return ops.batch_view(len(counts), sum(counts), ku.ints([sum(counts[:i]) for i in range(len(counts) + 1)]), ku.ints(starts), ku.ints(seqs),
                              ku.ints([i for i, n in enumerate(counts) for _ in range(n)]))

    def expect(i, pos, q):
        """From the bytes as they are."""
        pages = slots.page_table[seqs[i]].long()[:pos // 64 + 1]
        k, v = ((kv.pool[pages, w].to(torch.float32).double() * kv.scales[pages, w][..., None].double()).transpose(0, 1).flatten(1, 2)[:, :pos + 1] for w in (0, 1))
        z = q.double().view(G, H // G, D) @ k.transpose(1, 2) * D ** -0.5
        p = torch.softmax(z, -1)
        return (p @ v).flatten(), (p @ v.abs()).flatten()

    rows = torch.cat([r[:n] for r, n in zip(all_rows, prompts)])
    for s, n in zip(seqs, prompts):
        slots.extend(s, n)
    view, q, out = view_of(prompts, [0, 0, 0]), torch.empty((sum(prompts), H * D), dtype=torch.bfloat16, device=cuda), torch.empty((sum(prompts), H * D), dtype=torch.bfloat16, device=cuda)
    ops.kv8_append(view, rows, rows.shape[1], kv, H, rope=rope, rope_dims=D, interleaved=interleaved, q_out=q, q_out_ld=H * D, error_flag=flag)
    ops.kv8_unpack(view, kv, wide, error_flag=flag)
    ops.window_attn(view, q, H * D, wide, out, H * D, H, D ** -0.5, append=False, max_tokens_per_seq=max(prompts), error_flag=flag)
    at = 0
    for i, n in enumerate(prompts):
        for pos in range(n):
            want, size = expect(i, pos, q[at + pos])
            # keys and values in bf16 (2^-9 each, of scores up to about 4: 2^-6 of a weight), weights and output in bf16
            assert ((out[at + pos].double() - want).abs() <= 2.0 ** -5 * size + 2.0 ** -8 * want.abs()).all()
        at += n
    ws = ops.kv8_attn_workspace(3, H, G, D)
    row = torch.empty((3, rows.shape[1]), dtype=torch.bfloat16, device=cuda)
    view = view_of([1, 1, 1], prompts)
    start = view.keep[1]
    q1, o1 = torch.empty((3, H * D), dtype=torch.bfloat16, device=cuda), torch.empty((3, H * D), dtype=torch.bfloat16, device=cuda)

    def step():
        ops.kv8_append(view, row, row.shape[1], kv, H, rope=rope, rope_dims=D, interleaved=interleaved, q_out=q1, q_out_ld=H * D, error_flag=flag)
        ops.kv8_attn(view, q1, H * D, kv, o1, H * D, H, D ** -0.5, workspace=ws, error_flag=flag)

    for s in seqs:
        slots.extend(s, steps)
    row.copy_(torch.stack([r[n] for r, n in zip(all_rows, prompts)]))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for t in range(steps):
        row.copy_(torch.stack([r[n + t] for r, n in zip(all_rows, prompts)]))
        start.copy_(ku.ints([n + t for n in prompts]))
        graph.replay()
        for i, n in enumerate(prompts):
            want, size = expect(i, n + t, q1[i])
            assert ((o1[i].double() - want).abs() <= 2.0 ** -9 * size + 2.0 ** -8 * want.abs()).all()
    assert flag.item() == 0
    # a sequence forks: its last page is copied with its scales, and both read the same
    new, copies = slots.fork(seqs[0])
    assert copies
    ops.PagePools([kv]).copy(copies)
    a, b = copies[0]
    assert torch.equal(kv.pool[a].view(torch.uint8), kv.pool[b].view(torch.uint8)) and torch.equal(kv.scales[a], kv.scales[b])


def test_accepted_rows_move_with_their_scales(cuda):
    from poptransformer_b200 import ops
    s = ku.cached(ku.batch([6, 5], [60, 3], torch.bfloat16, torch.int8, n_kv=3, dim=64, seed=13))
    before = [[ku.history(s, i, s.starts[i] + s.counts[i], w) for w in (0, 1)] for i in (0, 1)]
    path, count = ku.ints([[0, 2, 5], [1, 4, -1]]), ku.ints([3, 2])
    ops.PagePools([s.cache]).move_rows(s.view, path, count, error_flag=s.flag)
    for i, kept in enumerate(([0, 2, 5], [1, 4])):
        for w in (0, 1):
            now = ku.history(s, i, s.starts[i] + len(kept), w)
            assert torch.equal(now[:, s.starts[i]:], before[i][w][:, [s.starts[i] + k for k in kept]]) and torch.equal(now[:, :s.starts[i]], before[i][w][:, :s.starts[i]])
    assert s.flag.item() == 0


def test_two_streams_with_workspaces_of_their_own(cuda):
    from poptransformer_b200 import ops
    batches = [ku.cached(ku.batch([1, 1], [n, 4000], torch.bfloat16, torch.int8, dim=128, n_kv=8, qpk=4, seed=n)) for n in (5000, 300)]
    streams = [torch.cuda.Stream() for _ in batches]
    outs = [torch.empty((2, s.heads * s.vdim), dtype=s.dtype, device=cuda) for s in batches]
    ws = [ops.kv8_attn_workspace(2, s.heads, s.n_kv, s.vdim) for s in batches]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, st, o, w in zip(batches, streams, outs, ws):
            with torch.cuda.stream(st):
                ku.attend(s, s.qkv, out=o, workspace=w)
    torch.cuda.synchronize()
    for s, o in zip(batches, outs):
        ku.check(s, s.qkv, o)
