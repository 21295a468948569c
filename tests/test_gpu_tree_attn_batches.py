"""Batches of drafted trees that a caller describes in other ways."""
import pytest
import torch

import tree_util as tu

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n_seq,n", [(17, 16), (300, 3), (2, 4)])
@pytest.mark.parametrize("dtype,plain", [(torch.bfloat16, False), (torch.float32, True)])
def test_the_most_tokens_of_a_sequence_need_not_be_given(cuda, n_seq, n, dtype, plain):
    from poptransformer_b200 import ops
    s = tu.batch([n] * n_seq, [(37 * i) % 90 for i in range(n_seq)], dtype=dtype, dim=64, n_kv=1, qpk=2, seed=41)
    before = s.cache.pool.clone()
    ws = ops.tree_attn_workspace(n_seq, min(256, n_seq * n), s.heads, s.n_kv, s.vdim)
    tu.check(s, before, tu.run(s, most=0, workspace=ws, plain=plain))
    assert s.flag.item() == 0


@pytest.mark.parametrize("dtype,plain", [(torch.bfloat16, False), (torch.float16, True), (torch.float32, True)])
def test_pages_behind_the_first_eight_gigabytes(cuda, dtype, plain):
    """Offsets that 32 bits do not hold, in attention, row moves and page copies."""
    from poptransformer_b200 import ops
    s = tu.batch([20, 9], [700, 130], dtype=dtype, dim=128, n_kv=8, qpk=2, rot=128, seed=42)
    small, used = s.cache.pool, s.cache.pool.shape[0]
    first = (9 << 30) // small[0].numel() // small.element_size()
    big = torch.empty((first + used + 20,) + tuple(small.shape[1:]), dtype=dtype, device=cuda)
    big[first:first + used] = small
    s.table = [[p + first for p in row] for row in s.table]
    s.cache.page_table += first
    s.cache.pool = big
    view = lambda: tu._pages(s, big, 0, 720)
    before = big[first:].clone()
    out = tu.run(s, plain=plain)
    keep, s.table = s.table, [[p - first for p in row] for row in s.table]
    s.cache.pool = big[first:]
    tu.check(s, before, out)
    s.table, s.cache.pool = keep, big
    K, V = view()
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda)
    pools = ops.PagePools([s.cache])
    pools.move_rows(s.view, i32([[0, 3, 4, 19], [0, 8, -1, -1]]), i32([4, 2]), error_flag=s.flag)
    K2, V2 = view()
    rows = list(range(700)) + [700, 703, 704, 719]
    assert torch.equal(K2[:, :704], K[:, rows]) and torch.equal(V2[:, :704], V[:, rows])
    pages = s.table[s.slot[0]][:5]
    held = big[pages].clone()
    pools.copy_pages(i32(pages), i32(range(first + used, first + used + 5)), error_flag=s.flag)
    pools.copy_pages(i32(pages), i32(range(5)), error_flag=s.flag)
    assert torch.equal(big[first + used:first + used + 5], held) and torch.equal(big[:5], held) and s.flag.item() == 0
