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
