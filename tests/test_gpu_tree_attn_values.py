"""Attention for trees of drafted tokens where values are infinite or NaN, and scores pass through caps of any size (tolerances: tree_util.reference)."""
import pytest
import torch

import tree_util as tu

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


@pytest.mark.parametrize("dtype,plain", [("bf16", False), ("fp16", False), ("bf16", True)])
@pytest.mark.parametrize("window", [0, 70])
def test_many_short_sequences_whose_second_halves_are_bad(cuda, dtype, plain, window):
    """Every sequence is one tile of keys that no row sees whole, and most values in its second half are NaN: one of the two warps that bring tiles in has all the
    work, tile after tile.  Rows that see none of those values keep their bits."""
    n, n_seq = 60, 600
    s = tu.batch([n] * n_seq, [64] * n_seq, "star", dtype=DT[dtype], dim=64, n_kv=1, qpk=1, page=128, seed=21)
    before = s.cache.pool.clone()
    want = tu.run(s, window=window, plain=plain).clone()
    some = tu.batch([n] * 4, [64] * 4, "star", dtype=DT[dtype], dim=64, n_kv=1, qpk=1, page=128, seed=22)
    held = some.cache.pool.clone()
    tu.check(some, held, tu.run(some, window=window, plain=plain), window=window)
    s.cache.pool.copy_(before)
    bad = (torch.arange(s.n_tok, device=cuda) % n) % 8 != 0      # (the root, which all see, is good)
    s.qkv[bad, 2 * 64:] = float("nan")
    for _ in range(5):
        s.cache.pool.copy_(before)
        got = tu.run(s, window=window, plain=plain)
        assert s.flag.item() == 0
        assert torch.equal(got[~bad], want[~bad]) and got[bad].isnan().all()
