"""Moves of accepted rows along paths as long as verification makes them."""
import random

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [255, 256, 257, 511, 512])
@pytest.mark.parametrize("every", [False, True])
def test_long_paths(cuda, n, every):
    """n rows of 600 (or of n: nothing moves); a path of 513 is refused and said."""
    from poptransformer_b200 import ops
    page, tokens, start = 16, n if every else 600, 37
    per = -(-(start + 600) // page)
    order = random.Random(n).sample(range(per + 4), per)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda)
    g = torch.Generator(device=cuda).manual_seed(n)
    caches = []
    table = i32([order])
    for dim in (8, 64):
        c = ops.PagedKVCache(1, 2, dim, per * page, page, cuda, table, dtype=torch.bfloat16, n_pages=per + 4)
        c.pool.copy_(torch.randn(c.pool.shape, generator=g, device=cuda))
        caches.append(c)
    before = [c.pool.clone() for c in caches]
    flag = i32([0])
    view = ops.batch_view(1, tokens, i32([0, tokens]), i32([start]), i32([0]), i32([0] * tokens))
    path = sorted(random.Random(n + 1).sample(range(tokens), n))
    ops.PagePools(caches).move_rows(view, i32([path]), i32([n]), error_flag=flag)
    assert flag.item() == 0
    at = lambda pool, j: pool[order[j // page], :, :, j % page]
    for c, b in zip(caches, before):
        want = b.clone()
        for i, r in enumerate(path):
            at(want, start + i).copy_(at(b, start + r))
        assert torch.equal(c.pool, want)


def test_a_path_that_is_too_long_is_left_alone(cuda):
    from poptransformer_b200 import ops
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda)
    c = ops.PagedKVCache(1, 1, 8, 640, 64, cuda, dtype=torch.float16)
    c.pool.copy_(torch.randn(c.pool.shape, device=cuda))
    before, flag = c.pool.clone(), i32([0])
    view = ops.batch_view(1, 600, i32([0, 600]), i32([0]), i32([0]), i32([0] * 600))
    ops.PagePools([c]).move_rows(view, i32([list(range(1, 514))]), i32([513]), error_flag=flag)
    assert flag.item() == 14 and torch.equal(c.pool, before)
