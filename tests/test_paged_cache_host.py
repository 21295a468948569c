"""Memory that a paged cache is given: how much there has to be, and where."""
import pytest
import torch

from poptransformer_b200 import ops


def _cache(pool, **kw):
    return ops.PagedKVCache(3, 2, 16, 40, 8, "cpu", **{**dict(dtype=torch.float16, pool=pool), **kw})      # 3 rows of 5 pages of 8 positions


def _pool(pages, **kw):
    return torch.zeros((pages, 2, 2, 8, 16), **{**dict(dtype=torch.float16), **kw})


def test_pools_that_are_too_small_are_refused():
    table = torch.zeros((3, 5), dtype=torch.int32)
    for pages, kw in ((14, {}), (0, {}), (15, dict(extra_pages=1)), (6, dict(n_pages=7)), (6, dict(n_pages=7, page_table=table)), (7, dict(n_pages=7, page_table=table, extra_pages=1)),
                      (0, dict(page_table=table))):
        with pytest.raises(ops.PtError, match="pages"):
            _cache(_pool(pages), **kw)
    for pages, kw in ((15, {}), (16, dict(extra_pages=1)), (40, {}), (7, dict(n_pages=7, page_table=table)), (2, dict(page_table=table))):
        pool = _pool(pages)
        c = _cache(pool, **kw)
        assert c.pool is pool
    assert int(_cache(_pool(15)).page_table.max()) == 14


def test_pools_of_another_kind_are_refused():
    table = torch.zeros((3, 5), dtype=torch.int32)
    for pool in (_pool(15, dtype=torch.bfloat16), _pool(15)[:, :1], torch.zeros((30, 2, 2, 8, 16), dtype=torch.float16)[::2], torch.zeros((), dtype=torch.float16)):
        with pytest.raises(ops.PtError, match="expected contiguous"):
            _cache(pool)
    for pool, kw in ((_pool(15, device="meta"), {}), (_pool(15, device="meta"), dict(page_table=table)), (_pool(15), dict(page_table=table.to("meta")))):
        with pytest.raises(ops.PtError, match="wanted on"):
            _cache(pool, **kw)
