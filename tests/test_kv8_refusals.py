"""Caches of eight bits and of other widths than the rows': what the calls beside them say before any launch."""
import pytest
import torch

from poptransformer_b200 import ops
from poptransformer_b200._lib import PtError


def cache(dtype=torch.int8, **kw):
    return ops.PagedKVCache(2, 2, 64, 128, 64, "cpu", dtype=dtype, **kw)


def calls(c, x):
    """Every call that takes a cache in the rows' type; what else it wants is not looked at before the cache is."""
    step = torch.zeros(1, dtype=torch.int32)
    return dict(window_attn=lambda: ops.window_attn(None, x, 384, c, x, 384, 2, 1.0), kv_append_attn=lambda: ops.kv_append_attn(x, step, c, 2, workspace=x),
                prefill_attn=lambda: ops.prefill_attn(x, c, 1, 1, 0, 2, 1.0, None, None), latent_prep=lambda: ops.latent_prep(None, x, 384, 0, 0, None, x, 384, c, 0.0, None),
                latent_context=lambda: ops.latent_context(None, step, 1, None, c, x, x, 384), latent_attn=lambda: ops.latent_attn(None, x, 384, None, c, x, 384, 1.0, None, x))


@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("rows", [torch.float16, torch.bfloat16, torch.float32])
def test_kernels_of_wide_caches_refuse_those_of_eight_bits(dtype, rows):
    x = torch.zeros((1, 6 * 64), dtype=rows)
    for name, call in calls(cache(dtype), x).items():
        with pytest.raises(PtError, match=name + ".*is written by kv8_append"):
            call()
    with pytest.raises(PtError, match="export.*is written by kv8_append"):
        cache(dtype).export(torch.zeros(1, dtype=torch.int32), 8)
    with pytest.raises(PtError, match="into.*is written by kv8_append"):
        ops.kv8_unpack(None, cache(dtype), cache(dtype))
    with pytest.raises(PtError, match="tree_attn.*one type is wanted"):
        ops.tree_attn(None, x, 384, cache(dtype), x, 384, 2, 1.0)


def test_a_pool_of_smaller_elements_than_the_rows_is_refused():
    """The kernels count in the rows' type: they would write behind such a pool's end."""
    for pool, rows in ((torch.uint8, torch.float16), (torch.uint8, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float16, torch.float32)):
        for name, call in calls(cache(pool), torch.zeros((1, 6 * 64), dtype=rows)).items():
            with pytest.raises(PtError, match=name + ".*elements of"):
                call()
    with pytest.raises(PtError, match="export.*elements of"):
        cache(torch.uint8).export(torch.zeros(1, dtype=torch.int32), 8)
