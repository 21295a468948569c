"""Caches of eight bits and of other widths than the rows': what the calls beside them say before any launch."""
import math
from types import SimpleNamespace

import pytest
import torch

from poptransformer_b200 import _lib, ops
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


def test_cache_objects_of_a_callers_own_need_no_scales(monkeypatch):
    """What the calls read of a cache of 16 or 32 bits is what they read before there were others."""
    monkeypatch.setattr(ops, "_ptr", lambda t: None if t is None else t.data_ptr())

    class Taken(Exception):
        pass

    class Library:
        def __getattr__(self, name):
            def call(*args):
                raise Taken(name)
            return call

    monkeypatch.setattr(ops._lib, "lib", Library)
    monkeypatch.setattr(ops, "_stream", lambda: None)
    full = cache(torch.float16)
    own = SimpleNamespace(**{n: getattr(full, n) for n in ("n_kv", "head_dim", "v_dim", "page_size", "max_pages", "max_len", "pool", "page_table")})
    w = SimpleNamespace(q_rank=8, rank=8, rot_dim=8, dim=8, vdim=8, heads=2, q_norm=None, kv_norm=None, w_k=None, w_v=None)
    view, step = _lib.BatchView(1, 1), torch.zeros(1, dtype=torch.int32)
    wide = torch.zeros((1, 3 * 2 * 64), dtype=torch.float16)
    for call, name in ((lambda: ops.window_attn(view, wide, 384, own, wide, 384, 2, 1.0), "pt_window_attn"), (lambda: ops.kv_append_attn(wide, step, own, 2, workspace=wide), "pt_kv_append_attn"),
                       (lambda: ops.prefill_attn(wide, own, 1, 1, 0, 2, 1.0, None, None), "pt_prefill_attn"), (lambda: ops.tree_attn(view, wide, 384, own, wide, 384, 2, 1.0), "pt_tree_attn"),
                       (lambda: ops.latent_prep(view, wide, 384, 0, 0, w, wide, 384, own, 0.0, None), "pt_latent_prep"),
                       (lambda: ops.latent_context(view, step, 1, w, own, wide, wide, 384), "pt_latent_context"),
                       (lambda: ops.latent_attn(view, wide, 384, w, own, wide, 384, 1.0, None, wide), "pt_latent_attn"),
                       (lambda: ops.PagePools([own]).copy_pages(step, step), "pt_kv_copy_pages")):
        with pytest.raises(Taken, match=name):
            call()


def test_pages_of_bytes_without_scales():
    """A program's own bytes (any widths, no scales) are torch.uint8, and the refusals of eight bits say so."""
    for dtype in (torch.int8, torch.float8_e4m3fn):
        made = cache(dtype)
        for kw in (dict(pool=made.pool), dict(v_dim=0), dict(v_dim=300)):
            with pytest.raises(PtError, match="torch.uint8"):
                cache(dtype, **kw)
        own = cache(torch.uint8, pool=made.pool.view(torch.uint8))
        assert own.scales is None and own.pool.data_ptr() == made.pool.data_ptr()
    assert cache(torch.uint8, v_dim=0).pool.shape == (4, 2 * 64 * 64) and cache(torch.uint8, v_dim=300).pool.shape == (4, 2 * 64 * 364)
    with pytest.raises(PtError, match="is wanted"):
        ops._kv8(cache(torch.uint8), "kv8_attn")


def test_a_changed_cache_is_looked_at_again(monkeypatch):
    """The structure that the kernels get is kept from call to call, and says what the cache says now."""
    monkeypatch.setattr(ops, "_ptr", lambda t: None if t is None else t.data_ptr())
    c = cache()
    first = ops._kv8(c, "kv8_attn")
    assert ops._kv8(c, "kv8_attn") is first and first.max_len == 128 and first.max_pages == 2
    c.max_len = 100                                   # positions from 100 on are refused from now on
    assert ops._kv8(c, "kv8_attn").max_len == 100
    c.max_len = 129                                   # more than the table has pages for
    with pytest.raises(PtError, match="page table"):
        ops._kv8(c, "kv8_attn")
    c.max_len, table = 128, torch.zeros((2, 5), dtype=torch.int32)
    c.page_table = table
    assert ops._kv8(c, "kv8_attn").max_pages == 5
    table.resize_(2, 2)                               # the same tensor at the same place
    assert ops._kv8(c, "kv8_attn").max_pages == 2
    c.page_size, c.max_len = 32, 64                   # (two pages of 32)
    with pytest.raises(PtError, match="pages of 32 positions"):
        ops._kv8(c, "kv8_attn")
    c.n_kv = 4                                        # the same bytes, as twice the heads of half of the positions
    made = ops._kv8(c, "kv8_attn")
    assert (made.n_kv, made.page_size, made.max_len) == (4, 32, 64)
    c.head_dim = 65
    with pytest.raises(PtError, match="heads of 65 and 64"):
        ops._kv8(c, "kv8_attn")


def test_a_table_of_angles_says_how_much_turns(monkeypatch):
    """kv8_append rotates as wide as its table is, like rotary; a width that is not the table's is refused, 0 too."""
    monkeypatch.setattr(ops, "_ptr", lambda t: None if t is None else t.data_ptr())
    monkeypatch.setattr(ops, "_here", lambda *a: None)
    monkeypatch.setattr(ops, "_stream", lambda: None)
    seen = []

    class Library:
        def pt_kv8_append(self, a, stream):
            seen.append(a._obj.rope_dims)
            return 0

    monkeypatch.setattr(ops._lib, "lib", Library)
    c, i = cache(), torch.zeros(2, dtype=torch.int32)
    view = _lib.BatchView(1, 1)
    view.keep = (i, i, i, i)
    x, rope = torch.zeros((1, 6 * 64), dtype=torch.float16), ops.rope_table(128, 32, device="cpu")
    for kw, dims in ((dict(rope=rope), 32), (dict(rope=rope, rope_dims=32), 32), (dict(), 0), (dict(rope_dims=0), 0), (dict(rope_dims=None), 0)):
        ops.kv8_append(view, x, 384, c, 2, **kw)
        assert seen.pop() == dims
    for kw in (dict(rope=rope, rope_dims=0), dict(rope=rope, rope_dims=64), dict(rope_dims=32), dict(rope=rope[:100]), dict(rope=rope.double()), dict(rope=rope[0]), dict(rope=rope[:, 0, 0])):
        with pytest.raises(PtError, match="rotated dimensions"):
            ops.kv8_append(view, x, 384, c, 2, **kw)
    assert not seen


def test_rotary_refuses_rows_that_want_a_gradient():
    """The call records none; without recording, such rows are as good as others."""
    rope, at = ops.rope_table(4, 64, device="cpu"), torch.zeros(1, dtype=torch.int32)
    leaf, plain = torch.zeros((1, 64), requires_grad=True), torch.zeros((1, 64))
    for x, out in ((leaf, None), (leaf * 2.0, None), (leaf, plain), (plain, leaf)):
        with pytest.raises(PtError, match="wants a gradient"):
            ops.rotary(x, 1, 64, rope, at, out=out)
        with torch.no_grad(), pytest.raises(PtError, match="device"):           # (the next check: everything is on the CPU here)
            ops.rotary(x, 1, 64, rope, at, out=out)
    with pytest.raises(PtError, match="device"):
        ops.rotary(leaf.detach(), 1, 64, rope, at)


def test_tables_of_angles_that_would_be_no_numbers():
    """Sizes that are no finite numbers, and bounds that leave nothing between them or stand in the wrong order."""
    for kw in (dict(base=math.nan), dict(base=math.inf), dict(scaling=dict(kind="linear", factor=math.inf)), dict(scaling=dict(kind="base", factor=math.nan)),
               dict(scaling=dict(kind="bands", factor=2.0, original=64, low=4.0, high=4.0)), dict(scaling=dict(kind="bands", factor=2.0, original=64, low=4.0, high=1.0)),
               dict(base=1.0, scaling=dict(kind="ramp", factor=2.0, original=64)), dict(base=0.5, scaling=dict(kind="ramp", factor=2.0, original=64)),
               dict(scaling=dict(kind="ramp", factor=2.0, original=64, slow=32, fast=32)), dict(scaling=dict(kind="ramp", factor=2.0, original=64, slow=40))):
        with pytest.raises(PtError, match="rope_table"):
            ops.rope_table(8, 8, device="cpu", **kw)
    for kw in (dict(base=0.5), dict(base=1.0), dict(scaling=dict(kind="bands", factor=2.0, original=64, low=1.0, high=4.0)), dict(scaling=dict(kind="ramp", factor=1.0, original=64))):
        assert ops.rope_table(8, 8, device="cpu", **kw).isfinite().all()
