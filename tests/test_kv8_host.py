"""Caches of eight bits: what is refused before any launch, and tables of angles."""
import ctypes
import math

import numpy as np
import pytest
import torch

from poptransformer_b200 import _lib, ops
from poptransformer_b200._lib import PtError


def cache(dtype=torch.int8, **kw):
    return ops.PagedKVCache(2, 2, 64, 128, 64, "cpu", dtype=dtype, **kw)


@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn])
def test_a_cache_of_eight_bits_has_scales(dtype):
    c = cache(dtype)
    assert c.pool.dtype == dtype and c.pool.shape == (4, 2, 2, 64, 64) and c.scales.shape == (4, 2, 2, 64) and c.scales.dtype == torch.float32
    assert cache(torch.float16).scales is None
    d = cache(dtype, pool=c.pool, scales=c.scales)
    assert d.pool is c.pool and d.scales is c.scales
    for kw in (dict(pool=c.pool), dict(scales=c.scales), dict(pool=c.pool, scales=c.scales[:3]), dict(pool=c.pool, scales=c.scales.double()), dict(v_dim=0), dict(v_dim=257)):
        with pytest.raises(PtError):
            cache(dtype, **kw)
    with pytest.raises(PtError, match="no scales"):
        cache(torch.float16, pool=torch.zeros((4, 2, 2, 64, 64), dtype=torch.float16), scales=c.scales)


def test_other_kernels_refuse_it():
    c = cache()
    x = torch.zeros((1, 6 * 64), dtype=torch.float16)
    for call in (lambda: c.export(torch.zeros(1, dtype=torch.int32), 8), lambda: ops.kv_append_attn(x, torch.zeros(1, dtype=torch.int32), c, 2, workspace=x),
                 lambda: ops.prefill_attn(x, c, 1, 1, 0, 2, 1.0, None, None), lambda: ops.window_attn(None, x, 384, c, x, 384, 2, 1.0), lambda: ops.tree_attn(None, x, 384, c, x, 384, 2, 1.0),
                 lambda: ops.kv8_unpack(None, c, c)):
        with pytest.raises(PtError):
            call()


def test_tensors_that_are_not_on_the_device_are_refused():
    """Launches go to the current device; what lies elsewhere is said, not read."""
    c = cache()
    i = torch.zeros(2, dtype=torch.int32)
    view = _lib.BatchView(1, 1)
    view.keep = (i, i, i, i)
    x = torch.zeros((1, 6 * 64), dtype=torch.float16)
    for call in (lambda: ops.kv8_append(view, x, 384, c, 2), lambda: ops.kv8_attn(view, x, 384, c, x, 384, 2, 1.0), lambda: ops.rotary(x, 6, 64, torch.zeros((4, 32, 2)), torch.zeros(1, dtype=torch.int32)),
                 lambda: ops.kv8_unpack(view, c, cache(torch.float16))):
        with pytest.raises(PtError, match="device"):
            call()


P = ctypes.c_void_p(4096)


def kv8(**kw):
    return _lib.Kv8Cache(*[{**dict(pool=4096, scales=4096, page_table=4096, fmt=0, n_kv=2, dim=64, vdim=64, page_size=16, max_pages=4, max_len=0), **kw}[n] for n, _ in _lib.Kv8Cache._fields_])


def view(**kw):
    return _lib.BatchView(*[{**dict(n_seq=1, n_tok=1, cu=4096, start=4096, slot=4096, tok_seq=4096), **kw}[n] for n, _ in _lib.BatchView._fields_])


def refused(fn, args):
    assert fn(ctypes.byref(args), None) == -1
    return _lib.lib().pt_last_error().decode()


BAD_CACHES = [dict(pool=None), dict(scales=None), dict(page_table=None), dict(fmt=2), dict(fmt=-1), dict(n_kv=0), dict(dim=0), dict(dim=257), dict(vdim=300), dict(vdim=0), dict(page_size=0),
              dict(max_pages=0), dict(max_len=65), dict(max_len=-1), dict(page_size=1 << 20, max_pages=1 << 12), dict(scales=4097)]
BAD_VIEWS = [dict(n_seq=0), dict(n_tok=-1), dict(cu=None), dict(start=None), dict(slot=None), dict(tok_seq=None)]


def append_args(at=None, of=None, **kw):
    d = dict(batch=of or view(), cache=at or kv8(), dtype=0, n_head=2, q=4096, k=4096, v=4096, ld=384, q_out=None, q_out_ld=128, rope_dims=0, interleaved=0, rope=None, error_flag=None)
    return _lib.Kv8AppendArgs(*[{**d, **kw}[n] for n, _ in _lib.Kv8AppendArgs._fields_])


def attn_args(at=None, of=None, **kw):
    d = dict(batch=of or view(), cache=at or kv8(), dtype=0, n_head=2, window=0, scale=1.0, softcap=0.0, q=4096, q_ld=128, out=4096, out_ld=128, plain=0, workspace=None, workspace_bytes=0, error_flag=None)
    return _lib.Kv8AttnArgs(*[{**d, **kw}[n] for n, _ in _lib.Kv8AttnArgs._fields_])


def unpack_args(at=None, of=None, **kw):
    d = dict(batch=of or view(), cache=at or kv8(), dtype=0, into=4096, into_table=4096, into_page_size=16, into_max_pages=4, into_max_len=0, error_flag=None)
    return _lib.Kv8UnpackArgs(*[{**d, **kw}[n] for n, _ in _lib.Kv8UnpackArgs._fields_])


@pytest.mark.parametrize("make,fn", [(append_args, "pt_kv8_append"), (attn_args, "pt_kv8_attn"), (unpack_args, "pt_kv8_unpack")])
def test_bad_caches_and_batches(make, fn):
    f = getattr(_lib.lib(), fn)
    for c in BAD_CACHES:
        assert fn in refused(f, make(at=kv8(**c))), c
    for v in BAD_VIEWS:
        assert fn in refused(f, make(of=view(**v))), v
    assert f(None, None) == -1
    for dtype in (3, -1):
        refused(f, make(dtype=dtype))


def test_bad_arguments():
    L = _lib.lib()
    for kw in (dict(k=None), dict(v=None), dict(ld=0), dict(rope_dims=3, rope=4096), dict(rope_dims=66, rope=4096), dict(rope_dims=-2, rope=4096), dict(rope_dims=8), dict(rope_dims=8, rope=4100),
               dict(q_out=4096, q=None), dict(q_out=4096, n_head=0), dict(q_out=4096, q_out_ld=100), dict(q_out=4096, q_out_ld=130)):
        assert "pt_kv8_append" in refused(L.pt_kv8_append, append_args(**kw)), kw
    for kw in (dict(q=None), dict(out=None), dict(n_head=3), dict(n_head=0), dict(q_ld=127), dict(out_ld=100), dict(window=-1), dict(softcap=-1.0), dict(softcap=1e-30), dict(softcap=1e30),
               dict(softcap=math.nan), dict(scale=math.nan), dict(scale=math.inf)):
        refused(L.pt_kv8_attn, attn_args(**kw))
    for kw in (dict(into=None), dict(into_table=None), dict(into_page_size=0), dict(into_max_pages=0), dict(into_max_len=65), dict(into_max_len=-1)):
        refused(L.pt_kv8_unpack, unpack_args(**kw))
    d = dict(rows=1, heads=2, dim=64, dtype=0, x=4096, x_ld=128, out=8192, out_ld=128, position=4096, positions=10, rope_dims=64, interleaved=0, inverse=0, rope=4096, error_flag=None)
    make = lambda **kw: _lib.RotaryArgs(*[{**d, **kw}[n] for n, _ in _lib.RotaryArgs._fields_])
    for kw in (dict(rows=-1), dict(heads=0), dict(dim=0), dict(dim=300), dict(dtype=7), dict(x=None), dict(out=None), dict(position=None), dict(rope=None), dict(positions=0), dict(rope_dims=0),
               dict(rope_dims=5), dict(rope_dims=66), dict(x_ld=127), dict(out_ld=64), dict(out=4096, out_ld=160)):
        assert "pt_rotary" in refused(L.pt_rotary, make(**kw)), kw


def test_outputs_that_others_still_read_are_refused():
    """An output is the input itself, columns of the same wider rows that are none of the input's, or memory of its own."""
    L = _lib.lib()
    d = dict(rows=5, heads=2, dim=64, dtype=0, x=1 << 20, x_ld=400, out=1 << 20, out_ld=400, position=4096, positions=10, rope_dims=64, interleaved=0, inverse=0, rope=4096, error_flag=None)
    make = lambda **kw: _lib.RotaryArgs(*[{**d, **kw}[n] for n, _ in _lib.RotaryArgs._fields_])
    for off, ld in ((2, 400), (254, 400), (2 * 300, 400), (-2, 400), (1, 400), (0, 404), (2 * 128, 401), (2 * 800 + 2, 400)):
        assert "apart" in refused(L.pt_rotary, make(out=(1 << 20) + off, out_ld=ld)), (off, ld)
    for off, ld in ((0, 400), (256, 400), (2 * 272, 400), (-256, 400), (2 * (4 * 400 + 128), 500), (-2 * (4 * 130 + 128), 130)):      # (these pass, and the next check refuses them: nothing is launched)
        assert "0 positions" in refused(L.pt_rotary, make(out=(1 << 20) + off, out_ld=ld, positions=0)), (off, ld)
    at = 1 << 20                                    # q | k | v: 2, 2 and 2 heads of 64 in rows of 384
    rows = dict(of=view(n_tok=3), q=at, k=at + 256, v=at + 512, ld=384, q_out_ld=384)
    for off in (2, 256, 512, 700, -2):
        assert "apart" in refused(L.pt_kv8_append, append_args(**rows, q_out=at + off)), off
    assert "apart" in refused(L.pt_kv8_append, append_args(**{**rows, "q_out_ld": 200}, q_out=at))
    for kw in (dict(q_out=at), dict(q_out=at + 2 * 3 * 384), dict(q_out=at - 2 * 3 * 384)):
        assert "rotated dimensions" in refused(L.pt_kv8_append, append_args(**{**rows, **kw}, rope_dims=3)), kw
    assert "apart" in refused(L.pt_kv8_attn, attn_args(of=view(n_tok=3), q=at, out=at + 2))
    assert "apart" in refused(L.pt_kv8_attn, attn_args(at=kv8(vdim=32), of=view(n_tok=3), q=at, out=at))
    assert "workspace" in refused(L.pt_kv8_attn, attn_args(of=view(n_tok=3), q=at, out=at))


def test_batches_without_tokens():
    L = _lib.lib()
    empty = view(n_tok=0, tok_seq=None)
    for fn, args in ((L.pt_kv8_append, append_args(of=empty)), (L.pt_kv8_attn, attn_args(of=empty, q=4096, out=8192))):
        assert fn(ctypes.byref(args), None) == 0


# ------------------------------------------------------------------------------------------ tables of angles
def test_rope_table():
    t = ops.rope_table(1000, 64, device="cpu")
    a = np.arange(1000)[:, None] * 10000.0 ** (-np.arange(32) / 32)
    assert t.shape == (1000, 32, 2) and np.abs(t.numpy() - np.stack([np.cos(a), np.sin(a)], -1)).max() <= 2.0 ** -24


def angles(t):
    return torch.atan2(t[..., 1].double(), t[..., 0].double())


def test_scaled_tables():
    plain = ops.rope_table(64, 32, device="cpu")
    by = ops.rope_table(256, 32, scaling=dict(kind="linear", factor=4.0), device="cpu")
    assert torch.allclose(by[::4], plain, atol=2.0 ** -22, rtol=0)
    # the base: the fastest pair as before, the slowest `factor` times slower
    by = ops.rope_table(64, 32, scaling=dict(kind="base", factor=8.0), device="cpu")
    f = 10000.0 ** (-np.arange(16) / 16)
    a = angles(by)[1].numpy()
    assert abs(a[0] - 1.0) < 1e-6 and abs(a[-1] - f[-1] / 8) < 1e-9
    # the ramp: fast pairs left, slow ones divided, all between; magnitudes
    by = ops.rope_table(64, 128, scaling=dict(kind="ramp", factor=16.0, original=4096), device="cpu")
    f = 10000.0 ** (-np.arange(64) / 64)
    a, turns = angles(by)[1].numpy(), 4096 * f / (2 * math.pi)
    assert np.allclose(by.double().norm(dim=-1).numpy(), 0.1 * math.log(16.0) + 1, atol=1e-6)
    assert np.allclose(a[turns > 40], f[turns > 40], rtol=1e-5) and np.allclose(a[turns < 0.8], f[turns < 0.8] / 16, rtol=1e-4)
    assert (a <= f * (1 + 1e-5)).all() and (a >= f / 16 * (1 - 1e-4)).all() and (np.diff(a) < 0).all()
    assert np.allclose(ops.rope_table(9, 128, scaling=dict(kind="ramp", factor=16.0, original=4096, magnitude=1.0), device="cpu").double().norm(dim=-1).numpy(), 1.0, atol=1e-6)


def test_bands_are_those_of_the_decoders():
    from poptransformer_b200.padetar import rope_frequencies
    s = dict(factor=8.0, low=1.0, high=4.0, original=512)
    f = rope_frequencies(64, 10000.0, s)
    a = np.arange(300)[:, None] * f
    t = ops.rope_table(300, 64, scaling=dict(kind="bands", **s), device="cpu")
    assert np.abs(t.numpy() - np.stack([np.cos(a), np.sin(a)], -1)).max() <= 2.0 ** -23


def test_tables_that_are_refused():
    for args, kw in (((8, 8), dict(base=0.0)), ((8, 8), dict(scaling=dict(kind="linear", factor=0.0))), ((8, 8), dict(scaling=dict(kind="ramp", factor=2.0, original=-5))),
                     ((0, 8), {}), ((8, 7), {}), ((8, 0), {}), ((8, 8), dict(scaling=dict(kind="no"))), ((8, 8), dict(scaling=dict(kind="linear"))), ((8, 8), dict(scaling=dict(factor=2.0))),
                     ((8, 2), dict(scaling=dict(kind="base", factor=2.0))), ((8, 8), dict(scaling=dict(kind="bands", factor=2.0, original=8, low=1)))):
        with pytest.raises(PtError):
            ops.rope_table(*args, device="cpu", **kw)
