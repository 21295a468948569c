"""Refusals of the speculative entry points, before anything is launched, and pages that sequences share."""
import ctypes
import random

import pytest
import torch

from poptransformer_b200 import _lib, ops
from poptransformer_b200.cache import SequenceSlots

P = 1 << 20      # an address that nothing reads


def _view(n_seq=2, n_tok=6):
    v = _lib.BatchView()
    v.n_seq, v.n_tok, v.cu, v.start, v.slot, v.tok_seq = n_seq, n_tok, P, P, P, P
    return v


def _attn(**kw):
    a = _lib.TreeAttnArgs()
    a.batch, a.dtype, a.n_head, a.n_kv, a.dim, a.vdim, a.page_size, a.max_pages, a.scale = _view(), ops.DT_BF16, 8, 2, 64, 64, 64, 10, 0.125
    a.q = a.k = a.v = a.pool = a.page_table = a.out = a.workspace = a.rope = P
    a.q_ld, a.kv_ld, a.out_ld, a.workspace_bytes = 8 * 64, 8 * 64, 8 * 64, 1 << 40
    for k, v in kw.items():
        setattr(a, k, v)
    return _lib.lib().pt_tree_attn(ctypes.byref(a), None), _lib.lib().pt_last_error().decode()


@pytest.mark.parametrize("kw,word", [
    (dict(batch=_view(0)), "bad batch"), (dict(batch=_view(1025, 2000)), "bad batch"), (dict(batch=_view(2, 0)), "bad batch"), (dict(n_head=7), "multiple"), (dict(n_kv=0), "multiple"),
    (dict(dim=0), "bad shape"), (dict(dim=264), "bad shape"), (dict(vdim=257), "bad shape"), (dict(page_size=0), "bad shape"), (dict(max_pages=0), "bad shape"), (dict(dtype=7), "type"),
    (dict(q=None), "null"), (dict(k=None), "null"), (dict(pool=None), "null"), (dict(out=None), "null"), (dict(page_table=None), "null"), (dict(q_ld=511), "strides"),
    (dict(kv_ld=127), "strides"), (dict(out_ld=511), "strides"), (dict(window=-1), "window"), (dict(softcap=-1.0), "softcap"), (dict(rope_dims=3), "rotated"), (dict(rope_dims=66), "rotated"),
    (dict(rope_dims=64, rope=None), "rotated"), (dict(max_len=641), "positions"), (dict(max_tokens_per_seq=257), "at most 256"), (dict(batch=_view(2, 300)), "at most 256"),
    (dict(out_cols=100), "out_cols"), (dict(out_cols=513), "out_cols"), (dict(workspace=None), "workspace"), (dict(workspace_bytes=100), "workspace"), (dict(workspace=P + 8), "workspace"),
    (dict(batch=_view(1024, 200000), max_tokens_per_seq=256, max_pages=1 << 20, n_kv=8), "too much")])
def test_tree_attn_refuses(kw, word):
    rc, said = _attn(**kw)
    assert rc == -1 and word in said, said


@pytest.mark.parametrize("softcap", [1e-30, 1e30, float("inf"), float("nan")])
def test_tree_attn_refuses_caps_that_fp32_cannot_divide_by(softcap):
    rc, said = _attn(softcap=softcap)
    assert rc == -1 and "softcap" in said, said


def test_tree_attn_refuses_positions_that_an_int_cannot_round_up():
    rc, said = _attn(page_size=(1 << 31) - 512, max_pages=1, max_len=100)
    assert rc == -1 and "positions" in said, said


def _verify(**kw):
    a = _lib.VerifyArgs()
    a.n_seq, a.n_tok, a.dtype, a.vocab, a.logits_ld, a.draft_ld, a.max_path = 2, 8, ops.DT_F32, 100, 100, 100, 4
    for f in ("cu", "logits", "token", "parent", "draft", "temperature", "uniform", "uniform_next", "path", "count", "out_token", "logprob"):
        setattr(a, f, P)
    for k, v in kw.items():
        setattr(a, k, v)
    return _lib.lib().pt_verify_drafts(ctypes.byref(a), None), _lib.lib().pt_last_error().decode()


@pytest.mark.parametrize("kw,word", [(dict(n_seq=0), "n_seq"), (dict(n_tok=-1), "n_tok"), (dict(vocab=0), "vocab"), (dict(max_path=0), "max_path"), (dict(cu=None), "null"),
                                     (dict(logits=None), "null"), (dict(token=None), "null"), (dict(path=None), "null"), (dict(count=None), "null"), (dict(out_token=None), "null"),
                                     (dict(dtype=5), "type"), (dict(logits_ld=99), "strides"), (dict(draft_ld=99), "strides"), (dict(uniform=None), "sampling"),
                                     (dict(uniform_next=None), "sampling")])
def test_verify_refuses(kw, word):
    rc, said = _verify(**kw)
    assert rc == -1 and word in said, said


def test_pages_refuse():
    L = _lib.lib()
    pool = lambda **kw: (_lib.KvPool * 1)(_lib.KvPool(**{**dict(pool=P, n_kv=2, dim=64, vdim=64, elem_bytes=2), **kw}))
    copy = lambda pools, n=3, page=64, pages=10, src=P, dst=P, k=1: L.pt_kv_copy_pages(pools, k, page, pages, src, dst, n, None, None)
    assert copy(pool(), n=0) == 0                      # nothing to do, nothing launched
    for rc in (copy(None), copy(pool(), k=0), copy(pool(), n=-1), copy(pool(), page=0), copy(pool(), pages=0), copy(pool(), src=None), copy(pool(), dst=None), copy(pool(pool=None)),
               copy(pool(n_kv=0)), copy(pool(dim=0)), copy(pool(vdim=-1)), copy(pool(elem_bytes=3)), copy(pool(dim=1 << 30))):
        assert rc == -1
    move = lambda pools, view, page=64, pages=10, table=P, path=P, ld=4, count=P: L.pt_kv_move_rows(pools, 1, page, pages, table, ctypes.byref(view) if view else None, path, ld, count, None, None)
    for rc in (move(None, _view()), move(pool(), None), move(pool(), _view(0)), move(pool(), _view(), page=0), move(pool(), _view(), pages=0), move(pool(), _view(), table=None),
               move(pool(), _view(), path=None), move(pool(), _view(), ld=0), move(pool(), _view(), count=None), move(pool(), _view(), page=1 << 16, pages=1 << 16)):
        assert rc == -1


def test_python_refuses():
    i32 = lambda *shape: torch.zeros(shape, dtype=torch.int32)
    logits = torch.zeros((4, 10))
    for kw in (dict(token=i32(3)), dict(parent=i32(3)), dict(draft=torch.zeros(4, 9)), dict(temperature=torch.ones(2)), dict(token=torch.zeros(4)), dict(parent=torch.zeros(4)),
               dict(temperature=torch.ones(2), uniform=torch.zeros(4), uniform_next=torch.zeros(1)), dict(draft=torch.zeros(4, 10).half()),
               dict(out=(i32(2, 3), i32(2), i32(2, 4), torch.zeros(2, 3))), dict(max_path=2, out=(i32(2, 3), i32(2), i32(2, 3), torch.zeros(2, 3)))):
        with pytest.raises(ops.PtError):
            ops.verify_drafts(**{**dict(logits=logits, cu=i32(3), token=i32(4)), **kw})
    with pytest.raises(ops.PtError):
        ops.PagePools([])
    with pytest.raises(ops.PtError):
        ops.PagedKVCache(1, 2, 64, 64, device="cpu", pool=torch.zeros((3, 2, 2, 64, 32), dtype=torch.float16))


class Model:
    """Slots beside what their pages hold, one number per position: a plain model of what a decoder writes."""

    def __init__(self, seqs, max_len, page, n_pages):
        self.slots, self.page = SequenceSlots(seqs, max_len, page, n_pages, device="cpu"), page
        self.pool = torch.zeros((n_pages, page), dtype=torch.int64)
        self.want, self.next = {}, 1

    def copy(self, pairs):
        dst = [b for _, b in pairs]
        assert len(set(dst)) == len(dst) and not set(dst) & {a for a, _ in pairs}
        for a, b in pairs:
            self.pool[b] = self.pool[a]

    def open(self):
        s = self.slots.open()
        self.want[s] = []
        return s

    def extend(self, s, n):
        start = self.slots.extend(s, n)
        assert start == len(self.want[s])
        for j in range(start, start + n):
            self.pool[self.slots.page_table[s, j // self.page], j % self.page] = self.next
            self.want[s].append(self.next)
            self.next += 1

    def check(self):
        for s, w in self.want.items():
            assert self.slots.length[s] == len(w)
            got = [int(self.pool[self.slots.page_table[s, j // self.page], j % self.page]) for j in range(len(w))]
            assert got == w
        used = {int(self.slots.page_table[s, j]) for s, w in self.want.items() for j in range(-(-len(w) // self.page))}
        assert len(used) + self.slots.free_pages == self.slots.n_pages and not used & set(self.slots._free_pages)


@pytest.mark.parametrize("seed", range(6))
def test_slots_fork_truncate_compact(seed):
    rng = random.Random(seed)
    m = Model(6, 40, 4, 30)
    refused = 0
    for _ in range(400):
        live = list(m.want)
        what = rng.choice(["open", "extend", "extend", "extend", "fork", "truncate", "truncate", "close", "compact"])
        try:
            if what == "open":
                m.open()
            elif what == "compact":
                m.copy(m.slots.compact())
                used = m.slots.n_pages - m.slots.free_pages
                assert all(int(p) < used for s, w in m.want.items() for p in m.slots.page_table[s, :-(-len(w) // m.page)])
            elif live:
                s = rng.choice(live)
                if what == "extend":
                    m.extend(s, rng.randint(1, 9))
                elif what == "fork":
                    n = rng.randint(0, len(m.want[s]))
                    new, pairs = m.slots.fork(s, n)
                    m.copy(pairs)
                    m.want[new] = m.want[s][:n]
                elif what == "truncate":
                    n = rng.randint(0, len(m.want[s]))
                    m.copy(m.slots.truncate(s, n))
                    del m.want[s][n:]
                elif what == "close":
                    m.slots.close(s)
                    del m.want[s]
        except ops.PtError:
            refused += 1
        m.check()
    assert refused
    for s in list(m.want):
        m.slots.close(s)
    assert m.slots.free_pages == 30 and not m.slots._owners


def test_slots_refuse():
    m = Model(2, 12, 4, 3)
    a = m.open()
    m.extend(a, 6)
    for n in (-1, 7):
        with pytest.raises(ops.PtError):
            m.slots.fork(a, n)
        with pytest.raises(ops.PtError):
            m.slots.truncate(a, n)
    b, pairs = m.slots.fork(a)                         # shares a page, copies one: the pool is empty
    m.copy(pairs)
    m.want[b] = list(m.want[a])
    with pytest.raises(ops.PtError):                   # no slot
        m.slots.fork(a)
    with pytest.raises(ops.PtError):                   # no page
        m.slots.extend(a, 3)
    m.check()
    m.copy(m.slots.truncate(a, 2))                     # a page of its own again: it gives one back and takes it
    del m.want[a][2:]
    m.check()
    m.copy(m.slots.truncate(b, 3))                     # now b alone has the shared page
    del m.want[b][3:]
    m.check()
