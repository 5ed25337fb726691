"""The refusals of the C entry points of rotary positions, pages and drafts: every one before any
device work, so they need no GPU."""
from __future__ import annotations

import pytest

from model import _hip as H

P = 4096  # a pointer that is never followed


@pytest.fixture(scope="module")
def lib():
    if not H.LIB_PATH.exists():
        import __graft_entry__
        __graft_entry__.build()
    return H.load()


def rotary(lib, **kw):
    a = dict(q=P, q_t=128, q_h=64, k=P, k_t=64, k_h=64, cos=P, sin=P, stride=32, rows=10, tab=0, pos=P, pb=4, qo=P, ko=P,
             T=1, heads=2, kv=1, hd=64, rd=64, flags=0, dtype=1, stream=None)
    a.update(kw)
    return lib.mhc_rotary(*a.values())


def append(lib, **kw):
    a = dict(q=P, q_t=128, q_h=64, k=P, k_t=64, k_h=64, v=P, v_t=64, v_h=64, qg=None, kg=None, gd=0, eps=1e-6, cos=P, sin=P,
             stride=32, rows=10, tab=0, cu=P, lens=P, depths=None, table=P, qo=P, kp=P, vp=P, sp=1024, st=64, sh=64, T=1, B=1,
             heads=2, kv=1, hd=64, rd=64, width=2, pages=3, page=16, flags=0, dtype=1, stream=None)
    a.update(kw)
    return lib.mhc_paged_append(*a.values())


def attend(lib, **kw):
    a = dict(q=P, q_t=128, q_h=64, k=P, v=P, sp=1024, st=64, sh=64, table=P, lens=P, cu=P, tree=None, words=0, out=P, ws=P,
             nbytes=0, B=1, Tq=1, heads=2, kv=1, hd=64, width=2, pages=3, page=16, dtype=1, scale=0.1, stream=None)
    a.update(kw)
    return lib.mhc_paged_attn_fwd(*a.values())


def keep(lib, **kw):
    a = dict(planes=P, table=P, lens=P, cu=P, kept=P, path=P, new=P, T=1, B=1, n=2, plane=4096, row=128, width=2, pages=3,
             page=16, stream=None)
    a.update(kw)
    return lib.mhc_paged_keep(*a.values())


def verify(lib, **kw):
    a = dict(p=P, q=None, dtype=0, tokens=P, parents=None, u=None, cu=P, kept=P, path=P, next=P, T=1, V=10, B=1, stream=None)
    a.update(kw)
    return lib.mhc_verify_drafts(*a.values())


BAD = [
    (rotary, [dict(T=-1), dict(heads=-1), dict(hd=0), dict(rd=63), dict(rd=66), dict(rd=-2), dict(dtype=3), dict(tab=7), dict(pb=2),
              dict(cos=None), dict(q=None), dict(ko=None), dict(pos=None), dict(stride=-1), dict(T=(1 << 30) + 1),
              dict(T=1 << 30, heads=1 << 20)]),
    (append, [dict(T=-1), dict(T=(1 << 29) + 1), dict(B=-1), dict(width=-1), dict(pages=-1), dict(page=8), dict(page=24),
              dict(page=1 << 21), dict(width=1 << 26), dict(sp=4), dict(st=-8), dict(st=1 << 23), dict(sh=12), dict(dtype=0),
              dict(heads=0), dict(kv=0), dict(qg=P, gd=9), dict(q=None), dict(v=None), dict(qo=None), dict(cu=None),
              dict(lens=None), dict(table=None), dict(kp=None), dict(sin=None)]),
    (attend, [dict(Tq=-1), dict(Tq=(1 << 29) + 1), dict(hd=80), dict(heads=3, kv=2), dict(kv=0), dict(dtype=0), dict(page=15),
              dict(scale=0.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(tree=P), dict(tree=P, words=-1),
              dict(q_t=4), dict(q_h=-8), dict(q_t=1 << 23), dict(st=1 << 23), dict(q=None), dict(q=P + 8), dict(k=P + 2),
              dict(out=None), dict(cu=None), dict(lens=None), dict(table=None), dict(width=1 << 26), dict(B=-1),
              dict(Tq=1 << 28, heads=16)]),
    (keep, [dict(T=-1), dict(n=-1), dict(row=8), dict(row=130), dict(row=1 << 25), dict(plane=100), dict(page=0), dict(planes=P + 4),
            dict(planes=None), dict(lens=None), dict(cu=None), dict(kept=None), dict(path=None), dict(new=None), dict(table=None)]),
    (verify, [dict(T=-1), dict(V=0), dict(V=(1 << 28) + 1), dict(B=-1), dict(B=1 << 22), dict(dtype=5), dict(q=P), dict(p=None),
              dict(p=P + 4), dict(q=P + 2, u=P), dict(tokens=None), dict(cu=None), dict(kept=None), dict(path=None), dict(next=None)]),
]


@pytest.mark.parametrize("call,args", [(c, a) for c, all_ in BAD for a in all_],
                         ids=lambda x: x.__name__ if callable(x) else "-".join(f"{k}={v}" for k, v in x.items()))
def test_refused(lib, call, args):
    assert call(lib, **args) == 1
    assert lib.mhc_last_error()


def test_nothing_to_do(lib):
    assert rotary(lib, T=0, q=None, k=None) == 0
    assert append(lib, T=0, q=None) == 0
    assert attend(lib, Tq=0, q=None) == 0
    assert keep(lib, B=0, lens=None) == 0
    assert verify(lib, B=0, p=None) == 0


def test_workspace_sizes(lib):
    ask = lib.mhc_paged_attn_workspace_bytes
    assert ask(1, 0, 8, 4, 96) == 0 and ask(64, 64, 8, 4, 96) > 0
    assert ask(300, 300, 8, 4, 96) == 0      # a workgroup a sequence and head fills the chip
    for bad in ((-1, 1, 8, 4, 96), (1, -1, 8, 4, 96), (1, 1, 8, 3, 96), (1, 1, 8, 4, 80), (1, 1 << 29, 16, 4, 96)):
        assert ask(*bad) == -1
    assert attend(lib, ws=None, nbytes=0) == 1 and attend(lib, nbytes=16) == 1
