"""The 4-bit cache's and the packed attention's entry points where no GPU is
needed: sizes, and arguments refused before anything is launched."""
import ctypes

import pytest

from freeml_b200 import _lib

P = 0x10000  # an aligned address that is never read: the calls below return before a launch
F = ctypes.c_float


def rc(name, *args):
    return getattr(_lib.load(), name)(*args)


def test_sizes():
    lib = _lib.load()
    for hd in (32, 64, 128):
        for page in (16, 32, 64, 128):
            assert lib.fml_kv4_block_bytes(hd, page) == page * hd * 5 // 4
    assert lib.fml_kv4_block_bytes(48, 16) == 0 and lib.fml_kv4_block_bytes(64, 24) == 0
    # a context that is never split needs no workspace; a longer one does, more for more heads
    assert lib.fml_attention_kv4_workspace_bytes(4, 8, 8, 64, 1, 16) == 0
    small, large = (lib.fml_attention_kv4_workspace_bytes(4, h, h, 64, 1000, 64) for h in (8, 64))
    assert 0 < small < large
    assert lib.fml_kv4_pages_workspace_bytes(1000, 0) >= 4 * 2000
    assert lib.fml_kv4_pages_workspace_bytes(1000, 7) >= 4 * (1000 + 5 * 7)


def packed(out=P, q=P, k=P, v=P, kind=2, starts=P, batch=1, rows=8, k_rows=8, heads=4, kv=2, hd=64, ldo=256, ldq=256, ldk=128,
           ldv=128, mode=1):
    return rc("fml_attention_packed", out, q, k, v, kind, starts, None, batch, rows, k_rows, heads, kv, hd, ldo, ldq, ldk, ldv,
              F(0.1), mode, None)


@pytest.mark.parametrize("bad", [dict(out=None), dict(q=None), dict(k=None), dict(starts=None), dict(kind=3), dict(hd=48),
                                 dict(heads=3), dict(kv=0), dict(heads=1), dict(ldq=255), dict(ldv=64), dict(mode=7),
                                 dict(rows=1 << 31), dict(k_rows=1 << 31)])
def test_packed_attention_refuses(bad):
    assert packed(**bad) == 1
    assert b"fml_attention_packed" in _lib.load().fml_last_error()


def test_nothing_to_do():
    assert packed(batch=0, q=None) == 0 and packed(rows=0, q=None) == 0
    assert rows_call(batch=0, pool=None) == 0 and rows_call(rows=0, pool=None) == 0
    assert attention(batch=0, q=None) == 0


def rows_call(pool=P, table=P, lens=P, k=P, v=P, kind=0, starts=P, batch=2, rows=4, ldk=128, ldv=128, pages=4, slots=2, most=2,
              page=16, kv=2, hd=64):
    return rc("fml_kv4_append", pool, table, lens, None, k, v, kind, starts, batch, rows, ldk, ldv, pages, slots, most, page, kv,
              hd, None)


@pytest.mark.parametrize("bad", [dict(pool=None), dict(pool=P + 8), dict(table=None), dict(lens=None), dict(k=None),
                                 dict(starts=None), dict(kind=-1), dict(page=24), dict(hd=16), dict(pages=0), dict(slots=0),
                                 dict(kv=0), dict(ldk=127), dict(most=1 << 28)])
def test_rows_refuse(bad):
    assert rows_call(**bad) == 1


def attention(out=P, q=P, kind=0, ldo=256, ldq=256, pool=P, table=P, lens=P, batch=2, pages=4, slots=2, most=64, page=64, heads=4,
              kv=2, hd=64, ws=P, size=1 << 30):
    return rc("fml_attention_kv4", out, q, kind, ldo, ldq, pool, table, lens, None, batch, pages, slots, most, page, heads, kv, hd,
              F(0.1), ws, size, None)


@pytest.mark.parametrize("bad", [dict(out=None), dict(q=None), dict(pool=P + 4), dict(kind=9), dict(ldo=255), dict(heads=3),
                                 dict(kv=0), dict(hd=96), dict(page=8), dict(pages=0), dict(ws=None), dict(ws=P + 8),
                                 dict(size=64), dict(most=1 << 27)])
def test_cache_attention_refuses(bad):
    assert attention(**bad) == 1


def pages_call(name, **bad):
    a = dict(pool=P, layers=2, stride=1 << 20, page_bytes=1280, refs=P, table=P, lens=P, a=P, b=P, n=2, pages=16, slots=4, most=4,
             page=16, status=P, ws=P, size=1 << 20)
    a.update(bad)
    if name == "fml_kv4_reserve":
        return rc(name, a["refs"], a["table"], a["lens"], a["a"], a["b"], a["n"], a["pages"], a["slots"], a["most"], a["page"],
                  a["status"], a["ws"], a["size"], None)
    if name == "fml_kv4_fork":
        return rc(name, a["pool"], a["layers"], a["stride"], a["page_bytes"], a["refs"], a["table"], a["lens"], a["a"], a["b"],
                  a["n"], a["pages"], a["slots"], a["most"], a["page"], a["status"], a["ws"], a["size"], None)
    return rc(name, a["pool"], a["layers"], a["stride"], a["page_bytes"], a["refs"], a["table"], a["pages"], a["slots"],
              a["most"], a["ws"], a["size"], None)


@pytest.mark.parametrize("name", ["fml_kv4_reserve", "fml_kv4_fork", "fml_kv4_compact"])
def test_page_operations_refuse(name):
    common = [dict(refs=None), dict(table=None), dict(pages=0), dict(pages=(1 << 21) + 1), dict(slots=0), dict(ws=None),
              dict(ws=P + 4), dict(size=8)]
    lists = [dict(lens=None), dict(b=None), dict(status=None), dict(page=20), dict(most=1 << 28), dict(n=1 << 30)]
    pools = [dict(pool=None), dict(pool=P + 1), dict(layers=0), dict(page_bytes=1288), dict(page_bytes=0),
             dict(stride=(1 << 20) + 8), dict(stride=1280)]
    for bad in common + (lists if name != "fml_kv4_compact" else []) + (pools if name != "fml_kv4_reserve" else []):
        assert pages_call(name, **bad) == 1, (name, bad)
    if name != "fml_kv4_compact":
        assert pages_call(name, n=0, refs=None) == 0


def test_free_refuses():
    for bad in (0, 1, 2, 9):
        args = [P, P, P, P, 2, 16, 4, 4, 0, P, None]
        args = [P, P, P, P, 2, 16, 4, 4, P, None]
        args[bad if bad != 9 else 8] = None
        assert rc("fml_kv4_free", *args) == 1
    assert rc("fml_kv4_free", None, None, None, None, 0, 0, 0, 0, None, None) == 0


def test_the_keeping_forms_refuse():
    """As the plain forms do, and without `kept`."""
    rows = [P, P, P, None, P, P, P, 0, P, 2, 4, 128, 128, 4, 2, 2, 16, 2, 64, None]
    for at in (0, 1, 2, 4, 5, 6, 8):
        assert rc("fml_kv4_append_keeping", *rows[:at], None, *rows[at + 1:]) == 1
    assert b"fml_kv4_append_keeping" in _lib.load().fml_last_error()
    assert rc("fml_kv4_append_keeping", *rows[:4], None, *rows[5:9], 0, *rows[10:]) == 0
    reserve = [P, P, P, P, P, P, 2, 16, 4, 4, 16, P, P, 1 << 20, None]
    for at in (0, 1, 2, 3, 5, 11, 12):
        assert rc("fml_kv4_reserve_keeping", *reserve[:at], None, *reserve[at + 1:]) == 1
    assert b"fml_kv4_reserve_keeping" in _lib.load().fml_last_error()
    assert rc("fml_kv4_reserve_keeping", *reserve[:6], 0, *reserve[7:]) == 0
