"""Argument checks of the entry points that take a 4-bit weight's row offsets (no GPU: the
C functions refuse before they touch a device)."""

import ctypes

import pytest

from moe_b200._lib import lib

BAD = -1
P = 1 << 20  # an address that no call here may follow


def host(*off):
    return (ctypes.c_int32 * len(off))(*off)


def few(**kw):
    a = dict(x=P, T=2, ldx=64, H=64, router=P, rdt=0, E=4, w1=P, s1=P, w2=P, s2=P, group=64,
             rows=host(0, 32, 64, 96, 128), total=128, off=P, mw=32, k=2, norm=1, act=1, out=P,
             ldo=64, ws=P, wsb=1 << 30, dtype=0, status=None, stream=None)
    a.update(kw)
    return lib.moe_few_tokens_int4(*a.values())


@pytest.mark.parametrize("kw", [
    dict(rows=None), dict(rows=host(0, 32, 64, 96, 112)), dict(rows=host(16, 32, 64, 96, 128)),
    dict(rows=host(0, 32, 24, 96, 128)), dict(rows=host(0, 40, 64, 96, 128)), dict(group=0),
    dict(group=16), dict(act=2), dict(act=3), dict(act=-1), dict(total=136), dict(E=0),
    dict(E=257, rows=host(*range(0, 258 * 16, 16)), total=257 * 16), dict(s1=None), dict(s2=P + 2),
    dict(T=65), dict(T=-1), dict(H=24), dict(k=5), dict(ldx=48), dict(ws=None), dict(wsb=64),
])
def test_few_tokens_int4_refuses(kw):
    assert few(**kw) == BAD


def test_few_tokens_int4_unsupported_types_and_no_tokens():
    assert few(dtype=2, rdt=2) == -2
    assert few(rdt=1) == -2 and few(dtype=1, rdt=0) == -2 and few(dtype=2) == -2
    assert few(T=0) == 0
    assert few(T=0, act=2, rows=host(0, 0, 32, 48, 64)) == 0
    assert few(T=0, E=1, k=1, rows=None) == 0


def down(**kw):
    a = dict(x=P, rows=2, ldx=32, w=P, s=P, group=64, off_rows=host(0, 32, 64, 96, 128), H=64,
             total=128, tok=P, off=P, cnt=None, E=4, mw=32, out=P, ldo=64, ws=P, wsb=1 << 30,
             dtype=0, status=None, stream=None)
    a.update(kw)
    return lib.moe_grouped_gemv_down_int4(*a.values())


@pytest.mark.parametrize("kw", [
    dict(off_rows=None), dict(off_rows=host(0, 32, 64, 96, 112)), dict(total=144), dict(E=3),
    dict(E=0), dict(group=16), dict(rows=-1), dict(rows=65537), dict(ldx=24), dict(ldo=48),
    dict(w=None), dict(s=P + 4), dict(tok=None), dict(ws=P + 4), dict(wsb=100), dict(mw=40),
])
def test_down_product_refuses(kw):
    assert down(**kw) == BAD


def test_down_product_unsupported_types_and_no_rows():
    assert down(dtype=2) == -2
    assert down(rows=0) == 0
    assert down(rows=0, E=1, off_rows=None) == 0
