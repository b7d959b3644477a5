"""Argument checks of the few-token and 4-bit entry points that need no GPU: the
C functions refuse before they touch a device."""

import copy
import ctypes
import pickle

import pytest
import torch

from moe_b200._lib import lib
from moe_b200.kernels import Int4Weight, moe_few_tokens, quantize_int4

BAD = -1


def rows(K, group, off=None):
    b, g = ctypes.c_int64(-7), ctypes.c_int64(-7)
    arr = None if off is None else (ctypes.c_int32 * len(off))(*off)
    rc = lib.moe_int4_rows(K, group, arr, 1 if off is None else len(off) - 1,
                           ctypes.addressof(b), ctypes.addressof(g))
    return (b.value, g.value) if rc == 0 else rc


def test_int4_rows():
    assert rows(64, 64) == (1, 1)
    assert rows(80, 32) == (2, 3)
    assert rows(1104, 128) == (18, 9)
    assert rows(336, 128, [0, 48, 64, 64, 208, 336]) == (1 + 1 + 0 + 3 + 2, 1 + 1 + 0 + 2 + 1)
    for bad in [(0, 64), (24, 64), (64, 16), (64, 96), (-16, 32)]:
        assert rows(*bad) == BAD
    for off in ([0, 32], [0, 24, 64], [16, 64], [0, 48, 32, 64], [0, 80], [0] * 258):
        assert rows(64, 32, off) == BAD


def test_workspace_sizes():
    f = lib.moe_few_tokens_workspace_bytes
    assert f(1, 16, 1, 1, 16, 0) > 0
    a, b = f(1, 768, 16, 2, 512, 1), f(64, 768, 16, 2, 512, 1)
    assert 0 < a < b
    for bad in [(65, 64, 4, 2, 32, 0), (-1, 64, 4, 2, 32, 0), (1, 24, 4, 2, 32, 0),
                (1, 64, 257, 2, 32, 0), (1, 64, 4, 5, 32, 0), (1, 64, 64, 33, 32, 0),
                (1, 64, 4, 0, 32, 0), (1, 64, 4, 2, 40, 0), (1, 64, 4, 2, 32, 3),
                (1, 32784, 4, 2, 32, 0), (1, 64, 4, 2, 32784, 0)]:
        assert f(*bad) == -1, bad
    g = lib.moe_grouped_gemv_int4_workspace_bytes
    assert g(1, 16, 16, 0, 1) > 0 and g(0, 16, 16, 2, 0) > 0
    for bad in [(-1, 16, 16, 0, 0), (65537, 16, 16, 0, 0), (1, 8, 16, 0, 0), (1, 16, 40, 0, 0),
                (1, 32784, 16, 0, 0), (1, 16, 32784, 0, 0), (1, 16, 16, 3, 0), (1, 16, 16, 1, 1)]:
        assert g(*bad) == -1, bad


# Addresses that no call here may follow: every call is refused on its arguments.
P = 1 << 20


def few(**kw):
    a = dict(x=P, T=2, ldx=64, H=64, router=P, E=4, w1=P, s1=None, w2=P, s2=None, group=0, b2=0,
             g2=0, total=128, off=P, mw=32, k=2, norm=1, act=1, out=P, ldo=64, ws=P, wsb=1 << 30,
             dtype=0, status=None, stream=None)
    a.update(kw)
    return lib.moe_few_tokens(*a.values())


@pytest.mark.parametrize("kw", [
    dict(T=65), dict(T=-1), dict(H=24), dict(H=0), dict(E=0), dict(E=257), dict(k=0), dict(k=5),
    dict(mw=0), dict(mw=40), dict(act=3), dict(act=-1), dict(x=None), dict(router=None),
    dict(w1=None), dict(w2=None), dict(off=None), dict(out=None), dict(ws=None), dict(wsb=64),
    dict(total=0), dict(total=40), dict(ldx=48), dict(ldx=65), dict(ldo=48), dict(x=P + 2),
    dict(w1=P + 8), dict(w2=P + 4), dict(router=P + 2), dict(ws=P + 4), dict(group=16),
    dict(group=64), dict(group=64, s1=P), dict(group=64, s1=P, s2=P, b2=-1),
])
def test_few_tokens_refuses(kw):
    assert few(**kw) == BAD


def test_few_tokens_unsupported_types_and_no_tokens():
    assert few(dtype=3, ldx=64) == -2
    assert few(dtype=2, group=64, s1=P, s2=P, b2=4, g2=4) == -2
    assert few(T=0) == 0


def gemv(**kw):
    a = dict(x=P, rows=2, ldx=64, w=P, s=P, group=64, blocks=1, groups=1, H=64, total=128, tok=P,
             off=P, cnt=None, E=4, mw=32, act=1, down=0, out=P, ldo=32, ws=P, wsb=1 << 30, dtype=0,
             status=None, stream=None)
    a.update(kw)
    return lib.moe_grouped_gemv_int4(*a.values())


@pytest.mark.parametrize("kw", [
    dict(rows=-1), dict(rows=65537), dict(H=24), dict(total=40), dict(E=0), dict(E=257),
    dict(mw=40), dict(act=3), dict(down=1, ldo=64), dict(group=0), dict(group=16), dict(x=None),
    dict(w=None), dict(s=None), dict(tok=None), dict(off=None), dict(out=None), dict(ws=None),
    dict(wsb=100), dict(ldx=48), dict(ldx=65), dict(ldo=16), dict(x=P + 2), dict(blocks=-1),
    dict(blocks=0), dict(groups=0), dict(group=32),
])
def test_gemv_refuses(kw):
    assert gemv(**kw) == BAD


def test_gemv_unsupported_types_and_no_rows():
    assert gemv(dtype=2) == -2
    assert gemv(rows=0) == 0


def test_quantize_refuses():
    q = lib.moe_int4_quantize
    assert q(None, 64, 64, 64, 0, 64, None, 1, P, P, 0, None) == BAD
    assert q(P, 64, 64, 48, 0, 64, None, 1, P, P, 0, None) == BAD
    assert q(P, 64, 64, 65, 0, 64, None, 1, P, P, 0, None) == BAD
    assert q(P + 2, 64, 64, 64, 0, 64, None, 1, P, P, 0, None) == BAD
    assert q(P, 64, 24, 24, 0, 64, None, 1, P, P, 0, None) == BAD
    assert q(P, 64, 64, 64, 0, 64, None, 1, P, P, 1, None) == -2
    assert lib.moe_int4_pack(P, 64, 64, 40, 64, None, 1, P, None) == BAD
    assert lib.moe_int4_dequantize(P, P, 64, 64, 64, None, 1, P, 64, 2, None) == -2
    assert lib.moe_int4_dequantize(P, None, 64, 64, 64, None, 1, P, 64, 0, None) == BAD


def test_weights_copy_and_pickle():
    rows = (0, 48, 64, 144)  # 1 + 1 + 2 block rows, 2 + 1 + 3 groups of 32
    q = Int4Weight(torch.randint(0, 256, (4, 2, 512), dtype=torch.uint8),
                   torch.randn(6, 32).bfloat16(), 144, 32, 32, rows)
    for c in (copy.deepcopy(q), pickle.loads(pickle.dumps(q)), q.to("cpu")):
        assert c.shape == (144, 32) and c.group_size == 32 and c.row_offsets == rows
        assert torch.equal(c.packed, q.packed) and torch.equal(c.scales, q.scales)
        assert list(c._segments()[0]) == list(rows) and c._segments()[1] == 3
    with pytest.raises(ValueError, match="packed"):
        Int4Weight(q.packed[:3], q.scales, 144, 32, 32, rows)
    with pytest.raises(ValueError, match="scales"):
        Int4Weight(q.packed, q.scales[:5], 144, 32, 32, rows)
    with pytest.raises(TypeError, match="bf16"):
        Int4Weight(q.packed, q.scales.float(), 144, 32, 32, rows)


def test_cpu_tensors_are_refused():
    x = torch.randn(2, 64)
    with pytest.raises(ValueError, match="CUDA"):
        moe_few_tokens(x, torch.randn(4, 64), torch.randn(64, 128), torch.randn(128, 64),
                       torch.tensor([0, 32, 64, 96, 128], dtype=torch.int32), 32, 2)
    with pytest.raises(ValueError, match="CUDA"):
        quantize_int4(torch.randn(64, 64), 32)
