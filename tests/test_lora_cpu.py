"""Adapter operators on the CPU: what the C entry refuses before it launches anything."""

import ctypes as C

import pytest

from emmy_b200 import lib as L


@pytest.fixture(scope="module")
def eq():
    from emmy_b200.build import build

    build()
    return L.load()


def test_lora_add_validates_before_it_launches(eq):
    null, one = C.c_void_p(0), C.c_void_p(4096)  # never dereferenced

    def call(t=4, k=64, n=64, r=8, l=3, s=1, widths=(64,), dtype=L.EQ_BF16, ws=null, ws_bytes=0, **ptr):
        array = (C.c_int64 * len(widths))(*widths) if widths else None
        get = lambda name: C.c_void_p(ptr[name]) if name in ptr else one
        return eq.eq_lora_add(get("y"), get("x"), get("a"), get("b"), get("scaling"), get("ids"), t, k, n, r, l, s, array, dtype, get("out"), ws, ws_bytes, null)

    assert call(t=0) == 0 and call(t=0, widths=None) == 0
    for bad in (dict(t=-1), dict(k=0), dict(n=0), dict(r=0), dict(l=0), dict(s=0), dict(dtype=L.EQ_F32), dict(dtype=9), dict(widths=(56,)), dict(widths=(72,)),
                dict(s=2, widths=(0, 64)), dict(s=2, widths=(60, 4)), dict(s=2, widths=(-8, 72)), dict(s=2, widths=None), dict(s=2, widths=(2**62, 2**62)),
                dict(y=0), dict(x=0), dict(a=0), dict(b=0), dict(scaling=0), dict(ids=0), dict(out=0)):
        assert call(**bad) == L.EQ_ERR_BAD_ARG, bad
    for bad in (dict(k=60), dict(n=60, widths=(60,)), dict(r=12), dict(r=2048), dict(l=5000), dict(s=9, widths=(8,) * 9, n=72), dict(t=2**40), dict(r=256, s=8, widths=(8,) * 8),
                dict(k=2**40), dict(n=2**40, widths=(2**40,)), dict(r=2**60, s=8, widths=(8,) * 8)):
        assert call(**bad) == L.EQ_ERR_UNSUPPORTED, bad
    for name in ("y", "x", "a", "b", "out"):
        assert call(**{name: 4104}) == L.EQ_ERR_BAD_ALIGN
    assert call(ids=4098) == L.EQ_ERR_BAD_ALIGN
    # a workspace above 256 rows only
    assert eq.eq_lora_workspace_bytes(256, 8, 1, 8) == 0 and eq.eq_lora_workspace_bytes(257, 8, 1, 8) > 257 * (4 + 4 * 8)
    assert call(t=257) == L.EQ_ERR_WORKSPACE
    assert call(t=257, ws=C.c_void_p(4096 + 128), ws_bytes=1 << 20) == L.EQ_ERR_WORKSPACE
    assert call(t=257, ws=one, ws_bytes=eq.eq_lora_workspace_bytes(257, 3, 1, 8) - 1) == L.EQ_ERR_WORKSPACE


def test_ops_refuse_cpu_tensors():
    torch = pytest.importorskip("torch")
    from emmy_b200 import ops_lora

    z = torch.zeros(8, 8, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops_lora.lora_add(z, z, z[None], z[None], torch.zeros(1), torch.zeros(8, dtype=torch.int32))
