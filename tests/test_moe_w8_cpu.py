"""The FP8 expert layer on the CPU: what the C entry refuses before it launches anything."""

import ctypes as C

import pytest

from emmy_b200 import lib as L


@pytest.fixture(scope="module")
def eq():
    from emmy_b200.build import build

    build()
    return L.load()


def test_moe_w8a16_validates_before_it_launches(eq):
    null, one = C.c_void_p(0), C.c_void_p(4096)  # never dereferenced

    def call(t=4, e=8, topk=2, h=256, i=128, block=1, dtype=L.EQ_BF16, ws=one, ws_bytes=1 << 30, **ptr):
        get = lambda name: C.c_void_p(ptr[name]) if name in ptr else one
        return eq.eq_moe_w8a16(get("gate_up"), get("gate_up_scale"), get("down"), get("down_scale"), block, e, topk, h, i, get("x"), get("logits"), t, dtype, get("y"), ws,
                               ws_bytes, null)

    assert call(t=0) == 0
    for bad in (dict(t=-1), dict(e=0), dict(topk=0), dict(h=0), dict(i=0), dict(block=2), dict(dtype=L.EQ_F32), dict(gate_up=0), dict(gate_up_scale=0), dict(down=0),
                dict(down_scale=0), dict(x=0), dict(logits=0), dict(y=0)):
        assert call(**bad) == L.EQ_ERR_BAD_ARG, bad
    for bad in (dict(e=1025), dict(topk=9), dict(topk=17, e=32), dict(h=192), dict(i=64), dict(t=2**40), dict(h=2**40), dict(i=2**40)):
        assert call(**bad) == L.EQ_ERR_UNSUPPORTED, bad
    for name in ("gate_up", "down", "x", "y"):
        assert call(**{name: 4104}) == L.EQ_ERR_BAD_ALIGN
    for name in ("gate_up_scale", "down_scale", "logits"):
        assert call(**{name: 4098}) == L.EQ_ERR_BAD_ALIGN
    need = eq.eq_moe_w8a16_workspace_bytes(4, 8, 2, 256, 128)
    assert need >= 4 * 2 * 128 * 4 + 4 * 256 * 2  # silu * up in f32, x in f16
    assert call(ws=null) == call(ws_bytes=need - 1) == call(ws=C.c_void_p(4096 + 128)) == L.EQ_ERR_WORKSPACE


def test_ops_refuse_cpu_tensors():
    torch = pytest.importorskip("torch")
    from emmy_b200 import ops_moe

    z = torch.zeros(1, 128, dtype=torch.bfloat16)
    w = torch.zeros(1, 256, 128, dtype=torch.uint8)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops_moe.moe_w8a16(z, torch.zeros(1, 1), w, torch.ones(1, 256), w[:, :128].contiguous(), torch.ones(1, 128), 1)
