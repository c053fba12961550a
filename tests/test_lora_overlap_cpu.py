"""Outputs that overlap what a call of the adapters still reads: refused by the C entry before it launches anything."""

import ctypes as C

import pytest

from emmy_b200 import lib as L

T, K, N, R, ADAPTERS = 300, 64, 64, 8, 3
AT = dict(y=1 << 30, x=2 << 30, a=3 << 30, b=4 << 30, scaling=5 << 30, ids=6 << 30, workspace=7 << 30)  # never dereferenced
SIZE = dict(y=T * N * 2, x=T * K * 2, a=ADAPTERS * R * K * 2, b=ADAPTERS * N * R * 2, scaling=ADAPTERS * 4, ids=T * 4)


@pytest.fixture(scope="module")
def eq():
    from emmy_b200.build import build

    build()
    return L.load()


def call(eq, out, **ptr):
    at = {**AT, **ptr}
    return eq.eq_lora_add(at["y"], at["x"], at["a"], at["b"], at["scaling"], at["ids"], T, K, N, R, ADAPTERS, 1, None, L.EQ_BF16, out, at["workspace"], 1 << 20, None)


def test_an_output_that_overlaps_another_argument_is_refused(eq):
    cases = [call(eq, AT["x"], y=AT["x"])]  # y is x, added to in place
    for name in AT:
        size = SIZE.get(name) or eq.eq_lora_workspace_bytes(T, ADAPTERS, 1, R)
        last = -(-size // 16) * 16 - 16
        cases += [call(eq, AT[name] + last), call(eq, AT[name] - SIZE["y"] + 16)]  # its last bytes, its first
        if name != "y":
            cases.append(call(eq, AT[name]))
    assert cases == [L.EQ_ERR_BAD_ARG] * len(cases) and b"overlaps" in eq.eq_last_error()
