"""The word that the adapters' bounded waits set, as a user reaches it: through the operator and through the module, eager, compiled and captured.
(No wait is made to run out: the word is written by the test.)"""

import pytest
import torch

from tests import test_gpu_adapters as ta
from tests import test_gpu_lora as tl

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def ran_out(workspace):
    workspace.view(torch.int32)[0] = 2


def check(workspace):
    from emmy_b200 import ops_lora

    ops_lora.lora_status(workspace)


def refuses(workspace):
    from emmy_b200.lib import EmmyqError

    with pytest.raises(EmmyqError, match="EQ_ERR_TIMEOUT"):
        check(workspace)


@pytest.mark.parametrize("t,n", [(300, 264), (2500, 264), (700, 20000)])  # every CTA's own list, a list, tiles
def test_of_the_operator(t, n):
    from emmy_b200 import ops_lora

    args = tl.make(t, 264, [n], 64, 5, BF16, seed=t)
    ws = ops_lora.lora_workspace(t, 5, 1, 64, "cuda")
    check(ws)  # nothing has run
    ran_out(ws)
    refuses(ws)
    tl.close(tl.call(args, [n], workspace=ws), *args, [n])  # a call begins anew
    check(ws)
    ran_out(ws)
    small = [v[:5] for v in args[:2]] + args[2:5] + [args[5][:5]]
    tl.close(tl.call(small, [n], workspace=ws), *small, [n])
    refuses(ws)  # up to 256 rows nothing waits, and the word is the last larger call's


def test_of_the_module():
    m = ta.filled(ta.base_of("fp8_block", 512, 384), 3, 12, BF16, (256, 128))
    g = torch.Generator("cuda").manual_seed(1)
    x = torch.randn(600, 512, generator=g, device="cuda").bfloat16()
    ids = torch.randint(-1, 3, (600,), generator=g, device="cuda", dtype=torch.int32)
    with torch.no_grad():
        want = m(x, ids)
        ws = m.workspace(600)
        layers = (m, torch.compile(m, fullgraph=True, backend="eager"), torch.compile(m, fullgraph=True, backend="aot_eager"))
        for layer in layers:
            ran_out(ws)
            assert torch.equal(layer(x, ids, ws), want)
            check(ws)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = m(x, ids, workspace=ws)
        ran_out(ws)
        graph.replay()
        check(ws)
        assert torch.equal(y, want)
        with pytest.raises(RuntimeError, match="EQ_ERR_WORKSPACE"):
            m(x, ids, ws[:-512])
    torch.library.opcheck(torch.ops.emmyq.lora_add_in, (want, x, m.lora_a, m.lora_b, m.scaling, ids, [256, 128], ws))
