"""The few-token layer's rows in another order: what a token gets does not depend on its place among the tokens, also where an
expert's rows take several passes, of which the last is not full."""
import pytest
import torch

from test_gpu_routed_layer import DEV, DTYPES, _call, _inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
# tokens, experts, experts per token: passes of 8, 16 and 32 rows of an expert, the hot one's last pass of 1 to 16 rows
@pytest.mark.parametrize("T,E,k", [(20, 16, 2), (21, 8, 2), (17, 8, 2), (24, 8, 2), (33, 4, 1), (37, 8, 4), (41, 4, 2), (48, 4, 2), (64, 8, 2)])
def test_order_of_the_tokens(T, E, k, dtype):
    i = _inputs(T, 2048, 1024, E, dtype, seed=T + E)
    i["x"] = (i["x"].abs() + 0.25).to(dtype)
    i["wr"][1] = 1.0                                     # every token's first expert
    want = _call(i, k)
    g = torch.Generator().manual_seed(0)
    for order in [torch.arange(T).flip(0)] + [torch.randperm(T, generator=g) for _ in range(3)]:
        order = order.to(DEV)
        got = _call(dict(i, x=i["x"][order]), k)
        assert torch.equal(got[1], want[1][order])
        assert torch.equal(got[0], want[0][order]), "%d values differ" % int((got[0] != want[0][order]).sum())
    again = _call(i, k)
    assert torch.equal(again[0], want[0])
