"""The batched serving operators on the GPU where their documentation allows a call that is easily got wrong:
the largest sums, weights far below a row's largest, scales of zero, outputs that lie beside or over inputs."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def S():
    from vtq import serving
    return serving


@pytest.mark.parametrize("t,n", [(1, 3), (40, 130), (200, 20), (300, 4900)])
def test_linear_i8_the_largest_sum(S, t, n):
    """131072 products of -128 and -128 are 2^31, which 32 signed bits hold as their lowest value: codes of the
    caller's own may be -128. (All values are exact in 32-bit floats: 131072 times at most 15 bits.)"""
    k = 131072
    code = torch.where(torch.arange(t, device="cuda") % 3 == 1, 127, -128)
    weight = torch.where(torch.arange(n, device="cuda") % 3 == 2, 127, -128)
    q = code.to(torch.int8)[:, None].expand(t, k).contiguous()
    W = S.I8Weight(weight.to(torch.int8)[:, None].expand(n, k), torch.ones(n, device="cuda"))
    y = S.linear_i8(q, W, x_scale=torch.ones(t, device="cuda"))
    assert torch.equal(y.double(), (code[:, None] * weight).double() * k)
    # one product short of it
    q[:, 77] = 0
    y = S.linear_i8(q, W, x_scale=torch.ones(t, device="cuda"))
    assert torch.equal(y, ((code[:, None] * weight).double() * (k - 1)).float())
