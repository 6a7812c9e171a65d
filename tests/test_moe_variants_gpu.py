"""The MXFP4 expert operators at the ends of their ranges and through every variant of their
kernels, against plain 64-bit forms."""
import pytest
import torch

import moe_ref as R
from mxfp4_b200 import capi
from omo_python_api import mxfp4_moe as moe
from test_moe_gpu import act_grad_ref

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


@pytest.fixture(autouse=True)
def _no_wait_gave_up(cuda):
    yield
    torch.cuda.synchronize()
    assert capi.reset_wait_timeouts() == 0


@pytest.mark.parametrize("name", R.ACTS)
def test_slopes_of_large_values(cuda, name):
    """|z| from 16 to 2^126, where the slopes are 0, 1, 2 z or (swiglu) one half times the other.
    One rounding to BF16 (2^-9 of the value, 2^-8 allowed); a logistic below 2^-126 is 0, which
    leaves at most 88 * 2^-126 times the other half (here at most 3) of a tail: 4e-36."""
    big = torch.exp2(torch.arange(4, 127).double())
    big = torch.cat((big, -big, 1.37 * big[:-1], -1.37 * big[:-1]))
    big = torch.cat((big, big[:-big.numel() % 64])).reshape(-1, 64).to(BF).cuda()
    pre = big
    if name == "swiglu":
        other = torch.tensor([1.25, -3.0], device=cuda).repeat(32).to(BF).expand_as(big)
        pre = torch.cat((torch.cat((big, other), 1), torch.cat((other, big), 1)))
    dy = torch.ones(pre.shape[0], 64, dtype=BF, device=cuda)
    got = moe.omo_bias_act_grad(dy, pre, None, name, bias_grad=False)
    want = act_grad_ref(dy, pre, name)
    R.check(got, want, 2.0 ** -8 * want.abs() + 4e-36)
