"""The feed-forward products where values and lengths are extreme: infinite pre-activations, tails of the activations in FP32,
sums of hundreds of thousands of terms.

Each test derives its own bound; u(t) is half a step of type t relative to the value: FP16 2^-11, BF16 2^-8, FP32 2^-24."""
import pytest

from tests.test_feed_forward import ACTS, BF16, F16, F32, SENTINEL, act64

pytestmark = pytest.mark.gpu


def torch_type(name):
    import torch

    return getattr(torch, name)


# ------------------------------------------------------------------------------------------------ infinite Z
@pytest.mark.parametrize("dtype,out", [(F16, F16), (BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize("rows", [2, 200])  # the short-A kernels, the grouped kernel
def test_infinite_pre_activations(cuda_device, rows, dtype, out):
    """Where Z is +infinity every activation is; where it is -infinity, relu is 0 and the products z * 0 are NaN, as in the
    formulas. Bits, no tolerance."""
    import torch

    from cuda_hgemm_b200 import api

    N, K = 4096, 64
    A = torch.zeros((rows, K), dtype=torch_type(dtype), device=cuda_device)
    A[0::2, 0], A[1::2, 0] = float("inf"), float("-inf")
    B = torch.ones((N, K), dtype=A.dtype, device=cuda_device)
    offsets = torch.tensor([0, rows], dtype=torch.int32, device=cuda_device)
    z = A[:, :1].double().expand(rows, N)
    for act in ACTS:
        want = act64(z, act).to(torch_type(out))
        assert torch.isposinf(want[0]).all()
        for grouped in (False, True):
            C = torch.full((rows, N), SENTINEL, dtype=torch_type(out), device=cuda_device)
            pre = torch.full_like(C, SENTINEL)
            if grouped:
                api.hgemm_grouped(A, B[None], C, offsets, act=act, pre=pre)
            else:
                api.hgemm_linear(A, B, C, act=act, pre=pre)
            assert torch.equal(pre, z.to(pre.dtype)), (act, grouped)
            assert torch.equal(torch.isnan(C), torch.isnan(want)), (act, grouped)
            assert torch.equal(torch.nan_to_num(C.float(), nan=1.0), torch.nan_to_num(want.float(), nan=1.0)), (act, grouped)
    assert api.last_device_error() == 0


def test_slopes_at_infinity(cuda_device):
    """The slopes' limits: 1 at +infinity and 0 at -infinity (none: 1)."""
    import torch

    from cuda_hgemm_b200 import api

    N, K = 512, 8
    A, B = torch.zeros((1, K), dtype=torch.float16, device=cuda_device), torch.zeros((N, K), dtype=torch.float16, device=cuda_device)
    dC = torch.full((1, N), 1.5, dtype=torch.float16, device=cuda_device)
    pre = torch.full((1, N), float("inf"), dtype=torch.float16, device=cuda_device)
    pre[:, 1::2] = float("-inf")
    for act in ACTS[1:]:
        dZ, dbias = torch.empty_like(dC), torch.empty(N, device=cuda_device)
        api.hgemm_linear_backward(dC, A, B, act=act, pre=pre, dZ=dZ, dbias=dbias)
        assert (dZ[:, 0::2] == 1.5).all() and (dZ[:, 1::2] == 0).all(), act
        assert (dbias[0::2] == 1.5).all() and (dbias[1::2] == 0).all(), act
