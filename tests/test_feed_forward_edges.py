"""The feed-forward products where values and lengths are extreme: infinite pre-activations, tails of the activations in FP32,
sums of hundreds of thousands of terms.

Each test derives its own bound; u(t) is half a step of type t relative to the value: FP16 2^-11, BF16 2^-8, FP32 2^-24."""
import pytest

from tests.test_feed_forward import (ACTS, BF16, F16, F32, SENTINEL, act64, assert_within, check_backward, check_forward, half_step, make, rounded,
                                     slope64, sum_error)

pytestmark = pytest.mark.gpu


def torch_type(name):
    import torch

    return getattr(torch, name)


@pytest.fixture
def most_memory(cuda_device):
    """GB free once what torch keeps from earlier tests is given back; this test's share is given back too."""
    import gc

    import torch

    gc.collect()
    torch.cuda.empty_cache()
    yield torch.cuda.mem_get_info()[0] >> 30
    gc.collect()
    torch.cuda.empty_cache()


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


# ------------------------------------------------------------------------------------------------ the activations' tails
def smooth64(z, act):
    """Value and slope in 64 bits without cancellation for negative z, and what FP32 arithmetic may lose of the gate (relative).

    The gate is Phi(z) for gelu and a logistic function else: an exponential of an argument a that is formed by up to six
    roundings to FP32 (constants included), each 2^-24 |a| absolute, hence relative in the exponential; the hardware's
    exponential and reciprocal, 2^-22 each; gelu's polynomial (1.2e-7 and at most four FP32 roundings) and three products: 2^-20
    covers them."""
    import math

    import torch

    if act == "gelu":
        gate, a = 0.5 * torch.special.erfc(-z * math.sqrt(0.5)), z * z / 2
        slope = torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    else:
        w = z if act == "silu" else 2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)
        dw = torch.ones_like(z) if act == "silu" else 2 * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z * z)
        gate, a = torch.sigmoid(w), w.abs()
        slope = gate * torch.sigmoid(-w) * dw
    return gate, slope, 2.0 ** -20 + 6 * 2.0 ** -24 * a


@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("rows", [16, 256])  # the short-A kernels, the grouped kernel
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_activations_in_fp32_relative_to_their_value(cuda_device, dtype, rows, act):
    """A product with the identity hands every z of a grid over [-6, 6] on exactly; C in FP32 is then the activation alone."""
    import torch

    from cuda_hgemm_b200 import api

    N = 4096 if rows == 16 else 64
    A = torch.linspace(-6, 6, rows * 64, device=cuda_device).view(rows, 64).to(torch_type(dtype))
    B = torch.eye(64, device=cuda_device).to(A.dtype).repeat(N // 64, 1)
    C = torch.full((rows, N), float("nan"), device=cuda_device)
    api.hgemm_linear(A, B, C, act=act)
    z = A.double().repeat(1, N // 64)
    gate, _, rel = smooth64(z, act)
    # (1 - tail for positive z: one more rounding; the product with z another)
    over = (C.double() - z * gate).abs() - (rel + 2.0 ** -22) * (z * gate).abs()
    at = over.argmax()
    assert over.max() <= 0, (z.flatten()[at].item(), C.flatten()[at].item(), (z * gate).flatten()[at].item())
    assert api.last_device_error() == 0


@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
def test_slopes_in_fp32_relative_to_their_terms(cuda_device, act):
    """With one row and a gradient of one, dbias is the slope itself: gate + z gate', each term to its own relative bound."""
    import torch

    from cuda_hgemm_b200 import api

    N, K = 8192, 8
    A, B = torch.zeros((1, K), dtype=torch.bfloat16, device=cuda_device), torch.zeros((N, K), dtype=torch.bfloat16, device=cuda_device)
    pre = torch.linspace(-6, 6, N, device=cuda_device).view(1, N)
    dbias = torch.empty(N, device=cuda_device)
    api.hgemm_linear_backward(torch.ones_like(pre), A, B, act=act, pre=pre, dbias=dbias)
    z = pre[0].double()
    gate, slope, rel = smooth64(z, act)
    # (for positive z the logistic form takes 1 - gate, whose error is that of the gate: 2^-20 of 1 and not of 1 - gate)
    factor = torch.zeros_like(z) if act == "gelu" else z.abs() * gate * (slope / (gate * (1 - gate).clamp(min=1e-30)))
    bound = (rel + 2.0 ** -22) * (gate + (z * slope).abs()) + torch.where(z > 0, factor * 2.0 ** -20, 0.0)
    over = (dbias.double() - (gate + z * slope)).abs() - bound
    at = over.argmax()
    assert over.max() <= 0, (z[at].item(), dbias[at].item(), (gate + z * slope)[at].item(), bound[at].item())


# ------------------------------------------------------------------------------------------------ launches
def test_no_launch_of_a_linear_layer_starts_early(cuda_device, native_lib):
    """Short-A kernels of one k-range, of ranges summed inside clusters, of ranges summed through the workspace, and on pairs: none
    starts while the kernel before it drains. The same shapes through the older entry point do."""
    import ctypes

    import torch

    from cuda_hgemm_b200 import _native, api

    forms = set()
    for M, N, K in ((1, 1024, 1024), (16, 14336, 4096), (16, 4096, 14336), (64, 1024, 8192), (100, 512, 4096), (128, 4096, 14336),
                    (128, 4096, 8192), (64, 14336, 4096)):
        A, B = torch.zeros((M, K), dtype=torch.float16, device=cuda_device), torch.zeros((N, K), dtype=torch.float16, device=cuda_device)
        C = torch.full((M, N), SENTINEL, dtype=torch.float16, device=cuda_device)
        args = _native.LinearArgs(in_type=_native.C_F16, c_type=_native.C_F16, act=_native.ACT_SILU)
        before = native_lib.b200_debug_early_skinny_launches()
        api.hgemm_linear(A, B, C, act="silu")
        assert native_lib.b200_debug_early_skinny_launches() == before, (M, N, K)
        assert (C == 0).all()
        torch.cuda.synchronize()
        api.b200Hgemm(A, B, C)
        torch.cuda.synchronize()
        early = native_lib.b200_debug_early_skinny_launches() - before
        forms.add((early, native_lib.b200_hgemm_linear_workspace_bytes(M, N, K, ctypes.byref(args)) > 0))
    assert (1, False) in forms and (2, True) in forms  # one kernel, and a kernel with its sum behind it
    assert api.last_device_error() == 0


# ------------------------------------------------------------------------------------------------ long sums
def graded(shape, dtype, device, seed, scale=1.0):
    """Positive values whose columns (dimension 1) differ in size, so that the results fall anywhere between two steps."""
    import torch

    gen = torch.Generator(device=device).manual_seed(seed)
    x = torch.rand(shape, generator=gen, device=device).mul_(0.5).add_(0.5)
    x *= (torch.rand((1, shape[1]), generator=gen, device=device) * 0.5 + 0.5) * scale
    return x.to(torch_type(dtype))


def mean_signed_error(got, ref):
    return ((got.double() - ref) / ref).mean().item()


LONG = 262144


@pytest.mark.parametrize("form", ["forward", "input gradient", "weight gradient", "weight gradient on pairs"])
@pytest.mark.parametrize("dtype,length", [(F16, LONG), (BF16, 2 * LONG)])
def test_16_bit_results_of_very_long_sums_do_not_shrink(cuda_device, dtype, length, form):
    """The tensor cores cut an accumulator off at every MMA (16 terms), which makes a sum of positive terms smaller: by 1e-7 a
    step, 1.7e-3 after 16384 of them. Longer sums are cut into pieces of 4096 terms (FP16) or 32768
    (BF16), which lose at most 2^-23 a step. What else can move the mean of `count` results is their one
    rounding: u / sqrt(3 count) is its standard deviation, four of them are allowed."""
    import torch

    from cuda_hgemm_b200 import api

    if form == "forward":
        A, B = graded((136, length), dtype, cuda_device, 1), graded((128, length), dtype, cuda_device, 2, 2.0 ** -6)
        A, B = A * graded((136, 1), dtype, cuda_device, 3), B * graded((128, 1), dtype, cuda_device, 4)
        got = torch.empty((136, 128), dtype=A.dtype, device=cuda_device)
        api.hgemm_linear(A, B, got)
        ref = A.double() @ B.double().T
    elif form == "input gradient":
        dC, B = graded((136, length), dtype, cuda_device, 1), graded((length, 128), dtype, cuda_device, 2, 2.0 ** -6)
        dC = dC * graded((136, 1), dtype, cuda_device, 3)
        A, got = torch.empty((136, 128), dtype=dC.dtype, device=cuda_device), torch.empty((136, 128), dtype=dC.dtype, device=cuda_device)
        api.hgemm_linear_backward(dC, A, B, dA=got)
        ref = dC.double() @ B.double()
    else:
        # one group of rows, whose sum is not cut into slices; enough columns for CTA pairs in the second case
        N, K = (136, 128) if form == "weight gradient" else (1160, 1096)
        dC, A = graded((length, N), dtype, cuda_device, 1), graded((length, K), dtype, cuda_device, 2, 2.0 ** -6)
        B, got = torch.empty((1, N, K), dtype=A.dtype, device=cuda_device), torch.empty((1, N, K), dtype=A.dtype, device=cuda_device)
        offsets = torch.tensor([0, length], dtype=torch.int32, device=cuda_device)
        api.hgemm_grouped_backward(dC, A, B, offsets, dB=got)
        got, ref = got[0], torch.zeros((N, K), dtype=torch.float64, device=cuda_device)
        for lo in range(0, length, 65536):
            ref += dC[lo:lo + 65536].double().T @ A[lo:lo + 65536].double()
    assert torch.isfinite(got).all()
    u = torch.finfo(got.dtype).eps / 2
    limit = (256 if dtype == F16 else 2048) * 2.0 ** -23 + 4 * u / (3 * got.numel()) ** 0.5
    assert abs(mean_signed_error(got, ref)) < limit
    assert api.last_device_error() == 0


# ------------------------------------------------------------------------------------------------ offsets
def test_offsets_out_of_order_over_more_than_a_billion_rows(cuda_device, most_memory):
    """Every other offset is 0 and the rest M: taken as they stand, 512 groups of M rows are more blocks of rows than 32 bits count.
    Put in order, the first group holds every row; nothing behind row M is written."""
    import torch

    from cuda_hgemm_b200 import api

    M, N, K, G = (1 << 30) + (1 << 27), 8, 8, 1024
    if most_memory < 60:
        pytest.skip("not enough free memory")
    A = torch.full((M, K), 0.5, dtype=torch.bfloat16, device=cuda_device)
    B = make((G, N, K), BF16, cuda_device, 1)
    room = torch.full((M + 64, N), SENTINEL, dtype=torch.bfloat16, device=cuda_device)
    offsets = torch.tensor([0, M] * (G // 2) + [0], dtype=torch.int32, device=cuda_device)
    api.hgemm_grouped(A, B, room[:M], offsets)
    assert (room[M:] == SENTINEL).all()
    check_forward(A[:1], B[0], None, None, "none", room[:1], None, "first row")
    for lo in range(0, M, 1 << 27):
        assert (room[lo:min(lo + (1 << 27), M)] == room[0]).all(), lo
    offsets = torch.tensor([0, M - 3] * (G // 2) + [M], dtype=torch.int32, device=cuda_device)
    api.hgemm_grouped(A, B, room[:M], offsets)
    check_forward(A[M - 3:], B[G - 1], None, None, "none", room[M - 3:M], None, "last rows")
    assert (room[:M - 3] == room[0]).view(-1, N)[:: 1 << 12].all() and (room[M:] == SENTINEL).all()
    assert api.last_device_error() == 0


# ------------------------------------------------------------------------------------------------ gradients of the weights
@pytest.mark.parametrize("shape", [(5000, 72, 200), (8191, 264, 136), (3000, 256, 256)], ids=str)
@pytest.mark.parametrize("dtype,act", [(F16, "none"), (BF16, "none"), (BF16, "gelu")])
def test_accumulated_over_slices(cuda_device, shape, dtype, act):
    """Enough rows and few enough tiles for the sum to be cut into slices, which are then added to what dB holds."""
    import ctypes

    import torch

    from cuda_hgemm_b200 import _native, api

    M, N, K = shape
    # the slices lie in the workspace: without dZ and dbias nothing else does
    alone = _native.LinearGrads(in_type=_native.C_F16, c_type=_native.C_F16, db_type=_native.C_F32, dC=256, dB=256)
    assert _native.load().b200_hgemm_backward_workspace_bytes(M, N, K, 1, ctypes.byref(alone)) >= 2 * 4 * N * K
    A, B = make((M, K), dtype, cuda_device, 1), make((N, K), dtype, cuda_device, 2)
    dC, pre = make((M, N), dtype, cuda_device, 3, 0.1), make((M, N), dtype, cuda_device, 4, 2.0)
    dZ = torch.empty_like(dC) if act != "none" else None
    was, was_bias = make((N, K), F32, cuda_device, 5, 30.0), make((N,), F32, cuda_device, 6, 30.0)
    dB, dbias = was.clone(), was_bias.clone()
    for _ in range(2):  # twice: the second call adds to the first one's result
        before, before_bias = dB.clone(), dbias.clone()
        api.hgemm_linear_backward(dC, A, B, act=act, pre=pre if act != "none" else None, dB=dB, dbias=dbias, dZ=dZ, accumulate=True)
        check_backward(dC, A, B, act, pre, dZ, None, dB, dbias, "slices", dB_was=before, dbias_was=before_bias)
    assert api.last_device_error() == 0


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("act", ACTS[1:])
@pytest.mark.parametrize("sizes", [None, [700, 0, 33, 1290]], ids=["linear", "grouped"])
def test_products_of_an_unrounded_dz(cuda_device, sizes, act, dtype):
    """dA and an FP32 dB, accumulated, against dZ in 64 bits. The products read dZ rounded to the inputs' type: each of its values, and
    with it each term of a sum, is off by u(type) at most, or by half of FP16's smallest step; the slope by 2^-19."""
    import torch

    from cuda_hgemm_b200 import api

    M, N, K = sum(sizes) if sizes else 1500, 264, 136
    bounds = [0]
    for r in sizes or [M]:
        bounds.append(bounds[-1] + r)
    G = len(bounds) - 1
    A, B = make((M, K), dtype, cuda_device, 1), make((G, N, K), dtype, cuda_device, 2, K ** -0.5)
    dC, pre = make((M, N), dtype, cuda_device, 3), make((M, N), dtype, cuda_device, 4, 2.0)
    was = make((G, N, K), F32, cuda_device, 5)
    dA, dB = torch.empty_like(A), was.clone()
    if sizes:
        offsets = torch.tensor(bounds, dtype=torch.int32, device=cuda_device)
        api.hgemm_grouped_backward(dC, A, B, offsets, act=act, pre=pre, dA=dA, dB=dB, accumulate=True)
    else:
        api.hgemm_linear_backward(dC, A, B[0], act=act, pre=pre, dA=dA, dB=dB[0], accumulate=True)
    dz = dC.double() * slope64(pre.double(), act)
    edz = half_step(dtype) * dz.abs() + 2.0 ** -19 * dC.double().abs() * 1.001 + (2.0 ** -25 if dtype == F16 else 0)
    for g in range(G):
        r = slice(bounds[g], bounds[g + 1])
        a, b, z, ez = A[r].double(), B[g].double(), dz[r], edz[r]
        err = ez @ b.abs() + sum_error(N, (z.abs() + ez) @ b.abs())
        assert_within(dA[r], z @ b, rounded(z @ b, err, dtype), f"dA {g}")
        ref = z.T @ a + was[g].double()
        err = ez.T @ a.abs() + sum_error(len(a), (z.abs() + ez).T @ a.abs()) + 2.0 ** -23 * (ref.abs() + was[g].double().abs())
        assert_within(dB[g], ref, rounded(ref, err, torch.float32), f"dB {g}")
    assert api.last_device_error() == 0


# ------------------------------------------------------------------------------------------------ the largest sizes, and in place
def test_most_groups_there_may_be(cuda_device):
    import torch

    from cuda_hgemm_b200 import api

    G, N, K = 1024, 72, 136
    sizes = [(7 * i * i) % 6 for i in range(G)]
    bounds = [0]
    for r in sizes:
        bounds.append(bounds[-1] + r)
    M = bounds[-1]
    A, B, bias = make((M, K), F16, cuda_device, 1), make((G, N, K), F16, cuda_device, 2, K ** -0.5), make((G, N), F16, cuda_device, 3)
    dC = make((M, N), F16, cuda_device, 4)
    C, dA, dB = torch.empty_like(dC), torch.empty_like(A), torch.full((G, N, K), SENTINEL, device=cuda_device)
    dbias = torch.full((G, N), SENTINEL, device=cuda_device)
    offsets = torch.tensor(bounds, dtype=torch.int32, device=cuda_device)
    api.hgemm_grouped(A, B, C, offsets, bias=bias, act="silu")
    api.hgemm_grouped_backward(dC, A, B, offsets, dA=dA, dB=dB, dbias=dbias)
    for g in range(G):
        r = slice(bounds[g], bounds[g + 1])
        if sizes[g]:
            check_forward(A[r], B[g], bias[g], None, "silu", C[r], None, f"group {g}")
            check_backward(dC[r], A[r], B[g], "none", None, None, dA[r], dB[g], dbias[g], f"group {g}")
        else:
            assert (dB[g] == 0).all() and (dbias[g] == 0).all()
    assert api.last_device_error() == 0


def test_a_stack_of_more_than_2_to_the_32_weights(cuda_device, most_memory):
    import torch

    from cuda_hgemm_b200 import api

    G, N, K = 272, 4096, 4096  # 4.6e9 weights
    if most_memory < 24:
        pytest.skip("not enough free memory")
    B = torch.zeros((G, N, K), dtype=torch.bfloat16, device=cuda_device)
    last = (0, 255, 256, G - 1)  # around element 2^32, and the ends
    for g in last:
        B[g] = make((N, K), BF16, cuda_device, g, K ** -0.5)
    A, dC = make((4 * G, K), BF16, cuda_device, 1), make((4 * G, N), BF16, cuda_device, 2)
    offsets = torch.arange(0, 4 * G + 1, 4, dtype=torch.int32, device=cuda_device)
    C, dA, dB = torch.full_like(dC, SENTINEL), torch.full_like(A, SENTINEL), torch.full_like(B, SENTINEL)
    api.hgemm_grouped(A, B, C, offsets)
    api.hgemm_grouped_backward(dC, A, B, offsets, dA=dA, dB=dB)
    for g in last:
        r = slice(4 * g, 4 * g + 4)
        check_forward(A[r], B[g], None, None, "none", C[r], None, f"group {g}")
        check_backward(dC[r], A[r], B[g], "none", None, None, dA[r], dB[g], None, f"group {g}")
    assert (C[8:4 * 255] == 0).all() and (dA[8:4 * 255] == 0).all()
    assert api.last_device_error() == 0


def test_nearly_2_to_the_31_rows(cuda_device, most_memory):
    """The most rows a call takes, 2^31 - 256: the last of them, and nothing behind them."""
    import torch

    from cuda_hgemm_b200 import api

    M, N, K = 0x7fffff00, 8, 8
    if most_memory < 110:
        pytest.skip("not enough free memory")
    A = torch.zeros((M, K), dtype=torch.float16, device=cuda_device)
    A[-700:] = make((700, K), F16, cuda_device, 1)
    B = make((2, N, K), F16, cuda_device, 2)
    room = torch.full((M + 64, N), SENTINEL, dtype=torch.float16, device=cuda_device)
    C = room[:M]
    last = slice(M - 700, M)
    api.hgemm_linear(A, B[0], C, act="relu")
    check_forward(A[last], B[0], None, None, "relu", C[last], None, "linear")
    offsets = torch.tensor([0, 5, M], dtype=torch.int32, device=cuda_device)
    api.hgemm_grouped(A, B, C, offsets)
    check_forward(A[last], B[1], None, None, "none", C[last], None, "grouped")
    assert (room[M:] == SENTINEL).all()
    # (a weight gradient of one group of so many rows is one tile's sum, which takes seconds; the linear layer's is cut into slices)
    dA, dB, dbias = torch.full((M + 64, K), SENTINEL, dtype=torch.float16, device=cuda_device), torch.empty((N, K), device=cuda_device), torch.empty(N, device=cuda_device)
    api.hgemm_grouped_backward(C, A, B, offsets, dA=dA[:M])
    check_backward(C[last], A[last], B[1], "none", None, None, dA[:M][last], None, None, "grouped")
    assert (dA[M:] == SENTINEL).all()
    api.hgemm_linear_backward(C, A, B[1], dA=dA[:M], dB=dB, dbias=dbias)
    check_backward(C[last], A[last], B[1], "none", None, None, dA[:M][last], dB, dbias, "linear")
    assert api.last_device_error() == 0


@pytest.mark.parametrize("shape", [(1, 64, 72), (64, 1024, 8192), (16, 4096, 4096), (300, 701, 200), (777, 1000, 1544), (2000, 4096, 128)], ids=str)
@pytest.mark.parametrize("dtype,out", [(F16, F16), (BF16, F32)])
def test_residual_in_place_on_every_kernel(cuda_device, shape, dtype, out):
    import torch

    from cuda_hgemm_b200 import api

    M, N, K = shape
    A, B = make((M, K), dtype, cuda_device, 1), make((N, K), dtype, cuda_device, 2, K ** -0.5)
    C = make((M, N), out, cuda_device, 3)
    was, pre = C.clone(), torch.empty_like(C)
    api.hgemm_linear(A, B, C, residual=C, act="gelu_tanh", pre=pre)
    check_forward(A, B, None, was, "gelu_tanh", C, pre, "in place")
    assert api.last_device_error() == 0
