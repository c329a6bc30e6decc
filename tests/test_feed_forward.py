"""The feed-forward products (linear layers and products grouped by expert, forward and backward) against the same
formulas in 64 bits, and what they refuse.

Tolerances, derived from the number formats (u(t) = half a step of type t, relative):

* a sum of L products of 16-bit values is formed 16 at a time in FP32: every step rounds (or truncates) to FP32, and
  adds at most 2^-22 of the sum of the magnitudes: (L/16 + 2) 2^-22 S, S = sum |a| |b|;
* bias and residual add one FP32 rounding each: 2^-23 of the value;
* an activation passes an error on at most 1.13 times (the largest slope, gelu's) and adds 2^-20 |z| of its own (the
  approximations of exp, 1/x and erfc are good to 2^-21 or better); a slope is off by 2^-19 at most;
* the result is rounded once: u(t) of its value, or half the smallest FP16 step, 2^-25.
"""
import ctypes

import pytest

from cuda_hgemm_b200 import _native

F16, BF16, F32 = "float16", "bfloat16", "float32"
ACTS = ("none", "relu", "gelu", "gelu_tanh", "silu")
SENTINEL = 7.25  # representable in every type


# ------------------------------------------------------------------------------------------------ formulas in 64 bits
def act64(z, act):
    import torch

    if act == "relu":
        return z.clamp(min=0)
    if act == "gelu":
        return z * 0.5 * torch.special.erfc(-z * 0.5 ** 0.5)
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh((2 / torch.pi) ** 0.5 * (z + 0.044715 * z ** 3)))
    if act == "silu":
        return z * torch.sigmoid(z)
    return z


def slope64(z, act):
    import torch

    z = z.detach().clone().requires_grad_(True)
    if act == "none":
        return torch.ones_like(z)
    if act == "relu":
        return (z.detach() > 0).to(z.dtype)
    (g,) = torch.autograd.grad(act64(z, act).sum(), z)
    return g


def half_step(dtype):
    import torch

    return torch.finfo(getattr(torch, dtype) if isinstance(dtype, str) else dtype).eps / 2


def sum_error(length, magnitude):
    return (length / 16 + 2) * 2.0 ** -22 * magnitude


def rounded(ref, err, dtype):
    """What a value within ``err`` of ``ref`` may be off by after one rounding to ``dtype``."""
    import torch

    u = half_step(dtype)
    floor = 2.0 ** -25 if dtype in (F16, torch.float16) else 0.0
    return err + u * (ref.abs() + err) + floor


def assert_within(got, ref, tol, what):
    import torch

    got = got.double()
    assert torch.isfinite(got).all(), f"{what}: not finite"
    over = (got - ref).abs() - tol
    worst = over.max().item() if over.numel() else -1.0
    if worst > 0:
        at = torch.nonzero(over == over.max())[0].tolist()
        raise AssertionError(f"{what}: off by {(got - ref).abs()[tuple(at)].item():.4g} at {at}, allowed "
                             f"{tol[tuple(at)].item():.4g} (value {ref[tuple(at)].item():.4g}); {(over > 0).sum().item()} elements")


def make(shape, dtype, device, seed, scale=1.0):
    import torch

    gen = torch.Generator(device=device).manual_seed(seed)
    return (torch.randn(shape, generator=gen, device=device) * scale).to(getattr(torch, dtype))


def check_forward(A, B, bias, residual, act, C, pre, what):
    a, b = A.double(), B.double()
    z = a @ b.T
    ez = sum_error(A.shape[1], a.abs() @ b.abs().T)
    if bias is not None:
        z = z + bias.double()
        ez = ez + 2.0 ** -23 * z.abs()
    if pre is not None:
        assert_within(pre, z, rounded(z, ez, pre.dtype), what + " pre")
    c = act64(z, act)
    ec = 1.13 * ez + (2.0 ** -20 * z.abs() if act not in ("none", "relu") else 0)
    if residual is not None:
        c = c + residual.double()
        ec = ec + 2.0 ** -23 * (c.abs() + residual.double().abs())
    assert_within(C, c, rounded(c, ec, C.dtype), what)


def check_backward(dC, A, B, act, pre, dZ, dA, dB, dbias, what, dB_was=None, dbias_was=None):
    """dZ against the formula; the products against the dZ that the kernels read (rounded once to the inputs' type)."""
    import torch

    d = dC.double()
    dz = d * slope64(pre.double(), act) if act != "none" else d
    edz = 2.0 ** -19 * d.abs() + 2.0 ** -23 * dz.abs()
    if dZ is not None:
        assert_within(dZ, dz, rounded(dz, edz, dZ.dtype), what + " dZ")
    read = (dZ if dZ is not None else dC).double()
    if dA is not None:
        ref = read @ B.double()
        err = sum_error(read.shape[1], read.abs() @ B.double().abs())
        assert_within(dA, ref, rounded(ref, err, dA.dtype), what + " dA")
    if dB is not None:
        ref = read.T @ A.double()
        err = sum_error(read.shape[0], read.abs().T @ A.double().abs())
        if dB_was is not None:
            ref = ref + dB_was.double()
            err = err + 2.0 ** -23 * (ref.abs() + dB_was.double().abs())
        assert_within(dB, ref, rounded(ref, err, dB.dtype), what + " dB")
    if dbias is not None:
        ref = dz.sum(0)
        err = edz.sum(0) + dz.shape[0] * 2.0 ** -24 * dz.abs().sum(0)
        if dbias_was is not None:
            ref = ref + dbias_was.double()
            err = err + 2.0 ** -23 * (ref.abs() + dbias_was.double().abs())
        assert_within(dbias, ref, rounded(ref, err, torch.float32), what + " dbias")


# ------------------------------------------------------------------------------------------------ linear, forward
LINEAR_SHAPES = [
    (1, 8, 8), (1, 64, 72), (3, 1, 16), (16, 1024, 512), (17, 33, 40), (64, 4099, 136), (16, 4096, 4096), (100, 512, 4096),
    (128, 4096, 1024), (128, 4096, 8192), (40, 1024, 4096), (129, 257, 64), (300, 700, 200), (777, 1000, 520), (1024, 2048, 256), (200, 4096, 4096),
    (777, 4099, 2056),
]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", LINEAR_SHAPES, ids=str)
@pytest.mark.parametrize("dtype,out", [(F16, F16), (BF16, BF16), (F16, F32), (BF16, F32)])
def test_linear_forward(cuda_device, shape, dtype, out):
    import torch

    from cuda_hgemm_b200 import api

    M, N, K = shape
    A = make((M, K), dtype, cuda_device, 1)
    B = make((N, K), dtype, cuda_device, 2, K ** -0.5)
    bias = make((N,), dtype, cuda_device, 3)
    residual = make((M, N), out, cuda_device, 4)
    for act in ACTS:
        for with_bias, with_residual, with_pre in ((True, False, True), (False, True, False), (True, True, True)):
            C = torch.full((M, N), SENTINEL, dtype=getattr(torch, out), device=cuda_device)
            pre = torch.full_like(C, SENTINEL) if with_pre else None
            api.hgemm_linear(A, B, C, bias=bias if with_bias else None, act=act, residual=residual if with_residual else None, pre=pre)
            check_forward(A, B, bias if with_bias else None, residual if with_residual else None, act, C, pre, f"{shape} {dtype} {act}")
    assert api.last_device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("act,with_pre", [("gelu", False), ("silu", True), ("none", False)])
def test_linear_forward_large_tiles(cuda_device, dtype, act, with_pre):
    """A shape the dispatch gives to the kernel with 256 x 256 outputs per CTA, with a tail in M."""
    import torch

    from cuda_hgemm_b200 import api

    M, N, K = 4200, 8192, 2048
    A, B = make((M, K), dtype, cuda_device, 1), make((N, K), dtype, cuda_device, 2, K ** -0.5)
    bias, residual = make((N,), dtype, cuda_device, 3), make((M, N), dtype, cuda_device, 4)
    C = torch.full((M, N), SENTINEL, dtype=A.dtype, device=cuda_device)
    pre = torch.full_like(C, SENTINEL) if with_pre else None
    api.hgemm_linear(A, B, C, bias=bias, act=act, residual=residual, pre=pre)
    check_forward(A, B, bias, residual, act, C, pre, act)
    assert api.last_device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_fp32_results_of_long_sums(cuda_device, dtype):
    """The tensor cores cut an accumulator off at every MMA, on average by half of 2^-23 of it: a sum of 512 (32 MMAs)
    is off by at most 32 * 2^-24 in the mean, and so is a longer one, whose pieces are added in FP32 (rounding to
    nearest adds at most 2^-24 each, a quarter of it in the mean). One accumulator for all of a sum of 16384 would be
    off by 32 times that."""
    import torch

    from cuda_hgemm_b200 import api

    limit = 32 * 2.0 ** -24 + 32 * 2.0 ** -24 / 4
    for M, N, K in ((16, 264, 16384), (200, 264, 16384), (512, 4096, 16384), (2000, 2568, 16384)):
        A, B = make((M, K), dtype, cuda_device, 1), make((N, K), dtype, cuda_device, 2)
        C = torch.empty((M, N), device=cuda_device)
        api.hgemm_linear(A, B, C)
        ref = A.double() @ B.double().T
        assert ((C.double() - ref).norm() / ref.norm()).item() < limit, (M, N, K)
    for M, N, K in ((16384, 72, 136), (16384, 2568, 2056)):
        A, dC = make((M, K), dtype, cuda_device, 1), make((M, N), dtype, cuda_device, 2)
        B = torch.zeros((N, K), dtype=A.dtype, device=cuda_device)
        dB = torch.empty((N, K), device=cuda_device)
        api.hgemm_linear_backward(dC, A, B, dB=dB)
        ref = dC.double().T @ A.double()
        assert ((dB.double() - ref).norm() / ref.norm()).item() < limit, (M, N, K)
    assert api.last_device_error() == 0


@pytest.mark.gpu
def test_linear_residual_in_place_and_no_rows(cuda_device):
    import torch

    from cuda_hgemm_b200 import api

    A, B = make((40, 64), BF16, cuda_device, 1), make((72, 64), BF16, cuda_device, 2)
    C = make((40, 72), BF16, cuda_device, 3)
    was = C.clone()
    api.hgemm_linear(A, B, C, residual=C, act="relu")
    check_forward(A, B, None, was, "relu", C, None, "in place")
    api.hgemm_linear(A[:0], B, C[:0], act="silu")
    dB, dbias = torch.full((72, 64), SENTINEL, device=cuda_device), torch.full((72,), SENTINEL, device=cuda_device)
    api.hgemm_linear_backward(C[:0], A[:0], B, dA=A[:0], dB=dB, dbias=dbias, accumulate=True)
    assert (dB == SENTINEL).all() and (dbias == SENTINEL).all()
    api.hgemm_linear_backward(C[:0], A[:0], B, dA=A[:0], dB=dB, dbias=dbias)
    assert (dB == 0).all() and (dbias == 0).all()


# ------------------------------------------------------------------------------------------------ linear, backward
BACKWARD_SHAPES = [
    (1, 8, 8), (1, 64, 72), (15, 136, 40), (16, 16, 16), (17, 128, 256), (33, 1024, 64), (64, 72, 1032), (130, 264, 520),
    (500, 1000, 136), (1000, 2304, 2304), (2049, 256, 128), (1024, 1024, 1024), (5000, 72, 200), (8191, 264, 136),
    (300, 4096, 2048), (1333, 4104, 2040),
]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", BACKWARD_SHAPES, ids=str)
@pytest.mark.parametrize("dtype,out", [(F16, F16), (BF16, BF16), (BF16, F32)])
def test_linear_backward(cuda_device, shape, dtype, out):
    import torch

    from cuda_hgemm_b200 import api

    M, N, K = shape
    A = make((M, K), dtype, cuda_device, 1)
    B = make((N, K), dtype, cuda_device, 2, K ** -0.5)
    dC, pre = make((M, N), out, cuda_device, 3, 0.1), make((M, N), out, cuda_device, 4, 2.0)
    for act in ACTS:
        for db_type in (dtype, F32):
            dZ = torch.full((M, N), SENTINEL, dtype=A.dtype, device=cuda_device) if act != "none" or out == F32 else None
            dA = torch.full((M, K), SENTINEL, dtype=A.dtype, device=cuda_device)
            dB = torch.full((N, K), SENTINEL, dtype=getattr(torch, db_type), device=cuda_device)
            dbias = torch.full((N,), SENTINEL, device=cuda_device)
            api.hgemm_linear_backward(dC, A, B, act=act, pre=pre if act != "none" else None, dA=dA, dB=dB, dbias=dbias, dZ=dZ)
            check_backward(dC, A, B, act, pre, dZ, dA, dB, dbias, f"{shape} {dtype} {act} {db_type}")
    assert api.last_device_error() == 0


@pytest.mark.gpu
def test_linear_backward_in_parts_and_accumulated(cuda_device):
    """Each gradient alone (dZ then lies in scratch) gives the bits of all together; dB and dbias add up in FP32; dZ may be dC."""
    import torch

    from cuda_hgemm_b200 import api

    M, N, K = 300, 264, 136
    A, B = make((M, K), BF16, cuda_device, 1), make((N, K), BF16, cuda_device, 2, 0.1)
    dC, pre = make((M, N), BF16, cuda_device, 3), make((M, N), BF16, cuda_device, 4)
    dZ, dA = torch.empty_like(dC), torch.empty_like(A)
    dB, dbias = torch.empty((N, K), device=cuda_device), torch.empty(N, device=cuda_device)
    api.hgemm_linear_backward(dC, A, B, act="gelu", pre=pre, dA=dA, dB=dB, dbias=dbias, dZ=dZ)
    check_backward(dC, A, B, "gelu", pre, dZ, dA, dB, dbias, "together")
    one = torch.empty_like(A)
    api.hgemm_linear_backward(dC, A, B, act="gelu", pre=pre, dA=one)
    assert torch.equal(one, dA)
    one = torch.empty_like(dB)
    api.hgemm_linear_backward(dC, A, B, act="gelu", pre=pre, dB=one)
    assert torch.equal(one, dB)
    one = torch.empty_like(dbias)
    api.hgemm_linear_backward(dC, A, B, act="gelu", pre=pre, dbias=one)
    assert torch.equal(one, dbias)
    more, more_bias = dB.clone(), dbias.clone()
    api.hgemm_linear_backward(dC, A, B, act="gelu", pre=pre, dB=more, dbias=more_bias, accumulate=True)
    check_backward(dC, A, B, "gelu", pre, dZ, None, more, more_bias, "accumulated", dB_was=dB, dbias_was=dbias)
    in_place = dC.clone()
    api.hgemm_linear_backward(in_place, A, B, act="gelu", pre=pre, dZ=in_place)
    assert torch.equal(in_place, dZ)
    assert api.last_device_error() == 0


# ------------------------------------------------------------------------------------------------ grouped
GROUPS = {
    "one row": [1],
    "no rows": [0, 0, 0],
    "few": [5, 0, 3],
    "edges": [16, 15, 17, 32, 31, 33, 1, 0],
    "decode": [2, 1, 0, 0, 4, 1, 1, 0, 3, 0, 2, 1, 0, 0, 0, 1],
    "uneven": [300, 1, 0, 257, 64],
    "one long": [2050],
    "one takes all": [0, 0, 900, 0],
    "many": [((7 * i * i) % 23) for i in range(70)],
    "even": [128] * 6,
}
GROUPED_SHAPES = [(8, 8), (64, 64), (136, 72), (200, 264), (512, 1032), (1288, 136), (136, 1288)]


def group_inputs(sizes, N, K, dtype, device, before=3, behind=5, gap=0):
    import torch

    M = before + sum(sizes) + behind
    bounds = [before]
    for s in sizes:
        bounds.append(bounds[-1] + s)
    A = make((M, K), dtype, device, 1)
    G = len(sizes)
    B = make((G, N + gap, K), dtype, device, 2, K ** -0.5)[:, :N]
    return M, bounds, torch.tensor(bounds, dtype=torch.int32, device=device), A, B


def forward_of_groups(device, sizes, N, K, dtype, out, act, with_bias, with_pre, gap=0):
    import torch

    from cuda_hgemm_b200 import api

    M, bounds, offsets, A, B = group_inputs(sizes, N, K, dtype, device, gap=gap)
    bias = make((len(sizes), N), dtype, device, 3) if with_bias else None
    # what belongs to no group must not matter
    A[:bounds[0]] = float("nan")
    A[bounds[-1]:] = float("inf")
    C = torch.full((M, N), SENTINEL, dtype=getattr(torch, out), device=device)
    pre = torch.full_like(C, SENTINEL) if with_pre else None
    api.hgemm_grouped(A, B, C, offsets, bias=bias, act=act, pre=pre)
    for g in range(len(sizes)):
        rows = slice(bounds[g], bounds[g + 1])
        check_forward(A[rows], B[g], None if bias is None else bias[g], None, act, C[rows], None if pre is None else pre[rows],
                      f"group {g} of {len(sizes)}, {sizes[g]} rows, {N}x{K} {dtype} {act}")
    for t in (C, pre):
        if t is not None:
            assert (t[:bounds[0]] == SENTINEL).all() and (t[bounds[-1]:] == SENTINEL).all()
    assert api.last_device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("sizes", GROUPS.values(), ids=GROUPS.keys())
@pytest.mark.parametrize("shape", GROUPED_SHAPES, ids=str)
def test_grouped_forward(cuda_device, sizes, shape):
    N, K = shape
    forward_of_groups(cuda_device, sizes, N, K, F16, F16, "none", False, False)
    forward_of_groups(cuda_device, sizes, N, K, BF16, BF16, "silu", True, True)
    forward_of_groups(cuda_device, sizes, N + 1, K, BF16, BF16, "gelu", True, True)
    forward_of_groups(cuda_device, sizes, N + 3, K, F16, F32, "relu", True, False)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,out", [(F16, F16), (BF16, BF16), (F16, F32)])
@pytest.mark.parametrize("act", ACTS)
def test_grouped_forward_on_pairs(cuda_device, dtype, out, act):
    """Enough tiles for the pair kernel: several blocks of rows per group, a stack with gaps, a ragged last block."""
    sizes = [400, 37, 0, 1031, 256, 300, 511, 222]
    forward_of_groups(cuda_device, sizes, 1416, 328, dtype, out, act, True, act != "none", gap=8)
    forward_of_groups(cuda_device, sizes, 1416, 2184, dtype, out, act, True, act != "none")  # (FP32: added up in pieces)


def backward_of_groups(device, sizes, N, K, dtype, out, act, db_type, gap=0, accumulate=False):
    import torch

    from cuda_hgemm_b200 import api

    M, bounds, offsets, A, B = group_inputs(sizes, N, K, dtype, device, gap=gap)
    G = len(sizes)
    dC, pre = make((M, N), out, device, 5, 0.1), make((M, N), out, device, 6, 2.0)
    for t in (A, dC, pre):  # what belongs to no group must not reach a sum
        t[:bounds[0]] = float("nan")
        t[bounds[-1]:] = float("inf")
    tdt = getattr(torch, dtype)
    dZ = torch.full((M, N), SENTINEL, dtype=tdt, device=device) if act != "none" or out == F32 else None
    dA = torch.full((M, K), SENTINEL, dtype=tdt, device=device)
    dB = torch.full((G, N, K), SENTINEL, dtype=getattr(torch, db_type), device=device)
    dbias = torch.full((G, N), SENTINEL, device=device)
    api.hgemm_grouped_backward(dC, A, B, offsets, act=act, pre=pre if act != "none" else None, dA=dA, dB=dB, dbias=dbias, dZ=dZ,
                               accumulate=accumulate)
    was = torch.full((N, K), SENTINEL, device=device) if accumulate else None
    was_bias = torch.full((N,), SENTINEL, device=device) if accumulate else None
    for g in range(G):
        rows = slice(bounds[g], bounds[g + 1])
        check_backward(dC[rows], A[rows], B[g], act, pre[rows], None if dZ is None else dZ[rows], dA[rows], dB[g], dbias[g],
                       f"group {g} of {G}, {sizes[g]} rows, {N}x{K} {dtype} {act} {db_type}", dB_was=was, dbias_was=was_bias)
    for t in (dA, dZ):
        if t is not None:
            assert (t[:bounds[0]] == SENTINEL).all() and (t[bounds[-1]:] == SENTINEL).all()
    assert api.last_device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("sizes", GROUPS.values(), ids=GROUPS.keys())
@pytest.mark.parametrize("shape", GROUPED_SHAPES, ids=str)
def test_grouped_backward(cuda_device, sizes, shape):
    N, K = shape
    backward_of_groups(cuda_device, sizes, N, K, F16, F16, "none", F32)
    backward_of_groups(cuda_device, sizes, N, K, BF16, BF16, "silu", BF16)
    backward_of_groups(cuda_device, sizes, N, K, F16, F32, "gelu_tanh", F16)
    backward_of_groups(cuda_device, sizes, N, K, BF16, BF16, "relu", F32, accumulate=True)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(1416, 328), (328, 1416), (1032, 776), (2048, 1024), (1344, 1088)], ids=str)
@pytest.mark.parametrize("dtype,db_type", [(F16, F16), (BF16, F32)])
def test_grouped_backward_on_pairs(cuda_device, shape, dtype, db_type):
    N, K = shape
    sizes = [400, 37, 0, 1031, 256, 300, 511, 222, 1, 63]
    backward_of_groups(cuda_device, sizes, N, K, dtype, dtype, "gelu", db_type, gap=8)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,db_type", [(F16, F16), (BF16, F32)])
def test_grouped_backward_of_long_groups(cuda_device, dtype, db_type):
    """Groups long enough for pairs in the weights' gradient too, most of them ending inside a block of 64 rows."""
    sizes = [2600, 37, 0, 4031, 777, 3000]
    backward_of_groups(cuda_device, sizes, 2040, 1528, dtype, dtype, "silu", db_type)
    backward_of_groups(cuda_device, sizes, 2048, 1536, dtype, dtype, "none", F32, accumulate=True)


@pytest.mark.gpu
def test_rows_of_the_next_group_stay_out_of_a_weight_gradient(cuda_device):
    """A NaN in one group's rows makes its own gradients NaN and nobody else's."""
    import torch

    from cuda_hgemm_b200 import api

    for N, K, sizes in ((136, 72, [5, 7, 70, 64, 3]), (2040, 1528, [1000, 7, 2070, 640, 3, 1290, 1])):  # single CTAs, pairs
        M, bounds, offsets, A, B = group_inputs(sizes, N, K, F16, cuda_device)
        dC = make((M, N), F16, cuda_device, 5)
        bad = 1
        A[bounds[bad]:bounds[bad + 1]] = float("nan")
        dC[bounds[bad]:bounds[bad + 1]] = float("inf")
        dB = torch.empty((len(sizes), N, K), device=cuda_device)
        dbias = torch.empty((len(sizes), N), device=cuda_device)
        api.hgemm_grouped_backward(dC, A, B, offsets, dB=dB, dbias=dbias)
        for g in range(len(sizes)):
            finite = torch.isfinite(dB[g]).all().item() and torch.isfinite(dbias[g]).all().item()
            assert finite == (g != bad), g
        assert api.last_device_error() == 0


@pytest.mark.gpu
def test_offsets_out_of_order_stay_inside_the_operands(cuda_device):
    """Such offsets are held within the rows there are: nothing outside the outputs is written, sound groups are right."""
    import torch

    from cuda_hgemm_b200 import api

    N, K, M = 136, 72, 200
    A, B = make((M, K), F16, cuda_device, 1), make((4, N, K), F16, cuda_device, 2)
    room = torch.full((M + 64, N), SENTINEL, dtype=torch.float16, device=cuda_device)
    for values in ([0, 50, 20, 150, 5000], [-7, 50, 2 ** 31 - 1, 60, 100], [-2 ** 31, -1, 0, 0, 200]):
        offsets = torch.tensor(values, dtype=torch.int32, device=cuda_device)
        C = room[:M]
        api.hgemm_grouped(A, B, C, offsets)
        dB = torch.empty((4, N, K), device=cuda_device)
        dA = torch.empty_like(A)
        api.hgemm_grouped_backward(C, A, B, offsets, dA=dA, dB=dB, act="silu", pre=C)
        assert (room[M:] == SENTINEL).all()
    check_forward(A, B[3], None, None, "none", room[:M], None, "last group")
    assert api.last_device_error() == 0


@pytest.mark.gpu
def test_more_than_2_to_the_32_elements(cuda_device):
    """An output of 4.6e9 elements: its last rows lie beyond what 32 bits count."""
    import torch

    from cuda_hgemm_b200 import api

    M, N, K = 70001, 65536, 8
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("not enough free memory")
    A, B = make((M, K), BF16, cuda_device, 1), make((N, K), BF16, cuda_device, 2)
    bias = make((N,), BF16, cuda_device, 3)
    C = torch.empty((M, N), dtype=torch.bfloat16, device=cuda_device)
    api.hgemm_linear(A, B, C, bias=bias, act="gelu")
    for rows in (slice(0, 3), slice(65534, 65539), slice(M - 3, M)):
        check_forward(A[rows], B, bias, None, "gelu", C[rows], None, str(rows))
    dA, dbias = torch.empty_like(A), torch.empty(N, device=cuda_device)
    dB = torch.empty((N, K), device=cuda_device)
    C[:M - 2] = 0  # what is left to sum lies in the last two rows
    api.hgemm_linear_backward(C, A, B, dA=dA, dB=dB, dbias=dbias)
    last = slice(M - 2, M)
    check_backward(C[last], A[last], B, "none", None, None, dA[last], dB, dbias, "last rows")
    assert (dA[:M - 2] == 0).all()
    offsets = torch.tensor([0, 5, M], dtype=torch.int32, device=cuda_device)
    C.fill_(SENTINEL)
    api.hgemm_grouped(A, torch.stack([B, B.flip(0)]), C, offsets, act="relu")
    check_forward(A[last], B.flip(0), None, None, "relu", C[last], None, "last group")
    assert api.last_device_error() == 0


@pytest.mark.gpu
def test_two_layers_of_experts_forward_and_backward(cuda_device):
    """Up projection with activation, down projection, and all their gradients, as a layer of experts runs them: against
    the 64-bit chain rule on the values the layers hand on, and the weights' gradient against differences."""
    import torch

    from cuda_hgemm_b200 import api

    sizes, D, H = [130, 0, 61, 300, 9], 264, 520
    M, bounds, offsets, X, W1 = group_inputs(sizes, H, D, BF16, cuda_device, before=0, behind=0)
    G = len(sizes)
    W2 = make((G, D, H), BF16, cuda_device, 7, H ** -0.5)
    b1 = make((G, H), BF16, cuda_device, 8)
    h, z = torch.empty((M, H), dtype=torch.bfloat16, device=cuda_device), torch.empty((M, H), dtype=torch.bfloat16, device=cuda_device)
    y = torch.empty((M, D), dtype=torch.bfloat16, device=cuda_device)
    api.hgemm_grouped(X, W1, h, offsets, bias=b1, act="silu", pre=z)
    api.hgemm_grouped(h, W2, y, offsets)
    dy = make((M, D), BF16, cuda_device, 9)
    dh, dW2 = torch.empty_like(h), torch.empty((G, D, H), device=cuda_device)
    api.hgemm_grouped_backward(dy, h, W2, offsets, dA=dh, dB=dW2)
    dx, dW1, db1 = torch.empty_like(X), torch.empty((G, H, D), device=cuda_device), torch.empty((G, H), device=cuda_device)
    dz = torch.empty_like(h)
    api.hgemm_grouped_backward(dh, X, W1, offsets, act="silu", pre=z, dA=dx, dB=dW1, dbias=db1, dZ=dz)
    for g in range(G):
        r = slice(bounds[g], bounds[g + 1])
        check_forward(X[r], W1[g], b1[g], None, "silu", h[r], z[r], f"up {g}")
        check_forward(h[r], W2[g], None, None, "none", y[r], None, f"down {g}")
        check_backward(dy[r], h[r], W2[g], "none", None, None, dh[r], dW2[g], None, f"down' {g}")
        check_backward(dh[r], X[r], W1[g], "silu", z[r], dz[r], dx[r], dW1[g], db1[g], f"up' {g}")
    # differences in 64 bits: loss = sum(dy * y(W1)); one weight of each group that has rows
    for g in (0, 2, 3, 4):
        r = slice(bounds[g], bounds[g + 1])

        def loss(w):
            return (dy[r].double() * (act64(X[r].double() @ w.T + b1[g].double(), "silu") @ W2[g].double().T)).sum().item()

        w = W1[g].double()
        for i, j in ((0, 0), (H - 1, D - 1), (77, 130)):
            step = torch.zeros_like(w)
            step[i, j] = 1e-4
            slope = (loss(w + step) - loss(w - step)) / 2e-4
            # what the chain rounds on its way, in the inputs' type: z once (before the slope), dh and dz once; the
            # slope of silu changes by at most half of what z does
            u = half_step(BF16)
            dz_abs = (dh[r, i].double().abs() + dz[r, i].double().abs() + dh[r, i].double().abs() * z[r, i].double().abs() * 0.5)
            tol = 2 * u * (dz_abs * X[r, j].double().abs()).sum().item() + 1e-4 * abs(slope) + 1e-5
            # dh itself is a rounded sum: its own bound enters through u * |dh|
            assert abs(dW1[g, i, j].item() - slope) <= tol, (g, i, j, dW1[g, i, j].item(), slope, tol)
    assert api.last_device_error() == 0


@pytest.mark.gpu
def test_captured_replayed_and_on_another_stream(cuda_device):
    """One graph of a forward and a backward call, replayed with other group sizes; and the calls on a side stream."""
    import torch

    from cuda_hgemm_b200 import api

    N, K, M = 264, 136, 400
    A, B = make((M, K), BF16, cuda_device, 1), make((3, N, K), BF16, cuda_device, 2, 0.1)
    dC = make((M, N), BF16, cuda_device, 3)
    offsets = torch.tensor([0, 100, 100, 400], dtype=torch.int32, device=cuda_device)
    C, pre = torch.zeros((M, N), dtype=torch.bfloat16, device=cuda_device), torch.zeros((M, N), dtype=torch.bfloat16, device=cuda_device)
    dA = torch.zeros_like(A)
    dB, dbias = torch.zeros((3, N, K), device=cuda_device), torch.zeros((3, N), device=cuda_device)

    def step():
        api.hgemm_grouped(A, B, C, offsets, act="gelu", pre=pre)
        api.hgemm_grouped_backward(dC, A, B, offsets, act="gelu", pre=pre, dA=dA, dB=dB, dbias=dbias)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for values in ([0, 100, 100, 400], [0, 0, 333, 390], [10, 11, 27, 28]):
        offsets.copy_(torch.tensor(values, dtype=torch.int32))
        graph.replay()
        got = [t.clone() for t in (C, pre, dA, dB, dbias)]
        step()
        for a, b in zip(got, (C, pre, dA, dB, dbias)):
            assert torch.equal(a, b)
        for g in range(3):
            r = slice(values[g], values[g + 1])
            check_forward(A[r], B[g], None, None, "gelu", C[r], pre[r], f"{values} {g}")
    assert api.last_device_error() == 0


@pytest.mark.gpu
def test_two_streams_at_once(cuda_device):
    """Forward and backward calls of two layers, each on its own stream, run into each other: the bits of a run alone."""
    import torch

    from cuda_hgemm_b200 import api

    layers = []
    for seed, (sizes, N, K) in enumerate((([300, 0, 5, 700], 520, 264), ([64, 900, 33], 1032, 520))):
        M, bounds, offsets, A, B = group_inputs(sizes, N, K, BF16, cuda_device)
        G = len(sizes)
        layers.append(dict(A=A, B=B, offsets=offsets, dC=make((M, N), BF16, cuda_device, 50 + seed), G=G, N=N, K=K, M=M))

    def outputs(l):
        new = lambda shape, dt: torch.zeros(shape, dtype=dt, device=cuda_device)  # noqa: E731
        return dict(C=new((l["M"], l["N"]), torch.bfloat16), pre=new((l["M"], l["N"]), torch.bfloat16), dA=new((l["M"], l["K"]), torch.bfloat16),
                    dB=new((l["G"], l["N"], l["K"]), torch.float32), dbias=new((l["G"], l["N"]), torch.float32),
                    D=new((16, l["N"]), torch.bfloat16))

    def step(l, o):
        api.hgemm_grouped(l["A"], l["B"], o["C"], l["offsets"], act="gelu", pre=o["pre"])
        api.hgemm_linear(l["A"][8:24], l["B"][0], o["D"], act="silu")
        api.hgemm_grouped_backward(l["dC"], l["A"], l["B"], l["offsets"], act="gelu", pre=o["pre"], dA=o["dA"], dB=o["dB"], dbias=o["dbias"])

    alone = []
    for l in layers:
        o = outputs(l)
        step(l, o)
        torch.cuda.synchronize()
        alone.append(o)
    streams = [torch.cuda.Stream() for _ in layers]
    together = [outputs(l) for l in layers]
    torch.cuda.synchronize()
    for _ in range(30):
        for l, o, s in zip(layers, together, streams):
            with torch.cuda.stream(s):
                step(l, o)
    torch.cuda.synchronize()
    for a, b in zip(alone, together):
        for name in a:
            assert torch.equal(a[name], b[name]), name
    assert api.last_device_error() == 0


@pytest.mark.gpu
def test_same_inputs_same_bits(cuda_device):
    import torch

    from cuda_hgemm_b200 import api

    sizes = [((13 * i * i) % 97) for i in range(40)]
    M, bounds, offsets, A, B = group_inputs(sizes, 264, 520, F16, cuda_device)
    dC = make((M, 264), F16, cuda_device, 5)
    results = []
    for _ in range(3):
        dA, dB = torch.zeros_like(A), torch.empty((40, 264, 520), device=cuda_device)
        dbias = torch.empty((40, 264), device=cuda_device)
        api.hgemm_grouped_backward(dC, A, B, offsets, act="silu", pre=dC, dA=dA, dB=dB, dbias=dbias)
        results.append((dA, dB, dbias))
    for r in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(r, results[0]))


# ------------------------------------------------------------------------------------------------ refusals
def test_refusals_come_before_any_device_work(native_lib):
    buf = ctypes.create_string_buffer(4096)
    p = (ctypes.addressof(buf) + 255) & ~255
    A = _native.LinearArgs
    ok = dict(in_type=_native.C_F16, c_type=_native.C_F16, act=0)

    def linear(A_=p, B_=p, C_=p, M=8, N=8, K=8, args=None, **kw):
        args = A(**{**ok, **kw}) if args is None else args
        return native_lib.b200_hgemm_linear(A_, B_, C_, M, N, K, ctypes.byref(args), None, 0, None)

    assert linear(A_=None) == linear(B_=None) == linear(C_=None) == _native.ERR_INVALID_ARG
    assert linear(N=0) == linear(K=0) == _native.ERR_INVALID_ARG
    assert linear(act=5) == linear(act=-1) == _native.ERR_INVALID_ARG
    assert linear(in_type=_native.C_F32) == linear(c_type=_native.C_BF16) == linear(c_type=7) == _native.ERR_INVALID_ARG
    assert linear(K=12) == _native.ERR_UNSUPPORTED
    assert linear(M=1 << 40) == _native.ERR_UNSUPPORTED
    assert linear(M=0, A_=None, C_=None) == _native.OK
    assert native_lib.b200_hgemm_linear(p, p, p, 8, 8, 8, None, None, 0, None) == _native.ERR_INVALID_ARG

    def grouped(offsets=p, G=2, stride=64, M=8, N=8, K=8, A_=p, B_=p, C_=p, **kw):
        return native_lib.b200_hgemm_grouped(A_, B_, C_, offsets, M, N, K, G, stride, ctypes.byref(A(**{**ok, **kw})), None)

    assert grouped(offsets=None) == grouped(G=0) == grouped(stride=56) == grouped(A_=None) == _native.ERR_INVALID_ARG
    assert grouped(offsets=p + 2) == grouped(stride=68) == grouped(C_=p + 8) == grouped(bias=p + 4) == grouped(pre=p + 2) == _native.ERR_MISALIGNED
    assert grouped(G=1025, stride=64) == _native.ERR_TOO_LARGE
    assert grouped(K=4, stride=64) == grouped(residual=p) == _native.ERR_UNSUPPORTED
    assert grouped(act=9) == grouped(in_type=2) == _native.ERR_INVALID_ARG
    assert grouped(M=0, A_=None, C_=None) == _native.OK


def test_backward_refusals_come_before_any_device_work(native_lib):
    buf = ctypes.create_string_buffer(4096)
    p = (ctypes.addressof(buf) + 255) & ~255
    ok = dict(in_type=_native.C_F16, c_type=_native.C_F16, act=0, db_type=_native.C_F16, accumulate=0, dC=p, dA=p, dB=p)

    def backward(A_=p, B_=p, M=8, N=8, K=8, ws=None, ws_bytes=0, **kw):
        return native_lib.b200_hgemm_linear_backward(A_, B_, M, N, K, ctypes.byref(_native.LinearGrads(**{**ok, **kw})), ws, ws_bytes, None)

    assert backward(dC=None) == backward(A_=None) == backward(B_=None) == backward(N=0) == backward(K=0) == _native.ERR_INVALID_ARG
    assert backward(act=1) == backward(act=7) == backward(db_type=1) == backward(c_type=1) == backward(in_type=2) == _native.ERR_INVALID_ARG
    assert backward(dA=None, dB=None) == _native.ERR_INVALID_ARG
    assert backward(N=12) == backward(K=20) == backward(accumulate=1) == _native.ERR_UNSUPPORTED
    assert backward(dA=p + 4) == backward(dbias=p + 4) == backward(dC=p + 8) == _native.ERR_MISALIGNED
    # dZ has to lie somewhere: in the workspace, which is too small or missing
    need = native_lib.b200_hgemm_backward_workspace_bytes(8, 8, 8, 1, ctypes.byref(_native.LinearGrads(**{**ok, "act": 2, "pre": p})))
    assert need >= 8 * 8 * 2
    assert backward(act=2, pre=p) == backward(act=2, pre=p, ws=p, ws_bytes=need - 1) == _native.ERR_WORKSPACE
    assert backward(act=2, pre=p, ws=p + 16, ws_bytes=need) == _native.ERR_MISALIGNED
    # nothing to keep: no activation, or the caller takes dZ
    assert native_lib.b200_hgemm_backward_workspace_bytes(8, 8, 8, 1, ctypes.byref(_native.LinearGrads(**ok))) == 0
    assert native_lib.b200_hgemm_backward_workspace_bytes(8, 8, 8, 1, ctypes.byref(_native.LinearGrads(**{**ok, "act": 2, "pre": p, "dZ": p}))) == 0

    def grouped(offsets=p, G=2, stride=64, **kw):
        return native_lib.b200_hgemm_grouped_backward(p, p, offsets, 8, 8, 8, G, stride, ctypes.byref(_native.LinearGrads(**{**ok, **kw})), None, 0, None)

    assert grouped(offsets=None) == grouped(G=0) == grouped(stride=8) == _native.ERR_INVALID_ARG
    assert grouped(G=5000) == _native.ERR_TOO_LARGE
    assert grouped(stride=65) == _native.ERR_MISALIGNED


def test_valid_calls_without_a_gpu_fail_loudly(native_lib):
    import torch

    if torch.cuda.is_available():
        pytest.skip("a GPU is present; the no-device answer cannot be observed")
    buf = ctypes.create_string_buffer(4096)
    p = (ctypes.addressof(buf) + 255) & ~255
    args = _native.LinearArgs(in_type=_native.C_BF16, c_type=_native.C_BF16, act=1)
    no_device = (_native.ERR_CUDA, _native.ERR_NO_SM100)
    assert native_lib.b200_hgemm_linear(p, p, p, 8, 8, 8, ctypes.byref(args), None, 0, None) in no_device
    assert native_lib.b200_hgemm_grouped(p, p, p, p, 8, 8, 8, 1, 64, ctypes.byref(args), None) in no_device
    grads = _native.LinearGrads(in_type=_native.C_F16, c_type=_native.C_F16, db_type=_native.C_F32, dC=p, dB=p)
    assert native_lib.b200_hgemm_linear_backward(p, p, 8, 8, 8, ctypes.byref(grads), None, 0, None) in no_device


def test_wrappers_refuse_what_is_not_on_a_gpu():
    import torch

    from cuda_hgemm_b200 import api

    a, b, c = torch.zeros(4, 8).half(), torch.zeros(8, 8).half(), torch.zeros(4, 8).half()
    with pytest.raises(TypeError):
        api.hgemm_linear(a, b, c)
    with pytest.raises(TypeError):
        api.hgemm_grouped(a, b[None], c, None)
    with pytest.raises(TypeError):
        api.hgemm_grouped(a, b[None], c, torch.zeros(2, dtype=torch.int32))
    with pytest.raises(TypeError):
        api.hgemm_linear_backward(c, a, b, dA=a)


@pytest.mark.gpu
def test_wrappers_refuse_mismatched_tensors(cuda_device):
    import torch

    from cuda_hgemm_b200 import api

    A, B, C = make((16, 64), F16, cuda_device, 1), make((24, 64), F16, cuda_device, 2), make((16, 24), F16, cuda_device, 3)
    W, off = make((2, 24, 64), F16, cuda_device, 2), torch.tensor([0, 8, 16], dtype=torch.int32, device=cuda_device)
    for call, error in (
        (lambda: api.hgemm_linear(A, B.bfloat16(), C), TypeError),
        (lambda: api.hgemm_linear(A, B, C.bfloat16()), TypeError),
        (lambda: api.hgemm_linear(A, B, C[:8]), ValueError),
        (lambda: api.hgemm_linear(A.T.contiguous().T, B, C), TypeError),
        (lambda: api.hgemm_linear(A, B, C, act="tanh"), ValueError),
        (lambda: api.hgemm_linear(A, B, C, bias=torch.zeros(24, device=cuda_device)), TypeError),
        (lambda: api.hgemm_linear(A, B, C, residual=C.float()), TypeError),
        (lambda: api.hgemm_linear(A, B, None), TypeError),
        (lambda: api.hgemm_grouped(A, W, C, off.long()), TypeError),
        (lambda: api.hgemm_grouped(A, W, C, off[:2]), ValueError),
        (lambda: api.hgemm_grouped(A, W.transpose(1, 2).contiguous().transpose(1, 2), C, off), ValueError),
        (lambda: api.hgemm_grouped(A, B, C, off), ValueError),
        (lambda: api.hgemm_linear_backward(C, A, B, act="silu", dA=A), ValueError),
        (lambda: api.hgemm_linear_backward(C, A, B), ValueError),
        (lambda: api.hgemm_linear_backward(C, A, B, dbias=torch.zeros(24, device=cuda_device).half()), TypeError),
        (lambda: api.hgemm_linear_backward(C, A, B, dB=torch.zeros_like(B), accumulate=True), api.HgemmError),
    ):
        with pytest.raises(error):
            call()
