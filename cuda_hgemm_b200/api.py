"""Python-side mirror of the kernel entry points, for tests and the benchmark.

The reference registers one callable per kernel, all of the shape
``void name(half *A, half *B, half *C, size_t M, size_t N, size_t K)`` (reference
src/main.cu:11-33). The functions here keep that argument order and meaning for torch CUDA
tensors: ``A`` is ``[M, K]`` row-major, ``B`` is ``[N, K]`` row-major (the reference's
"col-major K x N", src/common/tester.h:117-119), ``C`` is ``[M, N]`` row-major; all float16
and contiguous. Everything runs on torch's current stream and returns without synchronising.
torch is used for device memory and streams only; the arithmetic is the native library's.
"""
from __future__ import annotations

import contextlib
import ctypes

from . import _native
from ._native import HgemmError, Plan, check

__all__ = [
    "b200Hgemm", "b200HgemmCta1", "b200HgemmCta2", "b200HgemmSplitK", "b200HgemmStreamK", "b200HgemmSimt",
    "hgemm_linear", "hgemm_linear_backward", "hgemm_grouped", "hgemm_grouped_backward", "ACTIVATIONS",
    "hgemm_ex", "hgemm_host", "select_plan", "workspace_bytes", "last_device_error", "launch_count",
    "KERNEL_LOG_NAMES", "Plan", "HgemmError",
]

# log names, in the reference's style (no spaces: its plot tool splits lines on spaces,
# reference tools/performance/performance.py:57-62)
KERNEL_LOG_NAMES = {
    "b200Hgemm": "B200-Tcgen05-Auto",
    "b200HgemmCta1": "B200-Tcgen05-1Cta",
    "b200HgemmCta2": "B200-Tcgen05-2Cta",
    "b200HgemmSplitK": "B200-Tcgen05-SplitK",
    "b200HgemmStreamK": "B200-Tcgen05-StreamK",
    "b200HgemmSimt": "B200-Simt-Fp32Acc",
}


def _shape_of(A, B, C, c_dtypes=None):
    import torch

    for name, t in (("A", A), ("B", B), ("C", C)):
        ok_types = c_dtypes if (name == "C" and c_dtypes) else (torch.float16,)
        if not isinstance(t, torch.Tensor) or t.dtype not in ok_types or not t.is_cuda or not t.is_contiguous():
            raise TypeError(f"{name} must be a contiguous float16 CUDA tensor")
        if t.dim() != 2:
            raise ValueError(f"{name} must be 2-D")
    M, K = A.shape
    N, Kb = B.shape
    if Kb != K or tuple(C.shape) != (M, N):
        raise ValueError(f"shape mismatch: A {tuple(A.shape)}, B {tuple(B.shape)} (N x K), C {tuple(C.shape)}")
    if A.device != B.device or A.device != C.device:
        raise ValueError("A, B and C must live on one device")
    return int(M), int(N), int(K)


def _stream_of(t) -> int:
    import torch

    # torch's own number of the stream where this torch has it; the public call builds a Stream object: 3 us of a call's 17
    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
    return raw(t.get_device()) if raw is not None else int(torch.cuda.current_stream(t.device).cuda_stream)


def _call(symbol: str, A, B, C):
    import torch

    M, N, K = _shape_of(A, B, C)
    fn = getattr(_native.load(), symbol)
    with torch.cuda.device(A.device):
        check(fn(A.data_ptr(), B.data_ptr(), C.data_ptr(), M, N, K, _stream_of(A)))
    return C


def b200Hgemm(A, B, C):
    """Auto-dispatching GEMM (C ABI ``b200_hgemm``)."""
    return _call("b200_hgemm", A, B, C)


def b200HgemmCta1(A, B, C):
    """Single-CTA tcgen05 tiles (C ABI ``b200_hgemm_cta1``)."""
    return _call("b200_hgemm_cta1", A, B, C)


def b200HgemmCta2(A, B, C):
    """CTA-pair tcgen05 tiles (C ABI ``b200_hgemm_cta2``)."""
    return _call("b200_hgemm_cta2", A, B, C)


def b200HgemmSplitK(A, B, C):
    """Fixed k-slices per tile with an FP32 workspace reduce (C ABI ``b200_hgemm_splitk``)."""
    return _call("b200_hgemm_splitk", A, B, C)


def b200HgemmStreamK(A, B, C):
    """Equal k-ranges over all SMs (C ABI ``b200_hgemm_streamk``)."""
    return _call("b200_hgemm_streamk", A, B, C)


def b200HgemmSimt(A, B, C):
    """CUDA-core kernel for any shape (C ABI ``b200_hgemm_simt``)."""
    return _call("b200_hgemm_simt", A, B, C)


def hgemm_ex(A, B, C, plan: Plan):
    """Run an explicit plan (C ABI ``b200_hgemm_ex``): ``plan.variant`` one of the ``_native.VARIANT_*``
    kernel families, ``plan.bn`` the tile width (or, for the large-tile and short-A kernels, the
    arrangement: see ``include/b200_hgemm.h``), ``plan.parts`` the number of k-ranges where k is cut."""
    import torch

    M, N, K = _shape_of(A, B, C)
    with torch.cuda.device(A.device):
        check(_native.load().b200_hgemm_ex(A.data_ptr(), B.data_ptr(), C.data_ptr(), M, N, K, ctypes.byref(plan),
                                           _stream_of(A)))
    return C


def hgemm_fused(A, B, C, alpha: float = 1.0, beta: float = 0.0, bias=None, c_in=None, plan: Plan = None):
    """``C = alpha * A @ B.T + beta * c_in + bias`` in one kernel (C ABI ``b200_hgemm_fused``, or
    ``b200_hgemm_fused_ex`` when a ``plan`` is given). ``C`` may be float16, bfloat16 or float32; ``bias`` has one
    FP16 value per column of C; ``c_in`` is an ``[M, N]`` tensor of C's dtype (``C`` itself for an in-place update)."""
    import torch

    c_types = {torch.float16: _native.C_F16, torch.bfloat16: _native.C_BF16, torch.float32: _native.C_F32}
    if not isinstance(C, torch.Tensor) or C.dtype not in c_types or not C.is_cuda or not C.is_contiguous() or C.dim() != 2:
        raise TypeError("C must be a contiguous 2-D float16, bfloat16 or float32 CUDA tensor")
    M, N, K = _shape_of(A, B, C, c_dtypes=tuple(c_types))
    if bias is not None and (bias.dtype != torch.float16 or bias.numel() != N or not bias.is_contiguous()):
        raise ValueError("bias must be a contiguous float16 tensor with one value per column of C")
    if c_in is not None and (c_in.dtype != C.dtype or tuple(c_in.shape) != (M, N) or not c_in.is_contiguous()):
        raise ValueError("c_in must be a contiguous [M, N] tensor of C's dtype")
    epi = _native.Epilogue(alpha, beta, bias.data_ptr() if bias is not None else None,
                           c_in.data_ptr() if c_in is not None else None, c_types[C.dtype])
    lib = _native.load()
    with torch.cuda.device(A.device):
        if plan is None:
            check(lib.b200_hgemm_fused(A.data_ptr(), B.data_ptr(), C.data_ptr(), M, N, K, ctypes.byref(epi), _stream_of(A)))
        else:
            check(lib.b200_hgemm_fused_ex(A.data_ptr(), B.data_ptr(), C.data_ptr(), M, N, K, ctypes.byref(epi),
                                          ctypes.byref(plan), _stream_of(A)))
    return C


def hgemm_bkn(A, B_kn, C):
    """``C = A @ B_kn`` with ``B_kn`` stored ``[K, N]`` row-major (C ABI ``b200_hgemm_bkn``): no transpose is made."""
    import torch

    for name, t in (("A", A), ("B_kn", B_kn), ("C", C)):
        if not isinstance(t, torch.Tensor) or t.dtype != torch.float16 or not t.is_cuda or not t.is_contiguous() or t.dim() != 2:
            raise TypeError(f"{name} must be a contiguous 2-D float16 CUDA tensor")
    M, K = A.shape
    Kb, N = B_kn.shape
    if Kb != K or tuple(C.shape) != (M, N):
        raise ValueError("shape mismatch")
    with torch.cuda.device(A.device):
        check(_native.load().b200_hgemm_bkn(A.data_ptr(), B_kn.data_ptr(), C.data_ptr(), int(M), int(N), int(K), _stream_of(A)))
    return C


def hgemm_batched(A, B, C):
    """``C[i] = A[i] @ B[i].T`` for stacks ``A [batch, M, K]``, ``B [batch, N, K]`` (or one ``[N, K]`` matrix for all),
    ``C [batch, M, N]`` (C ABI ``b200_hgemm_batched``). The innermost two dimensions must be contiguous; the
    stack dimension may have any stride that is a multiple of 8 elements."""
    import torch

    for name, t in (("A", A), ("B", B), ("C", C)):
        if not isinstance(t, torch.Tensor) or t.dtype != torch.float16 or not t.is_cuda:
            raise TypeError(f"{name} must be a float16 CUDA tensor")
    if A.dim() != 3 or C.dim() != 3 or B.dim() not in (2, 3):
        raise ValueError("A and C must be [batch, rows, cols]; B [batch, N, K] or [N, K]")
    batch, M, K = A.shape
    N = B.shape[-2]
    if B.shape[-1] != K or tuple(C.shape) != (batch, M, N) or (B.dim() == 3 and B.shape[0] != batch):
        raise ValueError("shape mismatch")
    for name, t in (("A", A), ("B", B), ("C", C)):
        if t.stride(-1) != 1 or t.stride(-2) != t.shape[-1]:
            raise ValueError(f"the matrices of {name} must be contiguous")
    stride_b = B.stride(0) if B.dim() == 3 else 0
    with torch.cuda.device(A.device):
        check(_native.load().b200_hgemm_batched(A.data_ptr(), B.data_ptr(), C.data_ptr(), int(M), int(N), int(K), int(batch),
                                                int(A.stride(0)), int(stride_b), int(C.stride(0)), _stream_of(A)))
    return C


# activation names of the feed-forward products -> B200_ACT_*
ACTIVATIONS = {"none": _native.ACT_NONE, "relu": _native.ACT_RELU, "gelu": _native.ACT_GELU,
               "gelu_tanh": _native.ACT_GELU_TANH, "silu": _native.ACT_SILU}


def _type_code(dtype):
    import torch

    return _native.C_F16 if dtype is torch.float16 else _native.C_BF16 if dtype is torch.bfloat16 else _native.C_F32 if dtype is torch.float32 else None


def _act_code(act):
    try:
        return ACTIVATIONS[act]
    except (KeyError, TypeError):
        raise ValueError(f"act must be one of {', '.join(ACTIVATIONS)}") from None


def _operand(name, t, dtypes, shape, device):
    """A contiguous CUDA tensor of one of ``dtypes`` and of ``shape`` on device number ``device``; its address (``None`` for an
    absent one)."""
    if t is None:
        return None
    if getattr(t, "dtype", None) not in dtypes or not t.is_cuda or not t.is_contiguous():  # (also what is no tensor at all)
        raise TypeError(f"{name} must be a contiguous CUDA tensor of type {' or '.join(str(d)[6:] for d in dtypes)}")
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, not {tuple(t.shape)}")
    if t.get_device() != device:
        raise ValueError(f"{name} must live on cuda:{device}")
    return t.data_ptr()


def _rows_and_weights(A, B, offsets):
    """Shapes and input type of ``A [M, K]`` and ``B [N, K]``, or ``B [G, N, K]`` where ``offsets`` are given."""
    import torch

    grouped = offsets is not None
    dtype = getattr(A, "dtype", None)
    if (dtype is not torch.float16 and dtype is not torch.bfloat16) or not A.is_cuda:
        raise TypeError("A must be a float16 or bfloat16 CUDA tensor")
    if getattr(B, "dtype", None) is not dtype or not B.is_cuda:
        raise TypeError("B must be a CUDA tensor of A's type")
    a_shape, b_shape = A.shape, B.shape
    if len(a_shape) != 2:
        raise ValueError("A must be 2-D")
    if len(b_shape) != (3 if grouped else 2):
        raise ValueError(f"B must be {3 if grouped else 2}-D")
    if A.get_device() != B.get_device():
        raise ValueError("A and B must live on one device")
    M, K = a_shape
    N = b_shape[-2]
    if b_shape[-1] != K:
        raise ValueError(f"shape mismatch: A {tuple(a_shape)}, B {tuple(b_shape)}")
    if not A.is_contiguous():
        raise TypeError("A must be contiguous")
    if not grouped:
        if not B.is_contiguous():
            raise TypeError("B must be contiguous")
        return M, N, K, 1, N * K
    G = B.shape[0]
    # the matrices must be dense (a dimension of one element may have any stride); the stack may have gaps
    if (B.stride(2) != 1 and K > 1) or (B.stride(1) != K and N > 1):
        raise ValueError("the matrices of B must be contiguous")
    if getattr(offsets, "dtype", None) != torch.int32 or not offsets.is_cuda or not offsets.is_contiguous():
        raise TypeError("offsets must be a contiguous int32 CUDA tensor")
    if offsets.shape != (G + 1,):
        raise ValueError(f"offsets must have {G + 1} values, one more than B has matrices")
    if offsets.get_device() != A.get_device():
        raise ValueError("offsets must live on A's device")
    return M, N, K, G, B.stride(0) if G > 1 else N * K


_NOTHING = contextlib.nullcontext()


def _on_device(t):
    """A context in which ``t``'s device is the current one (nothing to do where it is already)."""
    import torch

    return _NOTHING if torch.cuda.current_device() == t.get_device() else torch.cuda.device(t.device)


def _scratch(nbytes, device):
    """Scratch memory of one call, from torch's caching allocator on the current stream (``None`` where none is needed)."""
    import torch

    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def _linear_args(A, C, bias, act, residual, pre, bias_shape, M, N):
    import torch

    dtype, device = A.dtype, A.get_device()
    c_ptr = _operand("C", C, (dtype, torch.float32), (M, N), device)
    if c_ptr is None:
        raise TypeError("C must be a CUDA tensor")
    return c_ptr, _native.LinearArgs(
        _type_code(dtype), _type_code(C.dtype), _act_code(act),
        None if bias is None else _operand("bias", bias, (dtype,), bias_shape, device),
        None if residual is None else _operand("residual", residual, (C.dtype,), (M, N), device),
        None if pre is None else _operand("pre", pre, (C.dtype,), (M, N), device))


def hgemm_linear(A, B, C, bias=None, act: str = "none", residual=None, pre=None):
    """``C = act(A @ B.T + bias) + residual`` in one kernel (C ABI ``b200_hgemm_linear``).

    ``A [M, K]``, ``B [N, K]`` and ``bias [N]`` are float16 or bfloat16 (all of one type), ``C``, ``residual`` and ``pre``
    ``[M, N]`` of that type or float32. ``act`` is one of ``ACTIVATIONS``. ``pre`` receives ``A @ B.T + bias``, which
    :func:`hgemm_linear_backward` needs; ``residual`` may be ``C`` itself. ``K`` is a multiple of 8; ``M`` may be 0."""
    M, N, K, _, _ = _rows_and_weights(A, B, None)
    c_ptr, args = _linear_args(A, C, bias, act, residual, pre, (N,), M, N)
    lib, ref = _native.load(), ctypes.byref(args)
    with _on_device(A):
        stream = _stream_of(A)
        status = lib.b200_hgemm_linear(A.data_ptr(), B.data_ptr(), c_ptr, M, N, K, ref, None, 0, stream)
        if status == _native.ERR_WORKSPACE:  # few shapes need any (k cut into more ranges than a cluster holds)
            nbytes = lib.b200_hgemm_linear_workspace_bytes(M, N, K, ref)
            ws = _scratch(nbytes, A.device)
            status = lib.b200_hgemm_linear(A.data_ptr(), B.data_ptr(), c_ptr, M, N, K, ref, ws.data_ptr(), nbytes, stream)
        check(status)
    return C


def hgemm_grouped(A, B, C, offsets, bias=None, act: str = "none", pre=None):
    """Rows ``offsets[g] : offsets[g + 1]`` of ``C = act(those rows of A @ B[g].T + bias[g])``, for every group in one
    launch (C ABI ``b200_hgemm_grouped``).

    ``A [M, K]``, ``B [G, N, K]`` (dense matrices, any distance between them that is a multiple of 8 elements) and
    ``bias [G, N]`` are float16 or bfloat16, ``C`` and ``pre`` ``[M, N]`` of that type or float32. ``offsets`` are ``G + 1``
    ascending int32 values on the device, read there by the kernel: the host never needs the group sizes. Groups may
    be empty; rows outside ``offsets[0] : offsets[G]`` are not written. ``K`` is a multiple of 8, ``G`` at most 1024."""
    if offsets is None:
        raise TypeError("offsets must be a contiguous int32 CUDA tensor")
    M, N, K, G, stride = _rows_and_weights(A, B, offsets)
    c_ptr, args = _linear_args(A, C, bias, act, None, pre, (G, N), M, N)
    with _on_device(A):
        check(_native.load().b200_hgemm_grouped(A.data_ptr(), B.data_ptr(), c_ptr, offsets.data_ptr(), M, N, K, G, stride,
                                                ctypes.byref(args), _stream_of(A)))
    return C


def _backward(dC, A, B, offsets, act, pre, dA, dB, dbias, dZ, accumulate):
    import torch

    M, N, K, G, stride = _rows_and_weights(A, B, offsets)
    dtype, device = A.dtype, A.get_device()
    if dC is None:
        raise TypeError("dC must be a CUDA tensor")
    dc_ptr = _operand("dC", dC, (dtype, torch.float32), (M, N), device)
    stack = (G,) if offsets is not None else ()
    code = _act_code(act)
    if code != _native.ACT_NONE and pre is None:
        raise ValueError("the gradient of an activation needs pre, the value before it")
    if dA is None and dB is None and dbias is None and dZ is None:
        raise ValueError("none of dA, dB, dbias and dZ was asked for")
    grads = _native.LinearGrads(
        _type_code(dtype), _type_code(dC.dtype), code, _type_code(dtype if dB is None else getattr(dB, "dtype", None)) or 0,
        1 if accumulate else 0, dc_ptr, _operand("pre", pre, (dC.dtype,), (M, N), device),
        _operand("dZ", dZ, (dtype,), (M, N), device), _operand("dA", dA, (dtype,), (M, K), device),
        _operand("dB", dB, (dtype, torch.float32), stack + (N, K), device),
        _operand("dbias", dbias, (torch.float32,), stack + (N,), device))
    lib = _native.load()
    with _on_device(A):
        nbytes = lib.b200_hgemm_backward_workspace_bytes(M, N, K, G, ctypes.byref(grads))
        ws = _scratch(nbytes, A.device)
        ws_ptr = ws.data_ptr() if ws is not None else None
        if offsets is None:
            check(lib.b200_hgemm_linear_backward(A.data_ptr(), B.data_ptr(), M, N, K, ctypes.byref(grads), ws_ptr, nbytes,
                                                 _stream_of(A)))
        else:
            check(lib.b200_hgemm_grouped_backward(A.data_ptr(), B.data_ptr(), offsets.data_ptr(), M, N, K, G, stride,
                                                  ctypes.byref(grads), ws_ptr, nbytes, _stream_of(A)))


def hgemm_linear_backward(dC, A, B, act: str = "none", pre=None, dA=None, dB=None, dbias=None, dZ=None, accumulate: bool = False):
    """The gradients of :func:`hgemm_linear` that are asked for (C ABI ``b200_hgemm_linear_backward``): with
    ``dZ = dC * act'(pre)``, ``dA = dZ @ B``, ``dB = dZ.T @ A`` and ``dbias`` the column sums of ``dZ``.

    ``dC`` and ``pre`` ``[M, N]`` have the forward pass's C type; ``dA [M, K]`` and ``dZ [M, N]`` the inputs' type, ``dB [N, K]``
    that type or float32, ``dbias [N]`` float32 (summed before ``dZ`` is rounded). Both products read ``dZ`` rounded to
    the inputs' type, so each term of a float32 ``dB`` behind an activation carries that rounding. With ``accumulate``
    the new ``dB`` (float32 then) and ``dbias`` are added to what the tensors hold. The gradient of the residual is
    ``dC``. ``N`` and ``K`` are multiples of 8; ``M`` may be 0. Returns ``(dA, dB, dbias)``."""
    _backward(dC, A, B, None, act, pre, dA, dB, dbias, dZ, accumulate)
    return dA, dB, dbias


def hgemm_grouped_backward(dC, A, B, offsets, act: str = "none", pre=None, dA=None, dB=None, dbias=None, dZ=None,
                           accumulate: bool = False):
    """The gradients of :func:`hgemm_grouped` (C ABI ``b200_hgemm_grouped_backward``), as
    :func:`hgemm_linear_backward` group by group: ``dB [G, N, K]``, ``dbias [G, N]``. A group without rows gets zeros; rows of
    ``dA`` and ``dZ`` outside every group are not written."""
    if offsets is None:
        raise TypeError("offsets must be a contiguous int32 CUDA tensor")
    _backward(dC, A, B, offsets, act, pre, dA, dB, dbias, dZ, accumulate)
    return dA, dB, dbias


def hgemm_host(A_host, B_host, C_host):
    """HOST tensors in, HOST tensor out (C ABI ``b200_hgemm_host``): uploads, multiplies, downloads, synchronises."""
    import torch

    for name, t in (("A", A_host), ("B", B_host), ("C", C_host)):
        if not isinstance(t, torch.Tensor) or t.dtype != torch.float16 or t.is_cuda or not t.is_contiguous():
            raise TypeError(f"{name} must be a contiguous float16 CPU tensor")
    M, K = A_host.shape
    N, Kb = B_host.shape
    if Kb != K or tuple(C_host.shape) != (M, N):
        raise ValueError("shape mismatch")
    check(_native.load().b200_hgemm_host(A_host.data_ptr(), B_host.data_ptr(), C_host.data_ptr(), int(M), int(N), int(K)))
    return C_host


def hgemm_host_a(A_host, B_dev, C_host, upload_after=None, gemm_after=None):
    """HOST ``A`` in, HOST ``C`` out, ``B`` already on the GPU (C ABI ``b200_hgemm_host_a``); the current stream's
    work on ``B_dev`` must be complete (this call synchronises that stream first). With ``upload_after`` /
    ``gemm_after`` (``torch.cuda.Event`` objects already recorded; C ABI ``b200_hgemm_host_a_after``) nothing is
    synchronised up front: A's uploads start behind the first event and the multiplies behind the second."""
    import torch

    for name, t in (("A", A_host), ("C", C_host)):
        if not isinstance(t, torch.Tensor) or t.dtype != torch.float16 or t.is_cuda or not t.is_contiguous():
            raise TypeError(f"{name} must be a contiguous float16 CPU tensor")
    if not B_dev.is_cuda or B_dev.dtype != torch.float16 or not B_dev.is_contiguous():
        raise TypeError("B must be a contiguous float16 CUDA tensor")
    M, K = A_host.shape
    N, Kb = B_dev.shape
    if Kb != K or tuple(C_host.shape) != (M, N):
        raise ValueError("shape mismatch")
    with torch.cuda.device(B_dev.device):
        if upload_after is None and gemm_after is None:
            torch.cuda.current_stream().synchronize()
            check(_native.load().b200_hgemm_host_a(A_host.data_ptr(), B_dev.data_ptr(), C_host.data_ptr(), int(M), int(N), int(K)))
        else:
            check(_native.load().b200_hgemm_host_a_after(
                A_host.data_ptr(), B_dev.data_ptr(), C_host.data_ptr(), int(M), int(N), int(K),
                upload_after.cuda_event if upload_after is not None else None,
                gemm_after.cuda_event if gemm_after is not None else None))
    return C_host


def select_plan(M: int, N: int, K: int) -> Plan:
    """The plan ``b200Hgemm`` would run for this shape on the current device (C ABI ``b200_hgemm_select``)."""
    plan = Plan()
    check(_native.load().b200_hgemm_select(M, N, K, ctypes.byref(plan)))
    return plan


def select_plan_untuned(M: int, N: int, K: int) -> Plan:
    """The plan the dispatch rules give, ignoring the table of tuned plans."""
    plan = Plan()
    check(_native.load().b200_hgemm_select_untuned(M, N, K, ctypes.byref(plan)))
    return plan


def load_plan_table(path) -> int:
    """Replace the table of tuned plans with the file at ``path`` (``None``: no table); returns the entry count."""
    n = _native.load().b200_hgemm_load_plan_table(None if path is None else str(path).encode())
    if n < 0:
        check(n)
    return n


def workspace_bytes(M: int, N: int, K: int, plan: Plan) -> int:
    return int(_native.load().b200_hgemm_workspace_bytes(M, N, K, ctypes.byref(plan)))


def last_device_error() -> int:
    return int(_native.load().b200_hgemm_last_device_error())


def enable_multicast(on: bool = True) -> bool:
    """Switch the single-GPU kernels with multicast operand loads on or off (C ABI
    ``b200_hgemm_enable_multicast``). Returns whether they are on afterwards: never in a process that is
    one rank of several or that holds a multi-device handle, and never without the companion library."""
    lib = _native.load()
    lib.b200_hgemm_enable_multicast(1 if on else 0)
    return lib.b200_hgemm_multicast_state() == _native.MULTICAST_ON


def synchronize(device=None) -> None:
    """Wait for torch's current stream and raise if a kernel on it gave up on a bounded wait
    (C ABI ``b200_hgemm_synchronize``)."""
    import torch

    with torch.cuda.device(device):
        check(_native.load().b200_hgemm_synchronize(int(torch.cuda.current_stream().cuda_stream)))


def launch_count() -> int:
    return int(_native.load().b200_hgemm_launch_count())
