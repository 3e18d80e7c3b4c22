"""Python entry points of the MI355X INT4 weight-only linear path.

Drop-in for the int4 part of the reference's ``kernelforge/ops.py``
(:171-214, :277-302): same function names, signatures, defaults, validation
order, exception types and messages, and the same
``torch.library.custom_op("kernelforge::int4_matmul")`` with a fake impl.
Underneath, every op calls the C ABI of ``libkf_int4.so`` (gfx950 HIP
kernels) on torch's current HIP stream; outputs and split-K workspaces come
from torch's caching allocator, so the ops are hipGraph-capturable.

Inference only: no backward formulas are registered.
"""

from __future__ import annotations

import contextlib
import ctypes
import math
from typing import NamedTuple, Optional

import torch
from torch.autograd import forward_ad
from torch._subclasses.fake_tensor import FakeTensor

from kernelforge import _lib

# Largest M that goes to the GEMV; above it int4_gemm runs the streaming MFMA kernel for small and
# medium M, then the LDS-DMA tiles.  The reference's rule (bench/sweep_int4_dispatch.py:51-57: the
# largest M at which the sum of GEMV times over the layer shapes beats the GEMM's) gives 3 on one MI355X
# (dispatch_sweep.py beside bench.py; GEMV / GEMM over 8 shapes, us: M = 3 32.2 / 35.3, M = 4 36.3 / 35.8,
# M = 5 43.7 / 36.5).  M = 4 stays on the GEMV all the same: the sums are 1.4% apart, and the GEMV
# multiplies by the exact q s where the GEMM's matrix cores take fp16(q s).
GEMV_MAX_M = 4
# The reference's int4_matmul sends M <= 7 to its GEMV, which accepts every N, and M >= 8
# to its GEMM, which rejects N % 64 != 0 (kernelforge/ops.py:193,204-214).  Our MFMA kernels
# need N % 64 == 0 as well, so between GEMV_MAX_M and 7 a shape the GEMM cannot take stays
# on the GEMV: int4_matmul accepts exactly what the reference's accepts and raises the same
# ValueError for the rest.
_GEMV_LIMIT_M = 7


def _use_gemv(m: int, n: int) -> bool:
    return m <= GEMV_MAX_M or (m <= _GEMV_LIMIT_M and n % 64 != 0)


def _stream_ptr(device: torch.device) -> int:
    """The raw handle of torch's current HIP stream on `device`."""
    return torch._C._cuda_getCurrentRawStream(device.index if device.index is not None else torch.cuda.current_device())


def _ptr(t: torch.Tensor) -> int:
    return t.data_ptr()


_PLAIN = (torch.Tensor, torch.nn.Parameter)


def _traced(tensors) -> bool:
    """True when a tracer must see the registered op instead of a kernel launch: torch is
    compiling, a TorchDispatchMode is active (FakeTensorMode, make_fx's proxy mode, ...), or an
    input is a tensor subclass (a FakeTensor made outside its mode, a functional tensor, ...).
    Eager calls on plain tensors return False and skip the op dispatcher."""
    if torch.compiler.is_compiling() or torch._C._len_torch_dispatch_stack() > 0:
        return True
    return any(t is not None and type(t) not in _PLAIN for t in tensors)


def _transformed() -> bool:
    """True inside a functorch transform (vmap, jvp, grad, functionalize), a forward-mode level or
    torch.jit.trace: a kernel launched on the tensors' memory would drop the tangent, the batch
    dimension or the record of the operation, where torch's own operations keep them."""
    return (torch._C._functorch.maybe_current_level() is not None or forward_ad._current_level >= 0
            or torch._C._get_tracing_state() is not None)


def _on(device: torch.device):
    """Makes `device` current for the launch; a no-op context when it already is (the common
    case, which then costs no device switch)."""
    if device.index is None or device.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(device)


def _eager_shape(x, packed, scales, group_size) -> tuple[int, int, int, int] | None:
    """(M, N, K, device index) of a call on a 2-D x that every check below accepts as it is: plain contiguous
    tensors of the right types and shapes on the current device, no tracer looking, a kernel for this M and N.
    None for anything else, which then takes the checked path step by step (same results, and the
    errors in their order).  One pass over the attributes: the checks one function at a time, the two
    reshapes and the device context cost 4 of an eager call's 11.5 us of host time (12.3 -> 7 us above the
    GEMV's M, with the plan kept per thread)."""
    if (torch.compiler.is_compiling() or torch._C._len_torch_dispatch_stack() > 0 or type(x) not in _PLAIN
            or type(packed) not in _PLAIN or type(scales) not in _PLAIN or packed.dim() != 2):
        return None
    m, k = x.shape
    n, words = packed.shape
    index = x.get_device()
    if (index < 0 or index != torch._C._cuda_getDevice() or packed.get_device() != index
            or scales.get_device() != index or x.dtype != torch.float16 or packed.dtype != torch.int32
            or scales.dtype != torch.float16 or words * 8 != k or not (group_size == 64 or group_size == 128)
            or k % group_size or scales.shape != (n, k // group_size) or not x.is_contiguous()
            or not packed.is_contiguous() or not scales.is_contiguous() or m < 1 or not x.is_cuda
            or (m > GEMV_MAX_M and n % 64 and m > _GEMV_LIMIT_M) or (x.data_ptr() | packed.data_ptr()) & 15):
        return None
    return m, n, k, index


def _check_int4(x: torch.Tensor, packed: torch.Tensor, scales: torch.Tensor, group_size: int) -> None:
    """Reference kernelforge/ops.py:171-182 (same order, types and messages)."""
    if not isinstance(x, torch.Tensor) or not x.is_cuda or x.dtype != torch.float16 or x.dim() != 2:
        raise TypeError("x must be a 2-D fp16 CUDA tensor [M, K]")
    if not x.is_contiguous():
        raise ValueError("x must be contiguous")
    if packed.dtype != torch.int32 or scales.dtype != torch.float16:
        raise TypeError("packed must be int32 and scales fp16 (see kernelforge.quantize)")
    k = x.shape[1]
    if k % group_size != 0:
        raise ValueError(f"K={k} is not a multiple of group_size={group_size}")
    if packed.shape[1] * 8 != k:
        raise ValueError(f"packed has K/8={packed.shape[1]} columns but x has K={k}")


def _check_native(x: torch.Tensor, packed: torch.Tensor, scales: torch.Tensor, group_size: int) -> None:
    """Tensor checks the reference makes in C++ (csrc/gemm/dequant_gemv.cu:5-19); RuntimeError like TORCH_CHECK.

    Valid inputs pass one combined test (a few microseconds less host time per problem); anything
    else goes through the checks one by one, which raise in the reference's order."""
    dev = x.get_device()
    if (type(x) in _PLAIN and type(packed) in _PLAIN and type(scales) in _PLAIN
            and x.is_cuda and packed.is_cuda and scales.is_cuda and x.is_contiguous() and packed.is_contiguous()
            and scales.is_contiguous() and packed.get_device() == dev and scales.get_device() == dev
            and packed.dim() == 2 and scales.dim() == 2 and (group_size == 64 or group_size == 128)
            and scales.shape[0] == packed.shape[0] and scales.shape[1] == x.shape[1] // group_size
            and not (x.data_ptr() | packed.data_ptr()) & 15):
        return
    _check_native_each(x, packed, scales, group_size)


def _check_native_each(x: torch.Tensor, packed: torch.Tensor, scales: torch.Tensor, group_size: int) -> None:
    """_check_native's conditions one at a time, raising the first that fails."""
    for name, t in (("x", x), ("packed", packed), ("scales", scales)):
        if isinstance(t, FakeTensor) or t.is_meta:
            raise RuntimeError(f"{name} has no device memory (a fake or meta tensor): trace through int4_linear / "
                               "kernelforge::int4_matmul, whose fake impl gives the output shape")
        if not t.is_cuda:
            raise RuntimeError(f"{name} must be a CUDA tensor")
        if not t.is_contiguous():
            raise RuntimeError(f"{name} must be contiguous")
        if t.device != x.device:
            raise RuntimeError(f"{name} is on {t.device} but x is on {x.device}")
    if packed.dim() != 2:
        raise RuntimeError("packed must be int32 [N, K / 8]")
    if scales.dim() != 2:
        raise RuntimeError("scales must be fp16 [N, K / group]")
    if group_size not in (64, 128):
        raise RuntimeError(f"group size must be 64 or 128, got {group_size}")
    k, n = x.shape[1], packed.shape[0]
    if scales.shape[0] != n or scales.shape[1] != k // group_size:
        raise RuntimeError("scales must be [N, K / group]")
    if x.data_ptr() % 16 or packed.data_ptr() % 16:
        raise RuntimeError("INT4 kernels need 16-byte aligned inputs")


def int4_gemv(x: torch.Tensor, packed: torch.Tensor, scales: torch.Tensor, group_size: int = 128) -> torch.Tensor:
    """Fused INT4 dequant GEMV for M in [1, 8]: x [M, K] fp16 @ W_hat^T -> [M, N] fp16.

    Reference kernelforge/ops.py:185-190; kernel csrc/kf_gemv.hip.
    """
    _check_int4(x, packed, scales, group_size)
    if not 1 <= x.shape[0] <= 8:
        raise ValueError(f"int4_gemv handles M in [1, 8], got M={x.shape[0]}")
    _check_native(x, packed, scales, group_size)
    return _launch_gemv(x, packed, scales, int(group_size))


def _launch_gemv(x: torch.Tensor, packed: torch.Tensor, scales: torch.Tensor, group_size: int) -> torch.Tensor:
    """kf_int4_gemv on validated inputs."""
    lib = _lib.load()
    m, k = x.shape
    n = packed.shape[0]
    dev = x.device
    y = torch.empty(m, n, dtype=torch.float16, device=dev)
    with _on(dev):
        status = lib.kf_int4_gemv(x.data_ptr(), packed.data_ptr(), scales.data_ptr(), y.data_ptr(), m, n, k,
                                  group_size, _stream_ptr(dev))
    _lib.check(status, "int4_gemv")
    return y


# The MFMA-16 block copy of a weight (kf_int4_reorder_mfma16): the weight in MFMA fragment order, a
# second copy in device memory.  No kernel reads it: the streaming kernels take the public layout through
# LDS in whole lines, faster than fragment-order loads of the copy were (see csrc/kf_stream.hip).  The
# layout's entry points stay for programs that hold such copies; MFMA16_CACHE and prepare_mfma16 are
# accepted and change neither memory nor route.
MFMA16_CACHE = False


def _mfma16_sizes(packed: torch.Tensor, scales: torch.Tensor, group_size: int) -> tuple[int, int]:
    """Bytes of the copy's packed words and scales, for a weight that it can be made of."""
    if packed.dtype != torch.int32 or scales.dtype != torch.float16 or not packed.is_cuda:
        raise TypeError("int4_reorder_mfma16 expects int32 packed and fp16 scales on a CUDA device")
    if not packed.is_contiguous() or not scales.is_contiguous():
        raise ValueError("packed and scales must be contiguous")
    pb, sb = ctypes.c_size_t(), ctypes.c_size_t()
    _lib.check(_lib.load().kf_int4_mfma16_sizes(packed.shape[0], packed.shape[1] * 8, int(group_size), ctypes.byref(pb),
                                                ctypes.byref(sb)), "mfma16 sizes")
    return pb.value, sb.value


def int4_reorder_mfma16(packed: torch.Tensor, scales: torch.Tensor,
                        group_size: int = 128) -> tuple[torch.Tensor, torch.Tensor]:
    """The MFMA-16 block copy (packed_r int32, scales_r fp16) of a packed weight; K % 128 == 0.

    An internal layout (the public packed format is unchanged); kernel csrc/kf_aux.hip.
    """
    packed_bytes, scales_bytes = _mfma16_sizes(packed, scales, group_size)
    n, k = packed.shape[0], packed.shape[1] * 8
    lib = _lib.load()
    packed_r = torch.empty(packed_bytes // 4, dtype=torch.int32, device=packed.device)
    scales_r = torch.empty(scales_bytes // 2, dtype=torch.float16, device=packed.device)
    with _on(packed.device):
        _lib.check(lib.kf_int4_reorder_mfma16(_ptr(packed), _ptr(scales), _ptr(packed_r), _ptr(scales_r), n, k,
                                              int(group_size), _stream_ptr(packed.device)), "int4_reorder_mfma16")
    return packed_r, scales_r


def prepare_mfma16(packed: torch.Tensor, scales: torch.Tensor, group_size: int = 128) -> None:
    """Checks that the MFMA-16 copy of a weight could be made; nothing is built or kept, as no kernel reads
    the copy (see MFMA16_CACHE)."""
    _mfma16_sizes(packed, scales, group_size)


def int4_gemm(x: torch.Tensor, packed: torch.Tensor, scales: torch.Tensor, group_size: int = 128) -> torch.Tensor:
    """Fused INT4 dequant GEMM on the MFMA matrix cores, any M, N a multiple of 64.

    Reference kernelforge/ops.py:196-201; kernels csrc/kf_stream.hip, csrc/kf_gemm.hip.
    """
    _check_int4(x, packed, scales, group_size)
    if packed.shape[0] % 64 != 0:
        raise ValueError(f"int4_gemm needs N to be a multiple of 64, got N={packed.shape[0]}")
    _check_native(x, packed, scales, group_size)
    if x.shape[0] < 1:  # csrc/gemm/dequant_gemm_tc.cu:14 (its TORCH_CHECK text)
        raise RuntimeError(f"bad M {x.shape[0]}")
    return _launch_gemm(x, packed, scales, int(group_size))


def _launch_gemm(x: torch.Tensor, packed: torch.Tensor, scales: torch.Tensor, group_size: int) -> torch.Tensor:
    """kf_int4_gemm on validated inputs."""
    lib = _lib.load()
    m, k = x.shape
    n = packed.shape[0]
    dev = x.device
    y = torch.empty(m, n, dtype=torch.float16, device=dev)
    with _on(dev):
        ws_bytes = lib.kf_int4_gemm_workspace_bytes(m, n, k, group_size)
        ws = torch.empty((ws_bytes + 3) // 4, dtype=torch.float32, device=dev) if ws_bytes else None
        status = lib.kf_int4_gemm(_ptr(x), _ptr(packed), _ptr(scales), _ptr(y),
                                  _ptr(ws) if ws is not None else None, ws_bytes, m, n, k, group_size,
                                  _stream_ptr(dev))
    _lib.check(status, "int4_gemm")
    return y


def gemm_plan(m: int, n: int, k: int, group_size: int = 128, device: torch.device | None = None) -> dict:
    """The kernel int4_gemm runs for an [m, k] x [n, k]^T problem on `device` (default: current).

    Returns {"kernel": the configuration's index (the streaming tiles, then the LDS-DMA tiles),
    "num_kernels": configurations, "splits": split-K factor, "tile": (BM, BN)}.  Diagnostics; no reference
    counterpart.
    """
    lib = _lib.load()
    out = [ctypes.c_int() for _ in range(5)]
    with torch.cuda.device(device if device is not None else torch.cuda.current_device()):
        status = lib.kf_int4_gemm_plan(int(m), int(n), int(k), int(group_size), *[ctypes.byref(v) for v in out])
    _lib.check(status, "gemm_plan")
    kernel, num, splits, bm, bn = (v.value for v in out)
    return {"kernel": kernel, "num_kernels": num, "splits": splits, "tile": (bm, bn)}


def int4_matmul(x: torch.Tensor, packed: torch.Tensor, scales: torch.Tensor, group_size: int = 128) -> torch.Tensor:
    """y = x @ W_hat^T for INT4 weights from kernelforge.quantize, choosing the kernel by M.

    M <= GEMV_MAX_M: the bandwidth-bound GEMV; larger M: the MFMA GEMM (M <= 7 with N not
    a multiple of 64 stays on the GEMV, as in the reference).  Reference kernelforge/ops.py:204-214.
    """
    if _use_gemv(x.shape[0], packed.shape[0]):
        return int4_gemv(x, packed, scales, group_size)
    return int4_gemm(x, packed, scales, group_size)


def _matmul_checked(x: torch.Tensor, packed: torch.Tensor, scales: torch.Tensor, group_size: int) -> torch.Tensor:
    """int4_matmul after _check_int4 has passed (int4_linear's eager path): the remaining checks of
    int4_gemv / int4_gemm in their order, then the launch, without validating twice."""
    m, n = x.shape[0], packed.shape[0]
    if _use_gemv(m, n):
        if not 1 <= m <= 8:
            raise ValueError(f"int4_gemv handles M in [1, 8], got M={m}")
        _check_native(x, packed, scales, group_size)
        return _launch_gemv(x, packed, scales, group_size)
    if n % 64 != 0:
        raise ValueError(f"int4_gemm needs N to be a multiple of 64, got N={n}")
    _check_native(x, packed, scales, group_size)
    return _launch_gemm(x, packed, scales, group_size)


_QUANT_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}  # KF_DTYPE_* of the C ABI


def int4_quantize(weight: torch.Tensor, group_size: int = 128) -> tuple[torch.Tensor, torch.Tensor]:
    """(packed int32 [N, K/8], scales fp16 [N, K/G]) of a weight [N, K] on the GPU.

    The gfx950 quantize + pack kernel; bit-identical to ``kernelforge.quantize.quantize_weight``
    of the same weight on the CPU (the reference's quantize_int4 + pack_int4,
    kernelforge/quantize.py:61-105).  fp32, fp16 or bf16 weights with finite values.
    """
    if weight.dim() != 2:
        raise ValueError(f"weight must be 2-D [N, K], got shape {tuple(weight.shape)}")
    if group_size not in (64, 128):
        raise ValueError(f"group_size must be one of (64, 128), got {group_size}")
    n, k = weight.shape
    if k % group_size:
        raise ValueError(f"K={k} is not a multiple of group_size={group_size}. Pad K or pick another group size.")
    if not weight.is_cuda:
        raise TypeError("int4_quantize needs a CUDA tensor")
    code = _QUANT_DTYPES.get(weight.dtype)
    if code is None:
        raise TypeError(f"int4_quantize supports float32, float16 and bfloat16 weights, got {weight.dtype}")
    w = weight if weight.is_contiguous() else weight.contiguous()
    if w.data_ptr() % 16:
        w = w.clone()
    lib = _lib.load()
    dev = w.device
    packed = torch.empty((n, k // 8), dtype=torch.int32, device=dev)
    scales = torch.empty((n, k // group_size), dtype=torch.float16, device=dev)
    index = w.get_device()
    with contextlib.nullcontext() if index == torch._C._cuda_getDevice() else torch.cuda.device(index):
        status = lib.kf_int4_quantize(w.data_ptr(), code, packed.data_ptr(), scales.data_ptr(), n, k, int(group_size),
                                      torch._C._cuda_getCurrentRawStream(index))
    if status:
        _lib.check(status, "int4_quantize")
    return packed, scales


def int4_dequant_fp16(packed: torch.Tensor, scales: torch.Tensor, group_size: int = 128) -> torch.Tensor:
    """W_hat = fp16(q * s) [N, K] on the GPU, the exact operand the GEMM feeds to the matrix cores.

    Counterpart of the reference's ``quantize.dequantize(qw, torch.float16)``
    (kernelforge/quantize.py:108-113), exported for bit-exactness checks.
    """
    if packed.dtype != torch.int32 or scales.dtype != torch.float16:
        raise TypeError("packed must be int32 and scales fp16 (see kernelforge.quantize)")
    if not packed.is_cuda or not scales.is_cuda:
        raise TypeError("packed and scales must be CUDA tensors")
    if not packed.is_contiguous() or not scales.is_contiguous():
        raise ValueError("packed and scales must be contiguous")
    n, k = packed.shape[0], packed.shape[1] * 8
    if scales.shape != (n, k // group_size):
        raise ValueError("scales must be [N, K / group]")
    lib = _lib.load()
    w_hat = torch.empty(n, k, dtype=torch.float16, device=packed.device)
    with _on(packed.device):
        status = lib.kf_int4_dequant_fp16(_ptr(packed), _ptr(scales), _ptr(w_hat), n, k, int(group_size),
                                          _stream_ptr(packed.device))
    _lib.check(status, "int4_dequant_fp16")
    return w_hat


def int4_gemv_grouped(xs: list[torch.Tensor], packed: list[torch.Tensor], scales: list[torch.Tensor],
                      group_size: int = 128, *, _checked: bool = False) -> list[torch.Tensor]:
    """Several independent INT4 GEMVs (common M in [1, 8]) in one kernel launch per 8 problems.

    Each output equals ``int4_gemv(xs[i], packed[i], scales[i], group_size)`` bit for bit.
    This is the multi-problem launch of the GEMV (no reference counterpart as
    an entry point): on MI355X a launch's fixed cost exceeds the time to stream
    a small decode linear, so independent linears (q|k|v, gate|up, or separate
    layers) should share a launch.  Kernel: csrc/kf_gemv.hip.
    """
    if not (len(xs) == len(packed) == len(scales)) or not xs:
        raise ValueError("xs, packed and scales must be non-empty lists of equal length")
    m = xs[0].shape[0] if isinstance(xs[0], torch.Tensor) and xs[0].dim() == 2 else -1
    for x, p, s in zip(xs, packed, scales):
        if not _checked:
            _check_int4(x, p, s, group_size)
        if x.shape[0] != m:
            raise ValueError(f"all problems must share M, got {x.shape[0]} and {m}")
        if x.device != xs[0].device:
            raise RuntimeError("all problems must be on one device")
        _check_native(x, p, s, group_size)
    if not 1 <= m <= 8:
        raise ValueError(f"int4_gemv handles M in [1, 8], got M={m}")
    lib = _lib.load()
    dev = xs[0].device
    # One tensor per output: the registered grouped op may not return outputs that alias each other.
    ns = [p.shape[0] for p in packed]
    ys = [torch.empty(m, n, dtype=torch.float16, device=dev) for n in ns]
    problem = _lib.GemvProblem
    with _on(dev):
        stream = _stream_ptr(dev)
        for b0 in range(0, len(xs), _lib.GEMV_MAX_GROUP):
            b1 = min(b0 + _lib.GEMV_MAX_GROUP, len(xs))
            probs = (problem * (b1 - b0))(*[problem(xs[i].data_ptr(), packed[i].data_ptr(), scales[i].data_ptr(),
                                                    ys[i].data_ptr(), ns[i], xs[i].shape[1]) for i in range(b0, b1)])
            status = lib.kf_int4_gemv_grouped(probs, b1 - b0, m, int(group_size), stream)
            _lib.check(status, "int4_gemv_grouped")
    return ys


@torch.library.custom_op("kernelforge::int4_matmul", mutates_args=())
def _int4_matmul_op(x: torch.Tensor, packed: torch.Tensor, scales: torch.Tensor, group_size: int) -> torch.Tensor:
    return int4_matmul(x, packed, scales, group_size)


@_int4_matmul_op.register_fake
def _(x, packed, scales, group_size):
    return x.new_empty(x.shape[0], packed.shape[0])


def _matmul_grouped(xs: list[torch.Tensor], packed: list[torch.Tensor], scales: list[torch.Tensor],
                    group_size: int, checked: bool = False) -> list[torch.Tensor]:
    """checked: _check_int4 has passed on every problem (int4_linear_grouped's eager path)."""
    if all(_use_gemv(x.shape[0], p.shape[0]) for x, p in zip(xs, packed)):
        return int4_gemv_grouped(xs, packed, scales, group_size, _checked=checked)
    if _groupable(xs, packed):
        return _launch_gemm_grouped(xs, packed, scales, group_size, checked)
    if xs[0].shape[0] <= _GEMV_LIMIT_M:
        return [int4_matmul(x, p, s, group_size) for x, p, s in zip(xs, packed, scales)]
    return [int4_gemm(x, p, s, group_size) for x, p, s in zip(xs, packed, scales)]


def _groupable(xs: list[torch.Tensor], packed: list[torch.Tensor]) -> bool:
    """Whether these problems go to kf_int4_gemm_grouped: one M above the GEMV's, one device, every N
    a multiple of 64."""
    m, dev = xs[0].shape[0], xs[0].device
    return (m > GEMV_MAX_M and len(xs) > 1 and
            all(x.shape[0] == m and x.device == dev and p.shape[0] % 64 == 0 for x, p in zip(xs, packed)))


def _launch_gemm_grouped(xs: list[torch.Tensor], packed: list[torch.Tensor], scales: list[torch.Tensor],
                         group_size: int, checked: bool) -> list[torch.Tensor]:
    """int4_gemm of every problem through kf_int4_gemm_grouped, KF_GEMV_MAX_GROUP problems per call."""
    for x, p, s in zip(xs, packed, scales):
        if not checked:
            _check_int4(x, p, s, group_size)
        _check_native(x, p, s, group_size)
    lib = _lib.load()
    dev, m, group_size = xs[0].device, xs[0].shape[0], int(group_size)
    ys = [torch.empty(m, p.shape[0], dtype=torch.float16, device=dev) for p in packed]
    with _on(dev):
        stream = _stream_ptr(dev)
        for b0 in range(0, len(xs), _lib.GEMV_MAX_GROUP):
            part = range(b0, min(b0 + _lib.GEMV_MAX_GROUP, len(xs)))
            probs = (_lib.GemvProblem * len(part))(*[
                _lib.GemvProblem(xs[i].data_ptr(), packed[i].data_ptr(), scales[i].data_ptr(), ys[i].data_ptr(),
                                 packed[i].shape[0], xs[i].shape[1]) for i in part])
            ws_bytes = lib.kf_int4_gemm_grouped_workspace_bytes(probs, len(part), m, group_size)
            ws = torch.empty((ws_bytes + 3) // 4, dtype=torch.float32, device=dev) if ws_bytes else None
            status = lib.kf_int4_gemm_grouped(probs, len(part), m, group_size, _ptr(ws) if ws is not None else None,
                                              ws_bytes, stream)
            _lib.check(status, "int4_gemm_grouped")
    return ys


@torch.library.custom_op("kernelforge::int4_matmul_grouped", mutates_args=())
def _int4_matmul_grouped_op(xs: list[torch.Tensor], packed: list[torch.Tensor], scales: list[torch.Tensor],
                            group_size: int) -> list[torch.Tensor]:
    return _matmul_grouped(xs, packed, scales, group_size)


@_int4_matmul_grouped_op.register_fake
def _(xs, packed, scales, group_size):
    return [x.new_empty(x.shape[0], p.shape[0]) for x, p in zip(xs, packed)]


def int4_linear_grouped(xs: list[torch.Tensor], packed: list[torch.Tensor], scales: list[torch.Tensor],
                        group_size: int = 128, biases: list[torch.Tensor | None] | None = None
                        ) -> list[torch.Tensor]:
    """``[int4_linear(xs[i], packed[i], scales[i], group_size, biases[i]) ...]`` with one GEMV launch
    for all problems at decode sizes (common flattened M <= GEMV_MAX_M) and as few GEMM launches as
    their plans allow above; results are bit-identical."""
    flat = []
    for x in xs:
        x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
        flat.append(x2 if x2.is_contiguous() else x2.contiguous())
    for x2, p, s in zip(flat, packed, scales):
        _check_int4(x2, p, s, group_size)
    if _traced([*flat, *packed, *scales]):
        ys = _int4_matmul_grouped_op(flat, list(packed), list(scales), int(group_size))
    else:  # eager: the op's implementation without the dispatcher (as in int4_linear), checked once
        ys = _matmul_grouped(flat, list(packed), list(scales), int(group_size), checked=True)
    out = []
    for i, y in enumerate(ys):
        b = biases[i] if biases is not None else None
        if b is not None:
            y = y + b
        out.append(y if xs[i].dim() == 2 else y.reshape(*xs[i].shape[:-1], packed[i].shape[0]))
    return out


def _launch(x: torch.Tensor, packed: torch.Tensor, scales: torch.Tensor, group_size: int, m: int, n: int, k: int,
            index: int) -> torch.Tensor:
    """int4_matmul of a call that _eager_shape accepted."""
    lib = _lib.load()
    if _use_gemv(m, n):
        y = x.new_empty((m, n))
        status = lib.kf_int4_gemv(x.data_ptr(), packed.data_ptr(), scales.data_ptr(), y.data_ptr(), m, n, k, group_size,
                                  torch._C._cuda_getCurrentRawStream(index))
        if status:
            _lib.check(status, "int4_gemv")
        return y
    y = x.new_empty((m, n))
    ws_bytes = lib.kf_int4_gemm_workspace_bytes(m, n, k, group_size)
    ws = x.new_empty((ws_bytes + 3) // 4, dtype=torch.float32) if ws_bytes else None
    status = lib.kf_int4_gemm(x.data_ptr(), packed.data_ptr(), scales.data_ptr(), y.data_ptr(),
                              ws.data_ptr() if ws is not None else None, ws_bytes, m, n, k, group_size,
                              torch._C._cuda_getCurrentRawStream(index))
    if status:
        _lib.check(status, "int4_gemm")
    return y


def int4_linear(x: torch.Tensor, packed: torch.Tensor, scales: torch.Tensor, group_size: int = 128,
                bias: torch.Tensor | None = None) -> torch.Tensor:
    """y = x @ W_hat^T (+ bias) for INT4 weights from kernelforge.quantize. x: [..., K] fp16.

    Leading dimensions are flattened into M like nn.Linear; the bias add is a
    separate fp16 add, as in the reference (kernelforge/ops.py:287-302).
    """
    shape = _eager_shape(x, packed, scales, group_size) if isinstance(x, torch.Tensor) and x.dim() == 2 else None
    if shape is not None:
        y = _launch(x, packed, scales, int(group_size), *shape)
        if bias is None:
            return y
        y = y + bias
        # A bias of more dimensions broadcasts the sum: back to the output's shape, or refused, as below.
        return y if y.dim() == 2 and y.numel() == shape[0] * shape[1] else y.reshape(shape[:2])
    lead = x.shape[:-1]
    x2 = x.reshape(-1, x.shape[-1])
    if not x2.is_contiguous():
        x2 = x2.contiguous()
    _check_int4(x2, packed, scales, group_size)
    # The registered op kernelforge::int4_matmul whenever torch compiles or any tracer or dispatch
    # mode is looking (torch.compile, FakeTensorMode, make_fx, ...), as the reference always calls
    # it; eager calls on plain tensors go straight to its implementation (same result), skipping
    # ~14 us of op dispatch.
    if _traced((x2, packed, scales)):
        y = _int4_matmul_op(x2, packed, scales, int(group_size))
    else:
        y = _matmul_checked(x2, packed, scales, int(group_size))
    if bias is not None:
        y = y + bias
    return y.reshape(*lead, packed.shape[0])


def int4_linear_fused(x: torch.Tensor, packed: torch.Tensor, scales: torch.Tensor, group_size: int = 128, *,
                      norm_weight: torch.Tensor | None = None, eps: float = 1e-5, up: torch.Tensor | None = None,
                      residual: torch.Tensor | None = None) -> torch.Tensor:
    """A decoder linear with the work around it: ``residual + int4_linear(prologue(x))``.

    prologue: with ``norm_weight``, RMSNorm ``x * rsqrt(mean(x^2) + eps) * norm_weight`` (fp32
    inside); with ``up``, SwiGLU ``silu(x) * up`` where x is the gate (the fp16 roundings of torch's
    ``silu(x) * up``); neither: x itself.  ``residual`` ([..., N] fp16), when given, is added to the
    fp16 result exactly as ``residual + y`` would be.

    At decode size (one row of x, K <= 10240) all of it is one GEMV launch
    (``kf_int4_gemv_fused``): the prologue runs on the workgroup's LDS copy of x and the residual
    joins the store, with the product bit-identical to ``int4_linear``'s.  Other sizes run the
    same steps as separate torch ops around ``int4_linear``.  No reference counterpart.
    """
    if norm_weight is not None and up is not None:
        raise ValueError("int4_linear_fused takes norm_weight or up, not both")
    lead = x.shape[:-1]
    k = x.shape[-1]
    n = packed.shape[0]
    x2 = x.reshape(-1, k)
    m = x2.shape[0]
    res2 = residual.reshape(-1, n) if residual is not None else None
    if res2 is not None and (res2.shape[0] != m or res2.dtype != torch.float16 or res2.device != x.device):
        raise ValueError(f"residual must be fp16 [..., {n}] on {x.device} with the leading dims of x")
    aux = norm_weight if norm_weight is not None else up
    if aux is not None and (aux.dtype != torch.float16 or aux.device != x.device):
        raise ValueError("norm_weight / up must be fp16 on the device of x")
    if up is not None and up.shape != x.shape:
        raise ValueError(f"up must have the shape of x, {tuple(x.shape)}, got {tuple(up.shape)}")
    if norm_weight is not None and norm_weight.shape != (k,):
        raise ValueError(f"norm_weight must be [{k}], got {tuple(norm_weight.shape)}")
    prologue = (_lib.KF_PROLOGUE_RMSNORM if norm_weight is not None
                else _lib.KF_PROLOGUE_SWIGLU if up is not None else _lib.KF_PROLOGUE_NONE)
    fused = (m == 1 and k <= _lib.KF_GEMV_FUSED_MAX_K and x.is_cuda and x2.is_contiguous()
             and (aux is None or aux.is_contiguous()) and (res2 is None or res2.is_contiguous()))
    if not fused:
        return _fused_composition(x2, packed, scales, group_size, prologue, aux, eps, res2).reshape(*lead, n)
    _check_int4(x2, packed, scales, group_size)
    if _traced((x2, packed, scales, aux, res2)):
        y = _int4_linear_fused_op(x2, packed, scales, int(group_size), prologue, aux, float(eps), res2)
    else:
        y = _launch_fused(x2, packed, scales, int(group_size), prologue, aux, float(eps), res2)
    return y.reshape(*lead, n)


def _fused_composition(x2: torch.Tensor, packed: torch.Tensor, scales: torch.Tensor, group_size: int, prologue: int,
                       aux: torch.Tensor | None, eps: float, res2: torch.Tensor | None) -> torch.Tensor:
    """int4_linear_fused's steps as separate torch ops around int4_linear (shapes the fused launch
    does not take); x2 [M, K] -> y [M, N]."""
    k = x2.shape[1]
    if prologue == _lib.KF_PROLOGUE_RMSNORM:
        x2 = torch.nn.functional.rms_norm(x2, (k,), aux, eps)
    elif prologue == _lib.KF_PROLOGUE_SWIGLU:
        x2 = torch.nn.functional.silu(x2) * aux.reshape(-1, k)
    y = int4_linear(x2, packed, scales, group_size)
    return y if res2 is None else res2 + y


def _launch_fused(x2: torch.Tensor, packed: torch.Tensor, scales: torch.Tensor, group_size: int, prologue: int,
                  aux: torch.Tensor | None, eps: float, res2: torch.Tensor | None) -> torch.Tensor:
    """kf_int4_gemv_fused on int4_linear_fused's validated one-row inputs; y [1, N].  x or the
    prologue operand off a 16-byte boundary (the launch's LDS copies need it) takes the
    composition instead, with the same result."""
    if x2.data_ptr() % 16 or (aux is not None and aux.data_ptr() % 16):
        return _fused_composition(x2, packed, scales, group_size, prologue, aux, eps, res2)
    _check_native(x2, packed, scales, group_size)
    lib = _lib.load()
    n, k = packed.shape[0], x2.shape[1]
    y = torch.empty(1, n, dtype=torch.float16, device=x2.device)
    with _on(x2.device):
        status = lib.kf_int4_gemv_fused(_ptr(x2), _ptr(packed), _ptr(scales), _ptr(y), 1, n, k, group_size,
                                        prologue, _ptr(aux) if aux is not None else None, eps,
                                        _ptr(res2) if res2 is not None else None, _stream_ptr(x2.device))
    _lib.check(status, "int4_gemv_fused")
    return y


@torch.library.custom_op("kernelforge::int4_linear_fused", mutates_args=())
def _int4_linear_fused_op(x: torch.Tensor, packed: torch.Tensor, scales: torch.Tensor, group_size: int,
                          prologue: int, aux: Optional[torch.Tensor], eps: float,
                          residual: Optional[torch.Tensor]) -> torch.Tensor:
    return _launch_fused(x, packed, scales, group_size, prologue, aux, eps, residual)


@_int4_linear_fused_op.register_fake
def _(x, packed, scales, group_size, prologue, aux, eps, residual):
    return x.new_empty(1, packed.shape[0])


def int4_qkv_rope_cache(x: torch.Tensor, packed: torch.Tensor, scales: torch.Tensor, group_size: int, *,
                        cos: torch.Tensor, sin: torch.Tensor, pos: torch.Tensor, cache_k: torch.Tensor,
                        cache_v: torch.Tensor, heads: int, kv_heads: int, head_dim: int,
                        norm_weight: torch.Tensor | None = None, eps: float = 1e-5) -> torch.Tensor:
    """The q|k|v projection of one decode token with RoPE and the KV-cache update in one launch.

    x: one row [..., K] fp16 (RMSNorm-ed first when ``norm_weight`` is given); packed / scales: the
    q|k|v weights concatenated along N = (heads + 2 kv_heads) head_dim; cos / sin: fp16
    [max_seq, head_dim] tables (sin with the rotate-half sign folded in: -sin on the first half);
    pos: int64 [1] on the device; cache_k: fp16 [kv_heads, head_dim, max_seq] (K transposed),
    cache_v: fp16 [kv_heads, max_seq, head_dim].  Returns y [..., N]: q and k rotated, v as is.
    k and v are also written at position pos of the caches; a pos outside [0, max_seq) writes no
    cache entry (and rotates with the tables' row 0).  Kernel: kf_int4_gemv_qkv_rope.
    No reference counterpart.
    """
    k = x.shape[-1]
    n = packed.shape[0]
    x2 = x.reshape(-1, k)
    if x2.shape[0] != 1:
        raise ValueError(f"int4_qkv_rope_cache takes one token, got {x2.shape[0]} rows")
    if (heads + 2 * kv_heads) * head_dim != n:
        raise ValueError(f"packed has N={n} rows, not (heads + 2 kv_heads) * head_dim")
    max_seq = cos.shape[0]
    for name, t, numel in (("cos", cos, max_seq * head_dim), ("sin", sin, max_seq * head_dim),
                           ("cache_k", cache_k, kv_heads * head_dim * max_seq),
                           ("cache_v", cache_v, kv_heads * max_seq * head_dim)):
        if t.dtype != torch.float16 or not t.is_contiguous() or t.numel() != numel or t.device != x.device:
            raise ValueError(f"{name} must be a contiguous fp16 tensor of {numel} elements on {x.device}")
    if pos.dtype != torch.int64 or pos.numel() != 1 or pos.device != x.device:
        raise ValueError("pos must be one int64 on the device of x")
    if norm_weight is not None and (norm_weight.dtype != torch.float16 or norm_weight.shape != (k,)
                                    or not norm_weight.is_contiguous()):
        raise ValueError(f"norm_weight must be a contiguous, 16-byte aligned fp16 [{k}]")
    x2 = x2.contiguous()
    _check_int4(x2, packed, scales, group_size)
    args = (x2, packed, scales, int(group_size), cos, sin, pos, cache_k, cache_v, int(heads), int(kv_heads),
            int(head_dim), norm_weight, float(eps))
    y = _int4_qkv_rope_cache_op(*args) if _traced((x2, packed, scales, cos, sin, pos, cache_k, cache_v,
                                                   norm_weight)) else _launch_qkv_rope(*args)
    return y.reshape(*x.shape[:-1], n)


def _launch_qkv_rope(x2, packed, scales, group_size, cos, sin, pos, cache_k, cache_v, heads, kv_heads, head_dim,
                     norm_weight, eps) -> torch.Tensor:
    """kf_int4_gemv_qkv_rope on int4_qkv_rope_cache's validated inputs; y [1, N]."""
    _check_native(x2, packed, scales, group_size)
    for name, t in (("cos", cos), ("sin", sin), ("pos", pos), ("cache_k", cache_k), ("cache_v", cache_v),
                    ("norm_weight", norm_weight)):
        if t is not None and (isinstance(t, FakeTensor) or t.is_meta):
            raise RuntimeError(f"{name} has no device memory (a fake or meta tensor)")
    if norm_weight is not None and norm_weight.data_ptr() % 16:
        raise ValueError(f"norm_weight must be a contiguous, 16-byte aligned fp16 [{x2.shape[1]}]")
    lib = _lib.load()
    n, k = packed.shape[0], x2.shape[1]
    y = torch.empty(1, n, dtype=torch.float16, device=x2.device)
    rc = _lib.RopeCache(_ptr(cos), _ptr(sin), _ptr(pos), _ptr(cache_k), _ptr(cache_v), heads, kv_heads, head_dim,
                        cos.shape[0])
    with _on(x2.device):
        status = lib.kf_int4_gemv_qkv_rope(_ptr(x2), _ptr(packed), _ptr(scales), _ptr(y), n, k, group_size,
                                           _ptr(norm_weight) if norm_weight is not None else None, eps,
                                           ctypes.byref(rc), _stream_ptr(x2.device))
    _lib.check(status, "int4_gemv_qkv_rope")
    return y


@torch.library.custom_op("kernelforge::int4_qkv_rope_cache", mutates_args=("cache_k", "cache_v"))
def _int4_qkv_rope_cache_op(x: torch.Tensor, packed: torch.Tensor, scales: torch.Tensor, group_size: int,
                            cos: torch.Tensor, sin: torch.Tensor, pos: torch.Tensor, cache_k: torch.Tensor,
                            cache_v: torch.Tensor, heads: int, kv_heads: int, head_dim: int,
                            norm_weight: Optional[torch.Tensor], eps: float) -> torch.Tensor:
    return _launch_qkv_rope(x, packed, scales, group_size, cos, sin, pos, cache_k, cache_v, heads, kv_heads,
                            head_dim, norm_weight, eps)


@_int4_qkv_rope_cache_op.register_fake
def _(x, packed, scales, group_size, cos, sin, pos, cache_k, cache_v, heads, kv_heads, head_dim, norm_weight, eps):
    return x.new_empty(1, packed.shape[0])



def decode_argmax_step(logits: torch.Tensor, token: torch.Tensor, pos: torch.Tensor, history: torch.Tensor,
                       mask: torch.Tensor | None = None) -> None:
    """The greedy step of a graph-captured decode loop in one launch (kf_decode_argmax_step).

    logits: fp16 [n] on the GPU; token, pos: int64 [1]; history: int64 [max_seq]; mask: None or
    fp16 with max_seq elements.  Computes idx = torch.argmax(logits) (same tie and NaN rules) and
    then, on the device: pos += 1; token = idx; history[pos] = idx and mask[pos] = 0 when pos <
    max_seq.  Asynchronous on the current stream; capturable.  No reference counterpart (the
    reference's decode loop does these steps as separate torch ops).
    """
    if logits.dtype != torch.float16 or logits.dim() != 1 or not logits.is_cuda or not logits.is_contiguous():
        raise TypeError("logits must be a contiguous 1-D fp16 CUDA tensor")
    for name, t in (("token", token), ("pos", pos)):
        if t.dtype != torch.int64 or t.numel() != 1 or t.device != logits.device:
            raise ValueError(f"{name} must be one int64 on {logits.device}")
    if history.dtype != torch.int64 or history.dim() != 1 or not history.is_contiguous() or \
            history.device != logits.device:
        raise ValueError(f"history must be a contiguous 1-D int64 tensor on {logits.device}")
    max_seq = history.numel()
    if mask is not None and (mask.dtype != torch.float16 or mask.numel() != max_seq or not mask.is_contiguous()
                             or mask.device != logits.device):
        raise ValueError(f"mask must be a contiguous fp16 tensor of {max_seq} elements on {logits.device}")
    if _traced((logits, token, pos, history, mask)):
        raise RuntimeError("decode_argmax_step updates device buffers in place and has no traceable form")
    lib = _lib.load()
    with _on(logits.device):
        status = lib.kf_decode_argmax_step(_ptr(logits), logits.numel(), _ptr(token), _ptr(pos), _ptr(history),
                                           max_seq, _ptr(mask) if mask is not None else None,
                                           _stream_ptr(logits.device))
    _lib.check(status, "decode_argmax_step")


# KF_ATTN_MAX_HEAD_DIM / KF_ATTN_MAX_SEQ of the C ABI.
_ATTN_MAX_HEAD_DIM, _ATTN_MAX_SEQ = 256, 8192


def decode_attention_fits(head_dim: int, max_seq: int) -> bool:
    """Whether decode_attention takes this head size and cache length."""
    return head_dim % 8 == 0 and 0 < head_dim <= _ATTN_MAX_HEAD_DIM and 0 < max_seq <= _ATTN_MAX_SEQ


def decode_attention_eager(q: torch.Tensor, cache_k: torch.Tensor, cache_v: torch.Tensor, mask: torch.Tensor) -> bool:
    """Whether these operands can go to decode_attention's launch: plain tensors outside any tracer or
    transform and not tracked by autograd, fp16 on q's device, caches contiguous and 16-byte aligned,
    mask rows contiguous."""
    tensors = (q, cache_k, cache_v, mask)
    if _traced(tensors) or _transformed() or (torch.is_grad_enabled() and any(t.requires_grad for t in tensors)):
        return False
    return (all(t.dtype == torch.float16 and t.device == q.device for t in tensors) and mask.stride(-1) == 1 and
            all(t.is_contiguous() and t.data_ptr() % 16 == 0 for t in (cache_k, cache_v)))


def decode_attention(q: torch.Tensor, cache_k: torch.Tensor, cache_v: torch.Tensor, mask: torch.Tensor, *,
                     kv_heads: int) -> torch.Tensor:
    """Attention of one decode token over the KV cache in one launch (kf_decode_attention).

    q fp16 [heads, d]; cache_k holds kv_heads x d x max_seq values (K transposed), cache_v kv_heads x
    max_seq x d, both contiguous; mask fp16 [heads, max_seq] additive, rows contiguous (an expanded
    row is fine).  Returns softmax(mask + q K / sqrt(d)) V, fp16 [heads, d], with fp32 scores and
    sums; query head h reads KV head h // (heads / kv_heads).  No reference counterpart (its decode
    loop runs torch's attention).
    """
    if q.dim() != 2 or mask.dim() != 2 or q.dtype != torch.float16 or not q.is_cuda:
        raise TypeError("q must be a 2-D fp16 CUDA tensor [heads, d] and mask [heads, max_seq]")
    heads, d = q.shape
    max_seq = mask.shape[1]
    if kv_heads < 1 or heads % kv_heads or mask.shape[0] != heads:
        raise ValueError(f"kv_heads={kv_heads} must divide heads={heads}, and mask must have {heads} rows")
    if not decode_attention_fits(d, max_seq):
        raise ValueError(f"decode_attention needs head_dim a multiple of 8 up to {_ATTN_MAX_HEAD_DIM} and max_seq up "
                         f"to {_ATTN_MAX_SEQ}, got {d} and {max_seq}")
    for name, t, numel in (("q", q, heads * d), ("cache_k", cache_k, kv_heads * d * max_seq),
                           ("cache_v", cache_v, kv_heads * max_seq * d)):
        if t.dtype != torch.float16 or not t.is_contiguous() or t.numel() != numel or t.device != q.device:
            raise ValueError(f"{name} must be a contiguous fp16 tensor of {numel} elements on {q.device}")
    if mask.dtype != torch.float16 or mask.device != q.device or (max_seq > 1 and mask.stride(1) != 1):
        raise ValueError(f"mask must be fp16 on {q.device} with contiguous rows")
    if _traced((q, cache_k, cache_v, mask)) or _transformed():
        raise RuntimeError("decode_attention launches a kernel; it cannot be traced or transformed")
    lib = _lib.load()
    out = torch.empty_like(q)
    with _on(q.device):
        status = lib.kf_decode_attention(_ptr(q), _ptr(cache_k), _ptr(cache_v), _ptr(mask), _ptr(out), q.shape[0],
                                         kv_heads, q.shape[1], mask.shape[1], mask.stride(0), _stream_ptr(q.device))
    _lib.check(status, "decode_attention")
    return out


# ---- several requests at once: a paged KV cache ---------------------------------------------------------
#
# cache_k, cache_v: fp16 or bf16 [num_pages, kv_heads, block_size, head_dim], the last dimension contiguous, block_size a
# power of two from 16 up.  block_table int32 [requests, width]: the pages of each request in order; token i of
# request r lies in slot block_table[r, i // block_size] * block_size + i % block_size.  One step of a server is
# paged_tables, the q|k|v projection, rope_paged_cache, paged_attention (or prompt_attention where the step
# is whole prompts only).  Inference only.

_HALF_TYPES = {torch.float16: 1, torch.bfloat16: 2}  # KF_DTYPE_F16, KF_DTYPE_BF16


class PagedStep(NamedTuple):
    """What paged_tables makes of a step's lengths."""

    cu_new: torch.Tensor      # int32 [requests + 1]: where each request's new tokens begin
    seq_lens: torch.Tensor    # int32 [requests]: tokens of each request, the new ones included
    positions: torch.Tensor   # int64 [max_tokens]: position of every new token in its request, -1 behind the last
    slots: torch.Tensor       # int64 [max_tokens]: its slot of the cache, -1 where it has none
    free_count: torch.Tensor  # int32 [1]: pages left on the stack


def _check_plain(what: str, tensors) -> None:
    """Refuses what a kernel launch would get wrong silently: transforms and gradients."""
    if _transformed():
        raise RuntimeError(f"{what} launches a kernel; it cannot be transformed")
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise RuntimeError(f"{what} is inference only; a tensor requires a gradient (use torch.no_grad())")


def _direct(index: int, tensors) -> bool:
    """Plain tensors on the current device `index`, seen by no tracer, transform or gradient: with right types and
    shapes their call goes straight to its launch.  One pass over the attributes, as in _eager_shape; anything else takes
    the checks one by one, which name what is wrong and take some microseconds more of host time."""
    if (index < 0 or torch.compiler.is_compiling() or torch._C._len_torch_dispatch_stack() > 0 or _transformed()
            or index != torch._C._cuda_getDevice()):
        return False
    grad = torch.is_grad_enabled()
    for t in tensors:
        if type(t) not in _PLAIN or t.get_device() != index or (grad and t.requires_grad):
            return False
    return True


def _check_memory(name: str, t: torch.Tensor, device: torch.device) -> None:
    if isinstance(t, FakeTensor) or t.is_meta:
        raise RuntimeError(f"{name} has no device memory (a fake or meta tensor)")
    if not t.is_cuda or t.device != device:
        raise RuntimeError(f"{name} must be on {device}, a CUDA device, got {t.device}")


def _check_int(name: str, t: torch.Tensor, dtype: torch.dtype, shape: tuple) -> None:
    if t.dtype != dtype or tuple(t.shape) != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {str(dtype)[6:]} tensor of shape {list(shape)}, got "
                         f"{str(t.dtype)[6:]} {list(t.shape)}")


def _check_table(block_table: torch.Tensor, requests: int) -> None:
    if (block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.shape[0] != requests
            or block_table.shape[1] < 1 or block_table.stride(1) != 1):
        raise ValueError(f"block_table must be int32 [{requests}, width] with contiguous rows, got "
                         f"{str(block_table.dtype)[6:]} {list(block_table.shape)}")


def _check_block_size(block_size: int) -> None:
    if block_size < 16 or block_size > 1 << 20 or block_size & (block_size - 1):
        raise ValueError(f"block_size must be a power of two from 16 to 2^20, got {block_size}")


def _check_cache(cache_k: torch.Tensor, cache_v: torch.Tensor, dtype: torch.dtype) -> None:
    """The two caches of one shape and type, laid out as the kernels read them."""
    if cache_k.dim() != 4 or cache_k.shape != cache_v.shape:
        raise ValueError(f"cache_k and cache_v must be [num_pages, kv_heads, block_size, head_dim], got "
                         f"{list(cache_k.shape)} and {list(cache_v.shape)}")
    if cache_k.numel() == 0:
        raise ValueError("cache_k and cache_v must not be empty")
    _check_block_size(cache_k.shape[2])
    for name, t in (("cache_k", cache_k), ("cache_v", cache_v)):
        if t.dtype != dtype:
            raise TypeError(f"{name} must have the type of the queries, {str(dtype)[6:]}, got {str(t.dtype)[6:]}")
        if not _rows_ok(t):
            raise ValueError(f"{name} must have a contiguous last dimension, other strides of multiples of 8 and a "
                             "16-byte aligned start")


def _caches_ok(cache_k: torch.Tensor, cache_v: torch.Tensor, dtype: torch.dtype) -> bool:
    """_check_cache as one test, for plain tensors; dtype one of _HALF_TYPES as well."""
    if cache_k.dim() != 4 or cache_k.dtype != dtype or cache_v.dtype != dtype or dtype not in _HALF_TYPES:
        return False
    shape = cache_k.shape
    a, b, c, one = cache_k.stride()
    e, f, g, last = cache_v.stride() if cache_v.dim() == 4 else (0, 0, 0, 0)
    block = shape[2]
    return (cache_v.shape == shape and one == 1 and last == 1 and not (a | b | c | e | f | g) & 7
            and a and b and c and e and f and g
            and not (cache_k.data_ptr() | cache_v.data_ptr()) & 15 and 16 <= block <= 1 << 20
            and not block & (block - 1) and cache_k.numel() > 0)


def _rows_ok(t: torch.Tensor) -> bool:
    """Whether the kernels can read t's last dimension in 16-byte pieces."""
    *strides, last = t.stride()
    return last == 1 and all(s % 8 == 0 for s in strides) and (isinstance(t, FakeTensor) or t.data_ptr() % 16 == 0)


def _check_heads(heads: int, kv_heads: int, head_dim: int) -> None:
    if heads < 1 or kv_heads < 1 or heads % kv_heads:
        raise ValueError(f"kv_heads={kv_heads} must divide heads={heads}")
    if head_dim < 8 or head_dim % 8 or head_dim > _ATTN_MAX_HEAD_DIM:
        raise ValueError(f"head_dim must be a multiple of 8 up to {_ATTN_MAX_HEAD_DIM}, got {head_dim}")


def _check_scale(scale: float | None, head_dim: int) -> float:
    if scale is None:
        return 1.0 / math.sqrt(head_dim)
    if not 0.0 < scale <= 2.35e38:  # finite in units of the exponent to base 2 as well
        raise ValueError(f"scale must be positive and at most 2.35e38, got {scale}")
    return float(scale)


def _own_places(t: torch.Tensor) -> bool:
    """Whether no dimension of a tensor that is written is expanded (stride 0)."""
    return all(s != 0 or n <= 1 for s, n in zip(t.stride(), t.shape))


def _check_out(out: torch.Tensor | None, q: torch.Tensor) -> None:
    if out is not None and (out.shape != q.shape or out.dtype != q.dtype or out.device != q.device
                            or not _rows_ok(out) or not _own_places(out)):
        raise ValueError(f"out must be {str(q.dtype)[6:]} {list(q.shape)} on {q.device} with a contiguous last dimension, "
                         "other strides of multiples of 8, none of them 0, and a 16-byte aligned start")


def paged_tables(block_table: torch.Tensor, context_lens: torch.Tensor, new_lens: torch.Tensor,
                 free_pages: torch.Tensor, free_count: torch.Tensor, *, block_size: int, max_tokens: int) -> PagedStep:
    """The tables of one step from the requests' lengths, in one launch (kf_paged_tables).

    block_table int32 [B, width] (updated in place); context_lens, new_lens int32 [B]: tokens of each request in
    the cache and tokens that this step adds (0 for a request that pauses). Pages that they need beyond those they
    hold come from the stack free_pages int32 [F] with free_count int32 [1] pages on it, the last first, and are
    entered into the table, -1 once the stack is empty; tokens whose page is -1 or past the table's width have no
    slot. max_tokens: rows of positions and slots (the step's tokens at least). free_pages and
    free_count are not changed: PagedStep.free_count is the count after the step. Lengths stay on the device, so a
    captured call follows them. No reference counterpart.
    """
    args = (block_table, context_lens, new_lens, free_pages, free_count, int(block_size), int(max_tokens))
    if _direct(block_table.get_device(), args[:5]) and block_table.dim() == 2:
        b, width = block_table.shape
        i32 = torch.int32
        if (context_lens.shape == (b,) and new_lens.shape == (b,) and free_count.shape == (1,) and free_pages.dim() == 1
                and block_table.dtype == i32 and context_lens.dtype == i32 and new_lens.dtype == i32
                and free_pages.dtype == i32 and free_count.dtype == i32 and b > 0 and width > 0 and max_tokens >= 0
                and block_table.stride(1) == 1 and (b == 1 or block_table.stride(0) >= width)
                and context_lens.is_contiguous() and new_lens.is_contiguous()
                and free_pages.is_contiguous() and 16 <= block_size <= 1 << 20 and not block_size & (block_size - 1)):
            cu_new, seq_lens, free_left = block_table.new_empty(2 * b + 2).split_with_sizes((b + 1, b, 1))
            odd = max_tokens & 1  # slots start at 16 bytes as well
            positions, _, slots = block_table.new_empty(2 * max_tokens + odd, dtype=torch.int64).split_with_sizes(
                (max_tokens, odd, max_tokens))
            return _run_paged_tables(*args, PagedStep(cu_new, seq_lens, positions, slots, free_left))
    b = block_table.shape[0] if block_table.dim() == 2 else -1
    _check_table(block_table, b)
    if b > 1 and block_table.stride(0) < block_table.shape[1]:
        raise ValueError("block_table is written: its rows must not overlap")
    _check_int("context_lens", context_lens, torch.int32, (b,))
    _check_int("new_lens", new_lens, torch.int32, (b,))
    _check_int("free_count", free_count, torch.int32, (1,))
    if free_pages.dtype != torch.int32 or free_pages.dim() != 1 or not free_pages.is_contiguous():
        raise ValueError("free_pages must be a contiguous 1-D int32 tensor")
    _check_block_size(block_size)
    if b < 1 or max_tokens < 0:
        raise ValueError(f"paged_tables needs at least one request and max_tokens >= 0, got {b} and {max_tokens}")
    _check_plain("paged_tables", args[:5])
    return PagedStep(*_paged_tables_op(*args)) if _traced(args[:5]) else _launch_paged_tables(*args)


def _launch_paged_tables(block_table, context_lens, new_lens, free_pages, free_count, block_size, max_tokens):
    dev = block_table.device
    for name, t in (("block_table", block_table), ("context_lens", context_lens), ("new_lens", new_lens),
                    ("free_pages", free_pages), ("free_count", free_count)):
        _check_memory(name, t, dev)
    b = block_table.shape[0]
    step = PagedStep(block_table.new_empty(b + 1), block_table.new_empty(b),
                     *(block_table.new_empty(max_tokens, dtype=torch.int64) for _ in range(2)), block_table.new_empty(1))
    with _on(dev):
        return _run_paged_tables(block_table, context_lens, new_lens, free_pages, free_count, block_size, max_tokens, step)


def _run_paged_tables(block_table, context_lens, new_lens, free_pages, free_count, block_size, max_tokens, step):
    """kf_paged_tables on checked arguments of the current device."""
    cu_new, seq_lens, positions, slots, free_left = step
    b, width = block_table.shape
    args = _lib.pack_paged_tables(block_table.data_ptr(), context_lens.data_ptr(), new_lens.data_ptr(),
                                  free_pages.data_ptr(), free_count.data_ptr(), cu_new.data_ptr(), seq_lens.data_ptr(),
                                  positions.data_ptr(), slots.data_ptr(), free_left.data_ptr(), block_table.stride(0), b,
                                  width, block_size, free_pages.numel(), max_tokens)
    status = _lib.load().kf_paged_tables(args, torch._C._cuda_getCurrentRawStream(block_table.get_device()))
    if status:
        _lib.check(status, "paged_tables")
    return step


@torch.library.custom_op("kernelforge::paged_tables", mutates_args=("block_table",))
def _paged_tables_op(block_table: torch.Tensor, context_lens: torch.Tensor, new_lens: torch.Tensor,
                     free_pages: torch.Tensor, free_count: torch.Tensor, block_size: int, max_tokens: int
                     ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    return tuple(_launch_paged_tables(block_table, context_lens, new_lens, free_pages, free_count, block_size, max_tokens))


@_paged_tables_op.register_fake
def _(block_table, context_lens, new_lens, free_pages, free_count, block_size, max_tokens):
    b = block_table.shape[0]
    return (block_table.new_empty(b + 1), block_table.new_empty(b), block_table.new_empty(max_tokens, dtype=torch.int64),
            block_table.new_empty(max_tokens, dtype=torch.int64), block_table.new_empty(1))


def rope_paged_cache(qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor,
                     slots: torch.Tensor, cache_k: torch.Tensor, cache_v: torch.Tensor, *,
                     heads: int) -> tuple[torch.Tensor, torch.Tensor]:
    """RoPE on q and k of a q|k|v projection, and k and v into the cache's slots, in one launch (kf_rope_paged_cache).

    qkv [T, (heads + 2 kv_heads) head_dim] (rows may be strided); cos, sin fp32 [max_pos, head_dim] (sin with the
    rotate-half sign folded in, as in int4_qkv_rope_cache); positions, slots int64 [T] (PagedStep's). Returns the
    rotated q [T, heads, head_dim] and k [T, kv_heads, head_dim], views of one tensor, rotated in 32 bits and
    rounded once; the caches get that k, and v as it is. A slot outside the cache writes no cache entry, nor does
    a position outside [0, max_pos), which rotates with row 0. Slots must be distinct. The form of
    int4_qkv_rope_cache for many tokens and a paged cache; no reference counterpart.
    """
    tensors = (qkv, cos, sin, positions, slots, cache_k, cache_v)
    if _direct(qkv.get_device(), tensors) and qkv.dim() == 2 and cos.dim() == 2 and _caches_ok(cache_k, cache_v, qkv.dtype):
        t, columns = qkv.shape
        kv_heads, d = cache_k.shape[1], cache_k.shape[3]
        row, one = qkv.stride()
        if (heads > 0 and heads % kv_heads == 0 and columns == (heads + 2 * kv_heads) * d and d % 8 == 0
                and d <= _ATTN_MAX_HEAD_DIM and t > 0 and one == 1 and row % 8 == 0 and cos.shape[0] > 0
                and cos.shape == sin.shape and cos.shape[1] == d and positions.shape == (t,) and slots.shape == (t,)
                and cos.dtype == torch.float32 and sin.dtype == torch.float32 and positions.dtype == torch.int64
                and slots.dtype == torch.int64 and cos.is_contiguous() and sin.is_contiguous()
                and positions.is_contiguous() and slots.is_contiguous()
                and not (qkv.data_ptr() | cos.data_ptr() | sin.data_ptr() | positions.data_ptr() | slots.data_ptr()) & 15):
            qk = _run_rope_paged(*tensors, int(heads))
            return qk.split_with_sizes((heads, kv_heads), 1)
    if qkv.dim() != 2 or qkv.dtype not in _HALF_TYPES:
        raise TypeError("qkv must be a 2-D fp16 or bf16 tensor [T, (heads + 2 kv_heads) head_dim]")
    _check_cache(cache_k, cache_v, qkv.dtype)
    if not _own_places(cache_k) or not _own_places(cache_v):
        raise ValueError("cache_k and cache_v are written: they must not be expanded")
    kv_heads, d = cache_k.shape[1], cache_k.shape[3]
    _check_heads(heads, kv_heads, d)
    t = qkv.shape[0]
    if qkv.shape[1] != (heads + 2 * kv_heads) * d:
        raise ValueError(f"qkv has {qkv.shape[1]} columns, not (heads + 2 kv_heads) head_dim = "
                         f"{(heads + 2 * kv_heads) * d}")
    if cos.dim() != 2 or cos.shape[0] < 1:
        raise ValueError(f"cos must be float32 [max_pos, {d}], got {list(cos.shape)}")
    _check_int("cos", cos, torch.float32, (cos.shape[0], d))
    _check_int("sin", sin, torch.float32, (cos.shape[0], d))
    _check_int("positions", positions, torch.int64, (t,))
    _check_int("slots", slots, torch.int64, (t,))
    _check_plain("rope_paged_cache", tensors)
    qk = (_rope_paged_op if _traced(tensors) else _launch_rope_paged)(*tensors, int(heads))
    return qk[:, :heads], qk[:, heads:]


def _launch_rope_paged(qkv, cos, sin, positions, slots, cache_k, cache_v, heads):
    dev = qkv.device
    for name, t in (("qkv", qkv), ("cos", cos), ("sin", sin), ("positions", positions), ("slots", slots),
                    ("cache_k", cache_k), ("cache_v", cache_v)):
        _check_memory(name, t, dev)
    if not _rows_ok(qkv):
        qkv = qkv.clone(memory_format=torch.contiguous_format)
    if qkv.shape[0] == 0:
        return qkv.new_empty(0, heads + cache_k.shape[1], cache_k.shape[3])
    cos, sin, positions, slots = (t if t.data_ptr() % 16 == 0 else t.clone() for t in (cos, sin, positions, slots))
    with _on(dev):
        return _run_rope_paged(qkv, cos, sin, positions, slots, cache_k, cache_v, heads)


def _run_rope_paged(qkv, cos, sin, positions, slots, cache_k, cache_v, heads):
    """kf_rope_paged_cache on checked arguments of the current device."""
    pages, kv_heads, block_size, d = cache_k.shape
    qk = qkv.new_empty((qkv.shape[0], heads + kv_heads, d))
    k_page, k_head, k_token, _ = cache_k.stride()
    v_page, v_head, v_token, _ = cache_v.stride()
    args = _lib.pack_rope_paged(qkv.data_ptr(), cos.data_ptr(), sin.data_ptr(), positions.data_ptr(), slots.data_ptr(),
                                qk.data_ptr(), cache_k.data_ptr(), cache_v.data_ptr(), qkv.stride(0), k_page, k_head,
                                k_token, v_page, v_head, v_token, qkv.shape[0], heads, kv_heads, d, cos.shape[0], pages,
                                block_size, _HALF_TYPES[qkv.dtype])
    status = _lib.load().kf_rope_paged_cache(args, torch._C._cuda_getCurrentRawStream(qkv.get_device()))
    if status:
        _lib.check(status, "rope_paged_cache")
    return qk


@torch.library.custom_op("kernelforge::rope_paged_cache", mutates_args=("cache_k", "cache_v"))
def _rope_paged_op(qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor,
                   slots: torch.Tensor, cache_k: torch.Tensor, cache_v: torch.Tensor, heads: int) -> torch.Tensor:
    return _launch_rope_paged(qkv, cos, sin, positions, slots, cache_k, cache_v, heads)


@_rope_paged_op.register_fake
def _(qkv, cos, sin, positions, slots, cache_k, cache_v, heads):
    return qkv.new_empty(qkv.shape[0], heads + cache_k.shape[1], cache_k.shape[3])


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor, *,
                     scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention over whole prompts, packed one after the other (kf_prompt_attention): one launch, or two for
    few row tiles over many keys.

    q [T, heads, head_dim], k and v [T, kv_heads, head_dim], fp16 or bf16, any strides of the first two dimensions
    (views of a fused projection are read in place; tokens of k and v up to 2^26 elements apart); cu_seqlens int32
    [B + 1] on the device: sequence s is rows cu_seqlens[s] .. cu_seqlens[s + 1] - 1, ascending from 0, empty ones
    allowed. Query head h reads KV head h // (heads / kv_heads); scale defaults to 1 / sqrt(head_dim). Scores, softmax
    and sums in 32 bits, probabilities rounded to the inputs' type for their product with v. Rows behind the last
    sequence are zeros in a new output and left as they are in ``out``, which must not overlap k or v. The form of
    decode_attention for prompts; no reference counterpart (its models run torch's attention).
    """
    tensors = (q, k, v, cu_seqlens)
    if _direct(q.get_device(), tensors) and out is None and q.dim() == 3 and k.dim() == 3 and v.dim() == 3:
        t, heads, d = q.shape
        kt, kv_heads, kd = k.shape
        dtype = q.dtype
        a, b, one = q.stride()
        c, e, two = k.stride()
        f, g, three = v.stride()
        if (dtype in _HALF_TYPES and k.dtype == dtype and v.dtype == dtype and v.shape == k.shape and kt == t and kd == d
                and t > 0 and kv_heads > 0 and heads > 0 and heads % kv_heads == 0 and 0 < d <= _ATTN_MAX_HEAD_DIM
                and not d & 7 and one == 1 and two == 1 and three == 1 and not (a | b | c | e | f | g) & 7
                and not (q.data_ptr() | k.data_ptr() | v.data_ptr()) & 15 and cu_seqlens.dtype == torch.int32
                and cu_seqlens.dim() == 1 and cu_seqlens.numel() > 1 and cu_seqlens.is_contiguous()):
            return _run_prompt(*tensors, _check_scale(scale, d), q.new_empty((t, heads, d)), True)
    if q.dim() != 3 or q.dtype not in _HALF_TYPES:
        raise TypeError("q must be a 3-D fp16 or bf16 tensor [T, heads, head_dim]")
    t, heads, d = q.shape
    if k.dim() != 3 or k.shape[0] != t or k.shape[2] != d or v.shape != k.shape:
        raise ValueError(f"k and v must be [{t}, kv_heads, {d}], got {list(k.shape)} and {list(v.shape)}")
    _check_heads(heads, k.shape[1], d)
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError(f"k and v must have the type of q, {str(q.dtype)[6:]}")
    if cu_seqlens.dim() != 1 or cu_seqlens.numel() < 2:
        raise ValueError("cu_seqlens must be int32 [B + 1] with B >= 1")
    _check_int("cu_seqlens", cu_seqlens, torch.int32, tuple(cu_seqlens.shape))
    scale = _check_scale(scale, d)
    _check_out(out, q)
    _check_plain("prompt_attention", tensors if out is None else (*tensors, out))
    if _traced(tensors):
        if out is not None:
            raise RuntimeError("prompt_attention with out updates it in place and has no traceable form")
        return _prompt_attention_op(*tensors, scale)
    return _launch_prompt(*tensors, scale, out)


def _launch_prompt(q, k, v, cu_seqlens, scale, out=None):
    dev = q.device
    for name, t in (("q", q), ("k", k), ("v", v), ("cu_seqlens", cu_seqlens)):
        _check_memory(name, t, dev)
    q, k, v = (t if _rows_ok(t) else t.clone(memory_format=torch.contiguous_format) for t in (q, k, v))
    zero_rest = out is None
    if out is None:
        out = q.new_empty(q.shape)
    if q.shape[0] == 0:
        return out
    with _on(dev):
        return _run_prompt(q, k, v, cu_seqlens, scale, out, zero_rest)


def _run_prompt(q, k, v, cu_seqlens, scale, out, zero_rest):
    """kf_prompt_attention on checked arguments of the current device."""
    t, heads, d = q.shape
    q_token, q_head, _ = q.stride()
    k_token, k_head, _ = k.stride()
    v_token, v_head, _ = v.stride()
    out_token, out_head, _ = out.stride()
    args = _lib.pack_prompt_attention(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), cu_seqlens.data_ptr(),
                                      q_token, q_head, k_token, k_head, v_token, v_head, out_token, out_head, t,
                                      cu_seqlens.numel() - 1, heads, k.shape[1], d, _HALF_TYPES[q.dtype], scale, zero_rest)
    lib = _lib.load()
    ws_bytes = lib.kf_prompt_attention_workspace_bytes(args)
    ws = q.new_empty((ws_bytes + 1) // 2) if ws_bytes else None  # two bytes a value
    status = lib.kf_prompt_attention(args, ws.data_ptr() if ws is not None else None, ws_bytes,
                                     torch._C._cuda_getCurrentRawStream(q.get_device()))
    if status:
        _lib.check(status, "prompt_attention")
    return out


@torch.library.custom_op("kernelforge::prompt_attention", mutates_args=())
def _prompt_attention_op(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor,
                         scale: float) -> torch.Tensor:
    return _launch_prompt(q, k, v, cu_seqlens, scale)


@_prompt_attention_op.register_fake
def _(q, k, v, cu_seqlens, scale):
    return q.new_empty(q.shape)


def paged_attention(q: torch.Tensor, cache_k: torch.Tensor, cache_v: torch.Tensor, block_table: torch.Tensor,
                    cu_new: torch.Tensor, seq_lens: torch.Tensor, *, max_new: int | None = None,
                    scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of every request's new tokens over its pages of the cache (kf_paged_attention).

    q [T, heads, head_dim], fp16 or bf16, any strides of the first two dimensions; block_table int32 [B, width];
    cu_new int32 [B + 1]: request r's new tokens are rows cu_new[r] .. cu_new[r + 1] - 1 of q, the last ones of
    its seq_lens[r] tokens (int32 [B]), whose keys and values the cache holds already (rope_paged_cache). One
    token per request (decode), chunks of prompts and batches of both. max_new: an upper bound of a request's new
    tokens, if the caller knows one; it and the table's width choose kernels and splits only (short requests are
    faster with a table, or a view of its first columns, that is not much wider than they need). Tokens whose page
    is not in the cache (-1) and those behind the table's last page are not attended to; a row with no key gets
    zeros. Rows behind the last request are zeros in a new output and left as they are in ``out``, which must not
    overlap the caches. Arithmetic as in prompt_attention; results do not change from run to run. The form of
    decode_attention for many requests; no reference counterpart.
    """
    tensors = (q, cache_k, cache_v, block_table, cu_new, seq_lens)
    if (_direct(q.get_device(), tensors) and out is None and q.dim() == 3 and block_table.dim() == 2
            and _caches_ok(cache_k, cache_v, q.dtype)):
        t, heads, d = q.shape
        _, kv_heads, _, kd = cache_k.shape
        b, width = block_table.shape
        a, c, one = q.stride()
        i32 = torch.int32
        if (d == kd and t > 0 and heads > 0 and heads % kv_heads == 0 and d <= _ATTN_MAX_HEAD_DIM and not d & 7 and one == 1
                and not (a | c) & 7 and not q.data_ptr() & 15 and b > 0 and width > 0 and block_table.stride(1) == 1
                and block_table.dtype == i32 and cu_new.dtype == i32 and seq_lens.dtype == i32 and cu_new.shape == (b + 1,)
                and seq_lens.shape == (b,) and cu_new.is_contiguous() and seq_lens.is_contiguous()
                and (max_new is None or max_new > 0)):
            return _run_paged(*tensors, int(max_new or 0), _check_scale(scale, d), q.new_empty((t, heads, d)), True)
    if q.dim() != 3 or q.dtype not in _HALF_TYPES:
        raise TypeError("q must be a 3-D fp16 or bf16 tensor [T, heads, head_dim]")
    _check_cache(cache_k, cache_v, q.dtype)
    if q.shape[2] != cache_k.shape[3]:
        raise ValueError(f"q has head_dim {q.shape[2]}, the caches {cache_k.shape[3]}")
    _check_heads(q.shape[1], cache_k.shape[1], q.shape[2])
    b = seq_lens.numel()
    _check_int("seq_lens", seq_lens, torch.int32, (b,))
    _check_int("cu_new", cu_new, torch.int32, (b + 1,))
    _check_table(block_table, b)
    if b < 1:
        raise ValueError("paged_attention needs at least one request")
    if max_new is not None and max_new < 1:
        raise ValueError(f"max_new must be positive, got {max_new}")
    scale = _check_scale(scale, q.shape[2])
    _check_out(out, q)
    _check_plain("paged_attention", tensors if out is None else (*tensors, out))
    if _traced(tensors):
        if out is not None:
            raise RuntimeError("paged_attention with out updates it in place and has no traceable form")
        return _paged_attention_op(*tensors, int(max_new or 0), scale)
    return _launch_paged(*tensors, int(max_new or 0), scale, out)


def _launch_paged(q, cache_k, cache_v, block_table, cu_new, seq_lens, max_new, scale, out=None):
    dev = q.device
    for name, t in (("q", q), ("cache_k", cache_k), ("cache_v", cache_v), ("block_table", block_table),
                    ("cu_new", cu_new), ("seq_lens", seq_lens)):
        _check_memory(name, t, dev)
    if not _rows_ok(q):
        q = q.clone(memory_format=torch.contiguous_format)
    zero_rest = out is None
    if out is None:
        out = q.new_empty(q.shape)
    if q.shape[0] == 0:
        return out
    with _on(dev):
        return _run_paged(q, cache_k, cache_v, block_table, cu_new, seq_lens, max_new, scale, out, zero_rest)


def _run_paged(q, cache_k, cache_v, block_table, cu_new, seq_lens, max_new, scale, out, zero_rest):
    """kf_paged_attention on checked arguments of the current device."""
    t, heads, d = q.shape
    pages, kv_heads, block_size, _ = cache_k.shape
    q_token, q_head, _ = q.stride()
    out_token, out_head, _ = out.stride()
    k_page, k_head, k_token, _ = cache_k.stride()
    v_page, v_head, v_token, _ = cache_v.stride()
    args = _lib.pack_paged_attention(q.data_ptr(), cache_k.data_ptr(), cache_v.data_ptr(), out.data_ptr(),
                                     block_table.data_ptr(), cu_new.data_ptr(), seq_lens.data_ptr(), q_token, q_head,
                                     out_token, out_head, k_page, k_head, k_token, v_page, v_head, v_token,
                                     block_table.stride(0), t, seq_lens.numel(), heads, kv_heads, d, _HALF_TYPES[q.dtype],
                                     block_table.shape[1], pages, block_size, max_new, scale, zero_rest)
    lib = _lib.load()
    ws_bytes = lib.kf_paged_attention_workspace_bytes(args)
    ws = q.new_empty((ws_bytes + 1) // 2) if ws_bytes else None  # two bytes a value
    status = lib.kf_paged_attention(args, ws.data_ptr() if ws is not None else None, ws_bytes,
                                    torch._C._cuda_getCurrentRawStream(q.get_device()))
    if status:
        _lib.check(status, "paged_attention")
    return out


@torch.library.custom_op("kernelforge::paged_attention", mutates_args=())
def _paged_attention_op(q: torch.Tensor, cache_k: torch.Tensor, cache_v: torch.Tensor, block_table: torch.Tensor,
                        cu_new: torch.Tensor, seq_lens: torch.Tensor, max_new: int, scale: float) -> torch.Tensor:
    return _launch_paged(q, cache_k, cache_v, block_table, cu_new, seq_lens, max_new, scale)


@_paged_attention_op.register_fake
def _(q, cache_k, cache_v, block_table, cu_new, seq_lens, max_new, scale):
    return q.new_empty(q.shape)
