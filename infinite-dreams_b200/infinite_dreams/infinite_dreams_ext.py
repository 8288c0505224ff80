"""Drop-in for the reference's compiled extension ``infinite_dreams_ext``.

The reference module (src/gemm_ext.cpp:123-132) exports three functions; the
same three names are exported here with the same argument meaning and the
same error behaviour (``RuntimeError`` with the reference's messages), backed
by the sm_100a kernel bank through its C ABI (include/gemm_sm100.h):

* ``gemm_forward(A, B, tile_m, tile_n, tile_k, stages, mma_sm=1, raster=0,
  group=8, split_k=1)`` -- explicit knobs (src/gemm_ext.cpp:57-93).  The
  reference's knobs were (tile_m, tile_n, tile_k, tm, tn); the register
  micro-tile (tm, tn) has no meaning for tcgen05, so the positions after
  tile_k carry the Blackwell knobs.  A tuple that is not in the menu raises
  (the reference returned an uninitialised tensor, gemm_ext.cpp:35 + F7).
* ``gemm_forward_cfg(A, B, cfg_id)`` -- menu id (src/gemm_ext.cpp:95-106).
* ``gemm_cfg_table_cpu()`` -- the menu as a CPU int32 tensor
  ``[num_cfg, len(CFG_COLUMNS)]`` (src/gemm_ext.cpp:108-120).

``gemm_ex`` goes beyond the reference: transposed operand views read in
place and a fused epilogue (alpha, beta * C, bias, ReLU / GELU).  So do the
products whose weight is picked by the row, in fp16 and bf16:
``grouped_gemm`` (rows sorted by expert, ragged counts) and its weight
gradient ``grouped_gemm_wgrad`` (``grouped.grouped_linear`` is the pair as a
differentiable function), and ``lora_gemm`` (a shared projection with the
low-rank adapter that each row picks).

Like the reference, inputs are made contiguous, C is allocated from torch's
caching allocator on A's device, and the launch is asynchronous on the
current stream.  Split-K / repacking workspace is cached per (device, stream)
and zero-initialised once, as the C ABI requires.
"""
from __future__ import annotations

import ctypes
import os
import threading
from typing import Dict, Optional, Tuple

import torch

from . import _capi
from ._capi import GemmError, lib

CFG_COLUMNS: Tuple[str, ...] = tuple(_capi.menu()[0])
NUM_CFG: int = int(lib.gemm_num_cfgs())

# The compiled torch binding of the same C ABI (csrc/torch_ext.cpp) takes the
# per-call Python work off small launches; the ctypes path below remains for
# builds without it (INFINITE_DREAMS_NO_TORCH_EXT=1 selects it explicitly).
_fast = None
if not os.environ.get("INFINITE_DREAMS_NO_TORCH_EXT"):
    try:
        from . import _torch_ext as _fast  # type: ignore[no-redef]
    except ImportError:
        _fast = None

_ws_lock = threading.Lock()
_workspaces: Dict[Tuple[int, int], torch.Tensor] = {}


def _workspace(device: torch.device, stream: torch.cuda.Stream, nbytes: int) -> Tuple[int, int]:
    if nbytes == 0:
        return 0, 0
    key = (device.index, stream.cuda_stream)
    with _ws_lock:
        ws = _workspaces.get(key)
        if ws is None or ws.numel() < nbytes:
            # Grow geometrically; zeros satisfies the "ticket region is zero" contract.
            size = max(nbytes, 0 if ws is None else 2 * ws.numel())
            with torch.cuda.stream(stream):
                ws = torch.zeros(size, dtype=torch.uint8, device=device)
            _workspaces[key] = ws
    return ws.data_ptr(), ws.numel()


def reset_workspaces() -> None:
    """Drops cached workspaces (needed after a device-side timeout)."""
    with _ws_lock:
        _workspaces.clear()
    if _fast is not None:
        _fast.reset_workspaces()


def _check_inputs(A: torch.Tensor, B: torch.Tensor) -> None:
    # Same checks and messages as src/gemm_ext.cpp:66-73,86.
    if not isinstance(A, torch.Tensor) or not A.is_cuda:
        raise RuntimeError("A must be CUDA tensor")
    if not isinstance(B, torch.Tensor) or not B.is_cuda:
        raise RuntimeError("B must be CUDA tensor")
    if A.dtype != torch.float16:
        raise RuntimeError("A must be float16")
    if B.dtype != torch.float16:
        raise RuntimeError("B must be float16")
    if A.dim() != 2:
        raise RuntimeError("A must be 2D (M x K)")
    if B.dim() != 2:
        raise RuntimeError("B must be 2D (K x N)")
    if A.size(1) != B.size(0):
        raise RuntimeError("Inner dimensions must match: A is (M x K), B is (K x N)")
    if A.get_device() != B.get_device():
        raise RuntimeError("A and B must be on the same CUDA device")


def _launch(A: torch.Tensor, B: torch.Tensor, cfg_id: int, out: Optional[torch.Tensor]) -> torch.Tensor:
    if A.get_device() != torch.cuda.current_device():
        with torch.cuda.device(A.device):
            return _launch_here(A, B, cfg_id, out)
    return _launch_here(A, B, cfg_id, out)


def _launch_here(A: torch.Tensor, B: torch.Tensor, cfg_id: int, out: Optional[torch.Tensor]) -> torch.Tensor:
    """Launch on A's device, which is the current device."""
    M, K = A.shape
    N = B.shape[1]
    dev = A.device
    A = A.contiguous()
    B = B.contiguous()
    if out is None:
        C = torch.empty((M, N), dtype=torch.float16, device=dev)
    else:
        if (out.dtype != torch.float16 or out.shape != (M, N) or out.device != dev
                or not out.is_contiguous()):
            raise RuntimeError("out must be a contiguous float16 (M x N) tensor on A's device")
        C = out
    stream = torch.cuda.current_stream(dev)
    a_ptr, b_ptr = A.data_ptr(), B.data_ptr()
    need = lib.gemm_workspace_bytes(a_ptr, b_ptr, M, N, K, K, N, cfg_id)
    ws_ptr, ws_len = _workspace(dev, stream, need) if need else (0, 0)
    st = lib.gemm_launch(a_ptr, b_ptr, C.data_ptr(), M, N, K, K, N, N, cfg_id,
                         ws_ptr or None, ws_len, stream.cuda_stream or None)
    if st:
        _capi.check(st, "gemm_launch")
    return C


def gemm_forward(A: torch.Tensor, B: torch.Tensor, tile_m: int, tile_n: int, tile_k: int, stages: int,
                 mma_sm: int = 1, raster: int = 0, group: int = 8, split_k: int = 1,
                 *, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """FP16 GEMM forward (CUDA) with explicit knobs; the tuple must be in the menu."""
    _check_inputs(A, B)
    if tile_m <= 0 or tile_n <= 0 or tile_k <= 0:
        raise RuntimeError("tile_m/tile_n/tile_k must be > 0")
    if stages <= 0 or mma_sm <= 0 or group <= 0 or split_k <= 0:
        raise RuntimeError("stages/mma_sm/group/split_k must be > 0")
    knobs = (tile_m, tile_n, tile_k, stages, mma_sm, raster, group, split_k)
    cfg_id = _capi.cfg_find(knobs)
    if cfg_id < 0:
        raise RuntimeError(f"knob tuple {knobs} is not in the kernel bank menu "
                           f"(columns {', '.join(CFG_COLUMNS)})")
    if _fast is not None:
        return _fast.gemm_forward_cfg(A, B, cfg_id, out)
    return _launch(A, B, cfg_id, out)


def gemm_forward_cfg(A: torch.Tensor, B: torch.Tensor, cfg_id: int, *,
                     out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """FP16 GEMM forward (CUDA) using cfg_id from the static menu."""
    if cfg_id < 0:
        raise RuntimeError("cfg_id must be >= 0")
    if cfg_id >= NUM_CFG:
        raise RuntimeError("cfg_id out of range")
    if _fast is not None:
        return _fast.gemm_forward_cfg(A, B, int(cfg_id), out)
    _check_inputs(A, B)
    return _launch(A, B, int(cfg_id), out)


def _operand(X: torch.Tensor) -> Tuple[torch.Tensor, int, int]:
    """(tensor, trans, pitch) for a logical [R, C] operand read in place.

    A row-major view (unit column stride) is passed as stored; a transposed
    view (unit row stride, e.g. ``W.t()``) is passed as its K-major storage
    with trans = 1, which the kernels read without a copy.  Anything else is
    made contiguous first.
    """
    R, C = X.shape
    s0, s1 = X.stride()
    if (s1 == 1 or C <= 1) and s0 >= max(C, 1):
        return X, 0, s0
    if (s0 == 1 or R <= 1) and s1 >= max(R, 1):
        return X, 1, s1
    X = X.contiguous()
    return X, 0, max(C, 1)


def gemm_ex(A: torch.Tensor, B: torch.Tensor, *, alpha: float = 1.0, beta: float = 0.0,
            C: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, activation: str = "none",
            cfg_id: Optional[int] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """out = act(alpha * A @ B + beta * C + bias), fp16, fused into the GEMM's epilogue.

    A is a logical [M, K] and B a logical [K, N] fp16 CUDA tensor; row-major
    and transposed views (``x.t()``) are read in place (gemm_launch_ex's
    trans flags), other strides are copied.  C ([M, N], read only when
    beta != 0) may be ``out`` itself for an in-place update; bias is [N].
    activation: "none", "relu" or "gelu" (erf form).  cfg_id defaults to the
    per-shape dispatch table entry, else the heuristic.
    """
    _check_inputs(A, B)
    if activation not in _capi.ACTIVATIONS:
        raise RuntimeError(f"activation must be one of {sorted(_capi.ACTIVATIONS)}")
    M, K = A.shape
    N = B.shape[1]
    dev = A.device
    if _fast is not None:
        if cfg_id is None:
            from . import dispatch
            cfg_id = dispatch.lookup(M, N, K, epilogue=(beta != 0.0 or activation != "none"))
        return _fast.gemm_ex(A, B, int(cfg_id), float(alpha), float(beta), C, bias, _capi.ACTIVATIONS[activation],
                             out)
    if beta != 0.0:
        if C is None:
            raise RuntimeError("beta != 0 needs C")
        if C.dtype != torch.float16 or tuple(C.shape) != (M, N) or C.device != dev:
            raise RuntimeError("C must be a float16 (M x N) tensor on A's device")
        if (C.stride(1) != 1 and N > 1) or (M > 1 and C.stride(0) < N):   # expanded rows too
            C = C.contiguous()
    if bias is not None:
        if bias.dtype != torch.float16 or bias.numel() != N or bias.device != dev:
            raise RuntimeError("bias must be a float16 tensor of N elements on A's device")
        bias = bias.reshape(N).contiguous()
    if cfg_id is None:
        from . import dispatch
        cfg_id = dispatch.lookup(M, N, K, epilogue=(beta != 0.0 or activation != "none"))
    elif not 0 <= int(cfg_id) < NUM_CFG:
        raise RuntimeError("cfg_id out of range")
    with torch.cuda.device(dev):
        A_s, ta, lda = _operand(A)
        B_s, tb, ldb = _operand(B)
        if out is None:
            out = torch.empty((M, N), dtype=torch.float16, device=dev)
        elif (out.dtype != torch.float16 or tuple(out.shape) != (M, N) or out.device != dev
              or (out.stride(1) != 1 and N > 1) or (M > 1 and out.stride(0) < N)):
            raise RuntimeError("out must be a float16 (M x N) tensor with unit column stride on A's device, its rows "
                               "apart")
        stream = torch.cuda.current_stream(dev)
        a_ptr, b_ptr = A_s.data_ptr(), B_s.data_ptr()
        need = lib.gemm_workspace_bytes_ex(a_ptr, b_ptr, M, N, K, lda, ldb, ta, tb, int(cfg_id))
        ws_ptr, ws_len = _workspace(dev, stream, need) if need else (0, 0)
        d_ptr, ldd = (C.data_ptr(), max(C.stride(0), N)) if beta != 0.0 else (None, 0)
        st = lib.gemm_launch_ex(a_ptr, b_ptr, out.data_ptr(), M, N, K, lda, ldb, max(out.stride(0), N), ta, tb,
                                float(alpha), float(beta), d_ptr, ldd,
                                bias.data_ptr() if bias is not None else None, _capi.ACTIVATIONS[activation],
                                int(cfg_id), ws_ptr or None, ws_len, stream.cuda_stream or None)
        if st:
            _capi.check(st, "gemm_launch_ex")
    return out


def _scratch(device: torch.device, nbytes: int):
    """(keep-alive, pointer, bytes) of one call's workspace, from torch's allocator and not the cached one.

    These operators' launches come in twos (repacking or the low-rank half,
    then the product), between which another thread's call on the same stream
    would overwrite a shared buffer; and two graphs captured on one stream may
    be replayed on two.
    """
    if nbytes == 0:
        return None, None, 0
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
    return ws, ws.data_ptr(), nbytes


def _is_16bit(t) -> bool:
    return t.dtype in (torch.float16, torch.bfloat16)


def _dtype_id(t: torch.Tensor) -> int:
    return _capi.GEMM_DTYPE_BF16 if t.dtype == torch.bfloat16 else _capi.GEMM_DTYPE_F16


def _check_like(t, A: torch.Tensor, name: str) -> None:
    """A is the operand that holds the rows; every other one goes by it."""
    if not isinstance(t, torch.Tensor) or t.device != A.device:
        raise RuntimeError(f"{name} must be on the rows' device")
    if t.dtype != A.dtype:
        raise RuntimeError(f"{name} must have the rows' dtype")


def _check_index(t, A: torch.Tensor, n: int, name: str) -> None:
    if not isinstance(t, torch.Tensor) or t.device != A.device:
        raise RuntimeError(f"{name} must be on the rows' device")
    if t.dtype not in (torch.int32, torch.int64):
        raise RuntimeError(f"{name} must be int32 or int64")
    if t.dim() != 1 or t.size(0) != n:
        raise RuntimeError(f"{name} must be 1D with {n} elements")


def _shares_memory(out: torch.Tensor, t: torch.Tensor) -> bool:
    """Whether t shares bytes with out, which is rows of adjacent elements (2D), or a stack of them (3D, row-major
    or transposed, its matrices apart)."""
    def extent(x):   # bytes from the first to the last element
        return (1 + sum((n - 1) * st for n, st in zip(x.shape, x.stride()))) * x.element_size()
    es, ts = out.element_size(), t.element_size()
    o0, t0 = out.data_ptr(), t.data_ptr()
    if t0 + extent(t) <= o0 or o0 + extent(out) <= t0:
        return False
    if extent(t) == t.numel() * ts and extent(out) == out.numel() * es:   # two dense blocks
        return True
    if (t.dim() == 2 and out.dim() == 2 and es == ts and t.stride(1) == 1 and out.stride(1) == 1 and t.size(0) > 1
            and out.size(0) > 1 and t.stride(0) == out.stride(0) and t.stride(0) >= max(t.size(1), out.size(1))):
        row = out.stride(0) * es
        c = (t0 - o0) % row   # columns of one buffer: where t's begin in out's rows
        return c < out.size(1) * es or c + t.size(1) * es > row
    # out: E matrices, se bytes apart, of R rows, sr apart, of `width` bytes
    d = out.dim()
    trans = d == 3 and out.stride(2) != 1 and out.size(2) > 1
    row_dim, col_dim = d - (1 if trans else 2), d - (2 if trans else 1)
    far = extent(out) + 1   # the pitch of one thing
    R, width, E = out.size(row_dim), out.size(col_dim) * es, out.size(0) if d == 3 else 1
    sr = out.stride(row_dim) * es if R > 1 else far
    se = out.stride(0) * es if E > 1 else far
    # t: runs of adjacent elements, the bytes [a, b) from out's first
    run_dims = [i for i in range(t.dim()) if t.stride(i) == 1 and t.size(i) > 1]
    run = (t.size(run_dims[-1]) if run_dims else 1) * ts
    a = torch.tensor([t0 - o0])
    for i in range(t.dim()):
        if i not in run_dims[-1:] and t.stride(i) != 0:
            a = (a[:, None] + torch.arange(t.size(i))[None, :] * (t.stride(i) * ts)).flatten()
    b = a + run
    e = torch.div(a, se, rounding_mode="floor")
    next_e = (e + 1).clamp_min(0)
    meet = (next_e < E) & (next_e * se < b)          # the next matrix begins before b
    left = a - e * se
    r = torch.div(left, sr, rounding_mode="floor")
    inside = ((r < R) & (left - r * sr < width)) | ((r + 1 < R) & (e * se + (r + 1) * sr < b))
    return bool((meet | ((e >= 0) & (e < E) & inside)).any())


def _check_apart(out: torch.Tensor, *tensors) -> None:
    """The kernels read operands while they write out."""
    if out.numel() == 0:
        return
    for t in tensors:
        if t is not None and t.numel() > 0 and _shares_memory(out, t):
            raise RuntimeError("out must not share memory with an operand")


def _count_write(out: torch.Tensor) -> None:
    """A graph that saved out notices that it was written; tensors made in inference mode keep no such count."""
    if not out.is_inference():
        torch.autograd.graph.increment_version(out)


def _check_no_grad(what: str, *tensors) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError(what)
    if any(t is not None and torch.autograd.forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError("the operator has no forward-mode derivative: an input's tangent would be lost")


def _stacked_operand(X: torch.Tensor) -> Tuple[torch.Tensor, int, int, int]:
    """(tensor, trans, pitch, matrix stride) of a stack of weights [E, R, C] read in place.

    Strides that are neither row-major nor transposed, or matrices that
    overlap (expanded weights), are copied.
    """
    E, R, C = X.shape
    se, s0, s1 = X.stride()
    if (s1 == 1 or C <= 1) and s0 >= max(C, 1) and (E == 1 or se >= (R - 1) * s0 + C):
        return X, 0, s0, se
    if (s0 == 1 or R <= 1) and s1 >= max(R, 1) and (E == 1 or se >= (C - 1) * s1 + R):
        return X, 1, s1, se
    return X.contiguous(), 0, max(C, 1), R * max(C, 1)


def _row_operand(X: torch.Tensor) -> torch.Tensor:
    ok = (X.stride(1) == 1 or X.size(1) <= 1) and (X.size(0) <= 1 or X.stride(0) >= X.size(1))
    return X if ok else X.contiguous()


def _pitch(X: torch.Tensor) -> int:
    return max(X.size(1), 1) if X.size(0) <= 1 else max(X.stride(0), 1)


def _rows_out(out: Optional[torch.Tensor], T: int, N: int, A: torch.Tensor) -> torch.Tensor:
    if out is None:
        return torch.empty((T, N), dtype=A.dtype, device=A.device)
    if (out.device != A.device or out.dtype != A.dtype or tuple(out.shape) != (T, N)
            or (out.stride(1) != 1 and N > 1) or (T > 1 and out.stride(0) < N)):
        raise RuntimeError("out must be a (T x N) tensor of the rows' dtype with unit column stride on their device")
    return out


def grouped_gemm(A: torch.Tensor, B: torch.Tensor, offsets: torch.Tensor, *, bias: Optional[torch.Tensor] = None,
                 activation: str = "none", out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """out[r] = act(A[r] @ B[e] + bias[e]) for the rows offsets[e] <= r < offsets[e + 1] of group e.

    A is [T, K] with its rows sorted by group, B a stack of weights [E, K, N]
    (row-major, or a transposed view of [E, N, K] storage; both are read in
    place), bias [E, N]; fp16 or bf16, all alike.  offsets: E + 1
    non-decreasing int32 or int64 row numbers on the device; the call never
    synchronises, and offsets that decrease or leave [0, T] are clamped and
    reported by ``check_device_errors``.  Groups may be empty.  Rows outside
    [offsets[0], offsets[E]) are zero in a new ``out`` and left as they are
    in a given one, which must not share memory with an operand.  The input gradient of a plain product is
    ``grouped_gemm(dy, B.transpose(1, 2), offsets)``.  At most 1024 groups.
    """
    if activation not in _capi.ACTIVATIONS:
        raise RuntimeError(f"activation must be one of {sorted(_capi.ACTIVATIONS)}")
    act = _capi.ACTIVATIONS[activation]
    if _fast is not None:
        return _fast.grouped_gemm(A, B, offsets, bias, act, out)
    if not isinstance(A, torch.Tensor) or not A.is_cuda:
        raise RuntimeError("A must be CUDA tensor")
    if not _is_16bit(A):
        raise RuntimeError("A must be float16 or bfloat16")
    if A.dim() != 2:
        raise RuntimeError("A must be 2D (T x K)")
    _check_like(B, A, "B")
    if B.dim() != 3:
        raise RuntimeError("B must be 3D (E x K x N)")
    if A.size(1) != B.size(1):
        raise RuntimeError("Inner dimensions must match: A is (T x K), B is (E x K x N)")
    if B.size(0) < 1:
        raise RuntimeError("B must hold at least one group")
    E, K, N = B.shape
    T = A.size(0)
    _check_index(offsets, A, E + 1, "offsets")
    if bias is not None:
        _check_like(bias, A, "bias")
        if tuple(bias.shape) != (E, N):
            raise RuntimeError("bias must be (E x N)")
    _check_no_grad("grouped_gemm computes no gradients: use grouped.grouped_linear, or call it under "
                   "torch.no_grad()", A, B, bias, out)
    with torch.cuda.device(A.device):
        As, off = _row_operand(A), offsets.contiguous()
        Bs, tb, ldb, sb = _stacked_operand(B)
        C = _rows_out(out, T, N, A)
        if out is not None:
            _check_apart(C, A, B, offsets, bias)
        bias = None if bias is None else bias.contiguous()
        stream = torch.cuda.current_stream(A.device)
        lda = _pitch(As)
        need = lib.gemm_grouped_workspace_bytes(As.data_ptr(), Bs.data_ptr(), T, N, K, E, lda, ldb, sb, tb)
        keep, ws_ptr, ws_len = _scratch(A.device, need)
        st = lib.gemm_grouped_launch(As.data_ptr(), Bs.data_ptr(), C.data_ptr(), off.data_ptr(),
                                     64 if off.dtype == torch.int64 else 32, T, N, K, E, lda, ldb, sb,
                                     max(_pitch(C), N), tb, bias.data_ptr() if bias is not None else None, act,
                                     0 if out is not None else 1, _dtype_id(A), ws_ptr, ws_len,
                                     stream.cuda_stream or None)
        _capi.check(st, "gemm_grouped_launch")
    if out is not None:
        _count_write(C)
    return C


def grouped_gemm_wgrad(A: torch.Tensor, G: torch.Tensor, offsets: torch.Tensor, *,
                       out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """out[e] = A[r].T @ G[r] over the rows r of group e: the weight gradient of ``grouped_gemm``.

    A is [T, K], G [T, N] (fp16 or bf16, alike), offsets as for
    ``grouped_gemm``; out is [E, K, N], row-major or a transposed view of
    [E, N, K] storage.  An empty group's matrix is zero; rows outside every
    group do not enter.
    """
    if _fast is not None:
        return _fast.grouped_gemm_wgrad(A, G, offsets, out)
    if not isinstance(A, torch.Tensor) or not A.is_cuda:
        raise RuntimeError("A must be CUDA tensor")
    if not _is_16bit(A):
        raise RuntimeError("A must be float16 or bfloat16")
    if A.dim() != 2:
        raise RuntimeError("A must be 2D (T x K)")
    _check_like(G, A, "G")
    if G.dim() != 2 or G.size(0) != A.size(0):
        raise RuntimeError("G must be 2D (T x N) with A's rows")
    if offsets.dim() != 1 or offsets.size(0) < 2:
        raise RuntimeError("offsets must be 1D with at least 2 elements")
    _check_index(offsets, A, offsets.size(0), "offsets")
    (T, K), N, E = A.shape, G.size(1), offsets.size(0) - 1
    _check_no_grad("grouped_gemm_wgrad computes no gradients: call it under torch.no_grad()", A, G, out)
    with torch.cuda.device(A.device):
        D = torch.empty((E, K, N), dtype=A.dtype, device=A.device) if out is None else out
        if D.device != A.device or D.dtype != A.dtype or tuple(D.shape) != (E, K, N):
            raise RuntimeError("out must be an (E x K x N) tensor of A's dtype on A's device")
        Ds, td, ldd, sd = _stacked_operand(D)
        if Ds.data_ptr() != D.data_ptr():
            raise RuntimeError("out must be row-major or a transposed view, its matrices apart")
        As, Gs, off = _row_operand(A), _row_operand(G), offsets.contiguous()
        if out is not None:
            _check_apart(D, A, G, offsets)
        L, R = (Gs, As) if td else (As, Gs)   # a gradient stored N x K: the operands exchanged
        stream = torch.cuda.current_stream(A.device)
        need = lib.gemm_grouped_wgrad_workspace_bytes(L.data_ptr(), R.data_ptr(), T, L.size(1), R.size(1), _pitch(L),
                                                      _pitch(R))
        keep, ws_ptr, ws_len = _scratch(A.device, need)
        st = lib.gemm_grouped_wgrad_launch(L.data_ptr(), R.data_ptr(), Ds.data_ptr(), off.data_ptr(),
                                           64 if off.dtype == torch.int64 else 32, T, L.size(1), R.size(1), E,
                                           _pitch(L), _pitch(R), ldd, sd, _dtype_id(A), ws_ptr, ws_len,
                                           stream.cuda_stream or None)
        _capi.check(st, "gemm_grouped_wgrad_launch")
    if out is not None:
        _count_write(D)
    return D


def lora_gemm(x: torch.Tensor, W: torch.Tensor, down: torch.Tensor, up: torch.Tensor, adapter: torch.Tensor, *,
              scale: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, activation: str = "none",
              out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """out[t] = act(x[t] @ W + scale[a] * (x[t] @ down[a]) @ up[a] + bias) with a = adapter[t].

    The shared projection W [K, N] of all rows, beside the low-rank adapter
    that each row picks: x is [T, K], down [L, K, R], up [L, R, N] (each
    weight row-major or a transposed view, read in place), fp16 or bf16, all
    alike.  adapter: T int32 or int64 numbers on the device, in any order;
    negative means none, a number past the last adapter counts as none and
    is reported by ``check_device_errors``.  scale is float32 [L], bias [N].
    Adapters of smaller ranks are padded with zeros; R is at most 1024.
    scale * (x @ down) is kept to 2^-16 of it, over the range of float32.
    One request's inf or NaN does not reach the rows of others.  A serving
    operator: it computes no gradients and refuses inputs that ask for them.
    """
    if activation not in _capi.ACTIVATIONS:
        raise RuntimeError(f"activation must be one of {sorted(_capi.ACTIVATIONS)}")
    act = _capi.ACTIVATIONS[activation]
    if _fast is not None:
        return _fast.lora_gemm(x, W, down, up, adapter, scale, bias, act, out)
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise RuntimeError("x must be CUDA tensor")
    if not _is_16bit(x):
        raise RuntimeError("x must be float16 or bfloat16")
    if x.dim() != 2:
        raise RuntimeError("x must be 2D (T x K)")
    for t, name in ((W, "W"), (down, "down"), (up, "up")):
        _check_like(t, x, name)
    T, K = x.shape
    if W.dim() != 2 or W.size(0) != K:
        raise RuntimeError("W must be 2D (K x N)")
    N = W.size(1)
    if down.dim() != 3 or down.size(1) != K:
        raise RuntimeError("down must be 3D (L x K x R)")
    L, R = down.size(0), down.size(2)
    if tuple(up.shape) != (L, R, N):
        raise RuntimeError("up must be 3D (L x R x N)")
    if K < 1 or L < 1 or R < 1:
        raise RuntimeError("K, the number of adapters and the rank must be at least 1")
    _check_index(adapter, x, T, "adapter")
    if scale is not None:
        if scale.device != x.device or scale.dtype != torch.float32 or tuple(scale.shape) != (L,):
            raise RuntimeError("scale must be a float32 tensor of L elements on x's device")
    if bias is not None:
        _check_like(bias, x, "bias")
        if tuple(bias.shape) != (N,):
            raise RuntimeError("bias must be (N)")
    _check_no_grad("lora_gemm is a serving operator and computes no gradients: call it under torch.no_grad()",
                   x, W, down, up, scale, bias, out)
    with torch.cuda.device(x.device):
        xs, ids = _row_operand(x), adapter.contiguous()
        Ws, tw, ldw = _operand(W)
        Ds, td, ldd, sd = _stacked_operand(down)
        Us, tu, ldu, su = _stacked_operand(up)
        C = _rows_out(out, T, N, x)
        if out is not None:
            _check_apart(C, x, W, down, up, adapter, scale, bias)
        scale, bias = (None if t is None else t.contiguous() for t in (scale, bias))
        stream = torch.cuda.current_stream(x.device)
        ldx = _pitch(xs)
        need = lib.gemm_lora_workspace_bytes(xs.data_ptr(), Ws.data_ptr(), Us.data_ptr(), T, N, K, L, R, ldx, ldw, tw,
                                             ldu, su, tu)
        keep, ws_ptr, ws_len = _scratch(x.device, need)
        st = lib.gemm_lora_launch(xs.data_ptr(), Ws.data_ptr(), Ds.data_ptr(), Us.data_ptr(), C.data_ptr(),
                                  ids.data_ptr(), 64 if ids.dtype == torch.int64 else 32, T, N, K, L, R, ldx, ldw, tw,
                                  ldd, sd, td, ldu, su, tu, max(_pitch(C), N),
                                  scale.data_ptr() if scale is not None else None,
                                  bias.data_ptr() if bias is not None else None, act, _dtype_id(x), ws_ptr, ws_len,
                                  stream.cuda_stream or None)
        _capi.check(st, "gemm_lora_launch")
    if out is not None:
        _count_write(C)
    return C


def gemm_cfg_table_cpu() -> torch.Tensor:
    """CPU int32 tensor [num_cfg, len(CFG_COLUMNS)], columns CFG_COLUMNS."""
    cols, rows = _capi.menu()
    return torch.tensor(rows, dtype=torch.int32).reshape(len(rows), len(cols))


def default_cfg(M: int, N: int, K: int) -> int:
    return int(lib.gemm_default_cfg(M, N, K))


def check_device_errors(device: Optional[int] = None) -> None:
    """Raises if a kernel on `device` gave up on a bounded wait, or was given offsets or adapter indices out of
    range, since the last call (synchronises)."""
    dev = torch.cuda.current_device() if device is None else int(device)
    code = ctypes.c_int(0)
    st = lib.gemm_device_error(dev, ctypes.byref(code))
    if st != _capi.GEMM_OK:
        message = lib.gemm_last_error().decode(errors="replace")
        if st != _capi.GEMM_ERR_INVALID_ARG:   # index data out of range leaves the workspaces clean
            reset_workspaces()
        raise GemmError(st, f"device {dev}: kernel error bits {code.value}: {message}")


__all__ = ["gemm_forward", "gemm_forward_cfg", "gemm_ex", "grouped_gemm", "grouped_gemm_wgrad", "lora_gemm",
           "gemm_cfg_table_cpu", "CFG_COLUMNS", "NUM_CFG",
           "default_cfg", "check_device_errors", "GemmError", "reset_workspaces"]
