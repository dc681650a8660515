"""The gated projection of a feed-forward block: ``act(x @ w_gate) * (x @ w_up)`` in one kernel.

:func:`gated_matmul` takes fp16 / bf16 operands and has gradients; :func:`gated_gemm` takes e4m3 / int8 operands with
scales, as :func:`helion_b200.rms_norm_quantize` and :func:`helion_b200.quantize_rows` make them.  The reference's
examples stop at one product with an epilogue (examples/matmul.py:26-56).
"""
from __future__ import annotations

import weakref
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .ops import _INT8_MAX_K, _OUT_DT, _changed, _empty_matrix, _require_cuda, _round_up, _stream_ptr

_ACTIVATIONS = {"silu": _lib.ACT_SILU, "gelu": _lib.ACT_GELU, "gelu_tanh": _lib.ACT_GELU_TANH}


def _check_gated(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, activation: str, what: str) -> int:
    xs, gs, us = x.shape, w_gate.shape, w_up.shape
    if not (len(xs) == len(gs) == len(us) == 2):
        raise ValueError(f"{what} expects 2-D inputs, got {tuple(xs)}, {tuple(gs)} and {tuple(us)}")
    if gs != us:
        raise ValueError(f"{what}: w_gate {tuple(gs)} and w_up {tuple(us)} differ in shape")
    if xs[1] != gs[0]:
        raise ValueError(f"{what}: size mismatch, x is {tuple(xs)} and the weights {tuple(gs)}")
    act = _ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"{what}: activation must be one of {sorted(_ACTIVATIONS)}, got {activation!r}")
    return act


def _rows_ready(t: torch.Tensor, per16: int) -> torch.Tensor:
    """``t`` itself where its rows are what the kernels read (unit column stride, 16-byte aligned), else a copy."""
    rs, cs = t.stride()
    if cs == 1 and rs % per16 == 0 and rs >= t.shape[1] and t.data_ptr() % 16 == 0:
        return t  # (a single row's stride counts too: it goes into a tensor map)
    return t.clone(memory_format=torch.contiguous_format)


def _weights_ready(w_gate: torch.Tensor, w_up: torch.Tensor, per16: int, row_major: bool):
    """Both weights in one layout the kernels read: column-major, or row-major where that is allowed and they are."""
    k = w_gate.shape[0]
    (g0, g1), (u0, u1) = w_gate.stride(), w_up.stride()
    if g0 == u0 == 1 and g1 >= k and u1 >= k and (g1 | u1) % per16 == 0 and (w_gate.data_ptr() | w_up.data_ptr()) % 16 == 0:
        return w_gate, w_up
    if row_major and g1 == u1 == 1 and g0 != 1 and u0 != 1:
        return _rows_ready(w_gate, per16), _rows_ready(w_up, per16)
    return _rows_ready(w_gate.t(), per16).t(), _rows_ready(w_up.t(), per16).t()


def _launch(x, w_gate, w_up, out, act: int, dev: int, what: str, scales=None, mode: int = _lib.SCALE_NONE, saved=(None, None)):
    m, k = x.shape
    sx = sg = su = None
    if scales is not None:
        sx, sg, su = scales[0].data_ptr(), scales[1].data_ptr(), scales[2].data_ptr()
    code = _lib.load().hb200_gated_gemm(
        x.data_ptr(), w_gate.data_ptr(), w_up.data_ptr(), out.data_ptr(), m, out.shape[1], k, x.stride(0),
        *w_gate.stride(), *w_up.stride(), out.stride(0), _OUT_DT[x.dtype], _OUT_DT[out.dtype], act, sx, sg, su, mode, *saved,
        dev, _stream_ptr(dev),
    )
    if code:
        _lib.raise_for(code, what)
    return out


class _LivingNodes:
    """Weak references to backward nodes, for any number of threads: every access to the dictionary is one operation of its
    own (a WeakSet that is iterated while another thread adds to it raises)."""

    def __init__(self):
        self._refs = {}

    def add(self, node) -> None:
        key = id(node)  # not taken by another node before this one's reference has left
        self._refs[key] = weakref.ref(node, lambda _: self._refs.pop(key, None))

    def snapshot(self) -> list:
        nodes = (ref() for ref in self._refs.copy().values())
        return [n for n in nodes if n is not None]

    def __len__(self) -> int:
        return len(self._refs)


# Backward nodes of eager forward passes on the default stream that are still alive (see _refuse_capture).
_eager_nodes = _LivingNodes()


class _GatedMatmul(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, act):
        dev = x.get_device()
        x = _rows_ready(x, 8)
        w_gate, w_up = _weights_ready(w_gate, w_up, 8, True)
        m, f = x.shape[0], w_gate.shape[1]
        out = _empty_matrix(x, m, f, x.dtype)
        # u * act'(g) and act(g) in fp32: the gradients of g and u are then rounded once, as operands of their products
        saved = _empty_matrix(x, 2 * m, f, torch.float32)
        p = saved.data_ptr()
        _launch(x, w_gate, w_up, out, act, dev, "gated_matmul", saved=(p, p + 4 * m * f))
        ctx.save_for_backward(x, w_gate, w_up, saved)
        if _stream_ptr(dev) == 0:
            _eager_nodes.add(ctx)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dh):
        x, w_gate, w_up, saved = ctx.saved_tensors
        want_x, want_gate, want_up, _ = ctx.needs_input_grad
        m, k = x.shape
        f = w_gate.shape[1]
        dev = _require_cuda(dh, x)
        dh = _rows_ready(dh, 8)
        dx = dw_gate = dw_up = None
        if want_x:
            dx = _empty_matrix(x, m, k, x.dtype)
        if want_gate or want_up:
            strides = (1, k) if w_gate.stride(0) == 1 else (f, 1)
            dw_gate, dw_up = x.new_empty_strided((k, f), strides), x.new_empty_strided((k, f), strides)
        lib = _lib.load()
        bytes_ = lib.hb200_gated_gemm_backward_workspace_bytes(m, f, k)
        workspace = _empty_matrix(x, 1, bytes_, torch.uint8)
        p = saved.data_ptr()
        code = lib.hb200_gated_gemm_backward(
            dh.data_ptr(), x.data_ptr(), w_gate.data_ptr(), w_up.data_ptr(), p, p + 4 * m * f,
            None if dx is None else dx.data_ptr(), None if dw_gate is None else dw_gate.data_ptr(),
            None if dw_up is None else dw_up.data_ptr(), m, f, k, dh.stride(0), x.stride(0), *w_gate.stride(), *w_up.stride(),
            _OUT_DT[x.dtype], workspace.data_ptr(), bytes_, dev, _stream_ptr(dev),
        )
        if code:
            _lib.raise_for(code, "gated_matmul backward")
        return dx, dw_gate if want_gate else None, dw_up if want_up else None, None


def _reachable(nodes) -> set:
    """All nodes of the graphs below ``nodes``, these included."""
    seen, todo = set(), list(nodes)
    while todo:
        node = todo.pop()
        if node not in seen:
            seen.add(node)
            todo += [n for n, _ in node.next_functions if n is not None]
    return seen


def _refuse_capture(*inputs: torch.Tensor) -> None:
    """Refuses a capture that living eager graphs over the leaves below ``inputs`` would break.

    Autograd ties a leaf's gradient accumulator to the stream it was made on for as long as any graph over that leaf
    lives.  A backward pass under capture then waits on that stream, which CUDA forbids for the default one: the capture
    would be lost in the middle of the backward pass.  So it is refused here, before anything is recorded.
    """
    here = _reachable(torch.autograd.graph.get_gradient_edge(t).node for t in inputs if t.requires_grad)
    # (both sets keep their nodes' Python objects, so that one node is one object in both)
    if any(hasattr(n, "variable") for n in here & _reachable(_eager_nodes.snapshot())):
        raise RuntimeError(
            "gated_matmul: an eager graph over the same leaf tensors, made on the default stream, is still alive; "
            "a backward pass cannot be captured next to it. Drop its results first, or make it on another stream"
        )


def gated_matmul(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, *, activation: str = "silu") -> torch.Tensor:
    """``act(x @ w_gate) * (x @ w_up)`` for fp16 or bf16 ``x [M,K]`` and weights ``[K,F]``, with gradients.

    Both products, the activation (``"silu"``, ``"gelu"`` or ``"gelu_tanh"``) and the product run in one kernel with
    fp32 accumulation; the result has the operands' dtype, rounded once.  The weights may be column-major (a transposed
    view of ``[F, K]`` storage) or row-major, both in the same layout (else one is copied).  When a gradient is needed
    the forward pass also keeps two fp32 ``[M,F]`` tensors; the backward pass returns ``x``'s and the weights' gradients
    in their dtype, and is not differentiable itself.  It rounds ``dh * u * act'(g)`` and ``dh * act(g)`` to the operands'
    dtype (in fp16 scaled so that their largest value fits) before the products that give the gradients, and computes
    both weights' gradients where one is wanted.  Operands whose ``K`` or ``F`` is not a multiple of 8 are padded, that is
    copied, in every call.

    Both passes can be captured into a CUDA graph, unless an eager graph over the same leaf tensors, made by this
    function on the default stream, is alive: a call under capture that needs gradients is refused then.  (Other eager
    graphs over them, made on the default stream by other operations alone, break a captured backward pass just as
    they do without this function, and are not seen here.)
    """
    if not (x.dtype == w_gate.dtype == w_up.dtype) or x.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError(f"gated_matmul expects three float16 or three bfloat16 tensors, got {x.dtype}, {w_gate.dtype} and {w_up.dtype}")
    act = _check_gated(x, w_gate, w_up, activation, "gated_matmul")
    dev = _require_cuda(x, w_gate, w_up)
    m, k = x.shape
    f = w_gate.shape[1]
    if m == 0 or f == 0 or k == 0:
        return (x @ w_gate) * (x @ w_up)  # without elements, or zeros: act(0) = 0
    grad = torch.is_grad_enabled() and (x.requires_grad or w_gate.requires_grad or w_up.requires_grad)
    if grad and _eager_nodes and torch.cuda.is_current_stream_capturing():
        _refuse_capture(x, w_gate, w_up)
    kp, fp = _round_up(k, 8), _round_up(f, 8)
    if kp != k or fp != f:  # odd K or F: the same kernels on zero-padded copies; zero columns give act(0) * 0
        pad = torch.nn.functional.pad
        weights = (pad(w.t(), (0, kp - k, 0, fp - f)).t() for w in (w_gate, w_up))
        return gated_matmul(pad(x, (0, kp - k)), *weights, activation=activation)[:, :f]
    if grad:
        return _GatedMatmul.apply(x, w_gate, w_up, act)
    x = _rows_ready(x, 8)
    w_gate, w_up = _weights_ready(w_gate, w_up, 8, True)
    return _launch(x, w_gate, w_up, _empty_matrix(x, m, f, x.dtype), act, dev, "gated_matmul")


def _gated_scales(scale_x, scale_gate, scale_up, m: int, f: int, dev: int):
    """Validate the three scales; returns them as contiguous fp32 tensors with the C-ABI scale mode."""
    if scale_x is None or scale_gate is None or scale_up is None:
        if not (scale_x is None and scale_gate is None and scale_up is None):
            raise ValueError("gated_gemm: pass scale_x, scale_gate and scale_up, or none of them")
        return None, _lib.SCALE_NONE
    scales = (scale_x, scale_gate, scale_up)
    if not (scale_x.dtype == scale_gate.dtype == scale_up.dtype == torch.float32):
        raise TypeError("gated_gemm: scale_x, scale_gate and scale_up must be float32 tensors")
    if not (scale_x.get_device() == scale_gate.get_device() == scale_up.get_device() == dev):
        raise ValueError("gated_gemm: scale_x, scale_gate and scale_up must live on the inputs' device")
    columns = ((1, f), (f,))
    if scale_x.shape in ((m, 1), (m,)) and scale_gate.shape in columns and scale_up.shape in columns:
        if scale_x.is_contiguous() and scale_gate.is_contiguous() and scale_up.is_contiguous():
            return scales, _lib.SCALE_ROWWISE
        return tuple(s.contiguous() for s in scales), _lib.SCALE_ROWWISE
    if scale_x.numel() == scale_gate.numel() == scale_up.numel() == 1:
        return scales, _lib.SCALE_TENSOR
    raise ValueError(
        "gated_gemm: scales must be one element each, or [M,1]/[M], [1,F]/[F] and [1,F]/[F]; got "
        f"{tuple(scale_x.shape)}, {tuple(scale_gate.shape)} and {tuple(scale_up.shape)} for M={m}, F={f}"
    )


def gated_gemm(
    x: torch.Tensor,
    w_gate: torch.Tensor,
    w_up: torch.Tensor,
    *,
    scale_x: Optional[torch.Tensor] = None,
    scale_gate: Optional[torch.Tensor] = None,
    scale_up: Optional[torch.Tensor] = None,
    activation: str = "silu",
    out_dtype: torch.dtype = torch.bfloat16,
    out: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """``act(g) * u`` with ``g = (x @ w_gate) * scale_x * scale_gate`` and ``u`` likewise, for e4m3 or int8 operands.

    ``x [M,K]`` and the weights ``[K,F]`` share one 8-bit dtype (``float8_e4m3fn`` or ``int8``).  The fp32 scales (all
    three or none) are one element each, or one for each row of ``x`` (``[M, 1]`` / ``[M]``) and each column of the
    weights (``[1, F]`` / ``[F]``).  One kernel, ``g`` and ``u`` in fp32, one rounding to ``out_dtype`` (fp16, bf16 or
    fp32).  Weights are best column-major (a transposed view of ``[F, K]`` storage); row-major ones are re-laid out in
    every call, and so is everything where ``K`` is not a multiple of 16 or ``F`` not one of 8.  ``K`` is at most 131056
    for int8 operands.  Up to 128 rows of ``x`` run in a kernel that streams the weights.  The result has no gradient;
    ``out`` has unit column stride and rows at multiples of 16 bytes, and must not overlap the inputs.
    """
    if not (x.dtype == w_gate.dtype == w_up.dtype) or x.dtype not in (torch.float8_e4m3fn, torch.int8):
        raise TypeError(f"gated_gemm expects three float8_e4m3fn or three int8 tensors, got {x.dtype}, {w_gate.dtype} and {w_up.dtype}")
    act = _check_gated(x, w_gate, w_up, activation, "gated_gemm")
    if x.dtype == torch.int8 and x.shape[1] > _INT8_MAX_K:
        raise ValueError(f"gated_gemm: K must be at most {_INT8_MAX_K} for int8 operands (the sums are int32), got {x.shape[1]}")
    if out_dtype not in (torch.float16, torch.bfloat16, torch.float32):
        raise TypeError(f"gated_gemm out_dtype must be float16, bfloat16 or float32, got {out_dtype}")
    dev = _require_cuda(x, w_gate, w_up)
    m, k = x.shape
    f = w_gate.shape[1]
    scales, mode = _gated_scales(scale_x, scale_gate, scale_up, m, f, dev)
    given = out
    if out is None:
        out = _empty_matrix(x, m, f, out_dtype)
    elif out.dtype != out_dtype or tuple(out.shape) != (m, f) or out.stride(1) != 1 or out.device != x.device:
        raise ValueError("gated_gemm: `out` must be a row-major [M, F] tensor of out_dtype on the inputs' device")
    if m == 0 or f == 0:
        return out
    if k == 0:
        return out.zero_()
    kp, fp = _round_up(k, 16), _round_up(f, 8)
    if kp != k or fp != f:  # odd K or F: the same kernels on zero-padded copies
        xp = x.new_zeros((m, kp))
        xp[:, :k].copy_(x)
        padded = []
        for w in (w_gate, w_up):
            wp = w.new_zeros((fp, kp))
            wp[:f, :k].copy_(w.t())
            padded.append(wp.t())
        if mode == _lib.SCALE_ROWWISE:
            scales = (scales[0], *(torch.nn.functional.pad(s.reshape(f), (0, fp - f)) for s in scales[1:]))
        res = _empty_matrix(x, m, fp, out_dtype)
        out.copy_(_launch(xp, *padded, res, act, dev, "gated_gemm", scales, mode)[:, :f])
        return out
    x = _rows_ready(x, 16)
    w_gate, w_up = _weights_ready(w_gate, w_up, 16, False)
    _launch(x, w_gate, w_up, out, act, dev, "gated_gemm", scales, mode)
    if given is not None:
        _changed(given)
    return out
