"""The operators of a decoding step, on torch tensors and torch's current stream.

The reference has no counterpart; they stand beside the kernels of
:mod:`hc_b200.workloads` (the int8 weight-only GEMM, the bf16 GEMM, the row
softmax) and go the same way: the native dispatcher checks the arguments, the
C-ABI (``include/hc_b200_kernels.h``, where the formulas are) picks a
precompiled sm_100a kernel.  Unlike the ``@kernel`` objects they launch
straight on the stream that is current when they are called, so that a call
costs one launch, is ordered with its neighbours by the stream alone and can
be captured into a CUDA graph.  Call an operator once before capturing it: its
kernel image is loaded at the first launch.
"""

from __future__ import annotations

import torch

from .hckernel.kernel import get_context

_native = None
_contexts = {}


def _launcher(t):
    """(native module, context, raw current stream) of the tensor's device."""
    global _native
    if _native is None:
        from ._native import _dispatcher

        _native = _dispatcher
    if not t.is_cuda:
        raise ValueError("hc_b200.serving: CUDA tensors expected, got one on the CPU")
    index = t.device.index
    ctx = _contexts.get(index)
    if ctx is None:
        ctx = _contexts[index] = get_context(f"cuda:{index}")
    return _native, ctx, torch._C._cuda_getCurrentRawStream(index)


def add_rms_norm(x, gain, residual=None, *, eps=1e-5, out_dtype=None, group=0, out=None,
                 scale=None, summed=None):
    """Root-mean-square norm of ``x + residual`` over the last axis.

    ``x`` [rows, cols] bfloat16 or float32, ``gain`` [cols] and ``residual`` of
    its type.  Returns ``(out, scale, summed)``: the normalised rows times the
    gain in ``x``'s type (``scale`` is then None), or with ``out_dtype``
    ``torch.int8`` / ``torch.float8_e4m3fn`` in 8 bits with one float32 scale
    per row and ``group`` columns (0: per row), ``scale`` [rows, groups];
    and the sum in ``x``'s type, None without a residual.  ``out``, ``scale``
    and ``summed`` may be given; ``summed`` may be the residual itself.
    """
    native, ctx, stream = _launcher(x)
    if out is None:
        out = torch.empty(x.shape, dtype=out_dtype or x.dtype, device=x.device)
    elif out_dtype is not None and out.dtype != out_dtype:
        raise TypeError(f"add_rms_norm: out is {out.dtype}, not {out_dtype}")
    if out.dtype == x.dtype:
        scale = None
    elif scale is None:
        cols = x.shape[-1]
        groups = -(-cols // group) if 0 < group < cols else 1
        scale = torch.empty((x.shape[0], groups), dtype=torch.float32, device=x.device)
    if summed is None and residual is not None:
        summed = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    native.add_rms_norm(ctx, x, gain, residual, summed, out, scale, group, eps, stream)
    return out, scale, summed


def gemm_w4(a, w, scale, zero=None, *, group, a_scale=None, a_group=0, out=None):
    """``out[m, n] = sum_k a[m, k] (u[n, k] - z[n, k // group]) s[n, k // group]``.

    ``w`` uint8 [N, ceil(K / 2)] holds u, two 4-bit numbers per byte along K
    (even k in the low half); ``scale`` bfloat16 or float32 and ``zero`` uint8
    (None: 8 throughout) are [N, ceil(K / group)], ``group`` a multiple of 32.
    ``a`` is bfloat16 [M, K], or int8 with ``a_scale`` float32 as
    :func:`add_rms_norm` returns them (``a_group``: its ``group``).  Returns
    ``out`` bfloat16 [M, N].

    Up to 64 rows stream the weights as they are.  More rows convert them to
    bfloat16 first, into scratch memory taken from torch's allocator for the
    length of the call, and run the bf16 GEMM.
    """
    native, ctx, stream = _launcher(a)
    m, k = a.shape
    n = w.shape[0]
    if out is None:
        out = torch.empty((m, n), dtype=torch.bfloat16, device=a.device)
    workspace = None
    if m > 64:
        need = native.w4_workspace_bytes(m, n, k, a.dtype == torch.int8)
        workspace = torch.empty(need, dtype=torch.uint8, device=a.device)
    native.gemm_w4(ctx, a, w, scale, zero, out, group, a_scale, a_group, workspace, stream)
    return out
