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

The kernels on tcgen05 bound their waits; one that runs out (it never does while
the GPU works) leaves NaN in place of what was not computed, and a code that the
context's ``kernel_status()`` returns once the stream has been synchronised.

No operator has a backward pass.  A call whose inputs require gradients is refused
while gradients are recorded (call it under ``torch.no_grad()``): its results would
be cut from the graph without a word.
"""

from __future__ import annotations

import torch

from .hckernel.kernel import get_context

_native = None
_contexts = {}


def _forward_only(name, *tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise RuntimeError(f"{name}: no backward pass, but an argument requires gradients "
                                   "(call it under torch.no_grad())")


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
    _forward_only("add_rms_norm", x, gain, residual, out, summed)
    native, ctx, stream = _launcher(x)
    if out is None:
        out = torch.empty_like(x, dtype=out_dtype)
    elif out_dtype is not None and out.dtype != out_dtype:
        raise TypeError(f"add_rms_norm: out is {out.dtype}, not {out_dtype}")
    if out.dtype == x.dtype:
        scale = None
    elif scale is None:
        cols = x.shape[-1]
        groups = -(-cols // group) if 0 < group < cols else 1
        scale = x.new_empty((x.shape[0], groups), dtype=torch.float32)
    if summed is None and residual is not None:
        summed = torch.empty_like(x)
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

    Up to 8 rows that fit in shared memory (``include/hc_b200_kernels.h``:
    at ``K`` = 8192 in bfloat16 6 to 8, by ``group``) stream the weights as
    they are; more rows run on the tensor cores with the weights rounded to
    bfloat16, and int8 activations with several scales per row (``a_group``)
    too.  Scratch memory is taken from torch's allocator for the length of
    the call.
    """
    _forward_only("gemm_w4", a, scale, a_scale, out)
    native, ctx, stream = _launcher(a)
    m, k = a.shape
    n = w.shape[0]
    if out is None:
        out = a.new_empty((m, n), dtype=torch.bfloat16)
    workspace = None
    # (A single row may report any stride; an unaligned array counts as one of odd pitch.)
    lda = 1 if a.data_ptr() % 16 else max(a.stride(0), k)
    ldw = 1 if w.data_ptr() % 16 else max(w.stride(0), (k + 1) // 2)
    need = native.w4_workspace_bytes(ctx, m, n, k, group, lda, ldw, a.dtype == torch.int8)
    if need:
        workspace = a.new_empty(need, dtype=torch.uint8)
    native.gemm_w4(ctx, a, w, scale, zero, out, group, a_scale, a_group, workspace, stream)
    return out


class KvCache:
    """A paged 8-bit key/value cache with one scale per block of tokens and head.

    ``k`` and ``v`` [pages, heads, block, dim], int8 or float8_e4m3fn, in any
    layout with contiguous 16-byte aligned rows; ``k_scale`` and ``v_scale``
    float32 [pages, heads].  ``block`` is a multiple of 16 up to 256, ``dim``
    a multiple of 16 up to 256.  Which page holds which block of which
    sequence is the caller's table, given with every call.
    """

    def __init__(self, k, v, k_scale, v_scale):
        _forward_only("KvCache", k_scale, v_scale)
        native, ctx, _ = _launcher(k)
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self._native = native.KvCache(ctx, k, v, k_scale, v_scale)
        self._root = k.shape[3] ** -0.5

    @classmethod
    def empty(cls, pages, heads, block, dim, dtype=torch.float8_e4m3fn, device="cuda"):
        """A cache with nothing in it (blocks are written before they are read)."""
        k, v = (torch.zeros((pages, heads, block, dim), dtype=torch.int8,
                            device=device).view(dtype) for _ in range(2))
        scales = (torch.zeros((pages, heads), dtype=torch.float32, device=device)
                  for _ in range(2))
        return cls(k, v, *scales)


def kv_append(cache, k, v, table, lengths, starts=None, *, max_new=None):
    """Writes new keys and values into the cache.

    ``k``, ``v`` bfloat16 [tokens, heads, dim]; ``table`` int32 [seqs, width]
    the page of each block of each sequence; ``lengths`` int32 [seqs] the
    tokens of each sequence, the new ones included; ``starts`` int32
    [seqs + 1] where each sequence's rows begin (None: one row per sequence),
    with ``max_new`` at least the most new tokens of a sequence.  A block's
    scale grows to what its new tokens need (earlier tokens are rounded
    again); pages that several sequences share must not be written.
    """
    _forward_only("kv_append", k, v)
    native, ctx, stream = _launcher(k)
    native.kv_append(ctx, cache._native, k, v, table, lengths, starts,
                     -1 if max_new is None else max_new, stream)


_scratch = {}
_COUNTER_BYTES = 4096  # HC_KV_COUNTER_BYTES of the C-ABI


def _attention_workspace(native, ctx, device, stream):
    """Scratch of the attention, its counters zeroed: one per stream, and one of its own
    for every call that is being captured, so that graphs may run beside each other."""
    if torch.cuda.current_device() == device.index:
        capturing = torch.cuda.is_current_stream_capturing()
    else:
        with torch.cuda.device(device):  # (the question is about the current device's stream)
            capturing = torch.cuda.is_current_stream_capturing()
    key = (device.index, stream)
    buf = None if capturing else _scratch.get(key)
    if buf is None:
        buf = torch.empty(native.kv_attention_workspace_bytes(ctx), dtype=torch.uint8,
                          device=device)
        buf[:_COUNTER_BYTES].zero_()
        if not capturing:
            _scratch[key] = buf
    return buf


def kv_attention(cache, q, table, lengths, starts=None, *, max_new=None, scale=None, window=0,
                 out=None, return_lse=False):
    """Attention of the new tokens over the cache they were appended to.

    ``q`` bfloat16 [tokens, heads, dim] with a multiple of the cache's heads;
    ``table``, ``lengths``, ``starts``, ``max_new`` as for :func:`kv_append`.
    A token sees its own position and those before it, with ``window`` > 0 at
    most that many; ``scale`` defaults to ``dim ** -0.5``.  Returns ``out`` in
    ``q``'s shape, and with ``return_lse`` also the natural logarithm of each
    row's sum of exponentials, float32 [tokens, heads].  A row that sees
    nothing gives zeros and -inf; rows of no sequence are not written.
    """
    _forward_only("kv_attention", q, out)
    native, ctx, stream = _launcher(q)
    if out is None:
        out = torch.empty_like(q)
    lse = None
    if return_lse:
        lse = q.new_empty(q.shape[:2], dtype=torch.float32)
    native.kv_attention(ctx, cache._native, q, out, lse, table, lengths, starts,
                        -1 if max_new is None else max_new,
                        cache._root if scale is None else scale, window,
                        _attention_workspace(native, ctx, q.device, stream), stream)
    return (out, lse) if return_lse else out
