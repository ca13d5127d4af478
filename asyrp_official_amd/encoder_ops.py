"""Operators of the transformer encoders in a training loss, as differentiable functions over the C ABI (include/asyrp.h).

The reference's loss runs an image and a text encoder around the DeltaBlock step (diffusion_latent.py:337-347, losses/clip_loss.py); their
attention and the seams between their residual blocks are the work there that is not a plain matrix product:
  packed_attention      attention over sequences packed behind each other, causal or not, with grouped key / value heads
  gated_residual_norm   norm behind a block, gate, residual sum with its scale, norm in front of the next block
Both run on the current stream of their tensors' device, keep nothing between calls, and may be captured into a graph.
"""
import ctypes as C
import math

import torch

from . import _lib
from .engine import AsyrpDeviceError, _ptr


def _tensor(t, name, dtypes, dim=None):
    if not (isinstance(t, torch.Tensor) and t.is_cuda):
        raise AsyrpDeviceError(f"{name} must be a CUDA(HIP) tensor — the operator has no CPU path")
    if t.dtype not in dtypes:
        raise ValueError(f"{name} must be one of {[str(d) for d in dtypes]}, got {t.dtype}")
    if dim is not None and t.dim() != dim:
        raise ValueError(f"{name} must have {dim} dimensions, got shape {tuple(t.shape)}")
    return t


def _same_device(first, *named):
    for name, t in named:
        if t is not None and t.device != first.device:
            raise AsyrpDeviceError(f"{name} lives on {t.device}, the other arguments on {first.device}")


def _stream(t):
    return C.c_void_p(torch.cuda.current_stream(t.device).cuda_stream)


# ---- attention ---------------------------------------------------------------------------------------------------------------------
def _heads_layout(t):
    """`t` [tokens, heads, head_dim] as the kernels read it: last axis contiguous, other strides multiples of 8 values, 16-byte address.
    Views of a fused q|k|v projection are; anything else is copied.  A dimension of one has no stride of its own."""
    ok = t.stride(2) == 1 and t.data_ptr() % 16 == 0 and all(t.shape[d] <= 1 or (t.stride(d) % 8 == 0 and t.stride(d) > 0) for d in (0, 1))
    return t if ok else t.contiguous().clone() if t.is_contiguous() else t.contiguous()


def _strides(t):
    return tuple(t.stride(d) if t.shape[d] > 1 else t.shape[2] for d in (0, 1))


def _attention_struct(q, k, v, out, cu, causal, scale, dout=None):
    p = _lib.PackedAttention()
    p.tokens, p.sequences, p.heads, p.kv_heads, p.head_dim = q.shape[0], cu.shape[0] - 1, q.shape[1], k.shape[1], q.shape[2]
    p.causal, p.dtype, p.scale = int(causal), _lib.DTYPES[q.dtype], scale
    p.q_stride[:], p.k_stride[:], p.v_stride[:], p.out_stride[:] = _strides(q), _strides(k), _strides(v), _strides(out)
    if dout is not None:
        p.dout_stride[:] = _strides(dout)
    return p


def _attention_forward(q, k, v, cu, causal, scale, out, want_lse):
    q, k, v = _heads_layout(q), _heads_layout(k), _heads_layout(v)
    fresh = out is None
    if fresh:
        out = torch.empty(q.shape, device=q.device, dtype=q.dtype)
    lse = torch.empty((q.shape[1], q.shape[0]), device=q.device, dtype=torch.float32) if want_lse else None
    p = _attention_struct(q, k, v, out, cu, causal, scale)
    _lib.check(_lib.load().asyrp_packed_attention_forward(q.device.index, C.byref(p), _ptr(q), _ptr(k), _ptr(v), _ptr(cu), _ptr(out), _ptr(lse),
                                                          int(fresh), _stream(q)))
    return q, k, v, out, lse


class _PackedAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, cu, causal, scale):
        q, k, v, out, lse = _attention_forward(q, k, v, cu, causal, scale, None, True)
        ctx.save_for_backward(q, k, v, cu, out, lse)
        ctx.causal, ctx.scale = causal, scale
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_out):
        q, k, v, cu, out, lse = ctx.saved_tensors
        d_out = _heads_layout(d_out)
        dq, dk, dv = (torch.empty(t.shape, device=t.device, dtype=t.dtype) for t in (q, k, v))
        delta = torch.empty_like(lse)
        p = _attention_struct(q, k, v, out, cu, ctx.causal, ctx.scale, d_out)
        _lib.check(_lib.load().asyrp_packed_attention_backward(q.device.index, C.byref(p), _ptr(q), _ptr(k), _ptr(v), _ptr(cu), _ptr(out), _ptr(lse),
                                                               _ptr(d_out), _ptr(delta), _ptr(dq), _ptr(dk), _ptr(dv), _stream(q)))
        return dq, dk, dv, None, None, None


def packed_attention(q, k, v, cu_seqlens, *, causal=False, scale=None, out=None):
    """softmax(scale q k^T) v within each of the sequences that lie behind each other in the rows of q, k and v.

    q [tokens, heads, head_dim], k and v [tokens, kv_heads, head_dim] in float16 or bfloat16, head_dim a multiple of 8 up to 128, heads a multiple
    of kv_heads (head h reads key / value head h // (heads // kv_heads)).  Any strides; views whose last axis is contiguous and whose other strides are
    multiples of 8 values are read in place, others are copied.  cu_seqlens: int32 on the same device, sequences + 1 ascending
    offsets from 0; sequence i is rows cu_seqlens[i] .. cu_seqlens[i + 1] - 1 and may be empty.  (Its values stay on the device and are not checked
    there: others than these give no defined result, but nothing outside the tensors is touched.)  scale: 1 / sqrt(head_dim) by default.

    Returns [tokens, heads, head_dim].  Rows behind the last sequence are zero there and in the gradients.  `out` (without gradients only;
    the result's type and shape, laid out as q may be) takes the result and keeps what it holds in those rows.  Sums and softmax statistics are float32;
    probabilities are rounded to the inputs' type before they multiply v.  A value that is not finite may reach every row of its own sequence, the
    rows before it included, and no other sequence.  Results do not depend on the order in which the card works."""
    _tensor(q, "q", (torch.float16, torch.bfloat16), 3)
    _tensor(k, "k", (q.dtype,), 3)
    _tensor(v, "v", (q.dtype,), 3)
    _tensor(cu_seqlens, "cu_seqlens", (torch.int32,), 1)
    _same_device(q, ("k", k), ("v", v), ("cu_seqlens", cu_seqlens), ("out", out))
    T, H, D = q.shape
    if k.shape != v.shape or k.shape[0] != T or k.shape[2] != D:
        raise ValueError(f"k and v must be [{T}, kv_heads, {D}] alike, got {tuple(k.shape)} and {tuple(v.shape)}")
    if H < 1 or k.shape[1] < 1 or H % k.shape[1]:
        raise ValueError(f"{H} query heads are no multiple of {k.shape[1]} key / value heads")
    if D % 8 or not 8 <= D <= 128:
        raise ValueError(f"head_dim must be a multiple of 8 from 8 to 128, got {D}")
    if cu_seqlens.shape[0] < 2:
        raise ValueError("cu_seqlens needs at least two offsets")
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if not math.isfinite(scale):
        raise ValueError(f"scale must be finite, got {scale}")
    cu = cu_seqlens.detach().contiguous()
    grad = torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)
    if out is not None:
        _tensor(out, "out", (q.dtype,), 3)
        if grad:
            raise ValueError("out= takes part in no graph: call without it, or under torch.no_grad()")
        if out.shape != q.shape or _heads_layout(out) is not out:
            raise ValueError(f"out must be {tuple(q.shape)} with its last axis contiguous, other strides multiples of 8 values and a 16-byte address")
    if grad:
        return _PackedAttention.apply(q, k, v, cu, bool(causal), scale)
    return _attention_forward(q, k, v, cu, bool(causal), scale, out, False)[3]


# ---- the seam between two residual blocks ------------------------------------------------------------------------------------------------
_KINDS = {"layer": _lib.NORM_LAYER, "rms": _lib.NORM_RMS}


class _GatedResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, y, gate, w1, b1, w2, b2, kind, after, before, scale, eps, keep):
        p = _lib.ResidualNorm()
        p.rows, p.width, p.gates = x.shape[0], x.shape[1], 0 if gate is None else gate.shape[0]
        p.kind, p.after, p.before = _KINDS[kind], int(after), int(before)
        p.stream_dtype, p.branch_dtype, p.residual_scale, p.eps = _lib.DTYPES[x.dtype], _lib.DTYPES[y.dtype], scale, eps
        h = torch.empty(x.shape, device=x.device, dtype=x.dtype)
        n = torch.empty(y.shape, device=x.device, dtype=y.dtype) if before else None
        stats = torch.empty((x.shape[0], 4), device=x.device, dtype=torch.float32) if keep else None
        _lib.check(_lib.load().asyrp_residual_norm_forward(x.device.index, C.byref(p), _ptr(x), _ptr(y), _ptr(gate), _ptr(w1), _ptr(b1), _ptr(w2), _ptr(b2),
                                                           _ptr(h), _ptr(n), _ptr(stats), _stream(x)))
        if keep:
            ctx.save_for_backward(x, y, gate, w1, b1, w2, b2, stats)
            ctx.p = p
            ctx.set_materialize_grads(False)
        return h, n

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh, dn):
        if dh is None and dn is None:
            return (None,) * 13
        x, y, gate, w1, b1, w2, b2, stats = ctx.saved_tensors
        p, need = ctx.p, ctx.needs_input_grad
        dh, dn = (None if t is None else _rows_layout(t) for t in (dh, dn))
        dx, dy = (torch.empty(t.shape, device=t.device, dtype=t.dtype) if n else None for t, n in ((x, need[0]), (y, need[1])))
        # without a gradient of n, the norm in front of the next block takes no part: its parameters' gradients are zero
        zero = dn is None or x.shape[0] == 0
        outs = [None if t is None or not n else torch.zeros_like(t) if z else torch.empty_like(t)
                for t, n, z in ((gate, need[2], x.shape[0] == 0), (w1, need[3], x.shape[0] == 0), (b1, need[4], x.shape[0] == 0), (w2, need[5], zero), (b2, need[6], zero))]
        lib = _lib.load()
        words = lib.asyrp_residual_norm_workspace(C.byref(p))
        if words < 0:
            _lib.check(int(words))
        ws = torch.empty(max(4, words), device=x.device, dtype=torch.float32)
        _lib.check(lib.asyrp_residual_norm_backward(x.device.index, C.byref(p), _ptr(x), _ptr(y), _ptr(gate), _ptr(w1), _ptr(b1), _ptr(w2), _ptr(stats), _ptr(dh),
                                                    _ptr(dn), _ptr(dx), _ptr(dy), _ptr(outs[0]), _ptr(outs[1]), _ptr(outs[2]), None if zero else _ptr(outs[3]),
                                                    None if zero else _ptr(outs[4]), _ptr(ws), _stream(x)))
        return (dx, dy, *outs, None, None, None, None, None, None)


def _rows_layout(t):
    """Contiguous rows; a copy also where the address is odd for the type's 16-byte loads is not needed: such rows are read value by value."""
    return t.contiguous()


def _vector(t, name, width):
    _tensor(t, name, tuple(_lib.DTYPES))
    if tuple(t.shape) != (width,):
        raise ValueError(f"{name} must be [{width}], got {tuple(t.shape)}")
    return t.float().contiguous()


def gated_residual_norm(x, y, *, gate=None, residual_scale=1.0, kind="layer", after=None, before=(None, None), eps=1e-5):
    """(h, n) with h = residual_scale * x + gate * N_after(y) and n = N_before(h): what lies between a block's output y and the next block's input n.

    x [..., width] is the residual stream, y alike the block's output; float32, float16 or bfloat16, both of one type or x in float32.  width: 1 to 8192.
    after / before: None (no such norm; without `before` n is None) or (weight, bias), each None or [width].  kind: "layer"
    ((t - mean) / sqrt(var + eps)) or "rms" (t / sqrt(mean t^2 + eps)), for both norms.  gate: None, [width], or [gates, width] where gates divides the rows (the product of
    x's other dimensions) and row r takes gate row r // (rows / gates): one gate per image of a batch, or one per row.
    h has x's type, n has y's.  Statistics, the sum h that the second norm sees and the sums of the parameters' gradients are float32; h and n are rounded once.
    Gates, weights and biases of any of the three types; their gradients come back in it."""
    types = tuple(_lib.DTYPES)
    _tensor(x, "x", types)
    _tensor(y, "y", types)
    if x.dim() < 1 or x.shape != y.shape:
        raise ValueError(f"x and y must have one shape of at least one dimension, got {tuple(x.shape)} and {tuple(y.shape)}")
    if x.dtype != y.dtype and x.dtype != torch.float32:
        raise ValueError(f"a stream in {x.dtype} takes a branch of the same type, got {y.dtype}")
    if kind not in _KINDS:
        raise ValueError(f"kind must be 'layer' or 'rms', got {kind!r}")
    width, shape = x.shape[-1], x.shape
    if not 1 <= width <= 8192:
        raise ValueError(f"the width must be 1 to 8192, got {width}")
    residual_scale, eps = float(residual_scale), float(eps)
    if not math.isfinite(residual_scale) or not math.isfinite(eps) or eps < 0:
        raise ValueError("residual_scale and eps must be finite, eps not negative")
    rows = math.prod(shape[:-1])
    if gate is not None:
        _tensor(gate, "gate", types)
        if gate.dim() == 1:
            gate = gate[None]
        if gate.dim() != 2 or gate.shape[1] != width or gate.shape[0] < 1 or rows % gate.shape[0]:
            raise ValueError(f"gate must be [{width}] or [gates, {width}] with gates dividing {rows} rows, got {tuple(gate.shape)}")
        gate = gate.float().contiguous()
    pairs = []
    for name, wb in (("after", after), ("before", before)):
        if wb is not None and (not isinstance(wb, (tuple, list)) or len(wb) != 2):
            raise ValueError(f"{name} must be None or (weight, bias)")
        pairs += [None if t is None else _vector(t, f"{name}[{i}]", width) for i, t in enumerate(wb or (None, None))]
    _same_device(x, ("y", y), ("gate", gate), *((n, t) for n, t in zip(("after weight", "after bias", "before weight", "before bias"), pairs)))
    x2, y2 = _rows_layout(x.reshape(rows, width)), _rows_layout(y.reshape(rows, width))
    keep = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x2, y2, gate, *pairs))
    h, n = _GatedResidualNorm.apply(x2, y2, gate, *pairs, kind, after is not None, before is not None, residual_scale, eps, keep)
    return h.view(shape), None if n is None else n.view(shape)
