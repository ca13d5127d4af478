"""Operators of the transformer encoders in a training loss, as differentiable functions over the C ABI (include/asyrp.h).

The reference's loss runs an image and a text encoder around the DeltaBlock step (diffusion_latent.py:337-347, losses/clip_loss.py); their
attention and the seams between their residual blocks are the work there that is not a plain matrix product:
  packed_attention      attention over sequences packed behind each other, causal or not, with grouped key / value heads
  gated_residual_norm   norm behind a block, gate, residual sum with its scale, norm in front of the next block
Both run on the current stream of their tensors' device, keep nothing between calls, and may be captured into a graph.  Their gradients are those of one backward pass
(no forward mode, no second derivative), and they cannot be traced.  (As with any autograd function: while a
backward pass is captured, no graph of the same leaves that was built outside the capture may be alive.)
"""
import math

import torch
from torch.autograd import forward_ad

from . import _lib
from .engine import AsyrpDeviceError

_HALF = (torch.float16, torch.bfloat16)
_INT32 = (torch.int32,)
_TYPES = tuple(_lib.DTYPES)
_raw_stream = torch._C._cuda_getCurrentRawStream      # the current stream's handle (torch.cuda.current_stream() without its object)


def _refuse_tensor(t, name, device):
    if not (isinstance(t, torch.Tensor) and t.is_cuda):
        raise AsyrpDeviceError(f"{name} must be a CUDA(HIP) tensor — the operator has no CPU path")
    raise AsyrpDeviceError(f"{name} lives on {t.device}, the other arguments on cuda:{device}")


def _tensor(t, name, device, dtypes):
    """`t` is a tensor of cuda:`device` (None: of any) and of one of the types; returns its device's index."""
    d = t.get_device() if isinstance(t, torch.Tensor) else -1          # -1 on the CPU
    if d < 0 or (d != device and device is not None):
        _refuse_tensor(t, name, device)
    if t.dtype not in dtypes:
        raise ValueError(f"{name} must be one of {[str(v) for v in dtypes]}, got {t.dtype}")
    return d


def _refuse_transforms(name, tensors):
    """The kernels work through addresses: a tangent of an argument would be dropped, and a trace would hold the empty result alone."""
    if torch._C._get_tracing_state() is not None:
        raise RuntimeError(f"{name} cannot be traced")
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError(f"{name} has no forward-mode derivative")


def _ptr(t):
    return None if t is None else t.data_ptr()


# ---- attention ---------------------------------------------------------------------------------------------------------------------
def _strides(t):
    """(token, head) strides of `t` [tokens, heads, head_dim] where the kernels can read it in place: last axis contiguous, the others
    multiples of 8 values and rows at most 2^23 apart, 16-byte address; None elsewhere.  An axis of one has no stride of its own."""
    (n, h, d), (a, b, c) = t.shape, t.stride()
    if n <= 1:
        a = d
    if h <= 1:
        b = d
    return (a, b) if c == 1 and a > 0 and b > 0 and not (a | b) & 7 and a <= 1 << 23 and not t.data_ptr() & 15 else None


def _apart(out, so, t):
    """No value of `t` lies where `out` is written: their spans do not meet, or they take different columns of the same rows (or of the same heads' blocks).  What is
    not read in place is copied before."""
    st = _strides(t)
    if st is None:
        return True
    extent = lambda t, s, axes: sum((t.shape[i] - 1) * s[i] for i in axes) + t.shape[2]  # noqa: E731
    gap = (out.data_ptr() - t.data_ptr()) // t.element_size()
    if gap >= extent(t, st, (0, 1)) or -gap >= extent(out, so, (0, 1)):
        return True
    return any(so[i] == st[i] and extent(t, st, (1 - i,)) <= gap % so[i] <= so[i] - extent(out, so, (1 - i,)) for i in (0, 1))


def _readable(t):
    st = _strides(t)
    if st is not None:
        return t, st
    t = t.clone(memory_format=torch.contiguous_format)
    return t, _strides(t)


def _attention_forward(q, k, v, cu, causal, scale, out, train):
    q, sq = _readable(q)
    k, sk = _readable(k)
    v, sv = _readable(v)
    fill = out is None
    if fill:
        out = q.new_empty(q.shape)
    T, H, D = q.shape
    sums = q.new_empty((H, T, 2), dtype=torch.float32) if train else None
    rest = q.new_empty(q.shape) if train else None
    spec = (T, cu.shape[0] - 1, H, k.shape[1], D, causal, _lib.DTYPES[q.dtype], scale, *sq, *sk, *sv, *_strides(out))
    lib, device, packed = _lib.load(), q.get_device(), _lib.PACKED_ATTENTION.pack(*spec, 0, 0)
    words = lib.asyrp_packed_attention_workspace(packed, 0)
    if words < 0:
        _lib.check(words)
    ws = q.new_empty((words,), dtype=torch.float32) if words else None
    rc = lib.asyrp_packed_attention_forward(device, packed, q.data_ptr(), k.data_ptr(), v.data_ptr(), cu.data_ptr(),
                                                    out.data_ptr(), _ptr(sums), _ptr(rest), _ptr(ws), fill, _raw_stream(device))
    if rc:
        _lib.check(rc)
    return q, k, v, out, sums, rest, spec


class _PackedAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, cu, causal, scale):
        q, k, v, out, sums, rest, ctx.spec = _attention_forward(q, k, v, cu, causal, scale, None, True)
        ctx.save_for_backward(q, k, v, cu, out, sums, rest)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_out):
        q, k, v, cu, out, sums, rest = ctx.saved_tensors
        d_out, sd = _readable(d_out)
        dq, dk, dv = q.new_empty(q.shape), k.new_empty(k.shape), v.new_empty(v.shape)
        lib, device, spec = _lib.load(), q.get_device(), _lib.PACKED_ATTENTION.pack(*ctx.spec, *sd)
        words = lib.asyrp_packed_attention_workspace(spec, 1)
        if words < 0:
            _lib.check(words)
        ws = q.new_empty((max(4, words),), dtype=torch.float32)
        rc = lib.asyrp_packed_attention_backward(device, spec, q.data_ptr(), k.data_ptr(), v.data_ptr(), cu.data_ptr(), out.data_ptr(), sums.data_ptr(),
                                                 rest.data_ptr(), d_out.data_ptr(), ws.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), _raw_stream(device))
        if rc:
            _lib.check(rc)
        return dq, dk, dv, None, None, None


def packed_attention(q, k, v, cu_seqlens, *, causal=False, scale=None, out=None):
    """softmax(scale q k^T) v within each of the sequences that lie behind each other in the rows of q, k and v.

    q [tokens, heads, head_dim], k and v [tokens, kv_heads, head_dim] in float16 or bfloat16, head_dim a multiple of 8 up to 128, heads a multiple
    of kv_heads (head h reads key / value head h // (heads // kv_heads)).  Any strides; views whose last axis is contiguous and whose other strides are
    multiples of 8 values are read in place, others are copied.  cu_seqlens: int32 on the same device, sequences + 1 ascending
    offsets from 0; sequence i is rows cu_seqlens[i] .. cu_seqlens[i + 1] - 1 and may be empty.  (Its values stay on the device and are not checked
    there: others than these give no defined result, but nothing outside the tensors is touched.)  scale: 1 / sqrt(head_dim) by default.

    Returns [tokens, heads, head_dim].  Rows behind the last sequence are zero there and in the gradients.  `out` (without gradients only;
    the result's type and shape, laid out as q may be, beside q, k and v and not over them) takes the result and keeps what it holds in those rows.  Sums and softmax statistics are float32;
    probabilities, and in the backward pass those and the scores' gradients, are rounded to the inputs' type before they multiply (float16: under powers of two that keep small
    ones' bits).  A call with gradients keeps the result, as much again for its roundings, and two float32 per token and head until its backward pass.  A value that is not finite may reach every row of its own sequence, the
    rows before it included, and no other sequence.  Results do not depend on the order in which the card works."""
    device = _tensor(q, "q", None, _HALF)
    same = (q.dtype,)
    _tensor(k, "k", device, same)
    _tensor(v, "v", device, same)
    _tensor(cu_seqlens, "cu_seqlens", device, _INT32)
    if q.dim() != 3 or k.dim() != 3:
        raise ValueError(f"q and k must be [tokens, heads, head_dim], got {tuple(q.shape)} and {tuple(k.shape)}")
    T, H, D = q.shape
    if k.shape != v.shape or k.shape[0] != T or k.shape[2] != D:
        raise ValueError(f"k and v must be [{T}, kv_heads, {D}] alike, got {tuple(k.shape)} and {tuple(v.shape)}")
    if H < 1 or k.shape[1] < 1 or H % k.shape[1]:
        raise ValueError(f"{H} query heads are no multiple of {k.shape[1]} key / value heads")
    if D % 8 or not 8 <= D <= 128:
        raise ValueError(f"head_dim must be a multiple of 8 from 8 to 128, got {D}")
    if cu_seqlens.dim() != 1 or cu_seqlens.shape[0] < 2:
        raise ValueError(f"cu_seqlens must be a vector of at least two offsets, got shape {tuple(cu_seqlens.shape)}")
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if not 0.0 < scale < math.inf:
        raise ValueError(f"scale must be positive and finite, got {scale}")
    _refuse_transforms("packed_attention", (q, k, v, out))
    cu, causal = cu_seqlens.contiguous(), bool(causal)
    grad = torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)
    if out is not None:
        _tensor(out, "out", device, same)
        if grad or (out.requires_grad and torch.is_grad_enabled()):
            raise ValueError("out= takes part in no graph: call without it, or under torch.no_grad()")
        so = _strides(out)
        if out.shape != q.shape or so is None:
            raise ValueError(f"out must be {tuple(q.shape)} with its last axis contiguous, other strides multiples of 8 values and a 16-byte address")
        if T and not ((so[0] >= (H - 1) * so[1] + D or so[1] >= (T - 1) * so[0] + D) and _apart(out, so, q) and _apart(out, so, k) and _apart(out, so, v)):
            raise ValueError("out must not overlap itself, q, k or v")
    if grad:
        return _PackedAttention.apply(q, k, v, cu, causal, scale)
    result = _attention_forward(q, k, v, cu, causal, scale, out, False)[3]
    if out is not None and not out.is_inference():
        torch.autograd.graph.increment_version(out)          # what an earlier operation keeps of it for its backward is no longer there
    return result


# ---- the seam between two residual blocks ------------------------------------------------------------------------------------------------
_KINDS = {"layer": _lib.NORM_LAYER, "rms": _lib.NORM_RMS}


def _norm_forward(x, y, gate, w1, b1, w2, b2, spec, before, device, stats=None):
    h = x.new_empty(x.shape)
    n = y.new_empty(y.shape) if before else None
    rc = _lib.load().asyrp_residual_norm_forward(device, spec, x.data_ptr(), y.data_ptr(), _ptr(gate), _ptr(w1), _ptr(b1), _ptr(w2), _ptr(b2), h.data_ptr(),
                                                 _ptr(n), _ptr(stats), _raw_stream(device))
    if rc:
        _lib.check(rc)
    return h, n


class _GatedResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, y, gate, w1, b1, w2, b2, spec, before, device):
        stats = x.new_empty((x.shape[0], 4), dtype=torch.float32)
        h, n = _norm_forward(x, y, gate, w1, b1, w2, b2, spec, before, device, stats)
        ctx.save_for_backward(x, y, gate, w1, b1, w2, b2, stats)
        ctx.spec, ctx.device = spec, device
        ctx.set_materialize_grads(False)
        return h, n

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh, dn):
        if dh is None and dn is None:
            return (None,) * 10
        x, y, gate, w1, b1, w2, b2, stats = ctx.saved_tensors
        need, device = ctx.needs_input_grad, ctx.device
        dh, dn = None if dh is None else dh.contiguous(), None if dn is None else dn.contiguous()
        dx, dy = x.new_empty(x.shape) if need[0] else None, y.new_empty(y.shape) if need[1] else None
        # without rows every sum is empty; without a gradient of n, the norm in front of the next block takes no part
        empty = x.shape[0] == 0
        outs = [None if t is None or not n else t.new_zeros(t.shape) if empty or (k > 2 and dn is None) else t.new_empty(t.shape)
                for k, t, n in zip(range(5), (gate, w1, b1, w2, b2), need[2:7])]
        late = outs[3:] if dn is not None else (None, None)
        lib = _lib.load()
        words = lib.asyrp_residual_norm_workspace(ctx.spec)
        if words < 0:
            _lib.check(words)
        ws = x.new_empty((max(4, words),), dtype=torch.float32)
        rc = lib.asyrp_residual_norm_backward(device, ctx.spec, x.data_ptr(), y.data_ptr(), _ptr(gate), _ptr(w1), _ptr(b1), _ptr(w2), stats.data_ptr(), _ptr(dh),
                                              _ptr(dn), _ptr(dx), _ptr(dy), _ptr(outs[0]), _ptr(outs[1]), _ptr(outs[2]), _ptr(late[0]), _ptr(late[1]), ws.data_ptr(),
                                              _raw_stream(device))
        if rc:
            _lib.check(rc)
        return (dx, dy, *outs, None, None, None)


def _vector(t, name, width, device):
    if t is None:
        return None
    _tensor(t, name, device, _TYPES)
    if t.dim() != 1 or t.shape[0] != width:
        raise ValueError(f"{name} must be [{width}], got {tuple(t.shape)}")
    return t if t.dtype == torch.float32 and t.is_contiguous() else t.float().contiguous()


def gated_residual_norm(x, y, *, gate=None, residual_scale=1.0, kind="layer", after=None, before=(None, None), eps=1e-5):
    """(h, n) with h = residual_scale * x + gate * N_after(y) and n = N_before(h): what lies between a block's output y and the next block's input n.

    x [..., width] is the residual stream, y alike the block's output; float32, float16 or bfloat16, both of one type or x in float32.  width: 1 to 8192.
    after / before: None (no such norm; without `before` n is None) or (weight, bias), each None or [width].  kind: "layer"
    ((t - mean) / sqrt(var + eps)) or "rms" (t / sqrt(mean t^2 + eps)), for both norms.  gate: None, [width], or [gates, width] where gates divides the rows (the product of
    x's other dimensions) and row r takes gate row r // (rows / gates): one gate per image of a batch, or one per row.
    h has x's type, n has y's.  Statistics, the sum h that the second norm sees and the sums of the parameters' gradients are float32; h and n are rounded once.
    Gates, weights and biases of any of the three types; their gradients come back in it."""
    device = _tensor(x, "x", None, _TYPES)
    _tensor(y, "y", device, _TYPES)
    shape = x.shape
    if not shape or shape != y.shape:
        raise ValueError(f"x and y must have one shape of at least one dimension, got {tuple(shape)} and {tuple(y.shape)}")
    if x.dtype != y.dtype and x.dtype != torch.float32:
        raise ValueError(f"a stream in {x.dtype} takes a branch of the same type, got {y.dtype}")
    if kind not in _KINDS:
        raise ValueError(f"kind must be 'layer' or 'rms', got {kind!r}")
    width, rows = shape[-1], math.prod(shape[:-1])
    if not 1 <= width <= 8192:
        raise ValueError(f"the width must be 1 to 8192, got {width}")
    residual_scale, eps = float(residual_scale), float(eps)
    if not math.isfinite(residual_scale) or not math.isfinite(eps) or eps < 0:
        raise ValueError("residual_scale and eps must be finite, eps not negative")
    if gate is not None:
        _tensor(gate, "gate", device, _TYPES)
        if gate.dim() == 1:
            gate = gate[None]
        if gate.dim() != 2 or gate.shape[1] != width or gate.shape[0] < 1 or rows % gate.shape[0]:
            raise ValueError(f"gate must be [{width}] or [gates, {width}] with gates dividing {rows} rows, got {tuple(gate.shape)}")
        gate = gate.float().contiguous()
    if any(pair is not None and (not isinstance(pair, (tuple, list)) or len(pair) != 2) for pair in (after, before)):
        raise ValueError("after and before must be None or (weight, bias)")
    w1, b1 = (None, None) if after is None else (_vector(after[0], "after[0]", width, device), _vector(after[1], "after[1]", width, device))
    w2, b2 = (None, None) if before is None else (_vector(before[0], "before[0]", width, device), _vector(before[1], "before[1]", width, device))
    if len(shape) != 2:
        x, y = x.reshape(rows, width), y.reshape(rows, width)
    _refuse_transforms("gated_residual_norm", (x, y, gate, w1, b1, w2, b2))
    args = (x.contiguous(), y.contiguous(), gate, w1, b1, w2, b2)
    spec = _lib.RESIDUAL_NORM.pack(rows, 0 if gate is None else gate.shape[0], width, _KINDS[kind], after is not None, before is not None, _lib.DTYPES[x.dtype],
                                   _lib.DTYPES[y.dtype], residual_scale, eps)
    grad = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in args)
    h, n = (_GatedResidualNorm.apply if grad else _norm_forward)(*args, spec, before is not None, device)
    if len(shape) == 2:
        return h, n
    return h.view(shape), None if n is None else n.view(shape)
