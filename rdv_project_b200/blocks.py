"""Operators of a conditioned image block: what stands between the
convolutions of ``conv.py`` in an image network, forward and backward.
The reference has none of them.

* ``group_norm(x, groups, weight, bias, eps, activation)``: group norm with
  an activation ("relu", "silu", "gelu") over channels-last maps
  ``[N, ..., C]`` -> rdvb_group_norm. ``group_norm_forward`` also returns the
  statistics that ``group_norm_backward`` takes.
* ``cross_attention(q, k, v, lengths, mask, scale)``: attention of positions
  ``q [B, Lq, heads, D]`` to an encoder's states ``k, v [B, Lk, kv_heads,
  D]`` -> rdvb_attention_forward. ``cross_attention_forward`` also returns the
  log sums that ``cross_attention_backward`` takes.
* ``dropout(x, p, seed, offset, residual)``: dropout whose mask comes from a
  counter and is never stored, with an optional residual added ->
  rdvb_dropout; ``dropout_backward`` recomputes the mask.
* ``GroupNormTensorOp`` and ``CrossAttentionTensorOp``: the first two as
  ``TensorOperation`` s (fp32 ``[rows, channels]``, one sample).

Elements are float32, float16 or bfloat16; results have their input's type,
sums and statistics are float32. 16-bit attention on the tensor cores rounds
probabilities and score gradients to that type before the products that take
them (float32 inputs, and 16-bit ones that the tensor cores do not take, keep
them in float32). The three main functions are
differentiable: where gradients are enabled and an input requires one, they
record themselves for torch's autograd, in reverse mode; inputs with a
forward-mode tangent are refused. Calls are asynchronous on the
current stream, with workspaces from torch's allocator.
"""
from __future__ import annotations

import math

import torch
from torch.autograd import forward_ad

from . import _native as N
from .core import RDVObject, _timed, as_device_tensor, current_device, stream_handle, wrap
from .tensor_ops import TensorOperation, _as_op_input, _f32_view

_DTYPES = {torch.float32: N.RDVB_F32, torch.float16: N.RDVB_F16, torch.bfloat16: N.RDVB_BF16}
_ACTIVATIONS = {None: N.RDVB_ACT_NONE, "relu": N.RDVB_ACT_RELU, "silu": N.RDVB_ACT_SILU, "gelu": N.RDVB_ACT_GELU}


def _tensor(x) -> torch.Tensor:
    """x on the current device (a CUDA tensor that is there is aliased)."""
    if isinstance(x, torch.Tensor) and x.is_cuda and x.get_device() == torch.cuda.current_device():
        return x
    current_device()
    return as_device_tensor(x)


def _workspace(nbytes: int, device):
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes > 0 else None


def _dense_like(t):
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _wants_grad(*tensors) -> bool:
    """Whether a call is to be recorded for its gradients. Forward-mode
    derivatives, which the kernels do not carry along, are refused."""
    tangents = forward_ad._current_level >= 0
    wants = False
    for t in tensors:
        if isinstance(t, RDVObject):
            t = t._tensor
        if tangents and isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError("the image block's operators have no forward-mode derivative")
        if getattr(t, "requires_grad", False):
            wants = True
    return wants and torch.is_grad_enabled()


# ---------------------------------------------------------------- group norm


def _channel_param(name, p, c):
    if p is None:
        return None
    p = _tensor(p)
    if p.dim() != 1 or p.shape[0] != c or p.dtype not in _DTYPES:
        raise ValueError(f"{name} must be [{c}] of float32, float16 or bfloat16, got {tuple(p.shape)} of {p.dtype}")
    return p.contiguous()


def _norm_args(x, groups, weight, bias, activation):
    x = _tensor(x).contiguous()
    if not (x.dim() >= 2):
        raise ValueError(f"x must be [N, ..., C], got {tuple(x.shape)}")
    if not (x.dtype in _DTYPES):
        raise ValueError(f"x must be float32, float16 or bfloat16, got {x.dtype}")
    c = x.shape[-1]
    if not (c > 0 and isinstance(groups, int) and groups > 0 and c % groups == 0):
        raise ValueError(f"groups ({groups}) must be a whole number that divides the channels ({c})")
    if not (activation in _ACTIVATIONS):
        raise ValueError(f"activation must be None, 'relu', 'silu' or 'gelu', got {activation!r}")
    w, b = _channel_param("weight", weight, c), _channel_param("bias", bias, c)
    if w is not None and b is not None and w.dtype != b.dtype:
        w, b = w.float(), b.float()
    kind = N.RDVB_F32 if w is None and b is None else _DTYPES[b.dtype if w is None else w.dtype]
    return x, w, b, kind, x.shape[0], math.prod(x.shape[1:-1]), c


def _group_norm(x, groups, weight, bias, eps, activation, want_stats):
    x, w, b, kind, n, rows, c = _norm_args(x, groups, weight, bias, activation)
    lib = N.lib()
    y = torch.empty_like(x)
    # a sample without rows has no statistics: zeros stand in their place
    stats = None
    if want_stats:
        stats = (torch.empty if rows else torch.zeros)((n, groups, 2), dtype=torch.float32, device=x.device)
    nbytes = lib.rdvb_group_norm_workspace_bytes(n, rows, c, groups, 0)
    ws = _workspace(nbytes, x.device)
    with _timed():
        N.check(lib.rdvb_group_norm(x.data_ptr(), _DTYPES[x.dtype], n, rows, c, groups, _ptr(w), _ptr(b), kind,
                                    _ACTIVATIONS[activation], eps, y.data_ptr(), _ptr(stats), _ptr(ws), nbytes,
                                    stream_handle()), "rdvb_group_norm")
    return y, stats


def group_norm_forward(x, groups: int, weight=None, bias=None, eps: float = 1e-5, activation=None):
    """(y, stats): group_norm(...) and its [N, groups, 2] means and reciprocal
    standard deviations, for group_norm_backward. Not recorded by autograd."""
    return _group_norm(x, groups, weight, bias, eps, activation, True)


def _as_param(grad, param):
    kind = getattr(param._tensor if isinstance(param, RDVObject) else param, "dtype", torch.float32)
    return grad if grad is None or kind not in _DTYPES else grad.to(kind)


def group_norm_backward(dy, x, stats, groups: int, weight=None, bias=None, activation=None):
    """(dx, dweight, dbias) of group_norm_forward's y for the gradient dy;
    dweight and dbias have their parameter tensor's type (float32 sums), None
    for a parameter that is None."""
    x, w, b, kind, n, rows, c = _norm_args(x, groups, weight, bias, activation)
    dy = _tensor(dy).contiguous()
    if not (dy.shape == x.shape and dy.dtype == x.dtype):
        raise ValueError("dy must have x's shape and type")
    stats = _tensor(stats).contiguous()
    if not (tuple(stats.shape) == (n, groups, 2) and stats.dtype == torch.float32):
        raise ValueError(f"stats must be float32 [{n}, {groups}, 2]")
    lib = N.lib()
    dx = torch.empty_like(x)
    dw = torch.empty(c, dtype=torch.float32, device=x.device) if w is not None else None
    db = torch.empty(c, dtype=torch.float32, device=x.device) if b is not None else None
    nbytes = lib.rdvb_group_norm_workspace_bytes(n, rows, c, groups, 1)
    ws = _workspace(nbytes, x.device)
    with _timed():
        N.check(lib.rdvb_group_norm_backward(
            dy.data_ptr(), x.data_ptr(), stats.data_ptr(), _DTYPES[x.dtype], n, rows, c, groups, _ptr(w), _ptr(b),
            kind, _ACTIVATIONS[activation], dx.data_ptr(), _ptr(dw), _ptr(db), _ptr(ws), nbytes, stream_handle()),
            "rdvb_group_norm_backward")
    return dx, _as_param(dw, weight), _as_param(db, bias)


class _GroupNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, groups, eps, activation):
        y, stats = group_norm_forward(x, groups, weight, bias, eps, activation)
        ctx.save_for_backward(x, weight, bias, stats)
        ctx.groups, ctx.activation = groups, activation
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, bias, stats = ctx.saved_tensors
        return (*group_norm_backward(dy, x, stats, ctx.groups, weight, bias, ctx.activation), None, None, None)


def group_norm(x, groups: int, weight=None, bias=None, eps: float = 1e-5, activation=None) -> torch.Tensor:
    """act(weight (x - mean) / sqrt(variance + eps) + bias) of channels-last x
    [N, ..., C], the mean and variance over each sample's positions and
    the C / groups channels of a group; weight, bias [C] or None."""
    if _wants_grad(x, weight, bias):
        return _GroupNorm.apply(_tensor(x), None if weight is None else _tensor(weight),
                                None if bias is None else _tensor(bias), groups, eps, activation)
    return _group_norm(x, groups, weight, bias, eps, activation, False)[0]


# ----------------------------------------------------------- cross attention


def _states(name, t):
    t = _tensor(t)
    if not (t.dim() == 4):
        raise ValueError(f"{name} must be [batch, positions, heads, D], got {tuple(t.shape)}")
    if not (t.dtype in _DTYPES):
        raise ValueError(f"{name} must be float32, float16 or bfloat16, got {t.dtype}")
    return t if t.stride(3) == 1 or t.shape[3] == 1 else t.contiguous()


def _key_lengths(lengths, b, lk):
    """lengths as the kernels take them: int32, dense. They clamp to [0, lk]
    themselves; here only types whose values could wrap are clamped."""
    kind = lengths.dtype
    if not (lengths.shape == (b,) and (kind == torch.int32 or not (
            kind.is_floating_point or kind.is_complex or kind == torch.bool))):
        raise ValueError(f"lengths must be whole numbers [{b}]")
    if kind == torch.int32:
        return lengths.contiguous()
    if kind in (torch.int64, torch.uint32, torch.uint64):
        wide = lengths.to(torch.int64)
        if kind == torch.uint64:  # 2**63 and more
            wide = wide.masked_fill(wide < 0, lk)
        lengths = wide.clamp(0, lk)
    return lengths.to(torch.int32).contiguous()


def _describe(q, k, v, lengths, mask, scale):
    """The rdvb_attention of a call, as bytes, and the tensors that it points into."""
    q, k, v = _states("q", q), _states("k", k), _states("v", v)
    b, lq, heads, d = q.shape
    lk, kv_heads = k.shape[1], k.shape[2]
    if not (k.shape == v.shape):
        raise ValueError(f"k and v must have one shape, got {tuple(k.shape)} and {tuple(v.shape)}")
    if not (k.shape[0] == b and k.shape[3] == d):
        raise ValueError(f"k and v must be [{b}, Lk, kv_heads, {d}], got {tuple(k.shape)}")
    if not (k.dtype == q.dtype and v.dtype == q.dtype):
        raise ValueError("q, k and v must have one type")
    if not (kv_heads > 0 and heads > 0 and heads % kv_heads == 0):
        raise ValueError(f"k's heads ({kv_heads}) must divide q's ({heads})")
    if lengths is not None:
        lengths = _key_lengths(_tensor(lengths), b, lk)
    if mask is not None:
        mask = _tensor(mask)
        if not (tuple(mask.shape) == (b, lk) and mask.dtype == torch.bool):
            raise ValueError(f"mask must be bool [{b}, {lk}]")
        mask = mask if mask.stride(1) == 1 or lk <= 1 else mask.contiguous()
    packed = N.ATTENTION_PACK(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), 0 if lengths is None else lengths.data_ptr(),
        0 if mask is None else mask.data_ptr(), 0 if mask is None else mask.stride(0),
        *q.stride()[:3], *k.stride()[:3], *v.stride()[:3], lq, lk, _DTYPES[q.dtype], b, heads, kv_heads, d,
        d ** -0.5 if scale is None else float(scale))
    return packed, (q, k, v, lengths, mask)


def _dense16(t):
    """t dense and 16-byte aligned, as the kernels read it."""
    t = _tensor(t).contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _cross_attention(q, k, v, lengths, mask, scale, want_lse):
    a, held = _describe(q, k, v, lengths, mask, scale)
    q = held[0]
    lib = N.lib()
    out = _dense_like(q)
    lse = torch.empty((q.shape[0], q.shape[2], q.shape[1]), dtype=torch.float32, device=q.device) if want_lse else None
    nbytes = lib.rdvb_attention_workspace_bytes(a, 0)
    ws = _workspace(nbytes, q.device)
    with _timed():
        N.check(lib.rdvb_attention_forward(a, out.data_ptr(), _ptr(lse), _ptr(ws), nbytes,
                                           stream_handle()), "rdvb_attention_forward")
    return out, lse


def cross_attention_forward(q, k, v, lengths=None, mask=None, scale=None):
    """(out, lse): cross_attention(...) and the float32 [B, heads, Lq] natural
    logs of the sums of exponentials, for cross_attention_backward. Not
    recorded by autograd."""
    return _cross_attention(q, k, v, lengths, mask, scale, True)


def cross_attention_backward(dout, q, k, v, out, lse, lengths=None, mask=None, scale=None):
    """(dq, dk, dv) of cross_attention_forward's out for the gradient dout,
    dense; dk and dv are summed over the query heads that share a key head and
    0 at states that no position attends to."""
    a, held = _describe(q, k, v, lengths, mask, scale)
    q, k = held[0], held[1]
    dout, out, lse = _dense16(dout), _dense16(out), _tensor(lse).contiguous()
    for name, t in (("dout", dout), ("out", out)):
        if not (t.shape == q.shape and t.dtype == q.dtype):
            raise ValueError(f"{name} must have q's shape and type")
    b, lq, heads = q.shape[:3]
    if not (tuple(lse.shape) == (b, heads, lq) and lse.dtype == torch.float32):
        raise ValueError(f"lse must be float32 [{b}, {heads}, {lq}]")
    lib = N.lib()
    dq, dk, dv = _dense_like(q), _dense_like(k), _dense_like(k)
    nbytes = lib.rdvb_attention_workspace_bytes(a, 1)
    ws = _workspace(nbytes, q.device)
    with _timed():
        N.check(lib.rdvb_attention_backward(
            a, dout.data_ptr(), out.data_ptr(), lse.data_ptr(), dq.data_ptr(), dk.data_ptr(),
            dv.data_ptr(), _ptr(ws), nbytes, stream_handle()), "rdvb_attention_backward")
    return dq, dk, dv


class _CrossAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lengths, mask, scale):
        out, lse = cross_attention_forward(q, k, v, lengths, mask, scale)
        ctx.save_for_backward(q, k, v, out, lse, lengths, mask)
        ctx.scale = scale
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        q, k, v, out, lse, lengths, mask = ctx.saved_tensors
        return (*cross_attention_backward(dout, q, k, v, out, lse, lengths, mask, ctx.scale), None, None, None)


def cross_attention(q, k, v, lengths=None, mask=None, scale=None) -> torch.Tensor:
    """softmax(scale q k^T) v of q [B, Lq, heads, D] against an encoder's
    states k, v [B, Lk, kv_heads, D], query head h reading key head h //
    (heads / kv_heads); D up to 256, scale None: D ** -0.5. A sample's
    positions attend to the states below lengths[sample] (whole numbers [B])
    where mask[sample] is True (bool [B, Lk]); with none of them the result is
    0. States outside them are not read. Any strides; views of a joint
    projection are read in place."""
    if _wants_grad(q, k, v):
        return _CrossAttention.apply(_tensor(q), _tensor(k), _tensor(v),
                                     None if lengths is None else _tensor(lengths),
                                     None if mask is None else _tensor(mask), scale)
    return _cross_attention(q, k, v, lengths, mask, scale, False)[0]


# ------------------------------------------------------------------- dropout


def _dropout(x, p, seed, offset, residual):
    x = _tensor(x).contiguous()
    if not (x.dtype in _DTYPES):
        raise ValueError(f"x must be float32, float16 or bfloat16, got {x.dtype}")
    p = float(p)
    if not (0.0 <= p and round(min(p, 2.0) * 2 ** 32) < 2 ** 32):
        raise ValueError(f"p must be in [0, 1 - 2**-32), got {p}")
    if not (isinstance(seed, int) and 0 <= seed < 2 ** 64):
        raise ValueError("seed must be a whole number in [0, 2**64)")
    if not (isinstance(offset, int) and 0 <= offset and offset + (x.numel() + 3) // 4 <= 2 ** 64):
        raise ValueError("offset must be a whole number >= 0 whose counters fit 64 bits")
    if residual is not None:
        residual = _tensor(residual).contiguous()
        if not (residual.shape == x.shape and residual.dtype == x.dtype):
            raise ValueError("residual must have x's shape and type")
    y = torch.empty_like(x)
    with _timed():
        N.check(N.lib().rdvb_dropout(x.data_ptr(), _ptr(residual), y.data_ptr(), _DTYPES[x.dtype], x.numel(), p, seed,
                                     offset, stream_handle()), "rdvb_dropout")
    return y


def dropout_backward(dy, p: float, seed: int, offset: int = 0) -> torch.Tensor:
    """The gradient of dropout(x, p, seed, offset) in x for the gradient dy."""
    return _dropout(dy, p, seed, offset, None)


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p, seed, offset):
        ctx.args = p, seed, offset
        return _dropout(x, p, seed, offset, residual)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        dx = dropout_backward(dy, *ctx.args) if ctx.needs_input_grad[0] else None
        return dx, dy if ctx.needs_input_grad[1] else None, None, None, None


def dropout(x, p: float, seed: int, offset: int = 0, residual=None) -> torch.Tensor:
    """residual + (x / (1 - p) where kept, else 0). Element i (in x's order) is
    kept iff word i % 4 of the Philox 4x32-10 block at counter offset + i // 4
    and key seed is at least round(p 2**32). A call uses (numel + 3) // 4
    counters: advance offset by as many for the next mask under one seed."""
    if _wants_grad(x, residual):
        return _Dropout.apply(_tensor(x), None if residual is None else _tensor(residual), p, seed, offset)
    return _dropout(x, p, seed, offset, residual)


# --------------------------------------------------------- tensor operations


class GroupNormTensorOp(TensorOperation):
    """group_norm of one sample x [rows, channels] (fp32)."""

    _TILE_ROWS = 1
    _TILE_COLS = 1

    def __init__(self, x, weight, bias, groups: int, activation=None, eps: float = 1e-5) -> None:
        data, shape, upstream = _as_op_input(x)
        assert len(shape) == 2, "GroupNormTensorOp requires a 2D (rows, channels) input"
        weight = weight if isinstance(weight, RDVObject) else wrap(weight)
        bias = bias if isinstance(bias, RDVObject) else wrap(bias)
        assert tuple(weight.shape) == (shape[1],), "weight must be [channels]"
        assert tuple(bias.shape) == (shape[1],), "bias must be [channels]"
        assert groups > 0 and shape[1] % groups == 0, f"groups ({groups}) must divide channels ({shape[1]})"
        assert activation in _ACTIVATIONS, "activation must be None, 'relu', 'silu' or 'gelu'"
        self.x_buf = data
        self.weight = weight
        self.bias = bias
        self.groups, self.activation, self.eps = groups, activation, eps
        self._upstream = upstream
        super().__init__(shape)

    def _run(self):
        x, w, b = _f32_view(self.x_buf), _f32_view(self.weight), _f32_view(self.bias)
        rows, c = x.shape
        lib = N.lib()
        nbytes = lib.rdvb_group_norm_workspace_bytes(1, rows, c, self.groups, 0)
        ws = _workspace(nbytes, x.device)
        N.check(lib.rdvb_group_norm(x.data_ptr(), N.RDVB_F32, 1, rows, c, self.groups, w.data_ptr(), b.data_ptr(),
                                    N.RDVB_F32, _ACTIVATIONS[self.activation], self.eps,
                                    self._result._tensor.data_ptr(), None, _ptr(ws), nbytes, stream_handle()),
                "rdvb_group_norm")


class CrossAttentionTensorOp(TensorOperation):
    """cross_attention of one sample: q [Lq, heads * D], k and v [Lk, kv_heads
    * D] (fp32), heads side by side in a row; kv_heads None: heads."""

    _TILE_ROWS = 1
    _TILE_COLS = 1

    def __init__(self, q, k, v, heads: int, kv_heads=None, scale=None) -> None:
        kv_heads = heads if kv_heads is None else kv_heads
        (self.q_buf, qs, up_q), (self.k_buf, ks, up_k), (self.v_buf, vs, up_v) = (_as_op_input(t) for t in (q, k, v))
        assert len(qs) == len(ks) == len(vs) == 2, "CrossAttentionTensorOp requires 2D (positions, channels) inputs"
        assert heads > 0 and kv_heads > 0 and heads % kv_heads == 0, \
            f"kv_heads ({kv_heads}) must divide heads ({heads})"
        assert qs[1] % heads == 0, f"q's own channels ({qs[1]}) must be a multiple of heads ({heads})"
        assert ks == vs, "k and v must share one shape"
        assert ks[1] == qs[1] // heads * kv_heads, "k's own channels must be kv_heads times q's channels per head"
        self.heads, self.kv_heads, self.scale = heads, kv_heads, scale
        ups = [u for u in (up_q, up_k, up_v) if u is not None]
        self._upstream = ups[0] if ups else None
        self._extra_upstreams = tuple(ups[1:])
        super().__init__(qs)

    def _run(self):
        q, k, v = (_f32_view(t) for t in (self.q_buf, self.k_buf, self.v_buf))
        a, _ = _describe(q.view(1, q.shape[0], self.heads, -1), k.view(1, k.shape[0], self.kv_heads, -1),
                         v.view(1, v.shape[0], self.kv_heads, -1), None, None, self.scale)
        lib = N.lib()
        nbytes = lib.rdvb_attention_workspace_bytes(a, 0)
        ws = _workspace(nbytes, q.device)
        N.check(lib.rdvb_attention_forward(a, self._result._tensor.data_ptr(), None, _ptr(ws), nbytes,
                                           stream_handle()), "rdvb_attention_forward")
