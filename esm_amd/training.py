"""Operators for fine-tuning the trunk: LayerNorm, block-diagonal attention and a paired preference loss, each with its
gradient, on hand-written gfx950 kernels (include/esmk.h, "Training").

Every operator comes in two forms:
  * `layer_norm`, `attention_varlen`, `preference_loss`: differentiable, for torch's autograd;
  * `*_forward` / `*_backward`: the two halves as plain functions, for programs that schedule them by themselves.  Capture
    THESE into a HIP graph (after one call outside the capture); a captured autograd backward ties the graph to the
    autograd nodes that exist at capture time.
Tensors live on one GPU; work is enqueued on that GPU's current stream and nothing waits for it.  Outputs and scratch memory
come from torch's allocator.  Wrong shapes, types or devices raise ValueError / TypeError before anything is launched.

The reference differentiates its own modules (esm/layers/attention.py:26-33,65-78, esm/layers/blocks.py:31) through
autograd; the loss has no counterpart there.
"""
from __future__ import annotations

import ctypes as C

import torch
from torch.autograd.function import once_differentiable

from . import _lib as L

_DTYPES = {torch.float32: L.F32, torch.bfloat16: L.BF16}
_INT_MAX = 2 ** 31 - 1


class _On:
    """Make the tensor's GPU the current one while a call is enqueued; gives that GPU's current stream."""

    def __init__(self, device):
        self.device, self.guard = device, None

    def __enter__(self):
        if self.device.index != torch.cuda.current_device():
            self.guard = torch.cuda.device(self.device)
            self.guard.__enter__()
        return torch.cuda.current_stream(self.device).cuda_stream

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)


def _need(t, name, dtypes, device=None):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    if t.dtype not in dtypes:
        raise TypeError(f"{name} has dtype {t.dtype}, wanted {' or '.join(str(d) for d in dtypes)}")
    if not t.is_cuda:
        raise L.EsmkError(f"esm_amd runs on the GPU only: {name} is on {t.device} (there is no CPU path)")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, the other tensors on {device}")


def _rows(t, d):
    """t [..., d] -> (t with dense equally spaced rows, distance of its rows); copies only where no such view exists."""
    if t.dim() == 2 and t.stride(1) == 1 and t.stride(0) >= d:
        return t, t.stride(0)
    if not t.is_contiguous():
        t = t.contiguous()
    return t, d


# ---------------------------------------------------------------------------------------------- layer norm

def _check_norm(x, weight, bias):
    _need(x, "x", _DTYPES)
    _need(weight, "weight", _DTYPES, x.device)
    if x.dim() < 1 or x.shape[-1] < 1 or weight.shape != x.shape[-1:]:
        raise ValueError(f"weight {tuple(weight.shape)} does not fit x {tuple(x.shape)}")
    if x.shape[-1] > 12288:
        raise ValueError(f"rows of {x.shape[-1]} elements: at most 12288")
    if bias is not None:
        _need(bias, "bias", _DTYPES, x.device)
        if bias.shape != weight.shape:
            raise ValueError(f"bias {tuple(bias.shape)} does not fit x {tuple(x.shape)}")
    if x.numel() // x.shape[-1] > _INT_MAX:
        raise ValueError("too many rows")


def _param(t):
    return None if t is None else t.detach().to(torch.float32).contiguous()


def layer_norm_forward(x, weight, bias=None, eps: float = 1e-5):
    """LayerNorm over the last dimension -> (y, stats).  x [..., d] fp32 or bf16 (rows may be slices of wider ones);
    weight, bias [d].  y has x's shape and dtype; stats fp32 [rows, 2] (mean, 1 / sqrt(var + eps)) is what
    `layer_norm_backward` wants.  Statistics are fp32."""
    _check_norm(x, weight, bias)
    d = x.shape[-1]
    M = x.numel() // d
    xr, ld = _rows(x, d)
    w, b = _param(weight), _param(bias)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    stats = torch.empty((M, 2), dtype=torch.float32, device=x.device)
    with _On(x.device) as stream:
        L.check(L.lib().esmk_layernorm_fwd(xr.data_ptr(), _DTYPES[x.dtype], ld, w.data_ptr(), L.ptr(b), y.data_ptr(),
                                           stats.data_ptr(), M, d, eps, stream), "esmk_layernorm_fwd")
    return y, stats


def layer_norm_backward(dy, x, weight, stats, bias: bool = True, param_grads: bool = True):
    """Gradients of `layer_norm_forward` -> (dx, dweight, dbias).  dx has x's dtype, dweight and dbias are fp32 [d] sums over
    all rows; dbias is None without `bias`, both are None without `param_grads` (a frozen norm)."""
    _check_norm(x, weight, None)
    _need(dy, "dy", (x.dtype,), x.device)
    _need(stats, "stats", (torch.float32,), x.device)
    d = x.shape[-1]
    M = x.numel() // d
    if dy.shape != x.shape or stats.shape != (M, 2) or not stats.is_contiguous():
        raise ValueError(f"dy {tuple(dy.shape)} / stats {tuple(stats.shape)} do not fit x {tuple(x.shape)}")
    xr, ldx = _rows(x, d)
    gr, ldg = _rows(dy, d)
    w = _param(weight)
    dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    dw = torch.empty(d, dtype=torch.float32, device=x.device) if param_grads else None
    db = torch.empty(d, dtype=torch.float32, device=x.device) if param_grads and bias else None
    lib = L.lib()
    nbytes = lib.esmk_layernorm_bwd_workspace_bytes(M, d) if param_grads else 0
    ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device) if nbytes else None
    with _On(x.device) as stream:
        L.check(lib.esmk_layernorm_bwd(gr.data_ptr(), ldg, xr.data_ptr(), ldx, _DTYPES[x.dtype], w.data_ptr(),
                                       stats.data_ptr(), dx.data_ptr(), L.ptr(dw), L.ptr(db), L.ptr(ws), nbytes, M, d,
                                       stream), "esmk_layernorm_bwd")
    return dx, dw, db


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, stats = layer_norm_forward(x, weight, bias, eps)
        ctx.save_for_backward(x, weight, stats)
        ctx.bias_dtype = None if bias is None else bias.dtype
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, stats = ctx.saved_tensors
        want_w, want_b = ctx.needs_input_grad[1], ctx.needs_input_grad[2]
        dx, dw, db = layer_norm_backward(dy, x, weight, stats, bias=want_b, param_grads=want_w or want_b)
        return (dx if ctx.needs_input_grad[0] else None, dw.to(weight.dtype) if want_w else None,
                db.to(ctx.bias_dtype) if want_b else None, None)


def layer_norm(x, weight, bias=None, eps: float = 1e-5):
    """Differentiable LayerNorm over the last dimension (see `layer_norm_forward`)."""
    return _LayerNorm.apply(x, weight, bias, eps)


# ---------------------------------------------------------------------------------------------- attention

def _strided(t, what):
    """A [tokens, heads, head_dim] tensor the kernels can address: dense head_dim, 16-byte rows; a copy where it is not."""
    s = t.stride()
    if s[2] == 1 and s[0] % 8 == 0 and s[1] % 8 == 0 and t.shape[2] <= s[0] < 2 ** 23 and t.data_ptr() % 16 == 0:
        return t
    t = t.contiguous()
    if t.shape[1] * t.shape[2] >= 2 ** 23:
        raise ValueError(f"{what}: a token of {t.shape[1]} heads x {t.shape[2]} is too wide")
    return t


def _check_attention(q, k, v, cu_seqlens, key_mask):
    _need(q, "q", (torch.bfloat16,))
    for t, n in ((k, "k"), (v, "v")):
        _need(t, n, (torch.bfloat16,), q.device)
    if q.dim() != 3 or k.dim() != 3 or k.shape != v.shape or q.shape[0] != k.shape[0] or q.shape[2] != k.shape[2]:
        raise ValueError(f"q [N, H, D], k and v [N, G, D]: got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    N, H, D = q.shape
    if D not in (64, 128):
        raise ValueError(f"head dim {D}: 64 or 128")
    if H < 1 or k.shape[1] < 1 or H % k.shape[1]:
        raise ValueError(f"{k.shape[1]} key heads do not divide {H} query heads")
    if N > 2 ** 30:
        raise ValueError("too many tokens")
    _need(cu_seqlens, "cu_seqlens", (torch.int32,), q.device)
    if cu_seqlens.dim() != 1 or cu_seqlens.numel() < 1 or not cu_seqlens.is_contiguous():
        raise ValueError("cu_seqlens must be a dense vector of at least one offset")
    if key_mask is not None:
        _need(key_mask, "key_mask", (torch.bool, torch.uint8), q.device)
        if key_mask.shape != (N,) or not key_mask.is_contiguous():
            raise ValueError(f"key_mask must be a dense vector of {N} values, got {tuple(key_mask.shape)}")


def _scale(scale, D):
    scale = D ** -0.5 if scale is None else float(scale)
    if not 0.0 < scale < 1e30:
        raise ValueError(f"scale must be positive and finite, got {scale}")
    return scale


def attention_varlen_forward(q, k, v, cu_seqlens, scale: float | None = None, key_mask=None):
    """Bidirectional attention inside packed sequences -> (out, lse).

    q [N, H, D], k and v [N, G, D] bf16, D 64 or 128; G divides H (query head h reads key head h // (H // G)).  Any strides
    over tokens and heads (slices of a fused qkv buffer are read in place; layouts without 16-byte rows are copied).
    cu_seqlens int32 [n + 1] on the GPU: sequence s is tokens cu_seqlens[s] .. cu_seqlens[s + 1]; empty sequences are allowed,
    and tokens in no sequence get zeros.  key_mask bool [N]: False keys take no part, whatever they hold (a padded [B, L]
    batch is cu_seqlens = L * arange(B + 1), key_mask = tokens != pad).  A query without any key gets zeros.
    out bf16 [N, H, D]; lse fp32 [H, N] natural logs (-inf without a key).  scale defaults to D ** -0.5.  Products take bf16
    and sum in fp32; probabilities are rounded to bf16 for the product with v."""
    _check_attention(q, k, v, cu_seqlens, key_mask)
    N, H, D = q.shape
    scale = _scale(scale, D)
    q, k, v = _strided(q, "q"), _strided(k, "k"), _strided(v, "v")
    out = torch.empty((N, H, D), dtype=torch.bfloat16, device=q.device)
    lse = torch.empty((H, N), dtype=torch.float32, device=q.device)
    st = (C.c_int64 * 8)(*q.stride()[:2], *k.stride()[:2], *v.stride()[:2], *out.stride()[:2])
    with _On(q.device) as stream:
        L.check(L.lib().esmk_attn_varlen_fwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(), st,
                                             cu_seqlens.data_ptr(), cu_seqlens.numel() - 1, L.ptr(key_mask), N, H,
                                             k.shape[1], D, scale, stream), "esmk_attn_varlen_fwd")
    return out, lse


def attention_varlen_backward(dout, q, k, v, out, lse, cu_seqlens, scale: float | None = None, key_mask=None):
    """Gradients of `attention_varlen_forward` -> (dq, dk, dv), dense bf16 in the shapes of q, k and v.  out and lse are the
    forward call's, on the same inputs.  Probabilities and their gradients are rounded to bf16 for the products with q, k and
    dout; every sum is fp32, and shared key heads sum over their query heads in fp32."""
    _check_attention(q, k, v, cu_seqlens, key_mask)
    N, H, D = q.shape
    scale = _scale(scale, D)
    for t, n in ((dout, "dout"), (out, "out")):
        _need(t, n, (torch.bfloat16,), q.device)
        if t.shape != q.shape:
            raise ValueError(f"{n} {tuple(t.shape)} does not fit q {tuple(q.shape)}")
    _need(lse, "lse", (torch.float32,), q.device)
    if lse.shape != (H, N) or not lse.is_contiguous():
        raise ValueError(f"lse must be dense [{H}, {N}], got {tuple(lse.shape)}")
    dout, q, k, v, out = (_strided(t, n) for t, n in ((dout, "dout"), (q, "q"), (k, "k"), (v, "v"), (out, "out")))
    dq = torch.empty((N, H, D), dtype=torch.bfloat16, device=q.device)
    dk = torch.empty((N, k.shape[1], D), dtype=torch.bfloat16, device=q.device)
    dv = torch.empty_like(dk)
    lib = L.lib()
    nbytes = lib.esmk_attn_varlen_bwd_workspace_bytes(N, H)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
    st = (C.c_int64 * 16)(*(s for t in (dout, q, k, v, out, dq, dk, dv) for s in t.stride()[:2]))
    with _On(q.device) as stream:
        L.check(lib.esmk_attn_varlen_bwd(dout.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
                                         lse.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), st,
                                         cu_seqlens.data_ptr(), cu_seqlens.numel() - 1, L.ptr(key_mask), N, H, k.shape[1], D,
                                         scale, ws.data_ptr(), nbytes, stream), "esmk_attn_varlen_bwd")
    return dq, dk, dv


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, cu_seqlens, scale, key_mask):
        out, lse = attention_varlen_forward(q, k, v, cu_seqlens, scale, key_mask)
        ctx.save_for_backward(q, k, v, out, lse, cu_seqlens, key_mask)
        ctx.scale = scale
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, out, lse, cu_seqlens, key_mask = ctx.saved_tensors
        return (*attention_varlen_backward(dout, q, k, v, out, lse, cu_seqlens, ctx.scale, key_mask), None, None, None)


def attention_varlen(q, k, v, cu_seqlens, scale: float | None = None, key_mask=None):
    """Differentiable attention inside packed sequences (see `attention_varlen_forward`) -> out."""
    return _Attention.apply(q, k, v, cu_seqlens, scale, key_mask)


# ---------------------------------------------------------------------------------------------- preference loss

def _check_preference(logits, targets):
    _need(logits, "logits", _DTYPES)
    _need(targets, "targets", (torch.int64,), logits.device)
    if logits.dim() != 2 or logits.shape[1] < 1 or targets.shape != logits.shape[:1]:
        raise ValueError(f"logits [N, V] and targets [N]: got {tuple(logits.shape)}, {tuple(targets.shape)}")
    if logits.shape[0] > _INT_MAX or logits.shape[1] > 2 ** 30:
        raise ValueError("logits are too large")


def _dense16(t):
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def preference_loss_forward(logits, targets, cu_seqlens, ref_logps, beta: float = 0.1, label_smoothing: float = 0.0,
                            nll_weight: float = 0.0):
    """Preference loss of packed sequence pairs -> (loss, logps, saved).

    logits [N, V] fp32 or bf16 over the packed tokens; targets int64 [N], a value outside [0, V) marks a token that is not
    scored; cu_seqlens int32 [2 P + 1]: sequences 2i (preferred) and 2i + 1 (other) are pair i; ref_logps fp32 [2 P] the
    frozen model's log-probabilities.
        logps[s] = sum over scored tokens of log softmax(logits)[target]
        m_i = beta * ((logps - ref_logps)[2i] - (logps - ref_logps)[2i + 1])
        loss = mean_i (1 - label_smoothing) softplus(-m_i) + label_smoothing softplus(m_i)
                      - nll_weight * logps[2i] / max(1, scored tokens of 2i)
    loss fp32 scalar, logps fp32 [2 P]; `saved` is for `preference_loss_backward`.  Sums over tokens and pairs are 64-bit."""
    _check_preference(logits, targets)
    dev = logits.device
    _need(cu_seqlens, "cu_seqlens", (torch.int32,), dev)
    _need(ref_logps, "ref_logps", (torch.float32,), dev)
    P = (cu_seqlens.numel() - 1) // 2
    if cu_seqlens.dim() != 1 or P < 1 or cu_seqlens.numel() != 2 * P + 1 or not cu_seqlens.is_contiguous():
        raise ValueError("cu_seqlens must be a dense vector of 2 * pairs + 1 offsets, one pair at least")
    if ref_logps.shape != (2 * P,):
        raise ValueError(f"ref_logps {tuple(ref_logps.shape)}: wanted ({2 * P},)")
    if not 0.0 <= label_smoothing <= 1.0:
        raise ValueError(f"label_smoothing {label_smoothing} is outside [0, 1]")
    N, V = logits.shape
    z, y, ref = _dense16(logits), targets.contiguous(), ref_logps.contiguous()
    lib = L.lib()
    nbytes = lib.esmk_pref_loss_saved_bytes(N, P)
    saved = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    logps = torch.empty(2 * P, dtype=torch.float32, device=dev)
    loss = torch.empty((), dtype=torch.float32, device=dev)
    with _On(dev) as stream:
        L.check(lib.esmk_pref_loss_fwd(z.data_ptr(), _DTYPES[z.dtype], y.data_ptr(), cu_seqlens.data_ptr(), P, ref.data_ptr(),
                                       beta, label_smoothing, nll_weight, N, V, saved.data_ptr(), nbytes, logps.data_ptr(),
                                       loss.data_ptr(), stream), "esmk_pref_loss_fwd")
    return loss, logps, saved


def preference_loss_backward(logits, targets, saved, grad_loss=None):
    """Gradient of the loss with respect to the logits, in their dtype; tokens that are not scored get zeros.  `saved` is the
    forward call's, on the same inputs; grad_loss: fp32 scalar on the GPU (None = 1)."""
    _check_preference(logits, targets)
    N, V = logits.shape
    _need(saved, "saved", (torch.uint8,), logits.device)
    if saved.numel() < L.lib().esmk_pref_loss_saved_bytes(N, 0) or not saved.is_contiguous():
        raise ValueError("saved does not belong to these logits")
    if grad_loss is not None:
        _need(grad_loss, "grad_loss", (torch.float32,), logits.device)
        if grad_loss.numel() != 1:
            raise ValueError("grad_loss must be one value")
    z, y = _dense16(logits), targets.contiguous()
    dz = torch.empty((N, V), dtype=z.dtype, device=z.device)
    with _On(z.device) as stream:
        L.check(L.lib().esmk_pref_loss_bwd(z.data_ptr(), _DTYPES[z.dtype], y.data_ptr(), saved.data_ptr(), L.ptr(grad_loss),
                                           dz.data_ptr(), N, V, stream), "esmk_pref_loss_bwd")
    return dz


class _Preference(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, cu_seqlens, ref_logps, beta, label_smoothing, nll_weight):
        loss, logps, saved = preference_loss_forward(logits, targets, cu_seqlens, ref_logps, beta, label_smoothing, nll_weight)
        ctx.save_for_backward(logits, targets, saved)
        ctx.mark_non_differentiable(logps)
        return loss, logps

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_loss, _):
        logits, targets, saved = ctx.saved_tensors
        return (preference_loss_backward(logits, targets, saved, grad_loss),) + (None,) * 6


def preference_loss(logits, targets, cu_seqlens, ref_logps, beta: float = 0.1, label_smoothing: float = 0.0,
                    nll_weight: float = 0.0):
    """Differentiable preference loss (see `preference_loss_forward`) -> (loss, logps); logps carries no gradient."""
    return _Preference.apply(logits, targets, cu_seqlens, ref_logps, beta, label_smoothing, nll_weight)
