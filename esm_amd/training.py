"""Operators for fine-tuning: LayerNorm, block-diagonal attention and a paired preference loss, each with its gradient, on
hand-written gfx950 kernels (include/esmk.h, "Training").

Every operator comes in two forms:
  * `layer_norm`, `attention_varlen`, `preference_loss`: differentiable, for torch's autograd;
  * `*_forward` / `*_backward`: the two halves as plain functions, for programs that schedule them by themselves.  Capture
    THESE into a HIP graph (after one call outside the capture); a captured autograd backward ties the graph to the
    autograd nodes that exist at capture time.
Tensors live on one GPU; work is enqueued on that GPU's current stream and nothing waits for it.  Outputs and scratch memory
come from torch's allocator.  Wrong shapes, types or devices raise ValueError / TypeError before anything is launched.

The models' own forward passes keep no graph: a program that trains writes its blocks from these operators and torch's.  The
reference differentiates its own modules (esm/layers/attention.py:26-33,65-78, esm/layers/blocks.py:31) through autograd; the
loss has no counterpart there.
"""
from __future__ import annotations

import ctypes as C

import torch
from torch.autograd.function import once_differentiable

from . import _lib as L

_DTYPES = {torch.float32: L.F32, torch.bfloat16: L.BF16}
_F32, _BF16, _I32, _I64, _U8 = (torch.float32,), (torch.bfloat16,), (torch.int32,), (torch.int64,), (torch.uint8,)
_MASK = (torch.bool, torch.uint8)
_Strides8, _Strides16 = C.c_int64 * 8, C.c_int64 * 16
Tensor, _DENSE = torch.Tensor, torch.contiguous_format


def _public_stream(gpu):
    return torch.cuda.current_stream(gpu).cuda_stream


# The current stream's handle.  torch's compiler-facing call spares the Stream object around it, 1 us of a small operator's 8 on the
# host; a torch without that call is asked the public way.
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _public_stream)


def _need(t, name, dtypes, gpu=None):
    """`t` has to be a tensor of one of `dtypes` on a GPU (on that one, if given)."""
    if isinstance(t, Tensor) and t.dtype in dtypes and t.is_cuda and (gpu is None or t.get_device() == gpu):
        return
    if not isinstance(t, Tensor):
        raise TypeError(f"{name} must be a tensor")
    if t.dtype not in dtypes:
        raise TypeError(f"{name} has dtype {t.dtype}, wanted {' or '.join(str(d) for d in dtypes)}")
    if not t.is_cuda:
        raise L.EsmkError(f"esm_amd runs on the GPU only: {name} is on {t.device} (there is no CPU path)")
    raise ValueError(f"{name} is on {t.device}, the other tensors on cuda:{gpu}")


def _call(gpu, name, *args):
    """One C entry point on the tensors' GPU and its current stream."""
    if gpu == torch.cuda.current_device():
        rc = getattr(L.lib(), name)(*args, _stream(gpu))
    else:
        with torch.cuda.device(gpu):
            rc = getattr(L.lib(), name)(*args, _stream(gpu))
    if rc:
        L.check(rc, name)


def _rows(t, d):
    """t [..., d] -> (t with dense equally spaced rows, distance of its rows); copies only where the rows are not dense or do not
    lie at one distance.  Slices [..., :d] of wider activations do, whatever their number of dimensions."""
    if t.is_contiguous():
        return t, d
    if t.stride(-1) == 1:
        ld = after = None  # distance of the rows, and what the next dimension's stride has to be
        for n, stride in zip(t.shape[-2::-1], t.stride()[-2::-1]):
            if n == 1:
                continue
            if ld is None:
                ld = stride
            elif stride != after:
                break
            after = stride * n
        else:
            if ld is not None and ld >= d:
                return t, ld
    return t.contiguous(), d


# ---------------------------------------------------------------------------------------------- layer norm

def _check_norm(x, weight, bias):
    _need(x, "x", _DTYPES)
    gpu, shape = x.get_device(), x.shape
    _need(weight, "weight", _DTYPES, gpu)
    if not shape or shape[-1] < 1 or weight.shape != shape[-1:]:
        raise ValueError(f"weight {tuple(weight.shape)} does not fit x {tuple(shape)}")
    d = shape[-1]
    if d > 12288:
        raise ValueError(f"rows of {d} elements: at most 12288")
    if bias is not None:
        _need(bias, "bias", _DTYPES, gpu)
        if bias.shape != weight.shape:
            raise ValueError(f"bias {tuple(bias.shape)} does not fit x {tuple(shape)}")
    M = x.numel() // d
    if M > 2 ** 30:
        raise ValueError("too many rows")
    return gpu, shape, M, d


def _param(t):
    return t if t.dtype is torch.float32 and t.is_contiguous() else t.detach().float().contiguous()


def layer_norm_forward(x, weight, bias=None, eps: float = 1e-5):
    """LayerNorm over the last dimension -> (y, stats).  x [..., d] fp32 or bf16 (rows may be slices of wider ones);
    weight, bias [d].  y has x's shape and dtype; stats fp32 [rows, 2] (mean, 1 / sqrt(var + eps)) is what
    `layer_norm_backward` wants.  Statistics are fp32."""
    gpu, shape, M, d = _check_norm(x, weight, bias)
    xr, ld = _rows(x, d)
    w, b = _param(weight), None if bias is None else _param(bias)
    y, stats = torch.empty_like(x, memory_format=_DENSE), w.new_empty((M, 2))
    _call(gpu, "esmk_layernorm_fwd", xr.data_ptr(), _DTYPES[x.dtype], ld, w.data_ptr(), None if b is None else b.data_ptr(),
          y.data_ptr(), stats.data_ptr(), M, d, eps)
    return y, stats


def layer_norm_backward(dy, x, weight, stats, bias: bool = True, param_grads: bool = True, input_grad: bool = True):
    """Gradients of `layer_norm_forward` -> (dx, dweight, dbias).  dx has x's dtype, dweight and dbias are fp32 [d] sums over
    all rows; dbias is None without `bias`, both are None without `param_grads` (a frozen norm), dx is None without `input_grad`
    (a norm of fixed inputs)."""
    gpu, shape, M, d = _check_norm(x, weight, None)
    _need(dy, "dy", (x.dtype,), gpu)
    _need(stats, "stats", _F32, gpu)
    if dy.shape != shape or stats.shape != (M, 2) or not stats.is_contiguous():
        raise ValueError(f"dy {tuple(dy.shape)} / stats {tuple(stats.shape)} do not fit x {tuple(shape)}")
    xr, ldx = _rows(x, d)
    gr, ldg = _rows(dy, d)
    w = _param(weight)
    if not (input_grad or param_grads):
        return None, None, None
    dx = torch.empty_like(x, memory_format=_DENSE) if input_grad else None
    dw = w.new_empty(d) if param_grads else None
    db = w.new_empty(d) if param_grads and bias else None
    nbytes = L.lib().esmk_layernorm_bwd_workspace_bytes(M, d) if param_grads else 0
    ws = w.new_empty(nbytes // 4) if nbytes else None
    _call(gpu, "esmk_layernorm_bwd", gr.data_ptr(), ldg, xr.data_ptr(), ldx, _DTYPES[x.dtype], w.data_ptr(), stats.data_ptr(),
          None if dx is None else dx.data_ptr(), None if dw is None else dw.data_ptr(), None if db is None else db.data_ptr(),
          None if ws is None else ws.data_ptr(), nbytes, M, d)
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
        want_x, want_w, want_b = ctx.needs_input_grad[:3]
        dx, dw, db = layer_norm_backward(dy, x, weight, stats, bias=want_b, param_grads=want_w or want_b, input_grad=want_x)
        return dx, dw.to(weight.dtype) if want_w else None, db.to(ctx.bias_dtype) if want_b else None, None


def layer_norm(x, weight, bias=None, eps: float = 1e-5):
    """Differentiable LayerNorm over the last dimension (see `layer_norm_forward`)."""
    return _LayerNorm.apply(x, weight, bias, eps)


# ---------------------------------------------------------------------------------------------- attention

def _strided(t, what):
    """A [tokens, heads, head_dim] tensor the kernels can address (dense head_dim, 16-byte rows; a copy where it is not), its
    address and its token and head strides."""
    tok, head, dim = t.stride()
    at = t.data_ptr()
    if dim != 1 or tok % 8 or head % 8 or at % 16 or not t.shape[2] <= tok < 2 ** 23:
        t = t.clone(memory_format=_DENSE)  # contiguous() would keep an unaligned dense tensor, or one token's odd strides
        if t.shape[1] * t.shape[2] >= 2 ** 23:
            raise ValueError(f"{what}: a token of {t.shape[1]} heads x {t.shape[2]} is too wide")
        tok, head, dim = t.stride()
        at = t.data_ptr()
    return t, at, tok, head


def _check_attention(q, k, v, cu_seqlens, key_mask):
    _need(q, "q", _BF16)
    gpu = q.get_device()
    _need(k, "k", _BF16, gpu)
    _need(v, "v", _BF16, gpu)
    qs, ks = q.shape, k.shape
    if len(qs) != 3 or len(ks) != 3 or ks != v.shape or qs[0] != ks[0] or qs[2] != ks[2]:
        raise ValueError(f"q [N, H, D], k and v [N, G, D]: got {tuple(qs)}, {tuple(ks)}, {tuple(v.shape)}")
    N, H, D = qs
    G = ks[1]
    if D != 64 and D != 128:
        raise ValueError(f"head dim {D}: 64 or 128")
    if H < 1 or G < 1 or H % G:
        raise ValueError(f"{G} key heads do not divide {H} query heads")
    if N > 2 ** 30:
        raise ValueError("too many tokens")
    _need(cu_seqlens, "cu_seqlens", _I32, gpu)
    if cu_seqlens.dim() != 1 or cu_seqlens.numel() < 1 or not cu_seqlens.is_contiguous():
        raise ValueError("cu_seqlens must be a dense vector of at least one offset")
    if key_mask is not None:
        _need(key_mask, "key_mask", _MASK, gpu)
        if key_mask.shape != (N,) or not key_mask.is_contiguous():
            raise ValueError(f"key_mask must be a dense vector of {N} values, got {tuple(key_mask.shape)}")
    return gpu, N, H, G, D


def _scale(scale, D):
    scale = D ** -0.5 if scale is None else float(scale)
    if not 1e-30 < scale < 1e30:
        raise ValueError(f"scale must be positive and finite (1e-30 .. 1e30), got {scale}")
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
    gpu, N, H, G, D = _check_attention(q, k, v, cu_seqlens, key_mask)
    scale = _scale(scale, D)
    (q, qp, qt, qh), (k, kp, kt, kh), (v, vp, vt, vh) = _strided(q, "q"), _strided(k, "k"), _strided(v, "v")
    out = torch.empty_like(q, memory_format=_DENSE)
    lse = q.new_empty((H, N), dtype=torch.float32)
    _call(gpu, "esmk_attn_varlen_fwd", qp, kp, vp, out.data_ptr(), lse.data_ptr(),
          _Strides8(qt, qh, kt, kh, vt, vh, H * D, D), cu_seqlens.data_ptr(), cu_seqlens.numel() - 1,
          None if key_mask is None else key_mask.data_ptr(), N, H, G, D, scale)
    return out, lse


def attention_varlen_backward(dout, q, k, v, out, lse, cu_seqlens, scale: float | None = None, key_mask=None,
                              kv_grads: bool = True):
    """Gradients of `attention_varlen_forward` -> (dq, dk, dv), dense bf16 in the shapes of q, k and v; dk and dv are None without
    `kv_grads` (fixed keys and values).  out and lse are the forward call's, on the same inputs.  Probabilities and their
    gradients are rounded to bf16 for the products with q, k and dout; every sum is fp32, and shared key heads sum over their
    query heads in fp32.  Sequences of at most 64 unmasked keys lose nothing of dq and dk but the rounding of the results:
    rowsum(dout out) is summed without the rounding of out, and the gradients of the probabilities enter in two bf16 parts.  That
    depends on a sequence's own keys, not on padding or on the rest of the call.  From 65 to 512 unmasked keys the two parts are
    used in small calls alone (about 256 blocks of 128 tokens, heads counted): dq and dk are then off by 1.8e-3 of their norm
    instead of 2.5e-3, so that a sequence's gradients are a little less exact in a larger batch."""
    gpu, N, H, G, D = _check_attention(q, k, v, cu_seqlens, key_mask)
    scale = _scale(scale, D)
    _need(dout, "dout", _BF16, gpu)
    _need(out, "out", _BF16, gpu)
    _need(lse, "lse", _F32, gpu)
    if dout.shape != q.shape or out.shape != q.shape:
        raise ValueError(f"dout {tuple(dout.shape)} / out {tuple(out.shape)} do not fit q {tuple(q.shape)}")
    if lse.shape != (H, N) or not lse.is_contiguous():
        raise ValueError(f"lse must be dense [{H}, {N}], got {tuple(lse.shape)}")
    dout, gp, gt, gh = _strided(dout, "dout")
    (q, qp, qt, qh), (k, kp, kt, kh), (v, vp, vt, vh) = _strided(q, "q"), _strided(k, "k"), _strided(v, "v")
    out, op, ot, oh = _strided(out, "out")
    dq = torch.empty_like(q, memory_format=_DENSE)
    dk, dv = (torch.empty_like(t, memory_format=_DENSE) if kv_grads else None for t in (k, v))
    nbytes = L.lib().esmk_attn_varlen_bwd_workspace_bytes(N, H)
    ws = lse.new_empty(nbytes // 4)
    _call(gpu, "esmk_attn_varlen_bwd", gp, qp, kp, vp, op, lse.data_ptr(), dq.data_ptr(),
          None if dk is None else dk.data_ptr(), None if dv is None else dv.data_ptr(),
          _Strides16(gt, gh, qt, qh, kt, kh, vt, vh, ot, oh, H * D, D, G * D, D, G * D, D), cu_seqlens.data_ptr(),
          cu_seqlens.numel() - 1, None if key_mask is None else key_mask.data_ptr(), N, H, G, D, scale, ws.data_ptr(), nbytes)
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
        return (*attention_varlen_backward(dout, q, k, v, out, lse, cu_seqlens, ctx.scale, key_mask,
                                           kv_grads=any(ctx.needs_input_grad[1:3])), None, None, None)


def attention_varlen(q, k, v, cu_seqlens, scale: float | None = None, key_mask=None):
    """Differentiable attention inside packed sequences (see `attention_varlen_forward`) -> out."""
    return _Attention.apply(q, k, v, cu_seqlens, scale, key_mask)


# ---------------------------------------------------------------------------------------------- preference loss

def _check_preference(logits, targets):
    _need(logits, "logits", _DTYPES)
    gpu, shape = logits.get_device(), logits.shape
    _need(targets, "targets", _I64, gpu)
    if len(shape) != 2 or shape[1] < 1 or targets.shape != shape[:1]:
        raise ValueError(f"logits [N, V] and targets [N]: got {tuple(shape)}, {tuple(targets.shape)}")
    if shape[0] >= 2 ** 26 or shape[1] > 2 ** 30:
        raise ValueError("logits are too large")
    return gpu, shape[0], shape[1]


def _dense16(t):
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def preference_loss_forward(logits, targets, cu_seqlens, ref_logps, beta: float = 0.1, label_smoothing: float = 0.0,
                            nll_weight: float = 0.0):
    """Preference loss of packed sequence pairs -> (loss, logps, saved).

    logits [N, V] fp32 or bf16 over the packed tokens (copied where they are not dense); targets int64 [N], a value outside
    [0, V) marks a token that is not scored; cu_seqlens int32 [2 P + 1]: sequences 2i (preferred) and 2i + 1 (other) are pair
    i; ref_logps fp32 [2 P] the frozen model's log-probabilities.
        logps[s] = sum over scored tokens of log softmax(logits)[target]
        m_i = beta * ((logps - ref_logps)[2i] - (logps - ref_logps)[2i + 1])
        loss = mean_i (1 - label_smoothing) softplus(-m_i) + label_smoothing softplus(m_i)
                      - nll_weight * logps[2i] / max(1, scored tokens of 2i)
    loss fp32 scalar, logps fp32 [2 P]; `saved` is for `preference_loss_backward`.  Sums over tokens and pairs are 64-bit."""
    gpu, N, V = _check_preference(logits, targets)
    _need(cu_seqlens, "cu_seqlens", _I32, gpu)
    _need(ref_logps, "ref_logps", _F32, gpu)
    P = (cu_seqlens.numel() - 1) // 2
    if cu_seqlens.dim() != 1 or P < 1 or cu_seqlens.numel() != 2 * P + 1 or not cu_seqlens.is_contiguous():
        raise ValueError("cu_seqlens must be a dense vector of 2 * pairs + 1 offsets, one pair at least")
    if P >= 2 ** 23:
        raise ValueError("too many pairs")
    if ref_logps.shape != (2 * P,):
        raise ValueError(f"ref_logps {tuple(ref_logps.shape)}: wanted ({2 * P},)")
    if not 0.0 <= label_smoothing <= 1.0:
        raise ValueError(f"label_smoothing {label_smoothing} is outside [0, 1]")
    z, y, ref = _dense16(logits), targets.contiguous(), ref_logps.contiguous()
    nbytes = L.lib().esmk_pref_loss_saved_bytes(N, P)
    saved = ref.new_empty(nbytes // 4)
    logps, loss = ref.new_empty(2 * P), ref.new_empty(())
    _call(gpu, "esmk_pref_loss_fwd", z.data_ptr(), _DTYPES[z.dtype], y.data_ptr(), cu_seqlens.data_ptr(), P, ref.data_ptr(),
          beta, label_smoothing, nll_weight, N, V, saved.data_ptr(), nbytes, logps.data_ptr(), loss.data_ptr())
    return loss, logps, saved


def preference_loss_backward(logits, targets, saved, grad_loss=None):
    """Gradient of the loss with respect to the logits, in their dtype; tokens that are not scored get zeros.  `saved` is the
    forward call's, on the same inputs; grad_loss: fp32 scalar on the GPU (None = 1)."""
    gpu, N, V = _check_preference(logits, targets)
    _need(saved, "saved", _F32, gpu)
    if 4 * saved.numel() < L.lib().esmk_pref_loss_saved_bytes(N, 0) or not saved.is_contiguous():
        raise ValueError("saved does not belong to these logits")
    if grad_loss is not None:
        _need(grad_loss, "grad_loss", _F32, gpu)
        if grad_loss.numel() != 1:
            raise ValueError("grad_loss must be one value")
    z, y = _dense16(logits), targets.contiguous()
    dz = torch.empty_like(z)
    _call(gpu, "esmk_pref_loss_bwd", z.data_ptr(), _DTYPES[z.dtype], y.data_ptr(), saved.data_ptr(),
          None if grad_loss is None else grad_loss.data_ptr(), dz.data_ptr(), N, V)
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
