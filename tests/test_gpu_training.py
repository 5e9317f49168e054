"""Training operators (esm_amd.training) against plain 64-bit computations of their formulas.

Tolerances are bounds, element by element, derived from where the kernels round: u = 2^-24 for fp32 arithmetic,
r = eps / 2 of the output type (2^-8 for bf16) for every rounding to it.  Each test states its bound where it forms it."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U, TINY = 2.0 ** -24, 2.0 ** -126
R = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def T():
    from esm_amd import training
    return training


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def within(got, want, tol, what):
    assert got.shape == want.shape, what
    assert torch.isfinite(got.double()).all(), f"{what}: not finite"
    over = (got.double() - want).abs() - tol
    assert (over <= 0).all(), f"{what}: {over.max().item():.3e} over the bound, {int((over > 0).sum())} of {over.numel()}"


# ------------------------------------------------------------------------------------------------ layer norm

def norm_oracle(x, w, b, dy, eps=1e-5):
    """64-bit (y, dx, dw, db) and their bounds for output type x.dtype."""
    r = R[x.dtype]
    x, w, dy = x.double(), w.double(), dy.double()
    b = torch.zeros_like(w) if b is None else b.double()
    d = x.shape[-1]
    mu = x.mean(-1, keepdim=True)
    rs = 1 / ((x - mu).pow(2).mean(-1, keepdim=True) + eps).sqrt()
    h = (x - mu) * rs
    y = h * w + b
    g = dy * w
    c1, c2 = g.mean(-1, keepdim=True), (g * h).mean(-1, keepdim=True)
    dx = rs * (g - c1 - h * c2)
    # A row sum is at most 24 additions in a lane, 6 between lanes, 8 between waves: 40 u of the mean of the magnitudes.
    # xc = x - mean: 41 u (|x| + mean|x|); rstd: relative 60 u plus the effect of xc; h: both.
    ax = x.abs()
    exc = 42 * U * (ax + ax.mean(-1, keepdim=True))
    ers = 64 * U + 2 * (exc * (x - mu).abs()).mean(-1, keepdim=True) * rs * rs  # relative
    eh = exc * rs + h.abs() * ers
    ty = r * y.abs() + (1 + r) * (eh * w.abs() + 4 * U * (h * w).abs() + U * y.abs())
    ec1 = 44 * U * g.abs().mean(-1, keepdim=True)
    ec2 = ((eh + 44 * U * h.abs()) * g.abs()).mean(-1, keepdim=True)
    inner = g.abs() + c1.abs() + (h * c2).abs()
    ti = 4 * U * inner + ec1 + eh * c2.abs() + h.abs() * ec2
    tdx = r * dx.abs() + (1 + r) * rs * (ti + inner * ers)
    # columns: a lane adds its rows, then 3 row slots, 16 partials and 32 groups: below M + 64 additions
    M = x.reshape(-1, d).shape[0]
    n = min(M, M // 512 + 8) + 64
    cols = lambda t: t.reshape(-1, d).sum(0)
    dw, db = cols(dy * h), cols(dy)
    tdw = cols(dy.abs() * eh) + n * U * cols((dy * h).abs())
    tdb = n * U * cols(dy.abs())
    return (y, dx, dw, db), (ty, tdx, tdw, tdb)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,d", [(1, 1), (2, 3), (5, 64), (17, 65), (66, 960), (301, 1152), (130, 1281), (1030, 512),
                                    (37, 2560), (33, 1537), (9, 4097), (7, 6145), (3, 12288), (4099, 33), (700, 256), (33, 255),
                                    (2049, 136), (5000, 7), (70, 129), (40000, 72), (129, 257), (512, 1152), (513, 1152), (600, 2560),
                                    (601, 1537), (530, 4097), (520, 6145), (515, 12288), (900, 1281), (512, 12288), (400, 4096)])
def test_layer_norm(rows, d, dtype):
    g = gen(rows * 31 + d)
    x = (randn(g, rows, d) * 2 + 0.5).to(dtype)
    w, b, dy = 1 + 0.2 * randn(g, d), 0.3 * randn(g, d), randn(g, rows, d).to(dtype)
    for bias in (None, b):
        y, stats = T().layer_norm_forward(x, w, bias)
        dx, dw, db = T().layer_norm_backward(dy, x, w, stats, bias=bias is not None)
        assert y.dtype == dx.dtype == dtype and dw.dtype == torch.float32 and (db is None) == (bias is None)
        want, tol = norm_oracle(x, w, bias, dy)
        for got, a, t, n in zip((y, dx, dw, db), want, tol, ("y", "dx", "dw", "db")):
            if got is not None:
                within(got, a, t, n)


def test_layer_norm_strides_ranks_and_parameter_types():
    g = gen(5)
    wide = randn(g, 70, 3 * 192).bfloat16()
    w, b = 1 + 0.1 * randn(g, 192), 0.1 * randn(g, 192)
    dyw = randn(g, 70, 2 * 192).bfloat16()
    for x, dy in ((wide[:, 192:384], dyw[:, :192]), (wide[:, 1:193], dyw[:, 3:195]), (wide[::2, :192], dyw[::2, :192]),
                  (wide[:, :192].t().contiguous().t(), dyw[:, :192]), (wide[:1, :192].expand(70, 192), dyw[:, :192])):
        y, st = T().layer_norm_forward(x, w, b)
        got = (y,) + T().layer_norm_backward(dy, x, w, st)
        y2, st2 = T().layer_norm_forward(x.contiguous(), w, b)
        for p, q in zip(got, (y2,) + T().layer_norm_backward(dy.contiguous(), x.contiguous(), w, st2)):
            want, tol = norm_oracle(x, w, b, dy)
            assert p.shape == q.shape
        for p, a, t in zip(got, want, tol):
            within(p, a, t, "strided")
    x3 = wide[:, :192].reshape(2, 35, 192)
    assert torch.equal(T().layer_norm_forward(x3, w, b)[0], T().layer_norm_forward(x3.reshape(70, 192), w, b)[0].view(2, 35, 192))
    x1 = wide[0, :192]
    assert T().layer_norm_forward(x1, w)[0].shape == (192,)
    # parameters in bf16 count as the values they hold
    assert torch.equal(T().layer_norm_forward(x1, w.bfloat16())[0], T().layer_norm_forward(x1, w.bfloat16().float())[0])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d", [64, 192, 1152])
def test_layer_norm_slices_of_wider_activations(d, dtype):
    """x and dy as slices of [B, L, 3 d] activations, read in place: the bits of the 2-D slices, and of copies."""
    g = gen(d)
    qkv, grads = randn(g, 3, 41, 3 * d).to(dtype), randn(g, 3, 41, 2 * d).to(dtype)
    w, b = 1 + 0.1 * randn(g, d), 0.1 * randn(g, d)
    for x, dy in ((qkv[..., :d], grads[..., d:]), (qkv[..., 2 * d:], grads[..., :d]), (qkv[:, :1, d:2 * d], grads[:, 3:4, :d]),
                  (qkv[:, :40, :d], grads[:, 1:, d:])):
        got = T().layer_norm_forward(x, w, b)
        got += T().layer_norm_backward(dy, x, w, got[1])
        xc, dc = x.reshape(-1, d).contiguous(), dy.reshape(-1, d).contiguous()
        want = T().layer_norm_forward(xc, w, b)
        want += T().layer_norm_backward(dc, xc, w, want[1])
        for p, q in zip(got, want):
            assert torch.equal(p.reshape(q.shape), q)
        leaf = x.detach().requires_grad_()
        T().layer_norm(leaf, w, b).backward(dy)
        assert torch.equal(leaf.grad.reshape(-1, d), want[2])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,d", [(1, 64), (200, 65), (512, 256), (513, 256), (3000, 129), (300, 960), (512, 12288), (600, 1152), (2049, 1281),
                                    (700, 6145)])
def test_layer_norm_each_gradient_alone(rows, d, dtype):
    """What is not wanted changes no bit of what is: input and parameter gradients alone, one parameter's alone (C interface)."""
    from esm_amd import _lib as L
    g = gen(rows + d)
    x, dy = randn(g, rows, d).to(dtype), randn(g, rows, d).to(dtype)
    w, b = 1 + 0.1 * randn(g, d), randn(g, d)
    y, st = T().layer_norm_forward(x, w, b)
    dx, dw, db = T().layer_norm_backward(dy, x, w, st)
    want, tol = norm_oracle(x, w, b, dy)
    for got, a, t in zip((dx, dw, db), want[1:], tol[1:]):
        within(got, a, t, "all")
    none = T().layer_norm_backward(dy, x, w, st, param_grads=False)
    assert torch.equal(none[0], dx) and none[1] is None and none[2] is None
    par = T().layer_norm_backward(dy, x, w, st, input_grad=False)
    assert par[0] is None and torch.equal(par[1], dw) and torch.equal(par[2], db)
    assert T().layer_norm_backward(dy, x, w, st, param_grads=False, input_grad=False) == (None, None, None)
    nbytes = L.lib().esmk_layernorm_bwd_workspace_bytes(rows, d)
    for with_x in (True, False):
        for p, q in ((dw, None), (None, db)):
            ws = torch.empty(nbytes // 4 + 1, device="cuda")
            gx, gw, gb = (None if t is None else torch.full_like(t, 7.0) for t in (dx if with_x else None, p, q))
            L.check(L.lib().esmk_layernorm_bwd(dy.data_ptr(), d, x.data_ptr(), d, 0 if dtype is torch.float32 else 1, w.data_ptr(), st.data_ptr(),
                                               L.ptr(gx), L.ptr(gw), L.ptr(gb), ws.data_ptr(), nbytes, rows, d,
                                               torch.cuda.current_stream().cuda_stream))
            for got, full in ((gx, dx), (gw, dw), (gb, db)):
                assert got is None or torch.equal(got, full)


def test_autograd_asks_for_no_gradient_that_is_not_wanted(monkeypatch):
    """Frozen inputs and parameters: the call is told, and what is asked for keeps its bits."""
    t = T()
    calls = []
    call = t._call
    monkeypatch.setattr(t, "_call", lambda gpu, name, *args: (calls.append((name, args)), call(gpu, name, *args))[1])
    g = gen(12)
    x, w, b, dy = randn(g, 700, 96), 1 + 0.1 * randn(g, 96), randn(g, 96), randn(g, 700, 96)
    y, st = t.layer_norm_forward(x, w, b)
    full = t.layer_norm_backward(dy, x, w, st)
    for wants in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (0, 1, 1), (1, 1, 1)):
        leaves = [u.clone().requires_grad_(bool(v)) for u, v in zip((x, w, b), wants)]
        t.layer_norm(*leaves).backward(dy)
        name, args = calls[-1]
        assert name == "esmk_layernorm_bwd" and [a is not None for a in args[7:10]] == [wants[0] == 1, wants[1] + wants[2] > 0, wants[2] == 1]
        for leaf, want in zip(leaves, full):
            assert leaf.grad is None if not leaf.requires_grad else torch.equal(leaf.grad, want)
    row = x[:1].clone().requires_grad_()  # a broadcast input's gradient is summed
    t.layer_norm(row.expand(700, 96), w, b).backward(dy)
    dx = t.layer_norm_backward(dy, x[:1].expand(700, 96), w, t.layer_norm_forward(x[:1].expand(700, 96), w)[1])[0]
    assert torch.equal(row.grad, dx.sum(0, keepdim=True))
    for r in (1, 70):  # few blocks and many
        q, k, v, cu, cut, dout, _ = attention_inputs(19, [130, 31, 64], 2 * r, r, 64, tail=2)
        full = attention_all(q, k, v, cut, dout)[2:]
        for wants in ((1, 0, 0), (1, 1, 0), (0, 0, 1), (1, 1, 1)):
            leaves = [u.clone().requires_grad_(bool(a)) for u, a in zip((q, k, v), wants)]
            t.attention_varlen(*leaves, cut).backward(dout)
            name, args = calls[-1]
            assert name == "esmk_attn_varlen_bwd" and [a is not None for a in args[6:9]] == [True] + 2 * [wants[1] + wants[2] > 0]
            for leaf, want in zip(leaves, full):
                assert leaf.grad is None if not leaf.requires_grad else torch.equal(leaf.grad, want)


def test_layer_norm_no_rows_gives_zero_parameter_gradients():
    x, w = torch.empty(0, 96, device="cuda"), torch.ones(96, device="cuda")
    y, st = T().layer_norm_forward(x, w)
    dx, dw, db = T().layer_norm_backward(torch.empty_like(x), x, w, st)
    assert y.shape == dx.shape == (0, 96) and not dw.any() and not db.any()


def test_layer_norm_far_rows():
    """Row offsets past 2^32 bytes."""
    big = torch.empty(300 * 2 ** 23, dtype=torch.bfloat16, device="cuda")
    for rows, ld, d in ((300, 2 ** 23, 64), (300, 2 ** 23, 320), (37, 2 ** 26, 64)):  # the last: strides that 16 rows cannot share
        x = big.as_strided((rows, d), (ld, 1))
        g = gen(3)
        x.copy_(randn(g, rows, d))
        w, dy = 1 + 0.1 * randn(g, d), randn(g, rows, d).bfloat16()
        y, st = T().layer_norm_forward(x, w)
        got = (y,) + T().layer_norm_backward(dy, x, w, st)
        xc = x.contiguous()
        want, tol = norm_oracle(xc, w, None, dy)
        for a, b, t in zip(got, want, tol):
            within(a, b, t, "far rows")
        if ld < 2 ** 26:
            y2, st2 = T().layer_norm_forward(xc, w)
            for a, b in zip(got, (y2,) + T().layer_norm_backward(dy, xc, w, st2)):
                assert torch.equal(a, b)


def test_layer_norm_more_than_2_31_elements():
    """Dense rows past 2^32 bytes of x, y, dy and dx: the last rows against the same rows alone, and column sums of rows that
    repeat."""
    g = gen(4)
    one, dy1 = randn(g, 1024, 1152).bfloat16(), randn(g, 1024, 1152).bfloat16()
    w, b = 1 + 0.1 * randn(g, 1152), 0.1 * randn(g, 1152)
    times = 1850
    x, dy = one.repeat(times, 1), dy1.repeat(times, 1)
    assert x.numel() > 2 ** 31
    y, st = T().layer_norm_forward(x, w, b)
    dx, dw, db = T().layer_norm_backward(dy, x, w, st)
    y1, st1 = T().layer_norm_forward(one, w, b)
    dx1, _, _ = T().layer_norm_backward(dy1, one, w, st1)
    for got, want in ((y, y1), (st, st1), (dx, dx1)):
        assert torch.equal(got[-1024:], want) and torch.equal(got[:1024], want)
    want, tol = norm_oracle(one, w, b, dy1)
    # a lane adds 1850 x 1024 / 512 rows of its workgroup's four slots, then 64 more sums: below 1000 u of the magnitudes
    h = ((one.double() - one.double().mean(-1, keepdim=True)) / (one.double().var(-1, unbiased=False, keepdim=True) + 1e-5).sqrt())
    within(dw, times * want[2], times * (tol[2] + 1000 * U * (dy1.double() * h).abs().sum(0)), "dw")
    within(db, times * want[3], times * (tol[3] + 1000 * U * dy1.double().abs().sum(0)), "db")


def test_layer_norm_autograd_and_differences():
    g = gen(11)
    x, w, b = randn(g, 21, 130), 1 + 0.2 * randn(g, 130), 0.2 * randn(g, 130)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    probe = randn(g, 21, 130)
    (T().layer_norm(*leaves) * probe).sum().backward()
    want, tol = norm_oracle(x, w, b, probe)
    for t, a, e in zip(leaves, want[1:], tol[1:]):
        within(t.grad, a, e, "autograd")
    # central differences of the 64-bit formula along a random direction; its own error is below 1e-8 of the slope's terms
    f = lambda x, w, b: (norm_oracle(x, w, b, probe.double())[0][0] * probe.double()).sum().item()
    for i, t in enumerate((x, w, b)):
        v = randn(g, *t.shape).double()
        at = lambda s: f(*[(u.double() + s * v if j == i else u.double()) for j, u in enumerate((x, w, b))])
        R[torch.float64] = 0.0
        slope = (at(1e-4) - at(-1e-4)) / 2e-4
        bound = (tol[1 + i] * v.abs()).sum().item() + 1e-6 * (want[1 + i].abs() * v.abs()).sum().item()
        assert abs((leaves[i].grad.double() * v).sum().item() - slope) <= bound
    # a frozen weight asks for no reduction; a broadcast input's gradient is summed
    row = randn(g, 1, 130).requires_grad_()
    T().layer_norm(row.expand(21, 130), w, b).sum().backward()
    assert row.grad.shape == (1, 130)


# ------------------------------------------------------------------------------------------------ attention

def attention_oracle(q, k, v, cu, scale, mask, dout, short=False, rest=False):
    """64-bit (out, lse, dq, dk, dv) and bounds.  Where the kernels round: P to bf16 before P V and P^T dO (r), dS to bf16
    before dS K and dS^T Q (r), outputs (r); delta uses the rounded out.  fp32: a score has D products (D u of their
    magnitudes) and moves P by that, relatively; sums over keys or queries L u.  Below the smallest normal number, 2^-126, a
    probability or a result may be flushed to zero: that much is added wherever one enters.  short: sequences of at most 64
    tokens, where delta is summed again as delta + rowsum(P (dP - delta)) and out's rounding leaves it.
    rest: dS in two bf16 parts, off by r r / 2 of it."""
    r = R[torch.bfloat16]
    N, H, D = q.shape
    G = k.shape[1]
    q, k, v, dout = (t.double() for t in (q, k, v, dout))
    z = lambda *s: torch.zeros(*s, dtype=torch.float64, device=q.device)
    o, dq, dk, dv = z(N, H, D), z(N, H, D), z(N, G, D), z(N, G, D)
    to, tdq, tdk, tdv = z(N, H, D), z(N, H, D), z(N, G, D), z(N, G, D)
    lse, tl = torch.full((H, N), -math.inf, dtype=torch.float64, device=q.device), z(H, N)
    for a, e in zip(cu, cu[1:]):
        keys = torch.arange(a, e, device=q.device)
        if mask is not None:
            keys = keys[mask[a:e].bool()]
        L = e - a
        if len(keys) == 0:
            continue
        for h in range(H):
            Q, K, V, dO = q[a:e, h], k[keys, h // (H // G)], v[keys, h // (H // G)], dout[a:e, h]
            S = Q @ K.t() * scale
            ls = torch.logsumexp(S, -1, keepdim=True)
            P = (S - ls).exp()
            O = P @ V
            eS = (D + 8) * U * scale * (Q.abs() @ K.abs().t()) + 4 * U * (S.abs() + ls.abs())  # abs, both S and S - lse
            eP = 2 * eS.amax(-1, keepdim=True) + (L + 32) * U                                  # rel. of P
            A = P @ V.abs()
            tO = (r + eP) * A * (1 + r) + r * O.abs() + eP * O.abs() + TINY * (1 + V.abs().sum(0) + L * O.abs())
            dP = dO @ V.t()
            dl = (dO * O).sum(-1, keepdim=True)
            dS = P * (dP - dl)
            eDl = (dO.abs() * tO).sum(-1, keepdim=True) + (D + 8) * U * (dO * O).abs().sum(-1, keepdim=True)
            eDP = (D + 8) * U * (dO.abs() @ V.abs().t())
            if short:
                assert L <= 64
                eDl = ((eP + (L + 32) * U) * P * ((dP - dl).abs() + eDl) + P * eDP).sum(-1, keepdim=True) + 2 * U * dl.abs()
            eds = P * (eDl + eDP + eP * (dP - dl).abs()) * (1 + r) + r * (r if rest else 1) * dS.abs() + TINY * (1 + (dP - dl).abs())  # abs, of the rounded dS
            n = (L + 32) * U
            o[a:e, h], to[a:e, h] = O, tO
            lse[h, a:e] = ls[:, 0]
            tl[h, a:e] = eS.amax(-1) + (L + 32) * U + 4 * U * ls[:, 0].abs()
            dq[a:e, h] = scale * dS @ K
            tdq[a:e, h] = scale * ((eds + n * dS.abs()) @ K.abs())
            dk[keys, h // (H // G)] += scale * dS.t() @ Q
            tdk[keys, h // (H // G)] += scale * ((eds + n * dS.abs()).t() @ Q.abs())
            dv[keys, h // (H // G)] += P.t() @ dO
            tdv[keys, h // (H // G)] += ((r + eP + n) * P + TINY).t() @ dO.abs()
    tdq, tdk, tdv = (t * (1 + r) + r * x.abs() + 4 * U * x.abs() + TINY for t, x in ((tdq, dq), (tdk, dk), (tdv, dv)))
    return (o, lse, dq, dk, dv), (to, tl, tdq, tdk, tdv)


def attention_inputs(seed, lens, H, G, D, tail=0, lead=0, q_gain=1.5):
    g = gen(seed)
    cu = [lead]
    for n in lens:
        cu.append(cu[-1] + n)
    N = cu[-1] + tail
    qkv = randn(g, N, H + 2 * G, D)
    qkv[:, :H] *= q_gain
    qkv = qkv.bfloat16()
    return qkv[:, :H], qkv[:, H:H + G], qkv[:, H + G:], cu, torch.tensor(cu, dtype=torch.int32, device="cuda"), randn(g, N, H, D).bfloat16(), g


def attention_all(q, k, v, cu, dout, scale=None, mask=None):
    out, lse = T().attention_varlen_forward(q, k, v, cu, scale, mask)
    return (out, lse) + T().attention_varlen_backward(dout, q, k, v, out, lse, cu, scale, mask)


def copies(N, n, G):
    """How often the heads have to be repeated for more than 256 blocks of 128 rows: fewer go other ways through the kernels."""
    return 256 // ((N // 128 + n + 2) * G) + 1


def check_attention(q, k, v, cu, cut, dout, scale=None, mask=None, short=False):
    """Few heads, and the same heads so often that the kernels for many blocks run, against one oracle."""
    want, tol = attention_oracle(q, k, v, cu, scale or q.shape[2] ** -0.5, mask, dout, short)
    none = want[1] == -math.inf
    want = (want[0], want[1].masked_fill(none, 0.0)) + want[2:]
    first = None
    for r in (1, copies(len(q), len(cu) - 1, k.shape[1])):
        got = attention_all(*(t.repeat(1, r, 1) if r > 1 else t for t in (q, k, v)), cut, dout.repeat(1, r, 1), scale, mask)
        first = first or got
        lse = got[1].view(r, *none.shape)
        assert torch.equal(lse == -math.inf, none.expand_as(lse))
        got = tuple(t.view(len(q), r, -1, q.shape[2]).transpose(0, 1) for t in got[:1] + got[2:])
        for a, b, t, n in zip((got[0], lse.masked_fill(none, 0.0)) + got[1:], want, tol, ("out", "lse", "dq", "dk", "dv")):
            within(a, b.expand_as(a), t, f"{n}, {r} copies")
            assert torch.equal(a[0], a[-1])
    return first


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens,H,G,tail", [([1], 1, 1, 0), ([2, 1, 3], 2, 1, 0), ([0, 5, 0], 2, 2, 3), ([64], 1, 1, 0),
                                           ([63, 65], 2, 2, 0), ([128, 129, 127], 3, 1, 9), ([200, 1, 77, 300], 4, 2, 0),
                                           ([1100], 2, 2, 1), ([31] * 70, 1, 1, 5)])
def test_attention(lens, H, G, tail, D):
    q, k, v, cu, cut, dout, _ = attention_inputs(len(lens) * 7 + D, lens, H, G, D, tail)
    check_attention(q, k, v, cu, cut, dout)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens,H,G,tail,lead", [([900, 3, 1300, 0, 512, 700], 9, 3, 140, 0), ([513, 1500, 640], 3, 1, 0, 200), ([700] * 3, 10, 2, 1, 1),
                                                ([17] * 62, 9, 9, 3, 0), ([17] * 63, 9, 9, 3, 0), ([130, 1] * 31, 2, 1, 0, 5),
                                                ([2100], 3, 3, 0, 300), ([0, 0, 0], 2, 2, 300, 0), ([300, 90], 64, 1, 5, 0)])
def test_attention_every_order_of_blocks(lens, H, G, tail, lead, D):
    """By length, by number (up to 62 sequences) and by groups; heads in eights and what is left of them; nothing but gaps."""
    q, k, v, cu, cut, dout, _ = attention_inputs(len(lens) + H + D, lens, H, G, D, tail, lead)
    got = check_attention(q, k, v, cu, cut, dout)
    for t in (got[0],) + got[2:]:
        assert not t[:lead].any() and not t[cu[-1]:].any()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("masked", [False, True])
def test_attention_short_sequences_have_an_exact_delta(D, masked):
    """dq and dk of sequences of one tile: what the rounding of out would leave in delta (all of dq and dk, for one token,
    where they are zero) is above these bounds."""
    q, k, v, cu, cut, dout, g = attention_inputs(50 + D, [1, 5, 64, 2, 33, 1, 63, 3] * 3, 4, 2, D, tail=2)
    mask = None
    if masked:
        mask = torch.rand(len(q), generator=g, device="cuda") > 0.2
        mask[cu[2]:cu[3]] = False
    got = check_attention(q, k, v, cu, cut, dout, mask=mask, short=True)
    # few blocks: dS's rounding has a second product, and dq's and dk's own rounding is left
    want, tol = attention_oracle(q, k, v, cu, D ** -0.5, mask, dout, short=True, rest=True)
    for a, b, t, n in zip(got[2:4], want[2:4], tol[2:4], ("dq", "dk")):
        within(a, b, t, n)


@pytest.mark.parametrize("D", [64, 128])
def test_attention_key_mask(D):
    """Scattered masked keys, a tile without any key, a sequence without any key, one key left."""
    q, k, v, cu, cut, dout, g = attention_inputs(3 + D, [150, 40, 260, 90], 4, 2, D, tail=6, lead=5)
    mask = torch.rand(len(q), generator=g, device="cuda") > 0.3
    mask[cu[1]:cu[2]] = False
    mask[cu[2] + 64:cu[2] + 128] = False
    mask[cu[3]:cu[4]] = False
    mask[cu[3] + 70] = True
    for m in (mask, mask.to(torch.uint8)):
        got = check_attention(q, k, v, cu, cut, dout, mask=m)
    assert not got[0][cu[1]:cu[2]].any() and not got[2][cu[1]:cu[2]].any()
    assert not got[0][:5].any() and not got[0][cu[-1]:].any() and not got[3][~mask].any() and not got[4][~mask].any()
    # what masked keys and tokens in no sequence hold does not matter, NaN and inf included
    k2, v2, d2, q2 = k.clone(), v.clone(), dout.clone(), q.clone()
    k2[~mask], v2[~mask] = math.nan, math.inf
    for t in (q2, k2, v2, d2):
        t[:5], t[cu[-1]:] = math.nan, math.nan
    d2[cu[1]:cu[2]] = math.inf  # queries without a key
    for a, b in zip(got, attention_all(q2, k2, v2, cut, d2, mask=mask)):
        assert torch.equal(a, b)
    many = lambda *ts: [t.repeat(1, copies(len(q), 4, 2), 1) for t in ts]
    q3, k3, v3, d3 = many(q, k, v, dout)
    q4, k4, v4, d4 = many(q2, k2, v2, d2)
    for a, b in zip(attention_all(q3, k3, v3, cut, d3, mask=mask), attention_all(q4, k4, v4, cut, d4, mask=mask)):
        assert torch.equal(a, b)


def test_attention_scales_and_large_scores():
    """Scores of several hundred (one key takes all), a tiny scale (all keys alike), values of 1e4."""
    for gain, scale in ((60.0, None), (1.0, 1e-4), (1.0, 2.0)):
        q, k, v, cu, cut, dout, _ = attention_inputs(9, [130, 70], 2, 2, 64, q_gain=gain)
        check_attention(q, k, v, cu, cut, dout, scale)
    q, k, v, cu, cut, dout, _ = attention_inputs(10, [130, 70], 2, 2, 64)
    check_attention(q, k, (v * 1e4).bfloat16(), cu, cut, dout)


def test_attention_layouts():
    """Head-major storage, an unaligned slice (copied), int strides past 2^31 elements."""
    q, k, v, cu, cut, dout, _ = attention_inputs(21, [90, 33], 4, 2, 64)
    base = attention_all(q.contiguous(), k.contiguous(), v.contiguous(), cut, dout)
    hm = lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)
    odd = torch.empty(len(q), 4, 65, dtype=torch.bfloat16, device="cuda")[:, :, 1:]
    odd.copy_(q)
    one = dout[:, :1].expand(-1, 4, -1)
    for args in ((q, k, v, dout), (hm(q), hm(k), hm(v), hm(dout)), (odd, k, v, dout)):
        for a, b in zip(base, attention_all(*args[:3], cut, args[3])):
            assert torch.equal(a, b)
    for a, b in zip(attention_all(q, k, v, cut, one), attention_all(q, k, v, cut, one.contiguous())):
        assert torch.equal(a, b)

    def shifted(t):  # dense, at an address that is no multiple of 16 bytes
        flat = t.new_empty(t.numel() + 1)[1:].view(t.shape)
        return flat.copy_(t)
    assert shifted(q).is_contiguous() and shifted(q).data_ptr() % 16
    for a, b in zip(base, attention_all(shifted(q), shifted(k), shifted(v), cut, shifted(dout))):
        assert torch.equal(a, b)
    # one token and one head: torch calls any strides of theirs dense
    lone = lambda t: t.new_empty(1, 1, 70)[:, :, :64].as_strided((1, 1, 64), (70, 3, 1)).copy_(t[:1, :1])
    assert lone(q).is_contiguous()
    first = cut.clamp(max=1)
    for a, b in zip(attention_all(lone(q), lone(k), lone(v), first, lone(dout)),
                    attention_all(q[:1, :1], k[:1, :1], v[:1, :1], first, dout[:1, :1])):
        assert torch.equal(a, b)
    N = 400
    big = torch.empty(N * (2 ** 23 - 8), dtype=torch.bfloat16, device="cuda")
    far = big.as_strided((N, 3, 64), (2 ** 23 - 8, 64, 1))
    far.copy_(randn(gen(2), N, 3, 64))
    cut = torch.tensor([0, 150, N], dtype=torch.int32, device="cuda")
    near = far.contiguous()
    for r in (1, copies(N, 2, 1)):  # heads that are all the same memory
        d = dout.new_ones(N, r, 64)
        at = lambda t, i: t[:, i:i + 1].expand(-1, r, -1)
        for a, b in zip(attention_all(at(far, 0), at(far, 1), at(far, 2), cut, d), attention_all(at(near, 0), at(near, 1), at(near, 2), cut, d)):
            assert torch.equal(a, b)


def test_attention_more_than_2_31_elements():
    """q, k, v, out and lse offsets past 32 bits of elements: 850 k tokens of 40 heads in 64-token sequences; the last ones
    against the same tokens alone."""
    N, H = 850_000 // 64 * 64, 40
    assert N * H * 64 > 2 ** 31
    g = gen(6)
    one = randn(g, 64 * 50, 3 * H, 64).bfloat16()
    qkv = one.repeat(-(-N // len(one)), 1, 1)[:N]
    q, k, v = qkv[:, :H].contiguous(), qkv[:, H:2 * H], qkv[:, 2 * H:]
    cu = torch.arange(N // 64 + 1, dtype=torch.int32, device="cuda") * 64
    dout = q
    got = attention_all(q, k, v, cu, dout)
    small = attention_all(one[:, :H], one[:, H:2 * H], one[:, 2 * H:], cu[:51], one[:, :H])
    m = (N // len(one)) * len(one)  # a whole copy ends here
    for a, b in zip(got, small):
        a = a[:, m - len(one):m] if a.dim() == 2 else a[m - len(one):m]
        assert torch.equal(a, b)
    del got, q, k, v, qkv, dout
    torch.cuda.empty_cache()


def test_attention_padded_batch_equals_packed():
    """[B, L] with a key mask over the padding = the packed sequences, for the real tokens."""
    lens, L = [70, 128, 1, 200], 200
    q, k, v, cu, cut, dout, g = attention_inputs(41, lens, 4, 2, 64)
    want = attention_all(q, k, v, cut, dout)
    at = torch.cat([torch.arange(n) + i * L for i, n in enumerate(lens)]).cuda()
    wide = lambda t: torch.randn(4 * L, *t.shape[1:], device="cuda", generator=g).bfloat16().index_copy(0, at, t.contiguous())
    mask = torch.zeros(4 * L, dtype=torch.bool, device="cuda").index_fill(0, at, True)
    d = wide(dout) * mask[:, None, None]
    got = attention_all(wide(q), wide(k), wide(v), torch.arange(5, dtype=torch.int32, device="cuda") * L, d, mask=mask)
    oracle, tol = attention_oracle(q, k, v, cu, 0.125, None, dout)
    for a, b, t, n in zip(got, oracle, tol, ("out", "lse", "dq", "dk", "dv")):
        within(a[:, at] if n == "lse" else a[at], b, t, n)
    assert torch.equal(got[0][at], want[0]) and not got[3][~mask].any()


def few_key_buffers(at, N, q, k, v, dout, g):
    """The packed tokens at the places `at` of a buffer of N tokens that holds anything elsewhere, with the mask of
    those places; dout is zero elsewhere."""
    wide = lambda t: randn(g, N, *t.shape[1:]).bfloat16().index_copy(0, at, t.contiguous())
    mask = torch.zeros(N, dtype=torch.bool, device="cuda").index_fill(0, at, True)
    return wide(q), wide(k), wide(v), wide(dout) * mask[:, None, None], mask


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("scattered", [False, True])
@pytest.mark.parametrize("L", [70, 130, 600, 1100])
def test_attention_few_live_keys_among_padding(L, scattered, D):
    """Sequences of 1 to 64 live keys, padded at their end or scattered among masked tokens: the bounds of the packed
    sequences, whose delta is free of out's rounding and whose dS has two parts.  The sums have the same terms; masked keys add
    zeros.  In few blocks and in many."""
    lens = [1, 2, 3, 5, 17, 33, 64]
    q, k, v, cu, cut, dout, g = attention_inputs(60 + L + D, lens, 4, 2, D)
    at = []
    for i, n in enumerate(lens):
        where = torch.randperm(L, generator=torch.Generator().manual_seed(i))[:n].sort()[0] if scattered else torch.arange(n)
        at.append(where + i * L)
    at = torch.cat(at).cuda()
    want, tol = attention_oracle(q, k, v, cu, D ** -0.5, None, dout, short=True, rest=True)
    wq, wk, wv, wd, mask = few_key_buffers(at, len(lens) * L, q, k, v, dout, g)
    wcu = torch.arange(len(lens) + 1, dtype=torch.int32, device="cuda") * L
    for r in (1, copies(len(mask), len(lens), 2)):
        many = lambda t: t.repeat(1, r, 1)
        got = attention_all(many(wq), many(wk), many(wv), wcu, many(wd), mask=mask)
        for a, b, t, n in zip(got[2:], want[2:], tol[2:], ("dq", "dk", "dv")):
            a = a.view(len(mask), r, -1, D).transpose(0, 1)
            within(a[:, at], b.expand_as(a[:, at]), t, f"{n}, {r} copies")
            assert n == "dq" or not a[:, ~mask].any()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("masked", [False, True])
def test_attention_gradients_of_few_keys_do_not_depend_on_the_rest_of_the_call(D, masked):
    """The same short sequences alone, among long ones, and with more heads: dS in two parts in all of them."""
    short = [1, 5, 64, 2, 33, 40, 63, 3]
    q, k, v, cu, cut, dout, g = attention_inputs(80 + D, short + [900, 70, 1300], 4, 2, D)
    n = sum(short)
    mask = None
    if masked:
        mask = torch.rand(len(q), generator=g, device="cuda") > 0.3
        mask[cu[2]:cu[3]:2] = True
    want, tol = attention_oracle(q[:n], k[:n], v[:n], cu[:len(short) + 1], D ** -0.5, None if mask is None else mask[:n], dout[:n],
                                 short=True, rest=True)
    alone = (q[:n], k[:n], v[:n], cut[:len(short) + 1], dout[:n], None if mask is None else mask[:n])
    r = copies(len(q), len(cu) - 1, 2)
    many = lambda t: t.repeat(1, r, 1)
    for args in (alone, (q, k, v, cut, dout, mask), (many(q), many(k), many(v), cut, many(dout), mask)):
        got = attention_all(*args[:5], mask=args[5])
        for a, b, t, name in zip(got[2:], want[2:], tol[2:], ("dq", "dk", "dv")):
            a = a[:n].view(n, -1, b.shape[1], D).transpose(0, 1)
            within(a, b.expand_as(a), t, f"{name}, {len(args[0])} tokens, {args[0].shape[1]} heads")


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("masked", [False, True])
def test_attention_small_calls_keep_two_parts_up_to_512_keys(D, masked):
    """dq and dk of 65 to 512 keys in few blocks, against 64 bits with the delta that the forward pass's rounded out gives.  What is
    left is the rounding of the result and, were dS rounded once, one as large and independent of it: 1.41 times the former.
    1.2 is asked of each sequence."""
    live = [65, 130, 300, 512]
    lens = [n + n // 3 if masked else n for n in live]  # with every fourth key masked as many take part
    q, k, v, cu, cut, dout, g = attention_inputs(90 + D, lens, 2, 2, D)
    mask = torch.arange(len(q), device="cuda") % 4 != 3 if masked else None
    got = attention_all(q, k, v, cut, dout, mask=mask)
    scale = D ** -0.5
    for a, b in zip(cu, cu[1:]):
        keep = torch.ones(b - a, dtype=torch.bool, device="cuda") if mask is None else mask[a:b]
        assert 64 < keep.sum() <= 512
        for h in range(2):
            Q, K, V, dO, O = (t[a:b, h].double() for t in (q, k, v, dout, got[0]))
            P = (Q @ K.t() * scale).masked_fill(~keep, -math.inf).softmax(-1)
            dS = scale * P * (dO @ V.t() - (dO * O).sum(-1, keepdim=True))
            for x, exact, name in ((got[2], dS @ K, "dq"), (got[3], dS.t() @ Q, "dk")):
                rounding = (exact.bfloat16().double() - exact).norm()
                assert (x[a:b, h].double() - exact).norm() <= 1.2 * rounding, f"{name} of {b - a} tokens"


def test_attention_rising_and_falling_scores():
    """Keys whose scores rise from tile to tile by far more than the reference point may lag, and fall again; large values."""
    N = 64 * 9
    q = torch.zeros(N, 1, 64, device="cuda")
    q[:, :, 0] = 8.0
    g = gen(77)
    k = 0.3 * randn(g, N, 1, 64)
    k[:, 0, 0] = torch.tensor([0.0, 3, 8, 20, 45, 44, 10, -60, 45.5], device="cuda").repeat_interleave(64)
    v = randn(g, N, 1, 64)
    q, k, v = q.bfloat16(), k.bfloat16(), v.bfloat16()
    cut = torch.tensor([0, N], dtype=torch.int32, device="cuda")
    dout = randn(g, N, 1, 64).bfloat16()
    check_attention(q, k, v, [0, N], cut, dout)
    check_attention(q, k.flip(0).contiguous(), (v * 1e30).bfloat16(), [0, N], cut, (dout * 1e-30).bfloat16())


def test_empty_inputs():
    e = torch.empty(0, 2, 64, dtype=torch.bfloat16, device="cuda")
    cut = torch.zeros(3, dtype=torch.int32, device="cuda")
    got = attention_all(e, e, e, cut, e)
    assert got[0].shape == (0, 2, 64) and got[1].shape == (2, 0) and got[2].shape == got[3].shape == (0, 2, 64)
    z, y = torch.empty(0, 7, device="cuda"), torch.empty(0, dtype=torch.int64, device="cuda")
    for P in (1, 3):
        ref = torch.randn(2 * P, device="cuda")
        loss, logps, saved = T().preference_loss_forward(z, y, torch.zeros(2 * P + 1, dtype=torch.int32, device="cuda"), ref, beta=0.5)
        want = torch.nn.functional.softplus(0.5 * (ref[0::2] - ref[1::2]).double()).mean().item()
        assert abs(loss.item() - want) <= 1e-6 and not logps.any()
        assert T().preference_loss_backward(z, y, saved).shape == (0, 7)


def test_layer_norm_parameters_in_bf16_get_gradients_in_bf16():
    g = gen(8)
    x = randn(g, 40, 96).bfloat16().requires_grad_()
    w, b = (1 + 0.1 * randn(g, 96)).bfloat16().requires_grad_(), randn(g, 96).bfloat16().requires_grad_()
    dy = randn(g, 40, 96).bfloat16()
    T().layer_norm(x, w, b).backward(dy)
    want, tol = norm_oracle(x.detach(), w.detach(), b.detach(), dy)
    for t, a, e in zip((x, w, b), want[1:], tol[1:]):
        assert t.grad.dtype == torch.bfloat16
        within(t.grad, a, e * (1 + R[torch.bfloat16]) + R[torch.bfloat16] * a.abs(), "bf16 parameters")


def test_attention_offsets_outside_the_buffer_are_clamped():
    q, k, v, cu, cut, dout, _ = attention_inputs(4, [90, 60], 2, 2, 64)
    bad = torch.tensor([-7, 90, 150 + 1000], dtype=torch.int32, device="cuda")
    for a, b in zip(attention_all(q, k, v, cut, dout), attention_all(q, k, v, bad, dout)):
        assert torch.equal(a, b)
    none = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = attention_all(q, k, v, none, dout)
    assert (out[1] == -math.inf).all() and not any(t.any() for t in (out[0],) + out[2:])


def test_attention_autograd_and_differences():
    q, k, v, cu, cut, dout, g = attention_inputs(31, [70, 45], 4, 2, 64)
    scale = 0.125
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    T().attention_varlen(*leaves, cut).backward(dout)
    want, tol = attention_oracle(q, k, v, cu, scale, None, dout)
    for i, (t, a, e) in enumerate(zip(leaves, want[2:], tol[2:])):
        within(t.grad, a, e, "autograd")
        d = randn(g, *t.shape).double()
        f = lambda s: (attention_oracle(*[(x.double() + s * d if j == i else x) for j, x in enumerate((q, k, v))], cu, scale,
                                        None, dout)[0][0] * dout.double()).sum().item()
        slope = (f(1e-4) - f(-1e-4)) / 2e-4
        assert abs((t.grad.double() * d).sum().item() - slope) <= (e * d.abs()).sum().item() + 1e-5 * (a.abs() * d.abs()).sum().item()


# ------------------------------------------------------------------------------------------------ preference loss

def preference_oracle(z, y, cu, ref, beta, eps, alpha, dtype):
    """64-bit (loss, logps, dz) and bounds: a token's log-probability is off by u (V + 64 + 4 |logp| + 4 |z_y - max|) at most
    (its sum has below V / 16 + 16 additions of terms that are off by 4 u (1 + |z - max|), and exp damps those)."""
    z = z.double()
    V = z.shape[1]
    P = (len(cu) - 1) // 2
    lp = torch.log_softmax(z, -1)
    l, tl, n = [], [], []
    used = []
    for a, b in zip(cu, cu[1:]):
        rows = torch.arange(a, b, device=z.device)
        rows = rows[(y[rows] >= 0) & (y[rows] < V)]
        x = lp[rows, y[rows]]
        l.append(x.sum())
        tl.append((U * (V / 16 + 64 + 8 * x.abs())).sum() + U * x.sum().abs())
        n.append(max(1, len(rows)))
        used.append(rows)
    ref = ref.double()
    loss, tloss, dz, tdz = 0.0, 0.0, torch.zeros_like(z), torch.zeros_like(z)
    r = R[dtype]
    for i in range(P):
        m = beta * ((l[2 * i] - ref[2 * i]) - (l[2 * i + 1] - ref[2 * i + 1]))
        tm = abs(beta) * (tl[2 * i] + tl[2 * i + 1])
        sp = lambda t: torch.nn.functional.softplus(t, threshold=1e9)
        loss = loss + ((1 - eps) * sp(-m) + eps * sp(m) - alpha * l[2 * i] / n[2 * i]) / P
        tloss = tloss + (tm + abs(alpha) * tl[2 * i] / n[2 * i]) / P
        gm = beta * (eps * torch.sigmoid(m) - (1 - eps) * torch.sigmoid(-m)) / P
        tg = abs(beta) * tm / 4 / P
        for j, c in ((2 * i, gm - alpha / n[2 * i] / P), (2 * i + 1, -gm)):
            rows = used[j]
            p = lp[rows].exp()
            hot = torch.nn.functional.one_hot(y[rows], V).double()
            dz[rows] = c * (hot - p)
            ep = p * U * (V / 16 + 64 + 8 * lp[rows].abs())
            tdz[rows] = (tg + 4 * U * abs(c)) * (hot - p).abs() + abs(c) * (ep + U * hot)
    tdz = tdz * (1 + r) + r * dz.abs() + 2e-38  # results below the smallest normal number may be flushed
    return (loss, torch.stack(l), dz), (tloss + 4 * U * abs(loss), torch.stack(tl) + U * torch.stack(l).abs(), tdz)


def preference_inputs(seed, lens, V, dtype, tail=0, spread=1.5, lead=0):
    g = gen(seed)
    cu = [lead]
    for n in lens:
        cu.append(cu[-1] + n)
    N = cu[-1] + tail
    z = (spread * randn(g, N, V)).to(dtype)
    y = torch.randint(0, V, (N,), generator=g, device="cuda")
    y[torch.rand(N, generator=g, device="cuda") < 0.25] = -100
    ref = -3.0 * torch.tensor([float(n) for n in lens], device="cuda") + randn(g, len(lens))
    return z, y, cu, torch.tensor(cu, dtype=torch.int32, device="cuda"), ref, g


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V,lens,tail", [(64, [5, 9], 0), (64, [1, 0, 0, 3], 2), (1, [4, 4], 0), (2, [3, 3], 0), (33, [70, 64, 1, 130], 7),
                                         (256, [40, 40], 0), (257, [17, 33], 1), (4096, [30, 41], 0), (4101, [20, 9, 11, 1], 5),
                                         (9001, [3, 2], 0), (64, [7] * 140, 0)])
def test_preference_loss(V, lens, tail, dtype):
    z, y, cu, cut, ref, _ = preference_inputs(V + len(lens), lens, V, dtype, tail)
    if len(y) > 6:
        y[3] = V  # out of range: not scored
    for beta, eps, alpha in ((0.1, 0.0, 0.0), (0.5, 0.1, 0.3), (0.05, 1.0, 1.0)):
        loss, logps, saved = T().preference_loss_forward(z, y, cut, ref, beta, eps, alpha)
        dz = T().preference_loss_backward(z, y, saved)
        want, tol = preference_oracle(z, y, cu, ref, beta, eps, alpha, dtype)
        for got, a, t, n in zip((loss, logps, dz), want, tol, ("loss", "logps", "dz")):
            within(got, a, t, n)
        assert dz.dtype == dtype and not dz[(y < 0) | (y >= V)].any() and not dz[cu[-1]:].any()


@pytest.mark.parametrize("lens", [[2500, 700, 1, 5000], [513, 2049, 512, 2048], [3] * 1300])
def test_preference_long_sequences_many_pairs_and_a_lead(lens):
    """Sequences beyond one turn of a workgroup, more pairs than a workgroup has threads, tokens before the first sequence."""
    z, y, cu, cut, ref, _ = preference_inputs(len(lens), lens, 33, torch.float32, tail=3, lead=11)
    loss, logps, saved = T().preference_loss_forward(z, y, cut, ref, 0.02, 0.1, 0.3)
    dz = T().preference_loss_backward(z, y, saved)
    want, tol = preference_oracle(z, y, cu, ref, 0.02, 0.1, 0.3, torch.float32)
    for got, a, t, n in zip((loss, logps, dz), want, tol, ("loss", "logps", "dz")):
        within(got, a, t, n)
    assert not dz[:11].any() and not dz[cu[-1]:].any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [60, 1024])
def test_preference_margin_of_a_long_sequence_has_no_bias(V, dtype):
    """A margin of 40000 tokens: errors that go either way add up to the root of their number, a bias to all of it.  A token's
    log-probability takes some dozens of roundings of at most u each: below 8 u in root mean square, and six standard deviations
    of 40000 of them are asked.  One logit above the others by log V: half of the sum lies that far below the maximum."""
    n = 40000
    g = gen(V)
    z = 0.3 * randn(g, n, V)
    z[:, V // 3] += math.log(V)
    z = z.to(dtype)
    y = torch.randint(0, V, (n,), generator=g, device="cuda")
    want = torch.log_softmax(z.double(), -1).gather(1, y[:, None]).sum()
    cut = torch.tensor([0, n, n], dtype=torch.int32, device="cuda")
    ref = torch.stack([want, torch.zeros_like(want)]).float()  # a margin near zero: the loss shows its error
    loss, logps, saved = T().preference_loss_forward(z, y, cut, ref, beta=1.0)
    m = want - ref[0].double()
    error = 6 * 8 * U * n ** 0.5
    exact = torch.nn.functional.softplus(-m)
    assert abs(loss.double() - exact) <= error * torch.sigmoid(-m) + U * exact
    dz = T().preference_loss_backward(z, y, saved)
    c = -torch.sigmoid(-m)
    p = torch.log_softmax(z.double(), -1).exp()
    grad = c * (torch.nn.functional.one_hot(y, V) - p)
    # the coefficient is off by the margin's error times sigmoid(m); a probability has a few roundings of its own
    tol = (error * torch.sigmoid(m) + 4 * U) * grad.abs() + 16 * U * c.abs() * p
    within(dz, grad, tol * (1 + R[dtype]) + R[dtype] * grad.abs(), "dz")


def test_preference_more_than_2_31_elements():
    """Logits and gradients past 2^32 bytes: the last pair against the same pair alone (half the weight among two pairs)."""
    z1, y1, cu, cut, ref, _ = preference_inputs(19, [300, 211], 4096, torch.bfloat16)
    times = 1040
    z, y = z1.repeat(times, 1), y1.repeat(times)
    assert z.numel() > 2 ** 31
    N = len(y)
    cu2 = torch.tensor([0, 400, N - 511, N - 211, N], dtype=torch.int32, device="cuda")
    loss, logps, saved = T().preference_loss_forward(z, y, cu2, torch.cat([ref, ref]))
    dz = T().preference_loss_backward(z, y, saved)
    a, b, c = T().preference_loss_forward(z1, y1, cut, ref)
    assert torch.equal(logps[2:], b)
    assert torch.equal(dz[-511:], T().preference_loss_backward(z1, y1, c, torch.full((), 0.5, device="cuda")))


def test_preference_skipped_tokens_may_hold_anything():
    z, y, cu, cut, ref, _ = preference_inputs(8, [20, 30, 10, 15], 65, torch.float32, tail=9)
    a = T().preference_loss_forward(z, y, cut, ref, 0.1, 0.1, 0.5)
    z2, y2 = z.clone(), y.clone()
    z2[y < 0] = math.nan
    z2[cu[-1]:] = math.inf
    b = T().preference_loss_forward(z2, y2, cut, ref, 0.1, 0.1, 0.5)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    assert torch.equal(T().preference_loss_backward(z, y, a[2]), T().preference_loss_backward(z2, y2, b[2]))
    # vocabulary entries that are ruled out (-inf, or the type's lowest value), and a long way between logits
    for fill in (-math.inf, torch.finfo(torch.float32).min):
        z3 = z.clone()
        z3[:, ::3] = fill
        y3 = torch.where(y % 3 == 0, torch.full_like(y, -100), y)
        for s in (1.0, 200.0):
            zs = torch.where(z3 == fill, z3, z3 * s)
            got = T().preference_loss_forward(zs, y3, cut, ref)
            dz = T().preference_loss_backward(zs, y3, got[2])
            zo = zs.double().masked_fill(z3 == fill, -1e30)
            want, tol = preference_oracle(zo, y3, cu, ref, 0.1, 0.0, 0.0, torch.float32)
            keep = z3 != fill
            within(got[0], want[0], tol[0], "loss")
            assert not dz[~keep].any()
            within(dz[keep], want[2][keep], tol[2][keep], "dz")


def test_preference_autograd_and_differences():
    z, y, cu, cut, ref, g = preference_inputs(13, [25, 31, 12, 40], 64, torch.float32)
    x = z.clone().requires_grad_()
    loss, logps = T().preference_loss(x, y, cut, ref, beta=0.3, label_smoothing=0.1, nll_weight=0.2)
    assert loss.requires_grad and not logps.requires_grad
    (loss * 2.5).backward()
    want, tol = preference_oracle(z, y, cu, ref, 0.3, 0.1, 0.2, torch.float32)
    within(x.grad, 2.5 * want[2], 2.5 * tol[2] + 2 * U * 2.5 * want[2].abs(), "autograd")
    v = randn(g, *z.shape).double()
    f = lambda s: preference_oracle(z.double() + s * v, y, cu, ref, 0.3, 0.1, 0.2, torch.float32)[0][0].item()
    slope = 2.5 * (f(1e-4) - f(-1e-4)) / 2e-4
    assert abs((x.grad.double() * v).sum().item() - slope) <= 3 * (tol[2] * v.abs()).sum().item() + 1e-6 * (want[2].abs() * v.abs()).sum().item()


# ------------------------------------------------------------------------------------------------ together

class Block:
    """A pre-norm attention sublayer (reference esm/layers/attention.py:26-33, blocks.py:146-155) and a vocabulary head."""

    def __init__(self, d, H, V, seed, dtype=torch.float32):
        g = gen(seed)
        p = lambda *s, m=0.0, w=0.1: (m + w * randn(g, *s)).to(dtype)
        self.d, self.H = d, H
        self.p = {"ln_w": p(d, m=1), "ln_b": p(d), "w_qkv": p(3 * d, d, w=d ** -0.5), "q_ln": p(d, m=1), "k_ln": p(d, m=1),
                  "w_o": p(d, d, w=d ** -0.5), "f_ln": p(d, m=1), "w_v": p(V, d, w=d ** -0.5)}

    def run(self, x, p, norm, attend):
        N, d = x.shape
        qkv = norm(x, p["ln_w"], p["ln_b"]) @ p["w_qkv"].t()
        q, k, v = norm(qkv[:, :d], p["q_ln"], None), norm(qkv[:, d:2 * d], p["k_ln"], None), qkv[:, 2 * d:]
        heads = lambda t: t.reshape(N, self.H, d // self.H)
        x = x + attend(heads(q), heads(k), heads(v)).reshape(N, d) @ p["w_o"].t()
        return norm(x, p["f_ln"], None) @ p["w_v"].t()


def plain_norm(x, w, b):
    h = (x - x.mean(-1, keepdim=True)) / ((x - x.mean(-1, keepdim=True)).pow(2).mean(-1, keepdim=True) + 1e-5).sqrt()
    return h * w + (0 if b is None else b)


def plain_attend(cu, keep):
    def go(q, k, v):
        out = torch.zeros_like(q)
        for a, b in zip(cu, cu[1:]):
            s = torch.einsum("qhd,khd->hqk", q[a:b], k[a:b]) * q.shape[2] ** -0.5
            s = s.masked_fill(~keep[a:b], -math.inf)
            out = torch.cat([out[:a], torch.einsum("hqk,khd->qhd", s.softmax(-1), v[a:b]), out[b:]])
        return out
    return go


def test_preference_step_through_a_block():
    """Loss and every parameter's gradient of norm -> qkv -> q/k norm -> attention -> residual -> norm -> head -> loss against
    64-bit autograd.  The bf16 roundings on the way (eleven per path: activations, q k v, P, dS, their gradients) are
    independent: relative errors of sqrt(11) 2^-8 = 1.3 % of the norm at most; 2 % is asked."""
    d, H, V = 128, 2, 64
    blk = Block(d, H, V, 1)
    z, y, cu, cut, ref, g = preference_inputs(17, [60, 75, 130, 20], V, torch.float32)
    N = cu[-1]
    keep = torch.rand(N, generator=g, device="cuda") > 0.2
    keep[cu[:-1]] = True
    x0 = randn(g, N, d)
    ref = -4.0 * torch.tensor([60.0, 75, 130, 20], device="cuda") * 0.75
    p16 = {n: t.clone().requires_grad_() for n, t in blk.p.items()}
    bf = lambda x, w, b: T().layer_norm(x.bfloat16(), w, b)
    low = {n: (t if "ln" in n else t.bfloat16()) for n, t in p16.items()}
    logits = blk.run(x0.bfloat16(), low, bf, lambda q, k, v: T().attention_varlen(q, k, v, cut, key_mask=keep))
    loss, logps = T().preference_loss(logits.float(), y, cut, ref, nll_weight=0.1)
    loss.backward()
    p64 = {n: (t.double() if "ln" in n else t.bfloat16().double()).requires_grad_() for n, t in blk.p.items()}
    lg = blk.run(x0.bfloat16().double(), p64, plain_norm, plain_attend(cu, keep))
    lp = torch.log_softmax(lg, -1)
    l = torch.stack([lp[a:b][y[a:b] >= 0].gather(1, y[a:b][y[a:b] >= 0][:, None]).sum() for a, b in zip(cu, cu[1:])])
    m = 0.1 * ((l - ref)[0::2] - (l - ref)[1::2])
    n = torch.tensor([int((y[a:b] >= 0).sum()) for a, b in zip(cu, cu[1:])], device="cuda")
    want = (torch.nn.functional.softplus(-m) - 0.1 * l[0::2] / n[0::2]).mean()
    want.backward()
    assert abs(loss.item() - want.item()) <= 0.02 * abs(want.item())
    assert (logps.double() - l).norm() <= 0.02 * l.norm()
    for name, t in p16.items():
        g64 = p64[name].grad
        assert (t.grad.double() - g64).norm() <= 0.02 * g64.norm(), name


def _step(x, dy, w, b, q, k, v, cu, dout, mask, z, y, cp, ref):
    n, st = T().layer_norm_forward(x, w, b)
    got = [n, st, *T().layer_norm_backward(dy, x, w, st)]
    got += attention_all(q, k, v, cu, dout, mask=mask)
    loss, lp, saved = T().preference_loss_forward(z, y, cp, ref, nll_weight=0.5)
    return got + [loss, lp, T().preference_loss_backward(z, y, saved)]


def _step_inputs(seed):
    g = gen(seed)
    q, k, v, _, cu, dout, _ = attention_inputs(seed, [100, 31, 200], 4, 2, 64, tail=3)
    z, y, _, cp, ref, _ = preference_inputs(seed, [40, 50, 33, 21], 64, torch.float32)
    return [randn(g, 600, 384).bfloat16(), randn(g, 600, 384).bfloat16(), 1 + 0.1 * randn(g, 384), randn(g, 384), q, k, v, cu,
            dout, torch.rand(len(q), generator=g, device="cuda") > 0.1, z, y, cp, ref]


def test_same_bits_again_on_other_streams_and_in_a_replayed_graph():
    a, b = _step_inputs(1), _step_inputs(2)
    b[7], b[12] = a[7], a[12]
    ea, eb = _step(*a), _step(*b)
    for p, q in zip(ea, _step(*a)):
        assert torch.equal(p, q)
    # two streams at once, each with its own outputs and scratch memory
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    got = []
    for s, args in ((s1, a), (s2, b), (s1, b), (s2, a)):
        with torch.cuda.stream(s):
            got.append(_step(*args))
    torch.cuda.synchronize()
    for out, want in zip(got, (ea, eb, eb, ea)):
        for p, q in zip(out, want):
            assert torch.equal(p, q)
    # one captured step, replayed with other inputs in its buffers and eager work in between
    bufs = [t.clone() for t in a]
    with torch.cuda.stream(s1):
        _step(*bufs)
    torch.cuda.synchronize()
    graph, graph2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = _step(*bufs)
    with torch.cuda.graph(graph2):
        outs2 = _step(*b)
    for args, want in ((b, eb), (a, ea), (b, eb)):
        for t, s in zip(bufs, args):
            t.copy_(s)
        graph.replay()
        graph2.replay()
        mid = _step(*a)
        torch.cuda.synchronize()
        for o, w in ((outs, want), (outs2, eb), (mid, ea)):
            for p, q in zip(o, w):
                assert torch.equal(p, q)


def test_the_stream_of_a_call_is_the_current_one():
    gpu = torch.cuda.current_device()
    side = torch.cuda.Stream()
    for s in (torch.cuda.current_stream(), side):
        with torch.cuda.stream(s):
            assert T()._stream(gpu) == T()._public_stream(gpu) == s.cuda_stream


@pytest.mark.parametrize("H,G", [(2, 1), (150, 75)])
def test_attention_graph_follows_the_offsets(H, G):
    """The order of the blocks is formed on the GPU: a captured step holds for other offsets, with few blocks and with many."""
    n = 700
    sets = []
    for seed, lens in ((1, [100, 31, 500]), (2, [1, 600, 20]), (3, [0, 0, 700]), (4, [233, 233, 234])):
        q, k, v, _, cu, dout, g = attention_inputs(seed, lens, H, G, 64, tail=n - sum(lens))
        sets.append([q.contiguous(), k.contiguous(), v.contiguous(), cu, dout, torch.rand(n, generator=g, device="cuda") > 0.1])
    step = lambda q, k, v, cu, dout, mask: attention_all(q, k, v, cu, dout) + attention_all(q, k, v, cu, dout, mask=mask)
    want = [step(*s) for s in sets]
    bufs = [t.clone() for t in sets[0]]
    s1 = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s1):
        step(*bufs)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(*bufs)
    for i in (1, 0, 2, 3, 1):
        for t, s in zip(bufs, sets[i]):
            t.copy_(s)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, want[i]):
            assert torch.equal(a, b)


def test_refusals_name_the_argument():
    t = T()
    x, w = torch.zeros(4, 64, device="cuda"), torch.ones(64, device="cuda")
    q = torch.zeros(8, 2, 64, dtype=torch.bfloat16, device="cuda")
    cu = torch.tensor([0, 8], dtype=torch.int32, device="cuda")
    y = torch.zeros(8, dtype=torch.int64, device="cuda")
    z = torch.zeros(8, 16, device="cuda")
    cp, ref = torch.tensor([0, 4, 8], dtype=torch.int32, device="cuda"), torch.zeros(2, device="cuda")
    y0, st = t.layer_norm_forward(x, w)
    o, lse = t.attention_varlen_forward(q, q, q, cu)
    for err, call in (
            (ValueError, lambda: t.layer_norm_forward(x, w[:32])), (ValueError, lambda: t.layer_norm_forward(x, w, w[:1])),
            (TypeError, lambda: t.layer_norm_forward(x.half(), w)), (ValueError, lambda: t.layer_norm_backward(x[:2], x, w, st)),
            (TypeError, lambda: t.layer_norm_backward(x.bfloat16(), x, w, st)),
            (ValueError, lambda: t.layer_norm_backward(x, x, w, st[:2])),
            (ValueError, lambda: t.layer_norm_forward(torch.zeros(1, 12289, device="cuda"), torch.ones(12289, device="cuda"))),
            (TypeError, lambda: t.attention_varlen_forward(q.float(), q, q, cu)),
            (ValueError, lambda: t.layer_norm_forward(x[:1, :1].expand(2 ** 30 + 1, 1), w[:1])),
            (ValueError, lambda: t.attention_varlen_forward(q[:, :, :32], q[:, :, :32], q[:, :, :32], cu)),
            (ValueError, lambda: t.attention_varlen_forward(q, q[:, :1].expand(8, 3, 64), q[:, :1].expand(8, 3, 64), cu)),
            (ValueError, lambda: t.attention_varlen_forward(q, q[:4], q[:4], cu)),
            (TypeError, lambda: t.attention_varlen_forward(q, q, q, cu.long())),
            (ValueError, lambda: t.attention_varlen_forward(q, q, q, cu, scale=-1.0)),
            (ValueError, lambda: t.attention_varlen_forward(q, q, q, cu, scale=0.0)),
            (ValueError, lambda: t.attention_varlen_forward(q, q, q, cu, key_mask=torch.ones(7, dtype=torch.bool, device="cuda"))),
            (ValueError, lambda: t.attention_varlen_backward(o, q, q, q, o, lse[:1], cu)),
            (ValueError, lambda: t.preference_loss_forward(z, y[:4], cp, ref)),
            (ValueError, lambda: t.preference_loss_forward(z, y, cu, ref)),
            (ValueError, lambda: t.preference_loss_forward(z, y, cp, ref[:1])),
            (ValueError, lambda: t.preference_loss_forward(z, y, cp[:1].expand(2 ** 24 + 1).contiguous(), ref)),
            (ValueError, lambda: t.preference_loss_forward(z, y, cp, ref, label_smoothing=1.5)),
            (TypeError, lambda: t.preference_loss_forward(z, y.int(), cp, ref)),
            (ValueError, lambda: t.preference_loss_backward(z, y, torch.zeros(8, device="cuda")))):
        with pytest.raises(err):
            call()
