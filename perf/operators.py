"""Cases of the operators that fine-tuning the trunk needs: LayerNorm with its gradients, block-diagonal attention with
its gradients, and the paired preference loss with its gradient.

`run` computes a case in plain torch operations (32 bits, 64 where a long sum needs them, rounded once at the end) or,
with `own` set, through esm_amd.training.  `exact` is the same mathematics in 64 bits, written apart from `run`.

Formulas
  layer norm   mu, var over the row; r = 1/sqrt(var + eps); h = (x - mu) r; y = h w + b
               g = dy w; dx = r (g - mean g - h mean(g h)); dw = sum_rows dy h; db = sum_rows dy
  attention    per sequence and head: S = scale Q K^T, masked keys -inf; P = softmax S; O = P V; lse = log sum exp S
               dV = P^T dO; D = rowsum(dO O); dS = P (dO V^T - D) scale; dQ = dS K; dK = dS^T Q
               query heads share key heads in groups; a row without keys gives O = 0, lse = -inf and no gradient;
               tokens behind the last sequence give zeros
  preference   l_s = sum of log softmax(z_t)[y_t] over the scored tokens of sequence s (0 <= y_t < V, others are skipped)
               m_i = beta ((l_2i - ref_2i) - (l_2i+1 - ref_2i+1))
               L = mean_i [(1 - e) softplus(-m_i) + e softplus(m_i) - a l_2i / max(1, scored_2i)];  dL/dz
"""
import random

import torch

own = False

_DT = {"bf16": torch.bfloat16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f32": 4}


def _ln(name, dir, rows, d, dtype, bias, wide=1):
    return {"name": name, "op": "layer_norm", "dir": dir, "rows": rows, "d": d, "dtype": dtype, "bias": bias, "wide": wide}


def _at(name, dir, n_seg, lo, hi, heads, kv_heads, head_dim, masked=False, tail=0, mix=0):
    return {"name": name, "op": "attention", "dir": dir, "n_seg": n_seg, "min_len": lo, "max_len": hi, "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "masked": masked, "tail": tail, "mix": mix}


def _pl(name, dir, pairs, lo, hi, vocab, dtype, tail=0, mix=0):
    return {"name": name, "op": "preference", "dir": dir, "pairs": pairs, "min_len": lo, "max_len": hi, "vocab": vocab,
            "dtype": dtype, "beta": 0.1, "smoothing": 0.05, "nll_weight": 0.2, "tail": tail, "mix": mix}


def listed():
    return [
        # the final norm of one short protein at scoring time: launch latency is all there is
        _ln("norm of one protein", "forward", 66, 960, "bf16", False),
        # a block's input norm over a 64 x 512 batch of the 1152-wide trunk: the ordinary training step
        _ln("norm of a batch", "train", 32768, 1152, "bf16", True),
        # q_ln inside the wide qkv projection of the 2560-wide trunk at 4 x 4096: rows of a wider buffer, no bias
        _ln("q norm of a wide trunk", "train", 16384, 2560, "bf16", False, wide=3),
        # fp32 rows of an odd width and an odd count: no vector of 16 bytes fits
        _ln("norm of odd rows", "train", 4099, 1281, "f32", True),
        # three short proteins, two heads: the smallest training batch
        _at("attention of three proteins", "train", 3, 21, 64, 2, 2, 64, mix=1),
        # the forward half of a 64 x 512 batch with 18 heads, as gradient checkpointing runs it
        _at("attention of a batch", "forward", 64, 512, 512, 18, 18, 64),
        # the same batch's training step
        _at("attention step of a batch", "train", 64, 512, 512, 18, 18, 64),
        # 4 x 4096 with 40 heads: long contexts, the largest
        _at("attention step of long chains", "train", 4, 4096, 4096, 40, 40, 64),
        # ragged complexes with padded residues masked out, shared key heads, head dim 128, buffer longer than the batch
        _at("attention step of ragged chains", "train", 24, 217, 1031, 16, 4, 128, masked=True, tail=77, mix=2),
        # one pair of short designs over the 64-entry sequence vocabulary
        _pl("preference of one pair", "train", 1, 90, 130, 64, "f32", mix=3),
        # 32 pairs of 512-residue designs over the sequence vocabulary
        _pl("preference of a batch", "train", 32, 512, 512, 64, "f32"),
        # 10 ragged pairs over the structure-token vocabulary, bf16 logits
        _pl("preference of structure tokens", "train", 10, 200, 1024, 4096, "bf16", tail=19, mix=4),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(("layer_norm", "attention", "preference"))
    way = rng.choice(("forward", "train", "train"))
    if op == "layer_norm":
        d = rng.choice((_log(rng, 33, 4096), 64 * rng.randint(1, 64)))
        rows = _log(rng, 1, min(32768, 32768 * 1152 // d))
        c = _ln("", way, rows, d, rng.choice(("bf16", "f32")), rng.random() < 0.5, rng.choice((1, 1, 3)))
    elif op == "attention":
        kv, group = rng.choice((1, 2, 3, 5, 8)), rng.choice((1, 1, 2, 4))
        head_dim = rng.choice((64, 64, 128))
        # from 4 keys on: where every query has one key alone, dq and dk are zero and their rounding is all that is left
        hi, n = _log(rng, 4, 4096), _log(rng, 1, 64)
        while n * hi > 32768 or n * hi * hi * kv * group * head_dim > 2 * 40 * 4096 ** 2 * 64:
            n, hi = (n // 2, hi) if n > 1 else (n, hi // 2)
        lo = hi if rng.random() < 0.3 else max(1, hi // rng.randint(2, 8))
        c = _at("", way, n, lo, hi, kv * group, kv, head_dim, rng.random() < 0.5 and lo >= 8, rng.choice((0, rng.randint(1, 200))), rng.randint(0, 10 ** 6))
    else:
        vocab = rng.choice((64, _log(rng, 5, 8192)))
        hi, pairs = _log(rng, 1, 1024), _log(rng, 1, 64)
        while 2 * pairs * hi * vocab > 32768 * 2560:
            pairs, hi = (pairs // 2, hi) if pairs > 1 else (pairs, hi // 2)
        lo = hi if rng.random() < 0.3 else max(1, hi // rng.randint(2, 8))
        c = _pl("", way, pairs, lo, hi, vocab, rng.choice(("bf16", "f32")), rng.choice((0, rng.randint(1, 200))), rng.randint(0, 10 ** 6))
        c["beta"], c["smoothing"], c["nll_weight"] = rng.choice((0.05, 0.1, 0.5)), rng.choice((0.0, 0.1)), rng.choice((0.0, 1.0))
    del c["name"]
    return c


def _lengths(case):
    """Lengths of the sequences, the longest among them: a property of the case, not of the seed."""
    n = case["n_seg"] if case["op"] == "attention" else 2 * case["pairs"]
    rng = random.Random(case["mix"])
    ls = [rng.randint(case["min_len"], case["max_len"]) for _ in range(n)]
    ls[rng.randrange(n)] = case["max_len"]
    return ls


def _offsets(lengths):
    cu = [0]
    for n in lengths:
        cu.append(cu[-1] + n)
    return cu


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    def rand(*shape):
        return torch.rand(*shape, generator=gen, device="cuda")

    s = dict(case)
    if case["op"] == "layer_norm":
        rows, d, dt = case["rows"], case["d"], _DT[case["dtype"]]
        # a residual stream: channels of unequal size and offset
        x = (randn(rows, case["wide"] * d) * (0.5 + rand(case["wide"] * d)) + 0.3 * randn(case["wide"] * d)).to(dt)
        s["x"] = x[:, :d]
        s["w"] = 1 + 0.1 * randn(d)
        s["b"] = 0.1 * randn(d) if case["bias"] else None
        s["dy"] = (0.02 * randn(rows, d)).to(dt) if case["dir"] == "train" else None
        return s
    lengths = _lengths(case)
    cu = _offsets(lengths)
    N = cu[-1] + case["tail"]
    s["cu"] = torch.tensor(cu, dtype=torch.int32, device="cuda")
    if case["op"] == "attention":
        H, G, D = case["heads"], case["kv_heads"], case["head_dim"]
        qkv = randn(N, H + 2 * G, D).to(torch.bfloat16)  # as the fused projection lays them out
        s["q"], s["k"], s["v"] = qkv[:, :H], qkv[:, H:H + G], qkv[:, H + G:]
        s["scale"] = 1.5 / D ** 0.5
        s["mask"] = None
        if case["masked"]:  # one key in eight is padding; every key of the first of several sequences is
            s["mask"] = rand(N) > 0.125
            if len(lengths) > 1:
                s["mask"][:lengths[0]] = False
        s["dout"] = (0.05 * randn(N, H, D)).to(torch.bfloat16) if case["dir"] == "train" else None
        return s
    V, P = case["vocab"], case["pairs"]
    z = 1.5 * randn(N, V)
    y = torch.randint(0, V, (N,), generator=gen, device="cuda")
    y[rand(N) > 0.75] = -100  # positions that are not scored
    s["z"], s["y"] = z.to(_DT[case["dtype"]]), y
    # the frozen model's log-probabilities: those of nearby logits
    t = (z + 0.2 * randn(N, V)).log_softmax(-1).gather(1, y.clamp(min=0)[:, None])[:, 0].masked_fill(y < 0, 0.0).double()
    t = torch.cat([t.new_zeros(1), t.cumsum(0)])
    s["ref"] = (t[s["cu"][1:].long()] - t[s["cu"][:-1].long()]).float()
    return s


# ------------------------------------------------------------------------------------------ plain forms

def _plain_norm(s):
    x, w, b = s["x"].float(), s["w"], s["b"]
    xc = x - x.mean(-1, keepdim=True)
    r = torch.rsqrt((xc * xc).mean(-1, keepdim=True) + 1e-5)
    h = xc * r
    y = h * w
    if b is not None:
        y = y + b
    y = y.to(s["x"].dtype)
    if s["dy"] is None:
        return y
    dy = s["dy"].float()
    g = dy * w
    dx = (g - g.mean(-1, keepdim=True) - h * (g * h).mean(-1, keepdim=True)) * r
    dw = (dy * h).sum(0)
    return (y, dx.to(s["x"].dtype), dw) + (() if b is None else (dy.sum(0),))


def _plain_attention(s):
    q, cu, L = s["q"], s["cu"].long(), s["max_len"]
    N, H, D = q.shape
    G = s["kv_heads"]
    # sequences side by side, padded to the longest, and the way back
    col = torch.arange(L, device=q.device)
    at = (cu[:-1, None] + col).clamp(max=N - 1)
    real = col < (cu[1:] - cu[:-1])[:, None]
    tok = torch.arange(N, device=q.device)
    seg = (torch.searchsorted(cu, tok, right=True) - 1).clamp(max=len(cu) - 2)
    pos, inside = (tok - cu[seg]).clamp(max=L - 1), tok < cu[-1]

    def pad(x):
        return x[at].float().transpose(1, 2).contiguous()

    def back(x):  # [S, heads, L, D] -> [N, heads, D]
        return (x[seg, :, pos] * inside[:, None, None]).to(torch.bfloat16)

    def share(x):
        return x if G == H else x.repeat_interleave(H // G, 1)

    def gather(x):
        return x if G == H else x.unflatten(1, (G, H // G)).sum(2)

    qp, kp, vp = pad(q), share(pad(s["k"])), share(pad(s["v"]))
    keep = real if s["mask"] is None else real & s["mask"][at]
    p = torch.matmul(qp, kp.transpose(-1, -2).contiguous()).mul_(s["scale"])
    p.masked_fill_(~keep[:, None, None, :], float("-inf"))
    top = p.amax(-1, keepdim=True)
    top = torch.where(top == float("-inf"), torch.zeros_like(top), top)
    p.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    some = total > 0
    p.div_(torch.where(some, total, torch.ones_like(total)))
    o = torch.matmul(p, vp)
    lse = torch.where(some, top + total.log(), torch.full_like(top, float("-inf")))[..., 0]
    lse = (lse[seg, :, pos] * 1.0).masked_fill(~inside[:, None], float("-inf")).t().contiguous()
    if s["dout"] is None:
        return back(o), lse
    do = pad(s["dout"]) * real[:, None, :, None]
    dv = torch.matmul(p.transpose(-1, -2).contiguous(), do)
    ds = torch.matmul(do, vp.transpose(-1, -2).contiguous())
    ds.sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(s["scale"])
    dq = torch.matmul(ds, kp)
    dk = torch.matmul(ds.transpose(-1, -2).contiguous(), qp)
    return back(o), lse, back(dq), back(gather(dk)), back(gather(dv))


def _plain_preference(s):
    z, y, cu = s["z"].float(), s["y"], s["cu"].long()
    N, V = z.shape
    S = len(cu) - 1
    tok = torch.arange(N, device=z.device)
    seg = torch.searchsorted(cu, tok, right=True) - 1
    used = (y >= 0) & (y < V) & (tok < cu[-1])
    at = torch.where(used, y, torch.zeros_like(y))[:, None]
    top = z.amax(-1, keepdim=True)
    e = (z - top).exp()
    total = e.sum(-1, keepdim=True)
    logp = ((z.gather(1, at) - top).double() - total.double().log())[:, 0]
    logp = torch.where(used, logp, torch.zeros_like(logp))
    l = torch.zeros(S + 1, dtype=torch.float64, device=z.device).index_add_(0, seg, logp)[:S]
    n = torch.zeros(S + 1, dtype=torch.float64, device=z.device).index_add_(0, seg, used.double())[:S].clamp(min=1)
    gain = l - s["ref"].double()
    m = s["beta"] * (gain[0::2] - gain[1::2])
    eps, a = s["smoothing"], s["nll_weight"]

    def softplus(x):
        return x.clamp(min=0) + (1 + (-x.abs()).exp()).log()

    loss = ((1 - eps) * softplus(-m) + eps * softplus(m) - a * l[0::2] / n[0::2]).mean().float()
    if s["dir"] == "forward":
        return loss, l.float()
    up = 1 / (1 + (-m).exp())
    gm = s["beta"] * (eps * up - (1 - eps) * (1 - up)) / (S // 2)
    coef = torch.zeros(S + 1, dtype=torch.float64, device=z.device)
    coef[0:S:2] = gm - a / n[0::2] / (S // 2)
    coef[1:S:2] = -gm
    coef = torch.where(used, coef[seg], torch.zeros_like(logp)).float()[:, None]
    dz = e.div_(total).mul_(-coef).scatter_add_(1, at, coef)
    return loss, l.float(), dz.to(s["z"].dtype)


def run(s):
    if own:
        from esm_amd import training as T
        if s["op"] == "layer_norm":
            y, stats = T.layer_norm_forward(s["x"], s["w"], s["b"])
            if s["dy"] is None:
                return y
            dx, dw, db = T.layer_norm_backward(s["dy"], s["x"], s["w"], stats, bias=s["b"] is not None)
            return (y, dx, dw) + (() if db is None else (db,))
        if s["op"] == "attention":
            out, lse = T.attention_varlen_forward(s["q"], s["k"], s["v"], s["cu"], scale=s["scale"], key_mask=s["mask"])
            if s["dout"] is None:
                return out, lse
            return (out, lse) + tuple(T.attention_varlen_backward(s["dout"], s["q"], s["k"], s["v"], out, lse, s["cu"],
                                                                  scale=s["scale"], key_mask=s["mask"]))
        loss, logps, saved = T.preference_loss_forward(s["z"], s["y"], s["cu"], s["ref"], beta=s["beta"],
                                                       label_smoothing=s["smoothing"], nll_weight=s["nll_weight"])
        if s["dir"] == "forward":
            return loss, logps
        return loss, logps, T.preference_loss_backward(s["z"], s["y"], saved)
    return {"layer_norm": _plain_norm, "attention": _plain_attention, "preference": _plain_preference}[s["op"]](s)


# ------------------------------------------------------------------------------------------ 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    train = case["dir"] == "train"
    if case["op"] == "layer_norm":
        x, w = s["x"].double(), s["w"].double()
        var, mu = torch.var_mean(x, -1, correction=0, keepdim=True)
        sd = (var + 1e-5).sqrt()
        h = (x - mu) / sd
        y = h * w + (0 if s["b"] is None else s["b"].double())
        if not train:
            return y
        dy = s["dy"].double()
        dh = dy * w
        d = case["d"]
        dx = (d * dh - dh.sum(-1, keepdim=True) - h * (dh * h).sum(-1, keepdim=True)) / (d * sd)
        return (y, dx, (dy * h).sum(0)) + (() if s["b"] is None else (dy.sum(0),))
    cu = _offsets(_lengths(case))
    if case["op"] == "attention":
        q, k, v, mask = s["q"], s["k"], s["v"], s["mask"]
        N, H, D = q.shape
        group = H // case["kv_heads"]
        o, dq = (torch.zeros(N, H, D, dtype=torch.float64, device=q.device) for _ in range(2))
        dk, dv = (torch.zeros(N, H // group, D, dtype=torch.float64, device=q.device) for _ in range(2))
        lse = torch.full((H, N), float("-inf"), dtype=torch.float64, device=q.device)
        for a, b in zip(cu, cu[1:]):
            keys = torch.arange(a, b, device=q.device)
            if mask is not None:
                keys = keys[mask[a:b]]
            if len(keys) == 0:
                continue
            step = max(1, (1 << 28) // ((b - a) * len(keys)))  # heads at a time: about 2 GB a matrix
            for h0 in range(0, H, step):
                hs = torch.arange(h0, min(H, h0 + step), device=q.device)
                gs = hs // group
                Q = q[a:b].double()[:, hs].transpose(0, 1).contiguous()
                K = k[keys].double()[:, gs].transpose(0, 1).contiguous()
                V = v[keys].double()[:, gs].transpose(0, 1).contiguous()
                S = Q @ K.transpose(1, 2).contiguous() * s["scale"]
                ls = torch.logsumexp(S, -1, keepdim=True)
                P = torch.exp(S - ls)
                O = P @ V
                o[a:b, hs] = O.transpose(0, 1)
                lse[hs, a:b] = ls[..., 0]
                if train:
                    dO = s["dout"][a:b].double()[:, hs].transpose(0, 1).contiguous()
                    dP = dO @ V.transpose(1, 2).contiguous()
                    dS = P * (dP - (P * dP).sum(-1, keepdim=True)) * s["scale"]
                    dq[a:b, hs] = (dS @ K).transpose(0, 1)
                    gk, gv = dS.transpose(1, 2).contiguous() @ Q, P.transpose(1, 2).contiguous() @ dO
                    for j in range(len(hs)):
                        dk[keys, (h0 + j) // group] += gk[j]
                        dv[keys, (h0 + j) // group] += gv[j]
        return (o, lse, dq, dk, dv) if train else (o, lse)
    z, y = s["z"].double(), s["y"]
    logp = torch.log_softmax(z, -1)
    P = case["pairs"]
    dz = torch.zeros_like(z)
    l = torch.zeros(2 * P, dtype=torch.float64, device=z.device)
    terms = []
    for i in range(2 * P):
        rows = torch.arange(cu[i], cu[i + 1], device=z.device)
        rows = rows[y[rows] >= 0]
        l[i] = logp[rows, y[rows]].sum()
    for i in range(P):
        m = case["beta"] * ((l[2 * i] - s["ref"][2 * i].double()) - (l[2 * i + 1] - s["ref"][2 * i + 1].double()))
        rows = torch.arange(cu[2 * i], cu[2 * i + 1], device=z.device)
        n = max(1, int((y[rows] >= 0).sum()))
        e = case["smoothing"]
        terms.append(-(1 - e) * torch.nn.functional.logsigmoid(m) - e * torch.nn.functional.logsigmoid(-m) - case["nll_weight"] * l[2 * i] / n)
        if train:
            gm = (-(1 - e) * torch.sigmoid(-m) + e * torch.sigmoid(m)) * case["beta"] / P
            for j, c in ((2 * i, gm - case["nll_weight"] / n / P), (2 * i + 1, -gm)):
                rows = torch.arange(cu[j], cu[j + 1], device=z.device)
                rows = rows[y[rows] >= 0]
                dz[rows] = -c * logp[rows].exp()
                dz[rows, y[rows]] += c
    loss = torch.stack(terms).mean()
    return (loss, l, dz) if train else (loss, l)


def work(case):
    train = case["dir"] == "train"
    if case["op"] == "layer_norm":
        n, size = case["rows"] * case["d"], _SIZE[case["dtype"]]
        # x in, y out; the step also reads dy and writes dx (x once: the row could stay on the chip)
        par = case["d"] * 4 * (2 if case["bias"] else 1)
        return {"bytes": n * size * (4 if train else 2) + par * (2 if train else 1), "flops": n * (20 if train else 8)}
    lengths = _lengths(case)
    n = sum(lengths) + case["tail"]
    if case["op"] == "attention":
        H, G, D = case["heads"], case["kv_heads"], case["head_dim"]
        q, kv = n * H * D * 2, n * G * D * 2
        pairs = sum(a * a for a in lengths) * H
        # forward: q k v in, o and lse out, two products; backward: do in, dq dk dv out, five more
        return {"bytes": 2 * q + 2 * kv + 4 * n * H + (2 * q + 2 * kv if train else 0), "flops": (14 if train else 4) * pairs * D}
    b = n * case["vocab"] * _SIZE[case["dtype"]]
    return {"bytes": b * (2 if train else 1) + 8 * n, "flops": n * case["vocab"] * (8 if train else 4)}
