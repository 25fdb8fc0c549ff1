"""Oracle of the context operators (attention, gated feed-forward, residual norm): their definitions in fp64 on the CPU, with gradients
from autograd, and bounds on what an implementation may be off that holds sums in fp32 and rounds the documented values to the inputs'
type.  Checker only.  The operators have no counterpart in the reference ("parity unpinned"): this is their definition."""
import torch

F32 = 2.0 ** -24
# fp32 inputs: products of three bf16 planes each; the three of nine products that are dropped are below 2^-22 |a b|, and as much again is
# allowed for the rest (the partial sums' rounding inside the matrix pipe)
PLANES = {torch.float32: 2.0 ** -21, torch.bfloat16: 0.0, torch.float16: 0.0}


def half_step(dtype):
    """Largest relative error of one rounding to ``dtype``: half of ``finfo.eps``."""
    return torch.finfo(dtype).eps / 2


def visible(b, nq, nk, q_lens, kv_lens, key_mask, causal):
    """bool [b, nq, nk]"""
    i, j = torch.arange(nq)[None, :, None], torch.arange(nk)[None, None, :]
    ql = torch.full((b,), nq) if q_lens is None else q_lens.long().clamp(0, nq)
    kl = torch.full((b,), nk) if kv_lens is None else kv_lens.long().clamp(0, nk)
    ql, kl = ql[:, None, None], kl[:, None, None]
    ok = (i < ql) & (j < kl)
    if causal:
        ok = ok & (j - kl <= i - ql)
    if key_mask is not None:
        ok = ok & key_mask[:, None, :]
    return ok


def attention(q, k, v, grad=None, q_lens=None, kv_lens=None, key_mask=None, causal=False, scale=None):
    """-> (values, bounds): dicts with out and, given ``grad``, grad_q / grad_k / grad_v.  CPU tensors of the operator's dtype."""
    dt = q.dtype
    u, (b, nq, h, d), nk, hk = half_step(dt), q.shape, k.shape[1], k.shape[2]
    scale = d ** -0.5 if scale is None else scale
    ok = visible(b, nq, nk, q_lens, kv_lens, key_mask, causal)[:, None]
    hidden = ~ok.any(dim=2)                                                  # [b, 1, nk]: keys that no point sees
    Q, K, V = (t.detach().double().permute(0, 2, 1, 3) for t in (q, k, v))
    K, V = K.repeat_interleave(h // hk, 1), V.repeat_interleave(h // hk, 1)
    K, V = K.masked_fill(hidden[..., None], 0.0), V.masked_fill(hidden[..., None], 0.0)
    dead = ~ok.any(dim=3)                                                    # [b, 1, nq]: points that see nothing
    Q = Q.masked_fill(dead[..., None], 0.0)
    S = Q @ K.mT * scale
    P = torch.softmax(S.masked_fill(~ok, float("-inf")).masked_fill(dead[..., None], 0.0), -1) * ok
    O = P @ V
    acc = (d + 8) * F32 + PLANES[dt]
    ds = acc * scale * (Q.abs() @ K.abs().mT)                                # error of a score
    top = lambda t: (t * ok).amax(-1, keepdim=True) if nk else t.new_zeros(b, h, nq, 1)  # noqa: E731
    rel = 2 * top(ds) + top(S.abs()) * 4 * F32 + 2.0 ** -19
    sums = (nk ** 0.5 + 8) * F32 + PLANES[dt]
    o_err = u * O.abs() + (u * (dt != torch.float32) + rel + sums) * (P @ V.abs()) + tiny(dt)
    back = lambda t: t.permute(0, 2, 1, 3)  # noqa: E731
    fold = lambda t: back(t.reshape(b, hk, h // hk, nk, d).sum(2))  # noqa: E731
    val, err = {"out": back(O)}, {"out": back(o_err)}
    if grad is None:
        return val, err
    G = grad.detach().double().permute(0, 2, 1, 3).masked_fill(dead[..., None], 0.0)
    dP, delta = G @ V.mT, (G * O).sum(-1, keepdim=True)
    dS = P * (dP - delta)
    p16 = u if dt != torch.float32 else 0.0
    e_p = (2 * rel + p16) * P                                                # error of a probability
    e_dp = acc * (G.abs() @ V.abs().mT) + (G.abs() * (o_err - u * O.abs() * (dt != torch.float32) + 4 * F32 * O.abs())).sum(-1, keepdim=True) + acc * (G.abs() * O.abs()).sum(-1, keepdim=True)
    if dt == torch.float16 and nk:
        # fp16 holds 2^E dS with 30000 <= 2^E bound <= 60000, bound = 2 d max|dO| max|V| (a power of two below 60000 / bound): below fp16's
        # normal range one rounding is off by up to half of its smallest step, 2^-25, which is 2^-25 2^-E <= 2^-25 bound / 30000 of dS.
        # (Seen: a grad_k of 2.8e-8, itself below the normal range, off by 2^-25 + 4.2e-9, the latter 2^-25 2^-4 times |q| summed.)
        e_p = e_p + 2.0 ** -35 * ok                                          # P is held as 2^10 P
        floor = 2.0 ** -25 * 2 * d * float(G.abs().max()) * float(V.abs().max()) / 30000 * ok
    else:
        floor = 0.0
    e_ds = floor + (p16 + 8 * F32) * dS.abs() + e_p * (dP - delta).abs() + P * e_dp
    sums_q = (nq ** 0.5 * (h // hk) ** 0.5 + 8) * F32 + PLANES[dt]
    val["grad_q"], val["grad_k"], val["grad_v"] = back(dS @ K * scale), fold(dS.mT @ Q * scale), fold(P.mT @ G)
    err["grad_q"] = back((e_ds + sums * dS.abs()) @ K.abs() * scale)
    err["grad_k"] = fold((e_ds + sums_q * dS.abs()).mT @ Q.abs() * scale)
    err["grad_v"] = fold((e_p + sums_q * P).mT @ G.abs())
    for n in ("grad_q", "grad_k", "grad_v"):
        err[n] = err[n] + u * val[n].abs() + tiny(dt)
    return val, err


def tiny(dtype):
    """Half of the smallest step of the type (results below its normal range)."""
    return {torch.float32: 1e-38, torch.bfloat16: 1e-38, torch.float16: 2.0 ** -25}[dtype]


def _act(name, z):
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "gelu":
        return 0.5 * z * (1 + torch.erf(z / 2 ** 0.5))
    return z.clamp(min=0)


def feed_forward(x, w_gate, w_up, w_down, b_gate=None, b_up=None, b_down=None, grad=None, activation="silu"):
    """-> (values, bounds) with y and, given ``grad``, the gradients of every tensor given; x [rows, width]."""
    dt = x.dtype
    u, rows, (hidden, width), out = half_step(dt), x.shape[0], w_gate.shape, w_down.shape[0]
    names = ["x", "w_gate", "w_up", "w_down"] + [n for n, t in (("b_gate", b_gate), ("b_up", b_up), ("b_down", b_down)) if t is not None]
    t = dict(x=x, w_gate=w_gate, w_up=w_up, w_down=w_down, b_gate=b_gate, b_up=b_up, b_down=b_down)
    leaf = {n: t[n].detach().double().requires_grad_(grad is not None) for n in names}
    zero = torch.zeros((), dtype=torch.float64)
    z = leaf["x"] @ leaf["w_gate"].mT + leaf.get("b_gate", zero)
    up = leaf["x"] @ leaf["w_up"].mT + leaf.get("b_up", zero)
    h = _act(activation, z) * up
    y = h @ leaf["w_down"].mT + leaf.get("b_down", zero)
    val = {"y": y.detach()}
    if grad is not None:
        for n, g in zip(names, torch.autograd.grad(y, [leaf[n] for n in names], grad.detach().double())):
            val["grad_" + n] = g
    with torch.no_grad():
        p16, pl = (u if dt != torch.float32 else 0.0), PLANES[dt]
        acc = lambda n: (n ** 0.5 * 2 + 8) * F32 + pl  # noqa: E731     sums of n products: 2 sqrt(n) roundings, 6 sigma of a random walk
        X, Wg, Wu, Wd = (leaf[n].abs() for n in names[:4])
        e_z = acc(width) * (X @ Wg.mT + z.abs())
        e_u = acc(width) * (X @ Wu.mT + up.abs())
        a = _act(activation, z)
        zz = z.detach().clone().requires_grad_(True)
        with torch.enable_grad():
            da, = torch.autograd.grad(_act(activation, zz).sum(), zz)
        e_a = 1.13 * e_z + 16 * F32 * a.abs() + 4 * F32                      # |act'| < 1.13
        e_h = e_a * up.abs() + a.abs() * e_u + e_a * e_u + p16 * h.abs()
        err = {"y": u * y.abs() + (e_h + acc(hidden) * h.abs()) @ Wd.mT + 4 * F32 * y.abs() + tiny(dt)}
        if grad is not None:
            G = grad.detach().double()
            dh = G @ leaf["w_down"]
            e_dh = acc(out) * (G.abs() @ Wd)
            e_da = e_z * (0.8 if activation != "relu" else 0.0) + 32 * F32   # |act''| < 0.8
            if activation == "relu":
                e_da = e_da + (z.abs() <= e_z)
            dz, du = dh * up * da, dh * a
            e_dz = e_dh * (up * da).abs() + dh.abs() * (e_u * da.abs() + (up.abs() + e_u) * e_da) + p16 * dz.abs() + 8 * F32 * dz.abs() + p16 * tiny(dt)
            e_du = e_dh * a.abs() + dh.abs() * e_a + p16 * du.abs() + 8 * F32 * du.abs()
            if dt == torch.float16:                                          # fp16 also has a smallest step
                e_dz, e_du, e_h = e_dz + tiny(dt), e_du + tiny(dt), e_h + tiny(dt)
            err["grad_x"] = (e_dz + acc(2 * hidden) * dz.abs()) @ Wg + (e_du + acc(2 * hidden) * du.abs()) @ Wu
            err["grad_w_gate"] = (e_dz + acc(rows) * dz.abs()).mT @ X
            err["grad_w_up"] = (e_du + acc(rows) * du.abs()).mT @ X
            err["grad_w_down"] = G.abs().mT @ (e_h + acc(rows) * h.abs())
            err["grad_b_gate"] = (e_dz + acc(rows) * dz.abs()).sum(0)
            err["grad_b_up"] = (e_du + acc(rows) * du.abs()).sum(0)
            err["grad_b_down"] = acc(rows) * G.abs().sum(0)
            for n in names:
                err["grad_" + n] = err["grad_" + n] + u * val["grad_" + n].abs() + tiny(dt)
    return val, err


def residual_norm(x, f=None, pre_weight=None, pre_bias=None, post_weight=None, post_bias=None, gate=None, scale=None, kind="layer", eps=1e-5,
                  grad_y=None, grad_u=None):
    """-> (values, bounds) with y, u and the gradients of every tensor given.  ``gate`` already broadcasts against x."""
    dt, c = x.dtype, x.shape[-1]
    u = half_step(dt)
    t = dict(x=x, f=f, pre_weight=pre_weight, pre_bias=pre_bias, post_weight=post_weight, post_bias=post_bias, gate=gate,
             scale=scale if isinstance(scale, torch.Tensor) else None)
    leaf = {n: v.detach().double().requires_grad_(True) for n, v in t.items() if v is not None}

    def norm(v, w, b):
        if kind == "layer":
            v = v - v.mean(-1, keepdim=True)
        v = v / torch.sqrt((v * v).mean(-1, keepdim=True) + eps)
        return v * w + (0.0 if b is None else b)

    z = None
    y = leaf["x"]
    if f is not None:
        z = norm(leaf["f"], leaf["post_weight"], leaf.get("post_bias")) if post_weight is not None else leaf["f"]
        k = leaf.get("scale", 1.0 if scale is None or isinstance(scale, torch.Tensor) else float(scale))
        z = z * k * leaf.get("gate", 1.0)
        y = y + z
    outs, grads = [y], [grad_y]
    val = {"y": y.detach()}
    if pre_weight is not None:
        outs.append(norm(y, leaf["pre_weight"], leaf.get("pre_bias")))
        grads.append(grad_u)
        val["u"] = outs[1].detach()
    pairs = [(o, g.detach().double()) for o, g in zip(outs, grads) if g is not None]
    if pairs:
        got = torch.autograd.grad([o for o, _ in pairs], list(leaf.values()), [g for _, g in pairs], allow_unused=True)
        for n, g in zip(leaf, got):
            val["grad_" + n] = torch.zeros_like(leaf[n]) if g is None else g
    # every value is a few fp32 operations on fp32 sums over the row (and, parameters, over the rows): relative to the row's largest
    # magnitude that is (2 sqrt(c) + 40) roundings, amplified where the spread is small against the values (1 / spread)
    err = {}
    for n, v in val.items():
        store = u if n in ("y", "u", "grad_x", "grad_f", "grad_gate") else half_step(torch.float32)
        over = v.abs()
        if n in ("y", "u", "grad_x", "grad_f"):
            size = over.amax(-1, keepdim=True) + (1.0 if n != "y" else 0.0)
        else:
            size = over.max() + 1.0 + (sum(float(g.abs().max()) for _, g in pairs) * x.numel() / c) ** 0.5
        err[n] = store * over + (2 * c ** 0.5 + 40) * 8 * F32 * size + tiny(dt)
    return val, err
