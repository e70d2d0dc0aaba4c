"""Linear attention by the gated delta rule from its definition, in 64 bits on the CPU, token by token: outputs, final state and the gradients,
and the tolerances that the kernels are held to.

Tolerances.  A value rounded to bfloat16 is off by at most u = 2^-8 of itself, one held as two bfloat16 parts by at most p = 2^-18 (the second part's
half step, of a rest that is at most 2^-9).  Roundings are independent of each other and of either sign, so n of them on the way of a term move the norm of a
sum by at most sqrt(n) times one, and a single value by at most n times one of |value| + 4 times the root mean square.
    Where a value is the sum of m terms that carry them, each up to 4 times its own root mean square, i.e. 4 / sqrt(m) times the result's, the errors of a
    value whose terms cancel add up to m times n / sqrt(m): sqrt(m) n times one.  out has 2 such terms (the state's, the scores'), dquery 2 of each
    head of a key head, dkey 4 (state, its cotangent, two scores).  (Without m, a dkey of two heads with resets, held to 4 2^-8 = 1.56e-2 of
    |value| + 4 root mean squares, was off by 1.80e-2.)
  * 16-bit results of 16-bit data.  out: the state, u and the scores as operands, and itself: n = 4.  dvalue: itself, n = 1.  dquery: a score
    (from parts), itself: n = 2.  dkey: u and dv as operands of a score, the score, itself: n = 4 (by the state: the state or its cotangent, dv or u,
    itself: 3).
  * 32-bit results of 16-bit data.  u: the state, r and the inverse in two parts each, and the product of their second parts that is left out:
    n = 4 of p.  A state adds u's in three parts; the gradient of beta takes two such numbers: n = 8.  Float sums are far below: sqrt(64) 2^-24.
    dlog_decay sums o.do - v.dv over the tokens of a chunk of 64, each term off by its own share (o.do: the state or u in two parts against a
    whole operand; u's own: n = 4; dv: n = 4), and <S, dS> behind the chunk, off by as much of each of its terms: their errors add in quadrature.
    What one chunk adds to these errors reaches the next through its token's maps (1 - b k k^T) e^a, whose norm is at most 1 for 0 <= b |k|^2 <= 2 and
    close to 1 where nothing decays: a result behind m chunks has m times as many roundings, independent of each other.  (Without m,
    the cotangent of the first state behind three chunks of reflections, b = 2, with decays above 0.999 was held to 2 2^-18 = 7.6e-6 of
    its norm and off by 8.6e-6.)
    (The kernels hold what 32-bit results depend on in three parts, which is off by less; the bounds count two.)
  * 32-bit data: products of floats, as for chunk_decay: 1e-5 (sqrt(2^14) 2^-24 = 2^-17, and room for the exponentials), and for dlog_decay by the same terms.
"""
import numpy as np
import torch

U16, P16, U32 = 2.0 ** -8, 2.0 ** -18, 1e-5
NAMES = ("hidden_final", "out", "dhidden_init", "dlog_decay", "dbeta", "dvalue", "dkey", "dquery")
ROUNDINGS = {"out": 4, "dvalue": 1, "dquery": 2, "dkey": 4, "hidden_final": 1, "dhidden_init": 1}      # of 16-bit results
PARTS = {"hidden_final": 4, "dhidden_init": 4, "dbeta": 8, "dlog_decay": 4}                             # of 32-bit results of 16-bit data


def reference(h0, a, b, v, k, q, lengths=None, dh=None, do=None, chunk=64):
    """(hidden_final, out) and, with cotangents, (dh0, da, db, dv, dk, dq, what da's error goes by), all float64.  `a`, `b` [B,T,H] or [H]."""
    h, v, k, q = (x.detach().double().cpu() for x in (h0, v, k, q))
    B, T, H, DV = v.shape
    HK, DK = k.shape[2:]
    G = H // HK
    wide = lambda x: x.detach().double().cpu().expand(B, T, H)  # noqa: E731
    a, b = wide(a), wide(b)
    n = [T] * B if lengths is None else [min(max(int(x), 0), T) for x in lengths]
    hT, out = h.clone(), torch.zeros(B, T, H, DV, dtype=torch.float64)
    grads = dh is not None
    if grads:
        dh, do = dh.detach().double().cpu(), do.detach().double().cpu()
        dh0 = torch.zeros_like(h)
        da, db, scale = (torch.zeros(B, T, H, dtype=torch.float64) for _ in range(3))
        dv, dk, dq = torch.zeros_like(v), torch.zeros_like(k), torch.zeros_like(q)
    heads = torch.arange(H) // G
    for i in range(B):
        s, kept, miss = h[i], [], []
        for t in range(n[i]):
            key = k[i, t][heads][:, :, None]
            s = a[i, t].exp()[:, None, None] * s
            kept.append(s)                            # decayed, not yet written to
            miss.append(v[i, t] - (s * key).sum(1))
            s = s + key * (b[i, t][:, None] * miss[t])[:, None, :]
            out[i, t] = (s * q[i, t][heads][:, :, None]).sum(1)
        hT[i] = s
        if not grads:
            continue
        d, after, so_far = dh[i], s, 0.0
        for t in reversed(range(n[i])):
            key, w = k[i, t][heads][:, :, None], b[i, t][:, None]
            if t == n[i] - 1 or (t + 1) % chunk == 0:
                so_far = (after * d).square().sum((-1, -2))
            dq[i, t] = (after * do[i, t][:, None, :]).sum(-1).view(HK, G, DK).sum(1)
            d = d + q[i, t][heads][:, :, None] * do[i, t][:, None, :]
            du = (d * key).sum(1)
            db[i, t] = (du * miss[t]).sum(-1)
            dv[i, t] = w * du
            dk[i, t] = (d * (w * miss[t])[:, None, :] - kept[t] * dv[i, t][:, None, :]).sum(-1).view(HK, G, DK).sum(1)
            d = d - key * dv[i, t][:, None, :]
            da[i, t] = (d * kept[t]).sum((-1, -2))
            so_far = so_far + (out[i, t] * do[i, t]).square().sum(-1) + (v[i, t] * dv[i, t]).square().sum(-1)
            scale[i, t] = so_far.sqrt()
            after = torch.where(a[i, t].exp()[:, None, None] > 0, kept[t] / a[i, t].exp()[:, None, None], 0.0) if t == 0 else None
            if t:
                prev = k[i, t - 1][heads][:, :, None]
                after = kept[t - 1] + prev * (b[i, t - 1][:, None] * miss[t - 1])[:, None, :]
            d = a[i, t].exp()[:, None, None] * d
        dh0[i] = d
    if not grads:
        return hT, out
    return hT, out, dh0, da, db, dv, dk, dq, scale


def check(name, got, exact, dtype, scale=None, chunks=1, group=1):
    """`got` (a tensor of the kernels, from data of `dtype`) against float64 `exact`; `scale`: what the error is a share of, where that is not the result; `chunks`: of a
    sequence; `group`: heads of a key head."""
    assert tuple(got.shape) == tuple(exact.shape), f"{name}: {tuple(got.shape)} != {tuple(exact.shape)}"
    x, y = got.detach().double().cpu(), exact
    assert torch.isfinite(x).all(), f"{name}: not finite"
    if not y.numel():
        return
    if got.dtype == torch.bfloat16:
        n, one = ROUNDINGS[name], U16
    elif dtype == torch.bfloat16:
        n, one = PARTS[name] * max(chunks, 1), P16
    else:
        n, one = 1, U32
    terms = {"out": 2, "dquery": 2 * group, "dkey": 4 * group}.get(name, 1)
    by = y if scale is None else torch.maximum(scale, y.abs())
    norm, off = float(by.norm()), float((x - y).norm())
    assert off <= n ** 0.5 * one * norm + 1e-30, f"{name}: error {off / max(norm, 1e-300):.3e} of the norm, {n ** 0.5 * one:.3e} is allowed"
    rms = norm / np.sqrt(y.numel())
    worst = float(((x - y).abs() / (by.abs() + 4 * rms + 1e-300)).max())
    assert worst <= terms ** 0.5 * n * one, f"{name}: a value is off by {worst:.3e}, {terms ** 0.5 * n * one:.3e} is allowed"


def inputs(B, T, H, HK, DK, DV, dtype=torch.bfloat16, hidden=torch.float32, decay="token", beta="token", keys="random", seed=0, device="cuda"):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    unit = lambda x: x / x.norm(dim=-1, keepdim=True)  # noqa: E731
    h0, v = r(B, H, DK, DV).to(hidden), r(B, T, H, DV).to(dtype)
    k, q = unit(r(B, T, HK, DK)), (unit(r(B, T, HK, DK)) * DK ** -0.5).to(dtype)
    if keys == "same":                    # every token asks for what the one before it wrote
        k = k[:, :1].expand(B, T, HK, DK)
    k = k.to(dtype).contiguous()
    if decay == "head":
        a = torch.log1p(-torch.exp2(-torch.arange(H, dtype=torch.float32) - 3.0))
    else:
        a = torch.nn.functional.logsigmoid({"token": 3.0, "hard": -2.0, "mild": 8.0, "resets": 3.0}[decay] + r(B, T, H))
        if decay == "resets":
            a = a.masked_fill(torch.rand(B, T, H, generator=g) < 0.05, -float("inf"))
        if decay == "hard":
            a = a.masked_fill(torch.rand(B, T, H, generator=g) < 0.1, -200.0)
    b = r(B, T, H).sigmoid()
    if beta == "ends":                    # nothing, all, and twice as much (the state's part along the key changes sign)
        b = torch.randint(0, 3, (B, T, H), generator=g).float()
    if beta == "head":
        b = r(H).sigmoid()
    dh, do = r(B, H, DK, DV).to(hidden), r(B, T, H, DV).to(dtype)
    return [x.to(device) for x in (h0, a, b, v, k, q, dh, do)]


def step(fn, h0, a, b, v, k, q, dh, do, lengths=None):
    arrays = [x.clone().requires_grad_() for x in (h0, a, b)] + [x.detach().requires_grad_() for x in (v, k, q)]
    hT, out = fn(*arrays, lengths)
    return (hT, out) + torch.autograd.grad((hT, out), arrays, (dh, do))


def check_step(got, h0, a, b, v, k, q, dh, do, lengths=None):
    exact = reference(h0, a, b, v, k, q, lengths, dh, do, 64 if v.dtype == torch.bfloat16 else 32)
    B, T, H = v.shape[:3]
    m = -(-T // 64)
    for name, x, y in zip(NAMES, got, exact):
        if name == "dlog_decay":
            scale = exact[8]
            if a.ndim == 1:               # the sum over tokens: their errors add in quadrature
                y, scale = y.sum((0, 1)), scale.square().sum((0, 1)).sqrt()
            check(name, x, y, v.dtype, scale, m)
        elif name == "dbeta" and b.ndim == 1:
            check(name, x, y.sum((0, 1)), v.dtype, y.square().sum((0, 1)).sqrt(), m)
        else:
            check(name, x, y, v.dtype, None, m, H // k.shape[2])
