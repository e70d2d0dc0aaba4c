"""Linear attention with one decay a head from its definition, in 64 bits on the CPU, token by token: outputs, final state and
the gradients, and the tolerances that the kernels are held to.

Tolerances.  With u = 2^-9 the rounding of a bfloat16 value and u32 = 2^-24 that of a float:
  * 16-bit results take at most three roundings to 16 bits: the scores, the state where it is an operand, and the result itself.  Each
    moves a value by at most u of itself; over a sum of terms of either sign the norm of the error stays within u of the sum's norm
    for each.  So the norm of the error is at most 3 u of the result's, and a single value is off by at most 3 u of the largest
    |value| plus as much of the norm's root mean square times 4 (a term can exceed the root mean square by that much).
  * 32-bit results (float data, states, the gradient of log_decay) accumulate float products: n of them in any order are off by at most
    sqrt(n) u32 of the norm in the mean; with n up to 2^14 products behind a value that is 2^-17, and 1e-5 leaves room for the exponentials
    (a unit in the last place each).
"""
import numpy as np
import torch

U16, U32 = 2.0 ** -9, 1e-5


def reference(h0, a, v, k, q, lengths=None, dh=None, do=None):
    """(hidden_final, out) and, with cotangents, (dh0, da, dv, dk, dq), all float64.  Arrays [B,..] as chunk_decay's; `a` [B,T,H] or [H]."""
    h, v, k, q = (x.detach().double().cpu() for x in (h0, v, k, q))
    B, T, H, DV = v.shape
    HK, DK = k.shape[2:]
    G = H // HK
    constant = a.ndim == 1
    a = a.detach().double().cpu().expand(B, T, H)
    n = [T] * B if lengths is None else [min(max(int(x), 0), T) for x in lengths]
    hT, out = h.clone(), torch.zeros(B, T, H, DV, dtype=torch.float64)
    grads = dh is not None
    if grads:
        dh, do = dh.detach().double().cpu(), do.detach().double().cpu()
        dh0, da = torch.zeros_like(h), torch.zeros(B, T, H, dtype=torch.float64)
        dv, dk, dq = torch.zeros_like(v), torch.zeros_like(k), torch.zeros_like(q)
    heads = torch.arange(H) // G
    for b in range(B):
        s, kept = h[b], []
        for t in range(n[b]):
            kept.append(s)
            s = a[b, t].exp()[:, None, None] * s + k[b, t][heads][:, :, None] * v[b, t][:, None, :]
            out[b, t] = (s * q[b, t][heads][:, :, None]).sum(1)
        hT[b] = s
        if not grads:
            continue
        d, after = dh[b], s
        for t in reversed(range(n[b])):
            dq[b, t] = (after * do[b, t][:, None, :]).sum(-1).view(HK, G, DK).sum(1)
            d = d + q[b, t][heads][:, :, None] * do[b, t][:, None, :]
            dk[b, t] = (d * v[b, t][:, None, :]).sum(-1).view(HK, G, DK).sum(1)
            dv[b, t] = (d * k[b, t][heads][:, :, None]).sum(1)
            d = a[b, t].exp()[:, None, None] * d
            da[b, t] = (d * kept[t]).sum((-1, -2))
            after = kept[t]
        dh0[b] = d
    if not grads:
        return hT, out
    return hT, out, dh0, (da.sum((0, 1)) if constant else da), dv, dk, dq


def check(name, got, exact, scale=None):
    """`got` (a tensor of the kernels) against float64 `exact`; `scale`: what the error is a share of, where that is not the result."""
    assert tuple(got.shape) == tuple(exact.shape), f"{name}: {tuple(got.shape)} != {tuple(exact.shape)}"
    x, y = got.detach().double().cpu(), exact
    assert torch.isfinite(x).all(), f"{name}: not finite"
    if not y.numel():
        return
    tol = 3 * U16 if got.dtype == torch.bfloat16 else U32
    norm = float(y.norm()) if scale is None else float(scale)
    off = float((x - y).norm())
    assert off <= tol * norm + 1e-30, f"{name}: error {off / max(norm, 1e-300):.3e} of the norm, {tol:.3e} is allowed"
    rms = norm / np.sqrt(y.numel())
    worst = float(((x - y).abs() / (y.abs() + 4 * rms + 1e-300)).max())
    assert worst <= 4 * tol, f"{name}: a value is off by {worst:.3e}, {4 * tol:.3e} is allowed"


def inputs(B, T, H, HK, DK, DV, dtype=torch.bfloat16, hidden=torch.float32, decay="token", seed=0, device="cuda"):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    h0, v = r(B, H, DK, DV).to(hidden), r(B, T, H, DV).to(dtype)
    k, q = (r(B, T, HK, DK) * DK ** -0.25).to(dtype), (r(B, T, HK, DK) * DK ** -0.5).to(dtype)
    if decay == "head":
        a = torch.log1p(-torch.exp2(-torch.arange(H, dtype=torch.float32) - 3.0))
    else:
        a = torch.nn.functional.logsigmoid({"token": 3.0, "hard": -2.0, "mild": 8.0, "resets": 3.0}[decay] + r(B, T, H))
        if decay == "resets":
            a = a.masked_fill(torch.rand(B, T, H, generator=g) < 0.05, -float("inf"))
        if decay == "hard":
            a = a.masked_fill(torch.rand(B, T, H, generator=g) < 0.1, -200.0)
    dh, do = r(B, H, DK, DV).to(hidden), r(B, T, H, DV).to(dtype)
    return [x.to(device) for x in (h0, a, v, k, q, dh, do)]


NAMES = ("hidden_final", "out", "dhidden_init", "dlog_decay", "dvalue", "dkey", "dquery")


def step(fn, h0, a, v, k, q, dh, do, lengths=None):
    arrays = [x.clone().requires_grad_() for x in (h0, a)] + [x.detach().requires_grad_() for x in (v, k, q)]
    hT, out = fn(*arrays, lengths)
    return (hT, out) + torch.autograd.grad((hT, out), arrays, (dh, do))


def check_step(got, h0, a, v, k, q, dh, do, lengths=None):
    exact = reference(h0, a, v, k, q, lengths, dh, do)
    for name, x, y in zip(NAMES, got, exact):
        scale = None
        if name == "dlog_decay" and a.ndim == 1:      # a sum over all tokens: its error goes by theirs
            B, T, H = v.shape[:3]
            each = reference(h0, a.expand(B, T, H), v, k, q, lengths, dh, do)[3]
            scale = each.abs().sum((0, 1)).norm()
        check(name, x, y, scale)
