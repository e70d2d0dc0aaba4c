"""What chunk_delta's results may be off by where nothing but their own rounding is left, and the chunked rule with its operands in parts, on the CPU.

16-bit results.  With y a value in 64 bits, e the error of what is rounded and h <= 2^-7 |y| the distance of neighbouring 16-bit numbers, a result that is
rounded once differs from y rounded in a share |e| / h of all values, there by h: the norm of the difference is at most sqrt(|e| |h|) of the norms.  In e every
operand that is a 32-bit number counts with p = 2^-18 (two bf16 parts: half a step of a rest of at most 2^-9), and so does the product of two second
parts that is left out:
    out      state: 1; scores, u and their second parts' product: 3
    dquery   state: none (three parts); the score: 1
    dkey     state, dv, their second parts: 3; cotangent of the state, u, theirs: 3; the score of dquery: 1; the score of dv and u: 4
    dvalue   none but its own
The terms of a sum may be twice as large as the sum together: |e| <= 2 sqrt(4) p |y| = 2^-16 |y|, and the difference sqrt(2^-16 2^-7) = 2^-11.5, of
which the few values that differ (50 and more of the sizes here) make at most 2^-11.  One operand rounded to 16 bits once has |e| = 2^-9 / sqrt(3) of a
term and more: above 2^-10 as soon as the term is as large as the rest.

32-bit results.  Operands in three parts are off by 2^-25 or less, so float sums remain.  In a chunk three products follow each other, of 12, 6 and 6
instructions an accumulator for 128 features and 64 tokens, each of which adds a few numbers: 64 additions together, sqrt(64) 2^-25 = 2^-22 of the norm;
the exponentials, two units each, as much again.  Chunks are independent of each other: sqrt(m) 2^-21 behind m of them.  The cotangent of the state goes
the same way from the other end.  A gradient of a gate takes one number of each way, whose errors add in quadrature, and its terms may be twice as large
as it: 2 sqrt(2 m) 2^-21.  Two parts instead of three are off by 2^-18 / sqrt(3) for each operand: 2^-18 and more with the three products of a chunk.

32-bit data.  The operands are whole, and all results are float sums: those of 16-bit data's 32-bit results, with chunks of 32 tokens; out and the gradients of
rows take a number of each way, or two of one, and their terms may be twice as large as they are: 2 sqrt(2 m) 2^-21.
"""
import torch

CHANGED = 2.0 ** -11
RESULTS = ("hidden_final", "out", "dhidden_init", "dlog_decay", "dbeta", "dvalue", "dkey", "dquery")


def changed(got, exact):
    """The norm of the difference between a 16-bit result and the exact one rounded, as a share of the norm."""
    y = exact.to(torch.bfloat16).double()
    return float((got.detach().double().cpu() - y).norm() / y.norm())


def off(got, exact, scale=None):
    return float((got.detach().double().cpu() - exact).norm() / (exact if scale is None else scale).norm())


def bound_of_floats(name, chunks):
    return (1.0 if name in ("hidden_final", "dhidden_init") else 8.0 ** 0.5) * chunks ** 0.5 * 2.0 ** -21


def parts_of(x, n):
    """n bf16 parts of x; 0: x as it is."""
    if not n:
        return [x]
    found = []
    for _ in range(n):
        found.append(x.bfloat16().float())
        x = x - found[-1]
    return found


def product(a, b, of_a, of_b):
    a, b = parts_of(a, of_a), parts_of(b, of_b)
    n = max(len(a), len(b))
    return sum(x @ y for i, x in enumerate(a) for j, y in enumerate(b) if i + j < n)


def emulated(h0, a, b, v, k, q, dh, do, many=3, few=2, out_scores=2, dkey_cotangent=2, C=64):
    """One training step on the CPU with float sums: what 32-bit results depend on in `many` parts, what only 16-bit ones do in `few`, but for the scores
    of out and the cotangent of a state in dkey.  One sequence, T a multiple of C, as many key heads as heads."""
    _, T, H, _ = v.shape
    N = T // C
    rows = lambda x: x[0].float().transpose(0, 1).reshape(H, N, C, -1)  # noqa: E731
    v, k, q, do = rows(v), rows(k), rows(q), rows(do)
    a, b = (x[0].T.reshape(H, N, C) for x in (a, b))
    L = a.double().cumsum(-1)
    weight = (L[..., :, None] - L[..., None, :]).tril().exp().float().tril()
    start, end, whole = L.exp().float()[..., None], (L[..., -1:] - L).exp().float()[..., None], L[..., -1].exp().float()[..., None, None]
    t = lambda x: x.transpose(-1, -2)  # noqa: E731
    P, M = weight * (q @ t(k)), (weight * (k @ t(k))).tril(-1)
    eye, wide = torch.eye(C), b[..., None]
    solve, solve_back = (torch.linalg.inv((eye + x).double()).float() for x in (M * t(wide), t(M * wide)))
    S, states, xs, out = h0[0].float(), [], [], []
    for n in range(N):
        states.append(S)
        x = product(solve[:, n], v[:, n] - start[:, n] * product(k[:, n], S, 0, many), many, many)
        u = wide[:, n] * x
        out.append(start[:, n] * product(q[:, n], S, 0, few) + product(P[:, n], u, out_scores, few if out_scores > 1 else 1))
        xs.append(x)
        S = whole[:, n] * S + product(t(k[:, n]), end[:, n] * u, 0, many)
    states.append(S)
    hT, d = S, dh[0].float()
    da, db, dv, dk, dq = (torch.zeros(H, N, C, *s) for s in ((), (), v.shape[3:], k.shape[3:], q.shape[3:]))
    for n in reversed(range(N)):
        x, S, o = xs[n], states[n], do[:, n]
        u = wide[:, n] * x
        behind = (states[n + 1] * d).double().sum((-1, -2))
        du = product(solve_back[:, n], product(t(P[:, n]), o, many, 0) + end[:, n] * product(k[:, n], d, 0, many), many, many)
        dx = wide[:, n] * du
        dv[:, n], db[:, n] = dx, (x * du).sum(-1)
        scores, from_state = product(o, t(u), 0, many), start[:, n] * product(o, t(S), 0, many)
        read = (P[:, n] * scores).sum(-1) + (q[:, n] * from_state).sum(-1) - (dx * v[:, n]).sum(-1)
        da[:, n] = (read.double().flip(-1).cumsum(-1).flip(-1) + behind[:, None]).float()
        both = (weight[:, n] * product(dx, t(u), few, few)).tril(-1)
        both, scores = both + t(both), weight[:, n] * scores
        dq[:, n] = from_state + product(scores, k[:, n], few, 0)
        dk[:, n] = (product(t(scores), q[:, n], few, 0) - product(both, k[:, n], few, 0) - start[:, n] * product(dx, t(S), few, few)
                    + end[:, n] * product(u, t(d), few, dkey_cotangent))
        d = whole[:, n] * d + product(t(q[:, n]), start[:, n] * o, 0, many) - product(t(k[:, n]), start[:, n] * dx, 0, many)
    back = lambda x: x.reshape(H, T, *x.shape[3:]).transpose(0, 1)[None]  # noqa: E731
    to = lambda x: back(x).bfloat16()  # noqa: E731
    return hT[None], to(torch.stack(out, 1)), d[None], back(da), back(db), to(dv), to(dk), to(dq)
