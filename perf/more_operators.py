"""Linear attention by the gated delta rule, and the log probabilities that its models are trained and scored by, as a model that serves and
trains calls them, in cases that can be timed and compared.

A case is a dict of plain values.  `op` names the call:
    prompt   chunk_delta without gradients (prompts)
    train    chunk_delta, forward and the gradients of all six arrays
    decode   delta_step: one token for each row of a batch, on a pool of states that is updated in place
    score    token_logprobs without gradients: given tokens' log probabilities, the entropy, the largest alternatives
    loss     token_logprobs, forward and the gradient of the logits

With `own` false `run` computes the same in elementary torch operations: products, sums, exp, comparisons, indexing.
"""
import math

import torch

own = False

FLOAT = {"bf16": torch.bfloat16, "fp32": torch.float32}

# a drawn case moves and computes no more than the largest listed one of its kind
MOST_BYTES = {"prompt": 272e6, "train": 210e6, "decode": 280e6, "score": 132e6, "loss": 525e6}
MOST_STATES = 4 * 4096 * 6 * 128 * 128      # tokens x state of a training step: what exact() keeps in 64 bits


def _chunk(op, B, T, H, HK, DK, DV, dtype="bf16", state="fp32", documents=False, ragged=False, fused=False):
    return {"op": op, "B": B, "T": T, "H": H, "HK": HK, "DK": DK, "DV": DV, "dtype": dtype, "state": state, "documents": documents,
            "ragged": ragged, "fused": fused}


def _decode(B, H, HK, DK, DV, state="fp32", dtype="bf16", pool=0, beams=0):
    return {"op": "decode", "B": B, "H": H, "HK": HK, "DK": DK, "DV": DV, "state": state, "dtype": dtype, "pool": pool,
            "beams": beams}


def _tokens(op, N, V, dtype="bf16", top=0, padded=False):
    return {"op": op, "N": N, "V": V, "dtype": dtype, "top": top, "padded": padded}


def listed():
    def named(name, case):
        return dict(case, name=name)

    return [
        # serving: a short question of one user: launches and the host path
        named("prompt_short", _chunk("prompt", 1, 37, 8, 8, 64, 64)),
        # serving: a batch of prompts of different lengths, padded to the longest, rows cut from one projection, four heads
        # to a key head
        named("prompts_ragged", _chunk("prompt", 16, 1337, 16, 4, 128, 128, ragged=True, fused=True)),
        # serving: one long document
        named("prompt_long", _chunk("prompt", 1, 32768, 8, 8, 128, 128)),
        # training: the sizes of the benchmark's own step
        named("train", _chunk("train", 4, 4096, 6, 6, 128, 128)),
        # training on packed documents (the decay at a document's start is -inf), eight heads to a key head
        named("train_shared_keys", _chunk("train", 2, 2050, 16, 2, 64, 128, documents=True)),
        # a small float32 step: research code and gradient checks
        named("train_fp32", _chunk("train", 1, 777, 4, 4, 64, 64, dtype="fp32")),
        # serving: one token of one sequence: latency
        named("decode_one", _decode(1, 16, 16, 128, 128)),
        # serving: one token of each of 128 sequences, whose states lie in a pool with room for more; idle rows among them
        named("decode_pool", _decode(128, 16, 4, 128, 128, pool=160)),
        # serving: the token that one user was answered with, and its five nearest alternatives
        named("score_one", _tokens("score", 1, 32000, dtype="fp32", top=5)),
        # serving: the next token of 500 sequences over a large vocabulary, with twenty alternatives each
        named("score_batch", _tokens("score", 500, 131072, top=20)),
        # training: a step's loss over 4096 tokens, some of which do not count
        named("loss", _tokens("loss", 4096, 32000)),
        # training: logits of an odd vocabulary, whose rows begin where the head's padding lets them
        named("loss_odd", _tokens("loss", 777, 50001, dtype="fp32", padded=True)),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """One more case of the ranges that the listed ones stand for: 1 to 32768 tokens, 1 to 32 heads of 32 to 256 features, 1 to 256 rows of a
    decoding batch, 1 to 8192 rows of logits over 1000 to 131072 tokens."""
    while True:
        op = rng.choice(["prompt", "prompt", "train", "train", "decode", "score", "loss"])
        DK, DV = rng.choice([32, 64, 96, 128, 128]), rng.choice([32, 64, 96, 128, 128, 256])
        H = rng.choice([1, 2, 3, 4, 6, 8, 12, 16, 32])
        HK = rng.choice([n for n in (H, H, 1, 2, 4) if n <= H and H % n == 0])
        dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
        if op in ("prompt", "train"):
            T = _log_int(rng, 1, 32768 if op == "prompt" else 8192)
            case = _chunk(op, _log_int(rng, 1, 32), T, H, HK, DK, DV, dtype, rng.choice(["fp32", "fp32", "bf16"]),
                          documents=rng.random() < 0.3, ragged=rng.random() < 0.3, fused=rng.random() < 0.3)
        elif op == "decode":
            beams = rng.choice([0, 0, 0, 2, 4, 5, 8])
            B = _log_int(rng, 1, 256) if not beams else beams * _log_int(rng, 1, 256 // beams)
            case = _decode(B, H, HK, DK, DV, rng.choice(["fp32", "fp32", "bf16"]), dtype,
                           B + rng.randrange(40) if rng.random() < 0.5 else 0, beams)
        else:
            case = _tokens(op, _log_int(rng, 1, 8192), _log_int(rng, 1000, 131072), dtype,
                           rng.choice([0, 1, 5, 8, 20]) if op == "score" else 0, rng.random() < 0.3)
        if work(case)["bytes"] > MOST_BYTES[op]:
            continue
        if op == "train" and case["B"] * case["T"] * H * DK * DV > MOST_STATES:
            continue
        return case


# ---- inputs ---------------------------------------------------------------------------------------
def _lengths(case, seed):
    """Lengths spread over 0..T, an empty row and a full one among them (where there are two); the seed moves them round."""
    B, T = case["B"], case["T"]
    n = [0 if (i == 0 and B > 2) else T if i == B - 1 else 1 + int((T - 1) * ((i * 0.6180339887) % 1.0)) for i in range(B)]
    return n[seed % B:] + n[:seed % B]


def _rows(r, lead, H, HK, DK, DV):
    """Queries, keys and values as a layer makes them: keys of length one, queries of length DK^-1/2."""
    unit = lambda x: x / x.norm(dim=-1, keepdim=True)  # noqa: E731
    return unit(r(*lead, HK, DK)) * DK ** -0.5, unit(r(*lead, HK, DK)), r(*lead, H, DV)


def _prepare_chunk(case, seed, g):
    B, T, H, HK, DK, DV = (case[n] for n in ("B", "T", "H", "HK", "DK", "DV"))
    dt, st = FLOAT[case["dtype"]], FLOAT[case["state"]]
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    q, k, v = _rows(r, (B, T), H, HK, DK, DV)
    if case["fused"]:                 # one projection's rows, cut into the three
        rows = torch.cat([x.reshape(B, T, -1) for x in (q, k, v)], dim=-1).to(dt)
        q, k, v = rows.split([HK * DK, HK * DK, H * DV], dim=-1)
        q, k, v = q.unflatten(-1, (HK, DK)), k.unflatten(-1, (HK, DK)), v.unflatten(-1, (H, DV))
    else:
        q, k, v = q.to(dt), k.to(dt), v.to(dt)
    a = torch.nn.functional.logsigmoid(3.0 + r(B, T, H))
    if case["documents"]:             # every 300th token or so starts a document: nothing before it counts
        starts = torch.rand(B, T, 1, device="cuda", generator=g) < 1 / 300
        a = a.masked_fill(starts, -math.inf)
    s = {"op": case["op"], "h0": r(B, H, DK, DV).to(st), "a": a, "b": r(B, T, H).sigmoid(), "v": v, "k": k, "q": q, "lengths": None}
    if case["ragged"]:
        n = _lengths(case, seed)
        s["lengths"] = torch.tensor(n, device="cuda", dtype=torch.int32)
        # what lies past a row's end is whatever was there: infinities and NaN among it
        past = torch.arange(T, device="cuda")[None, :] >= s["lengths"][:, None]
        v[past] = math.nan
        k[past] = math.inf
    if case["op"] == "train":
        s["dh"], s["do"] = r(B, H, DK, DV).to(st), r(B, T, H, DV).to(dt)
        for n in ("h0", "a", "b", "v", "k", "q"):
            s[n] = s[n].detach().requires_grad_()
    return s


def _prepare_decode(case, seed, g):
    B, H, HK, DK, DV, dt = case["B"], case["H"], case["HK"], case["DK"], case["DV"], FLOAT[case["dtype"]]
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    N = case["pool"] or B
    q, k, v = _rows(r, (B,), H, HK, DK, DV)
    s = {"op": "decode", "states": r(N, H, DK, DV).to(FLOAT[case["state"]]), "a": torch.nn.functional.logsigmoid(3.0 + r(B, H)),
         "b": r(B, H).sigmoid(), "v": v.to(dt), "k": k.to(dt), "q": q.to(dt), "slots": None, "parents": None}
    if case["pool"]:
        s["slots"] = torch.randperm(N, device="cuda", generator=g)[:B]
        if not case["beams"] and B > 8:
            s["slots"][seed % 7::16] = -1                  # rows without a sequence
    if case["beams"]:
        s["parents"] = torch.randint(case["beams"], (B // case["beams"], case["beams"]), device="cuda", generator=g)
    return s


def _prepare_tokens(case, seed, g):
    N, V = case["N"], case["V"]
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    row = V + -V % 64 + 64 if case["padded"] else V         # a head padded for its product: what lies behind is never a token
    logits = (2.5 * r(N, row) + 3.0 * r(N, 1)).to(FLOAT[case["dtype"]])[:, :V]
    logits.masked_fill_(torch.rand(V, device="cuda", generator=g) < 0.01, -math.inf)       # tokens that may not come
    logits[:, 0] = 0.5                                      # one of them all may, and it is the token where a mask took the drawn one
    tokens = torch.randint(V, (N,), device="cuda", generator=g)
    tokens = torch.where(logits.gather(1, tokens[:, None])[:, 0] == -math.inf, torch.zeros_like(tokens), tokens)
    s = {"op": case["op"], "logits": logits, "tokens": tokens, "top": case["top"]}
    if case["op"] == "loss":
        tokens[torch.rand(N, device="cuda", generator=g) < 0.1] = -100      # positions that do not count
        tokens[0] = 0
        s["dp"], s["de"] = r(N) / N, -0.01 * torch.rand(N, device="cuda", generator=g) / N
        s["logits"] = logits.detach().requires_grad_()
    return s


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] in ("prompt", "train"):
        return _prepare_chunk(case, seed, g)
    return _prepare_decode(case, seed, g) if case["op"] == "decode" else _prepare_tokens(case, seed, g)


# ---- one pass -------------------------------------------------------------------------------------
def run(s):
    with torch.set_grad_enabled(s["op"] in ("train", "loss")):
        if s["op"] in ("prompt", "train"):
            if own:
                from gla_jax_amd import chunk_delta
                hT, out = chunk_delta(s["h0"], s["a"], s["b"], s["v"], s["k"], s["q"], s["lengths"])
            else:
                hT, out = _plain_chunk(s["h0"], s["a"], s["b"], s["v"], s["k"], s["q"], s["lengths"])
            if s["op"] == "prompt":
                return hT, out
            arrays = [s[n] for n in ("h0", "a", "b", "v", "k", "q")]
            return (hT.detach(), out.detach()) + torch.autograd.grad((hT, out), arrays, (s["dh"], s["do"]))
        if s["op"] == "decode":
            if own:
                from gla_jax_amd import delta_step
                out = delta_step(s["states"], s["a"], s["b"], s["v"], s["k"], s["q"], slots=s["slots"], parents=s["parents"])
            else:
                out = _plain_step(s["states"], s["a"], s["b"], s["v"], s["k"], s["q"], s["slots"], s["parents"])
            return out, s["states"]
        if own:
            from gla_jax_amd import token_logprobs
            found = token_logprobs(s["logits"], s["tokens"], top=s["top"])
        else:
            found = _plain_logprobs(s["logits"], s["tokens"], s["top"])
        if s["op"] == "score":
            return found
        d, = torch.autograd.grad(found, [s["logits"]], (s["dp"], s["de"]))
        return tuple(x.detach() for x in found) + (d,)


def _sums(a):
    """The sums of a over (j, i] as a lower triangle [..., i, j], each formed from its own terms; -inf above the diagonal."""
    C = a.shape[-1]
    below = torch.ones(C, C, device=a.device, dtype=torch.bool).tril(-1)
    s = torch.where(below, a[..., :, None], torch.zeros_like(a[..., :, None])).cumsum(-2)
    return s.masked_fill(~(below | torch.eye(C, device=a.device, dtype=torch.bool)), -math.inf)


def _inverse(A):
    """(I + A)^-1 of strictly lower A [..., C, C], C a power of two: the inverses of the blocks of s rows on the diagonal give those of 2 s."""
    C = A.shape[-1]
    i = torch.arange(C, device=A.device)
    X, s = torch.eye(C, device=A.device).expand_as(A), 1
    while s < C:
        part = (i[:, None] // (2 * s) == i // (2 * s)) & (i[:, None] // s > i // s)
        X, s = X - X @ torch.where(part, A, torch.zeros_like(A)) @ X, 2 * s
    return X


def _plain_chunk(h0, a, b, v, k, q, lengths, C=64):
    """S_t = (1 - b_t k_t k_t') exp(a_t) S_{t-1} + b_t k_t v_t', o_t = S_t' q_t, in chunks of C tokens: with u what the tokens of a chunk
    write, (1 + A) u = b (v - exp(.) k S) for the state S before it."""
    B, T, H, DV = v.shape
    HK, DK = k.shape[2:]
    dtype = v.dtype
    v, k, q = v.float(), k.float().repeat_interleave(H // HK, dim=2), q.float().repeat_interleave(H // HK, dim=2)
    if lengths is not None:
        past = torch.arange(T, device=v.device)[None, :, None] >= lengths[:, None, None]
        a, b = a.masked_fill(past, 0.0), b.masked_fill(past, 0.0)
        v, k, q = (x.masked_fill(past[..., None], 0.0) for x in (v, k, q))
    N = -(-T // C)
    pad = N * C - T
    F = torch.nn.functional.pad
    a, b = (F(x, (0, 0, 0, pad)).transpose(1, 2).reshape(B, H, N, C) for x in (a, b))
    v, k, q = (F(x, (0, 0, 0, 0, 0, pad)).transpose(1, 2).reshape(B, H, N, C, x.shape[-1]) for x in (v, k, q))
    seg = _sums(a)
    weight, start = seg.exp(), a.cumsum(-1).exp()[..., None]
    inverse = _inverse(b[..., None] * (weight * (k @ k.transpose(-1, -2))).tril(-1))
    from_value, from_state = inverse @ (b[..., None] * v), inverse @ (b[..., None] * start * k)
    scores, from_start, to_end = weight * (q @ k.transpose(-1, -2)), start * q, (k * weight[..., -1, :, None]).transpose(-1, -2)
    whole = a.sum(-1).exp()[..., None, None]
    state, out = h0.float(), []
    for n in range(N):
        u = from_value[:, :, n] - from_state[:, :, n] @ state
        out.append(from_start[:, :, n] @ state + scores[:, :, n] @ u)
        state = whole[:, :, n] * state + to_end[:, :, n] @ u
    out = torch.stack(out, 2).reshape(B, H, N * C, DV).transpose(1, 2)[:, :T]
    return state.to(h0.dtype), out.to(dtype)


def _plain_step(states, a, b, v, k, q, slots, parents):
    B, H = a.shape
    HK, DK = k.shape[1:]
    at = torch.arange(B, device=a.device) if slots is None else slots
    live = at >= 0
    rows = torch.arange(B, device=a.device)
    if parents is not None:
        W = parents.shape[1]
        rows = (parents + torch.arange(B // W, device=a.device)[:, None] * W).reshape(-1)
    old = states[at[rows].clamp(min=0)].float() * a.exp()[..., None, None]
    k, q = k.float().repeat_interleave(H // HK, dim=1), q.float().repeat_interleave(H // HK, dim=1)
    u = b[..., None] * (v.float() - (old * k[..., :, None]).sum(-2))
    new = old + k[..., :, None] * u[..., None, :]
    out = (new * q[..., :, None]).sum(-2)
    to = at[live]
    states[to] = new[live].to(states.dtype)
    return torch.where(live[:, None, None], out, torch.zeros_like(out)).to(v.dtype)


def _plain_logprobs(logits, tokens, top):
    V = logits.shape[-1]
    x = logits.float()
    counts = (tokens >= 0) & (tokens < V)
    most = x.detach().amax(-1, keepdim=True)
    p = x - most - (x - most).exp().sum(-1, keepdim=True).log()
    given = p.gather(1, tokens.clamp(0, V - 1)[:, None])[:, 0]
    given = torch.where(counts, given, torch.zeros_like(given))
    finite = torch.where(x == -math.inf, torch.zeros_like(p), p)
    entropy = -(p.exp() * finite).sum(-1)
    entropy = torch.where(counts, entropy, torch.zeros_like(entropy))
    if not top:
        return given, entropy
    index = x.sort(dim=-1, descending=True, stable=True)[1][:, :top]
    near = p.gather(1, index).masked_fill(~counts[:, None], -math.inf)
    return given, entropy, near, index.masked_fill(~counts[:, None], -1)


# ---- what a pass cannot do without ----------------------------------------------------------------
def work(case):
    size = lambda t: 2 if t == "bf16" else 4  # noqa: E731
    e = size(case["dtype"])
    if case["op"] in ("score", "loss"):
        N, V, top = case["N"], case["V"], case["top"]
        if case["op"] == "score":
            return {"bytes": float(N * V * e + N * (16 + 12 * top)), "flops": 5.0 * N * V}
        return {"bytes": float(2 * N * V * e + N * 24), "flops": 12.0 * N * V}
    H, DK, DV = case["H"], case["DK"], case["DV"]
    if case["op"] in ("prompt", "train"):
        B, HK = case["B"], case["HK"]
        tokens = sum(_lengths(case, 0)) if case["ragged"] else B * case["T"]
        gates = tokens * H * 8
        state = B * H * DK * DV * size(case["state"])
        rows = tokens * (2 * HK * DK + 2 * H * DV) * e + (B * case["T"] - tokens) * H * DV * e + gates + 2 * state
        flops = 6.0 * tokens * H * DK * DV
        if case["op"] == "train":     # the cotangents, and a gradient for every array
            rows += tokens * H * DV * e + tokens * (2 * HK * DK + H * DV) * e + gates + 2 * state
            flops *= 3
        return {"bytes": float(rows), "flops": flops}
    B, HK = case["B"], case["HK"]
    state = B * H * DK * DV
    return {"bytes": float(2 * state * size(case["state"]) + B * (2 * HK * DK + 2 * H * DV) * e + B * H * 8),
            "flops": 8.0 * state}


# ---- the definition, in 64 bits -------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if s["op"] in ("prompt", "train"):
            return _exact_chunk(s)
        return _exact_step(s) if s["op"] == "decode" else _exact_logprobs(s)


def _exact_chunk(s):
    h, v, k, q = (s[n].double() for n in ("h0", "v", "k", "q"))
    B, T, H, DV = v.shape
    HK, DK = k.shape[2:]
    group = H // HK
    n = torch.full((B,), T, device=v.device) if s["lengths"] is None else s["lengths"].long()
    live = torch.arange(T, device=v.device)[None, :] < n[:, None]
    v, k, q = (torch.where(live[..., None, None], x, 0.0) for x in (v, k, q))
    decay, b = torch.where(live[..., None], s["a"].double().exp(), 1.0), torch.where(live[..., None], s["b"].double(), 0.0)
    of_head = torch.arange(H, device=v.device) // group
    out, kept, missed = torch.empty_like(v), [], torch.empty_like(v)
    train = s["op"] == "train"
    for t in range(T):
        if train:
            kept.append(h)
        kt = k[:, t, of_head, :, None]
        h = h * decay[:, t, :, None, None]
        missed[:, t] = v[:, t] - (h * kt).sum(-2)           # what the state does not yet answer its key with
        h = h + kt * (b[:, t, :, None] * missed[:, t])[:, :, None, :]
        out[:, t] = (h * q[:, t, of_head, :, None]).sum(-2)
    if not train:
        return h, out
    d, do = s["dh"].double(), torch.where(live[..., None, None], s["do"].double(), 0.0)
    da, db, dv = torch.empty_like(decay), torch.empty_like(b), torch.empty_like(v)
    dk, dq = (torch.zeros(B, T, HK, DK, device=v.device, dtype=torch.float64) for _ in range(2))
    after = h
    for t in reversed(range(T)):
        kt, bt = k[:, t, of_head, :, None], b[:, t, :, None]
        decayed = kept[t] * decay[:, t, :, None, None]
        dq[:, t] = (after * do[:, t, :, None, :]).sum(-1).view(B, HK, group, DK).sum(2)
        d = d + q[:, t, of_head, :, None] * do[:, t, :, None, :]
        du = (d * kt).sum(-2)
        db[:, t] = (du * missed[:, t]).sum(-1)
        dv[:, t] = bt * du
        each = (d * (bt * missed[:, t])[:, :, None, :] - decayed * dv[:, t, :, None, :]).sum(-1)
        dk[:, t] = each.view(B, HK, group, DK).sum(2)
        d = d - kt * dv[:, t, :, None, :]
        da[:, t] = (d * decayed).sum((-1, -2))
        after, d = kept[t], d * decay[:, t, :, None, None]
    for x in (da, db, dv, dk, dq):
        x[~live] = 0.0
    return h, out, d, da, db, dv, dk, dq


def _exact_step(s):
    B, H = s["a"].shape
    group = H // s["k"].shape[1]
    of_head = torch.arange(H, device=s["a"].device) // group
    states = s["states"].double()
    result = states.clone()
    out = torch.zeros(B, H, s["v"].shape[-1], device=states.device, dtype=torch.float64)
    slots = list(range(B)) if s["slots"] is None else s["slots"].tolist()
    parents = None if s["parents"] is None else s["parents"].tolist()
    for i in range(B):
        if slots[i] < 0:
            continue
        W = 1 if parents is None else len(parents[0])
        source = i if parents is None else i // W * W + parents[i // W][i % W]
        new = states[slots[source]] * s["a"][i].double().exp()[:, None, None]
        key = s["k"][i].double()[of_head][:, :, None]
        new = new + key * (s["b"][i].double()[:, None] * (s["v"][i].double() - (new * key).sum(1)))[:, None, :]
        result[slots[i]] = new
        out[i] = (new * s["q"][i].double()[of_head][:, :, None]).sum(1)
    return out, result


def _exact_logprobs(s):
    tokens, top = s["tokens"], s["top"]
    p = torch.log_softmax(s["logits"].double(), dim=-1)
    counts = (tokens >= 0) & (tokens < p.shape[-1])
    at = torch.where(counts, tokens, 0)[:, None]
    given = torch.where(counts, p.gather(1, at)[:, 0], 0.0)
    entropy = torch.where(counts, torch.special.entr(p.exp()).sum(-1), 0.0)
    if s["op"] == "loss":
        e, shift = torch.where(counts, s["de"].double(), 0.0)[:, None], torch.where(counts, s["dp"].double(), 0.0)[:, None]
        w = p.exp()
        d = -shift * w - e * torch.where(w > 0, w * (p + entropy[:, None]), 0.0)
        return given, entropy, d.scatter_add(1, at, shift)
    if not top:
        return given, entropy
    best = torch.where(counts[:, None], p.topk(top, dim=-1).values, -math.inf)
    return given, entropy, best, None                       # places have no error
