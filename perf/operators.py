"""Linear attention with one decay a head, as a model that serves and trains with it calls it, in cases that can be
timed and compared.

A case is a dict of plain values.  `op` names the call:
    prompt   chunk_decay without gradients (prompts)
    train    chunk_decay, forward and the gradients of all five arrays
    decode   decay_step: one token for each row of a batch, on a pool of states that is updated in place
    beams    beam_select and reorder_states: the next candidates of a beam search, and the states behind them

With `own` false `run` computes the same in elementary torch operations: products, sums, exp, comparisons, indexing.
"""
import math

import torch

own = False

FLOAT = {"bf16": torch.bfloat16, "fp32": torch.float32}

# a drawn case moves and computes no more than the largest listed one
MOST_BYTES = 280e6
MOST_STATES = 4 * 4096 * 6 * 128 * 128      # tokens x state of a training step: what exact() keeps in 64 bits


def _chunk(op, B, T, H, HK, DK, DV, dtype="bf16", decay="token", ragged=False, fused=False):
    return {"op": op, "B": B, "T": T, "H": H, "HK": HK, "DK": DK, "DV": DV, "dtype": dtype, "decay": decay,
            "ragged": ragged, "fused": fused}


def _decode(B, H, HK, DK, DV, state="fp32", dtype="bf16", pool=0, beams=0):
    return {"op": "decode", "B": B, "H": H, "HK": HK, "DK": DK, "DV": DV, "state": state, "dtype": dtype, "pool": pool,
            "beams": beams}


def _beams(G, W, V, H, DK, DV, dtype="bf16", state="fp32"):
    return {"op": "beams", "G": G, "W": W, "V": V, "H": H, "DK": DK, "DV": DV, "dtype": dtype, "state": state}


def listed():
    def named(name, case):
        return dict(case, name=name)

    return [
        # serving: a short question of one user: launches and the host path
        named("prompt_short", _chunk("prompt", 1, 37, 8, 8, 64, 64)),
        # serving: a batch of prompts of different lengths, padded to the longest, rows cut from one projection, four heads
        # to a key head
        named("prompts_ragged", _chunk("prompt", 16, 1337, 16, 4, 128, 128, ragged=True, fused=True)),
        # serving: one long document under one constant decay a head
        named("prompt_long", _chunk("prompt", 1, 32768, 8, 8, 128, 128, decay="head")),
        # training: the sizes of the benchmark's own step
        named("train", _chunk("train", 4, 4096, 6, 6, 128, 128)),
        # training on packed documents (the decay at a document's start is -inf), eight heads to a key head
        named("train_shared_keys", _chunk("train", 2, 2050, 16, 2, 64, 128, decay="documents")),
        # training with values twice as wide as keys
        named("train_wide_values", _chunk("train", 8, 1000, 4, 4, 128, 256)),
        # a small float32 step under one constant decay a head: research code and gradient checks
        named("train_fp32", _chunk("train", 1, 777, 4, 4, 64, 64, dtype="fp32", decay="head")),
        # serving: one token of one sequence: latency
        named("decode_one", _decode(1, 16, 16, 128, 128)),
        # serving: one token of each of 128 sequences, whose states lie in a pool with room for more; idle rows among them
        named("decode_pool", _decode(128, 16, 4, 128, 128, pool=160)),
        # beam search: one token for 16 searches of 8 beams, each from the state of the beam that it continues
        named("decode_beams", _decode(128, 16, 16, 64, 64, state="bf16", beams=8)),
        # beam search: the next candidates of one search of 4 beams, and its states
        named("beams_one", _beams(1, 4, 32000, 16, 128, 128, dtype="fp32")),
        # beam search: 16 searches of 8 beams over a large vocabulary
        named("beams_many", _beams(16, 8, 131072, 16, 64, 64)),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """One more case of the ranges that the listed ones stand for: 1 to 32768 tokens, 1 to 32 heads of 32 to 256 features,
    1 to 256 rows of a decoding batch, 1 to 16 beams over 1000 to 131072 tokens."""
    while True:
        op = rng.choice(["prompt", "prompt", "train", "train", "decode", "decode", "beams"])
        DK, DV = rng.choice([32, 64, 96, 128, 128]), rng.choice([32, 64, 96, 128, 128, 256])
        H = rng.choice([1, 2, 3, 4, 6, 8, 12, 16, 32])
        HK = rng.choice([n for n in (H, H, 1, 2, 4) if n <= H and H % n == 0])
        dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
        if op in ("prompt", "train"):
            T = _log_int(rng, 1, 32768 if op == "prompt" else 8192)
            case = _chunk(op, _log_int(rng, 1, 32), T, H, HK, DK, DV, dtype, rng.choice(["token", "head", "documents"]),
                          ragged=rng.random() < 0.3, fused=rng.random() < 0.3)
        elif op == "decode":
            beams = rng.choice([0, 0, 2, 4, 5, 8, 16])
            B = _log_int(rng, 1, 256) if not beams else beams * _log_int(rng, 1, 256 // beams)
            case = _decode(B, H, HK, DK, DV, rng.choice(["fp32", "fp32", "bf16"]), dtype,
                           B + rng.randrange(40) if rng.random() < 0.5 else 0, beams)
        else:
            case = _beams(_log_int(rng, 1, 32), rng.choice([1, 2, 3, 4, 5, 8, 12, 16]), _log_int(rng, 1000, 131072), H, DK, DV,
                          dtype, rng.choice(["fp32", "fp32", "bf16"]))
        if work(case)["bytes"] > MOST_BYTES:
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


def _log_decay(case, g):
    B, T, H = case["B"], case["T"], case["H"]
    if case["decay"] == "head":       # one constant for each head, from quick to slow, a little different for every seed
        i = torch.arange(H, device="cuda", dtype=torch.float32) * (7.0 / max(H - 1, 1)) + 4.0
        return torch.log1p(-torch.exp2(-i - 0.25 * torch.rand(H, device="cuda", generator=g)))
    a = torch.nn.functional.logsigmoid(3.0 + torch.randn(B, T, H, device="cuda", generator=g))
    if case["decay"] == "documents":  # every 300th token or so starts a document: nothing before it counts
        starts = torch.rand(B, T, 1, device="cuda", generator=g) < 1 / 300
        a = a.masked_fill(starts, -math.inf)
    return a


def _prepare_chunk(case, seed, g):
    B, T, H, HK, DK, DV = (case[n] for n in ("B", "T", "H", "HK", "DK", "DV"))
    dt = FLOAT[case["dtype"]]
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    q, k, v = r(B, T, HK, DK) * DK ** -0.5, r(B, T, HK, DK) * DK ** -0.25, r(B, T, H, DV)
    if case["fused"]:                 # one projection's rows, cut into the three
        rows = torch.cat([x.reshape(B, T, -1) for x in (q, k, v)], dim=-1).to(dt)
        q, k, v = rows.split([HK * DK, HK * DK, H * DV], dim=-1)
        q, k, v = q.unflatten(-1, (HK, DK)), k.unflatten(-1, (HK, DK)), v.unflatten(-1, (H, DV))
    else:
        q, k, v = q.to(dt), k.to(dt), v.to(dt)
    s = {"op": case["op"], "h0": r(B, H, DK, DV), "a": _log_decay(case, g), "v": v, "k": k, "q": q, "lengths": None}
    if case["ragged"]:
        n = _lengths(case, seed)
        s["lengths"] = torch.tensor(n, device="cuda", dtype=torch.int32)
        # what lies past a row's end is whatever was there: infinities and NaN among it
        past = torch.arange(T, device="cuda")[None, :] >= s["lengths"][:, None]
        v[past] = math.nan
        k[past] = math.inf
    if case["op"] == "train":
        s["dh"], s["do"] = r(B, H, DK, DV), r(B, T, H, DV).to(dt)
        for n in ("h0", "a", "v", "k", "q"):
            s[n] = s[n].detach().requires_grad_()
    return s


def _prepare_decode(case, seed, g):
    B, H, HK, DK, DV, dt = case["B"], case["H"], case["HK"], case["DK"], case["DV"], FLOAT[case["dtype"]]
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    N = case["pool"] or B
    s = {"op": "decode", "states": r(N, H, DK, DV).to(FLOAT[case["state"]]),
         "a": torch.nn.functional.logsigmoid(3.0 + r(B, H)), "v": r(B, H, DV).to(dt),
         "k": (r(B, HK, DK) * DK ** -0.25).to(dt), "q": (r(B, HK, DK) * DK ** -0.5).to(dt), "slots": None, "parents": None}
    if case["pool"]:
        s["slots"] = torch.randperm(N, device="cuda", generator=g)[:B]
        if not case["beams"] and B > 8:
            s["slots"][seed % 7::16] = -1                  # rows without a sequence
    if case["beams"]:
        s["parents"] = torch.randint(case["beams"], (B // case["beams"], case["beams"]), device="cuda", generator=g)
    return s


def _prepare_beams(case, seed, g):
    G, W, V = case["G"], case["W"], case["V"]
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    logits = 2.5 * r(G, W, V)
    logits.masked_fill_(torch.rand(V, device="cuda", generator=g) < 0.01, -math.inf)       # tokens that may not come
    logits += 1.5 * r(G, 1, 1) + 2.0 * r(G, W, 1)
    finished = torch.rand(G, W, device="cuda", generator=g) < (0.1 if W > 1 else 0.0)
    eos = 2
    logits[:, :, eos] = 0.5
    return {"op": "beams", "logits": logits.to(FLOAT[case["dtype"]]), "scores": -20.0 * torch.rand(G, W, device="cuda", generator=g),
            "finished": finished, "eos": eos, "states": r(G * W, case["H"], case["DK"], case["DV"]).to(FLOAT[case["state"]])}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] in ("prompt", "train"):
        return _prepare_chunk(case, seed, g)
    return _prepare_decode(case, seed, g) if case["op"] == "decode" else _prepare_beams(case, seed, g)


# ---- one pass -------------------------------------------------------------------------------------
def run(s):
    with torch.set_grad_enabled(s["op"] == "train"):
        if s["op"] in ("prompt", "train"):
            if own:
                from gla_jax_amd import chunk_decay
                hT, out = chunk_decay(s["h0"], s["a"], s["v"], s["k"], s["q"], s["lengths"])
            else:
                hT, out = _plain_chunk(s["h0"], s["a"], s["v"], s["k"], s["q"], s["lengths"])
            if s["op"] == "prompt":
                return hT, out
            arrays = [s[n] for n in ("h0", "a", "v", "k", "q")]
            return (hT.detach(), out.detach()) + torch.autograd.grad((hT, out), arrays, (s["dh"], s["do"]))
        if s["op"] == "decode":
            if own:
                from gla_jax_amd import decay_step
                out = decay_step(s["states"], s["a"], s["v"], s["k"], s["q"], slots=s["slots"], parents=s["parents"])
            else:
                out = _plain_step(s["states"], s["a"], s["v"], s["k"], s["q"], s["slots"], s["parents"])
            return out, s["states"]
        if own:
            from gla_jax_amd import beam_select, reorder_states
            scores, parents, tokens = beam_select(s["logits"], s["scores"], finished=s["finished"], eos=s["eos"])
            reorder_states(s["states"], parents)
        else:
            scores, parents, tokens = _plain_select(s["logits"], s["scores"], s["finished"], s["eos"])
            _plain_reorder(s["states"], parents)
        return scores, parents, tokens, s["states"]


def _sums(a):
    """The sums of a over (j, i] as a lower triangle [..., i, j], each formed from its own terms; -inf above the diagonal."""
    C = a.shape[-1]
    below = torch.ones(C, C, device=a.device, dtype=torch.bool).tril(-1)
    s = torch.where(below, a[..., :, None], torch.zeros_like(a[..., :, None])).cumsum(-2)
    return s.masked_fill(~(below | torch.eye(C, device=a.device, dtype=torch.bool)), -math.inf)


def _plain_chunk(h0, a, v, k, q, lengths, C=64):
    """S_t = exp(a_t) S_{t-1} + k_t v_t', o_t = S_t' q_t, in chunks of C tokens and, over the chunks, as one product with their
    decays."""
    B, T, H, DV = v.shape
    HK, DK = k.shape[2:]
    dtype = v.dtype
    a = (a.expand(B, T, H) if a.ndim == 1 else a).float()
    v, k, q = v.float(), k.float().repeat_interleave(H // HK, dim=2), q.float().repeat_interleave(H // HK, dim=2)
    if lengths is not None:
        past = torch.arange(T, device=v.device)[None, :, None] >= lengths[:, None, None]
        a = a.masked_fill(past, 0.0)
        v, k, q = (x.masked_fill(past[..., None], 0.0) for x in (v, k, q))
    N = -(-T // C)
    pad = N * C - T
    F = torch.nn.functional.pad
    a = F(a, (0, 0, 0, pad)).transpose(1, 2).reshape(B, H, N, C)
    v, k, q = (F(x, (0, 0, 0, 0, 0, pad)).transpose(1, 2).reshape(B, H, N, C, x.shape[-1]) for x in (v, k, q))
    seg = _sums(a)
    out = ((q @ k.transpose(-1, -2)) * seg.exp()) @ v
    own_part = (k * seg[..., -1, :].exp()[..., None]).transpose(-1, -2) @ v
    parts = torch.cat([h0.float()[:, :, None], own_part], dim=2).flatten(-2)
    over = _sums(F(a.sum(-1), (1, 0))).exp()
    states = (over @ parts).unflatten(-1, (DK, DV))
    out = out + a.cumsum(-1).exp()[..., None] * (q @ states[:, :, :-1])
    out = out.reshape(B, H, N * C, DV).transpose(1, 2)[:, :T]
    return states[:, :, -1].to(h0.dtype), out.to(dtype)


def _plain_step(states, a, v, k, q, slots, parents):
    B, H = a.shape
    HK, DK = k.shape[1:]
    at = torch.arange(B, device=a.device) if slots is None else slots
    live = at >= 0
    rows = torch.arange(B, device=a.device)
    if parents is not None:
        W = parents.shape[1]
        rows = (parents + torch.arange(B // W, device=a.device)[:, None] * W).reshape(-1)
    old = states[at[rows].clamp(min=0)].float()
    k, q = k.float().repeat_interleave(H // HK, dim=1), q.float().repeat_interleave(H // HK, dim=1)
    new = old * a.exp()[..., None, None] + k[..., :, None] * v.float()[..., None, :]
    out = (new * q[..., :, None]).sum(-2)
    to = at[live]
    states[to] = new[live].to(states.dtype)
    return torch.where(live[:, None, None], out, torch.zeros_like(out)).to(v.dtype)


def _plain_select(logits, scores, finished, eos):
    G, W, V = logits.shape
    x = logits.float()
    x = torch.where(torch.isnan(x), torch.full_like(x, -math.inf), x)
    top = x.amax(-1, keepdim=True)
    lse = top + (x - top).exp().sum(-1, keepdim=True).log()
    ended = torch.full((V,), -math.inf, device=x.device)
    ended[eos] = 0.0
    x = torch.where(finished[..., None], ended, x)
    lse = torch.where(finished[..., None], torch.zeros_like(lse), lse)
    value, token = x.sort(dim=-1, descending=True, stable=True)            # a beam's candidates: its W largest logits
    value, token = value[..., :W], token[..., :W]
    cand = scores[..., None] + (value - lse)
    cand = torch.where(torch.isnan(cand), torch.full_like(cand, -math.inf), cand).reshape(G, -1)
    # equal ones in the order of (beam, token)
    flat = (torch.arange(W, device=x.device)[:, None] * V + token).reshape(G, -1)
    order = flat.argsort(dim=-1)
    cand, flat = cand.gather(1, order), flat.gather(1, order)
    best, at = cand.sort(dim=-1, descending=True, stable=True)
    flat = flat.gather(1, at[:, :W])
    return best[:, :W], flat // V, flat % V


def _plain_reorder(states, parents):
    W = parents.shape[1]
    rows = (parents + torch.arange(parents.shape[0], device=parents.device)[:, None] * W).reshape(-1)
    states.copy_(states[rows])


# ---- what a pass cannot do without ----------------------------------------------------------------
def work(case):
    size = lambda t: 2 if t == "bf16" else 4  # noqa: E731
    H, DK, DV, e = case["H"], case["DK"], case["DV"], size(case["dtype"])
    if case["op"] in ("prompt", "train"):
        B, HK = case["B"], case["HK"]
        tokens = sum(_lengths(case, 0)) if case["ragged"] else B * case["T"]
        gates = H * 4 if case["decay"] == "head" else tokens * H * 4
        state = B * H * DK * DV * 4
        rows = tokens * (2 * HK * DK + 2 * H * DV) * e + (B * case["T"] - tokens) * H * DV * e + gates + 2 * state
        flops = 4.0 * tokens * H * DK * DV
        if case["op"] == "train":     # the cotangents, and a gradient for every array
            rows += tokens * H * DV * e + tokens * (2 * HK * DK + H * DV) * e + gates + 2 * state
            flops *= 3
        return {"bytes": float(rows), "flops": flops}
    if case["op"] == "decode":
        B, HK = case["B"], case["HK"]
        state = B * H * DK * DV
        return {"bytes": float(2 * state * size(case["state"]) + B * (2 * HK * DK + 2 * H * DV) * e + B * H * 4),
                "flops": 5.0 * state}
    G, W, V = case["G"], case["W"], case["V"]
    state = G * W * H * DK * DV * size(case["state"])
    return {"bytes": float(G * W * V * e + 2 * state + G * W * 28), "flops": 2.0 * G * W * V}


# ---- the definition, in 64 bits -------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if s["op"] in ("prompt", "train"):
            return _exact_chunk(s)
        if s["op"] == "decode":
            return _exact_step(s)
        return _exact_select(s)


def _exact_chunk(s):
    h, v, k, q = (s[n].double() for n in ("h0", "v", "k", "q"))
    B, T, H, DV = v.shape
    HK, DK = k.shape[2:]
    group = H // HK
    a = s["a"].double()
    a = a.expand(B, T, H) if a.ndim == 1 else a
    n = torch.full((B,), T, device=v.device) if s["lengths"] is None else s["lengths"].long()
    live = torch.arange(T, device=v.device)[None, :] < n[:, None]
    v, k, q = (torch.where(live[..., None, None], x, 0.0) for x in (v, k, q))
    decay = torch.where(live[..., None], a.exp(), 1.0)
    of_head = torch.arange(H, device=v.device) // group
    out, kept = torch.empty_like(v), []
    train = s["op"] == "train"
    for t in range(T):
        if train:
            kept.append(h)
        h = h * decay[:, t, :, None, None] + k[:, t, of_head, :, None] * v[:, t, :, None, :]
        out[:, t] = (h * q[:, t, of_head, :, None]).sum(-2)
    if not train:
        return h, out
    d, do = s["dh"].double(), torch.where(live[..., None, None], s["do"].double(), 0.0)
    da, dv = torch.empty_like(decay), torch.empty_like(v)
    dk, dq = (torch.zeros(B, T, HK, DK, device=v.device, dtype=torch.float64) for _ in range(2))
    after = h
    for t in reversed(range(T)):
        dq[:, t] = (after * do[:, t, :, None, :]).sum(-1).view(B, HK, group, DK).sum(2)
        d = d + q[:, t, of_head, :, None] * do[:, t, :, None, :]
        dk[:, t] = (d * v[:, t, :, None, :]).sum(-1).view(B, HK, group, DK).sum(2)
        dv[:, t] = (d * k[:, t, of_head, :, None]).sum(-2)
        d_decayed = d * decay[:, t, :, None, None]
        da[:, t] = (d_decayed * kept[t]).sum((-1, -2))
        after, d = kept[t], d_decayed
    for x in (dk, dq, dv):
        x[~live] = 0.0
    da[~live] = 0.0
    if s["a"].ndim == 1:
        da = da.sum((0, 1))
    return h, out, d, da, dv, dk, dq


def _exact_step(s):
    B, H = s["a"].shape
    group = H // s["k"].shape[1]
    of_head = torch.arange(H, device=s["a"].device) // group
    states = s["states"].double()
    result = states.clone()
    out = torch.zeros(B, H, s["v"].shape[-1], device=states.device, dtype=torch.float64)
    slots = list(range(B)) if s["slots"] is None else s["slots"].tolist()
    parents = None if s["parents"] is None else s["parents"].tolist()
    for b in range(B):
        if slots[b] < 0:
            continue
        W = 1 if parents is None else len(parents[0])
        source = b if parents is None else b // W * W + parents[b // W][b % W]
        new = (states[slots[source]] * s["a"][b].double().exp()[:, None, None]
               + s["k"][b].double()[of_head][:, :, None] * s["v"][b].double()[:, None, :])
        result[slots[b]] = new
        out[b] = (new * s["q"][b].double()[of_head][:, :, None]).sum(1)
    return out, result


def _exact_select(s):
    G, W, V = s["logits"].shape
    p = torch.log_softmax(s["logits"].double(), dim=-1)
    ended = torch.full((V,), -math.inf, device=p.device, dtype=torch.float64)
    ended[s["eos"]] = 0.0
    p = torch.where(s["finished"][..., None], ended, p) + s["scores"].double()[..., None]
    return p.reshape(G, W * V).topk(W, dim=-1).values, None, None, None     # places and copies have no error
