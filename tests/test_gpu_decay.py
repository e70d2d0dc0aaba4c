"""chunk_decay and decay_step against the recurrence in 64 bits, where they can go wrong."""
import pytest
import torch

from tests.decay_reference import check, check_step, inputs, reference, step

pytestmark = pytest.mark.gpu


def _chunk():
    from gla_jax_amd import chunk_decay
    return chunk_decay


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 96, 127, 129, 200])
def test_lengths_around_tiles_and_chunks(T, dtype):
    x = inputs(2, T, 3, 3, 32, 48, dtype, seed=T)
    check_step(step(_chunk(), *x), *x)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("DK, DV", [(16, 16), (16, 256), (64, 64), (64, 128), (80, 96), (128, 64), (128, 128), (96, 256), (144, 64), (256, 128),
                                    (256, 256), (240, 208)])
def test_head_dimensions(DK, DV, dtype):
    """Every width of a workgroup, filled and not, and keys and values that take two."""
    x = inputs(1, 83, 2, 2, DK, DV, dtype, seed=DK + DV)
    check_step(step(_chunk(), *x), *x)


@pytest.mark.parametrize("DK, DV", [(1, 1), (20, 12), (7, 33)])
def test_head_dimensions_that_are_padded(DK, DV):
    x = inputs(2, 70, 2, 1, DK, DV, seed=3)
    check_step(step(_chunk(), *x), *x)


@pytest.mark.parametrize("decay", ["token", "head", "hard", "mild", "resets"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_decays(decay, dtype):
    x = inputs(2, 150, 4, 2, 64, 64, dtype, decay=decay, seed=11)
    check_step(step(_chunk(), *x), *x)


def test_growth():
    """A positive log_decay: nothing here relies on decays below one."""
    h0, a, v, k, q, dh, do = inputs(1, 100, 2, 2, 32, 32, torch.float32, seed=5)
    x = (h0, -0.2 * a, v, k, q, dh, do)
    check_step(step(_chunk(), *x), *x)


@pytest.mark.parametrize("H, HK, DV", [(4, 1, 64), (6, 3, 64), (16, 2, 128), (8, 2, 256), (12, 4, 32)])
def test_heads_that_share_keys(H, HK, DV):
    x = inputs(2, 90, H, HK, 32, DV, seed=H)
    check_step(step(_chunk(), *x), *x)


@pytest.mark.parametrize("hidden", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_types_of_the_state(hidden, dtype):
    x = inputs(2, 66, 2, 2, 48, 64, dtype, hidden, seed=7)
    got = step(_chunk(), *x)
    assert got[0].dtype == got[2].dtype == hidden and got[1].dtype == dtype and got[3].dtype == torch.float32
    check_step(got, *x)


@pytest.mark.parametrize("B, T, H, DK, DV, dtype", [(1, 1500, 1, 128, 128, torch.bfloat16), (2, 777, 2, 64, 256, torch.bfloat16),
                                                    (1, 1000, 2, 256, 64, torch.bfloat16), (1, 500, 3, 32, 64, torch.float32)])
def test_few_long_sequences(B, T, H, DK, DV, dtype):
    """These run as segments side by side, the forward as others than the backward; shared heads and constant decays too."""
    x = inputs(B, T, H, 1, DK, DV, dtype, decay="head" if H == 3 else "token", seed=T)
    check_step(step(_chunk(), *x), *x)


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
@pytest.mark.parametrize("T, lengths", [(70, [0, 70, 1, 64, 65, 37]), (300, [300, 0, 5, 128, 129, 299]), (40, [0, 0, 0, 0, 0, 0])])
def test_ragged(T, lengths, index):
    """What lies behind a sequence's end is not read: NaN and infinities there leave everything alone, and gradients there are zero."""
    h0, a, v, k, q, dh, do = inputs(6, T, 2, 2, 32, 64, seed=T)
    n = torch.tensor(lengths, device="cuda", dtype=index)
    past = torch.arange(T, device="cuda")[None, :] >= n[:, None]
    clean = step(_chunk(), h0, a, v, k, q, dh, do, n)
    v, k, q, a = v.clone(), k.clone(), q.clone(), a.clone()
    v[past], k[past], q[past], a[past] = float("nan"), float("inf"), -float("inf"), float("nan")
    got = step(_chunk(), h0, a, v, k, q, dh, do, n)
    for x, y in zip(got, clean):
        assert torch.equal(x, y)
    assert not got[1][past].any() and not any(x[past].any() for x in got[3:])
    check_step(got, h0, torch.where(past[..., None], 0.0, a), *(torch.where(past[..., None, None], 0.0, x) for x in (v, k, q)), dh, do, n)
    for b, length in enumerate(lengths):
        if length == 0:
            assert torch.equal(got[0][b], h0[b]) and torch.equal(got[2][b], dh[b])


def test_lengths_outside_are_clipped():
    h0, a, v, k, q, dh, do = inputs(3, 50, 2, 2, 32, 32, seed=1)
    n = torch.tensor([-5, 1000, 50], device="cuda", dtype=torch.int32)
    hT, out = _chunk()(h0, a, v, k, q, n)
    assert torch.equal(hT[0], h0[0]) and not out[0].any()
    full = _chunk()(h0, a, v, k, q)
    check("out", out[1:], full[1][1:].double().cpu())


def test_nothing_to_do():
    h0, a, v, k, q, dh, do = inputs(2, 0, 3, 3, 32, 16, seed=2)
    got = step(_chunk(), h0, a, v, k, q, dh, do)
    assert torch.equal(got[0], h0) and got[1].shape == (2, 0, 3, 16) and torch.equal(got[2], dh) and got[3].shape == (2, 0, 3)
    head = torch.zeros(3, device="cuda")
    assert torch.equal(step(_chunk(), h0, head, v, k, q, dh, do)[3], head)
    empty = inputs(1, 5, 2, 2, 16, 16, seed=2)
    hT, out = _chunk()(*(x[:0] for x in empty[:5]))
    assert hT.shape == (0, 2, 16, 16) and out.shape == (0, 5, 2, 16)


def test_batch_axes():
    h0, a, v, k, q, dh, do = inputs(6, 33, 2, 1, 16, 32, seed=4)
    one = _chunk()(h0[0], a[0], v[0], k[0], q[0])
    many = _chunk()(*(x.reshape(2, 3, *x.shape[1:]) for x in (h0, a, v, k, q)))
    flat = _chunk()(h0, a, v, k, q)
    for x, y, z in zip(one, many, flat):
        assert torch.equal(y.reshape(z.shape), z) and torch.equal(x, z[0])
    n = torch.tensor([5, 33, 0, 7, 1, 20], device="cuda")
    ragged = _chunk()(*(x.reshape(2, 3, *x.shape[1:]) for x in (h0, a, v, k, q)), n.reshape(2, 3))
    for x, y in zip(ragged, _chunk()(h0, a, v, k, q, n)):
        assert torch.equal(x.reshape(y.shape), y)


def test_strides():
    """One projection's rows cut into the three, heads before tokens, one key head for all by a stride of zero, rows that begin on an
    odd address: all the same values."""
    B, T, H, D = 2, 70, 4, 32
    h0, a, v, k, q, dh, do = inputs(B, T, H, H, D, D, seed=6)
    want = step(_chunk(), h0, a, v, k, q, dh, do)
    fused = torch.cat([x.reshape(B, T, -1) for x in (q, k, v)], -1)
    cut = [x.unflatten(-1, (H, D)) for x in fused.split([H * D] * 3, -1)]
    heads_first = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (v, k, q)]
    odd = [torch.cat([x.new_zeros(1), x.flatten()])[1:].view(x.shape) for x in (v, k, q)]
    gates = a.transpose(1, 2).contiguous().transpose(1, 2)
    for vkq in ([cut[2], cut[1], cut[0]], heads_first, odd):
        assert any(not x.is_contiguous() or x.data_ptr() % 16 for x in vkq)
        for x, y in zip(step(_chunk(), h0, gates, *vkq, dh, do), want):
            assert torch.equal(x, y)
    shared = k[:, :, :1].expand(B, T, H, D)
    x = (h0, a, v, shared, q, dh, do)
    got = step(_chunk(), *x)
    check_step(got, *x)


def test_the_same_twice():
    """Sums run in one order: equal inputs give equal bits, also where parts are summed over workgroups."""
    x = inputs(2, 400, 8, 2, 64, 256, decay="head", seed=8)
    first = step(_chunk(), *x)
    for y, z in zip(first, step(_chunk(), *x)):
        assert torch.equal(y, z)


def test_another_stream():
    x = inputs(4, 500, 8, 8, 64, 64, seed=9)
    want = step(_chunk(), *x)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = step(_chunk(), *x)
    side.synchronize()
    for y, z in zip(got, want):
        assert torch.equal(y, z)


def test_gradients_against_differences():
    """Central differences of the definition in 64 bits, along a random direction of every array: the truncation is the
    step's square (1e-8), so what is allowed is that of the kernel's 32-bit gradients."""
    h0, a, v, k, q, dh, do = inputs(1, 40, 2, 1, 16, 16, torch.float32, seed=10)
    got = step(_chunk(), h0, a, v, k, q, dh, do)
    arrays = [x.double().cpu() for x in (h0, a, v, k, q)]
    value = lambda xs: sum((y * d.double().cpu()).sum() for y, d in zip(reference(*xs), (dh, do)))  # noqa: E731
    g = torch.Generator().manual_seed(1)
    for i in range(5):
        way = torch.randn(arrays[i].shape, generator=g, dtype=torch.float64)
        way /= way.norm()
        plus, minus = list(arrays), list(arrays)
        plus[i], minus[i] = arrays[i] + 1e-4 * way, arrays[i] - 1e-4 * way
        slope = float(value(plus) - value(minus)) / 2e-4
        mine = float((got[2 + i].double().cpu() * way).sum())
        assert abs(mine - slope) <= 1e-5 * float(got[2 + i].double().norm()) + 1e-6


def test_agrees_with_gates_for_every_feature():
    """chunk_gla with all features of a head under the same gate is the same recurrence."""
    from gla_jax_amd import recurrent_gla_naive
    h0, a, v, k, q, dh, do = inputs(2, 128, 2, 2, 64, 64, torch.float32, seed=12)
    hT, out = _chunk()(h0, a, v, k, q)
    hT2, out2 = recurrent_gla_naive(h0, a[..., None].expand(2, 128, 2, 64), v, k, q, False)
    check("hidden_final", hT, hT2.double().cpu())
    check("out", out, out2.double().cpu())


def test_transforms():
    """torch.func over the calls: a mapped call is the call of the batch; a second derivative is refused."""
    h0, a, v, k, q, dh, do = inputs(4, 40, 2, 2, 16, 32, torch.float32, seed=13)
    want = step(_chunk(), h0, a, v, k, q, dh, do)
    one = lambda *x: _chunk()(*x)  # noqa: E731
    got = torch.func.vmap(one)(h0, a, v, k, q)
    for x, y in zip(got, want):
        assert torch.equal(x, y)
    loss = lambda h, a, v, k, q, dh, do: sum((x * y).sum() for x, y in zip(_chunk()(h, a, v, k, q), (dh, do)))  # noqa: E731
    grads = torch.func.vmap(torch.func.grad(loss, argnums=(0, 1, 2, 3, 4)))(h0, a, v, k, q, dh, do)
    for x, y in zip(grads, want[2:]):
        check("gradient", x, y.double().cpu())
    n = torch.tensor([40, 0, 3, 17], device="cuda", dtype=torch.int32)
    mapped = torch.func.vmap(lambda h, a, v, k, q, n: _chunk()(h, a, v, k, q, n))(h0, a, v, k, q, n)
    for x, y in zip(mapped, _chunk()(h0, a, v, k, q, n)):
        assert torch.equal(x, y)
    head = torch.full((2,), -0.1, device="cuda")
    per_head = torch.func.vmap(torch.func.grad(loss, argnums=1), in_dims=(0, None, 0, 0, 0, 0, 0))(h0, head, v, k, q, dh, do)
    assert per_head.shape == (4, 2)
    total = step(_chunk(), h0, head, v, k, q, dh, do)[3]
    check("dlog_decay", per_head.sum(0), total.double().cpu(), scale=per_head.abs().sum())
    x = [y.clone().requires_grad_() for y in (h0, a, v, k, q)]
    (g,) = torch.autograd.grad(_chunk()(*x)[1].sum(), x[2], create_graph=True)
    with pytest.raises(NotImplementedError, match="second-order"):
        torch.autograd.grad(g.sum(), x[4])


def test_one_cotangent_alone():
    h0, a, v, k, q, dh, do = inputs(2, 50, 2, 2, 32, 32, seed=14)
    zero = torch.zeros_like
    for use in (0, 1):
        arrays = [x.clone().requires_grad_() for x in (h0, a, v, k, q)]
        res = _chunk()(*arrays)
        got = torch.autograd.grad(res[use], arrays, (dh, do)[use])
        want = step(_chunk(), h0, a, v, k, q, dh if use == 0 else zero(dh), do if use else zero(do))[2:]
        for x, y in zip(got, want):
            assert torch.equal(x, y)


def test_replays_from_a_graph():
    """The C entry points only enqueue kernels: a step records and replays, on new inputs, as the eager calls compute it."""
    from gla_jax_amd import chunk_decay, decay_step
    B, T, H, D = 2, 300, 4, 64
    dev = inputs(B, T, H, 2, D, D, decay="head", seed=20)
    states = torch.zeros(B, H, D, D, device="cuda")
    run = lambda: list(step(chunk_decay, *dev)) + [decay_step(states, dev[1], dev[2][:, 0], dev[3][:, 0], dev[4][:, 0])]  # noqa: E731
    run()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        replayed = run()
    for i in range(3):
        for x, y in zip(dev, inputs(B, T, H, 2, D, D, decay="head", seed=30 + i)):
            x.copy_(y)
        states.fill_(0.5)
        graph.replay()
        torch.cuda.synchronize()
        after = states.clone()
        states.fill_(0.5)
        for x, y in zip(replayed, run()):
            assert torch.equal(x, y)
        assert torch.equal(after, states)


def test_offsets_past_32_bits():
    """Rows behind 2^31 elements: the last heads of the last tokens, against a call on those heads alone."""
    T, H, D = 8448, 2048, 128
    v, k, q = (torch.empty(1, T, H, D, device="cuda", dtype=torch.bfloat16).normal_() for _ in range(3))
    a, h0 = torch.full((1, T, H), -0.05, device="cuda"), torch.zeros(1, H, D, D, device="cuda")
    assert v.numel() > 1 << 31
    hT, out = _chunk()(h0, a, v, k, q)
    last = slice(H - 2, H)
    hT2, out2 = _chunk()(h0[:, last], a[:, :, last], v[:, :, last], k[:, :, last], q[:, :, last])
    check("hidden_final", hT[:, last], hT2.double().cpu())
    check("out", out[:, -200:, last], out2[:, -200:].double().cpu())


# ---- decay_step ---------------------------------------------------------------------------------
def _step_reference(states, a, v, k, q, slots=None, parents=None):
    s, v, k, q = (x.double().cpu() for x in (states, v, k, q))
    B, H, DV = v.shape
    heads = torch.arange(H) // (H // k.shape[1])
    a = a.double().cpu().expand(B, H)
    new, out = s.clone(), torch.zeros(B, H, DV, dtype=torch.float64)
    where = [b if slots is None else int(slots[b]) for b in range(B)]
    there = lambda i: 0 <= i < s.shape[0]  # noqa: E731
    for b in range(B):
        if not there(where[b]):
            continue
        source = where[b]
        if parents is not None:
            W = parents.shape[1]
            p = int(parents[b // W, b % W])
            if 0 <= p < W and there(where[b // W * W + p]):
                source = where[b // W * W + p]
        x = a[b].exp()[:, None, None] * s[source] + k[b][heads][:, :, None] * v[b][:, None, :]
        new[where[b]] = x
        out[b] = (x * q[b][heads][:, :, None]).sum(1)
    return new, out


def _step_inputs(N, B, H, HK, DK, DV, dtype, state, seed):
    h0, a, v, k, q, _, _ = inputs(B, 1, H, HK, DK, DV, dtype, seed=seed)
    g = torch.Generator().manual_seed(seed)
    return torch.randn(N, H, DK, DV, generator=g).to(state).cuda(), a[:, 0], v[:, 0], k[:, 0], q[:, 0]


@pytest.mark.parametrize("state", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("DK, DV", [(16, 16), (48, 80), (64, 64), (128, 128), (144, 32), (256, 256)])
def test_single_tokens(DK, DV, dtype, state):
    from gla_jax_amd import decay_step
    states, a, v, k, q = _step_inputs(5, 5, 4, 2, DK, DV, dtype, state, DK)
    new, out = _step_reference(states, a, v, k, q)
    got = decay_step(states, a, v, k, q)
    check("out", got, out)
    check("states", states, new)


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_slots(index):
    """Rows in any order of a pool with room for more; rows without a state, and slots past the pool, change nothing."""
    from gla_jax_amd import decay_step
    states, a, v, k, q = _step_inputs(300, 290, 4, 4, 32, 32, torch.bfloat16, torch.float32, 3)
    slots = torch.randperm(300, generator=torch.Generator().manual_seed(0))[:290].to(index).cuda()
    slots[::7] = -1
    slots[5], slots[6] = 300, 2 ** 31 - 1
    new, out = _step_reference(states, a, v, k, q, slots)
    got = decay_step(states, a, v, k, q, slots=slots)
    check("out", got, out)
    check("states", states, new)
    assert not got[::7].any() and not got[5:7].any()


@pytest.mark.parametrize("pooled", [False, True])
@pytest.mark.parametrize("W, DK, state", [(1, 32, torch.float32), (2, 64, torch.bfloat16), (8, 64, torch.float32), (9, 256, torch.float32),
                                          (8, 256, torch.bfloat16), (16, 128, torch.float32), (17, 32, torch.float32), (64, 32, torch.bfloat16)])
def test_beams(W, DK, state, pooled):
    """Every beam goes on from the state of another, as that was before any was written."""
    from gla_jax_amd import decay_step
    G = 3
    states, a, v, k, q = _step_inputs(G * W + 4, G * W, 4, 2, DK, 64, torch.bfloat16, state, W)
    gen = torch.Generator().manual_seed(W)
    parents = torch.randint(-1, W + 1, (G, W), generator=gen).cuda()
    slots = None
    if pooled:
        slots = torch.randperm(G * W + 4, generator=gen)[:G * W].cuda()
        slots[W // 2] = -1
    new, out = _step_reference(states, a, v, k, q, slots, parents)
    got = decay_step(states, a, v, k, q, slots=slots, parents=parents)
    check("out", got, out)
    check("states", states, new)


def test_steps_go_on_from_a_prompt():
    """A prompt's state and single tokens after it are the whole sequence."""
    from gla_jax_amd import chunk_decay, decay_step
    h0, a, v, k, q, _, _ = inputs(3, 80, 4, 2, 64, 32, torch.float32, seed=21)
    hT, out = reference(h0, a, v, k, q)
    states, _ = chunk_decay(h0, a[:, :70], v[:, :70], k[:, :70], q[:, :70])
    for t in range(70, 80):
        check("out", decay_step(states, a[:, t], v[:, t], k[:, t], q[:, t]), out[:, t])
    check("states", states, hT)


def test_step_of_a_projection_and_a_constant_decay():
    from gla_jax_amd import decay_step
    states, _, v, k, q = _step_inputs(6, 6, 4, 4, 32, 32, torch.bfloat16, torch.float32, 5)
    a = torch.tensor([-0.01, -0.1, -1.0, -float("inf")], device="cuda")
    rows = torch.cat([x.reshape(6, -1) for x in (q, k, v)], -1)
    q2, k2, v2 = (x.unflatten(-1, (4, 32)) for x in rows.split([128] * 3, -1))
    new, out = _step_reference(states, a, v, k, q)
    check("out", decay_step(states, a, v2, k2, q2), out)
    check("states", states, new)


def test_pool_past_32_bits():
    from gla_jax_amd import decay_step
    N, H, D = 8448, 16, 128
    states = torch.zeros(N, H, D, D, device="cuda")
    assert states.numel() > 1 << 31
    _, a, v, k, q = _step_inputs(1, 2, H, H, D, D, torch.bfloat16, torch.float32, 6)
    states[-1] = 1.0
    slots = torch.tensor([N - 1, 0], device="cuda")
    new, out = _step_reference(states[[N - 1, 0]], a, v, k, q)
    check("out", decay_step(states, a, v, k, q, slots=slots), out)
    check("states", states[[N - 1, 0]], new)
    assert not states[1:N - 1].any()
