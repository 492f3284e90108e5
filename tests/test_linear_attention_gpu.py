"""Linear attention with a decay for each head against the 64-bit recurrence (tests/sequence_reference.py)."""
import math

import pytest
import torch

import sequence_reference as ref

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


@pytest.fixture(scope="module")
def ops():
    from dsp_amd import ops
    return ops


def decays(h, kind="mixed"):
    if kind == "mixed":  # from forgetting at once to never
        some = [-math.inf, -2.0, -0.7, -0.05, -0.002, 0.0]
        return [some[(3 * i + 4) % 6] for i in range(h)]
    return [math.log1p(-2.0 ** -(5 + i % 5)) for i in range(h)]


def make(dev, t, b, n, h, hq, hk, hv, dk, dv, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g).to(t).to(dev)  # noqa: E731
    return r(b, n, hq, dk), r(b, n, hk, dk), r(b, n, hv, dv), r(b, n, h, dv), \
        torch.randn(b, h, dk, dv, generator=g).to(dev), torch.randn(b, h, dk, dv, generator=g).to(dev)


def check_forward(q, k, v, ld, scale, state, out, end):
    h = len(ld)
    fq, fk, fv = (ref.heads_of(x, h) for x in (q, k, v))
    want, wend = ref.forward(fq, fk, fv, ld, scale, state)
    total, tend = ref.forward(fq.abs(), fk.abs(), fv.abs(), ld, abs(scale), None if state is None else state.abs())
    terms = q.shape[-1] + q.shape[1]
    ref.near(out, want, total, terms, q.dtype)
    if end is not None:
        ref.near(end, wend, tend, terms, torch.float32)


def check_backward(q, k, v, ld, scale, state, dout, dend, grads, dstate):
    h = len(ld)
    args = [ref.heads_of(x, h) for x in (q, k, v)]
    do = dout.detach().cpu().double()
    want = ref.backward(*args, ld, scale, state, do, dend)
    total = ref.backward(*(x.abs() for x in args), ld, abs(scale), None if state is None else state.abs(), do.abs(),
                         None if dend is None else dend.abs())
    terms = max(q.shape[-1], v.shape[-1]) + q.shape[1] + h
    for got, w, t in zip(grads, want, total):
        ref.near(got, ref.shared(w, got.shape[2]), ref.shared(t, got.shape[2]), terms, q.dtype)
    if dstate is not None:
        ref.near(dstate, want[3], total[3], terms, torch.float32)


SHAPES = [  # batch, n, heads, of q, of k, of v, dim_k, dim_v
    (1, 1, 1, 1, 1, 1, 1, 1),
    (2, 1, 3, 3, 3, 3, 16, 16),
    (1, 2, 2, 1, 2, 2, 33, 7),
    (2, 63, 2, 2, 2, 2, 64, 64),
    (1, 64, 4, 4, 2, 1, 48, 80),
    (3, 65, 2, 2, 2, 2, 128, 128),
    (1, 129, 4, 1, 1, 4, 128, 64),
    (1, 200, 2, 2, 2, 2, 100, 130),
    (1, 97, 2, 2, 1, 2, 256, 256),
    (1, 150, 1, 1, 1, 1, 192, 31),
    (1, 700, 2, 2, 2, 2, 64, 128),   # cut in time
    (1, 1091, 1, 1, 1, 1, 130, 72),  # cut in time, odd
]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("kind", TYPES)
def test_forward(ops, dev, kind, shape):
    q, k, v, _, s0, _ = make(dev, TYPES[kind], *shape)
    ld, scale = decays(shape[2]), shape[6] ** -0.5
    end = torch.full_like(s0, math.nan)
    out = ops.linear_attention(q, k, v, ld, scale=scale, state=s0, new_state=end)
    check_forward(q, k, v, ld, scale, s0, out, end)
    out = ops.linear_attention(q, k, v, ld, scale=scale)
    check_forward(q, k, v, ld, scale, None, out, None)


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("kind", TYPES)
def test_backward(ops, dev, kind, shape):
    q, k, v, do, s0, d1 = make(dev, TYPES[kind], *shape)
    ld, scale = decays(shape[2]), shape[6] ** -0.5
    ds = torch.full_like(s0, math.nan)
    grads = ops.linear_attention_backward(q, k, v, ld, do, scale=scale, state=s0, dnew_state=d1, dstate=ds)
    check_backward(q, k, v, ld, scale, s0, do, d1, grads, ds)
    grads = ops.linear_attention_backward(q, k, v, ld, do, scale=scale)
    check_backward(q, k, v, ld, scale, None, do, None, grads, None)


@pytest.mark.parametrize("kind", ["bf16", "fp32"])
def test_views_of_a_fused_projection(ops, dev, kind):
    """q, k, v as views of one buffer, o into a view, one of them off the 16-byte grid; keys broadcast over tokens' heads."""
    b, n, h, d = 2, 130, 3, 40
    g = torch.Generator().manual_seed(5)
    for off in (0, 1):
        fused = torch.randn(b, n, 3 * h * d + off, generator=g).to(TYPES[kind]).to(dev)
        q, k, v = (fused[..., off + i * h * d:off + (i + 1) * h * d].unflatten(-1, (h, d)) for i in range(3))
        wide = torch.full((b, n, h, 2 * d), 7.0, dtype=TYPES[kind], device=dev)
        ld = decays(h)
        ops.linear_attention(q, k, v, ld, scale=0.3, out=wide[..., :d])
        check_forward(q, k, v, ld, 0.3, None, wide[..., :d], None)
        assert (wide[..., d:] == 7).all()
    one = torch.randn(b, 1, h, d, generator=g).to(TYPES[kind]).to(dev).expand(b, n, h, d)  # the same key for every token
    out = ops.linear_attention(q, one, v, ld, scale=0.3)
    check_forward(q, one, v, ld, 0.3, None, out, None)
    do = torch.randn(b, h, n, d, generator=g).to(TYPES[kind]).to(dev).transpose(1, 2)
    grads = ops.linear_attention_backward(q, one, v, ld, do, scale=0.3)
    check_backward(q, one, v, ld, 0.3, None, do, None, grads, None)


LENGTHS = [[0, 1, 5, 64, 0, 200, 33], [3], [0, 0], [700, 0, 129]]


@pytest.mark.parametrize("lengths", LENGTHS, ids=str)
@pytest.mark.parametrize("kind", ["bf16", "fp32"])
def test_packed(ops, dev, kind, lengths):
    """Packed sequences, empty ones among them; rows in front and behind hold NaN and are left alone, or get zeros."""
    h, hk, dk, dv, front, back = 4, 2, 48, 64, 3, 5
    rows, b = front + sum(lengths) + back, len(lengths)
    q, k, v, do, _, _ = (x[0] for x in make(dev, TYPES[kind], 1, rows, h, h, hk, h, dk, dv, seed=9))
    s0, d1 = (torch.randn(b, h, dk, dv, generator=torch.Generator().manual_seed(i)).to(dev) for i in (1, 2))
    offsets = torch.tensor([front] + lengths, device=dev).cumsum(0)
    for x in (q, k, v, do):
        x[:front] = math.nan
        x[rows - back:] = math.nan
    ld = decays(h)
    for most in (max(lengths), None):
        end, ds = torch.full_like(s0, math.nan), torch.full_like(s0, math.nan)
        kept = torch.full((rows, h, dv), 7.0, dtype=TYPES[kind], device=dev)
        ops.linear_attention(q, k, v, ld, scale=0.5, state=s0, new_state=end, offsets=offsets, max_length=most, out=kept)
        out = ops.linear_attention(q, k, v, ld, scale=0.5, state=s0, offsets=offsets, max_length=most)
        grads = ops.linear_attention_backward(q, k, v, ld, do, scale=0.5, state=s0, dnew_state=d1, dstate=ds, offsets=offsets, max_length=most)
        inside = slice(front, rows - back)
        assert torch.equal(kept[inside], out[inside])
        for edge in (slice(0, front), slice(rows - back, rows)):
            assert (kept[edge] == 7).all() and (out[edge] == 0).all() and all((x[edge] == 0).all() for x in grads)
        for i, n in enumerate(lengths):
            at = slice(int(offsets[i]), int(offsets[i]) + n)
            a = [x[at][None] for x in (q, k, v)]
            check_forward(*a, ld, 0.5, s0[i:i + 1], out[at][None], end[i:i + 1])
            check_backward(*a, ld, 0.5, s0[i:i + 1], do[at][None], d1[i:i + 1], [x[at][None] for x in grads], ds[i:i + 1])


def test_padded(ops, dev):
    """A padded batch: what lies behind a sequence's length may be NaN, and out keeps what it held there."""
    lengths, n, h, dk, dv = [0, 1, 77, 150], 150, 2, 64, 72
    q, k, v, do, s0, d1 = make(dev, torch.bfloat16, 4, n, h, 1, h, h, dk, dv, seed=4)
    ln = torch.tensor(lengths, device=dev)
    for i, m in enumerate(lengths):
        for x in (q, k, v, do):
            x[i, m:] = math.nan
    ld = decays(h)
    end, ds = torch.empty_like(s0), torch.empty_like(s0)
    kept = torch.full((4, n, h, dv), 7.0, dtype=torch.bfloat16, device=dev)
    ops.linear_attention(q, k, v, ld, state=s0, new_state=end, lengths=ln, out=kept)
    grads = ops.linear_attention_backward(q, k, v, ld, do, state=s0, dnew_state=d1, dstate=ds, lengths=ln)
    for i, m in enumerate(lengths):
        assert (kept[i, m:] == 7).all() and all((x[i, m:] == 0).all() for x in grads)
        a = [x[i:i + 1, :m] for x in (q, k, v)]
        check_forward(*a, ld, 1.0, s0[i:i + 1], kept[i:i + 1, :m], end[i:i + 1])
        check_backward(*a, ld, 1.0, s0[i:i + 1], do[i:i + 1, :m], d1[i:i + 1], [x[i:i + 1, :m] for x in grads], ds[i:i + 1])


def test_lengths_outside_are_clamped(ops, dev):
    """Lengths and offsets are data: whatever they hold, the kernels stay inside the tensors."""
    q, k, v, _, _, _ = make(dev, torch.float32, 3, 40, 2, 2, 2, 2, 16, 16)
    out = ops.linear_attention(q, k, v, decays(2), lengths=torch.tensor([-5, 1 << 50, 40], device=dev))
    want = ops.linear_attention(q, k, v, decays(2), lengths=torch.tensor([0, 40, 40], device=dev))
    assert torch.equal(out, want)
    p = [x[0] for x in (q, k, v)]
    out = ops.linear_attention(*p, decays(2), offsets=torch.tensor([-9, 15, 1 << 40], device=dev))
    want = ops.linear_attention(*p, decays(2), offsets=torch.tensor([0, 15, 40], device=dev))
    assert torch.equal(out, want)


@pytest.mark.parametrize("kind", TYPES)
def test_states_carried_on(ops, dev, kind):
    """A prompt in two calls with the state in place, then single tokens, is the whole sequence; an empty call keeps it."""
    b, n, cut, h, dk, dv = 2, 300, 171, 3, 96, 80
    q, k, v, _, s0, _ = make(dev, TYPES[kind], b, n, h, h, h, h, dk, dv)
    ld = [-0.05, -0.4, 0.0]
    state, parts = s0.clone(), []
    for at in (slice(0, cut), slice(cut, cut), slice(cut, n - 4)):
        parts.append(ops.linear_attention(q[:, at], k[:, at], v[:, at], ld, scale=0.2, state=state, new_state=state))
    for t in range(n - 4, n):
        parts.append(ops.linear_attention_step(q[:, t], k[:, t], v[:, t], ld, state, scale=0.2)[:, None])
    check_forward(q, k, v, ld, 0.2, s0, torch.cat(parts, 1), state)


@pytest.mark.parametrize("n", [600, 1300])
def test_state_in_place_of_a_long_prompt(ops, dev, n):
    """Cut in time, with the state after the last token where the one before the first was: bit for bit the call with two."""
    q, k, v, _, s0, _ = make(dev, torch.bfloat16, 2, n, 3, 3, 3, 3, 64, 80)
    ld, end, both = [-0.001, -0.05, 0.0], torch.empty_like(s0), s0.clone()
    out = ops.linear_attention(q, k, v, ld, scale=0.2, state=s0, new_state=end)
    assert torch.equal(ops.linear_attention(q, k, v, ld, scale=0.2, state=both, new_state=both), out)
    assert torch.equal(both, end)
    lengths = torch.tensor([n, 40], device=dev)
    both = s0.clone()
    ops.linear_attention(q, k, v, ld, scale=0.2, state=s0, new_state=end, lengths=lengths)
    ops.linear_attention(q, k, v, ld, scale=0.2, state=both, new_state=both, lengths=lengths)
    assert torch.equal(both, end)


def test_nothing_from_nothing(ops, dev):
    """No tokens: gradients of nothing, and the state's gradient handed on."""
    q, k, v, do, s0, d1 = make(dev, torch.bfloat16, 2, 0, 2, 2, 2, 2, 16, 16)
    end, ds = torch.empty_like(s0), torch.empty_like(s0)
    assert ops.linear_attention(q, k, v, decays(2), state=s0, new_state=end).shape == (2, 0, 2, 16)
    assert torch.equal(end, s0)
    ops.linear_attention_backward(q, k, v, decays(2), do, dnew_state=d1, dstate=ds)
    assert torch.equal(ds, d1)
    ops.linear_attention(q, k, v, decays(2), new_state=end)
    assert (end == 0).all()
    rows, none = torch.ones(5, 2, 16, dtype=torch.bfloat16, device=dev), torch.zeros(1, dtype=torch.int64, device=dev)
    assert (ops.linear_attention(rows, rows, rows, decays(2), offsets=none) == 0).all()  # rows, but no sequence
    assert all((x == 0).all() for x in ops.linear_attention_backward(rows, rows, rows, decays(2), rows, offsets=none))


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("shape", [(1, 1, 1, 1, 1, 1, 1), (5, 4, 2, 1, 4, 64, 64), (3, 2, 2, 2, 2, 100, 30), (2, 3, 3, 3, 1, 256, 130), (70, 2, 2, 2, 2, 33, 256)], ids=str)
def test_step(ops, dev, kind, shape):
    b, h, hq, hk, hv, dk, dv = shape
    q, k, v, _, _, _ = (x[:, 0] for x in make(dev, TYPES[kind], b, 1, h, hq, hk, hv, dk, dv))
    ld = decays(h)
    s0 = torch.randn(b, h, dk, dv, generator=torch.Generator().manual_seed(8)).to(dev)
    state = s0.clone()
    out = ops.linear_attention_step(q, k, v, ld, state, scale=0.25)
    args = [ref.heads_of(x[:, None], h) for x in (q, k, v)]
    want, end = ref.forward(*args, ld, 0.25, s0)
    total, tend = ref.forward(*(x.abs() for x in args), ld, 0.25, s0.abs())
    ref.near(out[:, None], want, total, dk, TYPES[kind], operands=False)  # S and the products stay in fp32
    ref.near(state, end, tend, dk, torch.float32)


def test_step_slots(ops, dev):
    """Slots of a pool: skipped rows, slots that several rows name (in their order), states nobody names."""
    b, pool, h, dk, dv = 300, 9, 2, 32, 72
    q, k, v, _, _, _ = (x[:, 0] for x in make(dev, torch.float32, b, 1, h, h, 1, h, dk, dv))
    slots = torch.full((b,), -1)
    slots[::50], slots[7], slots[8], slots[299], slots[298] = 3, pool, 1 << 40, 0, 3
    s0 = torch.randn(pool, h, dk, dv, generator=torch.Generator().manual_seed(8)).to(dev)
    state, ld = s0.clone(), [-0.3, -0.01]
    out = ops.linear_attention_step(q, k, v, ld, state, slots=slots.to(dev))
    one, want = s0.clone(), torch.zeros(b, h, dv, device=dev)
    for i, s in enumerate(slots.tolist()):
        if 0 <= s < pool:
            want[i] = ops.linear_attention_step(q[i:i + 1], k[i:i + 1], v[i:i + 1], ld, one[s:s + 1])[0]
    assert torch.equal(out, want) and torch.equal(state, one)


def test_long_memory(ops, dev):
    """A decay of 1 - 2^-16 over 20,000 tokens: w^C rounded to fp32 alone would be 2^-25 off each chunk."""
    n = 20000
    q, k, v, _, _, _ = make(dev, torch.bfloat16, 1, n, 1, 1, 1, 1, 16, 16)
    k, v = k.abs(), v.abs()  # sums that grow: nothing hides the drift
    ld, end = [math.log1p(-2.0 ** -16)], torch.empty(1, 1, 16, 16, device=dev)
    ops.linear_attention(q, k, v, ld, new_state=end)
    w = torch.exp(ld[0] * torch.arange(n - 1, -1, -1, dtype=torch.float64))
    want = torch.einsum("td,tn->dn", k[0, :, 0].cpu().double() * w[:, None], v[0, :, 0].cpu().double())
    # 2^-25 and less for each of the 16 sums of a chunk's 64 products and each of 313 chunks, and for the weights
    assert ((end[0, 0].cpu().double() - want).abs() <= 400 * 2.0 ** -24 * want).all()


def test_masked_places_may_hold_anything(ops, dev):
    """A key whose product with an earlier query overflows, or is NaN, does not reach that query."""
    q, k, v, _, _, _ = make(dev, torch.float32, 1, 64, 1, 1, 1, 1, 32, 32)
    k[0, 40:] = 3e38
    q[0, :40] = q[0, :40].abs() * 10
    out = ops.linear_attention(q, k, v, [-0.1])
    want = ops.linear_attention(q[:, :40], k[:, :40], v[:, :40], [-0.1])
    assert torch.equal(out[:, :40], want)


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("kind", ["bf16", "fp32"])
def test_what_is_not_finite_stays_where_it_belongs(ops, dev, kind, bad):
    """One bad element of q, k, v or dout: the outputs that the recurrence carries it to are not finite, all others are as
    near as ever -- earlier tokens of the same chunk among them, in either direction of time."""
    b, n, h, dk, dv, at = 1, 150, 2, 48, 72, 70
    clean = make(dev, TYPES[kind], b, n, h, h, h, h, dk, dv, seed=11)
    ld, terms = [-0.05, -0.2], dk + dv + n
    for which in range(4):
        q, k, v, do, s0, d1 = (x.clone() for x in clean)
        (q, k, v, do)[which][0, at, 1, 5] = bad
        end, ds = torch.empty_like(s0), torch.empty_like(s0)
        out = ops.linear_attention(q, k, v, ld, scale=0.3, state=s0, new_state=end)
        grads = ops.linear_attention_backward(q, k, v, ld, do, scale=0.3, state=s0, dnew_state=d1, dstate=ds)
        args = [ref.heads_of(x, h) for x in (q, k, v)]
        pos = [ref.heads_of(x, h).abs() for x in clean[:3]]
        do64, cdo = do.cpu().double(), clean[3].cpu().double().abs()
        want = [*ref.forward(*args, ld, 0.3, s0), *ref.backward(*args, ld, 0.3, s0, do64, d1)]
        total = [*ref.forward(*pos, ld, 0.3, s0.abs()), *ref.backward(*pos, ld, 0.3, s0.abs(), cdo, d1.abs())]
        for i, (x, w, t) in enumerate(zip((out, end, *grads, ds), want, total)):
            fine = torch.isfinite(w)
            assert torch.equal(torch.isfinite(x.cpu()), fine), (which, i)
            ref.near(x.cpu()[fine], w[fine], t[fine], terms, x.dtype, operands=i not in (1, 5))


def test_offsets_past_32_bits(ops, dev):
    """Rows 2^17 bytes apart, 5 GB in all: the last ones are reached as the first ones are."""
    n, h, d = 40000, 1, 64
    big = torch.zeros(n, 1 << 16, dtype=torch.bfloat16, device=dev)
    g = torch.Generator().manual_seed(1)
    small = [torch.randn(n, h, d, generator=g).to(torch.bfloat16).to(dev) for _ in range(3)]
    views = [big[:, i * 128:i * 128 + d].unflatten(-1, (h, d)) for i in range(3)]
    for x, y in zip(views, small):
        x.copy_(y)
    wide = torch.empty(n, 1 << 16, dtype=torch.bfloat16, device=dev)[:, :d].unflatten(-1, (h, d))
    want = ops.linear_attention(*(x[None] for x in small), [-0.01])
    got = ops.linear_attention(*(x[None] for x in views), [-0.01], out=wide[None])
    assert torch.equal(got, want)
    do = small[0][None]
    for x, y in zip(ops.linear_attention_backward(*(x[None] for x in views), [-0.01], do), ops.linear_attention_backward(*(x[None] for x in small), [-0.01], do)):
        assert torch.equal(x, y)
    freq = 0.5 ** torch.arange(32, dtype=torch.float64).numpy()
    assert torch.equal(ops.rotary(views[0], freq), ops.rotary(small[0], freq))
    step = ops.linear_attention_step(views[0][-2:], views[1][-2:], views[2][-2:], [-0.1], torch.zeros(2, 1, d, d, device=dev))
    assert torch.equal(step, ops.linear_attention_step(small[0][-2:], small[1][-2:], small[2][-2:], [-0.1], torch.zeros(2, 1, d, d, device=dev)))


def test_differences(ops, dev):
    """The fp32 gradients along random directions against central differences of the forward call (64-bit sums of its fp32
    outputs: their errors, 2^-24 of about 100 terms, come in divided by the step 2^-4 -- the function is a cubic in the
    step for each operand alone, linear: the difference itself is exact)."""
    b, n, h, dk, dv = 1, 90, 2, 24, 40
    q, k, v, do, s0, d1 = make(dev, torch.float32, b, n, h, 1, h, h, dk, dv, seed=3)
    ld, ds = [-0.03, -0.2], torch.empty_like(s0)
    grads = [*ops.linear_attention_backward(q, k, v, ld, do, scale=0.3, state=s0, dnew_state=d1, dstate=ds), ds]

    def loss(args):
        end = torch.empty_like(s0)
        out = ops.linear_attention(*args[:3], ld, scale=0.3, state=args[3], new_state=end)
        parts = torch.cat(((out.double() * do.double()).flatten(), (end.double() * d1.double()).flatten()))
        return parts.sum().item(), parts.abs().sum().item()

    args = [q, k, v, s0]
    for i, gx in enumerate(grads):
        step = torch.randn(args[i].shape, generator=torch.Generator().manual_seed(i)).to(dev)
        up, down = list(args), list(args)
        up[i], down[i] = args[i] + step / 16, args[i] - step / 16
        (a, size), (c, _) = loss(up), loss(down)
        want, got = (a - c) * 8, (gx.double() * step.double()).sum().item()
        assert abs(want - got) <= 16 * 200 * 2.0 ** -24 * size, (i, want, got, size)


def test_repeats_streams_and_graphs(ops, dev):
    """Bit for bit the same: again, on two streams at once, and captured and replayed, with other work in between."""
    q, k, v, do, s0, d1 = make(dev, torch.bfloat16, 1, 1500, 4, 2, 1, 4, 64, 128, seed=6)
    ld = [-0.01, -0.02, -0.1, -0.5]

    def work():
        end, ds = torch.empty_like(s0), torch.empty_like(s0)
        out = ops.linear_attention(q, k, v, ld, scale=0.1, state=s0, new_state=end)
        grads = ops.linear_attention_backward(q, k, v, ld, do, scale=0.1, state=s0, dnew_state=d1, dstate=ds)
        st = end.clone()
        tok = ops.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, st, scale=0.1)
        return [out, end, *grads, ds, tok, st]

    want = work()
    assert all(torch.equal(x, y) for x, y in zip(want, work()))
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append([work() for _ in range(3)])
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for runs in got for run in runs for x, y in zip(run, want))
    graphs = []
    for _ in range(2):  # two graphs of the same calls: neither has the other's workspace
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = work()
        graphs.append((g, out))
    for _ in range(3):
        for (g, out), s in zip(graphs, streams):
            for x in out:
                x.zero_()
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        work()
        for _, out in graphs:
            assert all(torch.equal(x, y) for x, y in zip(out, want))


def test_library_workspace(ops, dev):
    """The C call with no workspace takes the library's own."""
    import ctypes as C
    from dsp_amd import capi
    import numpy as np
    q, k, v, _, _, _ = make(dev, torch.bfloat16, 1, 2048, 2, 2, 2, 2, 64, 64)
    a = ops._Attention(q, k, v, [-0.1, -0.2], None, None, None, 4)
    out = torch.empty_like(v)
    shape, ld = a.shape(out, "out", False), np.array([-0.1, -0.2]).tobytes()
    need = C.c_size_t(0)
    assert capi.lib().dsp_gpu_linear_attention_workspace(shape, 0, C.byref(need)) == 0 and need.value > 0
    stream = torch.cuda.current_stream().cuda_stream
    for _ in range(2):
        rc = capi.lib().dsp_gpu_linear_attention(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), shape, ld, 1.0, None, None, None, 0, stream)
        assert rc == 0
    assert torch.equal(out, ops.linear_attention(q, k, v, [-0.1, -0.2]))


def test_refusals(ops, dev):
    from dsp_amd.capi import DspGpuError
    q, k, v, do, s0, _ = make(dev, torch.bfloat16, 2, 8, 2, 2, 2, 2, 16, 16)
    ld, ln = [-0.1, -0.2], torch.tensor([8, 8], device=dev)
    off = torch.tensor([0, 8], device=dev)
    cases = [
        lambda: ops.linear_attention(q.double(), k, v, ld), lambda: ops.linear_attention(q, k.float(), v, ld),
        lambda: ops.linear_attention(q, k.cpu(), v, ld), lambda: ops.linear_attention(q[..., :8], k, v, ld),
        lambda: ops.linear_attention(q[:, :4], k, v, ld), lambda: ops.linear_attention(q[0], k[0], v[0], ld),
        lambda: ops.linear_attention(q, k, v, [-0.1, -0.2, -0.3]), lambda: ops.linear_attention(q, k, v, [0.1, -0.2]),
        lambda: ops.linear_attention(q, k, v, [math.nan, -0.2]), lambda: ops.linear_attention(q, k, v, [ld]),
        lambda: ops.linear_attention(q.transpose(-1, -2), k, v, ld), lambda: ops.linear_attention(q, k, v, ld, out=q),
        lambda: ops.linear_attention(q, k, v, ld, out=do.float()), lambda: ops.linear_attention(q, k, v, ld, state=s0[:1]),
        lambda: ops.linear_attention(q, k, v, ld, state=s0.half()), lambda: ops.linear_attention(q, k, v, ld, new_state=s0.cpu()),
        lambda: ops.linear_attention(q, k, v, ld, lengths=ln.int()), lambda: ops.linear_attention(q, k, v, ld, lengths=ln[:1]),
        lambda: ops.linear_attention(q, k, v, ld, lengths=ln.cpu()), lambda: ops.linear_attention(q, k, v, ld, offsets=off),
        lambda: ops.linear_attention(q[0], k[0], v[0], ld, offsets=off, lengths=ln), lambda: ops.linear_attention(q, k, v, ld, max_length=8),
        lambda: ops.linear_attention(q[0], k[0], v[0], ld, offsets=off[:0]), lambda: ops.linear_attention(q[0], k[0], v[0], ld, offsets=off, max_length=-1),
        lambda: ops.linear_attention(q, k, v, ld, scale=math.inf), lambda: ops.linear_attention_backward(q, k, v, ld, do[:, :4]),
        lambda: ops.linear_attention_backward(q, k, v, ld, do, dnew_state=s0, dstate=s0),
        lambda: ops.linear_attention_step(q, k, v, ld, s0), lambda: ops.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, None),
        lambda: ops.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, s0[:1]),
        lambda: ops.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, s0, slots=ln.int()),
        lambda: ops.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, s0.transpose(-1, -2), slots=ln),
    ]
    for i, call in enumerate(cases):
        with pytest.raises(DspGpuError) as e:
            call()
        assert e.value.code == -1, i


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotary_and_attention_together(ops, dev, layout):
    """A sequence layer as it is used: queries and keys of a fused projection rotated in place, the prompt mixed, then single
    tokens at their positions -- against the complex-pole recurrence in 64 bits, on the rotated values as rounded."""
    from dsp_amd import design
    b, n, new, h, d = 2, 140, 3, 4, 64
    g = torch.Generator().manual_seed(2)
    fused = torch.randn(b, n + new, 3, h, d, generator=g).to(torch.bfloat16).to(dev)
    raw = fused.clone()
    freq, ld, first = design.rotary_frequencies(32, scaling="ramp", factor=4.0), design.head_decays(h), 100000
    qk = fused[:, :, :2].flatten(2, 3)  # a view: queries and keys as 2 h heads
    assert qk.data_ptr() == fused.data_ptr()
    ops.rotary(qk[:, :n], freq, position=first, layout=layout, out=qk[:, :n])
    state = torch.zeros(b, h, d, d, device=dev)
    outs = [ops.linear_attention(fused[:, :n, 0], fused[:, :n, 1], fused[:, :n, 2], ld, scale=d ** -0.5, new_state=state)]
    for t in range(n, n + new):
        one = qk[:, t:t + 1]
        ops.rotary(one, freq, positions=torch.full((b, 1), first + t, device=dev), layout=layout, out=one)
        outs.append(ops.linear_attention_step(fused[:, t, 0], fused[:, t, 1], fused[:, t, 2], ld, state, scale=d ** -0.5)[:, None])
    angle = (first + torch.arange(n + new, dtype=torch.float64))[:, None] * torch.from_numpy(freq)
    x = raw[:, :, :2, :, :32].cpu().double()
    z = torch.complex(x[..., :16], x[..., 16:]) if layout == "half" else torch.view_as_complex(x.unflatten(-1, (16, 2)).contiguous())
    z = z * torch.polar(torch.ones_like(angle), angle)[:, None, None]
    want = torch.cat((z.real, z.imag), -1) if layout == "half" else torch.view_as_real(z).flatten(-2)
    got = fused[:, :, :2, :, :32].cpu().double()
    assert ((got - want).abs() <= 2.0 ** -8 * want.abs() * 1.001 + 1e-6 * x.abs().amax()).all()
    assert torch.equal(fused[:, :, :2, :, 32:], raw[:, :, :2, :, 32:]) and torch.equal(fused[:, :, 2], raw[:, :, 2])
    check_forward(fused[:, :, 0], fused[:, :, 1], fused[:, :, 2], list(ld), d ** -0.5, None, torch.cat(outs, 1), state)
