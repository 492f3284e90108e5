"""Linear attention on values at the ends of their types -- infinities, NaN, the largest finite numbers -- against the 64-bit
recurrence: which outputs are not finite, and that the others are as near as ever."""
import math

import pytest
import torch

import sequence_reference as ref
from test_linear_attention_gpu import TYPES, make

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from dsp_amd import ops
    return ops


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("ld", [[-2.0, -5.0], [-math.inf, -1.0]], ids=str)
@pytest.mark.parametrize("at", [0, 3, 66])
@pytest.mark.parametrize("kind", TYPES)
def test_what_is_not_finite_outlives_a_weight_that_underflows(ops, dev, kind, at, ld, bad):
    """0 * NaN is NaN: a head that forgets fast carries what is not finite on as a slow one does, within a chunk (where the
    decay between two tokens comes to 0 in fp32) as from one to the next."""
    b, n, h, dk, dv = 1, 200, 2, 48, 40
    clean = make(dev, TYPES[kind], b, n, h, h, h, h, dk, dv, seed=11)
    terms = dk + dv + n
    for which in range(4):
        for head in range(h):
            q, k, v, do, s0, d1 = (x.clone() for x in clean)
            (q, k, v, do)[which][0, at, head, 5] = bad
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
                assert torch.equal(torch.isfinite(x.cpu()), fine), (which, head, i)
                ref.near(x.cpu()[fine], w[fine], t[fine], terms, x.dtype, operands=i not in (1, 5))


def near(got, want, total, terms, dtype, factor, operands=True):
    """ref.near's bound, and what it leaves out below the normal range, where steps do not shrink any more: fp32's are 2^-149
    there and bf16's 2^-133.  Each of the 2 terms + 64 sums and products is off by up to half a step then, 2^-150; each of
    the `terms` operands that are rounded to bf16 by 2^-134; either is multiplied by one more factor, `factor` at most (or by
    none); and the result is rounded once."""
    got = got.detach().cpu().double()
    assert got.shape == want.shape and torch.isfinite(got).all()
    half, f = torch.finfo(dtype).eps / 2, max(1.0, factor)
    bound = half * want.abs() * 1.01 + (2 * terms + 64) * (2.0 ** -24 * total + 2.0 ** -150 * f) + 2.0 ** -150
    if dtype == torch.bfloat16:
        bound = bound + 2.0 ** -134
        if operands:
            bound = bound + half * 1.01 * total + 2.0 ** -134 * terms * f
    over = (got - want).abs() - bound
    assert (over <= 0).all(), f"off by up to {over.max():.3g} more than the bound ({(over > 0).sum()} of {over.numel()})"


@pytest.mark.parametrize("log_decay", [math.log1p(-1 / 32), -0.002, -0.3], ids=lambda x: f"{x:.3f}")
@pytest.mark.parametrize("kind", ["bf16", "fp32"])
def test_large_values_and_small_ones(ops, dev, kind, log_decay):
    """Values, states and gradients of 1e35 beside factors of 1e-35, and the other way round: what the recurrence keeps finite
    is finite, and as near as for values around one.  (Products with both factors large are left out: q . k, v . dout and
    what the state adds have to stay finite in fp32.)"""
    b, n, h, dk, dv, big, small = 2, 700, 1, 24, 40, 1e35, 1e-35
    ld, terms = [log_decay], dk + dv + n
    for size in (dict(v=big, k=small), dict(v=small, k=big), dict(s0=big, q=small, k=big, v=1.0), dict(do=big, q=small, d1=big * 1e-35)):
        q, k, v, do, s0, d1 = make(dev, TYPES[kind], b, n, h, h, h, h, dk, dv, seed=13)
        q, k, v, do, s0, d1 = (x * size.get(name, 1.0) for name, x in zip(("q", "k", "v", "do", "s0", "d1"), (q, k, v, do, s0, d1)))
        if "s0" in size:
            do = do * small
        end, ds = torch.empty_like(s0), torch.empty_like(s0)
        out = ops.linear_attention(q, k, v, ld, scale=0.3, state=s0, new_state=end)
        grads = ops.linear_attention_backward(q, k, v, ld, do, scale=0.3, state=s0, dnew_state=d1, dstate=ds)
        args = [x.cpu().double() for x in (q, k, v, do, s0, d1)]
        pos = [x.abs() for x in args]
        want = [*ref.forward(*args[:3], ld, 0.3, s0), *ref.backward(*args[:3], ld, 0.3, s0, args[3], d1)]
        total = [*ref.forward(*pos[:3], ld, 0.3, pos[4]), *ref.backward(*pos[:3], ld, 0.3, pos[4], pos[3], pos[5])]
        mq, mk, mv, mdo = (x.max().item() for x in pos[:4])  # last factors: v and q of o, k of the state, k and dout of dq, ...
        factor = [max(mq, mv), mk, max(mk, mdo), max(mq, mv), max(mk, mdo), mq]
        for i, (x, w, t, f) in enumerate(zip((out, end, *grads, ds), want, total, factor)):
            near(x, w, t, terms, x.dtype, f, operands=i not in (1, 5))


@pytest.mark.parametrize("n", [1, 64, 150, 700, 1400])
@pytest.mark.parametrize("kind", ["bf16", "fp32"])
def test_an_infinite_state_stays_infinite(ops, dev, kind, n):
    """w * inf = inf for every decay but zero, whichever way w^n rounds: after single tokens, a few chunks, and segments."""
    b, h, dk, dv = 1, 12, 24, 40
    q, k, v, _, s0, _ = make(dev, TYPES[kind], b, n, h, h, h, h, dk, dv, seed=14)
    ld = [0.0, -0.001, -0.002, -0.003, -0.01, -0.011, -0.02, -0.03, math.log(0.5) / 64, -0.1, -0.2, -0.3]
    s0[:, :, 3, 5], s0[:, :, 7, 6] = math.inf, -math.inf
    args = [x.cpu().double() for x in (q, k, v)]
    want, wend = ref.forward(*args, ld, 0.3, s0)
    end = torch.empty_like(s0)
    out = ops.linear_attention(q, k, v, ld, scale=0.3, state=s0, new_state=end)
    odd = ~torch.isfinite(wend)
    assert odd.sum() == 2 * h and torch.equal(end.cpu()[odd].double(), wend[odd]) and torch.isfinite(end.cpu()[~odd]).all()
    assert torch.equal(torch.isfinite(out.cpu()), torch.isfinite(want))
    if n == 1:
        state = s0.clone()
        one = ops.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, state, scale=0.3)
        odd_o = ~torch.isfinite(want[:, 0])
        assert torch.equal(state.cpu()[odd].double(), wend[odd]) and torch.isfinite(state.cpu()[~odd]).all()
        assert torch.equal(one.cpu()[odd_o].double(), want[:, 0][odd_o]) and torch.isfinite(one.cpu()[~odd_o]).all()
