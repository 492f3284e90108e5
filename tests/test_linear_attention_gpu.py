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
