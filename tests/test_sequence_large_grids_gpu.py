"""Sequence-layer calls of more than 2^32 threads, which one axis of a launch does not hold."""
import math

import pytest
import torch

import sequence_reference as ref
from test_linear_attention_gpu import check_backward, check_forward

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from dsp_amd import ops
    return ops


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotary(ops, dev, layout):
    """2 x 2^31 tokens of one pair each, 17 GB in place, a thread a pair: zeros, and rows that are not at either end and in
    the middle."""
    n = 1 << 31
    x = torch.zeros(2, n, 1, 2, dtype=torch.float16, device=dev)
    places = [(b, t) for b in (0, 1) for t in (0, 1, (1 << 24) * 8 + 5, n - 2, n - 1)]
    pair = torch.tensor([1.0, -0.5], dtype=torch.float16, device=dev)
    for b, t in places:
        x[b, t, 0] = pair
    assert ops.rotary(x, [0.75], layout=layout, out=x) is x
    for b, t in places:
        assert torch.equal(x[b, t, 0], ops.rotary(pair.view(1, 1, 2), [0.75], position=t, layout=layout)[0, 0]), (b, t)
        x[b, t, 0] = 0
    assert all(not x[b, i:i + (1 << 28)].any() for b in (0, 1) for i in range(0, n, 1 << 28))


def test_backward_of_shared_heads(ops, dev):
    """More than 2^24 rows whose gradients are added up over heads."""
    b, n, h = 16385, 1024, 2
    g = torch.Generator(dev).manual_seed(1)
    q, k, v = (torch.randn(b, n, 1, 1, generator=g, device=dev) for _ in range(3))
    do = torch.randn(b, n, h, 1, generator=g, device=dev)
    ld = [-0.1, -0.01]
    grads = ops.linear_attention_backward(q, k, v, ld, do, scale=0.5)
    for i in (0, 9000, b - 1):
        a = [x[i:i + 1] for x in (q, k, v)]
        check_backward(*a, ld, 0.5, None, do[i:i + 1], None, [x[i:i + 1] for x in grads], None)


def test_step(ops, dev):
    """65,537 rows of 256 heads."""
    b, h = 65537, 256
    g = torch.Generator(dev).manual_seed(2)
    q, k, v = (torch.randn(b, 1, 1, generator=g, device=dev) for _ in range(3))
    s0 = torch.randn(b, h, 1, 1, generator=g, device=dev)
    state, ld = s0.clone(), [-0.01 * i for i in range(h)]
    out = ops.linear_attention_step(q, k, v, ld, state, scale=0.5)
    w = torch.exp(torch.tensor(ld, dtype=torch.float64, device=dev))[:, None, None]
    kv = (k.double() * v.double())[:, :, None]
    want, size = s0.double() * w + kv, s0.double().abs() * w + kv.abs()
    assert ((state.double() - want).abs() <= 8 * 2.0 ** -24 * size).all()
    assert ((out.double() - 0.5 * q.double() * want[..., 0]).abs() <= 12 * 2.0 ** -24 * q.double().abs() * size[..., 0]).all()


def test_packed_states_in_place(ops, dev):
    """262,145 sequences of 64 heads, all but one of them empty, that one cut into joined segments: every state is kept but
    its own."""
    b, h, n, at = 262145, 64, 4096, 200000
    g = torch.Generator(dev).manual_seed(3)
    q, k, v = (torch.randn(n, 1, 1, generator=g, device=dev) for _ in range(3))
    s0 = torch.randn(b, h, 1, 1, generator=g, device=dev)
    offsets = torch.zeros(b + 1, dtype=torch.int64, device=dev)
    offsets[at + 1:] = n
    state, ld = s0.clone(), [math.log1p(-2.0 ** -(3 + i % 9)) for i in range(h)]
    out = ops.linear_attention(q, k, v, ld, scale=0.5, state=state, new_state=state, offsets=offsets)
    check_forward(q[None], k[None], v[None], ld, 0.5, s0[at:at + 1], out[None], state[at:at + 1])
    state[at] = s0[at]
    assert torch.equal(state, s0)
    assert ref.heads_of(q[None], h).shape == (1, n, h, 1)
