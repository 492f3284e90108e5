"""Linear attention cut in time into many segments (joined by a kernel of its own from seven on) against the 64-bit
recurrence: dense, padded and packed batches, both directions, with states before and gradients of the states after."""
import math

import pytest
import torch

from test_linear_attention_gpu import TYPES, check_backward, check_forward, make

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from dsp_amd import ops
    return ops


SLOW = [-0.0005, -0.02, 0.0, -0.004]  # states that outlive many segments

# One head of 64 columns: segments of 128 tokens, so the longest has up to 22 of them; single tokens, empty sequences, whole
# segments and one token more or less among them.
PACKED = [[2700, 0, 1, 128, 129, 257, 900], [127, 1, 0, 0, 1665, 128, 256], [5] * 40 + [1100] + [130] * 5]


@pytest.mark.parametrize("lengths", PACKED, ids=lambda x: str(sum(x)))
@pytest.mark.parametrize("kind", ["bf16", "fp32"])
def test_packed_sequences_of_many_segments(ops, dev, kind, lengths):
    h, dk, dv, front, back = 1, 24, 40, 61, 7
    rows, b = front + sum(lengths) + back, len(lengths)
    q, k, v, do, _, _ = (x[0] for x in make(dev, TYPES[kind], 1, rows, h, h, h, h, dk, dv, seed=3))
    s0, d1 = (torch.randn(b, h, dk, dv, generator=torch.Generator().manual_seed(i)).to(dev) for i in (1, 2))
    offsets = torch.tensor([front] + lengths, device=dev).cumsum(0)
    ld = SLOW[:h]
    for most in (max(lengths), None):
        end, ds = torch.full_like(s0, math.nan), torch.full_like(s0, math.nan)
        out = ops.linear_attention(q, k, v, ld, scale=0.3, state=s0, new_state=end, offsets=offsets, max_length=most)
        grads = ops.linear_attention_backward(q, k, v, ld, do, scale=0.3, state=s0, dnew_state=d1, dstate=ds, offsets=offsets, max_length=most)
        for edge in (slice(0, front), slice(rows - back, rows)):
            assert (out[edge] == 0).all() and all((x[edge] == 0).all() for x in grads)
        for i, n in enumerate(lengths):
            if n in lengths[:i] and n == 5:
                continue  # one of the short ones stands for all
            at = slice(int(offsets[i]), int(offsets[i]) + n)
            a = [x[at][None] for x in (q, k, v)]
            check_forward(*a, ld, 0.3, s0[i:i + 1], out[at][None], end[i:i + 1])
            check_backward(*a, ld, 0.3, s0[i:i + 1], do[at][None], d1[i:i + 1], [x[at][None] for x in grads], ds[i:i + 1])


def test_a_longest_length_below_the_longest(ops, dev):
    """Tokens from max_length on are left out: the call is that of the shortened sequences."""
    lengths, most, h, dk, dv = [1500, 300, 2000], 1100, 1, 16, 16
    q, k, v, do, _, _ = (x[0] for x in make(dev, torch.float32, 1, sum(lengths), h, h, h, h, dk, dv, seed=5))
    offsets = torch.tensor([0] + lengths, device=dev).cumsum(0)
    end, ds = (torch.empty(3, h, dk, dv, device=dev) for _ in range(2))
    out = ops.linear_attention(q, k, v, SLOW[:h], new_state=end, offsets=offsets, max_length=most)
    grads = ops.linear_attention_backward(q, k, v, SLOW[:h], do, dstate=ds, offsets=offsets, max_length=most)
    for i, n in enumerate(lengths):
        at, rest = (slice(int(offsets[i]) + a, int(offsets[i]) + b) for a, b in ((0, min(n, most)), (min(n, most), n)))
        a = [x[at][None] for x in (q, k, v)]
        check_forward(*a, SLOW[:h], 1.0, None, out[at][None], end[i:i + 1])
        check_backward(*a, SLOW[:h], 1.0, None, do[at][None], None, [x[at][None] for x in grads], ds[i:i + 1])
        assert (out[rest] == 0).all() and all((x[rest] == 0).all() for x in grads)


@pytest.mark.parametrize("shape", [(1, 1500, 2, 1, 2, 2, 40, 24), (2, 1000, 4, 2, 1, 4, 16, 72), (1, 1100, 1, 1, 1, 1, 200, 136)], ids=str)
@pytest.mark.parametrize("kind", TYPES)
def test_dense_sequences_of_many_segments(ops, dev, kind, shape):
    q, k, v, do, s0, d1 = make(dev, TYPES[kind], *shape, seed=7)
    ld, end, ds = SLOW[:shape[2]], torch.full_like(s0, math.nan), torch.full_like(s0, math.nan)
    out = ops.linear_attention(q, k, v, ld, scale=0.3, state=s0, new_state=end)
    check_forward(q, k, v, ld, 0.3, s0, out, end)
    grads = ops.linear_attention_backward(q, k, v, ld, do, scale=0.3, state=s0, dnew_state=d1, dstate=ds)
    check_backward(q, k, v, ld, 0.3, s0, do, d1, grads, ds)


def test_padded_sequences_of_many_segments(ops, dev):
    lengths, n, h, dk, dv = [1400, 0, 900, 1025], 1400, 2, 32, 48
    q, k, v, do, s0, d1 = make(dev, torch.bfloat16, 4, n, h, h, h, h, dk, dv, seed=8)
    ln, ld = torch.tensor(lengths, device=dev), SLOW[:h]
    end, ds = torch.empty_like(s0), torch.empty_like(s0)
    out = ops.linear_attention(q, k, v, ld, scale=0.3, state=s0, new_state=end, lengths=ln)
    grads = ops.linear_attention_backward(q, k, v, ld, do, scale=0.3, state=s0, dnew_state=d1, dstate=ds, lengths=ln)
    for i, m in enumerate(lengths):
        assert (out[i, m:] == 0).all() and all((x[i, m:] == 0).all() for x in grads)
        a = [x[i:i + 1, :m] for x in (q, k, v)]
        check_forward(*a, ld, 0.3, s0[i:i + 1], out[i:i + 1, :m], end[i:i + 1])
        check_backward(*a, ld, 0.3, s0[i:i + 1], do[i:i + 1, :m], d1[i:i + 1], [x[i:i + 1, :m] for x in grads], ds[i:i + 1])


@pytest.mark.parametrize("n", [300, 600, 2000])
@pytest.mark.parametrize("kind", ["bf16", "fp32"])
def test_states_in_place(ops, dev, kind, n):
    """The state after the last token over the one before the first: dense, padded and packed, one segment and many, bit for
    bit the call with two tensors (tests above hold that one to the recurrence)."""
    b, h, dk, dv = 3, 2, 40, 136
    q, k, v, _, s0, _ = make(dev, TYPES[kind], b, n, h, h, h, h, dk, dv, seed=12)
    packed = [x.flatten(0, 1) for x in (q, k, v)]
    calls = [((q, k, v), {}), ((q, k, v), dict(lengths=torch.tensor([n, 0, n // 2], device=dev))),
             (packed, dict(offsets=torch.tensor([0, n // 3, n // 3, 3 * n], device=dev))),
             (packed, dict(offsets=torch.tensor([5, 6, 200, 3 * n - 1], device=dev)))]
    for args, more in calls:
        end, both = torch.full_like(s0, math.nan), s0.clone()
        out = ops.linear_attention(*args, SLOW[:h], scale=0.3, state=s0, new_state=end, **more)
        again = ops.linear_attention(*args, SLOW[:h], scale=0.3, state=both, new_state=both, **more)
        assert torch.equal(again, out) and torch.equal(both, end)


def test_memory_of_many_short_packed_sequences(ops, dev):
    """1,000 sequences in 32,768 rows of 16 heads, max_length left out: 0.5 GB of tensors, and less than that of workspace."""
    rows, h, d = 32768, 16, 128
    q, k, v = (torch.randn(rows, h, d, device=dev, dtype=torch.bfloat16) for _ in range(3))
    offsets = (torch.arange(1001, device=dev) * rows) // 1000
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    out = ops.linear_attention(q, k, v, [-0.01] * h, offsets=offsets)
    grads = ops.linear_attention_backward(q, k, v, [-0.01] * h, out, offsets=offsets)
    torch.cuda.synchronize()
    new = (4 * rows * h * d) * 2
    assert torch.cuda.max_memory_allocated() - before <= new + 2 ** 27
    want = ops.linear_attention(q, k, v, [-0.01] * h, offsets=offsets, max_length=33)
    assert torch.equal(out, want)
    del grads


def test_very_many_packed_sequences(ops, dev):
    """60,000 sequences of 0 to 9 tokens and one of 2,000, max_length left out: the workgroups that start are those of
    segments that exist."""
    g = torch.Generator().manual_seed(2)
    lengths = torch.randint(0, 10, (60001,), generator=g)
    lengths[31234] = 2000
    rows, h, d = int(lengths.sum()), 4, 16
    offsets = torch.cat((torch.zeros(1, dtype=torch.int64), lengths)).cumsum(0)
    q, k, v = (torch.randn(rows, h, d, generator=g).to(dev) for _ in range(3))
    end = torch.full((60001, h, d, d), math.nan, device=dev)
    out = ops.linear_attention(q, k, v, SLOW, scale=0.3, new_state=end, offsets=offsets.to(dev))
    assert (end[(lengths == 0).to(dev)] == 0).all()
    for i in (0, 1, 31234, 59999, 60000):
        at = slice(int(offsets[i]), int(offsets[i + 1]))
        check_forward(*(x[at][None] for x in (q, k, v)), SLOW, 0.3, None, out[at][None], end[i:i + 1])


@pytest.mark.parametrize("most", [None, 700])
def test_a_captured_packed_call_with_other_offsets(ops, dev, most):
    """Offsets are data: a captured prompt with its state in place and its gradients, replayed on other sequences, are the eager
    calls on those -- with joined segments and with few."""
    h, dk, dv, rows, b = 2, 40, 72, 2100, 5
    q, k, v, do, _, _ = (x[0] for x in make(dev, torch.bfloat16, 1, rows, h, h, 1, h, dk, dv, seed=15))
    s0 = torch.randn(b, h, dk, dv, generator=torch.Generator().manual_seed(16)).to(dev)
    cuts = [[0, 700, 700, 1400, 1401, 2100], [0, 1, 129, 129, 800, 1500], [300, 300, 300, 300, 300, 300], [7, 650, 1206, 1334, 1400, 2093]]
    offsets, state, ds = torch.tensor(cuts[0], device=dev), s0.clone(), torch.empty_like(s0)
    more = dict(scale=0.3, offsets=offsets, max_length=most)

    def work():
        out = ops.linear_attention(q, k, v, SLOW[:h], state=state, new_state=state, **more)
        return [out, *ops.linear_attention_backward(q, k, v, SLOW[:h], do, state=s0, dnew_state=s0, dstate=ds, **more)]

    work()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = work()
    for cut in cuts[1:] + cuts:
        offsets.copy_(torch.tensor(cut))
        state.copy_(s0)
        want = [*work(), state.clone(), ds.clone()]
        state.copy_(s0)
        ds.fill_(math.nan)
        for x in got:
            x.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip([*got, state, ds], want)), cut
        end = torch.empty_like(s0)
        ops.linear_attention(q, k, v, SLOW[:h], state=s0, new_state=end, **more)
        assert torch.equal(state, end), cut
