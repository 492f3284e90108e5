"""Linear attention on values at the ends of their types -- infinities, NaN, the largest finite numbers -- against the 64-bit
recurrence: which outputs are not finite, and that the others are as near as ever."""
import math

import pytest
import torch

import sequence_reference as ref
from test_linear_attention_gpu import TYPES, check_backward, check_forward, make

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
