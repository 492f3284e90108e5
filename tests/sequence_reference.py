"""The sequence-layer operators in 64 bits on the CPU, token after token from their definitions, and how far a result may be.

Every output is a sum of products with weights >= 0 (decays), so the same loops on absolute values give A, the sum of the
absolute terms, that rounding errors are relative to:

    fp32 arithmetic     every term goes through at most dim + n sums and a dozen products and powers: (2 (dim + n) + 64) 2^-24 A
    bf16 operands       each pair (i, j) goes through P or through S, rounded once: eps/2 of its share of A  (bf16 inputs only;
                        fp16 and fp32 inputs are multiplied in fp32)
    the result          rounded once: eps/2 |result|
"""
import torch


def heads_of(x, h):
    """[batch, n, heads, dim] -> float64 [batch, n, h, dim], shared heads repeated."""
    return x.detach().cpu().double().repeat_interleave(h // x.shape[2], 2)


def forward(q, k, v, log_decay, scale, state):
    """q, k, v float64 [batch, n, h, dim] -> (o, state after)."""
    w = torch.exp(torch.as_tensor(log_decay, dtype=torch.float64))[:, None, None]
    b, n, h, dk = q.shape
    s = torch.zeros(b, h, dk, v.shape[-1], dtype=torch.float64) if state is None else state.detach().cpu().double()
    out = torch.zeros(b, n, h, v.shape[-1], dtype=torch.float64)
    for t in range(n):
        s = s * w + k[:, t, :, :, None] * v[:, t, :, None, :]
        out[:, t] = scale * (q[:, t, :, :, None] * s).sum(2)
    return out, s


def backward(q, k, v, log_decay, scale, state, dout, dend):
    """-> dq, dk, dv (for all h heads), gradient of the state before."""
    w = torch.exp(torch.as_tensor(log_decay, dtype=torch.float64))[:, None, None]
    b, n, h, dk_ = q.shape
    shape = (b, h, dk_, v.shape[-1])
    s = torch.zeros(shape, dtype=torch.float64) if state is None else state.detach().cpu().double()
    d = torch.zeros(shape, dtype=torch.float64) if dend is None else dend.detach().cpu().double()
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for t in range(n):
        s = s * w + k[:, t, :, :, None] * v[:, t, :, None, :]
        dq[:, t] = scale * (s * dout[:, t, :, None, :]).sum(3)
    for t in reversed(range(n)):
        d = d + scale * q[:, t, :, :, None] * dout[:, t, :, None, :]
        dk[:, t] = (d * v[:, t, :, None, :]).sum(3)
        dv[:, t] = (d * k[:, t, :, :, None]).sum(2)
        d = d * w
    return dq, dk, dv, d


def shared(x, heads):
    """Gradients of all h heads [batch, n, h, dim] -> of the `heads` that they share."""
    return x.unflatten(2, (heads, x.shape[2] // heads)).sum(3)


def near(got, want, total, terms, dtype, operands=True):
    """Every element of `got` within the bound above; `total` = A, `terms` = dim + n."""
    got = got.detach().cpu().double()
    assert got.shape == want.shape, (got.shape, want.shape)
    assert torch.isfinite(got).all()
    half = torch.finfo(dtype).eps / 2
    bound = half * want.abs() * 1.01 + (2 * terms + 64) * 2.0 ** -24 * total
    if dtype == torch.bfloat16 and operands:
        bound = bound + half * 1.01 * total
    if dtype == torch.float16:  # below 2^-14 steps are 2^-24: half of one
        bound = bound + 2.0 ** -25
    over = (got - want).abs() - bound
    assert (over <= 0).all(), f"off by up to {over.max():.3g} more than the bound ({(over > 0).sum()} of {over.numel()})"
