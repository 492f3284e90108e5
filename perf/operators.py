"""The sequence-layer operators measured: rotary positions and linear attention with a decay for each head.

    rotary      y = gain * (pairs of x rotated by pos * f_i), or back (the gradient)
    prompt      o_t = scale * q_t S_t,  S_t = decay * S_{t-1} + k_t v_t^T, over whole sequences, with the state after them
    backward    the gradients of q, k, v and of the state before, from those of o and of the state after
    step        one token for each row of a serving batch, on slots of a pool of states

Everything is [batch, time, head, dim]; a packed batch is [rows, head, dim] with offsets.  `run` computes the plain
form in fp32 (angles and powers of the decay in 64 bits), or calls the framework where `own` is true.
"""
import math
import random

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


def _rotary(name, dtype, batch, n, heads, dim, rot, layout, inverse=False, scaled=False, positions=False):
    return {"name": name, "op": "rotary", "dtype": dtype, "batch": batch, "n": n, "heads": heads, "dim": dim, "rot": rot,
            "layout": layout, "inverse": inverse, "scaled": scaled, "positions": positions}


def _mixer(name, op, dtype, batch, n, heads, heads_q, heads_k, heads_v, dim_k, dim_v, fast=False, state=False, packed=False):
    return {"name": name, "op": op, "dtype": dtype, "batch": batch, "n": n, "heads": heads, "heads_q": heads_q,
            "heads_k": heads_k, "heads_v": heads_v, "dim_k": dim_k, "dim_v": dim_v, "fast": fast, "state": state,
            "packed": packed}


def listed():
    return [
        # queries and keys of one serving step, every row at a far position of its own: latency
        _rotary("rotary_step", "bf16", 64, 1, 20, 128, 128, "half", positions=True),
        # queries of a long prompt, half of each head rotated, frequencies stretched for a longer context
        _rotary("rotary_prompt", "bf16", 1, 16384, 32, 128, 64, "half", scaled=True),
        # a training batch: the largest tensor
        _rotary("rotary_train", "bf16", 8, 8192, 40, 128, 128, "interleaved"),
        # the way back of an odd-sized fp32 batch
        _rotary("rotary_back", "fp32", 3, 1001, 6, 80, 40, "interleaved", inverse=True),
        # one token for one listener: the smallest call
        _mixer("step_one", "step", "bf16", 1, 1, 8, 8, 8, 8, 64, 64),
        # one token for each row of a serving batch
        _mixer("step_batch", "step", "bf16", 64, 1, 16, 16, 4, 16, 128, 128),
        # a short question of odd length
        _mixer("prompt_short", "prompt", "fp16", 1, 77, 8, 8, 8, 8, 64, 64, fast=True),
        # one long document: few heads, one sequence, so the time axis has to be split
        _mixer("prompt_long", "prompt", "bf16", 1, 32768, 16, 16, 16, 16, 128, 128),
        # prompts of very different lengths in one packed batch, continued from earlier states
        _mixer("prompt_packed", "prompt", "bf16", 16, 20011, 16, 16, 4, 16, 128, 128, state=True, packed=True),
        # fp32 all through, wide values
        _mixer("prompt_fp32", "prompt", "fp32", 2, 2048, 8, 8, 8, 8, 64, 128, fast=True),
        # a training step's way back
        _mixer("backward_train", "backward", "bf16", 4, 4096, 16, 16, 16, 16, 128, 128),
        # odd dimensions, queries and keys shared between heads, a state carried in and out
        _mixer("backward_shared", "backward", "bf16", 2, 1000, 12, 4, 4, 12, 48, 80, fast=True, state=True),
    ]


def _spread(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


def draw(rng):
    op = rng.choice(("rotary", "prompt", "prompt", "backward", "step"))
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    if op == "rotary":
        batch = _spread(rng, 1, 64)
        n = _spread(rng, 1, 65536 // batch)
        dim = rng.choice((32, 64, 80, 96, 128, 192, 256))
        heads = _spread(rng, 1, max(1, min(64, 300000000 // (batch * n * dim))))
        case = _rotary("", dtype, batch, n, heads, dim, rng.choice((dim, dim // 2, dim // 2 // 2 * 2)),
                       rng.choice(("half", "interleaved")), rng.random() < 0.3, rng.random() < 0.3, rng.random() < 0.5)
    else:
        dim_k = rng.choice((16, 32, 48, 64, 72, 96, 128, 128, 192, 256, rng.randrange(1, 257)))
        dim_v = rng.choice((16, 32, 48, 64, 80, 96, 128, 128, 192, 256, rng.randrange(1, 257)))
        share = [rng.choice((1, 1, 1, 2, 4)) for _ in range(3)]
        base = rng.choice((4, 8, 12, 16)) if max(share) > 1 else _spread(rng, 1, 32)
        heads = [base] + [base // s for s in share]
        if op == "step":
            batch, n = _spread(rng, 1, 128), 1
            batch = max(1, min(batch, 18000000 // (base * dim_k * dim_v)))
        else:
            most = 8000000000 // (base * dim_k * dim_v)
            batch = _spread(rng, 1, 32)
            n = _spread(rng, 1, max(1, min(32768, (most if op == "prompt" else most // 4)) // batch))
        packed = op == "prompt" and batch > 1 and rng.random() < 0.5
        case = _mixer("", op, dtype, batch, n * batch if packed else n, *heads, dim_k, dim_v, rng.random() < 0.5,
                      rng.random() < 0.5, packed)
    del case["name"]
    return case


def _lengths(case):
    """The lengths of a packed batch's sequences: very different ones, a single token and an empty one among them."""
    rng = random.Random(case["n"] * 31 + case["batch"])
    weights = [math.exp(rng.uniform(0.0, 4.0)) for _ in range(case["batch"])]
    total, out = case["n"], []
    for w in weights:
        out.append(int(total * w / sum(weights)))
    if case["batch"] > 3:
        out[1], out[2] = 0, 1
    big = out.index(max(out))
    out[big] += total - sum(out)
    return out


def _log_decay(case):
    """ln of each head's decay: 1 - decay spread evenly in its logarithm, from 1/32 to 1/512 (or from 1/2 to 1/64)."""
    h = case["heads"]
    first, last = (0.5, 1 / 64) if case["fast"] else (1 / 32, 1 / 512)
    return [math.log1p(-math.exp(math.log(first) + (math.log(last) - math.log(first)) * i / max(1, h - 1))) for i in range(h)]


def _frequencies(case):
    """Radians a position for each pair; `scaled`: slowed where fewer than 1 to 32 turns fit 4096 positions, by up to 8."""
    r = case["rot"]
    f = [10000.0 ** (-2.0 * i / r) for i in range(r // 2)]
    if case["scaled"]:
        for i, x in enumerate(f):
            turns = 4096 * x / (2 * math.pi)
            keep = min(1.0, max(0.0, (turns - 1.0) / 31.0))
            f[i] = x * (keep + (1.0 - keep) / 8.0)
    return f


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(dev).manual_seed(seed)
    t = _TYPES[case["dtype"]]

    def normal(*shape, dtype=t, by=1.0):
        x = torch.empty(shape, dtype=dtype, device=dev)
        return x.normal_(0.0, by, generator=gen)

    st = {"case": case}
    if case["op"] == "rotary":
        st["x"] = normal(case["batch"], case["n"], case["heads"], case["dim"])
        st["inv_freq"] = _frequencies(case)
        st["gain"] = 0.1 * math.log(8.0) + 1.0 if case["scaled"] else 1.0
        st["positions"] = None
        if case["positions"]:
            start = torch.randint(0, 1 << 20, (case["batch"], 1), generator=gen, device=dev)
            st["positions"] = start + torch.arange(case["n"], device=dev)
        return st
    b, n, h, dk, dv = (case[k] for k in ("batch", "n", "heads", "dim_k", "dim_v"))
    lead = (b,) if case["op"] == "step" else (n,) if case["packed"] else (b, n)
    st["q"] = normal(*lead, case["heads_q"], dk)
    st["k"] = normal(*lead, case["heads_k"], dk)
    st["v"] = normal(*lead, case["heads_v"], dv)
    st["log_decay"] = _log_decay(case)
    st["scale"] = dk ** -0.5
    if case["op"] == "step":
        slots = b + b // 4
        st["slots"] = torch.randperm(slots, generator=gen, device=dev)[:b]
        st["state"] = normal(slots, h, dk, dv, dtype=torch.float32, by=3.0)
        return st
    st["state"] = normal(b, h, dk, dv, dtype=torch.float32, by=3.0) if case["state"] else None
    if case["packed"]:
        lengths = _lengths(case)
        st["lengths"] = torch.tensor(lengths, device=dev)
        st["offsets"] = torch.tensor([0] + lengths, device=dev).cumsum(0)
        st["longest"] = max(lengths)
    if case["op"] == "backward":
        st["dout"] = normal(b, n, h, dv)
        st["dnew_state"] = normal(b, h, dk, dv, dtype=torch.float32, by=0.1) if case["state"] else None
    return st


# ---- plain forms -----------------------------------------------------------------------------------------------------


def _plain_rotary(st):
    case, x = st["case"], st["x"]
    n, r = case["n"], case["rot"]
    pos = st["positions"] if st["positions"] is not None else torch.arange(n, device=x.device)[None]
    angle = pos.double()[..., None] * torch.tensor(st["inv_freq"], dtype=torch.float64, device=x.device)
    c, s = torch.cos(angle).float()[:, :, None], torch.sin(angle).float()[:, :, None]
    if case["inverse"]:
        s = -s
    f = x.float()
    head, tail = f[..., :r], f[..., r:]
    if case["layout"] == "half":
        a, b = head[..., : r // 2], head[..., r // 2:]
        turned = torch.cat(((a * c - b * s) * st["gain"], (a * s + b * c) * st["gain"]), -1)
    else:
        a, b = head[..., 0::2], head[..., 1::2]
        turned = torch.stack(((a * c - b * s) * st["gain"], (a * s + b * c) * st["gain"]), -1).flatten(-2)
    return torch.cat((turned, tail), -1).to(x.dtype)


def _heads(x, h):
    """[batch, time, heads, dim] -> fp32 [batch, h, time, dim], shared heads repeated."""
    return x.float().repeat_interleave(h // x.shape[2], 2).transpose(1, 2).contiguous()


def _plain_mix(q, k, v, log_decay, scale_read, scale_write, state, late):
    """[batch, head, time, dim] fp32: outputs of every token, in chunks.  late = 1: the state decays before it is written to."""
    b, h, n, dk = q.shape
    dv = v.shape[-1]
    size = max(1, min(128, n))
    m = -(-n // size)
    pad = m * size - n
    if pad:
        q, k, v = (torch.nn.functional.pad(x, (0, 0, 0, pad)) for x in (q, k, v))
    q, k, v = q.view(b, h, m, size, dk), k.view(b, h, m, size, dk), v.view(b, h, m, size, dv)
    g = torch.tensor(log_decay, dtype=torch.float64, device=q.device)[:, None]
    i = torch.arange(size, device=q.device, dtype=torch.float64)
    gap = i[:, None] - i[None]
    weight = torch.where(gap >= 0, torch.exp(g[:, :, None] * gap.clamp(min=0)), torch.zeros_like(gap)).float()
    read = torch.exp(g * (i + 1 - late)).float()[:, None, :, None]
    write = torch.exp(g * (size - 1 - i + late)).float()[:, None, :, None]
    inside = (q @ k.transpose(-1, -2)) * (weight[:, None] * (scale_read * scale_write)) @ v
    writes = (k * (write * scale_write)).transpose(-1, -2) @ v
    c = torch.arange(m, device=q.device, dtype=torch.float64)
    before = c[:, None] - c[None] - 1
    carry = torch.where(before >= 0, torch.exp(g[:, :, None] * size * before.clamp(min=0)), torch.zeros_like(before)).float()
    starts = (carry @ writes.view(b, h, m, dk * dv)).view(b, h, m, dk, dv)
    if state is not None:
        starts = starts + state[:, :, None] * torch.exp(g * size * c).float()[:, :, None, None]
    out = inside + (q * (read * scale_read)) @ starts
    return out.view(b, h, m * size, dv)[:, :, :n]


def _plain_end(k, v, log_decay, lengths, state, late):
    """The state after each sequence: [batch, head, dk, dv]."""
    n = k.shape[2]
    g = torch.tensor(log_decay, dtype=torch.float64, device=k.device)[None, :, None]
    left = lengths.double()[:, None, None] - 1 - torch.arange(n, device=k.device, dtype=torch.float64)
    weight = torch.where(left >= 0, torch.exp(g * (left.clamp(min=0) + late)), torch.zeros_like(left)).float()
    end = (k * weight[..., None]).transpose(-1, -2) @ v
    if state is not None:
        end = end + state * torch.exp(g * lengths.double()[:, None, None]).float()[..., None]
    return end


def _plain_prompt(st):
    case = st["case"]
    h, q, k, v = case["heads"], st["q"], st["k"], st["v"]
    if case["packed"]:
        t = torch.arange(st["longest"], device=q.device)
        there = t[None] < st["lengths"][:, None]
        row = torch.where(there, st["offsets"][:-1, None] + t[None], torch.full_like(t, case["n"])[None])
        q, k, v = (torch.cat((x, torch.zeros_like(x[:1])))[row] for x in (q, k, v))
        lengths = st["lengths"]
    else:
        lengths = torch.full((case["batch"],), case["n"], device=q.device)
    fq, fk, fv = (_heads(x, h) for x in (q, k, v))
    out = _plain_mix(fq, fk, fv, st["log_decay"], st["scale"], 1.0, st["state"], 0).transpose(1, 2).to(q.dtype)
    end = _plain_end(fk, fv, st["log_decay"], lengths, st["state"], 0)
    return [out[there] if case["packed"] else out.contiguous(), end]


def _plain_shared(x, heads, t):
    """[batch, h, time, dim] -> [batch, time, heads, dim], the gradients of a shared head added up."""
    b, h, n, d = x.shape
    return x.view(b, heads, h // heads, n, d).sum(2).transpose(1, 2).to(t).contiguous()


def _plain_backward(st):
    case, t = st["case"], st["q"].dtype
    h, scale, log_decay = case["heads"], st["scale"], st["log_decay"]
    q, k, v, do = (_heads(st[x], h) for x in ("q", "k", "v", "dout"))
    s0, d1 = st["state"], st["dnew_state"]
    dq = _plain_mix(do, v, k, log_decay, scale, 1.0, None if s0 is None else s0.transpose(-1, -2), 0)
    rq, rk, rv, rdo = (x.flip(2) for x in (q, k, v, do))
    dk = _plain_mix(rv, rdo, rq, log_decay, 1.0, scale, None if d1 is None else d1.transpose(-1, -2), 1).flip(2)
    dv = _plain_mix(rk, rq, rdo, log_decay, 1.0, scale, d1, 1).flip(2)
    out = [_plain_shared(dq, case["heads_q"], t), _plain_shared(dk, case["heads_k"], t), _plain_shared(dv, case["heads_v"], t)]
    if s0 is not None:
        lengths = torch.full((case["batch"],), case["n"], device=q.device)
        out.append(_plain_end(rq * scale, rdo, log_decay, lengths, d1, 1))
    return out


def _plain_step(st):
    case, pool = st["case"], st["state"]
    h = case["heads"]
    q, k, v = (st[x].float().repeat_interleave(h // st[x].shape[1], 1) for x in ("q", "k", "v"))
    decay = torch.exp(torch.tensor(st["log_decay"], dtype=torch.float64, device=q.device)).float()[:, None, None]
    s = pool[st["slots"]] * decay + k[..., None] * v[..., None, :]
    pool[st["slots"]] = s
    out = (q[:, :, None] @ s)[:, :, 0] * st["scale"]
    return [out.to(st["q"].dtype), pool]


# ---- one pass --------------------------------------------------------------------------------------------------------


def run(st):
    op = st["case"]["op"]
    if not own:
        return {"rotary": _plain_rotary, "prompt": _plain_prompt, "backward": _plain_backward, "step": _plain_step}[op](st)
    from dsp_amd import ops

    case = st["case"]
    if op == "rotary":
        return ops.rotary(st["x"], st["inv_freq"], positions=st["positions"], layout=case["layout"],
                          inverse=case["inverse"], gain=st["gain"])
    if op == "step":
        out = ops.linear_attention_step(st["q"], st["k"], st["v"], st["log_decay"], st["state"], scale=st["scale"],
                                        slots=st["slots"])
        return [out, st["state"]]
    packed = {"offsets": st["offsets"], "max_length": st["longest"]} if case["packed"] else {}
    q, k, v = st["q"], st["k"], st["v"]
    end = torch.empty((case["batch"], case["heads"], case["dim_k"], case["dim_v"]), dtype=torch.float32, device=q.device)
    if op == "prompt":
        out = ops.linear_attention(q, k, v, st["log_decay"], scale=st["scale"], state=st["state"], new_state=end, **packed)
        return [out, end]
    if st["state"] is None:
        return list(ops.linear_attention_backward(q, k, v, st["log_decay"], st["dout"], scale=st["scale"]))
    return [*ops.linear_attention_backward(q, k, v, st["log_decay"], st["dout"], scale=st["scale"], state=st["state"],
                                           dnew_state=st["dnew_state"], dstate=end), end]


def work(case):
    size = _BYTES[case["dtype"]]
    if case["op"] == "rotary":
        rows = case["batch"] * case["n"]
        count = rows * case["heads"] * case["dim"]
        return {"bytes": 2 * size * count + (8 * rows if case["positions"] else 0),
                "flops": 3 * rows * case["heads"] * case["rot"]}
    b, n, h, dk, dv = (case[k] for k in ("batch", "n", "heads", "dim_k", "dim_v"))
    rows = n if case["packed"] else b * n
    ins = rows * ((case["heads_q"] + case["heads_k"]) * dk + case["heads_v"] * dv)
    outs = rows * h * dv
    pairs = [x * (x + 1) // 2 for x in (_lengths(case) if case["packed"] else [n] * b)]
    if case["op"] == "step":
        return {"bytes": size * (ins + outs) + 8 * b * h * dk * dv + 8 * b, "flops": 5 * b * h * dk * dv}
    each = 4 * b * h * dk * dv
    if case["op"] == "prompt":  # recurrent, or over all pairs where the sequences are short
        flops = h * min(4 * rows * dk * dv, 2 * sum(pairs) * (dk + dv) + 2 * rows * dk * dv)
        return {"bytes": size * (ins + outs) + each * (2 if case["state"] else 1), "flops": flops}
    flops = h * min(10 * rows * dk * dv, 4 * sum(pairs) * (dk + dv) + 2 * sum(pairs) * dk)
    return {"bytes": size * (2 * ins + outs) + (3 * each if case["state"] else 0), "flops": flops}


# ---- from the definitions, in 64 bits ----------------------------------------------------------------------------------


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "rotary":
        x = st["x"].double()
        dev, r = x.device, case["rot"]
        pos = torch.arange(case["n"], device=dev).expand(case["batch"], -1) if st["positions"] is None else st["positions"]
        out = x.clone()
        turn = -1.0 if case["inverse"] else 1.0
        for i, f in enumerate(st["inv_freq"]):
            j, l = (i, i + r // 2) if case["layout"] == "half" else (2 * i, 2 * i + 1)
            z = torch.polar(torch.full_like(pos, st["gain"], dtype=torch.float64), turn * f * pos.double())[:, :, None]
            y = torch.complex(x[..., j], x[..., l]) * z
            out[..., j], out[..., l] = y.real, y.imag
        return out
    h = case["heads"]
    axis = 1 if case["op"] == "step" or case["packed"] else 2
    q, k, v = (st[x].double().repeat_interleave(h // st[x].shape[axis], axis) for x in ("q", "k", "v"))
    decay = torch.exp(torch.tensor(st["log_decay"], dtype=torch.float64, device=q.device))[:, None, None]
    if case["op"] == "step":
        pool = st["state"].double()
        out = torch.zeros(case["batch"], h, case["dim_v"], dtype=torch.float64, device=q.device)
        for row, slot in enumerate(st["slots"].tolist()):
            pool[slot] = pool[slot] * decay + k[row, :, :, None] * v[row, :, None, :]
            out[row] = st["scale"] * torch.einsum("hd,hdn->hn", q[row], pool[slot])
        return [out, pool]
    dev = q.device
    if case["op"] == "prompt":
        shape = (case["batch"], h, case["dim_k"], case["dim_v"])
        s = torch.zeros(shape, dtype=torch.float64, device=dev) if st["state"] is None else st["state"].double()
        if case["packed"]:  # token t of every sequence that is so long, together
            offsets, lengths = st["offsets"].tolist(), st["lengths"].tolist()
            order = sorted(range(case["batch"]), key=lambda i: -lengths[i])
            start = torch.tensor([offsets[i] for i in order], device=dev)
            s = s[order].clone()
            out = torch.zeros(case["n"], h, case["dim_v"], dtype=torch.float64, device=dev)
            live = case["batch"]
            for t in range(lengths[order[0]]):
                while lengths[order[live - 1]] <= t:
                    live -= 1
                at = start[:live] + t
                s[:live] = s[:live] * decay + k[at][..., None] * v[at][..., None, :]
                out[at] = st["scale"] * torch.einsum("bhd,bhdn->bhn", q[at], s[:live])
            end = torch.empty_like(s)
            end[order] = s
            return [out, end]
        out = torch.empty(case["batch"], case["n"], h, case["dim_v"], dtype=torch.float64, device=dev)
        for t in range(case["n"]):
            s = s * decay + k[:, t, :, :, None] * v[:, t, :, None, :]
            out[:, t] = st["scale"] * torch.einsum("bhd,bhdn->bhn", q[:, t], s)
        return [out, s]
    do = st["dout"].double()
    shape = (case["batch"], h, case["dim_k"], case["dim_v"])
    s = torch.zeros(shape, dtype=torch.float64, device=dev) if st["state"] is None else st["state"].double()
    d = torch.zeros(shape, dtype=torch.float64, device=dev) if st["state"] is None else st["dnew_state"].double()
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    for t in range(case["n"]):
        s = s * decay + k[:, t, :, :, None] * v[:, t, :, None, :]
        dq[:, t] = st["scale"] * torch.einsum("bhdn,bhn->bhd", s, do[:, t])
    for t in reversed(range(case["n"])):
        d = d + st["scale"] * q[:, t, :, :, None] * do[:, t, :, None, :]
        dk[:, t] = torch.einsum("bhdn,bhn->bhd", d, v[:, t])
        dv[:, t] = torch.einsum("bhdn,bhd->bhn", d, k[:, t])
        d = d * decay
    out = []
    for x, heads in ((dq, case["heads_q"]), (dk, case["heads_k"]), (dv, case["heads_v"])):
        out.append(x.unflatten(2, (heads, h // heads)).sum(3))
    return out + ([d] if st["state"] is not None else [])
