"""Cases of two operators of a GPT's training step: queries and keys normalised per head and rotated in one pass, with its
gradient, and the update of a matrix whose momentum is made orthogonal by Newton-Schulz products.

A case is a dict of plain values with a `kind`:
  rotate       y = rotation(x * inv * gamma) of `heads` query and `kv` key heads of `dim` columns per token, inv = 1 / sqrt(mean
               x^2 + eps) of the head; the first `rot` columns rotate (halves, not neighbours), the others stay normalised
  gradient     its gradients: of queries and keys, and of the two weight vectors
  step         momentum, orthogonal factor and decayed update of `count` matrices of rows x cols, in place
  factor       the orthogonal factor alone, of matrices given in `dtype` and returned in it (`half`: products of operands
               rounded once to 16 bits; otherwise as exact as 32 bits)

`packed`: queries and keys lie in rows of a packed projection [q | k | v], and their gradients go to rows of another.
`placed`: every token has a position of its own (decoding); otherwise token t of a sequence has position t.
"""
from __future__ import annotations

import math
from types import SimpleNamespace

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
_EPS = 1e-6
_COEFFICIENTS = (3.4445, -4.7750, 2.0315)
_STEPS = 5
_LR, _MOMENTUM, _DECAY = 0.02, 0.95, 0.01


def listed():
    return [
        # one token of one sequence of the benchmark's model: the smallest call, all latency
        {"name": "rotate-token", "kind": "rotate", "tokens": 1, "seq": 1, "heads": 10, "kv": 10, "dim": 128, "rot": 128,
         "dtype": "f32", "weighted": True, "packed": False, "placed": True},
        # a token of each of 64 sequences, Qwen's 12 and 2 heads in rows of the packed projection
        {"name": "rotate-decode-64", "kind": "rotate", "tokens": 64, "seq": 1, "heads": 12, "kv": 2, "dim": 128, "rot": 128,
         "dtype": "bf16", "weighted": True, "packed": True, "placed": True},
        # prompts through odd heads of 80 columns, of which the first 40 rotate
        {"name": "rotate-ragged", "kind": "rotate", "tokens": 999, "seq": 333, "heads": 7, "kv": 3, "dim": 80, "rot": 40,
         "dtype": "f32", "weighted": False, "packed": True, "placed": False},
        # the benchmark's batch, 16 sequences of 2048
        {"name": "rotate-batch", "kind": "rotate", "tokens": 32768, "seq": 2048, "heads": 10, "kv": 10, "dim": 128, "rot": 128,
         "dtype": "f32", "weighted": True, "packed": False, "placed": False},
        # the backward pass of the Qwen-shaped layer, 4 sequences of 2048, bf16 activations
        {"name": "gradient-qwen", "kind": "gradient", "tokens": 8192, "seq": 2048, "heads": 12, "kv": 2, "dim": 128, "rot": 128,
         "dtype": "bf16", "weighted": True, "packed": True, "placed": False},
        # and that of the benchmark's batch
        {"name": "gradient-batch", "kind": "gradient", "tokens": 32768, "seq": 2048, "heads": 10, "kv": 10, "dim": 128,
         "rot": 128, "dtype": "f32", "weighted": True, "packed": False, "placed": False},
        # the two projections of the smallest model of the tests: 64 columns
        {"name": "step-tiny", "kind": "step", "count": 2, "rows": 64, "cols": 256, "dtype": "f32"},
        # a small model's projections, 6 layers of 384 columns
        {"name": "step-gpt2", "kind": "step", "count": 6, "rows": 384, "cols": 1536, "dtype": "f32"},
        # the attention projections of 5 layers of the benchmark's model
        {"name": "step-square", "kind": "step", "count": 20, "rows": 1280, "cols": 1280, "dtype": "f32"},
        # the second matrix of its feed-forward part, gradients kept as bf16
        {"name": "step-tall", "kind": "step", "count": 4, "rows": 5120, "cols": 1280, "dtype": "bf16"},
        # bf16 in and out, one 16-bit product each: what a sharded optimizer asks for before it sends the factor on
        {"name": "factor-half", "kind": "factor", "count": 4, "rows": 1536, "cols": 8960, "dtype": "bf16", "half": True},
        # odd sizes on both sides
        {"name": "factor-odd", "kind": "factor", "count": 3, "rows": 1001, "cols": 333, "dtype": "f32", "half": False},
    ]


def _log(rng, low, high):
    """An integer spread evenly over the logarithm of [low, high]."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["rotate", "gradient", "step", "step", "factor"])
    if kind in ("rotate", "gradient"):
        heads = rng.choice([1, 7, 10, 12, 16, 25, 32])
        dim = rng.choice([64, 128, 128, 256, 2 * _log(rng, 8, 128)])
        placed = kind == "rotate" and rng.random() < 0.4
        sequences = rng.choice([1, 4])
        length = _log(rng, 1, min(32768, 32768 * 20 * 128 // (2 * heads * dim)) // sequences)
        return {"kind": kind, "tokens": sequences * length, "seq": 1 if placed else length, "heads": heads,
                "kv": rng.choice([1, max(1, heads // 4), heads]), "dim": dim, "rot": rng.choice([dim, dim, dim // 4 * 2, 0]),
                "dtype": rng.choice(["f32", "bf16"]), "weighted": rng.random() < 0.7, "packed": rng.random() < 0.5, "placed": placed}
    while True:
        rows, cols = rng.choice([_log(rng, 16, 5120), _log(rng, 2, 160) * 32]), _log(rng, 16, 5120)
        count = _log(rng, 1, 32)
        if _flops(rows, cols) * count <= _flops(1280, 5120) * 4:
            break
    case = {"kind": kind, "count": count, "rows": rows, "cols": cols, "dtype": rng.choice(["f32", "bf16"])}
    if kind == "factor":
        case["half"] = case["dtype"] == "bf16" and rng.random() < 0.7
    return case


def _flops(rows, cols):
    """Of one matrix: x x^T and its square are symmetric, half of each is enough."""
    m, n = min(rows, cols), max(rows, cols)
    return _STEPS * (m * m * n + m * m * m + 2 * m * m * n)


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["kind"] in ("rotate", "gradient"):
        n = case["tokens"] * (case["heads"] + case["kv"]) * case["dim"]
        tables = min(case["tokens"], case["seq"] if not case["placed"] else 2048) * case["rot"] * 4
        return {"bytes": n * size * (2 if case["kind"] == "rotate" else 3) + tables, "flops": n * (8 if case["kind"] == "rotate" else 16)}
    n = case["count"] * case["rows"] * case["cols"]
    return {"bytes": n * (16 + size if case["kind"] == "step" else 2 * size), "flops": case["count"] * _flops(case["rows"], case["cols"])}


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dtype = _TYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(shape, device="cuda", generator=g)

    s = SimpleNamespace(case=dict(case), kind=case["kind"], calls=None)
    if s.kind in ("rotate", "gradient"):
        n, h, kv, d, rot = case["tokens"], case["heads"], case["kv"], case["dim"], case["rot"]
        s.rot, s.length = rot, 2048 if case["placed"] else case["seq"]
        # outputs of a projection: heads of different sizes, a few columns much larger than the others
        x = randn(n, h + kv * (2 if case["packed"] else 1), d) * torch.exp(randn(h + kv * (2 if case["packed"] else 1), 1))
        x[:, :, :: max(1, d // 3)] *= 8.0
        x = x.to(dtype)
        if case["packed"]:
            s.q, s.k = x[:, :h], x[:, h:h + kv]
        else:
            s.q, s.k = x[:, :h].contiguous(), x[:, h:].contiguous()
        angle = torch.arange(s.length, device="cuda", dtype=torch.float64)[:, None] * (
            1e5 ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / max(rot, 1)))
        s.cos, s.sin = angle.cos().float(), angle.sin().float()
        s.at = torch.randint(0, s.length, (n,), device="cuda", generator=g).int() if case["placed"] else None
        s.q_gamma, s.k_gamma = (1.0 + 0.3 * randn(2, d)).unbind(0) if case["weighted"] else (None, None)
        if s.kind == "gradient":
            s.dq_out, s.dk_out = (randn(n, h, d) / n).to(dtype), (randn(n, kv, d) / n).to(dtype)
            dx = torch.empty_like(x)
            s.dq, s.dk = (dx[:, :h], dx[:, h:h + kv]) if case["packed"] else (torch.empty_like(s.q), torch.empty_like(s.k))
            s.dgamma = torch.empty(2, d, device="cuda") if case["weighted"] else None
        else:
            s.q_out, s.k_out = torch.empty(n, h, d, device="cuda", dtype=dtype), torch.empty(n, kv, d, device="cuda", dtype=dtype)
        return s
    count, rows, cols = case["count"], case["rows"], case["cols"]

    def gradient():
        # a few strong directions over the noise of a batch, rows of different sizes
        r = min(8, rows, cols)
        strong = torch.matmul(randn(count, rows, r), randn(count, r, cols)) / math.sqrt(r)
        return (0.6 * strong + randn(count, rows, cols)) * torch.exp(0.3 * randn(count, rows, 1)) * 1e-3

    if s.kind == "factor":
        s.g = gradient().to(dtype)
        s.out = torch.empty_like(s.g)
    else:
        s.g = gradient().to(dtype)
        s.m = 0.7 * s.g.float() + 0.5 * gradient()
        s.p = 0.02 * randn(count, rows, cols)
        s.scale = 0.2 * math.sqrt(max(rows, cols))
    return s


# ------------------------------------------------------------------ plain forms
def _turn(x, cos, sin, rot):
    half = rot // 2
    lo, hi = x[..., :half], x[..., half:rot]
    return torch.cat([lo * cos - hi * sin, lo * sin + hi * cos, x[..., rot:]], -1)


def _tables(s):
    n = s.q.shape[0]
    at = s.at.long() if s.at is not None else torch.arange(n, device="cuda") % s.length
    return s.cos[at][:, None], s.sin[at][:, None]


def _plain_rotate(s):
    cos, sin = _tables(s)

    def one(x, gamma):
        x = x.float()
        y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + _EPS)
        return _turn(y if gamma is None else y * gamma, cos, sin, s.rot).to(s.q.dtype)
    return [one(s.q, s.q_gamma), one(s.k, s.k_gamma)]


def _plain_gradient(s):
    cos, sin = _tables(s)

    def one(x, dy, gamma):
        x = x.float()
        inv = torch.rsqrt(x.square().mean(-1, keepdim=True) + _EPS)
        y = x * inv
        dy = _turn(dy.float(), cos, -sin, s.rot)
        dgamma = (dy * y).sum((0, 1), dtype=torch.float64).float()
        if gamma is not None:
            dy = dy * gamma
        return (inv * (dy - y * (dy * y).mean(-1, keepdim=True))).to(s.q.dtype), dgamma
    dq, dq_gamma = one(s.q, s.dq_out, s.q_gamma)
    dk, dk_gamma = one(s.k, s.dk_out, s.k_gamma)
    return [dq, dk] + ([dq_gamma, dk_gamma] if s.q_gamma is not None else [])


def _plain_factor(u):
    a, b, c = _COEFFICIENTS
    norm = u.double().square().sum((-2, -1), keepdim=True).sqrt().clamp(min=1e-7)
    x = (u.double() / norm).float()
    if x.shape[-2] > x.shape[-1]:
        x = x.mT.contiguous()
    for _ in range(_STEPS):
        gram = torch.matmul(x, x.mT)
        x = a * x + torch.matmul(b * gram + c * torch.matmul(gram, gram), x)
    return x if x.shape == u.shape else x.mT


def _plain_step(s):
    g = s.g.float()
    s.m.add_(g - s.m, alpha=1.0 - _MOMENTUM)
    factor = _plain_factor(g + _MOMENTUM * (s.m - g))
    s.p.mul_(1.0 - _LR * _DECAY).sub_(factor, alpha=_LR * s.scale)
    return [s.p, s.m]


# ------------------------------------------------------------------ the framework's calls
_DEVICE = None


def _bind(s):
    """The call of a user's program on this state, on the tensors' own memory, and what it returns."""
    global _DEVICE
    import numpy as np

    import autograd_b200 as ag
    from autograd_b200 import _native as native
    from autograd_b200 import hostgraph as hg
    from autograd_b200.storage import CudaMemPointer, Storage

    if _DEVICE is None:
        _DEVICE = ag.create(0)  # on a stream of its own
    backend = _DEVICE[2]
    types = {torch.float32: np.float32, torch.bfloat16: np.uint16, torch.int32: np.int32}

    def tensor(t, shape=None):
        if t is None:
            return None
        shape = tuple(t.shape) if shape is None else shape
        h = hg.HostTensor(shape, types[t.dtype], requires_grad=False)
        h.storage = Storage(CudaMemPointer(t.data_ptr()), shape, types[t.dtype], "cuda", t.numel() * t.element_size())
        return h

    torch.cuda.synchronize()  # the inputs were made on torch's stream
    if s.kind in ("rotate", "gradient"):
        n, length = s.q.shape[0], s.case["seq"]

        def heads(t):
            return tensor(t, (n // length, length) + tuple(t.shape[1:]))

        kw = {"q_gamma": tensor(s.q_gamma), "k_gamma": tensor(s.k_gamma), "positions": tensor(s.at),
              "q_stride": s.q.stride(0), "k_stride": s.k.stride(0)}
        cos, sin = tensor(s.cos), tensor(s.sin)
        if s.kind == "rotate":
            return (backend.qk_norm_rope_forward, (heads(s.q), heads(s.k), cos, sin, heads(s.q_out), heads(s.k_out), _EPS), kw,
                    [s.q_out, s.k_out])
        out = [s.dq, s.dk]
        kw |= {"dq_stride": s.dq.stride(0), "dk_stride": s.dk.stride(0)}
        if s.dgamma is not None:
            kw |= {"dq_gamma": tensor(s.dgamma[0]), "dk_gamma": tensor(s.dgamma[1])}
            out += [s.dgamma[0], s.dgamma[1]]
            both = tensor(s.dgamma)
        args = (heads(s.dq_out), heads(s.dk_out), heads(s.q), heads(s.k), cos, sin, heads(s.dq), heads(s.dk), _EPS)

        def gradient(*args, **kw):
            # gradients of parameters accumulate, as everywhere in the framework: a step clears them first
            if s.dgamma is not None:
                backend.fill(both, 0.0)
            backend.qk_norm_rope_backward(*args, **kw)
        return gradient, args, kw, out
    if s.kind == "factor":
        precision = native.AG_CE_BF16 if s.case["half"] else native.AG_CE_3XTF32
        return (backend.orthogonalise, (tensor(s.g), tensor(s.out)),
                {"steps": _STEPS, "coefficients": _COEFFICIENTS, "precision": precision}, [s.out])
    return (backend.muon_step, (tensor(s.p), tensor(s.g), tensor(s.m), _LR),
            {"momentum": _MOMENTUM, "weight_decay": _DECAY, "scale": s.scale, "steps": _STEPS, "coefficients": _COEFFICIENTS},
            [s.p, s.m])


def run(state):
    if own:
        if state.calls is None:
            state.calls = _bind(state)
        fn, args, kw, out = state.calls
        fn(*args, **kw)
        return out
    if state.kind == "factor":
        return [_plain_factor(state.g.float()).to(state.g.dtype)]
    return {"rotate": _plain_rotate, "gradient": _plain_gradient, "step": _plain_step}[state.kind](state)


# ------------------------------------------------------------------ the definition in 64 bits
def _polynomial(g):
    """The factor of one matrix from its singular values: five times p(s) = a s + b s^3 + c s^5 on s / |s|.  Where the
    decomposition takes too long, the same polynomial of x x^T: t = a + b y + c y^2, y <- t y t, all of which commute."""
    a, b, c = _COEFFICIENTS
    if min(g.shape) ** 2 * max(g.shape) > 2e8:
        x = g.double() if g.shape[0] <= g.shape[1] else g.double().mT
        x = x / x.square().sum().sqrt().clamp(min=1e-7)
        y, one = x @ x.mT, torch.eye(x.shape[0], device=x.device, dtype=x.dtype)
        p = one
        for _ in range(_STEPS):
            t = a * one + y @ (b * one + c * y)
            p, y = t @ p, t @ y @ t
        return p @ x if g.shape[0] <= g.shape[1] else (p @ x).mT
    u, sv, vt = torch.linalg.svd(g.double(), full_matrices=False)
    sv = sv / sv.square().sum().sqrt().clamp(min=1e-7)
    for _ in range(_STEPS):
        sv = sv * (a + sv.square() * (b + c * sv.square()))
    return (u * sv) @ vt


def exact(case, seed):
    s = prepare(case, seed)
    if s.kind == "factor":
        return [torch.stack([_polynomial(g) for g in s.g])]
    if s.kind == "step":
        m = _MOMENTUM * s.m.double() + (1.0 - _MOMENTUM) * s.g.double()
        u = (1.0 - _MOMENTUM) * s.g.double() + _MOMENTUM * m
        factor = torch.stack([_polynomial(x) for x in u])
        return [s.p.double() * (1.0 - _LR * _DECAY) - _LR * s.scale * factor, m]
    n, rot = s.q.shape[0], s.rot
    place = torch.arange(n, device="cuda") % s.length if s.at is None else s.at.long()
    # the rotation as a product of complex numbers, the halves of a head being real and imaginary parts
    turn = torch.complex(s.cos.double()[place], s.sin.double()[place])[:, None]

    def rotated(y, by):
        z = torch.complex(y[..., :rot // 2], y[..., rot // 2:rot]) * by
        return torch.cat([z.real, z.imag, y[..., rot:]], -1)
    out = []
    if s.kind == "rotate":
        for x, gamma in ((s.q, s.q_gamma), (s.k, s.k_gamma)):
            x = x.double()
            norm = torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + _EPS)
            out.append(rotated(x / norm * (1.0 if gamma is None else gamma.double()), turn))
        return out
    sums = []
    for x, dy, gamma in ((s.q, s.dq_out, s.q_gamma), (s.k, s.dk_out, s.k_gamma)):
        x, w = x.double(), rotated(dy.double(), turn.conj())
        norm = torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + _EPS)
        sums.append((w * x / norm).sum((0, 1)))
        if gamma is not None:
            w = w * gamma.double()
        out.append(w / norm - x * ((w * x).sum(-1, keepdim=True) / (x.shape[-1] * norm ** 3)))
    return out + (sums if s.q_gamma is not None else [])
