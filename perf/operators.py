"""Cases of the operators on a head's logits: log-probabilities of given tokens, and distillation from a teacher's list.

A pass is one call on logits of `rows` x `vocab`.  A case is a dict of plain values with a `kind`:
  score    log-probability of each row's token, entropy of the row, its `top` likeliest tokens
  policy   the gradient of those log-probabilities and entropies, as a policy-gradient step needs it
  distill  loss against a teacher's `top` logits and its gradient, the upstream gradient being known (a training step)
  eval     that loss alone (validation)
  grad     its gradient alone, from the row statistics that the loss left (a graph runtime's backward pass)

`rest`: the teacher gives log-probabilities, and what they leave of its mass is compared with what the student's
probabilities of the same tokens leave of its own; otherwise its logits are a distribution over the listed tokens.
Teachers list fewer than `top` tokens in one row of twenty (the other slots have id -1); one row of twenty has no token
of its own (id -1) in `score` and `policy`.
"""
from __future__ import annotations

import math
from types import SimpleNamespace

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # a token of one sequence, with five alternatives beside it: the smallest call, all latency
        {"name": "score-token", "kind": "score", "rows": 1, "vocab": 32768, "top": 5, "dtype": "f32", "temperature": 1.0,
         "masked": 0.0},
        # a token of each of 8 sequences of a Qwen-sized model, sampled at temperature 0.8, twenty alternatives
        {"name": "score-decode-8", "kind": "score", "rows": 8, "vocab": 151936, "top": 20, "dtype": "bf16",
         "temperature": 0.8, "masked": 0.0},
        # prompts through a small head with an odd vocabulary, nine of ten tokens forbidden by a grammar
        {"name": "score-ragged", "kind": "score", "rows": 333, "vocab": 5003, "top": 20, "dtype": "f32", "temperature": 0.7,
         "masked": 0.9},
        # half of the benchmark's batch scored: no alternatives, every logit read once
        {"name": "score-batch", "kind": "score", "rows": 16384, "vocab": 32768, "top": 0, "dtype": "f32", "temperature": 1.0,
         "masked": 0.0},
        # a teacher's pass over 8192 tokens: the 64 likeliest tokens of each are what a student learns from
        {"name": "score-teacher", "kind": "score", "rows": 8192, "vocab": 32768, "top": 64, "dtype": "bf16",
         "temperature": 1.0, "masked": 0.0},
        # rollouts scored by the policy that made them, a Qwen-sized vocabulary, bf16 logits
        {"name": "score-rollouts", "kind": "score", "rows": 4096, "vocab": 151936, "top": 0, "dtype": "bf16",
         "temperature": 1.0, "masked": 0.0},
        # the smallest training step of the tests: 3 sequences of 64 over 640 tokens
        {"name": "policy-tiny", "kind": "policy", "rows": 192, "vocab": 640, "dtype": "f32", "temperature": 1.0, "masked": 0.0},
        # the policy-gradient step on the rollouts above, with an entropy bonus
        {"name": "policy-rollouts", "kind": "policy", "rows": 4096, "vocab": 151936, "dtype": "bf16", "temperature": 1.0,
         "masked": 0.0},
        # validation against a teacher with long lists
        {"name": "eval-512", "kind": "eval", "rows": 512, "vocab": 32768, "top": 128, "dtype": "f32", "temperature": 1.0,
         "rest": True},
        # the backward pass of a graph over 8192 tokens, row weights
        {"name": "grad-8192", "kind": "grad", "rows": 8192, "vocab": 32768, "top": 64, "dtype": "bf16", "temperature": 1.0,
         "rest": False},
        # a student of the GPT-2 vocabulary, rows that no 16 bytes divide, teacher's log-probabilities and their rest
        {"name": "distill-gpt2", "kind": "distill", "rows": 2000, "vocab": 50257, "top": 50, "dtype": "bf16",
         "temperature": 1.0, "rest": True},
        # half of the benchmark's batch distilled in fp32 at temperature 2
        {"name": "distill-batch", "kind": "distill", "rows": 16384, "vocab": 32768, "top": 32, "dtype": "f32",
         "temperature": 2.0, "rest": False},
    ]


def _log(rng, low, high):
    """An integer spread evenly over the logarithm of [low, high]."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["score", "score", "policy", "distill", "distill", "eval", "grad"])
    vocab = rng.choice([32768, 50257, 151936, _log(rng, 640, 151936), _log(rng, 640, 151936)])
    case = {"kind": kind, "rows": _log(rng, 1, max(1, min(16384, 500_000_000 // vocab))), "vocab": vocab,
            "dtype": rng.choice(["f32", "bf16"]), "temperature": rng.choice([0.7, 1.0, 1.0, 2.0])}
    if kind == "score":
        case["top"] = rng.choice([0, 0, 1, _log(rng, 2, 128), _log(rng, 2, 128)])
    elif kind != "policy":
        case["top"] = _log(rng, 1, 128)
        case["rest"] = rng.random() < 0.5
    if kind in ("score", "policy"):
        case["masked"] = rng.choice([0.0, 0.0, 0.5, 0.9])
    return case


def work(case):
    """Logits read once, gradients written once, what a row has beside them; exp, scale and sums of each logit."""
    n, v, kind = case["rows"], case["vocab"], case["kind"]
    size = 4 if case["dtype"] == "f32" else 2
    nbytes = n * v * size * (2 if kind in ("policy", "distill", "grad") else 1)
    if kind == "score":
        nbytes += n * (12 + 8 * case["top"])
    elif kind == "policy":
        nbytes += n * 28
    else:
        nbytes += n * (8 + 8 * case["top"])
    return {"bytes": nbytes, "flops": n * v * {"score": 6, "policy": 8, "eval": 5, "grad": 5, "distill": 8}[kind]}


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    n, v, kind, dtype = case["rows"], case["vocab"], case["kind"], _TYPES[case["dtype"]]

    def rand(*shape):
        return torch.rand(shape, device="cuda", generator=g)

    # what a head puts out: a frequency for every token, and what the context adds
    x = torch.randn(n, v, device="cuda", generator=g)
    x += -1.5 * torch.log(1.0 + v * rand(v))
    s = SimpleNamespace(case=dict(case), kind=kind, temperature=case["temperature"], vocab=v, rest=bool(case.get("rest")), calls=None)
    if kind in ("score", "policy"):
        s.top = case.get("top", 0)
        if case["masked"]:
            keep = rand(n, v) >= case["masked"]
            keep[:, 7] = True
            x.masked_fill_(~keep, -math.inf)
            s.ids = torch.where(rand(n) < 0.5, 7, keep.to(torch.int8).argmax(1)).to(torch.int32)
        else:
            s.ids = (rand(n).square() * v).to(torch.int32).clamp_(max=v - 1)
        s.ids[1::20] = -1
        x = x.to(dtype)
        if kind == "score":
            s.logprob, s.entropy = torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
            s.top_ids = torch.empty(n, s.top, device="cuda", dtype=torch.int32)
            s.top_logprobs = torch.empty(n, s.top, device="cuda")
        else:
            s.dlogprob = torch.randn(n, device="cuda", generator=g) / n
            s.dentropy = torch.full((n,), -0.01 / n, device="cuda")
            p = torch.softmax(x.double() / s.temperature, 1)
            entropy = torch.special.entr(p).sum(1)
    else:
        s.top = case["top"]
        first = (rand(n) * v).long()
        slot = torch.arange(s.top, device="cuda")
        s.teacher_ids = ((first[:, None] + slot * max(1, v // s.top)) % v).to(torch.int32)
        t = torch.randn(n, s.top, device="cuda", generator=g).mul_(2.0).sort(1, descending=True).values
        # a student that agrees with its teacher in part
        x.scatter_(1, s.teacher_ids.long(), 4.0 + 0.5 * t + torch.randn(n, s.top, device="cuda", generator=g))
        x = x.to(dtype)
        if s.rest:
            t = torch.log_softmax(t, 1) + torch.log(0.7 + 0.29 * rand(n, 1))
        s.teacher_logits = t
        s.teacher_ids[::20, s.top - s.top // 3:] = -1
        s.row_scale = rand(n) / n if kind == "grad" else None
        s.dloss = torch.full((1,), 1.0, device="cuda")
        s.loss, s.row_loss = torch.empty(1, device="cuda"), torch.empty(n, device="cuda")
    if kind in ("policy", "grad"):
        # what the forward call of the same program has left: largest logit, log of the sum, entropy or log of the rest
        z = x.double() / s.temperature
        top = z.amax(1)
        left = torch.zeros_like(top)
        if kind == "policy":
            left = entropy
        elif s.rest:
            p = torch.softmax(z, 1)
            left = p.scatter(1, s.teacher_ids.long().clamp(min=0), p.new_zeros(1, 1).expand(n, s.top)).sum(1).log()
        s.stats = torch.stack([x.double().amax(1), torch.logsumexp(z, 1) - top, left, torch.zeros_like(top)], 1).float()
    else:
        s.stats = torch.empty(n, 4, device="cuda")
    s.logits = x
    if kind in ("policy", "distill", "grad"):
        s.dlogits = torch.empty_like(x)
    return s


# ------------------------------------------------------------------ plain forms
def _normalised(s):
    """Log-probabilities in 32 bits, -inf where a logit is."""
    x = s.logits.float()
    d = (x - x.amax(1, keepdim=True)) / s.temperature
    return d - torch.log(torch.exp(d).sum(1, keepdim=True))


def _entropy(lp):
    return -(torch.exp(lp) * torch.where(lp > -math.inf, lp, 0.0)).sum(1)


def _plain_score(s):
    lp = _normalised(s)
    ids = s.ids.long()
    logprob = torch.where(ids >= 0, lp.gather(1, ids.clamp(min=0)[:, None])[:, 0], 0.0)
    out = [logprob, _entropy(lp)]
    if s.top:
        # the order of the floats as integers, then the lower index first: every key is another one
        bits = (s.logits.float() + 0.0).view(torch.int32)
        order = bits ^ ((bits >> 31) & 0x7FFFFFFF)
        key = order.long() * (1 << 32) + torch.arange(s.vocab - 1, -1, -1, device=order.device)
        at = s.vocab - 1 - torch.topk(key, s.top, 1).values % (1 << 32)
        out += [at.to(torch.int32), lp.gather(1, at)]
    return out


def _plain_policy(s):
    lp = _normalised(s)
    p, finite = torch.exp(lp), torch.where(lp > -math.inf, lp, 0.0)
    entropy = -(p * finite).sum(1, keepdim=True)
    ids = s.ids.long()[:, None]
    dlp = torch.where(ids >= 0, s.dlogprob[:, None], 0.0)
    g = -p * dlp - s.dentropy[:, None] * p * (finite + entropy)
    g.scatter_add_(1, ids.clamp(min=0), dlp)
    return [(g / s.temperature).to(s.logits.dtype)]


def _plain_teacher(s):
    """(slots in use, their tokens, teacher's probabilities, its logarithms, what it leaves)"""
    used = s.teacher_ids >= 0
    t = torch.where(used, s.teacher_logits, -math.inf)
    if s.rest:
        log_q = t
    else:
        t = (t - t.amax(1, keepdim=True)) / s.temperature
        log_q = t - torch.log(torch.exp(t).sum(1, keepdim=True))
    q = torch.exp(log_q)
    left = (1.0 - q.double().sum(1)).clamp(min=0.0).float() if s.rest else torch.zeros_like(q[:, 0])
    return used, s.teacher_ids.long().clamp(min=0), q, torch.where(used, log_q, 0.0), left


def _plain_distill(s):
    lp = _normalised(s)
    used, ids, q, log_q, left = _plain_teacher(s)
    n = s.logits.shape[0]
    scale = s.row_scale if s.row_scale is not None else torch.full((n,), 1.0 / n, device=lp.device)
    p = torch.exp(lp)
    listed_ = torch.zeros_like(p)
    listed_.scatter_add_(1, ids, used.float())
    outside = torch.where(listed_ > 0, 0.0, p).sum(1)
    out = []
    if s.kind != "grad":
        row_loss = (q * (log_q - lp.gather(1, ids))).sum(1)
        if s.rest:
            row_loss = row_loss + torch.where(left > 0, left * (torch.log(left) - torch.log(outside)), 0.0)
        out += [(row_loss * scale).sum().reshape(1), row_loss]
    if s.kind != "eval":
        g = p * (q.sum(1) + left)[:, None]
        if s.rest:
            g = g - torch.where(listed_ > 0, 0.0, p) * (left / outside)[:, None]
        g.scatter_add_(1, ids, -q)
        out.append((g * (s.dloss * scale / s.temperature)[:, None]).to(s.logits.dtype))
    return out


# ------------------------------------------------------------------ the framework's calls
_DEVICE = None


def _bind(s):
    """The call of a user's program on this state, on the tensors' own memory, and what it returns."""
    global _DEVICE
    import numpy as np

    import autograd_b200 as ag
    from autograd_b200 import hostgraph as hg
    from autograd_b200.storage import CudaMemPointer, Storage

    if _DEVICE is None:
        _DEVICE = ag.create(0)  # on a stream of its own
    backend = _DEVICE[2]
    types = {torch.float32: np.float32, torch.bfloat16: np.uint16, torch.int32: np.int32}

    def tensor(t):
        if t is None:
            return None
        h = hg.HostTensor(tuple(t.shape), types[t.dtype], requires_grad=False)
        h.storage = Storage(CudaMemPointer(t.data_ptr()), tuple(t.shape), types[t.dtype], "cuda", t.numel() * t.element_size())
        return h

    w = {k: tensor(t) for k, t in vars(s).items() if t is None or isinstance(t, torch.Tensor)}
    tau, rest = s.temperature, s.rest
    torch.cuda.synchronize()  # the inputs were made on torch's stream
    if s.kind == "score":
        fn, args, kw = backend.token_logprobs_forward, (w["logits"], w["ids"], w["logprob"]), {"entropy": w["entropy"], "temperature": tau}
        out = [s.logprob, s.entropy]
        if s.top:
            kw |= {"top_ids": w["top_ids"], "top_logprobs": w["top_logprobs"]}
            out += [s.top_ids, s.top_logprobs]
    elif s.kind == "policy":
        fn = backend.token_logprobs_backward
        args, kw = (w["logits"], w["ids"], w["stats"], w["dlogprob"], w["dentropy"], w["dlogits"]), {"temperature": tau}
        out = [s.dlogits]
    elif s.kind == "eval":
        fn, args = backend.distill_forward, (w["logits"], w["teacher_ids"], w["teacher_logits"], w["row_loss"])
        kw = {"loss": w["loss"], "row_scale": w["row_scale"], "temperature": tau, "rest": rest}
        out = [s.loss, s.row_loss]
    elif s.kind == "grad":
        fn = backend.distill_backward
        args = (w["logits"], w["teacher_ids"], w["teacher_logits"], w["stats"], w["dloss"], w["dlogits"])
        kw = {"row_scale": w["row_scale"], "temperature": tau, "rest": rest}
        out = [s.dlogits]
    else:
        fn = backend.distill_forward_backward
        args = (w["logits"], w["teacher_ids"], w["teacher_logits"], w["dloss"], w["row_loss"], w["dlogits"], w["stats"])
        kw = {"loss": w["loss"], "row_scale": w["row_scale"], "temperature": tau, "rest": rest}
        out = [s.loss, s.row_loss, s.dlogits]
    return fn, args, kw, out


def run(state):
    if own:
        if state.calls is None:
            state.calls = _bind(state)
        fn, args, kw, out = state.calls
        fn(*args, **kw)
        return out
    return {"score": _plain_score, "policy": _plain_policy}.get(state.kind, _plain_distill)(state)


# ------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    n, v, kind, tau = case["rows"], case["vocab"], case["kind"], case["temperature"]
    parts = []
    weight = torch.full((n,), 1.0 / n, device="cuda", dtype=torch.float64)
    if kind not in ("score", "policy") and s.row_scale is not None:
        weight = s.row_scale.double()
    step = max(1, (1 << 27) // v)
    for r in range(0, n, step):
        rows = slice(r, min(n, r + step))
        z = s.logits[rows].double() / tau
        z = z - torch.logsumexp(z, 1, keepdim=True)
        p = z.exp()
        if kind in ("score", "policy"):
            h = torch.special.entr(p).sum(1)
            ids = s.ids[rows].long()
            has = ids >= 0
            at = torch.where(has, ids, 0)[:, None]
            if kind == "score":
                got = [torch.where(has, torch.gather(z, 1, at)[:, 0], 0.0), h]
                if s.top:
                    best = torch.sort(s.logits[rows].double(), dim=1, descending=True, stable=True).indices[:, :s.top]
                    got += [best.to(torch.int32), torch.gather(z, 1, best)]
            else:
                a = torch.where(has, s.dlogprob[rows].double(), 0.0)[:, None]
                onehot = torch.zeros_like(p).scatter_(1, at, has[:, None].double())
                dh = torch.where(p > 0, p * (torch.where(p > 0, z, 0.0) + h[:, None]), 0.0)
                got = [(a * (onehot - p) - s.dentropy[rows].double()[:, None] * dh) / tau]
        else:
            ids, t = s.teacher_ids[rows].long(), s.teacher_logits[rows].double()
            has = ids >= 0
            at = torch.where(has, ids, 0)
            t = torch.where(has, t, -math.inf)
            q = t.exp() if s.rest else torch.softmax(t / tau, 1)
            target = torch.zeros_like(p).scatter_add_(1, at, q)                    # teacher's mass on every token
            inside = torch.zeros_like(p).scatter_add_(1, at, has.double()) > 0
            log_q = torch.where(has, q.log(), 0.0)
            loss = (q * (log_q - torch.gather(z, 1, at))).sum(1)
            g = p * q.sum(1, keepdim=True) - target
            if s.rest:
                left = (1.0 - q.sum(1)).clamp(min=0.0)
                out = torch.where(inside, 0.0, p).sum(1)
                loss = loss + torch.where(left > 0, left * (left.log() - out.log()), 0.0)
                g = g + left[:, None] * (p - torch.where(inside, 0.0, p) / out[:, None])
            got = [loss] if kind != "grad" else []
            if kind != "eval":
                got.append(g * (s.dloss.double() * weight[rows] / tau)[:, None])
        parts.append([u.cpu() if kind == "score" else u for u in got])
    out = [torch.cat(u) for u in zip(*parts)]
    if kind in ("eval", "distill"):
        out = [(out[0] * weight).sum().reshape(1)] + out
    return out
