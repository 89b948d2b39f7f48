"""Cases for the operators that learn from a language model's logits.

Four operators, all over rows of ``V`` logits (a vocabulary):

- ``topk``        a teacher's ``k`` largest logits with their places and the row's
                  logsumexp: what a station sends to the others in place of weights;
- ``distill``     the divergence of a student's row from such a record, and its
                  gradient by the student's logits;
- ``preference``  the paired log-ratio loss of chosen against rejected answers, and
                  its gradient by both answers' logits;
- ``policy``      the clipped policy loss with a KL term, and its gradient.

``own`` says whether ``run`` calls the framework or the plain forms below it.
"""
import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}

# The largest logits of one call: eight sequences of 256 over a vocabulary of
# 128256 in bf16, as one local step of the decoder configuration makes them.
_MOST_BYTES = 2048 * 128256 * 2


def listed():
    return [
        # the next token of one request, encoder vocabulary: latency alone
        {"name": "topk one row", "op": "topk", "rows": 1, "vocab": 30522, "k": 8, "dtype": "bf16"},
        # a teacher's pass over the benchmark's decoder batch, two sequences of 512
        {"name": "topk decoder batch", "op": "topk", "rows": 1024, "vocab": 128256, "k": 64, "dtype": "bf16"},
        # an odd vocabulary, rows that start anywhere, full precision
        {"name": "topk odd fp32", "op": "topk", "rows": 389, "vocab": 50021, "k": 33, "dtype": "fp32"},
        # one short sentence of the public set, softened
        {"name": "distill sentence", "op": "distill", "batch": 1, "seq": 15, "vocab": 30522, "k": 8,
         "dtype": "fp32", "temperature": 2.0, "tail": False, "pad": 0.0},
        # the encoder's batch of eight at 512, ragged, with the mass outside the record
        {"name": "distill encoder fp16", "op": "distill", "batch": 8, "seq": 512, "vocab": 30522, "k": 32,
         "dtype": "fp16", "temperature": 1.0, "tail": True, "pad": 0.4},
        # the decoder's vocabulary
        {"name": "distill decoder", "op": "distill", "batch": 8, "seq": 256, "vocab": 128256, "k": 64,
         "dtype": "bf16", "temperature": 2.0, "tail": True, "pad": 0.0},
        # one pair of short answers
        {"name": "preference pair", "op": "preference", "pairs": 1, "seq": 23, "vocab": 30522,
         "dtype": "bf16", "smoothing": 0.0, "sliced": False, "pad": 0.0},
        # logits that are a slice of one token more, ragged answers
        {"name": "preference ragged fp16", "op": "preference", "pairs": 3, "seq": 211, "vocab": 32003,
         "dtype": "fp16", "smoothing": 0.1, "sliced": True, "pad": 0.5},
        # four pairs at 256 tokens, the decoder's vocabulary
        {"name": "preference decoder", "op": "preference", "pairs": 4, "seq": 256, "vocab": 128256,
         "dtype": "bf16", "smoothing": 0.0, "sliced": False, "pad": 0.2},
        # one short rollout
        {"name": "policy rollout", "op": "policy", "batch": 1, "seq": 9, "vocab": 30522,
         "dtype": "bf16", "kl": 0.05, "pad": 0.0},
        # no reference model, full precision
        {"name": "policy encoder fp32", "op": "policy", "batch": 5, "seq": 333, "vocab": 30522,
         "dtype": "fp32", "kl": 0.0, "pad": 0.3},
        # eight rollouts of 256, the decoder's vocabulary
        {"name": "policy decoder", "op": "policy", "batch": 8, "seq": 256, "vocab": 128256,
         "dtype": "bf16", "kl": 0.05, "pad": 0.0},
    ]


def _log_between(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["topk", "distill", "preference", "policy"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    vocab = _log_between(rng, 600, 131072)
    size = 4 if dtype == "fp32" else 2
    rows = _log_between(rng, 1, max(1, min(8192, _MOST_BYTES // (size * vocab))))
    case = {"op": op, "vocab": vocab, "dtype": dtype}
    if op == "topk":
        case.update(rows=rows, k=_log_between(rng, 1, 128))
        return case
    pad = rng.choice([0.0, round(rng.uniform(0.05, 0.6), 2)])
    if op == "preference":
        pairs = max(1, min(_log_between(rng, 1, 16), rows // 2))
        case.update(pairs=pairs, seq=max(1, rows // (2 * pairs)), pad=pad,
                    smoothing=rng.choice([0.0, 0.05, 0.2]), sliced=rng.random() < 0.5)
        return case
    batch = min(_log_between(rng, 1, 32), rows)
    case.update(batch=batch, seq=rows // batch, pad=pad)
    if op == "distill":
        case.update(k=_log_between(rng, 1, 128), temperature=rng.choice([1.0, 1.5, 2.0, 4.0]),
                    tail=rng.random() < 0.5)
    else:
        case.update(kl=rng.choice([0.0, 0.02, 0.1]))
    return case


def _shape(case):
    """(sequences, tokens) of a case."""
    if case["op"] == "topk":
        return 1, case["rows"]
    if case["op"] == "preference":
        return 2 * case["pairs"], case["seq"]
    return case["batch"], case["seq"]


def _lengths(case):
    """Tokens of each sequence that count: from all of them down to 1 - pad."""
    batch, seq = _shape(case)
    pad = case.get("pad", 0.0)
    return [max(1, seq - int(pad * seq * i / batch)) for i in range(batch)]


# --------------------------------------------------------------------- inputs
def _row_logsumexp(x, t=1.0):
    """In float32, a slab of rows at a time: an input is made with it."""
    return torch.cat([(part.float() / t).logsumexp(-1) for part in x.split(256)])


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dtype, V = _TYPES[case["dtype"]], case["vocab"]
    batch, seq = _shape(case)
    R = batch * seq
    # fp16 training scales its loss, so that small gradients stay above the type's least
    scale = 4096.0 if case["dtype"] == "fp16" else 1.0
    state = {"case": case, "op": case["op"], "scale": torch.full((), scale, device=dev)}
    extra = 1 if case.get("sliced") else 0
    x = torch.randn(batch * (seq + extra), V, generator=g, device=dev, dtype=dtype).mul_(2.5)
    x = x.view(batch, seq + extra, V)

    if case["op"] == "topk":
        state["logits"] = x.view(R, V)
        return state

    # a trained model holds most of its rows for one token: every other row is sharp
    targets = torch.randint(0, V, (batch, seq), generator=g, device=dev)
    x = x[:, :seq]
    lift = torch.where(torch.rand(batch, seq, generator=g, device=dev) < 0.5, 9.0, 0.0)
    x.scatter_add_(-1, targets[..., None], lift[..., None].to(dtype))
    state["logits"] = x.detach().requires_grad_(True)
    keep = torch.arange(seq, device=dev)[None] < torch.tensor(_lengths(case), device=dev)[:, None]

    if case["op"] == "distill":
        t, k = case["temperature"], case["k"]
        teacher = x.reshape(R, V) + torch.randn(R, V, generator=g, device=dev, dtype=dtype)
        values, indices = teacher.topk(k, dim=-1)
        state.update(values=values.view(batch, seq, k), indices=indices.view(batch, seq, k), mask=keep)
        if case["tail"]:
            state["lse"] = _row_logsumexp(teacher, t).view(batch, seq)
        return state

    rows = x.detach().reshape(R, V)
    logps = rows.gather(-1, targets.view(R, 1))[:, 0].float() - _row_logsumexp(rows)
    logps = logps.view(batch, seq)
    if case["op"] == "preference":
        state["targets"] = torch.where(keep, targets, -100)
        drift = torch.randn(batch, generator=g, device=dev) * 8.0
        state["ref_logps"] = torch.where(keep, logps, 0.0).double().sum(-1).float() + drift
        return state

    # the policy has moved a little since the rollout; no token sits on the border of
    # the clip, where one rounding turns its gradient off
    moved = torch.randn(batch, seq, generator=g, device=dev) * 0.15
    for border in (math.log(1.2), math.log(0.8)):
        moved = torch.where((moved - border).abs() < 1e-3, moved + 4e-3, moved)
    state.update(actions=targets, mask=keep, old_logps=logps - moved,
                 advantages=torch.randn(batch, seq, generator=g, device=dev) * 0.7 + 0.5)
    if case["kl"]:
        state["ref_logps"] = logps + torch.randn(batch, seq, generator=g, device=dev) * 0.3
    return state


# ----------------------------------------------------------------- plain forms
def _softmax_parts(x):
    """x - max, log of the sum of its exponentials, and the probabilities."""
    x = x - x.amax(-1, keepdim=True)
    e = x.exp()
    s = e.sum(-1, keepdim=True)
    return x, s.log(), e / s


def _plain_topk(s):
    x, k = s["logits"], s["case"]["k"]
    # a key that sorts by value, and by the lower place where values are equal
    bits = (x.float() + 0.0).view(torch.int32)
    order = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).long() << 32
    places = (1 << 31) - 1 - torch.arange(x.shape[-1], device=x.device)
    keys = (order + places).topk(k, dim=-1).values
    indices = (1 << 31) - 1 - (keys & 0xFFFFFFFF)
    shifted = x.float()
    top = shifted.amax(-1)
    lse = top + (shifted - top[:, None]).exp().sum(-1).log()
    return x.gather(-1, indices), indices, lse


def _plain_distill(s):
    case, logits, idx, mask = s["case"], s["logits"].detach(), s["indices"], s["mask"]
    t = case["temperature"]
    x, log_s, q = _softmax_parts(logits.float() / t)
    log_q = x.gather(-1, idx) - log_s
    v = s["values"].float() / t
    weight = mask.float() / mask.sum().clamp_min(1)
    if case["tail"]:
        log_p = v.double() - s["lse"].double()[..., None]
        p = log_p.exp()
        p_tail = (1.0 - p.sum(-1, keepdim=True)).clamp_min(0.0)
        inside = torch.zeros_like(q, dtype=torch.bool).scatter_(-1, idx, True)
        q_tail = q.masked_fill(inside, 0.0).sum(-1, keepdim=True)
        rows = (p * (log_p - log_q)).sum(-1) + (torch.xlogy(p_tail, p_tail) - p_tail * q_tail.log())[..., 0]
        grad = q * torch.where(inside, 1.0, (1.0 - p_tail / q_tail).float())
    else:
        y, log_z, p = _softmax_parts(v)
        rows = (p * ((y - log_z) - log_q)).sum(-1)
        grad = q
    grad = grad.scatter_add(-1, idx, -p.float()) * (t * s["scale"] * weight)[..., None]
    loss = (rows.float() * weight).sum() * (t * t)
    return loss, grad.to(logits.dtype)


def _plain_logps(logits, targets):
    """Log-probability of each target, in 64 bits as differences of them follow, and the probabilities."""
    x = logits.float()
    top = x.amax(-1, keepdim=True)
    e = (x - top).exp()
    s = e.sum(-1, keepdim=True)
    logps = (x.gather(-1, targets[..., None]) - top).double() - s.double().log()
    return logps[..., 0], e / s


def _plain_logits_grad(q, targets, by_logp, dtype):
    """d(logp of target)/d(logits) is onehot - q, times the loss's derivative by logp."""
    grad = q * -by_logp[..., None]
    return grad.scatter_add_(-1, targets[..., None], by_logp[..., None]).to(dtype)


def _plain_preference(s):
    logits, targets, n = s["logits"].detach(), s["targets"], s["case"]["pairs"]
    beta, eps = 0.1, s["case"]["smoothing"]
    keep = targets != -100
    safe = targets.clamp_min(0)
    logps, q = _plain_logps(logits, safe)
    # sums over whole answers differ little from the reference's: in 64 bits
    rewards = beta * (torch.where(keep, logps, 0.0).sum(-1) - s["ref_logps"].double())
    z = rewards[:n] - rewards[n:]
    softplus = z.clamp_min(0.0) + (-z.abs()).exp().log1p()  # log(1 + exp(z))
    loss = ((1 - eps) * (softplus - z) + eps * softplus).mean()
    by_z = (1.0 / (1.0 + (-z).exp()) - (1 - eps)) / n
    by_logp = (torch.cat([by_z, -by_z]) * beta * s["scale"]).float()[:, None] * keep
    grad = _plain_logits_grad(q, safe, by_logp, logits.dtype)
    return loss.float(), rewards[:n].float(), rewards[n:].float(), grad


def _plain_policy(s):
    logits, actions, mask, adv = s["logits"].detach(), s["actions"], s["mask"], s["advantages"]
    kl_coef = s["case"]["kl"]
    logps, q = _plain_logps(logits, actions)
    weight = mask.float() / mask.sum().clamp_min(1)
    ratio = (logps - s["old_logps"]).exp()
    loss = -torch.minimum(ratio * adv, ratio.clamp(0.8, 1.2) * adv)
    moves = torch.where(adv > 0, ratio <= 1.2, ratio >= 0.8)
    by_logp = torch.where(moves, -adv * ratio, 0.0)
    kl = torch.zeros_like(logps)
    if kl_coef:
        d = s["ref_logps"] - logps
        kl = d.expm1() - d
        loss = loss + kl_coef * kl
        by_logp = by_logp - kl_coef * d.expm1()
    grad = _plain_logits_grad(q, actions, (by_logp * weight * s["scale"]).float(), logits.dtype)
    return ((loss * weight).sum().float(), torch.where(mask, logps, 0.0).float(),
            torch.where(mask, kl, 0.0).float(), grad)


_PLAIN = {"topk": _plain_topk, "distill": _plain_distill, "preference": _plain_preference, "policy": _plain_policy}


# ------------------------------------------------------------ the framework's
def _own_topk(s):
    from vantage6_amd.ops.distill import topk_logits

    return tuple(topk_logits(s["logits"], s["case"]["k"]))


def _own_distill(s):
    from vantage6_amd.ops.distill import distill_loss

    loss = distill_loss(s["logits"], s["values"], s["indices"], s.get("lse"),
                        temperature=s["case"]["temperature"], mask=s["mask"])
    return loss.detach(), torch.autograd.grad(loss, s["logits"], s["scale"])[0]


def _own_preference(s):
    from vantage6_amd.ops.preference import preference_loss

    loss, chosen, rejected = preference_loss(s["logits"], s["targets"], s["ref_logps"], beta=0.1,
                                             label_smoothing=s["case"]["smoothing"])
    return loss.detach(), chosen, rejected, torch.autograd.grad(loss, s["logits"], s["scale"])[0]


def _own_policy(s):
    from vantage6_amd.ops.preference import policy_loss

    loss, logps, kl = policy_loss(s["logits"], s["actions"], s["old_logps"], s["advantages"],
                                  s.get("ref_logps"), mask=s["mask"], clip_low=0.2, clip_high=0.2,
                                  kl_coef=s["case"]["kl"])
    return loss.detach(), logps, kl, torch.autograd.grad(loss, s["logits"], s["scale"])[0]


_OWN = {"topk": _own_topk, "distill": _own_distill, "preference": _own_preference, "policy": _own_policy}


def run(state):
    return _OWN[state["op"]](state) if own else _PLAIN[state["op"]](state)


# ------------------------------------------------------------------------ work
def work(case):
    size = _TYPES[case["dtype"]].itemsize
    batch, seq = _shape(case)
    R, V, k = batch * seq, case["vocab"], case.get("k", 0)
    live = R if case["op"] == "topk" else sum(_lengths(case))
    read, wrote = live * V * size, 0
    if case["op"] == "topk":
        return {"bytes": read + R * (k * (size + 8) + 4), "flops": 4 * R * V}
    wrote = R * V * size
    small = {"distill": R * (k * (size + 8) + 1 + (4 if case.get("tail") else 0)),
             "preference": R * 8 + 16 * batch,
             "policy": R * (8 + 4 + 4 + 1 + 8 + (4 if case.get("kl") else 0))}[case["op"]]
    return {"bytes": read + wrote + small, "flops": 7 * live * V}


# ----------------------------------------------------------------------- exact
def _exact_rows(logits, t=1.0):
    """Slabs of rows in 64 bits with their logsumexp, so that the largest case fits."""
    flat = logits.detach().reshape(-1, logits.shape[-1])
    for at in range(0, flat.shape[0], 256):
        x = flat[at:at + 256].double() / t
        yield at, x, torch.logsumexp(x, -1)


def _exact_topk(s):
    k, parts = s["case"]["k"], []
    for _, x, lse in _exact_rows(s["logits"]):
        values, indices = torch.sort(x, dim=-1, descending=True, stable=True)
        parts.append((values[:, :k].clone(), indices[:, :k].clone(), lse))
    return tuple(torch.cat(column) for column in zip(*parts))


def _exact_distill(s):
    case, logits = s["case"], s["logits"]
    t, k, V = case["temperature"], case["k"], case["vocab"]
    idx, values = s["indices"].reshape(-1, k), s["values"].reshape(-1, k).double() / t
    mask = s["mask"].reshape(-1).double()
    weight, total, grads = mask / mask.sum().clamp_min(1), 0.0, []
    for at, x, lse in _exact_rows(logits, t):
        n = x.shape[0]
        i, w = idx[at:at + n], weight[at:at + n]
        q = (x - lse[:, None]).exp()
        q_top = q.gather(-1, i)
        if case["tail"]:
            p = (values[at:at + n] - s["lse"].reshape(-1)[at:at + n].double()[:, None]).exp()
            outside = q.scatter(-1, i, 0.0).sum(-1)
            p_out = (1 - p.sum(-1)).clamp_min(0)
            rows = torch.xlogy(p, p / q_top).sum(-1) + torch.xlogy(p_out, p_out / outside)
            grad = q * (1 - p_out / outside)[:, None]
        else:
            p = torch.softmax(values[at:at + n], -1)
            rows = torch.xlogy(p, p / q_top).sum(-1)
            grad = q
        grad = grad.scatter(-1, i, q_top - p)
        total = total + (rows * w).sum()
        grads.append(grad * (t * w * s["scale"])[:, None])
    return total * t * t, torch.cat(grads).view(logits.shape)


def _exact_scores(logits, targets):
    flat = targets.reshape(-1, 1)
    return torch.cat([x.gather(-1, flat[at:at + x.shape[0]])[:, 0] - lse
                      for at, x, lse in _exact_rows(logits)]).view(targets.shape)


def _exact_grad(s, targets, by_logp):
    logits, by_logp = s["logits"], by_logp * s["scale"]
    flat, d, grads = targets.reshape(-1, 1), by_logp.reshape(-1, 1), []
    for at, x, lse in _exact_rows(logits):
        n = x.shape[0]
        one = torch.zeros_like(x).scatter_(-1, flat[at:at + n], 1.0)
        grads.append(d[at:at + n] * (one - (x - lse[:, None]).exp()))
    return torch.cat(grads).view(logits.shape)


def _exact_preference(s):
    n, eps, logits = s["case"]["pairs"], s["case"]["smoothing"], s["logits"]
    keep = (s["targets"] >= 0).double()
    targets = s["targets"].clamp_min(0)
    scores = (_exact_scores(logits, targets) * keep).sum(-1)
    rewards = 0.1 * (scores - s["ref_logps"].double())
    z = (rewards[:n] - rewards[n:]).requires_grad_(True)
    loss = -((1 - eps) * torch.nn.functional.logsigmoid(z) + eps * torch.nn.functional.logsigmoid(-z)).mean()
    by_z = torch.autograd.grad(loss, z)[0]
    by_logp = 0.1 * torch.cat([by_z, -by_z])[:, None] * keep
    return loss.detach(), rewards[:n], rewards[n:], _exact_grad(s, targets, by_logp)


def _exact_policy(s):
    mask, adv, logits = s["mask"].double(), s["advantages"].double(), s["logits"]
    scores = _exact_scores(logits, s["actions"]).requires_grad_(True)
    ratio = torch.exp(scores - s["old_logps"].double())
    loss, kl = -torch.min(ratio * adv, torch.clamp(ratio, 0.8, 1.2) * adv), torch.zeros_like(scores)
    if s["case"]["kl"]:
        d = s["ref_logps"].double() - scores
        kl = torch.expm1(d) - d
        loss = loss + s["case"]["kl"] * kl
    loss = (loss * mask).sum() / mask.sum().clamp_min(1)
    by_logp = torch.autograd.grad(loss, scores)[0]
    return loss.detach(), scores.detach() * mask, kl.detach() * mask, _exact_grad(s, s["actions"], by_logp)


def exact(case, seed):
    state = prepare(case, seed)
    return {"topk": _exact_topk, "distill": _exact_distill, "preference": _exact_preference,
            "policy": _exact_policy}[case["op"]](state)
