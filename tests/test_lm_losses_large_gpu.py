"""Losses and records over more logits than the caches hold, against 64 bits.

What a pass does depends on the bytes of its logits: a gradient of more than
64 MB is written past the caches, of more than 300 MB of logits only a part is
told to stay in them and the gradient goes in shorter segments, and more than
128 MB are streamed by topk. Every row is compared, in slabs on the device.
The tolerances are those of the small sizes (test_lm_losses.py): LP for a
log-probability, GRAD for a gradient, for every V up to 131072.
"""
import math

import pytest
import torch

from test_lm_losses import GRAD, LP, TYPES, half_step, need
from vantage6_amd.ops.distill import distill_loss, topk_logits
from vantage6_amd.ops.preference import policy_loss, preference_loss

pytestmark = pytest.mark.gpu

MB = 2 ** 20
SLAB = 128
# (dtype, sequences, tokens, V, logits that a row has behind those V). Sizes in
# bytes lie above 64 MB, where the gradient is streamed, or above 300 MB.
STREAMED = [(torch.bfloat16, 2, 350, 50021, 0), (torch.float16, 3, 401, 30522, 6),
            (torch.float32, 1, 361, 50021, 0)]
FAR = [(torch.bfloat16, 2, 850, 128257, 0), (torch.float32, 1, 850, 128256, 3),
       (torch.float16, 11, 1000, 16001, 0)]  # the last: a wave to each row


def large_logits(dtype, B, T, V, more, seed=0, least=64 * MB):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(B, T, V + more, generator=g, device="cuda").mul_(3.0).to(dtype)
    x = x[..., :V]
    assert x.numel() * x.element_size() > least
    return x


def ragged(B, T, seed=5):
    ends = torch.randint(T // 2, T + 1, (B, 1), generator=torch.Generator().manual_seed(seed))
    return (torch.arange(T)[None] < ends).cuda()


def slabs(x):
    """(first row, rows in 64 bits), of logits [B, T, V]."""
    B, T, V = x.shape
    for b in range(B):
        for t in range(0, T, SLAB):
            yield b * T + t, x[b, t:t + SLAB].double()


def close_grad(got, want, a, q):
    """got [n, V] against want; a [n] the rows' coefficients, q what scales."""
    least = 2.0 ** -24 if got.dtype == torch.float16 else 1e-37
    tol = (half_step(got.dtype) + GRAD) * want.abs() + GRAD * a.abs()[:, None] * q + least
    err = (got.double() - want).abs()
    assert (err <= tol).all(), (err - tol).max().item()


def scale_of(dtype, n):
    """An upstream gradient that undoes the mean, and in fp16 lifts the
    probabilities above the type's least values."""
    return n * (512.0 if dtype == torch.float16 else 1.0)


# ------------------------------------------------------------------------ topk
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V,k", [(4001, 24), (8200, 256), (30522, 32), (300001, 64)])
def test_topk_streamed(dtype, V, k):
    """Logits kept one by one, in vectors, in lines, and by larger blocks."""
    need("cuda")
    size = 4 if dtype == torch.float32 else 2
    rows = 128 * MB // (V * size) + 3
    x = large_logits(dtype, 1, rows, V, 0, least=128 * MB)
    x[0, 0, V // 2:] = 20.0  # a row of ties
    got = topk_logits(x, k, 2.0)
    for at, row in slabs(x):
        n = len(row)
        values, places = torch.sort(row + 0.0, dim=-1, descending=True, stable=True)
        assert torch.equal(got.indices[0, at:at + n], places[:, :k])
        assert torch.equal(got.values[0, at:at + n].double(), values[:, :k])
        torch.testing.assert_close(got.logsumexp[0, at:at + n].double(),
                                   torch.logsumexp(row / 2.0, -1), rtol=2.0 ** -23, atol=LP)


# --------------------------------------------------------------------- distill
def bordering_record(x, K, t, seed=1):
    """K places a row, each the first or the last of 32 logits, where segments
    end and begin. Over all rows every such place is one of a record."""
    B, T, V = x.shape
    g = torch.Generator(device="cuda").manual_seed(seed)
    blocks = torch.rand(B * T, V // 32, generator=g, device="cuda").argsort(-1)[:, :K]
    places = (blocks * 32 - torch.randint(0, 2, blocks.shape, generator=g, device="cuda"))
    places = places.clamp_min(0).view(B, T, K)
    noise = torch.randn(B, T, K, generator=g, device="cuda")
    values = (x.gather(-1, places).float() + 4.0 + noise).to(x.dtype)
    lse = torch.empty(B * T, dtype=torch.float64, device="cuda")
    for at, row in slabs(x):
        # of a teacher that differs from the student at these places alone
        n = len(row)
        row = row.scatter(-1, places.view(-1, K)[at:at + n], values.view(-1, K)[at:at + n].double())
        lse[at:at + n] = torch.logsumexp(row / t, -1)
    return values, places, lse.float().view(B, T)


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("case", STREAMED + FAR, ids=str)
def test_distill_large(case, tail):
    need("cuda")
    dtype, B, T, V, more = case
    t, K = 2.0, 200
    x = large_logits(*case, least=(300 if case in FAR else 64) * MB).detach().requires_grad_(True)
    values, places, lse = bordering_record(x.detach(), K, t)
    mask = ragged(B, T)
    live = mask.view(-1)
    n_live = int(live.sum())
    up = torch.tensor(scale_of(dtype, n_live), device="cuda")
    loss = distill_loss(x, values, places, lse if tail else None, temperature=t, mask=mask)
    grad, = torch.autograd.grad(loss, x, up)
    with torch.no_grad():
        each = distill_loss(x, values, places, lse if tail else None, temperature=t, mask=mask,
                            reduction="none").view(-1)
    grad = grad.reshape(B * T, V)
    a = t * live.double() * up.item() / n_live
    total = 0.0
    for at, row in slabs(x.detach()):
        s = slice(at, at + len(row))
        idx, v = places.view(-1, K)[s], values.view(-1, K)[s].double() / t
        lq = torch.log_softmax(row / t, -1)
        lp = v - (lse.view(-1)[s].double()[:, None] if tail else torch.logsumexp(v, -1, keepdim=True))
        p = lp.exp()
        rows, q = (p * (lp - lq.gather(-1, idx))).sum(-1), lq.exp()
        want = q
        if tail:
            rest = 1.0 - p.sum(-1, keepdim=True)
            assert (rest > 0).all()
            out = torch.logsumexp(lq.scatter(-1, idx, -math.inf), -1, keepdim=True)
            rows = rows + (rest * (rest.log() - out))[:, 0]
            want = (q - rest * (lq - out).exp()).scatter(-1, idx, q.gather(-1, idx))
        else:
            want = want * p.sum(-1, keepdim=True)
        want = want.scatter_add(-1, idx, -p)
        rows = torch.where(live[s], rows * t * t, 0.0)
        torch.testing.assert_close(each[s].double(), rows, rtol=2.0 ** -22, atol=2 * t * t * LP)
        total += rows.sum().item()
        # outside the record the gradient is that of q over its sum there
        close_grad(grad[s], want * a[s][:, None], a[s], q + want.abs() if tail else q)
    assert (grad[~live] == 0).all()
    assert abs(loss.item() - total / n_live) <= 2 * t * t * LP + 2.0 ** -22 * abs(loss.item())


# ------------------------------------------------------- preference and policy
def target_logps(x, targets):
    """[B * T] in 64 bits, 0 where the target is negative."""
    flat, parts = targets.reshape(-1), []
    for at, row in slabs(x):
        idx = flat[at:at + len(row)]
        lp = torch.log_softmax(row, -1).gather(-1, idx.clamp_min(0)[:, None])[:, 0]
        parts.append(torch.where(idx >= 0, lp, 0.0))
    return torch.cat(parts)


def check_onehot_grad(grad, x, targets, by_lp, big):
    """by_lp (onehot - q) in each row; an error of by_lp is one of ``big``."""
    flat = targets.reshape(-1)
    grad = grad.reshape(len(flat), -1)
    for at, row in slabs(x):
        s = slice(at, at + len(row))
        q = torch.softmax(row, -1)
        one = torch.zeros_like(q).scatter_(-1, flat[s].clamp_min(0)[:, None], 1.0)
        close_grad(grad[s], by_lp[s][:, None] * (one - q), big[s], (one - q).abs() + q)
    assert (grad[by_lp == 0] == 0).all()


@pytest.mark.parametrize("case", STREAMED + FAR, ids=str)
def test_policy_large(case):
    need("cuda")
    dtype, B, T, V, more = case
    x = large_logits(*case, least=(300 if case in FAR else 64) * MB).detach().requires_grad_(True)
    g = torch.Generator(device="cuda").manual_seed(3)
    actions = torch.randint(0, V, (B, T), generator=g, device="cuda")
    lp = target_logps(x.detach(), actions)
    moved = torch.randn(B * T, generator=g, device="cuda").double() * 0.3
    for border in (math.log(1.2), math.log(0.8)):
        moved = torch.where((moved - border).abs() < 1e-3, moved + 4e-3, moved)
    old = (lp - moved).float()
    ref = (lp + torch.randn(B * T, generator=g, device="cuda") * 0.3).float()
    adv = torch.randn(B * T, generator=g, device="cuda")
    mask = ragged(B, T)
    live = mask.view(-1)
    n_live, coef = int(live.sum()), 0.05
    up = torch.tensor(scale_of(dtype, n_live), device="cuda")
    out = policy_loss(x, actions, old.view(B, T), adv.view(B, T), ref.view(B, T), mask=mask,
                      kl_coef=coef)
    grad, = torch.autograd.grad(out.loss, x, up)
    torch.testing.assert_close(out.logps.view(-1).double(), torch.where(live, lp, 0.0),
                               rtol=2.0 ** -23, atol=LP)
    A, ratio = adv.double(), (lp - old.double()).exp()
    d = ref.double() - lp
    loss = -torch.minimum(ratio * A, ratio.clamp(0.8, 1.2) * A) + coef * (d.expm1() - d)
    by_lp = torch.where(torch.where(A > 0, ratio <= 1.2, ratio >= 0.8), -A * ratio, 0.0)
    by_lp = by_lp - coef * d.expm1()
    want = (loss * live).sum().item() / n_live
    # as in the small sizes: ratios of at most e^2, advantages of at most 5
    assert abs(out.loss.item() - want) <= 50 * LP + 2.0 ** -22 * abs(want)
    each = live.double() * up.item() / n_live
    check_onehot_grad(grad, x.detach(), actions, by_lp * each,
                      (by_lp.abs() + 2 * A.abs() + 3 * coef) * each)


@pytest.mark.parametrize("case", [(torch.bfloat16, 4, 175, 50021, 0), (torch.float16, 4, 301, 30522, 6),
                                  (torch.float32, 2, 181, 50021, 0), (torch.bfloat16, 4, 425, 128257, 0),
                                  (torch.float32, 2, 425, 128256, 3)], ids=str)
def test_preference_large(case):
    need("cuda")
    dtype, B, T, V, more = case
    x = large_logits(*case).detach().requires_grad_(True)
    g = torch.Generator(device="cuda").manual_seed(3)
    keep = ragged(B, T)
    targets = torch.where(keep, torch.randint(0, V, (B, T), generator=g, device="cuda"), -100)
    lp = target_logps(x.detach(), targets)
    sums, n, beta, eps = lp.view(B, T).sum(-1), B // 2, 0.1, 0.1
    ref = sums + torch.randn(B, generator=g, device="cuda").double() * 8.0
    out = preference_loss(x, targets, ref, beta=beta, label_smoothing=eps)
    up = torch.tensor(scale_of(dtype, n) / beta, device="cuda")
    grad, = torch.autograd.grad(out.loss, x, up)
    r = beta * (sums - ref)
    z = r[:n] - r[n:]
    logsig = torch.nn.functional.logsigmoid
    want = (-(1 - eps) * logsig(z) - eps * logsig(-z)).mean()
    # a reward sums T log-probabilities, a margin two of them
    lim = beta * T * LP
    torch.testing.assert_close(out.chosen_rewards.double(), r[:n], rtol=2.0 ** -23, atol=lim)
    torch.testing.assert_close(out.rejected_rewards.double(), r[n:], rtol=2.0 ** -23, atol=lim)
    torch.testing.assert_close(out.loss.double(), want, rtol=2.0 ** -22, atol=2 * lim)
    by_z = (torch.sigmoid(z) - (1 - eps)) / n
    by_lp = torch.cat([by_z, -by_z]) * beta * up.item()
    by_lp = torch.where(keep, by_lp[:, None], 0.0).view(-1)
    # sigmoid moves by a quarter of the margin's error at most, 2 lim
    big = by_lp.abs() + torch.where(keep, 0.5 * lim / GRAD * beta * up.item() / n, 0.0).view(-1)
    check_onehot_grad(grad, x.detach(), targets, by_lp, big)


def test_records_past_32_bits():
    """Rows behind 2^31 logits: a record's places and gradient there."""
    need("cuda")
    T, V, K, t = 18000, 128256, 64, 2.0
    x = torch.empty(1, T, V, dtype=torch.bfloat16, device="cuda")
    x.normal_(generator=torch.Generator(device="cuda").manual_seed(0))
    top = topk_logits(x, K, t)
    x.requires_grad_(True)
    # the record of another model: this one's, less sure of itself
    values = top.values * 0.5
    loss = distill_loss(x, values, top.indices, top.logsumexp, temperature=t, reduction="sum")
    grad, = torch.autograd.grad(loss, x)
    for r in (0, 9000, 16743, 16744, 17999):
        row = x.detach()[0, r].double()
        want, places = torch.sort(row, descending=True, stable=True)
        assert torch.equal(top.indices[0, r], places[:K])
        assert torch.equal(top.values[0, r].double(), want[:K])
        lse = torch.logsumexp(row / t, -1)
        assert abs(top.logsumexp[0, r].item() - lse.item()) <= LP + 2.0 ** -23 * lse.item()
        idx, lq = places[:K], torch.log_softmax(row / t, -1)
        p = (values[0, r].double() / t - top.logsumexp[0, r].double()).exp()
        rest = 1.0 - p.sum()
        out = torch.logsumexp(lq.scatter(-1, idx, -math.inf), -1)
        q = lq.exp()
        g = (q - rest * (lq - out).exp()).scatter(-1, idx, q[idx] - p) * t
        close_grad(grad[0, r][None], g[None], torch.tensor([t], device="cuda"), (q + g.abs() / t)[None])
