"""Losses and records over vocabulary logits, against 64-bit definitions.

Tolerances, for every V up to 131072. A thread adds at most 128 terms to one
of its sums and some 20 joins follow, each addition off by 2^-24; a term
2^((x-m)c) is off by 2^-23 from the instruction and by 2^-23 |a| ln 2 from
its argument a, and the mean of |a| ln 2 under the softmax is at most
ln V < 12. S, and with it a log-probability, is off by at most
(128 + 20 + 2 + 2 * 12) 2^-24 < 200 * 2^-24 = LP. A probability as small as
e^-88 has an argument off by 88 * 2^-23, so q is off by at most LP + 88 * 2^-23
< 2.3e-5 of itself, and the coefficient of a row (an exponential of an lp) by
2 LP of itself: a gradient a (q - p) by 6e-5 (|a| q + |gradient|), and by half
a step of its type. fp16 has steps of 2^-24 below its normal range.
"""
import math

import pytest
import torch

from vantage6_amd.ops.distill import distill_loss, topk_logits
from vantage6_amd.ops.preference import policy_loss, preference_loss

LP = 200 * 2.0 ** -24
GRAD = 6e-5
CPU_GPU = [pytest.param("cpu"), pytest.param("cuda", marks=pytest.mark.gpu)]
TYPES = [torch.bfloat16, torch.float16, torch.float32]
# (B, T, V): one token, a vocabulary of one, below a vector, odd, several
# segments, the models' vocabularies
SHAPES = [(1, 1, 1), (1, 2, 7), (2, 3, 257), (3, 5, 4099), (2, 2, 30522),
          (1, 3, 128256), (40, 30, 613)]


def need(device):
    if device == "cuda" and not torch.cuda.is_available():
        pytest.skip("needs a GPU")


def make_logits(B, T, V, dtype, device, seed=0, scale=3.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(B, T, V, generator=g) * scale).to(dtype).to(device)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def check_grad(got, want, a, q):
    """got [.., V] against want (64 bits), a [..] the row's coefficient."""
    assert got.shape == want.shape
    least = 2.0 ** -24 if got.dtype == torch.float16 else 1e-37
    want, a, q = want.double().cpu(), a.double().cpu().abs()[..., None], q.cpu()
    tol = (half_step(got.dtype) + GRAD) * want.abs() + GRAD * a * q + least
    err = (got.double().cpu() - want).abs()
    assert (err <= tol).all(), (err - tol).max().item()


def softmax64(logits, t=1.0):
    x = logits.detach().cpu().double() / t
    return torch.log_softmax(x, -1)


# ------------------------------------------------------------------------ topk
def topk_oracle(logits, k):
    """By value, then by place; NaN above all, -0 equal to 0."""
    x = logits.detach().cpu().double()
    values, places = [], []
    for row in x.reshape(-1, x.shape[-1]).tolist():
        order = sorted(range(len(row)), key=lambda j: (
            -(math.inf if row[j] != row[j] else row[j]),
            0 if row[j] != row[j] else 1, j))
        # a NaN sorts with +inf by value and before it by the flag
        places.append(order[:k])
        values.append([row[j] for j in order[:k]])
    shape = (*x.shape[:-1], k)
    return torch.tensor(values, dtype=torch.float64).view(shape), torch.tensor(places).view(shape)


def check_topk(logits, k, t=1.0):
    got = topk_logits(logits, k, t)
    values, places = topk_oracle(logits, k)
    assert got.values.dtype == logits.dtype and got.indices.dtype == torch.int64
    assert torch.equal(got.indices.cpu(), places)
    assert torch.equal(got.values.cpu().double().nan_to_num(7e77), values.nan_to_num(7e77))
    lse = torch.logsumexp(logits.detach().cpu().double() / t, -1)
    torch.testing.assert_close(got.logsumexp.cpu().double(), lse, rtol=2.0 ** -23,
                               atol=LP, equal_nan=True)


@pytest.mark.parametrize("device", CPU_GPU)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,V,k", [(1, 1, 1), (3, 5, 5), (2, 8, 3), (5, 257, 256),
                                   (4, 1001, 128), (2, 4099, 1), (3, 30522, 64),
                                   (1, 128256, 256), (2, 131075, 17)])
def test_topk(device, dtype, R, V, k):
    need(device)
    check_topk(make_logits(1, R, V, dtype, device)[0], k, 1.0 if R % 2 else 2.0)


@pytest.mark.parametrize("device", CPU_GPU)
@pytest.mark.parametrize("dtype", TYPES)
def test_topk_ties_and_masks(device, dtype):
    """Constant rows, few finite logits, the type's lowest value, NaN, +-0."""
    need(device)
    V = 5003
    x = make_logits(1, 8, V, dtype, "cpu")[0]
    x[0] = 1.5  # all equal
    x[1] = float("-inf")
    x[1, 77] = -2.0  # one finite
    x[2] = torch.finfo(dtype).min
    x[2, 4000] = 0.5
    x[3, 100] = x[3, 4000] = float("nan")
    x[3, 50] = float("inf")
    x[4] = torch.where(torch.arange(V) % 2 == 0, 0.0, -0.0).to(dtype)
    x[5] = float("-inf")
    x[6, 1000:] = -3.0  # a long run of equal logits behind a few
    x[6, :1000] = -5.0
    x[6, :3] = 4.0
    x[7, 4992:] = 9.0  # the largest in the last, partial vector
    for v in (V, 700, 4090):  # a long row, and ones that are kept whole
        check_topk(x[:, V - v:].to(device), 12)


@pytest.mark.parametrize("device", CPU_GPU)
@pytest.mark.parametrize("dtype", TYPES)
def test_topk_infinite_logits(device, dtype):
    """A logit of +inf and no NaN beside it: the logsumexp is +inf, at any
    place of a row, alone, several times, and beside -inf."""
    need(device)
    V = 5003
    x = make_logits(1, 6, V, dtype, "cpu")[0]
    x[0, 4500] = x[1, V - 1] = x[2, V - 700] = float("inf")
    x[3] = float("inf")
    x[4] = float("-inf")
    x[4, V - 300] = float("inf")
    x[5, V - 200] = float("inf")
    x[5, V - 100] = float("nan")  # with a NaN: a NaN
    for v in (V, 700, 1):  # a row in lines or in vectors, one kept whole, one logit
        for k, t in ((1, 1.0), (12, 2.0), (40, 0.5)):
            if k <= v:
                check_topk(x[:, V - v:].to(device), k, t)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V,k", [(600, 256), (2100, 200), (4096, 256), (4097, 256), (8200, 256),
                                 (33000, 256), (33000, 100), (262144, 33), (300001, 256)])
def test_topk_piece_sizes(dtype, V, k):
    """Around the sizes at which a row is cut into other pieces."""
    need("cuda")
    check_topk(make_logits(1, 3, V, dtype, "cuda")[0], k)


@pytest.mark.parametrize("device", CPU_GPU)
def test_topk_layouts(device):
    need(device)
    x = make_logits(3, 6, 515, torch.bfloat16, device)
    for view in (x[:, :-1], x[:, 1:, :512], x[:, :, 1:], x.transpose(0, 1), x[0, 0],
                 x[:1].expand(3, 6, 515), x[..., ::2], x.view(3, 2, 3, 515)):
        check_topk(view, 5)
    empty = topk_logits(x[:, :0], 3)
    assert empty.values.shape == empty.indices.shape == (3, 0, 3)
    assert empty.logsumexp.shape == (3, 0)


# --------------------------------------------------------------------- distill
def distill_oracle(logits, values, indices, lse, t, mask):
    """(loss of each row, live, gradient of the sum, coefficient), 64 bits."""
    V = logits.shape[-1]
    x = logits.detach().cpu().double().reshape(-1, V) / t
    K = indices.shape[-1]
    v = values.cpu().double().reshape(-1, K) / t
    idx = indices.cpu().long().reshape(-1, K)
    m = (torch.ones(len(x), dtype=torch.bool) if mask is None else mask.cpu().reshape(-1))
    L = None if lse is None else lse.cpu().double().reshape(-1)
    loss, live = torch.zeros(len(x), dtype=torch.float64), torch.zeros(len(x), dtype=torch.bool)
    grad = torch.zeros_like(x)
    for r in range(len(x)):
        use = (idx[r] >= 0) & (v[r] > -math.inf)
        if not m[r] or not use.any():
            continue
        live[r] = True
        lq = torch.log_softmax(x[r], -1)
        lp = v[r][use] - (torch.logsumexp(v[r][use], -1) if L is None else L[r])
        p, at = lp.exp(), idx[r][use]
        loss[r] = torch.where(p > 0, p * (lp - lq[at]), 0.0).sum()
        target = torch.zeros(V, dtype=torch.float64).scatter_add_(0, at, p)
        # -sum p log q - rest log q_out, with any sum of p: mass q - p - rest q_out
        q, mass = lq.exp(), p.sum()
        if L is not None:
            inside = torch.zeros(V, dtype=torch.bool)
            inside[idx[r][idx[r] >= 0]] = True
            rest = (1 - p.sum()).clamp_min(0)
            if (x[r][~inside] > -math.inf).any():
                log_out = torch.logsumexp(lq[~inside], -1)
                loss[r] += torch.xlogy(rest, rest) - rest * log_out
                # q_j rest / q_out, from logarithms as q_out may be tiny
                mass = mass + rest
                q = torch.where(inside, q, q - rest / mass * (lq - log_out).exp())
        grad[r] = t * (mass * q - target)
        loss[r] *= t * t
    rows = logits.shape[:-1]
    return loss.view(rows), live.view(rows), grad.view(logits.shape)


def make_record(logits, k, t, seed=1, tail=True):
    g = torch.Generator().manual_seed(seed)
    teacher = logits.detach().cpu().float() + torch.randn(logits.shape, generator=g)
    values, indices = teacher.topk(k, -1)
    lse = torch.logsumexp(teacher / t, -1) if tail else None
    return (values.to(logits.dtype).to(logits.device), indices.to(logits.device),
            None if lse is None else lse.to(logits.device))


def check_distill(logits, values, indices, lse, t=1.0, mask=None, reduction="mean", up=None):
    x = logits.detach().requires_grad_(True) if logits.is_leaf else logits
    loss = distill_loss(x, values, indices, lse, temperature=t, mask=mask, reduction=reduction)
    rows, live, grad = distill_oracle(logits, values, indices, lse, t, mask)
    assert loss.dtype == torch.float32
    n = max(int(live.sum()), 1) if reduction == "mean" else 1
    want = rows if reduction == "none" else rows.sum() / n
    # KL: sum p (log p - lp), each lp off by LP/t at most: t^2 LP and a rounding
    lim = 2 * t * t * LP * (1 if reduction != "sum" else max(int(live.sum()), 1))
    torch.testing.assert_close(loss.detach().cpu().double(), want, rtol=2.0 ** -22, atol=lim)
    if up is None:
        up = torch.ones_like(loss)
    got, = torch.autograd.grad(loss, x, up)
    scale = up.cpu().double()[..., None] if reduction == "none" else up.cpu().double() / n
    q = torch.where(live[..., None], softmax64(logits, t).exp(), 0.0)
    if lse is not None:
        # outside the record the gradient is q_out-normalised: q + rest * q / q_out
        q = q + grad.abs() / t
    coef = torch.ones(logits.shape[:-1], dtype=torch.float64) * t * (
        up.cpu().double() if reduction == "none" else up.item() / n)
    check_grad(got, grad * scale, coef, q)
    if not live.all():
        assert (got.cpu()[~live] == 0).all()
    return loss.detach(), got


@pytest.mark.parametrize("device", CPU_GPU)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("tail", [False, True])
def test_distill(device, dtype, shape, tail):
    need(device)
    B, T, V = shape
    t = 2.0 if T % 2 else 1.0
    x = make_logits(B, T, V, dtype, device)
    k = min(V, 1 if B == 1 and T == 1 else 19)
    values, indices, lse = make_record(x, k, t, tail=tail)
    mask = None
    if B > 1:
        mask = (torch.arange(T)[None] < torch.randint(1, T + 1, (B, 1),
                                                      generator=torch.Generator().manual_seed(5)))
        mask = mask.to(device)
    scale = 512.0 if dtype == torch.float16 else 1.0
    check_distill(x, values, indices, lse, t, mask,
                  up=torch.tensor(scale, device=device))


@pytest.mark.parametrize("device", CPU_GPU)
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("tail", [False, True])
def test_distill_reductions_and_upstream(device, reduction, tail):
    need(device)
    x = make_logits(2, 4, 1023, torch.float32, device)
    values, indices, lse = make_record(x, 6, 1.0, tail=tail)
    up = torch.randn(2, 4, generator=torch.Generator().manual_seed(3)).to(device)
    check_distill(x, values, indices.int(), lse, 1.0, None, reduction,
                  up if reduction == "none" else torch.tensor(-3.5, device=device))


@pytest.mark.parametrize("device", CPU_GPU)
@pytest.mark.parametrize("t", [0.05, 0.3, 0.7, 1.1, 1.5, 3.0, 4.0, 7.3, 100.0])
def test_temperatures(device, t):
    """Any temperature, whichever way log2(e)/t rounds; a last vector that is
    not whole and logits of -inf."""
    need(device)
    x = make_logits(1, 3, 1027, torch.float32, device, scale=3.0 * min(t, 2.0))
    x[..., 1000:] = float("-inf")
    for tail in (False, True):
        values, indices, lse = make_record(x, 6, t, tail=tail)
        check_distill(x, values, indices, lse, t)
    check_topk(x, 6, t)


@pytest.mark.parametrize("device", CPU_GPU)
@pytest.mark.parametrize("tail", [False, True])
def test_distill_odd_records(device, tail):
    """Absent entries, -inf values, the same index twice, an empty record, a
    masked row of NaN and inf, a record of the whole row, masked logits."""
    need(device)
    V, k = 300, 300
    x = make_logits(1, 8, V, torch.float32, "cpu")[0]
    teacher = x + 0.5
    values, indices = teacher.topk(k, -1)
    lse = torch.logsumexp(teacher, -1) if tail else None
    values, indices = values[:, :9].clone(), indices[:, :9].clone()
    indices[0, 3:] = -1  # a short record
    values[1, 2] = float("-inf")
    indices[2, 4] = indices[2, 1]  # the same place twice
    indices[3] = -1  # nothing
    values[4] = float("-inf")  # nothing either
    mask = torch.ones(8, dtype=torch.bool)
    mask[5] = False
    x[5, ::3] = float("nan")
    x[5, 1::3] = float("inf")
    outside = torch.ones(V, dtype=torch.bool)
    outside[indices[6]] = False
    x[6, outside] = float("-inf")  # no mass outside the record
    x[7, outside] = torch.finfo(torch.float32).min
    args = [None if a is None else a.to(device) for a in (x, values, indices, lse)]
    check_distill(*args, 1.0, mask.to(device))
    # no row counts
    loss, grad = check_distill(*args, 1.0, torch.zeros(8, dtype=torch.bool, device=device))
    assert loss.item() == 0.0 and (grad == 0).all()


@pytest.mark.parametrize("device", CPU_GPU)
@pytest.mark.parametrize("tail", [False, True])
def test_distill_empty_records_hold_anything(device, tail):
    """Rows whose record holds nothing, whatever their logits are."""
    need(device)
    x = make_logits(1, 5, 700, torch.float32, device)
    values, indices, lse = make_record(x, 6, 1.0, tail=tail)
    indices[0, 1], values[0, 3] = -1, float("-inf")
    want, grad = check_distill(x, values, indices, lse)
    x[0, 1], x[0, 3, ::2], x[0, 3, 1::2] = float("nan"), float("inf"), float("-inf")
    x.requires_grad_(True)
    loss = distill_loss(x, values, indices, lse)
    got, = torch.autograd.grad(loss, x)
    assert torch.equal(loss.detach(), want) and torch.equal(got, grad)


@pytest.mark.parametrize("device", CPU_GPU)
@pytest.mark.parametrize("tail", [False, True])
def test_distill_layouts(device, tail):
    """Slices, one row, more dimensions, rows that are one; records of another
    type, not contiguous, in another order; masks that are broadcast."""
    need(device)
    x = make_logits(3, 7, 515, torch.float32, device)
    for view in (x[:, :-1], x[:, 1:, :512], x[:, :6, 3:], x[0, 1:], x[1, 2],
                 x.transpose(0, 1)[1:], x[:, :6].reshape(3, 2, 3, 515),
                 x[:1].expand(3, 7, 515), x[..., ::2]):
        values, indices, lse = make_record(view, 9, 1.0, tail=tail)
        values, indices = values.flip(-1)[..., ::2], indices.flip(-1)[..., ::2]
        assert not values.is_contiguous() or values.dim() == 1
        for v, L in ((values, lse), (values.bfloat16(), lse), (values.half(), lse),
                     (values.double(), None if lse is None else lse.double())):
            mask = None
            if view.dim() > 1:
                mask = (torch.arange(view.shape[-2]) != 1).to(device).expand(view.shape[:-1])
            check_distill(view, v, indices, L, 1.0, mask)


@pytest.mark.parametrize("device", CPU_GPU)
def test_distill_whole_row_in_the_record(device):
    need(device)
    x = make_logits(1, 3, 200, torch.float32, device)
    values, indices, lse = make_record(x, 200, 1.0)
    check_distill(x, values, indices, lse)


@pytest.mark.parametrize("device", CPU_GPU)
def test_distill_rest_that_underflows(device):
    """The student gives the record everything: q outside is e^-200, and the
    rest's term is still its logarithm."""
    need(device)
    x = torch.full((1, 2, 500), -200.0, device=device)
    x[..., :3] = 0.0
    values = torch.zeros(1, 2, 3, device=device)
    indices = torch.arange(3, device=device).expand(1, 2, 3)
    lse = torch.full((1, 2), math.log(4.0), device=device)
    loss, grad = check_distill(x, values, indices, lse)
    assert loss.item() > 40.0
    assert abs(grad[..., 3:].sum().item() / -0.25 - 1) < 1e-4


@pytest.mark.parametrize("device", CPU_GPU)
def test_distill_index_outside_is_nan(device):
    need(device)
    x = make_logits(1, 3, 64, torch.float32, device)
    values, indices, _ = make_record(x, 4, 1.0)
    indices[0, 1, 2] = 64
    x.requires_grad_(True)
    loss = distill_loss(x, values, indices, reduction="none")
    assert torch.isnan(loss[0, 1]) and torch.isfinite(loss[0, [0, 2]]).all()
    grad, = torch.autograd.grad(loss.sum(), x)
    assert torch.isfinite(grad[0, [0, 2]]).all() and torch.isnan(grad[0, 1]).all()


@pytest.mark.parametrize("device", CPU_GPU)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("t", [1.0, 2.0])
def test_distill_rows_of_extreme_logits(device, dtype, t):
    """Rows of the type's lowest or largest value: uniform ones, and not sums of
    1e38 that cancel to 1e22. A place far below the others counts by its own
    probability, however small beside the sum of them."""
    need(device)
    V = 300
    fi = torch.finfo(dtype)
    x = make_logits(1, 4, V, dtype, "cpu")
    x[0, 0], x[0, 1] = fi.min, fi.max
    x[0, 2, 100:] = fi.max
    x[0, 3] = 0.0
    x[0, 3, 7] = fi.max
    g = torch.Generator().manual_seed(6)
    values = torch.randn(1, 4, 9, generator=g).to(dtype)
    indices = torch.stack([torch.randperm(180, generator=g)[:9] + 110 for _ in range(4)])[None]
    values[0, 3, 0], indices[0, 3, 0] = 55.0, 7
    lse = torch.logsumexp(values.double() / t, -1).float() + 0.4
    x, values, indices, lse = (a.to(device) for a in (x, values, indices, lse))
    for r in range(4):
        each = x[:, r:r + 1], values[:, r:r + 1], indices[:, r:r + 1]
        check_distill(*each, None, t)
        if r < 3:  # the last row's rest is as impossible as its places
            check_distill(*each, lse[:, r:r + 1], t)


@pytest.mark.parametrize("device", CPU_GPU)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("t", [0.3, 0.05])
def test_distill_extreme_logits_at_low_temperatures(device, dtype, t):
    """The type's lowest and largest values, which a division by a temperature
    below 1 takes past the largest number."""
    need(device)
    V = 300
    fi = torch.finfo(dtype)
    x = make_logits(1, 4, V, dtype, "cpu", scale=0.3)
    x[0, 0], x[0, 1] = fi.min, fi.max
    x[0, 2, 100:] = fi.max
    x[0, 3, :100] = fi.min
    g = torch.Generator().manual_seed(6)
    values = (torch.randn(1, 4, 9, generator=g) * t).to(dtype)
    indices = torch.stack([torch.randperm(180, generator=g)[:9] + 110 for _ in range(4)])[None]
    lse = torch.logsumexp(values.double() / t, -1).float() + 0.4
    args = [a.to(device) for a in (x, values, indices)]
    check_distill(*args, None, t)
    check_distill(*args, lse.to(device), t)


@pytest.mark.parametrize("device", CPU_GPU)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("t", [0.3, 1.0])
def test_distill_places_far_apart(device, dtype, t):
    """A masked logit in the record costs its own probability's worth, not
    infinity; below a logit of the largest value the others keep their shares."""
    need(device)
    V = 300
    fi = torch.finfo(dtype)
    x = make_logits(1, 2, V, dtype, "cpu")
    values, indices, _ = make_record(x, 9, t, tail=False)
    lse = torch.logsumexp(values.double() / t, -1).float() + 0.4
    x[0, 0, indices[0, 0, 3]] = fi.min
    values[0, 0, 3] = -200.0 * t
    args = [a.to(device) for a in (x, values, indices)]
    check_distill(*[a[:, :1] for a in args], None, t)
    check_distill(*[a[:, :1] for a in args], lse[:, :1].to(device), t)
    x[0, 1, indices[0, 1, 0]] = fi.max  # all the student's mass is on one place
    y = x[:, 1:].to(device).requires_grad_(True)
    loss = distill_loss(y, values[:, 1:].to(device), indices[:, 1:].to(device),
                        lse[:, 1:].to(device), temperature=t)
    got, = torch.autograd.grad(loss, y, torch.tensor(64.0, device=device))
    p = (values[0, 1].double() / t - lse[0, 1].double()).exp()
    rest, out = 1 - p.sum(), x[0, 1].double().index_fill(0, indices[0, 1], -math.inf)
    want = -rest * torch.softmax(out / t, -1)
    want[indices[0, 1]] = -p
    want[indices[0, 1, 0]] += 1.0
    assert torch.isfinite(loss)
    # sums of a place's p and the rest's share: as any gradient, q being the shares
    check_grad(got[0], want[None] * 64.0 * t, torch.tensor([64.0 * t]), want.abs()[None])


@pytest.mark.parametrize("device", CPU_GPU)
@pytest.mark.parametrize("tail", [False, True])
def test_distill_unlikely_index_outside_is_nan(device, tail):
    """An index outside the row is one however small its probability; a value
    of -inf there has none."""
    need(device)
    x = make_logits(1, 4, 64, torch.float32, device)
    values, indices, lse = make_record(x, 4, 1.0, tail=tail)
    indices[0, 1:, 2] = 64
    values[0, 1, 2] = -1e4  # exp of it is 0 in 64 bits too
    values[0, 2, 2] = float("-inf")
    values[0, 3] = torch.tensor([3.0, 2.0, -1e30, 1.0], device=device)
    x.requires_grad_(True)
    loss = distill_loss(x, values, indices, lse, reduction="none")
    grad, = torch.autograd.grad(loss.sum(), x)
    assert torch.isfinite(loss[0, [0, 2]]).all() and torch.isfinite(grad[0, [0, 2]]).all()
    assert torch.isnan(loss[0, [1, 3]]).all() and torch.isnan(grad[0, [1, 3]]).any(-1).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V,k", [(1, 1), (65, 65), (601, 200), (2047, 100), (4100, 3)])
def test_many_short_rows(dtype, V, k):
    """Rows that a wave each reads, some masked, in a slice that starts anywhere."""
    need("cuda")
    R = 2049
    x = make_logits(1, R, V + 3, dtype, "cuda")[..., 1:V + 1]
    g = torch.Generator().manual_seed(6)
    mask = (torch.rand(1, R, generator=g) < 0.8).to("cuda")
    up = torch.randn(1, R, generator=g).to("cuda") * (64.0 if dtype == torch.float16 else 1.0)
    check_policy(x, *make_rollout(x), mask, reduction="none", up=up)
    values, indices, lse = make_record(x, k, 1.5)
    x[0, ~mask[0]] = float("nan")
    check_distill(x, values, indices, lse, 1.5, mask, "none", up)
    check_distill(x, values, indices, None, 1.5, mask, "none", up)


# ------------------------------------------------------------------ preference
def preference_oracle(logits, targets, ref, beta, eps, ignore):
    N = logits.shape[0] // 2
    lq = softmax64(logits)
    tg = targets.cpu().long()
    keep = tg != ignore
    lp = torch.where(keep, lq.gather(-1, tg.clamp_min(0)[..., None])[..., 0], 0.0)
    r = beta * (lp.sum(-1) - ref.cpu().double())
    z = r[:N] - r[N:]
    loss = -((1 - eps) * torch.nn.functional.logsigmoid(z) + eps * torch.nn.functional.logsigmoid(-z))
    by_z = eps - torch.sigmoid(-z)  # sigmoid(z) - (1 - eps)
    a = beta * torch.cat([by_z, -by_z])[:, None] * keep
    one = torch.zeros_like(lq).scatter_(-1, tg.clamp_min(0)[..., None], 1.0)
    grad = torch.where(a[..., None] != 0, a[..., None] * (one - lq.exp()), 0.0)
    return loss, r, grad, a, lq.exp()


def check_preference(logits, targets, ref, beta=0.1, eps=0.0, ignore=-100, reduction="mean", up=None):
    x = logits.detach().requires_grad_(True) if logits.is_leaf else logits
    out = preference_loss(x, targets, ref, beta=beta, label_smoothing=eps, ignore_index=ignore,
                          reduction=reduction)
    rows, r, grad, a, q = preference_oracle(logits, targets, ref, beta, eps, ignore)
    N, T = len(rows), targets.shape[1]
    want = {"mean": rows.mean(), "sum": rows.sum(), "none": rows}[reduction]
    lim = 2 * beta * T * LP
    torch.testing.assert_close(out.loss.detach().cpu().double(), want, rtol=2.0 ** -22,
                               atol=lim * (N if reduction == "sum" else 1))
    rewards = torch.cat([out.chosen_rewards, out.rejected_rewards])
    torch.testing.assert_close(rewards.cpu().double(), r, rtol=2.0 ** -22, atol=lim)
    assert not rewards.requires_grad
    up = torch.ones_like(out.loss) if up is None else up
    got, = torch.autograd.grad(out.loss, x, up)
    u = up.cpu().double()
    each = u.repeat(2)[:, None] if reduction == "none" else u / (N if reduction == "mean" else 1)
    # the coefficient moves by lim of z's error beside the rounding of q
    slack = (lim / GRAD + 1) if lim > GRAD else 2
    check_grad(got, grad * each[..., None], a * each * slack, q + (q * 0 + grad.abs() / a.abs().clamp_min(1e-300)[..., None]) * (a != 0)[..., None])
    assert (got.cpu()[(targets == ignore).cpu()] == 0).all()
    return out, got


def make_pairs(N, T, V, device, seed=2):
    g = torch.Generator().manual_seed(seed)
    targets = torch.randint(0, V, (2 * N, T), generator=g)
    lengths = torch.randint(0, T + 1, (2 * N, 1), generator=g)
    targets = torch.where(torch.arange(T)[None] < lengths, targets, -100)
    ref = torch.randn(2 * N, generator=g) * 5 - 10.0 * (targets >= 0).sum(-1)
    return targets.to(device), ref.to(device)


@pytest.mark.parametrize("device", CPU_GPU)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_preference(device, dtype, shape):
    need(device)
    B, T, V = shape
    x = make_logits(2 * B, T, V, dtype, device)
    targets, ref = make_pairs(B, T, V, device)
    scale = 512.0 if dtype == torch.float16 else 1.0
    check_preference(x, targets, ref, eps=0.1 if B > 1 else 0.0,
                     up=torch.tensor(scale, device=device))


@pytest.mark.parametrize("device", CPU_GPU)
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_preference_reductions_and_layouts(device, reduction):
    need(device)
    x = make_logits(6, 6, 515, torch.float32, device)
    targets, ref = make_pairs(3, 5, 512, device)
    up = torch.tensor([0.5, -2.0, 3.0] if reduction == "none" else 1.75, device=device)
    for view in (x[:, :-1, :], x[:, 1:, :512], x[:, :5, 3:],
                 x[:, 1:].transpose(0, 1).contiguous().transpose(0, 1)):
        check_preference(view, targets, ref.double(), reduction=reduction, up=up)
    # another ignored index, whose token is a real one; int32 targets
    targets[:, 0] = 7
    check_preference(x[:, 1:], targets.clamp_min(0).int(), ref, ignore=7, reduction=reduction, up=up)


@pytest.mark.parametrize("device", CPU_GPU)
def test_preference_masked_rows_hold_anything(device):
    need(device)
    x = make_logits(4, 5, 130, torch.float32, device)
    targets, ref = make_pairs(2, 5, 130, device, seed=11)
    targets[0] = -100  # an answer of no tokens
    want, grad = check_preference(x, targets, ref)
    bad = x.clone()
    bad[targets == -100] = float("nan")
    bad.requires_grad_(True)
    got = preference_loss(bad, targets, ref)
    assert torch.equal(got.loss.detach(), want.loss.detach())
    g, = torch.autograd.grad(got.loss, bad)
    assert torch.equal(g, grad)


@pytest.mark.parametrize("device", CPU_GPU)
def test_preference_far_margins(device):
    """sigmoid and its logarithm far out: no overflow, no 0 * inf."""
    need(device)
    x = make_logits(4, 3, 64, torch.float32, device)
    targets = torch.zeros(4, 3, dtype=torch.int64, device=device)
    ref = torch.tensor([-1e6, 1e6, 0.0, 0.0], device=device)
    check_preference(x, targets, ref, reduction="none")
    # z = 40 and -40: a pair that is all but settled has a gradient of e^-40
    lp = softmax64(x)[..., 0].sum(-1)
    ref = lp - torch.tensor([400.0, -400.0, 0.0, 0.0], dtype=torch.float64)
    y = x.clone().requires_grad_(True)
    out = preference_loss(y, targets, ref.to(device), reduction="none")
    grad, = torch.autograd.grad(out.loss.sum(), y)
    want = [0.1 * math.exp(-40.0), 0.1]
    for pair in range(2):
        for row in (pair, pair + 2):
            a = grad[row, 0, 0].item() / (softmax64(x)[row, 0, 0].exp().item() - 1)
            a = a if row < 2 else -a
            # z is off by 6 LP of its rewards
            assert abs(a / want[pair] - 1) < 6 * LP + GRAD, (row, a)


@pytest.mark.parametrize("device", CPU_GPU)
def test_preference_impossible_answers(device):
    """A token whose logit is -inf: an impossible rejected answer costs
    nothing, an impossible chosen one everything, and neither is a NaN."""
    need(device)
    x = make_logits(4, 3, 64, torch.float32, device)
    x[[1, 2], 1, 5] = float("-inf")
    x.requires_grad_(True)
    targets = torch.full((4, 3), 5, device=device)
    out = preference_loss(x, targets, torch.zeros(4, device=device), reduction="none")
    assert out.loss.tolist() == [0.0, math.inf]
    assert out.rejected_rewards[0].item() == out.chosen_rewards[1].item() == -math.inf
    grad, = torch.autograd.grad(out.loss.sum(), x)
    assert (grad[[0, 2]] == 0).all() and torch.isfinite(grad[3]).all() and grad[3].abs().sum() > 0


@pytest.mark.parametrize("device", CPU_GPU)
def test_preference_target_outside_is_nan(device):
    need(device)
    x = make_logits(4, 3, 64, torch.float32, device).requires_grad_(True)
    targets = torch.zeros(4, 3, dtype=torch.int64, device=device)
    targets[1, 2] = 64
    targets[2, 0] = -7
    out = preference_loss(x[:2], targets[:2], torch.zeros(2, device=device), reduction="none")
    assert torch.isnan(out.loss).all()
    out = preference_loss(x[2:], targets[2:], torch.zeros(2, device=device), reduction="none")
    assert torch.isnan(out.loss).all()


# ---------------------------------------------------------------------- policy
def policy_oracle(logits, actions, old, adv, ref, mask, low, high, coef):
    lq = softmax64(logits)
    act = actions.cpu().long()
    live = torch.ones(act.shape, dtype=torch.bool) if mask is None else mask.cpu()
    lp = torch.where(live, lq.gather(-1, act[..., None])[..., 0], 0.0)
    A = torch.where(live, adv.cpu(), 0).double()
    ratio = (lp - torch.where(live, old.cpu(), 0).double()).exp()
    held = ratio.clamp(1 - low, 1 + high)
    loss = -torch.minimum(ratio * A, held * A)
    moves = torch.where(A > 0, ratio <= 1 + high, ratio >= 1 - low)
    by_lp = torch.where(moves, -A * ratio, 0.0)
    kl = torch.zeros_like(lp)
    if ref is not None:
        d = torch.where(live, ref.cpu(), 0).double() - lp
        kl = torch.expm1(d) - d
        loss = loss + coef * kl
        by_lp = by_lp - coef * torch.expm1(d)
    by_lp = by_lp * live
    one = torch.zeros_like(lq).scatter_(-1, act[..., None], 1.0)
    grad = torch.where(by_lp[..., None] != 0, by_lp[..., None] * (one - lq.exp()), 0.0)
    return loss * live, lp, kl * live, grad, by_lp, lq.exp(), live


def make_rollout(logits, seed=4, spread=0.3):
    """Old log-probabilities that keep 1e-3 from the borders of the clip."""
    g = torch.Generator().manual_seed(seed)
    rows = logits.shape[:-1]
    actions = torch.randint(0, logits.shape[-1], rows, generator=g)
    lp = softmax64(logits).gather(-1, actions[..., None])[..., 0]
    moved = torch.randn(rows, generator=g).double() * spread
    for border in (math.log(1.2), math.log(0.8), math.log(1.3)):
        moved = torch.where((moved - border).abs() < 1e-3, moved + 4e-3, moved)
    adv = torch.randn(rows, generator=g)
    ref = (lp + torch.randn(rows, generator=g) * 0.3).float()
    return [a.to(logits.device) for a in (actions, (lp - moved).float(), adv, ref)]


def check_policy(logits, actions, old, adv, ref, mask=None, low=0.2, high=0.2, coef=0.05,
                 reduction="mean", up=None):
    x = logits.detach().requires_grad_(True) if logits.is_leaf else logits
    out = policy_loss(x, actions, old, adv, ref, mask=mask, clip_low=low, clip_high=high,
                      kl_coef=coef, reduction=reduction)
    rows, lp, kl, grad, by_lp, q, live = policy_oracle(logits, actions, old, adv, ref, mask,
                                                       low, high, coef)
    n = max(int(live.sum()), 1)
    want = {"mean": rows.sum() / n, "sum": rows.sum(), "none": rows}[reduction]
    # a ratio of at most e^2 * |A| <= 5 and an exp(d) of at most e^2: 50 LP
    lim = 50 * LP * (n if reduction == "sum" else 1)
    torch.testing.assert_close(out.loss.detach().cpu().double(), want, rtol=2.0 ** -22, atol=lim)
    torch.testing.assert_close(out.logps.cpu().double(), lp, rtol=2.0 ** -23, atol=LP)
    torch.testing.assert_close(out.kl.cpu().double(), kl, rtol=2.0 ** -22, atol=10 * LP)
    assert not out.logps.requires_grad and not out.kl.requires_grad
    up = torch.ones_like(out.loss) if up is None else up
    got, = torch.autograd.grad(out.loss, x, up)
    u = up.cpu().double()
    each = u if reduction == "none" else u / (n if reduction == "mean" else 1)
    each = each * torch.ones_like(by_lp)
    # the terms of by_lp may cancel: its error is that of the larger ones
    big = (by_lp.abs() + (adv.cpu().double().abs() * 2 + coef * 3) * live) * each.abs()
    check_grad(got, grad * each[..., None], big, q + (1 - q) * (grad != 0))
    assert (got.cpu()[by_lp == 0] == 0).all()
    return out, got


@pytest.mark.parametrize("device", CPU_GPU)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_policy(device, dtype, shape):
    need(device)
    B, T, V = shape
    x = make_logits(B, T, V, dtype, device)
    actions, old, adv, ref = make_rollout(x)
    mask = None
    if B > 1:
        mask = (torch.arange(T)[None] < torch.randint(1, T + 1, (B, 1),
                                                      generator=torch.Generator().manual_seed(5)))
        mask = mask.to(device)
    scale = 512.0 if dtype == torch.float16 else 1.0
    check_policy(x, actions, old, adv, ref if T > 1 else None, mask, coef=0.05 if T > 1 else 0.0,
                 up=torch.tensor(scale, device=device))


def check_policy_grad(got, grad, by_lp, big, q, actions):
    """got against ``grad`` = by_lp (onehot - q). An error of by_lp, at most
    GRAD of ``big``, moves a place by |onehot - q| of it, one of q by q of it:
    1 - q is allowed at the action alone."""
    one = torch.zeros_like(q).scatter_(-1, actions.cpu().long()[..., None], 1.0)
    check_grad(got, grad, big, (one - q).abs() + q)
    assert (got.cpu()[by_lp == 0] == 0).all()


@pytest.mark.parametrize("device", CPU_GPU)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_policy_gradient_of_every_logit(device, dtype, shape):
    """The gradient of the sum, so that the small ones are no denormals."""
    need(device)
    B, T, V = shape
    base = make_logits(B, T, V + 2, dtype, device)
    up = 512.0 if dtype == torch.float16 else 1.0
    for view in (base[..., :V].contiguous(), base[..., 1:V + 1]):
        actions, old, adv, ref = make_rollout(view)
        x = view.detach().requires_grad_(True)
        out = policy_loss(x, actions, old, adv, ref, kl_coef=0.05, reduction="sum")
        got, = torch.autograd.grad(out.loss, x, torch.tensor(up, device=device))
        _, _, _, grad, by_lp, q, _ = policy_oracle(view, actions, old, adv, ref, None, 0.2, 0.2, 0.05)
        big = by_lp.abs() + adv.cpu().double().abs() * 2 + 0.05 * 3
        check_policy_grad(got, grad * up, by_lp, big * up, q, actions)


@pytest.mark.parametrize("V", [613, 4099, 30522, 128256])
def test_policy_gradient_check_sees_small_probabilities(V):
    """The check itself: a gradient that lacks what is below q = 1e-4, or one
    place of it, is not accepted."""
    x = make_logits(1, 3, V, torch.float32, "cpu")
    actions, old, adv, ref = make_rollout(x)
    _, _, _, grad, by_lp, q, _ = policy_oracle(x, actions, old, adv, ref, None, 0.2, 0.2, 0.05)
    assert (by_lp != 0).all()  # no row is clipped
    big = by_lp.abs() + adv.double().abs() * 2 + 0.05 * 3
    right = (grad, by_lp, big, q, actions)
    check_policy_grad(grad.float(), *right)
    away = torch.ones_like(q, dtype=torch.bool).scatter_(-1, actions[..., None], False)
    for lost in (away & (q < 1e-4), away & (torch.arange(V) == V - 1)):
        assert lost.any()
        with pytest.raises(AssertionError):
            check_policy_grad(grad.masked_fill(lost, 0.0).float(), *right)


@pytest.mark.parametrize("device", CPU_GPU)
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_policy_reductions_and_layouts(device, reduction):
    need(device)
    x = make_logits(3, 7, 515, torch.float32, device)
    for view in (x[:, :-1], x[:, 1:, :512], x[:, :6, 3:], x[0, 1:], x[1, 2],
                 x.transpose(0, 1)[1:], x[:, :6].reshape(3, 2, 3, 515)):
        actions, old, adv, ref = make_rollout(view)
        up = torch.randn(adv.shape if reduction == "none" else (),
                         generator=torch.Generator().manual_seed(1)).to(device)
        check_policy(view, actions.int(), old, adv, ref, low=0.2, high=0.3, reduction=reduction,
                     up=up)


@pytest.mark.parametrize("device", CPU_GPU)
def test_policy_masks(device):
    need(device)
    x = make_logits(2, 5, 130, torch.float32, device)
    actions, old, adv, ref = make_rollout(x)
    mask = torch.tensor([[1, 1, 0, 0, 1], [0, 0, 0, 0, 0]], dtype=torch.bool, device=device)
    want, grad = check_policy(x, actions, old, adv, ref, mask)
    for t in (x, old, adv, ref):
        t[~mask] = float("nan")
    actions[~mask] = -100
    x.requires_grad_(True)
    got = policy_loss(x, actions, old, adv, ref, mask=mask, kl_coef=0.05)
    g, = torch.autograd.grad(got.loss, x)
    assert torch.equal(got.loss.detach(), want.loss.detach()) and torch.equal(g, grad)
    assert torch.equal(got.kl, want.kl) and torch.equal(got.logps, want.logps)
    none = policy_loss(x, actions, old, adv, ref, mask=torch.zeros_like(mask), kl_coef=0.05)
    assert none.loss.item() == 0.0
    g, = torch.autograd.grad(none.loss, x)
    assert (g == 0).all()


@pytest.mark.parametrize("device", CPU_GPU)
def test_policy_impossible_old_tokens(device):
    """An old log-probability of -inf, or one far below: the ratio passes the
    largest number, the clip holds the loss and the gradient is 0. Where the
    advantage is negative nothing holds it."""
    need(device)
    x = make_logits(1, 6, 33, torch.float32, device)
    actions, old, adv, ref = make_rollout(x)
    old[0, 1], old[0, 2], old[0, 4] = float("-inf"), -1e30, -900.0
    adv[0] = torch.tensor([1.0, 0.5, 2.0, -1.0, 1.5, 1.0])
    check_policy(x, actions, old, adv, None, coef=0.0)
    check_policy(x, actions, old, adv, ref, coef=0.05, reduction="sum")
    adv[0, 1] = -0.5
    x.requires_grad_(True)
    out = policy_loss(x, actions, old, adv, reduction="none")
    assert out.loss[0, 1].item() == float("inf") and torch.isfinite(out.loss[0, 2:]).all()
    g, = torch.autograd.grad(out.loss.sum(), x)
    assert not torch.isfinite(g[0, 1]).any() and torch.isfinite(g[0, 2:]).all()


@pytest.mark.parametrize("device", CPU_GPU)
def test_policy_nan_advantage_is_nan(device):
    """A NaN advantage makes its token's loss a NaN, and its gradient with it,
    on whichever side of the clip the ratio lies."""
    need(device)
    x = make_logits(1, 4, 33, torch.float32, device)
    actions, old, adv, _ = make_rollout(x, spread=0.0)
    old = old - torch.tensor([0.0, 2.0, -2.0, 0.0], device=device)
    adv[0, :3] = float("nan")
    x.requires_grad_(True)
    out = policy_loss(x, actions, old, adv, reduction="none")
    g, = torch.autograd.grad(out.loss.sum(), x)
    assert torch.isnan(out.loss[0, :3]).all() and torch.isfinite(out.loss[0, 3])
    assert torch.isnan(g[0, :3]).all() and torch.isfinite(g[0, 3]).all()


@pytest.mark.parametrize("device", CPU_GPU)
def test_policy_kl_without_weight(device):
    """With a coefficient of 0 the KL is reported only, and one that passes the
    largest number changes neither loss nor gradient."""
    need(device)
    x = make_logits(1, 4, 64, torch.float32, device)
    actions = torch.tensor([[3, 9, 20, 63]], device=device)
    x[0, 1, 9] = -1000.0  # exp(999) is none in 64 bits either
    x[0, 2, 20] = torch.finfo(torch.float32).min
    old = softmax64(x).gather(-1, actions.cpu()[..., None])[..., 0].float().to(device)
    adv = torch.tensor([[1.0, -0.5, 2.0, -1.0]], device=device)
    ref = torch.full((1, 4), -1.0, device=device)
    x.requires_grad_(True)
    for reduction in ("none", "mean"):
        got = policy_loss(x, actions, old, adv, ref, kl_coef=0.0, reduction=reduction)
        want = policy_loss(x, actions, old, adv, reduction=reduction)
        assert torch.isfinite(want.loss).all() and torch.equal(got.loss, want.loss)
        a, b = (torch.autograd.grad(o.loss.sum(), x)[0] for o in (got, want))
        assert torch.isfinite(b).all() and torch.equal(a, b)
        assert torch.isinf(got.kl[0, 1:3]).all() and torch.isfinite(got.kl[0, [0, 3]]).all()


@pytest.mark.parametrize("device", CPU_GPU)
@pytest.mark.parametrize("dtype", TYPES)
def test_masked_logits(device, dtype):
    """-inf (a padded head) and the type's lowest value in a row: no gradient
    there, none lost elsewhere; a row of the lowest value alone is uniform."""
    need(device)
    x = make_logits(2, 3, 600, dtype, device)
    x[..., 500:] = float("-inf")
    x[1, ..., 400:500] = torch.finfo(dtype).min
    x[1, 2] = torch.finfo(dtype).min
    actions = torch.randint(0, 400, (2, 3), generator=torch.Generator().manual_seed(8)).to(device)
    old = softmax64(x).gather(-1, actions.cpu()[..., None])[..., 0].float().to(device)
    adv = torch.ones(2, 3, device=device)
    _, grad = check_policy(x, actions, old, adv, None, coef=0.0)
    assert (grad[0, :, 500:] == 0).all()


@pytest.mark.parametrize("device", CPU_GPU)
def test_policy_action_outside_and_bad_logits_are_nan(device):
    need(device)
    x = make_logits(1, 6, 64, torch.float32, device)
    x[0, 2, 5] = float("nan")
    x[0, 3, 5] = float("inf")
    x[0, 4] = float("-inf")
    x.requires_grad_(True)
    actions = torch.tensor([[64, -1, 3, 3, 3, 3]], device=device)
    zero = torch.zeros(1, 6, device=device)
    out = policy_loss(x, actions, zero, zero + 1, reduction="none")
    assert torch.isnan(out.loss[0, :5]).all() and torch.isfinite(out.loss[0, 5])
    g, = torch.autograd.grad(out.loss.sum(), x)
    assert torch.isnan(g[0, :5]).any(-1).all() and torch.isfinite(g[0, 5]).all()


# ------------------------------------------------------ gradients by differences
def test_gradients_by_differences():
    """The CPU definitions that the kernels are held to, in float64."""
    x = make_logits(4, 3, 11, torch.float64, "cpu", scale=1.0).requires_grad_(True)
    values, indices, lse = make_record(x, 4, 1.5)
    values = values.detach()
    for record in ((values, indices), (values, indices, lse.double())):
        assert torch.autograd.gradcheck(
            lambda y: distill_loss(y, *record, temperature=1.5), (x,))
    targets, ref = make_pairs(2, 3, 11, "cpu")
    assert torch.autograd.gradcheck(lambda y: preference_loss(
        y, targets, ref, label_smoothing=0.1).loss, (x,))
    actions, old, adv, kref = make_rollout(x)
    assert torch.autograd.gradcheck(lambda y: policy_loss(
        y, actions, old, adv, kref, kl_coef=0.1).loss, (x,))


@pytest.mark.gpu
def test_kernel_gradients_by_differences():
    """The kernels' own loss moves as their own gradient says. Central
    differences of step h along a direction: off by h^2 times a third
    derivative (< 1) and by two losses' rounding, 4 LP, over 2 h."""
    need("cuda")
    h = 0.05
    x = make_logits(4, 3, 203, torch.float32, "cuda", scale=1.0)
    d = make_logits(4, 3, 203, torch.float32, "cuda", seed=9, scale=1.0)
    d /= d.norm()
    values, indices, lse = make_record(x, 7, 1.0)
    targets, ref = make_pairs(2, 3, 203, "cuda")
    actions, old, adv, kref = make_rollout(x, spread=0.05)
    for fn in (lambda y: distill_loss(y, values, indices),
               lambda y: distill_loss(y, values, indices, lse),
               lambda y: preference_loss(y, targets, ref).loss,
               lambda y: policy_loss(y, actions, old, adv, kref, kl_coef=0.1, clip_low=0.9,
                                     clip_high=9.0).loss):
        y = x.clone().requires_grad_(True)
        g, = torch.autograd.grad(fn(y), y)
        slope = (g * d).sum().item()
        with torch.no_grad():
            moved = (fn(x + h * d).item() - fn(x - h * d).item()) / (2 * h)
        assert abs(moved - slope) <= h * h + 4 * LP / (2 * h), (moved, slope)


# -------------------------------------------------------------------- refusals
@pytest.mark.parametrize("device", CPU_GPU)
def test_refusals(device):
    need(device)
    x = make_logits(2, 3, 40, torch.float32, device)
    values, indices, lse = make_record(x, 4, 1.0)
    targets = torch.zeros(2, 3, dtype=torch.int64, device=device)
    rows = torch.zeros(2, 3, device=device)
    ref = torch.zeros(2, device=device)
    bad = [
        lambda: topk_logits(x, 0), lambda: topk_logits(x, 41),
        lambda: topk_logits(x.int(), 2), lambda: topk_logits(x, 2, 0.0),
        lambda: topk_logits(make_logits(1, 1, 400, torch.float32, device), 257),
        lambda: topk_logits(torch.zeros((), device=device), 1),
        lambda: topk_logits(x, 2, float("nan")),
        lambda: distill_loss(x, values, indices, temperature=-1.0),
        lambda: distill_loss(x, values, indices, reduction="max"),
        lambda: distill_loss(x, values[:, :2], indices),
        lambda: distill_loss(x, values, indices[..., :3]),
        lambda: distill_loss(x, values, indices.float()),
        lambda: distill_loss(x, indices, indices),
        lambda: distill_loss(x, values, indices, lse[:1]),
        lambda: distill_loss(x, values, indices, mask=rows),
        lambda: distill_loss(x, values, indices, mask=torch.ones(3, dtype=torch.bool, device=device)),
        lambda: distill_loss(x, values.clone().requires_grad_(True), indices),
        lambda: distill_loss(x, values[..., :0], indices[..., :0]),
        lambda: distill_loss(x, torch.zeros(2, 3, 257, device=device),
                             torch.zeros(2, 3, 257, dtype=torch.int64, device=device)),
        lambda: preference_loss(x[0], targets[0], ref),
        lambda: preference_loss(x[:1], targets[:1], ref[:1]),
        lambda: preference_loss(x, targets[:, :2], ref),
        lambda: preference_loss(x, targets.float(), ref),
        lambda: preference_loss(x, targets, ref[:1]),
        lambda: preference_loss(x, targets, ref.long()),
        lambda: preference_loss(x, targets, ref, beta=0.0),
        lambda: preference_loss(x, targets, ref, label_smoothing=0.5),
        lambda: preference_loss(x, targets, ref.clone().requires_grad_(True)),
        lambda: preference_loss(x[:, :0], targets[:, :0], ref),
        lambda: policy_loss(x, targets, rows[:1], rows),
        lambda: policy_loss(x, targets.bool(), rows, rows),
        lambda: policy_loss(x, targets, rows, rows, kl_coef=0.1),
        lambda: policy_loss(x, targets, rows, rows, clip_low=1.0),
        lambda: policy_loss(x, targets, rows, rows, clip_high=-0.1),
        lambda: policy_loss(x, targets, rows, rows, rows, kl_coef=-1.0),
        lambda: policy_loss(x, targets, rows, rows.clone().requires_grad_(True)),
        lambda: policy_loss(x, targets, rows, rows, mask=targets),
    ]
    if device == "cuda":
        bad += [lambda: topk_logits(x[0, 0, :1].expand(1 << 22, 1), 1),
                lambda: topk_logits(x.double(), 2),
                lambda: policy_loss(x, targets.cpu(), rows, rows),
                lambda: preference_loss(x, targets, ref.cpu()),
                lambda: distill_loss(x, values.cpu(), indices)]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")


@pytest.mark.parametrize("device", CPU_GPU)
def test_no_rows(device):
    need(device)
    x = torch.zeros(0, 3, 40, device=device, requires_grad=True)
    rows = torch.zeros(0, 3, device=device)
    ids = torch.zeros(0, 3, dtype=torch.int64, device=device)
    record = torch.zeros(0, 3, 2, device=device), torch.zeros(0, 3, 2, dtype=torch.int64, device=device)
    for loss in (distill_loss(x, *record), policy_loss(x, ids, rows, rows).loss,
                 policy_loss(x, ids, rows, rows, reduction="sum").loss):
        assert loss.item() == 0.0
        g, = torch.autograd.grad(loss, x)
        assert g.shape == x.shape
    assert distill_loss(x, *record, reduction="none").shape == (0, 3)


# ----------------------------------------------------- streams, graphs, memory
def all_losses(x, pairs, rollout, record, lse):
    return (distill_loss(x, *record, lse, temperature=2.0),
            preference_loss(x, *pairs).loss,
            policy_loss(x, *rollout, kl_coef=0.05).loss)


@pytest.mark.gpu
def test_same_bits_again_and_backward_twice():
    need("cuda")
    x = make_logits(4, 37, 5003, torch.bfloat16, "cuda").requires_grad_(True)
    values, indices, lse = make_record(x, 9, 2.0)
    pairs, rollout = make_pairs(2, 37, 5003, "cuda"), make_rollout(x)
    first = None
    for _ in range(3):
        losses = all_losses(x, pairs, rollout, (values, indices), lse)
        grads = [torch.autograd.grad(l, x, retain_graph=True)[0] for l in losses]
        again = [torch.autograd.grad(l, x)[0] for l in losses]
        now = [l.detach() for l in losses] + grads
        assert all(torch.equal(a, b) for a, b in zip(grads, again))
        assert first is None or all(torch.equal(a, b) for a, b in zip(first, now))
        first = now


@pytest.mark.gpu
def test_gradient_reaches_views_and_accumulates():
    need("cuda")
    base = make_logits(4, 6, 515, torch.float32, "cuda").requires_grad_(True)
    targets, ref = make_pairs(2, 5, 512, "cuda")
    for _ in range(2):
        preference_loss(base[:, :-1, :512], targets, ref).loss.backward()
    _, _, grad, _, _ = preference_oracle(base[:, :-1, :512], targets, ref, 0.1, 0.0, -100)
    assert (base.grad[:, -1] == 0).all() and (base.grad[..., 512:] == 0).all()
    torch.testing.assert_close(base.grad[:, :-1, :512].cpu().double(), grad, rtol=1e-3, atol=1e-6)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_rows_of_several_segments(dtype):
    """A vocabulary that no single block takes, beside many short rows."""
    need("cuda")
    scale = 512.0 if dtype == torch.float16 else 1.0
    for B, T, V in ((1, 2, 300001), (6, 301, 97)):
        x = make_logits(B, T, V, dtype, "cuda")
        up = torch.tensor(scale, device="cuda")
        values, indices, lse = make_record(x, 40, 2.0)
        check_distill(x, values, indices, lse, 2.0, up=up)
        check_distill(x, values, indices, None, 2.0, up=up)
        check_policy(x, *make_rollout(x), up=up)
        check_preference(x.repeat(2, 1, 1), *make_pairs(B, T, V, "cuda"), up=up)


@pytest.mark.gpu
def test_most_rows():
    """2**22 - 1 rows, the most of a call: as its first 6141, which it repeats."""
    need("cuda")
    n, times, V = 6141, 683, 3
    assert n * times == 2 ** 22 - 1
    base = make_logits(1, n, V, torch.float32, "cuda")
    x = base.repeat(1, times, 1).requires_grad_(True)
    top, want = topk_logits(x, 2), topk_logits(base, 2)
    for got, part in zip(top, want):
        assert torch.equal(got.unflatten(1, (times, n)), part[:, None].expand(
            1, times, n, *part.shape[2:]))
    values, indices, lse = make_record(base, 2, 1.0)
    small, grad = check_distill(base, values, indices, lse, reduction="none")
    loss = distill_loss(x, values.repeat(1, times, 1), indices.repeat(1, times, 1),
                        lse.repeat(1, times), reduction="none")
    got, = torch.autograd.grad(loss.sum(), x)
    for big, part in ((loss, small), (got, grad)):
        # both are within their tolerances of one value
        torch.testing.assert_close(big.detach().unflatten(1, (times, n)),
                                   part[:, None].expand(1, times, *part.shape[1:]),
                                   rtol=2.0 ** -21, atol=4 * LP)
    check_policy(x.detach(), *make_rollout(x.detach()))


@pytest.mark.gpu
def test_no_grad_and_inference_mode():
    need("cuda")
    x = make_logits(4, 9, 515, torch.bfloat16, "cuda").requires_grad_(True)
    values, indices, lse = make_record(x, 5, 2.0)
    args = make_pairs(2, 9, 515, "cuda"), make_rollout(x), (values, indices), lse
    want = [l.item() for l in all_losses(x, *args)]
    for mode in (torch.no_grad, torch.inference_mode):
        with mode():
            got = all_losses(x, *args)
            assert not any(l.requires_grad for l in got)
            assert [l.item() for l in got] == want
            assert topk_logits(x.clone(), 3).values.shape == (4, 9, 3)


@pytest.mark.parametrize("device", CPU_GPU)
def test_records_and_rollouts_of_inference_mode(device):
    """A teacher answers and a rollout is sampled in inference mode; what they
    give trains a model outside of it."""
    need(device)
    x = make_logits(4, 9, 515, torch.float32, device).requires_grad_(True)

    def made():
        record = topk_logits(x.detach() * 1.5, 7, 2.0)
        return make_pairs(2, 9, 515, device), make_rollout(x), record[:2], record[2]

    def step(pairs, rollout, record, lse):
        losses = all_losses(x, pairs, rollout, record, lse)
        return [l.detach() for l in losses] + [torch.autograd.grad(l, x)[0] for l in losses]

    want = step(*made())
    with torch.inference_mode():
        args = made()
    assert args[2][1].is_inference() and args[1][0].is_inference()
    assert all(torch.equal(a, b) for a, b in zip(want, step(*args)))


@pytest.mark.gpu
def test_changed_logits_are_noticed():
    """The gradient is made from the logits that the loss saw, or not at all."""
    need("cuda")
    x = make_logits(1, 3, 64, torch.float32, "cuda").requires_grad_(True)
    values, indices, _ = make_record(x, 4, 1.0)
    y = x * 1.0
    loss = distill_loss(y, values, indices)
    y.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


@pytest.mark.gpu
def test_second_derivative_is_refused():
    need("cuda")
    x = make_logits(1, 3, 64, torch.float32, "cuda").requires_grad_(True)
    values, indices, _ = make_record(x, 4, 1.0)
    loss = distill_loss(x, values, indices)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(loss, x, create_graph=True)


@pytest.mark.gpu
def test_another_stream():
    need("cuda")
    x = make_logits(4, 64, 30522, torch.bfloat16, "cuda").requires_grad_(True)
    values, indices, lse = make_record(x, 9, 2.0)
    pairs, rollout = make_pairs(2, 64, 30522, "cuda"), make_rollout(x)
    want = all_losses(x, pairs, rollout, (values, indices), lse)
    want = [(l.detach(), torch.autograd.grad(l, x)[0]) for l in want]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = all_losses(x, pairs, rollout, (values, indices), lse)
        got = [(l.detach(), torch.autograd.grad(l, x)[0]) for l in got]
        top = topk_logits(x, 5)
    side.synchronize()
    for (a, b), (c, d) in zip(want, got):
        assert torch.equal(a, c) and torch.equal(b, d)
    assert torch.equal(top.indices, topk_logits(x, 5).indices)


@pytest.mark.gpu
def test_two_streams_at_once():
    """Calls that overlap on two streams share nothing."""
    need("cuda")
    sides, want, got = [torch.cuda.Stream() for _ in range(2)], [], [[], []]
    sets = []
    for seed in (0, 1):
        x = make_logits(4, 64, 30522, torch.bfloat16, "cuda", seed=seed).requires_grad_(True)
        values, indices, lse = make_record(x, 9, 2.0, seed=seed)
        sets.append((x, make_pairs(2, 64, 30522, "cuda", seed=seed), make_rollout(x, seed=seed),
                     (values, indices), lse))

    def step(args):
        losses = all_losses(*args)
        grads = [torch.autograd.grad(l, args[0])[0] for l in losses]
        return [l.detach() for l in losses] + grads + list(topk_logits(args[0], 5))

    for args in sets:
        want.append(step(args))
    torch.cuda.synchronize()
    for _ in range(4):
        for i, side in enumerate(sides):
            with torch.cuda.stream(side):
                got[i].append(step(sets[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for out in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(out, want[i]))


@pytest.mark.gpu
def test_two_captured_graphs():
    """Forward and backward in two graphs that share nothing, replayed in turn
    on new inputs with eager calls between."""
    need("cuda")
    graphs, static = [], []
    for seed in (0, 1):
        x = make_logits(4, 21, 4099, torch.bfloat16, "cuda", seed=seed).requires_grad_(True)
        values, indices, lse = make_record(x, 9, 2.0)
        pairs, rollout = make_pairs(2, 21, 4099, "cuda"), make_rollout(x)

        def step(x=x, pairs=pairs, rollout=rollout, record=(values, indices), lse=lse):
            losses = all_losses(x, pairs, rollout, record, lse)
            grads = [torch.autograd.grad(l, x)[0] for l in losses]
            return [l.detach() for l in losses] + grads + list(topk_logits(x.detach(), 5))

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out, step))
        static.append(x)
    for turn in range(4):
        for (graph, out, step), x in zip(graphs, static):
            with torch.no_grad():
                x.copy_(make_logits(4, 21, 4099, torch.bfloat16, "cuda", seed=10 + turn))
            graph.replay()
            torch.cuda.synchronize()
            got = [o.clone() for o in out]
            assert all(torch.equal(a, b) for a, b in zip(got, step()))
            torch.cuda.synchronize()


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """Rows behind 2^31 logits: 4.6 GB of them, with the last rows checked."""
    need("cuda")
    T, V = 18000, 128256
    x = torch.empty(1, T, V, dtype=torch.bfloat16, device="cuda").normal_()
    x.requires_grad_(True)
    actions = torch.randint(0, V, (1, T), device="cuda")
    old = torch.full((1, T), -12.0, device="cuda")
    out = policy_loss(x, actions, old, torch.ones(1, T, device="cuda"), clip_high=1e6,
                      reduction="sum")
    grad, = torch.autograd.grad(out.loss, x)
    top = topk_logits(x, 3)
    for r in (0, 9000, 16744, 17999):
        row = x.detach()[0, r].double()
        lq = torch.log_softmax(row, -1)
        lp = lq[actions[0, r]]
        assert abs(out.logps[0, r].item() - lp.item()) <= LP + 2.0 ** -20
        a = (lp + 12.0).exp()
        want = a * lq.exp()
        want[actions[0, r]] -= a
        check_grad(grad[0, r], want, a, lq.exp().cpu())
        assert torch.equal(top.values[0, r], row.topk(3).values.bfloat16())


# ------------------------------------------------------------- used together
@pytest.mark.parametrize("device", CPU_GPU)
@pytest.mark.parametrize("tail", [False, True])
def test_station_learns_from_a_record(device, tail):
    """A teacher's record of its own answers pulls a student's logits to the
    teacher's: the gradient vanishes at the teacher and points there elsewhere."""
    need(device)
    g = torch.Generator().manual_seed(0)
    h = torch.randn(2, 6, 16, generator=g).to(device)
    wt = torch.randn(64, 16, generator=g).to(device)
    teacher = h @ wt.t()
    record = topk_logits(teacher, 64, 2.0)
    lse = record.logsumexp if tail else None
    w = wt.clone().requires_grad_(True)
    loss = distill_loss(h @ w.t(), record.values, record.indices, lse, temperature=2.0)
    at, = torch.autograd.grad(loss, w)
    # KL at the teacher is 0 up to LP; the gradient up to LP times |h| < 6
    assert abs(loss.item()) <= 8 * LP and at.abs().max().item() <= 12 * LP
    w = (wt * 0.5).requires_grad_(True)
    record = topk_logits(teacher, 8, 2.0)
    lse = record.logsumexp if tail else None
    loss = distill_loss(h @ w.t(), record.values, record.indices, lse, temperature=2.0)
    grad, = torch.autograd.grad(loss, w)
    with torch.no_grad():
        down = distill_loss(h @ (w - 1e-2 * grad).t(), record.values, record.indices, lse,
                            temperature=2.0)
    slope = (grad * grad).sum().item()
    assert down.item() < loss.item() - 0.5 * 1e-2 * slope


# ------------------------------------------------------------ through the engine
TINY = {
    "llama_1b": dict(vocab=131, hidden=64, layers=1, heads=1, kv_heads=1, ffn=128),
    # a head padded to 56 columns, of which 50 are real
    "bert_base": dict(vocab=50, hidden=64, layers=1, heads=1, ffn=64, max_seq=16, vocab_pad=56),
}


def objective_data(model, vocab, objective, n=6, S=8, seed=0):
    """A dataset as a station holds it, on the CPU."""
    from vantage6_amd.models import teacher_record

    g = torch.Generator().manual_seed(seed)
    if objective == "preference":
        mask = torch.ones(n, 2, S, dtype=torch.bool)
        mask[:, :, :3] = False
        return {"input_ids": torch.randint(0, vocab, (n, 2, S), generator=g), "mask": mask,
                "ref_logps": torch.randn(n, 2, generator=g) - 20.0}
    data = {"input_ids": torch.randint(0, vocab, (n, S), generator=g)}
    data["mask"] = torch.arange(S)[None] < torch.randint(3, S + 1, (n, 1), generator=g)
    if objective == "distill":
        device = next(model.parameters()).device
        record = teacher_record(model, data["input_ids"].to(device), 5, 2.0)
        assert (record["teacher_indices"] < vocab).all()
        return {**data, **{k: v.cpu() for k, v in record.items()}}
    data["old_logps"] = torch.randn(n, S - 1, generator=g) * 0.1 - math.log(vocab)
    data["ref_logps"] = torch.randn(n, S - 1, generator=g) * 0.1 - math.log(vocab)
    data["advantages"] = torch.randn(n, S - 1, generator=g)
    return data


OPTIONS = {"distill": {"temperature": 2.0}, "preference": {"beta": 0.2},
           "policy": {"kl_coef": 0.1, "clip_high": 0.3}}


@pytest.mark.parametrize("device", CPU_GPU)
@pytest.mark.parametrize("name", list(TINY))
@pytest.mark.parametrize("objective", list(OPTIONS))
def test_objectives_of_the_models(device, name, objective):
    """The factory's objective is the loss on the model's own logits, and its
    gradient reaches every weight."""
    need(device)
    from vantage6_amd.models import build_model, model_loss

    torch.manual_seed(0)
    dtype = torch.bfloat16 if device == "cuda" else torch.float32
    model = build_model(name, dtype=dtype, device=device, **TINY[name])
    vocab = TINY[name]["vocab"]
    batch = {k: v.to(device) for k, v in objective_data(model, vocab, objective).items()}
    if objective == "distill":
        batch["teacher_values"] = batch["teacher_values"] * 1.5  # not the model's own
    loss = model_loss(name, objective, **OPTIONS[objective])(model, batch)
    loss.backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in model.parameters())
    assert model.head.weight.grad[:vocab].abs().sum() > 0
    assert (model.head.weight.grad[vocab:] == 0).all()
    with torch.no_grad():
        ids = batch["input_ids"]
        if objective == "distill":
            rows, live, _ = distill_oracle(model(ids)[..., :vocab], batch["teacher_values"],
                                           batch["teacher_indices"], batch["teacher_lse"], 2.0,
                                           batch["mask"])
            want = rows.sum() / live.sum()
        elif objective == "preference":
            both = torch.cat([ids[:, 0], ids[:, 1]])
            targets = both[:, 1:].masked_fill(
                ~torch.cat([batch["mask"][:, 0], batch["mask"][:, 1]])[:, 1:], -100)
            ref = torch.cat([batch["ref_logps"][:, 0], batch["ref_logps"][:, 1]])
            want = preference_oracle(model(both[:, :-1])[..., :vocab], targets, ref, 0.2, 0.0,
                                     -100)[0].mean()
        else:
            rows, *_, live = policy_oracle(model(ids[:, :-1])[..., :vocab], ids[:, 1:],
                                           batch["old_logps"], batch["advantages"],
                                           batch["ref_logps"], batch["mask"][:, 1:], 0.2, 0.3, 0.1)
            want = rows.sum() / live.sum()
    # the same logits twice, one loss: its own error
    assert abs(loss.item() - want.item()) <= 50 * LP + 2.0 ** -22 * abs(want.item())


@pytest.mark.parametrize("device", CPU_GPU)
def test_preference_objective_with_another_ignore_index(device):
    """What the mask leaves out stays out under any ``ignore_index``."""
    need(device)
    from vantage6_amd.models import build_model, model_loss

    torch.manual_seed(2)
    name, vocab = "llama_1b", TINY["llama_1b"]["vocab"]
    model = build_model(name, device=device, **TINY[name])
    batch = {k: v.to(device) for k, v in objective_data(model, vocab, "preference").items()}
    with torch.no_grad():
        want, got = (model_loss(name, "preference", **o)(model, batch)
                     for o in ({}, {"ignore_index": -1}))
    assert torch.isfinite(want) and torch.equal(got, want)


@pytest.mark.parametrize("device", CPU_GPU)
@pytest.mark.parametrize("objective", list(OPTIONS))
def test_fit_rounds_with_an_objective(device, objective):
    need(device)
    from algorithms.fedavg import fit_rounds, make_batches
    from vantage6_amd.models import build_model

    torch.manual_seed(1)
    kw = dict(TINY["llama_1b"])
    teacher = build_model("llama_1b", device=device, **kw)
    data = objective_data(teacher, kw["vocab"], objective)
    out = fit_rounds(data, model="llama_1b", model_kwargs=kw, rounds=2, local_steps=2,
                     batch_size=4, lr=0.01, device=torch.device(device), objective=objective,
                     objective_options=OPTIONS[objective])
    assert out["rounds"] == 2 and all(math.isfinite(h["loss"]) for h in out["history"])
    batch = next(make_batches(data, 4, device))
    assert all(batch[k].dtype == data[k].dtype for k in data)  # measured values stay exact


@pytest.mark.parametrize("device", CPU_GPU)
def test_record_of_another_temperature(device):
    """A record's logsumexp holds at its temperature alone: the trainer refuses
    another, and a batch of it has a NaN for a loss. Without the logsumexp the
    record serves any."""
    need(device)
    from algorithms.fedavg import fit_rounds, make_batches
    from vantage6_amd.models import build_model, model_loss, teacher_record

    torch.manual_seed(1)
    kw = dict(TINY["llama_1b"])
    model = build_model("llama_1b", device=device, **kw)
    ids = torch.randint(0, kw["vocab"], (6, 8), generator=torch.Generator().manual_seed(2))
    for made in (1.0, 0.7):
        record = teacher_record(model, ids.to(device), 5, temperature=made)
        assert record["teacher_temperature"].shape == (6,)
        data = {"input_ids": ids, **{k: v.cpu() for k, v in record.items()}}
        batch = next(make_batches(data, 4, device))
        lse = batch.pop("teacher_lse")
        for used in (1.0, 0.7):
            loss = model_loss("llama_1b", "distill", temperature=used)
            assert torch.isfinite(loss(model, batch))
            got = loss(model, {**batch, "teacher_lse": lse})
            assert torch.isfinite(got) if used == made else torch.isnan(got)
            options = dict(model="llama_1b", model_kwargs=kw, rounds=1, local_steps=1, batch_size=4,
                           device=torch.device(device), objective="distill")
            if used == 1.0:  # the default
                run = lambda: fit_rounds(data, **options)
            else:
                run = lambda: fit_rounds(data, objective_options={"temperature": used}, **options)
            if used == made:
                assert math.isfinite(run()["final_loss"])
            else:
                with pytest.raises(ValueError, match="temperature"):
                    run()


@pytest.mark.parametrize("device", CPU_GPU)
def test_record_goes_into_the_loss_as_it_is(device):
    """``distill_loss(logits, **teacher_record(...))``: the record's entries are
    the loss's arguments, its temperature among them."""
    need(device)
    from vantage6_amd.models import build_model, teacher_record

    torch.manual_seed(1)
    kw = TINY["llama_1b"]
    model = build_model("llama_1b", device=device, **kw)
    ids = torch.randint(0, kw["vocab"], (2, 8), generator=torch.Generator().manual_seed(2))
    record = teacher_record(model, ids.to(device), 5, 2.0)
    x = make_logits(2, 8, kw["vocab"], torch.float32, device)
    want = distill_loss(x, record["teacher_values"], record["teacher_indices"],
                        record["teacher_lse"], temperature=2.0)
    assert torch.isfinite(want) and torch.equal(distill_loss(x, **record, temperature=2.0), want)
    assert torch.isnan(distill_loss(x, **record))  # at 1
    record["teacher_temperature"][0] = 1.0
    each = distill_loss(x, **record, reduction="none")
    assert torch.isfinite(each[0]).all() and torch.isnan(each[1]).all()
    mask = torch.tensor([[True], [False]], device=device).expand(2, 8)
    assert torch.isfinite(distill_loss(x, **record, mask=mask))
    lone = {k: v[0, 3] for k, v in record.items() if v.dim() > 1}
    one = torch.ones((), dtype=torch.float64, device=device)
    for shape, made in (((131,), one), ((1, 1, 1, 131), one.view(1))):
        args = {k: v.reshape((*shape[:-1], *v.shape)) for k, v in lone.items()}
        y = x[0, 3].reshape(shape)
        assert torch.isfinite(distill_loss(y, **args, teacher_temperature=made))
        assert torch.isnan(distill_loss(y, **args, teacher_temperature=made, temperature=0.7))
    no_lse = {k: v for k, v in record.items() if k != "teacher_lse"}
    assert torch.isfinite(distill_loss(x, **no_lse, temperature=0.7))
    for bad in (torch.ones(8, device=device), torch.ones(2, dtype=torch.int64, device=device)):
        with pytest.raises(ValueError):
            distill_loss(x, **{**record, "teacher_temperature": bad})


def test_objective_refusals():
    from algorithms.fedavg import fit_rounds
    from vantage6_amd.models import model_loss

    for call in (lambda: model_loss("resnet18", "distill"), lambda: model_loss("llama_1b", "lm"),
                 lambda: model_loss("llama_1b", temperature=2.0),
                 lambda: fit_rounds({"input_ids": torch.zeros(2, 4, dtype=torch.int64)},
                                    model="llama_1b", dp={"max_grad_norm": 1.0}, objective="policy",
                                    device=torch.device("cpu"))):
        with pytest.raises(ValueError):
            call()


@pytest.mark.gpu
@pytest.mark.parametrize("objective", list(OPTIONS))
def test_objective_in_a_captured_step(objective):
    """The trainer's captured local step, replayed, against eager steps: the
    same losses, bit for bit."""
    need("cuda")
    from algorithms.fedavg import _build, make_batches
    from vantage6_amd.models import build_model
    from vantage6_amd.parallel.comm import CommContext
    from vantage6_amd.parallel.fedavg import FedAvgConfig, FedAvgTrainer

    kw, dev = TINY["llama_1b"], torch.device("cuda", 0)
    torch.manual_seed(1)
    data = objective_data(build_model("llama_1b", device=dev, **kw), kw["vocab"], objective)
    losses = []
    for graph in (False, True):
        net, loss_fn = _build("llama_1b", kw, dev, objective=objective,
                              objective_options=OPTIONS[objective])
        # the same batch each time, whatever the capture draws
        fixed = next(make_batches(data, 4, dev))

        def batches():
            while True:
                yield fixed

        trainer = FedAvgTrainer(net, loss_fn, batches(), CommContext(device=dev),
                                FedAvgConfig(local_steps=1, lr=0.01), n_samples=6)
        if graph:
            assert trainer.enable_graph()
        losses.append([trainer.local_step() for _ in range(5)])
    assert losses[0] == losses[1] and len(set(losses[0])) > 1
