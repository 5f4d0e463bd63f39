"""Top logits and the distillation loss where a row's logits lie far apart or are large (B200).

The oracle and its bounds are those of test_distill_gpu.py.  Rows are masked with finite values at many depths and places, so that a
thread's, a warp's or a whole stage's first logits lie anywhere from nothing to hundreds below the row's largest, at
temperatures where exponentials at 1 and at tau differ much."""
import pytest
import torch

from test_distill_gpu import BF16, F32, U, _check_loss, _check_top, _logits, _ops, _reference, _targets, _teacher

pytestmark = pytest.mark.gpu

V = 50257
LOWS = (-60.0, -75.0, -76.0, -78.0, -80.0, -85.0, -87.0, -88.0, -89.0, -95.0, -100.0, -110.0, -128.0, -200.0, -250.0)
# a vector, a warp's, every thread's first vectors, a leading third and half, all but the last eight columns
PLACES = (8, 256, 3100, 16800, 25000, V - 8)


def _masked_rows(n, dtype, seed):
    z = _logits(n, V, dtype, seed)
    for r in range(n):
        combo = r % (len(LOWS) * len(PLACES) + 1)  # and a row without a mask
        if combo < len(LOWS) * len(PLACES):
            z[r, :PLACES[combo // len(LOWS)]] = LOWS[combo % len(LOWS)]
    return z


# 700 rows go to the persistent kernels (CTAs of their own for bf16, clusters for fp32), 91 to those of few rows
@pytest.mark.parametrize("n", [700, 91])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("tau,ce", [(1.0, 0.0), (1.0, 0.5), (0.5, 0.5), (1.5, 0.5), (2.0, 0.5), (3.5, 0.5), (4.0, 0.0),
                                    (4.0, 0.5), (8.0, 0.5), (30.0, 0.5)])
def test_finite_masks_at_every_depth(n, dtype, tau, ce):
    z = _masked_rows(n, dtype, 70)
    ids, t, lse = _teacher(z, 12, F32, 71, True, tau)
    y = _targets(n, V, ids, 72)
    _check_loss(z, ids, t, lse, y, tau, 0.8, ce, 0.5)
    _check_loss(z, ids, t, None, y, tau, 0.8, ce, 2.0 ** -13)


@pytest.mark.parametrize("n", [700, 91])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("tau", [1.0, 4.0])
def test_log_sum_exp_under_finite_masks(n, dtype, tau):
    _check_top(_masked_rows(n, dtype, 73), 8, tau)


# ------------------------------------------------------------------------------------ logits of large size
# A product of such a logit and log2(e) / tau has an error of many units; what follows must not depend on it.
LARGE = (-1e6, -1.2e7, -1e9, -1e10, -3e10, -7e11, -1e15, -1e20, -1e25, -1e30, 1e8, 1e10, 1e20)


def _compare(z, like, ids, t, lse, targets, tau, kd, ce, scale=1.0):
    """The kernels on ``z`` against the oracle on ``like``, which has the same probabilities."""
    loss, grad, tol, gtol = _reference(like, ids, t, lse, targets, tau, kd, ce, scale)
    zz = z.detach().requires_grad_(True)
    rows = _ops().distillation_loss(zz, ids, t, lse, targets, tau, kd, ce, scale, reduction="none")
    bad = ~((rows.double() - loss).abs() <= tol)
    assert not bad.any(), (bad.nonzero()[:5], rows[bad][:5], loss[bad][:5], tol[bad][:5])
    with torch.no_grad():
        assert torch.equal(_ops().distillation_loss(z, ids, t, lse, targets, tau, kd, ce, scale, reduction="none"), rows)
    (got,) = torch.autograd.grad(rows.sum(), zz)
    bad = ~((got.double() - grad).abs() <= gtol)
    assert not bad.any(), (bad.nonzero()[:5], got[bad][:5], grad[bad][:5], gtol[bad][:5])


@pytest.mark.parametrize("n", [700, 91])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("tau,ce", [(1.0, 0.0), (2.0, 0.5), (4.0, 0.5), (7.0, 0.5), (0.3, 0.5)])
def test_uniform_rows_of_large_logits(n, dtype, tau, ce):
    z = torch.tensor(LARGE, device="cuda").to(dtype).repeat(n // len(LARGE) + 1)[:n, None].expand(n, V).contiguous()
    ids, t, lse = _teacher(z, 12, F32, 74, True, tau)
    _compare(z, torch.zeros_like(z), ids, t, lse, _targets(n, V, ids, 75), tau, 0.8, ce)
    _check_top(z, 8, tau)


@pytest.mark.parametrize("n", [700, 91])
@pytest.mark.parametrize("tau,ce", [(1.0, 0.0), (2.0, 0.5), (4.0, 0.5), (7.0, 0.5), (0.3, 0.5)])
def test_a_shift_of_all_logits_changes_nothing(n, tau, ce):
    """fp32 logits in steps of 4 and shifts up to 2^25, whose sum is exact."""
    like = (_logits(n, V, F32, 76, spread=3.0) / 4).round() * 4
    shift = torch.tensor([0.0, 2.0 ** 20, -2.0 ** 23, -11629080.0, 11629080.0, 2.0 ** 24, -2.0 ** 25], device="cuda")
    z = like + shift.repeat(n // 7 + 1)[:n, None]
    assert torch.equal(z.double() - like.double(), (z - like).double())
    ids, t, lse = _teacher(like, 12, F32, 77, True, tau)
    _compare(z, like, ids, t, lse, _targets(n, V, ids, 78), tau, 0.8, ce)


@pytest.mark.parametrize("n", [700, 91])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("tau,ce", [(1.0, 0.0), (2.0, 0.5), (4.0, 0.5), (7.0, 0.5), (0.3, 0.5)])
def test_large_masks_are_as_good_as_infinite(n, dtype, tau, ce):
    z = _logits(n, V, dtype, 79)
    ids, t, lse = _teacher(z[:, 45000:].contiguous(), 12, F32, 80, True, tau)
    y = _targets(n, V - 45000, ids, 81)
    ids, y = torch.where(ids >= 0, ids + 45000, ids), torch.where(y >= 0, y + 45000, y)
    like, lows, places = z.clone(), [q for q in LARGE if q < 0], PLACES[:-1] + (45000,)
    for r in range(n):
        z[r, :places[r // len(lows) % len(places)]] = lows[r % len(lows)]
        like[r, :places[r // len(lows) % len(places)]] = float("-inf")
    _compare(z, like, ids, t, lse, y, tau, 0.8, ce)
    _check_top(z, 8, tau)


@pytest.mark.parametrize("n", [700, 91])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("tau", [1.0, 2.0, 7.0])
def test_only_the_listed_logits_are_not_masked(n, dtype, tau):
    """The rest is uniform: its loss m (log m - log q_rest) to 2^-16 of it (rounding of 2^-24 in a handful of numbers of its
    size), its gradient -kd tau m / columns to 2^-14 and half an ulp, that of a listed column tau (q (1 + m - ...) - p)."""
    lows = torch.tensor([q for q in LARGE if q < 0], device="cuda").to(dtype)
    z = lows.repeat(n // len(lows) + 1)[:n, None].expand(n, V).contiguous()
    g = torch.Generator(device="cuda").manual_seed(82)
    ids = (torch.randint(0, V - 60, (n, 1), device="cuda", generator=g) + 5 * torch.arange(10, device="cuda")).int()
    t = 2 * torch.randn(n, 10, device="cuda", generator=g)
    lse = torch.logsumexp(t / tau, 1) + 0.3
    mine = torch.randn(n, 10, device="cuda", generator=g).to(dtype)
    low = z[:, 0].double()
    z.scatter_(1, ids.long(), mine)
    p = torch.exp(t.double() / tau - lse.double()[:, None])
    m = 1 - p.sum(1)
    q = torch.softmax(mine.double() / tau, 1)
    log_rest = low / tau + torch.log(torch.tensor(V - 10.0, device="cuda").double()) - torch.logsumexp(mine.double() / tau, 1)
    want = tau * tau * ((p * (p.log() - q.log())).sum(1) + m * (m.log() - log_rest))
    zz = z.clone().requires_grad_(True)
    rows = _ops().distillation_loss(zz, ids, t, lse, temperature=tau, reduction="none")
    assert ((rows.double() - want).abs() <= 2.0 ** -16 * want).all()
    (got,) = torch.autograd.grad(rows.sum(), zz)
    half = 2.0 ** -8 if dtype == BF16 else 0.0
    rest = -tau * m / (V - 10)
    unlisted = torch.ones_like(got, dtype=torch.bool).scatter_(1, ids.long(), False)
    off = (got.double() - rest[:, None]).abs() / rest.abs()[:, None]
    assert off[unlisted].max() <= 2.0 ** -14 + half
    listed = tau * (q * (p.sum(1) + m)[:, None] - p)
    tol = tau * 64 * U * (1 + 20) * (q + p) + half * listed.abs()
    assert ((got.gather(1, ids.long()).double() - listed).abs() <= tol).all()


@pytest.mark.parametrize("n", [700, 3])
def test_a_rest_far_below_the_list(n):
    """The unlisted logits' mass lies e^-68.9 below the list's largest logit, one column of it far above the others, whose
    exponentials relative to the list vanish in fp32 (2^-126) although they are a thousandth of that mass."""
    v = 131072
    z = torch.full((n, v), -87.45, device="cuda")
    z[:, 70000] = -68.95
    ids = torch.tensor([[0, 5, 131071]], dtype=torch.int32, device="cuda").repeat(n, 1)
    z[:, ids[0].long()] = torch.tensor([0.0, -1.0, -2.0], device="cuda")
    t = torch.tensor([[1.0, 0.5, 0.0]], device="cuda").repeat(n, 1)
    lse = torch.logsumexp(t, 1) + 0.3
    _compare(z, z, ids, t, lse, None, 1.0, 1.0, 0.0)


# Rows off 16 bytes: their first and last columns are added one by one, after the others.
@pytest.mark.parametrize("n", [700, 91])
@pytest.mark.parametrize("dtype,v,offset", [(F32, 36226, 1), (BF16, 36226, 3), (BF16, 50257, 5)])
@pytest.mark.parametrize("tau,ce", [(1.0, 0.0), (1.3, 0.5), (2.0, 0.5), (4.0, 0.5), (6.0, 0.5)])
def test_finite_masks_and_the_rows_ends(n, dtype, v, offset, tau, ce):
    z = _logits(n, v, dtype, 83, ld=v, offset=offset, spread=0.3)
    lows = (-70.0, -80.0, -86.0, -87.0, -87.5, -88.0, -88.5, -90.0)
    places = (1, 9, 1001, 15003, 32507, v - 601, v - 9, v - 3, v - 1)
    for r in range(n):
        at, low = places[r // len(lows) % len(places)], lows[r % len(lows)]
        if r % 2:
            z[r, :at] = low
        else:  # the last columns alone lie below, or the first
            z[r, -at:] = low if r % 4 else z[r, -at:]
            z[r, -1] = 0.5
    ids, t, lse = _teacher(z, 5, F32, 84, True, tau)
    _check_loss(z, ids, t, lse, _targets(n, v, ids, 85), tau, 0.8, ce, 0.5)
    _check_top(z, 8, tau)
