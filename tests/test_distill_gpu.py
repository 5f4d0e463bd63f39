"""A teacher's top logits and the distillation loss against plain 64-bit PyTorch (B200).

Top logits are compared for equality (values, columns, order); the log-sum-exp and everything below within
bounds derived before the first run, in units of u = 2^-24:

* an exponential exp(x) of an fp32 difference x is off by a relative (8 + 2 |x|) u (rounding of x times a constant,
  and the hardware's 2^-22); a sum of exponentials relative to the largest is then off by 32 u (|x| e^-|x| < 1);
* log-sum-exp: 32 u plus the rounding of |max / tau| and of the result: 4 u (|max / tau| + |lse|);
* p_i = exp(a_i - L): relative E_p = (16 + 4 (|a_i| + |L|)) u;  m = 1 - sum p: absolute k-independent E_m = max E_p + 8 u;
* the loss of a row: every logarithm is off by 64 u (1 + |z|max / tau + |a|max + |L|) absolute, every p and m as above
  and multiplies a difference of logarithms of size D: together kd tau^2 (64 u S + (E_p + E_m) (D + 2)) with
  S = 1 + |z|max / tau + |a|max + |L|, plus ce 64 u (1 + |z|max);
* the gradient of a column: kd tau (q_j (P + m + m / q_rest) 64 u (1 + R) + q_j / q_rest E_m + p_j E_p + q_j E_m)
  + ce 64 u (softmax_j (1 + R tau) + [j = target]), R = max |z - top| / tau, plus half an ulp of the gradient's type.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF_ULP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0 ** -25}
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _ops():
    from tensor_train_ing_b200.ops import distill
    return distill


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _logits(n, v, dtype, seed, ld=None, offset=0, spread=2.0):
    """[n, v] logits whose rows are ``ld`` apart and start ``offset`` elements into the buffer."""
    ld = v if ld is None else ld
    flat = (torch.randn(n * ld + offset + 8, device="cuda", generator=_gen(seed)) * spread).to(dtype)
    return flat[offset:offset + n * ld].view(n, ld)[:, :v]


# ------------------------------------------------------------------------------------ top logits
def _check_top(z, k, tau=1.0):
    got = _ops().top_logits(z, k, temperature=tau)
    values, order = torch.sort(z.float(), dim=1, descending=True, stable=True)
    assert got.ids.dtype == torch.int32 and got.values.dtype == z.dtype and got.lse.dtype == F32
    assert torch.equal(got.ids.long(), order[:, :k])
    assert torch.equal(got.values.float().nan_to_num(nan=7e30), values[:, :k].nan_to_num(nan=7e30))
    lse = torch.logsumexp(z.double() / tau, 1)
    top = (z.double() / tau).amax(1)
    tol = 32 * U + 4 * U * (top.abs() + lse.abs())
    fine = torch.isfinite(lse)
    assert torch.equal(got.lse.double()[~fine].nan_to_num(nan=7e30), lse[~fine].nan_to_num(nan=7e30))
    assert ((got.lse.double() - lse).abs()[fine] <= tol[fine]).all()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("n,v,k", [(1, 1, 1), (3, 2, 2), (2, 7, 3), (5, 33, 33), (4, 256, 256), (7, 500, 8), (3, 1000, 256),
                                   (2, 4097, 64), (40, 8191, 17), (300, 8192, 1), (9, 50257, 64), (2, 50304, 256),
                                   (3, 131072, 128), (1, 200000, 32)])
def test_top_logits(n, v, k, dtype):
    _check_top(_logits(n, v, dtype, n + v + k), k, tau=1.0 + (k % 3))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("offset,ld", [(0, 1024), (1, 1001), (3, 1003), (5, 1024), (8, 1009)])
def test_top_logits_of_strided_and_misaligned_rows(dtype, offset, ld):
    _check_top(_logits(6, 1000, dtype, 3, ld=ld, offset=offset), 20)


def test_top_logits_strides_leading_shapes_and_streams():
    z = _logits(12, 3000, BF16, 1)
    want = _ops().top_logits(z, 5)
    got = _ops().top_logits(z.view(3, 4, 3000), 5)
    assert got.ids.shape == (3, 4, 5) and got.lse.shape == (3, 4)
    for a, b in zip(got, want):
        assert torch.equal(a.reshape(b.shape), b)
    for view in (z.t().contiguous().t(), z[::3], torch.stack([z, z], 2)[:, :, 0]):
        _check_top(view, 5)
    one = _ops().top_logits(z[0], 5)
    assert one.ids.shape == (5,) and torch.equal(one.ids, want.ids[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = _ops().top_logits(z, 5)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(again, want))
    empty = _ops().top_logits(z[:0], 5)
    assert empty.ids.shape == (0, 5) and empty.lse.shape == (0,)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("v", [100, 2000, 50257])
def test_ties_take_the_lowest_columns(v, dtype):
    z = torch.zeros(7, v, device="cuda", dtype=dtype)
    z[1] = -3.25
    z[2] = torch.arange(v, device="cuda") % 3  # a third of the row ties for the top
    z[3] = float("-inf")
    z[3, ::17] = -1.0  # fewer finite entries than a list may hold, all equal
    z[4] = torch.finfo(dtype).min
    z[5, 1::2] = -0.0  # equal to +0
    z[6] = torch.arange(v, device="cuda").to(dtype)  # ascending
    for k in (1, 40, min(v, 256)):
        _check_top(z, k)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("v", [64, 5000, 60000])
def test_infinities_and_nan(v, dtype):
    z = _logits(6, v, dtype, 11)
    z[0] = float("-inf")
    z[1, 5] = float("inf")
    z[2, [1, 9]] = float("nan")
    z[3] = float("nan")
    z[4, : v - 3] = float("-inf")
    z[5, ::2] = torch.finfo(dtype).min
    _check_top(z, 12)


# Many long rows: the persistent kernel
@pytest.mark.parametrize("dtype,v,ld,offset", [(BF16, 16384, 16384, 0), (BF16, 20001, 20001, 3), (F16, 50257, 50304, 0),
                                               (F32, 8200, 8200, 0), (F32, 30001, 30001, 2), (F32, 131072, 131072, 0),
                                               (BF16, 60003, 60003, 3), (F16, 300007, 300007, 5)])
@pytest.mark.parametrize("k", [1, 64, 256])
def test_top_logits_of_many_rows(dtype, v, ld, offset, k):
    n = 1501 if v < 30000 else 601
    z = _logits(n, v, dtype, v + k, ld=ld, offset=offset)
    z[3] = 0  # ties throughout
    z[4] = float("-inf")
    z[5, 100:] = float("-inf")
    z[6, 7] = float("nan")
    z[7] = torch.finfo(dtype).min
    z[8, ::3] = z[8].max() + 1  # more ties at the top than any list holds
    z[9, [0, v - 1]] = 50.0  # the ends of the row
    z[10, 5] = float("inf")
    z[n - 1] = torch.arange(v, device="cuda").to(dtype)
    _check_top(z, k, tau=1.5)


def test_top_logits_of_a_peaked_thread():
    """All large logits in the vectors one thread reads: the bound from thread maxima is then far too low."""
    z = _logits(3, 30000, F32, 2)
    for r in range(3):
        z[r, r * 8:r * 8 + 8] = 50 + torch.rand(8, device="cuda", generator=_gen(r))
        z[r, 4096 + r * 8:4096 + r * 8 + 8] = 40 + torch.rand(8, device="cuda", generator=_gen(r))
    _check_top(z, 16)
    _check_top(z, 256)


def test_rows_past_32_bit_offsets():
    """Element offsets of the last rows exceed 2^31."""
    n, v = 43000, 50304
    z = torch.empty(n, v, device="cuda", dtype=BF16)
    z.normal_(generator=_gen(4))
    last = z[-3:].clone()
    got = _ops().top_logits(z, 16)
    want = _ops().top_logits(last, 16)
    assert torch.equal(got.ids[-3:], want.ids) and torch.equal(got.lse[-3:], want.lse)
    ids = got.ids[-3:]
    zz = z.requires_grad_(True)
    loss = _ops().distillation_loss(zz, got.ids, got.values)
    (g,) = torch.autograd.grad(loss, zz)
    ll = last.requires_grad_(True)
    (gl,) = torch.autograd.grad(_ops().distillation_loss(ll, ids, got.values[-3:]), ll)
    assert torch.equal(g[-3:], gl)


# ------------------------------------------------------------------------------------ distillation loss
def _teacher(z, k, t_dtype, seed, rest, tau):
    """Distinct columns, falling logits, a few absent entries, one row without any."""
    n, v = z.shape
    g = _gen(seed)
    ids = torch.rand(n, v, device="cuda", generator=g).topk(k, dim=1).indices if v <= 60000 else \
        torch.randint(0, v - 4 * k, (n, 1), device="cuda", generator=g) + 3 * torch.arange(k, device="cuda")
    t = (4 - torch.rand(n, k, device="cuda", generator=g).cumsum(1)).to(t_dtype)
    if k > 1:
        ids = torch.where(torch.rand(n, k, device="cuda", generator=g) < 0.1, -1, ids)
    if n > 2:
        ids[1] = -1
    lse = torch.logsumexp(t.float() / tau, 1) + 0.3 * torch.rand(n, device="cuda", generator=g) + 0.05 if rest else None
    return ids.to(torch.int32), t, lse


def _reference(z, ids, t, lse, targets, tau, kd, ce, scale):
    """(loss rows, gradient, tolerances of both) in 64 bits, from the formulas of ops/distill.py."""
    z64 = z.detach().double()
    n, v = z64.shape
    a = t.double() / tau
    there = ids >= 0
    L = lse.double() if lse is not None else torch.logsumexp(a.masked_fill(~there, -math.inf), 1)
    L = torch.where(there.any(1) & torch.isfinite(L), L, torch.zeros_like(L))[:, None]
    logp = (a - L).masked_fill(~there, -math.inf)
    p = logp.exp()
    m = (1 - p.sum(1)) * there.any(1) if lse is not None else torch.zeros(n, device=z.device, dtype=torch.float64)
    m = torch.where(m > 2.0 ** -20, m, torch.zeros_like(m))
    logq = torch.log_softmax(z64 / tau, 1)
    q = logq.exp()
    at = ids.long().clamp_min(0)
    share = torch.zeros_like(z64).scatter_add_(1, at, p)
    listed = torch.zeros(n, v, device=z.device).scatter_add_(1, at, there.float()) > 0
    log_rest = torch.logsumexp(logq.masked_fill(listed, -math.inf), 1)
    m = torch.where(listed.all(1), torch.zeros_like(m), m)
    diff = torch.where(p > 0, logp - logq.gather(1, at), torch.zeros_like(p))
    rest_diff = torch.where(m > 0, m.clamp_min(1e-300).log() - log_rest, torch.zeros_like(m))
    kl = (p * diff).sum(1) + m * rest_diff
    loss = kd * tau * tau * kl
    inv_rest = torch.where(m > 0, 1 / log_rest.exp(), torch.zeros_like(m))[:, None]
    mass = (p.sum(1) + m)[:, None]
    grad = kd * tau * (q * mass - torch.where(listed, torch.zeros_like(q), q * m[:, None] * inv_rest) - share)
    zmax = z64.masked_fill(~torch.isfinite(z64), 0).abs().amax(1)
    amax = a.masked_fill(~(there & torch.isfinite(a)), 0).abs().amax(1)
    Ep = (16 + 4 * (amax + L[:, 0].abs())) * U
    Em = Ep + 8 * U
    D = torch.maximum(diff.abs().amax(1), rest_diff.abs())
    S = 1 + zmax / tau + amax + L[:, 0].abs()
    tol = kd * tau * tau * (64 * U * S + (Ep + Em) * (D + 2))
    R = ((z64.amax(1, keepdim=True) - z64) / tau).clamp_max(200.0)
    gtol = kd * tau * (q * (mass + m[:, None] * inv_rest) * 64 * U * (1 + R) + q * inv_rest * Em[:, None]
                       + share * Ep[:, None] + q * Em[:, None])
    if ce:
        logs = torch.log_softmax(z64, 1)
        hot = torch.zeros_like(z64).scatter_(1, targets.clamp_min(0)[:, None], 1.0)
        loss = loss - ce * logs.gather(1, targets.clamp_min(0)[:, None])[:, 0]
        grad = grad + ce * (logs.exp() - hot)
        tol = tol + ce * 64 * U * (1 + zmax)
        gtol = gtol + ce * 64 * U * (logs.exp() * (1 + R * tau) + hot)
    if targets is not None:
        dead = targets < 0
        loss = loss.masked_fill(dead, 0)
        grad = grad.masked_fill(dead[:, None], 0)
    gtol = scale * gtol + HALF_ULP[z.dtype] * 1.01 * (scale * grad).abs() + TINY[z.dtype]
    return scale * loss, scale * grad, scale * tol + 1e-37, gtol


def _check_loss(z, ids, t, lse=None, targets=None, tau=1.0, kd=1.0, ce=0.0, scale=1.0):
    loss, grad, tol, gtol = _reference(z, ids, t, lse, targets, tau, kd, ce, scale)
    kw = dict(teacher_lse=lse, targets=targets, temperature=tau, kd_weight=kd, ce_weight=ce, scale=scale)
    with torch.no_grad():
        rows = _ops().distillation_loss(z, ids, t, reduction="none", **kw)
    assert rows.dtype == F32
    bad = (rows.double() - loss).abs() > tol
    assert not bad.any(), (rows[bad], loss[bad], tol[bad])
    zz = z.detach().requires_grad_(True)
    total = _ops().distillation_loss(zz, ids, t, **kw)
    assert abs(float(total.detach()) - float(loss.sum())) <= float(tol.sum()) + 4 * U * float(loss.abs().sum())
    (got,) = torch.autograd.grad(total, zz)
    assert got.dtype == z.dtype and got.shape == z.shape
    bad = (got.double() - grad).abs() > gtol
    assert not bad.any(), (bad.nonzero()[:5], got[bad][:5], grad[bad][:5], gtol[bad][:5])


def _targets(n, v, ids, seed):
    g = _gen(seed)
    y = torch.randint(0, v, (n,), device="cuda", generator=g)
    y = torch.where(torch.rand(n, device="cuda", generator=g) < 0.4, ids[:, 0].long().clamp_min(0), y)
    if n > 3:
        y[3] = -100
    return y


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("n,v,k", [(1, 1, 1), (2, 2, 1), (4, 7, 7), (5, 33, 4), (9, 500, 8), (6, 1000, 300), (4, 4097, 64),
                                   (33, 8192, 33), (5, 50257, 64), (3, 131072, 128), (2, 200001, 1024)])
@pytest.mark.parametrize("tau,ce", [(1.0, 0.0), (2.0, 0.25), (1.0, 0.5)])
def test_loss_fp32(n, v, k, rest, tau, ce):
    z = _logits(n, v, F32, n + v)
    ids, t, lse = _teacher(z, k, F32, k, rest, tau)
    _check_loss(z, ids, t, lse, _targets(n, v, ids, 1), tau, 0.75, ce, 0.125)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("n,v,k", [(3, 5, 2), (9, 500, 8), (4, 4097, 64), (5, 50257, 64), (300, 1027, 16), (2, 131072, 256)])
@pytest.mark.parametrize("rest,tau,ce", [(False, 1.0, 0.0), (True, 1.5, 0.0), (True, 4.0, 0.5), (False, 2.0, 1.0)])
def test_loss_16_bits(n, v, k, rest, tau, ce, dtype):
    z = _logits(n, v, dtype, n + v)
    ids, t, lse = _teacher(z, k, dtype, k, rest, tau)
    _check_loss(z, ids, t, lse, _targets(n, v, ids, 2), tau, 1.0, ce, 1.0)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("offset,ld", [(0, 1024), (1, 1001), (3, 1003), (5, 1024), (8, 5000)])
def test_loss_of_strided_and_misaligned_rows(dtype, offset, ld):
    z = _logits(6, 1000, dtype, 3, ld=ld, offset=offset)
    ids, t, lse = _teacher(z, 20, F32, 5, True, 1.0)
    _check_loss(z, ids.long(), t, lse, None, 1.0, 1.0, 0.0, 1.0)


# Many long rows: the persistent kernel, of single CTAs and of clusters.  These take several rows each, with and without
# left-out ones between them; odd widths and offsets give rows with edges on either side.
@pytest.mark.parametrize("dtype,v,ld,offset", [(BF16, 8192, 8192, 0), (BF16, 9001, 9001, 3), (F16, 20011, 20032, 1),
                                               (F32, 4100, 4100, 0), (F32, 16001, 16001, 2), (BF16, 50257, 50257, 0),
                                               (BF16, 30011, 30011, 3), (F16, 40009, 40064, 5), (F32, 20480, 20480, 0),
                                               (F32, 50257, 50257, 1), (F32, 131072, 131072, 0), (F16, 200003, 200003, 5)])
@pytest.mark.parametrize("k,rest,tau,ce", [(1, False, 1.0, 0.0), (40, True, 2.0, 0.5), (200, True, 1.5, 0.25),
                                           (64, False, 4.0, 0.5)])
def test_loss_of_many_rows(dtype, v, ld, offset, k, rest, tau, ce):
    n = 601 if v > 9500 else 1201
    z = _logits(n, v, dtype, v + k, ld=ld, offset=offset)
    ids, t, lse = _teacher(z, k, F32, k, rest, tau)
    ids[5:9] = -1
    if k > 2:
        ids[20, 0], ids[20, 1], ids[20, 2] = 0, v - 1, 0  # both ends of the row, and a column named twice
        ids[21, :3] = 4099 % v
    y = _targets(n, v, ids, 5)
    y[torch.rand(n, device="cuda", generator=_gen(6)) < 0.3] = -100
    y[30:330] = -100
    y[20], y[22] = 0, v - 1
    _check_loss(z, ids, t, lse, y if ce or v % 2 else None, tau, 0.9, ce, 0.5)


def test_every_row_of_many_left_out():
    z = _logits(800, 30011, BF16, 50)
    ids, t, lse = _teacher(z, 8, F32, 51, True, 1.0)
    _check_loss(z, ids, t, lse, torch.full((800,), -100, device="cuda"))


def test_non_finite_rows_among_many():
    z = _logits(700, 20011, F32, 52)
    ids, t, lse = _teacher(z, 8, F32, 53, True, 1.0)
    clean = _ops().distillation_loss(z, ids, t, lse, reduction="none")
    bad = torch.zeros(700, dtype=torch.bool, device="cuda")
    bad[[3, 299, 699]] = True
    zz = z.clone()
    zz[3, 1], zz[299, 20010], zz[699, 4000] = float("nan"), float("nan"), float("inf")
    rows = _ops().distillation_loss(zz, ids, t, lse, reduction="none")
    assert torch.equal(rows[~bad], clean[~bad]) and not torch.isfinite(rows[bad]).any()
    low = z.clone()
    low[:, 5000:] = torch.finfo(F32).min
    low[10] = torch.finfo(F32).min  # a row at the lowest value throughout: uniform
    _check_loss(torch.cat([low[:10], low[11:]]), torch.cat([ids[:10], ids[11:]]).clamp_max(4999),
                torch.cat([t[:10], t[11:]]), torch.cat([lse[:10], lse[11:]]))
    flat = low.clone()
    flat[10] = 0
    a = _ops().distillation_loss(low, ids, t, lse, reduction="none")[10]
    assert a == _ops().distillation_loss(flat, ids, t, lse, reduction="none")[10]


@pytest.mark.parametrize("keep", [1, 2, 5])
def test_clusters_that_leave_out_most_rows(keep):
    z = _logits(1200, 50257, F32, 57)
    ids, t, lse = _teacher(z, 16, F32, 58, True, 2.0)
    y = _targets(1200, 50257, ids, 59)
    stride = torch.arange(1200, device="cuda") // 100  # rows of one cluster lie about a hundred apart
    y[(stride % 6) >= keep] = -100
    _check_loss(z, ids, t, lse, y, 2.0, 1.0, 0.5)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("low", [-1e4, -3e38, float("-inf")])
def test_rows_masked_at_their_start(dtype, low):
    z = _logits(700, 40009, dtype, 60)
    ids, t, lse = _teacher(z[:, 9000:].contiguous(), 8, F32, 61, True, 1.0)
    ids = torch.where(ids >= 0, ids + 9000, ids)
    z[:, :9000] = low
    y = torch.where(ids[:, 0] >= 0, ids[:, 0].long(), 30000)
    y[::3] = 20000
    _check_loss(z, ids, t, lse, y, 2.0, 1.0, 0.5)
    _check_loss(z, ids, t, lse, None, 1.0)
    _check_top(z, 8)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_logits_far_above_a_threads_first_ones(dtype):
    """Late logits so far above the first that sums relative to these overflow; in many rows and in few."""
    for n in (700, 5):
        z = _logits(n, 40009, dtype, 54)
        ids, t, lse = _teacher(z, 8, F32, 55, True, 1.0)
        z[::2, 30000:30100] += 300.0
        z[1, 39000] = 400.0
        kept = z[3, ids[3].long()].clone()
        z[3, :20000] = float("-inf")
        z[3, ids[3].long()] = kept  # a listed column at -inf makes the row's loss infinite
        _check_loss(z, ids, t, lse, None, 1.0)
        y = _targets(n, 40009, ids, 56)
        _check_loss(z, ids, t, lse, y, 2.0, 1.0, 0.5)
        _check_top(z, 8)


def test_types_of_the_list_mix():
    z = _logits(8, 3000, BF16, 6)
    for t_dtype in (F32, BF16, F16):
        ids, t, lse = _teacher(z, 12, t_dtype, 7, True, 1.0)
        _check_loss(z, ids, t, lse)
        _check_loss(z.float(), ids.long(), t, lse)


def test_rows_without_a_list_and_without_a_target():
    z = _logits(6, 700, F32, 8)
    ids, t, lse = _teacher(z, 5, F32, 9, True, 1.0)
    ids[:] = -1
    _check_loss(z, ids, t, lse)
    y = torch.full((6,), -100, device="cuda")
    _check_loss(z, ids, t, lse, y, ce=1.0)
    z[2] = float("nan")  # a left-out row is not read
    _check_loss(z.nan_to_num(), ids, t, lse, y, ce=1.0)
    zz = z.clone().requires_grad_(True)
    loss = _ops().distillation_loss(zz, ids, t, lse, y, ce_weight=1.0)
    assert loss == 0 and not torch.autograd.grad(loss, zz)[0].any()


def test_list_naming_every_column():
    z = _logits(5, 40, F32, 10)
    ids = torch.stack([torch.randperm(40, device="cuda", generator=_gen(i)) for i in range(5)]).int()
    t = torch.randn(5, 40, device="cuda", generator=_gen(3))
    _check_loss(z, ids, t, torch.logsumexp(t, 1))
    _check_loss(z, ids, t)


def test_repeated_columns_add_up():
    z = _logits(4, 900, F32, 12)
    ids, t, lse = _teacher(z, 6, F32, 13, True, 1.0)
    ids[:, 3] = ids[:, 0]
    ids[0] = 17
    lse = lse + 2.0
    _check_loss(z, ids, t, lse)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_masked_logits(dtype):
    """-inf and the type's lowest value among the student's logits: no mass, no gradient, nothing else changes."""
    z = _logits(4, 6000, dtype, 14)
    ids, t, lse = _teacher(z, 10, F32, 15, True, 1.0)
    ids = ids.clamp_max(4999)
    for low in (float("-inf"), torch.finfo(dtype).min):
        zz = z.clone()
        zz[:, 5000:] = low
        _check_loss(zz, ids, t, lse)
        _check_loss(zz, ids, t)
        g = zz.clone().requires_grad_(True)
        (got,) = torch.autograd.grad(_ops().distillation_loss(g, ids, t, lse), g)
        assert not got[:, 5000:].any()


def test_student_without_mass_outside_the_list():
    """Only the listed columns have finite logits, the teacher has mass elsewhere: an infinite divergence (or, with
    the lowest finite value in place of -inf, a huge one), and finite without the teacher's rest."""
    z = torch.full((2, 3000), float("-inf"), device="cuda")
    ids = torch.tensor([[3, 900, 2999], [0, 1, 2]], dtype=torch.int32, device="cuda")
    t = torch.tensor([[1.0, 0.5, 0.0], [2.0, 2.0, 2.0]], device="cuda")
    lse = torch.logsumexp(t, 1) + 0.2
    z.scatter_(1, ids.long(), torch.randn(2, 3, device="cuda", generator=_gen(1)))
    rows = _ops().distillation_loss(z, ids, t, lse, reduction="none")
    assert (rows == float("inf")).all()
    _check_loss(z, ids, t)
    z = z.clamp_min(torch.finfo(F32).min)
    rows = _ops().distillation_loss(z, ids, t, lse, reduction="none")
    assert torch.isfinite(rows).all() and (rows > 1e36).all()
    _check_loss(z, ids, t, lse)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_uniform_rows_at_the_lowest_value(dtype):
    z = torch.full((3, 300), torch.finfo(dtype).min, device="cuda", dtype=dtype)
    ids, t, _ = _teacher(z, 5, F32, 33, False, 1.0)
    rows = _ops().distillation_loss(z, ids, t, reduction="none")
    flat = _ops().distillation_loss(torch.zeros_like(z), ids, t, reduction="none")
    assert torch.equal(rows, flat)  # a shift of all logits changes nothing


def test_teacher_without_mass_on_an_entry():
    z = _logits(3, 500, F32, 16)
    ids, t, lse = _teacher(z, 9, F32, 17, False, 1.0)
    t[0, 2:5] = float("-inf")
    t[2] = float("-inf")  # nothing at all: the row has no divergence
    _check_loss(z, ids, t)


def test_non_finite_rows_stay_in_their_row():
    z = _logits(5, 9000, F32, 18)
    ids, t, lse = _teacher(z, 9, F32, 19, True, 1.0)
    z[2, 77] = float("nan")
    rows = _ops().distillation_loss(z, ids, t, lse, reduction="none")
    assert torch.isnan(rows[2]) and torch.isfinite(rows[[0, 1, 3, 4]]).all()
    zz = z.clone().requires_grad_(True)
    (g,) = torch.autograd.grad(_ops().distillation_loss(zz, ids, t, lse), zz)
    assert torch.isfinite(g[[0, 1, 3, 4]]).all()


def test_gradient_against_differences():
    """Directional differences of the kernel's own loss, step 2^-6: truncation of order h^2 / 6 of the third
    derivative (4e-5), rounding 64 u S / h (about 2e-4 of the loss): 3e-3 of the slope is safe."""
    z = _logits(4, 300, F32, 20)
    ids, t, lse = _teacher(z, 6, F32, 21, True, 2.0)
    y = torch.tensor([5, 6, 7, 8], device="cuda")
    f = lambda q: _ops().distillation_loss(q, ids, t, lse, y, temperature=2.0, ce_weight=0.3, reduction="none")  # noqa: E731
    zz = z.clone().requires_grad_(True)
    (g,) = torch.autograd.grad(f(zz).sum(), zz)
    v = torch.randn(z.shape, device="cuda", generator=_gen(5))
    v = v / v.norm() + g / g.norm()
    h = 2.0 ** -6
    with torch.no_grad():
        slope = (f(z + h * v).double() - f(z - h * v).double()).sum() / (2 * h)
    want = (g.double() * v.double()).sum()
    assert abs(slope - want) <= 3e-3 * abs(want)


def test_incoming_factors_and_a_single_backward():
    z = _logits(7, 1300, F32, 22)
    ids, t, lse = _teacher(z, 6, F32, 23, True, 1.0)
    zz = z.clone().requires_grad_(True)
    (g1,) = torch.autograd.grad(_ops().distillation_loss(zz, ids, t, lse), zz)
    (g2,) = torch.autograd.grad(_ops().distillation_loss(zz, ids, t, lse) * 3.0, zz)
    torch.testing.assert_close(g2, 3.0 * g1, rtol=2 * U, atol=0)
    w = torch.tensor([1.0, 0.0, 2.0, 1.0, -1.0, 0.5, 1.0], device="cuda")
    (g3,) = torch.autograd.grad((_ops().distillation_loss(zz, ids, t, lse, reduction="none") * w).sum(), zz)
    torch.testing.assert_close(g3, w[:, None] * g1, rtol=2 * U, atol=0)
    dev = torch.tensor(0.5, device="cuda")
    (g4,) = torch.autograd.grad(_ops().distillation_loss(zz, ids, t, lse, scale=dev), zz)
    torch.testing.assert_close(g4, 0.5 * g1, rtol=2 * U, atol=0)
    loss = _ops().distillation_loss(zz, ids, t, lse)
    torch.autograd.grad(loss, zz, retain_graph=True)
    with pytest.raises(RuntimeError, match="earlier backward"):
        torch.autograd.grad(loss, zz)


def test_through_a_student_and_leading_shapes():
    """The gradient reaches a student's parameters; (B, T, V) logits cut from a padded buffer."""
    g = _gen(24)
    w = torch.randn(640, 32, device="cuda", generator=g, requires_grad=True)
    x = torch.randn(2, 5, 32, device="cuda", generator=g)
    logits = (x @ w.t())[..., :601]
    ids, t, lse = _teacher(logits.detach().reshape(10, 601), 7, F32, 25, True, 1.0)
    y = torch.full((2, 5), 3, device="cuda")
    y[0, 2] = -100
    loss = _ops().distillation_loss(logits, ids.view(2, 5, 7), t.view(2, 5, 7), lse.view(2, 5), y, ce_weight=0.5)
    loss.backward()
    z = logits.detach().reshape(10, 601)
    _, grad, _, _ = _reference(z, ids, t, lse, y.view(-1), 1.0, 1.0, 0.5, 1.0)
    want = torch.zeros(640, 32, device="cuda", dtype=torch.float64)
    want[:601] = grad.t() @ x.view(10, 32).double()
    torch.testing.assert_close(w.grad.double(), want, rtol=1e-4, atol=1e-4)
    rows = _ops().distillation_loss(logits, ids.view(2, 5, 7), t.view(2, 5, 7), reduction="none")
    assert rows.shape == (2, 5)


def test_no_rows_same_bits_and_streams():
    z = _logits(64, 20000, BF16, 26)
    ids, t, lse = _teacher(z, 32, BF16, 27, True, 1.0)

    def both():
        zz = z.detach().requires_grad_(True)
        rows = _ops().distillation_loss(zz, ids, t, lse, reduction="none")
        return rows.detach(), torch.autograd.grad(rows.sum(), zz)[0]
    one = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        two = both()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(one, two))
    zz = z[:0].requires_grad_(True)
    loss = _ops().distillation_loss(zz, ids[:0], t[:0], lse[:0])
    assert loss == 0 and torch.autograd.grad(loss, zz)[0].shape == (0, 20000)


def test_top_logits_feed_the_loss():
    """A student equal to its teacher: no divergence and no gradient beyond rounding."""
    z = _logits(20, 5000, F32, 28)
    top = _ops().top_logits(z, 64, temperature=2.0)
    zz = z.clone().requires_grad_(True)
    loss = _ops().distillation_loss(zz, top.ids, top.values, top.lse, temperature=2.0, reduction="none")
    assert (loss.abs() <= 4 * 64 * U * 40).all()
    (g,) = torch.autograd.grad(loss.sum(), zz)
    assert (g.abs() <= 2 * 64 * U * 40).all()


def test_ids_outside_the_vocabulary_are_reported():
    from tensor_train_ing_b200.ops._ext import check_status
    z = _logits(3, 100, F32, 29)
    ids, t, _ = _teacher(z, 4, F32, 30, False, 1.0)
    check_status()
    bad = ids.clone()
    bad[0, 1] = 100
    got = _ops().distillation_loss(z, bad, t, reduction="none")
    with pytest.raises(RuntimeError, match="index out of range"):
        check_status()
    bad[0, 1] = -1
    assert torch.equal(got, _ops().distillation_loss(z, bad, t, reduction="none"))
    y = torch.tensor([1, 100, 2], device="cuda")
    got = _ops().distillation_loss(z, ids, t, targets=y, reduction="none")
    with pytest.raises(RuntimeError, match="index out of range"):
        check_status()
    assert got[1] == 0


def test_refusals():
    d = _ops()
    z = _logits(4, 50, F32, 31)
    ids = torch.zeros(4, 3, dtype=torch.int32, device="cuda")
    t = torch.zeros(4, 3, device="cuda")
    bad = [
        (ValueError, "CUDA", lambda: d.top_logits(z.cpu(), 2)),
        (TypeError, "float32", lambda: d.top_logits(z.double(), 2)),
        (ValueError, "k must be", lambda: d.top_logits(z, 0)),
        (ValueError, "k must be", lambda: d.top_logits(z, 51)),
        (ValueError, "k must be", lambda: d.top_logits(torch.zeros(1, 999, device="cuda"), 257)),
        (ValueError, "temperature", lambda: d.top_logits(z, 2, temperature=0.0)),
        (ValueError, "at least one column", lambda: d.top_logits(z[:, :0], 1)),
        (ValueError, "shared memory", lambda: d.top_logits(torch.empty(1, 1 << 20, device="cuda"), 2)),
        (ValueError, "same shape", lambda: d.distillation_loss(z, ids[:, :2], t)),
        (ValueError, "rows of logits", lambda: d.distillation_loss(z, ids[:2], t[:2])),
        (ValueError, "entries", lambda: d.distillation_loss(z, ids[:, :0], t[:, :0])),
        (TypeError, "int32 or int64", lambda: d.distillation_loss(z, ids.short(), t)),
        (TypeError, "teacher_logits", lambda: d.distillation_loss(z, ids, t.double())),
        (TypeError, "float32", lambda: d.distillation_loss(z.double(), ids, t)),
        (ValueError, "targets", lambda: d.distillation_loss(z, ids, t, ce_weight=0.5)),
        (ValueError, "targets has", lambda: d.distillation_loss(z, ids, t, targets=torch.zeros(3, device="cuda").long())),
        (RuntimeError, "targets", lambda: d.distillation_loss(z, ids, t, targets=torch.zeros(4, device="cuda"))),
        (ValueError, "teacher_lse has", lambda: d.distillation_loss(z, ids, t, t)),
        (ValueError, "temperature", lambda: d.distillation_loss(z, ids, t, temperature=-1.0)),
        (ValueError, "reduction", lambda: d.distillation_loss(z, ids, t, reduction="mean")),
        (ValueError, "scale", lambda: d.distillation_loss(z, ids, t, scale=torch.ones(2, device="cuda"))),
        (RuntimeError, "CUDA tensor", lambda: d.distillation_loss(z, ids.cpu(), t)),
    ]
    for kind, text, call in bad:
        with pytest.raises(kind, match=text):
            call()
    assert torch.isfinite(d.distillation_loss(z, ids, t))  # refused calls leave the context usable


# The loss forms first derivatives.  A second one, or a tangent, is refused and never left out of a sum.
@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("reduction", ["sum", "none"])
def test_second_derivatives_are_refused(reduction, dtype):
    z = _logits(6, 900, dtype, 32).requires_grad_(True)
    ids, t, lse = _teacher(z, 6, F32, 33, True, 1.0)
    s = torch.ones((), device="cuda", requires_grad=True)
    loss = lambda: _ops().distillation_loss(z, ids, t, lse, reduction=reduction).sum()  # noqa: E731
    (want,) = torch.autograd.grad(loss(), z)
    for leaf in (z, s):
        first = loss()
        (g,) = torch.autograd.grad(first * s, z, create_graph=True)
        assert torch.equal(g, want)
        for objective in (g.float().square().sum(), first.detach() * s + z.sum() + g.float().square().sum()):
            with pytest.raises(RuntimeError, match="distillation_loss.*second derivative"):
                torch.autograd.grad(objective, leaf, retain_graph=True, allow_unused=True)


@pytest.mark.parametrize("record", [False, True])
def test_tangents_are_refused(record):
    import torch.autograd.forward_ad as fwd
    z = _logits(6, 900, F32, 34)
    ids, t, lse = _teacher(z, 6, F32, 35, True, 1.0)
    with fwd.dual_level():
        dual = fwd.make_dual(z.requires_grad_(record), torch.ones_like(z))
        with pytest.raises(RuntimeError, match="distillation_loss.*forward-mode"):
            _ops().distillation_loss(dual, ids, t, lse)


@pytest.mark.parametrize("reduction", ["sum", "none"])
@pytest.mark.parametrize("n,v", [(6, 3001), (700, 50257), (6, 50257)])
def test_factors_reach_an_fp16_gradient_before_it_is_rounded(n, v, reduction):
    """What a loss scaler does: the loss is one over many tokens, the factor arrives in the backward.  The rounding to fp16
    comes after both, so nothing of the gradient is lost below 2^-25."""
    z = _logits(n, v, F16, 36, ld=v + 7)
    ids, t, lse = _teacher(z, 9, F32, 37, True, 2.0)
    y = _targets(n, v, ids, 38)
    weights = torch.ones(n, device="cuda") if reduction == "sum" else \
        torch.tensor([1.0, 0.5, -3.0], device="cuda").repeat(n // 3 + 1)[:n]
    scale, factor = 2.0 ** -17, 49152.0
    zz = z.detach().requires_grad_(True)
    loss = _ops().distillation_loss(zz, ids, t, lse, y, temperature=2.0, ce_weight=0.5, scale=scale, reduction=reduction)
    objective = factor * (loss if reduction == "sum" else (loss * weights).sum())
    (got,) = torch.autograd.grad(objective, zz, retain_graph=True)
    _, grad, _, gtol = _reference(z, ids, t, lse, y, 2.0, 1.0, 0.5, scale * factor)
    grad, gtol = grad * weights[:, None], gtol * weights.abs()[:, None].clamp_min(1)
    bad = (got.double() - grad).abs() > gtol
    assert got.dtype == F16 and not bad.any(), (bad.nonzero()[:5], got[bad][:5], grad[bad][:5], gtol[bad][:5])
    assert (got != 0).float().mean() > 0.3  # most of it would be zero without the factor
    with pytest.raises(RuntimeError, match="earlier backward"):
        torch.autograd.grad(objective, zz)


def _direct(z, ids, t, lse, y, tau, kd, ce, scale, dz):
    from tensor_train_ing_b200.ops._ext import lib
    return lib().distill_loss(z, ids, t, lse, y, tau, kd, ce, torch.full((1,), scale, device="cuda"), dz)


# What the trainer calls: fp32 logits cut from a padded buffer, a bf16 gradient as wide as that buffer.
@pytest.mark.parametrize("n,v,ld,offset", [(601, 50257, 50304, 0), (601, 50257, 50257, 1), (601, 131071, 131072, 0),
                                           (1201, 16385, 16448, 0), (1201, 20000, 20032, 4), (40, 50257, 50304, 0),
                                           (3, 500, 512, 2), (9, 4097, 4104, 3)])
@pytest.mark.parametrize("k,rest,tau,ce", [(1, False, 1.0, 0.0), (40, True, 2.0, 0.5), (64, True, 1.5, 0.25),
                                           (64, False, 4.0, 0.5)])
def test_fp32_logits_with_a_bf16_gradient(n, v, ld, offset, k, rest, tau, ce):
    z = _logits(n, v, F32, v + k, ld=ld, offset=offset)
    ids, t, lse = _teacher(z, k, F32, k, rest, tau)
    y = _targets(n, v, ids, 5)
    y[torch.rand(n, device="cuda", generator=_gen(6)) < 0.3] = -100
    y[0], y[1] = 0, v - 1
    loss, grad, tol, gtol = _reference(z, ids, t, lse, y, tau, 0.9, ce, 0.5)
    gtol = gtol + HALF_ULP[BF16] * 1.01 * grad.abs()
    for width, skip in ((ld, 0), (v, 0), (ld + 5, 1)):  # the buffer's width, the logits', rows off 16 bytes
        flat = torch.full((n * width + 1,), float("nan"), device="cuda", dtype=BF16)
        dz = flat[skip:skip + n * width].view(n, width)
        rows = _direct(z, ids, t, lse, y, tau, 0.9, ce, 0.5, dz)
        assert ((rows.double() - loss).abs() <= tol).all()
        bad = ~((dz[:, :v].double() - grad).abs() <= gtol)
        assert not bad.any(), (bad.nonzero()[:5], dz[:, :v][bad][:5], grad[bad][:5], gtol[bad][:5])
        assert not dz[:, v:].any() and flat[:skip].isnan().all() and flat[skip + n * width:].isnan().all()


@pytest.mark.parametrize("dtype,v,offset", [(F32, 20011, 1), (BF16, 50257, 3), (BF16, 901, 0)])
@pytest.mark.parametrize("n", [700, 12])
def test_columns_named_many_times_give_the_same_bits(n, dtype, v, offset):
    z = _logits(n, v, dtype, 60, offset=offset)
    ids, t, lse = _teacher(z, 300, F32, 61, True, 2.0)
    some = torch.tensor([0, 1, v - 1, v // 2, v // 3, 257, 258], device="cuda", dtype=torch.int32)
    ids = torch.where(torch.rand(n, 300, device="cuda", generator=_gen(62)) < 0.5, ids,
                      some[torch.randint(0, 7, (n, 300), device="cuda", generator=_gen(63))])
    lse = torch.logsumexp(t / 2.0, 1) + 0.2
    y = _targets(n, v, ids, 64)
    _check_loss(z, ids, t, lse, y, 2.0, 1.0, 0.5)
    once = None
    for _ in range(12):
        zz = z.detach().requires_grad_(True)
        rows = _ops().distillation_loss(zz, ids, t, lse, y, temperature=2.0, ce_weight=0.5, reduction="none")
        got = rows.detach(), torch.autograd.grad(rows.sum(), zz)[0]
        once = once or got
        assert torch.equal(got[0], once[0]) and torch.equal(got[1], once[1])


@pytest.mark.parametrize("n", [700, 7])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_teacher_rows_without_any_logit(n, dtype):
    teacher = _logits(n, 30011, dtype, 39)
    teacher[::5] = float("-inf")
    top = _ops().top_logits(teacher, 12, temperature=2.0)
    assert (top.lse[::5] == float("-inf")).all()
    z = _logits(n, 30011, dtype, 40)
    y = _targets(n, 30011, top.ids, 41)
    there = top.ids.clone()
    there[::5] = -1  # the same teacher, its empty rows without entries
    lse = top.lse.clone()
    lse[::5] = 0.0
    for ce, targets in ((0.0, None), (0.5, y)):
        def both(ids, lse):
            zz = z.detach().requires_grad_(True)
            rows = _ops().distillation_loss(zz, ids, top.values, lse, targets, 2.0, 1.0, ce, reduction="none")
            return rows.detach(), torch.autograd.grad(rows.sum(), zz)[0]
        got, want = both(top.ids, top.lse), both(there, lse)
        assert torch.isfinite(got[0]).all()
        torch.testing.assert_close(got[0], want[0], rtol=64 * U, atol=64 * U)
        torch.testing.assert_close(got[1].float(), want[1].float(), rtol=2 * HALF_ULP[dtype] + 64 * U * 20, atol=1e-9)


def test_factors_are_refused_where_they_have_no_kernel():
    from tensor_train_ing_b200.ops._ext import lib
    one = torch.ones(1, device="cuda")
    ids, t = torch.zeros(4, 2, dtype=torch.int32, device="cuda"), torch.zeros(4, 2, device="cuda")
    for dtype in (F32, BF16, F16):
        z = _logits(4, 50, dtype, 42)
        for dz in (None, torch.empty_like(z)):
            if dtype == F16 and dz is not None:
                continue
            with pytest.raises((RuntimeError, ValueError), match="factors"):
                lib().distill_loss(z, ids, t, None, None, 1.0, 1.0, 0.0, None, dz, one)
    with pytest.raises((RuntimeError, ValueError), match="factor"):
        z = _logits(4, 50, F16, 42)
        lib().distill_loss(z, ids, t, None, None, 1.0, 1.0, 0.0, None, torch.empty_like(z), torch.ones(3, device="cuda"))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_lists_from_inference_mode(dtype):
    teacher = _logits(6, 900, dtype, 43)
    with torch.inference_mode():
        top = _ops().top_logits(teacher, 8, temperature=2.0)
        y = _targets(6, 900, top.ids, 44)
        scale = torch.full((1,), 0.5, device="cuda")
    z = _logits(6, 900, dtype, 45).requires_grad_(True)
    loss = lambda *a: _ops().distillation_loss(z, *a, temperature=2.0, ce_weight=0.5, scale=0.5)  # noqa: E731
    (want,) = torch.autograd.grad(4.0 * loss(top.ids.clone(), top.values.clone(), top.lse.clone(), y.clone()), z)
    (got,) = torch.autograd.grad(4.0 * _ops().distillation_loss(z, top.ids, top.values, top.lse, y, temperature=2.0,
                                                              ce_weight=0.5, scale=scale), z)
    assert torch.equal(got, want) and got.any()


@pytest.mark.parametrize("which", range(6))
def test_fp16_inputs_changed_before_the_backward_are_reported(which):
    z = _logits(6, 900, F16, 46)
    ids, t, lse = _teacher(z, 6, F32, 47, True, 1.0)
    y, scale = _targets(6, 900, ids, 48), torch.ones(1, device="cuda")
    zz = z.clone().requires_grad_(True)
    logits = zz * 1
    inputs = [logits, ids, t, lse, y, scale]
    loss = _ops().distillation_loss(logits, ids, t, lse, y, ce_weight=0.5, scale=scale)
    with torch.no_grad():
        inputs[which].add_(0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation|changed in place"):
        torch.autograd.grad(8.0 * loss, zz)
