"""Top logits and the distillation loss where a row's logits lie far apart or are large (B200).

The oracle and its bounds are those of test_distill_gpu.py.  Rows are masked with finite values at many depths and places, so that a
thread's, a warp's or a whole stage's first logits lie anywhere from nothing to hundreds below the row's largest, at
temperatures where exponentials at 1 and at tau differ much."""
import pytest

from test_distill_gpu import BF16, F32, _check_loss, _check_top, _logits, _targets, _teacher

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
