"""Rows of the trainable layer norm whose values differ widely in size, on the GPU: a large value where a warp's
columns begin, and an offset far above the spread.  Errors are bounded by the rows' spread around their mean,
not by their distance from any one element."""
from __future__ import annotations

import pytest
import torch

import fp8_reference as R
import hc

pytestmark = pytest.mark.gpu

EPS = 1e-5
COLUMNS = 512  # of a warp in the row kernels, for the lengths below
ROWS = 7


def bounds(x, whole_rows):
    """How far xh, mean and rstd may be off in fp32.  With D = mean |x - mean| and W warps of 512 columns, each of which
    works around the mean of half of its columns: that lies within S D of the row's, S = 2 W (the mean deviation of
    1 / S of a row's elements is at most S times the row's), and within 2 D in the mean over the warps.
      each warp's residual sum has 16 additions at most, of magnitudes that are 3 D in the mean of the row;
      the warps' means are joined from their distances to the first one's, (2 + S) D in the mean, in 8 roundings;
      a column's own value passes roundings of its warp's distance (S D, six times) and of its own (twice);
      a sum of squares has 24 roundings and twice the mean's error, rstd half of that and 4 of rsqrt.
    Over 8192 columns a thread of 256 adds H / 256 terms, and 15 more additions follow."""
    x = x.double()
    H = x.shape[-1]
    mean = x.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean(-1, keepdim=True) + EPS)
    xh = (x - mean) * rstd
    dev = (x - mean).abs().mean(-1, keepdim=True)
    if whole_rows:
        S = 2 * H // COLUMNS
        shift, squares = R.U * (16 * 3 + 8 * (2 + S) + 6 * S) * dev, 24
    else:
        shift, squares = R.U * (H // 256 + 15) * dev, H // 256 + 24
    e_rstd = R.U * squares + 2 * shift * rstd
    d_xh = rstd * (shift + 2 * R.U * (x - mean).abs()) + xh.abs() * (2 * R.U + e_rstd)
    return (xh, mean, rstd), (1.01 * d_xh, 1.01 * shift + R.U * mean.abs(), e_rstd * rstd)


def rows(H, kind, where, big, aligned):
    x = torch.randn(ROWS, H, generator=torch.Generator().manual_seed(H))
    run = 32 * {"f32": 4, "f16": 8, "bf16": 8}[kind] if aligned else 32  # columns of a warp that lie side by side
    if where == "offset":
        x += big
    elif where == "first":
        x[:, 0] = big
    else:
        first = torch.arange(max(H // COLUMNS, 1)) * run
        x[:, first] = big * (1 + first / H)
    x[::2] *= -1
    x = x.to(R.DTYPES[kind])
    if aligned:
        return x.cuda()
    return torch.empty(1 + x.numel(), dtype=x.dtype, device="cuda")[1:].view(x.shape).copy_(x)


@pytest.mark.parametrize("where", ["first", "warps", "offset"])
@pytest.mark.parametrize("big", [1e2, 1e4, 1e6])
@pytest.mark.parametrize("kind,aligned", [("f32", True), ("f32", False), ("bf16", True)])
@pytest.mark.parametrize("H", [512, 1024, 2048, 4096, 8192, 16384])
def test_statistics_and_rows(cuda, H, kind, aligned, big, where):
    x = rows(H, kind, where, big, aligned)
    gamma, beta = torch.ones(H, device="cuda"), torch.zeros(H, device="cuda")
    (xh, mean, rstd), (d_xh, d_mean, d_rstd) = bounds(x, H <= 8192)
    y, got_mean, got_rstd = hc.layer_norm_fwd_train(x, gamma, beta, EPS)
    R.assert_within(got_mean, mean[:, 0], d_mean[:, 0], "mean")
    R.assert_within(got_rstd, rstd[:, 0], d_rstd[:, 0], "rstd")
    R.assert_within(y, xh, d_xh, "y")
    y, q, scale, got_rstd = hc.layer_norm_ckpt(x, gamma, beta, EPS)
    R.assert_within(got_rstd, rstd[:, 0], d_rstd[:, 0], "rstd of the checkpoint")
    R.assert_within(y, xh, d_xh, "y of the checkpoint")
    kept = (R.values(q, scale) - xh).abs()
    assert bool((kept <= d_xh + (xh.abs() + d_xh) * 2.0**-4 * (1 + 8 * R.U) + R.spread(scale, x.shape) * 2.0**-10 * (1 + 8 * R.U)).all())


@pytest.mark.parametrize("H", [5, 513, 1000, 1001, 6000, 9000])
def test_two_values_one_step_apart(cuda, H):
    """Rows of 1e6 with one element an fp32 step (2^-4) higher: the spread is that of the step, however the mean rounds."""
    x = torch.full((4, H), 1e6, device="cuda")
    for r, c in enumerate((0, 1, H // 2, H - 1)):
        x[r, c] += 2.0**-4
    gamma, beta = torch.ones(H, device="cuda"), torch.zeros(H, device="cuda")
    y, mean, rstd = hc.layer_norm_fwd_train(x, gamma, beta, EPS)
    ref, xh, m, r = R.layer_norm(x, gamma, beta, EPS)
    # differences of neighbours are exact; their mean and squares pass at most H / 256 + 40 roundings
    n = (H // 256 + 40) * R.U
    R.assert_within(mean, m[:, 0], R.U * m[:, 0].abs(), "mean")
    R.assert_within(rstd, r[:, 0], n * r[:, 0], "rstd")
    R.assert_within(y, ref, 2 * n * (xh.abs() + r * 2.0**-4), "y")


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("H", [64, 512, 520, 1001, 4096, 9000])
def test_squares_past_the_largest_fp32(cuda, H, kind):
    """Finite rows whose squares overflow: rstd is 0, so is xh, and no NaN comes of the corrections."""
    x = (1e25 * (torch.arange(4 * H).reshape(4, H) % 3 - 0.5)).to(R.DTYPES[kind]).cuda()
    x[1] *= -1
    x[2, :H // 2] *= 1e-3
    x[3, 0] *= 1e5
    gamma, beta = torch.ones(H, device="cuda"), torch.randn(H, generator=torch.Generator().manual_seed(1)).cuda()
    y, mean, rstd = hc.layer_norm_fwd_train(x, gamma, beta, EPS)
    assert bool((rstd == 0).all()) and bool(mean.isfinite().all())
    assert torch.equal(y, beta.to(y.dtype).expand_as(y))
    y, q, scale, rstd = hc.layer_norm_ckpt(x, gamma, beta, EPS)
    assert bool((rstd == 0).all()) and torch.equal(y, beta.to(y.dtype).expand_as(y)) and bool((q.float() == 0).all())
