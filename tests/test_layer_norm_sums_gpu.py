"""unet_layer_norm_*: sums of very many terms.  Equal terms that are no multiple of the running sum's step are rounded to the same
side again and again, so a long fp32 chain is off by more the longer it is.  The bounds here do not grow with the length."""
import ctypes

import pytest
import torch

import seq_ref
from gpu_util import DEV, empty
from unet_amd import capi

pytestmark = pytest.mark.gpu
U = seq_ref.U
UNEVEN = 1 + 0.49 * 2.0 ** -13  # rounded to 1 by a sum of 2^11 and more


def stream():
    return torch.cuda.current_stream().cuda_stream


def backward(dy, x, stats, w, dx, dw):
    rows, c = x.shape
    n = ctypes.c_size_t()
    capi.unet_layer_norm_backward_workspace_bytes(rows, c, ctypes.byref(n))
    ws = torch.empty(max(n.value, 1), dtype=torch.uint8, device=DEV)
    capi.unet_layer_norm_backward_f32(dy.data_ptr(), c, x.data_ptr(), c, stats.data_ptr(), None if w is None else w.data_ptr(), None, 0,
                                      None if dx is None else dx.data_ptr(), c, None if dw is None else dw.data_ptr(), rows, c, ws.data_ptr(), ws.numel(),
                                      stream())


@pytest.mark.parametrize("c", [1 << 22, (1 << 22) + 77])
def test_rows_of_millions_of_channels(c):
    """Row 0: all equal.  Row 1: +-a, so that the squares are all equal.  Row 2: random.  A thread's share is added up in double, 256
    shares in a tree of 8 sums: 16 U cover these, the division and the roundings of a term."""
    a = UNEVEN ** 0.5
    x = torch.stack([torch.full((c,), UNEVEN), a * (1 - 2.0 * (torch.arange(c) % 2)), torch.randn(c, generator=torch.Generator().manual_seed(1)) * 2 + 1])
    x = x.to(DEV)
    y, stats = empty((3, c)), empty((3, 2))
    eps = 1e-2
    capi.unet_layer_norm_f32(x.data_ptr(), c, y.data_ptr(), c, None, stats.data_ptr(), 3, c, eps, stream())
    xd = x.double()
    mean = xd.mean(1, keepdim=True)
    d = xd - mean
    var = (d * d).mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    e_mean = 16 * U * xd.abs().mean(1, keepdim=True)
    e_d = e_mean + U * d.abs()
    rel = ((d.abs() * e_d).mean(1, keepdim=True) + e_mean ** 2 + 16 * U * var) / (var + eps) + 4 * U
    e_xhat = rstd * e_d + (d * rstd).abs() * (rel + 2 * U)
    seq_ref.check(stats[:, :1], mean, e_mean, "mean")
    seq_ref.check(stats[:, 1:], rstd, rstd * rel, "rstd")
    seq_ref.check(y, d * rstd, e_xhat + 2 * U * (d * rstd).abs(), "y")

    dy, dx = torch.full_like(x, UNEVEN), empty((3, c))
    dy[1] = x[1]
    dy[2] += x[2].abs()
    backward(dy, x, stats, None, dx, None)
    g, xhat = dy.double(), d * rstd
    m0, m1 = g.mean(1, keepdim=True), (g * xhat).mean(1, keepdim=True)
    want = rstd * (g - m0 - xhat * m1)
    by_xhat = rstd * (e_xhat * m1.abs() + xhat.abs() * (g.abs() * e_xhat).mean(1, keepdim=True))
    size = rstd * (g.abs() + g.abs().mean(1, keepdim=True) + xhat.abs() * (g * xhat).abs().mean(1, keepdim=True))
    # the statistics that it was given are off by their own bounds: twice
    seq_ref.check(dx, want, 2 * (by_xhat + size * (rel + 24 * U)), "dx")


@pytest.mark.parametrize("rows,c", [((1 << 25) + 5, 4), ((1 << 23) + 3, 100), (1 << 20, 260)])
def test_columns_of_millions_of_rows(rows, c):
    """All rows of a column hold the same x and dy.  A lane adds at most 256 rows (each a rounding of the sum, of the product and
    of xhat behind the stored statistics), then 16 groups of a workgroup, at most 16 launches here, and 512 partial rows in double."""
    g = torch.Generator().manual_seed(3)
    one = torch.randn(1, c, generator=g).to(DEV)
    x, stats, dw = one.expand(rows, c).contiguous(), empty((rows, 2)), empty((c, 2))
    dy = torch.full_like(x, UNEVEN)
    dy[:, 1] = -UNEVEN / 3
    dx = empty((rows, c))
    capi.unet_layer_norm_f32(x.data_ptr(), c, dx.data_ptr(), c, None, stats.data_ptr(), rows, c, 1e-5, stream())
    assert torch.equal(stats, stats[:1].expand(rows, 2))
    backward(dy, x, stats, None, dx, dw)
    xhat = (one[0].double() - stats[0, 0].double()) * stats[0, 1].double()
    want = torch.stack([dy[0].double() * xhat, dy[0].double()], 1) * rows
    seq_ref.check(dw, want, (256 + 16 + 16 + 4) * U * want.abs(), "dweights")
    assert torch.equal(dx, dx[:1].expand(rows, c))  # every launch's rows


def test_rows_of_several_launches():
    """Different rows, strides and a skip gradient: each launch begins at its own rows.  dx alone is one launch of the same rows."""
    rows, c = 300001, 1100  # a workgroup holds a row; 131072 rows a launch
    gen = torch.Generator(device=DEV).manual_seed(4)
    x, dy, skip = (torch.randn(rows, c + p, generator=gen, device=DEV)[:, :c] for p in (4, 0, 8))
    w = torch.randn(c, 2, generator=gen, device=DEV)
    stats, dx, alone, dw = empty((rows, 2)), empty((rows, c)), empty((rows, c)), empty((c, 2))
    capi.unet_layer_norm_f32(x.data_ptr(), x.stride(0), dx.data_ptr(), c, w.data_ptr(), stats.data_ptr(), rows, c, 1e-5, stream())
    n = ctypes.c_size_t()
    capi.unet_layer_norm_backward_workspace_bytes(rows, c, ctypes.byref(n))
    ws = torch.full((n.value + 4096,), 255, dtype=torch.uint8, device=DEV)
    args = (dy.data_ptr(), dy.stride(0), x.data_ptr(), x.stride(0), stats.data_ptr(), w.data_ptr(), skip.data_ptr(), skip.stride(0))
    capi.unet_layer_norm_backward_f32(*args, dx.data_ptr(), c, dw.data_ptr(), rows, c, ws.data_ptr(), n.value, stream())
    capi.unet_layer_norm_backward_f32(*args, alone.data_ptr(), c, None, rows, c, None, 0, stream())
    assert torch.equal(dx, alone) and (ws[n.value:] == 255).all()
    want, size = torch.zeros(c, 2, dtype=torch.float64, device=DEV), torch.zeros(c, 2, dtype=torch.float64, device=DEV)
    for r in range(0, rows, 50000):
        d = dy[r:r + 50000].double()
        t = torch.stack([d * (x[r:r + 50000].double() - stats[r:r + 50000, :1].double()) * stats[r:r + 50000, 1:].double(), d], 2)
        want += t.sum(0)
        size += t.abs().sum(0)
    seq_ref.check(dw, want, (256 + 16 + 4) * U * size, "dweights")
