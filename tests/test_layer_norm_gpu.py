"""unet_layer_norm_* and unet_layer_norm_backward_* against the float64 definition (seq_ref.py, which also derives the
bounds): row lengths around every kernel's limits, strided and misaligned rows, in place, skipped halves, large offsets."""
import ctypes

import pytest
import torch

import seq_ref
from gpu_util import DEV, empty
from unet_amd import capi

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
FWD = {"f32": capi.unet_layer_norm_f32, "bf16": capi.unet_layer_norm_bf16}
BWD = {"f32": capi.unet_layer_norm_backward_f32, "bf16": capi.unet_layer_norm_backward_bf16}


def workspace(rows, c):
    n = ctypes.c_size_t()
    capi.unet_layer_norm_backward_workspace_bytes(rows, c, ctypes.byref(n))
    return torch.full((max(n.value, 1),), 255, dtype=torch.uint8, device=DEV)


def matrix(rows, c, dtype, seed, pad=0, scale=1.0, shift=0.0):
    """A [rows, c] view `pad` columns into a wider buffer (pad odd: rows start at odd elements)."""
    g = torch.Generator().manual_seed(seed)
    wide = (torch.randn(rows, c + 2 * pad, generator=g) * scale + shift).to(dtype).to(DEV)
    return wide[:, pad:pad + c]


def stream():
    return torch.cuda.current_stream().cuda_stream


# 16-lane rows, one and more wavefronts a row, the workgroup, rows that do not fit registers; lengths that end inside a piece
CASES = [(1, 1), (3, 2), (5, 7), (17, 32), (33, 77), (9, 128), (21, 129), (1, 256), (40, 321), (7, 512), (1000, 96), (3, 513), (6, 1000),
         (2500, 1024), (4, 1025), (5, 2048), (3, 4096), (2, 4099), (3, 8192), (70, 8200)]


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("rows,c", CASES)
@pytest.mark.parametrize("pad", [0, 3])
def test_forward_and_backward(name, rows, c, pad):
    dtype = TYPES[name]
    x = matrix(rows, c, dtype, rows * 7919 + c, pad, 1.5, 0.7)
    dy, skip = matrix(rows, c, dtype, c + 1, pad), matrix(rows, c, dtype, c + 2, pad + 1)
    w = (torch.randn(c, 2, generator=torch.Generator().manual_seed(c)) * 0.3 + torch.tensor([1.0, 0.0])).to(DEV)
    wide = torch.full((rows + 1, c + 5), 7.0, dtype=dtype, device=DEV)
    y, stats = wide[:rows, 1:1 + c], empty((rows, 2))
    FWD[name](x.data_ptr(), x.stride(0), y.data_ptr(), y.stride(0), w.data_ptr(), stats.data_ptr(), rows, c, 1e-5, stream())
    val, bnd = seq_ref.layer_norm(x, w, 1e-5, dy, skip)
    store = seq_ref.half_step(dtype) if name == "bf16" else 0.0
    seq_ref.check(y, val["y"], bnd["y"] + store * val["y"].abs(), "y")
    seq_ref.check(stats[:, :1], val["mean"], bnd["mean"], "mean")
    seq_ref.check(stats[:, 1:], val["rstd"], bnd["rstd"], "rstd")
    assert (wide[rows] == 7).all() and (wide[:, 0] == 7).all() and (wide[:, 1 + c:] == 7).all()

    wide = torch.full((rows + 1, c + 5), 7.0, dtype=dtype, device=DEV)
    dx, dw, ws = wide[:rows, 1:1 + c], empty((c, 2)), workspace(rows, c)

    def back(dx_, dw_, skip_=skip):
        BWD[name](dy.data_ptr(), dy.stride(0), x.data_ptr(), x.stride(0), stats.data_ptr(), w.data_ptr(),
                  None if skip_ is None else skip_.data_ptr(), 0 if skip_ is None else skip_.stride(0),
                  None if dx_ is None else dx_.data_ptr(), 0 if dx_ is None else dx_.stride(0), None if dw_ is None else dw_.data_ptr(), rows, c,
                  ws.data_ptr(), ws.numel(), stream())

    back(dx, dw)
    # the kernel reads the statistics it was given: their own bounds come on top, and act like an error of xhat
    seq_ref.check(dx, val["dx"], 2 * bnd["dx"] + store * val["dx"].abs(), "dx")
    seq_ref.check(dw, val["dw"], 2 * bnd["dw"], "dweights")
    assert (wide[rows] == 7).all() and (wide[:, 0] == 7).all() and (wide[:, 1 + c:] == 7).all()
    # each half alone gives the same bits; without the skip gradient
    dx2, dw2 = torch.empty(rows, c, dtype=dtype, device=DEV), empty((c, 2))
    back(dx2, None)
    back(None, dw2)
    assert torch.equal(dx2, dx) and torch.equal(dw2, dw)
    back(dx2, None, None)
    val, bnd = seq_ref.layer_norm(x, w, 1e-5, dy)
    seq_ref.check(dx2, val["dx"], 2 * bnd["dx"] + store * val["dx"].abs(), "dx without skip")


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("c", [64, 1000, 8200])
def test_in_place_and_without_weights(name, c):
    dtype, rows = TYPES[name], 37
    x, dy = matrix(rows, c, dtype, 5).clone(), matrix(rows, c, dtype, 6)
    y, stats = empty((rows, c), dtype), empty((rows, 2))
    FWD[name](x.data_ptr(), c, y.data_ptr(), c, None, stats.data_ptr(), rows, c, 1e-5, stream())
    val, bnd = seq_ref.layer_norm(x, None, 1e-5, dy)
    seq_ref.check(y, val["y"], bnd["y"] + seq_ref.half_step(dtype) * val["y"].abs(), "y")
    dx = empty((rows, c), dtype)
    args = (stats.data_ptr(), None, None, 0)
    BWD[name](dy.data_ptr(), c, x.data_ptr(), c, *args, dx.data_ptr(), c, None, rows, c, None, 0, stream())
    for which in ("grad", "inputs"):  # grad_inputs in the buffer of either operand, with the weight gradient from the same call
        g, xx = dy.clone(), x.clone()
        to, dw, ref, ws = (g if which == "grad" else xx), empty((c, 2)), empty((c, 2)), workspace(rows, c)
        BWD[name](dy.data_ptr(), c, x.data_ptr(), c, *args, None, 0, ref.data_ptr(), rows, c, ws.data_ptr(), ws.numel(), stream())
        BWD[name](g.data_ptr(), c, xx.data_ptr(), c, *args, to.data_ptr(), c, dw.data_ptr(), rows, c, ws.data_ptr(), ws.numel(), stream())
        assert torch.equal(to, dx) and torch.equal(dw, ref)
    FWD[name](x.data_ptr(), c, x.data_ptr(), c, None, None, rows, c, 1e-5, stream())
    assert torch.equal(x, y)


def test_constant_rows_infinities_and_nan_stay_in_their_row():
    c = 200
    x = matrix(6, c, torch.float32, 1).clone()
    x[1] = 3.0
    x[2, 5] = float("inf")
    x[4, 7] = float("nan")
    y, stats = empty((6, c)), empty((6, 2))
    capi.unet_layer_norm_f32(x.data_ptr(), c, y.data_ptr(), c, None, stats.data_ptr(), 6, c, 1e-5, stream())
    assert (y[1] == 0).all() and torch.isnan(y[2]).any() and torch.isnan(y[4]).all()
    ok = [0, 3, 5]
    val, bnd = seq_ref.layer_norm(x[ok], None, 1e-5)
    seq_ref.check(y[ok], val["y"], bnd["y"], "other rows")


def test_no_rows_clear_the_weight_gradient():
    dw = empty((9, 2))
    capi.unet_layer_norm_backward_f32(None, 9, None, 9, None, None, None, 0, None, 0, dw.data_ptr(), 0, 9, None, 0, stream())
    assert (dw == 0).all()


def test_rows_beyond_32_bits_of_offset():
    rows, c, ld = 300, 40, 1 << 23  # 2.5e9 elements, 5 GB
    buf = torch.zeros(rows * ld, dtype=torch.bfloat16, device=DEV)
    x = buf.view(rows, ld)[:, 8:8 + c]
    src = matrix(rows, c, torch.bfloat16, 3)
    x.copy_(src)
    y, y2 = empty((rows, c), torch.bfloat16), empty((rows, c), torch.bfloat16)
    capi.unet_layer_norm_bf16(src.data_ptr(), c, y.data_ptr(), c, None, None, rows, c, 1e-5, stream())
    capi.unet_layer_norm_bf16(x.data_ptr(), ld, y2.data_ptr(), c, None, None, rows, c, 1e-5, stream())
    assert torch.equal(y, y2)
    capi.unet_layer_norm_bf16(x.data_ptr(), ld, x.data_ptr(), ld, None, None, rows, c, 1e-5, stream())
    assert torch.equal(x, y)


def test_captured_and_replayed_beside_eager_work():
    rows, c = 3000, 768
    x, dy = matrix(rows, c, torch.bfloat16, 1), matrix(rows, c, torch.bfloat16, 2)
    w = torch.randn(c, 2, device=DEV)
    out = [empty((rows, c), torch.bfloat16), empty((rows, 2)), empty((rows, c), torch.bfloat16), empty((c, 2)), workspace(rows, c)]

    def step(y, stats, dx, dw, ws):
        capi.unet_layer_norm_bf16(x.data_ptr(), c, y.data_ptr(), c, w.data_ptr(), stats.data_ptr(), rows, c, 1e-5, stream())
        capi.unet_layer_norm_backward_bf16(dy.data_ptr(), c, x.data_ptr(), c, stats.data_ptr(), w.data_ptr(), None, 0, dx.data_ptr(), c,
                                           dw.data_ptr(), rows, c, ws.data_ptr(), ws.numel(), stream())

    step(*out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(*out)
    for i in range(4):
        x.copy_(matrix(rows, c, torch.bfloat16, 10 + i))
        ref = [torch.empty_like(t) for t in out]
        step(*ref)
        for t in out:
            t.fill_(0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out[:4], ref):
            assert torch.equal(a, b)
