"""unet_dropout_* against the stated generator (seq_ref.py, numpy): the mask bit for bit, whatever the stride, alignment and type."""
import pytest
import torch

import seq_ref
from gpu_util import DEV, empty
from unet_amd import capi

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
FWD = {"f32": capi.unet_dropout_f32, "bf16": capi.unet_dropout_bf16}
BWD = {"f32": capi.unet_dropout_backward_f32, "bf16": capi.unet_dropout_backward_bf16}


def stream():
    return torch.cuda.current_stream().cuda_stream


def matrix(rows, c, dtype, seed, pad=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(rows, c + 2 * pad, generator=g).to(dtype).to(DEV)[:, pad:pad + c]


def wanted(x, res, kept, p):
    """x / (1 - p) where kept, plus res: the scale, the product and the sum are each off by at most half a step of fp32."""
    x = x.double().cpu()
    v = torch.where(kept, x / (1 - p) if p < 1 else torch.zeros_like(x), torch.zeros_like(x))
    r = torch.zeros_like(x) if res is None else res.double().cpu()
    return v + r, 2.1 * seq_ref.U * v.abs() + (0 if res is None else 1) * seq_ref.U * (v + r).abs()


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("rows,c,pad", [(1, 1, 0), (1, 7, 1), (3, 8, 0), (5, 9, 0), (5, 9, 3), (64, 77, 0), (64, 77, 1), (33, 320, 8), (1000, 1024, 0),
                                        (7, 3, 2), (2, 100003, 0)])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 1.0])
@pytest.mark.parametrize("residual", [False, True])
def test_forward_and_backward(name, rows, c, pad, p, residual):
    dtype, seed, offset = TYPES[name], 0x123456789ABCDEF0 + c, (7 << 32) + rows
    x = matrix(rows, c, dtype, c, pad)
    res = matrix(rows, c, dtype, c + 1, pad + 1) if residual else None
    wide = torch.full((rows + 1, c + 3), 7.0, dtype=dtype, device=DEV)
    out = wide[:rows, 1:1 + c] if pad else torch.empty(rows, c, dtype=dtype, device=DEV)
    FWD[name](x.data_ptr(), x.stride(0), None if res is None else res.data_ptr(), 0 if res is None else res.stride(0), out.data_ptr(),
              out.stride(0), rows, c, p, seed, offset, None, stream())
    kept = seq_ref.dropout_kept(rows, c, p, seed, offset)
    val, bnd = wanted(x, res, kept, p)
    seq_ref.check(out, val, bnd + (seq_ref.half_step(dtype) * val.abs() if name == "bf16" else 0), "out")
    if pad:
        assert (wide[rows] == 7).all() and (wide[:, 0] == 7).all() and (wide[:, 1 + c:] == 7).all()
    if not residual:
        assert torch.equal((out != 0).cpu(), kept & (x != 0).cpu())
        back = empty((rows, c), dtype)
        BWD[name](x.data_ptr(), x.stride(0), back.data_ptr(), c, rows, c, p, seed, offset, None, stream())
        assert torch.equal(back, out)


def test_probability_is_resolved_to_32_bits():
    """p a little above and below the number of an element that shares its upper 16 bits with the threshold."""
    n, seed, offset = 1 << 20, 99, 5
    numbers = torch.from_numpy(seq_ref.dropout_numbers(n, seed, offset).astype("int64"))
    x, out = torch.ones(1, n, device=DEV), empty((1, n))
    for at in (0, 12345, n - 1):
        u = int(numbers[at])
        for t in (u, u + 1):
            capi.unet_dropout_f32(x.data_ptr(), n, None, 0, out.data_ptr(), n, 1, n, t / 2 ** 32, seed, offset, None, stream())
            assert torch.equal((out != 0).cpu()[0], numbers >= t)
            assert bool(out[0, at] != 0) == (t == u)


def test_dropped_elements_are_zero_whatever_they_hold():
    n = 4096
    x = torch.full((1, n), float("inf"), device=DEV)
    x[0, ::2] = float("nan")
    res, out = torch.full((1, n), 2.0, device=DEV), empty((1, n))
    capi.unet_dropout_f32(x.data_ptr(), n, res.data_ptr(), n, out.data_ptr(), n, 1, n, 0.3, 1, 2, None, stream())
    kept = seq_ref.dropout_kept(1, n, 0.3, 1, 2)
    assert (out.cpu()[~kept] == 2).all() and not torch.isfinite(out.cpu()[kept]).any()


def test_in_place():
    rows, c = 50, 321
    x, res = matrix(rows, c, torch.bfloat16, 1).clone(), matrix(rows, c, torch.bfloat16, 2).clone()
    out = torch.empty_like(x)
    args = (rows, c, 0.2, 3, 4, None, stream())
    capi.unet_dropout_bf16(x.data_ptr(), c, res.data_ptr(), c, out.data_ptr(), c, *args)
    r2 = res.clone()
    capi.unet_dropout_bf16(x.data_ptr(), c, r2.data_ptr(), c, r2.data_ptr(), c, *args)
    assert torch.equal(r2, out)
    capi.unet_dropout_bf16(x.data_ptr(), c, res.data_ptr(), c, x.data_ptr(), c, *args)
    assert torch.equal(x, out)


def test_more_elements_than_32_bits():
    """A matrix of 2^32 + 24 elements, 8.6 GB in place; its last rows against the generator."""
    c = 8
    rows = (1 << 29) + 3
    x = torch.ones(rows, c, dtype=torch.bfloat16, device=DEV)
    capi.unet_dropout_bf16(x.data_ptr(), c, None, 0, x.data_ptr(), c, rows, c, 0.5, 11, 12, None, stream())
    for first in (0, (1 << 32) - 800, (1 << 32)):
        n = min(1600, rows * c - first)
        numbers = seq_ref.dropout_numbers(n, 11, 12, first)
        assert torch.equal((x.view(-1)[first:first + n] != 0).cpu(), torch.from_numpy(numbers >= 2 ** 31))


def test_a_captured_graph_draws_a_new_mask_per_replay():
    rows, c = 77, 130
    x, out = matrix(rows, c, torch.float32, 1), empty((rows, c))
    count = torch.tensor([5], dtype=torch.int64, device=DEV)

    def call(to, offset, dev):
        capi.unet_dropout_f32(x.data_ptr(), c, None, 0, to.data_ptr(), c, rows, c, 0.4, 21, offset, dev, stream())

    call(out, 100, count.data_ptr())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(out, 100, count.data_ptr())
        count.add_(1)
    for i in range(4):
        out.fill_(0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        ref = empty((rows, c))
        call(ref, 105 + i, None)
        assert torch.equal(out, ref)
        assert int(count) == 6 + i
