"""Layer norm, dropout and dot-product attention without a GPU: what the entry points refuse, how much workspace
they ask for, and the float64 definitions that the GPU tests compare with against differences and autograd."""
import ctypes
import math

import numpy as np
import pytest
import torch

import seq_ref
from unet_amd import capi

P = 4096  # an address that no accepted call reaches: every call below is refused before any launch, or is empty


def ln(x=P, x_ld=8, y=P, y_ld=8, w=P, stats=P, rows=2, c=8, eps=1e-5, f=capi.unet_layer_norm_f32):
    f(x, x_ld, y, y_ld, w, stats, rows, c, eps, None)


@pytest.mark.parametrize("f", [capi.unet_layer_norm_f32, capi.unet_layer_norm_bf16])
@pytest.mark.parametrize("bad,match", [(dict(x=None), "NULL"), (dict(y=None), "NULL"), (dict(x_ld=7), "stride"), (dict(y_ld=7), "stride"),
                                       (dict(rows=-1), "rows"), (dict(c=0), "channels"), (dict(c=2 ** 26 + 1, x_ld=2 ** 27, y_ld=2 ** 27), "channels"), (dict(eps=-1.0), "eps"),
                                       (dict(eps=float("nan")), "eps"), (dict(x=P + 1), "misaligned"), (dict(w=P + 2), "misaligned")])
def test_layer_norm_refuses(f, bad, match):
    with pytest.raises(RuntimeError, match=match):
        ln(f=f, **bad)
    ln(f=f, rows=0, x=None, y=None)  # an empty call is fine


def ln_back(dy=P, dy_ld=8, x=P, x_ld=8, stats=P, w=P, skip=None, skip_ld=0, dx=P, dx_ld=8, dw=P, rows=2, c=8, ws=P, n=1 << 20,
            f=capi.unet_layer_norm_backward_f32):
    f(dy, dy_ld, x, x_ld, stats, w, skip, skip_ld, dx, dx_ld, dw, rows, c, ws, n, None)


@pytest.mark.parametrize("f", [capi.unet_layer_norm_backward_f32, capi.unet_layer_norm_backward_bf16])
@pytest.mark.parametrize("bad,match", [(dict(dy=None), "NULL"), (dict(x=None), "NULL"), (dict(stats=None), "NULL"), (dict(dy_ld=3), "stride"),
                                       (dict(x_ld=3), "stride"), (dict(dx_ld=3), "stride"), (dict(skip=P, skip_ld=3), "stride"),
                                       (dict(n=2 * 2 * 8 * 4 - 1), "workspace"), (dict(ws=None), "workspace"), (dict(ws=P + 4), "aligned"),
                                       (dict(rows=-1), "rows"), (dict(c=0), "channels"), (dict(dx=P + 1), "misaligned")])
def test_layer_norm_backward_refuses(f, bad, match):
    with pytest.raises(RuntimeError, match=match):
        ln_back(f=f, **bad)
    ln_back(f=f, rows=0, dw=None, dy=None, x=None, stats=None, ws=None, n=0)


def drop(x=P, x_ld=8, res=None, res_ld=0, y=P, y_ld=8, rows=2, c=8, p=0.1, off=None, f=capi.unet_dropout_f32):
    f(x, x_ld, res, res_ld, y, y_ld, rows, c, p, 1, 2, off, None)


@pytest.mark.parametrize("f", [capi.unet_dropout_f32, capi.unet_dropout_bf16])
@pytest.mark.parametrize("bad,match", [(dict(p=-0.01), "p ="), (dict(p=1.01), "p ="), (dict(p=float("nan")), "p ="), (dict(x=None), "NULL"),
                                       (dict(y=None), "NULL"), (dict(x_ld=7), "stride"), (dict(y_ld=7), "stride"), (dict(res=P, res_ld=7), "stride"),
                                       (dict(c=0), "channels"), (dict(rows=-1), "rows"), (dict(rows=2 ** 61), "too many"),
                                       (dict(x=P + 1), "misaligned"), (dict(off=P + 4), "misaligned")])
def test_dropout_refuses(f, bad, match):
    with pytest.raises(RuntimeError, match=match):
        drop(f=f, **bad)
    drop(f=f, rows=0, x=None, y=None)


def test_dropout_backward_refuses():
    for f in (capi.unet_dropout_backward_f32, capi.unet_dropout_backward_bf16):
        with pytest.raises(RuntimeError, match="p ="):
            f(P, 8, P, 8, 2, 8, 2.0, 1, 2, None, None)
        with pytest.raises(RuntimeError, match="stride"):
            f(P, 8, P, 7, 2, 8, 0.5, 1, 2, None, None)
        f(None, 8, None, 8, 0, 8, 0.5, 1, 2, None, None)


ATT = dict(q=P, q_ld=64, k=P, k_ld=32, v=P, v_ld=32, out=P, out_ld=64, lse=P, cu_q=P, cu_k=P, num_seqs=2, total_q=10, total_k=12, heads_q=4,
           heads_kv=2, head_dim=16, scale=0.25, causal=1, workspace=P, workspace_bytes=1 << 30, stream=None)
SHAPE = [(dict(heads_kv=3), "multiple"), (dict(heads_kv=0), "multiple"), (dict(heads_q=0), "multiple"), (dict(head_dim=0), "head_dim"),
         (dict(head_dim=129, q_ld=4096, k_ld=4096, v_ld=4096, out_ld=4096), "larger than 128"), (dict(num_seqs=-1), "num_seqs"),
         (dict(total_q=-1), "total_q"), (dict(total_k=2 ** 31), "too many"), (dict(total_q=2 ** 30), "too many"), (dict(scale=0.0), "scale"),
         (dict(scale=-1.0), "scale"), (dict(scale=float("inf")), "scale"), (dict(scale=float("nan")), "scale"), (dict(scale=3e38), "scale"), (dict(num_seqs=2 ** 30), "too many"), (dict(cu_q=None), "cu_q"),
         (dict(cu_k=None), "cu_k"), (dict(cu_k=P + 2), "misaligned"), (dict(q=None), "q is NULL"), (dict(k=None), "k is NULL"),
         (dict(v=None), "v is NULL"), (dict(q_ld=63), "stride of q"), (dict(k_ld=31), "stride of k"), (dict(v_ld=31), "stride of v"),
         (dict(q=P + 1), "misaligned")]


@pytest.mark.parametrize("f", [capi.unet_dot_attention_f32, capi.unet_dot_attention_bf16])
@pytest.mark.parametrize("bad,match", SHAPE + [(dict(out=None), "out is NULL"), (dict(out_ld=63), "stride of out"), (dict(lse=P + 2), "misaligned")])
def test_attention_refuses(f, bad, match):
    with pytest.raises(RuntimeError, match=match):
        f(*{**ATT, **bad}.values())
    f(*{**ATT, "total_q": 0, "q": None, "out": None}.values())
    f(*{**ATT, "num_seqs": 0, "cu_q": None, "cu_k": None}.values())


BACK = dict(grad_out=P, grad_out_ld=64, q=P, q_ld=64, k=P, k_ld=32, v=P, v_ld=32, out=P, out_ld=64, lse=P, grad_q=P, grad_q_ld=64, grad_k=P,
            grad_k_ld=32, grad_v=P, grad_v_ld=32, **{n: ATT[n] for n in list(ATT)[9:]})


@pytest.mark.parametrize("f", [capi.unet_dot_attention_backward_f32, capi.unet_dot_attention_backward_bf16])
@pytest.mark.parametrize("bad,match", [(b if "out_ld" not in b else {**b, "grad_out_ld": 4096, "grad_q_ld": 4096, "grad_k_ld": 4096, "grad_v_ld": 4096}, m)
                                       for b, m in SHAPE] +
                         [(dict(grad_out=None), "grad_out is NULL"), (dict(out=None), "out is NULL"), (dict(lse=None), "lse"),
                          (dict(grad_q=None), "grad_q is NULL"), (dict(grad_k=None), "grad_k is NULL"), (dict(grad_v=None), "grad_v is NULL"),
                          (dict(grad_v_ld=31), "stride of grad_v"), (dict(workspace_bytes=10 * 4 * 4 - 1), "workspace"),
                          (dict(workspace=None), "workspace"), (dict(workspace=P + 8), "aligned")])
def test_attention_backward_refuses(f, bad, match):
    with pytest.raises(RuntimeError, match=match):
        f(*{**BACK, **bad}.values())
    f(*{**BACK, "num_seqs": 0}.values())


def test_workspace_sizes():
    n = ctypes.c_size_t(7)
    capi.unet_layer_norm_backward_workspace_bytes(0, 5, ctypes.byref(n))
    assert n.value == 0
    capi.unet_layer_norm_backward_workspace_bytes(10 ** 9, 1024, ctypes.byref(n))
    assert n.value <= 8 << 20  # does not grow with the rows
    capi.unet_dot_attention_backward_workspace_bytes(3, 100, 50, 4, 2, 64, ctypes.byref(n))
    assert n.value >= 100 * 4 * 4
    with pytest.raises(RuntimeError, match="NULL"):
        capi.unet_dot_attention_workspace_bytes(3, 100, 50, 4, 2, 64, None)
    with pytest.raises(RuntimeError, match="multiple"):
        capi.unet_dot_attention_workspace_bytes(3, 100, 50, 4, 3, 64, ctypes.byref(n))


def test_generator_known_answers():
    # the published test vectors of Philox4x32-10
    zero = seq_ref.philox4x32_10(np.zeros((1, 4), np.uint64), (0, 0))[0]
    assert [int(w) for w in zero] == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    ones = seq_ref.philox4x32_10(np.full((1, 4), 0xFFFFFFFF, np.uint64), (0xFFFFFFFF, 0xFFFFFFFF))[0]
    assert [int(w) for w in ones] == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]


def test_generator_is_uniform_and_independent():
    n = 1 << 18
    a, b = seq_ref.dropout_numbers(n, 3, 0) / 2 ** 32, seq_ref.dropout_numbers(n, 3, 1) / 2 ** 32
    # means of n uniform numbers: standard deviation 1 / sqrt(12 n); products of independent ones likewise.  Six of them
    assert abs(a.mean() - 0.5) < 6 / math.sqrt(12 * n)
    assert abs(((a - 0.5) * (b - 0.5)).mean()) < 6 / 12 / math.sqrt(n)
    assert abs(((a[1:] - 0.5) * (a[:-1] - 0.5)).mean()) < 6 / 12 / math.sqrt(n)


def test_layer_norm_definition_against_autograd():
    g = torch.Generator().manual_seed(1)
    x, dy = (torch.randn(5, 13, generator=g, dtype=torch.float64) for _ in range(2))
    w = torch.randn(13, 2, generator=g, dtype=torch.float64)
    xs, ws = x.clone().requires_grad_(), w.clone().requires_grad_()
    y = torch.nn.functional.layer_norm(xs, (13,), ws[:, 0], ws[:, 1], 1e-5)
    y.backward(dy)
    val, _ = seq_ref.layer_norm(x, w, 1e-5, dy)
    for a, b in ((val["y"], y.detach()), (val["dx"], xs.grad), (val["dw"], ws.grad)):
        assert torch.allclose(a, b, rtol=1e-12, atol=1e-12)


@pytest.mark.parametrize("causal", [False, True])
def test_attention_definition_against_differences(causal):
    lens_q, lens_k, hq, hk, d, scale = [3, 4, 0, 2], [5, 2, 3, 2], 4, 2, 3, 0.6
    g = torch.Generator().manual_seed(2)
    mats = [torch.randn(sum(n), h * d, generator=g, dtype=torch.float64) for n, h in ((lens_q, hq), (lens_k, hk), (lens_k, hk))]
    do = torch.randn(sum(lens_q), hq * d, generator=g, dtype=torch.float64)

    def loss(q, k, v):
        return float((seq_ref.attention(q, k, v, lens_q, lens_k, hq, hk, d, scale, causal, torch.float32)[0]["out"] * do).sum())

    val, _ = seq_ref.attention(*mats, lens_q, lens_k, hq, hk, d, scale, causal, torch.float32, do)
    if causal:  # 4 queries over 2 keys: the first two see nothing
        assert not val["out"][3:5].any() and torch.isinf(val["lse"][3:5]).all() and not val["dq"][3:5].any()
    for i, name in enumerate(("dq", "dk", "dv")):
        for at in range(0, mats[i].numel(), 7):
            step = [m.clone() for m in mats]
            ends = []
            for sign in (1, -1):
                step[i].view(-1)[at] = mats[i].view(-1)[at] + sign * 1e-5
                ends.append(loss(*step))
            # central differences: third derivatives of order 1 times h^2, rounding 2^-52 / h
            assert abs((ends[0] - ends[1]) / 2e-5 - float(val[name].view(-1)[at])) < 1e-8
