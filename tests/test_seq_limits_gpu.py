"""Dot-product attention and layer norm at the ends of what their header allows: workspaces of other sizes than the call's own,
infinities that a query sees, the largest numbers, sums of a few and of very many terms.  Definitions and bounds: seq_ref.py."""
import ctypes

import pytest
import torch

import seq_ref
from gpu_util import DEV
from test_dot_attention_gpu import Call
from unet_amd import capi

pytestmark = pytest.mark.gpu


# ---- workspaces -----------------------------------------------------------------------------------------

def poisoned(f, *shape):
    """A workspace of the size that f names for the shape, 4 KB behind it, all bytes 255."""
    n = ctypes.c_size_t()
    f(*shape, ctypes.byref(n))
    whole = torch.full((n.value + 4096,), 255, dtype=torch.uint8, device=DEV)
    return whole[:n.value], whole[n.value:]


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lens_q,lens_k,hq,hk,d", [([1024], [1024], 8, 8, 64), ([300, 211], [300, 211], 4, 1, 100), ([1, 1], [5000, 3000], 8, 1, 128),
                                                   ([700], [700], 2, 1, 128), ([3] * 40, [9] * 40, 2, 2, 16), ([257], [4000], 1, 1, 40)])
def test_a_workspace_for_a_larger_call(name, causal, lens_q, lens_k, hq, hk, d):
    c = Call(name, lens_q, lens_k, hq, hk, d, causal, behind=2)
    large = (70, 60000, 600000, hq, hk, d)
    c.ws, behind = poisoned(capi.unet_dot_attention_workspace_bytes, *large)
    c.wsb, behind_b = poisoned(capi.unet_dot_attention_backward_workspace_bytes, *large)
    c.forward()
    c.backward()
    c.verify()
    assert (behind == 255).all() and (behind_b == 255).all()


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("lens_q,lens_k,hq,hk,d", [([1024], [1024], 8, 8, 64), ([1, 1], [5000, 3000], 8, 1, 128), ([700], [700], 2, 1, 128)])
def test_nothing_is_written_behind_a_workspace(name, lens_q, lens_k, hq, hk, d):
    c = Call(name, lens_q, lens_k, hq, hk, d, True)
    c.ws, behind = poisoned(capi.unet_dot_attention_workspace_bytes, *c.shape)
    c.wsb, behind_b = poisoned(capi.unet_dot_attention_backward_workspace_bytes, *c.shape)
    c.forward()
    c.backward()
    c.verify()
    assert (behind == 255).all() and (behind_b == 255).all()


# ---- the largest numbers --------------------------------------------------------------------------------

@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("lens_q,lens_k,hq,hk,d,pad", [([70, 9], [90, 9], 4, 2, 64, 0), ([300], [513], 66, 66, 100, 1), ([3, 1], [5000, 1], 8, 1, 128, 0),
                                                       ([130], [1500], 2, 1, 40, 0)])
def test_values_near_the_largest_number(name, lens_q, lens_k, hq, hk, d, pad):
    """A weighted mean is never larger than its terms, so the result is finite; the gradients of small dout are, too."""
    c = Call(name, lens_q, lens_k, hq, hk, d, True, pad)
    c.v *= 0.98 * torch.finfo(c.dtype).max / float(c.v.abs().max())  # half a step of bf16 on top: 0.984
    c.v[::3] = 0.98 * torch.finfo(c.dtype).max
    c.dout *= 2.0 ** -100
    c.forward()
    c.backward()
    c.verify()


# ---- infinities that a query sees -----------------------------------------------------------------------
# Both types treat them as the definition does: a score of -inf is a weight of 0, an infinite value makes an infinite output.

VISIBLE = [(4, 20), (60, 30), (130, 32), (4, 60), (60, 64), (80, 50), (130, 50), (4, 96), (66, 88), (4, 128), (66, 120)]  # heads, dim: each kernel of fp32
LENS_Q, LENS_K = [333, 40], [340, 33]


def visible(name, heads, dim, causal, pad):
    return Call(name, LENS_Q, LENS_K, heads, heads // 2, dim, causal, pad=pad, behind=1)


def seeing(c, key):
    """The queries that see a key (a truth value each), both numbered over all sequences."""
    s = 0 if key < c.lens_k[0] else 1
    query = torch.arange(c.nq)
    mine = (query >= c.lens_q[0]) == bool(s)
    at, nq, nk = (query - s * c.lens_q[0], c.lens_q[s], c.lens_k[s])
    return mine & (at + nk - nq >= key - s * c.lens_k[0]) if c.causal else mine


def check(c, val, bnd, names):
    for n in names:
        seq_ref.check(getattr(c, n)[:val[n].shape[0]], val[n], bnd[n], n)


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("causal,pad", [(False, 0), (True, 3)])
@pytest.mark.parametrize("heads,dim", VISIBLE)
def test_keys_with_infinite_scores(name, causal, pad, heads, dim):
    """Element 3 of the queries is positive and of some keys -inf: those keys have weight 0 with every query, so only grad_q's
    element 3, a product of 0 and the infinity, is NaN.  The definition has -1e30 in their place: weight 0 as well."""
    c = visible(name, heads, dim, causal, pad)
    bad = [7, 50, 51, 200, 345]
    c.q[:, 3::dim] = c.q[:, 3::dim].abs() + 0.125
    for key in bad:
        c.k[key, 3::dim] = -1e30
    val, bnd = c.exact()
    for key in bad:
        c.k[key, 3::dim] = -float("inf")
        val["dq"][seeing(c, key), 3::dim] = float("nan")
    c.forward()
    c.backward()
    check(c, val, bnd, ("out", "lse", "dq", "dk", "dv"))


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("causal,pad", [(False, 0), (True, 3)])
@pytest.mark.parametrize("heads,dim", VISIBLE)
def test_infinite_values_and_gradients(name, causal, pad, heads, dim):
    """An infinite element of V makes that element of the outputs infinite, one of grad_out that element of grad_v."""
    c = visible(name, heads, dim, causal, pad)
    clean, bnd = c.exact()
    val = {n: t.clone() for n, t in clean.items()}
    for key, e, inf in ((40, 1, float("inf")), (339, 1, float("inf")), (372, 4, float("inf")), (3, 5, -float("inf"))):
        c.v[key, e::dim] = inf
        val["out"][seeing(c, key), e::dim] = inf
    c.forward()
    check(c, val, bnd, ("out", "lse"))
    c = visible(name, heads, dim, causal, pad)
    val = {n: t.clone() for n, t in clean.items()}
    for query in (0, 331, 372):
        c.dout[query, 2::dim] = float("inf")
        val["dv"][torch.stack([seeing(c, key)[query] for key in range(c.nk)]), 2::dim] = float("inf")
    c.forward()
    c.backward()
    check(c, val, bnd, ("out", "lse", "dv"))


@pytest.mark.parametrize("heads,dim", VISIBLE)
def test_nan_whose_upper_half_is_an_infinity(heads, dim):
    c = visible("f32", heads, dim, True, 0)
    val, bnd = c.exact()
    for t, key in ((c.k, 60), (c.v, 345)):
        t[key] = torch.full_like(t[key], 0).view(torch.int32).fill_(0x7F800001).view(torch.float32)
        val["out"][seeing(c, key)] = float("nan")
    val["lse"][seeing(c, 60)] = float("nan")
    c.forward()
    assert (c.k[60].view(torch.int32) == 0x7F800001).all()
    check(c, val, bnd, ("out", "lse"))


@pytest.mark.parametrize("heads,dim", VISIBLE)
def test_scores_beyond_the_largest_number(heads, dim):
    """Products of -1e50 and more in one element: -inf in fp32, so weight 0, whatever their parts are."""
    c = visible("f32", heads, dim, True, 0)
    g = torch.Generator().manual_seed(1)
    c.q[:, 3::dim] = (torch.rand(c.tq, heads, generator=g) * 1e25 + 1e25).to(DEV)
    c.k[:, 3::dim] = 0.0
    c.k[[5, 100, 250], 3::dim] = -(torch.rand(3, c.hk, generator=g) * 1e25 + 1e25).to(DEV)
    c.forward()
    c.backward()
    c.verify()


@pytest.mark.parametrize("name", ["f32", "bf16"])
def test_infinities_in_split_sums(name):
    c = Call(name, [2, 1], [4000, 3500], 8, 2, 64, False)
    c.q[:, 3::64] = c.q[:, 3::64].abs() + 0.125
    bad = [0, 1, 3100, 5000]
    c.k[bad, 3::64] = -1e30
    val, bnd = c.exact()
    c.k[bad, 3::64] = -float("inf")
    c.v[[10, 6000], 1::64] = float("inf")
    val["out"][:, 1::64] = float("inf")
    c.forward()
    check(c, val, bnd, ("out", "lse"))


# ---- a few keys -----------------------------------------------------------------------------------------

def grad_q_of_few_keys(c, most):
    """grad_q in 64 bits and its bound for queries that see 1 to `most` keys, heads of up to 64 elements, bf16: what dS is made of
    is fp32, delta included (a sum over the weights: not dout * out, whose out was rounded to bf16), and dS goes into its
    product in two bf16 parts, off by half a step of the second, 2^-8 * 2^-8."""
    U, d, g = seq_ref.U, c.d, c.hq // c.hk
    q, k, v, do = (t.double().cpu().reshape(t.shape[0], -1, d) for t in (c.q, c.k, c.v, c.dout))
    val, bnd, rows = torch.zeros(c.nq, c.hq, d).double(), torch.zeros(c.nq, c.hq, d).double(), torch.zeros(c.nq, dtype=torch.bool)
    bq = bk = 0
    for nq, nk in zip(c.lens_q, c.lens_k):
        for i in range(nq):
            n = min(nk, i + 1 + nk - nq) if c.causal else nk
            if not 1 <= n <= most:
                continue
            rows[bq + i] = True
            for h in range(c.hq):
                qi, kj, vj, doi = q[bq + i, h], k[bk:bk + n, h // g], v[bk:bk + n, h // g], do[bq + i, h]
                s = kj @ qi * c.scale
                lse = torch.logsumexp(s, 0)
                p, dp = torch.exp(s - lse), vj @ doi
                ds = p * (dp - p @ dp)
                # as in seq_ref.attention: a score's roundings, the exponent's, those of the sum behind lse
                e_w = (d / 16 + 8) * U * c.scale * (kj.abs() @ qi.abs()) + 8 * U * (s.abs() + lse.abs() + 12)
                e_p = e_w + p @ e_w + 65 * U + 8 * U * lse.abs()
                e_dp = (d / 16 + 8) * U * (vj.abs() @ doi.abs())
                e_delta = p @ (e_dp + dp.abs() * (e_p + 40 * U))
                e_ds = p * (e_dp + e_delta) + ds.abs() * (e_p + 2.0 ** -16 + 4 * U)
                val[bq + i, h] = ds @ kj * c.scale
                bnd[bq + i, h] = c.scale * ((e_ds + 65 * U * ds.abs()) @ kj.abs()) + (seq_ref.half_step(c.dtype) + U) * val[bq + i, h].abs()
        bq, bk = bq + nq, bk + nk
    return val.reshape(c.nq, -1)[rows], bnd.reshape(c.nq, -1)[rows] + 1e-34, rows


@pytest.mark.parametrize("dim", [20, 32, 64])
@pytest.mark.parametrize("lens_q,lens_k,hq,hk,causal", [([50, 7], [32, 32], 6, 2, False), ([50, 7], [31, 1], 6, 2, False), ([40], [40], 32, 1, True),
                                                        ([40, 33], [40, 60], 3, 3, True)])
def test_grad_q_of_queries_that_see_up_to_32_keys(lens_q, lens_k, hq, hk, causal, dim):
    """Keys with a large part in common: dS adds up to zero, so that part falls out of grad_q, but an error of delta does not."""
    c = Call("bf16", lens_q, lens_k, hq, hk, dim, causal, spread=0.25)
    c.k += 4.0
    c.forward()
    c.backward()
    val, bnd, rows = grad_q_of_few_keys(c, 32)
    assert rows.any()
    seq_ref.check(c.dq[:c.nq][rows.to(DEV)], val, bnd, "dq")


# ---- each way to share the queries of fp32's 33 to 64 elements -------------------------------------------

@pytest.mark.parametrize("lens,hq,hk,dim,causal", [([128] * 12, 12, 12, 64, False), ([384] * 7, 8, 8, 48, True), ([300, 20], 60, 60, 40, False),
                                                   ([700], 32, 32, 64, True), ([65] * 9, 30, 30, 33, True)])
def test_fp32_of_up_to_64_elements(lens, hq, hk, dim, causal):
    c = Call("f32", lens, lens, hq, hk, dim, causal, behind=2)
    c.forward()
    c.backward()
    c.verify()
