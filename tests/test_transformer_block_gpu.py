"""Layer norm, attention, dropout and the residual connection as one transformer block uses them, forward and backward,
on images of different sizes packed one behind the other, against float64 autograd with the same dropout mask; and the whole
step captured into a graph, where a number in device memory gives every replay its own mask.

Between the operators stand plain matrix products.  They run in fp32 on float copies here, so that what is compared are the
operators: in fp32 every one of the about 20 steps of the chain is off by some 32 U of its own norm at most, 32 * 20 * U = 4e-5; in
bf16 a step rounds to half a step of 2^-8 at most, and 6 (output) or 14 (gradients) steps lie one behind the other."""
import ctypes
import math

import pytest
import torch

import seq_ref
from gpu_util import DEV, empty
from unet_amd import capi

pytestmark = pytest.mark.gpu
LENS, C, HEADS, KV, P, SEED = [64, 1, 144, 100], 96, 6, 3, 0.2, 77
D = C // HEADS


def stream():
    return torch.cuda.current_stream().cuda_stream


class Block:
    def __init__(self, dtype):
        self.dtype, self.tag = dtype, "bf16" if dtype == torch.bfloat16 else "f32"
        g = torch.Generator().manual_seed(4)
        self.t = sum(LENS)
        rand = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
        self.x, self.dy = rand(self.t, C).to(dtype).to(DEV), rand(self.t, C).to(dtype).to(DEV)
        self.w_ln = (rand(C, 2) * 0.2 + torch.tensor([1.0, 0.0])).to(DEV)
        self.w_qkv = (rand(C, C + 2 * KV * D) / math.sqrt(C)).to(dtype).to(DEV)
        self.w_out = (rand(C, C) / math.sqrt(C)).to(dtype).to(DEV)
        self.cu = torch.tensor([0] + LENS, dtype=torch.int32).cumsum(0).to(torch.int32).to(DEV)
        self.step = torch.tensor([3], dtype=torch.int64, device=DEV)  # added to the dropout's offset
        new = lambda *s: empty(s, dtype)  # noqa: E731
        self.norm, self.stats, self.att, self.lse = new(self.t, C), empty((self.t, 2)), new(self.t, C), empty((self.t, HEADS))
        self.y, self.dproj, self.dx = new(self.t, C), new(self.t, C), new(self.t, C)
        self.dqkv, self.dw_ln = new(self.t, C + 2 * KV * D), empty((C, 2))
        shape = (len(LENS), self.t, self.t, HEADS, KV, D)
        sizes = []
        for f, args in ((capi.unet_dot_attention_workspace_bytes, shape), (capi.unet_dot_attention_backward_workspace_bytes, shape),
                        (capi.unet_layer_norm_backward_workspace_bytes, (self.t, C))):
            n = ctypes.c_size_t()
            f(*args, ctypes.byref(n))
            sizes.append(n.value)
        self.ws = torch.empty(max(sizes) + 1, dtype=torch.uint8, device=DEV)  # one after the other on one stream: one workspace
        self.tail = (self.cu.data_ptr(), self.cu.data_ptr(), *shape, 1 / math.sqrt(D), 0, self.ws.data_ptr(), self.ws.numel())
        self.qkv = self.proj = self.dw_qkv = self.dw_out = None

    def op(self, name):
        return getattr(capi, f"unet_{name}_{self.tag}")

    def product(self, a, b):
        return (a.float() @ b.float()).to(self.dtype)

    def cut(self, m):
        return [m[:, :C], m[:, C:C + KV * D], m[:, C + KV * D:]]

    def run(self):
        s, x = stream(), self.x
        self.op("layer_norm")(x.data_ptr(), C, self.norm.data_ptr(), C, self.w_ln.data_ptr(), self.stats.data_ptr(), self.t, C, 1e-5, s)
        self.qkv = self.product(self.norm, self.w_qkv)
        pairs = lambda *ts: [v for t in ts for v in (t.data_ptr(), t.stride(0))]  # noqa: E731
        self.op("dot_attention")(*pairs(*self.cut(self.qkv), self.att), self.lse.data_ptr(), *self.tail, s)
        self.proj = self.product(self.att, self.w_out)
        self.op("dropout")(self.proj.data_ptr(), C, x.data_ptr(), C, self.y.data_ptr(), C, self.t, C, P, SEED, 10, self.step.data_ptr(), s)
        # backward
        self.op("dropout_backward")(self.dy.data_ptr(), C, self.dproj.data_ptr(), C, self.t, C, P, SEED, 10, self.step.data_ptr(), s)
        self.dw_out = self.att.float().t() @ self.dproj.float()
        datt = self.product(self.dproj, self.w_out.t())
        self.op("dot_attention_backward")(*pairs(datt, *self.cut(self.qkv), self.att), self.lse.data_ptr(), *pairs(*self.cut(self.dqkv)), *self.tail, s)
        self.dw_qkv = self.norm.float().t() @ self.dqkv.float()
        dnorm = self.product(self.dqkv, self.w_qkv.t())
        self.op("layer_norm_backward")(dnorm.data_ptr(), C, x.data_ptr(), C, self.stats.data_ptr(), self.w_ln.data_ptr(), self.dy.data_ptr(), C,
                                       self.dx.data_ptr(), C, self.dw_ln.data_ptr(), self.t, C, self.ws.data_ptr(), self.ws.numel(), s)

    def results(self):
        return {"y": self.y, "dx": self.dx, "dw_ln": self.dw_ln, "dw_qkv": self.dw_qkv, "dw_out": self.dw_out}

    def reference(self, offset):
        leaf = lambda t: t.double().cpu().requires_grad_()  # noqa: E731
        x, w_ln, w_qkv, w_out = leaf(self.x), leaf(self.w_ln), leaf(self.w_qkv), leaf(self.w_out)
        norm = torch.nn.functional.layer_norm(x, (C,), w_ln[:, 0], w_ln[:, 1], 1e-5)
        q, k, v = self.cut(norm @ w_qkv)
        parts, at = [], 0
        for n in LENS:
            rows = slice(at, at + n)
            at += n
            heads = []
            for h in range(HEADS):
                kv = slice(h // (HEADS // KV) * D, (h // (HEADS // KV) + 1) * D)
                s = q[rows, h * D:(h + 1) * D] @ k[rows, kv].T / math.sqrt(D)
                heads.append(torch.softmax(s, 1) @ v[rows, kv])
            parts.append(torch.cat(heads, 1))
        kept = seq_ref.dropout_kept(self.t, C, P, SEED, offset).double()
        y = x + torch.cat(parts) @ w_out * kept / (1 - P)
        y.backward(self.dy.double().cpu())
        return {"y": y.detach(), "dx": x.grad, "dw_ln": w_ln.grad, "dw_qkv": w_qkv.grad, "dw_out": w_out.grad}


def compare(got, want, dtype):
    for name, ref in want.items():
        bound = 32 * 20 * seq_ref.U if dtype == torch.float32 else (6 if name == "y" else 14) * 2.0 ** -8
        err = float((got[name].double().cpu() - ref).norm() / ref.norm())
        assert err <= bound, (name, err, bound)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_block_forward_and_backward(dtype):
    b = Block(dtype)
    b.run()
    compare(b.results(), b.reference(13), dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_block_captured_with_a_new_mask_per_replay(dtype):
    b = Block(dtype)
    b.run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.run()
        b.step.add_(1)
    for i in range(3):
        for t in (b.y, b.dx, b.dw_ln):
            t.fill_(0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        compare(b.results(), b.reference(13 + i), dtype)
        e = Block(dtype)
        e.step.fill_(3 + i)
        e.run()
        torch.cuda.synchronize()
        for name, t in e.results().items():
            if name in ("y", "dx", "dw_ln"):
                assert torch.equal(t, b.results()[name]), name
