"""unet_dot_attention_* and unet_dot_attention_backward_* against the float64 definition (seq_ref.py, which derives the bounds)."""
import ctypes
import math

import pytest
import torch

import seq_ref
from gpu_util import DEV, empty
from unet_amd import capi

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
FWD = {"f32": capi.unet_dot_attention_f32, "bf16": capi.unet_dot_attention_bf16}
BWD = {"f32": capi.unet_dot_attention_backward_f32, "bf16": capi.unet_dot_attention_backward_bf16}


def stream():
    return torch.cuda.current_stream().cuda_stream


def starts(lens, first=0):
    return torch.tensor([first] + list(lens), dtype=torch.int32).cumsum(0).to(torch.int32).to(DEV)


def workspace(f, *shape):
    n = ctypes.c_size_t()
    f(*shape, ctypes.byref(n))
    return torch.full((max(n.value, 1),), 255, dtype=torch.uint8, device=DEV)


class Call:
    """Packed inputs of a case with `behind` unused rows behind the last sequence, in buffers wider than the heads by `pad`
    columns (odd: misaligned), outputs inside buffers filled with 7."""

    def __init__(self, name, lens_q, lens_k, hq, hk, d, causal, pad=0, behind=0, seed=0, scale=None, spread=1.0):
        self.name, self.dtype, self.causal, self.d, self.hq, self.hk = name, TYPES[name], causal, d, hq, hk
        self.lens_q, self.lens_k, self.scale = lens_q, lens_k, scale or 1 / math.sqrt(d)
        self.nq, self.nk = sum(lens_q), sum(lens_k)
        self.tq, self.tk = self.nq + behind, self.nk + behind
        self.pad = pad
        g = torch.Generator().manual_seed(seed + 1)

        def rand(rows, cols, by=1.0):
            wide = (torch.randn(rows, cols + 2 * pad, generator=g) * by).to(self.dtype).to(DEV)
            return wide[:, pad:pad + cols]

        self.q, self.k, self.v = rand(self.tq, hq * d, spread), rand(self.tk, hk * d), rand(self.tk, hk * d)
        self.dout = rand(self.tq, hq * d)
        self.cu_q, self.cu_k = starts(lens_q), starts(lens_k)
        self.shape = (len(lens_q), self.tq, self.tk, hq, hk, d)
        self.ws = workspace(capi.unet_dot_attention_workspace_bytes, *self.shape)
        self.wsb = workspace(capi.unet_dot_attention_backward_workspace_bytes, *self.shape)
        self.out, self.lse = self.fresh(self.tq, hq), torch.full((self.tq, hq), 7.0, device=DEV)
        self.dq, self.dk, self.dv = self.fresh(self.tq, hq), self.fresh(self.tk, hk), self.fresh(self.tk, hk)

    def fresh(self, rows, heads):
        wide = torch.full((rows, heads * self.d + 2 * self.pad), 7.0, dtype=self.dtype, device=DEV)
        return wide[:, self.pad:self.pad + heads * self.d]

    def tail(self, ws):
        return (self.cu_q.data_ptr(), self.cu_k.data_ptr(), *self.shape, self.scale, int(self.causal), ws.data_ptr(), ws.numel(), stream())

    def pairs(self, *tensors):
        return [x for t in tensors for x in (t.data_ptr(), t.stride(0))]

    def forward(self, lse=True):
        FWD[self.name](*self.pairs(self.q, self.k, self.v, self.out), self.lse.data_ptr() if lse else None, *self.tail(self.ws))

    def backward(self):
        BWD[self.name](*self.pairs(self.dout, self.q, self.k, self.v, self.out), self.lse.data_ptr(),
                       *self.pairs(self.dq, self.dk, self.dv), *self.tail(self.wsb))

    def exact(self):
        n, m = self.nq, self.nk
        return seq_ref.attention(self.q[:n], self.k[:m], self.v[:m], self.lens_q, self.lens_k, self.hq, self.hk, self.d, self.scale, self.causal,
                                 self.dtype, self.dout[:n])

    def verify(self, names=("out", "lse", "dq", "dk", "dv")):
        val, bnd = self.exact()
        for what in names:
            t = getattr(self, what)
            n = self.nk if what in ("dk", "dv") else self.nq
            seq_ref.check(t[:n], val[what], bnd[what], what)
            assert (t[n:] == 7).all(), f"{what}: rows behind the last sequence were written"
            if self.pad and what != "lse":
                wide = t.as_strided((t.shape[0], t.stride(0)), (t.stride(0), 1), t.storage_offset() - self.pad)
                assert (wide[:, :self.pad] == 7).all() and (wide[:, -self.pad:] == 7).all(), f"{what}: columns beside it were written"


SHAPES = [  # lens_q, lens_k, heads, kv heads, head dim
    ([1], [1], 1, 1, 1),
    ([5, 0, 33], [5, 0, 33], 2, 1, 8),
    ([64, 1, 130], [64, 1, 130], 4, 2, 64),
    ([31, 32, 65, 127, 129], [31, 32, 65, 127, 129], 2, 2, 32),
    ([7, 200, 3], [100, 64, 0], 6, 2, 40),        # fewer keys than queries: rows that see nothing; no keys at all
    ([0, 3, 0], [5, 300, 1], 3, 3, 128),          # keys that no query sees
    ([257], [257], 8, 1, 80),
    ([300], [513], 5, 5, 33),
    ([20, 129], [20, 190], 14, 2, 100),           # groups of 7, a head dimension of 16-byte pieces and a half
    ([150], [700], 4, 4, 128),
    ([1, 1, 1], [2000, 1, 777], 16, 2, 64),       # single queries
    ([3, 9], [1500, 100], 12, 4, 96),
    ([2] * 70, [3] * 70, 2, 1, 16),               # many short sequences
]


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("pad,behind", [(0, 0), (1, 5), (8, 3)])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, [max(s[0]), max(s[1]), *s[2:]])))
def test_against_the_definition(name, causal, pad, behind, shape):
    c = Call(name, *shape, causal, pad, behind)
    c.forward()
    c.backward()
    c.verify()
    first = [t.clone() for t in (c.out, c.lse, c.dq, c.dk, c.dv)]
    c.forward(lse=False)
    c.backward()
    for a, b in zip(first, (c.out, c.lse, c.dq, c.dk, c.dv)):
        assert torch.equal(a, b)  # equal calls, equal bits


# long key sequences and few queries: the keys are split over workgroups and joined; and row counts for which the
# gradient of the keys is summed in parts
SPLIT = [([1, 1], [2500, 4100], 8, 1, 128), ([3, 0, 1], [5000, 600, 10], 6, 2, 40), ([5], [1999], 2, 2, 64), ([700, 1, 1300], [700, 1, 1300], 4, 1, 64),
         ([1100], [1500], 2, 1, 104), ([40], [20], 32, 1, 16), ([2, 300], [9000, 3], 3, 3, 32)]


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("shape", SPLIT, ids=lambda s: "x".join(map(str, [max(s[0]), max(s[1]), *s[2:]])))
@pytest.mark.parametrize("pad", [0, 1])
def test_split_sums(name, causal, shape, pad):
    c = Call(name, *shape, causal, pad=pad, behind=3)
    c.forward()
    c.backward()
    c.verify()
    first = [t.clone() for t in (c.out, c.lse, c.dq, c.dk, c.dv)]
    c.forward()
    c.backward()
    for a, b in zip(first, (c.out, c.lse, c.dq, c.dk, c.dv)):
        assert torch.equal(a, b)


# few heads and one or two sequences: dQ is summed in parts, and the workspace holds them where dK's and dV's need less
FEW = [([700], [700], 2, 1, 128), ([600, 9], [1300, 40], 1, 1, 100), ([900], [2100], 2, 2, 40), ([300], [2500], 4, 2, 20), ([65, 0, 1], [800, 300, 700], 1, 1, 96)]


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("pad", [0, 1])
@pytest.mark.parametrize("shape", FEW, ids=lambda s: "x".join(map(str, [max(s[0]), max(s[1]), *s[2:]])))
def test_few_heads(name, causal, pad, shape):
    c = Call(name, *shape, causal, pad=pad, behind=4)
    c.forward()
    c.backward()
    c.verify()
    first = [t.clone() for t in (c.out, c.lse, c.dq, c.dk, c.dv)]
    c.wsb.fill_(255)
    c.forward()
    c.backward()
    for a, b in zip(first, (c.out, c.lse, c.dq, c.dk, c.dv)):
        assert torch.equal(a, b)


def test_thousands_of_sequences():
    """More sequences than 64 x 64: found in three looks.  Empty ones among them."""
    g = torch.Generator().manual_seed(9)
    lens_q, lens_k = (torch.randint(0, 3, (4500,), generator=g).tolist() for _ in range(2))
    c = Call("bf16", lens_q, lens_k, 2, 1, 16, True, behind=3)
    c.forward()
    c.backward()
    c.verify()


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dim", [96, 128])
def test_many_queries(causal, dim):
    """Enough queries for the widest workgroups; a sequence that ends inside one, and queries that see nothing."""
    c = Call("bf16", [300, 700], [290, 701], 106, 53, dim, causal, behind=2)
    c.forward()
    c.backward()
    c.verify()


# one call for each way to share the queries of a head dimension's kernels: 32, 64 and 128 of them in a workgroup
SHARES = [(4, 20), (4, 60), (4, 96), (4, 128), (60, 30), (60, 64), (30, 80), (30, 128), (130, 32), (130, 50), (66, 88), (66, 120)]


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("pad", [0, 3])
@pytest.mark.parametrize("heads,dim", SHARES)
def test_shares_of_the_queries(name, causal, pad, heads, dim):
    c = Call(name, [333, 40], [340, 33], heads, heads // 2, dim, causal, pad=pad, behind=1)
    c.forward()
    c.backward()
    c.verify()


@pytest.mark.parametrize("power", [-100, -60, 60, 100, 113])
def test_fp32_over_its_range(power):
    """Values near both ends of fp32's range and gradients near the other: the results are linear in both, so their bounds
    scale with them.  The products leave out at most 2 * 2^-7 * 2^-15 of each term, 8 U, which is less than the chains of
    the bounds have.  113: every value is as large as the header allows, largest / (256 * 90 keys), rounded down to
    largest / 2^15: the weights on the way are up to 2^8, and 2^8 * 90 < 2^15."""
    c = Call("f32", [70, 9], [90, 9], 4, 2, 64, True)
    if power == 113:
        top = torch.finfo(torch.float32).max * 2.0 ** -15
        c.v[:] = top * torch.where(torch.arange(c.v.shape[1], device=DEV) % 2 == 0, 1.0, -1.0)
    else:
        c.v *= 2.0 ** power
    c.dout *= 2.0 ** -power
    c.forward()
    c.backward()
    c.verify()


def test_fp32_largest_numbers():
    """The largest finite fp32 number as an element of every key, times the smallest normal one in the queries: a part of
    the score of about 4 that needs all bits of the key.  (dK has 2^-126 of dS in that column: not looked at.)"""
    c = Call("f32", [40], [75], 2, 1, 32, True)
    c.k[:, 0] = torch.finfo(torch.float32).max
    c.q[:, 0] = 2.0 ** -126
    c.q[:, 32] = -2.0 ** -126
    c.dout *= 2.0 ** -30
    c.forward()
    c.backward()
    c.verify(("out", "lse", "dq", "dv"))


@pytest.mark.parametrize("bad", [float("nan"), float("-inf")])
def test_split_sums_keep_bad_keys_to_the_queries_that_see_them(bad):
    c = Call("bf16", [2, 1], [4000, 3500], 4, 2, 64, True)
    val, bnd = c.exact()
    c.k[3999] = bad  # seen by the second query alone
    c.v[3999] = bad
    c.forward()
    for n in ("out", "lse"):
        seq_ref.check(getattr(c, n)[[0, 2]], val[n][[0, 2]], bnd[n][[0, 2]], n)
    assert not torch.isfinite(c.out[1].float()).any()


@pytest.mark.parametrize("name", ["f32", "bf16"])
def test_large_scores(name):
    """Scores of several hundred: the running maximum moves often, most weights underflow."""
    c = Call(name, [190], [190], 2, 1, 64, True, scale=1.0, spread=12.0)
    c.forward()
    c.backward()
    c.verify()


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("where", [0, 40, 95])
def test_what_a_query_does_not_see_does_not_reach_it(name, bad, where):
    """Against the definition without the bad row, not bit by bit: tiles that hold it are summed row by row, and another order of
    an fp32 sum is another rounding.  The bounds hold for any order with at most 64 + n / 32 additions in a row: 32 for each
    of the at most two tiles that a bad row can be hidden in, one per tile and product elsewhere."""
    lens = [96, 50]
    clean = Call(name, lens, lens, 4, 2, 48, True, behind=4)
    val, bnd = clean.exact()

    def same(c, what, rows):
        seq_ref.check(getattr(c, what)[rows], val[what][rows], bnd[what][rows], what)

    for what in ("k", "v"):
        c = Call(name, lens, lens, 4, 2, 48, True, behind=4)
        getattr(c, what)[where] = bad
        getattr(c, what)[146:] = bad  # rows of no sequence
        c.forward()
        c.backward()
        blind = [i for i in range(146) if i < where or i >= 96]  # queries that do not see the bad key
        for n in ("out", "lse", "dq"):
            same(c, n, blind)
        if what == "v":
            assert not torch.isfinite(c.out[where:96].float()).any()
        for n in ("dk", "dv"):
            same(c, n, list(range(96, 146)))
    for what in ("q", "dout"):
        c = Call(name, lens, lens, 4, 2, 48, True, behind=4)
        getattr(c, what)[where] = bad
        c.forward()
        c.backward()
        for n in ("out", "dq"):
            same(c, n, [i for i in range(146) if i != where])
        for n in ("dk", "dv"):
            same(c, n, [i for i in range(146) if i > where])  # keys that the bad query does not see
        if what == "dout":
            assert not torch.isfinite(c.dv[:where + 1].float()).any()


def test_gradient_against_differences():
    """Along random directions: loss(x + h d) - loss(x - h d) of the fp32 forward, the loss taken in float64.  (A bf16
    forward is too coarse for differences; its gradient is tested against the formula.)"""
    c = Call("f32", [60, 45], [60, 70], 4, 2, 32, True)
    c.forward()
    c.backward()
    dout = c.dout.double()
    for t, grad in ((c.q, c.dq), (c.k, c.dk), (c.v, c.dv)):
        g = torch.Generator().manual_seed(3)
        d = torch.randn(t.shape, generator=g).to(DEV)
        keep, h, ends = t.clone(), 2.0 ** -7, []
        for sign in (1, -1):
            t.copy_(keep + sign * h * d)
            c.forward()
            ends.append(float((c.out.double() * dout).sum()))
        t.copy_(keep)
        got, want = (ends[0] - ends[1]) / (2 * h), float((grad.double() * d.double()).sum())
        # third-order term h^2/6 f''' with f''' of the order of the sum of |grad d| (inputs of order 1), rounding of the outputs
        # U * 50 * sum |dout out| / h
        size = float((grad.double() * d.double()).abs().sum())
        noise = 50 * seq_ref.U * float((dout * c.out.double()).abs().sum()) / h
        assert abs(got - want) <= h * h * size + noise, (got, want, size, noise)


def test_garbage_bounds_stay_inside_the_tensors():
    """Sequence bounds beyond the tensors are clipped: nothing outside them is touched."""
    c = Call("bf16", [40, 30], [40, 30], 2, 1, 32, False, behind=6)
    c.cu_q.copy_(torch.tensor([-5, 40, 1 << 30], dtype=torch.int32))
    c.cu_k.copy_(torch.tensor([-9, 40, 1 << 30], dtype=torch.int32))
    c.forward()
    c.backward()
    torch.cuda.synchronize()
    full = Call("bf16", [40, 36], [40, 36], 2, 1, 32, False)
    full.q, full.k, full.v, full.dout = c.q, c.k, c.v, c.dout
    full.forward()
    full.backward()
    assert torch.equal(c.out, full.out) and torch.equal(c.dk, full.dk)


def test_tokens_beyond_32_bits_of_offset():
    """Keys and values 2^23 elements apart: 300 of them reach past 2^31 elements."""
    c = Call("bf16", [40], [300], 2, 1, 64, True)
    c.forward()
    want = c.out.clone()
    ld = 1 << 23
    buf = torch.zeros(300 * ld, dtype=torch.bfloat16, device=DEV).view(300, ld)
    k, v = buf[:, 64:128], buf[:, 4096:4160]
    k.copy_(c.k)
    v.copy_(c.v)
    c.k, c.v = k, v
    c.forward()
    assert torch.equal(c.out, want)
    c.backward()
    c.verify()


def test_first_sequence_need_not_start_at_the_first_row():
    c = Call("bf16", [30, 50], [30, 50], 2, 2, 64, True, behind=20)
    c.cu_q.add_(9)
    c.cu_k.add_(9)
    c.forward()
    assert (c.out[:9] == 7).all() and (c.out[89:] == 7).all()
    val, bnd = seq_ref.attention(c.q[9:89], c.k[9:89], c.v[9:89], [30, 50], [30, 50], 2, 2, 64, c.scale, True, c.dtype)
    seq_ref.check(c.out[9:89], val["out"], bnd["out"], "out")


@pytest.mark.parametrize("name,lens_q", [("bf16", [200, 56, 300]), ("f32", [200, 56, 300]), ("bf16", [1, 1, 2])])
def test_captured_and_replayed_beside_eager_work(name, lens_q):
    lens_k = [900, 56, 300]
    c = Call(name, lens_q, lens_k, 8, 2, 64, True)
    names = ("out", "lse", "dq", "dk", "dv")
    c.forward()
    c.backward()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.forward()
        c.backward()
    for i in range(4):
        e = Call(name, lens_q, lens_k, 8, 2, 64, True, seed=10 + i)
        c.q.copy_(e.q)
        c.k.copy_(e.k)
        c.v.copy_(e.v)
        c.dout.copy_(e.dout)
        e.forward()
        e.backward()
        for n in names:
            getattr(c, n).fill_(0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for n in names:
            assert torch.equal(getattr(c, n), getattr(e, n)), n


def test_two_streams_at_once():
    calls = [Call("bf16", [400, 333], [400, 333], 8, 4, 64, True, seed=i) for i in range(2)]
    want = []
    for c in calls:
        c.forward()
        c.backward()
        want.append([t.clone() for t in (c.out, c.dq, c.dk, c.dv)])
        for t in (c.out, c.dq, c.dk, c.dv):
            t.fill_(0)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    for _ in range(3):
        for c, s in zip(calls, streams):
            with torch.cuda.stream(s):
                c.forward()
                c.backward()
    torch.cuda.synchronize()
    for c, w in zip(calls, want):
        for a, b in zip((c.out, c.dq, c.dk, c.dv), w):
            assert torch.equal(a, b)
