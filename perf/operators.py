"""The transformer-block operators of the C ABI (layer norm, dropout, dot-product attention) as calls on
real sizes: `listed()` and `draw()` name them, `prepare()` makes their data, `run()` is one pass.

With `own` false `run` computes an operator in elementary torch operations in 32 bits, rounded once at the
end; with `own` true it makes the calls of include/unet_hip.h through unet_amd.capi.  `exact()` is the
operator's definition in 64 bits.
"""
import ctypes
import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
_EPS = 1e-5
_LOW32 = 0xFFFFFFFF


# ---------------------------------------------------------------------------------------------- cases --

def _ln(name, rows, channels, dtype, train, pad=0):
    return {"name": name, "op": "layer_norm", "rows": rows, "channels": channels, "dtype": dtype, "train": train, "pad": pad}


def _drop(name, rows, channels, dtype, p, direction, pad=0):
    return {"name": name, "op": "dropout", "rows": rows, "channels": channels, "dtype": dtype, "p": p,
            "direction": direction, "pad": pad}


def _attn(name, lens, q_lens, heads, kv_heads, dim, dtype, causal, train):
    return {"name": name, "op": "attention", "lens": " ".join(map(str, lens)),
            "q_lens": "" if q_lens is None else " ".join(map(str, q_lens)), "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "dtype": dtype, "causal": causal, "train": train}


def listed():
    return [
        # one 256x256 image at the network's bottleneck: 16x16 tokens of 1024 channels, inference
        _ln("ln_bf16_one_image", 256, 1024, "bf16", False),
        # a training batch of 16 images at 64x64 tokens: forward and backward
        _ln("ln_bf16_train", 65536, 1024, "bf16", True),
        # the fp32 route with a channel count that is no multiple of anything, rows inside a wider buffer
        _ln("ln_f32_odd_train", 16383, 321, "f32", True, pad=7),
        # one image: the residual branch behind the attention of one block
        _drop("dropout_bf16_one_image", 256, 1024, "bf16", 0.1, "residual"),
        # the residual branch of a training batch
        _drop("dropout_bf16_train", 65536, 1024, "bf16", 0.1, "residual"),
        # the gradient on the fp32 route, odd channel count, rows inside a wider buffer
        _drop("dropout_f32_odd_grad", 16383, 321, "f32", 0.25, "backward", pad=7),
        # one image at the bottleneck, every token sees every token, inference
        _attn("attn_bf16_one_image", [256], None, 8, 8, 64, "bf16", False, False),
        # a training batch of 16 images at the bottleneck
        _attn("attn_bf16_batch_train", [256] * 16, None, 16, 16, 64, "bf16", False, True),
        # one long sequence (a 1024x1024 image in 8x8 patches is 16384 tokens, half of it), causal, grouped heads
        _attn("attn_bf16_long_train", [8192], None, 16, 4, 128, "bf16", True, True),
        # images of different sizes packed without padding; a head dimension between two tile widths
        _attn("attn_bf16_ragged_train", [1, 1000, 77, 2049, 529, 0, 1600, 33], None, 8, 2, 80, "bf16", True, True),
        # the fp32 route
        _attn("attn_f32_train", [1024, 900, 1024, 577], None, 8, 8, 64, "f32", False, True),
        # single new queries over long key sequences
        _attn("attn_bf16_single_query", [16384, 12001, 9000, 16001], [1, 1, 1, 1], 32, 4, 128, "bf16", True, False),
    ]


def _spread(rng, low, high):
    """An integer whose logarithm is uniform."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["layer_norm", "dropout", "attention", "attention"])
    if op == "attention":
        dtype = rng.choice(["bf16", "bf16", "f32"])
        kv_heads = rng.choice([1, 2, 4, 8])
        heads = kv_heads * rng.choice([1, 1, 2, 3, 4, 8])
        dim = rng.choice([16, 24, 32, 40, 48, 64, 64, 72, 80, 96, 100, 128, 128])
        train = rng.random() < 0.6
        few = not train and rng.random() < 0.5
        count = rng.choice([1, 1, 2, 3, 5, 8])
        top = 16384 if few else 4096
        lens = [_spread(rng, 1, top) for _ in range(count)]
        lens[0] = _spread(rng, 64, top)
        q_lens = [min(n, _spread(rng, 1, 16)) for n in lens] if few else None
        budget = 2 ** 29 if dtype == "bf16" else 2 ** 28  # score elements of the padded batch
        while heads * count * max(lens) * max(q_lens or lens) > budget:
            lens = [max(1, n // 2) for n in lens]
            q_lens = [min(a, b) for a, b in zip(lens, q_lens)] if few else None
        return {k: v for k, v in _attn("", lens, q_lens, heads, kv_heads, dim, dtype, few or rng.random() < 0.6, train).items()
                if k != "name"}
    dtype = rng.choice(["bf16", "f32"])
    channels = rng.choice([32, 64, 77, 96, 128, 256, 321, 512, 640, 768, 1000, 1024, 2048])
    rows = _spread(rng, 1, (2 ** 25 if dtype == "bf16" else 2 ** 24) // channels)
    pad = rng.choice([0, 0, 1, 8, 64])
    if op == "layer_norm":
        case = _ln("", rows, channels, dtype, rng.random() < 0.6, pad)
    else:
        case = _drop("", rows, channels, dtype, rng.choice([0.05, 0.1, 0.2, 0.5]), rng.choice(["plain", "residual", "backward"]), pad)
    return {k: v for k, v in case.items() if k != "name"}


def _lengths(case):
    lens = [int(n) for n in case["lens"].split()]
    return lens, [int(n) for n in case["q_lens"].split()] if case["q_lens"] else list(lens)


def _pairs(case):
    """Visible (query, key) pairs, one query head."""
    k_lens, q_lens = _lengths(case)
    total = 0
    for nq, nk in zip(q_lens, k_lens):
        if not case["causal"]:
            total += nq * nk
        else:
            seen = [max(0, min(nk, i + 1 + nk - nq)) for i in (0, nq - 1)] if nq else [0, 0]
            empty = max(0, nq - nk)
            total += (max(seen[0], 1) + seen[1]) * (nq - empty) // 2 if nq > empty else 0
    return total


def work(case):
    size = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "layer_norm":
        n = case["rows"] * case["channels"]
        moved, per = (2, 8) if not case["train"] else (4, 24)  # x -> y; with dy -> dx
        return {"bytes": moved * n * size + 8 * case["rows"] + 4 * case["channels"] * (2 if not case["train"] else 6), "flops": per * n}
    if case["op"] == "dropout":
        n = case["rows"] * case["channels"]
        return {"bytes": (3 if case["direction"] == "residual" else 2) * n * size, "flops": 3 * n}
    k_lens, q_lens = _lengths(case)
    q = sum(q_lens) * case["heads"] * case["dim"] * size
    kv = 2 * sum(k_lens) * case["kv_heads"] * case["dim"] * size
    rows = 4 * sum(q_lens) * case["heads"]
    flops = 4 * case["dim"] * case["heads"] * _pairs(case)
    moved = 2 * q + kv + rows
    if case["train"]:
        moved += 2 * q + kv  # dout in; dq, dk, dv out
        flops = flops * 7 // 2
    return {"bytes": moved, "flops": flops}


# --------------------------------------------------------------------------------------------- inputs --

def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed * 7919 + 13)

    def normal(rows, columns, dtype, pad=0, scale=1.0, shift=0.0):
        wide = torch.randn(rows, columns + pad, generator=gen, device="cuda")
        return (wide * scale + shift).to(dtype)[:, :columns]

    dtype = _TYPES[case["dtype"]]
    st = {"case": case}
    if case["op"] == "layer_norm":
        rows, ch, pad = case["rows"], case["channels"], case["pad"]
        st["x"] = normal(rows, ch, dtype, pad, 1.5, 0.3)
        st["weights"] = torch.randn(ch, 2, generator=gen, device="cuda") * 0.2 + torch.tensor([1.0, 0.0], device="cuda")
        if case["train"]:
            st["dy"] = normal(rows, ch, dtype, pad)
        return st
    if case["op"] == "dropout":
        rows, ch, pad = case["rows"], case["channels"], case["pad"]
        st["x"] = normal(rows, ch, dtype, pad)
        if case["direction"] == "residual":
            st["residual"] = normal(rows, ch, dtype, pad)
        st["seed"] = (seed * 0x9E3779B97F4A7C15 + 1) & (2 ** 63 - 1)
        st["offset"] = 1000 + seed
        return st
    k_lens, q_lens = _lengths(case)
    hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
    tq, tk = sum(q_lens), sum(k_lens)
    if case["q_lens"]:  # queries of their own; keys and values side by side, as a cache of finished tokens holds them
        st["q"] = normal(tq, hq * d, dtype)
        kv = normal(tk, 2 * hk * d, dtype)
        st["k"], st["v"] = kv[:, :hk * d], kv[:, hk * d:]
    else:  # one projection makes the three
        qkv = normal(tq, (hq + 2 * hk) * d, dtype)
        st["q"], st["k"], st["v"] = qkv[:, :hq * d], qkv[:, hq * d:(hq + hk) * d], qkv[:, (hq + hk) * d:]
    if case["train"]:
        st["dout"] = normal(tq, hq * d, dtype)

    def starts(lens):
        return torch.tensor([0] + lens, dtype=torch.int64).cumsum(0).to(torch.int32).cuda()

    st["cu_q"], st["cu_k"] = starts(q_lens), starts(k_lens)
    st["max_q"], st["max_k"] = max(q_lens), max(k_lens)
    return st


# ---------------------------------------------------------------------------------------- plain forms --

def _plain_layer_norm(st):
    x, w = st["x"].float(), st["weights"]
    mean = x.mean(1, keepdim=True)
    centred = x - mean
    rstd = 1.0 / torch.sqrt((centred * centred).mean(1, keepdim=True) + _EPS)
    xhat = centred * rstd
    out = {"y": (xhat * w[:, 0] + w[:, 1]).to(st["x"].dtype)}
    if st["case"]["train"]:
        dy = st["dy"].float()
        g = dy * w[:, 0]
        dx = rstd * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
        out["dx"] = dx.to(st["x"].dtype)
        out["dweights"] = torch.stack([(dy * xhat).sum(0), dy.sum(0)], 1)
    return out


def _mul32(a, constant):
    """High and low words of the 64-bit product of 32-bit words held in int64."""
    product = a * constant  # wraps modulo 2^64
    return (product >> 32) & _LOW32, product & _LOW32


def _philox(blocks, flag, seed, offset):
    """Philox4x32-10 (Salmon, Moraes, Dror, Shaw 2011): 10 rounds on the counter (block, offset) under the key `seed`."""
    c0, c1 = blocks & _LOW32, (blocks >> 32) | (flag << 31)
    c2, c3 = torch.full_like(blocks, offset & _LOW32), torch.full_like(blocks, offset >> 32)
    k0, k1 = seed & _LOW32, seed >> 32

    def round_of(words, k0, k1):
        hi0, lo0 = _mul32(words[0], 0xD2511F53)
        hi1, lo1 = _mul32(words[2], 0xCD9E8D57)
        return hi1 ^ words[1] ^ k0, lo1, hi0 ^ words[3] ^ k1, lo0

    words = (c0, c1, c2, c3)
    for i in range(10):
        words = round_of(words, (k0 + i * 0x9E3779B9) & _LOW32, (k1 + i * 0xBB67AE85) & _LOW32)
    words = torch.stack(words, 1)
    return torch.stack([words & 0xFFFF, words >> 16], 2).reshape(-1, 8)


def _plain_dropout(st):
    x, case = st["x"], st["case"]
    n = x.shape[0] * x.shape[1]
    blocks = torch.arange((n + 7) // 8, device=x.device)
    number = (_philox(blocks, 0, st["seed"], st["offset"]) << 16) | _philox(blocks, 1, st["seed"], st["offset"])
    keep = (number.reshape(-1)[:n] >= round(case["p"] * 2 ** 32)).reshape(x.shape)
    out = torch.where(keep, x.float() * (1.0 / (1.0 - case["p"])), torch.zeros((), device=x.device))
    if case["direction"] == "residual":
        out = out + st["residual"].float()
    return {"out": out.to(x.dtype)}


def _padded(cu, most):
    """Token index of (sequence, position) and which of them exist."""
    position = torch.arange(most, device=cu.device)
    here = position < (cu[1:] - cu[:-1])[:, None]
    return torch.where(here, cu[:-1, None] + position, 0), here


def _plain_attention(st):
    case = st["case"]
    hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
    scale = 1.0 / math.sqrt(d)
    tok_q, here_q = _padded(st["cu_q"], st["max_q"])
    tok_k, here_k = _padded(st["cu_k"], st["max_k"])
    s, lq, lk, g = tok_q.shape[0], st["max_q"], st["max_k"], hq // hk

    def split(t, tokens, here, heads, copies):  # -> [sequence, head, position, dim], absent tokens 0
        t = torch.where(here[..., None], t.float()[tokens.reshape(-1)].reshape(*tokens.shape, heads * d), 0.0)
        t = t.reshape(*tokens.shape, heads, d).transpose(1, 2)
        return t.repeat_interleave(copies, 1) if copies > 1 else t.contiguous()

    q = split(st["q"], tok_q, here_q, hq, 1)
    k = split(st["k"], tok_k, here_k, hk, g)
    v = split(st["v"], tok_k, here_k, hk, g)
    seen = here_k[:, None, :].expand(s, lq, lk)
    if case["causal"]:
        ends = (st["cu_k"][1:] - st["cu_k"][:-1] - st["cu_q"][1:] + st["cu_q"][:-1])[:, None, None]
        seen = seen & (torch.arange(lk, device=q.device)[None, None] <= torch.arange(lq, device=q.device)[None, :, None] + ends)
    scores = torch.matmul(q, k.transpose(2, 3).contiguous()) * scale
    scores.masked_fill_(~seen[:, None], float("-inf"))
    top = scores.amax(3, keepdim=True)
    top = torch.where(torch.isinf(top) & (top < 0), torch.zeros_like(top), top)
    p = torch.exp_(scores - top)
    total = p.sum(3, keepdim=True)
    p = p / torch.where(total > 0, total, torch.ones_like(total))
    o = torch.matmul(p, v)

    def joined(t, tokens, here, count, heads):  # back to [token, head * dim]
        t = t.transpose(1, 2).reshape(*tokens.shape, heads * d)
        out = t.new_zeros(count, heads * d)
        return out.index_copy_(0, tokens[here], t[here])

    count_q, count_k = st["q"].shape[0], st["k"].shape[0]
    dtype = st["q"].dtype
    out = {"out": joined(o, tok_q, here_q, count_q, hq).to(dtype)}
    lse = (top + torch.log(total)).squeeze(3).transpose(1, 2)
    out["lse"] = lse.new_empty(count_q, hq).index_copy_(0, tok_q[here_q], lse[here_q])
    if not case["train"]:
        return out
    do = split(st["dout"], tok_q, here_q, hq, 1)

    def of_group(t):
        return t.reshape(s, hk, g, lk, d).sum(2)

    dv = of_group(torch.matmul(p.transpose(2, 3).contiguous(), do))
    dp = torch.matmul(do, v.transpose(2, 3).contiguous())
    ds = p * (dp - (do * o).sum(3, keepdim=True))
    dq = torch.matmul(ds, k) * scale
    dk = of_group(torch.matmul(ds.transpose(2, 3).contiguous(), q)) * scale
    out["dq"] = joined(dq, tok_q, here_q, count_q, hq).to(dtype)
    out["dk"] = joined(dk, tok_k, here_k, count_k, hk).to(dtype)
    out["dv"] = joined(dv, tok_k, here_k, count_k, hk).to(dtype)
    return out


# ------------------------------------------------------------------------------- the framework's calls --

def _own_layer_norm(st):
    from unet_amd import capi
    case, x, w = st["case"], st["x"], st["weights"]
    rows, ch = x.shape
    stream = torch.cuda.current_stream().cuda_stream
    if "y" not in st:  # the buffers that a program keeps from step to step
        st["y"] = torch.empty(rows, ch, dtype=x.dtype, device=x.device)
        st["stats"] = torch.empty(rows, 2, device=x.device)
        if case["train"]:
            st["dx"], st["dweights"] = torch.empty_like(st["y"]), torch.empty_like(w)
            need = ctypes.c_size_t()
            capi.unet_layer_norm_backward_workspace_bytes(rows, ch, ctypes.byref(need))
            st["work"] = torch.empty(max(need.value, 1), dtype=torch.uint8, device=x.device)
    forward, backward = ((capi.unet_layer_norm_bf16, capi.unet_layer_norm_backward_bf16) if case["dtype"] == "bf16" else
                         (capi.unet_layer_norm_f32, capi.unet_layer_norm_backward_f32))
    y, stats = st["y"], st["stats"]
    forward(x.data_ptr(), x.stride(0), y.data_ptr(), ch, w.data_ptr(), stats.data_ptr() if case["train"] else None, rows, ch,
            _EPS, stream)
    if not case["train"]:
        return {"y": y}
    dy, dx, dw, ws = st["dy"], st["dx"], st["dweights"], st["work"]
    backward(dy.data_ptr(), dy.stride(0), x.data_ptr(), x.stride(0), stats.data_ptr(), w.data_ptr(), None, 0, dx.data_ptr(), ch,
             dw.data_ptr(), rows, ch, ws.data_ptr(), ws.numel(), stream)
    return {"y": y, "dx": dx, "dweights": dw}


def _own_dropout(st):
    from unet_amd import capi
    case, x = st["case"], st["x"]
    rows, ch = x.shape
    stream = torch.cuda.current_stream().cuda_stream
    if "out" not in st:
        st["out"] = torch.empty(rows, ch, dtype=x.dtype, device=x.device)
    out, bf16 = st["out"], case["dtype"] == "bf16"
    if case["direction"] == "backward":
        call = capi.unet_dropout_backward_bf16 if bf16 else capi.unet_dropout_backward_f32
        call(x.data_ptr(), x.stride(0), out.data_ptr(), ch, rows, ch, case["p"], st["seed"], st["offset"], None, stream)
    else:
        call = capi.unet_dropout_bf16 if bf16 else capi.unet_dropout_f32
        res = st.get("residual")
        call(x.data_ptr(), x.stride(0), None if res is None else res.data_ptr(), 0 if res is None else res.stride(0),
             out.data_ptr(), ch, rows, ch, case["p"], st["seed"], st["offset"], None, stream)
    return {"out": out}


def _own_attention(st):
    from unet_amd import capi
    case, q, k, v = st["case"], st["q"], st["k"], st["v"]
    hq, hk, d, bf16 = case["heads"], case["kv_heads"], case["dim"], case["dtype"] == "bf16"
    tq, tk, seqs = q.shape[0], k.shape[0], st["cu_q"].numel() - 1
    stream = torch.cuda.current_stream().cuda_stream
    if "out" not in st:
        new = {"dtype": q.dtype, "device": q.device}
        st["out"], st["lse"] = torch.empty(tq, hq * d, **new), torch.empty(tq, hq, device=q.device)
        need, more = ctypes.c_size_t(), ctypes.c_size_t()
        capi.unet_dot_attention_workspace_bytes(seqs, tq, tk, hq, hk, d, ctypes.byref(need))
        if case["train"]:
            st["dq"], st["dk"], st["dv"] = (torch.empty(n, h * d, **new) for n, h in ((tq, hq), (tk, hk), (tk, hk)))
            capi.unet_dot_attention_backward_workspace_bytes(seqs, tq, tk, hq, hk, d, ctypes.byref(more))
        st["work"] = torch.empty(max(need.value, more.value, 1), dtype=torch.uint8, device=q.device)
    forward, backward = ((capi.unet_dot_attention_bf16, capi.unet_dot_attention_backward_bf16) if bf16 else
                         (capi.unet_dot_attention_f32, capi.unet_dot_attention_backward_f32))
    out, lse, ws = st["out"], st["lse"], st["work"]
    shape = (st["cu_q"].data_ptr(), st["cu_k"].data_ptr(), seqs, tq, tk, hq, hk, d, 1.0 / math.sqrt(d), int(case["causal"]),
             ws.data_ptr(), ws.numel(), stream)
    forward(q.data_ptr(), q.stride(0), k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0), out.data_ptr(), hq * d,
            lse.data_ptr(), *shape)
    if not case["train"]:
        return {"out": out, "lse": lse}
    do, dq, dk, dv = st["dout"], st["dq"], st["dk"], st["dv"]
    backward(do.data_ptr(), do.stride(0), q.data_ptr(), q.stride(0), k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0),
             out.data_ptr(), hq * d, lse.data_ptr(), dq.data_ptr(), hq * d, dk.data_ptr(), hk * d, dv.data_ptr(), hk * d, *shape)
    return {"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv}


def run(st):
    op = st["case"]["op"]
    if own:
        return {"layer_norm": _own_layer_norm, "dropout": _own_dropout, "attention": _own_attention}[op](st)
    return {"layer_norm": _plain_layer_norm, "dropout": _plain_dropout, "attention": _plain_attention}[op](st)


# ------------------------------------------------------------------------------------------ in 64 bits --

def _exact_layer_norm(st):
    x, gamma, beta = st["x"].double(), st["weights"][:, 0].double(), st["weights"][:, 1].double()
    var, mean = torch.var_mean(x, 1, unbiased=False, keepdim=True)
    deviation = torch.sqrt(var + _EPS)
    normal = (x - mean) / deviation
    out = {"y": normal * gamma + beta}
    if st["case"]["train"]:
        dy, c = st["dy"].double(), x.shape[1]
        up = dy * gamma
        along = (up * normal).sum(1, keepdim=True)
        out["dx"] = (c * up - up.sum(1, keepdim=True) - normal * along) / (c * deviation)
        out["dweights"] = torch.stack([torch.einsum("rc,rc->c", dy, normal), dy.sum(0)], 1)
    return out


def _random_words(block, flag, seed, offset):
    """The four words of block's counter, with products taken in 16-bit halves."""
    def product(a, m):
        a_hi, a_lo, m_hi, m_lo = a >> 16, a & 0xFFFF, m >> 16, m & 0xFFFF
        mid = a_hi * m_lo + ((a_lo * m_lo) >> 16)
        low_mid = (mid & 0xFFFF) + a_lo * m_hi
        return a_hi * m_hi + (mid >> 16) + (low_mid >> 16), ((low_mid & 0xFFFF) << 16) | ((a_lo * m_lo) & 0xFFFF)

    word = [block % 2 ** 32, block // 2 ** 32 + flag * 2 ** 31,
            torch.zeros_like(block) + offset % 2 ** 32, torch.zeros_like(block) + offset // 2 ** 32]
    key = [seed % 2 ** 32, seed // 2 ** 32]
    for _ in range(10):
        high_a, low_a = product(word[0], 0xD2511F53)
        high_b, low_b = product(word[2], 0xCD9E8D57)
        word = [high_b ^ word[1] ^ key[0], low_b, high_a ^ word[3] ^ key[1], low_a]
        key = [(key[0] + 0x9E3779B9) % 2 ** 32, (key[1] + 0xBB67AE85) % 2 ** 32]
    return word


def _exact_dropout(st):
    x, p = st["x"].double(), st["case"]["p"]
    element = torch.arange(x.numel(), device=x.device)
    block = torch.arange((x.numel() + 7) // 8, device=x.device)
    number = torch.zeros_like(element)
    for flag in (0, 1):
        words = _random_words(block, flag, st["seed"], st["offset"])
        for lane in range(8):
            mine = number[lane::8]
            half = (words[lane // 2][:mine.numel()] >> (16 * (lane % 2))) & 0xFFFF
            number[lane::8] = mine * 65536 + half
    threshold = round(p * 2 ** 32)
    out = x / (1 - p) * (number >= threshold).reshape(x.shape)
    return {"out": out + st["residual"].double() if "residual" in st else out}


def _exact_attention(st):
    case = st["case"]
    hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
    scale = 1 / math.sqrt(d)
    tq, tk = st["q"].shape[0], st["k"].shape[0]
    names = ["out"] + (["dq"] if case["train"] else [])
    res = {n: torch.zeros(tq, hq, d, dtype=torch.float64, device="cuda") for n in names}
    res["lse"] = torch.zeros(tq, hq, dtype=torch.float64, device="cuda")
    if case["train"]:
        res["dk"], res["dv"] = (torch.zeros(tk, hk, d, dtype=torch.float64, device="cuda") for _ in range(2))
    cu_q, cu_k = st["cu_q"].tolist(), st["cu_k"].tolist()
    q_all, k_all, v_all = st["q"].reshape(tq, hq, d), st["k"].reshape(tk, hk, d), st["v"].reshape(tk, hk, d)
    for s in range(len(cu_q) - 1):
        rows, keys = slice(cu_q[s], cu_q[s + 1]), slice(cu_k[s], cu_k[s + 1])
        nq, nk = cu_q[s + 1] - cu_q[s], cu_k[s + 1] - cu_k[s]
        if not nq:
            continue
        hidden = None
        if case["causal"]:
            hidden = torch.ones(nq, nk, dtype=torch.bool, device="cuda").tril(nk - nq).logical_not()
        for h in range(hq):
            q, k, v = q_all[rows, h].double(), k_all[keys, h // (hq // hk)].double(), v_all[keys, h // (hq // hk)].double()
            scores = q @ k.T * scale
            if hidden is not None:
                scores = scores.masked_fill(hidden, -math.inf)
            lse = torch.logsumexp(scores, 1)
            p = torch.exp(scores - lse[:, None])
            o = p @ v
            res["out"][rows, h], res["lse"][rows, h] = o, lse
            if case["train"]:
                do = st["dout"].reshape(tq, hq, d)[rows, h].double()
                ds = p * (do @ v.T - (p * (do @ v.T)).sum(1, keepdim=True))
                res["dv"][keys, h // (hq // hk)] += p.T @ do
                res["dq"][rows, h] = ds @ k * scale
                res["dk"][keys, h // (hq // hk)] += ds.T @ q * scale
    order = ["out", "lse"] + (["dq", "dk", "dv"] if case["train"] else [])
    return {n: res[n] if n == "lse" else res[n].reshape(res[n].shape[0], -1) for n in order}


def exact(case, seed):
    st = prepare(case, seed)
    return {"layer_norm": _exact_layer_norm, "dropout": _exact_dropout, "attention": _exact_attention}[case["op"]](st)
