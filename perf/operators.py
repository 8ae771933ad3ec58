"""Cases of the attention operators of ``rvc_cuda.attention``, with their plain forms.

Four operators: ``attention`` and ``attention_backward`` (states of another
length, padding, shared key/value heads, the bias of distance), the bias of
distance on its own with its gradient, and the per-head norm of queries and
keys with the rotation of positions, forward and backward.
"""

import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _module():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rvc-vulkan_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from rvc_cuda import attention

    return attention


# ------------------------------------------------------------------------ cases


def _attn(name, op, dtype, B, Hq, Hkv, D, Lq, Lk, mask="none", causal=False, buckets=0, max_distance=0):
    c = {"op": op, "dtype": dtype, "B": B, "Hq": Hq, "Hkv": Hkv, "D": D, "Lq": Lq, "Lk": Lk, "mask": mask,
         "causal": causal, "buckets": buckets, "max_distance": max_distance}
    return dict(c, name=name) if name else c


def _bias(name, op, dtype, B, H, Lq, Lk, buckets, max_distance, both):
    c = {"op": op, "dtype": dtype, "B": B, "Hq": H, "Lq": Lq, "Lk": Lk, "buckets": buckets,
         "max_distance": max_distance, "both": both}
    return dict(c, name=name) if name else c


def _rope(name, op, dtype, B, L, Hq, Hkv, D, R, interleaved):
    c = {"op": op, "dtype": dtype, "B": B, "L": L, "Hq": Hq, "Hkv": Hkv, "D": D, "R": R, "interleaved": interleaved}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one new frame attends to the 499 encoder frames of a 10 s chunk: latency only
        _attn("frame_499", "attn", "bf16", 1, 12, 12, 64, 1, 499),
        # a serving batch of new tokens over long ragged states, four query heads to a key head: bandwidth
        _attn("tokens_ragged", "attn", "bf16", 32, 16, 4, 128, 1, 8192, mask="lens"),
        # HuBERT's heads and type (12 x 64, fp32), a padded batch: 10 s of queries on 30 s of states
        _attn("hubert_fp32", "attn", "fp32", 8, 12, 12, 64, 499, 1499, mask="lens"),
        # a long prompt over longer states, shared key heads: tensor-core rate
        _attn("cross_long", "attn", "bf16", 2, 16, 4, 128, 2048, 16384),
        # self attention with the bias of distance, an odd length
        _attn("self_bias", "attn", "fp16", 4, 16, 16, 64, 2047, 2047, buckets=320, max_distance=800),
        # training step of a decoder that reads 30 s of encoder states with holes in the mask
        _attn("cross_train", "attn_bwd", "bf16", 8, 12, 12, 64, 251, 1499, mask="keys"),
        # training step of a causal self attention with the table's gradient
        _attn("self_bias_train", "attn_bwd", "bf16", 4, 16, 16, 64, 2048, 2048, causal=True, buckets=32,
              max_distance=128),
        # the text encoder's heads (2 x 96) and type, trained on a padded batch
        _attn("text_fp32_train", "attn_bwd", "fp32", 4, 2, 2, 96, 1000, 1000, mask="lens", buckets=32,
              max_distance=128),
        # the bias as a tensor, for an attention that takes one
        _bias("bias_499", "bias", "fp32", 1, 12, 499, 1499, 320, 800, True),
        # its gradient over a batch of long self attentions, odd rows
        _bias("bias_grad_long", "bias_bwd", "bf16", 4, 16, 4095, 4095, 320, 800, True),
        # one new token of each of 64 sequences
        _rope("rope_tokens", "rope", "bf16", 64, 1, 16, 4, 128, 128, False),
        # the backward pass of a training step
        _rope("rope_train", "rope_bwd", "bf16", 8, 4096, 16, 4, 128, 128, False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attn", "attn", "attn_bwd", "attn_bwd", "bias", "bias_bwd", "rope", "rope_bwd"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op in ("attn", "attn_bwd"):
        D = rng.choice([32, 40, 64, 64, 80, 96, 128, 128])
        Hkv, g = rng.choice([1, 2, 3, 4, 8, 12, 16]), rng.choice([1, 1, 2, 4, 8])
        Hq = Hkv * g
        Lq = rng.choice([1, rng.randint(2, 16), _log(rng, 17, 4096), _log(rng, 17, 4096)])
        Lk = _log(rng, 1, 16384)
        # pairs of queries and keys at most: those of cross_long forward in 16 bits, a tenth in 32 or backward
        most = 2 * 16 * 2048 * 16384 * (1.0 if op == "attn" and dtype != "fp32" else 0.1)
        B = _log(rng, 1, 64)
        while B > 1 and (B * Hq * Lq * Lk > most or B * (Lq * Hq + 2 * Lk * Hkv) * D > 3e8):
            B //= 2
        while Hq * Lq * Lk > most:
            Lk = max(1, Lk // 2)
        causal = rng.random() < 0.25
        buckets, dist = rng.choice([(0, 0), (0, 0), (32, 128), (320, 800)])
        return _attn("", op, dtype, B, Hq, Hkv, D, Lq, Lk, rng.choice(["none", "lens", "lens", "keys"]), causal,
                     buckets, dist)
    if op in ("bias", "bias_bwd"):
        H, Lq, Lk = rng.choice([1, 2, 8, 12, 16]), _log(rng, 1, 4096), _log(rng, 1, 4096)
        buckets, dist = rng.choice([(32, 128), (64, 256), (320, 800)])
        B = rng.choice([1, 1, 2, 4]) if op == "bias_bwd" else 1
        while B > 1 and B * H * Lq * Lk > (1 << 29):
            B //= 2
        return _bias("", op, dtype, B, H, Lq, Lk, buckets, dist, rng.random() < 0.7)
    D = rng.choice([32, 64, 96, 128, 128])
    L = rng.choice([1, _log(rng, 2, 4096)])
    Hkv, g = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4])
    B = _log(rng, 1, 64)
    while B > 1 and B * L * Hkv * (g + 1) * D > 8 * 4096 * 20 * 128:
        B //= 2
    return _rope("", op, dtype, B, L, Hkv * g, Hkv, D, rng.choice([D, D, D // 2]), rng.random() < 0.5)


# ----------------------------------------------------------------------- inputs


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = DTYPES[case["dtype"]]

    def n(*shape, scale=1.0, dtype=None):
        return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype or t)

    s = {"case": case}
    if case["op"] in ("attn", "attn_bwd"):
        B, Hq, Hkv, D, Lq, Lk = (case[x] for x in ("B", "Hq", "Hkv", "D", "Lq", "Lk"))
        # keys and values are the two halves of one projection of the states
        kv = n(B, Lk, 2, Hkv, D)
        s |= {"q": n(B, Lq, Hq, D), "k": kv[:, :, 0], "v": kv[:, :, 1], "lens": None, "keep": None, "table": None,
              "q_offset": Lk - Lq if case["causal"] else 0}
        if case["mask"] == "lens":  # a padded batch: from a quarter to all of the states, one of them whole
            s["lens"] = torch.randint(min(Lk, max(1, Lk // 4)), Lk + 1, (B,), generator=g, device="cuda",
                                      dtype=torch.int32)
            s["lens"][B // 2] = Lk
        elif case["mask"] == "keys":  # a tenth of the states is dropped
            s["keep"] = torch.rand((B, Lk), generator=g, device="cuda") >= 0.1
        if case["buckets"]:
            s["table"] = n(case["buckets"], Hq, scale=0.5)
        if case["op"] == "attn_bwd":
            s["out"], s["lse"] = _attention(s)
            s["dout"] = n(B, Lq, Hq, D)
    elif case["op"] in ("bias", "bias_bwd"):
        s["table"] = n(case["buckets"], case["Hq"], scale=0.5)
        if case["op"] == "bias_bwd":
            s["dbias"] = n(case["B"], case["Hq"], case["Lq"], case["Lk"])
    else:
        B, L, Hq, Hkv, D, R = (case[x] for x in ("B", "L", "Hq", "Hkv", "D", "R"))
        # queries, keys and values come out of one projection
        qkv = n(B, L, Hq + 2 * Hkv, D, scale=1.5)
        s |= {"q": qkv[:, :, :Hq], "k": qkv[:, :, Hq:Hq + Hkv], "wq": 1.0 + n(D, scale=0.1, dtype=torch.float32),
              "wk": 1.0 + n(D, scale=0.1, dtype=torch.float32)}
        angle = torch.arange(8192, device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (
            -torch.arange(0, R, 2, device="cuda", dtype=torch.float64) / R)
        s |= {"cos": angle.cos().float(), "sin": angle.sin().float()}
        s["positions"] = torch.randint(0, 8192 - L + 1, (B, 1), generator=g, device="cuda") + torch.arange(
            L, device="cuda")
        if case["op"] == "rope_bwd":
            s |= {"dqo": n(B, L, Hq, D), "dko": n(B, L, Hkv, D)}
    if own and s.get("table") is not None:
        both = case.get("both", not case.get("causal", False))
        s["bias"] = _module().BucketBias(s["table"], max_distance=case["max_distance"], bidirectional=both)
    return s


# ------------------------------------------------------------------ plain forms


def _borders(case):
    """The smallest distance of every bucket past the first, on whole numbers."""
    both = case.get("both", not case.get("causal", False))
    n = case["buckets"] // 2 if both else case["buckets"]
    e, far = n // 2, case["max_distance"]
    # bucket e + k begins at the first r with (r / e)^(n - e) >= (far / e)^k
    return both, n, list(range(1, e + 1)) + [
        next(r for r in range(e, far + 1) if r ** (n - e) * e ** k >= far ** k * e ** (n - e)) for k in range(1, n - e)]


_BORDERS = {}


def _buckets(case, lo, hi, device):
    """The bucket of every relative position lo .. hi - 1."""
    key = (case["buckets"], case["max_distance"], case.get("both", not case.get("causal", False)))
    if key not in _BORDERS:
        _BORDERS[key] = _borders(case)
    both, n, borders = _BORDERS[key]
    r = torch.arange(lo, hi, device=device)
    far = r.abs() if both else (-r).clamp_min(0)
    b = torch.bucketize(far, torch.tensor(borders, device=device), right=True)
    return b + n * (r > 0) if both else b


def _diagonals(s):
    """bias [H, Lq, Lk] in 32 bits from the table: one value to a diagonal."""
    c = s["case"]
    Lq, Lk, off = c["Lq"], c["Lk"], s.get("q_offset", 0)
    d = s["table"].float()[_buckets(c, 1 - Lq - off, Lk - off, s["table"].device)].t()
    i, j = torch.arange(Lq, device=d.device), torch.arange(Lk, device=d.device)
    return d[:, j[None] - i[:, None] + Lq - 1]


def _table_gradient(s, ds):
    """Sums of ds [H, Lq, Lk] over the diagonals (each row one further right in a wider sheet), then over the buckets."""
    c = s["case"]
    H, Lq, Lk = ds.shape
    off = s.get("q_offset", 0)
    wide = torch.nn.functional.pad(ds.flip(1), (0, Lq)).reshape(H, -1)[:, :Lq * (Lk + Lq - 1)]
    sums = wide.reshape(H, Lq, Lk + Lq - 1).sum(1, dtype=torch.float64)
    grad = torch.zeros((c["buckets"], H), device=ds.device, dtype=torch.float64)
    return grad.index_add_(0, _buckets(c, 1 - Lq - off, Lk - off, ds.device), sums.t()).to(s["table"].dtype)


def _alive(s):
    c, dev = s["case"], s["q"].device
    j = torch.arange(c["Lk"], device=dev)
    a = torch.ones((1, 1, 1, 1, c["Lk"]), device=dev, dtype=torch.bool)
    if s["lens"] is not None:
        a = a & (j < s["lens"][:, None])[:, None, None, None]
    if s["keep"] is not None:
        a = a & s["keep"][:, None, None, None]
    if c["causal"]:
        a = a & (j <= torch.arange(c["Lq"], device=dev)[:, None] + s["q_offset"])
    return a


def _weights(s):
    """Softmax weights [B, Hkv, g, Lq, Lk] and their log sums, q [B, Hkv, g Lq, D], k, v [B, Hkv, Lk, D], in 32 bits."""
    c = s["case"]
    B, Hkv, Lq, Lk, D = c["B"], c["Hkv"], c["Lq"], c["Lk"], c["D"]
    g = c["Hq"] // Hkv
    q = s["q"].float().permute(0, 2, 1, 3).reshape(B, Hkv, g * Lq, D)
    k, v = s["k"].float().transpose(1, 2), s["v"].float().transpose(1, 2)
    x = torch.matmul(q * D ** -0.5, k.transpose(2, 3)).reshape(B, Hkv, g, Lq, Lk)
    if s["table"] is not None:
        x = x + _diagonals(s).reshape(1, Hkv, g, Lq, Lk)
    if s["lens"] is not None or s["keep"] is not None or c["causal"]:
        x = torch.where(_alive(s), x, -math.inf)
    m = x.amax(-1, keepdim=True)
    x = torch.exp(x - torch.where(m > -math.inf, m, 0.0))
    l = x.sum(-1, keepdim=True)
    return x / torch.where(l > 0, l, 1.0), (m + torch.log(l)).squeeze(-1), q, k, v


def _attention(s):
    c = s["case"]
    B, Hq, Lq, Lk, D = c["B"], c["Hq"], c["Lq"], c["Lk"], c["D"]
    p, lse, _, _, v = _weights(s)
    out = torch.matmul(p.reshape(B, c["Hkv"], -1, Lk), v).reshape(B, Hq, Lq, D)
    return out.transpose(1, 2).to(s["q"].dtype).contiguous(), lse.reshape(B, Hq, Lq)


def _attention_backward(s):
    c = s["case"]
    B, Hq, Hkv, Lq, Lk, D = c["B"], c["Hq"], c["Hkv"], c["Lq"], c["Lk"], c["D"]
    p, _, q, k, v = _weights(s)
    p = p.reshape(B, Hkv, -1, Lk)
    do = s["dout"].float().permute(0, 2, 1, 3).reshape(B, Hkv, -1, D)
    dv = torch.matmul(p.transpose(2, 3), do)
    dp = torch.matmul(do, v.transpose(2, 3))
    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
    dq = torch.matmul(ds, k) * D ** -0.5
    dk = torch.matmul(ds.transpose(2, 3), q) * D ** -0.5
    t = s["q"].dtype
    r = [dq.reshape(B, Hq, Lq, D).transpose(1, 2).to(t).contiguous(), dk.transpose(1, 2).to(t).contiguous(),
         dv.transpose(1, 2).to(t).contiguous()]
    if s["table"] is not None:
        r.append(_table_gradient(s, ds.reshape(B, Hq, Lq, Lk).sum(0)))
    return tuple(r)


def _pairs(x, R, interleaved):
    """The two members of every rotated pair."""
    return (x[..., 0:R:2], x[..., 1:R:2]) if interleaved else (x[..., :R // 2], x[..., R // 2:R])


def _turn(x, cos, sin, R, interleaved):
    a, b = _pairs(x, R, interleaved)
    y = torch.stack((a * cos - b * sin, a * sin + b * cos), -1 if interleaved else -2).flatten(-2)
    return torch.cat((y, x[..., R:]), -1)


def _norm_rope(s, x, w):
    c = s["case"]
    x = x.float()
    cos, sin = s["cos"][s["positions"]][:, :, None], s["sin"][s["positions"]][:, :, None]
    y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w
    return _turn(y, cos, sin, c["R"], c["interleaved"])


def _norm_rope_backward(s, dy, x, w):
    c = s["case"]
    x = x.float()
    cos, sin = s["cos"][s["positions"]][:, :, None], s["sin"][s["positions"]][:, :, None]
    g = _turn(dy.float(), cos, -sin, c["R"], c["interleaved"])
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)
    n = x * r
    dw = (g * n).sum((0, 1, 2), dtype=torch.float64).float()
    g = g * w
    return r * (g - n * (g * n).mean(-1, keepdim=True)), dw


def run(state):
    s, c = state, state["case"]
    op = c["op"]
    if own:
        A = _module()
        if op in ("attn", "attn_bwd"):
            how = {"kv_lens": s["lens"], "key_mask": s["keep"], "causal": c["causal"], "q_offset": s["q_offset"],
                   "bias": s.get("bias")}
            if op == "attn":
                return A.attention(s["q"], s["k"], s["v"], **how)
            return A.attention_backward(s["dout"], s["q"], s["k"], s["v"], s["out"], s["lse"], **how)
        if op == "bias":
            return A.relative_bias(s["bias"], c["Lq"], c["Lk"])
        if op == "bias_bwd":
            return A.relative_bias_backward(s["bias"], s["dbias"])
        how = {"positions": s["positions"], "interleaved": c["interleaved"]}
        if op == "rope":
            return A.qk_norm_rope(s["q"], s["k"], s["wq"], s["wk"], s["cos"], s["sin"], **how)
        return A.qk_norm_rope_backward(s["dqo"], s["dko"], s["q"], s["k"], s["wq"], s["wk"], s["cos"], s["sin"], **how)
    if op == "attn":
        return _attention(s)
    if op == "attn_bwd":
        return _attention_backward(s)
    if op == "bias":
        return _diagonals(s).to(s["table"].dtype)
    if op == "bias_bwd":
        return _table_gradient(s, s["dbias"].sum(0, dtype=torch.float32))
    t = s["q"].dtype
    if op == "rope":
        return _norm_rope(s, s["q"], s["wq"]).to(t), _norm_rope(s, s["k"], s["wk"]).to(t)
    dq, dwq = _norm_rope_backward(s, s["dqo"], s["q"], s["wq"])
    dk, dwk = _norm_rope_backward(s, s["dko"], s["k"], s["wk"])
    return dq.to(t), dk.to(t), dwq, dwk


# ------------------------------------------------------------------ what it costs


def _mean_keys(c):
    """Keys that a query meets on average: a padded batch holds five eighths of its states, a causal row half a square."""
    n = float(c["Lk"])
    if c["mask"] == "lens":
        n *= 0.625 if c["B"] > 1 else 1.0
    elif c["mask"] == "keys":
        n *= 0.9
    if c["causal"]:
        q = min(c["Lq"], c["Lk"])
        n *= (q * (c["Lk"] - (q - 1) / 2)) / (c["Lq"] * c["Lk"])
    return n


def work(case):
    c = case
    size = 4 if c["dtype"] == "fp32" else 2
    if c["op"] in ("attn", "attn_bwd"):
        keys = c["Lk"] * (0.625 if c["mask"] == "lens" and c["B"] > 1 else 1.0)
        rows, states = c["B"] * c["Lq"] * c["Hq"], c["B"] * keys * c["Hkv"]
        pairs = rows * _mean_keys(c) * c["D"]
        if c["op"] == "attn":
            return {"bytes": (2 * rows + 2 * states) * c["D"] * size + 4 * rows, "flops": 4 * pairs}
        return {"bytes": (4 * rows + 2 * states + 2 * c["B"] * c["Lk"] * c["Hkv"]) * c["D"] * size + 4 * rows,
                "flops": 10 * pairs}
    if c["op"] in ("bias", "bias_bwd"):
        n = c["B"] * c["Hq"] * c["Lq"] * c["Lk"]
        return {"bytes": n * size + 2 * c["buckets"] * c["Hq"] * size, "flops": n if c["op"] == "bias_bwd" else 0}
    n = c["B"] * c["L"] * (c["Hq"] + c["Hkv"]) * c["D"]
    table = 4 * min(8192, c["B"] * c["L"]) * c["R"] + 8 * c["B"] * c["L"]
    return {"bytes": (2 if c["op"] == "rope" else 3) * n * size + table, "flops": (8 if c["op"] == "rope" else 20) * n}


# --------------------------------------------------------------------- 64 bits


def _exact_bucket(c, r):
    """The definition with logarithms; a distance that falls on a border within 1e-9 belongs behind it."""
    both = c.get("both", not c.get("causal", False))
    n = c["buckets"] // 2 if both else c["buckets"]
    e = n // 2
    a = r.abs() if both else torch.where(r < 0, -r, torch.zeros_like(r))
    y = torch.log(a.clamp_min(1).double() / e) / math.log(c["max_distance"] / e) * (n - e)
    b = torch.where(a < e, a, torch.clamp(e + torch.floor(y + 1e-9).long(), max=n - 1))
    return torch.where(r > 0, b + n, b) if both else b


def _exact_attention(s, backward):
    c = s["case"]
    B, Hq, Hkv, Lq, Lk, D = (c[x] for x in ("B", "Hq", "Hkv", "Lq", "Lk", "D"))
    dev, f8 = s["q"].device, torch.float64
    i, j = torch.arange(Lq, device=dev)[:, None] + s["q_offset"], torch.arange(Lk, device=dev)[None]
    where = _exact_bucket(c, j - i) if s["table"] is not None else None
    out = torch.zeros((B, Lq, Hq, D), device=dev, dtype=f8)
    lse = torch.full((B, Hq, Lq), -math.inf, device=dev, dtype=f8)
    dq = torch.zeros((B, Lq, Hq, D), device=dev, dtype=f8)
    dk, dv = (torch.zeros((B, Lk, Hkv, D), device=dev, dtype=f8) for _ in range(2))
    dt = torch.zeros((max(1, c["buckets"]), Hq), device=dev, dtype=f8)
    for b in range(B):
        keep = torch.ones((Lq, Lk), device=dev, dtype=torch.bool)
        if s["lens"] is not None:
            keep &= j < s["lens"][b]
        if s["keep"] is not None:
            keep &= s["keep"][b][None]
        if c["causal"]:
            keep &= j <= i
        live = keep.any(1)
        for h in range(Hq):
            kh = h * Hkv // Hq
            q, k, v = s["q"][b, :, h].to(f8), s["k"][b, :, kh].to(f8), s["v"][b, :, kh].to(f8)
            x = torch.einsum("id,jd->ij", q, k) / math.sqrt(D)
            if where is not None:
                x += s["table"][:, h].to(f8)[where]
            x.masked_fill_(~keep, -math.inf)
            z = torch.logsumexp(x, 1)
            lse[b, h] = z
            p = torch.exp(x - torch.where(live, z, torch.zeros_like(z))[:, None])
            if not backward:
                out[b, :, h] = p @ v
                continue
            do = s["dout"][b, :, h].to(f8)
            dp = do @ v.T
            ds = p * dp - p * torch.einsum("ij,ij->i", p, dp)[:, None]
            dv[b, :, kh] += p.T @ do
            dq[b, :, h] = ds @ k / math.sqrt(D)
            dk[b, :, kh] += ds.T @ q / math.sqrt(D)
            if where is not None:
                dt[:, h] += torch.bincount(where.reshape(-1), weights=ds.reshape(-1), minlength=c["buckets"])
    if not backward:
        return out, lse
    return (dq, dk, dv) if where is None else (dq, dk, dv, dt)


def _exact_rope(s, x, w, dy):
    c = s["case"]
    R, half = c["R"], c["R"] // 2
    d = torch.arange(half, device=x.device)
    a, b = (2 * d, 2 * d + 1) if c["interleaved"] else (d, d + half)
    x, w = x.double(), w.double()
    turn = torch.complex(s["cos"].double(), s["sin"].double())[s["positions"]][:, :, None]
    r = 1.0 / torch.sqrt((x * x).sum(-1, keepdim=True) / c["D"] + 1e-6)
    if dy is None:
        y = x * r * w
        z = torch.complex(y[..., a], y[..., b]) * turn
        y[..., a], y[..., b] = z.real, z.imag
        return y
    g = dy.double().clone()
    z = torch.complex(g[..., a], g[..., b]) * turn.conj()
    g[..., a], g[..., b] = z.real, z.imag
    dw = torch.einsum("blhd,blhd->d", g, x * r)
    g = g * w
    return g * r - x * r ** 3 * (g * x).sum(-1, keepdim=True) / c["D"], dw


def exact(case, seed):
    s, c = prepare(case, seed), case
    if c["op"] in ("attn", "attn_bwd"):
        return _exact_attention(s, c["op"] == "attn_bwd")
    if c["op"] in ("bias", "bias_bwd"):
        r = torch.arange(c["Lk"], device="cuda")[None] - torch.arange(c["Lq"], device="cuda")[:, None]
        where = _exact_bucket(c, r)
        if c["op"] == "bias":
            return s["table"].double().t()[:, where]
        return torch.stack([torch.bincount(where.reshape(-1), weights=s["dbias"][:, h].double().sum(0).reshape(-1),
                                           minlength=c["buckets"]) for h in range(c["Hq"])], 1)
    if c["op"] == "rope":
        return _exact_rope(s, s["q"], s["wq"], None), _exact_rope(s, s["k"], s["wk"], None)
    dq, dwq = _exact_rope(s, s["q"], s["wq"], s["dqo"])
    dk, dwk = _exact_rope(s, s["k"], s["wk"], s["dko"])
    return dq, dk, dwq, dwk
