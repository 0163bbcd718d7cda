"""Performance cases of the decoder operators: cross attention, add + RMS norm, products with 4-bit weights.

Each case is one call as a program makes it that reads a relational model's
object embeddings with a decoder: the norm in front of a sublayer, the cross
attention from ragged queries (candidate actions, tokens) to the ragged object
states of a batch, and the 4-bit projections of the same sublayers when they
are served. ``run`` computes either the plain form (elementary torch
operations in float32, rounded once) or the package's operators.
"""

from __future__ import annotations

import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f16": 2, "f32": 4}
_EPS = 1e-6
_E4M3_MAX = 448.0
_KEEP = 0.9  # share of the keys that a key mask leaves


# ---- cases ---------------------------------------------------------------------------


def _norm(name, kind, dtype, rows, width):
    return {"name": name, "op": "norm", "kind": kind, "dtype": dtype, "rows": rows, "width": width}


def _attn(name, kind, dtype, seqs, q_min, q_max, kv_min, kv_max, heads, kv_heads, dim, masked=False):
    return {"name": name, "op": "attn", "kind": kind, "dtype": dtype, "seqs": seqs, "q_min": q_min, "q_max": q_max,
            "kv_min": kv_min, "kv_max": kv_max, "heads": heads, "kv_heads": kv_heads, "dim": dim, "masked": masked}


def _int4(name, dtype, rows, n, k, group, zeros, quantized=False):
    return {"name": name, "op": "int4", "kind": "forward", "dtype": dtype, "rows": rows, "n": n, "k": k,
            "group": group, "zeros": zeros, "quantized": quantized}


def listed():
    return [
        # one served query entering a sublayer: latency, output in 8 bits for the projection behind it
        _norm("norm_one_row_e4m3", "e4m3", "bf16", 1, 4096),
        # the object embeddings of a micro-batch of 512 states x 100 objects (the 30-layer model's width), training
        _norm("norm_train_objects", "train", "bf16", 51200, 128),
        # float32 training with a width that is no multiple of a vector and a prime row count
        _norm("norm_train_f32_odd", "train", "f32", 10007, 1001),
        # a wide decoder's prefill: bandwidth
        _norm("norm_forward_wide", "forward", "bf16", 16384, 8192),
        # 512 states: each state's candidate actions (ragged) read its 100 objects; embedding 128 as 4 heads
        _attn("attn_train_states", "train", "bf16", 512, 8, 160, 100, 100, 4, 4, 32),
        # the small float32 model: 256 states x 50 objects, embedding 32, some objects masked
        _attn("attn_train_f32_masked", "train", "f32", 256, 4, 40, 50, 50, 2, 2, 16, True),
        # long prompts over long encoder states with shared key/value heads, training
        _attn("attn_train_long", "train", "bf16", 4, 2048, 2048, 4001, 4096, 16, 4, 128),
        # ragged prefill in float16 with masked states
        _attn("attn_prefill_f16", "forward", "f16", 16, 100, 3001, 301, 6000, 16, 16, 64, True),
        # a served batch, one new token each over cached states of very different lengths
        _attn("attn_decode_batch", "forward", "bf16", 48, 1, 1, 1000, 32001, 32, 8, 128),
        # one readout query over the objects of one state: latency
        _attn("attn_decode_one", "forward", "bf16", 1, 1, 1, 50, 50, 4, 4, 32),
        # one token through a served square projection
        _int4("int4_one_row", "bf16", 1, 4096, 4096, 128, False),
        # a small served batch through a wide projection, zero points
        _int4("int4_rows", "f16", 7, 16384, 8192, 64, True),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["norm", "norm", "train", "forward", "decode", "int4", "int4"])
    if kind == "norm":
        while True:
            c = _norm("", rng.choice(["train", "forward", "e4m3"]), rng.choice(["bf16", "f16", "f32"]),
                      _log(rng, 1, 60000), _log(rng, 16, 8192))
            if rng.random() < 0.6:
                c["width"] = max(16, c["width"] // 8 * 8)
            if c["rows"] * c["width"] <= 1.2e8:
                break
    elif kind == "int4":
        while True:
            group = rng.choice([32, 64, 128])
            k = max(group, _log(rng, 128, 16384) // group * group)
            quantized = rng.random() < 0.25
            c = _int4("", "bf16" if quantized else rng.choice(["bf16", "f16", "f32"]), _log(rng, 1, 16),
                      _log(rng, 64, 16384), k, group, rng.random() < 0.5, quantized)
            if c["n"] * k <= 1.3e8:
                break
    else:
        while True:
            dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
            dim = rng.choice([16, 32, 40, 64, 80, 96, 128])
            kv_heads = rng.choice([1, 2, 4, 8])
            heads = kv_heads * rng.choice([1, 1, 2, 4])
            masked = rng.random() < 0.4
            if kind == "decode":
                kv_max = _log(rng, 20, 120000)
                q = rng.choice([1, 1, 1, 2, 3])
                c = _attn("", "forward", dtype, _log(rng, 1, 128), q, q, max(1, kv_max // rng.choice([1, 2, 16])),
                          kv_max, heads, kv_heads, dim, masked)
            else:
                q_max, kv_max = _log(rng, 8, 4096), _log(rng, 16, 8192)
                c = _attn("", kind, dtype, _log(rng, 1, 512), max(1, q_max // rng.choice([1, 2, 8])), q_max,
                          max(1, kv_max // rng.choice([1, 2, 8])), kv_max, heads, kv_heads, dim, masked)
            w = work(c)
            fits = (c["seqs"] * heads * c["q_max"] * kv_max <= 4.5e8 and
                    c["seqs"] * kv_max * kv_heads * dim <= 1.2e9)
            if fits and w["bytes"] <= 3.0e9 and w["flops"] <= (3e11 if dtype == "f32" else 9e11):
                break
    del c["name"]
    return c


def _lengths(n, lo, hi):
    """``n`` lengths over [lo, hi], spread by a low-discrepancy sequence (the same for every seed)."""

    return [lo + int((hi - lo + 1) * ((i * 0.6180339887498949 + 0.37) % 1.0)) for i in range(n)]


def work(case):
    c, e = case, _SIZE[case["dtype"]]
    if c["op"] == "norm":
        n = c["rows"] * c["width"]
        if c["kind"] == "train":  # x, residual, dy, dh in; y, h, dx (one gradient for both addends) out
            return {"bytes": 7 * n * e + 2 * c["width"] * e, "flops": 20 * n}
        if c["kind"] == "e4m3":
            return {"bytes": 3 * n * e + n + 4 * c["rows"] + c["width"] * e, "flops": 8 * n}
        return {"bytes": 4 * n * e + c["width"] * e, "flops": 6 * n}
    if c["op"] == "int4":
        w = c["n"] * c["k"]
        x = c["rows"] * (c["k"] + 4 if c["quantized"] else c["k"] * e)
        groups = w // c["group"]
        return {"bytes": w // 2 + groups * (3 if c["zeros"] else 2) + x + c["rows"] * c["n"] * e,
                "flops": 2 * c["rows"] * w}
    ql, kl = _lengths(c["seqs"], c["q_min"], c["q_max"]), _lengths(c["seqs"], c["kv_min"], c["kv_max"])
    if c["masked"]:  # the last sequence keeps no key
        kl = [int(_KEEP * s) for s in kl[:-1]] + [0]
    pairs = sum(t * s for t, s in zip(ql, kl))
    qn, kn = sum(ql) * c["heads"] * c["dim"], sum(kl) * c["kv_heads"] * c["dim"]
    mask = sum(_lengths(c["seqs"], c["kv_min"], c["kv_max"])) if c["masked"] else 0
    product = 2 * pairs * c["heads"] * c["dim"]
    if c["kind"] == "train":  # q, k, v, do in; o, dq, dk, dv out; 2 products forward, 5 backward
        return {"bytes": (4 * qn + 4 * kn) * e + mask, "flops": 7 * product}
    return {"bytes": (2 * qn + 2 * kn) * e + mask, "flops": 2 * product}


# ---- inputs --------------------------------------------------------------------------


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    t = _TYPES[c["dtype"]]
    train = c["kind"] == "train"

    def randn(*shape, scale=1.0, grad=False):
        x = (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * scale).to(t)
        return x.requires_grad_(grad)

    s = {"case": c}
    if c["op"] == "norm":
        shape = (c["rows"], c["width"])
        s["x"], s["residual"] = randn(*shape, grad=train), randn(*shape, scale=2.0, grad=train)
        s["weight"] = (1 + 0.1 * randn(c["width"]).float()).to(t).requires_grad_(train)
        if train:
            s["dy"], s["dh"] = randn(*shape), randn(*shape)
        return s
    if c["op"] == "int4":
        groups = c["k"] // c["group"]
        s["codes"] = torch.randint(0, 256, (c["n"], c["k"] // 2), generator=g, device="cuda", dtype=torch.uint8)
        spread = torch.rand((c["n"], groups), generator=g, device="cuda") + 0.5
        s["scales"] = (spread * (0.3 / math.sqrt(c["k"]))).half()
        s["zeros"] = (torch.randint(4, 12, (c["n"], groups), generator=g, device="cuda", dtype=torch.uint8)
                      if c["zeros"] else None)
        x = randn(c["rows"], c["k"])
        if c["quantized"]:
            s["x_scale"] = x.float().abs().amax(1) / _E4M3_MAX
            s["x"] = (x.float() / s["x_scale"][:, None]).to(torch.float8_e4m3fn)
        else:
            s["x"], s["x_scale"] = x, None
        if own:  # the served program's weight handle, laid out once
            from relmo_b200.ops import decoder

            s["handle"] = decoder.Int4Weight(s["codes"], s["scales"], s["zeros"])
        return s
    ql, kl = _lengths(c["seqs"], c["q_min"], c["q_max"]), _lengths(c["seqs"], c["kv_min"], c["kv_max"])
    s["q"] = randn(sum(ql), c["heads"], c["dim"], grad=train)
    s["k"] = randn(sum(kl), c["kv_heads"], c["dim"], grad=train)
    s["v"] = randn(sum(kl), c["kv_heads"], c["dim"], grad=train)
    if train:
        s["do"] = randn(sum(ql), c["heads"], c["dim"])
    s["mask"] = None
    if c["masked"]:
        s["mask"] = torch.rand(sum(kl), generator=g, device="cuda") < _KEEP
        s["mask"][sum(kl[:-1]):] = False  # a state whose objects are all masked
    s["q_lengths"], s["kv_lengths"] = ql, kl
    s["q_len"] = torch.tensor(ql, device="cuda")
    s["kv_len"] = torch.tensor(kl, device="cuda")
    if own:  # the batch's plan, made once beside its routing
        from relmo_b200.ops import decoder

        s["plan"] = decoder.attention_plan(ql, kl, device="cuda")
    return s


# ---- one pass ------------------------------------------------------------------------


def run(state):
    op = state["case"]["op"]
    if own:
        return {"norm": _norm_own, "attn": _attn_own, "int4": _int4_own}[op](state)
    with torch.no_grad():
        return {"norm": _norm_plain, "attn": _attn_plain, "int4": _int4_plain}[op](state)


def _norm_own(s):
    from relmo_b200.ops import decoder

    kind = s["case"]["kind"]
    if kind == "e4m3":
        q, scale, h = decoder.add_rms_norm_e4m3(s["x"], s["weight"], s["residual"], eps=_EPS)
        return {"q": q, "scale": scale, "h": h}
    y, h = decoder.add_rms_norm(s["x"], s["weight"], s["residual"], eps=_EPS)
    if kind == "forward":
        return {"y": y, "h": h}
    dx, dr, dw = torch.autograd.grad((y, h), (s["x"], s["residual"], s["weight"]), (s["dy"], s["dh"]))
    return {"y": y, "h": h, "dx": dx, "dresidual": dr, "dweight": dw}


def _norm_plain(s):
    kind, t = s["case"]["kind"], s["x"].dtype
    w = s["weight"].float()
    h = s["x"].float() + s["residual"].float()
    inv = torch.rsqrt((h * h).mean(1, keepdim=True) + _EPS)
    n = h * inv
    y = n * w
    if kind == "e4m3":
        scale = y.abs().amax(1) / _E4M3_MAX
        scale = torch.where(scale == 0, torch.ones_like(scale), scale)
        q = (y / scale[:, None]).clamp(-_E4M3_MAX, _E4M3_MAX).to(torch.float8_e4m3fn)
        return {"q": q, "scale": scale, "h": h.to(t)}
    if kind == "forward":
        return {"y": y.to(t), "h": h.to(t)}
    dy = s["dy"].float()
    dw = (dy * n).sum(0)
    dn = dy * w
    dx = inv * (dn - n * (dn * n).mean(1, keepdim=True)) + s["dh"].float()
    dx = dx.to(t)
    return {"y": y.to(t), "h": h.to(t), "dx": dx, "dresidual": dx, "dweight": dw.to(t)}


def _int4_own(s):
    from relmo_b200.ops import decoder

    if s["case"]["quantized"]:
        return decoder.int4_matvec(s["x"], s["handle"], x_scale=s["x_scale"], out_dtype=torch.bfloat16)
    return decoder.int4_matvec(s["x"], s["handle"])


def _int4_plain(s):
    c = s["case"]
    codes = torch.stack((s["codes"] & 15, s["codes"] >> 4), dim=-1).view(c["n"], -1, c["group"]).float()
    zeros = s["zeros"].float()[:, :, None] if c["zeros"] else 8.0
    w = ((codes - zeros) * s["scales"].float()[:, :, None]).view(c["n"], c["k"])
    x = s["x"].float()
    if c["quantized"]:
        return ((x @ w.t()) * s["x_scale"][:, None]).to(torch.bfloat16)
    return (x @ w.t()).to(s["x"].dtype)


def _attn_own(s):
    from relmo_b200.ops import decoder

    o = decoder.cross_attention(s["q"], s["k"], s["v"], s["plan"], key_mask=s["mask"])
    if s["case"]["kind"] != "train":
        return o
    dq, dk, dv = torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["do"])
    return {"o": o, "dq": dq, "dk": dk, "dv": dv}


def _padded(length, longest):
    """Rows of a [seqs, longest] padding of packed rows, which of them exist, and each packed row's place in it."""

    end = length.cumsum(0)
    at = torch.arange(longest, device=length.device)
    exists = at < length[:, None]
    row = torch.where(exists, (end - length)[:, None] + at, 0)
    return row, exists, end


def _place(end, length, longest, rows):
    r = torch.arange(rows, device=end.device)
    b = torch.searchsorted(end, r, right=True)
    return b * longest + r - (end - length)[b]


def _attn_plain(s):
    c, t = s["case"], s["q"].dtype
    tm, sm = max(s["q_lengths"]), max(s["kv_lengths"])
    hk, g, d = c["kv_heads"], c["heads"] // c["kv_heads"], c["dim"]
    scale = 1 / math.sqrt(d)
    qrow, qok, qend = _padded(s["q_len"], tm)
    krow, kok, kend = _padded(s["kv_len"], sm)
    if s["mask"] is not None:
        kok = kok & s["mask"][krow]
    q = s["q"].float()[qrow].view(-1, tm, hk, g, d).permute(0, 2, 3, 1, 4).reshape(-1, hk, g * tm, d)
    k = s["k"].float()[krow].transpose(1, 2)
    v = s["v"].float()[krow].transpose(1, 2)
    p = (q @ k.transpose(2, 3)).mul_(scale).masked_fill_(~kok[:, None, None, :], -math.inf)
    top = p.amax(-1, keepdim=True)
    p = p.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    p = p.div_(torch.where(total == 0, 1.0, total))
    qplace = _place(qend, s["q_len"], tm, s["q"].size(0))

    def packed(x):  # [seqs, kv heads, group * tm, d] -> rows of q
        return (x.view(-1, hk, g, tm, d).permute(0, 3, 1, 2, 4).reshape(-1, hk * g, d)[qplace]).to(t)

    o = packed(p @ v)
    if c["kind"] != "train":
        return o
    do = s["do"].float()[qrow] * qok[:, :, None, None]
    do = do.view(-1, tm, hk, g, d).permute(0, 2, 3, 1, 4).reshape(-1, hk, g * tm, d)
    dv = p.transpose(2, 3) @ do
    ds = do @ v.transpose(2, 3)
    ds = ds.sub_((p * ds).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    dq = packed(ds @ k)
    dk = ds.transpose(2, 3) @ q
    kplace = _place(kend, s["kv_len"], sm, s["k"].size(0))
    dk, dv = ((x.transpose(1, 2).reshape(-1, hk, d)[kplace]).to(t) for x in (dk, dv))
    return {"o": o, "dq": dq, "dk": dk, "dv": dv}


# ---- the definitions in 64 bits ------------------------------------------------------


def _to_e4m3_grid(x):
    """Nearest value of the 8-bit type with 3 mantissa bits, ties to even, largest 448."""

    _, e = torch.frexp(x.abs().clamp_min(2.0**-6))
    step = torch.exp2((e - 4).double())
    return (torch.round(x / step) * step).clamp(-_E4M3_MAX, _E4M3_MAX)


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"norm": _norm_exact, "attn": _attn_exact, "int4": _int4_exact}[case["op"]](s, case)


def _norm_exact(s, c):
    x, r, w = s["x"].double(), s["residual"].double(), s["weight"].double()
    h = x + r
    rms = torch.sqrt(h.square().sum(1) / c["width"] + _EPS)
    y = h / rms[:, None] * w
    if c["kind"] == "e4m3":
        top = y.abs().max(1).values
        scale = torch.where(top > 0, top / _E4M3_MAX, 1.0)
        return {"q": _to_e4m3_grid(y / scale[:, None]), "scale": scale, "h": h}
    if c["kind"] == "forward":
        return {"y": y, "h": h}
    dy, dh = s["dy"].double(), s["dh"].double()
    # y_i = w_i h_i / rms, d rms / d h_j = h_j / (width rms)
    inner = (dy * w * h).sum(1) / (c["width"] * rms**3)
    dx = dy * w / rms[:, None] - h * inner[:, None] + dh
    dw = torch.einsum("rc,rc,r->c", dy, h, 1 / rms)
    return {"y": y, "h": h, "dx": dx, "dresidual": dx, "dweight": dw}


def _int4_exact(s, c):
    out = []
    x = s["x"].float().double()
    if c["quantized"]:
        x = x * s["x_scale"].double()[:, None]
    for lo in range(0, c["n"], 1024):
        codes = s["codes"][lo:lo + 1024].long()
        w = torch.empty(codes.size(0), c["k"], device=codes.device, dtype=torch.float64)
        w[:, 0::2], w[:, 1::2] = codes % 16, codes // 16
        z = s["zeros"][lo:lo + 1024].double() if c["zeros"] else torch.full_like(s["scales"][lo:lo + 1024], 8).double()
        w -= z.repeat_interleave(c["group"], 1)
        w *= s["scales"][lo:lo + 1024].double().repeat_interleave(c["group"], 1)
        out.append(x @ w.T)
    return torch.cat(out, 1)


def _attn_exact(s, c):
    if work(c)["flops"] > 2e12:
        return None
    train = c["kind"] == "train"
    g, scale = c["heads"] // c["kv_heads"], c["dim"] ** -0.5
    o, dq = (torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda") for _ in range(2))
    dk, dv = (torch.zeros(s["k"].shape, dtype=torch.float64, device="cuda") for _ in range(2))
    qa = ka = 0
    for t, n in zip(s["q_lengths"], s["kv_lengths"]):
        qs, ks = slice(qa, qa + t), slice(ka, ka + n)
        qa, ka = qa + t, ka + n
        keep = None if s["mask"] is None else s["mask"][ks].nonzero().squeeze(1)
        q, k, v = s["q"][qs].double(), s["k"][ks].double(), s["v"][ks].double()
        if keep is not None:
            k, v = k[keep], v[keep]
        if k.size(0) == 0:
            continue
        k, v = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)
        p = torch.softmax(torch.einsum("thd,shd->hts", q, k) * scale, -1)
        o[qs] = torch.einsum("hts,shd->thd", p, v)
        if not train:
            continue
        do = s["do"][qs].double()
        delta = (do * o[qs]).sum(-1).t()[:, :, None]
        ds = p * (torch.einsum("thd,shd->hts", do, v) - delta) * scale
        dq[qs] = torch.einsum("hts,shd->thd", ds, k)
        gk = torch.einsum("hts,thd->shd", ds, q).view(k.size(0), -1, g, c["dim"]).sum(2)
        gv = torch.einsum("hts,thd->shd", p, do).view(k.size(0), -1, g, c["dim"]).sum(2)
        at = torch.arange(n, device="cuda") if keep is None else keep
        dk[ks].index_copy_(0, at, gk)
        dv[ks].index_copy_(0, at, gv)
    return {"o": o, "dq": dq, "dk": dk, "dv": dv} if train else o
