"""Measured cases of the training operators: attention's backward pass, layer norm forward and backward, and
rotary embedding over several position axes in both directions.

Each case names its operator ("op") and sizes.  `run` makes the framework's calls where `own` is true and computes
the same outputs with elementary torch operations in 32 bits where it is false; `exact` computes them in 64 bits.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-5


def _framework():
    """The package's modules (they lie flat in its folder)."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    pkg = os.path.join(root, "flash-attn-economical-gpu_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import flash_atten
    import training

    return flash_atten, training


# ------------------------------------------------------------------ cases
def _attn(name, dtype, B, Hq, Hkv, M, N, D, causal):
    return {"name": name, "op": "attn_bwd", "dtype": dtype, "B": B, "Hq": Hq, "Hkv": Hkv, "M": M, "N": N, "D": D,
            "causal": causal}


def listed():
    return [
        # A short prompt through a small model: launches and latency count, not throughput.
        _attn("attn_short", "bf16", 1, 4, 2, 300, 300, 128, True),
        # One 2048-token sequence of a 28/4-head decoder (the prefill the framework times), fine-tuned causally.
        _attn("attn_gqa28_2048", "bf16", 1, 28, 4, 2048, 2048, 128, True),
        # A training batch of short sequences, plain multi-head.
        _attn("attn_mha_1024", "bf16", 4, 32, 32, 1024, 1024, 128, True),
        # Long-context training, four query heads to a key/value head: the largest case.
        _attn("attn_gqa_8192", "bf16", 2, 16, 4, 8192, 8192, 128, True),
        # Cross attention of odd lengths in fp16 with 64-wide heads: queries of a decoder over an encoder's keys.
        _attn("attn_cross_d64", "fp16", 2, 8, 8, 1000, 1531, 64, False),
        # Wide heads.
        _attn("attn_d256_2048", "bf16", 2, 16, 16, 2048, 2048, 256, True),
        # A packed batch of documents, one token to two thousand, one with queries and no keys, one with neither.
        {"name": "attn_packed", "op": "attn_bwd_packed", "dtype": "bf16", "Hq": 28, "Hkv": 4, "D": 128,
         "causal": True, "lens_q": "1031,1,37,0,2048,300,129", "lens_k": "1031,1,0,0,2048,300,200"},
        # One decoded token: the norm as serving calls it.
        {"name": "ln_token", "op": "ln_fwd", "dtype": "bf16", "wdtype": "bf16", "rows": 1, "cols": 3584,
         "residual": False},
        # The norm in front of a block at 8192 tokens, with the residual add, and its backward with fp32 weights.
        {"name": "ln_fwd_8192", "op": "ln_fwd", "dtype": "bf16", "wdtype": "bf16", "rows": 8192, "cols": 3584,
         "residual": True},
        {"name": "ln_bwd_8192", "op": "ln_bwd", "dtype": "bf16", "wdtype": "fp32", "rows": 8192, "cols": 3584,
         "residual": True},
        # Rotary of text and image tokens (time, height, width) over a 16384-token batch's 28 + 4 heads.
        {"name": "rope_text_image", "op": "rope", "dtype": "bf16", "tokens": 16384, "Hq": 28, "Hkv": 4, "D": 128,
         "sections": "16,24,24", "table": 32768, "inverse": False},
        # Backward of a vision encoder's two-axis rotary, odd patch count, 80-wide heads.
        {"name": "rope_patches_bwd", "op": "rope", "dtype": "fp16", "tokens": 4099, "Hq": 16, "Hkv": 16, "D": 80,
         "sections": "20,20", "table": 256, "inverse": True},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


MOST_PAIRS = 2 * 16 * 8192 * 8192  # query-key pairs over all heads of the largest listed case


def draw(rng):
    op = rng.choice(["attn_bwd", "attn_bwd", "attn_bwd_packed", "ln_fwd", "ln_bwd", "rope"])
    if op == "attn_bwd":
        D = rng.choice([40, 64, 72, 80, 96, 128, 128, 160, 192, 256])
        Hkv, g = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 1, 2, 4, 5, 7])
        M = _log(rng, 1, 8192)
        N = M if rng.random() < 0.6 else _log(rng, 1, 8192)
        B = _log(rng, 1, 8)
        while B > 1 and B * Hkv * g * M * N * max(D, 128) > MOST_PAIRS * 128:
            B -= 1
        while g > 1 and B * Hkv * g * M * N * max(D, 128) > MOST_PAIRS * 128:
            g -= 1
        return {"op": op, "dtype": rng.choice(["bf16", "bf16", "fp16"]), "B": B, "Hq": Hkv * g, "Hkv": Hkv, "M": M,
                "N": N, "D": D, "causal": rng.random() < 0.6}
    if op == "attn_bwd_packed":
        n = rng.randint(2, 9)
        lq = [0 if rng.random() < 0.1 else _log(rng, 1, 2048) for _ in range(n)]
        lk = [x if rng.random() < 0.7 else 0 if rng.random() < 0.2 else _log(rng, 1, 2048) for x in lq]
        if not sum(lq):
            lq[0] = 65
        if not sum(lk):
            lk[0] = 130
        while sum(lq) > 5120 or sum(lk) > 5120:
            lq, lk = lq[:-1], lk[:-1]
        Hkv, g = rng.choice([1, 2, 4]), rng.choice([1, 2, 7])
        return {"op": op, "dtype": rng.choice(["bf16", "fp16"]), "Hq": Hkv * g, "Hkv": Hkv,
                "D": rng.choice([64, 80, 128, 128, 256]), "causal": rng.random() < 0.6,
                "lens_q": ",".join(map(str, lq)), "lens_k": ",".join(map(str, lk))}
    if op in ("ln_fwd", "ln_bwd"):
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        cols = _log(rng, 64, 16384)
        if rng.random() < 0.7:
            cols = max(64, cols // 64 * 64)
        rows = _log(rng, 1, max(1, min(32768, (1 << 27) // cols)))
        return {"op": op, "dtype": dtype, "wdtype": rng.choice([dtype, "fp32"]), "rows": rows, "cols": cols,
                "residual": rng.random() < 0.5}
    D = rng.choice([64, 80, 96, 128, 256])
    axes = rng.choice([1, 2, 3])
    half = D // 2 if rng.random() < 0.7 else D // 4
    cuts = sorted(rng.sample(range(1, half), axes - 1))
    sections = [b - a for a, b in zip([0] + cuts, cuts + [half])]
    Hkv = rng.choice([1, 4, 8])
    return {"op": op, "dtype": rng.choice(["bf16", "fp16", "fp32"]), "tokens": _log(rng, 1, 16384),
            "Hq": Hkv * rng.choice([1, 2, 4]), "Hkv": Hkv, "D": D, "sections": ",".join(map(str, sections)),
            "table": rng.choice([64, 4096, 32768]), "inverse": rng.random() < 0.5}


# ----------------------------------------------------------------- inputs
def _ints(text):
    return [int(x) for x in text.split(",")]


def _pair_mask(M, N, causal, device):
    """Visible (query, key) pairs of one dense sequence: key n to query m iff n <= m, or all."""
    m = torch.arange(M, device=device)[:, None]
    n = torch.arange(N, device=device)[None, :]
    return n <= m if causal else (n >= 0).expand(M, N)


def _packed_mask(cu_q, cu_k, Tq, Tk, causal):
    """Visible pairs of a packed batch: same sequence and, causally, key place <= query place in it."""
    tq = torch.arange(Tq, device=cu_q.device)
    tk = torch.arange(Tk, device=cu_k.device)
    sq = torch.searchsorted(cu_q[1:].long(), tq, right=True)
    sk = torch.searchsorted(cu_k[1:].long(), tk, right=True)
    mask = sq[:, None] == sk[None, :]
    if causal:
        mask = mask & ((tk - cu_k.long()[sk])[None, :] <= (tq - cu_q.long()[sq])[:, None])
    return mask


def _forward(q, k, v, mask, scale):
    """o and lse of [heads, rows, D] in 32 bits, as a forward pass leaves them: NaN and -inf in rows that see no key."""
    s = (q.float() @ k.float().transpose(-1, -2) * scale).masked_fill_(~mask, -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.exp(s.sub_(lse[..., None]))
    return p @ v.float(), lse


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    op, dt = case["op"], DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    if op == "attn_bwd":
        B, Hq, Hkv, M, N, D = (case[x] for x in ("B", "Hq", "Hkv", "M", "N", "D"))
        q, k, v = randn(B, Hq, M, D).to(dt), randn(B, Hkv, N, D).to(dt), randn(B, Hkv, N, D).to(dt)
        # Gradients as a loss scaled for 16 bits gives them: tokens differ in size by powers of two.
        dout = (randn(B, Hq, M, D) * torch.exp2(torch.round(randn(B, 1, M, 1)) - 2)).to(dt)
        o = torch.empty_like(q)
        lse = torch.empty(B, Hq, M, device=dev)
        mask = _pair_mask(M, N, case["causal"], dev)
        for b in range(B):
            kb, vb = (t[b].repeat_interleave(Hq // Hkv, 0) for t in (k, v))
            ob, lb = _forward(q[b], kb, vb, mask, D ** -0.5)
            o[b], lse[b] = ob.to(dt), lb
        return {"case": case, "dout": dout, "q": q, "k": k, "v": v, "o": o, "lse": lse}
    if op == "attn_bwd_packed":
        Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
        lq, lk = _ints(case["lens_q"]), _ints(case["lens_k"])
        cu_q = torch.tensor([0] + lq, device=dev).cumsum(0).to(torch.int32)
        cu_k = torch.tensor([0] + lk, device=dev).cumsum(0).to(torch.int32)
        Tq, Tk = sum(lq), sum(lk)
        q, k, v = randn(Tq, Hq, D).to(dt), randn(Tk, Hkv, D).to(dt), randn(Tk, Hkv, D).to(dt)
        dout = (randn(Tq, Hq, D) * torch.exp2(torch.round(randn(Tq, 1, 1)) - 2)).to(dt)
        mask = _packed_mask(cu_q, cu_k, Tq, Tk, case["causal"])
        ke, ve = (t.transpose(0, 1).repeat_interleave(Hq // Hkv, 0) for t in (k, v))
        o, lse = _forward(q.transpose(0, 1), ke, ve, mask, D ** -0.5)
        return {"case": case, "dout": dout, "q": q, "k": k, "v": v, "o": o.transpose(0, 1).to(dt).contiguous(),
                "lse": lse.contiguous(), "cu_q": cu_q, "cu_k": cu_k, "max_q": max(lq), "max_k": max(lk)}
    if op in ("ln_fwd", "ln_bwd"):
        rows, cols, wdt = case["rows"], case["cols"], DTYPES[case["wdtype"]]
        # A residual stream: columns of different size, an offset, rows of different size.
        col = torch.exp(0.5 * randn(cols))
        x = ((randn(rows, cols) * col + 0.3) * torch.exp(0.3 * randn(rows, 1))).to(dt)
        w = (1 + 0.2 * randn(cols)).to(wdt)
        b = (0.2 * randn(cols)).to(wdt)
        extra = randn(rows, cols).to(dt) if case["residual"] else None
        state = {"case": case, "x": x, "w": w, "b": b, "extra": extra}
        if op == "ln_bwd":
            xf = x.float()
            mean = xf.mean(1)
            state["mean"] = mean
            state["rstd"] = torch.rsqrt((xf - mean[:, None]).square().mean(1) + EPS)
            state["dy"] = (randn(rows, cols) * 0.25).to(dt)
        return state
    T, D, sections = case["tokens"], case["D"], _ints(case["sections"])
    half = sum(sections)
    # q and k as the projection leaves them: column blocks of one packed row per token.
    qkv = randn(T, case["Hq"] + 2 * case["Hkv"], D).to(dt)
    q, k = qkv[:, :case["Hq"]], qkv[:, case["Hq"]:case["Hq"] + case["Hkv"]]
    pos = torch.randint(0, case["table"], (len(sections), T), generator=g, device=dev, dtype=torch.int32)
    freq = 10000.0 ** (-torch.arange(half, device=dev, dtype=torch.float64) / half)
    ang = torch.arange(case["table"], device=dev, dtype=torch.float64)[:, None] * freq
    return {"case": case, "q": q, "k": k, "pos": pos, "cos": ang.cos().float(), "sin": ang.sin().float(),
            "sections": tuple(sections)}


# -------------------------------------------------------------- plain form
def _plain_attention(dout, q, k, v, o, lse, mask, scale):
    """Gradients for [..., heads, rows, D] with grouped key/value heads, in 32 bits."""
    Hq, Hkv = q.shape[-3], k.shape[-3]
    g = Hq // Hkv
    qf, dof, of = q.float(), dout.float(), o.float()
    kf, vf = (t.float().repeat_interleave(g, -3) for t in (k, v))
    p = torch.exp((qf @ kf.transpose(-1, -2)).mul_(scale).sub_(lse[..., None]))
    p = torch.where(mask, p, 0.0)
    dv = p.transpose(-1, -2) @ dof
    ds = (dof @ vf.transpose(-1, -2)).sub_((dof * of).sum(-1, keepdim=True)).mul_(p)
    del p
    ds = torch.where(mask, ds, 0.0)
    dq = (ds @ kf).mul_(scale)
    dk = (ds.transpose(-1, -2) @ qf).mul_(scale)
    del ds
    dk, dv = (t.unflatten(-3, (Hkv, g)).sum(-3) for t in (dk, dv))
    return dq, dk, dv


def _plain(state):
    case = state["case"]
    op, dt = case["op"], DTYPES[case["dtype"]]
    if op == "attn_bwd":
        mask = _pair_mask(case["M"], case["N"], case["causal"], state["q"].device)
        grads = _plain_attention(state["dout"], state["q"], state["k"], state["v"], state["o"], state["lse"], mask,
                                 case["D"] ** -0.5)
        return tuple(map(lambda t: t.to(dt), grads))
    if op == "attn_bwd_packed":
        q, k, v, o, dout = map(lambda n: state[n].transpose(0, 1), ("q", "k", "v", "o", "dout"))
        mask = _packed_mask(state["cu_q"], state["cu_k"], q.shape[1], k.shape[1], case["causal"])
        grads = _plain_attention(dout, q, k, v, o, state["lse"], mask, case["D"] ** -0.5)
        return tuple(map(lambda t: t.transpose(0, 1).to(dt), grads))
    if op == "ln_fwd":
        x = state["x"]
        if state["extra"] is not None:
            x = (x.float() + state["extra"].float()).to(dt)
        xf = x.float()
        mean = xf.mean(1)
        c = xf - mean[:, None]
        rstd = torch.rsqrt(c.square().mean(1) + EPS)
        y = (c * rstd[:, None] * state["w"].float() + state["b"].float()).to(dt)
        return (y, mean, rstd) if state["extra"] is None else (y, mean, rstd, x)
    if op == "ln_bwd":
        dy, rstd, wdt = state["dy"].float(), state["rstd"][:, None], state["w"].dtype
        xhat = (state["x"].float() - state["mean"][:, None]) * rstd
        gw = dy * state["w"].float()
        dx = rstd * (gw - gw.mean(1, keepdim=True) - xhat * (gw * xhat).mean(1, keepdim=True))
        if state["extra"] is not None:
            dx = dx + state["extra"].float()
        return dx.to(dt), (dy * xhat).sum(0).to(wdt), dy.sum(0).to(wdt)
    axis = torch.repeat_interleave(torch.arange(len(state["sections"]), device=state["pos"].device),
                                   torch.tensor(state["sections"], device=state["pos"].device),
                                   output_size=sum(state["sections"]))
    rows = state["pos"].long()[axis].t()  # [tokens, half]: the table row of each pair
    cos, sin = state["cos"].gather(0, rows)[:, None], state["sin"].gather(0, rows)[:, None]
    if case["inverse"]:
        sin = -sin
    half = cos.shape[-1]

    def rotate(x):
        lo, hi, rest = x[..., :half].float(), x[..., half:2 * half].float(), x[..., 2 * half:].float()
        return torch.cat((lo * cos - hi * sin, hi * cos + lo * sin, rest), -1).to(dt)

    return rotate(state["q"]), rotate(state["k"])


# ------------------------------------------------------------------- calls
def run(state):
    if not own:
        return _plain(state)
    flash_atten, training = _framework()
    case = state["case"]
    op = case["op"]
    if op == "attn_bwd":
        return flash_atten.attention_backward(state["dout"], state["q"], state["k"], state["v"], state["o"],
                                              state["lse"], causal=case["causal"])
    if op == "attn_bwd_packed":
        return flash_atten.attention_backward_varlen(state["dout"], state["q"], state["k"], state["v"], state["o"],
                                                     state["lse"], state["cu_q"], state["cu_k"], state["max_q"],
                                                     state["max_k"], causal=case["causal"])
    if op == "ln_fwd":
        return training.layernorm_forward(state["x"], state["w"], state["b"], eps=EPS, residual=state["extra"])
    if op == "ln_bwd":
        return training.layernorm_backward(state["dy"], state["x"], state["w"], state["mean"], state["rstd"],
                                           dresidual=state["extra"])
    return training.rope_multi_axis(state["q"], state["k"], state["pos"], state["cos"], state["sin"],
                                    state["sections"], inverse=case["inverse"])


# ------------------------------------------------------------- needed work
def _visible(M, N, causal):
    if not causal:
        return M * N
    return sum(min(m + 1, N) for m in range(M))


def work(case):
    op = case["op"]
    size = 4 if case["dtype"] == "fp32" else 2
    if op in ("attn_bwd", "attn_bwd_packed"):
        D, Hq, Hkv = case["D"], case["Hq"], case["Hkv"]
        if op == "attn_bwd":
            lens = [(case["M"], case["N"])] * case["B"]
        else:
            lens = list(zip(_ints(case["lens_q"]), _ints(case["lens_k"])))
        tq, tk = sum(m for m, _ in lens), sum(n for _, n in lens)
        pairs = sum(_visible(m, n, case["causal"]) for m, n in lens)
        # q, o, dout in and dq out; k, v in and dk, dv out; lse.
        return {"bytes": size * D * (4 * Hq * tq + 4 * Hkv * tk) + 4 * Hq * tq, "flops": 10 * Hq * pairs * D}
    if op in ("ln_fwd", "ln_bwd"):
        n, cols, w = case["rows"] * case["cols"], case["cols"], 4 if case["wdtype"] == "fp32" else 2
        if op == "ln_fwd":
            return {"bytes": size * n * (4 if case["residual"] else 2) + 2 * w * cols + 8 * case["rows"],
                    "flops": 8 * n}
        return {"bytes": size * n * (4 if case["residual"] else 3) + 3 * w * cols + 8 * case["rows"],
                "flops": 13 * n}
    sections = _ints(case["sections"])
    elems = case["tokens"] * (case["Hq"] + case["Hkv"]) * case["D"]
    rot = case["tokens"] * (case["Hq"] + case["Hkv"]) * 2 * sum(sections)
    rows = min(case["tokens"], case["table"])
    return {"bytes": 2 * size * elems + 4 * case["tokens"] * len(sections) + 8 * rows * sum(sections),
            "flops": 3 * rot}


# ------------------------------------------------------------ 64-bit values
def _exact_heads(dout, q, k, v, o, lse, visible, scale):
    """One sequence: [Hq, M, D] and [Hkv, N, D] in 64 bits, a head at a time."""
    Hq, Hkv = q.shape[0], k.shape[0]
    dq, dk, dv = (torch.zeros(t.shape, dtype=torch.float64, device=t.device) for t in (q, k, v))
    for h in range(Hq):
        kv = h // (Hq // Hkv)
        Q, K, V, dO, O = q[h].double(), k[kv].double(), v[kv].double(), dout[h].double(), o[h].double()
        logp = scale * torch.einsum("md,nd->mn", Q, K) - lse[h].double()[:, None]
        P = logp.exp().masked_fill(~visible, 0.0)
        dP = torch.einsum("md,nd->mn", dO, V)
        dS = (P * (dP - torch.einsum("md,md->m", dO, O)[:, None])).masked_fill(~visible, 0.0)
        dq[h] = scale * torch.einsum("mn,nd->md", dS, K)
        dk[kv] += scale * torch.einsum("mn,md->nd", dS, Q)
        dv[kv] += torch.einsum("mn,md->nd", P, dO)
    return dq, dk, dv


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "attn_bwd":
        visible = _pair_mask(case["M"], case["N"], case["causal"], s["q"].device)
        each = [_exact_heads(*(s[n][b] for n in ("dout", "q", "k", "v", "o", "lse")), visible, case["D"] ** -0.5)
                for b in range(case["B"])]
        return tuple(torch.stack(t) for t in zip(*each))
    if op == "attn_bwd_packed":
        dq, dk, dv = (torch.zeros(s[n].shape, dtype=torch.float64, device=s[n].device) for n in ("q", "k", "v"))
        q0 = k0 = 0
        for m, n in zip(_ints(case["lens_q"]), _ints(case["lens_k"])):
            Q, dO, O = (s[x][q0:q0 + m].transpose(0, 1) for x in ("q", "dout", "o"))
            K, V = (s[x][k0:k0 + n].transpose(0, 1) for x in ("k", "v"))
            got = _exact_heads(dO, Q, K, V, O, s["lse"][:, q0:q0 + m],
                               _pair_mask(m, n, case["causal"], Q.device), case["D"] ** -0.5)
            if n:
                dq[q0:q0 + m], dk[k0:k0 + n], dv[k0:k0 + n] = (t.transpose(0, 1) for t in got)
            q0, k0 = q0 + m, k0 + n
        return dq, dk, dv
    if op == "ln_fwd":
        x = s["x"]
        if s["extra"] is not None:
            x = (x.double() + s["extra"].double()).to(x.dtype)  # the sum is kept in x's own type
        x = x.double()
        mean = x.sum(1) / case["cols"]
        var = ((x - mean[:, None]) ** 2).sum(1) / case["cols"]
        rstd = 1 / torch.sqrt(var + EPS)
        y = (x - mean[:, None]) * rstd[:, None] * s["w"].double() + s["b"].double()
        return (y, mean, rstd) if s["extra"] is None else (y, mean, rstd, x)
    if op == "ln_bwd":
        x, dy, w, cols = s["x"].double(), s["dy"].double(), s["w"].double(), case["cols"]
        mean, rstd = s["mean"].double()[:, None], s["rstd"].double()[:, None]
        xh = (x - mean) * rstd
        a = (dy * w).sum(1, keepdim=True) / cols
        b = (dy * w * xh).sum(1, keepdim=True) / cols
        dx = rstd * (dy * w - a - b * xh)
        if s["extra"] is not None:
            dx = dx + s["extra"].double()
        return dx, (dy * xh).sum(0), dy.sum(0)
    outs = []
    for x in (s["q"], s["k"]):
        z = x.double().clone()
        half, at = sum(s["sections"]), 0
        for axis, n in enumerate(s["sections"]):
            c = s["cos"].double()[s["pos"][axis].long(), at:at + n][:, None]
            t = s["sin"].double()[s["pos"][axis].long(), at:at + n][:, None]
            t = -t if case["inverse"] else t
            lo, hi = x[..., at:at + n].double(), x[..., half + at:half + at + n].double()
            z[..., at:at + n] = lo * c - hi * t
            z[..., half + at:half + at + n] = hi * c + lo * t
            at += n
        outs.append(z)
    return tuple(outs)
