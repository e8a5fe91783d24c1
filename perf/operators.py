"""The operators on 4-bit block-scaled floating point and the few-token expert layer: what they are
measured on, their plain forms, and their definitions in 64 bits.

``own`` chooses between the plain form (elementary torch operations in 32 bits) and the calls a user
makes of the package.  Four operators:

* ``quantise``: rows to E2M1 codes with a scale per block of 16 (E4M3, and one fp32 scale for the whole
  matrix) or of 32 (E8M0), and back to numbers;
* ``product``: ``c[m,n] = a[m,k] . b[n,k]^T`` of two such matrices;
* ``decode``: router, both expert products and the weighted sum for at most 16 tokens, 16-bit experts;
* ``decode4``: the same with experts in the 4-bit format.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ----------------------------------------------------------------------------------------------------
# the cases
# ----------------------------------------------------------------------------------------------------
def listed():
    return [
        # one token's hidden state before a 4-bit projection
        {"name": "quantise 1 token", "op": "quantise", "rows": 1, "cols": 4096, "block": 16, "dtype": "bf16"},
        # a ragged batch of wide fp32 rows
        {"name": "quantise 1111 fp32 rows", "op": "quantise", "rows": 1111, "cols": 2080, "block": 16, "dtype": "fp32"},
        # a prompt's activations
        {"name": "quantise 16384 tokens", "op": "quantise", "rows": 16384, "cols": 4096, "block": 32, "dtype": "fp16"},
        # the projection of a single token: latency
        {"name": "product 1 token", "op": "product", "m": 1, "n": 4096, "k": 4096, "block": 16, "dtype": "bf16"},
        # a small batch with sizes that divide nothing
        {"name": "product 333 tokens", "op": "product", "m": 333, "n": 1399, "k": 2080, "block": 32, "dtype": "fp16"},
        # a prompt's up projection
        {"name": "product 8192 tokens", "op": "product", "m": 8192, "n": 14336, "k": 4096, "block": 16, "dtype": "bf16"},
        # single-token generation with 64 fine-grained experts
        {"name": "decode 1 token 64 experts", "op": "decode", "m": 1, "h": 2048, "i": 1408, "e": 64, "k": 6, "dtype": "fp16"},
        # the same layer with a handful of sequences
        {"name": "decode 5 tokens 64 experts", "op": "decode", "m": 5, "h": 2048, "i": 1408, "e": 64, "k": 6, "dtype": "bf16"},
        # single-token generation with 8 large experts
        {"name": "decode 1 token 8 experts", "op": "decode", "m": 1, "h": 4096, "i": 14336, "e": 8, "k": 2, "dtype": "bf16"},
        # the largest batch of the layer: every expert is read
        {"name": "decode 16 tokens 8 experts", "op": "decode", "m": 16, "h": 4096, "i": 14336, "e": 8, "k": 2, "dtype": "bf16"},
        # 4-bit experts, single token
        {"name": "decode4 1 token 8 experts", "op": "decode4", "m": 1, "h": 4096, "i": 14336, "e": 8, "k": 2, "block": 16, "dtype": "bf16"},
        # 4-bit experts, many of them, the largest batch
        {"name": "decode4 16 tokens 64 experts", "op": "decode4", "m": 16, "h": 2048, "i": 1408, "e": 64, "k": 6, "block": 32, "dtype": "bf16"},
    ]


def _log(rng, lo, hi, step):
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi)))) // step * step))


def draw(rng):
    op = rng.choice(["quantise", "product", "decode", "decode", "decode4", "decode4"])
    block = rng.choice([16, 32])
    if op == "quantise":
        return {"op": op, "rows": _log(rng, 1, 16384, 1), "cols": _log(rng, 64, 4096, 32), "block": block,
                "dtype": rng.choice(["bf16", "fp16", "fp32"])}
    if op == "product":
        return {"op": op, "m": _log(rng, 1, 8192, 1), "n": _log(rng, 16, 14336, 1), "k": _log(rng, 64, 4096, 32),
                "block": block, "dtype": rng.choice(["bf16", "fp16"])}
    e = rng.choice([4, 8, 16, 60, 64, 128])
    step = 8 if op == "decode" else 32
    h = _log(rng, 256, 4096, step)
    i = _log(rng, 256, min(14336, 8 * 14336 // e), step)
    case = {"op": op, "m": rng.randint(1, 16), "h": h, "i": i, "e": e, "k": rng.randint(1, min(8, e)),
            "dtype": rng.choice(["bf16", "fp16"])}
    if op == "decode4":
        case["block"] = block
        if block == 32:
            case["dtype"] = "bf16"      # E8M0 scales reach beyond what fp16 holds
    return case


# ----------------------------------------------------------------------------------------------------
# inputs
# ----------------------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _codes(g, *shape):
    """Random packed E2M1 pairs."""
    return torch.randint(0, 256, shape, generator=g, device="cuda", dtype=torch.uint8)


def _scales(g, block, std, *shape):
    """Block scales such that uniformly drawn codes (rms 2.9) stand for numbers of about ``std``; the E4M3 kind
    uses its upper range together with one fp32 scale per matrix, as quantising real weights does."""
    r = torch.rand(shape, generator=g, device="cuda")
    if block == 16:
        scale = (100.0 + 300.0 * r).to(torch.float8_e4m3fn)
        return scale, std / 2.9 / 250.0
    e = round(math.log2(std / 2.9)) + 127
    return (e - 1 + (3 * r).floor()).to(torch.uint8).view(torch.float8_e8m0fnu), None


def _fp4_matrix(g, block, std, lead, rows, cols):
    q = _codes(g, *lead, rows, cols // 2)
    scale, gs = _scales(g, block, std, *lead, rows, cols // block)
    if gs is None:
        return q, scale, None
    n = lead[0] if lead else 1
    gscale = gs * (0.75 + 0.5 * torch.rand(n, generator=g, device="cuda"))
    return q, scale, gscale


def prepare(case, seed):
    g = _gen(seed)
    dt = DTYPES[case["dtype"]]
    op = case["op"]
    if op == "quantise":
        x = torch.randn(case["rows"], case["cols"], generator=g, device="cuda")
        x[:, ::97] *= 8.0                                       # the outlier channels of real activations
        return {"op": op, "x": x.to(dt), "block": case["block"]}
    if op == "product":
        a = _fp4_matrix(g, case["block"], 1.0, (), case["m"], case["k"])
        b = _fp4_matrix(g, case["block"], 0.02, (), case["n"], case["k"])
        return {"op": op, "a": a, "b": b, "dtype": dt, "block": case["block"]}
    m, h, i, e = case["m"], case["h"], case["i"], case["e"]
    x = torch.randn(m, h, generator=g, device="cuda").to(dt)
    gate = (torch.randn(e, h, generator=g, device="cuda") * 0.02).to(dt).t()
    s = {"op": op, "x": x, "gate": gate, "k": case["k"]}
    if op == "decode":
        w1 = torch.empty(e, 2 * i, h, dtype=dt, device="cuda")
        w2 = torch.empty(e, h, i, dtype=dt, device="cuda")
        for j in range(e):
            w1[j] = torch.randn(2 * i, h, generator=g, device="cuda") * 0.02
            w2[j] = torch.randn(h, i, generator=g, device="cuda") * 0.02
        s["w1"], s["w2"] = w1, w2
    else:
        s["w1"] = _fp4_matrix(g, case["block"], 0.02, (e,), 2 * i, h)
        s["w2"] = _fp4_matrix(g, case["block"], 0.02, (e,), h, i)
        s["block"] = case["block"]
    return s


# ----------------------------------------------------------------------------------------------------
# the plain form
# ----------------------------------------------------------------------------------------------------
def _e2m1_index(a):
    """Index into 0, .5, 1, 1.5, 2, 3, 4, 6 of the nearest value, ties to the even index."""
    return ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))


def _table(device):
    return torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0],
                        device=device)


def _quantise_plain(x, block):
    xf = x.float().unflatten(-1, (-1, block))
    amax = xf.abs().amax(-1)
    if block == 16:
        top = amax.max()
        gscale = torch.where(top > 0, (top / torch.full_like(top, 2688.0)).clamp_min(2.0 ** -110), torch.ones_like(top))
        s = (amax / (6.0 * gscale)).clamp_max(448.0).to(torch.float8_e4m3fn).float()
        unit = s * gscale
        inv = torch.where(unit > 0, 1.0 / unit, torch.zeros_like(unit))
    else:
        gscale = None
        e = (torch.frexp(amax).exponent - 3).clamp_min(-127)
        e = torch.where(amax > 0, e, torch.full_like(e, -127))
        s = unit = torch.ldexp(torch.ones_like(amax), e)
        inv = torch.ldexp(torch.ones_like(amax), -e)
    r = xf * inv.unsqueeze(-1)
    value = _table(x.device)[_e2m1_index(r.abs()).int()].copysign(r) * unit.unsqueeze(-1)
    return value.flatten(-2).to(x.dtype), s, gscale


def _numbers(q, scale, gscale):
    """What codes and scales stand for, fp32."""
    pair = torch.stack((q & 15, q >> 4), -1).flatten(-2)
    block = pair.shape[-1] // scale.shape[-1]
    s = scale.float() if gscale is None else scale.float() * gscale.view(-1, *[1] * (scale.dim() - 1))
    return (_table(q.device)[pair.int()].unflatten(-1, (-1, block)) * s.unsqueeze(-1)).flatten(-2)


def _route_plain(x, gate, k):
    logits = x.float() @ gate.float()
    top, ids = torch.sort(logits, dim=1, descending=True, stable=True)
    top, ids = top[:, :k], ids[:, :k]
    w = (top - top[:, :1]).exp()
    return w / w.sum(1, keepdim=True), ids


def _pick(w, ids):
    """The experts that ``ids`` names, from a tensor or from the three tensors of the 4-bit format, in fp32."""
    if isinstance(w, tuple):
        q, scale, gscale = w
        scale = scale.view(torch.uint8)[ids].view(scale.dtype)
        return _numbers(q[ids], scale, None if gscale is None else gscale[ids])
    return w[ids].float()


def _layer_plain(s):
    x, k = s["x"], s["k"]
    w, ids = _route_plain(x, s["gate"], k)
    e = s["gate"].shape[1]
    m = x.shape[0]
    xf = x.float()
    if m * k < e:           # few assignments: only their experts
        h = torch.einsum("nch,nh->nc", _pick(s["w1"], ids.flatten()), xf.repeat_interleave(k, 0))
        i = h.shape[1] // 2
        act = h[:, :i] * torch.sigmoid(h[:, :i]) * h[:, i:]
        y = torch.einsum("nhi,ni->nh", _pick(s["w2"], ids.flatten()), act).view(m, k, -1)
        out = (y * w.unsqueeze(-1)).sum(1)
    else:                   # every expert on every token, and the weights of the routing
        every = torch.arange(e, device=x.device)
        h = torch.matmul(xf.unsqueeze(0), _pick(s["w1"], every).transpose(1, 2))
        i = h.shape[2] // 2
        act = h[..., :i] * torch.sigmoid(h[..., :i]) * h[..., i:]
        dense = torch.zeros(m, e, device=x.device).scatter_(1, ids, w)
        out = (torch.matmul(act, _pick(s["w2"], every).transpose(1, 2)) * dense.t().unsqueeze(-1)).sum(0)
    return out.to(x.dtype), w, ids.to(torch.int32)


def run(s):
    if s["op"] == "quantise":
        if own:
            import fast_route_b200 as fr
            q, scale, gscale = fr.quantize_fp4(s["x"], block=s["block"])
            value = fr.dequantize_fp4(q, scale, gscale, dtype=s["x"].dtype)
            out = {"value": value, "scale": scale}
        else:
            value, scale, gscale = _quantise_plain(s["x"], s["block"])
            out = {"value": value, "scale": scale.to(torch.float8_e4m3fn if s["block"] == 16 else torch.float8_e8m0fnu)}
        if gscale is not None:
            out["global"] = gscale.reshape(())
        return out
    if s["op"] == "product":
        (aq, asc, ag), (bq, bsc, bg) = s["a"], s["b"]
        if own:
            import fast_route_b200 as fr
            return fr.matmul_fp4(aq, asc, bq, bsc, a_global=ag, b_global=bg, dtype=s["dtype"])
        return (_numbers(aq, asc, ag) @ _numbers(bq, bsc, bg).t()).to(s["dtype"])
    if own:
        import fast_route_b200 as fr
        if s["op"] == "decode":
            out, w, ids = fr.fused_moe_decode(s["x"], s["gate"], s["w1"], s["w2"], s["k"], return_routing=True)
        else:
            (q1, s1, g1), (q2, s2, g2) = s["w1"], s["w2"]
            out, w, ids = fr.fused_moe_decode_fp4(s["x"], s["gate"], q1, s1, q2, s2, s["k"], w1_global=g1, w2_global=g2,
                                                  return_routing=True)
    else:
        out, w, ids = _layer_plain(s)
    return {"out": out, "weights": w, "ids": ids}


# ----------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ----------------------------------------------------------------------------------------------------
def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    op = case["op"]
    if op == "quantise":        # numbers in, codes and scales out; codes and scales in, numbers out
        n = case["rows"] * case["cols"]
        return {"bytes": 2.0 * n * size + 2.0 * n * (0.5 + 1.0 / case["block"]), "flops": 4.0 * n}
    if op == "product":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": (m + n) * k * (0.5 + 1.0 / case["block"]) + 2.0 * m * n, "flops": 2.0 * m * n * k}
    m, h, i, e, k = (case[c] for c in ("m", "h", "i", "e", "k"))
    active = e * (1.0 - (1.0 - k / e) ** m)         # expected number of different experts, even routing
    weight = 2.0 if op == "decode" else 0.5 + 1.0 / case["block"]
    return {"bytes": active * 3.0 * h * i * weight + 2.0 * h * e + 4.0 * m * h + 8.0 * m * k,
            "flops": 6.0 * m * k * h * i + 2.0 * m * h * e}


# ----------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ----------------------------------------------------------------------------------------------------
def _exact_values(nib):
    """E2M1 from its fields: sign, two bits of exponent (bias 1, zero: no implied one), one bit of fraction."""
    nib = nib.long()
    exp, frac = (nib >> 1) & 3, (nib & 1).double()
    mag = torch.where(exp == 0, frac * 0.5, torch.ldexp(1.0 + 0.5 * frac, exp - 1))
    return torch.where(nib >= 8, -mag, mag)


def _exact_scale(scale):
    """E4M3 and E8M0 from their fields."""
    b = scale.view(torch.uint8).long()
    if scale.dtype == torch.float8_e4m3fn:
        exp, frac = (b >> 3) & 15, (b & 7).double() / 8.0
        return torch.where(exp == 0, torch.ldexp(frac, torch.full_like(exp, -6)), torch.ldexp(1.0 + frac, exp - 7))
    return torch.ldexp(torch.ones(b.shape, dtype=torch.float64, device=b.device), b - 127)


def _exact_matrix(q, scale, gscale):
    rows, half = q.shape
    out = torch.empty(rows, 2 * half, dtype=torch.float64, device=q.device)
    out[:, 0::2] = _exact_values(q & 15)
    out[:, 1::2] = _exact_values(q >> 4)
    block = 2 * half // scale.shape[1]
    out *= _exact_scale(scale).repeat_interleave(block, 1)
    return out if gscale is None else out * gscale.double()


def _single(v):
    """A 64-bit number rounded to the nearest fp32, where the definition holds a value in fp32."""
    return v.float().double()


def _exact_quantise(x, block):
    rows = x.shape[0]
    xd = x.double().reshape(rows, -1, block)
    amax = xd.abs().max(-1).values
    if block == 16:
        top = amax.max()
        g = _single(top / 2688.0).clamp_min(2.0 ** -110) if float(top) > 0 else torch.ones_like(top)
        t = _single(amax / _single(6.0 * g)).clamp_max(448.0)
        exp = (torch.frexp(t).exponent - 1).clamp_min(-6)                # 3 bits of fraction below the leading one
        step = torch.ldexp(torch.ones_like(t), exp - 3)
        s = torch.round(t / step) * step
        unit = _single(s * g)
        inv = torch.where(unit > 0, _single(1.0 / unit.clamp_min(1e-300)), torch.zeros_like(unit))
    else:
        g = None
        exp = (torch.frexp(amax).exponent - 1 - 2).clamp_min(-127)
        exp = torch.where(amax > 0, exp, torch.full_like(exp, -127))
        s = unit = torch.ldexp(torch.ones_like(amax), exp)
        inv = 1.0 / unit
    r = _single(xd * inv.unsqueeze(-1))
    mag = r.abs().clamp_max(6.0)
    exp = (torch.frexp(mag).exponent - 1).clamp_min(0)                   # one bit of fraction below the leading one
    step = torch.ldexp(torch.ones_like(mag), exp - 1)
    v = (torch.round(mag / step) * step).copysign(r) * unit.unsqueeze(-1)
    return {"value": v.reshape(rows, -1), "scale": s, **({} if g is None else {"global": g.reshape(())})}


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "quantise":
        return _exact_quantise(s["x"], s["block"])
    if s["op"] == "product":
        a, b = _exact_matrix(*s["a"]), _exact_matrix(*s["b"])
        return a @ b.t()
    x, k = s["x"].double(), s["k"]
    m = x.shape[0]
    logits = x @ s["gate"].double()
    ids = torch.argsort(logits, dim=1, descending=True, stable=True)[:, :k]
    w = torch.softmax(logits.gather(1, ids), dim=1)
    out = torch.zeros_like(x)
    for e in sorted(set(ids.flatten().tolist())):
        t, j = (ids == e).nonzero(as_tuple=True)
        if s["op"] == "decode":
            w1, w2 = s["w1"][e].double(), s["w2"][e].double()
        else:
            w1 = _exact_matrix(*[None if p is None else p[e] for p in s["w1"]])
            w2 = _exact_matrix(*[None if p is None else p[e] for p in s["w2"]])
        h = x[t] @ w1.t()
        i = h.shape[1] // 2
        act = h[:, :i] / (1.0 + torch.exp(-h[:, :i])) * h[:, i:]
        out[t] += w[t, j].unsqueeze(1) * (act @ w2.t())
    return {"out": out, "weights": w, "ids": None}
