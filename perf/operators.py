"""Serving with a quantised state, as cases that can be timed and compared.

Kinds of case:

* rows     New rows of a prompt or a turn written into the arena held in 4 bits, and the rows read back
           for the prefix attention (FullRelation.forward with such an arena): cache4_write, cache4_read.
* decode   One decode step of one Relation layer over the arena held in 4 bits: RoPE and Givens of the new
           chunk, the softmax read of every past row, the append: relation_decode4.
* linear   A projection in 8-bit integers with a scale per token and per output channel: int8_linear.

4 bits: groups of 32 head dims share a bf16 scale s = bf16(max|x| / 6); a value is its e2m1 code (0, 0.5, 1,
1.5, 2, 3, 4, 6 and a sign; nearest to x (1 / s) in 32 bits, ties to the even code) times s. Two codes a byte,
the even dim in the low half; a row's codes are padded to whole groups.
8 bits: scale = max|x| / 127 in 32 bits, code = round(x (127 / max|x|)), ties to even.

`own` false: the operators from elementary torch operations. Heads and widths are those of the presets this
repository is measured on (192 x 4 heads, 768 x 8) and the generic head dim 128 (1024 x 8).
"""

from __future__ import annotations

import math

import torch

own = False

GROUP = 32
TINY = 2.0 ** -126   # a 4-bit group whose scale is below stores zeros
SMALL = 2.0 ** -120  # an 8-bit row whose largest magnitude is below stores zeros
TAU = 2.0
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ---- the cases -----------------------------------------------------------------------------------
def _rows(name, B, H, D, n, T, dtype="bf16", ragged=False):
    c = dict(kind="rows", B=B, H=H, D=D, n=n, T=T, dtype=dtype, ragged=ragged)
    return dict(c, name=name) if name else c


def _decode(name, B, H, D, S, dtype="bf16", ragged=False, odd=False):
    c = dict(kind="decode", B=B, H=H, D=D, S=S, dtype=dtype, ragged=ragged, odd=odd)
    return dict(c, name=name) if name else c


def _linear(name, M, K, N, dtype="bf16"):
    c = dict(kind="linear", M=M, K=K, N=N, dtype=dtype)
    return dict(c, name=name) if name else c


def listed():
    return [
        # a 1 KB turn after 4096 cached chunks, one conversation
        _rows("rows_turn_b1", 1, 8, 96, 4096, 311),
        # the prompts of eight conversations, padded to the longest, read in one go
        _rows("rows_prompt_b8", 8, 8, 96, 0, 4984, ragged=True),
        # the smallest preset in full precision, sixteen conversations at positions of their own
        _rows("rows_fp32_b16", 16, 4, 48, 1000, 241, "fp32", ragged=True),
        # the first chunks of one conversation on the smallest preset in full precision: latency
        _decode("decode_start_fp32", 1, 4, 48, 37, "fp32"),
        # the decode engine's step, one conversation
        _decode("decode_b1", 1, 8, 96, 4096),
        # the decode engine's step, sixteen conversations of about 16 KB
        _decode("decode_b16", 16, 8, 96, 4700, ragged=True, odd=True),
        # sixteen long conversations, head dim 128: the largest sweep
        _decode("decode_long_b16", 16, 8, 128, 32768, ragged=True),
        # the stacked projection of one token
        _linear("linear_token", 1, 768, 2304),
        # the output projection of sixteen sequences' tokens
        _linear("linear_b16", 16, 768, 768),
        # the stacked projection of one 16 KB window
        _linear("linear_prompt", 4964, 768, 2304),
        # full precision at widths that no tile divides
        _linear("linear_odd_fp32", 1000, 520, 271, "fp32"),
        # a large batch of prompts through a wide layer: the largest product
        _linear("linear_large", 65536, 1024, 4096),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["rows", "decode", "decode", "linear", "linear"])
    dtype = "fp32" if rng.random() < 0.25 else "bf16"
    if kind == "rows":
        H, D = rng.choice([(4, 48), (8, 64), (8, 96), (8, 128), (4, 40), (6, 112)])
        B, T = _log(rng, 1, 16), _log(rng, 1, 5000)
        n = rng.choice([0, _log(rng, 1, 5000)])
        most = 8 * 5000 * 96 * 8 // (B * H * D)
        T = max(1, min(T, most))
        n = max(0, min(n, most - T))
        return _rows(None, B, H, D, n, T, dtype, ragged=rng.random() < 0.5)
    if kind == "decode":
        H, D = rng.choice([(4, 48), (8, 64), (8, 96), (8, 128), (4, 40), (6, 112)])
        B = _log(rng, 1, 32)
        S = min(_log(rng, 1, 32768), 16 * 32768 // B)
        return _decode(None, B, H, D, S, dtype, ragged=rng.random() < 0.5, odd=rng.random() < 0.5)
    M, K, N = _log(rng, 1, 65536), _log(rng, 64, 4096), _log(rng, 64, 4096)
    M = max(1, min(M, 65536 * 1024 * 4096 // (K * N)))
    if rng.random() < 0.5:  # widths of a model rather than any
        K, N = max(64, K // 64 * 64), max(64, N // 64 * 64)
    return _linear(None, M, K, N, dtype)


# ---- inputs ----------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, scale=1.0):
    return torch.randn(*shape, generator=g, device="cuda") * scale


def _channels(g, H, D):
    """Head dims of unlike size, as keys and values have them: most near 1, a few several times larger."""
    c = 0.5 + torch.rand(H, 1, D, generator=g, device="cuda")
    return c * torch.where(torch.rand(H, 1, D, generator=g, device="cuda") < 0.05, 4.0, 1.0)


def _held(g, B, H, rows, D, amp):
    """Random rows already held in 4 bits: (codes, scales), a sequence at a time."""
    codes, scales = [], []
    for _ in range(B):
        c, s = _pack(_randn(g, 1, H, rows, D) * amp)
        codes.append(c)
        scales.append(s)
    return torch.cat(codes), torch.cat(scales)


def prepare(case, seed):
    c, g = case, _gen(seed)
    T = DTYPES[c["dtype"]]
    if c["kind"] == "linear":
        M, K, N = c["M"], c["K"], c["N"]
        x = _randn(g, M, K)
        x *= torch.where(torch.rand(K, generator=g, device="cuda") < 0.01, 8.0, 1.0)  # a few large channels
        w = (torch.rand(N, K, generator=g, device="cuda") * 2 - 1) / math.sqrt(K)
        wq, ws = _quantise8(w)
        padded = torch.zeros(N, -(-K // 128) * 128, dtype=torch.int8, device="cuda")
        padded[:, :K] = wq.to(torch.int8)
        return dict(c=c, x=x.to(T), wq=padded, ws=ws)
    B, H, D = c["B"], c["H"], c["D"]
    rows = c["n"] + c["T"] if c["kind"] == "rows" else c["S"] + 1
    cap = -(-rows // 256) * 256
    amp, amp_i = _channels(g, H, D), _channels(g, H, D)
    k, ks = _held(g, B, H, cap, D, amp)
    v, vs = _held(g, B, H, cap, D, amp_i)
    st = dict(c=c, cache=(k, ks, v, vs))
    if c["kind"] == "rows":
        new = lambda a: (_randn(g, B, H, c["T"], D) * a).to(T).transpose(1, 2).contiguous().transpose(1, 2)  # noqa: E731
        st["p2"], st["info"] = new(amp), new(amp_i)
        st["start"], st["lens"] = c["n"], None
        if c["ragged"]:
            low = lambda most: torch.randint(most // 2, most + 1, (B,), generator=g, device="cuda")  # noqa: E731
            st["start"], st["lens"] = low(c["n"]), low(c["T"])
            st["lens"][0] = c["T"]
        return st
    st["qkv"] = (_randn(g, B, 3, H, D) * torch.stack([torch.ones_like(amp), amp, amp_i])[:, :, 0]).to(T)
    S = torch.full((B,), c["S"], device="cuda")
    if c["ragged"]:
        S = torch.randint(c["S"] // 2, c["S"] + 1, (B,), generator=g, device="cuda")
        S[0] = c["S"]
    st["S"] = S
    st["lam"] = torch.full((), 0.5, device="cuda")
    st["theta"] = torch.rand(H // 2, generator=g, device="cuda") * 0.6 - 0.3
    st["inv_freq"] = 1.0 / 10000.0 ** (torch.arange(0, D, 2, device="cuda").float() / D)
    return st


# ---- the plain forms -------------------------------------------------------------------------------
def _over(a, b):
    """a / b rounded once: by a scalar, a quotient of tensors is a product with its rounded inverse."""
    like = a if torch.is_tensor(a) else b
    return torch.div(*(t if torch.is_tensor(t) else torch.full_like(like, t) for t in (a, b)))


def _pack(x):
    """fp32 rows [..., D] -> (codes uint8 [..., 16 G], scales bf16 [..., G])."""
    D = x.shape[-1]
    G = -(-D // GROUP)
    x = torch.nn.functional.pad(x, (0, G * GROUP - D)).unflatten(-1, (G, GROUP))
    top = x.abs().amax(-1)
    s = _over(top, 6.0).to(torch.bfloat16)
    s = torch.where(s.float() < TINY, 0.0, s.float())
    inv = torch.where(s > 0, _over(1.0, s), 0.0)
    t = x * inv[..., None]
    a = t.abs()
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    code = (code + 8 * (t < 0)).flatten(-2).to(torch.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), s.to(torch.bfloat16)


def _unpack(codes, scales, D):
    """The fp32 values of 4-bit rows."""
    n = torch.arange(8, device=codes.device).float()
    table = torch.where(n < 4, n / 2, torch.where(n < 6, n - 2, 2 * n - 8))
    table = torch.cat([table, -table])
    both = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    v = table[both.int()].unflatten(-1, (scales.shape[-1], GROUP)) * scales.float()[..., None]
    return v.flatten(-2)[..., :D]


def _quantise8(x):
    """fp32 rows [M, K] -> (whole numbers in fp32 [M, K], scales fp32 [M])."""
    top = x.abs().amax(-1)
    fine = top >= SMALL
    inv = torch.where(fine, _over(127.0, top), 0.0)
    return torch.round(x * inv[:, None]), torch.where(fine, _over(top, 127.0), 0.0)


def _plain_rows(st):
    c, (k, ks, v, vs) = st["c"], st["cache"]
    T, D, new = DTYPES[c["dtype"]], c["D"], c["T"]
    B = c["B"]
    t = torch.arange(new, device="cuda")
    start = st["start"] if torch.is_tensor(st["start"]) else torch.full((B,), st["start"], device="cuda")
    lens = st["lens"] if st["lens"] is not None else torch.full((B,), new, device="cuda")
    b, row = torch.arange(B, device="cuda")[:, None], start[:, None] + t
    live = (t < lens[:, None])[..., None, None]
    for codes, scales, x in ((k, ks, st["p2"]), (v, vs, st["info"])):
        for held, fresh in zip((codes, scales), _pack(x.float())):
            held[b, :, row] = torch.where(live, fresh.transpose(1, 2), held[b, :, row])
    upto = c["n"] + new
    return [_unpack(codes[:, :, :upto], scales[:, :, :upto], D).to(T) for codes, scales in ((k, ks), (v, vs))]


def _plain_decode(st):
    c, (k, ks, v, vs) = st["c"], st["cache"]
    T, B, H, D = DTYPES[c["dtype"]], c["B"], c["H"], c["D"]
    S, half = st["S"], D // 2
    r = lambda x: x.to(T).float()  # noqa: E731  (a value of the step's type)
    ang = (S.float()[:, None] * st["inv_freq"]).double()
    cs, sn = r(ang.cos())[:, None], r(ang.sin())[:, None]
    x1, x2, xi = st["qkv"].float().unbind(1)
    rope = lambda x: torch.cat([r(r(x[..., :half] * cs) - r(x[..., half:] * sn)),  # noqa: E731
                                r(r(x[..., half:] * cs) + r(x[..., :half] * sn))], -1)
    q, kn = rope(x1), rope(x2)
    first = torch.arange(int(c["odd"]), H, 2, device="cuda")
    second = (first + 1) % H
    gc, gs = r(st["theta"].double().cos())[:, None], r(st["theta"].double().sin())[:, None]
    inew = torch.empty_like(xi)
    inew[:, first] = r(r(gc * xi[:, first]) - r(gs * xi[:, second]))
    inew[:, second] = r(r(gs * xi[:, first]) + r(gc * xi[:, second]))
    past = torch.arange(c["S"], device="cuda")[None, None] < S[:, None, None]
    u = (_unpack(k[:, :, : c["S"]], ks[:, :, : c["S"]], D) * q[:, :, None]).sum(-1) / math.sqrt(D)
    e = torch.where(past, u / (1.0 + torch.exp(-u)), -math.inf)
    top = e.amax(-1, keepdim=True).clamp(min=-1e30)
    p = torch.exp(e - top)
    l = p.sum(-1, keepdim=True)  # noqa: E741
    ibar = (_unpack(v[:, :, : c["S"]], vs[:, :, : c["S"]], D) * p[..., None]).sum(-2) / l.clamp(min=1e-30)
    lse = top[..., 0] + torch.log(l[..., 0])
    own_score = torch.sigmoid((q * kn).sum(-1) / math.sqrt(D) / TAU)
    g = torch.sigmoid(lse - st["lam"] * torch.log(S.float() + 1.0)[:, None] - own_score)
    y = (1.0 - g)[..., None] * inew + g[..., None] * ibar
    b = torch.arange(B, device="cuda")
    rows = []
    for codes, scales, x in ((k, ks, kn), (v, vs, inew)):
        xc, xs = _pack(x)
        codes[b, :, S], scales[b, :, S] = xc, xs
        rows.append(_unpack(xc, xs, D).to(T)[:, :, None])
    return [y.to(T), g, *rows]


def _plain_linear(st):
    c = st["c"]
    q, s = _quantise8(st["x"].float())
    acc = torch.matmul(q, st["wq"][:, : c["K"]].float().t())
    return (acc * s[:, None] * st["ws"]).to(DTYPES[c["dtype"]])


def run(state):
    st, c = state, state["c"]
    if not own:
        return {"rows": _plain_rows, "decode": _plain_decode, "linear": _plain_linear}[c["kind"]](st)
    if c["kind"] == "linear":
        from mote_amd.int8 import Int8Weight, int8_linear

        return int8_linear(st["x"], Int8Weight(st["wq"], st["ws"], c["K"]))
    from mote_amd.cache4 import Cache4, cache4_read, cache4_write, decode4_workspace, relation_decode4

    cache, T = Cache4(*st["cache"]), DTYPES[c["dtype"]]
    if c["kind"] == "rows":
        cache4_write(cache, st["p2"], st["info"], st["start"], st["lens"])
        return list(cache4_read(cache, c["D"], 0, c["n"] + c["T"], dtype=T))
    if "workspace" not in st:  # kept by the decode step between its calls
        st["workspace"] = decode4_workspace(c["B"], c["H"], c["D"], cache.p2.shape[2], "cuda")
    p1, p2, info = st["qkv"].unbind(1)
    y, g = relation_decode4(p1, p2, info, st["S"], cache, st["lam"], TAU, st["inv_freq"], st["theta"], int(c["odd"]),
                            workspace=st["workspace"])
    return [y, g, *cache4_read(cache, c["D"], st["S"], 1, dtype=T)]


# ---- the work of a pass ------------------------------------------------------------------------------
def work(case):
    c = case
    e = 4 if c["dtype"] == "fp32" else 2
    if c["kind"] == "linear":
        M, K, N = c["M"], c["K"], c["N"]
        return {"bytes": M * K * e + N * K + 4 * N + M * N * e, "flops": 2 * M * N * K}
    B, H, D = c["B"], c["H"], c["D"]
    row = D // 2 + 2 * -(-D // GROUP)  # bytes of a row in 4 bits
    if c["kind"] == "rows":
        # the new rows read, their codes written, every row's codes read and its values written
        new, upto = (0.75 * c["T"] if c["ragged"] else c["T"]), c["n"] + c["T"]
        return {"bytes": 2 * B * H * (new * (D * e + row) + upto * (row + D * e)), "flops": 2 * B * H * D * (new + upto)}
    S = 0.75 * c["S"] if c["ragged"] else c["S"]
    # every past row's codes read; the new chunk read, its rows written and read back, y written
    return {"bytes": 2 * B * H * S * row + B * H * (6 * D * e + 4 * row + 4), "flops": 4 * B * H * S * D}


# ---- the definitions in 64 bits ------------------------------------------------------------------------
def _f32(x):
    """A 64-bit value rounded to 32 bits."""
    return x.float().double()


def _round4(x):
    """The values that fp64 rows [..., D] have in 4 bits (32-bit rounding points as the format defines them)."""
    out = torch.zeros_like(x)
    for d in range(0, x.shape[-1], GROUP):
        part = x[..., d: d + GROUP]
        s = _f32(part.abs().amax(-1, keepdim=True) / 6.0).float().bfloat16().double()
        s = torch.where(s < TINY, torch.zeros_like(s), s)
        inv = _f32(1.0 / s.clamp(min=TINY))
        t = _f32(part * inv)
        a = t.abs().clamp(max=6.0)
        step = torch.where(a < 2.0, 0.5, torch.where(a < 4.0, 1.0, 2.0))
        out[..., d: d + GROUP] = torch.sign(t) * torch.round(a / step) * step * s
    return out


def _values(codes, scales, D):
    """fp64 values of rows held in 4 bits, from the meaning of sign, exponent and mantissa bits."""
    nib = torch.empty(*codes.shape[:-1], 2 * codes.shape[-1], dtype=torch.int64, device=codes.device)
    nib[..., 0::2], nib[..., 1::2] = codes % 16, codes // 16
    sign, ex, man = 1.0 - 2.0 * (nib // 8), (nib // 2) % 4, (nib % 2).double()
    mag = torch.where(ex == 0, 0.5 * man, (1.0 + 0.5 * man) * 2.0 ** (ex - 1).double())
    return (sign * mag * scales.double().repeat_interleave(GROUP, -1))[..., :D]


def exact(case, seed):
    st = prepare(case, seed)
    c = case
    T = DTYPES[c["dtype"]]
    if c["kind"] == "linear":
        x = st["x"].double()
        top = x.abs().max(1).values
        ok = top >= SMALL
        q = torch.round(_f32(x * torch.where(ok, _f32(127.0 / top), 0.0)[:, None]))
        out = q @ st["wq"][:, : c["K"]].double().t()
        out *= torch.where(ok, _f32(top / 127.0), 0.0)[:, None]
        out *= st["ws"].double()
        return out
    k, ks, v, vs = st["cache"]
    B, H, D = c["B"], c["H"], c["D"]
    if c["kind"] == "rows":
        upto, outs = c["n"] + c["T"], []
        for codes, scales, new in ((k, ks, st["p2"]), (v, vs, st["info"])):
            out = torch.empty(B, H, upto, D, dtype=torch.float64, device="cuda")
            for b in range(B):
                out[b] = _values(codes[b, :, :upto], scales[b, :, :upto], D)
                n = int(st["start"][b]) if c["ragged"] else c["n"]
                m = int(st["lens"][b]) if c["ragged"] else c["T"]
                out[b, :, n: n + m] = _round4(new[b, :, :m].double())
            outs.append(out)
        return outs
    y, g = torch.empty(B, H, D, dtype=torch.float64, device="cuda"), torch.empty(B, H, dtype=torch.float64, device="cuda")
    kr, vr = torch.empty(B, H, 1, D, dtype=torch.float64, device="cuda"), torch.empty(B, H, 1, D, dtype=torch.float64, device="cuda")
    to_t = lambda x: x.float().to(T).double()  # noqa: E731  (the step's type: its tables, products and sums round to it)
    for b in range(B):
        n = int(st["S"][b])
        angle = _f32(float(n) * st["inv_freq"].double())
        co, si = to_t(torch.cos(angle)).repeat(2), to_t(torch.sin(angle)).repeat(2)
        turn = lambda x: to_t(to_t(x * co) + to_t(torch.cat([-x[:, D // 2:], x[:, : D // 2]], 1) * si))  # noqa: E731
        q, kn, raw = turn(st["qkv"][b, 0].double()), turn(st["qkv"][b, 1].double()), st["qkv"][b, 2].double()
        new = raw.clone()
        for p in range(H // 2):
            i, j = 2 * p + int(c["odd"]), (2 * p + 1 + int(c["odd"])) % H
            co_g, si_g = (to_t(f(st["theta"][p].double())) for f in (torch.cos, torch.sin))
            new[i] = to_t(to_t(co_g * raw[i]) - to_t(si_g * raw[j]))
            new[j] = to_t(to_t(si_g * raw[i]) + to_t(co_g * raw[j]))
        u = (_values(k[b, :, :n], ks[b, :, :n], D) * q[:, None]).sum(-1) / math.sqrt(D)
        e = u * torch.sigmoid(u)
        lse = torch.logsumexp(e, -1)
        mean = (torch.exp(e - lse[:, None])[..., None] * _values(v[b, :, :n], vs[b, :, :n], D)).sum(1)
        mine = torch.sigmoid((q * kn).sum(-1) / math.sqrt(D) / TAU)
        gate = torch.sigmoid(lse - st["lam"].double() * math.log(n + 1.0) - mine)
        g[b] = gate
        y[b] = (1.0 - gate[:, None]) * new + gate[:, None] * mean
        kr[b, :, 0], vr[b, :, 0] = _round4(kn), _round4(new)
    return [y, g, kr, vr]
