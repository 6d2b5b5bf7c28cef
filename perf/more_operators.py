"""Serving many conversations from a paged cache in 8 bits, as cases that can be timed and compared.

Kinds of case:

* rows     New rows of a prompt or a turn appended to the paged cache, and the rows read back for the prefix
           attention (FullRelation.forward with such an arena): cache8_write, cache8_read.
* decode   One decode step of one Relation layer over the paged cache: RoPE and Givens of the new chunk, the
           softmax read of every past row, the append: relation_decode8.
* fork     A prompt continued in several sequences: their old pages released, the prompt's pages shared, its newest
           rows copied, pages for the rows to come: pages_free, pages_fork, pages_reserve.
* compact  The pages in use moved into another pool, front to back: pages_compact.
* sample   The next token of every sequence from its logits and a random number: sample_tokens.

8 bits: the 64 rows of a block of one head share a scale s = max|x| / 448 in 32 bits; a value is the e4m3 code of
x (448 / max|x|) (32 bits, nearest, ties to even) times s in 32 bits. Only whole blocks are held in 8 bits, one a
page; a sequence's newest rows, fewer than 64, are held as they are. In a page of P2 the bytes lie [D / 16][64
rows][16 dims], in one of I~ [D dims][64 rows]; D is padded to a multiple of 16.

Sampling: w = exp((x - max) / T); tokens in the order of their logits, ties to the lowest index; kept are the first
k, of these the shortest run of at least p of their weight, and those with w >= min_p; the token is the first whose
running weight exceeds u times the weight kept. T = 0 takes the first.

`own` false: the operators from elementary torch operations. Heads and widths are those of the presets this
repository is measured on (192 x 4 heads, 768 x 8) and the generic head dim 128 (1024 x 8); vocabularies the
byte vocabulary of 271 ids and generic ones.
"""

from __future__ import annotations

import math

import torch

own = False

PAGE = 64
TOP = 448.0           # the largest e4m3 value
SMALL = 2.0 ** -112   # a block whose largest magnitude is below stores zeros
TAU = 2.0
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ---- the cases -----------------------------------------------------------------------------------
def _rows(name, B, H, D, n, T, dtype="bf16", ragged=False):
    c = dict(kind="rows", B=B, H=H, D=D, n=n, T=T, dtype=dtype, ragged=ragged)
    return dict(c, name=name) if name else c


def _decode(name, B, H, D, S, dtype="bf16", ragged=False, odd=False):
    c = dict(kind="decode", B=B, H=H, D=D, S=S, dtype=dtype, ragged=ragged, odd=odd)
    return dict(c, name=name) if name else c


def _fork(name, layers, B, H, D, S, more, dtype="bf16"):
    c = dict(kind="fork", layers=layers, B=B, H=H, D=D, S=S, more=more, dtype=dtype)
    return dict(c, name=name) if name else c


def _compact(name, layers, B, H, D, pages, live):
    c = dict(kind="compact", layers=layers, B=B, H=H, D=D, pages=pages, live=live)
    return dict(c, name=name) if name else c


def _sample(name, B, V, dtype="fp32", T=1.0, k=0, p=1.0, m=0.0, mixed=False):
    c = dict(kind="sample", B=B, V=V, dtype=dtype, T=T, k=k, p=p, m=m, mixed=mixed)
    return dict(c, name=name) if name else c


def listed():
    return [
        # a 1 KB turn after 4096 cached chunks, one conversation
        _rows("rows_turn_b1", 1, 8, 96, 4096, 311),
        # the prompts of eight conversations, padded to the longest
        _rows("rows_prompt_b8", 8, 8, 96, 0, 4984, ragged=True),
        # the first chunks of one conversation on the smallest preset in full precision: latency
        _decode("decode_start_fp32", 1, 4, 48, 101, "fp32"),
        # the decode engine's step, sixteen conversations of about 16 KB
        _decode("decode_b16", 16, 8, 96, 4700, ragged=True, odd=True),
        # sixteen long conversations, head dim 128: the largest sweep
        _decode("decode_long_b16", 16, 8, 128, 32768, ragged=True),
        # two continuations of a short prompt on a small preset, in full precision: latency
        _fork("fork_small_fp32", 4, 3, 4, 48, 150, 100, "fp32"),
        # one prompt continued fifteen times, twelve layers
        _fork("fork_prompt_b16", 12, 16, 8, 96, 4133, 512),
        # the pool of a small preset's engine after half of its conversations have ended
        _compact("compact_small", 4, 8, 4, 48, 300, 0.5),
        # the same of sixteen conversations and twelve layers
        _compact("compact_b16", 12, 16, 8, 96, 1200, 0.6),
        # the next byte of one conversation
        _sample("sample_byte_b1", 1, 271, T=0.8, p=0.95),
        # the next byte of many, each with settings of its own
        _sample("sample_byte_b256", 256, 271, "bf16", mixed=True),
        # a large vocabulary and a batch
        _sample("sample_large", 64, 131072, "fp32", T=0.9, k=2000, p=0.95, m=0.0001),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["rows", "decode", "decode", "fork", "compact", "sample", "sample"])
    dtype = "fp32" if rng.random() < 0.3 else "bf16"
    H, D = rng.choice([(4, 48), (8, 64), (8, 96), (8, 128), (4, 40), (6, 112)])
    if kind == "rows":
        B, T = _log(rng, 1, 16), _log(rng, 1, 5000)
        n = rng.choice([0, _log(rng, 1, 5000)])
        most = 8 * 5000 * 96 * 8 // (B * H * D)
        T = max(1, min(T, most))
        n = max(0, min(n, most - T))
        n = n if n % PAGE + T <= PAGE else n // PAGE * PAGE  # see prepare
        return _rows(None, B, H, D, n, T, dtype, ragged=rng.random() < 0.5)
    if kind == "decode":
        B = _log(rng, 1, 32)
        S = min(_log(rng, 1, 32768), 16 * 32768 // B)
        return _decode(None, B, H, D, S, dtype, ragged=rng.random() < 0.5, odd=rng.random() < 0.5)
    if kind == "fork":
        return _fork(None, _log(rng, 1, 12), _log(rng, 2, 16), H, D, _log(rng, 1, 4200), _log(rng, 1, 600), dtype)
    if kind == "compact":
        layers, B = _log(rng, 1, 12), _log(rng, 1, 16)
        most = 12 * 1200 * 8 * 96 // (layers * H * D)
        return _compact(None, layers, B, H, D, min(_log(rng, 8, 1200), most), rng.uniform(0.1, 1.0))
    V = _log(rng, 64, 131072)
    B = min(_log(rng, 1, 256), 64 * 131072 // V)
    if rng.random() < 0.4:
        return _sample(None, B, V, dtype, mixed=True)
    k = rng.choice([0, _log(rng, 1, V)])
    return _sample(None, B, V, dtype, T=rng.choice([0.0, rng.uniform(0.3, 1.5), 1.0]), k=k,
                   p=rng.choice([1.0, rng.uniform(0.5, 0.999)]), m=rng.choice([0.0, rng.uniform(0.0, 0.1)]))


# ---- inputs ----------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, scale=1.0):
    return torch.randn(*shape, generator=g, device="cuda") * scale


def _channels(g, H, D):
    """Head dims of unlike size, as keys and values have them: most near 1, a few several times larger."""
    c = 0.5 + torch.rand(H, 1, D, generator=g, device="cuda")
    return c * torch.where(torch.rand(H, 1, D, generator=g, device="cuda") < 0.05, 4.0, 1.0)


def _tables(g, needs, width, pages):
    """A page of its own for each of needs[b] blocks of sequence b, in no order; none (-1) behind them."""
    order = torch.randperm(pages, generator=g, device="cuda").int()
    table = torch.full((len(needs), width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(needs):
        table[b, :n] = order[at: at + n]
        at += n
    return table


def _cache(g, c, needs, width, amp, amp_i):
    """A pool whose pages all hold rows, the newest rows of every sequence, and the page table."""
    B, H, D, T = c["B"], c["H"], c["D"], DTYPES[c["dtype"]]
    pages = sum(needs) + 5
    parts = ([], [], [], [])
    for at in range(0, pages, 256):
        n = min(256, pages - at)
        for i, (a, pack) in enumerate(((amp, _pack_p2), (amp_i, _pack_info))):
            codes, scales = pack(_randn(g, n, H, PAGE, D) * a)
            parts[2 * i].append(codes)
            parts[2 * i + 1].append(scales)
    tails = [(_randn(g, B, H, PAGE, D) * a).to(T) for a in (amp, amp_i)]
    return (*(torch.cat(p) for p in parts), *tails, _tables(g, needs, width, pages))


def prepare(case, seed):
    c, g = case, _gen(seed)
    kind = c["kind"]
    if kind == "sample":
        B, V, T = c["B"], c["V"], DTYPES[c["dtype"]]
        st = dict(c=c, logits=(_randn(g, B, V) * 2.5).to(T), u=torch.rand(B, generator=g, device="cuda"))
        if c["mixed"]:
            one = lambda: torch.rand(B, generator=g, device="cuda")  # noqa: E731
            some = lambda x, off: torch.where(one() < 0.6, x, torch.full_like(x, off))  # noqa: E731
            st["set"] = (torch.where(one() < 0.1, 0.0, 0.3 + 1.2 * one()), some(1 + (one() ** 3 * V).long(), 0),
                         some(0.5 + 0.5 * one(), 1.0), some(0.1 * one(), 0.0))
        else:
            st["set"] = (c["T"], c["k"], c["p"], c["m"])
        return st
    B, H, D = c["B"], c["H"], c["D"]
    wide = -(-D // 16) * 16
    if kind == "compact":
        P, planes = c["pages"], 2 * c["layers"]
        codes = torch.randint(0, 127, (planes, P, H * wide * PAGE), generator=g, device="cuda", dtype=torch.uint8)
        scales = torch.rand(planes, P, H, generator=g, device="cuda")
        live = max(1, int(P * c["live"]))
        needs = [live // B + (b < live % B) for b in range(B)]
        table = _tables(g, needs, max(needs) + 3, P)
        if B > 1 and needs[1] > 1:  # a prompt that two conversations share
            table[1, : needs[1] // 2] = table[0, : needs[1] // 2]
        refs = torch.bincount(table[table >= 0].long(), minlength=P).int()
        new = live + 7
        into = (torch.zeros(planes, new, H * wide * PAGE, dtype=torch.uint8, device="cuda"),
                torch.zeros(planes, new, H, device="cuda"), torch.zeros(new, dtype=torch.int32, device="cuda"))
        return dict(c=c, pool=(codes, scales, refs), table=table, into=into)
    if kind == "fork":
        T, planes = DTYPES[c["dtype"]], 2 * c["layers"]
        S = torch.randint(1, c["S"] + 1, (B,), generator=g, device="cuda")
        S[0] = c["S"]
        width = (c["S"] + c["more"]) // PAGE + 2
        needs = [n // PAGE for n in S.tolist()]
        P = B * width + 11
        table = _tables(g, needs, width, P)
        refs = torch.bincount(table[table >= 0].long(), minlength=P).int()
        tails = _randn(g, planes, B, H, PAGE, D).to(T)
        return dict(c=c, S=S, table=table, refs=refs, tails=tails, dst=list(range(1, B)))
    amp, amp_i = _channels(g, H, D), _channels(g, H, D)
    low = lambda most: torch.randint(most // 2, most + 1, (B,), generator=g, device="cuda")  # noqa: E731
    T = DTYPES[c["dtype"]]
    if kind == "rows":
        # the old rows end with a block or the new ones stay within theirs: a pass that closes a block that was
        # begun before replaces the newest rows that it has read, and could not be repeated on the same state
        st = dict(c=c, start=c["n"], lens=None)
        if c["ragged"]:
            st["start"], st["lens"] = low(c["n"]) // PAGE * PAGE, low(c["T"])
            st["lens"][0] = c["T"]
        start = st["start"] if c["ragged"] else torch.full((B,), c["n"], device="cuda")
        st["held"] = start + (st["lens"] if c["ragged"] else c["T"])
        width = (c["n"] + c["T"]) // PAGE + 1
        st["cache"] = _cache(g, c, [n // PAGE for n in st["held"].tolist()], width, amp, amp_i)
        new = lambda a: (_randn(g, B, H, c["T"], D) * a).to(T).transpose(1, 2).contiguous().transpose(1, 2)  # noqa: E731
        st["p2"], st["info"] = new(amp), new(amp_i)
        return st
    S = torch.full((B,), c["S"], device="cuda")
    if c["ragged"]:
        S = low(c["S"])
        S[0] = c["S"]
    width = -(-(c["S"] + 1) // (4 * PAGE)) * 4  # the table reaches to a multiple of 256 rows
    st = dict(c=c, S=S, held=S + 1, cache=_cache(g, c, [(n + 1) // PAGE for n in S.tolist()], width, amp, amp_i))
    st["qkv"] = (_randn(g, B, 3, H, D) * torch.stack([torch.ones_like(amp), amp, amp_i])[:, :, 0]).to(T)
    st["lam"] = torch.full((), 0.5, device="cuda")
    st["theta"] = torch.rand(H // 2, generator=g, device="cuda") * 0.6 - 0.3
    st["inv_freq"] = 1.0 / 10000.0 ** (torch.arange(0, D, 2, device="cuda").float() / D)
    return st


# ---- the plain forms -------------------------------------------------------------------------------
def _over(a, b):
    """a / b rounded once: by a scalar, a quotient of tensors is a product with its rounded inverse."""
    like = a if torch.is_tensor(a) else b
    return torch.div(*(t if torch.is_tensor(t) else torch.full_like(like, t) for t in (a, b)))


def _block8(x):
    """fp32 blocks [..., 64, D] -> (codes uint8 [..., 64, D padded to 16], scales fp32 [...])."""
    D = x.shape[-1]
    top = x.abs().amax((-1, -2))
    fine = top >= SMALL
    s = torch.where(fine, _over(top, TOP), 0.0)
    t = x * torch.where(fine, _over(TOP, top), 0.0)[..., None, None]
    t = torch.nn.functional.pad(t, (0, -D % 16))
    return t.to(torch.float8_e4m3fn).view(torch.uint8), s


def _pack_p2(x):
    codes, s = _block8(x)
    return codes.unflatten(-1, (-1, 16)).transpose(-2, -3).contiguous(), s


def _pack_info(x):
    codes, s = _block8(x)
    return codes.transpose(-1, -2).contiguous(), s


def _unpack_p2(codes, s, D):
    """The fp32 values [..., 64, D] of pages of P2."""
    x = codes.transpose(-2, -3).flatten(-2)[..., :D].contiguous()
    return x.view(torch.float8_e4m3fn).float() * s[..., None, None]


def _unpack_info(codes, s, D):
    x = codes.transpose(-1, -2)[..., :D].contiguous()
    return x.view(torch.float8_e4m3fn).float() * s[..., None, None]


def _blocks(cache, D, n):
    """fp32 values of the first n blocks of every sequence, [B, H, n * 64, D] each."""
    k, ks, v, vs, _, _, table = cache
    at = table[:, :n].clamp(min=0).long()
    out = []
    for codes, s, unpack in ((k, ks, _unpack_p2), (v, vs, _unpack_info)):
        x = unpack(codes[at], s[at], D)  # [B, n, H, 64, D]
        out.append(x.transpose(1, 2).flatten(2, 3))
    return out


def _held_rows(cache, D, held, rows, T):
    """Rows [0, rows) of every sequence in T; zeros from row held[b] on."""
    pos = torch.arange(rows, device="cuda")
    whole = held // PAGE * PAGE
    outs = []
    for x, tail in zip(_blocks(cache, D, -(-rows // PAGE)), cache[4:6]):
        new = tail.float()[:, :, pos % PAGE]
        x = torch.nn.functional.pad(x, (0, 0, 0, max(0, rows - x.shape[2])))[:, :, :rows]
        x = torch.where((pos < whole[:, None])[:, None, :, None], x, new)
        outs.append(torch.where((pos < held[:, None])[:, None, :, None], x, 0.0).to(T))
    return outs


def _plain_rows(st):
    c, cache = st["c"], st["cache"]
    T, B, D, new = DTYPES[c["dtype"]], c["B"], c["D"], c["T"]
    k, ks, v, vs, kt, vt, table = cache
    start = st["start"] if torch.is_tensor(st["start"]) else torch.full((B,), st["start"], device="cuda")
    held = st["held"]
    # the rows of the blocks that the new ones touch: the newest old ones, then the new ones
    blocks = (new + PAGE - 1) // PAGE + 1
    pos = (start // PAGE * PAGE)[:, None] + torch.arange(blocks * PAGE, device="cuda")
    fresh = (pos >= start[:, None]) & (pos < held[:, None])
    b = torch.arange(B, device="cuda")[:, None]
    block = pos[:, ::PAGE] // PAGE
    done = (block + 1) * PAGE <= held[:, None]
    whole = done & (block < table.shape[1])
    at = table[b, torch.where(whole, block, 0)].long()
    for codes, scales, tail, x, pack in ((k, ks, kt, st["p2"], _pack_p2), (v, vs, vt, st["info"], _pack_info)):
        rows = torch.where(fresh[..., None, None], x.transpose(1, 2)[b, (pos - start[:, None]).clamp(0, new - 1)],
                           tail.transpose(1, 2)[b, pos % PAGE])  # [B, blocks * 64, H, D]
        rows = rows.unflatten(1, (blocks, PAGE)).transpose(2, 3)  # [B, blocks, H, 64, D]
        packed, s = pack(rows.float())
        codes[at[whole]] = packed[whole]
        scales[at[whole]] = s[whole]
        last = (held // PAGE - start // PAGE).clamp(max=blocks - 1)
        open_ = rows[torch.arange(B, device="cuda"), last]
        keep = (torch.arange(PAGE, device="cuda") < (held % PAGE)[:, None])[:, None, :, None]
        tail.copy_(torch.where(keep, open_, tail))
    return _held_rows(cache, D, held, c["n"] + new, T)


def _plain_decode(st):
    c, cache = st["c"], st["cache"]
    T, B, H, D = DTYPES[c["dtype"]], c["B"], c["H"], c["D"]
    S, half = st["S"], D // 2
    k, ks, v, vs, kt, vt, table = cache
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
    n = c["S"] // PAGE
    keys, values = _blocks(cache, D, n)
    keys, values = torch.cat([keys, kt.float()], 2), torch.cat([values, vt.float()], 2)
    pos = torch.arange((n + 1) * PAGE, device="cuda")
    past = torch.where(pos < n * PAGE, pos < (S // PAGE * PAGE)[:, None], pos - n * PAGE < (S % PAGE)[:, None])[:, None]
    u = (keys * q[:, :, None]).sum(-1) / math.sqrt(D)
    e = torch.where(past, u / (1.0 + torch.exp(-u)), -math.inf)
    top = e.amax(-1, keepdim=True).clamp(min=-1e30)
    p = torch.exp(e - top)
    l = p.sum(-1, keepdim=True)  # noqa: E741
    ibar = (values * p[..., None]).sum(-2) / l.clamp(min=1e-30)
    lse = top[..., 0] + torch.log(l[..., 0])
    own_score = torch.sigmoid((q * kn).sum(-1) / math.sqrt(D) / TAU)
    g = torch.sigmoid(lse - st["lam"] * torch.log(S.float() + 1.0)[:, None] - own_score)
    y = (1.0 - g)[..., None] * inew + g[..., None] * ibar
    b = torch.arange(B, device="cuda")
    block = S // PAGE
    whole = (S % PAGE == PAGE - 1)
    at = table[b, block].long()[whole]
    outs = []
    for codes, scales, tail, x, pack, unpack in ((k, ks, kt, kn, _pack_p2, _unpack_p2), (v, vs, vt, inew, _pack_info, _unpack_info)):
        tail[b, :, S % PAGE] = x.to(T)
        packed, s = pack(tail.float())
        codes[at], scales[at] = packed[whole], s[whole]
        row = torch.where(whole[:, None, None], unpack(packed, s, D)[b, :, S % PAGE], x)
        outs.append(row.to(T)[:, :, None])
    return [y.to(T), g, *outs]


def _plain_fork(st):
    c, S, table, refs, tails = st["c"], st["S"], st["table"], st["refs"], st["tails"]
    dst = torch.tensor(st["dst"], device="cuda")
    width, P = table.shape[1], refs.shape[0]
    block = torch.arange(width, device="cuda")
    table[dst] = torch.where(block < S[0] // PAGE, table[:1], -1).clone()
    S[dst] = S[0].clone()
    keep = (torch.arange(PAGE, device="cuda") < S[0] % PAGE)[:, None]
    tails[:, dst] = torch.where(keep, tails[:, :1], tails[:, dst]).clone()
    need = (block < ((S + c["more"]) // PAGE)[:, None]) & (table < 0)
    held = torch.zeros(P + 1, dtype=torch.int32, device="cuda")
    held.index_add_(0, torch.where(table < 0, P, table).long().flatten(), torch.ones_like(table).flatten())
    free = torch.nonzero(held[:P] == 0)[:, 0].int()
    rank = (need.flatten().cumsum(0) - 1).view_as(need)
    fits = need & (rank < free.shape[0])
    given = torch.where(fits, free[rank.clamp(0, free.shape[0] - 1)], table)
    table.copy_(given)
    held.zero_()
    held.index_add_(0, torch.where(table < 0, P, table).long().flatten(), torch.ones_like(table).flatten())
    refs.copy_(held[:P])
    return [table, refs, S, tails, (need & ~fits).sum().int().view(1)]


def _plain_compact(st):
    (codes, scales, refs), table, (codes2, scales2, refs2) = st["pool"], st["table"], st["into"]
    live = torch.nonzero(refs > 0)[:, 0]
    n = live.shape[0]
    codes2[:, :n] = codes[:, live]
    scales2[:, :n] = scales[:, live]
    refs2.zero_()
    refs2[:n] = refs[live]
    new = (refs > 0).int().cumsum(0).int() - 1
    moved = torch.where(table >= 0, new[table.clamp(min=0).long()], -1)
    return [moved, codes2, scales2, refs2, torch.zeros(1, dtype=torch.int32, device="cuda")]


def _plain_sample(st):
    x = st["logits"].double()
    B, V = x.shape
    col = lambda t, dt: (t if torch.is_tensor(t) else torch.full((B,), t, device="cuda")).to(dt)[:, None]  # noqa: E731
    f32 = lambda t: col(t, torch.float32).double()  # noqa: E731  (settings are 32-bit numbers)
    T, k, p, m = f32(st["set"][0]), col(st["set"][1], torch.int64), f32(st["set"][2]), f32(st["set"][3])
    xs, order = torch.sort(x, dim=-1, descending=True, stable=True)
    w = torch.exp((xs - xs[:, :1]) / torch.where(T > 0, T, 1.0))
    rank = torch.arange(V, device="cuda")
    w = torch.where((k <= 0) | (rank < k), w, 0.0)
    before = w.cumsum(-1) - w
    kept = (p >= 1.0) | (before < p * w.sum(-1, keepdim=True)) | (rank == 0)
    kept &= (w >= m) | (rank == 0)
    w = torch.where(kept, w, 0.0)
    run_ = w.cumsum(-1)
    at = (run_ <= st["u"].double()[:, None] * run_[:, -1:]).sum(-1).clamp(max=V - 1)
    at = torch.where(T[:, 0] > 0, at, 0)
    return order[torch.arange(B, device="cuda"), at]


def run(state):
    st, c = state, state["c"]
    kind = c["kind"]
    if not own:
        return {"rows": _plain_rows, "decode": _plain_decode, "fork": _plain_fork, "compact": _plain_compact,
                "sample": _plain_sample}[kind](st)
    if kind == "sample":
        from mote_amd.sample import sample_tokens

        T, k, p, m = st["set"]
        return sample_tokens(st["logits"], st["u"], temperature=T, top_k=k, top_p=p, min_p=m)
    if kind == "fork":
        from mote_amd.pages import pages_fork, pages_free, pages_reserve

        pages_free(st["refs"], st["table"], st["dst"])
        pages_fork(st["refs"], st["table"], st["S"], 0, st["dst"], st["tails"])
        missing = pages_reserve(st["refs"], st["table"], st["S"] + c["more"])
        return [st["table"], st["refs"], st["S"], st["tails"], missing]
    if kind == "compact":
        from mote_amd.pages import PagePool, pages_compact

        into = PagePool(*st["into"])
        table, missing = pages_compact(PagePool(*st["pool"]), st["table"], into)
        return [table, *into, missing]
    from mote_amd.cache8 import Cache8, cache8_read, cache8_write, decode8_workspace, relation_decode8

    cache, T = Cache8(*st["cache"]), DTYPES[c["dtype"]]
    if kind == "rows":
        cache8_write(cache, st["p2"], st["info"], st["start"], st["lens"])
        return list(cache8_read(cache, st["held"], 0, c["n"] + c["T"], dtype=T))
    if "workspace" not in st:  # kept by the decode step between its calls
        st["workspace"] = decode8_workspace(c["B"], c["H"], c["D"], PAGE * cache.table.shape[1], "cuda")
    p1, p2, info = st["qkv"].unbind(1)
    y, g = relation_decode8(p1, p2, info, st["S"], cache, st["lam"], TAU, st["inv_freq"], st["theta"], int(c["odd"]),
                            workspace=st["workspace"])
    return [y, g, *cache8_read(cache, st["held"], st["S"], 1, dtype=T)]


# ---- the work of a pass ------------------------------------------------------------------------------
def work(case):
    c = case
    e = 4 if c.get("dtype") == "fp32" else 2
    if c["kind"] == "sample":
        # every logit read; a difference, a scaling, an exponential and a sum each
        return {"bytes": c["B"] * (c["V"] * e + 12), "flops": 4 * c["B"] * c["V"]}
    B, H, D = c["B"], c["H"], c["D"]
    if c["kind"] == "fork":
        # the prompt's newest rows read once and written B - 1 times; the tables and counts
        width = (c["S"] + c["more"]) // PAGE + 2
        return {"bytes": 2 * c["layers"] * B * H * (c["S"] % PAGE) * D * e + 16 * B * width, "flops": B * width}
    if c["kind"] == "compact":
        live = max(1, int(c["pages"] * c["live"]))
        if B > 1:
            live -= (live // B + (1 < live % B)) // 2
        return {"bytes": 4 * c["layers"] * live * H * (PAGE * D + 4) + 8 * c["pages"], "flops": c["pages"]}
    if c["kind"] == "rows":
        # the new rows read, their codes written, every row's codes read and its values written
        new, upto = (0.75 * c["T"] if c["ragged"] else c["T"]), c["n"] + c["T"]
        return {"bytes": 2 * B * H * D * (new * (e + 1) + upto * (1 + e)), "flops": 2 * B * H * D * (new + upto)}
    S = 0.75 * c["S"] if c["ragged"] else c["S"]
    tail = min(S, PAGE // 2)
    # every past row read; the new chunk read, its rows written and read back, y written
    return {"bytes": 2 * B * H * ((S - tail) * D + tail * D * e) + B * H * (10 * D * e + 4), "flops": 4 * B * H * S * D}


# ---- the definitions in 64 bits ------------------------------------------------------------------------
def _f32(x):
    """A 64-bit value rounded to 32 bits."""
    return x.float().double()


def _round8(x):
    """The values that fp64 blocks [..., 64, D] have in 8 bits (32-bit rounding points as the format defines them)."""
    top = x.abs().flatten(-2).max(-1).values[..., None, None]
    ok = top >= SMALL
    t = _f32(x * torch.where(ok, _f32(TOP / top), 0.0))
    a = t.abs()
    step = 2.0 ** (torch.floor(torch.log2(a.clamp(min=2.0 ** -6))) - 3.0)  # three bits behind the leading one
    return _f32(torch.sign(t) * torch.round(a / step) * step * torch.where(ok, _f32(top / TOP), 0.0))


def _bytes8(codes):
    """fp64 values of e4m3 bytes, from the meaning of sign, exponent and mantissa bits."""
    n = torch.arange(256, device="cuda")
    ex, man = (n // 8) % 16, (n % 8).double()
    mag = torch.where(ex == 0, man * 2.0 ** -9, (1.0 + man / 8.0) * 2.0 ** (ex - 7).double())
    return (torch.where(n < 128, mag, -mag))[codes.int()]


def _row(cache, b, pos, which, D):
    """fp64 rows at whole-block positions pos [n] of sequence b, [H, n, D]: single bytes looked up in their pages."""
    codes, s, table = cache[2 * which], cache[2 * which + 1], cache[6]
    page, r = table[b, pos // PAGE].long(), pos % PAGE
    d = torch.arange(D, device="cuda")
    if which == 0:
        x = codes[page[:, None], :, d // 16, r[:, None], d % 16]  # [n, D, H]
    else:
        x = codes[page[:, None], :, d, r[:, None]]
    return _f32(_bytes8(x).permute(2, 0, 1) * s[page].double().t()[:, :, None])


def _exact_decode(st, c):
    cache = st["cache"]
    B, H, D, T = c["B"], c["H"], c["D"], DTYPES[c["dtype"]]
    new = lambda *s: torch.empty(*s, dtype=torch.float64, device="cuda")  # noqa: E731
    y, g, kr, vr = new(B, H, D), new(B, H), new(B, H, 1, D), new(B, H, 1, D)
    to_t = lambda x: x.float().to(T).double()  # noqa: E731  (the step's type: its tables, products and sums round to it)
    for b in range(B):
        n = int(st["S"][b])
        angle = _f32(float(n) * st["inv_freq"].double())
        co, si = to_t(torch.cos(angle)).repeat(2), to_t(torch.sin(angle)).repeat(2)
        turn = lambda x: to_t(to_t(x * co) + to_t(torch.cat([-x[:, D // 2:], x[:, : D // 2]], 1) * si))  # noqa: E731
        q, kn, raw = turn(st["qkv"][b, 0].double()), turn(st["qkv"][b, 1].double()), st["qkv"][b, 2].double()
        fresh = raw.clone()
        for p in range(H // 2):
            i, j = 2 * p + int(c["odd"]), (2 * p + 1 + int(c["odd"])) % H
            co_g, si_g = (to_t(f(st["theta"][p].double())) for f in (torch.cos, torch.sin))
            fresh[i] = to_t(to_t(co_g * raw[i]) - to_t(si_g * raw[j]))
            fresh[j] = to_t(to_t(si_g * raw[i]) + to_t(co_g * raw[j]))
        whole, rest = n // PAGE * PAGE, n % PAGE
        scores, rows = [], []
        for at in range(0, whole, 4096):
            pos = torch.arange(at, min(whole, at + 4096), device="cuda")
            scores.append((_row(cache, b, pos, 0, D) * q[:, None]).sum(-1))
            rows.append(pos)
        scores.append((cache[4][b, :, :rest].double() * q[:, None]).sum(-1))
        u = torch.cat(scores, 1) / math.sqrt(D)
        e = u * torch.sigmoid(u)
        lse = torch.logsumexp(e, -1)
        share = torch.exp(e - lse[:, None]) if n else e
        mean = (share[:, whole:, None] * cache[5][b, :, :rest].double()).sum(1)
        for pos in rows:
            mean += (share[:, pos, None] * _row(cache, b, pos, 1, D)).sum(1)
        mine = torch.sigmoid((q * kn).sum(-1) / math.sqrt(D) / TAU)
        gate = torch.sigmoid(lse - st["lam"].double() * math.log(n + 1.0) - mine)
        g[b] = gate
        y[b] = (1.0 - gate[:, None]) * fresh + gate[:, None] * mean
        for out, row, tail in ((kr, kn, cache[4]), (vr, fresh, cache[5])):
            out[b, :, 0] = row
            if rest == PAGE - 1:
                out[b, :, 0] = _round8(torch.cat([tail[b, :, :rest].double(), row[:, None]], 1))[:, -1]
    return [y, g, kr, vr]


def _exact_rows(st, c):
    cache, D, outs = st["cache"], c["D"], []
    for which, x in enumerate((st["p2"], st["info"])):
        out = torch.zeros(c["B"], c["H"], c["n"] + c["T"], D, dtype=torch.float64, device="cuda")
        for b in range(c["B"]):
            n, end = (int(st["start"][b]) if c["ragged"] else c["n"]), int(st["held"][b])
            whole = n // PAGE * PAGE
            out[b, :, :whole] = _row(cache, b, torch.arange(whole, device="cuda"), which, D)
            out[b, :, whole:n] = cache[4 + which][b, :, : n - whole].double()
            out[b, :, n:end] = x[b, :, : end - n].double()
            last = end // PAGE * PAGE
            if last > whole:
                out[b, :, whole:last] = _round8(out[b, :, whole:last].unflatten(1, (-1, PAGE))).flatten(1, 2)
        outs.append(out)
    return outs


def _exact_fork(st, c):
    table, S, P = st["table"].tolist(), st["S"].tolist(), st["refs"].shape[0]
    tails = st["tails"].double()
    for b in st["dst"]:
        table[b] = [t if j < S[0] // PAGE else -1 for j, t in enumerate(table[0])]
        S[b] = S[0]
        tails[:, b, :, : S[0] % PAGE] = tails[:, 0, :, : S[0] % PAGE]
    used, missing = {t for row in table for t in row if t >= 0}, 0
    free = iter([p for p in range(P) if p not in used])
    for b, row in enumerate(table):
        for j in range((S[b] + c["more"]) // PAGE):
            if row[j] < 0:
                row[j] = next(free, -1)
                missing += row[j] < 0
    refs = [0] * P
    for row in table:
        for t in row:
            if t >= 0:
                refs[t] += 1
    whole = lambda x: torch.tensor(x, device="cuda")  # noqa: E731
    return [whole(table).int(), whole(refs).int(), whole(S), tails, whole([missing]).int()]


def _exact_compact(st):
    (codes, scales, refs), (codes2, scales2, refs2) = st["pool"], st["into"]
    names, count = {}, refs.tolist()
    for p, n in enumerate(count):
        if n > 0:
            names[p] = len(names)
    counts = [0] * refs2.shape[0]
    for p, i in names.items():
        counts[i] = count[p]
        codes2[:, i].copy_(codes[:, p])
        scales2[:, i].copy_(scales[:, p])
    table = [[names[t] if t >= 0 else -1 for t in row] for row in st["table"].tolist()]
    return [torch.tensor(table, device="cuda").int(), codes2, scales2.double(), torch.tensor(counts, device="cuda").int(),
            torch.zeros(1, dtype=torch.int32, device="cuda")]


def _exact_sample(st):
    import numpy as np

    x, u = st["logits"].double().cpu().numpy(), st["u"].double().cpu().numpy()
    B, V = x.shape
    single = lambda t: np.broadcast_to(np.asarray(t.cpu() if torch.is_tensor(t) else t, dtype=np.float32), (B,))  # noqa: E731
    T, p, m = (single(st["set"][i]).astype(np.float64) for i in (0, 2, 3))
    k = st["set"][1].tolist() if torch.is_tensor(st["set"][1]) else [st["set"][1]] * B
    tokens = []
    for b in range(B):
        order = np.lexsort((np.arange(V), -x[b]))
        if T[b] <= 0:
            tokens.append(int(order[0]))
            continue
        order = order[: k[b]] if 0 < k[b] < V else order
        w = np.exp(((x[b][order] - x[b].max()) / T[b]).astype(np.longdouble))
        total = np.cumsum(w)
        kept = len(w)
        if p[b] < 1.0:
            kept = int(np.searchsorted(total, p[b] * total[-1], side="left")) + 1
        kept = max(1, min(kept, int((w >= m[b]).sum())))
        at = int(np.searchsorted(total[:kept], u[b] * total[kept - 1], side="right"))
        tokens.append(int(order[min(at, kept - 1)]))
    return torch.tensor(tokens, device="cuda")


def exact(case, seed):
    st, c = prepare(case, seed), case
    if c["kind"] == "sample":
        return _exact_sample(st)
    if c["kind"] == "fork":
        return _exact_fork(st, c)
    if c["kind"] == "compact":
        return _exact_compact(st)
    return _exact_rows(st, c) if c["kind"] == "rows" else _exact_decode(st, c)
