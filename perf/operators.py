"""The 4-bit decode operators on real work: what each reads and computes, in plain torch and through the package.

Three operators of the low-bit decode path of a StripedHyena2 target (``evspark_b200.q4``):

* ``linear``: tokens times a weight held in 4 bits with one scale per group of input features;
* ``append``: new keys and values rotated to their positions and put into a paged 4-bit cache, the
  queries rotated alongside; the appended span is read back as the values that the cache holds;
* ``attend``: attention of the new tokens over the paged 4-bit cache, causal, with shared key/value
  heads and rows of different lengths.

The 4-bit format: groups of 32 (cache: along head_dim) or 32, 64 or 128 (weights: along the input
features) values share a scale; a code c in 1..15 stands for (c - 8) * scale.  The scale is
absmax / 7 rounded to five significant bits, so that every (c - 8) * scale is exact in bf16.
A group whose absmax / 7 is below 2^-120 is held as zeros, one with a NaN, an infinity or
absmax / 7 above 2^120 as NaN.

Weight: codes uint8 [N, Kp / 2], two per byte, even feature in the low half, K padded with code 8 to
Kp = a multiple of 128; scales bf16 [Kp / group, N].  Cache: pool uint8 [pages, kv_heads, block], a
block holding P tokens of one head: K codes [P, Dh / 2], V codes [P, Dh / 2], K scales
[Dh / 32, P], V scales [Dh / 32, P] (bf16); page_table int32 [B, max_pages], lengths int32 [B] (the
tokens before this call), counts int32 [B] (new tokens of each row, the rest of T is padding).
"""

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
ROPE_BASE = 10000.0


def listed():
    return [
        # one native decode step through an out-projection of the 7B shape: the call is a few microseconds long
        dict(name="linear_step_out_7b", op="linear", M=1, N=4096, K=4096, group=128, dtype="bf16"),
        # a 13-token verify block through both MLP input projections of the 7B shape
        dict(name="linear_verify_mlp_in_7b", op="linear", M=13, N=22016, K=4096, group=64, dtype="bf16"),
        # a 13-token verify block through the MLP out-projection of the 40B shape: the longest sums
        dict(name="linear_verify_mlp_out_40b", op="linear", M=13, N=8192, K=22528, group=128, dtype="bf16"),
        # an fp32 model with odd sizes: padded columns, ragged row tiles, the smallest groups
        dict(name="linear_odd_fp32", op="linear", M=7, N=1003, K=717, group=32, dtype="fp32"),
        # one verify block's keys and values of the 7B shape
        dict(name="append_verify_7b", op="append", B=1, T=13, H=32, G=32, D=128, page=64, longest=1023, ragged=False, dtype="bf16"),
        # prompt chunks of eight streams of different lengths
        dict(name="append_prompts_7b", op="append", B=8, T=1024, H=32, G=32, D=128, page=64, longest=8192, ragged=True, dtype="bf16"),
        # shared heads, small pages and far positions, in fp32
        dict(name="append_grouped_fp32", op="append", B=5, T=37, H=12, G=4, D=64, page=16, longest=262144, ragged=True, dtype="fp32"),
        # one native decode step at a 1k context of the 7B shape
        dict(name="attend_step_1k_7b", op="attend", B=1, T=1, H=32, G=32, D=128, page=64, longest=1023, ragged=False, dtype="bf16"),
        # verify blocks of the 7B shape at 64k and 262k contexts
        dict(name="attend_verify_64k_7b", op="attend", B=1, T=13, H=32, G=32, D=128, page=64, longest=65536, ragged=False, dtype="bf16"),
        dict(name="attend_verify_262k_7b", op="attend", B=1, T=13, H=32, G=32, D=128, page=64, longest=262131, ragged=False, dtype="bf16"),
        # sixteen streams of different lengths, eight query heads to a key/value head
        dict(name="attend_streams_grouped", op="attend", B=16, T=13, H=64, G=8, D=128, page=32, longest=16384, ragged=True, dtype="bf16"),
        # an fp32 model with an odd head group and pages that end inside a tile
        dict(name="attend_odd_fp32", op="attend", B=3, T=5, H=6, G=2, D=64, page=16, longest=777, ragged=True, dtype="fp32"),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["linear", "append", "attend"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    if op == "linear":
        while True:
            case = dict(op=op, M=_spread(rng, 1, 64), N=_spread(rng, 64, 22016), K=_spread(rng, 64, 22528),
                        group=rng.choice([32, 64, 128]), dtype=dtype)
            if case["N"] * case["K"] <= 8192 * 22528 and case["M"] * case["N"] * case["K"] <= 13 * 8192 * 22528:
                return case
    shape = dict(D=rng.choice([32, 64, 128]), G=rng.choice([1, 2, 3, 4, 8, 16, 32]), page=rng.choice([16, 32, 64, 128]),
                 ragged=rng.random() < 0.6, dtype=dtype)
    shape["H"] = shape["G"] * rng.choice([1, 1, 2, 4, 5, 8])
    while True:
        case = dict(op=op, B=_spread(rng, 1, 16), T=_spread(rng, 1, 1024 if op == "append" else 16),
                    longest=_spread(rng, 1, 262131), **shape)
        pairs = case["B"] * case["longest"] * case["G"] * case["D"]
        if op == "append" and case["B"] * case["T"] * case["H"] * case["D"] <= 8 * 1024 * 32 * 128 and pairs <= 2 ** 29:
            return case
        if op == "attend" and pairs <= 2 ** 29 and pairs * case["T"] * (case["H"] // case["G"]) <= 2 ** 33:
            return case


def _round5(t):
    """t rounded to five significant bits (nearest, ties to even); t in 64 bits, not negative."""
    mantissa, exponent = torch.frexp(t)
    return torch.ldexp(torch.round(mantissa * 32.0) / 32.0, exponent)


def _quantize(x, group):
    """x [..., n] in 64 bits, n a multiple of group -> (codes uint8 [..., n], scales bf16 [..., n / group])."""
    g = x.unflatten(-1, (-1, group))
    t = g.abs().amax(-1) / 7.0
    s = torch.where(t < 2.0 ** -120, torch.zeros_like(t), _round5(t))
    s = torch.where(torch.isfinite(t) & (t <= 2.0 ** 120), s, torch.full_like(t, math.nan))
    held = torch.isfinite(s) & (s > 0)
    c = torch.round(g / torch.where(held, s, torch.ones_like(s))[..., None]).clamp(-7.0, 7.0)
    c = torch.where(held[..., None], c, torch.zeros_like(c)) + 8.0
    return c.flatten(-2).to(torch.uint8), s.to(torch.bfloat16)


def _pack(codes):
    pair = codes.unflatten(-1, (-1, 2))
    return pair[..., 0] | (pair[..., 1] << 4)


def _unpack(packed):
    """uint8 [..., n / 2] -> codes less 8, in fp32 [..., n]."""
    return torch.stack([packed & 15, packed >> 4], -1).flatten(-2).to(torch.float32) - 8.0


def _fields(pool, D, page):
    """Views of a pool's K codes, V codes [pages, heads, P, D / 2] and K scales, V scales [pages, heads, D / 32, P]."""
    n, f = page * D // 2, page * D // 16
    k, v = (pool[..., i * n:(i + 1) * n].unflatten(-1, (page, D // 2)) for i in (0, 1))
    ks, vs = (pool[..., 2 * n + i * f:2 * n + (i + 1) * f].view(torch.bfloat16).unflatten(-1, (D // 32, page)) for i in (0, 1))
    return k, v, ks, vs


def _block_bytes(D, page):
    return page * D + page * D // 8


def _pages_of(case, gen, device):
    """lengths, counts and a page table of scattered pages (-1 where a row has none), with the number of pages."""
    B, T, page = case["B"], case["T"], case["page"]
    longest = case["longest"]
    if case["ragged"]:
        lengths = (torch.rand(B, generator=gen, device=device) * longest).to(torch.int32)
        lengths[0] = longest
        counts = 1 + (torch.rand(B, generator=gen, device=device) * T).to(torch.int32).clamp(max=T - 1)
        counts[-1] = T
    else:
        lengths = torch.full((B,), longest, dtype=torch.int32, device=device)
        counts = torch.full((B,), T, dtype=torch.int32, device=device)
    most = (longest + T + page - 1) // page
    used = (lengths + counts + page - 1) // page
    held = torch.arange(most, device=device)[None, :] < used[:, None]
    total = int(held.sum())
    table = torch.full((B, most), -1, dtype=torch.int32, device=device)
    table[held] = torch.randperm(total, generator=gen, device=device).to(torch.int32)
    return lengths, counts, table, total


def prepare(case, seed):
    device = torch.device("cuda")
    gen = torch.Generator(device=device)
    gen.manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]
    if case["op"] == "linear":
        M, N, K, group = case["M"], case["N"], case["K"], case["group"]
        x = torch.randn(M, K, generator=gen, device=device).to(dtype)
        padded = -(-K // 128) * 128
        codes = torch.empty(N, padded // 2, dtype=torch.uint8, device=device)
        scales = torch.empty(padded // group, N, dtype=torch.bfloat16, device=device)
        for n0 in range(0, N, 1024):  # a slab at a time: the 64-bit copy of a whole weight would not be small
            w = torch.zeros(min(1024, N - n0), padded, dtype=torch.float64, device=device)
            w[:, :K] = torch.randn(w.shape[0], K, generator=gen, device=device) * K ** -0.5
            c, s = _quantize(w, group)
            codes[n0:n0 + w.shape[0]] = _pack(c)
            scales[:, n0:n0 + w.shape[0]] = s.t()
        state = dict(case, x=x, codes=codes, scales=scales)
        if own:
            from evspark_b200 import q4
            state["weight"] = q4.Q4Weight(codes, scales, (N, K), group)
        return state
    B, T, H, G, D, page = (case[n] for n in ("B", "T", "H", "G", "D", "page"))
    lengths, counts, table, total = _pages_of(case, gen, device)
    pool = torch.full((total, G, _block_bytes(D, page)), 0x88, dtype=torch.uint8, device=device)
    state = dict(case, lengths=lengths, counts=counts, table=table, pool=pool)
    if case["op"] == "append":
        # q, k and v as slices of one projection's output, as a fused projection leaves them
        qkv = torch.randn(B, T, (H + 2 * G) * D, generator=gen, device=device).to(dtype)
        state["q"] = qkv[..., :H * D].unflatten(-1, (H, D))
        state["k"] = qkv[..., H * D:(H + G) * D].unflatten(-1, (G, D))
        state["v"] = qkv[..., (H + G) * D:].unflatten(-1, (G, D))
        state["q_out"] = torch.zeros(B, T, H, D, dtype=dtype, device=device)
        state["read"] = tuple(torch.zeros(B, T, G, D, dtype=torch.bfloat16, device=device) for _ in range(2))
    else:
        kc, vc, ks, vs = _fields(pool, D, page)
        rows = max(1, 2 ** 27 // (G * page * D))
        for p0 in range(0, total, rows):  # codes of normal values, a slab of pages at a time
            n = min(rows, total - p0)
            for field in (kc, vc):
                c = (torch.randn(n, G, page, D, generator=gen, device=device) * 2.6).round_().clamp_(-7, 7) + 8
                field[p0:p0 + n] = _pack(c.to(torch.uint8))
        for field in (ks, vs):
            t = torch.exp(torch.randn(field.shape, generator=gen, device=device) * 0.3) * 0.35
            field.copy_(_round5(t.double()).to(torch.bfloat16))
        state["q"] = (torch.randn(B, T, H, D, generator=gen, device=device) * 2.0).to(dtype)
        state["out"] = torch.zeros(B, T, H, D, dtype=dtype, device=device)
    if own:
        from evspark_b200 import q4
        state["cache"] = q4.Q4Cache.from_pool(pool, head_dim=D, page_size=page)
        state["max_length"] = case["longest"] + T
    return state


def _rotate(x, positions):
    """Rotate-half position rotation of x [B, T, heads, D], in 64 bits (the angles of far positions need them)."""
    half = x.shape[-1] // 2
    freq = ROPE_BASE ** (-torch.arange(half, dtype=torch.float64, device=x.device) / half)
    angle = positions.double()[..., None, None] * freq
    c, s = torch.cos(angle), torch.sin(angle)
    a, b = x[..., :half].double(), x[..., half:].double()
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def _plain_linear(st):
    w = (_unpack(st["codes"]).unflatten(-1, (-1, st["group"])) * st["scales"].t().float()[..., None]).flatten(-2)
    return st["x"].float() @ w[:, :st["K"]].t()


def _plain_append(st):
    B, T, D, page = st["B"], st["T"], st["D"], st["page"]
    steps = torch.arange(T, device=st["q"].device)
    positions = st["lengths"].long()[:, None] + steps
    live = steps[None, :] < st["counts"][:, None]
    b, t = live.nonzero(as_tuple=True)
    at = positions[b, t]
    ids, slot = st["table"][b, at // page].long(), at % page
    k, v = _rotate(st["k"], positions), st["v"].double()
    kc, vc, ks, vs = _fields(st["pool"], D, page)
    (k_codes, k_scales), (v_codes, v_scales) = _quantize(k[b, t], 32), _quantize(v[b, t], 32)
    kc[ids, :, slot], vc[ids, :, slot] = _pack(k_codes), _pack(v_codes)
    ks[ids, :, :, slot], vs[ids, :, :, slot] = k_scales, v_scales
    st["q_out"][b, t] = _rotate(st["q"], positions)[b, t].to(st["q"].dtype)
    k_out, v_out = st["read"]
    k_out[b, t] = (_unpack(kc[ids, :, slot]).unflatten(-1, (-1, 32)) * ks[ids, :, :, slot].float()[..., None]).flatten(-2).bfloat16()
    v_out[b, t] = (_unpack(vc[ids, :, slot]).unflatten(-1, (-1, 32)) * vs[ids, :, :, slot].float()[..., None]).flatten(-2).bfloat16()
    return {"q": st["q_out"], "k": k_out, "v": v_out}


def _rows_of(codes, scales, table):
    """A cache field as values [B, heads, keys, D] in fp32, page by page in each row's order."""
    ids = table.long().clamp(min=0)
    c = _unpack(codes[ids]).unflatten(-1, (-1, 32))  # [B, pages, heads, P, D / 32, 32]
    return (c * scales[ids].float().transpose(-1, -2)[..., None]).flatten(-2).transpose(1, 2).flatten(2, 3)


def _plain_attend(st):
    B, T, H, G, D, page = (st[n] for n in ("B", "T", "H", "G", "D", "page"))
    kc, vc, ks, vs = _fields(st["pool"], D, page)
    k = _rows_of(kc, ks, st["table"])
    q = st["q"].float().unflatten(2, (G, H // G)).permute(0, 2, 1, 3, 4).flatten(2, 3)  # [B, G, T * (H / G), D]
    s = (q @ k.transpose(-1, -2)) * D ** -0.5
    del k
    steps = torch.arange(T, device=q.device)
    last = (st["lengths"][:, None] + steps).repeat_interleave(H // G, 1)  # [B, T * (H / G)]
    seen = torch.arange(s.shape[-1], device=q.device) <= last[..., None]
    s = torch.where(seen[:, None], s, torch.full((), -math.inf, device=q.device))
    p = torch.exp(s - s.amax(-1, keepdim=True))
    del s
    total = p.sum(-1, keepdim=True)
    # keys behind a row's last token are not its own: their values stay out of the sums
    behind = torch.arange(p.shape[-1], device=q.device) >= (st["lengths"] + st["counts"])[:, None]
    v = _rows_of(vc, vs, st["table"]).masked_fill_(behind[:, None, :, None], 0.0)
    o = ((p @ v) / total).unflatten(2, (T, H // G)).permute(0, 2, 1, 3, 4).flatten(2, 3)
    live = (steps[None, :] < st["counts"][:, None])[..., None, None]
    st["out"].copy_(torch.where(live, o, torch.zeros_like(o)))
    return st["out"]


def run(state):
    if own:
        from evspark_b200 import q4
        if state["op"] == "linear":
            return q4.q4_linear(state["x"], state["weight"])
        cache, table, lengths, counts = state["cache"], state["table"], state["lengths"], state["counts"]
        if state["op"] == "append":
            q = q4.q4_kv_append(cache, table, lengths, state["k"], state["v"], q=state["q"], counts=counts,
                                rope_base=ROPE_BASE, q_out=state["q_out"])
            k, v = q4.q4_kv_read(cache, table, lengths, state["T"], counts=counts, out=state["read"])
            return {"q": q, "k": k, "v": v}
        return q4.q4_attention(state["q"], cache, table, lengths, counts=counts, max_length=state["max_length"],
                               out=state["out"])
    return {"linear": _plain_linear, "append": _plain_append, "attend": _plain_attend}[state["op"]](state)


def work(case):
    size = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        return {"bytes": N * K // 2 + 2 * N * -(-K // case["group"]) + size * M * K + 4 * M * N, "flops": 2 * M * N * K}
    B, T, H, G, D = (case[n] for n in ("B", "T", "H", "G", "D"))
    held = D // 2 + D // 16  # bytes of one token's key (or value) of one head
    share = 0.5 if case["ragged"] else 1.0  # the mean of the ragged lengths and counts
    if case["op"] == "append":
        tokens = B * T * share
        moved = size * (2 * H + 2 * G) * D + 2 * 2 * G * held + 2 * 2 * G * D
        return {"bytes": int(tokens * moved), "flops": int(tokens * (3 * (H + G) * D + 4 * G * D))}
    keys = B * (case["longest"] * share + T)
    return {"bytes": int(keys * 2 * G * held + 2 * size * B * T * H * D), "flops": int(4 * keys * T * share * H * D)}


def exact(case, seed):
    """The operators' definitions in 64 bits, row by row and head by head."""
    st = prepare(case, seed)
    f64 = torch.float64

    def values(packed, scales, group):
        low, high = (packed % 16).to(f64) - 8, (packed // 16).to(f64) - 8
        c = torch.empty(*packed.shape[:-1], 2 * packed.shape[-1], dtype=f64, device=packed.device)
        c[..., 0::2], c[..., 1::2] = low, high
        return c * scales.to(f64).repeat_interleave(group, -1)

    if case["op"] == "linear":
        y = torch.empty(case["M"], case["N"], dtype=f64, device=st["x"].device)
        x = st["x"].to(f64)
        for n0 in range(0, case["N"], 2048):
            w = values(st["codes"][n0:n0 + 2048], st["scales"][:, n0:n0 + 2048].t(), case["group"])
            y[:, n0:n0 + 2048] = x @ w[:, :case["K"]].t()
        return y
    B, T, H, G, D, page = (case[n] for n in ("B", "T", "H", "G", "D", "page"))
    lengths, counts = st["lengths"].tolist(), st["counts"].tolist()
    if case["op"] == "append":
        def turned(x, b):
            half = D // 2
            j = torch.arange(half, dtype=f64, device=x.device)
            angle = (lengths[b] + torch.arange(T, device=x.device)).to(f64)[:, None, None] * torch.exp(-j / half * math.log(ROPE_BASE))
            z = torch.complex(x[..., :half].to(f64), x[..., half:].to(f64)) * torch.polar(torch.ones_like(angle), angle)
            return torch.cat([z.real, z.imag], -1)

        def held(x):
            g = x.reshape(*x.shape[:-1], D // 32, 32)
            t = g.abs().amax(-1, keepdim=True) / 7
            unit = torch.exp2(torch.floor(torch.log2(t)) - 4)
            unit = torch.where(t >= 32 * unit, 2 * unit, unit)
            s = torch.round(t / unit) * unit
            return (torch.round(g / s).clamp(-7, 7) * s).reshape(x.shape)

        q, k, v = (torch.zeros(*st[n].shape, dtype=f64, device=st["q"].device) for n in ("q", "k", "v"))
        for b in range(B):
            n = counts[b]
            q[b, :n] = turned(st["q"][b], b)[:n]
            k[b, :n] = held(turned(st["k"][b], b))[:n]
            v[b, :n] = held(st["v"][b].to(f64))[:n]
        return {"q": q, "k": k, "v": v}
    n, f = page * D // 2, page * D // 16
    out = torch.zeros(B, T, H, D, dtype=f64, device=st["q"].device)
    for b in range(B):
        end = lengths[b] + counts[b]
        ids = st["table"][b, :-(-end // page)].long()
        for g in range(G):
            block = st["pool"][ids, g]

            def field(i):
                codes = block[:, i * n:(i + 1) * n].reshape(-1, D // 2)[:end]
                scales = block[:, 2 * n + i * f:2 * n + (i + 1) * f].contiguous().view(torch.bfloat16)
                return values(codes, scales.reshape(-1, D // 32, page).transpose(1, 2).reshape(-1, D // 32)[:end], 32)

            k, v = field(0), field(1)
            heads = slice(g * (H // G), (g + 1) * (H // G))
            q = st["q"][b, :counts[b], heads].to(f64)
            s = torch.einsum("thd,kd->thk", q, k) / math.sqrt(D)
            hidden = torch.arange(end, device=s.device)[None, :] > lengths[b] + torch.arange(counts[b], device=s.device)[:, None]
            s = s.masked_fill(hidden[:, None, :], -math.inf)
            out[b, :counts[b], heads] = torch.softmax(s, -1) @ v
    return out
