"""Measured cases of the key/value cache operators: the cache is written in 4 or 8 bits as tokens arrive
(`KVCachePlan.append`), read back as fp16 (`KVCachePlan.read`), and attended over where it lies
(`KVCachePlan.attention`), for single tokens, a few tokens and whole prompts.

With `own` false, `run` computes them in elementary torch operations in fp32 on the same buffers, rounded once
at the end; with `own` true it makes the calls a user of the package makes.

The cache is one uint8 buffer [pages][heads_kv][2: K, V][page_size][row]. A row holds one head's vector of one
token: head_dim codes (4 bits: element d in nibble d % 2 of byte d / 2, the low one first; 8 bits: byte d), then
for each 32 elements an fp16 scale and an fp16 zero. A code c stands for fp16(c * scale + zero).
"""
import math

import torch

own = False

GROUP = 32       # elements that share a scale and a zero
F16_MAX = 65504.0


def row_bytes(case):
    return case["head_dim"] * case["bits"] // 8 + case["head_dim"] // GROUP * 4


def sequences_of(case):
    """(lengths, new tokens) of each sequence, by the case alone. `ragged` r spreads the lengths evenly from
    (1 - r) * length to length, and the new tokens likewise in another order. Both count the new tokens."""
    B, r = case["sequences"], case["ragged"]
    lengths, new = [], []
    for b in range(B):
        n = max(1, int(case["new"] * (1 - r * ((5 * b + 2) % B) / B))) if B > 1 else case["new"]
        ln = max(1, int(case["length"] * (1 - r * b / B)))
        if case["op"] == "read":
            n = ln
        lengths.append(max(ln, n))
        new.append(n)
    return lengths, new


def listed():
    base = {"sequences": 1, "heads_q": 8, "heads_kv": 8, "head_dim": 128, "bits": 4, "page_size": 64, "new": 1,
            "length": 1, "ragged": 0.0, "causal": True, "packed": False, "lse": False}

    def case(name, op, **kw):
        return {"name": name, "op": op, **base, **kw}

    return [
        # Each of 16 running sequences writes the token it just produced; the values are read back for the
        # layers that want them in fp16. Latency only.
        case("write one token each", "write_read", sequences=16, heads_q=32, new=1, length=1000, ragged=0.5),
        # Four prompts of up to 4096 tokens, 16 heads of 128 (the framework's B4 H16 S4096 D128), written from
        # a fused Q/K/V projection's output, so K and V rows are strided.
        case("write prompts", "write_read", sequences=4, heads_q=16, heads_kv=16, new=4096, length=4096, ragged=0.25,
             packed=True),
        # Prompt chunks of odd lengths into an 8-bit cache of small heads, grouped 8 / 2, small pages.
        case("write chunks, 8 bits", "write_read", sequences=7, heads_kv=2, head_dim=64, bits=8, page_size=16, new=333,
             length=1023, ragged=0.6),
        # Eight long sequences read back whole, e.g. to hand them to a dense kernel or move them off the GPU.
        case("read long", "read", sequences=8, heads_q=32, length=8192, ragged=0.3),
        # A few short sequences read back from an 8-bit cache: latency.
        case("read short, 8 bits", "read", sequences=3, heads_kv=2, head_dim=64, bits=8, page_size=16, length=300,
             ragged=0.5),
        # One sequence of the reference driver's heads (8 / 8 of 128) produces one token: the smallest call.
        case("attend one token, one sequence", "attend", length=1023),
        # A full serving batch: 64 sequences, ragged lengths up to 8192, grouped 32 / 8.
        case("attend one token, batch", "attend", sequences=64, heads_q=32, length=8192, ragged=0.7),
        # Two very long contexts: few rows, so the key axis is split over the whole GPU and joined.
        case("attend one token, long", "attend", sequences=2, heads_q=32, length=131072, ragged=0.1),
        # One token over an 8-bit cache, ungrouped heads of 64, an odd number of sequences.
        case("attend one token, 8 bits", "attend", sequences=33, heads_q=8, heads_kv=8, head_dim=64, bits=8,
             page_size=32, length=3001, ragged=0.8),
        # Six proposed tokens per sequence are checked at once, causal among themselves, 16-token pages.
        case("attend a few tokens", "attend", sequences=16, heads_q=32, page_size=16, new=6, length=4500, ragged=0.5,
             lse=True),
        # Four whole prompts attend over themselves (B4 H16 S4096 D128, causal), Q strided as projected.
        case("attend prompts", "attend", sequences=4, heads_q=16, heads_kv=16, new=4096, length=4096, packed=True),
        # Prompt chunks on top of a long context, 8 bits, heads of 64 grouped 16 / 2, odd ragged lengths.
        case("attend chunks, 8 bits", "attend", sequences=3, heads_q=16, heads_kv=2, head_dim=64, bits=8, page_size=32,
             new=1000, length=12001, ragged=0.4, lse=True),
    ]


def draw(rng):
    def log_int(lo, hi):
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))

    while True:
        hq, hkv = rng.choice([(8, 8), (16, 16), (16, 4), (32, 8), (32, 4), (16, 2), (8, 1), (6, 2), (10, 5), (4, 4)])
        c = {"op": rng.choice(["write_read", "read", "attend", "attend", "attend", "attend"]),
             "sequences": log_int(1, 64), "heads_q": hq, "heads_kv": hkv, "head_dim": rng.choice([64, 128, 128]),
             "bits": rng.choice([4, 4, 8]), "page_size": rng.choice([16, 32, 64, 128, 256]), "new": 1,
             "length": log_int(1, 131072), "ragged": round(rng.uniform(0.0, 0.9), 2), "causal": rng.random() < 0.85,
             "packed": rng.random() < 0.4, "lse": False}
        if c["op"] == "write_read":
            c["new"] = log_int(1, 8192)
            c["length"] = max(c["new"], c["length"])
        elif c["op"] == "attend":
            c["new"] = rng.choice([1, 1, log_int(2, 16), log_int(17, 4096)])
            c["length"] = max(c["new"], c["length"])
            c["lse"] = rng.random() < 0.3
        w = work(c)
        rows = c["sequences"] * c["new"]
        cached = c["sequences"] * c["length"] * c["heads_kv"] * c["head_dim"]
        scores = rows * c["length"] * c["heads_q"] if c["op"] == "attend" else 0
        if cached <= 64 * 8192 * 8 * 128 and scores <= 4 * 4096 * 16 * 4096 and rows * c["heads_q"] <= 1 << 18 \
                and w["flops"] <= 2.8e11 and w["bytes"] <= 4.5e8 and not (c["op"] == "read" and w["bytes"] > 3.4e8):
            return c


def work(case):
    lengths, new = sequences_of(case)
    D, Hq, Hk = case["head_dim"], case["heads_q"], case["heads_kv"]
    pair = 2 * Hk * row_bytes(case)      # one token's K and V in the cache
    values = 2 * Hk * D * 2              # and as fp16
    if case["op"] == "write_read":
        return {"bytes": sum(new) * (values + pair + values), "flops": 0}
    if case["op"] == "read":
        return {"bytes": sum(lengths) * (pair + values), "flops": 0}
    if case["causal"]:
        pairs = sum(n * ln - n * (n - 1) // 2 for ln, n in zip(lengths, new))
    else:
        pairs = sum(n * ln for ln, n in zip(lengths, new))
    rows = sum(new) * Hq
    return {"bytes": sum(lengths) * pair + rows * (2 * D * 2 + (4 if case["lse"] else 0)), "flops": 4 * D * Hq * pairs}


# ----------------------------------------------------------------------------------------------------------
# inputs
# ----------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    D, Hq, Hk, bits, page = (case[k] for k in ("head_dim", "heads_q", "heads_kv", "bits", "page_size"))
    lengths, new = sequences_of(case)
    B, tokens = len(lengths), sum(new)
    per_seq = (max(lengths) + page - 1) // page
    used = [(ln + page - 1) // page for ln in lengths]
    pages = sum(used) + 3                # a pool with a little room, handed out in no order
    order = torch.randperm(pages, generator=gen, device=dev).to(torch.int32)
    table = torch.zeros(B, per_seq, dtype=torch.int32, device=dev)
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = order[at:at + n]
        at += n
    offsets = [0]
    for n in new:
        offsets.append(offsets[-1] + n)
    channel = torch.exp(0.5 * torch.randn(Hk, D, generator=gen, device=dev))  # some channels of K are large

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=dev)

    s = {"case": case, "table": table, "lengths": torch.tensor(lengths, dtype=torch.int32, device=dev),
         "offsets": torch.tensor(offsets, dtype=torch.int32, device=dev),
         "cache": torch.zeros(pages, Hk * 2 * page * row_bytes(case), dtype=torch.uint8, device=dev)}
    width = (Hq + 2 * Hk) * D + 64 if case["packed"] else 0  # a fused projection's row, padded by 128 bytes

    def rows(heads, first, scale):       # [tokens][heads][D], a slice of a fused projection where packed
        x = (normal(tokens, heads, D) * scale).half()
        if not width:
            return x
        whole = torch.zeros(tokens, width, dtype=torch.float16, device=dev)
        part = whole[:, first:first + heads * D]
        part.copy_(x.view(tokens, heads * D))
        return part.view(tokens, heads, D)

    if case["op"] == "write_read":
        s["K"], s["V"] = rows(Hk, Hq * D, channel), rows(Hk, (Hq + Hk) * D, 1.0)
    else:
        pool = s["cache"].view(pages, Hk, 2, page, row_bytes(case))
        step = max(1, (1 << 26) // (Hk * 2 * page * D))
        for p in range(0, pages, step):
            x = normal(min(step, pages - p), Hk, 2, page, D)
            x[:, :, 0] *= channel[None, :, None, :]
            pool[p:p + step] = pack(x.half(), bits)
    if case["op"] == "attend":
        s["Q"] = rows(Hq, 0, 1.0)
        s["lse"] = torch.empty(tokens, Hq, dtype=torch.float32, device=dev) if case["lse"] else None
    if own:
        from example_matmul_metal4_b200.kv_cache import KVCacheBatch, KVCacheDimensions, KVCachePlan
        s["plan"] = KVCachePlan(KVCacheDimensions(pages, page, Hq, Hk, D, bits), causal=case["causal"])
        s["batch"] = KVCacheBatch(table, s["lengths"], s["offsets"], tokens, max(new))
    return s


# ----------------------------------------------------------------------------------------------------------
# the plain form
# ----------------------------------------------------------------------------------------------------------

def pack(x, bits):
    """fp16 [..., D] as cache rows, uint8 [..., row]: per group of 32 the zero is the smallest value and the scale
    fp16((largest - smallest) / (2^bits - 1)) rounded towards zero, so no code's value leaves fp16's range; NaN
    counts as 0 and infinities as the largest finite value."""
    top = (1 << bits) - 1
    g = torch.nan_to_num(x.float(), nan=0.0, posinf=F16_MAX, neginf=-F16_MAX).unflatten(-1, (-1, GROUP))
    low = g.amin(-1, keepdim=True)
    step = (g.amax(-1, keepdim=True) - low) / top
    near = step.half()
    scale = torch.where(near.float() > step, (near.view(torch.int16) - 1).view(torch.float16), near)
    s = scale.float()
    codes = torch.where(s > 0, torch.round((g - low) / s).clamp(max=top), torch.zeros_like(g))
    codes = codes.to(torch.uint8).flatten(-2)
    if bits == 4:
        codes = codes[..., 0::2] | (codes[..., 1::2] << 4)
    params = torch.cat([scale, low.half()], -1).flatten(-2)
    return torch.cat([codes, params.contiguous().view(torch.uint8)], -1)


def unpack(rows, case):
    """Cache rows, uint8 [..., row], as the fp32 values [..., D] they stand for."""
    D, bits = case["head_dim"], case["bits"]
    codes, params = rows[..., :D * bits // 8], rows[..., D * bits // 8:]
    if bits == 4:
        codes = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    p = params.contiguous().view(torch.float16).float().unflatten(-1, (D // GROUP, 2))
    c = codes.float().unflatten(-1, (D // GROUP, GROUP))
    return (c * p[..., 0:1] + p[..., 1:2]).half().float().flatten(-2)


def places(s, tokens):
    """Where the rows of K, V lie: the page of each token and its row there."""
    t = torch.arange(tokens, device=s["offsets"].device, dtype=torch.int32)
    b = torch.searchsorted(s["offsets"], t, right=True) - 1
    position = s["lengths"][b] - (s["offsets"][b + 1] - t)
    page = s["case"]["page_size"]
    return s["table"][b, (position // page).long()].long(), (position % page).long()


def plain_write(s):
    case, K, V = s["case"], s["K"], s["V"]
    pool = s["cache"].view(-1, case["heads_kv"], 2, case["page_size"], row_bytes(case))
    page, row = places(s, K.shape[0])
    pool[page, :, 0, row] = pack(K, case["bits"])
    pool[page, :, 1, row] = pack(V, case["bits"])


def plain_read(s, tokens):
    case = s["case"]
    pool = s["cache"].view(-1, case["heads_kv"], 2, case["page_size"], row_bytes(case))
    page, row = places(s, tokens)
    return {"K": unpack(pool[page, :, 0, row], case).half(), "V": unpack(pool[page, :, 1, row], case).half()}


def plain_attend(s):
    case, Q = s["case"], s["Q"]
    D, Hq, Hk = case["head_dim"], case["heads_q"], case["heads_kv"]
    dev, tokens, group, B = Q.device, Q.shape[0], Hq // Hk, case["sequences"]
    lengths, offsets = s["lengths"].long(), s["offsets"].long()
    new = offsets[1:] - offsets[:-1]
    N, pages_per = max(sequences_of(case)[1]), s["table"].shape[1]
    L = pages_per * case["page_size"]
    pool = s["cache"].view(-1, Hk, 2, case["page_size"], row_bytes(case))
    rows = pool[s["table"].long()].permute(0, 2, 3, 1, 4, 5).reshape(B, Hk, 2, L, -1)
    K, V = unpack(rows[:, :, 0], case), unpack(rows[:, :, 1], case)              # [B][Hk][L][D]
    i = torch.arange(N, device=dev)
    at = (offsets[:-1, None] + i).clamp(max=tokens - 1)                          # [B][N]
    q = Q[at].float().view(B, N, Hk, group, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, group * N, D)
    score = torch.matmul(q, K.transpose(-1, -2)).view(B, Hk, group, N, L) * (1.0 / math.sqrt(D))
    key = torch.arange(L, device=dev)
    last = lengths[:, None] - 1 - (new[:, None] - 1 - i if case["causal"] else torch.zeros_like(at))
    seen = (key <= last[..., None]) & (i[:, None] < new[:, None, None])          # [B][N][L]
    score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-3e38)
    p = score.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(B, Hk, group * N, L), V).view(B, Hk, group, N, D) / total.clamp(min=1e-37)
    b = torch.searchsorted(s["offsets"], torch.arange(tokens, device=dev, dtype=torch.int32), right=True) - 1
    n = torch.arange(tokens, device=dev) - offsets[b]
    got = {"O": out.permute(0, 3, 1, 2, 4)[b, n].reshape(tokens, Hq, D).half()}
    if case["lse"]:
        lse = (top + total.log()).squeeze(-1)                                    # [B][Hk][group][N]
        got["lse"] = lse.permute(0, 3, 1, 2)[b, n].reshape(tokens, Hq)
    return got


def run(state):
    op = state["case"]["op"]
    if own:
        plan, cache, batch = state["plan"], state["cache"], state["batch"]
        if op == "attend":
            got = {"O": plan.attention(state["Q"], cache, batch, lse=state["lse"])}
            if state["lse"] is not None:
                got["lse"] = state["lse"]
            return got
        if op == "write_read":
            plan.append(state["K"], state["V"], cache, batch)
        K, V = plan.read(cache, batch)
        return {"K": K, "V": V}
    if op == "attend":
        return plain_attend(state)
    if op == "write_read":
        plain_write(state)
        return plain_read(state, state["K"].shape[0])
    return plain_read(state, sum(sequences_of(state["case"])[1]))


# ----------------------------------------------------------------------------------------------------------
# the definition in 64 bits
# ----------------------------------------------------------------------------------------------------------

def _values64(raw, D, bits):
    """fp64 [n][heads][D] from rows uint8 [n][heads][row]: one element at a time of each group."""
    n, heads, _ = raw.shape
    out = torch.empty(n, heads, D, dtype=torch.float64, device=raw.device)
    codes = D * bits // 8
    for g in range(D // GROUP):
        par = raw[:, :, codes + 4 * g:codes + 4 * g + 4].contiguous().view(torch.float16).double()
        for d in range(g * GROUP, (g + 1) * GROUP):
            c = raw[:, :, d] if bits == 8 else (raw[:, :, d // 2] >> (4 * (d % 2))) & 15
            out[:, :, d] = (c.double() * par[:, :, 0] + par[:, :, 1]).half().double()
    return out


def _rounded64(x, bits):
    """fp64 values that fp16 x [n][heads][D] has after quantising, from the definition."""
    top = 2 ** bits - 1
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for g in range(0, x.shape[-1], GROUP):
        v = x[..., g:g + GROUP].double()
        v = torch.where(torch.isnan(v), torch.zeros_like(v), v).clamp(-F16_MAX, F16_MAX)
        low, high = v.min(-1, keepdim=True).values, v.max(-1, keepdim=True).values
        step = (high - low) / top
        # towards zero in fp16: 11 significant bits, spaced 2^-24 at the least
        unit = torch.exp2(torch.floor(torch.log2(step.clamp(min=2.0 ** -14))) - 10)
        scale = torch.floor(step / unit) * unit
        code = torch.where(scale > 0, ((v - low) / scale).round().clamp(max=top), torch.zeros_like(v))
        out[..., g:g + GROUP] = (code * scale + low).half().double()
    return out


def exact(case, seed):
    global own
    kept, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = kept
    lengths, new = sequences_of(case)
    D, Hq, Hk, bits, page = (case[k] for k in ("head_dim", "heads_q", "heads_kv", "bits", "page_size"))
    if case["op"] == "write_read":
        return {"K": _rounded64(s["K"], bits), "V": _rounded64(s["V"], bits)}
    pool = s["cache"].view(-1, Hk, 2, page, row_bytes(case))
    Ks, Vs, Os, Ls, at = [], [], [], [], 0
    for b, (ln, n) in enumerate(zip(lengths, new)):
        whole = pool[s["table"][b, :(ln + page - 1) // page].long()].permute(2, 0, 3, 1, 4).reshape(2, -1, Hk,
                                                                                                   row_bytes(case))
        K, V = _values64(whole[0, :ln], D, bits), _values64(whole[1, :ln], D, bits)
        if case["op"] == "read":
            Ks.append(K)
            Vs.append(V)
            continue
        O = torch.empty(n, Hq, D, dtype=torch.float64, device=K.device)
        lse = torch.empty(n, Hq, dtype=torch.float64, device=K.device)
        for h in range(Hq):
            hk = h // (Hq // Hk)
            S = s["Q"][at:at + n, h].double() @ K[:, hk].T / math.sqrt(D)
            if case["causal"]:
                row = torch.arange(ln - n, ln, device=K.device)
                S[torch.arange(ln, device=K.device)[None, :] > row[:, None]] = -math.inf
            lse[:, h] = torch.logsumexp(S, -1)
            O[:, h] = torch.exp(S - lse[:, h:h + 1]) @ V[:, hk]
        Os.append(O)
        Ls.append(lse)
        at += n
    if case["op"] == "read":
        return {"K": torch.cat(Ks), "V": torch.cat(Vs)}
    return {"O": torch.cat(Os), "lse": torch.cat(Ls)} if case["lse"] else {"O": torch.cat(Os)}
