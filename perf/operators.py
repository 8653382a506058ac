"""What is measured of the attention over selected blocks and of the quantised paged KV cache.

Four operators: `attend` (attention of each request's queries over the blocks listed for it, bf16 cache), `qattend` (the same
over a cache held in 4 or 8 bits), `append` (a decode step over the quantised cache: the new tokens' K/V rows are quantised into
it, then attended to), and `store` (K/V rows or whole blocks are quantised into the cache and read back).

Shapes: `req` requests of `lo`..`hi` blocks of `tokens` tokens (spread evenly over their logarithm), `hkv` KV heads, `hq` query
heads, `dim` values a head, `nq` query tokens a request at most; `tail`: contexts end inside their last block; `sparse`: the
blocks listed are a selection of a longer sequence, given with their positions in it; `hollow`: some requests list nothing.
"""
import math

import torch

own = False

DEV = "cuda:0"


# ------------------------------------------------------------------------------------------------------------ the cases

def _case(kind, name=None, **kw):
    c = dict(kind=kind, req=1, lo=1, hi=1, tokens=16, hkv=8, hq=32, dim=128, nq=1, bits=16, tail=True, sparse=False,
             hollow=False, blocks=False)
    c.update(kw)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # one short chat request at its first decode steps: latency is all there is
        _case("attend", "attend_one_short", req=1, lo=5, hi=5, tokens=16),
        # the decode batch of the retrieval benchmark: 64 requests, 5 % of 8k..128k tokens selected, 128-token blocks
        _case("attend", "attend_decode64", req=64, lo=16, hi=52, tokens=128, tail=False, sparse=True),
        # a draft of up to 5 tokens checked at once, 8 query heads a KV head, ragged tails, requests without blocks
        _case("attend", "attend_draft", req=24, lo=9, hi=160, tokens=16, hq=64, nq=5, sparse=True, hollow=True),
        # one very long prompt, every block attended
        _case("attend", "attend_long", req=1, lo=1023, hi=1023, tokens=128),
        # a small model: 64 values a head, 7 query heads on each of 2 KV heads, many short requests
        _case("attend", "attend_small_model", req=190, lo=1, hi=40, tokens=32, hkv=2, hq=14, dim=64),
        # few requests at moderate length over the 4-bit cache
        _case("qattend", "q4_few", req=3, lo=30, hi=110, tokens=16, bits=4),
        # a long-context decode batch over the 4-bit cache, all blocks attended
        _case("qattend", "q4_batch", req=32, lo=120, hi=500, tokens=64, bits=4),
        # the selection of the benchmark's batch over an 8-bit cache
        _case("qattend", "q8_decode64", req=64, lo=16, hi=52, tokens=128, bits=8, tail=False, sparse=True),
        # decode steps: new rows into the cache, then attention over it
        _case("append", "append_q4", req=48, lo=60, hi=130, tokens=64, bits=4),
        _case("append", "append_q8_small", req=5, lo=7, hi=30, tokens=16, bits=8, hq=64),
        # a prefill chunk goes into the 4-bit cache token by token and is read back
        _case("store", "store_tokens_q4", req=1, lo=509, hi=509, tokens=16, bits=4),
        # full blocks go into an 8-bit store and come back
        _case("store", "store_blocks_q8", req=1, lo=300, hi=300, tokens=128, bits=8, blocks=True),
    ]


def draw(rng):
    def log_int(a, b):
        return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))

    kind = rng.choice(["attend", "attend", "qattend", "qattend", "append", "store"])
    tokens = rng.choice([16, 32, 64, 128])
    bits = 16 if kind == "attend" else rng.choice([4, 8])
    hkv = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 3, 4, 5, 7, 8, 16])
    dim = rng.choice([64, 128, 128, 128, 256])
    if kind == "store":
        rows = log_int(8, 40000)
        return _case(kind, lo=max(1, rows // tokens), hi=max(1, rows // tokens), tokens=tokens, hkv=hkv, dim=dim, bits=bits,
                     blocks=rng.random() < 0.5)
    req = log_int(1, 200)
    hi = log_int(1, 1000)
    lo = max(1, int(hi * rng.uniform(0.1, 1.0)))
    nq = rng.choice([1, 1, 2, 4, 7]) if kind != "append" else 1
    values = req * tokens * hkv * dim
    cap = min((60e6 if kind == "attend" else 200e6) / values, 2e9 / (values * group * nq))
    hi = max(1, min(hi, int(cap)))
    lo = min(lo, hi)
    return _case(kind, req=req, lo=lo, hi=hi, tokens=tokens, hkv=hkv, hq=hkv * group, dim=dim, bits=bits,
                 nq=nq, tail=rng.random() < 0.8,
                 sparse=kind != "append" and rng.random() < 0.5, hollow=kind != "append" and rng.random() < 0.3)


def _counts(c):
    """Blocks of each request: spread evenly over the logarithm of [lo, hi]; the hollow ones list none."""
    R = c["req"]
    n = [int(round(c["lo"] * (c["hi"] / c["lo"]) ** ((i + 0.5) / R))) for i in range(R)]
    if c["hollow"]:
        n = [0 if i % 8 == 3 else x for i, x in enumerate(n)]
    return n


def _queries(c):
    return [1 + (i % c["nq"]) if i % 3 else c["nq"] for i in range(c["req"])]


def work(case):
    c, n, nq = case, _counts(case), _queries(case)
    row = c["dim"] * 2 if c["bits"] == 16 else c["dim"] * c["bits"] // 8 + 4      # one K or V row as it is held
    if c["kind"] == "store":
        rows = 2 * sum(n) * c["tokens"] * c["hkv"]
        return {"bytes": 2 * rows * (c["dim"] * 2 + row), "flops": 6 * rows * c["dim"]}
    toks = sum(n) * c["tokens"]
    io = 2 * sum(nq) * c["hq"] * c["dim"] * 2 + 8 * sum(n)
    if c["kind"] == "append":
        io += 2 * c["req"] * c["hkv"] * (c["dim"] * 2 + row)
    return {"bytes": 2 * toks * c["hkv"] * row + io,
            "flops": sum(4 * a * b for a, b in zip(n, nq)) * c["tokens"] * c["hq"] * c["dim"]}


# ----------------------------------------------------------------------------------------- the quantised cache, plain form
#
# uint8 [blocks, heads, tokens/16, group bytes].  A group holds 16 tokens of one KV head: K codes, V codes, then bf16 (scale,
# zero) of the 16 K rows and of the 16 V rows.  Both code parts come in panels of up to 64 bytes a token.  A K panel is
# [token][bytes].  A V panel is [token / 8][byte chunk 0..7][(token % 8) / 2][unit of 2 bytes in the chunk][token % 2][2 bytes].
# Codes lie in order of the dimension, the lower one in the lower bits.

def _panel(dim, bits):
    return min(64, dim * bits // 8)


def _codes_of(x, bits):
    """(codes as float64, scale and zero as bf16) of rows x [..., dim]; the quotient in 64 bits, so that ties are seen as such."""
    top = 2.0 ** bits - 1
    x = x.double()
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    scale = ((hi - lo) / top).float().to(torch.bfloat16)
    s = scale.double()
    codes = torch.where(s > 0, ((x - lo) / torch.where(s > 0, s, 1.0)).round().clamp(0, top), 0.0)
    return codes, scale, lo.to(torch.bfloat16)


def _pack(k, v, bits):
    """K, V rows [n, tokens, heads, dim] -> groups uint8 [n, heads, tokens/16, bytes]."""
    n, T, H, D = k.shape
    pb = _panel(D, bits)
    P, parts, params = D * bits // 8 // pb, [], []
    for which, x in enumerate((k, v)):
        codes, scale, zero = _codes_of(x, bits)
        b = codes.to(torch.uint8)
        if bits == 4:
            b = b[..., 0::2] | (b[..., 1::2] << 4)
        b = b.permute(0, 2, 1, 3).reshape(n, H, T // 16, 16, P, pb)
        if which == 0:
            b = b.permute(0, 1, 2, 4, 3, 5)
        else:
            b = b.reshape(n, H, T // 16, 2, 4, 2, P, 8, pb // 16, 2).permute(0, 1, 2, 6, 3, 7, 4, 8, 5, 9)
        parts.append(b.reshape(n, H, T // 16, -1))
        sz = torch.cat([scale, zero], -1).permute(0, 2, 1, 3).reshape(n, H, T // 16, 32).contiguous()
        params.append(sz.view(torch.uint8))
    return torch.cat(parts + params, -1)


def _unpack(g, dim, bits):
    """Groups uint8 [..., heads, tokens/16, bytes] -> K, V in fp32 [..., tokens, heads, dim]."""
    lead, (H, G) = g.shape[:-3], g.shape[-3:-1]
    g = g.reshape(-1, H, G, g.shape[-1])
    n, pb, half = g.shape[0], _panel(dim, bits), 16 * dim * bits // 8
    P, got = dim * bits // 8 // pb, []
    for which in (0, 1):
        b = g[..., which * half:(which + 1) * half]
        if which == 0:
            b = b.reshape(n, H, G, P, 16, pb).permute(0, 1, 2, 4, 3, 5)
        else:
            b = b.reshape(n, H, G, P, 2, 8, 4, pb // 16, 2, 2).permute(0, 1, 2, 4, 6, 8, 3, 5, 7, 9)
        b = b.reshape(n, H, G * 16, dim * bits // 8)
        if bits == 4:
            b = torch.stack([b & 15, b >> 4], -1).reshape(n, H, G * 16, dim)
        sz = g[..., 2 * half + which * 64:2 * half + which * 64 + 64].contiguous().view(torch.bfloat16).reshape(n, H, G * 16, 2).float()
        x = b.float() * sz[..., 0:1] + sz[..., 1:2]
        got.append(x.permute(0, 2, 1, 3).reshape(*lead, G * 16, H, dim))
    return got


# --------------------------------------------------------------------------------------------------------------- inputs

def _rows(gen, n, T, H, D, spread):
    """K or V rows: normal values, and for K a few channels that are several times the others, as trained models have."""
    x = torch.randn((n, T, H, D), generator=gen, device=DEV)
    return (x * spread).to(torch.bfloat16)


def prepare(case, seed):
    c = case
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    n, nq = _counts(c), _queries(c)
    T, H, Hq, D, bits = c["tokens"], c["hkv"], c["hq"], c["dim"], c["bits"]
    total = sum(n)
    pool = total + 3                                          # the pool holds a few blocks that nobody lists
    i32 = dict(dtype=torch.int32, device=DEV)
    spread = 1.0 + 4.0 * (torch.rand((H, D), generator=gen, device=DEV) < 0.03)
    s = {"case": c}
    if c["kind"] == "store":
        s["k"] = _rows(gen, pool, T, H, D, spread)
        s["v"] = _rows(gen, pool, T, H, D, 1.0)
        s["ids"] = torch.randperm(pool, generator=gen, device=DEV)[:total].to(torch.int32)
        s["cache"] = torch.zeros((pool, H, T // 16, 2 * 16 * (D * bits // 8) + 128), dtype=torch.uint8, device=DEV)
        s["k_back"] = torch.zeros((total, T, H, D), dtype=torch.bfloat16, device=DEV)
        s["v_back"] = torch.zeros_like(s["k_back"])
        if c["blocks"]:
            s["rows"] = torch.randperm(pool, generator=gen, device=DEV)[:total].to(torch.int32)   # cache block of each block written
        else:                                                 # the tokens of one sequence in its blocks, in order
            s["k"], s["v"] = s["k"][:total].reshape(total * T, H, D), s["v"][:total].reshape(total * T, H, D)
            s["rows"] = s["ids"]
            s["slots"] = (s["ids"].long()[:, None] * T + torch.arange(T, device=DEV)).reshape(-1)
        return s
    if bits == 16:
        s["k"], s["v"] = _rows(gen, pool, T, H, D, spread), _rows(gen, pool, T, H, D, 1.0)
    else:
        step = max(1, int(2e7 // (T * H * D)))
        s["cache"] = torch.cat([_pack(_rows(gen, min(step, pool - a), T, H, D, spread), _rows(gen, min(step, pool - a), T, H, D, 1.0), bits)
                                for a in range(0, pool, step)])
    s["ids"] = torch.randperm(pool, generator=gen, device=DEV)[:total].to(torch.int32)
    off = [0]
    for x in n:
        off.append(off[-1] + x)
    s["offsets"], s["most"] = torch.tensor(off, **i32), max(n)
    qoff = [0]
    for x in nq:
        qoff.append(qoff[-1] + x)
    s["q_offsets"], s["nq"] = torch.tensor(qoff, **i32), max(nq)
    s["q"] = torch.randn((qoff[-1], Hq, D), generator=gen, device=DEV).to(torch.bfloat16)
    # where the listed blocks stand in their sequences, and where the sequences end
    last = [x - 1 for x in n]
    if c["sparse"]:
        gap = torch.randint(0, 12, (total,), generator=gen, device=DEV)
        run_ = torch.cumsum(gap + 1, 0)
        first = torch.repeat_interleave(run_[s["offsets"][:-1].long().clamp(max=max(total - 1, 0))] - 1,
                                        torch.tensor(n, device=DEV), output_size=total)
        s["positions"] = (run_ - 1 - first).to(torch.int32)
        p = s["positions"].cpu()
        last = [int(p[off[i + 1] - 1]) if x else 0 for i, x in enumerate(n)]
    else:
        s["positions"] = None
    cut = torch.randint(0, T, (len(n),), generator=gen, device=DEV).cpu() if c["tail"] else [0] * len(n)
    s["ctx"] = torch.tensor([max(0, (l + 1) * T - int(x)) for l, x in zip(last, cut)], **i32) if c["tail"] or max(nq) > 1 else None
    if c["kind"] == "append":                                 # the last token of each request is the new one
        s["k_new"], s["v_new"] = (_rows(gen, c["req"], 1, H, D, x)[:, 0].contiguous() for x in (spread, 1.0))
        at = torch.tensor([(l + 1) * T - int(x) - 1 for l, x in zip(last, cut)], device=DEV)
        block = s["ids"].long()[s["offsets"][:-1].long() + at // T]
        s["slots"] = block * T + at % T
    return s


# ------------------------------------------------------------------------------------------------------------ plain form

def _attend_plain(s, k, v):
    """k, v: rows of the listed blocks padded to the longest list, [requests, blocks, T, H, D], fp32."""
    R, N, T, H, D = k.shape
    dev, off, qoff = k.device, s["offsets"].long(), s["q_offsets"].long()
    n, nq = off[1:] - off[:-1], qoff[1:] - qoff[:-1]
    j = torch.arange(s["nq"], device=dev)
    q = s["q"][(qoff[:-1, None] + j).clamp(max=s["q"].shape[0] - 1)].float()
    q = q.reshape(R, s["nq"], H, -1, D).permute(0, 2, 3, 1, 4).reshape(R, H, -1, D)
    listed_ = torch.arange(N, device=dev)[None] < n[:, None]
    place = torch.arange(N, device=dev).expand(R, N) if s["positions"] is None else _rows_of(s, s["positions"])
    place = place[:, :, None] * T + torch.arange(T, device=dev)
    end = torch.full((R, s["nq"]), 1 << 60, device=dev) if s["ctx"] is None else s["ctx"].long()[:, None] - (nq[:, None] - 1 - j)
    seen = (listed_[:, :, None] & torch.ones_like(place, dtype=torch.bool)).reshape(R, 1, -1) & (place.reshape(R, 1, -1) < end[:, :, None])
    any_seen = seen.any(1)
    v = torch.where(any_seen[:, :, None, None], v.reshape(R, N * T, H, D), 0.0)
    sc = q @ k.reshape(R, N * T, H, D).permute(0, 2, 3, 1) / math.sqrt(D)
    G = sc.shape[2] // s["nq"]
    sc = sc.reshape(R, H, G, s["nq"], N * T).masked_fill(~seen[:, None, None], -math.inf)
    m = sc.amax(-1, keepdim=True)
    p = torch.exp(sc - torch.where(torch.isinf(m), 0.0, m))
    l = p.sum(-1, keepdim=True)
    o = p.reshape(R, H, G * s["nq"], N * T) @ v.permute(0, 2, 1, 3)
    o = o.reshape(R, H, G, s["nq"], D)
    o = torch.where(l > 0, o / l, 0.0).permute(0, 3, 1, 2, 4).reshape(R, s["nq"], H * G, D)
    r = torch.repeat_interleave(torch.arange(R, device=dev), nq, output_size=s["q"].shape[0])
    return o[r, torch.arange(s["q"].shape[0], device=dev) - qoff[r]].to(torch.bfloat16)


def _rows_of(s, flat):
    """One value an entry of the lists, as rows of the longest list's length (what lies behind a shorter list is not used)."""
    off = s["offsets"].long()
    at = off[:-1, None] + torch.arange(s["most"], device=flat.device)
    return flat.long()[at.clamp(max=max(flat.numel() - 1, 0))]


def _run_plain(s):
    c = s["case"]
    T, H, D, bits = c["tokens"], c["hkv"], c["dim"], c["bits"]
    if c["kind"] == "store":
        rows = s["rows"].long()
        if c["blocks"]:
            k, v = s["k"][s["ids"].long()], s["v"][s["ids"].long()]
        else:
            k, v = s["k"].reshape(-1, T, H, D), s["v"].reshape(-1, T, H, D)
        s["cache"][rows] = _pack(k, v, bits)
        back = _unpack(s["cache"][rows], D, bits)
        s["k_back"].copy_(back[0])
        s["v_back"].copy_(back[1])
        return s["k_back"], s["v_back"]
    if c["kind"] == "append":
        block, t = s["slots"] // T, s["slots"] % T
        blocks = s["cache"][block]
        k, v = (x.reshape(-1, T, H, D) for x in _unpack(blocks, D, bits))
        new = _pack(*(x[:, None].expand(-1, T, -1, -1) for x in (s["k_new"], s["v_new"])), bits)   # the row at every token's place
        mine = _place_mask(t, T, D, bits)
        s["cache"][block] = torch.where(mine[:, None], new, blocks)
    ids = _rows_of(s, s["ids"])
    if bits == 16:
        return _attend_plain(s, s["k"][ids].float(), s["v"][ids].float())
    return _attend_plain(s, *_unpack(s["cache"][ids], D, bits))


def _place_mask(t, T, dim, bits):
    """Which bytes of a block's groups belong to token t: [n, tokens/16, bytes]."""
    mark = (torch.arange(T, device=t.device)[None] == t[:, None])
    n, pb = t.shape[0], _panel(dim, bits)
    P = dim * bits // 8 // pb
    m = mark.reshape(n, T // 16, 16)
    kpart = m[:, :, None, :, None].expand(-1, -1, P, -1, pb).reshape(n, T // 16, -1)
    vpart = m.reshape(n, T // 16, 1, 2, 1, 4, 1, 2, 1).expand(-1, -1, P, -1, 8, -1, pb // 16, -1, 2).reshape(n, T // 16, -1)
    spart = m[..., None].expand(-1, -1, -1, 4).reshape(n, T // 16, -1)
    return torch.cat([kpart, vpart, spart, spart], -1)


# ---------------------------------------------------------------------------------------------------- the framework's calls

def _run_own(s):
    import sys
    if "unified-cache-management_b200" not in sys.path:
        sys.path.insert(0, "unified-cache-management_b200")
    from ucmx import ops
    c = s["case"]
    if c["bits"] != 16:
        cache = ops.QuantKvCache(s["cache"], head_dim=c["dim"], bits=c["bits"])
    if c["kind"] == "store":
        if c["blocks"]:
            ops.quant_write_blocks(cache, s["k"], s["v"], s["ids"], out_slots=s["rows"])
        else:
            ops.quant_write_tokens(cache, s["k"], s["v"], s["slots"])
        ops.quant_read_blocks(cache, s["rows"], k_out=s["k_back"], v_out=s["v_back"])
        return s["k_back"], s["v_back"]
    lists = dict(block_ids=s["ids"], positions=s["positions"], ctx_lens=s["ctx"], q_offsets=s["q_offsets"] if s["nq"] > 1 else None,
                 max_q_tokens=s["nq"])
    if c["kind"] == "append":
        ops.quant_write_tokens(cache, s["k_new"], s["v_new"], s["slots"])
    if c["bits"] == 16:
        return ops.block_attention(s["q"], s["k"], s["v"], s["offsets"], **lists)
    return ops.quant_block_attention(s["q"], cache, s["offsets"], **lists)


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ----------------------------------------------------------------------------------------------------------- in 64 bits

def _bf16_value(a, b):
    """The number that two bytes (low, high) of a bf16 stand for."""
    bits = (a.to(torch.int32) | (b.to(torch.int32) << 8)) << 16
    return bits.view(torch.float32).double()


def _held(g, which, dim, bits):
    """K (0) or V (1) of groups [n, heads, tokens/16, bytes] in 64 bits, each value fetched from its place in the group."""
    n, H, G, _ = g.shape
    t = torch.arange(16, device=g.device)[:, None]
    d = torch.arange(dim, device=g.device)[None]
    pb, nb = min(64, dim * bits // 8), dim * bits // 8
    byte = d * bits // 8
    if which == 0:
        at = (byte // pb) * 16 * pb + t * pb + byte % pb
    else:
        x = byte % pb
        chunk = pb // 8
        at = 16 * nb + (byte // pb) * 16 * pb + (t // 8) * 8 * pb + (x // chunk) * 8 * chunk + ((t % 8) // 2) * 2 * chunk \
            + ((x % chunk) // 2) * 4 + (t % 2) * 2 + x % 2
    code = g[..., at.reshape(-1)].reshape(n, H, G, 16, dim)
    if bits == 4:
        code = torch.where(d % 2 == 1, code // 16, code % 16)
    p = 32 * nb + which * 64 + torch.arange(16, device=g.device) * 4
    scale, zero = _bf16_value(g[..., p], g[..., p + 1]), _bf16_value(g[..., p + 2], g[..., p + 3])
    x = code.double() * scale[..., None] + zero[..., None]
    return x.reshape(n, H, G * 16, dim)


def _nearest(x, bits):
    """What rows x [..., dim] read back as, in 64 bits, from the definition."""
    x, steps = x.double(), 2 ** bits - 1
    zero = x.min(-1, keepdim=True).values
    scale = ((x.max(-1, keepdim=True).values - zero) / steps).float().bfloat16().double()
    code = torch.round((x - zero) / scale.masked_fill(scale == 0, 1.0)).clamp(max=steps)
    return code * scale + zero


def exact(case, seed):
    c, s = case, prepare(case, seed)
    T, H, Hq, D, bits = c["tokens"], c["hkv"], c["hq"], c["dim"], c["bits"]
    if c["kind"] == "store":
        pick = (lambda x: x[s["ids"].long()]) if c["blocks"] else (lambda x: x.reshape(-1, T, H, D))
        return tuple(torch.cat([_nearest(y, bits) for y in pick(s[x]).split(64)]) for x in ("k", "v"))
    off, qoff = s["offsets"].tolist(), s["q_offsets"].tolist()
    ctx = s["ctx"].tolist() if s["ctx"] is not None else None
    out = torch.zeros((qoff[-1], Hq, D), dtype=torch.float64, device=DEV)
    for r in range(c["req"]):
        ids = s["ids"][off[r]:off[r + 1]].long()
        if not ids.numel():
            continue
        if bits == 16:
            k, v = (s[x][ids].double().reshape(-1, H, D).permute(1, 0, 2) for x in ("k", "v"))
        else:
            g = s["cache"][ids]
            k, v = (_held(g, w, D, bits).permute(1, 0, 2, 3).reshape(H, -1, D).clone() for w in (0, 1))
        place = s["positions"][off[r]:off[r + 1]].long() if s["positions"] is not None else torch.arange(len(ids), device=DEV)
        place = (place[:, None] * T + torch.arange(T, device=DEV)).reshape(-1)
        if c["kind"] == "append":
            here = int((place == ctx[r] - 1).nonzero()[0]) if ctx is not None else place.numel() - 1
            k[:, here], v[:, here] = _nearest(s["k_new"][r], bits), _nearest(s["v_new"][r], bits)
        many = qoff[r + 1] - qoff[r]
        for j in range(many):
            keep = place < ctx[r] - (many - 1 - j) if ctx is not None else place >= 0
            if not bool(keep.any()):
                continue
            q = s["q"][qoff[r] + j].double().reshape(H, -1, D)
            w = torch.softmax(q @ k[:, keep].transpose(1, 2) / math.sqrt(D), -1)
            out[qoff[r] + j] = (w @ v[:, keep]).reshape(Hq, D)
    return out
