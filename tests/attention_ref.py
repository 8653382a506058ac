"""Plain 64-bit forms of the quantised cache and of attention over listed blocks (torch on the CPU), and how far a kernel that
keeps its sums in 32 bits may be from them."""
import numpy as np
import torch


def to_codes(x, bits):
    """Rows x [..., dim] (bf16): codes (int64), scale and zero (float64, bf16 values) by the definition."""
    top = 2 ** bits - 1
    x = x.double()
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    scale = ((hi - lo) / top).float().to(torch.bfloat16).double()
    codes = torch.where(scale > 0, torch.round((x - lo) / torch.where(scale > 0, scale, 1.0)).clamp(0, top), 0.0)
    bad = ~torch.isfinite(x).all(-1, keepdim=True)
    nan = torch.tensor(float("nan"), dtype=torch.float64)
    return torch.where(bad, 0.0, codes).long(), torch.where(bad, nan, scale), torch.where(bad, nan, lo)


def places(which, dim, bits):
    """Byte of a group that holds the code of (token 0..15, dimension), and the bit shift inside it."""
    t, d = np.meshgrid(np.arange(16), np.arange(dim), indexing="ij")
    nb = dim * bits // 8
    P = min(64, nb)
    b = d * bits // 8
    panel, x = b // P, b % P
    if which == 0:
        at = panel * 16 * P + t * P + x
    else:
        c = P // 8
        at = 16 * nb + panel * 16 * P + (t // 8) * 8 * P + (x // c) * P + (t % 8 // 2) * (2 * c) + (x % c // 2) * 4 + (t % 2) * 2 + x % 2
    return torch.from_numpy(at), torch.from_numpy((d % 2) * 4 if bits == 4 else d * 0)


def held(data, dim, bits):
    """(codes, scale, zero) of K and of V of a cache uint8 [blocks, heads, groups, bytes]: [blocks, tokens, heads, dim | 1]."""
    nb, H, G, _ = data.shape
    out = []
    for which in (0, 1):
        at, sh = places(which, dim, bits)
        codes = (data[..., at.reshape(-1)].reshape(nb, H, G, 16, dim).long() >> sh) & (2 ** bits - 1)
        p = 32 * (dim * bits // 8) + which * 64
        sz = data[..., p:p + 64].contiguous().view(torch.bfloat16).reshape(nb, H, G, 16, 2).double()
        f = lambda x: x.reshape(nb, H, G * 16, -1).permute(0, 2, 1, 3)  # noqa: E731
        out.append((f(codes), f(sz[..., :1]), f(sz[..., 1:])))
    return out


def pack(k, v, bits):
    """K, V rows bf16 [blocks, tokens, heads, dim] -> the cache's bytes."""
    nb, T, H, D = k.shape
    data = torch.zeros((nb, H, T // 16, 32 * (D * bits // 8) + 128), dtype=torch.uint8)
    for which, x in enumerate((k, v)):
        codes, scale, zero = to_codes(x, bits)
        at, sh = places(which, D, bits)
        c = codes.permute(0, 2, 1, 3).reshape(nb, H, T // 16, 16, D) << sh
        flat = torch.zeros_like(data, dtype=torch.int64)
        flat.scatter_add_(-1, at.reshape(-1).expand(nb, H, T // 16, -1), c.reshape(nb, H, T // 16, -1))
        data |= flat.to(torch.uint8)
        sz = torch.cat([scale, zero], -1).to(torch.bfloat16).permute(0, 2, 1, 3).reshape(nb, H, T // 16, 32).contiguous()
        p = 32 * (D * bits // 8) + which * 64
        data[..., p:p + 64] = sz.view(torch.uint8)
    return data


def values(data, dim, bits):
    """K and V in float64 [blocks, tokens, heads, dim]."""
    return [c.double() * s + z for c, s, z in held(data, dim, bits)]


def attend(q, k, v, lists, *, scale=None, codes_err=0.0):
    """out, lse, tolerance of out, tolerance of lse (float64).  q [tokens, Hq, D]; k, v [blocks, T, H, D] float64;
    lists: per request (query rows, [(block, place), ...], ctx or None).

    Tolerances.  u = 2^-23 bounds one fp32 step, of the matrix unit's sums too (they may truncate).  A score is a sum of D products:
    off by at most delta = scale * (D + 4) * u * sum |q||k| (codes_err: what the split of a quantised row into codes and zero adds to
    |k|), and its use as a power of two by |score| * u * 2.  A weight is then off by a factor 1 + 2 delta (numerator and sum), by
    2^-16 for its two bf16 halves, by 4u for the power, and sums over n tokens by n*u.  All of that is of sum p|v|; the result is
    rounded to bf16 once: 2^-8 |out|."""
    D = q.shape[-1]
    scale = D ** -0.5 if scale is None else scale
    T, H = k.shape[1], k.shape[2]
    G = q.shape[1] // H
    q = q.double()
    out, tol = torch.zeros_like(q), torch.zeros_like(q)
    lse = torch.full(q.shape[:2], -float("inf"), dtype=torch.float64)
    ltol = torch.zeros_like(lse)
    u = 2.0 ** -23
    for rows, blocks, ctx in lists:
        n = len(rows)
        for j, row in enumerate(rows):
            end = float("inf") if ctx is None else ctx - (n - 1 - j)
            pick = [(b, t) for b, place in blocks for t in range(T) if place * T + t < end]
            if not pick:
                continue
            bi, ti = (torch.tensor(x) for x in zip(*pick))
            for h in range(H):
                kk, vv = k[bi, ti, h], v[bi, ti, h]
                qq = q[row, h * G:(h + 1) * G]
                s = scale * (qq @ kk.T)
                mag = (qq.abs() @ (kk.abs() + codes_err).T).amax(-1) * abs(scale)
                m = s.amax(-1, keepdim=True)
                p = torch.exp(s - m)
                l = p.sum(-1, keepdim=True)
                o = (p / l) @ vv
                delta = (D + 4) * u * mag + 4 * u * s.abs().amax(-1)
                absv = (p / l) @ (vv.abs() + codes_err)
                out[row, h * G:(h + 1) * G] = o
                tol[row, h * G:(h + 1) * G] = 2.0 ** -8 * o.abs() + absv * (2 * delta[:, None] + 2.0 ** -16 + (len(pick) + 8) * u)
                lse[row, h * G:(h + 1) * G] = (m + l.log())[:, 0]
                ltol[row, h * G:(h + 1) * G] = delta + (len(pick) + 8) * u + 4 * u * lse[row, h * G:(h + 1) * G].abs()
    return out, lse, tol, ltol


def check(got, want, tol, what=""):
    got = got.detach().cpu().double()
    same_nan = torch.isnan(got) == torch.isnan(want)
    assert bool(same_nan.all()), f"{what}: NaN in other places"
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]), what
    fine = ~torch.isnan(want) & ~inf
    over = ((got - want).abs() - tol)[fine]
    if over.numel():
        worst = float(over.max())
        assert worst <= 0, f"{what}: {worst} beyond the tolerance"
