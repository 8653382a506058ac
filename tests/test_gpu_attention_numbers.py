"""Attention over listed blocks: queries and values whose numbers are far apart."""
import pytest
import torch

import attention_ref as R
from test_gpu_block_attention import DEV, Setup, dev  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", [8, 4])
@pytest.mark.parametrize("first", [0, 1])
def test_small_query_values_beside_a_large_one(fmt, first):
    """One value of the query is 2^21 times the others and meets zeros in K; the others meet large numbers, and together they are the
    whole score.  The tolerance is the one of every other test: sums of D products of what the codes are held as."""
    from ucmx import ops
    D, T, n = 64, 16, 3
    top = 2 ** fmt - 1
    q = torch.zeros((1, 1, D))
    q[..., first::2] = 255 / 256 * 2.0 ** -11
    q[..., 1 - first] = 1024.0
    k = torch.zeros((n, T, 1, D))
    k[..., first::2] = 15.0 * 64.0
    k[1:, ::2, :, first::2] = 0.0                                         # tokens whose score is nothing
    k[..., 8 + first] = 15.0 * 64.0                                       # (a row of zeros has no scale)
    v = torch.randn((n, T, 1, D), generator=torch.Generator().manual_seed(1))
    q, k, v = (x.to(torch.bfloat16) for x in (q, k, v))
    data = R.pack(k, v, fmt)
    kd, vd = R.values(data, D, fmt)
    assert float((kd - k.double()).abs().max()) <= 960.0 / top            # (scale 64 at 4 bits: exact)
    out, want, tol, ltol = R.attend(q, kd, vd, [(range(1), [(i, i) for i in range(n)], None)], codes_err=960.0)
    lse = torch.zeros((1, 1), device=DEV)
    got = ops.quant_block_attention(q.to(DEV), ops.QuantKvCache(data.to(DEV), head_dim=D, bits=fmt), dev([0, n]), block_ids=dev(range(n)), lse=lse)
    R.check(got, out, tol, "out")
    R.check(lse, want, ltol, "lse")


@pytest.mark.parametrize("H,G,D,T,counts,nq", [
    (2, 1, 64, 16, [3, 1], None), (2, 4, 128, 16, [5, 40], None), (1, 8, 128, 32, [4, 2], None), (1, 12, 64, 16, [6], None),
    (1, 30, 128, 16, [7, 2], None), (1, 6, 256, 16, [3, 900], None), (1, 4, 128, 16, [5, 3], [3, 2]),
])
def test_an_infinity_that_is_seen_is_one(H, G, D, T, counts, nq):
    """A sum of weights above zero times values one of which is infinite is infinite."""
    s = Setup(81, 16, H, G, D, T, counts, nq).tails()
    for r, (rows, blocks, ctx) in enumerate(s.lists()):
        n = len(rows)
        for at, d, x in ((0, 5, "inf"), (ctx - n, 6, "-inf"), (ctx // 2, 33, "inf"), (ctx // 3, D - 1, "-inf")):
            at = min(at, ctx - n)
            s.v16[blocks[at // T][0], at % T, :, d] = float(x)
    s.vd = s.v16.double()
    out, _, tol, _ = s.want()
    assert bool(torch.isinf(out).any(-1).all()) and not bool(torch.isnan(out).any())
    R.check(s.run(), out, tol)


def test_scores_that_are_all_minus_infinity_count_as_unseen():
    for G, nq in ((1, 1), (4, 1), (8, 2)):
        s = Setup(82, 16, 2, G, 64, 16, [3, 40, 2], [nq] * 3).tails()
        s.q[:, :G, 7] = 1.0
        s.k16[s.ids[s.off[1]:s.off[2]].astype(int), :, 0, 7] = float("-inf")           # the second request's blocks, one head
        s.kd = s.k16.double()
        out, want, tol, ltol = s.want()
        rows = slice(int(s.qoff[1]), int(s.qoff[2]))
        assert bool(torch.isnan(out[rows, :G]).all())                                  # (the formula's own answer is no number)
        out[rows, :G], tol[rows, :G], want[rows, :G], ltol[rows, :G] = 0.0, 0.0, float("-inf"), 0.0
        lse = torch.zeros(s.q.shape[:2], device=DEV)
        got = s.run(lse=lse)
        R.check(got, out, tol)
        R.check(lse, want, ltol)
