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
