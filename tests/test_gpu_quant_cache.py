"""The quantised paged cache: codes, scales and zeros equal to the definition bit for bit (ties included), every place of the layout,
slots in any order, rows with infinities, and the way back."""
import numpy as np
import pytest
import torch

import attention_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
FORMS = [(4, 64), (4, 128), (4, 256), (8, 64), (8, 128), (8, 256)]


def rows(seed, *shape, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(torch.bfloat16)


def dev(a):
    return torch.as_tensor(np.asarray(a), dtype=torch.int32).to(DEV)


def same_rows(cache, k, v, bits, where=None):
    """The cache's codes, scales and zeros are those of K and V [blocks, tokens, heads, dim]."""
    got = R.held(cache.data.cpu(), k.shape[-1], bits)
    for (codes, scale, zero), x in zip(got, (k, v)):
        wc, ws, wz = R.to_codes(x, bits)
        pick = (lambda t: t) if where is None else (lambda t: t[where])
        assert torch.equal(pick(codes), pick(wc))
        assert torch.equal(pick(scale).nan_to_num(-7.0), pick(ws).nan_to_num(-7.0))
        assert torch.equal(pick(zero).nan_to_num(-7.0), pick(wz).nan_to_num(-7.0))


@pytest.mark.parametrize("bits,D", FORMS)
@pytest.mark.parametrize("T,H,n", [(16, 1, 1), (32, 3, 5), (128, 8, 3)])
def test_blocks_there_and_back(bits, D, T, H, n):
    from ucmx import _native, ops
    k, v = rows(1, n + 3, T, H, D), rows(2, n + 3, T, H, D, scale=5.0)
    ids = np.random.default_rng(0).permutation(n + 3)[:n]
    out = np.random.default_rng(1).permutation(n + 2)[:n]
    c = ops.QuantKvCache.alloc(n + 2, T, H, D, bits, DEV)
    ops.quant_write_blocks(c, k.to(DEV), v.to(DEV), dev(ids), out_slots=dev(out))
    kb, vb = ops.quant_read_blocks(c, dev(out))
    torch.cuda.synchronize()
    assert _native.device_error() == 0
    want_k, want_v = torch.zeros((n + 2, T, H, D), dtype=torch.bfloat16), torch.zeros((n + 2, T, H, D), dtype=torch.bfloat16)
    want_k[out], want_v[out] = k[ids], v[ids]
    same_rows(c, want_k, want_v, bits)
    assert torch.equal(c.data.cpu(), R.pack(want_k, want_v, bits))        # (blocks that were not written stay zero)
    for got, x in ((kb, k[ids]), (vb, v[ids])):
        codes, scale, zero = R.to_codes(x, bits)
        assert torch.equal(got.cpu(), (codes.double() * scale + zero).float().to(torch.bfloat16))


@pytest.mark.parametrize("bits,D", FORMS)
def test_tokens_one_by_one_in_any_order(bits, D):
    """Slots in order, shuffled, with gaps and skips, from rows of a wider tensor; tokens that are not named keep what they had."""
    from ucmx import _native, ops
    T, H, nb = 32, 2, 4
    c = ops.QuantKvCache.alloc(nb, T, H, D, bits, DEV)
    k0, v0 = rows(3, nb, T, H, D), rows(4, nb, T, H, D)
    ops.quant_write_blocks(c, k0.to(DEV), v0.to(DEV), dev(range(nb)))
    want_k, want_v = k0.clone().reshape(-1, H, D), v0.clone().reshape(-1, H, D)
    rng = np.random.default_rng(6)
    for slots in (np.arange(40) + 3, np.arange(33) * 2 + 1, rng.permutation(nb * T)[:77], np.asarray([5]), np.asarray([9, 8]),
                  np.where(rng.random(50) < 0.3, -1, rng.permutation(nb * T)[:50])):
        n = len(slots)
        k, v = rows(int(slots[0]) + 50, n, H, D), rows(int(slots[0]) + 90, n, H, D, scale=0.1)
        fused = torch.zeros((n, 5 * H * D), dtype=torch.bfloat16, device=DEV)
        ks, vs = fused[:, H * D:2 * H * D].view(n, H, D), fused[:, 3 * H * D:4 * H * D].view(n, H, D)
        ks.copy_(k)
        vs.copy_(v)
        ops.quant_write_tokens(c, ks, vs, torch.from_numpy(slots.astype(np.int64)).to(DEV))
        ok = slots >= 0
        want_k[slots[ok]], want_v[slots[ok]] = k[ok], v[ok]
        same_rows(c, want_k.view(nb, T, H, D), want_v.view(nb, T, H, D), bits)
    torch.cuda.synchronize()
    assert _native.device_error() == 0


@pytest.mark.parametrize("bits", [4, 8])
def test_ties_flat_rows_and_extremes(bits):
    """Rows whose values fall on ties, constant rows, rows of zeros and negative zeros, the type's largest and smallest numbers."""
    from ucmx import ops
    D, T = 128, 16
    top = 2 ** bits - 1
    x = torch.zeros((1, T, 2, D), dtype=torch.float64)
    steps = torch.arange(D, dtype=torch.float64)
    x[0, 0, 0] = steps % (2 * top + 1) * 0.5                              # scale 1: every half step is a tie
    x[0, 1, 0] = (steps % (2 * top + 1) * 0.5 - top / 2) * 2.0 ** -7
    x[0, 2, 0] = 3.25
    x[0, 3, 0] = -0.0
    x[0, 4, 0, ::3] = 2.0 ** -133
    x[0, 5, 0] = (steps - 64) * 2.0 ** -133
    big = torch.finfo(torch.bfloat16).max
    x[0, 6, 0, 0], x[0, 6, 0, 1], x[0, 6, 0, 2] = big, -big, big / 3
    x[0, 7, 0, 5] = -big
    x[0, 8, 0] = torch.where(steps % 2 == 0, -top / 2 * 2.0 ** -4, top / 2 * 2.0 ** -4)
    x[0, 8, 0, 3:9] = torch.tensor([2.0 ** -40, -2.0 ** -40, 2.0 ** -30, -2.0 ** -30, 0.0, 2.0 ** -130], dtype=torch.float64)   # beside a tie
    x[0, 9, 0] = (steps - 60) * 1e-36
    g = torch.Generator().manual_seed(9)
    x[0, :, 1] = torch.randn((T, D), generator=g, dtype=torch.float64) * 10.0 ** torch.arange(-20, 12, 2)[:T, None]
    k = x.to(torch.bfloat16)
    v = k.flip(1)
    c = ops.QuantKvCache.alloc(1, T, 2, D, bits, DEV)
    ops.quant_write_blocks(c, k.to(DEV), v.contiguous().to(DEV), dev([0]))
    same_rows(c, k, v, bits)


@pytest.mark.parametrize("bits", [4, 8])
def test_a_million_random_values_round_as_defined(bits):
    from ucmx import ops
    for seed, scale in ((21, 1.0), (22, 1e-3)):
        k, v = rows(seed, 16, 128, 4, 128, scale=scale), rows(seed + 5, 16, 128, 4, 128)
        k[..., 0] *= 16                                                   # a channel that stands out
        c = ops.QuantKvCache.alloc(16, 128, 4, 128, bits, DEV)
        ops.quant_write_blocks(c, k.to(DEV), v.to(DEV), dev(range(16)))
        same_rows(c, k, v, bits)


def test_rows_with_infinities_or_nan_read_back_as_nan():
    from ucmx import ops
    k, v = rows(7, 2, 16, 2, 64), rows(8, 2, 16, 2, 64)
    k[0, 3, 1, 60], k[1, 0, 0, 0], v[0, 15, 0, 9] = float("nan"), float("inf"), -float("inf")
    c = ops.QuantKvCache.alloc(2, 16, 2, 64, 4, DEV)
    ops.quant_write_blocks(c, k.to(DEV), v.to(DEV), dev([0, 1]))
    same_rows(c, k, v, 4)
    kb, vb = (x.cpu() for x in ops.quant_read_blocks(c, dev([0, 1])))
    assert torch.equal(torch.isnan(kb).all(-1), ~torch.isfinite(k).all(-1)) and torch.equal(torch.isnan(kb).any(-1), ~torch.isfinite(k).all(-1))
    assert torch.equal(torch.isnan(vb).all(-1), ~torch.isfinite(v).all(-1))


def test_ids_beyond_the_caches_are_dropped_and_reported():
    from ucmx import _native, ops
    k, v = rows(10, 3, 16, 2, 64).to(DEV), rows(11, 3, 16, 2, 64).to(DEV)
    c = ops.QuantKvCache.alloc(3, 16, 2, 64, 8, DEV)
    _native.device_error()
    ops.quant_write_blocks(c, k, v, dev([0, 3, 2, -1]), out_slots=dev([0, 1, 7, 2]))
    torch.cuda.synchronize()
    assert _native.device_error() == 3
    assert bool(c.data[0].any()) and not bool(c.data[1:].any())
    ops.quant_write_tokens(c, k[1][:3], v[1][:3], torch.tensor([16, 48, 2 ** 40], device=DEV))
    torch.cuda.synchronize()
    assert _native.device_error() == 3
    same_rows(c, torch.cat([k[:1], k[1:2], k[:1]]).cpu(), torch.cat([v[:1], torch.zeros_like(v[1:2]), v[:1]]).cpu(), 8, where=(0,))
    kb, vb = torch.full_like(k, 5.0), torch.full_like(v, 5.0)
    ops.quant_read_blocks(c, dev([0, 3, 0]), k_out=kb, v_out=vb, out_slots=dev([2, 1, 3]))
    torch.cuda.synchronize()
    assert _native.device_error() == 3
    assert bool((kb[:2] == 5.0).all()) and not bool((kb[2] == 5.0).all())


def test_write_then_attend_then_move():
    """As they are used together: prefill blocks are quantised, decode tokens are appended, blocks move to another place as plain
    bytes, and the attention over the block table reads them there; pooled, scored and selected blocks go into the same call."""
    from ucmx import ops
    T, H, G, D, bits = 16, 2, 4, 128, 4
    n = 12
    k, v = rows(31, n, T, H, D), rows(32, n, T, H, D)
    c = ops.QuantKvCache.alloc(2 * n, T, H, D, bits, DEV)
    ops.quant_write_blocks(c, k.to(DEV), v.to(DEV), dev(range(n - 1)))
    ctx = (n - 1) * T
    q = rows(33, 1, H * G, D)
    for step in range(5):                                                  # the last block fills token by token
        slot = torch.tensor([ctx], device=DEV)
        ops.quant_write_tokens(c, k[n - 1, step:step + 1].to(DEV), v[n - 1, step:step + 1].to(DEV), slot)
        ctx += 1
    stage = torch.zeros((n, 1, c.block_bytes), dtype=torch.uint8, device=DEV)
    ops.gather_blocks([c.data], dev(range(n)), stage)
    moved = np.random.default_rng(3).permutation(np.arange(n, 2 * n))
    ops.scatter_blocks([c.data], dev(moved), stage)
    got = ops.quant_block_attention(q.to(DEV), c, dev([0, n]), positions=dev(range(n)), block_table=dev(moved), table_offsets=dev([0, n]),
                                    ctx_lens=dev([ctx]))
    kd, vd = R.values(R.pack(k, v, bits), D, bits)
    err = 12.0
    out, _, tol, _ = R.attend(q, kd, vd, [(range(1), [(i, i) for i in range(n)], ctx)], codes_err=err)
    R.check(got, out, tol)
    # pool -> score -> select the best blocks -> attend to them, in bf16 and over the codes
    kk, vv = k.to(DEV), v.to(DEV)
    reps = ops.pool_blocks(kk, dev(range(n)))
    off, per = dev([0, n]), dev([5])
    scores = ops.score_dot_query(reps, off, q.to(DEV), total=n, n_kv_heads=H)
    sel, _, cnt = ops.topk_ragged(scores, off, per, out_stride=8, order=ops.ORDER_INDEX_ASC)
    a = ops.block_attention(q.to(DEV), kk, vv, dev([0, 8]), positions=sel.view(-1), block_table=dev(range(n)), table_offsets=off, req_counts=cnt)
    b = ops.quant_block_attention(q.to(DEV), c, dev([0, 8]), positions=sel.view(-1), block_table=dev(moved), table_offsets=off, req_counts=cnt,
                                  ctx_lens=dev([ctx]))
    blocks = [(int(i), int(i)) for i in sel.view(-1)[:5].cpu()]
    out, _, tol, _ = R.attend(q, k.double(), v.double(), [(range(1), blocks, None)])
    R.check(a, out, tol)
    out, _, tol, _ = R.attend(q, kd, vd, [(range(1), blocks, ctx)], codes_err=err)
    R.check(b, out, tol)


@pytest.mark.parametrize("bits,D", FORMS)
@pytest.mark.parametrize("H", [1, 7])
def test_many_rows_at_once(bits, D, H):
    """Enough rows that a warp goes through several heads, of an odd number; blocks and tokens, and the way back."""
    from ucmx import _native, ops
    n, T = (160, 64) if H == 7 else (640, 64)
    k, v = rows(41, n, T, H, D), rows(42, n, T, H, D, scale=3.0)
    kd, vd = k.to(DEV), v.to(DEV)
    c = ops.QuantKvCache.alloc(n, T, H, D, bits, DEV)
    order = np.random.default_rng(5).permutation(n)
    ops.quant_write_blocks(c, kd, vd, dev(order), out_slots=dev(order))
    want = R.pack(k, v, bits)
    assert torch.equal(c.data.cpu(), want)
    t = ops.QuantKvCache.alloc(n, T, H, D, bits, DEV)
    slots = torch.arange(n * T, device=DEV)
    slots[5::1000] = -1
    ops.quant_write_tokens(t, kd.view(-1, H, D), vd.view(-1, H, D), slots)
    ops.quant_write_tokens(t, kd.view(-1, H, D)[5::1000], vd.view(-1, H, D)[5::1000], torch.arange(n * T, device=DEV)[5::1000].contiguous())
    assert torch.equal(t.data.cpu(), want)
    kb, vb = ops.quant_read_blocks(c, dev(order))
    torch.cuda.synchronize()
    assert _native.device_error() == 0
    for got, x in ((kb, k), (vb, v)):
        codes, scale, zero = R.to_codes(x[order], bits)
        assert torch.equal(got.cpu(), (codes.double() * scale + zero).float().to(torch.bfloat16))
