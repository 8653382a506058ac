"""Attention over listed blocks (bf16, 8-bit and 4-bit caches) against the plain 64-bit form: head layouts, block sizes, list forms,
contexts that end anywhere, several query tokens, and the places where such a kernel goes wrong."""
import numpy as np
import pytest
import torch

import attention_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def dev(a):
    return torch.as_tensor(np.asarray(a), dtype=torch.int32).to(DEV)


class Setup:
    """A cache of `fmt` bits (16: bf16) with random rows, and ragged lists over it."""

    def __init__(self, seed, fmt, H, G, D, T, counts, nq=None, pool=None, k_scale=1.0):
        g = torch.Generator().manual_seed(seed)
        self.fmt, self.H, self.G, self.D, self.T, self.counts = fmt, H, G, D, T, list(counts)
        total = sum(counts)
        self.pool = pool or total + 2
        k = (torch.randn((self.pool, T, H, D), generator=g) * k_scale).to(torch.bfloat16)
        v = torch.randn((self.pool, T, H, D), generator=g).to(torch.bfloat16)
        if fmt == 16:
            self.k16, self.v16 = k, v
            self.kd, self.vd = k.double(), v.double()
            self.err = 0.0
        else:
            self.data = R.pack(k, v, fmt)
            self.kd, self.vd = R.values(self.data, D, fmt)
            self.err = max(float((x.amax(-1) - x.amin(-1)).max()) for x in (self.kd, self.vd))     # codes and zero are up to a range apart
        self.off = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        self.ids = torch.randperm(max(self.pool, total), generator=g)[:total].numpy().astype(np.int32) % self.pool
        self.nq = list(nq) if nq is not None else [1] * len(counts)
        self.qoff = np.concatenate([[0], np.cumsum(self.nq)]).astype(np.int32)
        self.q = torch.randn((int(self.qoff[-1]), H * G, D), generator=g).to(torch.bfloat16)
        self.positions = None
        self.ctx = None
        self.rng = np.random.default_rng(seed)

    def spread(self):
        """Blocks from places of a longer sequence, ascending."""
        self.positions = np.concatenate([np.sort(self.rng.choice(4 * n + 3, n, replace=False)) for n in self.counts if n] or [[]]).astype(np.int32)
        return self

    def tails(self):
        """Contexts that end inside a request's last block."""
        last = [(self.positions[self.off[i + 1] - 1] if self.positions is not None else n - 1) if n else 0 for i, n in enumerate(self.counts)]
        self.ctx = np.asarray([int(l) * self.T + int(self.rng.integers(1, self.T + 1)) for l in last], np.int32)
        return self

    def lists(self):
        out = []
        for r, n in enumerate(self.counts):
            a = self.off[r]
            place = self.positions[a:a + n] if self.positions is not None else range(n)
            blocks = [(int(b), int(p)) for b, p in zip(self.ids[a:a + n], place) if b >= 0 and p >= 0]
            out.append((range(self.qoff[r], self.qoff[r + 1]), blocks, None if self.ctx is None else int(self.ctx[r])))
        return out

    def want(self, **kw):
        return R.attend(self.q, self.kd, self.vd, self.lists(), codes_err=self.err, **kw)

    def args(self, **kw):
        a = dict(block_ids=dev(self.ids), positions=None if self.positions is None else dev(self.positions),
                 ctx_lens=None if self.ctx is None else dev(self.ctx))
        if max(self.nq, default=1) > 1 or sum(self.nq) != len(self.counts):
            a.update(q_offsets=dev(self.qoff), max_q_tokens=max(self.nq))
        a.update(kw)
        return a

    def cache(self):
        from ucmx import ops
        if not hasattr(self, "dev_cache"):
            self.dev_cache = (self.k16.to(DEV), self.v16.to(DEV)) if self.fmt == 16 else (
                ops.QuantKvCache(self.data.to(DEV), head_dim=self.D, bits=self.fmt),)
        return self.dev_cache

    def run(self, q=None, offsets=None, **kw):
        from ucmx import ops
        f = ops.block_attention if self.fmt == 16 else ops.quant_block_attention
        return f(self.q.to(DEV) if q is None else q, *self.cache(), dev(self.off) if offsets is None else offsets, **self.args(**kw))

    def check(self, **kw):
        from ucmx import _native
        lse = torch.full((self.q.shape[0], self.q.shape[1]), 7.0, device=DEV)
        got = self.run(lse=lse, **kw)
        torch.cuda.synchronize()
        assert _native.device_error() == 0
        out, want_lse, tol, ltol = self.want()
        R.check(got, out, tol, "out")
        R.check(lse, want_lse, ltol, "lse")
        return got


SHAPES = [  # H, G, D, T, blocks of each request
    (2, 4, 128, 16, [3, 1, 7]),
    (1, 1, 128, 16, [1]),
    (2, 3, 64, 32, [2, 5]),
    (1, 8, 128, 64, [4, 1]),
    (2, 5, 64, 16, [9, 2]),
    (1, 16, 128, 16, [6, 3]),
    (1, 7, 256, 16, [3, 2]),
    (2, 2, 256, 32, [2, 1]),
    (1, 12, 256, 16, [2]),
    (1, 32, 64, 16, [3]),
    (1, 40, 64, 16, [3, 2]),
    (8, 4, 128, 128, [2, 1]),
]


@pytest.mark.parametrize("fmt", [16, 8, 4])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(map(str, s[:4])))
def test_whole_blocks(fmt, shape):
    H, G, D, T, counts = shape
    Setup(11, fmt, H, G, D, T, counts).check()


@pytest.mark.parametrize("fmt", [16, 8, 4])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(map(str, s[:4])))
def test_selected_blocks_with_ragged_ends(fmt, shape):
    H, G, D, T, counts = shape
    Setup(12, fmt, H, G, D, T, counts).spread().tails().check()


@pytest.mark.parametrize("fmt", [16, 8, 4])
@pytest.mark.parametrize("H,G,D,T,counts,nq", [
    (2, 4, 128, 16, [4, 2, 6], [3, 1, 2]),          # 12 columns: a tile of 16
    (1, 1, 64, 32, [2, 3], [4, 2]),                 # four columns, a request with fewer
    (1, 2, 128, 16, [5], [37]),                     # 74 columns: three tiles of 32
    (1, 8, 256, 16, [3, 2], [5, 1]),                # 40 columns, tiles of 16
    (2, 7, 64, 64, [1, 2], [3, 2]),
])
def test_several_query_tokens(fmt, H, G, D, T, counts, nq):
    s = Setup(13, fmt, H, G, D, T, counts, nq)
    s.tails().check()
    s.ctx = np.asarray([(n - 1) * T + 1 for n in counts], np.int32)      # the last token opens its block: earlier queries end before it
    s.check()
    s.ctx = np.asarray([max(1, q - 2) for q in nq], np.int32)            # fewer tokens than queries: the first ones see nothing
    s.check()


@pytest.mark.parametrize("T", [1, 3, 5, 8, 17, 24, 100])
def test_any_block_size(T):
    Setup(14, 16, 2, 4, 128, T, [5, 1, 3]).tails().check()
    Setup(15, 16, 1, 6, 64, T, [4, 2], [2, 1]).spread().tails().check()


@pytest.mark.parametrize("fmt", [16, 4])
def test_empty_requests_and_contexts_of_zero_and_one(fmt):
    s = Setup(16, fmt, 2, 4, 128, 16, [0, 3, 0, 0, 2, 1, 0])
    s.check()
    s.ctx = np.asarray([5, 0, 0, 16, 1, 17, 1], np.int32)
    got = s.check()
    assert not bool(got[[0, 1, 2, 3, 6]].any())
    Setup(17, fmt, 1, 4, 128, 16, [0, 0]).check()                         # nothing at all
    Setup(17, fmt, 1, 4, 128, 16, [0], [3], pool=2).tails().check()


@pytest.mark.parametrize("fmt", [16, 8, 4])
def test_skipped_counted_and_repeated_entries(fmt):
    from ucmx import _native
    s = Setup(18, fmt, 2, 4, 128, 32, [5, 4, 6]).spread()
    s.ids[[1, 4, 9]] = -1
    s.positions[6] = -3
    s.ids[12] = s.ids[11]                                                 # the same block twice counts twice
    s.check()
    full_ids = s.ids.copy()
    s.ids[[2, 3, 4, 5, 6, 7, 8]] = -1                                     # what counts [2, 0, 6] leaves
    want = s.want()
    s.ids = full_ids
    _native.device_error()
    got = s.run(req_counts=dev([2, 0, 6]))
    R.check(got, want[0], want[2])
    assert _native.device_error() == 0


def test_ids_beyond_the_cache_or_the_table_are_dropped_and_reported():
    from ucmx import _native
    for fmt in (16, 4):
        s = Setup(19, fmt, 2, 4, 128, 16, [6, 5])
        keep = s.ids.copy()
        s.ids[[1, 7]] = -1
        want = s.want()
        s.ids = keep.copy()
        s.ids[1], s.ids[7] = s.pool, 2_000_000_000
        _native.device_error()
        got = s.run()
        torch.cuda.synchronize()
        assert _native.device_error() == 3
        R.check(got, want[0], want[2])
        # through a block table: places beyond a request's row of it
        s.ids = keep.copy()
        order = np.asarray([5, 0, 9, 2, 4, 1, 3, 0, 5, 4, 1], np.int32)
        s.positions = order
        table = keep
        s.ids = np.asarray([table[p] if p < 6 else -1 for p in order[:6]] + [table[6 + p] if p < 5 else -1 for p in order[6:]], np.int32)
        want = s.want()
        got = s.run(block_ids=None, block_table=dev(table), table_offsets=dev(s.off))
        torch.cuda.synchronize()
        assert _native.device_error() == 3
        R.check(got, want[0], want[2])


@pytest.mark.parametrize("fmt", [16, 8, 4])
def test_what_is_not_seen_may_be_anything(fmt):
    """NaN and infinities in tokens behind the context, and in blocks that nobody lists, reach no result."""
    s = Setup(20, fmt, 2, 4, 128, 32, [3, 2, 4], [1, 3, 2]).tails()
    seen = np.zeros((s.pool, s.T), bool)
    for rows, blocks, ctx in s.lists():
        for b, p in blocks:
            seen[b] |= p * s.T + np.arange(s.T) < ctx
    hide = torch.from_numpy(~seen)
    assert bool(hide.any())
    if fmt == 16:
        s.k16[hide], s.v16[hide] = float("inf"), float("nan")
    else:
        for b, t in hide.nonzero().tolist():
            p = 32 * (s.D * fmt // 8) + (t % 16) * 4
            s.data[b, :, t // 16, p:p + 4] = 255                          # a NaN for the scale and the zero
            s.data[b, :, t // 16, p + 64:p + 68] = 255
    s.check()


@pytest.mark.parametrize("fmt", [16, 8, 4])
@pytest.mark.parametrize("G,nq", [(1, 3), (4, 3), (4, 6), (2, 2)])
def test_a_bad_row_stays_with_the_queries_that_see_it(fmt, G, nq):
    """The last token's V row is NaN (and an infinity): the last query's result is, the earlier queries' are not."""
    s = Setup(21, fmt, 2, G, 128, 16, [3, 2], [nq, nq])
    s.ctx = np.asarray([3 * 16 - 5, 2 * 16], np.int32)
    for r, (rows, blocks, ctx) in enumerate(s.lists()):
        b, t = blocks[(ctx - 1) // 16][0], (ctx - 1) % 16
        if fmt == 16:
            s.v16[b, t, :, 5] = float("inf")
            s.v16[b, t, 1] = float("nan")
        else:
            p = 32 * (s.D * fmt // 8) + 64 + (t % 16) * 4
            s.data[b, :, t // 16, p:p + 4] = 255
    if fmt == 16:
        s.vd = s.v16.double()
        out, _, tol, _ = s.want()
        got = s.run().cpu().double()
        for rows, _, _ in s.lists():
            early, last = list(rows)[:-1], rows[-1]
            R.check(got[early], out[early], tol[early])
            assert bool(torch.isnan(got[last, G:]).all()) and not bool(torch.isfinite(got[last, :G, 5]).any())
            fine = [d for d in range(128) if d != 5]
            R.check(got[last, :G][:, fine], out[last, :G][:, fine], tol[last, :G][:, fine])
    else:
        s.vd = R.values(s.data, s.D, fmt)[1]
        s.err = 20.0                                                      # (the range of a NaN row says nothing)
        out, _, tol, _ = s.want()
        R.check(s.run(), out, tol)
        assert bool(torch.isnan(out).any())


def test_a_nan_that_is_seen_is_not_lost():
    for fmt in (16, 4):
        s = Setup(22, fmt, 2, 4, 128, 16, [40, 3])
        b = int(s.ids[31])
        if fmt == 16:
            s.k16[b, 3, 1, 7] = float("nan")
        else:
            s.data[b, 1, 0, 32 * 64 + 3 * 4:32 * 64 + 3 * 4 + 4] = 255
        got = s.run().cpu()
        assert bool(torch.isnan(got[0, 4:]).all()) and not bool(torch.isnan(got[0, :4]).any()) and not bool(torch.isnan(got[1]).any())


@pytest.mark.parametrize("fmt", [16, 8, 4])
@pytest.mark.parametrize("scale", [0.0, -0.3, 4.0])
def test_scales_and_large_scores(fmt, scale):
    """scale 4 gives scores of hundreds: one token takes all the weight, the running maximum moves a long way."""
    from ucmx import _native
    s = Setup(23, fmt, 2, 4, 128, 16, [9, 60], k_scale=3.0)
    lse = torch.empty((2, 8), device=DEV)
    got = s.run(scale=scale, lse=lse)
    out, wl, tol, ltol = s.want(scale=scale)
    R.check(got, out, tol)
    R.check(lse, wl, ltol)
    assert _native.device_error() == 0


@pytest.mark.parametrize("fmt", [16, 8, 4])
def test_long_lists_are_split_and_joined_in_order(fmt):
    """One long request beside short ones: the long one is cut over many thread blocks.  Twice the same bits; any order of the
    requests gives a request the same result to rounding."""
    s = Setup(24, fmt, 2, 4, 128, 16, [1, 1500, 3, 0, 700]).tails()
    a = s.check()
    b = s.run()
    assert torch.equal(a.view(torch.int16), b.view(torch.int16))
    Setup(25, fmt, 1, 16, 64, 16, [900], [3]).tails().check()
    Setup(26, fmt, 1, 3, 256, 16, [500, 2]).check()
    Setup(27, fmt, 4, 8, 128, 16, [300, 301, 299]).spread().tails().check()


def test_many_requests():
    n = 1500                                                               # more requests than thread blocks, many without blocks
    rng = np.random.default_rng(5)
    counts = [int(x) for x in rng.integers(0, 3, n)]
    Setup(28, 16, 1, 2, 64, 16, counts).check()
    Setup(29, 4, 1, 2, 64, 16, counts).tails().check()


def test_strided_queries_and_caches():
    """Queries inside a fused projection's rows; K and V of a block side by side; blocks of a wider allocation."""
    from ucmx import ops
    s = Setup(30, 16, 2, 4, 128, 16, [5, 3, 2])
    wide = torch.randn((3, 8 * 128 + 4 * 128), device=DEV).to(torch.bfloat16)
    qs = wide[:, :8 * 128].view(3, 8, 128)
    qs.copy_(s.q)
    both = torch.randn((s.pool, 2, s.T, 2, 128), device=DEV).to(torch.bfloat16)
    both[:, 0], both[:, 1] = s.k16.to(DEV), s.v16.to(DEV)
    out, _, tol, _ = s.want()
    R.check(ops.block_attention(qs, both[:, 0], both[:, 1], dev(s.off), **s.args()), out, tol)
    padded = torch.randn((s.pool, s.T, 3, 128), device=DEV).to(torch.bfloat16)
    padded[:, :, :2] = s.k16.to(DEV)
    R.check(ops.block_attention(qs, padded[:, :, :2], both[:, 1], dev(s.off), **s.args()), out, tol)
    f = Setup(31, 4, 2, 4, 128, 32, [5, 3, 2])
    store = torch.zeros((f.pool, f.data[0].numel() + 64), dtype=torch.uint8, device=DEV)
    view = store[:, :f.data[0].numel()].view(f.data.shape)
    view.copy_(f.data)
    out, _, tol, _ = f.want()
    R.check(ops.quant_block_attention(f.q.to(DEV), ops.QuantKvCache(view, head_dim=128, bits=4), dev(f.off), **f.args()), out, tol)


def test_rows_behind_the_last_request_stay_as_they_are():
    for fmt in (16, 8):
        s = Setup(32, fmt, 2, 4, 128, 16, [4, 0, 2], [2, 1, 3]).tails()
        q = torch.cat([s.q, torch.full((5, 8, 128), float("nan"), dtype=torch.bfloat16)]).to(DEV)
        out = torch.full((11, 8, 128), 3.0, dtype=torch.bfloat16, device=DEV)
        lse = torch.full((11, 8), 3.0, device=DEV)
        s.run(q=q, out=out, lse=lse)
        w = s.want()
        R.check(out[:6], w[0], w[2])
        assert bool((out[6:] == 3.0).all()) and bool((lse[6:] == 3.0).all())


@pytest.mark.parametrize("fmt", [16, 4])
def test_captured_and_replayed_with_other_lists(fmt):
    """A graph captured at its capacity is replayed with shorter lists, other contexts and another split."""
    s = Setup(33, fmt, 2, 4, 128, 16, [60, 200, 40, 10]).tails()
    cap = 400
    ids = torch.full((cap,), 1_000_000, dtype=torch.int32, device=DEV)    # what lies behind the lists is not read
    ids[:310] = dev(s.ids)
    off, ctx, q = dev(s.off), dev(s.ctx), s.q.to(DEV)
    out = torch.zeros((4, 8, 128), dtype=torch.bfloat16, device=DEV)
    from ucmx import _native, ops
    ws = ops.attention_workspace(q, 2, bits=fmt)
    f = ops.block_attention if fmt == 16 else ops.quant_block_attention
    cache = s.cache()
    f(q, *cache, off, block_ids=ids, ctx_lens=ctx, out=out, workspace=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        f(q, *cache, off, block_ids=ids, ctx_lens=ctx, out=out, workspace=ws)
    for seed, counts in ((34, [60, 200, 40, 10]), (35, [1, 3, 0, 90]), (36, [0, 0, 0, 1]), (37, [100, 100, 100, 100])):
        t = Setup(33, fmt, 2, 4, 128, 16, [60, 200, 40, 10])
        rng = np.random.default_rng(seed)
        t.counts, t.off = counts, np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        t.ids = rng.integers(0, t.pool, sum(counts)).astype(np.int32)
        t.tails()
        ids.fill_(1_000_000)
        ids[:len(t.ids)] = dev(t.ids)
        off.copy_(dev(t.off))
        ctx.copy_(dev(t.ctx))
        ws.fill_(255)                                                     # the workspace may hold anything
        graph.replay()
        torch.cuda.synchronize()
        w = t.want()
        R.check(out, w[0], w[2])
        assert _native.device_error() == 0


def test_two_streams_with_workspaces_of_their_own():
    s, t = (Setup(seed, fmt, 2, 4, 128, 16, [300, 20, 500]) for seed, fmt in ((38, 16), (39, 4)))
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    s.cache(), t.cache(), s.run(), t.run()
    torch.cuda.synchronize()
    outs = []
    for _ in range(5):
        with torch.cuda.stream(a):
            outs.append((s, s.run()))
        with torch.cuda.stream(b):
            outs.append((t, t.run()))
    torch.cuda.synchronize()
    wants = {id(x): x.want() for x in (s, t)}
    for x, got in outs:
        R.check(got, wants[id(x)][0], wants[id(x)][2])


def test_offsets_beyond_32_bits():
    """A cache of more than 2^32 bytes and 2^31 elements: the blocks at its end are the ones read."""
    from ucmx import ops
    T, H, D = 128, 8, 128
    per = T * H * D
    nb = 2 ** 31 // per + 40
    k = torch.zeros((nb, T, H, D), dtype=torch.bfloat16, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(3)
    used = [nb - 1, 0, nb - 7, nb - 30]
    for b in used:
        k[b] = torch.randn((T, H, D), generator=g, device=DEV).to(torch.bfloat16)
    q = torch.randn((1, 8, D), generator=g, device=DEV).to(torch.bfloat16)
    got = ops.block_attention(q, k, k, dev([0, 4]), block_ids=dev(used), ctx_lens=dev([4 * T - 3]))
    small = k[torch.tensor(used, device=DEV)].cpu().double()
    out, _, tol, _ = R.attend(q.cpu(), small, small, [(range(1), [(i, i) for i in range(4)], 4 * T - 3)])
    R.check(got, out, tol)
    del k
    nb = 2 ** 32 // 1088 // 4 + 50                                        # 4-bit, 64 values a head, 4 heads, T 16
    c = ops.QuantKvCache.alloc(nb, 16, 4, 64, 4, DEV)
    assert c.data.numel() > 2 ** 32
    x, y = (torch.randn((4, 16, 4, 64), generator=g, device=DEV).to(torch.bfloat16) for _ in range(2))
    used = [nb - 2, 1, nb - 1, nb - 40]
    ops.quant_write_blocks(c, x, y, dev([0, 1, 2, 3]), out_slots=dev(used))
    q = torch.randn((1, 8, 64), generator=g, device=DEV).to(torch.bfloat16)
    got = ops.quant_block_attention(q, c, dev([0, 4]), block_ids=dev(used))
    kd, vd = R.values(c.data[torch.tensor(used, device=DEV)].cpu(), 64, 4)
    out, _, tol, _ = R.attend(q.cpu(), kd, vd, [(range(1), [(i, i) for i in range(4)], None)], codes_err=8.0)
    R.check(got, out, tol)


@pytest.mark.parametrize("fmt", [16, 8])
def test_lists_inside_larger_arrays(fmt):
    """Some of a batch's requests, by a piece of its offsets: entries, tables and offsets stay where they are."""
    s = Setup(50, fmt, 2, 4, 128, 16, [4, 70, 5, 0, 40, 3]).tails()
    w = s.want()
    got = s.run(q=s.q[1:5].to(DEV), offsets=dev(s.off[1:6]), ctx_lens=dev(s.ctx[1:5]))
    R.check(got, w[0][1:5], w[2][1:5])
    t = Setup(51, fmt, 1, 8, 64, 32, [9, 30, 2], [2, 5, 3]).tails()      # with several tiles of columns
    w = t.want()
    qo = t.qoff[1:] - t.qoff[1]
    got = t.run(q=t.q[2:].to(DEV), offsets=dev(t.off[1:]), ctx_lens=dev(t.ctx[1:]), q_offsets=dev(qo), max_q_tokens=5)
    R.check(got, w[0][2:], w[2][2:])


@pytest.mark.parametrize("nq", [1, 5])
def test_offsets_that_do_not_ascend_are_reported(nq):
    """They index nothing outside the lists, the call ends and says so, and the next one is fine."""
    from ucmx import _native
    s = Setup(52, 16, 2, 8, 64, 16, [6, 90, 4, 8], [nq] * 4).tails()
    _native.device_error()
    for off in ([0, 6, 3, 90, 40], [0, 108, 0, 108, 0], [50, 40, 30, 20, 10], [0, 2_000_000_000, -5, 7, 108], [0, 6, 200, 100, 108]):
        s.run(offsets=dev(off))
        torch.cuda.synchronize()
    assert _native.device_error() == 3
    s.check()


def test_a_table_that_ends_early_is_reported():
    from ucmx import _native
    s = Setup(53, 4, 2, 4, 128, 16, [6, 5])
    table = s.ids.copy()
    place = np.asarray([0, 5, 2, 4, 1, 3, 0, 4, 2, 1, 3], np.int32)
    s.positions = place
    s.ids = np.asarray([table[p] for p in place[:6]] + [table[6 + p] if 6 + p < 9 else -1 for p in place[6:]], np.int32)
    w = s.want()
    _native.device_error()
    got = s.run(block_ids=None, block_table=dev(table[:9]), table_offsets=dev(s.off))
    torch.cuda.synchronize()
    assert _native.device_error() == 3
    R.check(got, w[0], w[2])


@pytest.mark.parametrize("fmt", [16, 4])
def test_several_tiles_of_columns(fmt):
    """More requests than are counted one by one; tiles of 32; tiles that are cut over many thread blocks."""
    rng = np.random.default_rng(60)
    n = 1100
    Setup(61, fmt, 1, 8, 64, 16, [int(x) for x in rng.integers(0, 3, n)], [int(x) for x in rng.integers(1, 7, n)]).tails().check()
    Setup(62, fmt, 2, 8, 128, 16, [300, 5, 120], [4, 8, 1]).tails().check()
    Setup(63, fmt, 1, 8, 256, 16, [400, 3], [5, 2]).tails().check()
    Setup(64, fmt, 2, 16, 64, 16, [250, 9], [3, 4]).spread().tails().check()


@pytest.mark.parametrize("fmt", [8, 4])
@pytest.mark.parametrize("T,H", [(16, 1), (16, 2), (32, 1)])
def test_blocks_that_follow_one_another_in_memory(fmt, T, H):
    """Neighbouring blocks in every place of a list: two slices are copied at once only where they are the ones wanted."""
    for seed in range(6):
        s = Setup(70 + seed, fmt, H, 4, 64, T, [40, 17], pool=200)
        rng = np.random.default_rng(seed)
        ids = rng.permutation(200)[:57]
        for i in rng.permutation(50)[:30]:
            ids[i + rng.integers(1, 8)] = (ids[i] + 1) % 200               # follows the block a few places before it
        if seed == 0:
            ids = np.arange(57)
        s.ids = ids.astype(np.int32)
        s.check()


@pytest.mark.parametrize("fmt", [16, 4])
@pytest.mark.parametrize("G,D", [(1, 64), (3, 128), (7, 128), (2, 256), (13, 64), (16, 128), (20, 256), (33, 64)])
def test_parts_by_the_hundred_are_joined(fmt, G, D):
    """One KV head and one long request: more parts than a warp has lanes, in each width of tile; contexts that leave the later parts
    empty, or all of them; a shorter request whose few parts are joined another way."""
    s = Setup(70, fmt, 1, G, D, 16, [1500, 90]).tails()
    s.check()
    for ctx in ([700 * 16 + 5, 41], [3, 0], [0, 90 * 16]):
        s.ctx = np.asarray(ctx, np.int32)
        s.check()


@pytest.mark.parametrize("fmt", [16, 4])
def test_a_workspace_whose_bytes_are_not_its_own_is_refused(fmt):
    s = Setup(71, fmt, 1, 2, 64, 16, [2])
    with pytest.raises(ValueError):
        s.run(workspace=torch.zeros(1, dtype=torch.uint8, device=DEV).expand(1 << 26))
    s.check()
