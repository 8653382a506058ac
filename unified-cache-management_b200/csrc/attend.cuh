// Attention of a ragged batch of queries over listed KV blocks: the kernel shared by the bf16 cache (attend.cu) and the
// quantised cache (attend_quant.cu).
//
//   out[c] = sum_t softmax_t(scale * q_c . k_t) v_t        over the tokens t of the request's listed blocks that c may see
//
// Shape of the work.  Few query rows (query heads of one KV head x query tokens of the request: the "columns") meet
// thousands of cached tokens, so the kernel is a stream over K and V: every listed token is read once per KV head and
// column tile, and everything else stays in registers.  The matrix instructions take TOKENS as their 16 rows and the
// columns as their 8 wide side (S^T = K Q^T, O^T = V^T P^T): 4 to 8 query heads per KV head then waste little, K and V
// are the wide operand straight from shared memory, and one column's softmax statistics live in one register per thread.
//
// Split.  The unit is a slice: up to 16 consecutive tokens of one listed block.  All slices of all (request, KV head,
// column tile) items are laid end to end and cut into equal parts, one per thread block, whatever the lengths of the
// requests are; an item that crosses cuts leaves partial results (running maximum, sum, unnormalised output) in the
// workspace, which a second small kernel joins in order.  The workspace needs no initial state, and the order of the
// sums is fixed by the shapes, so results do not change from run to run.
//
// Within a thread block each of the four warps takes every fourth slice with a ring of its own: one lane per row starts
// an asynchronous bulk copy, the warp waits on its own barrier, no other warp is involved until the item ends.
//
// Rounding.  Scores, maxima, sums and outputs are fp32.  The weights are the one operand that has to become bf16 for
// the second product; each is split into a bf16 value and the bf16 of what is left (2^-17 relative instead of 2^-9,
// which would be as large an error as the final rounding of the output).  With at most four columns the two halves
// share one instruction (columns 4..7 repeat 0..3), otherwise they are two.
#pragma once

#include "common.cuh"

namespace ucmx {
namespace attend {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kRows = 16;              // tokens of a slice
constexpr float kLn2 = 0.69314718055994531f;
constexpr float kLog2e = 1.4426950408889634f;
// A column's running maximum is only moved when a score passes it by this much (in powers of two): weights stay below
// 2^8, and most slices need neither the reduction over the warp nor the rescaling.
constexpr float kMaxSlack = 8.0f;

struct Params {
    const uint16_t* q;
    int64_t q_stride;                  // elements between query tokens
    const int32_t* q_offsets;          // [n_req+1] or NULL: one query token per request
    int32_t n_q_tokens, max_q;
    int32_t Hq, H, G;                  // query heads, KV heads, Hq / H
    const uint8_t* k;                  // bf16: K cache; quantised: the cache
    const uint8_t* v;
    int64_t k_block, v_block;          // bytes between blocks
    int64_t k_token, v_token;          // bytes between tokens (bf16)
    int32_t T, spe;                    // tokens per block, slices per block
    int64_t n_blocks;
    const int32_t* offsets;            // [n_req+1] into the lists
    const int32_t* counts;             // [n_req] or NULL
    const int32_t* block_ids;          // [total] or NULL: table[table_offsets[r] + position]
    const int32_t* positions;          // [total] or NULL: the i-th entry of a request stands at i
    const int32_t* table;
    const int32_t* table_offsets;      // [n_req+1]
    const int32_t* ctx;                // [n_req] or NULL
    int32_t n_req, total;
    int32_t col_tiles, cols_per_tile;
    float scale_log2;
    uint16_t* out;                     // [n_q_tokens, Hq, D]
    float* lse;                        // [n_q_tokens, Hq] or NULL
    float* ws;                         // partial results: 2 per thread block
    int32_t* err;
};

// One item's part inside a thread block's range.
struct Seg {
    int64_t begin, end;                // of the whole item, in the order of all slices
    int64_t lo, hi;                    // the part of it
    int32_t r, h, ct;
    int32_t first;                     // offsets[r]
    int32_t n;                         // entries of the request's list
};

// The last r with offsets[r] <= e (a warp probes 32 places at a time).  All lanes get it.
__device__ __forceinline__ int request_of(const int32_t* __restrict__ offsets, int n_req, int64_t e)
{
    const int lane = threadIdx.x & 31;
    int lo = 0, n = n_req;
    while (n > 1) {
        const int step = (n + 31) >> 5;
        const int at = lo + lane * step;
        const bool below = lane * step < n && (int64_t)__ldg(offsets + at) <= e;
        const int c = __popc(__ballot_sync(0xffffffffu, below));
        const int adv = (c > 0 ? c - 1 : 0) * step;
        lo += adv;
        n = min(step, n - adv);
    }
    return lo;
}

__device__ __forceinline__ int64_t entries_total(const Params& p)
{
    const int32_t n = __ldg(p.offsets + p.n_req);      // a captured batch may use less than its capacity
    return n < 0 ? 0 : n < p.total ? n : p.total;
}
__device__ __forceinline__ int64_t slices_per_entry(const Params& p) { return (int64_t)p.spe * p.H * p.col_tiles; }

__device__ __forceinline__ int64_t cut(int64_t all, int c, int n) { return all / n * c + all % n * c / n; }

// The item that holds position `at` (< hi); called by whole warps.
__device__ __forceinline__ Seg segment_at(const Params& p, int64_t at, int64_t hi)
{
    Seg s;
    const int64_t spe = slices_per_entry(p);
    s.r = request_of(p.offsets, p.n_req, at / spe);
    s.first = __ldg(p.offsets + s.r);
    s.n = min(__ldg(p.offsets + s.r + 1), p.total) - s.first;
    const int64_t item = (int64_t)s.n * p.spe;         // slices of one (KV head, column tile)
    const int64_t rel = at - (int64_t)s.first * spe;
    const int32_t i = (int32_t)(rel / item);
    s.h = i / p.col_tiles;
    s.ct = i - s.h * p.col_tiles;
    s.begin = (int64_t)s.first * spe + (int64_t)i * item;
    s.end = s.begin + item;
    s.lo = at;
    s.hi = s.end < hi ? s.end : hi;
    return s;
}

// Query rows of request r: first row and how many (clamped to the query tensor and to max_q).
__device__ __forceinline__ void queries_of(const Params& p, int r, int& q0, int& nq)
{
    if (p.q_offsets == nullptr) {
        q0 = r;
        nq = r < p.n_q_tokens ? 1 : 0;
        return;
    }
    q0 = __ldg(p.q_offsets + r);
    nq = __ldg(p.q_offsets + r + 1) - q0;
    if (q0 < 0 || nq < 0 || nq > p.max_q || q0 + (int64_t)nq > p.n_q_tokens) {
        if (p.err && threadIdx.x == 0) atomicExch(p.err, 3);
        nq = q0 < 0 || q0 >= p.n_q_tokens ? 0 : max(0, min(min(nq, p.max_q), p.n_q_tokens - q0));
    }
}

__device__ __forceinline__ float exp2_fast(float x) { return exp2f(x); }

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_trans(uint32_t (&r)[4], uint32_t addr)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x)
{
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi)
{
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ uint32_t sub_bf16x2(uint32_t a, uint32_t b)
{
    uint32_t r;
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ uint4 lds16(uint32_t a)
{
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ uint2 lds8(uint32_t a)
{
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t lds4(uint32_t a)
{
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
}

// Codes to centred integers in bf16 (exact): 4 bits: c - 8, two per register from bits [4i, 4i+4) of both halves.
// 0x4300 is 128.0 and a bf16 of that size counts in ones, so or-ing the code in adds it.
__device__ __forceinline__ uint32_t nibbles(uint32_t w, int i)
{
    return sub_bf16x2(((w >> (4 * i)) & 0x000f000fu) | 0x43004300u, 0x43084308u);
}
// 8 bits: c - 128 from bytes i and i+2.  The low seven bits are or-ed into 128.0; the top bit chooses what is taken off:
// 256.0 (0x4380) where it is clear, 128.0 (0x4300) where it is set.
__device__ __forceinline__ uint32_t bytes(uint32_t w, int i)
{
    const uint32_t x = w >> (8 * i);
    return sub_bf16x2((x & 0x007f007fu) | 0x43004300u, (~x & 0x00800080u) | 0x43004300u);
}

// FMT 16: bf16 cache, rows of K and V; 8 or 4: groups of the quantised cache.
template <int FMT, int D>
struct Layout {
    static constexpr int kRowBytes = D * FMT / 8;
    static constexpr int kPanel = FMT == 16 ? kRowBytes : kRowBytes < 64 ? kRowBytes : 64;   // bytes of a row in a panel
    static constexpr int kPanels = kRowBytes / kPanel;
    static constexpr int kPanelDims = D / kPanels;
    static constexpr int kGroup = 2 * kRows * kRowBytes + 2 * kRows * 4;  // quantised: codes of K and V, then their scales
    static constexpr int kRowStride = kRowBytes + 16;                     // bf16: rows in shared memory, off the bank period
    static constexpr int kStage = FMT == 16 ? 2 * kRows * kRowStride : kGroup;
    static constexpr int kStages = kStage > 8400 && D == 256 ? 2 : kStage > 8000 && FMT != 16 ? 2 : kStage > 4000 ? 3 : 4;
};

template <int FMT, int D, int NT, bool DUP>
struct Traits {
    using L = Layout<FMT, D>;
    static constexpr int kCols = DUP ? 4 : 8 * NT;       // columns of a tile
    static constexpr int kKSteps = D / 16;
    static constexpr int kMTiles = D / 16;
    static constexpr bool kQReg = kKSteps * NT <= 16;    // query fragments in registers (else in shared memory)
    static constexpr int kMergeLd = D + 4;
    static constexpr int kMergeCols = 4;                 // columns joined at a time
    static constexpr int kMergeSteps = DUP ? 1 : 2 * NT;
    static constexpr int kRingBytes = kWarps * L::kStages * L::kStage;
    static constexpr int kMergeBytes = kWarps * kMergeCols * kMergeLd * 4;
    static constexpr int kStatBytes = kWarps * kCols * 3 * 4;
    static constexpr int kQBytes = kQReg ? 0 : kKSteps * NT * 32 * 8;
    static constexpr int kBarBytes = 16 * kWarps * L::kStages;            // a barrier (8) and the stage's note (8)
    static constexpr int kSmem = kRingBytes + kMergeBytes + kStatBytes + kQBytes + kBarBytes;
    static constexpr int kPart = kCols * (D + 2);        // floats of a partial result: m, l, then the rows
    // thread blocks per SM: what shared memory holds (228 KB, 1 KB of it per block), and the registers of the accumulators
    static constexpr int kBySmem = 233472 / (kSmem + 1024);
    static constexpr int kByRegs = D * NT <= 128 ? 4 : 2;
    static constexpr int kOcc = kBySmem < 1 ? 1 : kBySmem < kByRegs ? kBySmem : kByRegs;
};

template <int FMT, int D, int NT, bool DUP>
__global__ void __launch_bounds__(kThreads, Traits<FMT, D, NT, DUP>::kOcc) attend_kernel(const Params p)
{
    using X = Traits<FMT, D, NT, DUP>;
    using L = typename X::L;
    extern __shared__ __align__(128) unsigned char smem[];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = lane >> 2, q4 = lane & 3;

    unsigned char* const ring = smem + warp * (L::kStages * L::kStage);
    float* const merge = reinterpret_cast<float*>(smem + X::kRingBytes);
    float* const stat = reinterpret_cast<float*>(smem + X::kRingBytes + X::kMergeBytes);     // [warp][3][cols]
    uint2* const q_frag = reinterpret_cast<uint2*>(smem + X::kRingBytes + X::kMergeBytes + X::kStatBytes);
    unsigned char* const bars = smem + X::kRingBytes + X::kMergeBytes + X::kStatBytes + X::kQBytes + warp * (16 * L::kStages);
    uint64_t* const full = reinterpret_cast<uint64_t*>(bars);
    int2* const note = reinterpret_cast<int2*>(bars + 8 * L::kStages);    // .x tokens copied (0: nothing), .y first position

    if (lane == 0) {
        for (int s = 0; s < L::kStages; ++s) mbar_init(&full[s], 1);
        mbar_init_fence();
    }
    __syncwarp();

    const int64_t all = entries_total(p) * slices_per_entry(p);
    const int64_t lo = cut(all, blockIdx.x, gridDim.x), hi = cut(all, blockIdx.x + 1, gridDim.x);
    early_start_allow();

    // requests that list nothing have no slices: their rows are written here
    for (int r = blockIdx.x; r < p.n_req; r += gridDim.x) {
        if (__ldg(p.offsets + r + 1) > __ldg(p.offsets + r) && __ldg(p.offsets + r) < p.total) continue;
        int q0, nq;
        queries_of(p, r, q0, nq);
        for (int64_t i = tid; i < (int64_t)nq * p.Hq * (D / 2); i += kThreads)
            reinterpret_cast<uint32_t*>(p.out)[(int64_t)q0 * p.Hq * (D / 2) + i] = 0u;
        if (p.lse)
            for (int i = tid; i < nq * p.Hq; i += kThreads) p.lse[(int64_t)q0 * p.Hq + i] = -INFINITY;
    }
    if (lo >= hi) return;

    // ---- the warp's loads run ahead of its arithmetic, across items: a cursor of their own
    Seg ps;
    ps.hi = -1;
    int64_t p_at = 0;                  // next slice to load of segment ps
    int64_t p_batch = 0;               // lane i knows slice p_batch + 4 i
    int32_t my_id = -1, my_nv = 0, my_pos = 0;
    int32_t p_sub = 0;                 // first token of my slice inside its block
    bool p_done = false;
    int64_t p_next = lo;               // where the next segment begins

    // what this lane has to know of slice `at` of segment ps
    auto look_up = [&](int64_t at) {
        my_id = -1;
        my_nv = 0;
        if (at >= ps.hi) return;
        const int32_t s = (int32_t)(at - ps.begin);
        const int32_t e = s / p.spe, sub = s - e * p.spe;
        p_sub = sub * kRows;
        int32_t cnt = ps.n;
        if (p.counts) cnt = min(cnt, __ldg(p.counts + ps.r));
        if (e >= cnt) return;
        const int32_t at_list = ps.first + e;
        const int32_t pos_block = p.positions ? __ldg(p.positions + at_list) : e;
        if (pos_block < 0) return;
        int32_t id;
        if (p.block_ids) {
            id = __ldg(p.block_ids + at_list);
        } else {
            const int32_t t0 = __ldg(p.table_offsets + ps.r), t1 = __ldg(p.table_offsets + ps.r + 1);
            if (pos_block >= t1 - t0) {
                if (p.err) atomicExch(p.err, 3);
                return;
            }
            id = __ldg(p.table + t0 + pos_block);
        }
        if (id < 0) return;
        if ((int64_t)id >= p.n_blocks) {
            if (p.err) atomicExch(p.err, 3);
            return;
        }
        int32_t nv = min(kRows, p.T - p_sub);
        if (p.ctx) {
            int q0, nq;
            queries_of(p, ps.r, q0, nq);
            const int64_t pos = (int64_t)pos_block * p.T + p_sub;
            const int32_t j = min(nq - 1, (ps.ct * X::kCols + X::kCols - 1) / p.G);     // the tile's last query token
            const int64_t end = (int64_t)__ldg(p.ctx + ps.r) - (nq - 1 - j);
            if (pos >= end) return;
            nv = (int32_t)min((int64_t)nv, end - pos);
            my_pos = (int32_t)pos;
        }
        my_id = id;
        my_nv = nv;
    };
    // start the loads of the warp's next slice into stage s; false when the range is exhausted
    auto issue = [&](int s) {
        while (!p_done && p_at >= ps.hi) {
            if (p_next >= hi) {
                p_done = true;
                break;
            }
            ps = segment_at(p, p_next, hi);
            p_next = ps.hi;
            p_at = ps.lo + warp;
            p_batch = p_at;
            look_up(p_at + (int64_t)lane * kWarps);
        }
        if (p_done) return;
        if (p_at >= p_batch + 32 * kWarps) {
            p_batch = p_at;
            look_up(p_at + (int64_t)lane * kWarps);
        }
        const int src = (int)((p_at - p_batch) / kWarps);
        const int32_t id = __shfl_sync(0xffffffffu, my_id, src);
        const int32_t nv = __shfl_sync(0xffffffffu, my_nv, src);
        const int32_t pos = __shfl_sync(0xffffffffu, my_pos, src);
        const int32_t sub = __shfl_sync(0xffffffffu, p_sub, src);
        p_at += kWarps;
        if (lane == 0) note[s] = make_int2(nv, pos);
        if (nv <= 0) return;
        unsigned char* const dst = ring + s * L::kStage;
        if (FMT == 16) {
            if (lane == 0) mbar_expect_tx(&full[s], (uint32_t)(2 * nv) * L::kRowBytes);
            __syncwarp();
            const int row = lane & 15;
            const bool is_v = lane >= 16;
            unsigned char* const d = dst + (is_v ? kRows : 0) * L::kRowStride + row * L::kRowStride;
            if (row < nv) {
                const uint8_t* const srcp = is_v ? p.v + (int64_t)id * p.v_block + (int64_t)(sub + row) * p.v_token
                                                 : p.k + (int64_t)id * p.k_block + (int64_t)(sub + row) * p.k_token;
                bulk_g2s(d, srcp + (int64_t)ps.h * L::kRowBytes, L::kRowBytes, &full[s]);
            } else if (is_v) {          // rows without a token: a weight of zero must meet a number
#pragma unroll
                for (int i = 0; i < L::kRowBytes / 16; ++i) *reinterpret_cast<uint4*>(d + i * 16) = make_uint4(0, 0, 0, 0);
                fence_proxy_async();
            }
        } else if (lane == 0) {
            mbar_expect_tx(&full[s], L::kGroup);
            const int64_t groups = p.T / kRows;
            bulk_g2s(dst, p.k + (int64_t)id * p.k_block + ((int64_t)ps.h * groups + sub / kRows) * L::kGroup, L::kGroup, &full[s]);
        }
    };

#pragma unroll 1
    for (int s = 0; s < L::kStages; ++s) issue(s);
    __syncwarp();

    int stage = 0;
    uint32_t phases = 0;
    bool dead = false;
    const uint32_t ring_u = smem_u32(ring);

    int64_t at = lo;
#pragma unroll 1
    while (at < hi) {
        const Seg sg = segment_at(p, at, hi);
        at = sg.hi;
        int q0, nq;
        queries_of(p, sg.r, q0, nq);
        const int cols = min(X::kCols, nq * p.G - sg.ct * X::kCols);      // may be <= 0: nothing to write
        const int c0 = sg.ct * X::kCols;
        // first position that each of the thread's columns may not see
        int32_t limit[NT][2], limit_min = INT32_MAX;
        if (p.ctx) {
            const int32_t ctx = __ldg(p.ctx + sg.r);
            limit_min = ctx - (nq - 1 - c0 / p.G);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int cc = DUP ? (2 * q4 + e) & 3 : nt * 8 + 2 * q4 + e;
                    limit[nt][e] = ctx - (nq - 1 - (c0 + cc) / p.G);
                }
        } else {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) limit[nt][0] = limit[nt][1] = INT32_MAX;
        }

        // ---- query fragments (the order of the values follows that of the codes), and their sums for the zeros
        uint32_t qf[X::kQReg ? X::kKSteps : 1][X::kQReg ? NT : 1][2];
        float qsum[NT][2];
        if (!X::kQReg) __syncthreads();            // the item before may still be read
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int cc = DUP ? g & 3 : nt * 8 + g;
            const int c = c0 + cc;
            const bool live = cc < cols;
            const int j = live ? c / p.G : 0;
            const uint16_t* const qp = p.q + (int64_t)(q0 + j) * p.q_stride + (int64_t)(sg.h * p.G + (live ? c - j * p.G : 0)) * D;
            float sum = 0.f;
            auto put = [&](int ks, uint32_t b0, uint32_t b1) {
                if (FMT != 16) sum += (bf16lo(b0) + bf16hi(b0)) + (bf16lo(b1) + bf16hi(b1));
                if (X::kQReg) {
                    qf[X::kQReg ? ks : 0][X::kQReg ? nt : 0][0] = b0;
                    qf[X::kQReg ? ks : 0][X::kQReg ? nt : 0][1] = b1;
                } else if (warp == (ks & 3)) {
                    q_frag[(ks * NT + nt) * 32 + lane] = make_uint2(b0, b1);
                }
            };
            if (FMT == 16) {
#pragma unroll
                for (int ks = 0; ks < X::kKSteps; ++ks) {
                    const uint32_t b0 = live ? __ldg(reinterpret_cast<const uint32_t*>(qp + ks * 16 + 2 * q4)) : 0u;
                    const uint32_t b1 = live ? __ldg(reinterpret_cast<const uint32_t*>(qp + ks * 16 + 8 + 2 * q4)) : 0u;
                    put(ks, b0, b1);
                }
            } else if (FMT == 4) {
                constexpr int kWords = L::kPanelDims / 32;       // words of 8 codes a lane has in a panel
#pragma unroll
                for (int i = 0; i < L::kPanels * kWords; ++i) {
                    const int base = (i / kWords) * L::kPanelDims + q4 * (L::kPanelDims / 4) + (i % kWords) * 8;
                    const uint4 x = live ? __ldg(reinterpret_cast<const uint4*>(qp + base)) : make_uint4(0, 0, 0, 0);
                    put(2 * i, __byte_perm(x.x, x.z, 0x5410), __byte_perm(x.x, x.z, 0x7632));
                    put(2 * i + 1, __byte_perm(x.y, x.w, 0x5410), __byte_perm(x.y, x.w, 0x7632));
                }
            } else {
#pragma unroll
                for (int ks = 0; ks < X::kKSteps; ++ks) {
                    const int base = (ks / 4) * L::kPanelDims + q4 * 16 + (ks % 4) * 4;
                    const uint2 x = live ? __ldg(reinterpret_cast<const uint2*>(qp + base)) : make_uint2(0, 0);
                    put(ks, __byte_perm(x.x, x.y, 0x5410), __byte_perm(x.x, x.y, 0x7632));
                }
            }
            if (FMT != 16) {
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                qsum[nt][0] = __shfl_sync(0xffffffffu, sum, (2 * q4) * 4) * p.scale_log2;
                qsum[nt][1] = __shfl_sync(0xffffffffu, sum, (2 * q4 + 1) * 4) * p.scale_log2;
            }
        }
        if (!X::kQReg) __syncthreads();

        float o[X::kMTiles][NT][4];
        float m[NT][2], l[NT][2], z[NT][2];       // m: what is taken off the scores (0 while nothing was seen)
        bool seen[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                m[nt][e] = -INFINITY;
                l[nt][e] = z[nt][e] = 0.f;
                seen[nt][e] = false;
            }
#pragma unroll
            for (int mt = 0; mt < X::kMTiles; ++mt)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[mt][nt][i] = 0.f;
        }

        // ---------------------------------------------------------------------------- the warp's slices of this item
#pragma unroll 1
        for (int64_t s = sg.lo + warp; s < sg.hi; s += kWarps) {
            const int2 nt_ = note[stage];
            const int nv = nt_.x, pos0 = nt_.y;
            const uint32_t st_u = ring_u + stage * L::kStage;
            if (nv > 0 && !dead) {
                if (!mbar_wait(&full[stage], (phases >> stage) & 1u)) {
                    if (p.err && lane == 0) atomicExch(p.err, 1);
                    dead = true;
                }
                phases ^= 1u << stage;
            }
            if (nv > 0 && !dead) {
                // ---- S^T = K Q^T
                float sc[NT][4];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) sc[nt][i] = 0.f;
                auto qk = [&](int ks, const uint32_t (&a)[4]) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        if (X::kQReg) {
                            mma(sc[nt], a, qf[X::kQReg ? ks : 0][X::kQReg ? nt : 0][0], qf[X::kQReg ? ks : 0][X::kQReg ? nt : 0][1]);
                        } else {
                            const uint2 b = q_frag[(ks * NT + nt) * 32 + lane];
                            mma(sc[nt], a, b.x, b.y);
                        }
                    }
                };
                if (FMT == 16) {
                    const uint32_t ka = st_u + (lane & 15) * L::kRowStride + (lane >> 4) * 16;
#pragma unroll
                    for (int ks = 0; ks < X::kKSteps; ++ks) {
                        uint32_t a[4];
                        ldsm4(a, ka + ks * 32);
                        qk(ks, a);
                    }
                } else {
                    constexpr int kChunk = L::kPanel / 4;        // bytes of a row in a panel that a lane reads
#pragma unroll
                    for (int pn = 0; pn < L::kPanels; ++pn) {
                        const uint32_t ka = st_u + pn * (kRows * L::kPanel) + g * L::kPanel + q4 * kChunk;
                        uint32_t x[4], y[4];                     // rows g and g + 8
                        if (kChunk == 16) {
                            const uint4 u = lds16(ka), w = lds16(ka + 8 * L::kPanel);
                            x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w;
                            y[0] = w.x; y[1] = w.y; y[2] = w.z; y[3] = w.w;
                        } else {
                            const uint2 u = lds8(ka), w = lds8(ka + 8 * L::kPanel);
                            x[0] = u.x; x[1] = u.y;
                            y[0] = w.x; y[1] = w.y;
                        }
#pragma unroll
                        for (int i = 0; i < kChunk / 4; ++i) {
                            if (FMT == 4) {
#pragma unroll
                                for (int half = 0; half < 2; ++half) {
                                    const uint32_t a[4] = {nibbles(x[i], 2 * half), nibbles(y[i], 2 * half),
                                                           nibbles(x[i], 2 * half + 1), nibbles(y[i], 2 * half + 1)};
                                    qk((pn * (kChunk / 4) + i) * 2 + half, a);
                                }
                            } else {
                                const uint32_t a[4] = {bytes(x[i], 0), bytes(y[i], 0), bytes(x[i], 1), bytes(y[i], 1)};
                                qk(pn * (kChunk / 4) + i, a);
                            }
                        }
                    }
                }

                // ---- scores in powers of two; rows g (values 0, 1) and g + 8 (values 2, 3)
                float ks0 = p.scale_log2, ks1 = p.scale_log2, kz0 = 0.f, kz1 = 0.f, vs0 = 1.f, vs1 = 1.f, vz0 = 0.f, vz1 = 0.f;
                if (FMT != 16) {
                    const float mid = FMT == 4 ? 8.f : 128.f;
                    const uint32_t pa = st_u + 2 * kRows * L::kRowBytes + g * 4;
                    const uint32_t k0 = lds4(pa), k1 = lds4(pa + 32), v0 = lds4(pa + 64), v1 = lds4(pa + 96);
                    kz0 = fmaf(bf16lo(k0), mid, bf16hi(k0));     // the centred codes' zero
                    kz1 = fmaf(bf16lo(k1), mid, bf16hi(k1));
                    ks0 = bf16lo(k0) * p.scale_log2;
                    ks1 = bf16lo(k1) * p.scale_log2;
                    vs0 = bf16lo(v0);
                    vs1 = bf16lo(v1);
                    vz0 = fmaf(vs0, mid, bf16hi(v0));
                    vz1 = fmaf(vs1, mid, bf16hi(v1));
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    if (FMT == 16) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) sc[nt][i] *= ks0;
                    } else {
                        sc[nt][0] = fmaf(sc[nt][0], ks0, kz0 * qsum[nt][0]);
                        sc[nt][1] = fmaf(sc[nt][1], ks0, kz0 * qsum[nt][1]);
                        sc[nt][2] = fmaf(sc[nt][2], ks1, kz1 * qsum[nt][0]);
                        sc[nt][3] = fmaf(sc[nt][3], ks1, kz1 * qsum[nt][1]);
                    }
                }
                const bool masked = nv < kRows || (p.ctx != nullptr && pos0 + kRows > limit_min);
                uint32_t hide = 0;                               // bit 4 nt + i: value i of tile nt is not seen
                if (masked) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int row = g + (i >> 1) * 8;
                            if (row >= nv || pos0 + row >= limit[nt][i & 1]) {
                                sc[nt][i] = -INFINITY;
                                hide |= 1u << (4 * nt + i);
                            }
                        }
                }
                // ---- running maximum: moved only when it is passed by more than the slack
                bool passed = false;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        passed |= fmaxf(sc[nt][e], sc[nt][e + 2]) > (seen[nt][e] ? m[nt][e] + kMaxSlack : -INFINITY);
                if (__any_sync(0xffffffffu, passed)) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            float x = fmaxf(sc[nt][e], sc[nt][e + 2]);
                            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                            const float now = fmaxf(m[nt][e], x);
                            if (now > -INFINITY) {
                                const float f = seen[nt][e] ? exp2_fast(m[nt][e] - now) : 0.f;
                                // (nothing but zeros and NaN can have been added before the first score)
                                if (seen[nt][e]) {
                                    l[nt][e] *= f;
                                    z[nt][e] *= f;
#pragma unroll
                                    for (int mt = 0; mt < X::kMTiles; ++mt) {
                                        o[mt][nt][e] *= f;
                                        o[mt][nt][e + 2] *= f;
                                    }
                                }
                                m[nt][e] = now;
                                seen[nt][e] = true;
                            }
                        }
                }
                // ---- weights, and their bf16 halves with tokens along the columns' other side
                uint32_t ph[NT][2], pl[NT][2];
                float wt[NT][4];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float (&w)[4] = wt[nt];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float off = seen[nt][i & 1] ? m[nt][i & 1] : 0.f;
                        w[i] = exp2_fast(sc[nt][i] - off);
                    }
                    l[nt][0] += w[0] + w[2];
                    l[nt][1] += w[1] + w[3];
                    if (FMT != 16) {
                        if (masked) {                            // what stands in rows that are not seen may be anything
                            const uint32_t hd = hide >> (4 * nt);
                            z[nt][0] += ((hd & 1u) ? 0.f : w[0] * vz0) + ((hd & 4u) ? 0.f : w[2] * vz1);
                            z[nt][1] += ((hd & 2u) ? 0.f : w[1] * vz0) + ((hd & 8u) ? 0.f : w[3] * vz1);
                            w[0] = (hd & 1u) ? 0.f : w[0] * vs0;
                            w[1] = (hd & 2u) ? 0.f : w[1] * vs0;
                            w[2] = (hd & 4u) ? 0.f : w[2] * vs1;
                            w[3] = (hd & 8u) ? 0.f : w[3] * vs1;
                        } else {
                            z[nt][0] = fmaf(w[0], vz0, fmaf(w[2], vz1, z[nt][0]));
                            z[nt][1] = fmaf(w[1], vz0, fmaf(w[3], vz1, z[nt][1]));
                            w[0] *= vs0;
                            w[1] *= vs0;
                            w[2] *= vs1;
                            w[3] *= vs1;
                        }
                    }
                    uint32_t a = pack_bf16(w[0], w[1]), b = pack_bf16(w[2], w[3]);
                    const uint32_t al = pack_bf16(w[0] - bf16lo(a), w[1] - bf16hi(a));
                    const uint32_t bl = pack_bf16(w[2] - bf16lo(b), w[3] - bf16hi(b));
                    if (DUP) {
                        ph[nt][0] = transpose8(q4 < 2 ? a : al);
                        ph[nt][1] = transpose8(q4 < 2 ? b : bl);
                    } else {
                        ph[nt][0] = transpose8(a);
                        ph[nt][1] = transpose8(b);
                        pl[nt][0] = transpose8(al);
                        pl[nt][1] = transpose8(bl);
                    }
                }
                // ---- O^T += V^T P^T
                auto pv = [&](int mt, const uint32_t (&a)[4]) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        mma(o[mt][nt], a, ph[nt][0], ph[nt][1]);
                        if (!DUP) mma(o[mt][nt], a, pl[nt][0], pl[nt][1]);
                    }
                };
                // A row that some columns see and others do not may hold an infinity or a NaN, and a weight of zero would not
                // keep it out of the product: such a slice (the last tokens of a request with several queries) is added up
                // column by column instead.
                bool wild = false;
                if (FMT == 16 && masked && pos0 + nv > limit_min) {
                    for (int i = lane; i < nv * (D / 8); i += 32) {
                        const uint4 x = lds16(st_u + (kRows + i / (D / 8)) * L::kRowStride + (i % (D / 8)) * 16);
                        const uint32_t y[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            wild |= (y[k] & 0x7f80u) == 0x7f80u || (y[k] & 0x7f800000u) == 0x7f800000u;
                    }
                    wild = __any_sync(0xffffffffu, wild);
                }
                if (FMT == 16 && wild) {
#pragma unroll 1
                    for (int row = 0; row < nv; ++row) {
                        const int src = (row & 7) * 4 + q4;
                        const uint32_t hd = __shfl_sync(0xffffffffu, hide, src);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                const float w0 = __shfl_sync(0xffffffffu, wt[nt][e], src);
                                const float w1 = __shfl_sync(0xffffffffu, wt[nt][e + 2], src);
                                const int bit = 4 * nt + e + (row >> 3) * 2;
                                if (((hd >> bit) & 1u) || (DUP && q4 >= 2)) continue;
                                const float w = row < 8 ? w0 : w1;
#pragma unroll
                                for (int mt = 0; mt < X::kMTiles; ++mt)
#pragma unroll
                                    for (int k = 0; k < 2; ++k) {
                                        const uint16_t b = *reinterpret_cast<const uint16_t*>(
                                            ring + stage * L::kStage + (kRows + row) * L::kRowStride + (mt * 16 + g + k * 8) * 2);
                                        o[mt][nt][e + 2 * k] += w * __uint_as_float((uint32_t)b << 16);
                                    }
                            }
                    }
                } else if (FMT == 16) {
                    const uint32_t va = st_u + kRows * L::kRowStride + ((lane & 7) + ((lane >> 4) & 1) * 8) * L::kRowStride +
                                        ((lane >> 3) & 1) * 16;
#pragma unroll
                    for (int mt = 0; mt < X::kMTiles; ++mt) {
                        uint32_t a[4];
                        ldsm4_trans(a, va + mt * 32);
                        pv(mt, a);
                    }
                } else {
                    constexpr int kChunk = L::kPanel / 4;        // bytes of a lane in half a panel: 2 tokens, 1/8 of the values
#pragma unroll
                    for (int pn = 0; pn < L::kPanels; ++pn) {
                        const uint32_t va = st_u + kRows * L::kRowBytes + pn * (kRows * L::kPanel) + lane * kChunk;
                        uint32_t x[4], y[4];                     // tokens 2 q4, 2 q4 + 1 and the two 8 behind them
                        if (kChunk == 16) {
                            const uint4 u = lds16(va), w = lds16(va + 8 * L::kPanel);
                            x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w;
                            y[0] = w.x; y[1] = w.y; y[2] = w.z; y[3] = w.w;
                        } else {
                            const uint2 u = lds8(va), w = lds8(va + 8 * L::kPanel);
                            x[0] = u.x; x[1] = u.y;
                            y[0] = w.x; y[1] = w.y;
                        }
#pragma unroll
                        for (int i = 0; i < kChunk / 4; ++i) {
                            if (FMT == 4) {
#pragma unroll
                                for (int half = 0; half < 2; ++half) {
                                    const uint32_t a[4] = {nibbles(x[i], 2 * half), nibbles(x[i], 2 * half + 1),
                                                           nibbles(y[i], 2 * half), nibbles(y[i], 2 * half + 1)};
                                    pv(pn * (L::kPanelDims / 16) + i * 2 + half, a);
                                }
                            } else {
                                const uint32_t a[4] = {bytes(x[i], 0), bytes(x[i], 1), bytes(y[i], 0), bytes(y[i], 1)};
                                pv(pn * (L::kPanelDims / 16) + i, a);
                            }
                        }
                    }
                }
            }
            __syncwarp();                                        // every lane is done with the stage
            if (!dead) issue(stage);
            __syncwarp();
            stage = stage + 1 == L::kStages ? 0 : stage + 1;
        }

        // ---------------------------------------------------------------------------------- join the four warps
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float a = l[nt][e], b = z[nt][e];
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) {
                    a += __shfl_xor_sync(0xffffffffu, a, x);
                    if (FMT != 16) b += __shfl_xor_sync(0xffffffffu, b, x);
                }
                const int cc = nt * 8 + 2 * q4 + e;
                if (g == 0 && cc < X::kCols) {
                    stat[(warp * 3 + 0) * X::kCols + cc] = m[nt][e];
                    stat[(warp * 3 + 1) * X::kCols + cc] = a;
                    stat[(warp * 3 + 2) * X::kCols + cc] = b;
                }
            }
        const bool whole = sg.lo == sg.begin && sg.hi == sg.end;
        float* const part = p.ws + (int64_t)(2 * blockIdx.x + (sg.lo == sg.begin ? 1 : 0)) * X::kPart;
#pragma unroll
        for (int step = 0; step < X::kMergeSteps; ++step) {
            if (step) __syncthreads();
#pragma unroll
            for (int k = 0; k < NT; ++k) {
                if (k != step >> 1) continue;
#pragma unroll
                for (int mt = 0; mt < X::kMTiles; ++mt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float x = o[mt][k][i];
                        if (DUP) x += __shfl_xor_sync(0xffffffffu, x, 2);
                        const int row = i >> 1;                  // rows g and g + 8 of the tile
                        const int d = FMT == 16 ? mt * 16 + g + row * 8
                                                : (mt / (L::kPanelDims / 16)) * L::kPanelDims + g * (L::kPanelDims / 8) +
                                                      (mt % (L::kPanelDims / 16)) * 2 + row;
                        if ((q4 >> 1) == (step & 1)) merge[(warp * X::kMergeCols + ((2 * q4 + (i & 1)) & 3)) * X::kMergeLd + d] = x;
                    }
            }
            __syncthreads();
            for (int i = tid; i < X::kMergeCols * (D / 2); i += kThreads) {
                const int cl = i / (D / 2), d = (i - cl * (D / 2)) * 2, cc = step * 4 + cl;
                if (cc >= cols) continue;
                float mw[kWarps], top = -INFINITY;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) top = fmaxf(top, mw[w] = stat[(w * 3) * X::kCols + cc]);
                const float off = top == -INFINITY ? 0.f : top;
                float sum = 0.f, zero = 0.f, a = 0.f, b = 0.f;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) {
                    const float f = exp2_fast(mw[w] - off);
                    const float* const row = merge + (w * X::kMergeCols + cl) * X::kMergeLd + d;
                    sum += f * stat[(w * 3 + 1) * X::kCols + cc];
                    if (FMT != 16) zero += f * stat[(w * 3 + 2) * X::kCols + cc];
                    a += f * row[0];
                    b += f * row[1];
                }
                a += zero;
                b += zero;
                if (whole) {
                    const int c = c0 + cc, j = c / p.G;
                    const int64_t row = (int64_t)(q0 + j) * p.Hq + sg.h * p.G + (c - j * p.G);
                    const float inv = sum == 0.f ? 0.f : 1.f / sum;
                    reinterpret_cast<uint32_t*>(p.out)[row * (D / 2) + d / 2] = sum == 0.f ? 0u : pack_bf16(a * inv, b * inv);
                    if (d == 0 && p.lse) p.lse[row] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * kLn2;
                } else {
                    *reinterpret_cast<float2*>(part + 2 * X::kCols + cc * D + d) = make_float2(a, b);
                    if (d == 0) {
                        part[cc] = top;
                        part[X::kCols + cc] = sum;
                    }
                }
            }
        }
        __syncthreads();
    }
    // a wait that ran out leaves copies behind: give them one more bounded wait before the block's memory is reused
    if (dead)
        for (int s = 0; s < L::kStages; ++s)
            if (note[s].x > 0) mbar_wait(&full[s], (phases >> s) & 1u);
}

// Joins the partial results of the item that crosses the cut between thread blocks blockIdx.x and blockIdx.x + 1 (the
// first cut of the item does it), eight columns per blockIdx.y.
template <int D, int COLS>
__global__ void __launch_bounds__(256) attend_join_kernel(const Params p, const int n_parts)
{
    constexpr int kC = COLS < 8 ? COLS : 8;
    constexpr int kJoinWarps = D == 256 ? 4 : 8;
    constexpr int kPart = COLS * (D + 2);
    constexpr int kV = D / 32;                        // values of a row per lane
    __shared__ float buf[kJoinWarps][kC][D];
    early_start_wait();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t all = entries_total(p) * slices_per_entry(p);
    const int b = blockIdx.x;
    const int64_t at = cut(all, b + 1, n_parts);
    if (at <= 0 || at >= all) return;
    const Seg s = segment_at(p, at, all);
    if (s.begin == at || s.begin < cut(all, b, n_parts)) return;     // nothing crosses here, or an earlier cut does it
    if (cut(all, b, n_parts) == at) return;                          // an empty range: the cut was an earlier one
    int last = b + 1;
    while (last + 1 < n_parts && cut(all, last + 1, n_parts) < s.end) ++last;
    int q0, nq;
    queries_of(p, s.r, q0, nq);
    const int y0 = blockIdx.y * 8;
    const int cols = min(COLS, nq * p.G - s.ct * COLS);
    if (y0 >= cols) return;

    // part i of the item: thread block b + i; the first one's is its trailing part, the others' are leading ones
    auto part_of = [&](int i) { return p.ws + (int64_t)(2 * (b + i) + (i == 0 ? 1 : 0)) * kPart; };
    const int n = last - b + 1;
    float top[kC], sum[kC], acc[kC][kV];
#pragma unroll
    for (int c = 0; c < kC; ++c) {
        float x = -INFINITY;
        for (int i = lane; i < n; i += 32)
            if (cut(all, b + i, n_parts) < cut(all, b + i + 1, n_parts)) x = fmaxf(x, part_of(i)[y0 + c]);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
        top[c] = x;
        sum[c] = 0.f;
#pragma unroll
        for (int v = 0; v < kV; ++v) acc[c][v] = 0.f;
    }
    if (warp < kJoinWarps)
        for (int i = warp; i < n; i += kJoinWarps) {
            if (cut(all, b + i, n_parts) == cut(all, b + i + 1, n_parts)) continue;
            const float* const part = part_of(i);
#pragma unroll
            for (int c = 0; c < kC; ++c) {
                const float f = exp2_fast(part[y0 + c] - (top[c] == -INFINITY ? 0.f : top[c]));
                sum[c] += f * part[COLS + y0 + c];
#pragma unroll
                for (int v = 0; v < kV; ++v) acc[c][v] += f * part[2 * COLS + (y0 + c) * D + v * 32 + lane];
            }
        }
    __shared__ float sums[kJoinWarps][kC];
    if (warp < kJoinWarps) {
#pragma unroll
        for (int c = 0; c < kC; ++c) {
            if (lane == 0) sums[warp][c] = sum[c];
#pragma unroll
            for (int v = 0; v < kV; ++v) buf[warp][c][v * 32 + lane] = acc[c][v];
        }
    }
    __syncthreads();
    for (int i = tid; i < kC * (D / 2); i += 256) {
        const int cl = i / (D / 2), d = (i - cl * (D / 2)) * 2, cc = y0 + cl;
        if (cc >= cols) continue;
        float l = 0.f, x = 0.f, y = 0.f;
#pragma unroll
        for (int w = 0; w < kJoinWarps; ++w) {
            l += sums[w][cl];
            x += buf[w][cl][d];
            y += buf[w][cl][d + 1];
        }
        const int c = s.ct * COLS + cc, j = c / p.G;
        const int64_t row = (int64_t)(q0 + j) * p.Hq + s.h * p.G + (c - j * p.G);
        const float inv = l == 0.f ? 0.f : 1.f / l;
        reinterpret_cast<uint32_t*>(p.out)[row * (D / 2) + d / 2] = l == 0.f ? 0u : pack_bf16(x * inv, y * inv);
        if (d == 0 && p.lse) {
            float t = -INFINITY;
#pragma unroll
            for (int k = 0; k < kC; ++k)
                if (k == cl) t = top[k];
            p.lse[row] = l == 0.f ? -INFINITY : (t + log2f(l)) * kLn2;
        }
    }
}

// ---------------------------------------------------------------------------------------------------- host side

// Columns of a tile for `cols` query rows of a KV head: the narrowest tile that takes them all, 32 (16 with 256 values a
// head) and several tiles beyond that.  A tile reads K and V once; a narrower one costs fewer instructions per token.
inline int tile_cols(int cols, int head_dim)
{
    if (cols <= 4) return 4;
    if (cols <= 8) return 8;
    if (cols <= 16 || head_dim == 256) return 16;
    return 32;
}

// what a launch needs for one shape
struct Plan {
    int32_t ctas;                      // thread blocks resident on the device at once
    int32_t part;                      // floats of a partial result
    int32_t cols;                      // columns of a tile
};

template <int FMT, int D, int NT, bool DUP>
int32_t run(const Params& p, bool launch, Plan* plan, cudaStream_t st)
{
    using X = Traits<FMT, D, NT, DUP>;
    plan->ctas = sm_count() * X::kOcc;
    plan->part = X::kPart;
    plan->cols = X::kCols;
    if (!launch) return UCMX_OK;
    auto kern = attend_kernel<FMT, D, NT, DUP>;
    UCMX_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, X::kSmem));
    const int64_t all = (int64_t)p.total * p.spe * p.H * p.col_tiles;
    // at least one slice per warp: below that more blocks only add partial results
    int64_t grid = (all + kWarps - 1) / kWarps;
    if (grid > plan->ctas) grid = plan->ctas;
    if (grid < 1) grid = 1;
    kern<<<(unsigned)grid, kThreads, X::kSmem, st>>>(p);
    UCMX_LAUNCH_CHECK("attend_kernel");
    if (grid == 1) return UCMX_OK;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid - 1, X::kCols <= 8 ? 1 : X::kCols / 8);
    cfg.blockDim = dim3(256);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    UCMX_CUDA(cudaLaunchKernelEx(&cfg, attend_join_kernel<D, X::kCols>, p, (int)grid));
    UCMX_LAUNCH_CHECK("attend_join_kernel");
    return UCMX_OK;
}

template <int FMT, int D>
int32_t run_cols(const Params& p, int cols, bool launch, Plan* plan, cudaStream_t st)
{
    switch (tile_cols(cols, D)) {
        case 4: return run<FMT, D, 1, true>(p, launch, plan, st);
        case 8: return run<FMT, D, 1, false>(p, launch, plan, st);
        case 16: return run<FMT, D, 2, false>(p, launch, plan, st);
        default:
            if constexpr (D != 256) return run<FMT, D, 4, false>(p, launch, plan, st);
            return UCMX_EUNSUPPORTED;
    }
}

template <int FMT>
int32_t run_format(const Params& p, int head_dim, int cols, bool launch, Plan* plan, cudaStream_t st)
{
    switch (head_dim) {
        case 64: return run_cols<FMT, 64>(p, cols, launch, plan, st);
        case 128: return run_cols<FMT, 128>(p, cols, launch, plan, st);
        case 256: return run_cols<FMT, 256>(p, cols, launch, plan, st);
        default: return UCMX_EUNSUPPORTED;
    }
}

// the three formats live in files of their own
int32_t run_bf16(const Params& p, int head_dim, int cols, bool launch, Plan* plan, cudaStream_t st);
int32_t run_q8(const Params& p, int head_dim, int cols, bool launch, Plan* plan, cudaStream_t st);
int32_t run_q4(const Params& p, int head_dim, int cols, bool launch, Plan* plan, cudaStream_t st);

}  // namespace attend
}  // namespace ucmx
