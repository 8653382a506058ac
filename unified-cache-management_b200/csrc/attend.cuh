// Attention of a ragged batch of queries over listed KV blocks: the kernel shared by the bf16 cache (attend.cu) and the
// quantised cache (attend_q8.cu, attend_q4.cu).
//
//   out[c] = sum_t softmax_t(scale * q_c . k_t) v_t        over the tokens t of the request's listed blocks that c may see
//
// Shape of the work.  Few query rows (query heads of one KV head x query tokens of the request: the "columns") meet
// thousands of cached tokens, so the kernel is a stream over K and V: every listed token is read once per KV head and
// column tile, and everything else stays in registers.  The matrix instructions take TOKENS as their 16 rows and the
// columns as their 8 wide side (S^T = K Q^T, O^T = V^T P^T): 4 to 8 query heads per KV head then waste little, K and V
// are the wide operand straight from shared memory, and one column's softmax statistics live in one register per thread.
// (With so few columns the warp-level instructions keep up with HBM: 8 % of their rate for the bf16 cache, 23 % for 4-bit
// codes, which have to pass through registers anyway.)
//
// Split.  The unit is a slice: up to 16 consecutive tokens of one listed block.  All slices of all (request, KV head,
// column tile) items are laid end to end, each item behind a lead of 16 or 24 units (what beginning and ending an item costs:
// 190 requests of 1 to 40 blocks take 26.6 us with a lead of 1, 14.6 so), and cut into equal parts, one per thread block, whatever
// the lengths of the requests are.  A short item stays with the thread block that it begins in; a longer one that crosses
// cuts leaves partial results (running maximum, sum, unnormalised output) in the workspace, which a second small kernel joins
// in order.  The workspace needs no initial state, and the order of the sums is fixed by the shapes, so results do not change
// from run to run.
//
// Within a thread block each of the four warps takes every fourth slice (pairs of slices of codes: alone they took 176 us
// where pairs take 142) with a ring of its own: one elected lane starts the copies - four swizzled tiles of a tensor map
// for 16 tokens of bf16, one bulk copy for two groups of codes - the warp waits on its own barrier, and no other warp is involved
// until the item ends.  The loads run ahead across items.
//
// Rounding.  Scores, maxima, sums and outputs are fp32.  The weights are the one operand that has to become bf16 for
// the second product; each is split into a bf16 value and the bf16 of what is left (2^-16 relative over a bf16 cache, where
// the first half is the value next below, 2^-17 over codes; 2^-9 without, which would be as large an error as the final rounding
// of the output).  With at most four columns the two halves share one instruction (columns 4..7 repeat 0..3), otherwise they are two.
//
// Measured on a B200 (128 values a head, 32 query heads on 8; device times of a call, both kernels; bytes of the listed K and V):
//   bf16, 64 requests, 16..52 blocks of 128 tokens: 162 us, 6.3 TB/s, 0.97 of a copy's rate: HBM.  One request of 130 944 tokens:
//   92 us, 5.8 TB/s.  8 bits, the first batch: 92 us, 5.7 TB/s: HBM, and eight warps per SM.
//   4 bits, 32 requests of 120..500 blocks of 64 tokens: 139 us, 4.3 TB/s: turning codes into 16-bit operands (326 instructions per
//   slice; 62 % of the issue slots, 55 % of the integer pipe's cycles).  Shortest call, 40 slices: 6 us.
#pragma once

#include <cuda.h>

#include <atomic>
#include <type_traits>

#include "common.cuh"
#include "split.cuh"

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
    int32_t box;                       // bf16: rows that one load brings, min(16, T)
    int64_t n_blocks;
    const int32_t* offsets;            // [n_req+1] into the lists
    const int32_t* counts;             // [n_req] or NULL
    const int32_t* block_ids;          // [total] or NULL: table[table_offsets[r] + position]
    const int32_t* positions;          // [total] or NULL: the i-th entry of a request stands at i
    const int32_t* table;
    const int32_t* table_offsets;      // [n_req+1]
    int32_t table_size;
    const int32_t* ctx;                // [n_req] or NULL
    int32_t n_req, total;
    int32_t col_tiles;
    float scale_log2;
    uint16_t* out;                     // [n_q_tokens, Hq, D]
    float* lse;                        // [n_q_tokens, Hq] or NULL
    float* ws;                         // partial results: 2 per thread block, then a Rec per thread block
    int32_t* err;
};

// K and V of the bf16 cache as tensors [block][token][head][value]; unused for the quantised cache.
struct Maps {
    CUtensorMap k, v;
};

// What a thread block tells the joining kernel about the item that begins in its range and goes on behind it.
struct __align__(16) Rec {
    int32_t parts;                     // 0: there is none
    int32_t q0, c0, cols, h;
    int32_t pad[3];
};
static_assert(alignof(Rec) <= 16 && sizeof(Rec) == 32, "records lie in a workspace that starts on 16 bytes, and no more is asked of it");

template <int LEAD>
__device__ __forceinline__ int32_t base_of(const Params& p, const int32_t* scan, int32_t r)
{
    return scan ? scan[r] : inside(__ldg(p.offsets + r), p.total) * p.spe + r * LEAD;
}

// The last r with base(r) <= e, and base(r), base(r+1); 31 intervals a step, the first of them at hand.
template <int LEAD>
__device__ __forceinline__ int request_of(const Params& p, const Share& w, int32_t e, int32_t& first, int32_t& next)
{
    const int lane = threadIdx.x & 31;
    int lo = 0, n = p.n_req, step = w.step;
    int32_t v = w.probes[lane];
    for (;;) {
        const int c = __popc(__ballot_sync(0xffffffffu, lane * step < n && v <= e));
        const int adv = (c > 0 ? c - 1 : 0) * step;
        if (step == 1) {
            first = __shfl_sync(0xffffffffu, v, c > 0 ? c - 1 : 0);
            next = __shfl_sync(0xffffffffu, v, c > 0 ? c : 1);
            return lo + adv;
        }
        lo += adv;
        n = min(step, n - adv);
        step = (n + 30) / 31;
        v = base_of<LEAD>(p, w.scan, lo + min(lane * step, n));
    }
}

// Query rows [q0, end) that no request of this call can have.
__device__ __forceinline__ bool bad_queries(const Params& p, int32_t q0, int32_t end)
{
    return q0 < 0 || end < q0 || end > p.n_q_tokens || end - q0 > p.max_q;
}

// Query rows of request r: first row and how many (clamped to the query tensor and to max_q).
__device__ __forceinline__ void queries_of(const Params& p, int r, int& q0, int& nq)
{
    if (p.q_offsets == nullptr) {
        q0 = r;
        nq = r < p.n_q_tokens ? 1 : 0;
        return;
    }
    const int32_t end = __ldg(p.q_offsets + r + 1);
    q0 = __ldg(p.q_offsets + r);
    nq = (int)((uint32_t)end - (uint32_t)q0);
    if (bad_queries(p, q0, end)) {
        if (p.err && threadIdx.x == 0) atomicExch(p.err, 3);
        nq = q0 < 0 || q0 >= p.n_q_tokens || end <= q0 ? 0 : min(min(nq, p.max_q), p.n_q_tokens - q0);
    }
}

// The item that holds unit `at` and the part of it that ends in this thread block; called by whole warps.  Items that cannot be are passed
// over (n < 0) and reported.
template <int COLS, int LEAD>
__device__ __forceinline__ Seg segment_at(const Params& p, const Share& w, int32_t at)
{
    Seg s;
    int32_t a, b, tiles = w.tiles;
    s.r = request_of<LEAD>(p, w, at / w.mult + w.zero, a, b);
    if (w.scan) {
        int q0, nq;
        queries_of(p, s.r, q0, nq);
        tiles = max(1, (nq * p.G + COLS - 1) / COLS);
        s.first = inside(__ldg(p.offsets + s.r), p.total);
    } else {
        s.first = (a - s.r * LEAD) / p.spe;
    }
    if (!place(s, w, a, b, tiles, p.H, p.spe, p.total, LEAD, at) && p.err && threadIdx.x == 0) atomicExch(p.err, 3);
    return s;
}

// 2^x for a weight: x is at most kMaxSlack, and what is below 2^-126 of the largest weight is nothing
__device__ __forceinline__ float exp2_fast(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// 64 values of `box` tokens of one head -> rows of 128 bytes, their 16-byte pieces XORed with the row (mod 8)
__device__ __forceinline__ void load_panel(unsigned char* dst, const CUtensorMap* map, int x, int h, int token, int block, uint64_t* bar)
{
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(
            smem_u32(dst)),
        "l"(map), "r"(x), "r"(h), "r"(token), "r"(block), "r"(smem_u32(bar))
        : "memory");
}
__device__ __forceinline__ void prefetch_l2(const void* at) { asm volatile("prefetch.global.L2 [%0];" ::"l"(at)); }
// One lane of a converged warp.  (Told this way the compiler issues a copy once; behind `lane == 0` it loops over the lanes.)
__device__ __forceinline__ bool one_lane()
{
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar)
{
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

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
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi)
{
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float f16lo(uint32_t x) { return __half2float(__ushort_as_half((unsigned short)x)); }
__device__ __forceinline__ float f16hi(uint32_t x) { return __half2float(__ushort_as_half((unsigned short)(x >> 16))); }
__device__ __forceinline__ uint32_t sub_f16x2(uint32_t a, uint32_t b)
{
    uint32_t r;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi)
{
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// Two weights (not negative) as the bf16 numbers next below them, 0 for 0: what is left of a weight above 0 is above 0, so that both halves
// of it make an infinity of V the same infinity.
__device__ __forceinline__ uint32_t pack_below(float lo, float hi)
{
    return __byte_perm(max(__float_as_uint(lo), 1u) - 1u, max(__float_as_uint(hi), 1u) - 1u, 0x7632);
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

template <int BYTES>
__device__ __forceinline__ void lds_words(uint32_t (&w)[4], uint32_t a)
{
    if (BYTES == 16) {
        const uint4 u = lds16(a);
        w[0] = u.x;
        w[1] = u.y;
        w[2] = u.z;
        w[3] = u.w;
    } else {
        const uint2 u = lds8(a);
        w[0] = u.x;
        w[1] = u.y;
    }
}

// (x & mask) | base in one instruction (written out it became two, each with a constant of its own)
__device__ __forceinline__ uint32_t mask_or(uint32_t x, uint32_t mask, uint32_t base)
{
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(x), "r"(mask), "r"(base));
    return r;
}
// V's codes as centred integers in bf16 (exact): 4 bits: c - 8, two per register from bits [4i, 4i+4) of both halves.
// 0x4300 is 128.0 and a bf16 of that size counts in ones, so or-ing the code in adds it.
__device__ __forceinline__ uint32_t v_nibbles(uint32_t w, int i)
{
    return sub_bf16x2(mask_or(w >> (4 * i), 0x000f000fu, 0x43004300u), 0x43084308u);
}
// 8 bits: c - 128 from bytes i and i+2.  The low seven bits are or-ed into 128.0; the top bit chooses what is taken off:
// 256.0 (0x4380) where it is clear, 128.0 (0x4300) where it is set.
__device__ __forceinline__ uint32_t v_bytes(uint32_t w, int i)
{
    const uint32_t x = w >> (8 * i);
    return sub_bf16x2(mask_or(x, 0x007f007fu, 0x43004300u), mask_or(~x, 0x00800080u, 0x43004300u));
}
// K's codes become fp16, whose eleven bits hold two nibble positions: half the shifts, and half or none of the subtractions.
// (The queries can follow: a column scaled by a power of two to where its largest value is 2^14 or more fits fp16 to 2^-39 of that
// value, to 2^-35 where a sixteenth of it is held (below).  The weights cannot: their range is not bounded.)
// 0x6400 is 1024.0, counting in ones.  4 bits: registers i = 0, 2 hold c - 8, registers i = 1, 3
// hold 1024 + 16 c, whose 1024 + 128 the accumulator starts below (kOddOffset times those queries' sum) and whose 16 is in the
// queries.  With that offset in all four the sums would lose four bits more.
__device__ __forceinline__ uint32_t k_nibbles(uint32_t w, int i)
{
    const uint32_t x = i < 2 ? w : w >> 8;
    if (i & 1) return mask_or(x, 0x00f000f0u, 0x64006400u);
    return sub_f16x2(mask_or(x, 0x000f000fu, 0x64006400u), 0x64086408u);
}
// 8 bits: 1024 + c of bytes 2i and 2i+1: one instruction; the accumulator starts 1024 + 128 times the queries' sum below.
__device__ __forceinline__ uint32_t k_bytes(uint32_t w, int i) { return __byte_perm(w, 0x64646464u, i ? 0x4342 : 0x4140); }
constexpr float kOddOffset = 1024.f + 128.f;

// FMT 16: bf16 cache, rows of K and V; 8 or 4: groups of the quantised cache.
template <int FMT, int D>
struct Layout {
    static constexpr int kRowBytes = D * FMT / 8;
    static constexpr int kPanel = FMT == 16 ? kRowBytes : kRowBytes < 64 ? kRowBytes : 64;   // bytes of a row in a panel
    static constexpr int kPanels = kRowBytes / kPanel;
    static constexpr int kPanelDims = D / kPanels;
    static constexpr int kGroup = 2 * kRows * kRowBytes + 2 * kRows * 4;  // quantised: codes of K and V, then their scales
    static constexpr int kBf16Panel = kRows * 128;                        // bf16: 64 values of 16 rows in shared memory
    // slices a warp takes at a time: two of the codes' (twice the independent work between waits), one of bf16 rows
    static constexpr int kUnits = FMT == 16 ? 1 : 2;
    static constexpr int kUnit = FMT == 16 ? 2 * kRows * kRowBytes : kGroup;
    static constexpr int kStage = kUnits * kUnit;
};

template <int FMT, int D, int NT, bool DUP>
struct Traits {
    using L = Layout<FMT, D>;
    static constexpr int kCols = DUP ? 4 : 8 * NT;       // columns of a tile
    // stages of a warp's ring: what keeps about twice the latency-bandwidth product of 45 KB in flight per SM and leaves
    // room for the thread blocks that the registers allow
    static constexpr int kStages = FMT == 16 && D <= 128 && NT == 1 ? 3 : 2;
    static constexpr int kKSteps = D / 16;
    static constexpr int kMTiles = D / 16;
    static constexpr bool kQReg = kKSteps * NT <= 16;    // query fragments in registers (else in shared memory)
    static constexpr int kMergeLd = D + 4;
    static constexpr int kMergeCols = NT == 1 ? 4 : D == 256 ? 4 : D == 128 && NT == 4 ? 8 : 16;   // columns joined at a time: what there is room for
    static constexpr int kMergeSteps = kCols / kMergeCols;
    static constexpr int kRingBytes = kWarps * kStages * L::kStage;
    static constexpr int kMergeBytes = kWarps * kMergeCols * kMergeLd * 4;
    static constexpr int kStatBytes = kWarps * kCols * 3 * 4;
    static constexpr bool kTiled = NT >= 2;              // requests may need several tiles
    static constexpr int kLead = lead_of(kTiled);
    static constexpr int kScanBytes = kTiled ? (kMaxScan + 1) * 4 : 0;
    static constexpr int kQBytes = kQReg ? 0 : kKSteps * NT * 32 * 8;
    static constexpr int kBarStride = kStages * (8 + 8 * L::kUnits) + 128 + 48;   // a warp's barriers, a note (8) per slice, 32 probes, a Seg
    static constexpr int kBarBytes = kWarps * kBarStride;
    static constexpr int kSmem = 1024 + kRingBytes + kMergeBytes + kStatBytes + kQBytes + kScanBytes + kBarBytes;   // (1024: alignment)
    static constexpr int kPart = kCols * (D + 2);        // floats of a partial result: m, l, then the rows
    // thread blocks per SM: what shared memory holds (228 KB, 1 KB of it per block), and the registers of the accumulators
    static constexpr int kBySmem = 233472 / (kSmem + 1024);
    static constexpr int kByRegs = D * NT > 128 ? 2 : NT == 1 ? 4 : 3;
    static constexpr int kOcc = kBySmem < 1 ? 1 : kBySmem < kByRegs ? kBySmem : kByRegs;
};

template <int FMT, int D, int NT, bool DUP>
__global__ void __launch_bounds__(kThreads, Traits<FMT, D, NT, DUP>::kOcc) attend_kernel(const Params p, const __grid_constant__ Maps maps)
{
    using X = Traits<FMT, D, NT, DUP>;
    using L = typename X::L;
    extern __shared__ __align__(128) unsigned char smem_raw[];
    unsigned char* const smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);   // the panels' pattern repeats every 1024 bytes
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = lane >> 2, q4 = lane & 3;

    unsigned char* const ring = smem + warp * (X::kStages * L::kStage);
    float* const merge = reinterpret_cast<float*>(smem + X::kRingBytes);
    float* const stat = reinterpret_cast<float*>(smem + X::kRingBytes + X::kMergeBytes);     // [warp][3][cols]
    uint2* const q_frag = reinterpret_cast<uint2*>(smem + X::kRingBytes + X::kMergeBytes + X::kStatBytes);
    int32_t* const scan = reinterpret_cast<int32_t*>(smem + X::kRingBytes + X::kMergeBytes + X::kStatBytes + X::kQBytes);
    unsigned char* const bars = reinterpret_cast<unsigned char*>(scan) + X::kScanBytes + warp * X::kBarStride;
    uint64_t* const full = reinterpret_cast<uint64_t*>(bars);
    int2* const note = reinterpret_cast<int2*>(bars + 8 * X::kStages);    // .x tokens copied (0: nothing), .y first position

    if (lane == 0) {
        for (int s = 0; s < X::kStages; ++s) mbar_init(&full[s], 1);
        mbar_init_fence();
    }
    __syncwarp();

    // This kernel may be placed on the SMs while the one ahead of it ends; it reads nothing before that, and lets the next one begin
    // only then (what a kernel that may begin early relies on is that everything ahead of this one is over).
    early_start_wait();
    early_start_allow();

    // ---- this thread block's share
    Share w;
    w.scan = nullptr;
    w.tiles = p.col_tiles;
    w.mult = p.H * p.col_tiles;
    if (X::kTiled && p.col_tiles > 1 && p.n_req <= kMaxScan) {
        constexpr int kEach = (kMaxScan + kThreads) / kThreads;
        const int32_t most = most_units(p.H);
        int32_t v[kEach], sum = 0;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int r = tid * kEach + i;
            v[i] = 0;
            if (r < p.n_req) {
                int q0, nq;
                queries_of(p, r, q0, nq);
                const int32_t units = base_of<X::kLead>(p, nullptr, r + 1) - base_of<X::kLead>(p, nullptr, r);
                v[i] = max(X::kLead, units) * ((nq * p.G + X::kCols - 1) / X::kCols);
            }
            sum = add_units(sum, v[i], most);
        }
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int32_t y = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum = add_units(sum, y, most);
        }
        int32_t* const warp_sum = reinterpret_cast<int32_t*>(stat);
        if (lane == 31) warp_sum[warp] = sum;
        int32_t before = __shfl_up_sync(0xffffffffu, sum, 1);
        if (lane == 0) before = 0;
        __syncthreads();
        for (int i = 0; i < warp; ++i) before = add_units(before, warp_sum[i], most);
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int r = tid * kEach + i;
            if (r <= p.n_req) scan[r] = before;
            before = add_units(before, v[i], most);
        }
        __syncthreads();
        w.scan = scan;
        w.mult = p.H;
    }
    w.step = (p.n_req + 30) / 31;
    int32_t* const probes = reinterpret_cast<int32_t*>(note + X::kStages * L::kUnits);
    const int32_t probe = base_of<X::kLead>(p, w.scan, min(lane * w.step, p.n_req));
    probes[lane] = probe;
    __syncwarp();
    w.probes = probes;
    share_out(w, __shfl_sync(0xffffffffu, probe, 0), __shfl_sync(0xffffffffu, probe, 31), blockIdx.x, gridDim.x, X::kLead);
    int32_t begin = w.lo;
    Seg* const head = reinterpret_cast<Seg*>(probes + 32);                // the first segment, for the loads and for the arithmetic
    static_assert(sizeof(Seg) <= 48, "a Seg has 48 bytes of shared memory");
    if (begin < w.hi) {
        Seg s = segment_at<X::kCols, X::kLead>(p, w, begin);
        if (passes_over(w, s, begin, X::kLead) && begin < w.hi) s = segment_at<X::kCols, X::kLead>(p, w, begin);
        if (lane == 0) *head = s;
        __syncwarp();
    }
    Rec* const rec = reinterpret_cast<Rec*>(p.ws + (int64_t)2 * gridDim.x * X::kPart) + blockIdx.x;
    if (tid == 0) rec->parts = 0;

    // ---- the warp's loads run ahead of its arithmetic, across items: a cursor of their own
    constexpr int kU = L::kUnits, kStep = kWarps * kU;
    Seg ps;
    ps.to = -1;
    int32_t p_at = 0;                  // next slice to load of segment ps
    int32_t p_look = 33;               // lanes p_look .. p_look + kU - 1 know the slices to load next; 32: look again, 33: at another segment
    int32_t p_entries = 0;             // entries of the request that count
    int32_t p_end = 0;                 // first position that no column of the tile sees
    int32_t p_all = 0;                 // first position that some column of the tile does not see
    // this lane's slice: where it lies (bf16: block and first token, codes: byte address), its first position, and
    // bits 0..4 tokens to load, bit 5 every column sees all 16, bit 6 (first of a step) the step's other slice follows in memory
    int32_t my_id = 0, my_sub = 0, my_pos = 0;
    const uint8_t* my_src = nullptr;
    uint32_t my_flags = 0;
    bool p_done = false;
    int32_t p_next = begin;            // where the next segment begins
    uint32_t plain = 0;                // bit s: the step in stage s needs no masks
    // what this lane has to know of slice s of segment ps; `fresh`: and all of them of the segment (after the list's entries have
    // been asked for: these are trips to memory that need not wait for one another)
    auto look_up = [&](int32_t s, bool fresh) {
        const int32_t e = s / p.spe, sub = (s - e * p.spe) * kRows;
        const bool mine = s < ps.to;
        const int32_t pos_block = mine && p.positions ? __ldg(p.positions + ps.first + e) : e;
        int32_t id = mine && p.block_ids ? __ldg(p.block_ids + ps.first + e) : -1;
        if (fresh) {
            p_entries = p.counts ? min(ps.n, __ldg(p.counts + ps.r)) : ps.n;
            int q0 = 0, nq = 1;
            if (X::kTiled || p.ctx) queries_of(p, ps.r, q0, nq);
            if (X::kTiled) {
                // the tile's query rows on their way into L2: the item begins some steps from here, and reads them before all else
                // (44 requests with 32 columns: 72 -> 69 us, 100 with 56 columns 137 -> 129; a tile of 8 has too few of them: the
                // shortest calls lose 0.2 us)
                static_assert(X::kCols * (D / 64) <= kThreads, "a line per thread");
                const int line = warp * 32 + lane, cc = ps.ct * X::kCols + line / (D / 64);
                if (line < X::kCols * (D / 64) && cc < nq * p.G) {
                    const int j = cc / p.G;
                    prefetch_l2(p.q + (int64_t)(q0 + j) * p.q_stride + (int64_t)(ps.h * p.G + cc - j * p.G) * D + line % (D / 64) * 64);
                }
            }
            if (p.ctx) {
                const int32_t ctx = __ldg(p.ctx + ps.r) - (nq - 1);
                p_end = ctx + min(nq - 1, (ps.ct * X::kCols + X::kCols - 1) / p.G);
                p_all = ctx + ps.ct * X::kCols / p.G;
            }
        }
        my_flags = 0;
        if (!mine || e >= p_entries || pos_block < 0) return;
        if (!p.block_ids) {
            const int32_t t0 = __ldg(p.table_offsets + ps.r);
            if (!in_row(t0, __ldg(p.table_offsets + ps.r + 1), p.table_size, pos_block)) {
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
        int32_t nv = min(kRows, p.T - sub);
        bool seen = nv == kRows;
        if (p.ctx) {
            const int64_t pos = (int64_t)pos_block * p.T + sub;
            if (pos >= p_end) return;
            nv = (int32_t)min((int64_t)nv, p_end - pos);
            my_pos = (int32_t)pos;
            seen = seen && pos + kRows <= p_all;
        }
        if (FMT == 16) {
            my_id = id;
            my_sub = sub;
        } else {
            my_src = p.k + (int64_t)id * p.k_block + (int64_t)(ps.h * p.spe + (sub >> 4)) * L::kGroup;
        }
        my_flags = (uint32_t)nv | (seen ? 32u : 0u);
    };
    // start the loads of the warp's next step into stage s; every step completes its barrier, with or without bytes
    auto issue = [&](int s) {
        if (p_at >= ps.to) {
            while (!p_done && p_at >= ps.to) {
                if (p_next < w.hi) ps = p_next == begin ? *head : segment_at<X::kCols, X::kLead>(p, w, p_next);
                if (p_next >= w.hi || !begins_here(w, ps, X::kLead)) {
                    p_done = true;
                    break;
                }
                p_next = ps.hi;
                p_at = ps.from + warp * kU;
                p_look = 33;
            }
            if (p_done) return;
        }
        if (p_look >= 32) {
            look_up(p_at + (lane / kU) * kStep + lane % kU, p_look > 32);
            p_look = 0;
            if (kU == 2) {
                const unsigned long long next = __shfl_down_sync(0xffffffffu, (unsigned long long)my_src, 1);
                const uint32_t other = __shfl_down_sync(0xffffffffu, my_flags, 1);
                if (lane % kU == 0 && (my_flags & 31u) && (other & 31u) && next == (unsigned long long)my_src + L::kGroup) my_flags |= 64u;
            }
        }
        const int from = p_look + lane % kU;
        const uint32_t flags = __shfl_sync(0xffffffffu, my_flags, from);
        unsigned char* const dst = ring + s * L::kStage;
        if (FMT == 16) {
            const int32_t id = __shfl_sync(0xffffffffu, my_id, p_look), sub = __shfl_sync(0xffffffffu, my_sub, p_look);
            if (one_lane()) {
                if (flags & 31u) {
                    mbar_expect_tx(&full[s], (uint32_t)(2 * p.box) * L::kRowBytes);
#pragma unroll
                    for (int i = 0; i < D / 64; ++i) {
                        load_panel(dst + i * L::kBf16Panel, &maps.k, i * 64, ps.h, sub, id, &full[s]);
                        load_panel(dst + (D / 64 + i) * L::kBf16Panel, &maps.v, i * 64, ps.h, sub, id, &full[s]);
                    }
                } else {
                    mbar_arrive(&full[s]);
                }
            }
        } else {
            const unsigned long long src = __shfl_sync(0xffffffffu, (unsigned long long)my_src, p_look);
            if (__any_sync(0xffffffffu, flags & 64u)) {          // two slices side by side: one copy
                if (one_lane()) {
                    mbar_expect_tx(&full[s], 2 * L::kGroup);
                    bulk_g2s(dst, (const void*)src, 2 * L::kGroup, &full[s]);
                }
            } else {
                const unsigned long long src1 = __shfl_sync(0xffffffffu, (unsigned long long)my_src, p_look + kU - 1);
                const uint32_t have = __ballot_sync(0xffffffffu, (flags & 31u) != 0u);       // bits 0 and 1: the two slices
                if (one_lane()) {
                    mbar_expect_tx(&full[s], __popc(have & 3u) * L::kGroup);
                    if (have & 1u) bulk_g2s(dst, (const void*)src, L::kGroup, &full[s]);
                    if (have & 2u) bulk_g2s(dst + L::kUnit, (const void*)src1, L::kGroup, &full[s]);
                }
            }
        }
        if (__all_sync(0xffffffffu, flags & 32u)) {
            plain |= 1u << s;
        } else {
            plain &= ~(1u << s);
            const int32_t pos = __shfl_sync(0xffffffffu, my_pos, from);
            if (lane < kU) note[s * kU + lane] = make_int2((int)(flags & 31u), pos);
        }
        p_at += kStep;
        p_look += kU;
    };

#pragma unroll 1
    for (int s = 0; s < X::kStages; ++s) issue(s);
    __syncwarp();
    // the offsets of all requests, shared out among the thread blocks: what no list and no batch can have is reported, whether or not it is
    // met below
    for (int r = blockIdx.x * kThreads + tid; r < p.n_req; r += gridDim.x * kThreads)
        if ((bad_offsets(__ldg(p.offsets + r), __ldg(p.offsets + r + 1), p.total) ||
             (p.q_offsets && bad_queries(p, __ldg(p.q_offsets + r), __ldg(p.q_offsets + r + 1)))) && p.err)
            atomicExch(p.err, 3);

    int stage = 0;
    uint32_t parity = 0;
    bool dead = false;
    const uint32_t ring_u = smem_u32(ring);

    int32_t at = begin;
#pragma unroll 1
    while (at < w.hi) {
        const Seg sg = at == begin ? *head : segment_at<X::kCols, X::kLead>(p, w, at);
        if (!begins_here(w, sg, X::kLead)) break;
        at = sg.hi;
        int q0, nq;
        queries_of(p, sg.r, q0, nq);
        const int cols = sg.n < 0 ? 0 : min(X::kCols, nq * p.G - sg.ct * X::kCols);      // may be <= 0: nothing to write
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

        // ---- query fragments.  bf16 cache: as they are.  Codes: in the order of the codes, scaled by a power of two per column
        // to fp16; `qoff` is what the accumulators start from, `qsum` and `qmul` turn them into scores.
        uint32_t qf[X::kQReg ? X::kKSteps : 1][X::kQReg ? NT : 1][2];
        float qsum[NT][2], qmul[NT][2], qoff[NT][2];
        if (!X::kQReg) __syncthreads();            // the item before may still be read
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int cc = DUP ? g & 3 : nt * 8 + g;
            const int c = c0 + cc;
            const bool live = cc < cols;
            const int j = live ? c / p.G : 0;
            const uint16_t* const qp = p.q + (int64_t)(q0 + j) * p.q_stride + (int64_t)(sg.h * p.G + (live ? c - j * p.G : 0)) * D;
            auto put = [&](int ks, uint32_t b0, uint32_t b1) {
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
                    if (!X::kQReg && (ks & 3) != warp) continue;
                    const uint32_t b0 = live ? __ldg(reinterpret_cast<const uint32_t*>(qp + ks * 16 + 2 * q4)) : 0u;
                    const uint32_t b1 = live ? __ldg(reinterpret_cast<const uint32_t*>(qp + ks * 16 + 8 + 2 * q4)) : 0u;
                    put(ks, b0, b1);
                }
            } else {
                // this lane's quarter of the column: pairs (values 2i, 2i+1) in the order of its code words
                constexpr int kRun = L::kPanelDims / 4;          // neighbouring values a lane has in a panel
                uint32_t raw[D / 8];
#pragma unroll
                for (int i = 0; i < D / 32; ++i) {
                    const int at = (i * 8 / kRun) * L::kPanelDims + q4 * kRun + (i * 8) % kRun;
                    const uint4 x = live ? __ldg(reinterpret_cast<const uint4*>(qp + at)) : make_uint4(0, 0, 0, 0);
                    raw[4 * i] = x.x;
                    raw[4 * i + 1] = x.y;
                    raw[4 * i + 2] = x.z;
                    raw[4 * i + 3] = x.w;
                }
                float most = 0.f;
#pragma unroll
                for (int i = 0; i < D / 8; ++i) most = fmaxf(most, fmaxf(fabsf(bf16lo(raw[i])), fabsf(bf16hi(raw[i]))));
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
                // powers of two (exact) that bring the largest value to [2^14, 2^15): its infinity would be 2^16, and what lies 2^28 below
                // it is still a normal number
                const uint32_t ex = min(max(__float_as_uint(most) >> 23, 15u), 253u);
                const float up = __uint_as_float((268u - ex) << 23), down = __uint_as_float((ex - 14u) << 23);
                float sum = 0.f, odd = 0.f;                      // of the rounded values; `odd`: of those that meet 1024 + 16 c
#pragma unroll
                for (int i = 0; i < D / 32; ++i) {
                    uint32_t b[4];
                    float f[8];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        f[2 * k] = bf16lo(raw[4 * i + k]) * up;
                        f[2 * k + 1] = bf16hi(raw[4 * i + k]) * up;
                    }
                    if (FMT == 4) {
                        // a code word's registers 0..3 hold values (0, 4), (1, 5), (2, 6), (3, 7)
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const float by = k & 1 ? 0.0625f : 1.f;
                            b[k] = pack_f16(f[k] * by, f[k + 4] * by);
                            const float both = f16lo(b[k]) + f16hi(b[k]);
                            if (k & 1) odd += both;
                            else sum += both;
                        }
                        put(2 * i, b[0], b[1]);
                        put(2 * i + 1, b[2], b[3]);
                    } else {
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            b[k] = pack_f16(f[2 * k], f[2 * k + 1]);
                            odd += f16lo(b[k]) + f16hi(b[k]);
                        }
                        put(2 * i, b[0], b[1]);
                        put(2 * i + 1, b[2], b[3]);
                    }
                }
                sum = FMT == 4 ? fmaf(odd, 16.f, sum) : odd;
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                odd += __shfl_xor_sync(0xffffffffu, odd, 1);
                odd += __shfl_xor_sync(0xffffffffu, odd, 2);
                const float mul = down * p.scale_log2;
                sum *= mul;
                odd *= -kOddOffset;
#pragma unroll
                for (int e = 0; e < 2; ++e) {                    // from the column's own lanes to those that hold its scores
                    const int from = (2 * q4 + e) * 4;
                    qsum[nt][e] = __shfl_sync(0xffffffffu, sum, from);
                    qmul[nt][e] = __shfl_sync(0xffffffffu, mul, from);
                    qoff[nt][e] = __shfl_sync(0xffffffffu, odd, from);
                }
            }
        }
        if (!X::kQReg) __syncthreads();

        float o[X::kMTiles][NT][4];
        float m[NT][2], l[NT][2], z[NT][2];
        float base[NT][2], pass[NT][2];           // what is taken off the scores (m, 0 before the first); what moves the maximum
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                m[nt][e] = -INFINITY;
                l[nt][e] = z[nt][e] = 0.f;
                base[nt][e] = 0.f;
                pass[nt][e] = -INFINITY;
            }
#pragma unroll
            for (int mt = 0; mt < X::kMTiles; ++mt)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[mt][nt][i] = 0.f;
        }

        // One step over the slices in the current stage.  MASKED: some column does not see some token of it (the ends of
        // sequences, blocks shorter than a slice); a form of its own, so that the others carry none of that.
        auto step = [&](auto masked_) {
            constexpr bool MASKED = decltype(masked_)::value;
            const uint32_t st_u = ring_u + stage * L::kStage;
            int nv[kU], pos0[kU];
            if (MASKED) {
                bool any = false;
#pragma unroll
                for (int u = 0; u < kU; ++u) {
                    const int2 n = note[stage * kU + u];
                    nv[u] = n.x;
                    pos0[u] = n.y;
                    any |= nv[u] > 0;
                }
                if (!any) return;
            }
            // ---- S^T = K Q^T
            float sc[kU][NT][4];
#pragma unroll
            for (int u = 0; u < kU; ++u) {
                const uint32_t un_u = st_u + u * L::kUnit;
                float s2[NT][4];                             // every other product: half the chain of dependent sums
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        sc[u][nt][i] = FMT == 16 ? 0.f : qoff[nt][i & 1];
                        s2[nt][i] = 0.f;
                    }
                auto qk = [&](int ks, const uint32_t (&a)[4]) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        uint32_t b0, b1;
                        if (X::kQReg) {
                            b0 = qf[X::kQReg ? ks : 0][X::kQReg ? nt : 0][0];
                            b1 = qf[X::kQReg ? ks : 0][X::kQReg ? nt : 0][1];
                        } else {
                            const uint2 b = q_frag[(ks * NT + nt) * 32 + lane];
                            b0 = b.x;
                            b1 = b.y;
                        }
                        float (&to)[4] = NT == 1 && (ks & 1) ? s2[nt] : sc[u][nt];
                        if (FMT == 16) mma(to, a, b0, b1);
                        else mma_f16(to, a, b0, b1);
                    }
                };
                if (FMT == 16) {
                    const uint32_t ka = un_u + (lane & 15) * 128;
#pragma unroll
                    for (int ks = 0; ks < X::kKSteps; ++ks) {
                        uint32_t a[4];
                        ldsm4(a, ka + (ks / 4) * L::kBf16Panel + ((((ks % 4) * 2 + (lane >> 4)) ^ (lane & 7)) << 4));
                        qk(ks, a);
                    }
                } else {
                    constexpr int kChunk = L::kPanel / 4;    // bytes of a row in a panel that a lane reads
#pragma unroll
                    for (int pn = 0; pn < L::kPanels; ++pn) {
                        const uint32_t ka = un_u + pn * (kRows * L::kPanel) + lane * kChunk;
                        uint32_t x[4], y[4];                 // rows g and g + 8
                        lds_words<kChunk>(x, ka);
                        lds_words<kChunk>(y, ka + 8 * L::kPanel);
#pragma unroll
                        for (int i = 0; i < kChunk / 4; ++i) {
                            if (FMT == 4) {
#pragma unroll
                                for (int half = 0; half < 2; ++half) {
                                    const uint32_t a[4] = {k_nibbles(x[i], 2 * half), k_nibbles(y[i], 2 * half),
                                                           k_nibbles(x[i], 2 * half + 1), k_nibbles(y[i], 2 * half + 1)};
                                    qk((pn * (kChunk / 4) + i) * 2 + half, a);
                                }
                            } else {
                                const uint32_t a[4] = {k_bytes(x[i], 0), k_bytes(y[i], 0), k_bytes(x[i], 1), k_bytes(y[i], 1)};
                                qk(pn * (kChunk / 4) + i, a);
                            }
                        }
                    }
                }
                if (NT == 1) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) sc[u][0][i] += s2[0][i];
                }
            }

            // ---- scores in powers of two; rows g (values 0, 1) and g + 8 (values 2, 3)
            float vs[kU][2], vz[kU][2];
#pragma unroll
            for (int u = 0; u < kU; ++u) {
                if (FMT == 16) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int i = 0; i < 4; ++i) sc[u][nt][i] *= p.scale_log2;
                } else {
                    constexpr float mid = FMT == 4 ? 8.f : 128.f;
                    const uint32_t pa = st_u + u * L::kUnit + 2 * kRows * L::kRowBytes + g * 4;
#pragma unroll
                    for (int row = 0; row < 2; ++row) {
                        const uint32_t k0 = lds4(pa + row * 32), v0 = lds4(pa + 64 + row * 32);
                        const float kz = fmaf(bf16lo(k0), mid, bf16hi(k0));      // the centred codes' zero
                        const float ksc = bf16lo(k0);
                        vs[u][row] = bf16lo(v0);
                        vz[u][row] = fmaf(vs[u][row], mid, bf16hi(v0));
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int e = 0; e < 2; ++e)
                                sc[u][nt][2 * row + e] = fmaf(sc[u][nt][2 * row + e], ksc * qmul[nt][e], kz * qsum[nt][e]);
                    }
                }
            }
            uint32_t hide[kU];                               // bit 4 nt + i: value i of tile nt is not seen
#pragma unroll
            for (int u = 0; u < kU; ++u) hide[u] = 0;
            if (MASKED) {
#pragma unroll
                for (int u = 0; u < kU; ++u)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int row = g + (i >> 1) * 8;
                            if (row >= nv[u] || pos0[u] + row >= limit[nt][i & 1]) {
                                sc[u][nt][i] = -INFINITY;
                                hide[u] |= 1u << (4 * nt + i);
                            }
                        }
            }
            // ---- running maximum: moved only when it is passed by more than the slack
            bool passed = false;
            float top[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    top[nt][e] = fmaxf(sc[0][nt][e], sc[0][nt][e + 2]);
                    if (kU == 2) top[nt][e] = fmaxf(top[nt][e], fmaxf(sc[kU - 1][nt][e], sc[kU - 1][nt][e + 2]));
                    passed |= top[nt][e] > pass[nt][e];
                }
            if (__any_sync(0xffffffffu, passed)) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float x = top[nt][e];
                        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                        const float now = fmaxf(m[nt][e], x);
                        // (before the first score nothing but zeros and NaN can have been added: both stay)
                        const float f = m[nt][e] > -INFINITY ? exp2_fast(m[nt][e] - now) : 1.f;
                        if (now > -INFINITY) {
                            m[nt][e] = base[nt][e] = now;
                            pass[nt][e] = now + kMaxSlack;
                        }
                        l[nt][e] *= f;
                        z[nt][e] *= f;
#pragma unroll
                        for (int mt = 0; mt < X::kMTiles; ++mt) {
                            o[mt][nt][e] *= f;
                            o[mt][nt][e + 2] *= f;
                        }
                    }
            }
            // ---- weights, and their bf16 halves with tokens along the columns' other side
            uint32_t ph[kU][NT][2], pl[kU][NT][2];
            float wt[kU][NT][4];
#pragma unroll
            for (int u = 0; u < kU; ++u)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float (&w)[4] = wt[u][nt];
#pragma unroll
                    for (int i = 0; i < 4; ++i) w[i] = exp2_fast(sc[u][nt][i] - base[nt][i & 1]);
                    l[nt][0] += w[0] + w[2];
                    l[nt][1] += w[1] + w[3];
                    if (FMT != 16) {
                        if (MASKED) {                        // what stands in rows that are not seen may be anything
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const bool hd = (hide[u] >> (4 * nt + i)) & 1u;
                                z[nt][i & 1] += hd ? 0.f : w[i] * vz[u][i >> 1];
                                w[i] = hd ? 0.f : w[i] * vs[u][i >> 1];
                            }
                        } else {
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                z[nt][i & 1] = fmaf(w[i], vz[u][i >> 1], z[nt][i & 1]);
                                w[i] *= vs[u][i >> 1];
                            }
                        }
                    }
                    const uint32_t a = FMT == 16 ? pack_below(w[0], w[1]) : pack_bf16(w[0], w[1]);
                    const uint32_t b = FMT == 16 ? pack_below(w[2], w[3]) : pack_bf16(w[2], w[3]);
                    const uint32_t al = pack_bf16(w[0] - bf16lo(a), w[1] - bf16hi(a));
                    const uint32_t bl = pack_bf16(w[2] - bf16lo(b), w[3] - bf16hi(b));
                    if (DUP) {
                        ph[u][nt][0] = transpose8(q4 < 2 ? a : al);
                        ph[u][nt][1] = transpose8(q4 < 2 ? b : bl);
                    } else {
                        ph[u][nt][0] = transpose8(a);
                        ph[u][nt][1] = transpose8(b);
                        pl[u][nt][0] = transpose8(al);
                        pl[u][nt][1] = transpose8(bl);
                    }
                }
            // A row that some columns see and others do not may hold an infinity or a NaN, and a weight of zero would not
            // keep it out of the product: such a slice (the last tokens of a request with several queries) is added up
            // column by column instead.
            bool wild = false;
            if (FMT == 16 && MASKED) {
                unsigned char* const v_rows = ring + stage * L::kStage + (D / 64) * L::kBf16Panel;
                // rows without a seen token: a weight of zero must meet a number
                for (int i = lane; i < (kRows - nv[0]) * (D / 8); i += 32) {
                    const int row = nv[0] + i / (D / 8), x = i % (D / 8);
                    *reinterpret_cast<uint4*>(v_rows + (x / 8) * L::kBf16Panel + row * 128 + (x % 8) * 16) = make_uint4(0, 0, 0, 0);
                }
                fence_proxy_async();                         // (the next load into the stage comes behind these stores)
                if (pos0[0] + nv[0] > limit_min) {
                    for (int i = lane; i < nv[0] * (D / 8); i += 32) {
                        const int row = i / (D / 8), x = i % (D / 8);
                        const uint4 q = *reinterpret_cast<const uint4*>(v_rows + (x / 8) * L::kBf16Panel + row * 128 + (x % 8) * 16);
                        const uint32_t y[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            wild |= (y[k] & 0x7f80u) == 0x7f80u || (y[k] & 0x7f800000u) == 0x7f800000u;
                    }
                    wild = __any_sync(0xffffffffu, wild);
                }
                __syncwarp();
            }
            if (FMT == 16 && wild) {
#pragma unroll 1
                for (int row = 0; row < nv[0]; ++row) {
                    const int src = (row & 7) * 4 + q4;
                    const uint32_t hd = __shfl_sync(0xffffffffu, hide[0], src);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const float w0 = __shfl_sync(0xffffffffu, wt[0][nt][e], src);
                            const float w1 = __shfl_sync(0xffffffffu, wt[0][nt][e + 2], src);
                            const int bit = 4 * nt + e + (row >> 3) * 2;
                            if (((hd >> bit) & 1u) || (DUP && q4 >= 2)) continue;
                            const float w = row < 8 ? w0 : w1;
#pragma unroll
                            for (int mt = 0; mt < X::kMTiles; ++mt)
#pragma unroll
                                for (int k = 0; k < 2; ++k) {
                                    const int x = mt * 2 + k;        // the 16-byte piece of value mt * 16 + k * 8 + g
                                    const uint16_t b = *reinterpret_cast<const uint16_t*>(
                                        ring + stage * L::kStage + (D / 64 + x / 8) * L::kBf16Panel + row * 128 +
                                        (((x % 8) ^ (row & 7)) << 4) + g * 2);
                                    o[mt][nt][e + 2 * k] += w * __uint_as_float((uint32_t)b << 16);
                                }
                        }
                }
            }
            // ---- O^T += V^T P^T
#pragma unroll
            for (int u = 0; u < kU; ++u) {
                const uint32_t un_u = st_u + u * L::kUnit;
                auto pv = [&](int mt, const uint32_t (&a)[4]) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        mma(o[mt][nt], a, ph[u][nt][0], ph[u][nt][1]);
                        if (!DUP) mma(o[mt][nt], a, pl[u][nt][0], pl[u][nt][1]);
                    }
                };
                if (FMT == 16) {
                    if (!wild) {
                        const uint32_t va = un_u + (D / 64) * L::kBf16Panel + ((lane & 7) + ((lane >> 4) & 1) * 8) * 128;
#pragma unroll
                        for (int mt = 0; mt < X::kMTiles; ++mt) {
                            uint32_t a[4];
                            ldsm4_trans(a, va + (mt / 4) * L::kBf16Panel + ((((mt % 4) * 2 + ((lane >> 3) & 1)) ^ (lane & 7)) << 4));
                            pv(mt, a);
                        }
                    }
                } else {
                    constexpr int kChunk = L::kPanel / 4;    // bytes of a lane in half a panel: 2 tokens, 1/8 of the values
#pragma unroll
                    for (int pn = 0; pn < L::kPanels; ++pn) {
                        const uint32_t va = un_u + kRows * L::kRowBytes + pn * (kRows * L::kPanel) + lane * kChunk;
                        uint32_t x[4], y[4];                 // tokens 2 q4, 2 q4 + 1 and the two 8 behind them
                        lds_words<kChunk>(x, va);
                        lds_words<kChunk>(y, va + 8 * L::kPanel);
#pragma unroll
                        for (int i = 0; i < kChunk / 4; ++i) {
                            if (FMT == 4) {
#pragma unroll
                                for (int half = 0; half < 2; ++half) {
                                    const uint32_t a[4] = {v_nibbles(x[i], 2 * half), v_nibbles(x[i], 2 * half + 1),
                                                           v_nibbles(y[i], 2 * half), v_nibbles(y[i], 2 * half + 1)};
                                    pv(pn * (L::kPanelDims / 16) + i * 2 + half, a);
                                }
                            } else {
                                const uint32_t a[4] = {v_bytes(x[i], 0), v_bytes(x[i], 1), v_bytes(y[i], 0), v_bytes(y[i], 1)};
                                pv(pn * (L::kPanelDims / 16) + i, a);
                            }
                        }
                    }
                }
            }
        };
        // ---------------------------------------------------------------------------- the warp's slices of this item
#pragma unroll 1
        for (int32_t s = sg.from + warp * kU; s < sg.to; s += kStep) {
            if (!dead && !mbar_wait(&full[stage], parity)) {
                if (p.err && lane == 0) atomicExch(p.err, 1);
                dead = true;
            }
            if (!dead) {
                if ((plain >> stage) & 1u) step(std::false_type());
                else step(std::true_type());
            }
            __syncwarp();                                        // every lane is done with the stage
            if (!dead) issue(stage);
            __syncwarp();
            if (++stage == X::kStages) {
                stage = 0;
                parity ^= 1u;
            }
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
        if (tid == 0 && sg.lo == sg.begin && sg.hi < sg.end)
            *rec = Rec{parts_of(w, sg, blockIdx.x, gridDim.x), q0, c0, cols, sg.h, {0, 0, 0}};
        float* const part = p.ws + (int64_t)(2 * blockIdx.x + (sg.lo == sg.begin ? 1 : 0)) * X::kPart;
#pragma unroll
        for (int step = 0; step < X::kMergeSteps; ++step) {
            if (step) __syncthreads();
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                if (nt * 8 / X::kMergeCols > step || (nt * 8 + 7) / X::kMergeCols < step) continue;
#pragma unroll
                for (int mt = 0; mt < X::kMTiles; ++mt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float x = o[mt][nt][i];
                        if (DUP) x += __shfl_xor_sync(0xffffffffu, x, 2);
                        const int row = i >> 1;                  // rows g and g + 8 of the tile
                        const int d = FMT == 16 ? mt * 16 + g + row * 8
                                                : (mt / (L::kPanelDims / 16)) * L::kPanelDims + g * (L::kPanelDims / 8) +
                                                      (mt % (L::kPanelDims / 16)) * 2 + row;
                        if ((nt * 8 + 2 * q4) / X::kMergeCols == step)
                            merge[(warp * X::kMergeCols + (nt * 8 + 2 * q4 + (i & 1)) % X::kMergeCols) * X::kMergeLd + d] = x;
                    }
            }
            __syncthreads();
            for (int i = tid; i < X::kMergeCols * (D / 4); i += kThreads) {
                const int cl = i / (D / 4), d = (i - cl * (D / 4)) * 4, cc = step * X::kMergeCols + cl;
                if (cc >= cols) continue;
                float mw[kWarps], top = -INFINITY;
#pragma unroll
                for (int k = 0; k < kWarps; ++k) top = fmaxf(top, mw[k] = stat[(k * 3) * X::kCols + cc]);
                const float off = top == -INFINITY ? 0.f : top;
                float sum = 0.f, zero = 0.f, a[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int k = 0; k < kWarps; ++k) {
                    const float f = exp2_fast(mw[k] - off);
                    const float4 x = *reinterpret_cast<const float4*>(merge + (k * X::kMergeCols + cl) * X::kMergeLd + d);
                    sum = fmaf(f, stat[(k * 3 + 1) * X::kCols + cc], sum);
                    if (FMT != 16) zero = fmaf(f, stat[(k * 3 + 2) * X::kCols + cc], zero);
                    a[0] = fmaf(f, x.x, a[0]);
                    a[1] = fmaf(f, x.y, a[1]);
                    a[2] = fmaf(f, x.z, a[2]);
                    a[3] = fmaf(f, x.w, a[3]);
                }
                if (FMT != 16) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) a[k] += zero;
                }
                if (whole) {
                    const int c = c0 + cc, j = c / p.G;
                    const int64_t row = (int64_t)(q0 + j) * p.Hq + sg.h * p.G + (c - j * p.G);
                    const float inv = sum == 0.f ? 0.f : 1.f / sum;
                    const uint2 y = sum == 0.f ? make_uint2(0u, 0u) : make_uint2(pack_bf16(a[0] * inv, a[1] * inv), pack_bf16(a[2] * inv, a[3] * inv));
                    *reinterpret_cast<uint2*>(p.out + row * D + d) = y;
                    if (d == 0 && p.lse) p.lse[row] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * kLn2;
                } else {
                    *reinterpret_cast<float4*>(part + 2 * X::kCols + cc * D + d) = make_float4(a[0], a[1], a[2], a[3]);
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
    if (dead) {
        for (int s = stage; s < X::kStages; ++s) mbar_wait(&full[s], parity);
        for (int s = 0; s < stage; ++s) mbar_wait(&full[s], parity ^ 1u);
    }
}

// Joins the partial results of the item that begins in thread block blockIdx.x and ends in a later one, eight columns per
// blockIdx.y.  Part 0 is that block's trailing result, the others are leading ones.  Latency is all there is to it, and as many
// thread blocks as can be at once: a few parts are joined column by column, one warp each; many of them by all warps together, two
// columns at a time.  (All warps over every item, eight columns in registers: 44 requests with 32 columns spent 21 us here, 5.7 so;
// 6 requests of 6 650..29 600 tokens, 256 values a head, 25 parts: 12 us; one request of 130 944 tokens, 37 parts a head: 11 us.)
template <int D, int COLS>
__global__ void __launch_bounds__(256, 4) attend_join_kernel(const Params p, const int n_blocks)
{
    constexpr int kC = COLS < 8 ? COLS : 8;
    constexpr int kJoinWarps = 8;
    constexpr int kPart = COLS * (D + 2);
    constexpr int kW = D < 128 ? 2 : 4;               // values of one load
    constexpr int kV = D / 32 / kW;                   // loads of a row per lane
    struct __align__(4 * kW) Vec {
        float x[kW];
    };
    __shared__ Vec buf[kJoinWarps][2][D / kW];
    __shared__ float sums[2];
    early_start_wait();
    const Rec rec = reinterpret_cast<const Rec*>(p.ws + (int64_t)2 * n_blocks * kPart)[blockIdx.x];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int y0 = blockIdx.y * 8;
    if (rec.parts == 0 || y0 >= rec.cols) return;

    const float* const first = p.ws + (int64_t)(2 * blockIdx.x + 1) * kPart + y0;
    const float* const rest = p.ws + (int64_t)2 * blockIdx.x * kPart + y0;
    auto part_of = [&](int i) { return i == 0 ? first : rest + (int64_t)2 * i * kPart; };
    auto row_of = [&](Vec (&x)[kV], int i, int c) {
        const Vec* const s = reinterpret_cast<const Vec*>(part_of(i) + 2 * COLS + y0 * (D - 1) + c * D);
#pragma unroll
        for (int v = 0; v < kV; ++v) x[v] = s[v * 32 + lane];
    };
    auto add = [&](float (&acc)[kV][kW], const Vec (&x)[kV], float w) {
#pragma unroll
        for (int v = 0; v < kV; ++v)
#pragma unroll
            for (int k = 0; k < kW; ++k) acc[v][k] = fmaf(w, x[v].x[k], acc[v][k]);
    };
    auto over_lanes = [](float x, auto op) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) x = op(x, __shfl_xor_sync(0xffffffffu, x, o));
        return x;
    };
    auto most = [](float x, float y) { return fmaxf(x, y); };
    auto plus = [](float x, float y) { return x + y; };
    auto put = [&](int cl, const float (&acc)[kV][kW], float top, float l) {       // one column's result, by a warp
        const int c = rec.c0 + y0 + cl, j = c / p.G;
        const int64_t row = (int64_t)(rec.q0 + j) * p.Hq + rec.h * p.G + (c - j * p.G);
        const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
        for (int v = 0; v < kV; ++v) {
            uint32_t y[kW / 2];
#pragma unroll
            for (int k = 0; k < kW / 2; ++k) y[k] = l == 0.f ? 0u : pack_bf16(acc[v][2 * k] * inv, acc[v][2 * k + 1] * inv);
            uint32_t* const to = reinterpret_cast<uint32_t*>(p.out + row * D) + (v * 32 + lane) * (kW / 2);
            if constexpr (kW == 4) *reinterpret_cast<uint2*>(to) = make_uint2(y[0], y[1]);
            else *to = y[0];
        }
        if (lane == 0 && p.lse) p.lse[row] = l == 0.f ? -INFINITY : (top + log2f(l)) * kLn2;
    };
    const int cols = min(kC, rec.cols - y0);
    if (rec.parts <= 8) {
        if (warp >= cols) return;
        const bool mine = lane < rec.parts;
        const float* const s = part_of(mine ? lane : 0) + warp;
        Vec x[2][kV];
        row_of(x[0], 0, warp);
        if (rec.parts > 1) row_of(x[1], 1, warp);
        const float m = mine ? s[0] : -INFINITY, l0 = mine ? s[COLS] : 0.f;
        const float top = over_lanes(m, most);
        const float f = exp2_fast(m - (top == -INFINITY ? 0.f : top));
        const float l = over_lanes(f * l0, plus);
        float acc[kV][kW] = {};
        add(acc, x[0], __shfl_sync(0xffffffffu, f, 0));
        if (rec.parts > 1) add(acc, x[1], __shfl_sync(0xffffffffu, f, 1));
#pragma unroll 2
        for (int i = 2; i < rec.parts; ++i) {
            row_of(x[0], i, warp);
            add(acc, x[0], __shfl_sync(0xffffffffu, f, i));
        }
        put(warp, acc, top, l);
        return;
    }
    float top[kC];
#pragma unroll
    for (int c = 0; c < kC; ++c) top[c] = -INFINITY;
    for (int i = lane; i < rec.parts; i += 32) {
        const float4* const s = reinterpret_cast<const float4*>(part_of(i));
#pragma unroll
        for (int c = 0; c < kC; c += 4) {
            const float4 x = s[c / 4];
            top[c] = fmaxf(top[c], x.x);
            top[c + 1] = fmaxf(top[c + 1], x.y);
            top[c + 2] = fmaxf(top[c + 2], x.z);
            top[c + 3] = fmaxf(top[c + 3], x.w);
        }
    }
#pragma unroll
    for (int c = 0; c < kC; ++c) top[c] = over_lanes(top[c], most);
#pragma unroll
    for (int c0 = 0; c0 < kC; c0 += 2) {
        if (c0 >= cols) break;
        if (c0) __syncthreads();
        float acc[2][kV][kW] = {}, sum[2] = {};
        const float off[2] = {top[c0] == -INFINITY ? 0.f : top[c0], top[c0 + 1] == -INFINITY ? 0.f : top[c0 + 1]};
#pragma unroll 1
        for (int from = 0; from < rec.parts; from += 32) {        // 32 parts at a time, their factors in the lanes
            float f[2] = {0.f, 0.f};
            if (from + lane < rec.parts) {
                const float* const s = part_of(from + lane) + c0;
                const float2 m = *reinterpret_cast<const float2*>(s), l = *reinterpret_cast<const float2*>(s + COLS);
                f[0] = exp2_fast(m.x - off[0]);
                f[1] = exp2_fast(m.y - off[1]);
                sum[0] = fmaf(f[0], l.x, sum[0]);
                sum[1] = fmaf(f[1], l.y, sum[1]);
            }
            const int end = min(32, rec.parts - from);
#pragma unroll
            for (int k = 0; k < 32 / kJoinWarps; ++k) {
                const int j = warp + k * kJoinWarps;
                if (j >= end) break;
                Vec x[2][kV];
                row_of(x[0], from + j, c0);
                row_of(x[1], from + j, c0 + 1);
                add(acc[0], x[0], __shfl_sync(0xffffffffu, f[0], j));
                add(acc[1], x[1], __shfl_sync(0xffffffffu, f[1], j));
            }
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
            for (int v = 0; v < kV; ++v) {
                Vec x;
#pragma unroll
                for (int k = 0; k < kW; ++k) x.x[k] = acc[e][v][k];
                buf[warp][e][v * 32 + lane] = x;
            }
            if (warp == 0) {
                sum[e] = over_lanes(sum[e], plus);
                if (lane == 0) sums[e] = sum[e];
            }
        }
        __syncthreads();
        if (warp < 2 && c0 + warp < cols) {
            float all[kV][kW] = {};
#pragma unroll
            for (int k = 0; k < kJoinWarps; ++k) {
                Vec x[kV];
#pragma unroll
                for (int v = 0; v < kV; ++v) x[v] = buf[k][warp][v * 32 + lane];
                add(all, x, 1.f);
            }
            put(c0 + warp, all, top[c0 + (warp ? 1 : 0)], sums[warp]);
        }
    }
}

// ---------------------------------------------------------------------------------------------------- host side

// Columns of a tile for `cols` query rows of a KV head.  A tile reads K and V once and pays for its matrix instructions and
// weights: a tile of 32 takes about 1.3 times one of 16 (24 requests of 6400 tokens, 128 values a head, 8 heads: 32 columns 129 us
// in one tile, 202 us in two; 40 columns 235 us in two, 223 us in three).  Codes are decoded once per tile, but beside 128
// accumulators there are no registers left for it: 16 is their widest (8 requests of 8192 tokens, 32 columns, 4 bits: 67 us against
// 78 us with 32), as it is with 256 values a head.
inline int tile_cols(int cols, int head_dim, int format)
{
    if (cols <= 4) return 4;
    if (cols <= 8) return 8;
    if (format != 16 || head_dim == 256) return 16;
    return 2 * ((cols + 15) / 16) <= 3 * ((cols + 31) / 32) ? 16 : 32;
}

// what a launch needs for one shape (asked for without maps: nothing is launched)
struct Plan {
    int32_t ctas;                      // thread blocks resident on the device at once
    int32_t part;                      // floats of a partial result
    int32_t cols;                      // columns of a tile
};

template <int FMT, int D, int NT, bool DUP>
int32_t run(const Params& p, const Maps* maps, Plan* plan, cudaStream_t st)
{
    using X = Traits<FMT, D, NT, DUP>;
    plan->ctas = sm_count() * X::kOcc;
    plan->part = X::kPart;
    plan->cols = X::kCols;
    if (!maps) return UCMX_OK;
    auto kern = attend_kernel<FMT, D, NT, DUP>;
    // the attribute sticks to the function on a device: once is enough (2 us of host time a call)
    static std::atomic<uint64_t> set{0};
    int dev = 0;
    UCMX_CUDA(cudaGetDevice(&dev));
    if (dev >= 64 || !((set.load(std::memory_order_acquire) >> dev) & 1u)) {
        UCMX_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, X::kSmem));
        if (dev < 64) set.fetch_or(1ull << dev, std::memory_order_release);
    }
    // (attend_common has bounded it) a thread block per lead: an item of a few slices has one of its own
    const int64_t all = ((int64_t)p.total * p.spe + (int64_t)p.n_req * X::kLead) * p.H * p.col_tiles;
    int64_t grid = (all + X::kLead - 1) / X::kLead;
    if (grid > plan->ctas) grid = plan->ctas;
    if (grid < 1) grid = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = X::kSmem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    UCMX_CUDA(cudaLaunchKernelEx(&cfg, kern, p, *maps));
    UCMX_LAUNCH_CHECK("attend_kernel");
    // no item can be split?  (A captured batch may use less than its capacity: then the shares are smaller, never larger.)
    const int64_t size = (all + grid - 1) / grid;
    if (grid == 1 || (int64_t)p.total * p.spe + X::kLead <= whole_of((int)(size < 64 ? size : 64), X::kLead)) return UCMX_OK;
    cfg.gridDim = dim3((unsigned)grid - 1, X::kCols <= 8 ? 1 : X::kCols / 8);
    cfg.blockDim = dim3(256);
    cfg.dynamicSmemBytes = 0;
    UCMX_CUDA(cudaLaunchKernelEx(&cfg, attend_join_kernel<D, X::kCols>, p, (int)grid));
    UCMX_LAUNCH_CHECK("attend_join_kernel");
    return UCMX_OK;
}

template <int FMT, int D>
int32_t run_cols(const Params& p, int cols, const Maps* maps, Plan* plan, cudaStream_t st)
{
    switch (tile_cols(cols, D, FMT)) {
        case 4: return run<FMT, D, 1, true>(p, maps, plan, st);
        case 8: return run<FMT, D, 1, false>(p, maps, plan, st);
        case 16: return run<FMT, D, 2, false>(p, maps, plan, st);
        default:
            if constexpr (D != 256 && FMT == 16) return run<FMT, D, 4, false>(p, maps, plan, st);
            return UCMX_EUNSUPPORTED;
    }
}

template <int FMT>
int32_t run_format(const Params& p, int head_dim, int cols, const Maps* maps, Plan* plan, cudaStream_t st)
{
    switch (head_dim) {
        case 64: return run_cols<FMT, 64>(p, cols, maps, plan, st);
        case 128: return run_cols<FMT, 128>(p, cols, maps, plan, st);
        case 256: return run_cols<FMT, 256>(p, cols, maps, plan, st);
        default: return UCMX_EUNSUPPORTED;
    }
}

// the three formats live in files of their own
int32_t run_bf16(const Params& p, int head_dim, int cols, const Maps* maps, Plan* plan, cudaStream_t st);
int32_t run_q8(const Params& p, int head_dim, int cols, const Maps* maps, Plan* plan, cudaStream_t st);
int32_t run_q4(const Params& p, int head_dim, int cols, const Maps* maps, Plan* plan, cudaStream_t st);

}  // namespace attend
}  // namespace ucmx
