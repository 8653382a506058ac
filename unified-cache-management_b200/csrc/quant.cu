// The quantised paged KV cache: rows of new tokens or whole bf16 blocks in, whole blocks back out.
//
// Per row x (one token, one KV head, K or V): zero = min x, scale = bf16((max x - min x) / L), code = nearest((x - zero) /
// scale), L = 15 or 255; the layout is described at ucmx_quant_geometry.  All three kernels are streams: a row of 128 values is
// 256 bytes on the bf16 side and 68 (132) on the other, with one reduction over the lanes that hold it in between.
//
// Sixteen values per lane in pieces of eight (what 16 bytes hold), so that a row is 4, 8 or 16 lanes and a warp holds eight, four
// or two neighbouring tokens of one head: what is done once per row is shared by that many.
// V's layout puts the codes of tokens 2i and 2i+1 side by side in pairs of bytes: neighbouring rows of the warp exchange words, so
// that V moves in 32-bit words like K (a token whose partner is not in the call stores 16-bit pieces).
//
// Arithmetic.  The range comes from packed bf16 maxima (of x and of -x; NaN wins).  Differences are taken of halves: exact, and no
// overflow for any finite row.  A reciprocal, a rounding to the integers by adding 2^23, and the residual x - code*scale, which is
// exact in fp32: where it is half a step or more (ties, and quotients the reciprocal put on the wrong side) the code is settled by
// it and by what the difference x - zero was rounded by.  A division per value, and fp64 for the ties, were the bound of this kernel.
//
// Measured on a B200 (8 heads of 128 values): 300 blocks of 128 tokens to 8 bits in 66 us (3.6 TB/s of both sides' bytes; floor
// 36 us), back in 42 us (5.7 TB/s); 8144 tokens to 4 bits in 20 us, back in 12 us.  Writing is bound by instructions (74 warp
// instructions a row, 69 % of the issue slots; 4 bits 61 %); reading comes within a sixth of the copy's rate with 81 % of them.
#include "common.cuh"

namespace ucmx {
namespace {

constexpr int kRows = 16;

template <int BITS, int D>
struct Q {
    static constexpr int kRowBytes = D * BITS / 8;
    static constexpr int kPanel = kRowBytes < 64 ? kRowBytes : 64;
    static constexpr int kPieces = 2;                    // pieces of 8 values a lane holds: lr, lr + kLanes
    static constexpr int kDims = 8 * kPieces;
    static constexpr int kLanes = D / kDims;             // lanes of a row
    static constexpr int kTokens = 32 / kLanes;          // rows of a warp: neighbouring tokens of one head
    static constexpr int kWords = BITS / 4;              // code words of a piece
    static constexpr int kGroup = 2 * kRows * kRowBytes + 2 * kRows * 4;
    static constexpr int kTop = (1 << BITS) - 1;
};

struct QuantParams {
    const uint16_t* k;                 // bf16 side: rows of tokens, or a paged cache
    const uint16_t* v;
    int64_t k_block, v_block;          // elements
    int64_t k_token, v_token;
    uint8_t* cache;
    int64_t block_stride;              // bytes
    int64_t n_blocks;                  // of the quantised cache
    int64_t n_src;                     // blocks of the bf16 cache
    const int64_t* slots;              // token form
    const int32_t* ids;                // block forms
    const int32_t* out_slots;
    int32_t T, H;
    int64_t n;                         // tokens or blocks
    uint32_t items;                    // pieces of work, one per warp
    uint32_t head_chunks;              // pieces that the heads are cut into,
    int32_t heads_per;                 // of this many heads
    int32_t* err;
};

constexpr float kMagic = 8388608.f;    // 2^23: floats of this size count in ones

__device__ __forceinline__ uint32_t pack2(float lo, float hi)
{
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b)
{
    uint32_t r;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ uint32_t min2(uint32_t a, uint32_t b)
{
    uint32_t r;
    asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

// two fp32 operations in one instruction
struct F2 {
    float x, y;
};
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c)
{
    F2 r;
    asm("{\n\t.reg .b64 a, b, c;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
        "fma.rn.f32x2 a, a, b, c;\n\tmov.b64 {%0, %1}, a;\n\t}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b)
{
    F2 r;
    asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}

// Settles a code whose residual is half a step or more.  c: the code so far; v, lo: the value and the row's smallest.
__device__ __forceinline__ float settle(float c, float v, float lo, float half_scale)
{
    const float a = 0.5f * v, b = -0.5f * lo, hx = a + b;
    const float r = fmaf(-c, half_scale, hx);
    const float bb = hx - a;
    const float err = (a - (hx - bb)) + (b - bb);        // what the difference was rounded by
    const float to = r > 0.f ? 1.f : -1.f;
    bool move = fabsf(r) > 0.5f * half_scale;
    if (!move) {                                         // a tie of the rounded difference
        move = __float_as_uint(c + kMagic) & 1u;         // of an exact one: the even code
        if (err != 0.f) {                                // which side the exact difference lies on (as far as fp64 would see it)
            const float unit = __uint_as_float(__float_as_uint(hx) & 0x7f800000u) * 1.1102230246251565e-16f;     // 2^-53 of hx's power of two
            if (fabsf(err) > unit) move = (err > 0.f) == (r > 0.f);
        }
    }
    return move ? c + to : c;
}

// byte offset of piece `pc` of a row (8 values) inside K's part of a group / of unit u (2 bytes of a row) inside V's part
template <int BITS, int D>
__device__ __forceinline__ int k_at(int t, int pc)
{
    using X = Q<BITS, D>;
    const int b = pc * X::kWords * 4;
    return (b / X::kPanel) * (kRows * X::kPanel) + t * X::kPanel + b % X::kPanel;
}
template <int BITS, int D>
__device__ __forceinline__ int v_at(int t, int u)
{
    using X = Q<BITS, D>;
    const int b = (u * 2) % X::kPanel;
    constexpr int kChunk = X::kPanel / 8;
    return (u * 2 / X::kPanel) * (kRows * X::kPanel) + (t >> 3) * (8 * X::kPanel) + (b / kChunk) * X::kPanel + ((t & 7) >> 1) * (2 * kChunk) +
           (b % kChunk) / 2 * 4 + (t & 1) * 2;
}

// Piece of work -> (token group, K or V, first head); heads are innermost, neighbouring warps read neighbouring rows.
struct Piece {
    uint32_t tg;
    int32_t kv, h;
};
__device__ __forceinline__ Piece piece_of(uint32_t item, const QuantParams& p)
{
    Piece x;
    const uint32_t a = item / p.head_chunks;
    x.h = (int32_t)(item - a * p.head_chunks) * p.heads_per;
    x.kv = (int32_t)(a & 1);
    x.tg = a >> 1;
    return x;
}

// heads_per heads of one token group per warp, HC at a time with their loads in flight at once.
template <int BITS, int D, bool BLOCKS, int HC>
__global__ void __launch_bounds__(256, 4) quant_write_kernel(const QuantParams p)
{
    using X = Q<BITS, D>;
    const int lane = threadIdx.x & 31, lr = lane % X::kLanes, row = lane / X::kLanes;
    const uint32_t item = blockIdx.x * 8 + (threadIdx.x >> 5);
    if (item >= p.items) return;
    const Piece x = piece_of(item, p);
    // ---- where the rows come from and where they go
    const uint16_t* src = x.kv ? p.v : p.k;
    int64_t block = -1;
    int t = 0;
    if (BLOCKS) {
        const uint32_t per_block = (uint32_t)p.T / X::kTokens;
        const uint32_t i = x.tg / per_block;
        t = (int)(x.tg - i * per_block) * X::kTokens + row;
        const int id = checked_block_id(p.ids, i, p.n_src, lane == 0 ? p.err : nullptr);
        const int64_t out = checked_out_row(p.out_slots, i, p.n_blocks, lane == 0 ? p.err : nullptr);
        if (id < 0 || out < 0) return;                   // (the same for the whole warp)
        block = out;
        src += (int64_t)id * (x.kv ? p.v_block : p.k_block) + (int64_t)t * (x.kv ? p.v_token : p.k_token);
    } else {
        const int64_t i = (int64_t)x.tg * X::kTokens + row;
        int64_t slot = i < p.n ? __ldg(p.slots + i) : -1;
        if (slot >= p.n_blocks * p.T) {
            if (p.err && lr == 0) atomicExch(p.err, 3);
            slot = -1;
        }
        if (slot >= 0) {
            block = slot < (1ll << 32) ? (int64_t)((uint32_t)slot / (uint32_t)p.T) : slot / p.T;
            t = (int)(slot - block * p.T);
        }
        src += i * (x.kv ? p.v_token : p.k_token);
    }
    const bool live = block >= 0;
    src += (int64_t)x.h * D + lr * 8;
    const int head_end = min(p.H, x.h + p.heads_per);
    // is the neighbouring row the other token of a pair?
    const int64_t place = live ? block * p.T + t : -2 - row;
    const int64_t other = __shfl_xor_sync(0xffffffffu, place, X::kLanes);
    const bool paired = live && other == (place ^ 1) && (place & 1) == (row & 1);
    const int tt = t % kRows;
    const int group_step = (p.T / kRows) * X::kGroup;
    uint8_t* group = p.cache + block * p.block_stride + (int64_t)x.h * group_step + (t / kRows) * X::kGroup;
#pragma unroll 1
    for (int h = x.h; h < head_end; h += HC, src += HC * D) {
        uint4 raw[HC][X::kPieces];
#pragma unroll
        for (int c = 0; c < HC; ++c)
#pragma unroll
            for (int i = 0; i < X::kPieces; ++i)
                raw[c][i] = live && h + c < head_end ? ld_stream16(src + c * D + i * X::kLanes * 8) : make_uint4(0, 0, 0, 0);
        // ---- each row's range: (max x, max -x) in one register
        uint32_t range[HC];
#pragma unroll
        for (int c = 0; c < HC; ++c) {
            uint32_t hi2 = raw[c][0].x, lo2 = raw[c][0].x;
#pragma unroll
            for (int i = 0; i < X::kPieces; ++i) {
                hi2 = max2(max2(max2(max2(hi2, raw[c][i].x), raw[c][i].y), raw[c][i].z), raw[c][i].w);
                lo2 = min2(min2(min2(min2(lo2, raw[c][i].x), raw[c][i].y), raw[c][i].z), raw[c][i].w);
            }
            lo2 ^= 0x80008000u;
            range[c] = max2(__byte_perm(hi2, lo2, 0x5410), __byte_perm(hi2, lo2, 0x7632));
#pragma unroll
            for (int o = 1; o < X::kLanes; o <<= 1) range[c] = max2(range[c], __shfl_xor_sync(0xffffffffu, range[c], o));
        }
        // ---- scale and zero: lane lr works them out for head lr % HC, the others fetch them
        uint32_t my_sz;
        float my_inv;
        {
            uint32_t r = range[0];
#pragma unroll
            for (int c = 1; c < HC; ++c)
                if (lr % HC == c) r = range[c];
            const float hi = bf16lo(r), lo = -bf16hi(r);
            const bool bad = !((hi - hi) + (lo - lo) == 0.f);
            my_sz = f32_to_bf16_bits(fmaf(0.5f, hi, -0.5f * lo) / (0.5f * (float)X::kTop)) | (__float_as_uint(lo) & 0xffff0000u);
            if (bad) my_sz = 0x7fc07fc0u;
            my_inv = __fdividef(1.f, 0.5f * bf16lo(my_sz));
        }
#pragma unroll
        for (int c = 0; c < HC; ++c, group += group_step) {
            if (h + c >= head_end) break;
            const uint32_t sz = HC == 1 ? my_sz : __shfl_sync(0xffffffffu, my_sz, row * X::kLanes + c);
            const float inv = HC == 1 ? my_inv : __shfl_sync(0xffffffffu, my_inv, row * X::kLanes + c);
            const float scale = bf16lo(sz), half_scale = 0.5f * scale, lo = bf16hi(sz), half_lo = 0.5f * lo;
            const float half = 0.5f * half_scale, most = (float)X::kTop * half_scale;
            uint8_t* const part = group + kRows * X::kRowBytes;
#pragma unroll
            for (int pc = 0; pc < X::kPieces; ++pc) {
                const uint32_t q[4] = {raw[c][pc].x, raw[c][pc].y, raw[c][pc].z, raw[c][pc].w};
                auto value = [&](int i) { return i & 1 ? bf16hi(q[i / 2]) : bf16lo(q[i / 2]); };
                // ---- codes, as floats
                float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                if (scale >= 1e-30f) {
                    float worst = 0.f, e[8];
#pragma unroll
                    for (int i = 0; i < 8; i += 2) {
                        F2 hx = fma2({value(i), value(i + 1)}, {0.5f, 0.5f}, {-half_lo, -half_lo});
                        if (BITS == 8) {                     // 255 steps of a scale that was rounded down may end beyond 255.5; 15 cannot
                            hx.x = fminf(hx.x, most);
                            hx.y = fminf(hx.y, most);
                        }
                        const F2 d = add2(fma2(hx, {inv, inv}, {kMagic, kMagic}), {-kMagic, -kMagic});
                        const F2 r = fma2(d, {-half_scale, -half_scale}, hx);
                        f[i] = d.x;
                        f[i + 1] = d.y;
                        e[i] = fabsf(r.x);
                        e[i + 1] = fabsf(r.y);
                        worst = fmaxf(worst, fmaxf(e[i], e[i + 1]));
                    }
                    if (worst >= half) {
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            if (e[i] >= half) f[i] = settle(f[i], value(i), lo, half_scale);
                    }
                } else if (scale > 0.f) {                    // the reciprocal would leave the range: in fp64.  (Neither: a scale of 0, or NaN)
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        f[i] = (float)fmin(rint(((double)value(i) - (double)lo) / (double)scale), (double)X::kTop);
                }
                // ---- 16 bits at a time: the codes side by side in one float of 2^23
                uint32_t w[X::kWords];
                constexpr int kIn16 = 16 / BITS;
#pragma unroll
                for (int i = 0; i < X::kWords; ++i) {
                    uint32_t half[2];
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const int at = (2 * i + j) * kIn16;
                        float a = kMagic + f[at];
#pragma unroll
                        for (int k = 1; k < kIn16; ++k) a = fmaf(f[at + k], (float)(1 << (BITS * k)), a);
                        half[j] = __float_as_uint(a);
                    }
                    w[i] = __byte_perm(half[0], half[1], 0x5410);
                }
                const int piece = pc * X::kLanes + lr;
                if (x.kv == 0) {
                    if (live) {
                        uint8_t* const d = group + k_at<BITS, D>(tt, piece);
                        if (X::kWords == 1) *reinterpret_cast<uint32_t*>(d) = w[0];
                        else *reinterpret_cast<uint2*>(d) = make_uint2(w[0], w[X::kWords - 1]);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < X::kWords; ++i) {
                        const uint32_t y = __shfl_xor_sync(0xffffffffu, w[i], X::kLanes);
                        const int u = (piece * X::kWords + i) * 2;
                        if (paired) {
                            *reinterpret_cast<uint32_t*>(part + v_at<BITS, D>(tt & ~1, u + (row & 1))) =
                                __byte_perm(w[i], y, (row & 1) ? 0x3276 : 0x5410);
                        } else if (live) {
                            *reinterpret_cast<uint16_t*>(part + v_at<BITS, D>(tt, u)) = (uint16_t)w[i];
                            *reinterpret_cast<uint16_t*>(part + v_at<BITS, D>(tt, u + 1)) = (uint16_t)(w[i] >> 16);
                        }
                    }
                }
            }
            if (live && lr == 0)
                *reinterpret_cast<uint32_t*>(group + 2 * kRows * X::kRowBytes + x.kv * (kRows * 4) + tt * 4) = sz;
        }
    }
}

template <int BITS, int D, int HC>
__global__ void __launch_bounds__(256) quant_read_kernel(const QuantParams p)
{
    using X = Q<BITS, D>;
    const int lane = threadIdx.x & 31, lr = lane % X::kLanes, row = lane / X::kLanes;
    const uint32_t item = blockIdx.x * 8 + (threadIdx.x >> 5);
    if (item >= p.items) return;
    const Piece x = piece_of(item, p);
    const uint32_t per_block = (uint32_t)p.T / X::kTokens;
    const uint32_t i = x.tg / per_block;
    const int t = (int)(x.tg - i * per_block) * X::kTokens + row;
    const int id = checked_block_id(p.ids, i, p.n_blocks, lane == 0 ? p.err : nullptr);
    const int64_t out = checked_out_row(p.out_slots, i, p.n_src, lane == 0 ? p.err : nullptr);
    if (id < 0 || out < 0) return;                       // (the same for the whole warp)
    const int group_step = (p.T / kRows) * X::kGroup;
    const uint8_t* const group = p.cache + (int64_t)id * p.block_stride + (int64_t)x.h * group_step + (t / kRows) * X::kGroup;
    const int tt = t % kRows;
    uint32_t w[HC][X::kPieces][X::kWords], sz[HC];
#pragma unroll
    for (int c = 0; c < HC; ++c) {
        if (x.h + c >= p.H) break;
        const uint8_t* const g = group + c * group_step;
#pragma unroll
        for (int pc = 0; pc < X::kPieces; ++pc) {
            const int piece = pc * X::kLanes + lr;
            if (x.kv == 0) {
                const uint8_t* const s = g + k_at<BITS, D>(tt, piece);
                if (X::kWords == 1) {
                    w[c][pc][0] = __ldg(reinterpret_cast<const uint32_t*>(s));
                } else {
                    const uint2 y = __ldg(reinterpret_cast<const uint2*>(s));
                    w[c][pc][0] = y.x;
                    w[c][pc][X::kWords - 1] = y.y;
                }
            } else {
#pragma unroll
                for (int j = 0; j < X::kWords; ++j)
                    w[c][pc][j] = __ldg(reinterpret_cast<const uint32_t*>(g + kRows * X::kRowBytes +
                                                                           v_at<BITS, D>(tt & ~1, (piece * X::kWords + j) * 2 + (row & 1))));
            }
        }
        sz[c] = __ldg(reinterpret_cast<const uint32_t*>(g + 2 * kRows * X::kRowBytes + x.kv * (kRows * 4) + tt * 4));
    }
    uint16_t* const dst = const_cast<uint16_t*>(x.kv ? p.v : p.k) + out * (x.kv ? p.v_block : p.k_block) +
                          (int64_t)t * (x.kv ? p.v_token : p.k_token) + (int64_t)x.h * D + lr * 8;
#pragma unroll
    for (int c = 0; c < HC; ++c) {
        if (x.h + c >= p.H) break;
        const float scale = bf16lo(sz[c]), zero = bf16hi(sz[c]);
#pragma unroll
        for (int pc = 0; pc < X::kPieces; ++pc) {
            float f[8];
#pragma unroll
            for (int j = 0; j < X::kWords; ++j) {
                uint32_t u = w[c][pc][j];
                if (x.kv) u = __byte_perm(u, __shfl_xor_sync(0xffffffffu, u, X::kLanes), (row & 1) ? 0x3276 : 0x5410);
                const uint32_t even = BITS == 4 ? u & 0x0f0f0f0fu : u, odd = BITS == 4 ? (u >> 4) & 0x0f0f0f0fu : 0u;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float a = __uint_as_float(__byte_perm(even, 0x4b000000u, 0x7440 + k)) - kMagic;
                    if (BITS == 4) {
                        const float b = __uint_as_float(__byte_perm(odd, 0x4b000000u, 0x7440 + k)) - kMagic;
                        f[2 * k] = fmaf(a, scale, zero);
                        f[2 * k + 1] = fmaf(b, scale, zero);
                    } else {
                        f[(j * 4 + k) % 8] = fmaf(a, scale, zero);
                    }
                }
            }
            st_stream16(dst + c * D + pc * X::kLanes * 8, make_uint4(pack2(f[0], f[1]), pack2(f[2], f[3]), pack2(f[4], f[5]), pack2(f[6], f[7])));
        }
    }
}

int32_t refuse(const char* why, int32_t code = UCMX_EPARAM)
{
    set_last_text(why);
    return code;
}

enum Form { kTokensForm, kBlocksForm, kReadForm };

constexpr char kTooMany[] = "quantised cache: more rows than one call takes";

template <int BITS, int D, int HC>
int32_t launch_heads(QuantParams& p, Form form, int64_t groups, int chunks, cudaStream_t st)
{
    p.heads_per = ((p.H + chunks - 1) / chunks + HC - 1) / HC * HC;
    p.head_chunks = (uint32_t)((p.H + p.heads_per - 1) / p.heads_per);
    const int64_t items = groups * 2 * p.head_chunks;
    if (items > INT32_MAX) return refuse(kTooMany, UCMX_EUNSUPPORTED);
    p.items = (uint32_t)items;
    const unsigned grid = (unsigned)((items + 7) / 8);
    if (form == kTokensForm)
        quant_write_kernel<BITS, D, false, HC><<<grid, 256, 0, st>>>(p);
    else if (form == kBlocksForm)
        quant_write_kernel<BITS, D, true, HC><<<grid, 256, 0, st>>>(p);
    else
        quant_read_kernel<BITS, D, HC><<<grid, 256, 0, st>>>(p);
    UCMX_LAUNCH_CHECK("quant_cache_kernel");
    return UCMX_OK;
}

template <int BITS, int D>
int32_t launch(QuantParams& p, Form form, cudaStream_t st)
{
    using X = Q<BITS, D>;
    const int64_t groups = form == kTokensForm ? p.n / X::kTokens + (p.n % X::kTokens != 0) : p.n * (p.T / X::kTokens);
    if (groups > INT32_MAX) return refuse(kTooMany, UCMX_EUNSUPPORTED);  // (what follows is counted in 64 bits)
    // Two heads of a warp in flight as soon as that still gives every SM its 32 warps; with the few tokens of a decode step one head
    // each, over twice as many warps.  Writing, a warp goes on through its tokens' heads (finding its place costs as much as two thirds
    // of a head) as long as that leaves two rounds of warps; reading, which HBM bounds, it does not.
    const int64_t full = (int64_t)sm_count() * 32;
    const int pairs = (p.H + 1) / 2;
    if (groups * 2 * pairs < full) return launch_heads<BITS, D, 1>(p, form, groups, p.H, st);
    int64_t chunks = form == kReadForm ? pairs : (2 * full + groups * 2 - 1) / (groups * 2);
    if (chunks > pairs) chunks = pairs;
    return launch_heads<BITS, D, 2>(p, form, groups, (int)chunks, st);
}

int32_t dispatch(QuantParams& p, const ucmx_quant_geometry* g, Form form, cudaStream_t st)
{
    p.err = error_word();
    const int which = (g->bits == 4 ? 0 : 1) * 1000 + g->head_dim;
    switch (which) {
        case 64: return launch<4, 64>(p, form, st);
        case 128: return launch<4, 128>(p, form, st);
        case 256: return launch<4, 256>(p, form, st);
        case 1064: return launch<8, 64>(p, form, st);
        case 1128: return launch<8, 128>(p, form, st);
        default: return launch<8, 256>(p, form, st);
    }
}

int32_t check_cache(const void* cache, const ucmx_quant_geometry* g)
{
    const size_t bytes = ucmx_quant_block_bytes(g);
    if (bytes == 0) return refuse("quantised cache: a geometry that the library does not hold", UCMX_EUNSUPPORTED);
    if (!cache || ((uintptr_t)cache & 15)) return refuse("quantised cache: must start on 16 bytes");
    if (g->n_blocks < 1 || g->block_stride < (int64_t)bytes || g->block_stride % 16)
        return refuse("quantised cache: block_stride must be a multiple of 16 and hold a block");
    return UCMX_OK;
}

// the bf16 side of the block forms
int32_t check_pair(QuantParams& p, const void* k, const ucmx_kv_geometry* kg, const void* v, const ucmx_kv_geometry* vg,
                   const ucmx_quant_geometry* g)
{
    if (!k || !v || ((uintptr_t)k & 15) || ((uintptr_t)v & 15)) return refuse("quantised cache: bf16 caches must start on 16 bytes");
    if (!kg || !vg || kg->reserved < 1 || vg->reserved < 1) return refuse("quantised cache: the geometries must carry the number of blocks");
    const ucmx_kv_geometry* both[2] = {kg, vg};
    for (const ucmx_kv_geometry* x : both) {
        if (x->block_tokens != g->block_tokens || x->n_kv_heads != g->n_kv_heads || x->head_dim != g->head_dim)
            return refuse("quantised cache: the bf16 blocks have another shape");
        if (x->token_stride < (int64_t)x->n_kv_heads * x->head_dim || x->token_stride % 8 || x->block_stride % 8 || x->block_stride < 0)
            return refuse("quantised cache: strides must be multiples of 8 elements and hold a token's heads");
    }
    p.k = (const uint16_t*)k;
    p.v = (const uint16_t*)v;
    p.k_block = kg->block_stride;
    p.v_block = vg->block_stride;
    p.k_token = kg->token_stride;
    p.v_token = vg->token_stride;
    p.n_src = kg->reserved < vg->reserved ? kg->reserved : vg->reserved;
    return UCMX_OK;
}

void set_cache(QuantParams& p, const void* cache, const ucmx_quant_geometry* g)
{
    p.cache = (uint8_t*)const_cast<void*>(cache);
    p.block_stride = g->block_stride;
    p.n_blocks = g->n_blocks;
    p.T = g->block_tokens;
    p.H = g->n_kv_heads;
}

}  // namespace
}  // namespace ucmx

using namespace ucmx;

extern "C" size_t ucmx_quant_block_bytes(const ucmx_quant_geometry* g)
{
    if (!g || (g->bits != 4 && g->bits != 8) || (g->head_dim != 64 && g->head_dim != 128 && g->head_dim != 256)) return 0;
    if (g->block_tokens < 16 || g->block_tokens % 16 || g->n_kv_heads < 1 || g->block_tokens > (1 << 20) || g->n_kv_heads > (1 << 16)) return 0;
    const size_t group = (size_t)(2 * 16) * (g->head_dim * g->bits / 8) + 2 * 16 * 4;
    return group * (size_t)(g->block_tokens / 16) * (size_t)g->n_kv_heads;
}

extern "C" int32_t ucmx_quant_write_tokens(const void* k, const void* v, int64_t k_stride, int64_t v_stride, int64_t n, const int64_t* slots,
                                           void* cache, const ucmx_quant_geometry* g, ucmx_stream_t stream)
{
    if (n < 0) return refuse("quant_write_tokens: a negative count");
    if (n == 0) return UCMX_OK;
    const int32_t rc = check_cache(cache, g);
    if (rc != UCMX_OK) return rc;
    if (!k || !v || !slots || ((uintptr_t)k & 15) || ((uintptr_t)v & 15)) return refuse("quant_write_tokens: rows must start on 16 bytes");
    const int64_t E = (int64_t)g->n_kv_heads * g->head_dim;
    if (k_stride < E || v_stride < E || k_stride % 8 || v_stride % 8)
        return refuse("quant_write_tokens: strides must be multiples of 8 elements and hold a token's heads");
    QuantParams p = {};
    p.k = (const uint16_t*)k;
    p.v = (const uint16_t*)v;
    p.k_token = k_stride;
    p.v_token = v_stride;
    p.slots = slots;
    p.n = n;
    set_cache(p, cache, g);
    return dispatch(p, g, kTokensForm, (cudaStream_t)stream);
}

extern "C" int32_t ucmx_quant_write_blocks(const void* k_cache, const ucmx_kv_geometry* kg, const void* v_cache, const ucmx_kv_geometry* vg,
                                           const int32_t* block_ids, const int32_t* out_slots, int32_t n, void* cache,
                                           const ucmx_quant_geometry* g, ucmx_stream_t stream)
{
    if (n < 0) return refuse("quant_write_blocks: a negative count");
    if (n == 0) return UCMX_OK;
    int32_t rc = check_cache(cache, g);
    QuantParams p = {};
    if (rc == UCMX_OK) rc = check_pair(p, k_cache, kg, v_cache, vg, g);
    if (rc != UCMX_OK) return rc;
    if (!block_ids) return refuse("quant_write_blocks: no block ids");
    p.ids = block_ids;
    p.out_slots = out_slots;
    p.n = n;
    set_cache(p, cache, g);
    return dispatch(p, g, kBlocksForm, (cudaStream_t)stream);
}

extern "C" int32_t ucmx_quant_read_blocks(const void* cache, const ucmx_quant_geometry* g, const int32_t* block_ids, const int32_t* out_slots,
                                          int32_t n, void* k_cache, const ucmx_kv_geometry* kg, void* v_cache, const ucmx_kv_geometry* vg,
                                          ucmx_stream_t stream)
{
    if (n < 0) return refuse("quant_read_blocks: a negative count");
    if (n == 0) return UCMX_OK;
    int32_t rc = check_cache(cache, g);
    QuantParams p = {};
    if (rc == UCMX_OK) rc = check_pair(p, k_cache, kg, v_cache, vg, g);
    if (rc != UCMX_OK) return rc;
    if ((kg->block_stride == 0 && kg->reserved > 1) || (vg->block_stride == 0 && vg->reserved > 1))
        return refuse("quant_read_blocks: all blocks of the output lie in one place");
    if (!block_ids) return refuse("quant_read_blocks: no block ids");
    p.ids = block_ids;
    p.out_slots = out_slots;
    p.n = n;
    set_cache(p, cache, g);
    return dispatch(p, g, kReadForm, (cudaStream_t)stream);
}
