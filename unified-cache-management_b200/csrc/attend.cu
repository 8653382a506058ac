// Attention over listed blocks: the C entries, their checks, and the bf16 cache's instances (kernel: attend.cuh).
#include <mutex>

#include "attend.cuh"

namespace ucmx {
namespace attend {

int32_t run_bf16(const Params& p, int head_dim, int cols, const Maps* maps, Plan* plan, cudaStream_t st)
{
    return run_format<16>(p, head_dim, cols, maps, plan, st);
}

namespace {

int32_t refuse(const char* why, int32_t code = UCMX_EPARAM)
{
    set_last_text(why);
    return code;
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn()
{
    static std::mutex mu;
    static EncodeTiledFn fn = nullptr;
    std::lock_guard<std::mutex> lk(mu);
    if (!fn) {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q = cudaDriverEntryPointSymbolNotFound;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = (EncodeTiledFn)p;
    }
    return fn;
}

// one side of the bf16 cache as a tensor [block][token][head][value], loaded 64 values x `box` tokens at a time
bool make_map(CUtensorMap* map, const uint8_t* base, const Params& p, int head_dim, int64_t token_bytes, int64_t block_bytes)
{
    EncodeTiledFn enc = encode_fn();
    if (!enc) return false;
    const cuuint64_t dims[4] = {(cuuint64_t)head_dim, (cuuint64_t)p.H, (cuuint64_t)p.T, (cuuint64_t)p.n_blocks};
    const cuuint64_t strides[3] = {(cuuint64_t)head_dim * 2, (cuuint64_t)token_bytes,
                                   (cuuint64_t)(block_bytes > 0 ? block_bytes : token_bytes)};   // (one block: any stride will do)
    const cuuint32_t box[4] = {64, 1, (cuuint32_t)p.box, 1}, one[4] = {1, 1, 1, 1};
    return enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<uint8_t*>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int32_t run_any(int bits, const Params& p, int head_dim, int cols, const Maps* maps, Plan* plan, cudaStream_t st)
{
    return bits == 16 ? run_bf16(p, head_dim, cols, maps, plan, st)
         : bits == 8  ? run_q8(p, head_dim, cols, maps, plan, st)
                      : run_q4(p, head_dim, cols, maps, plan, st);
}

size_t plan_bytes(const Plan& plan) { return (size_t)plan.ctas * (2 * plan.part * sizeof(float) + sizeof(Rec)); }

// what both entries check and fill in; the cache's part of `p` is set by the caller
int32_t attend_common(Params& p, int bits, int32_t head_dim, const void* q, int64_t q_stride, int32_t n_q_heads, int32_t n_kv_heads,
                      const int32_t* q_offsets, int32_t n_q_tokens, int32_t max_q_tokens, const ucmx_block_lists* l, float scale,
                      void* out, float* out_lse, void* workspace, size_t workspace_bytes, ucmx_stream_t stream)
{
    if (!l || l->n_req < 0 || l->total < 0 || l->table_size < 0 || n_q_tokens < 0) return refuse("attention: negative sizes or no lists");
    if (l->n_req == 0 || n_q_tokens == 0) return UCMX_OK;
    if (!q || !out || !l->offsets || !workspace) return refuse("attention: a pointer is missing");
    if (l->total > 0 && !l->block_ids && !(l->positions && l->table && l->table_offsets))
        return refuse("attention: block_ids, or positions with table and table_offsets");
    if (n_kv_heads < 1 || n_q_heads < n_kv_heads || n_q_heads % n_kv_heads) return refuse("attention: n_q_heads must be a multiple of n_kv_heads");
    if (max_q_tokens < 1 || (!q_offsets && max_q_tokens != 1)) return refuse("attention: more than one query token per request needs q_offsets");
    if (max_q_tokens > 1 && !l->ctx_lens) return refuse("attention: several query tokens per request need ctx_lens");
    if (q_stride % 8 || q_stride < (int64_t)n_q_heads * head_dim || ((uintptr_t)q & 15) || ((uintptr_t)out & 15) || ((uintptr_t)workspace & 15))
        return refuse("attention: query rows, out and workspace must start on 16 bytes");
    if (p.k_block % 16 || ((uintptr_t)p.k & 15) || ((uintptr_t)p.v & 15)) return refuse("attention: the cache must start on 16 bytes");
    if ((int64_t)max_q_tokens * (n_q_heads / n_kv_heads) > (1 << 20)) return refuse("attention: too many query rows per request", UCMX_EUNSUPPORTED);
    p.q = (const uint16_t*)q;
    p.q_stride = q_stride;
    p.q_offsets = q_offsets;
    p.n_q_tokens = n_q_tokens;
    p.max_q = max_q_tokens;
    p.Hq = n_q_heads;
    p.H = n_kv_heads;
    p.G = n_q_heads / n_kv_heads;
    p.spe = (p.T + kRows - 1) / kRows;
    p.offsets = l->offsets;
    p.counts = l->counts;
    p.block_ids = l->block_ids;
    p.positions = l->positions;
    p.table = l->table;
    p.table_offsets = l->table_offsets;
    p.table_size = l->table_size;
    p.ctx = l->ctx_lens;
    p.n_req = l->n_req;
    p.total = l->total;
    p.scale_log2 = scale * kLog2e;
    p.out = (uint16_t*)out;
    p.lse = out_lse;
    p.ws = (float*)workspace;
    p.err = error_word();
    const int cols = max_q_tokens * p.G;
    Plan plan;
    const int32_t rc = run_any(bits, p, head_dim, cols, nullptr, &plan, nullptr);
    if (rc != UCMX_OK) return refuse("attention: head_dim must be 64, 128 or 256", rc);
    if (workspace_bytes < plan_bytes(plan)) return refuse("attention: workspace too small");
    p.col_tiles = (cols + plan.cols - 1) / plan.cols;
    // the slices of all requests, heads and tiles, and a lead for each of them, are numbered in 32 bits
    const int64_t units = (int64_t)p.total * p.spe + (int64_t)p.n_req * kLeadMost;
    if (too_many_units(units, p.H, p.col_tiles))
        return refuse("attention: more than 2^31 pieces of 16 tokens in the lists of all heads", UCMX_EUNSUPPORTED);
    Maps maps = {};
    if (bits == 16 && p.total > 0) {
        p.box = p.T < kRows ? p.T : kRows;
        if (!make_map(&maps.k, p.k, p, head_dim, p.k_token, p.k_block) || !make_map(&maps.v, p.v, p, head_dim, p.v_token, p.v_block))
            return refuse("attention: no tensor map for a cache with these strides", UCMX_EUNSUPPORTED);
    }
    return run_any(bits, p, head_dim, cols, &maps, &plan, (cudaStream_t)stream);
}

}  // namespace
}  // namespace attend
}  // namespace ucmx

using namespace ucmx;
using namespace ucmx::attend;

extern "C" size_t ucmx_attention_workspace_bytes(int32_t bits, int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim, int32_t max_q_tokens)
{
    if ((bits != 16 && bits != 8 && bits != 4) || n_kv_heads < 1 || n_q_heads < n_kv_heads || max_q_tokens < 1) return 0;
    Plan plan;
    Params p = {};
    const int64_t cols = (int64_t)max_q_tokens * (n_q_heads / n_kv_heads);
    if (run_any(bits, p, head_dim, cols > 64 ? 64 : (int)cols, nullptr, &plan, nullptr) != UCMX_OK) return 0;
    return plan_bytes(plan);
}

extern "C" int32_t ucmx_block_attention(const void* q, int64_t q_stride, int32_t n_q_heads, const int32_t* q_offsets, int32_t n_q_tokens,
                                        int32_t max_q_tokens, const void* k_cache, const ucmx_kv_geometry* kg, const void* v_cache,
                                        const ucmx_kv_geometry* vg, const ucmx_block_lists* lists, float scale, void* out, float* out_lse,
                                        void* workspace, size_t workspace_bytes, ucmx_stream_t stream)
{
    if (!kg || !vg || !lists) return refuse("block_attention: geometry or lists missing");
    if (kg->block_tokens < 1 || kg->n_kv_heads < 1 || kg->reserved < 1) return refuse("block_attention: the geometry must carry tokens, heads and blocks");
    if (vg->block_tokens != kg->block_tokens || vg->n_kv_heads != kg->n_kv_heads || vg->head_dim != kg->head_dim)
        return refuse("block_attention: K and V blocks differ in shape");
    const int64_t E = (int64_t)kg->n_kv_heads * kg->head_dim;
    if (kg->token_stride < E || vg->token_stride < E || kg->token_stride % 8 || vg->token_stride % 8 || kg->block_stride % 8 || vg->block_stride % 8 ||
        kg->block_stride < 0 || vg->block_stride < 0)
        return refuse("block_attention: strides must be multiples of 8 elements and hold a token's heads");
    if ((kg->block_stride == 0 && kg->reserved > 1) || (vg->block_stride == 0 && vg->reserved > 1))
        return refuse("block_attention: all blocks of the cache lie in one place");
    if (lists->n_req > 0 && lists->total > 0 && n_q_tokens > 0 && (!k_cache || !v_cache)) return refuse("block_attention: no cache");
    Params p = {};
    p.k = (const uint8_t*)k_cache;
    p.v = (const uint8_t*)v_cache;
    p.k_block = kg->block_stride * 2;
    p.v_block = vg->block_stride * 2;
    p.k_token = kg->token_stride * 2;
    p.v_token = vg->token_stride * 2;
    p.T = kg->block_tokens;
    p.n_blocks = kg->reserved < vg->reserved ? kg->reserved : vg->reserved;
    return attend_common(p, 16, kg->head_dim, q, q_stride, n_q_heads, kg->n_kv_heads, q_offsets, n_q_tokens, max_q_tokens, lists, scale, out,
                         out_lse, workspace, workspace_bytes, stream);
}

extern "C" int32_t ucmx_quant_block_attention(const void* q, int64_t q_stride, int32_t n_q_heads, const int32_t* q_offsets, int32_t n_q_tokens,
                                              int32_t max_q_tokens, const void* cache, const ucmx_quant_geometry* g,
                                              const ucmx_block_lists* lists, float scale, void* out, float* out_lse, void* workspace,
                                              size_t workspace_bytes, ucmx_stream_t stream)
{
    if (!lists) return refuse("quant_block_attention: no lists");
    if (ucmx_quant_block_bytes(g) == 0) return refuse("quant_block_attention: a cache geometry that the library does not hold", UCMX_EUNSUPPORTED);
    if (g->n_blocks < 1 || g->block_stride < (int64_t)ucmx_quant_block_bytes(g) || g->block_stride % 16)
        return refuse("quant_block_attention: block_stride must be a multiple of 16 and hold a block");
    if (lists->n_req > 0 && lists->total > 0 && n_q_tokens > 0 && !cache) return refuse("quant_block_attention: no cache");
    Params p = {};
    p.k = (const uint8_t*)cache;
    p.k_block = g->block_stride;
    p.T = g->block_tokens;
    p.n_blocks = g->n_blocks;
    return attend_common(p, g->bits, g->head_dim, q, q_stride, n_q_heads, g->n_kv_heads, q_offsets, n_q_tokens, max_q_tokens, lists, scale, out,
                         out_lse, workspace, workspace_bytes, stream);
}
