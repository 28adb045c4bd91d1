// Attention over the quantised cache: entry points.
#include <algorithm>
#include <memory>
#include <new>
#include <type_traits>

#include "vx_kv_attention.cuh"

struct vx_kv_attention {
    const vx_context* ctx = nullptr;
    const vx_kv_cache* cache = nullptr;
    size_t heads = 0, max_seqs = 0;
    uint32_t grid[3] = {};  // thread blocks by groups of eight rows (1, 2), 0: four rows
    uint8_t* workspace = nullptr;
    size_t ml_offset = 0, counters_offset = 0;
};

namespace vx {

extern template vx_status kv_attention_setup<false, false>(uint32_t, uint32_t, int*, uint32_t*);
extern template vx_status kv_attention_setup<false, true>(uint32_t, uint32_t, int*, uint32_t*);
extern template vx_status kv_attention_setup<true, false>(uint32_t, uint32_t, int*, uint32_t*);
extern template vx_status kv_attention_setup<true, true>(uint32_t, uint32_t, int*, uint32_t*);
extern template vx_status kv_attention_launch<false, false>(uint32_t, uint32_t, uint32_t, cudaStream_t, const AttnParams&);
extern template vx_status kv_attention_launch<false, true>(uint32_t, uint32_t, uint32_t, cudaStream_t, const AttnParams&);
extern template vx_status kv_attention_launch<true, false>(uint32_t, uint32_t, uint32_t, cudaStream_t, const AttnParams&);
extern template vx_status kv_attention_launch<true, true>(uint32_t, uint32_t, uint32_t, cudaStream_t, const AttnParams&);

}  // namespace vx

namespace {

using namespace vx;

bool attn_dim(size_t d) { return d == 64 || d == 96 || d == 128 || d == 256; }
vx_status setup(const vx_kv_cache* c, uint32_t nt, int* per_sm, uint32_t* smem) {
    const bool k4 = c->g.k4, v4 = c->g.v4;
    if (k4) return v4 ? kv_attention_setup<true, true>(c->g.blocks, nt, per_sm, smem) : kv_attention_setup<true, false>(c->g.blocks, nt, per_sm, smem);
    return v4 ? kv_attention_setup<false, true>(c->g.blocks, nt, per_sm, smem) : kv_attention_setup<false, false>(c->g.blocks, nt, per_sm, smem);
}

vx_status launch(const vx_kv_cache* c, uint32_t nt, uint32_t grid, cudaStream_t s, const AttnParams& p) {
    const bool k4 = c->g.k4, v4 = c->g.v4;
    if (k4) return v4 ? kv_attention_launch<true, true>(c->g.blocks, nt, grid, s, p) : kv_attention_launch<true, false>(c->g.blocks, nt, grid, s, p);
    return v4 ? kv_attention_launch<false, true>(c->g.blocks, nt, grid, s, p) : kv_attention_launch<false, false>(c->g.blocks, nt, grid, s, p);
}

}  // namespace

extern "C" {

vx_status vx_kv_attention_create(vx_context* ctx, const vx_kv_cache* cache, size_t heads, size_t max_seqs, vx_kv_attention** out) {
    VX_REQUIRE(ctx && cache && out, VX_ERR_INVALID_ARGUMENT, "vx_kv_attention_create: null argument");
    *out = nullptr;
    VX_REQUIRE(ctx->device == cache->device, VX_ERR_INVALID_ARGUMENT, "vx_kv_attention_create: the cache is on device %d, the context on %d",
               cache->device, ctx->device);
    VX_REQUIRE(heads > 0 && heads % cache->g.heads == 0, VX_ERR_SHAPE, "vx_kv_attention_create: %zu query heads over %u heads of keys", heads,
               cache->g.heads);
    VX_REQUIRE(max_seqs > 0, VX_ERR_INVALID_ARGUMENT, "vx_kv_attention_create: max_seqs is 0");
    VX_REQUIRE(attn_dim(cache->head_dim), VX_ERR_UNSUPPORTED, "vx_kv_attention_create: heads of %zu values (64, 96, 128 and 256 are supported)",
               cache->head_dim);
    VX_REQUIRE(heads <= 65535 && max_seqs <= 0x0fffffffull, VX_ERR_UNSUPPORTED, "vx_kv_attention_create: too many heads or sequences");
    DeviceGuard guard(ctx->device);
    std::unique_ptr<vx_kv_attention> a(new (std::nothrow) vx_kv_attention());
    VX_REQUIRE(a, VX_ERR_OUT_OF_MEMORY, "host allocation failed");
    a->ctx = ctx;
    a->cache = cache;
    a->heads = heads;
    a->max_seqs = max_seqs;
    size_t rows = 0, blocks = 0;
    for (uint32_t nt = 0; nt <= 2; ++nt) {
        int per_sm = 0;
        uint32_t smem = 0;
        const vx_status st = setup(cache, nt, &per_sm, &smem);
        if (st != VX_OK) return st;
        VX_REQUIRE(per_sm > 0, VX_ERR_UNSUPPORTED, "vx_kv_attention_create: the kernel does not fit an SM");
        a->grid[nt] = (uint32_t)(ctx->sm_count * per_sm);
        rows = std::max(rows, (size_t)2 * a->grid[nt] * (nt == 0 ? 4 : 8 * nt));
        blocks = std::max(blocks, (size_t)a->grid[nt]);
    }
    a->ml_offset = rows * cache->head_dim * sizeof(float);
    a->counters_offset = a->ml_offset + rows * sizeof(float2);
    const size_t bytes = a->counters_offset + blocks * sizeof(uint32_t);
    cudaError_t e = device_malloc(ctx, reinterpret_cast<void**>(&a->workspace), bytes);
    if (e != cudaSuccess) {
        (void)cudaGetLastError();
        return fail(VX_ERR_OUT_OF_MEMORY, "allocating %zu bytes of attention workspace failed: %s", bytes, cudaGetErrorString(e));
    }
    e = cudaMemsetAsync(a->workspace + a->counters_offset, 0, blocks * sizeof(uint32_t), ctx->stream);
    if (e == cudaSuccess) e = cudaStreamSynchronize(ctx->stream);  // an error while the stream is being captured
    if (e != cudaSuccess) {
        (void)cudaGetLastError();
        cudaFree(a->workspace);
        return fail(VX_ERR_CUDA, "clearing the attention counters failed: %s", cudaGetErrorString(e));
    }
    *out = a.release();
    return VX_OK;
}

vx_status vx_kv_attention_free(vx_context* ctx, vx_kv_attention* a) {
    VX_REQUIRE(ctx, VX_ERR_INVALID_ARGUMENT, "vx_kv_attention_free: null context");
    if (!a) return VX_OK;
    VX_REQUIRE(ctx == a->ctx, VX_ERR_INVALID_ARGUMENT, "vx_kv_attention_free: made with another context");
    DeviceGuard guard(ctx->device);
    VX_CUDA(cudaStreamSynchronize(ctx->stream));
    VX_CUDA(cudaFree(a->workspace));
    delete a;
    return VX_OK;
}

vx_status vx_kv_attention_run(vx_context* ctx, const vx_kv_attention* a, const vx_kv_rows* rows, const float* q, size_t q_stride, float* out,
                              size_t out_stride, float scale, const uint32_t* mask, size_t mask_words) {
    VX_REQUIRE(ctx && a, VX_ERR_INVALID_ARGUMENT, "vx_kv_attention_run: null argument");
    VX_REQUIRE(ctx == a->ctx, VX_ERR_INVALID_ARGUMENT, "vx_kv_attention_run: the workspace was made with another context");
    AttnParams p{};
    const vx_status st = kv_rows_check("vx_kv_attention_run", rows, &p.r);
    if (st != VX_OK || p.r.rows == 0) return st;
    VX_REQUIRE(rows->seqs <= a->max_seqs, VX_ERR_INVALID_ARGUMENT, "vx_kv_attention_run: %zu sequences, made for %zu", rows->seqs, a->max_seqs);
    VX_REQUIRE(q && out, VX_ERR_INVALID_ARGUMENT, "vx_kv_attention_run: null q or out");
    const size_t width = a->heads * a->cache->head_dim;
    VX_REQUIRE(p.r.rows == 1 || (q_stride >= width && out_stride >= width), VX_ERR_INVALID_ARGUMENT,
               "vx_kv_attention_run: rows %zu and %zu elements apart, a row has %zu", q_stride, out_stride, width);
    // In place, every block has read its rows of q before any of its heads' results is written.
    VX_REQUIRE(q != out || p.r.rows == 1 || q_stride == out_stride, VX_ERR_INVALID_ARGUMENT,
               "vx_kv_attention_run: out is q with rows %zu instead of %zu elements apart", out_stride, q_stride);
    VX_REQUIRE(!mask || (mask_words > 0 && mask_words <= 0x7ffffffull), VX_ERR_INVALID_ARGUMENT, "vx_kv_attention_run: a mask of %zu words a row", mask_words);
    const uint32_t group = (uint32_t)(a->heads / a->cache->g.heads);
    VX_REQUIRE((uint64_t)p.r.rows * group <= 0x7fffffffull, VX_ERR_UNSUPPORTED, "vx_kv_attention_run: too many rows (%u)", p.r.rows);
    p.g = a->cache->g;
    p.q = q;
    p.out = out;
    p.q_stride = q_stride;
    p.out_stride = out_stride;
    p.group = group;
    p.scale_log2 = scale * 1.4426950408889634f;
    p.mask = mask;
    p.mask_words = (uint32_t)mask_words;
    p.part_o = reinterpret_cast<float*>(a->workspace);
    p.part_ml = reinterpret_cast<float2*>(a->workspace + a->ml_offset);
    p.counters = reinterpret_cast<uint32_t*>(a->workspace + a->counters_offset);
    // Rows of a sequence that share a head of keys, as the host can know them (the average), in groups of 4, 8 or 16.  Four
    // rows' two parts fill the eight columns of a product (9.3 us with, 10.7 without for one token of 4 heads to a head of
    // keys over 500; 73 and 80 us for 16 sequences of up to 16384).  Two groups of 8 in one block share the conversion of the
    // codes (30 us for 4 x 8 drafted tokens of 32 heads over 4000, 149 for 2 x 48 over 12000; one group at a time 34 and
    // 183); 32 rows spilled registers (35).
    const uint64_t each = ((uint64_t)p.r.rows + p.r.seqs - 1) / p.r.seqs * group;
    const uint32_t nt = each <= 4 ? 0 : each <= 8 ? 1 : 2;
    DeviceGuard guard(ctx->device);
    const vx_status ls = launch(a->cache, nt, a->grid[nt], ctx->stream, p);
    if (ls != VX_OK) return ls;
    ctx->launches++;
    return VX_OK;
}

}  // extern "C"
