// The quantised cache of keys and values: storage, quantising on write, reading back.
//
// Formats and arithmetic are those of vx_quantize (IEEE division, scale rounded to f16 before the codes are formed,
// half away from zero); vortx has no counterpart.  One block of threads takes one 32-token tile of one head, keys or
// values: eight lanes share a block of 32 values (a float4 each, the largest magnitude by three shuffles), so rows are
// read and written as whole 128-byte lines.  A tile that the call covers completely is put together in shared memory
// and goes out (comes in) as 16-byte vectors; the others' codes are stored where they belong one word at a time.
// Both are bound by the f32 side of the copy: 4 bytes a value next to 1.06 (Q8_0) or 0.56 (Q4_0).
#include <cfloat>
#include <memory>
#include <new>

#include "vx_decode.cuh"

namespace {

using namespace vx;

constexpr uint32_t kMaxBlocks = 16;  // head_dim <= 512
constexpr uint32_t kThreads = 256;

// Which tile of which sequence a thread block has.  Sequence s owns the numbers from row0 / 32 + 2 s on: n rows lie
// in at most n / 32 + 2 tiles whatever their alignment, and floor(a / 32) + floor(n / 32) <= floor((a + n) / 32).
struct TileOf {
    uint32_t seq, tile, t0, t1;  // tokens t0 .. t1 - 1 of the tile are the call's
    KvSeq q;
};
__device__ __forceinline__ TileOf tile_of(const KvRows& r, const KvGeometry& g, uint32_t x) {
    TileOf o;
    o.seq = warp_search(r.seqs, x, [&](uint32_t s) { return (uint32_t)min(max(r.begin[s], 0), (int32_t)r.rows) / 32 + 2 * s; });
    o.q = kv_seq(r, g, o.seq);
    const uint32_t base = o.q.row0 / 32 + 2 * o.seq;
    o.tile = o.q.first / 32 + (x - base);
    const uint64_t lo = (uint64_t)o.tile * 32, end = (uint64_t)o.q.first + o.q.n;
    o.t0 = o.q.first > lo ? o.q.first - (uint32_t)lo : 0;
    o.t1 = x < base || end <= lo ? 0 : (uint32_t)(end - lo < 32 ? end - lo : 32);
    return o;
}

__device__ __forceinline__ uint32_t code_bits(float v, float d, bool four) {
    float q = d != 0.0f ? roundf(__fdiv_rn(v, d)) : 0.0f;  // roundf: half away from zero
    if (four) return (uint32_t)(int)fminf(15.0f, fmaxf(0.0f, q + 8.0f));
    return (uint32_t)((int)fminf(127.0f, fmaxf(-127.0f, q)) + 128);
}

template <bool FOUR, bool VALUES>
__device__ void append_part(const KvRows& r, const KvGeometry& g, const TileOf& o, uint8_t* dst, const float* __restrict__ src,
                            size_t stride, uint32_t head, bool vec, uint8_t* image) {
    const uint32_t oct = threadIdx.x / 8, j = threadIdx.x % 8, nb = g.blocks;
    const bool whole = o.t0 == 0 && o.t1 == 32;
    uint8_t* to = whole ? image : dst;
    const uint32_t scales = kv_code_bytes(FOUR, nb);
    // the eight lanes of a block take part or stay out together
    for (uint32_t p0 = o.t0 * nb; p0 < o.t1 * nb; p0 += kThreads / 8) {
        const uint32_t p = p0 + oct;
        const bool live = p < o.t1 * nb;
        const uint32_t mask = __ballot_sync(0xffffffffu, live);
        if (!live) continue;
        const uint32_t token = p / nb, block = p - token * nb;
        const uint32_t row = o.q.row0 + (o.tile * 32 + token - o.q.first);
        const float* from = src + (size_t)row * stride + (size_t)head * nb * 32 + block * 32 + j * 4;
        float v[4];
        if (vec) {
            const float4 f = __ldcs(reinterpret_cast<const float4*>(from));
            v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
        } else {
#pragma unroll
            for (int n = 0; n < 4; ++n) v[n] = __ldcs(from + n);
        }
        // the element of largest magnitude, the first one on ties
        float amax = 0.0f, signed_max = 0.0f;
        bool bad = false;
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            const float a = fabsf(v[n]);
            bad |= !(a <= FLT_MAX);
            if (a > amax) {
                amax = a;
                signed_max = v[n];
            }
        }
        uint32_t at = j;
#pragma unroll
        for (int s = 1; s < 8; s *= 2) {
            const float a = __shfl_xor_sync(mask, amax, s), m = __shfl_xor_sync(mask, signed_max, s);
            const uint32_t i = __shfl_xor_sync(mask, at, s);
            bad |= (bool)__shfl_xor_sync(mask, (int)bad, s);
            if (a > amax || (a == amax && i < at)) {
                amax = a;
                signed_max = m;
                at = i;
            }
        }
        uint16_t dh = __half_as_ushort(__float2half_rn(FOUR ? __fdiv_rn(signed_max, 7.0f) : __fdiv_rn(amax, 127.0f)));
        if (bad || (dh & 0x7fffu) >= 0x7c00u) dh = 0x7fffu;
        const bool nan = dh == 0x7fffu;
        const float d = nan ? 0.0f : __half2float(__ushort_as_half(dh));
        uint32_t c[4];
#pragma unroll
        for (int n = 0; n < 4; ++n) c[n] = code_bits(nan ? 0.0f : v[n], d, FOUR);
        if (VALUES) {
            if (FOUR)
                *reinterpret_cast<uint16_t*>(to + v_word(true, block, token, j)) = (uint16_t)(c[0] | c[1] << 4 | c[2] << 8 | c[3] << 12);
            else
#pragma unroll
                for (int n = 0; n < 4; ++n) to[v_word(false, block, token, j) + 4 * n] = (uint8_t)c[n];
        } else {
            uint32_t w = c[0] | c[1] << 8 | c[2] << 16 | c[3] << 24;
            if (FOUR) w |= __shfl_xor_sync(mask, w, 4) << 4;  // byte i of a Q4_0 block: values i and i + 16
            if (!FOUR || j < 4) *reinterpret_cast<uint32_t*>(to + k_word(FOUR, block, token, j)) = w;
        }
        if (j == 0) *reinterpret_cast<uint16_t*>(to + scales + (VALUES ? v_scale(block, token) : k_scale(block, token))) = dh;
    }
    if (!whole) return;
    __syncthreads();
    const uint4* im = reinterpret_cast<const uint4*>(image);
    for (uint32_t i = threadIdx.x; i < kv_part_bytes(FOUR, nb) / 16; i += kThreads) reinterpret_cast<uint4*>(dst)[i] = im[i];
}

__global__ void __launch_bounds__(kThreads)
kv_append_kernel(KvRows r, KvGeometry g, const float* __restrict__ k, size_t k_stride, const float* __restrict__ v, size_t v_stride,
                 int k_vec, int v_vec) {
    __shared__ __align__(16) uint8_t image[kv_part_bytes(false, kMaxBlocks)];
    const uint32_t head = blockIdx.y;
    const TileOf o = tile_of(r, g, blockIdx.x);
    if (o.t0 >= o.t1) return;
    uint8_t* rec = kv_record(r, g, o.seq, o.tile, head);
    if (!rec) return;
    if (blockIdx.z == 0) {
        if (g.k4) append_part<true, false>(r, g, o, rec, k, k_stride, head, k_vec != 0, image);
        else append_part<false, false>(r, g, o, rec, k, k_stride, head, k_vec != 0, image);
    } else {
        if (g.v4) append_part<true, true>(r, g, o, rec + g.k_bytes, v, v_stride, head, v_vec != 0, image);
        else append_part<false, true>(r, g, o, rec + g.k_bytes, v, v_stride, head, v_vec != 0, image);
    }
}

template <bool FOUR, bool VALUES>
__device__ void read_part(const KvGeometry& g, const TileOf& o, const uint8_t* src, float* __restrict__ dst, size_t stride,
                          uint32_t head, bool vec, uint8_t* image) {
    const uint32_t oct = threadIdx.x / 8, j = threadIdx.x % 8, nb = g.blocks;
    const uint32_t scales = kv_code_bytes(FOUR, nb);
    if (src && o.t1 - o.t0 >= 8) {  // most of the tile is wanted: bring it in as vectors
        for (uint32_t i = threadIdx.x; i < kv_part_bytes(FOUR, nb) / 16; i += kThreads)
            reinterpret_cast<uint4*>(image)[i] = reinterpret_cast<const uint4*>(src)[i];
        __syncthreads();
        src = image;
    }
    for (uint32_t p = o.t0 * nb + oct; p < o.t1 * nb; p += kThreads / 8) {
        const uint32_t token = p / nb, block = p - token * nb;
        const uint32_t row = o.q.row0 + (o.tile * 32 + token - o.q.first);
        float f[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (src) {
            const uint16_t dh = *reinterpret_cast<const uint16_t*>(src + scales + (VALUES ? v_scale(block, token) : k_scale(block, token)));
            const float d = __half2float(__ushort_as_half(dh));
            uint32_t w;
            if (VALUES && FOUR) {
                w = *reinterpret_cast<const uint16_t*>(src + v_word(true, block, token, j));
            } else if (VALUES) {
                const uint8_t* at = src + v_word(false, block, token, j);
                w = at[0] | (uint32_t)at[4] << 8 | (uint32_t)at[8] << 16 | (uint32_t)at[12] << 24;
            } else {
                w = *reinterpret_cast<const uint32_t*>(src + k_word(FOUR, block, token, FOUR ? j % 4 : j));
            }
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                int q;
                if (!FOUR) q = (int)((w >> (8 * n)) & 255u) - 128;
                else if (VALUES) q = (int)((w >> (4 * n)) & 15u) - 8;
                else q = (int)((w >> (8 * n + (j < 4 ? 0 : 4))) & 15u) - 8;
                f[n] = __fmul_rn(d, (float)q);
            }
        }
        float* to = dst + (size_t)row * stride + (size_t)head * nb * 32 + block * 32 + j * 4;
        if (vec) {
            __stcs(reinterpret_cast<float4*>(to), make_float4(f[0], f[1], f[2], f[3]));
        } else {
#pragma unroll
            for (int n = 0; n < 4; ++n) __stcs(to + n, f[n]);
        }
    }
}

__global__ void __launch_bounds__(kThreads)
kv_read_kernel(KvRows r, KvGeometry g, float* __restrict__ k, size_t k_stride, float* __restrict__ v, size_t v_stride, int k_vec, int v_vec) {
    __shared__ __align__(16) uint8_t image[kv_part_bytes(false, kMaxBlocks)];
    const uint32_t head = blockIdx.y;
    const bool values = k == nullptr || blockIdx.z == 1;
    const TileOf o = tile_of(r, g, blockIdx.x);
    if (o.t0 >= o.t1) return;
    const uint8_t* rec = kv_record(r, g, o.seq, o.tile, head);
    if (!values) {
        if (g.k4) read_part<true, false>(g, o, rec, k, k_stride, head, k_vec != 0, image);
        else read_part<false, false>(g, o, rec, k, k_stride, head, k_vec != 0, image);
    } else {
        if (rec) rec += g.k_bytes;
        if (g.v4) read_part<true, true>(g, o, rec, v, v_stride, head, v_vec != 0, image);
        else read_part<false, true>(g, o, rec, v, v_stride, head, v_vec != 0, image);
    }
}

int vec_ok(const void* p, size_t stride) { return ((reinterpret_cast<uintptr_t>(p) & 15u) == 0 && stride % 4 == 0) ? 1 : 0; }

dim3 tiles_grid(const KvRows& r, const KvGeometry& g, unsigned parts) { return dim3(r.rows / 32 + 2 * r.seqs, g.heads, parts); }

}  // namespace

namespace vx {

vx_status kv_rows_check(const char* who, const vx_kv_rows* rows, KvRows* out) {
    VX_REQUIRE(rows, VX_ERR_INVALID_ARGUMENT, "%s: null rows", who);
    *out = KvRows{};
    if (rows->rows == 0 || rows->seqs == 0) return VX_OK;
    VX_REQUIRE(rows->table && rows->begin && rows->start, VX_ERR_INVALID_ARGUMENT, "%s: null page table, begin or start", who);
    VX_REQUIRE(rows->max_pages > 0, VX_ERR_INVALID_ARGUMENT, "%s: a page table of no pages", who);
    VX_REQUIRE(rows->rows <= 0x3fffffffull && rows->seqs <= 0x0fffffffull && rows->max_pages <= 0x7fffffffull, VX_ERR_UNSUPPORTED,
               "%s: too many rows (%zu), sequences (%zu) or pages (%zu)", who, rows->rows, rows->seqs, rows->max_pages);
    out->table = rows->table;
    out->begin = rows->begin;
    out->start = rows->start;
    out->max_pages = (uint32_t)rows->max_pages;
    out->seqs = (uint32_t)rows->seqs;
    out->rows = (uint32_t)rows->rows;
    return VX_OK;
}

}  // namespace vx

extern "C" {

vx_status vx_kv_cache_create(vx_context* ctx, vx_qtype k_type, vx_qtype v_type, size_t heads, size_t head_dim, size_t pages,
                             size_t page_tokens, vx_kv_cache** out) {
    VX_REQUIRE(ctx && out, VX_ERR_INVALID_ARGUMENT, "vx_kv_cache_create: null argument");
    *out = nullptr;
    VX_REQUIRE((k_type == VX_Q8_0 || k_type == VX_Q4_0) && (v_type == VX_Q8_0 || v_type == VX_Q4_0), VX_ERR_INVALID_ARGUMENT,
               "vx_kv_cache_create: unknown quantised type (%d, %d)", (int)k_type, (int)v_type);
    VX_REQUIRE(heads > 0 && pages > 0 && head_dim > 0 && head_dim % 32 == 0, VX_ERR_INVALID_ARGUMENT,
               "vx_kv_cache_create: heads (%zu) and pages (%zu) must be positive and head_dim (%zu) a positive multiple of 32", heads,
               pages, head_dim);
    VX_REQUIRE(page_tokens > 0 && page_tokens % kTileTokens == 0, VX_ERR_INVALID_ARGUMENT,
               "vx_kv_cache_create: page_tokens (%zu) must be a positive multiple of 32", page_tokens);
    VX_REQUIRE(head_dim <= kMaxBlocks * 32 && heads <= 65535 && pages <= 0x7fffffffull && page_tokens <= 0x7fffffe0ull,
               VX_ERR_UNSUPPORTED, "vx_kv_cache_create: head_dim (%zu) above 512, or too many heads, pages or tokens per page", head_dim);
    const uint32_t nb = (uint32_t)(head_dim / 32);
    const bool k4 = k_type == VX_Q4_0, v4 = v_type == VX_Q4_0;
    const size_t record = kv_part_bytes(k4, nb) + kv_part_bytes(v4, nb);
    const size_t tiles = page_tokens / kTileTokens;
    VX_REQUIRE(pages <= ((size_t)1 << 50) / (tiles * heads * record), VX_ERR_OUT_OF_MEMORY, "vx_kv_cache_create: %zu pages are too many", pages);
    DeviceGuard guard(ctx->device);
    std::unique_ptr<vx_kv_cache> c(new (std::nothrow) vx_kv_cache());
    VX_REQUIRE(c, VX_ERR_OUT_OF_MEMORY, "host allocation failed");
    c->k_type = k_type;
    c->v_type = v_type;
    c->head_dim = head_dim;
    c->page_tokens = page_tokens;
    c->device_bytes = pages * tiles * heads * record;
    c->device = ctx->device;
    c->g.pages = (uint32_t)pages;
    c->g.tiles_per_page = (uint32_t)tiles;
    c->g.heads = (uint32_t)heads;
    c->g.blocks = nb;
    c->g.k4 = k4;
    c->g.v4 = v4;
    c->g.k_bytes = kv_part_bytes(k4, nb);
    c->g.record_bytes = (uint32_t)record;
    cudaError_t e = device_malloc(ctx, reinterpret_cast<void**>(&c->g.base), c->device_bytes);
    if (e != cudaSuccess) {
        (void)cudaGetLastError();
        return fail(VX_ERR_OUT_OF_MEMORY, "allocating %zu bytes of cache failed: %s", c->device_bytes, cudaGetErrorString(e));
    }
    e = cudaMemsetAsync(c->g.base, 0, c->device_bytes, ctx->stream);
    // any context of the device may be the first to use it
    if (e == cudaSuccess) e = cudaStreamSynchronize(ctx->stream);
    if (e != cudaSuccess) {
        (void)cudaGetLastError();
        cudaFree(c->g.base);
        return fail(VX_ERR_CUDA, "clearing the cache failed: %s", cudaGetErrorString(e));
    }
    *out = c.release();
    return VX_OK;
}

vx_status vx_kv_cache_free(vx_context* ctx, vx_kv_cache* cache) {
    VX_REQUIRE(ctx, VX_ERR_INVALID_ARGUMENT, "vx_kv_cache_free: null context");
    if (!cache) return VX_OK;
    DeviceGuard guard(cache->device);
    VX_CUDA(cudaStreamSynchronize(ctx->stream));
    VX_CUDA(cudaFree(cache->g.base));
    delete cache;
    return VX_OK;
}

vx_status vx_kv_cache_info(const vx_kv_cache* cache, int32_t* k_type, int32_t* v_type, size_t* heads, size_t* head_dim, size_t* pages,
                           size_t* page_tokens, size_t* device_bytes) {
    VX_REQUIRE(cache, VX_ERR_INVALID_ARGUMENT, "vx_kv_cache_info: null cache");
    if (k_type) *k_type = cache->k_type;
    if (v_type) *v_type = cache->v_type;
    if (heads) *heads = cache->g.heads;
    if (head_dim) *head_dim = cache->head_dim;
    if (pages) *pages = cache->g.pages;
    if (page_tokens) *page_tokens = cache->page_tokens;
    if (device_bytes) *device_bytes = cache->device_bytes;
    return VX_OK;
}

vx_status vx_kv_append(vx_context* ctx, vx_kv_cache* cache, const vx_kv_rows* rows, const float* k, size_t k_stride, const float* v,
                       size_t v_stride) {
    VX_REQUIRE(ctx && cache, VX_ERR_INVALID_ARGUMENT, "vx_kv_append: null argument");
    VX_REQUIRE(ctx->device == cache->device, VX_ERR_INVALID_ARGUMENT, "vx_kv_append: the cache is on device %d, the context on %d",
               cache->device, ctx->device);
    KvRows r;
    const vx_status st = kv_rows_check("vx_kv_append", rows, &r);
    if (st != VX_OK || r.rows == 0) return st;
    const size_t width = cache->head_dim * cache->g.heads;
    VX_REQUIRE(k && v, VX_ERR_INVALID_ARGUMENT, "vx_kv_append: null keys or values");
    VX_REQUIRE(r.rows == 1 || (k_stride >= width && v_stride >= width), VX_ERR_INVALID_ARGUMENT,
               "vx_kv_append: rows %zu and %zu elements apart, a row has %zu", k_stride, v_stride, width);
    DeviceGuard guard(ctx->device);
    kv_append_kernel<<<tiles_grid(r, cache->g, 2), kThreads, 0, ctx->stream>>>(r, cache->g, k, k_stride, v, v_stride, vec_ok(k, k_stride),
                                                                              vec_ok(v, v_stride));
    VX_CUDA(cudaGetLastError());
    ctx->launches++;
    return VX_OK;
}

vx_status vx_kv_read(vx_context* ctx, const vx_kv_cache* cache, const vx_kv_rows* rows, float* k, size_t k_stride, float* v, size_t v_stride) {
    VX_REQUIRE(ctx && cache, VX_ERR_INVALID_ARGUMENT, "vx_kv_read: null argument");
    VX_REQUIRE(ctx->device == cache->device, VX_ERR_INVALID_ARGUMENT, "vx_kv_read: the cache is on device %d, the context on %d",
               cache->device, ctx->device);
    KvRows r;
    const vx_status st = kv_rows_check("vx_kv_read", rows, &r);
    if (st != VX_OK || r.rows == 0 || (!k && !v)) return st;
    const size_t width = cache->head_dim * cache->g.heads;
    VX_REQUIRE(r.rows == 1 || ((!k || k_stride >= width) && (!v || v_stride >= width)), VX_ERR_INVALID_ARGUMENT,
               "vx_kv_read: rows %zu and %zu elements apart, a row has %zu", k_stride, v_stride, width);
    DeviceGuard guard(ctx->device);
    kv_read_kernel<<<tiles_grid(r, cache->g, k && v ? 2 : 1), kThreads, 0, ctx->stream>>>(r, cache->g, k, k_stride, v, v_stride,
                                                                                         vec_ok(k, k_stride), vec_ok(v, v_stride));
    VX_CUDA(cudaGetLastError());
    ctx->launches++;
    return VX_OK;
}

}  // extern "C"
