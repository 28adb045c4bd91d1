// The quantised cache of keys and values: storage, quantising on write, reading back.
//
// Formats and arithmetic are those of vx_quantize (IEEE division, scale rounded to f16 before the codes are formed,
// half away from zero); vortx has no counterpart.  One block of threads takes a 32-token tile of some heads, keys or
// values: four lanes share a block of 32 values (two float4 each, the largest magnitude by two shuffles), so rows are read and
// written as whole 64-byte pieces, four loads per lane under way.  A tile that the call covers completely is put
// together in shared memory and goes out as 16-byte vectors; the others' codes are stored where they belong.
// The floor is the f32 side of the copy: 4 bytes a value next to 1.06 (Q8_0) or 0.56 (Q4_0).  Measured, 16 x 1024 tokens of
// 8 heads of 128 in Q4_0 (134 MB of f32, 19 MB of codes): append 47 us (3.3 TB/s; 29 lane operations
// per value, a fifth of which find out where things are, at 0.64 a cycle and scheduler: it waits for its loads and at the two
// barriers a head around the block's image); read 32 us (4.8 TB/s).  Eight lanes to a block took 66 and 36 us. One
// token: 4.6 us for both calls, recorded.
#include <algorithm>
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

// What the format prescribes rests on two f32 quotients, the scale's and v / d.  Products with a reciprocal are within
// 2^-22 of them and give the same f16 scale and the same code except next to a border between two of them; only there
// the division is made.  (With divisions throughout append took 89 us where it then took 66.)
//
// f16(top / n).  The border between two f16 numbers is at bit 12 of an f32 mantissa.
__device__ __forceinline__ uint16_t scale_of(float top, float n, float inv_n) {
    float q = top * inv_n;
    const uint32_t off = (__float_as_uint(q) & 0x1fffu) - 0x0ff8u;
    if (off <= 16u || (!(fabsf(q) >= 6.2e-5f) && q != 0.0f)) q = __fdiv_rn(top, n);  // f16's small numbers have other borders
    return __half_as_ushort(__float2half_rn(q));
}
// The codes of eight values in the words' low bytes, offset included: round half away from zero of v / d; r is 1 / d to 2^-22.
// `special`: the scale is no number, and all codes are zeros, or one of f16's small ones, whose error can take a code out
// of its range; else the largest is 7 or 127 (1 + 2^-11) before it is rounded.
template <bool FOUR>
__device__ __forceinline__ void codes_of(const float (&v)[8], float d, float r, bool special, uint32_t (&c)[8]) {
    constexpr float kMagic = 12582912.0f + (FOUR ? 8.0f : 128.0f);  // 1.5 2^23: the nearest integer in the sum's low bits
    float off = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float y = fmaf(v[i], r, kMagic);
        c[i] = __float_as_uint(y);
        off = fmaxf(off, fabsf(fmaf(v[i], r, kMagic - y)));
    }
    if (off > 0.4999f || special) {  // one of them next to a tie
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int n = d == d ? (int)roundf(__fdiv_rn(v[i], d)) : 0;
            c[i] = (uint32_t)(FOUR ? min(15, max(0, n + 8)) : min(127, max(-127, n)) + 128);
        }
    }
}
// Four low bytes.
__device__ __forceinline__ uint32_t word_of(const uint32_t (&c)[8], int i) {
    return __byte_perm(__byte_perm(c[i], c[i + 1], 0x0040), __byte_perm(c[i + 2], c[i + 3], 0x0040), 0x5410);
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float min_nan(float a, float b) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// The largest magnitude of a block that four lanes share, for Q4_0 with the sign of the first element that has it; NaN if
// there is one.
template <bool FOUR>
__device__ __forceinline__ float largest_of(const float (&v)[8], uint32_t lane, bool there) {
    float high = FOUR ? v[0] : fabsf(v[0]), low = v[0];
#pragma unroll
    for (int n = 1; n < 8; ++n) {
        high = max_nan(high, FOUR ? v[n] : fabsf(v[n]));
        if (FOUR) low = min_nan(low, v[n]);
    }
#pragma unroll
    for (int x = 1; x < 4; x *= 2) {
        high = max_nan(high, __shfl_xor_sync(0xffffffffu, high, x));
        if (FOUR) low = min_nan(low, __shfl_xor_sync(0xffffffffu, low, x));
    }
    if (!FOUR) return high;
    float top = high > -low ? high : low;
    if (__any_sync(0xffffffffu, there && high == -low)) {  // both signs (or zeros): which comes first
        float with[2] = {0.0f, 0.0f};
        bool has[2] = {false, false};
#pragma unroll
        for (int n = 7; n >= 0; --n)
            if (fabsf(v[n]) == fabsf(top)) {
                with[n / 4] = v[n];
                has[n / 4] = true;
            }
        const uint32_t first = __ballot_sync(0xffffffffu, has[0]) >> (lane & 28u) & 15u, second = __ballot_sync(0xffffffffu, has[1]) >> (lane & 28u) & 15u;
        const float one = __shfl_sync(0xffffffffu, first ? with[0] : with[1], (lane & 28u) + (first | second ? __ffs(first ? first : second) - 1 : 0));
        if (first | second) top = one;  // else NaN
    }
    return top;
}

// Pairs (token, block) that a thread has under way at a time.
constexpr uint32_t kBatch = 2, kStep = kThreads / 4;

// p / blocks for a pair's number p < 32 blocks <= 512: the error of the rounded-up reciprocal stays below 1 / blocks.
struct PerToken {
    uint32_t blocks, inverse;
    __device__ explicit PerToken(uint32_t nb) : blocks(nb), inverse((65536 + nb - 1) / nb) {}
    __device__ uint32_t token(uint32_t p) const { return (p * inverse) >> 16; }
};

template <bool FOUR, bool VALUES>
__device__ __forceinline__ void append_part(const KvRows& r, const KvGeometry& g, const TileOf& o, uint8_t* dst, const float* __restrict__ src,
                                            size_t stride, uint32_t head, bool vec, uint8_t* image) {
    const uint32_t quad = threadIdx.x / 4, j = threadIdx.x % 4, lane = threadIdx.x % 32, nb = g.blocks;
    const bool whole = o.t0 == 0 && o.t1 == 32;
    uint8_t* to = whole ? image : dst;
    const uint32_t scales = kv_code_bytes(FOUR, nb), end = o.t1 * nb;
    const PerToken per(nb);
    src += (size_t)head * nb * 32 + j * 4;
    for (uint32_t p0 = o.t0 * nb; p0 < end; p0 += kBatch * kStep) {
        float v[kBatch][8];  // values 4 j .. 4 j + 3 and 16 + 4 j .. of a block
#pragma unroll
        for (uint32_t i = 0; i < kBatch; ++i) {
            const uint32_t p = p0 + i * kStep + quad;
#pragma unroll
            for (int n = 0; n < 8; ++n) v[i][n] = 0.0f;
            if (p < end) {
                const uint32_t token = per.token(p), block = p - token * nb;
                const uint32_t row = o.q.row0 + (o.tile * 32 + token - o.q.first);
                const float* from = src + (size_t)row * stride + block * 32;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if (vec) {
                        const float4 f = __ldcs(reinterpret_cast<const float4*>(from + 16 * h));
                        v[i][4 * h] = f.x; v[i][4 * h + 1] = f.y; v[i][4 * h + 2] = f.z; v[i][4 * h + 3] = f.w;
                    } else {
#pragma unroll
                        for (int n = 0; n < 4; ++n) v[i][4 * h + n] = __ldcs(from + 16 * h + n);
                    }
                }
            }
        }
#pragma unroll
        for (uint32_t i = 0; i < kBatch; ++i) {
            const uint32_t p = p0 + i * kStep + quad, token = per.token(p), block = p - token * nb;
            const float top = largest_of<FOUR>(v[i], lane, p < end);
            uint16_t dh = scale_of(top, FOUR ? 7.0f : 127.0f, FOUR ? 1.0f / 7.0f : 1.0f / 127.0f);
            if ((dh & 0x7fffu) >= 0x7c00u) dh = 0x7fffu;
            // without a scale (all zeros, or too small for one) the codes are those of zeros
            const uint32_t size = dh & 0x7fffu;
            const float d = size == 0 ? 1.0f : __half2float(__ushort_as_half(dh)), inv = __fdividef(1.0f, d);
            uint32_t c[8];
            codes_of<FOUR>(v[i], d, inv, size - 1 < 0x3ffu || size == 0x7fffu, c);
            if (p >= end) continue;
            if (VALUES && FOUR) {
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    *reinterpret_cast<uint16_t*>(to + v_word(true, block, token, j + 4 * h)) =
                        (uint16_t)__byte_perm((c[4 * h] & 15u) | c[4 * h + 1] << 4, (c[4 * h + 2] & 15u) | c[4 * h + 3] << 4, 0x0040);
            } else if (VALUES) {
#pragma unroll
                for (int n = 0; n < 8; ++n) to[v_word(false, block, token, j + n / 4 * 4) + 4 * (n % 4)] = (uint8_t)c[n];
            } else if (FOUR) {  // byte i of a Q4_0 block: values i and i + 16
                *reinterpret_cast<uint32_t*>(to + k_word(true, block, token, j)) = word_of(c, 0) | word_of(c, 4) << 4;
            } else {
#pragma unroll
                for (int h = 0; h < 2; ++h) *reinterpret_cast<uint32_t*>(to + k_word(false, block, token, j + 4 * h)) = word_of(c, 4 * h);
            }
            if (j == 0) *reinterpret_cast<uint16_t*>(to + scales + (VALUES ? v_scale(block, token) : k_scale(block, token))) = dh;
        }
    }
    if (!whole) return;
    __syncthreads();
    const uint4* im = reinterpret_cast<const uint4*>(image);
    for (uint32_t i = threadIdx.x; i < kv_part_bytes(FOUR, nb) / 16; i += kThreads) reinterpret_cast<uint4*>(dst)[i] = im[i];
}

struct KvAppend {
    KvRows r;
    KvGeometry g;
    const float *k, *v;
    size_t k_stride, v_stride;
    int k_vec, v_vec;
    uint32_t heads;  // of a block
};

__global__ void __launch_bounds__(kThreads) kv_append_kernel(KvAppend p) {
    pdl_wait();
    pdl_launch();
    const KvRows& r = p.r;
    const KvGeometry& g = p.g;
    __shared__ __align__(16) uint8_t image[kv_part_bytes(false, kMaxBlocks)];
    const TileOf o = tile_of(r, g, blockIdx.x);
    if (o.t0 >= o.t1) return;
    const uint32_t first = blockIdx.y * p.heads, end = min(g.heads, first + p.heads);
    uint8_t* rec = kv_record(r, g, o.seq, o.tile, first);
    if (!rec) return;
    for (uint32_t head = first; head < end; ++head, rec += g.record_bytes) {
        if (head > first) __syncthreads();  // the last head's image has been copied
        if (blockIdx.z == 0) {
            if (g.k4) append_part<true, false>(r, g, o, rec, p.k, p.k_stride, head, p.k_vec != 0, image);
            else append_part<false, false>(r, g, o, rec, p.k, p.k_stride, head, p.k_vec != 0, image);
        } else {
            if (g.v4) append_part<true, true>(r, g, o, rec + g.k_bytes, p.v, p.v_stride, head, p.v_vec != 0, image);
            else append_part<false, true>(r, g, o, rec + g.k_bytes, p.v, p.v_stride, head, p.v_vec != 0, image);
        }
    }
}

template <bool FOUR, bool VALUES>
__device__ __forceinline__ void read_part(const KvGeometry& g, const TileOf& o, const uint8_t* src, float* __restrict__ dst, size_t stride,
                                          uint32_t head, bool vec) {
    const uint32_t quad = threadIdx.x / 4, j = threadIdx.x % 4, nb = g.blocks;
    const uint32_t scales = kv_code_bytes(FOUR, nb), end = o.t1 * nb;
    const PerToken per(nb);
    dst += (size_t)head * nb * 32 + j * 4;
    for (uint32_t p0 = o.t0 * nb; p0 < end; p0 += kBatch * kStep) {
        uint32_t w[kBatch][2], dh[kBatch];  // straight from the record: its neighbours' words come along in the L1
#pragma unroll
        for (uint32_t i = 0; i < kBatch; ++i) {
            const uint32_t p = p0 + i * kStep + quad, token = per.token(p), block = p - token * nb;
            w[i][0] = w[i][1] = FOUR ? 0x88888888u : 0x80808080u;  // zeros, for tokens without a place
            dh[i] = 0;
            if (src && p < end) {
                dh[i] = *reinterpret_cast<const uint16_t*>(src + scales + (VALUES ? v_scale(block, token) : k_scale(block, token)));
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if (VALUES && FOUR) {
                        w[i][h] = *reinterpret_cast<const uint16_t*>(src + v_word(true, block, token, j + 4 * h));
                    } else if (VALUES) {
                        const uint8_t* at = src + v_word(false, block, token, j + 4 * h);
                        w[i][h] = at[0] | (uint32_t)at[4] << 8 | (uint32_t)at[8] << 16 | (uint32_t)at[12] << 24;
                    } else if (!FOUR || h == 0) {
                        w[i][h] = *reinterpret_cast<const uint32_t*>(src + k_word(FOUR, block, token, FOUR ? j : j + 4 * h));
                    }
                }
            }
        }
#pragma unroll
        for (uint32_t i = 0; i < kBatch; ++i) {
            const uint32_t p = p0 + i * kStep + quad, token = per.token(p), block = p - token * nb;
            if (p >= end) continue;
            const uint32_t row = o.q.row0 + (o.tile * 32 + token - o.q.first);
            const float d = __half2float(__ushort_as_half((uint16_t)dh[i]));
            float* to = dst + (size_t)row * stride + block * 32;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float f[4];
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    const uint32_t shift = !FOUR ? 8 * n : VALUES ? 4 * n : 8 * n + 4 * h;
                    const uint32_t u = (w[i][FOUR && !VALUES ? 0 : h] >> shift) & (FOUR ? 15u : 255u);
                    f[n] = __fmul_rn(d, __uint_as_float(u | 0x4b000000u) - (FOUR ? 8388616.0f : 8388736.0f));  // 2^23 + u
                }
                if (vec) {
                    __stcs(reinterpret_cast<float4*>(to + 16 * h), make_float4(f[0], f[1], f[2], f[3]));
                } else {
#pragma unroll
                    for (int n = 0; n < 4; ++n) __stcs(to + 16 * h + n, f[n]);
                }
            }
        }
    }
}

struct KvRead {
    KvRows r;
    KvGeometry g;
    float *k, *v;
    size_t k_stride, v_stride;
    int k_vec, v_vec;
    uint32_t heads;
};

__global__ void __launch_bounds__(kThreads) kv_read_kernel(KvRead p) {
    pdl_wait();
    pdl_launch();
    const KvRows& r = p.r;
    const KvGeometry& g = p.g;
    const bool values = p.k == nullptr || blockIdx.z == 1;
    const TileOf o = tile_of(r, g, blockIdx.x);
    if (o.t0 >= o.t1) return;
    const uint32_t first = blockIdx.y * p.heads, end = min(g.heads, first + p.heads);
    const uint8_t* rec = kv_record(r, g, o.seq, o.tile, first);
    for (uint32_t head = first; head < end; ++head) {
        const uint8_t* part = rec ? rec + (size_t)(head - first) * g.record_bytes + (values ? g.k_bytes : 0) : nullptr;
        if (!values) {
            if (g.k4) read_part<true, false>(g, o, part, p.k, p.k_stride, head, p.k_vec != 0);
            else read_part<false, false>(g, o, part, p.k, p.k_stride, head, p.k_vec != 0);
        } else {
            if (g.v4) read_part<true, true>(g, o, part, p.v, p.v_stride, head, p.v_vec != 0);
            else read_part<false, true>(g, o, part, p.v, p.v_stride, head, p.v_vec != 0);
        }
    }
}

int vec_ok(const void* p, size_t stride) { return ((reinterpret_cast<uintptr_t>(p) & 15u) == 0 && stride % 4 == 0) ? 1 : 0; }

// Blocks for a call: finding out whose tile it is costs a block as much as a third of a head's work, so blocks take
// several heads where there are enough tiles to fill the GPU twice over all the same.
struct TileLaunch {
    dim3 grid;
    uint32_t heads;  // of a block
    TileLaunch(const vx_context* ctx, const KvRows& r, const KvGeometry& g, unsigned parts) {
        const uint32_t tiles = r.rows / 32 + 2 * r.seqs;
        const uint64_t one = (uint64_t)tiles * g.heads * parts, fill = (uint64_t)ctx->sm_count * 16;
        heads = (uint32_t)std::min<uint64_t>(std::max<uint64_t>(1, one / fill), g.heads);
        grid = dim3(tiles, (g.heads + heads - 1) / heads, parts);
    }
};

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
    // the kernels' code is loaded now, so that the first call may be one that is being recorded
    cudaFuncAttributes loaded;
    VX_CUDA(cudaFuncGetAttributes(&loaded, kv_append_kernel));
    VX_CUDA(cudaFuncGetAttributes(&loaded, kv_read_kernel));
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
    const TileLaunch l(ctx, r, cache->g, 2);
    const KvAppend p{r, cache->g, k, v, k_stride, v_stride, vec_ok(k, k_stride), vec_ok(v, v_stride), l.heads};
    VX_CUDA(launch_after(kv_append_kernel, l.grid, kThreads, 0, ctx->stream, p));
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
    const TileLaunch l(ctx, r, cache->g, k && v ? 2 : 1);
    const KvRead p{r, cache->g, k, v, k_stride, v_stride, vec_ok(k, k_stride), vec_ok(v, v_stride), l.heads};
    VX_CUDA(launch_after(kv_read_kernel, l.grid, kThreads, 0, ctx->stream, p));
    ctx->launches++;
    return VX_OK;
}

}  // extern "C"
