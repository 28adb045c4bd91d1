// A mixture-of-experts layer for a few tokens on block-quantised weights, in three launches:
//   route   logits = router x (a warp per expert and four tokens), x split into two f16 parts per block of 32
//           (vx_decode.cuh); the last block to finish picks the experts and lists every expert's tokens
//   inner   silu(gate x) * (up x): a thread block per (expert with tokens, 32 inner rows)
//   down    y = sum weight * (down h): a thread block per (32 output rows, share of all experts' columns)
// Bound by the weights' bytes: each is read once per 16 tokens of its expert.  In both products a warp has every
// eighth 64-byte column chunk of the unit's rows (16-byte cp.async copies, two chunks in flight per warp, no
// synchronisation between warps until the sums are added up), multiplies it on the tensor cores
// (m16n8k16: 16 rows of codes, columns 2 i and 2 i + 1 are the two parts of token i, so a thread holds both sums of a
// (row, token)) and scales every block's sums in f32.
#include <algorithm>
#include <memory>
#include <new>

#include "vx_decode.cuh"

namespace {

using namespace vx;

constexpr uint32_t kMoeWarps = 8, kMoeThreads = kMoeWarps * 32;
constexpr uint32_t kMaxExperts = 256, kMaxTopK = 16, kMaxTokens = 64;
constexpr uint32_t kGroup = 16;             // tokens of an expert per pass over its weights
constexpr uint32_t kPitch = 80;             // a row's 64-byte chunk in shared memory: eight rows meet different banks
constexpr uint32_t kScaleWords = 3;         // a chunk's scales (2 or 4 halves at any 2-byte offset), as 4-byte words
constexpr uint32_t kStages = 2;

struct Matrix {
    const uint8_t* quants;
    const uint16_t* scales;
};

struct MoeParams {
    const float* x;
    float* y;
    size_t x_stride, y_stride;
    const float* router;
    uint32_t tokens, experts, top_k, hidden, inner, splits;
    int normalise, down4, x_vec, gate4;
    Matrix gate, up, down;
    float* logits;       // [tokens][experts]
    uint8_t* xh;         // [tokens][2 parts][hidden / 32][64 bytes], B-operand order
    float* xs;           // [tokens][hidden / 32], what a block's parts are multiplied with
    uint8_t* hh;         // the inner vectors, per slot = token * top_k + place
    float* hs;
    uint32_t* plan;      // [0] experts with tokens, then [experts] which, [experts + 1] where their lists begin
    uint32_t* list;      // slots by expert, ascending
    float* weights;      // per slot
    float* part;         // [splits][tokens][hidden]
    uint32_t* counters;  // [0] route, [1 + i] output rows 32 i ..; zero between calls
    int32_t* ids_out;
    float* weights_out;
};

__device__ __forceinline__ uint32_t redux_max(uint32_t v) { return __reduce_max_sync(0xffffffffu, v); }
__device__ __forceinline__ uint32_t redux_min(uint32_t v) { return __reduce_min_sync(0xffffffffu, v); }

// Whether this block is the last of `count` to get here; everything the others wrote before is then visible.
__device__ __forceinline__ bool last_of(uint32_t* counter, uint32_t count, uint32_t* shared) {
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) *shared = atomicInc(counter, count - 1);  // back to 0 with the last one
    __syncthreads();
    const bool last = *shared == count - 1;
    if (last) __threadfence();
    return last;
}

// ------------------------------------------------------------------------------------------------- route ----
// Sums of one expert's row with tokens t0 .. t0 + 3.
__device__ __forceinline__ void logits_of(const MoeParams& p, uint32_t expert, uint32_t t0, uint32_t lane) {
    const float* w = p.router + (size_t)expert * p.hidden;
    const uint32_t n = min(4u, p.tokens - t0);
    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (p.x_vec) {
#pragma unroll 4
        for (uint32_t i = lane * 4; i < p.hidden; i += 128) {
            const float4 a = __ldg(reinterpret_cast<const float4*>(w + i));
#pragma unroll
            for (uint32_t t = 0; t < 4; ++t)
                if (t < n) {
                    const float4 b = *reinterpret_cast<const float4*>(p.x + (size_t)(t0 + t) * p.x_stride + i);
                    sum[t] = fmaf(a.x, b.x, fmaf(a.y, b.y, fmaf(a.z, b.z, fmaf(a.w, b.w, sum[t]))));
                }
        }
    } else {
#pragma unroll 4
        for (uint32_t i = lane; i < p.hidden; i += 32) {
            const float a = __ldg(w + i);
#pragma unroll
            for (uint32_t t = 0; t < 4; ++t)
                if (t < n) sum[t] = fmaf(a, p.x[(size_t)(t0 + t) * p.x_stride + i], sum[t]);
        }
    }
#pragma unroll
    for (uint32_t t = 0; t < 4; ++t) {
        const float s = warp_add(sum[t]);
        if (t < n && lane == 0) p.logits[(size_t)(t0 + t) * p.experts + expert] = s;
    }
}

// One block of 32 values (a lane each) as two parts in B-operand order.
__device__ __forceinline__ void split_block(float v, uint32_t lane, bool four, uint8_t* hi, uint8_t* lo, float* scale) {
    const float up = lift(warp_max(fabsf(v)));
    const float x = v * up;
    const __half h = __float2half_rn(x), l = __float2half_rn(x - __half2float(h));
    const uint32_t at = frag_lane(lane) * 16 + frag_half(four, lane) * 2;
    *reinterpret_cast<__half*>(hi + at) = h;
    *reinterpret_cast<__half*>(lo + at) = l;
    if (lane == 0) *scale = 1.0f / up;
}

__global__ void __launch_bounds__(kMoeThreads) moe_route_kernel(const MoeParams p) {
    __shared__ uint32_t last;
    __shared__ uint16_t chosen[kMaxTokens * kMaxTopK];
    __shared__ uint32_t scan[2][kMoeWarps];
    pdl_wait();
    pdl_launch();
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nb = p.hidden / 32;
    const uint32_t quads = (p.tokens + 3) / 4, dots = p.experts * quads, pieces = (nb + 15) / 16;
    for (uint32_t job = blockIdx.x * kMoeWarps + warp; job < dots + p.tokens * pieces; job += gridDim.x * kMoeWarps) {
        if (job < dots) {
            logits_of(p, job / quads, (job % quads) * 4, lane);
        } else {
            const uint32_t t = (job - dots) / pieces, b0 = (job - dots) % pieces * 16;
#pragma unroll 4
            for (uint32_t b = b0; b < min(b0 + 16, nb); ++b) {
                uint8_t* hi = p.xh + ((size_t)t * 2 * nb + b) * 64;
                split_block(p.x[(size_t)t * p.x_stride + b * 32 + lane], lane, p.gate4 != 0, hi, hi + (size_t)nb * 64,
                            p.xs + (size_t)t * nb + b);
            }
        }
    }
    if (!last_of(p.counters, gridDim.x, &last)) return;

    // ---- the top_k experts of every token, a warp each ---------------------------------------------------------
    for (uint32_t t = warp; t < p.tokens; t += kMoeWarps) {
        float v[kMaxExperts / 32];
        uint32_t key[kMaxExperts / 32];  // order of the numbers, NaN lowest; 0 and `gone`: not to be taken (again)
        uint32_t gone = 0;
        float all = 0.0f;
#pragma unroll
        for (uint32_t i = 0; i < kMaxExperts / 32; ++i) {
            const uint32_t e = lane + 32 * i;
            v[i] = e < p.experts ? __ldcg(p.logits + (size_t)t * p.experts + e) : -INFINITY;
            const uint32_t u = __float_as_uint(v[i]);
            key[i] = v[i] != v[i] ? 1u : (u >> 31 ? ~u : u | 0x80000000u);
            if (v[i] == 0.0f) key[i] = 0x80000000u;  // -0 and 0 are a tie
            if (e >= p.experts) gone |= 1u << i;
        }
        float top = 0.0f, chosen_value = 0.0f;
        for (uint32_t j = 0; j < p.top_k; ++j) {
            uint32_t best = 0, at = 0;
#pragma unroll
            for (uint32_t i = 0; i < kMaxExperts / 32; ++i)
                if (!(gone >> i & 1) && key[i] > best) {
                    best = key[i];
                    at = lane + 32 * i;
                }
            const uint32_t winner = redux_max(best);
            const uint32_t e = redux_min(best == winner ? at : 0xffffffffu);
            if (best == winner && at == e) gone |= 1u << (e / 32);
            const float f = winner == 1u ? NAN : __uint_as_float(winner >> 31 ? winner & 0x7fffffffu : ~winner);
            if (j == 0) top = f;
            if (lane == j) {
                chosen[t * p.top_k + j] = (uint16_t)e;
                chosen_value = f;
                if (p.ids_out) p.ids_out[(size_t)t * p.top_k + j] = (int32_t)e;
            }
        }
        if (p.normalise) {
            all = warp_add(lane < p.top_k ? expf(chosen_value - top) : 0.0f);
        } else {
#pragma unroll
            for (uint32_t i = 0; i < kMaxExperts / 32; ++i)
                if (lane + 32 * i < p.experts) all += expf(v[i] - top);
            all = warp_add(all);
        }
        if (lane < p.top_k) {
            const float w = expf(chosen_value - top) / all;
            p.weights[t * p.top_k + lane] = w;
            if (p.weights_out) p.weights_out[(size_t)t * p.top_k + lane] = w;
        }
    }
    __syncthreads();

    // ---- every expert's slots, ascending; a thread per expert -------------------------------------------------------
    const uint32_t e = threadIdx.x, slots = p.tokens * p.top_k;
    uint32_t count = 0;
    if (e < p.experts)
        for (uint32_t s = 0; s < slots; ++s) count += chosen[s] == e;
    uint32_t before = count, used = count ? 1 : 0, place = used;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const uint32_t a = __shfl_up_sync(0xffffffffu, before, o), b = __shfl_up_sync(0xffffffffu, place, o);
        if (lane >= (uint32_t)o) {
            before += a;
            place += b;
        }
    }
    if (lane == 31) {
        scan[0][warp] = before;
        scan[1][warp] = place;
    }
    __syncthreads();
    uint32_t active = 0;
    for (uint32_t w = 0; w < kMoeWarps; ++w) {
        if (w < warp) {
            before += scan[0][w];
            place += scan[1][w];
        }
        active += scan[1][w];
    }
    before -= count;
    place -= used;
    if (threadIdx.x == 0) {
        p.plan[0] = active;
        p.plan[1 + p.experts + active] = slots;
    }
    if (used) {
        p.plan[1 + place] = e;
        p.plan[1 + p.experts + place] = before;
        for (uint32_t s = 0; s < slots; ++s)
            if (chosen[s] == e) p.list[before++] = s;
    }
}

// ---------------------------------------------------------------------------------------------- products ----
// A warp's stage: ROWS rows of one column chunk (64 bytes: four Q4_0 or two Q8_0 blocks) and their scales.
template <bool FOUR, int TILES>
struct Stage {
    static constexpr uint32_t rows = TILES * 16, blocks = FOUR ? 4 : 2;
    static constexpr uint32_t scales = rows * kPitch, bytes = scales + rows * kScaleWords * 4;
};

// Copies chunk c of 32 rows that begin at row `row0` of the matrix into rows at .. at + 31 of the stage.
template <bool FOUR>
__device__ __forceinline__ void fetch_rows(const Matrix& m, size_t row0, uint32_t nb, uint32_t c, uint32_t stage, uint32_t scales, uint32_t at,
                                           uint32_t lane) {
    constexpr uint32_t B = FOUR ? 4 : 2;
    const uint32_t row_bytes = nb * (FOUR ? 16 : 32), col = c * 64 + (lane & 3) * 16;
    if (col < row_bytes) {
        const uint8_t* src = m.quants + (row0 + (lane >> 2)) * row_bytes + col;
        const uint32_t dst = stage + (at + (lane >> 2)) * kPitch + (lane & 3) * 16;
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) cp_async16(dst + i * 8 * kPitch, src + (size_t)i * 8 * row_bytes);
    }
    const size_t h0 = (row0 + lane) * nb + c * B;
    const uint32_t words = ((uint32_t)(h0 & 1) + min(B, nb - c * B) + 1) / 2;
    const uint8_t* src = reinterpret_cast<const uint8_t*>(m.scales) + (h0 >> 1) * 4;
    const uint32_t dst = scales + (at + lane) * (kScaleWords * 4);
#pragma unroll
    for (uint32_t i = 0; i < (FOUR ? 3 : 2); ++i)
        if (i < words) cp_async4(dst + i * 4, src + i * 4);
}

// The scales of one row's blocks of the chunk, as f32.
template <bool FOUR>
__device__ __forceinline__ void scales_of(uint32_t addr, uint32_t odd, float (&d)[FOUR ? 4 : 2]) {
    uint32_t w0 = lds32(addr), w1 = lds32(addr + 4);
    if (FOUR) {
        const uint32_t w2 = lds32(addr + 8);
        if (odd) {
            w0 = __funnelshift_r(w0, w1, 16);
            w1 = __funnelshift_r(w1, w2, 16);
        }
        const float2 a = __half22float2(bits_h2(w0)), b = __half22float2(bits_h2(w1));
        d[0] = a.x;
        d[1] = a.y;
        d[FOUR ? 2 : 0] = b.x;
        d[FOUR ? 3 : 1] = b.y;
    } else {
        if (odd) w0 = __funnelshift_r(w0, w1, 16);
        const float2 a = __half22float2(bits_h2(w0));
        d[0] = a.x;
        d[1] = a.y;
    }
}

// What a lane needs of the vectors: the B operand of token 4 n + g / 2 (part g % 2), the block scales of token 4 n + t.
template <int NT>
struct Vectors {
    const uint8_t* parts[NT];  // null: no such token
    const float* scale[NT];
};

// acc[m][n] += chunk's 16-row tiles times the vectors: rows g and g + 8 of tile m, token 4 n + t.
// odd[m]: bit 0 / 1 = whether the scales of rows g / g + 8 begin at an odd half.
template <bool FOUR, int TILES, int NT>
__device__ __forceinline__ void multiply(uint32_t stage, uint32_t c, uint32_t nb, const Vectors<NT>& x, const uint32_t (&odd)[TILES], uint32_t lane,
                                         float (&acc)[TILES][NT][2], const uint4 (&bq)[FOUR ? 4 : 2][NT], const float (&sx)[FOUR ? 4 : 2][NT]) {
    constexpr uint32_t B = FOUR ? 4 : 2;
    const uint32_t g = lane >> 2;
    float d[TILES][2][B];
#pragma unroll
    for (int m = 0; m < TILES; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h)
            scales_of<FOUR>(stage + Stage<FOUR, TILES>::scales + (m * 16 + h * 8 + g) * (kScaleWords * 4), (odd[m] >> h) & 1, d[m][h]);
#pragma unroll
    for (uint32_t j = 0; j < B; ++j) {
        if (c * B + j >= nb) break;
        uint32_t a[TILES][2][4];
        if (FOUR) {
#pragma unroll
            for (int m = 0; m < TILES; m += 2) {
                uint32_t w[4];
                ldmatrix_x4(w, stage + (m * 16 + lane) * kPitch + j * 16);
                a_of_nibbles(w[0], w[1], a[m]);
                a_of_nibbles(w[2], w[3], a[m + 1]);
            }
        } else {
#pragma unroll
            for (int m = 0; m < TILES; ++m) {
                uint32_t w[4];
                ldmatrix_x4(w, stage + (m * 16 + (lane & 15)) * kPitch + j * 32 + (lane >> 4) * 16);
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] ^= 0x80808080u;
                a_of_bytes(w, a[m]);
            }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int m = 0; m < TILES; ++m) {
                float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                mma_f16(s, a[m][0], bq[j][n].x, bq[j][n].y);
                mma_f16(s, a[m][1], bq[j][n].z, bq[j][n].w);
                acc[m][n][0] = fmaf((s[0] + s[1]) * sx[j][n], d[m][0][j], acc[m][n][0]);
                acc[m][n][1] = fmaf((s[2] + s[3]) * sx[j][n], d[m][1][j], acc[m][n][1]);
            }
    }
}

template <bool FOUR, int NT>
__device__ __forceinline__ void load_vectors(const Vectors<NT>& x, uint32_t c, uint32_t nb, uint4 (&bq)[FOUR ? 4 : 2][NT],
                                             float (&sx)[FOUR ? 4 : 2][NT]) {
    constexpr uint32_t B = FOUR ? 4 : 2;
#pragma unroll
    for (uint32_t j = 0; j < B; ++j)
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            bq[j][n] = make_uint4(0, 0, 0, 0);
            sx[j][n] = 0.0f;
            if (c * B + j < nb) {
                if (x.parts[n]) bq[j][n] = *reinterpret_cast<const uint4*>(x.parts[n] + (size_t)(c * B + j) * 64);
                if (x.scale[n]) sx[j][n] = x.scale[n][c * B + j];
            }
        }
}

// ------------------------------------------------------------------------------------------------- inner ----
template <bool FOUR>
constexpr uint32_t inner_smem() {
    constexpr uint32_t ring = kMoeWarps * kStages * Stage<FOUR, 4>::bytes, sums = kMoeWarps * 64 * (kGroup + 1) * 4;
    return ring > sums ? ring : sums;
}

template <bool FOUR, int NT>
__device__ void inner_unit(const MoeParams& p, uint32_t expert, uint32_t rows32, const uint32_t* slots, uint32_t count, uint8_t* smem) {
    using S = Stage<FOUR, 4>;
    constexpr uint32_t B = S::blocks;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint32_t nb = p.hidden / 32, chunks = (nb + B - 1) / B, nbf = p.inner / 32;
    const size_t row0 = (size_t)expert * p.inner + rows32 * 32;
    Vectors<NT> x;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const uint32_t i = 4 * n + g / 2, k = 4 * n + t;
        x.parts[n] = i < count ? p.xh + ((size_t)(slots[i] / p.top_k) * 2 + (g & 1)) * nb * 64 + t * 16 : nullptr;
        x.scale[n] = k < count ? p.xs + (size_t)(slots[k] / p.top_k) * nb : nullptr;
    }
    uint32_t odd[4];  // a chunk begins at an even block
#pragma unroll
    for (int m = 0; m < 4; ++m)
        odd[m] = (uint32_t)((row0 + (m & 1) * 16 + g) * nb & 1) | (uint32_t)((row0 + (m & 1) * 16 + 8 + g) * nb & 1) << 1;
    const uint32_t ring = smem_addr(smem) + warp * kStages * S::bytes;
    auto fetch = [&](uint32_t k) {
        const uint32_t c = warp + k * kMoeWarps;
        if (c < chunks) {
            const uint32_t st = ring + (k % kStages) * S::bytes;
            fetch_rows<FOUR>(p.gate, row0, nb, c, st, st + S::scales, 0, lane);
            fetch_rows<FOUR>(p.up, row0, nb, c, st, st + S::scales, 32, lane);
        }
        cp_async_commit();
    };
    float acc[4][NT][2];
#pragma unroll
    for (int m = 0; m < 4; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[m][n][0] = acc[m][n][1] = 0.0f;
#pragma unroll
    for (uint32_t k = 0; k < kStages; ++k) fetch(k);
    for (uint32_t k = 0; warp + k * kMoeWarps < chunks; ++k) {
        const uint32_t c = warp + k * kMoeWarps;
        uint4 bq[B][NT];
        float sx[B][NT];
        load_vectors<FOUR, NT>(x, c, nb, bq, sx);
        cp_async_wait<kStages - 1>();
        __syncwarp();
        multiply<FOUR, 4, NT>(ring + (k % kStages) * S::bytes, c, nb, x, odd, lane, acc, bq, sx);
        __syncwarp();
        fetch(k + kStages);
    }
    cp_async_wait<0>();
    __syncthreads();
    // ---- the eight warps' sums: gate rows 0..31, up rows 32..63 ------------------------------------------------------
    constexpr uint32_t W = 4 * NT + 1;
    float* sums = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int m = 0; m < 4; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int h = 0; h < 2; ++h) sums[(warp * 64 + m * 16 + h * 8 + g) * W + 4 * n + t] = acc[m][n][h];
    __syncthreads();
    for (uint32_t i = warp; i < count; i += kMoeWarps) {
        float a = 0.0f, b = 0.0f;
#pragma unroll
        for (uint32_t w = 0; w < kMoeWarps; ++w) {
            a += sums[(w * 64 + lane) * W + i];
            b += sums[(w * 64 + 32 + lane) * W + i];
        }
        const float h = a / (1.0f + expf(-a)) * b;
        const uint32_t slot = slots[i];
        uint8_t* hi = p.hh + ((size_t)slot * 2 * nbf + rows32) * 64;
        split_block(h, lane, p.down4 != 0, hi, hi + (size_t)nbf * 64, p.hs + (size_t)slot * nbf + rows32);
    }
    __syncthreads();
}

template <bool FOUR>
__global__ void __launch_bounds__(kMoeThreads, 2) moe_inner_kernel(const MoeParams p) {
    extern __shared__ __align__(128) uint8_t smem[];
    pdl_wait();
    pdl_launch();
    const uint32_t tiles = p.inner / 32, units = p.plan[0] * tiles;
    for (uint32_t u = blockIdx.x; u < units; u += gridDim.x) {
        const uint32_t a = u / tiles, rows32 = u - a * tiles, expert = p.plan[1 + a];
        const uint32_t begin = p.plan[1 + p.experts + a], end = p.plan[2 + p.experts + a];
        for (uint32_t at = begin; at < end; at += kGroup) {
            const uint32_t count = min(kGroup, end - at);
            if (count <= 4) inner_unit<FOUR, 1>(p, expert, rows32, p.list + at, count, smem);
            else if (count <= 8) inner_unit<FOUR, 2>(p, expert, rows32, p.list + at, count, smem);
            else inner_unit<FOUR, 4>(p, expert, rows32, p.list + at, count, smem);
        }
    }
}

// -------------------------------------------------------------------------------------------------- down ----
template <bool FOUR>
constexpr uint32_t down_ring() {
    return kMoeWarps * kStages * Stage<FOUR, 2>::bytes;
}

// This warp's chunks of one expert and up to 4 NT of its tokens; the weighted sums go to the warp's own rows of `mine`.
template <bool FOUR, int NT>
__device__ __forceinline__ void down_expert(const MoeParams& p, uint32_t expert, size_t row0, uint32_t c0, uint32_t c1, const uint32_t* slots,
                                            uint32_t count, uint32_t ring, float* mine, uint32_t lane) {
    using S = Stage<FOUR, 2>;
    constexpr uint32_t B = S::blocks;
    const uint32_t g = lane >> 2, t = lane & 3, nb = p.inner / 32;
    Vectors<NT> x;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const uint32_t i = 4 * n + g / 2, k = 4 * n + t;
        x.parts[n] = i < count ? p.hh + ((size_t)slots[i] * 2 + (g & 1)) * nb * 64 + t * 16 : nullptr;
        x.scale[n] = k < count ? p.hs + (size_t)slots[k] * nb : nullptr;
    }
    uint32_t odd[2];
#pragma unroll
    for (int m = 0; m < 2; ++m) odd[m] = (uint32_t)((row0 + m * 16 + g) * nb & 1) | (uint32_t)((row0 + m * 16 + 8 + g) * nb & 1) << 1;
    float acc[2][NT][2];
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[m][n][0] = acc[m][n][1] = 0.0f;
    auto fetch = [&](uint32_t c, uint32_t k) {
        if (c < c1) {
            const uint32_t st = ring + (k % kStages) * S::bytes;
            fetch_rows<FOUR>(p.down, row0, nb, c, st, st + S::scales, 0, lane);
        }
        cp_async_commit();
    };
#pragma unroll
    for (uint32_t k = 0; k < kStages; ++k) fetch(c0 + k * kMoeWarps, k);
    uint32_t k = 0;
    for (uint32_t c = c0; c < c1; c += kMoeWarps, ++k) {
        uint4 bq[B][NT];
        float sx[B][NT];
        load_vectors<FOUR, NT>(x, c, nb, bq, sx);
        cp_async_wait<kStages - 1>();
        __syncwarp();
        multiply<FOUR, 2, NT>(ring + (k % kStages) * S::bytes, c, nb, x, odd, lane, acc, bq, sx);
        __syncwarp();
        fetch(c + kStages * kMoeWarps, k);
    }
    cp_async_wait<0>();
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const uint32_t i = 4 * n + t;
        if (i < count) {
            const uint32_t slot = slots[i];
            const float w = p.weights[slot];
            float* to = mine + (slot / p.top_k) * 33;
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int h = 0; h < 2; ++h) to[m * 16 + h * 8 + g] = fmaf(w, acc[m][n][h], to[m * 16 + h * 8 + g]);
        }
    }
    __syncwarp();
}

template <bool FOUR>
__global__ void __launch_bounds__(kMoeThreads, 2) moe_down_kernel(const MoeParams p) {
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint32_t last;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float* sums = reinterpret_cast<float*>(smem + down_ring<FOUR>());  // [warps][tokens][33]
    float* mine = sums + warp * p.tokens * 33;
    for (uint32_t i = lane; i < p.tokens * 33; i += 32) mine[i] = 0.0f;
    __syncwarp();
    pdl_wait();
    pdl_launch();
    const uint32_t tile = blockIdx.x, split = blockIdx.y;
    const uint32_t nb = p.inner / 32, chunks = (nb + (FOUR ? 3 : 1)) / (FOUR ? 4 : 2), active = p.plan[0];
    const uint64_t all = (uint64_t)active * chunks;
    // this block's share of all experts' chunks; the warps take them in turn
    const uint32_t lo = (uint32_t)(all * split / p.splits), hi = (uint32_t)(all * (split + 1) / p.splits);
    const uint32_t ring = smem_addr(smem) + warp * kStages * Stage<FOUR, 2>::bytes;
    for (uint32_t a = lo / chunks; a < active && a * chunks < hi; ++a) {
        const uint32_t first = a * chunks, from = max(lo, first), to = min(hi, first + chunks);
        // the first chunk >= from whose number is the warp's, counted through all experts
        const uint32_t c0 = from + (warp + kMoeWarps - (from - lo) % kMoeWarps) % kMoeWarps;
        if (c0 >= to) continue;
        const uint32_t expert = p.plan[1 + a], begin = p.plan[1 + p.experts + a], end = p.plan[2 + p.experts + a];
        const size_t row0 = (size_t)expert * p.hidden + tile * 32;
        for (uint32_t at = begin; at < end; at += kGroup) {
            const uint32_t count = min(kGroup, end - at);
            if (count <= 4) down_expert<FOUR, 1>(p, expert, row0, c0 - first, to - first, p.list + at, count, ring, mine, lane);
            else if (count <= 8) down_expert<FOUR, 2>(p, expert, row0, c0 - first, to - first, p.list + at, count, ring, mine, lane);
            else down_expert<FOUR, 4>(p, expert, row0, c0 - first, to - first, p.list + at, count, ring, mine, lane);
        }
    }
    __syncthreads();
    for (uint32_t t = warp; t < p.tokens; t += kMoeWarps) {
        float s = 0.0f;
#pragma unroll
        for (uint32_t w = 0; w < kMoeWarps; ++w) s += sums[(w * p.tokens + t) * 33 + lane];
        if (p.splits == 1) p.y[(size_t)t * p.y_stride + tile * 32 + lane] = s;
        else p.part[((size_t)split * p.tokens + t) * p.hidden + tile * 32 + lane] = s;
    }
    if (p.splits == 1) return;
    if (!last_of(p.counters + 1 + tile, p.splits, &last)) return;
    for (uint32_t t = warp; t < p.tokens; t += kMoeWarps) {
        float s = 0.0f;
        for (uint32_t i = 0; i < p.splits; ++i) s += __ldcg(p.part + ((size_t)i * p.tokens + t) * p.hidden + tile * 32 + lane);
        p.y[(size_t)t * p.y_stride + tile * 32 + lane] = s;
    }
}

template <class K>
cudaError_t launch_pdl(K kernel, dim3 grid, uint32_t smem, cudaStream_t stream, const MoeParams& p) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(kMoeThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, p);
}

size_t round_up(size_t v, size_t a) { return (v + a - 1) / a * a; }

}  // namespace

struct vx_moe {
    const vx_context* ctx = nullptr;
    MoeParams p{};
    size_t max_tokens = 0;
    uint32_t inner_grid = 0, sm_count = 0;
    uint8_t* workspace = nullptr;
};

extern "C" {

vx_status vx_moe_create(vx_context* ctx, const float* router, size_t experts, const vx_qweights* gate, const vx_qweights* up,
                        const vx_qweights* down, size_t top_k, int32_t normalise, size_t max_tokens, vx_moe** out) {
    VX_REQUIRE(ctx && router && gate && up && down && out, VX_ERR_INVALID_ARGUMENT, "vx_moe_create: null argument");
    *out = nullptr;
    VX_REQUIRE(experts >= 1 && experts <= kMaxExperts, VX_ERR_UNSUPPORTED, "vx_moe_create: %zu experts (1 to %u)", experts, kMaxExperts);
    VX_REQUIRE(top_k >= 1 && top_k <= experts && top_k <= kMaxTopK, VX_ERR_UNSUPPORTED, "vx_moe_create: top_k %zu of %zu experts (1 to %u)", top_k,
               experts, kMaxTopK);
    VX_REQUIRE(max_tokens >= 1 && max_tokens <= kMaxTokens, VX_ERR_UNSUPPORTED, "vx_moe_create: max_tokens %zu (1 to %u)", max_tokens, kMaxTokens);
    VX_REQUIRE(gate->device == ctx->device && up->device == ctx->device && down->device == ctx->device, VX_ERR_INVALID_ARGUMENT,
               "vx_moe_create: weights of another device");
    VX_REQUIRE(gate->type == up->type, VX_ERR_UNSUPPORTED, "vx_moe_create: gate and up must have one type");
    VX_REQUIRE(gate->rows % experts == 0 && gate->rows == up->rows && gate->cols == up->cols, VX_ERR_SHAPE,
               "vx_moe_create: gate is %zu x %zu, up %zu x %zu, for %zu experts", gate->rows, gate->cols, up->rows, up->cols, experts);
    const size_t hidden = gate->cols, inner = gate->rows / experts;
    VX_REQUIRE(down->cols == inner && down->rows == experts * hidden, VX_ERR_SHAPE, "vx_moe_create: down is %zu x %zu, expected %zu x %zu",
               down->rows, down->cols, experts * hidden, inner);
    VX_REQUIRE(hidden <= 0x1000000 && inner <= 0x1000000, VX_ERR_UNSUPPORTED, "vx_moe_create: experts of %zu x %zu are too large", inner, hidden);
    DeviceGuard guard(ctx->device);
    std::unique_ptr<vx_moe> m(new (std::nothrow) vx_moe());
    VX_REQUIRE(m, VX_ERR_OUT_OF_MEMORY, "host allocation failed");
    m->ctx = ctx;
    m->max_tokens = max_tokens;
    m->sm_count = (uint32_t)ctx->sm_count;
    MoeParams& p = m->p;
    p.router = router;
    p.experts = (uint32_t)experts;
    p.top_k = (uint32_t)top_k;
    p.hidden = (uint32_t)hidden;
    p.inner = (uint32_t)inner;
    p.normalise = normalise != 0;
    p.gate4 = gate->type == VX_Q4_0;
    p.down4 = down->type == VX_Q4_0;
    p.gate = {gate->d_quants, gate->d_scales};
    p.up = {up->d_quants, up->d_scales};
    p.down = {down->d_quants, down->d_scales};
    // Output rows in tiles of 32; few tiles share out the columns too, so that about two blocks per SM have work.
    const uint32_t tiles = p.hidden / 32;
    p.splits = std::min(16u, std::max(1u, 2 * m->sm_count / tiles));
    const int inner_bytes = (int)(p.gate4 ? inner_smem<true>() : inner_smem<false>());
    const int down_bytes = (int)((p.down4 ? down_ring<true>() : down_ring<false>()) + kMoeWarps * max_tokens * 33 * 4);
    int per_sm = 0;
    if (p.gate4) {
        VX_CUDA(cudaFuncSetAttribute(moe_inner_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, inner_bytes));
        VX_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, moe_inner_kernel<true>, kMoeThreads, inner_bytes));
    } else {
        VX_CUDA(cudaFuncSetAttribute(moe_inner_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, inner_bytes));
        VX_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, moe_inner_kernel<false>, kMoeThreads, inner_bytes));
    }
    m->inner_grid = (uint32_t)std::max(1, per_sm) * m->sm_count;
    const int most = (int)((p.down4 ? down_ring<true>() : down_ring<false>()) + kMoeWarps * kMaxTokens * 33 * 4);
    if (p.down4) VX_CUDA(cudaFuncSetAttribute(moe_down_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, most));
    else VX_CUDA(cudaFuncSetAttribute(moe_down_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, most));
    (void)down_bytes;
    // ---- workspace ------------------------------------------------------------------------------------------------------
    const size_t slots = max_tokens * top_k, nbh = hidden / 32, nbf = inner / 32;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t o = at;
        at += round_up(bytes, 256);
        return o;
    };
    const size_t o_counters = take((1 + tiles) * 4), o_logits = take(max_tokens * experts * 4), o_xh = take(max_tokens * 2 * nbh * 64),
                 o_xs = take(max_tokens * nbh * 4), o_hh = take(slots * 2 * nbf * 64), o_hs = take(slots * nbf * 4),
                 o_plan = take((2 + 2 * experts) * 4), o_list = take(slots * 4), o_weights = take(slots * 4),
                 o_part = take(p.splits > 1 ? p.splits * max_tokens * hidden * 4 : 0);
    cudaError_t e = device_malloc(ctx, reinterpret_cast<void**>(&m->workspace), at);
    if (e != cudaSuccess) {
        (void)cudaGetLastError();
        return fail(VX_ERR_OUT_OF_MEMORY, "allocating %zu bytes of expert-layer workspace failed: %s", at, cudaGetErrorString(e));
    }
    e = cudaMemsetAsync(m->workspace, 0, (1 + tiles) * 4, ctx->stream);
    if (e != cudaSuccess) {
        (void)cudaGetLastError();
        cudaFree(m->workspace);
        return fail(VX_ERR_CUDA, "clearing the expert-layer counters failed: %s", cudaGetErrorString(e));
    }
    uint8_t* w = m->workspace;
    p.counters = reinterpret_cast<uint32_t*>(w + o_counters);
    p.logits = reinterpret_cast<float*>(w + o_logits);
    p.xh = w + o_xh;
    p.xs = reinterpret_cast<float*>(w + o_xs);
    p.hh = w + o_hh;
    p.hs = reinterpret_cast<float*>(w + o_hs);
    p.plan = reinterpret_cast<uint32_t*>(w + o_plan);
    p.list = reinterpret_cast<uint32_t*>(w + o_list);
    p.weights = reinterpret_cast<float*>(w + o_weights);
    p.part = reinterpret_cast<float*>(w + o_part);
    *out = m.release();
    return VX_OK;
}

vx_status vx_moe_free(vx_context* ctx, vx_moe* m) {
    VX_REQUIRE(ctx, VX_ERR_INVALID_ARGUMENT, "vx_moe_free: null context");
    if (!m) return VX_OK;
    VX_REQUIRE(ctx == m->ctx, VX_ERR_INVALID_ARGUMENT, "vx_moe_free: made with another context");
    DeviceGuard guard(ctx->device);
    VX_CUDA(cudaStreamSynchronize(ctx->stream));
    VX_CUDA(cudaFree(m->workspace));
    delete m;
    return VX_OK;
}

vx_status vx_moe_run(vx_context* ctx, const vx_moe* m, const float* x, size_t x_stride, float* y, size_t y_stride, size_t tokens, int32_t* ids,
                     float* weights) {
    VX_REQUIRE(ctx && m, VX_ERR_INVALID_ARGUMENT, "vx_moe_run: null argument");
    VX_REQUIRE(ctx == m->ctx, VX_ERR_INVALID_ARGUMENT, "vx_moe_run: the layer was made with another context");
    if (tokens == 0) return VX_OK;
    VX_REQUIRE(tokens <= m->max_tokens, VX_ERR_INVALID_ARGUMENT, "vx_moe_run: %zu tokens, made for %zu", tokens, m->max_tokens);
    VX_REQUIRE(x && y, VX_ERR_INVALID_ARGUMENT, "vx_moe_run: null x or y");
    MoeParams p = m->p;
    VX_REQUIRE(tokens == 1 || (x_stride >= p.hidden && y_stride >= p.hidden), VX_ERR_INVALID_ARGUMENT,
               "vx_moe_run: rows %zu and %zu elements apart, a row has %u", x_stride, y_stride, p.hidden);
    p.x = x;
    p.y = y;
    p.x_stride = x_stride;
    p.y_stride = y_stride;
    p.tokens = (uint32_t)tokens;
    p.ids_out = ids;
    p.weights_out = weights;
    p.x_vec = ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(p.router)) & 15u) == 0 && (tokens == 1 || x_stride % 4 == 0);
    DeviceGuard guard(ctx->device);
    const uint32_t nbh = p.hidden / 32, jobs = p.experts * ((p.tokens + 3) / 4) + p.tokens * ((nbh + 15) / 16);
    const uint32_t route_grid = std::min((jobs + kMoeWarps - 1) / kMoeWarps, m->sm_count * 4);
    VX_CUDA(launch_pdl(moe_route_kernel, dim3(route_grid), 0, ctx->stream, p));
    // as many units as there can be experts with tokens
    const uint64_t units = (uint64_t)std::min<uint64_t>(p.experts, (uint64_t)p.tokens * p.top_k) * (p.inner / 32);
    const uint32_t grid = (uint32_t)std::min<uint64_t>(units, m->inner_grid);
    if (p.gate4) VX_CUDA(launch_pdl(moe_inner_kernel<true>, dim3(grid), inner_smem<true>(), ctx->stream, p));
    else VX_CUDA(launch_pdl(moe_inner_kernel<false>, dim3(grid), inner_smem<false>(), ctx->stream, p));
    const uint32_t sums = kMoeWarps * p.tokens * 33 * 4;
    const dim3 down_grid(p.hidden / 32, p.splits);
    if (p.down4) VX_CUDA(launch_pdl(moe_down_kernel<true>, down_grid, down_ring<true>() + sums, ctx->stream, p));
    else VX_CUDA(launch_pdl(moe_down_kernel<false>, down_grid, down_ring<false>() + sums, ctx->stream, p));
    ctx->launches += 3;
    return VX_OK;
}

}  // extern "C"
