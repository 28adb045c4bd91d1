// A mixture-of-experts layer for a few tokens on block-quantised weights, in three launches:
//   route   logits = router x, in slices of the columns, and x split into two f16 parts, lifted together per chunk of a gate row
//   inner   silu(gate x) * (up x): four or eight warps per (expert with tokens, 32 inner rows)
//   down    y = sum weight * (down h): a thread block per (32 output rows, share of all experts' columns)
// Every block of the last two picks the experts from the logits itself (2.5 us; less than one block doing it for all would
// cost in waiting), and the down kernel does so, and starts to copy its weights, while the inner kernel still runs.
//
// The weights' bytes are the floor: each is read once per 8 tokens of its expert.  In both products a warp has every
// fourth or eighth chunk of the columns (64 bytes of a gate and an up row, 128 of a down row; codes and scales by
// cp.async copies that run ahead over the ends of units and experts; no synchronisation between warps until the
// sums are added up).  On the tensor cores (m16n8k16) 16 rows of codes are A; B's columns are the two parts of four
// tokens, or eight tokens, whose parts are then multiplied one after the other into the same sums.
// A code becomes its f16 number before it is multiplied (one logic operation or byte permutation and one f16 operation per
// pair).  Taking the bits of code + 8 or + 128 as a subnormal f16 number, and 8 or 128 times the vector's sum off afterwards,
// would save the f16 operation, but its error goes with 128 times the block's largest value, not with the row's own
// products: 1.5e-5 of sum |w||x| beside values 1000 times the others, and 5e-7 of the largest output on even inputs,
// where this form has 3e-7.
// Measured (recorded calls): 8 tokens, 2 of 8 experts of 14336 x 4096, Q4_0 gate and up, Q8_0 down: 197 us (alone: inner 117, 4.0
// TB/s, down 77, 5.7 TB/s); 32 tokens, 4 of 32 experts of 1408 x 2048, Q4_0: 76 us; 7 tokens, 3 of 16 experts of 608 x 1120,
// Q8_0: 18.1 us; one token, 8 of 64 experts of 1024 x 2048, Q4_0: 19.4 us.  The inner kernel reads at 0.61 of the copy rate with 76
// instructions per 32 x 32 weights (36 of them to take the codes apart) at 0.57 a cycle and scheduler: neither issue slots nor
// memory are full.  What it waits for most are the vectors' parts, which each warp reads from the L2 into its registers;
// 128 registers leave four warps a scheduler to hide that, and its Q4_0 forms spill 12 to 60 bytes.
#include <algorithm>
#include <cstddef>
#include <memory>
#include <new>
#include <type_traits>

#include "vx_decode.cuh"

namespace {

using namespace vx;

constexpr uint32_t kMoeWarps = 8, kMoeThreads = kMoeWarps * 32;
constexpr uint32_t kMaxExperts = 256, kMaxTopK = 16, kMaxTokens = 64;
constexpr uint32_t kGroup = 8;              // tokens of an expert per pass over its weights: what fits 128 registers
constexpr uint32_t kStages = 2;             // chunks in flight per warp
constexpr uint32_t kSlice = 512;            // columns of a router row per warp: four 16-byte loads a lane, all in flight

struct Matrix {
    const uint8_t* quants;
    const uint16_t* scales;
};

struct MoeParams {
    const float* x;
    float* y;
    size_t x_stride, y_stride;
    const float* router;
    uint32_t tokens, experts, top_k, hidden, inner, splits, slices;
    uint32_t row_log;    // of the experts, rounded up to a power of two of at least 4
    int normalise, down4, x_vec, gate4;
    Matrix gate, up, down;
    float* logits;       // [slices][tokens][experts]
    uint8_t* xh;         // [tokens][2 parts][hidden / 32][64 bytes], B-operand order
    float* xs;           // [tokens][chunks of a gate row]: what a chunk's sum is multiplied with
    uint8_t* hh;         // the inner vectors, per slot = token * top_k + place
    float* hs;           // [slots][inner / 32]: the same for a block's sum
    int32_t* ids_out;
    float* weights_out;
};

// ------------------------------------------------------------------------------------------------- route ----
// A slice of one expert's row with tokens t0 .. t0 + 3.
__device__ __forceinline__ void logits_of(const MoeParams& p, uint32_t expert, uint32_t t0, uint32_t slice, uint32_t lane) {
    const float* w = p.router + (size_t)expert * p.hidden;
    const uint32_t n = min(4u, p.tokens - t0), from = slice * kSlice, to = min(p.hidden, from + kSlice);
    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (p.x_vec) {
        float4 a[kSlice / 128], b[4][kSlice / 128];  // all asked for before any is used
#pragma unroll
        for (uint32_t k = 0; k < kSlice / 128; ++k) {
            const uint32_t i = from + k * 128 + lane * 4;
            a[k] = i < to ? __ldg(reinterpret_cast<const float4*>(w + i)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (uint32_t t = 0; t < 4; ++t)
                b[t][k] = t < n && i < to ? *reinterpret_cast<const float4*>(p.x + (size_t)(t0 + t) * p.x_stride + i) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
#pragma unroll
        for (uint32_t k = 0; k < kSlice / 128; ++k)
#pragma unroll
            for (uint32_t t = 0; t < 4; ++t)
                sum[t] = fmaf(a[k].x, b[t][k].x, fmaf(a[k].y, b[t][k].y, fmaf(a[k].z, b[t][k].z, fmaf(a[k].w, b[t][k].w, sum[t]))));
    } else {
#pragma unroll 4
        for (uint32_t i = from + lane; i < to; i += 32) {
            const float a = __ldg(w + i);
#pragma unroll
            for (uint32_t t = 0; t < 4; ++t)
                if (t < n) sum[t] = fmaf(a, p.x[(size_t)(t0 + t) * p.x_stride + i], sum[t]);
        }
    }
#pragma unroll
    for (uint32_t t = 0; t < 4; ++t) {
        if (t >= n) break;
        const float s = warp_add(sum[t]);
        if (lane == 0) p.logits[((size_t)slice * p.tokens + t0 + t) * p.experts + expert] = s;
    }
}

// The power of two that values, `most` the largest magnitude, are split with.  f16 ends just below 2^16: values from 2^105 on
// count as infinite.
__device__ __forceinline__ float split_lift(float most) { return fmaxf(lift(most), __uint_as_float((127u - 89u) << 23)); }
__device__ __forceinline__ float split_factor(float up) { return kCodeUnits * __uint_as_float(0x7f000000u - __float_as_uint(up)); }  // over up
// One block of 32 values (a lane each) as two parts in B-operand order.
__device__ __forceinline__ void split_block(float v, float up, uint32_t lane, bool four, uint8_t* hi, uint8_t* lo) {
    const float x = v * up;
    const __half h = __float2half_rn(x), l = __float2half_rn(x - __half2float(h));
    const uint32_t at = frag_lane(lane) * 16 + frag_half(four, lane) * 2;
    *reinterpret_cast<__half*>(hi + at) = h;
    *reinterpret_cast<__half*>(lo + at) = l;
}

__global__ void __launch_bounds__(kMoeThreads) moe_route_kernel(MoeParams p) {
    pdl_wait();
    pdl_launch();
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nb = p.hidden / 32;
    const uint32_t quads = (p.tokens + 3) / 4, dots = p.experts * quads * p.slices, pieces = (nb + 3) / 4;
    for (uint32_t job = blockIdx.x * kMoeWarps + warp; job < dots + p.tokens * pieces; job += gridDim.x * kMoeWarps) {
        if (job < dots) {
            const uint32_t slice = job % p.slices, rest = job / p.slices;
            logits_of(p, rest / quads, (rest % quads) * 4, slice, lane);
        } else {
            const uint32_t t = (job - dots) / pieces, b0 = (job - dots) % pieces * 4;
            float v[4];
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) v[i] = b0 + i < nb ? p.x[(size_t)t * p.x_stride + (b0 + i) * 32 + lane] : 0.0f;
            // a chunk of gate and up (four blocks in Q4_0, two in Q8_0) has one power of two
            const uint32_t each = p.gate4 ? 4 : 2, chunks = (nb + each - 1) / each;
            float m0 = fmaxf(fabsf(v[0]), fabsf(v[1])), m1 = fmaxf(fabsf(v[2]), fabsf(v[3]));
            if (p.gate4) m0 = m1 = fmaxf(m0, m1);
            const float up0 = split_lift(warp_max(m0)), up1 = split_lift(warp_max(m1));
            if (lane == 0) {
                float* factor = p.xs + (size_t)t * chunks + b0 / each;
                factor[0] = split_factor(up0);
                if (!p.gate4 && b0 + 2 < nb) factor[1] = split_factor(up1);
            }
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i)
                if (b0 + i < nb) {
                    uint8_t* hi = p.xh + ((size_t)t * 2 * nb + b0 + i) * 64;
                    split_block(v[i], i < 2 ? up0 : up1, lane, p.gate4 != 0, hi, hi + (size_t)nb * 64);
                }
        }
    }
}

// What every block of the products knows of the routing: the experts that have tokens, and for each the list of its
// slots (token * top_k + place), tokens ascending, and those tokens.
struct Plan {
    uint32_t active;
    uint16_t expert[kMaxExperts], begin[kMaxExperts + 2], list[kMaxTokens * kMaxTopK];
    uint8_t token[kMaxTokens * kMaxTopK];
    float weight[kMaxTokens * kMaxTopK];
};
struct PlanScratch {
    uint32_t tokens[2][kMaxExperts];  // which tokens an expert has
    uint32_t begin[kMaxExperts];      // of the expert's list
    uint16_t chosen[kMaxTokens * kMaxTopK];
    uint32_t scan[kMoeWarps];
    uint4 keys[1];                    // [tokens][experts, rounded up to a power of two]
};
constexpr uint32_t plan_scratch(uint32_t tokens) { return sizeof(PlanScratch) + tokens * kMaxExperts * 4; }

// Numbers as unsigned integers of the same order, NaN below all (0 is below that: no expert).
__device__ __forceinline__ uint32_t order_of(float v) {
    const uint32_t u = __float_as_uint(v);
    return v != v ? 1u : v == 0.0f ? 0x80000000u : u >> 31 ? ~u : u | 0x80000000u;  // -0 and 0 are a tie
}
__device__ __forceinline__ float value_of(uint32_t key) {
    return key == 1u ? NAN : __uint_as_float(key >> 31 ? key & 0x7fffffffu : ~key);
}

// All threads of the block; ends with a barrier.  An expert's place among a token's logits is how many are larger, or
// equal and earlier: a thread per (token, expert) counts, which needs no rounds of finding a largest one.
// WEIGHTS: the softmax as well; `outputs`: it and the experts go to the caller's arrays.
template <bool WEIGHTS>
__device__ __forceinline__ void make_plan(const MoeParams& p, Plan* plan, PlanScratch* w, bool outputs) {
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, row = 1u << p.row_log, quads = row / 4, all = p.tokens << p.row_log;
    uint32_t* keys = reinterpret_cast<uint32_t*>(w->keys);
    w->tokens[0][tid] = w->tokens[1][tid] = 0;
    for (uint32_t i0 = tid; i0 < all; i0 += 4 * kMoeThreads) {
        float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (uint32_t s0 = 0; s0 < p.slices; s0 += 4) {
            float part[4][4];  // sixteen loads in flight
#pragma unroll
            for (uint32_t x = 0; x < 4; ++x) {
                const uint32_t i = i0 + x * kMoeThreads, t = i >> p.row_log, e = i & (row - 1);
                const float* src = p.logits + ((size_t)s0 * p.tokens + t) * p.experts + e;
#pragma unroll
                for (uint32_t y = 0; y < 4; ++y, src += p.tokens * p.experts)
                    part[x][y] = i < all && e < p.experts && s0 + y < p.slices ? __ldcg(src) : 0.0f;
            }
#pragma unroll
            for (uint32_t x = 0; x < 4; ++x)
#pragma unroll
                for (uint32_t y = 0; y < 4; ++y) v[x] += part[x][y];
        }
#pragma unroll
        for (uint32_t x = 0; x < 4; ++x) {
            const uint32_t i = i0 + x * kMoeThreads;
            if (i < all) keys[i] = (i & (row - 1)) < p.experts ? order_of(v[x]) : 0u;
        }
    }
    __syncthreads();
    for (uint32_t i = tid; i < all; i += kMoeThreads) {
        const uint32_t t = i >> p.row_log, e = i & (row - 1), mine = keys[i];
        const uint4* of = w->keys + t * quads;
        uint32_t place = 0;
#pragma unroll 4
        for (uint32_t q = 0; q < quads; ++q) {
            const uint4 k = of[q];
            place += k.x > mine || (k.x == mine && 4 * q < e);
            place += k.y > mine || (k.y == mine && 4 * q + 1 < e);
            place += k.z > mine || (k.z == mine && 4 * q + 2 < e);
            place += k.w > mine || (k.w == mine && 4 * q + 3 < e);
        }
        if (mine && place < p.top_k) {
            w->chosen[t * p.top_k + place] = (uint16_t)e;
            atomicOr(&w->tokens[t >> 5][e], 1u << (t & 31));
            if (outputs && p.ids_out) p.ids_out[(size_t)t * p.top_k + place] = (int32_t)e;
        }
    }
    __syncthreads();
    // a thread per expert: where its list begins, and its place among those that have tokens
    const uint32_t count = __popc(w->tokens[0][tid]) + __popc(w->tokens[1][tid]), both = count | (count ? 0x10000u : 0u);
    uint32_t before = both;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const uint32_t v = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= (uint32_t)o) before += v;
    }
    if (lane == 31) w->scan[warp] = before;
    __syncthreads();
    uint32_t total = 0;
    before -= both;
#pragma unroll
    for (uint32_t i = 0; i < kMoeWarps; ++i) {
        if (i < warp) before += w->scan[i];
        total += w->scan[i];
    }
    w->begin[tid] = before & 0xffffu;
    if (count) {
        plan->expert[before >> 16] = (uint16_t)tid;
        plan->begin[before >> 16] = (uint16_t)before;
    }
    if (tid == 0) {
        plan->active = total >> 16;
        plan->begin[total >> 16] = (uint16_t)total;
    }
    if (WEIGHTS || outputs) {
        for (uint32_t t = warp; t < p.tokens; t += kMoeWarps) {
            const uint32_t* of = keys + (t << p.row_log);
            const float mine = lane < p.top_k ? value_of(of[w->chosen[t * p.top_k + lane]]) : 0.0f;
            const float top = __shfl_sync(0xffffffffu, mine, 0);
            float sum = 0.0f;
            if (p.normalise) {
                sum = lane < p.top_k ? expf(mine - top) : 0.0f;
            } else {
                for (uint32_t e = lane; e < p.experts; e += 32) sum += expf(value_of(of[e]) - top);
            }
            sum = warp_add(sum);
            if (lane < p.top_k) {
                const float f = expf(mine - top) / sum;
                plan->weight[t * p.top_k + lane] = f;
                if (outputs && p.weights_out) p.weights_out[(size_t)t * p.top_k + lane] = f;
            }
        }
    }
    __syncthreads();
    for (uint32_t slot = tid; slot < p.tokens * p.top_k; slot += kMoeThreads) {
        const uint32_t e = w->chosen[slot], t = slot / p.top_k, bits = w->tokens[t >> 5][e] & ((1u << (t & 31)) - 1u);
        const uint32_t at = w->begin[e] + __popc(bits) + (t >= 32 ? __popc(w->tokens[0][e]) : 0);
        plan->list[at] = (uint16_t)slot;
        plan->token[at] = (uint8_t)t;
    }
    __syncthreads();
}

// ---------------------------------------------------------------------------------------------- products ----
// A stage of a warp's ring: 4 KiB of codes, 32 rows of one matrix with 128 bytes each or of two matrices with 64 each
// (their 16-byte units swizzled, so that eight rows meet different banks), then the rows' scales.
template <bool FOUR, int MATS>
struct Chunk {
    static constexpr uint32_t bytes = MATS == 2 ? 64 : 128, units = bytes / 16;
    static constexpr uint32_t blocks = bytes / (FOUR ? 16 : 32);
    __host__ __device__ static uint32_t count(uint32_t nb) { return (nb + blocks - 1) / blocks; }
    __device__ static uint32_t swizzle(uint32_t row) { return (MATS == 2 ? row >> 1 : row) & (units - 1); }
};
constexpr uint32_t kCodes = 4096;

// Copies a chunk of 32 rows; src: the lane's 16 bytes of row lane / units.
template <bool FOUR, int MATS>
__device__ __forceinline__ void fetch_codes(const uint8_t* src, size_t row_bytes, uint32_t dst, uint32_t lane) {
    using C = Chunk<FOUR, MATS>;
    constexpr uint32_t rows = 32 / C::units;  // of a copy
#pragma unroll
    for (uint32_t i = 0; i < C::units; ++i) {
        const uint32_t row = lane / C::units + i * rows;
        cp_async16(dst + row * C::bytes + ((lane % C::units) ^ C::swizzle(row)) * 16, src + i * rows * row_bytes);
    }
}

// A chunk's scales.  WHOLE: a row's blocks are a multiple of the chunk's, so chunks are complete and their scales one
// aligned piece per row.  Else the 4-byte words that hold them; a row of an odd number of blocks may begin in the middle of one.
template <bool FOUR, int MATS, bool WHOLE>
struct Scales {
    static constexpr uint32_t B = Chunk<FOUR, MATS>::blocks, pitch = 2 * B + (WHOLE ? 0 : 4);
    // the lane's row; row: of the matrix, first: the chunk's first block
    __device__ static void fetch(const uint16_t* scales, size_t row, uint32_t first, uint32_t nb, uint32_t dst, uint32_t lane) {
        dst += lane * pitch;
        const size_t at = row * nb + first;
        if (WHOLE) {
            if (B == 8) cp_async16(dst, scales + at);
            else if (B == 4) cp_async8(dst, scales + at);
            else cp_async4(dst, scales + at);
        } else {
            const uint32_t odd = (uint32_t)at & 1u;
#pragma unroll
            for (uint32_t k = 0; k <= B / 2; ++k)
                if (first + 2 * k < nb + odd) cp_async4(dst + 4 * k, scales + (at - odd) + 2 * k);
        }
    }
    // Blocks j0 .. j0 + G - 1 of rows g, g + 8, g + 16, g + 24; `first` as above
    template <uint32_t G>
    struct Of {
        uint32_t pair[4][G / 2];
        __device__ __forceinline__ Of(uint32_t src, uint32_t j0, uint32_t g, uint32_t nb) {
            src += g * pitch + 2 * j0;
#pragma unroll
            for (int i = 0; i < 4; ++i, src += 8 * pitch) {
                if (!WHOLE) {
                    uint32_t w[G / 2 + 1];
#pragma unroll
                    for (uint32_t k = 0; k <= G / 2; ++k) w[k] = lds32(src + 4 * k);
#pragma unroll
                    for (uint32_t k = 0; k < G / 2; ++k) pair[i][k] = __funnelshift_r(w[k], w[k + 1], 16 * (g & nb & 1u));  // 32 rows begin with an even one
                } else if (G == 8) {
                    const uint4 v = lds128(src);
                    pair[i][0] = v.x;
                    pair[i][1] = v.y;
                    pair[i][G / 2 - 2] = v.z;
                    pair[i][G / 2 - 1] = v.w;
                } else if (G == 4) {
                    const uint2 v = lds64(src);
                    pair[i][0] = v.x;
                    pair[i][G / 2 - 1] = v.y;
                } else {
                    pair[i][0] = lds32(src);
                }
            }
        }
        __device__ __forceinline__ float operator()(int row, uint32_t j) const {
            const __half2 d = bits_h2(pair[row][j / 2]);
            return j % 2 ? __high2float(d) : __low2float(d);
        }
    };
};
template <bool FOUR, int MATS, bool WHOLE>
constexpr uint32_t kStage = kCodes + 32 * MATS * Scales<FOUR, MATS, WHOLE>::pitch;  // a multiple of 128
template <bool FOUR, int MATS, bool WHOLE>
constexpr uint32_t kRing = kMoeWarps * kStages * kStage<FOUR, MATS, WHOLE>;

// The vectors of a pass as a lane needs them, NT = 1 for up to four tokens, 2 for up to eight.  B's columns are both parts
// of four tokens, or eight tokens, of which the two parts are multiplied one after the other: a lane has the operand
// of token g / 2, part g % 2, or of token g, both parts, and the results and factors of NT tokens.  Where there is no such
// token, another one's: its results are not used.
template <int NT>
__device__ __forceinline__ uint32_t token_of(uint32_t n, uint32_t t) { return NT == 1 ? t : 2 * t + n; }
template <int NT>
struct Vectors {
    const uint8_t* px[NT];
    const float* pf[NT];
    // nb blocks and nf factors a vector
    template <class Row>
    __device__ __forceinline__ Vectors(const uint8_t* h, const float* f, uint32_t nb, uint32_t nf, const Row* rows, uint32_t count, uint32_t lane) {
        const uint32_t g = lane >> 2, t = lane & 3;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const uint32_t i = min(NT == 1 ? g / 2 : g, count - 1), k = min(token_of<NT>(n, t), count - 1);
            px[n] = h + (size_t)(rows[i] * 2u + (NT == 1 ? g & 1 : n)) * (nb * 64) + t * 16;
            pf[n] = f + (size_t)rows[k] * nf;
        }
    }
    __device__ __forceinline__ void advance(uint32_t blocks, uint32_t factors) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            px[n] += (size_t)blocks * 64;
            pf[n] += factors;
        }
    }
    __device__ __forceinline__ void load(int block, uint4* parts) const {
#pragma unroll
        for (int n = 0; n < NT; ++n) parts[n] = *reinterpret_cast<const uint4*>(px[n] + block * 64);
    }
    __device__ __forceinline__ void load_factor(int at, float* factor) const {
#pragma unroll
        for (int n = 0; n < NT; ++n) factor[n] = pf[n][at];
    }
};
// Blocks of the vectors that are in registers: a chunk's, four at most.  Factors: one for a chunk of two matrices (all its blocks are
// here then), one a block for a chunk of one.
template <bool FOUR, int MATS>
struct Ahead {
    static constexpr uint32_t B = Chunk<FOUR, MATS>::blocks;
    template <int NT>
    static constexpr uint32_t group = std::min(B, NT == 1 || MATS == 2 ? 4u : 2u);
    static constexpr uint32_t size = std::max(group<1>, 2 * group<2>);
    static_assert(MATS == 1 || (group<1> == B && group<2> == B), "a chunk of two matrices is one group");
    uint4 parts[size];
    float factor[MATS == 2 ? 2 : size];
    template <int NT>
    __device__ __forceinline__ void load(const Vectors<NT>& x, int block, uint32_t j) {
        x.load(block, parts + j * NT);
        if (MATS == 1) x.load_factor(block, factor + j * NT);
    }
    // the first blocks of a pass over chunks c0 .. c1 - 1
    template <int NT>
    __device__ __forceinline__ void start(Vectors<NT> x, uint32_t c0, uint32_t c1, uint32_t nb) {
        if (c0 >= c1) return;
        x.advance(c0 * B, MATS == 2 ? c0 : c0 * B);
#pragma unroll
        for (uint32_t j = 0; j < group<NT>; ++j)
            if (c0 * B + j < nb) load<NT>(x, j, j);
        if (MATS == 2) x.load_factor(0, factor);
    }
};

// Products of block j with the two 16-row tiles of 32 rows: use(m, n, h, sum), sum that of row 16 m + 8 h + g, token token_of(n, t).
// codes: where the lane's row begins, its unit swizzled; a stage begins at a multiple of 128 bytes, so the block's number goes into
// the address's bits.
template <bool FOUR, int MATS, int NT, class Use>
__device__ __forceinline__ void multiply(uint32_t codes, uint32_t j, const uint4* parts, Use use) {
    using C = Chunk<FOUR, MATS>;
    uint32_t a[2][2][4];
    if (FOUR) {
        uint32_t w[4];
        ldmatrix_x4(w, codes ^ j * 16);
#pragma unroll
        for (int i = 0; i < 2; ++i) a_of_nibbles(w[2 * i], w[2 * i + 1], a[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            uint32_t w[4];
            ldmatrix_x4(w, (codes ^ j * 32) + i * 16 * C::bytes);
#pragma unroll
            for (int h = 0; h < 4; ++h) w[h] ^= 0x80808080u;  // code + 128
            a_of_bytes(w, a[i]);
        }
    }
    float s[2][4];
    auto both = [&](auto product) {  // neighbouring products do not wait for each other
        product(0);
        product(1);
    };
    if (NT > 1) {
        both([&](int i) { mma_f16_new(s[i], a[i][0], parts[NT - 1].x, parts[NT - 1].y); });
        both([&](int i) { mma_f16(s[i], a[i][1], parts[NT - 1].z, parts[NT - 1].w); });
        both([&](int i) { mma_f16(s[i], a[i][0], parts[0].x, parts[0].y); });
    } else {
        both([&](int i) { mma_f16_new(s[i], a[i][0], parts[0].x, parts[0].y); });
    }
    both([&](int i) { mma_f16(s[i], a[i][1], parts[0].z, parts[0].w); });
    both([&](int i) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int h = 0; h < 2; ++h) use(i, n, h, NT == 1 ? s[i][2 * h] + s[i][2 * h + 1] : s[i][2 * h + n]);
    });
}

// Sums of chunks c0, c0 + TEAM, .. < c1 of 32 rows of each of MATS matrices.  next() waits for the next stage of the ring and
// says where it is, done() gives it back.  `ahead` holds the vectors' first blocks; a block's place is filled with
// the one that comes a group later as soon as it has been used.
template <bool FOUR, bool WHOLE, int MATS, uint32_t TEAM, int NT, class Next, class Done>
__device__ __forceinline__ void dot_chunks(Vectors<NT> x, Ahead<FOUR, MATS>& ahead, uint32_t nb, uint32_t c0, uint32_t c1, uint32_t lane,
                                           Next next, Done done, float (&acc)[MATS][2][NT][2]) {
    using S = Scales<FOUR, MATS, WHOLE>;
    constexpr uint32_t B = Chunk<FOUR, MATS>::blocks, G = Ahead<FOUR, MATS>::template group<NT>;
    using C = Chunk<FOUR, MATS>;
    // where the lane's row begins for ldmatrix, block 0: a row is a tile's of 32 (Q4_0) or of 16, then its second unit (Q8_0)
    const uint32_t lane_row = FOUR ? lane : lane & 15, lane_at = lane_row * C::bytes + ((FOUR ? 0 : lane >> 4) ^ C::swizzle(lane_row)) * 16;
    x.advance(c0 * B, MATS == 2 ? c0 : c0 * B);
#pragma unroll
    for (int a = 0; a < MATS; ++a)
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int n = 0; n < NT; ++n) acc[a][m][n][0] = acc[a][m][n][1] = 0.0f;
    for (uint32_t c = c0; c < c1; c += TEAM) {
        const uint32_t stage = next(), codes = stage + lane_at;
        const bool more = c + TEAM < c1;
#pragma unroll
        for (uint32_t j0 = 0; j0 < B; j0 += G)
#pragma unroll
            for (int a = 0; a < MATS; ++a) {
                const typename S::template Of<G> d(stage + kCodes + a * 32 * S::pitch, j0, lane >> 2, nb);
                float chunk[2][NT][2];  // of two matrices' chunks, whose blocks share a factor
#pragma unroll
                for (uint32_t j = 0; j < G; ++j) {
                    const uint32_t block = c * B + j0 + j;
                    if (WHOLE || block < nb)
                        multiply<FOUR, MATS, NT>(codes + a * (kCodes / 2), j0 + j, ahead.parts + j * NT, [&](int m, int n, int h, float sum) {
                            if (MATS == 1) acc[a][m][n][h] = fmaf(sum * ahead.factor[j * NT + n], d(2 * m + h, j), acc[a][m][n][h]);
                            else chunk[m][n][h] = j == 0 ? sum * d(2 * m + h, j) : fmaf(sum, d(2 * m + h, j), chunk[m][n][h]);
                        });
                    if (a == MATS - 1) {
                        const uint32_t later = j0 + j + (j0 + G < B ? G : TEAM * B + G - B);
                        if ((j0 + G < B || more) && (WHOLE || c * B + later < nb)) ahead.template load<NT>(x, later, j);
                    }
                }
                if (MATS == 2) {
#pragma unroll
                    for (int m = 0; m < 2; ++m)
#pragma unroll
                        for (int n = 0; n < NT; ++n)
#pragma unroll
                            for (int h = 0; h < 2; ++h) acc[a][m][n][h] = fmaf(chunk[m][n][h], ahead.factor[n], acc[a][m][n][h]);
                }
            }
        if (MATS == 2 && more) x.load_factor(TEAM, ahead.factor);
        x.advance(TEAM * B, MATS == 2 ? TEAM : TEAM * B);
        done();
    }
}

// ------------------------------------------------------------------------------------------------- inner ----
constexpr uint32_t kSums4 = 64 * 5;  // floats of a warp; two of them, or one for up to eight tokens
constexpr uint32_t kSums = std::max(2 * kSums4, 64 * (kGroup + 1)), kInnerSums = kMoeWarps * kSums * 4;
template <bool FOUR, bool WHOLE>
constexpr uint32_t kInnerSmem = kRing<FOUR, 2, WHOLE> + kInnerSums + sizeof(Plan);
static_assert(plan_scratch(kMaxTokens) <= kMoeWarps * kStages * kCodes + kInnerSums, "the plan is made where ring and sums are later");

// A pass over a unit's weights: 32 inner rows of an expert, up to kGroup of its tokens.  TEAM warps share its columns;
// team k of all has units k, k + teams, ...
struct InnerPass {
    uint32_t unit, a, at;  // a: expert number in the plan, at: of its list
    __device__ void enter(const Plan* plan, uint32_t tiles, uint32_t units) {
        if (unit >= units) return;
        a = unit / tiles;
        at = plan->begin[a];
    }
    __device__ void next(const Plan* plan, uint32_t tiles, uint32_t units, uint32_t step) {
        at += kGroup;
        if (at < plan->begin[a + 1]) return;
        unit += step;
        enter(plan, tiles, units);
    }
    __device__ uint32_t count(const Plan* plan) const { return plan->begin[a + 1] - at; }
    __device__ uint32_t rows32(uint32_t tiles) const { return unit - a * tiles; }
};

template <bool FOUR, bool WHOLE, uint32_t TEAM>
__global__ void __launch_bounds__(kMoeThreads, 2) moe_inner_kernel(MoeParams p) {
    extern __shared__ __align__(128) uint8_t smem[];
    using C = Chunk<FOUR, 2>;
    using S = Scales<FOUR, 2, WHOLE>;
    constexpr uint32_t kRing = ::kRing<FOUR, 2, WHOLE>, kStage = ::kStage<FOUR, 2, WHOLE>;
    Plan* plan = reinterpret_cast<Plan*>(smem + kRing + kInnerSums);
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    pdl_wait();
    pdl_launch();
    make_plan<false>(p, plan, reinterpret_cast<PlanScratch*>(smem), blockIdx.x == 0);
    const uint32_t nb = p.hidden / 32, chunks = C::count(nb), tiles = p.inner / 32, nbf = tiles, units = plan->active * tiles;
    const uint32_t ring = smem_addr(smem) + warp * kStages * kStage, row_bytes = nb * (FOUR ? 16 : 32);
    const uint32_t team = warp / TEAM, member = warp % TEAM, step = gridDim.x * (kMoeWarps / TEAM);
    float* sums = reinterpret_cast<float*>(smem + kRing) + team * TEAM * kSums;
    auto barrier = [&]() { asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "n"(TEAM * 32) : "memory"); };  // of the team

    // what is copied runs kStages chunks ahead of what is multiplied
    InnerPass ahead;
    ahead.unit = blockIdx.x * (kMoeWarps / TEAM) + team;
    ahead.enter(plan, tiles, units);
    InnerPass now = ahead;
    size_t ahead_row = 0, ahead_at = 0;  // first row, the lane's 16 bytes of the chunk to come
    uint32_t ahead_c = 0, used = 0;
    auto start = [&]() {  // of the pass `ahead`
        ahead_row = (size_t)plan->expert[ahead.a] * p.inner + ahead.rows32(tiles) * 32;
        ahead_at = (ahead_row + lane / C::units) * row_bytes + member * C::bytes + lane % C::units * 16;
        ahead_c = member;
    };
    if (ahead.unit < units) start();
    auto fetch = [&](uint32_t stage) {
        if (ahead_c >= chunks && member < chunks && ahead.unit < units) {
            ahead.next(plan, tiles, units, step);
            if (ahead.unit < units) start();
        }
        if (ahead_c < chunks && ahead.unit < units) {
            if (WHOLE || ahead_c * C::bytes + lane % C::units * 16 < row_bytes) {
                fetch_codes<FOUR, 2>(p.gate.quants + ahead_at, row_bytes, stage, lane);
                fetch_codes<FOUR, 2>(p.up.quants + ahead_at, row_bytes, stage + kCodes / 2, lane);
            }
            S::fetch(p.gate.scales, ahead_row + lane, ahead_c * C::blocks, nb, stage + kCodes, lane);
            S::fetch(p.up.scales, ahead_row + lane, ahead_c * C::blocks, nb, stage + kCodes + 32 * S::pitch, lane);
            ahead_at += TEAM * C::bytes;
            ahead_c += TEAM;
        }
        cp_async_commit();
    };
#pragma unroll
    for (uint32_t k = 0; k < kStages; ++k) fetch(ring + k * kStage);

    // Four tokens' sums are added up in two places in turn, with one barrier a pass; more tokens' use both, with three.
    uint32_t turn = 0;
    Ahead<FOUR, 2> vectors;
    auto begin = [&](auto groups) {
        constexpr int NT = decltype(groups)::value;
        return Vectors<NT>(p.xh, p.xs, nb, chunks, plan->token + now.at, min(kGroup, now.count(plan)), lane);
    };
    auto begin_ahead = [&]() {
        if (now.unit >= units) return;
        if (now.count(plan) <= 4) vectors.start(begin(std::integral_constant<int, 1>()), member, chunks, nb);
        else vectors.start(begin(std::integral_constant<int, 2>()), member, chunks, nb);
    };
    begin_ahead();
    while (now.unit < units) {
        const uint32_t count = min(kGroup, now.count(plan)), rows32 = now.rows32(tiles);
        const uint16_t* slots = plan->list + now.at;
        auto next = [&]() {
            cp_async_wait<kStages - 1>();
            __syncwarp();
            return ring + (used % kStages) * kStage;
        };
        auto done = [&]() {
            __syncwarp();
            fetch(ring + (used % kStages) * kStage);
            ++used;
        };
        auto pass = [&](auto groups) {
            constexpr int NT = decltype(groups)::value;
            float acc[2][2][NT][2];
            const Vectors<NT> x = begin(groups);
            dot_chunks<FOUR, WHOLE, 2, TEAM, NT>(x, vectors, nb, member, chunks, lane, next, done, acc);
            now.next(plan, tiles, units, step);
            begin_ahead();
            // the team's sums: gate rows 0..31, up rows 32..63
            constexpr uint32_t W = 4 * NT + 1;
            if (NT > 1) barrier();
            float* to = sums + (NT > 1 ? 0 : turn * TEAM * kSums4);
#pragma unroll
            for (int a = 0; a < 2; ++a)
#pragma unroll
                for (int m = 0; m < 2; ++m)
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int h = 0; h < 2; ++h) to[(member * 64 + a * 32 + m * 16 + h * 8 + g) * W + token_of<NT>(n, t)] = acc[a][m][n][h];
            barrier();
            for (uint32_t i = member; i < count; i += TEAM) {
                float a = 0.0f, b = 0.0f;
#pragma unroll
                for (uint32_t w = 0; w < TEAM; ++w) {
                    a += to[(w * 64 + lane) * W + i];
                    b += to[(w * 64 + 32 + lane) * W + i];
                }
                const float h = a / (1.0f + expf(-a)) * b;
                const uint32_t slot = slots[i];
                uint8_t* hi = p.hh + ((size_t)slot * 2 * nbf + rows32) * 64;
                const float up = split_lift(warp_max(fabsf(h)));
                split_block(h, up, lane, p.down4 != 0, hi, hi + (size_t)nbf * 64);
                if (lane == 0) p.hs[(size_t)slot * nbf + rows32] = split_factor(up);
            }
            if (NT > 1) barrier();
            turn ^= 1;
        };
        if (count <= 4) pass(std::integral_constant<int, 1>());
        else pass(std::integral_constant<int, 2>());
    }
    cp_async_wait<0>();
}

// -------------------------------------------------------------------------------------------------- down ----
// Shared memory: the ring, [warps][tokens][33] sums, as much of the plan as the tokens need.
constexpr uint32_t down_sums(uint32_t tokens) { return kMoeWarps * tokens * 33 * 4; }
template <bool FOUR, bool WHOLE>
constexpr uint32_t down_smem(uint32_t tokens, uint32_t slots) {
    return kRing<FOUR, 1, WHOLE> + down_sums(tokens) + (uint32_t)offsetof(Plan, weight) + slots * 4;
}
static_assert(plan_scratch(48) <= kMoeWarps * kStages * kCodes && plan_scratch(kMaxTokens) <= kMoeWarps * kStages * kCodes + down_sums(49),
              "the plan is made where ring and sums are later");

// A warp's way through the block's share of all experts' chunks, counted through: chunk `warp` of every eight, and
// for each expert a pass per kGroup tokens.
struct DownPass {
    uint32_t a, at, c, c1;  // expert number in the plan, its tokens from `at` on, chunks c, c + 8, .. < c1
    uint32_t c0;
    // enters expert a or the next one that has a chunk for this warp
    __device__ void enter(const Plan* plan, uint32_t chunks, uint32_t lo, uint32_t hi, uint32_t warp) {
        for (; a < plan->active && a * chunks < hi; ++a) {
            const uint32_t first = a * chunks, from = max(lo, first);
            c1 = min(hi, first + chunks) - first;
            c0 = from + (warp + kMoeWarps - (from - lo) % kMoeWarps) % kMoeWarps - first;
            if (c0 < c1) {
                at = plan->begin[a];
                c = c0;
                return;
            }
        }
        a = kMaxExperts;
    }
    __device__ bool valid() const { return a < kMaxExperts; }
    // on to the next pass over this expert's chunks, or to the next expert
    __device__ void next_pass(const Plan* plan, uint32_t chunks, uint32_t lo, uint32_t hi, uint32_t warp) {
        at += kGroup;
        if (at < plan->begin[a + 1]) {
            c = c0;
        } else {
            ++a;
            enter(plan, chunks, lo, hi, warp);
        }
    }
};

constexpr uint32_t kMaxSplits = 4;  // blocks of a cluster; eight did not all find room at once (19 against 12 us)

__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The float at shared-memory address `at` of block `rank` of the cluster.
__device__ __forceinline__ float cluster_load(uint32_t at, uint32_t rank) {
    uint32_t there;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(at), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(there) : "memory");
    return v;
}

template <bool FOUR, bool WHOLE>
__global__ void __launch_bounds__(kMoeThreads, 2) moe_down_kernel(MoeParams p) {
    extern __shared__ __align__(128) uint8_t smem[];
    using C = Chunk<FOUR, 1>;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    constexpr uint32_t kRing = ::kRing<FOUR, 1, WHOLE>, kStage = ::kStage<FOUR, 1, WHOLE>;
    Plan* plan = reinterpret_cast<Plan*>(smem + kRing + down_sums(p.tokens));
    float* sums = reinterpret_cast<float*>(smem + kRing);  // [warps][tokens][33]
    float* mine = sums + warp * p.tokens * 33;
    // The logits are the route kernel's, which had ended before any block of the inner kernel let this one start.
    make_plan<true>(p, plan, reinterpret_cast<PlanScratch*>(smem), false);
    for (uint32_t i = lane; i < p.tokens * 33; i += 32) mine[i] = 0.0f;
    __syncwarp();
    const uint32_t tile = blockIdx.x, split = blockIdx.y;
    const uint32_t nb = p.inner / 32, chunks = C::count(nb), row_bytes = nb * (FOUR ? 16 : 32);
    const uint64_t all = (uint64_t)plan->active * chunks;
    const uint32_t lo = (uint32_t)(all * split / p.splits), hi = (uint32_t)(all * (split + 1) / p.splits);
    const uint32_t ring = smem_addr(smem) + warp * kStages * kStage;

    DownPass ahead;
    ahead.a = lo / chunks;
    ahead.enter(plan, chunks, lo, hi, warp);
    DownPass now = ahead;
    size_t ahead_row = 0, ahead_at = 0;  // first row, the lane's 16 bytes of the chunk to come
    uint32_t used = 0;
    auto start = [&]() {
        if (!ahead.valid()) return;
        ahead_row = (size_t)plan->expert[ahead.a] * p.hidden + tile * 32;
        ahead_at = (ahead_row + lane / C::units) * row_bytes + ahead.c * C::bytes + lane % C::units * 16;
    };
    start();
    auto fetch = [&](uint32_t stage) {
        if (ahead.valid()) {
            if (WHOLE || ahead.c * C::bytes + lane % C::units * 16 < row_bytes)
                fetch_codes<FOUR, 1>(p.down.quants + ahead_at, row_bytes, stage, lane);
            Scales<FOUR, 1, WHOLE>::fetch(p.down.scales, ahead_row + lane, ahead.c * C::blocks, nb, stage + kCodes, lane);
            ahead_at += kMoeWarps * C::bytes;
            ahead.c += kMoeWarps;
            if (ahead.c >= ahead.c1) {
                ahead.next_pass(plan, chunks, lo, hi, warp);
                start();
            }
        }
        cp_async_commit();
    };
#pragma unroll
    for (uint32_t k = 0; k < kStages; ++k) fetch(ring + k * kStage);
    pdl_wait();  // for the inner vectors
    pdl_launch();
    Ahead<FOUR, 1> vectors;
    auto begin = [&](auto groups) {
        constexpr int NT = decltype(groups)::value;
        return Vectors<NT>(p.hh, p.hs, nb, nb, plan->list + now.at, min(kGroup, plan->begin[now.a + 1] - now.at), lane);
    };
    auto begin_ahead = [&]() {
        if (!now.valid()) return;
        if (plan->begin[now.a + 1] - now.at <= 4) vectors.start(begin(std::integral_constant<int, 1>()), now.c0, now.c1, nb);
        else vectors.start(begin(std::integral_constant<int, 2>()), now.c0, now.c1, nb);
    };
    begin_ahead();
    while (now.valid()) {
        const uint32_t count = min(kGroup, plan->begin[now.a + 1] - now.at);
        const uint16_t* slots = plan->list + now.at;
        auto next = [&]() {
            cp_async_wait<kStages - 1>();
            __syncwarp();
            return ring + (used % kStages) * kStage;
        };
        auto done = [&]() {
            __syncwarp();
            fetch(ring + (used % kStages) * kStage);
            ++used;
        };
        auto pass = [&](auto groups) {
            constexpr int NT = decltype(groups)::value;
            float acc[1][2][NT][2];
            const Vectors<NT> x = begin(groups);
            dot_chunks<FOUR, WHOLE, 1, kMoeWarps, NT>(x, vectors, nb, now.c0, now.c1, lane, next, done, acc);
            now.next_pass(plan, chunks, lo, hi, warp);
            begin_ahead();
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const uint32_t i = token_of<NT>(n, t);
                if (i < count) {
                    const uint32_t slot = slots[i];
                    const float w = plan->weight[slot];
                    float* to = mine + (slot / p.top_k) * 33;
#pragma unroll
                    for (int m = 0; m < 2; ++m)
#pragma unroll
                        for (int h = 0; h < 2; ++h) to[m * 16 + h * 8 + g] = fmaf(w, acc[0][m][n][h], to[m * 16 + h * 8 + g]);
                }
            }
            __syncwarp();
        };
        if (count <= 4) pass(std::integral_constant<int, 1>());
        else pass(std::integral_constant<int, 2>());
    }
    cp_async_wait<0>();
    __syncthreads();
    // The warps' sums, then the cluster's: its blocks have a share of the columns each, of the same rows.
    for (uint32_t k = warp; k < p.tokens; k += kMoeWarps) {
        float s = 0.0f;
#pragma unroll
        for (uint32_t w = 0; w < kMoeWarps; ++w) s += sums[(w * p.tokens + k) * 33 + lane];
        if (p.splits == 1) p.y[(size_t)k * p.y_stride + tile * 32 + lane] = s;
        else sums[k * 33 + lane] = s;  // row k of warp 0, which only this warp reads
    }
    if (p.splits == 1) return;
    cluster_barrier();
    for (uint32_t k = split * kMoeWarps + warp; k < p.tokens; k += p.splits * kMoeWarps) {
        const uint32_t at = smem_addr(sums + k * 33 + lane);
        float part[kMaxSplits], s = 0.0f;
#pragma unroll
        for (uint32_t i = 0; i < kMaxSplits; ++i) part[i] = i < p.splits ? cluster_load(at, i) : 0.0f;
#pragma unroll
        for (uint32_t i = 0; i < kMaxSplits; ++i) s += part[i];
        p.y[(size_t)k * p.y_stride + tile * 32 + lane] = s;
    }
    cluster_barrier();  // nobody leaves while its sums are being read
}

// The kernels for a matrix: its type, and whether its rows are whole chunks.
using MoeKernel = void (*)(MoeParams);
struct Launch {
    MoeKernel kernel;
    uint32_t smem;
};
template <bool FOUR, bool WHOLE>
Launch inner_of(uint32_t team) {
    return {team == 8 ? moe_inner_kernel<FOUR, WHOLE, 8> : moe_inner_kernel<FOUR, WHOLE, 4>, kInnerSmem<FOUR, WHOLE>};
}
template <bool FOUR>
Launch inner_of(uint32_t nb, uint32_t team) {
    return nb % Chunk<FOUR, 2>::blocks == 0 ? inner_of<FOUR, true>(team) : inner_of<FOUR, false>(team);
}
template <bool FOUR>
Launch down_of(uint32_t nb, uint32_t tokens, uint32_t slots) {
    if (nb % Chunk<FOUR, 1>::blocks == 0) return {moe_down_kernel<FOUR, true>, down_smem<FOUR, true>(tokens, slots)};
    return {moe_down_kernel<FOUR, false>, down_smem<FOUR, false>(tokens, slots)};
}
Launch inner_launch(const MoeParams& p, uint32_t team) {
    return p.gate4 ? inner_of<true>(p.hidden / 32, team) : inner_of<false>(p.hidden / 32, team);
}
Launch down_launch(const MoeParams& p, uint32_t tokens) {
    return p.down4 ? down_of<true>(p.inner / 32, tokens, tokens * p.top_k) : down_of<false>(p.inner / 32, tokens, tokens * p.top_k);
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
    p.splits = std::min(kMaxSplits, std::max(1u, 2 * m->sm_count / tiles));
    p.slices = (p.hidden + kSlice - 1) / kSlice;
    p.row_log = 2;
    while ((1u << p.row_log) < p.experts) ++p.row_log;
    int per_sm = 0;
    cudaFuncAttributes loaded;  // all kernels' code is loaded now, so that the first call may be one that is being recorded
    VX_CUDA(cudaFuncGetAttributes(&loaded, moe_route_kernel));
    for (uint32_t team : {4u, 8u}) {
        const Launch inner = inner_launch(p, team);
        VX_CUDA(cudaFuncSetAttribute(inner.kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)inner.smem));
        VX_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, inner.kernel, kMoeThreads, inner.smem));
    }
    m->inner_grid = (uint32_t)std::max(1, per_sm) * m->sm_count;
    // for every layer of these types, so the most that any needs
    MoeParams most = p;
    most.top_k = kMaxTopK;
    const Launch down_k = down_launch(most, kMaxTokens);
    VX_CUDA(cudaFuncSetAttribute(down_k.kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)down_k.smem));
    // ---- workspace ------------------------------------------------------------------------------------------------------
    const size_t slots = max_tokens * top_k, nbh = hidden / 32, nbf = inner / 32;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t o = at;
        at += round_up(bytes, 256);
        return o;
    };
    const size_t o_logits = take(p.slices * max_tokens * experts * 4), o_xh = take(max_tokens * 2 * nbh * 64), o_xs = take(max_tokens * nbh * 4),
                 o_hh = take(slots * 2 * nbf * 64), o_hs = take(slots * nbf * 4);
    const cudaError_t e = device_malloc(ctx, reinterpret_cast<void**>(&m->workspace), at);
    if (e != cudaSuccess) {
        (void)cudaGetLastError();
        return fail(VX_ERR_OUT_OF_MEMORY, "allocating %zu bytes of expert-layer workspace failed: %s", at, cudaGetErrorString(e));
    }
    uint8_t* w = m->workspace;
    p.logits = reinterpret_cast<float*>(w + o_logits);
    p.xh = w + o_xh;
    p.xs = reinterpret_cast<float*>(w + o_xs);
    p.hh = w + o_hh;
    p.hs = reinterpret_cast<float*>(w + o_hs);
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
    const uint32_t jobs = p.experts * ((p.tokens + 3) / 4) * p.slices + p.tokens * ((p.hidden / 32 + 3) / 4);
    const uint32_t route_grid = std::min((jobs + kMoeWarps - 1) / kMoeWarps, m->sm_count * 8);
    VX_CUDA(launch_after(moe_route_kernel, dim3(route_grid), kMoeThreads, 0, ctx->stream, p));
    // as many units as there can be experts with tokens
    const uint64_t units = (uint64_t)std::min<uint64_t>(p.experts, (uint64_t)p.tokens * p.top_k) * (p.inner / 32);
    // Eight warps share a unit's columns, or four do and a block has two units at a time: whichever takes fewer chunks one after the
    // other (8 experts of 8192 x 512, two tokens: 20 us with four, 26 with eight; 8 of 14336 x 4096, 8 tokens: 219 and 205).
    const uint32_t chunks = p.gate4 ? Chunk<true, 2>::count(p.hidden / 32) : Chunk<false, 2>::count(p.hidden / 32);
    auto turns = [&](uint32_t team) {
        const uint64_t at_once = (uint64_t)m->inner_grid * (kMoeWarps / team);
        return (units + at_once - 1) / at_once * ((chunks + team - 1) / team);
    };
    const uint32_t team = turns(4) < turns(8) ? 4 : 8, teams = kMoeWarps / team;
    const uint32_t grid = (uint32_t)std::min<uint64_t>((units + teams - 1) / teams, m->inner_grid);
    const Launch inner = inner_launch(p, team), down = down_launch(p, p.tokens);
    VX_CUDA(launch_after(inner.kernel, dim3(grid), kMoeThreads, inner.smem, ctx->stream, p));
    VX_CUDA(launch_after(down.kernel, dim3(p.hidden / 32, p.splits), kMoeThreads, down.smem, ctx->stream, p, dim3(1, p.splits)));
    ctx->launches += 3;
    return VX_OK;
}

}  // extern "C"
