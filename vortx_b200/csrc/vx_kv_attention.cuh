// Attention of a call's rows over the quantised cache: the kernel, included by the files that instantiate it for a
// pair of types (vx_kv_attention_*.cu), and what its host side needs to know.
//
// S^T = K Q^T and O^T = V^T P^T: the codes are the A operand (16 tokens or 16 values of the head high), the query rows are the
// 8-wide N dimension, so the few rows of a decode step (query heads that share a head of keys, times drafted tokens)
// fill the tensor cores' tiles.  A thread block has a head of a sequence, 4 (NT 0), 8 or 16 query rows and a run of 32-token
// tiles; its four or six warps take the tiles in turn, each with its own running maximum, sum and output (one pass over the
// cache, no synchronisation between tiles), two tiles in flight per warp (cp.async, a record is contiguous).
//   scores   per block of 32 values: sum of code * (q hi + q lo) on the tensor cores, times the block's scale, in f32
//   softmax  base 2 (log2 e is multiplied into q), running maximum per row, weights p <= 1
//   output   the value blocks' scales d are per token, so they go into the weights.  With 2^e the power of two below a
//            token's largest |d|, p 2^e is lifted so that the row's largest of the tile lies in [2^12, 2^13) and split into
//            two f16 parts, once per tile; the f16 scales become d 2^(1 - e), in [2, 4) for the largest; and the two parts of
//            the product, hi = p hi * d and lo = p lo * d + (p hi * d - hi), are three f16 operations per pair of
//            tokens and block (the difference is exact).  A token of no weight, however large, costs the others nothing.
//            That holds while a token's scales are within 2^14 of its largest, so that none becomes a small number of
//            f16; where a token with weight has a smaller one (or zeros in a block where others have more), p d is
//            taken in f32, lifted per row and block, and split (see `wide`)
// The runs are shares of all tiles of all (sequence, head, group of rows), see Share.  A share that covers the tiles of a
// (sequence, head, rows) only in part leaves maximum, sum and unnormalised output in the workspace, at most two per block,
// and the last block to finish a part joins them all, in their order.
// Measured (recorded), 32 heads over 8 of 128 in Q8_0: a token each of 16 sequences of up to 16384 tokens 73 us (392 MB at 5.4 TB/s,
// 0.82 of the copy rate), of one of 500 9.2 us; 4 x 8 drafted tokens over 4000 30 us, 2 x 48 over 12000 149 us; one token
// of 16 heads of 64 over 60001 in Q4_0 30 us (537 instructions a tile of 32 tokens; 16 warps of 128 registers were no faster).
// With many rows the products take 0.4 of what the tensor cores could do: the chain scores -> maximum -> weights ->
// output binds (0.5 instructions a cycle and scheduler with 8 warps of 255 registers as with 12 of 168).
// Looking for scales that f16 cannot hold costs 0 to 2 %, and 3 % where most tiles are a sequence's last; having them in every tile
// 10 to 45 %.
#pragma once

#include <type_traits>

#include "vx_decode.cuh"

namespace vx {

// Tiles per block below which fewer blocks work: one per warp (500 tokens, 8 heads of keys: 10.7 us, with two or four 13).
constexpr uint32_t kAttnMinTiles = 4;
// Items of so many tiles at most are not split, if there are blocks for all: two tiles of a warp one after the other cost less
// than joining two parts (250 tokens: 8.9 us, split 10.8).
constexpr uint32_t kAttnWhole = 8;
constexpr uint32_t kAttnJoin = 32;       // parts whose weights are in shared memory at a time

struct AttnParams {
    KvGeometry g;
    KvRows r;
    const float* q;
    float* out;
    size_t q_stride, out_stride;
    uint32_t group;          // query heads of one head of keys
    float scale_log2;        // scale * log2 e
    const uint32_t* mask;
    uint32_t mask_words;
    float* part_o;           // [2 * grid][rows of an item][D]
    float2* part_ml;         // [2 * grid][rows of an item] maximum (base 2), sum
    uint32_t* counters;      // [grid] parts that are done, of what begins in this block; zero between calls
};

// The (head, group of rows) of a sequence, and its tiles.
__device__ __forceinline__ uint64_t seq_items(const KvSeq& q, const KvGeometry& g, uint32_t group, uint32_t rows_per_item) {
    return (uint64_t)g.heads * (((uint64_t)q.n * group + rows_per_item - 1) / rows_per_item);
}
__device__ __forceinline__ uint32_t seq_tiles_of(const KvSeq& q, uint32_t tokens) { return (q.end + tokens - 1) / tokens; }
// a / b; most often both fit 32 bits, and a 64-bit division is a call.
__device__ __forceinline__ uint64_t quotient(uint64_t a, uint64_t b) {
    return ((a | b) >> 32) == 0 ? (uint32_t)a / (uint32_t)b : a / b;
}
// Shares of `total` tiles: the first `more` blocks have `each` + 1, the others `each`.
struct Shares {
    uint64_t each, more;
    __device__ Shares(uint64_t total, uint64_t blocks) : each(quotient(total, blocks)), more(total - each * blocks) {}
    __device__ uint64_t begin(uint64_t block) const { return block * each + (block < more ? block : more); }
    __device__ uint32_t block_of(uint64_t tile) const {  // every block has a tile
        const uint64_t large = more * (each + 1);
        return (uint32_t)(tile < large ? quotient(tile, each + 1) : more + quotient(tile - large, each));
    }
};

// A block's share: of units of `step` tiles of an item (sequence, head, group of rows).  One unit per block where that
// leaves the blocks nearly equal (few items next to the grid), else the same number of tiles, whichever items they are
// of.
struct Share {
    uint32_t seq = 0, step = 1;
    uint64_t pos = 0, hi = 0;  // units of the sequence: where the block is, where its share ends
    uint64_t origin = 0;       // units before the sequence
    Shares shares;
    __device__ explicit Share(const AttnParams&) : shares(0, 1) {}

    // All threads of the block (W warps); items have R rows, tiles TT tokens.  False: nothing to do.
    template <uint32_t R, uint32_t W, uint32_t TT>
    __device__ __forceinline__ bool find(const AttnParams& p, uint64_t* shared64) {
        const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
        auto tiles_of = [&](uint32_t s, uint64_t* items) {
            const KvSeq q = kv_seq(p.r, p.g, s);
            *items = seq_items(q, p.g, p.group, R);
            return seq_tiles_of(q, TT);
        };
        auto choose_step = [&](uint64_t tiles, uint64_t items, uint32_t most) {
            if (most <= kAttnWhole && items <= gridDim.x) {
                step = kAttnWhole;
                return;
            }
            const uint64_t even = quotient(tiles + gridDim.x - 1, gridDim.x);
            const uint64_t apart = items < gridDim.x ? quotient(tiles, gridDim.x - items) + 1 : ~0ull;  // sum ceil(tiles / apart) <= grid
            if (apart <= even + even / 4 + kAttnMinTiles) step = max((uint32_t)apart, kAttnMinTiles);
        };
        // blocks that have a share of `total` units; false for the others
        auto choose_shares = [&](uint64_t total) {
            uint64_t blocks = step > 1 ? total : quotient(total + kAttnMinTiles - 1, kAttnMinTiles);
            if (blocks > gridDim.x) blocks = gridDim.x;
            if (blockIdx.x >= blocks) return false;
            shares = Shares(total, blocks);
            return true;
        };
        // Up to 32 sequences: a lane each, every warp for itself.
        uint64_t my_items = 0;
        const uint32_t my_tiles = p.r.seqs <= 32 && lane < p.r.seqs ? tiles_of(lane, &my_items) : 0;
        if (p.r.seqs <= 32 && !__any_sync(0xffffffffu, my_items * my_tiles >> 26)) {
            const uint32_t tiles = __reduce_add_sync(0xffffffffu, (uint32_t)my_items * my_tiles);
            if (tiles == 0) return false;
            choose_step(tiles, __reduce_add_sync(0xffffffffu, my_tiles ? (uint32_t)my_items : 0u), __reduce_max_sync(0xffffffffu, my_items ? my_tiles : 0u));
            const uint32_t mine = (uint32_t)my_items * ((my_tiles + step - 1) / step);
            uint32_t upto = mine;
#pragma unroll
            for (int o = 1; o < 32; o *= 2) {
                const uint32_t v = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= (uint32_t)o) upto += v;
            }
            if (!choose_shares(__shfl_sync(0xffffffffu, upto, 31))) return false;
            const uint32_t lo = (uint32_t)shares.begin(blockIdx.x);
            seq = __ffs(__ballot_sync(0xffffffffu, lo < upto)) - 1;
            origin = __shfl_sync(0xffffffffu, upto - mine, seq);
            pos = lo - origin;
            hi = shares.begin(blockIdx.x + 1) - origin;
        } else {
            const uint32_t per = (p.r.seqs + W * 32 - 1) / (W * 32);
            const uint32_t s0 = min(p.r.seqs, tid * per), s1 = min(p.r.seqs, s0 + per);
            uint64_t tiles = 0, items = 0;
            for (uint32_t s = s0; s < s1; ++s) {
                uint64_t i;
                const uint32_t t_ = tiles_of(s, &i);
                if (t_) items += i;
                tiles += i * t_;
            }
#pragma unroll
            for (int o = 16; o > 0; o /= 2) {
                tiles += __shfl_xor_sync(0xffffffffu, tiles, o);
                items += __shfl_xor_sync(0xffffffffu, items, o);
            }
            if (lane == 0) {
                shared64[warp] = tiles;
                shared64[W + warp] = items;
            }
            __syncthreads();
            tiles = items = 0;
#pragma unroll
            for (uint32_t w = 0; w < W; ++w) {
                tiles += shared64[w];
                items += shared64[W + w];
            }
            if (tiles == 0) return false;
            choose_step(tiles, items, ~0u);  // with so many sequences, items seldom have a block each
            auto units_of = [&](uint32_t s) {
                uint64_t i;
                const uint32_t t_ = tiles_of(s, &i);
                return i * ((t_ + step - 1) / step);
            };
            uint64_t mine = 0;
            for (uint32_t s = s0; s < s1; ++s) mine += units_of(s);
            uint64_t before = mine;
#pragma unroll
            for (int o = 1; o < 32; o *= 2) {
                const uint64_t v = __shfl_up_sync(0xffffffffu, before, o);
                if (lane >= (uint32_t)o) before += v;
            }
            __syncthreads();
            if (lane == 31) shared64[warp] = before;
            __syncthreads();
            uint64_t total = 0;
            before -= mine;
            for (uint32_t w = 0; w < W; ++w) {
                if (w < warp) before += shared64[w];
                total += shared64[w];
            }
            if (!choose_shares(total)) return false;
            const uint64_t lo = shares.begin(blockIdx.x);
            hi = shares.begin(blockIdx.x + 1);
            __syncthreads();
            if (before <= lo && lo < before + mine) {  // one thread of the block
                uint64_t at = before;
                uint32_t s = s0;
                for (;; ++s) {
                    const uint64_t w = units_of(s);
                    if (lo < at + w) break;
                    at += w;
                }
                shared64[0] = s;
                shared64[1] = at;
            }
            __syncthreads();
            seq = (uint32_t)shared64[0];
            origin = shared64[1];
            pos = lo - origin;
            hi -= origin;
        }
        return true;
    }
};

// What a block does next: tiles [tile0, tile1) of a head of a sequence for R rows from row_first on.
struct Segment {
    KvSeq sq;
    uint32_t seq, head, row_first, row_count, tile0, tile1, seq_tiles, parts, c0, slot;
    bool whole;  // else one of `parts` parts, of blocks c0 ..
};
template <uint32_t R, uint32_t TT>
__device__ __forceinline__ bool next_segment(const AttnParams& p, Share& at, Segment& s) {
    while (at.pos < at.hi) {
        s.sq = kv_seq(p.r, p.g, at.seq);
        s.seq_tiles = seq_tiles_of(s.sq, TT);
        const uint32_t units = (s.seq_tiles + at.step - 1) / at.step;
        const uint64_t work = seq_items(s.sq, p.g, p.group, R) * units;
        if (at.pos >= work) {  // on to the next sequence
            at.pos -= work;
            at.hi -= work;
            at.origin += work;
            ++at.seq;
            continue;
        }
        s.seq = at.seq;
        const uint32_t groups = (uint32_t)(((uint64_t)s.sq.n * p.group + R - 1) / R);
        const uint32_t item = (uint32_t)quotient(at.pos, units), unit0 = (uint32_t)(at.pos - (uint64_t)item * units);
        s.head = item / groups;
        s.row_first = (item - s.head * groups) * R;
        s.row_count = min(R, s.sq.n * p.group - s.row_first);
        const uint32_t count = at.hi - at.pos < units - unit0 ? (uint32_t)(at.hi - at.pos) : units - unit0;
        s.tile0 = unit0 * at.step;
        s.tile1 = min(s.seq_tiles, (unit0 + count) * at.step);
        s.whole = count == units;
        s.slot = blockIdx.x * 2 + (unit0 == 0 ? 1 : 0);
        s.parts = 1;
        s.c0 = 0;
        if (!s.whole) {  // the first block's second slot, the others' first
            const uint64_t first = at.origin + (uint64_t)item * units;
            s.c0 = at.shares.block_of(first);
            s.parts = at.shares.block_of(first + units - 1) - s.c0 + 1;
        }
        at.pos += count;
        return true;
    }
    return false;
}

// Four neighbouring values of a row of the result.
__device__ __forceinline__ void put_row(const AttnParams& p, const Segment& s, uint32_t dim, uint32_t row, uint32_t col, float4 o, float n) {
    const uint32_t rr = s.row_first + row, i = rr / p.group;
    float* dst = p.out + (size_t)(s.sq.row0 + i) * p.out_stride + (size_t)(s.head * p.group + (rr - i * p.group)) * dim + col;
    dst[0] = o.x * n;
    dst[1] = o.y * n;
    dst[2] = o.z * n;
    dst[3] = o.w * n;
}
// A part that saw nothing is zeros, and NaN where a NaN was seen; neither is weighted.
__device__ __forceinline__ float part_weight(float m, float most) { return m == -INFINITY ? 1.0f : ex2(m - most); }

// The last block of a split (sequence, head, rows) joins the parts, in their order.  of_row: R pairs, weights: kAttnJoin R
// floats of shared memory.
template <uint32_t R, uint32_t DIM, uint32_t THREADS>
__device__ __forceinline__ void join_parts(const AttnParams& p, const Segment& s, float2* of_row, float* weights) {
    const uint32_t tid = threadIdx.x;
    auto slot_of = [&](uint32_t c) { return (size_t)(s.c0 + c) * 2 + (c == 0 ? 1 : 0); };
    constexpr uint32_t kLanes = 128 / R;  // that share a row: neighbours of the first four warps
    if (tid < 128) {
        const uint32_t row = tid / kLanes, at = tid % kLanes;
        float m = -INFINITY, l = 0.0f;
#pragma unroll 4
        for (uint32_t c = at; c < s.parts; c += kLanes) {
            const float2 f = __ldcg(&p.part_ml[slot_of(c) * R + row]);
            const float now = fmaxf(m, f.x);
            l = (m == -INFINITY ? l : l * ex2(m - now)) + f.y * part_weight(f.x, now);
            m = now;
        }
#pragma unroll
        for (uint32_t o = 1; o < kLanes; o *= 2) {
            const float m2 = __shfl_xor_sync(0xffffffffu, m, o), l2 = __shfl_xor_sync(0xffffffffu, l, o);
            const float now = fmaxf(m, m2);
            l = l * part_weight(m, now) + l2 * part_weight(m2, now);
            m = now;
        }
        if (at == 0) of_row[row] = make_float2(m, l == 0.0f ? 0.0f : 1.0f / l);
    }
    // so many rows at a time that a thread has at most four pieces of them
    constexpr uint32_t kRows = R * DIM <= 16 * THREADS ? R : 16 * THREADS / DIM, kEach = (kRows * DIM / 4 + THREADS - 1) / THREADS;
    for (uint32_t r0 = 0; r0 < R; r0 += kRows) {
        float4 o[kEach];
#pragma unroll
        for (uint32_t x = 0; x < kEach; ++x) o[x] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (uint32_t from = 0; from < s.parts; from += kAttnJoin) {
            const uint32_t count = min(kAttnJoin, s.parts - from);
            __syncthreads();
            for (uint32_t x = tid; x < count * kRows; x += THREADS)
                weights[x] = part_weight(__ldcg(&p.part_ml[slot_of(from + x / kRows) * R + r0 + x % kRows]).x, of_row[r0 + x % kRows].x);
            __syncthreads();
#pragma unroll 8
            for (uint32_t c = 0; c < count; ++c) {
                const float4* src = reinterpret_cast<const float4*>(p.part_o + (slot_of(from + c) * R + r0) * DIM);
#pragma unroll
                for (uint32_t x = 0; x < kEach; ++x) {
                    const uint32_t at = tid + x * THREADS;
                    if (at < kRows * DIM / 4) {
                        const float4 f = __ldcg(src + at);
                        const float w = weights[c * kRows + at / (DIM / 4)];
                        o[x].x = fmaf(w, f.x, o[x].x);
                        o[x].y = fmaf(w, f.y, o[x].y);
                        o[x].z = fmaf(w, f.z, o[x].z);
                        o[x].w = fmaf(w, f.w, o[x].w);
                    }
                }
            }
        }
#pragma unroll
        for (uint32_t x = 0; x < kEach; ++x) {
            const uint32_t at = tid + x * THREADS, row = r0 + at / (DIM / 4);
            if (at < kRows * DIM / 4 && row < s.row_count) put_row(p, s, DIM, row, at % (DIM / 4) * 4, o[x], of_row[row].y);
        }
    }
}

template <bool K4, bool V4, int NB, int NT, int W>
struct AttnLayout {  // of W warps
    static constexpr uint32_t k_bytes = kv_part_bytes(K4, NB), v_bytes = kv_part_bytes(V4, NB), record = k_bytes + v_bytes;
    static constexpr uint32_t rows = NT == 0 ? 4 : 8 * NT, dim = 32 * NB;
    static constexpr uint32_t ring = W * 2 * record;
    static constexpr uint32_t joined = W / 2 * rows * dim * 4;  // outputs of half the warps, after the loop
    static constexpr uint32_t tiles = ring > joined ? ring : joined;
    static constexpr uint32_t q_bytes = NB * (NT == 0 ? 1 : 2 * NT) * 512;
    // the weights' transposition buffer lies over the keys' codes, which have been read by then, where it fits
    static constexpr uint32_t p_warp = rows * 32 * 4;
    static constexpr bool p_over = p_warp <= kv_code_bytes(K4, NB);
    static constexpr uint32_t p_bytes = p_over ? 0 : W * p_warp;
    static constexpr uint32_t smem = tiles + q_bytes + p_bytes + rows * 4 + W * rows * 8 + 128;
};

// Twelve warps per SM, as 168 registers allow: three blocks of four where their shared memory fits, else two of six (154 us
// instead of the 160 of two blocks of four for 48 drafted tokens of 32 heads over 12000, with eight rows to a block).  Sixteen rows
// need more registers than that: two blocks of four, 255 registers (156 us with six and 168 for those tokens, 149 so; 16
// tokens over 500: 15.7 and 14.7; heads of 64 over 12000: 95.5 and 98).  The largest heads have one block.
// With eight or sixteen rows of 128 or 256 values some registers spill: up to 48 bytes, 256 for sixteen rows of 256.
constexpr bool attn_fits(uint32_t smem, uint32_t blocks) { return blocks * (smem + 1024) <= 228 * 1024; }
template <bool K4, bool V4, int NB, int NT>
constexpr int attn_warps() {
    if (NT == 2 && NB <= 4) return 4;
    if (attn_fits(AttnLayout<K4, V4, NB, NT, 4>::smem, 3)) return 4;
    if (attn_fits(AttnLayout<K4, V4, NB, NT, 6>::smem, 2)) return 6;
    if (attn_fits(AttnLayout<K4, V4, NB, NT, 4>::smem, 2)) return 4;
    return attn_fits(AttnLayout<K4, V4, NB, NT, 6>::smem, 1) ? 6 : 4;
}
template <bool K4, bool V4, int NB, int NT>
struct AttnShape : AttnLayout<K4, V4, NB, NT, attn_warps<K4, V4, NB, NT>()> {
    static constexpr int warps = attn_warps<K4, V4, NB, NT>();
    static constexpr int blocks = NB > 4 ? 1 : warps == 4 && NT < 2 ? 3 : 2;  // of an SM, for the registers
};

// 16-byte slot of the weights' transposition buffer: rows of eight slots, spread so that the writes (one float per
// lane, rows two apart) and the reads (a slot per lane) meet different banks.
__device__ __forceinline__ uint32_t p_slot(uint32_t row, uint32_t slot) { return row * 8 + (slot ^ ((row ^ (row >> 1)) & 1u)); }

template <bool K4, bool V4, int NB, int NT>
__global__ void __launch_bounds__(AttnShape<K4, V4, NB, NT>::warps * 32, AttnShape<K4, V4, NB, NT>::blocks)
kv_attention_kernel(AttnParams p) {
    using Shape = AttnShape<K4, V4, NB, NT>;
    constexpr uint32_t R = Shape::rows, W = Shape::warps, kHalf = W / 2, kPerWarp = (R + W - 1) / W;
    // Groups of eight columns, and rows of a group that a lane has results of: with four rows their two parts are the columns.
    constexpr bool kParts = NT == 0;
    constexpr int N = kParts ? 1 : NT, E = kParts ? 1 : 2;
    constexpr float kNone = -INFINITY;
    extern __shared__ __align__(128) uint8_t smem[];
    uint8_t* qf = smem + Shape::tiles;
    float* pbuf = reinterpret_cast<float*>(qf + Shape::q_bytes);
    float* inv_lift = pbuf + Shape::p_bytes / 4;
    float2* ml = reinterpret_cast<float2*>(inv_lift + R);
    uint64_t* shared64 = reinterpret_cast<uint64_t*>(ml + W * R);

    pdl_wait();
    pdl_launch();
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    auto row_of = [&](int n, int e) { return kParts ? t : n * 8 + 2 * t + e; };

    Share at(p);
    if (!at.template find<R, W, kTileTokens>(p, shared64)) return;

    const uint32_t ring = smem_addr(smem) + warp * 2 * Shape::record;

    Segment seg;
    while (next_segment<R, kTileTokens>(p, at, seg)) {
        const KvSeq& sq = seg.sq;
        const uint32_t seq = seg.seq, head = seg.head, row_first = seg.row_first, row_count = seg.row_count, tile0 = seg.tile0, tile1 = seg.tile1;
        // with no mask, nothing is attended to behind the last row's own token
        uint32_t last_tile = tile1;
        if (p.mask == nullptr) last_tile = min(last_tile, (sq.start + (row_first + row_count - 1) / p.group) / kTileTokens + 1);

        // ---- q's rows and the first two tiles of every warp come in together -----------------------------
        float qv[kPerWarp][NB];
#pragma unroll
        for (uint32_t x = 0; x < kPerWarp; ++x) {
            const uint32_t r = warp + x * W, rr = row_first + r, i = rr / p.group, hq = head * p.group + (rr - i * p.group);
            const float* src = p.q + (size_t)(sq.row0 + i) * p.q_stride + (size_t)hq * Shape::dim + lane;
#pragma unroll
            for (int b = 0; b < NB; ++b) qv[x][b] = r < row_count ? src[b * 32] : 0.0f;
        }
        const uint32_t mine0 = tile0 + warp;
        uint32_t have = 0;           // bit k & 1: tile number k has a page
        uint64_t ahead = 0;          // record of this lane's tile of the next 32 of this warp, 0 if it has no page
        auto look_ahead = [&](uint32_t tile) {
            const uint32_t x = tile + lane * W;
            ahead = x < last_tile ? reinterpret_cast<uint64_t>(kv_record(p.r, p.g, seq, x, head)) : 0;
        };
        auto fetch = [&](uint32_t k) {  // the warp's tile number k, which `ahead` has
            const uint64_t src = __shfl_sync(0xffffffffu, ahead, k & 31);
            if (src) {
                const uint32_t dst = ring + (k & 1) * Shape::record + lane * 16;
                const uint8_t* from = reinterpret_cast<const uint8_t*>(src) + lane * 16;
#pragma unroll
                for (uint32_t o = 0; o < Shape::record; o += 512)
                    if (o + 512 <= Shape::record || o + lane * 16 < Shape::record) cp_async16(dst + o, from + o);
            }
            cp_async_commit();
            have = src ? have | 1u << (k & 1) : have & ~(1u << (k & 1));
        };
        const uint32_t mine = mine0 < last_tile ? (last_tile - mine0 + W - 1) / W : 0;
        look_ahead(mine0);
        fetch(0);
        fetch(1);

        // ---- q: scaled, lifted by a power of two per row, split into two f16 parts in B-operand order ----------------
#pragma unroll
        for (uint32_t x = 0; x < kPerWarp; ++x) {
            const uint32_t r = warp + x * W;
            float most = 0.0f;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                qv[x][b] *= p.scale_log2;
                most = fmaxf(most, fabsf(qv[x][b]));
            }
            const float up = lift(warp_max(most));
            if (r >= R) break;
            if (lane == 0) inv_lift[r] = kCodeUnits / up;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const float v = qv[x][b] * up;
                const __half h = __float2half_rn(v), l = __float2half_rn(v - __half2float(h));
                uint8_t* dst = qf + frag_lane(lane) * 16 + frag_half(K4, lane) * 2 + (kParts ? b * 512 + r * 128 : ((b * N + r / 8) * 2) * 512 + (r % 8) * 64);
                *reinterpret_cast<__half*>(dst) = h;
                *reinterpret_cast<__half*>(dst + (kParts ? 64 : 512)) = l;
            }
        }
        __syncthreads();
        const uint32_t qs = smem_addr(qf) + lane * 16;
        float inv[N][E];
        float top[N][E], sum[N][E], acc[2 * NB][N][2 * E], unit[N][E];  // acc counts kCodeUnits / (2 unit)
#pragma unroll
        for (int n = 0; n < N; ++n) {
#pragma unroll
            for (int e = 0; e < E; ++e) {
                inv[n][e] = inv_lift[row_of(n, e)];
                top[n][e] = kNone;
                sum[n][e] = 0.0f;
                unit[n][e] = 1.0f;
            }
#pragma unroll
            for (int d = 0; d < 2 * NB; ++d)
#pragma unroll
                for (int c = 0; c < 2 * E; ++c) acc[d][n][c] = 0.0f;
        }

        for (uint32_t k = 0; k < mine; ++k) {
            const uint32_t tile = mine0 + k * W;
            cp_async_wait<1>();
            __syncwarp();
            if (have >> (k & 1) & 1) {
                const uint32_t rec = ring + (k & 1) * Shape::record, base = tile * kTileTokens;
                float* pwf = Shape::p_over ? reinterpret_cast<float*>(smem + (warp * 2 + (k & 1)) * Shape::record) : pbuf + warp * R * 32;
                const uint32_t pw = smem_addr(pwf);
                // ---- which of the tile's tokens each of the thread's rows attends to, if not to all -------------------------
                const bool masked = base + kTileTokens > sq.start;
                uint32_t may[N][E];
                if (masked) {
                    const uint32_t before = base < sq.start ? (1u << (sq.start - base)) - 1u : 0u;  // context
                    const uint32_t there = sq.end - base >= 32 ? 0xffffffffu : (1u << (sq.end - base)) - 1u;
                    const uint32_t j0 = base < sq.start ? 0u : base - sq.start, up = base < sq.start ? sq.start - base : 0u;
#pragma unroll
                    for (int n = 0; n < N; ++n)
#pragma unroll
                        for (int e = 0; e < E; ++e) {
                            const uint32_t rr = row_first + row_of(n, e), i = rr / p.group;
                            uint32_t bits = 0;  // of the call's tokens j0 ..
                            if (rr < sq.n * p.group) {
                                if (p.mask == nullptr) {
                                    bits = i < j0 ? 0u : i - j0 >= 31 ? 0xffffffffu : (2u << (i - j0)) - 1u;
                                } else {
                                    const uint32_t* row = p.mask + (size_t)(sq.row0 + i) * p.mask_words;
                                    const uint32_t w = j0 / 32;
                                    const uint32_t lo_ = w < p.mask_words ? row[w] : 0u, hi_ = w + 1 < p.mask_words ? row[w + 1] : 0u;
                                    bits = __funnelshift_r(lo_, hi_, j0 % 32);
                                }
                            }
                            may[n][e] = (before | bits << up) & there;
                        }
                }
                // ---- scores of 32 tokens: s[m][n][E h + e] = token 16 m + 8 h + g, row row_of(n, e)
                float s[2][N][2 * E];
#pragma unroll
                for (int m = 0; m < 2; ++m)
#pragma unroll
                    for (int n = 0; n < N; ++n)
#pragma unroll
                        for (int c = 0; c < 2 * E; ++c) s[m][n][c] = 0.0f;
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    uint32_t a[2][2][4];
                    if (K4) {
                        uint32_t w[4];
                        ldmatrix_x4(w, rec + b * 512 + lane * 16);
                        a_of_nibbles(w[0], w[1], a[0]);
                        a_of_nibbles(w[2], w[3], a[1]);
                    } else {
#pragma unroll
                        for (int m = 0; m < 2; ++m) {
                            uint32_t w[4];
                            ldmatrix_x4(w, rec + (2 * b + (lane >> 4)) * 512 + (m * 16 + (lane & 15)) * 16);
                            a_of_bytes(w, a[m]);
                        }
                    }
                    const uint2 ds = lds64(rec + kv_code_bytes(K4, NB) + b * 64 + g * 8);
                    const float2 d01 = __half22float2(bits_h2(ds.x)), d23 = __half22float2(bits_h2(ds.y));
                    // steps outside, tiles inside: neighbouring products do not wait for each other
                    float c[2][N][4];
                    uint4 qh[N], ql[N];
#pragma unroll
                    for (int n = 0; n < N; ++n) {
                        qh[n] = lds128(qs + (kParts ? b : (b * N + n) * 2) * 512);
                        if (!kParts) ql[n] = lds128(qs + ((b * N + n) * 2 + 1) * 512);
                    }
                    auto step = [&](auto use) {
#pragma unroll
                        for (int n = 0; n < N; ++n)
#pragma unroll
                            for (int m = 0; m < 2; ++m) use(n, m);
                    };
                    if (kParts) {
                        step([&](int n, int m) { mma_f16_new(c[m][n], a[m][0], qh[n].x, qh[n].y); });
                    } else {
                        step([&](int n, int m) { mma_f16_new(c[m][n], a[m][0], ql[n].x, ql[n].y); });
                        step([&](int n, int m) { mma_f16(c[m][n], a[m][1], ql[n].z, ql[n].w); });
                        step([&](int n, int m) { mma_f16(c[m][n], a[m][0], qh[n].x, qh[n].y); });
                    }
                    step([&](int n, int m) { mma_f16(c[m][n], a[m][1], qh[n].z, qh[n].w); });
                    step([&](int n, int m) {
                        const float d[2] = {m == 0 ? d01.x : d23.x, m == 0 ? d01.y : d23.y};
#pragma unroll
                        for (int h = 0; h < 2; ++h)
#pragma unroll
                            for (int e = 0; e < E; ++e)
                                s[m][n][E * h + e] = fmaf(d[h], kParts ? c[m][n][2 * h] + c[m][n][2 * h + 1] : c[m][n][2 * h + e], s[m][n][E * h + e]);
                    });
                }
#pragma unroll
                for (int m = 0; m < 2; ++m)
#pragma unroll
                    for (int n = 0; n < N; ++n)
#pragma unroll
                        for (int c = 0; c < 2 * E; ++c) s[m][n][c] *= inv[n][c % E];
                if (masked) {
                    __syncwarp();  // keeps this a branch that other tiles jump over
#pragma unroll
                    for (int m = 0; m < 2; ++m)
#pragma unroll
                        for (int n = 0; n < N; ++n)
#pragma unroll
                            for (int c = 0; c < 2 * E; ++c)
                                if (!(may[n][c % E] >> (m * 16 + (c / E) * 8 + g) & 1)) s[m][n][c] = kNone;
                }
                __syncwarp();  // the keys' codes have been read
                // ---- running maximum and sum; the weights change sides through shared memory -----------------------------
                float fall[N][E];
#pragma unroll
                for (int n = 0; n < N; ++n)
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        float mx = fmaxf(fmaxf(s[0][n][e], s[0][n][e + E]), fmaxf(s[1][n][e], s[1][n][e + E]));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                        const float now = fmaxf(top[n][e], mx), ref = now == kNone ? 0.0f : now;
                        fall[n][e] = ex2(top[n][e] - ref);
                        top[n][e] = now;
                        float add = 0.0f;
#pragma unroll
                        for (int m = 0; m < 2; ++m)
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                const float w = ex2(s[m][n][e + E * h] - ref);
                                add += w;
                                const uint32_t row = row_of(n, e), lo = g + 8 * h;  // token lo + 16 m
                                pwf[p_slot(row, (lo & 3) * 2 + m) * 4 + (lo >> 2)] = w;
                            }
                        sum[n][e] = fmaf(sum[n][e], fall[n][e], add);
                    }
                if (masked) {  // -0 for what a row does not attend to, 0 for a weight that is nothing
#pragma unroll
                    for (int n = 0; n < N; ++n)
#pragma unroll
                        for (int e = 0; e < E; ++e)
#pragma unroll
                            for (int m = 0; m < 2; ++m)
#pragma unroll
                                for (int h = 0; h < 2; ++h) {
                                    const uint32_t lo = g + 8 * h;
                                    if (!(may[n][e] >> (m * 16 + lo) & 1)) pwf[p_slot(row_of(n, e), (lo & 3) * 2 + m) * 4 + (lo >> 2)] = -0.0f;
                                }
                }
                __syncwarp();
                // ---- the value blocks' scales: tokens t + 4 i + 16 s of every lane, and the power of two that they allow
                const uint32_t vrec = rec + Shape::k_bytes, vscales = vrec + kv_code_bytes(V4, NB) + t * 16;
                uint4 dv[NB];
                __half2 most[4], least[4];
#pragma unroll
                for (int x = 0; x < 4; ++x) most[x] = bits_h2(0x04000400u);  // 2^-14: smaller scales keep their own size
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    dv[b] = lds128(vscales + b * 64);
                    const uint32_t d[4] = {dv[b].x, dv[b].y, dv[b].z, dv[b].w};
#pragma unroll
                    for (int x = 0; x < 4; ++x) {  // of NaN and a number, the number
                        most[x] = __hmax2(most[x], __habs2(bits_h2(d[x])));
                        least[x] = b == 0 ? __habs2(bits_h2(d[x])) : __hmin2(least[x], __habs2(bits_h2(d[x])));
                    }
                }
                __half2 back[4];  // 2^(1 - e)
                float pe[N][8];
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const uint32_t e = h2_bits(most[x]) & 0x7c007c00u;
                    back[x] = bits_h2(0x7c007c00u - e);
                    const float2 f = __half22float2(bits_h2(e));
                    pe[0][2 * x] = f.x;
                    pe[0][2 * x + 1] = f.y;
                }
                // whether a token may have a scale too far below its largest
                auto small_of = [&](const __half2 (&d)[4]) {
                    const __half2 low = __hmin2(__hmin2(__hmul2(d[0], back[0]), __hmul2(d[1], back[1])),
                                                __hmin2(__hmul2(d[2], back[2]), __hmul2(d[3], back[3])));
                    return !__hbge2(low, bits_h2(0x08000800u));  // 2^-13
                };
                const bool small_here = small_of(least);
                float largest[N], now[N][E];
#pragma unroll
                for (int n = N - 1; n >= 0; --n) {
                    largest[n] = 0.0f;
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const uint4 f = lds128(pw + p_slot(kParts ? g / 2 : n * 8 + g, t * 2 + x) * 16);
                        const uint32_t w[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            pe[n][4 * x + i] = __uint_as_float(w[i]) * pe[0][4 * x + i];
                            largest[n] = fmaxf(largest[n], pe[n][4 * x + i]);
                        }
                    }
                }
                // Each row has its own power of two: found by the four lanes with its weights, given to those with its output.
#pragma unroll
                for (int o = 1; o < 4; o *= 2)
#pragma unroll
                    for (int n = 0; n < N; ++n) largest[n] = fmaxf(largest[n], __shfl_xor_sync(0xffffffffu, largest[n], o));
#pragma unroll
                for (int n = 0; n < N; ++n) {
                    // 2^12 over the power of two below the largest; 2^64 at most, which a row without weights has (its output stays below 2^120)
                    const float up = __uint_as_float(min(((12u + 2u * 127u) << 23) - (__float_as_uint(largest[n]) & 0x7f800000u), (64u + 127u) << 23));
#pragma unroll
                    for (int e = 0; e < E; ++e) now[n][e] = __shfl_sync(0xffffffffu, up, kParts ? 8 * t : 8 * t + 4 * e);
#pragma unroll
                    for (int i = 0; i < 8; ++i) pe[n][i] *= up;
                }
#pragma unroll
                for (int n = 0; n < N; ++n)
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        fall[n][e] *= now[n][e] * __uint_as_float(0x7f000000u - __float_as_uint(unit[n][e]));  // powers of two
                        unit[n][e] = now[n][e];
                    }
                uint32_t ph[N][4], pl[N][4];  // pairs of tokens
                uint32_t minus[N][4];         // what hi is to be taken off for the lane's column: of the parts of four rows, the first has hi itself
#pragma unroll
                for (int n = 0; n < N; ++n)
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        split_f16(pe[n][2 * x], pe[n][2 * x + 1], &ph[n][x], &pl[n][x]);
                        minus[n][x] = kParts && !(g & 1) ? 0u : ph[n][x];
                        if (kParts && !(g & 1)) pl[n][x] = 0u;
                    }
                // ---- output ------------------------------------------------------------------------------------------
                auto weights = [&](int n, float (&w)[8]) {  // of the lane's row and tokens, once more
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const uint4 f = lds128(pw + p_slot(kParts ? g / 2 : n * 8 + g, t * 2 + x) * 16);
                        w[4 * x] = __uint_as_float(f.x);
                        w[4 * x + 1] = __uint_as_float(f.y);
                        w[4 * x + 2] = __uint_as_float(f.z);
                        w[4 * x + 3] = __uint_as_float(f.w);
                    }
                };
                auto output = [&](auto some_masked, auto in_f32) {
                    constexpr bool kMasked = decltype(some_masked)::value, kWide = decltype(in_f32)::value;
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        const __half2 d[4] = {__hmul2(bits_h2(dv[b].x), back[0]), __hmul2(bits_h2(dv[b].y), back[1]),
                                              __hmul2(bits_h2(dv[b].z), back[2]), __hmul2(bits_h2(dv[b].w), back[3])};
                        uint32_t a[2][2][4];  // [k-step][16 values][...]
                        if (V4) {
                            const uint4 w4 = lds128(vrec + b * 512 + lane * 16);
                            const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
                            for (int x = 0; x < 2; ++x)
#pragma unroll
                                for (int h = 0; h < 2; ++h) {
                                    const uint32_t u = w[2 * x + h], v = u >> 8;
                                    a[x][0][2 * h] = f16_of_low_nibbles(u);
                                    a[x][0][2 * h + 1] = f16_of_high_nibbles(u);
                                    a[x][1][2 * h] = f16_of_low_nibbles(v);
                                    a[x][1][2 * h + 1] = f16_of_high_nibbles(v);
                                }
                        } else {
#pragma unroll
                            for (int x = 0; x < 2; ++x) {
                                const uint4 w4 = lds128(vrec + b * 1024 + x * 512 + lane * 16);
                                a[x][0][0] = f16_of_bytes(w4.x, 0x4140);
                                a[x][0][1] = f16_of_bytes(w4.y, 0x4140);
                                a[x][0][2] = f16_of_bytes(w4.x, 0x4342);
                                a[x][0][3] = f16_of_bytes(w4.y, 0x4342);
                                a[x][1][0] = f16_of_bytes(w4.z, 0x4140);
                                a[x][1][1] = f16_of_bytes(w4.w, 0x4140);
                                a[x][1][2] = f16_of_bytes(w4.z, 0x4342);
                                a[x][1][3] = f16_of_bytes(w4.w, 0x4342);
                            }
                        }
                        uint32_t hi_[N][4], lo_[N][4];  // with four rows, the lane's part is in lo_
                        float back_to[N][E];            // what the block's sums count in the output's unit
                        if constexpr (!kWide) {
#pragma unroll
                            for (int n = 0; n < N; ++n)
#pragma unroll
                                for (int x = 0; x < 4; ++x) {
                                    const __half2 h = __hmul2(bits_h2(minus[n][x]), d[x]);
                                    const __half2 l = __hfma2(bits_h2(pl[n][x]), d[x], __hfma2(bits_h2(ph[n][x]), d[x], __hneg2(h)));
                                    hi_[n][x] = h2_bits(h);
                                    lo_[n][x] = h2_bits(l);
                                    if (kMasked) {  // what is no number in a masked place (weight -0) stays there
                                        const uint32_t on = ((ph[n][x] & 0xffffu) == 0x8000u ? 0u : 0xffffu) | (ph[n][x] >> 16 == 0x8000u ? 0u : 0xffff0000u);
                                        hi_[n][x] &= on;
                                        lo_[n][x] &= on;
                                    }
                                }
                        } else {
                            const uint32_t own[4] = {dv[b].x, dv[b].y, dv[b].z, dv[b].w};
#pragma unroll
                            for (int n = 0; n < N; ++n) {
                                float w[8], most_ = 0.0f;
                                weights(n, w);
#pragma unroll
                                for (int x = 0; x < 4; ++x) {
                                    const float2 f = __half22float2(bits_h2(own[x]));
                                    w[2 * x] = __float_as_uint(w[2 * x]) == 0x80000000u ? 0.0f : w[2 * x] * f.x;
                                    w[2 * x + 1] = __float_as_uint(w[2 * x + 1]) == 0x80000000u ? 0.0f : w[2 * x + 1] * f.y;
                                    most_ = fmaxf(most_, fmaxf(fabsf(w[2 * x]), fabsf(w[2 * x + 1])));
                                }
                                most_ = fmaxf(most_, __shfl_xor_sync(0xffffffffu, most_, 1));
                                most_ = fmaxf(most_, __shfl_xor_sync(0xffffffffu, most_, 2));
                                const float up = lift(most_), inverse = __uint_as_float(0x7f000000u - __float_as_uint(up));
#pragma unroll
                                for (int e = 0; e < E; ++e) back_to[n][e] = 2.0f * unit[n][e] * __shfl_sync(0xffffffffu, inverse, kParts ? 8 * t : 8 * t + 4 * e);
#pragma unroll
                                for (int x = 0; x < 4; ++x) {
                                    split_f16(w[2 * x] * up, w[2 * x + 1] * up, &hi_[n][x], &lo_[n][x]);
                                    if (kParts && !(g & 1)) lo_[n][x] = hi_[n][x];
                                }
                            }
                        }
                        // The tensor cores cut their f32 sums off instead of rounding them: a tile's sum is taken from
                        // zero and added to the output here, or the loss would grow with the number of tiles.
                        float o[N][2][4];
                        auto step = [&](auto use) {
#pragma unroll
                            for (int n = 0; n < N; ++n)
#pragma unroll
                                for (int m = 0; m < 2; ++m) use(n, m);
                        };
                        step([&](int n, int m) { mma_f16_new(o[n][m], a[0][m], lo_[n][0], lo_[n][1]); });
                        step([&](int n, int m) { mma_f16(o[n][m], a[1][m], lo_[n][2], lo_[n][3]); });
                        if (!kParts) {
                            step([&](int n, int m) { mma_f16(o[n][m], a[0][m], hi_[n][0], hi_[n][1]); });
                            step([&](int n, int m) { mma_f16(o[n][m], a[1][m], hi_[n][2], hi_[n][3]); });
                        }
                        step([&](int n, int m) {
#pragma unroll
                            for (int c = 0; c < 2 * E; ++c) {
                                const float sum_ = kParts ? o[n][m][2 * c] + o[n][m][2 * c + 1] : o[n][m][c];
                                acc[2 * b + m][n][c] = fmaf(acc[2 * b + m][n][c], fall[n][c % E], kWide ? sum_ * back_to[n][c % E] : sum_);
                            }
                        });
                    }
                };
                bool wide = __any_sync(0xffffffffu, small_here);
                if (wide) {  // most often the zeros behind a sequence's end: only tokens that a row gives weight count
                    uint32_t weighted[4] = {0u, 0u, 0u, 0u};
#pragma unroll
                    for (int n = 0; n < N; ++n) {
                        float w[8];
                        weights(n, w);
#pragma unroll
                        for (int x = 0; x < 4; ++x) weighted[x] |= (w[2 * x] > 0.0f ? 0xffffu : 0u) | (w[2 * x + 1] > 0.0f ? 0xffff0000u : 0u);
                    }
                    auto closer = [&](auto but_empty) {  // but_empty: not the blocks in which no token of the tile has anything
                        __half2 low[4] = {bits_h2(0x7bff7bffu), bits_h2(0x7bff7bffu), bits_h2(0x7bff7bffu), bits_h2(0x7bff7bffu)};
#pragma unroll
                        for (int b = 0; b < NB; ++b) {
                            const uint32_t d[4] = {dv[b].x, dv[b].y, dv[b].z, dv[b].w};
                            if (decltype(but_empty)::value && !__any_sync(0xffffffffu, ((d[0] | d[1] | d[2] | d[3]) & 0x7fff7fffu) != 0)) continue;
#pragma unroll
                            for (int x = 0; x < 4; ++x) low[x] = __hmin2(low[x], __habs2(bits_h2(d[x])));
                        }
#pragma unroll
                        for (int x = 0; x < 4; ++x) low[x] = bits_h2((h2_bits(low[x]) & weighted[x]) | (0x7bff7bffu & ~weighted[x]));
                        return (bool)__any_sync(0xffffffffu, small_of(low));
                    };
                    wide = closer(std::false_type()) && closer(std::true_type());
                }
                if (wide) {
                    output(std::false_type(), std::true_type());
                } else if (masked) {
                    __syncwarp();
                    output(std::true_type(), std::false_type());
                } else {
                    output(std::false_type(), std::false_type());
                }
            }
            __syncwarp();  // the tile and the weights have been read
            if (((k + 2) & 31) == 0) look_ahead(mine0 + (k + 2) * W);
            fetch(k + 2);
        }
        cp_async_wait<0>();

        // ---- the warps' parts become one -------------------------------------------------------------------------
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int e = 0; e < E; ++e) {
                float l = sum[n][e];
                l += __shfl_xor_sync(0xffffffffu, l, 4);
                l += __shfl_xor_sync(0xffffffffu, l, 8);
                l += __shfl_xor_sync(0xffffffffu, l, 16);
                if (g == 0) ml[warp * R + row_of(n, e)] = make_float2(top[n][e], l);
            }
        __syncthreads();
        float* joined = reinterpret_cast<float*>(smem);
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int e = 0; e < E; ++e) {
                float m = kNone;
#pragma unroll
                for (uint32_t w = 0; w < W; ++w) m = fmaxf(m, ml[w * R + row_of(n, e)].x);
                const float f = top[n][e] == kNone ? 0.0f : ex2(top[n][e] - m) * (0.5f * kCodeUnits * __uint_as_float(0x7f000000u - __float_as_uint(unit[n][e])));
#pragma unroll
                for (int d = 0; d < 2 * NB; ++d) {
                    acc[d][n][e] *= f;
                    acc[d][n][e + E] *= f;
                }
            }
        auto each = [&](auto use) {  // lane's four neighbouring values of every (row, block)
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
                for (int e = 0; e < E; ++e)
#pragma unroll
                    for (int b = 0; b < NB; ++b) use(n, e, b, row_of(n, e) * Shape::dim + b * 32 + g * 4);
        };
        auto store = [&](uint32_t half) {
            each([&](int n, int e, int b, uint32_t at) {
                *reinterpret_cast<float4*>(joined + half * R * Shape::dim + at) =
                    make_float4(acc[2 * b][n][e], acc[2 * b][n][e + E], acc[2 * b + 1][n][e], acc[2 * b + 1][n][e + E]);
            });
        };
        if (warp >= kHalf) store(warp - kHalf);
        __syncthreads();
        if (warp < kHalf) {
            each([&](int n, int e, int b, uint32_t at) {
                const float4 f = *reinterpret_cast<const float4*>(joined + warp * R * Shape::dim + at);
                acc[2 * b][n][e] += f.x;
                acc[2 * b][n][e + E] += f.y;
                acc[2 * b + 1][n][e] += f.z;
                acc[2 * b + 1][n][e + E] += f.w;
            });
            store(warp);
        }
        __syncthreads();
        for (uint32_t x = tid; x < R * Shape::dim / 4; x += W * 32) {
            const uint32_t row = x / (Shape::dim / 4), col = (x % (Shape::dim / 4)) * 4;
            float m = kNone, l = 0.0f;
#pragma unroll
            for (uint32_t w = 0; w < W; ++w) m = fmaxf(m, ml[w * R + row].x);
#pragma unroll
            for (uint32_t w = 0; w < W; ++w) l += ml[w * R + row].y * part_weight(ml[w * R + row].x, m);
            float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (uint32_t w = 0; w < kHalf; ++w) {
                const float4 f = *reinterpret_cast<const float4*>(joined + (w * R + row) * Shape::dim + col);
                o.x += f.x;
                o.y += f.y;
                o.z += f.z;
                o.w += f.w;
            }
            if (seg.whole) {
                if (row < row_count) put_row(p, seg, Shape::dim, row, col, o, l == 0.0f ? 0.0f : 1.0f / l);
            } else {
                *reinterpret_cast<float4*>(p.part_o + ((size_t)seg.slot * R + row) * Shape::dim + col) = o;
                if (col == 0) p.part_ml[(size_t)seg.slot * R + row] = make_float2(m, l);
            }
        }
        if (!seg.whole && last_of(p.counters + seg.c0, seg.parts, reinterpret_cast<uint32_t*>(shared64)))
            join_parts<R, Shape::dim, W * 32>(p, seg, ml, reinterpret_cast<float*>(smem));
        __syncthreads();
    }
}

template <bool K4, bool V4>
vx_status kv_attention_setup(uint32_t blocks, uint32_t nt, int* per_sm, uint32_t* smem);
template <bool K4, bool V4>
vx_status kv_attention_launch(uint32_t blocks, uint32_t nt, uint32_t grid, cudaStream_t stream, const AttnParams& p);

// Calls f with the kernel of a head size (blocks of 32) and group of rows, and its shared memory.
template <bool K4, bool V4, class F>
bool attn_pick(uint32_t nb, uint32_t nt, F f) {
    auto go = [&](auto b, auto n) {
        constexpr int B = decltype(b)::value, N = decltype(n)::value;
        f(kv_attention_kernel<K4, V4, B, N>, AttnShape<K4, V4, B, N>::smem, (uint32_t)AttnShape<K4, V4, B, N>::warps * 32);
        return true;
    };
    using std::integral_constant;
#define VX_ATTN_CASE(B, N) \
    if (nb == B && nt == N) return go(integral_constant<int, B>{}, integral_constant<int, N>{});
    VX_ATTN_CASE(2, 0)
    VX_ATTN_CASE(2, 1)
    VX_ATTN_CASE(2, 2)
    VX_ATTN_CASE(3, 0)
    VX_ATTN_CASE(3, 1)
    VX_ATTN_CASE(3, 2)
    VX_ATTN_CASE(4, 0)
    VX_ATTN_CASE(4, 1)
    VX_ATTN_CASE(4, 2)
    VX_ATTN_CASE(8, 0)
    VX_ATTN_CASE(8, 1)
    VX_ATTN_CASE(8, 2)
#undef VX_ATTN_CASE
    return false;
}

#define VX_ATTN_INSTANCE(K4, V4)                                                                                          \
    template <>                                                                                                           \
    vx_status kv_attention_setup<K4, V4>(uint32_t nb, uint32_t nt, int* per_sm, uint32_t* smem) {                         \
        cudaError_t e = cudaSuccess;                                                                                      \
        const bool known = attn_pick<K4, V4>(nb, nt, [&](auto kernel, uint32_t bytes, uint32_t threads) {                 \
            *smem = bytes;                                                                                                \
            e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);                    \
            if (e == cudaSuccess)                                                                                         \
                e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(per_sm, kernel, (int)threads, bytes);                   \
        });                                                                                                               \
        VX_REQUIRE(known, VX_ERR_UNSUPPORTED, "attention: no kernel for heads of %u values", nb * 32);                    \
        VX_CUDA(e);                                                                                                       \
        return VX_OK;                                                                                                     \
    }                                                                                                                     \
    template <>                                                                                                           \
    vx_status kv_attention_launch<K4, V4>(uint32_t nb, uint32_t nt, uint32_t grid, cudaStream_t stream, const AttnParams& p) { \
        cudaError_t e = cudaSuccess;                                                                                      \
        attn_pick<K4, V4>(nb, nt, [&](auto kernel, uint32_t bytes, uint32_t threads) { e = launch_after(kernel, dim3(grid), threads, bytes, stream, p); }); \
        VX_CUDA(e);                                                                                                       \
        return VX_OK;                                                                                                     \
    }

}  // namespace vx
