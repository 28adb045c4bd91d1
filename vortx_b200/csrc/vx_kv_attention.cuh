// Attention of a call's rows over the quantised cache: the kernel, included by the files that instantiate it for a
// pair of types (vx_kv_attention_*.cu), and what its host side needs to know.
//
// S^T = K Q^T and O^T = V^T P^T: the codes are the A operand (16 tokens or 16 values of the head high), the query rows are the
// 8-wide N dimension, so the few rows of a decode step (query heads that share a head of keys, times drafted tokens)
// fill the tensor cores' tiles.  A thread block has a head of a sequence, up to 8 NT query rows and a run of 32-token
// tiles; its four warps take the tiles in turn, each with its own running maximum, sum and output (one pass over the
// cache, no synchronisation between tiles), two tiles in flight per warp (cp.async, a record is contiguous).
//   scores   per block of 32 values: sum of code * (q hi + q lo) on the tensor cores, times the block's scale, in f32
//   softmax  base 2 (log2 e is multiplied into q), running maximum per row, weights p <= 1
//   output   the value blocks' scales are per token, so they go into the weights: w = p * d * c with c a power of two
//            that keeps the largest |d| c in [2^14, 2^15), w split into two f16 parts, times the codes
// The runs are equal shares of all tiles of all (sequence, head, group of rows): whatever the lengths, every block of
// the grid has the same number of tiles.  A share that covers the tiles of a (sequence, head, rows) only in part leaves maximum, sum
// and unnormalised output in the workspace, at most two per block, and kv_merge_kernel joins them in a fixed order.
#pragma once

#include "vx_decode.cuh"

namespace vx {

constexpr int kAttnWarps = 4;
constexpr uint32_t kAttnMinTiles = kAttnWarps;  // tiles per block below which fewer blocks work

struct AttnParams {
    KvGeometry g;
    KvRows r;
    const float* q;
    float* out;
    size_t q_stride, out_stride;
    uint32_t heads, group;   // query heads, of one head of keys
    float scale_log2;        // scale * log2 e
    const uint32_t* mask;
    uint32_t mask_words;
    float* part_o;           // [2 * grid][8 NT][D]
    float2* part_ml;         // [2 * grid][8 NT] maximum (base 2), sum
    uint64_t* plan;          // [0] all tiles, [1] blocks that work, [2 + s] tiles before sequence s
};

// Tiles of sequence s over all its (head, group of rows).
__device__ __forceinline__ uint64_t seq_work(const KvSeq& q, const KvGeometry& g, uint32_t group, uint32_t rows_per_item) {
    const uint64_t items = (uint64_t)g.heads * (((uint64_t)q.n * group + rows_per_item - 1) / rows_per_item);
    return items * ((q.end + kTileTokens - 1) / kTileTokens);
}
__device__ __forceinline__ uint64_t share_begin(uint64_t total, uint64_t blocks, uint64_t c) { return c * total / blocks; }
__device__ __forceinline__ uint64_t share_of(uint64_t total, uint64_t blocks, uint64_t x) { return ((x + 1) * blocks - 1) / total; }

template <bool K4, bool V4, int NB, int NT>
struct AttnShape {
    static constexpr uint32_t k_bytes = kv_part_bytes(K4, NB), v_bytes = kv_part_bytes(V4, NB), record = k_bytes + v_bytes;
    static constexpr uint32_t rows = 8 * NT, dim = 32 * NB;
    static constexpr uint32_t ring = kAttnWarps * 2 * record;
    static constexpr uint32_t joined = 2 * rows * dim * 4;  // outputs of two warps, after the loop
    static constexpr uint32_t tiles = ring > joined ? ring : joined;
    static constexpr uint32_t q_bytes = NB * NT * 2 * 512;
    static constexpr uint32_t p_bytes = kAttnWarps * rows * 32 * 4;
    static constexpr uint32_t smem = tiles + q_bytes + p_bytes + rows * 4 + kAttnWarps * rows * 8 + 64;
};

// 16-byte slot of the weights' transposition buffer: rows of eight slots, spread so that the writes (one float per
// lane, rows two apart) and the reads (a slot per lane) meet different banks.
__device__ __forceinline__ uint32_t p_slot(uint32_t row, uint32_t slot) { return row * 8 + (slot ^ ((row ^ (row >> 1)) & 1u)); }

template <bool K4, bool V4, int NB, int NT>
__global__ void __launch_bounds__(kAttnWarps * 32, NT == 1 ? (NB <= 4 ? 3 : 2) : (NT * NB <= 8 ? 3 : 2))
kv_attention_kernel(const AttnParams p) {
    using Shape = AttnShape<K4, V4, NB, NT>;
    constexpr uint32_t R = Shape::rows;
    constexpr float kNone = -INFINITY;
    extern __shared__ __align__(128) uint8_t smem[];
    uint8_t* qf = smem + Shape::tiles;
    float* pbuf = reinterpret_cast<float*>(qf + Shape::q_bytes);
    float* inv_lift = pbuf + kAttnWarps * R * 32;
    float2* ml = reinterpret_cast<float2*>(inv_lift + R);
    uint64_t* shared64 = reinterpret_cast<uint64_t*>(ml + kAttnWarps * R);

    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;

    // ---- this block's share -----------------------------------------------------------------------------------
    uint32_t seq;
    uint64_t pos, hi;   // position within the sequence's tiles, end of the share (in the same count)
    {
        const uint32_t per = (p.r.seqs + kAttnWarps * 32 - 1) / (kAttnWarps * 32);
        const uint32_t s0 = min(p.r.seqs, tid * per), s1 = min(p.r.seqs, s0 + per);
        uint64_t mine = 0;
        for (uint32_t s = s0; s < s1; ++s) mine += seq_work(kv_seq(p.r, p.g, s), p.g, p.group, R);
        uint64_t before = mine;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const uint64_t v = __shfl_up_sync(0xffffffffu, before, o);
            if (lane >= (uint32_t)o) before += v;
        }
        if (lane == 31) shared64[warp] = before;
        __syncthreads();
        uint64_t total = 0;
        before -= mine;
        for (uint32_t w = 0; w < kAttnWarps; ++w) {
            if (w < warp) before += shared64[w];
            total += shared64[w];
        }
        uint64_t blocks = (total + kAttnMinTiles - 1) / kAttnMinTiles;
        if (blocks > gridDim.x) blocks = gridDim.x;
        if (blocks < 1) blocks = 1;
        if (blockIdx.x == 0) {  // for the kernel that joins the parts
            if (tid == 0) {
                p.plan[0] = total;
                p.plan[1] = blocks;
            }
            uint64_t at = before;
            for (uint32_t s = s0; s < s1; ++s) {
                p.plan[2 + s] = at;
                at += seq_work(kv_seq(p.r, p.g, s), p.g, p.group, R);
            }
        }
        if (blockIdx.x >= blocks || total == 0) return;
        const uint64_t lo = share_begin(total, blocks, blockIdx.x);
        hi = share_begin(total, blocks, blockIdx.x + 1);
        __syncthreads();
        if (before <= lo && lo < before + mine) {  // one thread of the block
            uint64_t at = before;
            uint32_t s = s0;
            for (;; ++s) {
                const uint64_t w = seq_work(kv_seq(p.r, p.g, s), p.g, p.group, R);
                if (lo < at + w) break;
                at += w;
            }
            shared64[0] = s;
            shared64[1] = at;
        }
        __syncthreads();
        seq = (uint32_t)shared64[0];
        pos = lo - shared64[1];
        hi -= shared64[1];
    }

    const uint32_t ring = smem_addr(smem) + warp * 2 * Shape::record;
    const uint32_t pw = smem_addr(pbuf) + warp * R * 32 * 4;
    float* pwf = pbuf + warp * R * 32;

    while (pos < hi) {
        const KvSeq sq = kv_seq(p.r, p.g, seq);
        const uint64_t work = seq_work(sq, p.g, p.group, R);
        if (pos >= work) {  // on to the next sequence
            pos -= work;
            hi -= work;
            ++seq;
            continue;
        }
        const uint32_t seq_tiles = (sq.end + kTileTokens - 1) / kTileTokens;
        const uint32_t groups = (uint32_t)(((uint64_t)sq.n * p.group + R - 1) / R);
        const uint32_t item = (uint32_t)(pos / seq_tiles), tile0 = (uint32_t)(pos - (uint64_t)item * seq_tiles);
        const uint32_t head = item / groups, rt = item - head * groups;
        uint32_t tile1 = seq_tiles;
        if (hi - pos < seq_tiles - tile0) tile1 = tile0 + (uint32_t)(hi - pos);
        pos += tile1 - tile0;
        const uint32_t row_first = rt * R, row_count = min(R, sq.n * p.group - row_first);
        // with no mask, nothing is attended to behind the last row's own token
        uint32_t last_tile = tile1;
        if (p.mask == nullptr) last_tile = min(last_tile, (sq.start + (row_first + row_count - 1) / p.group) / kTileTokens + 1);

        // ---- the first two tiles of every warp, while q is laid out -----------------------------------------------
        const uint32_t mine0 = tile0 + warp;
        uint64_t ahead = 0;          // record of this lane's tile of the next 32 of this warp, 0 if it has no page
        auto look_ahead = [&](uint32_t tile) {
            const uint32_t x = tile + lane * kAttnWarps;
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
            return src != 0;
        };
        const uint32_t mine = mine0 < last_tile ? (last_tile - mine0 + kAttnWarps - 1) / kAttnWarps : 0;
        look_ahead(mine0);
        bool have[2];
        have[0] = fetch(0);
        have[1] = fetch(1);

        // ---- q: scaled, lifted by a power of two per row, split into two f16 parts in B-operand order ----------------
        for (uint32_t r = warp; r < R; r += kAttnWarps) {
            float v[NB], top = 0.0f;
            const uint32_t rr = row_first + r, i = rr / p.group, hq = head * p.group + (rr - i * p.group);
            const float* src = p.q + (size_t)(sq.row0 + i) * p.q_stride + (size_t)hq * Shape::dim;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                v[b] = r < row_count ? src[b * 32 + lane] * p.scale_log2 : 0.0f;
                top = fmaxf(top, fabsf(v[b]));
            }
            const float up = lift(warp_max(top));
            if (lane == 0) inv_lift[r] = 1.0f / up;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const float x = v[b] * up;
                const __half h = __float2half_rn(x), l = __float2half_rn(x - __half2float(h));
                uint8_t* dst = qf + ((b * NT + r / 8) * 2) * 512 + ((r % 8) * 4 + frag_lane(lane)) * 16 + frag_half(K4, lane) * 2;
                *reinterpret_cast<__half*>(dst) = h;
                *reinterpret_cast<__half*>(dst + 512) = l;
            }
        }
        __syncthreads();
        const uint32_t qs = smem_addr(qf) + lane * 16;
        float inv[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            inv[n][0] = inv_lift[n * 8 + 2 * t];
            inv[n][1] = inv_lift[n * 8 + 2 * t + 1];
        }

        float top[NT][2], sum[NT][2], acc[2 * NB][NT][4], lifted = __uint_as_float((28u + 127u) << 23);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            top[n][0] = top[n][1] = kNone;
            sum[n][0] = sum[n][1] = 0.0f;
#pragma unroll
            for (int d = 0; d < 2 * NB; ++d)
#pragma unroll
                for (int c = 0; c < 4; ++c) acc[d][n][c] = 0.0f;
        }

        for (uint32_t k = 0; k < mine; ++k) {
            const uint32_t tile = mine0 + k * kAttnWarps;
            cp_async_wait<1>();
            __syncwarp();
            if (have[k & 1]) {
                const uint32_t rec = ring + (k & 1) * Shape::record;
                // ---- scores of 32 tokens: s[m][n] = tokens 16 m + g (c 0, 1) and 16 m + g + 8 (c 2, 3), rows 8 n + 2 t, + 1
                float s[2][NT][4];
#pragma unroll
                for (int m = 0; m < 2; ++m)
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int c = 0; c < 4; ++c) s[m][n][c] = 0.0f;
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
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        const uint4 qh = lds128(qs + ((b * NT + n) * 2) * 512), ql = lds128(qs + ((b * NT + n) * 2 + 1) * 512);
#pragma unroll
                        for (int m = 0; m < 2; ++m) {
                            float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                            mma_f16(c, a[m][0], ql.x, ql.y);
                            mma_f16(c, a[m][1], ql.z, ql.w);
                            mma_f16(c, a[m][0], qh.x, qh.y);
                            mma_f16(c, a[m][1], qh.z, qh.w);
                            const float d0 = m == 0 ? d01.x : d23.x, d1 = m == 0 ? d01.y : d23.y;
                            s[m][n][0] = fmaf(d0, c[0], s[m][n][0]);
                            s[m][n][1] = fmaf(d0, c[1], s[m][n][1]);
                            s[m][n][2] = fmaf(d1, c[2], s[m][n][2]);
                            s[m][n][3] = fmaf(d1, c[3], s[m][n][3]);
                        }
                    }
                }
                const uint32_t base = tile * kTileTokens;
                const bool masked = base + kTileTokens > sq.start;
#pragma unroll
                for (int m = 0; m < 2; ++m)
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            s[m][n][c] *= inv[n][c & 1];
                            if (masked) {
                                const uint32_t token = base + m * 16 + (c >> 1) * 8 + g;
                                if (token >= sq.start) {
                                    const uint32_t j = token - sq.start, rr = row_first + n * 8 + 2 * t + (c & 1);
                                    bool may = token < sq.end && rr < sq.n * p.group;
                                    if (may) {
                                        const uint32_t i = rr / p.group;
                                        if (p.mask == nullptr) may = j <= i;
                                        else may = j / 32 < p.mask_words &&
                                                   ((p.mask[(size_t)(sq.row0 + i) * p.mask_words + j / 32] >> (j & 31)) & 1u);
                                    }
                                    if (!may) s[m][n][c] = kNone;
                                }
                            }
                        }
                // ---- running maximum and sum; the weights change sides through shared memory -----------------------------
                float fall[NT][2];
                bool rescale = false;
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float mx = fmaxf(fmaxf(s[0][n][e], s[0][n][e + 2]), fmaxf(s[1][n][e], s[1][n][e + 2]));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                        const float now = fmaxf(top[n][e], mx), ref = now == kNone ? 0.0f : now;
                        fall[n][e] = exp2f(top[n][e] - ref);
                        rescale |= fall[n][e] != 1.0f;
                        top[n][e] = now;
                        float add = 0.0f;
#pragma unroll
                        for (int m = 0; m < 2; ++m)
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                const float w = exp2f(s[m][n][e + 2 * h] - ref);
                                add += w;
                                const uint32_t row = n * 8 + 2 * t + e, lo = g + 8 * h;  // token lo + 16 m
                                pwf[p_slot(row, (lo & 3) * 2 + m) * 4 + (lo >> 2)] = w;
                            }
                        sum[n][e] = fmaf(sum[n][e], fall[n][e], add);
                    }
                __syncwarp();
                // ---- the value blocks' scales: tokens t + 4 i + 16 s of every lane, and the power of two that they allow
                const uint32_t vrec = rec + Shape::k_bytes, vscales = vrec + kv_code_bytes(V4, NB) + t * 16;
                uint4 dv[NB];
                __half2 big = __float2half2_rn(0.0f);
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    dv[b] = lds128(vscales + b * 64);
                    if (masked) {  // behind the sequence's end lies whatever the page held before
                        uint32_t* w = &dv[b].x;
#pragma unroll
                        for (int x = 0; x < 8; ++x)
                            if (base + t + 4 * (x & 3) + 16 * (x >> 2) >= sq.end) w[x / 2] &= x & 1 ? 0x0000ffffu : 0xffff0000u;
                    }
                    big = __hmax2(big, __hmax2(__hmax2(__habs2(bits_h2(dv[b].x)), __habs2(bits_h2(dv[b].y))),
                                               __hmax2(__habs2(bits_h2(dv[b].z)), __habs2(bits_h2(dv[b].w)))));
                }
                float largest = fmaxf(__low2float(big), __high2float(big));
                largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
                largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
                if (largest > 0.0f) {
                    const float up = fminf(lift(largest), lifted);
                    if (up < lifted) {
                        const float ratio = up / lifted;  // powers of two
                        rescale = true;
                        lifted = up;
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            fall[n][0] *= ratio;
                            fall[n][1] *= ratio;
                        }
                    }
                }
                if (__any_sync(0xffffffffu, rescale)) {
#pragma unroll
                    for (int d = 0; d < 2 * NB; ++d)
#pragma unroll
                        for (int n = 0; n < NT; ++n)
#pragma unroll
                            for (int c = 0; c < 4; ++c) acc[d][n][c] *= fall[n][c & 1];
                }
                float w8[NT][8];
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const uint4 f = lds128(pw + p_slot(n * 8 + g, t * 2 + x) * 16);
                        w8[n][4 * x] = __uint_as_float(f.x);
                        w8[n][4 * x + 1] = __uint_as_float(f.y);
                        w8[n][4 * x + 2] = __uint_as_float(f.z);
                        w8[n][4 * x + 3] = __uint_as_float(f.w);
                    }
                // ---- output ------------------------------------------------------------------------------------------
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    float d8[8];
                    const uint32_t raw[4] = {dv[b].x, dv[b].y, dv[b].z, dv[b].w};
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const float2 f = __half22float2(bits_h2(raw[x]));
                        d8[2 * x] = f.x * lifted;
                        d8[2 * x + 1] = f.y * lifted;
                    }
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
                            const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                const uint32_t u = __byte_perm(w[2 * h], w[2 * h + 1], 0x5140), v = __byte_perm(w[2 * h], w[2 * h + 1], 0x7362);
                                a[x][0][2 * h] = f16_of_bytes(u, 0x4140);
                                a[x][0][2 * h + 1] = f16_of_bytes(u, 0x4342);
                                a[x][1][2 * h] = f16_of_bytes(v, 0x4140);
                                a[x][1][2 * h + 1] = f16_of_bytes(v, 0x4342);
                            }
                        }
                    }
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        uint32_t hi_[4], lo_[4];
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            float u = w8[n][2 * x] * d8[2 * x], v = w8[n][2 * x + 1] * d8[2 * x + 1];
                            if (masked) {  // a NaN in a masked place stays there
                                if (w8[n][2 * x] == 0.0f) u = 0.0f;
                                if (w8[n][2 * x + 1] == 0.0f) v = 0.0f;
                            }
                            split_f16(u, v, &hi_[x], &lo_[x]);
                        }
#pragma unroll
                        for (int x = 0; x < 2; ++x)
#pragma unroll
                            for (int m = 0; m < 2; ++m) {
                                mma_f16(acc[2 * b + m][n], a[x][m], lo_[2 * x], lo_[2 * x + 1]);
                                mma_f16(acc[2 * b + m][n], a[x][m], hi_[2 * x], hi_[2 * x + 1]);
                            }
                    }
                }
            }
            __syncwarp();  // the tile and the weights have been read
            if (((k + 2) & 31) == 0) look_ahead(mine0 + (k + 2) * kAttnWarps);
            have[k & 1] = fetch(k + 2);
        }
        cp_async_wait<0>();

        // ---- the four warps' parts become one ------------------------------------------------------------------------
        const float down = 1.0f / lifted;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float l = sum[n][e];
                l += __shfl_xor_sync(0xffffffffu, l, 4);
                l += __shfl_xor_sync(0xffffffffu, l, 8);
                l += __shfl_xor_sync(0xffffffffu, l, 16);
                if (g == 0) ml[warp * R + n * 8 + 2 * t + e] = make_float2(top[n][e], l);
            }
        __syncthreads();
        float* joined = reinterpret_cast<float*>(smem);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const uint32_t row = n * 8 + 2 * t + e;
                float m = kNone;
#pragma unroll
                for (int w = 0; w < kAttnWarps; ++w) m = fmaxf(m, ml[w * R + row].x);
                const float f = top[n][e] == kNone ? 0.0f : exp2f(top[n][e] - m) * down;
#pragma unroll
                for (int d = 0; d < 2 * NB; ++d) {
                    acc[d][n][e] *= f;
                    acc[d][n][e + 2] *= f;
                }
            }
        auto each = [&](auto use) {  // lane's four neighbouring values of every (row, block)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                    for (int b = 0; b < NB; ++b) use(n, e, b, (n * 8 + 2 * t + e) * Shape::dim + b * 32 + g * 4);
        };
        auto store = [&](uint32_t half) {
            each([&](int n, int e, int b, uint32_t at) {
                *reinterpret_cast<float4*>(joined + half * R * Shape::dim + at) =
                    make_float4(acc[2 * b][n][e], acc[2 * b][n][e + 2], acc[2 * b + 1][n][e], acc[2 * b + 1][n][e + 2]);
            });
        };
        if (warp >= 2) store(warp - 2);
        __syncthreads();
        if (warp < 2) {
            each([&](int n, int e, int b, uint32_t at) {
                const float4 f = *reinterpret_cast<const float4*>(joined + warp * R * Shape::dim + at);
                acc[2 * b][n][e] += f.x;
                acc[2 * b][n][e + 2] += f.y;
                acc[2 * b + 1][n][e] += f.z;
                acc[2 * b + 1][n][e + 2] += f.w;
            });
            store(warp);
        }
        __syncthreads();
        const bool whole = tile0 == 0 && tile1 == seq_tiles;
        const uint32_t slot = blockIdx.x * 2 + (tile0 == 0 ? 1 : 0);
        for (uint32_t x = tid; x < R * Shape::dim / 4; x += kAttnWarps * 32) {
            const uint32_t row = x / (Shape::dim / 4), col = (x % (Shape::dim / 4)) * 4;
            float m = kNone, l = 0.0f;
#pragma unroll
            for (int w = 0; w < kAttnWarps; ++w) m = fmaxf(m, ml[w * R + row].x);
#pragma unroll
            for (int w = 0; w < kAttnWarps; ++w)
                if (ml[w * R + row].x != kNone || ml[w * R + row].y != 0.0f) l += ml[w * R + row].y * (ml[w * R + row].x == kNone ? 1.0f : exp2f(ml[w * R + row].x - m));
            const float4 u = *reinterpret_cast<const float4*>(joined + row * Shape::dim + col);
            const float4 v = *reinterpret_cast<const float4*>(joined + (R + row) * Shape::dim + col);
            float4 o = make_float4(u.x + v.x, u.y + v.y, u.z + v.z, u.w + v.w);
            if (whole) {
                if (row < row_count) {
                    const float n = l == 0.0f ? 0.0f : 1.0f / l;
                    const uint32_t rr = row_first + row, i = rr / p.group;
                    float* dst = p.out + (size_t)(sq.row0 + i) * p.out_stride + (size_t)(head * p.group + (rr - i * p.group)) * Shape::dim + col;
                    dst[0] = o.x * n;
                    dst[1] = o.y * n;
                    dst[2] = o.z * n;
                    dst[3] = o.w * n;
                }
            } else {
                *reinterpret_cast<float4*>(p.part_o + ((size_t)slot * R + row) * Shape::dim + col) = o;
                if (col == 0) p.part_ml[(size_t)slot * R + row] = make_float2(m, l);
            }
        }
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
        f(kv_attention_kernel<K4, V4, B, N>, AttnShape<K4, V4, B, N>::smem);
        return true;
    };
    using std::integral_constant;
#define VX_ATTN_CASE(B, N) \
    if (nb == B && nt == N) return go(integral_constant<int, B>{}, integral_constant<int, N>{});
    VX_ATTN_CASE(2, 1)
    VX_ATTN_CASE(2, 2)
    VX_ATTN_CASE(2, 4)
    VX_ATTN_CASE(3, 1)
    VX_ATTN_CASE(3, 2)
    VX_ATTN_CASE(4, 1)
    VX_ATTN_CASE(4, 2)
    VX_ATTN_CASE(4, 4)
    VX_ATTN_CASE(8, 1)
    VX_ATTN_CASE(8, 2)
#undef VX_ATTN_CASE
    return false;
}

#define VX_ATTN_INSTANCE(K4, V4)                                                                                          \
    template <>                                                                                                           \
    vx_status kv_attention_setup<K4, V4>(uint32_t nb, uint32_t nt, int* per_sm, uint32_t* smem) {                         \
        cudaError_t e = cudaSuccess;                                                                                      \
        const bool known = attn_pick<K4, V4>(nb, nt, [&](auto kernel, uint32_t bytes) {                                   \
            *smem = bytes;                                                                                                \
            e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);                    \
            if (e == cudaSuccess)                                                                                         \
                e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(per_sm, kernel, kAttnWarps * 32, bytes);                \
        });                                                                                                               \
        VX_REQUIRE(known, VX_ERR_UNSUPPORTED, "attention: no kernel for heads of %u values", nb * 32);                    \
        VX_CUDA(e);                                                                                                       \
        return VX_OK;                                                                                                     \
    }                                                                                                                     \
    template <>                                                                                                           \
    vx_status kv_attention_launch<K4, V4>(uint32_t nb, uint32_t nt, uint32_t grid, cudaStream_t stream, const AttnParams& p) { \
        attn_pick<K4, V4>(nb, nt, [&](auto kernel, uint32_t bytes) { kernel<<<grid, kAttnWarps * 32, bytes, stream>>>(p); }); \
        VX_CUDA(cudaGetLastError());                                                                                      \
        return VX_OK;                                                                                                     \
    }

}  // namespace vx
