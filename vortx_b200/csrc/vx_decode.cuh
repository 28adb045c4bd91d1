// Device pieces shared by the decode-step kernels (quantised cache, attention over it, expert layer).
//
// Products of block-quantised codes with f32 vectors on the tensor cores, to f32 accuracy.  A code (-127..127 or
// -8..7) is exact in f16.  An f32 value x is scaled by a power of two that brings the largest of its group (a row of q, a few
// blocks of an expert layer's input) to [2^14, 2^15) and split into two f16 parts, hi = f16(x), lo = f16(x - hi).  From 2^-2 on
// that keeps 22 significant bits, half a step 2^-23 relative: values down to 2^-16 of the group's largest.  Below, lo is one
// of f16's small numbers and the error an absolute 2^-25: at most 2^-39 of the largest, so 2^-21 relative for a value 2^-18 of
// the largest, 2^-15 for one of 2^-24.  Products of a code and a part are exact in the f32 accumulator; the two parts'
// sums are added in f32.  One rounding to fewer bits than f32 is therefore made, 22 bits instead of 24 of x, next to sums
// whose own f32 rounding is of that order; of a value so small that it is more, the group's largest is in the same sum (unless its
// code is zero).
#pragma once

#include <cuda_fp16.h>

#include <cstdint>

#include "vx_internal.h"
#include "vx_sm100.cuh"

namespace vx {

using sm100::smem_addr;

// D = A B + D, A 16 x 16 (rows of codes), B 16 x 8, f16 in, f32 sums.
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// D = A B.
__device__ __forceinline__ void mma_f16_new(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}

// Four 8 x 16-byte matrices; lane l passes the row address of row l % 8 of matrix l / 8 and receives, of each matrix,
// the 4-byte word l % 4 of row l / 4.
__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async8(uint32_t dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ uint32_t lds32(uint32_t a) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
    return v;
}

__device__ __forceinline__ uint32_t h2_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ __half2 bits_h2(uint32_t u) { return *reinterpret_cast<__half2*>(&u); }

// Codes to f16 pairs.  A byte or nibble u (code + 128 or + 8) alone in the low bits of a half is the f16 number u 2^-24, or 16 u
// 2^-24 at bits 4..7: one byte permutation or logic operation.  One exact f16 multiply-add makes it code 2^-9, a normal number
// (the tensor cores align products by the exponent field, so the leading zeros of a small one would be lost bits).
// Putting u under the exponent of 1024 needs a mask and an exponent, two constants, and took a quarter more instructions
// (8 experts of 14336 x 4096: 209 us, so 197).
constexpr float kCodeUnits = 512.0f;  // of 2^-9 in 1
__device__ __forceinline__ uint32_t fma_h2(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t d;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
    return d;
}
// bytes (two of `w`, picked by `sel`, e.g. 0x4140 = bytes 0 and 1) that hold code + 128
__device__ __forceinline__ uint32_t f16_of_bytes(uint32_t w, uint32_t sel) {
    return fma_h2(__byte_perm(w, 0, sel), 0x78007800u, 0xb400b400u);  // 2^15, -128 2^-9
}
// nibbles at bits 0..3 and 16..19 that hold code + 8
__device__ __forceinline__ uint32_t f16_of_low_nibbles(uint32_t w) { return fma_h2(w & 0x000f000fu, 0x78007800u, 0xa400a400u); }  // 2^15, -8 2^-9
// nibbles at bits 4..7 and 20..23
__device__ __forceinline__ uint32_t f16_of_high_nibbles(uint32_t w) { return fma_h2(w & 0x00f000f0u, 0x68006800u, 0xa400a400u); }  // 2^11

// Splits a and b: hi = their f16 parts as a pair (a low), lo = what those miss.
__device__ __forceinline__ void split_f16(float a, float b, uint32_t* hi, uint32_t* lo) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    *hi = h2_bits(h);
    *lo = h2_bits(__floats2half2_rn(a - f.x, b - f.y));
}

// The power of two that brings `largest` (> 0, finite) to [2^14, 2^15); 1 for zero, infinity and NaN, and exponents
// are kept where the power and its inverse are both normal numbers.
__device__ __forceinline__ float lift(float largest) {
    const uint32_t e = (__float_as_uint(largest) >> 23) & 0xffu;
    if (largest == 0.0f || e == 0xffu) return 1.0f;
    const int want = 14 - ((int)e - 127);
    return __uint_as_float((uint32_t)(min(126, max(-113, want)) + 127) << 23);
}

// 2^v to 2^-22 relative; results below the smallest normal number are 0.
__device__ __forceinline__ float ex2(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}

// Whether this block is the last of `count` that get here with this counter; what the others wrote before is then
// visible.  The counter is zero again afterwards.
__device__ __forceinline__ bool last_of(uint32_t* counter, uint32_t count, uint32_t* shared) {
    __syncthreads();
    if (threadIdx.x == 0) {
        __threadfence();  // the block's writes, which the barrier has put before this
        *shared = atomicInc(counter, count - 1);
        __threadfence();
    }
    __syncthreads();
    return *shared == count - 1;
}

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
__device__ __forceinline__ float warp_add(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Programmatic dependent launch: the kernel's reads of what the previous kernel of the stream wrote come after
// pdl_wait; pdl_launch lets the next kernel's blocks start being scheduled.
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// Where value x (0..31) of a block lies in the 16 bytes (8 halves) that lane t = (x % 16) / 4 of a quad holds as its
// B operand: k-step x / 16, then the order in which the A operand's codes come out of a word.
__host__ __device__ constexpr int frag_lane(int x) { return (x % 16) / 4; }
__host__ __device__ constexpr int frag_half(bool four_bit, int x) {
    const int m = x % 4;
    return (x / 16) * 4 + (four_bit ? (m == 1 ? 2 : m == 2 ? 1 : m) : m);
}

// The A operand (two k-steps) of 16 rows x 32 codes of one block.  Q8_0 (bytes hold code + 128): r = words of (rows
// 0..7, codes 0..15), (rows 8..15, codes 0..15), (rows 0..7, codes 16..31), (rows 8..15, codes 16..31).
__device__ __forceinline__ void a_of_bytes(const uint32_t (&r)[4], uint32_t (&a)[2][4]) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        a[s][0] = f16_of_bytes(r[2 * s], 0x4140);
        a[s][1] = f16_of_bytes(r[2 * s + 1], 0x4140);
        a[s][2] = f16_of_bytes(r[2 * s], 0x4342);
        a[s][3] = f16_of_bytes(r[2 * s + 1], 0x4342);
    }
}
// Q4_0: r0 / r1 = the word (4 bytes, 8 codes) of a row 0..7 / 8..15.
__device__ __forceinline__ void a_of_nibbles(uint32_t r0, uint32_t r1, uint32_t (&a)[2][4]) {
    const uint32_t s0 = r0 >> 8, s1 = r1 >> 8;
    a[0][0] = f16_of_low_nibbles(r0);
    a[0][1] = f16_of_low_nibbles(r1);
    a[0][2] = f16_of_low_nibbles(s0);
    a[0][3] = f16_of_low_nibbles(s1);
    a[1][0] = f16_of_high_nibbles(r0);
    a[1][1] = f16_of_high_nibbles(r1);
    a[1][2] = f16_of_high_nibbles(s0);
    a[1][3] = f16_of_high_nibbles(s1);
}

// ------------------------------------------------------------------------------------------ quantised cache ----
// A page is tokens / 32 tiles; a tile has one record per head, and a record holds 32 tokens of that head: the keys'
// codes and scales, then the values' codes and scales, in the order in which the attention kernel's warps take them
// (see the two offset functions), so a record is copied to shared memory as it is, 16 bytes per lane, and every
// later read of it is a full, conflict-free vector.
constexpr uint32_t kTileTokens = 32;

__host__ __device__ constexpr uint32_t kv_code_bytes(bool four_bit, uint32_t blocks) { return blocks * (four_bit ? 512u : 1024u); }
__host__ __device__ constexpr uint32_t kv_part_bytes(bool four_bit, uint32_t blocks) { return kv_code_bytes(four_bit, blocks) + blocks * 64u; }

// Keys, codes: 16-byte rows (16 bytes of Q8_0 codes + 128, or a whole Q4_0 block) of 32 tokens one after the other.
// Offset of the 4-byte word that holds values 4 j .. 4 j + 3 (Q8_0, j < 8) or bytes 4 j .. 4 j + 3 (Q4_0, j < 4).
__host__ __device__ constexpr uint32_t k_word(bool four_bit, uint32_t block, uint32_t token, uint32_t j) {
    return four_bit ? (block * 32 + token) * 16 + j * 4 : ((block * 2 + j / 4) * 32 + token) * 16 + (j % 4) * 4;
}
__host__ __device__ constexpr uint32_t k_scale(uint32_t block, uint32_t token) { return block * 64 + ((token % 8) * 4 + token / 8) * 2; }
// Values, codes: token = t + 4 i + 16 s; lane 4 j + t of a warp takes values 4 j .. 4 j + 3 of its tokens.
// Q4_0: two bytes (four nibbles, code + 8) of a token; Q8_0: value 4 j is this byte (code + 128), the next three follow four
// bytes apart, so a word has one value of four tokens.
__host__ __device__ constexpr uint32_t v_word(bool four_bit, uint32_t block, uint32_t token, uint32_t j) {
    const uint32_t t = token % 4, i = (token / 4) % 4, s = token / 16;
    return four_bit ? block * 512 + (j * 4 + t) * 16 + s * 8 + i * 2 : block * 1024 + s * 512 + (j * 4 + t) * 16 + i;
}
__host__ __device__ constexpr uint32_t v_scale(uint32_t block, uint32_t token) {
    return block * 64 + ((token % 4) * 8 + (token / 16) * 4 + (token / 4) % 4) * 2;
}

struct KvGeometry {
    uint8_t* base;
    uint32_t pages, tiles_per_page, heads, blocks;
    uint32_t k4, v4;                   // keys / values in four bits
    uint32_t k_bytes, record_bytes;    // the keys' part, the whole record
};
// The rows of one call as the device sees them (see vx_kv_rows).
struct KvRows {
    const int32_t *table, *begin, *start;
    uint32_t max_pages, seqs, rows;
};
struct KvSeq {
    uint32_t row0, n;      // rows [row0, row0 + n) of the call
    uint32_t first;        // the token that row row0 is
    uint32_t start, end;   // tokens before the call's, and with them, as far as the page table reaches
};
// Whatever the three arrays hold, the rows of a sequence lie in [0, rows) and its tokens in the page table.
__device__ __forceinline__ KvSeq kv_seq(const KvRows& r, const KvGeometry& g, uint32_t s) {
    const int32_t a = r.begin[s], b = r.begin[s + 1], p = r.start[s];
    KvSeq q;
    q.row0 = (uint32_t)min(max(a, 0), (int32_t)r.rows);
    q.n = (uint32_t)(min(max(b, (int32_t)q.row0), (int32_t)r.rows)) - q.row0;
    const uint64_t room = (uint64_t)r.max_pages * g.tiles_per_page * kTileTokens;
    const uint64_t most = room < 0x7fffffe0ull ? room : 0x7fffffe0ull;
    const uint64_t s0 = (uint64_t)(uint32_t)max(p, 0);
    q.first = (uint32_t)s0;
    q.start = (uint32_t)(s0 < most ? s0 : most);
    const uint64_t e = s0 + q.n;
    q.end = (uint32_t)(e < most ? e : most);
    if (p < 0) q.end = q.start = 0, q.n = 0;  // a sequence without a place has no rows
    return q;
}
// The last s of [0, seqs) with at(s) <= x, at() not decreasing and at(0) <= x; all lanes of a warp take part.
template <class At>
__device__ __forceinline__ uint32_t warp_search(uint32_t seqs, uint32_t x, At at) {
    uint32_t lo = 0, hi = seqs;
    const uint32_t lane = threadIdx.x & 31;
    while (hi - lo > 1) {
        const uint32_t step = (hi - lo + 31) / 32, i = lo + lane * step;
        const uint32_t below = __ballot_sync(0xffffffffu, i < hi && at(i) <= x);
        lo += (below ? 31 - __clz(below) : 0) * step;
        hi = min(hi, lo + step);
    }
    return lo;
}
// The record of a tile of a sequence, or null where the page table names no page of the cache.
__device__ __forceinline__ uint8_t* kv_record(const KvRows& r, const KvGeometry& g, uint32_t seq, uint32_t tile, uint32_t head) {
    const uint32_t page = tile / g.tiles_per_page;
    if (page >= r.max_pages) return nullptr;
    const int32_t id = r.table[(size_t)seq * r.max_pages + page];
    if (id < 0 || (uint32_t)id >= g.pages) return nullptr;
    return g.base + (((size_t)id * g.tiles_per_page + (tile - page * g.tiles_per_page)) * g.heads + head) * g.record_bytes;
}

}  // namespace vx

struct vx_kv_cache {
    vx::KvGeometry g{};
    vx_qtype k_type = VX_Q8_0, v_type = VX_Q8_0;
    size_t head_dim = 0, page_tokens = 0, device_bytes = 0;
    int device = 0;
};

namespace vx {
// Launches a kernel whose blocks may be scheduled while the stream's previous kernel ends (it calls pdl_wait first).
template <class P>
cudaError_t launch_after(void (*kernel)(P), dim3 grid, uint32_t threads, uint32_t smem, cudaStream_t stream, const P& p, dim3 cluster = dim3(1)) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2]{};
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = 1;
    if (cluster.x * cluster.y * cluster.z > 1) {
        attr[1].id = cudaLaunchAttributeClusterDimension;
        attr[1].val.clusterDim.x = cluster.x;
        attr[1].val.clusterDim.y = cluster.y;
        attr[1].val.clusterDim.z = cluster.z;
        cfg.numAttrs = 2;
    }
    cfg.attrs = attr;
    return cudaLaunchKernelEx(&cfg, kernel, p);
}

// The host's checks of a vx_kv_rows and what the kernels get of it.
vx_status kv_rows_check(const char* who, const vx_kv_rows* rows, KvRows* out);
}  // namespace vx
