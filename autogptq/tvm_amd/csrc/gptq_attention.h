// Device-side pieces shared by the attention kernels over a paged key/value cache, and their launchers.
//
// Rows.  The query heads that share a key/value head are rows of one matrix: token t of a request and head g of the group
// are row t * group + g, and a workgroup takes a tile of R consecutive rows of one request and one key/value head, so that
// every key and value is loaded once for the whole group.  Request b of B owns the tiles from
//   first_tile(b) = floor(starts[b] * group / R) + b:
// the floors of two neighbours lie at least floor(rows / R) apart, and the + b adds the tile of a remainder.  The bound
// floor(tokens * group / R) + B on the number of tiles, and the request of a tile, follow without any sum over requests;
// tiles past a request's rows leave at once.
//
// Keys.  A tile sees the keys [0, ns) (sinks that its window has left behind) and [lo, hi) of its request.  The two are
// walked as one list of n_seen keys; what single rows of the tile do not see in it is masked.  Nothing outside of the list
// is read: block table entries there may hold anything.
//
// Statistics.  Scores are kept in units of log2(e): p = 2^(c q.k - m) with c = scale * log2(e), m the running maximum, l
// the sum of p and o the sum of p v, all in 32 bits.  p is rounded to the cache's type for the matrix instruction (the
// largest p of a row is 1, so its error is at most the rounding of that type, relative to the largest share of a row).
// m is raised, and o and l scaled down, only when a score passes it by 2^8: until then p is at most 2^8, far from the
// largest fp16 and with the same relative rounding, and most tiles of keys need no pass over o.
#pragma once
#include <hip/hip_runtime.h>

#include "gptq_device.h"

namespace gptq {

constexpr int kMostKeys = 1 << 30;   // of a request: sums of positions and widths stay within 32 bits

struct AttentionParams {
    const void *q, *k, *v;
    void *out;
    const int32_t *tables, *starts, *contexts;
    int *counters;     // one per (tile, key/value head): zero between calls
    float *stats;      // [slot][row of tokens * heads][2]: m and l of a part
    float *parts;      // [slot][row][dim]: o of a part
    int tokens, requests, heads, kv_heads, group, dim;
    int blocks, block_size, table_width;
    int window, sinks;
    int shared;        // 1: every token sees the first `prefix` keys of the one table row, and the parts stay parts
    int prefix;
    int tiles, splits, chunk;   // tiles (bound), parts of a tile at most, keys of a part
    int first_slot;    // parts of the shared prefix that stand before a tile's own
    long long q_token, q_head, block_stride, slot_stride, head_stride, table_stride;   // in elements
    float c;
};

// A query tile: rows [row0, row0 + rows) of the request with the tokens [start, start + count), whose last one is at
// position context - 1.
struct QueryTile {
    int b, start, count, row0, rows;
    int position;      // of the request's first new token
    int ns, lo, seen;  // the list of keys: [0, ns) and [lo, lo + seen - ns)
    int t0, t1;        // first and last token of the tile
};

template <int R>
__device__ __forceinline__ bool find_tile(const AttentionParams &p, int tile, QueryTile &q)
{
    const int lane = threadIdx.x & 63;
    int context;
    if (p.shared) {
        q.b = 0, q.start = 0, q.count = p.tokens, q.row0 = tile * R;
        context = p.prefix;
    } else {
        int before = 0;
        if (p.requests > 1) {
            for (int b0 = 0; b0 < p.requests; b0 += 64) {
                const int b = b0 + lane;
                const bool there = b < p.requests;
                const int s = there ? min(max(p.starts[b], 0), p.tokens) : 0;
                before += __popcll(__ballot(there && (int)((uint32_t)s * (uint32_t)p.group / R) + b <= tile));
            }
            before = max(before, 1) - 1;
        }
        q.b = __builtin_amdgcn_readfirstlane(before);
        // (what the tensors say is cut to what the other arguments allow: wrong lengths give wrong sums, not wrong addresses)
        q.start = min(max(p.starts[q.b], 0), p.tokens);
        q.count = min(max(p.starts[q.b + 1] - q.start, 0), p.tokens - q.start);
        context = p.contexts[q.b];
        q.row0 = (tile - ((int)((uint32_t)q.start * (uint32_t)p.group / R) + q.b)) * R;
    }
    const int all = q.count * p.group;
    if (q.row0 < 0 || q.row0 >= all) return false;
    q.rows = min(R, all - q.row0);
    q.t0 = q.row0 / p.group;
    q.t1 = (q.row0 + q.rows - 1) / p.group;
    if (p.shared) {
        q.position = context, q.ns = 0, q.lo = 0, q.seen = context;
        return true;
    }
    q.position = context - q.count;
    const int held = (int)min((long long)p.table_width * p.block_size, (long long)kMostKeys);
    const int hi = max(min(min(context, q.position + q.t1 + 1), held), 0);
    q.lo = p.window > 0 ? min(max(q.position + q.t0 - p.window + 1, 0), hi) : 0;
    q.ns = min(p.sinks, q.lo);
    q.seen = q.ns + hi - q.lo;
    return true;
}

// The keys of a part: [begin, end) of the list, and how many parts the tile has.  A list that is longer than the host
// expected (splits * chunk) has longer parts.
__device__ __forceinline__ int tile_parts(const AttentionParams &p, int seen, int unit, int &chunk)
{
    chunk = max(p.chunk, ((seen + p.splits - 1) / p.splits + unit - 1) / unit * unit);
    return max(1, (seen + chunk - 1) / chunk);
}

// position of entry i of the list
__device__ __forceinline__ int key_position(const QueryTile &q, int i) { return i < q.ns ? i : i - q.ns + q.lo; }

// Whether a row at position `pos` sees entry i of the list, whose part ends at `end`.  (Without branches: every entry of a
// mixed tile is asked.)
__device__ __forceinline__ bool sees(const AttentionParams &p, const QueryTile &q, int i, int end, int pos)
{
    const int at = key_position(q, i);
    const int oldest = p.window > 0 ? pos - p.window : -1;      // the newest position that is no longer in the window
    const bool seen = (at <= pos) & ((at > oldest) | (at < p.sinks));
    return (i < end) & (seen | (p.shared != 0));
}

// where the row of key position `at` stands in a cache, in units of 16 bytes (head 0).  A block that the cache does not
// have counts as its first: the values are then undefined, the addresses are not.
__device__ __forceinline__ uint32_t key_row(const AttentionParams &p, const int32_t *table, int at)
{
    const uint32_t j = (uint32_t)at / (uint32_t)p.block_size;
    const uint32_t slot = (uint32_t)at - j * (uint32_t)p.block_size;
    uint32_t block = (uint32_t)table[j];
    if (block >= (uint32_t)p.blocks) block = 0;
    return (uint32_t)(((unsigned long long)block * (unsigned long long)p.block_stride + slot * (unsigned long long)p.slot_stride) >> 3);
}

// fp16 or bf16 operands of the matrix instructions
template <typename E>
struct Vec {
    typedef E e2 __attribute__((ext_vector_type(2)));
    typedef E e4 __attribute__((ext_vector_type(4)));
    typedef E e8 __attribute__((ext_vector_type(8)));
};
typedef float f2 __attribute__((ext_vector_type(2)));
typedef float f8 __attribute__((ext_vector_type(8)));
typedef float f16 __attribute__((ext_vector_type(16)));

__device__ __forceinline__ f4 mfma16(Vec<_Float16>::e8 a, Vec<_Float16>::e8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f4 mfma16(Vec<__bf16>::e8 a, Vec<__bf16>::e8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f16 mfma32(Vec<_Float16>::e8 a, Vec<_Float16>::e8 b, f16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f16 mfma32(Vec<__bf16>::e8 a, Vec<__bf16>::e8 b, f16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }

// Over the lanes l and l ^ 32, or all lanes of equal l % 16: lanes hand a register over without LDS.  The swap exchanges the upper
// half (every odd 16) of one register with the lower half (even 16) of another.  (The results are named before they are read as
// floats: the compiler takes element 0 for a bit cast of any element of a vector.)
__device__ __forceinline__ f2 swap_halves(float x)
{
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const uint32_t a = r[0], b = r[1];
    return (f2){__builtin_bit_cast(float, a), __builtin_bit_cast(float, b)};
}
__device__ __forceinline__ f2 swap_quarters(float x)
{
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const uint32_t a = r[0], b = r[1];
    return (f2){__builtin_bit_cast(float, a), __builtin_bit_cast(float, b)};
}
__device__ __forceinline__ float max_halves(float x) { const f2 r = swap_halves(x); return fmaxf(r[0], r[1]); }
__device__ __forceinline__ float add_halves(float x) { const f2 r = swap_halves(x); return r[0] + r[1]; }
__device__ __forceinline__ float max_quarters(float x) { const f2 r = swap_quarters(max_halves(x)); return fmaxf(r[0], r[1]); }
__device__ __forceinline__ float add_quarters(float x) { const f2 r = swap_quarters(add_halves(x)); return r[0] + r[1]; }

constexpr float kNone = -__builtin_inff();
// the reference of a row that has seen nothing yet (its p are 2^(-inf) = 0)
__device__ __forceinline__ float reference(float m) { return m == kNone ? 0.0f : m; }

__device__ __forceinline__ void store_stats(float *dst, float m, float l)
{
    const f2 v = {m, l};
    __hip_atomic_store((unsigned long long *)dst, __builtin_bit_cast(unsigned long long, v), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ f2 load_stats(const float *src)
{
    return __builtin_bit_cast(f2, __hip_atomic_load((const unsigned long long *)src, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
}

// row r of a tile -> row of the part arrays and of the output: token * heads + head
__device__ __forceinline__ long long out_row(const AttentionParams &p, const QueryTile &q, int h, int r)
{
    const int row = q.row0 + r, t = row / p.group, g = row - t * p.group;
    return (long long)(q.start + t) * p.heads + h * p.group + g;
}

// 4 results of a row as 4 values of the output's type, 8 bytes
template <typename E>
__device__ __forceinline__ void store_row4(void *out, long long at, f4 o)
{
    *(typename Vec<E>::e4 *)((E *)out + at) = __builtin_convertvector(o, typename Vec<E>::e4);
}

// Whether this workgroup joins the parts of its tile: the one that is last, or the only one (then behind a shared prefix).
__device__ __forceinline__ bool last_part(const AttentionParams &p, int counter, int parts, int *flag)
{
    if (parts > 1) return arrive_last(p.counters + counter, parts, flag);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // (the caller's barrier follows)
    return true;
}

// The last workgroup of a tile joins its parts, in their order: m = max m_i, l = sum l_i 2^(m_i - m), o likewise.
// `weights`: LDS for rows * slots floats (at most kJoinWeights; longer lists go through it in rounds of rows).
constexpr int kJoinWeights = 4096;
template <typename E, int THREADS>
__device__ void join_parts(const AttentionParams &p, const QueryTile &q, int h, int slots, float *weights)
{
    const long long all = (long long)p.tokens * p.heads;
    const int quads = p.dim / 4;
    const int round = max(1, min(q.rows, kJoinWeights / slots));
    for (int r0 = 0; r0 < q.rows; r0 += round) {
        const int rows = min(round, q.rows - r0);
        __syncthreads();
        // 16 lanes a row
        for (int r = threadIdx.x / 16; r < rows; r += THREADS / 16) {
            const long long at = out_row(p, q, h, r0 + r);
            float m = kNone, l = 0.0f;
            for (int s = threadIdx.x % 16; s < slots; s += 16) m = fmaxf(m, load_stats(p.stats + 2 * (s * all + at))[0]);
            for (int d = 8; d >= 1; d /= 2) m = fmaxf(m, __shfl_xor(m, d, 16));
            const float ref = reference(m);
            for (int s = threadIdx.x % 16; s < slots; s += 16) {
                const f2 ml = load_stats(p.stats + 2 * (s * all + at));
                const float w = __builtin_amdgcn_exp2f(ml[0] - ref);
                weights[r * slots + s] = w;
                l += w * ml[1];
            }
            for (int d = 8; d >= 1; d /= 2) l += __shfl_xor(l, d, 16);
            const float inv = l > 0.0f ? 1.0f / l : 0.0f;
            for (int s = threadIdx.x % 16; s < slots; s += 16) weights[r * slots + s] *= inv;
        }
        __syncthreads();
        for (int i = threadIdx.x; i < rows * quads; i += THREADS) {
            const int r = i / quads, d = (i - r * quads) * 4;
            const long long at = out_row(p, q, h, r0 + r);
            f4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
            for (int s = 0; s < slots; s++) {
                const float w = weights[r * slots + s];
                const f4 x = load_partial(p.parts + (s * all + at) * p.dim + d);
#pragma unroll
                for (int e = 0; e < 4; e++) o[e] += w * x[e];
            }
            store_row4<E>(p.out, at * p.dim + d, o);
        }
    }
}

// rows_of_a_wave = 16 * RT rows of a tile; dims: the compiled width (64, 128 or 256) that covers dim
int launch_attention_few(const AttentionParams &p, int type, int rt, void *stream);
int launch_attention_tile(const AttentionParams &p, int type, void *stream);
constexpr int kTileRows = 128;

}  // namespace gptq
