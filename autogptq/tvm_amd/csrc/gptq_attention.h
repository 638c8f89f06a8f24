// Device-side pieces shared by the attention kernels over a paged key/value cache, and their launchers.
//
// Rows.  The query heads that share a key/value head are rows of one matrix: token t of a request and head g of the group
// are row t * group + g, and a workgroup takes a tile of R consecutive rows of one request and one key/value head, so that
// every key and value is loaded once for the whole group.
//
// Keys.  A tile sees the keys [0, ns) (sinks that its window has left behind) and [lo, hi) of its request.  The two are
// walked as one list of n_seen keys; what single rows of the tile do not see in it is masked.  Nothing outside of the list
// is read: block table entries there may hold anything.  A short shared prefix may stand in front of the list, looked up in
// a table of its own.
//
// Parts.  The keys of a tile may be divided among workgroups.  Each leaves m, l and o of its part in the workspace.  Parts of few
// rows are joined by the workgroup that comes last, those of up to 128 by a launch of their own.
//
// Statistics.  Scores are kept in units of log2(e): p = 2^(c q.k - m) with c = scale * log2(e), m the row's reference, l the sum
// of p and o the sum of p v, all in 32 bits.  m is set `lift` below the running maximum, and raised, with o and l scaled down,
// only when a score passes it by `most`: most tiles of keys need no pass over o.  p is rounded to the cache's type for the matrix
// instruction.  bf16 has the exponents of 32 bits: every p keeps the relative rounding of the type.  fp16 keeps it from 2^-14 up
// and holds multiples of 2^-24 below, so its p are lifted to the upper end of the type: shares down to 2^-(14 + lift) of a row's
// largest have the type's relative rounding, smaller ones an error of at most 2^-(25 + lift) of the largest.  (Parts that are
// joined are of one type, hence of one lift, which o / l does not show.)
#pragma once
#include <hip/hip_runtime.h>

#include "gptq_device.h"

namespace gptq {

constexpr int kTileRows = 128;       // of a tile at most
constexpr int kMostKeys = 1 << 29;   // of a request, a prefix, a window: sums of positions and widths stay within 32 bits

struct AttentionParams {
    const void *q, *k, *v;
    void *out;
    const int32_t *tables, *starts, *contexts;
    const int32_t *prefix_blocks;
    int *counters;     // zero between calls
    float *stats, *parts;        // m and l, and o, of the parts of a shared prefix: [part][row of tokens * heads][2 or dim]
    float *own_stats, *own_parts;   // of a tile's own parts: as those, or (few-rows kernel) [place][row of the tile][2 or dim]
    int tokens, requests, heads, kv_heads, group, dim;
    int blocks, block_size, table_width;
    int window, sinks;
    int shared;        // 1: the launch computes the parts of a shared prefix of `prefix` keys
    int prefix;
    int front;         // keys of a prefix that stands in front of every list
    int tiles, splits, chunk;   // tiles (bound), parts of a tile at most, keys of a part
    int prefix_parts;  // parts of a shared prefix to be joined with a tile's own
    int team, most_units;       // few-rows kernel: workgroups of a key/value head, units of a tile at most
    long long q_token, q_head, head_stride, table_stride;   // in elements
    uint32_t block_step, slot_step;   // of a cache, in units of 16 bytes
    float c;
    uint32_t group_magic;    // x / group = x * magic >> 16 for x < group + kTileRows; 0: groups that are divided by
    int block_shift;         // log2(block_size), or -1
};

// x / group for the rows of a tile, counted from its first token's
__device__ __forceinline__ int tokens_of(const AttentionParams &p, int x)
{
    return p.group_magic ? (int)((uint32_t)x * p.group_magic >> 16) : x / p.group;
}

// A query tile: rows [row0, row0 + rows) of the request with the tokens [start, start + count), whose last one is at
// position context - 1.
struct QueryTile {
    int b, start, count, row0, rows;
    int position;      // of the request's first new token
    int front;         // the list of keys: [0, front) of a prefix, then [0, ns) and [lo, lo + seen - ns - front)
    int ns, lo, seen;
    int t0, t1;        // first and last token of the tile
    int g0;            // rows of the first token that belong to the tile before
};

// keys of a request that a table can name
__device__ __forceinline__ int held_keys(const AttentionParams &p)
{
    return (int)min((long long)p.table_width * p.block_size, (long long)kMostKeys);
}

// the rest of a tile whose request and rows are known
template <bool SHARED>
__device__ __forceinline__ void set_tile(const AttentionParams &p, QueryTile &q, int context)
{
    q.t0 = q.row0 / p.group;
    q.g0 = q.row0 - q.t0 * p.group;
    q.t1 = q.t0 + tokens_of(p, q.g0 + q.rows - 1);
    if (SHARED) {
        q.position = context, q.ns = 0, q.lo = 0, q.seen = q.front = context;
        return;
    }
    q.position = context - q.count;
    const int hi = max(min(min(context, q.position + q.t1 + 1), held_keys(p)), 0);
    q.lo = p.window > 0 ? min(max(q.position + q.t0 - p.window + 1, 0), hi) : 0;
    q.ns = min(p.sinks, q.lo);
    q.front = p.front;
    q.seen = q.front + q.ns + hi - q.lo;
}

// position of entry i of the list; entries of the front have negative ones
__device__ __forceinline__ int key_position(const QueryTile &q, int i)
{
    const int own = i - q.front;
    return own < q.ns ? own : own - q.ns + q.lo;
}

// What a row at position `pos` sees of a part of the list that ends at `end`: the entries below `high` that are not below
// `low`, and all below `free` (a prefix, sinks that the window has left behind, and what of the sinks it has not).
struct Sight {
    int low, high, free;
    __device__ __forceinline__ bool sees(int i) const { return (i < high) & ((i >= low) | (i < free)); }
};
__device__ __forceinline__ Sight sight(const AttentionParams &p, const QueryTile &q, int end, int pos)
{
    const int own = q.front + q.ns - q.lo;      // entry of position 0, were it in the window
    return {p.window > 0 ? pos - p.window + 1 + own : -kMostKeys, min(max(pos + 1 + own, q.front), end), max(q.front + q.ns, p.sinks + own)};
}

// whether every row from the tile's token at position `first` to the one at `last` sees entries [i0, i1) of the list
__device__ __forceinline__ bool all_see(const AttentionParams &p, const QueryTile &q, int i0, int i1, int first, int last)
{
    return i1 <= q.front || (key_position(q, i1 - 1) <= first &&
                             (p.window <= 0 || (i0 >= q.front + q.ns && key_position(q, i0) > last - p.window)));
}

// Where the row of entry i stands in a cache, in units of 16 bytes (head 0).  A block that the cache does not have counts
// as its first: the values are then undefined, the addresses are not.
__device__ __forceinline__ uint32_t key_row(const AttentionParams &p, const QueryTile &q, const int32_t *table, int i)
{
    const bool front = i < q.front;
    const uint32_t at = (uint32_t)(front ? i : key_position(q, i));
    const uint32_t j = p.block_shift >= 0 ? at >> p.block_shift : at / (uint32_t)p.block_size;
    const uint32_t slot = at - j * (uint32_t)p.block_size;
    uint32_t block = (uint32_t)(front ? p.prefix_blocks : table)[j];
    if (block >= (uint32_t)p.blocks) block = 0;
    return block * p.block_step + slot * p.slot_step;   // (the host has seen to it that no row passes 2^32)
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

// How far a score may pass a row's reference, and how far below the row's maximum the reference is set.  (fp16 holds 2^15.  A larger lift
// keeps smaller shares whole and raises references more often: prompts of 4096 tokens, 16 heads of 256, take 215, 217, 219, 222 and 231 us
// with 7, 9, 10, 11 and 13, and 243 with 15; 8192 of 32 heads of 128 600, 602, 602, 603, 615 and 626.)
template <typename E>
struct Shares {
    static constexpr float most = 8.0f, lift = 0.0f;
};
template <>
struct Shares<_Float16> {
    static constexpr float most = 15.0f, lift = 9.0f;
};

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

// Four values of a part, and its statistics.  Parts that a later launch reads need no way past the caches.
template <bool COHERENT>
__device__ __forceinline__ void put_part(float *to, f4 x)
{
    if constexpr (COHERENT) store_partial(to, x);
    else *(f4 *)to = x;
}
template <bool COHERENT>
__device__ __forceinline__ void put_stats(float *to, float m, float l)
{
    if constexpr (COHERENT) store_stats(to, m, l);
    else *(f2 *)to = (f2){m, l};
}

// row r of a tile: its token (in the request) and query head
__device__ __forceinline__ void token_head(const AttentionParams &p, const QueryTile &q, int h, int r, int &t, int &head)
{
    const int x = q.g0 + r, dt = tokens_of(p, x);
    t = q.t0 + dt;
    head = h * p.group + x - dt * p.group;
}
// ... and its row in the part arrays and the output: token * heads + head
__device__ __forceinline__ long long out_row(const AttentionParams &p, const QueryTile &q, int h, int r)
{
    int t, head;
    token_head(p, q, h, r, t, head);
    return (long long)(q.start + t) * p.heads + head;
}

// Zeros for the tokens that belong to no request (a step that is padded to a fixed size): those before `first` = starts[0] and from
// `last` = starts[requests] on, dealt to all threads of the launch.  (The two are asked for beside the lengths and used behind
// them: asked for alone they cost a small call 0.3 us, so nothing.)
__device__ __forceinline__ void clear_rest(const AttentionParams &p, int first, int last, long long thread, long long threads)
{
    first = min(max(first, 0), p.tokens), last = min(max(last, first), p.tokens);
    if (first == 0 && last == p.tokens) return;
    const long long token = (long long)p.heads * p.dim / 8;      // 16-byte chunks of one
    for (long long i = thread; i < token * (first + p.tokens - last); i += threads)
        ((u4 *)p.out)[i < token * first ? i : i + token * (last - first)] = (u4){0u, 0u, 0u, 0u};
}

// 4 results of a row as 4 values of the output's type, 8 bytes
template <typename E>
__device__ __forceinline__ void store_row4(void *out, long long at, f4 o)
{
    *(typename Vec<E>::e4 *)((E *)out + at) = __builtin_convertvector(o, typename Vec<E>::e4);
}

// Four values of a row with the row's statistics, and parts that join them: m = max m_i, l = sum l_i 2^(m_i - m), o likewise.
struct Sum {
    float m, l;
    f4 o;
    __device__ __forceinline__ void add(float mi, float li, f4 oi)
    {
        const float up = fmaxf(m, mi), to = reference(up), f = __builtin_amdgcn_exp2f(m - to), w = __builtin_amdgcn_exp2f(mi - to);
        m = up;
        l = f * l + w * li;
        o = f * o + w * oi;
    }
    __device__ __forceinline__ f4 result() const { return o * (l > 0.0f ? 1.0f / l : 0.0f); }
};
// The parts first, first + step, ... < count.  `stat` and `part` give the address of a part's statistics and of its four
// values; eight parts are asked for at a time.  Coherent: parts of other workgroups of this launch, past the caches.
template <bool COHERENT, typename Stat, typename Part>
__device__ __forceinline__ void add_parts(Sum &x, int first, int step, int count, Stat stat, Part part)
{
    for (int s0 = first; s0 < count; s0 += 8 * step) {
        f2 ml[8];
        f4 o[8];
#pragma unroll
        for (int u = 0; u < 8; u++) {
            const int s = min(s0 + u * step, count - 1);
            ml[u] = COHERENT ? load_stats(stat(s)) : *(const f2 *)stat(s);
            o[u] = COHERENT ? load_partial(part(s)) : *(const f4 *)part(s);
        }
#pragma unroll
        for (int u = 0; u < 8; u++)
            if (s0 + u * step < count) x.add(ml[u][0], ml[u][1], o[u]);
    }
}
// The parts of a shared prefix, which a launch before left.
__device__ __forceinline__ void add_prefix(const AttentionParams &p, Sum &x, long long at, int d)
{
    const long long all = (long long)p.tokens * p.heads;
    add_parts<false>(x, 0, 1, p.prefix_parts, [&](int s) { return p.stats + 2 * (s * all + at); },
                     [&](int s) { return p.parts + (s * all + at) * p.dim + d; });
}

// Joins the `parts` parts of a tile, in their order, behind those of a shared prefix.  place(part, row of the tile) is a row of
// own_stats and own_parts.  Where a tile has few rows several threads share a value's parts; where it has many a thread takes
// two values' at a time, four parts each.  `lds`: THREADS Sums; ITEMS: the most quads of values that a tile of the kernel has.
template <typename E, int THREADS, int ITEMS, typename Place>
__device__ void join_parts(const AttentionParams &p, const QueryTile &q, int h, int parts, void *lds, Place place)
{
    const int quads = p.dim / 4, items = q.rows * quads;
    if (ITEMS > 2 * THREADS && items >= 2 * THREADS) {
        for (int i = threadIdx.x; i < items; i += 2 * THREADS) {
            Sum x[2];
            int r[2], d[2];
            long long at[2];
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const int item = min(i + u * THREADS, items - 1);       // (the last one twice, if there is no other)
                r[u] = item / quads, d[u] = (item - r[u] * quads) * 4, at[u] = out_row(p, q, h, r[u]);
                x[u] = {kNone, 0.0f, {0.0f, 0.0f, 0.0f, 0.0f}};
                add_prefix(p, x[u], at[u], d[u]);
            }
            for (int s0 = 0; s0 < parts; s0 += 4) {
                f2 ml[2][4];
                f4 o[2][4];
#pragma unroll
                for (int s = 0; s < 4; s++)
#pragma unroll
                    for (int u = 0; u < 2; u++) {
                        if (s0 + s >= parts) continue;
                        const long long from = place(s0 + s, r[u]);
                        ml[u][s] = load_stats(p.own_stats + 2 * from);
                        o[u][s] = load_partial(p.own_parts + from * p.dim + d[u]);
                    }
#pragma unroll
                for (int s = 0; s < 4; s++)
#pragma unroll
                    for (int u = 0; u < 2; u++)
                        if (s0 + s < parts) x[u].add(ml[u][s][0], ml[u][s][1], o[u][s]);
            }
#pragma unroll
            for (int u = 0; u < 2; u++) store_row4<E>(p.out, at[u] * p.dim + d[u], x[u].result());
        }
        return;
    }
    Sum *half_way = (Sum *)lds;
    int teams = 1;
    while (8 * teams < parts && 2 * teams * items <= THREADS) teams *= 2;
    const int team = teams > 1 ? threadIdx.x / items : 0;
    for (int i = threadIdx.x - team * items; i < items && team < teams; i += teams > 1 ? items : THREADS) {
        const int r = i / quads, d = (i - r * quads) * 4;
        const long long at = out_row(p, q, h, r);
        Sum x = {kNone, 0.0f, {0.0f, 0.0f, 0.0f, 0.0f}};
        if (team == 0) add_prefix(p, x, at, d);
        add_parts<true>(x, team, teams, parts, [&](int s) { return p.own_stats + 2 * place(s, r); },
                        [&](int s) { return p.own_parts + place(s, r) * p.dim + d; });
        if (teams > 1) half_way[threadIdx.x] = x;
        else store_row4<E>(p.out, at * p.dim + d, x.result());
    }
    if (teams > 1) {
        __syncthreads();
        if ((int)threadIdx.x < items) {
            Sum x = half_way[threadIdx.x];
            for (int t = 1; t < teams; t++) {
                const Sum y = half_way[t * items + threadIdx.x];
                x.add(y.m, y.l, y.o);
            }
            const int r = threadIdx.x / quads, d = (threadIdx.x - r * quads) * 4;
            store_row4<E>(p.out, out_row(p, q, h, r) * p.dim + d, x.result());
        }
    }
}

int launch_attention_few(const AttentionParams &p, int type, int rt, void *stream);
int launch_attention_tile(const AttentionParams &p, int type, void *stream);

}  // namespace gptq
