// Attention over a paged cache for few rows a request: single tokens, drafts of a few, small groups of shared heads.
//
// What bounds it: memory.  Every visible key and value is read once (4 dim bytes in all), for 4 dim flops a row, and a tile
// has 16 RT rows.  So the kernel is a stream: four waves of a workgroup take every fourth block of 32 keys of the part and
// load keys and values straight into the registers of the matrix instructions, past LDS and without a barrier, the next
// 32 keys' loads in flight while the present ones are used.  (LDS holds the places of a wave's rows, and the waves' sums at the end.)
//
//   S^T[key, row] = K Q^T   keys are rows of the A operand: lane (i, g) = (lane % 16, lane / 16) loads 16 bytes of key i at
//                           dims 32 s + 8 g; a result lane holds for its row i the keys 4 g .. 4 g + 3
//   O^T[dim, row] += V^T P^T  the sum over keys may run in any order: lane group g takes the keys 4 g .. 4 g + 3 of both
//                           16-key halves, exactly those whose p it already holds, so p goes from the first product's
//                           result to the second's operand without leaving the lane.  V is loaded as it lies, whole rows
//                           (lane i: dims 8 i .. 8 i + 7 of the eight keys of its g), and turned in registers: half of
//                           two keys' dwords by one byte permute.  Operand row i of tile t is then dim 8 i + t, and a
//                           result lane holds eight neighbouring dims of a row.
//
// The division.  One to four workgroups fill a CU's registers, so a grid with a workgroup for every part that
// a request might have spends its time on those that find none (16 contexts of up to 32768 tokens: 146 us, with the
// division below 70).  Instead a head has `team` workgroups, as many as run at once, and each takes the same number of units
// of up to 256 keys of the requests' tiles, one after the other, in the order of the requests: a workgroup ends one tile, takes
// whole ones and begins another, and leaves at most two parts.  Every wave finds its place from the requests' lengths by
// itself, 64 requests at a time.
//
// Measured (32 heads in groups of 4, dim 128): 16 contexts of 32768 363 us, 5.9 TB/s of keys and values (a plain read of as much: 7.06);
// 64 of up to 32768 under a window of 4096 72.5 us; one of 512 8.5 us, a chain of reads of about 1 us each (lengths, table, keys, values, parts).
//
// A cache in MXFP4 (MX).  The same division and products; a row is dim / 2 bytes of codes and its groups' powers of two, which one
// instruction turns into two values each, exactly, so that the operands are what a cache of 16-bit values with the same contents has.  A
// quarter of the bytes at the same number of steps: what was hidden behind the stream now shows, so scales and places go through lists in
// LDS (one request for 64 keys in place of four lanes' reads of each), and every load stands a step or two ahead.  Measured as above: 16
// contexts of 32768 108 us, 5.3 TB/s of codes and scales.  It is not the conversions or the depth that bound it: with the loads alone it
// takes 106, and a plain kernel whose workgroups stream blocks of their own reaches 6.0 TB/s in whatever order.  64 under a window 26 us, one of 512
// 7.4, 24 requests of 5 tokens of 64 dims behind up to 6001 14.5 (a chain again).
#pragma once
#include "gptq_attention.h"
#include "gptq_mx.h"

#include <type_traits>

namespace gptq {

constexpr int kFewWaves = 4, kFewUnit = 256;

// Requests [base, base + 64), one a lane.
struct Requests {
    int start, count, context;
    int units, keys;       // of a tile: units, and the keys of one
    int total;             // units of all its tiles
};
template <int R, bool MX>
__device__ __forceinline__ Requests look_at(const AttentionParams &p, int base)
{
    // what the tensors say is cut to what the other arguments allow: wrong lengths give wrong sums, not wrong addresses
    const int b = base + (threadIdx.x & 63), last = p.requests - 1;
    Requests r;
    r.start = min(max(p.starts[min(b, last)], 0), p.tokens);
    r.count = min(max(p.starts[min(b, last) + 1] - r.start, 0), p.tokens - r.start);
    r.context = p.contexts[min(b, last)];
    if (b > last) r.count = 0;
    // the keys that any of its tokens sees: no tile's list is longer
    const int hi = max(min(r.context, held_keys(p)), 0);
    const int lo = p.window > 0 ? min(max(r.context - r.count - p.window + 1, 0), hi) : 0;
    const int seen = p.front + min(p.sinks, lo) + hi - lo;
    r.units = min(max(1, MX ? (seen + (1 << p.unit_bits) - 1) >> p.unit_bits : (seen + kFewUnit - 1) / kFewUnit), p.most_units);
    r.keys = max(32, ((seen + r.units - 1) / r.units + 31) / 32 * 32);
    const int tiles = (int)(((uint32_t)r.count * (uint32_t)p.group + R - 1) / R);
    r.total = MX && p.few_rows && tiles > 1 ? 0 : tiles * r.units;
    return r;
}
// DP: compiled width, the dims past p.dim do not count; FULL: there are none; RT: 16-row operands a wave holds; SHARED: the parts of a
// shared prefix; MX: a cache in MXFP4
template <typename E, int DP, bool FULL, int RT, bool SHARED, bool MX>
__global__ __launch_bounds__(64 * kFewWaves, few_resident(RT, DP, MX)) void attention_few_kernel(const AttentionParams given)
{
    typedef typename Vec<E>::e8 e8;
    constexpr int R = 16 * RT, NW = kFewWaves;
    constexpr int KS = DP / 32;                    // matrix instructions along dim for S
    constexpr int FIRST = DP == 64 ? 0 : KS / 2;   // the first of them that may hold dims past p.dim (wider kernels take dims above DP / 2)
    constexpr int VE = DP >= 128 ? 8 : DP / 16;    // dims a lane loads of a value row at a time
    constexpr int VH = DP / 16 / VE;               // ... that many times
    constexpr int VW = VE / 2;                     // dwords of that
    constexpr int OD = DP + 4;                     // row of O in LDS
    __shared__ uint32_t list[MX ? 1 : NW][2][64];
    __shared__ float stat_m[NW][16 * RT], stat_l[NW][16 * RT];
    __shared__ __align__(16) float join[NW * 16 * OD];
    __shared__ int flag;

    // neighbours take different heads: they go to the compute dies in turn, and a head's workgroups to the same one
    const int h = blockIdx.x % given.kv_heads, member = blockIdx.x / given.kv_heads;
    // this workgroup's units [at, stop), and the 64 requests that the first of them lies in or behind
    int at = 0, stop = 1, share = 1, base = 0, before = 0, upto = 0;
    Requests look = {};
    if (!SHARED) {
        look = look_at<R, MX>(given, 0);
        clear_rest(given, given.starts[0], given.starts[given.requests], blockIdx.x * (64ll * kFewWaves) + threadIdx.x, gridDim.x * (64ll * kFewWaves));
        upto = sum_upto(look.total);
        int total = __builtin_amdgcn_readlane(upto, 63), most = 0;       // units in all, and of a tile at most
        if (MX) most = max_lanes(look.total ? look.units : 0);
        for (int b = 64; b < given.requests; b += 64) {
            const Requests x = look_at<R, MX>(given, b);
            if (MX) most = max(most, max_lanes(x.total ? x.units : 0));
            total += __builtin_amdgcn_readlane(sum_upto(x.total), 63);
        }
        // (Whole tiles of two units rather than their halves, once every CU has a workgroup: the second unit costs less than
        // the join.  32 contexts of 300 tokens, 8 heads: 12.0 us, in halves 13.9; 4 of 512, where CUs are left, 10.4 in halves.)
        share = max((total + given.team - 1) / given.team, total * given.kv_heads > 256 && total <= 2 * given.requests ? 2 : 1);
        if constexpr (MX) {
            // A part costs a workgroup some 6 us around its keys, 256 of them 1.2 (a quarter of the bytes, but as many steps as of a cache in
            // 16 bits), and its join a tenth: fewer and longer parts where a tile has many units, more so once memory is the
            // bound, and whole tiles where each CU has two of them.  (8 key/value heads, us with the shortest parts and so: 1
            // context of 32768 29.2 / 17.6, of 8192 12.4 / 11.2; 4 of 32768 38.7 / 33.0, 16 of 8192 34.4 / 31.8; 64 of 1024 19.7 / 16.4.)
            const int tile_units = (total + given.requests - 1) / given.requests;
            int least = (int)__builtin_sqrtf((float)most * (1.0f / 6.0f));
            if ((long long)total * given.kv_heads >= 4096 && tile_units >= 8) least = max(least, 8);
            if ((long long)given.requests * given.kv_heads >= 512 && tile_units <= 4) least = max(least, tile_units);
            share = max(share, least);
        }
        at = member * share;
        stop = min(at + share, total);
        if (at >= stop) return;
    }
    for (;;) {
        // The arguments, and what follows from the lane, are taken anew for every part: kept in registers over all of them
        // they cost 20 vector registers and some 90 spilled scalar ones.  (The compiler cannot see through the two values.)
        size_t first_argument = 0;
        int thread = threadIdx.x;
        asm volatile("" : "+s"(first_argument), "+v"(thread));
        const int lane = thread & 63, i16 = lane & 15, g = lane >> 4;
        const int wave = __builtin_amdgcn_readfirstlane(thread >> 6);
        const AttentionParams &p = *(const AttentionParams *)((const __attribute__((address_space(4))) char *)__builtin_amdgcn_kernarg_segment_ptr() + first_argument);
        const int dim = FULL ? DP : p.dim;
        const char *kbase = (const char *)p.k + (long long)h * p.head_stride * (MX ? 1 : 2);
        const char *vbase = (const char *)p.v + (long long)h * p.head_stride * (MX ? 1 : 2);
        // a tile and a part [begin, end) of its list; the tile's parts belong to the members from `first` on
        QueryTile q;
        int begin, end, first = member, parts = 1, context = p.prefix, keys = p.chunk;
        if (SHARED) {
            q.b = 0, q.start = 0, q.count = p.tokens, q.row0 = member * R;
            begin = blockIdx.y, end = begin + 1;
            at = stop;
        } else {
            while (at - before >= __builtin_amdgcn_readlane(upto, 63)) {
                before += __builtin_amdgcn_readlane(upto, 63);
                base += 64;
                look = look_at<R, MX>(p, base);
                upto = sum_upto(look.total);
            }
            const int owner = __popcll(__ballot(upto <= at - before));
            const int units = __builtin_amdgcn_readlane(look.units, owner);
            keys = __builtin_amdgcn_readlane(look.keys, owner);
            q.b = base + owner;
            q.start = __builtin_amdgcn_readlane(look.start, owner);
            q.count = __builtin_amdgcn_readlane(look.count, owner);
            context = __builtin_amdgcn_readlane(look.context, owner);
            begin = at - before - (__builtin_amdgcn_readlane(upto, owner) - __builtin_amdgcn_readlane(look.total, owner));
            const int tile = begin / units;
            q.row0 = tile * R;
            begin -= tile * units;
            end = min(units, begin + stop - at);
            first = (at - begin) / share;
            parts = (at - begin + units - 1) / share - first + 1;
            at += end - begin;
        }
        q.rows = min(R, q.count * p.group - q.row0);
        set_tile<SHARED>(p, q, context);
        begin = min(begin * keys, q.seen), end = min(end * keys, q.seen);
        const int32_t *table = p.tables + (long long)q.b * p.table_stride;
        // blocks of 32 keys: a wave takes every fourth, and looks two of its own up at a time, one a half of its lanes (past
        // the end: the last key's row again)
        const int blocks = (end - begin + 31) / 32, busy = min(blocks, NW);   // ... waves that have keys
        auto look_up = [&](int n) { return key_row(p, q, table, min(begin + (n + (lane >> 5) * NW) * 32 + (lane & 31), end - 1)); };
        uint32_t next = 0;
        if (!MX && wave < blocks) next = look_up(wave);

        // the query rows as B operands, and what they see
        e8 qf[RT][KS];
        Sight my[RT];
    #pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            int t, hg;
            token_head(p, q, h, min(16 * rt + i16, q.rows - 1), t, hg);
            my[rt] = sight(p, q, end, q.position + t);
            const char *src = (const char *)p.q + ((long long)(q.start + t) * p.q_token + (long long)hg * p.q_head) * 2;
    #pragma unroll
            for (int s = 0; s < KS; s++) {
                const int d = !MX ? 32 * s + 8 * g : DP == 64 ? 16 * g + 8 * s : 128 * (s / 4) + 32 * g + 8 * (s % 4);
                u4 x = {0u, 0u, 0u, 0u};
                if (d < dim) x = *(const u4 *)(src + d * 2);
                qf[rt][s] = __builtin_bit_cast(e8, x);
            }
        }

        float m[RT], l[RT];
        f4 o[RT][VH][VE];
    #pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            m[rt] = kNone, l[rt] = 0.0f;
    #pragma unroll
            for (int vh = 0; vh < VH; vh++)
    #pragma unroll
                for (int t = 0; t < VE; t++) o[rt][vh][t] = (f4){0.0f, 0.0f, 0.0f, 0.0f};
        }

        // (Dims past p.dim: of keys their lanes load nothing and hold zeros, since an infinity times the query's zeros would be a NaN;
        // of values they are the last ones again, and reach dims of o that are not stored.)
        u4 kr[2][KS];
        if constexpr (!FULL && !MX) {
#pragma unroll
            for (int a = 0; a < 2; a++)
#pragma unroll
                for (int s = FIRST; s < KS; s++) kr[a][s] = (u4){0u, 0u, 0u, 0u};
        }
        uint32_t vr[8][VH][VW];
        auto load_keys = [&](const uint32_t *rows) {
#pragma unroll
            for (int a = 0; a < 2; a++) {
                const char *src = kbase + (unsigned long long)rows[16 * a + i16] * 16;
#pragma unroll
                for (int s = 0; s < KS; s++) {
                    if (FULL || s < FIRST || 32 * s + 8 * g < dim) kr[a][s] = *(const u4 *)(src + (32 * s + 8 * g) * 2);
                }
            }
        };
        auto load_values = [&](const uint32_t *rows) {
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const char *src = vbase + (unsigned long long)rows[16 * (j / 4) + 4 * g + j % 4] * 16;
#pragma unroll
                for (int vh = 0; vh < VH; vh++) {
                    const char *from = src + min(128 * vh + VE * i16, dim - VE) * 2;
                    if constexpr (VW == 4) {
                        const u4 x = *(const u4 *)from;
#pragma unroll
                        for (int w = 0; w < 4; w++) vr[j][vh][w] = x[w];
                    } else {
                        const u2 x = *(const u2 *)from;
#pragma unroll
                        for (int w = 0; w < 2; w++) vr[j][vh][w] = x[w];
                    }
                }
            }
        };
        auto hand_over = [&]() {   // what lanes of this wave wrote to LDS is there for the others of it
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        };

        if constexpr (MX) {
            // Keys and values are codes.  A lane's of a key are the groups g and 4 + g (half of one at rows of two), which lie side by side: the
            // order of dims in the first product is theirs.  Of a value a lane has the same dims as above.  While a wave uses 32 keys the next
            // 32 are on their way (a second set of registers for 64 brings nothing: what bounds a long call is how fast
            // workgroups that each stream their own blocks are served, 6.0 TB/s; a fourth workgroup a CU in their place lets
            // 64 contexts of 1024 take 20.0 us in place of 24.2), and the scales and places of the step behind it; the table's entries two steps
            // ahead.  None of this stands behind a condition, for which the compiler would wait for all of it: past the end
            // every lane asks for the last key again, which no row sees there.
            typedef unsigned long long u64;
            constexpr int GW = DP > 128 ? 2 : 1;           // words of a row's scales
            const int groups = mx_groups(dim);
            auto has_group = [&](int u) { return FULL || (DP == 64 ? g / 2 : 4 * u + g) < groups; };
            // the wave's lists, which lie where its sums go at the end: where rows stand, and their scales
            u64 *const places = (u64 *)(join + wave * 16 * OD);
            uint32_t *const scales = (uint32_t *)(places + 2 * 64);
            static_assert(2 * 64 * 8 + 2 * 2 * GW * 64 * 4 <= 16 * OD * 4, "");
            auto scales_at = [&](int turn, int kv, int word) { return scales + ((turn * 2 + kv) * GW + word) * 64; };
            const uint32_t value_turn = mx_turn(DP == 64 ? i16 / 8 : i16 / 4);
            const char *const key_base = kbase + (DP == 64 ? 8 : 16) * g;
            const char *const value_base = vbase + (FULL ? VE / 2 * i16 : min(VE / 2 * i16, 16 * groups - VE / 2));
            const int value_step = FULL ? 64 : min(64, 16 * groups - VE / 2 - min(VE / 2 * i16, 16 * groups - VE / 2));   // to a lane's second eight dims

            float c = p.c;                                 // (in a vector register, not asked for again at every step)
            asm("" : "+v"(c));

            struct Scales {
                uint32_t word[2][GW];
            };
            // (In 64 bits throughout: of a 32-bit product and sum the compiler takes the upper half from any register, and waits for
            // what is on its way there.)
            auto entry_of = [&](int n) { return key_entry<true>(p, q, table, min(begin + (n + (lane >> 5) * NW) * 32 + (lane & 31), end - 1)); };
            auto block_of = [&](Entry e) { return (u64)(e.block < (uint32_t)p.blocks ? e.block : 0); };
            auto place_of = [&](Entry e) { return (block_of(e) * p.block_step + (u64)e.slot * p.slot_step) * 16; };
            auto load_scales = [&](Entry e) {
                Scales x;
                const u64 at = (block_of(e) * p.scale_block + (u64)e.slot * p.scale_slot) * (DP / 32);
#pragma unroll
                for (int kv = 0; kv < 2; kv++) {
                    const char *from = (const char *)(kv ? p.v_scales : p.k_scales) + (long long)h * p.scale_head + at;
                    if constexpr (DP == 64) {
                        x.word[kv][0] = *(const uint16_t *)from;
                    } else if constexpr (DP == 128) {
                        x.word[kv][0] = *(const uint32_t *)from;
                    } else {
                        const u2 y = *(const u2 *)from;
                        x.word[kv][0] = y[0], x.word[kv][GW - 1] = y[1];
                    }
                }
                return x;
            };
            auto enter_scales = [&](int turn, const Scales &x) {
#pragma unroll
                for (int kv = 0; kv < 2; kv++)
#pragma unroll
                    for (int w = 0; w < GW; w++) scales_at(turn, kv, w)[lane] = x.word[kv][w];
            };
            uint32_t kc[2][KS], vc[8][VH];
            if constexpr (!FULL) {
#pragma unroll
                for (int a = 0; a < 2; a++)
#pragma unroll
                    for (int s = 0; s < KS; s++) kc[a][s] = 0u;
            }
            auto load_key_codes = [&](const u64 *rows, uint32_t (&to)[2][KS]) {
#pragma unroll
                for (int a = 0; a < 2; a++) {
                    const char *src = key_base + rows[16 * a + i16];
                    if constexpr (DP == 64) {
                        if (has_group(0)) {
                            const u2 x = *(const u2 *)src;
                            to[a][0] = x[0], to[a][1] = x[1];
                        }
                    } else {
#pragma unroll
                        for (int u = 0; u < KS / 4; u++)
                            if (has_group(u)) {
                                const u4 x = *(const u4 *)(src + 64 * u);
#pragma unroll
                                for (int w = 0; w < 4; w++) to[a][4 * u + w] = x[w];
                            }
                    }
                }
            };
            auto load_value_codes = [&](const u64 *rows, uint32_t (&to)[8][VH]) {
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const char *src = value_base + rows[16 * (j / 4) + 4 * g + j % 4];
#pragma unroll
                    for (int vh = 0; vh < VH; vh++) to[j][vh] = VE == 8 ? *(const uint32_t *)(src + vh * value_step) : *(const uint16_t *)src;
                }
            };

            if (wave < blocks) {
                Entry entry = entry_of(wave), after = entry_of(wave + 2 * NW);
                Scales these = load_scales(entry), next_scales = load_scales(after);
                places[lane] = place_of(entry);
                u64 next_place = place_of(after);
                entry = entry_of(wave + 4 * NW);
                hand_over();
                load_key_codes(places, kc);
                asm volatile("" ::: "memory");     // (in the order of the loop's: its waits count from either)
                load_value_codes(places, vc);
                asm volatile("" ::: "memory");
                enter_scales(0, these);
                hand_over();
                int turn = 0;
                for (int n = wave; n < blocks; n += 2 * NW, turn ^= 1) {
                    places[(turn ^ 1) * 64 + lane] = next_place;
                    enter_scales(turn ^ 1, next_scales);
                    next_place = place_of(entry);
                    next_scales = load_scales(entry);
                    entry = entry_of(n + 6 * NW);
                    hand_over();
#pragma unroll
                    for (int half = 0; half < 2; half++) {
                        const int v0 = begin + (n + half * NW) * 32;
                        if (half == 1 && v0 >= end) goto summed;       // (not around the loop's head: its waits count on both halves)
                        const u64 *rows = half ? places + (turn ^ 1) * 64 : places + turn * 64 + 32;
                        // S^T
                        f4 s[RT][2];
#pragma unroll
                        for (int a = 0; a < 2; a++)
#pragma unroll
                            for (int u = 0; u < (KS + 3) / 4; u++) {
                                // (a lane without a group has zeros, of which no scale must make anything else)
                                uint32_t scale = (uint32_t)((const unsigned char *)scales_at(turn, 0, u))[4 * (32 * half + 16 * a + i16) + (DP == 64 ? g / 2 : g)] << 23;
                                if (!has_group(u)) scale = 127u << 23;
#pragma unroll
                                for (int x = 4 * u; x < KS && x < 4 * u + 4; x++) {
                                    const e8 key = __builtin_bit_cast(e8, mx_values<E>(kc[a][x], scale));
#pragma unroll
                                    for (int rt = 0; rt < RT; rt++) s[rt][a] = mfma16(key, qf[rt][x], x == 0 ? (f4){0.0f, 0.0f, 0.0f, 0.0f} : s[rt][a]);
                                }
                            }
                        load_key_codes(rows, kc);
                        // what a row does not see
                        if (v0 + 32 > end || (q.t0 != q.t1 && !all_see(p, q, v0, v0 + 32, q.position + q.t0, q.position + q.t1))) {
#pragma unroll
                            for (int a = 0; a < 2; a++)
#pragma unroll
                                for (int e = 0; e < 4; e++)
#pragma unroll
                                    for (int rt = 0; rt < RT; rt++)
                                        if (!my[rt].sees(v0 + 16 * a + 4 * g + e)) s[rt][a][e] = kNone;
                        }
                        e8 pe[RT];
#pragma unroll
                        for (int rt = 0; rt < RT; rt++) {
                            float top = max2(max2(max2(s[rt][0][0], s[rt][0][1]), max2(s[rt][0][2], s[rt][0][3])),
                                             max2(max2(s[rt][1][0], s[rt][1][1]), max2(s[rt][1][2], s[rt][1][3])));
                            f2 two = swap_halves(top);
                            two = swap_quarters(max2(two[0], two[1]));
                            top = max2(two[0], two[1]) * c;
                            if (__ballot(top > m[rt] + Shares<E>::most)) {
                                const float up = fmaxf(m[rt], top - Shares<E>::lift);
                                const float down = __builtin_amdgcn_exp2f(m[rt] - reference(up));
                                m[rt] = up;
                                l[rt] *= down;
#pragma unroll
                                for (int vh = 0; vh < VH; vh++)
#pragma unroll
                                    for (int t = 0; t < VE; t++) o[rt][vh][t] *= down;
                            }
                            const float ref = reference(m[rt]);
                            f8 pr;
#pragma unroll
                            for (int j = 0; j < 8; j++) {
                                pr[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[rt][j / 4][j % 4], c, -ref));
                                l[rt] += pr[j];
                            }
                            pe[rt] = __builtin_convertvector(pr, e8);
                        }
                        // the operands of V: 8 keys of this lane's group, one dim each
#pragma unroll
                        for (int vh = 0; vh < VH; vh++) {
                            uint32_t scale[8];
#pragma unroll
                            for (int j = 0; j < 8; j += 4) {
                                const u4 words = *(const u4 *)(scales_at(turn, 1, vh) + 32 * half + 4 * j + 4 * g);
#pragma unroll
                                for (int k = 0; k < 4; k++) scale[j + k] = mx_scale(words[k], value_turn);
                            }
                            auto two_dims = [&](auto which) {
                                constexpr int W = decltype(which)::value;
                                u4 even, odd;
#pragma unroll
                                for (int j = 0; j < 4; j++) {
                                    const uint32_t a = mx_pair<E, W>(vc[2 * j][vh], scale[2 * j]), b = mx_pair<E, W>(vc[2 * j + 1][vh], scale[2 * j + 1]);
                                    even[j] = __builtin_amdgcn_perm(b, a, 0x05040100u);
                                    odd[j] = __builtin_amdgcn_perm(b, a, 0x07060302u);
                                }
#pragma unroll
                                for (int rt = 0; rt < RT; rt++) {
                                    o[rt][vh][2 * W] = mfma16(__builtin_bit_cast(e8, even), pe[rt], o[rt][vh][2 * W]);
                                    o[rt][vh][2 * W + 1] = mfma16(__builtin_bit_cast(e8, odd), pe[rt], o[rt][vh][2 * W + 1]);
                                }
                            };
                            two_dims(std::integral_constant<int, 0>());
                            two_dims(std::integral_constant<int, 1>());
                            if constexpr (VW == 4) {
                                two_dims(std::integral_constant<int, 2>());
                                two_dims(std::integral_constant<int, 3>());
                            }
                        }
                        load_value_codes(rows, vc);
                        asm volatile("" ::: "memory");      // (these are asked for here, not where they are used)
                    }
                }
            summed:
                hand_over();      // (the lists are read before sums go where they are)
            }
        } else if (wave < blocks) {
            list[wave][0][lane] = next;
            hand_over();
            load_keys(list[wave][0]);
            load_values(list[wave][0]);
            if (wave + 2 * NW < blocks) next = look_up(wave + 2 * NW);
            int turn = 0;
            for (int n = wave; n < blocks; n += 2 * NW, turn ^= 1) {
                if (n + 2 * NW < blocks) {
                    list[wave][turn ^ 1][lane] = next;
                    hand_over();
                    if (n + 4 * NW < blocks) next = look_up(n + 4 * NW);
                }
#pragma unroll
                for (int half = 0; half < 2; half++) {
                    const int block = n + half * NW, v0 = begin + block * 32;
                    if (half == 1 && block >= blocks) break;
                    // the rows of this wave's next block
                    const uint32_t *rows = half ? list[wave][turn ^ 1] : list[wave][turn] + 32;
                    const bool load = block + NW < blocks;
                    // S^T
                    f4 s[RT][2];
#pragma unroll
                    for (int rt = 0; rt < RT; rt++)
#pragma unroll
                        for (int a = 0; a < 2; a++) {
                            s[rt][a] = (f4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                            for (int x = 0; x < KS; x++) s[rt][a] = mfma16(__builtin_bit_cast(e8, kr[a][x]), qf[rt][x], s[rt][a]);
                        }
                    if (load) load_keys(rows);
                    // what a row does not see
                    const bool tail = v0 + 32 > end;
                    const bool mixed = q.t0 != q.t1 && !all_see(p, q, v0, v0 + 32, q.position + q.t0, q.position + q.t1);
#pragma unroll
                    for (int rt = 0; rt < RT; rt++)
#pragma unroll
                        for (int a = 0; a < 2; a++)
#pragma unroll
                            for (int e = 0; e < 4; e++) s[rt][a][e] *= p.c;
                    if (tail || mixed) {
#pragma unroll
                        for (int a = 0; a < 2; a++)
#pragma unroll
                            for (int e = 0; e < 4; e++)
#pragma unroll
                                for (int rt = 0; rt < RT; rt++)
                                    if (!my[rt].sees(v0 + 16 * a + 4 * g + e)) s[rt][a][e] = kNone;
                    }
                    e8 pe[RT];
#pragma unroll
                    for (int rt = 0; rt < RT; rt++) {
                        float top = fmaxf(fmaxf(fmaxf(s[rt][0][0], s[rt][0][1]), fmaxf(s[rt][0][2], s[rt][0][3])),
                                          fmaxf(fmaxf(s[rt][1][0], s[rt][1][1]), fmaxf(s[rt][1][2], s[rt][1][3])));
                        top = max_quarters(top);
                        if (__ballot(top > m[rt] + Shares<E>::most)) {
                            const float up = fmaxf(m[rt], top - Shares<E>::lift);
                            const float down = __builtin_amdgcn_exp2f(m[rt] - reference(up));
                            m[rt] = up;
                            l[rt] *= down;
#pragma unroll
                            for (int vh = 0; vh < VH; vh++)
#pragma unroll
                                for (int t = 0; t < VE; t++) o[rt][vh][t] *= down;
                        }
                        const float ref = reference(m[rt]);
                        f8 pr;
#pragma unroll
                        for (int j = 0; j < 8; j++) {
                            pr[j] = __builtin_amdgcn_exp2f(s[rt][j / 4][j % 4] - ref);
                            l[rt] += pr[j];
                        }
                        pe[rt] = __builtin_convertvector(pr, e8);
                    }
                    // the operands of V: 8 keys of this lane's group, one dim each
#pragma unroll
                    for (int vh = 0; vh < VH; vh++)
#pragma unroll
                        for (int w = 0; w < VW; w++) {
                            u4 even, odd;
#pragma unroll
                            for (int j = 0; j < 4; j++) {
                                even[j] = __builtin_amdgcn_perm(vr[2 * j + 1][vh][w], vr[2 * j][vh][w], 0x05040100u);
                                odd[j] = __builtin_amdgcn_perm(vr[2 * j + 1][vh][w], vr[2 * j][vh][w], 0x07060302u);
                            }
#pragma unroll
                            for (int rt = 0; rt < RT; rt++) {
                                o[rt][vh][2 * w] = mfma16(__builtin_bit_cast(e8, even), pe[rt], o[rt][vh][2 * w]);
                                o[rt][vh][2 * w + 1] = mfma16(__builtin_bit_cast(e8, odd), pe[rt], o[rt][vh][2 * w + 1]);
                            }
                        }
                    if (load) load_values(rows);
                }
            }
        }

        // the four waves, 16 rows at a time
        const bool whole = parts == 1 && !SHARED;
        const long long all = (long long)p.tokens * p.heads;
        const long long mine = ((2 * member + (first == member)) * p.kv_heads + h) * R;
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            l[rt] = add_quarters(l[rt]);
            if (g == 0 && wave < busy) stat_m[wave][16 * rt + i16] = m[rt], stat_l[wave][16 * rt + i16] = l[rt];
        }
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            if (rt > 0) __syncthreads();
            if (wave < busy && 16 * rt + i16 < q.rows) {
                float *to = join + (wave * 16 + i16) * OD;
#pragma unroll
                for (int vh = 0; vh < VH; vh++)
#pragma unroll
                    for (int e = 0; e < 4; e++)
#pragma unroll
                        for (int t = 0; t < VE; t += 4)
                            *(f4 *)(to + 128 * vh + VE * (4 * g + e) + t) = (f4){o[rt][vh][t][e], o[rt][vh][t + 1][e], o[rt][vh][t + 2][e], o[rt][vh][t + 3][e]};
            }
            __syncthreads();
            for (int x = MX ? thread : (int)threadIdx.x; x < 16 * (DP / 4); x += 64 * NW) {
                const int r = x / (DP / 4), d = x % (DP / 4) * 4, row = 16 * rt + r;
                if (row >= q.rows || d >= dim) continue;
                float top = kNone, sum = 0.0f, ms[NW];
#pragma unroll
                for (int w = 0; w < NW; w++) {
                    ms[w] = w < busy ? stat_m[w][row] : kNone;
                    top = fmaxf(top, ms[w]);
                }
                const float ref = reference(top);
                f4 total = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int w = 0; w < NW; w++) {
                    const f4 y = *(const f4 *)(join + (w * 16 + r) * OD + d);
                    const float f = __builtin_amdgcn_exp2f(ms[w] - ref), lw = stat_l[w][row];
                    if (w < busy) {
                        total += f * y;
                        sum += f * lw;
                    }
                }
                const long long at_row = out_row(p, q, h, row);
                if (whole) {
                    Sum x = {top, sum, total};
                    add_prefix(p, x, at_row, d);
                    store_row4<E>(p.out, at_row * dim + d, x.result());
                } else {
                    const long long to = SHARED ? blockIdx.y * all + at_row : mine + row;
                    put_part<!SHARED>((SHARED ? p.parts : p.own_parts) + to * dim + d, total);
                    if (d == 0) put_stats<!SHARED>((SHARED ? p.stats : p.own_stats) + 2 * to, top, sum);
                }
            }
        }
        if (parts > 1 && arrive_last(p.counters + first * p.kv_heads + h, parts, &flag))
            join_parts<E, 64 * NW, 16 * RT * DP / 4>(p, q, h, parts, join, [&](int part, int r) {
                return (long long)((2 * (first + part) + (part == 0)) * p.kv_heads + h) * R + r;
            });
        if (at >= stop) break;
        look = look_at<R, MX>(p, base);
        upto = sum_upto(look.total);
        __syncthreads();
    }
}

template <typename E, bool SHARED, bool MX>
static void launch_few(const AttentionParams &p, int rt, hipStream_t stream)
{
    const dim3 grid((unsigned)(p.kv_heads * (SHARED ? p.tiles : p.team)), SHARED ? (unsigned)p.splits : 1u);
#define GPTQ_FEW(DP, RT) \
    if (p.dim == DP) hipLaunchKernelGGL((attention_few_kernel<E, DP, true, RT, SHARED, MX>), grid, dim3(64 * kFewWaves), 0, stream, p); \
    else hipLaunchKernelGGL((attention_few_kernel<E, DP, false, RT, SHARED, MX>), grid, dim3(64 * kFewWaves), 0, stream, p)
    if (p.dim <= 64) {
        if (rt == 1) {
            GPTQ_FEW(64, 1);
        } else {
            GPTQ_FEW(64, 2);
        }
    } else if (p.dim <= 128) {
        if (rt == 1) {
            GPTQ_FEW(128, 1);
        } else {
            GPTQ_FEW(128, 2);
        }
    } else {
        GPTQ_FEW(256, 1);
    }
#undef GPTQ_FEW
}

template <bool MX>
static int launch_few_of(const AttentionParams &p, int type, int rt, void *stream_v)
{
    hipStream_t stream = (hipStream_t)stream_v;
    if (type == GPTQ_HIP_TYPE_FP16) p.shared ? launch_few<_Float16, true, MX>(p, rt, stream) : launch_few<_Float16, false, MX>(p, rt, stream);
    else p.shared ? launch_few<__bf16, true, MX>(p, rt, stream) : launch_few<__bf16, false, MX>(p, rt, stream);
    return hipGetLastError() == hipSuccess ? GPTQ_HIP_OK : GPTQ_HIP_ERR_LAUNCH;
}

}  // namespace gptq
