// Attention over a paged cache for many rows a request: prompts, pieces of prompts, a batch behind a shared prefix.
//
// What bounds it: the matrix instructions and the exponentials beside them.  A workgroup of four waves takes 128 rows, 32 a
// wave, and walks the tile's keys 64 at a time; keys and values go through LDS, so that a row from the cache is read once
// for 128 rows.
//
//   S^T = K Q^T    32 x 32 results: a lane holds 16 keys of one row for each 32 keys, the maximum and the sum of a row are
//             the lane's own and one exchange with lane ^ 32.
//   O^T += V^T P^T  the sum over keys runs in the order in which the lane already holds p (keys 4 h + 8 x + y of 16, h =
//             lane / 32); the operand of V in the same order comes from LDS through the transposing read.
//   order     the products of S run one tile of keys ahead of the softmax and the products with V, so that a wave has matrix
//             instructions to issue between its exponentials.
//   staging   direct requests from the cache into LDS (16 bytes a lane, no registers), two buffers for keys and two for
//             values, one barrier a tile: while tile n is summed, the keys of n + 2 and the values of n + 1 arrive.  The
//             rows' places come from a ring of lists in LDS, filled every four tiles by all waves at once, a tile each (one
//             wave doing it for every tile held the others up at every barrier).
//   parts     where a batch has fewer tiles than the card holds workgroups, each tile's keys are divided; a second launch joins
//             the parts, 16 rows a workgroup.  (The last workgroup of a tile doing it, one for up to 128 rows, cost 16 pieces of
//             20 tokens behind 2048 keys, dim 128, a third more, 5 of up to 333 behind up to 9001, dim 80, a sixth.)
//   LDS       rows as they lie in the cache; the 16-byte chunk c of row r stands at c ^ t(r), the four low bits of r turned by two.
//             Sixteen lanes read the same chunk of 16 keys at a time, and 32 lanes four chunks of four rows of values: t puts each on banks of
//             its own (c ^ r and c ^ 2 r, which served sixteen lanes of the latter, cost a third of the cycles of LDS and 1 % of the
//             time).  The swizzle is in the requests' source addresses.
//
// Measured (32 heads in groups of 4, dim 128): a prompt of 8192 tokens 587 to 619 us on different cards, 889 to 937 TFLOP/s; the matrix
// pipes are busy in half of the cycles, at 1.8 GHz; a wave waits for data or the barrier 31 % of its time, and 31 % to issue.  Without
// the exponentials it takes 6 % less, without the requests 18 %, without the reads of values 3 %.  Not better: 64 rows a wave (spills,
// 1537 us), eight waves a workgroup (the same), a wave's priority raised around its products (fewer cycles, the same time).
//
// A cache in MXFP4 (MX).  LDS holds the same values at the same places.  A tile's codes come into registers a tile ahead, four threads a
// row, and are turned into values (two an instruction, exactly) and written to LDS between the products, whose pipe they leave alone.
// Measured as above: a prompt of 8192 tokens 573 to 586 us, 938 to 960 TFLOP/s; 128 single tokens behind a prefix of 16384 67 us, two launches and
// the parts between them; 5 pieces of up to 333 behind up to 9001, dim 80, 68 us.
#pragma once
#include <algorithm>
#include <type_traits>

#include "gptq_attention.h"
#include "gptq_mx.h"

namespace gptq {

constexpr int kTileKeys = 64;   // keys of a step
constexpr int kJoinRows = 16;

// Request b, or requests [base, base + 64), one a lane, as the kernel of tiles sees them.
struct TileRequests {
    int start, count, context;
    int tiles, keys;       // tiles, and the keys that any of its tokens sees: no tile's list is longer
};
__device__ __forceinline__ TileRequests look_at_tile(const AttentionParams &p, int b, bool there)
{
    // what the tensors say is cut to what the other arguments allow: wrong lengths give wrong sums, not wrong addresses
    const int first = p.starts[b], end = p.starts[b + 1];
    TileRequests r;
    r.context = p.contexts[b];
    r.start = min(max(first, 0), p.tokens);
    r.count = there ? min(max(end - r.start, 0), p.tokens - r.start) : 0;
    const uint32_t rows = (uint32_t)r.count * (uint32_t)p.group;
    r.tiles = rows <= (uint32_t)p.few_rows ? 0 : (int)((rows + kTileRows - 1) / kTileRows);
    const int hi = max(min(r.context, held_keys(p)), 0), lo = p.window > 0 ? min(max(r.context - r.count - p.window + 1, 0), hi) : 0;
    r.keys = p.front + min(p.sinks, lo) + hi - lo;
    return r;
}
__device__ __forceinline__ TileRequests look_at_tiles(const AttentionParams &p, int base)
{
    const int b = base + (threadIdx.x & 63);
    return look_at_tile(p, min(b, p.requests - 1), b < p.requests);
}

// Keys of a part, before they are cut to the tile's list.  Up to kEvenRequests requests: the smallest parts, in steps of 64 keys, with which all tiles
// together have no more parts than run at once, if those are not longer than 1.5 times an even share, or than the host's; else the host's.  (The host
// knows the longest context only and divides as if all had it, and counts no tiles that are not full.  Where tiles of short lists leave the
// long ones no parts, the host's take several rounds, but are done sooner: dim 256, 5 pieces of up to 333 tokens behind up to 9001 keys 510 us as they
// fit at once, 367 so, 8 behind up to 9000 533 / 393.)  Every workgroup finds them for itself, of the
// same numbers by the same operations; that and the places for twice as many parts cost 4 us, so that it is for long contexts:
// measured beside the choice.
template <int N>
__device__ __forceinline__ int even_keys(const AttentionParams &p, const TileRequests (&r)[N])
{
    int steps[N], most = 0;      // of a tile
    float all = 0.0f;
#pragma unroll
    for (int n = 0; n < N; n++) {
        steps[n] = r[n].tiles ? (r[n].keys + kTileKeys - 1) / kTileKeys : 0;
        most = max(most, max_lanes(steps[n]));
        // (of wrong lengths the sums may be anything: every choice is a right one, and the same in every workgroup)
        all += (float)__builtin_amdgcn_readlane(sum_upto(r[n].tiles * ((steps[n] + 7) / 8)), 63) * 8.0f;
    }
    const int share = (int)min(all * 1.5f * (float)p.kv_heads / (float)p.even, 1e6f), least = max(4, (most + p.splits - 1) / p.splits);
    auto fit = [&](int part) {
        const float per = __builtin_amdgcn_rcpf((float)part);
        int parts = 0;
#pragma unroll
        for (int n = 0; n < N; n++) parts += r[n].tiles * (int)ceilf((float)steps[n] * per);
        return (long long)__builtin_amdgcn_readlane(sum_upto(parts), 63) * p.kv_heads <= p.even;
    };
    const int given = max(least, p.chunk / kTileKeys);
    int few = least, many = max(least, min(most, max(share, given)));      // steps of a part
    if (!fit(many)) few = many = given;
    while (few < many) {
        const int mid = (few + many) / 2;
        if (fit(mid)) many = mid;
        else few = mid + 1;
    }
    return __builtin_amdgcn_readfirstlane(few * kTileKeys);
}

// The tile and the part of workgroup `at` of those of a key/value head, or (JOIN) tile `at`; the keys of a part, and how many parts the tile has.
// The requests come one after the other, the last rows of a request first (they see the most keys), and of up to 64 the longest contexts
// first where not all workgroups run at once.  If all tiles of up to 64 requests have as many parts, the first parts come before the second
// ones: the last ones are the shortest, and share a CU where there are more workgroups than CUs (4 pieces of 64 tokens behind 1000, five parts,
// 320 workgroups, us a request after the other and so: 16 bits, dim 64 18.4 / 17.1, dim 128 25.8 / 24.0, MXFP4 28.5 / 25.3).  Workgroups
// without work are the last ones: between others they cost more than themselves, since workgroups go to the parts of the card in turn,
// whichever have room (64 pieces of 32 tokens behind 4096, 32 heads in groups of 4, every second workgroup without a tile: 278 us, 175 so).  There are at
// most floor(tokens * group / kTileRows) + requests tiles.  A list that is longer than the host expected (splits * chunk) has longer parts.
// False for a workgroup without work.
// What small calls have no use for stands out of their way, and is short: all of it is on the way of code into an empty cache (16 bits, a chunk of 17 tokens, dim 64,
// 6.9 to 6.6 us with the order of the arguments, 100 pieces of 20 tokens 16.8 to 16.1 with 64 requests at a time).
template <bool EVEN, bool JOIN>
__device__ __forceinline__ bool find_tile(const AttentionParams &p, int at, QueryTile &q, int &split, int &chunk, int &parts)
{
    const int lane = threadIdx.x & 63;
    int base = p.chunk, context = p.prefix;
    split = 0, q.row0 = -1;
    // parts of a request's tiles: as many as its longest list has
    auto parts_of = [&](const TileRequests &r) {
        return JOIN || p.splits == 1 ? 1 : r.keys > (long long)p.splits * base ? p.splits : max(1, (r.keys + base - 1) / base);
    };
    // workgroup `at` of those of request b, the `owner` of r
    auto take = [&](const TileRequests &r, int b, int owner, int at, bool known) {
        q.b = b, q.start = __builtin_amdgcn_readlane(r.start, owner), q.count = __builtin_amdgcn_readlane(r.count, owner);
        context = __builtin_amdgcn_readlane(r.context, owner);
        const int tiles = max(1, __builtin_amdgcn_readlane(r.tiles, owner));
        if (!JOIN && p.splits > 1 && !known) split = __builtin_amdgcn_readfirstlane(at / tiles), at -= split * tiles;
        q.row0 = (tiles - 1 - at) * kTileRows;
    };
    if (p.shared) {
        split = at / p.tiles;
        q.b = 0, q.start = 0, q.count = p.tokens, q.row0 = (at - split * p.tiles) * kTileRows;
    } else if (p.requests == 1) {       // (lengths by scalar reads, nothing to search: 0.2 us sooner, and as much in the join: 40 tokens behind 960, dim 128, 19.0 us, 18.5 so)
        const TileRequests r = look_at_tile(p, 0, true);
        const int each = parts_of(r);
        if (at >= r.tiles * each) return false;
        if (!JOIN && p.splits > 1) split = at / r.tiles, at -= split * r.tiles;
        q.b = 0, q.start = r.start, q.count = r.count, context = r.context, q.row0 = (r.tiles - 1 - at) * kTileRows;
    } else if (__builtin_expect(p.requests <= 64, 1)) {
        const TileRequests r[1] = {look_at_tiles(p, 0)};
        if (EVEN && p.even) base = even_keys(p, r);
        int own = r[0].tiles, from = lane;
        bool alike = false;
        if (!JOIN && p.splits > 1) {
            const int mine = parts_of(r[0]);
            const unsigned long long with = __ballot(own > 0);
            if (!with) return false;
            const int each = __builtin_amdgcn_readlane(mine, __builtin_ctzll(with));
            alike = !__ballot(own > 0 && mine != each);
            if (alike) {
                const int all = __builtin_amdgcn_readlane(sum_upto(own), 63);
                split = __builtin_amdgcn_readfirstlane(at / all), at -= split * all;
                if (split >= each) return false;
            } else {
                own *= mine;
            }
        }
        int upto = sum_upto(own);
        const int total = __builtin_amdgcn_readlane(upto, 63);
        if (at >= total) return false;
        if (!JOIN && __builtin_expect(total * p.kv_heads > (p.dim > 128 ? 256 : 512), 0)) {
            const uint32_t key = (uint32_t)min(max(r[0].context, 0), (1 << 25) - 1) << 6 | (63 - lane);
            int longer = 0;
            for (int j = 0; j < p.requests; j++) longer += (uint32_t)__builtin_amdgcn_readlane((int)key, j) > key;
            if (lane >= p.requests) longer = lane;
            from = __builtin_amdgcn_ds_permute(4 * longer, lane);
            own = __builtin_amdgcn_ds_permute(4 * longer, own);
            upto = sum_upto(own);
        }
        const int place = __popcll(__ballot(upto <= at)), owner = __builtin_amdgcn_readlane(from, place);
        take(r[0], owner, owner, at - (__builtin_amdgcn_readlane(upto, place) - __builtin_amdgcn_readlane(own, place)), alike);
    } else {
        constexpr int N = EVEN ? kEvenRequests / 64 : 1;     // (waves of requests at a time)
        for (int b0 = 0; b0 < p.requests && q.row0 < 0; b0 += 64 * N) {
            TileRequests r[N];
#pragma unroll
            for (int n = 0; n < N; n++) r[n] = look_at_tiles(p, b0 + 64 * n);
            if (EVEN && p.even) base = even_keys(p, r);      // (there are no more requests)
#pragma unroll
            for (int n = 0; n < N; n++) {
                const int own = r[n].tiles * parts_of(r[n]), upto = sum_upto(own), total = __builtin_amdgcn_readlane(upto, 63);
                if (q.row0 < 0 && at < total) {
                    const int owner = __popcll(__ballot(upto <= at));
                    take(r[n], b0 + 64 * n + owner, owner, at - (__builtin_amdgcn_readlane(upto, owner) - __builtin_amdgcn_readlane(own, owner)), false);
                }
                at -= total;
            }
        }
    }
    const int all = q.row0 < 0 ? 0 : q.count * p.group;
    if (q.row0 < 0 || q.row0 >= all) return false;
    q.rows = min(kTileRows, all - q.row0);
    if (p.shared) set_tile<true>(p, q, context);
    else set_tile<false>(p, q, context);
    chunk = max(base, ((q.seen + p.splits - 1) / p.splits + kTileKeys - 1) / kTileKeys * kTileKeys);
    parts = max(1, (q.seen + chunk - 1) / chunk);
    if (EVEN && p.even) {      // the last one no shorter
        chunk = max(kTileKeys, ((q.seen + parts - 1) / parts + kTileKeys - 1) / kTileKeys * kTileKeys);
        parts = max(1, (q.seen + chunk - 1) / chunk);
    }
    chunk = __builtin_amdgcn_readfirstlane(chunk), parts = __builtin_amdgcn_readfirstlane(parts);
    return JOIN || split < parts;
}

// 16 bytes of `src` to LDS at lds + 16 * lane.  Inline assembly, so that the compiler does not wait for every outstanding
// request before each read of LDS; the kernel waits for them at its barrier.
__device__ __forceinline__ void request16(const char *src, uint32_t lds)
{
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "s"(lds) : "m0", "memory");
}

// a 4 x 16 block of 16-bit values of a row-major matrix, as 16 lanes hold its columns: lane x gets rows 0 .. 3 of column x,
// and gives the address of four values of row x / 4 from column 4 (x % 4) on
template <typename E>
__device__ __forceinline__ u2 read_turned(uint32_t at)
{
    typedef short s4 __attribute__((ext_vector_type(4)));
    return __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4 *)(uintptr_t)at));
}
__device__ __forceinline__ u4 read16(uint32_t at) { return *(const __attribute__((address_space(3))) u4 *)(uintptr_t)at; }

// DP: row of LDS (a power of two), DC: dims that are computed, the multiple of 16 that covers p.dim; MX: a cache in MXFP4
template <typename E, int DP, int DC, bool MX>
__global__ __launch_bounds__(256, DP == 256 ? 1 : DP == 128 ? 2 : 3) void attention_tile_kernel(const AttentionParams p)
{
    typedef typename Vec<E>::e8 e8;
    constexpr int KT = kTileKeys;
    constexpr int CH = DP / 8;              // 16-byte chunks of a row
    constexpr int RP = 256 / CH;            // rows that the workgroup requests at a time
    constexpr int PASSES = KT / RP;
    constexpr int TILE = KT * DP * 2;       // bytes of a tile of keys or values
    constexpr int KA = KT / 32, SX = DC / 16, DT = (DC + 31) / 32, PX = KT / 16;
    const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char *)smem;
    uint32_t *list = (uint32_t *)(smem + 4 * TILE);     // [8][KT]; MX: and as many places of scales

    const int lane = threadIdx.x & 63, col = lane & 31, hh = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int h = blockIdx.x % p.kv_heads;
    int split, chunk, parts;
    QueryTile q;
    const int first_token = p.shared ? 0 : p.starts[0], end_token = p.shared ? p.tokens : p.starts[p.requests];
    const bool found = find_tile<MX, false>(p, blockIdx.y * p.tiles + blockIdx.x / p.kv_heads, q, split, chunk, parts);
    if (!p.shared) clear_rest(p, first_token, end_token, (blockIdx.y * (long long)gridDim.x + blockIdx.x) * 256 + threadIdx.x, 256ll * gridDim.x * gridDim.y);
    if (!found) return;
    const int begin = split * chunk, end = min(q.seen, begin + chunk);
    const int32_t *table = p.tables + (long long)q.b * p.table_stride;
    const char *kbase = (const char *)p.k + (long long)h * p.head_stride * (MX ? 1 : 2);
    const char *vbase = (const char *)p.v + (long long)h * p.head_stride * (MX ? 1 : 2);

    const int r = 32 * wave + col;
    int qt, hg;
    token_head(p, q, h, min(r, q.rows - 1), qt, hg);
    const int pos = q.position + qt;
    e8 qf[SX];
    {
        const char *src = (const char *)p.q + ((long long)(q.start + qt) * p.q_token + (long long)hg * p.q_head) * 2;
#pragma unroll
        for (int x = 0; x < SX; x++) {
            const int d = 16 * x + 8 * hh;
            u4 y = {0u, 0u, 0u, 0u};
            if (d < p.dim) y = *(const u4 *)(src + d * 2);
            qf[x] = __builtin_bit_cast(e8, y);
        }
    }
    // positions of this wave's first and last row
    const bool works = 32 * wave < q.rows;
    const int pos_first = q.position + q.t0 + tokens_of(p, q.g0 + min(32 * wave, q.rows - 1));
    const int pos_last = q.position + q.t0 + tokens_of(p, q.g0 + min(32 * wave + 31, q.rows - 1));

    const Sight my = sight(p, q, end, pos);
    const int tiles = (end - begin + KT - 1) / KT;
    // Rows of tile n for the requests: four tiles at a time, one a wave.  A thread's rows of a tile stand side by side.
    auto look_up = [&](int n) {
        const int i = min(begin + min(n, tiles - 1) * KT + lane, end - 1);
        if constexpr (MX) return key_entry<true>(p, q, table, i);
        else return key_row(p, q, table, i);
    };
    auto enter = [&](int n, auto place) {
        if constexpr (MX) {
            list[(n & 7) * KT + lane] = row_of(p, place);
            list[(8 + (n & 7)) * KT + lane] = scales_of(p, place);
        } else {
            list[(n & 7) * KT + lane % RP * PASSES + lane / RP] = place;
        }
    };
    typedef uint32_t Rows __attribute__((ext_vector_type(PASSES)));
    // the swizzle of a row.  (Rows of 64 dims alternate between the halves of the banks, so that three bits do; the lowest two, of which
    // rows of values differ, must both count.)
    auto turn = [](int row) { return DP == 64 ? ((row ^ row >> 1) << 2 & 4) | (row >> 2 & 3) : (row << 2 & 12) | (row >> 2 & 3); };
    // this thread's chunk of the rows it requests
    const int myrow = threadIdx.x / CH, place = threadIdx.x % CH;
    auto rows_of = [&](int n) { return *(const Rows *)(list + (n & 7) * KT + myrow * PASSES); };
    auto request = [&](const Rows &rows, const char *from, uint32_t to) {
#pragma unroll
        for (int j = 0; j < PASSES; j++) {
            const int c = place ^ turn(j * RP + myrow);
            if (p.dim == DP || c * 8 < p.dim)
                request16(from + (unsigned long long)rows[j] * 16 + c * 16, __builtin_amdgcn_readfirstlane(to + wave * 1024 + j * 4096));
        }
    };
    auto request_keys = [&](const Rows &rows, int buf) { request(rows, kbase, lds + buf * TILE); };
    auto request_values = [&](const Rows &rows, int buf) { request(rows, vbase, lds + (2 + buf) * TILE); };
    auto meet = [&]() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); };

    // MX: four threads hold a row of a tile, DP / 4 dims each, and write them to LDS as values.  (Rows end with a group: what of a
    // thread's dims lies behind them is zero.)
    constexpr int DW = DP / 32;             // words of codes
    struct Coded {
        uint32_t codes[DW], scales;
    };
    const int groups = MX ? mx_groups(p.dim) : 0;
    // (Taken anew for every use: what follows from the thread would else stand in registers that the kernel does not have.)
    auto this_thread = [&]() {
        int t = threadIdx.x;
        asm volatile("" : "+v"(t));
        return t;
    };
    // MX: the row whose codes a thread holds: the eight lanes that LDS takes at a time write eight chunks whose lowest bits differ
    auto row_of_codes = [](int thread) { return thread >> 6 << 4 | (thread << 2 & 12) | (thread >> 2 & 3); };
    // Where its part of a row goes, from a tile's beginning.  (Dynamic LDS begins at 0, so that the swizzle is in the low bits of the sum.)
    auto find_place = [&]() {
        const int thread = this_thread(), code_row = row_of_codes(thread), chunk = (thread >> 4 & 3) * DW;
        return (uint32_t)(code_row * (DP * 2) + (chunk ^ turn(code_row)) * 16);
    };
    const uint32_t kept_place = MX && DP <= 128 ? find_place() : 0;
    auto place_of_part = [&]() { return DP <= 128 ? kept_place : find_place(); };
    auto fetch = [&](int n, const char *from, const void *scales) {
        const int thread = this_thread(), code_row = row_of_codes(thread), code_part = thread >> 4 & 3;
        Coded x = {};
        const int first = code_part * DP / 128;              // the thread's first group
        x.scales = 0x7f7fu;
        if (first < groups) {
            const char *src = from + (unsigned long long)list[(n & 7) * KT + code_row] * 16 + code_part * (DP / 8);
            const char *at = (const char *)scales + (long long)h * p.scale_head + (unsigned long long)list[(8 + (n & 7)) * KT + code_row] * DW + first;
            if constexpr (DW == 2) {
                const u2 y = *(const u2 *)src;
                x.codes[0] = y[0], x.codes[1] = y[1];
            } else {
#pragma unroll
                for (int u = 0; u < DW / 4; u++)
                    if (first + u < groups) {
                        const u4 y = *(const u4 *)(src + 16 * u);
#pragma unroll
                        for (int w = 0; w < 4; w++) x.codes[4 * u + w] = y[w];
                    }
            }
            x.scales = DW == 8 ? *(const uint16_t *)at : *(const unsigned char *)at;
            if (DW == 8 && first + 1 >= groups) x.scales = (x.scales & 0xffu) | 0x7f00u;
        }
        return x;
    };
    // (words [w0, w1) of a part)
    auto put = [&](const Coded &x, int w0, int w1, uint32_t row) {
#pragma unroll
        for (int w = 0; w < DW; w++)
            if (w >= w0 && w < w1)
                *(__attribute__((address_space(3))) u4 *)(uintptr_t)(row ^ (w * 16)) = mx_values<E>(x.codes[w], (w < 4 ? x.scales : x.scales >> 8) << 23);
    };
    auto put_keys = [&](const Coded &x, int buf, int w0 = 0, int w1 = 8) { put(x, w0, w1, lds + buf * TILE + place_of_part()); };
    auto put_values = [&](const Coded &x, int buf, int w0 = 0, int w1 = 8) { put(x, w0, w1, lds + (2 + buf) * TILE + place_of_part()); };
    auto meet_lds = [&]() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); };

    float m = kNone, l = 0.0f;
    f16 o[DT];
#pragma unroll
    for (int dt = 0; dt < DT; dt++) o[dt] = (f16)(0.0f);

    // Where this lane's operands stand in the first buffers.  The rest of an address is an immediate: 32 keys on, or 8 or 16
    // values, leave the swizzle as it is.
    uint32_t kat[SX], vat[2][DT];
#pragma unroll
    for (int x = 0; x < SX; x++) kat[x] = lds + col * (DP * 2) + (((2 * x + hh) ^ turn(col)) * 16);
#pragma unroll
    for (int up = 0; up < 2; up++)
#pragma unroll
        for (int dt = 0; dt < DT; dt++) {
            const int key = 8 * up + 4 * hh + (col & 15) / 4, c = 4 * dt + 2 * (col >> 4) + (col & 3) / 2;
            vat[up][dt] = lds + 2 * TILE + key * (DP * 2) + ((c ^ turn(key)) * 16) + (col & 1) * 8;
        }
    static_assert(CH >= 8, "the swizzle repeats every 16 rows");

    f16 s[KA];
    // S^T for the keys in the buffer BUF
    auto scores = [&](auto buf) {
        constexpr int BUF = decltype(buf)::value * TILE;
#pragma unroll
        for (int a = 0; a < KA; a++) s[a] = (f16)(0.0f);
#pragma unroll
        for (int x0 = 0; x0 < SX; x0 += 4) {
            u4 kf[4][KA];
#pragma unroll
            for (int x = x0; x < SX && x < x0 + 4; x++)
#pragma unroll
                for (int a = 0; a < KA; a++) kf[x - x0][a] = read16(kat[x] + (BUF + 32 * a * DP * 2));
#pragma unroll
            for (int x = x0; x < SX && x < x0 + 4; x++)
#pragma unroll
                for (int a = 0; a < KA; a++) s[a] = mfma32(__builtin_bit_cast(e8, kf[x - x0][a]), qf[x], s[a]);
        }
    };
    // softmax of tile n, whose scores are in s, and its products with the values in the buffer BUF; then the next scores.  `beside`
    // is called between the products, four times.
    auto sum = [&](int n, auto buf, auto beside) {
        constexpr int BUF = decltype(buf)::value * TILE;
        u2 vf[PX][DT][2];
        auto read_values = [&](int x) {
#pragma unroll
            for (int dt = 0; dt < DT; dt++)
#pragma unroll
                for (int up = 0; up < 2; up++) vf[x][dt][up] = read_turned<E>(vat[up][dt] + (BUF + 16 * x * DP * 2));
        };
        // (a step of 16 keys ahead, but for the widest rows, which leave no registers for it, and those of 64, where the registers
        // let a third workgroup into a CU: a prompt of 4096 tokens 106 us, 97 so)
        constexpr bool EARLY = DT > 2 && DT <= 6;
        if (EARLY) read_values(0);
        __builtin_amdgcn_sched_barrier(0);
        const int v0 = begin + n * KT, v1 = min(v0 + KT, end);
        if (v0 + KT > end || !all_see(p, q, v0, v1, pos_first, pos_last)) {
#pragma unroll
            for (int a = 0; a < KA; a++)
#pragma unroll
                for (int i = 0; i < 16; i++)
                    if (!my.sees(v0 + 4 * hh + 32 * a + 8 * (i / 4) + i % 4)) s[a][i] = kNone;
        }
        float top = kNone;
#pragma unroll
        for (int a = 0; a < KA; a++)
#pragma unroll
            for (int i = 0; i < 16; i++) top = fmaxf(top, s[a][i]);
        top = max_halves(top) * p.c;
        if (__ballot(top > m + Shares<E>::most)) {
            const float up = fmaxf(m, top - Shares<E>::lift);
            const float down = __builtin_amdgcn_exp2f(m - reference(up));
            m = up;
            l *= down;
#pragma unroll
            for (int dt = 0; dt < DT; dt++) o[dt] *= down;
        }
        const float ref = reference(m);
#pragma unroll
        for (int x = 0; x < PX; x++) {
            if (!EARLY) read_values(x);
            else if (x + 1 < PX) read_values(x + 1);
            f8 pr;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                pr[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[x / 2][(x & 1) * 8 + j], p.c, -ref));
                l += pr[j];
            }
            const e8 pe = __builtin_convertvector(pr, e8);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int dt = 0; dt < DT; dt++) {
                const u4 y = {vf[x][dt][0][0], vf[x][dt][0][1], vf[x][dt][1][0], vf[x][dt][1][1]};
                o[dt] = mfma32(__builtin_bit_cast(e8, y), pe, o[dt]);
            }
            beside(x);
        }
        scores(std::integral_constant<int, 1 - decltype(buf)::value>());
    };

    if constexpr (MX) {
        if (tiles > 0) {
            enter(wave, look_up(wave));
            Entry next = look_up(4 + wave);
            meet_lds();
            Coded keys = fetch(0, kbase, p.k_scales), values = fetch(0, vbase, p.v_scales);
            Coded more = fetch(1, kbase, p.k_scales);
            put_keys(keys, 0);
            put_values(values, 0);
            put_keys(more, 1);
            keys = fetch(2, kbase, p.k_scales);
            values = fetch(1, vbase, p.v_scales);
            meet_lds();
            if (works) scores(std::integral_constant<int, 0>());
            meet_lds();
            // Tile n: the keys of n + 2 and the values of n + 1, which came while tile n - 1 was summed, go where those of n and n - 1 were.
            // They are turned into values between the products: the matrix pipes are busy then.
            auto step = [&](int n, auto buf) {
                constexpr int BUF = decltype(buf)::value;
                if ((n & 3) == 0) {      // (the places of tile n + 4 are read a tile from here at the earliest)
                    enter(n + 4 + wave, next);
                    next = look_up(n + 8 + wave);
                }
                // (past the end: the last key's row, into buffers that nobody reads)
                auto stage = [&](int x) {
                    static_assert(PX == 4, "");
                    if (x < 2) put_keys(keys, BUF, x * DW / 2, (x + 1) * DW / 2);
                    else put_values(values, 1 - BUF, (x - 2) * DW / 2, (x - 1) * DW / 2);
                    if (x == 1) keys = fetch(n + 3, kbase, p.k_scales);
                    if (x == 3) values = fetch(n + 2, vbase, p.v_scales);
                };
                if (works) {
                    sum(n, buf, stage);
                } else {
                    for (int x = 0; x < 4; x++) stage(x);
                }
                meet_lds();
            };
            for (int n = 0; n < tiles; n += 2) {
                step(n, std::integral_constant<int, 0>());
                if (n + 1 < tiles) step(n + 1, std::integral_constant<int, 1>());
            }
        }
    } else if (tiles > 0) {
        if (p.dim < DC) {   // the chunks of keys that no request fills (of values they only reach dims that are not stored)
            for (int x = threadIdx.x; x < 2 * TILE / 16; x += 256) ((u4 *)smem)[x] = (u4){0u, 0u, 0u, 0u};
        }
        enter(wave, look_up(wave));
        uint32_t next = look_up(4 + wave);
        meet();
        Rows keys = rows_of(0);
        request_keys(keys, 0);
        request_values(keys, 0);
        keys = rows_of(1);
        if (1 < tiles) request_keys(keys, 1);
        meet();
        if (works) scores(std::integral_constant<int, 0>());
        meet();
        // tile n: the keys of n + 2 go where those of n were, the values of n + 1 where those of n - 1 were
        auto step = [&](int n, auto buf) {
            constexpr int BUF = decltype(buf)::value;
            if (n + 1 < tiles) request_values(keys, 1 - BUF);
            if (n + 2 < tiles) {
                keys = rows_of(n + 2);
                request_keys(keys, BUF);
            }
            if ((n & 3) == 0) {      // (the places of tile n + 4 are read two tiles from here at the earliest)
                enter(n + 4 + wave, next);
                next = look_up(n + 8 + wave);
            }
            if (works) sum(n, buf, [](int) {});
            meet();
        };
        for (int n = 0; n < tiles; n += 2) {
            step(n, std::integral_constant<int, 0>());
            if (n + 1 < tiles) step(n + 1, std::integral_constant<int, 1>());
        }
    }

    l = add_halves(l);
    const bool whole = parts == 1 && p.prefix_parts == 0 && !p.shared;
    const long long all = (long long)p.tokens * p.heads;
    float *stats = p.shared ? p.stats : p.own_stats, *outs = p.shared ? p.parts : p.own_parts;
    const int row = MX ? 32 * wave + (this_thread() & 31) : r;
    if (row < q.rows) {
        const long long at = out_row(p, q, h, row);
        const long long slot = split * all;
        const float inv = l > 0.0f ? 1.0f / l : 0.0f;
        if (!whole && hh == 0) put_stats<false>(stats + 2 * (slot + at), m, l);
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int d = 32 * dt + 8 * i + 4 * hh;
                if (d >= p.dim) continue;
                const f4 y = {o[dt][4 * i], o[dt][4 * i + 1], o[dt][4 * i + 2], o[dt][4 * i + 3]};
                if (whole) store_row4<E>(p.out, at * p.dim + d, y * inv);
                else put_part<false>(outs + (slot + at) * p.dim + d, y);
            }
    }
}

template <typename E, bool MX>
static void launch_tile(const AttentionParams &p, hipStream_t stream)
{
    const dim3 grid((unsigned)(p.kv_heads * p.tiles), (unsigned)p.splits);
#define GPTQ_TILE(DP, DC) \
    hipLaunchKernelGGL((attention_tile_kernel<E, DP, DC, MX>), grid, dim3(256), 4 * kTileKeys * DP * 2 + (MX ? 16 : 8) * kTileKeys * 4, stream, p)
    if (p.dim <= 64) GPTQ_TILE(64, 64);
    else if (p.dim <= 80) GPTQ_TILE(128, 80);
    else if (p.dim <= 96) GPTQ_TILE(128, 96);
    else if (p.dim <= 128) GPTQ_TILE(128, 128);
    else if (p.dim <= 192) GPTQ_TILE(256, 192);
    else GPTQ_TILE(256, 256);
#undef GPTQ_TILE
    if (!p.shared && (p.splits > 1 || p.prefix_parts > 0))
        launch_attention_join(p, __is_same(E, _Float16) ? GPTQ_HIP_TYPE_FP16 : GPTQ_HIP_TYPE_BF16, grid.x, stream);
}

template <bool MX>
static int launch_tile_of(const AttentionParams &p, int type, void *stream)
{
    if (type == GPTQ_HIP_TYPE_FP16) launch_tile<_Float16, MX>(p, (hipStream_t)stream);
    else launch_tile<__bf16, MX>(p, (hipStream_t)stream);
    return hipGetLastError() == hipSuccess ? GPTQ_HIP_OK : GPTQ_HIP_ERR_LAUNCH;
}

}  // namespace gptq
