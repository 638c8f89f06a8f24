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
//             the parts, 16 rows a workgroup.  (The last workgroup of a tile doing it, one for up to 128 rows: 16 pieces of
//             20 tokens behind 2048 keys, dim 128, 73.6 us against 54.5; 5 of up to 333 behind up to 9001, dim 80, 77.7
//             against 66.6.)
//   LDS       rows as they lie in the cache; the 16-byte chunks of row r stand at chunk ^ r (keys) and chunk ^ 2 r (values),
//             without which all lanes of a read would stand on the same banks.  Some still do: a third of the cycles of LDS are
//             conflicts.  The swizzle is in the requests' source addresses.
//
// Measured (32 heads in groups of 4, dim 128): a prompt of 8192 tokens 587 to 613 us on different cards, 897 to 937 TFLOP/s; the matrix
// pipes are busy in half of the cycles, at 1.8 GHz; a wave waits for data or the barrier 31 % of its time, and 31 % to issue.  Without
// the exponentials it takes 6 % less, without the requests 18 %, without the reads of values 3 %.  Not better: 64 rows a wave (spills,
// 1537 us), eight waves a workgroup (the same), a wave's priority raised around its products (fewer cycles, the same time).
#include <algorithm>
#include <type_traits>

#include "gptq_attention.h"

namespace gptq {

constexpr int kTileKeys = 64;   // keys of a step
constexpr int kJoinRows = 16;

// The tile of a workgroup.  Request b owns the tiles from first_tile(b) = floor(starts[b] * group / R) + b: the floors of two
// neighbours lie at least floor(rows / R) apart, and the + b adds the tile of a remainder.  So the bound
// floor(tokens * group / R) + requests on the number of tiles, and the request of a tile, follow without any sum over
// requests.  False for a tile past its request's rows.
template <int R>
__device__ __forceinline__ bool find_tile(const AttentionParams &p, int tile, QueryTile &q)
{
    const int lane = threadIdx.x & 63;
    int context = p.prefix;
    if (p.shared) {
        q.b = 0, q.start = 0, q.count = p.tokens, q.row0 = tile * R;
    } else {
        // what the tensors say is cut to what the other arguments allow: wrong lengths give wrong sums, not wrong addresses
        int before = 0;
#pragma unroll 4
        for (int b0 = 0; b0 < p.requests; b0 += 64) {
            const int b = b0 + lane;
            const int s = min(max(p.starts[min(b, p.requests)], 0), p.tokens);
            before += __popcll(__ballot(b < p.requests && (int)((uint32_t)s * (uint32_t)p.group / R) + b <= tile));
        }
        q.b = __builtin_amdgcn_readfirstlane(max(before, 1) - 1);
        q.start = min(max(p.starts[q.b], 0), p.tokens);
        q.count = min(max(p.starts[q.b + 1] - q.start, 0), p.tokens - q.start);
        context = p.contexts[q.b];
        q.row0 = (tile - ((int)((uint32_t)q.start * (uint32_t)p.group / R) + q.b)) * R;
    }
    const int all = q.count * p.group;
    if (q.row0 < 0 || q.row0 >= all) return false;
    q.rows = min(R, all - q.row0);
    if (p.shared) set_tile<true>(p, q, context);
    else set_tile<false>(p, q, context);
    return true;
}

// The keys of a part, and how many parts the tile has.  A list that is longer than the host expected (splits * chunk) has
// longer parts.
__device__ __forceinline__ int tile_parts(const AttentionParams &p, int seen, int unit, int &chunk)
{
    chunk = max(p.chunk, ((seen + p.splits - 1) / p.splits + unit - 1) / unit * unit);
    return max(1, (seen + chunk - 1) / chunk);
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

// DP: row of LDS (a power of two), DC: dims that are computed, the multiple of 16 that covers p.dim
template <typename E, int DP, int DC>
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
    uint32_t *list = (uint32_t *)(smem + 4 * TILE);     // [8][KT]

    const int lane = threadIdx.x & 63, col = lane & 31, hh = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    // the last rows of a request see the most keys: they come first
    const int h = blockIdx.x % p.kv_heads, tile = p.tiles - 1 - blockIdx.x / p.kv_heads, split = blockIdx.y;
    QueryTile q;
    const int first_token = p.shared ? 0 : p.starts[0], end_token = p.shared ? p.tokens : p.starts[p.requests];
    const bool found = find_tile<kTileRows>(p, tile, q);
    if (!p.shared) clear_rest(p, first_token, end_token, (blockIdx.y * (long long)gridDim.x + blockIdx.x) * 256 + threadIdx.x, 256ll * gridDim.x * gridDim.y);
    if (!found) return;
    int chunk;
    const int parts = tile_parts(p, q.seen, KT, chunk);
    if (split >= parts) return;
    const int begin = split * chunk, end = min(q.seen, begin + chunk);
    const int32_t *table = p.tables + (long long)q.b * p.table_stride;
    const char *kbase = (const char *)p.k + (long long)h * p.head_stride * 2;
    const char *vbase = (const char *)p.v + (long long)h * p.head_stride * 2;

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
        return key_row(p, q, table, min(begin + min(n, tiles - 1) * KT + lane, end - 1));
    };
    auto enter = [&](int n, uint32_t row) {
        list[(n & 7) * KT + lane % RP * PASSES + lane / RP] = row;
    };
    typedef uint32_t Rows __attribute__((ext_vector_type(PASSES)));
    // this thread's chunk of the rows it requests
    const int myrow = threadIdx.x / CH, place = threadIdx.x % CH;
    auto rows_of = [&](int n) { return *(const Rows *)(list + (n & 7) * KT + myrow * PASSES); };
    auto request = [&](const Rows &rows, const char *from, uint32_t to, int twist) {
#pragma unroll
        for (int j = 0; j < PASSES; j++) {
            const int c = place ^ ((twist * (j * RP + myrow)) & (CH - 1));
            if (p.dim == DP || c * 8 < p.dim)
                request16(from + (unsigned long long)rows[j] * 16 + c * 16, __builtin_amdgcn_readfirstlane(to + wave * 1024 + j * 4096));
        }
    };
    auto request_keys = [&](const Rows &rows, int buf) { request(rows, kbase, lds + buf * TILE, 1); };
    auto request_values = [&](const Rows &rows, int buf) { request(rows, vbase, lds + (2 + buf) * TILE, 2); };
    auto meet = [&]() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); };

    float m = kNone, l = 0.0f;
    f16 o[DT];
#pragma unroll
    for (int dt = 0; dt < DT; dt++) o[dt] = (f16)(0.0f);

    // Where this lane's operands stand in the first buffers.  The rest of an address is an immediate: 32 keys on, or 8 or 16
    // values, leave the swizzle as it is.
    uint32_t kat[SX], vat[2][DT];
#pragma unroll
    for (int x = 0; x < SX; x++) kat[x] = lds + col * (DP * 2) + (((2 * x + hh) ^ (col & (CH - 1))) * 16);
#pragma unroll
    for (int up = 0; up < 2; up++)
#pragma unroll
        for (int dt = 0; dt < DT; dt++) {
            const int key = 8 * up + 4 * hh + (col & 15) / 4, c = 4 * dt + 2 * (col >> 4) + (col & 3) / 2;
            vat[up][dt] = lds + 2 * TILE + key * (DP * 2) + ((c ^ ((2 * key) & (CH - 1))) * 16) + (col & 1) * 8;
        }
    static_assert(CH <= 32, "the swizzle repeats every 32 rows, of keys, and every 16, of values");

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
    // softmax of tile n, whose scores are in s, and its products with the values in the buffer BUF; then the next scores
    auto sum = [&](int n, auto buf) {
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
        }
        scores(std::integral_constant<int, 1 - decltype(buf)::value>());
    };

    if (tiles > 0) {
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
            if (works) sum(n, buf);
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
    if (r < q.rows) {
        const long long at = out_row(p, q, h, r);
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

// Joins the parts of tiles that are divided, or stand behind a shared prefix: kJoinRows rows of a tile a workgroup.
template <typename E>
__global__ __launch_bounds__(256) void attention_join_kernel(const AttentionParams p)
{
    const int h = blockIdx.x % p.kv_heads, tile = blockIdx.x / p.kv_heads, r0 = blockIdx.y * kJoinRows;
    QueryTile q;
    if (!find_tile<kTileRows>(p, tile, q) || r0 >= q.rows) return;
    int chunk;
    const int parts = tile_parts(p, q.seen, kTileKeys, chunk);
    if (parts == 1 && p.prefix_parts == 0) return;
    const long long all = (long long)p.tokens * p.heads;
    const int quads = p.dim / 4;
    for (int i = threadIdx.x; i < min(kJoinRows, q.rows - r0) * quads; i += 256) {
        const int r = i / quads, d = (i - r * quads) * 4;
        const long long at = out_row(p, q, h, r0 + r);
        Sum x = {kNone, 0.0f, {0.0f, 0.0f, 0.0f, 0.0f}};
        add_prefix(p, x, at, d);
        add_parts<false>(x, 0, 1, parts, [&](int s) { return p.own_stats + 2 * (s * all + at); },
                         [&](int s) { return p.own_parts + (s * all + at) * p.dim + d; });
        store_row4<E>(p.out, at * p.dim + d, x.result());
    }
}

template <typename E>
static void launch_tile(const AttentionParams &p, hipStream_t stream)
{
    const dim3 grid((unsigned)(p.kv_heads * p.tiles), (unsigned)p.splits);
    // A CU holds three workgroups of rows of 64.  Where those that have rows are two a CU at most (and not many others run beside them) three
    // would stand on some and one on others; LDS for two keeps it even.  Behind 4096 keys, 32 heads in groups of 4, us with LDS for two and
    // for three: 8 pieces of 128 tokens (512 with rows of 640, two parts) 62 / 72, of 256 (512 of 576) 94 / 114, of 288 (576 of 640) 141 / 117,
    // of 320 (640 of 704) 155 / 124; 16 of 64 behind 1000 (512 of 768, two parts) 39 / 30.  With 8 heads: 8 of 512 (512 of 544, two
    // parts) 61 / 71, of 288 (576 of 640) 54 / 45; on the wrong side 8 of 256 (512 of 576, four parts) 52 / 43.
    const long long groups = (long long)p.kv_heads * p.splits, full = ((long long)p.tokens * p.group + kTileRows - 1) / kTileRows;
    const int least = groups * full <= 512 && groups * p.tiles <= 640 ? 56 * 1024 : 0;
#define GPTQ_TILE(DP, DC) \
    hipLaunchKernelGGL((attention_tile_kernel<E, DP, DC>), grid, dim3(256), std::max(4 * kTileKeys * DP * 2 + 8 * kTileKeys * 4, least), stream, p)
    if (p.dim <= 64) GPTQ_TILE(64, 64);
    else if (p.dim <= 80) GPTQ_TILE(128, 80);
    else if (p.dim <= 96) GPTQ_TILE(128, 96);
    else if (p.dim <= 128) GPTQ_TILE(128, 128);
    else if (p.dim <= 192) GPTQ_TILE(256, 192);
    else GPTQ_TILE(256, 256);
#undef GPTQ_TILE
    if (!p.shared && (p.splits > 1 || p.prefix_parts > 0))
        hipLaunchKernelGGL(attention_join_kernel<E>, dim3(grid.x, kTileRows / kJoinRows), dim3(256), 0, stream, p);
}

int launch_attention_tile(const AttentionParams &p, int type, void *stream)
{
    if (type == GPTQ_HIP_TYPE_FP16) launch_tile<_Float16>(p, (hipStream_t)stream);
    else launch_tile<__bf16>(p, (hipStream_t)stream);
    return hipGetLastError() == hipSuccess ? GPTQ_HIP_OK : GPTQ_HIP_ERR_LAUNCH;
}

}  // namespace gptq
