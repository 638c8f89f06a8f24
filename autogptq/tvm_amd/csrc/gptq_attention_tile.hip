// Attention over a paged cache for many rows a request: prompts, pieces of prompts, a batch behind a shared prefix.
//
// What bounds it: the matrix instructions and the exponentials beside them.  A workgroup of four waves takes 128 rows, 32 a
// wave, and walks the tile's keys KT at a time; keys and values go through LDS, so that a row from the cache is read once
// for 128 rows.
//
//   staging   direct requests from the cache into LDS (16 bytes a lane, no registers), one tile of keys ahead, two buffers
//             and one barrier a tile.  The rows' places come from a list in LDS that the first KT threads keep two tiles
//             ahead of the requests and whose block table entries they ask for three tiles ahead.
//   LDS       rows as they lie in the cache; the 16-byte chunks of row r stand at chunk ^ r (keys) and chunk ^ 2 r (values),
//             which spreads the lanes of a read over all banks.  The swizzle is in the requests' source addresses.
//   S^T = K Q^T    32 x 32 results: a lane holds 16 keys of one row for each 32 keys, the maximum and the sum of a row are
//             the lane's own and one exchange with lane ^ 32.
//   O^T += V^T P^T  the sum over keys runs in the order in which the lane already holds p (keys 4 h + 8 x + y of 16, h =
//             lane / 32); the operand of V in the same order comes from LDS through the transposing read.
#include "gptq_attention.h"

namespace gptq {

// 16 bytes of `src` to LDS at lds + 16 * lane.  Inline assembly, so that the compiler does not wait for every outstanding
// request before each read of LDS; the kernel waits for them at its barrier.
__device__ __forceinline__ void request16(const char *src, uint32_t lds)
{
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "s"(lds) : "memory");
}

// a 4 x 16 block of 16-bit values of a row-major matrix, as 16 lanes hold its columns: lane x gets rows 0 .. 3 of column x,
// and gives the address of four values of row x / 4 from column 4 (x % 4) on
template <typename E>
__device__ __forceinline__ u2 read_turned(uint32_t at)
{
    typedef short s4 __attribute__((ext_vector_type(4)));
    return __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4 *)at));
}
__device__ __forceinline__ u4 read16(uint32_t at) { return *(const __attribute__((address_space(3))) u4 *)at; }

template <typename E, int DP, int KT>
__global__ __launch_bounds__(256, DP == 256 ? 1 : 2) void attention_tile_kernel(const AttentionParams p)
{
    typedef typename Vec<E>::e8 e8;
    constexpr int CH = DP / 8;              // 16-byte chunks of a row
    constexpr int RP = 256 / CH;            // rows that the workgroup requests at a time
    constexpr int PASSES = KT / RP;
    constexpr int TILE = KT * DP * 2;       // bytes of a tile of keys or values
    constexpr int KA = KT / 32, DT = DP / 32;
    const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char *)smem;
    uint32_t *list = (uint32_t *)(smem + 4 * TILE);     // [2][KT]
    int *flag = (int *)(list + 2 * KT);

    const int lane = threadIdx.x & 63, col = lane & 31, hh = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int h = blockIdx.x % p.kv_heads, rest = blockIdx.x / p.kv_heads;
    // the last rows of a request see the most keys: they come first
    const int tile = p.tiles - 1 - rest % p.tiles, split = rest / p.tiles;
    QueryTile q;
    if (!find_tile<kTileRows>(p, tile, q)) return;
    int chunk;
    const int parts = tile_parts(p, q.seen, KT, chunk);
    if (split >= parts) return;
    const int begin = split * chunk, end = min(q.seen, begin + chunk);
    const int32_t *table = p.tables + (p.shared ? 0 : (long long)q.b * p.table_stride);
    const char *kbase = (const char *)p.k + (long long)h * p.head_stride * 2;
    const char *vbase = (const char *)p.v + (long long)h * p.head_stride * 2;

    const int r = 32 * wave + col;
    const int qrow = q.row0 + min(r, q.rows - 1), qt = qrow / p.group, hg = h * p.group + qrow - qt * p.group;
    const int pos = q.position + qt;
    e8 qf[DP / 16];
    {
        const char *src = (const char *)p.q + ((long long)(q.start + qt) * p.q_token + (long long)hg * p.q_head) * 2;
#pragma unroll
        for (int s = 0; s < DP / 16; s++) {
            const int d = 16 * s + 8 * hh;
            u4 x = {0u, 0u, 0u, 0u};
            if (d < p.dim) x = *(const u4 *)(src + d * 2);
            qf[s] = __builtin_bit_cast(e8, x);
        }
    }
    // positions of this wave's first and last row
    const bool works = 32 * wave < q.rows;
    const int pos_first = q.position + (q.row0 + min(32 * wave, q.rows - 1)) / p.group;
    const int pos_last = q.position + (q.row0 + min(32 * wave + 31, q.rows - 1)) / p.group;

    const int tiles = (end - begin + KT - 1) / KT;
    auto look_up = [&](int n) {
        return key_row(p, table, key_position(q, min(begin + n * KT + (int)threadIdx.x, end - 1)));
    };
    // this thread's chunk of the rows it requests (RP is a multiple of 8, CH at most 32: the swizzle may change with the pass)
    const int myrow = threadIdx.x / CH, place = threadIdx.x % CH;
    auto request = [&](int n) {
        const uint32_t *rows = list + (n & 1) * KT;
        const uint32_t kdst = lds + (n & 1) * TILE + wave * 1024, vdst = kdst + 2 * TILE;
#pragma unroll
        for (int j = 0; j < PASSES; j++) {
            const int row = j * RP + myrow;
            const int kc = place ^ (row & (CH - 1)), vc = place ^ ((2 * row) & (CH - 1));
            const unsigned long long at = (unsigned long long)rows[row] * 16;
            if (p.dim == DP || kc * 8 < p.dim) request16(kbase + at + kc * 16, __builtin_amdgcn_readfirstlane(kdst + j * 4096));
            if (p.dim == DP || vc * 8 < p.dim) request16(vbase + at + vc * 16, __builtin_amdgcn_readfirstlane(vdst + j * 4096));
        }
    };
    auto meet = [&]() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); };

    float m = kNone, l = 0.0f;
    f16 o[DT];
#pragma unroll
    for (int dt = 0; dt < DT; dt++) o[dt] = (f16)(0.0f);

    if (tiles > 0) {
        if (p.dim < DP) {   // the chunks that no request fills
            for (int x = threadIdx.x; x < 4 * TILE / 16; x += 256) ((u4 *)smem)[x] = (u4){0u, 0u, 0u, 0u};
        }
        uint32_t next = 0;
        if (threadIdx.x < KT) {
            list[threadIdx.x] = look_up(0);
            list[KT + threadIdx.x] = look_up(min(1, tiles - 1));
            next = look_up(min(2, tiles - 1));
        }
        meet();
        request(0);
        meet();
        for (int n = 0; n < tiles; n++) {
            if (n + 1 < tiles) request(n + 1);
            if (threadIdx.x < KT && n + 2 < tiles) {
                list[(n & 1) * KT + threadIdx.x] = next;    // (of tile n + 2; tile n's places were read before the last barrier)
                next = look_up(min(n + 3, tiles - 1));
            }
            const int v0 = begin + n * KT, v1 = min(v0 + KT, end);
            // does this wave see any of it, does every row see all of it?
            const int at0 = key_position(q, v0), at1 = key_position(q, v1 - 1);
            bool any = works, clear = v0 + KT <= end;
            if (!p.shared) {
                any = any && at0 <= pos_last && (p.window <= 0 || v0 < q.ns || at1 > pos_first - p.window);
                clear = clear && at1 <= pos_first && (p.window <= 0 || (v0 >= q.ns && at0 > pos_last - p.window));
            }
            if (any) {
                const uint32_t kb = lds + (n & 1) * TILE, vb = kb + 2 * TILE;
                f16 s[KA];
#pragma unroll
                for (int a = 0; a < KA; a++) {
                    s[a] = (f16)(0.0f);
                    const int key = 32 * a + col;
                    const uint32_t krow = kb + key * (DP * 2);
#pragma unroll
                    for (int x = 0; x < DP / 16; x++) {
                        const u4 kf = read16(krow + (((2 * x + hh) ^ (key & (CH - 1))) * 16));
                        s[a] = mfma32(__builtin_bit_cast(e8, kf), qf[x], s[a]);
                    }
                }
                if (!clear) {
#pragma unroll
                    for (int a = 0; a < KA; a++)
#pragma unroll
                        for (int i = 0; i < 16; i++) {
                            const bool seen = sees(p, q, v0 + 32 * a + 4 * hh + 8 * (i / 4) + i % 4, end, pos);
                            s[a][i] = seen ? s[a][i] : kNone;
                        }
                }
                float top = kNone;
#pragma unroll
                for (int a = 0; a < KA; a++)
#pragma unroll
                    for (int i = 0; i < 16; i++) top = fmaxf(top, s[a][i]);
                top = max_halves(top) * p.c;
                if (__ballot(top > m + 8.0f)) {
                    const float up = fmaxf(m, top);
                    const float down = __builtin_amdgcn_exp2f(m - reference(up));
                    m = up;
                    l *= down;
#pragma unroll
                    for (int dt = 0; dt < DT; dt++) o[dt] *= down;
                }
                const float ref = reference(m);
                e8 pe[KT / 16];
#pragma unroll
                for (int x = 0; x < KT / 16; x++) {
                    f8 pr;
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        pr[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[x / 2][(x & 1) * 8 + j], p.c, -ref));
                        l += pr[j];
                    }
                    pe[x] = __builtin_convertvector(pr, e8);
                }
#pragma unroll
                for (int x = 0; x < KT / 16; x++) {
                    const int key = 16 * x + 4 * hh + (col & 15) / 4;
#pragma unroll
                    for (int dt = 0; dt < DT; dt++) {
                        const int c16 = 4 * dt + 2 * (col >> 4) + (col & 3) / 2;
                        const u2 lo = read_turned<E>(vb + key * (DP * 2) + ((c16 ^ ((2 * key) & (CH - 1))) * 16) + (col & 1) * 8);
                        const u2 hi = read_turned<E>(vb + (key + 8) * (DP * 2) + ((c16 ^ ((2 * (key + 8)) & (CH - 1))) * 16) + (col & 1) * 8);
                        o[dt] = mfma32(__builtin_bit_cast(e8, ((u4){lo[0], lo[1], hi[0], hi[1]})), pe[x], o[dt]);
                    }
                }
            }
            meet();
        }
    }

    l = add_halves(l);
    const bool whole = parts == 1 && p.first_slot == 0 && !p.shared;
    if (r < q.rows) {
        const long long at = out_row(p, q, h, r);
        const long long all = (long long)p.tokens * p.heads;
        const long long slot = (long long)(p.first_slot + split) * all;
        const float inv = l > 0.0f ? 1.0f / l : 0.0f;
        if (!whole && hh == 0) store_stats(p.stats + 2 * (slot + at), m, l);
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int d = 32 * dt + 8 * i + 4 * hh;
                if (d >= p.dim) continue;
                const f4 y = {o[dt][4 * i], o[dt][4 * i + 1], o[dt][4 * i + 2], o[dt][4 * i + 3]};
                if (whole) store_row4<E>(p.out, at * p.dim + d, y * inv);
                else store_partial(p.parts + (slot + at) * p.dim + d, y);
            }
    }
    if (whole || p.shared) return;
    if (last_part(p, tile * p.kv_heads + h, parts, flag))
        join_parts<E, 256>(p, q, h, p.first_slot + parts, (float *)smem);
}

template <typename E>
static void launch_tile(const AttentionParams &p, hipStream_t stream)
{
    const dim3 grid((unsigned)((long long)p.kv_heads * p.tiles * p.splits));
#define GPTQ_TILE(DP, KT) hipLaunchKernelGGL((attention_tile_kernel<E, DP, KT>), grid, dim3(256), 4 * KT * DP * 2 + 2 * KT * 4 + 16, stream, p)
    if (p.dim <= 64) GPTQ_TILE(64, 64);
    else if (p.dim <= 128) GPTQ_TILE(128, 64);
    else GPTQ_TILE(256, 32);
#undef GPTQ_TILE
}

int launch_attention_tile(const AttentionParams &p, int type, void *stream)
{
    if (type == GPTQ_HIP_TYPE_FP16) launch_tile<_Float16>(p, (hipStream_t)stream);
    else launch_tile<__bf16>(p, (hipStream_t)stream);
    return hipGetLastError() == hipSuccess ? GPTQ_HIP_OK : GPTQ_HIP_ERR_LAUNCH;
}

}  // namespace gptq
