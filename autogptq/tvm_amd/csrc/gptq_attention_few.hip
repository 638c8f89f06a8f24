// Attention over a paged cache for few rows a request: single tokens, drafts of a few, small groups of shared heads.
//
// What bounds it: memory.  Every visible key and value is read once (4 dim bytes in all), for 4 dim flops a row, and a tile
// has 16 RT rows.  So the kernel is a stream: four waves of a workgroup take every fourth group of 64 keys of the part and
// load keys and values straight into the registers of the matrix instructions, without LDS and without a barrier, the next
// 32 keys' loads in flight while the present ones are used.
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
// The four waves join through LDS at the end, parts of a tile through the workspace (the workgroup that is last adds them
// in order).
#include "gptq_attention.h"

namespace gptq {

// DP: compiled width, dims past p.dim are zero; RT: 16-row operands a wave holds
template <typename E, int DP, int RT>
__global__ __launch_bounds__(256) void attention_few_kernel(const AttentionParams p)
{
    typedef typename Vec<E>::e8 e8;
    constexpr int R = 16 * RT;
    constexpr int KS = DP / 32;                    // matrix instructions along dim for S
    constexpr int VE = DP >= 128 ? 8 : DP / 16;    // dims a lane loads of a value row at a time
    constexpr int VH = DP / 16 / VE;               // ... that many times
    constexpr int VW = VE / 2;                     // dwords of that
    constexpr int OD = DP + 4;                     // row of O in LDS
    __shared__ uint32_t list[4][2][64];
    __shared__ float stat_m[4][16 * RT], stat_l[4][16 * RT];
    __shared__ __align__(16) float join[4 * 16 * OD > kJoinWeights ? 4 * 16 * OD : kJoinWeights];
    __shared__ int flag;

    const int lane = threadIdx.x & 63, i16 = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    // heads of a tile side by side: they go to the compute dies in turn, and a head's tiles to the same one
    const int h = blockIdx.x % p.kv_heads, rest = blockIdx.x / p.kv_heads;
    const int tile = rest % p.tiles, split = rest / p.tiles;
    QueryTile q;
    if (!find_tile<R>(p, tile, q)) return;
    int chunk;
    const int parts = tile_parts(p, q.seen, 256, chunk);
    if (split >= parts) return;
    const int begin = split * chunk, end = min(q.seen, begin + chunk);
    const int32_t *table = p.tables + (p.shared ? 0 : (long long)q.b * p.table_stride);
    const char *kbase = (const char *)p.k + (long long)h * p.head_stride * 2;
    const char *vbase = (const char *)p.v + (long long)h * p.head_stride * 2;

    // the query rows as B operands, and their positions
    e8 qf[RT][KS];
    int pos[RT];
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        const int r = 16 * rt + i16;
        const int row = q.row0 + min(r, q.rows - 1), t = row / p.group, hg = h * p.group + row - t * p.group;
        pos[rt] = q.position + t;
        const char *src = (const char *)p.q + ((long long)(q.start + t) * p.q_token + (long long)hg * p.q_head) * 2;
#pragma unroll
        for (int s = 0; s < KS; s++) {
            const int d = 32 * s + 8 * g;
            u4 x = {0u, 0u, 0u, 0u};
            if (d < p.dim) x = *(const u4 *)(src + d * 2);
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

    const int groups = (end - begin + 63) / 64;
    u4 kr[2][KS];
    uint32_t vr[8][VH][VW];
    // the row of the list's entry that this lane looks up in a group (past the end: the last one's again)
    auto look_up = [&](int n) { return key_row(p, table, key_position(q, min(begin + n * 64 + lane, end - 1))); };
    auto load_keys = [&](const uint32_t *rows, int half) {
#pragma unroll
        for (int a = 0; a < 2; a++) {
            const char *src = kbase + (unsigned long long)rows[32 * half + 16 * a + i16] * 16;
#pragma unroll
            for (int s = 0; s < KS; s++) {
                const int d = 32 * s + 8 * g;
                kr[a][s] = (u4){0u, 0u, 0u, 0u};
                if (DP == p.dim || d < p.dim) kr[a][s] = *(const u4 *)(src + d * 2);
            }
        }
    };
    auto load_values = [&](const uint32_t *rows, int half) {
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const char *src = vbase + (unsigned long long)rows[32 * half + 16 * (j / 4) + 4 * g + j % 4] * 16;
#pragma unroll
            for (int vh = 0; vh < VH; vh++) {
                const int d = 128 * vh + VE * i16;
                const bool in = DP == p.dim || d < p.dim;
                if constexpr (VW == 4) {
                    u4 x = {0u, 0u, 0u, 0u};
                    if (in) x = *(const u4 *)(src + d * 2);
#pragma unroll
                    for (int w = 0; w < 4; w++) vr[j][vh][w] = x[w];
                } else {
                    u2 x = {0u, 0u};
                    if (in) x = *(const u2 *)(src + d * 2);
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

    if (wave < groups) {
        uint32_t next = look_up(wave);
        list[wave][0][lane] = next;
        hand_over();
        load_keys(list[wave][0], 0);
        load_values(list[wave][0], 0);
        next = look_up(min(wave + 4, groups - 1));
        int turn = 0;
        for (int n = wave; n < groups; n += 4, turn ^= 1) {
            list[wave][turn ^ 1][lane] = next;
            hand_over();
            next = look_up(min(n + 8, groups - 1));
            const uint32_t *rows = list[wave][turn], *rows_next = list[wave][turn ^ 1];
#pragma unroll
            for (int half = 0; half < 2; half++) {
                const int v0 = begin + n * 64 + 32 * half;
                if (half == 1 && v0 >= end) break;
                // S^T of 32 keys
                f4 s[RT][2];
#pragma unroll
                for (int rt = 0; rt < RT; rt++)
#pragma unroll
                    for (int a = 0; a < 2; a++) {
                        s[rt][a] = (f4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                        for (int x = 0; x < KS; x++) s[rt][a] = mfma16(__builtin_bit_cast(e8, kr[a][x]), qf[rt][x], s[rt][a]);
                    }
                if (half == 0) load_keys(rows, 1);
                else load_keys(rows_next, 0);
                // what a row does not see
                const bool tail = v0 + 32 > end;
                const bool mixed = q.t0 != q.t1 && !p.shared &&
                                   !(v0 >= q.ns && key_position(q, v0 + 31) <= q.position + q.t0 &&
                                     (p.window <= 0 || key_position(q, v0) > q.position + q.t1 - p.window));
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
                        for (int e = 0; e < 4; e++) {
#pragma unroll
                            for (int rt = 0; rt < RT; rt++) {
                                const bool seen = sees(p, q, v0 + 16 * a + 4 * g + e, end, pos[rt]);
                                s[rt][a][e] = seen ? s[rt][a][e] : kNone;
                            }
                        }
                }
                // the operands of V: 8 keys of this lane's group, one dim each
                e8 vt[VH][VE];
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
                        vt[vh][2 * w] = __builtin_bit_cast(e8, even);
                        vt[vh][2 * w + 1] = __builtin_bit_cast(e8, odd);
                    }
                if (half == 0) load_values(rows, 1);
                else load_values(rows_next, 0);
#pragma unroll
                for (int rt = 0; rt < RT; rt++) {
                    float top = fmaxf(fmaxf(fmaxf(s[rt][0][0], s[rt][0][1]), fmaxf(s[rt][0][2], s[rt][0][3])),
                                      fmaxf(fmaxf(s[rt][1][0], s[rt][1][1]), fmaxf(s[rt][1][2], s[rt][1][3])));
                    top = max_quarters(top);
                    if (__ballot(top > m[rt] + 8.0f)) {
                        const float up = fmaxf(m[rt], top);
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
                    const e8 pe = __builtin_convertvector(pr, e8);
#pragma unroll
                    for (int vh = 0; vh < VH; vh++)
#pragma unroll
                        for (int t = 0; t < VE; t++) o[rt][vh][t] = mfma16(vt[vh][t], pe, o[rt][vh][t]);
                }
            }
        }
    }

    // the four waves of a part, 16 rows at a time
    const bool whole = parts == 1 && p.first_slot == 0 && !p.shared;
    const long long all = (long long)p.tokens * p.heads;
    const long long slot = (long long)(p.first_slot + split) * all;
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        l[rt] = add_quarters(l[rt]);
        if (g == 0) stat_m[wave][16 * rt + i16] = m[rt], stat_l[wave][16 * rt + i16] = l[rt];
    }
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        if (rt > 0) __syncthreads();
        float *mine = join + (wave * 16 + i16) * OD;
#pragma unroll
        for (int vh = 0; vh < VH; vh++)
#pragma unroll
            for (int e = 0; e < 4; e++)
#pragma unroll
                for (int t = 0; t < VE; t += 4)
                    *(f4 *)(mine + 128 * vh + VE * (4 * g + e) + t) = (f4){o[rt][vh][t][e], o[rt][vh][t + 1][e], o[rt][vh][t + 2][e], o[rt][vh][t + 3][e]};
        __syncthreads();
        for (int x = threadIdx.x; x < 16 * (DP / 4); x += 256) {
            const int r = x / (DP / 4), d = x % (DP / 4) * 4, row = 16 * rt + r;
            if (row >= q.rows || d >= p.dim) continue;
            float top = kNone, sum = 0.0f;
#pragma unroll
            for (int w = 0; w < 4; w++) top = fmaxf(top, stat_m[w][row]);
            const float ref = reference(top);
            f4 total = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int w = 0; w < 4; w++) {
                const float f = __builtin_amdgcn_exp2f(stat_m[w][row] - ref);
                const f4 y = *(const f4 *)(join + (w * 16 + r) * OD + d);
                sum += f * stat_l[w][row];
#pragma unroll
                for (int e = 0; e < 4; e++) total[e] += f * y[e];
            }
            const long long at = out_row(p, q, h, row);
            if (whole) {
                store_row4<E>(p.out, at * p.dim + d, total * (sum > 0.0f ? 1.0f / sum : 0.0f));
            } else {
                store_partial(p.parts + (slot + at) * p.dim + d, total);
                if (d == 0) store_stats(p.stats + 2 * (slot + at), top, sum);
            }
        }
    }
    if (whole || p.shared) return;
    if (last_part(p, tile * p.kv_heads + h, parts, &flag))
        join_parts<E, 256>(p, q, h, p.first_slot + parts, join);
}

template <typename E>
static void launch_few(const AttentionParams &p, int rt, hipStream_t stream)
{
    const dim3 grid((unsigned)((long long)p.kv_heads * p.tiles * p.splits));
#define GPTQ_FEW(DP, RT) hipLaunchKernelGGL((attention_few_kernel<E, DP, RT>), grid, dim3(256), 0, stream, p)
    if (p.dim <= 64) {
        if (rt == 1) GPTQ_FEW(64, 1);
        else GPTQ_FEW(64, 2);
    } else if (p.dim <= 128) {
        if (rt == 1) GPTQ_FEW(128, 1);
        else GPTQ_FEW(128, 2);
    } else {
        GPTQ_FEW(256, 1);
    }
#undef GPTQ_FEW
}

int launch_attention_few(const AttentionParams &p, int type, int rt, void *stream)
{
    if (type == GPTQ_HIP_TYPE_FP16) launch_few<_Float16>(p, rt, (hipStream_t)stream);
    else launch_few<__bf16>(p, rt, (hipStream_t)stream);
    return hipGetLastError() == hipSuccess ? GPTQ_HIP_OK : GPTQ_HIP_ERR_LAUNCH;
}

}  // namespace gptq
