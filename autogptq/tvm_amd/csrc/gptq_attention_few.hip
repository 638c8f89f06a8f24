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
// The division.  Two to four workgroups fill a CU's registers, so a grid with a workgroup for every part that
// a request might have spends its time on those that find none (16 contexts of up to 32768 tokens: 146 us, with the
// division below 70).  Instead a head has `team` workgroups, as many as run at once, and each takes the same number of units
// of up to 256 keys of the requests' tiles, one after the other, in the order of the requests: a workgroup ends one tile, takes
// whole ones and begins another, and leaves at most two parts.  Every wave finds its place from the requests' lengths by
// itself, 64 requests at a time.
//
// Measured (32 heads in groups of 4, dim 128): 16 contexts of 32768 363 us, 5.9 TB/s of keys and values (a plain read of as much: 7.06);
// 64 of up to 32768 under a window of 4096 72.5 us; one of 512 8.5 us, a chain of reads of about 1 us each (lengths, table, keys, values, parts).
#include "gptq_attention.h"

namespace gptq {

constexpr int kFewWaves = 4, kFewUnit = 256;

// Requests [base, base + 64), one a lane.
struct Requests {
    int start, count, context;
    int units, keys;       // of a tile: units, and the keys of one
    int total;             // units of all its tiles
};
template <int R>
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
    r.units = min(max(1, (seen + kFewUnit - 1) / kFewUnit), p.most_units);
    r.keys = max(32, ((seen + r.units - 1) / r.units + 31) / 32 * 32);
    r.total = (int)(((uint32_t)r.count * (uint32_t)p.group + R - 1) / R) * r.units;
    return r;
}
// the sum over the lanes up to this one
__device__ __forceinline__ int sum_upto(int x)
{
#define GPTQ_ADD(CONTROL, ROWS) x += __builtin_amdgcn_update_dpp(0, x, CONTROL, ROWS, 0xf, false)
    GPTQ_ADD(0x111, 0xf);   // within rows of 16: from 1, 2, 4, 8 lanes before
    GPTQ_ADD(0x112, 0xf);
    GPTQ_ADD(0x114, 0xf);
    GPTQ_ADD(0x118, 0xf);
    GPTQ_ADD(0x142, 0xa);   // the last lane of rows 0 and 2 into rows 1 and 3
    GPTQ_ADD(0x143, 0xc);   // that of row 1 into rows 2 and 3
#undef GPTQ_ADD
    return x;
}

// DP: compiled width, the dims past p.dim do not count; FULL: there are none; RT: 16-row operands a wave holds; SHARED: the parts of a
// shared prefix
template <typename E, int DP, bool FULL, int RT, bool SHARED>
__global__ __launch_bounds__(64 * kFewWaves, DP > 128 ? 1 : (RT == 1 ? 3 : 2) + (DP == 64)) void attention_few_kernel(const AttentionParams given)
{
    typedef typename Vec<E>::e8 e8;
    constexpr int R = 16 * RT, NW = kFewWaves;
    constexpr int KS = DP / 32;                    // matrix instructions along dim for S
    constexpr int FIRST = DP == 64 ? 0 : KS / 2;   // the first of them that may hold dims past p.dim (wider kernels take dims above DP / 2)
    constexpr int VE = DP >= 128 ? 8 : DP / 16;    // dims a lane loads of a value row at a time
    constexpr int VH = DP / 16 / VE;               // ... that many times
    constexpr int VW = VE / 2;                     // dwords of that
    constexpr int OD = DP + 4;                     // row of O in LDS
    __shared__ uint32_t list[NW][2][64];
    __shared__ float stat_m[NW][16 * RT], stat_l[NW][16 * RT];
    __shared__ __align__(16) float join[NW * 16 * OD];
    __shared__ int flag;

    // neighbours take different heads: they go to the compute dies in turn, and a head's workgroups to the same one
    const int h = blockIdx.x % given.kv_heads, member = blockIdx.x / given.kv_heads;
    // this workgroup's units [at, stop), and the 64 requests that the first of them lies in or behind
    int at = 0, stop = 1, share = 1, base = 0, before = 0, upto = 0;
    Requests look = {};
    if (!SHARED) {
        look = look_at<R>(given, 0);
        clear_rest(given, given.starts[0], given.starts[given.requests], blockIdx.x * (64ll * kFewWaves) + threadIdx.x, gridDim.x * (64ll * kFewWaves));
        upto = sum_upto(look.total);
        int total = __builtin_amdgcn_readlane(upto, 63);
        for (int b = 64; b < given.requests; b += 64) total += __builtin_amdgcn_readlane(sum_upto(look_at<R>(given, b).total), 63);
        // (Whole tiles of two units rather than their halves, once every CU has a workgroup: the second unit costs less than
        // the join.  32 contexts of 300 tokens, 8 heads: 12.0 us, in halves 13.9; 4 of 512, where CUs are left, 10.4 in halves.)
        share = max((total + given.team - 1) / given.team, total * given.kv_heads > 256 && total <= 2 * given.requests ? 2 : 1);
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
        const char *kbase = (const char *)p.k + (long long)h * p.head_stride * 2;
        const char *vbase = (const char *)p.v + (long long)h * p.head_stride * 2;

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
                look = look_at<R>(p, base);
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
        if (wave < blocks) next = look_up(wave);

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
                const int d = 32 * s + 8 * g;
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
        if constexpr (!FULL) {
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

        if (wave < blocks) {
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
            for (int x = threadIdx.x; x < 16 * (DP / 4); x += 64 * NW) {
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
        look = look_at<R>(p, base);
        upto = sum_upto(look.total);
        __syncthreads();
    }
}

template <typename E, bool SHARED>
static void launch_few(const AttentionParams &p, int rt, hipStream_t stream)
{
    const dim3 grid((unsigned)(p.kv_heads * (SHARED ? p.tiles : p.team)), SHARED ? (unsigned)p.splits : 1u);
#define GPTQ_FEW(DP, RT) \
    if (p.dim == DP) hipLaunchKernelGGL((attention_few_kernel<E, DP, true, RT, SHARED>), grid, dim3(64 * kFewWaves), 0, stream, p); \
    else hipLaunchKernelGGL((attention_few_kernel<E, DP, false, RT, SHARED>), grid, dim3(64 * kFewWaves), 0, stream, p)
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

int launch_attention_few(const AttentionParams &p, int type, int rt, void *stream_v)
{
    hipStream_t stream = (hipStream_t)stream_v;
    if (type == GPTQ_HIP_TYPE_FP16) p.shared ? launch_few<_Float16, true>(p, rt, stream) : launch_few<_Float16, false>(p, rt, stream);
    else p.shared ? launch_few<__bf16, true>(p, rt, stream) : launch_few<__bf16, false>(p, rt, stream);
    return hipGetLastError() == hipSuccess ? GPTQ_HIP_OK : GPTQ_HIP_ERR_LAUNCH;
}

}  // namespace gptq
