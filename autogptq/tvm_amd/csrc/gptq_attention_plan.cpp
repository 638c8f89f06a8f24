// The host side of the attention over a paged cache: argument checks, the choice between the two kernels, and how a call is
// divided among workgroups.
#include <algorithm>
#include <array>

#include "gptq_attention.h"
#include "gptq_mx.h"

namespace gptq {

int check_cache(const gptq_hip_cache *c)
{
    if (!c || !c->k || !c->v || ((uintptr_t)c->k | (uintptr_t)c->v) % 16 != 0) return GPTQ_HIP_ERR_BAD_ARG;
    if (c->type != GPTQ_HIP_TYPE_FP16 && c->type != GPTQ_HIP_TYPE_BF16) return GPTQ_HIP_ERR_BAD_ARG;
    if (c->blocks < 1 || c->block_size < 1 || c->heads < 1 || c->dim < 8 || c->dim % 8 != 0) return GPTQ_HIP_ERR_BAD_ARG;
    if (c->block_stride < 0 || c->slot_stride < 0 || c->head_stride < 0) return GPTQ_HIP_ERR_BAD_ARG;
    if ((c->block_stride | c->slot_stride | c->head_stride) % 8 != 0) return GPTQ_HIP_ERR_BAD_ARG;
    // slots are 32-bit numbers, and so is the place of a row in units of 16 bytes
    if (c->dim > 256 || (long long)c->blocks * c->block_size >= 1ll << 31) return GPTQ_HIP_ERR_UNSUPPORTED;
    const unsigned __int128 rows = (unsigned __int128)(c->blocks - 1) * (unsigned long long)c->block_stride +
                                   (unsigned __int128)(c->block_size - 1) * (unsigned long long)c->slot_stride;
    if (rows / 8 >= 1ull << 32) return GPTQ_HIP_ERR_UNSUPPORTED;
    return GPTQ_HIP_OK;
}

int check_cache_mx(const gptq_hip_cache_mx *c)
{
    if (!c || !c->k || !c->v || !c->k_scales || !c->v_scales || ((uintptr_t)c->k | (uintptr_t)c->v) % 16 != 0) return GPTQ_HIP_ERR_BAD_ARG;
    if (c->type != GPTQ_HIP_TYPE_FP16 && c->type != GPTQ_HIP_TYPE_BF16) return GPTQ_HIP_ERR_BAD_ARG;
    if (c->blocks < 1 || c->block_size < 1 || c->heads < 1 || c->dim < 8 || c->dim % 8 != 0) return GPTQ_HIP_ERR_BAD_ARG;
    if (c->dim > 256 || (long long)c->blocks * c->block_size >= 1ll << 31) return GPTQ_HIP_ERR_UNSUPPORTED;
    const long long scale = mx_scale_bytes(c->dim);
    if (((uintptr_t)c->k_scales | (uintptr_t)c->v_scales) % scale != 0) return GPTQ_HIP_ERR_BAD_ARG;
    for (const auto &[unit, block, slot, head] : {std::array{16ll, c->block_stride, c->slot_stride, c->head_stride},
                                                  std::array{scale, c->scale_block_stride, c->scale_slot_stride, c->scale_head_stride}}) {
        if (block < 0 || slot < 0 || head < 0 || (block | slot | head) % unit != 0) return GPTQ_HIP_ERR_BAD_ARG;
        // the places of rows are 32-bit numbers of units
        const unsigned __int128 rows = (unsigned __int128)(c->blocks - 1) * (unsigned long long)block +
                                       (unsigned __int128)(c->block_size - 1) * (unsigned long long)slot;
        if (rows / unit >= 1ull << 32) return GPTQ_HIP_ERR_UNSUPPORTED;
    }
    return GPTQ_HIP_OK;
}

namespace {

constexpr size_t kAttentionCounters = 65536;             // bytes: one int per (tile, key/value head) of a divided call
constexpr size_t kMostParts = (size_t)1 << 29;           // bytes that the parts of a divided call may take

long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }

// How a launch is divided among workgroups.
struct Division {
    int rt = 0;        // 16-row operands a wave of the few-rows kernel, 0: the tile kernel
    int tiles = 0;     // of rows: all there can be
    int splits = 1, chunk = 1;          // parts of a tile at most, keys of a part
    int even = 0;      // kernel of tiles: the keys of a part follow from the lengths, for this many workgroups
    int team = 1, most_units = 1, unit_bits = 8;       // few-rows kernel on own contexts: see there
    int rows() const { return rt ? 16 * rt : kTileRows; }
};

// Rows of one request and key/value head (on average) up to which the few-rows kernel takes them.
int few_operands(long long rows, int dim)
{
    if (rows <= 16) return 1;
    if (rows <= 32 && dim <= 128) return 2;
    return 0;
}
// Parts of tiles that see `keys` keys: enough that `busy` workgroups become `want`, none of fewer than 256 keys.
void divide(Division &d, long long want, long long busy, long long keys, long long most_parts)
{
    const long long unit = d.rt ? 256 : 64;
    const long long s = std::max(1ll, std::min({ceil_div(want, busy), ceil_div(keys, 256), most_parts}));
    d.chunk = (int)(ceil_div(ceil_div(std::max(keys, 1ll), s), unit) * unit);
    d.splits = (int)std::max(1ll, ceil_div(keys, d.chunk));
}
// Own contexts on the tile kernel: two workgroups a CU (also where it holds three: 768 for dim 64 bring nothing), since they differ in length (32 heads in groups of 4; us with 256, 512 and
// 1024 workgroups: 16 pieces of 20 tokens behind 2048 keys, dim 128: 43, 40, 53, dim 256: 85, 100, 127; 8 of 256 behind 4096: dim
// 128: 161, 160, 190, dim 256: 431, 431, 510; 723 tokens of 7 heads behind up to 9001, dim 80: 94, 71, 81).  A shared prefix: parts of one length, which the
// next launch reads again, so one a CU (512 rows behind 16384 keys: 256 workgroups 80 us, 512 84, 1024 111); rows that fit the
// few-rows kernel two.
constexpr long long kOwnWorkgroups = 512, kPrefixWorkgroups = 256;

constexpr long long kMostPrefixParts = 1024;

struct Plan {
    Division own, shared, few;
    bool prefix = false;             // a launch of its own for the shared prefix
    bool mixed = false;              // `few` for requests of up to few.rows() rows, `own` for the others
    size_t prefix_rows = 0, own_rows = 0, bytes = 0;     // rows of the parts in the workspace
};

// mx: the cache is held in MXFP4
int plan(const gptq_hip_attention &a, bool mx, Plan &pl)
{
    const long long group = a.heads / a.cache.heads, T = a.tokens, B = a.requests, H = a.cache.heads;
    const long long all = T * a.heads, row = a.cache.dim * 4 + 8;
    const long long room = std::max(1ll, (long long)(kMostParts / (size_t)(all * row)));
    Division &d = pl.own;
    d.rt = few_operands(ceil_div(T * group, B), a.cache.dim);
    d.tiles = (int)(T * group / d.rows() + B);
    if (d.tiles * H >= 1ll << 24) return GPTQ_HIP_ERR_UNSUPPORTED;
    long long keys = (long long)a.table_width * a.cache.block_size;
    if (a.max_context > 0) keys = std::min<long long>(keys, a.max_context);
    if (a.window > 0) keys = std::min<long long>(keys, (long long)a.window + a.sinks + d.rows() / group + 1);
    // A short prefix stands in front of every request's keys instead of taking a launch of its own, which costs 4 us and less
    // as the tiles read it again (32 heads in groups of 4, dim 128): 8 requests behind 1000 keys 11.3 us against 15.4, 16
    // behind 1000 14.1 / 17.5, 64 behind 250 17.1 / 22.0, 8 behind 4000 17.2 / 17.8, 16 behind 2000 21.5 / 18.0, 32 behind 1000
    // 23.8 / 18.9.  A cache in MXFP4, whose re-reads are a quarter of the bytes, has it there a little longer: 16 behind 2000 14.2 / 20.5,
    // behind 4000 18.3 / 21.7, 64 behind 1000 21.9 / 27.0, 8 behind 16000 30.3 / 28.8.
    const bool alone = B == 1 && T * group <= d.rows();      // no other reader
    pl.prefix = a.prefix_length > 0 &&
                !(d.rt && (alone || (long long)d.tiles * a.prefix_length * H * a.cache.dim * 4 <= (mx ? 384ll : 256ll) << 20));
    if (pl.prefix) {
        Division &s = pl.shared;
        s.rt = few_operands(T * group, a.cache.dim);
        s.tiles = (int)ceil_div(T * group, s.rows());
        // (MXFP4, us with 256 and 512 workgroups: few rows, 8 behind 16384 21.6 / 27.7, 4 behind 32768 22.2 / 26.5; tiles, where two share a CU's
        // matrix pipes and its conversions, 128 behind 32768 119 / 107.5, behind 16384 73.6 / 71.0, in parts of 512 keys 64 behind 16384
        // 49.0 / 52.3, 128 behind 8192 49.8 / 50.8.)
        const bool two = mx ? !s.rt && a.cache.dim <= 128 && s.tiles * H * a.prefix_length >= 512ll * 1024 : s.rt != 0;
        divide(s, two ? 2 * kPrefixWorkgroups : kPrefixWorkgroups, s.tiles * H, a.prefix_length, std::min(room, kMostPrefixParts));
        pl.prefix_rows = (size_t)(s.splits * all);
    } else {
        keys += a.prefix_length;
    }
    // the few-rows kernel on own contexts, with d.tiles tiles
    auto by_units = [&](Division &d) {
        const long long most = B * (T * group / d.rows() + 1);    // tiles, whatever the lengths on the GPU say
        if (most > 1ll << 30) return GPTQ_HIP_ERR_UNSUPPORTED;
        d.most_units = (int)std::min((1ll << 30) / most, 1ll << 20);
        // MXFP4: units of 128 keys in place of 256 where each of them has a CU to itself, since a wave's second 32 keys wait for memory once more; not
        // for one unit, which needs no join, nor for more than eight.  (Contexts of single tokens, 8 key/value heads, us in units of 128 and 256: one of 200 7.5 / 6.5,
        // 300 7.5 / 8.1, 512 7.5 / 8.1, 640 7.6 / 8.1, 768 7.8 / 8.2, 1024 8.0 / 8.2, 1536 8.8 / 8.3; four of 1024, 256 units, 8.1 / 8.3; eight of 512, 256 units, 7.8 / 8.2, of
        // 520, 320 units, 8.4 / 8.2; sixteen of 300, 384 units, 8.5 / 8.3; dim 256, three of 768 9.0 / 9.5.)
        const long long team = 256ll * few_resident(d.rt, a.cache.dim, mx) / H;
        if (mx && keys > 256 && keys <= 1024 && B * H * ceil_div(keys, 128) <= 256) d.unit_bits = 7;
        const long long units = (d.tiles + 0ll) * std::max(1ll, ceil_div(keys, 1ll << d.unit_bits));
        d.team = (int)std::max(1ll, std::min(team, units));
        if (d.team * H > (long long)(kAttentionCounters / 4)) return GPTQ_HIP_ERR_UNSUPPORTED;
        pl.own_rows = std::max(pl.own_rows, (size_t)(2 * d.team * H * d.rows()));
        return GPTQ_HIP_OK;
    };
    if (d.rt) {
        const int rc = by_units(d);
        if (rc != GPTQ_HIP_OK) return rc;
    } else {
        // MXFP4: single tokens that a batch of pieces may hold have a launch of the few-rows kernel to themselves, where they would cost
        // the kernel of tiles more than such a launch finds nothing in.  (us without and with it: 63 up to 32768 and a piece of 512 behind
        // 4096 646 / 126, 7 up to 8192 and 256 behind 2044 72 / 59, 63 up to 4000 and a prompt of 2048 151 / 102, with 2 key/value
        // heads 7 up to 16384 and 512 behind 4096 58.0 / 55.4; nothing in it: 32 of 64 behind 4096 225 / 227; below the bound 8 of
        // 128 behind 4096 102 / 104, 3 up to 2500 and 256 behind 2044, 2 heads, 25 / 34.  Long pieces among so many single tokens that
        // the mean fits the few-rows kernel stay there: 255 up to 1000 and 1024 behind 7168 236, in two launches 259.)
        Division &f = pl.few;
        f.rt = few_operands(group, a.cache.dim);
        f.tiles = (int)B;
        pl.mixed = mx && f.rt && B > 1 && B * H * keys >= 512ll * 1024 && by_units(f) == GPTQ_HIP_OK;
        const bool even = mx && B > 1 && B <= kEvenRequests && keys >= 6144;
        long long busy = std::max(pl.mixed && even ? 1 : B, ceil_div(T * group, d.rows())) * H;
        // MXFP4: no more parts than the card holds workgroups (512, of rows of more than 128 dims 256), and none where every CU has a tile of up
        // to 2048 keys, since the parts' way through memory and their join cost some 17 us.  (8 key/value heads, us so and in parts for 512
        // workgroups: 32 pieces of 32 tokens behind 512 22 / 39, 1024 35 / 47, 2048 61 / 66, 4096 103 / 102; 20 of 20, two parts or four,
        // behind 1024 32 / 40, 4096 65 / 78; dim 256, 24 of 20 behind 1024 71 / 105, 4096 245 / 297, 40 of 20 behind 512 83 / 101,
        // 4096, where 320 tiles would wait for one another, in two parts 445, undivided 535.)
        long long want = kOwnWorkgroups;
        if (mx && !even) {
            busy = B * ceil_div(T * group, B * d.rows()) * H;      // (as many as requests of one length have)
            if (a.cache.dim > 128) want /= 2;
            if (busy >= 256 && keys <= 2048) want = 1;
            else if (a.cache.dim > 128 && busy > want) want = 2 * want;
            else want = std::max(1ll, want / busy) * busy;
        }
        divide(d, want, busy, keys, room);
        // MXFP4: parts by the lengths on the GPU (even_keys).  8 key/value heads, us by the longest context and so: lengths of all sizes, 3 pieces of up to 300 tokens
        // behind up to 20000 keys 163 / 110, 10 of up to 64 161 / 74, 20 of up to 33 behind 16000 134 / 73, 200 of 20 to 60 behind 8000, 2 heads, 245 / 157, 30 of
        // 30 to 60 behind 7000 166 / 105; the same from half the longest on 216 / 215, all alike 229 / 242; 12 of 130 behind 12000, alike, 393 / 407.  From 2048 keys
        // on: 24 of 50 behind 3000, of all sizes 79 / 54, from half on 99 / 106, alike 108 / 119: there the finding costs too large a share.
        if (even && d.splits > 1) {
            d.even = (int)(a.cache.dim > 128 ? kOwnWorkgroups / 2 : kOwnWorkgroups);     // (as many as the card holds)
            d.splits = (int)std::max(1ll, std::min({2ll * d.splits, ceil_div(keys, 256), room}));
        }
        if (d.splits > 1 || pl.prefix) pl.own_rows = std::max(pl.own_rows, (size_t)(d.splits * all));
    }
    const size_t rows = pl.prefix_rows + pl.own_rows;
    pl.bytes = rows ? kAttentionCounters + (rows * 8 + 255) / 256 * 256 + rows * a.cache.dim * 4 : 0;
    return GPTQ_HIP_OK;
}

// rc: what the checks of the cache said
int check(const gptq_hip_attention *a, int rc)
{
    if (!a) return GPTQ_HIP_ERR_BAD_ARG;
    if (rc != GPTQ_HIP_OK) return rc;
    if (a->tokens < 0 || a->requests < 0 || a->table_width < 0 || a->max_context < 0 || a->window < 0 || a->sinks < 0 ||
        a->prefix_length < 0)
        return GPTQ_HIP_ERR_BAD_ARG;
    if (a->heads < 1 || a->heads % a->cache.heads != 0 || !(a->scale > 0.0f) || a->scale > 3e38f) return GPTQ_HIP_ERR_BAD_ARG;
    if (a->prefix_length > 0 && (a->window > 0 || !a->prefix_blocks)) return GPTQ_HIP_ERR_BAD_ARG;
    if (a->tokens == 0) return GPTQ_HIP_OK;
    if (a->requests < 1 || !a->q || !a->out || !a->starts || !a->contexts || (a->table_width > 0 && !a->tables)) return GPTQ_HIP_ERR_BAD_ARG;
    if (((uintptr_t)a->q | (uintptr_t)a->out) % 16 != 0 || (a->q_token_stride | a->q_head_stride) % 8 != 0) return GPTQ_HIP_ERR_BAD_ARG;
    if (a->table_stride < a->table_width) return GPTQ_HIP_ERR_BAD_ARG;
    // row numbers are 32-bit
    if ((long long)a->tokens * a->heads >= 1ll << 30 || a->requests >= 1 << 24 ||
        a->prefix_length > kMostKeys)
        return GPTQ_HIP_ERR_UNSUPPORTED;
    return GPTQ_HIP_OK;
}

// mx: nullptr, or the cache in MXFP4, whose shape is a.cache's
int attend(const gptq_hip_attention *a, const gptq_hip_cache_mx *mx, void *workspace, size_t workspace_bytes, void *stream)
{
    Plan pl;
    int rc = plan(*a, mx != nullptr, pl);
    if (rc != GPTQ_HIP_OK) return rc;
    if (pl.bytes && (!workspace || (uintptr_t)workspace % 16 != 0 || workspace_bytes < pl.bytes)) return GPTQ_HIP_ERR_WORKSPACE;

    AttentionParams p = {};
    const gptq_hip_cache &c = a->cache;
    p.q = a->q, p.k = c.k, p.v = c.v, p.out = a->out;
    if (pl.bytes) {
        const size_t rows = pl.prefix_rows + pl.own_rows;
        p.counters = (int *)workspace;
        p.stats = (float *)((char *)workspace + kAttentionCounters);
        p.parts = (float *)((char *)p.stats + (rows * 8 + 255) / 256 * 256);
        p.own_stats = p.stats + 2 * pl.prefix_rows;
        p.own_parts = p.parts + pl.prefix_rows * c.dim;
    }
    p.tokens = a->tokens, p.requests = a->requests, p.heads = a->heads, p.kv_heads = c.heads, p.group = a->heads / c.heads;
    p.dim = c.dim, p.blocks = c.blocks, p.block_size = c.block_size;
    p.q_token = a->q_token_stride, p.q_head = a->q_head_stride;
    if (mx) {
        const long long scales = mx_scale_bytes(c.dim);
        p.head_stride = mx->head_stride, p.block_step = (uint32_t)(mx->block_stride / 16), p.slot_step = (uint32_t)(mx->slot_stride / 16);
        p.k_scales = mx->k_scales, p.v_scales = mx->v_scales, p.scale_head = mx->scale_head_stride;
        p.scale_block = (uint32_t)(mx->scale_block_stride / scales), p.scale_slot = (uint32_t)(mx->scale_slot_stride / scales);
    } else {
        p.head_stride = c.head_stride, p.block_step = (uint32_t)(c.block_stride / 8), p.slot_step = (uint32_t)(c.slot_stride / 8);
    }
    p.c = a->scale * 1.44269504088896340736f;
    if ((long long)p.group * (p.group + kTileRows) < 65536) p.group_magic = 65535u / (uint32_t)p.group + 1u;
    p.block_shift = c.block_size & (c.block_size - 1) ? -1 : __builtin_ctz((unsigned)c.block_size);
    while (p.block_bits < 31 && 1ll << p.block_bits < c.block_size) p.block_bits++;
    p.block_magic = (uint32_t)(((1ull << (29 + p.block_bits)) + (unsigned)c.block_size - 1) / (unsigned)c.block_size);
    auto launch = [&](const Division &d) {
        p.tiles = d.tiles, p.splits = d.splits, p.chunk = d.chunk, p.team = d.team, p.most_units = d.most_units, p.unit_bits = d.unit_bits, p.even = d.even;
        if (d.rt) return mx ? launch_attention_few_mx(p, c.type, d.rt, stream) : launch_attention_few(p, c.type, d.rt, stream);
        return mx ? launch_attention_tile_mx(p, c.type, stream) : launch_attention_tile(p, c.type, stream);
    };
    p.prefix_blocks = a->prefix_blocks;
    if (pl.prefix) {
        p.shared = 1, p.prefix = a->prefix_length;
        rc = launch(pl.shared);
        if (rc != GPTQ_HIP_OK) return rc;
        p.shared = 0, p.prefix_parts = pl.shared.splits;
    } else {
        p.front = a->prefix_length;
    }
    p.tables = a->tables, p.table_width = a->table_width, p.table_stride = a->table_stride;
    p.starts = a->starts, p.contexts = a->contexts;
    p.window = std::min(a->window, kMostKeys), p.sinks = std::min(a->sinks, kMostKeys);
    if (pl.mixed) {      // (both keep their parts at the same place, one after the other)
        p.few_rows = pl.few.rows();
        rc = launch(pl.few);
        if (rc != GPTQ_HIP_OK) return rc;
    }
    return launch(pl.own);
}

// a call on a cache in MXFP4, with that cache's shape
gptq_hip_attention with_shape_of(const gptq_hip_attention &a, const gptq_hip_cache_mx &mx)
{
    gptq_hip_attention b = a;
    b.cache = {mx.k, mx.v, mx.type, mx.blocks, mx.block_size, mx.heads, mx.dim, 0, 0, 0};
    return b;
}

}  // namespace
}  // namespace gptq

extern "C" size_t gptq_hip_attention_workspace_bytes(const gptq_hip_attention *a)
{
    gptq::Plan pl;
    if (!a || gptq::check(a, gptq::check_cache(&a->cache)) != GPTQ_HIP_OK || a->tokens == 0 || gptq::plan(*a, false, pl) != GPTQ_HIP_OK) return 0;
    return pl.bytes;
}

extern "C" int gptq_hip_attend(const gptq_hip_attention *a, void *workspace, size_t workspace_bytes, void *stream)
{
    if (!a) return GPTQ_HIP_ERR_BAD_ARG;
    const int rc = gptq::check(a, gptq::check_cache(&a->cache));
    if (rc != GPTQ_HIP_OK || a->tokens == 0) return rc;
    return gptq::attend(a, nullptr, workspace, workspace_bytes, stream);
}

extern "C" size_t gptq_hip_attention_mx_workspace_bytes(const gptq_hip_cache_mx *cache, const gptq_hip_attention *given)
{
    if (!cache || !given) return 0;
    const gptq_hip_attention a = gptq::with_shape_of(*given, *cache);
    gptq::Plan pl;
    if (gptq::check(&a, gptq::check_cache_mx(cache)) != GPTQ_HIP_OK || a.tokens == 0 || gptq::plan(a, true, pl) != GPTQ_HIP_OK) return 0;
    return pl.bytes;
}

extern "C" int gptq_hip_attend_mx(const gptq_hip_cache_mx *cache, const gptq_hip_attention *given, void *workspace, size_t workspace_bytes, void *stream)
{
    if (!cache || !given) return GPTQ_HIP_ERR_BAD_ARG;
    const gptq_hip_attention a = gptq::with_shape_of(*given, *cache);
    const int rc = gptq::check(&a, gptq::check_cache_mx(cache));
    if (rc != GPTQ_HIP_OK || a.tokens == 0) return rc;
    return gptq::attend(&a, cache, workspace, workspace_bytes, stream);
}
