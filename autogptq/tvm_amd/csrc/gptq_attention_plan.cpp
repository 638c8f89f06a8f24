// The host side of the attention over a paged cache: argument checks, the choice between the two kernels, and how a call is
// divided among workgroups.
#include <algorithm>

#include "gptq_attention.h"

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

namespace {

constexpr size_t kAttentionCounters = 65536;             // bytes: one int per (tile, key/value head) of a divided call
constexpr size_t kMostParts = (size_t)1 << 29;           // bytes that the parts of a divided call may take

long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }

// How a launch is divided among workgroups.
struct Division {
    int rt = 0;        // 16-row operands a wave of the few-rows kernel, 0: the tile kernel
    int tiles = 0;     // of rows: all there can be
    int splits = 1, chunk = 1;          // parts of a tile at most, keys of a part
    int team = 1, most_units = 1;       // few-rows kernel on own contexts: see there
    int rows() const { return rt ? 16 * rt : kTileRows; }
};

// Rows of one request and key/value head (on average) up to which the few-rows kernel takes them.
int few_operands(long long rows, int dim)
{
    if (rows <= 16) return 1;
    if (rows <= 32 && dim <= 128) return 2;
    return 0;
}
// workgroups of the few-rows kernel that a CU holds (registers)
int few_resident(int rt, int dim) { return dim > 128 ? 1 : (rt == 1 ? 3 : 2) + (dim <= 64); }

// Parts of tiles that see `keys` keys: enough that `busy` workgroups become `want`, none of fewer than 256 keys.
void divide(Division &d, long long want, long long busy, long long keys, long long most_parts)
{
    const long long unit = d.rt ? 256 : 64;
    const long long s = std::max(1ll, std::min({ceil_div(want, busy), ceil_div(keys, 256), most_parts}));
    d.chunk = (int)(ceil_div(ceil_div(std::max(keys, 1ll), s), unit) * unit);
    d.splits = (int)std::max(1ll, ceil_div(keys, d.chunk));
}
// Own contexts on the tile kernel: two workgroups a CU (also where it holds three: 768 for dim 64 bring nothing), since they differ in length (32 heads in groups of 4; us with 256, 512 and
// 1024 workgroups: 16 pieces of 20 tokens behind 2048 keys, dim 128: 51, 54, 62, dim 256: 136, 124, 140; 8 of 256 behind 4096: dim
// 128: 182, 181, 216, dim 256: 462, 464, 542; 723 tokens of 7 heads behind up to 9001, dim 80: 107, 87, 90).  A shared prefix: parts of one length, which the
// next launch reads again, so one a CU (512 rows behind 16384 keys: 256 workgroups 80 us, 512 84, 1024 111); rows that fit the
// few-rows kernel two.
constexpr long long kOwnWorkgroups = 512, kPrefixWorkgroups = 256;

constexpr long long kMostPrefixParts = 1024;

struct Plan {
    Division own, shared;
    bool prefix = false;             // a launch of its own for the shared prefix
    size_t prefix_rows = 0, own_rows = 0, bytes = 0;     // rows of the parts in the workspace
};

int plan(const gptq_hip_attention &a, Plan &pl)
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
    // 23.8 / 18.9.
    const bool alone = B == 1 && T * group <= d.rows();      // no other reader
    pl.prefix = a.prefix_length > 0 &&
                !(d.rt && (alone || (long long)d.tiles * a.prefix_length * H * a.cache.dim * 4 <= 256ll << 20));
    if (pl.prefix) {
        Division &s = pl.shared;
        s.rt = few_operands(T * group, a.cache.dim);
        s.tiles = (int)ceil_div(T * group, s.rows());
        divide(s, s.rt ? 2 * kPrefixWorkgroups : kPrefixWorkgroups, s.tiles * H, a.prefix_length, std::min(room, kMostPrefixParts));
        pl.prefix_rows = (size_t)(s.splits * all);
    } else {
        keys += a.prefix_length;
    }
    if (d.rt) {
        const long long most = B * (T * group / d.rows() + 1);    // tiles, whatever the lengths on the GPU say
        if (most > 1ll << 30) return GPTQ_HIP_ERR_UNSUPPORTED;
        d.most_units = (int)std::min((1ll << 30) / most, 1ll << 20);
        const long long units = (d.tiles + 0ll) * std::max(1ll, ceil_div(keys, 256));
        d.team = (int)std::max(1ll, std::min(256ll * few_resident(d.rt, a.cache.dim) / H, units));
        if (d.team * H > (long long)(kAttentionCounters / 4)) return GPTQ_HIP_ERR_UNSUPPORTED;
        pl.own_rows = (size_t)(2 * d.team * H * d.rows());
    } else {
        divide(d, kOwnWorkgroups, std::max(B, ceil_div(T * group, d.rows())) * H, keys, room);
        if (d.splits > 1 || pl.prefix) pl.own_rows = (size_t)(d.splits * all);
    }
    const size_t rows = pl.prefix_rows + pl.own_rows;
    pl.bytes = rows ? kAttentionCounters + (rows * 8 + 255) / 256 * 256 + rows * a.cache.dim * 4 : 0;
    return GPTQ_HIP_OK;
}

int check(const gptq_hip_attention *a)
{
    if (!a) return GPTQ_HIP_ERR_BAD_ARG;
    const int rc = check_cache(&a->cache);
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

}  // namespace
}  // namespace gptq

extern "C" size_t gptq_hip_attention_workspace_bytes(const gptq_hip_attention *a)
{
    gptq::Plan pl;
    if (gptq::check(a) != GPTQ_HIP_OK || a->tokens == 0 || gptq::plan(*a, pl) != GPTQ_HIP_OK) return 0;
    return pl.bytes;
}

extern "C" int gptq_hip_attend(const gptq_hip_attention *a, void *workspace, size_t workspace_bytes, void *stream)
{
    int rc = gptq::check(a);
    if (rc != GPTQ_HIP_OK || a->tokens == 0) return rc;
    gptq::Plan pl;
    rc = gptq::plan(*a, pl);
    if (rc != GPTQ_HIP_OK) return rc;
    if (pl.bytes && (!workspace || (uintptr_t)workspace % 16 != 0 || workspace_bytes < pl.bytes)) return GPTQ_HIP_ERR_WORKSPACE;

    gptq::AttentionParams p = {};
    const gptq_hip_cache &c = a->cache;
    p.q = a->q, p.k = c.k, p.v = c.v, p.out = a->out;
    if (pl.bytes) {
        const size_t rows = pl.prefix_rows + pl.own_rows;
        p.counters = (int *)workspace;
        p.stats = (float *)((char *)workspace + gptq::kAttentionCounters);
        p.parts = (float *)((char *)p.stats + (rows * 8 + 255) / 256 * 256);
        p.own_stats = p.stats + 2 * pl.prefix_rows;
        p.own_parts = p.parts + pl.prefix_rows * c.dim;
    }
    p.tokens = a->tokens, p.requests = a->requests, p.heads = a->heads, p.kv_heads = c.heads, p.group = a->heads / c.heads;
    p.dim = c.dim, p.blocks = c.blocks, p.block_size = c.block_size;
    p.q_token = a->q_token_stride, p.q_head = a->q_head_stride;
    p.head_stride = c.head_stride, p.block_step = (uint32_t)(c.block_stride / 8), p.slot_step = (uint32_t)(c.slot_stride / 8);
    p.c = a->scale * 1.44269504088896340736f;
    if ((long long)p.group * (p.group + gptq::kTileRows) < 65536) p.group_magic = 65535u / (uint32_t)p.group + 1u;
    p.block_shift = c.block_size & (c.block_size - 1) ? -1 : __builtin_ctz((unsigned)c.block_size);
    auto launch = [&](const gptq::Division &d) {
        p.tiles = d.tiles, p.splits = d.splits, p.chunk = d.chunk, p.team = d.team, p.most_units = d.most_units;
        return d.rt ? gptq::launch_attention_few(p, c.type, d.rt, stream) : gptq::launch_attention_tile(p, c.type, stream);
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
    p.window = std::min(a->window, gptq::kMostKeys), p.sinks = std::min(a->sinks, gptq::kMostKeys);
    return launch(pl.own);
}
