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

struct Division {
    int rt = 0;       // 16-row operands a wave of the few-rows kernel, 0: the tile kernel
    int tiles = 0, splits = 1, chunk = 1;
    int rows() const { return rt ? 16 * rt : kTileRows; }
    int unit() const { return rt ? 256 : 64; }
};

// Rows of one request and key/value head (on average) up to which the few-rows kernel takes them.
int few_operands(long long rows, int dim)
{
    if (rows <= 16) return 1;
    if (rows <= 32 && dim <= 128) return 2;
    return 0;
}

// How a call whose tiles see up to `keys` keys is divided: `busy` workgroups would run without a division.
void divide(Division &d, long long busy, long long keys, long long most_parts)
{
    const long long want = d.rt ? 1024 : 512;
    long long s = std::min(ceil_div(want, busy), ceil_div(keys, 256));
    if (d.rt) s = std::max(s, ceil_div(keys, 4096));     // requests of different lengths end together
    s = std::max(1ll, std::min(s, most_parts));
    d.chunk = (int)(ceil_div(ceil_div(std::max(keys, 1ll), s), d.unit()) * d.unit());
    d.splits = (int)std::max(1ll, ceil_div(keys, d.chunk));
}

struct Plan {
    Division own, shared;
    size_t slots = 0, rows = 0, bytes = 0;
};

int plan(const gptq_hip_attention &a, Plan &pl)
{
    const long long group = a.heads / a.cache.heads, T = a.tokens, B = a.requests, H = a.cache.heads;
    const size_t part = (size_t)T * a.heads * (a.cache.dim * 4 + 8);
    const long long room = std::max<long long>(1, (long long)(kMostParts / part));
    long long shared_parts = 0;
    if (a.prefix_length > 0) {
        Division &d = pl.shared;
        d.rt = few_operands(T * group, a.cache.dim);
        d.tiles = (int)ceil_div(T * group, d.rows());
        divide(d, d.tiles * H, a.prefix_length, room);
        shared_parts = d.splits;
        if (d.tiles * H * d.splits >= 1ll << 31) return GPTQ_HIP_ERR_UNSUPPORTED;
    }
    Division &d = pl.own;
    d.rt = few_operands(ceil_div(T * group, B), a.cache.dim);
    d.tiles = (int)(T * group / d.rows() + B);
    long long keys = (long long)a.table_width * a.cache.block_size;
    if (a.max_context > 0) keys = std::min<long long>(keys, a.max_context);
    if (a.window > 0) keys = std::min<long long>(keys, (long long)a.window + a.sinks + d.rows() / group + 1);
    const bool counted = d.tiles * H <= (long long)(kAttentionCounters / 4);
    divide(d, std::max(B, ceil_div(T * group, d.rows())) * H, keys, counted ? room : 1);
    if ((long long)d.tiles * H * d.splits >= 1ll << 31) return GPTQ_HIP_ERR_UNSUPPORTED;
    pl.rows = (size_t)T * a.heads;
    pl.slots = d.splits > 1 || shared_parts ? (size_t)(shared_parts + d.splits) : 0;
    pl.bytes = pl.slots ? kAttentionCounters + (pl.slots * pl.rows * 8 + 255) / 256 * 256 + pl.slots * pl.rows * a.cache.dim * 4 : 0;
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
        p.counters = (int *)workspace;
        p.stats = (float *)((char *)workspace + gptq::kAttentionCounters);
        p.parts = (float *)((char *)p.stats + (pl.slots * pl.rows * 8 + 255) / 256 * 256);
    }
    p.tokens = a->tokens, p.requests = a->requests, p.heads = a->heads, p.kv_heads = c.heads, p.group = a->heads / c.heads;
    p.dim = c.dim, p.blocks = c.blocks, p.block_size = c.block_size;
    p.q_token = a->q_token_stride, p.q_head = a->q_head_stride;
    p.block_stride = c.block_stride, p.slot_stride = c.slot_stride, p.head_stride = c.head_stride;
    p.c = a->scale * 1.44269504088896340736f;
    auto launch = [&](const gptq::Division &d) {
        p.tiles = d.tiles, p.splits = d.splits, p.chunk = d.chunk;
        return d.rt ? gptq::launch_attention_few(p, c.type, d.rt, stream) : gptq::launch_attention_tile(p, c.type, stream);
    };
    if (a->prefix_length > 0) {
        p.shared = 1, p.prefix = a->prefix_length;
        p.tables = a->prefix_blocks;
        p.table_width = (int)gptq::ceil_div(a->prefix_length, c.block_size);
        rc = launch(pl.shared);
        if (rc != GPTQ_HIP_OK) return rc;
        p.shared = 0, p.first_slot = pl.shared.splits;
    }
    p.tables = a->tables, p.table_width = a->table_width, p.table_stride = a->table_stride;
    p.starts = a->starts, p.contexts = a->contexts;
    p.window = std::min(a->window, gptq::kMostKeys), p.sinks = std::min(a->sinks, gptq::kMostKeys);
    return launch(pl.own);
}
