// A paged key/value cache: block tables and slot maps from the lengths of the requests, and the write of a step's keys and
// values into their slots.
#include <hip/hip_runtime.h>

#include "gptq_internal.h"
#include "gptq_unpack.h"

namespace gptq {

// ---------------------------------------------------------------------------------------------------------------------
// Tables.  What a request gets follows from two running sums over the requests, of its new tokens and of its new blocks;
// what a token gets follows from its request's.  A few thousand integers: the call is bound by the launch and by its chain
// of dependent reads.  So it is ONE launch without any meeting of its workgroups: every one makes the two sums for itself
// (a few numbers a thread, the sums and the lengths in LDS) and then takes its share of the new table entries, and of the
// tokens, up to four neighbours a thread, each found by a binary search in LDS.  A slot in a new block is taken from the free list
// itself, not from the table entry that another workgroup may not have written yet.  Few tokens take a thread
// each.  (170890 tokens of 333 requests 6.6 us, 7.5 with a token a thread and the lengths from memory; 64 tokens of 64 requests
// 3.6 us, 5.3 with four a thread.  A launch with one read and one write takes 2.4.)
// ---------------------------------------------------------------------------------------------------------------------
struct CacheTables {
    const int32_t *lengths, *counts, *free_blocks;
    int32_t *tables, *starts, *contexts, *slots, *positions, *taken;
    long long table_stride;
    int table_width, free_count, requests, tokens, block_size, block_shift;   // block_shift: log2(block_size), or -1
};

constexpr int kTableThreads = 256;

// the running sum over the threads of a workgroup: what stands before this thread's value, and the whole sum
__device__ __forceinline__ int2 sum_before(int value, int2 *waves, int2 &total, int other)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int a = value, b = other;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int x = __shfl_up(a, d), y = __shfl_up(b, d);
        if (lane >= d) a += x, b += y;
    }
    if (lane == 63) waves[wave] = make_int2(a, b);
    __syncthreads();
    int2 before = make_int2(a - value, b - other);
    total = make_int2(0, 0);
#pragma unroll
    for (int w = 0; w < kTableThreads / 64; w++) {
        if (w < wave) before.x += waves[w].x, before.y += waves[w].y;
        total.x += waves[w].x, total.y += waves[w].y;
    }
    return before;
}

// the last entry of the ascending list sums[0 .. n] that is at most x, below n (an entry whose successor is larger)
__device__ __forceinline__ int owner(const int *sums, int n, int x)
{
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (sums[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

extern __shared__ int table_sums[];   // starts [B + 1], new blocks before [B + 1], lengths [B]

// PER: neighbouring tokens of a thread
template <int PER>
__global__ __launch_bounds__(kTableThreads) void cache_tables_kernel(const CacheTables p)
{
    __shared__ int2 waves[kTableThreads / 64];
    const int B = p.requests, s = p.block_size;
    int *starts = table_sums, *before = starts + B + 1, *lengths = before + B + 1;
    // consecutive requests a thread; negative lengths and counts count as none
    const int each = (B + kTableThreads - 1) / kTableThreads, b0 = threadIdx.x * each, b1 = min(b0 + each, B);
    auto count = [&](int b) { return max(p.counts[b], 0); };
    auto block_of = [&](int at) { return p.block_shift >= 0 ? at >> p.block_shift : at / s; };
    auto blocks = [&](int tokens) { return tokens > 0 ? block_of(tokens - 1) + 1 : 0; };
    int mine = 0, fresh = 0;
    for (int b = b0; b < b1; b++) {
        const int held = max(p.lengths[b], 0), n = count(b);
        lengths[b] = held;
        mine += n;
        fresh += blocks(held + n) - blocks(held);
    }
    int2 total;
    int2 sum = sum_before(mine, waves, total, fresh);
    for (int b = b0; b < b1; b++) {
        const int held = lengths[b], n = count(b);
        starts[b] = sum.x, before[b] = sum.y;
        if (blockIdx.x == 0) p.starts[b] = sum.x, p.contexts[b] = held + n;
        sum.x += n;
        sum.y += blocks(held + n) - blocks(held);
    }
    if (threadIdx.x == 0) {
        starts[B] = total.x, before[B] = total.y;
        if (blockIdx.x == 0) p.starts[B] = total.x, p.taken[0] = total.y;
    }
    __syncthreads();
    const int step = gridDim.x * kTableThreads, first = blockIdx.x * kTableThreads + threadIdx.x;
    // new entries of the tables, in the order in which the free blocks are dealt out
    for (int i = first; i < min(total.y, p.free_count); i += step) {
        const int b = owner(before, B, i), j = blocks(lengths[b]) + i - before[b];
        if (j < p.table_width) p.tables[(long long)b * p.table_stride + j] = p.free_blocks[i];
    }
    for (int t0 = PER * first; t0 < p.tokens; t0 += PER * step) {
        // where each one's block stands, then all the reads together
        int at[PER], slot[PER], b = t0 < total.x ? owner(starts, B, t0) : 0;
        const int32_t *from[PER];
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int t = t0 + i;
            at[i] = slot[i] = -1;
            from[i] = nullptr;
            if (t < total.x) {
                while (t >= starts[b + 1]) b++;     // (there is one: t is below the last sum)
                at[i] = lengths[b] + t - starts[b];
                const int j = block_of(at[i]), have = blocks(lengths[b]), nth = before[b] + j - have;
                slot[i] = at[i] - j * s;
                if (j < p.table_width && j < have) from[i] = p.tables + (long long)b * p.table_stride + j;
                else if (j < p.table_width && nth < p.free_count) from[i] = p.free_blocks + nth;
            }
        }
        int block[PER];
#pragma unroll
        for (int i = 0; i < PER; i++) block[i] = from[i] ? *from[i] : -1;
#pragma unroll
        for (int i = 0; i < PER; i++) slot[i] = block[i] >= 0 ? block[i] * s + slot[i] : -1;
        if constexpr (PER == 4) {
            if (t0 + 4 <= p.tokens) {
                *(int4 *)(p.slots + t0) = make_int4(slot[0], slot[1], slot[2], slot[3]);
                *(int4 *)(p.positions + t0) = make_int4(at[0], at[1], at[2], at[3]);
                continue;
            }
        }
#pragma unroll
        for (int i = 0; i < PER; i++)
            if (t0 + i < p.tokens) p.slots[t0 + i] = slot[i], p.positions[t0 + i] = at[i];
    }
}

// ---------------------------------------------------------------------------------------------------------------------
// Write.  Bound by memory: every row is read and written once, 16 bytes a thread.  Tokens of a step that are no longer wanted
// (slot -1) and slots outside of the cache are skipped.  (8192 tokens of 8 heads of 128: 67 MB in 11.2 us, 6.0 TB/s; 64 tokens
// 2.6 us, of which a launch is 2.4.)
// ---------------------------------------------------------------------------------------------------------------------
struct CacheWrite {
    const char *k, *v;
    char *k_cache, *v_cache;
    const int32_t *slots;
    long long k_token, k_head, v_token, v_head, block_stride, slot_stride, head_stride;   // in bytes
    uint32_t tokens, chunks, row_chunks;   // 16-byte chunks of a head, of a token
    int block_size, blocks;
};

__global__ __launch_bounds__(256) void cache_write_kernel(const CacheWrite p)
{
    const unsigned long long i = (unsigned long long)blockIdx.x * 256 + threadIdx.x;
    const uint32_t t = (uint32_t)(i / p.row_chunks), x = (uint32_t)(i - (unsigned long long)t * p.row_chunks);
    if (t >= p.tokens) return;
    const int slot = p.slots[t];
    const uint32_t h = x / p.chunks, c = x - h * p.chunks;
    const u4 k = *(const u4 *)(p.k + t * p.k_token + h * p.k_head + c * 16);
    const u4 v = *(const u4 *)(p.v + t * p.v_token + h * p.v_head + c * 16);
    if (slot < 0 || slot / p.block_size >= p.blocks) return;
    const long long at = (long long)(slot / p.block_size) * p.block_stride + (long long)(slot % p.block_size) * p.slot_stride +
                         (long long)h * p.head_stride + c * 16;
    *(u4 *)(p.k_cache + at) = k;
    *(u4 *)(p.v_cache + at) = v;
}

}  // namespace gptq

extern "C" int gptq_hip_cache_tables(const int32_t *lengths, const int32_t *counts, int32_t *tables, long long table_stride,
                                     int table_width, const int32_t *free_blocks, int free_count, int requests, int tokens,
                                     int block_size, int32_t *starts, int32_t *contexts, int32_t *slots, int32_t *positions,
                                     int32_t *taken, void *stream)
{
    if (requests < 0 || tokens < 0 || block_size < 1 || table_width < 0 || free_count < 0 || table_stride < table_width)
        return GPTQ_HIP_ERR_BAD_ARG;
    if (!starts || !taken || (requests > 0 && (!lengths || !counts || !contexts || (table_width > 0 && !tables))) ||
        (free_count > 0 && !free_blocks) || (tokens > 0 && (!slots || !positions)))
        return GPTQ_HIP_ERR_BAD_ARG;
    if (((uintptr_t)slots | (uintptr_t)positions) % 16 != 0) return GPTQ_HIP_ERR_BAD_ARG;
    if (requests > GPTQ_HIP_CACHE_MAX_REQUESTS) return GPTQ_HIP_ERR_UNSUPPORTED;   // the sums over the requests stand in LDS
    const gptq::CacheTables p = {lengths, counts, free_blocks, tables, starts, contexts, slots, positions, taken,
                                 table_stride, table_width, free_count, requests, tokens, block_size,
                                 block_size & (block_size - 1) ? -1 : __builtin_ctz((unsigned)block_size)};
    const int lds = 4 * (3 * requests + 2);
    if (tokens <= 32768)
        hipLaunchKernelGGL(gptq::cache_tables_kernel<1>, dim3(tokens <= 256 ? 1 : (tokens + 255) / 256), dim3(gptq::kTableThreads), lds, (hipStream_t)stream, p);
    else
        hipLaunchKernelGGL(gptq::cache_tables_kernel<4>, dim3(tokens / 1024 < 512 ? (tokens + 1023) / 1024 : 512), dim3(gptq::kTableThreads), lds, (hipStream_t)stream, p);
    return hipGetLastError() == hipSuccess ? GPTQ_HIP_OK : GPTQ_HIP_ERR_LAUNCH;
}

extern "C" int gptq_hip_cache_write(const gptq_hip_cache *cache, const void *k, const void *v, long long k_token_stride,
                                    long long k_head_stride, long long v_token_stride, long long v_head_stride,
                                    const int32_t *slots, int tokens, void *stream)
{
    const int rc = gptq::check_cache(cache);
    if (rc != GPTQ_HIP_OK) return rc;
    if (tokens < 0) return GPTQ_HIP_ERR_BAD_ARG;
    if (tokens == 0) return GPTQ_HIP_OK;
    if (!k || !v || !slots || ((uintptr_t)k | (uintptr_t)v) % 16 != 0) return GPTQ_HIP_ERR_BAD_ARG;
    if ((k_token_stride | k_head_stride | v_token_stride | v_head_stride) % 8 != 0) return GPTQ_HIP_ERR_BAD_ARG;
    const uint32_t chunks = (uint32_t)cache->dim / 8, row = chunks * (uint32_t)cache->heads;
    const gptq::CacheWrite p = {(const char *)k, (const char *)v, (char *)cache->k, (char *)cache->v, slots,
                                2 * k_token_stride, 2 * k_head_stride, 2 * v_token_stride, 2 * v_head_stride,
                                2 * cache->block_stride, 2 * cache->slot_stride, 2 * cache->head_stride,
                                (uint32_t)tokens, chunks, row, cache->block_size, cache->blocks};
    const unsigned long long grid = ((unsigned long long)tokens * row + 255) / 256;
    if (grid >= 1ull << 31) return GPTQ_HIP_ERR_UNSUPPORTED;
    hipLaunchKernelGGL(gptq::cache_write_kernel, dim3((unsigned)grid), dim3(256), 0, (hipStream_t)stream, p);
    return hipGetLastError() == hipSuccess ? GPTQ_HIP_OK : GPTQ_HIP_ERR_LAUNCH;
}
