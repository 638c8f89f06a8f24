// A paged key/value cache held in MXFP4: the write that quantises a step's keys and values into their slots, and the read that
// gives the rows of slots back (of caches in fp16 and bf16 too).
#include <hip/hip_runtime.h>

#include "gptq_internal.h"
#include "gptq_mx.h"

namespace gptq {

// What a type's largest magnitudes and exponents are.  The exponents a write chooses keep every value of a group (1/2 to 6 times 2^e)
// within the type, fp16's subnormal steps included.
template <typename E>
struct MxLimits {
    static constexpr uint32_t infinite = 0x7c00u, lowest = 127 - 23, highest = 127 + 13;
};
template <>
struct MxLimits<__bf16> {
    static constexpr uint32_t infinite = 0x7f80u, lowest = 127 - 125, highest = 127 + 125;
};

// ---------------------------------------------------------------------------------------------------------------------
// Write.  Four lanes hold a group, 16 bytes each.  Its largest magnitude m is a maximum over their bit patterns (positive 16-bit floats are
// ordered as integers); with 2^x <= m < 2^(x + 1) the exponent is x - 2, which puts m into [4, 8) where 6 is the largest code, or x - 1 from
// 1.75 2^x on (root mean square error of normal values with the step at 1.5, 1.75, 1.875 and never: 0.1155, 0.1119, 0.1121, 0.1150
// sigma).  The conversion divides by 2^e and rounds to the nearest code, ties to even, and so does the format's definition:
// nothing here is rounded twice.  Bound by memory; 8 heads of 128: 8192 tokens 9.1 us (the caches hold what it writes: 4.7 TB/s in and
// out), 64 tokens 2.9, a launch.
// ---------------------------------------------------------------------------------------------------------------------
struct CacheWriteMx {
    const char *k, *v;
    char *k_codes, *v_codes, *k_scales, *v_scales;
    const int32_t *slots;
    long long k_token, k_head, v_token, v_head, block_stride, slot_stride, head_stride, scale_block, scale_slot, scale_head;   // in bytes
    uint32_t tokens, chunks, row_chunks;   // eights of values of a head, with the padding, and of a token
    int block_size, blocks, dim;
};

// over the four lanes of a group
__device__ __forceinline__ uint32_t max_group(uint32_t x)
{
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0xb1, 0xf, 0xf, true));   // lanes 1 0 3 2
    return max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x4e, 0xf, 0xf, true));   // lanes 2 3 0 1
}

template <typename E>
__device__ __forceinline__ void put_group(u4 x, char *codes, char *scales, uint32_t chunk)
{
    typedef unsigned short us2 __attribute__((ext_vector_type(2)));
    typedef E e2 __attribute__((ext_vector_type(2)));
    us2 top = {0, 0};
#pragma unroll
    for (int w = 0; w < 4; w++) {
        const uint32_t size = x[w] & 0x7fff7fffu;
        top = __builtin_elementwise_max(top, __builtin_bit_cast(us2, size));
    }
    const uint32_t most = max_group(max((uint32_t)top[0], (uint32_t)top[1]));
    const float m = (float)__builtin_bit_cast(E, (unsigned short)most);
    // (a mantissa of 1.75 or more carries into the exponent)
    const int e = (int)((__builtin_bit_cast(uint32_t, m) + 0x200000u) >> 23) - 2;
    const uint32_t scale = (uint32_t)min(max(e, (int)MxLimits<E>::lowest), (int)MxLimits<E>::highest);
    const float s = __builtin_bit_cast(float, scale << 23);
    uint32_t c = 0;
#define GPTQ_MX(W) \
    if constexpr (__is_same(E, _Float16)) c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, __builtin_bit_cast(e2, (uint32_t)x[W]), s, W); \
    else c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(e2, (uint32_t)x[W]), s, W);
    GPTQ_MX(0)
    GPTQ_MX(1)
    GPTQ_MX(2)
    GPTQ_MX(3)
#undef GPTQ_MX
    const bool finite = most < MxLimits<E>::infinite;
    *(uint32_t *)(codes + chunk * 4) = finite ? c : 0u;
    if (chunk % 4 == 0) scales[chunk / 4] = (char)(finite ? scale : 255u);
}

template <typename E>
__global__ __launch_bounds__(256) void cache_write_mx_kernel(const CacheWriteMx p)
{
    const unsigned long long i = (unsigned long long)blockIdx.x * 256 + threadIdx.x;
    const uint32_t t = (uint32_t)(i / p.row_chunks), x = (uint32_t)(i - (unsigned long long)t * p.row_chunks);
    if (t >= p.tokens) return;     // (a group's lanes are of one token)
    const int slot = p.slots[t];
    const uint32_t h = x / p.chunks, c = x - h * p.chunks;
    u4 k = {0u, 0u, 0u, 0u}, v = {0u, 0u, 0u, 0u};
    if ((int)c * 8 < p.dim) {
        k = *(const u4 *)(p.k + t * p.k_token + h * p.k_head + c * 16);
        v = *(const u4 *)(p.v + t * p.v_token + h * p.v_head + c * 16);
    }
    if (slot < 0 || slot / p.block_size >= p.blocks) return;
    const long long block = slot / p.block_size, at = slot % p.block_size;
    const long long codes = block * p.block_stride + at * p.slot_stride + (long long)h * p.head_stride;
    const long long scales = block * p.scale_block + at * p.scale_slot + (long long)h * p.scale_head;
    put_group<E>(k, p.k_codes + codes, p.k_scales + scales, c);
    put_group<E>(v, p.v_codes + codes, p.v_scales + scales, c);
}

// ---------------------------------------------------------------------------------------------------------------------
// Read.  Bound by memory: a thread takes eight values of a row.  Slots that the cache does not have give zeros.
// ---------------------------------------------------------------------------------------------------------------------
struct CacheRead {
    const char *k, *v, *k_scales, *v_scales;
    char *k_out, *v_out;
    const int32_t *slots;
    long long block_stride, slot_stride, head_stride, scale_block, scale_slot, scale_head;   // in bytes
    uint32_t tokens, chunks, row_chunks;   // eights of values of a head, of a token
    int block_size, blocks;
};

// MX: rows of codes, given as values of E; else rows of 16-bit values as they are.  PAST: results go past the caches.
template <typename E, bool MX, bool PAST>
__global__ __launch_bounds__(256) void cache_read_kernel(const CacheRead p)
{
    const unsigned long long i = (unsigned long long)blockIdx.x * 256 + threadIdx.x;
    const uint32_t t = (uint32_t)(i / p.row_chunks), x = (uint32_t)(i - (unsigned long long)t * p.row_chunks);
    if (t >= p.tokens) return;
    const int slot = p.slots[t];
    const uint32_t h = x / p.chunks, c = x - h * p.chunks;
    u4 k = {0u, 0u, 0u, 0u}, v = {0u, 0u, 0u, 0u};
    if (slot >= 0 && slot / p.block_size < p.blocks) {
        const long long block = slot / p.block_size, at = slot % p.block_size;
        const long long row = block * p.block_stride + at * p.slot_stride + (long long)h * p.head_stride;
        if constexpr (MX) {
            const long long scales = block * p.scale_block + at * p.scale_slot + (long long)h * p.scale_head + c / 4;
            const uint32_t kc = *(const uint32_t *)(p.k + row + c * 4), vc = *(const uint32_t *)(p.v + row + c * 4);
            const uint32_t ks = *(const unsigned char *)(p.k_scales + scales), vs = *(const unsigned char *)(p.v_scales + scales);
            k = mx_values<E>(kc, ks << 23);
            v = mx_values<E>(vc, vs << 23);
        } else {
            k = *(const u4 *)(p.k + row + c * 16);
            v = *(const u4 *)(p.v + row + c * 16);
        }
    }
    u4 *const k_out = (u4 *)(p.k_out + i * 16), *const v_out = (u4 *)(p.v_out + i * 16);
    if constexpr (PAST) {
        __builtin_nontemporal_store(k, k_out);
        __builtin_nontemporal_store(v, v_out);
    } else {
        *k_out = k;
        *v_out = v;
    }
}

template <typename E, bool MX>
static void launch_read(const CacheRead &p, unsigned grid, hipStream_t stream)
{
    // MiB of results, us past the caches and through them, 8 heads of 128: MXFP4 8 5.4 / 5.4, 12 5.4 / 5.3, 16 5.4 / 5.9, 20 5.3 / 6.7, 24 6.8 / 7.7, 32 8.8 / 9.2, 128
    // 27.8 / 28.5 (6.2 TB/s), 256 53 / 83; 16 bits, whose rows are read in as much, 8 5.4 / 5.4, 12 5.6 / 5.9, 16 7.2 / 7.1, 24 9.2 / 9.4, 32 11.9 / 11.8, 64 21.3 / 22.7,
    // 80 25.8 / 28.6, 128 48.5 / 41.7 (three calls' rows and results in turn, of which the last cache then keeps a part), 256 96 / 104
    const bool past = (unsigned long long)p.tokens * p.row_chunks * 32 > 12ull << 20;
    if (past) hipLaunchKernelGGL((cache_read_kernel<E, MX, true>), dim3(grid), dim3(256), 0, stream, p);
    else hipLaunchKernelGGL((cache_read_kernel<E, MX, false>), dim3(grid), dim3(256), 0, stream, p);
}

}  // namespace gptq

extern "C" int gptq_hip_cache_write_mx(const gptq_hip_cache_mx *c, const void *k, const void *v, long long k_token_stride,
                                       long long k_head_stride, long long v_token_stride, long long v_head_stride,
                                       const int32_t *slots, int tokens, void *stream)
{
    const int rc = gptq::check_cache_mx(c);
    if (rc != GPTQ_HIP_OK) return rc;
    if (tokens < 0) return GPTQ_HIP_ERR_BAD_ARG;
    if (tokens == 0) return GPTQ_HIP_OK;
    if (!k || !v || !slots || ((uintptr_t)k | (uintptr_t)v) % 16 != 0) return GPTQ_HIP_ERR_BAD_ARG;
    if ((k_token_stride | k_head_stride | v_token_stride | v_head_stride) % 8 != 0) return GPTQ_HIP_ERR_BAD_ARG;
    const uint32_t chunks = 4u * (uint32_t)gptq::mx_groups(c->dim), row = chunks * (uint32_t)c->heads;
    const unsigned long long grid = ((unsigned long long)tokens * row + 255) / 256;
    if (grid >= 1ull << 31 || (unsigned long long)chunks * (unsigned)c->heads >= 1ull << 32) return GPTQ_HIP_ERR_UNSUPPORTED;
    const gptq::CacheWriteMx p = {(const char *)k, (const char *)v, (char *)c->k, (char *)c->v, (char *)c->k_scales, (char *)c->v_scales, slots,
                                  2 * k_token_stride, 2 * k_head_stride, 2 * v_token_stride, 2 * v_head_stride,
                                  c->block_stride, c->slot_stride, c->head_stride, c->scale_block_stride, c->scale_slot_stride, c->scale_head_stride,
                                  (uint32_t)tokens, chunks, row, c->block_size, c->blocks, c->dim};
    if (c->type == GPTQ_HIP_TYPE_FP16) hipLaunchKernelGGL(gptq::cache_write_mx_kernel<_Float16>, dim3((unsigned)grid), dim3(256), 0, (hipStream_t)stream, p);
    else hipLaunchKernelGGL(gptq::cache_write_mx_kernel<__bf16>, dim3((unsigned)grid), dim3(256), 0, (hipStream_t)stream, p);
    return hipGetLastError() == hipSuccess ? GPTQ_HIP_OK : GPTQ_HIP_ERR_LAUNCH;
}

namespace {

int read_rows(gptq::CacheRead p, int type, bool mx, int heads, int dim, void *k, void *v, const int32_t *slots, int tokens, void *stream)
{
    if (tokens < 0) return GPTQ_HIP_ERR_BAD_ARG;
    if (tokens == 0) return GPTQ_HIP_OK;
    if (!k || !v || !slots || ((uintptr_t)k | (uintptr_t)v) % 16 != 0) return GPTQ_HIP_ERR_BAD_ARG;
    p.k_out = (char *)k, p.v_out = (char *)v, p.slots = slots;
    p.tokens = (uint32_t)tokens, p.chunks = (uint32_t)dim / 8, p.row_chunks = p.chunks * (uint32_t)heads;
    const unsigned long long grid = ((unsigned long long)tokens * p.row_chunks + 255) / 256;
    if (grid >= 1ull << 31 || (unsigned long long)p.chunks * (unsigned)heads >= 1ull << 32) return GPTQ_HIP_ERR_UNSUPPORTED;
    if (!mx) gptq::launch_read<_Float16, false>(p, (unsigned)grid, (hipStream_t)stream);
    else if (type == GPTQ_HIP_TYPE_FP16) gptq::launch_read<_Float16, true>(p, (unsigned)grid, (hipStream_t)stream);
    else gptq::launch_read<__bf16, true>(p, (unsigned)grid, (hipStream_t)stream);
    return hipGetLastError() == hipSuccess ? GPTQ_HIP_OK : GPTQ_HIP_ERR_LAUNCH;
}

}  // namespace

extern "C" int gptq_hip_cache_read(const gptq_hip_cache *c, const int32_t *slots, int tokens, void *k, void *v, void *stream)
{
    const int rc = gptq::check_cache(c);
    if (rc != GPTQ_HIP_OK) return rc;
    gptq::CacheRead p = {};
    p.k = (const char *)c->k, p.v = (const char *)c->v;
    p.block_stride = 2 * c->block_stride, p.slot_stride = 2 * c->slot_stride, p.head_stride = 2 * c->head_stride;
    p.block_size = c->block_size, p.blocks = c->blocks;
    return read_rows(p, c->type, false, c->heads, c->dim, k, v, slots, tokens, stream);
}

extern "C" int gptq_hip_cache_read_mx(const gptq_hip_cache_mx *c, const int32_t *slots, int tokens, void *k, void *v, void *stream)
{
    const int rc = gptq::check_cache_mx(c);
    if (rc != GPTQ_HIP_OK) return rc;
    gptq::CacheRead p = {};
    p.k = (const char *)c->k, p.v = (const char *)c->v, p.k_scales = (const char *)c->k_scales, p.v_scales = (const char *)c->v_scales;
    p.block_stride = c->block_stride, p.slot_stride = c->slot_stride, p.head_stride = c->head_stride;
    p.scale_block = c->scale_block_stride, p.scale_slot = c->scale_slot_stride, p.scale_head = c->scale_head_stride;
    p.block_size = c->block_size, p.blocks = c->blocks;
    return read_rows(p, c->type, true, c->heads, c->dim, k, v, slots, tokens, stream);
}
