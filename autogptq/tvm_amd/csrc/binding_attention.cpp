// torch.ops.gptq_hip.{cache_tables, cache_write, cache_read, paged_attention, shared_prefix_attention} and the same of a cache held in
// MXFP4 (..._mx): the serving entry points of
// libgptq_hip.so as dispatcher-visible operators (see binding.cpp for the products).  They check devices, dtypes, shapes and
// strides, allocate what they return, and launch on the current HIP stream of the tensors' device.
#include <ATen/ATen.h>
#include <ATen/hip/EmptyTensor.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <torch/library.h>

#include <array>
#include <cmath>
#include <tuple>

#include "binding.h"

namespace {

using namespace gptq_torch;

void on_gpu(const Tensor &t, const char *name, const Tensor &like)
{
    TORCH_CHECK(t.is_cuda(), name, " is on ", t.device(), ": the GPTQ kernels run on a ROCm GPU only and there is no CPU fallback");
    TORCH_CHECK(t.device() == like.device(), name, " is on ", t.device(), ", the others on ", like.device());
}

// int32 [n], contiguous (n < 0: any length)
void need_ints(const Tensor &t, const char *name, int64_t n, const Tensor &like)
{
    on_gpu(t, name, like);
    TORCH_CHECK(t.scalar_type() == at::kInt, name, " must be int32, got ", t.scalar_type());
    TORCH_CHECK(t.dim() == 1 && t.is_contiguous() && (n < 0 || t.size(0) == n), name, " must be a contiguous vector",
                n < 0 ? std::string() : " of " + std::to_string(n));
}

// int32 [rows, width], rows any distance apart
void need_tables(const Tensor &t, int64_t rows, const Tensor &like)
{
    on_gpu(t, "tables", like);
    TORCH_CHECK(t.scalar_type() == at::kInt, "tables must be int32, got ", t.scalar_type());
    TORCH_CHECK(t.dim() == 2 && t.size(0) == rows && t.size(1) < (1LL << 31), "tables must be [", rows, ", width]");
    TORCH_CHECK((t.size(1) <= 1 || t.stride(1) == 1) && (rows <= 1 || t.stride(0) >= t.size(1)),
                "the rows of tables must be contiguous and not overlap");
}
int64_t row_stride(const Tensor &t) { return std::max<int64_t>(t.size(0) > 1 ? t.stride(0) : t.size(1), t.size(1)); }

void no_grad(const Tensor &t, const char *name)
{
    TORCH_CHECK(!(t.requires_grad() && at::GradMode::is_enabled()), name, " requires grad: the cache operators have no backward");
}

// the stride of a dimension that has one (of a single entry it says nothing)
int64_t step(const Tensor &t, int64_t d) { return t.size(d) > 1 ? t.stride(d) : 0; }

// [tokens, heads, dim] rows the kernels can load 16 bytes at a time; else a copy
Tensor loadable(const Tensor &t)
{
    const bool fits = t.stride(2) == 1 && step(t, 0) % 8 == 0 && step(t, 1) % 8 == 0 && (uintptr_t)t.data_ptr() % 16 == 0;
    return fits ? t : t.clone(at::MemoryFormat::Contiguous);
}

gptq_hip_cache describe(const Tensor &k, const Tensor &v)
{
    on_gpu(v, "v_cache", k);
    TORCH_CHECK(k.scalar_type() == at::kHalf || k.scalar_type() == at::kBFloat16, "the cache must be float16 or bfloat16, got ",
                k.scalar_type());
    TORCH_CHECK(v.scalar_type() == k.scalar_type(), "k_cache is ", k.scalar_type(), ", v_cache ", v.scalar_type());
    TORCH_CHECK(k.dim() == 4 && k.sizes() == v.sizes(), "k_cache and v_cache must be [blocks, block_size, heads, dim] alike, got ",
                k.sizes(), " and ", v.sizes());
    const int64_t block = step(k, 0), slot = step(k, 1), head = step(k, 2);
    TORCH_CHECK(block == step(v, 0) && slot == step(v, 1) && head == step(v, 2) && k.stride(3) == v.stride(3), "k_cache and v_cache must have the same strides");
    TORCH_CHECK(k.numel() > 0, "the cache is empty");
    TORCH_CHECK(k.size(3) % 8 == 0 && k.size(3) <= 256, "dim must be a multiple of 8 up to 256, got ", k.size(3));
    TORCH_CHECK(k.stride(3) == 1 && block % 8 == 0 && slot % 8 == 0 && head % 8 == 0 &&
                    (uintptr_t)k.data_ptr() % 16 == 0 && (uintptr_t)v.data_ptr() % 16 == 0,
                "a head's dim elements must lie side by side in the cache, 16-byte aligned (strides ", k.strides(), ")");
    TORCH_CHECK(k.size(0) < (1LL << 31) && k.size(1) < (1LL << 31) && k.size(0) * k.size(1) < (1LL << 31) && k.size(2) < (1LL << 31),
                "the cache has too many slots");
    gptq_hip_cache c;
    c.k = k.data_ptr(), c.v = v.data_ptr();
    c.type = k.scalar_type() == at::kHalf ? GPTQ_HIP_TYPE_FP16 : GPTQ_HIP_TYPE_BF16;
    c.blocks = (int)k.size(0), c.block_size = (int)k.size(1), c.heads = (int)k.size(2), c.dim = (int)k.size(3);
    c.block_stride = block, c.slot_stride = slot, c.head_stride = head;
    return c;
}

// bytes [blocks, block_size, heads, n] whose rows lie side by side; the steps of its first three dimensions
std::array<int64_t, 3> rows_of(const Tensor &t, const char *name, int64_t n, int64_t unit)
{
    TORCH_CHECK(t.scalar_type() == at::kByte, name, " must be uint8, got ", t.scalar_type());
    TORCH_CHECK(t.dim() == 4 && t.size(3) == n, name, " must be [blocks, block_size, heads, ", n, "], got ", t.sizes());
    TORCH_CHECK(t.numel() > 0, "the cache is empty");
    const std::array<int64_t, 3> steps = {step(t, 0), step(t, 1), step(t, 2)};
    TORCH_CHECK(t.stride(3) == 1 && steps[0] % unit == 0 && steps[1] % unit == 0 && steps[2] % unit == 0 && (uintptr_t)t.data_ptr() % unit == 0,
                "the rows of ", name, " must be contiguous and ", unit, "-byte aligned (strides ", t.strides(), ")");
    return steps;
}

gptq_hip_cache_mx describe_mx(const Tensor &k, const Tensor &k_scales, const Tensor &v, const Tensor &v_scales, int64_t dim, at::ScalarType type)
{
    on_gpu(v, "v_codes", k);
    on_gpu(k_scales, "k_scales", k);
    on_gpu(v_scales, "v_scales", k);
    TORCH_CHECK(type == at::kHalf || type == at::kBFloat16, "an MXFP4 cache holds float16 or bfloat16 values, not ", type);
    TORCH_CHECK(dim >= 8 && dim % 8 == 0 && dim <= 256, "dim must be a multiple of 8 up to 256, got ", dim);
    const int64_t row = (dim + 31) / 32 * 16, scales = dim <= 64 ? 2 : dim <= 128 ? 4 : 8;
    const auto at = rows_of(k, "k_codes", row, 16), scale_at = rows_of(k_scales, "k_scales", scales, scales);
    TORCH_CHECK(rows_of(v, "v_codes", row, 16) == at && rows_of(v_scales, "v_scales", scales, scales) == scale_at && v.sizes() == k.sizes() &&
                    v_scales.sizes() == k_scales.sizes(), "keys and values must have the same shapes and strides");
    for (int d = 0; d < 3; d++)
        TORCH_CHECK(k.size(d) == k_scales.size(d), "codes and scales must be of the same rows, got ", k.sizes(), " and ", k_scales.sizes());
    TORCH_CHECK(k.size(0) < (1LL << 31) && k.size(1) < (1LL << 31) && k.size(0) * k.size(1) < (1LL << 31) && k.size(2) < (1LL << 31),
                "the cache has too many slots");
    gptq_hip_cache_mx c;
    c.k = k.data_ptr(), c.v = v.data_ptr(), c.k_scales = k_scales.data_ptr(), c.v_scales = v_scales.data_ptr();
    c.type = type == at::kHalf ? GPTQ_HIP_TYPE_FP16 : GPTQ_HIP_TYPE_BF16;
    c.blocks = (int)k.size(0), c.block_size = (int)k.size(1), c.heads = (int)k.size(2), c.dim = (int)dim;
    c.block_stride = at[0], c.slot_stride = at[1], c.head_stride = at[2];
    c.scale_block_stride = scale_at[0], c.scale_slot_stride = scale_at[1], c.scale_head_stride = scale_at[2];
    return c;
}

void *current_stream(const Tensor &t)
{
    return (void *)c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.get_device()).stream();
}

void raised(int rc, const char *what)
{
    TORCH_CHECK(rc == GPTQ_HIP_OK, what, " failed: ", gptq_hip_strerror(rc), " [status ", rc, "]");
}

// (the dispatcher counts the writes of torch's own operators only)
void written(const Tensor &t)
{
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

Tensor fresh(at::IntArrayRef sizes, const Tensor &like)
{
    return at::detail::empty_cuda(sizes, like.scalar_type(), like.device(), std::nullopt);
}

}  // namespace

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> gptq_torch::cache_tables(const Tensor &lengths, const Tensor &counts, const Tensor &tables,
                                                                const Tensor &free_blocks, int64_t tokens, int64_t block_size)
{
    need_ints(lengths, "lengths", -1, lengths);
    const int64_t B = lengths.size(0);
    need_ints(counts, "counts", B, lengths);
    need_tables(tables, B, lengths);
    need_ints(free_blocks, "free_blocks", -1, lengths);
    TORCH_CHECK(tokens >= 0 && tokens < (1LL << 31), "tokens must be the number of new tokens, got ", tokens);
    TORCH_CHECK(block_size > 0 && block_size < (1LL << 31), "block_size must be positive, got ", block_size);
    TORCH_CHECK(B <= GPTQ_HIP_CACHE_MAX_REQUESTS, "at most ", GPTQ_HIP_CACHE_MAX_REQUESTS, " requests, got ", B);
    TORCH_CHECK(free_blocks.size(0) < (1LL << 31), "too many free blocks");
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(lengths.device());
    // the five results are parts of one allocation (five would cost the host as much as the launch)
    const int64_t sizes[5] = {B + 1, B, tokens, tokens, 1};
    int64_t all = 0;
    for (int64_t n : sizes) all += (n + 3) / 4 * 4;
    const Tensor memory = fresh({all}, lengths);
    Tensor out[5];
    int64_t at = 0;
    for (int i = 0; i < 5; i++) {
        out[i] = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(memory.storage()), memory.key_set(), memory.dtype());
        out[i].unsafeGetTensorImpl()->set_storage_offset(at);
        out[i].unsafeGetTensorImpl()->set_sizes_contiguous({sizes[i]});
        at += (sizes[i] + 3) / 4 * 4;
    }
    const Tensor &starts = out[0], &contexts = out[1], &slots = out[2], &positions = out[3], &taken = out[4];
    raised(gptq_hip_cache_tables((const int32_t *)lengths.data_ptr(), (const int32_t *)counts.data_ptr(), (int32_t *)tables.data_ptr(),
                                 row_stride(tables), (int)tables.size(1), (const int32_t *)free_blocks.data_ptr(),
                                 (int)free_blocks.size(0), (int)B, (int)tokens, (int)block_size, (int32_t *)starts.data_ptr(),
                                 (int32_t *)contexts.data_ptr(), (int32_t *)slots.data_ptr(), (int32_t *)positions.data_ptr(),
                                 (int32_t *)taken.data_ptr(), current_stream(lengths)),
           "gptq_hip_cache_tables");
    written(tables);
    return {out[0], out[1], out[2], out[3], out[4]};
}

void gptq_torch::cache_write(const Tensor &k, const Tensor &v, const Tensor &k_cache, const Tensor &v_cache, const Tensor &slots)
{
    on_gpu(k_cache, "k_cache", k_cache);
    const gptq_hip_cache c = describe(k_cache, v_cache);
    no_grad(k_cache, "k_cache");
    no_grad(v_cache, "v_cache");
    for (const Tensor *t : {&k, &v}) {
        const char *name = t == &k ? "k" : "v";
        on_gpu(*t, name, k_cache);
        no_grad(*t, name);
        TORCH_CHECK(t->scalar_type() == k_cache.scalar_type(), name, " is ", t->scalar_type(), ", the cache ", k_cache.scalar_type());
        TORCH_CHECK(t->dim() == 3 && t->size(1) == c.heads && t->size(2) == c.dim, name, " must be [tokens, ", c.heads, ", ", c.dim,
                    "], got ", t->sizes());
        TORCH_CHECK(t->size(0) < (1LL << 31), "too many tokens");
    }
    need_ints(slots, "slots", k.size(0), k_cache);
    TORCH_CHECK(v.size(0) == k.size(0), "k has ", k.size(0), " tokens, v ", v.size(0));
    if (k.size(0) == 0) return;
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(k_cache.device());
    const Tensor ks = loadable(k), vs = loadable(v);
    raised(gptq_hip_cache_write(&c, ks.data_ptr(), vs.data_ptr(), step(ks, 0), step(ks, 1), step(vs, 0), step(vs, 1),
                                (const int32_t *)slots.data_ptr(), (int)k.size(0), current_stream(k_cache)),
           "gptq_hip_cache_write");
    written(k_cache);
    written(v_cache);
}

void gptq_torch::cache_write_mx(const Tensor &k, const Tensor &v, const Tensor &k_codes, const Tensor &k_scales, const Tensor &v_codes,
                                const Tensor &v_scales, const Tensor &slots)
{
    on_gpu(k_codes, "k_codes", k_codes);
    TORCH_CHECK(k.dim() == 3, "k must be [tokens, heads, dim], got ", k.sizes());
    const gptq_hip_cache_mx c = describe_mx(k_codes, k_scales, v_codes, v_scales, k.size(2), k.scalar_type());
    for (const Tensor *t : {&k, &v}) {
        const char *name = t == &k ? "k" : "v";
        on_gpu(*t, name, k_codes);
        no_grad(*t, name);
        TORCH_CHECK(t->scalar_type() == k.scalar_type(), name, " is ", t->scalar_type(), ", k ", k.scalar_type());
        TORCH_CHECK(t->dim() == 3 && t->size(1) == c.heads && t->size(2) == c.dim, name, " must be [tokens, ", c.heads, ", ", c.dim,
                    "], got ", t->sizes());
        TORCH_CHECK(t->size(0) < (1LL << 31), "too many tokens");
    }
    need_ints(slots, "slots", k.size(0), k_codes);
    TORCH_CHECK(v.size(0) == k.size(0), "k has ", k.size(0), " tokens, v ", v.size(0));
    if (k.size(0) == 0) return;
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(k_codes.device());
    const Tensor ks = loadable(k), vs = loadable(v);
    raised(gptq_hip_cache_write_mx(&c, ks.data_ptr(), vs.data_ptr(), step(ks, 0), step(ks, 1), step(vs, 0), step(vs, 1),
                                   (const int32_t *)slots.data_ptr(), (int)k.size(0), current_stream(k_codes)),
           "gptq_hip_cache_write_mx");
    for (const Tensor *t : {&k_codes, &k_scales, &v_codes, &v_scales}) written(*t);
}

std::tuple<Tensor, Tensor> gptq_torch::cache_read(const Tensor &k_cache, const Tensor &v_cache, const Tensor &slots)
{
    on_gpu(k_cache, "k_cache", k_cache);
    const gptq_hip_cache c = describe(k_cache, v_cache);
    no_grad(k_cache, "k_cache");
    no_grad(v_cache, "v_cache");
    need_ints(slots, "slots", -1, k_cache);
    TORCH_CHECK(slots.size(0) < (1LL << 31), "too many tokens");
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(k_cache.device());
    Tensor k = fresh({slots.size(0), c.heads, c.dim}, k_cache), v = fresh(k.sizes(), k_cache);
    raised(gptq_hip_cache_read(&c, (const int32_t *)slots.data_ptr(), (int)slots.size(0), k.data_ptr(), v.data_ptr(), current_stream(k_cache)),
           "gptq_hip_cache_read");
    return {k, v};
}

std::tuple<Tensor, Tensor> gptq_torch::cache_read_mx(const Tensor &k_codes, const Tensor &k_scales, const Tensor &v_codes, const Tensor &v_scales,
                                                     const Tensor &slots, int64_t dim, at::ScalarType dtype)
{
    on_gpu(k_codes, "k_codes", k_codes);
    const gptq_hip_cache_mx c = describe_mx(k_codes, k_scales, v_codes, v_scales, dim, dtype);
    need_ints(slots, "slots", -1, k_codes);
    TORCH_CHECK(slots.size(0) < (1LL << 31), "too many tokens");
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(k_codes.device());
    Tensor k = at::detail::empty_cuda({slots.size(0), c.heads, dim}, dtype, k_codes.device(), std::nullopt);
    Tensor v = at::detail::empty_cuda(k.sizes(), dtype, k_codes.device(), std::nullopt);
    raised(gptq_hip_cache_read_mx(&c, (const int32_t *)slots.data_ptr(), (int)slots.size(0), k.data_ptr(), v.data_ptr(), current_stream(k_codes)),
           "gptq_hip_cache_read_mx");
    return {k, v};
}

// A call but for its cache.  `cache` is the shape that q has to fit; on_cache: a tensor of it.
struct Call {
    const Tensor &q, &prefix_blocks;
    int64_t prefix_length;
    const Tensor &tables, &starts, &contexts;
    int64_t max_context, window, sinks;
    double scale;
};
template <typename Launch>
static Tensor attend(const Call &call, const gptq_hip_cache &cache, const Tensor &on_cache, Launch launch)
{
    const Tensor &q = call.q, &tables = call.tables;
    gptq_hip_attention a;
    a.cache = cache;
    TORCH_CHECK(q.dim() == 3 && q.size(2) == cache.dim, "q must be [tokens, heads, ", cache.dim, "], got ", q.sizes());
    TORCH_CHECK(q.size(1) > 0 && q.size(1) % cache.heads == 0, "q has ", q.size(1), " heads, no multiple of the cache's ", cache.heads);
    need_ints(call.contexts, "contexts", -1, on_cache);
    const int64_t B = call.contexts.size(0);
    need_ints(call.starts, "starts", B + 1, on_cache);
    need_tables(tables, B, on_cache);
    TORCH_CHECK(B > 0 || q.size(0) == 0, "q has tokens, but there is no request");
    TORCH_CHECK(q.size(0) * q.size(1) < (1LL << 30) && B < (1LL << 24), "too many tokens or requests");
    for (const auto &[value, name] : {std::pair<int64_t, const char *>{call.max_context, "max_context"}, {call.window, "window"}, {call.sinks, "sinks"}, {call.prefix_length, "prefix_length"}})
        TORCH_CHECK(value >= 0 && value < (1LL << 31), name, " must not be negative, got ", value);
    const double scale = call.scale == 0.0 ? 1.0 / std::sqrt((double)cache.dim) : call.scale;
    TORCH_CHECK(std::isfinite(scale) && scale > 0, "scale must be positive, got ", scale);
    a.prefix_blocks = nullptr;
    if (call.prefix_length > 0) {
        need_ints(call.prefix_blocks, "prefix_blocks", -1, on_cache);
        const int64_t blocks = (call.prefix_length + cache.block_size - 1) / cache.block_size;
        TORCH_CHECK(call.prefix_blocks.size(0) >= blocks, "a prefix of ", call.prefix_length, " tokens takes ", blocks, " blocks, prefix_blocks has ",
                    call.prefix_blocks.size(0));
        a.prefix_blocks = (const int32_t *)call.prefix_blocks.data_ptr();
    }
    Tensor out = fresh(q.sizes(), q);
    if (q.size(0) == 0) return out;
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(on_cache.device());
    const Tensor qs = loadable(q);
    a.q = qs.data_ptr(), a.out = out.data_ptr();
    a.tables = (const int32_t *)tables.data_ptr(), a.starts = (const int32_t *)call.starts.data_ptr(), a.contexts = (const int32_t *)call.contexts.data_ptr();
    a.tokens = (int)q.size(0), a.requests = (int)B, a.heads = (int)q.size(1), a.table_width = (int)tables.size(1);
    a.max_context = (int)call.max_context, a.window = (int)call.window, a.sinks = (int)call.sinks, a.prefix_length = (int)call.prefix_length;
    a.q_token_stride = step(qs, 0), a.q_head_stride = step(qs, 1), a.table_stride = row_stride(tables);
    a.scale = (float)scale;
    launch(a, current_stream(on_cache));
    return out;
}

static Tensor attend_plain(const char *what, const Tensor &k_cache, const Tensor &v_cache, const Call &call)
{
    on_gpu(k_cache, "k_cache", k_cache);
    const gptq_hip_cache cache = describe(k_cache, v_cache);
    on_gpu(call.q, "q", k_cache);
    no_grad(call.q, "q");
    no_grad(k_cache, "k_cache");
    no_grad(v_cache, "v_cache");
    TORCH_CHECK(call.q.scalar_type() == k_cache.scalar_type(), "q is ", call.q.scalar_type(), ", the cache ", k_cache.scalar_type());
    return attend(call, cache, k_cache, [&](const gptq_hip_attention &a, void *stream) {
        const WorkspaceLease ws(call.q, gptq_hip_attention_workspace_bytes(&a), stream, kAttentionWorkspace);
        raised(gptq_hip_attend(&a, ws.data(), ws.size(), stream), what);
    });
}

static Tensor attend_mx(const char *what, const Tensor &k_codes, const Tensor &k_scales, const Tensor &v_codes, const Tensor &v_scales, const Call &call)
{
    on_gpu(k_codes, "k_codes", k_codes);
    on_gpu(call.q, "q", k_codes);
    no_grad(call.q, "q");
    TORCH_CHECK(call.q.dim() == 3, "q must be [tokens, heads, dim], got ", call.q.sizes());
    const gptq_hip_cache_mx mx = describe_mx(k_codes, k_scales, v_codes, v_scales, call.q.size(2), call.q.scalar_type());
    const gptq_hip_cache shape = {mx.k, mx.v, mx.type, mx.blocks, mx.block_size, mx.heads, mx.dim, 0, 0, 0};
    return attend(call, shape, k_codes, [&](const gptq_hip_attention &a, void *stream) {
        const WorkspaceLease ws(call.q, gptq_hip_attention_mx_workspace_bytes(&mx, &a), stream, kAttentionWorkspace);
        raised(gptq_hip_attend_mx(&mx, &a, ws.data(), ws.size(), stream), what);
    });
}

Tensor gptq_torch::paged_attention(const Tensor &q, const Tensor &k_cache, const Tensor &v_cache, const Tensor &tables, const Tensor &starts,
                       const Tensor &contexts, int64_t max_context, int64_t window, int64_t sinks, double scale)
{
    return attend_plain("gptq_hip_attend", k_cache, v_cache, {q, Tensor(), 0, tables, starts, contexts, max_context, window, sinks, scale});
}

Tensor gptq_torch::shared_prefix_attention(const Tensor &q, const Tensor &k_cache, const Tensor &v_cache, const Tensor &prefix_blocks,
                               int64_t prefix_length, const Tensor &tables, const Tensor &starts, const Tensor &contexts,
                               int64_t max_context, double scale)
{
    return attend_plain("gptq_hip_attend (shared prefix)", k_cache, v_cache,
                        {q, prefix_blocks, prefix_length, tables, starts, contexts, max_context, 0, 0, scale});
}

Tensor gptq_torch::paged_attention_mx(const Tensor &q, const Tensor &k_codes, const Tensor &k_scales, const Tensor &v_codes, const Tensor &v_scales,
                                      const Tensor &tables, const Tensor &starts, const Tensor &contexts, int64_t max_context, int64_t window,
                                      int64_t sinks, double scale)
{
    return attend_mx("gptq_hip_attend_mx", k_codes, k_scales, v_codes, v_scales,
                     {q, Tensor(), 0, tables, starts, contexts, max_context, window, sinks, scale});
}

Tensor gptq_torch::shared_prefix_attention_mx(const Tensor &q, const Tensor &k_codes, const Tensor &k_scales, const Tensor &v_codes,
                                              const Tensor &v_scales, const Tensor &prefix_blocks, int64_t prefix_length, const Tensor &tables,
                                              const Tensor &starts, const Tensor &contexts, int64_t max_context, double scale)
{
    return attend_mx("gptq_hip_attend_mx (shared prefix)", k_codes, k_scales, v_codes, v_scales,
                     {q, prefix_blocks, prefix_length, tables, starts, contexts, max_context, 0, 0, scale});
}

using namespace gptq_torch;

TORCH_LIBRARY_FRAGMENT(gptq_hip, m)
{
    m.def("cache_tables(Tensor lengths, Tensor counts, Tensor(a!) tables, Tensor free_blocks, int tokens, int block_size) -> "
          "(Tensor, Tensor, Tensor, Tensor, Tensor)");
    m.def("cache_write(Tensor k, Tensor v, Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor slots) -> ()");
    m.def("cache_read(Tensor k_cache, Tensor v_cache, Tensor slots) -> (Tensor, Tensor)");
    m.def("cache_write_mx(Tensor k, Tensor v, Tensor(a!) k_codes, Tensor(b!) k_scales, Tensor(c!) v_codes, Tensor(d!) v_scales, "
          "Tensor slots) -> ()");
    m.def("cache_read_mx(Tensor k_codes, Tensor k_scales, Tensor v_codes, Tensor v_scales, Tensor slots, int dim, ScalarType dtype) -> "
          "(Tensor, Tensor)");
    m.def("paged_attention(Tensor q, Tensor k_cache, Tensor v_cache, Tensor tables, Tensor starts, Tensor contexts, "
          "int max_context, int window, int sinks, float scale) -> Tensor");
    m.def("shared_prefix_attention(Tensor q, Tensor k_cache, Tensor v_cache, Tensor prefix_blocks, int prefix_length, "
          "Tensor tables, Tensor starts, Tensor contexts, int max_context, float scale) -> Tensor");
    m.def("paged_attention_mx(Tensor q, Tensor k_codes, Tensor k_scales, Tensor v_codes, Tensor v_scales, Tensor tables, Tensor starts, "
          "Tensor contexts, int max_context, int window, int sinks, float scale) -> Tensor");
    m.def("shared_prefix_attention_mx(Tensor q, Tensor k_codes, Tensor k_scales, Tensor v_codes, Tensor v_scales, Tensor prefix_blocks, "
          "int prefix_length, Tensor tables, Tensor starts, Tensor contexts, int max_context, float scale) -> Tensor");
}

// The CPU key gets the same functions, whose first check says that there is no CPU fallback.
TORCH_LIBRARY_IMPL(gptq_hip, CUDA, m)
{
    m.impl("cache_tables", &cache_tables);
    m.impl("cache_write", &cache_write);
    m.impl("cache_read", &cache_read);
    m.impl("cache_write_mx", &cache_write_mx);
    m.impl("cache_read_mx", &cache_read_mx);
    m.impl("paged_attention", &paged_attention);
    m.impl("shared_prefix_attention", &shared_prefix_attention);
    m.impl("paged_attention_mx", &paged_attention_mx);
    m.impl("shared_prefix_attention_mx", &shared_prefix_attention_mx);
}

TORCH_LIBRARY_IMPL(gptq_hip, CPU, m)
{
    m.impl("cache_tables", &cache_tables);
    m.impl("cache_write", &cache_write);
    m.impl("cache_read", &cache_read);
    m.impl("cache_write_mx", &cache_write_mx);
    m.impl("cache_read_mx", &cache_read_mx);
    m.impl("paged_attention", &paged_attention);
    m.impl("shared_prefix_attention", &shared_prefix_attention);
    m.impl("paged_attention_mx", &paged_attention_mx);
    m.impl("shared_prefix_attention_mx", &shared_prefix_attention_mx);
}
