// Shared by the translation units of the torch operator library (binding.cpp: torch.ops.gptq_hip.* and the torch class;
// python_call.cpp: the module call from Python): the per-stream workspaces and a layer's constant tensors bound to one
// row count.
#pragma once
#include <ATen/ATen.h>

#include <mutex>
#include <optional>
#include <tuple>

#include "gptq_hip.h"

namespace gptq_torch {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

inline const void *ptr(const OptTensor &t) { return t.has_value() && t->defined() ? t->data_ptr() : nullptr; }
inline bool has(const OptTensor &t) { return t.has_value() && t->defined(); }

// x, or a copy of it where the kernels' 16-byte loads ask for one (a contiguous view at an odd offset)
inline Tensor aligned(const Tensor &x) { return (uintptr_t)x.data_ptr() % 16 == 0 ? x : x.clone(); }

void raise(int rc, const char *what, int64_t M, int64_t K, int64_t N, int64_t bits, int64_t gs);

constexpr int kAttentionWorkspace = 2;
int workspace_kind(const gptq_hip_plan &plan);

// 0, or a number of the graph capture that the stream is in (no two captures have the same)
unsigned long long capture_of(void *stream);

// The workspace of a stream for the launches of one call (none for nbytes = 0).  Held over all of them: a call is up to three
// launches that hand x or partial sums on through the workspace, and those of another thread on the same stream must not
// come between.
//
// Launches that are captured keep the address for as long as their graph lives, and replay on any stream beside anything, so
// they never get the workspace of eager calls, which is replaced when a call needs more: each capture has one of its own, out of
// the memory pool of its graph, cleared by a launch that is captured with them.  (One launch a capture, not a call.  A capture that
// needs more on the way gets another: the pool hands the first one's memory to what the graph does later on the same stream.)
struct Workspace {
    std::mutex busy;
    Tensor bytes;                      // of eager calls
    Tensor captured;                   // of the capture `capture`; let go with the first call outside of it
    unsigned long long capture = 0;
};
class WorkspaceLease {
public:
    WorkspaceLease(const Tensor &like, size_t nbytes, void *stream, int kind = 0);
    void *data() const { return bytes ? bytes->data_ptr() : nullptr; }
    size_t size() const { return bytes ? (size_t)bytes->numel() : 0; }

private:
    const Tensor *bytes = nullptr;
    std::unique_lock<std::mutex> held;
};

// One layer's constant tensors, a row count and the plan for it: what a call needs beside x.
// kind: 0 = checkpoint tensors (qweight, qzeros, scales, g_idx?), 1 = sorted copy (qweight_sorted, qzeros, scales,
// kmap), 2 = tiled copy (qtile, sz, -, xsrc?, kinv?).
struct Bound {
    int kind = 0, bits = 0, group_size = 0;
    int M = 0, K = 0, N = 0;
    Tensor a, b, c;
    OptTensor d, e, bias;
    gptq_hip_plan plan{};
    size_t ws_need = 0;

    // fills plan and ws_need for M, K and N; a status of the library
    int choose();
    // y = x @ W (+ bias) on the current stream of the layer's device; x fp16 [M, K] and y fp16 [M, N], contiguous,
    // on that device, which is the current one.  A status of the library.
    int launch(const Tensor &x, void *y, void *stream) const;
};

// the same product as the operator torch.ops.gptq_hip.*, through the dispatcher
Tensor dispatch(const Bound &q, const Tensor &x);

// the operators' checks of a layer's tensors (devices, dtypes, shapes), once, when they are bound
void check_bound(const Bound &q);

// the serving operators torch.ops.gptq_hip.* of binding_attention.cpp
std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> cache_tables(const Tensor &lengths, const Tensor &counts, const Tensor &tables,
                                                                const Tensor &free_blocks, int64_t tokens, int64_t block_size);
void cache_write(const Tensor &k, const Tensor &v, const Tensor &k_cache, const Tensor &v_cache, const Tensor &slots);
std::tuple<Tensor, Tensor> cache_read(const Tensor &k_cache, const Tensor &v_cache, const Tensor &slots);
void cache_write_mx(const Tensor &k, const Tensor &v, const Tensor &k_codes, const Tensor &k_scales, const Tensor &v_codes, const Tensor &v_scales,
                    const Tensor &slots);
std::tuple<Tensor, Tensor> cache_read_mx(const Tensor &k_codes, const Tensor &k_scales, const Tensor &v_codes, const Tensor &v_scales,
                                         const Tensor &slots, int64_t dim, at::ScalarType dtype);
Tensor paged_attention(const Tensor &q, const Tensor &k_cache, const Tensor &v_cache, const Tensor &tables, const Tensor &starts,
                       const Tensor &contexts, int64_t max_context, int64_t window, int64_t sinks, double scale);
Tensor shared_prefix_attention(const Tensor &q, const Tensor &k_cache, const Tensor &v_cache, const Tensor &prefix_blocks,
                               int64_t prefix_length, const Tensor &tables, const Tensor &starts, const Tensor &contexts,
                               int64_t max_context, double scale);
Tensor paged_attention_mx(const Tensor &q, const Tensor &k_codes, const Tensor &k_scales, const Tensor &v_codes, const Tensor &v_scales,
                          const Tensor &tables, const Tensor &starts, const Tensor &contexts, int64_t max_context, int64_t window,
                          int64_t sinks, double scale);
Tensor shared_prefix_attention_mx(const Tensor &q, const Tensor &k_codes, const Tensor &k_scales, const Tensor &v_codes, const Tensor &v_scales,
                                  const Tensor &prefix_blocks, int64_t prefix_length, const Tensor &tables, const Tensor &starts,
                                  const Tensor &contexts, int64_t max_context, double scale);

}  // namespace gptq_torch
