// The attention kernel of tiles on caches in fp16 and bf16 (see gptq_attention_tile.h), and the join of divided tiles.
#include "gptq_attention_tile.h"

namespace gptq {

// Joins the parts of tiles that are divided, or stand behind a shared prefix: kJoinRows rows of a tile a workgroup.  EVEN: the parts' keys follow from the
// lengths.
template <typename E, bool EVEN>
__global__ __launch_bounds__(256) void attention_join_kernel(const AttentionParams p)
{
    const int h = blockIdx.x % p.kv_heads, tile = blockIdx.x / p.kv_heads, r0 = blockIdx.y * kJoinRows;
    QueryTile q;
    int split, chunk, parts;
    if (!find_tile<EVEN, true>(p, tile, q, split, chunk, parts) || r0 >= q.rows) return;
    if (parts == 1 && p.prefix_parts == 0) return;
    const long long all = (long long)p.tokens * p.heads;
    const int quads = p.dim / 4;
    for (int i = threadIdx.x; i < min(kJoinRows, q.rows - r0) * quads; i += 256) {
        const int r = i / quads, d = (i - r * quads) * 4;
        const long long at = out_row(p, q, h, r0 + r);
        Sum x = {kNone, 0.0f, {0.0f, 0.0f, 0.0f, 0.0f}};
        add_prefix(p, x, at, d);
        add_parts<false>(x, 0, 1, parts, [&](int s) { return p.own_stats + 2 * (s * all + at); },
                         [&](int s) { return p.own_parts + (s * all + at) * p.dim + d; });
        store_row4<E>(p.out, at * p.dim + d, x.result());
    }
}

void launch_attention_join(const AttentionParams &p, int type, unsigned tiles, void *stream)
{
    const dim3 grid(tiles, kTileRows / kJoinRows);
    auto join = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, (hipStream_t)stream, p); };
    if (type == GPTQ_HIP_TYPE_FP16) p.even ? join(attention_join_kernel<_Float16, true>) : join(attention_join_kernel<_Float16, false>);
    else p.even ? join(attention_join_kernel<__bf16, true>) : join(attention_join_kernel<__bf16, false>);
}

int launch_attention_tile(const AttentionParams &p, int type, void *stream) { return launch_tile_of<false>(p, type, stream); }

}  // namespace gptq
