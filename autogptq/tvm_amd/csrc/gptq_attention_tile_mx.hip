// The attention kernel of tiles on caches in MXFP4 (see gptq_attention_tile.h).
#include "gptq_attention_tile.h"

int gptq::launch_attention_tile_mx(const AttentionParams &p, int type, void *stream) { return launch_tile_of<true>(p, type, stream); }
