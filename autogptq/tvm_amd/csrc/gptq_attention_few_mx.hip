// The few-rows attention kernel on caches in MXFP4 (see gptq_attention_few.h).
#include "gptq_attention_few.h"

int gptq::launch_attention_few_mx(const AttentionParams &p, int type, int rt, void *stream) { return launch_few_of<true>(p, type, rt, stream); }
