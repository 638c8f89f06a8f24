// The few-rows attention kernel on caches in fp16 and bf16 (see gptq_attention_few.h).
#include "gptq_attention_few.h"

int gptq::launch_attention_few(const AttentionParams &p, int type, int rt, void *stream) { return launch_few_of<false>(p, type, rt, stream); }
