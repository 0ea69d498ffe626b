#define FK_PA_D 64
#define FK_PA_KV kKvBf16
#define FK_PA_NAME d64_bf16
#include "paged_attention_tc_launch.inc"
