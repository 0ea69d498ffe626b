#define FK_PA_D 128
#define FK_PA_KV kKvBf16
#define FK_PA_NAME d128_bf16
#include "paged_attention_tc_launch.inc"
