#define FK_PA_D 64
#define FK_PA_KV kKvFp8
#define FK_PA_NAME d64_fp8
#include "paged_attention_tc_launch.inc"
