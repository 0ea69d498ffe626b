#define FK_PA_D 128
#define FK_PA_KV kKvFp8
#define FK_PA_NAME d128_fp8
#include "paged_attention_tc_launch.inc"
