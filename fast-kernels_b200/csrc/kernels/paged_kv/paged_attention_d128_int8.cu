#define FK_PA_D 128
#define FK_PA_KV kKvInt8
#define FK_PA_NAME d128_int8
#include "paged_attention_tc_launch.inc"
