#define FK_PA_D 64
#define FK_PA_KV kKvInt8
#define FK_PA_NAME d64_int8
#include "paged_attention_tc_launch.inc"
