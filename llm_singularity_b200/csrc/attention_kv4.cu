// Attention over a 4-bit cache, bfloat16 rows (attention_kv4.cuh).
#include "attention_kv4.cuh"

LSB_KV4_ENTRY_POINTS(__nv_bfloat16)
