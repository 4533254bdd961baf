// Attention over a 4-bit cache, 32-bit rows (attention_kv4.cuh).
#include "attention_kv4.cuh"

LSB_KV4_ENTRY_POINTS(float)
