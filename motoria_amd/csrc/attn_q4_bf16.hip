// Attention over a cache in 4 bits, rows of bf16 (attn_q4.inc).
#define ROWS_TYPE __bf16
#define ROWS_LAUNCH launch_bf16
#include "attn_q4.inc"
