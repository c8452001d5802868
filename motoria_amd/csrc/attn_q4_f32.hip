// Attention over a cache in 4 bits, rows of f32 (attn_q4.inc).
#define ROWS_TYPE float
#define ROWS_LAUNCH launch_f32
#include "attn_q4.inc"
