// Attention over a cache in 4 bits, rows of f16 (attn_q4.inc).
#define ROWS_TYPE _Float16
#define ROWS_LAUNCH launch_f16
#include "attn_q4.inc"
