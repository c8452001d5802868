// The shared-prefix attention of bf16 caches.
#include "attn_shared.inc"

int mhip_shared::launch_bf16(mhip_ctx *c, const Job &a, const Cut &k) { return by_head<__bf16>(c, a, k); }
