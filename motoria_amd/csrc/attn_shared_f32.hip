// The shared-prefix attention of fp32 caches.
#include "attn_shared.inc"

int mhip_shared::launch_f32(mhip_ctx *c, const Job &a, const Cut &k) { return by_head<float>(c, a, k); }
