// The shared-prefix attention of fp16 caches.
#include "attn_shared.inc"

int mhip_shared::launch_f16(mhip_ctx *c, const Job &a, const Cut &k) { return by_head<_Float16>(c, a, k); }
