// Attention over a bf16 cache: instances (attn_cached.h).
#include "attn_cached.h"

ITTS_ATTN_CACHED_INSTANCES(false, 64)
ITTS_ATTN_CACHED_INSTANCES(false, 128)
