// Attention over an e4m3 cache, head size 64: instances (attn_cached.h).
#include "attn_cached.h"

ITTS_ATTN_CACHED_INSTANCES(true, 64)
