// Attention over a paged cache on the bf16 matrix cores.
#include "kv_flash.h"
