// Kernels of a serving loop: a paged cache of keys and values (append, keep,
// attention) and rules on logits.
#include "kv_append.h"
#include "kv_attention.h"
#include "kv_rows.h"
#include "logit_rules.h"
