// Host-side interface between the C ABI of the decode step (qmk_api.cu) and the paged-cache entry points (qmk_paged.cu).
#pragma once
#include "../../include/qmk_b200.h"

// What qmk_prefix_attention checks before it launches anything.
int qmk_prefix_attention_check(const qmk_prefix_attention_args* a, int device);
