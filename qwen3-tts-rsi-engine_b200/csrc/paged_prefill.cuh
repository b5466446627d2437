// The tensor-core form of q3t_paged_prefill_attention (paged_prefill.cu); arguments are checked by the caller.
#pragma once

#include <stddef.h>
#include <stdint.h>

#include "q3t.h"

namespace q3t {

// Whether sizes and scale are within what the tiled kernel takes (its counters are 32-bit, its scale positive).
bool prefill_tiles_supported(int64_t rows, int64_t capacity, double scale);
size_t prefill_tiles_workspace(int64_t rows, int64_t sequences, int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                               int64_t capacity);
int launch_prefill_tiles(const q3t_paged_prefill& call, unsigned* status, void* stream, const char* name);

}  // namespace q3t
