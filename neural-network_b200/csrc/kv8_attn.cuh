// Attention over the 8-bit paged cache: what the handle keeps for it.
#pragma once

#include "kv8.cuh"

namespace specdec {

// Workspaces and kernel attributes of a handle's attention (its device current).
void kv8_attn_create(specdec_kv8 *h);
void kv8_attn_destroy(specdec_kv8 *h);

// Checked views of the caller's records (throw OpError).
Kv8Layer kv8_layer(const specdec_kv8 *h, const specdec_kv8_layer *l);
Kv8Batch kv8_batch(const specdec_kv8 *h, const specdec_kv8_batch *b, int n_tokens);

}  // namespace specdec
