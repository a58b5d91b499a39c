// What the engine needs of the paged cache beyond include/eii.h.
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

#include "eii.h"

namespace eii {

// eii_paged_attention with prob_bits 16 for rows that see positions 0 .. pos[r], q dense, the context written as
// the row-blocked byte planes that the O projection reads.  The handle's device is current.
int paged_attention_planes(eii_paged* p, const eii_pages& pages, const int16_t* q, int n_rows, const int32_t* seq,
                           const int32_t* pos, int max_len, int shift_s, int shift_c, int bits_c, uint8_t* planes,
                           int n_planes, int offset, cudaStream_t st);

}  // namespace eii
