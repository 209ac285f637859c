// Layout of the paged key/value cache held in 4 bits.
//
// The pool is [num_pages][kv_heads] blocks of page * (D + D/8) bytes; a block holds one page of one head:
//   keys' codes    [page][D/2]
//   values' codes  [page][D/2]
//   keys' pairs    [page][D/64] x {scale, centre} fp16
//   values' pairs  [page][D/64] x {scale, centre} fp16
// A value is scale * (code - 8) + centre, one pair per 64 consecutive channels.  One block is contiguous, so a page
// of a head is ONE bulk copy (four with codes and pairs of keys and values in arrays of their own: at 16-position
// pages and head_dim 64 those would be copies of 64 to 512 bytes).
//
// Codes of a row: 32-bit word u*G + g (G = D/64, u = 0..7) holds channels 64g + 8u .. + 7, lowest nibble first.  A
// lane that takes G consecutive words thus has eight channels of EACH group, which is what both products of decode
// attention want: their operands must not mix groups, whose scales differ.
#pragma once

#include "common.cuh"

namespace i8tk {

__host__ __device__ constexpr int kv4_row_bytes(int D) { return D / 2; }
__host__ __device__ constexpr int kv4_pair_bytes(int D) { return D / 16; }
__host__ __device__ constexpr int kv4_block_bytes(int page, int D) { return page * (D + D / 8); }
inline bool kv4_page_ok(int page) { return page == 16 || page == 32 || page == 64 || page == 128; }

}  // namespace i8tk
