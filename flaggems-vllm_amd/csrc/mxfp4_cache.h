// The paged key/value cache in MXFP4, shared by its writer and its reader.
//
// A block holds `page` tokens of every key/value head.  Per (block, head), one
// after the other:
//   page x D/2   bytes of key codes (E2M1, two to a byte, the even dim low)
//   page x D/2   bytes of value codes
//   page x D/32  bytes of key scales (UE8M0, byte b stands for 2^(b - 127))
//   page x D/32  bytes of value scales
// so that a head's block is one run of page * (D + D/16) bytes, 136 a token at
// D = 128 (512 in bf16).  page is a multiple of 16: 16 tokens are what one
// matrix instruction takes, and their codes and scales are whole runs of 16
// bytes that no block's end cuts.
#pragma once

#include <stdint.h>

namespace fgv {

constexpr int kMxBlock = 32;  // values under one scale

constexpr int mx_token_bytes(int dim) { return dim + dim / 16; }

// First byte of the part of a head's block: 0 key codes, 1 value codes, 2 key scales, 3 value scales.
__host__ __device__ constexpr int64_t mx_part(int part, int64_t page, int dim) {
    return part < 2 ? part * page * (dim / 2) : page * dim + (part - 2) * page * (dim / kMxBlock);
}

}  // namespace fgv
