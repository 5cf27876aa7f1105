// Which elements of a row paged_token's lanes read, as plain C++ that the host walks over every head dim (tests/test_paged_reads.py).
#pragma once

namespace limn {

// Head dims whose rows the tiled kernels of a paged cache serve: whole 16-byte chunks, up to 128.
constexpr bool paged_dim(long hd, int element_bytes) { return hd >= 1 && hd <= 128 && hd % (16 / element_bytes) == 0; }

// The tile width that paged_token runs a head dim at.
constexpr int token_width(long hd) { return hd <= 64 ? 64 : 128; }

// Of 16 lanes with W dims each, lane n has those from W n on, where there are any (W n < hd), and reads W of them from here on: a row
// that ends among them (float32 of 68, 76, .. 124 dims, W = 8) is read to its end and no further, with dims of the lane before.
constexpr int value_dim(int n, int W, int hd) { return W * n + W <= hd ? W * n : hd - W; }

}  // namespace limn
