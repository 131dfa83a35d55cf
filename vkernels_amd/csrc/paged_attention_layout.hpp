// paged_attention_layout.hpp — which bytes of a key or value row the lanes of a wavefront load, as pure
// functions of integers.  The kernel (paged_attention.hip) calls them; tests/test_paged_attention_layout.py
// compiles them for the host and checks for every width and type that no lane reads a byte outside
// its row and that every byte of the row is read.
#pragma once

#ifndef __HIPCC__
#ifndef __host__
#define __host__
#define __device__
#endif
#endif

namespace vk {

// The width that the kernel is compiled for, of a head of D values.
__host__ __device__ constexpr inline int pa_padded_width(int D, bool fp8) {
  if (D <= 64) return 64;
  if (D <= 96 && !fp8) return 96;
  return D <= 128 ? 128 : D <= 192 ? 192 : 256;
}

// Keys: lane (col, quad) loads 16 bytes of row col in each of `pa_key_loads` loads, 64 bytes of a row
// together (padded rows are multiples of that).
__host__ __device__ constexpr inline int pa_key_loads(int padded_row_bytes) { return padded_row_bytes / 64; }

// Values: the lanes that share a row, the 16-byte pieces of a padded row rounded up to a power of two,
// so that a load takes whole rows.
__host__ __device__ constexpr inline int pa_value_pieces(int padded_row_bytes) {
  return padded_row_bytes <= 64 ? 4 : padded_row_bytes <= 128 ? 8 : padded_row_bytes <= 256 ? 16 : 32;
}

// Where in a row of `row_bytes` a 16-byte piece is read from.  A row of 96 or 192 values has fewer pieces
// than lanes, and so has one that is narrower than its padded width: a lane without a piece of its own
// reads the first one again (a row's end may be the end of the cache's memory).
__host__ __device__ constexpr inline int pa_piece_at(int at, int row_bytes) { return at < row_bytes ? at : 0; }
__host__ __device__ constexpr inline int pa_key_at(int quad, int load) { return quad * 16 + load * 64; }
__host__ __device__ constexpr inline int pa_value_at(int piece, int row_bytes) { return pa_piece_at(piece * 16, row_bytes); }

}  // namespace vk
