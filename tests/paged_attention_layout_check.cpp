// Host-side walk over the bytes of a key and a value row that the paged attention's lanes load (the functions
// of vkernels_amd/csrc/paged_attention_layout.hpp, compiled for the CPU).  For a head width and an element
// size it checks
//   - every 16-byte load of a key or value row ends within the row's bytes;
//   - every byte of the row is read, by the lane that stands for it;
//   - the value loads of a tile cover its 32 rows, each once.
// Usage: paged_attention_layout_check D elem_bytes ; exit status 0 = all hold.
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "paged_attention_layout.hpp"

using namespace vk;

#define CHECK(cond, ...)                                  \
  do {                                                    \
    if (!(cond)) {                                        \
      std::fprintf(stderr, "FAILED %s: ", #cond);         \
      std::fprintf(stderr, __VA_ARGS__);                  \
      std::fprintf(stderr, "\n");                         \
      return 1;                                           \
    }                                                     \
  } while (0)

int main(int argc, char** argv) {
  if (argc != 3) return 2;
  const int D = std::atoi(argv[1]), elem = std::atoi(argv[2]);
  const int row = D * elem, padded = pa_padded_width(D, elem == 1) * elem;
  CHECK(padded >= row && padded % 64 == 0, "padded %d of %d bytes", padded, row);

  std::vector<int> seen(row, 0);
  for (int load = 0; load < pa_key_loads(padded); ++load)
    for (int quad = 0; quad < 4; ++quad) {
      const int at = pa_key_at(quad, load), from = pa_piece_at(at, row);
      CHECK(from >= 0 && from + 16 <= row, "key quad %d load %d reads [%d, %d) of %d", quad, load, from, from + 16, row);
      if (at < row)
        for (int i = 0; i < 16; ++i) ++seen[at + i];
    }
  for (int i = 0; i < row; ++i) CHECK(seen[i] == 1, "key byte %d is taken %d times", i, seen[i]);

  const int pieces = pa_value_pieces(padded);
  CHECK(pieces * 16 >= padded && 64 % pieces == 0, "%d pieces", pieces);
  const int rows_per_load = 64 / pieces, loads = 32 / rows_per_load;
  CHECK(loads * rows_per_load == 32 && loads % 2 == 0, "%d loads of %d rows", loads, rows_per_load);
  std::vector<int> taken(32 * row, 0);
  for (int load = 0; load < loads; ++load)
    for (int lane = 0; lane < 64; ++lane) {
      const int piece = lane % pieces, r = load * rows_per_load + lane / pieces;
      const int from = pa_value_at(piece, row);
      CHECK(r < 32 && from >= 0 && from + 16 <= row, "value lane %d reads [%d, %d) of %d", lane, from, from + 16, row);
      if (piece * 16 < row)
        for (int i = 0; i < 16; ++i) ++taken[r * row + piece * 16 + i];
    }
  for (int i = 0; i < 32 * row; ++i) CHECK(taken[i] == 1, "value byte %d of row %d is taken %d times", i % row, i / row, taken[i]);
  return 0;
}
