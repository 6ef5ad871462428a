// Shared memory of the one-kernel int8 expert layer (moe_i8.cu), in host arithmetic alone: a test compiles this by itself and checks that no stage
// is read beyond its end.
#pragma once

namespace b2q {
namespace mi8 {
constexpr int WARPS = 8, WORKERS = 32 * WARPS;              // the warps that multiply
constexpr int MAX_TOK = 16, MAX_K = 32, MAX_PAIRS = MAX_TOK * MAX_K, MAX_E = 1024;
constexpr int PASS = 16;                                   // groups of eight columns whose sums are held at a time
constexpr int TABLE_MAX = 24 * 1024;                       // bytes of the down part's sums, and of its scales
constexpr int XR = 4;                                      // pairs of a down stage; an expert with more fetches its rows again, from L2
constexpr int PIECE = 2048;                                // longest k of a stage: 256 elements of eight bytes in a TMA box
constexpr int MAX_STAGES = 32, BAR_BYTES = 16 * MAX_STAGES + 16;
constexpr int SMEM_MAX = 232448 - 1024;                    // of a CTA, static part included
constexpr int STATIC_BYTES = 21104;                        // the static part, at most

struct Sizes {
  int grid, pitch, row_cap, xr;                            // xr: pairs of a down stage
  int front;                                               // bytes of the tokens' codes, or of the tables that take their place
  int up_piece, down_piece, down_rows;                     // k of a stage; weight rows of a down stage
  int stages, stage_bytes, smem;                           // smem: the dynamic part
};

inline int room(int fixed) { return SMEM_MAX - STATIC_BYTES - fixed; }

// k of a stage: the whole row where six stages of that fit, else what fits (a TMA box has 2048 bytes of a row at most)
inline int piece_of(int K, int rows, int more, int fixed) {
  const int fits = (room(fixed) / 6 - more) / rows;
  if (K <= fits && K <= PIECE) return K;
  const int v = fits < PIECE ? fits : PIECE;
  return v / 64 * 64;
}

// pitch: bytes between two tokens' codes
inline Sizes sizes_of(int T, int k, int H, int I, int pitch, int sms) {
  Sizes s{};
  const int pairs = T * k;
  s.grid = sms < H ? sms : H;
  s.pitch = pitch;
  s.xr = T < XR ? T : XR;
  s.row_cap = (H + s.grid - 1) / s.grid;
  const int tables = 2 * pairs * s.row_cap * 4, codes = T * pitch;
  s.front = ((codes > tables ? codes : tables) + 255) / 256 * 256;
  const int fixed = s.front + 2 * PASS * T * 16 * 4 + BAR_BYTES;
  s.up_piece = piece_of(H, 8, 0, fixed);
  // up to sixteen rows that are one run of memory, if there are more than eight and they fit; else eight
  const int most = s.row_cap < 16 ? s.row_cap : 16;
  s.down_rows = s.row_cap > 8 && piece_of(I, most + s.xr, 16 * s.xr, fixed) == I ? most : 8;
  s.down_piece = piece_of(I, s.down_rows + s.xr, 16 * s.xr, fixed);
  const int up = 8 * s.up_piece, down = s.down_rows * s.down_piece + s.xr * (s.down_piece + 16);
  s.stage_bytes = ((up > down ? up : down) + 127) / 128 * 128;
  s.stages = room(fixed) / s.stage_bytes;
  if (s.stages > MAX_STAGES) s.stages = MAX_STAGES;
  s.smem = s.stages * s.stage_bytes + fixed;
  return s;
}
}  // namespace mi8
}  // namespace b2q
