// window.h - arguments and launches of attention over packed sequences
// (k_window.h), checked and filled by window.cpp. Strides are in elements.
#pragma once

#include "attention.h"

namespace relx {

constexpr int kFew = 128; // tokens of a row whose D the backward sums from its weights

struct WindowArgs {
  Heads q, k, v, o;
  Heads dout, dq, dk, dv;
  const int32_t *starts;
  float *lse;        // [heads, rows]
  float *stats;      // [heads, 2, rows]: -lse / scale (both in powers of two), and -D
  float *first_sums; // [pieces, kv_heads, sinks, 2, width]: what pieces of rows add to the first tokens' gradients
  // a workgroup's rows: tokens, times heads of a group (in `parts` where those are many)
  FastDiv tile_tokens, tile_heads;
  FastDiv key_tokens, first_tokens; // tokens of its keys; rows that share sums of the first tokens
  FastDiv longer;                   // the fewest rows of a sequence that some window leaves
  int32_t row_pieces, key_pieces, first_pieces; // numbers of such pieces, at most
  int32_t first_blocks;                         // of 32 first tokens
  int32_t rows, sequences, heads, kv_heads, parts, dim, window, sinks;
  float scale, plain_scale; // of a score, times log2 e, and as it is
  int32_t few_pieces;       // of a sequence's rows, at most, that see up to kFew tokens; 0: any may
};
hipError_t window_launch_f16(const WindowArgs &a, bool back, hipStream_t s);
hipError_t window_launch_bf16(const WindowArgs &a, bool back, hipStream_t s);

} // namespace relx
