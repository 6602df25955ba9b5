// attend_share.h - which tokens of a tile the lanes of a wave bring
// (k_attend.h), apart from the kernels so that the host can go through them.
#pragma once

namespace relx {

// A wave's NT tokens of a tile, DP elements of CELL bytes each, 16 bytes a lane
// and load. Where a load has room for more tokens than the wave has, the lanes
// past them bring nothing.
template <int DP, int CELL, int NT> struct Share {
  static constexpr int LB = 16 / CELL; // elements of a lane's load
  static constexpr int TL = DP / LB;   // lanes of a token
  static constexpr int TPI = 64 / TL;  // tokens of a load
  static constexpr int LOADS = NT > TPI ? NT / TPI : 1;
  static constexpr bool brings(int lane) { return NT >= TPI || lane / TL < NT; }
  // The token that a lane addresses in a load. Loads through registers are not
  // masked (a branch round each of them), so lanes that bring nothing read the
  // first token again, which is in the cache as theirs may not be.
  static constexpr int token(int lane) { return brings(lane) ? lane / TL : 0; }
};

} // namespace relx
