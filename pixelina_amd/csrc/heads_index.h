// Which values of an attention head a lane of heads_device.h holds; without a device, so
// that a test on the host enumerates them.
#pragma once

namespace pixhip {

// How a lane's values lie: SCALAR pairs p = lane + G j, any size and alignment;
// HALVES float4s of either half of the rotated part (pairs (i, i + rotary / 2));
// ADJACENT 8 values in a row (pairs (2i, 2i + 1)).  The wide ones need a rotary
// size that is a multiple of 8, a head size that is one of 4, and 16-byte aligned
// rows (HeadTurn::vec).
enum { kTurnScalar = 0, kTurnHalves = 1, kTurnAdjacent = 2 };

// Value indices of the lane's quads (wide forms); the second may lie past the head.
template <int MODE>
constexpr void turn_quads(int lp, int rotary, int& o1, int& o2)
{
    if (MODE == kTurnAdjacent) {
        o1 = 8 * lp;
        o2 = o1 + 4;
    } else if (lp < rotary / 8) {
        o1 = 4 * lp;
        o2 = rotary / 2 + 4 * lp;
    } else {
        o1 = rotary + 8 * (lp - rotary / 8);
        o2 = o1 + 4;
    }
}

// Value indices of pair j of a lane of G (the scalar form); at or past the head's size: none.
template <int G>
constexpr void turn_pair(int lp, int j, int rotary, bool interleaved, int& ia, int& ib)
{
    const int p = lp + G * j, half = rotary / 2;
    if (p >= half) {
        ia = rotary + 2 * (p - half);
        ib = ia + 1;
    } else {
        ia = interleaved? 2 * p : p;
        ib = interleaved? ia + 1 : p + half;
    }
}

}  // namespace pixhip
