// Which LDS buffer of the tiled row attention kernel (rows_tile.hpp) holds which staged rows, and when
// they are touched. Host code too: the order is checked on the CPU by walking a share's iterations.
#pragma once

#if defined(__HIPCC__)
#define LOGKV_HD __host__ __device__
#else
#define LOGKV_HD
#endif

namespace logkv {

// A share's tiles are walked in iterations 0, 1, ..., each opened by the block's only barrier, so a
// buffer must not be written in an iteration that reads it. RB 32-row blocks a tile (and wave). In
// iteration t, in this order:
//
//   block kb     reads                                  writes
//   0 .. RB - 1  V(t), block kb                         -
//                K and bias of the block to come:       -
//                (t, kb + 1), behind the last (t + 1, 0)
//                (RB > 1) K of the one after that       -
//   RB - 1       -                                      V(t + 1), behind it K and bias of t + 2
//
//   K(t) of block 0 is read last in iteration t - 1, of a later block in iteration t. So with one block
//   the tile behind the next takes K(t)'s buffer in iteration t; with more it needs a third one.
//   V(t) is read in iteration t alone: two buffers.
template <int RB>
struct RowsSchedule {
  static constexpr int kAhead = 2;                    // K of tile t + kAhead is stored in iteration t
  static constexpr int kKBuffers = RB > 1 ? 3 : 2;    // of K and the bias
  static constexpr int kVBuffers = 2;
  // Iteration, relative to a tile's own, in which its K and bias are read last.
  static constexpr int kLastKRead = RB > 1 ? 0 : -1;
  // The tile whose K the stored one takes the place of, relative to the iteration, has been read before.
  static_assert(kAhead - kKBuffers + kLastKRead < 0, "K is overwritten in an iteration that reads it");
  static LOGKV_HD constexpr int next_k(int buffer) { return buffer + 1 < kKBuffers ? buffer + 1 : 0; }
  static LOGKV_HD constexpr int next_v(int buffer) { return buffer ^ 1; }
};

}  // namespace logkv
