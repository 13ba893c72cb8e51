// Parameters of the rotary positions' kernels (rotary.hip).
#pragma once
#include "gated_scan_dev.h"

namespace issm {

constexpr int ROT_MAX_D = 1024;

struct RotP {
  int L, D, R, tokens, H[2];      // tokens = B L; H: heads of the two sides, 0 of one that is absent
  int lpr, pairs, blocks[2];
  unsigned first;                 // the launch's first workgroup, where there are more than one launches
  int group, heads_each, groups[2];   // heads of a token that a wave has at a time, times how often; and of a side, backwards
  Div by_parts, by_L;
  float inv_D;
  const void* x[2];
  long s[2][3], ds[2][3];         // element strides of batch, token and head: of x (without a norm, backwards, of what is turned back), of dy
  const void* dy[2];
  void* y[2];                     // (tokens, H, D): results, or gradients
  const void* w[2];               // (D)
  void* dw[2];                    // (D) in the weights' type, or NULL
  float* part;                    // (blocks, D)
  const float* table;             // (rows, R): R / 2 cosines, R / 2 sines
  long rows;
  const void* pos;                // or NULL: the token's place in its sequence
  long pos_b, pos_l;
  int pos64, w_bf;
  float eps, sign;
};

// Workgroups that walk a side's rows backwards: enough for all CUs, and few enough that their partial sums are soon read again
// (4096 x 4 tokens of 16 and 4 heads of 64, bf16: 512 27.3 us, 768 29.6, 1536 33.0)
inline int rotary_bwd_blocks(long rows) { return rows <= 0 ? 0 : (int)(rows < 512 * 16 ? (rows + 15) / 16 : 512); }

}  // namespace issm
