// Parameters and device parts of the gated linear recurrence (gated_scan.hip).
#pragma once
#include "issm_dev.h"

namespace issm {

constexpr int GS_THREADS = 512, GS_CG = 16, GS_TT = GS_THREADS / GS_CG, GS_S = 4, GS_TILE = GS_TT * GS_S;   // tokens of a tile

struct GScanP {
  int B, L, C, ncb, nk;           // ncb, nk: blocks of channels, tiles of tokens
  const void *x, *g, *i, *dy;     // i, dy: or NULL
  long xb, xl, gb, gl, ib, il, dyb, dyl;   // strides of batch and token in elements; negative ones walk from the end
  const float *A, *h0, *dlast;    // (C); (B, C) or NULL
  const int* ids;                 // or NULL
  long ids_b, ids_l;
  void *y, *dx, *dg, *di;         // yb, yl: strides of all four
  long yb, yl;
  float *last, *hs, *dh0, *part, *dA;   // (B, C); (B, nk, C) states before the tiles; (B, C); partial sums of dA; (C)
  unsigned* tickets;              // tiles of a row on workgroups of their own: a counter for each row of a block of channels, GS_TICKET apart, and
  unsigned long long* words;      // what its tiles tell the ones behind them, (B, ncb, nk, 64); all bits set before the launch
};
constexpr int GS_TICKET = 32;

// What a tile tells the ones behind it of a channel, in one access of 8 bytes, so that nothing needs an order of its own: the map of its tokens,
// H below P, or the state behind it, H below the bits of -0 (P is never negative: a tile with a cut knows the state behind it), or, all bits set,
// nothing yet.
constexpr unsigned GS_STATE = 0x80000000u, GS_NOTHING = 0xffffffffu;
__device__ __forceinline__ void tell(unsigned long long* at, float H, unsigned high) {
  __hip_atomic_store(at, (unsigned long long)high << 32 | __float_as_uint(H), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ unsigned map_bits(float P) { return P != P ? 0x7fc00000u : __float_as_uint(P); }

struct GStepP {
  int rows, C, ncb;
  long slots, state_s;
  const void *x, *g, *i;
  long xs, gs, is;
  const float* A;
  float* state;
  const void* at;                 // or NULL: row r has state r
  int at64;
  void* y;
};

inline int gscan_blocks(int C) { return C >= 4 ? (C + GS_CG * 4 - 1) / (GS_CG * 4) : 1; }
inline int gscan_tiles(int L) { return (int)(((long)L + GS_TILE - 1) / GS_TILE); }

// The first of a thread's V channels: where fewer than V are left they are the last V, and two threads compute the same values
template <int V>
__device__ __forceinline__ int first_channel(int c, int C) { return min(c, C - V); }
// and the channel of one of a block's slots
template <int V>
__device__ __forceinline__ int slot_channel(int c, int slot, int C) { return first_channel<V>(c + slot / V * V, C) + slot % V; }

// V elements side by side, at any element's address: types that promise no more than an element's alignment (the target takes
// wide accesses at any address)
template <int N>
struct __attribute__((packed, aligned(2))) Half {
  uint16_t v[N];
};
template <int N>
struct __attribute__((packed, aligned(4))) Word {
  float v[N];
};
template <bool BF, int V>
struct Piece {
  using Mem = typename std::conditional<BF, Half<V>, Word<V>>::type;
  Mem m;
  __device__ __forceinline__ void load(const void* p, long off) {
    if constexpr (BF) m = *(const Mem*)((const uint16_t*)p + off);
    else m = *(const Mem*)((const float*)p + off);
  }
  __device__ __forceinline__ float operator[](int v) const {
    if constexpr (BF) return bf16_to_f(m.v[v]);
    else return m.v[v];
  }
  static __device__ __forceinline__ void store(void* p, long off, const float (&f)[V]) {
    Mem m;
    if constexpr (BF) {
#pragma unroll
      for (int v = 0; v < V; ++v) m.v[v] = f_to_bf16(f[v]);
      *(Mem*)((uint16_t*)p + off) = m;
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v) m.v[v] = f[v];
      *(Mem*)((float*)p + off) = m;
    }
  }
};

__device__ __forceinline__ float sigmoid(float x) { return __builtin_amdgcn_rcpf(1.0f + ex2(-LOG2E * x)); }
// and 1 - sigmoid, without its cancellation (e bounded, so that e * 0 does not arise; a NaN stays one)
__device__ __forceinline__ void sigmoid2(float x, float& s, float& rest) {
  float z = -LOG2E * x;
  z = z > 126.0f ? 126.0f : z;
  const float e = ex2(z);
  s = __builtin_amdgcn_rcpf(1.0f + e);
  rest = e * s;
}
// a = exp(l) and beta = sqrt(1 - a^2).  Near 0, -expm1(l) as its series: what is left out is below 2^-24 of it at |l| = 1/4 (l^6 / 7! = 4.8e-8)
template <bool NRM>
__device__ __forceinline__ void decay(float l, float& a, float& beta) {
  const float e = ex2(LOG2E * l);
  float q = fmaf(l, 1.0f / 720.0f, 1.0f / 120.0f);
  q = fmaf(l, q, 1.0f / 24.0f);
  q = fmaf(l, q, 1.0f / 6.0f);
  q = fmaf(l, q, 0.5f);
  q = fmaf(l, q, 1.0f);
  const bool near = fabsf(l) < 0.25f;
  const float d = near ? -l * q : 1.0f - e;
  a = near ? 1.0f - d : e;
  if (NRM) beta = __builtin_amdgcn_sqrtf(fmaf(d, a, d));
}

}  // namespace issm
