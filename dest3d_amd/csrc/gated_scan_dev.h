// Parameters and device parts of the gated linear recurrence (gated_scan.hip).
#pragma once
#include "issm_dev.h"

namespace issm {

// A workgroup: GS_TT segments of tokens times GS_CG groups of channels, and a wave that joins the segments' maps
constexpr int GS_THREADS = 512, GS_CG = 16, GS_TT = (GS_THREADS - 64) / GS_CG;
// Tokens of a thread: forward, in workgroups that share a row and in ones that walk it, and backward.  The forward leaves the states in front of
// the backward's tiles.  (Bf16, 1 x 131072 x 2048, shared: forward 4 tokens 529 us, 2 714; backward, in an earlier form, 2 tokens 1181, 4 1231.
// 16 x 4096 x 2048, walked: forward 2 tokens 246, 4, which spill, 355.  The shared forward's 4 spill a little too, at four waves a SIMD: in bf16 with an
// in_gate 5 registers, packed 20 or 29, without buffers 12 to 23; so do the shared backward's forms without buffers, 16 and 18.)
constexpr int GS_S_SHARED = 4, GS_S_WALKED = 2, GS_S_BACK = 2, GS_TILE_BACK = GS_TT * GS_S_BACK;

struct GScanP {
  int B, L, C, ncb, nk, nb;       // ncb, nk, nb: blocks of channels, tiles of tokens, the backward's
  bool nrm, lines;                // lines: blocks of channels end inside cache lines
  const void *x, *g, *i, *dy;     // i, dy: or NULL
  long xb, xl, gb, gl, ib, il, dyb, dyl;   // strides of batch and token in elements; negative ones walk from the end
  const float *A, *h0, *dlast;    // (C); (B, C) or NULL
  const int* ids;                 // or NULL
  long ids_b, ids_l;
  void *y, *dx, *dg, *di;         // yb, yl: strides of all four
  long yb, yl;
  float *last, *hs, *dh0, *part, *dA;   // (B, C); (B, tiles of the backward, C) states in front of them; (B, C); partial sums of dA; (C)
  unsigned* tickets;              // tiles of a row on workgroups of their own: a counter for each row of a block of channels, GS_TICKET apart, and
  unsigned long long* words;      // what its tiles tell the ones behind them, (B, ncb, GS_LOOK + nk, 64); all bits set before the launch
};
// Words of a look.  (Bf16, 1 x 131072 x 2048, forward and backward: 2 593 and 1239 us, 4 529 and 1126, 8 534 and 1170, 16 571 and 1762.)
constexpr int GS_TICKET = 32, GS_LOOK = 4;

// What a tile tells the ones behind it of a channel, in one access of 8 bytes, so that nothing needs an order of its own: the map of its tokens,
// H below P, or the state behind it, H below the bits of -0 (P is a number, never negative: a tile with a cut knows the state behind it), or, all
// bits set, nothing yet.
constexpr unsigned GS_STATE = 0x80000000u, GS_NOTHING = 0xffffffffu;
__device__ __forceinline__ void tell(unsigned long long* at, float H, unsigned high) {
  __hip_atomic_store(at, (unsigned long long)high << 32 | __float_as_uint(H), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

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
inline int gscan_tiles(int L, int S) { return (int)(((long)L + GS_TT * S - 1) / (GS_TT * S)); }

// The first of a thread's V channels: where fewer than V are left they are the last V, and two threads compute the same values
template <int V>
__device__ __forceinline__ int first_channel(int c, int C) { return min(c, C - V); }
// and the channel of one of a block's slots
template <int V>
__device__ __forceinline__ int slot_channel(int c, int slot, int C) { return first_channel<V>(c + slot / V * V, C) + slot % V; }

// V elements side by side, at any element's address: types that promise no more than an element's alignment (the target takes
// wide accesses at any address).  Pairs of bf16 stay one register: as halves the compiler keeps each in a register of its own.
template <int N>
struct __attribute__((packed, aligned(2))) Half {
  unsigned v[N / 2];
  __device__ __forceinline__ float operator[](int i) const { return __uint_as_float(i & 1 ? v[i / 2] & 0xffff0000u : v[i / 2] << 16); }
  __device__ __forceinline__ void put(const float (&f)[N]) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) v[i] = pack_bf16(f[2 * i], f[2 * i + 1]);
  }
};
template <>
struct Half<1> {
  uint16_t v;
  __device__ __forceinline__ float operator[](int) const { return bf16_to_f(v); }
  __device__ __forceinline__ void put(const float (&f)[1]) { v = f_to_bf16(f[0]); }
};
template <int N>
struct __attribute__((packed, aligned(4))) Word {
  float v[N];
  __device__ __forceinline__ float operator[](int i) const { return v[i]; }
  __device__ __forceinline__ void put(const float (&f)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = f[i];
  }
};
template <bool BF, int V>
struct Piece {
  using Mem = typename std::conditional<BF, Half<V>, Word<V>>::type;
  using Element = typename std::conditional<BF, uint16_t, float>::type;
  Mem m;
  __device__ __forceinline__ void load(const void* p, long off) { m = *(const Mem*)((const Element*)p + off); }
  __device__ __forceinline__ float operator[](int v) const { return m[v]; }
  // Its registers as something new to the compiler: two ways behind a branch that begin with the same conversions would have all of them in
  // front of it, in registers of their own
  template <bool WAY>
  __device__ __forceinline__ void apart() {
    unsigned(&w)[sizeof(Mem) / 4] = (unsigned(&)[sizeof(Mem) / 4])m;
#pragma unroll
    for (unsigned i = 0; i < sizeof(Mem) / 4; ++i) {
      if constexpr (WAY) asm volatile("; near" : "+v"(w[i]));
      else asm volatile("; any" : "+v"(w[i]));
    }
  }
  __device__ __forceinline__ void keep(bool there) {   // or zeros
    float f[V];
#pragma unroll
    for (int v = 0; v < V; ++v) f[v] = there ? m[v] : 0.0f;
    m.put(f);
  }
  static __device__ __forceinline__ void store(void* p, long off, const float (&f)[V]) {
    Mem m;
    m.put(f);
    *(Mem*)((Element*)p + off) = m;
  }
};

__device__ __forceinline__ float sigmoid(float x) { return __builtin_amdgcn_rcpf(1.0f + ex2(-LOG2E * x)); }
// a = exp(l) and beta = sqrt(1 - a^2).  Up to |l| = 1/4, -expm1(l) as its series: what is left out is below 2^-24 of it (l^6 / 7! = 4.8e-8).
// NEAR: no l is beyond that (the same values, without the other form's exponential)
constexpr float GS_NEAR = 0.25f;
template <bool NEAR>
__device__ __forceinline__ void decay(float l, bool nrm, float& a, float& beta) {
  float q = fmaf(l, 1.0f / 720.0f, 1.0f / 120.0f);
  q = fmaf(l, q, 1.0f / 24.0f);
  q = fmaf(l, q, 1.0f / 6.0f);
  q = fmaf(l, q, 0.5f);
  q = fmaf(l, q, 1.0f);
  float d = -l * q;
  a = 1.0f - d;
  if (!NEAR) {
    const float e = ex2(LOG2E * l);
    const bool near = fabsf(l) < GS_NEAR;
    d = near ? d : 1.0f - e;
    a = near ? a : e;
  }
  beta = nrm ? __builtin_amdgcn_sqrtf(fmaf(d, a, d)) : 1.0f;
}

// The sum of rows strand, strand + 64, ... of a column, four requests at a time, in their order
__device__ __forceinline__ float strand_sum(const float* column, int stride, int strand, int rows) {
  float sum = 0.0f;
  int r = strand;
  for (; r + 192 < rows; r += 256) {
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = column[(long)(r + 64 * i) * stride];
#pragma unroll
    for (int i = 0; i < 4; ++i) sum += v[i];
  }
  for (; r < rows; r += 64) sum += column[(long)r * stride];
  return sum;
}

}  // namespace issm
