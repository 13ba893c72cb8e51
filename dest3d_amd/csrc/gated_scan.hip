// Gated linear recurrence for gfx950: a state of one number for each channel.
//   r = sigmoid(gate),  l = A r,  a = exp(l),  beta = sqrt(1 - a^2)  (or 1),  u = sigmoid(in_gate) x  (or x)
//   h_t = a_t h_{t-1} + beta_t u_t;   at a cut (the sequence id changes) h_t = beta_t u_t
// and backwards, with G_t the whole gradient of h_t and c_t what of it reaches h_{t-1}:
//   G_t = dy_t + c_{t+1},   c_t = a_t G_t (0 at a cut),   dh0 = c_0
//   dx = G beta s,   din_gate = G beta x s (1 - s),   dl = c_t h_{t-1} - G u a^2 / beta,   dgate = dl l (1 - r),   dA = sum dl r
//
// a and beta come from d = 1 - a = -expm1(l): a decay next to one that is rounded with a bias of half a place adds that bias up over
// all tokens it remembers (1000 at a = 0.999), while 1 - d is rounded to nearest, and 1 - a^2 = d (1 + a) has no cancellation.
//
// A workgroup takes tiles of GS_TT * S tokens and GS_CG * V channels: a thread V channels of S tokens one behind the other, whose map
// h -> P h + H it leaves in LDS.  A wave without tokens of its own, a channel a lane, joins the maps of the tile and gives every thread its first
// state; with the tokens' requests out of its way its looks at other tiles come back at once (a wave's loads return in their order).
// GS_CG * V = 64 channels are rows' pieces of 128 bytes in bf16: with half of that a row of
// 131072 tokens of 2048 channels, 585 us at the time, took 715.
//
// Bound by bytes, and where rows are few by waiting for the states in front (a copy of 1 GiB: 5.1 TB/s).  us forward and backward, with in_gate and beta,
// calls one behind the other, their launches that clear the words and sum dA included (kernels alone, 8 x 4096 x 2048: 129 and 238):
//   bf16, 2048 channels      all |A| < 1/4              wide decays     packed
//   16 x 4096, walked        246, 4.4 TB/s   423, 4.4   256   449       256   522
//   8 x 4096, by 2 and 3     139, 3.9        261, 3.6   132   256       156   278
//   1 x 131072, by 16 and 24 527, 4.1       1115, 3.4   530  1137       584  1162    (copies that did not wait: 465 and 852)
//   fp32, 1024 channels: 32 x 4096, walked 454, 4.7, and 780, 4.8 (packed 461 and 798); 8 x 4096, by 4 and 6, 120, 4.5, and 213, 4.4 (packed 125 and 226)
// What the forms pay: packed ones look at the ids of each token, and shared ones spill there (gated_scan_dev.h); rows without buffers (odd widths in bf16, odd
// addresses) have 64-bit places: 16 x 4096 x 2047 253 and 483, 8 x 4096 x 2047 180 and 339, whose shared forms spill too.
#include "gated_scan_dev.h"

// (every multiply-add is written as one: the forms of a kernel that do the same sums are to give the same bits)
#pragma clang fp contract(off)

namespace issm {

// A thread's rows of one tensor in a tile: S tokens, V channels each.
// BUF: behind a buffer that ends with the tile's rows (those past the end of the sequence read zero and are not stored): a row is one 32-bit
// addition.  It takes rows that start at whole dwords and lie within 2^31 bytes of a tile; the others have 64-bit addresses, clamped to the last token.
template <bool BF, int V, int S, bool BUF>
struct Rows {
  static constexpr int SIZE = BF ? 2 : 4, T = GS_TT * S;
  typedef unsigned u2 __attribute__((ext_vector_type(2)));
  typedef unsigned u4 __attribute__((ext_vector_type(4)));
  __amdgpu_buffer_rsrc_t buf;
  unsigned off, step;
  char* base;
  long ls;
  int t0, end;
  // tile k of a sequence of L tokens, the thread's first row t0
  __device__ __forceinline__ Rows(const void* q, long bs, long ls_, int b, int k, int L, int C, int t0_, int c0) {
    if constexpr (BUF) {
      const int rows = min(T, L - k * T), j = t0_ - k * T;
      const unsigned gap = (unsigned)(ls_ < 0 ? -ls_ : ls_);
      buf = __builtin_amdgcn_make_buffer_rsrc((char*)const_cast<void*>(q) + (b * bs + (k * (long)T + (ls_ < 0 ? rows - 1 : 0)) * ls_) * SIZE, 0,
                                              ((rows - 1) * gap + C) * SIZE, 0x00027000);
      off = ((unsigned)(ls_ < 0 ? rows - 1 - j : j) * gap + c0) * SIZE;
      step = (unsigned)ls_ * SIZE;
    } else {
      base = (char*)const_cast<void*>(q) + (b * bs + c0) * SIZE;
      ls = ls_ * SIZE;
      t0 = t0_;
      end = L - 1;
    }
  }
  __device__ __forceinline__ void load(Piece<BF, V> (&v)[S]) const {
#pragma unroll
    for (int s = 0; s < S; ++s) {
      if constexpr (!BUF) v[s].load(base + min(t0 + s, end) * ls, 0);
      else if constexpr (BF) v[s].m = __builtin_bit_cast(Half<V>, (u2)__builtin_amdgcn_raw_buffer_load_b64(buf, off + s * step, 0, 0));
      else v[s].m = __builtin_bit_cast(Word<V>, (u4)__builtin_amdgcn_raw_buffer_load_b128(buf, off + s * step, 0, 0));
    }
  }
  __device__ __forceinline__ void store(int s, const float (&f)[V]) const {
    if constexpr (BUF) {
      if constexpr (BF) {
        Half<V> m;
        m.put(f);
        __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u2, m), buf, off + s * step, 0, 0);
      } else {
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u4, f), buf, off + s * step, 0, 0);
      }
    } else if (t0 + s <= end) {
      Piece<BF, V>::store(base + (t0 + s) * ls, 0, f);
    }
  }
};

// The ids of the thread's S tokens and of the one before them, and at which of the S a sequence starts; the id before the first token is 0
template <int S>
struct Ids {
  int id[S + 1];
  __device__ __forceinline__ void load(const GScanP& p, int b, int t0) {
    const int* ids = p.ids + b * p.ids_b;
#pragma unroll
    for (int s = 0; s <= S; ++s) id[s] = ids[(long)min(max(t0 + s - 1, 0), p.L - 1) * p.ids_l];
  }
  __device__ __forceinline__ unsigned cuts(int t0) const {
    unsigned m = (t0 ? id[0] : 0) != id[1] ? 1u : 0u;
#pragma unroll
    for (int s = 1; s < S; ++s) m |= id[s + 1] != id[s] ? 1u << s : 0u;
    return m;
  }
};
// What is done at each token, APART: for a wave without a cut among its tokens as in rows that are not packed
template <bool SEQ, bool APART, class F>
__device__ __forceinline__ void with_cuts(unsigned cut, F f) {
  if (SEQ && (!APART || __any(cut != 0))) f([&](int s) { return (cut >> s & 1) != 0; });
  else f([](int) { return false; });
}

// The maps of a tile's segments, as the threads leave them, a channel a lane.  P < 0 marks a segment with a cut: nothing passes through it.
// Returns the tile's own map.
template <bool SEQ, int TT, int W>
__device__ __forceinline__ void tile_map(const float (&sP)[TT][W], const float (&sH)[TT][W], int w, bool back, float& P, float& H) {
  P = 1.0f;
  H = 0.0f;
#pragma unroll 8
  for (int i = 0; i < TT; ++i) {
    const int j = back ? TT - 1 - i : i;
    const float q = sP[j][w], f = sH[j][w];
    const bool cut = SEQ && q < 0.0f;
    H = cut ? f : fmaf(q, H, f);
    P = cut || (SEQ && P < 0.0f) ? -1.0f : P * q;
  }
}
// What every segment starts from, in place of its H; returns the state behind them.  ZEROS: a state of 0 stays 0, whatever a segment multiplies it by.
template <bool SEQ, bool ZEROS, int TT, int W>
__device__ __forceinline__ float tile_starts(const float (&sP)[TT][W], float (&sH)[TT][W], int w, bool back, float h) {
#pragma unroll 8
  for (int i = 0; i < TT; ++i) {
    const int j = back ? TT - 1 - i : i;
    const float q = sP[j][w], f = sH[j][w];
    sH[j][w] = h;
    h = (SEQ && q < 0.0f) || (ZEROS && h == 0.0f) ? f : fmaf(q, h, f);
  }
  return h;
}
// Whether a tile's map is one in numbers.  Without beta decays may grow (A > 0): a product beyond fp32 would make a state of 0 NaN and small ones infinite.
// The state behind such a tile is its segments', one behind the other, and the tiles behind it wait for that state.
__device__ __forceinline__ bool in_range(float P, float H) { return __builtin_isfinite(P) && __builtin_isfinite(H); }

template <int TT, int W>
__device__ __forceinline__ void column_sum(const float (&s)[TT][W], int w, float* to) {
  float sum = 0.0f;
#pragma unroll 8
  for (int j = 0; j < TT; ++j) sum += s[j][w];
  *to = sum;
}
// A thread's rows of A; whether no decay of the wave's leaves the series
template <int V>
__device__ __forceinline__ bool decays(const float* from, float (&A)[V]) {
  bool near = true;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    A[v] = from[v];
    near = near && fabsf(A[v]) < GS_NEAR;
  }
  return __all(near);
}

// The state in front of the o-th tile of a row (in the order of the walk), a channel a lane, from what the tiles in front of it have told:
// the nearest state among the last GS_LOOK of them, and the maps from there on, in the order in which the tiles themselves apply
// them -- whichever of the states is found, the bits are the same.  (A tile out of range tells no map: its state is waited for.)
// Every wait ends: tiles are taken in their order (tickets), so the tiles in front of this one are on workgroups that run, and the first of them
// that has not told its state waits for none that has not.  (After GS_POLLS looks, seconds, it would end with NaN: should memory be overwritten
// from elsewhere, no workgroup stays.)
constexpr int GS_POLLS = 1 << 22;
struct Look {
  unsigned H[GS_LOOK], P[GS_LOOK];
  __device__ __forceinline__ void ask(const unsigned long long* at) {   // at: the lane's word of the tile
#pragma unroll
    for (int i = 0; i < GS_LOOK; ++i) {   // (in front of a row's first tile lie GS_LOOK that tell nothing)
      const unsigned long long w = __hip_atomic_load(at - 64 * (i + 1), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      P[i] = (unsigned)(w >> 32);
      H[i] = (unsigned)w;
    }
  }
  // (the first look asked for before)
  __device__ __forceinline__ float back(const unsigned long long* at, int o, float first) {
    int n = GS_LOOK;
    for (int polls = 0;;) {
      n = GS_LOOK;
      bool told = true;
#pragma unroll
      for (int i = 0; i < GS_LOOK; ++i) {   // i == o: the state that the row starts from
        if (told && n == GS_LOOK && (i == o || P[i] == GS_STATE)) n = i;
        told = told && P[i] != GS_NOTHING;
      }
      if (__all(n < GS_LOOK) || ++polls == GS_POLLS) break;
      __builtin_amdgcn_s_sleep(1);
      ask(at);
    }
    float h = __builtin_nanf("");
#pragma unroll
    for (int i = GS_LOOK - 1; i >= 0; --i) {
      const float f = __uint_as_float(H[i]);
      h = i == n ? (i == o ? first : f) : i < n ? fmaf(__uint_as_float(P[i]), h, f) : h;
    }
    return h;
  }
};
// (its answer is one less than the ticket: the counter starts with all bits set)
__device__ __forceinline__ int ticket(unsigned* counter) {
  return (int)__hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__global__ __launch_bounds__(256) void k_gscan_clear(uint4* p, long n) {
  for (long i = blockIdx.x * 256L + threadIdx.x; i < n; i += gridDim.x * 256L) p[i] = make_uint4(~0u, ~0u, ~0u, ~0u);
}

// The row of a block of channels that a workgroup is of.  Where blocks of channels share cache lines (p.lines), an XCD's workgroups (every eighth one) take
// rows that lie side by side, so that such a line is in one L2: 8 x 4096 x 1000 bf16 67 us forward and 145 backward, 83 and 169 without; 64 x 1024 x 1000
// 126 and 228, 145 and 310; 4 x 5001 x 801 fp32, packed, 58 and 143, 67 and 155.  Where there are no such lines the other order is as fast or faster
// (8 x 4096 x 2048 136 and 254, 136 and 254 side by side; 1 x 131072 x 2048 526 and 1126, 544 and 1165), and where a workgroup has hardly more than a tile:
// XCDs do not get the same number of rows (3 x 3000 x 333 fp32 22 and 35, 22 and 38; 2 x 1000 x 290 11 and 16, 12 and 19).
template <bool SHARED>
__device__ __forceinline__ int chain_of(const GScanP& p) {
  const unsigned rows = p.B * p.ncb, each = gridDim.x >> 3, xcd = blockIdx.x & 7, nth = blockIdx.x >> 3;
  if (!p.lines) return SHARED ? blockIdx.x % rows : blockIdx.x;
  if (!SHARED || gridDim.x == rows) return xcd * each + min(xcd, gridDim.x & 7) + nth;
  // (its rows in turn, the first and last of which may be another XCD's too; none is left out: rows that share their tiles so have GS_WG * NCU workgroups
  // or more, an XCD more of them than rows)
  const unsigned first = (xcd * rows) >> 3, mine = (((xcd + 1) * rows + 7) >> 3) - first;
  return first + nth % mine;
}

// A row of a block of channels is one workgroup's, tile behind tile, or (SHARED) that of several: each takes the next tile that none has taken.
// One barrier a tile.  From a tile's barrier to the next one's the maps' wave has its maps, looks for the state in front of it and gives the
// threads theirs; meanwhile the others ask for the inputs of the tile behind it, finish the one before it, whose states lie there, and leave
// the maps of the one behind it.  So a state in front of a tile may be late by all of that before it costs time.
template <int W>
struct Maps {
  float P[GS_TT][W], H[GS_TT][W];
};
template <int W>
struct FwdShared {
  Maps<W> maps[2];   // of two tiles in turn
  int turn[2];       // the tile behind them
};
// Forward, the maps' wave
template <int V, int S, bool SEQ, bool SHARED, int W>
__device__ __forceinline__ void chain_fwd(const GScanP& p, FwdShared<W>& sh, int chain, int cb, int b, int k) {
  const int w = threadIdx.x & 63, mine = slot_channel<V>(cb * W, w, p.C);
  const bool on = W == 64 || w < W;
  unsigned long long* words = p.words + ((long)chain * (p.nk + GS_LOOK) + GS_LOOK) * 64 + w;
  unsigned* counter = p.tickets + (long)chain * GS_TICKET;
  const float first = on && p.h0 ? p.h0[(long)b * p.C + mine] : 0.0f;
  float carry = first;
  __builtin_amdgcn_s_setprio(3);
  for (int n = 0; k < p.nk; n ^= 1) {
    int next = k + 1;
    if (SHARED) {
      if (w == 0) sh.turn[n] = ticket(counter) + 1;
      next = __builtin_amdgcn_readfirstlane(sh.turn[n]);
    }
    Look look;
    if (SHARED && k > 0) look.ask(words + (long)k * 64);
    __syncthreads();
    Maps<W>& m = sh.maps[n];
    if (on) {
      float Pt, Ht;
      tile_map<SEQ, GS_TT, W>(m.P, m.H, w, false, Pt, Ht);
      const bool cut_off = SEQ && Pt < 0.0f, whole = in_range(Pt, Ht);
      if (SHARED && k > 0) {
        if (whole) tell(words + (long)k * 64, Ht, cut_off ? GS_STATE : __float_as_uint(Pt));
        carry = look.back(words + (long)k * 64, k, first);
      }
      float behind = cut_off ? Ht : fmaf(Pt, carry, Ht);
      if (SHARED && k + 1 < p.nk && whole) tell(words + (long)k * 64, behind, GS_STATE);
      const float walked = __any(!whole) ? tile_starts<SEQ, true, GS_TT, W>(m.P, m.H, w, false, carry) : tile_starts<SEQ, false, GS_TT, W>(m.P, m.H, w, false, carry);
      if (!whole) {
        behind = walked;
        if (SHARED && k + 1 < p.nk) tell(words + (long)k * 64, behind, GS_STATE);
      }
      if (p.hs)
#pragma unroll
        for (int i = 0; i < S / GS_S_BACK; ++i) {
          const int t = k * (S / GS_S_BACK) + i;
          if (t < p.nb) p.hs[((long)b * p.nb + t) * p.C + mine] = m.H[i * (GS_TT * GS_S_BACK / S)][w];
        }
      carry = behind;
    }
    k = next;
  }
  __syncthreads();
}
// IG, NRM: whether there is an in_gate, a beta; 2: asked when run.
template <bool BF, int V, int S, int IG, int NRM, bool SEQ, bool SHARED, bool BUF>
__global__ __launch_bounds__(GS_THREADS, BF ? 4 : 2) void k_gscan_fwd(GScanP p) {
  constexpr int W = GS_CG * V, T = GS_TT * S;
  __shared__ FwdShared<W> sh;
  const int chain = chain_of<SHARED>(p), cb = chain % p.ncb, b = chain / p.ncb;
  const int tid = threadIdx.x, cg = tid % GS_CG, tt = tid / GS_CG, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int k = 0;
  if (SHARED) {
    if (tid == 0) sh.turn[1] = ticket(p.tickets + (long)chain * GS_TICKET) + 1;
    __syncthreads();
    k = __builtin_amdgcn_readfirstlane(sh.turn[1]);   // (turn[1] is written again behind the first tile's barrier)
  }
  if (wave == GS_THREADS / 64 - 1) return chain_fwd<V, S, SEQ, SHARED, W>(p, sh, chain, cb, b, k);
  const bool ig = IG == 2 ? p.i != nullptr : IG == 1, nrm = NRM == 2 ? p.nrm : NRM == 1;
  const int c0 = first_channel<V>(cb * W + cg * V, p.C);
  Piece<BF, V> x[S], g[S], in[S];
  auto request = [&](int k) {
    const int t0 = k * T + tt * S;
    Rows<BF, V, S, BUF>(p.x, p.xb, p.xl, b, k, p.L, p.C, t0, c0).load(x);
    Rows<BF, V, S, BUF>(p.g, p.gb, p.gl, b, k, p.L, p.C, t0, c0).load(g);
    if (ig) Rows<BF, V, S, BUF>(p.i, p.ib, p.il, b, k, p.L, p.C, t0, c0).load(in);
  };
  float A[V];
  const bool all_near = decays<V>(p.A + c0, A);
  struct Tile {   // of a tile whose states are looked for
    float a[S][V], f[S][V];
    unsigned cut;
    int k;
  };
  auto begin = [&](Tile& q, int k, Maps<W>& m) {
    const int t0 = k * T + tt * S;
    q.k = k;
    Ids<S> ids;
    if (SEQ) ids.load(p, b, t0);
    auto gates = [&](auto near) {
#pragma unroll
      for (int s = 0; s < S; ++s) {
        if (V > 1) {
          x[s].template apart<near.value>();
          g[s].template apart<near.value>();
          if (ig) in[s].template apart<near.value>();
        }
#pragma unroll
        for (int v = 0; v < V; ++v) {
          float u = x[s][v], beta;
          if (ig) u *= sigmoid(in[s][v]);
          decay<near.value>(A[v] * sigmoid(g[s][v]), nrm, q.a[s][v], beta);
          q.f[s][v] = nrm ? beta * u : u;
        }
        __builtin_amdgcn_sched_barrier(0);   // (a token's values at a time are enough to fill the pipeline, and all at once cost registers)
      }
    };
    if (all_near) gates(std::true_type());
    else gates(std::false_type());
    if ((k + 1) * T > p.L) {   // behind the end: the identity
#pragma unroll
      for (int s = 0; s < S; ++s)
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const bool there = t0 + s < p.L;
          q.a[s][v] = there ? q.a[s][v] : 1.0f;
          q.f[s][v] = there ? q.f[s][v] : 0.0f;
        }
    }
    q.cut = SEQ ? ids.cuts(t0) : 0u;
    with_cuts<SEQ, true>(q.cut, [&](auto cut) {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float P = 1.0f, H = 0.0f;
#pragma unroll
        for (int s = 0; s < S; ++s) {
          H = cut(s) ? q.f[s][v] : fmaf(q.a[s][v], H, q.f[s][v]);
          P *= q.a[s][v];
        }
        m.P[tt][cg * V + v] = SEQ && q.cut ? -1.0f : P;
        m.H[tt][cg * V + v] = H;
      }
    });
  };
  auto finish = [&](const Tile& q, const Maps<W>& m) {
    const int t0 = q.k * T + tt * S;
    float h[V];
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = m.H[tt][cg * V + v];
    const Rows<BF, V, S, BUF> y(p.y, p.yb, p.yl, b, q.k, p.L, p.C, t0, c0);
    with_cuts<SEQ, true>(q.cut, [&](auto cut) {
#pragma unroll
      for (int s = 0; s < S; ++s) {
#pragma unroll
        for (int v = 0; v < V; ++v) h[v] = cut(s) ? q.f[s][v] : fmaf(q.a[s][v], h[v], q.f[s][v]);
        y.store(s, h);
        if (t0 + s == p.L - 1 && p.last) Piece<false, V>::store(p.last, (long)b * p.C + c0, h);
      }
    });
  };
  Tile one, two;
  one.k = two.k = -1;
  if (k < p.nk) request(k);
  // (a thread reads and writes no slots of the maps but its own: those of the tile that it finishes take the next one's)
  while (k < p.nk) {
    begin(one, k, sh.maps[0]);
    __syncthreads();
    k = SHARED ? __builtin_amdgcn_readfirstlane(sh.turn[0]) : k + 1;
    if (k < p.nk) request(k);
    if (two.k >= 0) finish(two, sh.maps[1]);
    two.k = -1;
    if (k >= p.nk) break;
    begin(two, k, sh.maps[1]);
    __syncthreads();
    k = SHARED ? __builtin_amdgcn_readfirstlane(sh.turn[1]) : k + 1;
    if (k < p.nk) request(k);
    finish(one, sh.maps[0]);
    one.k = -1;
  }
  __syncthreads();
  if (one.k >= 0) finish(one, sh.maps[0]);
  if (two.k >= 0) finish(two, sh.maps[1]);
}

// Backwards the tiles' order o is from the last to the first.  The maps' wave: c, what the tokens behind a tile give to its last state, and h
// (two barriers a tile: what the threads keep of a tile is too much to keep two of, and three workgroups a CU stand in for each other)
template <int W>
struct BackMaps : Maps<W> {
  int turn;
  float C[GS_TT][W];
  float dA[2][GS_TT][W];   // what the threads give to dA, of two tiles in turn
};
template <int V, int S, bool SEQ, bool SHARED, int W>
__device__ __forceinline__ void chain_bwd(const GScanP& p, BackMaps<W>& m, int chain, int cb, int b, int o) {
  const int w = threadIdx.x & 63, mine = slot_channel<V>(cb * W, w, p.C);
  const bool on = W == 64 || w < W;
  unsigned long long* words = p.words + ((long)chain * (p.nk + GS_LOOK) + GS_LOOK) * 64 + w;
  unsigned* counter = p.tickets + (long)chain * GS_TICKET;
  const float first = on && p.dlast ? p.dlast[(long)b * p.C + mine] : 0.0f;
  float carry = first;
  int past = -1, n = 0;   // the tile before this one, how many tiles
  // a tile's sum to a row of its own: which workgroup took it is chance
  auto sum_up = [&] {
    if (SHARED && p.part && on && past >= 0) column_sum(m.dA[(n & 1) ^ 1], w, p.part + ((long)b * p.nk + p.nk - 1 - past) * p.C + mine);
  };
  __builtin_amdgcn_s_setprio(3);
  while (o < p.nk) {
    int next = o;
    if (SHARED && w == 0) next = ticket(counter);
    const float before = on ? p.hs[((long)b * p.nk + p.nk - 1 - o) * p.C + mine] : 0.0f;
    Look look;
    if (SHARED && o > 0) look.ask(words + (long)o * 64);
    if (SHARED && w == 0) m.turn = next + 1;
    __syncthreads();
    next = SHARED ? __builtin_amdgcn_readfirstlane(m.turn) : o + 1;
    if (on) {
      float Pt, Ct;
      tile_map<SEQ, GS_TT, W>(m.P, m.C, w, true, Pt, Ct);
      const bool cut_off = SEQ && Pt < 0.0f, whole = in_range(Pt, Ct);
      if (SHARED && o > 0) {
        if (whole) tell(words + (long)o * 64, Ct, cut_off ? GS_STATE : __float_as_uint(Pt));
        carry = look.back(words + (long)o * 64, o, first);
      }
      float behind = cut_off ? Ct : fmaf(Pt, carry, Ct);
      if (SHARED && o + 1 < p.nk && whole) tell(words + (long)o * 64, behind, GS_STATE);
      const bool zeros = __any(!whole);
      const float walked = zeros ? tile_starts<SEQ, true, GS_TT, W>(m.P, m.C, w, true, carry) : tile_starts<SEQ, false, GS_TT, W>(m.P, m.C, w, true, carry);
      if (!whole) {
        behind = walked;
        if (SHARED && o + 1 < p.nk) tell(words + (long)o * 64, behind, GS_STATE);
      }
      if (zeros) tile_starts<SEQ, true, GS_TT, W>(m.P, m.H, w, false, before);
      else tile_starts<SEQ, false, GS_TT, W>(m.P, m.H, w, false, before);
      carry = behind;
    }
    __syncthreads();
    sum_up();
    past = o;
    ++n;
    o = next;
  }
  __syncthreads();
  sum_up();
}
template <bool BF, int V, int S, int IG, int NRM, bool SEQ, bool SHARED, bool BUF>
__global__ __launch_bounds__(GS_THREADS, BF && SHARED ? 6 : 2) void k_gscan_bwd(GScanP p) {
  constexpr int W = GS_CG * V, T = GS_TT * S;
  __shared__ BackMaps<W> m;
  const int chain = chain_of<SHARED>(p), cb = chain % p.ncb, b = chain / p.ncb;
  const int tid = threadIdx.x, cg = tid % GS_CG, tt = tid / GS_CG, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int k0 = 0;
  if (SHARED) {
    if (tid == 0) m.turn = ticket(p.tickets + (long)chain * GS_TICKET) + 1;
    __syncthreads();
    k0 = __builtin_amdgcn_readfirstlane(m.turn);
    __syncthreads();
  }
  float dA[V];
#pragma unroll
  for (int v = 0; v < V; ++v) dA[v] = 0.0f;
  const int c0 = first_channel<V>(cb * W + cg * V, p.C);
  if (wave == GS_THREADS / 64 - 1) {
    chain_bwd<V, S, SEQ, SHARED, W>(p, m, chain, cb, b, k0);
  } else {
    const bool ig = IG == 2 ? p.i != nullptr : IG == 1, nrm = NRM == 2 ? p.nrm : NRM == 1;
    float A[V];
    const bool all_near = decays<V>(p.A + c0, A);
    int o = k0, n = 0;
    while (o < p.nk) {
      const int k = p.nk - 1 - o, t0 = k * T + tt * S;
      Piece<BF, V> x[S], g[S], in[S], dy[S];
      Rows<BF, V, S, BUF>(p.x, p.xb, p.xl, b, k, p.L, p.C, t0, c0).load(x);
      Rows<BF, V, S, BUF>(p.g, p.gb, p.gl, b, k, p.L, p.C, t0, c0).load(g);
      if (ig) Rows<BF, V, S, BUF>(p.i, p.ib, p.il, b, k, p.L, p.C, t0, c0).load(in);
      if (p.dy) {
        Rows<BF, V, S, BUF>(p.dy, p.dyb, p.dyl, b, k, p.L, p.C, t0, c0).load(dy);
      } else {
#pragma unroll
        for (int s = 0; s < S; ++s) dy[s].keep(false);
      }
      Ids<S> ids;
      if (SEQ) ids.load(p, b, t0);
      float a[S][V], r[S][V], beta[S][V], sg[S][V];
      auto gates = [&](auto near) {
#pragma unroll
        for (int s = 0; s < S; ++s) {
          if (V > 1) {
            g[s].template apart<near.value>();
            if (ig) in[s].template apart<near.value>();
          }
#pragma unroll
          for (int v = 0; v < V; ++v) {
            sg[s][v] = ig ? sigmoid(in[s][v]) : 1.0f;
            r[s][v] = sigmoid(g[s][v]);
            decay<near.value>(A[v] * r[s][v], nrm, a[s][v], beta[s][v]);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      };
      if (all_near) gates(std::true_type());
      else gates(std::false_type());
      if ((k + 1) * T > p.L) {   // behind the end: the identity, and nothing to any sum
#pragma unroll
        for (int s = 0; s < S; ++s) {
          const bool there = t0 + s < p.L;
          x[s].keep(there);
          dy[s].keep(there);
#pragma unroll
          for (int v = 0; v < V; ++v) {
            a[s][v] = there ? a[s][v] : 1.0f;
            r[s][v] = there ? r[s][v] : 0.0f;
            sg[s][v] = there ? sg[s][v] : 0.0f;
            beta[s][v] = there ? beta[s][v] : 0.0f;
          }
        }
      }
      auto fed = [&](int s, int v) {   // the forward's beta u, rounded as there
        const float u = ig ? x[s][v] * sg[s][v] : x[s][v];
        return nrm ? beta[s][v] * u : u;
      };
      const unsigned cuts = SEQ ? ids.cuts(t0) : 0u;
      with_cuts<SEQ, !(BF && SHARED)>(cuts, [&](auto cut) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
          float P = 1.0f, H = 0.0f, C = 0.0f;
#pragma unroll
          for (int s = 0; s < S; ++s) {
            H = cut(s) ? fed(s, v) : fmaf(a[s][v], H, fed(s, v));
            P *= a[s][v];
          }
#pragma unroll
          for (int s = S - 1; s >= 0; --s) C = cut(s) ? 0.0f : a[s][v] * (dy[s][v] + C);
          m.P[tt][cg * V + v] = SEQ && cuts ? -1.0f : P;
          m.H[tt][cg * V + v] = H;
          m.C[tt][cg * V + v] = C;
        }
      });
      __syncthreads();
      const int next = SHARED ? __builtin_amdgcn_readfirstlane(m.turn) : o + 1;
      __syncthreads();
      // (from here to the next barrier a thread reads and writes no slots of the maps but its own)
      float h[V], c[V], before[S][V], sum[V];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        h[v] = m.H[tt][cg * V + v];
        c[v] = m.C[tt][cg * V + v];
        sum[v] = 0.0f;
      }
      with_cuts<SEQ, !(BF && SHARED)>(cuts, [&](auto cut) {
#pragma unroll
      for (int s = 0; s < S; ++s)
#pragma unroll
        for (int v = 0; v < V; ++v) {
          before[s][v] = cut(s) ? 0.0f : h[v];
          h[v] = cut(s) ? fed(s, v) : fmaf(a[s][v], h[v], fed(s, v));
        }
      const Rows<BF, V, S, BUF> to_x(p.dx, p.yb, p.yl, b, k, p.L, p.C, t0, c0), to_g(p.dg, p.yb, p.yl, b, k, p.L, p.C, t0, c0),
          to_i(p.di, p.yb, p.yl, b, k, p.L, p.C, t0, c0);
#pragma unroll
      for (int s = S - 1; s >= 0; --s) {
        float dx[V], dg[V], di[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float G = dy[s][v] + c[v], l = A[v] * r[s][v], xv = x[s][v];
          c[v] = cut(s) ? 0.0f : a[s][v] * G;
          float dl = c[v] * before[s][v], du = G;
          if (nrm) {
            const float bt = beta[s][v];   // (0 where nothing decays: its part is left out)
            dl = fmaf(-(G * (xv * sg[s][v])) * (a[s][v] * a[s][v]), bt == 0.0f ? 0.0f : __builtin_amdgcn_rcpf(bt), dl);
            du *= bt;
          }
          dx[v] = du * sg[s][v];
          di[v] = dx[v] * xv * (1.0f - sg[s][v]);
          dg[v] = dl * l * (1.0f - r[s][v]);
          // (an empty gate, as behind the end, gives nothing to any sum: the state may be infinite there, or a last state's gradient)
          sum[v] = r[s][v] == 0.0f ? sum[v] : fmaf(dl, r[s][v], sum[v]);
        }
        if (p.dx) to_x.store(s, dx);
        if (p.dg) to_g.store(s, dg);
        if (ig && p.di) to_i.store(s, di);
        if (t0 + s == 0 && p.dh0) Piece<false, V>::store(p.dh0, (long)b * p.C + c0, c);
      }
      });
#pragma unroll
      for (int v = 0; v < V; ++v) {
        if (SHARED) m.dA[n & 1][tt][cg * V + v] = sum[v];
        else dA[v] += sum[v];
      }
      ++n;
      o = next;
    }
    if (!SHARED)
#pragma unroll
      for (int v = 0; v < V; ++v) m.dA[0][tt][cg * V + v] = dA[v];
    __syncthreads();
  }
  if (!SHARED && p.part && tid < W) column_sum(m.dA[0], tid, p.part + (long)b * p.C + slot_channel<V>(cb * W, tid, p.C));
}

// dA: the sums of `rows` partial rows, in an order that their number alone decides: 16 channels and 64 strands of rows a workgroup
__global__ __launch_bounds__(1024) void k_gscan_sum(const float* part, int rows, int C, float* out) {
  __shared__ float s[64][17];
  const int c = threadIdx.x & 15, strand = threadIdx.x >> 4, d = blockIdx.x * 16 + c;
  s[strand][c] = strand_sum(part + min(d, C - 1), C, strand, rows);
  __syncthreads();
  if (strand || d >= C) return;
  float sum = 0.0f;
#pragma unroll 16
  for (int i = 0; i < 64; ++i) sum += s[i][c];
  out[d] = sum;
}

// One token a row, four channels a thread.  Rows whose slot is none of the pool's give zeros and touch no state.  Several rows of one slot are
// taken in their order, by the first of them: a workgroup looks over all rows' slots, each of its waves over a quarter of them.
// Bound by its bytes where rows are many (512 rows of 4096 channels bf16, 33.6 MB, 7.8 us, 9.2 with their slots
// named; 10.0 with every wave looking at all of them), by a launch and two trips to memory where they are few (one row of 2048 2.5 us).
template <bool BF>
struct Four {   // the channels that there are of four
  Piece<BF, 4> m;
  __device__ __forceinline__ void load(const void* q, long off, int n) {
    if (n >= 4) return m.load(q, off);
    float f[4];
#pragma unroll
    for (int v = 0; v < 4; ++v) f[v] = v < n ? ldv(q, off + v, BF) : 0.0f;
    m.m.put(f);
  }
  static __device__ __forceinline__ void store(void* q, long off, int n, const float (&f)[4]) {
    if (n >= 4) return Piece<BF, 4>::store(q, off, f);
#pragma unroll
    for (int v = 0; v < 4; ++v)
      if (v < n) stv(q, off + v, BF, f[v]);
  }
};
template <bool BF, bool IG, bool NRM>
__global__ __launch_bounds__(256) void k_gscan_step(GStepP p) {
  const int lane = threadIdx.x & 63, row = blockIdx.x / p.ncb;
  const int c0 = (blockIdx.x % p.ncb * 256 + threadIdx.x) * 4, n = min(4, p.C - c0);   // (n <= 0: no channel, but a look at the slots)
  auto slot_of = [&](int r) { return p.at64 ? ((const long*)p.at)[r] : (long)((const int*)p.at)[r]; };
  Four<BF> x, g, in;
  float A[4];
  auto request = [&](int r) {
    x.load(p.x, r * p.xs + c0, n);
    g.load(p.g, r * p.gs + c0, n);
    if (IG) in.load(p.i, r * p.is + c0, n);
  };
  request(row);
#pragma unroll
  for (int v = 0; v < 4; ++v) A[v] = v < n ? p.A[c0 + v] : 0.0f;
  const long slot = p.at ? slot_of(row) : row;
  const float none[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (slot < 0 || slot >= p.slots) return Four<BF>::store(p.y, (long)row * p.C + c0, n, none);
  float* state = p.state + slot * p.state_s;
  Four<false> old;
  old.load(state, c0, n);
  int next = p.rows;   // the next row of the slot
  if (p.at) {
    __shared__ int first_of[4], next_of[4];
    const int wave = threadIdx.x >> 6;
    int first = p.rows;
    for (int q = 64 * wave; q < p.rows; q += 512) {
      long s[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) s[i] = slot_of(min(q + 256 * i + lane, p.rows - 1));
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = q + 256 * i + lane;
        const bool same = r < p.rows && s[i] == slot;
        first = same ? min(first, r) : first;
        next = same && r > row ? min(next, r) : next;
      }
    }
    if (__any(first < p.rows))
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) {
        first = min(first, __shfl_xor(first, o, 64));
        next = min(next, __shfl_xor(next, o, 64));
      }
    if (lane == 0) {
      first_of[wave] = first;
      next_of[wave] = next;
    }
    __syncthreads();
    if (min(min(first_of[0], first_of[1]), min(first_of[2], first_of[3])) < row) return;
    next = min(min(next_of[0], next_of[1]), min(next_of[2], next_of[3]));
  }
  float h[4];
#pragma unroll
  for (int v = 0; v < 4; ++v) h[v] = old.m[v];
  for (int r = row;;) {
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      float u = x.m[v], a, beta;
      if (IG) u *= sigmoid(in.m[v]);
      decay<false>(A[v] * sigmoid(g.m[v]), NRM, a, beta);
      h[v] = fmaf(a, h[v], NRM ? beta * u : u);
    }
    Four<BF>::store(p.y, (long)r * p.C + c0, n, h);
    if (next >= p.rows) break;
    r = next;
    request(r);
    next = p.rows;
    for (int q = r + 1; q < p.rows && next == p.rows; q += 64) {
      const unsigned long long hit = __ballot(q + lane < p.rows && slot_of(min(q + lane, p.rows - 1)) == slot);
      if (hit) next = q + __ffsll(hit) - 1;
    }
  }
  Four<false>::store(state, c0, n, h);
}

template <bool BF, int V, int IG, int NRM, bool SEQ, bool SHARED, bool BUF>
static void launch_one(const GScanP& p, bool back, int blocks, hipStream_t st) {
  if (back) k_gscan_bwd<BF, V, GS_S_BACK, IG, NRM, SEQ, SHARED, BUF><<<blocks, GS_THREADS, 0, st>>>(p);
  else k_gscan_fwd<BF, V, SHARED ? GS_S_SHARED : GS_S_WALKED, IG, NRM, SEQ, SHARED, BUF><<<blocks, GS_THREADS, 0, st>>>(p);
}
template <bool BF, int V, int IG, int NRM, bool SHARED, bool BUF>
static void launch_packed(const GScanP& p, bool back, int blocks, hipStream_t st) {
  p.ids ? launch_one<BF, V, IG, NRM, true, SHARED, BUF>(p, back, blocks, st) : launch_one<BF, V, IG, NRM, false, SHARED, BUF>(p, back, blocks, st);
}
template <bool BF, int V, int IG, int NRM, bool BUF>
static void launch_shared(const GScanP& p, bool back, int blocks, hipStream_t st) {
  p.words ? launch_packed<BF, V, IG, NRM, true, BUF>(p, back, blocks, st) : launch_packed<BF, V, IG, NRM, false, BUF>(p, back, blocks, st);
}
// Rows that buffers take: whole dwords, a tile's rows (and one more) within 2^31 bytes
static bool behind_buffers(const GScanP& p, bool bf, bool back) {
  if (p.C < 4) return false;
  const long most = (1L << 31) / (4 * (GS_TT * GS_S_SHARED + 1)), odd = bf ? 1 : 0;
  auto takes = [&](const void* q, long b, long l) { return !q || (((uintptr_t)q & 3) == 0 && !((b | l) & odd) && labs(l) < most); };
  return !(p.C & odd) && p.C < most && takes(p.x, p.xb, p.xl) && takes(p.g, p.gb, p.gl) && takes(p.i, p.ib, p.il) &&
         (back ? takes(p.dy, p.dyb, p.dyl) && takes(p.dx, 0, 0) && takes(p.dg, 0, 0) && takes(p.di, 0, 0) : takes(p.y, 0, 0));
}
template <bool BF>
static void launch_form(const GScanP& p, bool buffers, bool back, int blocks, hipStream_t st) {
  if (!buffers) {
    if (p.C >= 4) launch_shared<BF, 4, 2, 2, false>(p, back, blocks, st);
    else launch_shared<BF, 1, 2, 2, false>(p, back, blocks, st);
  } else if (p.i) {
    p.nrm ? launch_shared<BF, 4, 1, 1, true>(p, back, blocks, st) : launch_shared<BF, 4, 1, 0, true>(p, back, blocks, st);
  } else {
    p.nrm ? launch_shared<BF, 4, 0, 1, true>(p, back, blocks, st) : launch_shared<BF, 4, 0, 0, true>(p, back, blocks, st);
  }
}

// Workgroups that share a row of a block of channels, of `rows` in all: as many as it takes for GS_WG a CU, forward and backward; rows enough to fill
// the GPU twice are walked.  (As many as fit in bf16.  Of the fp32 forms one fits forward, for its registers, and of some two backward; the
// others start when those end, which costs nothing: with one and two a CU 8 x 4096 x 1024 fp32 takes 121 and 214 us for 120 and 212, 4 x 5001 x 801, packed,
// 60 and 143 for 58 and 145, 1 x 65536 x 1024 223 and 462 for 220 and 447.)
// us forward and backward, shared and walked: bf16, 8 x 4096 x 2048 (256 rows) 139 and 261, 173 and 339; 16 x 4096 x 2048 (512) 268 and 497, 248 and 422;
// 1 x 131072 x 2048 (32) 522 and 1121, 4583 and 9183; fp32, 8 x 4096 x 1024 (128) 120 and 212, 180 and 363.  Just above 512 rows, where some
// walk alone behind the others, two workgroups a row would be faster: 9 x 4096 x 3712 (522) 264 and 450, walked 333 and 668; 11 x 4096 x 4096 (704) 354 and
// 625, 376 and 736.
constexpr int GS_WG = 2, GS_WG_BACK = 3, GS_ROWS_WALKED = 2 * NCU;
static int sharing(int rows, int tiles, bool back) {
  return rows >= GS_ROWS_WALKED ? 1 : max(1, min(tiles, ((back ? GS_WG_BACK : GS_WG) * NCU + rows - 1) / rows));
}
// A call's tiles of a row, how many workgroups share it, and its workspace: partial sums of dA, a row for each tile where tiles are shared and for
// each row where it is walked, then (shared) the tickets and what the tiles tell, in whole 16 bytes each.  All of it goes by sizes alone.
struct GScanPlan {
  int share, nk;
  size_t part, tickets, words;
  GScanPlan(int B, int L, int C, bool back, bool dA) {
    const int ncb = gscan_blocks(C), rows = B * ncb, S = back ? GS_S_BACK : GS_S_SHARED;
    share = sharing(rows, gscan_tiles(L, S), back);
    nk = gscan_tiles(L, share > 1 || back ? S : GS_S_WALKED);
    part = dA ? ((size_t)B * (share > 1 ? nk : 1) * C * 4 + 255) & ~(size_t)255 : 0;
    tickets = share > 1 ? (size_t)rows * GS_TICKET * 4 : 0;
    words = share > 1 ? (size_t)rows * (nk + GS_LOOK) * 64 * 8 : 0;
  }
};
size_t gscan_workspace(int B, int L, int C, bool back, bool dA) {
  const GScanPlan plan(B, L, C, back, back && dA);
  return plan.part + plan.tickets + plan.words;
}

int launch_gscan(GScanP p, bool bf, bool back, void* workspace, hipStream_t st) {
  const GScanPlan plan(p.B, p.L, p.C, back, back && p.dA);
  const bool shared = plan.share > 1;
  p.ncb = gscan_blocks(p.C);
  p.nb = gscan_tiles(p.L, GS_S_BACK);
  p.nk = plan.nk;
  p.lines = (p.C * (bf ? 2L : 4L)) % 128 != 0 && (!shared || 2 * p.nk >= 3 * plan.share);
  char* ws = (char*)workspace;
  if (plan.part) p.part = (float*)ws;
  if (shared) {
    ws += plan.part;
    p.tickets = (unsigned*)ws;
    p.words = (unsigned long long*)(ws + plan.tickets);
    const long n = (long)((plan.tickets + plan.words) / 16);
    k_gscan_clear<<<(int)min((n + 1023) / 1024, 1024L), 256, 0, st>>>((uint4*)ws, n);
  }
  const int blocks = p.B * p.ncb * plan.share;
  bf ? launch_form<true>(p, behind_buffers(p, bf, back), back, blocks, st) : launch_form<false>(p, behind_buffers(p, bf, back), back, blocks, st);
  if (p.part) k_gscan_sum<<<(p.C + 15) / 16, 1024, 0, st>>>(p.part, shared ? p.B * p.nk : p.B, p.C, p.dA);
  return (int)hipGetLastError();
}

template <bool BF>
static void launch_step(const GStepP& p, bool nrm, hipStream_t st) {
  const unsigned grid = (unsigned)p.rows * p.ncb;
  if (p.i) nrm ? k_gscan_step<BF, true, true><<<grid, 256, 0, st>>>(p) : k_gscan_step<BF, true, false><<<grid, 256, 0, st>>>(p);
  else nrm ? k_gscan_step<BF, false, true><<<grid, 256, 0, st>>>(p) : k_gscan_step<BF, false, false><<<grid, 256, 0, st>>>(p);
}
// Rows with slots go in launches of at most GS_STEP_ROWS, one behind the other: a row looks at its launch's slots only, so that the looking grows with
// the rows and not with their square, and a slot's rows stay in their order.  (8192 rows bf16 of 4096 channels by 1024, 2048, 4096, 8192: 169, 162,
// 174, 217 us; of 256: 43, 34, 36, 44.)
constexpr int GS_STEP_ROWS = 2048;
int launch_gscan_step(GStepP p, bool bf, bool nrm, hipStream_t st) {
  p.ncb = (p.C + 1023) / 1024;
  const int rows = p.rows, most = p.at ? GS_STEP_ROWS : rows;
  const long size = bf ? 2 : 4, index = p.at64 ? 8 : 4;
  auto on = [](auto*& q, long bytes) { q = q ? (std::remove_reference_t<decltype(q)>)((const char*)q + bytes) : q; };
  for (int r = 0; r < rows; r += most) {
    p.rows = min(most, rows - r);
    bf ? launch_step<true>(p, nrm, st) : launch_step<false>(p, nrm, st);
    on(p.x, most * p.xs * size);
    on(p.g, most * p.gs * size);
    on(p.i, most * p.is * size);
    on(p.at, most * index);
    on(p.y, (long)most * p.C * size);
  }
  return (int)hipGetLastError();
}

}  // namespace issm
