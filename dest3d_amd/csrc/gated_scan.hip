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
// A workgroup takes tiles of TT * S tokens and CG * V channels: a thread V channels of S tokens one behind the other, whose map
// h -> P h + H it leaves in LDS; the first wave, a channel a lane, joins the TT maps of the tile and gives every thread its first state.
#include "gated_scan_dev.h"

// (every multiply-add is written as one: the forms of a kernel that do the same sums are to give the same bits)
#pragma clang fp contract(off)

namespace issm {

// A tile's inputs of one thread: S tokens, V channels each
template <bool BF, int V, int S>
struct Raw {
  Piece<BF, V> v[S];
  __device__ __forceinline__ void load(const void* base, long bs, long ls, int b, int t0, int c0, int last) {
#pragma unroll
    for (int s = 0; s < S; ++s) v[s].load(base, b * bs + (long)min(t0 + s, last) * ls + c0);   // (behind the end: the last token again)
  }
};

// Which of the thread's S tokens a sequence starts at; the id before the first token is 0
template <int S>
__device__ __forceinline__ unsigned cuts(const GScanP& p, int b, int t0) {
  const int* ids = p.ids + b * p.ids_b;
  int id[S + 1];
#pragma unroll
  for (int s = 0; s <= S; ++s) {
    const int t = t0 + s - 1;
    id[s] = t < 0 ? 0 : ids[(long)min(t, p.L - 1) * p.ids_l];
  }
  unsigned m = 0;
#pragma unroll
  for (int s = 0; s < S; ++s) m |= id[s + 1] != id[s] ? 1u << s : 0u;
  return m;
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
template <bool SEQ, int TT, int W>
__device__ __forceinline__ void tile_starts(const float (&sP)[TT][W], float (&sH)[TT][W], int w, bool back, float h) {
#pragma unroll 8
  for (int i = 0; i < TT; ++i) {
    const int j = back ? TT - 1 - i : i;
    const float q = sP[j][w], f = sH[j][w];
    sH[j][w] = h;
    h = SEQ && q < 0.0f ? f : fmaf(q, h, f);
  }
}

// The state in front of the o-th tile of a row (in the order of the walk), a channel a lane, from what the tiles in front of it have told:
// the nearest state among the last GS_LOOK of them, and the maps from there on, in the order in which the tiles themselves apply
// them -- whichever of the states is found, the bits are the same.
// Every wait ends: tiles are taken in their order (tickets), so the tiles in front of this one are on workgroups that run, and the first of them
// that has not told its state waits for none that has not.  (After GS_POLLS looks, seconds, it would end with NaN: should memory be overwritten
// from elsewhere, no workgroup stays.)
constexpr int GS_LOOK = 8, GS_POLLS = 1 << 22;
__device__ __forceinline__ float look_back(const unsigned long long* words, int o, float first, int lane) {
  float H[GS_LOOK], P[GS_LOOK];
  int n = GS_LOOK;
  for (int polls = 0; polls < GS_POLLS; ++polls) {
    unsigned long long w[GS_LOOK];
#pragma unroll
    for (int i = 0; i < GS_LOOK; ++i)
      w[i] = __hip_atomic_load(words + (long)max(o - 1 - i, 0) * 64 + lane, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    n = GS_LOOK;
    bool told = true;
#pragma unroll
    for (int i = 0; i < GS_LOOK; ++i) {
      unsigned high = (unsigned)(w[i] >> 32);
      H[i] = __uint_as_float((unsigned)w[i]);
      if (o - 1 - i < 0) {   // in front of the first: the state that the row starts from
        high = GS_STATE;
        H[i] = first;
      }
      P[i] = __uint_as_float(high);
      if (told && n == GS_LOOK && high == GS_STATE) n = i;
      told = told && high != GS_NOTHING;
    }
    if (__all(n < GS_LOOK)) break;
    __builtin_amdgcn_s_sleep(2);
  }
  float h = __builtin_nanf("");
#pragma unroll
  for (int i = GS_LOOK - 1; i >= 0; --i) h = i == n ? H[i] : i < n ? fmaf(P[i], h, H[i]) : h;
  return h;
}
// The tile's ticket; one barrier
__device__ __forceinline__ int ticket(unsigned* counter, int* shared) {
  if (threadIdx.x == 0) *shared = (int)(__hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1u);
  __syncthreads();
  return *shared;
}
__global__ __launch_bounds__(256) void k_gscan_clear(uint4* p, long n) {
  for (long i = blockIdx.x * 256L + threadIdx.x; i < n; i += gridDim.x * 256L) p[i] = make_uint4(~0u, ~0u, ~0u, ~0u);
}

// LOOK: a tile a workgroup; else a row's tiles one behind the other on one
template <bool BF, int V, int S, bool IG, bool NRM, bool SEQ, bool LOOK>
__global__ __launch_bounds__(GS_THREADS) void k_gscan_fwd(GScanP p) {
  constexpr int TT = GS_TT, W = GS_CG * V, T = TT * S;
  __shared__ float sP[TT][W], sH[TT][W];
  const int tid = threadIdx.x, cg = tid % GS_CG, tt = tid / GS_CG;
  const int chain = LOOK ? blockIdx.x % (p.B * p.ncb) : blockIdx.x, cb = chain % p.ncb, b = chain / p.ncb;
  const int c0 = first_channel<V>(cb * W + cg * V, p.C), mine = slot_channel<V>(cb * W, tid, p.C);
  float A[V];
#pragma unroll
  for (int v = 0; v < V; ++v) A[v] = p.A[c0 + v];
  float carry = 0.0f;
  if (tid < W && p.h0) carry = p.h0[(long)b * p.C + mine];
  __shared__ int turn;
  const int k0 = LOOK ? ticket(p.tickets + (long)chain * GS_TICKET, &turn) : 0, k1 = LOOK ? k0 + 1 : p.nk;
  unsigned long long* words = p.words + (long)chain * p.nk * 64;
  for (int k = k0; k < k1; ++k) {
    const int t0 = k * T + tt * S;
    Raw<BF, V, S> x, g, in;
    x.load(p.x, p.xb, p.xl, b, t0, c0, p.L - 1);
    g.load(p.g, p.gb, p.gl, b, t0, c0, p.L - 1);
    if (IG) in.load(p.i, p.ib, p.il, b, t0, c0, p.L - 1);
    const unsigned cut = SEQ ? cuts<S>(p, b, t0) : 0u;
    float a[S][V], f[S][V], P[V], H[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      P[v] = 1.0f;
      H[v] = 0.0f;
    }
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float u = x.v[s][v];
        if (IG) u *= sigmoid(in.v[s][v]);
        float beta;
        decay<NRM>(A[v] * sigmoid(g.v[s][v]), a[s][v], beta);
        f[s][v] = NRM ? beta * u : u;
      }
    if (t0 + S > p.L) {   // behind the end: the identity
#pragma unroll
      for (int s = 0; s < S; ++s)
        if (t0 + s >= p.L)
#pragma unroll
          for (int v = 0; v < V; ++v) {
            a[s][v] = 1.0f;
            f[s][v] = 0.0f;
          }
    }
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const bool z = SEQ && (cut >> s & 1);
        H[v] = z ? f[s][v] : fmaf(a[s][v], H[v], f[s][v]);
        P[v] = z || (SEQ && P[v] < 0.0f) ? -1.0f : P[v] * a[s][v];
      }
#pragma unroll
    for (int v = 0; v < V; ++v) {
      sP[tt][cg * V + v] = P[v];
      sH[tt][cg * V + v] = H[v];
    }
    __syncthreads();
    if (tid < W) {
      float Pt, Ht;
      tile_map<SEQ, TT, W>(sP, sH, tid, false, Pt, Ht);
      if (LOOK && k > 0) {
        const bool cut_off = SEQ && Pt < 0.0f;
        tell(words + (long)k * 64 + tid, Ht, cut_off ? GS_STATE : map_bits(Pt));
        carry = look_back(words, k, carry, tid);
      }
      if (p.hs) p.hs[((long)b * p.nk + k) * p.C + mine] = carry;
      const float behind = SEQ && Pt < 0.0f ? Ht : fmaf(Pt, carry, Ht);
      if (LOOK && k + 1 < p.nk) tell(words + (long)k * 64 + tid, behind, GS_STATE);
      tile_starts<SEQ, TT, W>(sP, sH, tid, false, carry);
      carry = behind;
    }
    __syncthreads();
    float h[V];
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = sH[tt][cg * V + v];
#pragma unroll
    for (int s = 0; s < S; ++s) {
#pragma unroll
      for (int v = 0; v < V; ++v) h[v] = SEQ && (cut >> s & 1) ? f[s][v] : fmaf(a[s][v], h[v], f[s][v]);
      const int t = t0 + s;
      if (t < p.L) Piece<BF, V>::store(p.y, b * p.yb + t * p.yl + c0, h);
      if (t == p.L - 1 && p.last) Piece<false, V>::store(p.last, (long)b * p.C + c0, h);
    }
    if (!LOOK) __syncthreads();   // (the next tile's maps go where these states are read)
  }
}

template <bool BF, int V, int S, bool IG, bool NRM, bool SEQ, bool LOOK>
__global__ __launch_bounds__(GS_THREADS) void k_gscan_bwd(GScanP p) {
  constexpr int TT = GS_TT, W = GS_CG * V, T = TT * S;
  __shared__ float sP[TT][W], sH[TT][W], sC[TT][W];
  const int tid = threadIdx.x, cg = tid % GS_CG, tt = tid / GS_CG;
  const int chain = LOOK ? blockIdx.x % (p.B * p.ncb) : blockIdx.x, cb = chain % p.ncb, b = chain / p.ncb;
  const int c0 = first_channel<V>(cb * W + cg * V, p.C), mine = slot_channel<V>(cb * W, tid, p.C);
  float A[V], dA[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    A[v] = p.A[c0 + v];
    dA[v] = 0.0f;
  }
  float carry = 0.0f;   // what the tokens behind the tile give to its last state
  if (tid < W && p.dlast) carry = p.dlast[(long)b * p.C + mine];
  __shared__ int turn;
  const int o0 = LOOK ? ticket(p.tickets + (long)chain * GS_TICKET, &turn) : 0, o1 = LOOK ? o0 + 1 : p.nk;
  unsigned long long* words = p.words + (long)chain * p.nk * 64;
  for (int o = o0; o < o1; ++o) {   // from the last tile to the first
    const int k = p.nk - 1 - o;
    const int t0 = k * T + tt * S;
    Raw<BF, V, S> x, g, in, dy;
    x.load(p.x, p.xb, p.xl, b, t0, c0, p.L - 1);
    g.load(p.g, p.gb, p.gl, b, t0, c0, p.L - 1);
    if (IG) in.load(p.i, p.ib, p.il, b, t0, c0, p.L - 1);
    if (p.dy) dy.load(p.dy, p.dyb, p.dyl, b, t0, c0, p.L - 1);
    const unsigned cut = SEQ ? cuts<S>(p, b, t0) : 0u;
    float a[S][V], f[S][V], d[S][V], P[V], H[V], Cm[V];
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float u = x.v[s][v];
        if (IG) u *= sigmoid(in.v[s][v]);
        float beta;
        decay<NRM>(A[v] * sigmoid(g.v[s][v]), a[s][v], beta);
        f[s][v] = NRM ? beta * u : u;
        d[s][v] = p.dy ? dy.v[s][v] : 0.0f;
      }
    if (t0 + S > p.L) {
#pragma unroll
      for (int s = 0; s < S; ++s)
        if (t0 + s >= p.L)
#pragma unroll
          for (int v = 0; v < V; ++v) {
            a[s][v] = 1.0f;
            f[s][v] = d[s][v] = 0.0f;
          }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
      P[v] = 1.0f;
      H[v] = Cm[v] = 0.0f;
    }
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const bool z = SEQ && (cut >> s & 1);
        H[v] = z ? f[s][v] : fmaf(a[s][v], H[v], f[s][v]);
        P[v] = z || (SEQ && P[v] < 0.0f) ? -1.0f : P[v] * a[s][v];
      }
#pragma unroll
    for (int s = S - 1; s >= 0; --s)
#pragma unroll
      for (int v = 0; v < V; ++v) Cm[v] = SEQ && (cut >> s & 1) ? 0.0f : a[s][v] * (d[s][v] + Cm[v]);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      sP[tt][cg * V + v] = P[v];
      sH[tt][cg * V + v] = H[v];
      sC[tt][cg * V + v] = Cm[v];
    }
    __syncthreads();
    if (tid < W) {
      float Pt, Ct;
      const float before = p.hs[((long)b * p.nk + k) * p.C + mine];
      tile_map<SEQ, TT, W>(sP, sC, tid, true, Pt, Ct);
      if (LOOK && o > 0) {
        tell(words + (long)o * 64 + tid, Ct, SEQ && Pt < 0.0f ? GS_STATE : map_bits(Pt));
        carry = look_back(words, o, carry, tid);
      }
      const float behind = SEQ && Pt < 0.0f ? Ct : fmaf(Pt, carry, Ct);
      if (LOOK && o + 1 < p.nk) tell(words + (long)o * 64 + tid, behind, GS_STATE);
      tile_starts<SEQ, TT, W>(sP, sC, tid, true, carry);
      tile_starts<SEQ, TT, W>(sP, sH, tid, false, before);
      carry = behind;
    }
    __syncthreads();
    float h[V], c[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      h[v] = sH[tt][cg * V + v];
      c[v] = sC[tt][cg * V + v];
    }
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
      for (int v = 0; v < V; ++v) {   // f becomes the state before the token
        const bool z = SEQ && (cut >> s & 1);
        const float now = z ? f[s][v] : fmaf(a[s][v], h[v], f[s][v]);
        f[s][v] = z ? 0.0f : h[v];
        h[v] = now;
      }
#pragma unroll
    for (int s = S - 1; s >= 0; --s) {
      float dx[V], dg[V], di[V];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float G = d[s][v] + c[v];
        c[v] = SEQ && (cut >> s & 1) ? 0.0f : a[s][v] * G;
        float r, rr, sg = 1.0f, ss = 0.0f, av, beta;
        sigmoid2(g.v[s][v], r, rr);
        if (IG) sigmoid2(in.v[s][v], sg, ss);
        const float l = A[v] * r, xv = x.v[s][v];
        decay<NRM>(l, av, beta);
        float dl = c[v] * f[s][v], du = G;
        if (NRM) {
          // (where nothing decays, beta = 0, the quotient's limit times l is 0)
          dl = fmaf(-(G * (xv * sg)) * (av * av), beta == 0.0f ? 0.0f : __builtin_amdgcn_rcpf(beta), dl);
          du *= beta;
        }
        dx[v] = du * sg;
        di[v] = du * xv * sg * ss;
        dg[v] = dl * l * rr;
        if (t0 + s < p.L) dA[v] = fmaf(dl, r, dA[v]);
      }
      const int t = t0 + s;
      if (t < p.L) {
        const long o = b * p.yb + t * p.yl + c0;
        if (p.dx) Piece<BF, V>::store(p.dx, o, dx);
        if (p.dg) Piece<BF, V>::store(p.dg, o, dg);
        if (IG && p.di) Piece<BF, V>::store(p.di, o, di);
      }
      if (t == 0 && p.dh0) Piece<false, V>::store(p.dh0, (long)b * p.C + c0, c);
    }
    if (!LOOK) __syncthreads();
  }
  if (!p.part) return;
  if (LOOK) __syncthreads();
#pragma unroll
  for (int v = 0; v < V; ++v) sP[tt][cg * V + v] = dA[v];
  __syncthreads();
  if (tid < W) {
    float sum = 0.0f;
#pragma unroll 8
    for (int j = 0; j < TT; ++j) sum += sP[j][tid];
    p.part[((long)b * (LOOK ? p.nk : 1) + (LOOK ? p.nk - 1 - o0 : 0)) * p.C + mine] = sum;
  }
}

// dA: the sums of `rows` partial rows, in their order
__global__ __launch_bounds__(1024) void k_gscan_sum(const float* part, int rows, int C, float* out) {
  __shared__ float s[16][64];
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, c = blockIdx.x * 64 + lane;
  float sum = 0.0f;
  if (c < C)
    for (int r = wv; r < rows; r += 16) sum += part[(long)r * C + c];
  s[wv][lane] = sum;
  __syncthreads();
  if (wv || c >= C) return;
  sum = 0.0f;
#pragma unroll
  for (int i = 0; i < 16; ++i) sum += s[i][lane];
  out[c] = sum;
}

// One token a row.  Rows whose slot is none of the pool's give zeros and touch no state.  Several rows of one slot are taken in their order, by
// the first of them: a wave looks over all rows' slots, 64 at a time.
template <bool BF, bool IG, bool NRM>
__global__ __launch_bounds__(256) void k_gscan_step(GStepP p) {
  const int lane = threadIdx.x & 63, row = blockIdx.x / p.ncb;
  const int c0 = (blockIdx.x % p.ncb * 256 + threadIdx.x) * 4, n = min(4, p.C - c0);   // (n <= 0: no channel, but votes)
  auto slot_of = [&](int r) { return p.at64 ? ((const long*)p.at)[r] : (long)((const int*)p.at)[r]; };
  long slot = row;
  if (p.at) {
    slot = slot_of(row);
    if (slot < 0 || slot >= p.slots) {
      for (int v = 0; v < n; ++v) stv(p.y, (long)row * p.C + c0 + v, BF, 0.0f);
      return;
    }
    bool before = false;
    for (int r = lane; r < row; r += 64) before |= slot_of(r) == slot;
    if (__any(before)) return;
  }
  float* state = p.state + slot * p.state_s;
  float A[4], h[4];
#pragma unroll
  for (int v = 0; v < 4; ++v) {
    A[v] = v < n ? p.A[c0 + v] : 0.0f;
    h[v] = v < n ? state[c0 + v] : 0.0f;
  }
  for (int r = row;;) {
#pragma unroll
    for (int v = 0; v < 4; ++v)
      if (v < n) {
        float u = ldv(p.x, r * p.xs + c0 + v, BF), a, beta;
        if (IG) u *= sigmoid(ldv(p.i, r * p.is + c0 + v, BF));
        decay<NRM>(A[v] * sigmoid(ldv(p.g, r * p.gs + c0 + v, BF)), a, beta);
        h[v] = fmaf(a, h[v], NRM ? beta * u : u);
        stv(p.y, (long)r * p.C + c0 + v, BF, h[v]);
      }
    if (!p.at) break;
    int next = p.rows;   // the next row of the slot
    for (int q = r + 1; q < p.rows && next == p.rows; q += 64) {
      const unsigned long long hit = __ballot(q + lane < p.rows && slot_of(min(q + lane, p.rows - 1)) == slot);
      if (hit) next = q + __ffsll(hit) - 1;
    }
    if (next == p.rows) break;
    r = next;
  }
#pragma unroll
  for (int v = 0; v < 4; ++v)
    if (v < n) state[c0 + v] = h[v];
}

template <bool BF, int V, bool IG, bool NRM, bool SEQ>
static void launch_dir(const GScanP& p, bool back, int blocks, hipStream_t st) {
  if (back) {
    if (p.words) k_gscan_bwd<BF, V, GS_S, IG, NRM, SEQ, true><<<blocks, GS_THREADS, 0, st>>>(p);
    else k_gscan_bwd<BF, V, GS_S, IG, NRM, SEQ, false><<<blocks, GS_THREADS, 0, st>>>(p);
  } else {
    if (p.words) k_gscan_fwd<BF, V, GS_S, IG, NRM, SEQ, true><<<blocks, GS_THREADS, 0, st>>>(p);
    else k_gscan_fwd<BF, V, GS_S, IG, NRM, SEQ, false><<<blocks, GS_THREADS, 0, st>>>(p);
  }
}
template <bool BF, int V, bool IG, bool NRM>
static void launch_packed(const GScanP& p, bool back, int blocks, hipStream_t st) {
  p.ids ? launch_dir<BF, V, IG, NRM, true>(p, back, blocks, st) : launch_dir<BF, V, IG, NRM, false>(p, back, blocks, st);
}
template <bool BF, int V>
static void launch_form(const GScanP& p, bool nrm, bool back, int blocks, hipStream_t st) {
  if (p.i) nrm ? launch_packed<BF, V, true, true>(p, back, blocks, st) : launch_packed<BF, V, true, false>(p, back, blocks, st);
  else nrm ? launch_packed<BF, V, false, true>(p, back, blocks, st) : launch_packed<BF, V, false, false>(p, back, blocks, st);
}

// Whether a row's tiles go on workgroups of their own: up to where the rows of blocks of channels fill the GPU twice.  In us, forward and backward,
// bf16: 256 of them (8 x 4096 x 2048) 140 and 366, walked 169 and 312; 512 (32 x 2048 x 1024) 143 and 371, walked 129 and 315;
// 32 (1 x 4096 x 2048) 22.5 and 51.5, walked 139 and 254
bool gscan_looks(int B, int L, int C) { return gscan_tiles(L) > 1 && (long)B * gscan_blocks(C) < 2 * NCU; }
// Bytes of a call's workspace: partial sums of dA, then the tickets and what the tiles tell, in whole 16 bytes each
static size_t part_bytes(int B, int L, int C) { return ((size_t)B * (gscan_looks(B, L, C) ? gscan_tiles(L) : 1) * C * 4 + 255) & ~(size_t)255; }
static size_t ticket_bytes(int B, int C) { return (size_t)B * gscan_blocks(C) * GS_TICKET * 4; }
static size_t word_bytes(int B, int L, int C) { return (size_t)B * gscan_blocks(C) * gscan_tiles(L) * 64 * 8; }
size_t gscan_workspace(int B, int L, int C, bool back) {
  return (back ? part_bytes(B, L, C) : 0) + (gscan_looks(B, L, C) ? ticket_bytes(B, C) + word_bytes(B, L, C) : 0);
}

int launch_gscan(GScanP p, bool bf, bool nrm, bool back, void* workspace, hipStream_t st) {
  const bool wide = p.C >= 4;
  p.ncb = gscan_blocks(p.C);
  p.nk = gscan_tiles(p.L);
  int blocks = p.B * p.ncb, rows = p.B;
  char* ws = (char*)workspace;
  if (back) {
    p.part = p.dA ? (float*)ws : nullptr;
    ws += part_bytes(p.B, p.L, p.C);
  }
  if (gscan_looks(p.B, p.L, p.C)) {
    p.tickets = (unsigned*)ws;
    p.words = (unsigned long long*)(ws + ticket_bytes(p.B, p.C));
    const long n = (long)((ticket_bytes(p.B, p.C) + word_bytes(p.B, p.L, p.C)) / 16);
    k_gscan_clear<<<(int)min((n + 1023) / 1024, 1024L), 256, 0, st>>>((uint4*)ws, n);
    blocks *= p.nk;
    rows *= p.nk;
  }
  if (bf) wide ? launch_form<true, 4>(p, nrm, back, blocks, st) : launch_form<true, 1>(p, nrm, back, blocks, st);
  else wide ? launch_form<false, 4>(p, nrm, back, blocks, st) : launch_form<false, 1>(p, nrm, back, blocks, st);
  if (p.part) k_gscan_sum<<<(p.C + 63) / 64, 1024, 0, st>>>(p.part, rows, p.C, p.dA);
  return (int)hipGetLastError();
}

template <bool BF>
static void launch_step(const GStepP& p, bool nrm, hipStream_t st) {
  const unsigned grid = (unsigned)p.rows * p.ncb;
  if (p.i) nrm ? k_gscan_step<BF, true, true><<<grid, 256, 0, st>>>(p) : k_gscan_step<BF, true, false><<<grid, 256, 0, st>>>(p);
  else nrm ? k_gscan_step<BF, false, true><<<grid, 256, 0, st>>>(p) : k_gscan_step<BF, false, false><<<grid, 256, 0, st>>>(p);
}
int launch_gscan_step(GStepP p, bool bf, bool nrm, hipStream_t st) {
  p.ncb = (p.C + 1023) / 1024;
  bf ? launch_step<true>(p, nrm, st) : launch_step<false>(p, nrm, st);
  return (int)hipGetLastError();
}

}  // namespace issm
