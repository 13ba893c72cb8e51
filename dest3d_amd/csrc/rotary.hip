// Rotary positions, with or without the norm of each head before them, for gfx950.
//   v = x / sqrt(mean x^2 + eps) w  (or x);   y1 = v1 c - v2 s,  y2 = v1 s + v2 c   for the pairs of the first R of a head's D features,
// pair j of features (j, j + R/2) or (2j, 2j + 1), c and s from the row of a table that the token's position names; the others are v.
// Backwards, with g = the gradient turned back (s negated):  dw = sum g xh,  dx = rstd (w g - xh mean(w g xh)),  xh = x rstd.
//
// A lane owns V pairs of a row (one head of one token), so that a rotation is its own affair; LPR lanes, a power of two, share a row and
// its sums.  The 64 / LPR rows that a wave has at a time are `group` heads of 64 / LPR / group tokens; it goes on to their other heads, or, where
// a token has no more, to other tokens, and asks for NB of its rows before it works on the first.  Angles and weights stay with the lane.
// Rows are bound by their bytes, read and written once: bf16, 16384 tokens of 32 and 8 heads of 128, with the norm, 70 us, 4.8 TB/s (a copy
// of 256 MiB 5.4); 65536 of 16 and 4, alone, 130 us, 5.2; the norm's gradients of 16384 tokens of 16 and 4, 252 MB, 53 us behind other work and 47
// over and over, 4.8 and 5.4.  Rows with angles and weights asked for each by itself, four at a time: 97, 151 and 63 us.
#include "rotary_dev.h"

// (every multiply-add is written as one: the forms of a kernel that do the same sums are to give the same bits)
#pragma clang fp contract(off)

namespace issm {

// A token: its place and its row of the table
struct Token {
  unsigned b, l;
  const float* turn; // NULL: the position is none of the table's
};
__device__ __forceinline__ Token token_of(const RotP& p, unsigned token) {
  Token t;
  t.b = token;
  t.l = p.by_L(t.b);
  long pos = t.l;
  if (p.pos) {
    const long o = t.b * p.pos_b + t.l * p.pos_l;
    pos = p.pos64 ? ((const long*)p.pos)[o] : (long)((const int*)p.pos)[o];
  }
  t.turn = pos >= 0 && pos < p.rows ? p.table + pos * p.R : nullptr;
  return t;
}
__device__ __forceinline__ long place(const Token& t, unsigned h, const long (&s)[3]) { return t.b * s[0] + t.l * s[1] + h * s[2]; }

// Pair q's two features; the unturned ones behind R are paired the same way
template <bool INTER>
__device__ __forceinline__ void features(const RotP& p, int q, int& one, int& two) {
  if (INTER) {
    one = 2 * q;
    two = one + 1;
  } else {
    const int half = p.R >> 1, rest = (p.D - p.R + 1) >> 1;
    const bool turned = q < half;
    one = turned ? q : p.R + q - half;
    two = one + (turned ? half : rest);
  }
}

// A lane's part of a row, as it lies
template <bool BF, int V, int NI, bool INTER>
struct Part {
  static constexpr bool WIDE = INTER && V > 1;
  Piece<BF, WIDE ? 2 * V : V> m[NI], n[WIDE ? 1 : NI];
  // (lanes without pairs read the row's first; what they have is counted in no sum and not stored)
  __device__ __forceinline__ void load(const RotP& p, const void* x, long at, int li) {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int q = (i * p.lpr + li) * V;
      int o, t;
      features<INTER>(p, q < p.pairs ? q : 0, o, t);
      m[i].load(x, at + o);
      if constexpr (!WIDE) n[i].load(x, at + (V > 1 || t < p.D ? t : o));
    }
  }
};
// and as numbers
template <bool BF, int V, int NI, bool INTER>
struct Nums {
  float one[NI][V], two[NI][V];
  __device__ __forceinline__ void take(const RotP& p, const Part<BF, V, NI, INTER>& part, int li) {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int q = (i * p.lpr + li) * V;
      const bool ok = q < p.pairs;
      bool ok2 = ok;
      if (V == 1) {
        int o, t;
        features<INTER>(p, q, o, t);
        ok2 = ok && t < p.D;
      }
#pragma unroll
      for (int v = 0; v < V; ++v) {
        if constexpr (INTER && V > 1) {
          one[i][v] = ok ? part.m[i][2 * v] : 0.0f;
          two[i][v] = ok ? part.m[i][2 * v + 1] : 0.0f;
        } else {
          one[i][v] = ok ? part.m[i][v] : 0.0f;
          two[i][v] = ok2 ? part.n[i][v] : 0.0f;
        }
      }
    }
  }
  __device__ __forceinline__ void store(const RotP& p, void* y, long at, int li) const {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int q = (i * p.lpr + li) * V;
      if (q >= p.pairs) continue;
      int o, t;
      features<INTER>(p, q, o, t);
      if constexpr (INTER && V > 1) {
        float f[2 * V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
          f[2 * v] = one[i][v];
          f[2 * v + 1] = two[i][v];
        }
        Piece<BF, 2 * V>::store(y, at + o, f);
      } else {
        Piece<BF, V>::store(y, at + o, one[i]);
        if (V > 1 || t < p.D) Piece<BF, V>::store(y, at + t, two[i]);
      }
    }
  }
  __device__ __forceinline__ float dot(const Nums& other) const {
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int v = 0; v < V; ++v) s = fmaf(one[i][v], other.one[i][v], fmaf(two[i][v], other.two[i][v], s));
    return s;
  }
};
// A lane's angles: cosines and `sign` times the sines; 1 and 0 for the features that are not turned
template <int V, int NI>
struct Angles {
  float c[NI][V], s[NI][V];
  __device__ __forceinline__ void load(const RotP& p, const float* row, int li, float sign) {
    const int half = p.R >> 1;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int q = (i * p.lpr + li) * V;
      const bool turned = q < half;
      const float* at = (row ? row : p.table) + (turned ? q : 0);
      const Word<V> a = *(const Word<V>*)at, b = *(const Word<V>*)(at + half);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        c[i][v] = turned ? (row ? a.v[v] : __builtin_nanf("")) : 1.0f;
        s[i][v] = turned ? (row ? sign * b.v[v] : __builtin_nanf("")) : 0.0f;
      }
    }
  }
  template <bool BF, bool INTER>
  __device__ __forceinline__ void turn(const RotP& p, Nums<BF, V, NI, INTER>& x, int li) const {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const bool turned = (i * p.lpr + li) * V < p.R >> 1;   // (the others as they are, infinite ones too)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float a = x.one[i][v], b = x.two[i][v];
        x.one[i][v] = turned ? fmaf(a, c[i][v], -(b * s[i][v])) : a;
        x.two[i][v] = turned ? fmaf(a, s[i][v], b * c[i][v]) : b;
      }
    }
  }
};
// The weights of a side, whichever their type
template <int V, int NI, bool INTER>
struct Weights : Nums<false, V, NI, INTER> {
  __device__ __forceinline__ void load(const RotP& p, const void* w, int li) {
    if (p.w_bf) {
      Part<true, V, NI, INTER> raw;
      raw.load(p, w, 0, li);
      Nums<true, V, NI, INTER> x;
      x.take(p, raw, li);
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int v = 0; v < V; ++v) {
          this->one[i][v] = x.one[i][v];
          this->two[i][v] = x.two[i][v];
        }
    } else {
      Part<false, V, NI, INTER> raw;
      raw.load(p, w, 0, li);
      this->take(p, raw, li);
    }
  }
};

// Sums over the lpr lanes of a row, of N rows at a time
template <int CTRL>
__device__ __forceinline__ float dpp_add(float v) {
  return v + __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), CTRL, 0xf, 0xf, true));
}
template <int N>
__device__ __forceinline__ void row_sums(float (&v)[N], int lpr) {
  if (lpr > 1)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = dpp_add<0xb1>(v[i]);    // lanes 1, 0, 3, 2
  if (lpr > 2)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = dpp_add<0x4e>(v[i]);    // 2, 3, 0, 1
  if (lpr > 4)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = dpp_add<0x141>(v[i]);   // mirrored in 8
  if (lpr > 8)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = dpp_add<0x140>(v[i]);   // mirrored in 16
  if (lpr > 16)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor(v[i], 16, 64);
  if (lpr > 32)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor(v[i], 32, 64);
}

// MANY: the lane's rows are of NB tokens, one head of each; else `heads_each` heads of one token
template <bool BF, int V, int NI, bool INTER, bool NORM, int NB, bool MANY>
__global__ __launch_bounds__(256) void k_rotary(RotP p) {
  const int lane = threadIdx.x & 63, li = lane & (p.lpr - 1), sub = lane / p.lpr, tokens = 64 / p.lpr / p.group;   // tokens at a time
  unsigned unit = (p.first + blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned part = p.by_parts(unit);
  const int heads = p.H[0] + p.H[1], h0 = (int)part * p.heads_each * p.group + sub % p.group, mine = sub / p.group;
  const long t0 = (long)unit * (MANY ? NB : 1) * tokens + mine;
  if ((long)unit * (MANY ? NB : 1) * tokens >= p.tokens) return;
  Weights<V, NI, INTER> wq, wk;
  Angles<V, NI> angles;
  Token token;
  if (!MANY) token = token_of(p, (unsigned)min(t0, (long)p.tokens - 1));
  for (int n0 = 0; n0 < (MANY ? 1 : p.heads_each); n0 += NB) {
    Part<BF, V, NI, INTER> raw[NB];
    int side[NB];
    unsigned h[NB];
    Token at[NB];
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      if (!MANY && n0 + j >= p.heads_each) continue;
      const int all = min(h0 + (MANY ? 0 : (n0 + j) * p.group), heads - 1);
      side[j] = all >= p.H[0];
      h[j] = all - (side[j] ? p.H[0] : 0);
      at[j] = MANY ? token_of(p, (unsigned)min(t0 + j * tokens, (long)p.tokens - 1)) : token;
      raw[j].load(p, p.x[side[j]], place(at[j], h[j], p.s[side[j]]), li);
    }
    if (n0 == 0) {
      if (!MANY) angles.load(p, token.turn, li, p.sign);
      if (NORM) {
        wq.load(p, p.w[p.H[0] ? 0 : 1], li);
        wk.load(p, p.w[p.H[1] ? 1 : 0], li);
      }
    }
    Nums<BF, V, NI, INTER> x[NB];
    float ss[NB];
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      if (!MANY && n0 + j >= p.heads_each) {
        ss[j] = 0.0f;
        continue;
      }
      x[j].take(p, raw[j], li);
      if (NORM) ss[j] = x[j].dot(x[j]);
    }
    if (NORM) row_sums(ss, p.lpr);
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      if (!MANY && n0 + j >= p.heads_each) continue;
      if (NORM) {
        const float rstd = __builtin_amdgcn_rsqf(ss[j] * p.inv_D + p.eps);
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
          for (int v = 0; v < V; ++v) {
            x[j].one[i][v] *= rstd * (side[j] ? wk.one[i][v] : wq.one[i][v]);
            x[j].two[i][v] *= rstd * (side[j] ? wk.two[i][v] : wq.two[i][v]);
          }
      }
      if (MANY) angles.load(p, at[j].turn, li, p.sign);
      angles.turn(p, x[j], li);
      const long t = t0 + (MANY ? j * tokens : 0);
      if (t < p.tokens && h0 + (MANY ? 0 : (n0 + j) * p.group) < heads) x[j].store(p, p.y[side[j]], (t * p.H[side[j]] + h[j]) * p.D, li);
    }
  }
}

// Workgroups [0, blocks[0]) walk the queries' rows, those behind them the keys'; each leaves its sums of dw.  A row a lane at a time, MANY or not: two rows
// asked for at a time leave too few waves (4096 x 4 tokens of 16 and 4 heads of 128, bf16: 52.9 us for 46.6)
template <bool BF, int V, int NI, bool INTER, bool MANY>
__global__ __launch_bounds__(256) void k_rotary_norm_bwd(RotP p) {
  extern __shared__ float sums[];   // (4, D)
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), li = lane & (p.lpr - 1), sub = lane / p.lpr;
  const int side = (int)blockIdx.x >= p.blocks[0], block = blockIdx.x - (side ? p.blocks[0] : 0);
  const int heads = p.H[side], group = p.groups[side], tokens = 64 / p.lpr / group, mine = sub / group, h0 = sub % group;
  const int each = (heads + group - 1) / group;
  Weights<V, NI, INTER> w;
  w.load(p, p.w[side], li);
  Nums<false, V, NI, INTER> dw;
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int v = 0; v < V; ++v) dw.one[i][v] = dw.two[i][v] = 0.0f;
  for (long u = ((long)block * 4 + wave) * tokens; u < p.tokens; u += (long)p.blocks[side] * 4 * tokens) {
    Angles<V, NI> angles;
    Token token;
    if (!MANY) token = token_of(p, (unsigned)min(u + mine, (long)p.tokens - 1));
    for (int n0 = 0; n0 < (MANY ? 1 : each); ++n0) {
      const int n = h0 + (MANY ? 0 : n0 * group);
      const long t = u + mine;
      const unsigned h = min(n, heads - 1);
      if (MANY) token = token_of(p, (unsigned)min(t, (long)p.tokens - 1));
      const bool there = n < heads && t < p.tokens;
      Part<BF, V, NI, INTER> rx, rg;
      rx.load(p, p.x[side], place(token, h, p.s[side]), li);
      rg.load(p, p.dy[side], place(token, h, p.ds[side]), li);
      if (!MANY && n0 == 0) angles.load(p, token.turn, li, -1.0f);
      Nums<BF, V, NI, INTER> x, g;
      x.take(p, rx, li);
      g.take(p, rg, li);
      if (MANY) angles.load(p, token.turn, li, -1.0f);
      angles.turn(p, g, li);
      float both[2];   // sums of x^2 and of w g x
      both[0] = x.dot(x);
      float s = 0.0f;
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int v = 0; v < V; ++v)
          s = fmaf(g.one[i][v] * w.one[i][v], x.one[i][v], fmaf(g.two[i][v] * w.two[i][v], x.two[i][v], s));
      both[1] = s;
      row_sums(both, p.lpr);
      const float rstd = __builtin_amdgcn_rsqf(both[0] * p.inv_D + p.eps), mean = both[1] * rstd * p.inv_D;
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float x1 = x.one[i][v] * rstd, x2 = x.two[i][v] * rstd, g1 = g.one[i][v], g2 = g.two[i][v];
          dw.one[i][v] = there ? fmaf(g1, x1, dw.one[i][v]) : dw.one[i][v];
          dw.two[i][v] = there ? fmaf(g2, x2, dw.two[i][v]) : dw.two[i][v];
          x.one[i][v] = rstd * fmaf(-x1, mean, g1 * w.one[i][v]);
          x.two[i][v] = rstd * fmaf(-x2, mean, g2 * w.two[i][v]);
        }
      if (there) x.store(p, p.y[side], (t * heads + h) * p.D, li);
    }
  }
  // the rows of a wave, then the waves
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int v = 0; v < V; ++v) {
      for (int o = 32; o >= p.lpr; o >>= 1) {
        dw.one[i][v] += __shfl_xor(dw.one[i][v], o, 64);
        dw.two[i][v] += __shfl_xor(dw.two[i][v], o, 64);
      }
      const int q = (i * p.lpr + li) * V + v;
      int one, two;
      if (sub == 0 && q < p.pairs) {
        features<INTER>(p, q, one, two);
        sums[wave * p.D + one] = dw.one[i][v];
        if (two < p.D) sums[wave * p.D + two] = dw.two[i][v];
      }
    }
  __syncthreads();
  for (int d = threadIdx.x; d < p.D; d += 256)
    p.part[(long)blockIdx.x * p.D + d] = (sums[d] + sums[p.D + d]) + (sums[2 * p.D + d] + sums[3 * p.D + d]);
}

// dw of both sides, from the workgroups' sums in their order: 16 columns and 64 strands of rows a workgroup
__global__ __launch_bounds__(1024) void k_rotary_dw(RotP p) {
  __shared__ float s[64][17];
  const int c = threadIdx.x & 15, strand = threadIdx.x >> 4, d = blockIdx.x * 16 + c, side = blockIdx.y, n = p.blocks[side];
  if (!p.dw[side]) return;
  const float* part = p.part + (long)(side ? p.blocks[0] : 0) * p.D + min(d, p.D - 1);
  s[strand][c] = strand_sum(part, p.D, strand, n);
  __syncthreads();
  if (strand || d >= p.D) return;
  float sum = 0.0f;
#pragma unroll 16
  for (int i = 0; i < 64; ++i) sum += s[i][c];
  stv(p.dw[side], d, p.w_bf, sum);
}

// Units of work: a wave each, as few heads a wave as it takes to have WAVES of them
constexpr long WAVES = 4096;
template <bool BF, int V, int NI, bool INTER, bool NORM>
static void launch_rows(RotP& p, hipStream_t st) {
  constexpr int NB = NI > 1 || !NORM ? 1 : 2;   // (16384 tokens of 32 and 8 heads of 128, bf16, with the norm, 1, 2, 4: 73.6, 68.5, 95.0 us; 65536 of 16
                                                // and 4, without, 1 and 2: 129 and 136)
  const int rows = 64 / p.lpr, heads = p.H[0] + p.H[1];
  p.group = 1;
  while (p.group < heads && p.group < rows) p.group *= 2;
  const int tokens = rows / p.group, each = (heads + p.group - 1) / p.group;
  const long units = (p.tokens + (long)tokens - 1) / tokens;
  long parts = 1;
  while (parts < each && units * parts < WAVES) ++parts;
  p.heads_each = (each + (int)parts - 1) / (int)parts;
  parts = (each + p.heads_each - 1) / p.heads_each;
  p.by_parts = div_by((unsigned)parts);
  const bool many = p.heads_each == 1 && units * parts >= 2 * WAVES;   // (waves enough with several tokens each)
  const long waves = (many ? (units + NB - 1) / NB : units) * parts, blocks = (waves + 3) / 4;
  constexpr long MOST = (1L << 24) - 1;   // (a launch has fewer than 2^32 threads: 2^26 rows of 33 pairs go in two)
  for (long b = 0; b < blocks; b += MOST) {
    p.first = (unsigned)b;
    const unsigned n = (unsigned)min(blocks - b, MOST);
    if (many) k_rotary<BF, V, NI, INTER, NORM, NB, true><<<n, 256, 0, st>>>(p);
    else k_rotary<BF, V, NI, INTER, NORM, NB, false><<<n, 256, 0, st>>>(p);
  }
}
template <bool BF, int V, int NI, bool INTER>
static void launch_norm_bwd(RotP& p, hipStream_t st) {
  const int rows = 64 / p.lpr;
  bool many = true;
  for (int i = 0; i < 2; ++i) {
    p.groups[i] = 1;
    while (p.groups[i] < p.H[i] && p.groups[i] < rows) p.groups[i] *= 2;
    many = many && p.H[i] <= p.groups[i];
  }
  const unsigned blocks = p.blocks[0] + p.blocks[1], bytes = 4 * p.D * sizeof(float);
  if (many) k_rotary_norm_bwd<BF, V, NI, INTER, true><<<blocks, 256, bytes, st>>>(p);
  else k_rotary_norm_bwd<BF, V, NI, INTER, false><<<blocks, 256, bytes, st>>>(p);
}

// V: the widest that both parts of a head, turned and not, are whole multiples of, if 64 lanes hold a row; up to 16 bytes an access forward (16384 tokens
// of 32 and 8 heads of 128, bf16, 8 and 4: 68.5 and 86.7 us), 4 backwards, where wider ones leave too few waves (46.8 and 43.7 us, heads of 64 29.6 and 25.9)
template <bool BF, bool INTER>
static void launch_widths(RotP& p, bool norm, bool back, hipStream_t st) {
  const int half = p.R / 2, rest = p.D - p.R;
  int V = 1;
  for (int v = BF && !back ? 8 : 4; v > 1; v >>= 1)
    if (half % v == 0 && rest % (2 * v) == 0) {
      V = v;
      break;
    }
  p.pairs = half + (rest + 1) / 2;
  if ((p.pairs + V - 1) / V > 64) V = 1;
  const int lanes = (p.pairs + V - 1) / V;
  p.lpr = 1;
  while (p.lpr < lanes && p.lpr < 64) p.lpr *= 2;
#define ROT(v, ni) \
  (back ? launch_norm_bwd<BF, v, ni, INTER>(p, st) : norm ? launch_rows<BF, v, ni, INTER, true>(p, st) : launch_rows<BF, v, ni, INTER, false>(p, st))
  if constexpr (BF)
    if (V == 8) return norm ? launch_rows<BF, 8, 1, INTER, true>(p, st) : launch_rows<BF, 8, 1, INTER, false>(p, st);
  if (V == 4) return ROT(4, 1);
  if (V == 2) return ROT(2, 1);
  if (lanes <= 64) return ROT(1, 1);
  return ROT(1, ROT_MAX_D / 128);
#undef ROT
}

static void divisors(RotP& p) {
  p.by_L = div_by(p.L);
  p.inv_D = 1.0f / (float)p.D;
}

int launch_rotary(RotP p, bool bf, bool inter, bool norm, hipStream_t st) {
  divisors(p);
  if (bf) inter ? launch_widths<true, true>(p, norm, false, st) : launch_widths<true, false>(p, norm, false, st);
  else inter ? launch_widths<false, true>(p, norm, false, st) : launch_widths<false, false>(p, norm, false, st);
  return (int)hipGetLastError();
}

int launch_rotary_norm_bwd(RotP p, bool bf, bool inter, hipStream_t st) {
  divisors(p);
  for (int i = 0; i < 2; ++i) p.blocks[i] = rotary_bwd_blocks((long)p.tokens * p.H[i]);
  if (bf) inter ? launch_widths<true, true>(p, true, true, st) : launch_widths<true, false>(p, true, true, st);
  else inter ? launch_widths<false, true>(p, true, true, st) : launch_widths<false, false>(p, true, true, st);
  k_rotary_dw<<<dim3((p.D + 15) / 16, 2), 1024, 0, st>>>(p);
  return (int)hipGetLastError();
}

}  // namespace issm
