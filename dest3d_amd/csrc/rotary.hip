// Rotary positions, with or without the norm of each head before them, for gfx950.
//   v = x / sqrt(mean x^2 + eps) w  (or x);   y1 = v1 c - v2 s,  y2 = v1 s + v2 c   for the pairs of the first R of a head's D features,
// pair j of features (j, j + R/2) or (2j, 2j + 1), c and s from the row of a table that the token's position names; the others are v.
// Backwards, with g = the gradient turned back (s negated):  dw = sum g xh,  dx = rstd (w g - xh mean(w g xh)),  xh = x rstd.
//
// A lane owns V pairs of a row (one head of one token), so that a rotation is its own affair; LPR lanes, a power of two, share a row and
// its sums, 64 / LPR rows a wave.  Rows are bound by their bytes (read and written once): each wave asks for NR times 64 / LPR rows
// before it works on the first.
#include "rotary_dev.h"

// (every multiply-add is written as one: the forms of a kernel that do the same sums are to give the same bits)
#pragma clang fp contract(off)

namespace issm {

// A row of either side: where it is, and its token's row of the table
struct Row {
  int side;
  unsigned b, l, h;
  long at, out;      // element offsets
  const float* turn; // NULL: the position is none of the table's
};
__device__ __forceinline__ long place(const Row& r, const long (&s)[3]) { return r.b * s[0] + r.l * s[1] + r.h * s[2]; }
__device__ __forceinline__ Row row_of(const RotP& p, unsigned n, int side) {
  Row r;
  unsigned token = n;
  if (side < 0) {    // of both sides, token by token
    r.h = p.by_heads(token);
    r.side = (int)r.h >= p.H[0];
    r.h -= r.side ? p.H[0] : 0;
  } else {
    r.h = (side ? p.by_k : p.by_q)(token);
    r.side = side;
  }
  r.b = token;
  r.l = p.by_L(r.b);
  r.at = place(r, p.s[r.side]);
  r.out = ((long)token * p.H[r.side] + r.h) * p.D;
  long pos = r.l;
  if (p.pos) {
    const long o = r.b * p.pos_b + r.l * p.pos_l;
    pos = p.pos64 ? ((const long*)p.pos)[o] : (long)((const int*)p.pos)[o];
  }
  r.turn = pos >= 0 && pos < p.rows ? p.table + pos * p.R : nullptr;
  return r;
}

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

// A lane's part of a row
template <bool BF, int V, int NI, bool INTER>
struct Part {
  float one[NI][V], two[NI][V];
  __device__ __forceinline__ void load(const RotP& p, const void* x, long at, int li, bool there) {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int q = (i * p.lpr + li) * V;
      const bool ok = there && q < p.pairs;
      int o, t;
      features<INTER>(p, ok ? q : 0, o, t);
      const long base = there ? at : 0;
      if constexpr (INTER && V > 1) {
        Piece<BF, 2 * V> m;
        m.load(x, base + o);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          one[i][v] = ok ? m[2 * v] : 0.0f;
          two[i][v] = ok ? m[2 * v + 1] : 0.0f;
        }
      } else {
        const bool ok2 = ok && (V > 1 || t < p.D);
        Piece<BF, V> m, n;
        m.load(x, base + o);
        n.load(x, base + (V > 1 || t < p.D ? t : o));
#pragma unroll
        for (int v = 0; v < V; ++v) {
          one[i][v] = ok ? m[v] : 0.0f;
          two[i][v] = ok2 ? n[v] : 0.0f;
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
  // by the angles' cosines and sign times their sines
  __device__ __forceinline__ void turn(const RotP& p, const float* row, int li, float sign) {
    const int half = p.R >> 1;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int q = (i * p.lpr + li) * V;
      if (q >= half) continue;
      Word<V> c, s;
      if (row) {
        c = *(const Word<V>*)(row + q);
        s = *(const Word<V>*)(row + half + q);
      } else {
#pragma unroll
        for (int v = 0; v < V; ++v) c.v[v] = s.v[v] = __builtin_nanf("");
      }
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float sn = sign * s.v[v], a = one[i][v], b = two[i][v];
        one[i][v] = fmaf(a, c.v[v], -(b * sn));
        two[i][v] = fmaf(a, sn, b * c.v[v]);
      }
    }
  }
  __device__ __forceinline__ float dot(const Part& other) const {
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int v = 0; v < V; ++v) s = fmaf(one[i][v], other.one[i][v], fmaf(two[i][v], other.two[i][v], s));
    return s;
  }
  __device__ __forceinline__ void scale(const Part& w, float f) {
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        one[i][v] *= f * w.one[i][v];
        two[i][v] *= f * w.two[i][v];
      }
  }
};

__device__ __forceinline__ float row_sum(float v, int lpr) {
  for (int o = lpr >> 1; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

template <bool BF, int V, int NI, bool INTER, bool NORM, int NR>
__global__ __launch_bounds__(256) void k_rotary(RotP p) {
  const int lane = threadIdx.x & 63, li = lane & (p.lpr - 1), sub = lane / p.lpr, per = 64 / p.lpr;
  const long first = ((long)blockIdx.x * 4 + (threadIdx.x >> 6)) * (NR * per) + sub;
  Row row[NR];
  Part<BF, V, NI, INTER> x[NR];
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    const long i = first + n * per;
    row[n] = row_of(p, (unsigned)min(i, p.all - 1), -1);   // (rows behind the last are the last, not stored)
    x[n].load(p, p.x[row[n].side], row[n].at, li, true);
  }
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    if (NORM) {
      Part<BF, V, NI, INTER> w;
      if (p.w_bf) {
        Part<true, V, NI, INTER> wb;
        wb.load(p, p.w[row[n].side], 0, li, true);
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
          for (int v = 0; v < V; ++v) {
            w.one[i][v] = wb.one[i][v];
            w.two[i][v] = wb.two[i][v];
          }
      } else {
        Part<false, V, NI, INTER> wf;
        wf.load(p, p.w[row[n].side], 0, li, true);
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
          for (int v = 0; v < V; ++v) {
            w.one[i][v] = wf.one[i][v];
            w.two[i][v] = wf.two[i][v];
          }
      }
      const float ss = row_sum(x[n].dot(x[n]), p.lpr);
      x[n].scale(w, 1.0f / sqrtf(ss / (float)p.D + p.eps));
    }
    x[n].turn(p, row[n].turn, li, p.sign);
    if (first + n * per < p.all) x[n].store(p, p.y[row[n].side], row[n].out, li);
  }
}

// Workgroups [0, blocks[0]) walk the queries' rows, those behind them the keys'; each leaves its sums of dw
template <bool BF, int V, int NI, bool INTER>
__global__ __launch_bounds__(256) void k_rotary_norm_bwd(RotP p) {
  extern __shared__ float sums[];   // (4, D)
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, li = lane & (p.lpr - 1), sub = lane / p.lpr, per = 64 / p.lpr;
  const int side = (int)blockIdx.x >= p.blocks[0], block = blockIdx.x - (side ? p.blocks[0] : 0);
  const long rows = (long)p.tokens * p.H[side];
  Part<BF, V, NI, INTER> w, dw;
  if (p.w_bf) {
    Part<true, V, NI, INTER> wb;
    wb.load(p, p.w[side], 0, li, true);
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        w.one[i][v] = wb.one[i][v];
        w.two[i][v] = wb.two[i][v];
      }
  } else {
    Part<false, V, NI, INTER> wf;
    wf.load(p, p.w[side], 0, li, true);
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        w.one[i][v] = wf.one[i][v];
        w.two[i][v] = wf.two[i][v];
      }
  }
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int v = 0; v < V; ++v) dw.one[i][v] = dw.two[i][v] = 0.0f;
  for (long i0 = ((long)block * 4 + wave) * per; i0 < rows; i0 += (long)p.blocks[side] * 4 * per) {
    const long n = i0 + sub;
    const bool there = n < rows;
    const Row row = row_of(p, (unsigned)(there ? n : rows - 1), side);
    Part<BF, V, NI, INTER> x, g;
    x.load(p, p.x[side], row.at, li, there);
    g.load(p, p.dy[side], place(row, p.ds[side]), li, there);
    g.turn(p, row.turn, li, -1.0f);
    const float ss = row_sum(x.dot(x), p.lpr);
    const float rstd = 1.0f / sqrtf(ss / (float)p.D + p.eps);
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        x.one[i][v] *= rstd;
        x.two[i][v] *= rstd;
        if (there) {
          dw.one[i][v] = fmaf(g.one[i][v], x.one[i][v], dw.one[i][v]);
          dw.two[i][v] = fmaf(g.two[i][v], x.two[i][v], dw.two[i][v]);
        }
        g.one[i][v] *= w.one[i][v];
        g.two[i][v] *= w.two[i][v];
      }
    const float mean = row_sum(g.dot(x), p.lpr) / (float)p.D;
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        g.one[i][v] = rstd * fmaf(-x.one[i][v], mean, g.one[i][v]);
        g.two[i][v] = rstd * fmaf(-x.two[i][v], mean, g.two[i][v]);
      }
    if (there) g.store(p, p.y[side], row.out, li);
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

// dw of both sides, from the workgroups' sums in their order
__global__ __launch_bounds__(1024) void k_rotary_dw(RotP p) {
  __shared__ float s[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, d = blockIdx.x * 64 + lane, side = blockIdx.y;
  const int first = side ? p.blocks[0] : 0;
  float sum = 0.0f;
  if (d < p.D)
    for (int r = wave; r < p.blocks[side]; r += 16) sum += p.part[(long)(first + r) * p.D + d];
  s[wave][lane] = sum;
  __syncthreads();
  if (wave || d >= p.D || !p.dw[side]) return;
  sum = 0.0f;
#pragma unroll
  for (int i = 0; i < 16; ++i) sum += s[i][lane];
  stv(p.dw[side], d, p.w_bf, sum);
}

template <bool BF, int V, int NI, bool INTER>
static bool launch_rows(const RotP& p, bool norm, hipStream_t st) {
  constexpr int NR = NI > 1 ? 1 : 4;
  const long per = 4L * NR * (64 / p.lpr);
  const long blocks = (p.all + per - 1) / per;
  if (blocks >= 1L << 24) return false;   // (a launch has fewer than 2^32 threads)
  if (norm) k_rotary<BF, V, NI, INTER, true, NR><<<blocks, 256, 0, st>>>(p);
  else k_rotary<BF, V, NI, INTER, false, NR><<<blocks, 256, 0, st>>>(p);
  return true;
}
template <bool BF, int V, int NI, bool INTER>
static bool launch_norm_bwd(const RotP& p, hipStream_t st) {
  k_rotary_norm_bwd<BF, V, NI, INTER><<<p.blocks[0] + p.blocks[1], 256, 4 * p.D * sizeof(float), st>>>(p);
  return true;
}

// V: the widest that both parts of a head, turned and not, are whole multiples of, up to 16 bytes an access, if 64 lanes hold a row
template <bool BF, bool INTER>
static bool launch_widths(RotP& p, bool norm, bool back, hipStream_t st) {
  const int half = p.R / 2, rest = p.D - p.R;
  int V = 1;
  for (int v = BF ? 8 : 4; v > 1; v >>= 1)
    if (half % v == 0 && rest % (2 * v) == 0) {
      V = v;
      break;
    }
  p.pairs = half + (rest + 1) / 2;
  if ((p.pairs + V - 1) / V > 64) V = 1;
  const int lanes = (p.pairs + V - 1) / V;
  p.lpr = 1;
  while (p.lpr < lanes && p.lpr < 64) p.lpr *= 2;
#define ROT(v, ni) (back ? launch_norm_bwd<BF, v, ni, INTER>(p, st) : launch_rows<BF, v, ni, INTER>(p, norm, st))
  if constexpr (BF)
    if (V == 8) return ROT(8, 1);
  if (V == 4) return ROT(4, 1);
  if (V == 2) return ROT(2, 1);
  if (lanes <= 64) return ROT(1, 1);
  return ROT(1, ROT_MAX_D / 128);
#undef ROT
}

static void divisors(RotP& p) {
  p.by_heads = div_by(p.H[0] + p.H[1]);
  p.by_q = div_by(p.H[0] ? p.H[0] : 1);
  p.by_k = div_by(p.H[1] ? p.H[1] : 1);
  p.by_L = div_by(p.L);
  p.all = (long)p.tokens * (p.H[0] + p.H[1]);
}

int launch_rotary(RotP p, bool bf, bool inter, bool norm, hipStream_t st) {
  divisors(p);
  bool ok;
  if (bf) ok = inter ? launch_widths<true, true>(p, norm, false, st) : launch_widths<true, false>(p, norm, false, st);
  else ok = inter ? launch_widths<false, true>(p, norm, false, st) : launch_widths<false, false>(p, norm, false, st);
  return ok ? (int)hipGetLastError() : (int)hipErrorInvalidConfiguration;
}

int launch_rotary_norm_bwd(RotP p, bool bf, bool inter, hipStream_t st) {
  divisors(p);
  for (int i = 0; i < 2; ++i) p.blocks[i] = rotary_bwd_blocks((long)p.tokens * p.H[i]);
  if (bf) inter ? launch_widths<true, true>(p, true, true, st) : launch_widths<true, false>(p, true, true, st);
  else inter ? launch_widths<false, true>(p, true, true, st) : launch_widths<false, false>(p, true, true, st);
  k_rotary_dw<<<dim3((p.D + 63) / 64, 2), 1024, 0, st>>>(p);
  return (int)hipGetLastError();
}

}  // namespace issm
