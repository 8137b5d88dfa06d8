// Device code of paged caches that may hold 8 bits: written by positions of several axes, slots moved together, and attention of
// drafted tokens (csrc/rx_lm.h states what they compute).
#pragma once
#include "rx_lm_norm_kernels.h"

template <bool B, typename X, typename Y> struct rx_lm_if { typedef X type; };
template <typename X, typename Y> struct rx_lm_if<false, X, Y> { typedef Y type; };
constexpr int rx_lm_pow2(const int n) { return n <= 1 ? 1 : 2 * rx_lm_pow2((n + 1) / 2); }

// A token's heads, EACH of them after one another, to a group of LANES lanes, NE elements of 16 bytes to a lane: what a head's
// largest magnitude is found over, and what the cosines and sines of its dimensions are loaded for once.  Every lane loads the
// pairs' other elements itself.
template <typename E, typename C, int HQ, int HK, int DK, int DV, int P, int S, int B, int M, int L, int R2, int A, int S0, int S1, int S2, bool PAIRS, bool BY_SLOT, int T,
          bool WHOLE, int EACH, typename I>
RX_DEV void rx_kv_write(const typename E::S* q, const typename E::S* k, const typename E::S* v, const float* cos, const float* sin, const I* angle, const I* position,
                        const I* sequence, const I* pages, typename E::S* qo, typename C::S* kc, typename C::S* vc, float* ks, float* vs) {
  typedef typename E::S X;
  constexpr int NE = 16 / sizeof(X), LANES = rx_lm_pow2(((DK > DV ? DK : DV) + NE - 1) / NE);
  constexpr int GQ = (HQ + EACH - 1) / EACH, GK = (HK + EACH - 1) / EACH, ALL = GQ + 2 * GK;   // groups of a token
  constexpr bool BITS8 = rx_lm_is8<C>::value;
  typedef rx_vec<X, NE> W;
  const int lane = threadIdx.x % LANES, d = lane * NE;
  for (long long i = ((long long)blockIdx.x * 256 + threadIdx.x) / LANES; i < (long long)T * ALL; i += (long long)gridDim.x * (256 / LANES)) {
    const long long t = i / ALL;
    const int u = (int)(i % ALL), kind = u < GQ ? 0 : u < GQ + GK ? 1 : 2, first = (u - (kind == 0 ? 0 : kind == 1 ? GQ : GQ + GK)) * EACH;
    const I pos = position[t], seq = sequence[t];
    bool known = pos >= 0 && pos < (I)(M * S) && seq >= 0 && seq < B;
    I row[A] = {};
    if constexpr (R2 > 0) {
#pragma unroll
      for (int a = 0; a < A; ++a) {
        row[a] = angle[(long long)a * T + t];
        known = known && row[a] >= 0 && row[a] < L;
      }
    }
    int page = -1, slot = 0;
    if (known) {
      const I p = pages[(long long)seq * M + (int)pos / S];
      page = p >= 0 && p < P ? (int)p : -1;
      slot = (int)pos % S;
    }
    const int D = kind == 2 ? DV : DK, heads = kind == 0 ? HQ : HK;
    const X* in = (kind == 0 ? q : kind == 1 ? k : v) + t * heads * D;
    float c[NE], s[NE];
    const bool turns = R2 > 0 && L > 0 && known && kind < 2;
#pragma unroll
    for (int e = 0; e < NE; ++e) {
      c[e] = 1.0f;
      s[e] = 0.0f;
      if (turns && d + e < 2 * R2) {
        const int a = PAIRS ? (d + e) >> 1 : d + e < R2 ? d + e : d + e - R2;
        const I r = A == 1 || a < S0 ? row[0] : A == 2 || a < S1 ? row[A > 1 ? 1 : 0] : A == 3 || a < S2 ? row[A > 2 ? 2 : 0] : row[A > 3 ? 3 : 0];
        c[e] = cos[(long long)r * R2 + a];
        s[e] = sin[(long long)r * R2 + a];
      }
    }
#pragma unroll
    for (int n = 0; n < EACH; ++n) {
      const int head = first + n;
      if (head >= heads) break;
      const X* x = in + (long long)head * D;
      W own{}, other{};
      if constexpr (WHOLE) {
        if (d < D) own = rx_load<W>(x + d);
        if (!PAIRS && R2 > 0 && turns && d < 2 * R2) other = rx_load<W>(x + (d < R2 ? d + R2 : d - R2));
      } else {
#pragma unroll
        for (int e = 0; e < NE; ++e) {
          const int f = d + e;
          if (f < D) own.v[e] = x[f];
          if (turns && f < 2 * R2) other.v[e] = x[PAIRS ? f ^ 1 : f < R2 ? f + R2 : f - R2];
        }
      }
      float y[NE];
#pragma unroll
      for (int e = 0; e < NE; ++e) {
        const int f = d + e;
        const float a = E::up(own.v[e]), b = E::up(WHOLE && PAIRS ? own.v[e ^ 1] : other.v[e]);
        const bool second = PAIRS ? (f & 1) != 0 : f >= R2;
        y[e] = turns && f < 2 * R2 ? (second ? a * c[e] + b * s[e] : a * c[e] - b * s[e]) : a;
      }
      if (kind == 0 || !BITS8) {
        W o;
#pragma unroll
        for (int e = 0; e < NE; ++e) o.v[e] = kind == 0 && !known ? E::down(0.0f) : kind == 2 ? own.v[e] : E::down(y[e]);
        if (kind != 0 && page < 0) continue;
        // (of the cache only where it has the type of k)
        X* to = kind == 0 ? qo + (t * HQ + head) * DK
                          : (X*)(kind == 1 ? kc + rx_lm_slot<S, HK, DK, BY_SLOT>(page, slot, head) : vc + rx_lm_slot<S, HK, DV, BY_SLOT>(page, slot, head));
        if constexpr (WHOLE) {
          if (d < D) rx_store_nt(to + d, o);
        } else {
#pragma unroll
          for (int e = 0; e < NE; ++e)
            if (d + e < D) to[d + e] = o.v[e];
        }
      } else if constexpr (BITS8) {
        rx_u32 top = 0;
#pragma unroll
        for (int e = 0; e < NE; ++e) {
          const rx_u32 bits = d + e < D ? rx_f2u(y[e]) & 0x7fffffffu : 0u;
          top = bits > top ? bits : top;
        }
        if constexpr (LANES == 64) top = rx_wave_reduce(top, rx_lm_umax());
        else top = rx_group_reduce<LANES>(top, rx_lm_umax());
        if (page < 0) continue;
        const float scale = rx_lm_scale_of<C>(top);
        const rx_vec<rx_u8, NE> o = rx_lm_codes<C>(y, scale);
        rx_u8* to = kind == 1 ? kc + rx_lm_slot<S, HK, DK, BY_SLOT>(page, slot, head) : vc + rx_lm_slot<S, HK, DV, BY_SLOT>(page, slot, head);
        if constexpr (WHOLE) {
          if (d < D) rx_store_nt(to + d, o);
        } else {
#pragma unroll
          for (int e = 0; e < NE; ++e)
            if (d + e < D) to[d + e] = o.v[e];
        }
        if (lane == 0) (kind == 1 ? ks : vs)[rx_lm_slot<S, HK, 1, false>(page, slot, head)] = scale;
      }
    }
  }
}

// ---------------------------------------------------------------------------
// slots moved together: a thread takes the same bytes (a unit) of all of a sequence's steps, and loads them all before it stores the
// first, so that a slot may be moved from and moved to.
// ---------------------------------------------------------------------------
template <int S, typename U, int A, typename F, typename G>
RX_DEV void rx_lm_move(U* base, const int (&from)[A], const int (&to)[A], F page_of, G place) {
  U held[A];
#pragma unroll
  for (int a = 0; a < A; ++a)
    if (to[a] >= 0) held[a] = base[place(page_of(from[a]), from[a] % S)];
#pragma unroll
  for (int a = 0; a < A; ++a)
    if (to[a] >= 0) base[place(page_of(to[a]), to[a] % S)] = held[a];
}
template <typename U, int KU, int VU, int HK, int P, int S, int B, int M, int A, bool BY_SLOT, bool SCALES, typename I>
RX_DEV void rx_kv_move(const I* lengths, const I* path, const I* pages, U* kc, U* vc, float* ks, float* vs) {
  constexpr int UNITS = HK * (KU + VU) + (SCALES ? 2 * HK : 0);
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < (long long)B * UNITS; i += (long long)gridDim.x * 256) {
    const long long b = i / UNITS;
    const int u = (int)(i % UNITS);
    const I n = lengths[b];
    if (n < 0 || n >= (I)(M * S)) continue;
    int from[A], to[A];                                 // positions; -1: not moved
#pragma unroll
    for (int a = 0; a < A; ++a) {
      const I p = path[b * A + a];
      from[a] = to[a] = -1;
      if (p < 0 || p == a || p >= (I)(M * S) - n || a >= (I)(M * S) - n) continue;
      const int f = (int)(n + p), t = (int)n + a;
      const I fp = pages[b * M + f / S], tp = pages[b * M + t / S];
      if (fp < 0 || fp >= P || tp < 0 || tp >= P) continue;
      from[a] = f;
      to[a] = t;
    }
    auto page_of = [&](const int at) { return (long long)pages[b * M + at / S]; };
    if (u < HK * KU) rx_lm_move<S>(kc, from, to, page_of, [&](const long long page, const int slot) { return rx_lm_slot<S, HK, KU, BY_SLOT>(page, slot, u / KU) + u % KU; });
    else if (u < HK * (KU + VU))
      rx_lm_move<S>(vc, from, to, page_of, [&](const long long page, const int slot) { return rx_lm_slot<S, HK, VU, BY_SLOT>(page, slot, (u - HK * KU) / VU) + (u - HK * KU) % VU; });
    else if constexpr (SCALES) {
      const int h = u - HK * (KU + VU);
      rx_lm_move<S>(h < HK ? ks : vs, from, to, page_of, [&](const long long page, const int slot) { return rx_lm_slot<S, HK, 1, false>(page, slot, h % HK); });
    }
  }
}

// ---------------------------------------------------------------------------
// attention of drafted tokens
// ---------------------------------------------------------------------------
// As the attention of one token per sequence (rx_paged_attention): one pass with running maxima and sums, scores as K Q' and results
// as V' P' on the matrix cores, where the columns are rows of the result: (drafted token, query head) pairs of one key head, token
// by token.  A step is 32 positions.  Which rows see a position matters only in steps that hold drafted tokens or the window's edge.
struct rx_lm_tree_span : rx_lm_span { int prefix; };   // positions before the drafted tokens
template <int S, int B, int M, int N, int W, typename I>
RX_DEV rx_lm_tree_span rx_lm_tree_span_of(const I len) {
  rx_lm_tree_span s;
  s.prefix = len < 0 ? 0 : len > (I)(M * S) ? M * S : (int)len;
  s.n = len < 0 ? 0 : s.prefix + N < M * S ? s.prefix + N : M * S;
  s.lo = W && s.prefix > W ? s.prefix - W : 0;
  s.units = (s.n - (s.lo & ~31) + 31) >> 5;
  if (s.units == 0) s.units = 1;
  s.cost = s.units + (B > 1 ? 4 : 0);
  return s;
}

// N elements of a row from element d on as 32-bit words, zeros past its end
template <typename X, int D, int N, bool ONCE>
RX_DEV rx_vec<rx_u32, N * sizeof(X) / 4> rx_lm_part(const X* row, const int d) {
  constexpr int BYTES = N * sizeof(X);
  typedef rx_vec<rx_u32, BYTES / 4> R;
  R v{};
  if constexpr (D % N == 0) {
    if (d < D) v = ONCE ? rx_load_nt<R>(row + d) : rx_load<R>(row + d);
  } else {
    rx_vec<X, N> w{};
#pragma unroll
    for (int k = 0; k < N; ++k)
      if (d + k < D) w.v[k] = row[d + k];
    v = __builtin_bit_cast(R, w);
  }
  return v;
}
// two of a word's four numbers of 8 bits as bf16, which holds them exactly
template <typename C>
RX_DEV rx_u32 rx_lm_pair_up(const rx_u32 w, const bool high) {
  typedef __bf16 P __attribute__((ext_vector_type(2)));
  P p;
  if constexpr (__is_same(C, rx_lm_f8)) {
    p = high ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true) : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false);
  } else {
    p[0] = (__bf16)(float)(rx_i8)(w >> (high ? 16 : 0));
    p[1] = (__bf16)(float)(rx_i8)(w >> (high ? 24 : 8));
  }
  return __builtin_bit_cast(rx_u32, p);
}
// eight of them
template <typename C>
RX_DEV rx_u32x4 rx_lm_eight_up(const rx_u32 a, const rx_u32 b) {
  return rx_u32x4{rx_lm_pair_up<C>(a, false), rx_lm_pair_up<C>(a, true), rx_lm_pair_up<C>(b, false), rx_lm_pair_up<C>(b, true)};
}

// What the rows of a wavefront have seen: maxima, sums, unscaled results, for NT tiles of 16 rows.
// E: of the queries and the result, C: of the caches, F: of the products.  Caches of 8 bits are multiplied as bf16, which holds their numbers
// exactly; queries of more digits than bf16's go in as a sum of up to three bf16 (f16: two hold it exactly, f32: three leave 2^-24).
// KF: fragments of a key (16 bytes of its dimensions to each of four lanes), PERMUTED: in the order that 16 bytes of 8-bit numbers give.
template <typename E, typename C, int DK, int DV, int NT, bool PERMUTED>
struct rx_lm_tree {
  static constexpr bool BITS8 = rx_lm_is8<C>::value, WIDE = !BITS8 && sizeof(typename E::S) == 4;   // WIDE: products in f32
  typedef typename rx_lm_if<BITS8, rx_lm_bf16, E>::type F;
  static constexpr int NE = WIDE ? 4 : 8;                                                           // elements of a fragment
  static constexpr int KF = PERMUTED ? 2 * ((DK + 63) / 64) : (DK + 4 * NE - 1) / (4 * NE);
  static constexpr int VE = WIDE || DV <= 64 ? 4 : 8, NV = (DV + 16 * VE - 1) / (16 * VE);           // dimensions of a lane, times 16 lanes
  static constexpr int NQ = !BITS8 ? 1 : sizeof(typename E::S) == 4 ? 3 : E::BF16 ? 1 : 2;
  // weights enter the product as a sum of as many numbers: one alone is off by as much as the result's own rounding
  static constexpr int NP = WIDE ? 1 : sizeof(typename E::S) == 4 ? 3 : 2;
  static constexpr float SHIFT = !WIDE && !F::BF16 ? 15.0f : 0.0f;   // f16 weights are taken times 2^15: the smallest would be lost below 2^-24
  rx_u32x4 q[NT][NQ][KF];
  float m[NT], l[NT];
  rx_f32x4 acc[NT][NV][VE];

  RX_MEM void clear() {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      m[t] = -rx_lm_inf();
      l[t] = 0.0f;
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < VE; ++e) acc[t][j][e] = rx_f32x4{0, 0, 0, 0};
    }
  }
  // first dimension of fragment k in the lanes g4
  RX_MEM static int dim(const int k, const int g4) { return PERMUTED ? k / 2 * 64 + g4 * 16 + (k & 1) * 8 : (k * 4 + g4) * NE; }
  RX_MEM void load(const int t, const typename E::S* row, const bool there) {
    const int g4 = (threadIdx.x & 63) >> 4;
#pragma unroll
    for (int k = 0; k < KF; ++k) {
      if constexpr (!BITS8) {
        q[t][0][k] = there ? rx_lm_row16<E, DK>(row, dim(k, g4)) : rx_u32x4{0, 0, 0, 0};
      } else {
        rx_vec<rx_u16, 8> part[NQ];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float x = there && dim(k, g4) + e < DK ? E::up(row[dim(k, g4) + e]) : 0.0f;
          const bool finite = __builtin_fabsf(x) <= RX_LM_FLT_MAX;
#pragma unroll
          for (int n = 0; n < NQ; ++n) {
            part[n].v[e] = rx_f32_to_bf16(x);
            x = finite ? x - rx_bf16_to_f32(part[n].v[e]) : 0.0f;
          }
        }
#pragma unroll
        for (int n = 0; n < NQ; ++n) q[t][n][k] = __builtin_bit_cast(rx_u32x4, part[n]);
      }
    }
  }
  // One step.  kf: keys of positions r and 16 + r; value(j, e): dimension VE r + e (of 16 VE) of the eight positions 4 g4 + (0..3) and
  // 16 further as an operand; seen[t]: which of those eight the lane's row sees, where `some` do not; factor: of the scores;
  // ks, vs: the scales of the eight positions, ks times factor already.
  template <typename V>
  RX_MEM void step(const rx_u32x4 (&kf)[2][KF], V value, const bool some, const unsigned (&seen)[NT], const float factor, const float (&ks)[8], const float (&vs)[8]) {
    rx_u32x4 w[NT][NP];                                   // 16-bit weights of the eight positions
    float wide[NT][8];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      rx_f32x4 s[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
      for (int n = 0; n < NQ; ++n)
#pragma unroll
        for (int k = 0; k < KF; ++k) {
          s[0] = rx_lm_mma<F>(kf[0][k], q[t][n][k], s[0]);
          s[1] = rx_lm_mma<F>(kf[1][k], q[t][n][k], s[1]);
        }
      float x[8], top = -rx_lm_inf();
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = s[i >> 2][i & 3] * (BITS8 ? ks[i] : factor);
      // (not below the lowest number: a maximum of -inf says that there was no position)
      if (some) {
#pragma unroll
        for (int i = 0; i < 8; ++i) top = __builtin_fmaxf(top, (seen[t] >> i) & 1u ? __builtin_fmaxf(x[i], -RX_LM_FLT_MAX) : -rx_lm_inf());
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) top = __builtin_fmaxf(top, x[i]);
        top = __builtin_fmaxf(top, -RX_LM_FLT_MAX);
      }
      top = __builtin_fmaxf(m[t], rx_lm_max4(top));
      if (__any(top != m[t])) {
        const float shrink = top == m[t] ? 1.0f : __builtin_amdgcn_exp2f(m[t] - top);
        l[t] *= shrink;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int e = 0; e < VE; ++e) acc[t][j][e] *= shrink;
        m[t] = top;
      }
      float p[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) p[i] = __builtin_amdgcn_exp2f(x[i] - top + SHIFT);
      if (some) {
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = (seen[t] >> i) & 1u ? p[i] : 0.0f;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) l[t] += p[i];
      if constexpr (BITS8) {
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = some && !((seen[t] >> i) & 1u) ? 0.0f : p[i] * vs[i];
      }
      if constexpr (WIDE) {
#pragma unroll
        for (int i = 0; i < 8; ++i) wide[t][i] = p[i];
      } else {
#pragma unroll
        for (int n = 0; n < NP; ++n) {
          rx_vec<rx_u16, 8> o;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            o.v[i] = F::down(p[i]);
            if (n + 1 < NP) p[i] -= F::up(o.v[i]);
          }
          w[t][n] = __builtin_bit_cast(rx_u32x4, o);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        const rx_u32x4 a0 = value(j, e, 0);
        const rx_u32x4 a1 = WIDE ? value(j, e, 1) : a0;    // (f32: positions 4 .. 7)
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          if constexpr (WIDE) {
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[t][j][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(rx_u2f((i < 4 ? a0 : a1)[i & 3]), wide[t][i], acc[t][j][e], 0, 0, 0);
          } else {
#pragma unroll
            for (int n = 0; n < NP; ++n) acc[t][j][e] = rx_lm_mma<F>(a0, w[t][n], acc[t][j][e]);
          }
        }
      }
  }
  // Infinities and NaN among the values of a step that some rows do not see (a weight of zero would make them NaN there): they are
  // taken out of the values before the step, and added here to the rows that see them.  at(p, d): value of position p (of 32).
  template <typename A>
  RX_MEM void add_special(const unsigned (&seen)[NT], A at) {
    const int r = threadIdx.x & 15, g4 = (threadIdx.x & 63) >> 4;
    for (int p = 0; p < 32; ++p) {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const unsigned bits = rx_lane_from(seen[t], (((p >> 2) & 3) << 4) + r);
        const bool sees = (bits >> ((p >> 4) * 4 + (p & 3))) & 1u;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int e = 0; e < VE; ++e)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int d = (j * 16 + g4 * 4 + i) * VE + e;
              const float v = sees && d < DV ? at(p, d) : 0.0f;
              if (!(__builtin_fabsf(v) <= RX_LM_FLT_MAX)) acc[t][j][e][i] += v;
            }
      }
    }
  }
};

// bits of a word's numbers that are infinite or NaN
template <typename X>
RX_DEV rx_u32 rx_lm_special(const rx_u32 w) {
  if constexpr (__is_same(X, rx_lm_i8)) {
    return 0;
  } else if constexpr (__is_same(X, rx_lm_f8)) {
    rx_u32 o = 0;
#pragma unroll
    for (int b = 0; b < 32; b += 8) o |= ((w >> b) & 0x7fu) == 0x7fu ? 0xffu << b : 0u;
    return o;
  } else if constexpr (sizeof(typename X::S) == 4) {
    return (w & 0x7f800000u) == 0x7f800000u ? ~0u : 0u;
  } else {
    constexpr rx_u32 e = X::BF16 ? 0x7f80u : 0x7c00u;
    return ((w & e) == e ? 0xffffu : 0u) | (((w >> 16) & e) == e ? 0xffff0000u : 0u);
  }
}

// MASK: 0 every drafted token sees itself and those before it, 2 [N, N] for all sequences, 3 [B, N, N].  NT: tiles of 16 rows to a
// wavefront.  WR: wavefronts that have rows of their own: 1 (few rows) the four share the positions, and read the caches into their
// registers; 4 (many rows) they share keys and values, which pass through LDS, 8-bit numbers as bf16, the next step's being loaded
// while this one's are multiplied.  R, HW, ONCE, DIES, Q: as for rx_paged_attention.
template <typename E, typename C, int N, int HQ, int HK, int DK, int DV, int P, int S, int B, int M, int W, bool BY_SLOT, int MASK, int NT, int WR, int R, int HW, bool ONCE, bool DIES,
          int Q, typename I>
RX_DEV void rx_tree_attention(const typename E::S* q, const typename C::S* kc, const typename C::S* vc, const I* pages, const I* lengths, const rx_u8* mask, const float* ks,
                              const float* vs, typename E::S* out, float* lse, float* part, float* stat, int* arrived, const float scale) {
  constexpr bool SHARED = WR > 1, BITS8 = rx_lm_is8<C>::value;
  typedef rx_lm_tree<E, C, DK, DV, NT, BITS8 && !SHARED> A;
  typedef typename A::F F;
  typedef typename C::S T;
  constexpr int G = HQ / HK, ROWS = N * G, TR = 16 * NT * WR, RT = ROWS < TR ? ROWS : TR, TILES = (ROWS + TR - 1) / TR, COLUMNS = HK / HW * TILES, WPH = 4 / HW;
  constexpr int KF = A::KF, VE = A::VE, NV = A::NV;
  constexpr int BLOCK = 2048;                          // positions whose pages are held in LDS
  constexpr int HR = RT < 16 ? RT : 16, WIDTH = 16 * VE < DV ? 16 * VE : DV;   // rows and dimensions that are joined at a time
  constexpr int VD = DV % 4 == 0 ? 4 : 1;
  constexpr int FE = 16 / sizeof(typename F::S), KP = KF * 4 * A::NE + FE, VP = NV * 16 * VE + FE;   // rows of keys and values in LDS: 16 bytes longer, for its banks
  typedef rx_vec<rx_u32, VE * sizeof(typename F::S) / 4> FV;   // a lane's part of a value
  __shared__ union {
    int page[SHARED ? 1 : BLOCK / S + 2];
    float o[SHARED ? 1 : 4][HR][WIDTH + 4];
    rx_lm_joined<VD> j[256];
  } lds;
  __shared__ float join_m[4][16], join_l[4][16];
  __shared__ __attribute__((aligned(16))) typename F::S kt[SHARED ? 2 : 1][SHARED ? 32 : 1][SHARED ? KP : FE];
  __shared__ __attribute__((aligned(16))) typename F::S vt[SHARED ? 2 : 1][SHARED ? 32 : 1][SHARED ? VP : FE];
  __shared__ float st_k[2][32], st_v[2][32];
  __shared__ unsigned st_ok[2];
  __shared__ int last;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, r = lane & 15, g4 = lane >> 4;
  const int id = DIES ? (int)rx_xcd_remap(blockIdx.x, R * COLUMNS) : (int)blockIdx.x, column = id % COLUMNS, mine = id / COLUMNS, tile = column % TILES;
  const int head0 = column / TILES * HW, head = head0 + (SHARED ? 0 : wave / WPH);
  const int row0 = tile * TR + (SHARED ? wave * 16 * NT : 0);                 // first row of this wavefront
  const int rows = ROWS - tile * TR < TR ? ROWS - tile * TR : TR;             // of the workgroup
  const rx_lm_stretch st = rx_lm_stretch_of<B, R, Q>([&](const int at) { return rx_lm_tree_span_of<S, B, M, N, W>(lengths[at]).cost; }, mine);
  auto result_of = [&](const int b, const int row, const int h) { return ((long long)b * N + row / G) * HQ + h * G + row % G; };   // row of the results
  int buf = 0;
  if constexpr (SHARED && (DK + FE - 1) / FE * FE < KF * 4 * A::NE) {          // what no chunk of a key covers
    for (int i = threadIdx.x; i < 64 * KP; i += 256) (&kt[0][0][0])[i] = F::down(0.0f);
    __syncthreads();
  }

  int b = st.b, unit = st.unit;
  for (int left = st.count; left > 0; ++b, unit = 0) {
  const rx_lm_tree_span span = rx_lm_tree_span_of<S, B, M, N, W>(lengths[b]);
  const int step = span.cost - unit < left ? span.cost - unit : left, take = span.units - unit < step ? span.units - unit : step;
  const long long begin = st.first + (st.count - left) - unit;                // the sequence's first unit in the row
  left -= step;
  if (take <= 0) continue;
  const int p0 = (span.lo & ~31) + unit * 32, p1 = P == 0 ? p0 : p0 + take * 32 < span.n ? p0 + take * 32 : span.n;
  const bool whole = take == span.units;                                      // the whole sequence is in this stretch
  A a;
  a.clear();
  int token[NT], first[NT];                                                   // of the lane's rows: the drafted token, and the first position of the prefix that it sees
  bool inside[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int row = row0 + t * 16 + r;
    inside[t] = row < ROWS;
    token[t] = inside[t] ? row / G : 0;
    first[t] = 0;
    a.load(t, q + result_of(b, inside[t] ? row : 0, head) * DK, inside[t]);
    if constexpr (W > 0) {                                                    // the window's last places are taken by the drafted tokens that it sees
      int sees = 0;
      if constexpr (MASK == 0) sees = token[t] + 1;
      else
        for (int j = 0; j < N; ++j) sees += mask[((long long)(MASK == 3 ? b : 0) * N + token[t]) * N + j] != 0;
      first[t] = span.prefix - (W - sees) > 0 ? span.prefix - (W - sees) : 0;
    }
  }
  const int edge = W > 0 && span.prefix - W + N > 0 ? span.prefix - W + N : 0;   // every row sees the prefix from here on
  // bits of the lane's eight positions of a step that its rows see
  auto seen_by = [&](const int t0, const unsigned ok, unsigned (&seen)[NT]) {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      seen[t] = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int at = (i & 4) * 4 + g4 * 4 + (i & 3), p = t0 + at, j = p - span.prefix;
        bool see = (ok >> at) & 1u;
        if (see) {
          if (j < 0) see = p >= first[t];
          else if constexpr (MASK == 0) see = j <= token[t];
          else see = mask[((long long)(MASK == 3 ? b : 0) * N + token[t]) * N + j] != 0;
        }
        seen[t] |= see ? 1u << i : 0u;
      }
    }
  };
  auto some_of = [&](const int t0, const unsigned ok) { return ok != ~0u || t0 + 32 > span.prefix || (W > 0 && t0 < edge); };

  if constexpr (!SHARED) {
    constexpr int KR = BITS8 ? (DK + 63) / 64 : KF;    // 16-byte loads of a key by its four lanes
    typedef rx_vec<rx_u32, VE * sizeof(T) / 4> CV;
    for (int s0 = p0; s0 < p1; s0 += BLOCK) {
      const int s1 = s0 + BLOCK < p1 ? s0 + BLOCK : p1;
      const int page0 = s0 / S, npages = (s1 - 1) / S - page0 + 1;
      __syncthreads();
      for (int i = threadIdx.x; i < npages; i += 256) {
        const I page = pages[(long long)b * M + page0 + i];
        lds.page[i] = page >= 0 && page < P ? (int)page : -1;
      }
      __syncthreads();
      // page of a position, -1 where it is not to be looked at
      auto where = [&](const int t) { return t >= span.lo && t < s1 ? lds.page[t / S - page0] : -1; };
      for (int t0 = s0 + wave % WPH * 32; t0 < s1; t0 += WPH * 32) {
        const int ta = t0 + r, tb = ta + 16, pa = where(ta), pb = where(tb);
        const unsigned ok = ((unsigned)__ballot(pa >= 0) & 0xffffu) | ((unsigned)__ballot(pb >= 0) << 16);
        if (!ok) continue;
        rx_vec<rx_u32, 4> raw[2][KR];
        const T* ka = kc + rx_lm_slot<S, HK, DK, BY_SLOT>(pa < 0 ? 0 : pa, ta % S, head);
        const T* kb = kc + rx_lm_slot<S, HK, DK, BY_SLOT>(pb < 0 ? 0 : pb, tb % S, head);
#pragma unroll
        for (int k = 0; k < KR; ++k) {
          raw[0][k] = rx_lm_part<T, DK, 16 / sizeof(T), ONCE>(ka, (k * 4 + g4) * (16 / sizeof(T)));
          raw[1][k] = rx_lm_part<T, DK, 16 / sizeof(T), ONCE>(kb, (k * 4 + g4) * (16 / sizeof(T)));
        }
        // values of positions t0 + 4 g4 + (0..3) and 16 further: where a page's slots are a multiple of four, on two pages
        CV vf[NV][8];
        float kscale[8] = {}, vscale[8] = {};
        int pv = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int tv = t0 + (i & 4) * 4 + g4 * 4 + (i & 3);
          if (S % 4 != 0 || i % 4 == 0) {
            pv = where(S % 4 == 0 ? (tv + 3 < s1 ? tv + 3 : s1 - 1) : tv);   // (the group's first positions may lie before span.lo)
            if (S % 4 == 0 && tv >= s1) pv = -1;
          }
          const T* v = vc + rx_lm_slot<S, HK, DV, BY_SLOT>(pv < 0 ? 0 : pv, tv % S, head);
#pragma unroll
          for (int j = 0; j < NV; ++j) vf[j][i] = rx_lm_part<T, DV, VE, ONCE>(v, (j * 16 + r) * VE);
          if constexpr (BITS8) {
            const long long at = rx_lm_slot<S, HK, 1, false>(pv < 0 ? 0 : pv, tv % S, head);
            if constexpr (S % 4 == 0) {
              if (i % 4 == 0) {
                const rx_vec<float, 4> x = rx_load<rx_vec<float, 4>>(ks + at), y = rx_load<rx_vec<float, 4>>(vs + at);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  kscale[i + e] = x.v[e] * scale;
                  vscale[i + e] = y.v[e];
                }
              }
            } else {
              kscale[i] = ks[at] * scale;
              vscale[i] = vs[at];
            }
          }
        }
        const unsigned there = (ok >> (g4 * 4)) & 0x000f000fu;   // bit i: position 4 g4 + i, bit 16 + i: 16 further
        if (ok != ~0u) {
          // what lies in other slots may be anything, and NaN times a weight of zero is not zero
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (!((there >> ((i & 4) * 4 + (i & 3))) & 1u)) {
#pragma unroll
              for (int j = 0; j < NV; ++j) vf[j][i] = CV{};
            }
        }
        unsigned seen[NT] = {};
        rx_u32 special = 0;
        const bool some = some_of(t0, ok);
        if (some) {
          seen_by(t0, ok, seen);
#pragma unroll
          for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
              for (int n = 0; n < (int)(sizeof(CV) / 4); ++n) {
                const rx_u32 x = rx_lm_special<C>(vf[j][i].v[n]);
                vf[j][i].v[n] &= ~x;
                special |= x;
              }
        }
        rx_u32x4 kf[2][KF];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int k = 0; k < KF; ++k) {
            if constexpr (BITS8) kf[h][k] = rx_lm_eight_up<C>(raw[h][k / 2].v[k % 2 * 2], raw[h][k / 2].v[k % 2 * 2 + 1]);
            else kf[h][k] = __builtin_bit_cast(rx_u32x4, raw[h][k]);
          }
        a.step(kf, [&](const int j, const int e, const int half) {
          rx_u32x4 o;
          if constexpr (A::WIDE) {
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = vf[j][half * 4 + i].v[e];
          } else if constexpr (BITS8) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              o[k] = rx_lm_pair_up<C>(__builtin_amdgcn_perm(vf[j][2 * k + 1].v[e >> 2], vf[j][2 * k].v[e >> 2], e & 2 ? 0x07030602u : 0x05010400u), e & 1);
          } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) o[k] = __builtin_amdgcn_perm(vf[j][2 * k + 1].v[e >> 1], vf[j][2 * k].v[e >> 1], e & 1 ? 0x07060302u : 0x05040100u);
          }
          return o;
        }, some, seen, scale, kscale, vscale);
        if (some && __any(special != 0)) {
          a.add_special(seen, [&](const int p, const int d) {
            const int page = where(t0 + p);
            return page < 0 ? 0.0f : C::up(vc[rx_lm_slot<S, HK, DV, BY_SLOT>(page, (t0 + p) % S, head) + d]);
          });
        }
      }
    }
  } else {
    constexpr int CE = 16 / sizeof(T), CK = (DK + CE - 1) / CE, CV = (DV + CE - 1) / CE, LK = (32 * CK + 255) / 256, LV = (32 * CV + 255) / 256;
    rx_vec<rx_u32, 4> rk[LK], rv[LV];
    int pk[LK], pv[LV], ps = -1;                        // pages of the next step's loads; of position threadIdx.x
    float sk = 0.0f, sv = 0.0f;
    bool there = false;
    auto page_of = [&](const int t) {
      if (t < span.lo || t >= p1) return -1;
      const I page = pages[(long long)b * M + t / S];
      return page >= 0 && page < P ? (int)page : -1;
    };
    auto find = [&](const int t0) {
#pragma unroll
      for (int n = 0; n < LK; ++n) pk[n] = n * 256 + (int)threadIdx.x < 32 * CK ? page_of(t0 + (n * 256 + (int)threadIdx.x) / CK) : -1;
#pragma unroll
      for (int n = 0; n < LV; ++n) pv[n] = n * 256 + (int)threadIdx.x < 32 * CV ? page_of(t0 + (n * 256 + (int)threadIdx.x) / CV) : -1;
      ps = threadIdx.x < 32 ? page_of(t0 + (int)threadIdx.x) : -1;
    };
    auto fetch = [&](const int t0) {
#pragma unroll
      for (int n = 0; n < LK; ++n) {
        const int i = n * 256 + (int)threadIdx.x, t = t0 + i / CK;
        rk[n] = rx_vec<rx_u32, 4>{};
        if (pk[n] >= 0) rk[n] = rx_lm_part<T, DK, CE, ONCE>(kc + rx_lm_slot<S, HK, DK, BY_SLOT>(pk[n], t % S, head), i % CK * CE);
      }
#pragma unroll
      for (int n = 0; n < LV; ++n) {
        const int i = n * 256 + (int)threadIdx.x, t = t0 + i / CV;
        rv[n] = rx_vec<rx_u32, 4>{};
        if (pv[n] >= 0) rv[n] = rx_lm_part<T, DV, CE, ONCE>(vc + rx_lm_slot<S, HK, DV, BY_SLOT>(pv[n], t % S, head), i % CV * CE);
      }
      there = ps >= 0;
      if constexpr (BITS8) {
        sk = there ? ks[rx_lm_slot<S, HK, 1, false>(ps, (t0 + (int)threadIdx.x) % S, head)] * scale : 0.0f;
        sv = there ? vs[rx_lm_slot<S, HK, 1, false>(ps, (t0 + (int)threadIdx.x) % S, head)] : 0.0f;
      }
    };
    auto store = [&](typename F::S* to, const rx_vec<rx_u32, 4>& x) {
      if constexpr (BITS8) {
        *(rx_u32x4*)to = rx_lm_eight_up<C>(x.v[0], x.v[1]);
        *(rx_u32x4*)(to + 8) = rx_lm_eight_up<C>(x.v[2], x.v[3]);
      } else {
        *(rx_u32x4*)to = __builtin_bit_cast(rx_u32x4, x);
      }
    };
    if (p0 < p1) {
      find(p0);
      fetch(p0);
      find(p0 + 32);
    }
    for (int t0 = p0; t0 < p1; t0 += 32, buf ^= 1) {
#pragma unroll
      for (int n = 0; n < LK; ++n) {
        const int i = n * 256 + (int)threadIdx.x;
        if (LK * 256 == 32 * CK || i < 32 * CK) store(&kt[buf][i / CK][i % CK * CE], rk[n]);
      }
#pragma unroll
      for (int n = 0; n < LV; ++n) {
        const int i = n * 256 + (int)threadIdx.x;
        if (LV * 256 == 32 * CV || i < 32 * CV) store(&vt[buf][i / CV][i % CV * CE], rv[n]);
      }
      if (wave == 0) {
        const unsigned long long all = __ballot(there);
        if (lane == 0) st_ok[buf] = (unsigned)all;
        if (BITS8 && lane < 32) {
          st_k[buf][lane] = sk;
          st_v[buf][lane] = sv;
        }
      }
      __syncthreads();      // (the other buffer's readers have arrived here before it is written again)
      if (t0 + 32 < p1) {
        fetch(t0 + 32);
        find(t0 + 64);
      }
      const unsigned ok = st_ok[buf];
      if (!ok || row0 >= ROWS) continue;
      rx_u32x4 kf[2][KF];
      FV vf[NV][8];
      float kscale[8] = {}, vscale[8] = {};
#pragma unroll
      for (int k = 0; k < KF; ++k) {
        kf[0][k] = *(const rx_u32x4*)&kt[buf][r][(k * 4 + g4) * A::NE];
        kf[1][k] = *(const rx_u32x4*)&kt[buf][16 + r][(k * 4 + g4) * A::NE];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < NV; ++j) vf[j][i] = *(const FV*)&vt[buf][(i & 4) * 4 + g4 * 4 + (i & 3)][(j * 16 + r) * VE];
      if constexpr (BITS8) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          kscale[i] = st_k[buf][(i & 4) * 4 + g4 * 4 + (i & 3)];
          vscale[i] = st_v[buf][(i & 4) * 4 + g4 * 4 + (i & 3)];
        }
      }
      unsigned seen[NT] = {};
      rx_u32 special = 0;
      const bool some = some_of(t0, ok);
      if (some) {
        seen_by(t0, ok, seen);
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
          for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int n = 0; n < (int)(sizeof(FV) / 4); ++n) {
              const rx_u32 x = (j * 16 + r) * VE < DV ? rx_lm_special<F>(vf[j][i].v[n]) : ~0u;
              vf[j][i].v[n] &= ~x;
              special |= (j * 16 + r) * VE < DV ? x : 0u;
            }
      }
      a.step(kf, [&](const int j, const int e, const int half) {
        rx_u32x4 o;
        if constexpr (A::WIDE) {
#pragma unroll
          for (int i = 0; i < 4; ++i) o[i] = vf[j][half * 4 + i].v[e];
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k) o[k] = __builtin_amdgcn_perm(vf[j][2 * k + 1].v[e >> 1], vf[j][2 * k].v[e >> 1], e & 1 ? 0x07060302u : 0x05040100u);
        }
        return o;
      }, some, seen, scale, kscale, vscale);
      if (some && __any(special != 0)) a.add_special(seen, [&](const int p, const int d) { return F::up(vt[buf][p][d]); });
    }
  }

  if constexpr (!SHARED) {
    // the four wavefronts' parts
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      if (t * 16 >= rows) break;
      const float total = rx_lm_sum4(a.l[t]);
      __syncthreads();
      if (g4 == 0) {
        join_m[wave][r] = a.m[t];
        join_l[wave][r] = total;
      }
      __syncthreads();
      float top = -rx_lm_inf();
#pragma unroll
      for (int w = 0; w < WPH; ++w) top = __builtin_fmaxf(top, join_m[wave / WPH * WPH + w][r]);
      const float f = top == -rx_lm_inf() ? 0.0f : __builtin_amdgcn_exp2f(a.m[t] - top);
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if (j) __syncthreads();
        if (r < HR) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < VE; ++e) {
              const int d = (g4 * 4 + i) * VE + e;
              if (d < WIDTH) lds.o[wave][r][d] = a.acc[t][j][e][i] * f;
            }
        }
        __syncthreads();
        for (int k = threadIdx.x; k < HW * HR * WIDTH; k += 256) {
          const int hw = k / (HR * WIDTH), h = k / WIDTH % HR, d = j * 16 * VE + k % WIDTH, row = t * 16 + h;
          if (row >= rows || d >= DV) continue;
          float o = 0.0f, sum = 0.0f, hi = -rx_lm_inf();
#pragma unroll
          for (int i = 0; i < WPH; ++i) hi = __builtin_fmaxf(hi, join_m[hw * WPH + i][h]);
#pragma unroll
          for (int i = 0; i < WPH; ++i) {
            const int w = hw * WPH + i;
            o += lds.o[w][h][k % WIDTH];
            sum += hi == -rx_lm_inf() ? 0.0f : join_l[w][h] * __builtin_amdgcn_exp2f(join_m[w][h] - hi);
          }
          if (whole) {
            const long long at = result_of(b, tile * TR + row, head0 + hw);
            out[at * DV + d] = E::down(hi == -rx_lm_inf() ? 0.0f : o / sum);
            if (lse && d == 0) lse[at] = hi == -rx_lm_inf() ? -rx_lm_inf() : (hi - A::SHIFT + __builtin_log2f(sum)) * 0.6931471805599453f;
          } else {
            const long long at = (((long long)id * 2 + (unit == 0)) * HW + hw) * RT + row;
            rx_lm_put_shared(part + at * DV + d, o);
            if (d == 0) {
              rx_lm_put_shared(stat + at * 2, hi - A::SHIFT);
              rx_lm_put_shared(stat + at * 2 + 1, sum);
            }
          }
        }
      }
    }
  } else {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const float sum = rx_lm_sum4(a.l[t]), hi = a.m[t];
      if (!inside[t]) continue;
      const int row = row0 + t * 16 + r - tile * TR;
      const long long at = whole ? result_of(b, tile * TR + row, head) : ((long long)id * 2 + (unit == 0)) * RT + row;
      if (g4 == 0) {
        if (!whole) {
          rx_lm_put_shared(stat + at * 2, hi - A::SHIFT);
          rx_lm_put_shared(stat + at * 2 + 1, sum);
        } else if (lse) {
          lse[at] = hi == -rx_lm_inf() ? -rx_lm_inf() : (hi - A::SHIFT + __builtin_log2f(sum)) * 0.6931471805599453f;
        }
      }
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int e = 0; e < VE; ++e) {
            const int d = (j * 16 + g4 * 4 + i) * VE + e;
            if (d >= DV) continue;
            if (whole) out[at * DV + d] = E::down(hi == -rx_lm_inf() ? 0.0f : a.acc[t][j][e][i] / sum);
            else rx_lm_put_shared(part + at * DV + d, a.acc[t][j][e][i]);
          }
    }
  }
  if (whole) continue;
  const int from = rx_lm_stretch_with(st.total, st.parts, begin), to = rx_lm_stretch_with(st.total, st.parts, begin + span.units - 1);
  if (!rx_lm_last_to_arrive(arrived + b * COLUMNS + column, to - from + 1, &last)) continue;
  // VD outputs to a thread, DV / VD apart, so that lanes read consecutive words; where there are fewer than threads, the parts are
  // shared too, and joined once more
  const int outs = HW * rows * (DV / VD), ways = outs < 256 ? 256 / outs : 1, parts = to - from + 1;
  for (int k0 = 0; k0 < outs; k0 += 256) {
    const int k = ways > 1 ? (int)threadIdx.x % outs : k0 + (int)threadIdx.x, way = ways > 1 ? (int)threadIdx.x / outs : 0;
    const bool on = k < outs && way < ways;
    const int hw = k / (rows * (DV / VD)), h = k / (DV / VD) % rows, d = k % (DV / VD);
    const int w1 = on ? from + parts * (way + 1) / ways : 0;
    rx_lm_joined<VD> j = {-rx_lm_inf(), 0.0f, {}};
    for (int w = on ? from + parts * way / ways : 0; w < w1; w += 8) {
      float pm[8], psum[8], po[8][VD];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int v = w + i < w1 ? w + i : w1 - 1;
        const long long at = (((long long)(v * COLUMNS + column) * 2 + (v == from)) * HW + hw) * RT + h;
        pm[i] = rx_lm_get_shared(stat + at * 2);
        psum[i] = rx_lm_get_shared(stat + at * 2 + 1);
#pragma unroll
        for (int e = 0; e < VD; ++e) po[i][e] = rx_lm_get_shared(part + at * DV + d + e * (DV / VD));
      }
      float hi = j.m;
#pragma unroll
      for (int i = 0; i < 8; ++i) hi = __builtin_fmaxf(hi, pm[i]);
      j.to(hi);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (w + i < w1) j.add(pm[i], psum[i], po[i]);
    }
    if (ways > 1) {
      lds.j[threadIdx.x] = j;
      __syncthreads();
      if (way == 0)
        for (int n = 1; n < ways; ++n) {
          const rx_lm_joined<VD> o = lds.j[n * outs + k];
          j.to(__builtin_fmaxf(j.m, o.m));
          j.add(o.m, o.s, o.o);
        }
    }
    if (!on || way) continue;
    const long long at = result_of(b, tile * TR + h, head0 + hw);
#pragma unroll
    for (int e = 0; e < VD; ++e) out[at * DV + d + e * (DV / VD)] = E::down(j.m == -rx_lm_inf() ? 0.0f : j.o[e] / j.s);
    if (lse && d == 0) lse[at] = j.m == -rx_lm_inf() ? -rx_lm_inf() : (j.m + __builtin_log2f(j.s)) * 0.6931471805599453f;
  }
  }
}
