// Device code of paged caches that may hold 8 bits: written by positions of several axes, slots moved together, and attention of
// drafted tokens (csrc/rx_lm.h states what they compute).
#pragma once
#include "rx_lm_norm_kernels.h"

template <bool B, typename X, typename Y> struct rx_lm_if { typedef X type; };
template <typename X, typename Y> struct rx_lm_if<false, X, Y> { typedef Y type; };
constexpr int rx_lm_pow2(const int n) { return n <= 1 ? 1 : 2 * rx_lm_pow2((n + 1) / 2); }

// the row of the angles that pair a is turned by: of the axis whose section holds it
template <int A, int S0, int S1, int S2, typename I>
RX_DEV I rx_lm_axis_row(const int a, const I r0, const I r1, const I r2, const I r3) {
  I r = r0;
  if constexpr (A > 1) r = a < S0 ? r : r1;
  if constexpr (A > 2) r = a < S1 ? r : r2;
  if constexpr (A > 3) r = a < S2 ? r : r3;
  return r;
}
// A token's heads, EACH of them after one another, to a group of LANES lanes, NE elements of 16 bytes to a lane: what a head's
// largest magnitude is found over, and what the cosines and sines of its dimensions are loaded for once.  Every lane loads the
// pairs' other elements itself.  8191 tokens of 32 and 8 heads of 128 in bf16 into 8 bits, 189 MB, take 38.6 us, 4.9 TB/s, with inputs in the
// last-level cache, and 47 us from memory: the index arithmetic and the divisions take about half of the vector units' time.  48 tokens take 3.4 us, a launch and four dependent loads.
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
  // (32 bits where they count all groups: a division of 64 is a dozen operations more)
  typedef typename rx_lm_if<((long long)T * ALL < (1ll << 30)), rx_u32, rx_u64>::type Z;
  for (Z i = (Z)(((rx_u64)blockIdx.x * 256 + threadIdx.x) / LANES); i < (Z)T * ALL; i += (Z)gridDim.x * (256 / LANES)) {
    const long long t = (long long)(i / ALL);
    const int u = (int)(i % ALL), kind = u < GQ ? 0 : u < GQ + GK ? 1 : 2, first = (u - (kind == 0 ? 0 : kind == 1 ? GQ : GQ + GK)) * EACH;
    const I pos = position[t], seq = sequence[t];
    bool known = pos >= 0 && pos < (I)(M * S) && seq >= 0 && seq < B;
    I row0 = 0, row1 = 0, row2 = 0, row3 = 0;
    if constexpr (R2 > 0) {
      row0 = angle[t];
      if constexpr (A > 1) row1 = angle[(long long)T + t];
      if constexpr (A > 2) row2 = angle[2ll * T + t];
      if constexpr (A > 3) row3 = angle[3ll * T + t];
      auto inside = [&](const I r) { return r >= 0 && r < L; };
      known = known && inside(row0) && (A < 2 || inside(row1)) && (A < 3 || inside(row2)) && (A < 4 || inside(row3));
    }
    int page = -1, slot = 0;
    if (known) {
      const I p = pages[(long long)seq * M + (rx_u32)pos / S];
      page = p >= 0 && p < P ? (int)p : -1;
      slot = (int)((rx_u32)pos % S);
    }
    const int D = kind == 2 ? DV : DK, heads = kind == 0 ? HQ : HK;
    const X* in = (kind == 0 ? q : kind == 1 ? k : v) + t * heads * D;
    float c[NE], s[NE];
    const bool turns = R2 > 0 && L > 0 && known && kind < 2;
    auto axis_row = [row0, row1, row2, row3](const int a) { return rx_lm_axis_row<A, S0, S1, S2>(a, row0, row1, row2, row3); };
    // Sections of at least a lane's pairs: they lie in at most two of them, and come from the rows of the first and the last (8191 tokens of three axes
    // 43.8 -> 38.6 us, together with 32-bit indices).
    constexpr int NP = PAIRS ? NE / 2 : NE;
    constexpr bool TWO = WHOLE && R2 % 4 == 0 && NP % 4 == 0 && (A < 2 || (S0 >= NP && (A < 3 ? R2 - S0 : S1 - S0) >= NP)) && (A < 3 || (A < 4 ? R2 - S1 : S2 - S1) >= NP) && (A < 4 || R2 - S2 >= NP);
#pragma unroll
    for (int e = 0; e < NE; ++e) {
      c[e] = 1.0f;
      s[e] = 0.0f;
    }
    if constexpr (TWO) {
      if (turns && d < 2 * R2) {
        typedef rx_vec<float, 4> Q;
        const int a0 = PAIRS ? d >> 1 : d < R2 ? d : d - R2;
        const I r0 = axis_row(a0), r1 = axis_row(a0 + NP - 1);
        Q v[2][2][NP / 4];
#pragma unroll
        for (int k = 0; k < NP / 4; ++k) {
          v[0][0][k] = rx_load<Q>(cos + (long long)r0 * R2 + a0 + 4 * k);
          v[0][1][k] = rx_load<Q>(sin + (long long)r0 * R2 + a0 + 4 * k);
          if constexpr (A > 1) {
            v[1][0][k] = rx_load<Q>(cos + (long long)r1 * R2 + a0 + 4 * k);
            v[1][1][k] = rx_load<Q>(sin + (long long)r1 * R2 + a0 + 4 * k);
          }
        }
#pragma unroll
        for (int e = 0; e < NE; ++e) {
          const int p = PAIRS ? e / 2 : e;
          c[e] = v[0][0][p / 4].v[p % 4];
          s[e] = v[0][1][p / 4].v[p % 4];
          if constexpr (A > 1) {
            const bool last = axis_row(a0 + p) != r0;
            c[e] = last ? v[1][0][p / 4].v[p % 4] : c[e];
            s[e] = last ? v[1][1][p / 4].v[p % 4] : s[e];
          }
        }
      }
    } else {
#pragma unroll
      for (int e = 0; e < NE; ++e)
        if (turns && d + e < 2 * R2) {
          const int a = PAIRS ? (d + e) >> 1 : d + e < R2 ? d + e : d + e - R2;
          const I r = axis_row(a);
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
// first, so that a slot may be moved from and moved to.  A chain of four dependent loads and a store: 48 sequences of 5 steps in 8 bits
// (0.4 MB) 5.0 us, 256 of 16 steps in bf16 (16 MB) 6.9; with the page table read once more for the addresses 7.4 and 11.7.
// ---------------------------------------------------------------------------
template <int S, typename U, int A, typename G>
RX_DEV void rx_lm_move(U* base, const int (&from)[A], const int (&there)[A], const int (&here)[A], const int n, G place) {
  U held[A];
#pragma unroll
  for (int a = 0; a < A; ++a)
    if (from[a] >= 0) held[a] = base[place(there[a], (rx_u32)from[a] % S)];
#pragma unroll
  for (int a = 0; a < A; ++a)
    if (from[a] >= 0) base[place(here[a], (rx_u32)(n + a) % S)] = held[a];
}
template <typename U, int KU, int VU, int HK, int P, int S, int B, int M, int A, bool BY_SLOT, bool SCALES, typename I>
RX_DEV void rx_kv_move(const I* lengths, const I* path, const I* pages, U* kc, U* vc, float* ks, float* vs) {
  constexpr int UNITS = HK * (KU + VU) + (SCALES ? 2 * HK : 0);
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < (long long)B * UNITS; i += (long long)gridDim.x * 256) {
    const long long b = i / UNITS;
    const int u = (int)(i % UNITS);
    // all loads of one kind before the first of the next: lengths and path, pages, units
    const I len = lengths[b];
    I p[A];
#pragma unroll
    for (int a = 0; a < A; ++a) p[a] = path[b * A + a];
    if (len < 0 || len >= (I)(M * S)) continue;
    const int n = (int)len;
    int from[A], there[A], here[A];                     // position that is moved (-1: none), its page and the page it is moved to
#pragma unroll
    for (int a = 0; a < A; ++a) {
      const bool moves = p[a] >= 0 && p[a] != a && p[a] < (I)(M * S - n) && a < M * S - n;
      from[a] = moves ? n + (int)p[a] : -1;
      const I fp = pages[b * M + (rx_u32)(moves ? from[a] : 0) / S], tp = pages[b * M + (rx_u32)(moves ? n + a : 0) / S];
      there[a] = fp >= 0 && fp < P ? (int)fp : -1;
      here[a] = tp >= 0 && tp < P ? (int)tp : -1;
    }
#pragma unroll
    for (int a = 0; a < A; ++a)
      if (there[a] < 0 || here[a] < 0) from[a] = -1;
    if (u < HK * KU)
      rx_lm_move<S>(kc, from, there, here, n, [u](const int page, const int slot) { return rx_lm_slot<S, HK, KU, BY_SLOT>(page, slot, u / KU) + u % KU; });
    else if (u < HK * (KU + VU))
      rx_lm_move<S>(vc, from, there, here, n, [u](const int page, const int slot) { return rx_lm_slot<S, HK, VU, BY_SLOT>(page, slot, (u - HK * KU) / VU) + (u - HK * KU) % VU; });
    else if constexpr (SCALES) {
      const int h = u - HK * (KU + VU);
      rx_lm_move<S>(h < HK ? ks : vs, from, there, here, n, [h](const int page, const int slot) { return rx_lm_slot<S, HK, 1, false>(page, slot, h % HK); });
    }
  }
}

// ---------------------------------------------------------------------------
// attention of drafted tokens
// ---------------------------------------------------------------------------
// As the attention of one token per sequence (rx_paged_attention): one pass with running maxima and sums, scores as K Q' and results
// as V' P' on the matrix cores, where the columns are rows of the result: (drafted token, query head) pairs of one key head, token
// by token.  A step is 32 positions.  Which rows see a position matters only in steps that hold drafted tokens or the window's edge.
//
// One token over 8 sequences of 131072 positions in 8 bits, 64 query heads of 8, 2.2 GB: 379 us, 5.8 TB/s, bound by memory (rows of 128
// bytes are two half lines to a load; three and four wavefronts to a SIMD 384 and 427 us).  64 drafted tokens of 16 sequences of 4001 positions, 64
// query heads of 8, 136 GFLOP in f16: 264 us, 517 TFLOP/s, bound by the vector units (65 % of the time; the matrix cores a third): softmax, the weights'
// second numbers, addresses.  16 tokens of 64 sequences of up to 8192 in 8 bits: 72 us, half of it vector units, half a step's chain.
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

// two numbers (no products) rounded to a 16-bit type, by one operation: what is unpacked again is not rounded again
template <typename F>
RX_DEV rx_u32 rx_lm_pair_down(const float x, const float y) {
  rx_u32 p;
  if constexpr (F::BF16) {
    typedef __bf16 P __attribute__((ext_vector_type(2)));
    p = __builtin_bit_cast(rx_u32, P{(__bf16)x, (__bf16)y});
  } else {
    typedef _Float16 P __attribute__((ext_vector_type(2)));
    p = __builtin_bit_cast(rx_u32, P{(_Float16)x, (_Float16)y});
  }
  rx_pin(p);
  return p;
}
// the largest of the four lanes l, l ^ 16, l ^ 32, l ^ 48, by exchanges of rows of lanes
RX_DEV float rx_lm_rows_max(const float x) {
  const auto a = __builtin_amdgcn_permlane16_swap(rx_f2u(x), rx_f2u(x), false, false);
  const float y = __builtin_fmaxf(rx_u2f(a[0]), rx_u2f(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(rx_f2u(y), rx_f2u(y), false, false);
  return __builtin_fmaxf(rx_u2f(b[0]), rx_u2f(b[1]));
}
// offset of a slot's head in a cache, of pages whose elements 32 bits count where they do
template <int S, int H, int D, bool BY_SLOT>
RX_DEV rx_u64 rx_lm_at(const rx_u32 page, const rx_u32 slot, const rx_u32 head) {
  if constexpr ((long long)S * H * D < (1ll << 31)) return (rx_u64)page * (rx_u32)(S * H * D) + (BY_SLOT ? slot * (H * D) + head * D : head * (S * D) + slot * D);
  else return rx_lm_slot<S, H, D, BY_SLOT>(page, slot, head);
}

// What the rows of a wavefront have seen: maxima, sums, unscaled results, for NT tiles of 16 rows.
// E: of the queries and the result, C: of the caches, F: of the products.  Caches of 8 bits are multiplied as bf16, which holds their numbers
// exactly; queries of more digits than bf16's go in as a sum of bf16, which holds them exactly too (f16: two, f32: three).
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
  bool careful[NT];                                                                                 // a row's maximum is beyond 2^20, or the factor zero
  rx_f32x4 acc[NT][NV][VE];

  RX_MEM void clear() {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      m[t] = -rx_lm_inf();
      l[t] = 0.0f;
      careful[t] = false;
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
      if constexpr (NQ == 1) {
        q[t][0][k] = there ? rx_lm_row16<E, DK>(row, dim(k, g4)) : rx_u32x4{0, 0, 0, 0};
      } else {
        rx_vec<rx_u16, 8> part[NQ];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float x = there && dim(k, g4) + e < DK ? E::up(row[dim(k, g4) + e]) : 0.0f;
          const bool finite = __builtin_fabsf(x) <= RX_LM_FLT_MAX;
#pragma unroll
          for (int n = 0; n < NQ; ++n) {
            // (digits cut off, not rounded: 8 and 8 and 8 are all that f32 has, and neither a part nor a sum of them exceeds the number)
            part[n].v[e] = finite ? (rx_u16)(rx_f2u(x) >> 16) : rx_f32_to_bf16(x);
            x = finite ? x - rx_bf16_to_f32(part[n].v[e]) : 0.0f;
          }
        }
#pragma unroll
        for (int n = 0; n < NQ; ++n) q[t][n][k] = __builtin_bit_cast(rx_u32x4, part[n]);
      }
    }
  }
  // One step.  kf: keys of positions r and 16 + r; value(j, e): dimension VE r + e (of 16 VE) of the eight positions 4 g4 + (0..3) and
  // 16 further as an operand, after load_values(); factor: of the scores; ks, vs: the scales of the eight positions, ks times factor already.
  // Where `some` rows do not see some of the positions, seen[t] says which of those eight the lane's row sees: their scores become -inf, and
  // the rest is the same code, since code that runs once or twice is paid for by loading it.
  template <typename V, typename L>
  RX_MEM void step(const rx_u32x4 (&kf)[2][KF], L load_values, V value, const bool some, const unsigned (&seen)[NT], const float factor, const float (&ks)[8], const float (&vs)[8]) {
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
      // Where all positions have one factor the largest score is that of the products, times it, and weights take one operation more.
      const bool down = !BITS8 && factor < 0.0f;
      float x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = BITS8 ? s[i >> 2][i & 3] * ks[i] : s[i >> 2][i & 3];
      if (__builtin_expect(some, 0)) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = (seen[t] >> i) & 1u ? x[i] : down ? rx_lm_inf() : -rx_lm_inf();
      }
      float far = x[0];
#pragma unroll
      for (int i = 1; i < 8; ++i) far = down ? __builtin_fminf(far, x[i]) : __builtin_fmaxf(far, x[i]);
      // (not below the lowest number, so that differences from it are numbers)
      const float top = __builtin_fmaxf(m[t], rx_lm_rows_max(__builtin_fmaxf(BITS8 ? far : far * factor, -RX_LM_FLT_MAX)));
      if (__builtin_expect(__any(top != m[t]), 0)) {
        const float shrink = __builtin_amdgcn_exp2f(m[t] - top);
        l[t] *= shrink;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int e = 0; e < VE; ++e) acc[t][j][e] *= shrink;
        m[t] = top;
        careful[t] = !BITS8 && (factor == 0.0f || __any(__builtin_fabsf(top) >= 0x1p20f));
      }
      // One operation to a weight's exponent, whose error, the roundings of `top` and `base`, is below 2^-3 up to a maximum of 2^20.  Beyond, where
      // weights would grow without bound, differences are taken from the rounded products, of which the maximum is one; with a factor of zero
      // too, whose product with a masked score would be no number.  (The branch is 1 % of the time of 64 tokens of 64 heads.)
      float base = SHIFT - top, times = factor;
      if (!BITS8 && __builtin_expect(careful[t], 0)) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = !some || ((seen[t] >> i) & 1u) ? x[i] * factor - top + SHIFT : -rx_lm_inf();
        base = 0.0f;
        times = 1.0f;
      }
      float p[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) p[i] = __builtin_amdgcn_exp2f(BITS8 ? x[i] + base : __builtin_fmaf(x[i], times, base));
      l[t] += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
      if constexpr (BITS8) {
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] *= vs[i];
      }
      if constexpr (WIDE) {
#pragma unroll
        for (int i = 0; i < 8; ++i) wide[t][i] = p[i];
      } else {
#pragma unroll
        for (int n = 0; n < NP; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const rx_u32 pair = rx_lm_pair_down<F>(p[2 * i], p[2 * i + 1]);
            w[t][n][i] = pair;
            if (n + 1 < NP) {
              p[2 * i] -= F::up((rx_u16)pair);
              p[2 * i + 1] -= F::up((rx_u16)(pair >> 16));
            }
          }
      }
    }
    load_values();
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

// Parts of a result in memory as rx_lm_put_shared writes single numbers, four at a time: 16 bytes that one thread writes, device-wide
// (sc1, as the compiler has device-scope atomic accesses), and reads after they have been counted in.
RX_DEV void rx_lm_put_shared4(const __amdgpu_buffer_rsrc_t to, const unsigned byte, const rx_f32x4 v) {
  __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(rx_u32x4, v), to, byte, 0, 16);
}
RX_DEV rx_f32x4 rx_lm_get_shared4(const __amdgpu_buffer_rsrc_t from, const unsigned byte) {
  return __builtin_bit_cast(rx_f32x4, __builtin_amdgcn_raw_buffer_load_b128(from, byte, 0, 16));
}
RX_DEV __amdgpu_buffer_rsrc_t rx_lm_shared(float* base, const unsigned bytes) { return __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, bytes, 0x00020000); }

// Reads of LDS that other loads are on their way to.  The compiler has every read of its own wait for all loads into LDS, whichever place they
// go to; these are of places that have arrived, and wait for nothing but themselves.
RX_DEV rx_u32 rx_lm_lds(const void* p) { return (rx_u32)(unsigned long long)(RX_LDS const void*)p; }
// four places, and the four OFF bytes further
template <int OFF>
RX_DEV void rx_lm_lds_eight(rx_u32x4 (&x)[4], rx_u32x4 (&y)[4], const rx_u32 (&a)[4]) {
  asm volatile(
      "ds_read_b128 %0, %8\n\tds_read_b128 %1, %9\n\tds_read_b128 %2, %10\n\tds_read_b128 %3, %11\n\t"
      "ds_read_b128 %4, %8 offset:%12\n\tds_read_b128 %5, %9 offset:%12\n\tds_read_b128 %6, %10 offset:%12\n\tds_read_b128 %7, %11 offset:%12\n\ts_waitcnt lgkmcnt(0)"
      : "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3]), "=&v"(y[0]), "=&v"(y[1]), "=&v"(y[2]), "=&v"(y[3])
      : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]), "n"(OFF)
      : "memory");
}
template <int OFF>
RX_DEV void rx_lm_lds_eight(rx_u32x2 (&x)[4], rx_u32x2 (&y)[4], const rx_u32 (&a)[4]) {
  asm volatile(
      "ds_read_b64 %0, %8\n\tds_read_b64 %1, %9\n\tds_read_b64 %2, %10\n\tds_read_b64 %3, %11\n\t"
      "ds_read_b64 %4, %8 offset:%12\n\tds_read_b64 %5, %9 offset:%12\n\tds_read_b64 %6, %10 offset:%12\n\tds_read_b64 %7, %11 offset:%12\n\ts_waitcnt lgkmcnt(0)"
      : "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3]), "=&v"(y[0]), "=&v"(y[1]), "=&v"(y[2]), "=&v"(y[3])
      : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]), "n"(OFF)
      : "memory");
}
template <int OFF>
RX_DEV void rx_lm_lds_eight(rx_u32 (&x)[4], rx_u32 (&y)[4], const rx_u32 (&a)[4]) {
  asm volatile(
      "ds_read_b32 %0, %8\n\tds_read_b32 %1, %9\n\tds_read_b32 %2, %10\n\tds_read_b32 %3, %11\n\t"
      "ds_read_b32 %4, %8 offset:%12\n\tds_read_b32 %5, %9 offset:%12\n\tds_read_b32 %6, %10 offset:%12\n\tds_read_b32 %7, %11 offset:%12\n\ts_waitcnt lgkmcnt(0)"
      : "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3]), "=&v"(y[0]), "=&v"(y[1]), "=&v"(y[2]), "=&v"(y[3])
      : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]), "n"(OFF)
      : "memory");
}
// two places, and the two OFF bytes further
template <int OFF>
RX_DEV void rx_lm_lds_four(rx_u32x4& x0, rx_u32x4& x1, rx_u32x4& y0, rx_u32x4& y1, const rx_u32 a0, const rx_u32 a1) {
  asm volatile("ds_read_b128 %0, %4\n\tds_read_b128 %1, %5\n\tds_read_b128 %2, %4 offset:%6\n\tds_read_b128 %3, %5 offset:%6\n\ts_waitcnt lgkmcnt(0)"
               : "=&v"(x0), "=&v"(x1), "=&v"(y0), "=&v"(y1)
               : "v"(a0), "v"(a1), "n"(OFF)
               : "memory");
}
RX_DEV void rx_lm_lds_words(int (&x)[4], const rx_u32 (&a)[4]) {
  asm volatile("ds_read_b32 %0, %4\n\tds_read_b32 %1, %5\n\tds_read_b32 %2, %6\n\tds_read_b32 %3, %7\n\ts_waitcnt lgkmcnt(0)"
               : "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3])
               : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3])
               : "memory");
}

// MASK: 0 every drafted token sees itself and those before it, 2 [N, N] for all sequences, 3 [B, N, N].  NT: tiles of 16 rows to a
// wavefront.  WR: wavefronts that have rows of their own: 1 (few rows) the four share the positions, and read the caches into their
// registers; 4 (many rows) they share keys and values, which pass through LDS: with a RING of that many stages of 32 positions, loaded without
// registers; without one (rows that are no whole 16 bytes) through registers, 8-bit numbers as bf16, the next step's being loaded while this
// one's are multiplied.  R, ONCE, DIES, Q: as for rx_paged_attention.
template <typename E, typename C, int N, int HQ, int HK, int DK, int DV, int P, int S, int B, int M, int W, bool BY_SLOT, int MASK, int NT, int WR, int RING, int R, bool ONCE,
          bool DIES, int Q, typename I>
RX_DEV void rx_tree_attention(const typename E::S* q, const typename C::S* kc, const typename C::S* vc, const I* pages, const I* lengths, const rx_u8* mask, const float* ks,
                              const float* vs, typename E::S* out, float* lse, float* part, float* stat, int* arrived, const float scale) {
  constexpr bool SHARED = WR > 1, BITS8 = rx_lm_is8<C>::value;
  typedef rx_lm_tree<E, C, DK, DV, NT, BITS8 && (!SHARED || RING)> A;
  typedef typename A::F F;
  typedef typename C::S T;
  constexpr int G = HQ / HK, ROWS = N * G, TR = 16 * NT * WR, RT = ROWS < TR ? ROWS : TR, TILES = (ROWS + TR - 1) / TR, COLUMNS = HK * TILES;
  constexpr int KF = A::KF, VE = A::VE, NV = A::NV;
  constexpr int BLOCK = RING ? 1024 * (S < 256 ? S : 256) : 2048;   // positions whose pages are held in LDS
  constexpr int HR = RT < 16 ? RT : 16, WIDTH = 16 * VE < DV ? 16 * VE : DV;   // rows and dimensions that are joined at a time
  constexpr int VD = DV % 4 == 0 ? 4 : 1;
  constexpr int FE = 16 / sizeof(typename F::S), KP = KF * 4 * A::NE + FE, VP = NV * 16 * VE + FE;   // rows of keys and values in LDS: 16 bytes longer, for its banks
  typedef rx_vec<rx_u32, VE * sizeof(typename F::S) / 4> FV;   // a lane's part of a value
  // A stage of the ring: 32 keys and 32 values in chunks of 16 bytes, as many to a row as the next power of two holds, chunk c of row i at
  // place c ^ turn(i), so that sixteen rows' chunks lie on different banks.
  constexpr int CE = 16 / sizeof(T), CK = (DK + CE - 1) / CE, CV = (DV + CE - 1) / CE, PK = rx_lm_pow2(CK) < 4 ? 4 : rx_lm_pow2(CK), PV = rx_lm_pow2(CV) < 4 ? 4 : rx_lm_pow2(CV);
  constexpr int STAGE = 32 * 16 * (PK + PV);
  constexpr int ROOM = SHARED ? 4 * 16 * (16 * VE + 4) * 4 : 16;   // for the results of four wavefronts' 16 rows
  __shared__ __attribute__((aligned(1024))) rx_u8 ring[RING * STAGE > ROOM ? RING * STAGE : ROOM];
  __shared__ int table[RING ? BLOCK / S + 2 : 1];
  __shared__ float ring_s[RING ? RING : 1][64];
  __shared__ union {
    int page[SHARED ? 1 : BLOCK / S + 2];
    float o[SHARED ? 1 : 4][HR][WIDTH + 4];
    rx_lm_joined<VD> j[256];
  } lds;
  __shared__ float join_m[4][16], join_l[4][16];
  __shared__ __attribute__((aligned(16))) typename F::S kt[SHARED && !RING ? 2 : 1][SHARED && !RING ? 32 : 1][SHARED && !RING ? KP : FE];
  __shared__ __attribute__((aligned(16))) typename F::S vt[SHARED && !RING ? 2 : 1][SHARED && !RING ? 32 : 1][SHARED && !RING ? VP : FE];
  __shared__ float st_k[2][32], st_v[2][32];
  __shared__ unsigned st_ok[2];
  __shared__ int last, any;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, r = lane & 15, g4 = lane >> 4;
  const int id = DIES ? (int)rx_xcd_remap(blockIdx.x, R * COLUMNS) : (int)blockIdx.x, column = id % COLUMNS, mine = id / COLUMNS, tile = column % TILES;
  const int head = column / TILES;
  const int row0 = tile * TR + (SHARED ? wave * 16 * NT : 0);                 // first row of this wavefront
  const int rows = ROWS - tile * TR < TR ? ROWS - tile * TR : TR;             // of the workgroup
  const rx_lm_stretch st = rx_lm_stretch_of<B, R, Q>([&](const int at) { return rx_lm_tree_span_of<S, B, M, N, W>(lengths[at]).cost; }, mine);
  auto result_of = [&](const int b, const int row, const int h) { return ((long long)b * N + row / G) * HQ + h * G + row % G; };   // row of the results
  const __amdgpu_buffer_rsrc_t parts_at = rx_lm_shared(part, (unsigned)R * COLUMNS * 2 * RT * DV * 4);
  int buf = 0;
  if constexpr (SHARED && !RING && (DK + FE - 1) / FE * FE < KF * 4 * A::NE) {          // what no chunk of a key covers
    for (int i = threadIdx.x; i < 64 * KP; i += 256) (&kt[0][0][0])[i] = F::down(0.0f);
    __syncthreads();
  }

  // (what all lanes have alike is kept in scalar registers)
  int b = __builtin_amdgcn_readfirstlane(st.b), unit = __builtin_amdgcn_readfirstlane(st.unit);
  for (int left = __builtin_amdgcn_readfirstlane(st.count); left > 0; ++b, unit = 0) {
  rx_lm_tree_span span = rx_lm_tree_span_of<S, B, M, N, W>(lengths[b]);
  span.n = __builtin_amdgcn_readfirstlane(span.n);
  span.lo = __builtin_amdgcn_readfirstlane(span.lo);
  span.units = __builtin_amdgcn_readfirstlane(span.units);
  span.cost = __builtin_amdgcn_readfirstlane(span.cost);
  span.prefix = __builtin_amdgcn_readfirstlane(span.prefix);
  const int step = span.cost - unit < left ? span.cost - unit : left, take = span.units - unit < step ? span.units - unit : step;
  const long long begin = st.first + (st.count - left) - unit;                // the sequence's first unit in the row
  left -= step;
  if (take <= 0) continue;
  const int p0 = (span.lo & ~31) + unit * 32, p1 = P == 0 ? p0 : p0 + take * 32 < span.n ? p0 + take * 32 : span.n;
  const bool whole = take == span.units;                                      // the whole sequence is in this stretch
  A a;
  a.clear();
  // With a window the last of its places are taken by the drafted tokens that a token sees; where it begins among the positions before them.
  auto first_of = [&](const int token) {
    if constexpr (W == 0) return 0;
    int sees = 0;
    if constexpr (MASK == 0) sees = token + 1;
    else
      for (int j = 0; j < N; ++j) sees += mask[((long long)(MASK == 3 ? b : 0) * N + token) * N + j] != 0;
    return span.prefix - (W - sees) > 0 ? span.prefix - (W - sees) : 0;
  };
  auto sees = [&](const int token, const int first, const int p) {
    if (p < span.prefix) return p >= first;
    if constexpr (MASK == 0) return p - span.prefix <= token;
    else return mask[((long long)(MASK == 3 ? b : 0) * N + token) * N + (p - span.prefix)] != 0;
  };
  int token[NT], first[NT];                                                   // of the lane's rows
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    int row = row0 + t * 16 + r;
    rx_pin(row);
    const bool inside = row < ROWS;
    token[t] = inside ? row / G : 0;
    first[t] = first_of(token[t]);
    a.load(t, q + result_of(b, inside ? row : 0, head) * DK, inside);
  }
  // Rows differ in what they see of the steps before `edge` and of those from `mixed` on.
  const int edge = W > 0 && span.prefix - W + N > 0 ? (span.prefix - W + N + 31) & ~31 : 0, mixed = span.prefix & ~31;
  // bits of the lane's eight positions of a step that its rows see
  auto seen_by = [&](const int t0, const unsigned ok, unsigned (&seen)[NT]) {
    int g = g4;
    rx_pin(g);
    // (all of the mask's loads before the first of them is looked at: one under a condition waits for the one before)
    rx_u8 drafted[NT][8];
    if constexpr (MASK != 0) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int j = t0 + (i & 4) * 4 + g * 4 + (i & 3) - span.prefix;
          drafted[t][i] = mask[((long long)(MASK == 3 ? b : 0) * N + token[t]) * N + (j < 0 ? 0 : j < N ? j : N - 1)];
        }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      seen[t] = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int at = (i & 4) * 4 + g * 4 + (i & 3), p = t0 + at;
        bool see = p >= first[t];
        if constexpr (MASK == 0) see = p < span.prefix ? see : p - span.prefix <= token[t];
        else see = p < span.prefix ? see : drafted[t][i] != 0;
        seen[t] |= ((ok >> at) & 1u) && see ? 1u << i : 0u;
      }
    }
  };
  auto differ = [&](const int t0) { return t0 >= mixed || (W > 0 && t0 < edge); };
  rx_u32 special = 0;                                                         // infinities or NaN have been taken out of values
  unsigned saw[NT] = {};                                                      // positions that the lane's rows have seen
  bool all = false;                                                           // in a step that all rows see alike
  auto look = [&](const int t0, const unsigned ok, unsigned (&seen)[NT]) {
    seen_by(t0, ok, seen);
#pragma unroll
    for (int t = 0; t < NT; ++t) saw[t] |= seen[t];
  };

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
      auto where = [&](const int t) { return t >= span.lo && t < s1 ? lds.page[(rx_u32)t / S - page0] : -1; };
      for (int t0 = s0 + wave * 32; t0 < s1; t0 += 128) {
        const int ta = t0 + r, tb = ta + 16, pa = where(ta), pb = where(tb);
        const unsigned ok = ((unsigned)__ballot(pa >= 0) & 0xffffu) | ((unsigned)__ballot(pb >= 0) << 16);
        if (!ok) continue;
        rx_vec<rx_u32, 4> raw[2][KR];
        const T* ka = kc + rx_lm_at<S, HK, DK, BY_SLOT>(pa < 0 ? 0 : pa, (rx_u32)ta % S, head);
        const T* kb = kc + rx_lm_at<S, HK, DK, BY_SLOT>(pb < 0 ? 0 : pb, (rx_u32)tb % S, head);
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
          const T* v = vc + rx_lm_at<S, HK, DV, BY_SLOT>(pv < 0 ? 0 : pv, (rx_u32)tv % S, head);
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
        // (the mask's loads start behind those of keys and values, before any of them is waited for)
        unsigned seen[NT] = {};
        const bool some = ok != ~0u || differ(t0);
        if (__builtin_expect(some, 0)) look(t0, ok, seen);
        else all = true;
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
        rx_u32x4 kf[2][KF];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int k = 0; k < KF; ++k) {
            if constexpr (BITS8) kf[h][k] = rx_lm_eight_up<C>(raw[h][k / 2].v[k % 2 * 2], raw[h][k / 2].v[k % 2 * 2 + 1]);
            else kf[h][k] = __builtin_bit_cast(rx_u32x4, raw[h][k]);
          }
        auto value = [&](const int j, const int e, const int half) {
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
        };
        if (__builtin_expect(some, 0)) {
          if (differ(t0)) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              if (BITS8 && !(__builtin_fabsf(vscale[i]) <= RX_LM_FLT_MAX)) {
                special |= (there >> ((i & 4) * 4 + (i & 3))) & 1u;
                vscale[i] = 0.0f;
              }
#pragma unroll
              for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int n = 0; n < (int)(sizeof(CV) / 4); ++n) {
                  const rx_u32 x = rx_lm_special<C>(vf[j][i].v[n]);
                  vf[j][i].v[n] &= ~x;
                  special |= x;
                }
            }
          }
          if constexpr (BITS8) {
#pragma unroll
            for (int i = 0; i < 8; ++i) vscale[i] = (there >> ((i & 4) * 4 + (i & 3))) & 1u ? vscale[i] : 0.0f;
          }
        }
        a.step(kf, [] {}, value, some, seen, scale, kscale, vscale);
      }
    }
  } else if constexpr (RING > 0) {
    // Keys and values pass through LDS without registers, RING - 1 steps ahead: the loads of a step are started when the step before
    // last has been used, and waited for by count.
    constexpr int PER = (PK + PV) / 8, COUNT = PER + (BITS8 ? 1 : 0), AHEAD = RING - 1;   // loads of a wavefront in a step
    static_assert((PK + PV) % 8 == 0, "a step's loads are shared equally");
    typedef rx_vec<rx_u32, VE * sizeof(T) / 4> CVEC;
    constexpr int KR = BITS8 ? KF / 2 : KF;
    auto turn = [](const int row, const int places) { return places >= 16 ? row & 15 : (row / (16 / places)) & (places - 1); };
    const int key_turn = turn(r, PK);
    for (int s0 = p0; s0 < p1; s0 += BLOCK) {
      const int s1 = s0 + BLOCK < p1 ? s0 + BLOCK : p1, page0 = (rx_u32)s0 / S, npages = (rx_u32)(s1 - 1) / S - page0 + 1;
      __syncthreads();
      for (int i = threadIdx.x; i < npages; i += 256) {
        const I page = pages[(long long)b * M + page0 + i];
        table[i] = page >= 0 && page < P ? (int)page : -1;
      }
      __syncthreads();
      // Pages of a step's rows: of the rows that the lane loads, and of position lane mod 32.  Positions that are not to be looked at have the table's
      // first or last entry, and are told by `here`.
      auto entry = [&](const int t) { return rx_lm_lds(table) + 4 * ((rx_u32)(t < s1 ? t : s1 - 1) / S - page0); };
      auto here = [&](const int t, const int page) { return t >= span.lo && t < s1 && page >= 0; };
      auto start = [&](const int t0, const int stage) {
        constexpr int LOOK = PER + (BITS8 ? 1 : 0);
        int page[(LOOK + 3) / 4 * 4];
#pragma unroll
        for (int n = 0; n < LOOK; n += 4) {
          rx_u32 a[4];
          int w[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int at = (n + k) * 4 + wave, i = (at < PK / 2 ? at : at - PK / 2) * 64 + lane;
            a[k] = n + k < PER ? entry(t0 + i / (at < PK / 2 ? PK : PV)) : entry(t0 + (lane & 31));
          }
          rx_lm_lds_words(w, a);
#pragma unroll
          for (int k = 0; k < 4; ++k) page[n + k] = w[k];
        }
#pragma unroll
        for (int n = 0; n < PER; ++n) {
          const int at = n * 4 + wave;                    // kilobyte of the stage: keys, then values
          const bool key = at < PK / 2;
          const int i = (key ? at : at - PK / 2) * 64 + lane, places = key ? PK : PV, row = i / places, c = (i % places) ^ turn(row, places);
          const int chunk = c < (key ? CK : CV) ? c : (key ? CK : CV) - 1;
          const rx_u32 slot = (rx_u32)(t0 + row) % S, p = page[n] < 0 ? 0 : page[n];
          const T* from = key ? kc + rx_lm_at<S, HK, DK, BY_SLOT>(p, slot, head) + chunk * CE : vc + rx_lm_at<S, HK, DV, BY_SLOT>(p, slot, head) + chunk * CE;
          __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from, (RX_LDS void*)(ring + stage * STAGE + at * 1024), 16, 0, 0);
        }
        if constexpr (BITS8) {                            // (every wavefront the same, so that all count the same loads)
          const float* from = (lane < 32 ? ks : vs) + rx_lm_slot<S, HK, 1, false>(page[PER] < 0 ? 0 : page[PER], (rx_u32)(t0 + (lane & 31)) % S, head);
          __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from, (RX_LDS void*)&ring_s[stage][0], 4, 0, 0);
        }
      };
      int next = 0, now = 0;
#pragma unroll
      for (int n = 0; n < AHEAD; ++n) {
        start(s0 + n * 32, next);
        next = next + 1 == RING ? 0 : next + 1;
      }
      for (int t0 = s0; t0 < s1; t0 += 32) {
        rx_wait_vmcnt<(AHEAD - 1) * COUNT>();
        rx_lds_barrier();                                 // (and the stage that is loaded next has been read)
        start(t0 + AHEAD * 32, next);                     // (past the end: slots that nothing reads)
        const int stage = now;
        next = next + 1 == RING ? 0 : next + 1;
        now = now + 1 == RING ? 0 : now + 1;
        const rx_u32 keys = rx_lm_lds(ring) + stage * STAGE + r * (PK * 16), values = rx_lm_lds(ring) + stage * STAGE + 512 * PK, scales = rx_lm_lds(ring_s) + stage * 256 + g4 * 16;
        unsigned ok;
        {
          const rx_u32 a[4] = {entry(t0 + (lane & 31)), entry(t0), entry(t0), entry(t0)};
          int w[4];
          rx_lm_lds_words(w, a);
          ok = (unsigned)__ballot(lane < 32 && here(t0 + lane, w[0]));
        }
        if (__builtin_expect(!ok, 0)) continue;
        const bool some = ok != ~0u || differ(t0);
        if (__builtin_expect(some, 0)) {
          // What lies in other slots may be anything, and NaN times a weight of zero is not zero; the same of infinities and NaN in slots that some
          // rows see, which are taken out here.
          rx_u8* const tile_v = ring + stage * STAGE + 512 * PK;
          for (int i = threadIdx.x; i < 32 * PV; i += 256) {
            const int row = i / PV;
            const bool exists = (ok >> row) & 1u, whole_row = ((i % PV) ^ turn(row, PV)) < CV;
            rx_vec<rx_u32, 4> x = rx_load<rx_vec<rx_u32, 4>>(tile_v + i * 16);
#pragma unroll
            for (int n = 0; n < 4; ++n) {
              const rx_u32 out_of = exists && differ(t0) ? rx_lm_special<C>(x.v[n]) : 0u;
              x.v[n] &= exists ? ~out_of : 0u;
              special |= whole_row ? out_of : 0u;
            }
            rx_store(tile_v + i * 16, x);
          }
          if (BITS8 && threadIdx.x < 32) {
            const bool exists = (ok >> threadIdx.x) & 1u, finite = __builtin_fabsf(ring_s[stage][32 + threadIdx.x]) <= RX_LM_FLT_MAX;
            if (!exists || (!finite && differ(t0))) ring_s[stage][32 + threadIdx.x] = 0.0f;
            special |= exists && !finite && differ(t0) ? 1u : 0u;
          }
          rx_lds_barrier();
        }
        if (__builtin_expect(row0 >= ROWS, 0)) continue;
        rx_u32x4 kf[2][KF];
#pragma unroll
        for (int k0 = 0; k0 < KR; k0 += 4) {
          rx_u32x4 x[4], y[4];
          rx_u32 a[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) a[k] = keys + (((k0 + k < KR ? k0 + k : KR - 1) * 4 + g4) ^ key_turn) * 16;
          if constexpr (KR <= 2) rx_lm_lds_four<256 * PK>(x[0], x[1], y[0], y[1], a[0], a[1]);
          else rx_lm_lds_eight<256 * PK>(x, y, a);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if (k0 + k >= KR) break;
            // (places past a key's end hold its last chunk again, and an infinity there times a query's zero is NaN; 8 bits have no infinity)
            if (!BITS8 && CK % 4 != 0 && k0 + k == KR - 1 && g4 >= CK % 4) x[k] = y[k] = rx_u32x4{0, 0, 0, 0};
            if constexpr (BITS8) {
              kf[0][2 * (k0 + k)] = rx_lm_eight_up<C>(x[k][0], x[k][1]);
              kf[0][2 * (k0 + k) + 1] = rx_lm_eight_up<C>(x[k][2], x[k][3]);
              kf[1][2 * (k0 + k)] = rx_lm_eight_up<C>(y[k][0], y[k][1]);
              kf[1][2 * (k0 + k) + 1] = rx_lm_eight_up<C>(y[k][2], y[k][3]);
            } else {
              kf[0][k0 + k] = x[k];
              kf[1][k0 + k] = y[k];
            }
          }
        }
        CVEC vf[NV][8];
        float kscale[8] = {}, vscale[8] = {};
        if constexpr (BITS8) {
          rx_u32x4 x0, x1, y0, y1;
          rx_lm_lds_four<128>(x0, x1, y0, y1, scales, scales + 64);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            kscale[i] = rx_u2f(x0[i]) * scale;
            kscale[4 + i] = rx_u2f(x1[i]) * scale;
            vscale[i] = rx_u2f(y0[i]);
            vscale[4 + i] = rx_u2f(y1[i]);
          }
        }
        // (not before the weights are done: keys and values in registers at once leave none for a second wavefront)
        auto load_values = [&] {
          typedef typename rx_lm_if<sizeof(CVEC) == 16, rx_u32x4, typename rx_lm_if<sizeof(CVEC) == 8, rx_u32x2, rx_u32>::type>::type X;
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int j = 0; j < NV; ++j) {
            rx_u32 a[4];
            X x[4], y[4];
            const int byte = (j * 16 + r) * VE * (int)sizeof(T);
#pragma unroll
            for (int i = 0; i < 4; ++i) a[i] = values + (g4 * 4 + i) * (PV * 16) + (((byte / 16) & (PV - 1)) ^ turn(g4 * 4 + i, PV)) * 16 + byte % 16;
            rx_lm_lds_eight<256 * PV>(x, y, a);        // (rows 16 further have the same turn)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              vf[j][i] = __builtin_bit_cast(CVEC, x[i]);
              vf[j][4 + i] = __builtin_bit_cast(CVEC, y[i]);
            }
          }
        };
        auto value = [&](const int j, const int e, const int half) {
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
        };
        unsigned seen[NT] = {};
        if (__builtin_expect(some, 0)) look(t0, ok, seen);
        else all = true;
        a.step(kf, load_values, value, some, seen, scale, kscale, vscale);
      }
      rx_wait_vmcnt<0>();
    }
  } else {
    constexpr int LK = (32 * CK + 255) / 256, LV = (32 * CV + 255) / 256;
    rx_vec<rx_u32, 4> rk[LK], rv[LV];
    I pk[LK], pv[LV], ps = 0;                           // page table's entries of the next step's loads; of position threadIdx.x
    float sk = 0.0f, sv = 0.0f;
    bool there = false;
    const I* table = pages + (long long)b * M;
    // (No condition between a load and the next: each would wait for the data of the one before.  Positions past the end are the last.)
    auto entry = [&](const int t) { return table[(rx_u32)(t < p1 ? t : p1 - 1) / S]; };
    auto known = [&](const int t, const I page) { return t >= span.lo && t < p1 && page >= 0 && page < P; };
    auto find = [&](const int t0) {
#pragma unroll
      for (int n = 0; n < LK; ++n) pk[n] = entry(t0 + (n * 256 + (int)threadIdx.x) / CK);
#pragma unroll
      for (int n = 0; n < LV; ++n) pv[n] = CV == CK ? pk[n < LK ? n : 0] : entry(t0 + (n * 256 + (int)threadIdx.x) / CV);
      ps = entry(t0 + (int)threadIdx.x);
    };
    auto fetch = [&](const int t0) {
      bool on[LK];
#pragma unroll
      for (int n = 0; n < LK; ++n) {
        const int i = n * 256 + (int)threadIdx.x, t = t0 + i / CK;
        on[n] = known(t, pk[n]);
        rk[n] = rx_lm_part<T, DK, CE, ONCE>(kc + rx_lm_at<S, HK, DK, BY_SLOT>(on[n] ? (rx_u32)pk[n] : 0u, (rx_u32)t % S, head), i % CK * CE);
      }
#pragma unroll
      for (int n = 0; n < LV; ++n) {
        const int i = n * 256 + (int)threadIdx.x, t = t0 + i / CV;
        const bool in = CV == CK ? on[n < LK ? n : 0] : known(t, pv[n]);
        rv[n] = rx_lm_part<T, DV, CE, ONCE>(vc + rx_lm_at<S, HK, DV, BY_SLOT>(in ? (rx_u32)pv[n] : 0u, (rx_u32)t % S, head), i % CV * CE);
      }
      there = threadIdx.x < 32 && known(t0 + (int)threadIdx.x, ps);
      if constexpr (BITS8) {
        const long long at = rx_lm_slot<S, HK, 1, false>(there ? (long long)ps : 0, (t0 + (int)threadIdx.x) % S, head);
        sk = ks[at];
        sv = vs[at];
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
          st_k[buf][lane] = there ? sk * scale : 0.0f;
          st_v[buf][lane] = there ? sv : 0.0f;
        }
      }
      __syncthreads();      // (the other buffer's readers have arrived here before it is written again)
      if (__builtin_expect(t0 + 32 < p1, 1)) {
        fetch(t0 + 32);
        find(t0 + 64);
      }
      const unsigned ok = __builtin_amdgcn_readfirstlane(st_ok[buf]);
      if (__builtin_expect(!ok || row0 >= ROWS, 0)) continue;
      rx_u32x4 kf[2][KF];
      FV vf[NV][8];
      float kscale[8] = {}, vscale[8] = {};
#pragma unroll
      for (int k = 0; k < KF; ++k) {
        kf[0][k] = *(const rx_u32x4*)&kt[buf][r][(k * 4 + g4) * A::NE];
        kf[1][k] = *(const rx_u32x4*)&kt[buf][16 + r][(k * 4 + g4) * A::NE];
      }
      // (not before the weights are done: keys and values in registers at once leave none for a second wavefront)
      auto load_values = [&] {
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
          for (int j = 0; j < NV; ++j) vf[j][i] = *(const FV*)&vt[buf][(i & 4) * 4 + g4 * 4 + (i & 3)][(j * 16 + r) * VE];
      };
      if constexpr (BITS8) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          kscale[i] = st_k[buf][(i & 4) * 4 + g4 * 4 + (i & 3)];
          vscale[i] = st_v[buf][(i & 4) * 4 + g4 * 4 + (i & 3)];
        }
      }
      auto value = [&](const int j, const int e, const int half) {
        rx_u32x4 o;
        if constexpr (A::WIDE) {
#pragma unroll
          for (int i = 0; i < 4; ++i) o[i] = vf[j][half * 4 + i].v[e];
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k) o[k] = __builtin_amdgcn_perm(vf[j][2 * k + 1].v[e >> 1], vf[j][2 * k].v[e >> 1], e & 1 ? 0x07060302u : 0x05040100u);
        }
        return o;
      };
      unsigned seen[NT] = {};
      const bool some = ok != ~0u || differ(t0);
      if (__builtin_expect(some, 0)) look(t0, ok, seen);
      else all = true;
      if constexpr (BITS8) {
        if (__builtin_expect(some, 0)) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (!(__builtin_fabsf(vscale[i]) <= RX_LM_FLT_MAX) && differ(t0)) {
              special |= 1u;              // (those of slots that do not exist are zero already)
              vscale[i] = 0.0f;
            }
        }
      }
      a.step(kf, [&] {
        load_values();
        if (__builtin_expect(some, 0)) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const bool exists = (ok >> ((i & 4) * 4 + g4 * 4 + (i & 3))) & 1u;
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
              for (int n = 0; n < (int)(sizeof(FV) / 4); ++n) {
                // (what lies in other slots, and past a value's end, may be anything, and NaN times a weight of zero is not zero)
                const bool in = exists && (j * 16 + r) * VE < DV;
                const rx_u32 x = in && differ(t0) ? rx_lm_special<F>(vf[j][i].v[n]) : 0u;
                vf[j][i].v[n] &= in ? ~x : 0u;
                special |= x;
              }
          }
        }
      }, value, some, seen, scale, kscale, vscale);
    }
  }

  // Rows that have seen nothing: no maximum, no sum.
#pragma unroll
  for (int t = 0; t < NT; ++t)
    if (!all && rx_lm_rows_max(saw[t] ? 1.0f : 0.0f) == 0.0f) {
      a.m[t] = -rx_lm_inf();
      a.l[t] = 0.0f;
    }
  // (indices from here on are worked out here: what does not depend on the sequence would wait in registers through all of its steps)
  int tid = threadIdx.x;
  rx_pin(tid);
  const int er = tid & 15, eg = (tid & 63) >> 4;
  if constexpr (!SHARED) {
    // the four wavefronts' parts
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      if (t * 16 >= rows) break;
      const float total = rx_lm_sum4(a.l[t]);
      __syncthreads();
      if (eg == 0) {
        join_m[wave][er] = a.m[t];
        join_l[wave][er] = total;
      }
      __syncthreads();
      float top = -rx_lm_inf();
#pragma unroll
      for (int w = 0; w < 4; ++w) top = __builtin_fmaxf(top, join_m[w][er]);
      const float f = top == -rx_lm_inf() ? 0.0f : __builtin_amdgcn_exp2f(a.m[t] - top);
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if (j) __syncthreads();
        if (er < HR) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < VE; ++e) {
              const int d = (eg * 4 + i) * VE + e;
              if (d < WIDTH) lds.o[wave][er][d] = a.acc[t][j][e][i] * f;
            }
        }
        __syncthreads();
        for (int k = tid; k < HR * (WIDTH / VD); k += 256) {
          const int h = k / (WIDTH / VD), c = k % (WIDTH / VD) * VD, d = j * 16 * VE + c, row = t * 16 + h;
          if (row >= rows || d >= DV) continue;
          float o[VD] = {}, sum = 0.0f, hi = -rx_lm_inf();
#pragma unroll
          for (int w = 0; w < 4; ++w) hi = __builtin_fmaxf(hi, join_m[w][h]);
#pragma unroll
          for (int w = 0; w < 4; ++w) {
#pragma unroll
            for (int e = 0; e < VD; ++e) o[e] += lds.o[w][h][c + e];
            sum += hi == -rx_lm_inf() ? 0.0f : join_l[w][h] * __builtin_amdgcn_exp2f(join_m[w][h] - hi);
          }
          if (whole) {
            const long long at = result_of(b, tile * TR + row, head);
            rx_vec<typename E::S, VD> x;
#pragma unroll
            for (int e = 0; e < VD; ++e) x.v[e] = E::down(hi == -rx_lm_inf() ? 0.0f : o[e] / sum);
            rx_store(out + at * DV + d, x);
            if (lse && d == 0) lse[at] = hi == -rx_lm_inf() ? -rx_lm_inf() : (hi - A::SHIFT + __builtin_log2f(sum)) * 0.6931471805599453f;
          } else {
            const long long at = ((long long)id * 2 + (unit == 0)) * RT + row;
            if constexpr (VD == 4) rx_lm_put_shared4(parts_at, (unsigned)(at * DV + d) * 4, rx_f32x4{o[0], o[1], o[2], o[3]});
            else rx_lm_put_shared(part + at * DV + d, o[0]);
            if (d == 0) rx_lm_put_shared((rx_u64*)stat + at, (rx_u64)rx_f2u(hi - A::SHIFT) | (rx_u64)rx_f2u(sum) << 32);
          }
        }
      }
    }
  } else {
    // Every wavefront's rows through its own part of LDS, so that a loop of a few instructions writes rows of consecutive words.
    __syncthreads();
    float* const o = (float*)ring + wave * (16 * (16 * VE + 4));
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const float total = rx_lm_sum4(a.l[t]);
      if (eg == 0) {
        join_m[wave][er] = a.m[t];
        join_l[wave][er] = total;
      }
#pragma unroll
      for (int j = 0; j < NV; ++j) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int e = 0; e < VE; e += 4)
            rx_store(o + er * (16 * VE + 4) + (eg * 4 + i) * VE + e, rx_vec<float, 4>{{a.acc[t][j][e][i], a.acc[t][j][e + 1][i], a.acc[t][j][e + 2][i], a.acc[t][j][e + 3][i]}});
        for (int k = tid & 63; k < 16 * (16 * VE / VD); k += 64) {
          const int h = k / (16 * VE / VD), c = k % (16 * VE / VD) * VD, d = j * 16 * VE + c, row = row0 + t * 16 + h;
          if (row >= ROWS || d >= DV) continue;
          const rx_vec<float, VD> x = rx_load<rx_vec<float, VD>>(o + h * (16 * VE + 4) + c);
          const float hi = join_m[wave][h], sum = join_l[wave][h];
          if (whole) {
            const long long at = result_of(b, row, head);
            rx_vec<typename E::S, VD> y;
#pragma unroll
            for (int e = 0; e < VD; ++e) y.v[e] = E::down(hi == -rx_lm_inf() ? 0.0f : x.v[e] / sum);
            rx_store(out + at * DV + d, y);
            if (lse && d == 0) lse[at] = hi == -rx_lm_inf() ? -rx_lm_inf() : (hi - A::SHIFT + __builtin_log2f(sum)) * 0.6931471805599453f;
          } else {
            const long long at = ((long long)id * 2 + (unit == 0)) * RT + row - tile * TR;
            if constexpr (VD == 4) rx_lm_put_shared4(parts_at, (unsigned)(at * DV + d) * 4, rx_f32x4{x.v[0], x.v[1], x.v[2], x.v[3]});
            else rx_lm_put_shared(part + at * DV + d, x.v[0]);
            if (d == 0) rx_lm_put_shared((rx_u64*)stat + at, (rx_u64)rx_f2u(hi - A::SHIFT) | (rx_u64)rx_f2u(sum) << 32);
          }
        }
      }
    }
  }
  // Infinities and NaN among the values of steps whose rows differ have been taken out (a weight of zero would make them NaN in rows that
  // do not see them): they are added to the results of the rows that do.
  if ((p1 > mixed || (W > 0 && p0 < edge)) && p0 < p1) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // this wavefront's results
  if ((p1 > mixed || (W > 0 && p0 < edge)) && p0 < p1 && __builtin_expect(rx_block_any(special != 0, &any), 0)) {
    for (int k = tid; k < rows * DV; k += 256) {
      const int row = k / DV, d = k % DV, token = (tile * TR + row) / G, first = first_of(token);
      float more = 0.0f;
      for (int p = p0; p < p1; ++p) {
        if (!differ(p & ~31)) {
          p = mixed > p ? mixed - 1 : p;
          continue;
        }
        if (p < span.lo || !sees(token, first, p)) continue;
        const I page = pages[(long long)b * M + p / S];
        if (page < 0 || page >= P) continue;
        float v = C::up(vc[rx_lm_slot<S, HK, DV, BY_SLOT>(page, p % S, head) + d]);
        if constexpr (BITS8) v *= vs[rx_lm_slot<S, HK, 1, false>(page, p % S, head)];
        if (!(__builtin_fabsf(v) <= RX_LM_FLT_MAX)) more += v;
      }
      if (more == 0.0f) continue;
      if (whole) {
        const long long at = result_of(b, tile * TR + row, head) * DV + d;
        out[at] = E::down(E::up(out[at]) + more);
      } else {
        const long long at = (((long long)id * 2 + (unit == 0)) * RT + row) * DV + d;
        rx_lm_put_shared(part + at, rx_lm_get_shared(part + at) + more);
      }
    }
  }
  if (whole) continue;
  const int from = rx_lm_stretch_with(st.total, st.parts, begin), to = rx_lm_stretch_with(st.total, st.parts, begin + span.units - 1);
  if (!rx_lm_last_to_arrive(arrived + b * COLUMNS + column, to - from + 1, &last)) continue;
  // VD outputs to a thread; where there are fewer than threads, the parts are shared too, and joined once more; where there are more,
  // a thread has up to four times VD, so that sixteen loads are on their way.
  constexpr int MORE = RT * (DV / VD) >= 1024 ? 4 : RT * (DV / VD) >= 512 ? 2 : 1, AT = 16 / MORE;
  const int outs = rows * (DV / VD), ways = outs < 256 ? 256 / outs : 1, parts = to - from + 1;
  for (int k0 = 0; k0 < outs; k0 += 256 * MORE) {
    const int way = ways > 1 ? tid / outs : 0, k1 = ways > 1 ? tid % outs : k0 + tid;
    const bool on = k1 < outs && way < ways;
    const int w1 = on ? from + parts * (way + 1) / ways : 0;
    rx_lm_joined<VD> j[MORE];
#pragma unroll
    for (int u = 0; u < MORE; ++u) j[u] = {-rx_lm_inf(), 0.0f, {}};
    for (int w = on ? from + parts * way / ways : 0; w < w1; w += AT) {
      float pm[MORE][AT], psum[MORE][AT], po[MORE][AT][VD];
#pragma unroll
      for (int u = 0; u < MORE; ++u) {
        const int k = k1 + 256 * u < outs ? k1 + 256 * u : k1, h = k / (DV / VD), d = k % (DV / VD) * VD;
#pragma unroll
        for (int i = 0; i < AT; ++i) {
          const int v = w + i < w1 ? w + i : w1 - 1;
          const long long at = ((long long)(v * COLUMNS + column) * 2 + (v == from)) * RT + h;
          const rx_u64 both = rx_lm_get_shared((const rx_u64*)stat + at);
          pm[u][i] = rx_u2f((rx_u32)both);
          psum[u][i] = rx_u2f((rx_u32)(both >> 32));
          if constexpr (VD == 4) {
            const rx_f32x4 x = rx_lm_get_shared4(parts_at, (unsigned)(at * DV + d) * 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) po[u][i][e] = x[e];
          } else {
            po[u][i][0] = rx_lm_get_shared(part + at * DV + d);
          }
        }
      }
#pragma unroll
      for (int u = 0; u < MORE; ++u) {
        float hi = j[u].m;
#pragma unroll
        for (int i = 0; i < AT; ++i) hi = __builtin_fmaxf(hi, pm[u][i]);
        j[u].to(hi);
#pragma unroll
        for (int i = 0; i < AT; ++i)
          if (w + i < w1) j[u].add(pm[u][i], psum[u][i], po[u][i]);
      }
    }
    if (ways > 1) {
      lds.j[tid] = j[0];
      __syncthreads();
      if (way == 0)
        for (int n = 1; n < ways; ++n) {
          const rx_lm_joined<VD> o = lds.j[n * outs + k1];
          j[0].to(__builtin_fmaxf(j[0].m, o.m));
          j[0].add(o.m, o.s, o.o);
        }
    }
    if (!on || way) continue;
#pragma unroll
    for (int u = 0; u < MORE; ++u) {
      const int k = k1 + 256 * u, h = k / (DV / VD), d = k % (DV / VD) * VD;
      if (k >= outs) break;
      const long long at = result_of(b, tile * TR + h, head);
      rx_vec<typename E::S, VD> x;
#pragma unroll
      for (int e = 0; e < VD; ++e) x.v[e] = E::down(j[u].m == -rx_lm_inf() ? 0.0f : j[u].o[e] / j[u].s);
      rx_store(out + at * DV + d, x);
      if (lse && d == 0) lse[at] = j[u].m == -rx_lm_inf() ? -rx_lm_inf() : (j[u].m + __builtin_log2f(j[u].s)) * 0.6931471805599453f;
    }
  }
  }
}
