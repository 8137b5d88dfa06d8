// Device code of the language-model operators (csrc/rx_lm.h states what they compute).
#pragma once
#include "rx_preamble.h"
#include "rx_gemm_kernels.h"

// element types: storage, and conversion to and from the f32 that everything is computed in
struct rx_lm_f32 {
  typedef float S;
  static constexpr bool BF16 = false;
  RX_MEM static float up(S x) { return x; }
  RX_MEM static S down(float x) { return x; }
};
struct rx_lm_bf16 {
  typedef rx_u16 S;
  static constexpr bool BF16 = true;
  RX_MEM static float up(S x) { return rx_bf16_to_f32(x); }
  RX_MEM static S down(float x) { return rx_f32_to_bf16(x); }
};
struct rx_lm_f16 {
  typedef rx_u16 S;
  static constexpr bool BF16 = false;
  RX_MEM static float up(S x) { return rx_f16_to_f32(x); }
  // (apart from the product that x comes from: the two together become one instruction that rounds once, not to f32 first)
  RX_MEM static S down(float x) { return rx_f32_to_f16(rx_apart(x)); }
};

#define RX_LM_LOG2E 1.4426950408889634f
RX_DEV float rx_lm_inf() { return __builtin_inff(); }

// ---------------------------------------------------------------------------
// embedding: a thread per vector of VEC elements
// ---------------------------------------------------------------------------
template <typename E, int V, int D, int T, int VEC, typename I>
RX_DEV void rx_embedding(const typename E::S* table, const I* ids, typename E::S* out, const float scale) {
  constexpr int C = D / VEC;   // vectors of a row
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= (long long)T * C) return;
  const int t = (int)(i / C), c = (int)(i % C);
  const I id = ids[t];
  rx_vec<typename E::S, VEC> x{};
  if (id >= 0 && id < V) {
    x = rx_load<rx_vec<typename E::S, VEC>>(table + (long long)id * D + c * VEC);
#pragma unroll
    for (int k = 0; k < VEC; ++k) x.v[k] = E::down(E::up(x.v[k]) * scale);
  }
  rx_store(out + (long long)t * D + c * VEC, x);
}

// gradient: a workgroup per row of the table, which goes through the tokens
template <typename E, typename O, int D, int T, typename I>
RX_DEV void rx_embedding_grad(const typename E::S* dy, const I* ids, typename O::S* out, const float scale) {
  const int row = blockIdx.x;
  __shared__ int found[256];
  for (int c0 = 0; c0 < D; c0 += 256) {
    const int c = c0 + (int)threadIdx.x;
    float sum = 0.0f;
    for (int t0 = 0; t0 < T; t0 += 256) {
      const int t = t0 + (int)threadIdx.x;
      const bool hit = t < T && ids[t] == row;
      if (!__syncthreads_or(hit)) continue;
      found[threadIdx.x] = hit;
      __syncthreads();
      for (int k = 0; k < 256; ++k)
        if (found[k] && c < D) sum += E::up(dy[(long long)(t0 + k) * D + c]);
      __syncthreads();
    }
    if (c < D) out[(long long)row * D + c] = O::down(sum * scale);
  }
}

// ---------------------------------------------------------------------------
// paged cache
// ---------------------------------------------------------------------------
// offset of a slot's head in a cache of pages of S slots, H heads of D elements
template <int S, int H, int D, bool BY_SLOT>
RX_DEV long long rx_lm_slot(long long page, int slot, int head) {
  return BY_SLOT ? ((page * S + slot) * H + head) * D : ((page * H + head) * S + slot) * D;
}

// one element of a head after rotation: x cos - y sin for the first of a pair, y cos + x sin for the second
template <typename E, int R2, bool PAIRS>
RX_DEV float rx_lm_rotated(const typename E::S* head, int d, const float* cos, const float* sin) {
  const float x = E::up(head[d]);
  if (d >= 2 * R2) return x;
  const int a = PAIRS ? d >> 1 : (d < R2 ? d : d - R2);
  const bool second = PAIRS ? (d & 1) : d >= R2;
  const float y = E::up(head[second ? (PAIRS ? d - 1 : d - R2) : (PAIRS ? d + 1 : d + R2)]);
  return second ? x * cos[a] + y * sin[a] : x * cos[a] - y * sin[a];
}

// a workgroup per token
template <typename E, int HQ, int HK, int DK, int DV, int P, int S, int B, int M, int L, int R2, bool PAIRS, bool BY_SLOT, typename I>
RX_DEV void rx_kv_append(const typename E::S* q, const typename E::S* k, const typename E::S* v, const float* cos, const float* sin, const I* position, const I* sequence,
                         const I* pages, typename E::S* qo, typename E::S* kc, typename E::S* vc) {
  const long long t = blockIdx.x;
  const I pos = position[t], seq = sequence[t];
  const bool known = pos >= 0 && pos < (R2 ? (long long)L : (long long)M * S) && pos < (long long)M * S && seq >= 0 && seq < B;
  const float* c = cos + (known ? (long long)pos * R2 : 0);
  const float* s = sin + (known ? (long long)pos * R2 : 0);
  for (int i = threadIdx.x; i < HQ * DK; i += 256)
    qo[t * (HQ * DK) + i] = known ? E::down(rx_lm_rotated<E, R2, PAIRS>(q + t * (HQ * DK) + i / DK * DK, i % DK, c, s)) : E::down(0.0f);
  if (!known) return;
  const I page = pages[(long long)seq * M + pos / S];
  if (page < 0 || page >= P) return;
  const int slot = (int)(pos % S);
  for (int i = threadIdx.x; i < HK * DK; i += 256)
    kc[rx_lm_slot<S, HK, DK, BY_SLOT>(page, slot, i / DK) + i % DK] = E::down(rx_lm_rotated<E, R2, PAIRS>(k + t * (HK * DK) + i / DK * DK, i % DK, c, s));
  for (int i = threadIdx.x; i < HK * DV; i += 256) vc[rx_lm_slot<S, HK, DV, BY_SLOT>(page, slot, i / DV) + i % DV] = v[t * (HK * DV) + i];
}

// ---- attention of one token per sequence ----
// One pass over keys and values with the running maximum and sum of the softmax, on the matrix cores without LDS: a wavefront
// takes 32 positions at a time.  Scores are K Q' (MFMA rows are positions, columns the query heads of one key head), the result
// is V' P' (rows are dimensions, columns heads): column h of both lies in the lanes l with l mod 16 = h, so the maximum, the
// sum and the weights of a head stay in its lanes, and the weights leave the first product in the registers in which the
// second one takes them (which of its k is which position is free as long as V follows suit).  V' needs the values of one
// dimension at consecutive positions: a lane loads 16 bytes (8 dimensions) of 8 positions, and bytes are permuted in registers.
//
// The positions of all sequences are cut into about ITEMS chunks, equal within a sequence and as long as the sum of the lengths
// asks for (multiples of 128: four wavefronts, 32 each), so that a batch of uneven lengths fills the chip; every workgroup works
// the cut out from the lengths.  A sequence of one chunk is finished here; those of several leave (maximum, sum, unscaled
// result) and rx_paged_attention_join combines them.
struct rx_lm_cut { int n, lo, size, count; };   // length, first position, positions of a chunk (from lo rounded down to 128), chunks
template <int S, int M, int W, typename I>
RX_DEV int rx_lm_length(const I len) { return len < 0 ? 0 : len > (I)(M * S) ? M * S : (int)len; }
template <int W>
RX_DEV int rx_lm_first(const int n) { return W && n > W ? n - W : 0; }
template <int W>
RX_DEV rx_lm_cut rx_lm_cut_of(const int n, const int chunk) {
  rx_lm_cut c;
  c.n = n;
  c.lo = rx_lm_first<W>(n);
  const int tokens = n - (c.lo & ~127);
  const int k = tokens > chunk ? (tokens + chunk - 1) / chunk : 1;
  c.size = tokens > 0 ? ((tokens + k - 1) / k + 127) & ~127 : 128;
  c.count = tokens > c.size ? (tokens + c.size - 1) / c.size : 1;
  return c;
}
// chunk length for all sequences: every wavefront works it out for itself
template <int S, int B, int M, int W, int COLUMNS, int ITEMS, typename I>
RX_DEV int rx_lm_chunk(const I* lengths) {
  const int lane = threadIdx.x & 63;
  long long total = 0;
  for (int b = lane; b < B; b += 64) {
    const int n = rx_lm_length<S, M, W>(lengths[b]);
    total += n - (rx_lm_first<W>(n) & ~127);
  }
  if constexpr (B > 1) total = rx_wave_reduce(total, rx_op_add());
  else total = rx_lane_from(total, 0);
  const long long per = (total * COLUMNS + ITEMS - 1) / ITEMS;
  return per < 128 ? 128 : (int)((per + 127) & ~127ll);
}
// the sequence that item `item` (in units of COLUMNS items) belongs to, and the number of chunks before it; B where there is none
template <int S, int B, int M, int W, typename I>
RX_DEV int rx_lm_find(const I* lengths, const int chunk, const int item, int* before) {
  const int lane = threadIdx.x & 63;
  int sum = 0;
  for (int b0 = 0; b0 < B; b0 += 64) {
    const int b = b0 + lane;
    const int count = b < B ? rx_lm_cut_of<W>(rx_lm_length<S, M, W>(lengths[b]), chunk).count : 0;
    const int upto = sum + rx_wave_scan(count, rx_op_add());
    const unsigned long long past = __ballot(b < B && upto > item);
    if (past) {
      const int first = __builtin_ctzll(past);
      *before = rx_lane_from(upto - count, first);
      return __builtin_amdgcn_readfirstlane(b0 + first);
    }
    sum = rx_lane_from(upto, 63);
  }
  return B;
}

// maximum over the four lanes that hold one head's positions (l, l ^ 16, l ^ 32, l ^ 48)
RX_DEV float rx_lm_max4(float x) {
  x = __builtin_fmaxf(x, rx_lane_from(x, (threadIdx.x & 63) ^ 16));
  return __builtin_fmaxf(x, rx_lane_from(x, (threadIdx.x & 63) ^ 32));
}
RX_DEV float rx_lm_sum4(float x) {
  x += rx_lane_from(x, (threadIdx.x & 63) ^ 16);
  return x + rx_lane_from(x, (threadIdx.x & 63) ^ 32);
}

// 16 bytes of a head's row from element d on; zeros past its end (D: elements of the row)
template <typename E, int D>
RX_DEV rx_u32x4 rx_lm_row16(const typename E::S* row, const int d) {
  constexpr int NE = 16 / sizeof(typename E::S);
  rx_u32x4 v = {0, 0, 0, 0};
  if constexpr (D % NE == 0) {
    if (d < D) v = *(const rx_u32x4*)(row + d);
  } else {
    rx_vec<typename E::S, NE> w{};
#pragma unroll
    for (int k = 0; k < NE; ++k)
      if (d + k < D) w.v[k] = row[d + k];
    v = __builtin_bit_cast(rx_u32x4, w);
  }
  return v;
}

template <typename E>
RX_DEV rx_f32x4 rx_lm_mma(const rx_u32x4 a, const rx_u32x4 b, rx_f32x4 c) {
  if constexpr (sizeof(typename E::S) == 4) {
    const rx_f32x4 x = __builtin_bit_cast(rx_f32x4, a), y = __builtin_bit_cast(rx_f32x4, b);
#pragma unroll
    for (int k = 0; k < 4; ++k) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[k], y[k], c, 0, 0, 0);
    return c;
  } else if constexpr (E::BF16) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(rx_bf16x8, a), __builtin_bit_cast(rx_bf16x8, b), c, 0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(rx_f16x8, a), __builtin_bit_cast(rx_f16x8, b), c, 0, 0, 0);
  }
}

// HT: query heads of an item (those of one key head, up to 16 NT of them at a time); COLUMNS: items per chunk of a sequence
template <typename E, int HQ, int HK, int DK, int DV, int P, int S, int B, int M, int W, bool BY_SLOT, int NT, int ITEMS, bool JOIN, typename I>
RX_DEV void rx_paged_attention(const typename E::S* q, const typename E::S* kc, const typename E::S* vc, const I* pages, const I* lengths, typename E::S* out, float* lse,
                               float* part, float* stat, const float scale) {
  typedef typename E::S T;
  constexpr int NE = 16 / sizeof(T);                   // elements of 16 bytes
  constexpr int G = HQ / HK, GT = G < 16 * NT ? G : 16 * NT, TILES = (G + GT - 1) / GT, COLUMNS = HK * TILES;
  constexpr int NK = (DK + 4 * NE - 1) / (4 * NE);     // 16-byte loads of a position's key by its four lanes
  constexpr int NV = (DV + 16 * NE - 1) / (16 * NE);   // of a position's value by sixteen lanes
  constexpr int BLOCK = 2048;                          // positions whose pages are held in LDS
  constexpr float SHIFT = sizeof(T) == 2 && !E::BF16 ? 15.0f : 0.0f;   // f16 weights are taken times 2^15: the smallest would be lost below 2^-24
  constexpr int HR = GT < 16 ? GT : 16, WIDTH = 16 * NE < DV ? 16 * NE : DV;   // heads and dimensions that are joined at a time
  __shared__ union {
    int page[BLOCK / S + 2];
    float o[4][HR][WIDTH + 4];
  } lds;
  __shared__ float join_m[4][16], join_l[4][16];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, r = lane & 15, g4 = lane >> 4;
  const int chunk = JOIN ? rx_lm_chunk<S, B, M, W, COLUMNS, ITEMS>(lengths) : 1 << 30;

  const int item = blockIdx.x;
  int before = 0;
  const int b = B == 1 ? (item / COLUMNS < rx_lm_cut_of<W>(rx_lm_length<S, M, W>(lengths[0]), chunk).count ? 0 : B)
                       : JOIN ? rx_lm_find<S, B, M, W>(lengths, chunk, item / COLUMNS, &before) : (before = item / COLUMNS);
  if (b >= B) return;
  const rx_lm_cut cut = rx_lm_cut_of<W>(rx_lm_length<S, M, W>(lengths[b]), chunk);
  const int column = item % COLUMNS, head = column / TILES, tile = column % TILES;
  const int p0 = (cut.lo & ~127) + (item / COLUMNS - before) * cut.size;
  const int p1 = P == 0 ? p0 : p0 + cut.size < cut.n ? p0 + cut.size : cut.n;
  const int h0 = head * G + tile * GT;                 // first query head
  const int heads = G - tile * GT < GT ? G - tile * GT : GT;

  rx_u32x4 qf[NT][NK];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int k = 0; k < NK; ++k)
      qf[t][k] = t * 16 + r < heads ? rx_lm_row16<E, DK>(q + ((long long)b * HQ + h0 + t * 16 + r) * DK, (k * 4 + g4) * NE) : rx_u32x4{0, 0, 0, 0};

  float m[NT], l[NT];
  rx_f32x4 acc[NT][NV][NE];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    m[t] = -rx_lm_inf();
    l[t] = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < NE; ++e) acc[t][j][e] = rx_f32x4{0, 0, 0, 0};
  }

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
    auto where = [&](const int t) { return t >= cut.lo && t < s1 ? lds.page[t / S - page0] : -1; };
    for (int t0 = s0 + wave * 32; t0 < s1; t0 += 128) {
      const int ta = t0 + r, tb = ta + 16, pa = where(ta), pb = where(tb);
      const unsigned ok = ((unsigned)__ballot(pa >= 0) & 0xffffu) | ((unsigned)__ballot(pb >= 0) << 16);
      if (!ok) continue;
      rx_u32x4 kf[2][NK], vf[NV][8];
      const T* ka = kc + rx_lm_slot<S, HK, DK, BY_SLOT>(pa < 0 ? 0 : pa, ta % S, head);
      const T* kb = kc + rx_lm_slot<S, HK, DK, BY_SLOT>(pb < 0 ? 0 : pb, tb % S, head);
#pragma unroll
      for (int k = 0; k < NK; ++k) {
        kf[0][k] = rx_lm_row16<E, DK>(ka, (k * 4 + g4) * NE);
        kf[1][k] = rx_lm_row16<E, DK>(kb, (k * 4 + g4) * NE);
      }
      // values of positions t0 + 4 g4 + (0..3) and 16 further: where a page's slots are a multiple of four, on two pages
      int pv = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int tv = t0 + (i & 4) * 4 + g4 * 4 + (i & 3);
        if (S % 4 != 0 || i % 4 == 0) {
          pv = where(S % 4 == 0 ? (tv + 3 < s1 ? tv + 3 : s1 - 1) : tv);   // (the group's first positions may lie before cut.lo)
          if (S % 4 == 0 && tv >= s1) pv = -1;
        }
        const T* v = vc + rx_lm_slot<S, HK, DV, BY_SLOT>(pv < 0 ? 0 : pv, tv % S, head);
#pragma unroll
        for (int j = 0; j < NV; ++j) vf[j][i] = rx_lm_row16<E, DV>(v, (j * 16 + r) * NE);
      }
      const unsigned mine = (ok >> (g4 * 4)) & 0x000f000fu;      // bit i: position 4 g4 + i, bit 16 + i: 16 further
      if (ok != ~0u) {
        // what lies in other slots may be anything, and NaN times a weight of zero is not zero
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (!((mine >> ((i & 4) * 4 + (i & 3))) & 1u)) {
#pragma unroll
            for (int j = 0; j < NV; ++j) vf[j][i] = rx_u32x4{0, 0, 0, 0};
          }
      }
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        rx_f32x4 s[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
        for (int k = 0; k < NK; ++k) {
          s[0] = rx_lm_mma<E>(kf[0][k], qf[t][k], s[0]);
          s[1] = rx_lm_mma<E>(kf[1][k], qf[t][k], s[1]);
        }
        float x[8], top = -rx_lm_inf();
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = s[i >> 2][i & 3] * scale;
        if (ok != ~0u) {
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] = (mine >> ((i & 4) * 4 + (i & 3))) & 1u ? x[i] : -rx_lm_inf();
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) top = __builtin_fmaxf(top, x[i]);
        top = __builtin_fmaxf(m[t], rx_lm_max4(top));
        const float base = top == -rx_lm_inf() ? 0.0f : top;     // (a head whose scores are all -inf so far)
        if (__any(top != m[t])) {
          const float shrink = __builtin_amdgcn_exp2f(m[t] - base);
          l[t] *= shrink;
#pragma unroll
          for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int e = 0; e < NE; ++e) acc[t][j][e] *= shrink;
          m[t] = top;
        }
        rx_vec<T, 8> w;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float p = __builtin_amdgcn_exp2f(x[i] - base + SHIFT);
          l[t] += p;                                             // (in f32: lse is as exact as the scores)
          w.v[i] = E::down(p);                                   // rounded to the cache's type, in which the matrix cores take it
        }
        if constexpr (NE == 8) {
          const rx_u32x4 p = __builtin_bit_cast(rx_u32x4, w);
#pragma unroll
          for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              rx_u32x4 a;
#pragma unroll
              for (int k = 0; k < 4; ++k) a[k] = __builtin_amdgcn_perm(vf[j][2 * k + 1][e >> 1], vf[j][2 * k][e >> 1], e & 1 ? 0x07060302u : 0x05040100u);
              acc[t][j][e] = rx_lm_mma<E>(a, p, acc[t][j][e]);
            }
        } else {
#pragma unroll
          for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int e = 0; e < NE; ++e)
#pragma unroll
              for (int i = 0; i < 8; ++i)
                acc[t][j][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(rx_f32x4, vf[j][i])[e], w.v[i], acc[t][j][e], 0, 0, 0);
        }
      }
    }
  }

  // the four wavefronts' parts of the chunk
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    if (t * 16 >= heads) break;
    const float total = rx_lm_sum4(l[t]);
    __syncthreads();
    if (g4 == 0) {
      join_m[wave][r] = m[t];
      join_l[wave][r] = total;
    }
    __syncthreads();
    float top = -rx_lm_inf();
#pragma unroll
    for (int w = 0; w < 4; ++w) top = __builtin_fmaxf(top, join_m[w][r]);
    const float f = top == -rx_lm_inf() ? 0.0f : __builtin_amdgcn_exp2f(m[t] - top);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (j) __syncthreads();
      if (r < HR) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int e = 0; e < NE; ++e) {
            const int d = (g4 * 4 + i) * NE + e;
            if (d < WIDTH) lds.o[wave][r][d] = acc[t][j][e][i] * f;
          }
      }
      __syncthreads();
      for (int k = threadIdx.x; k < HR * WIDTH; k += 256) {
        const int h = k / WIDTH, d = j * 16 * NE + k % WIDTH;
        if (t * 16 + h >= heads) break;
        if (d >= DV) continue;
        float o = 0.0f, sum = 0.0f, hi = -rx_lm_inf();
#pragma unroll
        for (int w = 0; w < 4; ++w) hi = __builtin_fmaxf(hi, join_m[w][h]);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          o += lds.o[w][h][k % WIDTH];
          sum += hi == -rx_lm_inf() ? 0.0f : join_l[w][h] * __builtin_amdgcn_exp2f(join_m[w][h] - hi);
        }
        const int qh = h0 + t * 16 + h;
        if (!JOIN || cut.count == 1) {
          out[((long long)b * HQ + qh) * DV + d] = E::down(sum == 0.0f ? 0.0f : o / sum);
          if (lse && d == 0) lse[(long long)b * HQ + qh] = sum == 0.0f ? -rx_lm_inf() : (hi - SHIFT + __builtin_log2f(sum)) * 0.6931471805599453f;
        } else {
          part[((long long)item * GT + t * 16 + h) * DV + d] = o;
          if (d == 0) {
            stat[((long long)item * GT + t * 16 + h) * 2] = hi - SHIFT;
            stat[((long long)item * GT + t * 16 + h) * 2 + 1] = sum;
          }
        }
      }
    }
  }
}

// a workgroup per query head of a sequence of several chunks: the chunks' results in their order
template <typename E, int HQ, int HK, int DV, int S, int B, int M, int W, int NT, int ITEMS, typename I>
RX_DEV void rx_paged_attention_join(const I* lengths, const float* part, const float* stat, typename E::S* out, float* lse) {
  constexpr int G = HQ / HK, GT = G < 16 * NT ? G : 16 * NT, TILES = (G + GT - 1) / GT, COLUMNS = HK * TILES;
  const int b = blockIdx.y, qh = blockIdx.x, lane = threadIdx.x & 63;
  const int chunk = rx_lm_chunk<S, B, M, W, COLUMNS, ITEMS>(lengths);
  const rx_lm_cut cut = rx_lm_cut_of<W>(rx_lm_length<S, M, W>(lengths[b]), chunk);
  if (cut.count == 1) return;
  int before = 0;
  for (int k = lane; k < b; k += 64) before += rx_lm_cut_of<W>(rx_lm_length<S, M, W>(lengths[k]), chunk).count;
  if constexpr (B > 1) before = rx_wave_reduce(before, rx_op_add());
  const int tile = qh % G / GT, h = qh % G % GT, column = qh / G * TILES + tile;
  float top = -rx_lm_inf();
  for (int c = 0; c < cut.count; ++c) top = __builtin_fmaxf(top, stat[((long long)((before + c) * COLUMNS + column) * GT + h) * 2]);
  for (int d = threadIdx.x; d < DV; d += 256) {
    float o = 0.0f, sum = 0.0f;
    for (int c = 0; c < cut.count; ++c) {
      const long long at = (long long)((before + c) * COLUMNS + column) * GT + h;
      const float f = top == -rx_lm_inf() ? 0.0f : __builtin_amdgcn_exp2f(stat[at * 2] - top);
      o += f * part[at * DV + d];
      sum += f * stat[at * 2 + 1];
    }
    out[((long long)b * HQ + qh) * DV + d] = E::down(sum == 0.0f ? 0.0f : o / sum);
    if (lse && d == 0) lse[(long long)b * HQ + qh] = sum == 0.0f ? -rx_lm_inf() : (top + __builtin_log2f(sum)) * 0.6931471805599453f;
  }
}

// ---------------------------------------------------------------------------
// token log probabilities
// ---------------------------------------------------------------------------
// order of logits as whole numbers: larger value first, then the lower index; NaN counts as the largest, zeros are equal
RX_DEV rx_u32 rx_lm_order(float x) {
  if (x != x) return 0xffffffffu;
  const rx_u32 u = rx_f2u(x + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
RX_DEV rx_u64 rx_lm_key(float x, int j) { return ((rx_u64)rx_lm_order(x) << 32) | (rx_u32)~j; }

// a workgroup per row
template <typename E, int V, int K, typename I>
RX_DEV void rx_token_logprobs(const typename E::S* logits, const I* targets, float* logprob, float* lse, float* entropy, float* values, int* ids) {
  const long long t = blockIdx.x;
  const typename E::S* x = logits + t * V;
  __shared__ float red[4];
  __shared__ rx_u64 red64[4];
  float m = -rx_lm_inf();
  for (int j = threadIdx.x; j < V; j += 256) m = rx_max(m, E::up(x[j]));
  m = rx_block_reduce<float, rx_op_max, 4>(m, rx_op_max(), red);
  float s = 0.0f, sx = 0.0f;
  if (m != -rx_lm_inf())
    for (int j = threadIdx.x; j < V; j += 256) {
      const float v = E::up(x[j]);
      const float e = expf(v - m);
      s += e;
      if (v != -rx_lm_inf()) sx += e * (v - m);
    }
  __syncthreads();
  s = rx_block_reduce<float, rx_op_add, 4>(s, rx_op_add(), red);
  __syncthreads();
  sx = rx_block_reduce<float, rx_op_add, 4>(sx, rx_op_add(), red);
  const float l = s == 0.0f ? -rx_lm_inf() : m + logf(s);
  if (threadIdx.x == 0) {
    const I y = targets[t];
    lse[t] = l;
    entropy[t] = s == 0.0f ? 0.0f : logf(s) - sx / s;
    logprob[t] = y < 0 || y >= V ? 0.0f : s == 0.0f ? -rx_lm_inf() : E::up(x[y]) - l;
  }
  rx_u64 below = ~0ull;   // keys from here on have been taken
  for (int k = 0; k < K; ++k) {
    rx_u64 best = 0;
    for (int j = threadIdx.x; j < V; j += 256) {
      const rx_u64 key = rx_lm_key(E::up(x[j]), j);
      if (key < below && key > best) best = key;
    }
    __syncthreads();
    best = rx_block_reduce<rx_u64, rx_op_max, 4>(best, rx_op_max(), red64);
    if (threadIdx.x == 0) {
      const int j = (int)~(rx_u32)best;
      ids[t * K + k] = j;
      values[t * K + k] = s == 0.0f ? -rx_lm_inf() : E::up(x[j]) - l;
    }
    below = best;
  }
}

// d x_j = g (delta_jy - p_j) - h p_j (x_j - lse + H): a workgroup per row
template <typename E, int V, typename I>
RX_DEV void rx_token_logprobs_grad(const typename E::S* logits, const I* targets, const float* lse, const float* entropy, const float* d_logprob, const float* d_entropy,
                                   typename E::S* out) {
  const long long t = blockIdx.x;
  const typename E::S* x = logits + t * V;
  const I y = targets[t];
  const bool counts = y >= 0 && y < V;
  const float l = lse[t], H = entropy[t], g = counts ? d_logprob[t] : 0.0f, h = d_entropy[t];
  for (int j = threadIdx.x; j < V; j += 256) {
    const float z = E::up(x[j]) - l, p = l == -rx_lm_inf() ? 0.0f : expf(z);
    float d = p == 0.0f ? 0.0f : -p * (g + h * (z + H));
    if (counts && j == y) d += g;
    out[t * V + j] = E::down(d);
  }
}
