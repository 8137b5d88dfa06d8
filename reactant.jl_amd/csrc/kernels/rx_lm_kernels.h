// Device code of the language-model operators (csrc/rx_lm.h states what they compute).
#pragma once
#include "rx_preamble.h"

// element types: storage, and conversion to and from the f32 that everything is computed in
struct rx_lm_f32 {
  typedef float S;
  RX_MEM static float up(S x) { return x; }
  RX_MEM static S down(float x) { return x; }
};
struct rx_lm_bf16 {
  typedef rx_u16 S;
  RX_MEM static float up(S x) { return rx_bf16_to_f32(x); }
  RX_MEM static S down(float x) { return rx_f32_to_bf16(x); }
};
struct rx_lm_f16 {
  typedef rx_u16 S;
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

// attention of one token: a wavefront per query head goes through the positions, with the running maximum and sum
template <typename E, int HQ, int HK, int DK, int DV, int P, int S, int M, int W, bool BY_SLOT, typename I>
RX_DEV void rx_paged_attention(const typename E::S* q, const typename E::S* kc, const typename E::S* vc, const I* pages, const I* lengths, typename E::S* out, float* lse,
                               const float scale) {
  const int h = blockIdx.x, lane = threadIdx.x;
  const long long b = blockIdx.y;
  constexpr int NK = (DK + 63) / 64, NV = (DV + 63) / 64;
  float qr[NK], acc[NV] = {};
#pragma unroll
  for (int j = 0; j < NK; ++j) qr[j] = lane + 64 * j < DK ? E::up(q[(b * HQ + h) * DK + lane + 64 * j]) * scale : 0.0f;
  const I len = lengths[b];
  const int n = len < 0 ? 0 : len > (I)(M * S) ? M * S : (int)len;
  float m = -rx_lm_inf(), sum = 0.0f;
  for (int t = W && n > W ? n - W : 0; t < n; ++t) {
    const I page = pages[b * M + t / S];
    if (page < 0 || page >= P) continue;
    const typename E::S* kp = kc + rx_lm_slot<S, HK, DK, BY_SLOT>(page, t % S, h / (HQ / HK));
    const typename E::S* vp = vc + rx_lm_slot<S, HK, DV, BY_SLOT>(page, t % S, h / (HQ / HK));
    float d = 0.0f;
#pragma unroll
    for (int j = 0; j < NK; ++j)
      if (lane + 64 * j < DK) d = __builtin_fmaf(qr[j], E::up(kp[lane + 64 * j]), d);
    d = rx_wave_reduce(d, rx_op_add());
    const float m2 = rx_max(m, d), r = m2 == -rx_lm_inf() ? 1.0f : expf(m - m2), p = m2 == -rx_lm_inf() ? 0.0f : expf(d - m2);
    sum = sum * r + p;
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (lane + 64 * j < DV) acc[j] = acc[j] * r + p * E::up(vp[lane + 64 * j]);
    m = m2;
  }
#pragma unroll
  for (int j = 0; j < NV; ++j)
    if (lane + 64 * j < DV) out[(b * HQ + h) * DV + lane + 64 * j] = E::down(sum == 0.0f ? 0.0f : acc[j] / sum);
  if (lse && lane == 0) lse[b * HQ + h] = sum == 0.0f ? -rx_lm_inf() : m + logf(sum);
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
