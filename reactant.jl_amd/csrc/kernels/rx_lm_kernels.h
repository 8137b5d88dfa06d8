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

// Values handed to the workgroup of the same launch that arrives last, on whichever die it runs: written and read past the
// caches that belong to one die (device-scope atomic accesses), and counted in once the writes have arrived.  No workgroup
// waits for another.  The counter is zero before the launch, and again after it.
template <typename T>
RX_DEV void rx_lm_put_shared(T* p, const T v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
template <typename T>
RX_DEV T rx_lm_get_shared(const T* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
RX_DEV bool rx_lm_last_to_arrive(int* counter, const int expected, int* flag) {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // this wavefront's writes
  __syncthreads();
  if (threadIdx.x == 0) {
    const bool l = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == expected - 1;
    if (l) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    *flag = l;
  }
  __syncthreads();
  const bool l = *flag != 0;
  __syncthreads();
  return l;
}

#define RX_LM_LOG2E 1.4426950408889634f
#define RX_LM_FLT_MAX 3.4028234663852886e38f
RX_DEV float rx_lm_inf() { return __builtin_inff(); }

// ---------------------------------------------------------------------------
// embedding: EACH vectors of VEC elements to a thread, 256 apart, loaded before the first is stored.  Bound by memory: 16384 tokens
// of 4096 bf16 from 32000 rows, 186 MB with each row read once, take 32 us (5.8 TB/s), with
// non-temporal stores, which leave the caches to the table's repeated rows; 44 us without.
// ---------------------------------------------------------------------------
template <typename E, int V, int D, int T, int VEC, int EACH, typename I>
RX_DEV void rx_embedding(const typename E::S* table, const I* ids, typename E::S* out, const float scale) {
  constexpr int C = D / VEC;   // vectors of a row
  typedef rx_vec<typename E::S, VEC> W;
  for (long long i0 = (long long)blockIdx.x * (256 * EACH) + threadIdx.x; i0 < (long long)T * C; i0 += (long long)gridDim.x * (256 * EACH)) {
    W x[EACH];
    bool known[EACH];
#pragma unroll
    for (int n = 0; n < EACH; ++n) {
      const long long i = i0 + 256 * n < (long long)T * C ? i0 + 256 * n : i0;
      const I id = ids[i / C];
      known[n] = id >= 0 && id < V;
      x[n] = V ? rx_load<W>(table + (known[n] ? (long long)id * D : 0) + i % C * VEC) : W{};
    }
#pragma unroll
    for (int n = 0; n < EACH; ++n) {
      const long long i = i0 + 256 * n;
      if (i >= (long long)T * C) break;
#pragma unroll
      for (int k = 0; k < VEC; ++k) x[n].v[k] = known[n] ? E::down(E::up(x[n].v[k]) * scale) : E::down(0.0f);
      rx_store_nt(out + i * VEC, x[n]);
    }
  }
}

// Gradient.  The tokens are sorted by row, in their order within a row, by one launch without exchange between workgroups: a
// workgroup has the counters of ROWS rows in LDS and goes through all tokens twice.  The first time it counts its rows' tokens,
// for every wavefront's stretch of the tokens apart, and the tokens of rows before its own, which is where its part of the
// sorted list starts; the second time every wavefront puts its tokens into their places.  All counts are whole numbers, so the
// list is the same every run.  `start` [V + 1] is where a row's tokens start in `order`; `row_of` is the row of a place.
// 16384 tokens, 65536 rows, 256 workgroups of 256 rows: 9.7 us, two passes over the ids (which a wavefront keeps in registers
// between the two, up to 32 of them a lane) and their chains of LDS counters; atomics on sums of rows in memory would need no list,
// but their order, and with it the sums' last bits, would be another every run.
template <int V, int T, int ROWS, typename I>
RX_DEV void rx_lm_sort(const I* ids, int* start, int* order, int* row_of) {
  constexpr int WAVES = 16, EACH = ((T + WAVES - 1) / WAVES + 63) / 64, STRETCH = EACH * 64;
  constexpr int KEPT = EACH <= 32 ? EACH : 1;                   // a wavefront's tokens stay in registers where they fit
  __shared__ int counts[WAVES][ROWS], sums[WAVES];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, r0 = blockIdx.x * ROWS, t0 = wave * STRETCH, t1 = t0 + STRETCH < T ? t0 + STRETCH : T;
  int kept[KEPT];                                               // -1: no row of the table
  if constexpr (KEPT == EACH) {
#pragma unroll
    for (int k = 0; k < KEPT; ++k) {
      const I id = ids[t0 + lane + 64 * k < T ? t0 + lane + 64 * k : T - 1];
      kept[k] = t0 + lane + 64 * k < T && id >= 0 && id < V ? (int)id : -1;
    }
  }
  for (int k = threadIdx.x; k < WAVES * ROWS; k += 1024) counts[k / ROWS][k % ROWS] = 0;
  __syncthreads();
  int below = 0;
  auto tally = [&](const int id) {
    if (id >= 0 && id < r0) ++below;
    else if (id >= r0 && id < (long long)r0 + ROWS) atomicAdd(&counts[wave][id - r0], 1);
  };
  if constexpr (KEPT == EACH) {
#pragma unroll
    for (int k = 0; k < KEPT; ++k) tally(kept[k]);
  } else {
#pragma unroll 4
    for (int t = t0 + lane; t < t1; t += 64) {
      const I id = ids[t];
      tally(id >= 0 && id < V ? (int)id : -1);
    }
  }
  below = rx_wave_reduce(below, rx_op_add());
  if (lane == 0) sums[wave] = below;
  __syncthreads();
  below = 0;
  for (int w = 0; w < WAVES; ++w) below += sums[w];
  __syncthreads();
  // places: rows one after the other, a row's stretches one after the other
  int carry = below;
  for (int k0 = 0; k0 < ROWS; k0 += 1024) {
    const int k = k0 + (int)threadIdx.x;
    int total = 0;
    if (k < ROWS)
      for (int w = 0; w < WAVES; ++w) total += counts[w][k];
    const int upto = rx_wave_scan(total, rx_op_add());
    if (lane == 63) sums[wave] = upto;
    __syncthreads();
    int at = carry + upto - total;
    for (int w = 0; w < WAVES; ++w) {
      if (w < wave) at += sums[w];
      carry += sums[w];
    }
    if (k < ROWS) {
      if (r0 + k < V) start[r0 + k] = at;
      for (int w = 0; w < WAVES; ++w) {
        const int n = counts[w][k];
        counts[w][k] = at;
        at += n;
      }
    }
    __syncthreads();
  }
  if (threadIdx.x == 0 && r0 + ROWS >= V) start[V] = carry;
  auto place = [&](const int id, const int t) {                 // (whole wavefronts: the lanes compare their rows)
    const bool mine = id >= r0 && id < (long long)r0 + ROWS;
    const int row = mine ? id - r0 : -1;
    unsigned long long left = __ballot(mine);
    while (left) {
      const int leader = __builtin_ctzll(left), its = __builtin_amdgcn_readlane(row, leader);
      const unsigned long long same = __ballot(row == its);
      int at = 0;
      if (lane == leader) at = atomicAdd(&counts[wave][its], __popcll(same));
      at = __builtin_amdgcn_readlane(at, leader) + __popcll(same & ((1ull << lane) - 1));
      if (row == its) {
        order[at] = t;
        row_of[at] = id;
      }
      left &= ~same;
    }
  };
  if constexpr (KEPT == EACH) {
#pragma unroll
    for (int k = 0; k < KEPT; ++k) place(kept[k], t0 + lane + 64 * k);
  } else {
    for (int t = t0 + lane; t < t0 + STRETCH; t += 64) {
      const I id = t < t1 ? ids[t] : (I)-1;
      place(id >= 0 && id < V ? (int)id : -1, t);
    }
  }
}

template <long long N, typename S>
RX_DEV void rx_lm_zero(S* out) {
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < N; i += (long long)gridDim.x * 256) out[i] = (S)0;
}
template <int N>
struct rx_lm_acc { float v[N]; };
// adds the listed tokens' rows, in their order: the vectors c, c + 256, .. (EACH of them, those past the row's end are its last)
template <typename E, int D, int VEC, int EACH, int AHEAD>
RX_DEV int rx_lm_add_rows(const typename E::S* dy, const int* order, int from, const int to, const int c, rx_lm_acc<VEC> (&a)[EACH]) {
  typedef rx_vec<typename E::S, VEC> W;
  for (; AHEAD == 4 ? from < to : from + AHEAD <= to; from += AHEAD) {
    W w[AHEAD][EACH];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const typename E::S* row = dy + (long long)order[AHEAD > 4 || from + k < to ? from + k : to - 1] * D;
#pragma unroll
      for (int n = 0; n < EACH; ++n) w[k][n] = rx_load<W>(row + (c + 256 * n < D / VEC ? c + 256 * n : D / VEC - 1) * VEC);
    }
#pragma unroll
    for (int k = 0; k < AHEAD; ++k)
#pragma unroll
      for (int n = 0; n < EACH; ++n)
#pragma unroll
        for (int e = 0; e < VEC; ++e) a[n].v[e] += AHEAD > 4 || k == 0 || from + k < to ? E::up(w[k][n].v[e]) : 0.0f;
  }
  return from;
}
// eight tokens at a time, the last ones four at a time: loads one after the other would wait for one another
template <typename E, int D, int VEC, int EACH>
RX_DEV void rx_lm_sum_rows(const typename E::S* dy, const int* order, int from, const int to, const int c, rx_lm_acc<VEC> (&a)[EACH]) {
  from = rx_lm_add_rows<E, D, VEC, EACH, 8>(dy, order, from, to, c, a);
  rx_lm_add_rows<E, D, VEC, EACH, 4>(dy, order, from, to, c, a);
}
template <typename O, int VEC>
RX_DEV void rx_lm_put(typename O::S* out, const rx_lm_acc<VEC>& a, const float scale) {
  rx_vec<typename O::S, VEC> w;
#pragma unroll
  for (int e = 0; e < VEC; ++e) w.v[e] = O::down(a.v[e] * scale);
  rx_store_nt(out, w);
}

// Rows of up to LONG tokens: EACH vectors of a row to a thread (C vectors a row; several short rows to a workgroup), its tokens
// summed in their order.  A row of more would keep one thread's loads waiting for one another: those are summed in pieces, the
// places [LONG p, LONG p + LONG) of the list by the first workgroups (a piece touches at most two such rows: it may end one
// and start another), and the workgroup that arrives last adds a row's pieces in their order.
// Bound by memory: 65536 x 4096 in f32 from 16384 tokens in bf16, 1.2 GB of which 1.07 are written, take 221 us, 5.5 TB/s (a fill
// reaches 6.8, a copy 6.2).  The loads of four rows ahead of all sums: 242 us.
template <typename E, typename O, int V, int D, int T, int VEC, int LONG, int EACH>
RX_DEV void rx_embedding_grad_rows(const typename E::S* dy, const int* start, const int* order, const int* row_of, typename O::S* out, float* part, int* arrived, const float scale) {
  constexpr int C = D / VEC, TILES = (C + 256 * EACH - 1) / (256 * EACH), NP = (T + LONG - 1) / LONG;
  constexpr int LANES = C < 256 ? C : 256, ROWS = 256 / LANES;   // threads along a row, rows of a workgroup
  if (blockIdx.x < NP * TILES) {
    __shared__ int flag;
    const int piece = blockIdx.x / TILES, tile = blockIdx.x % TILES, c = tile * (256 * EACH) + (int)threadIdx.x, all = start[V];
    const int a = piece * LONG, e = a + LONG < all ? a + LONG : all;
    if (a >= e) return;
    const int first = row_of[a], last = row_of[e - 1];
    for (int k = 0; k < 2; ++k) {
      const int row = k ? last : first;
      if (k && last == first) break;
      const int s0 = start[row], s1 = start[row + 1];
      if (s1 - s0 <= LONG) continue;
      rx_lm_acc<VEC> sum[EACH] = {};
      if (c < C) {
        rx_lm_sum_rows<E, D, VEC, EACH>(dy, order, s0 > a ? s0 : a, s1 < e ? s1 : e, c, sum);
#pragma unroll
        for (int n = 0; n < EACH; ++n)
#pragma unroll
          for (int q = 0; q < VEC; ++q)
            if (c + 256 * n < C) rx_lm_put_shared(part + ((long long)(piece * 2 + k) * VEC + q) * C + c + 256 * n, sum[n].v[q]);
      }
      const int from = s0 / LONG, to = (s1 - 1) / LONG, starts = row_of[from * LONG] != row;   // its first piece's second row?
      if (!rx_lm_last_to_arrive(arrived + from * TILES + tile, to - from + 1, &flag) || c >= C) continue;
#pragma unroll
      for (int n = 0; n < EACH; ++n) {
        if (c + 256 * n >= C) break;
        rx_lm_acc<VEC> total = {};
#pragma unroll 4
        for (int p = from; p <= to; ++p)
#pragma unroll
          for (int q = 0; q < VEC; ++q) total.v[q] += rx_lm_get_shared(part + ((long long)(p * 2 + (p == from && starts)) * VEC + q) * C + c + 256 * n);
        rx_lm_put<O, VEC>(out + ((long long)row * C + c + 256 * n) * VEC, total, scale);
      }
    }
    return;
  }
  const int l = (int)threadIdx.x % LANES, r = (int)threadIdx.x / LANES;
  if (r >= ROWS) return;
  const long long work = (long long)((V + ROWS - 1) / ROWS) * TILES;
  for (long long i = blockIdx.x - NP * TILES; i < work; i += gridDim.x - NP * TILES) {
    const int row = (int)(i / TILES) * ROWS + r, c = (int)(i % TILES) * (256 * EACH) + l;
    if (row >= V || c >= C) continue;
    const int s0 = start[row], s1 = start[row + 1];
    if (s1 - s0 > LONG) continue;
    rx_lm_acc<VEC> sum[EACH] = {};
    rx_lm_sum_rows<E, D, VEC, EACH>(dy, order, s0, s1, c, sum);
#pragma unroll
    for (int n = 0; n < EACH; ++n)
      if (c + 256 * n < C) rx_lm_put<O, VEC>(out + ((long long)row * C + c + 256 * n) * VEC, sum[n], scale);
  }
}

// Few tokens (up to 768): one launch, without a sorted list in memory.  A workgroup takes the rows of about 1024 vectors, lists
// the tokens of these rows as it goes through all of them (a wavefront's matches in the order of its lanes, the wavefronts' one
// after the other), ranks the listed tokens by row, and every thread sums those of its vectors' rows.  513 tokens, 10007 x 1024 in
// f32, 43 MB: 9.2 us, where writing alone takes 6.3 and two launches with a sorted list 12.8.
template <typename E, typename O, int V, int D, int T, int VEC, typename I>
RX_DEV void rx_embedding_grad_few(const typename E::S* dy, const I* ids, typename O::S* out, const float scale) {
  constexpr int C = D / VEC, ROWS = C < 1024 ? 1024 / C : 1, LOADS = (T + 255) / 256;
  static_assert(LOADS <= 3, "tokens of a thread");
  __shared__ int found[T], of[T], sorted[T], start[ROWS + 1], sums[LOADS][4];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  int id[LOADS];
#pragma unroll
  for (int k = 0; k < LOADS; ++k) {
    const int t = k * 256 + (int)threadIdx.x;
    const I i = ids[t < T ? t : T - 1];
    id[k] = t < T && i >= 0 && i < V ? (int)i : -1;
  }
  for (long long r0 = (long long)blockIdx.x * ROWS; r0 < V; r0 += (long long)gridDim.x * ROWS) {
    unsigned long long hits[LOADS];
#pragma unroll
    for (int k = 0; k < LOADS; ++k) {
      hits[k] = __ballot(id[k] >= r0 && id[k] < r0 + ROWS);
      if (lane == 0) sums[k][wave] = __popcll(hits[k]);
    }
    __syncthreads();
    int n = 0;
#pragma unroll
    for (int k = 0; k < LOADS; ++k) {
      int at = n;
      for (int w = 0; w < 4; ++w) {
        if (w < wave) at += sums[k][w];
        n += sums[k][w];
      }
      if (id[k] >= r0 && id[k] < r0 + ROWS) {
        at += __popcll(hits[k] & ((1ull << lane) - 1));
        found[at] = k * 256 + (int)threadIdx.x;
        of[at] = id[k] - (int)r0;
      }
    }
    __syncthreads();
    for (int k = threadIdx.x; k < n; k += 256) {
      const int row = of[k];
      int rank = 0;
      for (int i = 0; i < n; ++i) rank += of[i] < row || (of[i] == row && i < k);
      sorted[rank] = found[k];
    }
    for (int k = threadIdx.x; k <= ROWS; k += 256) {
      int before = 0;
      for (int i = 0; i < n; ++i) before += of[i] < k;
      start[k] = before;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < ROWS * C; i += 256) {
      const int row = i / C, c = i % C;
      if (r0 + row >= V) break;
      rx_lm_acc<VEC> sum[1] = {};
      rx_lm_sum_rows<E, D, VEC, 1>(dy, sorted, start[row], start[row + 1], c, sum);
      rx_lm_put<O, VEC>(out + ((r0 + row) * C + c) * VEC, sum[0], scale);
    }
    __syncthreads();
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

// One element of a head after rotation: x cos - y sin for the first of a pair, y cos + x sin for the second.  The products are
// rounded, then their sum: `x * c - y * s` in f32.
template <typename E, int R2, bool PAIRS>
RX_DEV float rx_lm_rotated(const typename E::S* head, int d, const float* cos, const float* sin) {
  const float x = E::up(head[d]);
  if (d >= 2 * R2) return x;
  const int a = PAIRS ? d >> 1 : (d < R2 ? d : d - R2);
  const bool second = PAIRS ? (d & 1) : d >= R2;
  const float y = E::up(head[second ? (PAIRS ? d - 1 : d - R2) : (PAIRS ? d + 1 : d + R2)]);
  return second ? x * cos[a] + y * sin[a] : x * cos[a] - y * sin[a];
}

// where a token goes: its position, and the slot's page and number (page -1: nowhere)
struct rx_lm_place { long long pos; int page, slot; bool known; };
template <int P, int S, int B, int M, int L, int R2, typename I>
RX_DEV rx_lm_place rx_lm_place_of(const I* position, const I* sequence, const I* pages, const long long t) {
  const I pos = position[t], seq = sequence[t];
  rx_lm_place p = {0, -1, 0, pos >= 0 && pos < (R2 && L < (long long)M * S ? (long long)L : (long long)M * S) && seq >= 0 && seq < B};
  if (!p.known) return p;
  p.pos = pos;
  const I page = pages[(long long)seq * M + (int)pos / S];
  p.page = page >= 0 && page < P ? (int)page : -1;
  p.slot = (int)pos % S;
  return p;
}

// heads of any width: a workgroup per token
template <typename E, int HQ, int HK, int DK, int DV, int P, int S, int B, int M, int L, int R2, bool PAIRS, bool BY_SLOT, int T, typename I>
RX_DEV void rx_kv_append_any(const typename E::S* q, const typename E::S* k, const typename E::S* v, const float* cos, const float* sin, const I* position, const I* sequence,
                             const I* pages, typename E::S* qo, typename E::S* kc, typename E::S* vc) {
  for (long long t = blockIdx.x; t < T; t += gridDim.x) {
    const rx_lm_place p = rx_lm_place_of<P, S, B, M, L, R2>(position, sequence, pages, t);
    const float* c = cos + p.pos * R2;
    const float* s = sin + p.pos * R2;
    for (int i = threadIdx.x; i < HQ * DK; i += 256)
      qo[t * (HQ * DK) + i] = p.known ? E::down(rx_lm_rotated<E, R2, PAIRS>(q + t * (HQ * DK) + i / DK * DK, i % DK, c, s)) : E::down(0.0f);
    if (p.page < 0) continue;
    for (int i = threadIdx.x; i < HK * DK; i += 256)
      kc[rx_lm_slot<S, HK, DK, BY_SLOT>(p.page, p.slot, i / DK) + i % DK] = E::down(rx_lm_rotated<E, R2, PAIRS>(k + t * (HK * DK) + i / DK * DK, i % DK, c, s));
    for (int i = threadIdx.x; i < HK * DV; i += 256) vc[rx_lm_slot<S, HK, DV, BY_SLOT>(p.page, p.slot, i / DV) + i % DV] = v[t * (HK * DV) + i];
  }
}

// Heads of whole vectors: a thread takes the same dimensions of HEADS heads of a token (their cosines and sines are loaded
// once): the two vectors of a rotated stretch of pairs, or one vector that is not rotated, or whose pairs are inside of it.
// 8191 tokens of 32 and 8 heads of 128 in f16, half of the dimensions rotated, take 38 us, 5.4 TB/s of reading and writing, of which
// a copy of this size reaches 6.2; 48 tokens take 2.8 us, what a launch and four dependent loads last.
template <typename E, int HQ, int HK, int DK, int DV, int P, int S, int B, int M, int L, int R2, bool PAIRS, bool BY_SLOT, int T, int HEADS, typename I>
RX_DEV void rx_kv_append(const typename E::S* q, const typename E::S* k, const typename E::S* v, const float* cos, const float* sin, const I* position, const I* sequence,
                         const I* pages, typename E::S* qo, typename E::S* kc, typename E::S* vc) {
  typedef typename E::S X;
  constexpr int NE = 16 / sizeof(X);
  typedef rx_vec<X, NE> W;
  constexpr int TURNED = PAIRS ? 2 * R2 / NE : R2 / NE, UNITS = TURNED + (DK - 2 * R2) / NE;   // of a head: rotated ones first
  constexpr int GQ = (HQ + HEADS - 1) / HEADS, GK = (HK + HEADS - 1) / HEADS, VV = (HK * DV / NE + HEADS - 1) / HEADS;
  constexpr int ALL = (GQ + GK) * UNITS + VV;                                                     // threads of a token
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < (long long)T * ALL; i += (long long)gridDim.x * 256) {
    const long long t = i / ALL;
    const int u = (int)(i % ALL);
    const rx_lm_place p = rx_lm_place_of<P, S, B, M, L, R2>(position, sequence, pages, t);
    if (u >= (GQ + GK) * UNITS) {                                                                 // values
#pragma unroll
      for (int h = 0; h < HEADS; ++h) {
        const int w = (u - (GQ + GK) * UNITS) + h * VV, head = w / (DV / NE), d = w % (DV / NE) * NE;
        if (w >= HK * DV / NE) break;
        const W x = rx_load<W>(v + t * (HK * DV) + head * DV + d);
        if (p.page >= 0) rx_store_nt(vc + rx_lm_slot<S, HK, DV, BY_SLOT>(p.page, p.slot, head) + d, x);
      }
      continue;
    }
    const int group = u / UNITS, n = u % UNITS;
    const bool query = group < GQ;
    const bool turned = n < TURNED;
    const int d = turned ? n * NE : 2 * R2 + (n - TURNED) * NE;                                   // first dimension
    float c[NE] = {}, s[NE] = {};
    if (R2 && L && turned) {
      const long long at = p.pos * R2 + (PAIRS ? d / 2 : d);
#pragma unroll
      for (int e = 0; e < (PAIRS ? NE / 2 : NE); ++e) {
        c[e] = cos[at + e];
        s[e] = sin[at + e];
      }
    }
#pragma unroll
    for (int h = 0; h < HEADS; ++h) {
      const int head = (query ? group : group - GQ) * HEADS + h;
      if (head >= (query ? HQ : HK)) break;
      const X* x = query ? q + (t * HQ + head) * DK + d : k + (t * HK + head) * DK + d;
      X* y = query ? qo + (t * HQ + head) * DK + d : kc + rx_lm_slot<S, HK, DK, BY_SLOT>(p.page < 0 ? 0 : p.page, p.slot, head) + d;
      W a = rx_load<W>(x), b{};
      if (R2 && turned) {
        if constexpr (PAIRS) {
#pragma unroll
          for (int e = 0; e < NE; e += 2) {
            const float f = E::up(a.v[e]), g = E::up(a.v[e + 1]);
            a.v[e] = E::down(f * c[e / 2] - g * s[e / 2]);
            a.v[e + 1] = E::down(g * c[e / 2] + f * s[e / 2]);
          }
        } else {
          b = rx_load<W>(x + R2);
#pragma unroll
          for (int e = 0; e < NE; ++e) {
            const float f = E::up(a.v[e]), g = E::up(b.v[e]);
            a.v[e] = E::down(f * c[e] - g * s[e]);
            b.v[e] = E::down(g * c[e] + f * s[e]);
          }
        }
      }
      if (query && !p.known) a = b = W{};
      if (query || p.page >= 0) {
        rx_store_nt(y, a);
        if (!PAIRS && R2 && turned) rx_store_nt(y + R2, b);
      }
    }
  }
}

// ---- attention of one token per sequence ----
// One pass over keys and values with the running maximum and sum of the softmax, on the matrix cores without LDS: a wavefront
// takes 32 positions at a time.  Scores are K Q' (MFMA rows are positions, columns the query heads of one key head), the result
// is V' P' (rows are dimensions, columns heads): column h of both lies in the lanes l with l mod 16 = h, so the maximum, the
// sum and the weights of a head stay in its lanes, and the weights leave the first product in the registers in which the
// second one takes them (which of its k is which position is free as long as V follows suit).  V' needs the values of one
// dimension at consecutive positions: a lane loads 16 bytes (8 dimensions) of 8 positions, and bytes are permuted in registers.
//
// The positions of all sequences, in units of 32, are one row that R workgroups per key head (and tile of query heads) share in
// equal stretches, whatever the lengths: a stretch may end one sequence, hold others, and start one more.  Every workgroup
// works its stretch out from the lengths.  Sequences inside of one stretch are finished there.  Of a longer one every workgroup
// leaves (maximum, sum, unscaled result) of its part, and the one that arrives last combines them, in the order of the
// positions.  A workgroup has at most two such parts: one that a workgroup before it has started, and one that it starts.
//
// Bound by reading the caches where they are long: 8 sequences of 131072 positions, 8 key heads of 128 in bf16, 64 query heads, 4.3
// GB, take 627 us, 6.8 TB/s, what reading alone reaches (the first form, a workgroup per query head and dot products on the vector
// units: 192 ms); 64 sequences of 1 to 8192 positions, 257 MB, 52 us, 4.9 TB/s: what is missing is the start and the end of the launch.
// A chain of dependent steps where they are short: lengths, pages, keys and values, two products, the parts, the count, the parts
// again: 8.5 us for one sequence of 1000 positions.  Loads one step ahead of the products gained nothing (two wavefronts to a SIMD
// cover one another) and spilled registers in f32.
struct rx_lm_span { int n, lo, units, cost; };   // length, first position, units from lo rounded down to 32 (an empty sequence has one); what it counts in the row
template <int S, int B, int M, int W, typename I>
RX_DEV rx_lm_span rx_lm_span_of(const I len) {
  rx_lm_span s;
  s.n = len < 0 ? 0 : len > (I)(M * S) ? M * S : (int)len;
  s.lo = W && s.n > W ? s.n - W : 0;
  s.units = (s.n - (s.lo & ~31) + 31) >> 5;
  if (s.units == 0) s.units = 1;
  s.cost = s.units + (B > 1 ? 4 : 0);   // going over to another sequence takes as long as about four units (64 of 1 to 8192 positions: 0: 67 us, 2: 60, 4: 59, 8: 60, 12: 62)
  return s;
}
struct rx_lm_stretch { int b, unit, count; long long first, total; int parts; };   // sequence and its unit to start at, units; first unit in the row, units of the row, stretches
// Stretch r of up to R: at least four units each, one for every wavefront, and fewer for long sequences: the workgroup that joins n
// parts takes as long over each as n workgroups gain by it, so the longest sequence of u units is to have about sqrt(Q u).  (One of
// 65536 positions, 8 query heads of one key head of 128: 512 parts 79 us, 91 parts 31, 64 parts 32; of 4000: 31 parts 11.8.)
RX_DEV long long rx_lm_stretch_start(const long long total, const int parts, const int r) { return total * r / parts; }
// `cost(b)`: what sequence b counts in the row
template <int B, int R, int Q, typename F>
RX_DEV rx_lm_stretch rx_lm_stretch_of(F cost, const int r) {
  const int lane = threadIdx.x & 63;
  rx_lm_stretch s = {B, 0, 0, 0, 0, 0};
  int units = 0, longest = 0;
  for (int b0 = 0; b0 < B; b0 += 64) {
    units = b0 + lane < B ? cost(b0 + lane) : 0;
    s.total += units;
    longest = units > longest ? units : longest;
  }
  if constexpr (B > 1) s.total = rx_wave_reduce(s.total, rx_op_add());
  else s.total = rx_lane_from(s.total, 0);
  s.parts = s.total < 4ll * R ? (int)((s.total + 3) / 4) : R;
  if constexpr (R > 1) {
    longest = B > 1 ? rx_wave_reduce(longest, rx_op_max()) : rx_lane_from(longest, 0);
    const float most = (float)s.total * __builtin_amdgcn_sqrtf((float)Q / (float)longest) + 1.0f;
    s.parts = most < (float)s.parts ? (int)most : s.parts;
  }
  if (r >= s.parts) return s;
  s.first = rx_lm_stretch_start(s.total, s.parts, r);
  s.count = (int)(rx_lm_stretch_start(s.total, s.parts, r + 1) - s.first);
  long long sum = 0;
  for (int b0 = 0; b0 < B; b0 += 64) {
    if (B > 64) units = b0 + lane < B ? cost(b0 + lane) : 0;
    const long long upto = sum + (B > 1 ? rx_wave_scan((long long)units, rx_op_add()) : (long long)units);
    const unsigned long long past = __ballot(b0 + lane < B && upto > s.first);
    if (past) {
      const int at = __builtin_ctzll(past);
      s.b = b0 + at;
      s.unit = (int)(s.first - rx_lane_from(upto - units, at));
      return s;
    }
    sum = rx_lane_from(upto, 63);
  }
  return s;
}
// the stretch that holds a unit of the row
RX_DEV int rx_lm_stretch_with(const long long total, const int parts, const long long unit) {
  int r = (int)(unit * parts / total);
  while (r + 1 < parts && rx_lm_stretch_start(total, parts, r + 1) <= unit) ++r;
  while (r > 0 && rx_lm_stretch_start(total, parts, r) > unit) --r;
  return r;
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
template <typename E, int D, bool ONCE = false>
RX_DEV rx_u32x4 rx_lm_row16(const typename E::S* row, const int d) {
  constexpr int NE = 16 / sizeof(typename E::S);
  rx_u32x4 v = {0, 0, 0, 0};
  if constexpr (D % NE == 0) {
    if (d < D) v = ONCE ? __builtin_nontemporal_load((const rx_u32x4*)(row + d)) : *(const rx_u32x4*)(row + d);
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

// (maximum, sum, unscaled result) of parts of a sequence; the maximum goes up before parts are added
template <int N>
struct rx_lm_joined {
  float m, s, o[N];
  RX_MEM float weight(const float x, const float hi) const { return x == -rx_lm_inf() ? 0.0f : __builtin_amdgcn_exp2f(x - hi); }
  RX_MEM void to(const float hi) {
    const float f = weight(m, hi);
    s *= f;
#pragma unroll
    for (int e = 0; e < N; ++e) o[e] *= f;
    m = hi;
  }
  RX_MEM void add(const float x, const float sum, const float (&v)[N]) {
    const float f = weight(x, m);
    s += sum * f;
#pragma unroll
    for (int e = 0; e < N; ++e) o[e] += v[e] * f;
  }
};

// HW: key heads of a workgroup, whose four wavefronts share the units of a head, or have a head each; COLUMNS: groups of HW key
// heads, times the tiles of up to 16 NT query heads that read one; R: stretches; ONCE: the caches are read past the L2; DIES: a
// stretch's columns are neighbours on one die; VECTOR: f32 caches with one query head a key head, by the vector units, since 15
// of the matrix cores' 16 columns would be empty at a sixteenth of their 16-bit rate.  A lane multiplies its parts of two keys, and
// the values of its eight positions, in the same registers; every column holds the one head.
template <typename E, int HQ, int HK, int DK, int DV, int P, int S, int B, int M, int W, bool BY_SLOT, int NT, int R, int HW, bool ONCE, bool DIES, bool VECTOR, int Q, typename I>
RX_DEV void rx_paged_attention(const typename E::S* q, const typename E::S* kc, const typename E::S* vc, const I* pages, const I* lengths, typename E::S* out, float* lse,
                               float* part, float* stat, int* arrived, const float scale) {
  typedef typename E::S T;
  constexpr int NE = 16 / sizeof(T);                   // elements of 16 bytes
  constexpr int G = HQ / HK, GT = G < 16 * NT ? G : 16 * NT, TILES = (G + GT - 1) / GT, COLUMNS = HK / HW * TILES, WPH = 4 / HW;
  constexpr int NK = (DK + 4 * NE - 1) / (4 * NE);     // 16-byte loads of a position's key by its four lanes
  constexpr int NV = (DV + 16 * NE - 1) / (16 * NE);   // of a position's value by sixteen lanes
  constexpr int BLOCK = 2048;                          // positions whose pages are held in LDS
  constexpr float SHIFT = sizeof(T) == 2 && !E::BF16 ? 15.0f : 0.0f;   // f16 weights are taken times 2^15: the smallest would be lost below 2^-24
  constexpr int HR = GT < 16 ? GT : 16, WIDTH = 16 * NE < DV ? 16 * NE : DV;   // heads and dimensions that are joined at a time
  __shared__ union {
    int page[BLOCK / S + 2];
    float o[4][HR][WIDTH + 4];
    rx_lm_joined<DV % 4 == 0 ? 4 : 1> j[256];
  } lds;
  __shared__ float join_m[4][16], join_l[4][16];
  __shared__ int last;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, r = lane & 15, g4 = lane >> 4;
  const int id = DIES ? (int)rx_xcd_remap(blockIdx.x, R * COLUMNS) : (int)blockIdx.x, column = id % COLUMNS, mine = id / COLUMNS, tile = column % TILES;
  const int head0 = column / TILES * HW, head = head0 + wave / WPH;
  const int h0 = head * G + tile * GT;                 // first query head of this wavefront
  const int heads = G - tile * GT < GT ? G - tile * GT : GT;
  const rx_lm_stretch st = rx_lm_stretch_of<B, R, Q>([&](const int at) { return rx_lm_span_of<S, B, M, W>(lengths[at]).cost; }, mine);

  int b = st.b, unit = st.unit;
  for (int left = st.count; left > 0; ++b, unit = 0) {
  const rx_lm_span span = rx_lm_span_of<S, B, M, W>(lengths[b]);
  const int step = span.cost - unit < left ? span.cost - unit : left, take = span.units - unit < step ? span.units - unit : step;
  const long long begin = st.first + (st.count - left) - unit;   // the sequence's first unit in the row
  left -= step;
  if (take <= 0) continue;
  const int p0 = (span.lo & ~31) + unit * 32, p1 = P == 0 ? p0 : p0 + take * 32 < span.n ? p0 + take * 32 : span.n;
  const bool whole = take == span.units;               // the whole sequence is in this stretch
  rx_u32x4 qf[NT][NK];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int k = 0; k < NK; ++k)
      qf[t][k] = VECTOR || t * 16 + r < heads ? rx_lm_row16<E, DK>(q + ((long long)b * HQ + h0 + (VECTOR ? 0 : t * 16 + r)) * DK, (k * 4 + g4) * NE) : rx_u32x4{0, 0, 0, 0};

  float m[NT], l[NT];
  rx_f32x4 acc[NT][NV][NE];                            // (VECTOR: only the first of four)
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
    auto where = [&](const int t) { return t >= span.lo && t < s1 ? lds.page[t / S - page0] : -1; };
    for (int t0 = s0 + wave % WPH * 32; t0 < s1; t0 += WPH * 32) {
      const int ta = t0 + r, tb = ta + 16, pa = where(ta), pb = where(tb);
      const unsigned ok = ((unsigned)__ballot(pa >= 0) & 0xffffu) | ((unsigned)__ballot(pb >= 0) << 16);
      if (!ok) continue;
      rx_u32x4 kf[2][NK], vf[NV][8];
      const T* ka = kc + rx_lm_slot<S, HK, DK, BY_SLOT>(pa < 0 ? 0 : pa, ta % S, head);
      const T* kb = kc + rx_lm_slot<S, HK, DK, BY_SLOT>(pb < 0 ? 0 : pb, tb % S, head);
#pragma unroll
      for (int k = 0; k < NK; ++k) {
        kf[0][k] = rx_lm_row16<E, DK, ONCE>(ka, (k * 4 + g4) * NE);
        kf[1][k] = rx_lm_row16<E, DK, ONCE>(kb, (k * 4 + g4) * NE);
      }
      // values of positions t0 + 4 g4 + (0..3) and 16 further: where a page's slots are a multiple of four, on two pages
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
        for (int j = 0; j < NV; ++j) vf[j][i] = rx_lm_row16<E, DV, ONCE>(v, (j * 16 + r) * NE);
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
      // The weights, in f32 for the sum.  For the product the matrix cores take them in the cache's type: as two numbers, the
      // second what the first one's rounding leaves, since the first alone is off by as much as the result's own rounding.
      rx_vec<T, 8> w[NT], rest[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        rx_f32x4 s[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
        for (int k = 0; k < NK; ++k) {
          if constexpr (VECTOR) {
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
              for (int e = 0; e < 4; ++e) s[c][e] = __builtin_fmaf(__builtin_bit_cast(rx_f32x4, kf[c][k])[e], __builtin_bit_cast(rx_f32x4, qf[t][k])[e], s[c][e]);
          } else {
            s[0] = rx_lm_mma<E>(kf[0][k], qf[t][k], s[0]);
            s[1] = rx_lm_mma<E>(kf[1][k], qf[t][k], s[1]);
          }
        }
        if constexpr (VECTOR) {
          // position r's and 16 + r's scores, and from them those of the positions whose values this lane holds
          const float a = rx_lm_sum4((s[0][0] + s[0][1]) + (s[0][2] + s[0][3])), b = rx_lm_sum4((s[1][0] + s[1][1]) + (s[1][2] + s[1][3]));
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            s[0][i] = rx_lane_from(a, g4 * 4 + i);
            s[1][i] = rx_lane_from(b, g4 * 4 + i);
          }
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
        // (not below the lowest number: a maximum of -inf says that there was no position, and scores that are all -inf or NaN
        // leave a sum of nothing, or NaN, beside it: the result is NaN, not the zeros of an empty sequence)
        top = __builtin_fmaxf(__builtin_fmaxf(m[t], rx_lm_max4(top)), -RX_LM_FLT_MAX);
        if (__any(top != m[t])) {
          const float shrink = __builtin_amdgcn_exp2f(m[t] - top);
          l[t] *= shrink;
#pragma unroll
          for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int e = 0; e < NE; ++e) {
              if constexpr (VECTOR) acc[t][j][e][0] *= shrink;
              else acc[t][j][e] *= shrink;
            }
          m[t] = top;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float p = __builtin_amdgcn_exp2f(x[i] - top + SHIFT);
          l[t] += p;
          w[t].v[i] = E::down(p);
          rest[t].v[i] = E::down(p - E::up(w[t].v[i]));
        }
      }
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < NE; ++e) {
          if constexpr (NE == 8) {
            rx_u32x4 a;                                          // dimension 8 r + e of the eight positions
#pragma unroll
            for (int k = 0; k < 4; ++k) a[k] = __builtin_amdgcn_perm(vf[j][2 * k + 1][e >> 1], vf[j][2 * k][e >> 1], e & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
              acc[t][j][e] = rx_lm_mma<E>(a, __builtin_bit_cast(rx_u32x4, w[t]), acc[t][j][e]);
              acc[t][j][e] = rx_lm_mma<E>(a, __builtin_bit_cast(rx_u32x4, rest[t]), acc[t][j][e]);
            }
          } else {
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
              for (int i = 0; i < 8; ++i)
                if constexpr (VECTOR) acc[t][j][e][0] = __builtin_fmaf(__builtin_bit_cast(rx_f32x4, vf[j][i])[e], w[t].v[i], acc[t][j][e][0]);
                else acc[t][j][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(rx_f32x4, vf[j][i])[e], w[t].v[i], acc[t][j][e], 0, 0, 0);
          }
        }
    }
  }

  // the four wavefronts' parts
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
    for (int w = 0; w < WPH; ++w) top = __builtin_fmaxf(top, join_m[wave / WPH * WPH + w][r]);
    const float f = top == -rx_lm_inf() ? 0.0f : __builtin_amdgcn_exp2f(m[t] - top);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (j) __syncthreads();
      if constexpr (VECTOR) {
#pragma unroll
        for (int e = 0; e < NE; ++e) {
          const float sum = rx_lm_sum4(acc[t][j][e][0]) * f;
          if (g4 == 0 && r * NE + e < WIDTH) lds.o[wave][0][r * NE + e] = sum;
        }
      } else if (r < HR) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int e = 0; e < NE; ++e) {
            const int d = (g4 * 4 + i) * NE + e;
            if (d < WIDTH) lds.o[wave][r][d] = acc[t][j][e][i] * f;
          }
      }
      __syncthreads();
      for (int k = threadIdx.x; k < HW * HR * WIDTH; k += 256) {
        const int hw = k / (HR * WIDTH), h = k / WIDTH % HR, d = j * 16 * NE + k % WIDTH;
        if (t * 16 + h >= heads || d >= DV) continue;
        float o = 0.0f, sum = 0.0f, hi = -rx_lm_inf();
#pragma unroll
        for (int i = 0; i < WPH; ++i) hi = __builtin_fmaxf(hi, join_m[hw * WPH + i][h]);
#pragma unroll
        for (int i = 0; i < WPH; ++i) {
          const int w = hw * WPH + i;
          o += lds.o[w][h][k % WIDTH];
          sum += hi == -rx_lm_inf() ? 0.0f : join_l[w][h] * __builtin_amdgcn_exp2f(join_m[w][h] - hi);
        }
        const int qh = (head0 + hw) * G + tile * GT + t * 16 + h;
        if (whole) {
          out[((long long)b * HQ + qh) * DV + d] = E::down(hi == -rx_lm_inf() ? 0.0f : o / sum);
          if (lse && d == 0) lse[(long long)b * HQ + qh] = hi == -rx_lm_inf() ? -rx_lm_inf() : (hi - SHIFT + __builtin_log2f(sum)) * 0.6931471805599453f;
        } else {
          const long long at = (((long long)id * 2 + (unit == 0)) * HW + hw) * GT + t * 16 + h;
          rx_lm_put_shared(part + at * DV + d, o);
          if (d == 0) {
            rx_lm_put_shared(stat + at * 2, hi - SHIFT);
            rx_lm_put_shared(stat + at * 2 + 1, sum);
          }
        }
      }
    }
  }
  if (whole) continue;
  const int from = rx_lm_stretch_with(st.total, st.parts, begin), to = rx_lm_stretch_with(st.total, st.parts, begin + span.units - 1);
  if (!rx_lm_last_to_arrive(arrived + b * COLUMNS + column, to - from + 1, &last)) continue;
  // VD outputs to a thread, DV / VD apart, so that lanes read consecutive words (16000 positions of 4 key heads of 64, 125 parts: 28 us
  // with consecutive outputs to a thread, 22 so); where there are fewer than threads, the parts are shared too, and joined once more
  constexpr int VD = DV % 4 == 0 ? 4 : 1;
  const int outs = HW * heads * (DV / VD), ways = outs < 256 ? 256 / outs : 1, parts = to - from + 1;
  for (int k0 = 0; k0 < outs; k0 += 256) {
    const int k = ways > 1 ? (int)threadIdx.x % outs : k0 + (int)threadIdx.x, way = ways > 1 ? (int)threadIdx.x / outs : 0;
    const bool on = k < outs && way < ways;
    const int hw = k / (heads * (DV / VD)), h = k / (DV / VD) % heads, d = k % (DV / VD), qh = (head0 + hw) * G + tile * GT + h;
    const int w1 = on ? from + parts * (way + 1) / ways : 0;
    rx_lm_joined<VD> j = {-rx_lm_inf(), 0.0f, {}};
    for (int w = on ? from + parts * way / ways : 0; w < w1; w += 8) {
      float pm[8], ps[8], po[8][VD];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int v = w + i < w1 ? w + i : w1 - 1;
        const long long at = (((long long)(v * COLUMNS + column) * 2 + (v == from)) * HW + hw) * GT + h;
        pm[i] = rx_lm_get_shared(stat + at * 2);
        ps[i] = rx_lm_get_shared(stat + at * 2 + 1);
#pragma unroll
        for (int e = 0; e < VD; ++e) po[i][e] = rx_lm_get_shared(part + at * DV + d + e * (DV / VD));
      }
      float hi = j.m;
#pragma unroll
      for (int i = 0; i < 8; ++i) hi = __builtin_fmaxf(hi, pm[i]);
      j.to(hi);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (w + i < w1) j.add(pm[i], ps[i], po[i]);
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
#pragma unroll
    for (int e = 0; e < VD; ++e) out[((long long)b * HQ + qh) * DV + d + e * (DV / VD)] = E::down(j.m == -rx_lm_inf() ? 0.0f : j.o[e] / j.s);
    if (lse && d == 0) lse[(long long)b * HQ + qh] = j.m == -rx_lm_inf() ? -rx_lm_inf() : (j.m + __builtin_log2f(j.s)) * 0.6931471805599453f;
  }
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
RX_DEV float rx_lm_unorder(rx_u32 o) { return rx_u2f(o & 0x80000000u ? o & 0x7fffffffu : ~o); }
RX_DEV rx_u64 rx_lm_key(float x, int j) { return ((rx_u64)rx_lm_order(x) << 32) | (rx_u32)~j; }

// A row of V elements as vectors of 16 bytes that are aligned in memory: vector v holds the elements [v NE - off, v NE - off + NE),
// off being how far the row starts inside of a vector.  The vectors at both ends may reach over the row.
template <typename E, int V>
struct rx_lm_row {
  typedef typename E::S S;
  static constexpr int NE = 16 / sizeof(S), SHIFTS = V % NE ? 1 : 0, VECTORS = (V + NE - 1) / NE + SHIFTS;
  const S* x;
  int off;
  const rx_vec<S, NE>* vectors;   // counted from the tensor's start: a uniform load's address is made of aligned parts (a scalar load drops the low bits of each part)
  RX_MEM rx_lm_row(const S* all, const long long t)
      : x(all + t * V), off(SHIFTS ? (int)((t * (V % NE)) % NE) : 0), vectors((const rx_vec<S, NE>*)all + (t * V - off) / NE) {}
  RX_MEM int first(const int v) const { return v * NE - off; }
  RX_MEM bool whole(const int v) const { return V >= 2 * NE && v * NE >= off && (v + 1) * NE - off <= V; }
  // the whole vector nearest to v, so that the loads of a loop carry no conditions; get() corrects those at the ends
  RX_MEM rx_vec<S, NE> load(const int v) const {
    if constexpr (V >= 2 * NE) {
      const int lo = off > 0 ? 1 : 0, hi = (V + off) / NE - 1;
      return rx_load_nt<rx_vec<S, NE>>(vectors + (v < lo ? lo : v > hi ? hi : v));
    } else {
      return rx_vec<S, NE>{};
    }
  }
  RX_MEM void get(const rx_vec<S, NE>& r, const int v, const float fill, float (&e)[NE]) const {
#pragma unroll
    for (int k = 0; k < NE; ++k) e[k] = E::up(r.v[k]);
    if (!whole(v)) {
#pragma unroll
      for (int k = 0; k < NE; ++k) e[k] = first(v) + k >= 0 && first(v) + k < V ? E::up(x[first(v) + k]) : fill;
    }
  }
};

// Running (maximum m, sum s of e^(x - m), sum t of e^(x - m) log2 e^(x - m)); the last gives the entropy.  An exponential is
// 2^(x L - c), one fused multiply-add and the hardware's 2^y, with c the rounded product m L: that s belongs to c and not to m
// is undone exactly where sums of another maximum come in and in the log of s.  (L is log2 e rounded to f32, off by 1e-8 of itself, which
// turns e^x into e^(x (1 + 1e-8)).)  From 1e8 on c is off by up to 8 and more, and a sum soon has no room for the factor: the sums
// of such a maximum belong to m, with differences from it (`rx_lm_careful`).  A row goes there from half of that on, so that what a
// thread lost whose own maximum was lower is e^-5e7 and less of the row's.
struct rx_lm_yes { static constexpr bool value = true; };
struct rx_lm_no { static constexpr bool value = false; };
struct rx_lm_sums { float m, s, t; };
RX_DEV bool rx_lm_plain(const float m) { return __builtin_fabsf(m) < 1e8f; }   // its sums belong to c
// what the rounding of c took from m L, exactly
RX_DEV float rx_lm_left(const float m) { return rx_lm_plain(m) ? __builtin_fmaf(m, RX_LM_LOG2E, -(m * RX_LM_LOG2E)) : 0.0f; }
RX_DEV float rx_lm_apart(const float m, const float of) {
  return rx_lm_plain(m) && rx_lm_plain(of) ? m * RX_LM_LOG2E - of * RX_LM_LOG2E : (m - of) * RX_LM_LOG2E - rx_lm_left(m) + rx_lm_left(of);
}
RX_DEV rx_lm_sums rx_lm_rebase(const rx_lm_sums a, const float m) {
  if (a.m == m || a.m == -rx_lm_inf()) return {m, a.s, a.t};   // (nothing so far: the sums are 0, or NaN)
  const float d = rx_lm_apart(a.m, m), f = __builtin_amdgcn_exp2f(d);
  return {m, a.s * f, f == 0.0f ? 0.0f : (a.t + a.s * d) * f};
}
struct rx_op_lm_sums {
  RX_MEM rx_lm_sums operator()(const rx_lm_sums& a, const rx_lm_sums& b) const {
    const float m = __builtin_fmaxf(a.m, b.m);
    const rx_lm_sums x = rx_lm_rebase(a, m), y = rx_lm_rebase(b, m);
    return {m, x.s + y.s, x.t + y.t};
  }
};
// log of the sum of e^(x - m)
RX_DEV float rx_lm_log_sum(const rx_lm_sums a) { return (__builtin_log2f(a.s) - rx_lm_left(a.m)) * 0.6931471805599453f; }
RX_DEV float rx_lm_lse(const rx_lm_sums a) { return a.s == 0.0f ? -rx_lm_inf() : a.m + rx_lm_log_sum(a); }
// x - lse, the difference from the maximum first: lse's own rounding would be far larger than the result where logits are
RX_DEV float rx_lm_log_probability(const float x, const rx_lm_sums a) { return a.s == 0.0f ? -rx_lm_inf() : (x - a.m) - rx_lm_log_sum(a); }
// the sums of a workgroup's threads
RX_DEV rx_lm_sums rx_lm_block_sums(rx_lm_sums a, rx_lm_sums* red /* 4 */) {
  a = rx_lm_rebase(a, rx_wave_reduce(a.m, rx_op_max()));
  a.s = rx_wave_reduce(a.s, rx_op_add());
  a.t = rx_wave_reduce(a.t, rx_op_add());
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = a;
  __syncthreads();
  return rx_op_lm_sums()(rx_op_lm_sums()(red[0], red[1]), rx_op_lm_sums()(red[2], red[3]));
}
// elements [j0, j1) of a row in two passes, the second with the maximum of all
template <typename E>
RX_DEV rx_lm_sums rx_lm_careful(const typename E::S* x, const int j0, const int j1, rx_lm_sums* red) {
  rx_lm_sums a = {-rx_lm_inf(), 0.0f, 0.0f};
  for (int j = j0 + (int)threadIdx.x; j < j1; j += 256) a.m = __builtin_fmaxf(a.m, E::up(x[j]));
  a.m = rx_lm_block_sums(a, red).m;
  const float base = a.m == -rx_lm_inf() ? 0.0f : a.m, c = base * RX_LM_LOG2E;
  const bool plain = rx_lm_plain(a.m);
  for (int j = j0 + (int)threadIdx.x; j < j1; j += 256) {
    const float e = E::up(x[j]), d = plain ? __builtin_fmaf(e, RX_LM_LOG2E, -c) : (e - base) * RX_LM_LOG2E, p = __builtin_amdgcn_exp2f(d);
    a.s += p;
    a.t = __builtin_fmaf(p, __builtin_fmaxf(d, -1e30f), a.t);
  }
  return rx_lm_block_sums(a, red);
}
RX_DEV float rx_lm_max3(const float a, const float b, const float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));   // (without the compiler's quieting of its operands)
  return r;
}
template <int N>
RX_DEV float rx_lm_max_of(const float (&e)[N]) {
  float m = rx_lm_max3(e[0], e[1], e[2]);
#pragma unroll
  for (int k = 3; k < N; k += 2) m = rx_lm_max3(m, e[k], e[k + 1 < N ? k + 1 : k]);
  return m;
}

// the K largest of `n` keys in LDS (n up to what the caller holds), the i-th largest given to put(i, key)
template <int K, typename F>
RX_DEV void rx_lm_select(const rx_u64* keys, const int n, F put) {
  for (int i = threadIdx.x; i < n; i += 256) {
    const rx_u64 mine = keys[i];
    int rank = 0;
    for (int k = 0; k < n; ++k) rank += keys[k] > mine;
    if (rank < K) put(rank, mine);
  }
}

// log probability, lse and entropy of a row, and the K largest keys in `best`, from the row's sums
template <typename E, int V, typename I>
RX_DEV void rx_lm_row_results(const long long t, const rx_lm_sums a, const typename E::S* x, const I* targets, float* logprob, float* lse, float* entropy) {
  const I y = targets[t];
  lse[t] = rx_lm_lse(a);
  entropy[t] = a.s == 0.0f ? 0.0f : (__builtin_log2f(a.s) - a.t / a.s) * 0.6931471805599453f;
  logprob[t] = y < 0 || y >= V ? 0.0f : rx_lm_log_probability(E::up(x[y]), a);
}

// A workgroup per segment of a row (SPLIT segments; one: the whole row), in one pass with the running sums, and the alternatives
// almost without a second one.  With k alternatives asked for, the k-th largest of the maxima of 64 groups of four threads (of all
// threads for many alternatives) is no larger than the k-th largest element.  Every thread leaves the maximum of each of its
// SECTIONS stretches in LDS (the upper half of its order), so only the few stretches whose maximum reaches that bound are read
// again, and the elements that reach it, hardly more than k, are ranked by (value, index).  Where too many do, because they are equal (a constant row, a mask that
// leaves fewer than k tokens), the larger ones are taken, and of the equal ones the first in the row.  A row with a NaN, or
// with more larger ones than LDS holds (far from any distribution), is searched k times.
// Of a split row every workgroup leaves its sums and keys, and the one that arrives last combines them.
// 4096 rows of 131072 logits in bf16 with 20 alternatives, 1.07 GB: 180 us, 6.0 TB/s; bound by the reads and, nearly as much, by the
// vector units: an exponential, two fused multiply-adds, a maximum and the conversion of every element.  (Two passes, sums after the
// maximum: 252 us; alternatives by k searches through the row: 12.25 ms.)  32 rows of 32000: 11.5 us of dependent steps.
template <typename E, int V, int K, int T, int SPLIT, typename I>
RX_DEV void rx_token_logprobs(const typename E::S* logits, const I* targets, float* logprob, float* lse, float* entropy, float* values, int* ids, float* part_sums, rx_u64* part_keys,
                              int* arrived) {
  typedef typename E::S S;
  constexpr int NE = 16 / sizeof(S), UNROLL = 4, ROUND = 256 * UNROLL, VECTORS = rx_lm_row<E, V>::VECTORS;
  constexpr int CAP = K * SPLIT > 1024 ? K * SPLIT : 1024, LIST = 1024;
  constexpr int ROUNDS = ((VECTORS + SPLIT - 1) / SPLIT + ROUND - 1) / ROUND, EACH = (ROUNDS + 15) / 16, SECTIONS = (ROUNDS + EACH - 1) / EACH;   // rounds of a section
  __shared__ rx_lm_sums red[4];
  __shared__ rx_u64 keys[K ? CAP : 1], red64[4];
  __shared__ rx_u16 reach[K ? SECTIONS : 1][256], listed[K ? LIST : 1];
  constexpr int GROUPS = K <= 48 ? 64 : 256;                   // 4096 x 65536 in bf16: 20 of 64 groups 100 us, of 256 116; 48: 120 and 122; 64: 283 (a bound that hundreds reach) and 129
  __shared__ rx_u32 group[GROUPS], bound;
  __shared__ int count, nlist, last;
  for (long long item = blockIdx.x; item < (long long)T * SPLIT; item += gridDim.x) {
    const long long t = item / SPLIT;
    const int seg = (int)(item % SPLIT), v0 = (int)((long long)VECTORS * seg / SPLIT), v1 = (int)((long long)VECTORS * (seg + 1) / SPLIT);
    const rx_lm_row<E, V> row(logits, t);
    const int j0 = row.first(v0) > 0 ? row.first(v0) : 0, j1 = row.first(v1) < V ? row.first(v1) : V;   // its elements
    rx_lm_sums a = {-rx_lm_inf(), 0.0f, 0.0f};
    float high = -rx_lm_inf();                                 // of the section
    auto round = [&](const int v, auto ends) {                 // vectors v, v + 256, ..; ends: some may not be whole, or in the segment
      rx_vec<S, NE> r[UNROLL];
      float e[UNROLL][NE], top[UNROLL];
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) r[u] = decltype(ends)::value ? row.load(v + 256 * u) : rx_load_nt<rx_vec<S, NE>>(row.vectors + v + 256 * u);
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) {
        if constexpr (decltype(ends)::value) {
          row.get(r[u], v + 256 * u, -rx_lm_inf(), e[u]);
          if (SPLIT > 1 && v + 256 * u >= v1) {
#pragma unroll
            for (int k = 0; k < NE; ++k) e[u][k] = -rx_lm_inf();
          }
        } else {
#pragma unroll
          for (int k = 0; k < NE; ++k) e[u][k] = E::up(r[u].v[k]);
        }
        top[u] = rx_lm_max_of(e[u]);
      }
      high = rx_lm_max3(rx_lm_max3(high, top[0], top[1]), top[2], top[3]);
      if (high > a.m) a = rx_lm_rebase(a, high);
      const float c = rx_lm_plain(a.m) ? a.m * RX_LM_LOG2E : 0.0f;
#pragma unroll
      for (int u = 0; u < UNROLL; ++u)
#pragma unroll
        for (int k = 0; k < NE; ++k) {
          const float d = __builtin_fmaf(e[u][k], RX_LM_LOG2E, -c), p = __builtin_amdgcn_exp2f(d);
          a.s += p;
          a.t = __builtin_fmaf(p, __builtin_fmaxf(d, -1e30f), a.t);   // (0 times -inf is no 0)
        }
    };
    static_assert(UNROLL == 4, "maxima of four vectors");
    __syncthreads();                                            // (the item before is through with the LDS)
    int at = v0 + (int)threadIdx.x, nth = 0;
    for (int v = v0; v < v1; v += ROUND, at += ROUND, ++nth) {
      if (v + ROUND <= v1 && row.whole(v) && row.whole(v + ROUND - 1)) round(at, rx_lm_no());
      else round(at, rx_lm_yes());
      if (K > 0 && (nth % EACH == EACH - 1 || v + ROUND >= v1)) {
        reach[nth / EACH][threadIdx.x] = (rx_u16)(rx_lm_order(high) >> 16);
        high = -rx_lm_inf();
      }
    }
    const float own = a.m;
    a = rx_lm_block_sums(a, red);
    if (!(a.s < rx_lm_inf()) || (__builtin_fabsf(a.m) >= 5e7f && a.m != -rx_lm_inf())) a = rx_lm_careful<E>(row.x, j0, j1, red);
    int n = 0;
    if constexpr (K > 0) {
      rx_u32 quad = rx_lm_order(own);
      if constexpr (GROUPS == 64) {
        quad = rx_max(quad, rx_dpp_t<rx_u32, 0xB1, 0xf>(quad));
        quad = rx_max(quad, rx_dpp_t<rx_u32, 0x4E, 0xf>(quad));
        if ((threadIdx.x & 3) == 0) group[threadIdx.x >> 2] = quad;
      } else {
        group[threadIdx.x] = quad;
      }
      if (threadIdx.x == 0) count = nlist = 0;
      __syncthreads();
      if (threadIdx.x < GROUPS) {
        const rx_u32 g = group[threadIdx.x];
        int rank = 0;
#pragma unroll 16
        for (int k = 0; k < GROUPS; ++k) {
          const rx_u32 o = group[k];
          rank += o > g || (o == g && k < (int)threadIdx.x);
        }
        if (rank == K - 1) bound = g;
      }
      __syncthreads();
      const rx_u32 least = bound;
      auto take = [&](const float x, const int j, const bool also_equal) {
        const rx_u32 o = rx_lm_order(x);
        if (o > least || (also_equal && o == least)) {
          const int i = atomicAdd(&count, 1);
          if (i < CAP) keys[i] = rx_lm_key(x, j);
        }
      };
      const bool nan = a.s != a.s;
      if (!nan) {
        for (int k = 0; k < nth; k += EACH)                     // sections that reach the bound
          if (reach[k / EACH][threadIdx.x] >= least >> 16) {
            const int i = atomicAdd(&nlist, 1);
            if (i < LIST) listed[i] = (rx_u16)(k / EACH << 8 | threadIdx.x);
          }
        __syncthreads();
        if (nlist <= LIST)
          for (int k = threadIdx.x; k < nlist * EACH * UNROLL; k += 256) {
            const int what = listed[k / (EACH * UNROLL)], v = v0 + (what >> 8) * (EACH * ROUND) + k % (EACH * UNROLL) * 256 + (what & 255), j = row.first(v);
            if (v >= v1) continue;
            float e[NE];
            row.get(row.load(v), v, -rx_lm_inf(), e);
#pragma unroll
            for (int q = 0; q < NE; ++q)
              if (j + q >= 0 && j + q < V) take(e[q], j + q, true);
          }
        __syncthreads();
      }
      n = count;
      bool search = nan;
      if (!nan && (nlist > LIST || n > CAP)) {
        __syncthreads();
        if (threadIdx.x == 0) count = 0;
        __syncthreads();
        for (int j = j0 + (int)threadIdx.x; j < j1; j += 256) take(E::up(row.x[j]), j, false);
        __syncthreads();
        n = count;
        search = n > CAP - 256;
        __syncthreads();                                        // (every wavefront has read the count before one adds to it)
        for (int j = j0; !search && n < K && j < j1; j += 256) {
          const int mine = j + (int)threadIdx.x;
          if (mine < j1 && rx_lm_order(E::up(row.x[mine])) == least) keys[atomicAdd(&count, 1)] = rx_lm_key(E::up(row.x[mine]), mine);
          __syncthreads();
          n = count;
          __syncthreads();
        }
      }
      if (search) {
        rx_u64 below = 0;
        for (int k = 0; k < K; ++k) {
          rx_u64 top = 0;
          for (int j = j0 + (int)threadIdx.x; j < j1; j += 256) {
            const rx_u64 key = rx_lm_key(E::up(row.x[j]), j);
            if ((k == 0 || key < below) && key > top) top = key;   // (a NaN at index 0 has the largest key there is)
          }
          __syncthreads();
          top = rx_block_reduce<rx_u64, rx_op_max, 4>(top, rx_op_max(), red64);
          if (threadIdx.x == 0) keys[k] = top;
          below = top;
        }
        n = K;
        __syncthreads();
      }
    }
    if constexpr (SPLIT > 1) {
      if (threadIdx.x == 0) {
        rx_lm_put_shared(part_sums + item * 3, a.m);
        rx_lm_put_shared(part_sums + item * 3 + 1, a.s);
        rx_lm_put_shared(part_sums + item * 3 + 2, a.t);
      }
      if constexpr (K > 0) rx_lm_select<K>(keys, n, [&](const int rank, const rx_u64 key) { rx_lm_put_shared(part_keys + item * K + rank, key); });
      if (!rx_lm_last_to_arrive(arrived + t, SPLIT, &last)) continue;
      if constexpr (K > 0)
        for (int k = threadIdx.x; k < K * SPLIT; k += 256) keys[k] = rx_lm_get_shared(part_keys + t * (SPLIT * K) + k);
      n = K * SPLIT;
      a = {-rx_lm_inf(), 0.0f, 0.0f};
      if (threadIdx.x < SPLIT) a = {rx_lm_get_shared(part_sums + (t * SPLIT + threadIdx.x) * 3), rx_lm_get_shared(part_sums + (t * SPLIT + threadIdx.x) * 3 + 1),
                                    rx_lm_get_shared(part_sums + (t * SPLIT + threadIdx.x) * 3 + 2)};
      a = rx_lm_block_sums(a, red);
    }
    if (threadIdx.x == 0) rx_lm_row_results<E, V>(t, a, row.x, targets, logprob, lse, entropy);
    if constexpr (K > 0) {
      rx_lm_select<K>(keys, n, [&](const int rank, const rx_u64 key) {
        const int j = (int)~(rx_u32)key;
        ids[t * K + rank] = j;
        values[t * K + rank] = rx_lm_log_probability(E::up(row.x[j]), a);
      });
    }
  }
}

// d x_j = g (delta_jy - p_j) - h p_j (x_j - lse + H): a thread per vector of a row, a workgroup per 256 of them.  4096 rows of
// 50021 logits in bf16 take 135 us, 6.1 TB/s of reading and writing, as a copy reaches; two vectors to a thread 138, four 142.
template <typename E, int V, int T, typename I>
RX_DEV void rx_token_logprobs_grad(const typename E::S* logits, const I* targets, const float* lse, const float* entropy, const float* d_logprob, const float* d_entropy,
                                   typename E::S* out) {
  typedef typename E::S S;
  constexpr int NE = 16 / sizeof(S), VECTORS = rx_lm_row<E, V>::VECTORS, PARTS = (VECTORS + 255) / 256;
  for (long long item = blockIdx.x; item < (long long)T * PARTS; item += gridDim.x) {
    const long long t = item / PARTS;
    const int v = (int)(item % PARTS) * 256 + (int)threadIdx.x;
    const rx_lm_row<E, V> row(logits, t);
    const int j = row.first(v);
    const rx_vec<S, NE> r = row.load(v);
    const I y = targets[t];
    const bool counts = y >= 0 && y < V;
    const float l = lse[t] == -rx_lm_inf() ? rx_lm_inf() : lse[t];   // (a row of nothing: all probabilities 0)
    const float g = counts ? d_logprob[t] : 0.0f, h = d_entropy[t], c = g + h * entropy[t];
    if (v >= VECTORS) continue;
    float e[NE];
    row.get(r, v, 0.0f, e);
    rx_vec<S, NE> w;
#pragma unroll
    for (int k = 0; k < NE; ++k) {
      const float z = e[k] - l, p = __builtin_amdgcn_exp2f(z * RX_LM_LOG2E);
      float d = -p * __builtin_fmaf(h, __builtin_fmaxf(z, -200.0f), c);   // (p is 0 from there on, and 0 times -inf is no 0)
      if (counts && (long long)y - j == k) d += g;
      w.v[k] = E::down(d);
    }
    S* o = out + t * V + j;
    if (row.whole(v)) rx_store_nt(o, w);
    else {
#pragma unroll
      for (int k = 0; k < NE; ++k)
        if (j + k >= 0 && j + k < V) o[k] = w.v[k];
    }
  }
}
