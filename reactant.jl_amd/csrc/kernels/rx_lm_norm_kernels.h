// Device code of numbers in 8 bits with scales, and of root-mean-square norms (csrc/rx_lm.h states what they compute).
#pragma once
#include "rx_lm_kernels.h"

// Numbers of 8 bits that stand for their product with a scale: floats of 4 exponent and 3 mantissa bits, or whole numbers.
struct rx_lm_f8 {
  typedef rx_u8 S;
  static constexpr float LARGEST = 448.0f;
  RX_MEM static float up(S x) { return rx_e4m3_to_f32(x); }
  // two numbers in the low 16 bits; |x| and |y| at most a rounding above LARGEST
  RX_MEM static rx_u32 pair(float x, float y) {
    return (rx_u32)__builtin_amdgcn_cvt_pk_fp8_f32(rx_clamp_ordered(x, -LARGEST, LARGEST), rx_clamp_ordered(y, -LARGEST, LARGEST), 0, false) & 0xffffu;
  }
};
struct rx_lm_i8 {
  typedef rx_u8 S;
  static constexpr float LARGEST = 127.0f;
  RX_MEM static float up(S x) { return (float)(rx_i8)x; }
  RX_MEM static rx_u32 pair(float x, float y) {
    return ((rx_u32)(int)__builtin_rintf(rx_clamp_ordered(x, -LARGEST, LARGEST)) & 0xffu) | (((rx_u32)(int)__builtin_rintf(rx_clamp_ordered(y, -LARGEST, LARGEST)) & 0xffu) << 8);
  }
};
template <typename C> struct rx_lm_is8 { static constexpr bool value = false; };
template <> struct rx_lm_is8<rx_lm_f8> { static constexpr bool value = true; };
template <> struct rx_lm_is8<rx_lm_i8> { static constexpr bool value = true; };

// A row's scale from the bits of its largest magnitude (as whole numbers, infinities and NaN compare above all others): the
// largest over LARGEST, but not from less than 2^-100, so that it is a normal number whose quotients are finite.  NaN where the row
// holds an infinity or NaN: its numbers, all zero, stand for NaN then.
template <typename C>
RX_DEV float rx_lm_scale_of(const rx_u32 largest) {
  if (largest >= 0x7f800000u) return __builtin_nanf("");
  return __builtin_fmaxf(rx_u2f(largest), 0x1p-100f) / C::LARGEST;
}
// numbers of N values of a row of that scale: quotients in f32, rounded to nearest, ties to even
template <typename C, int N>
RX_DEV rx_vec<rx_u8, N> rx_lm_codes(const float (&x)[N], const float scale) {
  rx_vec<rx_u8, N> c;
  const bool there = scale == scale;
#pragma unroll
  for (int e = 0; e < N; e += 2) {
    const rx_u32 p = there ? C::pair(x[e] / scale, e + 1 < N ? x[e + 1] / scale : 0.0f) : 0u;
    c.v[e] = (rx_u8)p;
    if (e + 1 < N) c.v[e + 1] = (rx_u8)(p >> 8);
  }
  return c;
}

struct rx_lm_umax {
  RX_MEM rx_u32 operator()(rx_u32 a, rx_u32 b) const { return a > b ? a : b; }
};

// Sum or maximum over the lanes of a row: a wavefront, or a workgroup, whose exchange alternates between two places so that
// one barrier is enough.  The wavefronts' values are joined two by two: at most 6 + 4 roundings of a sum behind a lane's own.
template <int WAVES, typename T, typename OP>
RX_DEV T rx_lm_join_waves(const T (&v)[WAVES], OP op) {
  T x[WAVES];
#pragma unroll
  for (int w = 0; w < WAVES; ++w) x[w] = v[w];
#pragma unroll
  for (int n = WAVES / 2; n > 0; n /= 2)
#pragma unroll
    for (int w = 0; w < n; ++w) x[w] = op(x[w], x[w + n]);
  return x[0];
}
template <int LANES, typename T, typename OP>
RX_DEV T rx_lm_row_reduce(T v, OP op, T (*red)[LANES / 64], const int turn) {
  v = rx_wave_reduce(v, op);
  if constexpr (LANES > 64) {
    if ((threadIdx.x & 63) == 0) red[turn & 1][threadIdx.x >> 6] = v;
    __syncthreads();
    v = rx_lm_join_waves(red[turn & 1], op);
  }
  return v;
}

// ---------------------------------------------------------------------------
// norm: a row to a wavefront or a workgroup of LANES lanes, EACH vectors of VEC elements to a lane, LANES apart; the row stays in
// registers between the sum of its squares, its largest magnitude and its results.  Bound by memory: 16384 rows of 4096 bf16 with their
// residual, into 8 bits, 470 MB, take 77 us, 6.1 TB/s, a copy's rate.  48 rows take 3.7 us, a launch and a row's chain.  Rows of up to 512 elements
// leave lanes idle: 84 MB of 256, 128 and 64 bf16 without residual 42, 73 and 134 us, where 24 is a copy's time.
// ---------------------------------------------------------------------------
template <typename E, typename O, int D, int ROWS, int LANES, int VEC, int EACH, bool RES>
RX_DEV void rx_rms_norm(const typename E::S* x, const typename E::S* res, const typename E::S* weight, typename E::S* h, typename O::S* y, float* scale, const float eps) {
  constexpr int C = D / VEC, BLOCK = LANES < 256 ? 256 : LANES, LINES = BLOCK / LANES;
  typedef rx_vec<typename E::S, VEC> W;
  __shared__ float sums[2][LANES / 64];
  __shared__ rx_u32 tops[2][LANES / 64];
  const int lane = threadIdx.x % LANES;
  int turn = 0;
  for (long long row = (long long)blockIdx.x * LINES + threadIdx.x / LANES; row < ROWS; row += (long long)gridDim.x * LINES, ++turn) {
    W a[EACH], b[EACH], w[EACH];
#pragma unroll
    for (int n = 0; n < EACH; ++n) {
      const int c = lane + n * LANES < C ? lane + n * LANES : C - 1;
      a[n] = rx_load_nt<W>(x + row * D + c * VEC);
      if constexpr (RES) b[n] = rx_load_nt<W>(res + row * D + c * VEC);
    }
#pragma unroll
    for (int n = 0; n < EACH; ++n) w[n] = rx_load<W>(weight + (lane + n * LANES < C ? lane + n * LANES : C - 1) * VEC);
    float v[EACH][VEC], sum = 0.0f;
#pragma unroll
    for (int n = 0; n < EACH; ++n) {
      const bool in = lane + n * LANES < C;
      W o;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        v[n][e] = E::up(a[n].v[e]);
        if constexpr (RES) {
          v[n][e] += E::up(b[n].v[e]);
          o.v[e] = E::down(v[n][e]);
        }
        if (in) sum += v[n][e] * v[n][e];
      }
      if constexpr (RES)
        if (in) rx_store_nt(h + row * D + (lane + n * LANES) * VEC, o);
    }
    sum = rx_lm_row_reduce<LANES>(sum, rx_op_add(), sums, turn);
    const float r = rx_rsqrt(sum / (float)D + eps);
    rx_u32 top = 0;
#pragma unroll
    for (int n = 0; n < EACH; ++n)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        v[n][e] = v[n][e] * r * E::up(w[n].v[e]);
        const rx_u32 bits = rx_f2u(v[n][e]) & 0x7fffffffu;
        top = bits > top ? bits : top;                            // (lanes past the end repeat the last vector)
      }
    float s = 0.0f;
    if constexpr (rx_lm_is8<O>::value) {
      s = rx_lm_scale_of<O>(rx_lm_row_reduce<LANES>(top, rx_lm_umax(), tops, turn));
      if (lane == 0) scale[row] = s;
    }
#pragma unroll
    for (int n = 0; n < EACH; ++n) {
      if (lane + n * LANES >= C) break;
      rx_vec<typename O::S, VEC> o;
      if constexpr (rx_lm_is8<O>::value) {
        o = rx_lm_codes<O>(v[n], s);
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) o.v[e] = O::down(v[n][e]);
      }
      rx_store_nt(y + row * D + (lane + n * LANES) * VEC, o);
    }
  }
}

// Gradient.  With u = h r the norm is y = u weight; back through it goes g = dy weight, and dx = dh + r (g - u mean(g u)).  A
// workgroup goes through its rows, GROUPS apart, and keeps its part of the weight's gradient, sum of dy u, in registers; the parts
// are added by a second launch, in the order of the workgroups: the same bits every run.  Bound by memory: 16384 rows of 4096 bf16, 537 MB,
// take 89 us, 6.0 TB/s, and 4.7 us for the parts (loading the next row while this one is added up: 90).
template <typename E, int D, int ROWS, int LANES, int VEC, int EACH, bool RES, int GROUPS>
RX_DEV void rx_rms_norm_grad(const typename E::S* h, const typename E::S* weight, const typename E::S* dy, const typename E::S* dh, typename E::S* dx, float* part, const float eps) {
  constexpr int C = D / VEC, BLOCK = LANES < 256 ? 256 : LANES, LINES = BLOCK / LANES;
  typedef rx_vec<typename E::S, VEC> W;
  __shared__ rx_vec<float, 2> sums[2][LANES / 64];
  __shared__ float joined[LINES > 1 ? LINES : 1][LINES > 1 ? D : 1];
  const int lane = threadIdx.x % LANES, line = threadIdx.x / LANES;
  float acc[EACH][VEC] = {};
  int turn = 0;
  W w[EACH];
#pragma unroll
  for (int n = 0; n < EACH; ++n) w[n] = rx_load<W>(weight + (lane + n * LANES < C ? lane + n * LANES : C - 1) * VEC);
  for (long long row = (long long)blockIdx.x * LINES + line; row < ROWS; row += (long long)GROUPS * LINES, ++turn) {
    W a[EACH], b[EACH], d[EACH];
#pragma unroll
    for (int n = 0; n < EACH; ++n) {
      const long long at = row * D + (lane + n * LANES < C ? lane + n * LANES : C - 1) * VEC;
      a[n] = rx_load_nt<W>(h + at);
      b[n] = rx_load_nt<W>(dy + at);
      if constexpr (RES) d[n] = rx_load_nt<W>(dh + at);
    }
    rx_vec<float, 2> s = {{0.0f, 0.0f}};                          // squares of h, products g h
#pragma unroll
    for (int n = 0; n < EACH; ++n)
      if (lane + n * LANES < C)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float v = E::up(a[n].v[e]);
          s.v[0] += v * v;
          s.v[1] += E::up(b[n].v[e]) * E::up(w[n].v[e]) * v;
        }
    s.v[0] = rx_wave_reduce(s.v[0], rx_op_add());
    s.v[1] = rx_wave_reduce(s.v[1], rx_op_add());
    if constexpr (LANES > 64) {
      if ((threadIdx.x & 63) == 0) sums[turn & 1][threadIdx.x >> 6] = s;
      __syncthreads();
      s = rx_lm_join_waves(sums[turn & 1], [](const rx_vec<float, 2>& a, const rx_vec<float, 2>& b) { return rx_vec<float, 2>{{a.v[0] + b.v[0], a.v[1] + b.v[1]}}; });
    }
    const float r = rx_rsqrt(s.v[0] / (float)D + eps), m = s.v[1] * r / (float)D;
#pragma unroll
    for (int n = 0; n < EACH; ++n) {
      if (lane + n * LANES >= C) break;
      W o;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float u = E::up(a[n].v[e]) * r, g = E::up(b[n].v[e]);
        float t = r * (g * E::up(w[n].v[e]) - u * m);
        if constexpr (RES) t += E::up(d[n].v[e]);
        o.v[e] = E::down(t);
        acc[n][e] += g * u;
      }
      rx_store_nt(dx + row * D + (lane + n * LANES) * VEC, o);
    }
  }
  if constexpr (LINES > 1) {                                      // the wavefronts' rows, in their order
#pragma unroll
    for (int n = 0; n < EACH; ++n)
      if (lane + n * LANES < C)
#pragma unroll
        for (int e = 0; e < VEC; ++e) joined[line][(lane + n * LANES) * VEC + e] = acc[n][e];
    __syncthreads();
    for (int i = threadIdx.x; i < D; i += BLOCK) {
      float t = joined[0][i];
#pragma unroll
      for (int k = 1; k < LINES; ++k) t += joined[k][i];
      part[(long long)blockIdx.x * D + i] = t;
    }
  } else {
#pragma unroll
    for (int n = 0; n < EACH; ++n)
      if (lane + n * LANES < C)
#pragma unroll
        for (int e = 0; e < VEC; ++e) part[(long long)blockIdx.x * D + (lane + n * LANES) * VEC + e] = acc[n][e];
  }
}
// The weight's gradient from the workgroups' parts: 64 columns to a workgroup, a vector of four to each of 16 lanes, whose 64 lines of
// lanes take every 64th part, eight of them at a time.
template <typename O, int D, int GROUPS>
RX_DEV void rx_rms_norm_weight(const float* part, typename O::S* dweight) {
  constexpr int VEC = D % 4 == 0 ? 4 : 1, LANES = 16, LINES = 1024 / LANES;
  typedef rx_vec<float, VEC> W;
  __shared__ W lines[LINES][LANES];
  const int lane = threadIdx.x % LANES, line = threadIdx.x / LANES, c = (blockIdx.x * LANES + lane) * VEC;
  W t{};
  if (c < D) {
    for (int g0 = line; g0 < GROUPS; g0 += 8 * LINES) {
      W x[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) x[k] = rx_load<W>(part + (long long)(g0 + k * LINES < GROUPS ? g0 + k * LINES : g0) * D + c);
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (g0 + k * LINES < GROUPS)
#pragma unroll
          for (int e = 0; e < VEC; ++e) t.v[e] += x[k].v[e];
    }
  }
  lines[line][lane] = t;
  __syncthreads();
  const int o = threadIdx.x;
  if (o >= LANES * VEC || blockIdx.x * LANES * VEC + o >= D) return;
  float sum = 0.0f;
#pragma unroll 8
  for (int k = 0; k < LINES; ++k) sum += lines[k][o / VEC].v[o % VEC];
  dweight[blockIdx.x * LANES * VEC + o] = O::down(sum);
}
