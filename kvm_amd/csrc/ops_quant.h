// Products in 8-bit integers with a scale for each row of activations and of weights (ops 315-317). Semantics: mvm_ops_kvm.def.
#pragma once
#include "common.h"
#include "ops_basic.h"
#include "ops_gemm.h"
#include "ops_decode.h"
#include "ops_serve.h"
#include "gemv_q8_geo.h"

namespace kvm {

typedef int i32x16_t __attribute__((ext_vector_type(16)));

// ---------------------------------------------------------------------------------------------- rows in 8 bits
// v of a row (x, RMS-normalised x, silu(x) * x2) in vectors of 8: thread t has vectors t, t + 256, .. How x (and x2) are read, FORM: 1 f32, 2 bf16
// rows that start at whole words, 3 other bf16 rows, all by 16-byte loads through a descriptor that ends with the row's K values (any alignment of a
// word, zeros behind the end: only bf16 values that share a word with the last one are masked); 0 element by element, where x and x2 are of two types.
// A form of its own for each: a branch on the type between two loads makes each wait for the one before.
template <int FORM> struct RawRow {
  u32x4_t a, b; uint32_t c;
  __device__ __forceinline__ void load(const View& X, long long row, int j, int K) {   // vector j of the row
    const long long e0 = row * X.cols;
    if constexpr (FORM == 0) {
      const int n = K - 8 * j;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        a[e] = e < n ? __float_as_uint(X.ld(e0 + 8 * j + e)) : 0u;
        b[e] = e + 4 < n ? __float_as_uint(X.ld(e0 + 8 * j + 4 + e)) : 0u;
      }
    } else if constexpr (FORM == 1) {
      const __amdgpu_buffer_rsrc_t rs = buf_rsrc((const void*)(X.f() + e0), 4ll * K);
      a = __builtin_amdgcn_raw_buffer_load_b128(rs, 32 * j, 0, 0);
      b = __builtin_amdgcn_raw_buffer_load_b128(rs, 32 * j + 16, 0, 0);
    } else {
      const uintptr_t p = (uintptr_t)(X.h() + e0);
      const __amdgpu_buffer_rsrc_t rs = buf_rsrc((const void*)(p & ~(uintptr_t)3), (2ll * K + (p & 2) + 3) & ~3ll);   // (a last half word with its whole word)
      a = __builtin_amdgcn_raw_buffer_load_b128(rs, 16 * j, 0, 0);
      if constexpr (FORM == 3) c = __builtin_amdgcn_raw_buffer_load_b32(rs, 16 * j + 16, 0, 0);
    }
  }
  __device__ __forceinline__ void get(const View& X, long long row, int j, int K, float (&v)[8]) const {
    if constexpr (FORM <= 1) {
#pragma unroll
      for (int e = 0; e < 4; ++e) { v[e] = __uint_as_float(a[e]); v[4 + e] = __uint_as_float(b[e]); }
    } else {
      uint32_t w[4] = {a.x, a.y, a.z, a.w};
      if constexpr (FORM == 3) {
        const uint32_t odd = (uint32_t)((uintptr_t)(X.h() + row * X.cols) & 2) * 8;        // bits that the row starts into its word
        w[0] = __builtin_amdgcn_alignbit(a.y, a.x, odd); w[1] = __builtin_amdgcn_alignbit(a.z, a.y, odd);
        w[2] = __builtin_amdgcn_alignbit(a.w, a.z, odd); w[3] = __builtin_amdgcn_alignbit(c, a.w, odd);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = __uint_as_float(e & 1 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16);
    }
    if (FORM >= 2 && (FORM == 3 || (K & 1)))
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = 8 * j + e < K ? v[e] : 0.f;
  }
};
struct RowsSrc {
  View x, x2, g; int K, pro; float eps;
  __device__ int form() const {
    if (pro == 2 && x2.dtype != x.dtype) return 0;
    if (x.dtype != 2) return 1;
    return ((x.cols | (pro == 2 ? x2.cols : 0)) & 1) == 0 && (((uintptr_t)x.p | (pro == 2 ? (uintptr_t)x2.p : 0)) & 3) == 0 ? 2 : 3;
  }
};
// NV vectors of RB rows on their way, with what stands in front of them.
template <int FORM, int NV, int RB> struct RowsRaw {
  RawRow<FORM> x[RB][NV], y[RB][NV];
  RawRow<1> g[NV];
  __device__ __forceinline__ void load(const RowsSrc& S, long long r0, int nr, int j0) {
#pragma unroll
    for (int i = 0; i < RB; ++i)
#pragma unroll
      for (int u = 0; u < NV; ++u) x[i][u].load(S.x, r0 + min(i, nr - 1), j0 + u * KVM_THREADS, S.K);
    if (S.pro == 1)
#pragma unroll
      for (int u = 0; u < NV; ++u) g[u].load(S.g, 0, j0 + u * KVM_THREADS, S.K);
    if (S.pro == 2)
#pragma unroll
      for (int i = 0; i < RB; ++i)
#pragma unroll
        for (int u = 0; u < NV; ++u) y[i][u].load(S.x2, r0 + min(i, nr - 1), j0 + u * KVM_THREADS, S.K);
  }
  // x * rstd * gamma, or silu(x) * x2: rounded after each product
  __device__ __forceinline__ void shape(const RowsSrc& S, long long row, int i, int u, int j, float rstd, float (&v)[8]) const {
    float w[8];
    if (S.pro == 1) {
      g[u].get(S.g, 0, j, S.K, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) { const float t = v[e] * rstd; v[e] = t * w[e]; }
    } else if (S.pro == 2) {
      y[i][u].get(S.x2, row, j, S.K, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = silu_f(v[e]) * w[e];
    }
  }
};
__device__ __forceinline__ uint32_t q8_big(const float (&v)[8], uint32_t big) {   // magnitudes by their bits: what is not finite is largest
#pragma unroll
  for (int e = 0; e < 8; ++e) big = max(big, __float_as_uint(v[e]) & 0x7fffffffu);
  return big;
}
// Sum of doubles over a wave in registers (as lanes_all and rows_all move floats): through LDS four rows' sums took a third of a round.
template <int CTRL> __device__ __forceinline__ double dpp_d(double v) {
  const unsigned long long u = __builtin_bit_cast(unsigned long long, v);
  const unsigned lo = __builtin_amdgcn_update_dpp(0, (int)(unsigned)u, CTRL, 0xf, 0xf, true), hi = __builtin_amdgcn_update_dpp(0, (int)(unsigned)(u >> 32), CTRL, 0xf, 0xf, true);
  return __builtin_bit_cast(double, ((unsigned long long)hi << 32) | lo);
}
__device__ __forceinline__ double wave_all_d(double v) {
  v += dpp_d<0xB1>(v); v += dpp_d<0x4E>(v); v += dpp_d<0x141>(v); v += dpp_d<0x140>(v);
  auto both = [](double x, bool far) {
    const unsigned long long u = __builtin_bit_cast(unsigned long long, x);
    const unsigned lo = (unsigned)u, hi = (unsigned)(u >> 32);
    auto a = far ? __builtin_amdgcn_permlane32_swap(lo, lo, false, false) : __builtin_amdgcn_permlane16_swap(lo, lo, false, false);
    auto b = far ? __builtin_amdgcn_permlane32_swap(hi, hi, false, false) : __builtin_amdgcn_permlane16_swap(hi, hi, false, false);
    return __builtin_bit_cast(double, ((unsigned long long)b[0] << 32) | a[0]) + __builtin_bit_cast(double, ((unsigned long long)b[1] << 32) | a[1]);
  };
  return both(both(v, false), true);
}
// One sum or maximum per row over the workgroup, the waves' in order; red: 4 * RB of LDS.
template <int RB> __device__ __forceinline__ void q8_rows_sum(double (&s)[RB], LDS double* red) {
#pragma unroll
  for (int i = 0; i < RB; ++i) s[i] = wave_all_d(s[i]);
  __syncthreads();
  if (lane() == 0)
#pragma unroll
    for (int i = 0; i < RB; ++i) red[4 * i + wave()] = s[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < RB; ++i) s[i] = (red[4 * i] + red[4 * i + 1]) + (red[4 * i + 2] + red[4 * i + 3]);
}
template <int RB> __device__ __forceinline__ void q8_rows_max(uint32_t (&b)[RB], LDS double* red_) {
  LDS uint32_t* red = (LDS uint32_t*)red_ + 8 * RB;
#pragma unroll
  for (int i = 0; i < RB; ++i) b[i] = __float_as_uint(rows_max(lanes_max<16>(__uint_as_float(min(b[i], 0x7f800000u)))));
  __syncthreads();
  if (lane() == 0)
#pragma unroll
    for (int i = 0; i < RB; ++i) red[4 * i + wave()] = b[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < RB; ++i) b[i] = max(max(red[4 * i], red[4 * i + 1]), max(red[4 * i + 2], red[4 * i + 3]));
}
constexpr int Q8_RED = 12;     // doubles of LDS per row in flight
// nr <= RB rows from r0 on, K <= 2048 NV, from `raw` (requested before), held in registers: one reduction for the norm and one for the scale whatever RB
// is; `next` is called once the rows are out of raw, to request others under the reductions. put(i, j, w0, w1): vector j of row r0 + i as bytes;
// scaled(i, s). Sums of squares in double, so that rstd is the f32 nearest to the exact one.
template <int FORM, int NV, int RB, class Put, class Scaled, class Next>
__device__ __forceinline__ void q8_rows(const RowsSrc& S, RowsRaw<FORM, NV, RB>& raw, long long r0, int nr, LDS double* red, Put put, Scaled scaled, Next next) {
  const int nvec = (S.K + 7) >> 3;
  float v[RB][NV][8];
  double ss[RB] = {};
#pragma unroll
  for (int i = 0; i < RB; ++i)
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      if (NV > 2 && u * 8 * KVM_THREADS >= S.K) break;
      raw.x[i][u].get(S.x, r0 + min(i, nr - 1), tid() + u * KVM_THREADS, S.K, v[i][u]);
      if (S.pro == 1 && i < nr)
#pragma unroll
        for (int e = 0; e < 8; ++e) ss[i] += (double)v[i][u][e] * (double)v[i][u][e];
    }
  if (S.pro == 1) q8_rows_sum<RB>(ss, red);
  uint32_t big[RB] = {};
  float mine = 0.f;                                                    // lane i brings the reciprocal root of row i (division and root are 100 instructions)
  if (S.pro == 1) {
    double x = ss[0];
#pragma unroll
    for (int i = 1; i < RB; ++i) x = lane() == i ? ss[i] : x;
    mine = (float)(1.0 / sqrt(x / S.K + (double)S.eps));
  }
#pragma unroll
  for (int i = 0; i < RB; ++i) {
    if (i >= nr) break;
    const float rstd = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(mine), i));
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      if (NV > 2 && u * 8 * KVM_THREADS >= S.K) break;
      raw.shape(S, r0 + i, i, u, tid() + u * KVM_THREADS, rstd, v[i][u]);
      big[i] = q8_big(v[i][u], big[i]);
    }
  }
  next();
  q8_rows_max<RB>(big, red);
#pragma unroll
  for (int i = 0; i < RB; ++i) {
    if (i >= nr) break;
    const float s = q8_scale(__uint_as_float(big[i])), inv = s > 0.f ? 1.f / s : 0.f;
    if (tid() == 0) scaled(i, s);
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      if (NV > 2 && u * 8 * KVM_THREADS >= S.K) break;
      uint32_t w0, w1;
      q8_pack(v[i][u], s, inv, w0, w1);
      if (tid() + u * KVM_THREADS < nvec) put(i, tid() + u * KVM_THREADS, w0, w1);
    }
  }
}
// A row of any length, read three times.
template <int FORM, class Put, class Scaled>
__device__ __forceinline__ void q8_row_long(const RowsSrc& S, long long r, LDS double* red, Put put, Scaled scaled) {
  const int nvec = (S.K + 7) >> 3;
  double ss[1] = {};
  RowsRaw<FORM, 1, 1> raw;
  float v[8];
  auto get = [&](int j, float rstd, bool shaped) {
    raw.load(S, r, 1, j);
    raw.x[0][0].get(S.x, r, j, S.K, v);
    if (shaped) raw.shape(S, r, 0, 0, j, rstd, v);
  };
  if (S.pro == 1) {
    for (int j = tid(); j < nvec; j += KVM_THREADS) {
      get(j, 0.f, false);
#pragma unroll
      for (int e = 0; e < 8; ++e) ss[0] += (double)v[e] * (double)v[e];
    }
    q8_rows_sum<1>(ss, red);
  }
  const float rstd = (float)(1.0 / sqrt(ss[0] / S.K + (double)S.eps));
  uint32_t big[1] = {};
  for (int j = tid(); j < nvec; j += KVM_THREADS) { get(j, rstd, true); big[0] = q8_big(v, big[0]); }
  q8_rows_max<1>(big, red);
  const float s = q8_scale(__uint_as_float(big[0])), inv = s > 0.f ? 1.f / s : 0.f;
  if (tid() == 0) scaled(0, s);
  for (int j = tid(); j < nvec; j += KVM_THREADS) {
    uint32_t w0, w1;
    get(j, rstd, true);
    q8_pack(v, s, inv, w0, w1);
    put(0, j, w0, w1);
  }
}

// Op 315. Bound: bytes (K * (2 to 8) read, K written a row). Four rows of up to 4,096 values at once, one of up to 16,384, so that the two
// reductions' waits are shared; the next rows are requested before this round's maximum. 4,001 rows of 4,096 bf16 values with the norm:
// 43 us a call (49 MB, 1.1 TB/s with the launch); 7 us for four rows, about half of it instructions of rounding and norm, the rest waits of one wave a
// SIMD. Masks on every value and sums of doubles through LDS made it 49 where this took 41.
template <int FORM, int NV> __device__ __noinline__ void rows_q8_t(const Ctx& c) {
  constexpr int RB = NV && NV <= 2 ? 4 : 1;
  const RowsSrc S{uview(c, 0), uview(c, 1), uview(c, 2), rfl(c.i(7)), rfl(c.i(8)), c.f(9)};
  const View q = uview(c, 3), qs = uview(c, 4);
  const int r0 = rfl(c.i(5)), r1 = rfl(c.i(6)), words = min(q.cols, ((S.K + 15) >> 4) << 2), nvec = (S.K + 7) >> 3;
  const bool pair = (q.cols & 1) == 0 && ((uintptr_t)q.p & 7) == 0;
  LDS double* red = (LDS double*)c.smem;
  RowsRaw<FORM, NV ? NV : 1, RB> raw;
  if (NV > 0 && r0 < r1) raw.load(S, r0, min(RB, r1 - r0), tid());
  for (int r = r0; r < r1; r += RB) {
    auto word = [&](GLOBAL int* p, int k, uint32_t w) { if (k < words) stwt32i(p + k, (int)w); };
    auto put = [&](int i, int j, uint32_t w0, uint32_t w1) {
      GLOBAL int* p = q.i() + (long long)(r + i) * q.cols;
      if (pair && 2 * j + 1 < words) stwt64(p + 2 * j, (uint64_t)w0 | ((uint64_t)w1 << 32));
      else { word(p, 2 * j, w0); word(p, 2 * j + 1, w1); }
      if (j == nvec - 1 && (nvec & 1)) { word(p, 2 * nvec, 0); word(p, 2 * nvec + 1, 0); }   // up to the multiple of 16 bytes
    };
    auto scaled = [&](int i, float s) { stwt32(qs.f() + (r + i), s); };
    auto next = [&]() { if (r + RB < r1) raw.load(S, r + RB, min(RB, r1 - r - RB), tid()); };
    if constexpr (NV > 0) q8_rows<FORM, NV, RB>(S, raw, r, min(RB, r1 - r), red, put, scaled, next);
    else q8_row_long<FORM>(S, r, red, put, scaled);
  }
}
__device__ __noinline__ void op_rows_q8(const Ctx& c) {
  const RowsSrc S{c.buf(0), c.buf(1), c.buf(2), c.i(7), c.i(8), c.f(9)};
  const int form = rfl(S.form());
  if (S.K <= 2048 && form) { if (form == 1) rows_q8_t<1, 1>(c); else if (form == 2) rows_q8_t<2, 1>(c); else rows_q8_t<3, 1>(c); }
  else if (S.K <= 4096) { if (form == 1) rows_q8_t<1, 2>(c); else if (form == 2) rows_q8_t<2, 2>(c); else if (form == 3) rows_q8_t<3, 2>(c); else rows_q8_t<0, 0>(c); }
  else if (S.K <= 16384 && form) { if (form == 1) rows_q8_t<1, 8>(c); else if (form == 2) rows_q8_t<2, 8>(c); else rows_q8_t<3, 8>(c); }
  else if (form == 1) rows_q8_t<1, 0>(c);
  else if (form >= 2) rows_q8_t<3, 0>(c);
  else rows_q8_t<0, 0>(c);
}

// ---------------------------------------------------------------------------------------------- product tiles
// Arguments of op 316 (a, sa, w, sw, out, bias, res, m0, n0, M, N, K, tile), wave-uniform.
struct TileQ8 {
  View a, sa, w, sw, out, bias, res; int m0, n0, M, N, K;
  __device__ explicit TileQ8(const Ctx& c)
      : a(uview(c, 0)), sa(uview(c, 1)), w(uview(c, 2)), sw(uview(c, 3)), out(uview(c, 4)), bias(uview(c, 5)), res(uview(c, 6)),
        m0(rfl(c.i(7))), n0(rfl(c.i(8))), M(rfl(c.i(9))), N(rfl(c.i(10))), K(rfl(c.i(11))) {}
  __device__ float scaled(int sum, float s, float t) const { const float y = (float)sum * s; return y * t; }
  __device__ void put(int m, int n, int sum, float s) const {
    float y = scaled(sum, s, sw.f()[n]);
    if (bias.ok()) y += bias.f()[n];
    if (res.ok()) y += res.at(m, n);
    out.st((long long)m * out.cols + n, y);
  }
};
// The staged tile [TM][TN] of sums times their rows' scales (16-byte pieces swizzled by row as in gemm_store): a lane has 4 columns, whose scales
// (and bias) it brings; the waves take rows in turn. Without a residual nothing is loaded; with one, those of 8 rows are requested together.
template <int TM, int TN, bool OBF, bool RES> __device__ __forceinline__ void q8_rows_out(const TileQ8& g, const LDS float* et, f32x4n sw, f32x4n bias) {
  constexpr int LPR = TN / 4, RPI = 64 / LPR, NI = TM / KVM_WAVES / RPI, NB = NI < 8 ? NI : 8;
  const int l = lane(), w = wave(), ch = l % LPR, n = g.n0 + 4 * ch;
  const int re = g.res.dtype == 2 ? 2 : 4, left = g.M - g.m0;
  const View ov{(char*)g.out.p + (long long)g.m0 * g.out.cols * (OBF ? 2 : 4), left, g.out.cols, g.out.dtype, 0};
  Ld4 lr;
  if constexpr (RES) lr.init(View{(char*)g.res.p + (long long)g.m0 * g.res.cols * re, g.res.rows - g.m0, g.res.cols, g.res.dtype, 0});
  const __amdgpu_buffer_rsrc_t orsrc = wt_rsrc(ov.p, (long long)min(TM, left) * ov.cols * (OBF ? 2 : 4));
  for (int k0 = 0; k0 < NI; k0 += NB) {
    u32x4_t raw[NB];
    if constexpr (RES)
#pragma unroll
      for (int u = 0; u < NB; ++u) raw[u] = lr.raw(min(((k0 + u) * KVM_WAVES + w) * RPI + l / LPR, left - 1) * g.res.cols + n);
#pragma unroll
    for (int u = 0; u < NB; ++u) {
      const int r = ((k0 + u) * KVM_WAVES + w) * RPI + l / LPR;
      if (r >= left) continue;
      f32x4n y = *(const LDS f32x4n*)(et + r * TN + 4 * (ch ^ epi_swz<TN>(r)));
      y.x *= sw.x; y.y *= sw.y; y.z *= sw.z; y.w *= sw.w;
      if (g.bias.ok()) y += bias;
      if constexpr (RES) y += lr.cvt(raw[u]);
      if constexpr (OBF) stwt_bf4_buf(orsrc, (r * ov.cols + n) * 2, y);
      else stwt_buf(orsrc, (r * ov.cols + n) * 4, y);
    }
  }
}
// Rows of out or res that are no whole vectors, and the last columns of a ragged N: an element at a time, a row's neighbours in neighbouring lanes.
template <int TM, int TN> __device__ __noinline__ void q8_elements_out(const Ctx& c) {
  const TileQ8 g(c);
  const LDS float* et = (const LDS float*)c.smem;
  const int cols = min(TN, g.N - g.n0), rows = min(TM, g.M - g.m0), l = tid() % TN, r1 = KVM_THREADS / TN;
  if (l >= cols) return;
  const int n = g.n0 + l;
  const float sw = g.sw.f()[n], bias = g.bias.ok() ? g.bias.f()[n] : 0.f;
  constexpr int U = 4;
  for (int r0 = tid() / TN; r0 < rows; r0 += U * r1) {
    float x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) x[u] = g.res.ok() ? g.res.at(g.m0 + min(r0 + u * r1, rows - 1), n) : 0.f;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = r0 + u * r1;
      if (r >= rows) break;
      float y = et[r * TN + 4 * ((l >> 2) ^ epi_swz<TN>(r)) + (l & 3)] * sw;
      if (g.bias.ok()) y += bias;
      if (g.res.ok()) y += x[u];
      g.out.st((long long)(g.m0 + r) * g.out.cols + n, y);
    }
  }
}
// The first n bytes of a lane's 16, the others 0.
__device__ __forceinline__ bf16x8 first_bytes(bf16x8 f, int n) {
  u32x4_t x = __builtin_bit_cast(u32x4_t, f);
#pragma unroll
  for (int d = 0; d < 4; ++d) x[d] &= n >= 4 * d + 4 ? 0xffffffffu : n <= 4 * d ? 0u : 0xffffffffu >> (8 * (4 - (n & 3)));
  return __builtin_bit_cast(bf16x8, x);
}
// A tile on the matrix units, v_mfma_i32_32x32x32_i8: a row of bytes moves like a row of half as many bf16 values (DOp: HBM straight into
// LDS, NS stages of 64 bytes a row, fragments of 16 bytes a lane), and the schedule is gemm_lds_b's: fragments of the next half under the products
// of this one, constant waits, the last stage peeled. The sums are exact, so nothing depends on the tile's shape. K's tail is cut off in A
// alone: a byte of B meets a 0. 128 x 256: 0.54 us for 64 bytes of K and 11 us besides (4,001 x 12,288 x 4,096: 1,550 TOPS in the tiles; stages 4 or
// 5 alike); bound by the loads into LDS beside the fragments' reads.
template <int TM, int TN> __device__ __noinline__ void q8_tile(const Ctx& c) {
  constexpr int WM = TM / 2, WN = TN / 2, BM = WM / 32, BN = WN / 32, SA = TM * DK, SB = TN * DK, ST = SA + SB;
  constexpr int NS = KVM_LDS_BYTES / (ST * 2) < 8 ? KVM_LDS_BYTES / (ST * 2) : 8;
  static_assert(NS * ST * 2 <= KVM_LDS_BYTES && TM * TN * 4 <= KVM_LDS_BYTES, "LDS");
  const TileQ8 g(c);
  const View A{g.a.p, g.a.rows, 2 * g.a.cols, 2, 0}, B{g.w.p, g.w.rows, 2 * g.w.cols, 2, 0};
  LDS uint16_t* lds = (LDS uint16_t*)c.smem;
  const int wm0 = (wave() >> 1) * WM, wn0 = (wave() & 1) * WN;
  DOp<TM, true> da;
  DOp<TN, true> db;
  da.init(A, g.m0, g.M);
  db.init(B, g.n0, g.N);
  i32x16_t acc[BM][BN];
#pragma unroll
  for (int i = 0; i < BM; ++i)
#pragma unroll
    for (int j = 0; j < BN; ++j) acc[i][j] = i32x16_t{};
  float sa[BM];                                    // of the rows whose sums the lane gets
#pragma unroll
  for (int i = 0; i < BM; ++i) sa[i] = g.sa.f()[min(g.m0 + wm0 + i * 32 + (lane() & 31), g.M - 1)];
  const int nst = (g.K + 2 * DK - 1) / (2 * DK);
  constexpr int NLA = DOp<TM, true>::NL, NLS = NLA + DOp<TN, true>::NL, NF = BM + BN, NM = BM * BN, PF = (NF + NM - 1) / NM, PX = (NF + NLS + NM - 1) / NM;
  __syncthreads();                                 // the previous task may still read this LDS
  const unsigned lb = (unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)(uintptr_t)lds);
#pragma unroll
  for (int p = 0; p < NS - 1; ++p) { da.issue(lb + p * ST * 2, p, nst); db.issue(lb + (p * ST + SA) * 2, p, nst); }
  bf16x8 fa0[BM], fb0[BN], fa1[BM], fb1[BN];
  auto read_one = [&](const LDS uint16_t* st, int kk, int f, bf16x8 (&fa)[BM], bf16x8 (&fb)[BN]) {
    if (f < BM) fa[f] = da.frag(st, wm0 + f * 32, kk);
    else fb[f - BM] = db.frag(st + SA, wn0 + (f - BM) * 32, kk);
  };
  auto mfma_one = [&](int m, const bf16x8 (&fa)[BM], const bf16x8 (&fb)[BN]) {
    const int i = m / BN, j = m % BN;
    acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(__builtin_bit_cast(i32x4_t, fb[j]), __builtin_bit_cast(i32x4_t, fa[i]), acc[i][j], 0, 0, 0);
  };
  wait_vm_c<(NS - 2) * NLS>();
  __syncthreads();
#pragma unroll
  for (int f = 0; f < NF; ++f) read_one(lds, 0, f, fa0, fb0);
  for (int s = 0; s + 1 < nst; ++s) {
    const LDS uint16_t* la = lds + (s % NS) * ST;
#pragma unroll
    for (int m = 0; m < NM; ++m) {
      mfma_one(m, fa0, fb0);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int f = m * PF; f < (m + 1) * PF && f < NF; ++f) read_one(la, 1, f, fa1, fb1);
      __builtin_amdgcn_sched_barrier(0);
    }
    wait_vm_c<(NS - 3) * NLS>();                 // this thread's loads of stage s + 1 have landed
    asm volatile("s_barrier" ::: "memory");        // ... everyone's, and every wave is past stage s - 1
    const int sn = s + NS - 1;
    const unsigned nb = lb + ((s + NS - 1) % NS) * ST * 2;
    const LDS uint16_t* ln = lds + ((s + 1) % NS) * ST;
#pragma unroll
    for (int m = 0; m < NM; ++m) {
      mfma_one(m, fa1, fb1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int x = m * PX; x < (m + 1) * PX && x < NF + NLS; ++x) {
        if (x < NF) read_one(ln, 0, x, fa0, fb0);
        else if (x - NF < NLA) da.issue_one(nb, sn, x - NF, nst);
        else db.issue_one(nb + SA * 2, sn, x - NF - NLA, nst);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  {
    const LDS uint16_t* la = lds + ((nst - 1) % NS) * ST;
#pragma unroll
    for (int f = 0; f < NF; ++f) read_one(la, 1, f, fa1, fb1);
    const int kr = g.K - (nst - 1) * 2 * DK;       // bytes of the last stage
    if (kr < 2 * DK) {
      const int k0 = kr - 16 * (lane() >> 5);
#pragma unroll
      for (int i = 0; i < BM; ++i) { fa0[i] = first_bytes(fa0[i], k0); fa1[i] = first_bytes(fa1[i], k0 - 32); }
    }
#pragma unroll
    for (int m = 0; m < NM; ++m) mfma_one(m, fa0, fb0);
#pragma unroll
    for (int m = 0; m < NM; ++m) mfma_one(m, fa1, fb1);
  }
  const int l = lane(), n = g.n0 + 4 * (l % (TN / 4));
  const bool vec = g.n0 + TN <= g.N && (g.out.cols & 3) == 0 && vec_base(g.out) && (!g.res.ok() || ((g.res.cols & 3) == 0 && vec_base(g.res))) &&
                   (long long)TM * max(g.res.cols, g.out.cols) * 4 < 0x7fffffffll;
  f32x4n sw = {0.f, 0.f, 0.f, 0.f}, bias = sw;
  if (vec)
#pragma unroll
    for (int i = 0; i < 4; ++i) { sw[i] = g.sw.f()[n + i]; if (g.bias.ok()) bias[i] = g.bias.f()[n + i]; }
  wait_vm_c<0>();                                  // the placeholder loads have written their LDS bytes
  __syncthreads();
  LDS float* et = (LDS float*)c.smem;              // D^T: lane has row l % 32 of block i, columns 8 q + 4 (l / 32) .. + 3 of block j
#pragma unroll
  for (int i = 0; i < BM; ++i) {
    const int r = wm0 + i * 32 + (l & 31);
#pragma unroll
    for (int j = 0; j < BN; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int chunk = (wn0 + j * 32 + 8 * q) / 4 + (l >> 5);
        *(LDS f32x4n*)(et + r * TN + 4 * (chunk ^ epi_swz<TN>(r))) = f32x4n{(float)acc[i][j][4 * q] * sa[i], (float)acc[i][j][4 * q + 1] * sa[i], (float)acc[i][j][4 * q + 2] * sa[i],
                                                                          (float)acc[i][j][4 * q + 3] * sa[i]};
      }
  }
  __syncthreads();
  if (!vec) q8_elements_out<TM, TN>(c);
  else if (g.out.dtype == 2) { if (g.res.ok()) q8_rows_out<TM, TN, true, true>(g, et, sw, bias); else q8_rows_out<TM, TN, true, false>(g, et, sw, bias); }
  else if (g.res.ok()) q8_rows_out<TM, TN, false, true>(g, et, sw, bias);
  else q8_rows_out<TM, TN, false, false>(g, et, sw, bias);
}
// Rows of bytes that do not lie in whole 16-byte vectors: an output at a time, four products an instruction.
__device__ __forceinline__ int q8_dot(const GLOBAL int* a, const GLOBAL int* w, int K) {
  int s = 0;
  for (int k = 0; k < K >> 2; ++k) s = __builtin_amdgcn_sdot4(a[k], w[k], s, false);
  if (K & 3) s = __builtin_amdgcn_sdot4((int)((uint32_t)a[K >> 2] & (0xffffffffu >> (8 * (4 - (K & 3))))), w[K >> 2], s, false);
  return s;
}
__device__ __noinline__ void matmul_q8_simt(const Ctx& c, int tm, int tn) {
  const TileQ8 g(c);
  const int rows = min(rfl(tm), g.M - g.m0), cols = min(rfl(tn), g.N - g.n0);
  for (int e = tid(); e < rows * cols; e += KVM_THREADS) {
    const int m = g.m0 + e / cols, n = g.n0 + e % cols;
    g.put(m, n, q8_dot(g.a.i() + (long long)m * g.a.cols, g.w.i() + (long long)n * g.w.cols, g.K), g.sa.f()[m]);
  }
}
// Whether rows r0 .. of X lie in whole vectors that a descriptor from row r0 on reaches in 31 bits.
__device__ __forceinline__ bool q8_fast(const View& X, int R, int K) {
  return (X.cols & 3) == 0 && vec_base(X) && (long long)R * X.cols * 4 + K < 0x7fffff00ll;
}
__device__ __noinline__ void op_matmul_q8(const Ctx& c) {
  const int tile = rfl(c.i(12)), tm = tile == 2 ? 64 : 128, tn = tile == 0 ? 256 : tile == 1 ? 128 : 64;
  if (!q8_fast(c.buf(0), tm, c.i(11)) || !q8_fast(c.buf(2), tn, c.i(11))) matmul_q8_simt(c, tm, tn);
  else if (tile == 0) q8_tile<128, 256>(c);
  else if (tile == 1) q8_tile<128, 128>(c);
  else q8_tile<64, 64>(c);
}

// ---------------------------------------------------------------------------------------------- rows of weights, streamed
// Op 317. Bound: the weights' bytes (N * K), as the bf16 stream of ops 134 and 301, whose ring and cursor it uses (a row of bytes is a row of
// half as many bf16 values); K is rounded up to whole steps of all waves, the bytes behind K are 0 in the staged rows. A step of a wave is two
// v_mfma_i32_16x16x64_i8. A call: 12,288 x 4,096 for one row with the norm 38 us, of which the weights' 50 MB take ~15, launch ~13 and the row's
// norm and rounding inside every task ~6; 4,096 x 12,288 for 8 rows behind rows_q8 50.
struct GemvQ8 {
  View x, x2, g, w, sw, out, bias, res, sx; int n0, n1, K, M, pro, Ke;
  __device__ explicit GemvQ8(const Ctx& c)
      : x(uview(c, 0)), x2(uview(c, 1)), g(uview(c, 2)), w(uview(c, 3)), sw(uview(c, 4)), out(uview(c, 5)), bias(uview(c, 6)), res(uview(c, 7)), sx(uview(c, 8)),
        n0(rfl(c.i(9))), n1(rfl(c.i(10))), K(rfl(c.i(11))), M(rfl(c.i(12))), pro(rfl(c.i(13))) { Ke = ((K + 511) >> 9) << 8; }
  __device__ View stream() const { return View{w.p, w.rows, 2 * w.cols, 2, 0}; }
  __device__ bool fast() const { return q8_fast(w, n1 - n0 + 16, 4 * Ke); }   // (all parts of K are less than twice as long)
  __device__ void put(int m, int n, int sum, float s) const {
    float y = (float)sum * s;
    y *= sw.f()[n];
    if (bias.ok()) y += bias.f()[n];
    if (res.ok()) y += res.at(m, n);
    out.st((long long)m * out.cols + n, y);
  }
};
// Where byte o (a multiple of 4) of row m's staged range lies: its 16-byte pieces swizzled by row, so that 16 rows' reads of one piece touch every
// bank once without padding between the rows, which direct loads could not leave.
__device__ __forceinline__ int gq_at(int m, int pitch, int o) { return m * pitch + (o ^ (m << 4)); }
// Row m's bytes [lo, lo + n) (n a multiple of 256, zeros behind K) to LDS and the scales, for all rows.
template <int FORM, int NV> __device__ __noinline__ void gemv_q8_stage(const Ctx& c, LDS char* vs_, int pitch_, int lo_, int n_, LDS float* scale, LDS double* red) {
  const int pitch = rfl(pitch_), lo = rfl(lo_), n = rfl(n_);
  const GemvQ8 G(c);
  const RowsSrc S{G.x, G.x2, G.g, G.K, G.pro, c.f(14)};
  RowsRaw<FORM, NV ? NV : 1, 1> raw;
  if (NV > 0) raw.load(S, 0, 1, tid());
  for (int m = 0; m < G.M; ++m) {
    auto next = [&]() { if (m + 1 < G.M) raw.load(S, m + 1, 1, tid()); };
    auto put = [&](int, int j, uint32_t w0, uint32_t w1) {
      const int o = 8 * j - lo;
      if (o >= 0 && o < n) { *(LDS uint32_t*)(vs_ + gq_at(m, pitch, o)) = w0; *(LDS uint32_t*)(vs_ + gq_at(m, pitch, o + 4)) = w1; }
    };
    auto scaled = [&](int, float s) { scale[m] = s; };
    if constexpr (NV > 0) q8_rows<FORM, NV, 1>(S, raw, m, 1, red, put, scaled, next);
    else q8_row_long<FORM>(S, m, red, put, scaled);
    for (int o = max(0, ((G.K + 7) & ~7) - lo) + 4 * tid(); o < n; o += 4 * KVM_THREADS) *(LDS int*)(vs_ + gq_at(m, pitch, o)) = 0;
  }
}
__device__ __forceinline__ void gemv_q8_rows(const Ctx& c, const GemvQ8& G, LDS char* vs, int pitch, int lo, int n, LDS float* scale, LDS double* red) {
  if (G.pro == 3) {                                // bytes that are there already
    if (q8_fast(G.x, G.M, lo + n) && pitch == n) { // direct loads, 1 KiB a wave; what lies behind K is cleared once they have landed
      const i32x4_t rs = dma_rsrc(G.x.p, (long long)G.x.rows * G.x.cols * 4);
      for (int b = wave(); b < G.M * n / 1024; b += KVM_WAVES) {
        const int o = 1024 * b + 16 * lane(), m = o / pitch;
        dma16(rs, m * G.x.cols * 4 + lo + ((o - m * pitch) ^ (m << 4)), 0, vs + 1024 * b);
      }
      for (int o = (G.M * n & ~1023) + 4 * tid(); o < G.M * n; o += 4 * KVM_THREADS) {   // half a block may be left
        const int m = o / pitch, k = lo + ((o - m * pitch) ^ (m << 4));
        *(LDS int*)(vs + o) = k < G.K ? G.x.i()[(long long)m * G.x.cols + (k >> 2)] : 0;
      }
      wait_vm_c<0>();
      __syncthreads();
      const int k0 = max(0, (G.K - lo) & ~3);
      for (int m = 0; m < G.M; ++m)
        for (int o = k0 + 4 * tid(); o < n; o += 4 * KVM_THREADS) {
          LDS int* y = (LDS int*)(vs + gq_at(m, pitch, o));
          *y = G.K - lo - o > 0 ? *y & (int)(0xffffffffu >> (8 * (4 - (G.K - lo - o)))) : 0;
        }
    } else {
      for (int m = 0; m < G.M; ++m)
        for (int o = 4 * tid(); o < n; o += 4 * KVM_THREADS) {
          const int k = lo + o;
          int v = k < G.K ? G.x.i()[(long long)m * G.x.cols + (k >> 2)] : 0;
          if (G.K - k < 4 && k < G.K) v &= (int)(0xffffffffu >> (8 * (4 - (G.K - k))));
          *(LDS int*)(vs + gq_at(m, pitch, o)) = v;
        }
    }
    if (tid() < G.M) scale[tid()] = G.sx.f()[tid()];
    return;
  }
  const RowsSrc S{G.x, G.x2, G.g, G.K, G.pro, 0.f};
  const int form = rfl(S.form());
#define KVM_STAGE(F, N) gemv_q8_stage<F, N>(c, vs, pitch, lo, n, scale, red)
  if (G.K <= 4096) { if (form == 1) KVM_STAGE(1, 2); else if (form == 2) KVM_STAGE(2, 2); else if (form == 3) KVM_STAGE(3, 2); else KVM_STAGE(0, 0); }
  else if (G.K <= 16384 && form) { if (form == 1) KVM_STAGE(1, 8); else if (form == 2) KVM_STAGE(2, 8); else KVM_STAGE(3, 8); }
  else if (form == 1) KVM_STAGE(1, 0);
  else if (form >= 2) KVM_STAGE(3, 0);
  else KVM_STAGE(0, 0);
#undef KVM_STAGE
}
// LDS of one call with a ring of R steps a wave: [ring][rows: M x 2 KC bytes][scales][reductions][sums: 4 x blocks x M x 16], blocks the 16-output
// blocks of the task, at most GV_GRP. KC (pairs of bytes): a part of K in whole steps of all waves, K all parts of it together.
struct GqGeo { int K, KC, pitch, vs, scale, red, part, grp; };
__device__ __forceinline__ GqGeo gq_geo(int Ke, int M, int R, int n) {
  GqGeo g;
  g.grp = min((n + 15) >> 4, GV_GRP);
  const int rest = R * KVM_WAVES * GV_STEP + 64 + Q8_RED * 8 + KVM_WAVES * g.grp * M * 16 * 4;
  g.KC = gq_part_steps(Ke >> 8, M * 512, KVM_LDS_BYTES - rest) << 8;
  g.K = (Ke + g.KC - 1) / g.KC * g.KC; g.pitch = 2 * g.KC;
  g.vs = R * KVM_WAVES * GV_STEP;
  g.scale = g.vs + M * g.pitch;
  g.red = g.scale + 64;
  g.part = g.red + Q8_RED * 8;
  return g;
}
static_assert(4 * KVM_WAVES * GV_STEP + 64 + Q8_RED * 8 + KVM_WAVES * GV_GRP * 16 * 16 * 4 + 16 * 512 <= KVM_LDS_BYTES, "LDS");
static_assert(12 * KVM_WAVES * GV_STEP + 64 + Q8_RED * 8 + KVM_WAVES * GV_GRP * 4 * 16 * 4 + 4 * 512 <= KVM_LDS_BYTES, "LDS");
template <int R> __device__ __forceinline__ void gemv_q8_prefetch_r(const GemvQ8& G, LDS char* smem) {
  GvStream<> ws;
  const GqGeo geo = gq_geo(G.Ke, G.M, R, G.n1 - G.n0);
  ws.init(G.stream(), G.n0, G.n1, geo.K, geo.KC);
  LDS char* ring = smem + wave() * R * GV_STEP;
#pragma unroll
  for (int j = 0; j < R; ++j) ws.template issue<R>(ring);
}
__device__ __noinline__ void gemv_q8_prefetch(const Ctx& c) {
  const GemvQ8 G(c);
  if (!G.fast()) return;
  if (gv_pre_ring(G.M) == 12) gemv_q8_prefetch_r<12>(G, c.smem);
  else gemv_q8_prefetch_r<4>(G, c.smem);
}
template <int R> __device__ __noinline__ void gemv_q8_stream(const Ctx& c) {
  const GemvQ8 G(c);
  const int M = G.M, PM = 16 * M;
  const GqGeo geo = gq_geo(G.Ke, M, R, G.n1 - G.n0);
  const int K = geo.K, KC = geo.KC;                                             // in pairs of bytes
  LDS char* vs = c.smem + geo.vs;
  LDS float* scale = (LDS float*)(c.smem + geo.scale);
  LDS int* part = (LDS int*)(c.smem + geo.part);
  const int l = lane(), wv = wave(), nrb = (G.n1 - G.n0 + 15) / 16;
  LDS char* ring = c.smem + wv * R * GV_STEP;
  GvStream<> ws;
  ws.init(G.stream(), G.n0, G.n1, K, KC);
  if (rfl(c.pre)) {
#pragma unroll
    for (int j = 0; j < R; ++j) ws.template skip<R>();                           // issued before the dependency wait
  } else {
#pragma unroll
    for (int j = 0; j < R; ++j) ws.template issue<R>(ring);
  }
  const bool arow = (l & 15) < M;
  const int vm = arow ? l & 15 : 0, vx = vm << 4;
  const LDS char* va = vs + vm * geo.pitch;
  const LDS char* rl = ring + 16 * l;
  int cslot = 0;
  for (int g0 = 0; g0 < nrb; g0 += GV_GRP) {
    const int ng = min(GV_GRP, nrb - g0);
    for (int e = l; e < ng * PM; e += 64) part[wv * geo.grp * PM + e] = 0;
    for (int kc = 0; kc < K; kc += KC) {
      const int kq = KC / 2, ns = KC / 256;                                      // bytes of a wave's quarter, its steps
      __syncthreads();
      if (KC != K || g0 == 0) gemv_q8_rows(c, G, vs, geo.pitch, 2 * kc, 2 * KC, scale, (LDS double*)(c.smem + geo.red));
      __syncthreads();
      const int vk = wv * kq + 16 * (l >> 4);
      i32x4_t acc = {0, 0, 0, 0};
      int rb = 0, st = 0;
      for (int tt = 0; tt < ng * ns; ++tt) {                                     // one flat loop: no full wait at an inner loop's head
        wait_vm_c<2 * (R - 1)>();
        const LDS char* slot = rl + cslot * GV_STEP;
        const i32x4_t w0 = *(const LDS i32x4_t*)slot, w1 = *(const LDS i32x4_t*)(slot + 1024);
        const i32x4_t a0 = *(const LDS i32x4_t*)(va + ((vk + st * 128) ^ vx)), a1 = *(const LDS i32x4_t*)(va + ((vk + st * 128 + 64) ^ vx));
        acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(arow ? a0 : i32x4_t{}, w0, acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(arow ? a1 : i32x4_t{}, w1, acc, 0, 0, 0);
        wait_lds();
        ws.template issue<R>(ring);
        cslot = cslot + 1 == R ? 0 : cslot + 1;
        if (++st == ns) {                                                        // D[m][n]: lane holds m = 4 (l / 16) + i, n = l % 16
          LDS int* pp = part + (wv * geo.grp + rb) * PM + (l & 15);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int m = 4 * (l >> 4) + i;
            if (m < M) pp[m * 16] += acc[i];
          }
          acc = i32x4_t{0, 0, 0, 0};
          st = 0; ++rb;
        }
      }
    }
    __syncthreads();
    for (int e = tid(); e < ng * PM; e += KVM_THREADS) {
      const int rb = e / PM, m = (e / 16) % M, n = G.n0 + (g0 + rb) * 16 + e % 16;
      if (n < G.n1) G.put(m, n, part[e] + part[geo.grp * PM + e] + part[2 * geo.grp * PM + e] + part[3 * geo.grp * PM + e], scale[m]);
    }
    __syncthreads();                                                            // read before the next group clears them
  }
  wait_vm_c<0>();                                                               // the ring's trailing loads have landed
}
// Weights that do not lie in whole 16-byte vectors: rows in LDS 4,096 bytes at a time, an output to a thread.
__device__ __noinline__ void gemv_q8_simt(const Ctx& c) {
  const GemvQ8 G(c);
  constexpr int CH = 4096;
  LDS char* vs = c.smem;                                                        // [16][CH]
  LDS float* scale = (LDS float*)(vs + 16 * CH);
  LDS double* red = (LDS double*)(scale + 16);
  for (int e0 = 0; e0 < (G.n1 - G.n0) * G.M; e0 += KVM_THREADS) {
    const int e = e0 + tid(), m = e % G.M, n = G.n0 + e / G.M;
    int s = 0;
    for (int k0 = 0; k0 < G.K; k0 += CH) {
      __syncthreads();
      gemv_q8_rows(c, G, vs, CH, k0, CH, scale, red);
      __syncthreads();
      const int nw = (min(CH, G.K - k0) + 3) >> 2;
      if (n < G.n1)
        for (int k = 0; k < nw; ++k) s = __builtin_amdgcn_sdot4(*(const LDS int*)(vs + gq_at(m, CH, 4 * k)), G.w.i()[(long long)n * G.w.cols + (k0 >> 2) + k], s, false);
    }
    if (n < G.n1) G.put(m, n, s, scale[m]);
  }
}
__device__ __noinline__ void op_gemv_q8(const Ctx& c) {
  const GemvQ8 G(c);
  if (G.n0 >= G.n1) return;
  if (!G.fast()) gemv_q8_simt(c);
  else if (rfl(c.pre) && gv_pre_ring(G.M) == 12) gemv_q8_stream<12>(c);
  else gemv_q8_stream<4>(c);
}

}  // namespace kvm
