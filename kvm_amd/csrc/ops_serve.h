// Serving operators of a decode step: a key / value cache held in 8 bits (ops 312, 313) and the adjustment of logits before
// a token is chosen (op 314). Semantics: mvm_ops_kvm.def.
#pragma once
#include "common.h"
#include "ops_basic.h"
#include "ops_attn.h"
#include "ops_stream.h"

namespace kvm {

// ---------------------------------------------------------------------------------------------- 8-bit KV cache
// Rotation of position t by frequency i: theta^(-2 i / hd) and the angle in double (at positions of 10^5 an f32 angle is off
// by up to 4e-3), there reduced to a quarter turn around 0; sine and cosine by their Taylor series in f32, whose next terms are
// below 2e-9 at pi / 4. (The library's sincosf, with its path for large arguments, is ten times the code.)
__device__ __forceinline__ double q8_freq(int i, int hd, double ln_theta) { return exp(-2.0 * i / hd * ln_theta); }
__device__ __forceinline__ void q8_turn(long long t, double freq, float& sn, float& co) {
  const double turns = (double)t * freq * 0.15915494309189533577, quarter = rint(4.0 * turns);      // 1 / (2 pi)
  const float x = (float)((turns - 0.25 * quarter) * 6.28318530717958647693), y = x * x;
  const float s = x + x * y * (-1.f / 6 + y * (1.f / 120 + y * (-1.f / 5040 + y * (1.f / 362880))));
  const float c = 1.f + y * (-1.f / 2 + y * (1.f / 24 + y * (-1.f / 720 + y * (1.f / 40320 + y * (-1.f / 3628800)))));
  const int k = (int)((long long)quarter & 3);
  sn = k & 1 ? c : s; co = k & 1 ? s : c;
  if (k & 2) sn = -sn;
  if (k == 1 || k == 2) co = -co;
}
// The 8-bit number of x in a block of scale s: x / s rounded to the nearest whole number, ties to even, with no
// error from the reciprocal: one fused multiply-add gives the sign of (k + 1/2) s - |x| exactly. `inv` is 1 / s, 0 where s is 0.
__device__ __forceinline__ int q8_of(float x, float s, float inv) {
  const float a = fabsf(x), k = floorf(a * inv), d = fmaf(k + 0.5f, s, -a);
  int q = (int)k;
  if (d < 0.f || (d == 0.f && (q & 1))) ++q;
  q = s > 0.f ? min(q, 127) : 0;                                       // a NaN scale stands for itself: its bytes are 0
  return x < 0.f ? -q : q;
}
// The scale of a block from its largest magnitude (infinity for a block with a value that is not finite), times 1 / 127 as f32 has it:
// NaN for such a block, 0 where it falls below the normal numbers.
__device__ __forceinline__ float q8_scale(float amax) {
  const float s = amax * (1.f / 127.f);
  return !(amax < INFINITY) ? __uint_as_float(0x7fc00000u) : s < 1.17549435e-38f ? 0.f : s;
}
// Largest magnitude so far; a value that is not finite makes it infinity, for good.
__device__ __forceinline__ float q8_amax(float amax, float x) { return fabsf(x) < INFINITY ? fmaxf(amax, fabsf(x)) : INFINITY; }

typedef u32x4_t u32x4a4 __attribute__((aligned(4)));                   // 16 and 8 bytes at any element of a 4-byte buffer
typedef u32x2_t u32x2a4 __attribute__((aligned(4)));
// Whether rows of X can be read and written in vectors of 8 elements at columns that are multiples of 8.
__device__ __forceinline__ bool rows8_ok(const View& X) { return ((uintptr_t)X.p & 15) == 0 && (X.cols & 7) == 0; }
// Eight values as they lie in memory (bf16: the first half), so that a batch of loads is requested before any is converted.
struct Raw8 {
  u32x4_t lo, hi;
  __device__ __forceinline__ void load(const View& X, long long o) {
    if (X.dtype == 2) lo = *(const GLOBAL u32x4_t*)(X.h() + o);
    else { lo = *(const GLOBAL u32x4_t*)(X.f() + o); hi = *(const GLOBAL u32x4_t*)(X.f() + o + 4); }
  }
  __device__ __forceinline__ void get(bool half, float (&v)[8]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = __uint_as_float(!half ? lo[i] : i & 1 ? lo[i / 2] & 0xffff0000u : lo[i / 2] << 16);
      v[4 + i] = __uint_as_float(!half ? hi[i] : i & 1 ? lo[2 + i / 2] & 0xffff0000u : lo[2 + i / 2] << 16);
    }
  }
};
template <int CTRL> __device__ __forceinline__ float dpp(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
// Reduction over N = 8 or 16 neighbouring lanes, in registers: neighbours, pairs, then the mirrored half row and row.
template <int N, class F> __device__ __forceinline__ float lanes_all(float v, F f) {
  v = f(v, dpp<0xB1>(v));
  v = f(v, dpp<0x4E>(v));
  v = f(v, dpp<0x141>(v));
  return N == 16 ? f(v, dpp<0x140>(v)) : v;
}
template <int N> __device__ __forceinline__ float lanes_sum(float v) { return lanes_all<N>(v, [](float a, float b) { return a + b; }); }
template <int N> __device__ __forceinline__ float lanes_max(float v) { return lanes_all<N>(v, [](float a, float b) { return fmaxf(a, b); }); }
// Over the four rows of 16 lanes of a wave: lane n of each gets f over lanes n, n + 16, n + 32, n + 48.
template <class F> __device__ __forceinline__ float rows_all(float v, F f) {
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = f(__uint_as_float(a[0]), __uint_as_float(a[1]));
  auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return f(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float rows_sum(float v) { return rows_all(v, [](float a, float b) { return a + b; }); }
__device__ __forceinline__ float rows_max(float v) { return rows_all(v, [](float a, float b) { return fmaxf(a, b); }); }
// A head of HD values spread over HD / 8 neighbouring lanes, 8 each: RMS norm (gamma: the gains, or none) and rotation of
// position t (freq: the HD / 2 frequencies in LDS, or none), in f32. The other half of a pair is HD / 16 lanes away; the lanes
// share out the row's angles through `ang`, HD floats of LDS for each row in flight (HD / 8 lanes of one wave).
template <int HD> __device__ __forceinline__ void head8_turn(float (&v)[8], const GLOBAL float* gamma, float eps, const LDS double* freq, long long t, LDS float* ang) {
  constexpr int LPR = HD / 8;
  const int ln = lane() % LPR;
  if (freq) {
#pragma unroll 1
    for (int i = ln; i < HD / 2; i += LPR) { float sn, co; q8_turn(t, freq[i], sn, co); ang[i] = sn; ang[HD / 2 + i] = co; }
    __builtin_amdgcn_wave_barrier();                                   // one wave's LDS operations stay in order
  }
  if (gamma) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss += v[i] * v[i];
    const float rs = 1.f / sqrtf(lanes_sum<LPR>(ss) / HD + eps);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = v[i] * rs * gamma[8 * ln + i];
  }
  if (freq) {
    const float sign = ln >= LPR / 2 ? 1.f : -1.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int k = 8 * (ln % (LPR / 2)) + i;
      v[i] = v[i] * ang[HD / 2 + k] + sign * __shfl_xor(v[i], LPR / 2, 64) * ang[k];
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// Arguments of op 312 as every form reads them; Tmax = blk * ks.cols.
struct AppendQ8 {
  View kn, vn, kq, ks, vq, vs, kt, vt, lens, kg;
  int b0, b1, h0, h1, p, P, n, Hkv, hd, blk, nblk;
  float theta, eps;
  __device__ explicit AppendQ8(const Ctx& c)
      : kn(c.buf(0)), vn(c.buf(1)), kq(c.buf(2)), ks(c.buf(3)), vq(c.buf(4)), vs(c.buf(5)), kt(c.buf(6)), vt(c.buf(7)), lens(c.buf(8)), kg(c.buf(9)),
        b0(c.i(10)), b1(c.i(11)), h0(c.i(12)), h1(c.i(13)), p(c.i(14)), P(c.i(15)), n(c.i(16)), Hkv(c.i(17)), hd(c.i(18)), blk(c.i(19)),
        nblk(ks.cols), theta(c.f(20)), eps(c.f(21)) {}
  // The lengths of the task's sequences are all checked before anything is written.
  __device__ bool lengths_ok(const Ctx& c) const {
    bool bad = false;
    for (int b = b0 + tid(); b < b1; b += KVM_THREADS) {
      const int L = lens.i()[b];
      if (L < -1 || (long long)L + n > (long long)blk * nblk) { bad = true; c.fail(KVM_ERR_OP_KVLEN, b, L); }
    }
    return !__syncthreads_or(bad);
  }
  // Whether a block becomes full in this task's share.
  __device__ bool finishes() const {
    bool any = false;
    for (int b = b0 + tid(); b < b1; b += KVM_THREADS) { const int L = lens.i()[b]; any = any || (L >= 0 && (L + n) / blk > L / blk); }
    return __syncthreads_or(any);
  }
};

// One row of new keys, element by element: head norm and rotation in f32 (row in LDS, hd values), rounded to the tail's type.
__device__ __forceinline__ void q8_new_key(const AppendQ8& A, LDS float* x, long long row, int h, long long t, LDS float* red) {
  for (int k = tid(); k < A.hd; k += KVM_THREADS) x[k] = A.kn.at(row, h * A.hd + k);
  __syncthreads();
  if (A.kg.ok()) {
    float ss = 0.f;
    for (int k = tid(); k < A.hd; k += KVM_THREADS) ss += x[k] * x[k];
    const float rs = 1.f / sqrtf(block_sum(ss, red) / A.hd + A.eps);
    for (int k = tid(); k < A.hd; k += KVM_THREADS) x[k] = x[k] * rs * A.kg.f()[k];
    __syncthreads();
  }
  if (A.theta > 0.f) {
    const int half = A.hd / 2;
    for (int i = tid(); i < half; i += KVM_THREADS) {
      float sn, co; q8_turn(t, q8_freq(i, A.hd, log((double)A.theta)), sn, co);
      const float x1 = x[i], x2 = x[i + half];
      x[i] = x1 * co - x2 * sn; x[i + half] = x1 * sn + x2 * co;
    }
    __syncthreads();
  }
}

// KV append in 8 bits, any alignment and head size: token by token into an f32 copy of the block in LDS, which is quantised
// when it is full and stored to the tail otherwise.
__device__ __noinline__ void op_kv_append_q8(const Ctx& c) {
  const AppendQ8 A(c);
  if (!A.lengths_ok(c)) return;
  LDS float* x = (LDS float*)c.smem;                                   // [blk][hd], one of K and V at a time
  LDS float* red = x + 128 * 128;
  LDS float* row = red + 16;
  for (int b = A.b0; b < A.b1; ++b) {
    const int L = A.lens.i()[b];
    if (L < 0) continue;
    const int j0 = L / A.blk, jE = (L + A.n) / A.blk;                  // touched blocks j0 .. jE, the last one unfinished
    const int mid = max(0, jE - j0 - 1), m0 = (int)((long long)mid * A.p / A.P), m1 = (int)((long long)mid * (A.p + 1) / A.P);
    for (int h = A.h0; h < A.h1; ++h) {
      const long long pair = (long long)b * A.Hkv + h;
      for (int which = 0; which < 2; ++which) {
        const View& src = which ? A.vn : A.kn; const View& tail = which ? A.vt : A.kt;
        const View& Q = which ? A.vq : A.kq; const View& SC = which ? A.vs : A.ks;
        // part 0: the first block (it may hold older tokens), then the unfinished one (its rows in the tail are read before
        // they are overwritten); the blocks between are shared out
        for (int u = A.p == 0 ? -1 : 0; u <= m1 - m0; ++u) {
          if (u == m1 - m0 && A.p != 0) break;
          const int j = u < 0 ? j0 : u < m1 - m0 ? j0 + 1 + m0 + u : jE;
          const bool full = j < jE;
          if (u < 0 && !full) continue;                                // nothing finishes: the unfinished block only
          const long long t0 = (long long)j * A.blk;
          const int r0 = full ? 0 : (int)(max((long long)L, t0) - t0), r1 = full ? A.blk : (int)(L + A.n - t0);
          float amax = 0.f;
          __syncthreads();
          for (int r = r0; r < r1; ++r) {
            const long long t = t0 + r;
            if (t < L) for (int k = tid(); k < A.hd; k += KVM_THREADS) row[k] = tail.at(pair * A.blk + r, k);
            else if (which == 0) q8_new_key(A, row, (long long)b * A.n + (t - L), h, t, red);
            else for (int k = tid(); k < A.hd; k += KVM_THREADS) row[k] = src.at((long long)b * A.n + (t - L), h * A.hd + k);
            for (int k = tid(); k < A.hd; k += KVM_THREADS) {
              const float v = tail.dtype == 2 ? round_bf(row[k]) : row[k];
              if (full) { x[r * A.hd + k] = v; amax = q8_amax(amax, v); }
              else tail.st((pair * A.blk + r) * tail.cols + k, v);
            }
            __syncthreads();
          }
          if (!full) continue;
          const float s = q8_scale(block_max(amax, red)), inv = s > 0.f ? 1.f / s : 0.f;
          if (tid() == 0) stwt32(SC.f() + (pair * SC.cols + j), s);
          const long long w0 = (pair * A.nblk + j) * A.blk * (A.hd / 4);
          for (int e = tid(); e < A.blk * A.hd / 4; e += KVM_THREADS) {
            int w = 0;
            for (int i = 0; i < 4; ++i) {
              const int o = 4 * e + i;                                 // byte of the block: [blk][hd] of keys, [hd][blk] of values
              w |= (q8_of(x[which ? (o % A.blk) * A.hd + o / A.blk : o], s, inv) & 255) << (8 * i);
            }
            stwt32i(Q.i() + (w0 + e), w);
          }
        }
      }
    }
  }
}

// KV append in 8 bits at head sizes 64 and 128, rows in whole vectors. Bound: a few dependent loads (length, row) and the launch
// for single tokens, bytes for prompts. A row is HD / 8 lanes of 8 values, so a pass of the workgroup takes 16 or 32 rows.
// The tail rows of all pairs of the task go in one range, a row to HD / 8 lanes; blocks that become full (of single tokens one call in
// blk) are a function of their own, whose registers the tail rows' callers need not save.
// A full block is in registers as a whole, all its loads requested before any is used, K and V with one reduction of both maxima.
// Keys to be normalised or rotated
// go through LDS first, row by row. Keys are stored as they lie, 8 bytes a lane; values turn through LDS.
template <int HD> struct AppendLds {
  LDS double* freq; LDS float* red; LDS float* keys; LDS float* angs; LDS unsigned char* turn;
  __device__ explicit AppendLds(LDS char* p)
      : freq((LDS double*)p), red((LDS float*)(freq + HD / 2)), keys(red + 16), angs(keys + 128 * HD), turn((LDS unsigned char*)(angs + KVM_THREADS * 8)) {}
};
template <int HD, int NP> __device__ __noinline__ void append_q8_blocks(const Ctx& c) {
  constexpr int LPR = HD / 8, RPP = KVM_THREADS / LPR;                 // lanes a row, rows a pass; NP passes hold a block
  const AppendQ8 A(c);
  const AppendLds<HD> M(c.smem);                                       // keys [blk][HD], turn [HD][blk + 4]
  const int ln = tid() % LPR, rw = tid() / LPR, blk = A.blk;
  const GLOBAL float* gamma = A.kg.ok() ? A.kg.f() : nullptr;
  const LDS double* rot = A.theta > 0.f ? M.freq : nullptr;
  const bool turned = gamma || rot, nkh = A.kn.dtype == 2, nvh = A.vn.dtype == 2, tkh = A.kt.dtype == 2, tvh = A.vt.dtype == 2;
  const int nh = A.h1 - A.h0;
  for (int u = 0; u < (A.b1 - A.b0) * nh; ++u) {
    const int b = A.b0 + u / nh, h = A.h0 + u % nh, L = rfl(A.lens.i()[b]);
    if (L < 0) continue;
    const long long pair = (long long)b * A.Hkv + h;
    const int j0 = L / blk, jE = (L + A.n) / blk, mid = max(0, jE - j0 - 1);
    const int m0 = (int)((long long)mid * A.p / A.P), m1 = (int)((long long)mid * (A.p + 1) / A.P);
    for (int it = A.p == 0 && jE > j0 ? m0 - 1 : m0; it < m1; ++it) {  // (p = 0: m0 = 0, and -1 is the first block)
      const int j = j0 + 1 + it, old = max(0, L - j * blk);            // rows below `old` are in the tail
      const long long new0 = (long long)b * A.n + ((long long)j * blk - L), tail0 = pair * blk;
      if (turned) {
        __syncthreads();
#pragma unroll 1
        for (int r = rw; r < blk; r += RPP) {
          float x[8];
          Raw8 w;
          if (r >= old) {
            w.load(A.kn, (new0 + r) * A.kn.cols + h * HD + 8 * ln); w.get(nkh, x);
            head8_turn<HD>(x, gamma, A.eps, rot, (long long)j * blk + r, M.angs + rw * HD);
          } else { w.load(A.kt, (tail0 + r) * A.kt.cols + 8 * ln); w.get(tkh, x); }
#pragma unroll
          for (int e = 0; e < 8; ++e) M.keys[r * HD + 8 * ln + e] = x[e];
        }
      }
      Raw8 rk[NP], rv[NP];
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const int r = i * RPP + rw;
        if (r >= blk) break;
        const bool in_tail = r < old;
        if (!turned) rk[i].load(in_tail ? A.kt : A.kn, in_tail ? (tail0 + r) * A.kt.cols + 8 * ln : (new0 + r) * A.kn.cols + h * HD + 8 * ln);
        rv[i].load(in_tail ? A.vt : A.vn, in_tail ? (tail0 + r) * A.vt.cols + 8 * ln : (new0 + r) * A.vn.cols + h * HD + 8 * ln);
      }
      float k[NP][8], v[NP][8], ka = 0.f, va = 0.f;
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const int r = i * RPP + rw;
        if (r >= blk) break;
        if (turned) {
#pragma unroll
          for (int e = 0; e < 8; ++e) k[i][e] = M.keys[r * HD + 8 * ln + e];    // this thread's own
        } else rk[i].get(r < old ? tkh : nkh, k[i]);
        rv[i].get(r < old ? tvh : nvh, v[i]);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (tkh) k[i][e] = round_bf(k[i][e]);
          if (tvh) v[i][e] = round_bf(v[i][e]);
          ka = q8_amax(ka, k[i][e]); va = q8_amax(va, v[i][e]);
        }
      }
      ka = rows_max(lanes_max<16>(ka)); va = rows_max(lanes_max<16>(va));
      __syncthreads();                                                 // the block before is out of `turn` and `red`
      if (lane() == 0) { M.red[wave()] = ka; M.red[4 + wave()] = va; }
      __syncthreads();
      const float sk = q8_scale(fmaxf(fmaxf(M.red[0], M.red[1]), fmaxf(M.red[2], M.red[3]))), ik = sk > 0.f ? 1.f / sk : 0.f;
      const float sv = q8_scale(fmaxf(fmaxf(M.red[4], M.red[5]), fmaxf(M.red[6], M.red[7]))), iv = sv > 0.f ? 1.f / sv : 0.f;
      if (tid() == 0) { stwt32(A.ks.f() + (pair * A.ks.cols + j), sk); stwt32(A.vs.f() + (pair * A.vs.cols + j), sv); }
      const long long byte0 = (pair * A.nblk + j) * blk * HD;
      const __amdgpu_buffer_rsrc_t ok = wt_rsrc((const char*)A.kq.p + byte0, blk * HD), ov = wt_rsrc((const char*)A.vq.p + byte0, blk * HD);
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const int r = i * RPP + rw;
        if (r >= blk) break;
        uint32_t w[2] = {0, 0};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          w[e / 4] |= (uint32_t)(q8_of(k[i][e], sk, ik) & 255) << (8 * (e % 4));
          M.turn[(8 * ln + e) * (blk + 4) + r] = (unsigned char)q8_of(v[i][e], sv, iv);
        }
        __builtin_amdgcn_raw_buffer_store_b64(u32x2_t{w[0], w[1]}, ok, r * HD + 8 * ln, 0, 16 /* SC1 */);
      }
      __syncthreads();
      for (int e = tid(); e < HD * blk / 16; e += KVM_THREADS) {
        const LDS uint32_t* x = (const LDS uint32_t*)(M.turn + (16 * e / blk) * (blk + 4) + 16 * e % blk);
        stwt_buf(ov, 16 * e, __builtin_bit_cast(f32x4n, u32x4_t{x[0], x[1], x[2], x[3]}));
      }
    }
  }
}
template <int HD> __device__ __forceinline__ void append_q8_t(const Ctx& c) {
  constexpr int LPR = HD / 8, RPP = KVM_THREADS / LPR;
  const AppendQ8 A(c);
  if (!A.lengths_ok(c)) return;
  const AppendLds<HD> M(c.smem);
  const int ln = tid() % LPR, rw = tid() / LPR, blk = A.blk, nh = A.h1 - A.h0;
  const GLOBAL float* gamma = A.kg.ok() ? A.kg.f() : nullptr;
  const LDS double* rot = A.theta > 0.f ? M.freq : nullptr;
  if (rot && tid() < HD / 2) M.freq[tid()] = q8_freq(tid(), HD, log((double)A.theta));
  if (A.finishes()) {                                                  // (a barrier on both ways)
    if (blk <= 4 * RPP) append_q8_blocks<HD, 4>(c);
    else append_q8_blocks<HD, 128 / RPP>(c);
  }
  if (A.p != 0) return;
  __syncthreads();                                                     // old rows of the tail have been read
  const int most = min(A.n, blk - 1), rows = (A.b1 - A.b0) * nh * most;   // rows of an unfinished block: no more than that
  for (int u = rw; u < rows; u += RPP) {
    const int b = A.b0 + u / (nh * most), h = A.h0 + u / most % nh, L = A.lens.i()[b];
    if (L < 0) continue;
    const long long t = max((long long)L, (long long)((L + A.n) / blk) * blk) + u % most;
    if (t >= (long long)L + A.n) continue;
    const long long row = (long long)b * A.n + (t - L), at = ((long long)b * A.Hkv + h) * blk + t % blk;
    Raw8 rk, rv;
    rk.load(A.kn, row * A.kn.cols + h * HD + 8 * ln);
    rv.load(A.vn, row * A.vn.cols + h * HD + 8 * ln);
    float k[8], v[8];
    rk.get(A.kn.dtype == 2, k); rv.get(A.vn.dtype == 2, v);
    if (gamma || rot) head8_turn<HD>(k, gamma, A.eps, rot, t, M.angs + rw * HD);
    st8(A.kt, at * A.kt.cols + 8 * ln, k);
    st8(A.vt, at * A.vt.cols + 8 * ln, v);
  }
}
__device__ __noinline__ bool op_kv_append_q8_fast(const Ctx& c) {
  if (!rows8_ok(c.buf(0)) || !rows8_ok(c.buf(1)) || !rows8_ok(c.buf(6)) || !rows8_ok(c.buf(7))) return false;
  if (c.i(18) == 128) append_q8_t<128>(c);
  else if (c.i(18) == 64) append_q8_t<64>(c);
  else return false;
  return true;
}

// Arguments of op 313. A pair is a sequence and a kv head; its R = n * G query rows: row r = i * G + g is token i of head kvh * G + g.
struct DecodeQ8 {
  View q, kq, ks, vq, vs, kt, vt, lens, part, o, cnt, qg;
  int b0, b1, s, S, n, H, Hkv, hd, blk, G, R;
  float scale, theta, eps;
  __device__ explicit DecodeQ8(const Ctx& c)
      : q(c.buf(0)), kq(c.buf(1)), ks(c.buf(2)), vq(c.buf(3)), vs(c.buf(4)), kt(c.buf(5)), vt(c.buf(6)), lens(c.buf(7)), part(c.buf(8)), o(c.buf(9)),
        cnt(c.buf(10)), qg(c.buf(11)), b0(c.i(12)), b1(c.i(13)), s(c.i(14)), S(c.i(15)), n(c.i(16)), H(c.i(17)), Hkv(c.i(18)), hd(c.i(19)), blk(c.i(20)),
        scale(c.f(21)), theta(c.f(22)), eps(c.f(23)) { G = H / Hkv; R = n * G; }
  __device__ long long at(const View& X, int b, int h, int r) const { return ((long long)b * n + r / G) * X.cols + (h * G + r % G) * hd; }
  __device__ bool length_ok(const Ctx& c, int b, int L) const {
    if (L >= -1 && (long long)L + n <= (long long)blk * ks.cols) return true;
    c.fail(KVM_ERR_OP_KVLEN, b, L);
    return false;
  }
  __device__ void zeros(int b, int h) const { for (int e = tid(); e < R * hd; e += KVM_THREADS) o.st(at(o, b, h, e / hd) + e % hd, 0.f); }
};

// Decode attention over the 8-bit cache, any alignment and head size: whole pairs, every S-th one; 256 tokens at a time, a thread
// to a token for the scores and to an output element for P V, each row with its running maximum and sum.
__device__ __forceinline__ void attn_q8_pair(const Ctx& c, const DecodeQ8& D, int b, int kvh, int L) {
  constexpr float LOG2E = 1.44269504088896340736f;
  const int n = L + D.n, whole = n / D.blk * D.blk;
  __syncthreads();
  LDS float* q = (LDS float*)c.smem;                                   // [32][128]
  LDS float* p = q + 32 * 128;                                         // [32][256]
  LDS float* st = p + 32 * 256;                                        // [32] factors of the last step, then flags and sums
  LDS float* red = st + 32;
  const int hd = D.hd, half = hd / 2;
  for (int r = 0; r < D.R; ++r) {
    for (int k = tid(); k < hd; k += KVM_THREADS) q[r * hd + k] = D.q.ld(D.at(D.q, b, kvh, r) + k);
    __syncthreads();
    if (D.qg.ok()) {
      float ss = 0.f;
      for (int k = tid(); k < hd; k += KVM_THREADS) ss += q[r * hd + k] * q[r * hd + k];
      const float rs = 1.f / sqrtf(block_sum(ss, red) / hd + D.eps);
      for (int k = tid(); k < hd; k += KVM_THREADS) q[r * hd + k] *= rs * D.qg.f()[k];
      __syncthreads();
    }
    if (D.theta > 0.f)
      for (int i = tid(); i < half; i += KVM_THREADS) {
        float sn, co; q8_turn(L + r / D.G, q8_freq(i, hd, log((double)D.theta)), sn, co);
        const float x1 = q[r * hd + i], x2 = q[r * hd + i + half];
        q[r * hd + i] = x1 * co - x2 * sn; q[r * hd + i + half] = x1 * sn + x2 * co;
      }
  }
  __syncthreads();
  const long long pair = (long long)b * D.Hkv + kvh, bytes0 = pair * D.ks.cols * D.blk * hd;
  const GLOBAL signed char* K = (const GLOBAL signed char*)D.kq.p + bytes0;
  const GLOBAL signed char* V = (const GLOBAL signed char*)D.vq.p + bytes0;
  float acc[16];                                                       // of rows tid / hd, + 256 / hd, .. (hd < 16: some of them)
  const int d = tid() % hd, rows = KVM_THREADS / hd, ra = tid() / hd;
  LDS float* m_run = red + 16; LDS float* l_run = m_run + 32;
  for (int r = tid(); r < D.R; r += KVM_THREADS) { m_run[r] = -INFINITY; l_run[r] = 0.f; }
  for (int i = 0; i < 16; ++i) acc[i] = 0.f;
  for (int t0 = 0; t0 < n; t0 += KVM_THREADS) {
    const int t = t0 + tid(), cnt = min(n - t0, KVM_THREADS);
    __syncthreads();
    for (int r = 0; r < D.R; ++r) {
      float a = -INFINITY;
      if (t < n && t <= L + r / D.G) {
        a = 0.f;
        if (t < whole) {
          for (int k = 0; k < hd; ++k) a += q[r * hd + k] * (float)K[(long long)t * hd + k];
          a *= D.ks.f()[pair * D.ks.cols + t / D.blk];
        } else for (int k = 0; k < hd; ++k) a += q[r * hd + k] * D.kt.at(pair * D.blk + t - whole, k);
        a *= D.scale * LOG2E;
      }
      p[r * KVM_THREADS + tid()] = a;
      const float mx = fmaxf(m_run[r], block_max(a, red));
      const float e = a == -INFINITY ? 0.f : exp2f(a - mx), sum = block_sum(e, red);
      p[r * KVM_THREADS + tid()] = e;
      if (tid() == 0) { const float f = mx == -INFINITY ? 1.f : exp2f(m_run[r] - mx); st[r] = f; l_run[r] = l_run[r] * f + sum; m_run[r] = mx; }
    }
    __syncthreads();
    if (ra < rows)
      for (int i = 0; i < 16; ++i) {
        const int r = ra + i * rows;
        if (r >= D.R) break;
        float a = acc[i] * st[r];
        for (int u = 0; u < cnt; ++u) {
          const int tt = t0 + u;
          if (tt > L + r / D.G) break;
          const float v = tt < whole ? (float)V[(long long)(tt / D.blk) * D.blk * hd + d * D.blk + tt % D.blk] * D.vs.f()[pair * D.vs.cols + tt / D.blk]
                                     : D.vt.at(pair * D.blk + tt - whole, d);
          a += p[r * KVM_THREADS + u] * v;
        }
        acc[i] = a;
      }
  }
  __syncthreads();
  if (ra < rows)
    for (int i = 0; i < 16; ++i) {
      const int r = ra + i * rows;
      if (r >= D.R) break;
      D.o.st(D.at(D.o, b, kvh, r) + d, acc[i] / l_run[r]);
    }
}
__device__ __noinline__ void op_attn_decode_q8(const Ctx& c) {
  const DecodeQ8 D(c);
  for (int p = D.s; p < (D.b1 - D.b0) * D.Hkv; p += D.S) {
    const int b = D.b0 + p / D.Hkv, h = p % D.Hkv, L = D.lens.i()[b];
    if (L == -1) D.zeros(b, h);
    else if (L >= -1 && (long long)L + D.n <= (long long)D.blk * D.ks.cols) attn_q8_pair(c, D, b, h, L);
    else { if (tid() == 0) D.length_ok(c, b, L); return; }
  }
}

// ---- The work of a call over its tasks: every pair costs Q8_PAIR (query rows, the unfinished block, the end) and one per unit of 64
// tokens of its whole blocks; the pairs in order, by sequence and head, are cut into equal shares, in the tasks alike from the
// lengths. A cut within Q8_SNAP of a pair's end moves there: a small piece costs more than it balances. A pair that is cut has one piece in
// each of consecutive tasks; the first has the unfinished block.
constexpr int Q8_PAIR = 8, Q8_SNAP = 12, Q8_SHARE = 24, Q8_SEQS = 1024;
// (32 bits are enough: a unit is 4 KB and more of cache, whose buffers hold less than 2^33 bytes.)
struct WorkQ8 {
  const LDS int* pre;          // [seqs + 1] cost of the sequences before, for one head
  int seqs, Hkv, share, total;
  // The pair at x: its sequence and head, where it starts, its cost.
  struct At { int b, h, start, cost; };
  __device__ __forceinline__ At find(int x) const {
    int b = 0;
    for (int j0 = 0; j0 < seqs; j0 += 64) b += __popcll(__ballot(j0 + lane() < seqs && pre[j0 + lane()] * Hkv <= x));
    b = rfl(b) - 1;
    const int p0 = rfl(pre[b]), cost = rfl(pre[b + 1]) - p0, h = (int)((unsigned)(x - p0 * Hkv) / (unsigned)cost);
    return At{b, h, p0 * Hkv + h * cost, cost};
  }
  // Where task i starts.
  __device__ __forceinline__ int cut(int i) const {
    const int x = (int)min((long long)i * share, (long long)total);
    if (x == total) return total;
    const At a = find(x);
    const int off = x - a.start;
    return off < Q8_SNAP ? a.start : a.cost - off < Q8_SNAP ? a.start + a.cost : x;
  }
  // The first task that starts inside the pair, and how many do.
  __device__ __forceinline__ int first_inside(const At& a) const { return (int)((unsigned)(a.start + Q8_SNAP + share - 1) / (unsigned)share); }
  __device__ __forceinline__ int inside(const At& a) const {
    if (a.cost < 2 * Q8_SNAP) return 0;
    return max(0, (int)((unsigned)(a.start + a.cost - Q8_SNAP + share) / (unsigned)share) - first_inside(a));
  }
};
// Lengths and cost sums of the call's sequences into LDS; false if a length is out of range (reported).
__device__ __forceinline__ bool q8_work(const Ctx& c, const DecodeQ8& D, LDS int* pre, LDS int* len, LDS int* tot, WorkQ8& W) {
  constexpr int PER = Q8_SEQS / KVM_THREADS;
  const int seqs = D.b1 - D.b0;
  int cost[PER], sum = 0;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int k = tid() * PER + i;
    cost[i] = 0;
    if (k < seqs) {
      const int L = D.lens.i()[D.b0 + k];
      bad = bad || !D.length_ok(c, D.b0 + k, L);
      len[k] = L;
      cost[i] = L < 0 ? 1 : Q8_PAIR + (int)(((((unsigned)L + D.n) & -(unsigned)D.blk) + 63) >> 6);
      sum += cost[i];
    }
  }
  int upto = sum;
  for (int o = 1; o < 64; o <<= 1) { const int y = __shfl_up(upto, o, 64); if (lane() >= o) upto += y; }
  if (lane() == 63) tot[wave()] = upto;
  if (__syncthreads_or(bad)) return false;
  int at = upto - sum;
  for (int w = 0; w < KVM_WAVES; ++w) at += w < wave() ? tot[w] : 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int k = tid() * PER + i;
    if (k < seqs) { pre[k] = at; at += cost[i]; if (k == seqs - 1) pre[seqs] = at; }
  }
  __syncthreads();
  W.pre = pre; W.seqs = seqs; W.Hkv = D.Hkv;
  W.total = rfl(pre[seqs]) * D.Hkv;
  // equal shares, but none below Q8_SHARE unless there are tasks enough for a pair each
  W.share = max((int)((unsigned)(W.total + D.S - 1) / (unsigned)D.S), min(Q8_SHARE, (int)((unsigned)(W.total + seqs * D.Hkv - 1) / (unsigned)(seqs * D.Hkv))));
  return true;
}
// The piece of a pair that counts itself last merges them; maxima are in units of log2. Piece k lies in the partials of task i0 + k - 1,
// the first one in their second half. A wave takes a row at a time: lane i has the maximum and sum of piece i, the weights go from
// there to all lanes, which add up to two head dims each, the loads of 16 pieces in flight.
__device__ __forceinline__ void q8_arrive(const Ctx& c, const DecodeQ8& D, int b, int h, int i0, int live, LDS int* flag) {
  wait_stores();
  __syncthreads();
  GLOBAL int* cnt = D.cnt.i() + ((long long)b * D.Hkv + h);
  if (tid() == 0) *flag = add_relaxed((int*)cnt, 1);
  __syncthreads();
  const int old = *flag;
  if (old < 0 || old >= live) { if (tid() == 0) c.fail(KVM_ERR_OP_RANGE, b * D.Hkv + h, old); return; }
  if (old != live - 1) return;
  fence_acquire();                                                     // the other pieces' partials, stored before their counts
  constexpr int SB = 16;
  const int l = lane(), hd = D.hd, d0 = min(l, hd - 1), d1 = min(l + 64, hd - 1);
  for (int r = wave(); r < D.R; r += KVM_WAVES) {
    auto piece = [&](int k) { return D.part.f() + ((long long)(2 * i0 - 2 + (k ? 2 * k : 1)) * D.R + r) * D.part.cols; };
    float M = -INFINITY, a0 = 0.f, a1 = 0.f, z = 0.f;
    for (int s0 = 0; s0 < live; s0 += 64) {
      const bool mine = s0 + l < live;
      const GLOBAL float* y = piece(min(s0 + l, live - 1));
      const float m = mine ? y[hd] : -INFINITY, x = mine ? y[hd + 1] : 0.f;
      const float top = fmaxf(M, rows_max(lanes_max<16>(m))), f = M == -INFINITY ? 0.f : exp2f(M - top), e = m == -INFINITY ? 0.f : exp2f(m - top);
      z = z * f + e * x; a0 *= f; a1 *= f; M = top;
      for (int s1 = 0; s1 < 64 && s0 + s1 < live; s1 += SB) {
        float x0[SB], x1[SB];
#pragma unroll
        for (int i = 0; i < SB; ++i) {
          const GLOBAL float* w = piece(min(s0 + s1 + i, live - 1));
          x0[i] = w[d0]; x1[i] = w[d1];
        }
#pragma unroll
        for (int i = 0; i < SB; ++i) {
          const float w = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(e), s1 + i));
          if (s0 + s1 + i < live) { a0 += w * x0[i]; a1 += w * x1[i]; }
        }
      }
    }
    z = rows_sum(lanes_sum<16>(z));
    if (l < hd) D.o.st(D.at(D.o, b, h, r) + l, a0 / z);
    if (l + 64 < hd) D.o.st(D.at(D.o, b, h, r) + l + 64, a1 / z);
  }
  if (tid() == 0) st_relaxed((int*)cnt, 0);
}

// Decode attention over the 8-bit cache at head sizes 64 and 128, on the matrix units. Bound: streaming the cache's bytes.
// Each wave takes units of 64 tokens in turn, K and V straight from memory into registers in the layout of the operands:
//   scores  v_mfma_f32_16x16x32_f16, A = 16 keys, B = up to 16 query rows (NT such tiles). A lane's 16-byte load of a key
//           feeds two products, so the head dims run in the order of those loads, for the queries alike.
//   P V     the same instruction with A = V transposed (16 head dims x 32 tokens: the cache keeps a block's values as
//           [hd][blk], so this too is a 16-byte load), B = P. Tokens go to the rows of the score tiles (row m of tile a: token
//           16 (m / 4) + 4 a + m % 4) such that the scores' output registers are the B operand, in the loads' order.
// A byte becomes an f16 by two instructions for two of them (0x6400 | (q + 128) is 1024 + q + 128), exactly. Queries and
// probabilities are f16 pairs, the value and its remainder (22 bits: queries scaled by a power of two per row, probabilities
// to 2^12, so that no remainder that matters falls below f16's numbers), two products each, summed in f32. A block's key
// scale multiplies its scores; its value scale the probabilities, relative to the largest so far (vref, a power of two).
// Each unit's P V is summed on its own and added to the running one in f32 (the units' chained sums round towards -inf).
// The unfinished block is f32 work of all lanes: at most blk - 1 tokens.
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
// Eight signed bytes (two words) as f16.
__device__ __forceinline__ f16x8 q8_half(uint32_t w0, uint32_t w1) {
  const f16x2 off = {(_Float16)-1152.f, (_Float16)-1152.f};
  w0 ^= 0x80808080u; w1 ^= 0x80808080u;
  f16x2 x[4] = {__builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, w0, 0x04010400u)), __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, w0, 0x04030402u)),
                __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, w1, 0x04010400u)), __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, w1, 0x04030402u))};
  f16x8 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) { x[i] += off; r[2 * i] = x[i].x; r[2 * i + 1] = x[i].y; }
  return r;
}
template <int HD> struct UnitQ8 { u32x4_t k[4][HD / 64], v[HD / 16]; float ks, vs; };
// LDS of a task. The work and the frequencies stay through its pieces; the tail's scores and values give way to the waves' P V.
template <int HD> struct DecodeLds {
  LDS int* pre; LDS int* len; LDS double* freq; LDS float* qs; LDS float* to; LDS float* st; LDS float* cr; LDS float* ts; LDS float* tv;
  __device__ explicit DecodeLds(LDS char* p)
      : pre((LDS int*)p),                                              // [Q8_SEQS + 1]
        len(pre + Q8_SEQS + 4),                                        // [Q8_SEQS]
        freq((LDS double*)(len + Q8_SEQS)),                            // [HD / 2]
        qs((LDS float*)(freq + HD / 2)),                               // [32][HD + 4] queries
        to(qs + 32 * (HD + 4)),                                        // [32][HD] the tail's P V
        st(to + 32 * HD),                                              // [5][2][32] maxima and sums of the waves and the tail
        cr(st + 320),                                                  // [32] factors from a product to a score
        ts(cr + 32),                                                   // [32][128] the tail's scores
        tv(ts + 32 * 128) {}                                           // [128][HD] its values
  static_assert((2 * Q8_SEQS + 4 + HD + 32 * (HD + 4) + 32 * HD + 352 + 32 * 128 + 128 * HD) * 4 <= KVM_LDS_BYTES, "decode attention LDS map");
};
// One piece of a pair: units [u0, u1), with `first` also the unfinished block; `live` pieces in all, piece 1 in task i0's partials.
template <int HD, int NT> __device__ __noinline__ void attn_q8_piece(const Ctx& c, int b, int kvh, int L, int u0, int u1, bool first, int i0, int live) {
  constexpr float LOG2E = 1.44269504088896340736f, PS = 4096.f;
  constexpr int KH = HD / 64, VT = HD / 16, LPR = HD / 8, RPP = KVM_THREADS / LPR, QS = HD + 4;
  const DecodeLds<HD> M(c.smem);
  LDS float *const qs = M.qs, *const to = M.to, *const st = M.st, *const cr = M.cr, *const ts = M.ts, *const tv = M.tv;
  const DecodeQ8 D(c);
  const int blk = rfl(D.blk), lb = 31 - __clz(blk), n = L + D.n, whole = n & -blk, nt = first ? n - whole : 0;
  const bool tail = nt > 0;
  const int l = lane(), w = wave(), nn = l & 15, qq = l >> 4, ln = tid() % LPR, rw = tid() / LPR;
  const long long pair = (long long)b * D.Hkv + kvh, byte0 = pair * D.ks.cols * blk * HD;
  const GLOBAL char* K = (const GLOBAL char*)D.kq.p + byte0;
  const GLOBAL char* V = (const GLOBAL char*)D.vq.p + byte0;
  const GLOBAL float* KS = D.ks.f() + pair * D.ks.cols;
  const GLOBAL float* VS = D.vs.f() + pair * D.vs.cols;
  auto load = [&](UnitQ8<HD>& U, int u) {                              // tokens past the last whole block: the last ones again, masked below
    const int t0 = u << 6, rest = whole - t0;
    const GLOBAL char* kb = K + (long long)t0 * HD;
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
      for (int h = 0; h < KH; ++h) U.k[a][h] = *(const GLOBAL u32x4a4*)(kb + min(16 * (nn >> 2) + 4 * a + (nn & 3), rest - 1) * HD + 16 * (qq + 4 * h));
    const int tt = (t0 & (blk - 1)) + min(16 * qq, rest - 16), j = tt >> lb;   // from the start of the block of t0
    const GLOBAL char* vb = V + ((long long)(t0 >> lb) << lb) * HD + j * blk * HD + (tt & (blk - 1));
#pragma unroll
    for (int d = 0; d < VT; ++d) U.v[d] = *(const GLOBAL u32x4a4*)(vb + (16 * d + nn) * blk);
    U.ks = KS[(t0 >> lb) + j]; U.vs = VS[(t0 >> lb) + j];
  };
  // everything that a short context needs is requested at once: query rows, the unfinished block, the first unit
  constexpr int QP = (16 * NT + RPP - 1) / RPP, TP = 4;
  Raw8 rq[QP], rk[TP], rv[TP];
#pragma unroll
  for (int i = 0; i < QP; ++i) if (i * RPP + rw < D.R) rq[i].load(D.q, D.at(D.q, b, kvh, i * RPP + rw) + 8 * ln);
  auto load_tail = [&](int t0) {
#pragma unroll
    for (int i = 0; i < TP; ++i) {
      const long long t = pair * blk + min(t0 + i * RPP + rw, nt - 1);
      if (t0 + i * RPP < nt) { rk[i].load(D.kt, t * D.kt.cols + 8 * ln); rv[i].load(D.vt, t * D.vt.cols + 8 * ln); }
    }
  };
  if (tail) load_tail(0);
  UnitQ8<HD> U;
  if (u0 + w < u1) load(U, u0 + w);
  // query rows: norm, rotation, then scaled so that the largest magnitude of a row lies in [2^10, 2^11)
#pragma unroll
  for (int i = 0; i < QP; ++i) {
    const int r = i * RPP + rw;
    if (r >= 16 * NT) break;
    float x[8] = {};
    if (r < D.R) {
      rq[i].get(D.q.dtype == 2, x);
      head8_turn<HD>(x, D.qg.ok() ? D.qg.f() : nullptr, D.eps, D.theta > 0.f ? M.freq : nullptr, L + r / D.G, ts + rw * HD);
    }
    float big = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) big = fmaxf(big, fabsf(x[e]));
    big = lanes_max<LPR>(big);
    const int ex = max(20, (int)(__float_as_uint(big) >> 23));
    const float up = __uint_as_float((uint32_t)(264 - ex) << 23), down = __uint_as_float((uint32_t)(ex - 10) << 23);
#pragma unroll
    for (int e = 0; e < 8; ++e) qs[r * QS + 8 * ln + e] = x[e] * up;
    if (ln == 0) cr[r] = down * D.scale * LOG2E;
  }
  __syncthreads();
  if (tail) {                                                          // scores of the unfinished block, then its own softmax and P V
    for (int t0 = 0; t0 < nt; t0 += TP * RPP) {
      if (t0) load_tail(t0);
      float x[TP][8];
#pragma unroll
      for (int i = 0; i < TP; ++i) {
        const int t = t0 + i * RPP + rw;
        if (t >= nt) break;
        float y[8];
        rk[i].get(D.kt.dtype == 2, x[i]);
        rv[i].get(D.vt.dtype == 2, y);
#pragma unroll
        for (int e = 0; e < 8; ++e) tv[t * HD + 8 * ln + e] = y[e];
      }
      for (int r = 0; r < D.R; ++r) {
        float q[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) q[e] = qs[r * QS + 8 * ln + e];
        const int seen = min(nt, L + r / D.G + 1 - whole);
#pragma unroll
        for (int i = 0; i < TP; ++i) {
          const int t = t0 + i * RPP + rw;
          float a = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) a += q[e] * x[i][e];
          a = lanes_sum<LPR>(a);
          if (ln == 0 && t < nt) ts[r * 128 + t] = t < seen ? a * cr[r] : -INFINITY;
        }
      }
    }
    __syncthreads();
    for (int r = w; r < D.R; r += KVM_WAVES) {
      const float a = l < nt ? ts[r * 128 + l] : -INFINITY, b = 64 + l < nt ? ts[r * 128 + 64 + l] : -INFINITY;
      const float m = rows_max(lanes_max<16>(fmaxf(a, b)));
      const float pa = a == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(a - m), pb = b == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(b - m);
      const float z = rows_sum(lanes_sum<16>(pa + pb));
      ts[r * 128 + l] = pa; ts[r * 128 + 64 + l] = pb;
      if (l == 0) { st[256 + r] = m; st[288 + r] = z; }
    }
    __syncthreads();
    constexpr int RB = 2 * KVM_THREADS / HD;                           // two rows a thread, RB in all
    for (int r0 = tid() / HD; r0 < D.R; r0 += RB) {
      const int d = tid() % HD, r1 = min(r0 + RB / 2, D.R - 1);
      const int s0 = min(nt, L + r0 / D.G + 1 - whole), s1 = min(nt, L + r1 / D.G + 1 - whole);   // values not to be seen do not count, NaN neither
      float a[2][4] = {};
      for (int t = 0; t < s1; t += 8)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float x = tv[(t + e) * HD + d], y0 = ts[r0 * 128 + t + e] * x, y1 = ts[r1 * 128 + t + e] * x;
          a[0][e % 4] += t + e < s0 ? y0 : 0.f; a[1][e % 4] += t + e < s1 ? y1 : 0.f;
        }
      to[r0 * HD + d] = (a[0][0] + a[0][1]) + (a[0][2] + a[0][3]);
      to[r1 * HD + d] = (a[1][0] + a[1][1]) + (a[1][2] + a[1][3]);
    }
  }
  // the queries as B operands: row nn of tile g, dims 16 (qq + 4 h) + 8 p ..
  f16x8 qh[NT][KH][2], ql[NT][KH][2];
  float mrun[NT], lrun[NT], crow[NT];
  int lim[NT];
  f32x4n o[NT][VT];
#pragma unroll
  for (int g = 0; g < NT; ++g) {
    const int r = 16 * g + nn;
#pragma unroll
    for (int h = 0; h < KH; ++h)
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float x = qs[r * QS + 16 * (qq + 4 * h) + 8 * p + e];
          const _Float16 hi = (_Float16)x;
          qh[g][h][p][e] = hi; ql[g][h][p][e] = (_Float16)(x - (float)hi);
        }
    crow[g] = cr[r]; mrun[g] = -INFINITY; lrun[g] = 0.f;
    lim[g] = r < D.R ? min(whole, L + r / D.G + 1) : 0;
#pragma unroll
    for (int d = 0; d < VT; ++d) o[g][d] = f32x4n{0.f, 0.f, 0.f, 0.f};
  }
  float vref = 1.17549435e-38f;
  for (int u = u0 + w; u < u1; u += KVM_WAVES) {
    UnitQ8<HD> N;
    if (u + KVM_WAVES < u1) load(N, u + KVM_WAVES);
    const float vm0 = U.vs == U.vs ? U.vs : 0.f, vm = rows_max(vm0);
    float fv = 1.f;
    if (vm > vref) {                                                   // uniform: the four lane groups hold the unit's scales
      const float nv = __uint_as_float((__float_as_uint(vm) & 0x7f800000u) + 0x00800000u);
      fv = vref * __uint_as_float(0x7f000000u - __float_as_uint(nv));
      vref = nv;
    }
    const float pv = U.vs * __uint_as_float(0x7f000000u - __float_as_uint(vref)) * PS;
    float sc[NT][16];
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      f32x4n hi[NT], lo[NT];
#pragma unroll
      for (int g = 0; g < NT; ++g) hi[g] = lo[g] = f32x4n{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int h = 0; h < KH; ++h)
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          const f16x8 k = q8_half(U.k[a][h][2 * p], U.k[a][h][2 * p + 1]);
#pragma unroll
          for (int g = 0; g < NT; ++g) {
            hi[g] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, qh[g][h][p], hi[g], 0, 0, 0);
            lo[g] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, ql[g][h][p], lo[g], 0, 0, 0);
          }
        }
#pragma unroll
      for (int g = 0; g < NT; ++g)
#pragma unroll
        for (int i = 0; i < 4; ++i) sc[g][4 * a + i] = (hi[g][i] + lo[g][i]) * (crow[g] * U.ks);
    }
    f16x8 ph[NT][2], pl[NT][2];
    float fo[NT];
#pragma unroll
    for (int g = 0; g < NT; ++g) {
      const int seen = lim[g] - 64 * u - 16 * qq;                      // of this lane's 16 tokens
      float m = mrun[g];
#pragma unroll
      for (int i = 0; i < 16; ++i) if (i < seen) m = fmaxf(m, sc[g][i]);
      m = rows_max(m);
      const float base = m == -INFINITY ? 0.f : m;                     // nothing seen yet (or NaN, which stays)
      const float f = __builtin_amdgcn_exp2f(mrun[g] - base);
      float z = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float e = i < seen ? __builtin_amdgcn_exp2f(sc[g][i] - base) : 0.f, x = i < seen ? e * pv : 0.f;
        z += e;
        const _Float16 hi = (_Float16)x;
        ph[g][i / 8][i % 8] = hi; pl[g][i / 8][i % 8] = (_Float16)(x - (float)hi);
      }
      lrun[g] = lrun[g] * f + z;
      mrun[g] = m;
      fo[g] = f * fv;
    }
#pragma unroll
    for (int d = 0; d < VT; ++d) {
      const f16x8 v0 = q8_half(U.v[d].x, U.v[d].y), v1 = q8_half(U.v[d].z, U.v[d].w);
#pragma unroll
      for (int g = 0; g < NT; ++g) {
        f32x4n x = f32x4n{0.f, 0.f, 0.f, 0.f};
        x = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, ph[g][0], x, 0, 0, 0);
        x = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, ph[g][1], x, 0, 0, 0);
        x = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, pl[g][0], x, 0, 0, 0);
        x = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, pl[g][1], x, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < 4; ++i) o[g][d][i] = fmaf(o[g][d][i], fo[g], x[i]);
      }
    }
    U = N;
  }
  // the waves' and the tail's states, then their sum over all of them
  __syncthreads();
  LDS float* ow = ts;                                                  // [4][R][HD], over the tail's scores and values
#pragma unroll
  for (int g = 0; g < NT; ++g) {
    const int r = 16 * g + nn;
    const float z = rows_sum(lrun[g]);
    if (r < D.R) {
#pragma unroll
      for (int d = 0; d < VT; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) ow[(w * D.R + r) * HD + 16 * d + 4 * qq + i] = o[g][d][i] * (vref * (1.f / PS));
      if (qq == 0) { st[64 * w + r] = mrun[g]; st[64 * w + 32 + r] = z; }
    }
  }
  __syncthreads();
  for (int e = tid(); e < D.R * HD; e += KVM_THREADS) {
    const int r = e / HD, d = e % HD;
    float M = tail ? st[256 + r] : -INFINITY, a = 0.f, z = 0.f;
#pragma unroll
    for (int v = 0; v < KVM_WAVES; ++v) M = fmaxf(M, st[64 * v + r]);
#pragma unroll
    for (int v = 0; v < KVM_WAVES; ++v) {
      const float m = st[64 * v + r], f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - M);
      a += f * ow[(v * D.R + r) * HD + d]; z += f * st[64 * v + 32 + r];
    }
    if (tail) {
      const float m = st[256 + r], f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - M);
      a += f * to[r * HD + d]; z += f * st[288 + r];
    }
    if (live == 1) { D.o.st(D.at(D.o, b, kvh, r) + d, a / z); continue; }
    GLOBAL float* x = D.part.f() + ((long long)(2 * D.s + first) * D.R + r) * D.part.cols;
    stwt32(x + d, a);
    if (d == 0) { stwt32(x + HD, M); stwt32(x + HD + 1, z); }
  }
  if (live > 1) q8_arrive(c, D, b, kvh, i0, live, (LDS int*)qs);
}
template <int HD> __device__ __forceinline__ void attn_q8_t(const Ctx& c) {
  const DecodeLds<HD> M(c.smem);
  const DecodeQ8 D(c);
  WorkQ8 W;
  if (!q8_work(c, D, M.pre, M.len, (LDS int*)M.ts, W)) return;
  if (D.theta > 0.f && tid() < HD / 2) M.freq[tid()] = q8_freq(tid(), HD, log((double)D.theta));
  const int stop = W.cut(D.s + 1);
  for (int at = W.cut(D.s); at < stop;) {
    const WorkQ8::At P = W.find(at);
    const int off = at - P.start, end = min(P.cost, stop - P.start), L = rfl(M.len[P.b]), b = D.b0 + P.b;
    at = P.start + end;
    if (L < 0) { D.zeros(b, P.h); continue; }
    const bool cut = off > 0 || end < P.cost;
    const int u0 = max(0, off - Q8_PAIR), u1 = max(0, end - Q8_PAIR), i0 = cut ? W.first_inside(P) : 0, live = cut ? W.inside(P) + 1 : 1;
    __syncthreads();                                                   // frequencies; the piece before is out of LDS
    if (D.R > 16) attn_q8_piece<HD, 2>(c, b, P.h, L, u0, u1, off == 0, i0, live);
    else attn_q8_piece<HD, 1>(c, b, P.h, L, u0, u1, off == 0, i0, live);
  }
}
__device__ __noinline__ bool op_attn_decode_q8_fast(const Ctx& c) {
  if (!rows8_ok(c.buf(0)) || !rows8_ok(c.buf(5)) || !rows8_ok(c.buf(6))) return false;
  if (c.i(19) == 128) attn_q8_t<128>(c);
  else if (c.i(19) == 64) attn_q8_t<64>(c);
  else return false;
  return true;
}

// ---------------------------------------------------------------------------------------------- logits
// Adjusted logits (op 314): the token counts of the sequence in LDS, one word per logit of a chunk (generated: bits 0..19, bias
// slot: bits 20..30, prompt: bit 31), then the logits against them. Bound: the bytes of the logits, and per task the history, which
// every task of a row reads as a whole (a few KB, from the L2), and the clearing of the words. Logits go in vectors of 4
// from any element (a bf16 row from its first aligned one), eight per thread requested before the ones before are used;
// most have the word 0 and only meet the mask. A token's entries in the bias list meet by an atomic maximum of (2047 - entry),
// which leaves the slot of the first; the others are added to it in list order, one after another (they are few).
constexpr int ADJ_CHUNK = 26624, ADJ_BIAS = 2047, ADJ_NB = 8;
struct AdjustArgs {
  View x, out, par, hist, plen, hlen, last, bidx, bval, mask, mrow;
  int r0, r1, v0, v1, V;
  __device__ explicit AdjustArgs(const Ctx& c)
      : x(c.buf(0)), out(c.buf(1)), par(c.buf(2)), hist(c.buf(3)), plen(c.buf(4)), hlen(c.buf(5)), last(c.buf(6)), bidx(c.buf(7)), bval(c.buf(8)),
        mask(c.buf(9)), mrow(c.buf(10)), r0(c.i(11)), r1(c.i(12)), v0(c.i(13)), v1(c.i(14)), V(c.i(15)) {}
  // All rows of the task are checked before anything is written.
  __device__ bool rows_ok(const Ctx& c) const {
    bool bad = false;
    for (int r = r0 + tid(); r < r1; r += KVM_THREADS) {
      const int n = hist.ok() ? hlen.i()[r] : 0, pl = hist.ok() ? plen.i()[r] : 0, m = mrow.ok() ? mrow.i()[r] : 0;
      if (n < 0 || pl < 0 || pl > n || (hist.ok() && n + (last.ok() ? 1 : 0) > hist.cols)) { bad = true; c.fail(KVM_ERR_OP_RANGE, r, n); }
      if (mrow.ok() && (m < -1 || m >= mask.rows)) { bad = true; c.fail(KVM_ERR_OP_RANGE, r, m); }
    }
    return !__syncthreads_or(bad);
  }
};
__device__ __forceinline__ float adjusted(float x, uint32_t w, float rep, float freq, float pres, const LDS float* bsum) {
  if (w) {
    const uint32_t times = w & 0xfffffu, slot = (w >> 20) & 2047u;
    if (times || (w >> 31)) x = x > 0.f ? x / rep : x * rep;
    if (times) { x -= freq * (float)times; x -= pres; }
    if (slot) x += bsum[ADJ_BIAS - slot];
  }
  return x;
}
__device__ __forceinline__ void lds_or(LDS uint32_t* p, uint32_t v) { __hip_atomic_fetch_or(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP); }
__device__ __noinline__ void op_logits_adjust(const Ctx& c) {
  const AdjustArgs A(c);
  if (!A.rows_ok(c)) return;
  LDS uint32_t* cnt = (LDS uint32_t*)c.smem;                           // [ADJ_CHUNK + 8]
  LDS float* bsum = (LDS float*)(cnt + ADJ_CHUNK + 8);                 // [ADJ_BIAS + 1] an entry's value, the first one's the sum
  LDS int* later = (LDS int*)(bsum + ADJ_BIAS + 1);                    // [ADJ_BIAS + 1] first entry of the same token, or -1
  static_assert((ADJ_CHUNK + 8 + 2 * (ADJ_BIAS + 1)) * 4 <= KVM_LDS_BYTES, "logits LDS map");
  constexpr int NB = ADJ_NB;
  const int nb = A.bidx.ok() ? A.bidx.cols : 0;
  const bool xh = A.x.dtype == 2, oh = A.out.dtype == 2;
  for (int r = A.r0; r < A.r1; ++r) {
    const float rep = A.par.at(r, 0), freq = A.par.at(r, 1), pres = A.par.at(r, 2);
    const int n = A.hist.ok() ? A.hlen.i()[r] : 0, pl = A.hist.ok() ? A.plen.i()[r] : 0, last = A.last.ok() ? A.last.i()[r] : -1;
    const GLOBAL int* hist = A.hist.ok() ? A.hist.i() + (long long)r * A.hist.cols : nullptr;
    const GLOBAL int* bidx = nb ? A.bidx.i() + (long long)r * A.bidx.cols : nullptr;
    const int mr = A.mask.ok() ? (A.mrow.ok() ? A.mrow.i()[r] : r) : -1;
    const GLOBAL int* mask = mr >= 0 ? A.mask.i() + (long long)mr * A.mask.cols : nullptr;
    for (int c0 = A.v0; c0 < A.v1; c0 += ADJ_CHUNK) {
      const int len = min(A.v1 - c0, ADJ_CHUNK);
      const GLOBAL char* xp = (const GLOBAL char*)A.x.p + ((long long)r * A.x.cols + c0) * (xh ? 2 : 4);
      const GLOBAL char* op = (const GLOBAL char*)A.out.p + ((long long)r * A.out.cols + c0) * (oh ? 2 : 4);
      // vectors start where bf16 storage is 4-byte aligned, on both sides; rows that never are go one by one
      const int px = xh ? (int)((uintptr_t)xp >> 1) & 1 : 0, po = oh ? (int)((uintptr_t)op >> 1) & 1 : 0;
      const int peel = min(len, max(px, po)), nv = xh && oh && px != po ? 0 : (len - peel) / 4;
      const bool whole = ((c0 + peel) & 3) == 0;                       // no vector's mask bits lie in two words
      LDS uint32_t* w = cnt + (4 - peel) % 4;                          // word of logit c0 + i: w[i], a vector's at 16 bytes
      const __amdgpu_buffer_rsrc_t ro = wt_rsrc((const char*)op, (long long)len * (oh ? 2 : 4));
      u32x4_t x[NB];
      uint32_t m0[NB], m1[NB];
      auto request = [&](int q0) {
#pragma unroll
        for (int u = 0; u < NB; ++u) {
          const int i = peel + 4 * min(q0 + u * KVM_THREADS, nv - 1), v = c0 + i;
          if (xh) { const u32x2_t t = *(const GLOBAL u32x2a4*)(xp + 2 * i); x[u].x = t.x; x[u].y = t.y; }
          else x[u] = *(const GLOBAL u32x4a4*)(xp + 4 * i);
          m0[u] = m1[u] = ~0u;
          if (mask) { m0[u] = mask[v >> 5]; if (!whole) m1[u] = mask[(v + 3) >> 5]; }
        }
      };
      if (tid() < nv) request(tid());
      __syncthreads();
      for (int i = tid(); i < (len + 11) / 4; i += KVM_THREADS) ((LDS u32x4_t*)cnt)[i] = u32x4_t{0, 0, 0, 0};
      __syncthreads();
      if (nb) {
        for (int j = tid(); j < nb; j += KVM_THREADS) {
          const int v = bidx[j] - c0;
          if (v >= 0 && v < len) __hip_atomic_fetch_max(&w[v], (uint32_t)(ADJ_BIAS - j) << 20, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
        }
        __syncthreads();
        bool many = false;
        for (int j = tid(); j < nb; j += KVM_THREADS) {
          const int v = bidx[j] - c0, first = v >= 0 && v < len ? ADJ_BIAS - (int)(w[v] >> 20) : j;
          bsum[j] = A.bval.f()[(long long)r * A.bval.cols + j];
          later[j] = first == j ? -1 : first;
          many = many || first != j;
        }
        if (__syncthreads_or(many) && wave() == 0)                     // entries of one token, in list order
          for (int j0 = 0; j0 < nb; j0 += 64) {
            const int mine = j0 + lane() < nb ? later[j0 + lane()] : -1;
            for (uint64_t left = __ballot(mine >= 0); left; left &= left - 1) {
              const int j = __ffsll((long long)left) - 1, to = __builtin_amdgcn_readlane(mine, j);
              if (lane() == 0) bsum[to] += bsum[j0 + j];
            }
          }
      }
      auto said = [&](int k, int token) {
        const int v = token - c0;
        if (v < 0 || v >= len) return;
        if (k < pl) lds_or(&w[v], 0x80000000u);
        else __hip_atomic_fetch_add(&w[v], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
      };
      for (int k0 = 4 * tid(); k0 < n / 4 * 4; k0 += 16 * KVM_THREADS) {
        u32x4_t h[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) h[u] = *(const GLOBAL u32x4a4*)(hist + min(k0 + 4 * u * KVM_THREADS, n / 4 * 4 - 4));
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int k = k0 + 4 * u * KVM_THREADS;
          if (k >= n / 4 * 4) break;
#pragma unroll
          for (int e = 0; e < 4; ++e) said(k + e, (int)h[u][e]);
        }
      }
      if (tid() < n % 4) said(n / 4 * 4 + tid(), hist[n / 4 * 4 + tid()]);
      if (tid() == 4) said(n, last);
      __syncthreads();
      for (int q0 = tid(); q0 < nv; q0 += NB * KVM_THREADS) {
        f32x4n y[NB];
        uint32_t bits[NB];
#pragma unroll
        for (int u = 0; u < NB; ++u) {
          const int sh = (c0 + peel + 4 * (q0 + u * KVM_THREADS)) & 31;
          if (xh) y[u] = __builtin_bit_cast(f32x4n, u32x4_t{x[u].x << 16, x[u].x & 0xffff0000u, x[u].y << 16, x[u].y & 0xffff0000u});
          else y[u] = __builtin_bit_cast(f32x4n, x[u]);
          bits[u] = (uint32_t)((((uint64_t)m1[u] << 32) | m0[u]) >> sh);
        }
        if (q0 + NB * KVM_THREADS < nv) request(q0 + NB * KVM_THREADS);
#pragma unroll
        for (int u = 0; u < NB; ++u) {
          const int q = q0 + u * KVM_THREADS, i = peel + 4 * q;
          if (q >= nv) break;
          const u32x4_t t = *(const LDS u32x4_t*)(w + i);
          if (t.x | t.y | t.z | t.w) {
#pragma unroll
            for (int e = 0; e < 4; ++e) y[u][e] = adjusted(y[u][e], t[e], rep, freq, pres, bsum);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) if (!((bits[u] >> e) & 1)) y[u][e] = -INFINITY;
          if (oh) stwt_bf4_buf(ro, 2 * i, y[u]);
          else stwt_buf(ro, 4 * i, y[u]);
        }
      }
      for (int k = tid(); k < len - 4 * nv; k += KVM_THREADS) {         // before the first vector and behind the last
        const int i = k < peel ? k : k + 4 * nv, v = c0 + i;
        float y = adjusted(A.x.at(r, v), w[i], rep, freq, pres, bsum);
        if (mask && !((mask[v >> 5] >> (v & 31)) & 1)) y = -INFINITY;
        A.out.st((long long)r * A.out.cols + v, y);
      }
    }
    if (A.last.ok() && A.v0 == 0 && tid() == 0) stwt32i(A.hist.i() + ((long long)r * A.hist.cols + n), last);
  }
}

}  // namespace kvm
