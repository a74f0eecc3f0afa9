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
// by up to 4e-3), reduced to one turn there; sine and cosine in f32.
__device__ __forceinline__ double q8_freq(int i, int hd, double ln_theta) { return exp(-2.0 * i / hd * ln_theta); }
__device__ __forceinline__ void q8_turn(long long t, double freq, float& sn, float& co) {
  const double turns = (double)t * freq * 0.15915494309189533577;      // 1 / (2 pi)
  sincosf((float)((turns - rint(turns)) * 6.28318530717958647693), &sn, &co);
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
__device__ __forceinline__ void row8(const View& X, long long o, float (&v)[8]) {
  if (X.dtype == 2) {
    const u16x8_t h = *(const GLOBAL u16x8_t*)(X.h() + o);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = bf2f(h[i]);
  } else {
    const f32x4n a = *(const GLOBAL f32x4n*)(X.f() + o), b = *(const GLOBAL f32x4n*)(X.f() + o + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[i] = a[i]; v[4 + i] = b[i]; }
  }
}
// A head of HD values spread over HD / 8 neighbouring lanes, 8 each: RMS norm (g: this lane's gains, or none) and rotation of
// position t (freq: the HD / 2 frequencies in LDS, or none), in f32. The other half of a pair is HD / 16 lanes away; the lanes
// share out the row's angles through `ang`, 2 HD floats of LDS for each row in flight (HD / 8 lanes of one wave).
template <int HD> __device__ __forceinline__ void head8_turn(float (&v)[8], const GLOBAL float* gamma, float eps, const LDS double* freq, long long t, LDS float* ang) {
  constexpr int LPR = HD / 8;
  const int ln = lane() % LPR;
  if (gamma) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss += v[i] * v[i];
#pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1) ss += __shfl_xor(ss, o, 64);
    const float rs = 1.f / sqrtf(ss / HD + eps);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = v[i] * rs * gamma[8 * ln + i];
  }
  if (freq) {
#pragma unroll 1
    for (int i = ln; i < HD / 2; i += LPR) { float sn, co; q8_turn(t, freq[i], sn, co); ang[i] = sn; ang[HD / 2 + i] = co; }
    __builtin_amdgcn_wave_barrier();                                   // one wave's LDS operations stay in order
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
// for single tokens, bytes for prompts. A row is HD / 8 lanes of 8 values, so a pass of the workgroup takes 16 or 32 rows: a
// finished block is in registers as a whole (K and V together, one load round, one reduction of both maxima). Keys to be
// normalised or rotated go through LDS first, row by row. Keys are stored as they lie, 8 bytes a lane; values turn through LDS.
// Tail rows of all pairs of the task go in one range, a row to HD / 8 lanes.
template <int HD> __device__ __noinline__ void append_q8_t(const Ctx& c) {
  constexpr int LPR = HD / 8, RPP = KVM_THREADS / LPR, NP = 128 / RPP;    // lanes a row, rows a pass, passes of the largest block
  const AppendQ8 A(c);
  if (!A.lengths_ok(c)) return;
  LDS double* freq = (LDS double*)c.smem;                              // [HD / 2]
  LDS float* red = (LDS float*)(freq + HD / 2);                        // [8]
  LDS float* keys = red + 16;                                          // [blk][HD]
  LDS float* angs = keys + 128 * HD;                                   // [RPP][2 HD / 2]
  LDS unsigned char* turn = (LDS unsigned char*)(angs + RPP * HD);     // [HD][blk + 4]
  const int ln = tid() % LPR, rw = tid() / LPR, blk = A.blk;
  const GLOBAL float* gamma = A.kg.ok() ? A.kg.f() : nullptr;
  const LDS double* rot = A.theta > 0.f ? freq : nullptr;
  if (rot && tid() < HD / 2) freq[tid()] = q8_freq(tid(), HD, log((double)A.theta));
  __syncthreads();
  const int nh = A.h1 - A.h0;
  for (int u = 0; u < (A.b1 - A.b0) * nh; ++u) {
    const int b = A.b0 + u / nh, h = A.h0 + u % nh, L = A.lens.i()[b];
    if (L < 0) continue;
    const long long pair = (long long)b * A.Hkv + h;
    const int j0 = L / blk, jE = (L + A.n) / blk, mid = max(0, jE - j0 - 1);
    const int m0 = (int)((long long)mid * A.p / A.P), m1 = (int)((long long)mid * (A.p + 1) / A.P);
    for (int it = A.p == 0 && jE > j0 ? m0 - 1 : m0; it < m1; ++it) {  // (p = 0: m0 = 0, and -1 is the first block)
      const int j = j0 + 1 + it;
      const long long t0 = (long long)j * blk;
      auto new_row = [&](const View& X, long long t) { return ((long long)b * A.n + (t - L)) * X.cols + h * HD + 8 * ln; };
      if (gamma || rot) {
        __syncthreads();
#pragma unroll 1
        for (int r = rw; r < blk; r += RPP) {
          float x[8];
          if (t0 + r >= L) {
            row8(A.kn, new_row(A.kn, t0 + r), x);
            head8_turn<HD>(x, gamma, A.eps, rot, t0 + r, angs + rw * HD);
          } else row8(A.kt, (pair * blk + r) * A.kt.cols + 8 * ln, x);
#pragma unroll
          for (int e = 0; e < 8; ++e) keys[r * HD + 8 * ln + e] = x[e];
        }
      }
      float k[NP][8], v[NP][8];
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const int r = i * RPP + rw;
        if (r >= blk) break;
        if (gamma || rot) {
#pragma unroll
          for (int e = 0; e < 8; ++e) k[i][e] = keys[r * HD + 8 * ln + e];      // this thread's own
        }
        if (t0 + r < L) {
          if (!(gamma || rot)) row8(A.kt, (pair * blk + r) * A.kt.cols + 8 * ln, k[i]);
          row8(A.vt, (pair * blk + r) * A.vt.cols + 8 * ln, v[i]);
        } else {
          if (!(gamma || rot)) row8(A.kn, new_row(A.kn, t0 + r), k[i]);
          row8(A.vn, new_row(A.vn, t0 + r), v[i]);
        }
      }
      float ka = 0.f, va = 0.f;
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        if (i * RPP + rw >= blk) break;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (A.kt.dtype == 2) k[i][e] = round_bf(k[i][e]);
          if (A.vt.dtype == 2) v[i][e] = round_bf(v[i][e]);
          ka = q8_amax(ka, k[i][e]); va = q8_amax(va, v[i][e]);
        }
      }
      ka = wave_max(ka); va = wave_max(va);
      __syncthreads();                                                 // the block before is out of `turn` and `red`
      if (lane() == 0) { red[wave()] = ka; red[4 + wave()] = va; }
      __syncthreads();
      const float sk = q8_scale(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]))), ik = sk > 0.f ? 1.f / sk : 0.f;
      const float sv = q8_scale(fmaxf(fmaxf(red[4], red[5]), fmaxf(red[6], red[7]))), iv = sv > 0.f ? 1.f / sv : 0.f;
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
          turn[(8 * ln + e) * (blk + 4) + r] = (unsigned char)q8_of(v[i][e], sv, iv);
        }
        __builtin_amdgcn_raw_buffer_store_b64(u32x2_t{w[0], w[1]}, ok, r * HD + 8 * ln, 0, 16 /* SC1 */);
      }
      __syncthreads();
      for (int e = tid(); e < HD * blk / 16; e += KVM_THREADS) {
        const LDS uint32_t* x = (const LDS uint32_t*)(turn + (16 * e / blk) * (blk + 4) + 16 * e % blk);
        stwt_buf(ov, 16 * e, __builtin_bit_cast(f32x4n, u32x4_t{x[0], x[1], x[2], x[3]}));
      }
    }
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
    float k[8], v[8];
    row8(A.kn, row * A.kn.cols + h * HD + 8 * ln, k);
    row8(A.vn, row * A.vn.cols + h * HD + 8 * ln, v);
    if (gamma || rot) head8_turn<HD>(k, gamma, A.eps, rot, t, angs + rw * HD);
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

// Arguments of op 313; R = n * G query rows of a task, row r = i * G + g is token i of head kvh * G + g.
struct DecodeQ8 {
  View q, kq, ks, vq, vs, kt, vt, lens, part, o, cnt, qg;
  int b, kvh, s, S, n, H, Hkv, hd, blk, G, R, L;
  float scale, theta, eps;
  __device__ explicit DecodeQ8(const Ctx& c)
      : q(c.buf(0)), kq(c.buf(1)), ks(c.buf(2)), vq(c.buf(3)), vs(c.buf(4)), kt(c.buf(5)), vt(c.buf(6)), lens(c.buf(7)), part(c.buf(8)), o(c.buf(9)),
        cnt(c.buf(10)), qg(c.buf(11)), b(c.i(12)), kvh(c.i(13)), s(c.i(14)), S(c.i(15)), n(c.i(16)), H(c.i(17)), Hkv(c.i(18)), hd(c.i(19)), blk(c.i(20)),
        scale(c.f(21)), theta(c.f(22)), eps(c.f(23)) { G = H / Hkv; R = n * G; L = lens.i()[b]; }
  __device__ long long q_at(int r) const { return ((long long)b * n + r / G) * q.cols + (kvh * G + r % G) * hd; }
  __device__ long long o_at(int r) const { return ((long long)b * n + r / G) * o.cols + (kvh * G + r % G) * hd; }
  // This split's partial of row r: unnormalised P V, then the maximum and the sum.
  __device__ long long part_at(int split, int r) const { return ((((long long)b * S + split) * H + kvh * G) * n + r) * part.cols; }
  // false: nothing to do (a length out of range is reported; a slot that serves no sequence gives zeros).
  __device__ bool begin(const Ctx& c) const {
    if (L < -1 || (long long)L + n > (long long)blk * ks.cols) { if (tid() == 0) c.fail(KVM_ERR_OP_KVLEN, b, L); return false; }
    if (L >= 0) return true;
    if (s == 0) for (int e = tid(); e < R * hd; e += KVM_THREADS) o.st(o_at(e / hd) + e % hd, 0.f);
    return false;
  }
};
// The split that counts itself last merges the `live` splits' partials; maxima are in units of log2.
__device__ __forceinline__ void q8_arrive(const Ctx& c, const DecodeQ8& D, int live, LDS int* flag) {
  wait_stores();
  __syncthreads();
  GLOBAL int* cnt = D.cnt.i() + ((long long)D.b * D.Hkv + D.kvh);
  if (tid() == 0) *flag = add_relaxed((int*)cnt, 1);
  __syncthreads();
  const int old = *flag;
  if (old < 0 || old >= live) { if (tid() == 0) c.fail(KVM_ERR_OP_RANGE, D.b * D.Hkv + D.kvh, old); return; }
  if (old != live - 1) return;
  fence_acquire();                                                     // the other splits' partials, stored before their counts
  constexpr int SB = 16;                                               // splits in flight: their loads wait for memory together
  for (int e = tid(); e < D.R * D.hd; e += KVM_THREADS) {
    const int r = e / D.hd, d = e % D.hd;
    float M = -INFINITY, a = 0.f, l = 0.f;
    for (int s0 = 0; s0 < live; s0 += SB) {
      float x[SB], m[SB], z[SB], top = M;
#pragma unroll
      for (int i = 0; i < SB; ++i) {
        const GLOBAL float* y = D.part.f() + D.part_at(min(s0 + i, live - 1), r);
        x[i] = y[d]; m[i] = y[D.hd]; z[i] = y[D.hd + 1];
      }
#pragma unroll
      for (int i = 0; i < SB; ++i) top = fmaxf(top, m[i]);
      const float f = M == -INFINITY ? 0.f : exp2f(M - top);
      a *= f; l *= f; M = top;
#pragma unroll
      for (int i = 0; i < SB; ++i) {
        const float w = m[i] == -INFINITY ? 0.f : exp2f(m[i] - M);
        if (s0 + i < live) { a += w * x[i]; l += w * z[i]; }
      }
    }
    D.o.st(D.o_at(r) + d, a / l);
  }
  if (tid() == 0) st_relaxed((int*)cnt, 0);
}

// Decode attention over the 8-bit cache, any alignment and head size: 256 tokens at a time, a thread to a token for the scores
// and to an output element for P V, each row with its running maximum and sum.
__device__ __noinline__ void op_attn_decode_q8(const Ctx& c) {
  const DecodeQ8 D(c);
  if (!D.begin(c)) return;
  constexpr float LOG2E = 1.44269504088896340736f;
  const int n = D.L + D.n, whole = n / D.blk * D.blk, live = min(D.S, (n + 255) / 256);
  if (D.s >= live) return;
  const int per = ((n + live - 1) / live + 255) / 256 * 256, j0 = min(n, D.s * per), j1 = min(n, j0 + per);
  LDS float* q = (LDS float*)c.smem;                                   // [32][128]
  LDS float* p = q + 32 * 128;                                         // [32][256]
  LDS float* st = p + 32 * 256;                                        // [32] factors of the last step, then flags and sums
  LDS float* red = st + 32;
  const int hd = D.hd, half = hd / 2;
  for (int r = 0; r < D.R; ++r) {
    for (int k = tid(); k < hd; k += KVM_THREADS) q[r * hd + k] = D.q.ld(D.q_at(r) + k);
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
        float sn, co; q8_turn(D.L + r / D.G, q8_freq(i, hd, log((double)D.theta)), sn, co);
        const float x1 = q[r * hd + i], x2 = q[r * hd + i + half];
        q[r * hd + i] = x1 * co - x2 * sn; q[r * hd + i + half] = x1 * sn + x2 * co;
      }
  }
  __syncthreads();
  const long long pair = (long long)D.b * D.Hkv + D.kvh, bytes0 = pair * D.ks.cols * D.blk * hd;
  const GLOBAL signed char* K = (const GLOBAL signed char*)D.kq.p + bytes0;
  const GLOBAL signed char* V = (const GLOBAL signed char*)D.vq.p + bytes0;
  float acc[16];                                                       // of rows tid / hd, + 256 / hd, .. (hd < 16: some of them)
  const int d = tid() % hd, rows = KVM_THREADS / hd, ra = tid() / hd;
  LDS float* m_run = red + 16; LDS float* l_run = m_run + 32;
  for (int r = tid(); r < D.R; r += KVM_THREADS) { m_run[r] = -INFINITY; l_run[r] = 0.f; }
  for (int i = 0; i < 16; ++i) acc[i] = 0.f;
  for (int t0 = j0; t0 < j1; t0 += KVM_THREADS) {
    const int t = t0 + tid(), cnt = min(j1 - t0, KVM_THREADS);
    __syncthreads();
    for (int r = 0; r < D.R; ++r) {
      float a = -INFINITY;
      if (t < j1 && t <= D.L + r / D.G) {
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
          if (tt > D.L + r / D.G) break;
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
      if (live == 1) { D.o.st(D.o_at(r) + d, acc[i] / l_run[r]); continue; }
      GLOBAL float* x = D.part.f() + D.part_at(D.s, r);
      stwt32(x + d, acc[i]);
      if (d == 0) { stwt32(x + hd, m_run[r]); stwt32(x + hd + 1, l_run[r]); }
    }
  if (live > 1) q8_arrive(c, D, live, (LDS int*)st);
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
// The unfinished block is f32 work of all lanes in the last split: at most blk - 1 tokens.
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
template <int HD, int NT> __device__ __noinline__ void attn_q8_t(const Ctx& c) {
  constexpr float LOG2E = 1.44269504088896340736f, PS = 4096.f;
  constexpr int KH = HD / 64, VT = HD / 16, LPR = HD / 8, RPP = KVM_THREADS / LPR, QS = HD + 4;
  const DecodeQ8 D(c);
  if (!D.begin(c)) return;
  const int n = D.L + D.n, blk = rfl(D.blk), lb = 31 - __clz(blk), whole = rfl(n & -blk), nt = n - whole;
  const int units = (whole + 63) >> 6, live = min(D.S, max(1, units));
  if (D.s >= live) return;
  const int u0 = (int)(((long long)D.s * units + live - 1) / live), u1 = (int)(((long long)(D.s + 1) * units + live - 1) / live);
  const bool tail = D.s == live - 1 && nt > 0;
  const int l = lane(), w = wave(), nn = l & 15, qq = l >> 4, ln = tid() % LPR, rw = tid() / LPR;
  // LDS: queries, the tail's P V and its stats stay; the tail's scores and values give way to the waves' P V at the end
  LDS float* qs = (LDS float*)c.smem;                                  // [32][HD + 4]
  LDS float* to = qs + 32 * QS;                                        // [32][HD]
  LDS float* st = to + 32 * HD;                                        // [5][2][32] maxima and sums of the waves and the tail
  LDS float* cr = st + 320;                                            // [32] factors from a product to a score
  LDS double* freq = (LDS double*)(cr + 32);                           // [HD / 2]
  LDS float* ts = (LDS float*)(freq + HD / 2);                         // [32][128]
  LDS float* tv = ts + 32 * 128;                                       // [128][HD]
  static_assert((32 * (HD + 4) + 32 * HD + 352 + HD + 32 * 128 + 128 * HD) * 4 <= KVM_LDS_BYTES, "decode attention LDS map");
  const long long pair = (long long)D.b * D.Hkv + D.kvh, byte0 = pair * D.ks.cols * blk * HD;
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
  UnitQ8<HD> U;
  if (D.theta > 0.f && tid() < HD / 2) freq[tid()] = q8_freq(tid(), HD, log((double)D.theta));
  if (u0 + w < u1) load(U, u0 + w);
  __syncthreads();
  // query rows: norm, rotation, then scaled so that the largest magnitude of a row lies in [2^10, 2^11)
  for (int r = rw; r < 16 * NT; r += RPP) {
    float x[8] = {};
    if (r < D.R) {
      row8(D.q, D.q_at(r) + 8 * ln, x);
      head8_turn<HD>(x, D.qg.ok() ? D.qg.f() : nullptr, D.eps, D.theta > 0.f ? freq : nullptr, D.L + r / D.G, ts + rw * HD);
    }
    float big = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) big = fmaxf(big, fabsf(x[i]));
#pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1) big = fmaxf(big, __shfl_xor(big, o, 64));
    const int ex = max(20, (int)(__float_as_uint(big) >> 23));
    const float up = __uint_as_float((uint32_t)(264 - ex) << 23), down = __uint_as_float((uint32_t)(ex - 10) << 23);
#pragma unroll
    for (int i = 0; i < 8; ++i) qs[r * QS + 8 * ln + i] = x[i] * up;
    if (ln == 0) cr[r] = down * D.scale * LOG2E;
  }
  __syncthreads();
  if (tail) {                                                          // scores of the unfinished block, then its own softmax and P V
    for (int t0 = 0; t0 < nt; t0 += 4 * RPP) {
      float x[4][8], y[4][8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int t = min(t0 + i * RPP + rw, nt - 1);
        row8(D.kt, (pair * blk + t) * D.kt.cols + 8 * ln, x[i]);
        row8(D.vt, (pair * blk + t) * D.vt.cols + 8 * ln, y[i]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int t = t0 + i * RPP + rw;
        if (t >= nt) break;
#pragma unroll
        for (int e = 0; e < 8; ++e) tv[t * HD + 8 * ln + e] = y[i][e];
        for (int r = 0; r < D.R; ++r) {
          float a = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) a += qs[r * QS + 8 * ln + e] * x[i][e];
#pragma unroll
          for (int o = LPR / 2; o > 0; o >>= 1) a += __shfl_xor(a, o, 64);
          if (ln == 0) ts[r * 128 + t] = whole + t <= D.L + r / D.G ? a * cr[r] : -INFINITY;
        }
      }
    }
    __syncthreads();
    for (int r = w; r < D.R; r += KVM_WAVES) {
      const float a = l < nt ? ts[r * 128 + l] : -INFINITY, b = 64 + l < nt ? ts[r * 128 + 64 + l] : -INFINITY;
      const float m = wave_max(fmaxf(a, b)), pa = a == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(a - m), pb = b == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(b - m);
      const float z = wave_sum(pa + pb);
      ts[r * 128 + l] = pa; ts[r * 128 + 64 + l] = pb;
      if (l == 0) { st[256 + r] = m; st[288 + r] = z; }
    }
    __syncthreads();
    for (int r = tid() / HD; r < D.R; r += KVM_THREADS / HD) {
      const int d = tid() % HD, seen = min(nt, D.L + r / D.G + 1 - whole);   // a value that the row may not see does not count, NaN neither
      float a = 0.f;
      for (int t = 0; t < seen; ++t) a += ts[r * 128 + t] * tv[t * HD + d];
      to[r * HD + d] = a;
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
    lim[g] = r < D.R ? min(whole, D.L + r / D.G + 1) : 0;
#pragma unroll
    for (int d = 0; d < VT; ++d) o[g][d] = f32x4n{0.f, 0.f, 0.f, 0.f};
  }
  float vref = 1.17549435e-38f;
  for (int u = u0 + w; u < u1; u += KVM_WAVES) {
    UnitQ8<HD> N;
    if (u + KVM_WAVES < u1) load(N, u + KVM_WAVES);
    const float vm0 = U.vs == U.vs ? U.vs : 0.f, vm1 = fmaxf(vm0, __shfl_xor(vm0, 16, 64)), vm = fmaxf(vm1, __shfl_xor(vm1, 32, 64));
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
      m = fmaxf(m, __shfl_xor(m, 16, 64));
      m = fmaxf(m, __shfl_xor(m, 32, 64));
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
    float z = lrun[g] + __shfl_xor(lrun[g], 16, 64);
    z += __shfl_xor(z, 32, 64);
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
    if (live == 1) { D.o.st(D.o_at(r) + d, a / z); continue; }
    GLOBAL float* x = D.part.f() + D.part_at(D.s, r);
    stwt32(x + d, a);
    if (d == 0) { stwt32(x + HD, M); stwt32(x + HD + 1, z); }
  }
  if (live > 1) q8_arrive(c, D, live, (LDS int*)qs);
}
__device__ __noinline__ bool op_attn_decode_q8_fast(const Ctx& c) {
  if (!rows8_ok(c.buf(0)) || !rows8_ok(c.buf(5)) || !rows8_ok(c.buf(6))) return false;
  const int hd = c.i(19);
  const bool two = c.i(16) * (c.i(17) / c.i(18)) > 16;
  if (hd == 128) { if (two) attn_q8_t<128, 2>(c); else attn_q8_t<128, 1>(c); }
  else if (hd == 64) { if (two) attn_q8_t<64, 2>(c); else attn_q8_t<64, 1>(c); }
  else return false;
  return true;
}

// ---------------------------------------------------------------------------------------------- logits
// Adjusted logits (op 314): the token counts of the sequence in LDS, one word per logit of a chunk (generated: bits 0..19,
// bias slot + 1: bits 20..30, prompt: bit 31), then the logits against them. Bound: the bytes of the logits, and per task the
// history, which every task of a row reads as a whole (a few KB, from the L2), and the clearing of the words. Logits go
// in vectors of 4 from any element (a bf16 row from its first aligned one), eight loads in flight per thread; most have the
// word 0 and only meet the mask. Entries of one token in the bias list share the slot of the first, with their sum in list order.
constexpr int ADJ_CHUNK = 26624, ADJ_BIAS = 2047;
struct AdjustArgs {
  View x, out, par, hist, plen, hlen, last, bidx, bval, mask, mrow;
  int r0, r1, v0, v1, V;
  __device__ explicit AdjustArgs(const Ctx& c)
      : x(c.buf(0)), out(c.buf(1)), par(c.buf(2)), hist(c.buf(3)), plen(c.buf(4)), hlen(c.buf(5)), last(c.buf(6)), bidx(c.buf(7)), bval(c.buf(8)),
        mask(c.buf(9)), mrow(c.buf(10)), r0(c.i(11)), r1(c.i(12)), v0(c.i(13)), v1(c.i(14)), V(c.i(15)) {}
  __device__ bool rows_ok(const Ctx& c) const {
    for (int r = r0; r < r1; ++r) {
      const int n = hist.ok() ? hlen.i()[r] : 0, pl = hist.ok() ? plen.i()[r] : 0, m = mrow.ok() ? mrow.i()[r] : 0;
      if (n < 0 || pl < 0 || pl > n || (hist.ok() && n + (last.ok() ? 1 : 0) > hist.cols)) { if (tid() == 0) c.fail(KVM_ERR_OP_RANGE, r, n); return false; }
      if (mrow.ok() && (m < -1 || m >= mask.rows)) { if (tid() == 0) c.fail(KVM_ERR_OP_RANGE, r, m); return false; }
    }
    return true;
  }
};
__device__ __forceinline__ float adjusted(float x, uint32_t w, float rep, float freq, float pres, const LDS float* bsum) {
  if (w) {
    const uint32_t times = w & 0xfffffu, slot = (w >> 20) & 2047u;
    if (times || (w >> 31)) x = x > 0.f ? x / rep : x * rep;
    if (times) { x -= freq * (float)times; x -= pres; }
    if (slot) x += bsum[slot - 1];
  }
  return x;
}
__device__ __noinline__ void op_logits_adjust(const Ctx& c) {
  const AdjustArgs A(c);
  if (!A.rows_ok(c)) return;
  LDS uint32_t* cnt = (LDS uint32_t*)c.smem;                           // [ADJ_CHUNK + 8]
  LDS float* bsum = (LDS float*)(cnt + ADJ_CHUNK + 8);                 // [ADJ_BIAS + 1]
  LDS int* bidx = (LDS int*)(bsum + ADJ_BIAS + 1);                     // [ADJ_BIAS + 1]; -1 for an entry that is not its token's first
  static_assert((ADJ_CHUNK + 8 + 2 * (ADJ_BIAS + 1)) * 4 <= KVM_LDS_BYTES, "logits LDS map");
  constexpr int NB = 8;
  const int nb = A.bidx.ok() ? A.bidx.cols : 0;
  const bool xh = A.x.dtype == 2, oh = A.out.dtype == 2;
  for (int r = A.r0; r < A.r1; ++r) {
    const float rep = A.par.at(r, 0), freq = A.par.at(r, 1), pres = A.par.at(r, 2);
    const int n = A.hist.ok() ? A.hlen.i()[r] : 0, pl = A.hist.ok() ? A.plen.i()[r] : 0, last = A.last.ok() ? A.last.i()[r] : -1;
    const GLOBAL int* hist = A.hist.ok() ? A.hist.i() + (long long)r * A.hist.cols : nullptr;
    const int mr = A.mask.ok() ? (A.mrow.ok() ? A.mrow.i()[r] : r) : -1;
    const GLOBAL int* mask = mr >= 0 ? A.mask.i() + (long long)mr * A.mask.cols : nullptr;
    if (nb) {
      __syncthreads();
      for (int j = tid(); j < nb; j += KVM_THREADS) bidx[j] = A.bidx.i()[(long long)r * A.bidx.cols + j];
      __syncthreads();
      int mine[(ADJ_BIAS + KVM_THREADS) / KVM_THREADS];
#pragma unroll
      for (int i = 0; i < (ADJ_BIAS + KVM_THREADS) / KVM_THREADS; ++i) {
        const int j = tid() + i * KVM_THREADS;
        mine[i] = -1;
        if (j >= nb) continue;
        const int v = bidx[j];
        if (v < A.v0 || v >= A.v1) continue;
        float s = 0.f;
        bool first = true;
        for (int k = 0; k < nb; ++k)
          if (bidx[k] == v) { first = first && k >= j; s += A.bval.f()[(long long)r * A.bval.cols + k]; }
        bsum[j] = s;
        if (first) mine[i] = v;
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < (ADJ_BIAS + KVM_THREADS) / KVM_THREADS; ++i) if (tid() + i * KVM_THREADS < nb) bidx[tid() + i * KVM_THREADS] = mine[i];
    }
    for (int c0 = A.v0; c0 < A.v1; c0 += ADJ_CHUNK) {
      const int len = min(A.v1 - c0, ADJ_CHUNK);
      const GLOBAL char* xp = (const GLOBAL char*)A.x.p + ((long long)r * A.x.cols + c0) * (xh ? 2 : 4);
      const GLOBAL char* op = (const GLOBAL char*)A.out.p + ((long long)r * A.out.cols + c0) * (oh ? 2 : 4);
      // vectors start where bf16 storage is 4-byte aligned, on both sides; rows that never are go one by one
      const int px = xh ? (int)((uintptr_t)xp >> 1) & 1 : 0, po = oh ? (int)((uintptr_t)op >> 1) & 1 : 0;
      const int peel = min(len, max(px, po)), nv = xh && oh && px != po ? 0 : (len - peel) / 4;
      LDS uint32_t* w = cnt + (4 - peel) % 4;                          // word of logit c0 + i: w[i], a vector's at 16 bytes
      const __amdgpu_buffer_rsrc_t ro = wt_rsrc((const char*)op, (long long)len * (oh ? 2 : 4));
      __syncthreads();
      for (int i = tid(); i < (len + 11) / 4; i += KVM_THREADS) ((LDS u32x4_t*)cnt)[i] = u32x4_t{0, 0, 0, 0};
      __syncthreads();
      for (int j = tid(); j < nb; j += KVM_THREADS) {
        const int v = bidx[j] - c0;
        if (v >= 0 && v < len) __hip_atomic_fetch_or(&w[v], (uint32_t)(j + 1) << 20, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
      }
      auto said = [&](int k, int token) {
        const int v = token - c0;
        if (v < 0 || v >= len) return;
        if (k < pl) __hip_atomic_fetch_or(&w[v], 0x80000000u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
        else __hip_atomic_fetch_add(&w[v], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
      };
      for (int k0 = 4 * tid(); k0 < n / 4 * 4; k0 += 4 * NB * KVM_THREADS) {
        u32x4_t h[NB];
#pragma unroll
        for (int u = 0; u < NB; ++u) h[u] = *(const GLOBAL u32x4a4*)(hist + min(k0 + 4 * u * KVM_THREADS, n / 4 * 4 - 4));
#pragma unroll
        for (int u = 0; u < NB; ++u) {
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
        u32x4_t x[NB];
        uint64_t bits[NB];
#pragma unroll
        for (int u = 0; u < NB; ++u) {
          const int i = peel + 4 * min(q0 + u * KVM_THREADS, nv - 1);
          if (xh) { const u32x2_t t = *(const GLOBAL u32x2a4*)(xp + 2 * i); x[u] = u32x4_t{t.x << 16, t.x & 0xffff0000u, t.y << 16, t.y & 0xffff0000u}; }
          else x[u] = *(const GLOBAL u32x4a4*)(xp + 4 * i);
          const int v = c0 + i;
          bits[u] = ~0ull;
          if (mask) bits[u] = (((uint64_t)(uint32_t)mask[(v + 3) >> 5] << 32) | (uint32_t)mask[v >> 5]) >> (v & 31);
        }
#pragma unroll
        for (int u = 0; u < NB; ++u) {
          const int q = q0 + u * KVM_THREADS, i = peel + 4 * q;
          if (q >= nv) break;
          f32x4n y = __builtin_bit_cast(f32x4n, x[u]);
          const u32x4_t t = *(const LDS u32x4_t*)(w + i);
          if (t.x | t.y | t.z | t.w) {
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = adjusted(y[e], t[e], rep, freq, pres, bsum);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) if (!((bits[u] >> e) & 1)) y[e] = -INFINITY;
          if (oh) stwt_bf4_buf(ro, 2 * i, y);
          else stwt_buf(ro, 4 * i, y);
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
