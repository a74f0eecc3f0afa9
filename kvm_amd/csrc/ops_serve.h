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

// Arguments of op 312 as every form reads them; Tmax = blk * ks.cols.
struct AppendQ8 {
  View kn, vn, kq, ks, vq, vs, kt, vt, lens, kg;
  int b0, b1, h0, h1, p, P, n, Hkv, hd, blk, nblk;
  float theta, eps;
  __device__ explicit AppendQ8(const Ctx& c)
      : kn(c.buf(0)), vn(c.buf(1)), kq(c.buf(2)), ks(c.buf(3)), vq(c.buf(4)), vs(c.buf(5)), kt(c.buf(6)), vt(c.buf(7)), lens(c.buf(8)), kg(c.buf(9)),
        b0(c.i(10)), b1(c.i(11)), h0(c.i(12)), h1(c.i(13)), p(c.i(14)), P(c.i(15)), n(c.i(16)), Hkv(c.i(17)), hd(c.i(18)), blk(c.i(19)),
        nblk(ks.cols), theta(c.f(20)), eps(c.f(21)) {}
  // Every length is checked before anything is written: all workers of the operator refuse alike.
  __device__ bool lengths_ok(const Ctx& c) const {
    for (int b = b0; b < b1; ++b) {
      const int L = lens.i()[b];
      if (L < -1 || (long long)L + n > (long long)blk * nblk) { if (tid() == 0) c.fail(KVM_ERR_OP_KVLEN, b, L); return false; }
    }
    return true;
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
  for (int e = tid(); e < D.R * D.hd; e += KVM_THREADS) {
    const int r = e / D.hd, d = e % D.hd;
    float M = -INFINITY, a = 0.f, l = 0.f;
    for (int s = 0; s < live; ++s) M = fmaxf(M, D.part.f()[D.part_at(s, r) + D.hd]);
    for (int s = 0; s < live; ++s) {
      const GLOBAL float* x = D.part.f() + D.part_at(s, r);
      const float m = x[D.hd], w = m == -INFINITY ? 0.f : exp2f(m - M);
      a += w * x[d]; l += w * x[D.hd + 1];
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

// ---------------------------------------------------------------------------------------------- logits
// Adjusted logits (op 314): the token counts of the sequence in LDS, one word per logit of a chunk (generated: bits 0..19,
// bias slot + 1: bits 20..30, prompt: bit 31), then the logits one by one. Each task reads the whole history, a few KB, against
// its range of logits. Entries of one token in the bias list share the slot of the first, with their sum in list order.
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
  LDS uint32_t* cnt = (LDS uint32_t*)c.smem;                           // [ADJ_CHUNK]
  LDS float* bsum = (LDS float*)(cnt + ADJ_CHUNK);                     // [ADJ_BIAS + 1]
  LDS int* bidx = (LDS int*)(bsum + ADJ_BIAS + 1);
  const int nb = A.bidx.ok() ? A.bidx.cols : 0;
  for (int r = A.r0; r < A.r1; ++r) {
    const float rep = A.par.at(r, 0), freq = A.par.at(r, 1), pres = A.par.at(r, 2);
    const int n = A.hist.ok() ? A.hlen.i()[r] : 0, pl = A.hist.ok() ? A.plen.i()[r] : 0, last = A.last.ok() ? A.last.i()[r] : -1;
    const GLOBAL int* hist = A.hist.ok() ? A.hist.i() + (long long)r * A.hist.cols : nullptr;
    const int mr = A.mask.ok() ? (A.mrow.ok() ? A.mrow.i()[r] : r) : -1;
    const GLOBAL int* mask = mr >= 0 ? A.mask.i() + (long long)mr * A.mask.cols : nullptr;
    __syncthreads();
    for (int j = tid(); j < nb; j += KVM_THREADS) bidx[j] = A.bidx.i()[(long long)r * nb + j];
    __syncthreads();
    for (int j = tid(); j < nb; j += KVM_THREADS) {
      const int v = bidx[j];
      float s = 0.f;
      if (v >= A.v0 && v < A.v1) for (int k = 0; k < nb; ++k) if (bidx[k] == v) s += A.bval.f()[(long long)r * A.bval.cols + k];
      bsum[j] = s;
    }
    for (int c0 = A.v0; c0 < A.v1; c0 += ADJ_CHUNK) {
      const int c1 = min(A.v1, c0 + ADJ_CHUNK);
      __syncthreads();
      for (int i = tid(); i < c1 - c0; i += KVM_THREADS) cnt[i] = 0;
      __syncthreads();
      for (int j = tid(); j < nb; j += KVM_THREADS) {
        const int v = bidx[j];
        bool first = v >= c0 && v < c1;
        for (int k = 0; first && k < j; ++k) first = bidx[k] != v;
        if (first) __hip_atomic_fetch_or(&cnt[v - c0], (uint32_t)(j + 1) << 20, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
      }
      for (int k = tid(); k <= n; k += KVM_THREADS) {
        const int v = k < n ? hist[k] : last;
        if (v < c0 || v >= c1) continue;
        if (k < pl) __hip_atomic_fetch_or(&cnt[v - c0], 0x80000000u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
        else __hip_atomic_fetch_add(&cnt[v - c0], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
      }
      __syncthreads();
      for (int v = c0 + tid(); v < c1; v += KVM_THREADS) {
        float y = adjusted(A.x.at(r, v), cnt[v - c0], rep, freq, pres, bsum);
        if (mask && !((mask[v >> 5] >> (v & 31)) & 1)) y = -INFINITY;
        A.out.st((long long)r * A.out.cols + v, y);
      }
    }
    if (A.last.ok() && A.v0 == 0 && tid() == 0) stwt32i(A.hist.i() + ((long long)r * A.hist.cols + n), last);
  }
}

}  // namespace kvm
