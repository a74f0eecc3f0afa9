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
// Eight values of a block of scale s as two words of bytes, the lowest first. x / s is rounded by adding 1.5 * 2^23, exactly so where
// x * inv is not within 2^-12 of the middle between two whole numbers (it is off by 127 * 2^-22 at most), by q8_of in the others.
// A NaN scale (or 0) comes with inv = 0.
__device__ __forceinline__ void q8_pack(const float (&x)[8], float s, float inv, uint32_t& w0, uint32_t& w1) {
  constexpr float MAGIC = 12582912.f;
  uint32_t y[8];
  float far = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float z = fmaf(x[e], inv, MAGIC);
    far = fmaxf(far, fabsf(fmaf(x[e], inv, -(z - MAGIC))));
    y[e] = __float_as_uint(z);
  }
  if (far > 0.5f - 0x1p-12f)
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = (uint32_t)q8_of(x[e], s, inv);
  w0 = __builtin_amdgcn_perm(__builtin_amdgcn_perm(y[3], y[2], 0x0c0c0400u), __builtin_amdgcn_perm(y[1], y[0], 0x0c0c0400u), 0x05040100u);
  w1 = __builtin_amdgcn_perm(__builtin_amdgcn_perm(y[7], y[6], 0x0c0c0400u), __builtin_amdgcn_perm(y[5], y[4], 0x0c0c0400u), 0x05040100u);
  if (!(s > 0.f)) w0 = w1 = 0;
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
// Between LDS stores of a wave's lanes and loads of the same words by others of them: one wave's LDS operations are carried out in order,
// the fences keep them in order in the program. Not behind a loop that lanes leave one by one: where such a loop ends an `if`, the compiler
// (LLVM 22) drops the restore of EXEC between the loop and the barrier, and registers that it reloads there come back in no lane.
// With angles by sincosf and registers short, that left query rows of NaN. Loops in front of it have the same rounds for all lanes.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}
// A head of HD values spread over HD / 8 neighbouring lanes, 8 each: RMS norm (gamma: the gains, or none) and rotation of
// position t (freq: the HD / 2 frequencies in LDS, or none), in f32. The other half of a pair is HD / 16 lanes away; the lanes
// share out the row's angles through `ang`, HD floats of LDS for each row in flight (HD / 8 lanes of one wave).
template <int HD> __device__ __forceinline__ void head8_turn(float (&v)[8], const GLOBAL float* gamma, float eps, const LDS double* freq, long long t, LDS float* ang) {
  constexpr int LPR = HD / 8;
  const int ln = lane() % LPR;
  if (freq) {
#pragma unroll 1
    for (int j = 0; j < HD / 2 / LPR; ++j) {
      const int i = ln + j * LPR;
      float sn, co; q8_turn(t, freq[i], sn, co);
      ang[i] = sn; ang[HD / 2 + i] = co;
    }
    wave_sync();
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
    wave_sync();
  }
}

// Arguments of op 312 as every form reads them; Tmax = blk * ks.cols.
struct AppendQ8 {
  View kn, vn, kq, ks, vq, vs, kt, vt, lens, kg;
  int b0, b1, h0, h1, p, P, n, Hkv, hd, blk, nblk;
  float theta, eps;
  __device__ explicit AppendQ8(const Ctx& c)
      : kn(uview(c, 0)), vn(uview(c, 1)), kq(uview(c, 2)), ks(uview(c, 3)), vq(uview(c, 4)), vs(uview(c, 5)), kt(uview(c, 6)), vt(uview(c, 7)), lens(uview(c, 8)), kg(uview(c, 9)),
        b0(rfl(c.i(10))), b1(rfl(c.i(11))), h0(rfl(c.i(12))), h1(rfl(c.i(13))), p(rfl(c.i(14))), P(rfl(c.i(15))), n(rfl(c.i(16))), Hkv(rfl(c.i(17))), hd(rfl(c.i(18))), blk(rfl(c.i(19))),
        nblk(ks.cols), theta(c.f(20)), eps(c.f(21)) {}
  // The lengths of the task's sequences are all checked before anything is written (-1: one is out of range, reported); otherwise
  // whether a block becomes full.
  __device__ int lengths(const Ctx& c, LDS int* word) const {
    bool bad = false, full = false;
    for (int b = b0 + tid(); b < b1; b += KVM_THREADS) {
      const int L = lens.i()[b];
      if (L < -1 || (long long)L + n > (long long)blk * nblk) { bad = true; c.fail(KVM_ERR_OP_KVLEN, b, L); }
      else full = full || (L >= 0 && (L + n) / blk > L / blk);
    }
    const int mine = (__ballot(bad) ? 1 : 0) | (__ballot(full) ? 2 : 0);
    if (lane() == 0) word[wave()] = mine;
    __syncthreads();
    const int all = word[0] | word[1] | word[2] | word[3];
    return all & 1 ? -1 : all >> 1;
  }
  // Task p's share [m0, m1) of `full` blocks that become full; p = 0 has the first one in any case.
  __device__ void share(int full, int& m0, int& m1) const {
    const int per = (int)((unsigned)(full + P - 1) / (unsigned)P);
    m0 = (int)min((long long)p * per, (long long)full); m1 = min(m0 + per, full);
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

// KV append in 8 bits, any alignment and head size (16-byte vectors need aligned rows and 64 or 128 dims; this form is the plain one,
// 4,001 tokens of 8 heads of 96 dims 175 us where 128 dims take 32): token by token into an f32 copy of the block in LDS, which is quantised
// when it is full and stored to the tail otherwise.
__device__ __noinline__ void op_kv_append_q8(const Ctx& c) {
  const AppendQ8 A(c);
  if (A.lengths(c, (LDS int*)c.smem) < 0) return;
  LDS float* x = (LDS float*)c.smem;                                   // [blk][hd], one of K and V at a time
  LDS float* red = x + 128 * 128;
  LDS float* row = red + 16;
  for (int b = A.b0; b < A.b1; ++b) {
    const int L = A.lens.i()[b];
    if (L < 0) continue;
    const int j0 = L / A.blk, jE = (L + A.n) / A.blk;                  // touched blocks j0 .. jE, the last one unfinished
    int m0, m1;
    A.share(jE - j0, m0, m1);
    for (int h = A.h0; h < A.h1; ++h) {
      const long long pair = (long long)b * A.Hkv + h;
      for (int which = 0; which < 2; ++which) {
        const View& src = which ? A.vn : A.kn; const View& tail = which ? A.vt : A.kt;
        const View& Q = which ? A.vq : A.kq; const View& SC = which ? A.vs : A.ks;
        // task 0: the first block (it may hold older tokens) among its share, then the unfinished one (its rows in the tail are read
        // before they are overwritten)
        for (int u = m0; u < m1 + (A.p == 0); ++u) {
          const int j = u < m1 ? j0 + u : jE;
          const bool full = j < jE;
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
// A full block is in registers as a whole, all its loads requested before any is used, K and V together with one reduction of both
// maxima (of the largest blocks one after the other: their registers would be most of a worker's scratch). Keys to be normalised or
// rotated go through LDS first, row by row. Keys are stored as they lie, 8 bytes a lane; values turn through LDS. One token of a
// sequence: 4 us a task, 5 with norm and rotation; a block of 64 tokens of 128 dims: 6 us, 8 with them.
template <int HD> struct AppendLds {
  LDS double* freq; LDS float* red; LDS float* keys; LDS float* angs; LDS unsigned char* turn;
  __device__ explicit AppendLds(LDS char* p)
      : freq((LDS double*)p), red((LDS float*)(freq + HD / 2)), keys(red + 16), angs(keys + 128 * HD), turn((LDS unsigned char*)(angs + KVM_THREADS * 8)) {}
};
template <int HD, int NP> __device__ __noinline__ void append_q8_blocks(const Ctx& c) {
  constexpr int LPR = HD / 8, RPP = KVM_THREADS / LPR;                 // lanes a row, rows a pass; NP passes hold a block
  constexpr int NX = NP > 4 ? 1 : 2;                                   // K and V at once, blocks of more than four passes one after the other
  const AppendQ8 A(c);
  const AppendLds<HD> M(c.smem);                                       // keys [blk][HD], turn [HD][blk + 4]
  const int ln = tid() % LPR, rw = tid() / LPR, blk = A.blk;
  const GLOBAL float* gamma = A.kg.ok() ? A.kg.f() : nullptr;
  const LDS double* rot = A.theta > 0.f ? M.freq : nullptr;
  const bool turned = gamma || rot, kround = A.kt.dtype == 2 && (turned || A.kn.dtype != 2), vround = A.vt.dtype == 2 && A.vn.dtype != 2, nkh = A.kn.dtype == 2, nvh = A.vn.dtype == 2, tkh = A.kt.dtype == 2, tvh = A.vt.dtype == 2;
  const int nh = A.h1 - A.h0;
  for (int u = 0; u < (A.b1 - A.b0) * nh; ++u) {
    const int b = A.b0 + u / nh, h = A.h0 + u % nh, L = rfl(A.lens.i()[b]);
    if (L < 0) continue;
    const long long pair = (long long)b * A.Hkv + h;
    const int lb = 31 - __clz(blk), j0 = L >> lb, jE = (L + A.n) >> lb;
    int m0, m1;
    A.share(jE - j0, m0, m1);
    for (int j = j0 + m0; j < j0 + m1; ++j) {
      const int old = max(0, L - j * blk);            // rows below `old` are in the tail
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
#pragma unroll 1
      for (int x0 = 0; x0 < 2; x0 += NX) {
        Raw8 raw[NX][NP];
        float v[NX][NP][8], scale[NX], inv[NX];
        auto of = [&](int x, const View& k, const View& w) { return NX == 2 ? (x ? w : k) : (x0 ? w : k); };   // of K or of V
#pragma unroll
        for (int x = 0; x < NX; ++x) {
          const View tl = of(x, A.kt, A.vt), nw = of(x, A.kn, A.vn);
          if ((NX == 2 ? x : x0) == 0 && turned) continue;
#pragma unroll
          for (int i = 0; i < NP; ++i) {
            const int r = i * RPP + rw;
            if (r >= blk) break;
            raw[x][i].load(r < old ? tl : nw, r < old ? (tail0 + r) * tl.cols + 8 * ln : (new0 + r) * nw.cols + h * HD + 8 * ln);
          }
        }
#pragma unroll
        for (int x = 0; x < NX; ++x) {
          const bool key = (NX == 2 ? x : x0) == 0, round = key ? kround : vround, th = key ? tkh : tvh, nh_ = key ? nkh : nvh;
          uint32_t big = 0;                                            // largest magnitude by its bits: what is not finite is largest
#pragma unroll
          for (int i = 0; i < NP; ++i) {
            const int r = i * RPP + rw;
            if (r >= blk) break;
            if (key && turned) {
#pragma unroll
              for (int e = 0; e < 8; ++e) v[x][i][e] = M.keys[r * HD + 8 * ln + e];     // this thread's own
            } else raw[x][i].get(r < old ? th : nh_, v[x][i]);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              if (round) v[x][i][e] = round_bf(v[x][i][e]);
              big = max(big, __float_as_uint(v[x][i][e]) & 0x7fffffffu);
            }
          }
          scale[x] = rows_max(lanes_max<16>(__uint_as_float(min(big, 0x7f800000u))));
        }
        __syncthreads();                                               // the block before is out of `turn` and `red`
#pragma unroll
        for (int x = 0; x < NX; ++x) if (lane() == 0) M.red[4 * x + wave()] = scale[x];
        __syncthreads();
#pragma unroll
        for (int x = 0; x < NX; ++x) {
          const LDS float* m = M.red + 4 * x;
          scale[x] = q8_scale(fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])));
          inv[x] = scale[x] > 0.f ? 1.f / scale[x] : 0.f;
          const View sc = of(x, A.ks, A.vs);
          if (tid() == 0) stwt32(sc.f() + (pair * sc.cols + j), scale[x]);
        }
        const long long byte0 = (pair * A.nblk + j) * blk * HD;
        const __amdgpu_buffer_rsrc_t ok = wt_rsrc((const char*)A.kq.p + byte0, blk * HD), ov = wt_rsrc((const char*)A.vq.p + byte0, blk * HD);
#pragma unroll
        for (int x = 0; x < NX; ++x) {
          const bool key = (NX == 2 ? x : x0) == 0;
#pragma unroll
          for (int i = 0; i < NP; ++i) {
            const int r = i * RPP + rw;
            if (r >= blk) break;
            uint32_t w0, w1;
            q8_pack(v[x][i], scale[x], inv[x], w0, w1);
            if (key) __builtin_amdgcn_raw_buffer_store_b64(u32x2_t{w0, w1}, ok, r * HD + 8 * ln, 0, 16 /* SC1 */);
            else {
              LDS unsigned char* col = M.turn + 8 * ln * (blk + 4) + r;
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                col[e * (blk + 4)] = (unsigned char)(w0 >> (8 * e));
                col[(4 + e) * (blk + 4)] = (unsigned char)(w1 >> (8 * e));
              }
            }
          }
        }
        if (NX == 1 && x0 == 0) continue;
        __syncthreads();
        for (int e = tid(); e < HD * blk / 16; e += KVM_THREADS) {
          const LDS uint32_t* w = (const LDS uint32_t*)(M.turn + (16 * e >> lb) * (blk + 4) + (16 * e & (blk - 1)));
          stwt_buf(ov, 16 * e, __builtin_bit_cast(f32x4n, u32x4_t{w[0], w[1], w[2], w[3]}));
        }
      }
    }
  }
}
template <int HD> __device__ __forceinline__ void append_q8_t(const Ctx& c) {
  constexpr int LPR = HD / 8, RPP = KVM_THREADS / LPR;
  const AppendQ8 A(c);
  const AppendLds<HD> M(c.smem);
  const int full = A.lengths(c, (LDS int*)M.red);
  if (full < 0) return;
  const int ln = tid() % LPR, rw = tid() / LPR, blk = A.blk, nh = A.h1 - A.h0;
  const GLOBAL float* gamma = A.kg.ok() ? A.kg.f() : nullptr;
  const LDS double* rot = A.theta > 0.f ? M.freq : nullptr;
  if (rot && tid() < HD / 2) M.freq[tid()] = q8_freq(tid(), HD, log((double)A.theta));
  __syncthreads();
  if (full) {
    if (blk <= 4 * RPP) append_q8_blocks<HD, 4>(c);
    else append_q8_blocks<HD, 128 / RPP>(c);
  }
  if (A.p != 0) return;
  __syncthreads();                                                     // old rows of the tail have been read
  const int most = min(A.n, blk - 1), rows = (A.b1 - A.b0) * nh * most;   // rows of an unfinished block: no more than that
  constexpr int NR = 4;                                                // rows in flight
  for (int u0 = rw; u0 < rows; u0 += NR * RPP) {
    Raw8 rk[NR], rv[NR];
    long long t[NR] = {-1, -1, -1, -1}, at[NR];
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      const int u = u0 + i * RPP;
      if (u >= rows) break;
      const int b = A.b0 + u / (nh * most), h = A.h0 + u / most % nh, L = A.lens.i()[b];
      const long long x = max((long long)L, (long long)((L + A.n) & -blk)) + u % most, row = (long long)b * A.n + (x - L);
      if (L < 0 || x >= (long long)L + A.n) continue;
      t[i] = x; at[i] = ((long long)b * A.Hkv + h) * blk + (x & (blk - 1));
      rk[i].load(A.kn, row * A.kn.cols + h * HD + 8 * ln);
      rv[i].load(A.vn, row * A.vn.cols + h * HD + 8 * ln);
    }
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      if (t[i] < 0) continue;
      float k[8], v[8];
      rk[i].get(A.kn.dtype == 2, k); rv[i].get(A.vn.dtype == 2, v);
      if (gamma || rot) head8_turn<HD>(k, gamma, A.eps, rot, t[i], M.angs + rw * HD);
      st8(A.kt, at[i] * A.kt.cols + 8 * ln, k);
      st8(A.vt, at[i] * A.vt.cols + 8 * ln, v);
    }
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
      : q(uview(c, 0)), kq(uview(c, 1)), ks(uview(c, 2)), vq(uview(c, 3)), vs(uview(c, 4)), kt(uview(c, 5)), vt(uview(c, 6)), lens(uview(c, 7)), part(uview(c, 8)), o(uview(c, 9)),
        cnt(uview(c, 10)), qg(uview(c, 11)), b0(rfl(c.i(12))), b1(rfl(c.i(13))), s(rfl(c.i(14))), S(rfl(c.i(15))), n(rfl(c.i(16))), H(rfl(c.i(17))), Hkv(rfl(c.i(18))), hd(rfl(c.i(19))), blk(rfl(c.i(20))),
        scale(c.f(21)), theta(c.f(22)), eps(c.f(23)) { G = H / Hkv; R = n * G; }
  __device__ long long at(const View& X, int b, int h, int r) const { return ((long long)b * n + r / G) * X.cols + (h * G + r % G) * hd; }
  __device__ bool length_ok(const Ctx& c, int b, int L) const {
    if (L >= -1 && (long long)L + n <= (long long)blk * ks.cols) return true;
    c.fail(KVM_ERR_OP_KVLEN, b, L);
    return false;
  }
  __device__ void zeros(int b, int h) const { for (int e = tid(); e < R * hd; e += KVM_THREADS) o.st(at(o, b, h, e / hd) + e % hd, 0.f); }
};

// Decode attention over the 8-bit cache, any alignment and head size (a byte a load: 24 sequences of up to 4,096 tokens 2.6 ms at 96
// dims, 62 us at 128): whole pairs, every S-th one; 256 tokens at a time, a thread
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
  bool bad = false;                                                    // all lengths of the call are checked before anything is written
  for (int b = D.b0 + tid(); b < D.b1; b += KVM_THREADS) bad = bad || !D.length_ok(c, b, D.lens.i()[b]);
  if (__syncthreads_or(bad)) return;
  for (int p = D.s; p < (D.b1 - D.b0) * D.Hkv; p += D.S) {
    const int b = D.b0 + p / D.Hkv, h = p % D.Hkv, L = D.lens.i()[b];
    if (L == -1) D.zeros(b, h);
    else attn_q8_pair(c, D, b, h, L);
  }
}

// ---- The work of a call over its tasks: every pair costs Q8_PAIR (query rows, the unfinished block, the end) and one per unit of 64
// tokens of its whole blocks; the pairs in order, by sequence and head, are cut into equal shares, in the tasks alike from the
// lengths. A cut within Q8_SNAP of a pair's end moves there: a small piece costs more than it balances. A pair that is cut has one piece in
// each of consecutive tasks; the first has the unfinished block.
// Measured (pair, snap, smallest share), us of a launch in a row of them: one sequence of 32,000 tokens 38 (12, 14, 16), 44 (8, 12, 24),
// 45 (16, 20, 32), 59 (24, 28, 56); 24 sequences of up to 4,096 tokens 57, 60, 61, 65; 6 sequences of 1,531, four tokens each 30, 32, 31, 30.
constexpr int Q8_PAIR = 12, Q8_SNAP = 14, Q8_SHARE = 16, Q8_SEQS = 1024;
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
// Inclusive sum over the lanes of a wave: within rows of 16, then the rows' last sums.
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
  return v;
}
// Lengths and cost sums of the call's sequences into LDS; false if a length is out of range (reported). Up to 64 sequences by every wave
// for itself (the same words from all four, no barrier), more by the workgroup.
__device__ __forceinline__ bool q8_work(const Ctx& c, const DecodeQ8& D, LDS int* pre, LDS int* len, LDS int* tot, WorkQ8& W) {
  constexpr int PER = Q8_SEQS / KVM_THREADS;
  const int seqs = D.b1 - D.b0;
  auto cost_of = [&](int L) { return L < 0 ? 1 : Q8_PAIR + (int)(((((unsigned)L + D.n) & -(unsigned)D.blk) + 63) >> 6); };
  if (seqs <= 64) {
    const int L = lane() < seqs ? D.lens.i()[D.b0 + lane()] : -1;
    if (__ballot(lane() < seqs && !D.length_ok(c, D.b0 + lane(), L))) return false;
    const int cost = lane() < seqs ? cost_of(L) : 0, upto = wave_scan(cost);
    if (lane() < seqs) { len[lane()] = L; pre[lane()] = upto - cost; }
    if (lane() == seqs - 1) pre[seqs] = upto;
    wave_sync();
  } else {
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
        cost[i] = cost_of(L);
        sum += cost[i];
      }
    }
    const int upto = wave_scan(sum);
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
  }
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

// Decode attention over the 8-bit cache at head sizes 64 and 128, on the matrix units. Bound: streaming the cache's bytes, and
// where few workers stream at once the 415 vector instructions and 56 products of a unit. 128 sequences of 8,000 tokens, 8 kv heads
// of 128: 2.1 GB in 470 us (4.5 TB/s, a copy reaches 4.8). A piece costs 9 to 12 us beside its units (dependent loads: lengths, rows,
// first unit; the unfinished block; the waves' sum), a unit about 0.5.
// Each wave takes units of 64 tokens in turn, K and V straight from memory into registers in the layout of the operands, one to two
// units ahead:
//   scores  v_mfma_i32_16x16x64_i8, A = 16 keys as they lie, B = up to 16 query rows (NT such tiles) as three signed bytes of a
//           fixed-point number per value (22 bits below a power of two above the row's largest): whole numbers, summed exactly.
//           A lane's 16-byte load of a key is its part of the operand.
//   P V     v_mfma_f32_16x16x32_f16, A = V transposed (16 head dims x 32 tokens: the cache keeps a block's values as [hd][blk], so
//           this too is a 16-byte load), B = P. Tokens go to the rows of the score tiles (row m of tile a: token 16 (m / 4) + 4 a +
//           m % 4) such that the scores' output registers are the B operand, in the loads' order.
// A byte of V becomes an f16 by two instructions for two of them (0x6400 | (v + 128) is 1024 + v + 128), exactly. Probabilities are
// f16 pairs, the value and its remainder, two products each, summed in f32. A block's key scale multiplies its scores; its value
// scale the probabilities, and the pairs hold these products relative to a power of two above the row's largest so far (vtop, which
// shrinks with the row's running maximum; the running P V is in its units), times 2^12: 22 bits of a product, none closer than 2^-36
// of the largest. (Relative to the largest scale alone, a block without weight left 12 bits of the others at scales 2^26 apart and
// nothing at 2^36.) Each unit's P V is summed on its own and added to the running one in f32 (the units' chained sums round
// towards -inf). The unfinished block, at most blk - 1 tokens, is f32 work
// of all lanes (a wave to a row, the tail in its registers and no barrier, was 15 us slower for 24 ragged sequences).
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
template <int HD> struct KeysQ8 { u32x4_t k[4][HD / 64]; float s; };
template <int HD> struct ValuesQ8 { u32x4_t v[HD / 16]; float s; };
// LDS of a task. The work stays through its pieces; the tail's scores and values give way to the waves' P V.
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
        ts(cr + 32),                                                   // [32][128] the tail's scores; before, the rows' angles
        tv(ts + 32 * 128) {}                                           // [128][HD] its values
  static_assert((2 * Q8_SEQS + 4 + HD + 32 * (HD + 4) + 32 * HD + 352 + 32 * 128 + 128 * HD) * 4 <= KVM_LDS_BYTES, "decode attention LDS map");
};
// One piece of a pair: units [u0, u1), with `first` also the unfinished block; `live` pieces in all, piece 1 in task i0's partials.
template <int HD, int NT> __device__ __noinline__ void attn_q8_piece(const Ctx& c, int b_, int kvh_, int L_, int u0_, int u1_, bool first_, int i0_, int live_) {
  const int b = rfl(b_), kvh = rfl(kvh_), L = rfl(L_), u0 = rfl(u0_), u1 = rfl(u1_), i0 = rfl(i0_), live = rfl(live_);
  const bool first = rfl(first_) != 0;
  constexpr float LOG2E = 1.44269504088896340736f, PS = 4096.f;
  constexpr int KH = HD / 64, VT = HD / 16, LPR = HD / 8, RPP = KVM_THREADS / LPR, QS = HD + 4;
  const DecodeLds<HD> M(c.smem);
  LDS float *const qs = M.qs, *const to = M.to, *const st = M.st, *const cr = M.cr, *const ts = M.ts, *const tv = M.tv;
  const DecodeQ8 D(c);
  const int blk = D.blk, lb = 31 - __clz(blk), n = L + D.n, whole = n & -blk, nt = first ? n - whole : 0;
  const bool tail = nt > 0;
  const int l = lane(), w = rfl(wave()), nn = l & 15, qq = l >> 4, ln = tid() % LPR, rw = tid() / LPR;
  const long long pair = (long long)b * D.Hkv + kvh, byte0 = pair * D.ks.cols * blk * HD;
  const GLOBAL char* K = (const GLOBAL char*)D.kq.p + byte0;
  const GLOBAL char* V = (const GLOBAL char*)D.vq.p + byte0;
  const GLOBAL float* KS = D.ks.f() + pair * D.ks.cols;
  const GLOBAL float* VS = D.vs.f() + pair * D.vs.cols;
  // (tokens past the last whole block: the last ones again, masked later)
  auto load_keys = [&](KeysQ8<HD>& U, int u) {
    const int t0 = u << 6, rest = whole - t0;
    const GLOBAL char* kb = K + (long long)t0 * HD;
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
      for (int h = 0; h < KH; ++h) U.k[a][h] = *(const GLOBAL u32x4a4*)(kb + (min(16 * (nn >> 2) + 4 * a + (nn & 3), rest - 1) * HD + 16 * (qq + 4 * h)));
    U.s = KS[(t0 + min(16 * qq, rest - 16)) >> lb];
  };
  auto load_values = [&](ValuesQ8<HD>& U, int u) {
    const int t0 = u << 6, tt = (t0 & (blk - 1)) + min(16 * qq, whole - t0 - 16), j = tt >> lb;   // from the start of the block of t0
    const GLOBAL char* vb = V + ((long long)(t0 >> lb) << lb) * HD;
    const int at = j * blk * HD + (tt & (blk - 1)) + nn * blk;
#pragma unroll
    for (int d = 0; d < VT; ++d) U.v[d] = *(const GLOBAL u32x4a4*)(vb + (at + 16 * d * blk));
    U.s = VS[(t0 >> lb) + j];
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
  constexpr int NK = NT * HD > 128 ? 1 : 2;                            // units of keys under way; two tiles of 128 have registers for one
  KeysQ8<HD> keys[NK];
  ValuesQ8<HD> U;
  if (u0 + w < u1) { load_keys(keys[0], u0 + w); load_values(U, u0 + w); }
  if (NK > 1 && u0 + w + KVM_WAVES < u1) load_keys(keys[NK - 1], u0 + w + KVM_WAVES);
  if (D.theta > 0.f && tid() < HD / 2) M.freq[tid()] = q8_freq(tid(), HD, log((double)D.theta));
  __syncthreads();                                                     // frequencies; the work and the piece before are out of LDS
  // query rows: norm, rotation, then scaled by a power of two to magnitudes below 2^22
#pragma unroll
  for (int i = 0; i < QP; ++i) {
    const int r = i * RPP + rw;
    if (r >= 16 * NT) break;
    float x[8] = {};
    if (r < D.R) {
      rq[i].get(D.q.dtype == 2, x);
      head8_turn<HD>(x, D.qg.ok() ? D.qg.f() : nullptr, D.eps, D.theta > 0.f ? M.freq : nullptr, L + r / D.G, ts + rw * HD);
    }
    uint32_t big = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) big = max(big, __float_as_uint(x[e]) & 0x7fffffffu);
    const float top = lanes_max<LPR>(__uint_as_float(min(big, 0x7f800000u)));
    const int ex = max(24, (int)(__float_as_uint(top) >> 23));
    const float up = __uint_as_float((uint32_t)(275 - ex) << 23), down = __uint_as_float((uint32_t)(ex - 21) << 23);
#pragma unroll
    for (int e = 0; e < 8; ++e) qs[r * QS + 8 * ln + e] = top < INFINITY ? x[e] * up : 0.f;
    if (ln == 0) cr[r] = top < INFINITY ? down * D.scale * LOG2E : __uint_as_float(0x7fc00000u);   // a row that is not finite is NaN
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
      for (int r0 = 0; r0 < D.R; r0 += 4) {
        float a[4][TP];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float q[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) q[e] = qs[min(r0 + k, D.R - 1) * QS + 8 * ln + e];
#pragma unroll
          for (int i = 0; i < TP; ++i) {
            a[k][i] = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) a[k][i] += q[e] * x[i][e];
          }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int i = 0; i < TP; ++i) a[k][i] = lanes_sum<LPR>(a[k][i]);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int r = r0 + k, seen = min(nt, L + r / D.G + 1 - whole);
          const float f = cr[min(r, D.R - 1)];
#pragma unroll
          for (int i = 0; i < TP; ++i) {
            const int t = t0 + i * RPP + rw;
            if (ln == 0 && t < nt && r < D.R) ts[r * 128 + t] = t < seen ? a[k][i] * f : -INFINITY;
          }
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
  // the queries as B operands: row nn of tile g, dims 64 h + 16 qq .., byte p of the fixed-point numbers
  // (two tiles keep them in LDS, over the tail's scores: the same from every wave)
  i32x4_t qb[NT == 1 ? KH : 1][3];
  LDS i32x4_t* ql = (LDS i32x4_t*)ts + l;                              // [NT][KH][3][64]
  auto query = [&](int g, int h, int p) { return NT == 1 ? qb[NT == 1 ? h : 0][p] : ql[((g * KH + h) * 3 + p) * 64]; };
  if (NT > 1 && tail) __syncthreads();                                 // the scores have been read
  float mrun[NT], lrun[NT], crow[NT], vtop[NT];                        // vtop: largest probability times value scale so far
  int lim[NT];
  f32x4n o[NT][VT];
#pragma unroll
  for (int g = 0; g < NT; ++g) {
    const int r = 16 * g + nn;
#pragma unroll
    for (int h = 0; h < KH; ++h) {
      i32x4_t q[3];
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        uint32_t y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = ((uint32_t)(int)rintf(qs[r * QS + 64 * h + 16 * qq + 4 * v + e]) + 0x808080u) ^ 0x808080u;
        const uint32_t a01 = __builtin_amdgcn_perm(y[1], y[0], 0x05010400u), a23 = __builtin_amdgcn_perm(y[3], y[2], 0x05010400u);
        q[0][v] = (int)__builtin_amdgcn_perm(a23, a01, 0x05040100u);
        q[1][v] = (int)__builtin_amdgcn_perm(a23, a01, 0x07060302u);
        q[2][v] = (int)__builtin_amdgcn_perm(__builtin_amdgcn_perm(y[3], y[2], 0x0c0c0602u), __builtin_amdgcn_perm(y[1], y[0], 0x0c0c0602u), 0x05040100u);
      }
#pragma unroll
      for (int p = 0; p < 3; ++p) { if (NT == 1) qb[h][p] = q[p]; else ql[((g * KH + h) * 3 + p) * 64] = q[p]; }
    }
    crow[g] = cr[r]; mrun[g] = -INFINITY; lrun[g] = vtop[g] = 0.f;
    lim[g] = r < D.R ? min(whole, L + r / D.G + 1) : 0;
#pragma unroll
    for (int d = 0; d < VT; ++d) o[g][d] = f32x4n{0.f, 0.f, 0.f, 0.f};
  }
  auto above = [](float x) { return __uint_as_float((__float_as_uint(x) & 0x7f800000u) + 0x00800000u); };   // a power of two, and 1 / it
  auto one_over = [](float p) { return __uint_as_float(0x7f000000u - __float_as_uint(p)); };
  // one unit, its keys in C: the keys of this wave's unit after the next (of its next) are requested into C once the scores are there,
  // the next unit's values once the P V is
  auto unit = [&](int u, KeysQ8<HD>& C) {
    float sc[NT][16];
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      i32x4_t s[NT][3];
#pragma unroll
      for (int g = 0; g < NT; ++g)
#pragma unroll
        for (int p = 0; p < 3; ++p) s[g][p] = i32x4_t{0, 0, 0, 0};
#pragma unroll
      for (int h = 0; h < KH; ++h)
#pragma unroll
        for (int g = 0; g < NT; ++g)
#pragma unroll
          for (int p = 0; p < 3; ++p) s[g][p] = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4_t, C.k[a][h]), query(g, h, p), s[g][p], 0, 0, 0);
#pragma unroll
      for (int g = 0; g < NT; ++g)
#pragma unroll
        for (int i = 0; i < 4; ++i) sc[g][4 * a + i] = fmaf((float)((s[g][2][i] << 8) + s[g][1][i]), 256.f, (float)s[g][0][i]) * (crow[g] * C.s);
    }
    if (u + NK * KVM_WAVES < u1) load_keys(C, u + NK * KVM_WAVES);
    const bool all = 64 * (u + 1) <= min(whole, L + 1);                // every row sees every token
    f16x8 ph[NT][2], pl[NT][2];
    float fo[NT];
#pragma unroll
    for (int g = 0; g < NT; ++g) {
      float sg = U.s, ml = -INFINITY;
      if (!all) {
        const int seen = lim[g] - 64 * u - 16 * qq;                    // of this lane's 16 tokens, which lie in one block
#pragma unroll
        for (int i = 0; i < 16; ++i) sc[g][i] = i < seen ? sc[g][i] : -INFINITY;
        sg = seen > 0 ? sg : 0.f;                                      // the scale of a block that is not seen does not count, NaN neither
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) ml = fmaxf(ml, sc[g][i]);
      const float m = rows_max(fmaxf(mrun[g], ml));
      const float base = m == -INFINITY ? 0.f : m;                     // nothing seen yet (or NaN, which stays)
      const float f = __builtin_amdgcn_exp2f(mrun[g] - base), el = __builtin_amdgcn_exp2f(ml - base);
      sg = el > 0.f ? sg : 0.f * sg;                                   // no weight: the scale does not count (but NaN)
      const float top = fmaxf(vtop[g] * f, rows_max(fmaxf(el, 0x1p-112f) * sg));   // (2^-112: sg / top stays below 2^113)
      const float pg = sg * one_over(above(top)) * PS;
      float z = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float e = __builtin_amdgcn_exp2f(sc[g][i] - base), x = e * pg;
        z += e;
        const _Float16 hi = (_Float16)x;
        ph[g][i / 8][i % 8] = hi; pl[g][i / 8][i % 8] = (_Float16)(x - (float)hi);
      }
      lrun[g] = lrun[g] * f + z;
      mrun[g] = m;
      fo[g] = f * above(vtop[g]) * one_over(above(top));
      vtop[g] = top;
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
    if (u + KVM_WAVES < u1) load_values(U, u + KVM_WAVES);
  };
  for (int u = u0 + w; u < u1; u += NK * KVM_WAVES) {
    unit(u, keys[0]);
    if (NK > 1 && u + KVM_WAVES < u1) unit(u + KVM_WAVES, keys[NK - 1]);
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
        for (int i = 0; i < 4; ++i) ow[(w * D.R + r) * HD + 16 * d + 4 * qq + i] = o[g][d][i] * (1.f / PS) * above(vtop[g]);
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
  if (D.b0 == D.b1 || !q8_work(c, D, M.pre, M.len, (LDS int*)M.st, W)) return;
  const int stop = W.cut(D.s + 1);
  for (int at = W.cut(D.s); at < stop;) {
    const WorkQ8::At P = W.find(at);
    const int off = at - P.start, end = min(P.cost, stop - P.start), L = rfl(M.len[P.b]), b = D.b0 + P.b;
    at = P.start + end;
    if (L < 0) { D.zeros(b, P.h); continue; }
    const bool cut = off > 0 || end < P.cost;
    const int u0 = max(0, off - Q8_PAIR), u1 = max(0, end - Q8_PAIR), i0 = cut ? W.first_inside(P) : 0, live = cut ? W.inside(P) + 1 : 1;
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
// Adjusted logits (op 314). Bound: the bytes of the logits, and per task the history, which every task of a row reads as a whole (a few
// KB, from the L2). The task's logits go through as a stream that knows only the mask, in vectors of 4 from any element (a bf16
// row from its first aligned one), NB of a thread requested ahead (64 KB of f32, 32 KB of bf16), each again as soon as it is stored;
// vectors of 8 bf16 logits have stores of 16 bytes 32 apart, 7 us more for a task of 50,257 logits. Rows in place without a mask
// have no stream.
// The few tokens that the history or the biases name meet in LDS, one word each (generated: bits 0..19, bias slot: bits 20..30,
// prompt: bit 31), before the first vectors of the stream have come; behind the stream their logits are written again, each once, four
// of a thread in flight. The words lie at the tokens themselves where the range fits (22,528 logits) and are taken out of there by an
// exchange against 0 into a list; a longer range has them in an open-addressed table while it names at most 6,144 tokens, and is
// done in chunks otherwise: 256 rows of 50,257 bf16 logits, 777 tokens each, 31 us in three chunks, 25 with the table (tasks alone).
// A token's entries in the bias list meet by an atomic maximum of (2047 - entry), which leaves the slot of the first; the others are
// added to it in list order, one after another (they are few). Adjusting in the stream itself ran its divisions for every wave that
// met one named token: a task of 50,257 logits 47 us, now 22.
constexpr int ADJ_CHUNK = 22528, ADJ_BIAS = 2047, ADJ_LIST = 2048, ADJ_SLOTS = 8192, ADJ_NAMED = 6144;
struct AdjustArgs {
  View x, out, par, hist, plen, hlen, last, bidx, bval, mask, mrow;
  int r0, r1, v0, v1, V;
  __device__ explicit AdjustArgs(const Ctx& c)
      : x(uview(c, 0)), out(uview(c, 1)), par(uview(c, 2)), hist(uview(c, 3)), plen(uview(c, 4)), hlen(uview(c, 5)), last(uview(c, 6)), bidx(uview(c, 7)), bval(uview(c, 8)),
        mask(uview(c, 9)), mrow(uview(c, 10)), r0(rfl(c.i(11))), r1(rfl(c.i(12))), v0(rfl(c.i(13))), v1(rfl(c.i(14))), V(rfl(c.i(15))) {}
  __device__ bool row_ok(const Ctx& c, int r, int n, int pl, int m) const {
    if (n < 0 || pl < 0 || pl > n || (hist.ok() && n + (last.ok() ? 1 : 0) > hist.cols)) { c.fail(KVM_ERR_OP_RANGE, r, n); return false; }
    if (mrow.ok() && (m < -1 || m >= mask.rows)) { c.fail(KVM_ERR_OP_RANGE, r, m); return false; }
    return true;
  }
  // All rows of a task are checked before anything is written (a single one when it is read).
  __device__ bool rows_ok(const Ctx& c) const {
    bool bad = false;
    for (int r = r0 + tid(); r < r1; r += KVM_THREADS)
      bad = bad || !row_ok(c, r, hist.ok() ? hlen.i()[r] : 0, hist.ok() ? plen.i()[r] : 0, mrow.ok() ? mrow.i()[r] : 0);
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
  LDS uint32_t* cnt = (LDS uint32_t*)c.smem;                           // [ADJ_CHUNK]
  LDS float* bsum = (LDS float*)(cnt + ADJ_CHUNK);                     // [ADJ_BIAS + 1] an entry's value, the first one's the sum
  LDS int* later = (LDS int*)(bsum + ADJ_BIAS + 1);                    // [ADJ_BIAS + 1] first entry of the same token, or -1
  LDS uint32_t* list = (LDS uint32_t*)(later + ADJ_BIAS + 1);          // [ADJ_LIST][2] tokens and words taken out of cnt, then how many
  LDS int* listed = (LDS int*)(list + 2 * ADJ_LIST);
  // a longer range of a row that names at most ADJ_NAMED tokens: an open-addressed table over cnt, and its slots in use
  LDS uint32_t *keys = cnt, *words = cnt + ADJ_SLOTS, *used = words + ADJ_SLOTS;
  static_assert(2 * ADJ_SLOTS + ADJ_NAMED <= ADJ_CHUNK && ADJ_NAMED < ADJ_SLOTS && (ADJ_SLOTS & (ADJ_SLOTS - 1)) == 0, "logits table");
  static_assert((ADJ_CHUNK + 2 * (ADJ_BIAS + 1) + 2 * ADJ_LIST + 1) * 4 <= KVM_LDS_BYTES, "logits LDS map");
  constexpr int NH = 4, NB = 16;                                       // vectors of tokens, and of logits, in flight
  const int nb = A.bidx.ok() ? A.bidx.cols : 0, len = A.v1 - A.v0;
  const bool xh = A.x.dtype == 2, oh = A.out.dtype == 2;
  if (A.r1 - A.r0 > 1 && !A.rows_ok(c)) return;
  for (int r = A.r0; r < A.r1 && len > 0; ++r) {
    const float rep = A.par.at(r, 0), freq = A.par.at(r, 1), pres = A.par.at(r, 2);
    const int n = A.hist.ok() ? rfl(A.hlen.i()[r]) : 0, pl = A.hist.ok() ? rfl(A.plen.i()[r]) : 0, last = A.last.ok() ? rfl(A.last.i()[r]) : -1;
    const int mr = A.mask.ok() ? (A.mrow.ok() ? rfl(A.mrow.i()[r]) : r) : -1;
    if (!A.row_ok(c, r, n, pl, mr)) return;
    const GLOBAL int* hist = A.hist.ok() ? A.hist.i() + (long long)r * A.hist.cols : nullptr;
    const GLOBAL int* bidx = nb ? A.bidx.i() + (long long)r * A.bidx.cols : nullptr;
    const GLOBAL float* bval = nb ? A.bval.f() + (long long)r * A.bval.cols : nullptr;
    const GLOBAL int* mask = mr >= 0 ? A.mask.i() + (long long)mr * A.mask.cols : nullptr;
    const bool named = n || nb || last >= 0, table = len > ADJ_CHUNK && n + nb < ADJ_NAMED;
    // The stream: vectors start where bf16 storage is 4-byte aligned, on both sides; rows that never are go one by one.
    const GLOBAL char* xp = (const GLOBAL char*)A.x.p + ((long long)r * A.x.cols + A.v0) * (xh ? 2 : 4);
    const GLOBAL char* op = (const GLOBAL char*)A.out.p + ((long long)r * A.out.cols + A.v0) * (oh ? 2 : 4);
    const int px = xh ? (int)((uintptr_t)xp >> 1) & 1 : 0, po = oh ? (int)((uintptr_t)op >> 1) & 1 : 0;
    const int peel = min(len, max(px, po)), nv = (!mask && A.out.p == A.x.p) || (xh && oh && px != po) ? 0 : (len - peel) / 4;
    u32x4_t x[NB];                                                     // (bf16: the first half)
    uint32_t m0[NB], m1[NB];
    auto request = [&](int u, int base) {
      const int i = peel + 4 * min(base + tid() + u * KVM_THREADS, nv - 1), v = A.v0 + i;
      if (xh) { const u32x2_t t = *(const GLOBAL u32x2a4*)(xp + 2ll * i); x[u].x = t.x; x[u].y = t.y; }
      else x[u] = *(const GLOBAL u32x4a4*)(xp + 4ll * i);
      m0[u] = m1[u] = ~0u;
      if (mask) { m0[u] = mask[v >> 5]; m1[u] = mask[(v + 3) >> 5]; }  // a vector's bits may lie in two words
    };
    // The tokens of this thread, four at a time: of the history, and (fewer than four, and the token chosen last) behind it.
    u32x4_t h[NH];
    auto tokens = [&](int k0) {
#pragma unroll
      for (int u = 0; u < NH; ++u) if (k0 + 4 * u * KVM_THREADS < n / 4 * 4) h[u] = *(const GLOBAL u32x4a4*)(hist + k0 + 4 * u * KVM_THREADS);
    };
    auto visit = [&](auto f) {                                         // f(position, token)
      for (int k0 = 4 * tid(); k0 < n / 4 * 4; k0 += 4 * NH * KVM_THREADS) {
        if (n >= 4 * NH * KVM_THREADS) tokens(k0);                     // else they are there
#pragma unroll
        for (int u = 0; u < NH; ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e) if (k0 + 4 * u * KVM_THREADS < n / 4 * 4) f(k0 + 4 * u * KVM_THREADS + e, (int)h[u][e]);
      }
      const int rest = n / 4 * 4 + tid();
      if (rest <= n) f(rest, rest < n ? hist[rest] : last);
    };
    if (n && n < 4 * NH * KVM_THREADS) tokens(4 * tid());
    for (int c0 = A.v0, most; c0 < A.v1 && (named || c0 == A.v0); c0 += most) {
      most = table ? len : min(len - (c0 - A.v0), ADJ_CHUNK);
      // the word of token c0 + v (a token that is not in the table goes in: its slots are never all in use)
      auto word = [&](uint32_t v) {
        if (!table) return cnt + v;
        uint32_t s = v * 2654435769u >> (32 - __builtin_ctz(ADJ_SLOTS));
        for (;; s = (s + 1) & (ADJ_SLOTS - 1)) {
          uint32_t old = ~0u;
          if (__hip_atomic_compare_exchange_strong(keys + s, &old, v, __ATOMIC_RELAXED, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP)) {
            used[__hip_atomic_fetch_add(listed, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP)] = s;
            break;
          }
          if (old == v) break;
        }
        return words + s;
      };
      if (c0 == A.v0 && nv) {
#pragma unroll
        for (int u = 0; u < NB; ++u) request(u, 0);
      }
      if (named) {                                                     // counts and bias slots of the chunk's tokens
        __syncthreads();
        if (table) {
          for (int i = tid(); i < 2 * ADJ_SLOTS / 4; i += KVM_THREADS) ((LDS u32x4_t*)cnt)[i] = i < ADJ_SLOTS / 4 ? u32x4_t{~0u, ~0u, ~0u, ~0u} : u32x4_t{0, 0, 0, 0};
          if (tid() == 0) *listed = 0;
        } else
          for (int i = tid(); i < (most + 3) / 4; i += KVM_THREADS) ((LDS u32x4_t*)cnt)[i] = u32x4_t{0, 0, 0, 0};
        __syncthreads();
        if (nb) {
          for (int j = tid(); j < nb; j += KVM_THREADS) {
            const int v = bidx[j] - c0;
            bsum[j] = bval[j];
            if (v >= 0 && v < most) __hip_atomic_fetch_max(word(v), (uint32_t)(ADJ_BIAS - j) << 20, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
          }
          __syncthreads();
          bool many = false;
          for (int j = tid(); j < nb; j += KVM_THREADS) {
            const int v = bidx[j] - c0, one = v >= 0 && v < most ? ADJ_BIAS - (int)(*word(v) >> 20) : j;
            later[j] = one == j ? -1 : one;
            many = many || one != j;
          }
          if (__syncthreads_or(many) && wave() == 0)                   // entries of one token, in list order
            for (int j0 = 0; j0 < nb; j0 += 64) {
              const int mine = j0 + lane() < nb ? later[j0 + lane()] : -1;
              for (uint64_t left = __ballot(mine >= 0); left; left &= left - 1) {
                const int j = __ffsll((long long)left) - 1, to = __builtin_amdgcn_readlane(mine, j);
                if (lane() == 0) bsum[to] += bsum[j0 + j];
              }
            }
        }
        visit([&](int k, int t) {
          const unsigned v = (unsigned)(t - c0);
          if (t < 0 || v >= (unsigned)most) return;
          LDS uint32_t* w = word(v);
          if (k < pl) lds_or(w, 0x80000000u);
          else __hip_atomic_fetch_add(w, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
        });
      }
      if (c0 == A.v0 && (mask || A.out.p != A.x.p)) {
        for (int base = 0; base < nv; base += NB * KVM_THREADS) {
          // a descriptor for the round's vectors: what lies past the last one is out of its range and not stored
          const __amdgpu_buffer_rsrc_t ro = wt_rsrc((const char*)op + (peel + 4ll * base) * (oh ? 2 : 4), (long long)min(4 * NB * KVM_THREADS, 4 * (nv - base)) * (oh ? 2 : 4));
#pragma unroll
          for (int u = 0; u < NB; ++u) {
            const int i = 4 * (tid() + u * KVM_THREADS);
            const uint32_t bits = (uint32_t)((((uint64_t)m1[u] << 32) | m0[u]) >> ((A.v0 + peel + 4 * base + i) & 31));
            f32x4n y;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              y[e] = __uint_as_float(!xh ? x[u][e] : e & 1 ? x[u][e / 2] & 0xffff0000u : x[u][e / 2] << 16);
              if (!((bits >> e) & 1)) y[e] = -INFINITY;
            }
            if (oh) stwt_bf4_buf(ro, 2 * i, y); else stwt_buf(ro, 4 * i, y);
            if (base + NB * KVM_THREADS < nv) request(u, base + NB * KVM_THREADS);
          }
        }
        for (int k = tid(); k < len - 4 * nv; k += KVM_THREADS) {       // before the first vector and behind the last
          const int v = A.v0 + (k < peel ? k : k + 4 * nv);
          A.out.st((long long)r * A.out.cols + v, !mask || ((mask[v >> 5] >> (v & 31)) & 1) ? A.x.at(r, v) : -INFINITY);
        }
      }
      // The named tokens again, each once: the table's, or those taken out of the counts (what the list cannot hold stays for a next round).
      for (bool more = named; more;) {
        wait_stores();                                                 // the stream's values of these logits are out
        if (!table && tid() == 0) *listed = 0;
        __syncthreads();
        if (!table) {
          auto take = [&](int t) {
            const unsigned v = (unsigned)(t - c0);
            if (t < 0 || v >= (unsigned)most) return;
            const uint32_t w = __hip_atomic_exchange(&cnt[v], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
            if (!w) return;
            const int k = __hip_atomic_fetch_add(listed, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
            if (k < ADJ_LIST) { list[2 * k] = v; list[2 * k + 1] = w; }
            else __hip_atomic_store(&cnt[v], w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
          };
          visit([&](int, int t) { take(t); });
          for (int j = tid(); j < nb; j += KVM_THREADS) take(bidx[j]);
          __syncthreads();
        }
        const int found = table ? *listed : min(*listed, ADJ_LIST);
        more = !table && *listed > ADJ_LIST;
        for (int k0 = tid(); k0 < found; k0 += 4 * KVM_THREADS) {      // four logits of a thread in flight
          float z[4];
          uint32_t m[4], w[4];
          int t[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int k = min(k0 + i * KVM_THREADS, found - 1);
            const uint32_t s = table ? used[k] : 0;
            t[i] = c0 + (int)(table ? keys[s] : list[2 * k]); w[i] = table ? words[s] : list[2 * k + 1];
            z[i] = A.x.at(r, t[i]); m[i] = mask ? (uint32_t)mask[t[i] >> 5] : ~0u;
          }
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (k0 + i * KVM_THREADS < found) A.out.st((long long)r * A.out.cols + t[i], (m[i] >> (t[i] & 31)) & 1 ? adjusted(z[i], w[i], rep, freq, pres, bsum) : -INFINITY);
        }
        if (more) __syncthreads();
      }
    }
    if (A.last.ok() && A.v0 == 0 && tid() == 0) stwt32i(A.hist.i() + ((long long)r * A.hist.cols + n), last);
  }
}

}  // namespace kvm
