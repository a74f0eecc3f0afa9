// A KV cache in pages: append of new tokens with head norm and rotation (op 318) and their attention (op 319). Semantics: mvm_ops_kvm.def.
#pragma once
#include "common.h"
#include "ops_basic.h"
#include "ops_attn.h"
#include "ops_serve.h"

namespace kvm {

constexpr int PG_SEQS = 1024;

// What both operators check before they write: row numbers that do not fall and end within the buffers, lengths within the table. All
// threads of the workgroup call it; the row numbers are in LDS afterwards (cu: B + 1 words).
__device__ __forceinline__ bool paged_call_ok(const Ctx& c, const View& cu, const View& lens, int B, int rows, long long room, LDS int* scu) {
  bool bad = false;
  for (int b = tid(); b <= B; b += KVM_THREADS) {
    const int r = cu.i()[b], p = b ? cu.i()[b - 1] : 0, L = b ? lens.i()[b - 1] : 0;
    scu[b] = r;
    if (r < p || p < 0 || r > rows || (r > p && b && (L < 0 || (long long)L + (r - p) > room))) { bad = true; c.fail(KVM_ERR_OP_KVLEN, b - 1, L); }
  }
  return !__syncthreads_or(bad);
}
// The sequence of row r < scu[B]: the last one that starts at or before it (ones without rows start where the next does).
__device__ __forceinline__ int paged_owner(const LDS int* scu, int B, int r) {
  int lo = 0, hi = B;                                                  // scu[lo] <= r < scu[hi]
  while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if (scu[mid] <= r) lo = mid; else hi = mid; }
  return lo;
}

// ---------------------------------------------------------------------------------------------- append
struct AppendPaged {
  View q, k, v, qo, kc, vc, table, lens, cu, qg, kg; int r0, r1, B, H, Hkv, hd, page, lp; float theta, eps; int pages;
  __device__ explicit AppendPaged(const Ctx& c)
      : q(uview(c, 0)), k(uview(c, 1)), v(uview(c, 2)), qo(uview(c, 3)), kc(uview(c, 4)), vc(uview(c, 5)), table(uview(c, 6)), lens(uview(c, 7)), cu(uview(c, 8)), qg(uview(c, 9)),
        kg(uview(c, 10)), r0(rfl(c.i(11))), r1(rfl(c.i(12))), B(rfl(c.i(13))), H(rfl(c.i(14))), Hkv(rfl(c.i(15))), hd(rfl(c.i(16))), page(rfl(c.i(17))), theta(c.f(18)), eps(c.f(19)) {
    lp = 31 - __clz(page);
    pages = (int)((unsigned)kc.rows / (unsigned)(Hkv * page));
    if (!q.ok()) H = 0;
  }
  __device__ int rows() const { return q.ok() ? min(min(q.rows, qo.rows), min(k.rows, v.rows)) : min(k.rows, v.rows); }
  // Position of row r and its place in the pages (of head 0); the page is checked.
  __device__ bool place(const LDS int* scu, int r, int& t, long long& at) const {
    const int b = paged_owner(scu, B, r);
    t = lens.i()[b] + (r - scu[b]);
    const int p = table.i()[(long long)b * table.cols + (t >> lp)];
    at = (((long long)p * Hkv) << lp) + (t & (page - 1));
    return (unsigned)p < (unsigned)pages;
  }
};
// One of three values by `what` (values, not references: a choice between fields would put the arguments into scratch memory).
template <class T> __device__ __forceinline__ T pick(int what, T a, T b, T c) { return what == 0 ? a : what == 1 ? b : c; }
__device__ __forceinline__ View pick_view(int what, const View& a, const View& b, const View& c) {
  return View{pick<void*>(what, a.p, b.p, c.p), 0, pick<int>(what, a.cols, b.cols, c.cols), pick<int>(what, a.dtype, b.dtype, c.dtype), 0};
}
// LDS of a task: rows in flight with their positions, places and angles.
constexpr int AP_ROWS = 32;
struct AppendPagedLds {
  LDS double* freq; LDS long long* at; LDS int* pos; LDS int* cu; LDS float* ang;
  __device__ explicit AppendPagedLds(LDS char* p) : freq((LDS double*)p), at((LDS long long*)(freq + 128)), pos((LDS int*)(at + AP_ROWS)), cu(pos + AP_ROWS), ang((LDS float*)(cu + PG_SEQS + 4)) {}
  static constexpr int BYTES = 128 * 8 + AP_ROWS * 12 + (PG_SEQS + 4) * 4 + AP_ROWS * 256 * 4;
};
static_assert(AppendPagedLds::BYTES <= KVM_LDS_BYTES, "LDS");
// Checks the call and the task's own pages (nothing is written before); the rows that have a token begin at `r` and end at `end`. Frequencies, and
// positions and places of the first AP_ROWS rows, are in LDS then.
__device__ __forceinline__ bool append_paged_begin(const Ctx& c, const AppendPaged& A, const AppendPagedLds& M, int& r, int& end) {
  if (A.theta > 0.f && tid() >= KVM_THREADS - A.hd / 2) {              // (under the loads of what follows)
    const int i = KVM_THREADS - 1 - tid();
    M.freq[i] = q8_freq(i, A.hd, log((double)A.theta));
  }
  if (!paged_call_ok(c, A.cu, A.lens, A.B, A.rows(), (long long)A.table.cols << A.lp, M.cu)) return false;
  r = max(A.r0, rfl(M.cu[0])); end = min(A.r1, rfl(M.cu[A.B]));
  bool bad = false;
  for (int u = r + tid(); u < end; u += KVM_THREADS) {
    int t; long long at;
    if (!A.place(M.cu, u, t, at)) { bad = true; c.fail(KVM_ERR_OP_RANGE, u, t); }
    if (u < r + AP_ROWS) { M.pos[u - r] = t; M.at[u - r] = at; }
  }
  return !__syncthreads_or(bad);
}
// Positions, places (the first rows' are there) and angles of rows [r, r + nr).
__device__ __forceinline__ void append_paged_rows(const AppendPaged& A, const AppendPagedLds& M, int r, int nr, bool first) {
  const int half = A.hd / 2;
  if (!first) {
    __syncthreads();
    if (tid() < nr) {
      int t; long long at;
      A.place(M.cu, r + tid(), t, at);
      M.pos[tid()] = t; M.at[tid()] = at;
    }
    __syncthreads();
  }
  if (A.theta > 0.f) {
    for (int e = tid(); e < nr * half; e += KVM_THREADS) {
      const int u = e / half, i = e % half;
      float sn, co; q8_turn(M.pos[u], M.freq[i], sn, co);
      M.ang[u * A.hd + i] = sn; M.ang[u * A.hd + half + i] = co;
    }
    __syncthreads();
  }
}
// Any head size and alignment: a wave to a (row, head), a lane to pairs of dims.
__device__ __noinline__ void op_qkv_append_paged(const Ctx& c) {
  const AppendPaged A(c);
  const AppendPagedLds M(c.smem);
  int begin, end;
  if (!append_paged_begin(c, A, M, begin, end)) return;
  const int half = A.hd / 2, heads = A.H + 2 * A.Hkv, l = lane();
  for (int r = begin; r < end; r += AP_ROWS) {
    const int nr = min(AP_ROWS, end - r);
    append_paged_rows(A, M, r, nr, r == begin);
    for (int u = wave(); u < nr * heads; u += KVM_WAVES) {
      const int row = u / heads, s = u % heads, what = s < A.H ? 0 : s < A.H + A.Hkv ? 1 : 2, h = what == 0 ? s : what == 1 ? s - A.H : s - A.H - A.Hkv;
      const View src = pick_view(what, A.q, A.k, A.v), dst = pick_view(what, A.qo, A.kc, A.vc), g = pick_view(what, A.qg, A.kg, View{nullptr, 0, 0, 0, 0});
      const long long from = (long long)(r + row) * src.cols + (long long)h * A.hd;
      const long long to = what == 0 ? (long long)(r + row) * dst.cols + (long long)h * A.hd : (M.at[row] + ((long long)h << A.lp)) * dst.cols;
      float x[2][2], ss = 0.f;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int i = l + 64 * j;
        x[j][0] = i < half ? src.ld(from + i) : 0.f; x[j][1] = i < half ? src.ld(from + half + i) : 0.f;
        ss += x[j][0] * x[j][0] + x[j][1] * x[j][1];
      }
      const float rs = g.ok() ? 1.f / sqrtf(wave_sum(ss) / A.hd + A.eps) : 1.f;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int i = l + 64 * j;
        if (i >= half) continue;
        float a = x[j][0], b = x[j][1];
        if (g.ok()) { a = a * rs * g.f()[i]; b = b * rs * g.f()[half + i]; }
        if (what < 2 && A.theta > 0.f) {
          const float sn = M.ang[row * A.hd + i], co = M.ang[row * A.hd + half + i], y = a * co - b * sn;
          b = a * sn + b * co; a = y;
        }
        dst.st(to + i, a); dst.st(to + half + i, b);
      }
    }
  }
}
// Head sizes 64 and 128, rows in whole vectors, one type for the new rows and one for where they go. Bound: bytes for prompts, a few dependent
// loads (row numbers, length, page, row) and the launch for single tokens. A (row, head) is HD / 8 lanes of 8 values; a row's angles are
// computed once for all its heads; four items' loads are requested together. A call (launch ~13 us): 96 tokens of 48 heads of 128 24 us, prompts of
// 1,900 rows of 24 heads of 64 in f32 40 us (24 MB).
template <int HD, bool FROM16> __device__ __noinline__ void append_paged_t(const Ctx& c) {
  constexpr int LPR = HD / 8, RPP = KVM_THREADS / LPR, NR = 4;
  const AppendPaged A(c);
  const AppendPagedLds M(c.smem);
  const int ln = tid() % LPR, rw = tid() / LPR;
  const unsigned heads = A.H + 2 * A.Hkv;
  const bool to16 = A.kc.dtype == 2, qn = A.qg.ok(), kn = A.kg.ok(), turn = A.theta > 0.f;
  const float sign = ln >= LPR / 2 ? 1.f : -1.f;
  float qg[8], kg[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) { qg[e] = qn ? A.qg.f()[8 * ln + e] : 1.f; kg[e] = kn ? A.kg.f()[8 * ln + e] : 1.f; }
  // the row and head of item u of this range: what it is (0 query, 1 key, 2 value) and its head
  struct Item { int row, what, h; };
  auto item = [&](int u) {
    const int row = (int)((unsigned)u / heads), s = u - row * (int)heads, what = s < A.H ? 0 : s < A.H + A.Hkv ? 1 : 2;
    return Item{row, what, s - (what == 0 ? 0 : what == 1 ? A.H : A.H + A.Hkv)};
  };
  Raw8 raw[NR];
  auto request = [&](int r, int items, int u0) {
#pragma unroll
      for (int i = 0; i < NR; ++i) {
        const Item t = item(min(u0 + i * RPP, items - 1));
        const View x = pick_view(t.what, A.q, A.k, A.v);
        raw[i].load(View{x.p, 0, x.cols, FROM16 ? 2 : 0, 0}, (long long)(r + t.row) * x.cols + t.h * HD + 8 * ln);
      }
  };
  if (A.r0 >= A.r1) return;
  request(A.r0, min(AP_ROWS, A.r1 - A.r0) * (int)heads, rw);           // the first rows, before it is known whose they are
  int begin, end;
  if (!append_paged_begin(c, A, M, begin, end)) return;
  for (int r = begin; r < end; r += AP_ROWS) {
    const int nr = min(AP_ROWS, end - r), items = nr * (int)heads;
    if (r != A.r0) request(r, items, rw);
    append_paged_rows(A, M, r, nr, r == begin);
    for (int u0 = rw; u0 < items; u0 += NR * RPP) {
      if (u0 != rw) request(r, items, u0);
#pragma unroll
      for (int i = 0; i < NR; ++i) {
        const int u = u0 + i * RPP;
        if (u >= items) break;
        const Item t = item(u);
        float x[8];
        raw[i].get(FROM16, x);
        if (t.what == 0 ? qn : t.what == 1 && kn) {
          float ss = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) ss += x[e] * x[e];
          const float rs = 1.f / sqrtf(lanes_sum<LPR>(ss) / HD + A.eps);
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = x[e] * rs * (t.what == 0 ? qg[e] : kg[e]);
        }
        if (turn && t.what < 2) {
          const LDS float* ang = M.ang + t.row * HD + 8 * (ln % (LPR / 2));
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = x[e] * ang[HD / 2 + e] + sign * __shfl_xor(x[e], LPR / 2, 64) * ang[e];
        }
        const View y = pick_view(t.what, A.qo, A.kc, A.vc);
        const long long at = (t.what == 0 ? (long long)(r + t.row) : M.at[t.row] + ((long long)t.h << A.lp)) * y.cols + (t.what == 0 ? t.h * HD : 0) + 8 * ln;
        if (to16) { stwt_bf4(y.h() + at, x[0], x[1], x[2], x[3]); stwt_bf4(y.h() + at + 4, x[4], x[5], x[6], x[7]); }
        else { stwt_f4(y.f() + at, f32x4n{x[0], x[1], x[2], x[3]}); stwt_f4(y.f() + at + 4, f32x4n{x[4], x[5], x[6], x[7]}); }
      }
    }
  }
}
__device__ __noinline__ bool op_qkv_append_paged_fast(const Ctx& c) {
  const View q = c.buf(0), k = c.buf(1), v = c.buf(2), qo = c.buf(3), kc = c.buf(4), vc = c.buf(5);
  if ((q.ok() && (!rows8_ok(q) || !rows8_ok(qo) || q.dtype != k.dtype || qo.dtype != kc.dtype)) || v.dtype != k.dtype || vc.dtype != kc.dtype) return false;
  if (!rows8_ok(k) || !rows8_ok(v) || !rows8_ok(kc) || !rows8_ok(vc)) return false;
  const bool half = k.dtype == 2;
  if (c.i(16) == 128) { if (half) append_paged_t<128, true>(c); else append_paged_t<128, false>(c); }
  else if (c.i(16) == 64) { if (half) append_paged_t<64, true>(c); else append_paged_t<64, false>(c); }
  else return false;
  return true;
}

// ---------------------------------------------------------------------------------------------- attention
struct AttnPaged {
  View q, kc, vc, table, lens, cu, part, o, cnt; int s, S, B, H, Hkv, hd, page, tile, G, lp, pages; float sl2;
  __device__ explicit AttnPaged(const Ctx& c)
      : q(uview(c, 0)), kc(uview(c, 1)), vc(uview(c, 2)), table(uview(c, 3)), lens(uview(c, 4)), cu(uview(c, 5)), part(uview(c, 6)), o(uview(c, 7)), cnt(uview(c, 8)),
        s(rfl(c.i(9))), S(rfl(c.i(10))), B(rfl(c.i(11))), H(rfl(c.i(12))), Hkv(rfl(c.i(13))), hd(rfl(c.i(14))), page(rfl(c.i(15))), tile(rfl(c.i(16))) {
    G = H / Hkv;
    lp = 31 - __clz(page);
    pages = (int)((unsigned)kc.rows / (unsigned)(Hkv * page));
    sl2 = __int_as_float(rfl(__float_as_int(c.f(17) * 1.44269504088896340736f)));
  }
  // Storage of one type throughout at head sizes 64 and 128 in whole vectors: the matrix units (0 no, 1 f32, 2 bf16)
  __device__ int fast() const {
    const int t = q.dtype;
    if (kc.dtype != t || vc.dtype != t || o.dtype != t || (hd != 64 && hd != 128) || !rows8_ok(q) || !rows8_ok(kc) || !rows8_ok(vc) || !rows8_ok(o)) return 0;
    if ((part.cols & 1) || ((uintptr_t)part.p & 7) || (long long)Hkv * page * max(kc.cols, vc.cols) * 4 >= 0x7fffff00ll) return 0;   // (partial rows as pairs of words)
    return t == 2 ? 2 : 1;
  }
};
// A tile's rows: row r is token tok0 + r / G of the sequence's new ones, head h * G + r % G; it sees keys 0 .. L + tok0 + r / G.
struct TilePaged { int b, h, L, row0, tok0, ntok; long long start, cost; };
// A piece of a tile: keys [k0, k1), k0 a multiple of 64; piece k of `live`, the second of which falls to task i0.
struct PiecePaged { int k0, k1, k, live, i0; };

// The work of a call over its tasks: a tile costs PG_TILE and one per key up to the last that it sees; tiles in order of sequence, kv head
// and token are cut into equal shares, in all tasks alike from the lengths. A cut within PG_SNAP of a tile's end moves there: a small piece
// costs more than it balances; where there is a task for every tile and none is longer than a share by PG_CUT, about what the partials and the
// merge of a cut cost, no tile is cut: a tile costs 1 then, a task has one or none, and these are spread over all tasks (shared out by their keys
// some tasks had two and others none: 1,000 tokens of 32 heads behind 3,750, 256 tiles, 272 us in place of 175). Tiles of up to 32 rows are a
// sequence's new tokens as a whole (the waves share the keys); longer ones have `tile` rows (the waves share the rows).
constexpr int PG_TILE = 256, PG_SNAP = 320, PG_SHARE = 512, PG_CUT = 1024;
struct WorkPaged {
  const LDS long long* pre;    // [B + 1] cost of the sequences before
  const LDS int *cu, *len;
  int B, Hkv, G, rows;
  long long share, total;
  int S;
  bool whole;                  // tiles are not cut, the costs are numbers of tiles
  __device__ __forceinline__ int tokens(int n) const { return max(1, min(n, rows / G)); }   // of a tile, whose rows fit in the partials'
  // cost of the first j tiles of TT tokens of one head, none of them the last, ragged one
  __device__ __forceinline__ long long upto(long long j, long long L, long long TT) const { return whole ? j : j * (PG_TILE + L) + TT * (j * (j + 1) / 2); }
  __device__ __forceinline__ long long head_cost(int n, int L) const {
    if (n <= 0) return 0;
    const int TT = tokens(n), nt = (n + TT - 1) / TT;
    return whole ? nt : upto(nt - 1, L, TT) + PG_TILE + L + n;
  }
  __device__ __forceinline__ TilePaged find(long long x) const {
    int b = 0;
    for (int j0 = 0; j0 < B; j0 += 64) b += __popcll(__ballot(j0 + lane() < B && pre[min(j0 + lane(), B)] <= x));
    b = rfl(b) - 1;
    const int L = rfl(len[b]), r0 = rfl(cu[b]), n = rfl(cu[b + 1]) - r0, TT = tokens(n), nt = (n + TT - 1) / TT;
    const long long p0 = pre[b], hc = head_cost(n, L);
    const int h = rfl((int)((x - p0) / hc));
    const long long rest = x - p0 - h * hc;
    int lo = 0, hi = nt;                                               // upto(lo) <= rest, rest < upto(hi) or hi is the end
    while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if (upto(mid, L, TT) <= rest) lo = mid; else hi = mid; }
    lo = rfl(lo);
    TilePaged t;
    t.b = b; t.h = h; t.L = L; t.row0 = r0 + lo * TT; t.tok0 = lo * TT; t.ntok = min(TT, n - lo * TT);
    t.start = p0 + h * hc + upto(lo, L, TT);
    t.cost = whole ? 1 : PG_TILE + (long long)L + t.tok0 + t.ntok;
    return t;
  }
  __device__ __forceinline__ long long cut(int i) const {
    if (whole) return i == S ? total : (unsigned)i * (unsigned)total / (unsigned)S;   // (i < S and total <= S, at most 65,536)
    const long long x = min(i * share, total);
    if (x == total) return total;
    const TilePaged t = find(x);
    const long long off = x - t.start;
    return off < PG_SNAP ? t.start : t.cost - off < PG_SNAP ? t.start + t.cost : x;
  }
  // The piece [x, end) of a tile: its keys, and which of how many pieces it is.
  __device__ __forceinline__ PiecePaged piece(const TilePaged& t, long long x, long long end) const {
    auto key = [&](long long off) { return (int)(max(0ll, off - PG_TILE) & ~63ll); };
    PiecePaged p;
    p.k0 = x == t.start ? 0 : key(x - t.start);
    p.k1 = end == t.start + t.cost ? t.L + t.tok0 + t.ntok : key(end - t.start);
    const long long first = (t.start + PG_SNAP + share - 1) / share, last = (t.start + t.cost - PG_SNAP) / share;
    const int inside = whole || t.cost < 2 * PG_SNAP ? 0 : (int)max(0ll, last - first + 1);
    p.i0 = rfl((int)first); p.live = rfl(inside + 1);
    p.k = x == t.start ? 0 : rfl((int)(x / share - first + 1));
    p.k0 = rfl(p.k0); p.k1 = rfl(p.k1);
    return p;
  }
};
// LDS that stays over a task's pieces: the work; the forms' own memory begins behind it.
constexpr int PG_WORK = (PG_SEQS + 2) * 8 + (PG_SEQS + 4) * 4 + PG_SEQS * 4 + 128;

// Where piece k of a tile keeps its partial rows: the second half of the task in front of i0 for the first one, the first half of its own task
// for the others (a task has at most one piece of each kind).
__device__ __forceinline__ GLOBAL float* paged_partial(const AttnPaged& D, const PiecePaged& p, int k, int r) {
  return D.part.f() + ((long long)(2 * p.i0 - 2 + (k ? 2 * k : 1)) * D.tile + r) * D.part.cols;
}
__device__ __forceinline__ long long paged_out(const AttnPaged& D, const TilePaged& t, int r) {
  return (long long)(t.row0 + r / D.G) * D.o.cols + (long long)(t.h * D.G + r % D.G) * D.hd;
}
// The piece that counts itself last merges the tile's rows, in the pieces' order whichever it is; maxima are in units of log2. A piece of weight 0
// counts too: a NaN or an infinity that a row sees there stays one.
// Few rows: a thread has four dims of a row and a share of the pieces, 16 of them requested at once with their maxima and sums; the shares meet
// in LDS. Many rows: first the pieces' weights, to LDS, then four dims of four rows a thread at once.
template <bool PAIRS> __device__ __forceinline__ f32x4n paged_dims(const GLOBAL float* y, int d, int hd) {
  if (PAIRS) { const u32x2_t a = *(const GLOBAL u32x2_t*)(y + d), b = *(const GLOBAL u32x2_t*)(y + d + 2); return f32x4n{__uint_as_float(a.x), __uint_as_float(a.y), __uint_as_float(b.x), __uint_as_float(b.y)}; }
  f32x4n x;
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = y[min(d + i, hd - 1)];
  return x;
}
__device__ __forceinline__ void paged_put(const AttnPaged& D, const TilePaged& t, int r, int d, f32x4n x, bool pairs) {
  const long long o = paged_out(D, t, r) + d;
  if (pairs && D.o.dtype == 2) stwt_bf4(D.o.h() + o, x.x, x.y, x.z, x.w);
  else if (pairs) stwt_f4(D.o.f() + o, x);
  else
    for (int i = 0; i < min(4, D.hd - d); ++i) D.o.st(o + i, x[i]);
}
__device__ __forceinline__ float paged_top(float m, float x) { return x > m || x != x ? x : m; }              // a NaN stays
__device__ __forceinline__ float paged_weight(float m, float top) { return m == -INFINITY ? 0.f : exp2f(m - top); }
template <bool PAIRS> __device__ __noinline__ void paged_merge_few(const Ctx& c, int row0_, int h_, int ntok_, int live_, int i0_) {
  const AttnPaged D(c);
  const int live = rfl(live_), R = rfl(ntok_) * D.G, hd = D.hd, C4 = (hd + 3) >> 2, items = R * C4, split = min(live, KVM_THREADS / items);
  const TilePaged t{0, rfl(h_), 0, rfl(row0_), 0, rfl(ntok_), 0, 0};
  const PiecePaged p{0, 0, 0, live, rfl(i0_)};
  const int e = tid() % items, g = tid() / items, r = e / C4, d = 4 * (e % C4);
  f32x4n a = {0.f, 0.f, 0.f, 0.f};
  float M = -INFINITY, z = 0.f;
  constexpr int U = 16;
  for (int k0 = g < split ? g : live; k0 < live; k0 += U * split) {
    float m[U], s[U], top = M;
    f32x4n x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const GLOBAL float* y = paged_partial(D, p, min(k0 + u * split, live - 1), r);
      m[u] = y[hd]; s[u] = y[hd + 1];
      x[u] = paged_dims<PAIRS>(y, d, hd);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      m[u] = k0 + u * split < live ? m[u] : -INFINITY;
      top = paged_top(top, m[u]);
    }
    const float f = paged_weight(M, top);
    a *= f; z *= f; M = top;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float w = paged_weight(m[u], top);
      a += w * x[u]; z += w * s[u];                                    // (behind the last piece: that one again, with weight 0)
    }
  }
  LDS float* sh = (LDS float*)(c.smem + PG_WORK);                      // [256][6]
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) sh[6 * tid() + i] = a[i];
  sh[6 * tid() + 4] = M; sh[6 * tid() + 5] = z;
  __syncthreads();
  if (g == 0) {
    float top = M;
    for (int k = 1; k < split; ++k) top = paged_top(top, sh[6 * (tid() + k * items) + 4]);
    const float f = paged_weight(M, top);
    a *= f; z *= f;
    for (int k = 1; k < split; ++k) {
      const LDS float* y = sh + 6 * (tid() + k * items);
      const float w = paged_weight(y[4], top);
      a += w * f32x4n{y[0], y[1], y[2], y[3]}; z += w * y[5];
    }
    paged_put(D, t, r, d, f32x4n{a.x / z, a.y / z, a.z / z, a.w / z}, PAIRS);
  }
}
constexpr int PG_WEIGHTS = 8192;   // weights of pieces in LDS; tiles cut into more take them as they go
static_assert(PG_WORK + (256 + 2 * PG_WEIGHTS) * 4 <= KVM_LDS_BYTES, "LDS");
// (forms of their own: a branch between two loads makes each wait for the one before, 50 us for two pieces of 128 rows)
template <bool PAIRS, bool TABLE, int NI, int U> __device__ __forceinline__ void paged_sum_many(const AttnPaged& D, const TilePaged& t, const PiecePaged& p, int R, const LDS float* M, const LDS float* Z, const LDS float* W) {
  const int hd = D.hd, C4 = (hd + 3) >> 2, items = R * C4;
  for (int e0 = tid(); e0 < items; e0 += NI * KVM_THREADS) {
    f32x4n a[NI];
    int r[NI], d[NI];
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int e = min(e0 + i * KVM_THREADS, items - 1);
      r[i] = e / C4; d[i] = 4 * (e - r[i] * C4);
      a[i] = f32x4n{0.f, 0.f, 0.f, 0.f};
    }
    for (int k0 = 0; k0 < p.live; k0 += U) {
      f32x4n x[NI][U];
      float w[NI][U];
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const GLOBAL float* y = paged_partial(D, p, min(k0 + u, p.live - 1), r[i]);
          x[i][u] = paged_dims<PAIRS>(y, d[i], hd);
          if (!TABLE) w[i][u] = y[hd];
        }
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const float v = TABLE ? W[min(k0 + u, p.live - 1) * R + r[i]] : paged_weight(w[i][u], M[r[i]]);
          if (k0 + u < p.live) a[i] += v * x[i][u];
        }
    }
#pragma unroll
    for (int i = 0; i < NI; ++i)
      if (e0 + i * KVM_THREADS < items) { const float z = Z[r[i]]; paged_put(D, t, r[i], d[i], f32x4n{a[i].x / z, a[i].y / z, a[i].z / z, a[i].w / z}, PAIRS); }
  }
}
template <bool PAIRS> __device__ __noinline__ void paged_merge_many(const Ctx& c, int row0_, int h_, int ntok_, int live_, int i0_) {
  const AttnPaged D(c);
  const int live = rfl(live_), R = rfl(ntok_) * D.G, hd = D.hd;
  const TilePaged t{0, rfl(h_), 0, rfl(row0_), 0, rfl(ntok_), 0, 0};
  const PiecePaged p{0, 0, 0, live, rfl(i0_)};
  LDS float* M = (LDS float*)(c.smem + PG_WORK);                       // [128] maxima, [128] sums, [live][R] weights, the pieces' sums
  LDS float* Z = M + 128;
  LDS float* W = Z + 128;
  const bool table = live * R <= PG_WEIGHTS;
  if (table) {                                                         // maxima and sums of all pieces in one round of loads
    LDS float* S = W + PG_WEIGHTS;
    constexpr int NB = 8;
    for (int e0 = tid(); e0 < live * R; e0 += NB * KVM_THREADS) {
      float x[NB], y[NB];
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const int e = min(e0 + i * KVM_THREADS, live * R - 1), k = e / R;
        const GLOBAL float* v = paged_partial(D, p, k, e - k * R) + hd;
        x[i] = v[0]; y[i] = v[1];
      }
#pragma unroll
      for (int i = 0; i < NB; ++i) if (e0 + i * KVM_THREADS < live * R) { W[e0 + i * KVM_THREADS] = x[i]; S[e0 + i * KVM_THREADS] = y[i]; }
    }
    __syncthreads();
    if (tid() < R) {
      float top = -INFINITY, z = 0.f;
      for (int k = 0; k < live; ++k) top = paged_top(top, W[k * R + tid()]);
      for (int k = 0; k < live; ++k) {
        const float w = paged_weight(W[k * R + tid()], top);
        W[k * R + tid()] = w;
        z += w * S[k * R + tid()];
      }
      M[tid()] = top; Z[tid()] = z;
    }
    __syncthreads();
  } else {
    for (int r0 = 0; r0 < R; r0 += KVM_THREADS / 8) {                    // eight lanes to a row
      const int r = r0 + (tid() >> 3), sub = tid() & 7;
      float m = -INFINITY, z = 0.f;
      for (int k0 = sub; k0 < live; k0 += 32) {
        float x[4], y[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const GLOBAL float* v = paged_partial(D, p, min(k0 + 8 * u, live - 1), min(r, R - 1)) + hd;
          x[u] = v[0]; y[u] = v[1];
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (k0 + 8 * u < live && x[u] != -INFINITY) {
            const float top = paged_top(m, x[u]);
            z = paged_weight(m, top) * z + exp2f(x[u] - top) * y[u];
            m = top;
          }
      }
      const float top = lanes_all<8>(m, [](float a, float b) { return a != a ? a : paged_top(a, b); }), f = paged_weight(m, top);
      z = lanes_sum<8>(f * z);
      if (sub == 0 && r < R) { M[r] = top; Z[r] = z; }
    }
    __syncthreads();
  }
  if (!table) paged_sum_many<PAIRS, false, 4, 4>(D, t, p, R, M, Z, W);
  else if (live == 2) paged_sum_many<PAIRS, true, 8, 2>(D, t, p, R, M, Z, W);
  else paged_sum_many<PAIRS, true, 4, 4>(D, t, p, R, M, Z, W);
}
__device__ __forceinline__ void paged_arrive(const Ctx& c, const AttnPaged& D, const TilePaged& t, const PiecePaged& p, LDS int* flag) {
  wait_stores();
  __syncthreads();
  if (tid() == 0) *flag = add_relaxed((int*)D.cnt.i() + p.i0, 1);
  __syncthreads();
  const int old = rfl(*flag);
  if (old < 0 || old >= p.live) { if (tid() == 0) c.fail(KVM_ERR_OP_RANGE, p.i0, old); return; }
  if (old != p.live - 1) return;
  fence_acquire();                                                     // the other pieces' partials, stored before their counts
  const bool few = t.ntok * D.G * ((D.hd + 3) >> 2) <= KVM_THREADS / 2, pairs = rfl(D.fast()) != 0;
  if (few) { if (pairs) paged_merge_few<true>(c, t.row0, t.h, t.ntok, p.live, p.i0); else paged_merge_few<false>(c, t.row0, t.h, t.ntok, p.live, p.i0); }
  else if (pairs) paged_merge_many<true>(c, t.row0, t.h, t.ntok, p.live, p.i0);
  else paged_merge_many<false>(c, t.row0, t.h, t.ntok, p.live, p.i0);
  if (tid() == 0) st_relaxed((int*)D.cnt.i() + p.i0, 0);
}

enum { PG_DONE, PG_AGAIN, PG_FAILED };   // a piece is written; is to be done by the general form; has a page that is none

// Any storage, head size and alignment, in f32, and pieces of the other forms with results that are not finite (a key that a row does not see
// has weight 0 there, which an infinity or NaN in its value would turn into NaN; here it is skipped): 32 rows by 32 keys at a time in LDS, the
// next keys' loads in flight; scores a thread to a key and four rows, eight threads to a row for the softmax and its P V.
__device__ __noinline__ int attn_paged_general(const Ctx& c, int b_, int h_, int L_, int row0_, int tok0_, int ntok_, int k0_, int k1_, int k_, int live_, int i0_) {
  const AttnPaged D(c);
  const TilePaged t{rfl(b_), rfl(h_), rfl(L_), rfl(row0_), rfl(tok0_), rfl(ntok_), 0, 0};
  const PiecePaged p{rfl(k0_), rfl(k1_), rfl(k_), rfl(live_), rfl(i0_)};
  constexpr int KB = 32, NF = 8;                                       // keys a step; vectors of 4 a thread at 256 dims
  const int hd = D.hd, C4 = (hd + 3) >> 2, HP = 4 * C4 + 4, R = t.ntok * D.G;
  LDS float* qs = (LDS float*)(c.smem + PG_WORK);                      // [32][HP]
  LDS float* ks = qs + 32 * HP;                                        // [KB][HP]
  LDS float* vs = ks + KB * HP;
  LDS float* ps = vs + KB * HP;                                        // [32][KB + 4]; below 0: not seen
  const bool vec = (hd & 3) == 0 && rows8_ok(D.kc) && rows8_ok(D.vc);
  const GLOBAL int* tb = D.table.i() + (long long)t.b * D.table.cols;
  bool bad = false;
  f32x4n kr[NF], vr[NF];
  auto at4 = [&](const View& X, long long o, int d) {
    if (vec) return ld4(X, o + d);
    return f32x4n{X.ld(o + d), d + 1 < hd ? X.ld(o + d + 1) : 0.f, d + 2 < hd ? X.ld(o + d + 2) : 0.f, d + 3 < hd ? X.ld(o + d + 3) : 0.f};
  };
  auto fetch = [&](int kb) {
#pragma unroll
    for (int i = 0; i < NF; ++i) {
      const int e = tid() + i * KVM_THREADS;
      if (e >= KB * C4) break;
      const int key = min(kb + e / C4, p.k1 - 1), d = 4 * (e % C4);
      int id = tb[key >> D.lp];
      if ((unsigned)id >= (unsigned)D.pages) { bad = true; id = 0; }
      const long long row = ((((long long)id * D.Hkv) + t.h) << D.lp) + (key & (D.page - 1));
      kr[i] = at4(D.kc, row * D.kc.cols, d);
      vr[i] = at4(D.vc, row * D.vc.cols, d);
    }
  };
  for (int rg = 0; rg < R; rg += 32) {
    __syncthreads();
    for (int e = tid(); e < 32 * C4; e += KVM_THREADS) {
      const int r = rg + e / C4, d = 4 * (e % C4);
      const long long o = (long long)(t.row0 + min(r, R - 1) / D.G) * D.q.cols + (long long)(t.h * D.G + min(r, R - 1) % D.G) * hd;
#pragma unroll
      for (int i = 0; i < 4; ++i) qs[(e / C4) * HP + d + i] = d + i < hd ? D.q.ld(o + d + i) : 0.f;
    }
    fetch(p.k0);
    const int row = tid() >> 3, sub = tid() & 7, rr = min(rg + row, R - 1), lim = t.L + t.tok0 + rr / D.G;
    float m = -INFINITY, lsum = 0.f;
    f32x4n acc[NF];
#pragma unroll
    for (int i = 0; i < NF; ++i) acc[i] = f32x4n{0.f, 0.f, 0.f, 0.f};
    for (int kb = p.k0; kb < p.k1; kb += KB) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < NF; ++i) {
        const int e = tid() + i * KVM_THREADS;
        if (e >= KB * C4) break;
        *(LDS f32x4n*)(ks + (e / C4) * HP + 4 * (e % C4)) = kr[i];
        *(LDS f32x4n*)(vs + (e / C4) * HP + 4 * (e % C4)) = vr[i];
      }
      __syncthreads();
      if (kb + KB < p.k1) fetch(kb + KB);
      {
        const int key = tid() & 31, r4 = 4 * (tid() >> 5);
        float a[4] = {0.f, 0.f, 0.f, 0.f};
        for (int d = 0; d < 4 * C4; d += 4) {
          const f32x4n kk = *(const LDS f32x4n*)(ks + key * HP + d);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const f32x4n qq = *(const LDS f32x4n*)(qs + (r4 + i) * HP + d);
            a[i] += qq.x * kk.x; a[i] += qq.y * kk.y; a[i] += qq.z * kk.z; a[i] += qq.w * kk.w;
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) ps[(r4 + i) * (KB + 4) + key] = a[i] * D.sl2;
      }
      __syncthreads();
      float x[4], mx = -INFINITY;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = kb + 4 * sub + i;
        const bool on = key <= lim && key < p.k1;
        x[i] = on ? ps[row * (KB + 4) + 4 * sub + i] : -INFINITY;
        mx = fmaxf(mx, x[i]);
        if (on && x[i] != x[i]) mx = x[i];                             // a NaN score stays one (fmaxf drops it)
      }
      mx = lanes_all<8>(mx, [](float a, float b) { return a != a ? a : b != b ? b : fmaxf(a, b); });
      const float top = mx != mx ? mx : fmaxf(m, mx), f = m == -INFINITY ? 0.f : exp2f(m - top);
      float sum = 0.f;
      __syncthreads();                                                 // scores are read before weights overwrite them
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = kb + 4 * sub + i;
        const bool on = key <= lim && key < p.k1;
        const float e = !on ? -1.f : x[i] == -INFINITY ? 0.f : exp2f(x[i] - top);   // (all of a block may be -inf, and later ones not)
        if (on) sum += e;
        ps[row * (KB + 4) + 4 * sub + i] = e;
      }
      sum = lanes_sum<8>(sum);
      lsum = lsum * f + sum;
      m = top;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < NF; ++i) acc[i] *= f;
      const int n = min(KB, p.k1 - kb);
      for (int u = 0; u < n; ++u) {
        const float e = ps[row * (KB + 4) + u];
        if (e < 0.f) continue;
#pragma unroll
        for (int i = 0; i < NF; ++i)
          if (sub + 8 * i < C4) acc[i] += e * *(const LDS f32x4n*)(vs + u * HP + 4 * (sub + 8 * i));
      }
    }
    if (__syncthreads_or(bad)) { if (tid() == 0) c.fail(KVM_ERR_OP_RANGE, t.b, p.k0); return PG_FAILED; }
    if (rg + row < R) {
#pragma unroll
      for (int i = 0; i < NF; ++i)
        for (int e = 0; e < 4; ++e) {
          const int d = 4 * (sub + 8 * i) + e;
          if (d >= hd) break;
          if (p.live == 1) D.o.st(paged_out(D, t, rg + row) + d, acc[i][e] / lsum);
          else stwt32(paged_partial(D, p, p.k, rg + row) + d, acc[i][e]);
        }
      if (p.live > 1 && sub == 0) { GLOBAL float* y = paged_partial(D, p, p.k, rg + row) + hd; stwt32(y, m); stwt32(y + 1, lsum); }
    }
  }
  return PG_DONE;
}

// The end of a piece whose waves have keys of their own: their states (maxima m and sums ls of row l % 16 of each tile, ls a share for each quarter
// of the wave, P V in acc: dims DPL (4 (l / 16) + q) + i) meet in LDS; the rows go out, or to the piece's partials.
template <int HD, int NT, bool HALF>
__device__ __forceinline__ int paged_waves(const Ctx& c, const AttnPaged& D, const TilePaged& t, const PiecePaged& p, const f32x4_t (&acc)[NT][HD / 16], const float (&m)[NT],
                                           const float (&ls)[NT], bool bad) {
  constexpr int DPL = HD / 16, RW = 16 * NT;
  const int l = lane(), w = rfl(wave()), m16 = l & 15, qq = l >> 4, R = t.ntok * D.G;
  LDS float* st = (LDS float*)(c.smem + PG_WORK);                      // [4][2][32] maxima and sums
  LDS float* ol = st + 256;                                            // [4][RW][HD + 4]
  __syncthreads();
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const float z = rows_sum(ls[n]);
    if (qq == 0) { st[64 * w + 16 * n + m16] = m[n]; st[64 * w + 32 + 16 * n + m16] = z; }
  }
  __syncthreads();
  float nf = 0.f;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = 16 * n + m16;
    const float top = fmaxf(fmaxf(st[r], st[64 + r]), fmaxf(st[128 + r], st[192 + r]));
    const float f = m[n] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[n] - top);
    float z = 0.f;
#pragma unroll
    for (int v = 0; v < 4; ++v) z += (st[64 * v + r] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(st[64 * v + r] - top)) * st[64 * v + 32 + r];
    nf += z * 0.f + (top == -INFINITY ? 0.f : top * 0.f);
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int i = 0; i < DPL; ++i) {
        const float y = acc[n][i][q] * f;
        nf += y * 0.f;
        ol[(w * RW + r) * (HD + 4) + DPL * (4 * qq + q) + i] = y;
      }
  }
  const int again = __syncthreads_or(nf != 0.f ? 1 : 0), out = __syncthreads_or(bad ? 1 : 0);
  if (out) { if (tid() == 0) c.fail(KVM_ERR_OP_RANGE, t.b, p.k0); return PG_FAILED; }
  if (again) return PG_AGAIN;                                            // something is not finite: by the general form
  for (int e = tid(); e < R * (HD / 4); e += KVM_THREADS) {
    const int r = e / (HD / 4), d = 4 * (e % (HD / 4));
    f32x4n a = *(const LDS f32x4n*)(ol + r * (HD + 4) + d);
#pragma unroll
    for (int v = 1; v < 4; ++v) a += *(const LDS f32x4n*)(ol + (v * RW + r) * (HD + 4) + d);
    const float top = fmaxf(fmaxf(st[r], st[64 + r]), fmaxf(st[128 + r], st[192 + r]));
    float z = 0.f;
#pragma unroll
    for (int v = 0; v < 4; ++v) z += (st[64 * v + r] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(st[64 * v + r] - top)) * st[64 * v + 32 + r];
    if (p.live == 1) {
      a *= 1.f / z;
      if constexpr (HALF) stwt_bf4(D.o.h() + paged_out(D, t, r) + d, a.x, a.y, a.z, a.w);
      else stwt_f4(D.o.f() + paged_out(D, t, r) + d, a);
    }
    else {
      GLOBAL float* y = paged_partial(D, p, p.k, r);
      stwt_f4(y + d, a);
      if (d == 0) { stwt32(y + HD, top); stwt32(y + HD + 1, z); }
    }
  }
  return PG_DONE;
}

// ---- The matrix units: bf16 storage, head sizes 64 and 128.
// Tiles of up to 32 rows (single tokens, drafted ones): bound by the bytes of keys and values. The four waves take units of 32 keys in turn,
// each for itself, K and V straight from the pages into registers, a unit ahead, the page numbers two:
//   scores  v_mfma_f32_16x16x32_bf16, A = 16 keys (row m of tile a: key 8 (m / 4) + 4 a + m % 4), B = 16 query rows (NT such tiles). A lane's
//           16-byte load of a key is its part of the operand, and the rows' order makes the scores' registers the B operand of
//   P V     the same instruction, A = V transposed: a lane loads HD / 16 dims of 8 keys, whole rows of the page to 16 lanes, and turns them
//           in registers (one byte permute for two values), dims DPL m + i to row m of product i.
// A probability goes into the second product as two bf16 operands, its rounding and the rounding of what that leaves (16 bits: rounded once to bf16
// it put the results 0.0023 from 64 bits where the store's own rounding is 0.0017; here the second half of the products costs 1%, the tiles of more
// rows 13 to 19%); the running maximum moves only when a row's grows by more than 2^8. The waves' states meet in LDS. A call: 48 single tokens
// behind 5,000 others each (0.98 GB) 241 us, 4.1 TB/s; one behind 32,000 64 us, of which launch, the pieces' entry and the merge are 40.
// The sum of eight weights onto s.
__device__ __forceinline__ float sum8(const float (&p)[8], float s) { return s + (((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]))); }
template <int HD, int NT> __device__ __noinline__ int attn_paged_keys(const Ctx& c, int b_, int h_, int L_, int row0_, int tok0_, int ntok_, int k0_, int k1_, int k_, int live_, int i0_) {
  constexpr int NK = HD / 32, DPL = HD / 16, RW = 16 * NT;
  const AttnPaged D(c);
  const TilePaged t{rfl(b_), rfl(h_), rfl(L_), rfl(row0_), rfl(tok0_), rfl(ntok_), 0, 0};
  const PiecePaged p{rfl(k0_), rfl(k1_), rfl(k_), rfl(live_), rfl(i0_)};
  const int l = lane(), w = rfl(wave()), m16 = l & 15, qq = l >> 4, R = t.ntok * D.G, klast = p.k1 - 1;
  const GLOBAL int* tb = D.table.i() + (long long)t.b * D.table.cols;
  const GLOBAL char* kb = (const GLOBAL char*)D.kc.p + (((long long)t.h << D.lp) * D.kc.cols) * 2;
  const GLOBAL char* vb = (const GLOBAL char*)D.vc.p + (((long long)t.h << D.lp) * D.vc.cols) * 2;
  const unsigned kpage = (unsigned)(D.Hkv << D.lp) * D.kc.cols * 2, vpage = (unsigned)(D.Hkv << D.lp) * D.vc.cols * 2;   // bytes (below 2^31)
  const int pm = D.page - 1, kpitch = D.kc.cols * 2, vpitch = D.vc.cols * 2;
  bf16x8 qf[NT][NK];
  int lim[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = min(16 * n + m16, R - 1);
    lim[n] = t.L + t.tok0 + r / D.G;
    const GLOBAL uint16_t* q = D.q.h() + (long long)(t.row0 + r / D.G) * D.q.cols + (long long)(t.h * D.G + r % D.G) * HD + 8 * qq;
#pragma unroll
    for (int kk = 0; kk < NK; ++kk) qf[n][kk] = *(const GLOBAL bf16x8*)(q + 32 * kk);
  }
  struct Ids { int k, v; };
  struct Unit { u32x4_t k[2][NK]; u32x4_t v[8]; };                     // (HD 64: the first half of v)
  bool bad = false;
  const int nu = (p.k1 - p.k0 + 31) >> 5;                              // units of the piece; this wave: w, w + 4, ..
  auto ids = [&](Ids& I, int u) {
    const int key0 = p.k0 + 32 * u;
    I.k = tb[min(key0 + 8 * (m16 >> 2), klast) >> D.lp];
    I.v = tb[min(key0 + 8 * qq, klast) >> D.lp];
  };
  auto load = [&](Unit& U, const Ids& I, int u) {
    const int key0 = p.k0 + 32 * u;
    bad = bad || (unsigned)I.k >= (unsigned)D.pages || (unsigned)I.v >= (unsigned)D.pages;
    const unsigned ik = (unsigned)I.k < (unsigned)D.pages ? I.k : 0u, iv = (unsigned)I.v < (unsigned)D.pages ? I.v : 0u;
    const GLOBAL char* kp = kb + (unsigned long long)ik * kpage;
    const GLOBAL char* vp = vb + (unsigned long long)iv * vpage;
#pragma unroll
    for (int a = 0; a < 2; ++a) {
      const GLOBAL char* y = kp + ((min(key0 + 8 * (m16 >> 2) + 4 * a + (m16 & 3), klast) & pm) * kpitch + 16 * qq);
#pragma unroll
      for (int kk = 0; kk < NK; ++kk) U.k[a][kk] = *(const GLOBAL u32x4_t*)(y + 64 * kk);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const GLOBAL char* y = vp + ((min(key0 + 8 * qq + j, klast) & pm) * vpitch + 2 * DPL * m16);
      if constexpr (DPL == 8) U.v[j] = *(const GLOBAL u32x4_t*)y;
      else { const u32x2_t x = *(const GLOBAL u32x2_t*)y; U.v[j].x = x.x; U.v[j].y = x.y; }
    }
  };
  f32x4_t acc[NT][DPL];
  float m[NT], ls[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    m[n] = -INFINITY; ls[n] = 0.f;
#pragma unroll
    for (int i = 0; i < DPL; ++i) acc[n][i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  auto compute = [&](const Unit& U, int u) {
    const int key0 = p.k0 + 32 * u;
    bf16x8 vt[DPL];
#pragma unroll
    for (int d = 0; d < DPL / 2; ++d) {
      u32x4_t lo, hi;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        lo[j] = __builtin_amdgcn_perm(U.v[2 * j + 1][d], U.v[2 * j][d], 0x05040100u);
        hi[j] = __builtin_amdgcn_perm(U.v[2 * j + 1][d], U.v[2 * j][d], 0x07060302u);
      }
      vt[2 * d] = __builtin_bit_cast(bf16x8, lo); vt[2 * d + 1] = __builtin_bit_cast(bf16x8, hi);
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      f32x4_t s[2];
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        s[a] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kk = 0; kk < NK; ++kk) s[a] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, U.k[a][kk]), qf[n][kk], s[a], 0, 0, 0);
      }
      float x[8], mx = -INFINITY;
      const bool edge = key0 + 31 > t.L + t.tok0;                      // some row does not see the whole unit
#pragma unroll
      for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float y = s[a][r] * D.sl2;
          x[4 * a + r] = edge && key0 + 8 * qq + 4 * a + r > lim[n] ? -INFINITY : y;
          mx = fmaxf(mx, x[4 * a + r]);
        }
      mx = rows_max(mx);
      if (__ballot(mx > m[n] + 8.f)) {
        const float top = fmaxf(m[n], mx), f = m[n] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[n] - top);
        ls[n] *= f;
#pragma unroll
        for (int i = 0; i < DPL; ++i) acc[n][i] *= f;
        m[n] = top;
      }
      const float base = m[n] == -INFINITY ? 0.f : m[n];
      float pv[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) pv[i] = __builtin_amdgcn_exp2f(x[i] - base);
      const Pieces<2> pb = split_bf16<2>(pv);
      ls[n] = sum8(pv, ls[n]);
#pragma unroll
      for (int k = 1; k >= 0; --k)
#pragma unroll
        for (int i = 0; i < DPL; ++i) acc[n][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vt[i], pb.p[k], acc[n][i], 0, 0, 0);
    }
  };
  if (w < nu) {
    Ids i0, i1;
    Unit u0, u1;
    ids(i0, w); ids(i1, min(w + 4, nu - 1));
    load(u0, i0, w);
    int u = w;
    for (; u + 8 < nu; u += 8) {                                       // (no branch between a unit's loads and the products of the one before)
      ids(i0, u + 8);
      load(u1, i1, u + 4);
      compute(u0, u);
      ids(i1, min(u + 12, nu - 1));
      load(u0, i0, u + 8);
      compute(u1, u + 4);
    }
    if (u + 4 < nu) {
      load(u1, i1, u + 4);
      compute(u0, u);
      compute(u1, u + 4);
    } else compute(u0, u);
  }
  return paged_waves<HD, NT, true>(c, D, t, p, acc, m, ls, bad);
}

// The same tiles in f32 storage, v_mfma_f32_16x16x4_f32 (exact products): units of 16 keys; a lane's 16-byte load of a key is four dims of it, of
// which product i takes the i-th from all lanes (k = l / 16), and the scores' registers r are, row by row, P's operand for the keys 4 k + r,
// whose values the lane has loaded. A call: 100 rows of 16 heads of 64 behind ~1,000 tokens each 53 us, its tasks' chain of dependent loads.
template <int HD, int NT> __device__ __noinline__ int attn_paged_keys_f32(const Ctx& c, int b_, int h_, int L_, int row0_, int tok0_, int ntok_, int k0_, int k1_, int k_, int live_, int i0_) {
  constexpr int NK = HD / 16, DPL = HD / 16, NV = DPL / 4;
  const AttnPaged D(c);
  const TilePaged t{rfl(b_), rfl(h_), rfl(L_), rfl(row0_), rfl(tok0_), rfl(ntok_), 0, 0};
  const PiecePaged p{rfl(k0_), rfl(k1_), rfl(k_), rfl(live_), rfl(i0_)};
  const int l = lane(), w = rfl(wave()), m16 = l & 15, qq = l >> 4, R = t.ntok * D.G, klast = p.k1 - 1;
  const GLOBAL int* tb = D.table.i() + (long long)t.b * D.table.cols;
  const GLOBAL char* kb = (const GLOBAL char*)D.kc.p + (((long long)t.h << D.lp) * D.kc.cols) * 4;
  const GLOBAL char* vb = (const GLOBAL char*)D.vc.p + (((long long)t.h << D.lp) * D.vc.cols) * 4;
  const unsigned kpage = (unsigned)(D.Hkv << D.lp) * D.kc.cols * 4, vpage = (unsigned)(D.Hkv << D.lp) * D.vc.cols * 4;
  const int pm = D.page - 1, kpitch = D.kc.cols * 4, vpitch = D.vc.cols * 4;
  f32x4n qf[NT][NK];
  int lim[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = min(16 * n + m16, R - 1);
    lim[n] = t.L + t.tok0 + r / D.G;
    const GLOBAL float* q = D.q.f() + (long long)(t.row0 + r / D.G) * D.q.cols + (long long)(t.h * D.G + r % D.G) * HD + 4 * qq;
#pragma unroll
    for (int kk = 0; kk < NK; ++kk) qf[n][kk] = *(const GLOBAL f32x4n*)(q + 16 * kk);
  }
  struct Unit { f32x4n k[NK], v[4][NV]; };
  bool bad = false;
  const int nu = (p.k1 - p.k0 + 15) >> 4;
  auto ids = [&](int u) { return tb[min(p.k0 + 16 * u, klast) >> D.lp]; };   // (a unit lies within a page)
  auto load = [&](Unit& U, int id, int u) {
    const int key0 = p.k0 + 16 * u;
    bad = bad || (unsigned)id >= (unsigned)D.pages;
    const unsigned i = (unsigned)id < (unsigned)D.pages ? id : 0u;
    const GLOBAL char* kp = kb + (unsigned long long)i * kpage + ((min(key0 + m16, klast) & pm) * kpitch + 16 * qq);
    const GLOBAL char* vp = vb + (unsigned long long)i * vpage + 4 * DPL * m16;
#pragma unroll
    for (int kk = 0; kk < NK; ++kk) U.k[kk] = *(const GLOBAL f32x4n*)(kp + 64 * kk);
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int j = 0; j < NV; ++j) U.v[r][j] = *(const GLOBAL f32x4n*)(vp + ((min(key0 + 4 * qq + r, klast) & pm) * vpitch + 16 * j));
  };
  f32x4_t acc[NT][DPL];
  float m[NT], ls[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    m[n] = -INFINITY; ls[n] = 0.f;
#pragma unroll
    for (int i = 0; i < DPL; ++i) acc[n][i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  auto compute = [&](const Unit& U, int u) {
    const int key0 = p.k0 + 16 * u;
    const bool edge = key0 + 15 > t.L + t.tok0;                        // some row does not see the whole unit
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      f32x4_t s[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};      // (two chains: a product waits for the one before the last)
#pragma unroll
      for (int kk = 0; kk < NK; ++kk)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[i & 1] = __builtin_amdgcn_mfma_f32_16x16x4f32(U.k[kk][i], qf[n][kk][i], s[i & 1], 0, 0, 0);
      float x[4], mx = -INFINITY;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float y = (s[0][r] + s[1][r]) * D.sl2;
        x[r] = edge && key0 + 4 * qq + r > lim[n] ? -INFINITY : y;
        mx = fmaxf(mx, x[r]);
      }
      mx = rows_max(mx);
      if (__ballot(mx > m[n] + 8.f)) {
        const float top = fmaxf(m[n], mx), f = m[n] == -INFINITY ? 0.f : exp2f(m[n] - top);
        ls[n] *= f;
#pragma unroll
        for (int i = 0; i < DPL; ++i) acc[n][i] *= f;
        m[n] = top;
      }
      const float base = m[n] == -INFINITY ? 0.f : m[n];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float e = exp2f(x[r] - base);
        ls[n] += e;
#pragma unroll
        for (int i = 0; i < DPL; ++i) acc[n][i] = __builtin_amdgcn_mfma_f32_16x16x4f32(U.v[r][i >> 2][i & 3], e, acc[n][i], 0, 0, 0);
      }
    }
  };
  if (w < nu) {
    Unit u0, u1;
    int i0 = ids(w), i1 = ids(w + 4), u = w;
    load(u0, i0, w);
    for (; u + 8 < nu; u += 8) {
      i0 = ids(u + 8);
      load(u1, i1, u + 4);
      compute(u0, u);
      i1 = ids(u + 12);
      load(u0, i0, u + 8);
      compute(u1, u + 4);
    }
    if (u + 4 < nu) {
      load(u1, i1, u + 4);
      compute(u0, u);
      compute(u1, u + 4);
    } else compute(u0, u);
  }
  return paged_waves<HD, NT, false>(c, D, t, p, acc, m, ls, bad);
}

// Tiles of up to 128 rows (chunks of prompts): bound by the matrix units, the vector work of the softmax and LDS alike. A wave has 32 rows; blocks of
// 64 keys come from the pages straight into LDS for all of them, three stages, the places of up to PG_IDS pieces of pages in LDS. In transposed
// space: S^T = K Q^T by v_mfma_f32_32x32x16_bf16 (a lane owns a query row), O^T += V^T P^T with P^T's registers as they are. V lies row by row;
// a lane reads HD / 32 dims of 8 keys and turns them in registers (a byte permute for two values), dims HD / 32 * m + i to row m of product i:
// transposing reads of LDS run at a third of the rate. P^T is two operands, as above. 32 keys at a time, the scores of the next ones under the
// softmax of these: with 64 the fragments and scores under way pass 256 registers. A block of 64 keys takes 128 rows 2.3 us (470 TFLOP/s over
// 256 CUs; 1.9 with P^T rounded once), some 630 instructions a wave of which 48 are products; 1,000 tokens of 32 heads behind 3,750 175 us a call.
constexpr int PG_IDS = 2048, PG_NS = 3;
__device__ __forceinline__ void dma16_at(unsigned long long src, unsigned dst) {   // 16 bytes a lane from its own address to LDS byte dst (uniform) + 16 * lane
  asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, off" :: "s"(dst), "v"(src) : "memory", "m0");
}
// 8 keys of HD / 32 dims each (HD 128: 4 in two words; 64: 2 in one) as HD / 32 operands of 8 keys.
template <int HD> struct VTurn {
  static constexpr int NW = HD / 64;
  uint32_t w[8][NW];
  __device__ __forceinline__ void read(const LDS uint16_t* v, int key0, int g, int m) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const LDS uint16_t* y = v + (key0 + 8 * (j >> 2) + 4 * g + (j & 3)) * HD + 2 * NW * m;
      if constexpr (NW == 2) { const u32x2_t x = *(const LDS u32x2_t*)y; w[j][0] = x.x; w[j][1] = x.y; }
      else w[j][0] = *(const LDS uint32_t*)y;
    }
  }
  __device__ __forceinline__ bf16x8 turned(int d) const {
    u32x4_t r;
#pragma unroll
    for (int j = 0; j < 4; ++j) r[j] = __builtin_amdgcn_perm(w[2 * j + 1][d >> 1], w[2 * j][d >> 1], d & 1 ? 0x07060302u : 0x05040100u);
    return __builtin_bit_cast(bf16x8, r);
  }
};
// Maximum over a lane and the one 32 away, in registers: through LDS it would wait for all reads of LDS under way (a block of 64 keys 2.8 us in place of
// 2.0).
__device__ __forceinline__ float halves_max(float v) {
  auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
template <int HD> __device__ __noinline__ int attn_paged_rows(const Ctx& c, int b_, int h_, int L_, int row0_, int tok0_, int ntok_, int k0_, int k1_, int k_, int live_, int i0_) {
  typedef FaL<HD> FL;
  constexpr int NKK = HD / 16, NDB = HD / 32, ST = 2 * FA_KB * HD;
  static_assert(PG_WORK + PG_IDS * 4 + PG_NS * ST * 2 <= KVM_LDS_BYTES, "LDS");
  const AttnPaged D(c);
  const TilePaged t{rfl(b_), rfl(h_), rfl(L_), rfl(row0_), rfl(tok0_), rfl(ntok_), 0, 0};
  const PiecePaged p{rfl(k0_), rfl(k1_), rfl(k_), rfl(live_), rfl(i0_)};
  const int w = rfl(wave()), l = lane(), g = l >> 5, qi = l & 31, R = t.ntok * D.G, row = 32 * w + qi, rr = min(row, R - 1);
  const bool qok = row < R, wave_on = 32 * w < R;
  const int lim = t.L + t.tok0 + rr / D.G;
  const int wfirst = rfl(t.L + t.tok0 + min(32 * w, R - 1) / D.G), wlast = rfl(t.L + t.tok0 + min(32 * w + 31, R - 1) / D.G);
  const GLOBAL int* tb = D.table.i() + (long long)t.b * D.table.cols;
  // a piece of a page is up to 64 tokens: number v = (page * Hkv) * (pieces of a page) + piece lies v * (piece's bytes) behind kb and vb
  const int lsub = min(D.lp, 6), kpitch = D.kc.cols * 2, vpitch = D.vc.cols * 2;
  const unsigned ksub = (unsigned)kpitch << lsub, vsub = (unsigned)vpitch << lsub;
  const unsigned long long kb = (unsigned long long)(uintptr_t)D.kc.p + ((unsigned long long)t.h << D.lp) * kpitch;
  const unsigned long long vb = (unsigned long long)(uintptr_t)D.vc.p + ((unsigned long long)t.h << D.lp) * vpitch;
  LDS int* sid = (LDS int*)(c.smem + PG_WORK);
  LDS uint16_t* lds = (LDS uint16_t*)(sid + PG_IDS);
  bf16x8 qf[NKK];
  {
    const GLOBAL uint16_t* q = D.q.h() + (long long)(t.row0 + rr / D.G) * D.q.cols + (long long)(t.h * D.G + rr % D.G) * HD + 8 * g;
#pragma unroll
    for (int kk = 0; kk < NKK; ++kk) qf[kk] = *(const GLOBAL bf16x8*)(q + 16 * kk);
  }
  f32x16 oacc[NDB];
#pragma unroll
  for (int d = 0; d < NDB; ++d) oacc[d] = f32x16{};
  float m = -INFINITY, lsum = 0.f;
  bool bad = false;
  const unsigned lds0 = (unsigned)rfl((int)(unsigned)(uintptr_t)lds) + w * 1024u;   // where this wave's first KiB of stage 0 lies
  int lrow[FL::NL];                                                    // rows of a block that the lane loads pieces of, and these within a piece of a page
  unsigned koff[FL::NL], voff[FL::NL];
#pragma unroll
  for (int q = 0; q < FL::NL; ++q) {
    const int u = 64 * (q * KVM_WAVES + w) + l, r = u / FL::UPR, ph = u % FL::UPR, at = r & ((1 << lsub) - 1);
    lrow[q] = r;
    koff[q] = (unsigned)(at * kpitch + 16 * (ph ^ FL::kswz(r))); voff[q] = (unsigned)(at * vpitch + 16 * ph);
  }
  const int seg = PG_IDS << lsub;
  for (long long s0_ = p.k0; s0_ < p.k1; s0_ += seg) {
    const int s0 = (int)s0_, s1 = (int)min((long long)p.k1, s0_ + seg), nkb = (s1 - s0 + 63) >> 6, last = s1 - 1 - s0;
    __syncthreads();                                                   // the stages and places before are read
    for (int e = tid(); e <= last >> lsub; e += KVM_THREADS) {
      const int key = s0 + (e << lsub);
      int id = tb[key >> D.lp];
      if ((unsigned)id >= (unsigned)D.pages) { bad = true; id = 0; }
      sid[e] = ((id * D.Hkv) << (D.lp - lsub)) + ((key & (D.page - 1)) >> lsub);
    }
    __syncthreads();
    // (keys behind the last one: the last one again, not seen)
    auto issue = [&](int blk) {
      const unsigned d = lds0 + (unsigned)((blk % PG_NS) * ST * 2);
      const int first = (blk * FA_KB) >> lsub;
      if (blk * FA_KB + FA_KB - 1 <= last) {
        unsigned v[FL::NL];
#pragma unroll
        for (int q = 0; q < FL::NL; ++q) v[q] = (unsigned)sid[first + (lrow[q] >> lsub)];
#pragma unroll
        for (int q = 0; q < FL::NL; ++q) {
          dma16_at(kb + ((unsigned long long)v[q] * ksub + koff[q]), d + q * KVM_WAVES * 1024);
          dma16_at(vb + ((unsigned long long)v[q] * vsub + voff[q]), d + FA_KB * HD * 2 + q * KVM_WAVES * 1024);
        }
      } else {
#pragma unroll 1
        for (int q = 0; q < FL::NL; ++q) {
          const int u = 64 * (q * KVM_WAVES + w) + l, r = u / FL::UPR, ph = u % FL::UPR;
          const int key = min(blk * FA_KB + r, last), at = key & ((1 << lsub) - 1);
          const unsigned v = (unsigned)sid[key >> lsub];
          dma16_at(kb + ((unsigned long long)v * ksub + (unsigned)(at * kpitch + 16 * (ph ^ FL::kswz(r)))), d + q * KVM_WAVES * 1024);
          dma16_at(vb + ((unsigned long long)v * vsub + (unsigned)(at * vpitch + 16 * ph)), d + FA_KB * HD * 2 + q * KVM_WAVES * 1024);
        }
      }
    };
    bf16x8 kfr[NKK];                                                   // of the keys after the step's, and the step's own values
    VTurn<HD> vt[2];
    auto read = [&](const LDS uint16_t* K, int nk, const LDS uint16_t* V, int vk) {
#pragma unroll
      for (int kk = 0; kk < NKK; ++kk) kfr[kk] = FL::frag_kc(K, nk, kk);
#pragma unroll
      for (int u = 0; u < 2; ++u) vt[u].read(V, vk + 16 * u, g, qi);
    };
    // Keys [key0, key0 + 32): scores sa; the scores of the next 32 to sn. Then what the next step needs is read: K of the keys after it (from
    // nk on at Kn), V of its own (from vk on at Vn), under the last products and its maximum.
    auto step = [&](int key0, f32x16& sa, f32x16& sn, const LDS uint16_t* Kn, int nk, const LDS uint16_t* Vn, int vk) {
      if (!wave_on || key0 > wlast) return;                            // no row of the wave sees a key of these
      if (key0 + 31 > wfirst) {
        asm volatile("" ::: "memory");                                 // stays a branch: flattened, its selects run in every step
        const int seen = lim - key0 - 4 * g;
#pragma unroll
        for (int r = 0; r < 16; ++r) sa[r] = 8 * (r >> 2) + (r & 3) > seen ? -INFINITY : sa[r];
      }
      float mx = fmaxf(fmaxf(sa[0], sa[1]), sa[2]);
#pragma unroll
      for (int r = 3; r + 1 < 16; r += 2) mx = fmaxf(fmaxf(mx, sa[r]), sa[r + 1]);
      mx = fmaxf(mx, sa[15]);
      mx = halves_max(mx) * D.sl2;
      if (__ballot(mx > m + 8.f)) {
        const float top = fmaxf(m, mx), f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top);
        lsum *= f;
#pragma unroll
        for (int d = 0; d < NDB; ++d) oacc[d] *= f;
        m = top;
      }
      const float base = m == -INFINITY ? 0.f : m;
      Pieces<2> pf[2];
      float ps = 0.f;
      sn = f32x16{};
      // a product of the next scores, two exponentials and what belongs to them, in turn; then the products of P, their operands and the reads
      // between them
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        float pv[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) pv[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sa[8 * u + i], D.sl2, -base));
        pf[u] = split_bf16<2>(pv);
        ps = sum8(pv, ps);
      }
#pragma unroll
      for (int kk = 0; kk < NKK; ++kk) sn = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kfr[kk], qf[kk], sn, 0, 0, 0);
      lsum += ps;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int d = 0; d < NDB; ++d) oacc[d] = mfma_pieces(vt[u].turned(d), pf[u], oacc[d]);
      read(Kn, nk, Vn, vk);
#pragma unroll
      for (int i = 0; i < NKK; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);             // a matrix instruction,
        __builtin_amdgcn_sched_group_barrier(0x002, 6 * 8 / NKK, 0);   // vector instructions,
        __builtin_amdgcn_sched_group_barrier(0x400, 2 * 8 / NKK, 0);   // exponentials
      }
#pragma unroll
      for (int i = 0; i < 2 * NDB; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, 4, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);             // a read of LDS
      }
    };
    issue(0);
    if (nkb > 1) issue(1);
    wait_vm(nkb > 1 ? 2 * FL::NL : 0);
    __syncthreads();
    f32x16 sa = {}, sn;
#pragma unroll
    for (int kk = 0; kk < NKK; ++kk) sa = __builtin_amdgcn_mfma_f32_32x32x16_bf16(FL::frag_kc(lds, 0, kk), qf[kk], sa, 0, 0, 0);
    read(lds, 32, lds + FA_KB * HD, 0);
    for (int blk = 0; blk < nkb; ++blk) {
      const LDS uint16_t* Ks = lds + (blk % PG_NS) * ST;
      const LDS uint16_t* Kn = lds + ((blk + 1) % PG_NS) * ST;
      wait_vm_c<0>();                                                  // block blk + 1 has landed
      __syncthreads();                                                 // ... everyone's, and every wave is past block blk - 1
      if (blk + 2 < nkb) issue(blk + 2);
      step(s0 + blk * FA_KB, sa, sn, Kn, 0, Ks + FA_KB * HD, 32);
      step(s0 + blk * FA_KB + 32, sn, sa, Kn, 32, Kn + FA_KB * HD, 0);
    }
  }
  lsum += __shfl_xor(lsum, 32, 64);
  float nf = lsum * 0.f + (m == -INFINITY ? 0.f : m * 0.f);
#pragma unroll
  for (int d = 0; d < NDB; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) nf += oacc[d][r] * 0.f;
  if (__syncthreads_or(bad ? 1 : 0)) { if (tid() == 0) c.fail(KVM_ERR_OP_RANGE, t.b, p.k0); return PG_FAILED; }
  if (__syncthreads_or(qok && nf != 0.f ? 1 : 0)) return PG_AGAIN;
  // through LDS, whole rows go out
  LDS float* ol = (LDS float*)(c.smem + PG_WORK);                      // [128][HD + 4]
  static_assert(PG_WORK + 128 * (HD + 4) * 4 <= KVM_LDS_BYTES, "LDS");
  const float inv = p.live == 1 ? 1.f / lsum : 1.f;
#pragma unroll
  for (int r = 0; r < 16; ++r) {                                       // register r of the products: NDB dims in a row
    LDS float* y = ol + row * (HD + 4) + NDB * (8 * (r >> 2) + 4 * g + (r & 3));
#pragma unroll
    for (int d = 0; d < NDB; ++d) y[d] = oacc[d][r] * inv;
  }
  if (p.live > 1 && qok && g == 0) { GLOBAL float* y = paged_partial(D, p, p.k, row) + HD; stwt32(y, m); stwt32(y + 1, lsum); }
  __syncthreads();
  for (int e = tid(); e < R * (HD / 8); e += KVM_THREADS) {
    const int r = e / (HD / 8), d = 8 * (e % (HD / 8));
    const f32x4n a = *(const LDS f32x4n*)(ol + r * (HD + 4) + d), b = *(const LDS f32x4n*)(ol + r * (HD + 4) + d + 4);
    if (p.live == 1) {
      GLOBAL uint16_t* o = D.o.h() + paged_out(D, t, r) + d;
      stwt_bf4(o, a.x, a.y, a.z, a.w); stwt_bf4(o + 4, b.x, b.y, b.z, b.w);
    } else {
      GLOBAL float* y = paged_partial(D, p, p.k, r) + d;
      stwt_f4(y, a); stwt_f4(y + 4, b);
    }
  }
  return PG_DONE;
}

template <int HD> __device__ __forceinline__ int attn_paged_fast(const Ctx& c, const TilePaged& t, const PiecePaged& p, int R, int kind) {
  if (kind == 1) {
    if (R <= 16) return attn_paged_keys_f32<HD, 1>(c, t.b, t.h, t.L, t.row0, t.tok0, t.ntok, p.k0, p.k1, p.k, p.live, p.i0);
    if (R <= 32) return attn_paged_keys_f32<HD, 2>(c, t.b, t.h, t.L, t.row0, t.tok0, t.ntok, p.k0, p.k1, p.k, p.live, p.i0);
    return PG_AGAIN;
  }
  if (R <= 16) return attn_paged_keys<HD, 1>(c, t.b, t.h, t.L, t.row0, t.tok0, t.ntok, p.k0, p.k1, p.k, p.live, p.i0);
  if (R <= 32) return attn_paged_keys<HD, 2>(c, t.b, t.h, t.L, t.row0, t.tok0, t.ntok, p.k0, p.k1, p.k, p.live, p.i0);
  return attn_paged_rows<HD>(c, t.b, t.h, t.L, t.row0, t.tok0, t.ntok, p.k0, p.k1, p.k, p.live, p.i0);
}
__device__ __noinline__ void op_attn_paged(const Ctx& c) {
  const AttnPaged D(c);
  LDS long long* pre = (LDS long long*)c.smem;                         // [PG_SEQS + 2]
  LDS int* scu = (LDS int*)(pre + PG_SEQS + 2);                        // [PG_SEQS + 4]
  LDS int* len = scu + PG_SEQS + 4;                                    // [PG_SEQS]
  LDS int* flag = len + PG_SEQS;                                       // [4], then 12 words of 8 bytes: the waves' sums, longest tiles and numbers of tiles
  LDS long long* tot = (LDS long long*)(flag + 4);
  if (!paged_call_ok(c, D.cu, D.lens, D.B, min(D.q.rows, D.o.rows), (long long)D.table.cols << D.lp, scu)) return;
  WorkPaged W;
  W.pre = pre; W.cu = scu; W.len = len; W.B = D.B; W.Hkv = D.Hkv; W.G = D.G;
  const int fast = D.fast();
  W.rows = fast == 2 ? D.tile : min(D.tile, max(32, D.G));             // (the other forms take 32 rows at a time)
  W.whole = false; W.S = D.S;
  for (;;) {                                                           // what the sequences cost and the sums in front of each: in keys, then maybe in tiles
    constexpr int PER = PG_SEQS / KVM_THREADS;
    long long cost[PER], sum = 0, most = 0, tiles = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int b = tid() * PER + i;
      cost[i] = 0;
      if (b < D.B) {
        const int L = D.lens.i()[b], n = scu[b + 1] - scu[b];
        len[b] = L;
        if (n > 0) {
          const int TT = W.tokens(n);
          cost[i] = W.head_cost(n, L) * D.Hkv;
          sum += cost[i];
          most = max(most, PG_TILE + (long long)L + n);
          tiles += (long long)((n + TT - 1) / TT) * D.Hkv;
        }
      }
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) { most = max(most, (long long)__shfl_xor(most, d, 64)); tiles += __shfl_xor(tiles, d, 64); }
    if (lane() == 0) { tot[4 + wave()] = most; tot[8 + wave()] = tiles; }
    long long upto = sum;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) { const long long y = __shfl_up(upto, d, 64); if (lane() >= d) upto += y; }
    if (lane() == 63) tot[wave()] = upto;
    __syncthreads();
    long long at = upto - sum;
    for (int w = 0; w < wave(); ++w) at += tot[w];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int b = tid() * PER + i;
      if (b < D.B) { pre[b] = at; at += cost[i]; if (b == D.B - 1) pre[D.B] = at; }
    }
    __syncthreads();
    W.total = pre[D.B];
    if (W.whole) break;
    W.share = max((W.total + D.S - 1) / D.S, (long long)PG_SHARE);
    if (rfl(tot[8] + tot[9] + tot[10] + tot[11] > D.S || max(max(tot[4], tot[5]), max(tot[6], tot[7])) > W.share + PG_CUT)) break;
    W.whole = true;
    __syncthreads();                                                   // the sums are read
  }
  // Neighbouring shares read the same keys: eight runs of shares, one for the tasks s, s + 8, .. (where tasks go to workers in order, those of one
  // XCD and its L2).
  const int mine = D.S % 8 == 0 ? (D.s & 7) * (D.S >> 3) + (D.s >> 3) : D.s;
  long long x = W.cut(mine);
  const long long end = W.cut(mine + 1);
  while (x < end) {
    const TilePaged t = W.find(x);
    const long long stop = min(end, t.start + t.cost);
    const PiecePaged p = W.piece(t, x, stop);
    int r = !fast ? PG_AGAIN : D.hd == 128 ? attn_paged_fast<128>(c, t, p, t.ntok * D.G, fast) : attn_paged_fast<64>(c, t, p, t.ntok * D.G, fast);
    if (rfl(r) == PG_AGAIN) r = attn_paged_general(c, t.b, t.h, t.L, t.row0, t.tok0, t.ntok, p.k0, p.k1, p.k, p.live, p.i0);
    if (rfl(r) == PG_FAILED) return;
    if (p.live > 1) paged_arrive(c, D, t, p, flag);
    __syncthreads();
    x = stop;
  }
}

}  // namespace kvm
