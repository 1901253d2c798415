// Attention of a step's rows over 8-bit pages: the units of a plan (attend.hpp), and the join of their partial results.
//
//   s = scale ks (q . k), capped and biased as asked;  out = sum softmax(s) vs v
//
// Both bodies hold scores transposed, S^T = K Q^T: a lane has scores of ONE virtual row, so its softmax is arithmetic in its
// own registers and one or two lane swaps, and its weights are already the operand of O^T = V^T P^T (any order of the
// keys will do inside a product, as long as V's operand has the same). Codes become fp16, which holds them exactly; q is
// fp16 times a power of two of its row (2^14 <= largest < 2^15: exact, but for what lies below 2^-39 of that); weights
// are two fp16 parts, 2^-23 of each but for what lies below 2^-35 of the row's largest weight times |vs|, taken relative to a
// reference that this passes by 2^6 at most (accumulators are rescaled only when a page passes that); sums and statistics are
// fp32. (One part, 2^-12, shows beside bf16 results, more where values cancel: 2^-10 of a result in the norm from a softmax in
// fp32, for 2^-13. The second one costs small tiles 1 to 4 %, large ones 8 to 34: prompts of 8192 2293 us for 1712, 64 tokens
// behind a prefix of 8192 49.8 for 43.2. Its order among the products makes no difference.)
#include "codes8.hpp"
#include "attend.hpp"

#include <type_traits>

namespace kvs {
namespace {

struct AttendP {
  const uint16_t* q;
  int64_t q_sn, q_sh;
  const uint8_t* k;
  const uint8_t* v;
  int64_t k_sb, k_sh, v_sb, v_sh;
  uint32_t k_st, v_st;
  const float* k_scale;
  const float* v_scale;
  int64_t ks_sb, ks_sh, vs_sb, vs_sh;
  const int* block_table;
  const int* shared_table;
  int64_t bt_stride, st_stride;
  const float* slopes;
  uint16_t* out;
  float* lse;
  float* part_acc;
  float* part_ml;
  const int* head;
  const AttendUnit* units;
  const AttendJoin* joins;
  const AttendRow* rows;
  int n_rows, Hq, Hkv, G, num_pages, window;
  float scale, softcap;
};

typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef __attribute__((__vector_size__(4 * sizeof(__fp16)))) __fp16 fp16x4_t;

__device__ __forceinline__ float swap32_max(float v) {
  const uint32_t a = __float_as_uint(v);
  const u32x2 r = __builtin_amdgcn_permlane32_swap(a, a, false, false);
  return fmaxf(__uint_as_float(r.x), __uint_as_float(r.y));
}
__device__ __forceinline__ float swap32_sum(float v) {
  const uint32_t a = __float_as_uint(v);
  const u32x2 r = __builtin_amdgcn_permlane32_swap(a, a, false, false);
  return __uint_as_float(r.x) + __uint_as_float(r.y);
}

constexpr int JOIN_GRID = 2048;  // workgroups of the join: eight a CU

// A virtual row: its row of q and out, query head, position, prefix.
struct Row {
  int n, hq, pos, pre;
};
__device__ __forceinline__ Row virtual_row(const AttendP& p, const AttendUnit& u, int h, int i) {
  // (rows past the tile's last are that one again: computed and not stored)
  const int v = u.v0 + min(i, u.nv - 1), r = v / p.G;
  Row x;
  x.hq = h * p.G + (v - r * p.G);
  if (u.kind & 2) {
    const AttendRow y = p.rows[u.row0 + r];
    x.n = y.row, x.pos = y.pos, x.pre = y.pre;
  } else {
    x.n = u.row0 + r, x.pos = u.p0 + r, x.pre = u.pre;
  }
  return x;
}

// What a row sees of the unit's keys, as indices: from <= t < end, or t < pre (both ends at most the unit's len).
struct Sight {
  int from, end, pre;
};
__device__ __forceinline__ Sight sight(const AttendP& p, const AttendUnit& u, const Row& r) {
  Sight s;
  s.end = min(r.pos - u.base + 1, u.len);
  s.from = p.window > 0 ? max(r.pos - u.base + 1 - p.window, 0) : 0;
  s.pre = min(r.pre - u.base, u.len);
  return s;
}
__device__ __forceinline__ bool sees(const Sight& s, int t) { return ((t >= s.from) & (t < s.end)) | (t < s.pre); }

__device__ __forceinline__ int wave_min_int(int v) {
#pragma unroll
  for (int m = 1; m < WAVE; m *= 2) v = min(v, __shfl_xor(v, m, WAVE));
  return __builtin_amdgcn_readfirstlane(v);
}
__device__ __forceinline__ int wave_max_int(int v) { return ~wave_min_int(~v); }

// The rows of a wavefront (or tile) together.
struct Reach {
  int from_min, from_max, end_min, end_max, pre_min, pre_max;
};
__device__ __forceinline__ Reach reach(const Sight& s) {
  return Reach{wave_min_int(s.from), wave_max_int(s.from), wave_min_int(s.end), wave_max_int(s.end), wave_min_int(s.pre),
               wave_max_int(s.pre)};
}
__device__ __forceinline__ Reach both(const Reach& a, const Reach& b) {
  return Reach{min(a.from_min, b.from_min), max(a.from_max, b.from_max), min(a.end_min, b.end_min),
               max(a.end_max, b.end_max),   min(a.pre_min, b.pre_min),   max(a.pre_max, b.pre_max)};
}
// Every row sees all of a page's keys, those of [t0, t0 + 64) before len (from len on its rows read as zeros); all 64 of them;
// no row sees any.
__device__ __forceinline__ bool sees_keys(const Reach& r, int t0, int len) {
  const int t1 = min(t0 + BLK, len);
  return t1 <= r.pre_min || (t1 <= r.end_min && t0 >= r.from_max);
}
__device__ __forceinline__ bool sees_all(const Reach& r, int t0, int len) { return t0 + BLK <= len && sees_keys(r, t0, len); }
__device__ __forceinline__ bool sees_none(const Reach& r, int t0) {
  return t0 >= r.pre_max && (t0 >= r.end_max || t0 + BLK <= r.from_min);
}

// A NaN among V's codes (e4m3's 0x7f and 0xff) must reach the rows that see its key and no others, but a weight of 0 times NaN
// is NaN. So where a page is cut, its NaN codes are made zeros before the product; a unit that had any looks through its cut
// pages again at the end and puts them into the accumulators of the rows that see them. (Put in page by page instead, the
// registers that this takes in the loop cost 20 to 30 % of every pass over e4m3.)
// Bytes of w that are NaN, as 0x80.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }
__device__ __forceinline__ uint32_t without_nan(uint32_t w, uint32_t& any) {
  const uint32_t z = nan_bytes(w);
  any |= z;
  return w & ~((z >> 7) * 0xffu);
}

// Running state of a row. m: a score in log2 units, the row's largest when the state was last looked at; l: this lane's part of
// sum 2^(s - m). ar + ax: the accumulators' reference, a score and the exponent of its page's vs (apart, since in one float a large
// score takes the exponent's bits). c and d: LIFT - ax - ar (while the row has seen nothing: infinite, or 0) and ar + ax - LIFT - m.
//   LIFT: the exponent in fp16, whose finest is 2^-24, of a weight at the reference. (7 and 10 take the same time within 1 %; beside a key
// of value 0 with most of a row's weight, weights 2^-26 below it are off by 2^-6 each with 7 at worst, by 2^-9 with 10.)
constexpr int LIFT = 10;
struct State {
  float m = NEG_INF, l = 0.f, ar = NEG_INF, ax = 0.f, c, d = 0.f;
  __device__ explicit State(bool blind) : c(blind ? -NEG_INF : 0.f) {}
};
// What a wavefront's rows share: the largest exponent of vs so far; a reference has passed 2^10.
struct Common {
  int top = -1000;
  bool odd = false;
};
// A page's vs. plain: a positive number of middling size, and not 2^40 below another one.
struct Weight {
  float part, lv, ev;  // vs = part 2^ev
  bool plain;
  __device__ Weight(float v, Common& w) {
    const int e = static_cast<int>(__float_as_uint(v) >> 23);  // (a negative one from 256 on)
    const int x = max((e & 0xff) - 127, -126);
    part = ldexpf(v, -x);
    w.top = max(w.top, x);
    plain = e >= 27 && e <= 227 && x >= w.top - 40 && !w.odd;
    lv = flog2(v);
    ev = static_cast<float>(x);
  }
};

// Capped and biased scores, in log2 units, of raw products s times f (a score in natural units): tanh y as
// 1 - 2 / (e^2y + 1), off by 2^-24 of the cap, or where the wavefront's scores are all below an eighth of the cap as
// y - y^3 / 3 + 2 y^5 / 15 - 17 y^7 / 315, off by 2^-29 of y. d0: distance of key t0 (|t - t0| below 64), or its negative.
template <int N, class T>
__device__ __forceinline__ void modify(float (&s)[N], float f, float cap, bool biased, float slope, float d0, T&& at) {
  if (cap > 0.f) {
    const float g = f / cap;
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) top = fmaxf(top, fabsf(s[i]));
    if (__ballot(!(top * fabsf(g) <= 0.125f)) == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float y = s[i] * g, z = y * y;
        s[i] = fmaf(y * z, fmaf(z, fmaf(z, -17.f / 315.f, 2.f / 15.f), -1.f / 3.f), y);
      }
    } else {
      const float g2 = 2.f * LOG2E * g;
#pragma unroll
      for (int i = 0; i < N; ++i) s[i] = fmaf(__builtin_amdgcn_rcpf(fexp2(s[i] * g2) + 1.f), -2.f, 1.f);
    }
    f = cap;
  }
  if (biased) {
    const float a = f * LOG2E, b = slope * LOG2E;
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] = fmaf(s[i], a, -b * fabsf(d0 - at(i)));
  } else {
    const float a = f * LOG2E;
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] *= a;
  }
}

// (v_maximum3_f32: half the instructions of fmaxf, which makes each operand canonical first)
template <int N>
__device__ __forceinline__ float most_of(const float (&s)[N]) {
  float x = s[0];
#pragma unroll
  for (int i = 1; i < N; ++i) x = __builtin_elementwise_maximum(x, s[i]);
  return x;
}
template <int N>
__device__ __forceinline__ float least_of(const float (&s)[N]) {
  float x = s[0];
#pragma unroll
  for (int i = 1; i < N; ++i) x = __builtin_elementwise_minimum(x, s[i]);
  return x;
}

// A pair of weights in two parts of fp16, the second what the first leaves: 22 bits.
__device__ __forceinline__ void two_parts(float x, float y, uint32_t& hi, uint32_t& lo) {
  hi = pack_h(x, y);
  lo = mix_h(x, y, 1.f, -__builtin_bit_cast(f16x2_t, hi));
}

// One page of a row: s in, w + wl = 2^LIFT p vs / 2^(ar + ax) as fp16 pairs out, tokens in order; s f is the score in log2 units (neg: f <
// 0). alpha: the factor of the accumulators, true if it is not 1 for all.
//   The plain way takes 2^(s f + c + log2 vs) at once, from which l is found too: an fma, an exponential, a sum and one and a
// half conversions a score. Its one rounding more, of c + log2 vs, is 2^-14 at most where no reference passes 2^10; and no weight that
// l could feel is below 2^-126: a score at most 2^60 below the row's largest lies at most 2^64 below ar, and vs at most 2^40
// below 2^ax. It holds while no weight leaves fp16. BLIND: taken without the page's largest score, and taken back where a lane's
// sum passes fp16's largest (or is NaN: a row's first keys, whose c is infinite, and masked ones before them); else only after the
// reference has been moved to where no weight passes 2^15.
//   Elsewhere weights are taken relative to the page's largest score and multiplied by their factor.
template <bool BLIND, int N, class F>
__device__ __forceinline__ bool soften(float (&s)[N], float f, bool neg, const Weight& v, State& st, Common& com, float& alpha,
                                       uint32_t (&w)[N / 2], uint32_t (&wl)[N / 2], F&& swap) {
  alpha = 1.f;
  auto plain = [&]() {
    float sum[4];
    const float c = st.c + v.lv;
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const float x = fexp2(fmaf(s[i], f, c)), y = fexp2(fmaf(s[i + 1], f, c));
      sum[i % 4] = i < 4 ? x : sum[i % 4] + x, sum[i % 4 + 1] = i < 4 ? y : sum[i % 4 + 1] + y;
      two_parts(x, y, w[i / 2], wl[i / 2]);
    }
    return (sum[0] + sum[1]) + (sum[2] + sum[3]);
  };
  if (BLIND && v.plain && !com.odd) {  // uniform
    const float all = plain();
    if (__ballot(!(all <= 65504.f)) == 0) {
      st.l = fmaf(all, fexp2(st.d - v.lv), st.l);
      return false;
    }
  }
  const float mt = neg ? swap(-least_of(s)) * -f : swap(most_of(s)) * f;
  const float past = (mt - st.ar) + (v.ev - st.ax);  // (NaN, which passes nothing, where nothing came yet)
  const bool move = BLIND || __ballot((past > 14.f - LIFT) | (mt > st.m + 4.f)) != 0;
  if (move) {
    const bool on = past > 0.f;
    alpha = on ? fexp2(-past) : 1.f;
    st.ar = on ? mt : st.ar;
    st.ax = on ? v.ev : st.ax;
    const float m = fmaxf(st.m, mt), mu = m == NEG_INF ? 0.f : m;
    st.l *= fexp2(st.m - mu);
    st.m = m;
    const bool none = st.ar == NEG_INF;
    st.c = none ? (BLIND ? -NEG_INF : 0.f) : (LIFT - st.ax) - st.ar;
    st.d = none ? 0.f : ((st.ar - mu) + st.ax) - LIFT;
    com.odd |= __ballot(!none & (fabsf(st.ar) > 0x1p10f)) != 0;
  }
  if (!BLIND && v.plain && !com.odd) {  // uniform
    st.l = fmaf(plain(), fexp2(st.d - v.lv), st.l);
    return move;
  }
  const float mtu = mt == NEG_INF ? 0.f : mt;
  // (scores so large that mt's rounding would show in s f - mt: rounded alike)
  if (__ballot(fabsf(mtu) > 0x1p17f) != 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] *= f;
    f = 1.f;
  }
  // below 2^15 (none for a row that sees nothing of the page, whatever vs is)
  const float fv = mt == NEG_INF ? 0.f : v.part * fexp2(((mt - st.ar) + (v.ev - st.ax)) + LIFT);
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    const float x = fexp2(fmaf(s[i], f, -mtu)), y = fexp2(fmaf(s[i + 1], f, -mtu));
    sum[i % 4] += x, sum[i % 4 + 1] += y;
    two_parts(x * fv, y * fv, w[i / 2], wl[i / 2]);
  }
  st.l = fmaf((sum[0] + sum[1]) + (sum[2] + sum[3]), mt == NEG_INF ? 0.f : fexp2(mt - st.m), st.l);
  return move;
}

// q of a row in fp16: its power of two taken out, the factor of its scores.
__device__ __forceinline__ float q_factor(float amax, float bad, float& up) {
  constexpr int TOP = 14;
  const int ex = min(max(static_cast<int>(__float_as_uint(amax) >> 23) - 127, TOP - 126), 127);
  up = __uint_as_float(static_cast<uint32_t>(127 + TOP - ex) << 23);
  return __uint_as_float(static_cast<uint32_t>(127 - TOP + ex) << 23) + bad;
}
__device__ __forceinline__ void q_extent(const u32x4& x, float& amax, float& bad) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float a = bf_lo(x[e]), b = bf_hi(x[e]);
    amax = fmaxf(amax, fmaxf(fabsf(a), fabsf(b)));
    bad = fmaf(a, 0.f, fmaf(b, 0.f, bad));  // NaN of an infinity or NaN
  }
}
__device__ __forceinline__ u32x4 q_half(const u32x4& x, float up) {
  u32x4 r;
#pragma unroll
  for (int e = 0; e < 4; ++e) r[e] = pack_h(bf_lo(x[e]) * up, bf_hi(x[e]) * up);
  return r;
}

// Pages of 64 steps of a unit, one a lane: table entry (-1: past the unit's), page (-1: none) and scales, gathered in three
// stages while the 64 before them run.
struct Pages {
  int blk, pg;
  float ks, vs;
};
struct PageList {
  const AttendP& p;
  const AttendUnit& u;
  const int* table;
  int h, first, n;
  Pages cur, nxt;
  __device__ PageList(const AttendP& p_, const AttendUnit& u_, int h_, int first_, int n_)
      : p(p_), u(u_), h(h_), first(first_), n(n_) {
    table = (u.kind & 2) ? p.shared_table + u.table * p.st_stride : p.block_table + u.table * p.bt_stride;
    block(cur, 0), page(cur), scales(cur);
    nxt = cur;
  }
  __device__ __forceinline__ void block(Pages& x, int k0) {
    const int k = k0 + static_cast<int>(threadIdx.x % WAVE);
    x.blk = -1;
    if (k < n) {
      const int i = u.i0 + first + NWAVE * k;
      x.blk = i < u.a1 ? i : i - u.a1 + u.b0;
    }
  }
  __device__ __forceinline__ void page(Pages& x) { x.pg = x.blk >= 0 ? table[x.blk] : -1; }
  __device__ __forceinline__ void scales(Pages& x) {
    if (x.pg < 0 || x.pg >= p.num_pages) x.pg = -1;
    x.ks = x.vs = 0.f;
    if (x.pg >= 0) {
      x.ks = p.k_scale[x.pg * p.ks_sb + h * p.ks_sh];
      x.vs = p.v_scale[x.pg * p.vs_sb + h * p.vs_sh];
    }
  }
  // Before step k's own use of the list: what is to be had for the steps 64 on.
  __device__ __forceinline__ void advance(int k) {
    const int ph = k & 63;
    if (k - ph + 64 < n) {
      if (ph == 0) block(nxt, k + 64);
      if (ph == 16) page(nxt);
      if (ph == 32) scales(nxt);
    }
  }
  __device__ __forceinline__ void turn(int k) {  // after the last read of step k's scales
    if ((k & 63) == 63) cur = nxt;
  }
  __device__ __forceinline__ int blk(int k) const { return __builtin_amdgcn_readlane(cur.blk, k & 63); }
  __device__ __forceinline__ int pg(int k) const { return __builtin_amdgcn_readlane(cur.pg, k & 63); }
  __device__ __forceinline__ float ks(int k) const { return lane_value(cur.ks, k & 63); }
  __device__ __forceinline__ float vs(int k) const { return lane_value(cur.vs, k & 63); }
};

// The rows of a page that hold keys, as a buffer resource: rows past the sequence's last read zeros.
template <int D>
__device__ __forceinline__ rsrc_t page_res(const uint8_t* base, int64_t sb, uint32_t st, int pg, int rows) {
  const uint64_t at = reinterpret_cast<uint64_t>(base) + max(pg, 0) * sb;
  const uint64_t lo = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(at)));
  const uint64_t hi = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(at >> 32)));
  return make_rsrc(reinterpret_cast<const void*>(hi << 32 | lo), rows > 0 ? (rows - 1) * st + D : 0u);
}

// A row's result, or its partial result: four dims.
__device__ __forceinline__ void store4(const AttendP& p, const AttendUnit& u, int h, int i, const Row& r, int d, int D, f32x4_t a,
                                       float m, float l) {
  if (u.part >= 0) {
    const int64_t at = static_cast<int64_t>(u.part + i) * p.Hkv + h;
    *reinterpret_cast<f32x4_t*>(p.part_acc + at * D + d) = a;
    if (d == 0) *reinterpret_cast<float2*>(p.part_ml + at * 2) = make_float2(m, l);
    return;
  }
  const int64_t at = static_cast<int64_t>(r.n) * p.Hq + r.hq;
#pragma unroll
  for (int e = 0; e < 4; ++e) a[e] = l == 0.f ? 0.f : a[e] / l;
  *reinterpret_cast<u32x2*>(p.out + at * D + d) =
      u32x2{f2bf(a[0]) | static_cast<uint32_t>(f2bf(a[1])) << 16, f2bf(a[2]) | static_cast<uint32_t>(f2bf(a[3])) << 16};
  if (d == 0) p.lse[at] = l == 0.f ? NEG_INF : (m + flog2(l)) * LN2;
}

// NaN over those of a stored row's four dims that have 0x80 in z.
__device__ __forceinline__ void store_nan(const AttendP& p, const AttendUnit& u, int h, int i, const Row& r, int d, int D, uint32_t z) {
  for (int e = 0; e < 4; ++e)
    if (z >> (8 * e + 7) & 1) {
      if (u.part >= 0)
        p.part_acc[(static_cast<int64_t>(u.part + i) * p.Hkv + h) * D + d + e] = __builtin_nanf("");
      else
        p.out[(static_cast<int64_t>(r.n) * p.Hq + r.hq) * D + d + e] = 0x7fc0;
    }
}

// ---- Few rows: four independent wavefronts, a page a step each, no barrier but the one before their states are joined. Keys
// come from memory as operands and become fp16 in registers (the layouts of attn_decode8.hip), 16 rows a product.
template <int D>
struct Few {
  float acc[NWAVE][TILE_FEW][D];
  float m[NWAVE][TILE_FEW], l[NWAVE][TILE_FEW], x[NWAVE][TILE_FEW];
};

template <int D, bool I8, bool MOD>
__device__ __forceinline__ void few_rows(const AttendP& p, const AttendUnit& u, int h, Few<D>& L) {
  static_assert(TILE_FEW == 16, "rows of a product");
  constexpr int KC = Lay8<D>::KC, KS = Lay8<D>::KS, VN = Lay8<D>::VN, VD = Lay8<D>::VD;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / WAVE), lane = tid % WAVE;
  const int j4 = lane >> 4, c16 = lane & 15;
  const int nw = u.n > wave ? (u.n - wave + NWAVE - 1) / NWAVE : 0;
  PageList list(p, u, h, wave, nw);
  const uint32_t koff = c16 * p.k_st + 16 * j4;
  const uint32_t voff = D == 128 ? 4 * j4 * p.v_st + 8 * c16 : (4 * j4 + (c16 >> 3)) * p.v_st + 8 * (c16 & 7);
  const bool up_half = (lane & 8) != 0;
  const uint8_t* kb = p.k + h * p.k_sh;
  const uint8_t* vb = p.v + h * p.v_sh;
  auto res = [&](const uint8_t* base, int64_t sb, uint32_t st, int blk, int pg) {
    return page_res<D>(base, sb, st, pg, pg >= 0 ? min(BLK, u.len - blk * BLK) : 0);
  };
  u32x4 kr[4][KC];
  u32x2 vr[VN];
  int blk = list.blk(0), pg = nw > 0 ? list.pg(0) : -1;
  load_k8<D>(kr, res(kb, p.k_sb, p.k_st, blk, pg), koff, p.k_st);
  load_v8<D>(vr, res(vb, p.v_sb, p.v_st, blk, pg), voff, p.v_st);

  const Row r = virtual_row(p, u, h, c16);
  u32x4 qh[KS];
  float qf;
  {
    const uint16_t* qp = p.q + r.n * p.q_sn + r.hq * p.q_sh + 16 * j4;
    float amax = 0.f, bad = 0.f, up;
#pragma unroll
    for (int x = 0; x < KS; ++x) qh[x] = ld16(qp + 64 * (x / 2) + 8 * (x % 2));
#pragma unroll
    for (int x = 0; x < KS; ++x) q_extent(qh[x], amax, bad);
    qf = q_factor(swap_max(amax), swap_sum(bad), up) * (MOD ? p.scale : p.scale * LOG2E);
#pragma unroll
    for (int x = 0; x < KS; ++x) qh[x] = q_half(qh[x], up);
  }
  const Sight see = sight(p, u, r);
  const Reach re = reach(see);
  const int at = r.pos - u.base - 4 * j4;  // the row's own index, less the lane's first token
  const float slope = MOD && p.slopes != nullptr ? p.slopes[r.hq] : 0.f;
  State st(false);
  Common com;
  bool nan = false;  // a cut page held one
  f32x4_t acc[VD];
#pragma unroll
  for (int j = 0; j < VD; ++j) acc[j] = f32x4_t{0.f, 0.f, 0.f, 0.f};

  for (int k = 0; k < nw; ++k) {
    list.advance(k);
    const float ks = list.ks(k), vs = list.vs(k);
    list.turn(k);
    int blk_n = -1, pg_n = -1;
    if (k + 1 < nw) blk_n = list.blk(k + 1), pg_n = list.pg(k + 1);
    float s[16];
#pragma unroll
    for (int nt = 0; nt < 4; ++nt) {
      f32x4_t c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int x = 0; x < KS; ++x) {
        const u32x2 w0 = widen4<I8>(kr[nt][x / 2][2 * (x % 2)]), w1 = widen4<I8>(kr[nt][x / 2][2 * (x % 2) + 1]);
        c = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, u32x4{w0.x, w0.y, w1.x, w1.y}),
                                                   __builtin_bit_cast(f16x8_t, qh[x]), c, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) s[4 * nt + i] = c[i];
    }
    __builtin_amdgcn_sched_barrier(0);
    load_k8<D>(kr, res(kb, p.k_sb, p.k_st, blk_n, pg_n), koff, p.k_st);
    __builtin_amdgcn_sched_barrier(0);

    const int t0 = blk * BLK;
    const bool whole = sees_all(re, t0, u.len);
    if constexpr (!I8)
      if (!sees_keys(re, t0, u.len)) {
        uint32_t any = 0;
#pragma unroll
        for (int i = 0; i < VN; ++i) vr[i] = u32x2{without_nan(vr[i].x, any), without_nan(vr[i].y, any)};
        nan |= __ballot(any != 0) != 0;
      }
    float f = qf * ks;
    bool neg = (__float_as_int(ks) ^ __float_as_int(p.scale)) < 0;  // uniform
    if constexpr (MOD) {
      modify(s, f, p.softcap, p.slopes != nullptr, slope, static_cast<float>(at - t0),
             [](int i) { return static_cast<float>(16 * (i / 4) + i % 4); });
      f = 1.f, neg = false;
    }
    if (!whole || pg < 0) {  // uniform
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int t = t0 + mf_tok(i / 4, i % 4, j4);
        s[i] = (sees(see, t) & (pg >= 0)) ? s[i] * f : NEG_INF;
      }
      f = 1.f, neg = false;
    }
    uint32_t w[8], wl[8];
    float alpha;
    if (soften<false>(s, f, neg, Weight(vs, com), st, com, alpha, w, wl, [](float x) { return swap_max(x); }))
#pragma unroll
      for (int j = 0; j < VD; ++j) acc[j] *= alpha;
#pragma unroll
    for (int d = 0; d < VD / 4; ++d)
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        u32x4 x[4];  // four dims, tokens in pairs
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          uint32_t a, c;
          v_pair8<D>(vr, 2 * q + y / 2, 2 * (y % 2), d, up_half, a, c);
          const u32x2 w01 = widen4<I8>(__builtin_amdgcn_perm(c, a, 0x05010400u));
          const u32x2 w23 = widen4<I8>(__builtin_amdgcn_perm(c, a, 0x07030602u));
          x[0][y] = w01.x, x[1][y] = w01.y, x[2][y] = w23.x, x[3][y] = w23.y;
        }
        const u32x4 pw = {w[4 * q], w[4 * q + 1], w[4 * q + 2], w[4 * q + 3]};
        const u32x4 pl = {wl[4 * q], wl[4 * q + 1], wl[4 * q + 2], wl[4 * q + 3]};
#pragma unroll
        for (int y = 0; y < 4; ++y)
          acc[4 * d + y] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, x[y]), __builtin_bit_cast(f16x8_t, pw),
                                                                  acc[4 * d + y], 0, 0, 0);
#pragma unroll
        for (int y = 0; y < 4; ++y)
          acc[4 * d + y] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, x[y]), __builtin_bit_cast(f16x8_t, pl),
                                                                  acc[4 * d + y], 0, 0, 0);
      }
    __builtin_amdgcn_sched_barrier(0);
    load_v8<D>(vr, res(vb, p.v_sb, p.v_st, blk_n, pg_n), voff, p.v_st);
    blk = blk_n;
    pg = pg_n;
  }

  // ---- the four states joined: lane (c16, j4) holds row c16's dims mf_vdim(4 j4 + i) + j
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float* o = L.acc[wave][c16] + mf_vdim<D>(4 * j4 + i);
#pragma unroll
    for (int j = 0; j < VD; j += 4)
      *reinterpret_cast<float4*>(o + j) = make_float4(acc[j][i], acc[j + 1][i], acc[j + 2][i], acc[j + 3][i]);
  }
  const float sum = swap_sum(st.l);
  if (j4 == 0) {
    const float mu = st.m == NEG_INF ? 0.f : st.m;
    L.m[wave][c16] = st.m, L.l[wave][c16] = sum;
    L.x[wave][c16] = st.ar == NEG_INF ? NEG_INF : (st.ar - mu) + (st.ax - LIFT);
  }
  if (!I8 && nan)  // NaN of cut pages
    for (int k = 0; k < nw; ++k) {
      const int i0 = u.i0 + wave + NWAVE * k, b = i0 < u.a1 ? i0 : i0 - u.a1 + u.b0, g = list.table[b];
      if (g < 0 || g >= p.num_pages || sees_keys(re, b * BLK, u.len)) continue;
      for (int t = b * BLK; t < min(b * BLK + BLK, u.len); ++t) {
        if (!sees(see, t)) continue;
        for (int d = 4 * j4; d < D; d += 16) {
          const uint32_t z = nan_bytes(*reinterpret_cast<const uint32_t*>(vb + g * p.v_sb + (t - b * BLK) * p.v_st + d));
          for (int e = 0; e < 4; ++e)
            if ((z >> (8 * e + 7) & 1) != 0) L.acc[wave][c16][d + e] = __builtin_nanf("");
        }
      }
    }
  __syncthreads();
  for (int o = tid; o < u.nv * (D / 4); o += NT) {
    const int row = o / (D / 4), d = o % (D / 4) * 4;
    float m[NWAVE], M = NEG_INF, l = 0.f;
#pragma unroll
    for (int w = 0; w < NWAVE; ++w) m[w] = L.m[w][row], M = fmaxf(M, m[w]);
    const float mu = M == NEG_INF ? 0.f : M;
    f32x4_t a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < NWAVE; ++w) {
      const float mw = m[w] == NEG_INF ? 0.f : m[w];
      const Pow2 x((mw - mu) + L.x[w][row]);
      l += L.l[w][row] * fexp2(m[w] - mu);
      a += *reinterpret_cast<const f32x4_t*>(&L.acc[w][row][d]) * x.a * x.b;
    }
    store4(p, u, h, row, virtual_row(p, u, h, row), d, D, a, M, l);
  }
}

// ---- Many rows: the four wavefronts hold 32 rows each and read the same pages, fp16 in LDS, two at a time: while one is
// multiplied the next one's codes are on their way and converted, once for all rows. 32 x 32 products: K as it lies in
// LDS, V by transposing reads. Chunks of 16 bytes are placed so that neither reads nor writes conflict: K chunk c of
// row r at c ^ r, V's at c ^ 5 (r % 4) (64 dims: r / 2 in both).
//   Products and vector instructions bound it together: products take the matrix unit 1536 clocks a page of 128 dims and wavefront,
// beside them vector instructions run at half their rate or so, and two wavefronts a SIMD take turns at best (prompts of 8192:
// 2293 us, the matrix units busy for half of the clocks). So: operands asked for four products ahead (read and waited for one by one,
// prompts took 1850 us with one part a weight, for 1780), addresses that a page's turn does not change (two pages a turn,
// 1745 to 1737), maxima only where they are needed (1650), and nothing in the loop that waits for the codes asked for last (the
// page list in groups).
template <int D>
struct Many {
  uint8_t k[2][BLK * D * 2], v[2][BLK * D * 2];
  Reach reach[NWAVE];
  int nan;  // a cut page held one
};

template <int D, bool I8, bool MOD>
__device__ __forceinline__ void many_rows(const AttendP& p, const AttendUnit& u, int h, Many<D>& L) {
  constexpr int KS = D / 16, ND = D / 32, NC = D / 64;  // steps of a score product; dim tiles; 16-byte loads a thread
  constexpr int AHEAD = 4;  // operands are read that many products before theirs
  constexpr uint32_t ROW = 2 * D;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / WAVE), lane = tid % WAVE;
  const int c32 = lane & 31, half = lane >> 5;
  const int n = u.n;
  const uint8_t* kb = p.k + h * p.k_sh;
  const uint8_t* vb = p.v + h * p.v_sh;
  const int* table = (u.kind & 2) ? p.shared_table + u.table * p.st_stride : p.block_table + u.table * p.bt_stride;
  // the pages of 64 steps from g0 on, one a lane, of which the loop takes GROUP before it asks again: it looks up to two ahead
  constexpr int GROUP = 60;
  int g0 = 0, what;            // table entry (-1: no page)
  uint32_t k_lo, v_lo, kv_hi;  // addresses, 48 bits each
  float k_sc, v_sc;
  auto gather = [&](int first) {
    g0 = first;
    const int j = first + lane, i = u.i0 + j, b = i < u.a1 ? i : i - u.a1 + u.b0;
    int pg = j < n ? table[b] : -1;
    if (pg >= p.num_pages) pg = -1;
    what = pg >= 0 ? b : -1;
    const int at = max(pg, 0);
    const uint64_t ka = reinterpret_cast<uint64_t>(kb) + at * p.k_sb, va = reinterpret_cast<uint64_t>(vb) + at * p.v_sb;
    k_lo = static_cast<uint32_t>(ka), v_lo = static_cast<uint32_t>(va);
    kv_hi = (static_cast<uint32_t>(ka >> 32) & 0xffffu) | static_cast<uint32_t>(va >> 32) << 16;
    k_sc = pg >= 0 ? p.k_scale[pg * p.ks_sb + h * p.ks_sh] : 0.f;
    v_sc = pg >= 0 ? p.v_scale[pg * p.vs_sb + h * p.vs_sh] : 0.f;
    // (waited for here: first used in the loop, they would be waited for there at each turn, with the codes asked for last)
    asm volatile("" : "+v"(k_sc), "+v"(v_sc));
  };
  auto entry = [&](int k) { return static_cast<int>(lane_u32(static_cast<uint32_t>(what), k - g0)); };
  auto of_step = [&](uint32_t lo, int shift, uint32_t st, int k) {  // rows past the sequence's last read zeros
    const uint64_t at = static_cast<uint64_t>(lane_u32(kv_hi, k - g0) >> shift & 0xffffu) << 32 | lane_u32(lo, k - g0);
    const int b = entry(k);
    return make_rsrc(reinterpret_cast<const void*>(at), b >= 0 ? (min(BLK, u.len - b * BLK) - 1) * st + D : 0u);
  };
  // staging: thread t holds 16 NC codes of row t / 4
  const uint32_t srow = tid >> 2, sc = 2 * NC * (tid & 3);  // its first 16-byte chunk in LDS
  const uint32_t kso = srow * p.k_st + 16 * NC * (tid & 3), vso = srow * p.v_st + 16 * NC * (tid & 3);
  const uint32_t kx = D == 128 ? srow & 15 : (srow >> 1) & 7, vx = 5 * (D == 128 ? srow & 3 : (srow >> 1) & 1);
  u32x4 kc[NC], vc[NC];
  auto fetch = [&](int k) {
    const rsrc_t rk = of_step(k_lo, 0, p.k_st, k), rv = of_step(v_lo, 16, p.v_st, k);
#pragma unroll
    for (int c = 0; c < NC; ++c) kc[c] = bload16(rk, kso + 16 * c, 0);
#pragma unroll
    for (int c = 0; c < NC; ++c) vc[c] = bload16(rv, vso + 16 * c, 0);
  };
  auto widen16 = [&](const u32x4& x, uint8_t* row, uint32_t chunk, uint32_t swz) {
    const u32x2 a = widen4<I8>(x[0]), b = widen4<I8>(x[1]), c = widen4<I8>(x[2]), d = widen4<I8>(x[3]);
    *reinterpret_cast<u32x4*>(row + ((chunk ^ swz) << 4)) = u32x4{a.x, a.y, b.x, b.y};
    *reinterpret_cast<u32x4*>(row + (((chunk + 1) ^ swz) << 4)) = u32x4{c.x, c.y, d.x, d.y};
  };
  auto stage = [&](auto buf, bool cut) {
    uint8_t* k = L.k[buf] + srow * ROW;
    uint8_t* v = L.v[buf] + srow * ROW;
    if constexpr (!I8)
      if (cut) {  // uniform
        uint32_t any = 0;
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e) vc[c][e] = without_nan(vc[c][e], any);
        if (any != 0) L.nan = 1;
      }
#pragma unroll
    for (int c = 0; c < NC; ++c) widen16(kc[c], k, sc + 2 * c, kx);
#pragma unroll
    for (int c = 0; c < NC; ++c) widen16(vc[c], v, sc + 2 * c, vx);
  };
  gather(0);
  fetch(0);

  // ---- this wavefront's rows
  const bool busy = 32 * wave < u.nv;
  const Row r = virtual_row(p, u, h, 32 * wave + c32);
  u32x4 qh[KS];
  float qf;
  {
    const uint16_t* qp = p.q + r.n * p.q_sn + r.hq * p.q_sh + 8 * half;
    float amax = 0.f, bad = 0.f, up;
#pragma unroll
    for (int x = 0; x < KS; ++x) qh[x] = ld16(qp + 16 * x);
#pragma unroll
    for (int x = 0; x < KS; ++x) q_extent(qh[x], amax, bad);
    qf = q_factor(swap32_max(amax), swap32_sum(bad), up) * (MOD ? p.scale : p.scale * LOG2E);
#pragma unroll
    for (int x = 0; x < KS; ++x) qh[x] = q_half(qh[x], up);
  }
  const Sight see = sight(p, u, r);
  const Reach re = reach(see);
  const int at = r.pos - u.base - 4 * half;
  const float slope = MOD && p.slopes != nullptr ? p.slopes[r.hq] : 0.f;
  State st(!MOD);
  Common com;
  f32x16_t acc[ND];
#pragma unroll
  for (int j = 0; j < ND; ++j)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[j][i] = 0.f;
  // operand addresses: K chunk 2 x + half of row c32 (step x: ^ 32 x), V dims 32 j + .. of a group's rows (tile j: ^ 64 j)
  const uint32_t ka = c32 * ROW + ((half ^ (D == 128 ? c32 & 15 : (c32 >> 1) & 7)) << 4);
  const uint32_t vrow = 4 * half + ((lane & 15) >> 2), vch = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
  const uint32_t va = vrow * ROW + ((vch ^ 5 * (D == 128 ? vrow & 3 : (vrow >> 1) & 1)) << 4) + 8 * (lane & 1);

  Reach all = re;
  if constexpr (!I8) {  // of the whole tile
    if (lane == 0) L.reach[wave] = re;
    if (tid == 0) L.nan = 0;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NWAVE; ++w) all = both(all, L.reach[w]);
    for (int* x : {&all.from_min, &all.from_max, &all.end_min, &all.end_max, &all.pre_min, &all.pre_max})
      *x = __builtin_amdgcn_readfirstlane(*x);
  }
  auto is_cut = [&](int k) {
    const int b = entry(k);
    return b >= 0 && !sees_keys(all, b * BLK, u.len);
  };
  stage(std::integral_constant<int, 0>{}, !I8 && is_cut(0));
  fetch(1);
  __syncthreads();
  auto step = [&](int k, auto buf) {
    const float ks = lane_value(k_sc, k - g0), vs = lane_value(v_sc, k - g0);
    const int blk = entry(k), t0 = blk * BLK;
    if (busy && blk >= 0 && !sees_none(re, t0)) {
      const uint8_t* kl = L.k[buf];
      const uint8_t* vl = L.v[buf];
      float s[32];
      u32x4 a[2 * KS];  // operands, read a few products ahead
      auto read_k = [&](int x) {
        if (x < 2 * KS) a[x] = *reinterpret_cast<const u32x4*>(kl + ((ka ^ (32 * (x % KS))) + 32 * (x / KS) * ROW));
      };
#pragma unroll
      for (int x = 0; x < AHEAD; ++x) read_k(x);
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        f32x16_t c;
#pragma unroll
        for (int i = 0; i < 16; ++i) c[i] = 0.f;
#pragma unroll
        for (int x = 0; x < KS; ++x) {
          read_k(kt * KS + x + AHEAD);
          __builtin_amdgcn_sched_barrier(0);
          c = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a[kt * KS + x]),
                                                     __builtin_bit_cast(f16x8_t, qh[x]), c, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) s[16 * kt + i] = c[i];
      }
      u32x4 b[4 * ND];
      auto read_v = [&](int y) {
        if (y < 4 * ND) {
          typedef __attribute__((address_space(3))) fp16x4_t lds_t;
          const uint8_t* x = vl + ((va ^ (64 * (y % ND))) + 16 * (y / ND) * ROW);
          const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds_t*)(x)));
          const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds_t*)(x + 8 * ROW)));
          b[y] = u32x4{lo.x, lo.y, hi.x, hi.y};
        }
      };
      float f = qf * ks;
      bool neg = (__float_as_int(ks) ^ __float_as_int(p.scale)) < 0;  // uniform
      if constexpr (MOD) {
        modify(s, f, p.softcap, p.slopes != nullptr, slope, static_cast<float>(at - t0),
               [](int i) { return static_cast<float>(32 * (i / 16) + 8 * (i % 16 / 4) + i % 4); });
        f = 1.f, neg = false;
      }
      if (!sees_all(re, t0, u.len)) {
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const int t = t0 + 32 * (i / 16) + 8 * (i % 16 / 4) + 4 * half + i % 4;
          s[i] = sees(see, t) ? s[i] * f : NEG_INF;
        }
        f = 1.f, neg = false;
      }
      uint32_t w[16], wl[16];
      float alpha;
      if (soften<!MOD>(s, f, neg, Weight(vs, com), st, com, alpha, w, wl, [](float x) { return swap32_max(x); }))
#pragma unroll
        for (int j = 0; j < ND; ++j) acc[j] *= alpha;
#pragma unroll
      for (int y = 0; y < AHEAD; ++y) read_v(y);
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const u32x4 pw = {w[4 * g], w[4 * g + 1], w[4 * g + 2], w[4 * g + 3]};
        const u32x4 pl = {wl[4 * g], wl[4 * g + 1], wl[4 * g + 2], wl[4 * g + 3]};
#pragma unroll
        for (int j = 0; j < ND; ++j) {
          read_v(g * ND + j + AHEAD);
          __builtin_amdgcn_sched_barrier(0);
          acc[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, b[g * ND + j]),
                                                          __builtin_bit_cast(f16x8_t, pw), acc[j], 0, 0, 0);
          acc[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, b[g * ND + j]),
                                                          __builtin_bit_cast(f16x8_t, pl), acc[j], 0, 0, 0);
        }
      }
    }
    if (k + 1 < n) {
      stage(std::integral_constant<int, buf ^ 1>{}, !I8 && is_cut(k + 1));
      fetch(k + 2);
    }
    __syncthreads();
  };
  for (int first = 0; first < n; first += GROUP) {
    if (first > 0) gather(first);
    const int end = min(first + GROUP, n);
    for (int k = first; k < end; k += 2) {
      step(k, std::integral_constant<int, 0>{});
      if (k + 1 < end) step(k + 1, std::integral_constant<int, 1>{});
    }
  }

  // ---- results: lane holds row c32's dims 32 j + 8 (i / 4) + 4 half + i % 4
  const int i0 = 32 * wave + c32;
  const float l = swap32_sum(st.l);
  if (i0 >= u.nv) return;
  const float mu = st.m == NEG_INF ? 0.f : st.m;
  const Pow2 x(st.ar == NEG_INF ? NEG_INF : (st.ar - mu) + (st.ax - LIFT));
#pragma unroll
  for (int j = 0; j < ND; ++j)
#pragma unroll
    for (int i = 0; i < 16; i += 4)
      store4(p, u, h, i0, r, 32 * j + 2 * i + 4 * half, D,
             f32x4_t{acc[j][i], acc[j][i + 1], acc[j][i + 2], acc[j][i + 3]} * x.a * x.b, st.m, l);
  if (I8 || L.nan == 0) return;
  // NaN of cut pages over what was stored
  for (int k = 0; k < n; ++k) {
    const int i = u.i0 + k, b = i < u.a1 ? i : i - u.a1 + u.b0, g = table[b];
    if (g < 0 || g >= p.num_pages || sees_keys(all, b * BLK, u.len)) continue;
    for (int t = b * BLK; t < min(b * BLK + BLK, u.len); ++t) {
      if (!sees(see, t)) continue;
      const uint8_t* row = vb + g * p.v_sb + (t - b * BLK) * p.v_st;
      for (int d = 4 * half; d < D; d += 8) store_nan(p, u, h, i0, r, d, D, nan_bytes(*reinterpret_cast<const uint32_t*>(row + d)));
    }
  }
}

// Workgroups a CU: two for 128 dims (with three they spill 40 registers, 24 tokens behind a window of 4096 63.7 us for 47.2), three for
// 64 (two, with one part a weight: prompts of 2111 behind a prefix 174 us for 154; with two parts large tiles spill 6 registers).
template <int D, bool I8, bool MOD, bool LARGE>
__global__ void __launch_bounds__(NT, D == 128 ? 2 : 3) attend_kernel(const AttendP p) {
  __shared__ __attribute__((aligned(16))) uint8_t raw[sizeof(Few<D>) > (LARGE ? sizeof(Many<D>) : 0) ? sizeof(Few<D>) : sizeof(Many<D>)];
  const int i = blockIdx.x / p.Hkv, h = blockIdx.x % p.Hkv;
  const AttendUnit u = p.units[i];  // (the grid is as long as the array: not waited for twice)
  if (i >= p.head[H_UNITS]) return;
  if constexpr (LARGE) {
    if (u.kind & 1) {
      many_rows<D, I8, MOD>(p, u, h, *reinterpret_cast<Many<D>*>(raw));
      return;
    }
  }
  few_rows<D, I8, MOD>(p, u, h, *reinterpret_cast<Few<D>*>(raw));
}

// The join: a workgroup takes runs of up to 8 virtual rows of a joined tile and KV head, a thread four dims of a row and a class
// of its partial results; their first accumulators are asked for before the weights are found. Rows that no request brings are
// cleared by the workgroups in turn.
template <int D>
__global__ void __launch_bounds__(NT) join_kernel(const AttendP p) {
  constexpr int RW = JOIN_ROWS, MOST = 2 * MAX_TILE_UNITS, TR = D / 4, U = 4;
  __shared__ float sW[RW][MOST];
  __shared__ float sM[RW], sL[RW];
  __shared__ __attribute__((aligned(16))) f32x4_t sA[NT];
  const int tid = threadIdx.x, wave = tid / WAVE, lane = tid % WAVE;
  const int first = p.head[H_FIRST], last = p.head[H_LAST], n_out = p.n_rows - (last - first);
  for (int i = blockIdx.x; i < n_out; i += gridDim.x) {
    const int64_t n = i < first ? i : i - first + last;
    for (int x = tid; x < p.Hq * (D / 8); x += NT) *reinterpret_cast<u32x4*>(p.out + n * p.Hq * D + 8 * x) = u32x4{0, 0, 0, 0};
    for (int x = tid; x < p.Hq; x += NT) p.lse[n * p.Hq + x] = NEG_INF;
  }
  const int total = p.head[H_JOINS] * p.Hkv;
  for (int w = blockIdx.x; w < total; w += gridDim.x) {
    const int h = w % p.Hkv;
    const AttendJoin o = p.joins[w / p.Hkv];
    // partial result s of row i: own pages' first, then the prefix's
    const int np = o.ns + o.more_ns;
    auto at = [&](int i, int s) {
      const int r = s < o.ns ? o.part + i + s * o.step : o.more + i + (s - o.ns) * o.more_step;
      return static_cast<int64_t>(r) * p.Hkv + h;
    };
    const int R = o.n > 4 ? 8 : o.n > 2 ? 4 : o.n;      // rows side by side, NC classes of partials
    const int NC = NT / TR / R, i = tid / TR % R, cls = tid / TR / R, d = tid % TR * 4;
    const bool row = i < o.n;
    auto load = [&](int s) {
      return row && s < np ? *reinterpret_cast<const f32x4_t*>(p.part_acc + at(i, s) * D + d) : f32x4_t{0.f, 0.f, 0.f, 0.f};
    };
    f32x4_t x[U];
#pragma unroll
    for (int e = 0; e < U; ++e) x[e] = load(cls + NC * e);
#pragma unroll
    for (int g = 0; g < RW / NWAVE; ++g) {
      const int j = wave + NWAVE * g;
      if (j < o.n) {  // uniform
        float m[MOST / WAVE], l[MOST / WAVE], M = NEG_INF, L = 0.f;
#pragma unroll
        for (int e = 0; e < MOST / WAVE; ++e) {
          const int s = lane + WAVE * e;
          m[e] = NEG_INF, l[e] = 0.f;
          if (s < np) {
            const float2 t = *reinterpret_cast<const float2*>(p.part_ml + at(j, s) * 2);
            m[e] = t.x, l[e] = t.y;
          }
          M = fmaxf(M, m[e]);
        }
        M = wave_max(M);
        const float mu = M == NEG_INF ? 0.f : M;
#pragma unroll
        for (int e = 0; e < MOST / WAVE; ++e) {
          const int s = lane + WAVE * e;
          const float v = l[e] == 0.f ? 0.f : fexp2(m[e] - mu);
          L += l[e] * v;
          if (s < np) sW[j][s] = l[e] == 0.f ? -1.f : v;  // (an empty partial counts for nothing, a NaN counts)
        }
        L = wave_sum(L);
        if (lane == 0) sM[j] = M, sL[j] = L;
      }
    }
    __syncthreads();
    f32x4_t a = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = cls; s0 < np; s0 += NC * U) {
      f32x4_t y[U];  // the next round's, asked for before this one's are added
#pragma unroll
      for (int e = 0; e < U; ++e) y[e] = load(s0 + NC * (U + e));
#pragma unroll
      for (int e = 0; e < U; ++e) {
        const float v = row && s0 + NC * e < np ? sW[i][s0 + NC * e] : -1.f;
        if (v != -1.f) a += x[e] * v;
      }
#pragma unroll
      for (int e = 0; e < U; ++e) x[e] = y[e];
    }
    sA[tid] = a;
    __syncthreads();
    if (cls == 0 && row) {
      for (int c = 1; c < NC; ++c) a += sA[tid + c * R * TR];
      const int v = o.v0 + i, r = v / p.G;
      AttendUnit u{};
      u.part = -1;
      store4(p, u, h, 0, Row{o.row0 + r, h * p.G + (v - r * p.G), 0, 0}, d, D, a, sM[i], sL[i]);
    }
    __syncthreads();
  }
}

template <int D, bool I8>
hipError_t launch_d(const AttendP& p, const AttendSizes& z, hipStream_t s) {
  const dim3 grid(static_cast<uint32_t>(z.units * p.Hkv)), nt(NT);
  const bool mod = p.softcap > 0.f || p.slopes != nullptr;
  if (z.large) {
    if (mod)
      hipLaunchKernelGGL((attend_kernel<D, I8, true, true>), grid, nt, 0, s, p);
    else
      hipLaunchKernelGGL((attend_kernel<D, I8, false, true>), grid, nt, 0, s, p);
  } else {
    if (mod)
      hipLaunchKernelGGL((attend_kernel<D, I8, true, false>), grid, nt, 0, s, p);
    else
      hipLaunchKernelGGL((attend_kernel<D, I8, false, false>), grid, nt, 0, s, p);
  }
  return hipGetLastError();
}

}  // namespace

hipError_t launch_attend(const kvskip_attend_args& a, const AttendSizes& z, hipStream_t s) {
  AttendP p;
  p.q = static_cast<const uint16_t*>(a.q), p.q_sn = a.q_sn, p.q_sh = a.q_sh;
  p.k = static_cast<const uint8_t*>(a.k), p.k_sb = a.k_sb, p.k_sh = a.k_sh, p.k_st = static_cast<uint32_t>(a.k_st);
  p.v = static_cast<const uint8_t*>(a.v), p.v_sb = a.v_sb, p.v_sh = a.v_sh, p.v_st = static_cast<uint32_t>(a.v_st);
  p.k_scale = a.k_scale, p.ks_sb = a.ks_sb, p.ks_sh = a.ks_sh;
  p.v_scale = a.v_scale, p.vs_sb = a.vs_sb, p.vs_sh = a.vs_sh;
  p.block_table = a.block_table, p.bt_stride = a.bt_stride;
  p.shared_table = a.shared_table, p.st_stride = a.st_stride;
  p.slopes = a.slopes;
  p.out = static_cast<uint16_t*>(a.out), p.lse = a.lse, p.part_acc = a.part_acc, p.part_ml = a.part_ml;
  const int* work = a.plan.work;
  p.head = work;
  p.units = reinterpret_cast<const AttendUnit*>(work + z.at_units);
  p.joins = reinterpret_cast<const AttendJoin*>(work + z.at_joins);
  p.rows = reinterpret_cast<const AttendRow*>(work + z.at_rows);
  p.n_rows = a.plan.rows, p.Hq = a.plan.Hq, p.Hkv = a.plan.Hkv, p.G = a.plan.Hq / a.plan.Hkv;
  p.num_pages = a.num_pages, p.window = a.plan.window < (1 << 30) ? a.plan.window : 1 << 30;
  p.scale = a.scale;
  // (scores over the cap stay in fp32's range: below 2^-64 capped scores are all alike, and those that feel one above 2^96
  // leave one key any weight)
  p.softcap = a.softcap > 0.f ? fminf(fmaxf(a.softcap, 0x1p-64f), 0x1p96f) : 0.f;
  const bool i8 = a.format == KVSKIP_INT8;
  const hipError_t e = a.D == 128 ? (i8 ? launch_d<128, true>(p, z, s) : launch_d<128, false>(p, z, s))
                                  : (i8 ? launch_d<64, true>(p, z, s) : launch_d<64, false>(p, z, s));
  if (e != hipSuccess) return e;
  const int64_t joins = z.joins * p.Hkv;
  const dim3 grid(static_cast<uint32_t>(joins < JOIN_GRID ? joins : JOIN_GRID));
  if (a.D == 128)
    hipLaunchKernelGGL(join_kernel<128>, grid, dim3(NT), 0, s, p);
  else
    hipLaunchKernelGGL(join_kernel<64>, grid, dim3(NT), 0, s, p);
  return hipGetLastError();
}

}  // namespace kvs
