// Pages of a serving loop's cache: a step's block tables and slot map from the requests' lengths (page_map), and its
// new keys and values into the pages that the slot map names (cache_write).
//
// page_map. Request b holds h_b pages and has n_b tokens after the step, a_b of them new; need_b = ceil(n_b / 64).
// Pages past need_b go back on the free stack first (request by request); then take_b = max(need_b - h_b, 0) come off
// it, the k-th page taken by the step from position avail - 1 - k. Everything but two prefix sums (pages given, pages
// taken, and new tokens) is independent per request, row or page: one workgroup makes the sums, and the rows' slots and
// the tables' new entries follow from them with a binary search in LDS. The result has no atomics and depends on
// nothing but the inputs. It is bound by latency: lengths, then pages, then the stores, one after another.
//
// cache_write. The rows of one page lie next to each other in the slot map (a run). A workgroup takes a run of one KV
// head's keys or values: its rows are loaded once, into registers, the largest magnitude goes through LDS, and the codes
// are stored 8 bytes a lane in the page's order (a head's page is one contiguous piece). Bound by HBM: 2 bytes read and 1
// written an element. A scale is a power of two (or what a caller brought, as long as it suffices: its quotients are
// rounded once too): dividing by it is exact, so a code depends on its value and scale alone, and when a later row needs a larger scale, the rows that are there move to it without rounding again (e4m3:
// but for subnormal codes; int8 rounds once more per doubling, less than the final step in sum).
#include <type_traits>

#include "common.hpp"
#include "internal.hpp"

namespace kvs {
namespace {

// ------------------------------------------------------------------ page_map
constexpr int PT = 1024;  // threads of the summing workgroup
constexpr int PF = 256;   // threads of a filling workgroup

// A step's sums, in LDS: first row of each request (starts[B]: all rows), pages given back before it, pages taken
// before it (or -1: not served), pages held before the step.
struct Step {
  int starts[MAX_PAGE_B + 1];
  int given[MAX_PAGE_B];
  int taken[MAX_PAGE_B];
  int held[MAX_PAGE_B];
};

__device__ __forceinline__ int pages_of(int n) { return n / BLK + (n % BLK != 0); }

// A request's sizes from its lengths: false if its tokens do not fit a table row.
__device__ __forceinline__ bool page_need(const kvskip_page_args& p, int b, int& n, int& a, int& h, int& need) {
  n = max(p.seq_lens[b], 0);
  a = min(max(p.new_lens[b], 0), n);
  h = min(max(p.held[b], 0), p.width);
  need = pages_of(n);
  return need <= p.width;
}

// The last b with first[b] <= i (of requests with one value the last: the others have nothing there).
__device__ __forceinline__ int request_of(const int* first, int B, int i) {
  int lo = 0, hi = B - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (first[mid] <= i)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

// The k-th page taken by the step: from the stack as it was, or of those given back by this step (position g of them).
__device__ __forceinline__ int taken_page(const kvskip_page_args& p, const Step& s, int count, int avail, int k) {
  const int g = avail - 1 - k - count;
  if (g < 0) return p.free_pages[avail - 1 - k];
  const int b = request_of(s.given, p.B, g);
  return p.block_table[b * p.bt_stride + pages_of(max(p.seq_lens[b], 0)) + g - s.given[b]];
}

// Row i's slot, or -1.
__device__ __forceinline__ int row_slot(const kvskip_page_args& p, const Step& s, int count, int avail, int i) {
  if (i >= s.starts[p.B]) return -1;
  const int b = request_of(s.starts, p.B, i), before = s.taken[b];
  if (before < 0) return -1;
  const int n = max(p.seq_lens[b], 0), a = min(max(p.new_lens[b], 0), n);
  const int pos = n - a + (i - s.starts[b]), j = pos / BLK, h = s.held[b];
  const int pg = j < h ? p.block_table[b * p.bt_stride + j] : taken_page(p, s, count, avail, before + j - h);
  return pg >= 0 && pg < p.num_pages ? pg * BLK + pos % BLK : -1;
}

// The rows' slots and the pages that change hands, once the sums are in LDS: `threads` threads, this one number t; a
// wavefront moves the pages of one request (of 64 at a time it skips those with none to move). Nothing that is written
// is read here (a request's length after the step, where lens_out replaces it, is the same if it is served, and not used
// if it is not): entries given back are read below what a request keeps or in rows that take none, stack positions from
// `count` on are not read.
__device__ __forceinline__ void page_fill(const kvskip_page_args& p, const Step& s, int count, int avail, int t, int threads) {
  for (int i = t; i < p.rows; i += threads) p.slots[i] = row_slot(p, s, count, avail, i);
  const int lane = threadIdx.x % WAVE, w = __builtin_amdgcn_readfirstlane(t / WAVE), nw = threads / WAVE;
  for (int b0 = w; b0 < p.B; b0 += nw * WAVE) {
    const int mine = b0 + nw * lane;
    bool any = false;
    if (mine < p.B) {
      const int need = pages_of(max(p.seq_lens[mine], 0));
      any = s.taken[mine] >= 0 && need != s.held[mine];
    }
    for (uint64_t todo = __ballot(any); todo != 0; todo &= todo - 1) {
      const int b = b0 + nw * __builtin_ctzll(todo), h = s.held[b], need = pages_of(max(p.seq_lens[b], 0));
      int32_t* row = p.block_table + b * p.bt_stride;
      for (int j = h + lane; j < need; j += WAVE) row[j] = taken_page(p, s, count, avail, s.taken[b] + j - h);
      for (int j = need + lane; j < h; j += WAVE) {
        const int at = count + s.given[b] + j - need;
        if (at < p.num_pages) p.free_pages[at] = row[j];
      }
    }
  }
}

// The sums; ONE: also page_fill (the whole operator in one launch: of one workgroup, or of several that all make the sums,
// the first of which writes them). A thread holds two neighbouring requests; the three
// prefix sums (pages given, pages taken, rows) meet in LDS together, once, and what needs the total of pages given back
// (who is served, with how many pages) a second time.
template <bool ONE>
__global__ void __launch_bounds__(PT) page_sums_kernel(const kvskip_page_args p) {
  static_assert(MAX_PAGE_B == 2 * PT, "two requests a thread");
  constexpr int NW = PT / WAVE;
  __shared__ Step s;
  __shared__ int tot[3][NW], tot2[2][NW];
  const int tid = threadIdx.x, lane = tid % WAVE, wave = tid / WAVE;
  const int count = min(max(*p.free_count, 0), p.num_pages);
  int v[2][3], h[2], need[2];  // of request 2 tid + r: pages given, pages taken, rows
  int n[2], was[2];     // tokens after the step; before it
  bool fits[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int b = 2 * tid + r;
    int a = 0;
    h[r] = need[r] = n[r] = was[r] = 0;
    fits[r] = b < p.B && page_need(p, b, n[r], a, h[r], need[r]);
    was[r] = n[r] - a;
    v[r][2] = min(a, p.rows + 1);
    if (p.lens_out != nullptr && b < p.B) {
      const int sum = p.seq_lens[b], add = p.new_lens[b];
      if (sum < 0 && add > 0) {  // past 31 bits: more rows than any map has
        was[r] = static_cast<int>(static_cast<uint32_t>(sum) - static_cast<uint32_t>(add));
        v[r][2] = p.rows + 1;
      }
    }
  }
  int incl[3], all[3];
  auto sums = [&](auto k0, auto k1) {
#pragma unroll
    for (int k = k0; k < k1; ++k) {
      incl[k] = wave_incl_scan(v[0][k] + v[1][k]);
      if (lane == WAVE - 1) tot[k][wave] = incl[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = k0; k < k1; ++k) {
      const int x = wave_incl_scan(lane < NW ? tot[k][lane] : 0);
      all[k] = __builtin_amdgcn_readlane(x, NW - 1);
      incl[k] += (wave > 0 ? __shfl(x, wave - 1, WAVE) : 0) - v[0][k] - v[1][k];  // now exclusive
    }
  };
  auto pages = [&] {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      v[r][0] = fits[r] ? max(h[r] - need[r], 0) : 0;
      v[r][1] = fits[r] ? max(need[r] - h[r], 0) : 0;
    }
  };
  typedef std::integral_constant<int, 0> I0;
  typedef std::integral_constant<int, 2> I2;
  typedef std::integral_constant<int, 3> I3;
  if (p.lens_out == nullptr) {  // uniform
    pages();
    sums(I0{}, I3{});
  } else {  // a request whose rows do not all fit the map moves no pages: rows first
    sums(I2{}, I3{});
    int before = incl[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      before += v[r][2];
      fits[r] = fits[r] && (v[r][2] == 0 || before <= p.rows);
    }
    pages();
    sums(I0{}, I2{});
  }
  const int avail = min(count + all[0], p.num_pages);
  int used = 0, left = 0;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int b = 2 * tid + r;
    const bool served = fits[r] && (v[r][1] == 0 || incl[1] + v[r][1] <= avail);
    if (b < p.B) {
      s.starts[b] = incl[2];
      s.given[b] = incl[0];
      s.taken[b] = served ? incl[1] : -1;
      s.held[b] = h[r];
      if (!ONE || blockIdx.x == 0) {
        p.starts[b] = incl[2];
        p.held_out[b] = served ? need[r] : h[r];
        if (p.lens_out != nullptr) p.lens_out[b] = served ? n[r] : was[r];
      }
      used += served ? v[r][1] : 0;
      left += served ? 0 : 1;
    }
#pragma unroll
    for (int k = 0; k < 3; ++k) incl[k] += v[r][k];
  }
  used = wave_sum_int(used);
  left = wave_sum_int(left);
  if (lane == 0) tot2[0][wave] = used, tot2[1][wave] = left;
  if (tid == 0) {
    s.starts[p.B] = all[2];
    if (!ONE || blockIdx.x == 0) p.starts[p.B] = all[2];
  }
  __syncthreads();
  if ((!ONE || blockIdx.x == 0) && wave == NW - 1) {
    used = wave_sum_int(lane < NW ? tot2[0][lane] : 0);
    left = wave_sum_int(lane < NW ? tot2[1][lane] : 0);
    if (lane == 0) {
      *p.short_out = left;
      *p.free_count_out = avail - used;
    }
  }
  if constexpr (ONE) {
    page_fill(p, s, count, avail, blockIdx.x * PT + tid, gridDim.x * PT);
  } else {  // what the filling launch needs beside starts
    if (tid == 0) p.work[0] = count, p.work[1] = avail;
    for (int b = tid; b < p.B; b += PT) {
      p.work[2 + b] = s.given[b];
      p.work[2 + p.B + b] = s.taken[b];
      p.work[2 + 2 * p.B + b] = s.held[b];
    }
  }
}

__global__ void __launch_bounds__(PF) page_fill_kernel(const kvskip_page_args p) {
  __shared__ Step s;
  const int tid = threadIdx.x;
  const int count = p.work[0], avail = p.work[1];
  for (int b = tid; b < p.B; b += PF) {
    s.starts[b] = p.starts[b];
    s.given[b] = p.work[2 + b];
    s.taken[b] = p.work[2 + p.B + b];
    s.held[b] = p.work[2 + 2 * p.B + b];
  }
  if (tid == 0) s.starts[p.B] = p.starts[p.B];
  __syncthreads();
  page_fill(p, s, count, avail, blockIdx.x * PF + tid, gridDim.x * PF);
}

// ------------------------------------------------------------------ cache_write
enum : int { FMT_E4M3 = 0, FMT_INT8 = 1, FMT_BF16 = 2 };

// The smallest power of two s with amax <= qmax s (amax finite, > 0), at least 2^-126: qmax = (1 + f) 2^k, so s is
// 2^(e - k) for an amax of mantissa up to 1 + f, else twice that.
template <int FMT>
__device__ __forceinline__ float pow2_scale(float amax) {
  constexpr uint32_t FRAC = FMT == FMT_E4M3 ? 0x600000u : 0x7c0000u | 0x020000u;  // 448 = 1.75 2^8, 127 = 1.984375 2^6
  constexpr int K = FMT == FMT_E4M3 ? 8 : 6;
  const uint32_t u = __float_as_uint(amax);
  const int e = static_cast<int>(u >> 23) - K + ((u & 0x7fffffu) > FRAC ? 1 : 0);
  return __uint_as_float(static_cast<uint32_t>(max(e, 1)) << 23);
}

__device__ __forceinline__ u32x2 bload8(rsrc_t r, uint32_t voff, uint32_t soff) {
  return __builtin_amdgcn_raw_buffer_load_b64(r, static_cast<int>(voff), static_cast<int>(soff), 0);
}
__device__ __forceinline__ uint32_t bload4(rsrc_t r, uint32_t voff) {
  return static_cast<uint32_t>(__builtin_amdgcn_raw_buffer_load_b32(r, static_cast<int>(voff), 0, 0));
}
__device__ __forceinline__ void bstore4(uint32_t v, rsrc_t r, uint32_t voff) {
  __builtin_amdgcn_raw_buffer_store_b32(v, r, static_cast<int>(voff), 0, 0);
}
__device__ __forceinline__ void bstore16(u32x4 v, rsrc_t r, uint32_t voff) {
  __builtin_amdgcn_raw_buffer_store_b128(v, r, static_cast<int>(voff), 0, 0);
}

// Two values (already divided by the scale) as codes in the low half; infinities at the largest value of their sign,
// NaN as NaN (e4m3) or 0 (int8).
template <int FMT>
__device__ __forceinline__ uint32_t code1(float x) {
  if constexpr (FMT == FMT_INT8) {
    const float r = __builtin_rintf(x);
    return r != r ? 0u : static_cast<uint32_t>(static_cast<int>(fminf(fmaxf(r, -127.f), 127.f))) & 0xffu;
  }
  return 0u;
}
template <int FMT>
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d) {
  if constexpr (FMT == FMT_E4M3) {
    auto lim = [](float x) { return x != x ? x : fminf(fmaxf(x, -448.f), 448.f); };
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(lim(a), lim(b), 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(lim(c), lim(d), w, true);
    return static_cast<uint32_t>(w);
  } else {
    return code1<FMT>(a) | code1<FMT>(b) << 8 | code1<FMT>(c) << 16 | code1<FMT>(d) << 24;
  }
}

// Four codes as values.
template <int FMT>
__device__ __forceinline__ void values4(uint32_t w, float (&x)[4]) {
  if constexpr (FMT == FMT_E4M3) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), false);
    const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), true);
    x[0] = lo[0], x[1] = lo[1], x[2] = hi[0], x[3] = hi[1];
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = static_cast<float>(static_cast<int8_t>(w >> (8 * i) & 0xffu));
  }
}

// A quotient or product y, rounded to fp32, whose exact value lies off it towards the sign of r: rounded to odd instead, so
// that rounding it once more, to a code, gives the code of the exact value. (Far from every code's border y stays: below
// 2^-20 the code is 0, past 2^10 the largest.)
__device__ __forceinline__ float to_odd(float y, float r) {
  const uint32_t u = __float_as_uint(y);
  const bool off = r != 0.f && (u & 1u) == 0u && fabsf(y) >= 0x1p-20f && fabsf(y) <= 0x1p10f;
  return off ? __uint_as_float((r > 0.f) == (y > 0.f) ? u + 1u : u - 1u) : y;
}

// Powers of two (normal ones): dividing by them is multiplying by their reciprocal.
__device__ __forceinline__ bool is_pow2(float s) {
  const uint32_t u = __float_as_uint(s);
  return (u & 0x7fffffu) == 0u && u != 0u;
}

constexpr int CT = 256;

// Keys or values of one KV head: what a run needs.
struct Side {
  const char* rows;  // row 0 of the head
  char* pool;        // page 0 of the head
  float* scale;
  int64_t sn, psb, ssb;
  uint32_t st, pst;
};

// One run of `len` rows (at most 64) from row rs of the map on, this lane's slot within the page `at`, by T threads: the
// workgroup's (its wavefronts meet once, over `meet`: their maxima and, from the thread that will store the new one, the
// scale that the page holds, so that no wavefront loads it while that thread may have passed the barrier), or one
// wavefront's for a run that one load takes.
template <int FMT, int D, int T>
__device__ __forceinline__ void write_run(const Side& s, int pg, int rs, int len, int at, float* meet) {
  constexpr int LPR = D / 8, RPI = T / LPR;                     // lanes a row, rows a load
  constexpr int NI = T == WAVE ? 1 : BLK / RPI, NO = BLK / RPI;  // loads of a run, of a page
  constexpr int EB = FMT == FMT_BF16 ? 2 : 1;
  constexpr uint32_t OOB = 0xf0000000u;
  const int lane = threadIdx.x % WAVE, t = threadIdx.x % T, c = t % LPR, r0 = t / LPR;
  const int first = __builtin_amdgcn_readfirstlane(at);
  const uint64_t run = len == WAVE ? ~0ull : (1ull << len) - 1;
  uint64_t keep = run, fresh = run << first;  // rows of the run that are kept; rows of the page they fill
  const bool linear = (__ballot(at == first + lane) & run) == run;
  if (!linear) {  // not one after another: of rows with one slot the last
    bool last = lane < len;
    fresh = 0;
    for (int l = 0; l < len; ++l) {
      const int r = __builtin_amdgcn_readlane(at, l);
      fresh |= 1ull << r;
      last = last && !(l > lane && r == at);
    }
    keep = __ballot(last);
  }
  // Rows through buffer resources: the source's are consecutive and end with the run (rows past it read zero); so are the
  // page's, but where a slot comes twice, which costs a shuffle a row.
  const rsrc_t src = make_rsrc(s.rows + rs * s.sn, (len - 1) * s.st + 2 * D);
  const rsrc_t dst = make_rsrc(s.pool + pg * s.psb, 63 * s.pst + EB * D);
  float* scale = FMT == FMT_BF16 ? nullptr : s.scale + pg * s.ssb;
  float held = 0.f;  // asked for before the rows: whoever waits for those has it
  if (FMT != FMT_BF16 && (T == WAVE || t == 0)) held = *scale;
  u32x4 x[NI];
#pragma unroll
  for (int i = 0; i < NI; ++i) x[i] = bload16<BUF_NT>(src, r0 * s.st + 16 * c, RPI * i * s.st);
  auto dst_off = [&](int i) -> uint32_t {
    const int r = RPI * i + r0;
    const int row = linear ? first + r : __shfl(at, r, WAVE);
    return keep >> r & 1 ? row * s.pst + 8 * EB * c : OOB;
  };
  if constexpr (FMT == FMT_BF16) {
#pragma unroll
    for (int i = 0; i < NI; ++i)
      if (RPI * i < len) bstore16(x[i], dst, dst_off(i));
  } else {
    // the largest magnitude of the rows that are kept, of bf16 bits without the sign: an infinity counts as the largest
    // finite value, NaN not
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      uint32_t m = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t lo = x[i][e] & 0x7fffu, hi = x[i][e] >> 16 & 0x7fffu;
        m = max(m, max(lo <= 0x7f80u ? lo : 0u, hi <= 0x7f80u ? hi : 0u));
      }
      if (keep != run) m = keep >> (RPI * i + r0) & 1 ? m : 0u;
      top = max(top, m);
    }
    float amax = wave_max(__uint_as_float(min(top, 0x7f7fu) << 16));
    if constexpr (T > WAVE) {
      if (lane == 0) meet[t / WAVE] = amax;
      if (t == 0) meet[T / WAVE] = held;
      // a barrier for LDS alone: __syncthreads would wait for the stores of the run before too
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
      __builtin_amdgcn_s_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
#pragma unroll
      for (int w = 0; w < T / WAVE; ++w) amax = fmaxf(amax, meet[w]);
      held = meet[T / WAVE];
    }
    const bool anew = fresh & 1;
    const float was = !anew && held > 0.f && held < __builtin_huge_valf() ? held : 0.f;
    constexpr float QMAX = FMT == FMT_E4M3 ? 448.f : 127.f;
    const float now = amax > QMAX * was ? pow2_scale<FMT>(amax) : was;
    const float inv = now > 0.f ? 1.f / now : 0.f;
    if (__builtin_expect(now == 0.f || is_pow2(now), 1)) {  // uniform; the reciprocal is exact
#pragma unroll
      for (int i = 0; i < NI; ++i)
        if (RPI * i < len) {  // uniform
          const u32x4 w = x[i];
          bstore_b64(u32x2{codes4<FMT>(bf_lo(w.x) * inv, bf_hi(w.x) * inv, bf_lo(w.y) * inv, bf_hi(w.y) * inv),
                           codes4<FMT>(bf_lo(w.z) * inv, bf_hi(w.z) * inv, bf_lo(w.w) * inv, bf_hi(w.w) * inv)},
                     dst, dst_off(i), 0);
        }
    } else {
      // a scale that the caller brought: quotients to odd (both sides times 2^80 where the remainder could underflow; the
      // product with the reciprocal, improved once, is within a step of the quotient, which is what to_odd needs). A rare path
      // that is to cost the others no registers: four values at a time, loaded again
      const float lift = now < 0x1p-60f ? 0x1p80f : 1.f, den = now * lift, rec = 1.f / den;
      auto over = [&](uint32_t bits) {
        const float num = __uint_as_float(bits) * lift, q0 = num * rec, q = fmaf(fmaf(-q0, den, num), rec, q0);
        // (infinities, NaN and zeros of either sign as they are)
        return fabsf(q0) >= 0x1p-20f && fabsf(q0) <= 0x1p10f ? to_odd(q, fmaf(-q, den, num)) : q0;
      };
#pragma unroll 1
      for (int i = 0; i < 2 * NI; ++i) {
        const int r = RPI * (i / 2) + r0, half = i % 2;
        const u32x2 w = bload8(src, r * s.st + 16 * c + 8 * half, 0);
        const uint32_t off = dst_off(i / 2) + 4 * half;
        bstore4(codes4<FMT>(over(w.x << 16), over(w.x & 0xffff0000u), over(w.y << 16), over(w.y & 0xffff0000u)), dst, off);
      }
    }
    if (__builtin_expect(now != was && !anew, 0)) {  // uniform: the page's other rows move to the larger scale
      const float f = was * inv;  // exact: a scale that grows is a power of two
      if (__builtin_expect(was != 0.f && !is_pow2(was), 0)) {  // as above
        auto moved = [&](float code) { return to_odd(code * f, fmaf(code, f, -(code * f))); };
#pragma unroll 1
        for (int i = 0; i < 2 * NO; ++i) {
          const int r = RPI * (i / 2) + r0;
          const uint32_t off = fresh >> r & 1 ? OOB : r * s.pst + 8 * c + 4 * (i % 2);
          float a[4];
          values4<FMT>(bload4(dst, off), a);
          bstore4(codes4<FMT>(moved(a[0]), moved(a[1]), moved(a[2]), moved(a[3])), dst, off);
        }
      } else
#pragma unroll 1
      for (int i0 = 0; i0 < NO; i0 += NO < 4 ? NO : 4) {
        u32x2 old[NO < 4 ? NO : 4];
#pragma unroll
        for (int i = 0; i < (NO < 4 ? NO : 4); ++i) {
          const int r = RPI * (i0 + i) + r0;
          old[i] = bload8(dst, fresh >> r & 1 ? OOB : r * s.pst + 8 * c, 0);
        }
#pragma unroll
        for (int i = 0; i < (NO < 4 ? NO : 4); ++i) {
          const int r = RPI * (i0 + i) + r0;
          float a[4], b[4];
          values4<FMT>(old[i].x, a);
          values4<FMT>(old[i].y, b);
          bstore_b64(u32x2{codes4<FMT>(a[0] * f, a[1] * f, a[2] * f, a[3] * f),
                           codes4<FMT>(b[0] * f, b[1] * f, b[2] * f, b[3] * f)},
                     dst, fresh >> r & 1 ? OOB : r * s.pst + 8 * c, 0);
        }
      }
    }
    if (t == 0 && !(now == held)) *scale = now;
  }
}

// Workgroup (KV head's keys or values, window): the runs that start in rows [w0, w0 + win) of the map. Consecutive
// workgroups take the heads, keys then values, of one window: together they read and write whole rows (heads by windows
// instead: 72 us against 63 for 44 000 rows of 8 heads). Workgroups per CU, four (the compiler's choice of registers) /
// eight, us: prompts of 44 000 rows of 64 dims 39 / 33 in int8, 35 / 32 in e4m3, of 512 rows 6.2 / 7.3 and 5.9 / 6.1; of
// 128 dims and very different lengths 51.1 / 53.4, of 512 rows 7.4 / 9.2 and 7.2 / 8.5 (4096 single rows 34.7 / 30.9). Five of
// 128 dims is what 96 registers allow; with 97 to 128, four resident, the prompts take 55.2 for 51.5.
template <int FMT, int D>
__global__ void __launch_bounds__(CT, (D == 64 ? 8 : 5)) cache_write_kernel(const kvskip_write_args p, int win) {
  constexpr int EB = FMT == FMT_BF16 ? 2 : 1, RPW = WAVE / (D / 8);
  __shared__ float sMax[2][CT / WAVE + 1];
  const int lane = threadIdx.x % WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
  const bool isv = static_cast<int>(blockIdx.x) >= p.Hkv;
  const int h = blockIdx.x - (isv ? p.Hkv : 0);
  Side s;
  s.rows = static_cast<const char*>(isv ? p.v : p.k) + h * (isv ? p.v_sh : p.k_sh) * 2;
  s.sn = (isv ? p.v_sn : p.k_sn) * 2;
  s.st = static_cast<uint32_t>(s.sn);
  s.pool = static_cast<char*>(isv ? p.v_pool : p.k_pool) + h * (isv ? p.vp_sh : p.kp_sh) * EB;
  s.psb = (isv ? p.vp_sb : p.kp_sb) * EB;
  s.pst = static_cast<uint32_t>((isv ? p.vp_st : p.kp_st) * EB);
  s.scale = FMT == FMT_BF16 ? nullptr : (isv ? p.v_scale : p.k_scale) + h * (isv ? p.vs_sh : p.ks_sh);
  s.ssb = isv ? p.vs_sb : p.ks_sb;
  // slots of the window's 64 rows, of the 64 after them and of the row before: -1 for none
  const int slots = p.num_pages * BLK;
  const int w0 = blockIdx.y * win;
  auto slot_at = [&](int i) {
    const int x = i >= 0 && i < p.N ? p.slot_map[i] : -1;
    return x < slots ? max(x, -1) : -1;
  };
  const int s0 = slot_at(w0 + lane), s1 = slot_at(w0 + WAVE + lane), before = slot_at(w0 + lane - 1);
  uint64_t leaders = __ballot(lane < win && s0 >= 0 && (before < 0 || s0 / BLK != before / BLK));
  auto run_slots = [&](int l0) {  // of the run that starts at row w0 + l0, 64 rows
    const int in0 = __shfl(s0, (l0 + lane) & 63, WAVE), in1 = __shfl(s1, (l0 + lane) & 63, WAVE);
    return l0 + lane < WAVE ? in0 : in1;
  };
  auto length = [&](int mine, int pg) {
    const uint64_t on = __ballot(mine >= 0 && mine / BLK == pg);
    return on == ~0ull ? WAVE : static_cast<int>(__builtin_ctzll(~on));
  };
  // Runs that one load of a wavefront takes (new tokens of many requests) go to the wavefronts one each; the others to
  // the whole workgroup, in turn (4096 rows of as many pages, each run by the workgroup and with __syncthreads: 120 us,
  // so 34).
  int number = 0, turn = 0;
  for (; leaders != 0; leaders &= leaders - 1) {
    const int l0 = __builtin_ctzll(leaders);
    const int pg = __builtin_amdgcn_readlane(s0, l0) / BLK;
    int rs = w0 + l0, mine = run_slots(l0);
    int len = length(mine, pg);
    if (len <= RPW) {
      if (number++ % (CT / WAVE) == wave) write_run<FMT, D, WAVE>(s, pg, rs, len, mine % BLK, nullptr);
      continue;
    }
    // a run is longer than 64 rows only where it names a slot twice: its later rows come later
    while (true) {
      turn ^= 1;
      write_run<FMT, D, CT>(s, pg, rs, len, mine % BLK, sMax[turn]);
      if (len < WAVE) break;
      rs += WAVE;
      mine = slot_at(rs + lane);
      len = length(mine, pg);
      if (len == 0) break;
      __syncthreads();  // the next 64 rows of the run read and write the same page and scale
    }
  }
}

template <int FMT>
void launch_write_d(const kvskip_write_args& p, dim3 grid, int win, hipStream_t s) {
  if (p.D == 128)
    hipLaunchKernelGGL((cache_write_kernel<FMT, 128>), grid, dim3(CT), 0, s, p, win);
  else
    hipLaunchKernelGGL((cache_write_kernel<FMT, 64>), grid, dim3(CT), 0, s, p, win);
}

}  // namespace

// One launch of one workgroup up to ONE_ROWS rows of the map. Above, one launch of many workgroups where what they write
// is none of what the others read (the state's outputs are buffers of their own), else the sums and a filling launch. us,
// one workgroup / two launches: 24 requests of one new token 5.1 / 8.6, 2048 of one 8.3 / 12.8, 4 of 1024 6.3 / 8.1, 16 of
// 512 9.8 / 8.1, 64 of 2048 114 / 11.7; two launches / one of many workgroups: 257 mixed requests 10.0 / 6.9, 64 prompts
// of up to 4096 tokens 10.0 / 6.9.
constexpr int ONE_ROWS = 4096;

int page_work_ints(int B, int rows) { return rows <= ONE_ROWS ? 0 : 2 + 3 * B; }

static bool apart(const void* a, int64_t na, const void* b, int64_t nb) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return x + 4 * na <= y || y + 4 * nb <= x;
}

hipError_t launch_page_map(const kvskip_page_args& p, hipStream_t s) {
  const void* in[] = {p.seq_lens, p.new_lens, p.held, p.free_count};
  const int64_t n_in[] = {p.B, p.B, p.B, 1};
  const void* out[] = {p.starts, p.held_out, p.free_count_out, p.short_out, p.lens_out};
  const int64_t n_out[] = {p.B + 1, p.B, 1, 1, p.B};
  bool own = true;
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4 + (p.lens_out != nullptr); ++j) own = own && apart(in[i], n_in[i], out[j], n_out[j]);
  if (p.rows <= ONE_ROWS || own) {
    const int wgs = p.rows <= ONE_ROWS ? 1 : min(256, (p.rows + PT - 1) / PT);
    hipLaunchKernelGGL((page_sums_kernel<true>), dim3(wgs), dim3(PT), 0, s, p);
    return hipGetLastError();
  }
  hipLaunchKernelGGL((page_sums_kernel<false>), dim3(1), dim3(PT), 0, s, p);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(page_fill_kernel, dim3(min(512, (p.rows + PF - 1) / PF)), dim3(PF), 0, s, p);
  return hipGetLastError();
}

hipError_t launch_cache_write(const kvskip_write_args& p, hipStream_t s) {
  // Rows of the map a workgroup looks at: few enough that 4096 workgroups find work, at most 64 (a page of a prompt then
  // is one or two workgroups' and none ends with nothing to do), at least four (one new token a wavefront). 44 000 rows of
  // prompts, 8 heads, us: 4096 workgroups 51, with windows of 16 rows 83; 4096 single rows 34, by windows of 64 35.
  int win = 4;
  while (win < WAVE && static_cast<int64_t>(p.N) * 2 * p.Hkv > 4096 * win) win *= 2;
  const dim3 grid(2 * p.Hkv, (p.N + win - 1) / win);
  if (p.format == KVSKIP_BF16)
    launch_write_d<FMT_BF16>(p, grid, win, s);
  else if (p.format == KVSKIP_INT8)
    launch_write_d<FMT_INT8>(p, grid, win, s);
  else
    launch_write_d<FMT_E4M3>(p, grid, win, s);
  return hipGetLastError();
}

}  // namespace kvs
