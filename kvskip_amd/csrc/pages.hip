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
// written an element. A scale is a power of two: dividing by it is exact, so a code depends on its value and scale
// alone, and when a later row needs a larger scale, the rows that are there move to it without rounding again (e4m3:
// but for subnormal codes; int8 rounds once more per doubling, less than the final step in sum).
#include <cstdlib>
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

// Exclusive prefix of v over the workgroup's PT threads and its total; `tmp` holds one int a wavefront.
__device__ __forceinline__ int block_scan(int v, int* tmp, int& total) {
  const int wave = threadIdx.x / WAVE, lane = threadIdx.x % WAVE;
  const int incl = wave_incl_scan(v);
  __syncthreads();
  if (lane == WAVE - 1) tmp[wave] = incl;
  __syncthreads();
  const int x = wave_incl_scan(lane < PT / WAVE ? tmp[lane] : 0);
  total = __builtin_amdgcn_readlane(x, PT / WAVE - 1);
  return incl - v + (wave > 0 ? __shfl(x, wave - 1, WAVE) : 0);
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
// is read here: entries given back are read below what a request keeps or in rows that take none, stack positions from
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

// The sums; ONE: also page_fill (the whole operator in one launch).
template <bool ONE>
__global__ void __launch_bounds__(PT) page_sums_kernel(const kvskip_page_args p) {
  __shared__ Step s;
  __shared__ int tmp[PT / WAVE];
  const int tid = threadIdx.x;
  const int count = min(max(*p.free_count, 0), p.num_pages);
  int given = 0;
  for (int b0 = 0; b0 < p.B; b0 += PT) {
    const int b = b0 + tid;
    int n, a, h, need, g = 0, all;
    if (b < p.B && page_need(p, b, n, a, h, need)) g = max(h - need, 0);
    const int at = given + block_scan(g, tmp, all);
    if (b < p.B) s.given[b] = at;
    given += all;
  }
  const int avail = min(count + given, p.num_pages);
  int taken = 0, rows = 0, short_ = 0, used = 0;
  for (int b0 = 0; b0 < p.B; b0 += PT) {
    const int b = b0 + tid;
    int n = 0, a = 0, h = 0, need = 0, all;
    const bool fits = b < p.B && page_need(p, b, n, a, h, need);
    const int t = fits ? max(need - h, 0) : 0;
    const int before = taken + block_scan(t, tmp, all);
    taken += all;
    const bool served = fits && (t == 0 || before + t <= avail);
    const int start = rows + block_scan(min(a, p.rows + 1), tmp, all);
    rows += all;
    if (b < p.B) {
      s.starts[b] = start;
      s.taken[b] = served ? before : -1;
      s.held[b] = h;
      p.starts[b] = start;
      p.held_out[b] = served ? need : h;
    }
    // (not served, pages used: counts of at most 2^11 requests and 2^25 pages)
    short_ += __syncthreads_count(b < p.B && !served);
    block_scan(served ? t : 0, tmp, all);
    used += all;
  }
  if (tid == 0) {
    s.starts[p.B] = rows;
    p.starts[p.B] = rows;
    *p.short_out = short_;
    *p.free_count_out = avail - used;
  }
  __syncthreads();
  if constexpr (ONE) {
    page_fill(p, s, count, avail, tid, PT);
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

// One wavefront a workgroup: (window, KV head, keys or values), the runs that start in rows [w0, w0 + win) of the map.
template <int FMT, int D>
__global__ void __launch_bounds__(WAVE) cache_write_kernel(const kvskip_write_args p, int win) {
  constexpr int LPR = D / 8, RPI = WAVE / LPR, NI = BLK / RPI;  // lanes a row, rows a load, loads a page
  constexpr int EB = FMT == FMT_BF16 ? 2 : 1;
  const int lane = threadIdx.x, c = lane % LPR, r0 = lane / LPR;
  const int h = blockIdx.y;
  const bool isv = blockIdx.z != 0;
  const uint16_t* rows = static_cast<const uint16_t*>(isv ? p.v : p.k) + h * (isv ? p.v_sh : p.k_sh) + 8 * c;
  const int64_t sn = isv ? p.v_sn : p.k_sn;
  char* pool = static_cast<char*>(isv ? p.v_pool : p.k_pool) + h * (isv ? p.vp_sh : p.kp_sh) * EB + 8 * EB * c;
  const int64_t psb = (isv ? p.vp_sb : p.kp_sb) * EB, pst = (isv ? p.vp_st : p.kp_st) * EB;
  const int slots = p.num_pages * BLK;
  // slots of the window's 64 rows, of the 64 after them and of the row before: -1 for none
  const int w0 = blockIdx.x * win;
  auto slot_at = [&](int i) {
    const int s = i >= 0 && i < p.N ? p.slot_map[i] : -1;
    return s < slots ? max(s, -1) : -1;
  };
  int s0 = slot_at(w0 + lane), s1 = slot_at(w0 + WAVE + lane);
  const int prev = slot_at(w0 + lane - 1);
  uint64_t leaders = __ballot(lane < win && s0 >= 0 && (prev < 0 || s0 / BLK != prev / BLK));
  while (leaders != 0) {
    const int l0 = __builtin_ctzll(leaders);
    leaders &= leaders - 1;
    const int pg = __builtin_amdgcn_readlane(s0, l0) / BLK;
    // the run's slots, 64 rows at a time (it is longer only where it names a slot twice: later rows come later)
    int rs = w0 + l0;
    const int in0 = __shfl(s0, (l0 + lane) & 63, WAVE), in1 = __shfl(s1, (l0 + lane) & 63, WAVE);
    int mine = l0 + lane < WAVE ? in0 : in1;
    while (true) {
      const uint64_t on = __ballot(mine >= 0 && mine / BLK == pg);
      const int len = on == ~0ull ? WAVE : __builtin_ctzll(~on);
      if (len == 0) break;
      const int at = mine % BLK, first = __builtin_amdgcn_readfirstlane(at);
      const uint64_t run = len == WAVE ? ~0ull : (1ull << len) - 1;
      uint64_t keep = run, fresh = run << first;  // rows of the run that are kept; rows of the page they fill
      if ((__ballot(at == first + lane) & run) != run) {  // not one after another: of rows with one slot the last
        bool last = lane < len;
        fresh = 0;
        for (int l = 0; l < len; ++l) {
          const int r = __builtin_amdgcn_readlane(at, l);
          fresh |= 1ull << r;
          last = last && !(l > lane && r == at);
        }
        keep = __ballot(last);
      }
      u32x4 x[NI];
      int to[NI];  // this lane's row of the page, or -1
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int r = RPI * i + r0;
        to[i] = -1;
        x[i] = u32x4{0u, 0u, 0u, 0u};
        if (RPI * i < len) {  // uniform
          const int row = __shfl(at, r, WAVE);
          if (keep >> r & 1) {
            to[i] = row;
            x[i] = ld16_nt(rows + (rs + r) * sn);
          }
        }
      }
      char* out = pool + pg * psb;
      if constexpr (FMT == FMT_BF16) {
#pragma unroll
        for (int i = 0; i < NI; ++i)
          if (to[i] >= 0) *reinterpret_cast<u32x4*>(out + to[i] * pst) = x[i];
      } else {
        float* scale = (isv ? p.v_scale : p.k_scale) + pg * (isv ? p.vs_sb : p.ks_sb) + h * (isv ? p.vs_sh : p.ks_sh);
        const bool anew = fresh & 1;
        const float held = *scale;
        const float was = !anew && held > 0.f && held < __builtin_huge_valf() ? held : 0.f;
        // the largest magnitude, of bf16 bits without the sign: an infinity counts as the largest finite value, NaN not
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t lo = x[i][e] & 0x7fffu, hi = x[i][e] >> 16 & 0x7fffu;
            top = max(top, max(lo <= 0x7f80u ? lo : 0u, hi <= 0x7f80u ? hi : 0u));
          }
        const float amax = wave_max(__uint_as_float(min(top, 0x7f7fu) << 16));
        constexpr float QMAX = FMT == FMT_E4M3 ? 448.f : 127.f;
        const float now = amax > QMAX * was ? pow2_scale<FMT>(amax) : was;
        const float inv = now > 0.f ? 1.f / now : 0.f;  // exact where now is a power of two
#pragma unroll
        for (int i = 0; i < NI; ++i)
          if (to[i] >= 0) {
            const u32x4 w = x[i];
            *reinterpret_cast<u32x2*>(out + to[i] * pst) =
                u32x2{codes4<FMT>(bf_lo(w.x) * inv, bf_hi(w.x) * inv, bf_lo(w.y) * inv, bf_hi(w.y) * inv),
                      codes4<FMT>(bf_lo(w.z) * inv, bf_hi(w.z) * inv, bf_lo(w.w) * inv, bf_hi(w.w) * inv)};
          }
        if (now != was && !anew) {  // uniform: the page's other rows move to the larger scale
          const float f = was * inv;
          u32x2 old[NI];
#pragma unroll
          for (int i = 0; i < NI; ++i)
            if (!(fresh >> (RPI * i + r0) & 1)) old[i] = *reinterpret_cast<const u32x2*>(out + (RPI * i + r0) * pst);
#pragma unroll
          for (int i = 0; i < NI; ++i)
            if (!(fresh >> (RPI * i + r0) & 1)) {
              float a[4], b[4];
              values4<FMT>(old[i].x, a);
              values4<FMT>(old[i].y, b);
              *reinterpret_cast<u32x2*>(out + (RPI * i + r0) * pst) =
                  u32x2{codes4<FMT>(a[0] * f, a[1] * f, a[2] * f, a[3] * f),
                        codes4<FMT>(b[0] * f, b[1] * f, b[2] * f, b[3] * f)};
            }
        }
        if (lane == 0 && !(now == held)) *scale = now;
      }
      if (len < WAVE) break;
      rs += WAVE;
      mine = slot_at(rs + lane);
      // (the next 64 rows of the run read and write the same page and scale: after this chunk's stores)
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
    }
  }
}

template <int FMT>
void launch_write_d(const kvskip_write_args& p, dim3 grid, int win, hipStream_t s) {
  if (p.D == 128)
    hipLaunchKernelGGL((cache_write_kernel<FMT, 128>), grid, dim3(WAVE), 0, s, p, win);
  else
    hipLaunchKernelGGL((cache_write_kernel<FMT, 64>), grid, dim3(WAVE), 0, s, p, win);
}

}  // namespace

// One launch up to ONE_ROWS rows of the map, else the sums and a filling launch.
constexpr int ONE_ROWS = 4096;

int page_work_ints(int B, int rows) { return rows <= ONE_ROWS ? 0 : 2 + 3 * B; }

hipError_t launch_page_map(const kvskip_page_args& p, hipStream_t s) {
  if (p.rows <= ONE_ROWS) {
    hipLaunchKernelGGL((page_sums_kernel<true>), dim3(1), dim3(PT), 0, s, p);
    return hipGetLastError();
  }
  hipLaunchKernelGGL((page_sums_kernel<false>), dim3(1), dim3(PT), 0, s, p);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(page_fill_kernel, dim3(min(512, (p.rows + PF - 1) / PF)), dim3(PF), 0, s, p);
  return hipGetLastError();
}

hipError_t launch_cache_write(const kvskip_write_args& p, hipStream_t s) {
  static const int wv = getenv("KVS_WIN") ? atoi(getenv("KVS_WIN")) : 16;
  const int win = static_cast<int64_t>(p.N) * p.Hkv <= 16384 ? 1 : wv;
  const dim3 grid((p.N + win - 1) / win, p.Hkv, 2);
  if (p.format == KVSKIP_BF16)
    launch_write_d<FMT_BF16>(p, grid, win, s);
  else if (p.format == KVSKIP_INT8)
    launch_write_d<FMT_INT8>(p, grid, win, s);
  else
    launch_write_d<FMT_E4M3>(p, grid, win, s);
  return hipGetLastError();
}

}  // namespace kvs
