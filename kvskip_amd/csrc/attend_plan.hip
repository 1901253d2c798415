// Plan of the attention of a step's rows: tiles of virtual rows, the pages that each one sees, and their cut into units of
// about equal work (attend.hpp has the records). One workgroup, integers only; a step's layers share it.
//
//   1. a request's tiles are counted and summed (LDS holds every request's first tile), a shared prefix's rows listed;
//   2. every tile finds its pages: [0, a1) that prefix_lens shows it and [b0, ...) up to its last row, from its first
//      row's window on; the pages' sum gives the chunk that a unit takes;
//   3. partial rows and the runs of rows to join are counted in tile order, so that results never depend on when a workgroup ran;
//   4. units are written longest first, by a counting sort over 32 classes of length (their order inside a class is
//      whatever the atomics gave: it decides when a unit starts and nothing else).
// Every record lies inside its array by attend_sizes' bounds: a row belongs to one request, so tiles are at most the rows' share
// and one more a request and prefix; ceil(pages / chunk) over all of them is at most TARGET_UNITS / Hkv more than their number;
// a tile cut in two or more has at most 2 pages / chunk units of at most a tile's rows.
#include "attn_common.hpp"
#include "attend.hpp"

namespace kvs {

namespace {

constexpr int PT = 1024;  // threads
constexpr int CLASSES = 32;

// Workgroups that run at once: two a CU. (Units for one round of them, 24 tokens of up to 20011 behind a window of 4096: 47.1 us
// with 1024 units in about two rounds, 39.0; 16 tokens of up to 32000 54.3, 47.4; one of 32768 33.9, 24.0.)
constexpr int SLOTS = 512;
constexpr int TARGET_UNITS = 2 * SLOTS;  // units of a queued plan: those that end early take another
constexpr int LEAST_PAGES = 4;           // of a chunk: a unit's four wavefronts take a page each
// Of a chunk of a queued plan: partial results cost more than a shorter last round saves. (Least 4, 16 and 32, us, with one part a
// weight: 9 prompts of up to 763 behind bidirectional prefixes 86.5, 63.5, 63.3; 7 of up to 1412 in a window of 234 72, 43, 43; 64
// tokens behind a prefix of 8192 46.8, 42, 61.) A tile is cut evenly into ceil(pages / chunk) units, which hold half a chunk or more.
constexpr int LEAST_QUEUED = 16;

struct PlanP {
  kvskip_attend_plan_args a;
  int few, many;  // heights (many 0: small tiles only)
  int at_units, at_joins, at_tiles, at_rows;
};

struct Group {
  int rows, row0, len, height, tile0, min_pos, max_pre;
};

struct Request {
  int first, n, end, len, base, pre, group;  // its rows among the call's; the row after its last; group -1: behind no prefix
  __device__ int pos0() const { return base + len - (end - first); }
};
constexpr int MOST_END = 1 << 28;  // (no request has more tokens and rows before them: positions stay in 32 bits)

__device__ __forceinline__ Request request(const PlanP& p, int b) {
  Request r;
  r.first = min(max(p.a.starts[b], 0), p.a.rows);
  r.end = min(p.a.starts[b + 1], MOST_END);
  r.n = min(max(r.end, r.first), p.a.rows) - r.first;
  r.len = min(max(p.a.seq_lens[b], 0), p.a.T);
  r.group = p.a.shared > 0 ? p.a.shared_of[b] : -1;
  if (r.group < 0 || r.group >= p.a.shared) r.group = -1;
  r.base = r.group >= 0 ? min(max(p.a.shared_lens[r.group], 0), p.a.shared_T) : 0;
  if (r.base == 0) r.group = -1;
  r.pre = p.a.prefix_lens != nullptr ? min(max(p.a.prefix_lens[b], 0), r.base + r.len) : 0;
  return r;
}

// Rows of a request are numbered from its own tiles' height.
__device__ __forceinline__ int height(const PlanP& p, int virt) { return p.many == 0 || virt <= p.few ? p.few : p.many; }

// Exclusive sums over the workgroup in thread order, `total` of all.
__device__ __forceinline__ int block_scan(int v, int* sW, int& total) {
  const int wave = threadIdx.x / WAVE, lane = threadIdx.x % WAVE;
  const int incl = wave_incl_scan(v);
  if (lane == WAVE - 1) sW[wave] = incl;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < PT / WAVE; ++w) {
    before += w < wave ? sW[w] : 0;
    total += sW[w];
  }
  __syncthreads();
  return before + incl - v;
}

// The pages that a tile sees: [0, a1), then [b0, a1's end ...): `pages` in all.
struct Span {
  int a1, b0, pages;
};
__device__ __forceinline__ Span span(int lo, int hi, int base, int len, int pre, int window) {
  const int end = min(len, max(hi - base + 1, 0));
  const int from = window > 0 ? max(lo - window + 1 - base, 0) : 0;
  const int shown = min(max(pre - base, 0), len);
  Span s;
  s.a1 = (shown + BLK - 1) / BLK;
  s.b0 = max(from / BLK, s.a1);
  s.pages = s.a1 + max((end + BLK - 1) / BLK - s.b0, 0);
  return s;
}

__global__ void __launch_bounds__(PT) attend_plan_kernel(const PlanP p) {
  __shared__ int sTile[MAX_ATTEND_B + 1];  // a request's first tile
  __shared__ int sPlace[MAX_ATTEND_B];     // its first row among those of its prefix
  __shared__ Group sGr[MAX_SHARED];
  __shared__ int sW[PT / WAVE];
  __shared__ int sClass[CLASSES];
  __shared__ int sMost, sFit;
  const int tid = threadIdx.x, G = p.a.Hq / p.a.Hkv, window = p.a.window;
  int* work = p.a.work;
  AttendUnit* units = reinterpret_cast<AttendUnit*>(work + p.at_units);
  AttendJoin* joins = reinterpret_cast<AttendJoin*>(work + p.at_joins);
  AttendTile* tiles = reinterpret_cast<AttendTile*>(work + p.at_tiles);
  AttendRow* rows = reinterpret_cast<AttendRow*>(work + p.at_rows);

  // ---- 1. requests (starts that do not rise would give rows to two of them: then no row belongs to any)
  if (tid < CLASSES) sClass[tid] = 0;
  if (tid == 0) sMost = 1, sFit = INT32_MAX;
  bool fall = false;
  for (int b = tid; b < p.a.B; b += PT) fall |= p.a.starts[b + 1] < p.a.starts[b];
  const int B = __syncthreads_or(fall) ? 0 : p.a.B;
  int own = 0;
  for (int b0 = 0; b0 < B; b0 += PT) {
    const int b = b0 + tid;
    int t = 0;
    if (b < B) {
      const Request r = request(p, b);
      const int virt = r.n * G, h = height(p, virt);
      t = (virt + h - 1) / h;
    }
    int total;
    const int at = own + block_scan(t, sW, total);
    if (b < B) sTile[b] = at;
    own += total;
  }
  if (tid == 0) sTile[B] = own;
  int row0 = 0;
  for (int g = 0; g < p.a.shared; ++g) {
    if (tid == 0) sGr[g] = Group{0, row0, 0, 0, 0, INT32_MAX, 0};
    __syncthreads();
    int count = 0;
    for (int b0 = 0; b0 < B; b0 += PT) {
      const int b = b0 + tid;
      Request r{0, 0, 0, 0, 0, 0, -1};
      if (b < B) r = request(p, b);
      const bool in = r.group == g && r.n > 0;
      int total;
      const int at = count + block_scan(in ? r.n : 0, sW, total);
      if (in) {
        sPlace[b] = at;
        atomicMin(&sGr[g].min_pos, r.pos0());
        atomicMax(&sGr[g].max_pre, r.pre);
        sGr[g].len = r.base;  // (the same of all)
      }
      count += total;
    }
    if (tid == 0) sGr[g].rows = count;
    row0 += count;
    __syncthreads();
  }
  if (tid == 0) {
    int at = own;
    for (int g = 0; g < p.a.shared; ++g) {
      const int virt = sGr[g].rows * G, h = height(p, virt);
      sGr[g].height = h;
      sGr[g].tile0 = at;
      at += (virt + h - 1) / h;
    }
    sW[0] = at;
  }
  __syncthreads();
  const int n_tiles = sW[0];
  __syncthreads();
  // rows: positions, and those behind a prefix
  const int first = B > 0 ? min(max(p.a.starts[0], 0), p.a.rows) : 0, last = B > 0 ? min(max(p.a.starts[B], first), p.a.rows) : 0;
  for (int i = tid; i < p.a.rows; i += PT)
    if (i < first || i >= last) p.a.positions[i] = -1;
  for (int b = tid / WAVE; b < B; b += PT / WAVE) {
    const Request r = request(p, b);
    const int place = r.group >= 0 && r.n > 0 ? sGr[r.group].row0 + sPlace[b] : 0;
    for (int i = tid % WAVE; i < r.n; i += WAVE) {
      p.a.positions[r.first + i] = r.pos0() + i;
      if (r.group >= 0) rows[place + i] = AttendRow{r.first + i, r.pos0() + i, r.pre, 0};
    }
  }

  // ---- 2. tiles
  int64_t sum = 0;
  for (int t = tid; t < n_tiles; t += PT) {
    AttendTile x;
    if (t < own) {
      int lo = 0, hi = B - 1;  // the last request whose first tile is at most t, of those that have any
      while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (sTile[mid] <= t)
          lo = mid;
        else
          hi = mid - 1;
      }
      const Request r = request(p, lo);
      const int virt = r.n * G, h = height(p, virt), v0 = (t - sTile[lo]) * h, v1 = min(v0 + h, virt) - 1;
      x = AttendTile{lo, v0, span(r.pos0() + v0 / G, r.pos0() + v1 / G, r.base, r.len, r.pre, window).pages, -1};
    } else {
      int g = 0;
      while (g + 1 < p.a.shared && sGr[g + 1].tile0 <= t) ++g;
      const Group& r = sGr[g];
      x = AttendTile{~g, (t - r.tile0) * r.height, span(r.min_pos, INT32_MAX - 1, 0, r.len, r.max_pre, window).pages, -1};
    }
    tiles[t] = x;
    sum += x.pages;
  }
  __shared__ unsigned long long sSum;
  if (tid == 0) sSum = 0;
  __syncthreads();
  atomicAdd(&sSum, static_cast<unsigned long long>(sum));
  __syncthreads();
  // the shortest of 16 chunks whose units all run at once, or where there is none a queue's
  const int64_t all_pages = static_cast<int64_t>(sSum);
  const int room = max(SLOTS / p.a.Hkv, 1);
  if (n_tiles <= room) {  // uniform
    const int wave = tid / WAVE, c0 = static_cast<int>(max(static_cast<int64_t>(LEAST_PAGES), (all_pages + room - 1) / room));
    const int c = c0 + (c0 * wave + PT / WAVE - 1) / (PT / WAVE);
    int n = 0;
    for (int t = tid % WAVE; t < n_tiles; t += WAVE) n += (tiles[t].pages + c - 1) / c;
    if (wave_sum_int(n) <= room && tid % WAVE == 0) atomicMin(&sFit, c);
  }
  __syncthreads();
  const int queued = static_cast<int>(max(static_cast<int64_t>(LEAST_QUEUED), (all_pages * p.a.Hkv + TARGET_UNITS - 1) / TARGET_UNITS));
  const int chunk = sFit != INT32_MAX ? sFit : queued;
  auto cut = [&](int pages) { return min(max((pages + chunk - 1) / chunk, 1), MAX_TILE_UNITS); };

  // ---- 3. partial rows in tile order; the longest unit
  int parts = 0;
  for (int t0 = 0; t0 < n_tiles; t0 += PT) {
    const int t = t0 + tid;
    int nv = 0, ns = 0;
    bool partial = false;
    if (t < n_tiles) {
      const AttendTile x = tiles[t];
      int virt, group;
      if (x.who >= 0) {
        const Request r = request(p, x.who);
        virt = r.n * G, group = r.group;
        nv = min(height(p, virt), virt - x.v0);
      } else {
        group = ~x.who;
        nv = min(sGr[group].height, sGr[group].rows * G - x.v0);
      }
      ns = cut(x.pages);
      partial = group >= 0 || ns > 1;
      atomicMax(&sMost, (x.pages + ns - 1) / ns);
    }
    int total;
    const int at = parts + block_scan(partial ? nv * ns : 0, sW, total);
    parts += total;
    if (t < n_tiles) tiles[t].part = partial ? at : -1, tiles[t].nv = nv, tiles[t].ns = ns;
  }
  __syncthreads();  // (the joins read the tiles of a prefix, other threads')
  // runs of rows to join: up to JOIN_ROWS of a tile, of one tile of the prefix
  int n_joins = 0;
  for (int t0 = 0; t0 < own; t0 += PT) {
    const int t = t0 + tid;
    AttendTile x{};
    int group = -1, place = 0, runs = 0;
    Request r{};
    if (t < own) {
      x = tiles[t];
      if (x.part >= 0) {
        r = request(p, x.who);
        group = r.group;
        place = group >= 0 ? sPlace[x.who] * G + x.v0 : 0;
      }
    }
    auto run = [&](int i) {  // length of the one at row i
      const int n = min(x.nv - i, JOIN_ROWS);
      return group >= 0 ? min(n, sGr[group].height - (place + i) % sGr[group].height) : n;
    };
    if (x.part >= 0 && t < own)
      for (int i = 0; i < x.nv; i += run(i)) ++runs;
    int total;
    int j = n_joins + block_scan(runs, sW, total);
    n_joins += total;
    if (runs > 0)
      for (int i = 0; i < x.nv; i += run(i), ++j) {
        AttendJoin o{r.first, x.v0 + i, run(i), x.part + i, x.ns, x.nv, 0, 0, 0, {0, 0, 0}};
        if (group >= 0) {
          const int v = place + i, h = sGr[group].height;
          const AttendTile y = tiles[sGr[group].tile0 + v / h];
          o.more = y.part + v % h, o.more_ns = y.ns, o.more_step = y.nv;
        }
        joins[j] = o;
      }
  }
  // ---- 4. units, longest first
  const int most = sMost;
  auto cls = [&](int pages, int ns) {
    const int per = (pages + ns - 1) / ns;
    return CLASSES - 1 - static_cast<int>(static_cast<int64_t>(per) * (CLASSES - 1) / most);
  };
  for (int t = tid; t < n_tiles; t += PT) {
    const int pages = tiles[t].pages, ns = tiles[t].ns;
    atomicAdd(&sClass[cls(pages, ns)], ns);
  }
  __syncthreads();
  if (tid == 0) {
    int at = 0;
    for (int c = 0; c < CLASSES; ++c) {
      const int n = sClass[c];
      sClass[c] = at;
      at += n;
    }
    work[H_UNITS] = at;
    work[H_JOINS] = n_joins;
    work[H_FIRST] = first;
    work[H_LAST] = last;
  }
  __syncthreads();
  for (int t = tid; t < n_tiles; t += PT) {
    const AttendTile x = tiles[t];
    const int ns = x.ns;
    AttendUnit u{};
    u.nv = x.nv;
    u.v0 = x.v0;
    Span s;
    if (x.who >= 0) {
      const Request r = request(p, x.who);
      const int virt = r.n * G;
      u.kind = height(p, virt) == p.many ? 1 : 0;
      u.row0 = r.first;
      u.p0 = r.pos0();
      u.pre = r.pre;
      u.table = x.who;
      u.len = r.len;
      u.base = r.base;
      s = span(u.p0 + u.v0 / G, u.p0 + (u.v0 + u.nv - 1) / G, r.base, r.len, r.pre, window);
    } else {
      const Group& g = sGr[~x.who];
      u.kind = 2 | (g.height == p.many ? 1 : 0);
      u.row0 = g.row0;
      u.table = ~x.who;
      u.len = g.len;
      s = span(g.min_pos, INT32_MAX - 1, 0, g.len, g.max_pre, window);
    }
    u.a1 = s.a1;
    u.b0 = s.b0;
    const int at = atomicAdd(&sClass[cls(x.pages, ns)], ns);
    for (int i = 0; i < ns; ++i) {
      u.i0 = static_cast<int>(static_cast<int64_t>(x.pages) * i / ns);
      u.n = static_cast<int>(static_cast<int64_t>(x.pages) * (i + 1) / ns) - u.i0;
      u.part = x.part >= 0 ? x.part + i * u.nv : -1;
      units[at + i] = u;
    }
  }
}

}  // namespace

AttendSizes attend_sizes(const kvskip_attend_plan_args& p) {
  AttendSizes z{};
  const int64_t G = p.Hq / p.Hkv, virt = static_cast<int64_t>(p.rows) * G;
  const int64_t most = p.max_rows > 0 && p.max_rows < p.rows ? p.max_rows : p.rows;
  z.large = most * G > TILE_FEW || (p.shared > 0 && virt > TILE_FEW);
  z.few = TILE_FEW;
  z.many = z.large ? TILE_MANY : 0;
  // a small tile holds a whole request where large ones occur, so a batch has at most one short tile a request
  const int64_t h = z.large ? z.many : z.few;
  z.tiles = virt / h + p.B + (p.shared > 0 ? virt / h + p.shared : 0);
  // a run a JOIN_ROWS rows, one more a tile, and one more where a tile of a prefix ends inside it
  z.joins = virt / JOIN_ROWS + z.tiles;
  const int64_t cut = TARGET_UNITS / p.Hkv + 1;  // units beyond one a tile: the sum of floor(pages / chunk)
  z.units = z.tiles + cut;
  const int64_t tall = virt < h ? virt : h;
  z.part_rows = 2 * cut * tall + (p.shared > 0 ? 2 * virt : 0);
  auto up = [](int64_t n) { return (n + 15) / 16 * 16; };
  z.at_units = HEAD;
  z.at_joins = z.at_units + up(z.units * (sizeof(AttendUnit) / 4));
  z.at_tiles = z.at_joins + up(z.joins * (sizeof(AttendJoin) / 4));
  z.at_rows = z.at_tiles + up(z.tiles * (sizeof(AttendTile) / 4));
  z.total = z.at_rows + (p.shared > 0 ? up(static_cast<int64_t>(p.rows) * (sizeof(AttendRow) / 4)) : 0);
  return z;
}

hipError_t launch_attend_plan(const kvskip_attend_plan_args& a, const AttendSizes& z, hipStream_t s) {
  PlanP p;
  p.a = a;
  p.a.window = a.window < (1 << 30) ? a.window : 1 << 30;  // (positions are below 2^29: no limit)
  p.few = z.few, p.many = z.many;
  p.at_units = static_cast<int>(z.at_units), p.at_joins = static_cast<int>(z.at_joins);
  p.at_tiles = static_cast<int>(z.at_tiles), p.at_rows = static_cast<int>(z.at_rows);
  hipLaunchKernelGGL(attend_plan_kernel, dim3(1), dim3(PT), 0, s, p);
  return hipGetLastError();
}

}  // namespace kvs
