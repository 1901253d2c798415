// Split-K decode attention over a cache held in 8 bits (e4m3 or int8) with a scale for each 64-token block and KV
// head: dense or over block lists, contiguous or paged, one length or a ragged batch, with optional block statistics.
//
//   s_t = scale ks[blk] (q . k_t),  p_t = exp(s_t - m),  out = sum_t p_t vs[blk] v_t / sum_t p_t
//
// The work is cut as the bf16 pass cuts it (attn_common.hpp: workgroups of four independent wavefronts, a block per
// wavefront and step, the split merge a second launch); what differs is inside a block:
//   scores    e4m3  codes to fp16, exactly (the hardware's conversion), and products with q on v_mfma_f32_16x16x32_f16, q
//                   in fp16 times a power of two of its head, so that its largest value is near 2^15: whole, but for what
//                   lies below 2^-39 of that. (The matrix unit also takes e4m3 itself, q cut to two parts of it: a
//                   quarter of the products and no conversions, but it sums them to 12 to 16 bits of the largest only,
//                   measured, where fp16 products are summed in fp32.)
//             int8  K's codes as they lie in memory, q in four digits of 8 bits, together in steps of 2^-29 of its head's
//                   largest value (v_mfma_i32_16x16x64_i8, exact sums), the digits on the columns that the group's heads
//                   leave free.
//   weights   e = 2^(s - block maximum) times 2^(mt - r) vs in two fp16 parts, 22 bits (softmax sums are taken before, in
//             fp32). Up to 8 heads the low parts are the operand rows that the group's heads leave free, with accumulators
//             of their own (no further product); 9 to 16 heads take a second product for them, onto the same accumulators.
//             r is the accumulators' reference, at most 2^7 below the largest weight times |vs| so far: they are rescaled
//             only when a block passes that. (fp16 holds nothing finer than 2^-24, so beside its 2^-22 a weight is off by up
//             to 2^-32 of the largest p |vs| of the wavefront.) One part: 32 sequences
//             of 65536 tokens 612.5 us for 613.8, a ragged batch of 24 of 64 dims 35.1 for 35.5.
//   V         codes to fp16, exactly (e4m3 by the hardware's conversion, int8 by placing the byte under the exponent of 1024
//             and taking 1152 off), rows paired by byte permutation, and P V on v_mfma_f32_16x16x32_f16.
//   items     lane l of a wavefront holds block, page and scales of the wavefront's step 64 i + l (one gather per 64
//             steps, the next one fetched during this one in three stages, since a page needs its list entry and a
//             scale its page); the loop takes them by readlane, so no step waits for them.
//   memory    each block has a buffer resource of its own, based at the block's first row and ending with the
//             sequence's last token: no offset of a cache of any length passes 32 bits, rows past the end read zeros
//             (whatever codes a page holds there), and an empty block reads nothing.
#include "attn_common.hpp"

namespace kvs {
namespace {

typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));

// Four codes of a dword as fp16: codes 0, 1 and codes 2, 3.
template <bool I8>
__device__ __forceinline__ u32x2 widen4(uint32_t w) {
  uint32_t lo, hi;
  if constexpr (I8) {
    const uint32_t u = w ^ 0x80808080u;  // x + 128
    const f16x2_t off = {-1152.f16, -1152.f16};
    lo = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2_t, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) + off);
    hi = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2_t, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) + off);
  } else {
    lo = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, false));
    hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, true));
  }
  return u32x2{lo, hi};
}

__device__ __forceinline__ u32x2 bload8(rsrc_t r, uint32_t voff, uint32_t soff) {
  return __builtin_amdgcn_raw_buffer_load_b64(r, static_cast<int>(voff), static_cast<int>(soff), BUF_NT);
}

// Sizes of a block's registers: K as 16-byte chunks of a row (lane r = lane % 16, j = lane / 16 holds bytes 16 j + 64 c
// of row 16 nt + r, which are k-steps 2 c and 2 c + 1 of the scores' products; q is laid out alike), V as 8 bytes of a
// row (D 128: a 16-lane group loads one row; D 64: two, and lanes c and c ^ 8 exchange halves).
template <int D>
struct Lay8 {
  static constexpr int KC = D / 64;
  static constexpr int KS = D / 32;
  static constexpr int VN = BLK * D / (WAVE * 8);
  static constexpr int VD = D / 16;
};

template <int D>
__device__ __forceinline__ void load_k8(u32x4 (&kr)[4][Lay8<D>::KC], rsrc_t r, uint32_t koff, uint32_t st) {
#pragma unroll
  for (int nt = 0; nt < 4; ++nt)
#pragma unroll
    for (int c = 0; c < Lay8<D>::KC; ++c) kr[nt][c] = bload16<BUF_NT>(r, koff + 64 * c, 16 * nt * st);
}

template <int D>
__device__ __forceinline__ void load_v8(u32x2 (&vr)[Lay8<D>::VN], rsrc_t r, uint32_t voff, uint32_t st) {
#pragma unroll
  for (int i = 0; i < Lay8<D>::VN; ++i) {
    const int t = D == 128 ? mf_tok(i / 4, i % 4, 0) : mf_tok(i / 2, 2 * (i % 2), 0);
    vr[i] = bload8(r, voff, t * st);
  }
}

// Dword d (4 dims) of tokens (nt, i) and (nt, i + 1), i even, of this lane's column.
template <int D>
__device__ __forceinline__ void v_pair8(const u32x2 (&vr)[Lay8<D>::VN], int nt, int i, int d, bool up, uint32_t& a,
                                        uint32_t& c) {
  if constexpr (D == 128) {
    a = vr[4 * nt + i][d];
    c = vr[4 * nt + i + 1][d];
  } else {  // up: lanes c >= 8, which loaded the second token's row
    const u32x2 x = vr[2 * nt + i / 2];
    const uint32_t other = dppu<DPP_ROR8>(up ? x.x : x.y);
    a = up ? other : x.x;
    c = up ? x.y : other;
  }
}

// Two values as fp16, to nearest even, the first in the low half.
__device__ __forceinline__ uint32_t pack_h(float a, float b) {
  typedef float f32x2_t __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_t{a, b}), f16x2_t));
}

// (a, b) c + h as fp16, rounded once (v_fma_mixlo_f16, v_fma_mixhi_f16).
__device__ __forceinline__ uint32_t mix_h(float a, float b, float c, f16x2_t h) {
  return __builtin_bit_cast(uint32_t, f16x2_t{static_cast<_Float16>(fmaf(a, c, static_cast<float>(h.x))),
                                              static_cast<_Float16>(fmaf(b, c, static_cast<float>(h.y)))});
}

typedef int i32x4_t __attribute__((ext_vector_type(4)));

// q as the B operands of the scores' products: column c is head c % GP.
//   e4m3  x[ks]: fp16 of the dims of k-step ks, 64 (ks / 2) + 16 j + 8 (ks % 2) .. + 7
//   int8  y[n][c]: dims 64 c + 16 j .. + 15 of one digit: GP 4 the digits on the four column groups, GP 8 on two groups of
//         two products, GP 16 four products. z: the weight of this lane's column in the last one
//         (the digits of a product before it weigh 2^(8 digits a product) more).
template <int D, int GP, bool I8>
struct Q8 {
  static constexpr int NY = GP / 4, KC = D / 64, KS = D / 32;
  u32x4 x[I8 ? 1 : KS];
  u32x4 y[I8 ? NY : 1][KC];
  float z;
};

template <int D, int GP, bool I8>
__device__ __forceinline__ void make_q8(Q8<D, GP, I8>& qb, const u32x4 (&qr)[D / 32], float up, int lane) {
  typedef Q8<D, GP, I8> Q;
  const int c = lane & 15;
  if constexpr (I8) {
#pragma unroll
    for (int n = 0; n < Q::NY; ++n) {
      const int digit = GP == 4 ? c / 4 : GP == 8 ? 2 * n + c / 8 : n;  // 0 (weight 2^24) .. 3 (1)
      if (n == Q::NY - 1) qb.z = __uint_as_float((127u + 24u - 8u * digit) << 23);
      // a digit's byte of each of two values; the lower three are held with 128 added
      const uint32_t pick = 0x0c0c0000u | (7u - digit) << 8 | (3u - digit), flip = digit == 0 ? 0u : 0x80808080u;
#pragma unroll
      for (int k = 0; k < Q::KC; ++k)
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          uint32_t v[4];
#pragma unroll
          for (int o = 0; o < 4; ++o) {
            const uint32_t two = qr[2 * k + u / 2][2 * (u % 2) + o / 2];
            // (below 2^30: the top digit is within +-64)
            v[o] = static_cast<uint32_t>(static_cast<int>(__builtin_rintf((o % 2 ? bf_hi(two) : bf_lo(two)) * up))) + 0x00808080u;
          }
          qb.y[n][k][u] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(v[3], v[2], pick), __builtin_amdgcn_perm(v[1], v[0], pick),
                                                0x05040100u) ^ flip;
        }
    }
  } else {
#pragma unroll
    for (int ks = 0; ks < Q::KS; ++ks)
#pragma unroll
      for (int e = 0; e < 4; ++e) qb.x[ks][e] = pack_h(bf_lo(qr[ks][e]) * up, bf_hi(qr[ks][e]) * up);
  }
}

// Scores of a block's tokens from K's codes (times the power of two of q): s[nt][i] of head c % GP on every lane.
template <int D, int GP, bool I8>
__device__ __forceinline__ void qk8(float (&s)[4][4], const u32x4 (&kr)[4][D / 64], const Q8<D, GP, I8>& qb, int lane) {
  typedef Q8<D, GP, I8> Q;
#pragma unroll
  for (int nt = 0; nt < 4; ++nt) {
    if constexpr (I8) {
#pragma unroll
      for (int n = 0; n < Q::NY; ++n) {
        i32x4_t a = {0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < Q::KC; ++k)
          a = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4_t, kr[nt][k]),
                                                    __builtin_bit_cast(i32x4_t, qb.y[n][k]), a, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float x = static_cast<float>(a[i]);
          s[nt][i] = n == 0 ? x : fmaf(s[nt][i], GP == 8 ? 65536.f : 256.f, x);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (GP <= 8) s[nt][i] *= qb.z;
        if constexpr (GP <= 8) s[nt][i] += dpp<DPP_ROR8>(s[nt][i]);
        if constexpr (GP == 4) s[nt][i] += dpp<0x124>(s[nt][i]);  // row_ror:4
      }
    } else {
      f32x4_t a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < Q::KS; ++ks) {
        const u32x2 w0 = widen4<I8>(kr[nt][ks / 2][2 * (ks % 2)]), w1 = widen4<I8>(kr[nt][ks / 2][2 * (ks % 2) + 1]);
        const u32x4 w = {w0.x, w0.y, w1.x, w1.y};
        a = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, w), __builtin_bit_cast(f16x8_t, qb.x[ks]), a,
                                                   0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) s[nt][i] = a[i];
    }
  }
}

// acc *= alpha of each row's head (alpha: this lane's head's).
template <int D, int GP>
__device__ __forceinline__ void rescale8(f32x4_t (&acc)[D / 16], float alpha, int lane) {
  float r[4];
  if constexpr (GP == 16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = __shfl(alpha, 4 * (lane >> 4) + i, WAVE);
  } else {
    r[0] = dpp<0x150>(alpha), r[1] = dpp<0x151>(alpha), r[2] = dpp<0x152>(alpha), r[3] = dpp<0x153>(alpha);  // row_newbcast
    if constexpr (GP == 8) {
      const bool odd = (lane & 16) != 0;  // rows 4 .. 7
      r[0] = odd ? dpp<0x154>(alpha) : r[0], r[1] = odd ? dpp<0x155>(alpha) : r[1];
      r[2] = odd ? dpp<0x156>(alpha) : r[2], r[3] = odd ? dpp<0x157>(alpha) : r[3];
    }
  }
#pragma unroll
  for (int j = 0; j < D / 16; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[j][i] *= r[i];
}

// LDS of the epilogue: the wavefronts' accumulators by part and head, and each head's (m, l, reference of the accumulators, its
// two parts) of all wavefronts.
template <int D, int GP>
struct Merge8 {
  static constexpr int NP = GP == 16 ? 1 : 2;  // parts of the weights with accumulators of their own
  float acc[NWAVE * NP * GP * D];
  f32x4_t m[GP], l[GP], r[GP], x[GP];
};

// The wavefronts' states merged: out / out_f32 / lse (whole: all of the list) or the split partials; a thread four dims of
// a head. (A dim a thread, every value of the wavefronts a load of its own: 0.9 us for 4 heads of 128 dims, 1.3 for 7.)
template <int D, int GP>
__device__ __forceinline__ void finish8(const Attn8P& p, int b, int h, int split, bool whole, const Merge8<D, GP>& L) {
  static_assert(NWAVE == 4, "a vector holds a value of each wavefront");
  constexpr int NP = Merge8<D, GP>::NP;
  const int S = p.num_splits;
  __syncthreads();
  const int64_t hq0 = static_cast<int64_t>(b) * p.Hq + static_cast<int64_t>(h) * p.G;
  for (int o = threadIdx.x; o < p.G * (D / 4); o += NT) {
    const int g = o / (D / 4), d = o % (D / 4) * 4;
    const f32x4_t m = L.m[g], l = L.l[g], r = L.r[g], rx = L.x[g];
    const float M = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
    const float mu = M == NEG_INF ? 0.f : M;
    f32x4_t A = {0.f, 0.f, 0.f, 0.f};
    float Ls = 0.f;
#pragma unroll
    for (int w = 0; w < NWAVE; ++w) {
      Ls += l[w] * fexp2(m[w] - mu);
      f32x4_t x = *reinterpret_cast<const f32x4_t*>(L.acc + (w * NP * GP + g) * D + d);
      if constexpr (NP == 2) x -= *reinterpret_cast<const f32x4_t*>(L.acc + ((w * NP + 1) * GP + g) * D + d);
      A += x * fexp2((r[w] - mu) + (rx[w] - 7.f));
    }
    const int64_t hq = hq0 + g;
    if (whole) {
      // (a NaN sum, from a NaN of q or the cache, comes out as NaN)
#pragma unroll
      for (int i = 0; i < 4; ++i) A[i] = Ls == 0.f ? 0.f : A[i] / Ls;
      *reinterpret_cast<u32x2*>(p.out + hq * D + d) =
          u32x2{f2bf(A[0]) | static_cast<uint32_t>(f2bf(A[1])) << 16, f2bf(A[2]) | static_cast<uint32_t>(f2bf(A[3])) << 16};
      if (p.out_f32) *reinterpret_cast<f32x4_t*>(p.out_f32 + hq * D + d) = A;
      if (p.lse && d == 0) p.lse[hq] = Ls == 0.f ? NEG_INF : (M + flog2(Ls)) * LN2;
    } else {
      *reinterpret_cast<f32x4_t*>(p.part_acc + (hq * S + split) * D + d) = A;
      if (d == 0) *reinterpret_cast<float2*>(p.part_ml + (hq * S + split) * 2) = make_float2(M, Ls);
    }
  }
}

// (-inf, 0) statistics of blocks a .. a + len - 1 of the KV head whose first query head is hq0: thread t of `stride`.
__device__ __forceinline__ void empty_stats(const Attn8P& p, int64_t hq0, int a, int len, int t, int stride) {
  for (int g = 0; g < p.G; ++g)
    for (int x = t; x < len; x += stride) {
      const int64_t i = (hq0 + g) * p.nb + a + x;
      p.blk_max[i] = NEG_INF;
      p.blk_sum[i] = 0.f;
    }
}

// A wavefront's items of 64 steps, one per lane: block (-1: none of the cache's), page (0 of a contiguous cache; -1:
// nothing to read, an empty block), scales.
struct Items {
  int blk, pg;
  float ks, vs;
};

// Workgroups per CU that the registers are to allow: a ragged batch's hide each other's starts and ends (48 sequences of
// up to 16384 tokens at 4 a CU, two of them running at a time 96.9 us, three 89.1). 16 heads of 128 dims would spill.
template <int D, int GP>
constexpr int WG8 = D == 64 ? 4 : GP == 16 ? 2 : 3;

template <int D, int GP, bool I8, bool STATS, bool RAG>
__global__ void __launch_bounds__(NT, (WG8<D, GP>)) decode8_kernel(const Attn8P p) {
  constexpr int KC = Lay8<D>::KC, KS = Lay8<D>::KS, VN = Lay8<D>::VN, VD = Lay8<D>::VD;
  __shared__ __attribute__((aligned(16))) Merge8<D, GP> sL;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / WAVE), lane = tid % WAVE;
  const int j4 = lane >> 4, c16 = lane & 15;
  const bool masked = p.block_idx != nullptr, paged = p.block_table != nullptr;
  const int G = p.G;

  // ---- this workgroup's work, as decode_body finds it: list positions / blocks [i0, i0 + n) of the n_items of (b, h)
  int split, h, b, n_items, i0, n, Tb = p.T, nbb = p.nb;
  bool whole = p.num_splits == 1;
  if constexpr (!RAG) {
    work_coords(blockIdx.x, p.num_splits, p.Hkv, p.B, split, h, b);
    n_items = masked ? min(max(p.block_cnt[b * p.Hkv + h], 0), p.max_blocks) : p.nb;
    const int per = (n_items + p.num_splits - 1) / p.num_splits;
    i0 = min(n_items, split * per);
    n = min(n_items, i0 + per) - i0;
  } else {
    const int W = p.num_splits + p.B;
    const bool global = masked && p.list_partition != 0;
    const int it = global ? static_cast<int>(blockIdx.x) : xcd_remap(blockIdx.x, W * p.Hkv);
    int chunk, C;
    if (global) {
      C = global_lookup(p, it, b, h, chunk, n_items);
    } else {
      h = it / W;
      C = ragged_lookup(p, h, it % W, masked, b, chunk, n_items);
    }
    {  // (sequence, KV head)s with nothing to read: no partials, statistics written by one workgroup per KV head
      const int eh = global ? (it < p.Hkv ? it : -1) : (it % W == 0 ? h : -1);
      if (eh >= 0) {
        for (int b0 = wave * WAVE; b0 < p.B; b0 += NT) {
          const int bb = b0 + lane;
          uint64_t none = __ballot(bb < p.B && ragged_items(p, bb, eh, masked) == 0);
          while (none != 0) {
            const int be = b0 + __builtin_ctzll(none);
            none &= none - 1;
            if (lane == 0) p.counts[be * p.Hkv + eh] = 0;
            if constexpr (STATS) empty_stats(p, static_cast<int64_t>(be) * p.Hq + static_cast<int64_t>(eh) * G, 0, p.nb, lane, WAVE);
          }
        }
      }
    }
    if (b < 0) return;
    split = chunk;
    // (a list of one chunk is finished here, and the merge has nothing to do: 64 sequences of up to 4096 tokens 53.5 us,
    // 50.2 so)
    whole = n_items <= C;
    if (chunk == 0 && tid == 0) p.counts[b * p.Hkv + h] = (n_items + C - 1) / C;
    if ((global && (G > 4 || grid_queued(p))) || p.B == 1) {
      i0 = chunk * C;
      n = min(n_items, i0 + C) - i0;
    } else {
      const int k = max(1, (n_items + C - 1) / C);
      i0 = chunk * n_items / k;
      n = (chunk + 1) * n_items / k - i0;
    }
    Tb = seq_len(p, b);
    nbb = (Tb + BLK - 1) / BLK;
  }
  // scalar registers for the addressing that follows
  split = __builtin_amdgcn_readfirstlane(split), h = __builtin_amdgcn_readfirstlane(h), b = __builtin_amdgcn_readfirstlane(b);
  n_items = __builtin_amdgcn_readfirstlane(n_items), i0 = __builtin_amdgcn_readfirstlane(i0), n = __builtin_amdgcn_readfirstlane(n);
  Tb = __builtin_amdgcn_readfirstlane(Tb), nbb = __builtin_amdgcn_readfirstlane(nbb);
  const int64_t bh = static_cast<int64_t>(b) * p.Hkv + h, hq0 = bh * G;
  const int* list = masked ? p.block_idx + bh * p.max_blocks : nullptr;
  const int* table = paged ? p.block_table + static_cast<int64_t>(b) * p.bt_stride : nullptr;
  const int nw = n > wave ? (n - wave + NWAVE - 1) / NWAVE : 0;
  const int rot = item_rotation(p, h, split + (RAG && p.B > 1 ? n_items : 0), nw);

  // ---- items of steps k0 .. k0 + 63, in three stages
  auto item_block = [&](Items& x, int k0) {
    const int k = k0 + lane;
    x.blk = -1;
    if (k < nw) {
      const int pos = i0 + wave + NWAVE * rotated(k, rot, nw);
      x.blk = masked ? list[pos] : pos;
    }
  };
  auto item_page = [&](Items& x) {
    if (x.blk < 0 || x.blk >= p.nb) x.blk = -1;
    x.pg = x.blk >= 0 && x.blk < nbb ? 0 : -1;
    if (paged && x.pg == 0) x.pg = table[x.blk];
  };
  auto item_scales = [&](Items& x) {
    if (paged && (x.pg < 0 || x.pg >= p.num_pages)) x.pg = -1;
    x.ks = x.vs = 0.f;
    if (x.pg >= 0) {
      const int64_t i = paged ? x.pg : b;
      const int e = paged ? 0 : x.blk;
      x.ks = p.k_scale[i * p.ks_sb + h * p.ks_sh + e];
      x.vs = p.v_scale[i * p.vs_sb + h * p.vs_sh + e];
    }
  };
  const uint32_t k_st = static_cast<uint32_t>(p.k_st), v_st = static_cast<uint32_t>(p.v_st);
  const uint32_t koff = c16 * k_st + 16 * j4;
  const uint32_t voff = D == 128 ? 4 * j4 * v_st + 8 * c16 : (4 * j4 + (c16 >> 3)) * v_st + 8 * (c16 & 7);
  const bool up = (lane & 8) != 0;
  // up to 8 heads: this lane's operand row takes the weights' high parts (0) or, negative, their low ones (-1)
  const float part = (c16 / GP) % 2 == 1 ? -1.f : 0.f;
  const char* kb = reinterpret_cast<const char*>(p.k) + h * p.k_sh;
  const char* vb = reinterpret_cast<const char*>(p.v) + h * p.v_sh;
  // (through readfirstlane: left to itself the compiler added the offset up in vector registers and wrapped every load in
  // a loop over the resource's values)
  auto block_res = [&](const char* base, int64_t sb, uint32_t st, int blk, int pg) {
    const int rows = pg >= 0 ? min(BLK, Tb - blk * BLK) : 0;
    const int64_t off = paged ? max(pg, 0) * sb : b * sb + static_cast<int64_t>(max(blk, 0)) * BLK * st;
    const uint64_t at = reinterpret_cast<uint64_t>(base) + off;
    const uint64_t lo = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(at)));
    const uint64_t hi = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(at >> 32)));
    return make_rsrc(reinterpret_cast<const void*>(hi << 32 | lo), rows > 0 ? (rows - 1) * st + D : 0u);
  };

  __shared__ int2 sGap[STATS ? NT : 1];  // masked statistics: the list entries around a lane's gap
  int2 gap = make_int2(-1, 0);
  if constexpr (STATS) {
    const int t = wave + NWAVE * lane;
    if (masked && t < n) {
      gap.y = list[i0 + t];
      if (i0 + t > 0) gap.x = list[i0 + t - 1];
    }
  }
  // ---- the first block and q: nothing is waited for before the first block's loads but its page
  Items cur, nxt;
  item_block(cur, 0);
  item_page(cur);
  item_scales(cur);
  nxt = cur;
  u32x4 qr[KS];
  const int qg = c16 % GP;
  const uint16_t* qp = p.q + b * p.q_sb + (static_cast<int64_t>(h) * G + min(qg, G - 1)) * p.q_sh + 16 * j4;
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) qr[ks] = ld16(qp + 64 * (ks / 2) + 8 * (ks % 2));
  u32x4 kr[4][KC];
  u32x2 vr[VN];
  int blk = __builtin_amdgcn_readlane(cur.blk, 0), pg = nw > 0 ? __builtin_amdgcn_readlane(cur.pg, 0) : -1;
  __builtin_amdgcn_sched_barrier(0);
  load_k8<D>(kr, block_res(kb, p.k_sb, k_st, blk, pg), koff, k_st);
  __builtin_amdgcn_sched_barrier(0);
  load_v8<D>(vr, block_res(vb, p.v_sb, v_st, blk, pg), voff, v_st);
  __builtin_amdgcn_sched_barrier(0);

  // ---- q in the codes' type, and the factor that takes its power of two out again
  Q8<D, GP, I8> qb;
  float qf;
  {
    float amax = 0.f, bad = 0.f;  // bad: NaN where q has an infinity or NaN
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      if (qg >= G) qr[ks] = u32x4{0u, 0u, 0u, 0u};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x = bf_lo(qr[ks][e]), y = bf_hi(qr[ks][e]);
        amax = fmaxf(amax, fmaxf(fabsf(x), fabsf(y)));
        bad = fmaf(x, 0.f, fmaf(y, 0.f, bad));
      }
    }
    amax = swap_max(amax);
    bad = swap_sum(bad);
    constexpr int TOP = I8 ? 29 : 14;                               // 2^TOP <= q's largest value < 2^(TOP + 1)
    const int ex = min(max(static_cast<int>(__float_as_uint(amax) >> 23) - 127, TOP - 126), 127);
    qf = p.scale_log2 * __uint_as_float(static_cast<uint32_t>(127 - TOP + ex) << 23) + bad;
    make_q8<D, GP, I8>(qb, qr, __uint_as_float(static_cast<uint32_t>(127 + TOP - ex) << 23), lane);
  }

  if constexpr (STATS) sGap[tid] = gap;  // (registers are short in the loop)
  const uint32_t nb4 = 4u * static_cast<uint32_t>(p.nb);
  const rsrc_t rs_max = make_rsrc(STATS ? p.blk_max + hq0 * p.nb : nullptr, STATS ? G * nb4 : 0);
  const rsrc_t rs_sum = make_rsrc(STATS ? p.blk_sum + hq0 * p.nb : nullptr, STATS ? G * nb4 : 0);
  constexpr uint32_t OOB = 0x80000000u;
  const uint32_t v_stat = c16 < G && j4 == 0 ? c16 * nb4 : OOB;

  // running (m, l) of this lane's head c16 % GP, its accumulators' reference ar + ax: a block's maximum and the exponent of
  // its vs (apart, since in one float a large maximum takes the exponent's bits)
  float mr = NEG_INF, lr = 0.f, ar = NEG_INF, ax = 0.f;
  f32x4_t acc[VD];
#pragma unroll
  for (int j = 0; j < VD; ++j) acc[j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  if (nw > 0) {
    for (int k = 0; k < nw; ++k) {
      // the next 64 steps' items, stage by stage
      const int ph = k & 63;
      const float ks = lane_value(cur.ks, ph), vs = lane_value(cur.vs, ph);
      if (k - ph + 64 < nw) {
        if (ph == 0) item_block(nxt, k + 64);
        if (ph == 16) item_page(nxt);
        if (ph == 32) item_scales(nxt);
        if (ph == 63) cur = nxt;
      }
      const int kn = (k + 1) & 63;
      int blk_n = -1, pg_n = -1;
      if (k + 1 < nw) {
        blk_n = __builtin_amdgcn_readlane(cur.blk, kn);
        pg_n = __builtin_amdgcn_readlane(cur.pg, kn);
      }
      const rsrc_t rk_n = block_res(kb, p.k_sb, k_st, blk_n, pg_n), rv_n = block_res(vb, p.v_sb, v_st, blk_n, pg_n);

      // scores of this block, s[nt][i] of head c16 % GP, token 16 nt + 4 j4 + i: in log2 units times 1 / f
      float s[4][4], e[4][4];
      float f = qf * ks;
      qk8<D, GP, I8>(s, kr, qb, lane);
      if ((__float_as_int(ks) ^ __float_as_int(p.scale_log2)) < 0) {  // uniform: a negative scale, f made positive
        f = -f;
#pragma unroll
        for (int t = 0; t < 16; ++t) s[t / 4][t % 4] = -s[t / 4][t % 4];
      }
      const int t0 = blk * BLK, lim = pg >= 0 ? Tb : -BLK;
      if (t0 + BLK > lim) {  // uniform: the block that the sequence's end cuts, or an empty one
#pragma unroll
        for (int nt = 0; nt < 4; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[nt][i] = t0 + mf_tok(nt, i, j4) >= lim ? NEG_INF : s[nt][i] * f;
        f = 1.f;
      }
      __builtin_amdgcn_sched_barrier(0);
      load_k8<D>(kr, rk_n, koff, k_st);
      __builtin_amdgcn_sched_barrier(0);

      const float mt = block_max_mf(s) * f;  // f >= 0
      const float mtu = mt == NEG_INF ? 0.f : mt;
      // (scores so large that mt's rounding would show, or overflow, in s f - mt: rounded alike instead, so that the largest
      // weight is 1 whatever the scores are)
      if (__ballot(fabsf(mtu) > 0x1p17f) != 0) {
#pragma unroll
        for (int t = 0; t < 16; ++t) s[t / 4][t % 4] *= f;
        f = 1.f;
      }
      float r4[4];
#pragma unroll
      for (int nt = 0; nt < 4; ++nt) {
#pragma unroll
        for (int i = 0; i < 4; ++i) e[nt][i] = fexp2(fmaf(s[nt][i], f, -mtu));
        r4[nt] = (e[nt][0] + e[nt][1]) + (e[nt][2] + e[nt][3]);
      }
      const float st = swap_sum((r4[0] + r4[1]) + (r4[2] + r4[3]));
      const float m_new = fmaxf(mr, mt);
      const float mu = m_new == NEG_INF ? 0.f : m_new;
      const float cf = mt == NEG_INF ? 0.f : fexp2(mt - mu);
      lr = lr * fexp2(mr - mu) + st * cf;
      mr = m_new;
      // the accumulators' reference: mt + log2 |vs| (its whole part) of the largest block so far, left where it is for as
      // long as a block passes it by at most 2^7
      const float ev = static_cast<float>(max(static_cast<int>(__float_as_uint(vs) >> 23 & 0xffu) - 127, -100));
      const float past = (mt - ar) + (ev - ax);  // (NaN, which passes nothing, where nothing came yet)
      if (__ballot(past > 7.f) != 0) {
        const bool on = past > 0.f;
        rescale8<D, GP>(acc, on ? fexp2(-past) : 1.f, lane);
        ar = on ? mt : ar;
        ax = on ? ev : ax;
      }
      const float fv = vs * fexp2((mt - (ar == NEG_INF ? 0.f : ar)) - ax) * 0x1p7f;  // below 2^15
      if constexpr (STATS) {
        const uint32_t blk4 = 4u * static_cast<uint32_t>(max(blk, 0));
        const uint32_t at = blk >= 0 ? v_stat : OOB;
        bstore_f32(mt * LN2, rs_max, at, blk4);
        bstore_f32(st, rs_sum, at, blk4);
      }

      // the weights as operands: row c of a product is head c % GP, up to 8 heads the high parts in rows below GP and the
      // low ones in the GP rows after them (the rows from 2 GP on are not read)
      u32x4 w8[2], wl[2];
#pragma unroll
      for (int q = 0; q < 2; ++q)
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const float x = e[2 * q + u / 2][2 * (u % 2)] * fv, y = e[2 * q + u / 2][2 * (u % 2) + 1] * fv;
          const f16x2_t hi = __builtin_bit_cast(f16x2_t, pack_h(x, y));
          if constexpr (GP == 16) {
            w8[q][u] = __builtin_bit_cast(uint32_t, hi);
            wl[q][u] = mix_h(x, y, 1.f, -hi);
          } else {  // high rows hi - 0 x, low ones hi - x
            w8[q][u] = mix_h(x, y, part, hi);
          }
        }
#pragma unroll
      for (int d = 0; d < VD / 4; ++d) {
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          u32x4 w[4];  // four dims, tokens in pairs
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            uint32_t a, c;
            v_pair8<D>(vr, 2 * q + u / 2, 2 * (u % 2), d, up, a, c);
            const u32x2 w01 = widen4<I8>(__builtin_amdgcn_perm(c, a, 0x05010400u));
            const u32x2 w23 = widen4<I8>(__builtin_amdgcn_perm(c, a, 0x07030602u));
            w[0][u] = w01.x, w[1][u] = w01.y, w[2][u] = w23.x, w[3][u] = w23.y;
          }
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            acc[4 * d + x] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, w8[q]),
                                                                    __builtin_bit_cast(f16x8_t, w[x]), acc[4 * d + x], 0, 0, 0);
            if constexpr (GP == 16)
              acc[4 * d + x] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                  __builtin_bit_cast(f16x8_t, wl[q]), __builtin_bit_cast(f16x8_t, w[x]), acc[4 * d + x], 0, 0, 0);
          }
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      load_v8<D>(vr, rv_n, voff, v_st);
      blk = blk_n;
      pg = pg_n;
    }
  }

  // ---- the wavefront's state into LDS (row 4 j4 + i of the products is part and head of Merge8), then the merge
  {
    constexpr int NP = Merge8<D, GP>::NP;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = 4 * j4 + i;
      if (row < NP * GP && row % GP < G) {
        float* a = sL.acc + (wave * NP * GP + row) * D + mf_vdim<D>(c16);
#pragma unroll
        for (int j = 0; j < VD; j += 4)
          *reinterpret_cast<float4*>(a + j) = make_float4(acc[j][i], acc[j + 1][i], acc[j + 2][i], acc[j + 3][i]);
      }
    }
    if (lane < G) {
      sL.m[lane][wave] = mr, sL.l[lane][wave] = lr, sL.r[lane][wave] = ar, sL.x[lane][wave] = ax;
    }
  }
  finish8<D, GP>(p, b, h, split, whole, sL);

  if constexpr (STATS) {
    // the blocks that the list skips, and those past the sequence's end: the gap before each of this split's entries
    // and, on the split of the last one, what follows it
    if (masked) {
      if (n_items == 0 && split == 0) empty_stats(p, hq0, 0, p.nb, tid, NT);
      for (int j = 0; wave + NWAVE * j < n; ++j) {  // uniform over the wavefront
        int before, now;
        if (j < WAVE) {
          const int2 g = sGap[wave * WAVE + j];  // this wavefront's own
          before = __builtin_amdgcn_readfirstlane(g.x);
          now = __builtin_amdgcn_readfirstlane(g.y);
        } else {
          const int k = i0 + wave + NWAVE * j;
          now = __builtin_amdgcn_readfirstlane(list[k]);
          before = __builtin_amdgcn_readfirstlane(list[k - 1]);
        }
        const int a = min(max(before, -1), p.nb - 1) + 1, len = min(max(now, 0), p.nb) - a;
        empty_stats(p, hq0, a, len, lane, WAVE);
      }
    }
    if (n > 0 && i0 + n == n_items) {
      const int last = masked ? min(max(list[n_items - 1], -1), p.nb - 1) : nbb - 1;
      empty_stats(p, hq0, last + 1, p.nb - last - 1, tid, NT);
    }
  }
}

// Split merge: workgroup (b, query head), a thread four dims of a class of splits. A wavefront takes the partials'
// maxima and sums a split a lane, so the weights 2^(m_s - M) are in LDS after one barrier, under which the accumulators
// are already on their way. Its workgroup takes the place (xcd_remap) of its KV head's splits, whose L2 holds the partials.
// A ragged list's partials are counted by the pass; one of a single chunk has its result already. (The merge of the bf16
// passes, four workgroups a head that count chunks anew, took 10.5 us for 64 sequences of up to 4096 tokens, 8.4 for 16 of
// up to 32000 of 28 heads; this one 4.6 and 4.8, of which a launch alone is 3.3. Of a dim a thread: 4.7 and 4.8, and one
// sequence of 32768 tokens in 32 splits 18.1 us a call for 17.2 with four.)
template <int D>
__global__ void __launch_bounds__(NT) combine8_kernel(const Attn8P p) {
  constexpr int NC = NT * 4 / D, U = 4;
  __shared__ float sW[MAX_SPLITS];
  __shared__ __attribute__((aligned(16))) float sA[NC * D];
  const int tid = threadIdx.x, lane = tid % WAVE, cls = tid / (D / 4), d = tid % (D / 4) * 4;
  const int hq = xcd_remap(blockIdx.x, p.B * p.Hq), S = p.num_splits;
  const int n = p.seq_lens == nullptr ? S : __builtin_amdgcn_readfirstlane(p.counts[hq / p.Hq * p.Hkv + hq % p.Hq / p.G]);
  if (p.seq_lens != nullptr && n == 1) return;
  const float* ml = p.part_ml + static_cast<int64_t>(hq) * S * 2;
  const float* acc = p.part_acc + static_cast<int64_t>(hq) * S * D + d;
  auto load = [&](int s) {
    return s < n ? *reinterpret_cast<const f32x4_t*>(acc + s * D) : f32x4_t{0.f, 0.f, 0.f, 0.f};
  };
  float ms[MAX_SPLITS / WAVE], ls[MAX_SPLITS / WAVE];
#pragma unroll
  for (int r = 0; r < MAX_SPLITS / WAVE; ++r) {
    const int s = lane + WAVE * r;
    ms[r] = NEG_INF, ls[r] = 0.f;
    if (s < n) {
      const float2 t = *reinterpret_cast<const float2*>(ml + 2 * s);
      ms[r] = t.x, ls[r] = t.y;
    }
  }
  f32x4_t x[U];
#pragma unroll
  for (int u = 0; u < U; ++u) x[u] = load(cls + NC * u);
  float M = NEG_INF, L = 0.f;
#pragma unroll
  for (int r = 0; r < MAX_SPLITS / WAVE; ++r) M = fmaxf(M, ms[r]);
  M = wave_max(M);
  const float mu = M == NEG_INF ? 0.f : M;
#pragma unroll
  for (int r = 0; r < MAX_SPLITS / WAVE; ++r) {
    // (an empty partial, l = 0, may hold anything in its accumulators and counts for nothing; a NaN counts)
    const float w = ls[r] == 0.f ? 0.f : fexp2(ms[r] - mu);
    L += ls[r] * w;
    if (tid < WAVE && lane + WAVE * r < n) sW[lane + WAVE * r] = ls[r] == 0.f ? -1.f : w;
  }
  L = wave_sum(L);
  __syncthreads();
  f32x4_t A = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = cls; s0 < n; s0 += NC * U) {
    f32x4_t y[U];  // the next round's, asked for before this one's are added
#pragma unroll
    for (int u = 0; u < U; ++u) y[u] = load(s0 + NC * (U + u));
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float w = s0 + NC * u < n ? sW[s0 + NC * u] : -1.f;
      if (w != -1.f) A += x[u] * w;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) x[u] = y[u];
  }
  *reinterpret_cast<f32x4_t*>(sA + cls * D + d) = A;
  __syncthreads();
  if (tid < D) {
    float a = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c) a += sA[c * D + tid];
    const float o = L == 0.f ? 0.f : a / L;
    const int64_t at = static_cast<int64_t>(hq) * D + tid;
    p.out[at] = f2bf(o);
    if (p.out_f32) p.out_f32[at] = o;
    if (p.lse && tid == 0) p.lse[hq] = L == 0.f ? NEG_INF : (M + flog2(L)) * LN2;
  }
}

template <int D, int GP, bool I8, bool STATS>
void launch8_r(const Attn8P& p, hipStream_t s) {
  if (p.seq_lens != nullptr)
    hipLaunchKernelGGL((decode8_kernel<D, GP, I8, STATS, true>), attn_grid(p), dim3(NT), 0, s, p);
  else
    hipLaunchKernelGGL((decode8_kernel<D, GP, I8, STATS, false>), attn_grid(p), dim3(NT), 0, s, p);
}

template <int D, int GP, bool I8>
void launch8(const Attn8P& p, bool stats, hipStream_t s) {
  stats ? launch8_r<D, GP, I8, true>(p, s) : launch8_r<D, GP, I8, false>(p, s);
}

template <int D>
void launch8_d(const Attn8P& p, bool i8, bool stats, hipStream_t s) {
  if (p.G <= 4)
    i8 ? launch8<D, 4, true>(p, stats, s) : launch8<D, 4, false>(p, stats, s);
  else if (p.G <= 8)
    i8 ? launch8<D, 8, true>(p, stats, s) : launch8<D, 8, false>(p, stats, s);
  else
    i8 ? launch8<D, 16, true>(p, stats, s) : launch8<D, 16, false>(p, stats, s);
}

}  // namespace

hipError_t launch_decode8(const Attn8P& p, int D, bool i8, bool stats, hipStream_t s) {
  D == 128 ? launch8_d<128>(p, i8, stats, s) : launch8_d<64>(p, i8, stats, s);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.num_splits == 1) return e;
  if (D == 128)
    hipLaunchKernelGGL(combine8_kernel<128>, dim3(p.B * p.Hq), dim3(NT), 0, s, p);
  else
    hipLaunchKernelGGL(combine8_kernel<64>, dim3(p.B * p.Hq), dim3(NT), 0, s, p);
  return hipGetLastError();
}

}  // namespace kvs
