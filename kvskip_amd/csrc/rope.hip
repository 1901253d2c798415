// Norms of queries and keys for each head, and their rotation, in one pass over both.
//
//   y = x / sqrt(mean x^2 + eps) w;  pairs (a, b) of y: (a cos t - b sin t, b cos t + a sin t),  t = position * frequency
//
// Bound by memory: every element is read and written once. A lane holds four pairs of a head (eight elements, as two pieces
// of 8 bytes: halves of the head, or neighbours), so a rotation needs no other lane, and a head's sum of squares is three
// to five lane swaps over its 8, 16 or 32 lanes. Sines and cosines belong to a token: its workgroup makes them once,
// in LDS, for all of its heads. Angles of far positions need more than 24 bits (131071 * 1.0 in fp32 is off by 0.004):
// position * frequency / 2 pi is reduced to a turn in 64 bits, and the sine of what is left taken in 32.
#include "common.hpp"
#include "attend.hpp"

namespace kvs {
namespace {

constexpr int RT = 256;     // threads
constexpr int MAX_TT = 8;   // tokens of a workgroup

// Elements of a lane's unit u: two runs of four.
__device__ __forceinline__ void unit_at(const kvskip_rope_args& p, int u, int& a, int& b) {
  if (p.pairs != 0 || 8 * u >= p.rot)
    a = 8 * u, b = 8 * u + 4;
  else
    a = 4 * u, b = p.rot / 2 + 4 * u;
}

__device__ __forceinline__ void load_weight(float (&w)[8], const void* src, bool f32, int a, int b) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int d = (e < 4 ? a : b) + e % 4;
    w[e] = src == nullptr ? 1.f
           : f32          ? static_cast<const float*>(src)[d]
                          : __uint_as_float(static_cast<uint32_t>(static_cast<const uint16_t*>(src)[d]) << 16);
  }
}

__device__ __forceinline__ uint32_t pack_bf(float a, float b) {
  typedef float f32x2_t __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_t{a, b}), bf16x2_t));
}

template <int LU>
__device__ __forceinline__ float unit_sum(float v) {
  v = sum8(v);
  if constexpr (LU >= 16) v += dpp<DPP_ROR8>(v);
  if constexpr (LU >= 32) v += xshfl(v, 16);
  return v;
}

// LU lanes a head (at least D / 8), TT tokens a workgroup.
template <int LU, int TT>
__global__ void __launch_bounds__(RT) norm_rope_kernel(const kvskip_rope_args p) {
  __shared__ __attribute__((aligned(16))) float2 sCS[TT * 128];
  const int tid = threadIdx.x, half = p.rot / 2, H = p.Hq + p.Hkv;
  const int n0 = blockIdx.x * TT, nt = min(TT, p.rows - n0);
  for (int e = tid; e < nt * half; e += RT) {
    const int t = e / half, i = e - t * half;
    int axis = 0, end = p.sections[0];
    while (axis + 1 < p.axes && i >= end) end += p.sections[++axis];
    const double turns = static_cast<double>(p.positions[axis * p.pos_stride + n0 + t]) * static_cast<double>(p.inv_freq[i]) *
                         0.15915494309189533577;
    float s, c;
    sincospif(2.f * static_cast<float>(turns - rint(turns)), &s, &c);
    sCS[t * half + i] = make_float2(c * p.mscale, s * p.mscale);
  }
  const int u = tid % LU;
  const bool on = 8 * u < p.D, turned = 8 * u < p.rot;
  int a = 0, b = 4;
  if (on) unit_at(p, u, a, b);
  float wq[8], wk[8];
  load_weight(wq, p.q_weight, p.q_weight_f32 != 0, a, b);
  load_weight(wk, p.k_weight, p.k_weight_f32 != 0, a, b);
  __syncthreads();
  constexpr int SLOTS = RT / LU, NB = 4;
  const float inv_d = 1.f / static_cast<float>(p.D);
  for (int w0 = tid / LU; w0 < nt * H; w0 += SLOTS * NB) {
    u32x2 x[NB], y[NB];
    uint16_t* to[NB];
    int tok[NB];
    bool is_q[NB], live[NB];
#pragma unroll
    for (int g = 0; g < NB; ++g) {  // all loads, then the heads one by one
      const int w = w0 + SLOTS * g, wc = min(w, nt * H - 1), t = wc / H, hd = wc - t * H;
      live[g] = w < nt * H && on;
      tok[g] = t;
      is_q[g] = hd < p.Hq;
      const int64_t n = n0 + t;
      const uint16_t* from = is_q[g] ? static_cast<const uint16_t*>(p.q) + n * p.q_sn + hd * p.q_sh
                                     : static_cast<const uint16_t*>(p.k) + n * p.k_sn + (hd - p.Hq) * p.k_sh;
      to[g] = is_q[g] ? static_cast<uint16_t*>(p.q_out) + n * p.qo_sn + hd * p.qo_sh
                      : static_cast<uint16_t*>(p.k_out) + n * p.ko_sn + (hd - p.Hq) * p.ko_sh;
      x[g] = y[g] = u32x2{0u, 0u};
      if (live[g]) {
        x[g] = *reinterpret_cast<const u32x2*>(from + a);
        y[g] = *reinterpret_cast<const u32x2*>(from + b);
      }
    }
#pragma unroll
    for (int g = 0; g < NB; ++g) {
      float v[8] = {bf_lo(x[g].x), bf_hi(x[g].x), bf_lo(x[g].y), bf_hi(x[g].y),
                    bf_lo(y[g].x), bf_hi(y[g].x), bf_lo(y[g].y), bf_hi(y[g].y)};
      if ((is_q[g] ? p.q_weight : p.k_weight) != nullptr) {  // (a head's lanes alike)
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) s = fmaf(v[e], v[e], s);
        const float r = rsqrtf(unit_sum<LU>(s) * inv_d + p.eps);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = v[e] * r * (is_q[g] ? wq[e] : wk[e]);
      }
      if (turned) {
        const float2* cs = sCS + tok[g] * half + 4 * u;
        float o[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 z = cs[e];
          const float f = p.pairs != 0 ? v[2 * e] : v[e], h = p.pairs != 0 ? v[2 * e + 1] : v[e + 4];
          const float f1 = fmaf(f, z.x, -h * z.y), h1 = fmaf(h, z.x, f * z.y);
          o[e] = f1, o[e + 4] = h1;
        }
        if (p.pairs != 0) {
#pragma unroll
          for (int e = 0; e < 4; ++e) v[2 * e] = o[e], v[2 * e + 1] = o[e + 4];
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = o[e];
        }
      }
      if (live[g]) {
        *reinterpret_cast<u32x2*>(to[g] + a) = u32x2{pack_bf(v[0], v[1]), pack_bf(v[2], v[3])};
        *reinterpret_cast<u32x2*>(to[g] + b) = u32x2{pack_bf(v[4], v[5]), pack_bf(v[6], v[7])};
      }
    }
  }
}

template <int LU>
void launch_lu(const kvskip_rope_args& a, hipStream_t s) {
  // (eight tokens a workgroup as soon as every CU has one: fewer sines a token's head)
  if (a.rows >= 256 * MAX_TT)
    hipLaunchKernelGGL((norm_rope_kernel<LU, MAX_TT>), dim3((a.rows + MAX_TT - 1) / MAX_TT), dim3(RT), 0, s, a);
  else
    hipLaunchKernelGGL((norm_rope_kernel<LU, 1>), dim3(a.rows), dim3(RT), 0, s, a);
}

}  // namespace

hipError_t launch_norm_rope(const kvskip_rope_args& a, hipStream_t s) {
  if (a.D <= 64)
    launch_lu<8>(a, s);
  else if (a.D <= 128)
    launch_lu<16>(a, s);
  else
    launch_lu<32>(a, s);
  return hipGetLastError();
}

}  // namespace kvs
