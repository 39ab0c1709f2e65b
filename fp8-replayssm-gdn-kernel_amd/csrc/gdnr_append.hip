// gdnr_append.hip -- the entry of a full-attention layer, in one pass over its
// q, k and v rows: per head of q and k
//   x <- w x / sqrt(mean x^2 + eps)          (with a weight)
//   x0, x1 <- x0 c - x1 s, x1 c + x0 s       on the first `rotary` elements,
// where a pair is (i, i + rotary / 2), or (2i, 2i + 1) interleaved, and c, s
// come from the table's row of the token's position; q goes to q_out, k and v
// to their slot of the paged cache (v as it is). f32 arithmetic, rounded once.
//
// Bound by its bytes: every row is read once and written once. A lane owns 8
// elements of a head (16 bytes), so a head takes D / 8 lanes and a wave
// instruction moves 512 / D heads; a wave walks the heads of one token and
// keeps its table row and the weights in registers. The pair's other element
// sits rotary / 16 lanes away (a lane exchange of the raw bits) or in the same
// lane (interleaved).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "gdnr_device.h"
#include "gdnr_internal.h"

namespace gdnr {
namespace {

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

// sum over the aligned group of LANES lanes (8, 16 or 32), in every lane of it
template <int LANES>
__device__ __forceinline__ float group_sum(float x) {
  x = sum8(x);
  if constexpr (LANES >= 16) x += dpp_f<kDppMirror>(x);
  if constexpr (LANES == 32) x += __shfl_xor(x, 16);
  return x;
}

template <class Act>
__device__ __forceinline__ void unpack8(u32x4_t w, float* f) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 p = Act::from_pair(w[i]);
    f[2 * i] = p.x, f[2 * i + 1] = p.y;
  }
}
template <class Act>
__device__ __forceinline__ u32x4_t pack8(const float* f) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) Act::st2(&w[i], f[2 * i], f[2 * i + 1]);
  return u32x4_t{w[0], w[1], w[2], w[3]};
}

template <class Act, int D>
__global__ __launch_bounds__(256) void append_kernel(const AppendArgs a) {
  constexpr int LPH = D / 8;       // lanes per head
  constexpr int HPW = 64 / LPH;    // heads a wave instruction moves
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t unit = (int64_t)blockIdx.x * 4 + wave;
  const int t = (int)(unit / a.splits), part = (int)(unit - (int64_t)t * a.splits);
  if (t >= a.T) return;  // wave-uniform
  const int cl = lane & (LPH - 1), sub = lane / LPH;
  const int heads = a.HQ + 2 * a.HKV;
  const int pos = min(max(__builtin_amdgcn_readfirstlane(a.position[t * a.po_s]), 0), a.positions - 1);
  const int slot = __builtin_amdgcn_readfirstlane(a.slot[t * a.sl_s]);
  const bool kept = slot >= 0 && slot < a.slots;  // any other slot appends nothing
  const int page = kept ? slot / a.page : 0, at = kept ? slot - page * a.page : 0;

  // cosines and signed sines of this lane's elements; a lane past the rotary
  // part turns by nothing
  const int half = a.rotary / 2, e0 = 8 * cl;
  const bool turned = e0 < a.rotary;
  float c[8], s[8];
  if (turned) {
    const float* row = a.table + pos * a.tb_p;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int i = a.interleaved ? (e0 + e) >> 1 : (e0 < half ? e0 + e : e0 + e - half);
      c[e] = row[i];
      const float sine = row[half + i];
      s[e] = (a.interleaved ? !(e & 1) : e0 < half) ? -sine : sine;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) c[e] = 1.f, s[e] = 0.f;
  }
  const int partner = a.interleaved || !turned ? lane : (e0 < half ? lane + half / 8 : lane - half / 8);
  const int ep = 8 * (partner & (LPH - 1));

  for (int head = part * HPW; head < heads; head += a.splits * HPW) {
    const int hh = head + sub;
    const bool on = hh < heads, is_q = hh < a.HQ, is_k = !is_q && hh < a.HQ + a.HKV;
    const uint8_t* src = !on ? nullptr
                         : is_q ? (const uint8_t*)a.q + (t * a.q_t + hh * a.q_h) * 2
                         : is_k ? (const uint8_t*)a.k + (t * a.k_t + (hh - a.HQ) * a.k_h) * 2
                                : (const uint8_t*)a.v + (t * a.v_t + (hh - a.HQ - a.HKV) * a.v_h) * 2;
    u32x4_t w = {0, 0, 0, 0};
    if (on) w = *(const u32x4_t*)(src + 16 * cl);
    if (head < a.HQ + a.HKV) {  // wave-uniform: some head of these is q or k
      u32x4_t wp;
#pragma unroll
      for (int i = 0; i < 4; ++i) wp[i] = (uint32_t)__shfl((int)w[i], partner);
      float x[8], xp[8], y[8], sq = 0.f;
      unpack8<Act>(w, x);
      unpack8<Act>(wp, xp);
      const float* weight = is_q ? a.q_weight : a.k_weight;
      const bool norm = weight != nullptr && (is_q || is_k);
#pragma unroll
      for (int e = 0; e < 8; ++e) sq = fmaf(x[e], x[e], sq);
      const float r = 1.f / sqrtf(group_sum<LPH>(sq) * (1.f / D) + a.eps);
      if (norm) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] *= r * weight[e0 + e], xp[e] *= r * weight[ep + e];
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float other = a.interleaved ? x[e ^ 1] : xp[e];
        y[e] = turned ? fmaf(other, s[e], x[e] * c[e]) : x[e];
      }
      if (is_q || is_k) w = pack8<Act>(y);
    }
    if (is_q) {
      *(u32x4_t*)((uint8_t*)a.q_out + (t * a.qo_t + hh * a.qo_h) * 2 + 16 * cl) = w;
    } else if (on && kept) {
      uint8_t* dst = is_k ? (uint8_t*)a.k_cache + (page * a.kc_p + at * a.kc_t + (hh - a.HQ) * a.kc_h) * 2
                          : (uint8_t*)a.v_cache + (page * a.vc_p + at * a.vc_t + (hh - a.HQ - a.HKV) * a.vc_h) * 2;
      *(u32x4_t*)(dst + 16 * cl) = w;
    }
  }
}

template <class Act, int D>
int launch_append_dim(AppendArgs a, hipStream_t s) {
  // waves for every compute unit twice over, while a wave still has heads
  const int heads = a.HQ + 2 * a.HKV, most = (heads + 512 / D - 1) / (512 / D);
  const int want = (int)((8 * (int64_t)device_cus() + a.T - 1) / a.T);
  a.splits = want < 1 ? 1 : want < most ? want : most;
  const int64_t units = (int64_t)a.T * a.splits;
  hipLaunchKernelGGL((append_kernel<Act, D>), dim3((uint32_t)((units + 3) / 4)), dim3(256), 0, s, a);
  return (int)hipGetLastError();
}

template <class Act>
int launch_append_act(const AppendArgs& a, hipStream_t s) {
  if (a.D == 64) return launch_append_dim<Act, 64>(a, s);
  if (a.D == 128) return launch_append_dim<Act, 128>(a, s);
  return launch_append_dim<Act, 256>(a, s);
}

}  // namespace

int launch_append(const AppendArgs& a, int act_dt, void* stream) {
  return act_dt == DT_BF16 ? launch_append_act<ActBF16>(a, (hipStream_t)stream) : launch_append_act<ActF16>(a, (hipStream_t)stream);
}

}  // namespace gdnr
