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
// lane (interleaved). 8192 tokens of 32 + 2 x 8 heads of 128 take 47.4 us (4.3
// TB/s, 0.87 of a copy's rate), 14001 tokens of heads of 64, interleaved, 69.9 (as a
// copy); one token takes 3.4 us, its chain of loads.
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

// 4 N floats from p (4-byte aligned; 16 bytes an instruction)
typedef float f32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));
template <int N>
__device__ __forceinline__ void load_floats(const float* p, float* f) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const f32x4_a4 x = ((const f32x4_a4*)p)[i];
#pragma unroll
    for (int j = 0; j < 4; ++j) f[4 * i + j] = x[j];
  }
}

constexpr int kAhead = 4;  // groups of heads a wave asks for at once

template <class Act, int D, bool INTERLEAVED>
__global__ __launch_bounds__(256) void append_kernel(const AppendArgs a) {
  constexpr int LPH = D / 8;       // lanes per head
  constexpr int HPW = 64 / LPH;    // heads a wave instruction moves
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t unit = (int64_t)blockIdx.x * 4 + wave;
  const int t = (int)(unit / a.splits), part = (int)(unit - (int64_t)t * a.splits);
  if (t >= a.T) return;  // wave-uniform
  const int cl = lane & (LPH - 1), sub = lane / LPH;
  const int pos = min(max(__builtin_amdgcn_readfirstlane(a.position[t * a.po_s]), 0), a.positions - 1);
  const int slot = __builtin_amdgcn_readfirstlane(a.slot[t * a.sl_s]);
  const bool kept = slot >= 0 && slot < a.slots;  // any other slot appends nothing
  const int page = kept ? slot / a.page : 0, at = kept ? slot - page * a.page : 0;

  // this lane's elements, and its partner's that they turn with
  const int half = a.rotary / 2, e0 = 8 * cl;
  const bool turned = e0 < a.rotary, low = e0 < half;
  const int partner = INTERLEAVED || !turned ? lane : (low ? lane + half / 8 : lane - half / 8);
  const int ep = 8 * (partner & (LPH - 1));
  // its cosines and signed sines
  float c[8], s[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) c[e] = 1.f, s[e] = 0.f;
  if (turned) {
    const float* angles = a.table + pos * a.tb_p;
    if constexpr (INTERLEAVED) {
      float x[4], y[4];
      load_floats<1>(angles + e0 / 2, x);
      load_floats<1>(angles + half + e0 / 2, y);
#pragma unroll
      for (int e = 0; e < 8; ++e) c[e] = x[e >> 1], s[e] = (e & 1) ? y[e >> 1] : -y[e >> 1];
    } else {
      const float* own = angles + (low ? e0 : e0 - half);
      load_floats<2>(own, c);
      load_floats<2>(own + half, s);
      if (low) {
#pragma unroll
        for (int e = 0; e < 8; ++e) s[e] = -s[e];
      }
    }
  }

  const int q_groups = (a.HQ + HPW - 1) / HPW, kv_groups = (a.HKV + HPW - 1) / HPW;
  // one kind of heads: its rows in groups of HPW heads, group `first` and every
  // `splits`-th from there
  auto heads_of = [&](const void* from, int64_t from_t, int64_t from_h, void* to, int64_t to_row, int64_t to_h, int heads,
                      int first, const float* weight, bool rotate) {
    const int groups = (heads + HPW - 1) / HPW;
    if (first >= groups) return;
    const uint8_t* src = (const uint8_t*)from + (t * from_t + sub * from_h + e0) * 2;
    uint8_t* dst = (uint8_t*)to + (to_row + sub * to_h + e0) * 2;
    u32x4_t w[kAhead];
    auto ask = [&](int g0) {
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int g = g0 + u * a.splits;
        w[u] = u32x4_t{0, 0, 0, 0};
        if (g * HPW + sub < heads) w[u] = *(const u32x4_t*)(src + g * HPW * from_h * 2);
      }
    };
    ask(first);
    // y = r (x cw + x_partner sw): the weight, cosine and signed sine in one
    float cw[8], sw[8];
    if (rotate) {
      float own[8], other[8];
      if (weight) {
        load_floats<2>(weight + e0, own);
        load_floats<2>(weight + ep, other);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int o = INTERLEAVED ? e ^ 1 : e;
        cw[e] = weight ? own[e] * c[e] : c[e], sw[e] = weight ? other[o] * s[e] : s[e];
      }
    }
    for (int g0 = first; g0 < groups; g0 += kAhead * a.splits) {
      if (g0 != first) ask(g0);
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int g = g0 + u * a.splits;
        if (g >= groups) break;  // wave-uniform
        if (rotate) {
          float x[8], z[8], sq = 0.f, r = 1.f;
          unpack8<Act>(w[u], x);
          if constexpr (INTERLEAVED) {
#pragma unroll
            for (int e = 0; e < 8; ++e) z[e] = x[e ^ 1];
          } else {
            u32x4_t wp;
#pragma unroll
            for (int i = 0; i < 4; ++i) wp[i] = (uint32_t)__shfl((int)w[u][i], partner);
            unpack8<Act>(wp, z);
          }
          if (weight) {
#pragma unroll
            for (int e = 0; e < 8; ++e) sq = fmaf(x[e], x[e], sq);
            float eps = a.eps;
            if constexpr (std::is_same<Act, ActBF16>::value) {  // (f16's squares stay in range)
              if (__any(sq >= kLargeSquares)) {
                const float f = row_factor<LPH>(x);
                sq = 0.f, eps *= f * f;
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] *= f, z[e] *= f, sq = fmaf(x[e], x[e], sq);
              }
            }
            r = 1.f / sqrtf(group_sum<LPH>(sq) * (1.f / D) + eps);
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] *= cw[e];
          if (turned) {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = fmaf(z[e], sw[e], x[e]);
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] *= r;
          w[u] = pack8<Act>(x);
        }
        if (g * HPW + sub < heads) *(u32x4_t*)(dst + g * HPW * to_h * 2) = w[u];
      }
    }
  };
  heads_of(a.q, a.q_t, a.q_h, a.q_out, t * a.qo_t, a.qo_h, a.HQ, part, a.q_weight, true);
  if (!kept) return;
  // (the groups go round: the kinds' first ones fall to different waves)
  const int k_first = (part + a.splits - q_groups % a.splits) % a.splits;
  const int v_first = (k_first + a.splits - kv_groups % a.splits) % a.splits;
  heads_of(a.k, a.k_t, a.k_h, a.k_cache, page * a.kc_p + at * a.kc_t, a.kc_h, a.HKV, k_first, a.k_weight, true);
  heads_of(a.v, a.v_t, a.v_h, a.v_cache, page * a.vc_p + at * a.vc_t, a.vc_h, a.HKV, v_first, nullptr, false);
}

template <class Act, int D>
int launch_append_dim(AppendArgs a, hipStream_t s) {
  // waves for every compute unit twice over, while a wave still has heads
  constexpr int HPW = 512 / D;
  const int most = (a.HQ + HPW - 1) / HPW + 2 * ((a.HKV + HPW - 1) / HPW);
  const int want = (int)((8 * (int64_t)device_cus() + a.T - 1) / a.T);
  a.splits = want < 1 ? 1 : want < most ? want : most;
  const dim3 grid((uint32_t)(((int64_t)a.T * a.splits + 3) / 4));
  if (a.interleaved) hipLaunchKernelGGL((append_kernel<Act, D, true>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((append_kernel<Act, D, false>), grid, dim3(256), 0, s, a);
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
