// gdnr_prefill.hip -- the gated delta rule over packed sequences of any
// length, from the raw rows of the production contract: per sequence and
// value head, with the state S [V, K] of the sequence's slot,
//   q, k <- x / sqrt(sum x^2 + 1e-6), g = -exp(A_log) softplus_20(a + dt_bias),
//   beta = sigmoid(b);
//   S <- e^g S;  S <- S + beta (v - S k) k^T;  o = scale S q   for each token,
// the state left in its slot after the last one (the recurrence of
// prototype/gdn_replay_fp8_reference.py:137-163 on the inputs of
// prototype/gdn_replayssm_fp8_kernel.py:500-562).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "gdnr_device.h"
#include "gdnr_internal.h"

namespace gdnr {
namespace {

constexpr int K = kKeyDim;

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

// sum over the aligned 16-lane group, in every lane of it
__device__ __forceinline__ float sum16(float x) {
  x = sum8(x);
  return x + dpp_f<kDppMirror>(x);
}

// N consecutive elements at p (N * kBytes a multiple of 8, p aligned to it up
// to 16) as raw words, and their values
template <class Act, int N>
struct Raw {
  static constexpr int W = N * Act::kBytes / 4;
  uint32_t w[W];
  __device__ __forceinline__ void load(const void* p) {
    if constexpr (W % 4 == 0) {
#pragma unroll
      for (int i = 0; i < W / 4; ++i) {
        const u32x4_t x = ((const u32x4_t*)p)[i];
#pragma unroll
        for (int j = 0; j < 4; ++j) w[4 * i + j] = x[j];
      }
    } else {
      const uint2 x = *(const uint2*)p;
      w[0] = x.x, w[1] = x.y;
    }
  }
  __device__ __forceinline__ float operator[](int i) const {
    if constexpr (Act::kBytes == 4) return __uint_as_float(w[i]);
    else return Act::from_bits((i & 1) ? w[i / 2] >> 16 : w[i / 2]);
  }
};

// The tokens [begin, end) of sequence n, clamped to the rows there are.
__device__ __forceinline__ void sequence_rows(const PrefillArgs& a, int n, int& begin, int& end) {
  const int b = __builtin_amdgcn_readfirstlane(a.cu[n * a.cu_s]), e = __builtin_amdgcn_readfirstlane(a.cu[(n + 1) * a.cu_s]);
  begin = min(max(b, 0), a.T);
  end = min(max(e, begin), a.T);
}
// Its slot (out of range: the null slot) and whether it continues from it.
__device__ __forceinline__ int sequence_slot(const PrefillArgs& a, int n) {
  const int s = __builtin_amdgcn_readfirstlane(a.slot[n * a.sl_s]);
  return s >= 0 && s < a.n_slots ? s : 0;
}
__device__ __forceinline__ bool sequence_started(const PrefillArgs& a, int n) {
  return !a.started || __builtin_amdgcn_readfirstlane((int)a.started[n * a.sd_s]) != 0;
}

// log decay and write strength of one token of one value head
__device__ __forceinline__ float log_decay(float x, float a_log) {
  return -expf(a_log) * (x > 20.f ? x : log1pf(expf(x)));
}
__device__ __forceinline__ float sigmoid(float x) { return 1.f / (1.f + expf(-x)); }

// ---------------------------------------------------------------- recurrent
// Token by token, all arithmetic in f32: a wave owns 16 V-rows of one
// value head, a lane 8 columns of 4 of them, in registers from the first token
// to the last. Rows of S are independent, so nothing is shared between waves.
// One read and one write of the state carry a call of a few tokens; a long
// sequence is bound by the chain of a token's row sums (S k must be known
// before S q of the next).
constexpr int kRecRows = 16;  // V-rows per wave

template <class Act, class St, bool GATE_F32>
__global__ __launch_bounds__(256) void recurrent_kernel(const PrefillArgs a) {
  using Gate = typename std::conditional<GATE_F32, ActF32, Act>::type;
  constexpr int ES = Act::kBytes;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tiles = a.V / kRecRows, unit = blockIdx.x * 4 + wave;
  const int n = blockIdx.y;
  if (unit >= a.HV * tiles) return;  // wave-uniform
  const int hv = unit / tiles, row0 = (unit - hv * tiles) * kRecRows, h = hv / a.G;
  const int cl = lane & 15, grp = lane >> 4;
  int begin, end;
  sequence_rows(a, n, begin, end);
  const bool started = sequence_started(a, n);
  if (begin == end && started) return;
  uint8_t* sp = (uint8_t*)a.state + ((int64_t)sequence_slot(a, n) * a.st_s + hv * a.st_h + (int64_t)(row0 + 4 * grp) * a.st_v + 8 * cl) * St::kBytes;
  const int64_t srow = a.st_v * St::kBytes;
  float S[4][8];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    Raw<St, 8> x;
    if (started) x.load(sp + r * srow);
#pragma unroll
    for (int e = 0; e < 8; ++e) S[r][e] = started ? x[e] : 0.f;
  }
  const float a_log = a.a_log[hv * a.al_s], dt_bias = a.dt_bias[hv * a.db_s];
  Raw<Act, 8> q, k, qn, kn;
  Raw<Act, 4> v, vn;
  float ag, bg, agn, bgn;
  auto fetch = [&](int t) {
    const uint8_t* row = (const uint8_t*)a.mixed + (int64_t)t * a.mx_t * ES;
    qn.load(row + (h * K + 8 * cl) * ES);
    kn.load(row + ((a.H + h) * K + 8 * cl) * ES);
    vn.load(row + (2 * a.H * K + hv * a.V + row0 + 4 * grp) * ES);
    agn = Gate::ld(a.a, (int64_t)t * a.a_t + hv * a.a_h);
    bgn = Gate::ld(a.bgate, (int64_t)t * a.bg_t + hv * a.bg_h);
  };
  if (begin < end) fetch(begin);
  for (int t = begin; t < end; ++t) {
    q = qn, k = kn, v = vn, ag = agn, bg = bgn;
    if (t + 1 < end) fetch(t + 1);
    float qf[8], kf[8], qq = 0.f, kk = 0.f, qk = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      qf[e] = q[e], kf[e] = k[e];
      qq = fmaf(qf[e], qf[e], qq);
      kk = fmaf(kf[e], kf[e], kk);
      qk = fmaf(qf[e], kf[e], qk);
    }
    const float rq = 1.f / sqrtf(sum16(qq) + 1e-6f), rk = 1.f / sqrtf(sum16(kk) + 1e-6f);
    const float gamma = expf(log_decay(ag + dt_bias, a_log)), beta = sigmoid(bg);
    qk = sum16(qk) * rq * rk;
    float o[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      float sk = 0.f, sq = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        S[r][e] *= gamma;
        sk = fmaf(S[r][e], kf[e], sk);
        sq = fmaf(S[r][e], qf[e], sq);
      }
      sk = sum16(sk) * rk;
      sq = sum16(sq) * rq;
      const float u = beta * (v[r] - sk), uk = u * rk;
#pragma unroll
      for (int e = 0; e < 8; ++e) S[r][e] = fmaf(uk, kf[e], S[r][e]);
      o[r] = a.out_scale * fmaf(u, qk, sq);  // S q of the updated state
    }
    if (cl == 0) {
      uint8_t* op = (uint8_t*)a.out + ((int64_t)t * a.o_t + hv * a.o_h + row0 + 4 * grp) * ES;
      Act::st2(op, o[0], o[1]);
      Act::st2(op + 2 * ES, o[2], o[3]);
    }
  }
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int e = 0; e < 8; e += 2) St::st2(sp + r * srow + e * St::kBytes, S[r][e], S[r][e + 1]);
}

template <class Act, class St, bool GATE_F32>
int launch_recurrent(const PrefillArgs& a, hipStream_t s) {
  const int units = a.HV * (a.V / kRecRows);
  hipLaunchKernelGGL((recurrent_kernel<Act, St, GATE_F32>), dim3((units + 3) / 4, a.N), dim3(256), 0, s, a);
  return (int)hipGetLastError();
}

template <class Act, bool GATE_F32>
int launch_state(const PrefillArgs& a, int state_dt, hipStream_t s) {
  if (state_dt == DT_BF16) return launch_recurrent<Act, ActBF16, GATE_F32>(a, s);
  if (state_dt == DT_F16) return launch_recurrent<Act, ActF16, GATE_F32>(a, s);
  return launch_recurrent<Act, ActF32, GATE_F32>(a, s);
}

}  // namespace

int launch_prefill(const PrefillArgs& a, int state_dt, int act_dt, bool gate_f32, void* stream) {
  hipStream_t s = (hipStream_t)stream;
  if (act_dt == DT_F32) return launch_state<ActF32, true>(a, state_dt, s);
  if (act_dt == DT_BF16) return gate_f32 ? launch_state<ActBF16, true>(a, state_dt, s) : launch_state<ActBF16, false>(a, state_dt, s);
  return gate_f32 ? launch_state<ActF16, true>(a, state_dt, s) : launch_state<ActF16, false>(a, state_dt, s);
}

}  // namespace gdnr
