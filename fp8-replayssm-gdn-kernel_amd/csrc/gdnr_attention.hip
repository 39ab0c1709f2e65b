// gdnr_attention.hip -- attention of new tokens over a paged cache, causal:
// token j of a sequence of L new tokens whose context holds C keys (the new
// ones last) sees the keys i <= C - L + j,
//   o = sum_i p_i v_i / sum_i p_i,  p_i = exp(scale q k_i - max);
// a row that sees no key gives 0. Heads are grouped: query head h reads the
// keys of head h / G.
//
// One pass over the keys with a running maximum and sum (f32). The rows of a
// workgroup are the (token, query head of the group) pairs of one key head, 16
// to a tile, so the keys of a group are read once. Its four waves take 32 keys
// each in turn and join at the end. The scores are formed transposed,
// K (keys x D) by Q^T: a lane then holds 8 keys of one row, which is, as it
// stands, the operand of V^T (D x keys) by P^T -- the contraction may take the
// keys in any order as long as both operands do. V passes through LDS, where
// the transposing read turns it.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "gdnr_device.h"
#include "gdnr_internal.h"

namespace gdnr {
namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4_t lds_s16x4;

constexpr int kRows = 16;     // rows of a tile
constexpr int kKeys = 32;     // keys of a wave's step
constexpr int kWaves = 4;

template <class Act>
__device__ __forceinline__ f32x4_t mfma(u32x4_t a, u32x4_t b, f32x4_t c) {
  if constexpr (std::is_same<Act, ActBF16>::value)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
}
template <class Act>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t w;
  Act::st2(&w, lo, hi);
  return w;
}
// 4 rows (keys) x 16 columns at p (row stride in bytes), transposed: lane i of
// each 16-lane group receives column i of the group's 4 rows
__device__ __forceinline__ uint2 transposed4(const uint8_t* p) {
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p));
}
// whether any of 8 values is an infinity or a NaN
template <class Act>
__device__ __forceinline__ bool nonfinite8(u32x4_t w) {
  constexpr uint32_t kExp = std::is_same<Act, ActBF16>::value ? 0x7F80u : 0x7C00u;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) bad |= (w[i] & kExp) == kExp || ((w[i] >> 16) & kExp) == kExp;
  return bad;
}
// over the lanes of one column (lane & 15), in each of them
__device__ __forceinline__ float column_max(float x) {
  x = fmaxf(x, __shfl_xor(x, 16));
  return fmaxf(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ float column_sum(float x) {
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}

// Number of sequences n < N with cu[n] / per + n * every <= x (cu clamped to
// [0, T]; it does not decrease).
__device__ __forceinline__ int sequences_up_to(const AttentionArgs& a, int x, int per, int every) {
  const int lane = threadIdx.x & 63;
  int count = 0;
  for (int n0 = 0; n0 < a.N; n0 += 64) {
    const int n = n0 + lane;
    bool below = false;
    if (n < a.N) below = min(max(a.cu[n * a.cu_s], 0), a.T) / per + n * every <= x;
    count += __popcll(__ballot(below));
  }
  return count;
}

struct Span {
  int begin, end, context;
};
// tokens and context length of sequence n, clamped to what there is
__device__ __forceinline__ Span span_of(const AttentionArgs& a, int n) {
  Span s;
  s.begin = min(max(__builtin_amdgcn_readfirstlane(a.cu[n * a.cu_s]), 0), a.T);
  s.end = min(max(__builtin_amdgcn_readfirstlane(a.cu[(n + 1) * a.cu_s]), s.begin), a.T);
  s.context = min(max(__builtin_amdgcn_readfirstlane(a.context[n * a.cx_s]), 0), a.max_context);
  return s;
}
// keys that token t of the sequence sees
__device__ __forceinline__ int visible(const Span& s, int t) { return min(max(s.context - s.end + t + 1, 0), s.context); }

template <int D>
constexpr int v_stride() { return 2 * D + 32; }  // bytes between V rows in LDS: 16 rows' 32-byte pieces on distinct banks
template <int D>
constexpr int o_stride() { return 4 * D + 16; }
template <int D>
constexpr int lds_bytes() {
  const int v = kWaves * kKeys * v_stride<D>(), o = kWaves * kRows * o_stride<D>();
  return (v > o ? v : o) + kWaves * kRows * 8;
}

template <class Act, int D>
__global__ __launch_bounds__(256) void attention_kernel(const AttentionArgs a) {
  constexpr int KSTEPS = D / 32, DT = D / 16, LPR = D / 8, KPI = 64 / LPR, NV = kKeys / KPI;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, grp = lane >> 4;
  const int gt = min(a.G, kRows), tb = kRows / gt;  // heads and tokens of a tile
  const int n = sequences_up_to(a, blockIdx.x, tb, 1) - 1;
  if (n < 0) return;
  const Span sq = span_of(a, n);
  const int tok0 = sq.begin + ((int)blockIdx.x - sq.begin / tb - n) * tb;
  if (tok0 >= sq.end) return;
  const int head_tiles = (a.G + kRows - 1) / kRows;
  const int hk = blockIdx.y / head_tiles, ht = blockIdx.y - hk * head_tiles;
  const int last = min(tok0 + tb, sq.end) - 1;
  const int k_begin = (int)blockIdx.z * a.piece, k_end = min(visible(sq, last), k_begin + a.piece);
  if (k_begin >= k_end && (a.pieces > 1 || blockIdx.z > 0)) return;

  // this lane's row
  const int rt = tok0 + col / gt, rh = ht * kRows + col % gt;
  const bool live = col / gt < tb && rt < sq.end && rh < a.G;
  const int vis = live ? visible(sq, rt) : 0;
  const int vis_all = visible(sq, tok0);  // every live row sees these
  u32x4_t q[KSTEPS];
  {
    const uint8_t* qp = (const uint8_t*)a.q + (rt * a.q_t + (hk * a.G + rh) * a.q_h) * 2 + 16 * grp;
#pragma unroll
    for (int i = 0; i < KSTEPS; ++i) q[i] = live ? *(const u32x4_t*)(qp + 64 * i) : u32x4_t{0, 0, 0, 0};
  }

  uint8_t* vt = lds + wave * kKeys * v_stride<D>();
  const double inv_page = 1.0 / a.page;
  const int32_t* table = a.table + n * a.tb_n;
  const uint8_t* kbase = (const uint8_t*)a.k_cache + hk * a.kc_h * 2 + 16 * grp;
  const uint8_t* vbase = (const uint8_t*)a.v_cache + hk * a.vc_h * 2 + 16 * (lane % LPR);
  // rows of a step's keys, in 16-byte units from the caches' bases: lane l
  // finds key l & 31's
  uint32_t k_row, v_row;
  auto find_rows = [&](int key0) {
    const int key = min(key0 + (lane & 31), k_end - 1);
    int p = (int)((double)key * inv_page), r = key - p * a.page;
    if (r < 0) --p, r += a.page;
    if (r >= a.page) ++p, r -= a.page;
    const int at = min(max(table[p], 0), a.n_pages - 1);
    k_row = (uint32_t)((at * a.kc_p + r * a.kc_t) >> 3);
    v_row = (uint32_t)((at * a.vc_p + r * a.vc_t) >> 3);
  };
  u32x4_t kf[2][KSTEPS], vf[NV];
  auto load = [&](int key0) {
    find_rows(key0);
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      const uint8_t* p = kbase + (uint64_t)(uint32_t)__shfl((int)k_row, 16 * m + col) * 16;
#pragma unroll
      for (int i = 0; i < KSTEPS; ++i) kf[m][i] = *(const u32x4_t*)(p + 64 * i);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int r = i * KPI + lane / LPR;
      const uint8_t* p = vbase + (uint64_t)(uint32_t)__shfl((int)v_row, r) * 16;
      vf[i] = *(const u32x4_t*)p;
      // (a key past the end repeats the last one, weighted 0: not its value,
      // which may be infinite)
      if (key0 + r >= k_end) vf[i] = u32x4_t{0, 0, 0, 0};
    }
  };

  f32x4_t o[DT];
#pragma unroll
  for (int i = 0; i < DT; ++i) o[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  float m_run = -__builtin_inff(), l_run = 0.f;
  int key0 = k_begin + wave * kKeys;
  if (key0 < k_end) load(key0);
  for (; key0 < k_end; key0 += kWaves * kKeys) {
    const bool masked = key0 + kKeys > min(vis_all, k_end);
    bool bad = false;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      *(u32x4_t*)(vt + (i * KPI + lane / LPR) * v_stride<D>() + 16 * (lane % LPR)) = vf[i];
      if (masked) bad |= nonfinite8<Act>(vf[i]);
    }
    f32x4_t s[2];
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      s[m] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < KSTEPS; ++i) s[m] = mfma<Act>(kf[m][i], q[i], s[m]);
    }
    if (key0 + kWaves * kKeys < k_end) load(key0 + kWaves * kKeys);
    float x[8], top = -__builtin_inff();
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[e] = s[e >> 2][e & 3] * a.scale_log2;
      const int key = key0 + 16 * (e >> 2) + 4 * grp + (e & 3);
      if (masked && key >= min(vis, k_end)) x[e] = -__builtin_inff();
      top = fmaxf(top, x[e]);
    }
    top = column_max(top);
    if (__any(top > m_run)) {
      const float m_new = fmaxf(m_run, top);
      const float f = m_new == -__builtin_inff() ? 1.f : __builtin_amdgcn_exp2f(m_run - m_new);
      l_run *= f;
#pragma unroll
      for (int i = 0; i < DT; ++i) o[i] *= f;
      m_run = m_new;
    }
    const float base = m_run == -__builtin_inff() ? 0.f : m_run;
    float p[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) p[e] = __builtin_amdgcn_exp2f(x[e] - base), l_run += p[e];
    if (__any(bad)) {
      // a value that some rows must not see is infinite or NaN, and a product
      // with its weight 0 would show it to them: this step key by key
#pragma unroll
      for (int e = 0; e < 8; ++e)
#pragma nounroll
        for (int g = 0; g < 4; ++g) {
          const int key = 16 * (e >> 2) + 4 * g + (e & 3);
          const float pk = __shfl(p[e], col + 16 * g);
          const bool seen = key0 + key < min(vis, k_end);
#pragma unroll
          for (int i = 0; i < DT; ++i) {
            const uint2 w = *(const uint2*)(vt + key * v_stride<D>() + 32 * i + 8 * grp);
            const float2 lo = Act::from_pair(w.x), hi = Act::from_pair(w.y);
            const f32x4_t v = {lo.x, lo.y, hi.x, hi.y};
            if (seen) o[i] += pk * v;
          }
        }
      continue;
    }
    // (the sum is of the unrounded weights; rounding them to the cache's type
    // costs the output about its own rounding)
    const u32x4_t pf = {pack2<Act>(p[0], p[1]), pack2<Act>(p[2], p[3]), pack2<Act>(p[4], p[5]), pack2<Act>(p[6], p[7])};
#pragma unroll
    for (int i = 0; i < DT; ++i) {
      const uint8_t* at = vt + (4 * grp + (col >> 2)) * v_stride<D>() + 32 * i + 8 * (col & 3);
      const uint2 lo = transposed4(at), hi = transposed4(at + 16 * v_stride<D>());
      o[i] = mfma<Act>(u32x4_t{lo.x, lo.y, hi.x, hi.y}, pf, o[i]);
    }
  }
  l_run = column_sum(l_run);

  // join the waves: every row's sums at the largest maximum
  __syncthreads();
  float* ml = (float*)(lds + lds_bytes<D>() - kWaves * kRows * 8);
  uint8_t* ow = lds + wave * kRows * o_stride<D>() + col * o_stride<D>() + 16 * grp;
#pragma unroll
  for (int i = 0; i < DT; ++i) *(f32x4_t*)(ow + 64 * i) = o[i];
  if (grp == 0) ml[2 * (wave * kRows + col)] = m_run, ml[2 * (wave * kRows + col) + 1] = l_run;
  __syncthreads();
  const int row = threadIdx.x >> 4, dl = threadIdx.x & 15;
  const int t = tok0 + row / gt, head = ht * kRows + row % gt;
  if (row / gt >= tb || t >= sq.end || head >= a.G) return;
  float top = -__builtin_inff(), l = 0.f, f[kWaves];
#pragma unroll
  for (int w = 0; w < kWaves; ++w) top = fmaxf(top, ml[2 * (w * kRows + row)]);
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    f[w] = top == -__builtin_inff() ? 1.f : __builtin_amdgcn_exp2f(ml[2 * (w * kRows + row)] - top);
    l += f[w] * ml[2 * (w * kRows + row) + 1];
  }
  const int qh = hk * a.G + head;
  const float norm = a.pieces > 1 ? 1.f : visible(sq, t) == 0 ? 0.f : 1.f / l;
#pragma unroll
  for (int i = 0; i < D / 64; ++i) {
    const int d = 64 * i + 4 * dl;
    f32x4_t sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) sum += f[w] * *(const f32x4_t*)(lds + (w * kRows + row) * o_stride<D>() + 4 * d);
    sum *= norm;
    if (a.pieces > 1) {
      *(f32x4_t*)(a.part + (((int64_t)blockIdx.z * a.T + t) * a.HQ + qh) * D + d) = sum;
    } else {
      *(uint2*)((uint8_t*)a.out + (t * a.o_t + qh * a.o_h + d) * 2) = make_uint2(pack2<Act>(sum[0], sum[1]), pack2<Act>(sum[2], sum[3]));
    }
  }
  if (a.pieces > 1 && dl == 0) {
    float* p = a.part_ml + (((int64_t)blockIdx.z * a.T + t) * a.HQ + qh) * 2;
    p[0] = top, p[1] = l;
  }
}

// The pieces of a row joined in their order, one wave a row.
template <class Act, int D>
__global__ __launch_bounds__(256) void join_kernel(const AttentionArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int t = __builtin_amdgcn_readfirstlane((int)(row / a.HQ)), h = (int)(row - (int64_t)t * a.HQ);
  if (t >= a.T) return;
  const int n = sequences_up_to(a, t, 1, 0) - 1;
  if (n < 0) return;
  const Span sq = span_of(a, n);
  if (t >= sq.end) return;
  const int vis = visible(sq, t), pieces = (vis + a.piece - 1) / a.piece;
  constexpr int E = D / 64;
  float acc[E] = {}, top = -__builtin_inff(), l = 0.f;
  for (int z = 0; z < pieces; ++z) {
    const int64_t at = ((int64_t)z * a.T + t) * a.HQ + h;
    const float m = a.part_ml[2 * at], lz = a.part_ml[2 * at + 1];
    const float m_new = fmaxf(top, m);
    const float fo = m_new == -__builtin_inff() ? 1.f : __builtin_amdgcn_exp2f(top - m_new);
    const float fz = m_new == -__builtin_inff() ? 1.f : __builtin_amdgcn_exp2f(m - m_new);
    l = l * fo + lz * fz;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = acc[e] * fo + fz * a.part[at * D + E * lane + e];
    top = m_new;
  }
  const float norm = vis == 0 ? 0.f : 1.f / l;
  uint8_t* op = (uint8_t*)a.out + (t * a.o_t + h * a.o_h + E * lane) * 2;
  if constexpr (E == 1) {
    Act::st(op, 0, acc[0] * norm);
  } else {
#pragma unroll
    for (int e = 0; e < E; e += 2) Act::st2(op + 2 * e, acc[e] * norm, acc[e + 1] * norm);
  }
}

template <class Act, int D>
int launch_dim(const AttentionArgs& a, hipStream_t s) {
  const int gt = a.G < kRows ? a.G : kRows, tb = kRows / gt, head_tiles = (a.G + kRows - 1) / kRows;
  if (lds_bytes<D>() > 64 * 1024) {  // (enabled per kernel and device; idempotent, cheap)
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(attention_kernel<Act, D>),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, lds_bytes<D>());
    if (e != hipSuccess) return (int)e;
  }
  hipLaunchKernelGGL((attention_kernel<Act, D>), dim3(a.T / tb + a.N, a.HKV * head_tiles, a.pieces), dim3(256), lds_bytes<D>(), s, a);
  if (a.pieces > 1)
    hipLaunchKernelGGL((join_kernel<Act, D>), dim3((uint32_t)(((int64_t)a.T * a.HQ + 3) / 4)), dim3(256), 0, s, a);
  return (int)hipGetLastError();
}
template <class Act>
int launch_act(const AttentionArgs& a, hipStream_t s) {
  if (a.D == 64) return launch_dim<Act, 64>(a, s);
  if (a.D == 128) return launch_dim<Act, 128>(a, s);
  return launch_dim<Act, 256>(a, s);
}

}  // namespace

int launch_attention(const AttentionArgs& a, int act_dt, void* stream) {
  return act_dt == DT_BF16 ? launch_act<ActBF16>(a, (hipStream_t)stream) : launch_act<ActF16>(a, (hipStream_t)stream);
}

}  // namespace gdnr
