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

// whether the squares of a key or query may pass f32's range
template <class Act>
constexpr bool kMayBeLarge = !std::is_same<Act, ActF16>::value;

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
// One read and one write of the state carry a call of a few tokens (8 sequences
// of 4 tokens, HV=32, V=128, bf16: 9.1 us, of which the 15.5 MB of states and
// rows take 3.1 at a copy's rate; launch, the reads' latency and 240 instructions
// a token and wave the rest, one after the other since all waves start together).
// A long sequence is bound by the chain of a token's row sums (S k must be known
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
  if ((begin == end && started) || end - begin >= a.chunk_from) return;
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
  auto fetch = [&](int t) {
    const uint8_t* row = (const uint8_t*)a.mixed + (int64_t)t * a.mx_t * ES;
    qn.load(row + (h * K + 8 * cl) * ES);
    kn.load(row + ((a.H + h) * K + 8 * cl) * ES);
    vn.load(row + (2 * a.H * K + hv * a.V + row0 + 4 * grp) * ES);
  };
  // the gates of 64 tokens at once, a lane a token
  float gamma64 = 0.f, beta64 = 0.f;
  auto gates = [&](int t) {
    const int64_t at = min(t + lane, end - 1);
    gamma64 = expf(log_decay(Gate::ld(a.a, at * a.a_t + hv * a.a_h) + dt_bias, a_log));
    beta64 = sigmoid(Gate::ld(a.bgate, at * a.bg_t + hv * a.bg_h));
  };
  if (begin < end) fetch(begin);
  for (int t = begin; t < end; ++t) {
    q = qn, k = kn, v = vn;
    if (t + 1 < end) fetch(t + 1);
    if (((t - begin) & 63) == 0) gates(t);
    float qf[8], kf[8], qq = 0.f, kk = 0.f, qk = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      qf[e] = q[e], kf[e] = k[e];
      qq = fmaf(qf[e], qf[e], qq);
      kk = fmaf(kf[e], kf[e], kk);
      qk = fmaf(qf[e], kf[e], qk);
    }
    if constexpr (kMayBeLarge<Act>) {
      if (__any(fmaxf(qq, kk) >= kLargeSquares)) {
        const float fq = row_factor<16>(qf), fk = row_factor<16>(kf);
        qq = 0.f, kk = 0.f, qk = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          qf[e] *= fq, kf[e] *= fk;
          qq = fmaf(qf[e], qf[e], qq);
          kk = fmaf(kf[e], kf[e], kk);
          qk = fmaf(qf[e], kf[e], qk);
        }
      }
    }
    const float rq = __builtin_amdgcn_rsqf(sum16(qq) + 1e-6f), rk = __builtin_amdgcn_rsqf(sum16(kk) + 1e-6f);
    const float gamma = readlane_f(gamma64, (t - begin) & 63), beta = readlane_f(beta64, (t - begin) & 63);
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

// ---------------------------------------------------------------- chunked
// C tokens at once. With G_t = sum of the log decays up to t in the chunk and
// S0 the state before it,
//   (I + M) U = beta (V - e^G (K S0^T)),   M_ti = beta_t e^(G_t - G_i) k_t.k_i  (i < t)
//   O  = scale (e^G (Q S0^T) + A U),       A_ti = e^(G_t - G_i) q_t.k_i         (i <= t)
//   S1 = e^(G_C) S0 + sum_t e^(G_C - G_t) u_t k_t^T,
// (U's rows are the corrections beta (v - S k) of the recurrence, unrolled).
// T = (I + M)^-1 and A depend on the chunk alone: chunk_prep_kernel forms them
// for every chunk at once, with the unit keys and queries. chunk_scan_kernel
// then walks a sequence's chunks with matrix products.
//
// Numbers: the products run on f16 operands with f32 sums. Unit keys and
// queries, A and T (|T| <= 1: products of contractions) are safe in f16; V,
// S0, R and U get a power of two per V-row and chunk, from the largest of the
// row's v and state, that keeps them in range (V-rows do not mix, so each
// keeps its own precision whatever its neighbours hold; a chunk whose tokens
// differ too much for one such factor is walked token by token). An f16 operand costs
// 2^-12 of itself, an eighth of what storing bf16 does: bf16 outputs and states
// are bound by their own rounding. Where a result keeps more than bf16 (f16
// or f32 activations or state), SPLIT carries every operand as a sum of two
// f16 values and each product as three, good to some 2^-22. The state between
// chunks, sums and decays are f32 (the sums of log decays f64, so that
// differences of long sums stay exact).
//
// A token whose key or gates are not finite, and a V-row whose v or state is
// not, would reach earlier tokens through products with 0: both are computed
// as zeros and everything from their token on is written as NaN.
constexpr int C = 64;                   // tokens of a chunk
constexpr int kTri = 6;                 // 16 x 32 operand tiles of a lower triangle of 64
constexpr float kFix = 1024.f;          // SPLIT: factor of unit operands, keeps their low halves normal

typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef float f32x2v_t __attribute__((ext_vector_type(2)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4_t lds_s16x4;

__device__ __forceinline__ f32x4_t mfma(u32x4_t a, u32x4_t b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const f32x2v_t v = {lo, hi};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2_t));
}
__device__ __forceinline__ float2 unpack_f16(uint32_t w) {
  const f16x2_t h = __builtin_bit_cast(f16x2_t, w);
  return make_float2((float)h[0], (float)h[1]);
}

// 8 values as an MFMA operand: f16, or f16 plus the f16 of what that leaves
template <bool SPLIT>
struct Operand {
  u32x4_t hi, lo;
};
template <bool SPLIT>
__device__ __forceinline__ Operand<SPLIT> operand(f32x4_t a, f32x4_t b) {
  Operand<SPLIT> o;
  const float x[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    o.hi[i] = pack_f16(x[2 * i], x[2 * i + 1]);
    if constexpr (SPLIT) {
      const float2 h = unpack_f16(o.hi[i]);
      o.lo[i] = pack_f16(x[2 * i] - h.x, x[2 * i + 1] - h.y);
    }
  }
  return o;
}
template <bool SPLIT>
__device__ __forceinline__ f32x4_t product(const Operand<SPLIT>& a, const Operand<SPLIT>& b, f32x4_t c) {
  if constexpr (SPLIT) {
    c = mfma(a.lo, b.hi, c);
    c = mfma(a.hi, b.lo, c);
  }
  return mfma(a.hi, b.hi, c);
}

// Workspace: per chunk slot and key head the unit keys and queries [C][K] f16
// (SPLIT: high, then low), a row's pieces as unit_at places them; per slot and
// value head the tokens' {beta}[C], {-beta e^G}[C], {e^(G_C - G)}[C], {e^G}[C],
// first bad token (an int) in 64 words, {e^g}[C], padded to 2 KiB, then the operand
// tiles of T - I and of A (64 lanes x 16 bytes each; SPLIT: high, then low). The
// chunks of a sequence take slots one after the other.
constexpr int kScalars = 2048;
__host__ __device__ constexpr int64_t plane_bytes(bool split) { return C * K * 2 * (split ? 2 : 1); }  // keys, or queries
__host__ __device__ constexpr int64_t unit_bytes(bool split) { return 2 * plane_bytes(split); }
__host__ __device__ constexpr int64_t tri_bytes(bool split) { return kTri * 1024 * (split ? 2 : 1); }
__host__ __device__ constexpr int64_t head_bytes(bool split) { return kScalars + 2 * tri_bytes(split); }

// One of 64 sequences n, a lane's, among them (a.N and more: none): its tokens,
// whether it is walked in chunks, and how many before it and in all of the 64 are.
struct Lengths {
  int begin, end, chunked_before, chunked_all;
  bool chunked;
};
__device__ __forceinline__ Lengths lengths_of(const PrefillArgs& a, int n) {
  Lengths x = {0, 0, 0, 0, false};
  if (n < a.N) {
    x.begin = min(max(a.cu[n * a.cu_s], 0), a.T), x.end = min(max(a.cu[(n + 1) * a.cu_s], x.begin), a.T);
    x.chunked = x.end - x.begin >= a.chunk_from;
  }
  const uint64_t m = __ballot(x.chunked);
  x.chunked_before = __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0));
  x.chunked_all = __popcll(m);
  return x;
}
// most sequences that may be walked in chunks
__host__ __device__ inline int64_t chunked_most(int64_t T, int64_t N, int32_t chunk_from) {
  return chunk_from && T / chunk_from < N ? T / chunk_from : N;
}
// slots of chunks: sequence n's are those from begin / C + the sequences in chunks
// before it on
__host__ __device__ inline int64_t chunk_slots(int64_t T, int64_t N, int32_t chunk_from) {
  return T / C + chunked_most(T, N, chunk_from);
}

struct Work {
  uint8_t* unit;  // [slots][H]
  uint8_t* head;  // [slots][HV]
};
__host__ __device__ inline Work work_of(const PrefillArgs& a, bool split) {
  return {a.work, a.work + chunk_slots(a.T, a.N, a.chunk_from) * a.H * unit_bytes(split)};
}

// Byte of 4 elements (k = 4 k4 ..) of row t. A 16-byte piece holds the 8 elements
// that a lane gives to a product over 32 columns (4 g .. + 3 of each half of
// them), and row t keeps its piece p at p ^ (t & 15), so that the 16 rows of a
// fragment lie on distinct LDS banks.
__host__ __device__ constexpr int unit_at(int t, int k4) {
  return 2 * K * t + 16 * ((4 * (k4 >> 3) + (k4 & 3)) ^ (t & 15)) + 8 * ((k4 >> 2) & 1);
}

// index of the tile (16 rows of t, 32 columns of i) in a lower triangle
__host__ __device__ constexpr int tri(int tt, int ts) { return tt < 2 ? tt : 2 * (tt - 1) + ts; }

// A sum of log2 decays as two floats, hi the rounded sum and lo what that leaves.
// 2^(a - b): the difference of the hi's is off by 2^-24 of itself at most, which
// SPLIT corrects along with the lo's.
template <bool SPLIT>
__device__ __forceinline__ float exp2_diff(float2 a, float2 b) {
  const float d = a.x - b.x, e = __builtin_amdgcn_exp2f(d);
  const float t = d - a.x;  // (two-sum: what a.x - b.x rounded off)
  const float rest = (SPLIT ? (a.x - (d - t)) - (b.x + t) : 0.f) + (a.y - b.y);
  return fmaf(e, 0.6931471805599453f * rest, e);
}
__device__ __forceinline__ double readlane_d(double x, int lane) {
  const uint64_t b = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)b, lane), hi = __builtin_amdgcn_readlane((int)(uint32_t)(b >> 32), lane);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
template <int CTRL>
__device__ __forceinline__ double dpp_d(double x) {  // lanes with no source get 0
  const uint64_t b = __builtin_bit_cast(uint64_t, x);
  return __builtin_bit_cast(double, (uint64_t)dpp_u<CTRL>((uint32_t)(b >> 32)) << 32 | dpp_u<CTRL>((uint32_t)b));
}
// sum over the lanes up to this one, and over all 64: within rows of 16 lanes,
// then the rows before
__device__ __forceinline__ double prefix_sum(double x, double& total) {
  x += dpp_d<0x111>(x);
  x += dpp_d<0x112>(x);
  x += dpp_d<0x114>(x);
  x += dpp_d<0x118>(x);
  const double r0 = readlane_d(x, 15), r1 = r0 + readlane_d(x, 31), r2 = r1 + readlane_d(x, 47);
  total = r2 + readlane_d(x, 63);
  const int row = (threadIdx.x & 63) >> 4;
  return x + (row == 0 ? 0.0 : row == 1 ? r0 : row == 2 ? r1 : r2);
}

// One chunk of one key head: 4 waves. The Gram products are formed transposed
// (rows i on a lane's registers, columns t on lanes), which is the order that
// the scan's operands take them in. Bound by its bytes: 8192 tokens of 16 key and
// 32 value heads read 84 MB and write 123 MB (counters) in 52 us (4.0 TB/s, four fifths
// of a copy's rate); one workgroup alone takes 11.9 us, which four of
// them a compute unit cover.
template <class Act, bool GATE_F32, bool SPLIT>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(SPLIT ? 2 : 4, SPLIT ? 2 : 4))) void chunk_prep_kernel(const PrefillArgs a) {
  using Gate = typename std::conditional<GATE_F32, ActF32, Act>::type;
  constexpr int ES = Act::kBytes, RS = 2 * K + 16, P = SPLIT ? 2 : 1;  // LDS row of a key or query, halves
  constexpr int kUnits = 2 * P * C * RS, MS = 68 * 4, kM = C * MS;      // [i][t] f32 of M, per head
  __shared__ __attribute__((aligned(16))) uint8_t lds[kUnits > 2 * kM ? kUnits : 2 * kM];
  __shared__ float2 Gs[2][C];  // sums of log2 decays
  __shared__ float betas[2][C];
  __shared__ int bad_key;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, grp = lane >> 4;
  const int slot = blockIdx.x, h = blockIdx.y, g_first = 2 * blockIdx.z;

  // the slot's sequence and first row
  int n = -1, first_slot = 0, before = 0;
  for (int n0 = 0; n0 < a.N; n0 += 64) {
    const Lengths own = lengths_of(a, n0 + lane);
    const int from = own.begin / C + before + own.chunked_before;
    const uint64_t at = __ballot(own.chunked && from <= slot);
    if (at) {
      n = n0 + 63 - __builtin_clzll(at);
      first_slot = __builtin_amdgcn_readlane(from, 63 - __builtin_clzll(at));
    }
    before += own.chunked_all;
  }
  if (n < 0) return;
  int begin, end;
  sequence_rows(a, n, begin, end);
  const int row0 = begin + (slot - first_slot) * C, len = min(end - row0, C);
  if (len <= 0) return;
  const Work w = work_of(a, SPLIT);
  if (threadIdx.x == 0) bad_key = C;

  // every row's keys and queries, 16 lanes a row, and the gates of the first
  // two of its value heads are asked for at once
  uint8_t* unit = w.unit + ((int64_t)slot * a.H + h) * unit_bytes(SPLIT);
  Raw<Act, 8> rows[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int t = min(16 * (i & 3) + 4 * wave + grp, len - 1);
    rows[i].load((const uint8_t*)a.mixed + ((int64_t)(row0 + t) * a.mx_t + (i >= 4 ? h : a.H + h) * K + 8 * col) * ES);
  }
  float ga = 0.f, gb = 0.f, g_log = 0.f, g_bias = 0.f;
  auto load_gates = [&](int g0) {
    const int hv = h * a.G + min(g0 + wave, a.G - 1);
    const int64_t at = row0 + min(lane, len - 1);
    ga = Gate::ld(a.a, at * a.a_t + hv * a.a_h), gb = Gate::ld(a.bgate, at * a.bg_t + hv * a.bg_h);
    g_log = a.a_log[hv * a.al_s], g_bias = a.dt_bias[hv * a.db_s];
  };
  load_gates(g_first);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const bool is_q = i >= 4;
    const int t = 16 * (i & 3) + 4 * wave + grp;
    float x[8], ss = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = t < len ? rows[i][e] : 0.f, ss = fmaf(x[e], x[e], ss);
    if constexpr (kMayBeLarge<Act>) {
      if (__any(ss >= kLargeSquares)) {
        const float f = row_factor<16>(x);
        ss = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] *= f, ss = fmaf(x[e], x[e], ss);
      }
    }
    ss = sum16(ss);
    float f = __builtin_amdgcn_rsqf(ss + 1e-6f);
    if (!is_q && !(ss < __builtin_inff())) {
      if (col == 0) atomicMin(&bad_key, t);
      f = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = 0.f;
    }
    if constexpr (SPLIT) f *= kFix;
    const Operand<SPLIT> o = operand<SPLIT>(f32x4_t{x[0] * f, x[1] * f, x[2] * f, x[3] * f}, f32x4_t{x[4] * f, x[5] * f, x[6] * f, x[7] * f});
    const int plane = (is_q ? P : 0);
    *(u32x4_t*)(lds + (plane * C + t) * RS + 16 * col) = o.hi;
    if constexpr (SPLIT) *(u32x4_t*)(lds + ((plane + 1) * C + t) * RS + 16 * col) = o.lo;
    if (g_first) continue;  // (the first workgroup of the group writes them)
    *(uint2*)(unit + plane * C * 2 * K + unit_at(t, 2 * col)) = make_uint2(o.hi[0], o.hi[1]);
    *(uint2*)(unit + plane * C * 2 * K + unit_at(t, 2 * col + 1)) = make_uint2(o.hi[2], o.hi[3]);
    if constexpr (SPLIT) {
      *(uint2*)(unit + (plane + 1) * C * 2 * K + unit_at(t, 2 * col)) = make_uint2(o.lo[0], o.lo[1]);
      *(uint2*)(unit + (plane + 1) * C * 2 * K + unit_at(t, 2 * col + 1)) = make_uint2(o.lo[2], o.lo[3]);
    }
  }
  __syncthreads();

  // wave w: columns t of tile w, rows i of tiles 0..w
  f32x4_t kk[4], qk[4];
  auto fragment = [&](int plane, int tile, int step) {
    Operand<SPLIT> o;
    o.hi = *(const u32x4_t*)(lds + (plane * C + 16 * tile + col) * RS + 64 * step + 16 * grp);
    if constexpr (SPLIT) o.lo = *(const u32x4_t*)(lds + ((plane + 1) * C + 16 * tile + col) * RS + 64 * step + 16 * grp);
    return o;
  };
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    kk[c] = f32x4_t{0.f, 0.f, 0.f, 0.f}, qk[c] = kk[c];
    if (c > wave) continue;
#pragma unroll
    for (int s = 0; s < K / 32; ++s) {
      const Operand<SPLIT> ki = fragment(0, c, s);
      kk[c] = product<SPLIT>(ki, fragment(0, wave, s), kk[c]);
      qk[c] = product<SPLIT>(ki, fragment(P, wave, s), qk[c]);
    }
    if constexpr (SPLIT) kk[c] *= 1.f / (kFix * kFix), qk[c] *= 1.f / kFix;  // (A keeps one factor)
  }

  // the group's value heads, two at a time
  for (int g0 = g_first; g0 < a.G; g0 += 2 * gridDim.z) {
    const int heads = min(2, a.G - g0);
    __syncthreads();  // the units (or the last heads' M) are no longer read
    if (wave < heads) {
      const int hv = h * a.G + g0 + wave, t = lane;
      float g = 0.f, beta = 0.f;
      bool bad = t >= bad_key;
      if (g0 != g_first) load_gates(g0);
      if (t < len) {
        g = log_decay(ga + g_bias, g_log);
        beta = sigmoid(gb);
        bad |= g != g || beta != beta || g > 3e38f;
      }
      const uint64_t bads = __ballot(bad && t < len);
      const int first = bads ? __ffsll((unsigned long long)bads) - 1 : C;
      if (t >= first) g = 0.f, beta = 0.f;
      // (a decay of e^-1e4 is 0 in every format; a sum of such stays exact)
      double last;
      const double sum = prefix_sum((double)fmaxf(g, -1e4f) * 1.4426950408889634, last);
      const float2 G = make_float2((float)sum, (float)(sum - (double)(float)sum));
      const float2 end = make_float2((float)last, (float)(last - (double)(float)last));
      Gs[wave][t] = G;
      betas[wave][t] = beta;
      float* sc = (float*)(w.head + ((int64_t)slot * a.HV + hv) * head_bytes(SPLIT));
      const float grow = exp2_diff<SPLIT>(G, make_float2(0.f, 0.f));
      sc[t] = beta;
      sc[C + t] = -beta * grow * (SPLIT ? 1.f / kFix : 1.f);
      sc[2 * C + t] = exp2_diff<SPLIT>(end, G);
      sc[3 * C + t] = grow;
      if (t == 0) ((int*)sc)[4 * C] = first;
      sc[5 * C + t] = expf(g);
    }
    __syncthreads();
#pragma nounroll
    for (int e = 0; e < heads; ++e) {
      uint8_t* tiles = w.head + ((int64_t)slot * a.HV + h * a.G + g0 + e) * head_bytes(SPLIT) + kScalars;
      const int t = 16 * wave + col;
      const float2 Gt = Gs[e][t];
      const float bt = betas[e][t];
      f32x4_t at[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        at[c] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        if (c > wave) continue;
        f32x4_t m;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int i = 16 * c + 4 * grp + j;
          const float2 Gi = Gs[e][i];
          const float decay = exp2_diff<SPLIT>(i <= t ? Gt : Gi, Gi);
          at[c][j] = i <= t ? decay * qk[c][j] : 0.f;
          m[j] = i < t ? bt * decay * kk[c][j] : 0.f;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) *(float*)(lds + e * kM + (16 * c + 4 * grp + j) * MS + t * 4) = m[j];
      }
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        if (2 * s > wave) continue;
        const Operand<SPLIT> o = operand<SPLIT>(at[2 * s], at[2 * s + 1]);
        uint8_t* p = tiles + (kTri * P + tri(wave, s)) * 1024 + 16 * lane;
        *(u32x4_t*)p = o.hi;
        if constexpr (SPLIT) *(u32x4_t*)(p + kTri * 1024) = o.lo;
      }
    }
    __syncthreads();
    // T = (I + M)^-1 by blocks of 16, wave w the block row w. First its
    // diagonal block, a lane a column of it (lanes of group e: head g0 + e): (I + M) x
    // = e_c, each entry, once known, taken out of all below it. It takes M's place.
    if (grp < heads) {
      uint8_t* m = lds + grp * kM + 16 * wave * (MS + 4);  // [i][t]
      float x[16];
#pragma unroll
      for (int t = 0; t < 16; ++t) x[t] = col == t ? 1.f : 0.f;
#pragma unroll
      for (int i = 0; i < 15; ++i)
#pragma unroll
        for (int q = (i + 1) / 4; q < 4; ++q) {
          const f32x4_t mi = *(const f32x4_t*)(m + i * MS + 16 * q);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (4 * q + j > i) x[4 * q + j] = fmaf(-x[i], mi[j], x[4 * q + j]);
        }
#pragma unroll
      for (int q = 0; q < 4; ++q) *(f32x4_t*)(m + col * MS + 16 * q) = f32x4_t{x[4 * q], x[4 * q + 1], x[4 * q + 2], x[4 * q + 3]};
    }
    __syncthreads();
    // Then T_wJ = -(sum over L = J+1..w of T_wL M_LJ) T_JJ, the nearest block
    // first, transposed (rows of J on registers, t on lanes): what one product
    // leaves is the next one's right operand, and M and T_JJ are read from LDS
    // as they lie.
#pragma nounroll
    for (int e = 0; e < heads; ++e) {
      const uint8_t* m = lds + e * kM;
      f32x4_t x[4];
#pragma unroll
      for (int c = 3; c >= 0; --c) {
        x[c] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        if (c == wave)
#pragma unroll
          for (int j = 0; j < 4; ++j) x[c][j] = *(const float*)(m + (16 * c + 4 * grp + j) * MS + (16 * c + col) * 4);
        if (c >= wave) continue;
        const f32x4_t tl = *(const f32x4_t*)(m + (16 * c + col) * MS + (16 * c + 4 * grp) * 4);
        f32x4_t y = x[c];
#pragma unroll
        for (int l = c + 1; l < 4; ++l) {
          if (l > wave) continue;
          const f32x4_t ml = *(const f32x4_t*)(m + (16 * c + col) * MS + (16 * l + 4 * grp) * 4);
#pragma unroll
          for (int j = 0; j < 4; ++j) y = __builtin_amdgcn_mfma_f32_16x16x4f32(ml[j], x[l][j], y, 0, 0, 0);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) x[c] = __builtin_amdgcn_mfma_f32_16x16x4f32(-tl[j], y[j], x[c], 0, 0, 0);
      }
      uint8_t* tiles = w.head + ((int64_t)slot * a.HV + h * a.G + g0 + e) * head_bytes(SPLIT) + kScalars;
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (c == wave && 4 * grp + j == col) x[c][j] = 0.f;  // T - I
          if constexpr (SPLIT) x[c][j] *= kFix;
        }
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        if (2 * s > wave) continue;
        const Operand<SPLIT> o = operand<SPLIT>(x[2 * s], x[2 * s + 1]);
        uint8_t* p = tiles + tri(wave, s) * 1024 + 16 * lane;
        *(u32x4_t*)p = o.hi;
        if constexpr (SPLIT) *(u32x4_t*)(p + kTri * 1024) = o.lo;
      }
    }
  }
}

// max(m, |a|, |b|), NaN propagating (one v_maximum3_f32)
__device__ __forceinline__ float max3_abs(float m, float a, float b) {
  return __builtin_elementwise_maximum(__builtin_elementwise_maximum(m, __builtin_fabsf(a)), __builtin_fabsf(b));
}
__device__ __forceinline__ bool finite(float x) { return __builtin_fabsf(x) < __builtin_inff(); }
// over the lanes of one column (lane & 15), in each of them; NaN propagating
__device__ __forceinline__ float column_max(float x) {
  const uint32_t b = __float_as_uint(x);
  const auto half = __builtin_amdgcn_permlane32_swap(b, b, false, false);
  const uint32_t h = __float_as_uint(__builtin_elementwise_maximum(__uint_as_float(half[0]), __uint_as_float(half[1])));
  const auto row = __builtin_amdgcn_permlane16_swap(h, h, false, false);
  return __builtin_elementwise_maximum(__uint_as_float(row[0]), __uint_as_float(row[1]));
}

// (code that is left out of the way of what runs for every chunk)
__device__ __forceinline__ bool rare(bool x) { return __builtin_expect(x, false); }
// whether each of the 16 columns has a lane in the mask
__device__ __forceinline__ bool all_columns(uint64_t lanes) {
  lanes |= lanes >> 32;
  return ((lanes | lanes >> 16) & 0xFFFF) == 0xFFFF;
}

// Of a 16-row tile as a product leaves it (rows 4 grp + j, column lane & 15),
// each lane's 4 rows against the columns of its 4 neighbours: row 4 grp + (lane & 3)
// at columns lane & 12 to (lane & 12) + 3, to p (this lane's own place there),
// rounded to the activations' type, where `in`. One store in place of four.
template <class Act>
__device__ __forceinline__ void store_turned(uint8_t* p, const f32x4_t& x, int lane, bool in) {
  const bool odd = lane & 1, upper = lane & 2;
  if constexpr (Act::kBytes == 2) {
    auto pack = [](float lo, float hi) {
      if constexpr (std::is_same<Act, ActBF16>::value) return pack_bf16x2(lo, hi);
      else return pack_f16(lo, hi);
    };
    const uint32_t a = pack(x[0], x[1]), b = pack(x[2], x[3]);
    const uint32_t take = odd ? 0x03020706u : 0x05040100u;  // bytes 0-3 own, 4-7 the neighbour's
    const uint32_t r01 = __builtin_amdgcn_perm(dpp_u<kDppXor1>(a), a, take), r23 = __builtin_amdgcn_perm(dpp_u<kDppXor1>(b), b, take);
    const uint32_t y = dpp_u<kDppXor2>(upper ? r01 : r23);
    if (in) *(uint2*)p = upper ? make_uint2(y, r23) : make_uint2(r01, y);
  } else {
    const float a = dpp_f<kDppXor1>(odd ? x[0] : x[1]), b = dpp_f<kDppXor1>(odd ? x[2] : x[3]);
    const float2 r01 = odd ? make_float2(a, x[1]) : make_float2(x[0], a), r23 = odd ? make_float2(b, x[3]) : make_float2(x[2], b);
    const float y0 = dpp_f<kDppXor2>(upper ? r01.x : r23.x), y1 = dpp_f<kDppXor2>(upper ? r01.y : r23.y);
    if (in) *(f32x4_t*)p = upper ? f32x4_t{y0, y1, r23.x, r23.y} : f32x4_t{r01.x, r01.y, y0, y1};
  }
}

// KIB KiB (an even number) from memory to LDS, by COUNT waves of which this is wave w
template <int KIB, int COUNT>
__device__ __forceinline__ void dma_part(const uint8_t* src, uint32_t lds_addr, int w) {
#pragma unroll
  for (int i = 0; i < (KIB + 4 * COUNT - 1) / (4 * COUNT); ++i) {
    const int x = i * COUNT + w;  // wave-uniform
    if (x < KIB / 4) dma_kib<4>(src + x * 4096, lds_addr + x * 4096);
    else if (KIB % 4 && x == KIB / 4) dma_kib<2>(src + x * 4096, lds_addr + x * 4096);
  }
}

// The sequence at a place of the launch's order (-1: none) and its first slot: of each
// 64 sequences those of most chunks first. Workgroups start in order as others end,
// so that the last to start are then short ones (24 sequences of up to 1096 tokens:
// the scan 186 us as given, 168 so). The place is looked for bit by bit of the chunk
// counts.
__device__ __forceinline__ int longest_first(const PrefillArgs& a, int place, int& first_slot) {
  const int lane = threadIdx.x & 63, most = min((int)chunked_most(a.T, a.N, a.chunk_from), 64), group = place / most, base = 64 * group;
  first_slot = 0;
  if (a.N == 1) return 0;  // (in chunks)
  int before = 0;
  if (a.chunk_from == 0) before = base;
  else
    for (int n0 = 0; n0 < base; n0 += 64) before += lengths_of(a, n0 + lane).chunked_all;
  const Lengths own = lengths_of(a, base + lane);
  const uint32_t size = (uint32_t)(own.end - own.begin + C - 1) / C;
  uint64_t left = __ballot(own.chunked);
  int k = place - group * most;  // the place among those left
  if (k >= own.chunked_all) return -1;
  for (int bit = 31 - __builtin_clz((uint32_t)(a.T / C + 1)); bit >= 0; --bit) {
    const uint64_t set = __ballot(size >> bit & 1) & left;
    const int larger = __popcll(set);
    left &= k < larger ? set : ~set;
    if (k >= larger) k -= larger;
  }
  const int rank = __builtin_amdgcn_mbcnt_hi((uint32_t)(left >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)left, 0));
  const int at = __builtin_ctzll(__ballot((left >> lane & 1) && rank == k));
  first_slot = __builtin_amdgcn_readlane(own.begin / C + before + own.chunked_before, at);
  return __builtin_amdgcn_readfirstlane(base + at);
}

// LDS of the scan: a chunk's keys, scalars and T tiles twice (the next chunk's
// arrive while this one's are used); its queries and A tiles twice, or once
// under SPLIT, whose operands are twice as large. With ROLES also the chunk's v
// twice, and what the state's wave hands over (4 operands of S, 2 of U, scale
// and first bad token; SPLIT: once).
template <bool SPLIT, bool ROLES, int ES>
struct ScanLds {
  static constexpr int KEYS = (int)(plane_bytes(SPLIT) + kScalars + tri_bytes(SPLIT));
  static constexpr int QUERIES = (int)(plane_bytes(SPLIT) + tri_bytes(SPLIT));
  static constexpr int VALUES = ROLES ? C * 16 * ES : 0;
  static constexpr int HANDED = ROLES ? (SPLIT ? 13 : 7) * 1024 : 0;
  static constexpr int BUFS = SPLIT ? 1 : 2;  // of queries and of what is handed over
  static constexpr int QUERIES_AT = 2 * KEYS, VALUES_AT = QUERIES_AT + BUFS * QUERIES, HANDED_AT = VALUES_AT + 2 * VALUES;
  static constexpr int BYTES = HANDED_AT + BUFS * HANDED;
};

// A sequence's chunks in order. A wave has 16 V-rows of one value head, the
// columns (lane & 15) of every product, so what one product leaves in registers
// (rows k or t: 4 grp + j of a 16-row tile) is the next one's operand as it
// stands: both operands of a product may take its contraction in any order, and
// the keys', queries', T's and A's fragments are read in that one.
//
// The chain over the chunks is the state's: K S0^T, R, U, S1. The outputs hang
// off it. With ROLES (three waves a workgroup) one wave carries the chain and
// hands S0's and U's operands through LDS to a second one, which forms the
// outputs of chunk c while the first is at chunk c + 1; a third fetches what
// either reads (48 copies a chunk, whose issue alone costs a wave 850 cycles).
// Otherwise WAVES waves do all of it for 16 V-rows each on shared operands.
//
// Bound by the chain: 128 chunks of one sequence, HV=32, V=128, bf16 take 173 us,
// 1.35 a chunk (2600 cycles of the chain's wave: 240 vector instructions of 4
// cycles and 38 products of 16 one after the other, and the latencies between
// them; the outputs' wave has 1600 to do). With 8 waves a workgroup two waves a
// SIMD hide half of each other's latency: 3.7 us a chunk of 128 V-rows.
template <class Act, class St, bool SPLIT, int WAVES, bool ROLES>
__global__ __launch_bounds__(64 * WAVES) __attribute__((amdgpu_waves_per_eu(2, 2))) void chunk_scan_kernel(const PrefillArgs a) {
  constexpr int ES = Act::kBytes;
  using L = ScanLds<SPLIT, ROLES, ES>;
  constexpr int RS = 2 * K, COLS = ROLES ? 16 : 16 * WAVES;
  constexpr float kUp = SPLIT ? kFix : 1.f, kDown = 1.f / kUp;
  static_assert(!ROLES || WAVES == 3, "one wave a role");
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, grp = lane >> 4;
  const bool chain = !ROLES || wave == 0, outputs = !ROLES || wave == 1, fetches = !ROLES || wave == 2;
  // Workgroups go to the 8 XCDs in turn: those of one key head, which read the
  // same keys and queries, to one of them.
  int first_slot;
  const int blocks = a.V / COLS, n = longest_first(a, blockIdx.y, first_slot);
  if (n < 0) return;
  int unit_id = blockIdx.x;
  if (a.H % 8 == 0) {
    const int per = a.G * blocks, j = unit_id >> 3;
    unit_id = ((unit_id & 7) + 8 * (j / per)) * per + j % per;
  }
  const int hv = unit_id / blocks, h = hv / a.G;
  const int v0 = (unit_id - hv * blocks) * COLS + (ROLES ? 0 : wave * 16) + col;  // this lane's V-row
  int begin, end;
  sequence_rows(a, n, begin, end);
  const bool started = sequence_started(a, n);
  if (begin == end && started) return;
  const int len = end - begin, chunks = (len + C - 1) / C;
  const int64_t slot0 = a.N == 1 ? begin / C : first_slot;
  if (slot0 + chunks > chunk_slots(a.T, a.N, a.chunk_from)) return;  // (offsets that decrease)
  const uint8_t *unit, *head;  // of chunk 0
  const int64_t unit_step = a.H * unit_bytes(SPLIT), head_step = a.HV * head_bytes(SPLIT);
  {
    const Work w = work_of(a, SPLIT);
    unit = w.unit + slot0 * unit_step + h * unit_bytes(SPLIT);
    head = w.head + slot0 * head_step + hv * head_bytes(SPLIT);
  }

  // Operands from memory to LDS as they lie.
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_void_t*)lds;
  constexpr int kTeam = ROLES ? 1 : WAVES;  // waves that fetch a part
  const int member = ROLES ? 0 : wave;
  auto fetch_keys = [&](int c) {
    const uint32_t to = lds0 + (c & 1) * L::KEYS;
    dma_part<(int)plane_bytes(SPLIT) / 1024, kTeam>(unit + c * unit_step, to, member);
    dma_part<(int)(kScalars + tri_bytes(SPLIT)) / 1024, kTeam>(head + c * head_step, to + plane_bytes(SPLIT), member);
  };
  auto queries_at = [&](int c) { return L::QUERIES_AT + (c % L::BUFS) * L::QUERIES; };
  auto fetch_queries = [&](int c) {
    const uint32_t to = lds0 + queries_at(c);
    dma_part<(int)plane_bytes(SPLIT) / 1024, kTeam>(unit + c * unit_step + plane_bytes(SPLIT), to, member);
    dma_part<(int)tri_bytes(SPLIT) / 1024, kTeam>(head + c * head_step + kScalars + tri_bytes(SPLIT), to + plane_bytes(SPLIT), member);
  };
  // 16 tokens by 32 columns k of keys or queries at b
  auto rows_of = [&](const uint8_t* b, int tile, int step) {
    Operand<SPLIT> o;
    const uint8_t* p = b + (16 * tile + col) * RS + 16 * ((4 * step + grp) ^ col);
    o.hi = *(const u32x4_t*)p;
    if constexpr (SPLIT) o.lo = *(const u32x4_t*)(p + C * RS);
    return o;
  };
  auto triangle = [&](const uint8_t* tiles, int tt, int ts) {
    Operand<SPLIT> o;
    const uint8_t* p = tiles + tri(tt, ts) * 1024 + 16 * lane;
    o.hi = *(const u32x4_t*)p;
    if constexpr (SPLIT) o.lo = *(const u32x4_t*)(p + kTri * 1024);
    return o;
  };
  // The LDS operands of a product are read a stage or more before they are
  // used, which the fences keep the compiler from undoing: a read just before
  // its product costs its latency some 60 times a chunk.
  constexpr int AHEAD = SPLIT ? 1 : 2;  // k-steps of 4 fragments read before the first product
  Operand<SPLIT> f[AHEAD + 1][4], tf[kTri], bs[4], ub[2];
  auto read_rows = [&](const uint8_t* b, int s) {
#pragma unroll
    for (int tt = 0; tt < 4; ++tt) f[s % (AHEAD + 1)][tt] = rows_of(b, tt, s);
  };
  auto read_triangle = [&](const uint8_t* tiles) {
#pragma unroll
    for (int tt = 0; tt < 4; ++tt)
#pragma unroll
      for (int s = 0; s <= tt / 2; ++s) tf[tri(tt, s)] = triangle(tiles, tt, s);
  };
  auto by_state = [&](const uint8_t* b, f32x4_t(&x)[4]) {  // rows 0 .. AHEAD - 1 already asked for
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      if (s + AHEAD < 4) read_rows(b, s + AHEAD);
      GDNR_COMPILER_FENCE();
#pragma unroll
      for (int tt = 0; tt < 4; ++tt) x[tt] = product<SPLIT>(f[s % (AHEAD + 1)][tt], bs[s], s == 0 ? f32x4_t{0.f, 0.f, 0.f, 0.f} : x[tt]);
    }
  };
  auto by_triangle = [&](f32x4_t(&x)[4]) {
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int tt = 2 * s; tt < 4; ++tt) x[tt] = product<SPLIT>(tf[tri(tt, s)], ub[s], x[tt]);
  };

  // the state, transposed: tile kt of 16 columns k, rows 4 grp + j; times sc
  uint8_t* sp = (uint8_t*)a.state + ((int64_t)sequence_slot(a, n) * a.st_s + hv * a.st_h + (int64_t)v0 * a.st_v + 4 * grp) * St::kBytes;
  f32x4_t S[8];
  float sc = 1.f, inv = 1.f;
  typename Act::Bits vn[16];  // the next chunk's v: rows t of this lane, as raw bits
  const int64_t v_row = a.mx_t * ES, o_row = a.o_t * ES;
  const uint8_t* vp = (const uint8_t*)a.mixed + (int64_t)begin * v_row + (2 * a.H * K + hv * a.V) * ES;
  uint8_t* op = (uint8_t*)a.out + (int64_t)begin * o_row + hv * a.o_h * ES;
  const uint32_t v_lane = (uint32_t)(4 * grp * v_row) + v0 * ES, o_lane = (uint32_t)((4 * grp + (lane & 3)) * o_row) + (v0 & ~3) * ES;
  auto fetch_v = [&](int c) {
    const uint8_t* p = vp + c * C * v_row;
    if constexpr (ROLES) {  // rows of 16 V-rows' values, to LDS
#pragma unroll
      for (int i = 0; i < ES; ++i) {
        const int x = 64 * i + lane, t = x / ES;
        dma16(p + (uint32_t)min(t, len - 1 - c * C) * v_row + (v0 - col) * ES + 16 * (x % ES),
              lds0 + L::VALUES_AT + (c & 1) * L::VALUES + 1024 * i);
      }
    } else if ((c + 1) * C <= len) {
#pragma unroll
      for (int i = 0; i < 16; ++i) vn[i] = Act::ld_bits(p + (16 * (i >> 2) + (i & 3)) * v_row + v_lane, 0);
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) vn[i] = Act::ld_bits(p + (uint32_t)min(16 * (i >> 2) + (i & 3) + 4 * grp, len - 1 - c * C) * v_row + v0 * ES, 0);
    }
  };
  bool any_bad = false;
  int first = C;  // first token of the chunk whose results are NaN in this V-row
  bool by_token = false;  // the chunk's outputs are written already
  const float not_first = grp == 0 ? 0.f : __builtin_inff();

  // what is handed over: operands of S (0 .. 3) and U (4, 5), then scale and first
  // bad token; SPLIT: the operands' low halves after that
  auto place = [&](int c, int i) { return (u32x4_t*)(lds + L::HANDED_AT + (c % L::BUFS) * L::HANDED + 1024 * i + 16 * lane); };
  constexpr int kLow = 7;
  auto hand_over = [&](int c, int i, const Operand<SPLIT>& o) {
    *place(c, i) = o.hi;
    if constexpr (SPLIT) *place(c, kLow + i) = o.lo;
  };

  // A chunk token by token in f32, from its keys in LDS and its queries where the
  // preparation left them: the state and the outputs. (53 us a chunk, 106 SPLIT: for
  // rows that hold values of very different magnitude.)
  auto walk = [&](int c, const uint8_t* b, const float* scal) {
    const uint8_t* queries = unit + c * unit_step + plane_bytes(SPLIT);
    uint8_t* orow = op + c * C * o_row + (int64_t)v0 * ES;
    auto four = [](const uint8_t* p, float* x) {
      const uint2 w = *(const uint2*)p;
      const float2 lo = unpack_f16(w.x), hi = unpack_f16(w.y);
      x[0] = lo.x, x[1] = lo.y, x[2] = hi.x, x[3] = hi.y;
      if constexpr (SPLIT) {
        const uint2 u = *(const uint2*)(p + plane_bytes(false));
        const float2 l = unpack_f16(u.x), h = unpack_f16(u.y);
        x[0] = kDown * (x[0] + l.x), x[1] = kDown * (x[1] + l.y), x[2] = kDown * (x[2] + h.x), x[3] = kDown * (x[3] + h.y);
      }
    };
    auto total_of = [](float x) {  // over the lanes of a column
      x += __shfl_xor(x, 16);
      return x + __shfl_xor(x, 32);
    };
#pragma unroll
    for (int kt = 0; kt < 8; ++kt) S[kt] *= inv;
    sc = 1.f, inv = 1.f;
    const int count = min(C, len - c * C);
#pragma nounroll
    for (int t = 0; t < count; ++t) {
      float x;
      if constexpr (ROLES) x = Act::ld(lds + L::VALUES_AT + (c & 1) * L::VALUES + 16 * ES * t, col);
      else x = Act::ld(vp + (c * C + t) * v_row, v0);
      if (!finite(x)) x = 0.f;
      const float beta = scal[t], gamma = scal[5 * C + t];
      // (operands are read where they are used, four tiles at a time: kept over the
      // token they would cost the other path registers)
      float x4[4], sk = 0.f, o = 0.f;
#pragma unroll
      for (int kt = 0; kt < 8; ++kt) {
        if (kt % 4 == 0) GDNR_COMPILER_FENCE();
        four(b + unit_at(t, 4 * kt + grp), x4);
#pragma unroll
        for (int j = 0; j < 4; ++j) S[kt][j] *= gamma, sk = fmaf(S[kt][j], x4[j], sk);
      }
      const float u = beta * (x - total_of(sk));
#pragma unroll
      for (int kt = 0; kt < 8; ++kt) {
        if (kt % 4 == 0) GDNR_COMPILER_FENCE();
        four(b + unit_at(t, 4 * kt + grp), x4);
#pragma unroll
        for (int j = 0; j < 4; ++j) S[kt][j] = fmaf(u, x4[j], S[kt][j]);
        four(queries + unit_at(t, 4 * kt + grp), x4);
#pragma unroll
        for (int j = 0; j < 4; ++j) o = fmaf(S[kt][j], x4[j], o);
      }
      GDNR_COMPILER_FENCE();
      o = a.out_scale * total_of(o);
      if (grp == 0) Act::st(orow + t * o_row, 0, t >= first ? __builtin_nanf("") : o);
    }
    if (any_bad && first < C) {
#pragma unroll
      for (int kt = 0; kt < 8; ++kt) S[kt] = f32x4_t{1.f, 1.f, 1.f, 1.f} * __builtin_nanf("");
    }
  };

  // the chain: chunk c's R and U from S, then S after it
  auto state_step = [&](int c) {
    const uint8_t* b = lds + (c & 1) * L::KEYS;
    const float* scal = (const float*)(b + plane_bytes(SPLIT));
    const uint8_t* tiles = b + plane_bytes(SPLIT) + kScalars;
    const f32x4_t* beta4 = (const f32x4_t*)scal;
    const f32x4_t* held4 = (const f32x4_t*)(scal + C);
    const f32x4_t* end4 = (const f32x4_t*)(scal + 2 * C);
    auto turned = [&](int tile, int step) {  // 16 columns k of the keys by 32 tokens
      Operand<SPLIT> o;
      const int row = 4 * grp + (col >> 2);
      const uint8_t* p = b + 32 * step * RS + unit_at(row, 4 * tile + (col & 3));
      auto read = [](const uint8_t* q) { return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)q)); };
      const uint2 x = read(p), y = read(p + 16 * RS);
      o.hi = u32x4_t{x.x, x.y, y.x, y.y};
      if constexpr (SPLIT) {
        const uint2 z = read(p + C * RS), u = read(p + (C + 16) * RS);
        o.lo = u32x4_t{z.x, z.y, u.x, u.y};
      }
      return o;
    };
    const float total = scal[4 * C - 1];
    const int bad_token = __builtin_amdgcn_readfirstlane(((const int*)scal)[4 * C]);
    float v[4][4];
    if constexpr (ROLES) {
      const uint8_t* p = lds + L::VALUES_AT + (c & 1) * L::VALUES;
#pragma unroll
      for (int tt = 0; tt < 4; ++tt) {
        if constexpr (ES == 2) {
          const uint2 x = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 32 * (16 * tt + 4 * grp + (col >> 2)) + 8 * (col & 3))));
          const float2 lo = Act::from_pair(x.x), hi = Act::from_pair(x.y);
          v[tt][0] = lo.x, v[tt][1] = lo.y, v[tt][2] = hi.x, v[tt][3] = hi.y;
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) v[tt][j] = *(const float*)(p + 64 * (16 * tt + 4 * grp + j) + 4 * col);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i >> 2][i & 3] = Act::from_bits(vn[i]);
    }
    if (rare((c + 1) * C > len)) {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (c * C + 16 * (i >> 2) + 4 * grp + (i & 3) >= len) v[i >> 2][i & 3] = 0.f;
    }
    if constexpr (!ROLES) {
      if (SPLIT) fetch_queries(c);
      if (c + 1 < chunks) fetch_keys(c + 1), fetch_v(c + 1);
    }
#pragma unroll
    for (int s = 0; s < AHEAD; ++s) read_rows(b, s);
    GDNR_COMPILER_FENCE();

    // |S k| is at most |S| as a vector, and a token adds at most its v to that, at a
    // right angle or less: |R| and |U| are at most 10 times the bound. A row's f16
    // operands are off by some 2^-33 of it. Where a token that is much smaller may need
    // what that rounds off, the chunk is walked token by token: a later token's v, or a
    // state that has decayed meanwhile, must not cost it its bits. That needs four tokens
    // that are all that small, or one of the chunk's first (SPLIT: in four rows).
    constexpr float kSmall = SPLIT ? 0x1p-9f : 0x1p-18f;
    float bound, state_part, least;
    auto of_four_rows = [](float x) {
      x = __builtin_fabsf(x);
      x = fmaxf(x, dpp_f<kDppXor1>(x));
      return fmaxf(x, dpp_f<kDppXor2>(x));
    };
    auto largest = [&]() {
      float x = 0.f, x2 = 0.f, y[4];
#pragma unroll
      for (int kt = 0; kt < 8; ++kt) x = max3_abs(x, S[kt][0], S[kt][1]), x2 = max3_abs(x2, S[kt][2], S[kt][3]);
#pragma unroll
      for (int tt = 0; tt < 4; ++tt) y[tt] = max3_abs(max3_abs(0.f, v[tt][0], v[tt][1]), v[tt][2], v[tt][3]);
      if constexpr (SPLIT) least = fminf(fminf(of_four_rows(v[0][0]), of_four_rows(v[0][1])), of_four_rows(v[0][2]));
      else least = fminf(fminf(__builtin_fabsf(v[0][0]), __builtin_fabsf(v[0][1])), __builtin_fabsf(v[0][2]));
      least = fminf(fmaxf(least, not_first), y[0]);
      least = fminf(fminf(fminf(least, 0x1p127f), y[1]), fminf(y[2], y[3]));
      state_part = 12.f * inv * __builtin_elementwise_maximum(x, x2);
      bound = column_max(max3_abs(max3_abs(state_part, y[0], y[1]), y[2], y[3]));
    };
    largest();
    first = C;
    any_bad = by_token = false;
    if (rare(bad_token < C || __ballot(!(least >= kSmall * bound)) != 0)) {
      // V-rows with a value that is not finite (the bound then neither): zeros here, NaN
      // from its token on
      any_bad = bad_token < C || __ballot(!finite(bound)) != 0;
      float at = C;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float& x = v[i >> 2][i & 3];
        if (!finite(x)) at = fminf(at, (float)(16 * (i >> 2) + 4 * grp + (i & 3))), x = 0.f;
      }
#pragma unroll
      for (int kt = 0; kt < 8; ++kt)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (!finite(S[kt][j])) S[kt][j] = 0.f, at = 0.f;
      first = min(C - (int)column_max(C - at), bad_token);
      largest();
      // a row is safe where what it starts with, decayed by the whole chunk, is not
      // small; or where no token's v of it and its three neighbours is
      const float start = fmaxf(state_part, grp == 0 ? __builtin_fabsf(v[0][0]) : 0.f);
      const uint64_t safe = __ballot(total * start >= kSmall * bound);
      least = __builtin_inff();
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float x = of_four_rows(v[i >> 2][i & 3]);
        if (c * C + 16 * (i >> 2) + 4 * grp + (i & 3) < len) least = fminf(least, x);
      }
      least = -column_max(-least);
      by_token = !all_columns(safe | __ballot(least >= kSmall * bound));
      if (by_token) {
        walk(c, b, scal);
        if constexpr (ROLES) *place(c, 6) = u32x4_t{0, 0, 0, 1};
        return;
      }
    }
    // Each row's power of two puts its bound between 2^8 and 2^12. It stays what
    // it was while it does: then nothing is rescaled.
    float ratio = 1.f;
    const float scaled = bound * sc;
    if (!(scaled < 0x1p12f && scaled >= 0x1p8f)) {
      const uint32_t ex = min(max((__float_as_uint(bound) >> 23) + 3, 21u), 257u);
      const float s_new = __uint_as_float((268u - ex) << 23);
      ratio = fminf(s_new * inv, 0x1p126f);
      sc = s_new, inv = __uint_as_float((ex - 14u) << 23);
    }
    if (__any(ratio != 1.f)) {
#pragma unroll
      for (int kt = 0; kt < 8; ++kt) S[kt] *= ratio;
    }
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      bs[s] = operand<SPLIT>(S[2 * s], S[2 * s + 1]);
      if constexpr (ROLES) hand_over(c, s, bs[s]);
    }
    if constexpr (ROLES) *place(c, 6) = u32x4_t{__float_as_uint(inv), (uint32_t)first, any_bad, by_token};

    f32x4_t u[4];
    by_state(b, u);  // K S0^T
    GDNR_COMPILER_FENCE();
    f32x4_t be[4], bg[4], ed[4];
#pragma unroll
    for (int tt = 0; tt < 4; ++tt) be[tt] = beta4[4 * tt + grp], bg[tt] = held4[4 * tt + grp];
    if constexpr (!SPLIT) read_triangle(tiles);
    GDNR_COMPILER_FENCE();
    // R = beta (v - e^G (K S0^T))
#pragma unroll
    for (int tt = 0; tt < 4; ++tt)
#pragma unroll
      for (int j = 0; j < 4; ++j) u[tt][j] = fmaf(bg[tt][j], u[tt][j], be[tt][j] * (v[tt][j] * sc));
#pragma unroll
    for (int s = 0; s < 2; ++s) ub[s] = operand<SPLIT>(u[2 * s], u[2 * s + 1]);
    constexpr int KT = SPLIT ? 2 : 4;  // tiles of the keys read ahead
    Operand<SPLIT> kf[2][KT];
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) kf[0][kt] = turned(kt, 0);
#pragma unroll
    for (int tt = 0; tt < 4; ++tt) ed[tt] = end4[4 * tt + grp];
    GDNR_COMPILER_FENCE();
    // U = R + (T - I) R
    if constexpr (SPLIT) {
      read_triangle(tiles);
#pragma unroll
      for (int tt = 0; tt < 4; ++tt) u[tt] *= kUp;
    }
    by_triangle(u);
#pragma unroll
    for (int kt = 0; kt < 8; ++kt) S[kt] *= total * kUp;
    Operand<SPLIT> ud[2];
    if constexpr (SPLIT) {
#pragma unroll
      for (int tt = 0; tt < 4; ++tt) u[tt] *= kDown;
    }
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      ud[s] = operand<SPLIT>(u[2 * s] * ed[2 * s], u[2 * s + 1] * ed[2 * s + 1]);
      ub[s] = operand<SPLIT>(u[2 * s], u[2 * s + 1]);
      if constexpr (ROLES) hand_over(c, 4 + s, ub[s]);
    }
    // the state after the chunk, KT tiles of one half of the tokens at a time
#pragma unroll
    for (int i = 0; i < 16 / KT; ++i) {
      if (i + 1 < 16 / KT) {
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) kf[(i + 1) & 1][kt] = turned(((i + 1) * KT + kt) % 8, (i + 1) * KT / 8);
      }
      GDNR_COMPILER_FENCE();
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
        f32x4_t& x = S[(i * KT + kt) % 8];
        x = product<SPLIT>(kf[i & 1][kt], ud[i * KT / 8], x);
      }
    }
    if constexpr (SPLIT) {
#pragma unroll
      for (int kt = 0; kt < 8; ++kt) S[kt] *= kDown;
    }
    if (rare(any_bad) && first < C) {
#pragma unroll
      for (int kt = 0; kt < 8; ++kt) S[kt] = f32x4_t{1.f, 1.f, 1.f, 1.f} * __builtin_nanf("");
    }
  };

  // the outputs of chunk c from bs, ub, inv, first, any_bad and e^G (gr)
  f32x4_t gr[4];
  auto read_grow = [&](int c) {
    const f32x4_t* grow4 = (const f32x4_t*)(lds + (c & 1) * L::KEYS + plane_bytes(SPLIT) + 3 * C * 4);
#pragma unroll
    for (int tt = 0; tt < 4; ++tt) gr[tt] = grow4[4 * tt + grp];
  };
  auto output_step = [&](int c) {
    const uint8_t* b = lds + queries_at(c);
#pragma unroll
    for (int s = 0; s < AHEAD; ++s) read_rows(b, s);
    f32x4_t o[4];
    if constexpr (!ROLES) read_grow(c);
    GDNR_COMPILER_FENCE();
    if constexpr (!SPLIT) read_triangle(b + plane_bytes(SPLIT));
    by_state(b, o);  // Q S0^T
    if constexpr (SPLIT) read_triangle(b + plane_bytes(SPLIT));
#pragma unroll
    for (int tt = 0; tt < 4; ++tt) o[tt] *= gr[tt];
    by_triangle(o);
    const float scale = kDown * a.out_scale * inv;
#pragma unroll
    for (int tt = 0; tt < 4; ++tt) o[tt] *= scale;
    if (rare(any_bad)) {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (16 * (i >> 2) + 4 * grp + (i & 3) >= first) o[i >> 2][i & 3] = __builtin_nanf("");
    }
    // (what is on its way to LDS is waited for before the stores, which then
    // have a whole chunk to drain)
    if constexpr (!ROLES) {
      GDNR_WAIT_VMCNT(0);
    } else if (L::BUFS == 1 && c + 1 < chunks) {
      GDNR_WAIT_LGKM0();  // (this chunk's have been read)
      fetch_queries(c + 1);
      GDNR_WAIT_VMCNT(0);
    }
    uint8_t* orow = op + c * C * o_row + o_lane;
#pragma unroll
    for (int tt = 0; tt < 4; ++tt)
      store_turned<Act>(orow + 16 * tt * o_row, o[tt], lane, !by_token && c * C + 16 * tt + 4 * grp + (lane & 3) < len);
  };

  if (chain) {
#pragma unroll
    for (int kt = 0; kt < 8; ++kt) {
      Raw<St, 4> x;
      if (started) x.load(sp + 16 * kt * St::kBytes);
#pragma unroll
      for (int j = 0; j < 4; ++j) S[kt][j] = started ? x[j] : 0.f;
    }
  }
  if (fetches && chunks) {
    fetch_keys(0), fetch_v(0);
    if (!ROLES && !SPLIT) fetch_queries(0);
  }
  GDNR_WAIT_VMCNT(0);
  if constexpr (ROLES) {
    for (int c = 0; c <= chunks; ++c) {
      __syncthreads();  // chunk c's keys and v are in LDS, chunk c - 1 is handed over
      if (outputs) {
        if (c > 0) {
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            bs[s].hi = *place(c - 1, s);
            if constexpr (SPLIT) bs[s].lo = *place(c - 1, kLow + s);
          }
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            ub[s].hi = *place(c - 1, 4 + s);
            if constexpr (SPLIT) ub[s].lo = *place(c - 1, kLow + 4 + s);
          }
          const u32x4_t x = *place(c - 1, 6);
          inv = __uint_as_float(x[0]), first = (int)x[1], any_bad = __builtin_amdgcn_readfirstlane(x[2]) != 0;
          by_token = __builtin_amdgcn_readfirstlane(x[3]) != 0;
        }
        if (L::BUFS == 1 && c == 0 && chunks) fetch_queries(0);
      }
      if constexpr (L::BUFS == 1) __syncthreads();  // what was handed over is in registers
      if (chain && c < chunks) {
        state_step(c);
      }
      if (outputs) {
        if (c > 0) output_step(c - 1);
        else GDNR_WAIT_VMCNT(0);
        if (c < chunks) read_grow(c);
      }
      if (fetches) {
        if (c + 1 < chunks) fetch_keys(c + 1), fetch_v(c + 1);
        if (L::BUFS == 2 && c < chunks) fetch_queries(c);
        GDNR_WAIT_VMCNT(0);
      }
    }
  } else {
    for (int c = 0; c < chunks; ++c) {
      // chunk c's operands are in LDS (every wave waited for its part), those of
      // c - 1 are no longer read
      __syncthreads();
      if (!SPLIT && c + 1 < chunks) fetch_queries(c + 1);
      state_step(c);
      if constexpr (SPLIT) {  // the one buffer of queries was filled meanwhile
        GDNR_WAIT_VMCNT(0);
        __syncthreads();
      }
      output_step(c);
    }
  }
  if (chain) {
#pragma unroll
    for (int kt = 0; kt < 8; ++kt)
#pragma unroll
      for (int j = 0; j < 4; j += 2) St::st2(sp + (16 * kt + j) * St::kBytes, S[kt][j] * inv, S[kt][j + 1] * inv);
  }
}

// Whether results keep more than bf16 does.
bool needs_split(int act_dt, int state_dt) { return act_dt != DT_BF16 || state_dt != DT_BF16; }

// Which sequences are walked in chunks (PrefillArgs::chunk_from). The host knows
// their number and the sum of their tokens. All of them from an average of 16
// tokens a sequence on (SPLIT: 32). us a call, token by token and in chunks, HV=32,
// V=128, bf16: one sequence of 16 tokens 14.9 and 16.8, of 24 20.0 and 16.5; 64
// sequences of 8 72 and 109, of 16 125 and 109; f16 with an f32 state, 4 sequences of
// 32 25.6 and 28.3, of 64 46 and 29. Below that a batch may still hold a long one
// beside many short: from kLongWalk tokens in all, those of a chunk and more are
// walked in chunks and the others token by token. us a call, all token by token and
// so, bf16: 900 tokens beside 63 single ones 598 and 104, 120 beside 15 85 and 31;
// where none is long the kernels with nothing to do cost 4: 16 sequences of 12
// tokens 29 and 33, 64 of 8 70 and 72.
constexpr int kLongWalk = 128;
int32_t chunk_start(int64_t T, int64_t N, bool split) {
  if (T >= (split ? 32 : 16) * N) return 0;
  return T >= kLongWalk ? C : INT32_MAX;
}

// A workgroup takes a key head's value heads two after two; while that leaves
// compute units idle each two have one of their own, which forms the keys' part
// again (26 chunks of 4 key heads and 12 value heads, f16 with an f32 state: 20.5
// us in one part, 16.5 in two).
template <class Act, bool GATE_F32, bool SPLIT>
int launch_prep(const PrefillArgs& a, hipStream_t s) {
  const int64_t chunks = chunk_slots(a.T, a.N, a.chunk_from);
  const uint32_t parts = chunks * a.H < device_cus() ? (a.G + 1) / 2 : 1;
  hipLaunchKernelGGL((chunk_prep_kernel<Act, GATE_F32, SPLIT>), dim3((uint32_t)chunks, a.H, parts), dim3(256), 0, s, a);
  return (int)hipGetLastError();
}
// sequences that the scan has places for
int places(const PrefillArgs& a) {
  const int most = (int)std::min<int64_t>(chunked_most(a.T, a.N, a.chunk_from), 64);
  return a.N / 64 * most + std::min(a.N % 64, most);
}
template <class Act, class St, bool SPLIT, int WAVES, bool ROLES>
int launch_scan_as(const PrefillArgs& a, hipStream_t s) {
  constexpr int lds = ScanLds<SPLIT, ROLES, Act::kBytes>::BYTES;
  static_assert(lds <= kMaxStepLds, "the operands fit");
  const auto kernel = chunk_scan_kernel<Act, St, SPLIT, WAVES, ROLES>;
  const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  if (e != hipSuccess) return (int)e;
  hipLaunchKernelGGL(kernel, dim3(a.HV * (a.V / (ROLES ? 16 : 16 * WAVES)), places(a)), dim3(64 * WAVES), lds, s, a);
  return (int)hipGetLastError();
}
// A workgroup's LDS leaves room for one on a compute unit, so the scan's time is
// the rounds its workgroups take over the card times what a chunk costs them:
// with 8 waves (128 V-rows) 3.7 us, 4 waves 2.8, the three roles (16 V-rows) 1.4;
// with SPLIT operands 7.0, 5.0 and 3.3, and with 2 waves (32 V-rows) 4.7. The
// cheapest product runs, the wider one of equals (it reads the operands once for
// more rows). us a call of 1024 tokens a sequence, HV=32, V=128, with 8 waves, 4
// and the roles: 1 sequence 78, 62 and 47; 2: 80, 65 and 73; 4: 88, 75 and 124;
// 6: 109, 133 and 186; 8: 127, 147 and 238. f16 with an f32 state, HV=12, 512
// tokens a sequence, with 4 waves, 2 and the roles: 1 sequence 63, 59 and 46; 4:
// 67, 65 and 71; 16: 137, 164 and 185, with 8 waves 105.
template <class Act, class St, bool SPLIT>
int launch_scan(const PrefillArgs& a, hipStream_t s) {
  const int64_t rows = (int64_t)places(a) * a.HV * a.V, cus = device_cus();
  const auto cost = [&](int columns, int chunk) {
    return a.V % columns ? INT64_MAX : (rows / columns + cus - 1) / cus * chunk;
  };
  const int64_t eight = cost(128, SPLIT ? 70 : 37), four = cost(64, SPLIT ? 50 : 28), one = cost(16, SPLIT ? 33 : 14);
  if constexpr (SPLIT) {
    const int64_t two = cost(32, 47);
    if (two <= one && two < four && two < eight) return launch_scan_as<Act, St, SPLIT, 2, false>(a, s);
  }
  if (eight <= four && eight <= one) return launch_scan_as<Act, St, SPLIT, 8, false>(a, s);
  if (four <= one) return launch_scan_as<Act, St, SPLIT, 4, false>(a, s);
  return launch_scan_as<Act, St, SPLIT, 3, true>(a, s);
}

template <class Act, class St, bool GATE_F32>
int launch_recurrent(const PrefillArgs& a, hipStream_t s) {
  const int units = a.HV * (a.V / kRecRows);
  hipLaunchKernelGGL((recurrent_kernel<Act, St, GATE_F32>), dim3((units + 3) / 4, a.N), dim3(256), 0, s, a);
  return (int)hipGetLastError();
}

template <class Act, class St, bool GATE_F32>
int launch_forms(const PrefillArgs& a, hipStream_t s) {
  constexpr bool SPLIT = !(std::is_same<Act, ActBF16>::value && std::is_same<St, ActBF16>::value);
  int rc = a.chunk_from ? launch_recurrent<Act, St, GATE_F32>(a, s) : 0;
  if (rc || a.chunk_from == INT32_MAX) return rc;
  rc = launch_prep<Act, GATE_F32, SPLIT>(a, s);
  return rc ? rc : launch_scan<Act, St, SPLIT>(a, s);
}
template <class Act, bool GATE_F32>
int launch_state(const PrefillArgs& a, int state_dt, hipStream_t s) {
  if (state_dt == DT_BF16) return launch_forms<Act, ActBF16, GATE_F32>(a, s);
  if (state_dt == DT_F16) return launch_forms<Act, ActF16, GATE_F32>(a, s);
  return launch_forms<Act, ActF32, GATE_F32>(a, s);
}

}  // namespace

int64_t prefill_work_bytes(int64_t T, int64_t N, int32_t H, int32_t HV, int act_dt, int state_dt) {
  const bool split = needs_split(act_dt, state_dt);
  const int32_t from = chunk_start(T, N, split);
  return from == INT32_MAX ? 0 : chunk_slots(T, N, from) * (H * unit_bytes(split) + HV * head_bytes(split));
}

int launch_prefill(const PrefillArgs& args, int state_dt, int act_dt, bool gate_f32, void* stream) {
  PrefillArgs a = args;
  a.chunk_from = chunk_start(a.T, a.N, needs_split(act_dt, state_dt));
  hipStream_t s = (hipStream_t)stream;
  if (act_dt == DT_F32) return launch_state<ActF32, true>(a, state_dt, s);
  if (act_dt == DT_BF16) return gate_f32 ? launch_state<ActBF16, true>(a, state_dt, s) : launch_state<ActBF16, false>(a, state_dt, s);
  return gate_f32 ? launch_state<ActF16, true>(a, state_dt, s) : launch_state<ActF16, false>(a, state_dt, s);
}

}  // namespace gdnr
