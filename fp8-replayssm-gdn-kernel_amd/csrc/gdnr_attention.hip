// gdnr_attention.hip -- attention of new tokens over a paged cache, causal:
// token j of a sequence of L new tokens whose context holds C keys (the new
// ones last) sees the keys i <= C - L + j,
//   o = sum_i p_i v_i / sum_i p_i,  p_i = exp(scale q k_i - max);
// a row that sees no key gives 0. Heads are grouped: query head h reads the
// keys of head h / G.
//
// One pass over the keys with a running reference near the maximum and sums (f32). The rows of a
// workgroup are the (token, query head of the group) pairs of one key head, so
// the keys of a group are read once. The scores are formed transposed,
// K (keys x D) by Q^T: a lane then holds 8 keys of one row, which is, as it
// stands, the operand of V^T (D x keys) by P^T -- the contraction may take the
// keys in any order as long as both operands do. V passes through LDS, where
// the transposing read turns it.
//
// few_kernel: sequences of up to 16 rows (a decoded token of a group of up to
// 16 heads). Bound by the cache's bytes: 16 rows a workgroup, whose four waves
// take 32 keys each in turn, and long contexts in pieces. 64 decodes over up to
// 8192 keys, heads of 256: 144 us, 4.4 TB/s (0.88 of a copy's rate); one decode
// over 8192 keys 8.5 us, the chain lengths -> pages -> keys -> values.
// tile_kernel: the others. Bound by the matrix products and the exponentials:
// 128 rows a workgroup (64 at D = 256), 32 (16) a wave, all on the same keys.
// 2048 tokens over 8192 keys, 32 heads of 128: 248 us, 969 TFLOP/s (a square
// product of 8192 in the library: 1130); 32 of 64 159 us, 757; 16 of 256 320, 752.
// A context is cut into pieces where the rows alone do not fill the card, and
// join_kernel adds the pieces in their order.
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
constexpr int kKeys = 32;     // few_kernel: keys of a wave's step
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
// 16 x 32 ones: their product with rounded weights is the weights' sum, in every
// row of the result
template <class Act>
__device__ __forceinline__ u32x4_t ones() {
  constexpr uint32_t kOne = std::is_same<Act, ActBF16>::value ? 0x3F803F80u : 0x3C003C00u;
  return u32x4_t{kOne, kOne, kOne, kOne};
}
// 4 rows (keys) x 16 columns at p (row stride in bytes), transposed: lane i of
// each 16-lane group receives column i of the group's 4 rows
__device__ __forceinline__ uint2 transposed4(const uint8_t* p) {
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p));
}
// A weight is 2^(score - reference). f16 has all its bits down to 2^-14 alone,
// and a long tail of small weights under one large key is what the output consists of
// where that key's value is 0: there the reference lies kHead below the
// maximum that it was taken from, so that a weight that is 2^-25 of the largest keeps
// all its bits and one of 2^-36 still counts. kLag: how far tile_kernel's scores
// may pass that maximum before the reference follows; 2^(kHead + kLag + 1/2) fits
// the type. (With a lag of 8 and no head, thousands of keys 18 below one whose value
// is 0 gave outputs off by 0.7 to 6.7%; f16 rounds to 0.02%.) bf16 has f32's exponents.
template <class Act>
constexpr bool is_f16() { return !std::is_same<Act, ActBF16>::value; }
template <class Act>
constexpr float kHead = is_f16<Act>() ? 11.f : 0.f;
template <class Act>
constexpr float kLag = is_f16<Act>() ? 4.f : 8.f;
// whether a maximum has passed the reference's own by more than lag (a
// difference: exact where they are large)
template <class Act>
__device__ __forceinline__ bool passed(float top, float reference, float lag) {
  if constexpr (is_f16<Act>()) return top - reference > kHead<Act> + lag;
  else return top > reference + lag;
}
// the reference of a maximum (where top is so large that its neighbours are
// further apart than that: itself)
template <class Act>
__device__ __forceinline__ float reference(float top) {
  if constexpr (!is_f16<Act>()) return top;
  const float r = top - kHead<Act>;
  return top - r > kHead<Act> + 0.5f ? top : r;
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
  const uint32_t b = __float_as_uint(x);
  const auto half = __builtin_amdgcn_permlane32_swap(b, b, false, false);
  const uint32_t h = __float_as_uint(fmaxf(__uint_as_float(half[0]), __uint_as_float(half[1])));
  const auto row = __builtin_amdgcn_permlane16_swap(h, h, false, false);
  return fmaxf(__uint_as_float(row[0]), __uint_as_float(row[1]));
}
// x *= f, x += d and x += a b in the registers where x lies: of the two sides of a
// branch, the one that leaves x alone then has nothing to copy
__device__ __forceinline__ void scale_in_place(f32x4_t& x, float f) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float y = x[i];
    asm volatile("v_mul_f32 %0, %1, %0" : "+v"(y) : "v"(f));
    x[i] = y;
  }
}
__device__ __forceinline__ void shift_in_place(f32x4_t& x, float d) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float y = x[i];
    asm volatile("v_add_f32 %0, %1, %0" : "+v"(y) : "v"(d));
    x[i] = y;
  }
}
__device__ __forceinline__ void add_in_place(f32x4_t& x, float a, f32x4_t b) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float y = x[i];
    asm volatile("v_fmac_f32 %0, %1, %2" : "+v"(y) : "v"(a), "v"(b[i]));
    x[i] = y;
  }
}
// page and offset of a key (1 / page is off by a rounding: by at most one page)
__device__ __forceinline__ void page_of(int key, int page, double inv_page, int& p, int& r) {
  p = (int)((double)key * inv_page), r = key - p * page;
  if (r < 0) --p, r += page;
  if (r >= page) ++p, r -= page;
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

struct Block {  // a workgroup's place in its kernel's grid, or that grid
  int x, y, z;
};
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
// whether few_kernel takes the sequence (tile_kernel otherwise)
__device__ __forceinline__ bool few_rows(const AttentionArgs& a, const Span& s) {
  return (int64_t)(s.end - s.begin) * min(a.G, kRows) <= a.few_rows;
}
// place of token t among the pieces of its kind (0: few rows)
__device__ __forceinline__ int64_t piece_row(const AttentionArgs& a, int kind, int n, const Span& s, int t) {
  return kind == 0 && a.few_rows == kRows ? (int64_t)n * (kRows / min(a.G, kRows)) + (t - s.begin) : t;
}
// keys that token t of the sequence sees
__device__ __forceinline__ int visible(const Span& s, int t) { return min(max(s.context - s.end + t + 1, 0), s.context); }

// 16-byte piece p of row r of a tile of D-element rows in LDS lies at p ^ key:
// 16 rows' pieces then fall on distinct banks (rows of 128 bytes lie two to a
// bank window)
template <int D>
__device__ __forceinline__ int row_key(int r) { return D == 64 ? (r >> 1) & 7 : r & 15; }

template <int D>
constexpr int o_stride() { return 4 * D + 16; }
template <int D>
constexpr int lds_bytes() {
  const int v = kWaves * kKeys * 2 * D, o = kWaves * kRows * o_stride<D>();
  return (v > o ? v : o) + kWaves * kRows * 8;
}

// A wave's step: its keys' scores from registers (a lane holds whole pieces of
// two keys' rows, as the product takes them), its values from its part of the
// LDS. The next step's keys are asked for once the scores have used this one's,
// its values once the outputs have; two to four workgroups a compute unit
// cover the waits.
template <class Act, int D>
__device__ __forceinline__ void few_step(const AttentionArgs& a, uint8_t* lds, const Block blk) {
  constexpr int KSTEPS = D / 32, DT = D / 16, PPR = D / 8, RPI = 64 / PPR, NV = kKeys / RPI;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, grp = lane >> 4;
  const int gt = min(a.G, kRows), tb = kRows / gt;  // heads and tokens of a tile
  // beside tile_kernel, one tile holds all rows of each sequence that is taken here
  int n = blk.y;
  if (a.few_rows > kRows) n = sequences_up_to(a, n, tb, 1) - 1;
  if (n < 0) return;
  const Span sq = span_of(a, n);
  const int tok0 = a.few_rows > kRows ? sq.begin + (blk.y - sq.begin / tb - n) * tb : sq.begin;
  if (tok0 >= sq.end || !few_rows(a, sq)) return;
  const int head_tiles = (a.G + kRows - 1) / kRows;
  const int hk = blk.x / head_tiles, ht = blk.x - hk * head_tiles;
  const int last = min(tok0 + tb, sq.end) - 1;
  const int piece = a.piece[0], pieces = a.pieces[0];
  const int k_begin = blk.z * piece, k_end = min(visible(sq, last), k_begin + piece);
  if (k_begin >= k_end && (pieces > 1 || blk.z > 0)) return;

  // this lane's row
  const int rt = tok0 + col / gt, rh = ht * kRows + col % gt;
  const bool live = col / gt < tb && rt < sq.end && rh < a.G;
  const int vis = live ? min(visible(sq, rt), k_end) : 0;
  const int vis_all = min(visible(sq, tok0), k_end);  // every live row sees these
  u32x4_t q[KSTEPS];
  {
    const uint8_t* qp = (const uint8_t*)a.q + (rt * a.q_t + (hk * a.G + rh) * a.q_h) * 2 + 16 * grp;
#pragma unroll
    for (int i = 0; i < KSTEPS; ++i) q[i] = live ? *(const u32x4_t*)(qp + 64 * i) : u32x4_t{0, 0, 0, 0};
  }

  uint8_t* vt = lds + wave * kKeys * 2 * D;
  const uint32_t vt_lds = (uint32_t)(uintptr_t)(lds_void_t*)vt;
  const double inv_page = 1.0 / a.page;
  const int32_t* table = a.table + n * a.tb_n;
  const uint8_t* kbase = (const uint8_t*)a.k_cache + hk * a.kc_h * 2 + 16 * grp;
  const uint8_t* vbase = (const uint8_t*)a.v_cache + hk * a.vc_h * 2;
  const uint32_t k_page = (uint32_t)(a.kc_p >> 3), k_tok = (uint32_t)(a.kc_t >> 3);
  const uint32_t v_page = (uint32_t)(a.vc_p >> 3), v_tok = (uint32_t)(a.vc_t >> 3);
  // rows of a step's keys, in 16-byte units from the caches' bases: lane l
  // finds key l & 31's page a step before its rows are asked for
  int pg = 0, off = 0;
  auto find_rows = [&](int key0) {
    int p;
    page_of(min(key0 + (lane & 31), k_end - 1), a.page, inv_page, p, off);
    pg = table[p];
  };
  uint32_t k_row, v_row;
  u32x4_t kf[2][KSTEPS];
  auto load_keys = [&]() {
    const uint32_t at = min(max(pg, 0), a.n_pages - 1);
    k_row = at * k_page + off * k_tok, v_row = at * v_page + off * v_tok;
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      const uint8_t* p = kbase + (uint64_t)(uint32_t)__shfl((int)k_row, 16 * m + col) * 16;
#pragma unroll
      for (int i = 0; i < KSTEPS; ++i) kf[m][i] = *(const u32x4_t*)(p + 64 * i);
    }
  };
  auto copy_values = [&]() {
    uint32_t vr[NV];
    int sub = lane / PPR;
    asm volatile("" : "+v"(sub));  // (places formed here, not kept)
#pragma unroll
    for (int i = 0; i < NV; ++i) vr[i] = (uint32_t)__shfl((int)v_row, i * RPI + sub);
    GDNR_COMPILER_FENCE();
#pragma unroll
    for (int i = 0; i < NV; ++i)
      dma16(vbase + (vr[i] + (uint64_t)((lane % PPR) ^ row_key<D>(i * RPI + sub))) * 16, vt_lds + i * 1024);
  };

  f32x4_t o[DT];
#pragma unroll
  for (int i = 0; i < DT; ++i) o[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  float m_run = -__builtin_inff();         // the reference
  f32x4_t l_run = {0.f, 0.f, 0.f, 0.f};  // (every row of it)
  constexpr int STEP = kWaves * kKeys;
  int key0 = k_begin + wave * kKeys;
  if (key0 < k_end) {
    find_rows(key0);
    load_keys();
    copy_values();
    find_rows(key0 + STEP);
  }
  // one step; MASKED: some of its keys are not seen by every row
  auto step = [&](auto tag) {
    constexpr bool MASKED = decltype(tag)::value;
    const bool more = key0 + STEP < k_end;
    f32x4_t s[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int i = 0; i < KSTEPS; ++i)
#pragma unroll
      for (int m = 0; m < 2; ++m) s[m] = mfma<Act>(kf[m][i], q[i], s[m]);
    GDNR_WAIT_VMCNT(0);  // the step's values are in LDS
    if (more) {
      load_keys();
      find_rows(key0 + 2 * STEP);
    }
    float x[8], top = -__builtin_inff();
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[e] = s[e >> 2][e & 3] * a.scale_log2;
      if (MASKED && key0 + 16 * (e >> 2) + 4 * grp + (e & 3) >= vis) x[e] = -__builtin_inff();
      top = fmaxf(top, x[e]);
    }
    top = column_max(top);
    if (__any(passed<Act>(top, m_run, 0.f))) {
      const float m_new = fmaxf(m_run, reference<Act>(top));
      const float f = m_new == -__builtin_inff() ? 1.f : __builtin_amdgcn_exp2f(m_run - m_new);
      scale_in_place(l_run, f);
#pragma unroll
      for (int i = 0; i < DT; ++i) scale_in_place(o[i], f);
      m_run = m_new;
    }
    const float base = m_run == -__builtin_inff() ? 0.f : m_run;
    float p[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) p[e] = __builtin_amdgcn_exp2f(x[e] - base);
    bool bad = false;
    if constexpr (MASKED) {
#pragma nounroll
      for (int i = lane; i < kKeys * PPR; i += 64) bad |= nonfinite8<Act>(*(const u32x4_t*)(vt + 16 * i));
      bad = __any(bad);
      if (bad) {
        // a value that some rows must not see is infinite or NaN, and a product
        // with its weight 0 would show it to them: this step key by key
#pragma nounroll
        for (int key = 0; key < kKeys; ++key) {
          float pk = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (4 * (key >> 4) + (key & 3) == e) pk = p[e];
          pk = __shfl(pk, col + 16 * ((key >> 2) & 3));
          const uint32_t seen = key0 + key < vis ? ~0u : 0u;
          shift_in_place(l_run, pk);
#pragma unroll
          for (int i = 0; i < DT; ++i) {
            const uint2 w = *(const uint2*)(vt + key * 2 * D + 16 * ((2 * i + (grp >> 1)) ^ row_key<D>(key)) + 8 * (grp & 1));
            const float2 lo = Act::from_pair(w.x & seen), hi = Act::from_pair(w.y & seen);
            add_in_place(o[i], pk, f32x4_t{lo.x, lo.y, hi.x, hi.y});
          }
        }
      }
    }
    if (!bad) {
      // (the weights are rounded to the cache's type, which costs the output
      // about its own rounding; their sum is of the rounded ones, so that a row
      // that one key rules loses nothing)
      const u32x4_t pf = {pack2<Act>(p[0], p[1]), pack2<Act>(p[2], p[3]), pack2<Act>(p[4], p[5]), pack2<Act>(p[6], p[7])};
      l_run = mfma<Act>(ones<Act>(), pf, l_run);
      uint32_t v_key = row_key<D>(4 * grp + (col >> 2)) ^ ((col & 3) >> 1);
      asm volatile("" : "+v"(v_key));  // (addresses formed here, not kept)
      const uint8_t* vl = vt + (4 * grp + (col >> 2)) * 2 * D + 8 * (col & 1);
#pragma unroll
      for (int i0 = 0; i0 < DT; i0 += 4) {
        uint2 lo[4], hi[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint8_t* at = vl + 16 * ((2 * (i0 + i)) ^ v_key);
          lo[i] = transposed4(at), hi[i] = transposed4(at + 32 * D);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i0 + i] = mfma<Act>(u32x4_t{lo[i].x, lo[i].y, hi[i].x, hi[i].y}, pf, o[i0 + i]);
      }
    }
    if (more) {
      GDNR_WAIT_LGKM0();  // the step's values have been read
      copy_values();
    }
  };
  for (; key0 + kKeys <= vis_all; key0 += STEP) step(std::false_type{});
  for (; key0 < k_end; key0 += STEP) step(std::true_type{});
  // join the waves: every row's sums at the largest maximum
  __syncthreads();
  float* ml = (float*)(lds + lds_bytes<D>() - kWaves * kRows * 8);
  uint8_t* ow = lds + wave * kRows * o_stride<D>() + col * o_stride<D>() + 16 * grp;
#pragma unroll
  for (int i = 0; i < DT; ++i) *(f32x4_t*)(ow + 64 * i) = o[i];
  if (grp == 0) ml[2 * (wave * kRows + col)] = m_run, ml[2 * (wave * kRows + col) + 1] = l_run[0];
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
  const float norm = pieces > 1 ? 1.f : visible(sq, t) == 0 ? 0.f : 1.f / l;
  const int64_t part_at = (blk.z * a.part_rows[0] + piece_row(a, 0, n, sq, t)) * a.HQ + qh;
#pragma unroll
  for (int i = 0; i < D / 64; ++i) {
    const int d = 64 * i + 4 * dl;
    f32x4_t sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) sum += f[w] * *(const f32x4_t*)(lds + (w * kRows + row) * o_stride<D>() + 4 * d);
    sum *= norm;
    if (pieces > 1) {
      *(f32x4_t*)(a.part[0] + part_at * D + d) = sum;
    } else {
      *(uint2*)((uint8_t*)a.out + (t * a.o_t + qh * a.o_h + d) * 2) = make_uint2(pack2<Act>(sum[0], sum[1]), pack2<Act>(sum[2], sum[3]));
    }
  }
  if (pieces > 1 && dl == 0) {
    float* p = a.part_ml[0] + part_at * 2;
    p[0] = top, p[1] = l;
  }
}

template <int D>
struct Tile {
  static constexpr int NT = D == 256 ? 1 : 2;      // 16-row tiles a wave
  static constexpr int ROWS = kWaves * NT * 16;    // rows a workgroup
  static constexpr int KEYS = 8192 / D;            // keys a step
  static constexpr int KB = KEYS * 2 * D;          // bytes of a step's keys (and of its values)
  static constexpr int LDS = 4 * KB;               // two steps' keys and values
};

// 128 rows against the same keys. A step's keys and values go from the cache
// straight to LDS while the step before is computed. A wave keeps its rows'
// queries, scores and outputs in registers; the keys' fragment it reads from
// LDS serves both of its row tiles.
template <class Act, int D>
__device__ __forceinline__ void tile_step(const AttentionArgs& a, uint8_t* lds, const Block blk) {
  using TL = Tile<D>;
  constexpr int KSTEPS = D / 32, DT = D / 16, NT = TL::NT, KEYS = TL::KEYS, MT = KEYS / 16, PPR = D / 8;
  constexpr int RPI = 64 / PPR;                     // rows of an LDS copy
  constexpr int COPIES = KEYS / RPI / kWaves;       // copies of keys (and of values) a wave and step
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, grp = lane >> 4;
  const int gt = min(a.G, TL::ROWS), tb = TL::ROWS / gt;  // heads and tokens of a workgroup
  const int n = sequences_up_to(a, blk.y, tb, 1) - 1;
  if (n < 0) return;
  const Span sq = span_of(a, n);
  // Later tokens see more keys: the last tile first, so that the last to start
  // are short; and where two workgroups share a compute unit, the second ones in
  // the other direction, the longest beside the shortest. us a call, first tile
  // first, last first, and so, 32 heads of 128: 4096 tokens 196, 169 and 164; 2048
  // over 8192 keys 266, 257 and 248.
  const int tiles = (sq.end - sq.begin + tb - 1) / tb;
  int place = blk.y - sq.begin / tb - n;
  if (place >= tiles || few_rows(a, sq)) return;
  if (place >= a.turn && place < 2 * a.turn) place = a.turn + min(2 * a.turn, tiles) - 1 - place;
  const int tok0 = sq.begin + (tiles - 1 - place) * tb;
  const int head_tiles = (a.G + TL::ROWS - 1) / TL::ROWS;
  const int hk = blk.x / head_tiles, ht = blk.x - hk * head_tiles;
  const int last = min(tok0 + tb, sq.end) - 1;
  const int piece = a.piece[1], pieces = a.pieces[1];
  const int k_begin = blk.z * piece, k_end = min(visible(sq, last), k_begin + piece);
  if (k_begin >= k_end && (pieces > 1 || blk.z > 0)) return;

  // this lane's rows
  int rt[NT], rh[NT], vis[NT];
  bool live[NT];
  u32x4_t q[NT][KSTEPS];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int r = (wave * NT + nt) * 16 + col;
    rt[nt] = tok0 + r / gt, rh[nt] = ht * TL::ROWS + r % gt;
    live[nt] = r / gt < tb && rt[nt] < sq.end && rh[nt] < a.G;
    vis[nt] = live[nt] ? min(visible(sq, rt[nt]), k_end) : 0;
    const uint8_t* qp = (const uint8_t*)a.q + (rt[nt] * a.q_t + (hk * a.G + rh[nt]) * a.q_h) * 2 + 16 * grp;
#pragma unroll
    for (int i = 0; i < KSTEPS; ++i) q[nt][i] = live[nt] ? *(const u32x4_t*)(qp + 64 * i) : u32x4_t{0, 0, 0, 0};
  }
  const int vis_all = min(visible(sq, tok0), k_end);  // every live row sees these
  // scores grow with the products: a negative scale turns the queries' signs
  if (a.scale_log2 < 0.f) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < KSTEPS; ++i) q[nt][i] ^= 0x80008000u;
  }
  const float scale = fmaxf(fabsf(a.scale_log2), 1e-37f);  // (a masked -inf stays one)

  // copies: wave w's rows of a step are those of copies w, w + 4, ...; lane l
  // finds row l of them, in 16-byte units from the caches' bases
  constexpr int OWN = COPIES * RPI;
  const double inv_page = 1.0 / a.page;
  const int32_t* table = a.table + n * a.tb_n;
  const uint8_t* kbase = (const uint8_t*)a.k_cache + hk * a.kc_h * 2;
  const uint8_t* vbase = (const uint8_t*)a.v_cache + hk * a.vc_h * 2;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_void_t*)lds + wave * 1024;
  const uint32_t k_page = (uint32_t)(a.kc_p >> 3), k_tok = (uint32_t)(a.kc_t >> 3);
  const uint32_t v_page = (uint32_t)(a.vc_p >> 3), v_tok = (uint32_t)(a.vc_t >> 3);
  const int own = lane % OWN, own_row = ((own / RPI) * kWaves + wave) * RPI + own % RPI;
  int pg, off;
  auto find_rows = [&](int key0) {
    int p;
    page_of(min(key0 + own_row, k_end - 1), a.page, inv_page, p, off);
    pg = table[p];
  };
  auto copy = [&](int buf) {
    const uint32_t at = min(max(pg, 0), a.n_pages - 1);
    const uint32_t k_row = at * k_page + off * k_tok, v_row = at * v_page + off * v_tok;
    uint32_t kr[COPIES], vr[COPIES];
#pragma unroll
    for (int i = 0; i < COPIES; ++i) {
      const int from = i * RPI + lane / PPR;
      kr[i] = (uint32_t)__shfl((int)k_row, from), vr[i] = (uint32_t)__shfl((int)v_row, from);
    }
    GDNR_COMPILER_FENCE();
#pragma unroll
    for (int i = 0; i < COPIES; ++i) {
      const uint64_t piece16 = (lane % PPR) ^ row_key<D>((i * kWaves + wave) * RPI + lane / PPR);
      const uint32_t to = lds0 + buf * 2 * TL::KB + i * kWaves * 1024;
      dma16(kbase + (kr[i] + piece16) * 16, to);
      dma16(vbase + (vr[i] + piece16) * 16, to + TL::KB);
    }
  };

  f32x4_t o[NT][DT];
  f32x4_t l_run[NT];  // (every row of it)
  float m_run[NT];  // the references
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    m_run[nt] = -__builtin_inff(), l_run[nt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < DT; ++i) o[nt][i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  if (k_begin < k_end) {
    find_rows(k_begin);
    copy(0);
    if (k_begin + KEYS < k_end) find_rows(k_begin + KEYS);
  }
  int buf = 0, key0 = k_begin;
  // one step; MASKED: some of its keys are not seen by every row
  auto step = [&](auto tag) {
    constexpr bool MASKED = decltype(tag)::value;
    GDNR_WAIT_VMCNT(0);
    __syncthreads();  // the step's keys and values are in LDS; the other buffer is no longer read
    const uint8_t* kt = lds + buf * 2 * TL::KB;
    const uint8_t* vt = kt + TL::KB;
    // (the fragments' addresses are formed where they are used: kept across
    // steps they would take the registers of the operands)
    uint32_t k_key = row_key<D>(col) ^ grp, v_key = row_key<D>(4 * grp + (col >> 2)) ^ ((col & 3) >> 1);
    asm volatile("" : "+v"(k_key), "+v"(v_key));
    const uint8_t* kl = kt + col * 2 * D;
    const uint8_t* vl = vt + (4 * grp + (col >> 2)) * 2 * D + 8 * (col & 1);

    // S^T = K Q^T, two key tiles at a time
    f32x4_t s[MT][NT];
    u32x4_t kf[2][2][2];
    constexpr int KH = 2, STAGES = MT / 2 * (KSTEPS / KH);
    auto read_keys = [&](int st) {  // stage: key tiles 2 m2, 2 m2 + 1, k-steps KH h ..
      const int m2 = st / (KSTEPS / KH), h = st % (KSTEPS / KH);
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int i = 0; i < KH; ++i) {
          kf[st & 1][m][i] = *(const u32x4_t*)(kl + 16 * (2 * m2 + m) * 2 * D + 16 * ((4 * (KH * h + i)) ^ k_key));
        }
    };
    read_keys(0);
    GDNR_COMPILER_FENCE();
    if (key0 + KEYS < k_end) {
      copy(buf ^ 1);
      if (key0 + 2 * KEYS < k_end) find_rows(key0 + 2 * KEYS);
    }
    GDNR_COMPILER_FENCE();
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int st = 0; st < STAGES; ++st) {
      if (st + 1 < STAGES) read_keys(st + 1);
      GDNR_COMPILER_FENCE();
      const int m2 = st / (KSTEPS / KH), h = st % (KSTEPS / KH);
#pragma unroll
      for (int i = 0; i < KH; ++i)
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            s[2 * m2 + m][nt] = mfma<Act>(kf[st & 1][m][i], q[nt][KH * h + i],
                                          i + h == 0 ? f32x4_t{0.f, 0.f, 0.f, 0.f} : s[2 * m2 + m][nt]);
    }
    GDNR_COMPILER_FENCE();
    __builtin_amdgcn_s_setprio(0);
    // the values' fragments of 32 keys, read before the weights are formed
    u32x4_t vf[DT];
    auto read_values = [&](int half) {
#pragma unroll
      for (int i = 0; i < DT; ++i) {
        const uint8_t* p = vl + 32 * half * 2 * D + 16 * ((2 * i) ^ v_key);
        const uint2 lo = transposed4(p), hi = transposed4(p + 32 * D);
        vf[i] = u32x4_t{lo.x, lo.y, hi.x, hi.y};
      }
    };
    read_values(0);
    GDNR_COMPILER_FENCE();

    if constexpr (MASKED) {
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (key0 + 16 * m + 4 * grp + j >= vis[nt]) s[m][nt][j] = -__builtin_inff();
    }
    // The reference follows the scores only when their maximum has passed its
    // own by kLag: a weight then grows by 2^kLag at most, and the outputs are
    // rarely rescaled.
    float top[NT];
    bool behind = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      top[nt] = s[0][nt][0];
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int j = 0; j < 4; ++j) top[nt] = fmaxf(top[nt], s[m][nt][j]);
      top[nt] = column_max(top[nt]);
      behind |= passed<Act>(top[nt] * scale, m_run[nt], kLag<Act>);
    }
    if (__any(behind)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float m_new = fmaxf(m_run[nt], reference<Act>(top[nt] * scale));
        const float f = m_new == -__builtin_inff() ? 1.f : __builtin_amdgcn_exp2f(m_run[nt] - m_new);
        scale_in_place(l_run[nt], f);
#pragma unroll
        for (int i = 0; i < DT; ++i) scale_in_place(o[nt][i], f);
        m_run[nt] = m_new;
      }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float base = m_run[nt] == -__builtin_inff() ? 0.f : -m_run[nt], f = scale;
      if (__any(fabsf(base) > 0x1p24f)) {
        // (a rounding of such a product may pass the exponent's range: both
        // sides of the difference are rounded alike)
#pragma unroll
        for (int m = 0; m < MT; ++m) scale_in_place(s[m][nt], f), shift_in_place(s[m][nt], base);
        base = 0.f, f = 1.f;
      }
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[m][nt][j] = __builtin_amdgcn_exp2f(fmaf(s[m][nt][j], f, base));
    }
    if constexpr (MASKED) {
      bool bad = false;
#pragma nounroll
      for (int i = lane; i < KEYS * PPR; i += 64) bad |= nonfinite8<Act>(*(const u32x4_t*)(vt + 16 * i));
      if (__any(bad)) {
        // a value that some rows must not see is infinite or NaN, and a product
        // with its weight 0 would show it to them: this step key by key
#pragma nounroll
        for (int key = 0; key < KEYS; ++key)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float pk = 0.f;
#pragma unroll
            for (int e = 0; e < 4 * MT; ++e)
              if (4 * (key >> 4) + (key & 3) == e) pk = s[e >> 2][nt][e & 3];
            pk = __shfl(pk, col + 16 * ((key >> 2) & 3));
            const uint32_t seen = key0 + key < vis[nt] ? ~0u : 0u;
            shift_in_place(l_run[nt], pk);
#pragma unroll
            for (int i = 0; i < DT; ++i) {
              const uint2 w = *(const uint2*)(vt + key * 2 * D + 16 * ((2 * i + (grp >> 1)) ^ row_key<D>(key)) + 8 * (grp & 1));
              const float2 lo = Act::from_pair(w.x & seen), hi = Act::from_pair(w.y & seen);
              add_in_place(o[nt][i], pk, f32x4_t{lo.x, lo.y, hi.x, hi.y});
            }
          }
        return;
      }
    }
    // O^T += V^T P^T. (The weights are rounded to the cache's type, which costs
    // the output about its own rounding; their sum is of the rounded ones, so
    // that a row that one key rules loses nothing.)
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int half = 0; half < MT / 2; ++half) {
      u32x4_t pf[NT];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const f32x4_t x = s[2 * half][nt], y = s[2 * half + 1][nt];
        pf[nt] = u32x4_t{pack2<Act>(x[0], x[1]), pack2<Act>(x[2], x[3]), pack2<Act>(y[0], y[1]), pack2<Act>(y[2], y[3])};
        l_run[nt] = mfma<Act>(ones<Act>(), pf[nt], l_run[nt]);
      }
#pragma unroll
      for (int i = 0; i < DT; ++i)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) o[nt][i] = mfma<Act>(vf[i], pf[nt], o[nt][i]);
      if (half + 1 < MT / 2) {
        GDNR_COMPILER_FENCE();
        read_values(half + 1);
        GDNR_COMPILER_FENCE();
      }
    }
    __builtin_amdgcn_s_setprio(0);
  };
  for (; key0 + KEYS <= vis_all; key0 += KEYS, buf ^= 1) step(std::false_type{});
  for (; key0 < k_end; key0 += KEYS, buf ^= 1) step(std::true_type{});

#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const float l = l_run[nt][0];
    if (!live[nt]) continue;
    const int qh = hk * a.G + rh[nt];
    if (pieces > 1) {
      const int64_t at = (blk.z * a.part_rows[1] + piece_row(a, 1, n, sq, rt[nt])) * a.HQ + qh;
#pragma unroll
      for (int i = 0; i < DT; ++i) *(f32x4_t*)(a.part[1] + at * D + 16 * i + 4 * grp) = o[nt][i];
      if (grp == 0) a.part_ml[1][2 * at] = m_run[nt], a.part_ml[1][2 * at + 1] = l;
    } else {
      const float norm = vis[nt] == 0 ? 0.f : 1.f / l;
      uint8_t* p = (uint8_t*)a.out + (rt[nt] * a.o_t + qh * a.o_h + 4 * grp) * 2;
#pragma unroll
      for (int i = 0; i < DT; ++i) {
        const f32x4_t x = o[nt][i] * norm;
        *(uint2*)(p + 32 * i) = make_uint2(pack2<Act>(x[0], x[1]), pack2<Act>(x[2], x[3]));
      }
    }
  }
}

// The kernels: each walk alone, or both in one launch (the tiles' workgroups
// first) where a batch has sequences of either kind: the few rows' latency then
// hides behind the tiles' products (16 sequences, three of them with 400 tokens,
// 50.5 us a call in two launches, 39.7 in one).
template <class Act, int D>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, D == 64 ? 4 : 2))) void few_kernel(const AttentionArgs a) {
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  few_step<Act, D>(a, lds, Block{(int)blockIdx.x, (int)blockIdx.y, (int)blockIdx.z});
}
template <class Act, int D>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2))) void tile_kernel(const AttentionArgs a) {
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  tile_step<Act, D>(a, lds, Block{(int)blockIdx.x, (int)blockIdx.y, (int)blockIdx.z});
}
// few and tile: the two grids, x fastest
template <class Act, int D>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2))) void both_kernel(const AttentionArgs a, const Block few, const Block tile) {
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const auto block = [](int i, const Block& grid) {
    const int row = i / grid.x, z = row / grid.y;
    return Block{i - row * grid.x, row - z * grid.y, z};
  };
  const int tiles = tile.x * tile.y * tile.z, i = blockIdx.x;
  if (i < tiles) tile_step<Act, D>(a, lds, block(i, tile));
  else few_step<Act, D>(a, lds, block(i - tiles, few));
}

// The pieces of a row joined in their order. D / 4 lanes a row, the rows of a
// wave consecutive heads of one token (one look at its sequence for them all).
// Bound by the chain of loads lengths -> maxima and sums -> pieces: 4.5 us for
// one token of 16 heads in 32 pieces (with 4 pieces in flight the call takes 13.8
// us, 8 12.7, 16 12.3, 32 13.2).
template <class Act, int D>
__global__ __launch_bounds__(256) void join_kernel(const AttentionArgs a) {
  constexpr int W = D / 4, R = 64 / W, BATCH = 16;  // lanes a row, rows a wave, pieces in flight
  const int lane = threadIdx.x & 63, l = lane % W, t = blockIdx.x;
  const int h_own = (int)(blockIdx.y * 4 + (threadIdx.x >> 6)) * R + lane / W, h = min(h_own, a.HQ - 1);
  const int n = sequences_up_to(a, t, 1, 0) - 1;
  if (n < 0) return;
  const Span sq = span_of(a, n);
  const int kind = few_rows(a, sq) ? 0 : 1, piece = a.piece[kind];
  if (t < sq.begin || t >= sq.end || a.pieces[kind] == 1) return;
  const int64_t row0 = piece_row(a, kind, n, sq, t) * a.HQ + h, step = a.part_rows[kind] * a.HQ;
  const float* ml0 = a.part_ml[kind] + 2 * row0;
  const float* p0 = a.part[kind] + row0 * D + 4 * l;
  const int vis = visible(sq, t), pieces = (vis + piece - 1) / piece;
  f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
  float top = -__builtin_inff(), sum = 0.f;
  for (int z0 = 0; z0 < pieces; z0 += W) {
    // a lane a piece: its maximum and sum; then the pieces' outputs
    const int count = min(W, pieces - z0);
    const bool in = l < count;
    const float2 ml = *(const float2*)(ml0 + 2 * min(z0 + l, pieces - 1) * step);
    float m_new = fmaxf(top, in ? ml.x : -__builtin_inff());
#pragma unroll
    for (int d = 1; d < W; d *= 2) m_new = fmaxf(m_new, __shfl_xor(m_new, d));
    const float base = m_new == -__builtin_inff() ? 0.f : m_new;
    const float fo = z0 ? __builtin_amdgcn_exp2f(top - base) : 0.f, fz = in ? __builtin_amdgcn_exp2f(ml.x - base) : 0.f;
    float part = in ? fz * ml.y : 0.f;
#pragma unroll
    for (int d = 1; d < W; d *= 2) part += __shfl_xor(part, d);
    if (z0) sum *= fo, acc *= fo;
    sum += part;
    for (int i0 = 0; i0 < count; i0 += BATCH) {
      f32x4_t x[BATCH];
#pragma unroll
      for (int i = 0; i < BATCH; ++i) x[i] = *(const f32x4_t*)(p0 + min(z0 + i0 + i, pieces - 1) * step * D);
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        const float f = __shfl(fz, (lane & ~(W - 1)) + min(i0 + i, W - 1));
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] = i0 + i < count ? fmaf(f, x[i][e], acc[e]) : acc[e];
      }
    }
    top = m_new;
  }
  if (h_own >= a.HQ) return;
  acc *= vis == 0 ? 0.f : 1.f / sum;
  *(uint2*)((uint8_t*)a.out + (t * a.o_t + h * a.o_h + 4 * l) * 2) = make_uint2(pack2<Act>(acc[0], acc[1]), pack2<Act>(acc[2], acc[3]));
}

template <class Act, int D>
int launch_dim(AttentionArgs a, hipStream_t s) {
  const auto grid = [&](int rows, int pieces) {  // key heads first: a head's workgroups share an XCD
    const int gt = a.G < rows ? a.G : rows, tb = rows / gt;
    const bool one_tile = rows == kRows && a.few_rows == kRows;
    return Block{a.HKV * ((a.G + rows - 1) / rows), one_tile ? a.N : a.T / tb + a.N, pieces};
  };
  const auto launch = [&](auto kernel, dim3 blocks, int lds, auto... more) {
    if (lds > 64 * 1024) {  // (enabled per kernel and device; idempotent, cheap)
      const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
      if (e != hipSuccess) return (int)e;
    }
    hipLaunchKernelGGL(kernel, blocks, dim3(256), lds, s, a, more...);
    return (int)hipGetLastError();
  };
  constexpr int few_lds = lds_bytes<D>(), tile_lds = Tile<D>::LDS;
  const Block few = grid(kRows, a.pieces[0]), tile = grid(Tile<D>::ROWS, a.pieces[1]);
  if (a.N == 1 && a.pieces[1] == 1)  // (the second of two to a compute unit start there)
    a.turn = device_cus() / tile.x;
  const int64_t fews = (int64_t)few.x * few.y * few.z, tiles = (int64_t)tile.x * tile.y * tile.z;
  int rc = 0;
  if (fews && tiles && fews + tiles < 1 << 24) {  // (a dimension of a grid ends at 2^32 threads)
    rc = launch(both_kernel<Act, D>, dim3((uint32_t)(fews + tiles)), few_lds > tile_lds ? few_lds : tile_lds, few, tile);
  } else {
    if (fews) rc = launch(few_kernel<Act, D>, dim3(few.x, few.y, few.z), few_lds);
    if (!rc && tiles) rc = launch(tile_kernel<Act, D>, dim3(tile.x, tile.y, tile.z), tile_lds);
  }
  if (rc) return rc;
  if (a.pieces[0] > 1 || a.pieces[1] > 1) {
    constexpr int R = 256 / D;  // heads a wave
    hipLaunchKernelGGL((join_kernel<Act, D>), dim3(a.T, (a.HQ + 4 * R - 1) / (4 * R)), dim3(256), 0, s, a);
  }
  return (int)hipGetLastError();
}
template <class Act>
int launch_act(const AttentionArgs& a, hipStream_t s) {
  if (a.D == 64) return launch_dim<Act, 64>(a, s);
  if (a.D == 128) return launch_dim<Act, 128>(a, s);
  return launch_dim<Act, 256>(a, s);
}

}  // namespace

// Which kernels run (pieces 0: not that one), and the keys of a workgroup's
// piece. The lengths are on the device; the host knows their number and sum.
// Where a sequence has 16 rows or fewer on average, few_kernel takes all of
// them; a single longer one is tile_kernel's; otherwise each takes its kind. A
// context is cut while a kernel would have fewer than eight (few) or two
// (tile) workgroups a compute unit, into whole steps of 128 keys, at least 256:
// a shorter piece costs as much to join as to walk. us a call with half, this and
// twice as many workgroups: 64 decodes 145, 144 and 150; three chunks of 400
// tokens beside 13 decodes 46.5, 39.8 and 40.2; a chunk of 2048 tokens over 8192
// keys 248 as it is (one piece) and 284 with twice as many. One decode over 8192
// keys with pieces of 256 keys 12.6, of 128 14.2. (A prompt hidden by an average of
// 16 rows loses nothing on few_kernel: 960 tokens beside 63 single ones over 2000 keys, 8
// heads of 128 148 us, each kind on its kernel 153; 400 beside 63, heads of 64, 56 and 63.)
void plan_attention(AttentionArgs* a) {
  const int64_t cus = device_cus(), rows = (int64_t)a->T * (a->G < kRows ? a->G : kRows);
  const bool all_few = rows <= (int64_t)kRows * a->N, all_tile = !all_few && a->N == 1;
  a->few_rows = all_few ? INT32_MAX : all_tile ? 0 : kRows;
  const auto plan = [&](int kind, int64_t tiles, int64_t want) {
    const int64_t groups = tiles * a->HKV;
    int64_t p = a->max_context;
    if (groups < want) p = (a->max_context * groups + want - 1) / want;
    p = (p + 127) / 128 * 128;
    if (p < 256) p = 256;
    a->piece[kind] = (int32_t)(p < INT32_MAX ? p : INT32_MAX);
    a->pieces[kind] = a->max_context ? (int32_t)((a->max_context + p - 1) / p) : 1;
  };
  const auto tiles_of = [&](int tile_rows) {
    const int64_t gt = a->G < tile_rows ? a->G : tile_rows;
    return (a->T / (tile_rows / gt) + 1) * ((a->G + tile_rows - 1) / tile_rows);
  };
  a->pieces[0] = a->pieces[1] = 0;
  if (!all_tile) plan(0, all_few && a->T > a->N ? tiles_of(kRows) : (int64_t)a->N * ((a->G + kRows - 1) / kRows), 8 * cus);
  if (!all_few) plan(1, tiles_of(a->D == 256 ? 64 : 128), 2 * cus);
}

// The kinds' pieces one after the other, then their maxima and sums. Where both
// kinds occur, the sequences of few rows have one tile of tokens each (their
// number of pieces goes by the number of sequences: it would be charged to every
// token of a prompt beside them). A kind in one piece takes nothing.
int64_t place_pieces(AttentionArgs* a, float* work) {
  int64_t rows[2];
  for (int kind = 0; kind < 2; ++kind) {
    const bool by_sequence = kind == 0 && a->few_rows == kRows;
    a->part_rows[kind] = by_sequence ? (int64_t)a->N * (kRows / (a->G < kRows ? a->G : kRows)) : a->T;
    rows[kind] = a->pieces[kind] > 1 ? a->pieces[kind] * a->part_rows[kind] * a->HQ : 0;
  }
  if (work) {
    a->part[0] = work, a->part[1] = work + rows[0] * a->D;
    a->part_ml[0] = a->part[1] + rows[1] * a->D, a->part_ml[1] = a->part_ml[0] + 2 * rows[0];
  }
  return (rows[0] + rows[1]) * (a->D + 2) * 4;
}

int launch_attention(const AttentionArgs& a, int act_dt, void* stream) {
  return act_dt == DT_BF16 ? launch_act<ActBF16>(a, (hipStream_t)stream) : launch_act<ActF16>(a, (hipStream_t)stream);
}

}  // namespace gdnr
