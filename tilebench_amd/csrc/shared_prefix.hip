// Paged attention of a batch whose sequences share prefixes (decode, drafted
// tokens and prompt chunks in one call).
//
//   out = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale * q . k_j - m),   lse = m + log sum_j p_j
//
// over the tokens j of the sequence's group prefix followed by its own tokens,
// up to the query's own position (the queries are the last n_q tokens).
//
// Rows.  The query heads of one key/value head and the queries of one sequence
// read the same tokens, so they are rows of one product: row r of a run of
// queries is query r / grp, head r % grp of the group.  Three kinds of work:
//   tiles   64 or 128 rows of a group of more than 16 rows: over the shared prefix, and
//           on over the own tokens of those sequences that have more than 16 rows
//   few     the own tokens of one sequence of up to 16 rows, or the prefix of a
//           group of up to 16 rows: the block's four wavefronts split the tokens
//   combine joins the partial results of a row (one slot per split) by their maxima
// so a prefix is read once per tile however many sequences share it.
//
// One wavefront's step over TOK tokens in LDS (attend_tile):
//   S^T = K Q^T    K rows from LDS, Q in registers; a lane holds one row's scores
//   P^T            exp2 of the scores against the running maximum, in registers; the
//                  tokens a lane holds are in the order of the next product's operand
//   O^T = V^T P^T  V^T by transposing LDS reads (ds_read_b64_tr_b16 / _b8) in that order
// so scores never leave registers, and the maximum, sum and output of a row belong to
// the lanes that hold the row.  Sums and statistics are fp32.  P is rounded to the
// inputs' type for the second product (2^-11 or 2^-8 of each weight, unbiased).
//
// e4m3 caches: codes are converted exactly to the inputs' type; the keys' scales
// multiply the scores, the values' scales the weights.
//
// Values that a row does not attend to never reach it: masked scores are selected
// away, and in a tile that some rows see in part infinities and NaN among the
// values count as zeros in the product and are marked in LDS for the rows that
// attend to them, to be added at the end.
#include "tb_common.h"

#include <type_traits>

namespace tb {
namespace prefix {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2v __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

enum { F16 = 1, BF16 = 2 };
constexpr int THREADS = 256, WAVES = 4;
constexpr int FEW = 16;      // rows of a sequence or group that the token-splitting blocks take
constexpr int FILL = 512;    // blocks that fill the device: two on each of 256 CUs
constexpr int MAX_SPLIT = 64;
constexpr float NEG_INF = -__builtin_inff();

struct Args {
  const void* q;
  int64_t q_st, q_sh;
  const char* kc;
  const char* vc;
  int64_t c_page, c_head, c_slot;
  const float* ks;
  const float* vs;
  int64_t s_page, s_head, s_slot;
  const int* prefix_pages;  // [G, Wp]
  const int* prefix_lens;   // [G]
  const int* group_offsets; // [G + 1]
  const int* pages;         // [B, W]
  const int* lens;          // [B]
  const int* cu_q;          // [B + 1]
  void* out;
  float* lse;
  float* part_o;  // [slots][T * Hq][D]
  float2* part_ml;  // [slots][T * Hq]: maximum (log2) and sum; sum -1: the row is final
  int T, Hq, Hkv, grp, G, Wp, B, W;
  int n_pages, page_shift;
  int S1, S2;       // slots of tiles and prefixes, slots of own tokens
  int direct;       // own tokens in one slot and nothing else: results are final
  float scale_log2;     // of |scale|, or 1 for a scale of 0
  uint32_t flip, keep;  // applied to q
  int near;  // 64 slots of a page lie within 2 GiB
  int big;  // some sequence may have more than FEW rows
  int tile_blocks;
};

// The kernel's arguments, read again from memory.  Epilogues and other code off the loops take theirs from here: fields
// that are only needed there would hold scalar registers through the loops, which then spill.
__device__ __forceinline__ Args reload() {
  typedef const __attribute__((address_space(4))) Args* ptr;
  ptr p = (ptr)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *(const Args*)p;
}

template <int DT>
struct Ty;
template <>
struct Ty<F16> {
  typedef f16x8 v8;
  typedef _Float16 el;
  static __device__ __forceinline__ f32x4 mfma(v8 a, v8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x16 mfma(v8 a, v8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t up8(uint32_t w, bool hi) {
    return hi ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true))
              : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false));
  }
  static constexpr uint32_t EXP = 0x7C00u;  // exponent bits: all ones in infinities and NaN
};
template <>
struct Ty<BF16> {
  typedef bf16x8 v8;
  typedef __bf16 el;
  static __device__ __forceinline__ f32x4 mfma(v8 a, v8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x16 mfma(v8 a, v8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t up8(uint32_t w, bool hi) {
    return hi ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true))
              : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false));
  }
  static constexpr uint32_t EXP = 0x7F80u;
};

// ------------------------------------------------------------------ LDS tiles
//
// A tile holds rows of RB bytes, one per token; the 16-byte chunk c of row t sits at
// position c ^ f(t), so that the lanes of one LDS access (16 rows at one chunk for
// keys, the rows and chunks of one transposing read for values) fall into different
// banks.  SH is the side of the product's tiles (16 or 32).
template <int RB>
__device__ __forceinline__ constexpr int swizzle_k(int t) {
  return RB == 256 ? (t & 15) : RB == 128 ? ((t >> 1) & 7) : ((t >> 2) & 3);
}
template <int RB, int SH, bool E8>
__device__ __forceinline__ constexpr int swizzle_v(int t) {
  if (!E8 && SH == 16) return RB == 256 ? (t & 7) << 1 : ((t >> 1) & 3) << 1;
  if (!E8) return RB == 256 ? (t & 3) << 2 : ((t >> 1) & 1) << 2;
  if (SH == 16) return RB == 128 ? ((t >> 1) & 3) | ((t >> 4) & 1) << 2 : ((t >> 2) & 1) | ((t >> 4) & 1) << 1;
  return RB == 128 ? (((t >> 1) & 1) | ((t >> 3) & 1) << 1) << 1 : ((t >> 3) & 1) << 1;
}

typedef __attribute__((address_space(3))) char lds_char;
__device__ __forceinline__ uint32_t lds_addr(const void* p) {
  return (uint32_t)(uintptr_t)(lds_char*)p;
}
template <typename V>
__device__ __forceinline__ V lds_read(uint32_t addr) {
  return *(const __attribute__((address_space(3))) V*)(uintptr_t)addr;
}

// 16 (or 4) bytes a lane from global memory to LDS at lds + 16 (4) * lane.
__device__ __forceinline__ void dma16(uint32_t lds, const char* p) {
  asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, off"
               :
               : "s"(__builtin_amdgcn_readfirstlane((int)lds)), "v"(p)
               : "memory", "m0");
}
// the same from a uniform address plus a 32-bit offset of each lane
__device__ __forceinline__ void dma16(uint32_t lds, const char* p, uint32_t off) {
  const uint64_t u = (uint64_t)(uintptr_t)p;
  const uint64_t base = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)u) |
                        (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(u >> 32)) << 32;
  asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, %2"
               :
               : "s"(__builtin_amdgcn_readfirstlane((int)lds)), "v"(off), "s"(base)
               : "memory", "m0");
}
__device__ __forceinline__ void dma4(uint32_t lds, const char* p) {
  asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dword %1, off"
               :
               : "s"(__builtin_amdgcn_readfirstlane((int)lds)), "v"(p)
               : "memory", "m0");
}
// Waits until at most N of this wavefront's vector memory operations are pending.
template <int N>
__device__ __forceinline__ void wait_vm() {
  asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory");
}
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory"); }

// e4m3 scales of a tile, for each 32 tokens: 32 of the keys, 32 of the values.
__device__ __forceinline__ uint32_t scale_at(uint32_t sbase, int tok) { return sbase + (tok >> 5) * 256 + (tok & 31) * 4; }

// The tokens of one prefix or sequence: a row of a page table and a length.
struct Tokens {
  const int* table;
  int width, len;
};

// 64 consecutive entries of a page table, one a lane (ids outside the pool clamped to it).
struct Window {
  int ids = 0, first = 0x7FFFFFFF;
  __device__ __forceinline__ void cover(const Tokens& s, int lo, int hi, int n_pages) {
    if (lo >= first && hi < first + 64) return;
    first = lo;
    int id = s.table[min(lo + (int)(threadIdx.x & 63), s.width - 1)];
    id = min(max(id, 0), n_pages - 1);
    asm volatile("" : "+v"(id));  // the wait for the load belongs here, not at the uses in the loop
    ids = id;
  }
};

// Copies of NI KiB of token rows into a tile: rows lane / (RB / 16) + i * RPI from token t0 on, the 16-byte chunk of a
// lane at its swizzled place.
template <int RB, int NI>
struct Copier {
  static constexpr int LANES = RB / 16, RPI = 64 / LANES, ROWS = NI * RPI;
  // swizzle(r) is linear in the bits of r: that of the lane's row and that of the copy's first row
  template <typename Swizzle>
  static __device__ __forceinline__ void run(const Args& a, const Window& w, const Tokens& s, const char* pool,
                                             uint32_t lds, int t0, int esize, Swizzle swizzle) {
    const int lane = threadIdx.x & 63, r = lane / LANES, chunk = (lane % LANES) ^ swizzle(r);
    const int mask = (1 << a.page_shift) - 1;
    if (a.near && mask + 1 >= ROWS && t0 + ROWS <= s.len) {  // whole and in one page
      const int page = __builtin_amdgcn_readlane(w.ids, (t0 >> a.page_shift) - w.first);
      const char* p = pool + (page * a.c_page + (t0 & mask) * a.c_slot) * esize;
      const uint32_t row = (uint32_t)(r * (int)a.c_slot * esize);
      const int64_t step = RPI * a.c_slot * esize;
#pragma unroll
      for (int i = 0; i < NI; ++i)
        dma16(lds + i * 1024, p + i * step, row + (uint32_t)((chunk ^ swizzle(i * RPI)) << 4));
      return;
    }
#pragma unroll 1
    for (int i = 0; i < NI; ++i) {
      const int tok = min(t0 + r + i * RPI, s.len - 1);  // past the end: the last token again (masked)
      const int page = __builtin_amdgcn_ds_bpermute(((tok >> a.page_shift) - w.first) << 2, w.ids);
      dma16(lds + i * 1024, pool + (page * a.c_page + (tok & mask) * a.c_slot) * esize + ((chunk ^ swizzle(i * RPI)) << 4));
    }
  }
};

__device__ __forceinline__ uint32_t as_uint(float x) { return __builtin_bit_cast(uint32_t, x); }
__device__ __forceinline__ float as_float(uint32_t x) { return __builtin_bit_cast(float, x); }

// ------------------------------------------------------------------ one step
//
// State of one wavefront: SH rows (lane l: row l % SH), head dimension D.
template <int DT, bool E8, int D, int SH>
struct Wave {
  typedef Ty<DT> Y;
  typedef typename Y::v8 v8;
  typedef typename std::conditional<SH == 16, f32x4, f32x16>::type acc_t;
  static constexpr int RB = D * (E8 ? 1 : 2);
  static constexpr int NG = 64 / SH;        // lane groups that share the rows
  static constexpr int KS = 8 * NG;         // depth of one product instruction
  static constexpr int STEPS = D / KS;      // of S^T
  static constexpr int DT_N = D / SH;       // output tiles
  static constexpr int REGS = SH * SH / 64; // accumulator registers of a tile

  // log2 of the largest weight when m is set, and how far weights may grow past it before m is set again.  fp16:
  // weights down to 2^-32 (e4m3: 2^-28) of the largest are kept; with e4m3 values their scales are multiplied in, which leaves
  // room for scales up to 2^10 (a row of fp16 values has at most 146).
  static constexpr float LIFT = DT == BF16 ? 0.0f : E8 ? 4.0f : 8.0f;
  static constexpr float SLACK = DT == BF16 || !E8 ? 6.0f : 2.0f;

  v8 q[STEPS];
  acc_t o[DT_N];
  float m, l;  // reference of the weights (log2), this lane's part of their sum

  // channel of element 0 of operand `s` in this lane's group
  static __device__ __forceinline__ int channel(int s, int g) {
    return E8 ? (s / 2) * NG * 16 + g * 16 + (s % 2) * 8 : s * NG * 8 + g * 8;
  }
  // flip, keep: the sign bits of a negative scale and nothing of q for a scale of 0 (scale_log2 is positive)
  __device__ __forceinline__ void init(const typename Y::el* row, bool valid, uint32_t flip, uint32_t keep) {
    const int g = (threadIdx.x & 63) / SH;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      u32x4 x{};
      if (valid) x = *(const u32x4*)(row + channel(s, g));
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = (x[i] & keep) ^ flip;
      q[s] = __builtin_bit_cast(v8, x);
    }
#pragma unroll
    for (int d = 0; d < DT_N; ++d) o[d] = acc_t{};
    m = NEG_INF;
    l = 0.0f;
  }
  // token (within a tile of SH) of accumulator register r
  static __device__ __forceinline__ int token_of(int r, int g) {
    return SH == 16 ? g * 4 + r : 8 * (r / 4) + 4 * g + r % 4;
  }
  // over the lane groups, which hold the same rows (a swap of a value's halves with a copy's gives every lane both)
  static __device__ __forceinline__ float over_groups_max(float x) {
    if (SH == 16) {
      const auto y = __builtin_amdgcn_permlane16_swap(as_uint(x), as_uint(x), false, false);
      x = fmaxf(as_float(y[0]), as_float(y[1]));
    }
    const auto z = __builtin_amdgcn_permlane32_swap(as_uint(x), as_uint(x), false, false);
    return fmaxf(as_float(z[0]), as_float(z[1]));
  }
  static __device__ __forceinline__ float over_groups_sum(float x) {
    if (SH == 16) {
      const auto y = __builtin_amdgcn_permlane16_swap(as_uint(x), as_uint(x), false, false);
      x = as_float(y[0]) + as_float(y[1]);
    }
    const auto z = __builtin_amdgcn_permlane32_swap(as_uint(x), as_uint(x), false, false);
    return as_float(z[0]) + as_float(z[1]);
  }

  // S^T of TOK tokens: TOK / SH tiles
  template <int TOK>
  __device__ __forceinline__ void scores(uint32_t kbase, acc_t (&s)[TOK / SH]) {
    const int lane = threadIdx.x & 63, row = lane % SH, g = lane / SH;
    const uint32_t a0 = kbase + row * RB, x = (uint32_t)(swizzle_k<RB>(row) ^ g) << 4;
#pragma unroll
    for (int t = 0; t < TOK / SH; ++t) s[t] = acc_t{};
    if (E8) {
#pragma unroll
      for (int c = 0; c < STEPS / 2; ++c) {
        const uint32_t at = a0 + (x ^ (uint32_t)(c * NG * 16));
#pragma unroll
        for (int t = 0; t < TOK / SH; ++t) {
          const u32x4 w = lds_read<u32x4>(at + t * SH * RB);
          u32x4 lo, hi;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            lo[2 * i] = Y::up8(w[i], false);
            lo[2 * i + 1] = Y::up8(w[i], true);
            hi[2 * i] = Y::up8(w[2 + i], false);
            hi[2 * i + 1] = Y::up8(w[2 + i], true);
          }
          s[t] = Y::mfma(__builtin_bit_cast(v8, lo), q[2 * c], s[t]);
          s[t] = Y::mfma(__builtin_bit_cast(v8, hi), q[2 * c + 1], s[t]);
        }
      }
    } else {
#pragma unroll
      for (int c = 0; c < STEPS; ++c) {
        const uint32_t at = a0 + (x ^ (uint32_t)(c * NG * 16));
#pragma unroll
        for (int t = 0; t < TOK / SH; ++t) s[t] = Y::mfma(lds_read<v8>(at + t * SH * RB), q[c], s[t]);
      }
    }
  }

  // Scores of the tokens that a row does not see: -inf.  left: tokens up to the row's limit, from the lane group's first.
  template <int TOK>
  static __device__ __forceinline__ void hide(acc_t (&s)[TOK / SH], int left) {
    __builtin_amdgcn_sched_barrier(0);  // comparisons hoisted over the products would take all scalar registers
#pragma unroll
    for (int t = 0; t < TOK / SH; ++t) {
#pragma unroll
      for (int r = 0; r < REGS; ++r) s[t][r] = t * SH + token_of(r, 0) < left ? s[t][r] : NEG_INF;
      __builtin_amdgcn_sched_barrier(0);
    }
  }

  // Scores -> weights exp2(score - m), the operands of the second product.  m follows the running maximum in steps:
  // while no row of the wavefront passes its m by 2^SLACK beyond the lift, sums and outputs stay as they are.
  template <int TOK>
  __device__ __forceinline__ void weights(acc_t (&s)[TOK / SH], int t0, int limit, bool full, float scale,
                                          uint32_t sbase, int tok0, v8 (&p)[TOK / KS]) {
    const int g = (threadIdx.x & 63) / SH;
    float top = NEG_INF;
    if (!full) hide<TOK>(s, limit - t0 - 4 * g);
#pragma unroll
    for (int t = 0; t < TOK / SH; ++t)
#pragma unroll
      for (int r = 0; r < REGS; r += 4) {
        const int tok = t * SH + token_of(r, g);
        if (E8) {
          const f32x4 k = lds_read<f32x4>(scale_at(sbase, tok0 + tok));
#pragma unroll
          for (int i = 0; i < 4; ++i) s[t][r + i] *= full || s[t][r + i] > NEG_INF ? k[i] : 1.0f;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) top = fmaxf(top, s[t][r + i]);
        if (E8 && r % 8 == 4) __builtin_amdgcn_sched_barrier(0);  // all scales at once would spill
      }
    top = over_groups_max(top) * scale;
    if (__any(top > m + (LIFT + SLACK))) {
      const float ref = fmaxf(m, top - LIFT);
      const float alpha = __builtin_amdgcn_exp2f(m - (ref == NEG_INF ? 0.0f : ref));
      m = ref;
      l *= alpha;
#pragma unroll
      for (int d = 0; d < DT_N; ++d)
#pragma unroll
        for (int r = 0; r < REGS; ++r) o[d][r] *= alpha;
    }
    const float use = m == NEG_INF ? 0.0f : m;
    float sum = 0.0f;
#pragma unroll
    for (int t = 0; t < TOK / SH; ++t)
#pragma unroll
      for (int r = 0; r < REGS; r += 4) {
        f32x4 v;
        if (E8) v = lds_read<f32x4>(scale_at(sbase, tok0 + t * SH + token_of(r, g)) + 128);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][r + i], scale, -use));
          sum += w;
          s[t][r + i] = !E8 ? w : full || w > 0.0f ? w * v[i] : 0.0f;
        }
        if (E8 && r % 8 == 4) __builtin_amdgcn_sched_barrier(0);
      }
    l += sum;
#pragma unroll
    for (int k = 0; k < TOK / KS; ++k)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        p[k][e] = SH == 16 ? (typename Y::el)s[2 * k + e / 4][e % 4]
                           : (typename Y::el)s[k * 16 / SH][(k % 2) * 8 + e];
  }

  // V^T of output tile d, tokens of step k, as the first operand.
  struct Values {
    uint32_t at, x;  // address of the lane's first row, its swizzled chunk
    __device__ __forceinline__ explicit Values(uint32_t vbase) {
      const int lane = threadIdx.x & 63, i = lane & 15;
      const int gx = lane / SH;                          // the group's four tokens
      const int sub = SH == 32 ? (lane >> 4) & 1 : 0;    // 16 of a tile's 32 channels
      if (E8) {
        const int r = i >> 1, tok = gx * 4 + (r & 3) + (r >> 2) * (KS / 2);
        at = vbase + tok * RB + (i & 1) * 8;
        x = (uint32_t)(sub ^ swizzle_v<RB, SH, E8>(tok)) << 4;
      } else {
        const int r = i >> 2, b = i & 3, tok = gx * 4 + r;
        at = vbase + tok * RB + (b & 1) * 8;
        x = (uint32_t)((sub * 2 + (b >> 1)) ^ swizzle_v<RB, SH, E8>(tok)) << 4;
      }
    }
    __device__ __forceinline__ v8 read(int d, int k) const {
      if (E8) {
        const uint32_t p = at + (x ^ (uint32_t)(d * (SH / 16) * 16)) + k * KS * RB;
        const i32x2 w = __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) i32x2*)(uintptr_t)p);
        u32x4 u;
        u[0] = Y::up8((uint32_t)w[0], false);
        u[1] = Y::up8((uint32_t)w[0], true);
        u[2] = Y::up8((uint32_t)w[1], false);
        u[3] = Y::up8((uint32_t)w[1], true);
        return __builtin_bit_cast(v8, u);
      }
      // rows tok and tok + KS / 2: the swizzle of both is the same (it repeats every KS / 2 rows at most)
      const uint32_t p = at + (x ^ (uint32_t)(d * (SH / 8) * 16)) + k * KS * RB;
      typedef __attribute__((address_space(3))) s16x4* ptr;
      struct { s16x4 a, b; } u;
      u.a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ptr)(uintptr_t)p);
      u.b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ptr)(uintptr_t)(p + KS / 2 * RB));
      return __builtin_bit_cast(v8, u);
    }
  };

  // O^T += V^T P^T
  template <int TOK>
  __device__ __forceinline__ void values(uint32_t vbase, const v8 (&p)[TOK / KS]) {
    const Values v(vbase);
#pragma unroll
    for (int k = 0; k < TOK / KS; ++k)
#pragma unroll
      for (int d = 0; d < DT_N; ++d) o[d] = Y::mfma(v.read(d, k), p[k], o[d]);
  }

  // Infinities and NaN among the values of tokens that some rows do not see.  They are replaced by zeros in the tile
  // and marked for the rows that see their token: a byte for each row and each run of D / 64 channels, four bits a
  // channel (1: +inf, 2: -inf, 4: NaN), added to the row's output at the end.
  //
  // Tokens tok0 .. tok0 + ROWS - 1 of the tile at vbase, t0 being the tile's first token; limit_of(r): the limit of row r.
  template <int ROWS, typename Limit>
  static __device__ __forceinline__ void set_apart(uint32_t vbase, int tok0, int t0, int rows, uint32_t marks,
                                                   Limit limit_of) {
    const int lane = threadIdx.x & 63;
    const uint32_t exps = E8 ? 0x7F7F7F7Fu : Y::EXP | Y::EXP << 16, ones = E8 ? 0x7F7F7F7Fu : 0x7FFF7FFFu;
    uint32_t good = ~0u;  // the top bit of an element: not (all exponent bits, or the NaN code)
#pragma unroll
    for (int i = 0; i < ROWS * RB / 1024; ++i) {
      const u32x4 x = lds_read<u32x4>(vbase + tok0 * RB + i * 1024 + lane * 16);
#pragma unroll
      for (int e = 0; e < 4; ++e) good &= exps - (x[e] & exps) + ones;
    }
    if (!__any((~good & ~ones) != 0)) return;
    constexpr int PER = D / 64, ESIZE = E8 ? 1 : 2;
    const int at = lane * PER * ESIZE;
#pragma unroll 1
    for (int tok = tok0; tok < tok0 + ROWS; ++tok) {
      const uint32_t p = vbase + tok * RB + (((at >> 4) ^ swizzle_v<RB, SH, E8>(tok)) << 4) + (at & 15);
      uint32_t is = 0;
#pragma unroll
      for (int e = 0; e < PER; ++e) {
        uint32_t x = E8 ? lds_read<uint8_t>(p + e) : lds_read<uint16_t>(p + 2 * e);
        if (E8) x = (x & 0x7Fu) == 0x7Fu ? 0x7FFFu : 0u;
        if ((x & Y::EXP) != Y::EXP) continue;
        is |= ((x & 0x7FFFu) != Y::EXP ? 4u : x & 0x8000u ? 2u : 1u) << (4 * e);
        if (E8)
          *(__attribute__((address_space(3))) uint8_t*)(uintptr_t)(p + e) = 0;
        else
          *(__attribute__((address_space(3))) uint16_t*)(uintptr_t)(p + 2 * e) = 0;
      }
      if (!__any(is != 0)) continue;
#pragma unroll 1
      for (int r = 0; r < rows; ++r) {
        if (t0 + tok >= limit_of(r) || is == 0) continue;
        __hip_atomic_fetch_or((__attribute__((address_space(3))) uint32_t*)(uintptr_t)(marks + r * 64 + (lane & ~3)),
                              is << (8 * (lane & 3)), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
      }
    }
  }
  // x, or what the marks of row r make of channels c .. c + 3
  static __device__ __forceinline__ f32x4 marked(f32x4 x, uint32_t marks, int r, int c) {
    constexpr int PER = D / 64;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t m = (lds_read<uint8_t>(marks + r * 64 + (c + i) / PER) >> (4 * (i % PER))) & 15u;
      if (m & 1u) x[i] += __builtin_inff();
      if (m & 2u) x[i] -= __builtin_inff();
      if (m & 4u) x[i] = __builtin_nanf("");
    }
    return x;
  }
};

// ------------------------------------------------------------------ rows and lengths

struct Seq {
  int q0, n_q, own;  // first query, queries, own tokens
};
__device__ __forceinline__ int clamp_int(int x, int lo, int hi) { return min(max(x, lo), hi); }
__device__ __forceinline__ int query_start(const Args& a, int b) { return clamp_int(a.cu_q[b], 0, a.T); }
__device__ __forceinline__ Seq sequence(const Args& a, int b) {
  Seq s;
  s.q0 = query_start(a, b);
  s.n_q = max(query_start(a, b + 1) - s.q0, 0);
  s.own = clamp_int(a.lens[b], 0, a.W << a.page_shift);
  return s;
}
struct Group {
  int b0, b1, q0, rows, len;  // sequences, first query, rows per key/value head, prefix tokens
};
__device__ __forceinline__ Group group(const Args& a, int g) {
  Group r;
  r.b0 = a.group_offsets && g > 0 ? clamp_int(a.group_offsets[g], 0, a.B) : 0;
  r.b1 = a.group_offsets && g + 1 < a.G ? clamp_int(a.group_offsets[g + 1], r.b0, a.B) : a.B;
  r.q0 = query_start(a, r.b0);
  r.rows = max(query_start(a, r.b1) - r.q0, 0) * a.grp;
  r.len = a.prefix_lens ? clamp_int(a.prefix_lens[g], 0, a.Wp << a.page_shift) : 0;
  return r;
}
// The sequence of query t among b0 .. b1 - 1 (the last one that starts at or before it).
__device__ __forceinline__ int sequence_of(const Args& a, int t, int b0, int b1) {
  int lo = b0, hi = b1;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.cu_q[mid] <= t) lo = mid; else hi = mid;
  }
  return lo;
}

// A row without tokens has the sum 0: its output is 0 and its lse -inf.
__device__ __forceinline__ float inverse(float sum) { return sum == 0.0f ? 0.0f : 1.0f / sum; }
__device__ __forceinline__ float natural_lse(float m, float sum) {
  return sum == 0.0f ? NEG_INF : (m + __builtin_amdgcn_logf(sum)) * 0.69314718055994530942f;
}

template <typename el>
__device__ __forceinline__ void store4(el* p, f32x4 x) {
  struct alignas(8) { el e[4]; } v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v.e[i] = (el)x[i];
  *(decltype(v)*)p = v;
}

// ------------------------------------------------------------------ few rows

template <int DT, bool E8, int D>
struct FewLayout {
  static constexpr int RB = D * (E8 ? 1 : 2);
  static constexpr int TOK = RB == 256 ? 32 : 64;  // tokens of a wavefront's step
  static constexpr int TILE_BYTES = TOK * RB;
  static constexpr int WAVE_BYTES = 2 * TILE_BYTES + (E8 ? 2 * TOK * 4 : 0);
  static constexpr int MERGE_ROW = D + 4;  // floats; rows four banks apart
  static constexpr int MERGE_BYTES = WAVES * FEW * MERGE_ROW * 4 + WAVES * FEW * 8;
  static constexpr int MARKS = WAVES * WAVE_BYTES > MERGE_BYTES ? WAVES * WAVE_BYTES : MERGE_BYTES;
  static constexpr int LIMITS = MARKS + FEW * 64;
  static constexpr int LDS = LIMITS + FEW * 4;
};

// What a block of few rows does: rows 0 .. rows - 1 (at most 16) from query q0 on over the tokens of `src`, of which it
// takes split `split` of `splits`; results to slot `slot`.
struct FewTask {
  int h, q0, rows, split, splits, slot;
  Tokens src;
  bool own;    // own tokens of the sequence `seq`, or the prefix of sequences b0 .. b1 - 1
  Seq seq;
  int b0, b1;
};

template <int DT, bool E8, int D>
__device__ __forceinline__ void attend_few(const Args& a, char* smem, const FewTask& f) {
  constexpr int SH = 16;
  typedef FewLayout<DT, E8, D> L;
  typedef Wave<DT, E8, D, SH> W;
  typedef typename W::Y::el el;
  constexpr int TOK = L::TOK, RB = L::RB, NI = TOK * RB / 1024, ESIZE = E8 ? 1 : 2;
  typedef Copier<RB, NI> Copy;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int row = lane % SH, h = f.h;
  const Tokens src = f.src;
  const bool valid = row < f.rows;
  const int t = f.q0 + row / a.grp, hq = h * a.grp + row % a.grp;

  // tokens of `src` that the row attends to: its position is that of the last n_q tokens of its sequence
  int limit = 0x7FFFFFFF;
  if (valid) {
    const Seq s = f.own ? f.seq : sequence(a, sequence_of(a, t, f.b0, f.b1));
    const int end = s.own - s.n_q + (t - s.q0) + 1;  // own tokens up to and with the query
    limit = clamp_int(f.own ? end : src.len + end, 0, src.len);
  }

  W w;
  w.init((const el*)a.q + t * a.q_st + hq * a.q_sh, valid, a.flip, a.keep);

  const int tiles = (src.len + TOK - 1) / TOK;
  const int lo = (int)((int64_t)tiles * f.split / f.splits), hi = (int)((int64_t)tiles * (f.split + 1) / f.splits);
  const int n0 = lo + (hi - lo) * wave / WAVES, n1 = lo + (hi - lo) * (wave + 1) / WAVES;

  const uint32_t kbase = lds_addr(smem) + wave * L::WAVE_BYTES, vbase = kbase + L::TILE_BYTES;
  const uint32_t sbase = vbase + L::TILE_BYTES, marks = lds_addr(smem) + L::MARKS, limits = lds_addr(smem) + L::LIMITS;
  for (int i = threadIdx.x; i < FEW * 16; i += THREADS) *(uint32_t*)(smem + L::MARKS + 4 * i) = 0;
  if (wave == 0 && lane < SH) *(int*)(smem + L::LIMITS + 4 * lane) = limit;
  __syncthreads();
  const char* kp = a.kc + h * a.c_head * ESIZE;
  const char* vp = a.vc + h * a.c_head * ESIZE;
  Window win;
  auto cover = [&](int n) __attribute__((always_inline)) {
    const int t0 = n * TOK;
    win.cover(src, t0 >> a.page_shift, min(t0 + TOK - 1, src.len - 1) >> a.page_shift, a.n_pages);
  };
  auto fill_keys = [&](int n) __attribute__((always_inline)) {
    Copy::run(a, win, src, kp, kbase, n * TOK, ESIZE, [](int r) { return swizzle_k<RB>(r); });
  };
  auto fill_values = [&](int n) __attribute__((always_inline)) {
    Copy::run(a, win, src, vp, vbase, n * TOK, ESIZE, [](int r) { return swizzle_v<RB, SH, E8>(r); });
  };
  auto fill_scales = [&](int n) __attribute__((always_inline)) {  // 32 tokens a copy: keys' scales, then values'
#pragma unroll
    for (int i = 0; i < TOK / 32; ++i) {
      const int tok = min(n * TOK + i * 32 + (lane & 31), src.len - 1);
      const int page = __builtin_amdgcn_ds_bpermute(((tok >> a.page_shift) - win.first) << 2, win.ids);
      const int64_t off = page * a.s_page + h * a.s_head + (tok & ((1 << a.page_shift) - 1)) * a.s_slot;
      dma4(sbase + i * 256, (const char*)((lane < 32 ? a.ks : a.vs) + off));
    }
  };

  // Keys and values have one buffer each: the next keys are fetched from when the
  // scores are done, the next values from when the outputs are.
  if (n0 < n1) {
    cover(n0);
    if (E8) fill_scales(n0);
    fill_keys(n0);
    fill_values(n0);
  }
  for (int n = n0; n < n1; ++n) {
    const int t0 = n * TOK;
    const bool full = __all(limit >= t0 + TOK);
    typename W::acc_t s[TOK / SH];
    typename W::v8 p[TOK / W::KS];
    wait_vm<NI>();  // keys (and scales) are there; the values may be on their way
    w.template scores<TOK>(kbase, s);
    if (E8) w.template weights<TOK>(s, t0, limit, full, a.scale_log2, sbase, 0, p);
    wait_lds();
    if (n + 1 < n1) {
      cover(n + 1);
      if (E8) fill_scales(n + 1);
      fill_keys(n + 1);
    }
    if (!E8) w.template weights<TOK>(s, t0, limit, full, a.scale_log2, sbase, 0, p);
    if (n + 1 < n1) wait_vm<NI + (E8 ? TOK / 32 : 0)>(); else wait_vm<0>();
    if (!full) {
      W::template set_apart<TOK>(vbase, 0, t0, f.rows, marks, [&](int r) { return lds_read<int>(limits + 4 * r); });
      wait_lds();
    }
    w.template values<TOK>(vbase, p);
    wait_lds();
    if (n + 1 < n1) fill_values(n + 1);
  }

  // join the four wavefronts
  float l = W::over_groups_sum(w.l);
  float* merge = (float*)smem;
  float2* ml = (float2*)(merge + WAVES * FEW * L::MERGE_ROW);
  __syncthreads();  // every wavefront is done with its tiles
  if (lane < SH) ml[wave * FEW + row] = float2{w.m, l};
  __syncthreads();
  float top = NEG_INF;
#pragma unroll
  for (int i = 0; i < WAVES; ++i) top = fmaxf(top, ml[i * FEW + row].x);
  const float alpha = __builtin_amdgcn_exp2f(w.m - (top == NEG_INF ? 0.0f : top));
  const int g = lane / SH;
#pragma unroll
  for (int d = 0; d < W::DT_N; ++d)
#pragma unroll
    for (int r = 0; r < W::REGS; r += 4) {
      f32x4 x;
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = w.o[d][r + i] * alpha;
      *(f32x4*)(merge + (wave * FEW + row) * L::MERGE_ROW + d * SH + W::token_of(r, g)) = x;
    }
  __syncthreads();
  const Args b = reload();
  for (int i = threadIdx.x; i < f.rows * (D / 4); i += THREADS) {
    const int r = i / (D / 4), c = (i % (D / 4)) * 4;
    float m = NEG_INF, sum = 0.0f;
#pragma unroll
    for (int k = 0; k < WAVES; ++k) m = fmaxf(m, ml[k * FEW + r].x);
    const float use = m == NEG_INF ? 0.0f : m;
    f32x4 x{};
#pragma unroll
    for (int k = 0; k < WAVES; ++k) {
      const float2 e = ml[k * FEW + r];
      sum += e.y * __builtin_amdgcn_exp2f(e.x - use);
      x += *(const f32x4*)(merge + (k * FEW + r) * L::MERGE_ROW + c);
    }
    x = W::marked(x, marks, r, c);
    const int64_t id = (int64_t)(f.q0 + r / b.grp) * b.Hq + h * b.grp + r % b.grp;
    if (b.direct) {
      store4((el*)b.out + id * D + c, x * inverse(sum));
      if (c == 0) b.lse[id] = natural_lse(m, sum);
    } else {
      *(f32x4*)(b.part_o + ((int64_t)f.slot * b.T * b.Hq + id) * D + c) = x;
      if (c == 0) b.part_ml[(int64_t)f.slot * b.T * b.Hq + id] = float2{m, sum};
    }
  }
}

// Outputs of queries t0 .. t1 - 1 that attend to nothing.
template <int DT, int D>
__device__ __forceinline__ void empty_rows(const Args& a, int h, int t0, int t1) {
  for (int t = t0; t < t1; ++t) {
    const int64_t id = (int64_t)t * a.Hq + h * a.grp;
    for (int i = threadIdx.x; i < a.grp * D; i += THREADS) ((typename Ty<DT>::el*)a.out)[id * D + i] = 0;
    for (int i = threadIdx.x; i < a.grp; i += THREADS) a.lse[id + i] = NEG_INF;
  }
}

// Block `index`: own tokens of sequence b (b < B) or prefix of group b - B; key/value head; split.
template <int DT, bool E8, int D>
__device__ __forceinline__ void few_rows(const Args& a, char* smem, int index) {
  constexpr int TOK = FewLayout<DT, E8, D>::TOK;
  const int own_blocks = a.B * a.Hkv * a.S2;
  FewTask f;
  f.own = index < own_blocks;
  if (!f.own) index -= own_blocks;
  const int heads = (f.own ? a.B : a.G) * a.Hkv, unit = index % heads, b = unit / a.Hkv;
  f.h = unit % a.Hkv;
  f.split = index / heads;
  f.slot = f.own ? a.S1 + f.split : f.split;
  if (f.own) {
    if (a.direct && b == 0) {  // rows of no sequence
      const int first = query_start(a, 0);
      empty_rows<DT, D>(a, f.h, 0, first);
      empty_rows<DT, D>(a, f.h, max(query_start(a, a.B), first), a.T);
    }
    f.seq = sequence(a, b);
    f.q0 = f.seq.q0;
    f.rows = f.seq.n_q * a.grp;
    f.src = Tokens{a.pages + (int64_t)b * a.W, a.W, f.seq.own};
    if (a.direct && f.rows > FEW) {  // more queries than max_q announced: nothing was planned for them
      empty_rows<DT, D>(a, f.h, f.q0, f.q0 + f.seq.n_q);
      return;
    }
  } else {
    const Group gr = group(a, b);
    f.q0 = gr.q0;
    f.rows = gr.rows;
    f.src = Tokens{a.prefix_pages + (int64_t)b * a.Wp, a.Wp, gr.len};
    f.b0 = gr.b0;
    f.b1 = gr.b1;
    if (f.rows > FEW) return;  // its tiles write these slots
  }
  // splits of at least two steps a wavefront
  f.splits = clamp_int((f.src.len + 8 * TOK - 1) / (8 * TOK), 1, f.own ? a.S2 : a.S1);
  if (f.rows > FEW || f.split >= f.splits) {
    for (int r = threadIdx.x; r < f.rows; r += THREADS)
      a.part_ml[((int64_t)f.slot * a.T + f.q0 + r / a.grp) * a.Hq + f.h * a.grp + r % a.grp] = float2{NEG_INF, 0.0f};
    return;
  }
  if (f.rows > 0) attend_few<DT, E8, D>(a, smem, f);
}

// ------------------------------------------------------------------ tiles of rows
//
// RW wavefronts side by side hold the tile's 32 * RW rows, 4 / RW wavefronts share the tokens of a step.
template <int DT, bool E8, int D, int RW>
struct TileLayout {
  static constexpr int RB = D * (E8 ? 1 : 2);
  static constexpr int ROWS = 32 * RW;
  static constexpr int TOK = RB == 256 ? 64 : 128;  // tokens of a step
  static constexpr int TILE_BYTES = TOK * RB;
  static constexpr int STAGE = 2 * TILE_BYTES + (E8 ? 2 * TOK * 4 : 0);
  static constexpr int MERGE_ROW = D + 4;
  static constexpr int MARKS = 2 * STAGE;
  static constexpr int ROW_INFO = MARKS + ROWS * 64;
  static constexpr int LDS = ROW_INFO + ROWS * 12;
  static_assert(RW == 4 || MARKS >= ROWS * (MERGE_ROW * 4 + 8), "the merge reuses the stages");
};

// Unit (group, row tile, key/value head) and split of tile block `index`; false past the last one.  Units come in
// rounds of FILL blocks; those of a last, partial round are cut into up to S1 splits that fill the device.  A head's
// units lie S1 and Hkv apart in block numbers, so with 8 heads they run on one XCD, whose L2 then holds the keys and
// values that they share.
struct TileUnit {
  int g, tile, h, split, splits;
};
template <int ROWS>
__device__ __forceinline__ bool find_tile(const Args& a, int index, TileUnit& u) {
  const int lane = threadIdx.x & 63;
  auto count = [&](int x) __attribute__((always_inline)) {  // tiles of group x
    if (x >= a.G) return 0;
    const Group gr = group(a, x);
    return gr.rows > FEW ? (gr.rows + ROWS - 1) / ROWS : 0;
  };
  int n = 0, total = 0;
  for (int x0 = (a.G - 1) / 64 * 64; x0 >= 0; x0 -= 64) {  // downwards: ends with the first groups in registers
    n = count(x0 + lane);
    total += n;
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) total += __shfl_xor(total, d);
  const int units = __builtin_amdgcn_readfirstlane(total) * a.Hkv;
  const int whole = units / FILL * FILL, tail = units - whole;
  const int splits = tail ? clamp_int(FILL / tail, 1, a.S1) : 1;
  int unit = index;
  u.split = 0;
  u.splits = 1;
  if (index >= whole) {
    index -= whole;
    if (index >= tail * splits) return false;
    unit = whole + index % tail;
    u.split = index / tail;
    u.splits = splits;
  }
  u.h = unit % a.Hkv;
  const int tile = unit / a.Hkv;
  int seen = 0;
  for (int x0 = 0; x0 < a.G; x0 += 64) {
    if (x0 > 0) n = count(x0 + lane);
    int incl = n;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int o = __shfl_up(incl, d);
      if (lane >= d) incl += o;
    }
    const int here = __builtin_amdgcn_readfirstlane(__shfl(incl, 63));
    if (tile < seen + here) {
      const int l = __builtin_ctzll(__ballot(seen + incl > tile));
      u.g = __builtin_amdgcn_readfirstlane(x0 + l);
      u.tile = __builtin_amdgcn_readfirstlane(tile - seen - __shfl(incl - n, l));
      return true;
    }
    seen += here;
  }
  return false;
}

template <int DT, bool E8, int D, int RW>
__device__ __forceinline__ void row_tile(const Args& a, char* smem, int index) {
  typedef TileLayout<DT, E8, D, RW> L;
  constexpr int SH = 32, TOK = L::TOK, RB = L::RB, ESIZE = E8 ? 1 : 2;
  constexpr int MINE = TOK / WAVES;            // tokens that a wavefront fetches
  constexpr int NI = MINE * RB / 1024;         // in copies of 1 KiB
  typedef Copier<RB, NI> Copy;
  constexpr int SHARE = TOK * RW / WAVES;      // tokens that a wavefront attends to
  constexpr int MOST = E8 ? 32 : 64;           // in steps of so many (e4m3: 64 would spill)
  constexpr int STEP = SHARE > MOST ? MOST : SHARE;
  static_assert(NI >= 1, "a wavefront fetches whole copies");
  typedef Wave<DT, E8, D, SH> W;
  typedef typename W::Y::el el;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int wr = wave % RW, wt = wave / RW;
  TileUnit u;
  if (!find_tile<L::ROWS>(a, index, u)) return;
  const int h = u.h;
  const Group gr = group(a, u.g);
  const int row = u.tile * L::ROWS + wr * SH + lane % SH;
  const bool valid = row < gr.rows;
  const int t = gr.q0 + row / a.grp, hq = h * a.grp + row % a.grp;

  int b = -1, end = 0, own_limit = 0;
  bool big = false;
  if (valid) {
    b = sequence_of(a, t, gr.b0, gr.b1);
    const Seq s = sequence(a, b);
    end = s.own - s.n_q + (t - s.q0) + 1;
    own_limit = clamp_int(end, 0, s.own);
    big = s.n_q * a.grp > FEW;
  }
  const int prefix_limit = valid ? clamp_int(gr.len + end, 0, gr.len) : 0;

  W w;
  w.init((const el*)a.q + t * a.q_st + hq * a.q_sh, valid, a.flip, a.keep);

  // The tile's tokens: the prefix, then the own tokens (as far as a row of the tile sees them) of each of its
  // sequences with more than 16 rows.  Steps are counted over all of them and shared out to the splits.
  int b_first = gr.b0, b_last = gr.b0 - 1, t_last = 0;
  if (a.big) {
    t_last = gr.q0 + (min((u.tile + 1) * L::ROWS, gr.rows) - 1) / a.grp;
    b_first = sequence_of(a, gr.q0 + u.tile * L::ROWS / a.grp, gr.b0, gr.b1);
    b_last = sequence_of(a, t_last, gr.b0, gr.b1);
  }
  auto own_tokens = [&](int x) __attribute__((always_inline)) {
    const Args again = reload();
    const Seq s = sequence(again, x);
    if (s.n_q * again.grp <= FEW) return 0;
    const int last = min(t_last, s.q0 + s.n_q - 1);
    return clamp_int(s.own - s.n_q + (last - s.q0) + 1, 0, s.own);
  };
  int steps = (gr.len + TOK - 1) / TOK;
  for (int x = b_first; x <= b_last; ++x) steps += (own_tokens(x) + TOK - 1) / TOK;
  steps = __builtin_amdgcn_readfirstlane(steps);
  int skip = (int)((int64_t)steps * u.split / u.splits);
  int todo = (int)((int64_t)steps * (u.split + 1) / u.splits) - skip;

  const uint32_t base = lds_addr(smem), marks = base + L::MARKS, info = base + L::ROW_INFO;
  for (int i = threadIdx.x; i < L::ROWS * 16; i += THREADS) *(uint32_t*)(smem + L::MARKS + 4 * i) = 0;
  // of every row, for the marks: sequence (-1: no row), prefix tokens and own tokens that it sees
  if (wt == 0 && lane < SH) {
    int* p = (int*)(smem + L::ROW_INFO) + wr * SH + lane;
    p[0] = b;
    p[L::ROWS] = prefix_limit;
    p[2 * L::ROWS] = own_limit;
  }
  const char* kp = a.kc + h * a.c_head * ESIZE;
  const char* vp = a.vc + h * a.c_head * ESIZE;

  for (int x = b_first - 1; x <= b_last && todo > 0; ++x) {
    const bool pre = x < b_first;
    const int len = __builtin_amdgcn_readfirstlane(pre ? gr.len : own_tokens(x));
    const int n_all = (len + TOK - 1) / TOK;
    if (skip >= n_all) {
      skip -= n_all;
      continue;
    }
    const int n0 = skip, n1 = min(n_all, skip + todo);
    skip = 0;
    todo -= n1 - n0;
    const Args again = reload();
    const Tokens src = pre ? Tokens{again.prefix_pages + (int64_t)u.g * again.Wp, again.Wp, len}
                           : Tokens{again.pages + (int64_t)x * again.W, again.W, len};
    int limit = pre ? prefix_limit : b == x ? own_limit : 0;
    const bool some = valid && limit > 0;
    if (!valid) limit = 0x7FFFFFFF;
    Window win;
    auto fill = [&](int n) __attribute__((always_inline)) {
      const int t0 = n * TOK + wave * MINE;  // the wavefront's first token
      const uint32_t kb = base + (n & 1) * L::STAGE + wave * MINE * RB;
      win.cover(src, min(t0, src.len - 1) >> a.page_shift, min(t0 + MINE - 1, src.len - 1) >> a.page_shift, a.n_pages);
      Copy::run(a, win, src, kp, kb, t0, ESIZE, [](int r) { return swizzle_k<RB>(r); });
      Copy::run(a, win, src, vp, kb + L::TILE_BYTES, t0, ESIZE, [](int r) { return swizzle_v<RB, SH, E8>(r); });
      if (E8) {
        static_assert(MINE == 32 || !E8, "the scales of 32 tokens a copy");
        const int tok = min(t0 + (lane & 31), src.len - 1);
        const int page = __builtin_amdgcn_ds_bpermute(((tok >> a.page_shift) - win.first) << 2, win.ids);
        const int64_t off = page * a.s_page + h * a.s_head + (tok & ((1 << a.page_shift) - 1)) * a.s_slot;
        dma4(base + (n & 1) * L::STAGE + 2 * L::TILE_BYTES + wave * 256, (const char*)((lane < 32 ? a.ks : a.vs) + off));
      }
    };
    // both stages may still be read from the segment before; the rows' limits are there after this
    __syncthreads();
    fill(n0);
    auto limit_of = [&](int r) {
      const int rb = lds_read<int>(info + 4 * r);
      return rb < 0 ? 0 : pre ? lds_read<int>(info + 4 * (L::ROWS + r))
                              : rb == x ? lds_read<int>(info + 4 * (2 * L::ROWS + r)) : 0;
    };
    int seen_by_all = 0x7FFFFFFF;  // tokens that every row of the tile sees
#pragma unroll
    for (int r = 0; r < L::ROWS; r += 64)
      if (lds_read<int>(info + 4 * (r + lane)) >= 0) seen_by_all = min(seen_by_all, limit_of(r + lane));
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) seen_by_all = min(seen_by_all, __shfl_xor(seen_by_all, d));
    seen_by_all = __builtin_amdgcn_readfirstlane(seen_by_all);
    for (int n = n0; n < n1; ++n) {
      const uint32_t stage = base + (n & 1) * L::STAGE;
      wait_vm<0>();
      if ((n + 1) * TOK > seen_by_all)  // each wavefront looks at the tokens it has fetched
        W::template set_apart<MINE>(stage + L::TILE_BYTES, wave * MINE, n * TOK, L::ROWS, marks, limit_of);
      wait_lds();
      __builtin_amdgcn_s_barrier();  // the step's tokens are there, the other stage is free
      if (n + 1 < n1) fill(n + 1);
#pragma unroll
      for (int c = 0; c < SHARE / STEP; ++c) {
        const int tok0 = wt * SHARE + c * STEP, t0 = n * TOK + tok0;
        if (!__any(some && limit > t0)) continue;
        const bool full = __all(limit >= t0 + STEP);
        const uint32_t kb = stage + tok0 * RB;
        typename W::acc_t s[STEP / SH];
        typename W::v8 p[STEP / W::KS];
        w.template scores<STEP>(kb, s);
        w.template weights<STEP>(s, t0, limit, full, a.scale_log2, stage + 2 * L::TILE_BYTES, tok0, p);
        w.template values<STEP>(kb + L::TILE_BYTES, p);
      }
    }
  }

  float l = W::over_groups_sum(w.l), alpha = 1.0f;
  const int gx = lane / SH;
  float* merge = (float*)smem;
  float2* ml = (float2*)(merge + L::ROWS * L::MERGE_ROW);
  __syncthreads();  // all marks are made
  if (RW < WAVES) {
    // the wavefronts that share a row: the second hands its results to the first
    static_assert(RW == WAVES || RW * 2 == WAVES, "two halves");
    const int r = wr * SH + lane % SH;
    if (wt == 1) {
#pragma unroll
      for (int d = 0; d < W::DT_N; ++d)
#pragma unroll
        for (int i = 0; i < W::REGS; i += 4) {
          f32x4 x;
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = w.o[d][i + e];
          *(f32x4*)(merge + r * L::MERGE_ROW + d * SH + W::token_of(i, gx)) = x;
        }
      if (gx == 0) ml[r] = float2{w.m, l};
    }
    __syncthreads();
    if (wt == 1) return;
    const float2 other = ml[r];
    const float top = fmaxf(w.m, other.x), use = top == NEG_INF ? 0.0f : top;
    alpha = __builtin_amdgcn_exp2f(w.m - use);
    const float beta = __builtin_amdgcn_exp2f(other.x - use);
    l = l * alpha + other.y * beta;
    w.m = top;
#pragma unroll
    for (int d = 0; d < W::DT_N; ++d)
#pragma unroll
      for (int i = 0; i < W::REGS; i += 4) {
        const f32x4 x = *(const f32x4*)(merge + r * L::MERGE_ROW + d * SH + W::token_of(i, gx));
#pragma unroll
        for (int e = 0; e < 4; ++e) w.o[d][i + e] = w.o[d][i + e] * alpha + x[e] * beta;
      }
  }
  if (!valid) return;
  const Args e = reload();
  const int64_t id = (int64_t)t * e.Hq + hq, slots = (int64_t)e.T * e.Hq, slot = u.split * slots + id;
  const bool final = u.splits == 1 && big;
  const float inv = final ? inverse(l) : 1.0f;
#pragma unroll
  for (int d = 0; d < W::DT_N; ++d)
#pragma unroll
    for (int r = 0; r < W::REGS; r += 4) {
      f32x4 x;
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = w.o[d][r + i] * inv;
      const int c = d * SH + W::token_of(r, gx);
      x = W::marked(x, marks, wr * SH + lane % SH, c);
      if (final)
        store4((el*)e.out + id * D + c, x);
      else if (!(l == 0.0f))
        *(f32x4*)(e.part_o + slot * D + c) = x;
    }
  if (gx == 0) {
    e.part_ml[slot] = float2{w.m, final ? -1.0f : l};
    if (final) e.lse[id] = natural_lse(w.m, l);
    if (u.split == 0 && !final)  // the slots that other tiles use
      for (int k = u.splits; k < e.S1; ++k) e.part_ml[k * slots + id] = float2{NEG_INF, 0.0f};
  }
}

// Tile blocks first (the longest ones), then those of few rows.
template <int DT, bool E8, int D, int RW>
__global__ void __launch_bounds__(THREADS, 2) attend(Args a) {
  extern __shared__ __align__(16) char smem[];
  const int index = (int)blockIdx.x;
  if (index < a.tile_blocks)
    row_tile<DT, E8, D, RW>(a, smem, index);
  else
    few_rows<DT, E8, D>(a, smem, index - a.tile_blocks);
}

// ------------------------------------------------------------------ combine

// One wavefront a row: lane s reads the maximum and sum of slots s and s + 64, then all lanes add the slots' outputs
// in order, eight of them in flight.
template <int DT, int D>
__global__ void __launch_bounds__(THREADS) combine(Args a) {
  typedef typename Ty<DT>::el el;
  constexpr int PER = D / 64, AT_ONCE = 8;
  struct alignas(4 * PER) Part { float x[PER]; };
  struct alignas(2 * PER) Out { el x[PER]; };
  const int lane = threadIdx.x & 63;
  const int64_t rows = (int64_t)a.T * a.Hq, id = (int64_t)blockIdx.x * WAVES + (threadIdx.x >> 6);
  if (id >= rows) return;
  const int slots = a.S1 + a.S2;
  float2 ml[2] = {float2{NEG_INF, 0.0f}, float2{NEG_INF, 0.0f}};
  const int t = (int)(id / a.Hq), first = query_start(a, 0), end = query_start(a, a.B);
#pragma unroll
  for (int i = 0; i < 2; ++i)
    if (lane + 64 * i < slots) ml[i] = a.part_ml[(lane + 64 * i) * rows + id];
  if (t < first || t >= end) ml[0] = ml[1] = float2{NEG_INF, 0.0f};  // a row of no sequence
  if (__any(ml[0].y < 0.0f)) return;  // written by its tile
  float top = fmaxf(ml[0].x, ml[1].x);
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
  float weight[2], sum = 0.0f;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    weight[i] = __builtin_amdgcn_exp2f(ml[i].x - (top == NEG_INF ? 0.0f : top));
    sum += weight[i] * ml[i].y;
  }
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d);
  float x[PER] = {};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    unsigned long long live = __ballot(!(ml[i].y == 0.0f));  // a NaN counts
    while (live) {
      Part p[AT_ONCE];
      float w[AT_ONCE];
#pragma unroll
      for (int k = 0; k < AT_ONCE; ++k) {
        const int s = live ? __builtin_ctzll(live) : 0;
        w[k] = live ? __shfl(weight[i], s) : 0.0f;
        p[k] = Part{};
        if (live) p[k] = *(const Part*)(a.part_o + ((s + 64 * i) * rows + id) * D + lane * PER);
        live &= live - 1;
      }
#pragma unroll
      for (int k = 0; k < AT_ONCE; ++k)
#pragma unroll
        for (int e = 0; e < PER; ++e) x[e] += w[k] * p[k].x[e];
    }
  }
  const float inv = inverse(sum);
  Out o;
#pragma unroll
  for (int e = 0; e < PER; ++e) o.x[e] = (el)(x[e] * inv);
  *(Out*)((el*)a.out + id * D + lane * PER) = o;
  if (lane == 0) a.lse[id] = natural_lse(top, sum);
}

// ------------------------------------------------------------------ host

struct Plan {
  int64_t tile_blocks = 0;  // an upper bound
  int row_waves = 2;        // tiles of 64 or 128 rows
  int S1 = 0, S2 = 1;
  int64_t few_blocks = 0;
  bool combine = true;
  int64_t bytes = 0;
};

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline int64_t between(int64_t x, int64_t lo, int64_t hi) { return x < lo ? lo : x > hi ? hi : x; }

// Tiles of 128 rows where they fill the device by themselves, else of 64 (fewer splits, so fewer partial results).
// Splits of at least 256 tokens.
inline Plan make_plan(int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t G, int64_t Wp, int64_t B, int64_t W,
                      int64_t page, int64_t max_q) {
  Plan p;
  const int64_t grp = Hq / Hkv, rows = T * grp, groups = G > 0 ? G : 1;
  const bool big = max_q * grp > FEW;
  if (rows > FEW && (Wp > 0 || big)) {
    p.row_waves = ceil_div(rows, 128) * Hkv >= FILL ? 4 : 2;
    const int64_t tile = 32 * p.row_waves;
    const int64_t tokens = (Wp + (big ? W : 0)) * page;
    // a last round of `tail` units is cut into FILL / tail splits; with one group the number of tiles is known
    const int64_t units = ceil_div(rows, tile) * Hkv, tail = units % FILL;
    const int64_t most = groups == 1 ? (units < FILL ? FILL / units : tail ? FILL / tail : 1) : FILL / Hkv;
    p.S1 = (int)between(most, 1, between(ceil_div(tokens, 256), 1, units < FILL ? MAX_SPLIT : 8));
    p.tile_blocks = (rows / tile + groups) * Hkv + FILL;
  } else if (Wp > 0) {
    p.S1 = (int)between(FILL / (groups * Hkv), 1, between(ceil_div(Wp * page, 256), 1, MAX_SPLIT));
  }
  p.S2 = (int)between(FILL / (B * Hkv), p.S1 > 0 ? 4 : 1, between(ceil_div(W * page, 256), 1, MAX_SPLIT));
  if (p.S2 > ceil_div(W * page, 256)) p.S2 = (int)ceil_div(W * page, 256);
  p.few_blocks = B * Hkv * p.S2 + (p.S1 > 0 ? groups * Hkv * p.S1 : 0);
  p.combine = !(p.S1 == 0 && p.S2 == 1);
  p.bytes = p.combine ? (int64_t)(p.S1 + p.S2) * T * Hq * (D * 4 + 8) : 0;
  return p;
}

template <int DT, bool E8, int D, int RW>
tb_status launch(Args& a, const Plan& p, hipStream_t stream, const char* what) {
  constexpr int few = FewLayout<DT, E8, D>::LDS, tile = TileLayout<DT, E8, D, RW>::LDS;
  constexpr size_t lds = few > tile ? few : tile;
  static_assert(lds <= 81920, "two blocks a CU");
  if (tb_status s = reserve_lds((const void*)attend<DT, E8, D, RW>, lds, what)) return s;
  hipLaunchKernelGGL((attend<DT, E8, D, RW>), dim3((unsigned)(p.tile_blocks + p.few_blocks)), dim3(THREADS), lds, stream,
                     a);
  if (tb_status s = launch_status(what)) return s;
  if (!p.combine) return TB_OK;
  hipLaunchKernelGGL((combine<DT, D>), dim3((unsigned)ceil_div((int64_t)a.T * a.Hq, WAVES)), dim3(THREADS), 0, stream, a);
  return launch_status(what);
}

template <int DT, bool E8, int D>
tb_status launch_rows(Args& a, const Plan& p, hipStream_t stream, const char* what) {
  return p.row_waves == 4 ? launch<DT, E8, D, 4>(a, p, stream, what) : launch<DT, E8, D, 2>(a, p, stream, what);
}

template <int DT>
tb_status launch_for(bool e8, int64_t D, Args& a, const Plan& p, hipStream_t stream, const char* what) {
  if (D == 64) return e8 ? launch_rows<DT, true, 64>(a, p, stream, what) : launch_rows<DT, false, 64>(a, p, stream, what);
  return e8 ? launch_rows<DT, true, 128>(a, p, stream, what) : launch_rows<DT, false, 128>(a, p, stream, what);
}

tb_status check_sizes(const char* what, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t G, int64_t Wp, int64_t B,
                      int64_t W, int64_t page_size, int64_t max_q) {
  TB_CHECK_ARG(T >= 0 && B >= 0 && G >= 0 && Wp >= 0 && W >= 0 && max_q >= 0, "%s: negative size", what);
  TB_CHECK_ARG(Hkv >= 1 && Hq >= Hkv && Hq % Hkv == 0, "%s: %lld query heads do not share %lld key/value heads",
               what, (long long)Hq, (long long)Hkv);
  TB_CHECK_ARG(D == 64 || D == 128, "%s: the head dimension must be 64 or 128 (got %lld)", what, (long long)D);
  TB_CHECK_ARG(page_size >= 1 && page_size <= 4096 && (page_size & (page_size - 1)) == 0,
               "%s: the page size must be a power of two up to 4096 (got %lld)", what, (long long)page_size);
  TB_CHECK_ARG((Wp == 0) == (G == 0), "%s: %lld groups with page tables of %lld", what, (long long)G, (long long)Wp);
  const int64_t most = (1ll << 31) - 1;
  // row, token and block numbers are 32-bit in the kernels
  TB_CHECK_ARG(T * Hq <= most && B * Hkv <= most / MAX_SPLIT / 4 && G * Hkv <= most / MAX_SPLIT / 4 && W <= most / 2 / page_size &&
                   Wp <= most / 2 / page_size && max_q * Hq <= most,
               "%s: sizes past 2^31", what);
  return TB_OK;
}

}  // namespace prefix
}  // namespace tb

extern "C" tb_status tb_shared_prefix_attention_workspace_size(int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t G,
                                                               int64_t Wp, int64_t B, int64_t W, int64_t page_size,
                                                               int64_t max_q, int64_t* bytes) {
  using namespace tb::prefix;
  const char* what = "tb_shared_prefix_attention_workspace_size";
  TB_CHECK_ARG(bytes, "%s: null pointer", what);
  if (tb_status s = check_sizes(what, T, Hq, Hkv, D, G, Wp, B, W, page_size, max_q)) return s;
  *bytes = T == 0 ? 0 : make_plan(T, Hq, Hkv, D, G, Wp, B, W, page_size, max_q).bytes;
  return TB_OK;
}

extern "C" tb_status tb_shared_prefix_attention(const void* q, const void* k_cache, const void* v_cache,
                                                const float* k_scale, const float* v_scale,
                                                const int32_t* prefix_pages, const int32_t* prefix_lens,
                                                const int32_t* group_offsets, const int32_t* pages,
                                                const int32_t* lens, const int32_t* cu_q, void* out, float* lse,
                                                int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t G, int64_t Wp,
                                                int64_t B, int64_t W, int64_t max_q, int64_t n_pages,
                                                int64_t page_size, int64_t q_st, int64_t q_sh, int64_t c_page,
                                                int64_t c_head, int64_t c_slot, int64_t s_page, int64_t s_head,
                                                int64_t s_slot, double scale, int dtype, int cache_dtype,
                                                void* workspace, int64_t workspace_bytes, hipStream_t stream) {
  using namespace tb::prefix;
  const char* what = "tb_shared_prefix_attention";
  if (tb_status s = check_sizes(what, T, Hq, Hkv, D, G, Wp, B, W, page_size, max_q)) return s;
  TB_CHECK_ARG(dtype == F16 || dtype == BF16, "%s: unknown dtype %d", what, dtype);
  TB_CHECK_ARG(cache_dtype == dtype || cache_dtype == 3, "%s: the cache holds %d, the queries are %d (3 is e4m3)", what,
               cache_dtype, dtype);
  TB_CHECK_ARG((cache_dtype == 3) == (k_scale != nullptr) && (cache_dtype == 3) == (v_scale != nullptr),
               "%s: scales belong to e4m3 caches, and only to them", what);
  TB_CHECK_ARG(scale - scale == 0.0, "%s: the scale must be finite", what);
  TB_CHECK_ARG(n_pages >= 1 && n_pages <= ((1ll << 31) - 1) / page_size, "%s: bad number of pages %lld", what,
               (long long)n_pages);
  if (T == 0) return TB_OK;
  TB_CHECK_ARG(B >= 1 && W >= 1, "%s: queries without sequences", what);
  TB_CHECK_ARG(q && k_cache && v_cache && pages && lens && cu_q && out && lse, "%s: null pointer", what);
  TB_CHECK_ARG(G == 0 || (prefix_pages && prefix_lens && group_offsets), "%s: null pointer", what);
  TB_CHECK_ALIGN(q, 16, "q");
  TB_CHECK_ALIGN(k_cache, 16, "k_cache");
  TB_CHECK_ALIGN(v_cache, 16, "v_cache");
  TB_CHECK_ALIGN(out, 16, "out");
  const int64_t chunk = cache_dtype == 3 ? 16 : 8;  // elements of 16 bytes
  TB_CHECK_ARG(q_st % 8 == 0 && q_sh % 8 == 0, "%s: q's strides must be multiples of 8 elements", what);
  TB_CHECK_ARG(c_page % chunk == 0 && c_head % chunk == 0 && c_slot % chunk == 0,
               "%s: the cache's strides must be multiples of 16 bytes", what);
  const Plan p = make_plan(T, Hq, Hkv, D, G, Wp, B, W, page_size, max_q);
  if (p.bytes > 0 && (!workspace || workspace_bytes < p.bytes)) {
    tb::set_error("%s: needs a workspace of %lld bytes, got %lld", what, (long long)p.bytes,
                  (long long)(workspace ? workspace_bytes : 0));
    return TB_E_WORKSPACE;
  }
  if (p.bytes > 0) TB_CHECK_ALIGN(workspace, 16, "workspace");
  Args a{};
  a.q = q;
  a.q_st = q_st;
  a.q_sh = q_sh;
  a.kc = (const char*)k_cache;
  a.vc = (const char*)v_cache;
  a.c_page = c_page;
  a.c_head = c_head;
  a.c_slot = c_slot;
  a.ks = k_scale;
  a.vs = v_scale;
  a.s_page = s_page;
  a.s_head = s_head;
  a.s_slot = s_slot;
  a.prefix_pages = prefix_pages;
  a.prefix_lens = G > 0 ? prefix_lens : nullptr;
  a.group_offsets = G > 0 ? group_offsets : nullptr;
  a.pages = pages;
  a.lens = lens;
  a.cu_q = cu_q;
  a.out = out;
  a.lse = lse;
  a.part_o = (float*)workspace;
  a.part_ml = (float2*)((char*)workspace + (int64_t)(p.S1 + p.S2) * T * Hq * D * 4);
  a.T = (int)T;
  a.Hq = (int)Hq;
  a.Hkv = (int)Hkv;
  a.grp = (int)(Hq / Hkv);
  a.G = G > 0 ? (int)G : 1;
  a.Wp = (int)Wp;
  a.B = (int)B;
  a.W = (int)W;
  a.n_pages = (int)n_pages;
  a.page_shift = __builtin_ctzll((unsigned long long)page_size);
  a.S1 = p.S1;
  a.S2 = p.S2;
  a.direct = !p.combine;
  a.scale_log2 = scale == 0.0 ? 1.0f : (float)((scale < 0.0 ? -scale : scale) * 1.44269504088896340736);
  a.flip = scale < 0.0 ? 0x80008000u : 0u;
  a.keep = scale == 0.0 ? 0u : ~0u;
  a.near = c_slot >= 0 && c_slot < (1 << 23);
  a.big = max_q * a.grp > FEW;
  a.tile_blocks = (int)p.tile_blocks;
  const bool e8 = cache_dtype == 3;
  return dtype == F16 ? launch_for<F16>(e8, D, a, p, stream, what) : launch_for<BF16>(e8, D, a, p, stream, what);
}
