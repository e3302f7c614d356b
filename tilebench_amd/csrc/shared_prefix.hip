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
//   tiles   64 or 128 rows of a group: over the shared prefix, and on over the own
//           tokens of those sequences that have more than 16 rows
//   streams the own tokens of the sequences of up to 16 rows, laid end to end and
//           shared out evenly to the wavefronts
//   combine joins the partial results of a row (one slot per split) by their maxima
// so a prefix is read once per tile however many sequences share it.  Short calls
// are done by a block for each sequence and head (attend_each).
//
// One wavefront's step over TOK tokens in LDS:
//   S^T = K Q^T    K rows from LDS, Q in registers; a lane holds one row's scores
//   P^T            exp2 of the scores against the running maximum, in registers; the
//                  tokens a lane holds are in the order of the next product's operand
//   O^T = V^T P^T  V^T by transposing LDS reads (ds_read_b64_tr_b16 / _b8) in that order
// so scores never leave registers, and the maximum, sum and output of a row belong to
// the lanes that hold the row.  Sums and statistics are fp32.  P is rounded to the
// inputs' type for the second product (2^-11 or 2^-8 of each weight, unbiased).
//
// e4m3 caches: codes are converted exactly to the inputs' type (in tiles once on
// the way to LDS); the keys' scales multiply the scores, the values' scales the
// weights.
//
// What bounds it, and what it takes (kernel, us, in a kernel trace):
//   prompts behind 6000 tokens (bf16, 32 heads)   525   matrix cores 44 % busy at 1.9 GHz, vector work
//              47 %: the exponentials take as long again; 910 TFLOP/s of a call (matrix products 1325)
//   8 queries about 131001 tokens (64 heads)      107   memory, 5.2 TB/s
//   64 decodes behind 8192, up to 1024 own         31   half of it the first loads and the last
//              results of blocks that live for 20 us
//   96 x 1-2 queries, four e4m3 prefixes           91   vector work: 19 instructions a product
// and 6 to 13 for the combine.  Why tiles of 64 or 128 rows, streams and shares are as they are is said
// at each; the first kernel, with a launch for each kind of work, took 772, 171, 83 and 169 in all.
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
typedef float f32x2 __attribute__((ext_vector_type(2)));

enum { F16 = 1, BF16 = 2 };
constexpr int THREADS = 256, WAVES = 4;
constexpr int FEW = 16;      // rows of a sequence that the token-splitting blocks take
constexpr int FILL = 512;    // blocks that fill the device: two on each of 256 CUs
constexpr int MAX_SPLIT = 64;
constexpr int64_t PARTIALS = 512 << 20;  // bytes of partial results from which only rows that need them have some
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
  float* part_o;    // [slots][D]: partial outputs, those of a row together (see Slots)
  float2* part_ml;  // [slots]: maximum (log2) and sum
  int* n_tile;      // [T * Hq]: slots that the row's tiles used, -1 where its result is final
  int* n_own;       // [T * Hq]: slots that its own tokens used
  int* tile_at;     // [T * Hq], compact: the first of the tiles' slots, -1 for the one beside the own tokens'
  int* own_at;      // [T * Hq], compact: which of own_rows the row is
  int compact, tile_slots, own_rows;
  int direct_rows;  // own_rows are the rows of the call, else FEW for each sequence and key/value head
  int own_first, own_stride;  // slots: own row n has its from own_first + n * own_stride on
  int T, Hq, Hkv, grp, G, Wp, B, W;
  Divisor by_grp, by_heads;  // grp, Hkv
  int n_pages, page_shift;
  int S1, S2;       // slots of tiles, slots of own tokens
  int tile_fill;    // blocks that the tiles are shared out to
  int streams;      // wavefronts that the own tokens are shared out to
  int stream_least; // steps of one of them at least
  float scale_log2;     // of |scale|, or 1 for a scale of 0
  uint32_t flip, keep;  // applied to q
  int joint;   // sequences read their prefix themselves
  int rounds;  // at least FILL units of tiles
  int near;  // 64 slots of a page lie within 2 GiB
  int big;  // some sequence may have more than FEW rows
  int tile_blocks;
};

// The kernel's arguments once more, from LDS.  Epilogues and other code off the loops take theirs from here: fields that
// are only needed there would hold scalar registers through the loops, which then spill, and reading the argument
// segment again takes 2 us.
constexpr int ARG_WORDS = sizeof(Args) / 4;
static_assert(ARG_WORDS <= THREADS && sizeof(Args) % 4 == 0, "a word a thread");
__device__ __forceinline__ uint32_t argument_word() {
  const __attribute__((address_space(4))) uint32_t* p =
      (const __attribute__((address_space(4))) uint32_t*)__builtin_amdgcn_kernarg_segment_ptr();
  return p[min((int)threadIdx.x, ARG_WORDS - 1)];
}
template <typename V>
__device__ __forceinline__ V lds_read(uint32_t addr);
__device__ __forceinline__ Args saved_args(uint32_t at) {
  struct {
    uint32_t w[ARG_WORDS];
  } x;
#pragma unroll
  for (int i = 0; i < ARG_WORDS; ++i) x.w[i] = lds_read<uint32_t>(at + 4 * i);
  return __builtin_bit_cast(Args, x);
}
__device__ __forceinline__ const int* uniform(const int* p) {
  const uint64_t u = (uint64_t)(uintptr_t)p;
  return (const int*)(uintptr_t)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)u) |
                                 (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(u >> 32)) << 32);
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
  return RB == 128 ? ((t >> 1) & 3) | ((t >> 4) & 1) << 2 : ((t >> 2) & 1) | ((t >> 4) & 1) << 1;
}

typedef __attribute__((address_space(3))) char lds_char;
__device__ __forceinline__ uint32_t lds_addr(const void* p) {
  return (uint32_t)(uintptr_t)(lds_char*)p;
}
template <typename V>
__device__ __forceinline__ V lds_read(uint32_t addr) {
  return *(const __attribute__((address_space(3))) V*)(uintptr_t)addr;
}

// 16 (or 4) bytes a lane from global memory to LDS at lds + 16 (4) * lane.  One wait state lies between a scalar write of
// m0 and such a load, which would else find the m0 before it: the compiler keeps none within inline asm.
__device__ __forceinline__ void dma16(uint32_t lds, const char* p) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
               :
               : "s"(__builtin_amdgcn_readfirstlane((int)lds)), "v"(p)
               : "memory", "m0");
}
// the same from a uniform address plus a 32-bit offset of each lane.  The address is copied by a scalar instruction,
// which is that wait state too: it may come from a vector one (readfirstlane), and five would lie between that and a load.
__device__ __forceinline__ void dma16(uint32_t lds, const char* p, uint32_t off) {
  const uint64_t u = (uint64_t)(uintptr_t)p;
  const uint64_t base = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)u) |
                        (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(u >> 32)) << 32;
  uint64_t at;
  asm volatile("s_mov_b32 m0, %1\n\ts_mov_b64 %0, %3\n\tglobal_load_lds_dwordx4 %2, %0"
               : "=&s"(at)
               : "s"(__builtin_amdgcn_readfirstlane((int)lds)), "v"(off), "s"(base)
               : "memory", "m0");
}
__device__ __forceinline__ void dma4(uint32_t lds, const char* p) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off"
               :
               : "s"(__builtin_amdgcn_readfirstlane((int)lds)), "v"(p)
               : "memory", "m0");
}
// Waits until at most N of this wavefront's vector memory operations are pending.
template <int N>
__device__ __forceinline__ void wait_vm() {
  asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory");
}
// A barrier for LDS contents that leaves vector memory operations pending (__syncthreads waits for them).
__device__ __forceinline__ void block_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" : : : "memory");
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
  __device__ __forceinline__ void reset() { first = 0x7FFFFFFF; }
  __device__ __forceinline__ void cover(const Tokens& s, int lo, int hi, int n_pages) {
    if (lo >= first && hi - 64 < first) return;
    first = lo;
    int id = ((const __attribute__((address_space(1))) int*)s.table)[min(lo + (int)(threadIdx.x & 63), s.width - 1)];
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
// E8: the tiles hold e4m3 codes (else 16-bit values); SC: keys and values have scales.
template <int DT, bool E8, int D, int SH, bool SC = E8>
struct Wave {
  static_assert(SH == 16 || !E8, "tiles of 32 rows hold 16-bit values");
  typedef Ty<DT> Y;
  typedef typename Y::v8 v8;
  typedef typename std::conditional<SH == 16, f32x4, f32x16>::type acc_t;
  static constexpr int RB = D * (E8 ? 1 : 2), SIDE = SH;
  static constexpr int NG = 64 / SH;        // lane groups that share the rows
  static constexpr int KS = 8 * NG;         // depth of one product instruction
  static constexpr int STEPS = D / KS;      // of S^T
  static constexpr int DT_N = D / SH;       // output tiles
  static constexpr int REGS = SH * SH / 64; // accumulator registers of a tile

  // log2 of the largest weight when m is set, and how far weights may grow past it before m is set again.  fp16:
  // weights down to 2^-32 of the largest are kept.
  static constexpr float LIFT = DT == BF16 ? 0.0f : 8.0f, SLACK = 6.0f;
  // fp16 operands that are weight * scale of the value: the same holds for these products, the largest of which m follows.
  // (A bound made of the largest weight and the largest scale would not do: beside a token of no weight whose scale is
  // 2^30 times as large, products that count fell out of fp16's range.)  Weights reach 2^REACH; scales that have nothing
  // to give even so, below 2^-45, have nothing to give to an fp16 output either.  bf16 has fp32's range.
  static constexpr bool RANGED = SC && DT == F16;
  static constexpr float REACH = 32.0f;

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

  // Scores (weights) of the tokens that a row does not see: `instead`.  left: tokens up to the row's limit, from the lane
  // group's first.
  template <int TOK>
  static __device__ __forceinline__ void hide(acc_t (&s)[TOK / SH], int left, float instead) {
    __builtin_amdgcn_sched_barrier(0);  // comparisons hoisted over the products would take all scalar registers
#pragma unroll
    for (int t = 0; t < TOK / SH; ++t) {
#pragma unroll
      for (int r = 0; r < REGS; ++r) s[t][r] = t * SH + token_of(r, 0) < left ? s[t][r] : instead;
      __builtin_amdgcn_sched_barrier(0);
    }
  }

  // Scores -> weights exp2(score - m), the operands of the second product.  m follows the running maximum in steps:
  // while no row of the wavefront passes its m by 2^SLACK beyond the lift, sums and outputs stay as they are.
  template <int TOK>
  __device__ __forceinline__ void weights(acc_t (&s)[TOK / SH], int t0, int limit, bool full, float scale,
                                          uint32_t sbase, int tok0, v8 (&p)[TOK / KS]) {
    const int g = (threadIdx.x & 63) / SH;
    if (SC) {
#pragma unroll
      for (int t = 0; t < TOK / SH; ++t)
#pragma unroll
        for (int r = 0; r < REGS; r += 4) {
          const f32x4 k = lds_read<f32x4>(scale_at(sbase, tok0 + t * SH + token_of(r, g)));
#pragma unroll
          for (int i = 0; i < 4; ++i) s[t][r + i] *= k[i];
        }
    }
    if (!full) hide<TOK>(s, limit - t0 - 4 * g, NEG_INF);
    float top = NEG_INF;
#pragma unroll
    for (int t = 0; t < TOK / SH; ++t)
#pragma unroll
      for (int r = 0; r < REGS; ++r) top = fmaxf(top, s[t][r]);
    top = over_groups_max(top) * scale;
    constexpr float lift = RANGED ? REACH : LIFT, slack = RANGED ? 0.0f : SLACK;
    if (__any(top > m + (lift + slack))) {
      const float ref = fmaxf(m, top - lift);
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
        if (SC) v = lds_read<f32x4>(scale_at(sbase, tok0 + t * SH + token_of(r, g)) + 128);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][r + i], scale, -use));
          sum += w;
          s[t][r + i] = SC ? w * v[i] : w;
        }
      }
    if (SC && !full) hide<TOK>(s, limit - t0 - 4 * g, 0.0f);  // whatever their scales are
    if (RANGED) {
      float most = 0.0f;
#pragma unroll
      for (int t = 0; t < TOK / SH; ++t)
#pragma unroll
        for (int r = 0; r < REGS; ++r) most = fmaxf(most, fabsf(s[t][r]));
      most = over_groups_max(most);
      constexpr float room = 1 << (int)(LIFT + SLACK);
      if (__any(most > room)) {
        const float ref = most > room ? m + (__builtin_amdgcn_logf(fminf(most, 0x1p100f)) - LIFT) : m;
        const float alpha = __builtin_amdgcn_exp2f(m - (ref == NEG_INF ? 0.0f : ref));
        m = ref;
        l *= alpha;
        sum *= alpha;
#pragma unroll
        for (int t = 0; t < TOK / SH; ++t)
#pragma unroll
          for (int r = 0; r < REGS; ++r) s[t][r] *= alpha;
#pragma unroll
        for (int d = 0; d < DT_N; ++d)
#pragma unroll
          for (int r = 0; r < REGS; ++r) o[d][r] *= alpha;
      }
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
      const int sub = SH == 32 ? (lane >> 4) & 1 : 0;    // 16 of a 16-bit tile's 32 channels
      if (E8) {
        const int r = i >> 1, tok = gx * 4 + (r & 3) + (r >> 2) * (KS / 2);
        at = vbase + tok * RB + (i & 1) * 8;
        x = (uint32_t)swizzle_v<RB, SH, E8>(tok) << 4;
      } else {
        const int r = i >> 2, b = i & 3, tok = gx * 4 + r;
        at = vbase + tok * RB + (b & 1) * 8;
        x = (uint32_t)((sub * 2 + (b >> 1)) ^ swizzle_v<RB, SH, E8>(tok)) << 4;
      }
    }
    __device__ __forceinline__ v8 read(int d, int k) const {
      if (E8) {
        const uint32_t p = at + (x ^ (uint32_t)(d * 16)) + k * KS * RB;
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
  // Tokens tok0 .. tok0 + ROWS - 1 of the tile at vbase, t0 being the tile's first token; limit_of(r): the limit of row
  // r; the word `any` is set if there are any.
  template <int ROWS, typename Limit>
  static __device__ __forceinline__ void set_apart(uint32_t vbase, int tok0, int t0, int rows, uint32_t marks,
                                                   uint32_t any, Limit limit_of) {
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
    *(__attribute__((address_space(3))) int*)(uintptr_t)any = 1;
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
__device__ __forceinline__ int prefix_length(const Args& a, int g) {
  return a.prefix_lens ? clamp_int(a.prefix_lens[g], 0, a.Wp << a.page_shift) : 0;
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
  r.len = prefix_length(a, g);
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

// The sequences of a group: up to 64 of them are held one a lane (one round of loads, then shuffles), more are looked
// up in memory.
struct SeqTable {
  int b0, n, start = 0x7FFFFFFF, next = 0x7FFFFFFF, own = 0;
  __device__ __forceinline__ void load(const Args& a, int first, int last) {
    const int lane = threadIdx.x & 63;
    b0 = first;
    n = last - first;
    if (n <= 64 && lane < n) {
      start = query_start(a, b0 + lane);
      next = query_start(a, b0 + lane + 1);
      own = clamp_int(a.lens[b0 + lane], 0, a.W << a.page_shift);
    }
  }
  // number (from b0) of the sequence of query t; every lane takes part
  __device__ __forceinline__ int find(const Args& a, int t) const {
    if (n > 64) return sequence_of(a, t, b0, b0 + n) - b0;
    int at = 0;
#pragma unroll
    for (int step = 32; step > 0; step >>= 1) {
      const int c = __shfl(start, at + step);
      if (at + step < n && c <= t) at += step;
    }
    return at;
  }
  __device__ __forceinline__ Seq get(const Args& a, int i) const {
    if (n > 64) return sequence(a, b0 + i);
    Seq s;
    s.q0 = __shfl(start, i);
    s.n_q = max(__shfl(next, i) - s.q0, 0);
    s.own = __shfl(own, i);
    return s;
  }
};

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

// ------------------------------------------------------------------ results of a block
//
// Layout in LDS at the end: the outputs of PARTS wavefronts for each of ROWS rows (fp32, 16-byte chunks swizzled by the
// row), their references and sums, the marks.  Threads then take runs of four channels: whole rows are stored at once,
// by a short loop (unrolled over a wavefront's registers it took 4 us, most of it fetching instructions).
template <int D>
__device__ __forceinline__ uint32_t out_at(uint32_t base, int part_row, int chunk) {
  return base + part_row * D * 4 + ((chunk ^ (part_row & 15)) << 4);
}
template <typename W, int D>
__device__ __forceinline__ void stash(const W& w, uint32_t outs, uint32_t stats, int part_row) {
  const float l = W::over_groups_sum(w.l);
  const int g = (threadIdx.x & 63) / W::SIDE;
#pragma unroll
  for (int d = 0; d < W::DT_N; ++d)
#pragma unroll
    for (int r = 0; r < W::REGS; r += 4) {
      f32x4 x;
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = w.o[d][r + i];
      *(__attribute__((address_space(3))) f32x4*)(uintptr_t)out_at<D>(outs, part_row, (d * W::SIDE + W::token_of(r, g)) / 4) = x;
    }
  if (g == 0) *(__attribute__((address_space(3))) f32x2*)(uintptr_t)(stats + part_row * 8) = f32x2{w.m, l};
}
// Rows that sequence b's of key/value head h follow among own_rows, where these are FEW for each.
__device__ __forceinline__ int64_t own_rows_before(const Args& a, int b, int h) { return ((int64_t)b * a.Hkv + h) * FEW; }
// The first slot of own row `n`: S2 for its streams and, compact, one for a tile that was not split.
__device__ __forceinline__ int64_t own_slot(const Args& a, int64_t n) { return a.own_first + n * a.own_stride; }

// rows: how many; q0: query of row `first`.  own_row: the rows' places among own_rows, any + 4: the splits of the split
// units before this one (both compact).  big(r): its result is complete if the unit was not split.
template <typename W, int D, int ROWS, int PARTS, bool TILES, typename Big>
__device__ __forceinline__ void finish(uint32_t args, uint32_t outs, uint32_t stats, uint32_t marks, uint32_t any,
                                       int rows, int q0, int first, int h, int split, int splits, uint32_t own_row,
                                       Big big) {
  const Args a = saved_args(args);
  const bool marked = lds_read<int>(any) != 0;
  const int slots = a.S1 + a.S2, before = TILES ? lds_read<int>(any + 4) : 0;
  typedef typename W::Y::el el;
#pragma unroll 4
  for (int i = threadIdx.x; i < rows * (D / 4); i += THREADS) {
    const int r = i / (D / 4), c = i % (D / 4);
    f32x4 x = lds_read<f32x4>(out_at<D>(outs, r, c));
    f32x2 ml = lds_read<f32x2>(stats + r * 8);  // reference, sum
    if (PARTS > 1) {
      float m = ml[0], sum = 0.0f;
#pragma unroll
      for (int k = 1; k < PARTS; ++k) m = fmaxf(m, lds_read<f32x2>(stats + (k * ROWS + r) * 8)[0]);
      const float use = m == NEG_INF ? 0.0f : m;
      f32x4 y{};
#pragma unroll
      for (int k = 0; k < PARTS; ++k) {
        const f32x2 e = lds_read<f32x2>(stats + (k * ROWS + r) * 8);
        const float f = __builtin_amdgcn_exp2f(e[0] - use);
        sum += e[1] * f;
        y += lds_read<f32x4>(out_at<D>(outs, k * ROWS + r, c)) * f;
      }
      x = y;
      ml = f32x2{m, sum};
    }
    if (marked) x = W::marked(x, marks, r, c * 4);
    const int qi = a.by_grp.divide(first + r);
    const int64_t id = (int64_t)(q0 + qi) * a.Hq + h * a.grp + a.by_grp.rest(first + r, qi);
    const bool own_here = !TILES || big(r), final = own_here && splits == 1;
    int64_t slot = id * slots + split;
    if (TILES && a.compact)
      slot = splits > 1 ? before * ROWS + r * splits + split
                        : own_slot(a, a.direct_rows ? id : lds_read<int>(own_row + 4 * r)) + a.S2;
    if (final)
      store4((el*)a.out + id * D + c * 4, x * inverse(ml[1]));
    else if (!(ml[1] == 0.0f))
      *(f32x4*)(a.part_o + slot * D + c * 4) = x;
    if (c == 0) {
      if (final) a.lse[id] = natural_lse(ml[0], ml[1]);
      if (TILES && !final) a.part_ml[slot] = float2{ml[0], ml[1]};
      if (TILES && split == 0) {
        a.n_tile[id] = final ? -1 : splits;
        if (a.compact) a.tile_at[id] = splits > 1 ? before * ROWS + r * splits : -1;
        if (own_here) a.n_own[id] = 0;
      }
    }
  }
}

// ------------------------------------------------------------------ few rows

template <int DT, bool E8, int D>
struct FewLayout {
  static constexpr int RB = D * (E8 ? 1 : 2);
  static constexpr int TOK = RB == 256 ? 32 : 64;  // tokens of a wavefront's step
  static constexpr int TILE_BYTES = TOK * RB;
  static constexpr int WAVE_BYTES = 2 * TILE_BYTES + (E8 ? 2 * TOK * 4 : 0);
  static constexpr int OUT_BYTES = WAVES * FEW * D * 4;
  static constexpr int MARKS = WAVES * WAVE_BYTES > OUT_BYTES ? WAVES * WAVE_BYTES : OUT_BYTES;
  static constexpr int LIMITS = MARKS + FEW * 64, STATS = LIMITS + 2 * FEW * 4, ANY = STATS + WAVES * FEW * 8;
  static constexpr int ARGS = ANY + 16, LDS = ARGS + sizeof(Args);
};

// What a block of few rows does: rows 0 .. rows - 1 (at most 16) from query q0 on, over prefix tokens and then own tokens
// (either may be none).
struct FewTask {
  int h, q0, rows;
  Tokens prefix, own;
  int n_q, seen;  // queries of the sequence, its own tokens
};

template <int DT, bool E8, int D>
__device__ __forceinline__ void attend_few(const Args& a, char* smem, const FewTask& f, uint32_t arg_word) {
  constexpr int SH = 16;
  typedef FewLayout<DT, E8, D> L;
  typedef Wave<DT, E8, D, SH> W;
  typedef typename W::Y::el el;
  constexpr int TOK = L::TOK, RB = L::RB, NI = TOK * RB / 1024, ESIZE = E8 ? 1 : 2;
  typedef Copier<RB, NI> Copy;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int row = lane % SH, h = f.h;
  const bool valid = row < f.rows;
  const int qi = a.by_grp.divide(row), hq = h * a.grp + a.by_grp.rest(row, qi), t = f.q0 + qi;

  W w;
  w.init((const el*)a.q + t * a.q_st + hq * a.q_sh, valid, a.flip, a.keep);

  const int pre = (f.prefix.len + TOK - 1) / TOK, tiles = pre + (f.own.len + TOK - 1) / TOK;
  const int n0 = tiles * wave / WAVES, n1 = tiles * (wave + 1) / WAVES;

  const uint32_t kbase = lds_addr(smem) + wave * L::WAVE_BYTES, vbase = kbase + L::TILE_BYTES;
  const uint32_t sbase = vbase + L::TILE_BYTES, marks = lds_addr(smem) + L::MARKS, limits = lds_addr(smem) + L::LIMITS;
  const char* kp = a.kc + h * a.c_head * ESIZE;
  const char* vp = a.vc + h * a.c_head * ESIZE;
  // step n: of the prefix while n < pre, then of the own tokens
  auto source = [&](int n) __attribute__((always_inline)) { return n < pre ? f.prefix : f.own; };
  auto first_token = [&](int n) __attribute__((always_inline)) { return (n < pre ? n : n - pre) * TOK; };
  Window win;
  auto cover = [&](int n) __attribute__((always_inline)) {
    if (n == pre) win.reset();
    const Tokens src = source(n);
    const int t0 = first_token(n);
    win.cover(src, t0 >> a.page_shift, min(t0 + TOK - 1, src.len - 1) >> a.page_shift, a.n_pages);
  };
  auto fill_keys = [&](int n) __attribute__((always_inline)) {
    Copy::run(a, win, source(n), kp, kbase, first_token(n), ESIZE, [](int r) { return swizzle_k<RB>(r); });
  };
  auto fill_values = [&](int n) __attribute__((always_inline)) {
    Copy::run(a, win, source(n), vp, vbase, first_token(n), ESIZE, [](int r) { return swizzle_v<RB, SH, E8>(r); });
  };
  auto fill_scales = [&](int n) __attribute__((always_inline)) {  // 32 tokens a copy: keys' scales, then values'
    const Tokens src = source(n);
#pragma unroll
    for (int i = 0; i < TOK / 32; ++i) {
      const int tok = min(first_token(n) + i * 32 + (lane & 31), src.len - 1);
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

  // Tokens that the row attends to (its position is that of the last n_q tokens of its sequence), worked out while
  // the first ones are on their way.
  int prefix_limit = 0x7FFFFFFF, own_limit = 0x7FFFFFFF;
  if (valid) {
    const int end = f.seen - f.n_q + qi + 1;  // own tokens up to and with the query
    prefix_limit = clamp_int(f.prefix.len + end, 0, f.prefix.len);
    own_limit = clamp_int(end, 0, f.own.len);
  }
  for (int i = threadIdx.x; i < FEW * 16; i += THREADS) *(uint32_t*)(smem + L::MARKS + 4 * i) = 0;
  if (threadIdx.x < ARG_WORDS) *(uint32_t*)(smem + L::ARGS + 4 * threadIdx.x) = arg_word;
  if (wave == 0 && lane < SH) {
    ((int*)(smem + L::LIMITS))[lane] = prefix_limit;
    ((int*)(smem + L::LIMITS))[FEW + lane] = own_limit;
    if (lane == 0) *(int*)(smem + L::ANY) = 0;
  }
  block_barrier();

  for (int n = n0; n < n1; ++n) {
    const int t0 = first_token(n), limit = n < pre ? prefix_limit : own_limit;
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
      const uint32_t at = limits + (n < pre ? 0 : 4 * FEW);
      W::template set_apart<TOK>(vbase, 0, t0, f.rows, marks, lds_addr(smem) + L::ANY, [&](int r) { return lds_read<int>(at + 4 * r); });
      wait_lds();
    }
    w.template values<TOK>(vbase, p);
    wait_lds();
    if (n + 1 < n1) fill_values(n + 1);
  }

  block_barrier();  // every wavefront is done with its tiles
  const uint32_t outs = lds_addr(smem), stats = outs + L::STATS;
  stash<W, D>(w, outs, stats, wave * FEW + row);
  block_barrier();
  finish<W, D, FEW, WAVES, false>(outs + L::ARGS, outs, stats, marks, outs + L::ANY, f.rows, f.q0, 0, h, 0, 1, 0,
                                  [](int) { return true; });
}

// Outputs of queries t0 .. t1 - 1 that attend to nothing, every step-th one.
template <int DT, int D>
__device__ __forceinline__ void empty_rows(const Args& a, int h, int t0, int t1, int step) {
  for (int64_t t = t0; t < t1; t += step) {
    const int64_t id = t * a.Hq + h * a.grp;
    for (int i = threadIdx.x; i < a.grp * D; i += THREADS) ((typename Ty<DT>::el*)a.out)[id * D + i] = 0;
    for (int i = threadIdx.x; i < a.grp; i += THREADS) a.lse[id + i] = NEG_INF;
  }
}

// A block for each sequence and key/value head (with the sequence's prefix where the call is `joint`); results are final.
template <int DT, bool E8, int D>
__global__ void __launch_bounds__(THREADS, 2) attend_each(Args a) {
  extern __shared__ __align__(16) char smem[];
  const uint32_t arg_word = argument_word();
  const int b = a.by_heads.divide((int)blockIdx.x);
  FewTask f;
  f.h = a.by_heads.rest((int)blockIdx.x, b);
  // rows of no sequence, dealt out to the blocks
  const int first = query_start(a, 0), end = max(query_start(a, a.B), first);
  if (b < first) empty_rows<DT, D>(a, f.h, b, first, a.B);
  if (b < a.T - end) empty_rows<DT, D>(a, f.h, end + b, a.T, a.B);
  const Seq s = sequence(a, b);
  f.q0 = s.q0;
  f.n_q = s.n_q;
  f.rows = s.n_q * a.grp;
  f.seen = s.own;
  f.own = Tokens{a.pages + (int64_t)b * a.W, a.W, s.own};
  f.prefix = Tokens{nullptr, 0, 0};
  if (a.joint) {
    int lo = 0, hi = a.G;  // the last group that starts at or before the sequence
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (a.group_offsets[mid] <= b) lo = mid; else hi = mid;
    }
    f.prefix = Tokens{a.prefix_pages + (int64_t)lo * a.Wp, a.Wp, prefix_length(a, lo)};
  }
  if (f.rows > FEW)  // more queries than max_q announced: nothing was planned for them
    empty_rows<DT, D>(a, f.h, f.q0, f.q0 + s.n_q, 1);
  else if (f.rows > 0)
    attend_few<DT, E8, D>(a, smem, f, arg_word);
}

// ------------------------------------------------------------------ own tokens in streams
//
// Units are the sequences of up to 16 rows, once for each key/value head; their steps of TOK tokens, laid end to end,
// are shared out evenly to all wavefronts.  A wavefront runs through its share without a pause where one unit ends and
// the next begins: the next unit's first keys are fetched while the last values of the one before are used.  Unit by
// unit its results go to a slot, the n-th of those wavefronts that the unit's steps fall to.  (A block for each unit,
// its wavefronts joined at the end, left the memory idle for half of its 11 us at 400 tokens.)
template <int DT, bool E8, int D>
struct StreamLayout {
  static constexpr int RB = D * (E8 ? 1 : 2);
  static constexpr int TOK = RB == 256 ? 32 : 64;  // tokens of a step
  static constexpr int TILE_BYTES = TOK * RB;
  static constexpr int WAVE_BYTES = 2 * TILE_BYTES + (E8 ? 2 * TOK * 4 : 0);
  static constexpr int MARKS = WAVES * WAVE_BYTES, MARK_BYTES = FEW * 64 + FEW * 4 + 16;  // marks, limits, any
  static constexpr int ARGS = MARKS + WAVES * MARK_BYTES, LDS = ARGS + sizeof(Args);
};

template <int DT, bool E8, int D>
__device__ __forceinline__ void stream_rows(const Args& a, char* smem, int index, uint32_t arg_word) {
  constexpr int SH = 16;
  typedef StreamLayout<DT, E8, D> L;
  typedef Wave<DT, E8, D, SH> W;
  typedef typename W::Y::el el;
  constexpr int TOK = L::TOK, RB = L::RB, NI = TOK * RB / 1024, ESIZE = E8 ? 1 : 2;
  typedef Copier<RB, NI> Copy;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int row = lane % SH, qi = a.by_grp.divide(row), head = a.by_grp.rest(row, qi);

  if (threadIdx.x < ARG_WORDS) *(uint32_t*)(smem + L::ARGS + 4 * threadIdx.x) = arg_word;
  block_barrier();  // the only one: the wavefronts go their own ways from here

  // Steps of sequence x0 + lane, 64 sequences at a time.  Sequences of more than 16 rows have none (their tiles take
  // their tokens; without tiles an empty one, which marks them empty); without own tokens one, an empty one.
  Seq s;
  int steps = 0;
  auto count = [&](int x) __attribute__((always_inline)) {
    steps = 0;
    s = Seq{0, 0, 0};
    if (x >= a.B) return;
    s = sequence(a, x);
    const int rows = s.n_q * a.grp;
    if (rows > FEW) s.own = 0;
    steps = rows == 0 || (rows > FEW && a.big) ? 0 : max((s.own + TOK - 1) / TOK, 1);
  };
  int total = 0;
  for (int x0 = (a.B - 1) / 64 * 64; x0 >= 0; x0 -= 64) {  // downwards: ends with the first sequences in registers
    count(x0 + lane);
    total += steps;
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) total += __shfl_xor(total, d);
  total = __builtin_amdgcn_readfirstlane(total) * a.Hkv;
  const int per = max((total + a.streams - 1) / a.streams, a.stream_least);
  const int mine = index * WAVES + wave;
  int left = min(per, total - mine * per);  // steps to do (mine * per < streams * per < 2^31: see the plan)
  if (left <= 0) return;

  // the unit that the first step belongs to: sequence x0 + at, head h, step n; `start` is its first step of all
  int x0 = 0, at = 0, h = 0, n = 0, start = 0;
  {
    const int want = mine * per;
    int seen = 0;
    for (;; x0 += 64) {
      if (x0 >= a.B) return;  // not with lengths that stay as they are during the call
      if (a.B > 64) count(x0 + lane);
      int incl = steps * a.Hkv;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(incl, d);
        if (lane >= d) incl += o;
      }
      const int here = __builtin_amdgcn_readlane(incl, 63);
      if (want < seen + here) {
        at = __builtin_ctzll(__ballot(seen + incl > want));
        const int each = __builtin_amdgcn_readlane(steps, at);
        start = seen + __builtin_amdgcn_readlane(incl, at) - each * a.Hkv;
        h = (int)((uint32_t)(want - start) / (uint32_t)each);
        start += h * each;
        n = want - start;
        break;
      }
      seen += here;
    }
  }

  struct UnitOf {
    int q0, n_q, own, h, slot, last;  // last: its steps
    Tokens src;
  };
  auto unit_here = [&](const Args& a) __attribute__((always_inline)) {
    UnitOf u;
    u.q0 = __builtin_amdgcn_readlane(s.q0, at);
    u.n_q = __builtin_amdgcn_readlane(s.n_q, at);
    u.own = __builtin_amdgcn_readlane(s.own, at);
    u.last = __builtin_amdgcn_readlane(steps, at);
    u.h = h;
    u.slot = mine - (int)((uint32_t)start / (uint32_t)per);
    u.src = Tokens{uniform(a.pages + (int64_t)(x0 + at) * a.W), __builtin_amdgcn_readfirstlane(a.W), u.own};
    return u;
  };
  // on to the next unit (there is one: steps are left)
  auto next_unit = [&]() __attribute__((always_inline)) {
    start += __builtin_amdgcn_readlane(steps, at);
    n = 0;
    if (++h < a.Hkv) return;
    h = 0;
    for (;;) {
      if (++at == 64) {
        at = 0;
        x0 += 64;
        count(x0 + lane);
        if (x0 >= a.B) {  // not with lengths that stay as they are during the call
          left = 0;
          return;
        }
      }
      const unsigned long long some = __ballot(steps > 0) >> at;
      if (some) {
        at += __builtin_ctzll(some);
        return;
      }
      at = 63;
    }
  };

  const uint32_t kbase = lds_addr(smem) + wave * L::WAVE_BYTES, vbase = kbase + L::TILE_BYTES;
  const uint32_t sbase = vbase + L::TILE_BYTES;
  const uint32_t marks = lds_addr(smem) + L::MARKS + wave * L::MARK_BYTES, limits = marks + FEW * 64, any = limits + FEW * 4;
  auto clear_marks = [&]() __attribute__((always_inline)) {
    *(__attribute__((address_space(3))) u32x4*)(uintptr_t)(marks + lane * 16) = u32x4{};
    if (lane == 0) *(__attribute__((address_space(3))) int*)(uintptr_t)any = 0;
  };
  static_assert(FEW * 64 == 64 * 16, "16 bytes a lane");
  clear_marks();

  Window win;
  auto cover = [&](const Tokens& src, int n) __attribute__((always_inline)) {
    win.cover(src, n * TOK >> a.page_shift, min(n * TOK + TOK - 1, src.len - 1) >> a.page_shift, a.n_pages);
  };
  auto fill_scales = [&](const UnitOf& u, int n) __attribute__((always_inline)) {  // 32 tokens a copy
#pragma unroll
    for (int i = 0; i < TOK / 32; ++i) {
      const int tok = min(n * TOK + i * 32 + (lane & 31), u.src.len - 1);
      const int page = __builtin_amdgcn_ds_bpermute(((tok >> a.page_shift) - win.first) << 2, win.ids);
      const int64_t off = page * a.s_page + u.h * a.s_head + (tok & ((1 << a.page_shift) - 1)) * a.s_slot;
      dma4(sbase + i * 256, (const char*)((lane < 32 ? a.ks : a.vs) + off));
    }
  };
  auto fill_keys = [&](const UnitOf& u, int n) __attribute__((always_inline)) {
    if (u.src.len == 0) return;
    cover(u.src, n);
    if (E8) fill_scales(u, n);
    Copy::run(a, win, u.src, a.kc + u.h * a.c_head * ESIZE, kbase, n * TOK, ESIZE, [](int r) { return swizzle_k<RB>(r); });
  };
  auto fill_values = [&](const UnitOf& u, int n) __attribute__((always_inline)) {
    if (u.src.len == 0) return;
    Copy::run(a, win, u.src, a.vc + u.h * a.c_head * ESIZE, vbase, n * TOK, ESIZE,
              [](int r) { return swizzle_v<RB, SH, E8>(r); });
  };
  auto queries = [&](W& w, const UnitOf& u) __attribute__((always_inline)) {
    const bool valid = row < u.n_q * a.grp;
    w.init((const el*)a.q + (u.q0 + qi) * a.q_st + (u.h * a.grp + head) * a.q_sh, valid, a.flip, a.keep);
  };

  // the unit's sequence, which only its results need
  auto note = [&]() __attribute__((always_inline)) {
    if (lane == 0) *(__attribute__((address_space(3))) int*)(uintptr_t)(any + 4) = x0 + at;
  };
  note();
  UnitOf u = unit_here(a);
  W w;
  queries(w, u);
  fill_keys(u, n);
  fill_values(u, n);
  int limit = 0;
  auto set_limits = [&]() __attribute__((always_inline)) {
    const bool valid = row < u.n_q * a.grp;
    limit = valid ? clamp_int(u.own - u.n_q + qi + 1, 0, u.own) : 0x7FFFFFFF;
    if (lane < SH) *(__attribute__((address_space(3))) int*)(uintptr_t)(limits + 4 * lane) = limit;
  };
  set_limits();

  for (;;) {
    const int t0 = n * TOK;
    const bool ends = n + 1 == u.last, more = left > 1;
    UnitOf v = u;   // the next step's unit
    W next;         // its queries
    int n_next = n + 1;
    typename W::acc_t s2[TOK / SH];
    typename W::v8 p[TOK / W::KS];
    const bool full = __all(limit >= t0 + TOK), nothing = u.src.len == 0;
    if (!nothing) {
      wait_vm<NI>();  // keys (and scales) are there; the values may be on their way
      w.template scores<TOK>(kbase, s2);
      if (E8) w.template weights<TOK>(s2, t0, limit, full, a.scale_log2, sbase, 0, p);
      wait_lds();
    }
    if (more) {
      if (ends) {
        next_unit();
        n_next = 0;
        v = unit_here(saved_args(lds_addr(smem) + L::ARGS));
        queries(next, v);
        win.reset();
      }
      fill_keys(v, n_next);
    }
    if (!nothing) {
      if (!E8) w.template weights<TOK>(s2, t0, limit, full, a.scale_log2, sbase, 0, p);
      if (more && v.src.len > 0) wait_vm<NI + (E8 ? TOK / 32 : 0)>(); else wait_vm<0>();
      if (!full) {
        W::template set_apart<TOK>(vbase, 0, t0, min(u.n_q * a.grp, FEW), marks, any,
                                   [&](int r) { return lds_read<int>(limits + 4 * r); });
        wait_lds();
      }
      w.template values<TOK>(vbase, p);
      wait_lds();
    }
    if (ends || !more) {
      // this unit's results
      const Args b = saved_args(lds_addr(smem) + L::ARGS);
      const float l = W::over_groups_sum(w.l);
      const bool marked = lds_read<int>(any) != 0;
      const int g = lane / SH, rows = u.n_q * b.grp;
      if (row < rows && rows <= FEW) {
        const int64_t id = (int64_t)(u.q0 + qi) * b.Hq + u.h * b.grp + head;
        const int64_t own_row = b.direct_rows ? id : own_rows_before(b, lds_read<int>(any + 4), u.h) + row;
        const int64_t slot = own_slot(b, own_row) + u.slot;
        if (!(l == 0.0f)) {
#pragma unroll
          for (int d = 0; d < W::DT_N; ++d) {
            f32x4 x = w.o[d];
            const int c = d * SH + W::token_of(0, g);
            if (marked) x = W::marked(x, marks, row, c);
            *(f32x4*)(b.part_o + slot * D + c) = x;
          }
        }
        if (g == 0) {
          b.part_ml[slot] = float2{w.m, l};
          if (ends) b.n_own[id] = u.slot + 1;
          if (ends && b.compact) b.own_at[id] = (int)own_row;
        }
      }
      if (rows > FEW)  // more queries than max_q announced: nothing was planned for them
        for (int r = lane; r < rows; r += 64) {
          const int q = b.by_grp.divide(r);
          b.n_own[(int64_t)(u.q0 + q) * b.Hq + u.h * b.grp + b.by_grp.rest(r, q)] = 0;
        }
      if (!more) return;
      if (marked) clear_marks();
      u = v;
      note();
      w = next;
      set_limits();
    }
    n = n_next;
    --left;
    fill_values(v, n);
  }
}

// ------------------------------------------------------------------ tiles of rows
//
// RW wavefronts side by side hold the tile's 32 * RW rows, 4 / RW wavefronts share the tokens of a step.
template <int DT, bool E8, int D, int RW>
struct TileLayout {
  static constexpr int RB = D * 2;  // the tiles hold 16-bit values; e4m3 codes are converted on the way
  static constexpr int ROWS = 32 * RW;
  static constexpr int TOK = RB == 256 ? 64 : 128;  // tokens of a step
  static constexpr int TILE_BYTES = TOK * RB;
  static constexpr int STAGE = 2 * TILE_BYTES + (E8 ? 2 * TOK * 4 : 0);
  static constexpr int MARKS = 2 * STAGE;
  static constexpr int ROW_INFO = MARKS + ROWS * 64, STATS = ROW_INFO + ROWS * 16, ANY = STATS + WAVES * 32 * 8;
  static constexpr int ARGS = ANY + 16, LDS = ARGS + sizeof(Args);
  static_assert(MARKS >= WAVES * 32 * D * 4, "the outputs reuse the stages");
};

// Which entry (group) block `index` works for, which of its units and which split of that.  Entries have
// `units` units of `steps` steps (set by count(entry), an entry a lane, 64 at a time); a unit is cut into splits of
// about the same number of steps, `fill` blocks in all at most (units beside: an entry's last split may be short), of
// `least` steps at least and `most` splits at most.
// before: if asked for (`number`), the splits of the units before this one that are split too.
struct Unit {
  int entry, lane, at, split, splits, before;
};
template <typename Count>
__device__ __forceinline__ bool share_out(int entries, int index, int fill, int least, int most, bool number,
                                          Unit& u, int& total, Count count) {
  const int lane = threadIdx.x & 63;
  int units = 0, steps = 0;
  total = 0;
  float all = 0.0f;
  for (int x0 = (entries - 1) / 64 * 64; x0 >= 0; x0 -= 64) {  // downwards: ends with the first entries in registers
    count(x0 + lane, units, steps);
    total += units;
    all += (float)units * (float)steps;
  }
  if (entries > 1) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      total += __shfl_xor(total, d);
      all += __shfl_xor(all, d);
    }
  }
  total = __builtin_amdgcn_readfirstlane(total);
  if (index >= total + fill) return false;
  // steps of a split: sum of units * ceil(steps / share) <= sum of units * (steps / share + 1) <= fill
  const int room = max(fill - total, fill / 4);
  const float share = fmaxf(as_float(__builtin_amdgcn_readfirstlane(as_uint(all))) / (float)room, (float)least);
  int seen = 0, split_before = 0;
  for (int x0 = 0; x0 < entries; x0 += 64) {
    if (entries > 64) count(x0 + lane, units, steps);
    int cuts = (int)ceilf((float)steps / share);
    if (entries == 1) cuts = min(fill / max(units, 1), (steps + least - 1) / least);
    cuts = clamp_int(cuts, 1, most);
    int incl = units * cuts;
    const int n = incl;
    if (entries > 1) {
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(incl, d);
        if (lane >= d) incl += o;
      }
    }
    const int here = __builtin_amdgcn_readlane(incl, entries > 1 ? 63 : 0);
    int split_incl = cuts > 1 ? n : 0;
    const int split_n = split_incl;
    if (number && entries > 1) {
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(split_incl, d);
        if (lane >= d) split_incl += o;
      }
    }
    if (index < seen + here) {
      u.lane = entries > 1 ? __builtin_ctzll(__ballot(seen + incl > index)) : 0;
      const int at = index - seen - __builtin_amdgcn_readlane(incl - n, u.lane);
      const int of = __builtin_amdgcn_readlane(units, u.lane);
      u.entry = x0 + u.lane;
      u.splits = __builtin_amdgcn_readlane(cuts, u.lane);
      u.split = (int)((uint32_t)at / (uint32_t)of);
      u.at = at - u.split * of;
      u.before = split_before + __builtin_amdgcn_readlane(split_incl - split_n, u.lane) + u.at * u.splits;
      // Groups that overlap can hold more units than 32 bits count.
      return (uint32_t)u.split < (uint32_t)u.splits && (!number || (uint32_t)u.before <= (uint32_t)(2 * FILL - u.splits));
    }
    seen += here;
    split_before += __builtin_amdgcn_readlane(split_incl, 63);
  }
  return false;
}

// Unit (group, row tile, key/value head) and split of tile block `index`; false past the last one.
//
// At least FILL units: rounds of FILL whole units, then those of a last, partial round cut into splits that fill the
// device.  Fewer are shared out by their steps.  A head's units lie Hkv apart in block numbers, so with 8 heads they
// run on one XCD, whose L2 then holds the keys and values that they share.
struct TileUnit {
  Group gr;
  int g, tile, h, split, splits, before;
};
template <int ROWS, int TOK>
__device__ __forceinline__ bool find_tile(const Args& a, int index, TileUnit& t) {
  Group gr;
  auto count = [&](int x, int& units, int& steps) __attribute__((always_inline)) {
    units = steps = 0;
    if (x >= a.G) return;
    gr = group(a, x);
    units = (gr.rows + ROWS - 1) / ROWS * a.Hkv;
    steps = (gr.len + (a.big ? a.W << a.page_shift : 0) + TOK - 1) / TOK;  // own tokens: the most there may be
  };
  Unit u;
  int total, split = 0, splits = 0, before = 0;
  if (a.rounds) {
    // units in order, uncut: of the count of units, which of them this block takes
    if (a.G == 1) {
      int steps;
      count(0, total, steps);
    } else {
      total = 0;
      for (int x0 = 0; x0 < a.G; x0 += 64) {
        int units, steps;
        count(x0 + (threadIdx.x & 63), units, steps);
        total += units;
      }
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) total += __shfl_xor(total, d);
    }
    total = __builtin_amdgcn_readfirstlane(total);
    const int whole = total / FILL * FILL, tail = total - whole;
    splits = 1;
    if (index >= whole) {
      if (tail == 0) return false;
      splits = clamp_int(FILL / tail, 1, a.S1);
      index -= whole;
      if (index >= tail * splits) return false;
      split = index / tail;
      index -= split * tail;
      before = index * splits;
      index += whole;
    }
  }
  if (!share_out(a.G, index, a.tile_fill, 256 / TOK, a.rounds ? 1 : a.S1, a.compact && !a.rounds, u, total, count))
    return false;
  t.before = a.rounds ? before : u.before;
  t.split = a.rounds ? split : u.split;
  t.splits = a.rounds ? splits : u.splits;
  t.g = u.entry;
  t.tile = a.by_heads.divide(u.at);
  t.h = a.by_heads.rest(u.at, t.tile);
  t.gr.b0 = __builtin_amdgcn_readlane(gr.b0, u.lane);
  t.gr.b1 = __builtin_amdgcn_readlane(gr.b1, u.lane);
  t.gr.q0 = __builtin_amdgcn_readlane(gr.q0, u.lane);
  t.gr.rows = __builtin_amdgcn_readlane(gr.rows, u.lane);
  t.gr.len = __builtin_amdgcn_readlane(gr.len, u.lane);
  return true;
}

template <int DT, bool E8, int D, int RW>
__device__ __forceinline__ void row_tile(const Args& a, char* smem, int index, uint32_t arg_word) {
  typedef TileLayout<DT, E8, D, RW> L;
  constexpr int SH = 32, TOK = L::TOK, RB = L::RB, ESIZE = E8 ? 1 : 2;
  constexpr int MINE = TOK / WAVES;            // tokens that a wavefront fetches
  constexpr int NI = MINE * D * ESIZE / 1024;  // in copies of 1 KiB
  constexpr int SHARE = TOK * RW / WAVES;      // tokens of a step that a wavefront attends to
  constexpr int BIG = 1 << 30;                 // on a row's sequence number: it has more than 16 rows
  constexpr int MOST = E8 ? 32 : 64;           // in steps of so many (with scales 64 would spill)
  constexpr int STEP = SHARE > MOST ? MOST : SHARE;
  static_assert(NI >= 1, "a wavefront fetches whole copies");
  typedef Copier<RB, NI> Copy;
  typedef Wave<DT, false, D, SH, E8> W;
  typedef typename W::Y::el el;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int wr = wave % RW, wt = wave / RW;
  TileUnit u;
  if (!find_tile<L::ROWS, TOK>(a, index, u)) return;
  const int h = u.h;
  const Group gr = u.gr;
  const int row = u.tile * L::ROWS + wr * SH + lane % SH;
  const bool valid = row < gr.rows;
  const int qi = a.by_grp.divide(row), hq = h * a.grp + a.by_grp.rest(row, qi), t = gr.q0 + qi;

  SeqTable table;
  table.load(a, gr.b0, gr.b1);
  W w;
  w.init((const el*)a.q + t * a.q_st + hq * a.q_sh, valid, a.flip, a.keep);

  // The tile's tokens: the prefix, then the own tokens (as far as a row of the tile sees them) of each of its
  // sequences with more than 16 rows.  Steps are counted over all of them and shared out to the splits.
  int x_first = 0, x_last = -1, t_last = 0;  // sequences, from the group's first
  if (a.big) {
    t_last = gr.q0 + a.by_grp.divide(min((u.tile + 1) * L::ROWS, gr.rows) - 1);
    x_first = __builtin_amdgcn_readfirstlane(table.find(a, gr.q0 + a.by_grp.divide(u.tile * L::ROWS)));
    x_last = __builtin_amdgcn_readfirstlane(table.find(a, t_last));
  }
  auto own_tokens = [&](const Args& a, int x) __attribute__((always_inline)) {
    const Seq s = table.get(a, x);
    const int last = min(t_last, s.q0 + s.n_q - 1);
    return __builtin_amdgcn_readfirstlane(
        s.n_q * a.grp <= FEW ? 0 : clamp_int(s.own - s.n_q + (last - s.q0) + 1, 0, s.own));
  };
  int steps = (gr.len + TOK - 1) / TOK;
  for (int x = x_first; x <= x_last; ++x) steps += (own_tokens(a, x) + TOK - 1) / TOK;
  steps = __builtin_amdgcn_readfirstlane(steps);
  int skip = (int)((int64_t)steps * u.split / u.splits);
  int todo = (int)((int64_t)steps * (u.split + 1) / u.splits) - skip;

  const uint32_t base = lds_addr(smem), marks = base + L::MARKS, info = base + L::ROW_INFO, any = base + L::ANY;
  const char* kp = a.kc + h * a.c_head * ESIZE;
  const char* vp = a.vc + h * a.c_head * ESIZE;

  // the run of steps at hand: steps n0 .. n1 - 1 of the prefix (x < x_first) or of sequence x
  int x = x_first - 2, n0 = 0, n1 = 0;
  Tokens src{nullptr, 0, 0};
  Window win;
  auto next_run = [&](const Args& a) __attribute__((always_inline)) {
    while (todo > 0 && x < x_last) {
      ++x;
      const int len = x < x_first ? gr.len : own_tokens(a, x);
      const int all = (len + TOK - 1) / TOK;
      if (skip >= all) {
        skip -= all;
        continue;
      }
      n0 = skip;
      n1 = min(all, skip + todo);
      skip = 0;
      todo -= n1 - n0;
      src.table = uniform(x < x_first ? a.prefix_pages + (int64_t)u.g * a.Wp : a.pages + (int64_t)(gr.b0 + x) * a.W);
      src.width = __builtin_amdgcn_readfirstlane(x < x_first ? a.Wp : a.W);
      src.len = len;
      win.reset();
      return true;
    }
    return false;
  };
  // e4m3 codes pass through registers: rows lane / LANES + i * (64 / LANES), 16 codes a lane, and one scale a lane (of
  // the keys of the wavefront's tokens, then of their values).  Two sets, for even and odd steps: a step's loads have
  // two steps' time.
  constexpr int LANES = D / 16;
  struct Codes {
    u32x4 x[2][E8 ? NI : 1];
    float scale;
  };
  Codes codes[2];
  auto fetch = [&](int n, Codes& c) __attribute__((always_inline)) {
    const int t0 = n * TOK + wave * MINE;  // the wavefront's first token
    win.cover(src, min(t0, src.len - 1) >> a.page_shift, min(t0 + MINE - 1, src.len - 1) >> a.page_shift, a.n_pages);
    if (!E8) {
      const uint32_t kb = base + (n & 1) * L::STAGE + wave * MINE * RB;
      Copy::run(a, win, src, kp, kb, t0, ESIZE, [](int r) { return swizzle_k<RB>(r); });
      Copy::run(a, win, src, vp, kb + L::TILE_BYTES, t0, ESIZE, [](int r) { return swizzle_v<RB, SH, false>(r); });
      return;
    }
    const int mask = (1 << a.page_shift) - 1;
    auto offset = [&](int r, int64_t page_stride, int64_t slot_stride) __attribute__((always_inline)) {
      const int tok = min(t0 + r, src.len - 1);
      const int page = __builtin_amdgcn_ds_bpermute(((tok >> a.page_shift) - win.first) << 2, win.ids);
      return page * page_stride + (tok & mask) * slot_stride;
    };
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int64_t off = offset(lane / LANES + i * (64 / LANES), a.c_page, a.c_slot) + (lane % LANES) * 16;
      c.x[0][i] = *(const u32x4*)(kp + off);
      c.x[1][i] = *(const u32x4*)(vp + off);
    }
    const int64_t off = offset(lane % MINE, a.s_page, a.s_slot) + h * a.s_head;
    c.scale = ((lane / MINE) & 1 ? a.vs : a.ks)[off];
  };
  auto place = [&](int n, const Codes& c) __attribute__((always_inline)) {
    if (!E8) return;
    const uint32_t stage = base + (n & 1) * L::STAGE;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int r = wave * MINE + lane / LANES + i * (64 / LANES);
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        const uint32_t row = stage + kv * L::TILE_BYTES + r * RB;
        const int swizzle = kv ? swizzle_v<RB, SH, false>(r) : swizzle_k<RB>(r);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          u32x4 x;
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = W::Y::up8(c.x[kv][i][half * 2 + e / 2], e & 1);
          *(__attribute__((address_space(3))) u32x4*)(uintptr_t)(row + ((((lane % LANES) * 2 + half) ^ swizzle) << 4)) = x;
        }
      }
    }
    if (lane < 2 * MINE)
      *(__attribute__((address_space(3))) float*)(uintptr_t)(
          scale_at(stage + 2 * L::TILE_BYTES, wave * MINE + lane % MINE) + (lane / MINE) * 128) = c.scale;
  };
  bool have = next_run(a);
  if (have) {
    fetch(n0, codes[0]);
    if (E8 && n0 + 1 < n1) fetch(n0 + 1, codes[1]);
  }

  // What the rows see, worked out while the first tokens are on their way.
  int mine = -1, prefix_limit = 0, own_limit = 0, own_row = 0;  // sequence from the group's first
  bool big = false;
  {
    const int i = table.find(a, t);
    const Seq s = table.get(a, i);
    if (valid) {
      const int end = s.own - s.n_q + (t - s.q0) + 1;  // own tokens up to and with the query
      mine = i;
      prefix_limit = clamp_int(gr.len + end, 0, gr.len);
      own_limit = clamp_int(end, 0, s.own);
      big = s.n_q * a.grp > FEW;
      if (a.compact && !big) own_row = (int)own_rows_before(a, gr.b0 + i, h) + (t - s.q0) * a.grp + hq - h * a.grp;
    }
  }
  for (int i = threadIdx.x; i < L::ROWS * 16; i += THREADS) *(uint32_t*)(smem + L::MARKS + 4 * i) = 0;
  if (threadIdx.x < ARG_WORDS) *(uint32_t*)(smem + L::ARGS + 4 * threadIdx.x) = arg_word;
  // of every row, for the marks: sequence (-1: no row), prefix tokens and own tokens that it sees; its place among own_rows
  if (wt == 0 && lane < SH) {
    int* p = (int*)(smem + L::ROW_INFO) + wr * SH + lane;
    p[0] = big ? mine | BIG : mine;
    p[L::ROWS] = prefix_limit;
    p[2 * L::ROWS] = own_limit;
    p[3 * L::ROWS] = own_row;
    if (wr == 0 && lane == 0) {
      *(int*)(smem + L::ANY) = 0;
      *(int*)(smem + L::ANY + 4) = u.before;
    }
  }
  if (have) place(n0, codes[0]);
  block_barrier();

  while (have) {
    const bool pre = x < x_first;
    int limit = pre ? prefix_limit : mine == x ? own_limit : 0;
    const bool some = valid && limit > 0;
    if (!valid) limit = 0x7FFFFFFF;
    auto limit_of = [&](int r) {
      const int rb = lds_read<int>(info + 4 * r);  // (a sequence whose own tokens are read here has the BIG bit)
      return rb < 0 ? 0 : pre ? lds_read<int>(info + 4 * (L::ROWS + r))
                              : rb == (x | BIG) ? lds_read<int>(info + 4 * (2 * L::ROWS + r)) : 0;
    };
    int seen_by_all = 0x7FFFFFFF;  // tokens that every row of the tile sees
#pragma unroll
    for (int r = 0; r < L::ROWS; r += 64)
      if (lds_read<int>(info + 4 * (r + lane)) >= 0) seen_by_all = min(seen_by_all, limit_of(r + lane));
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) seen_by_all = min(seen_by_all, __shfl_xor(seen_by_all, d));
    seen_by_all = __builtin_amdgcn_readfirstlane(seen_by_all);
    // one step; `now` held the step's codes, `other` those of the next
    auto step = [&](int n, Codes& now, Codes& other) __attribute__((always_inline)) {
      const uint32_t stage = base + (n & 1) * L::STAGE;
      if (!E8) wait_vm<0>();
      if ((n + 1) * TOK > seen_by_all)  // each wavefront looks at the tokens it has fetched
        W::template set_apart<MINE>(stage + L::TILE_BYTES, wave * MINE, n * TOK, L::ROWS, marks, any, limit_of);
      block_barrier();  // the step's tokens are there, the other stage is free
      if (!E8 && n + 1 < n1) fetch(n + 1, other);
      if (E8 && n + 2 < n1) fetch(n + 2, now);
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
      if (n + 1 < n1) place(n + 1, other);
    };
    for (int n = n0; n < n1; n += E8 ? 2 : 1) {
      step(n, codes[0], codes[1]);
      if (E8 && n + 1 < n1) step(n + 1, codes[1], codes[0]);
    }
    if (todo > 0) {
      have = next_run(saved_args(base + L::ARGS));
      if (have) {
        block_barrier();  // both stages may still be read
        fetch(n0, codes[0]);
        if (E8 && n0 + 1 < n1) fetch(n0 + 1, codes[1]);
        place(n0, codes[0]);
      }
    } else {
      have = false;
    }
  }

  block_barrier();  // all marks are made, the stages are free
  stash<W, D>(w, base, base + L::STATS, wave * SH + lane % SH);
  block_barrier();
  const int first = u.tile * L::ROWS;
  finish<W, D, L::ROWS, WAVES / RW, true>(
      base + L::ARGS, base, base + L::STATS, marks, any, min(gr.rows - first, L::ROWS), gr.q0, first, h, u.split, u.splits,
      info + 4 * 3 * L::ROWS, [&](int r) { return lds_read<int>(info + 4 * r) >= 0 && (lds_read<int>(info + 4 * r) & BIG); });
}

// Tiles first: they take longer (64 decodes behind 8192 tokens: 30.6 us, the other way round 35.6).
template <int DT, bool E8, int D, int RW>
__global__ void __launch_bounds__(THREADS, 2) attend(Args a) {
  extern __shared__ __align__(16) char smem[];
  const int index = (int)blockIdx.x;
  const uint32_t arg_word = argument_word();
  if (index < a.tile_blocks)
    row_tile<DT, E8, D, RW>(a, smem, index, arg_word);
  else
    stream_rows<DT, E8, D>(a, smem, index - a.tile_blocks, arg_word);
}

// ------------------------------------------------------------------ combine

// The slots of a row: those of its tiles, as slots 0 .. tile - 1 of S1, and those of its streams, S1 .. S1 + own - 1.
//
// Where all of them for every row take at most 512 MB, they lie together, slot s of row `id` at id * (S1 + S2) + s, and the
// maxima and sums of all are read along with the counts, one round of loads less (those of unused slots mean nothing).
// Otherwise (`compact`) only rows that need slots have them: each row of a split tile as many as the tile has splits (a
// tile of x > 1 shares is cut into fewer than 2 x, of at most FILL shares in all, so there are at most 2 * FILL such
// splits; in a last round of tiles FILL), and each row of a sequence of up to 16 rows S2 for its streams and one for a tile
// that was not split.  Their places are read along with the counts (combine at 4385 queries of 32 heads: 13.2 us, with
// slots for every row 12.5, which took 1 GB).
template <bool COMPACT>
struct Slots {
  int tile = 0, own = 0, tile_at = 0, own_at = 0;
  Slots() = default;
  __device__ __forceinline__ Slots(const Args& a, int64_t id, int first, int end) {
    const int t = (int)(id / a.Hq);
    const int n_tile = a.S1 > 0 ? a.n_tile[id] : 0, n_own = a.n_own[id];
    if (COMPACT) {
      tile_at = a.S1 > 0 ? a.tile_at[id] : 0;
      own_at = a.own_at[id];
    }
    const bool inside = t >= first && t < end;  // else a row of no sequence
    tile = inside ? min(n_tile, a.S1) : 0;
    own = inside ? clamp_int(n_own, 0, a.S2) : 0;
  }
  // those that lane k holds
  __device__ __forceinline__ Slots of(int k) const {
    Slots s;
    s.tile = __builtin_amdgcn_readlane(tile, k);
    s.own = __builtin_amdgcn_readlane(own, k);
    s.tile_at = __builtin_amdgcn_readlane(tile_at, k);
    s.own_at = __builtin_amdgcn_readlane(own_at, k);
    return s;
  }
  __device__ __forceinline__ bool has(const Args& a, int slot) const {
    return slot < a.S1 ? slot < tile : slot < a.S1 + own;
  }
  // where a slot that the row has lies (offsets that the sequences do not cover are read as any others, hence the limits)
  __device__ __forceinline__ int64_t at(const Args& a, int64_t id, int slot) const {
    if (!COMPACT) return id * (a.S1 + a.S2) + slot;
    const int64_t mine = own_slot(a, clamp_int(own_at, 0, a.own_rows - 1));
    if (slot >= a.S1) return mine + slot - a.S1;
    return tile_at < 0 ? mine + a.S2 : clamp_int(tile_at, 0, max(a.tile_slots - a.S1, 0)) + slot;
  }
};

// One wavefront a row: lane n reads the maximum and sum of slots n and n + 64, then all lanes add the slots' outputs in
// order, sixteen of them in flight.  A wavefront looks through `run` rows for those that their tile has not written
// already (most of a prompt's); its rows lie far apart, since the others lie together.
template <int DT, int D, bool COMPACT>
__global__ void __launch_bounds__(THREADS) combine(Args a, int run) {
  typedef typename Ty<DT>::el el;
  constexpr int PER = D / 64, AT_ONCE = 16;
  struct alignas(4 * PER) Part { float x[PER]; };
  struct alignas(2 * PER) Out { el x[PER]; };
  const int lane = threadIdx.x & 63, n = a.S1 + a.S2;
  const int64_t rows = (int64_t)a.T * a.Hq, all = (int64_t)gridDim.x * WAVES;
  const int64_t id0 = (int64_t)blockIdx.x * WAVES + (threadIdx.x >> 6);
  const int first = query_start(a, 0), end = query_start(a, a.B);
  bool open = lane < run && id0 + lane * all < rows;
  Slots<COMPACT> held;
  if (open && (COMPACT || run > 1)) {
    held = Slots<COMPACT>(a, id0 + lane * all, first, end);
    open = held.tile >= 0;
  }
  for (unsigned long long rest = __ballot(open); rest; rest &= rest - 1) {
    const int k = __builtin_ctzll(rest);
    const int64_t id = id0 + k * all;
    float2 ml[2] = {float2{NEG_INF, 0.0f}, float2{NEG_INF, 0.0f}};
    if (!COMPACT) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (lane + 64 * i < n) ml[i] = a.part_ml[id * n + lane + 64 * i];
    }
    const Slots<COMPACT> slots = COMPACT ? held.of(k) : Slots<COMPACT>(a, id, first, end);
    if (slots.tile < 0) continue;
    if (COMPACT) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (slots.has(a, lane + 64 * i)) ml[i] = a.part_ml[slots.at(a, id, lane + 64 * i)];
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (!slots.has(a, lane + 64 * i)) ml[i] = float2{NEG_INF, 0.0f};
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
      unsigned long long live = __ballot(!(ml[i].y == 0.0f));  // an empty slot's output is not there; a NaN counts
      while (live) {
        Part p[AT_ONCE];
        float w[AT_ONCE];
#pragma unroll
        for (int k = 0; k < AT_ONCE; ++k) {
          const int s = live ? __builtin_ctzll(live) : 0;
          w[k] = live ? __shfl(weight[i], s) : 0.0f;
          p[k] = Part{};
          if (live) p[k] = *(const Part*)(a.part_o + slots.at(a, id, s + 64 * i) * D + lane * PER);
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
}

// The same with a block a row, for many slots (of few rows: they lie together): lanes 0 .. 31 and 32 .. 63 of each wavefront read a slot's output each.
template <int DT, int D>
__global__ void __launch_bounds__(THREADS) combine_many(Args a) {
  typedef typename Ty<DT>::el el;
  constexpr int PER = D / 32, HALVES = 2 * WAVES;
  struct alignas(4 * PER) Part { float x[PER]; };
  __shared__ float joined[HALVES][D];
  const int lane = threadIdx.x & 63, half = (int)threadIdx.x >> 5, at = lane & 31, n = a.S1 + a.S2;
  const int64_t rows = (int64_t)a.T * a.Hq, id = blockIdx.x;
  float2 ml[2] = {float2{NEG_INF, 0.0f}, float2{NEG_INF, 0.0f}};
#pragma unroll
  for (int i = 0; i < 2; ++i)
    if (lane + 64 * i < n) ml[i] = a.part_ml[id * n + lane + 64 * i];
  const Slots<false> slots(a, id, query_start(a, 0), query_start(a, a.B));
  if (slots.tile < 0) return;  // written by its tile
#pragma unroll
  for (int i = 0; i < 2; ++i)
    if (!slots.has(a, lane + 64 * i)) ml[i] = float2{NEG_INF, 0.0f};
  float top = fmaxf(ml[0].x, ml[1].x);
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
  float weight[2], sum = 0.0f;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    weight[i] = ml[i].y == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(ml[i].x - (top == NEG_INF ? 0.0f : top));
    sum += weight[i] * ml[i].y;
  }
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d);
  float x[PER] = {};
#pragma unroll 8
  for (int s0 = 0; s0 < n; s0 += HALVES) {  // all lanes take part: the shuffles read any lane
    const int s = s0 + half;
    const float w0 = __shfl(weight[0], s & 63), w1 = __shfl(weight[1], s & 63);
    const float l0 = __shfl(ml[0].y, s & 63), l1 = __shfl(ml[1].y, s & 63);
    const float w = s < 64 ? w0 : w1, l = s < 64 ? l0 : l1;
    Part p{};
    if (s < n && !(l == 0.0f)) p = *(const Part*)(a.part_o + (id * n + s) * D + at * PER);  // an empty one is not there
#pragma unroll
    for (int k = 0; k < PER; ++k) x[k] += w * p.x[k];
  }
#pragma unroll
  for (int k = 0; k < PER; ++k) joined[half][at * PER + k] = x[k];
  __syncthreads();
  for (int c = threadIdx.x; c < D; c += THREADS) {
    float y = 0.0f;
#pragma unroll
    for (int k = 0; k < HALVES; ++k) y += joined[k][c];
    ((el*)a.out)[id * D + c] = (el)(y * inverse(sum));
  }
  if (threadIdx.x == 0) a.lse[id] = natural_lse(top, sum);
}

// ------------------------------------------------------------------ host

struct Plan {
  int64_t tile_blocks = 0, stream_blocks = 0, each_blocks = 0;  // upper bounds
  int row_waves = 2;                                            // tiles of 64 or 128 rows
  int tile_fill = FILL;
  int S1 = 0, S2 = 0, stream_least = 0;
  bool joint = false, rounds = false, many = false;  // many: slots a row
  bool compact = false, direct_rows = true;
  int64_t tile_slots = 0, own_rows = 0, slots = 0;  // compact; of partial results
  int64_t bytes = 0;
};

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline int64_t between(int64_t x, int64_t lo, int64_t hi) { return x < lo ? lo : x > hi ? hi : x; }

// Short calls, and calls of many sequences without prefixes: a block for each sequence and head, which saves the combine
// (a second launch and the partial results, about 5 us) for at most 16 MB of prefixes read again.  Otherwise tiles of
// 128 rows, or of 64 where groups have few; splits of at least 256 tokens; the own tokens in streams.
inline Plan make_plan(int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t G, int64_t Wp, int64_t B, int64_t W,
                      int64_t page, int64_t max_q, bool e8) {
  Plan p;
  const int64_t grp = Hq / Hkv, rows = T * grp, groups = G > 0 ? G : 1;
  const bool big = max_q * grp > FEW;
  p.joint = Wp > 0 && !big && (Wp + W) * page <= 1024 && B * Hkv * Wp * page * D * 4 <= (16 << 20);
  if (p.joint || (Wp == 0 && !big && (B * Hkv >= 2 * FILL || W * page <= 512))) {
    p.each_blocks = B * Hkv;
    return p;
  }
  int64_t tiles = 0;  // blocks of them that run at once
  if (Wp > 0 || big) {
    // a group's rows padded to tiles, those of 64 counted 5 / 4 (they read each token twice as often)
    const int64_t each = ceil_div(rows, groups);
    p.row_waves = ceil_div(each, 128) * 128 <= ceil_div(each, 64) * 80 ? 4 : 2;
    const int64_t tile = 32 * p.row_waves, units = ceil_div(rows, tile) * Hkv;
    const int64_t tokens = (Wp + (big ? W : 0)) * page, cuts = ceil_div(tokens, 256);
    p.rounds = units >= FILL;
    // Where there is more to read of own tokens than of prefixes by all tiles, tiles leave every CU's second place to
    // the streams (64 decodes of up to 1024 own tokens behind 32768: 76 us, else 81); where less, they take both places
    // (96 sequences of up to 1400 own tokens in four groups of up to 15689: 124 us, else 139).
    p.tile_fill = !big && B * W * Hkv >= units * Wp ? FILL / 2 : FILL;
    p.S1 = (int)between(cuts, 1, p.rounds ? 8 : MAX_SPLIT);
    if (groups == 1 && !p.rounds) p.S1 = (int)between(p.tile_fill / between(units, 1, FILL), 1, p.S1);
    p.tile_blocks = (rows / tile + groups) * Hkv + FILL;
    tiles = p.rounds ? FILL : between(units * p.S1, 1, p.tile_fill);
    p.many = p.tile_fill / units > 24 && T * Hq <= 16384;  // at most 21 units of 128 rows: never compact
  }
  // A sequence falls to at most S2 - 1 full streams and one more; S2 up to 64, as far as 512 MB of partial results go, but
  // at least 4.
  const int64_t tok = (e8 || D == 64) ? 64 : 32, most = ceil_div(W * page, tok), row_bytes = D * 4 + 8;
  auto streams = [&](int64_t rows_of_streams) {
    const int64_t slots = between(PARTIALS / (rows_of_streams * row_bytes), 4, MAX_SPLIT);
    p.stream_least = (int)ceil_div(most, slots - 1);
    p.S2 = (int)(ceil_div(most, p.stream_least) + 1);
  };
  streams(T * Hq);
  p.slots = (p.S1 + p.S2) * T * Hq;
  p.compact = p.slots * row_bytes > PARTIALS;
  if (p.compact) {
    p.own_rows = big ? between(B * Hkv * FEW, 1, T * Hq) : T * Hq;
    p.direct_rows = p.own_rows == T * Hq;
    streams(p.own_rows);
    p.tile_slots = p.S1 > 1 ? (p.rounds ? 1 : 2) * FILL * 32 * p.row_waves : 0;
    p.slots = p.tile_slots + p.own_rows * (p.S2 + 1);
  }
  // Streams fill the device after tiles that do so (those four groups: 118 us, with half as many 124), or beside few
  // tiles most of it (64 decodes of 1024 to 4096 own tokens behind 1000: 130 us, with FILL / 2 152); beside as many
  // tiles as they are, all run at once (64 decodes of up to 1024 behind 8192: 41 us, with FILL 44).
  const int64_t fill = tiles > FILL / 2 || tiles == 0 ? FILL : tiles <= FILL / 4 ? FILL * 3 / 4 : FILL / 2;
  p.stream_blocks = between(ceil_div(B * Hkv * most, WAVES * p.stream_least), 1, fill);
  p.bytes = p.slots * row_bytes + (p.compact ? 4 : 2) * T * Hq * 4;
  return p;
}

template <int DT, bool E8, int D, int RW>
tb_status launch(Args& a, const Plan& p, hipStream_t stream, const char* what) {
  constexpr int own = StreamLayout<DT, E8, D>::LDS, tile = TileLayout<DT, E8, D, RW>::LDS;
  constexpr size_t lds = own > tile ? own : tile;
  static_assert(lds <= 81920, "two blocks a CU");
  if (tb_status s = reserve_lds((const void*)attend<DT, E8, D, RW>, lds, what)) return s;
  hipLaunchKernelGGL((attend<DT, E8, D, RW>), dim3((unsigned)(p.tile_blocks + p.stream_blocks)), dim3(THREADS), lds, stream,
                     a);
  if (tb_status s = launch_status(what)) return s;
  const int64_t rows = (int64_t)a.T * a.Hq, most = WAVES << 22;  // a launch holds 2^32 threads
  const int64_t run = rows > most ? 64 : a.big && rows >= 32768 ? 16 : 1;
  if (p.many) {  // 65 to 108 slots (8 queries about 131001 tokens): 116.6 us in all, by wavefronts 118.7
    hipLaunchKernelGGL((combine_many<DT, D>), dim3((unsigned)rows), dim3(THREADS), 0, stream, a);
  } else {
    const auto kernel = p.compact ? combine<DT, D, true> : combine<DT, D, false>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)ceil_div(rows, WAVES * run)), dim3(THREADS), 0, stream, a, (int)run);
  }
  return launch_status(what);
}

template <int DT, bool E8, int D>
tb_status launch_each(Args& a, const Plan& p, hipStream_t stream, const char* what) {
  constexpr size_t lds = FewLayout<DT, E8, D>::LDS;
  static_assert(lds <= 81920, "two blocks a CU");
  if (tb_status s = reserve_lds((const void*)attend_each<DT, E8, D>, lds, what)) return s;
  hipLaunchKernelGGL((attend_each<DT, E8, D>), dim3((unsigned)p.each_blocks), dim3(THREADS), lds, stream, a);
  return launch_status(what);
}

template <int DT, bool E8, int D>
tb_status launch_rows(Args& a, const Plan& p, hipStream_t stream, const char* what) {
  if (p.each_blocks) return launch_each<DT, E8, D>(a, p, stream, what);
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
  TB_CHECK_ARG(T <= most && Hq <= most && B <= most && G <= most && max_q <= most && T * Hq <= most &&
                   max_q * Hq <= most && B * Hkv <= most / MAX_SPLIT / 4 && G * Hkv <= most / MAX_SPLIT / 4 &&
                   W <= most / 4 / page_size && Wp <= most / 4 / page_size,
               "%s: sizes past 2^31", what);
  TB_CHECK_ARG(B == 0 || W == 0 || Hkv * B <= (1ll << 30) / ceil_div(W * page_size, 32),
               "%s: %lld sequences times %lld key/value heads times tables of %lld tokens in steps of 32 exceed 2^30", what,
               (long long)B, (long long)Hkv, (long long)(W * page_size));
  return TB_OK;
}

}  // namespace prefix
}  // namespace tb

extern "C" tb_status tb_shared_prefix_attention_workspace_size(int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t G,
                                                               int64_t Wp, int64_t B, int64_t W, int64_t page_size,
                                                               int64_t max_q, int cache_dtype, int64_t* bytes) {
  using namespace tb::prefix;
  const char* what = "tb_shared_prefix_attention_workspace_size";
  TB_CHECK_ARG(bytes, "%s: null pointer", what);
  if (tb_status s = check_sizes(what, T, Hq, Hkv, D, G, Wp, B, W, page_size, max_q)) return s;
  *bytes = T == 0 || B == 0 || W == 0 ? 0 : make_plan(T, Hq, Hkv, D, G, Wp, B, W, page_size, max_q, cache_dtype == 3).bytes;
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
  TB_CHECK_ARG(fabs(scale) < 1e38, "%s: the scale must be finite (in 32 bits)", what);
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
  const Plan p = make_plan(T, Hq, Hkv, D, G, Wp, B, W, page_size, max_q, cache_dtype == 3);
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
  a.part_ml = (float2*)((char*)workspace + p.slots * D * 4);
  a.n_tile = (int*)((char*)workspace + p.slots * (D * 4 + 8));
  a.n_own = a.n_tile + T * Hq;
  a.tile_at = a.n_own + T * Hq;  // these two compact only
  a.own_at = a.tile_at + T * Hq;
  a.compact = p.compact;
  a.direct_rows = p.direct_rows;
  a.own_first = p.compact ? (int)p.tile_slots : p.S1;
  a.own_stride = p.compact ? p.S2 + 1 : p.S1 + p.S2;
  a.tile_slots = (int)p.tile_slots;
  a.own_rows = (int)p.own_rows;
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
  a.streams = (int)(p.stream_blocks * WAVES);
  a.stream_least = p.stream_least;
  a.scale_log2 = scale == 0.0 ? 1.0f : (float)((scale < 0.0 ? -scale : scale) * 1.44269504088896340736);
  a.flip = scale < 0.0 ? 0x80008000u : 0u;
  a.keep = scale == 0.0 ? 0u : ~0u;
  a.joint = p.joint;
  a.rounds = p.rounds;
  a.tile_fill = p.tile_fill;
  a.by_grp = tb::Divisor((uint32_t)a.grp);
  a.by_heads = tb::Divisor((uint32_t)Hkv);
  a.near = c_slot >= 0 && c_slot < (1 << 23);
  a.big = max_q * a.grp > FEW;
  a.tile_blocks = (int)p.tile_blocks;
  const bool e8 = cache_dtype == 3;
  return dtype == F16 ? launch_for<F16>(e8, D, a, p, stream, what) : launch_for<BF16>(e8, D, a, p, stream, what);
}
