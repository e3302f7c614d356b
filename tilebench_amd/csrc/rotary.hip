// Rotary positions with several axes, and their fusion with appending to a
// paged key/value cache (memory-bound).
//
//   angle[t, i] = positions[axes[i], t] * inv_freq[i]          i = 0 .. R/2 - 1
//   (a, b) -> (a cos - b sin, b cos + a sin)                   for every pair i of a head
//
// with the pairs (x[i], x[i + R/2]) or, interleaved, (x[2i], x[2i+1]); channels
// R .. D-1 pass through.  The transpose of a rotation is the rotation by the
// negated angle, so the gradient is the same kernel with the sine negated.
//
// Angles.  A 32-bit product loses 2^-24 of the angle: 4e-3 rad at position
// 65536, more than an fp16 ulp of the result.  The product and its reduction
// to [-1/2, 1/2] turns are done in 64 bits, sine and cosine of the reduced angle
// in 32 (1 ulp).  They depend on (token, pair) only, so a block computes them
// once per token into LDS and all heads read them there: 64 per token instead of
// 64 per head and token.
//
// Layout of the work.  A head is D / (2 VEC) items of 2 VEC elements, one item a
// lane; LP = the next power of two lanes hold a head, so that the absolute
// maximum of an 8-bit cache row is a shuffle reduction and the row is read
// once.  VEC = 8 makes 16-byte accesses; VEC = 4 and 1 serve heads, rotations
// or strides that are not multiples of 16 (all widths give the same bits).
//
// 8-bit cache rows: s = absmax / 448 over the fp32 values (rotated, never
// rounded to 16 bits before), code = e4m3(x / s), both IEEE; a row of zeros
// stores s = 0 and codes 0; a row with inf or NaN reads back as NaN.
#include "tb_common.h"

namespace tb {
namespace rotary {

constexpr int THREADS = 256, MAX_TOKENS = 4, MAX_D = 512;

enum { F32 = 0, F16 = 1, BF16 = 2 };
enum { DENSE = 0, CACHE = 1, CACHE_E4M3 = 2 };

template <int DT>
struct Elem;
template <>
struct Elem<F32> {
  typedef float type;
  static __device__ __forceinline__ float up(float x) { return x; }
  static __device__ __forceinline__ float down(float x) { return x; }
};
template <>
struct Elem<F16> {
  typedef _Float16 type;
  static __device__ __forceinline__ float up(_Float16 x) { return (float)x; }
  static __device__ __forceinline__ _Float16 down(float x) { return (_Float16)x; }
};
template <>
struct Elem<BF16> {
  typedef uint16_t type;
  static __device__ __forceinline__ float up(uint16_t x) { return __builtin_bit_cast(float, (uint32_t)x << 16); }
  static __device__ __forceinline__ uint16_t down(float x) { return (uint16_t)bf16_bits(x); }
};

// One of q, k, v: `heads` rows a token, at element strides st (token) and sh (head).
struct Source {
  const void* p;
  int64_t st, sh;
  int heads;
};

struct Args {
  Source src[3];       // q, k, v (v.heads = 0 without a cache)
  void* out[3];        // dense outputs [T, heads, D]; k and v: the cache pools
  float* scale[2];     // scales of k and v (8-bit caches)
  int64_t cp, ch, cs;  // cache strides in elements: page, head, slot
  int64_t sp, sh, ss;  // scale strides
  const int* positions;  // [A, T]
  const float* inv_freq;
  const int* axes;  // null: every pair follows axis 0
  const int* slots;
  int64_t n_slots;
  int page_shift;
  int64_t T;
  int D, P, A;  // P = R / 2 pairs
  int lp_shift, items, tokens;
  int interleaved, inverse;
};

template <typename E, int VEC>
struct alignas(VEC * sizeof(E) < 16 ? VEC * sizeof(E) : 16) Chunk {
  E e[VEC];
};

// cos and sin of position * frequency: the turns and their nearest whole number in 64 bits.
__device__ __forceinline__ float2 cos_sin(int pos, float freq, bool inverse) {
  const double turns = (double)pos * (double)freq * 0.15915494309189533577;
  const float x = (float)(2.0 * (turns - __builtin_rint(turns)));
  float s, c;
  sincospif(x, &s, &c);
  return float2{c, inverse ? -s : s};
}

template <int DT, int VEC, int MODE>
__global__ void __launch_bounds__(THREADS) rotate_heads(Args a) {
  typedef Elem<DT> E;
  typedef typename E::type T;
  typedef Chunk<T, VEC> C;
  constexpr int PASSES = VEC == 1 ? MAX_D / 128 : 1;  // items of a lane
  __shared__ float2 trig[MAX_TOKENS * MAX_D / 2];

  const int tid = threadIdx.x;
  const int64_t t0 = (int64_t)blockIdx.x * a.tokens;
  const int here = (int)min((int64_t)a.tokens, a.T - t0);  // tokens of this block
  const int rows = a.src[0].heads + a.src[1].heads + a.src[2].heads;
  const int lp = 1 << a.lp_shift, lane = tid & (lp - 1), per_pass = THREADS >> a.lp_shift;
  const int total = here * rows, stride = per_pass * (int)gridDim.y;
  const int rot_items = a.P / VEC;

  C x1[PASSES], x2[PASSES];
  auto offset1 = [&](int j) __attribute__((always_inline)) {
    return j < rot_items && !a.interleaved ? j * VEC : 2 * j * VEC;
  };
  auto offset2 = [&](int j) __attribute__((always_inline)) {
    return j < rot_items && !a.interleaved ? a.P + j * VEC : (2 * j + 1) * VEC;
  };
  // head `row` of the token tile: its section and head within it
  auto locate = [&](int row, int& sec, int& head, int& tok) __attribute__((always_inline)) {
    tok = row / rows;
    head = row - tok * rows;
    sec = 0;
    if (head >= a.src[0].heads) {
      head -= a.src[0].heads;
      sec = 1;
      if (head >= a.src[1].heads) {
        head -= a.src[1].heads;
        sec = 2;
      }
    }
  };
  auto load = [&](int row) __attribute__((always_inline)) {
    int sec, head, tok;
    locate(row, sec, head, tok);
    const Source& s = a.src[sec];
    const T* p = (const T*)s.p + (t0 + tok) * s.st + head * s.sh;
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      const int j = lane + i * lp;
      if (j < a.items) {
        x1[i] = *(const C*)(p + offset1(j));
        x2[i] = *(const C*)(p + offset2(j));
      }
    }
  };

  // the first rows are on their way while the angles are computed
  int row = (int)blockIdx.y * per_pass + (tid >> a.lp_shift);
  if (row < total) load(row);
  for (int i = tid; i < here * a.P; i += THREADS) {
    const int tok = i / a.P, pair = i - tok * a.P;
    const int ax = a.axes ? min(max(a.axes[pair], 0), a.A - 1) : 0;
    trig[i] = cos_sin(a.positions[ax * a.T + t0 + tok], a.inv_freq[pair], a.inverse);
  }
  __syncthreads();

  for (; row < total; row += stride) {
    int sec, head, tok;
    locate(row, sec, head, tok);
    float y1[PASSES][VEC], y2[PASSES][VEC];
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      const int j = lane + i * lp;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        y1[i][e] = j < a.items ? E::up(x1[i].e[e]) : 0.0f;
        y2[i][e] = j < a.items ? E::up(x2[i].e[e]) : 0.0f;
      }
      if (sec < 2 && j < rot_items) {
        const float2* cs = trig + tok * a.P + j * VEC;
        if (VEC > 1 && a.interleaved) {
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            float* y = 2 * e < VEC ? &y1[i][(2 * e) % VEC] : &y2[i][(2 * e) % VEC];
            const float p = y[0], q = y[1];
            y[0] = p * cs[e].x - q * cs[e].y;
            y[1] = q * cs[e].x + p * cs[e].y;
          }
        } else {
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            const float p = y1[i][e], q = y2[i][e];
            y1[i][e] = p * cs[e].x - q * cs[e].y;
            y2[i][e] = q * cs[e].x + p * cs[e].y;
          }
        }
      }
    }
    const int64_t t = t0 + tok;
    // the next row's loads go out before this row's stores
    const int next = row + stride;
    if (next < total) load(next);

    int64_t at;
    if (MODE == DENSE || sec == 0) {
      at = (t * a.src[sec].heads + head) * a.D;
    } else {
      const int64_t slot = a.slots[t];
      if (slot < 0 || slot >= a.n_slots) continue;  // a padded token: nothing is written
      const int64_t page = slot >> a.page_shift, in = slot & ((1 << a.page_shift) - 1);
      at = page * a.cp + head * a.ch + in * a.cs;
      if (MODE == CACHE_E4M3) {
        // the largest magnitude as bits: NaN above inf above every number
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < PASSES; ++i)
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            m = max(m, __builtin_bit_cast(uint32_t, y1[i][e]) & 0x7FFFFFFFu);
            m = max(m, __builtin_bit_cast(uint32_t, y2[i][e]) & 0x7FFFFFFFu);
          }
        for (int d = lp >> 1; d > 0; d >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, d));
        const float s = __builtin_bit_cast(float, m) / 448.0f;
        if (lane == 0) a.scale[sec - 1][page * a.sp + head * a.sh + in * a.ss] = s;
        uint8_t* dst = (uint8_t*)a.out[sec] + at;
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
          const int j = lane + i * lp;
          if (j >= a.items) continue;
          Chunk<uint8_t, VEC> c1, c2;
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            c1.e[e] = m == 0 ? 0 : (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(y1[i][e] / s, 0.0f, 0, false);
            c2.e[e] = m == 0 ? 0 : (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(y2[i][e] / s, 0.0f, 0, false);
          }
          *(Chunk<uint8_t, VEC>*)(dst + offset1(j)) = c1;
          *(Chunk<uint8_t, VEC>*)(dst + offset2(j)) = c2;
        }
        continue;
      }
    }
    T* dst = (T*)a.out[sec] + at;
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      const int j = lane + i * lp;
      if (j >= a.items) continue;
      C c1, c2;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        c1.e[e] = E::down(y1[i][e]);
        c2.e[e] = E::down(y2[i][e]);
      }
      *(C*)(dst + offset1(j)) = c1;
      *(C*)(dst + offset2(j)) = c2;
    }
  }
}

template <int DT, int VEC, int MODE>
tb_status launch(const Args& a, dim3 grid, hipStream_t stream, const char* what) {
  hipLaunchKernelGGL((rotate_heads<DT, VEC, MODE>), grid, dim3(THREADS), 0, stream, a);
  return launch_status(what);
}

template <int DT, int MODE>
tb_status launch_vec(int vec, const Args& a, dim3 grid, hipStream_t stream, const char* what) {
  if (vec == 8) return launch<DT, 8, MODE>(a, grid, stream, what);
  if (vec == 4) return launch<DT, 4, MODE>(a, grid, stream, what);
  return launch<DT, 1, MODE>(a, grid, stream, what);
}

// The widest access that every head, rotation, stride and pointer allows.
struct Width {
  int vec = 8;
  void lengths(int64_t P, int64_t D) {
    while (vec > 1 && (P % vec || (D - 2 * P) % (2 * vec))) vec = vec == 8 ? 4 : 1;
  }
  void tensor(const void* p, int64_t elem, int64_t s0, int64_t s1, int64_t s2) {
    while (vec > 1) {
      const int64_t bytes = vec * elem < 16 ? vec * elem : 16;
      if ((uintptr_t)p % bytes == 0 && s0 % vec == 0 && s1 % vec == 0 && s2 % vec == 0) return;
      vec = vec == 8 ? 4 : 1;
    }
  }
};

// Fills the launch geometry.  Blocks of one pass over their rows for up to 2048
// of them (a decode batch: as many loads as possible at once), beyond that
// blocks of four tokens, whose threads make several passes and share the angles.
inline dim3 geometry(Args& a, int vec) {
  a.items = a.D / (2 * vec);
  int lp_shift = 0;
  while ((1 << lp_shift) < a.items && lp_shift < 6) ++lp_shift;
  a.lp_shift = lp_shift;
  const int64_t rows = a.src[0].heads + a.src[1].heads + a.src[2].heads;
  const int64_t per_pass = THREADS >> lp_shift;
  const int64_t split = (rows + per_pass - 1) / per_pass;
  if (a.T * split <= 2048) {
    a.tokens = 1;
    return dim3((unsigned)a.T, (unsigned)split);
  }
  a.tokens = MAX_TOKENS;
  return dim3((unsigned)((a.T + MAX_TOKENS - 1) / MAX_TOKENS), 1);
}

inline tb_status check_rotation(const char* what, int64_t T, int64_t Hq, int64_t Hk, int64_t D, int64_t R, int64_t A) {
  TB_CHECK_ARG(T >= 0 && T < (1ll << 31), "%s: bad number of tokens %lld", what, (long long)T);
  TB_CHECK_ARG(Hq >= 1 && Hk >= 0 && Hq <= 65536 && Hk <= 65536, "%s: bad numbers of heads %lld, %lld", what,
               (long long)Hq, (long long)Hk);
  TB_CHECK_ARG(D >= 2 && D <= MAX_D && D % 2 == 0, "%s: the head dimension must be even and at most %d (got %lld)", what,
               MAX_D, (long long)D);
  TB_CHECK_ARG(R >= 2 && R <= D && R % 2 == 0, "%s: the rotated channels must be even, 2 .. D (got %lld of %lld)", what,
               (long long)R, (long long)D);
  TB_CHECK_ARG(A >= 1 && A <= 8, "%s: need 1 .. 8 axes (got %lld)", what, (long long)A);
  return TB_OK;
}

}  // namespace rotary
}  // namespace tb

extern "C" tb_status tb_rotary_axes(const void* q, void* q_out, const void* k, void* k_out, const int32_t* positions,
                                    const float* inv_freq, const int32_t* axes, int64_t T, int64_t Hq, int64_t Hk,
                                    int64_t D, int64_t R, int64_t A, int64_t q_st, int64_t q_sh, int64_t k_st,
                                    int64_t k_sh, int dtype, int interleaved, int inverse, hipStream_t stream) {
  using namespace tb::rotary;
  const char* what = "tb_rotary_axes";
  if (tb_status s = check_rotation(what, T, Hq, Hk, D, R, A)) return s;
  TB_CHECK_ARG(dtype >= F32 && dtype <= BF16, "%s: unknown dtype %d", what, dtype);
  TB_CHECK_ARG(A == 1 || axes, "%s: %lld axes need the axis of every pair", what, (long long)A);
  if (T == 0) return TB_OK;  // tensors without elements have null pointers
  TB_CHECK_ARG(q && q_out && positions && inv_freq && (Hk == 0 || (k && k_out)), "%s: null pointer", what);
  Args a{};
  a.src[0] = Source{q, q_st, q_sh, (int)Hq};
  a.src[1] = Source{k, k_st, k_sh, (int)Hk};
  a.out[0] = q_out;
  a.out[1] = k_out;
  a.positions = positions;
  a.inv_freq = inv_freq;
  a.axes = axes;
  a.T = T;
  a.D = (int)D;
  a.P = (int)(R / 2);
  a.A = (int)A;
  a.interleaved = interleaved != 0;
  a.inverse = inverse != 0;
  const int64_t elem = dtype == F32 ? 4 : 2;
  Width w;
  w.lengths(a.P, D);
  w.tensor(q, elem, q_st, q_sh, 0);
  w.tensor(q_out, elem, D, 0, 0);
  if (Hk) {
    w.tensor(k, elem, k_st, k_sh, 0);
    w.tensor(k_out, elem, D, 0, 0);
  }
  const dim3 grid = geometry(a, w.vec);
  if (dtype == F32) return launch_vec<F32, DENSE>(w.vec, a, grid, stream, what);
  if (dtype == F16) return launch_vec<F16, DENSE>(w.vec, a, grid, stream, what);
  return launch_vec<BF16, DENSE>(w.vec, a, grid, stream, what);
}

extern "C" tb_status tb_rope_kv_append(const void* q, const void* k, const void* v, void* q_out,
                                       const int32_t* positions, const float* inv_freq, const int32_t* axes,
                                       const int32_t* slots, void* k_cache, void* v_cache, float* k_scale,
                                       float* v_scale, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t R,
                                       int64_t A, int64_t q_st, int64_t q_sh, int64_t k_st, int64_t k_sh, int64_t v_st,
                                       int64_t v_sh, int64_t pages, int64_t page_size, int64_t c_page, int64_t c_head,
                                       int64_t c_slot, int64_t s_page, int64_t s_head, int64_t s_slot, int dtype,
                                       int cache_dtype, int interleaved, hipStream_t stream) {
  using namespace tb::rotary;
  const char* what = "tb_rope_kv_append";
  if (tb_status s = check_rotation(what, T, Hq, Hkv, D, R, A)) return s;
  TB_CHECK_ARG(Hkv >= 1, "%s: need at least one key/value head", what);
  TB_CHECK_ARG(dtype == F16 || dtype == BF16, "%s: unknown dtype %d", what, dtype);
  TB_CHECK_ARG(cache_dtype == dtype || cache_dtype == 3, "%s: the cache holds %d, the inputs are %d (3 is e4m3)", what,
               cache_dtype, dtype);
  TB_CHECK_ARG((cache_dtype == 3) == (k_scale != nullptr) && (cache_dtype == 3) == (v_scale != nullptr),
               "%s: scales belong to e4m3 caches, and only to them", what);
  TB_CHECK_ARG(A == 1 || axes, "%s: %lld axes need the axis of every pair", what, (long long)A);
  TB_CHECK_ARG(page_size >= 1 && page_size <= 4096 && (page_size & (page_size - 1)) == 0,
               "%s: the page size must be a power of two up to 4096 (got %lld)", what, (long long)page_size);
  TB_CHECK_ARG(pages >= 1 && pages <= ((1ll << 31) - 1) / page_size, "%s: bad number of pages %lld", what,
               (long long)pages);
  if (T == 0) return TB_OK;
  TB_CHECK_ARG(q && k && v && q_out && positions && inv_freq && slots && k_cache && v_cache, "%s: null pointer", what);
  Args a{};
  a.src[0] = Source{q, q_st, q_sh, (int)Hq};
  a.src[1] = Source{k, k_st, k_sh, (int)Hkv};
  a.src[2] = Source{v, v_st, v_sh, (int)Hkv};
  a.out[0] = q_out;
  a.out[1] = k_cache;
  a.out[2] = v_cache;
  a.scale[0] = k_scale;
  a.scale[1] = v_scale;
  a.cp = c_page;
  a.ch = c_head;
  a.cs = c_slot;
  a.sp = s_page;
  a.sh = s_head;
  a.ss = s_slot;
  a.positions = positions;
  a.inv_freq = inv_freq;
  a.axes = axes;
  a.slots = slots;
  a.n_slots = pages * page_size;
  a.page_shift = __builtin_ctzll((unsigned long long)page_size);
  a.T = T;
  a.D = (int)D;
  a.P = (int)(R / 2);
  a.A = (int)A;
  a.interleaved = interleaved != 0;
  const int64_t c_elem = cache_dtype == 3 ? 1 : 2;
  Width w;
  w.lengths(a.P, D);
  w.tensor(q, 2, q_st, q_sh, 0);
  w.tensor(k, 2, k_st, k_sh, 0);
  w.tensor(v, 2, v_st, v_sh, 0);
  w.tensor(q_out, 2, D, 0, 0);
  w.tensor(k_cache, c_elem, c_page, c_head, c_slot);
  w.tensor(v_cache, c_elem, c_page, c_head, c_slot);
  const dim3 grid = geometry(a, w.vec);
  if (cache_dtype == 3)
    return dtype == F16 ? launch_vec<F16, CACHE_E4M3>(w.vec, a, grid, stream, what)
                        : launch_vec<BF16, CACHE_E4M3>(w.vec, a, grid, stream, what);
  return dtype == F16 ? launch_vec<F16, CACHE>(w.vec, a, grid, stream, what)
                      : launch_vec<BF16, CACHE>(w.vec, a, grid, stream, what);
}
