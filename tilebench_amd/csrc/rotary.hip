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
// 65536, more than an fp16 ulp of the result.  The product, its reduction and sine
// and cosine are done in 64 bits, which cost what 32 bits do here, and rounded to
// 32.  They depend on (token, pair) only: a wavefront computes its
// token's once into LDS and its lanes read them there for 8 rows of 128.
//
// Layout of the work.  A head is D / (2 VEC) items of 2 VEC elements, one item a
// lane, two accesses of 16 bytes (VEC = 8; 4 for fp32).  A wavefront takes 64
// items of one token and the four of a block follow each other in memory; no
// barrier, no loop.  Where a row's maximum is needed (8-bit caches), a power of
// two of lanes holds it, so the row is read once and the maximum is a shuffle.
// VEC = 4 and 1 serve heads, rotations or strides that are not multiples of 16
// bytes (all widths give the same bits).
//
// What bounds it: bytes in flight.  A wavefront lives for its chain of loads, a
// microsecond or more each, so axes, frequencies, positions, slots and rows are all asked
// for before the first of them is waited for: 20001 tokens of 32 + 8 fp16 heads
// of 128 take 74 us (5.5 TB/s), and 80 us (5.1 TB/s) with the positions' loads
// behind the axes'.  A 410 MB copy takes 64 us.  Wavefronts with 2, 3 and 4 times the
// items take 80, 95 and 124 us (before that change); four tokens to a block and
// a loop over their heads 83 us; 8-byte accesses 96 us.  Replayed from a graph, 4800
// tokens of 16 + 16 bf16 heads of 80 take 11.2 us (4.4 TB/s), 7001 tokens into a bf16
// cache 30.3 us (5.7 TB/s), 4096 into an 8-bit cache 21.0 us (4.4 TB/s), one token 3.0 us.
//
// 8-bit cache rows: s = absmax / 448 and code = e4m3(x / s), as in 64 bits: the
// scale is rounded to 32 bits, the quotient to 32 and then to 8.  Keys are rotated
// (by sines and cosines of 2^-36), compared and divided in 64 bits; with 32 a few
// quotients in a million fall on the other side of a border between codes (4096
// tokens on one card: 19.0 us, so 20.5, values in 64 bits too 21.3).  Values are divided in 32
// bits, the quotient corrected by the exact remainder.  A row of zeros stores s = 0
// and codes 0; a row with inf or NaN reads back as NaN.
#include "tb_common.h"

namespace tb {
namespace rotary {

constexpr int THREADS = 256, WAVES = 4, MAX_D = 512;

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
  static __device__ __forceinline__ _Float16 down(float x) {
    asm("" : "+v"(x));  // or single values would be rounded once, within the product (v_fma_mixlo_f16), and wide ones twice
    return (_Float16)x;
  }
};
template <>
struct Elem<BF16> {
  typedef __bf16 type;
  static __device__ __forceinline__ float up(__bf16 x) { return (float)x; }
  static __device__ __forceinline__ __bf16 down(float x) { return (__bf16)x; }
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
  int items, lanes;    // items of a head, lanes that hold it
  Divisor by_lanes, by_portions;
  int rows, portions;  // heads of a token; wavefronts that share them
  int64_t t0, end;     // tokens of the launch
  int interleaved, inverse;
};

template <typename E, int VEC>
struct alignas(VEC * sizeof(E) < 16 ? VEC * sizeof(E) : 16) Chunk {
  E e[VEC];
};

// cos and sin of position * frequency, in 64 bits: the nearest whole turn and quarter turn are taken off, which is
// exact, and the Taylor series are summed over the rest, |angle| <= pi / 4 (x^13 / 13! < 2^-37 and x^14 / 14! < 2^-41 are
// left out).
__device__ __forceinline__ double2 cos_sin(int pos, float freq, bool inverse) {
  double turns = (double)pos * (double)freq * 0.15915494309189533577;
  turns -= __builtin_rint(turns);
  const double quarter = __builtin_rint(4.0 * turns);
  const double x = __builtin_fma(4.0, turns, -quarter) * 1.57079632679489661923, z = x * x;
  double s = -1.0 / 39916800.0, c = 1.0 / 479001600.0;
  c = __builtin_fma(c, z, -1.0 / 3628800.0);
  s = __builtin_fma(s, z, 1.0 / 362880.0);
  c = __builtin_fma(c, z, 1.0 / 40320.0);
  s = __builtin_fma(s, z, -1.0 / 5040.0);
  c = __builtin_fma(c, z, -1.0 / 720.0);
  s = __builtin_fma(s, z, 1.0 / 120.0);
  c = __builtin_fma(c, z, 1.0 / 24.0);
  s = __builtin_fma(s, z, -1.0 / 6.0);
  c = __builtin_fma(c, z, -0.5);
  const double sine = __builtin_fma(s * z, x, x), cosine = __builtin_fma(c, z, 1.0);
  const int n = (int)quarter;
  const double u = n & 1 ? sine : cosine, v = n & 1 ? cosine : sine;
  return double2{(n + 1) & 2 ? -u : u, ((n & 2) != 0) != inverse ? -v : v};
}

__device__ __forceinline__ uint32_t upper(double x) {
  return (uint32_t)(__builtin_bit_cast(uint64_t, x) >> 32) & 0x7FFFFFFFu;
}

// x / (s + rest) rounded to 32 bits, for s in [2^-60, 2^60] with the rounded reciprocal inv: the product with that,
// corrected once by the exact remainder.
struct Reciprocal {
  float s, rest, inv;
  __device__ __forceinline__ float operator()(float x) const {
    const float q = x * inv;
    return fmaf(fmaf(-q, rest, fmaf(-q, s, x)), inv, q);
  }
};
struct Reciprocal64 {
  double inv;
  __device__ __forceinline__ float operator()(double x) const { return (float)(x * inv); }
};

// e4m3 codes of N (1 or a multiple of 4) quotients.
template <int N, typename F, typename Quotient>
__device__ __forceinline__ void codes(const F* x, Quotient quotient, uint8_t* c) {
  float y[N < 4 ? 4 : N] = {};
#pragma unroll
  for (int e = 0; e < N; ++e) y[e] = quotient(x[e]);
#pragma unroll
  for (int e = 0; e < N; e += 4) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[e], y[e + 1], 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(y[e + 2], y[e + 3], w, true);
    __builtin_memcpy(c + e, &w, N < 4 ? N : 4);
  }
}

// The pairs of an item, (x1[e], x2[e]) or neighbours within its 2 N elements, by the angles of its N pairs.
template <int N, bool INTER, typename F, typename CosSin>
__device__ __forceinline__ void rotate(F (&x1)[N], F (&x2)[N], const CosSin* cs) {
#pragma unroll
  for (int e = 0; e < N; ++e) {
    F& u = INTER && N > 1 ? (2 * e < N ? x1[(2 * e) % N] : x2[(2 * e) % N]) : x1[e];
    F& v = INTER && N > 1 ? (2 * e < N ? x1[(2 * e + 1) % N] : x2[(2 * e + 1) % N]) : x2[e];
    const F p = u, q = v;
    u = fma(p, cs[e].x, -(q * cs[e].y));  // written out, so that all widths round alike
    v = fma(q, cs[e].x, p * cs[e].y);
  }
}

template <int DT, int VEC, int MODE, bool INTER>
__global__ void __launch_bounds__(THREADS) rotate_heads(Args a) {
  typedef Elem<DT> E;
  typedef typename E::type T;
  typedef Chunk<T, VEC> C;
  constexpr int PASSES = VEC == 1 ? MAX_D / 128 : 1;  // items of a lane
  // cosines and sines of the block's wavefronts; 8-bit caches have them in 64 bits too
  extern __shared__ __align__(16) char smem[];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const uint32_t portion = blockIdx.x * WAVES + wave, token = (uint32_t)a.by_portions.divide((int)portion);
  const int64_t t = a.t0 + token;
  if (t >= a.end) return;  // no barrier follows
  float2* const trig = (float2*)smem + wave * a.P;
  double2* const fine = (double2*)(smem + WAVES * a.P * sizeof(float2)) + wave * a.P;
  const int n = (int)(portion - token * (uint32_t)a.portions) * 64 + lane;
  const int row = a.by_lanes.divide(n), item = n - row * a.lanes;
  const bool is_k = row >= a.src[0].heads, is_v = MODE != DENSE && row >= a.src[0].heads + a.src[1].heads;
  const int head = row - (is_k ? a.src[0].heads : 0) - (is_v ? a.src[1].heads : 0);
  const bool in = row < a.rows;
  auto offset1 = [&](int j) __attribute__((always_inline)) { return j * VEC < a.P && !INTER ? j * VEC : 2 * j * VEC; };
  auto offset2 = [&](int j) __attribute__((always_inline)) {
    return j * VEC < a.P && !INTER ? a.P + j * VEC : (2 * j + 1) * VEC;
  };

  // What the angles are made of is asked for first, then the row: it is on its way while they are computed.  No load
  // waits for another (each takes a microsecond in a busy memory system).
  const int places = a.axes && a.A > 1 ? min(lane, a.A - 1) : 0;
  const int axis = a.axes ? a.axes[min(lane, a.P - 1)] : 0;
  const float freq = a.inv_freq[min(lane, a.P - 1)];
  const int place = a.positions[places * a.T + t];  // lane i: on axis i
  const int64_t slot = MODE == DENSE ? 0 : a.slots[t];
  C x1[PASSES], x2[PASSES];
  if (in) {
    const T* p = is_v   ? (const T*)a.src[2].p + t * a.src[2].st
                 : is_k ? (const T*)a.src[1].p + t * a.src[1].st
                        : (const T*)a.src[0].p + t * a.src[0].st;
    p += head * (is_v ? a.src[2].sh : is_k ? a.src[1].sh : a.src[0].sh);
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      const int j = item + i * 64;
      if (j < a.items) {
        x1[i] = *(const C*)(p + offset1(j));
        x2[i] = *(const C*)(p + offset2(j));
      }
    }
  }
  for (int i = lane;; i += 64) {
    const bool mine = i < a.P, more = i >= 64;
    const int ax = more && mine && a.axes ? a.axes[i] : axis;
    const int pos = __shfl(place, min(max(ax, 0), a.A - 1));
    if (mine) {
      const double2 cs = cos_sin(pos, more ? a.inv_freq[i] : freq, a.inverse);
      trig[i] = float2{(float)cs.x, (float)cs.y};
      if (MODE == CACHE_E4M3) fine[i] = cs;
    }
    if (i - lane + 64 >= a.P) break;
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");

  // where a row of the caches goes (a padded token: nowhere)
  const bool kept = in && (MODE == DENSE || !is_k || (slot >= 0 && slot < a.n_slots));
  const int64_t page = slot >> a.page_shift, within = slot & ((1 << a.page_shift) - 1);
  if (MODE == CACHE_E4M3 && is_v) {  // values are not rotated: 32 bits hold them
    float y1[PASSES][VEC], y2[PASSES][VEC];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < PASSES; ++i)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        y1[i][e] = item + i * 64 < a.items ? E::up(x1[i].e[e]) : 0.0f;
        y2[i][e] = item + i * 64 < a.items ? E::up(x2[i].e[e]) : 0.0f;
        top = max(top, __builtin_bit_cast(uint32_t, y1[i][e]) & 0x7FFFFFFFu);
        top = max(top, __builtin_bit_cast(uint32_t, y2[i][e]) & 0x7FFFFFFFu);
      }
    for (int d = a.lanes >> 1; d > 0; d >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, d));
    if (!kept) return;
    const float most = __builtin_bit_cast(float, top), s = most / 448.0f;
    const Reciprocal by{s, fmaf(-448.0f, s, most) / 448.0f, 1.0f / s};
    const bool normal = s >= 0x1p-60f && s <= 0x1p60f;
    const double inv = most == 0.0f ? 0.0 : 448.0 / (double)most;
    if (item == 0) a.scale[1][page * a.sp + head * a.sh + within * a.ss] = s;
    uint8_t* dst = (uint8_t*)a.out[2] + page * a.cp + head * a.ch + within * a.cs;
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      const int j = item + i * 64;
      if (j >= a.items) continue;
      Chunk<uint8_t, VEC> c1, c2;
      if (normal) {
        codes<VEC>(y1[i], by, c1.e);
        codes<VEC>(y2[i], by, c2.e);
      } else {
        codes<VEC>(y1[i], Reciprocal64{inv}, c1.e);
        codes<VEC>(y2[i], Reciprocal64{inv}, c2.e);
      }
      *(Chunk<uint8_t, VEC>*)(dst + offset1(j)) = c1;
      *(Chunk<uint8_t, VEC>*)(dst + offset2(j)) = c2;
    }
    return;
  }
  if (MODE == CACHE_E4M3 && is_k) {
    double y1[PASSES][VEC], y2[PASSES][VEC], most = 0.0;
    uint32_t top = 0;  // the largest magnitude's upper half: NaN above inf above every number
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      const int j = item + i * 64;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        y1[i][e] = j < a.items ? E::up(x1[i].e[e]) : 0.0f;
        y2[i][e] = j < a.items ? E::up(x2[i].e[e]) : 0.0f;
      }
      if (j * VEC < a.P) rotate<VEC, INTER>(y1[i], y2[i], fine + j * VEC);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        most = fmax(most, fmax(fabs(y1[i][e]), fabs(y2[i][e])));
        top = max(top, max(upper(y1[i][e]), upper(y2[i][e])));
      }
    }
    for (int d = a.lanes >> 1; d > 0; d >>= 1) {
      most = fmax(most, __shfl_xor(most, d));
      top = max(top, (uint32_t)__shfl_xor((int)top, d));
    }
    if (!kept) return;
    if (top >= 0x7FF00000u) most = top > 0x7FF00000u ? __builtin_nan("") : __builtin_inf();
    const double inv = most == 0.0 ? 0.0 : 448.0 / most;
    if (item == 0) a.scale[0][page * a.sp + head * a.sh + within * a.ss] = (float)(most * (1.0 / 448.0));
    uint8_t* dst = (uint8_t*)a.out[1] + page * a.cp + head * a.ch + within * a.cs;
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      const int j = item + i * 64;
      if (j >= a.items) continue;
      Chunk<uint8_t, VEC> c1, c2;
      codes<VEC>(y1[i], Reciprocal64{inv}, c1.e);
      codes<VEC>(y2[i], Reciprocal64{inv}, c2.e);
      *(Chunk<uint8_t, VEC>*)(dst + offset1(j)) = c1;
      *(Chunk<uint8_t, VEC>*)(dst + offset2(j)) = c2;
    }
    return;
  }
  if (!kept) return;
  const int64_t at = MODE != DENSE && is_k ? page * a.cp + head * a.ch + within * a.cs
                                           : (t * (is_k ? a.src[1].heads : a.src[0].heads) + head) * a.D;
  T* dst = (T*)(is_v ? a.out[2] : is_k ? a.out[1] : a.out[0]) + at;
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const int j = item + i * 64;
    if (j >= a.items) continue;
    float y1[VEC], y2[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      y1[e] = E::up(x1[i].e[e]);
      y2[e] = E::up(x2[i].e[e]);
    }
    if (!is_v && j * VEC < a.P) rotate<VEC, INTER>(y1, y2, trig + j * VEC);
    C c1, c2;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      c1.e[e] = E::down(y1[e]);
      c2.e[e] = E::down(y2[e]);
    }
    *(C*)(dst + offset1(j)) = c1;
    *(C*)(dst + offset2(j)) = c2;
  }
}

template <int DT, int VEC, int MODE>
tb_status launch(Args& a, hipStream_t stream, const char* what) {
  a.items = a.D / (2 * VEC);
  a.lanes = a.items;
  if (MODE == CACHE_E4M3 || VEC == 1)  // a power of two: the row's maximum is taken over its lanes
    for (a.lanes = 1; a.lanes < a.items && a.lanes < 64;) a.lanes *= 2;
  a.by_lanes = Divisor((uint32_t)a.lanes);
  a.rows = a.src[0].heads + a.src[1].heads + a.src[2].heads;
  a.portions = (a.rows * a.lanes + 63) / 64;
  a.by_portions = Divisor((uint32_t)a.portions);
  const size_t lds = WAVES * a.P * (sizeof(float2) + (MODE == CACHE_E4M3 ? sizeof(double2) : 0));
  const int64_t most = (1 << 25) / a.portions;  // tokens of a launch: it holds 2^32 threads
  for (a.t0 = 0; a.t0 < a.T; a.t0 += most) {
    const int64_t tokens = a.T - a.t0 < most ? a.T - a.t0 : most;
    a.end = a.t0 + tokens;
    const dim3 grid((unsigned)((tokens * a.portions + WAVES - 1) / WAVES));
    if (a.interleaved)
      hipLaunchKernelGGL((rotate_heads<DT, VEC, MODE, true>), grid, dim3(THREADS), lds, stream, a);
    else
      hipLaunchKernelGGL((rotate_heads<DT, VEC, MODE, false>), grid, dim3(THREADS), lds, stream, a);
    if (tb_status s = launch_status(what)) return s;
  }
  return TB_OK;
}

template <int DT, int MODE>
tb_status launch_vec(int vec, Args& a, hipStream_t stream, const char* what) {
  if constexpr (DT != F32)
    if (vec == 8) return launch<DT, 8, MODE>(a, stream, what);
  if (vec == 4) return launch<DT, 4, MODE>(a, stream, what);
  return launch<DT, 1, MODE>(a, stream, what);
}

// The widest access that every head, rotation, stride and pointer allows.
struct Width {
  int vec;
  explicit Width(int64_t elem) : vec(elem == 4 ? 4 : 8) {}
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
  Width w(elem);
  w.lengths(a.P, D);
  w.tensor(q, elem, q_st, q_sh, 0);
  w.tensor(q_out, elem, D, 0, 0);
  if (Hk) {
    w.tensor(k, elem, k_st, k_sh, 0);
    w.tensor(k_out, elem, D, 0, 0);
  }
  if (dtype == F32) return launch_vec<F32, DENSE>(w.vec, a, stream, what);
  if (dtype == F16) return launch_vec<F16, DENSE>(w.vec, a, stream, what);
  return launch_vec<BF16, DENSE>(w.vec, a, stream, what);
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
  Width w(2);
  w.lengths(a.P, D);
  w.tensor(q, 2, q_st, q_sh, 0);
  w.tensor(k, 2, k_st, k_sh, 0);
  w.tensor(v, 2, v_st, v_sh, 0);
  w.tensor(q_out, 2, D, 0, 0);
  w.tensor(k_cache, c_elem, c_page, c_head, c_slot);
  w.tensor(v_cache, c_elem, c_page, c_head, c_slot);
  if (cache_dtype == 3)
    return dtype == F16 ? launch_vec<F16, CACHE_E4M3>(w.vec, a, stream, what)
                        : launch_vec<BF16, CACHE_E4M3>(w.vec, a, stream, what);
  return dtype == F16 ? launch_vec<F16, CACHE>(w.vec, a, stream, what)
                      : launch_vec<BF16, CACHE>(w.vec, a, stream, what);
}
