// Microscaled 4-bit floating point (MXFP4): quantisation and reading back.
//
// A row of K values is K / 32 blocks.  A block's scale is the power of two
// 2^e, e = floor(log2(largest magnitude)) - 2 held to -127 .. 127, stored as the
// byte e + 127; its values are e2m1 codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a
// sign) of x * 2^-e, rounded to nearest even, magnitudes beyond 6 to 6 (x * 2^-e
// is below 8).  Two codes a byte, the lower channel in the low four bits.  A block
// of zeros has scale 0; one with inf or NaN has scale 255, the NaN of these
// scales, and zero codes.  Scaling by a power of two is exact, so codes and scales
// have one right value each.
//
// Gated: the values are silu(g) * u = g / (1 + exp(-g)) * u, and codes and scales those of the product in
// 64 bits.  Nearly all are settled in fp32: a value comes with a bound of its error, both ends of that range are rounded,
// and where they agree (and the block's exponent does) that is the answer; a wavefront with a value next to a
// border computes in 64 bits (about one in a thousand on N(0, 1) gates; zeros are settled like other values).  16008 x 1408
// bf16, calls replayed over changing inputs: 26 us, with zeros among the values or half of the rows 25, with all in 64 bits 66.
//
// Both are bound by memory: 4096 x 7168 bf16 (74 MB) 15.7 us to codes, 4.7 TB/s, and 16.3 back, replayed over changing
// operands (back from codes just written: 13.0); 16384 x 4096 31 and 30 us, 5.5 and 5.8 TB/s.  Four lanes share a block, eight channels each: a
// lane's 16-bit channels are one 16-byte load (a wavefront reads 1 KiB runs), its
// codes one 4-byte store, and the block's largest magnitude takes two exchanges
// between lanes.  A thread takes four units in turn: loads of all four first hold registers and take a seventh
// longer, one or two units a thread make no difference.
#include "tb_common.h"

namespace tb {
namespace mxfp4 {

constexpr int THREADS = 256, UNIT = 8;   // channels of a lane
constexpr int CHUNK = 1024;              // units of a thread block: one row's, or several short rows'

// Units of a launch: thread block (x, y) takes rows x * rows_per_block .. and columns y * cols .. of units.
struct Shape {
  int64_t M;
  int64_t x_row;      // elements
  int64_t scale_row;  // bytes
  int upr;            // units of a row: K / 8
  int cols, rows;     // units of a row and rows that a thread block takes
  Divisor by_cols;
};

__device__ __forceinline__ float half_bits(uint32_t v, int dtype) {
  return dtype == 1 ? (float)__builtin_bit_cast(_Float16, (uint16_t)v) : __builtin_bit_cast(float, v << 16);
}

template <int DTYPE>
__device__ __forceinline__ void load_unit(const void* x, int64_t at, float (&v)[UNIT]) {
  if constexpr (DTYPE == 0) {
    const f32x4* p = reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(x) + at);
    const f32x4 a = p[0], b = p[1];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = a[i], v[4 + i] = b[i];
  } else {
    const u32x4 a = *reinterpret_cast<const u32x4*>(reinterpret_cast<const uint16_t*>(x) + at);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = half_bits(a[i] & 0xFFFFu, DTYPE);
      v[2 * i + 1] = half_bits(a[i] >> 16, DTYPE);
    }
  }
}

// The largest of the four lanes that share a block.
__device__ __forceinline__ uint32_t max4(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, true));  // lanes 1 0 3 2
  return max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xF, 0xF, true));  // lanes 2 3 0 1
}

__device__ __forceinline__ float power(int biased) {  // 2^(biased - 127)
  return __builtin_bit_cast(float, biased == 0 ? 0x00400000u : (uint32_t)biased << 23);
}

// The e2m1 codes of eight values below 8 in magnitude, or beyond 6 by any amount.
__device__ __forceinline__ uint32_t codes8(const float (&v)[UNIT]) {
  uint32_t c = 0;
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[0], v[1], 1.f, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2], v[3], 1.f, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[4], v[5], 1.f, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[6], v[7], 1.f, 3);
}

// Scale byte and codes of the lane's part of a block; all four lanes take part.
// Scaled in fp32: exact, or below 2^-126, which is code 0 either way.
__device__ __forceinline__ uint32_t quantise(const float (&v)[UNIT], int& byte) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < UNIT; ++i) top = max(top, __builtin_bit_cast(uint32_t, v[i]) & 0x7FFFFFFFu);
  top = max4(top);
  if (top >= 0x7F800000u) {
    byte = 255;
    return 0;
  }
  byte = max((int)(top >> 23) - 2, 0);  // magnitudes below 2^-126 included
  const float inverse = power(254 - byte);
  float q[UNIT];
#pragma unroll
  for (int i = 0; i < UNIT; ++i) q[i] = v[i] * inverse;
  return codes8(q);
}

// The same of products silu(g) * u in fp32, with bounds; false where these do not settle a code or the scale.
// Relative error: 1 ulp each of exp2 and of the reciprocal, half of the sum, the two products and the ends' own roundings,
// together 5 * 2^-23, and the exponent's own, |t| ln 2 times the rounding of t and of log2(e), below |t| 2^-23.  Beyond |g| = 80, for tiny
// blocks (products below the normals) and for what is not finite the bounds do not hold.  Nor for gates below the normals:
// g / 2 has few bits there, which a large u makes those of an ordinary product (halves of 16-bit types' gates are exact, and
// of a normal gate it loses 2^-23 at most).
template <int DTYPE>
__device__ __forceinline__ bool quantise_gated_bounded(const float (&g)[UNIT], const float (&u)[UNIT], int& byte, uint32_t& codes) {
  float lo[UNIT], hi[UNIT];
  uint32_t top_lo = 0, top_hi = 0;
  float most = 0.f;
  bool small = false;  // a gate below the normals, but not 0
#pragma unroll
  for (int i = 0; i < UNIT; ++i) {
    if constexpr (DTYPE == 0) small |= __builtin_amdgcn_classf(g[i], 0x90);
    const float t = g[i] * 1.44269504f;
    const float v = g[i] * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-t)) * u[i];
    const float b = __builtin_fmaf(__builtin_fabsf(t), 0x1p-23f, 0x1p-20f);
    most = fmaxf(most, __builtin_fabsf(g[i]));
    lo[i] = v * (1.f - b);  // a sum v - b v would make +0 of -0
    hi[i] = __builtin_fmaf(b, v, v);
    top_lo = max(top_lo, __builtin_bit_cast(uint32_t, lo[i]) & 0x7FFFFFFFu);
    top_hi = max(top_hi, __builtin_bit_cast(uint32_t, hi[i]) & 0x7FFFFFFFu);
  }
  top_lo = max4(top_lo);
  top_hi = max4(top_hi);
  byte = max((int)(top_hi >> 23) - 2, 0);
  const float inverse = power(max(254 - byte, 0));
#pragma unroll
  for (int i = 0; i < UNIT; ++i) {
    lo[i] *= inverse;
    hi[i] *= inverse;
  }
  codes = codes8(hi);
  // a block of zeros is one in 64 bits too, or of products below 2^-149: scale 0 and zero codes with their signs either way
  return (top_hi == 0 || (top_lo >> 23 == top_hi >> 23 && top_hi < 0x7F800000u && top_lo >= 0x0D800000u)) && most <= 80.f &&
         !small && codes == codes8(lo);
}

// The same of products silu(g) * u in 64 bits.  What goes on to the 4-bit rounding
// is cut to fp32 with the last bit set where anything was cut off: a value next to a
// border between codes stays on its side.
__device__ __forceinline__ uint32_t quantise_gated(const float (&g)[UNIT], const float (&u)[UNIT], int& byte) {
  double v[UNIT];
  uint32_t top = 0;  // the high word orders magnitudes by their exponents
#pragma unroll
  for (int i = 0; i < UNIT; ++i) {
    v[i] = (double)g[i] / (1.0 + exp(-(double)g[i])) * (double)u[i];
    top = max(top, (uint32_t)(__builtin_bit_cast(uint64_t, v[i]) >> 32) & 0x7FFFFFFFu);
  }
  top = max4(top);
  if (top >= 0x7FF00000u) {
    byte = 255;
    return 0;
  }
  byte = min(max((int)(top >> 20) - 1023 + 127 - 2, 0), 254);
  const double inverse = __builtin_bit_cast(double, (uint64_t)(1023 + 127 - byte) << 52);
  float q[UNIT];
#pragma unroll
  for (int i = 0; i < UNIT; ++i) {
    const double s = v[i] * inverse;
    const float cut = __double2float_rz(s);
    q[i] = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, cut) | (uint32_t)((double)cut != s));
  }
  return codes8(q);
}

template <int DTYPE, bool GATED>
__global__ void __launch_bounds__(THREADS)
    mxfp4_quant_kernel(const void* __restrict__ x, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, Shape s) {
  const int64_t row0 = (int64_t)blockIdx.x * s.rows;
  const int col0 = (int)blockIdx.y * s.cols;
  const int n = (int)min((int64_t)s.rows, s.M - row0) * s.cols;
  // a row is a whole number of blocks of four units, so the lanes of a block are all in or all out
  for (int i = threadIdx.x; i < n; i += THREADS) {
    const int r = s.by_cols.divide(i), c = col0 + s.by_cols.rest(i, r);
    if (c >= s.upr) continue;
    const int64_t row = row0 + r, at = row * s.x_row + (int64_t)c * UNIT;
    float v[UNIT];
    load_unit<DTYPE>(x, at, v);
    int byte;
    uint32_t q;
    if constexpr (GATED) {
      float u[UNIT];
      load_unit<DTYPE>(x, at + (int64_t)s.upr * UNIT, u);
      if (!__all(quantise_gated_bounded<DTYPE>(v, u, byte, q))) q = quantise_gated(v, u, byte);
    } else {
      q = quantise(v, byte);
    }
    reinterpret_cast<uint32_t*>(codes)[row * s.upr + c] = q;
    if ((c & 3) == 0) scales[row * s.scale_row + (c >> 2)] = (uint8_t)byte;
  }
}

// value = code * 2^(scale - 127) in fp32 (exact, or beyond its range), rounded once to the type.
template <int DTYPE>
__global__ void __launch_bounds__(THREADS)
    mxfp4_dequant_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, void* __restrict__ y, Shape s) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  const int64_t row0 = (int64_t)blockIdx.x * s.rows;
  const int col0 = (int)blockIdx.y * s.cols;
  const int n = (int)min((int64_t)s.rows, s.M - row0) * s.cols;
  for (int i = threadIdx.x; i < n; i += THREADS) {
    const int r = s.by_cols.divide(i), c = col0 + s.by_cols.rest(i, r);
    if (c >= s.upr) continue;
    const int64_t row = row0 + r, at = row * s.upr + c;
    const uint32_t q = reinterpret_cast<const uint32_t*>(codes)[at];
    const int byte = scales[row * s.scale_row + (c >> 2)];
    const float scale = byte == 255 ? __builtin_nanf("") : power(byte);
    f32x2 v[4];
    v[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.f, 0);
    v[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.f, 1);
    v[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.f, 2);
    v[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.f, 3);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = f32x2{v[j][0] * scale, v[j][1] * scale};
    if constexpr (DTYPE == 0) {
      f32x4* const p = reinterpret_cast<f32x4*>(reinterpret_cast<float*>(y) + at * UNIT);
      p[0] = f32x4{v[0][0], v[0][1], v[1][0], v[1][1]};
      p[1] = f32x4{v[2][0], v[2][1], v[3][0], v[3][1]};
    } else {
      u32x4 o;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (DTYPE == 1)
          o[j] = as_u32(f16x2{(_Float16)v[j][0], (_Float16)v[j][1]});
        else
          o[j] = __builtin_bit_cast(uint32_t, __builtin_convertvector(v[j], bf16x2));
      }
      *reinterpret_cast<u32x4*>(reinterpret_cast<uint16_t*>(y) + at * UNIT) = o;
    }
  }
}

// Sizes of a launch over M rows of K values.
inline tb_status shape_of(const char* fn, int64_t M, int64_t K, int64_t x_row, int64_t scale_row, Shape* s, dim3* grid) {
  TB_CHECK_ARG(M > 0 && K > 0, "%s: sizes must be positive", fn);
  TB_CHECK_ARG(K % 32 == 0, "%s: K must be a multiple of 32 (got %lld)", fn, (long long)K);
  TB_CHECK_ARG(scale_row >= K / 32, "%s: rows of scales overlap", fn);
  const int64_t upr = K / UNIT;
  s->M = M;
  s->x_row = x_row;
  s->scale_row = scale_row;
  s->cols = (int)(upr < CHUNK ? upr : CHUNK);
  s->rows = CHUNK / s->cols;
  const int64_t gx = (M + s->rows - 1) / s->rows, gy = (upr + s->cols - 1) / s->cols;
  TB_CHECK_ARG(gx < (1ll << 23) && gy < 65536, "%s: problem too large (M=%lld K=%lld)", fn, (long long)M, (long long)K);
  s->upr = (int)upr;
  s->by_cols = Divisor((uint32_t)s->cols);
  *grid = dim3((unsigned)gx, (unsigned)gy);
  return TB_OK;
}

}  // namespace mxfp4
}  // namespace tb

extern "C" tb_status tb_mxfp4_quant(const void* x, uint8_t* codes, uint8_t* scales, int64_t M, int64_t K, int64_t x_row,
                                    int64_t scale_row, int gated, int dtype, hipStream_t stream) {
  using namespace tb::mxfp4;
  const char* const fn = "tb_mxfp4_quant";
  TB_CHECK_ARG(x && codes && scales, "%s: null pointer", fn);
  TB_CHECK_ARG(dtype >= 0 && dtype <= 2, "%s: unknown type %d", fn, dtype);
  Shape s;
  dim3 grid;
  if (tb_status st = shape_of(fn, M, K, x_row, scale_row, &s, &grid)) return st;
  TB_CHECK_ARG(x_row >= 0 && x_row % (dtype == 0 ? 4 : 8) == 0, "%s: rows of x must start on 16 bytes (stride %lld)", fn,
               (long long)x_row);
  TB_CHECK_ALIGN(x, 16, "x");
  TB_CHECK_ALIGN(codes, 4, "codes");
  auto* const kernel = gated ? (dtype == 0 ? &mxfp4_quant_kernel<0, true>
                                : dtype == 1 ? &mxfp4_quant_kernel<1, true> : &mxfp4_quant_kernel<2, true>)
                             : (dtype == 0 ? &mxfp4_quant_kernel<0, false>
                                : dtype == 1 ? &mxfp4_quant_kernel<1, false> : &mxfp4_quant_kernel<2, false>);
  hipLaunchKernelGGL(kernel, grid, dim3(THREADS), 0, stream, x, codes, scales, s);
  return tb::launch_status(fn);
}

extern "C" tb_status tb_mxfp4_dequant(const uint8_t* codes, const uint8_t* scales, void* y, int64_t M, int64_t K,
                                      int64_t scale_row, int dtype, hipStream_t stream) {
  using namespace tb::mxfp4;
  const char* const fn = "tb_mxfp4_dequant";
  TB_CHECK_ARG(codes && scales && y, "%s: null pointer", fn);
  TB_CHECK_ARG(dtype >= 0 && dtype <= 2, "%s: unknown type %d", fn, dtype);
  Shape s;
  dim3 grid;
  if (tb_status st = shape_of(fn, M, K, K, scale_row, &s, &grid)) return st;
  TB_CHECK_ALIGN(codes, 4, "codes");
  TB_CHECK_ALIGN(y, 16, "y");
  auto* const kernel = dtype == 0 ? &mxfp4_dequant_kernel<0>
                       : dtype == 1 ? &mxfp4_dequant_kernel<1> : &mxfp4_dequant_kernel<2>;
  hipLaunchKernelGGL(kernel, grid, dim3(THREADS), 0, stream, codes, scales, y, s);
  return tb::launch_status(fn);
}
