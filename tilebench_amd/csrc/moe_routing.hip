// Routing to experts: scores, a bias for balance, groups, top-k, renormalised weights.
//
// Per row of logits x [E]:
//   s = 1 / (1 + exp(-x)), or exp(x - max) / sum of these (softmax);
//   c = s + bias: what experts are chosen by; s alone is what they are weighted by;
//   with groups of E / G consecutive experts, a group's score is the sum of its one or two largest c, and
//   only the experts of the top_groups best groups (equal scores: lowest group) can be chosen;
//   the k largest c of these, descending, equal ones by ascending expert; weights s of the
//   chosen, over their sum if asked for, times scale.
// All in 64 bits: neighbouring scores of a few hundred experts differ by less than
// fp32 rounds them, and a choice must not depend on how an exponential was computed.
// NaN ranks above every number, as in tb_moe_topk_gating.  A softmax row of
// -inf alone has scores 0; weights that sum to 0 stay 0.
//
// Two ways to the same results.
//
// Lanes (k <= 8, finite logits below 700 in magnitude, finite biases, lanes that do not straddle groups).  LPR
// lanes own a row, lane l its experts per * l .. per * l + per - 1, so a wavefront takes 64 / LPR rows.
//   1. scores: exp and the quotient written out in fp64 (unit(): 25 instructions, the library's exp and
//      division 50);
//   2. every lane sorts its choices, values only, and keeps the eight largest; the first one or two make the
//      groups' scores, and lanes of groups that are not among the best drop their lists;
//   3. lists of two lanes merge into the larger eight (max of one with the other reversed, then three rounds of a
//      bitonic network), over log2(LPR) rounds by DPP: every lane has the k-th largest value;
//   4. a lane's experts above it, and as many of those equal to it as fit (lowest first), go to an LDS list in the order
//      of their numbers; lane j takes the j-th, computes its score again and counts those before it.
//
// Rows (everything else): one wavefront a row, lane l holds experts l, 64 + l, ...; choices are compared as
// 64-bit keys in the order of their values (0: cannot be chosen), k rounds of a maximum over the wavefront.
// Rows of the first kind that hold inf, NaN or large logits are taken this way by their wavefront, one after the other; the
// rows beside them stay with the lanes, so that a row's results are its own (the ways' exponentials differ in their last bits).
//
// Bound by the chain of steps (1 row to a few hundred: 6 us, the launch included) and by fp64 instructions: 16384 x 256
// fp32 logits, sigmoid, 4 of 8 groups, k 8: 16 us with 40 % of the issue slots taken (18 MB, 3 us of HBM), and 64 one row to a
// wavefront.  A lane has 16 experts at
// most, two sorts of eight and a merge; more lanes a row mean more merges, of lists that are the same in all lanes by then.
// The second way: with k 12 69 us, with a quarter of the logits at -inf (k 8 or 12) 71 and 69, with one such row in seven 30.
#include "tb_common.h"

// a score is rounded before its bias is added, wherever it is computed
#pragma clang fp contract(off)

namespace tb {
namespace routing {

constexpr int WAVES = 4;

struct Args {
  const void* logits;
  const float* bias;
  float* weights;
  int32_t* ids;
  int64_t T, row;
  double scale;
  int E, k, groups, top_groups, group_top, softmax, renormalize, dtype;
  // route_lanes: experts of a lane, lanes of a group, whether these are a power of two, loads of 16 bytes, words of LDS of a wavefront
  int per, span, span_shift, vec, wave_words;
};

__device__ __forceinline__ float half_value(uint16_t v, int dtype) {
  return dtype == 1 ? (float)__builtin_bit_cast(_Float16, v) : __builtin_bit_cast(float, (uint32_t)v << 16);
}
__device__ __forceinline__ float logit(const void* p, int64_t i, int dtype) {
  if (dtype == 0) return reinterpret_cast<const float*>(p)[i];
  return half_value(reinterpret_cast<const uint16_t*>(p)[i], dtype);
}

// What the wavefront's lanes wrote to LDS is there for its other lanes.
__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// Order of doubles as an order of unsigned numbers above 0; -0 as 0, every NaN on top.
__device__ __forceinline__ uint64_t key_of(double c) {
  if (c != c) return ~0ull;
  const uint64_t b = __builtin_bit_cast(uint64_t, c + 0.0);
  return (b >> 63) ? ~b : b | (1ull << 63);
}
__device__ __forceinline__ double value_of(uint64_t key) {
  return __builtin_bit_cast(double, (key >> 63) ? (key == ~0ull ? 0x7FF8000000000000ull : key & ~(1ull << 63)) : ~key);
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) v += __shfl_xor(v, d);
  return v;
}

// The largest key of the wavefront and the lowest index that has it, in every lane.
__device__ __forceinline__ void wave_best(uint64_t& key, int& at) {
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) {
    const uint64_t k = (uint64_t)__shfl_xor((unsigned long long)key, d);
    const int i = __shfl_xor(at, d);
    if (k > key || (k == key && i < at)) key = k, at = i;
  }
}

// Row t by the whole wavefront; lds holds 2 E words.
template <int V>
__device__ void route_row(const Args& p, int64_t t, uint64_t* lds) {
  const int lane = threadIdx.x & 63;
  double* const ls = reinterpret_cast<double*>(lds);
  uint64_t* const lk = lds + p.E;

  double s[V];
  if (p.softmax) {
    float x[V], top = -__builtin_inff();
    bool nan = false;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int e = 64 * j + lane;
      x[j] = e < p.E ? logit(p.logits, t * p.row + e, p.dtype) : -__builtin_inff();
      nan |= x[j] != x[j];
      top = fmaxf(top, x[j]);
    }
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
    double sum = 0.0;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      s[j] = top == -__builtin_inff() && !nan ? 0.0 : exp((double)x[j] - (double)top);
      if (64 * j + lane < p.E) sum += s[j];
    }
    sum = wave_sum(sum);
#pragma unroll
    for (int j = 0; j < V; ++j) s[j] = sum == 0.0 ? 0.0 : s[j] / sum;
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int e = 64 * j + lane;
      s[j] = e < p.E ? 1.0 / (1.0 + exp(-(double)logit(p.logits, t * p.row + e, p.dtype))) : 0.0;
    }
  }
  uint64_t key[V];
  wave_fence();  // the row before may still be read
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int e = 64 * j + lane;
    key[j] = e < p.E ? key_of(p.bias ? s[j] + (double)p.bias[e] : s[j]) : 0;
    if (e < p.E) ls[e] = s[j], lk[e] = key[j];
  }
  wave_fence();

  if (p.groups > 1) {
    const int per = p.E / p.groups;
    uint64_t score = 0;
    if (lane < p.groups) {
      uint64_t a = 0, b = 0;  // the two largest
      for (int i = 0; i < per; ++i) {
        const uint64_t v = lk[lane * per + i];
        b = v > a ? a : v > b ? v : b;
        a = v > a ? v : a;
      }
      score = p.group_top == 2 ? key_of(value_of(a) + value_of(b)) : a;
    }
    uint64_t kept = 0;  // a bit per group
    for (int g = 0; g < p.top_groups; ++g) {
      uint64_t best = score;
      int at = lane;
      wave_best(best, at);
      kept |= 1ull << at;
      if (lane == at) score = 0;
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int e = 64 * j + lane;
      if (e < p.E && !((kept >> (e / per)) & 1)) key[j] = 0;
    }
  }

  int id = 0;  // lane j: the j-th choice
  for (int j = 0; j < p.k; ++j) {
    uint64_t best = 0;
    int at = 0;
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (key[i] > best) best = key[i], at = 64 * i + lane;
    if (best == 0) at = 1 << 20;  // nothing left in this lane
    wave_best(best, at);
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (at == 64 * i + lane) key[i] = 0;
    if (lane == j) id = at;
  }
  const double w = lane < p.k ? ls[id] : 0.0;
  const double sum = p.renormalize ? wave_sum(w) : 1.0;
  if (lane < p.k) {
    p.weights[t * p.k + lane] = (float)(sum == 0.0 ? 0.0 : w / sum * p.scale);
    p.ids[t * p.k + lane] = id;
  }
}

template <int V>
__global__ void __launch_bounds__(64 * WAVES) route_rows(Args p) {
  extern __shared__ uint64_t lds[];
  const int wave = threadIdx.x >> 6;
  const int64_t t = (int64_t)blockIdx.x * WAVES + wave;
  if (t < p.T) route_row<V>(p, t, lds + wave * 2 * p.E);  // no barrier: a row is one wavefront's
}

// ------------------------------------------------------------------ lanes

// exp(y) for y <= 700: y = n ln 2 + r with |r| <= 0.35 (ln 2 as a part of 44 bits, whose product with n is exact, and a
// rest), then the series of exp(r) up to r^13; the next term is below 2^-57.
__device__ __forceinline__ double exp64(double y) {
  const double n = __builtin_rint(y * 1.4426950408889634074);
  double r = __builtin_fma(n, -0x1.62e42fefa38p-1, y);
  r = __builtin_fma(n, -0x1.ef35793c7673p-45, r);
  double e = 1.0 / 6227020800.0;
  constexpr double C[13] = {1.0 / 479001600.0, 1.0 / 39916800.0, 1.0 / 3628800.0, 1.0 / 362880.0, 1.0 / 40320.0,
                            1.0 / 5040.0,      1.0 / 720.0,      1.0 / 120.0,     1.0 / 24.0,     1.0 / 6.0,
                            0.5,               1.0,              1.0};
#pragma unroll
  for (int i = 0; i < 13; ++i) e = __builtin_fma(e, r, C[i]);
  return __builtin_amdgcn_ldexp(e, (int)n);
}

// 1 / d for a normal d: two Newton steps.
__device__ __forceinline__ double inverse(double d) {
  double r = __builtin_amdgcn_rcp(d);
  r = __builtin_fma(__builtin_fma(-d, r, 1.0), r, r);
  return __builtin_fma(__builtin_fma(-d, r, 1.0), r, r);
}

// The score of a logit: of a softmax row exp(x - top) * share, share = 1 / sum.
__device__ __forceinline__ double unit(float x, int softmax, float top, double share) {
  const double e = exp64(softmax ? (double)x - (double)top : -(double)x);
  return softmax ? e * share : inverse(1.0 + e);
}

// v of a lane of the other half of 2, 4, 8 or 16 lanes (by DPP), or of 32 or 64.
template <int HALF>
__device__ __forceinline__ double other(double v) {
  if constexpr (HALF >= 16) {
    return __shfl_xor(v, HALF);
  } else {
    // lane ^ 1, lane ^ 2, 7 - lane within 8, 15 - lane within 16
    constexpr int CTRL = HALF == 1 ? 0xB1 : HALF == 2 ? 0x4E : HALF == 4 ? 0x141 : 0x140;
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_mov_dpp((int)(uint32_t)b, CTRL, 0xF, 0xF, true);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_mov_dpp((int)(uint32_t)(b >> 32), CTRL, 0xF, 0xF, true);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
  }
}

// No value here is NaN: one instruction each.
__device__ __forceinline__ double larger(double a, double b) { return __builtin_fmax(a, b); }
__device__ __forceinline__ double smaller(double a, double b) { return __builtin_fmin(a, b); }
__device__ __forceinline__ void order(double& a, double& b) {
  const double hi = larger(a, b), lo = smaller(a, b);
  a = hi;
  b = lo;
}

// Eight values in any order, descending (Batcher's network of 19).
__device__ __forceinline__ void sort8(double (&v)[8]) {
  constexpr int A[19] = {0, 2, 4, 6, 0, 1, 4, 5, 1, 5, 0, 1, 2, 3, 2, 3, 1, 3, 5};
  constexpr int B[19] = {1, 3, 5, 7, 2, 3, 6, 7, 2, 6, 4, 5, 6, 7, 4, 5, 2, 4, 6};
#pragma unroll
  for (int i = 0; i < 19; ++i) order(v[A[i]], v[B[i]]);
}
// ... of two descending lists, the eight largest: after this maximum they rise and fall once, which three rounds sort.
__device__ __forceinline__ void merge8(double (&a)[8], const double (&b)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) a[i] = larger(a[i], b[7 - i]);
#pragma unroll
  for (int d = 4; d >= 1; d >>= 1)
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (!(i & d)) order(a[i], a[i + d]);
}

template <int HALF, int LPR>
__device__ __forceinline__ void merge_lanes(double (&a)[8]) {
  if constexpr (HALF < LPR) {
    double b[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) b[i] = other<HALF>(a[i]);
    merge8(a, b);
    merge_lanes<2 * HALF, LPR>(a);
  }
}

template <int LPR>
__device__ __forceinline__ double row_sum(double v) {
  v += other<1>(v);
  v += other<2>(v);
  if constexpr (LPR > 4) v += other<4>(v);
  if constexpr (LPR > 8) v += other<8>(v);
  if constexpr (LPR > 16) v += other<16>(v);
  if constexpr (LPR > 32) v += other<32>(v);
  return v;
}

// V floats from byte offset `at` of a buffer, zeros past its end (no branch).
template <int V>
__device__ __forceinline__ void load_floats(const buf_rsrc_t& from, uint32_t at, float (&x)[V]) {
#pragma unroll
  for (int q = 0; q < V / 4; ++q) {
    const f32x4 v = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(from, at + 16u * q, 0, 0));
#pragma unroll
    for (int i = 0; i < 4; ++i) x[4 * q + i] = v[i];
  }
}
template <int V>
__device__ __forceinline__ void load_halves(const buf_rsrc_t& from, uint32_t at, int dtype, float (&x)[V]) {
#pragma unroll
  for (int q = 0; q < V / 8; ++q) {
    const u32x4 v = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(from, at + 16u * q, 0, 0));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[8 * q + 2 * i] = half_value((uint16_t)v[i], dtype);
      x[8 * q + 2 * i + 1] = half_value((uint16_t)(v[i] >> 16), dtype);
    }
  }
}

template <int LPR, int V, int WPB>
__global__ void __launch_bounds__(64 * WPB) route_lanes(Args p) {
  constexpr int ROWS = 64 / LPR;  // of a wavefront
  extern __shared__ uint64_t lds[];
  const int lane = threadIdx.x & 63, l = lane % LPR, base = lane - l;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t t0 = ((int64_t)blockIdx.x * WPB + wave) * ROWS, t = t0 + lane / LPR;
  if (t0 >= p.T) return;  // no barrier: a row is one wavefront's
  bool live = t < p.T;
  const int e0 = l * p.per;
  int n = live ? min(max(p.E - e0, 0), p.per) : 0;
  uint64_t* const own_lds = lds + wave * p.wave_words;

  float x[V], b[V];
  load_floats<V>(buf_rsrc(p.bias, p.bias ? (uint32_t)p.E * 4u : 0u), (uint32_t)e0 * 4u, b);
  if (p.vec) {
    const int size = p.dtype ? 2 : 4, rows = (int)min((int64_t)ROWS, p.T - t0);
    const uint32_t bytes = (((uint32_t)(rows - 1) * (uint32_t)p.row + (uint32_t)p.E) * size + 3u) & ~3u;
    const buf_rsrc_t from = buf_rsrc(reinterpret_cast<const uint8_t*>(p.logits) + t0 * p.row * size, bytes);
    const uint32_t at = ((uint32_t)(lane / LPR) * (uint32_t)p.row + (uint32_t)e0) * size;
    if (p.dtype == 0)
      load_floats<V>(from, at, x);
    else
      load_halves<V>(from, at, p.dtype, x);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) x[j] = j < n ? logit(p.logits, t * p.row + e0 + j, p.dtype) : 0.f;
  }
  double c[V];
  // inf and NaN make `odd` NaN; the largest magnitude decides the rest
  float odd = 0.f, most = 0.f;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    x[j] = j < n ? x[j] : 0.f;  // what lies behind the lane's experts
    b[j] = j < n ? b[j] : 0.f;
    odd = __builtin_fmaf(x[j], 0.f, odd);
    odd = __builtin_fmaf(b[j], 0.f, odd);
    most = fmaxf(most, fabsf(x[j]));
  }
  if (const uint64_t odd_lanes = __ballot(odd != 0.f || !(most < 700.f))) {
    // these rows by the whole wavefront, the others go on: a row takes the way of its own values
    constexpr uint64_t ROW = LPR == 64 ? ~0ull : (1ull << (LPR & 63)) - 1;
    int left = 0;
    for (int r = 0; r < ROWS && t0 + r < p.T; ++r) {
      if (odd_lanes >> (r * LPR) & ROW)
        route_row<LPR * V / 64>(p, t0 + r, own_lds);
      else
        ++left;
    }
    if (left == 0) return;
    wave_fence();  // the last of them may still be read
    if (odd_lanes >> base & ROW) {
      live = false;
      n = 0;
    }
  }
  float top = 0.f;
  double share = 1.0;
  if (p.softmax) {
    top = -__builtin_inff();
#pragma unroll
    for (int j = 0; j < V; ++j) top = j < n ? fmaxf(top, x[j]) : top;
#pragma unroll
    for (int d = 1; d < LPR; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
    double sum = 0.0;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      c[j] = exp64((double)x[j] - (double)top);
      sum += j < n ? c[j] : 0.0;
    }
    share = inverse(row_sum<LPR>(sum));
#pragma unroll
    for (int j = 0; j < V; ++j) c[j] *= share;
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) c[j] = unit(x[j], 0, 0.f, 1.0);
  }
#pragma unroll
  for (int j = 0; j < V; ++j) c[j] = j < n ? c[j] + (double)b[j] : -__builtin_inf();  // -inf: no expert

  double a[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) a[i] = c[i];
  sort8(a);
  if constexpr (V == 16) {
    double d[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) d[i] = c[8 + i];
    sort8(d);
    merge8(a, d);
  }
  bool keep = true;
  if (p.groups > 1) {
    // a group is `span` consecutive lanes
    double first = a[0], second = a[1];
    for (int d = 1; d < p.span; d = p.span_shift ? 2 * d : d + 1) {
      // a power of two: halves meet; otherwise every lane's own two go round
      const int from = p.span_shift ? lane ^ d : base + l / p.span * p.span + (l % p.span + d) % p.span;
      const double f = __shfl(p.span_shift ? first : a[0], from), g = __shfl(p.span_shift ? second : a[1], from);
      second = larger(smaller(first, f), larger(second, g));
      first = larger(first, f);
    }
    const double score = p.group_top == 2 ? first + second : first;
    const int own = l / p.span;
    int before = 0;
    for (int g = 0; g < p.groups; ++g) {
      const double s = __shfl(score, base + g * p.span);
      before += s > score || (s == score && g < own);
    }
    keep = before < p.top_groups && own < p.groups;
#pragma unroll
    for (int i = 0; i < 8; ++i) a[i] = keep ? a[i] : -__builtin_inf();
  }
  merge_lanes<1, LPR>(a);
  double kth = a[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) kth = p.k == i + 1 ? a[i] : kth;

  uint32_t above = 0, equal = 0;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    above |= c[j] > kth ? 1u << j : 0u;
    equal |= c[j] == kth ? 1u << j : 0u;
  }
  if (!keep || n == 0) above = equal = 0;
  const int mine = __popc(above) | __popc(equal) << 16;
  int upto = mine;
#pragma unroll
  for (int d = 1; d < LPR; d <<= 1) {
    const int o = __shfl_up(upto, d, LPR);
    if (l >= d) upto += o;
  }
  const int room = p.k - (__shfl(upto, base + LPR - 1) & 0xFFFF);  // for experts that equal the k-th
  const int equal_before = (upto - mine) >> 16;
  int at = ((upto - mine) & 0xFFFF) + min(equal_before, room);
  for (int drop = __popc(equal) - max(room - equal_before, 0); drop > 0; --drop) equal &= ~(0x80000000u >> __builtin_clz(equal));
  int* const list = reinterpret_cast<int*>(own_lds) + lane / LPR * 8;
  for (uint32_t sel = above | equal; sel; sel &= sel - 1) list[at++] = e0 + __builtin_ctz(sel);
  wave_fence();

  // lane j < k: the j-th of them; fewer lanes than eight a row do not exist
  const bool in = live && l < p.k;
  const int id = in ? list[l] : 0;
  const double s = in ? unit(logit(p.logits, t * p.row + id, p.dtype), p.softmax, top, share) : 0.0;
  const double ch = in && p.bias ? s + (double)p.bias[id] : s;
  int rank = 0;
  for (int j = 0; j < p.k; ++j) {
    const double o = __shfl(ch, base + j);
    rank += o > ch || (o == ch && j < l);
  }
  double sum = 1.0;
  if (p.renormalize) {
    sum = s;
    sum += other<1>(sum);
    sum += other<2>(sum);
    sum += other<4>(sum);
  }
  if (in) {
    p.weights[t * p.k + rank] = (float)(sum == 0.0 ? 0.0 : s / sum * p.scale);
    p.ids[t * p.k + rank] = id;
  }
}

constexpr int LANE_WAVES = 2;

// Lanes that own a row; 0: a whole wavefront does (route_rows).
int lanes_of_row(int64_t E, int64_t k, int64_t groups) {
  const int64_t lanes = E <= 64 ? 8 : E <= 256 ? 16 : E <= 512 ? 32 : 64, per = (E + lanes - 1) / lanes;
  return k <= 8 && (groups == 1 || (E / groups) % per == 0) ? (int)lanes : 0;
}

template <int LPR, int V>
tb_status launch_lanes_as(const char* fn, const Args& p, hipStream_t stream) {
  auto* const kernel = &route_lanes<LPR, V, LANE_WAVES>;
  constexpr int rows = 64 / LPR * LANE_WAVES;
  const size_t lds = (size_t)LANE_WAVES * 8 * (size_t)p.wave_words;
  if (tb_status st = tb::reserve_lds(reinterpret_cast<const void*>(kernel), lds, fn)) return st;
  hipLaunchKernelGGL(kernel, dim3((unsigned)((p.T + rows - 1) / rows)), dim3(64 * LANE_WAVES), lds, stream, p);
  return tb::launch_status(fn);
}

tb_status launch_lanes(const char* fn, const Args& p, int lpr, hipStream_t stream) {
  if (lpr == 8) return launch_lanes_as<8, 8>(fn, p, stream);
  if (lpr == 32) return launch_lanes_as<32, 16>(fn, p, stream);
  if (lpr == 64) return launch_lanes_as<64, 16>(fn, p, stream);
  return p.E <= 128 ? launch_lanes_as<16, 8>(fn, p, stream) : launch_lanes_as<16, 16>(fn, p, stream);
}

}  // namespace routing
}  // namespace tb

extern "C" tb_status tb_moe_expert_routing(const void* logits, const float* bias, float* weights, int32_t* ids, int64_t T,
                                           int64_t E, int64_t k, int64_t groups, int64_t top_groups, int64_t group_top,
                                           int64_t row, int softmax, int renormalize, double scale, int dtype,
                                           hipStream_t stream) {
  using namespace tb::routing;
  const char* const fn = "tb_moe_expert_routing";
  TB_CHECK_ARG(logits && weights && ids, "%s: null pointer", fn);
  TB_CHECK_ARG(T > 0 && E > 0 && E <= 1024, "%s: need rows and 1 to 1024 experts (got %lld and %lld)", fn, (long long)T,
               (long long)E);
  TB_CHECK_ARG(groups > 0 && groups <= 64 && E % groups == 0, "%s: need 1 to 64 groups of equal size (got %lld of %lld)",
               fn, (long long)groups, (long long)E);
  TB_CHECK_ARG(top_groups > 0 && top_groups <= groups, "%s: need 1 to %lld chosen groups (got %lld)", fn,
               (long long)groups, (long long)top_groups);
  TB_CHECK_ARG(group_top == 1 || (group_top == 2 && E / groups >= 2),
               "%s: a group's score is its one or two largest choices (got %lld of %lld)", fn, (long long)group_top,
               (long long)(E / groups));
  TB_CHECK_ARG(k > 0 && k <= 32 && k <= E / groups * top_groups, "%s: need 1 <= k <= 32 of the %lld experts left (got %lld)",
               fn, (long long)(E / groups * top_groups), (long long)k);
  TB_CHECK_ARG(row >= 0, "%s: negative stride", fn);
  TB_CHECK_ARG(dtype >= 0 && dtype <= 2, "%s: unknown type %d", fn, dtype);
  TB_CHECK_ALIGN(logits, dtype ? 2 : 4, "logits");
  Args p{logits, bias, weights, ids, T, row, scale, (int)E, (int)k, (int)groups, (int)top_groups, (int)group_top,
         softmax, renormalize, dtype};
  TB_CHECK_ARG(T < (1ll << 24), "%s: problem too large", fn);
  if (const int lpr = lanes_of_row(E, k, groups)) {
    const int size = dtype ? 2 : 4;
    p.per = (int)((E + lpr - 1) / lpr);
    p.span = (int)(E / groups) / p.per;
    p.span_shift = groups > 1 && (p.span & (p.span - 1)) == 0;
    // loads of 16 bytes need addresses on 4, and offsets within a wavefront's rows below 2^31
    p.vec = tb::aligned(logits, 4) && row * size % 4 == 0 && p.per * size % 4 == 0 && row < (1ll << 24);
    p.wave_words = (int)(2 * E > 64 / lpr * 4 ? 2 * E : 64 / lpr * 4);  // route_row's, or the lists of eight
    return launch_lanes(fn, p, lpr, stream);
  }
  const int64_t blocks = (T + WAVES - 1) / WAVES;
  const size_t lds = (size_t)WAVES * 2 * 8 * (size_t)E;
  auto* const kernel = E <= 64 ? &route_rows<1> : E <= 128 ? &route_rows<2> : E <= 256 ? &route_rows<4>
                       : E <= 512 ? &route_rows<8> : &route_rows<16>;
  if (tb_status st = tb::reserve_lds(reinterpret_cast<const void*>(kernel), lds, fn)) return st;
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(64 * WAVES), lds, stream, p);
  return tb::launch_status(fn);
}

extern "C" tb_status tb_moe_expert_routing_kernel(int64_t E, int64_t k, int64_t groups, const char** kernel, int32_t* lanes,
                                                  int32_t* threads) {
  using namespace tb::routing;
  const char* const fn = "tb_moe_expert_routing_kernel";
  TB_CHECK_ARG(kernel && lanes && threads, "%s: null output", fn);
  TB_CHECK_ARG(E > 0 && E <= 1024 && k > 0 && k <= 32 && groups > 0 && E % groups == 0, "%s: no routing has these sizes", fn);
  const int n = lanes_of_row(E, k, groups);
  *kernel = n ? "route_lanes" : "route_rows";
  *lanes = n ? n : 64;
  *threads = 64 * (n ? LANE_WAVES : WAVES);
  return TB_OK;
}
