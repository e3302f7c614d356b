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
// One wavefront a row: lane l holds experts l, 64 + l, ...; choices are compared as
// 64-bit keys in the order of their values (0: cannot be chosen).
#include "tb_common.h"

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
};

__device__ __forceinline__ float logit(const void* p, int64_t i, int dtype) {
  if (dtype == 0) return reinterpret_cast<const float*>(p)[i];
  const uint16_t v = reinterpret_cast<const uint16_t*>(p)[i];
  return dtype == 1 ? (float)__builtin_bit_cast(_Float16, v) : __builtin_bit_cast(float, (uint32_t)v << 16);
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

template <int V>
__global__ void __launch_bounds__(64 * WAVES) moe_routing_kernel(Args p) {
  extern __shared__ uint64_t lds[];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t t = (int64_t)blockIdx.x * WAVES + wave;
  if (t >= p.T) return;  // no barrier below: a row is one wavefront's
  double* const ls = reinterpret_cast<double*>(lds) + wave * 2 * p.E;
  uint64_t* const lk = lds + wave * 2 * p.E + p.E;

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
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int e = 64 * j + lane;
    key[j] = e < p.E ? key_of(p.bias ? s[j] + (double)p.bias[e] : s[j]) : 0;
    if (e < p.E) ls[e] = s[j], lk[e] = key[j];
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // the other lanes' parts of the row's LDS
  __builtin_amdgcn_wave_barrier();

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
  const int64_t blocks = (T + WAVES - 1) / WAVES;
  TB_CHECK_ARG(blocks < (1ll << 23), "%s: problem too large", fn);
  const Args p{logits, bias, weights, ids, T, row, scale, (int)E, (int)k, (int)groups, (int)top_groups, (int)group_top,
               softmax, renormalize, dtype};
  const size_t lds = (size_t)WAVES * 2 * 8 * (size_t)E;
  auto* const kernel = E <= 64 ? &moe_routing_kernel<1> : E <= 128 ? &moe_routing_kernel<2> : E <= 256 ? &moe_routing_kernel<4>
                       : E <= 512 ? &moe_routing_kernel<8> : &moe_routing_kernel<16>;
  if (tb_status st = tb::reserve_lds(reinterpret_cast<const void*>(kernel), lds, fn)) return st;
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(64 * WAVES), lds, stream, p);
  return tb::launch_status(fn);
}
