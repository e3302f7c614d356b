// Products of MXFP4 matrices: Y = T(sum_k a[m, k] * w[n, k]), dense (tb_mxfp4_gemm)
// and over rows sorted by expert (tb_moe_mxfp4_grouped_gemm).
//
// Both operands are e2m1 codes, two a byte, K contiguous, with one power of two for
// 32 channels (mxfp4.hip).  v_mfma_scale_f32_32x32x64_f8f6f4 takes them as they are:
// lane (r = lane % 32, h = lane / 32) gives row r's channels 32 h .. 32 h + 31 of the
// 64, which are 16 bytes of codes and one block, and one byte of its scale register
// is that block's scale.  Products and their sums within a block need few bits, so
// the fp32 accumulators round only where blocks of very different scales meet.
//
// K advances in steps of 128 bytes a row, 256 channels or 8 blocks.  Past the end of
// K a step's scales are cleared in both operands: the products are then at most 36 *
// 2^-254, nothing in fp32, whatever the codes there are (every code is finite).  The
// transposed product (W first) leaves a lane four consecutive columns of one row.
//
// Rows: expert e has the rows offsets[e] .. offsets[e + 1] - 1; the host knows only
// their total, so the grid is an upper bound and every block looks its expert up.
// Offsets and row numbers are held to their ranges on the device.
#include "gemm_tile.h"
#include "small_plan.h"
#include "tb_common.h"

#include <type_traits>

namespace tb {
namespace ntg {
namespace mx {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x2v __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2v __attribute__((ext_vector_type(2)));

constexpr int STEP = 128;       // bytes of codes of a row and step
constexpr int STEP_BLOCKS = 8;  // its scales
constexpr uint32_t RSRC_DW3 = 0x00020000u;

struct Args {
  const uint8_t *a, *sa, *w, *sw;
  uint16_t* y;
  const int *offsets, *gather, *scatter;  // grouped
  const float* weights;
  int64_t sw_expert;                      // bytes between experts' scales
  int M, N, K, E, a_rows;
  int sa_row, sw_row;                     // bytes between rows of scales
  int tiles_m, tiles_n;                   // grouped: tiles_m is the upper bound
  int bf16, vec;                          // output type; rows of Y start on 16 bytes
  Divisor by_topk, by_tiles_n, by_band;   // of tiles_n and of 8 tiles_n
};

// A tile: expert, first row, rows, first column.
struct Place {
  int e, m0, rows, n0;
};

// Block b's share of n consecutive blocks, runs of them on one XCD.
__device__ __forceinline__ int xcd_run(int b, int n) {
  const int x = b & 7, q = n >> 3, rem = n & 7;
  return x * q + min(x, rem) + (b >> 3);
}

// v plus those of the lanes before (DPP: by 1, 2, 4 and 8 within rows of 16, then the rows' last lanes go on).
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, true);
  return v;
}

// A run of row tiles: expert, its rows, the tiles before it and its own.
struct Run {
  int e, begin, end, before, tiles;
};

// Rows lo .. hi - 1 of lane's expert of the 64 from b on, and their tiles.
__device__ __forceinline__ int tiles_of(const Args& p, int b, int shift, int& lo, int& hi) {
  const int i = b + (threadIdx.x & 63);
  lo = i < p.E ? min(max(p.offsets[i], 0), p.M) : 0;
  hi = i < p.E ? min(max(p.offsets[i + 1], 0), p.M) : 0;
  return hi > lo ? ((hi - lo - 1) >> shift) + 1 : 0;
}

// The tile of this block.  Runs of consecutive tiles go to one XCD and walk 8 row tiles (of an expert), then the next
// columns, so that a run's operands stay in its L2.  Grouped: every wavefront counts the tiles of all experts, 64 at a
// time, since runs have to share out the tiles there are, not the grid, which is an upper bound (64 experts of 512 rows,
// N = 2816, K = 4096: 264 us, with runs of the grid, where the last XCDs find nothing, 396).
template <bool GROUPED, int TM, int TN>
__device__ __forceinline__ bool place(const Args& p, Place& at) {
  int idx;
  Run run{0, 0, p.M, 0, p.tiles_m};
  if constexpr (GROUPED) {
    constexpr int SHIFT = TM == 32 ? 5 : TM == 64 ? 6 : TM == 128 ? 7 : 8;
    static_assert(TM == 1 << SHIFT, "rows of a tile");
    int lo, hi, total = 0, own = 0, upto = 0;
    for (int b = 0; b < p.E; b += 64) {
      own = tiles_of(p, b, SHIFT, lo, hi);
      upto = wave_scan(own);
      total = min(total + __builtin_amdgcn_readlane(upto, 63), p.tiles_m);  // more only if segments overlap
    }
    if ((int)blockIdx.x >= total * p.tiles_n) return false;
    idx = xcd_run(blockIdx.x, total * p.tiles_n);
    const int tile = p.by_tiles_n.divide(idx);
    int before = 0;
    uint64_t past = 0;
    for (int b = 0; b < p.E; b += 64) {
      if (p.E > 64) {
        own = tiles_of(p, b, SHIFT, lo, hi);
        upto = wave_scan(own);
      }
      past = __ballot(tile < before + upto);
      run.e = b;
      if (past) break;
      before += __builtin_amdgcn_readlane(upto, 63);
    }
    const int src = __builtin_ctzll(past | 1ull << 63);
    run.e += src;
    run.begin = __builtin_amdgcn_readlane(lo, src);
    run.end = __builtin_amdgcn_readlane(hi, src);
    run.tiles = __builtin_amdgcn_readlane(own, src);
    run.before = before + __builtin_amdgcn_readlane(upto, src) - run.tiles;
    idx -= run.before * p.tiles_n;
  } else {
    idx = xcd_run(blockIdx.x, gridDim.x);
  }
  const int band = p.by_band.divide(idx), in = idx - band * 8 * p.tiles_n;
  const int rows = min(run.tiles - band * 8, 8), col = rows == 8 ? in >> 3 : in / rows;
  at.e = run.e;
  at.m0 = run.begin + (band * 8 + in - col * rows) * TM;
  at.rows = min(TM, run.end - at.m0);
  at.n0 = col * TN;
  return true;
}

// Row of A of product row m (-1: none).
__device__ __forceinline__ int row_of_a(const Args& p, int m) {
  const int g = p.gather[m];
  const int row = g < 0 ? -1 : p.by_topk.divide(g);
  return row < p.a_rows ? row : -1;
}

__device__ __forceinline__ i32x4 rsrc4(const void* p, uint32_t bytes) {
  const uint64_t base = (uint64_t)(uintptr_t)p;
  i32x4 r;
  r[0] = __builtin_amdgcn_readfirstlane((int)(uint32_t)base);
  r[1] = __builtin_amdgcn_readfirstlane((int)(uint32_t)(base >> 32) & 0xFFFF);
  r[2] = __builtin_amdgcn_readfirstlane((int)bytes);
  r[3] = (int)RSRC_DW3;
  return r;
}

// Bytes of `rows` rows of K / 32 scales, up to the end of the last 4 (a load of 4 that ends past the last scale must
// still be made; it stays within 4 aligned bytes that hold one).
__device__ __forceinline__ uint32_t scale_bytes(int rows, int stride, int K) {
  return ((uint32_t)(rows - 1) * (uint32_t)stride + (uint32_t)(K / 32) + 3u) & ~3u;
}

// The operands of a tile: bases, sizes of buffers, and the offset of an A row.
struct Operands {
  const uint8_t *a, *sa, *w, *sw;
  uint32_t a_bytes, sa_bytes, w_bytes, sw_bytes;
};

template <bool GROUPED>
__device__ __forceinline__ Operands operands(const Args& p, const Place& at, int tn) {
  const int K2 = p.K / 2, cols = min(tn, p.N - at.n0);
  Operands o;
  const bool whole = GROUPED && p.gather;  // rows from all over A: below 2 GiB, the host has checked
  const int first = whole ? 0 : at.m0, rows = whole ? p.a_rows : at.rows;
  o.a = p.a + (int64_t)first * K2;
  o.sa = p.sa + (int64_t)first * p.sa_row;
  o.a_bytes = (uint32_t)rows * (uint32_t)K2;
  o.sa_bytes = scale_bytes(rows, p.sa_row, p.K);
  o.w = p.w + ((int64_t)at.e * p.N + at.n0) * K2;
  o.sw = p.sw + at.e * p.sw_expert + (int64_t)at.n0 * p.sw_row;
  o.w_bytes = (uint32_t)cols * (uint32_t)K2;
  o.sw_bytes = scale_bytes(cols, p.sw_row, p.K);
  return o;
}

// Row of the buffer of A that holds row i of the tile (-1: none).
template <bool GROUPED>
__device__ __forceinline__ int buffer_row(const Args& p, const Place& at, int i) {
  if (i >= at.rows) return -1;
  if constexpr (GROUPED)
    if (p.gather) return row_of_a(p, at.m0 + i);
  return i;
}

// Row of Y of the tile's row i (-1: none), and the factor of that row.
template <bool GROUPED>
__device__ __forceinline__ int row_of_y(const Args& p, const Place& at, int i) {
  if (i >= at.rows) return -1;
  const int m = at.m0 + i;
  if constexpr (GROUPED)
    if (p.scatter) {
      const int y = p.scatter[m];
      return (unsigned)y < (unsigned)p.M ? y : -1;
    }
  return m;
}

__device__ __forceinline__ uint32_t pack2(float a, float b, int bf16) {
  if (bf16) return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2v{a, b}), bf16x2v));
  return as_u32(f16x2{(_Float16)a, (_Float16)b});
}

// Bytes 2 s + h, s = 0 .. 3, of a step's eight scales: substep s takes byte s.
__device__ __forceinline__ uint32_t pick_scales(const u32x2& v, int h) { return perm(v[1], v[0], h ? 0x07050301u : 0x06040200u); }

// ... those of the last step that K reaches; the others cleared.
__device__ __forceinline__ uint32_t tail_mask(int K, int h) {
  const int left = K / 32 - (K / 32 - 1) / STEP_BLOCKS * STEP_BLOCKS;
  uint32_t m = 0;
#pragma unroll
  for (int s = 0; s < 4; ++s) m |= 2 * s + h < left ? 0xFFu << (8 * s) : 0u;
  return m;
}

template <int S>
__device__ __forceinline__ f32x16 mfma(const i32x4& w, const i32x4& a, const f32x16& c, uint32_t sw, uint32_t sa) {
  const i32x8 w8 = __builtin_shufflevector(w, w, 0, 1, 2, 3, -1, -1, -1, -1);
  const i32x8 a8 = __builtin_shufflevector(a, a, 0, 1, 2, 3, -1, -1, -1, -1);
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w8, a8, c, 4, 4, S, (int)sw, S, (int)sa);
}

// ------------------------------------------------------------------ few rows
// Up to 32 rows are bound by reading the weights once.  A block owns 32 rows x 32
// columns and its KS wavefronts split K; each loads its fragments straight into
// registers, D steps ahead, with no LDS and no barrier in the loop.  A load instruction
// covers 32 bytes of 32 rows, the four of a step one 128-byte line each.  The partial
// sums are added in wavefront order, so results are reproducible bit for bit.
// 1 x 4096 x 4096: 5.6 us with its launch, a chain of load, products and join (8.9 MB, 1.4 us of HBM).
constexpr int SK_N = 32, SK_ROW = SK_N + 4;

template <int KS, int D, bool GROUPED>
__global__ void __launch_bounds__(64 * KS, KS / 4) mx_skinny(Args p) {
  __shared__ __attribute__((aligned(16))) float part[KS][32 * SK_ROW];
  Place at;
  if (!place<GROUPED, 32, SK_N>(p, at)) return;
  const int t = threadIdx.x, lane = t & 63, r = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int K2 = p.K / 2, nk = (K2 + STEP - 1) / STEP;
  const int k0 = (int)((int64_t)nk * wave / KS), k1 = (int)((int64_t)nk * (wave + 1) / KS);
  const Operands o = operands<GROUPED>(p, at, SK_N);
  const buf_rsrc_t ra = buf_rsrc(o.a, o.a_bytes), rsa = buf_rsrc(o.sa, o.sa_bytes);
  const buf_rsrc_t rw = buf_rsrc(o.w, o.w_bytes), rsw = buf_rsrc(o.sw, o.sw_bytes);
  const int arow = buffer_row<GROUPED>(p, at, r);
  const bool col = at.n0 + r < p.N;
  const uint32_t a_off = arow >= 0 ? (uint32_t)arow * (uint32_t)K2 + 16u * h : BUF_OOB;
  const uint32_t sa_off = arow >= 0 ? (uint32_t)arow * (uint32_t)p.sa_row : BUF_OOB;
  const uint32_t w_off = col ? (uint32_t)r * (uint32_t)K2 + 16u * h : BUF_OOB;
  const uint32_t sw_off = col ? (uint32_t)r * (uint32_t)p.sw_row : BUF_OOB;
  const uint32_t tail = tail_mask(p.K, h);

  struct Frag {
    i32x4 w[4], a[4];
    u32x2 sw, sa;
  };
  auto load = [&](Frag& f, int k) __attribute__((always_inline)) {
    const bool live = k < k1;  // uniform: past the wavefront's steps nothing is read
    const uint32_t soff = (uint32_t)(live ? k : 0) * STEP, ssoff = (uint32_t)(live ? k : 0) * STEP_BLOCKS;
    const uint32_t wo = live ? w_off : BUF_OOB, ao = live ? a_off : BUF_OOB;
#pragma unroll
    for (int s = 0; s < 4; ++s)
      f.w[s] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(rw, wo + 32u * s, soff, 0));
    f.sw = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(rsw, live ? sw_off : BUF_OOB, ssoff, 0));
#pragma unroll
    for (int s = 0; s < 4; ++s)
      f.a[s] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(ra, ao + 32u * s, soff, 0));
    f.sa = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(rsa, live ? sa_off : BUF_OOB, ssoff, 0));
  };
  f32x16 acc = f32x16{};
  auto mma = [&](const Frag& f, int k) __attribute__((always_inline)) {
    const uint32_t keep = k == nk - 1 ? tail : ~0u;
    const uint32_t sw = pick_scales(f.sw, h) & keep, sa = pick_scales(f.sa, h) & keep;
    acc = mfma<0>(f.w[0], f.a[0], acc, sw, sa);
    acc = mfma<1>(f.w[1], f.a[1], acc, sw, sa);
    acc = mfma<2>(f.w[2], f.a[2], acc, sw, sa);
    acc = mfma<3>(f.w[3], f.a[3], acc, sw, sa);
  };
  Frag f[D];
#pragma unroll
  for (int d = 0; d < D; ++d) load(f[d], k0 + d);
  for (int k = k0; k < k1; k += D) {
#pragma unroll
    for (int d = 0; d < D; ++d) {
      if (d > 0 && k + d >= k1) break;  // uniform
      mma(f[d], k + d);
      __builtin_amdgcn_sched_barrier(0);
      load(f[d], k + d + D);
      __builtin_amdgcn_sched_barrier(0);
    }
  }

  // element 4 g + e: row r, column 8 g + 4 h + e of the tile
#pragma unroll
  for (int g = 0; g < 4; ++g)
    *reinterpret_cast<f32x4*>(&part[wave][r * SK_ROW + 8 * g + 4 * h]) =
        f32x4{acc[4 * g], acc[4 * g + 1], acc[4 * g + 2], acc[4 * g + 3]};
  __syncthreads();
  for (int q = t; q < 32 * (SK_N / 4); q += 64 * KS) {
    const int row = q / (SK_N / 4), c = q % (SK_N / 4) * 4, n = at.n0 + c;
    const int yrow = row_of_y<GROUPED>(p, at, row);
    if (yrow < 0 || n >= p.N) continue;
    f32x4 v = *reinterpret_cast<const f32x4*>(&part[0][row * SK_ROW + c]);
#pragma unroll
    for (int w = 1; w < KS; ++w) {
      const f32x4 u = *reinterpret_cast<const f32x4*>(&part[w][row * SK_ROW + c]);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += u[e];
    }
    if constexpr (GROUPED) {
      const float s = p.weights ? p.weights[yrow] : 1.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] *= s;
    }
    u32x2 out;
    out[0] = pack2(v[0], v[1], p.bf16);
    out[1] = pack2(v[2], v[3], p.bf16);
    uint16_t* const y = p.y + (int64_t)yrow * p.N + n;
    if (p.vec) {  // N % 8 == 0: four columns are all in or all out
      *reinterpret_cast<u32x2*>(y) = out;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n + e < p.N) y[e] = (uint16_t)(out[e / 2] >> (16 * (e & 1)));
    }
  }
}

// ------------------------------------------------------------------ tiles
// One tile per block: NW wavefronts, WM x NW / WM, of FI x FJ fragments of 32 x 32.  256 x 256 takes eight (but for long
// K), so that one of a SIMD's two works while the other waits at a barrier, for its reads or for its stores (4096 tokens
// through 64 experts' down: 222 us, four of 4 x 4 fragments 237).  8192 x 8192 x 8192: 270 us, 4.1 PFLOP/s; its matrix
// instructions alone, in this order, 190 (the card then holds 1.8 GHz), without the DMAs 232, without fragment reads 268.
// Both operands and their scales stream HBM -> LDS by DMA.  Codes: ST stages of one step, rows of 128 bytes, 16-byte chunk
// c of row i at slot c ^ ((i ^ (i >> 3)) & 7), so that their writes and fragment reads are free of conflicts (rows of 64 bytes
// and twice the stages: 1.3 to 1.4 times slower, a DMA then takes 16 lines for its KiB instead of 8).  Rows of scales lie one
// after the other: 32 of them 8 CS bytes apart conflict (cycles of it an LDS instruction of any kind: CS = 8 2.9, 4 1.2, 2 0.4).
// Scales: two buffers of CS steps, 8 CS bytes of a row at once, since a load of a row's 8 bytes takes a whole line's time
// and, from HBM, a whole line.  A step is four substeps of one MFMA per fragment pair.  While a substep's MFMAs run, the
// next one's fragments are read (one ds_read_b128 each); the barrier sits before the last substep, when every wavefront
// has read the stage: it then takes the DMAs of the step ST later.
template <int FI_, int FJ_, int ST_, int CS_, int WM_ = 2, int NW_ = 4>
struct Tile {
  static constexpr int FI = FI_, FJ = FJ_, ST = ST_, CS = CS_, WM = WM_, NW = NW_;
  static constexpr int TM = 32 * FI * WM, TN = 32 * FJ * (NW / WM);
  static constexpr int A_ST = TM * STEP, STAGE = (TM + TN) * STEP;     // A rows, then W rows
  static constexpr int SROW = CS * STEP_BLOCKS, SC = (TM + TN) * SROW, SC_OFF = ST * STAGE;
  static constexpr int NS = SC / 1024, DS = (NS + NW - 1) / NW;   // scale DMAs of a buffer, of a wavefront
  static constexpr int PAD_OFF = SC_OFF + 2 * SC;                      // those of wavefronts that have none land here
  static constexpr int LDS_BYTES = PAD_OFF + (NS % NW ? 1024 : 0);
  static_assert(LDS_BYTES <= 160 * 1024 && SC % 1024 == 0 && TM * SROW % 1024 == 0, "LDS layout");
  // A buffer of scales goes out after the wait of step k, k % CS == 0, and is read after that of step k + CS - 1, which leaves
  // a stage's DMAs ST - 2 times under way: those of CS - 1 stages were issued behind the scales.
  static_assert(CS >= 2 && CS >= ST - 1, "scales have to have landed when they are read");
};

// The tile at `at`, or with half of C's FI the first half of its rows.
template <class C, int FI, bool GROUPED>
__device__ __forceinline__ void tile_product(const Args& p, const Place& at, uint8_t* lds) {
  constexpr int FJ = C::FJ, ST = C::ST, CS = C::CS, WN = C::NW / C::WM;
  const int t = threadIdx.x, lane = t & 63, r = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6), wm = wave / WN, wn = wave % WN;
  const int K2 = p.K / 2, nk = (K2 + STEP - 1) / STEP;
  const Operands o = operands<GROUPED>(p, at, C::TN);
  const i32x4 ra = rsrc4(o.a, o.a_bytes), rw = rsrc4(o.w, o.w_bytes);
  const i32x4 rsa = rsrc4(o.sa, o.sa_bytes), rsw = rsrc4(o.sw, o.sw_bytes);
  const uint32_t lds0 = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(uintptr_t)(
      __attribute__((address_space(3))) void*)lds);
  auto live_rsrc = [](bool live, i32x4 v) __attribute__((always_inline)) {
    v[2] = __builtin_amdgcn_readfirstlane(live ? v[2] : 0);
    return v;
  };

  // A wavefront's DMAs: of a step 8 A rows each (lane L: row + L / 8, slot L % 8), then 8 W rows each; of a scale
  // buffer 16 bytes a lane, SROW / 16 lanes a row.
  constexpr int DA = C::TM / (8 * C::NW), DW = C::TN / (8 * C::NW), PER = DA + DW, DS = C::DS, SL = C::SROW / 16;
  uint32_t off[PER], soff[DS];
#pragma unroll
  for (int d = 0; d < PER; ++d) {
    const int row = 8 * (d < DA ? DA * wave + d : DW * wave + d - DA) + (lane >> 3);
    const uint32_t c = (uint32_t)((lane & 7) ^ ((row ^ (row >> 3)) & 7)) * 16u;
    const int at_row = d < DA ? buffer_row<GROUPED>(p, at, row) : at.n0 + row < p.N ? row : -1;
    off[d] = at_row >= 0 ? (uint32_t)at_row * (uint32_t)K2 + c : BUF_OOB;
  }
#pragma unroll
  for (int d = 0; d < DS; ++d) {
    const int q = wave + C::NW * d, row = 64 / SL * q + lane / SL, wrow = row - C::TM;
    const int at_row = q >= C::NS ? -1 : row < C::TM ? buffer_row<GROUPED>(p, at, row) : at.n0 + wrow < p.N ? wrow : -1;
    soff[d] = at_row >= 0 ? (uint32_t)at_row * (uint32_t)(row < C::TM ? p.sa_row : p.sw_row) + 16u * (lane % SL) : BUF_OOB;
  }
  // past the last step: empty buffers (zeros, no traffic)
  auto issue_one = [&](int k, int st, int d) __attribute__((always_inline)) {
    const bool live = k < nk;
    const uint32_t dst = lds0 + (uint32_t)(st * C::STAGE), from = (uint32_t)(live ? k : 0) * STEP;
    if (d < DA)
      dma16(dst + (uint32_t)((DA * wave + d) * 1024), off[d], live_rsrc(live, ra), from);
    else
      dma16(dst + (uint32_t)(C::A_ST + (DW * wave + d - DA) * 1024), off[d], live_rsrc(live, rw), from);
  };
  auto issue_scales = [&](int buffer, int d) __attribute__((always_inline)) {  // of the steps from CS * buffer on
    const bool live = buffer * CS < nk;
    const int q = wave + C::NW * d;
    dma16(lds0 + (uint32_t)(q < C::NS ? C::SC_OFF + (buffer & 1) * C::SC + q * 1024 : C::PAD_OFF), soff[d],
          live_rsrc(live, q * (64 / SL) < C::TM ? rsa : rsw), (uint32_t)(live ? buffer : 0) * C::SROW);
  };

  // fragment f (f < FI: A rows 32 (FI wm + f) .., then W rows 32 (FJ wn + f - FI) ..) of substep s: chunk 2 s + h of
  // the lane's row; a substep flips bits 5 and 6 of the address
  typedef __attribute__((address_space(3))) uint8_t lds_u8;
  constexpr int NFR = FI + FJ;
  uint32_t base[NFR], sbase[NFR];
#pragma unroll
  for (int f = 0; f < NFR; ++f) {
    const int row = 32 * (f < FI ? FI * wm + f : FJ * wn + f - FI) + r;
    base[f] = lds0 + (uint32_t)((f < FI ? 0 : C::A_ST) + row * STEP + ((h ^ ((row ^ (row >> 3)) & 7)) << 4));
    sbase[f] = lds0 + (uint32_t)(C::SC_OFF + ((f < FI ? 0 : C::TM) + row) * C::SROW);
  }
  struct Frag {
    i32x4 v[NFR];
  };
  auto read_one = [&](Frag& fr, int st, int s, int f) __attribute__((always_inline)) {
    typedef __attribute__((address_space(3))) const i32x4 lds_i4;
    fr.v[f] = *(lds_i4*)((lds_u8*)(uintptr_t)(base[f] ^ (uint32_t)(s << 5)) + st * C::STAGE);
  };
  const uint32_t tail = tail_mask(p.K, h);
  // the scales read beside a step's last substep are picked apart when the next one starts: there the wait for them is
  // the fragments' too
  u32x2 raw[NFR];
  uint32_t sc[NFR];
  auto read_scale = [&](int k, int f) __attribute__((always_inline)) {
    typedef __attribute__((address_space(3))) const u32x2 lds_u2;
    const uint32_t at_step = (uint32_t)(((k / CS) & 1) * C::SC + k % CS * STEP_BLOCKS);
    raw[f] = *(lds_u2*)((lds_u8*)(uintptr_t)(sbase[f] + at_step));
  };

  f32x16 acc[FI][FJ];
#pragma unroll
  for (int i = 0; i < FI; ++i)
#pragma unroll
    for (int j = 0; j < FJ; ++j) acc[i][j] = f32x16{};

  // Codes of step k + 1 have landed when those of the ST - 2 steps behind are all that is outstanding; scales among them
  // only make the wait longer (that they have landed themselves is Tile's assertion).
  // DMAs of a step that go out beside the last substep; the others beside the next one's first (8192 x 8192 x 8192 on eight
  // wavefronts: a quarter 265 us, half 269, three quarters 278)
  constexpr int NOW = C::NW == 8 ? PER / 4 : PER / 2;
  constexpr int VM0 = PER * (ST - 2) + NOW, VM1 = PER * (ST - 2);
  static_assert(VM0 < 64, "vmcnt range");
  constexpr int WAIT_PRO = (VM0 & 15) | ((VM0 >> 4) << 14) | (7 << 4) | (15 << 8);
  constexpr int WAIT_STEP = (VM1 & 15) | ((VM1 >> 4) << 14) | (7 << 4) | (0 << 8);
  auto barrier = [&]() __attribute__((always_inline)) {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
#pragma unroll
  for (int d = 0; d < DS; ++d) issue_scales(0, d);
#pragma unroll
  for (int st = 0; st < ST; ++st)
#pragma unroll
    for (int d = 0; d < (st < ST - 1 ? PER : NOW); ++d) issue_one(st, st, d);
  // Thread i holds the tile's row i: where it goes, and its factor.  The loads come after the DMAs (the wait for the first
  // is theirs too), the factor arrives during the steps.
  int yrow = -1;
  float factor = 1.f;
  if constexpr (GROUPED) {
    if (t < C::TM) yrow = row_of_y<GROUPED>(p, at, t);
    if (p.weights && yrow >= 0) factor = p.weights[yrow];
  }
  __builtin_amdgcn_s_waitcnt(WAIT_PRO);
  barrier();
  Frag f0, f1;
#pragma unroll
  for (int f = 0; f < NFR; ++f) {
    read_one(f0, 0, 0, f);
    read_scale(0, f);
  }

  constexpr int NQ = FI * FJ;  // MFMAs of a substep
  // Substep s of step k on stage st; beside its q-th MFMA go out the reads of the next substep's fragments, and DMAs
  auto substep = [&](auto sub, int k, int st, const Frag& cur, Frag& other) __attribute__((always_inline)) {
    constexpr int S = decltype(sub)::value;
    const int next = (st + 1) % ST;
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
      const int i = q / FJ, j = q % FJ;
      acc[i][j] = mfma<S>(cur.v[FI + j], cur.v[i], acc[i][j], sc[FI + j], sc[i]);
#pragma unroll
      for (int f = 0; f < NFR; ++f)
        if (f * NQ / NFR == q) {
          if constexpr (S < 3) {
            read_one(other, st, S + 1, f);
          } else {
            read_one(other, next, 0, f);
            read_scale(k + 1, f);
          }
        }
      if constexpr (S == 3) {
#pragma unroll
        for (int d = 0; d < NOW; ++d)
          if (d * NQ / NOW == q) issue_one(k + ST, st, d);
      }
      if constexpr (S == 0) {
#pragma unroll
        for (int d = NOW; d < PER; ++d)
          if ((d - NOW) * NQ / (PER - NOW) == q) issue_one(k + ST - 1, (st + ST - 1) % ST, d);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  auto step = [&](int k, int st) __attribute__((always_inline)) {
#pragma unroll
    for (int f = 0; f < NFR; ++f) sc[f] = pick_scales(raw[f], h) & (k == nk - 1 ? tail : ~0u);
    substep(std::integral_constant<int, 0>{}, k, st, f0, f1);
    substep(std::integral_constant<int, 1>{}, k, st, f1, f0);
    substep(std::integral_constant<int, 2>{}, k, st, f0, f1);
    // step k + 1 landed, and every wavefront has read this stage, and the scales of the steps before
    __builtin_amdgcn_s_waitcnt(WAIT_STEP);
    barrier();
    if (k % CS == 0) {
#pragma unroll
      for (int d = 0; d < DS; ++d) issue_scales(k / CS + 1, d);
    }
    substep(std::integral_constant<int, 3>{}, k, st, f1, f0);
  };
  for (int k = 0; k < nk; k += ST) {
#pragma unroll
    for (int st = 0; st < ST; ++st)
      if (k + st < nk) step(k + st, st);
  }
  // grouped: the rows of Y and their factors, where the first stage was
  int* const map = reinterpret_cast<int*>(lds);
  float* const factors = reinterpret_cast<float*>(lds + C::TM * 4);
  __builtin_amdgcn_s_waitcnt(0);  // the DMAs issued past the end
  if constexpr (GROUPED) {
    __syncthreads();
    if (t < C::TM) {
      map[t] = yrow;
      factors[t] = factor;
    }
    __syncthreads();
  }

  // element 4 g + e of fragment (i, j): row 32 (FI wm + i) + r, column 32 (FJ wn + j) + 8 g + 4 h + e.  The halves of the
  // wavefront swap groups g and g + 1, after which a lane holds eight consecutive columns: 32 bytes of a row a store.
#pragma unroll
  for (int i = 0; i < FI; ++i) {
    const int row = 32 * (FI * wm + i) + r;
    const float s = GROUPED ? factors[row] : 1.f;
    const int to = GROUPED ? map[row] : row < at.rows ? at.m0 + row : -1;
    uint16_t* const y = p.y + (int64_t)to * p.N + at.n0;
#pragma unroll
    for (int j = 0; j < FJ; ++j)
#pragma unroll
      for (int g = 0; g < 4; g += 2) {
        uint32_t v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float a0 = acc[i][j][4 * g + 2 * e], a1 = acc[i][j][4 * g + 2 * e + 1];
          v[e] = GROUPED ? pack2(a0 * s, a1 * s, p.bf16) : pack2(a0, a1, p.bf16);
        }
        typedef uint32_t u2 __attribute__((ext_vector_type(2)));
        const u2 lo = __builtin_amdgcn_permlane32_swap(v[0], v[2], false, false);
        const u2 hi = __builtin_amdgcn_permlane32_swap(v[1], v[3], false, false);
        const int col = 32 * (FJ * wn + j) + 8 * (g + h), n = at.n0 + col;
        if (to < 0 || n >= p.N) continue;
        const u32x4 out = {lo[0], hi[0], lo[1], hi[1]};
        if (p.vec) {
          *reinterpret_cast<u32x4*>(y + col) = out;
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (n + e < p.N) y[col + e] = (uint16_t)(out[e / 2] >> (16 * (e & 1)));
        }
      }
  }
}

template <int FI, int FJ, int ST, int CS, int WM, bool GROUPED, int NW>
__global__ void __launch_bounds__(64 * NW, NW / 4) mx_tile(Args p) {
  typedef Tile<FI, FJ, ST, CS, WM, NW> C;
  extern __shared__ __attribute__((aligned(128))) uint8_t lds[];
  Place at;
  if (!place<GROUPED, C::TM, C::TN>(p, at)) return;
  if constexpr (GROUPED && FI == 4) {
    if (at.rows <= C::TM / 2) {
      tile_product<C, FI / 2, GROUPED>(p, at, lds);
      return;
    }
  }
  tile_product<C, FI, GROUPED>(p, at, lds);
}

constexpr int SKINNY_KS = 4, SKINNY_D = 1;  // 8 wavefronts or two steps ahead: 2 to 10 % slower

// Row tiles of TM rows: exact for a dense product, an upper bound for a grouped one.
inline int64_t row_tiles(int64_t M, int64_t tm, int64_t E) { return E ? M / tm + (E < M ? E : M) : (M + tm - 1) / tm; }

// f(shape) of a tile in LDS: launch and describe take the same one.
template <bool GROUPED, class F>
tb_status with_tile(plan::MxTile tile, const F& f) {
  if constexpr (GROUPED)
    if (tile == plan::MX_32x128) return f(Tile<1, 1, 3, 4, 1>{});
  switch (tile) {
    case plan::MX_64x64: return f(Tile<1, 1, 4, 8>{});
    case plan::MX_128x128: return f(Tile<2, 2, 2, 2>{});
    case plan::MX_256x128: return f(Tile<2, 2, 3, 2, 4, 8>{});
    case plan::MX_128_DEEP: return f(Tile<2, 2, 4, 4>{});
    case plan::MX_256_LONG:
      if constexpr (!GROUPED) return f(Tile<4, 4, 2, 2>{});
      [[fallthrough]];
    default: return f(Tile<4, 2, 2, 2, 2, 8>{});
  }
}

template <bool GROUPED, class K>
tb_status launch_kernel(const char* fn, K kernel, int tm, int tn, int threads, size_t lds, Args& p, hipStream_t stream) {
  const int64_t tiles_m = row_tiles(p.M, tm, GROUPED ? p.E : 0), tiles_n = (p.N + tn - 1) / tn;
  TB_CHECK_ARG(tiles_m * tiles_n < (1ll << 23), "%s: problem too large", fn);
  p.tiles_m = (int)tiles_m;
  p.tiles_n = (int)tiles_n;
  p.by_tiles_n = tb::Divisor((uint32_t)tiles_n);
  p.by_band = tb::Divisor((uint32_t)tiles_n * 8);
  if (lds)
    if (tb_status st = tb::reserve_lds(reinterpret_cast<const void*>(kernel), lds, fn)) return st;
  hipLaunchKernelGGL(kernel, dim3((unsigned)(tiles_m * tiles_n)), dim3(threads), lds, stream, p);
  return tb::launch_status(fn);
}

template <bool GROUPED>
tb_status launch(const char* fn, Args& p, hipStream_t stream) {
  const plan::MxTile tile = plan::pick_mx_tile(p.M, p.N, p.K, GROUPED ? p.E : 0);
  if (tile == plan::MX_32x32)
    return launch_kernel<GROUPED>(fn, &mx_skinny<SKINNY_KS, SKINNY_D, GROUPED>, 32, SK_N, 64 * SKINNY_KS, 0, p, stream);
  return with_tile<GROUPED>(tile, [&](auto shape) {
    typedef decltype(shape) C;
    return launch_kernel<GROUPED>(fn, &mx_tile<C::FI, C::FJ, C::ST, C::CS, C::WM, GROUPED, C::NW>, C::TM, C::TN, 64 * C::NW, C::LDS_BYTES, p, stream);
  });
}

// The checks that both products share.
tb_status check(const char* fn, const Args& p, int64_t M, int64_t N, int64_t K, int64_t sa_row, int64_t sw_row, int dtype) {
  TB_CHECK_ARG(p.a && p.sa && p.w && p.sw && p.y, "%s: null pointer", fn);
  TB_CHECK_ARG(M > 0 && N > 0 && K > 0, "%s: sizes must be positive", fn);
  TB_CHECK_ARG(M < (1ll << 31) - 256 && N < (1ll << 31) - 256, "%s: problem too large", fn);
  TB_CHECK_ARG(K % 32 == 0, "%s: K must be a multiple of 32 (got %lld)", fn, (long long)K);
  TB_CHECK_ARG(K <= 1ll << 22, "%s: K must be at most 2^22 (got %lld)", fn, (long long)K);
  TB_CHECK_ARG(dtype == 1 || dtype == 2, "%s: the output is fp16 (1) or bf16 (2), got type %d", fn, dtype);
  TB_CHECK_ARG(sa_row >= K / 32 && sw_row >= K / 32 && sa_row % 4 == 0 && sw_row % 4 == 0 && sa_row < (1ll << 22) &&
                   sw_row < (1ll << 22),
               "%s: rows of scales must hold K / 32 bytes and start on 4 bytes (strides %lld and %lld)", fn,
               (long long)sa_row, (long long)sw_row);
  TB_CHECK_ALIGN(p.a, 16, "a");
  TB_CHECK_ALIGN(p.w, 16, "w");
  TB_CHECK_ALIGN(p.sa, 4, "sa");
  TB_CHECK_ALIGN(p.sw, 4, "sw");
  TB_CHECK_ALIGN(p.y, 2, "y");
  return TB_OK;
}

void fill(Args& p, int64_t M, int64_t N, int64_t K, int64_t sa_row, int64_t sw_row, int dtype) {
  p.M = (int)M;
  p.N = (int)N;
  p.K = (int)K;
  p.sa_row = (int)sa_row;
  p.sw_row = (int)sw_row;
  p.bf16 = dtype == 2;
  p.vec = N % 8 == 0 && tb::aligned(p.y, 16);
}

}  // namespace mx
}  // namespace ntg
}  // namespace tb

void tb::describe_mxfp4(int64_t M, int64_t N, int64_t K, int64_t experts, tb_tile* out) {
  using namespace tb::ntg::mx;
  const plan::MxTile tile = plan::pick_mx_tile(M, N, K, experts);
  auto f = [&](auto shape) {
    typedef decltype(shape) C;
    *out = tb_tile{"mx_tile", C::TM, C::TN, C::NW, 1, 1, C::ST};
    return TB_OK;
  };
  if (tile == plan::MX_32x32)
    *out = tb_tile{"mx_skinny", 32, SK_N, SKINNY_KS, SKINNY_KS, 1};
  else if (experts)
    with_tile<true>(tile, f);
  else
    with_tile<false>(tile, f);
}

extern "C" tb_status tb_mxfp4_gemm(const uint8_t* a, const uint8_t* sa, const uint8_t* w, const uint8_t* sw, void* y,
                                   int64_t M, int64_t N, int64_t K, int64_t sa_row, int64_t sw_row, int dtype,
                                   hipStream_t stream) {
  using namespace tb::ntg::mx;
  Args p{};
  p.a = a;
  p.sa = sa;
  p.w = w;
  p.sw = sw;
  p.y = static_cast<uint16_t*>(y);
  if (tb_status st = check("tb_mxfp4_gemm", p, M, N, K, sa_row, sw_row, dtype)) return st;
  fill(p, M, N, K, sa_row, sw_row, dtype);
  return launch<false>("tb_mxfp4_gemm", p, stream);
}

extern "C" tb_status tb_moe_mxfp4_grouped_gemm(const uint8_t* a, const uint8_t* sa, const uint8_t* w, const uint8_t* sw,
                                               const int32_t* offsets, const int32_t* gather, const int32_t* scatter,
                                               const float* weights, void* y, int64_t R, int64_t a_rows,
                                               int64_t experts, int64_t N, int64_t K, int64_t topk, int64_t sa_row,
                                               int64_t sw_row, int64_t sw_expert, int dtype, hipStream_t stream) {
  using namespace tb::ntg::mx;
  const char* const fn = "tb_moe_mxfp4_grouped_gemm";
  Args p{};
  p.a = a;
  p.sa = sa;
  p.w = w;
  p.sw = sw;
  p.y = static_cast<uint16_t*>(y);
  p.offsets = offsets;
  p.gather = gather;
  p.scatter = scatter;
  p.weights = weights;
  if (tb_status st = check(fn, p, R, N, K, sa_row, sw_row, dtype)) return st;
  TB_CHECK_ARG(offsets, "%s: null pointer", fn);
  TB_CHECK_ARG(experts > 0 && experts <= 4096, "%s: need 0 < experts <= 4096 (got %lld)", fn, (long long)experts);
  TB_CHECK_ARG(a_rows > 0 && topk > 0 && topk < (1ll << 31), "%s: sizes must be positive", fn);
  TB_CHECK_ARG(gather || a_rows >= R, "%s: A has %lld rows for %lld product rows", fn, (long long)a_rows, (long long)R);
  TB_CHECK_ARG(!gather || (a_rows * (K / 2) < (1ll << 31) && a_rows * sa_row < (1ll << 31)),
               "%s: gathered rows come from an A smaller than 2 GiB (%lld rows of K = %lld)", fn, (long long)a_rows,
               (long long)K);
  TB_CHECK_ARG(sw_expert % 4 == 0 && sw_expert >= (N - 1) * sw_row + K / 32,
               "%s: experts' scales must not overlap and start on 4 bytes (stride %lld)", fn, (long long)sw_expert);
  TB_CHECK_ALIGN(offsets, 4, "offsets");
  fill(p, R, N, K, sa_row, sw_row, dtype);
  p.E = (int)experts;
  p.a_rows = (int)(a_rows < (1ll << 31) - 1 ? a_rows : (1ll << 31) - 1);
  p.sw_expert = sw_expert;
  p.by_topk = tb::Divisor((uint32_t)topk);
  return launch<true>(fn, p, stream);
}
