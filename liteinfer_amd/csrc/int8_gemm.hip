// out = x w^T in 8-bit integers: x [m, k] quantised on the way in with a scale
// for each row (token), w [n, k] held as codes with a scale for each of its
// rows (output channel).
//     sx[i]  = max(largest |x[i, :]| / 127, 2^-126)
//     c[i]   = rint(x[i, :] / sx[i])              (as a product with 1 / sx[i])
//     out[i, j] = (sum_k c[i, k] w[j, k]) * sx[i] * sw[j]
// The sums are int32 and exact (k <= LI_INT8_MAX_K keeps 127^2 k below 2^31);
// scales and their products are fp32, the output is rounded once. A row that
// holds a value that is not finite gets a NaN scale, so its outputs are NaN.
//
// Everything moves in bytes as a 16-bit product of half the k would: an
// operand of v_mfma_i32_16x16x64_i8 is 16 codes (16 bytes) a lane, lane
// (r, g) = (lane % 16, lane / 16) holding bytes 16 g .. of 64 of row r.
// Operand A is 16 rows of w, B 16 rows of x, so lane (r, g) ends with outputs
// 4 g .. 4 g + 3 of row r: four neighbours in memory.
//
// Codes past k are zero in x (its codes are laid out in rows of a multiple
// of kPadK), so whatever is read of w there does not count; reads of w are
// held to its rows' last 16 bytes.
#include "li_mfma.h"

#include <type_traits>

namespace {

using namespace li;

typedef int v4i __attribute__((ext_vector_type(4)));

constexpr int kPadK = 256;
constexpr float kStep = 1.0f / 127.0f;
constexpr float kLeast = 1.17549435e-38f;  // 2^-126
constexpr uint32_t kInfBits = 0x7f800000u;

template <typename E>
using Vec8 = __attribute__((__vector_size__(8 * sizeof(E)), __aligned__(16))) E;

// A row's scale (as bits) and its codes' factor, from the bits of its largest
// magnitude (which order what is not finite above the rest).
struct RowScale {
  uint32_t bits;
  float inv;  // 0: not finite, every code 0
};
__device__ __forceinline__ RowScale row_scale(uint32_t largest) {
  const bool lost = largest >= kInfBits;
  const float s = fmaxf(__uint_as_float(lost ? 0u : largest) * kStep, kLeast);
  return {lost ? 0x7fc00000u : __float_as_uint(s), lost ? 0.f : 1.f / s};
}

__device__ __forceinline__ uint32_t code_of(float x, float inv) {
  return (uint32_t)(int)fminf(fmaxf(rintf(x * inv), -127.f), 127.f) & 255u;
}

template <typename E>
__device__ __forceinline__ uint2 codes_of(const Vec8<E>& x, float inv, bool lost) {
  uint32_t w[2] = {0u, 0u};
  if (!lost) {
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e / 4] |= code_of(li_to_float(x[e]), inv) << (8 * (e % 4));
  }
  return uint2{w[0], w[1]};
}

template <typename E>
__device__ __forceinline__ uint32_t largest_of(const Vec8<E>& x) {
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(li_to_float(x[e])) & 0x7fffffffu);
  return top;
}

// ---------------------------------------------------------------------------
// Quantising rows: one work-group a row. Up to kHold x 2,048 values stay in
// registers between the maximum and the codes; longer rows are read twice.
// Memory-bound.
// ---------------------------------------------------------------------------

constexpr int kQuantHold = 2048;

// Eight values of a row from column d (zeros past k), whatever its alignment.
template <typename E, bool kVec>
__device__ __forceinline__ Vec8<E> row_values(const E* row, int d, int k) {
  if constexpr (kVec) {
    if (d + 8 <= k) return *reinterpret_cast<const Vec8<E>*>(row + d);
  }
  Vec8<E> v;
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = d + e < k ? row[d + e] : li_from_float<E>(0.f);
  return v;
}

template <typename E, bool kVec, int kQuantThreads>
__global__ __launch_bounds__(kQuantThreads) void quantize_rows(const E* x, int64_t x_s, int8_t* codes, int64_t c_s,
                                                               float* scales, int k, int padded) {
  constexpr int kHold = kQuantHold / kQuantThreads;
  const int tid = threadIdx.x;
  const E* row = x + (int64_t)blockIdx.x * x_s;
  Vec8<E> held[kHold];
  uint32_t top = 0;
#pragma unroll
  for (int u = 0; u < kHold; ++u) {
    const int d = 8 * (tid + kQuantThreads * u);
    if (d < k) {
      held[u] = row_values<E, kVec>(row, d, k);
      top = max(top, largest_of<E>(held[u]));
    }
  }
  for (int d = 8 * (tid + kQuantThreads * kHold); d < k; d += 8 * kQuantThreads)
    top = max(top, largest_of<E>(row_values<E, kVec>(row, d, k)));
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, off, 64));
  __shared__ uint32_t tops[kQuantThreads / 64];
  if ((tid & 63) == 0) tops[tid >> 6] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kQuantThreads / 64; ++w) top = max(top, tops[w]);
  const RowScale s = row_scale(top);
  const bool lost = top >= kInfBits;
  int8_t* out = codes + (int64_t)blockIdx.x * c_s;
#pragma unroll
  for (int u = 0; u < kHold; ++u) {
    const int d = 8 * (tid + kQuantThreads * u);
    if (d < k) *reinterpret_cast<uint2*>(out + d) = codes_of<E>(held[u], s.inv, lost);
    else if (d < padded) *reinterpret_cast<uint2*>(out + d) = uint2{0u, 0u};
  }
  for (int d = 8 * (tid + kQuantThreads * kHold); d < padded; d += 8 * kQuantThreads)
    *reinterpret_cast<uint2*>(out + d) = d < k ? codes_of<E>(row_values<E, kVec>(row, d, k), s.inv, lost) : uint2{0u, 0u};
  if (tid == 0) reinterpret_cast<uint32_t*>(scales)[blockIdx.x] = s.bits;
}

// ---------------------------------------------------------------------------
// The product.
// ---------------------------------------------------------------------------

struct GemmArgs {
  const char* x;     // codes [m, x_s], zero from k to a multiple of kPadK
  const float* xs;   // [m]
  const char* w;     // codes [n, w_s]
  const float* ws;   // [n]
  char* out;         // T rows (splits == 1)
  int32_t* part;     // [splits][m][n] sums (splits > 1)
  int64_t x_s, w_s;  // row strides in bytes
  int64_t o_s;       // out: in elements
  int m, n, k;
  int splits;
  int vec;           // four outputs side by side may be stored at once
  int rows16;        // 16-bit rows of the output are 16-byte aligned
  int mt, nt;        // tiles of rows of x, of w
};

// Four sums for outputs n .. n + 3 of row m.
template <typename T>
__device__ __forceinline__ void store4(const GemmArgs& a, const v4i& acc, int split, int m, int n) {
  if (m >= a.m || n >= a.n) return;
  if (a.splits > 1) {
    int32_t* p = a.part + ((int64_t)split * a.m + m) * a.n + n;
    if (a.vec && n + 4 <= a.n) {
      *reinterpret_cast<v4i*>(p) = acc;
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (n + r < a.n) p[r] = acc[r];
    }
    return;
  }
  const float sx = a.xs[m];
  T* o = reinterpret_cast<T*>(a.out) + m * a.o_s + n;
  float v[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) v[r] = n + r < a.n ? (float)acc[r] * sx * a.ws[n + r] : 0.f;
  if (a.vec && n + 4 <= a.n) {
    if constexpr (sizeof(T) == 4) *reinterpret_cast<floatx4_t*>(o) = floatx4_t{v[0], v[1], v[2], v[3]};
    else *reinterpret_cast<uint2*>(o) = uint2{li_pack2<T>(v[0], v[1]), li_pack2<T>(v[2], v[3])};
  } else {
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (n + r < a.n) o[r] = li_from_float<T>(v[r]);
  }
}

// Waits until at most `newer` stages of kPer loads each are in flight.
template <int R, int kPer>
__device__ __forceinline__ void wait_stages(int newer) {
  static_assert(R >= 2 && R <= 4 && (R - 2) * kPer < 64, "vmcnt range");
  if (R > 3 && newer >= 2) li_wait_vm<(R > 3 ? 2 * kPer : 0)>();
  else if (R > 2 && newer >= 1) li_wait_vm<(R > 2 ? kPer : 0)>();
  else li_wait_vm<0>();
}

// This work-group's tile: {tile of x's rows x runs + run, tile of w's rows}.
// Work-group i runs on XCD i % 8; each XCD takes a run of tiles in columns of
// `kColumn` along x's rows, so that the 32 it works on at a time read few
// rows of either operand (4 x 8 tiles: 12 rows of tiles, where 17 x 2 read
// 19), all of them at about the same k, from its L2.
constexpr int kColumn = 4;
__device__ __forceinline__ int2 tile_of(const GemmArgs& a, int splits) {
  const int across = a.mt * splits, total = across * a.nt;
  const int per = total / 8, rest = total % 8;
  const int xcd = (int)(blockIdx.x % 8u), at = (int)(blockIdx.x / 8u);
  const int t = xcd * per + min(xcd, rest) + at;
  const int column = t / (kColumn * a.nt), in = t - column * kColumn * a.nt;
  const int wide = min(kColumn, across - column * kColumn);
  return int2{column * kColumn + in % wide, in / wide};
}

// A work-group of WM x WN waves takes BM rows of x by BN rows of w and a run
// of k, both operands straight into LDS in a ring of R stages of RB bytes a
// row, chunk c (16 bytes) of row r at c ^ swizzle(r). A 16-byte LDS read is
// served 16 lanes at a time, lanes 0-3, 12-15, 20-23 and 24-27 together, then
// 4-11, 16-19 and 28-31, then the same of the upper half: eight rows of one
// chunk with eight others of the next, which the swizzles keep in 16 different
// bank groups. R - 1 stages are in flight, one barrier a stage; the operands of
// one step of 64 k are read while the step before is multiplied, across the
// barrier too, one read with every few products.
// 64 x 64 of 256-byte stages: 61 x 14336 by 4096 in 13.5 us, w at 4.3 TB/s.
// 128 x 128 of 128-byte stages: 1000 x 4096 by 6144 in 55 us, 0.9 P operations
// a second, LDS as busy as the matrix units (two reads of operands a product).
template <int RB>
__device__ __forceinline__ int swizzle(int row) {
  return (row / (256 / RB)) % (RB / 16);
}
template <typename T, int BM, int BN, int WM, int WN, int RB, int R>
__global__ __launch_bounds__(64 * WM * WN) void ring_gemm(GemmArgs a) {
  constexpr int kWaves = WM * WN;
  constexpr int kCh = RB / 16;                 // chunks of a row
  constexpr int kRows = 64 / kCh;              // rows one load fills
  constexpr int kLoads = (BM + BN) / kRows, kPer = kLoads / kWaves;
  static_assert(kPer >= 1 && kPer * kWaves == kLoads, "the waves split a stage's loads evenly");
  constexpr int kFm = BM / WM / 16, kFn = BN / WN / 16, kK = RB / 64;
  constexpr int kStage = (BM + BN) * RB;
  __shared__ __attribute__((aligned(1024))) char ring[R][kStage];
  const int lane = (int)(threadIdx.x & 63);
  const int wv = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int r16 = lane & 15, g = lane >> 4;

  const int2 tile = tile_of(a, a.splits);
  const int split = (int)(tile.x % (unsigned)a.splits), tm = (int)(tile.x / (unsigned)a.splits), tn = tile.y;
  const int stages = (a.k + RB - 1) / RB;
  const int s0 = (int)((int64_t)stages * split / a.splits), s1 = (int)((int64_t)stages * (split + 1) / a.splits);
  const int ns = s1 - s0;

  // Load i of this wave fills rows kRows * (wv * kPer + i) .. of the stage
  // (x's rows first); a lane brings one chunk. Rows past the last repeat it.
  const char* src[kPer];
  int col[kPer], cap[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int row = kRows * (wv * kPer + i) + lane / kCh;
    col[i] = 16 * ((lane % kCh) ^ swizzle<RB>(row)) + s0 * RB;
    src[i] = row < BM ? a.x + (int64_t)min(tm * BM + row, a.m - 1) * a.x_s
                      : a.w + (int64_t)min(tn * BN + row - BM, a.n - 1) * a.w_s;
    // w's rows end at their last chunk; x's go on in zeros.
    cap[i] = row < BM ? 0x7fffffff : (a.k + 15) / 16 * 16 - 16;
  }
  const uint32_t base = lds_addr(&ring[0][0]);
  auto issue = [&](int st) {
    const uint32_t dst = base + (uint32_t)(st % R) * kStage + (uint32_t)wv * kPer * 1024;
#pragma unroll
    for (int i = 0; i < kPer; ++i) dma16<false>(src[i] + min(col[i] + st * RB, cap[i]), dst + 1024 * i);
  };

  v4i acc[kFm][kFn];
#pragma unroll
  for (int i = 0; i < kFm; ++i)
#pragma unroll
    for (int j = 0; j < kFn; ++j) acc[i][j] = v4i{0, 0, 0, 0};
  const int wm = wv % WM, wn = wv / WM;
  uint32_t off[kK];
#pragma unroll
  for (int j = 0; j < kK; ++j) off[j] = (uint32_t)(r16 * RB + 16 * ((4 * j + g) ^ swizzle<RB>(r16)));

  v4i x0[kFm], w0[kFn], x1[kFm] = {}, w1[kFn] = {};
  auto read = [&](int st, int j, v4i (&xf)[kFm], v4i (&wf)[kFn]) __attribute__((always_inline)) {
    const uint32_t stage = base + (uint32_t)(st % R) * kStage + off[j];
    const uint32_t xc = stage + (uint32_t)wm * (BM / WM) * RB, wc = stage + (uint32_t)(BM + wn * (BN / WN)) * RB;
#pragma unroll
    for (int f = 0; f < kFn; ++f) wf[f] = lds_read_frag<v4i>(wc + f * 16 * RB);
#pragma unroll
    for (int i = 0; i < kFm; ++i) xf[i] = lds_read_frag<v4i>(xc + i * 16 * RB);
  };
  auto multiply = [&](const v4i (&xf)[kFm], const v4i (&wf)[kFn]) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kFm; ++i)
#pragma unroll
      for (int f = 0; f < kFn; ++f) acc[i][f] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[f], xf[i], acc[i][f], 0, 0, 0);
  };
  auto interleave = [&]() __attribute__((always_inline)) {
    constexpr int kReads = kFm + kFn, kEach = (kFm * kFn + kReads - 1) / kReads;
#pragma unroll
    for (int i = 0; i < kReads; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);  // an LDS read
      __builtin_amdgcn_sched_group_barrier(0x008, kEach, 0);
    }
  };
  // Stage st has landed; every wave is done with stage st - 1, whose place
  // the next loads take.
  auto enter = [&](int st) __attribute__((always_inline)) {
    wait_stages<R, kPer>(min(R - 2, ns - 1 - st));
    lds_barrier();
    if (st + R - 1 < ns) issue(st + R - 1);
  };

#pragma unroll
  for (int st = 0; st < R - 1; ++st)
    if (st < ns) issue(st);
  static_assert(kK % 2 == 0, "an even number of steps leaves the last in the second set");
  for (int st = 0; st < ns; ++st) {
    enter(st);
#pragma unroll
    for (int j = 0; j < kK; j += 2) {
      read(st, j, x0, w0);
      multiply(x1, w1);
      interleave();
      read(st, j + 1, x1, w1);
      multiply(x0, w0);
      interleave();
    }
    __builtin_amdgcn_sched_barrier(0);
  }
  multiply(x1, w1);
#pragma unroll
  for (int i = 0; i < kFm; ++i)
#pragma unroll
    for (int f = 0; f < kFn; ++f)
      store4<T>(a, acc[i][f], split, tm * BM + wm * (BM / WM) + 16 * i + r16, tn * BN + wn * (BN / WN) + 16 * f + 4 * g);
}

// Up to 16 rows: bound by the reading of w. A work-group takes 16 of w's rows,
// each of its four waves a quarter of k with a ring of its own (no barriers;
// XR of x's rows beside w's 16, R stages of 256 bytes a row in flight), and
// the waves' sums meet in LDS: no second kernel joins runs of k. (Tiles of 64
// of w's rows, k cut over the grid and a second kernel took 12.9 us a call at
// 1 x 4096 by 6144 where this takes 9.1, quantising included, 21.4 for 14.0 at
// 1 x 14336 by 4096, 21.8 for 15.9 with 16 rows. Operands loaded straight into
// registers and x quantised in every work-group: 20.1, 61 and 45.) 117 MB of w
// come at 5.6 TB/s; what is left at 25 MB is two launches and a wave's eight
// stages. XR = 4 where it does (4 rows: 9.1, as 16: 10.5).
template <typename T, int XR, int R>
__global__ __launch_bounds__(256) void few_gemm(GemmArgs a) {
  constexpr int kPer = (16 + XR) / 4;  // loads a stage, four rows each
  constexpr uint32_t kStage = 1024 * kPer;
  __shared__ __attribute__((aligned(1024))) char ring[4 * R * kStage];
  const int lane = (int)(threadIdx.x & 63);
  const int wv = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int r16 = lane & 15, g = lane >> 4;
  const int n0 = 16 * (int)blockIdx.x;
  const int stages = (a.k + 255) / 256, part = (stages + 3) / 4;
  const int s0 = wv * part, ns = min(part, stages - s0);
  const char* src[kPer];
  int col[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int row = (i < 4 ? 4 * i : 4 * (i - 4)) + g;
    col[i] = 16 * (r16 ^ swizzle<256>(row)) + s0 * 256;
    src[i] = i < 4 ? a.w + (int64_t)min(n0 + row, a.n - 1) * a.w_s : a.x + (int64_t)min(row, a.m - 1) * a.x_s;
  }
  const int cap = (a.k + 15) / 16 * 16 - 16;  // w's rows end at their last chunk; x's go on in zeros
  const uint32_t base = lds_addr(&ring[0]);
  const uint32_t mine = base + (uint32_t)wv * (R * kStage);
  auto issue = [&](int st) __attribute__((always_inline)) {
    const uint32_t to = mine + (uint32_t)(st % R) * kStage;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int at = col[i] + st * 256;
      if (i < 4) dma16<true>(src[i] + min(at, cap), to + 1024 * i);
      else dma16<false>(src[i] + at, to + 1024 * i);
    }
  };
  uint32_t woff[4], xoff[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    woff[j] = mine + (uint32_t)(r16 * 256 + 16 * ((4 * j + g) ^ swizzle<256>(r16)));
    xoff[j] = mine + 4096 + (uint32_t)(r16 % XR * 256 + 16 * ((4 * j + g) ^ swizzle<256>(r16 % XR)));
  }
  v4i acc = {0, 0, 0, 0};
#pragma unroll
  for (int st = 0; st < R; ++st)
    if (st < ns) issue(st);
  for (int st = 0; st < ns; ++st) {
    wait_stages<R + 1, kPer>(min(R - 1, ns - 1 - st));
    const uint32_t at = (uint32_t)(st % R) * kStage;
    v4i wf[4], xf[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      wf[j] = lds_read_frag<v4i>(woff[j] + at);
      xf[j] = lds_read_frag<v4i>(xoff[j] + at);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");  // read before the next loads write there
    if (st + R < ns) issue(st + R);
#pragma unroll
    for (int j = 0; j < 4; ++j) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[j], xf[j], acc, 0, 0, 0);
  }
  // (Every load of the wave is in: its ring is free.)
  *reinterpret_cast<__attribute__((address_space(3))) v4i*>((uintptr_t)(mine + 16 * lane)) = acc;
  __syncthreads();
  if (wv) return;
  v4i sum = {0, 0, 0, 0};
#pragma unroll
  for (int p = 0; p < 4; ++p) sum += lds_read_frag<v4i>(base + p * (R * kStage) + 16 * lane);
  store4<T>(a, sum, 0, r16, n0 + 4 * g);
}

// acc += w x^T in place. (As a builtin the accumulators of a wave that has 256
// of them were moved about: a thousand moves between registers in the loop.)
__device__ __forceinline__ void add_product(v4i& acc, const v4i& w, const v4i& x) {
  asm volatile("v_mfma_i32_16x16x64_i8 %0, %1, %2, %0" : "+a"(acc) : "v"(w), "v"(x));
}
// The products issued before are complete: their accumulators may be read,
// moved or written by other instructions. (The compiler does not see what an
// asm block issues, so it counts no such wait itself.)
__device__ __forceinline__ void products_done() {
  asm volatile("s_nop 15\n\ts_nop 7" : : : "memory");
  __builtin_amdgcn_sched_barrier(0);
}

// The same for many rows: 256 x 256 outputs of four waves, 128 x 128 each, one
// wave a SIMD with its 256 accumulators in the accumulation registers and two
// steps' operands (64 k) in the others; or 256 x 128, 128 x 64 a wave, with a
// ring of three stages for two. (Eight waves of 128 x 64 read half as much
// again from LDS, which with the loads' writes was as busy as the matrix
// units: 472 us for the whole call at the size below, now 435.) A step is FM
// groups of FN products; the first of them read the next step's operands, and
// each group issues its part of the loads of the stage R - 1 ahead. (Stages of
// 64 bytes a row in a ring of five instead of 128 in one of two ask the L2 for
// its lines twice: 480 us against 440.)
// Bound by the matrix units at the clock they leave: 4096 x 4096 by 28672 in
// 430 us, 2.2 P operations a second, products 51% of the cycles at 1.87 GHz
// (the same product's int32 sums alone take the library 529 us); the rest is
// the wait for a stage (1.6 us for 1.1 us of products) and, once a tile, the
// first stage and the store.
template <typename T, int FM, int FN, int R>
__global__ __launch_bounds__(256, 1) void wide_gemm(GemmArgs a) {
  constexpr int BM = 32 * FM, BN = 32 * FN;  // 2 x 2 waves of FM x FN groups of 16
  constexpr int RB = 128;                    // bytes of k a stage, two steps
  constexpr int kRows = 1024 / RB, kPer = (BM + BN) / kRows / 4;  // rows a load, loads a wave and stage
  constexpr int kK = RB / 64;
  constexpr int kEach = (kPer + FM - 1) / FM;  // loads with a group of products
  constexpr uint32_t kStage = (BM + BN) * RB;
  static_assert(kK == 2 && kEach <= FN && 2 * (FM + FN) <= FM * FN, "two steps a stage; room for its loads and reads");
  __shared__ __attribute__((aligned(1024))) char ring[R * kStage];
  const int lane = (int)(threadIdx.x & 63);
  const int wv = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int r16 = lane & 15, g = lane >> 4;
  const int2 tile = tile_of(a, 1);
  const int tm = tile.x, tn = tile.y;
  const int ns = (a.k + RB - 1) / RB;  // (x's codes are zero up to a multiple of kPadK)

  // A stage's rows, x's first, a quarter to a wave; rows past an operand's
  // last repeat it, and w's rows end at their last chunk.
  const char* xsrc = a.x + (int64_t)tm * BM * a.x_s;
  const char* wsrc = a.w + (int64_t)tn * BN * a.w_s;
  const int wcap = (a.k + 15) / 16 * 16 - 16;
  const char* src[kPer];
  uint32_t row_at[kPer];
  int col[kPer], cap[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int row = kRows * (wv * kPer + i) + lane / (RB / 16);
    const bool of_x = kRows * (wv * kPer + i) < BM;
    row_at[i] = of_x ? (uint32_t)min(row, a.m - 1 - tm * BM) * (uint32_t)a.x_s
                     : (uint32_t)min(row - BM, a.n - 1 - tn * BN) * (uint32_t)a.w_s;
    col[i] = 16 * ((lane % (RB / 16)) ^ swizzle<RB>(row));
    src[i] = of_x ? xsrc : wsrc;
    cap[i] = of_x ? 0x7fffffff : wcap;
  }
  const uint32_t base = lds_addr(&ring[0]);
  const uint32_t mine = base + (uint32_t)wv * kPer * 1024;
  auto load = [&](int st, uint32_t to, int i) __attribute__((always_inline)) {
    dma16_at(src[i], row_at[i] + (uint32_t)min(col[i] + st * RB, cap[i]), mine + to + 1024 * i);
  };

  v4i acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = v4i{0, 0, 0, 0};
  const int wm = wv & 1, wn = wv >> 1;
  uint32_t xoff[kK], woff[kK];
#pragma unroll
  for (int j = 0; j < kK; ++j) {
    const uint32_t o = base + (uint32_t)(r16 * RB + 16 * ((4 * j + g) ^ swizzle<RB>(r16)));
    xoff[j] = o + (uint32_t)wm * (BM / 2) * RB;
    woff[j] = o + (uint32_t)(BM + wn * (BN / 2)) * RB;
  }
  v4i x0[FM], x1[FM], w0[FN], w1[FN];
  uint32_t here = 0, fill = (R - 1) * kStage;  // the ring's stage that is read from, and the one to load into
  // Stage st is here (all of it, once every wave has come), and the one before it is free.
  auto enter = [&]() __attribute__((always_inline)) {
    here = here == (R - 1) * kStage ? 0 : here + kStage;
    fill = fill == (R - 1) * kStage ? 0 : fill + kStage;
    li_wait_vm<(R - 2) * kPer>();
    lds_barrier();
  };
  // One step, its operands in (xa, wa); leaves the next step's in (xb, wb): of
  // the same stage, or of stage `st`, entered first. (Past the last stage the
  // last is loaded once more and what is read is not used: without branches
  // the accumulators stay where they are.)
  auto step = [&](int st, int j, const v4i (&xa)[FM], const v4i (&wa)[FN], v4i (&xb)[FM], v4i (&wb)[FN])
      __attribute__((always_inline)) {
    const bool entered = j == 0;
    if (entered) enter();
    const int ahead = min(st + R - 1, ns - 1);
#pragma unroll
    for (int i = 0; i < FM; ++i) {
#pragma unroll
      for (int f = 0; f < FN; ++f) {
        if (entered && f < kEach && i * kEach + f < kPer) load(ahead, fill, i * kEach + f);
        const int r = (FN * i + f) / 2;
        if (f % 2 == 0 && r < FN) wb[r] = lds_read_frag<v4i>(woff[j] + here + r * 16 * RB);
        else if (f % 2 == 0 && r < FN + FM) xb[r - FN] = lds_read_frag<v4i>(xoff[j] + here + (r - FN) * 16 * RB);
        add_product(acc[i][f], wa[f], xa[i]);
        if (f % 2) __builtin_amdgcn_sched_barrier(0);
      }
    }
  };

#pragma unroll
  for (int st = 0; st < R; ++st)
#pragma unroll
    for (int i = 0; i < kPer; ++i) load(min(st, ns - 1), (uint32_t)st * kStage, i);
  li_wait_vm<(R - 1) * kPer>();
  lds_barrier();
#pragma unroll
  for (int i = 0; i < FN; ++i) w0[i] = lds_read_frag<v4i>(woff[0] + i * 16 * RB);
#pragma unroll
  for (int i = 0; i < FM; ++i) x0[i] = lds_read_frag<v4i>(xoff[0] + i * 16 * RB);
  for (int st = 0; st < ns; ++st) {
    step(st, 1, x0, w0, x1, w1);
    step(st + 1, 0, x1, w1, x0, w0);
    // Here, not after the loop, where moves of accumulators may come first
    // (24 cycles in 4,096 of the largest tile).
    products_done();
  }
  li_wait_vm<0>();
  lds_barrier();  // every load is in and every wave has read its last operands: the ring is free
  const int m0 = tm * BM + wm * (BM / 2), n0 = tn * BN + wn * (BN / 2);
  if constexpr (sizeof(T) == 2) {
    if (a.rows16 && n0 + BN / 2 <= a.n) {
      // A lane holds four neighbours of a row, 16 rows to an instruction: stored
      // as they are every store would write 32-byte pieces (the stores alone
      // took a quarter of the call). Each wave turns its rows in its own part
      // of the ring instead, chunk c of row r at c ^ r % kCh, and stores whole
      // rows.
      constexpr int kRowBytes = BN, kCh = kRowBytes / 16, kRowsEach = 64 / kCh;
      static_assert(R * kStage >= 4 * (BM / 2) * kRowBytes, "the ring holds the waves' rows");
      const uint32_t rows = base + (uint32_t)wv * (BM / 2 * kRowBytes);
      floatx4_t ws[FN];
#pragma unroll
      for (int f = 0; f < FN; ++f) {
#pragma unroll
        for (int r = 0; r < 4; ++r) ws[f][r] = a.ws[n0 + 16 * f + 4 * g + r];
      }
      typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
#pragma unroll
      for (int i = 0; i < FM; ++i) {
        const int row = 16 * i + r16;
        const float sx = a.xs[min(m0 + row, a.m - 1)];
#pragma unroll
        for (int f = 0; f < FN; ++f) {
          float v[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) v[r] = (float)acc[i][f][r] * sx * ws[f][r];
          const int c = 2 * f + (g >> 1);
          *reinterpret_cast<__attribute__((address_space(3))) u32x2_t*>(
              (uintptr_t)(rows + row * kRowBytes + 16 * (c ^ (row % kCh)) + 8 * (g & 1))) =
              u32x2_t{li_pack2<T>(v[0], v[1]), li_pack2<T>(v[2], v[3])};
        }
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int i = 0; i < BM / 2 / kRowsEach; ++i) {
        const int row = kRowsEach * i + lane / kCh, c = lane % kCh;
        const u32x4_t v = lds_read_frag<u32x4_t>(rows + row * kRowBytes + 16 * (c ^ (row % kCh)));
        if (m0 + row < a.m)
          __builtin_nontemporal_store(v, reinterpret_cast<u32x4_t*>(a.out + ((int64_t)(m0 + row) * a.o_s + n0 + 8 * c) * 2));
      }
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int f = 0; f < FN; ++f) {
      store4<T>(a, acc[i][f], 0, m0 + 16 * i + r16, n0 + 16 * f + 4 * g);
      __builtin_amdgcn_sched_barrier(0);
    }
}

// out = the splits' sums, scaled and rounded.
template <typename T>
__global__ __launch_bounds__(256) void reduce_sums(GemmArgs a) {
  const int64_t quads = (a.n + 3) / 4;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= a.m * quads) return;
  const int m = (int)(i / quads), n = (int)(i - m * quads) * 4;
  v4i s = {0, 0, 0, 0};
#pragma unroll 4
  for (int p = 0; p < a.splits; ++p) {
    const int32_t* src = a.part + ((int64_t)p * a.m + m) * a.n + n;
    if (a.vec && n + 4 <= a.n) {
      s += *reinterpret_cast<const v4i*>(src);
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (n + r < a.n) s[r] += src[r];
    }
  }
  GemmArgs whole = a;
  whole.splits = 1;
  store4<T>(whole, s, 0, m, n);
}

// Of tiles of 256 rows the last, where it would hold few, runs after the
// others as a product of its own: a row of tiles costs its share of a round
// of the GPU whatever it holds (4099 x 4096 by 28672: 521 us -> 488).
constexpr int kFewLeft = 64;
constexpr int64_t kWideStride = int64_t(1) << 23;  // 255 rows of it and a row's bytes stay below 2^32

// Which kernel a product runs on and the runs its k is cut into.
enum Kind { kFew, kSome, kMany, kHalf, kMost };
struct Plan {
  Kind kind;
  int bm, bn, splits;
};
// Tiles of 64 x 64 while they fit the GPU at once: against 128 x 128 they give
// 16 us for 20 at 100 x 4096 by 4096, 17 for 22 at 256 rows, 12 for 18 at 300 x
// 2048 by 2048; with more of them than compute units 128 x 128 wins (52 for 40
// at 100 x 4096 by 28672).
// Above, the last round of tiles (one a compute unit) decides, by what it
// leaves idle: a round of 128 x 128, 256 x 128 and 256 x 256 takes about 30, 37
// and 62 us at k = 4096. 256 x 128 against 128 x 128: 46 us for 69 at 256 x 4096
// by 28672 (1 round, 2), 43 for 63 at 1000 by 6144 and 46 for 67 at 2048 by 4096
// (1, 2), but 113 for 89 at 1000 x 14336 by 4096 (1, 1). 256 x 256 against 256 x
// 128: 72 for 77 at 512 by 28672 and 69 for 77 at 2000 by 6144 (1, 2), but 126
// for 115 at 600 by 28672 (2, 3) and 67 for 43 at 1000 by 6144 (1, 1).
// Tiles that leave a quarter of the GPU idle cut k, to runs of 1,024 at least:
// 40 us -> 24 at 64 x 14336 by 4096, 77 -> 28 at 100 rows.
Plan plan_of(int m, int n, int k) {
  const int cus = li::device_cu_count();
  const auto rounds = [&](int64_t tm, int64_t tn) { return (tm * tn + cus - 1) / cus; };
  const int left = m % 256, tall = left && left <= kFewLeft && m > left ? m / 256 : cdiv(m, 256);
  const int64_t many = 5 * rounds(cdiv(m, 128), cdiv(n, 128)), half = 6 * rounds(tall, cdiv(n, 128));
  const int64_t most = 10 * rounds(tall, cdiv(n, 256));
  Plan p{};
  if (m <= 16) p = {kFew, 16, 16, 1};
  else if (m <= 64 || (int64_t)cdiv(m, 64) * cdiv(n, 64) <= cus) p = {kSome, 64, 64, 1};
  else if (many <= std::min(half, most)) p = {kMany, 128, 128, 1};
  else if (half <= most) p = {kHalf, 256, 128, 1};
  else p = {kMost, 256, 256, 1};
  const int64_t tiles = (int64_t)cdiv(m, p.bm) * cdiv(n, p.bn);
  if ((p.kind == kSome || p.kind == kMany) && tiles * 4 < cus * 3)
    p.splits = std::max<int>(1, std::min<int64_t>(cus / tiles, cdiv(k, 1024)));
  return p;
}

size_t align256(size_t x) { return (x + 255) & ~size_t(255); }

struct Space {
  int64_t x_s;
  size_t scales, part, need;  // byte offsets: the codes come first
};
Space space_of(int m, int n, int k) {
  Space s;
  const Plan p = plan_of(m, n, k);
  s.x_s = (int64_t)(k + kPadK - 1) / kPadK * kPadK;
  s.scales = align256((size_t)m * s.x_s);
  s.part = s.scales + align256((size_t)m * sizeof(float));
  s.need = s.part + (p.splits > 1 ? align256((size_t)p.splits * m * n * sizeof(int32_t)) : 0);
  return s;
}

int check_extents(const char* who, int m, int n, int k) {
  if (m < 0 || n <= 0 || k <= 0) return li::fail(LI_EINVAL, "%s: bad extents (%d, %d, %d)", who, m, n, k);
  if (k > LI_INT8_MAX_K)
    return li::fail(LI_EUNSUPPORTED, "%s: sums of %d products pass 32 bits, %d at most", who, k, LI_INT8_MAX_K);
  return LI_OK;
}

// Few long rows take four times the threads each: 61 rows of 14,336 bring a
// call from 24.6 us to 23.1, 256 of 4,096 from 23.1 to 21.5; 600 of 14,336
// lose by it (80.5 -> 82.5), as their work-groups fill the GPU anyway.
constexpr int kQuantWideRows = 512, kQuantWideK = 2048;
template <typename E>
void launch_quantize(const void* x, int64_t x_s, void* codes, int64_t c_s, float* scales, int m, int k, int padded,
                     hipStream_t s) {
  const bool vec = li::aligned16(x) && (x_s * (int64_t)sizeof(E)) % 16 == 0;
  const E* xp = static_cast<const E*>(x);
  int8_t* cp = static_cast<int8_t*>(codes);
#define LI_QUANTIZE(VEC, THREADS) \
  hipLaunchKernelGGL((quantize_rows<E, VEC, THREADS>), dim3((unsigned)m), dim3(THREADS), 0, s, xp, x_s, cp, c_s, scales, k, padded)
  const bool wide = m < kQuantWideRows && k > kQuantWideK;
  if (vec && wide) LI_QUANTIZE(true, 1024);
  else if (vec) LI_QUANTIZE(true, 256);
  else LI_QUANTIZE(false, 256);
#undef LI_QUANTIZE
}

template <typename T, int BM, int BN, int WM, int WN, int RB, int R>
void launch_ring(GemmArgs a, hipStream_t s) {
  a.mt = cdiv(a.m, BM);
  a.nt = cdiv(a.n, BN);
  const dim3 grid((unsigned)(a.mt * a.nt * a.splits)), block(64 * WM * WN);
  hipLaunchKernelGGL((ring_gemm<T, BM, BN, WM, WN, RB, R>), grid, block, 0, s, a);
}

template <typename T, int FM, int FN, int R>
void launch_wide(GemmArgs a, hipStream_t s) {
  a.mt = cdiv(a.m, 32 * FM);
  a.nt = cdiv(a.n, 32 * FN);
  hipLaunchKernelGGL((wide_gemm<T, FM, FN, R>), dim3((unsigned)(a.mt * a.nt)), dim3(256), 0, s, a);
}

template <typename T>
void launch_gemm(const GemmArgs& a, Kind kind, hipStream_t s) {
  const int left = a.m % 256;
  if (kind >= kHalf && left && left <= kFewLeft && a.m > left) {
    GemmArgs whole = a, rest = a;
    whole.m = a.m - left;
    launch_gemm<T>(whole, kind, s);
    rest.x += (int64_t)whole.m * a.x_s;
    rest.xs += whole.m;
    rest.out += (int64_t)whole.m * a.o_s * (int64_t)sizeof(T);
    rest.m = left;
    launch_gemm<T>(rest, left <= 16 ? kFew : kSome, s);
    return;
  }
  switch (kind) {
    case kFew:
      if (a.m <= 4) hipLaunchKernelGGL((few_gemm<T, 4, 3>), dim3((unsigned)cdiv(a.n, 16)), dim3(256), 0, s, a);
      else hipLaunchKernelGGL((few_gemm<T, 16, 2>), dim3((unsigned)cdiv(a.n, 16)), dim3(256), 0, s, a);
      break;
    case kSome: launch_ring<T, 64, 64, 2, 2, 256, 4>(a, s); break;
    case kMany: launch_ring<T, 128, 128, 2, 2, 128, 4>(a, s); break;
    case kHalf: launch_wide<T, 8, 4, 3>(a, s); break;
    case kMost: launch_wide<T, 8, 8, 2>(a, s); break;
  }
  if (a.splits > 1) {
    const int64_t work = (int64_t)a.m * ((a.n + 3) / 4);
    hipLaunchKernelGGL(reduce_sums<T>, dim3((unsigned)cdiv64(work, 256)), dim3(256), 0, s, a);
  }
}

}  // namespace

extern "C" int li_quantize_rows(const void* x, int64_t x_stride, void* codes, int64_t codes_stride, float* scales,
                                int rows, int k, int padded, int dtype, void* stream) {
  li::clear_error();
  if (dtype != LI_F32 && dtype != LI_F16 && dtype != LI_BF16)
    return li::fail(LI_EINVAL, "li_quantize_rows: unknown dtype %d", dtype);
  if (rows < 0 || k <= 0 || padded < k || codes_stride < padded)
    return li::fail(LI_EINVAL, "li_quantize_rows: bad extents (%d, %d, %d)", rows, k, padded);
  if (rows == 0) return LI_OK;
  if (!x || !codes || !scales) return li::fail(LI_EINVAL, "li_quantize_rows: null pointer");
  if ((reinterpret_cast<uintptr_t>(codes) & 7) || codes_stride % 8 || padded % 8)
    return li::fail(LI_EINVAL, "li_quantize_rows: rows of codes must be 8-byte aligned and padded");
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == LI_F32) launch_quantize<float>(x, x_stride, codes, codes_stride, scales, rows, k, padded, s);
  else if (dtype == LI_F16) launch_quantize<li_f16>(x, x_stride, codes, codes_stride, scales, rows, k, padded, s);
  else launch_quantize<li_bf16>(x, x_stride, codes, codes_stride, scales, rows, k, padded, s);
  return li::check_launch("li_quantize_rows");
}

extern "C" int li_linear_int8_plan(int m, int n, int k, size_t* workspace_bytes) {
  li::clear_error();
  if (int rc = check_extents("li_linear_int8_plan", m, n, k)) return rc;
  if (workspace_bytes) *workspace_bytes = m ? space_of(m, n, k).need : 0;
  return LI_OK;
}

extern "C" int li_linear_int8(const void* x, int64_t x_stride, const void* w, int64_t w_stride, const float* w_scales,
                              void* out, int64_t out_stride, int m, int n, int k, void* workspace,
                              size_t workspace_bytes, int dtype, void* stream) {
  li::clear_error();
  const int esize = li::dtype_size(dtype);
  if (dtype != LI_F32 && dtype != LI_F16 && dtype != LI_BF16)
    return li::fail(LI_EINVAL, "li_linear_int8: unknown dtype %d", dtype);
  if (int rc = check_extents("li_linear_int8", m, n, k)) return rc;
  if (m == 0) return LI_OK;
  if (!x || !w || !w_scales || !out) return li::fail(LI_EINVAL, "li_linear_int8: null pointer");
  if (!li::aligned16(w) || w_stride % 16 || w_stride < (k + 15) / 16 * 16)
    return li::fail(LI_EINVAL, "li_linear_int8: rows of w must start at multiples of 16 bytes and be padded to them");
  if (out_stride < n || x_stride < 0) return li::fail(LI_EINVAL, "li_linear_int8: rows overlap");
  const Plan p = plan_of(m, n, k);
  const Space sp = space_of(m, n, k);
  if (!workspace || !li::aligned16(workspace) || workspace_bytes < sp.need)
    return li::fail(LI_EWORKSPACE, "li_linear_int8: workspace of %zu bytes given, %zu needed", workspace_bytes, sp.need);
  if ((int64_t)cdiv(m, p.bm) * cdiv(n, p.bn) * p.splits > 0x7fffffffLL)
    return li::fail(LI_EUNSUPPORTED, "li_linear_int8: %d x %d outputs are too many tiles", m, n);
  char* wp = static_cast<char*>(workspace);
  float* xs = reinterpret_cast<float*>(wp + sp.scales);
  if (int rc = li_quantize_rows(x, x_stride, wp, sp.x_s, xs, m, k, (int)sp.x_s, dtype, stream)) return rc;
  GemmArgs a{};
  a.x = wp;
  a.xs = xs;
  a.w = static_cast<const char*>(w);
  a.ws = w_scales;
  a.out = static_cast<char*>(out);
  a.part = reinterpret_cast<int32_t*>(wp + sp.part);
  a.x_s = sp.x_s;
  a.w_s = w_stride;
  a.o_s = out_stride;
  a.m = m;
  a.n = n;
  a.k = k;
  a.splits = p.splits;
  a.vec = n % 4 == 0 && out_stride % 4 == 0 && (reinterpret_cast<uintptr_t>(out) % (4 * esize)) == 0;
  a.rows16 = out_stride % 8 == 0 && li::aligned16(out);
  hipStream_t s = static_cast<hipStream_t>(stream);
  // (The large tiles reach their rows by 32-bit offsets.)
  const Kind kind = p.kind >= kHalf && w_stride > kWideStride ? kMany : p.kind;
  if (dtype == LI_F32) launch_gemm<float>(a, kind, s);
  else if (dtype == LI_F16) launch_gemm<li_f16>(a, kind, s);
  else launch_gemm<li_bf16>(a, kind, s);
  return li::check_launch("li_linear_int8");
}
