// Slot-write into an int8 paged cache with a scale for every (block of
// tokens, KV head), with the rotary embedding of q and k applied on the way
// or, as a plain scatter, without it.
//
// What a store holds. Row `slot` of KV head h stands for
//     codes[slot, h, :] * scale[slot / block_size, h],   codes in -127 .. 127,
// K and V each with scales of their own. Writing the rows W of one block:
//     old   = 0 if a row of W is the block's first, else scale[b, h]
//     new   = max(old, largest |x| over W / 127, 2^-126)
//     codes = rint(x / new)           the rows of W
//     codes = rint(codes * old / new) the block's other rows, if new > old
// so a block's scale only grows while it fills, a row is re-expressed when it
// does (each time off by at most half a step of the new scale), and writing a
// block's first slot starts it anew. A value that is not finite makes the
// scale NaN: everything the block holds for that head then reads as NaN until
// it is started anew (a code has no NaN of its own).
// All of it is fp32: the rotation
//     out[i]       = x[i] cos[i] - x[i + D/2] sin[i]
//     out[i + D/2] = x[i + D/2] cos[i + D/2] + x[i] sin[i + D/2]
// is formed in fp32 with no FMA and rounded once (q to its dtype, k to its
// code), unlike the 16-bit pools' write, which rounds every product to follow
// the separate torch ops of liteinfer/models/llama.py:85-98.
//
// Work split. The tokens of one block stand next to each other in the slot
// list (a sequence's positions are consecutive, and a block belongs to one
// sequence): a *run*. One wave takes one (run, KV head, K or V): it finds the
// run's rows by their offset in the block, loads them once, reduces the
// largest magnitude over the wave, and writes rows and scale: no two waves
// touch one scale, so nothing is atomic and nothing depends on order. A wave
// looks for runs that begin in its `span` tokens of the list. A slot named
// twice in a run keeps the later token. The q heads are rotated by the
// launch's other work-groups.
//
// Bound by launch and two dependent round trips (slots, then rows and the old
// scale) at a decode step (4 to 128 tokens, 32 / 8 heads: 6 us), by memory in
// a long pass (5,569 tokens at head_dim 128: 152 MB in 37.5 us, 4.1 TB/s where
// a copy moves 4.8).
#include "li_common.h"

#include <cmath>

namespace {

struct AppendArgs {
  const char* q;  // nullptr: a plain scatter (no rotation, no q)
  const char* k;
  const char* v;
  const char* cos;
  const char* sin;
  char* qo;
  int8_t* kp;
  int8_t* vp;
  float* kscale;
  float* vscale;
  int64_t qs[4], ks[4], vs[4], os[4];  // element strides: batch, head, token, dim
  int64_t cs[3];                        // cos / sin element strides: batch, token, dim
  int64_t tokens;                       // T
  int64_t n;                            // B * T
  const int64_t* slots;
  int64_t num_slots;
  int64_t ps_slot, ps_head;
  int64_t scale_s;  // scales: element stride of a block
  int block_size;
  int num_heads, num_kv_heads, head_dim;
  int span;             // list entries per wave
  int64_t kv_groups;    // work-groups of the K / V part
  int* bad;             // nullable: counts tokens whose slot is out of range
};

constexpr float kStep = 1.0f / 127.0f;
constexpr float kLeast = 1.17549435e-38f;  // 2^-126: 1 / new stays finite
constexpr uint32_t kInfBits = 0x7f800000u;
constexpr int kWavesPerGroup = 4;
constexpr int kPairs = 8;  // element pairs (i, i + D/2) of one lane

template <typename E>
using Vec8 = __attribute__((__vector_size__(8 * sizeof(E)), __aligned__(16))) E;

__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// Largest magnitude as fp32 bits: infinities and NaNs order above every
// finite value, so a maximum over the bits keeps them.
__device__ __forceinline__ uint32_t wave_max_bits(uint32_t v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, off, 64));
  return v;
}

// What writing rows of largest magnitude `largest` does to a block of scale
// `held` (both as bits: the sources build with -fno-honor-nans, under which a
// NaN in a float select or compare need not survive).
struct Growth {
  uint32_t bits;  // the new scale
  bool lost;      // it is a NaN: the rows' codes are 0, the others stay
  bool grown;     // the other rows are re-expressed, times `ratio`
  float inv, ratio;
};
__device__ __forceinline__ Growth grow(uint32_t held, bool anew, uint32_t largest) {
  Growth g;
  const uint32_t before = anew ? 0u : held;
  g.lost = largest >= kInfBits || (before & 0x7fffffffu) > kInfBits;
  const float old = __uint_as_float(g.lost ? 0u : before);
  const float now = fmaxf(old, fmaxf(__uint_as_float(g.lost ? 0u : largest) * kStep, kLeast));
  g.bits = g.lost ? 0x7fc00000u : __float_as_uint(now);
  g.grown = !g.lost && now > old;
  g.inv = 1.f / now;
  g.ratio = old * g.inv;
  return g;
}

__device__ __forceinline__ int code_of(float x, float inv) {
  return (int)fminf(fmaxf(rintf(x * inv), -127.f), 127.f);
}

__device__ __forceinline__ uint32_t pack4(int a, int b, int c, int d) {
  return (uint32_t)(a & 255) | (uint32_t)(b & 255) << 8 | (uint32_t)(c & 255) << 16 | (uint32_t)(d & 255) << 24;
}

// Four codes re-expressed with a larger scale.
__device__ __forceinline__ uint32_t requant4(uint32_t w, float ratio) {
  int c[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) c[e] = (int)rintf((float)(int)(int8_t)(w >> (8 * e)) * ratio);
  return pack4(c[0], c[1], c[2], c[3]);
}

__device__ __forceinline__ void rotate(float lo, float hi, float c_lo, float s_lo, float c_hi, float s_hi,
                                       float& out_lo, float& out_hi) {
#pragma clang fp contract(off)  // as the formula: two products, then their sum
  const float a = lo * c_lo, b = hi * s_lo, c = hi * c_hi, d = lo * s_hi;
  out_lo = a - b;
  out_hi = c + d;
}

// This wave's next run that begins in list entries [i, end): its first entry
// (-1: none), its block, and, in win[o], the last list entry that names
// offset o of the block (-1: none). The list's entries out of range are
// passed over. Every lane calls it and gets the same answer.
__device__ __forceinline__ int64_t find_run(const AppendArgs& a, int64_t i, int64_t end, int* win, uint32_t& block) {
  const int lane = (int)(threadIdx.x & 63);
  const uint32_t bs = (uint32_t)a.block_size;
  auto slot_at = [&](int64_t t) -> int64_t {
    const int64_t s = t < a.n ? a.slots[t] : -1;
    return s < a.num_slots ? s : -1;
  };
  for (; i < end; ++i) {
    const int64_t slot = slot_at(i);
    if (slot < 0) continue;
    block = (uint32_t)slot / bs;
    int64_t p = i - 1;
    int64_t before = -1;
    while (p >= 0 && (before = slot_at(p)) < 0) --p;
    if (p >= 0 && (uint32_t)before / bs == block) continue;  // inside a run that began earlier
    for (int o = lane; o < a.block_size; o += 64) win[o] = -1;
    __builtin_amdgcn_wave_barrier();
    // 64 entries at a time, until a valid one of another block.
    for (int64_t t0 = i; t0 < a.n; t0 += 64) {
      const int64_t s = slot_at(t0 + lane);
      const bool valid = s >= 0;
      const uint32_t b = valid ? (uint32_t)s / bs : 0;
      const uint64_t other = __ballot(valid && b != block);
      const int stop = other ? __ffsll((long long)other) - 1 : 64;
      if (valid && lane < stop) atomicMax(&win[(uint32_t)s - block * bs], (int)(t0 + lane));
      if (other) break;
    }
    __builtin_amdgcn_wave_barrier();
    return i;
  }
  return -1;
}

// One lane's pairs [8 c, 8 c + 8) of a row, rotated if the row is K's.
template <typename E, bool kRope>
__device__ __forceinline__ void load_pairs(const AppendArgs& a, bool is_k, int64_t t, int h, int c, float (&lo)[kPairs],
                                           float (&hi)[kPairs]) {
  const int half = a.head_dim / 2, d0 = kPairs * c;
  const int64_t b = t / a.tokens, tt = t - b * a.tokens;
  const E* src = is_k ? reinterpret_cast<const E*>(a.k) + b * a.ks[0] + h * a.ks[1] + tt * a.ks[2] + d0
                      : reinterpret_cast<const E*>(a.v) + b * a.vs[0] + h * a.vs[1] + tt * a.vs[2] + d0;
  const Vec8<E> x = *reinterpret_cast<const Vec8<E>*>(src), y = *reinterpret_cast<const Vec8<E>*>(src + half);
  if (kRope && is_k) {
    const E* cr = reinterpret_cast<const E*>(a.cos) + b * a.cs[0] + tt * a.cs[1] + d0;
    const E* sr = reinterpret_cast<const E*>(a.sin) + b * a.cs[0] + tt * a.cs[1] + d0;
    const Vec8<E> cl = *reinterpret_cast<const Vec8<E>*>(cr), ch = *reinterpret_cast<const Vec8<E>*>(cr + half);
    const Vec8<E> sl = *reinterpret_cast<const Vec8<E>*>(sr), sh = *reinterpret_cast<const Vec8<E>*>(sr + half);
#pragma unroll
    for (int e = 0; e < kPairs; ++e)
      rotate(li_to_float(x[e]), li_to_float(y[e]), li_to_float(cl[e]), li_to_float(sl[e]), li_to_float(ch[e]),
             li_to_float(sh[e]), lo[e], hi[e]);
  } else {
#pragma unroll
    for (int e = 0; e < kPairs; ++e) {
      lo[e] = li_to_float(x[e]);
      hi[e] = li_to_float(y[e]);
    }
  }
}

// Rows with a contiguous last axis, 16-byte aligned, head_dim a multiple of
// 16: D / 16 lanes per row, rows_per = 64 / (D / 16) rows at a time. The
// first kHold rounds of a block's rows stay in registers between the maximum
// and the codes; a block of more rows reads the others again (they are in the
// cache by then).
template <typename E, bool kRope>
__device__ __forceinline__ void append_run_vec(const AppendArgs& a, const int* win, uint32_t block, int h, bool is_k) {
  constexpr int kHold = 2;
  const int lane = (int)(threadIdx.x & 63);
  const int half = a.head_dim / 2;
  const int per_row = half / kPairs, rows_per = 64 / per_row;
  const int c = lane % per_row, r0 = lane / per_row;
  const bool idle = r0 >= rows_per;
  const int bs = a.block_size;
  uint32_t* scale = reinterpret_cast<uint32_t*>((is_k ? a.kscale : a.vscale) + (int64_t)block * a.scale_s + h);
  const uint32_t held = *scale;
  int8_t* codes = (is_k ? a.kp : a.vp) + (int64_t)block * bs * a.ps_slot + h * a.ps_head + kPairs * c;

  float lo[kHold][kPairs], hi[kHold][kPairs];
  uint32_t largest = 0;
  auto fold = [&](const float (&x)[kPairs], const float (&y)[kPairs]) {
#pragma unroll
    for (int e = 0; e < kPairs; ++e) largest = max(largest, max(abs_bits(x[e]), abs_bits(y[e])));
  };
  auto token = [&](int o) -> int { return !idle && o < bs ? win[o] : -1; };
#pragma unroll
  for (int u = 0; u < kHold; ++u) {
    const int t = token(u * rows_per + r0);
    if (t >= 0) {
      load_pairs<E, kRope>(a, is_k, t, h, c, lo[u], hi[u]);
      fold(lo[u], hi[u]);
    }
  }
  for (int o = kHold * rows_per + r0; o < bs; o += rows_per) {
    const int t = token(o);
    if (t < 0) continue;
    float x[kPairs], y[kPairs];
    load_pairs<E, kRope>(a, is_k, t, h, c, x, y);
    fold(x, y);
  }
  largest = wave_max_bits(largest);

  const bool anew = win[0] >= 0;
  const Growth g = grow(held, anew, largest);

  auto store = [&](int o, const float (&x)[kPairs], const float (&y)[kPairs]) {
    int8_t* row = codes + o * a.ps_slot;
    int cx[kPairs], cy[kPairs];
#pragma unroll
    for (int e = 0; e < kPairs; ++e) {
      cx[e] = g.lost ? 0 : code_of(x[e], g.inv);
      cy[e] = g.lost ? 0 : code_of(y[e], g.inv);
    }
    *reinterpret_cast<uint2*>(row) = uint2{pack4(cx[0], cx[1], cx[2], cx[3]), pack4(cx[4], cx[5], cx[6], cx[7])};
    *reinterpret_cast<uint2*>(row + half) = uint2{pack4(cy[0], cy[1], cy[2], cy[3]), pack4(cy[4], cy[5], cy[6], cy[7])};
  };
  auto again = [&](int o) {  // a row that is not written
    if (!g.grown) return;
    uint2* p0 = reinterpret_cast<uint2*>(codes + o * a.ps_slot);
    uint2* p1 = reinterpret_cast<uint2*>(codes + o * a.ps_slot + half);
    uint2 x = {0u, 0u}, y = {0u, 0u};
    if (!anew) {
      x = *p0;
      y = *p1;
      x = uint2{requant4(x.x, g.ratio), requant4(x.y, g.ratio)};
      y = uint2{requant4(y.x, g.ratio), requant4(y.y, g.ratio)};
    }
    *p0 = x;
    *p1 = y;
  };
#pragma unroll
  for (int u = 0; u < kHold; ++u) {
    const int o = u * rows_per + r0;
    if (idle || o >= bs) continue;
    if (win[o] >= 0) store(o, lo[u], hi[u]);
    else again(o);
  }
  for (int o = kHold * rows_per + r0; o < bs; o += rows_per) {
    const int t = token(o);
    if (idle) break;
    if (t < 0) {
      again(o);
      continue;
    }
    float x[kPairs], y[kPairs];
    load_pairs<E, kRope>(a, is_k, t, h, c, x, y);
    store(o, x, y);
  }
  if (lane == 0) *scale = g.bits;
}

// One pair of a row with any strides.
template <typename E, bool kRope>
__device__ __forceinline__ void load_pair(const AppendArgs& a, bool is_k, int64_t t, int h, int d, float& lo, float& hi) {
  const int half = a.head_dim / 2;
  const int64_t b = t / a.tokens, tt = t - b * a.tokens;
  const int64_t* st = is_k ? a.ks : a.vs;
  const E* src = reinterpret_cast<const E*>(is_k ? a.k : a.v) + b * st[0] + h * st[1] + tt * st[2];
  lo = li_to_float(src[d * st[3]]);
  hi = li_to_float(src[(d + half) * st[3]]);
  if (kRope && is_k) {
    const E* cr = reinterpret_cast<const E*>(a.cos) + b * a.cs[0] + tt * a.cs[1];
    const E* sr = reinterpret_cast<const E*>(a.sin) + b * a.cs[0] + tt * a.cs[1];
    float x, y;
    rotate(lo, hi, li_to_float(cr[d * a.cs[2]]), li_to_float(sr[d * a.cs[2]]), li_to_float(cr[(d + half) * a.cs[2]]),
           li_to_float(sr[(d + half) * a.cs[2]]), x, y);
    lo = x;
    hi = y;
  }
}

// Any strides and any even head_dim: lanes take element pairs, rows one after
// the other, each read twice. (The last element of an odd head_dim, which only
// a scatter can have, is in no pair.)
template <typename E, bool kRope>
__device__ __forceinline__ void append_run_elem(const AppendArgs& a, const int* win, uint32_t block, int h, bool is_k) {
  const int lane = (int)(threadIdx.x & 63);
  const int half = a.head_dim / 2, bs = a.block_size;
  const bool odd = a.head_dim & 1;  // scatters only
  uint32_t* scale = reinterpret_cast<uint32_t*>((is_k ? a.kscale : a.vscale) + (int64_t)block * a.scale_s + h);
  const uint32_t held = *scale;
  int8_t* codes = (is_k ? a.kp : a.vp) + (int64_t)block * bs * a.ps_slot + h * a.ps_head;
  auto last = [&](int t) -> float {  // the last element of an odd row
    const int64_t b = t / a.tokens, tt = t - b * a.tokens;
    const int64_t* st = is_k ? a.ks : a.vs;
    return li_to_float(reinterpret_cast<const E*>(is_k ? a.k : a.v)[b * st[0] + h * st[1] + tt * st[2] +
                                                                     (a.head_dim - 1) * st[3]]);
  };
  uint32_t largest = 0;
  for (int o = 0; o < bs; ++o) {
    const int t = win[o];
    if (t < 0) continue;
    for (int d = lane; d < half; d += 64) {
      float x, y;
      load_pair<E, kRope>(a, is_k, t, h, d, x, y);
      largest = max(largest, max(abs_bits(x), abs_bits(y)));
    }
    if (odd) largest = max(largest, abs_bits(last(t)));
  }
  largest = wave_max_bits(largest);
  const bool anew = win[0] >= 0;
  const Growth g = grow(held, anew, largest);
  for (int o = 0; o < bs; ++o) {
    const int t = win[o];
    int8_t* row = codes + o * a.ps_slot;
    if (t < 0) {
      if (g.grown)
        for (int d = lane; d < a.head_dim; d += 64) row[d] = anew ? 0 : (int8_t)(int)rintf((float)row[d] * g.ratio);
      continue;
    }
    for (int d = lane; d < half; d += 64) {
      float x, y;
      load_pair<E, kRope>(a, is_k, t, h, d, x, y);
      row[d] = (int8_t)(g.lost ? 0 : code_of(x, g.inv));
      row[d + half] = (int8_t)(g.lost ? 0 : code_of(y, g.inv));
    }
    if (odd && lane == 0) row[a.head_dim - 1] = (int8_t)(g.lost ? 0 : code_of(last(t), g.inv));
  }
  if (lane == 0) *scale = g.bits;
}

// K / V work-groups first, then the rotation of q. Wave u of the K / V part
// takes list entries [span * c, span * (c + 1)) for KV head h of K or V, with
// u = (c * 2 + kind) * heads + h.
template <typename E, bool kRope, bool kVec>
__global__ __launch_bounds__(64 * kWavesPerGroup) void append_int8(AppendArgs a) {
  extern __shared__ int win_of[];
  const int lane = (int)(threadIdx.x & 63);
  if ((int64_t)blockIdx.x < a.kv_groups) {
    const int wave = (int)(threadIdx.x >> 6);
    int* win = win_of + wave * a.block_size;
    const int64_t u = (int64_t)blockIdx.x * kWavesPerGroup + wave;
    const int h = (int)(u % a.num_kv_heads);
    const bool is_k = (u / a.num_kv_heads) % 2 == 0;
    const int64_t begin = u / a.num_kv_heads / 2 * a.span;
    if (begin >= a.n) return;
    const int64_t end = min(begin + a.span, a.n);
    if (h == 0 && is_k && a.bad) {
      int missed = 0;
      for (int64_t t = begin + lane; t < end; t += 64) missed += a.slots[t] < 0 || a.slots[t] >= a.num_slots;
#pragma unroll
      for (int off = 32; off > 0; off >>= 1) missed += __shfl_xor(missed, off, 64);
      if (missed && lane == 0) atomicAdd(a.bad, missed);
    }
    uint32_t block;
    for (int64_t i = begin; (i = find_run(a, i, end, win, block)) >= 0; ++i) {
      if constexpr (kVec) append_run_vec<E, kRope>(a, win, block, h, is_k);
      else append_run_elem<E, kRope>(a, win, block, h, is_k);
      __builtin_amdgcn_wave_barrier();  // win is read before the next run's is made
    }
    return;
  }
  if constexpr (kRope) {
    const int half = a.head_dim / 2;
    const int pairs = kVec ? half / kPairs : half;
    const int64_t per_token = (int64_t)a.num_heads * pairs;
    const int64_t total = a.n * per_token;
    const int64_t stride = (int64_t)(gridDim.x - a.kv_groups) * blockDim.x;
    for (int64_t w = ((int64_t)blockIdx.x - a.kv_groups) * blockDim.x + threadIdx.x; w < total; w += stride) {
      // (32-bit divisions while the work fits them.)
      const int64_t t = total < (int64_t)1 << 31 ? (int64_t)((uint32_t)w / (uint32_t)per_token) : w / per_token;
      const int rem = (int)(w - t * per_token);
      const int h = rem / pairs, c = rem - h * pairs;
      const int64_t b = t / a.tokens, tt = t - b * a.tokens;
      const int64_t so = b * a.qs[0] + h * a.qs[1] + tt * a.qs[2], to = b * a.os[0] + h * a.os[1] + tt * a.os[2];
      const int64_t co = b * a.cs[0] + tt * a.cs[1];
      if constexpr (kVec) {
        const int d0 = kPairs * c;
        const E* src = reinterpret_cast<const E*>(a.q) + so + d0;
        const E* cr = reinterpret_cast<const E*>(a.cos) + co + d0;
        const E* sr = reinterpret_cast<const E*>(a.sin) + co + d0;
        E* dst = reinterpret_cast<E*>(a.qo) + to + d0;
        const Vec8<E> x = *reinterpret_cast<const Vec8<E>*>(src), y = *reinterpret_cast<const Vec8<E>*>(src + half);
        const Vec8<E> cl = *reinterpret_cast<const Vec8<E>*>(cr), ch = *reinterpret_cast<const Vec8<E>*>(cr + half);
        const Vec8<E> sl = *reinterpret_cast<const Vec8<E>*>(sr), sh = *reinterpret_cast<const Vec8<E>*>(sr + half);
        Vec8<E> lo, hi;
#pragma unroll
        for (int e = 0; e < kPairs; ++e) {
          float l, m;
          rotate(li_to_float(x[e]), li_to_float(y[e]), li_to_float(cl[e]), li_to_float(sl[e]), li_to_float(ch[e]),
                 li_to_float(sh[e]), l, m);
          lo[e] = li_from_float<E>(l);
          hi[e] = li_from_float<E>(m);
        }
        *reinterpret_cast<Vec8<E>*>(dst) = lo;
        *reinterpret_cast<Vec8<E>*>(dst + half) = hi;
      } else {
        const E* src = reinterpret_cast<const E*>(a.q) + so;
        const E* cr = reinterpret_cast<const E*>(a.cos) + co;
        const E* sr = reinterpret_cast<const E*>(a.sin) + co;
        E* dst = reinterpret_cast<E*>(a.qo) + to;
        const int64_t d = c, e = c + half;
        float l, m;
        rotate(li_to_float(src[d * a.qs[3]]), li_to_float(src[e * a.qs[3]]), li_to_float(cr[d * a.cs[2]]),
               li_to_float(sr[d * a.cs[2]]), li_to_float(cr[e * a.cs[2]]), li_to_float(sr[e * a.cs[2]]), l, m);
        dst[d * a.os[3]] = li_from_float<E>(l);
        dst[e * a.os[3]] = li_from_float<E>(m);
      }
    }
  }
}

// Whether every row is 16-byte aligned with a contiguous last axis (codes:
// 8-byte halves).
bool vec_ok(const AppendArgs& a, int esize) {
  if (a.head_dim % (2 * kPairs) != 0 || a.head_dim > 2 * kPairs * 64) return false;
  auto ok = [&](const char* p, const int64_t* st, int dims) {
    if (!li::aligned16(p) || st[dims - 1] != 1) return false;
    for (int j = 0; j < dims - 1; ++j)
      if ((st[j] * esize) % 16 != 0) return false;
    return true;
  };
  if (!ok(a.k, a.ks, 4) || !ok(a.v, a.vs, 4)) return false;
  if (a.q && (!ok(a.q, a.qs, 4) || !ok(a.qo, a.os, 4) || !ok(a.cos, a.cs, 3) || !ok(a.sin, a.cs, 3))) return false;
  return (reinterpret_cast<uintptr_t>(a.kp) & 7) == 0 && (reinterpret_cast<uintptr_t>(a.vp) & 7) == 0 &&
         a.ps_slot % 8 == 0 && a.ps_head % 8 == 0;
}

template <typename E, bool kRope>
void launch(const AppendArgs& a, bool vec, unsigned grid, hipStream_t s) {
  const size_t lds = (size_t)kWavesPerGroup * a.block_size * sizeof(int);
  const dim3 block(64 * kWavesPerGroup);
  if (vec) hipLaunchKernelGGL((append_int8<E, kRope, true>), dim3(grid), block, lds, s, a);
  else hipLaunchKernelGGL((append_int8<E, kRope, false>), dim3(grid), block, lds, s, a);
}

// Entries of the list that one wave looks for runs in: one while the waves
// of entries that begin no run cost less than the runs one wave takes one
// after the other.
constexpr int64_t kSingleEntries = 1024;
constexpr int kSpan = 16;

int append_impl(const char* who, AppendArgs& a, int64_t batch, int dtype, hipStream_t s) {
  const int esize = li::dtype_size(dtype);
  if (esize == 0 || dtype == LI_FP8_E4M3) return li::fail(LI_EINVAL, "%s: unknown dtype %d", who, dtype);
  if (batch < 0 || a.tokens < 0 || a.num_kv_heads <= 0 || a.head_dim <= 0 || a.num_slots < 0 ||
      (a.q && a.num_heads <= 0))
    return li::fail(LI_EINVAL, "%s: negative or empty extent", who);
  if (a.block_size < 1 || a.block_size > LI_INT8_MAX_BLOCK)
    return li::fail(LI_EUNSUPPORTED, "%s: blocks of %d slots are outside 1..%d", who, a.block_size, LI_INT8_MAX_BLOCK);
  if (a.num_slots % a.block_size != 0)
    return li::fail(LI_EINVAL, "%s: %lld slots are no whole blocks of %d", who, (long long)a.num_slots, a.block_size);
  if (a.num_slots >= (int64_t)1 << 31)
    return li::fail(LI_EUNSUPPORTED, "%s: %lld slots, int8 pools hold fewer than 2^31", who, (long long)a.num_slots);
  a.n = batch * a.tokens;
  if (a.n == 0) return LI_OK;
  if (a.n >= (int64_t)1 << 30) return li::fail(LI_EUNSUPPORTED, "%s: %lld tokens are too many", who, (long long)a.n);
  if (!a.k || !a.v || !a.slots || !a.kp || !a.vp || !a.kscale || !a.vscale)
    return li::fail(LI_EINVAL, "%s: null pointer", who);
  if (a.ps_head < a.head_dim || a.ps_slot < (int64_t)a.num_kv_heads * a.head_dim)
    return li::fail(LI_EINVAL, "%s: pool strides (%lld, %lld) overlap rows of %d x %d", who, (long long)a.ps_slot,
                    (long long)a.ps_head, a.num_kv_heads, a.head_dim);
  if (a.scale_s < a.num_kv_heads)
    return li::fail(LI_EINVAL, "%s: a scale stride of %lld overlaps rows of %d heads", who, (long long)a.scale_s,
                    a.num_kv_heads);
  a.span = a.n <= kSingleEntries ? 1 : kSpan;
  const int64_t waves = li::cdiv64(a.n, a.span) * 2 * a.num_kv_heads;
  a.kv_groups = li::cdiv64(waves, kWavesPerGroup);
  const bool vec = vec_ok(a, esize);
  int64_t grid = a.kv_groups;
  if (a.q) {
    const int64_t work = a.n * a.num_heads * (vec ? a.head_dim / 2 / kPairs : a.head_dim / 2);
    grid += std::min<int64_t>(li::cdiv64(work, 64 * kWavesPerGroup), 65536);
  }
  if (grid > 0x7fffffffLL) return li::fail(LI_EUNSUPPORTED, "%s: a grid of %lld work-groups is too large", who, (long long)grid);
  if (a.q) {
    if (dtype == LI_F32) launch<float, true>(a, vec, (unsigned)grid, s);
    else if (dtype == LI_BF16) launch<li_bf16, true>(a, vec, (unsigned)grid, s);
    else launch<li_f16, true>(a, vec, (unsigned)grid, s);
  } else {
    if (dtype == LI_F32) launch<float, false>(a, vec, (unsigned)grid, s);
    else if (dtype == LI_BF16) launch<li_bf16, false>(a, vec, (unsigned)grid, s);
    else launch<li_f16, false>(a, vec, (unsigned)grid, s);
  }
  return li::check_launch(who);
}

}  // namespace

extern "C" int li_kv_scatter_int8(const void* k, const void* v, const int64_t* k_strides, const int64_t* v_strides,
                                  int64_t batch, int64_t tokens, const int64_t* slots, void* key_pool,
                                  void* value_pool, float* key_scales, float* value_scales, int64_t num_slots,
                                  int block_size, int64_t pool_stride_slot, int64_t pool_stride_head,
                                  int64_t scale_stride_block, int num_kv_heads, int head_dim, int src_dtype,
                                  int32_t* bad_slots, void* stream) {
  li::clear_error();
  if (!k_strides || !v_strides) return li::fail(LI_EINVAL, "li_kv_scatter_int8: strides must not be null");
  AppendArgs a{};
  a.k = static_cast<const char*>(k);
  a.v = static_cast<const char*>(v);
  for (int j = 0; j < 4; ++j) {
    a.ks[j] = k_strides[j];
    a.vs[j] = v_strides[j];
  }
  a.kp = static_cast<int8_t*>(key_pool);
  a.vp = static_cast<int8_t*>(value_pool);
  a.kscale = key_scales;
  a.vscale = value_scales;
  a.tokens = tokens;
  a.slots = slots;
  a.num_slots = num_slots;
  a.ps_slot = pool_stride_slot;
  a.ps_head = pool_stride_head;
  a.scale_s = scale_stride_block;
  a.block_size = block_size;
  a.num_kv_heads = num_kv_heads;
  a.head_dim = head_dim;
  a.bad = bad_slots;
  return append_impl("li_kv_scatter_int8", a, batch, src_dtype, static_cast<hipStream_t>(stream));
}

extern "C" int li_rope_kv_write_int8(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides,
                                     const void* v, const int64_t* v_strides, const void* cos, const void* sin,
                                     const int64_t* cs_strides, int64_t batch, int64_t tokens, const int64_t* slots,
                                     void* q_out, const int64_t* q_out_strides, void* key_pool, void* value_pool,
                                     float* key_scales, float* value_scales, int64_t num_slots, int block_size,
                                     int64_t pool_stride_slot, int64_t pool_stride_head, int64_t scale_stride_block,
                                     int num_heads, int num_kv_heads, int head_dim, int dtype, int32_t* bad_slots,
                                     void* stream) {
  li::clear_error();
  if (!q_strides || !k_strides || !v_strides || !cs_strides || !q_out_strides)
    return li::fail(LI_EINVAL, "li_rope_kv_write_int8: strides must not be null");
  if (head_dim % 2 != 0) return li::fail(LI_EINVAL, "li_rope_kv_write_int8: head_dim %d is odd", head_dim);
  if (batch * tokens > 0 && (!q || !q_out || !cos || !sin))
    return li::fail(LI_EINVAL, "li_rope_kv_write_int8: null pointer");
  AppendArgs a{};
  a.q = static_cast<const char*>(q);
  a.k = static_cast<const char*>(k);
  a.v = static_cast<const char*>(v);
  a.cos = static_cast<const char*>(cos);
  a.sin = static_cast<const char*>(sin);
  a.qo = static_cast<char*>(q_out);
  for (int j = 0; j < 4; ++j) {
    a.qs[j] = q_strides[j];
    a.ks[j] = k_strides[j];
    a.vs[j] = v_strides[j];
    a.os[j] = q_out_strides[j];
  }
  for (int j = 0; j < 3; ++j) a.cs[j] = cs_strides[j];
  a.kp = static_cast<int8_t*>(key_pool);
  a.vp = static_cast<int8_t*>(value_pool);
  a.kscale = key_scales;
  a.vscale = value_scales;
  a.tokens = tokens;
  a.slots = slots;
  a.num_slots = num_slots;
  a.ps_slot = pool_stride_slot;
  a.ps_head = pool_stride_head;
  a.scale_s = scale_stride_block;
  a.block_size = block_size;
  a.num_heads = num_heads;
  a.num_kv_heads = num_kv_heads;
  a.head_dim = head_dim;
  a.bad = bad_slots;
  return append_impl("li_rope_kv_write_int8", a, batch, dtype, static_cast<hipStream_t>(stream));
}
