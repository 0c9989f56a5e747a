// An int8 pool's contexts laid out in fp16, for a packed pass.
//
// The query blocks of a chunk all read its context's keys and values, each
// stage of them from LDS on the matrix cores in 16 bits. Converting a stage
// where it is folded would convert it once for every (query block of 256
// rows) and stand in the way of the softmax, which is what bounds the
// ping-pong kernel next to its MFMAs; converting each context once, before
// the pass, costs 1 + 2 + 2 bytes a value of memory traffic instead of 1.
//
// fp16 keeps 11 bits of code * scale where bf16 keeps 8, but reaches from
// 2^-24 to 65504 only. So K and V are divided by a power of two for each
// sequence and KV head, found from the largest scale s < 2^(e + 1) of the
// blocks the context lies in (a value is at most 128 s):
//     V by 2^(e - 7), to at most 2^15: values down to 2^-29 of the largest
//       keep all 11 bits;
//     K by 2^(e + 4), to at most 2^4: the query takes the power, and what
//       falls below fp16 of either moves a score by 2^-14 at most.
// The query and the output are multiplied by the same powers. Each division
// is exact (scales are multiplied by the inverse), each value rounded once.
//
// Where V's scale is not finite, the row of K is laid out as NaN and V's as
// zeros: who reads the key gets a NaN weight, and so the NaN in every dim that
// V would give, while a query in front of it, for whom the key is masked, does
// not multiply its weight of zero by a NaN.
//
// Two launches, both bound by memory and its latency. largest_scales:
// work-groups take kThreads positions of a sequence each (kParts of them at
// most) and keep the largest scale of each head of the blocks they lie in.
// copy_contexts: a work-group takes tiles of kTileKeys consecutive positions
// of one sequence, all heads, K and V: 16 codes (16 bytes) a thread and step, read and written in the order they lie in. Which
// sequence a tile belongs to is found by a scan of the sequences' lengths, 64
// at a time, in every wave.
//
// Three chunks of 2,048 over 8,192 keys (32 / 8 heads, head_dim 128, 190 MB
// moved) take 8 + 44 us here of 820; 101 over 4,096 (head_dim 64) 7 + 9 of 44,
// all latency.
#include "li_attention.h"

namespace li {
namespace {

constexpr int kTileKeys = 16;
constexpr int kUnroll = 4;  // steps of a thread whose codes are in flight
constexpr int kThreads = 256;
constexpr int kMaxGroups = 4096;
constexpr int kParts = 64;
constexpr int kMaxHeads = 1024;  // (their scales are held in LDS)
constexpr uint32_t kInfBits = 0x7f800000u;

struct CopyArgs {
  const int8_t* kp;
  const int8_t* vp;
  int64_t p_s0, p_s1;
  const float* ks;
  const float* vs;
  int64_t sc_s;
  int block_size;
  const int64_t* st;
  int64_t st_s;
  const int32_t* ctx;
  const int32_t* qsl;
  int batch, num_kv_heads, head_dim, max_context;
  int rows_elsewhere;
  int64_t capacity;
  void* keys;
  void* values;
  int64_t* table;
  float2* units;
  uint32_t* largest;  // [batch][parts][2 (K, V)][num_kv_heads], a scale's bits
  int parts;
};

// Positions of a sequence that are laid out.
__device__ __forceinline__ int copied_keys(const CopyArgs& a, int seq) {
  const int nq = a.qsl[seq + 1] - a.qsl[seq];
  const int c = a.ctx[seq];
  if (nq < 1 || (nq == 1 && a.rows_elsewhere)) return 0;
  return min(max(c, 0), a.max_context);
}

__device__ __forceinline__ void widen(const u32x4_t x, float scale, li_f16* dst) {
  u32x4_t out[2];
#pragma unroll
  for (int u = 0; u < 8; ++u) {
    const uint32_t w = x[u / 2] >> (16 * (u % 2));
    out[u / 4][u % 4] = li_pack2<li_f16>((float)(int)(int8_t)w * scale, (float)(int)(int8_t)(w >> 8) * scale);
  }
  reinterpret_cast<u32x4_t*>(dst)[0] = out[0];
  reinterpret_cast<u32x4_t*>(dst)[1] = out[1];
}

__device__ __forceinline__ void fill(uint32_t two, li_f16* dst) {
  const u32x4_t x = {two, two, two, two};
  reinterpret_cast<u32x4_t*>(dst)[0] = x;
  reinterpret_cast<u32x4_t*>(dst)[1] = x;
}

// The exponent e (biased) of a scale s < 2^(e + 1), held where every power
// below is a normal number.
__device__ __forceinline__ int exponent_of(uint32_t bits) { return min(max((int)(bits >> 23), 32), 249); }
__device__ __forceinline__ float power(int biased) { return __uint_as_float((uint32_t)biased << 23); }
// What K (col < heads) or V is multiplied by, and the inverse.
__device__ __forceinline__ float inverse_unit(uint32_t bits, bool of_v) {
  const int e = exponent_of(bits);
  return power(of_v ? 261 - e : 250 - e);
}
__device__ __forceinline__ float unit_of(uint32_t bits, bool of_v) {
  const int e = exponent_of(bits);
  return power(of_v ? e - 7 : e + 4);
}

// Largest scales of a part of a sequence's blocks (those that are not finite
// aside: their values are not either, whatever they are divided by). A thread
// that holds the first position of a run in one block reads its scales.
__global__ __launch_bounds__(kThreads) void largest_scales(CopyArgs a) {
  extern __shared__ uint32_t top[];  // [2 num_kv_heads]
  const int seq = (int)(blockIdx.x / (unsigned)a.parts), part = (int)(blockIdx.x % (unsigned)a.parts);
  const int tid = threadIdx.x, cols = 2 * a.num_kv_heads;
  const int keys = copied_keys(a, seq);
  const int64_t* slots = a.st + (int64_t)seq * a.st_s;
  for (int c = tid; c < cols; c += kThreads) top[c] = 0;
  __syncthreads();
  for (int64_t p = (int64_t)part * kThreads + tid; p < keys; p += (int64_t)a.parts * kThreads) {
    const uint32_t block = (uint32_t)slots[p] / (uint32_t)a.block_size;
    if (tid > 0 && (uint32_t)slots[p - 1] / (uint32_t)a.block_size == block) continue;
    const float* ks = a.ks + (int64_t)block * a.sc_s;
    const float* vs = a.vs + (int64_t)block * a.sc_s;
#pragma unroll 4
    for (int h = 0; h < a.num_kv_heads; ++h) {
      const uint32_t k = __float_as_uint(ks[h]) & 0x7fffffffu, v = __float_as_uint(vs[h]) & 0x7fffffffu;
      if (k < kInfBits) atomicMax(&top[h], k);
      if (v < kInfBits) atomicMax(&top[a.num_kv_heads + h], v);
    }
  }
  __syncthreads();
  uint32_t* out = a.largest + (int64_t)blockIdx.x * cols;
  for (int c = tid; c < cols; c += kThreads) out[c] = top[c];
}

__global__ __launch_bounds__(kThreads) void copy_contexts(CopyArgs a) {
  extern __shared__ uint32_t top[];  // [2 num_kv_heads]: of sequence `held`
  const int lane = (int)(threadIdx.x & 63);
  const int per_row = a.head_dim / 16;  // 16-code steps of a head's row
  const int steps = a.num_kv_heads * per_row;
  const int cols = 2 * a.num_kv_heads;
  int held = -1;
  for (int64_t tile = blockIdx.x;; tile += gridDim.x) {
    // The sequence holding tile `tile`, its first tile and its first row.
    int64_t tiles_before = 0, rows_before = 0;
    int seq = -1, keys = 0;
    for (int s0 = 0; s0 < a.batch && seq < 0; s0 += 64) {
      const int c = s0 + lane < a.batch ? copied_keys(a, s0 + lane) : 0;
      int64_t t_incl = (c + kTileKeys - 1) / kTileKeys, r_incl = c;
      const int64_t t_own = t_incl, r_own = r_incl;
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) {
        const int64_t t_up = __shfl_up(t_incl, off, 64), r_up = __shfl_up(r_incl, off, 64);
        if (lane >= off) {
          t_incl += t_up;
          r_incl += r_up;
        }
      }
      const uint64_t hit = __ballot(tiles_before + t_incl > tile);
      const int at = hit ? __ffsll((long long)hit) - 1 : 63;
      const int64_t t_last = __shfl(t_incl, at, 64), r_last = __shfl(r_incl, at, 64);
      if (hit) {
        seq = s0 + at;
        keys = __shfl(c, at, 64);
        tiles_before += t_last - __shfl(t_own, at, 64);
        rows_before += r_last - __shfl(r_own, at, 64);
      } else {
        tiles_before += t_last;
        rows_before += r_last;
      }
    }
    if (seq < 0) return;  // past the last tile
    const int p0 = (int)(tile - tiles_before) * kTileKeys;
    const int count = min(kTileKeys, keys - p0);
    const int64_t* slots = a.st + (int64_t)seq * a.st_s + p0;
    const int64_t row0 = rows_before + p0;
    if ((int)threadIdx.x < count) {
      const int64_t r = row0 + threadIdx.x;
      a.table[(int64_t)seq * a.max_context + p0 + threadIdx.x] = r < a.capacity ? r : 0;
    }
    for (int e0 = 0; e0 < count * steps; e0 += kUnroll * kThreads) {
      u32x4_t k[kUnroll], v[kUnroll];
      float ks[kUnroll], vs[kUnroll];
      int head[kUnroll];
      int64_t dst[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int e = e0 + u * kThreads + (int)threadIdx.x;
        const int key = e / steps, rem = e - key * steps;
        const int64_t r = row0 + key;
        dst[u] = -1;
        if (e >= count * steps || r >= a.capacity) continue;
        const int h = rem / per_row, c = rem - h * per_row;
        const uint32_t slot = (uint32_t)slots[key];
        const int64_t at = (int64_t)(slot / (uint32_t)a.block_size) * a.sc_s + h;
        const int64_t src = (int64_t)slot * a.p_s0 + h * a.p_s1 + 16 * c;
        k[u] = *reinterpret_cast<const u32x4_t*>(a.kp + src);
        v[u] = *reinterpret_cast<const u32x4_t*>(a.vp + src);
        ks[u] = a.ks[at];
        vs[u] = a.vs[at];
        head[u] = h;
        dst[u] = (r * a.num_kv_heads + h) * a.head_dim + 16 * c;
      }
      // The sequence's largest scales, joined while the codes come.
      if (seq != held) {
        const uint32_t* of = a.largest + (int64_t)seq * a.parts * cols;
        __syncthreads();
        for (int c = threadIdx.x; c < cols; c += kThreads) top[c] = 0;
        __syncthreads();
        for (int e = threadIdx.x; e < a.parts * cols; e += kThreads) atomicMax(&top[e % cols], of[e]);
        __syncthreads();
        held = seq;
        if (p0 == 0) {
          for (int h = threadIdx.x; h < a.num_kv_heads; h += kThreads)
            a.units[(int64_t)seq * a.num_kv_heads + h] =
                float2{unit_of(top[h], false), unit_of(top[a.num_kv_heads + h], true)};
        }
      }
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        if (dst[u] < 0) continue;
        li_f16* kd = static_cast<li_f16*>(a.keys) + dst[u];
        li_f16* vd = static_cast<li_f16*>(a.values) + dst[u];
        if ((__float_as_uint(vs[u]) & 0x7fffffffu) < kInfBits) {
          widen(k[u], ks[u] * inverse_unit(top[head[u]], false), kd);
          widen(v[u], vs[u] * inverse_unit(top[a.num_kv_heads + head[u]], true), vd);
        } else {
          fill(0x7e007e00u, kd);
          fill(0u, vd);
        }
      }
    }
  }
}

}  // namespace

bool copy_contexts_applies(const AttnArgs& a) {
  return a.head_dim % 16 == 0 && a.num_kv_heads <= kMaxHeads && aligned16(a.kp) && aligned16(a.vp) && a.p_s0 % 16 == 0 && a.p_s1 % 16 == 0;
}

static int parts_of(int max_context) { return std::max(1, std::min(kParts, cdiv(max_context, kThreads))); }

size_t context_units_scratch(int batch, int num_kv_heads, int max_context) {
  return (size_t)batch * parts_of(max_context) * 2 * num_kv_heads * sizeof(uint32_t);
}

int launch_copy_contexts(const AttnArgs& a, bool rows_elsewhere, int64_t capacity, void* keys, void* values,
                         int64_t* table, float2* units, uint32_t* largest, hipStream_t s) {
  CopyArgs c{};
  c.kp = static_cast<const int8_t*>(a.kp);
  c.vp = static_cast<const int8_t*>(a.vp);
  c.p_s0 = a.p_s0;
  c.p_s1 = a.p_s1;
  c.ks = a.ks;
  c.vs = a.vs;
  c.sc_s = a.sc_s;
  c.block_size = a.block_size;
  c.st = a.st;
  c.st_s = a.st_s;
  c.ctx = a.ctx;
  c.qsl = a.qsl;
  c.batch = a.batch;
  c.num_kv_heads = a.num_kv_heads;
  c.head_dim = a.head_dim;
  c.max_context = a.max_context;
  c.rows_elsewhere = rows_elsewhere;
  c.capacity = capacity;
  c.keys = keys;
  c.values = values;
  c.table = table;
  c.units = units;
  c.largest = largest;
  c.parts = parts_of(a.max_context);
  const size_t lds = 2 * (size_t)a.num_kv_heads * sizeof(uint32_t);
  const dim3 block(kThreads);
  hipLaunchKernelGGL(largest_scales, dim3((unsigned)(a.batch * c.parts)), block, lds, s, c);
  if (int rc = check_launch("largest_scales")) return rc;
  const int64_t tiles = cdiv64(capacity, kTileKeys) + a.batch;  // (each sequence's last may be partial)
  hipLaunchKernelGGL(copy_contexts, dim3((unsigned)std::min<int64_t>(tiles, kMaxGroups)), block, lds, s, c);
  return check_launch("copy_contexts");
}

}  // namespace li
