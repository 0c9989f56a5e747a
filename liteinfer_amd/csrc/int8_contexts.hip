// An int8 pool's contexts laid out in the query's 16-bit type, for a packed
// pass.
//
// The query blocks of a chunk all read its context's keys and values, each
// stage of them from LDS on the matrix cores in 16 bits. Converting a stage
// where it is folded would convert it once for every (query block of 256
// rows) and stand in the way of the softmax, which is what bounds the
// ping-pong kernel next to its MFMAs; converting each context once, before
// the pass, costs 1 + 2 + 2 bytes a value of memory traffic instead of 1:
// 6,144 queries over 3 x 10,240 keys (32 / 8 heads, head_dim 128) take
// this kernel a few percent of the pass. Every value is code * scale in fp32,
// rounded to the type, as the dense kernels gather it.
//
// A work-group takes tiles of kTileKeys consecutive positions of one
// sequence, all heads, K and V: 16 codes (16 bytes) a thread and step, read
// and written in the order they lie in. Which sequence a tile belongs to is
// found by a scan of the sequences' lengths, 64 at a time, in every wave.
// Bound by memory.
#include "li_attention.h"

namespace li {
namespace {

constexpr int kTileKeys = 16;
constexpr int kThreads = 256;
constexpr int kMaxGroups = 4096;

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
};

// Positions of a sequence that are laid out.
__device__ __forceinline__ int copied_keys(const CopyArgs& a, int seq) {
  const int nq = a.qsl[seq + 1] - a.qsl[seq];
  const int c = a.ctx[seq];
  if (nq < 1 || (nq == 1 && a.rows_elsewhere)) return 0;
  return min(max(c, 0), a.max_context);
}

template <typename T>
__device__ __forceinline__ void widen(const u32x4_t x, float scale, T* dst) {
  u32x4_t out[2];
#pragma unroll
  for (int u = 0; u < 8; ++u) {
    const uint32_t w = x[u / 2] >> (16 * (u % 2));
    out[u / 4][u % 4] = li_pack2<T>((float)(int)(int8_t)w * scale, (float)(int)(int8_t)(w >> 8) * scale);
  }
  reinterpret_cast<u32x4_t*>(dst)[0] = out[0];
  reinterpret_cast<u32x4_t*>(dst)[1] = out[1];
}

template <typename T>
__global__ __launch_bounds__(kThreads) void copy_contexts(CopyArgs a) {
  const int lane = (int)(threadIdx.x & 63);
  const int per_row = a.head_dim / 16;  // 16-code steps of a head's row
  const int steps = a.num_kv_heads * per_row;
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
    for (int e = threadIdx.x; e < count * steps; e += kThreads) {
      const int key = e / steps, rem = e - key * steps;
      const int64_t r = row0 + key;
      if (r >= a.capacity) continue;
      const int h = rem / per_row, c = rem - h * per_row;
      const uint32_t slot = (uint32_t)slots[key];
      const int64_t at = (int64_t)(slot / (uint32_t)a.block_size) * a.sc_s + h;
      const int64_t src = (int64_t)slot * a.p_s0 + h * a.p_s1 + 16 * c;
      const u32x4_t k = *reinterpret_cast<const u32x4_t*>(a.kp + src), v = *reinterpret_cast<const u32x4_t*>(a.vp + src);
      const float ks = a.ks[at], vs = a.vs[at];
      const int64_t dst = (r * a.num_kv_heads + h) * a.head_dim + 16 * c;
      widen<T>(k, ks, static_cast<T*>(a.keys) + dst);
      widen<T>(v, vs, static_cast<T*>(a.values) + dst);
    }
  }
}

}  // namespace

bool copy_contexts_applies(const AttnArgs& a) {
  return a.head_dim % 16 == 0 && aligned16(a.kp) && aligned16(a.vp) && a.p_s0 % 16 == 0 && a.p_s1 % 16 == 0;
}

int launch_copy_contexts(const AttnArgs& a, int dtype, bool rows_elsewhere, int64_t capacity, void* keys, void* values,
                         int64_t* table, hipStream_t s) {
  if (dtype != LI_BF16 && dtype != LI_F16) return fail(LI_EINVAL, "copy_contexts: 16-bit types only");
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
  const int64_t tiles = cdiv64(capacity, kTileKeys) + a.batch;  // (each sequence's last may be partial)
  const dim3 grid((unsigned)std::min<int64_t>(tiles, kMaxGroups)), block(kThreads);
  if (dtype == LI_BF16) hipLaunchKernelGGL(copy_contexts<li_bf16>, grid, block, 0, s, c);
  else hipLaunchKernelGGL(copy_contexts<li_f16>, grid, block, 0, s, c);
  return check_launch("copy_contexts");
}

}  // namespace li
