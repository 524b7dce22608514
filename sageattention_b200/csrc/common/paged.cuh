// What the two attention kernels over the paged 8-bit KV cache share: their parameters, the list of key tiles that is dealt
// to the CTAs in equal shares, and the merge of results that were cut.
//
// A unit is (request, KV head, ROWS query rows): the heads of a group, for each of the request's query tokens.  Its keys, as
// far as its last row sees them, are cut into tiles of TILE; all tiles of all units are one list (request, head, rows, keys),
// and CTA c takes tiles [c, c + 1) * ceil(total / CTAs) of it, so ragged lengths need no plan on the host.  A CTA can hold
// the end of one unit and the beginning of another, each a partial result of its own (slots 2 c and 2 c + 1).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>
#include "fp4.cuh"
#include "launch.cuh"

namespace nvfp4 {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct PagedParams {
  const void* q;
  int64_t sqt, sqh;                           // element strides of token and head
  const int32_t* cu;                          // [requests + 1] first query token, or null: one token a request
  int64_t tokens;
  const uint8_t *k, *v;
  int64_t k_block, v_block;                   // bytes from block to block
  const float *ks, *vs;
  int64_t ks_block, vs_block;
  const int32_t* table;
  int64_t table_row;
  const int32_t* lengths;
  int requests, width, blocks, log_block, hk, g;
  float scale_log2;                           // scaling * log2(e)
  void* out;                                  // [tokens, H, D]
  float* lse;                                 // [tokens, H] or null
  int4* cut;                                  // [CTAs] the unit that a CTA began and did not finish: first row, head, rows, pieces
  float *ws_m, *ws_l, *ws_acc;                // [2 * CTAs][ROWS] partial results
  int* status;
};

// What a request asks for: its query tokens [t0, t0 + n), its keys, its units.
template <int ROWS, int TILE>
struct Request {
  int t0, n, len, row_tiles;

  __device__ __forceinline__ Request() {}
  __device__ __forceinline__ Request(const PagedParams& p, int r) {
    if (p.cu == nullptr) {
      t0 = r;
      n = 1;
    } else {
      const int64_t a = min(max((int64_t)p.cu[r], (int64_t)0), p.tokens), b = min((int64_t)p.cu[r + 1], p.tokens);
      t0 = (int)a;
      n = (int)max(b - a, (int64_t)0);
    }
    len = (int)min((int64_t)max(p.lengths[r], 0), (int64_t)p.width << p.log_block);
    row_tiles = len == 0 ? 0 : (int)(((int64_t)n * p.g + ROWS - 1) / ROWS);
  }
  __device__ __forceinline__ int rows(const PagedParams& p, int row_tile) const { return min(n * p.g - row_tile * ROWS, ROWS); }
  // keys that row i of the request sees
  __device__ __forceinline__ int seen(const PagedParams& p, int i) const { return len - n + 1 + i / p.g; }
  // keys that the last row of a unit sees, in keys and in tiles: one at least, so that every unit is in the list
  __device__ __forceinline__ int limit(const PagedParams& p, int row_tile) const {
    return max(seen(p, row_tile * ROWS + rows(p, row_tile) - 1), 0);
  }
  __device__ __forceinline__ int tiles(const PagedParams& p, int row_tile) const {
    return max((limit(p, row_tile) + TILE - 1) / TILE, 1);
  }
  __device__ __forceinline__ int64_t head_tiles(const PagedParams& p) const {
    int64_t sum = 0;
    for (int j = 0; j < row_tiles; ++j) sum += tiles(p, j);
    return sum;
  }
};

// A place in the list: tile `tile` of the `tiles` of a unit.
template <int ROWS, int TILE>
struct Cursor {
  Request<ROWS, TILE> q;
  int r, head, row_tile, tile, tiles;

  __device__ __forceinline__ void next_unit(const PagedParams& p) {
    tile = 0;
    if (++row_tile >= q.row_tiles) {
      row_tile = 0;
      if (++head >= p.hk) {
        head = 0;
        do {
          if (++r >= p.requests) return;
          q = Request<ROWS, TILE>(p, r);
        } while (q.row_tiles == 0);
      }
    }
    tiles = q.tiles(p, row_tile);
  }
};

// The share of this CTA: tiles [begin, end) of the list, and the place of `begin`.  All threads; `list` has THREADS / 32 + 2
// words of shared memory.
struct Share {
  int64_t begin, end, share;
};
template <int THREADS, int ROWS, int TILE>
__device__ __forceinline__ Share deal_tiles(const PagedParams& p, int64_t* list, Cursor<ROWS, TILE>& at) {
  constexpr int kW = THREADS / 32;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  auto block_sum = [&](int64_t x, int64_t& before) -> int64_t {
    int64_t inc = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += y;
    }
    if (lane == 31) list[warp] = inc;
    __syncthreads();
    int64_t base = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kW; ++w) {
      if (w < warp) base += list[w];
      all += list[w];
    }
    __syncthreads();
    before = base + inc - x;
    return all;
  };
  auto weight = [&](int r) -> int64_t {
    return r < p.requests ? p.hk * Request<ROWS, TILE>(p, r).head_tiles(p) : 0;
  };
  // of up to THREADS requests a thread keeps its one
  const int64_t first = weight(tid);
  int64_t mine = first, before;
  for (int r = tid + THREADS; r < p.requests; r += THREADS) mine += weight(r);
  const int64_t total = block_sum(mine, before);
  Share s;
  s.share = (total + gridDim.x - 1) / gridDim.x;
  s.begin = (int64_t)blockIdx.x * s.share;
  s.end = min(total, s.begin + s.share);
  if (s.begin >= s.end) return s;
  if (tid == 0) list[kW] = -1;
  int64_t base = 0;
  for (int r0 = 0;; r0 += THREADS) {
    const int64_t w = r0 == 0 ? first : weight(r0 + tid);
    const int64_t all = block_sum(w, before);
    if (s.begin >= base + before && s.begin < base + before + w) {
      list[kW] = r0 + tid;
      list[kW + 1] = s.begin - base - before;
    }
    __syncthreads();
    if (list[kW] >= 0) break;
    base += all;
  }
  at.r = (int)list[kW];
  at.q = Request<ROWS, TILE>(p, at.r);
  const int64_t in = list[kW + 1], per_head = at.q.head_tiles(p);
  at.head = (int)(in / per_head);
  int64_t rest = in % per_head;
  at.row_tile = 0;
  while ((at.tiles = at.q.tiles(p, at.row_tile)) <= rest) {
    rest -= at.tiles;
    ++at.row_tile;
  }
  at.tile = (int)rest;
  return s;
}
// pieces of a unit that the CTA begins with `tiles` of its tiles, as its first segment or not
template <int ROWS, int TILE>
__device__ __forceinline__ int4 cut_unit(const PagedParams& p, const Cursor<ROWS, TILE>& u, int tiles, int64_t share, bool first) {
  return make_int4(u.q.t0 * p.g + u.row_tile * ROWS, u.head, u.q.rows(p, u.row_tile),
                   1 + (int)((u.tiles - tiles + share - 1) / share) + (first ? 1 << 30 : 0));
}

__device__ __forceinline__ float ex2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <typename T>
__device__ __forceinline__ void store4(T* p, const float (&x)[4]) {
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
  } else {
    *reinterpret_cast<uint2*>(p) = make_uint2(pack_16x2<T>(x[0], x[1]), pack_16x2<T>(x[2], x[3]));
  }
}
// row of `out` that row i (token * g + head of its group) of KV head `head` is
__device__ __forceinline__ int64_t out_row(const PagedParams& p, int64_t i, int head) {
  return (i / p.g) * (p.hk * p.g) + (int64_t)head * p.g + i % p.g;
}
// log-sum-exp of a sum relative to 2^top
__device__ __forceinline__ float lse_of(float top, float sum) { return sum == 0.0f ? -INFINITY : (top + log2f(sum)) * kLn2; }

// Rows of no request, and of requests without keys: zeros and -inf.
template <typename T, int D, int ROWS, int TILE>
__device__ __forceinline__ void clear_untouched(const PagedParams& p) {
  const int h = p.hk * p.g;
  auto clear = [&](int64_t t0, int64_t t1) {
    T* out = static_cast<T*>(p.out);
    for (int64_t i = t0 * h * D + threadIdx.x * 4; i < t1 * h * D; i += blockDim.x * 4) {
      const float z[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      store4<T>(out + i, z);
    }
    if (p.lse != nullptr)
      for (int64_t i = t0 * h + threadIdx.x; i < t1 * h; i += blockDim.x) p.lse[i] = -INFINITY;
  };
  for (int r = blockIdx.x; r < p.requests; r += gridDim.x) {
    const Request<ROWS, TILE> q(p, r);
    if (q.len == 0) clear(q.t0, q.t0 + q.n);
  }
  if (p.cu != nullptr && blockIdx.x == gridDim.x - 1) {
    auto inside = [&](int t) { return min(max((int64_t)t, (int64_t)0), p.tokens); };
    clear(0, inside(p.cu[0]));
    clear(inside(p.cu[p.requests]), p.tokens);
  }
}

// Exact merge of the pieces of a cut unit, one warp a row, in the order of the keys.
constexpr int kCombineWarps = 4;
template <typename T, int D, int ROWS>
__global__ void __launch_bounds__(32 * kCombineWarps) paged_combine_kernel(PagedParams p) {
  griddep_wait();
  griddep_launch();
  const int lane = threadIdx.x & 31, row = blockIdx.y * kCombineWarps + (threadIdx.x >> 5);
  const int4 u = p.cut[blockIdx.x];
  if (row >= u.z) return;
  const int pieces = u.w & ((1 << 30) - 1), first = 2 * (int)blockIdx.x + (u.w >> 30 ? 0 : 1);
  auto at = [&](int i) { return (int64_t)(i == 0 ? first : 2 * ((int)blockIdx.x + i)) * ROWS + row; };
  float top = -INFINITY;
  for (int i = lane; i < pieces; i += 32) top = fmaxf(top, p.ws_m[at(i)]);
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  float sum[D / 128][4], total = 0.0f;
#pragma unroll
  for (int c = 0; c < D / 128; ++c)
#pragma unroll
    for (int k = 0; k < 4; ++k) sum[c][k] = 0.0f;
#pragma unroll 4
  for (int i = 0; i < pieces; ++i) {
    const float f = top == -INFINITY ? 1.0f : ex2_approx(p.ws_m[at(i)] - top);        // no key: zeros, or NaN
    total += f * p.ws_l[at(i)];
#pragma unroll
    for (int c = 0; c < D / 128; ++c) {
      const float4 v = *reinterpret_cast<const float4*>(p.ws_acc + at(i) * D + c * 128 + lane * 4);
      sum[c][0] += f * v.x;
      sum[c][1] += f * v.y;
      sum[c][2] += f * v.z;
      sum[c][3] += f * v.w;
    }
  }
  const int64_t row_out = out_row(p, u.x + row, u.y);
  const float inv = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
  for (int c = 0; c < D / 128; ++c) {
#pragma unroll
    for (int k = 0; k < 4; ++k) sum[c][k] *= inv;
    store4<T>(static_cast<T*>(p.out) + row_out * D + c * 128 + lane * 4, sum[c]);
  }
  if (lane == 0 && p.lse != nullptr) p.lse[row_out] = lse_of(top, total);
}
template <typename T, int D, int ROWS>
int launch_combine(const PagedParams& p, int grid, cudaStream_t st) {
  const int64_t rows = p.cu == nullptr ? p.g : p.tokens * p.g;
  return launch("nvfp4_kv8_attention combine", paged_combine_kernel<T, D, ROWS>,
                dim3(grid, (unsigned)(((rows < ROWS ? rows : ROWS) + kCombineWarps - 1) / kCombineWarps)), 32 * kCombineWarps, 0, st, p);
}

// ---- the kernel for long chunks (paged_chunk.cu)
constexpr int64_t paged_slot_bytes(int64_t rows, int64_t d) { return 2 * rows * (d + 2) * 4 + 16; }      // of a CTA
inline int64_t paged_chunk_rows(int d) { return d == 128 ? 256 : 128; }
int launch_paged_chunk(const PagedParams& p, int q_dtype, int d, int ctas, cudaStream_t st);

}  // namespace nvfp4
