// What the two attention kernels over the paged 8-bit KV cache share: their parameters, the list of key tiles that is dealt
// to the CTAs in equal shares, and the merge of results that were cut.
//
// A unit is (request, KV head, ROWS query rows): the heads of a group, for each of the request's query tokens.  Its keys, as
// far as its last row sees them, are cut into tiles of TILE; all tiles of all units are one list (request, head, rows, keys),
// and CTA c takes entries [c, c + 1) * ceil(total / CTAs) of it, so ragged lengths need no plan on the host.  In front of a
// unit's tiles the list has unit_cost() entries without work, for what a unit costs besides (its query, its merge).  With one, two,
// three and four of them: decode of 160 requests of 1 to 4100 keys 23.1, 22.7, 24.2, 24.3 us; drafts of 32 requests 79.5, 70.0,
// 67.7, 69.4; chunks and single tokens in one batch at D 256 87.6, 82.7, 79.0, 79.4.  A CTA can hold
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
  uint32_t g_mul, g_shift;                    // division by g (set_group)
  float scale_log2;                           // scaling * log2(e)
  void* out;                                  // [tokens, H, D]
  float* lse;                                 // [tokens, H] or null
  int4* cut;                                  // [CTAs] the unit that a CTA began and did not finish: first row, head, rows, pieces
  float *ws_m, *ws_l, *ws_acc;                // [2 * CTAs][ROWS] partial results
  int* status;
};

// i / g for 0 <= i < 2^31: with 2^shift the next power of two from g on, i / g = (i + hi(i * mul)) >> shift for
// mul = floor(2^32 (2^shift - g) / g) + 1 (division by an invariant integer by multiplication).
inline void set_group(PagedParams& p, int g) {
  p.g = g;
  p.g_shift = 0;
  while ((1ll << p.g_shift) < g) ++p.g_shift;
  p.g_mul = (uint32_t)(((1ull << 32) * ((1ull << p.g_shift) - (uint64_t)g)) / (uint64_t)g + 1);
}
__device__ __forceinline__ int token_of(const PagedParams& p, int i) {
  return (int)((__umulhi((uint32_t)i, p.g_mul) + (uint32_t)i) >> p.g_shift);
}

__host__ __device__ constexpr int unit_cost(int rows) { return rows <= 8 ? 2 : 3; }

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
  __device__ __forceinline__ int seen(const PagedParams& p, int i) const { return len - n + 1 + token_of(p, i); }
  // keys that the last row of a unit sees, in keys and in tiles: one at least, so that every unit is in the list
  __device__ __forceinline__ int limit(const PagedParams& p, int row_tile) const {
    return max(seen(p, row_tile * ROWS + rows(p, row_tile) - 1), 0);
  }
  __device__ __forceinline__ int tiles(const PagedParams& p, int row_tile) const {
    return max((limit(p, row_tile) + TILE - 1) / TILE, 1);
  }
  __device__ __forceinline__ int64_t head_entries(const PagedParams& p) const {
    int64_t sum = (int64_t)unit_cost(ROWS) * row_tiles;
#pragma unroll 1
    for (int j = 0; j < row_tiles; ++j) sum += tiles(p, j);
    return sum;
  }
};

// The rest of a CTA's share, segment by segment: open() gives tiles [from, to) of a unit, close() goes on to the next one.
template <int ROWS, int TILE>
struct Walk {
  static constexpr int kUnitCost = unit_cost(ROWS);
  Request<ROWS, TILE> q;
  int r, head, row_tile, entry, tiles;        // entry: -kUnitCost .. -1 without work, then the unit's tiles
  int from, to;
  int64_t left;                               // entries

  __device__ __forceinline__ bool open() {
    if (left <= 0) return false;
    const int take = (int)min((int64_t)(tiles - entry), left);
    left -= take;
    from = max(entry, 0);
    to = entry + take;
    return to > 0;                            // else the share ends in front of the unit's tiles
  }
  __device__ __forceinline__ void close(const PagedParams& p) {
    if (left <= 0) return;
    entry = -kUnitCost;
    if (++row_tile >= q.row_tiles) {
      row_tile = 0;
      if (++head >= p.hk) {
        head = 0;
        do {
          if (++r >= p.requests) {            // not within a share
            left = 0;
            return;
          }
          q = Request<ROWS, TILE>(p, r);
        } while (q.row_tiles == 0);
      }
    }
    tiles = q.tiles(p, row_tile);
  }
  __device__ __forceinline__ bool whole() const { return from == 0 && to == tiles; }
};

// The share of this CTA; returns the entries of a full share.  All threads; `list` has THREADS / 32 + 2 words of shared memory.
template <int THREADS, int ROWS, int TILE>
__device__ __forceinline__ int64_t deal_tiles(const PagedParams& p, int64_t* list, Walk<ROWS, TILE>& at) {
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
    return r < p.requests ? p.hk * Request<ROWS, TILE>(p, r).head_entries(p) : 0;
  };
  constexpr int kUnitCost = unit_cost(ROWS);
  // a thread has `each` requests in a row
  const int each = (p.requests + THREADS - 1) / THREADS, r0 = tid * each;
  int64_t mine = 0, before;
  if (each == 1) {
    mine = weight(r0);
  } else {
#pragma unroll 1
    for (int i = 0; i < each; ++i) mine += weight(r0 + i);
  }
  const int64_t total = block_sum(mine, before);
  const int64_t share = (total + gridDim.x - 1) / gridDim.x, begin = (int64_t)blockIdx.x * share;
  at.left = min(total, begin + share) - begin;
  if (at.left <= 0) return share;
  if (begin >= before && begin < before + mine) {
    int r = r0;
    int64_t rest = begin - before;
    if (each > 1) {
#pragma unroll 1
      for (int64_t w; rest >= (w = weight(r)); ++r) rest -= w;
    }
    list[kW] = r;
    list[kW + 1] = rest;
  }
  __syncthreads();
  at.r = (int)list[kW];
  at.q = Request<ROWS, TILE>(p, at.r);
  int64_t rest = list[kW + 1];
  at.head = 0;
  if (at.q.row_tiles == 1) {                  // the common case without a 64-bit division
    at.row_tile = 0;
    at.tiles = at.q.tiles(p, 0);
    const int unit = at.tiles + kUnitCost;
    if (rest >= unit) {
      at.head = (int)((uint64_t)rest >> 31 ? rest / unit : (int)rest / unit);
      rest -= (int64_t)at.head * unit;
    }
  } else {
    const int64_t per_head = at.q.head_entries(p);
    at.head = (int)(rest / per_head);
    rest %= per_head;
    at.row_tile = 0;
#pragma unroll 1
    while ((at.tiles = at.q.tiles(p, at.row_tile)) + kUnitCost <= rest) {
      rest -= at.tiles + kUnitCost;
      ++at.row_tile;
    }
  }
  at.entry = (int)rest - kUnitCost;
  return share;
}
// pieces of a unit whose first tiles are this segment, the CTA's first one or not
template <int ROWS, int TILE>
__device__ __forceinline__ int4 cut_unit(const PagedParams& p, const Walk<ROWS, TILE>& u, int64_t share, bool first) {
  return make_int4(u.q.t0 * p.g + u.row_tile * ROWS, u.head, u.q.rows(p, u.row_tile),
                   1 + (int)((u.tiles - u.to + share - 1) / share) + (first ? 1 << 30 : 0));
}

__device__ __forceinline__ float ex2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Product of a query row's scale and a key's, at most the largest float: with inf a score that is 0 would become NaN.
__device__ __forceinline__ float scale_product(float a, float b) {
  float y;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a * b), "f"(3.402823466e38f));
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
__device__ __forceinline__ int64_t out_row(const PagedParams& p, int i, int head) {
  const int t = token_of(p, i);
  return (int64_t)t * (p.hk * p.g) + head * p.g + (i - t * p.g);
}
// query row of row i of the request whose tokens begin at t0
template <typename T>
__device__ __forceinline__ const T* query_row(const PagedParams& p, int t0, int i, int head) {
  const int t = token_of(p, i);
  return static_cast<const T*>(p.q) + (t0 + t) * p.sqt + (head * p.g + (i - t * p.g)) * p.sqh;
}
// log-sum-exp of a sum relative to 2^top
__device__ __forceinline__ float lse_of(float top, float sum) { return sum == 0.0f ? -INFINITY : (top + log2f(sum)) * kLn2; }

// Rows of no request, and of requests without keys: zeros and -inf.  The rows in front of the first request and behind the
// last one may be most of a captured step's, so all CTAs take part: a call of 32 single tokens and 8160 such rows
// of H 32 D 128 (67 MB) takes 66 us, and took 1078 with one.
template <typename T, int D, int ROWS, int TILE>
__device__ __forceinline__ void clear_untouched(const PagedParams& p) {
  const int h = p.hk * p.g;
  auto clear = [&](int64_t t0, int64_t t1, int64_t first, int64_t step) {    // tokens t0 .. t1 - 1 by threads first, first + step, ...
    constexpr int kRow = D * sizeof(T) / 16;
#pragma unroll 1
    for (int64_t i = t0 * h * kRow + first; i < t1 * h * kRow; i += step) static_cast<uint4*>(p.out)[i] = make_uint4(0, 0, 0, 0);
    if (p.lse != nullptr) {
#pragma unroll 1
      for (int64_t i = t0 * h + first; i < t1 * h; i += step) p.lse[i] = -INFINITY;
    }
  };
  if (p.cu != nullptr) {
    auto inside = [&](int t) { return min(max((int64_t)t, (int64_t)0), p.tokens); };
    const int64_t front = inside(p.cu[0]), behind = inside(p.cu[p.requests]);
    const int64_t first = (int64_t)blockIdx.x * blockDim.x + threadIdx.x, step = (int64_t)gridDim.x * blockDim.x;
#pragma unroll 1
    for (int x = 0; x < 2; ++x) clear(x == 0 ? 0 : behind, x == 0 ? front : p.tokens, first, step);
  }
#pragma unroll 1
  for (int r = (int)blockIdx.x; r < p.requests; r += gridDim.x) {
    const Request<ROWS, TILE> q(p, r);
    if (q.len == 0) clear(q.t0, q.t0 + q.n, threadIdx.x, blockDim.x);
  }
}

// Exact merge of the pieces of a cut unit, L lanes a row, in the order of the keys.  Bound by trips to L2: the maxima, sums
// and rows of up to four pieces are asked for at once.  Pieces lie row by row, a warp a row; or (kColumns) four columns of
// all rows behind each other, as threads that have a row each store them, two rows a warp, so that sectors are whole.
constexpr int kCombineWarps = 4;
template <typename T, int D, int ROWS, bool kColumns>
__global__ void __launch_bounds__(32 * kCombineWarps) paged_combine_kernel(PagedParams p) {
  griddep_wait();
  griddep_launch();
  constexpr int L = kColumns ? 16 : 32;
  const int lane = threadIdx.x % L, row = (int)(blockIdx.y * blockDim.x + threadIdx.x) / L;
  const int4 u = p.cut[blockIdx.x];
  if (row >= u.z) return;
  const int pieces = u.w & ((1 << 30) - 1), first = 2 * (int)blockIdx.x + (u.w >> 30 ? 0 : 1);
  auto slot = [&](int i) { return (int64_t)(i == 0 ? first : 2 * ((int)blockIdx.x + i)); };
  constexpr int kAtOnce = 4, kC = D / (4 * L);
  float top = -INFINITY, total = 0.0f, sum[kC][4];
#pragma unroll
  for (int c = 0; c < kC; ++c)
#pragma unroll
    for (int k = 0; k < 4; ++k) sum[c][k] = 0.0f;
  for (int i0 = 0; i0 < pieces; i0 += kAtOnce) {
    float m[kAtOnce], l[kAtOnce];
    float4 v[kAtOnce][kC];
#pragma unroll
    for (int x = 0; x < kAtOnce; ++x) {
      const int64_t a = slot(min(i0 + x, pieces - 1)) * ROWS;                // behind the last piece: that one again, not counted
      m[x] = p.ws_m[a + row];
      l[x] = p.ws_l[a + row];
#pragma unroll
      for (int c = 0; c < kC; ++c) {
        const int four = c * L + lane;
        v[x][c] = *(reinterpret_cast<const float4*>(p.ws_acc + a * D) + (kColumns ? four * ROWS + row : row * (D / 4) + four));
      }
    }
    float now = top;
#pragma unroll
    for (int x = 0; x < kAtOnce; ++x) now = fmaxf(now, m[x]);
    const float ref = now == -INFINITY ? 0.0f : now;
    const float f = top == -INFINITY ? 1.0f : ex2_approx(top - ref);         // no key so far: zeros, or NaN
    total *= f;
#pragma unroll
    for (int c = 0; c < kC; ++c)
#pragma unroll
      for (int k = 0; k < 4; ++k) sum[c][k] *= f;
#pragma unroll
    for (int x = 0; x < kAtOnce; ++x) {
      if (i0 + x >= pieces) break;
      const float g = m[x] == -INFINITY ? 1.0f : ex2_approx(m[x] - ref);
      total += g * l[x];
#pragma unroll
      for (int c = 0; c < kC; ++c) {
        sum[c][0] += g * v[x][c].x;
        sum[c][1] += g * v[x][c].y;
        sum[c][2] += g * v[x][c].z;
        sum[c][3] += g * v[x][c].w;
      }
    }
    top = now;
  }
  const int64_t row_out = out_row(p, u.x + row, u.y);
  const float inv = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
  for (int c = 0; c < kC; ++c) {
#pragma unroll
    for (int k = 0; k < 4; ++k) sum[c][k] *= inv;
    store4<T>(static_cast<T*>(p.out) + row_out * D + (c * L + lane) * 4, sum[c]);
  }
  if (lane == 0 && p.lse != nullptr) p.lse[row_out] = lse_of(top, total);
}
template <typename T, int D, int ROWS, bool kColumns>
int launch_combine(const PagedParams& p, int grid, cudaStream_t st) {
  const int64_t rows = p.cu == nullptr ? p.g : p.tokens * p.g;
  constexpr int kRowsBlock = kCombineWarps * (kColumns ? 2 : 1);
  return launch("nvfp4_kv8_attention combine", paged_combine_kernel<T, D, ROWS, kColumns>,
                dim3(grid, (unsigned)(((rows < ROWS ? rows : ROWS) + kRowsBlock - 1) / kRowsBlock)), 32 * kCombineWarps, 0, st, p);
}

// ---- the kernel for long chunks (paged_chunk.cu)
constexpr int64_t paged_slot_bytes(int64_t rows, int64_t d) { return 2 * rows * (d + 2) * 4 + 16; }      // of a CTA
inline int64_t paged_chunk_rows(int d) { return d == 128 ? 256 : 128; }
int launch_paged_chunk(const PagedParams& p, int q_dtype, int d, int ctas, cudaStream_t st);

}  // namespace nvfp4
