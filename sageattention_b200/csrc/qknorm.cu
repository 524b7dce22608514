// RMS norm of every head's queries and keys and their rotation by position, in one pass; and its backward pass.
//
//   r = 1 / sqrt(mean(x^2) + eps),  n = x r,  y = rot_p(n w)            rot_p: element i with element i + D/2, by angle i of position p
//   g' = rot_p^-1(dy),  dw = sum over rows g' n,  dx = r (g' w - n mean(g' w n))
//
// What bounds it: HBM; a row is read once and written once (backward: two reads, a write).  A row is D/16 lanes, each with eight
// elements of either half, so that a rotation stays within a lane and every access is 16 bytes wide; a warp has rows of several
// heads of a token (a step), STEPS steps together, for which it loads cos and sin once.  Statistics, rotation and weight
// gradients are fp32, two an instruction, rounded once to the type of the operand.  Squares are fp32 too: a row whose mean square is
// beyond it (values of 2^60) becomes 0, one whose squares vanish in it (below 2^-74) has eps alone.
//
// Forward: tasks of queries and keys by turns, so that what is in flight lies together, on the blocks that are resident at once: 16001
// tokens of H 32 Hk 8 D 128 in bf16 (views of a projection, 328 MB) 61.6 us, a copy of as many bytes 51.  On the same buffers
// again and again (16384 tokens) 57.2; all queries first 61.8; more blocks than resident 58 to 64; four steps a task 63, as there
// are fewer warps.  fp32 rows are twice as many registers, so a task is one step (8000 tokens 61.9 us, with two steps and 216 bytes of spills
// 76.8; 4000 of H 16 Hk 4 D 256 41.6, 46.8; 32 tokens 2.5, 3.4).  More under way does not help (rows asked into L2 a task ahead 63.6 instead of 61.6, two ahead 64.2), nor do
// loads past L1 (63.3) or stores that L2 gives up first (62.4).
// Backward: registers hold too few rows for the loads to stay under way (104 us with four steps, 110 with two), so a warp's rows
// come by bulk copies, the next task's while this one's are used, and a block is of queries or of keys, whose sums it keeps: 16384
// tokens, 503 MB, 84.9 us, an addition of two tensors of that size 73 (queries first, then keys, in every block: 90.8; three stages
// 96, four warps a block 87.5; tasks of keys that do not fill a stage 88.8; the forward pass by bulk copies 60.5 instead of 57.2).
#include <limits.h>
#include "common/abi.cuh"
#include "common/fp4.cuh"
#include "common/launch.cuh"
#include "common/pairs.cuh"
#include "common/sm100.cuh"

namespace nvfp4 {
namespace {

// One of the two operands: queries or keys.
struct Operand {
  const void* x;
  const void* g;                               // incoming gradient (backward)
  void* y;                                     // result, or gradient of x
  int64_t xz, xs, xh, gz, gs, gh, yz, ys, yh;  // element strides of batch entry, token, head
  const void* w;
  int heads, log_heads;                        // rows of a step: 2^log_heads heads of a token, the others are further tokens
  int steps;                                   // of a token in a task; tasks whose tokens take fewer have more of them, one after the other
  uint32_t chunks;                             // so many tasks have all heads of their tokens
  uint32_t tasks;
};
struct NormParams {
  Operand o[2];
  const float *cs, *sn;                        // [table_rows, D/2]
  int64_t table_rows, pos0, pos_batch;
  const int32_t* positions;                    // of token s of entry z: [z * pos_batch + s], or null: pos0 + s
  uint32_t tokens, s;                          // z * s, s
  int w_fp32;
  float eps;
  uint32_t key_blocks;                         // backward: blocks that have keys
  int stage_bytes;                             // of a task's rows and angles
  float* part;                                 // [blocks][D] sums of the weights' gradients, the queries' blocks first
  int* status;
};

template <typename T, int D>
struct Shape {
  static constexpr int kLanes = D / 16;        // of a row
  static constexpr int kRows = 32 / kLanes;    // of a step
  static constexpr int kRowBytes = D * sizeof(T);
};

__device__ __forceinline__ uint64_t pair_of(float lo, float hi) { return pair(__float_as_uint(lo), __float_as_uint(hi)); }
__device__ __forceinline__ float low(uint64_t v) { return __uint_as_float((uint32_t)v); }
__device__ __forceinline__ float high(uint64_t v) { return __uint_as_float((uint32_t)(v >> 32)); }
__device__ __forceinline__ uint64_t minus(uint64_t v) { return v ^ 0x8000000080000000ull; }
template <typename T> __device__ __forceinline__ uint64_t pair_of_16x2(uint32_t w);
template <> __device__ __forceinline__ uint64_t pair_of_16x2<__nv_bfloat16>(uint32_t w) { return pair(w << 16, w & 0xFFFF0000u); }
template <> __device__ __forceinline__ uint64_t pair_of_16x2<__half>(uint32_t w) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
  return pair_of(f.x, f.y);
}
__device__ __forceinline__ uint4 lds_v4(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}

// Eight elements as they lie, and as pairs.
template <typename T>
struct Eight {
  uint4 v[8 * sizeof(T) / 16];
  __device__ __forceinline__ void zero() {
    for (uint4& x : v) x = make_uint4(0, 0, 0, 0);
  }
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < (int)(sizeof(v) / 16); ++i) v[i] = reinterpret_cast<const uint4*>(p)[i];
  }
  __device__ __forceinline__ void load(uint32_t shared) {
#pragma unroll
    for (int i = 0; i < (int)(sizeof(v) / 16); ++i) v[i] = lds_v4(shared + i * 16);
  }
  __device__ __forceinline__ void pairs(uint64_t (&x)[4]) const {
    if constexpr (sizeof(T) == 4) {
      x[0] = pair(v[0].x, v[0].y);
      x[1] = pair(v[0].z, v[0].w);
      x[2] = pair(v[1].x, v[1].y);
      x[3] = pair(v[1].z, v[1].w);
    } else {
      x[0] = pair_of_16x2<T>(v[0].x);
      x[1] = pair_of_16x2<T>(v[0].y);
      x[2] = pair_of_16x2<T>(v[0].z);
      x[3] = pair_of_16x2<T>(v[0].w);
    }
  }
};
template <typename T>
__device__ __forceinline__ void store8(T* p, const uint64_t (&x)[4]) {
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<float4*>(p)[0] = make_float4(low(x[0]), high(x[0]), low(x[1]), high(x[1]));
    reinterpret_cast<float4*>(p)[1] = make_float4(low(x[2]), high(x[2]), low(x[3]), high(x[3]));
  } else {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack_16x2<T>(low(x[0]), high(x[0])), pack_16x2<T>(low(x[1]), high(x[1])),
                                              pack_16x2<T>(low(x[2]), high(x[2])), pack_16x2<T>(low(x[3]), high(x[3])));
  }
}
template <typename T>
__device__ __forceinline__ void load_weights(const NormParams& p, const void* w, int at, uint64_t (&x)[4]) {
  if (p.w_fp32) {
    Eight<float> e;
    e.load(static_cast<const float*>(w) + at);
    e.pairs(x);
  } else {
    Eight<T> e;
    e.load(static_cast<const T*>(w) + at);
    e.pairs(x);
  }
}
// sum of a pair's halves over the lanes of a row
template <int LANES>
__device__ __forceinline__ float row_sum(uint64_t v) {
  float x = low(v) + high(v);
#pragma unroll
  for (int m = 1; m < LANES; m <<= 1) x += __shfl_xor_sync(0xffffffffu, x, m);
  return x;
}

// Token `token` of a call, as batch entry and token of it, and its position.
struct Token {
  uint32_t z, s;
  __device__ __forceinline__ Token(const NormParams& p, uint32_t token) : z(token / p.s), s(token - token / p.s * p.s) {}
  __device__ __forceinline__ int64_t position(const NormParams& p) const {
    return p.positions != nullptr ? (int64_t)p.positions[z * p.pos_batch + s] : p.pos0 + s;
  }
};

constexpr int kFwdThreads = 128, kFwdWarps = kFwdThreads / 32, kFwdBlocks = 6;         // blocks of an SM

// Rounds of tasks: each has the same tokens' queries, then their keys.
template <typename T, int D, int STEPS>
__global__ void __launch_bounds__(kFwdThreads, kFwdBlocks) qk_norm_rope_kernel(NormParams p, uint32_t round_q, uint32_t round, uint32_t all) {
  using S = Shape<T, D>;
  const int lane = threadIdx.x & 31, group = lane / S::kLanes, col = lane % S::kLanes * 8;
  griddep_wait();
  griddep_launch();
  const uint32_t warps = gridDim.x * kFwdWarps;
  for (uint32_t i = blockIdx.x * kFwdWarps + (threadIdx.x >> 5); i < all; i += warps) {
    uint32_t sub = i % round;
    const int which = sub >= round_q;
    if (which) sub -= round_q;
    const Operand& o = p.o[which];
    // the task's number among those of its operand
    const uint32_t t = i / round * (which ? round - round_q : round_q) + sub;
    const uint32_t chunk = t % o.chunks, token = t / o.chunks * (uint32_t)(S::kRows >> o.log_heads) + (uint32_t)(group >> o.log_heads);
    const int head = (int)(chunk * o.steps << o.log_heads) + (group & ((1 << o.log_heads) - 1));
    const int left = token < p.tokens ? (o.heads - head + (1 << o.log_heads) - 1) >> o.log_heads : 0;      // this lane's steps
    const Token at(p, token < p.tokens ? token : 0);
    const int64_t x_step = o.xh << o.log_heads, y_step = o.yh << o.log_heads;
    const T* px = static_cast<const T*>(o.x) + at.z * o.xz + at.s * o.xs + head * o.xh + col;
    T* py = static_cast<T*>(o.y) + at.z * o.yz + at.s * o.ys + head * o.yh + col;
    Eight<T> xa[STEPS], xb[STEPS];
#pragma unroll
    for (int k = 0; k < STEPS; ++k) {
      if (k < left) {
        xa[k].load(px + k * x_step);
        xb[k].load(px + k * x_step + D / 2);
      } else {
        xa[k].zero();
        xb[k].zero();
      }
    }
    const int64_t pos = at.position(p);
    uint64_t ac[4], as[4], bc[4], bs[4];                   // weights times cos and sin
    {
      uint64_t wa[4], wb[4], c[4], s[4];
      if (pos >= 0 && pos < p.table_rows) {
        Eight<float> e;
        e.load(p.cs + pos * (D / 2) + col);
        e.pairs(c);
        e.load(p.sn + pos * (D / 2) + col);
        e.pairs(s);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) c[e] = s[e] = pair(0x7FC00000u, 0x7FC00000u);
      }
      load_weights<T>(p, o.w, col, wa);
      load_weights<T>(p, o.w, D / 2 + col, wb);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        ac[e] = mul_pair(wa[e], c[e]);
        as[e] = mul_pair(wa[e], s[e]);
        bc[e] = mul_pair(wb[e], c[e]);
        bs[e] = mul_pair(wb[e], minus(s[e]));
      }
    }
#pragma unroll
    for (int k = 0; k < STEPS; ++k) {
      uint64_t a[4], b[4];
      xa[k].pairs(a);
      xb[k].pairs(b);
      uint64_t sum = mul_pair(a[0], a[0]), sum_b = mul_pair(b[0], b[0]);
#pragma unroll
      for (int e = 1; e < 4; ++e) {
        sum = fma_pair(a[e], a[e], sum);
        sum_b = fma_pair(b[e], b[e], sum_b);
      }
      const float r = rsqrtf(row_sum<S::kLanes>(add_pair(sum, sum_b)) * (1.0f / D) + p.eps);
      const uint64_t r2 = pair_of(r, r);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint64_t u = mul_pair(a[e], r2), v = mul_pair(b[e], r2);
        a[e] = fma_pair(u, ac[e], mul_pair(v, bs[e]));
        b[e] = fma_pair(v, bc[e], mul_pair(u, as[e]));
      }
      if (k < left) {
        store8<T>(py + k * y_step, a);
        store8<T>(py + k * y_step + D / 2, b);
      }
    }
  }
}

constexpr int kBwdWarps = 2, kBwdBlocks = 6, kStages = 2;
constexpr int kBwdStatic = 2048;               // shared memory of a block besides its stages, at most, with what the system reserves

// Whether block b of `blocks` has keys, and its number among those of its operand: every blocks / key_blocks-th one.
struct Share {
  int which;
  uint32_t rank, count;
  __device__ __forceinline__ Share(const NormParams& p, uint32_t b, uint32_t blocks) {
    const uint32_t before = (uint32_t)((uint64_t)b * p.key_blocks / blocks), behind = (uint32_t)((uint64_t)(b + 1) * p.key_blocks / blocks);
    which = behind > before;
    rank = which ? before : b - before;
    count = which ? p.key_blocks : blocks - p.key_blocks;
  }
};

// A stage of a warp: rows of x [tokens][heads][D], of g, cos and sin [tokens][2][D/2].  Sums of a lane's columns stay in registers
// over all its rows, then go, row group by row group and warp by warp in that order, into the block's place of `part`.
template <typename T, int D, int STEPS>
__global__ void __launch_bounds__(32 * kBwdWarps, kBwdBlocks) qk_norm_rope_bwd_kernel(NormParams p) {
  using S = Shape<T, D>;
  constexpr int kOperand = S::kRows * STEPS * S::kRowBytes, kAngles = D * 4;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t bars[kBwdWarps][kStages];
  __shared__ bool inside_s[kBwdWarps][kStages][S::kRows * STEPS];      // a token's position lies within the tables
  __shared__ int64_t place_s[kBwdWarps][kStages][S::kRows * STEPS];    // where its gradient's rows are
  __shared__ int expired;
  const int lane = threadIdx.x & 31, warp = warp_index(), group = lane / S::kLanes, col = lane % S::kLanes * 8;
  if (threadIdx.x == 0) expired = 0;
  if (lane == 0) {
    for (int i = 0; i < kStages; ++i) mbar_init(&bars[warp][i], 1);
    mbar_fence_init();
  }
  __syncthreads();
  griddep_wait();
  griddep_launch();
  const Share share(p, blockIdx.x, gridDim.x);
  const Operand& o = p.o[share.which];
  const uint32_t warps = share.count * kBwdWarps, first = share.rank * kBwdWarps + warp;
  const int tokens_step = S::kRows >> o.log_heads, tokens = tokens_step * (STEPS / o.steps), heads = o.steps << o.log_heads;       // of a task
  const bool dense = o.xh == D && o.gh == D;               // a token's heads are one run
  const uint32_t stages = smem_u32(smem) + warp * kStages * p.stage_bytes;
  uint64_t da[4], db[4], wa[4], wb[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) da[e] = db[e] = 0;
  load_weights<T>(p, o.w, col, wa);
  load_weights<T>(p, o.w, D / 2 + col, wb);

  // Lane j asks for token j's rows and angles, or (heads apart) for row j of the task.  The positions of the task behind are on
  // their way meanwhile.
  uint32_t next = first, asked = 0;
  const int of = dense ? lane : lane / heads;              // this lane's token of a task
  int64_t pos = -1;
  auto look_up = [&]() {
    const uint32_t token = next / o.chunks * (uint32_t)tokens + of;
    pos = next < o.tasks && of < tokens && token < p.tokens ? Token(p, token).position(p) : -1;
  };
  auto ask = [&]() {
    if (next < o.tasks) {
      const uint32_t stage = asked % kStages, token = next / o.chunks * (uint32_t)tokens + of;
      const int head0 = next % o.chunks * heads, run = min(o.heads - head0, heads);
      const int in = dense ? 0 : lane - of * heads;        // first of this lane's heads
      const bool there = of < tokens && token < p.tokens, rows = there && in < run, angles = there && in == 0;
      const bool inside = pos >= 0 && pos < p.table_rows;
      const uint32_t bytes = dense ? run * S::kRowBytes : S::kRowBytes;
      uint64_t* bar = &bars[warp][stage];
      const uint32_t total = __reduce_add_sync(0xffffffffu, (rows ? 2 * bytes : 0) + (angles && inside ? kAngles : 0));
      if (lane == 0) mbar_expect_tx(bar, total);
      __syncwarp();
      const uint32_t to = stages + stage * p.stage_bytes;
      if (rows) {
        const Token at(p, token);
        const uint32_t row = to + (of * heads + in) * S::kRowBytes;
        bulk_load(row, static_cast<const T*>(o.x) + at.z * o.xz + at.s * o.xs + (head0 + in) * o.xh, bytes, bar);
        bulk_load(row + kOperand, static_cast<const T*>(o.g) + at.z * o.gz + at.s * o.gs + (head0 + in) * o.gh, bytes, bar);
      }
      if (angles) {
        const Token at(p, token);
        place_s[warp][stage][of] = at.z * o.yz + at.s * o.ys;
        inside_s[warp][stage][of] = inside;
        if (inside) {
          bulk_load(to + 2 * kOperand + of * kAngles, p.cs + pos * (D / 2), kAngles / 2, bar);
          bulk_load(to + 2 * kOperand + of * kAngles + kAngles / 2, p.sn + pos * (D / 2), kAngles / 2, bar);
        }
      }
      next += warps;
      ++asked;
    }
    look_up();
  };
  look_up();
  for (int i = 0; i < kStages - 1; ++i) ask();
  const int shift = o.steps > 2 ? 2 : o.steps - 1;         // steps of a token's place in a task: four, two or one
  const int sub = group & ((1 << o.log_heads) - 1);        // this lane's head of a step
  uint32_t n = 0;
  for (uint32_t i = first; i < o.tasks; i += warps, ++n) {
    ask();
    const uint32_t stage = n % kStages, token0 = i / o.chunks * (uint32_t)tokens;
    const int head = (int)(i % o.chunks) * heads + sub;
    mbar_wait_warp(&bars[warp][stage], n / kStages & 1, &expired, 80);
    const uint32_t from = stages + stage * p.stage_bytes;
#pragma unroll
    for (int k = 0; k < STEPS; ++k) {                      // straight on: steps of several tokens overlap
      const int in = (k >> shift) * tokens_step + (group >> o.log_heads), step = k & ((1 << shift) - 1);      // token of the task, its step
      const int at_head = head + (step << o.log_heads);
      const bool mine = token0 + in < p.tokens && in < tokens && step < o.steps && at_head < o.heads;
      if (!__any_sync(0xffffffffu, mine)) break;
      const uint32_t row = from + (in * heads + sub + (step << o.log_heads)) * S::kRowBytes + col * sizeof(T);
      const uint32_t angles = from + 2 * kOperand + in * kAngles + col * 4;
      T* py = static_cast<T*>(o.y) + place_s[warp][stage][in] + at_head * o.yh + col;
      uint64_t c[4], s[4];
      Eight<float> cos, sin;
      cos.load(angles);
      sin.load(angles + kAngles / 2);
      cos.pairs(c);
      sin.pairs(s);
      if (!inside_s[warp][stage][in]) {
#pragma unroll
        for (int e = 0; e < 4; ++e) c[e] = s[e] = pair(0x7FC00000u, 0x7FC00000u);
      }
      // rows of no head are what the stage held, and go nowhere
      Eight<T> xa, xb, ya, yb;
      xa.load(row);
      xb.load(row + S::kRowBytes / 2);
      ya.load(row + kOperand);
      yb.load(row + kOperand + S::kRowBytes / 2);
      uint64_t a[4], b[4], ga[4], gb[4], sum = 0, sum_b = 0, dot = 0, dot_b = 0;
      xa.pairs(a);
      xb.pairs(b);
      ya.pairs(ga);
      yb.pairs(gb);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        sum = fma_pair(a[e], a[e], sum);
        sum_b = fma_pair(b[e], b[e], sum_b);
        const uint64_t u = fma_pair(ga[e], c[e], mul_pair(gb[e], s[e])), v = fma_pair(gb[e], c[e], mul_pair(ga[e], minus(s[e])));
        ga[e] = u;
        gb[e] = v;
        dot = fma_pair(mul_pair(u, wa[e]), a[e], dot);
        dot_b = fma_pair(mul_pair(v, wb[e]), b[e], dot_b);
      }
      const float r = rsqrtf(row_sum<S::kLanes>(add_pair(sum, sum_b)) * (1.0f / D) + p.eps);
      const float m = row_sum<S::kLanes>(add_pair(dot, dot_b)) * r * (1.0f / D);     // mean(g' w n)
      const uint64_t r2 = pair_of(r, r), m2 = pair_of(-m, -m);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        a[e] = mul_pair(a[e], r2);
        b[e] = mul_pair(b[e], r2);
        if (mine) {
          da[e] = fma_pair(ga[e], a[e], da[e]);
          db[e] = fma_pair(gb[e], b[e], db[e]);
        }
        a[e] = mul_pair(fma_pair(a[e], m2, mul_pair(ga[e], wa[e])), r2);
        b[e] = mul_pair(fma_pair(b[e], m2, mul_pair(gb[e], wb[e])), r2);
      }
      if (mine) {
        store8<T>(py, a);
        store8<T>(py + D / 2, b);
      }
    }
    __syncwarp();                                          // the stage may be filled again
  }
  if (p.part != nullptr) {
    float* const sums = reinterpret_cast<float*>(smem) + warp * D;       // where the stages were: all of them have been read
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 4; ++e) {
#pragma unroll
      for (int m = S::kLanes; m < 32; m <<= 1) {
        da[e] = add_pair(da[e], __shfl_xor_sync(0xffffffffu, da[e], m));
        db[e] = add_pair(db[e], __shfl_xor_sync(0xffffffffu, db[e], m));
      }
      if (group == 0) {
        *reinterpret_cast<uint64_t*>(&sums[col + 2 * e]) = da[e];
        *reinterpret_cast<uint64_t*>(&sums[D / 2 + col + 2 * e]) = db[e];
      }
    }
    __syncthreads();
    const uint32_t place = share.which ? gridDim.x - p.key_blocks + share.rank : share.rank;
    for (int i = threadIdx.x; i < D; i += 32 * kBwdWarps) {
      float t = 0.0f;
#pragma unroll
      for (int w = 0; w < kBwdWarps; ++w) t += reinterpret_cast<const float*>(smem)[w * D + i];
      p.part[(int64_t)place * D + i] = t;
    }
  }
  __syncthreads();
  report_error(&expired, p.status);
}

// Columns of the blocks' sums, in block order: 32 columns a block of threads, 32 threads a column.
template <typename W>
__global__ void __launch_bounds__(1024) qk_norm_weights_kernel(const float* part, int query_blocks, int blocks, int d, W* dwq, W* dwk) {
  __shared__ float sums[32][33];
  griddep_wait();
  griddep_launch();
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5, which = (int)blockIdx.x * 32 >= d, col = blockIdx.x * 32 - which * d + lane;
  float t = 0.0f;
#pragma unroll 8
  for (int b = (which ? query_blocks : 0) + slice; b < (which ? blocks : query_blocks); b += 32) t += part[(int64_t)b * d + col];
  sums[slice][lane] = t;
  __syncthreads();
  t = sums[lane][slice];
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) t += __shfl_xor_sync(0xffffffffu, t, m);
  W* to = which ? dwk : dwq;
  if (lane == 0 && to != nullptr) to[blockIdx.x * 32 - which * d + slice] = from_f32<W>(t);
}

// Tasks of at most `steps` steps, of further tokens too where one takes fewer (`fill`).  Returns the tokens of a task.
int plan_operand(Operand& o, int64_t tokens, int rows, int steps, bool fill) {
  o.log_heads = 0;
  while ((2 << o.log_heads) <= rows && (2 << o.log_heads) <= o.heads) ++o.log_heads;
  const int want = (o.heads + (1 << o.log_heads) - 1) >> o.log_heads;
  o.steps = want < steps ? want : steps;
  const int at_once = (rows >> o.log_heads) * (fill ? steps / o.steps : 1);
  o.chunks = (uint32_t)((want + o.steps - 1) / o.steps);
  o.tasks = (uint32_t)((tokens + at_once - 1) / at_once * o.chunks);
  return at_once;
}
int sm_count() {
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms;
}

template <typename T, int D>
int run_forward(NormParams p, cudaStream_t st) {
  constexpr int kSteps = sizeof(T) == 4 ? 1 : 2, kRows = Shape<T, D>::kRows;
  const int64_t tq = plan_operand(p.o[0], p.tokens, kRows, kSteps, false), tk = plan_operand(p.o[1], p.tokens, kRows, kSteps, false);
  const int64_t tokens = tq > tk ? tq : tk;                // a round has those of the operand that takes more of them at once
  const uint32_t round_q = (uint32_t)(tokens / tq * p.o[0].chunks), round = round_q + (uint32_t)(tokens / tk * p.o[1].chunks);
  const int64_t all = (p.tokens + tokens - 1) / tokens * round, most = (int64_t)kFwdBlocks * sm_count(), want = (all + kFwdWarps - 1) / kFwdWarps;
  NVFP4_REQUIRE(all < (1ll << 31), "nvfp4_qk_norm_rope: too many rows");
  return launch("nvfp4_qk_norm_rope", qk_norm_rope_kernel<T, D, kSteps>, dim3((unsigned)(want < most ? want : most)), kFwdThreads, 0, st, p,
                round_q, round, (uint32_t)all);
}
template <typename T, int D>
int run_backward(NormParams p, int w_dtype, void* dwq, void* dwk, cudaStream_t st) {
  constexpr int kSteps = sizeof(T) == 4 ? 2 : 4, kRows = Shape<T, D>::kRows;
  const int of_q = plan_operand(p.o[0], p.tokens, kRows, kSteps, true), of_k = plan_operand(p.o[1], p.tokens, kRows, kSteps, true);
  p.stage_bytes = 2 * kRows * kSteps * Shape<T, D>::kRowBytes + (of_q > of_k ? of_q : of_k) * D * 4;
  const int smem = kBwdWarps * kStages * p.stage_bytes, fit = kSmemPerSm / (smem + kBwdStatic);
  const int64_t tq = p.o[0].tasks, tk = p.o[1].tasks, most = (int64_t)(fit < kBwdBlocks ? fit : kBwdBlocks) * sm_count();
  const int64_t want = (tq + kBwdWarps - 1) / kBwdWarps + (tk + kBwdWarps - 1) / kBwdWarps, blocks = want < most ? want : most;
  const int64_t keys = blocks * tk / (tq + tk);
  p.key_blocks = (uint32_t)(keys < 1 ? 1 : keys > blocks - 1 ? blocks - 1 : keys);
  // the largest that any call needs: the attribute is set once a kernel
  constexpr int kMost = kBwdWarps * kStages * (2 * kRows * kSteps * Shape<T, D>::kRowBytes + kRows * kSteps * D * 4);
  const auto kern = qk_norm_rope_bwd_kernel<T, D, kSteps>;
  if (int rc = allow_smem("nvfp4_qk_norm_rope_bwd", reinterpret_cast<const void*>(kern), kMost)) return rc;
  if (int rc = launch("nvfp4_qk_norm_rope_bwd", kern, dim3((unsigned)blocks), 32 * kBwdWarps, smem, st, p)) return rc;
  if (p.part == nullptr) return 0;
  const dim3 grid(2 * D / 32);
  const int query_blocks = (int)(blocks - p.key_blocks);
  switch (w_dtype) {
    case NVFP4_DT_BF16:
      return launch("nvfp4_qk_norm_rope_bwd", qk_norm_weights_kernel<__nv_bfloat16>, grid, 1024, 0, st, p.part, query_blocks, (int)blocks, D,
                    static_cast<__nv_bfloat16*>(dwq), static_cast<__nv_bfloat16*>(dwk));
    case NVFP4_DT_FP16:
      return launch("nvfp4_qk_norm_rope_bwd", qk_norm_weights_kernel<__half>, grid, 1024, 0, st, p.part, query_blocks, (int)blocks, D,
                    static_cast<__half*>(dwq), static_cast<__half*>(dwk));
    default:
      return launch("nvfp4_qk_norm_rope_bwd", qk_norm_weights_kernel<float>, grid, 1024, 0, st, p.part, query_blocks, (int)blocks, D,
                    static_cast<float*>(dwq), static_cast<float*>(dwk));
  }
}

// The arguments that both directions share, checked; 1: there is nothing to do.
int set_up(const char* what, NormParams& p, int dtype, int64_t z, int64_t s, int64_t h, int64_t hk, int d, const void* wq,
           const void* wk, int w_dtype, const float* cos_tab, const float* sin_tab, int64_t table_rows, const int32_t* positions, int64_t pos_batch, int64_t pos0, float eps) {
  NVFP4_REQUIRE(d == 128 || d == 256, "%s: D must be 128 or 256", what);
  NVFP4_REQUIRE(dtype >= NVFP4_DT_BF16 && dtype <= NVFP4_DT_FP32, "%s: unknown dtype %d", what, dtype);
  NVFP4_REQUIRE(w_dtype == dtype || w_dtype == NVFP4_DT_FP32, "%s: weights must be of the operands' type or fp32", what);
  NVFP4_REQUIRE(z >= 0 && s >= 0 && h >= 1 && hk >= 1 && h < (1 << 20) && hk < (1 << 20), "%s: sizes out of range", what);
  NVFP4_REQUIRE(s == 0 || z <= (1ll << 30) / s, "%s: too many tokens", what);
  NVFP4_REQUIRE(z * s * (h > hk ? h : hk) < (1ll << 31), "%s: too many rows", what);
  NVFP4_REQUIRE((((uintptr_t)cos_tab | (uintptr_t)sin_tab) & 15) == 0, "%s: cos / sin tables must be 16-byte aligned", what);
  NVFP4_REQUIRE((((uintptr_t)wq | (uintptr_t)wk) & 15) == 0, "%s: weights must be 16-byte aligned", what);
  NVFP4_REQUIRE(eps >= 0.0f, "%s: eps must not be negative", what);
  p.cs = cos_tab;
  p.sn = sin_tab;
  p.table_rows = table_rows;
  p.positions = positions;
  p.pos_batch = pos_batch;
  p.pos0 = pos0;
  p.tokens = (uint32_t)(z * s);
  p.s = (uint32_t)s;
  p.w_fp32 = w_dtype == NVFP4_DT_FP32;
  p.eps = eps;
  return z * s == 0 ? 1 : 0;
}
bool rows_aligned(const void* x, const int64_t* strides, int dtype) {
  const int64_t size = dtype == NVFP4_DT_FP32 ? 4 : 2;
  return ((uintptr_t)x & 15) == 0 && ((strides[0] | strides[1] | strides[2]) * size & 15) == 0;
}

}  // namespace
}  // namespace nvfp4

using namespace nvfp4;

extern "C" int nvfp4_qk_norm_rope(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides, int dtype, int64_t z,
                                  int64_t s, int64_t h, int64_t hk, int d, const void* wq, const void* wk, int w_dtype,
                                  const float* cos_tab, const float* sin_tab, int64_t table_rows, const int32_t* positions,
                                  int64_t pos_batch, int64_t pos0, float eps, void* out_q, const int64_t* oq_strides, void* out_k,
                                  const int64_t* ok_strides, nvfp4_stream_t stream) {
  const char* what = "nvfp4_qk_norm_rope";
  NormParams p{};
  const int rc = set_up(what, p, dtype, z, s, h, hk, d, wq, wk, w_dtype, cos_tab, sin_tab, table_rows, positions, pos_batch, pos0, eps);
  if (rc != 0) return rc < 0 ? rc : 0;
  NVFP4_REQUIRE(rows_aligned(q, q_strides, dtype) && rows_aligned(k, k_strides, dtype) && rows_aligned(out_q, oq_strides, dtype) &&
                    rows_aligned(out_k, ok_strides, dtype),
                "%s: rows must be 16-byte aligned", what);
  p.o[0] = {q, nullptr, out_q, q_strides[0], q_strides[1], q_strides[2], 0, 0, 0, oq_strides[0], oq_strides[1], oq_strides[2], wq, (int)h, 0, 0, 0, 0};
  p.o[1] = {k, nullptr, out_k, k_strides[0], k_strides[1], k_strides[2], 0, 0, 0, ok_strides[0], ok_strides[1], ok_strides[2], wk, (int)hk, 0, 0, 0, 0};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case NVFP4_DT_BF16: return d == 128 ? run_forward<__nv_bfloat16, 128>(p, st) : run_forward<__nv_bfloat16, 256>(p, st);
    case NVFP4_DT_FP16: return d == 128 ? run_forward<__half, 128>(p, st) : run_forward<__half, 256>(p, st);
    default: return d == 128 ? run_forward<float, 128>(p, st) : run_forward<float, 256>(p, st);
  }
}

extern "C" int nvfp4_qk_norm_rope_bwd_plan(int d, int sm_count, size_t* workspace_bytes) {
  NVFP4_REQUIRE(d == 128 || d == 256, "nvfp4_qk_norm_rope_bwd_plan: D must be 128 or 256");
  NVFP4_REQUIRE(sm_count >= 1 && workspace_bytes != nullptr, "nvfp4_qk_norm_rope_bwd_plan: bad argument");
  *workspace_bytes = (size_t)kBwdBlocks * sm_count * d * sizeof(float);
  return 0;
}

extern "C" int nvfp4_qk_norm_rope_bwd(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides, const void* grad_q,
                                      const int64_t* gq_strides, const void* grad_k, const int64_t* gk_strides, int dtype, int64_t z,
                                      int64_t s, int64_t h, int64_t hk, int d, const void* wq, const void* wk, int w_dtype,
                                      const float* cos_tab, const float* sin_tab, int64_t table_rows, const int32_t* positions,
                                      int64_t pos_batch, int64_t pos0, float eps, void* dq, const int64_t* dq_strides, void* dk,
                                      const int64_t* dk_strides, void* dwq, void* dwk, void* workspace, size_t workspace_bytes,
                                      int* status, nvfp4_stream_t stream) {
  const char* what = "nvfp4_qk_norm_rope_bwd";
  NormParams p{};
  const int rc = set_up(what, p, dtype, z, s, h, hk, d, wq, wk, w_dtype, cos_tab, sin_tab, table_rows, positions, pos_batch, pos0, eps);
  if (rc < 0) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (rc == 1) {                               // no rows: the weights' gradients are sums of nothing
    for (void* w : {dwq, dwk})
      if (w != nullptr)
        if (const cudaError_t e = cudaMemsetAsync(w, 0, (size_t)d * (w_dtype == NVFP4_DT_FP32 ? 4 : 2), st); e != cudaSuccess)
          return fail((int)e, "%s: %s", what, cudaGetErrorString(e));
    return 0;
  }
  NVFP4_REQUIRE(rows_aligned(q, q_strides, dtype) && rows_aligned(k, k_strides, dtype) && rows_aligned(grad_q, gq_strides, dtype) &&
                    rows_aligned(grad_k, gk_strides, dtype) && rows_aligned(dq, dq_strides, dtype) && rows_aligned(dk, dk_strides, dtype),
                "%s: rows must be 16-byte aligned", what);
  p.status = status;
  if (dwq != nullptr || dwk != nullptr) {
    NVFP4_REQUIRE(workspace != nullptr && ((uintptr_t)workspace & 3) == 0 &&
                      workspace_bytes >= (size_t)kBwdBlocks * sm_count() * d * sizeof(float),
                  "%s: workspace too small", what);
    p.part = static_cast<float*>(workspace);
  }
  p.o[0] = {q, grad_q, dq, q_strides[0], q_strides[1], q_strides[2], gq_strides[0], gq_strides[1], gq_strides[2], dq_strides[0],
            dq_strides[1], dq_strides[2], wq, (int)h, 0, 0, 0, 0};
  p.o[1] = {k, grad_k, dk, k_strides[0], k_strides[1], k_strides[2], gk_strides[0], gk_strides[1], gk_strides[2], dk_strides[0],
            dk_strides[1], dk_strides[2], wk, (int)hk, 0, 0, 0, 0};
  switch (dtype) {
    case NVFP4_DT_BF16:
      return d == 128 ? run_backward<__nv_bfloat16, 128>(p, w_dtype, dwq, dwk, st) : run_backward<__nv_bfloat16, 256>(p, w_dtype, dwq, dwk, st);
    case NVFP4_DT_FP16: return d == 128 ? run_backward<__half, 128>(p, w_dtype, dwq, dwk, st) : run_backward<__half, 256>(p, w_dtype, dwq, dwk, st);
    default: return d == 128 ? run_backward<float, 128>(p, w_dtype, dwq, dwk, st) : run_backward<float, 256>(p, w_dtype, dwq, dwk, st);
  }
}
