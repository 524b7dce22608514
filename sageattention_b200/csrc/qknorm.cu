// RMS norm of every head's queries and keys and their rotation by position, in one pass; and its backward pass.
//
//   r = 1 / sqrt(mean(x^2) + eps),  n = x r,  y = rot_p(n w)            rot_p: element i with element i + D/2, by angle i of position p
//   g' = rot_p^-1(dy),  dw = sum over rows g' n,  dx = r (g' w - n mean(g' w n))
//
// What bounds it: HBM; a row is read once and written once (backward: two reads, a write).  A row is D/16 lanes, each with eight
// elements of either half, so that a rotation stays within a lane and every access is 16 bytes wide; a warp has the rows of
// several heads of a token, whose cos and sin it loads once for all of them.  Statistics, rotation and weight gradients are
// fp32, rounded once to the type of the operand.
#include <limits.h>
#include "common/abi.cuh"
#include "common/fp4.cuh"
#include "common/launch.cuh"

namespace nvfp4 {
namespace {

constexpr int kThreads = 128, kWarps = kThreads / 32;

// One of the two operands: queries or keys.
struct Operand {
  const void* x;
  const void* g;                               // incoming gradient (backward)
  void* y;                                     // result, or gradient of x
  int64_t xz, xs, xh, gz, gs, gh, yz, ys, yh;  // element strides of batch entry, token, head
  const void* w;
  int heads, log_heads;                        // rows of a warp's step: 2^log_heads heads of a token, the others are further tokens
  uint32_t chunks;                             // steps times heads of a step cover the heads in so many tasks
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
  float* part;                                 // [blocks][2][D] sums of the weights' gradients
};

template <typename T, int D>
struct Shape {
  static constexpr int kLanes = D / 16;        // of a row
  static constexpr int kRows = 32 / kLanes;    // of a warp
  static constexpr int kVec = 8 * sizeof(T) / 16;
};

template <typename T, int D>
struct Row {                                   // eight elements of either half, as they lie
  uint4 v[2][Shape<T, D>::kVec];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < Shape<T, D>::kVec; ++i) v[h][i] = reinterpret_cast<const uint4*>(p + h * (D / 2))[i];
  }
  __device__ __forceinline__ void values(float (&a)[8], float (&b)[8]) const {
    const T *pa = reinterpret_cast<const T*>(v[0]), *pb = reinterpret_cast<const T*>(v[1]);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      a[i] = to_f32<T>(pa[i]);
      b[i] = to_f32<T>(pb[i]);
    }
  }
};
template <typename T, int D>
__device__ __forceinline__ void store_row(T* p, const float (&a)[8], const float (&b)[8]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const float(&x)[8] = h == 0 ? a : b;
    if constexpr (sizeof(T) == 4) {
      reinterpret_cast<float4*>(p + h * (D / 2))[0] = make_float4(x[0], x[1], x[2], x[3]);
      reinterpret_cast<float4*>(p + h * (D / 2))[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
      *reinterpret_cast<uint4*>(p + h * (D / 2)) =
          make_uint4(pack_16x2<T>(x[0], x[1]), pack_16x2<T>(x[2], x[3]), pack_16x2<T>(x[4], x[5]), pack_16x2<T>(x[6], x[7]));
    }
  }
}
__device__ __forceinline__ void load8(const float* p, float (&x)[8]) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
  x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}

template <typename T, int D>
struct Task {
  using S = Shape<T, D>;
  int lane, group, col;                        // column of this lane's elements of the first half
  float wa[8], wb[8];

  __device__ __forceinline__ Task() {
    lane = threadIdx.x & 31;
    group = lane / S::kLanes;
    col = lane % S::kLanes * 8;
  }
  __device__ __forceinline__ void weights(const NormParams& p, const Operand& o) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      wa[i] = p.w_fp32 ? static_cast<const float*>(o.w)[col + i] : to_f32<T>(static_cast<const T*>(o.w)[col + i]);
      wb[i] = p.w_fp32 ? static_cast<const float*>(o.w)[D / 2 + col + i] : to_f32<T>(static_cast<const T*>(o.w)[D / 2 + col + i]);
    }
  }
  // where task `t` of an operand lies: this lane's token (or none) and its first head
  uint32_t token, z, s;
  int head;
  bool there;
  __device__ __forceinline__ void find(const NormParams& p, const Operand& o, uint32_t t, int steps) {
    const uint32_t chunk = t % o.chunks, first = t / o.chunks * (uint32_t)(S::kRows >> o.log_heads);
    token = first + (uint32_t)(group >> o.log_heads);
    there = token < p.tokens;
    z = token / p.s;
    s = token - z * p.s;
    head = (int)(chunk * (uint32_t)steps << o.log_heads) + (group & ((1 << o.log_heads) - 1));
  }
  // cos and sin of the token; outside the tables NaN
  __device__ __forceinline__ void angles(const NormParams& p, float (&c)[8], float (&sn)[8]) const {
    const int64_t pos = !there ? 0 : p.positions != nullptr ? (int64_t)p.positions[z * p.pos_batch + s] : p.pos0 + s;
    if (pos >= 0 && pos < p.table_rows) {
      load8(p.cs + pos * (D / 2) + col, c);
      load8(p.sn + pos * (D / 2) + col, sn);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) c[i] = sn[i] = __int_as_float(0x7FC00000);
    }
  }
  // sum over the lanes of a row
  __device__ __forceinline__ float row_sum(float x) const {
#pragma unroll
    for (int m = 1; m < S::kLanes; m <<= 1) x += __shfl_xor_sync(0xffffffffu, x, m);
    return x;
  }
};

template <typename T, int D, int STEPS>
__global__ void __launch_bounds__(kThreads) qk_norm_rope_kernel(NormParams p) {
  using S = Shape<T, D>;
  Task<T, D> at;
  griddep_wait();
  griddep_launch();
  const uint32_t warps = gridDim.x * kWarps, all = p.o[0].tasks + p.o[1].tasks;
  int had = -1;
  for (uint32_t i = blockIdx.x * kWarps + (threadIdx.x >> 5); i < all; i += warps) {
    const int which = i >= p.o[0].tasks;
    const Operand& o = p.o[which];
    at.find(p, o, which ? i - p.o[0].tasks : i, STEPS);
    const T* px = static_cast<const T*>(o.x) + at.z * o.xz + at.s * o.xs + at.col;
    T* py = static_cast<T*>(o.y) + at.z * o.yz + at.s * o.ys + at.col;
    Row<T, D> x[STEPS];
#pragma unroll
    for (int k = 0; k < STEPS; ++k)
      if (at.there && at.head + (k << o.log_heads) < o.heads) x[k].load(px + (at.head + (k << o.log_heads)) * o.xh);
    float c[8], s[8];
    at.angles(p, c, s);
    if (had != which) at.weights(p, o);
    had = which;
#pragma unroll
    for (int k = 0; k < STEPS; ++k) {
      const int head = at.head + (k << o.log_heads);
      const bool mine = at.there && head < o.heads;
      float a[8], b[8], sum = 0.0f;
      x[k].values(a, b);
#pragma unroll
      for (int e = 0; e < 8; ++e) sum = fmaf(a[e], a[e], fmaf(b[e], b[e], sum));
      const float r = rsqrtf(at.row_sum(sum) * (1.0f / D) + p.eps);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float u = a[e] * r * at.wa[e], v = b[e] * r * at.wb[e];
        a[e] = u * c[e] - v * s[e];
        b[e] = v * c[e] + u * s[e];
      }
      if (mine) store_row<T, D>(py + head * o.yh, a, b);
    }
  }
}

// The rows of an operand after those of the other; sums of a lane's columns stay in registers over all its rows, then go, row
// group by row group and warp by warp in that order, into the block's own place of `part`.
template <typename T, int D, int STEPS>
__global__ void __launch_bounds__(kThreads) qk_norm_rope_bwd_kernel(NormParams p) {
  using S = Shape<T, D>;
  __shared__ float sums[kWarps][D];
  Task<T, D> at;
  griddep_wait();
  griddep_launch();
  const uint32_t warps = gridDim.x * kWarps;
  const int warp = threadIdx.x >> 5;
#pragma unroll 1
  for (int which = 0; which < 2; ++which) {
    const Operand& o = p.o[which];
    float da[8], db[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) da[e] = db[e] = 0.0f;
    at.weights(p, o);
    for (uint32_t i = blockIdx.x * kWarps + warp; i < o.tasks; i += warps) {
      at.find(p, o, i, STEPS);
      const T* px = static_cast<const T*>(o.x) + at.z * o.xz + at.s * o.xs + at.col;
      const T* pg = static_cast<const T*>(o.g) + at.z * o.gz + at.s * o.gs + at.col;
      T* py = static_cast<T*>(o.y) + at.z * o.yz + at.s * o.ys + at.col;
      Row<T, D> x[STEPS], g[STEPS];
#pragma unroll
      for (int k = 0; k < STEPS; ++k) {
        const int head = at.head + (k << o.log_heads);
        if (at.there && head < o.heads) {
          x[k].load(px + head * o.xh);
          g[k].load(pg + head * o.gh);
        }
      }
      float c[8], s[8];
      at.angles(p, c, s);
#pragma unroll
      for (int k = 0; k < STEPS; ++k) {
        const int head = at.head + (k << o.log_heads);
        const bool mine = at.there && head < o.heads;
        float a[8], b[8], ga[8], gb[8], sum = 0.0f, dot = 0.0f;
        x[k].values(a, b);
        g[k].values(ga, gb);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          sum = fmaf(a[e], a[e], fmaf(b[e], b[e], sum));
          const float u = ga[e] * c[e] + gb[e] * s[e], v = gb[e] * c[e] - ga[e] * s[e];
          ga[e] = u;
          gb[e] = v;
          dot = fmaf(u * at.wa[e], a[e], fmaf(v * at.wb[e], b[e], dot));
        }
        const float r = rsqrtf(at.row_sum(sum) * (1.0f / D) + p.eps);
        const float m = at.row_sum(dot) * r * (1.0f / D);        // mean(g' w n)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          a[e] *= r;
          b[e] *= r;
          if (mine) {
            da[e] = fmaf(ga[e], a[e], da[e]);
            db[e] = fmaf(gb[e], b[e], db[e]);
          }
          a[e] = r * (ga[e] * at.wa[e] - a[e] * m);
          b[e] = r * (gb[e] * at.wb[e] - b[e] * m);
        }
        if (mine) store_row<T, D>(py + head * o.yh, a, b);
      }
    }
    if (p.part == nullptr) continue;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
#pragma unroll
      for (int m = S::kLanes; m < 32; m <<= 1) {
        da[e] += __shfl_xor_sync(0xffffffffu, da[e], m);
        db[e] += __shfl_xor_sync(0xffffffffu, db[e], m);
      }
      if (at.group == 0) {
        sums[warp][at.col + e] = da[e];
        sums[warp][D / 2 + at.col + e] = db[e];
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < D; i += kThreads) {
      float t = 0.0f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) t += sums[w][i];
      p.part[((int64_t)blockIdx.x * 2 + which) * D + i] = t;
    }
    __syncthreads();
  }
}

// Columns of the blocks' sums, in block order: 32 columns a block of threads, 32 threads a column.
template <typename W>
__global__ void __launch_bounds__(1024) qk_norm_weights_kernel(const float* part, int blocks, int d, W* dwq, W* dwk) {
  __shared__ float sums[32][33];
  griddep_wait();
  griddep_launch();
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5, col = blockIdx.x * 32 + lane;
  float t = 0.0f;
  for (int b = slice; b < blocks; b += 32) t += part[(int64_t)b * 2 * d + col];
  sums[slice][lane] = t;
  __syncthreads();
  t = sums[lane][slice];
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) t += __shfl_xor_sync(0xffffffffu, t, m);
  if (lane == 0) {
    const int c = blockIdx.x * 32 + slice;
    W* to = c < d ? dwq : dwk;
    if (to != nullptr) to[c < d ? c : c - d] = from_f32<W>(t);
  }
}

void plan_operand(Operand& o, int64_t tokens, int rows, int steps) {
  o.log_heads = 0;
  while ((2 << o.log_heads) <= rows && (2 << o.log_heads) <= o.heads) ++o.log_heads;
  const int64_t per = (int64_t)steps << o.log_heads, at_once = rows >> o.log_heads;
  o.chunks = (uint32_t)((o.heads + per - 1) / per);
  o.tasks = (uint32_t)((tokens + at_once - 1) / at_once * o.chunks);
}

constexpr int kBlocksPerSm = 8;
int blocks_of(const NormParams& p, int sms) {
  const int64_t want = ((int64_t)p.o[0].tasks + p.o[1].tasks + kWarps - 1) / kWarps, most = (int64_t)kBlocksPerSm * sms;
  return (int)(want < most ? want : most);
}
int sm_count() {
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms;
}

template <typename T, int D>
int run_forward(NormParams p, cudaStream_t st) {
  constexpr int kSteps = sizeof(T) == 4 ? 2 : 4;
  for (Operand& o : p.o) plan_operand(o, p.tokens, Shape<T, D>::kRows, kSteps);
  return launch("nvfp4_qk_norm_rope", qk_norm_rope_kernel<T, D, kSteps>, dim3((unsigned)blocks_of(p, sm_count())), kThreads, 0, st, p);
}
template <typename T, int D>
int run_backward(NormParams p, int w_dtype, void* dwq, void* dwk, cudaStream_t st) {
  constexpr int kSteps = sizeof(T) == 4 ? 1 : 2;
  for (Operand& o : p.o) plan_operand(o, p.tokens, Shape<T, D>::kRows, kSteps);
  const int blocks = blocks_of(p, sm_count());
  if (int rc = launch("nvfp4_qk_norm_rope_bwd", qk_norm_rope_bwd_kernel<T, D, kSteps>, dim3((unsigned)blocks), kThreads, 0, st, p)) return rc;
  if (p.part == nullptr) return 0;
  const dim3 grid(2 * D / 32);
  switch (w_dtype) {
    case NVFP4_DT_BF16:
      return launch("nvfp4_qk_norm_rope_bwd", qk_norm_weights_kernel<__nv_bfloat16>, grid, 1024, 0, st, p.part, blocks, D,
                    static_cast<__nv_bfloat16*>(dwq), static_cast<__nv_bfloat16*>(dwk));
    case NVFP4_DT_FP16:
      return launch("nvfp4_qk_norm_rope_bwd", qk_norm_weights_kernel<__half>, grid, 1024, 0, st, p.part, blocks, D,
                    static_cast<__half*>(dwq), static_cast<__half*>(dwk));
    default:
      return launch("nvfp4_qk_norm_rope_bwd", qk_norm_weights_kernel<float>, grid, 1024, 0, st, p.part, blocks, D,
                    static_cast<float*>(dwq), static_cast<float*>(dwk));
  }
}

// The arguments that both directions share, checked; 1: there is nothing to do.
int set_up(const char* what, NormParams& p, int dtype, int64_t z, int64_t s, int64_t h, int64_t hk, int d, int w_dtype, const float* cos_tab,
           const float* sin_tab, int64_t table_rows, const int32_t* positions, int64_t pos_batch, int64_t pos0, float eps) {
  NVFP4_REQUIRE(d == 128 || d == 256, "%s: D must be 128 or 256", what);
  NVFP4_REQUIRE(dtype >= NVFP4_DT_BF16 && dtype <= NVFP4_DT_FP32, "%s: unknown dtype %d", what, dtype);
  NVFP4_REQUIRE(w_dtype == dtype || w_dtype == NVFP4_DT_FP32, "%s: weights must be of the operands' type or fp32", what);
  NVFP4_REQUIRE(z >= 0 && s >= 0 && h >= 1 && hk >= 1 && h < (1 << 20) && hk < (1 << 20), "%s: sizes out of range", what);
  NVFP4_REQUIRE(s == 0 || z <= (1ll << 30) / s, "%s: too many tokens", what);
  NVFP4_REQUIRE(z * s * (h > hk ? h : hk) < (1ll << 31), "%s: too many rows", what);
  NVFP4_REQUIRE((((uintptr_t)cos_tab | (uintptr_t)sin_tab) & 15) == 0, "%s: cos / sin tables must be 16-byte aligned", what);
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
  const int rc = set_up(what, p, dtype, z, s, h, hk, d, w_dtype, cos_tab, sin_tab, table_rows, positions, pos_batch, pos0, eps);
  if (rc != 0) return rc < 0 ? rc : 0;
  NVFP4_REQUIRE(rows_aligned(q, q_strides, dtype) && rows_aligned(k, k_strides, dtype) && rows_aligned(out_q, oq_strides, dtype) &&
                    rows_aligned(out_k, ok_strides, dtype),
                "%s: rows must be 16-byte aligned", what);
  p.o[0] = {q, nullptr, out_q, q_strides[0], q_strides[1], q_strides[2], 0, 0, 0, oq_strides[0], oq_strides[1], oq_strides[2], wq, (int)h, 0, 0, 0};
  p.o[1] = {k, nullptr, out_k, k_strides[0], k_strides[1], k_strides[2], 0, 0, 0, ok_strides[0], ok_strides[1], ok_strides[2], wk, (int)hk, 0, 0, 0};
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
  *workspace_bytes = (size_t)kBlocksPerSm * sm_count * 2 * d * sizeof(float);
  return 0;
}

extern "C" int nvfp4_qk_norm_rope_bwd(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides, const void* grad_q,
                                      const int64_t* gq_strides, const void* grad_k, const int64_t* gk_strides, int dtype, int64_t z,
                                      int64_t s, int64_t h, int64_t hk, int d, const void* wq, const void* wk, int w_dtype,
                                      const float* cos_tab, const float* sin_tab, int64_t table_rows, const int32_t* positions,
                                      int64_t pos_batch, int64_t pos0, float eps, void* dq, const int64_t* dq_strides, void* dk,
                                      const int64_t* dk_strides, void* dwq, void* dwk, void* workspace, size_t workspace_bytes,
                                      nvfp4_stream_t stream) {
  const char* what = "nvfp4_qk_norm_rope_bwd";
  NormParams p{};
  const int rc = set_up(what, p, dtype, z, s, h, hk, d, w_dtype, cos_tab, sin_tab, table_rows, positions, pos_batch, pos0, eps);
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
  if (dwq != nullptr || dwk != nullptr) {
    NVFP4_REQUIRE(workspace != nullptr && ((uintptr_t)workspace & 3) == 0 &&
                      workspace_bytes >= (size_t)kBlocksPerSm * sm_count() * 2 * d * sizeof(float),
                  "%s: workspace too small", what);
    p.part = static_cast<float*>(workspace);
  }
  p.o[0] = {q, grad_q, dq, q_strides[0], q_strides[1], q_strides[2], gq_strides[0], gq_strides[1], gq_strides[2], dq_strides[0],
            dq_strides[1], dq_strides[2], wq, (int)h, 0, 0, 0};
  p.o[1] = {k, grad_k, dk, k_strides[0], k_strides[1], k_strides[2], gk_strides[0], gk_strides[1], gk_strides[2], dk_strides[0],
            dk_strides[1], dk_strides[2], wk, (int)hk, 0, 0, 0};
  switch (dtype) {
    case NVFP4_DT_BF16:
      return d == 128 ? run_backward<__nv_bfloat16, 128>(p, w_dtype, dwq, dwk, st) : run_backward<__nv_bfloat16, 256>(p, w_dtype, dwq, dwk, st);
    case NVFP4_DT_FP16: return d == 128 ? run_backward<__half, 128>(p, w_dtype, dwq, dwk, st) : run_backward<__half, 256>(p, w_dtype, dwq, dwk, st);
    default: return d == 128 ? run_backward<float, 128>(p, w_dtype, dwq, dwk, st) : run_backward<float, 256>(p, w_dtype, dwq, dwk, st);
  }
}
