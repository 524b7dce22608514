// Paged 8-bit KV cache: block tables and slot maps from request lengths, and the quantising write.
#include <type_traits>
#include "common/abi.cuh"
#include "common/fp4.cuh"
#include "common/kv8.cuh"
#include "common/launch.cuh"

namespace nvfp4 {
namespace {

// ------------------------------------------------------------------------------------------ tables
constexpr int kTableThreads = 1024;
constexpr int kSearchRows = 4096;        // prefix sums of as many requests are searched in shared memory

// Exclusive prefix sum over the block of two counts at once, and their totals.
struct Sums {
  int64_t a, b;
};
__device__ __forceinline__ Sums block_exclusive(Sums mine, Sums* warp_sums, Sums& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  Sums x = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t a = __shfl_up_sync(0xffffffffu, x.a, o), b = __shfl_up_sync(0xffffffffu, x.b, o);
    if (lane >= o) {
      x.a += a;
      x.b += b;
    }
  }
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  if (warp == 0) {
    Sums w = lane < warps ? warp_sums[lane] : Sums{0, 0};
    const Sums own = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t a = __shfl_up_sync(0xffffffffu, w.a, o), b = __shfl_up_sync(0xffffffffu, w.b, o);
      if (lane >= o) {
        w.a += a;
        w.b += b;
      }
    }
    if (lane == 31) warp_sums[32] = w;
    if (lane < warps) warp_sums[lane] = {w.a - own.a, w.b - own.b};
  }
  __syncthreads();
  total = warp_sums[32];
  const Sums base = warp_sums[warp];
  __syncthreads();                       // warp_sums may be written again
  return {base.a + x.a - mine.a, base.b + x.b - mine.b};
}

// last r with prefix[r] <= t, for prefix[0] <= t < prefix[rows]
__device__ __forceinline__ int row_of(const int32_t* prefix, int rows, int64_t t) {
  int lo = 0, hi = rows;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (prefix[mid] <= t) lo = mid;
    else hi = mid;
  }
  return lo;
}

struct TableParams {
  const int32_t* wanted;                 // new tokens, or tokens to keep
  int32_t* lengths;
  int32_t* table;
  int64_t table_row;
  int32_t* free_blocks;
  int32_t* free_count;
  int requests, width, blocks, log_block;
  int64_t slots;
  int64_t* slot_map;
  int32_t* positions;
  int32_t* cu;
  int32_t* shortage;
  int32_t* off;                          // [requests + 1] blocks popped (pushed) in front of a request's
  int32_t* base;                         // free blocks before the call, or -1: nothing was reserved
};

__device__ __forceinline__ int64_t blocks_of(int64_t tokens, int log_block) {
  return (tokens + (1 << log_block) - 1) >> log_block;
}

// Slots first, first + step, ... of the map.  A fresh block starts with the token at its offset 0, whose thread also enters
// it in the table: fresh blocks come off the stack, so no thread reads an entry that another one writes.
__device__ __forceinline__ void fill_slots(const TableParams& p, const int32_t* cu, int64_t first, int64_t step) {
  const int64_t base = *p.base;
  const int64_t used = base < 0 ? 0 : cu[p.requests];
  for (int64_t t = first; t < p.slots; t += step) {
    int64_t slot = -1, pos = 0;
    if (t < used) {
      const int r = row_of(cu, p.requests, t);
      const int64_t start = (int64_t)p.lengths[r] - (cu[r + 1] - cu[r]);       // lengths are those after the call
      pos = start + (t - cu[r]);
      const int64_t j = pos >> p.log_block, had = blocks_of(start, p.log_block), in = pos & ((1 << p.log_block) - 1);
      int32_t* entry = p.table + r * p.table_row + j;
      int32_t block;
      if (j < had) {
        block = *entry;
      } else {
        block = p.free_blocks[base - 1 - (p.off[r] + (j - had))];
        if (in == 0) *entry = block;
      }
      slot = ((int64_t)block << p.log_block) + in;
    }
    p.slot_map[t] = slot;
    p.positions[t] = (int32_t)pos;
  }
}

// New tokens n_r of every request: cu_seqlens = prefix sums of n_r; blocks needed = ceil((len + n) / B) - ceil(len / B),
// popped from the stack in request order.  All or nothing: a short pool, a narrow table or too few slots change nothing.
// One block of threads, which latency bounds; with `fill` it writes the slot map too, else reserve_fill_kernel does.
__global__ void __launch_bounds__(kTableThreads) reserve_kernel(TableParams p, int fill) {
  __shared__ Sums warp_sums[33];
  __shared__ int32_t cu_s[kSearchRows + 1];
  __shared__ int too_wide;
  if (threadIdx.x == 0) too_wide = 0;
  griddep_wait();
  griddep_launch();
  __syncthreads();
  const int64_t avail = min(max(*p.free_count, 0), p.blocks);
  auto counts = [&](int r, int64_t& len, int64_t& n) -> Sums {
    len = n = 0;
    if (r >= p.requests) return {0, 0};
    len = max(p.lengths[r], 0);
    n = max(p.wanted[r], 0);
    const int64_t want = blocks_of(len + n, p.log_block);
    // (a later chunk of requests would find lengths of an earlier one updated; each thread updates only what it has read)
    if (want > p.width || len + n > INT32_MAX) too_wide = 1;
    return {n, want - blocks_of(len, p.log_block)};
  };
  // totals first: all or nothing
  Sums total{0, 0}, part;
  int64_t len, n;
  for (int r0 = 0; r0 < p.requests; r0 += kTableThreads) {
    block_exclusive(counts(r0 + threadIdx.x, len, n), warp_sums, part);
    total.a += part.a;
    total.b += part.b;
  }
  const bool ok = total.a <= p.slots && total.b <= avail && !too_wide;
  Sums run{0, 0};
  int32_t* cu = p.requests <= kSearchRows ? cu_s : p.cu;
  for (int r0 = 0; r0 < p.requests; r0 += kTableThreads) {
    const int r = r0 + threadIdx.x;
    const Sums mine = counts(r, len, n);
    const Sums at = block_exclusive(mine, warp_sums, part);
    if (r < p.requests) {
      const int32_t c = ok ? (int32_t)(run.a + at.a) : 0;
      p.cu[r] = c;
      cu[r] = c;
      p.off[r] = (int32_t)(run.b + at.b);
      if (ok) p.lengths[r] = (int32_t)(len + n);
    }
    run.a += part.a;
    run.b += part.b;
  }
  if (threadIdx.x == 0) {
    p.cu[p.requests] = cu[p.requests] = ok ? (int32_t)total.a : 0;
    *p.base = ok ? (int32_t)avail : -1;
    *p.shortage = ok ? 0 : 1;
    if (ok) *p.free_count = (int32_t)(avail - total.b);
  }
  __syncthreads();                       // lengths, off and base for the whole block
  if (fill) fill_slots(p, cu, threadIdx.x, kTableThreads);
}

__global__ void __launch_bounds__(256) reserve_fill_kernel(TableParams p) {
  __shared__ int32_t cu_s[kSearchRows + 1];
  griddep_wait();
  griddep_launch();
  const int32_t* cu = p.cu;
  if (p.requests <= kSearchRows) {
    for (int i = threadIdx.x; i <= p.requests; i += blockDim.x) cu_s[i] = p.cu[i];
    __syncthreads();
    cu = cu_s;
  }
  fill_slots(p, cu, (int64_t)blockIdx.x * blockDim.x + threadIdx.x, (int64_t)gridDim.x * blockDim.x);
}

// Freed blocks first, first + step, ...: the last one popped goes back first, so a trim to the lengths before a
// reservation leaves the stack as that found it.
__device__ __forceinline__ void push_blocks(const TableParams& p, const int32_t* off, int64_t first, int64_t step) {
  const int64_t gone = off[p.requests], top = (int64_t)*p.base + gone - 1;
  for (int64_t f = first; f < gone; f += step) {
    const int r = row_of(off, p.requests, f);
    int32_t* entry = p.table + r * p.table_row + blocks_of(p.lengths[r], p.log_block) + (f - off[r]);
    if (top - f < p.blocks) p.free_blocks[top - f] = *entry;
    *entry = -1;
  }
}

__global__ void __launch_bounds__(kTableThreads) trim_kernel(TableParams p, int fill) {
  __shared__ Sums warp_sums[33];
  __shared__ int32_t off_s[kSearchRows + 1];
  griddep_wait();
  griddep_launch();
  const int64_t avail = min(max(*p.free_count, 0), p.blocks);
  int32_t* off = p.requests <= kSearchRows ? off_s : p.off;
  int64_t run = 0;
  for (int r0 = 0; r0 < p.requests; r0 += kTableThreads) {
    const int r = r0 + threadIdx.x;
    int64_t len = 0, keep = 0;
    if (r < p.requests) {
      // no more than the table holds, whatever the lengths say: the entries beyond are not this request's
      len = min((int64_t)max(p.lengths[r], 0), (int64_t)p.width << p.log_block);
      keep = min((int64_t)max(p.wanted[r], 0), len);
    }
    Sums part;
    const Sums at = block_exclusive({blocks_of(len, p.log_block) - blocks_of(keep, p.log_block), 0}, warp_sums, part);
    if (r < p.requests) {
      off[r] = p.off[r] = (int32_t)(run + at.a);
      p.lengths[r] = (int32_t)keep;
    }
    run += part.a;
  }
  if (threadIdx.x == 0) {
    off[p.requests] = p.off[p.requests] = (int32_t)run;
    *p.base = (int32_t)avail;
    *p.free_count = (int32_t)min(avail + run, (int64_t)p.blocks);
  }
  __syncthreads();
  if (fill) push_blocks(p, off, threadIdx.x, kTableThreads);
}

__global__ void __launch_bounds__(256) trim_push_kernel(TableParams p) {
  __shared__ int32_t off_s[kSearchRows + 1];
  griddep_wait();
  griddep_launch();
  const int32_t* off = p.off;
  if (p.requests <= kSearchRows) {
    for (int i = threadIdx.x; i <= p.requests; i += blockDim.x) off_s[i] = p.off[i];
    __syncthreads();
    off = off_s;
  }
  push_blocks(p, off, (int64_t)blockIdx.x * blockDim.x + threadIdx.x, (int64_t)gridDim.x * blockDim.x);
}

// ------------------------------------------------------------------------------------------ write
struct WriteParams {
  const void* x[2];                      // keys, values
  int64_t st[2], sh[2];                  // element strides of token and head
  uint8_t* cache[2];
  int64_t block[2];                      // bytes from block to block
  float* scale[2];
  int64_t scale_block[2];
  const int64_t* slot_map;
  int64_t tokens, slots;
  int log_block;
};

constexpr int kWriteThreads = 256;
constexpr int kMaxBlock = 128;

// A block of threads per (window of tokens, head, K or V).  Tokens of one cache block that follow each other are a run;
// the window that holds a run's first token does the whole of it.  Per run: maximum of its values, scale, older codes of
// the block rounded again where the scale has grown, codes of the run.  HBM bounds long prompts: every value is read once
// (the first kHold rows of a thread stay in registers, others come from L1 or L2), every code written once; single tokens
// are bound by three dependent trips to memory (slots, values and scale, codes).
template <typename T, int D, int W>
__global__ void __launch_bounds__(kWriteThreads) kv8_write_kernel(WriteParams p) {
  constexpr int kPer = 16 / sizeof(T);                       // values of a 16-byte load
  constexpr int kLoads = D / kPer;                           // loads of a row
  constexpr int kLanes = kLoads < 32 ? kLoads : 32, kVec = kLoads / kLanes;
  constexpr int kRows = kWriteThreads / kLanes;              // rows of a pass of the block
  constexpr int kHold = sizeof(T) == 4 ? 2 : 4;
  constexpr int kSpan = W + kMaxBlock;
  static_assert(kSpan <= kWriteThreads, "one thread looks at one token");
  __shared__ int64_t slot_s[kSpan + 1];                      // slot of token t0 - 1 + i, or -1
  __shared__ int lead_s[kSpan];                              // first token of the token's run, or -1
  __shared__ uint32_t amax_s[W];                             // of the run that starts there
  __shared__ float scale_s[W], ratio_s[W];
  __shared__ int warp_last[kWriteThreads / 32], grown_s[W], n_grown, end_s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int kv = blockIdx.z, head = blockIdx.y;
  const int64_t t0 = (int64_t)blockIdx.x * W;
  const int bs = 1 << p.log_block;
  if (tid == 0) n_grown = 0;
  if (tid < W) amax_s[tid] = 0;
  griddep_wait();
  griddep_launch();
  if (tid <= kSpan) {
    const int64_t t = t0 - 1 + tid;
    const int64_t s = t >= 0 && t < p.tokens ? p.slot_map[t] : -1;
    slot_s[tid] = s < p.slots ? s : -1;
  }
  if (tid == 0) end_s = kSpan;
  __syncthreads();
  // runs: a token leads one where its slot does not follow the slot before, or opens a block
  const bool in = tid < kSpan;
  const int64_t slot = in ? slot_s[tid + 1] : -1;
  const bool valid = slot >= 0;
  const bool leads = valid && (slot_s[tid] < 0 || slot != slot_s[tid] + 1 || (slot & (bs - 1)) == 0);
  int lead = leads ? tid : -1;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int before = __shfl_up_sync(0xffffffffu, lead, o);
    if (lane >= o) lead = max(lead, before);
  }
  if (lane == 31) warp_last[warp] = lead;
  // the window ends behind the last run that starts in it
  if (in && tid >= W && (leads || !valid)) atomicMin(&end_s, tid);
  __syncthreads();
  for (int w = 0; w < warp; ++w) lead = max(lead, warp_last[w]);
  if (in) lead_s[tid] = valid ? lead : -1;
  __syncthreads();
  const int end = end_s;

  const T* x = static_cast<const T*>(p.x[kv]) + head * p.sh[kv];
  const int row0 = tid / kLanes, col = (tid % kLanes) * kPer;
  auto values = [&](int i, uint4 (&raw)[kVec]) {
    const T* px = x + (t0 + i) * p.st[kv] + col;
#pragma unroll
    for (int v = 0; v < kVec; ++v) raw[v] = *reinterpret_cast<const uint4*>(px + v * kLanes * kPer);
  };
  auto unpack = [](const uint4& raw, float (&f)[kPer]) {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (std::is_same<T, float>::value) {
        f[k] = __uint_as_float(w[k]);
      } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        f[2 * k] = __uint_as_float(w[k] << 16);
        f[2 * k + 1] = __uint_as_float(w[k] & 0xFFFF0000u);
      } else {
        const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&w[k]));
        f[2 * k] = h.x;
        f[2 * k + 1] = h.y;
      }
    }
  };
  auto measure = [&](int i, const uint4 (&raw)[kVec]) {
    uint32_t m = 0;
#pragma unroll
    for (int v = 0; v < kVec; ++v) {
      float f[kPer];
      unpack(raw[v], f);
#pragma unroll
      for (int k = 0; k < kPer; ++k) m = max(m, kv8_magnitude(f[k]));
    }
    if (m != 0) atomicMax(&amax_s[lead_s[i]], m);            // a maximum: no order
  };
  auto store = [&](int i, const uint4 (&raw)[kVec]) {
    const int run = lead_s[i];
    const int64_t s = slot_s[i + 1];
    uint8_t* pc = p.cache[kv] + (s >> p.log_block) * p.block[kv] + ((int64_t)head * bs + (s & (bs - 1))) * D + col;
    const float sc = scale_s[run], inv = ratio_s[run];
#pragma unroll
    for (int v = 0; v < kVec; ++v) {
      float f[kPer];
      unpack(raw[v], f);
      if (inv != 0.0f) {
#pragma unroll
        for (int k = 0; k < kPer; ++k) f[k] *= inv;
      } else {
#pragma unroll 1
        for (int k = 0; k < kPer; ++k) f[k] = __fdiv_rn(f[k], sc);
      }
      uint32_t w[kPer / 4];
#pragma unroll
      for (int k = 0; k < kPer / 4; ++k) w[k] = e4m3x4(f[4 * k], f[4 * k + 1], f[4 * k + 2], f[4 * k + 3]);
      if constexpr (kPer == 8) *reinterpret_cast<uint2*>(pc) = make_uint2(w[0], w[1]);
      else *reinterpret_cast<uint32_t*>(pc + v * kLanes * kPer) = w[0];
    }
  };
  uint4 held[kHold][kVec];
#pragma unroll
  for (int k = 0; k < kHold; ++k) {
    const int i = row0 + k * kRows;
    if (i < end && lead_s[i] >= 0) values(i, held[k]);
  }
#pragma unroll
  for (int k = 0; k < kHold; ++k) {
    const int i = row0 + k * kRows;
    if (i < end && lead_s[i] >= 0) measure(i, held[k]);
  }
  for (int i = row0 + kHold * kRows; i < end; i += kRows) {
    uint4 raw[kVec];
    if (lead_s[i] >= 0) {
      values(i, raw);
      measure(i, raw);
    }
  }
  __syncthreads();
  // scale of every run, and the runs whose block holds codes of a smaller one
  if (tid < W && lead_s[tid] == tid) {
    const int64_t s = slot_s[tid + 1];
    float* ps = p.scale[kv] + (s >> p.log_block) * p.scale_block[kv] + head;
    float now = kv8_scale(amax_s[tid]);
    if ((s & (bs - 1)) != 0) {
      const float was = *ps;
      if (was >= now) {
        now = was;
      } else {
        grown_s[atomicAdd(&n_grown, 1)] = tid;
        amax_s[tid] = __float_as_uint(was);
        *ps = now;
      }
    } else {
      *ps = now;
    }
    scale_s[tid] = now;
    // the reciprocal of a power of two is exact; a scale that something else wrote is divided by
    ratio_s[tid] = (__float_as_uint(now) & 0x7FFFFFu) == 0 && now <= 0x1p126f && now >= 0x1p-126f ? 1.0f / now : 0.0f;
  }
  __syncthreads();
  for (int gi = 0; gi < n_grown; ++gi) {
    const int run = grown_s[gi];
    const int64_t s = slot_s[run + 1];
    const float was = __uint_as_float(amax_s[run]), now = scale_s[run];
    uint4* pc = reinterpret_cast<uint4*>(p.cache[kv] + (s >> p.log_block) * p.block[kv] + (int64_t)head * bs * D);
    for (int c = tid; c < (int)(s & (bs - 1)) * (D / 16); c += kWriteThreads) {
      uint4 v = pc[c];
      uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        uint32_t lo, hi;
        half4_of_e4m3x4(w[k], lo, hi);
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo));
        const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
        w[k] = e4m3x4(__fdiv_rn(a.x * was, now), __fdiv_rn(a.y * was, now), __fdiv_rn(b.x * was, now),
                      __fdiv_rn(b.y * was, now));
      }
      pc[c] = v;
    }
  }
#pragma unroll
  for (int k = 0; k < kHold; ++k) {
    const int i = row0 + k * kRows;
    if (i < end && lead_s[i] >= 0) store(i, held[k]);
  }
  for (int i = row0 + kHold * kRows; i < end; i += kRows) {
    uint4 raw[kVec];
    if (lead_s[i] >= 0) {
      values(i, raw);
      store(i, raw);
    }
  }
}

template <typename T, int D>
int launch_write(const WriteParams& p, int64_t hk, cudaStream_t st) {
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  const int64_t wide = (p.tokens + 63) / 64;
  if (wide * hk * 2 >= 2 * sms)
    return launch_streaming("nvfp4_kv8_write", kv8_write_kernel<T, D, 64>, dim3((unsigned)wide, (unsigned)hk, 2), kWriteThreads, 0,
                            st, p);
  return launch_streaming("nvfp4_kv8_write", kv8_write_kernel<T, D, 16>, dim3((unsigned)((p.tokens + 15) / 16), (unsigned)hk, 2),
                          kWriteThreads, 0, st, p);
}

int log2_block(int block_size) {
  switch (block_size) {
    case 16: return 4;
    case 32: return 5;
    case 64: return 6;
    case 128: return 7;
    default: return -1;
  }
}

// slots (tokens) that one launch of a single block of threads fills, and table entries that it can be asked to give back
constexpr int64_t kSingleFill = 4096;

}  // namespace
}  // namespace nvfp4

using namespace nvfp4;

extern "C" int nvfp4_paged_reserve(const int32_t* new_lens, int32_t* lengths, int32_t* table, int64_t table_row,
                                   const int32_t* free_blocks, int32_t* free_count, int64_t requests, int64_t width,
                                   int64_t blocks, int block_size, int64_t slots, int64_t* slot_map, int32_t* positions,
                                   int32_t* cu_seqlens, int32_t* shortage, int32_t* workspace, nvfp4_stream_t stream) {
  const int lb = log2_block(block_size);
  NVFP4_REQUIRE(lb >= 0, "nvfp4_paged_reserve: block_size must be 16, 32, 64 or 128");
  NVFP4_REQUIRE(requests >= 1 && requests < (1 << 30) && width >= 1 && width < (1 << 30) && blocks >= 0 && blocks < INT32_MAX,
                "nvfp4_paged_reserve: sizes out of range");
  NVFP4_REQUIRE(slots >= 0 && slots < INT32_MAX, "nvfp4_paged_reserve: slot count out of range");
  TableParams p{new_lens, lengths, table, table_row, const_cast<int32_t*>(free_blocks), free_count, (int)requests, (int)width,
                (int)blocks, lb, slots, slot_map, positions, cu_seqlens, shortage, workspace, workspace + requests + 1};
  const bool one = slots <= kSingleFill;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  int rc = launch("nvfp4_paged_reserve", reserve_kernel, dim3(1), kTableThreads, 0, st, p, one ? 1 : 0);
  if (rc != 0 || one) return rc;
  const int64_t grid = (slots + 1023) / 1024;
  return launch("nvfp4_paged_reserve", reserve_fill_kernel, dim3((unsigned)(grid < 1184 ? grid : 1184)), 256, 0, st, p);
}

extern "C" int nvfp4_paged_trim(const int32_t* keep_lens, int32_t* lengths, int32_t* table, int64_t table_row,
                                int32_t* free_blocks, int32_t* free_count, int64_t requests, int64_t width, int64_t blocks,
                                int block_size, int32_t* workspace, nvfp4_stream_t stream) {
  const int lb = log2_block(block_size);
  NVFP4_REQUIRE(lb >= 0, "nvfp4_paged_trim: block_size must be 16, 32, 64 or 128");
  NVFP4_REQUIRE(requests >= 1 && requests < (1 << 30) && width >= 1 && width < (1 << 30) && blocks >= 0 && blocks < INT32_MAX,
                "nvfp4_paged_trim: sizes out of range");
  NVFP4_REQUIRE(requests * width < INT32_MAX, "nvfp4_paged_trim: the table has too many entries");
  TableParams p{keep_lens, lengths, table, table_row, free_blocks, free_count, (int)requests, (int)width, (int)blocks, lb, 0,
                nullptr, nullptr, nullptr, nullptr, workspace, workspace + requests + 1};
  const bool one = requests * width <= kSingleFill;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  int rc = launch("nvfp4_paged_trim", trim_kernel, dim3(1), kTableThreads, 0, st, p, one ? 1 : 0);
  if (rc != 0 || one) return rc;
  const int64_t grid = (requests * width + 1023) / 1024;
  return launch("nvfp4_paged_trim", trim_push_kernel, dim3((unsigned)(grid < 148 ? grid : 148)), 256, 0, st, p);
}

extern "C" int nvfp4_kv8_write(const void* key, const void* value, int dtype, int64_t tokens, int64_t hk, int d, int64_t skt,
                               int64_t skh, int64_t svt, int64_t svh, const int64_t* slot_map, uint8_t* k_cache,
                               int64_t k_block, uint8_t* v_cache, int64_t v_block, float* k_scale, int64_t ks_block,
                               float* v_scale, int64_t vs_block, int64_t blocks, int block_size, nvfp4_stream_t stream) {
  const int lb = log2_block(block_size);
  NVFP4_REQUIRE(lb >= 0, "nvfp4_kv8_write: block_size must be 16, 32, 64 or 128");
  NVFP4_REQUIRE(d == 128 || d == 256, "nvfp4_kv8_write: D must be 128 or 256");
  NVFP4_REQUIRE(tokens >= 0 && tokens < (1ll << 31) && hk >= 1 && hk <= 65535 && blocks >= 0, "nvfp4_kv8_write: sizes out of range");
  const int64_t size = dtype == NVFP4_DT_FP32 ? 4 : 2;
  NVFP4_REQUIRE((((uintptr_t)key | (uintptr_t)value) & 15) == 0 && ((skt | skh | svt | svh) * size & 15) == 0,
                "nvfp4_kv8_write: rows of keys and values must be 16-byte aligned");
  NVFP4_REQUIRE((((uintptr_t)k_cache | (uintptr_t)v_cache) & 15) == 0 && ((k_block | v_block) & 15) == 0,
                "nvfp4_kv8_write: cache blocks must be 16-byte aligned");
  if (tokens == 0) return 0;
  const WriteParams p{{key, value}, {skt, svt}, {skh, svh}, {k_cache, v_cache}, {k_block, v_block}, {k_scale, v_scale},
                      {ks_block, vs_block}, slot_map, tokens, blocks << lb, lb};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case NVFP4_DT_BF16: return d == 128 ? launch_write<__nv_bfloat16, 128>(p, hk, st) : launch_write<__nv_bfloat16, 256>(p, hk, st);
    case NVFP4_DT_FP16: return d == 128 ? launch_write<__half, 128>(p, hk, st) : launch_write<__half, 256>(p, hk, st);
    case NVFP4_DT_FP32: return d == 128 ? launch_write<float, 128>(p, hk, st) : launch_write<float, 256>(p, hk, st);
  }
  return fail(-1, "nvfp4_kv8_write: unknown dtype %d", dtype);
}
