// Paged 8-bit KV cache: block tables and slot maps from request lengths, and the quantising write.
#include <limits.h>
#include <type_traits>
#include "common/abi.cuh"
#include "common/fp4.cuh"
#include "common/kv8.cuh"
#include "common/launch.cuh"
#include "common/sm100.cuh"

namespace nvfp4 {
namespace {

// ------------------------------------------------------------------------------------------ tables
constexpr int kTableThreads = 1024;
constexpr int kSearchRows = 2048;        // prefix sums of as many requests are searched in shared memory
constexpr int64_t kAlone = 8192;         // entries that one block of threads sees to

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
  int32_t* scratch;                      // [requests + 2] prefix sums of blocks, where one kernel hands them to another
};

__device__ __forceinline__ int64_t blocks_of(int64_t tokens, int log_block) {
  return (tokens + (1 << log_block) - 1) >> log_block;
}

// All blocks of threads of a kernel that is one cluster.
__device__ __forceinline__ void all_blocks() {
  if (gridDim.z > 1) cluster_sync_all();
  else __syncthreads();
}

// Slots and positions, by warps `warp`, `warp` + `warps`, ...: a thread has four tokens 32 apart (four neighbours would be stores of
// 32 sectors an instruction), whose look-ups are under way together.  A fresh block starts with the token at its offset 0,
// whose thread also enters it in the table: fresh blocks come off the stack, so no thread reads an entry that another one
// writes.  start_of(r): tokens that request r held.
template <typename F>
__device__ __forceinline__ void fill_slots(const TableParams& p, const int32_t* cu, const int32_t* off, int avail, int used, int warp,
                                           int warps, F start_of) {
  constexpr int kFour = 4;
  const int slots = (int)p.slots, mask = (1 << p.log_block) - 1;
  int r = -1, next = 0, begin = 0, had = 0;                // request of the last token: its end, position 0, blocks it had
  const int32_t* fresh = nullptr;                          // where its block j comes from: fresh[-j]
  int32_t* row = nullptr;
  for (int64_t t0 = 32 * kFour * (int64_t)warp + (threadIdx.x & 31); t0 < slots; t0 += 32 * kFour * (int64_t)warps) {
    int32_t* entry[kFour];
    const int32_t* from[kFour];
    int block[kFour], pos[kFour];
#pragma unroll
    for (int x = 0; x < kFour; ++x) {
      const int t = (int)t0 + 32 * x;
      from[x] = nullptr;
      pos[x] = 0;
      if (t < used) {
        if (t >= next) {
          // the request behind, mostly
          if (r >= 0 && t < cu[r + 2 <= p.requests ? r + 2 : p.requests]) ++r;
          else r = row_of(cu, p.requests, t);
          const int start = start_of(r);
          next = cu[r + 1];
          begin = start - cu[r];
          had = (int)blocks_of(start, p.log_block);
          row = p.table + r * p.table_row;
          fresh = p.free_blocks + ((int64_t)avail - 1 - (off[r] - had));
        }
        pos[x] = begin + t;
        const int j = pos[x] >> p.log_block;
        entry[x] = row + j;
        from[x] = j < had ? entry[x] : fresh - j;
      }
    }
#pragma unroll
    for (int x = 0; x < kFour; ++x) block[x] = from[x] != nullptr ? *from[x] : -1;
#pragma unroll
    for (int x = 0; x < kFour; ++x) {
      const int t = (int)t0 + 32 * x;
      if (t >= slots) break;
      const int in = pos[x] & mask;
      if (from[x] != nullptr && in == 0) *entry[x] = block[x];
      p.slot_map[t] = from[x] != nullptr ? ((int64_t)block[x] << p.log_block) + in : -1;
      p.positions[t] = pos[x];
    }
  }
}

// New tokens n_r of every request: cu_seqlens = prefix sums of n_r; blocks needed = ceil((len + n) / B) - ceil(len / B),
// popped from the stack in request order.  All or nothing: a short pool, a narrow table or too few slots change nothing.
// One block of threads, whose latency is what it costs; a long list of slots is filled by reserve_fill_kernel behind it.  (As
// one cluster of eight, 200000 slots of 512 requests took 22 us: 90 instructions a token on eight SMs.)
__global__ void __launch_bounds__(kTableThreads) reserve_kernel(TableParams p, int fill) {
  __shared__ Sums warp_sums[33];
  __shared__ int32_t cu_s[kSearchRows + 1], off_s[kSearchRows + 1], len_s[kSearchRows];
  __shared__ int too_wide;
  const int tid = threadIdx.x, threads = blockDim.x;
  if (tid == 0) too_wide = 0;
  griddep_wait();
  griddep_launch();
  __syncthreads();
  const int avail = min(max(*p.free_count, 0), p.blocks);
  const bool in_smem = p.requests <= kSearchRows;
  auto counts = [&](int r) -> Sums {
    if (r >= p.requests) return {0, 0};
    const int64_t len = max(p.lengths[r], 0), n = max(p.wanted[r], 0), want = blocks_of(len + n, p.log_block);
    if (in_smem) len_s[r] = (int)len;
    if (want > p.width || len + n > INT32_MAX) too_wide = 1;
    return {n, want - blocks_of(len, p.log_block)};
  };
  // prefix sums of tokens and of blocks
  int32_t* cu = in_smem ? cu_s : p.cu;
  int32_t* off = in_smem ? off_s : p.scratch + 1;
  Sums total{0, 0};
  for (int r0 = 0; r0 < p.requests; r0 += threads) {
    Sums part;
    const Sums at = block_exclusive(counts(r0 + tid), warp_sums, part);
    if (r0 + tid < p.requests) {
      cu[r0 + tid] = (int32_t)min(total.a + at.a, (int64_t)INT32_MAX);
      off[r0 + tid] = (int32_t)min(total.b + at.b, (int64_t)INT32_MAX);
    }
    total.a += part.a;
    total.b += part.b;
  }
  const bool ok = total.a <= p.slots && total.b <= avail && !too_wide;
  if (tid == 0) cu[p.requests] = (int32_t)min(total.a, (int64_t)INT32_MAX);
  __syncthreads();
  if (fill)
    fill_slots(p, cu, off, avail, ok ? (int)total.a : 0, tid >> 5, threads >> 5,
               [&](int r) { return in_smem ? len_s[r] : max(p.lengths[r], 0); });
  __syncthreads();                       // lengths and, of many requests, p.cu have been read
  for (int r = tid; r <= p.requests; r += threads) {
    p.cu[r] = ok ? cu[r] : 0;
    if (r == p.requests) break;
    if (!fill) p.scratch[1 + r] = off[r];
    if (ok) p.lengths[r] = max(p.lengths[r], 0) + max(p.wanted[r], 0);
  }
  if (tid == 0) {
    *p.shortage = ok ? 0 : 1;
    if (ok) *p.free_count = (int32_t)(avail - total.b);
    if (!fill) p.scratch[0] = avail;
  }
}

__global__ void __launch_bounds__(256) reserve_fill_kernel(TableParams p) {
  __shared__ int32_t cu_s[kSearchRows + 1], off_s[kSearchRows + 1];
  griddep_wait();
  griddep_launch();
  const int32_t* cu = p.cu;
  const int32_t* off = p.scratch + 1;
  if (p.requests <= kSearchRows) {
    for (int i = threadIdx.x; i <= p.requests; i += blockDim.x) {
      cu_s[i] = cu[i];
      if (i < p.requests) off_s[i] = off[i];
    }
    __syncthreads();
    cu = cu_s;
    off = off_s;
  }
  const int warps = blockDim.x >> 5;
  fill_slots(p, cu, off, p.scratch[0], cu[p.requests], (int)blockIdx.x * warps + (threadIdx.x >> 5), (int)gridDim.x * warps,
             [&](int r) { return p.lengths[r] - (cu[r + 1] - cu[r]); });
}

// Every request keeps its first tokens.  A cluster: every block of threads makes the prefix sums for itself and does its share of
// the entries, the first one updates lengths and stack when all have read them.  Freed blocks go on the stack with the last one popped first, so a trim to the lengths
// before a reservation leaves the stack as that found it.
__global__ void __launch_bounds__(kTableThreads) trim_kernel(TableParams p) {
  __shared__ Sums warp_sums[33];
  __shared__ int32_t off_s[kSearchRows + 1], stay_s[kSearchRows];
  const int tid = threadIdx.x, threads = blockDim.x;
  const bool first = blockIdx.z == 0;
  griddep_wait();
  griddep_launch();
  const int64_t avail = min(max(*p.free_count, 0), p.blocks);
  // no more than the table holds, whatever the lengths say: the entries beyond are not this request's
  auto held = [&](int r) { return min((int64_t)max(p.lengths[r], 0), (int64_t)p.width << p.log_block); };
  auto kept = [&](int r) { return min((int64_t)max(p.wanted[r], 0), held(r)); };
  const bool in_smem = p.requests <= kSearchRows;
  int32_t* off = in_smem ? off_s : p.scratch;
  int64_t gone = 0;
  for (int r0 = 0; r0 < p.requests; r0 += threads) {
    const int r = r0 + tid;
    Sums part;
    int64_t mine = 0;
    if (r < p.requests) {
      const int64_t stay = blocks_of(kept(r), p.log_block);
      if (in_smem) stay_s[r] = (int)stay;
      mine = blocks_of(held(r), p.log_block) - stay;
    }
    const Sums at = block_exclusive({mine, 0}, warp_sums, part);
    if (r < p.requests && (in_smem || first)) off[r] = (int32_t)(gone + at.a);
    gone += part.a;
  }
  if (tid == 0 && (in_smem || first)) off[p.requests] = (int32_t)gone;
  if (in_smem) __syncthreads();
  else all_blocks();
  const int64_t top = avail + gone - 1;
  for (int64_t f = (int64_t)blockIdx.z * threads + tid; f < gone; f += (int64_t)gridDim.z * threads) {
    const int r = row_of(off, p.requests, f);
    int32_t* entry = p.table + r * p.table_row + (in_smem ? stay_s[r] : blocks_of(kept(r), p.log_block)) + (f - off[r]);
    if (top - f < p.blocks) p.free_blocks[top - f] = *entry;
    *entry = -1;
  }
  all_blocks();
  if (!first) return;
  for (int r = tid; r < p.requests; r += threads) p.lengths[r] = (int32_t)kept(r);
  if (tid == 0) *p.free_count = (int32_t)min(avail + gone, (int64_t)p.blocks);
}

unsigned table_threads(int64_t entries, int64_t requests) {
  const int64_t most = entries > requests ? entries : requests;
  unsigned threads = 128;
  while (threads < kTableThreads && threads < most) threads *= 2;
  return threads;
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
  int log_block, operands, per;          // operands: key head 0, value head 0, key head 1, ...
};

constexpr int kWriteThreads = 256;
constexpr int kMaxBlock = 128;

// A block of threads per window of W tokens and `per` of the 2 Hk operands (a head's keys, its values).  Tokens of one cache
// block that follow each other are a run; the window that holds a run's first token does the whole of it.  Which tokens
// make runs is found once; then, operand by operand: maximum of every run's values, scale, older codes of the block
// rounded again where the scale has grown, codes of the run, while the next operand's values are on their way into shared
// memory (every thread copies what it will use itself).  What is copied are the W tokens from the window's first run on: blocks
// begin anywhere in a window, and with the window's own tokens half of what it has to do lay behind them.  So every value
// is read once (but for what is behind those, of windows of many short runs) and every code written once.  Single tokens
// (kSmall) are bound by dependent trips to memory (slots, scale, codes) and copied before it is known whose they are.
// Measured: 17000 tokens of Hk 8 D 128 in bf16, 105 MB, 31.3 us = 3.35 TB/s, half of the copy rate: 1130 instructions a warp,
// issue 0.67; one token of each of many requests 4 us, 2.2 in a graph.
template <typename T, int D, int W, bool kSmall>
__global__ void __launch_bounds__(kWriteThreads) kv8_write_kernel(WriteParams p) {
  constexpr int kPer = 16 / sizeof(T);                       // values of a 16-byte load
  constexpr int kLoads = D / kPer;                           // loads of a row
  constexpr int kLanes = kLoads < 32 ? kLoads : 32, kVec = kLoads / kLanes;
  constexpr int kRows = kWriteThreads / kLanes;              // rows of a pass of the block
  constexpr int kHold = (W + kRows - 1) / kRows;             // rows of the window that a thread sees to
  constexpr int kSpan = W + kMaxBlock - 1;                   // tokens that runs of the window can reach
  static_assert(kSpan + 1 <= kWriteThreads, "one thread fetches one slot, that in front of the window among them");
  // [2][W rows].  Where it begins inside a sector, as behind the static words it may, prompts take 34.1 us instead of 31.3.
  extern __shared__ __align__(128) uint8_t values_s[];
  struct Run {
    int64_t block;                                           // of the cache
    int at;                                                  // offset of the run's token 0 in it, less its place in the window
    float scale, inv;                                        // inv 0: divide
  };
  __shared__ int64_t slot_s[kSpan + 1];                      // slot of token t0 - 1 + i, or -1
  __shared__ int lead_s[kSpan];                              // first token of the token's run, or -1
  __shared__ Run run_s[W];                                   // by first token
  __shared__ uint32_t amax_s[2][W];
  __shared__ int warp_last[kWriteThreads / 32], grown_s[W], n_grown[2], begin_s, end_s;
  __shared__ float was_s[W];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t t0 = (int64_t)blockIdx.x * W;
  const int bs = 1 << p.log_block;
  if (tid < 2) n_grown[tid] = 0;
  if (tid < W) amax_s[0][tid] = amax_s[1][tid] = 0;
  const int row0 = tid / kLanes, col = (tid % kLanes) * kPer;
  auto values = [&](int c, int i, uint4 (&raw)[kVec]) {
    const T* px = static_cast<const T*>(p.x[c & 1]) + (c >> 1) * p.sh[c & 1] + (t0 + i) * p.st[c & 1] + col;
#pragma unroll
    for (int v = 0; v < kVec; ++v) raw[v] = *reinterpret_cast<const uint4*>(px + v * kLanes * kPer);
  };
  const uint32_t own = smem_u32(values_s) + row0 * (D * sizeof(T)) + (tid % kLanes) * 16;
  constexpr uint32_t kStage = W * D * sizeof(T), kStep = kRows * D * sizeof(T);
  int shift = 0;                                             // first token copied
  auto fetch = [&](int c, int stage) {
    const T* px = static_cast<const T*>(p.x[c & 1]) + (c >> 1) * p.sh[c & 1] + (t0 + shift + row0) * p.st[c & 1] + col;
    const int64_t step = kRows * p.st[c & 1];
#pragma unroll
    for (int k = 0; k < kHold; ++k, px += step) {
      const int i = row0 + k * kRows;
      if (i < W && t0 + shift + i < p.tokens) {
#pragma unroll
        for (int v = 0; v < kVec; ++v)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(own + stage * kStage + k * kStep + v * kLanes * 16),
                       "l"(px + v * kLanes * kPer)
                       : "memory");
      }
    }
    cp_async_commit();
  };
  auto fetched = [&](int stage, int k, uint4 (&raw)[kVec]) {
#pragma unroll
    for (int v = 0; v < kVec; ++v) {
      const uint32_t a = own + stage * kStage + k * kStep + v * kLanes * 16;
      asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(raw[v].x), "=r"(raw[v].y), "=r"(raw[v].z), "=r"(raw[v].w) : "r"(a) : "memory");
    }
  };
  const int first = blockIdx.y * p.per, last = min(first + p.per, p.operands);
  griddep_wait();
  griddep_launch();
  int64_t my_slot = -1;
  if (tid <= kSpan) {
    const int64_t t = t0 - 1 + tid;
    if (t >= 0 && t < p.tokens) my_slot = p.slot_map[t];
  }
  if (kSmall) {
    fetch(first, 0);
  } else {                                                   // into L2, while it is found out which of them are this block's
    constexpr int kLines = D * (int)sizeof(T) / 128;
    for (int x = tid; x < W * kLines; x += kWriteThreads)
      if (t0 + x / kLines < p.tokens)
        prefetch_l2(reinterpret_cast<const uint8_t*>(static_cast<const T*>(p.x[first & 1]) + (first >> 1) * p.sh[first & 1] +
                                                     (t0 + x / kLines) * p.st[first & 1]) + x % kLines * 128);
  }
  if (tid <= kSpan) slot_s[tid] = my_slot < p.slots ? my_slot : -1;
  if (tid == 0) {
    begin_s = W;
    end_s = kSpan;
  }
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
  if (!kSmall && leads && tid < W) atomicMin(&begin_s, tid);
  const int offset = (int)(slot & (bs - 1));
  if (leads && tid < W) run_s[tid] = {slot >> p.log_block, offset - tid, 0.0f, 0.0f};
  __syncthreads();
  for (int w = 0; w < warp; ++w) lead = max(lead, warp_last[w]);
  if (in) lead_s[tid] = valid ? lead : -1;
  const bool mine = leads && tid < W;                        // this thread settles the scale of the run
  __syncthreads();
  const int end = end_s;
  if (!kSmall) {
    shift = begin_s;
    if (shift == W) return;                                  // no run starts here
    fetch(first, 0);
  }
  int lead_of[kHold];                                        // of this thread's rows
#pragma unroll
  for (int k = 0; k < kHold; ++k) {
    const int i = row0 + k * kRows;
    lead_of[k] = i < W && shift + i < end ? lead_s[shift + i] : -1;
  }
  // one run for all rows of the warp, as blocks of long prompts have it: -1 if there are several
  int only = -1;
  {
    int low = INT_MAX, high = -1;
#pragma unroll
    for (int k = 0; k < kHold; ++k) {
      if (lead_of[k] >= 0) low = min(low, lead_of[k]);
      high = max(high, lead_of[k]);
    }
    low = __reduce_min_sync(0xffffffffu, low);
    high = __reduce_max_sync(0xffffffffu, high);
    if (low == high) only = low;
  }

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
  // Largest magnitude of a thread's values, as float bits.  16-bit types two at a time (a NaN is passed over), and once more
  // one by one where a value is infinite.
  auto measure = [&](const uint4 (&raw)[kVec]) -> uint32_t {
    uint32_t m = 0;
    bool slow = sizeof(T) == 4;
    if constexpr (sizeof(T) == 2) {
      using T2 = typename std::conditional<std::is_same<T, __nv_bfloat16>::value, __nv_bfloat162, __half2>::type;
      constexpr uint32_t kInf = std::is_same<T, __nv_bfloat16>::value ? 0x7F80u : 0x7C00u;
      auto two = [](uint32_t w) { return *reinterpret_cast<const T2*>(&w); };
      T2 t = two(0u);
#pragma unroll
      for (int v = 0; v < kVec; ++v)
        t = __hmax2(t, __hmax2(__hmax2(__habs2(two(raw[v].x)), __habs2(two(raw[v].y))),
                               __hmax2(__habs2(two(raw[v].z)), __habs2(two(raw[v].w)))));
      const uint32_t w = *reinterpret_cast<const uint32_t*>(&t), top = max(w & 0xFFFFu, w >> 16);
      slow = top >= kInf;
      const uint16_t h = (uint16_t)top;
      m = __float_as_uint(to_f32<T>(*reinterpret_cast<const T*>(&h)));
    }
    if (slow) {
      m = 0;
#pragma unroll
      for (int v = 0; v < kVec; ++v) {
        float f[kPer];
        unpack(raw[v], f);
#pragma unroll
        for (int k = 0; k < kPer; ++k) m = max(m, kv8_magnitude(f[k]));
      }
    }
    return m;
  };
  auto store = [&](int c, int i, const Run& run, const uint4 (&raw)[kVec]) {
    uint8_t* pc = p.cache[c & 1] + run.block * p.block[c & 1] + (((c >> 1) << p.log_block) + run.at + i) * D + col;
#pragma unroll
    for (int v = 0; v < kVec; ++v) {
      float f[kPer];
      unpack(raw[v], f);
      if (run.inv != 0.0f) {
#pragma unroll
        for (int k = 0; k < kPer; ++k) f[k] *= run.inv;
      } else {
#pragma unroll
        for (int k = 0; k < kPer; ++k) f[k] = __fdiv_rn(f[k], run.scale);
      }
      uint32_t w[kPer / 4];
#pragma unroll
      for (int k = 0; k < kPer / 4; ++k) w[k] = e4m3x4(f[4 * k], f[4 * k + 1], f[4 * k + 2], f[4 * k + 3]);
      if constexpr (kPer == 8) *reinterpret_cast<uint2*>(pc) = make_uint2(w[0], w[1]);
      else *reinterpret_cast<uint32_t*>(pc + v * kLanes * kPer) = w[0];
    }
  };

  for (int c = first, turn = 0; c < last; ++c, turn ^= 1) {
    float* ps = p.scale[c & 1] + (mine ? run_s[tid].block * p.scale_block[c & 1] : 0) + (c >> 1);
    const float was = mine && offset != 0 ? *ps : 0.0f;
    if (c + 1 < last) {
      fetch(c + 1, turn ^ 1);
      cp_async_wait<1>();
    } else {
      cp_async_wait<0>();
    }
    // maxima have no order
    auto count = [&](uint32_t m, int run) {                  // of a row, by its lanes; all lanes of the warp
#pragma unroll
      for (int o = kLanes / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
      if (tid % kLanes == 0 && run >= 0) atomicMax(&amax_s[turn][run], m);
    };
    uint32_t top = 0;
#pragma unroll
    for (int k = 0; k < kHold; ++k) {
      uint4 raw[kVec];
      fetched(turn, k, raw);
      const uint32_t m = lead_of[k] >= 0 ? measure(raw) : 0;
      if (only >= 0) top = max(top, m);
      else count(m, lead_of[k]);
    }
    if (only >= 0) {
      top = __reduce_max_sync(0xffffffffu, top);
      if (lane == 0) atomicMax(&amax_s[turn][only], top);
    }
    for (int i0 = shift + W; i0 < end; i0 += kRows) {
      const int i = i0 + row0, run = i < end ? lead_s[i] : -1;
      uint4 raw[kVec];
      uint32_t m = 0;
      if (run >= 0) {
        values(c, i, raw);
        m = measure(raw);
      }
      count(m, run);
    }
    __syncthreads();
    // scale of every run, and the runs whose block holds codes of a smaller one
    if (mine) {
      float now = kv8_scale(amax_s[turn][tid]);
      amax_s[turn][tid] = 0;
      if (offset == 0) {
        *ps = now;
      } else if (was >= now) {
        now = was;
      } else {
        grown_s[atomicAdd(&n_grown[turn], 1)] = tid;
        was_s[tid] = was;
        *ps = now;
      }
      run_s[tid].scale = now;
      // the reciprocal of a power of two is exact; a scale that something else wrote is divided by
      run_s[tid].inv = (__float_as_uint(now) & 0x7FFFFFu) == 0 && now <= 0x1p126f && now >= 0x1p-126f ? 1.0f / now : 0.0f;
    }
    __syncthreads();
    const int grown = n_grown[turn];
    for (int gi = 0; gi < grown; ++gi) {
      const Run run = run_s[grown_s[gi]];
      const float old = was_s[grown_s[gi]];
      uint4* pc = reinterpret_cast<uint4*>(p.cache[c & 1] + run.block * p.block[c & 1] + (int64_t)((c >> 1) << p.log_block) * D);
      for (int x = tid; x < (run.at + grown_s[gi]) * (D / 16); x += kWriteThreads) {
        uint4 v = pc[x];
        uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          uint32_t lo, hi;
          half4_of_e4m3x4(w[k], lo, hi);
          const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo));
          const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
          w[k] = e4m3x4(__fdiv_rn(a.x * old, run.scale), __fdiv_rn(a.y * old, run.scale), __fdiv_rn(b.x * old, run.scale),
                        __fdiv_rn(b.y * old, run.scale));
        }
        pc[x] = v;
      }
    }
    for (int i = shift + W + row0; i < end; i += kRows) {
      uint4 raw[kVec];
      if (lead_s[i] >= 0) {
        values(c, i, raw);
        store(c, i, run_s[lead_s[i]], raw);
      }
    }
    if (only >= 0) {
      const Run run = run_s[only];
#pragma unroll
      for (int k = 0; k < kHold; ++k) {
        uint4 raw[kVec];
        fetched(turn, k, raw);
        if (lead_of[k] >= 0) store(c, shift + row0 + k * kRows, run, raw);
      }
    } else {
#pragma unroll
      for (int k = 0; k < kHold; ++k) {
        uint4 raw[kVec];
        fetched(turn, k, raw);
        if (lead_of[k] >= 0) store(c, shift + row0 + k * kRows, run_s[lead_of[k]], raw);
      }
    }
    if (c + 1 < last) {
      if (tid == 0) n_grown[turn ^ 1] = 0;                   // read last two barriers ago
      __syncthreads();                                       // run_s may be written again
    }
  }
}

template <typename T, int D, int W, bool kSmall>
int launch_window(WriteParams p, int per, cudaStream_t st) {
  constexpr int kBytes = 2 * W * D * (int)sizeof(T);
  const auto kern = kv8_write_kernel<T, D, W, kSmall>;
  if (int rc = allow_smem("nvfp4_kv8_write", reinterpret_cast<const void*>(kern), kBytes)) return rc;
  p.per = per;
  return launch("nvfp4_kv8_write", kern, dim3((unsigned)((p.tokens + W - 1) / W), (unsigned)((p.operands + per - 1) / per)),
                kWriteThreads, kBytes, st, p);
}
// Windows of 64 tokens (128 of the largest blocks), or of 16 where those would not give two blocks an SM.
template <typename T, int D>
int launch_write(WriteParams p, int64_t hk, cudaStream_t st) {
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  p.operands = (int)(2 * hk);
  const int64_t wide = (p.tokens + 63) / 64 * p.operands;
  if (wide < 2 * sms) return launch_window<T, D, 16, true>(p, 1, st);
  const int per = wide >= 2 * 8 * sms ? 2 : 1;               // 17000 tokens of Hk 8 D 128: one 37.7, two 34.8, four 39.8 us
  if constexpr (D * sizeof(T) <= 512)
    if (p.log_block == 7) return launch_window<T, D, 128, false>(p, per, st);
  return launch_window<T, D, 64, false>(p, per, st);
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
  NVFP4_REQUIRE(slots >= 0 && slots < (1ll << 30), "nvfp4_paged_reserve: slot count out of range");
  const TableParams p{new_lens, lengths, table, table_row, const_cast<int32_t*>(free_blocks), free_count, (int)requests, (int)width,
                      (int)blocks, lb, slots, slot_map, positions, cu_seqlens, shortage, workspace};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool alone = slots <= kAlone;
  const int rc = launch("nvfp4_paged_reserve", reserve_kernel, dim3(1), table_threads(alone ? slots : 0, requests), 0, st, p, alone ? 1 : 0);
  if (rc != 0 || alone) return rc;
  const int64_t grid = (slots + 1023) / 1024;
  return launch("nvfp4_paged_reserve", reserve_fill_kernel, dim3((unsigned)(grid < 592 ? grid : 592)), 256, 0, st, p);
}

extern "C" int nvfp4_paged_trim(const int32_t* keep_lens, int32_t* lengths, int32_t* table, int64_t table_row,
                                int32_t* free_blocks, int32_t* free_count, int64_t requests, int64_t width, int64_t blocks,
                                int block_size, int32_t* workspace, nvfp4_stream_t stream) {
  const int lb = log2_block(block_size);
  NVFP4_REQUIRE(lb >= 0, "nvfp4_paged_trim: block_size must be 16, 32, 64 or 128");
  NVFP4_REQUIRE(requests >= 1 && requests < (1 << 30) && width >= 1 && width < (1 << 30) && blocks >= 0 && blocks < INT32_MAX,
                "nvfp4_paged_trim: sizes out of range");
  NVFP4_REQUIRE(requests * width < INT32_MAX, "nvfp4_paged_trim: the table has too many entries");
  const TableParams p{keep_lens, lengths, table, table_row, free_blocks, free_count, (int)requests, (int)width, (int)blocks, lb, 0,
                      nullptr, nullptr, nullptr, nullptr, workspace};
  // one block of threads, or a cluster of eight for wide tables; of a table's entries a call gives few back, mostly
  const int64_t entries = requests * width / 4;
  const unsigned cluster = entries > kAlone ? 8 : 1;
  return launch_cluster("nvfp4_paged_trim", trim_kernel, dim3(1, 1, cluster), cluster, table_threads(entries, requests), 0,
                        static_cast<cudaStream_t>(stream), p);
}

extern "C" int nvfp4_kv8_write(const void* key, const void* value, int dtype, int64_t tokens, int64_t hk, int d, int64_t skt,
                               int64_t skh, int64_t svt, int64_t svh, const int64_t* slot_map, uint8_t* k_cache,
                               int64_t k_block, uint8_t* v_cache, int64_t v_block, float* k_scale, int64_t ks_block,
                               float* v_scale, int64_t vs_block, int64_t blocks, int block_size, nvfp4_stream_t stream) {
  const int lb = log2_block(block_size);
  NVFP4_REQUIRE(lb >= 0, "nvfp4_kv8_write: block_size must be 16, 32, 64 or 128");
  NVFP4_REQUIRE(d == 128 || d == 256, "nvfp4_kv8_write: D must be 128 or 256");
  NVFP4_REQUIRE(tokens >= 0 && tokens < (1ll << 31) && hk >= 1 && hk <= 32767 && blocks >= 0, "nvfp4_kv8_write: sizes out of range");
  const int64_t size = dtype == NVFP4_DT_FP32 ? 4 : 2;
  NVFP4_REQUIRE((((uintptr_t)key | (uintptr_t)value) & 15) == 0 && ((skt | skh | svt | svh) * size & 15) == 0,
                "nvfp4_kv8_write: rows of keys and values must be 16-byte aligned");
  NVFP4_REQUIRE((((uintptr_t)k_cache | (uintptr_t)v_cache) & 15) == 0 && ((k_block | v_block) & 15) == 0,
                "nvfp4_kv8_write: cache blocks must be 16-byte aligned");
  if (tokens == 0) return 0;
  const WriteParams p{{key, value}, {skt, svt}, {skh, svh}, {k_cache, v_cache}, {k_block, v_block}, {k_scale, v_scale},
                      {ks_block, vs_block}, slot_map, tokens, blocks << lb, lb, 0, 0};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case NVFP4_DT_BF16: return d == 128 ? launch_write<__nv_bfloat16, 128>(p, hk, st) : launch_write<__nv_bfloat16, 256>(p, hk, st);
    case NVFP4_DT_FP16: return d == 128 ? launch_write<__half, 128>(p, hk, st) : launch_write<__half, 256>(p, hk, st);
    case NVFP4_DT_FP32: return d == 128 ? launch_write<float, 128>(p, hk, st) : launch_write<float, 256>(p, hk, st);
  }
  return fail(-1, "nvfp4_kv8_write: unknown dtype %d", dtype);
}
