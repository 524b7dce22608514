// Paged 8-bit KV cache: the tokens of an accepted path moved together, in all layers at once.
//
// Path a_0 < a_1 < ... of a request's n newest tokens, which lie at positions len - n ..: token a_j goes to position len - n + j.
// Once a_j is not j it is above j from there on, so what moves is the path's tail, to places in front of where it lies, and a
// block that receives tokens receives all behind its first one.  Within blocks of equal scales codes are copied; else a code is
// the one rounding of the value it stood for to the receiving block's scale, which becomes the smallest power of two that holds
// what came from blocks of larger scales where that is more than it was, and older codes are rounded again to it.
//
// A warp has one head's keys or values of a layer, a block of threads eight such of one request, which share what the tables say of
// the tokens that move to a block.  What bounds it: trips to memory one behind the other (count, path, tables, scales, codes); a
// call moves a few tokens of a request.
#include <limits.h>
#include "common/abi.cuh"
#include "common/fp4.cuh"
#include "common/kv8.cuh"
#include "common/launch.cuh"

namespace nvfp4 {
namespace {

constexpr int kWarps = 8, kThreads = 32 * kWarps;
constexpr int kMaxBlock = 128;

struct KeepParams {
  const int32_t *accepted, *count, *cu, *lengths, *table;
  int64_t table_row, tokens;
  int requests, width, blocks, log_block, hk, units;       // units: layers * 2 * hk
  uint8_t* cache[2];
  int64_t block[2], layer[2];                  // bytes
  float* scale[2];
  int64_t scale_block[2], scale_layer[2];
  int32_t* keep;
};

template <int D>
__global__ void __launch_bounds__(kThreads) keep_path_kernel(KeepParams p) {
  constexpr int kLanes = D / 16, kRows = 32 / kLanes;      // lanes of a token, tokens of a warp's load
  constexpr int kAhead = 4;                                // loads of a lane under way together
  __shared__ int first_s, end_s;                           // the path's tail that moves: [first_s, end_s)
  __shared__ int64_t from_s[kMaxBlock];                    // of a receiving block's tokens: block * block size + offset, or -1
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, r = blockIdx.x;
  griddep_wait();
  griddep_launch();
  const int64_t t0 = min(max((int64_t)p.cu[r], (int64_t)0), p.tokens);
  const int n = (int)max(min((int64_t)p.cu[r + 1], p.tokens) - t0, (int64_t)0);
  const int len = max(p.lengths[r], 0), m = min(max(p.count[r], 0), n), base = len - n;
  if (tid == 0) {
    first_s = m;
    end_s = m;
  }
  __syncthreads();
  // the path ends in front of an entry that does not ascend or is no token; its tail begins where a_j > j
  for (int j = tid; j < m; j += kThreads) {
    const int a = p.accepted[t0 + j], before = j > 0 ? p.accepted[t0 + j - 1] : -1;
    if (a <= before || a >= n) atomicMin(&end_s, j);
    else if (a != j) atomicMin(&first_s, j);
  }
  __syncthreads();
  const int first = first_s, end = end_s;
  if (tid == 0 && blockIdx.y == 0) p.keep[r] = max(base + end, 0);
  if (first >= end || base < 0) return;
  const int bs = 1 << p.log_block, mask = bs - 1;
  const int unit = blockIdx.y * kWarps + warp;
  const int head = unit % p.hk, operand = unit / p.hk & 1, layer = unit / (2 * p.hk);
  uint8_t* const codes = unit < p.units ? p.cache[operand] + layer * p.layer[operand] + ((int64_t)head << p.log_block) * D : nullptr;
  float* const scales = unit < p.units ? p.scale[operand] + layer * p.scale_layer[operand] + head : nullptr;
  const int32_t* const row = p.table + r * p.table_row;
  auto block_at = [&](int64_t pos) -> int {
    const int64_t e = pos >> p.log_block;
    const int b = e < p.width ? row[e] : -1;
    return (unsigned)b < (unsigned)p.blocks ? b : -1;
  };
  for (int j0 = first; j0 < end;) {
    const int to = base + j0, offset = to & mask, count = min(end - j0, bs - offset);      // tokens j0 .. of one block
    __syncthreads();
    for (int i = tid; i < count; i += kThreads) {
      const int64_t pos = (int64_t)base + p.accepted[t0 + j0 + i];
      const int b = block_at(pos);
      from_s[i] = b < 0 ? -1 : ((int64_t)b << p.log_block) + (pos & mask);
    }
    const int into = block_at(to);
    __syncthreads();
    j0 += count;
    if (into < 0 || codes == nullptr) continue;
    uint8_t* const dst = codes + into * p.block[operand];
    const float was = scales[into * p.scale_block[operand]];
    auto scale_of = [&](int i) { return scales[(from_s[i] >> p.log_block) * p.scale_block[operand]]; };
    auto source = [&](int i) { return codes + (from_s[i] >> p.log_block) * p.block[operand] + (from_s[i] & mask) * D + lane % kLanes * 16; };
    bool larger = false, other = false;
    for (int i = lane; i < count; i += 32)
      if (from_s[i] >= 0) {
        const float s = scale_of(i);
        larger |= s > was;
        other |= s != was;
      }
    larger = __any_sync(0xffffffffu, larger);
    other = __any_sync(0xffffffffu, other);
    float now = was;
    if (larger) {
      uint32_t top = 0;
      for (int i = lane / kLanes; i < count; i += kRows) {
        if (from_s[i] < 0) continue;
        const float s = scale_of(i);
        if (!(s > was)) continue;
        const uint4 v = *reinterpret_cast<const uint4*>(source(i));
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          uint32_t lo, hi;
          half4_of_e4m3x4(w[k], lo, hi);
          const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo)), b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
          top = max(max(top, max(kv8_magnitude(a.x * s), kv8_magnitude(a.y * s))), max(kv8_magnitude(b.x * s), kv8_magnitude(b.y * s)));
        }
      }
      top = __reduce_max_sync(0xffffffffu, top);
      if (top != 0) now = fmaxf(was, kv8_scale(top));
    }
    auto again = [&](uint4& v, float s) {                  // codes of scale s to codes of `now`
      uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        uint32_t lo, hi;
        half4_of_e4m3x4(w[k], lo, hi);
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo)), b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
        w[k] = e4m3x4(__fdiv_rn(a.x * s, now), __fdiv_rn(a.y * s, now), __fdiv_rn(b.x * s, now), __fdiv_rn(b.y * s, now));
      }
    };
    if (now != was) {
      for (int x = lane; x < offset * kLanes; x += 32) {
        uint4 v = reinterpret_cast<const uint4*>(dst)[x];
        again(v, was);
        reinterpret_cast<uint4*>(dst)[x] = v;
      }
      if (lane == 0) scales[into * p.scale_block[operand]] = now;
    }
    // all of a round's tokens are read before any is written; those of later rounds lie behind what is written
    for (int i0 = lane / kLanes; i0 - lane / kLanes < count; i0 += kAhead * kRows) {
      uint4 v[kAhead];
#pragma unroll
      for (int a = 0; a < kAhead; ++a) {
        const int i = i0 + a * kRows;
        if (i < count && from_s[i] >= 0) v[a] = *reinterpret_cast<const uint4*>(source(i));
      }
      __syncwarp();
#pragma unroll
      for (int a = 0; a < kAhead; ++a) {
        const int i = i0 + a * kRows;
        if (i >= count || from_s[i] < 0) continue;
        if (other) {
          // a block that receives keeps its scale in `now`, but its own tokens were of the one before
          const float s = (from_s[i] >> p.log_block) == into ? was : scale_of(i);
          if (s != now) again(v[a], s);
        }
        *reinterpret_cast<uint4*>(dst + (offset + i) * D + lane % kLanes * 16) = v[a];
      }
      __syncwarp();
    }
  }
}

}  // namespace
}  // namespace nvfp4

using namespace nvfp4;

extern "C" int nvfp4_paged_keep_path(const int32_t* accepted, const int32_t* num_accepted, const int32_t* cu_seqlens, int64_t tokens,
                                     const int32_t* lengths, const int32_t* table, int64_t table_row, int64_t requests, int64_t width,
                                     uint8_t* k_cache, int64_t k_layer, int64_t k_block, uint8_t* v_cache, int64_t v_layer,
                                     int64_t v_block, float* k_scale, int64_t ks_layer, int64_t ks_block, float* v_scale,
                                     int64_t vs_layer, int64_t vs_block, int64_t layers, int64_t blocks, int64_t hk, int block_size, int d,
                                     int32_t* keep_lens, nvfp4_stream_t stream) {
  NVFP4_REQUIRE(d == 128 || d == 256, "nvfp4_paged_keep_path: D must be 128 or 256");
  int lb = 4;
  while (lb < 7 && (1 << lb) != block_size) ++lb;
  NVFP4_REQUIRE((1 << lb) == block_size, "nvfp4_paged_keep_path: block_size must be 16, 32, 64 or 128");
  NVFP4_REQUIRE(requests >= 1 && requests < (1 << 30) && width >= 1 && width < (1 << 30) && blocks >= 0 && blocks < INT32_MAX &&
                    tokens >= 0 && tokens < INT32_MAX && hk >= 1 && layers >= 0,
                "nvfp4_paged_keep_path: sizes out of range");
  const int64_t most = 65535 * kWarps;         // units of a grid
  NVFP4_REQUIRE(hk <= most && layers <= most / (2 * hk), "nvfp4_paged_keep_path: too many layers and heads");
  NVFP4_REQUIRE((((uintptr_t)k_cache | (uintptr_t)v_cache) & 15) == 0 && ((k_block | v_block | k_layer | v_layer) & 15) == 0,
                "nvfp4_paged_keep_path: cache blocks must be 16-byte aligned");
  const int units = (int)(layers * 2 * hk);
  const KeepParams p{accepted, num_accepted, cu_seqlens, lengths, table, table_row, tokens, (int)requests, (int)width, (int)blocks, lb,
                     (int)hk, units, {k_cache, v_cache}, {k_block, v_block}, {k_layer, v_layer}, {k_scale, v_scale},
                     {ks_block, vs_block}, {ks_layer, vs_layer}, keep_lens};
  const dim3 grid((unsigned)requests, (unsigned)((units + kWarps - 1) / kWarps > 0 ? (units + kWarps - 1) / kWarps : 1));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return d == 128 ? launch("nvfp4_paged_keep_path", keep_path_kernel<128>, grid, kThreads, 0, st, p)
                  : launch("nvfp4_paged_keep_path", keep_path_kernel<256>, grid, kThreads, 0, st, p);
}
