// Paged 8-bit KV cache: the tokens of an accepted path moved together, in all layers at once.
//
// Path a_0 < a_1 < ... of a request's n newest tokens, which lie at positions len - n ..: token a_j goes to position len - n + j.
// Once a_j is not j it is above j from there on, so what moves is the path's tail, to places in front of where it lies, and a
// block that receives tokens receives all behind its first one.  Within blocks of equal scales codes are copied; else a code is
// the one rounding of the value it stood for to the receiving block's scale, which becomes the smallest power of two that holds
// what came from blocks of larger scales where that is more than it was, and older codes are rounded again to it.  Codes behind the
// path stay, and are no tokens any more: their block's scale may have grown.
//
// A warp has a head's keys or values of a layer (a unit) after the other, a block of threads those of one request, which share
// what the tables say of the tokens that move to a block.  What bounds it: trips to memory one behind the other (count, path,
// table, codes with their scales); a call moves a few tokens of a request.  Paths of 64 requests in 16 layers of Hk 8 D 128, blocks of
// 16: 9.5 us, one more with the scales in a trip of their own; units of a request on the blocks that are resident at once, several a
// warp, 15 to 18.
#include <float.h>
#include <limits.h>
#include "common/abi.cuh"
#include "common/fp4.cuh"
#include "common/kv8.cuh"
#include "common/launch.cuh"

namespace nvfp4 {
namespace {

constexpr int kWarps = 8, kThreads = 32 * kWarps;
constexpr int kMaxBlock = 128;
// Blocks of an SM, with 48 registers a thread, out of which 96 bytes are spilled: four loads ahead, at 80
// registers and three blocks, took 11.6 us instead of 9.5.
constexpr int kResident = 5;

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

// x s / now, of which `about` is an approximation to 2^-22, as a float that is rounded to the code that the quotient itself would be:
// on the right side of the border between codes that it lies at.  Borders have five significant bits at most, so both sides of the
// comparison are exact in 64 bits.
__device__ __forceinline__ float beside(float about, float x, float s, float now) {
  const uint32_t u = __float_as_uint(about) & 0x7FFFFFFFu, border = (u + 0x40000u) & 0x7FF80000u;
  const double d = fabs((double)x * (double)s) - (double)__uint_as_float(border) * fabs((double)now);
  const uint32_t v = d > 0.0 ? max(u, border + 1) : d < 0.0 ? min(u, border - 1) : d == 0.0 ? border : u;
  return copysignf(__uint_as_float(v), about);
}
// Codes of scale s as codes of scale `now`, each the one rounding of its value.  Between powers of two a code times their quotient
// is exact; other scales take a call of their own, which hardly any makes: in place it costs 40 registers.
__device__ __noinline__ uint4 codes_divided(uint4 v, float s, float now) {
  float f = __fdiv_rn(s, now);
  if (f > FLT_MAX) f = FLT_MAX;                            // 0 stays 0
  uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    uint32_t lo, hi;
    half4_of_e4m3x4(w[k], lo, hi);
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo)), b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
    w[k] = e4m3x4(beside(a.x * f, a.x, s, now), beside(a.y * f, a.y, s, now), beside(b.x * f, b.x, s, now), beside(b.y * f, b.y, s, now));
  }
  return v;
}
__device__ __forceinline__ uint4 codes_again(uint4 v, float s, float now) {
  if (now == 0.0f) return v;                               // all that came is 0
  const uint32_t a = __float_as_uint(s), b = __float_as_uint(now);
  const int e = (int)(a >> 23) - (int)(b >> 23);           // of the quotient, where both are normal powers of two
  const bool powers = ((a | b) & 0x807FFFFFu) == 0 && a != 0 && b != 0 && a < 0x7F800000u && b < 0x7F800000u && e > -126 && e < 127;
  if (!powers) return codes_divided(v, s, now);
  const float f = __uint_as_float((uint32_t)(e + 127) << 23);
  uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    uint32_t lo, hi;
    half4_of_e4m3x4(w[k], lo, hi);
    const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&lo)), y = __half22float2(*reinterpret_cast<const __half2*>(&hi));
    w[k] = e4m3x4(x.x * f, x.y * f, y.x * f, y.y * f);
  }
  return v;
}

template <int D>
__global__ void __launch_bounds__(kThreads, kResident) keep_path_kernel(KeepParams p) {
  constexpr int kLanes = D / 16, kRows = 32 / kLanes;      // lanes of a token, tokens of a warp's load
  constexpr int kAhead = 2;                                // loads of a lane under way together
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
  const int32_t* const row = p.table + r * p.table_row;
  auto block_at = [&](int64_t pos) -> int {
    const int64_t e = pos >> p.log_block;
    const int b = e < p.width ? row[e] : -1;
    return (unsigned)b < (unsigned)p.blocks ? b : -1;
  };
  const int sub = lane / kLanes, piece = lane % kLanes * 16;           // this lane's token of a load, its bytes
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
    if (into < 0) continue;
    // keys or values of one head of a layer
    struct Unit {
      uint8_t* codes;
      float* scales;
      int64_t block, scale_block;
    };
    auto unit_of = [&](int u) -> Unit {
      const int head = u % p.hk, operand = u / p.hk & 1, layer = u / (2 * p.hk);
      return {p.cache[operand] + layer * p.layer[operand] + ((int64_t)head << p.log_block) * D,
              p.scale[operand] + layer * p.scale_layer[operand] + head, p.block[operand], p.scale_block[operand]};
    };
    auto scale_of = [&](const Unit& x, int i) { return x.scales[(from_s[i] >> p.log_block) * x.scale_block]; };
    auto source = [&](const Unit& x, int i) {
      return reinterpret_cast<const uint4*>(x.codes + (from_s[i] >> p.log_block) * x.block + (from_s[i] & mask) * D + piece);
    };
    auto magnitude = [](const uint4& v, float s) -> uint32_t {           // the largest, as float bits
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
      uint32_t top = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        uint32_t lo, hi;
        half4_of_e4m3x4(w[k], lo, hi);
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo)), b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
        top = max(max(top, max(kv8_magnitude(a.x * s), kv8_magnitude(a.y * s))), max(kv8_magnitude(b.x * s), kv8_magnitude(b.y * s)));
      }
      return top;
    };
    // the block's scale once the largest value that comes from larger scales is known; older codes follow it
    auto grow = [&](const Unit& x, float was, uint32_t top) -> float {
      top = __reduce_max_sync(0xffffffffu, top);
      const float now = top != 0 ? fmaxf(was, kv8_scale(top)) : was;
      if (now != was) {
        uint4* old = reinterpret_cast<uint4*>(x.codes + into * x.block);
        for (int i = lane; i < offset * kLanes; i += 32) {
          const uint4 v = old[i];
          old[i] = codes_again(v, was, now);
        }
        if (lane == 0) x.scales[into * x.scale_block] = now;
      }
      return now;
    };
    for (int u = blockIdx.y * kWarps + warp; u < p.units; u += gridDim.y * kWarps) {
      const Unit x = unit_of(u);
      // Rounds of tokens, each read before any of it is written; those of later rounds lie behind what is written.  The first
      // one's codes come with the scales, whatever those turn out to be.
      uint4 v[kAhead];
      float s[kAhead];
      auto read = [&](int i0) {
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
          const int i = i0 + sub + a * kRows;
          s[a] = 0.0f;
          if (i < count && from_s[i] >= 0) {
            v[a] = *source(x, i);
            s[a] = scale_of(x, i);
          }
        }
      };
      const float was = x.scales[into * x.scale_block];
      read(0);
      bool larger = false;
#pragma unroll
      for (int a = 0; a < kAhead; ++a) larger |= s[a] > was;
      for (int i = kAhead * kRows + lane; i < count; i += 32) larger |= from_s[i] >= 0 && scale_of(x, i) > was;
      float now = was;
      if (__any_sync(0xffffffffu, larger)) {
        uint32_t top = 0;
#pragma unroll
        for (int a = 0; a < kAhead; ++a)
          if (s[a] > was) top = max(top, magnitude(v[a], s[a]));
        for (int i = kAhead * kRows + sub; i < count; i += kRows) {
          if (from_s[i] < 0) continue;
          const float t = scale_of(x, i);
          if (t > was) top = max(top, magnitude(*source(x, i), t));
        }
        now = grow(x, was, top);
      }
      for (int i0 = 0;;) {
        __syncwarp();
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
          const int i = i0 + sub + a * kRows;
          if (i >= count || from_s[i] < 0) continue;
          // the block that receives has its new scale by now, but its own tokens were of the one before
          const float t = (from_s[i] >> p.log_block) == into ? was : s[a];
          if (t != now) v[a] = codes_again(v[a], t, now);
          *reinterpret_cast<uint4*>(x.codes + into * x.block + (offset + i) * D + piece) = v[a];
        }
        if ((i0 += kAhead * kRows) >= count) break;
        __syncwarp();
        read(i0);
      }
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
  NVFP4_REQUIRE(hk <= (1 << 20) && layers <= (1 << 28) / (2 * hk), "nvfp4_paged_keep_path: too many layers and heads");
  NVFP4_REQUIRE((((uintptr_t)k_cache | (uintptr_t)v_cache) & 15) == 0 && ((k_block | v_block | k_layer | v_layer) & 15) == 0,
                "nvfp4_paged_keep_path: cache blocks must be 16-byte aligned");
  const int units = (int)(layers * 2 * hk);
  const int64_t want = ((int64_t)units + kWarps - 1) / kWarps, y = want < 65535 ? want : 65535;
  const KeepParams p{accepted, num_accepted, cu_seqlens, lengths, table, table_row, tokens, (int)requests, (int)width, (int)blocks, lb,
                     (int)hk, units, {k_cache, v_cache}, {k_block, v_block}, {k_layer, v_layer}, {k_scale, v_scale},
                     {ks_block, vs_block}, {ks_layer, vs_layer}, keep_lens};
  const dim3 grid((unsigned)requests, (unsigned)(y > 1 ? y : 1));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return d == 128 ? launch("nvfp4_paged_keep_path", keep_path_kernel<128>, grid, kThreads, 0, st, p)
                  : launch("nvfp4_paged_keep_path", keep_path_kernel<256>, grid, kThreads, 0, st, p);
}
