// Attention over the paged 8-bit KV cache for many query rows a request: chunks of prompts, drafts to verify.
//
// The mathematics of paged_attn.cu on the tensor cores of sm_100: S = Q K^T and O += P V as tcgen05.mma kind::f16 of halves, 128
// rows an instruction, accumulators in tensor memory.  Codes become halves on their way into shared memory; kind::f8f6f4 would
// take them as they are, but round q and the weights to three bits of mantissa.
//
// Warps: two softmax groups (a thread a row; at D = 256 one group), four converting warps (at D = 256 four an operand), one that
// issues the products, three that fetch query rows.  A job is 128 rows against 64 keys (128 at D = 256); a group goes through
// its jobs one after the other, S of job j in place j & 1 of the group's two, P over the upper half of the S it came from.
//   rows > 128 (D = 128): group g has rows 128 g .., both go through every key tile
//   rows <= 128 (D = 128): the groups take turns at the key tiles and keep results of their own, merged at the end
// Products are issued in the order PV(j), S(j + 2): S(j + 1) is there when the softmax of job j ends.
//
// Precision: scores, maxima, sums and outputs are fp32.  A bf16 row of q becomes halves times a power of two, exact unless
// below 2^-26 of its maximum.  K and V are halves relative to the largest scale of their tile where its scales are within
// 2^kNear of each other, which keeps every code exact (a scale that is no power of two is rounded to eleven bits).  In a tile
// whose scales lie further apart each block is relative to its own, and the softmax brings them together key by key, for what a row
// sees: scores by their K scales, weights by their V scales relative to the largest of them.  A weight is a half relative to a
// reference that the running maximum may have left behind by 2^kLag, times 2^kLift (2^15 at most): its rounding is 2^-11 of itself,
// and of weights below 2^-(14 + kLift) of the largest 2^-(25 + kLift) of that.
//
// What bounds it: at D = 128 the chain of a softmax warp, 2000 clocks a job: waiting for S 300, masks 160, maximum 175, the
// reference 110, exponentials 1040 (512 on the special-function unit, which two warps share).  A 2048-token chunk over 10240
// keys, Hk 8 G 4: 342 us = 900 TFLOP/s, tensor pipe 0.46, issue 0.53.  With 128 rows or fewer the converting warps, 3700
// clocks a tile: 32 requests of 36 rows and 300 to 8190 keys 112 us = 1.5 TB/s.  At D = 256 the softmax warps, one a scheduler:
// 4000 clocks a tile; seven requests of 0 to 777 tokens over 800 to 6007 keys 45.7 us.  Where all tiles hold
// scales far apart the chunk takes 1.8 times as long (two exponentials a score, one after the other), 32 requests of 36 rows
// 1.1 times.  Turns of the two groups at the exponentials changed nothing, a quarter of them as polynomials took 359 us instead of 337.
#include <cuda_fp16.h>
#include <type_traits>
#include "common/abi.cuh"
#include "common/bwd_util.cuh"
#include "common/kv8.cuh"
#include "common/launch.cuh"
#include "common/paged.cuh"
#include "common/pairs.cuh"
#include "common/sm100.cuh"

namespace nvfp4 {
namespace {

constexpr int kTile = 128;                    // keys of a tile
constexpr int kSub = 128 * 128;               // bytes of a 128-row sub-tile of 64 halves
constexpr int kLoaders = 3;                   // warps that fetch query rows
constexpr int kInfo = 8;                      // tiles whose scales are kept: more than can be under way
// P is held times 2^kLift relative to a reference that may lag behind the running maximum by 2^kLag
constexpr float kLift = 3.0f, kLag = 12.0f;
constexpr int kNear = 15;                     // codes are multiples of 2^-9, halves of 2^-24

template <int D>
struct Cfg {
  static constexpr int kGroups = D == 128 ? 2 : 1;
  static constexpr int kRows = 128 * kGroups;
  static constexpr int kStages = D == 128 ? 2 : 1;
  static constexpr int kSoft = 4 * kGroups;                // softmax warps
  // converting warpgroups: one for K and V, or (D = 256, where one took 3600 clocks a tile) one for each
  static constexpr int kConvert = D == 128 ? 1 : 2;
  static constexpr int kIssue = kSoft + 4 * kConvert;      // first warp of the last warpgroup, which issues the products
  static constexpr int kThreads = 32 * (kIssue + 4);       // whole warpgroups: registers move between them
  static constexpr int kRegsSoft = D == 128 ? 144 : 168, kRegsConvert = D == 128 ? 152 : 128, kRegsIssue = D == 128 ? 72 : 80;
  // an increase waits for registers of this launch, which has 128 a thread (65536 / 512): more than those would wait forever
  static_assert(kThreads == 512 && kSoft * kRegsSoft + 4 * kConvert * kRegsConvert + 4 * kRegsIssue <= kThreads / 32 * 128, "registers");
  static constexpr int kOperand = D / 64 * kSub;           // 128 rows of q, or a tile of keys or values
  static constexpr int kQ = 0, kK = kGroups * kOperand, kV = kK + kStages * kOperand, kTail = kV + kStages * kOperand;
  static constexpr int kN = D == 128 ? 64 : 128;           // keys of a job
  static constexpr int kJobs = kTile / kN;                 // jobs of a tile
  // Products issued from straight code or (1) from loops: an instruction per 64 halves' step at D = 128, where the straight
  // code took 359 us of the 2048-row chunk and loops 380; at D = 256 products are longer and the straight code larger than
  // the instruction cache keeps (mixed batch 77 us straight, 70 in loops).
  static constexpr int kIssueUnroll = D == 128 ? 2 : 1;
  static constexpr int kO = 256;                           // tensor memory: S of (group, place), O behind
  static __device__ __forceinline__ uint32_t s_at(int group, int place) { return (group * 2 + place) * kN; }
};

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(
          taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

__device__ __forceinline__ void store_sector(void* dst, const uint32_t (&w)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]),
               "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}

__device__ __forceinline__ float max3(float a, uint32_t b, uint32_t c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(__uint_as_float(b)), "f"(__uint_as_float(c)));
  return d;
}

// Registers of a warpgroup.  The shares are at most what the launch has (512 threads of 128).
template <int N>
__device__ __forceinline__ void more_registers() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void fewer_registers() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// What a tile's softmax has to know: factor of its scores, log2 of what its values were divided by, which 16-key groups are there
// (a bit each).  Where the scales lie apart `there` is 0, `apart` says which groups are there, and each has exponents of its own.
struct TileInfo {
  float k_factor, v_log2;
  uint32_t there, apart;
  int8_t k_exp[8], v_exp[8];
};

// exponent (floor of log2) of a scale
__device__ __forceinline__ int scale_exp(float s) { return min(max((int)(__float_as_uint(s) >> 23 & 0xFF) - 127, -112), 126); }
__device__ __forceinline__ float exp2_int(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// Shared memory behind the tiles.  All of it is dynamic, and within 195 KB: with that the SM's split leaves 60 KB of L1, whose
// lines hold what the converting warps have asked for, and with more than 195 KB 28.
template <int D, bool kTree>
struct Tail {
  using C = Cfg<D>;
  uint64_t k_full[2], k_free[2], v_full[2], v_free[2], s_full[2][2], p_full[2][2], o_full[2], o_free[2], pv_done[2], q_full, q_free;
  int64_t list[C::kThreads / 32 + 2];
  Walk<C::kRows, kTile, kTree> place;
  int64_t share;                                           // entries of a full share
  uint32_t tmem_base;
  int expired;
  TileInfo info[kInfo];
  float c[C::kRows];
  float m[C::kGroups][128];
  __device__ __forceinline__ float* l() { return c + C::kRows - 128; }       // of rows that a unit of one group's rows does not have
};
constexpr int kSmemPercent = 85;
template <int D, bool kTree>
constexpr int smem_bytes() {
  static_assert(Cfg<D>::kTail + sizeof(Tail<D, kTree>) <= 195 * 1024, "L1");
  return Cfg<D>::kTail + (int)sizeof(Tail<D, kTree>);
}

template <typename T, int D, bool kTree>
__global__ void __launch_bounds__(Cfg<D>::kThreads, 1) paged_chunk_kernel(PagedParams p) {
  using C = Cfg<D>;
  using Place = Walk<C::kRows, kTile, kTree>;
  extern __shared__ __align__(1024) uint8_t smem[];        // at 1024 without static shared memory in front of it, see below
  auto& sh = *reinterpret_cast<Tail<D, kTree>*>(smem + C::kTail);
  auto &k_full = sh.k_full, &k_free = sh.k_free, &v_full = sh.v_full, &v_free = sh.v_free, &pv_done = sh.pv_done, &o_full = sh.o_full,
       &o_free = sh.o_free;
  auto &s_full = sh.s_full, &p_full = sh.p_full;
  uint64_t &q_full = sh.q_full, &q_free = sh.q_free;
  int& expired = sh.expired;                               // a wait ran out: site, else 0
  auto& info_s = sh.info;
  auto& c_s = sh.c;
  const int tid = threadIdx.x, lane = tid & 31, warp = warp_index();
  volatile int* err = &expired;

  if (smem_u32(smem) & 1023) {                             // what the products' descriptors take for granted
    griddep_wait();
    if (tid == 0) {
      p.cut[blockIdx.x] = make_int4(0, 0, 0, 0);           // nothing to be merged
      if (p.status != nullptr) atomicExch(p.status, 72);
    }
    return;
  }
  if (tid == 0) {
    expired = 0;
    for (int i = 0; i < 2; ++i) {
      mbar_init(&k_full[i], 4);
      mbar_init(&k_free[i], 1);
      mbar_init(&v_full[i], 4);
      mbar_init(&v_free[i], 1);
      for (int k = 0; k < 2; ++k) {
        mbar_init(&s_full[i][k], 1);
        mbar_init(&p_full[i][k], 4);
      }
      mbar_init(&pv_done[i], 1);
      mbar_init(&o_full[i], 1);
      mbar_init(&o_free[i], 4);
    }
    mbar_init(&q_full, kLoaders);
    mbar_init(&q_free, C::kSoft + 1);
    mbar_fence_init();
  }
  if (warp == C::kIssue) tmem_alloc(&sh.tmem_base, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  griddep_launch();
  griddep_wait();
  const uint32_t tmem = sh.tmem_base;
  {
    Place from;
    const int64_t share = deal_tiles<C::kThreads>(p, sh.list, from);
    if (tid == 0) {
      sh.place = from;
      sh.share = share;
      p.cut[blockIdx.x] = make_int4(0, 0, 0, 0);
    }
  }
  __syncthreads();                                         // every role has its own copy from here on

  if (warp >= C::kSoft && warp < C::kIssue) {
    if (C::kRegsConvert > 128) more_registers<C::kRegsConvert>();
    Place ahead = sh.place;
    bool more = ahead.open();                              // there is a tile to be looked up: `tile` of `ahead`
    int tile = ahead.from;
    // ------------------------------------------------------------------ codes to halves
    const int w = warp & 3, t = w * 32 + lane;
    const bool does_k = C::kConvert == 1 || warp < C::kSoft + 4;
    // 16-byte pieces of a tile: eight lanes take 64 bytes of two neighbouring keys, whose halves then lie in different banks
    constexpr int kPieces = D / 16;                        // per thread and operand
    const int in_key = (lane >> 2) & 1, in_chunk = lane & 3, pair8 = w * 4 + (lane >> 3);
    auto key_of = [&](int i) { return (i / (D / 64)) * 32 + pair8 * 2 + in_key; };
    auto chunk_of = [&](int i) { return (i % (D / 64)) * 4 + in_chunk; };
    // Codes wait in registers, from the time that their tile's predecessor is converted on: asked for when all of that one's are
    // (piece by piece between the conversions the chunk took 4 us more; before there was L1 for a tile of K
    // and V it was the better way).
    uint4 kr[kPieces], vr[C::kConvert == 1 ? kPieces : 1];   // where a warp does one operand, its codes are in the first
    // lanes 0 to 7: block of keys 16 lane .. of the tile being converted (`now`), asked for (`next`), and of the one behind
    int id_now = -1, id_next = -1, id_ahead = -1;
    float ks_now = 0.0f, vs_now = 0.0f, ks_next = 0.0f, vs_next = 0.0f;
    int key0 = 0, limit = 0, head = 0;                     // of the tile asked for
    int key0_now = 0, limit_now = 0, head_now = 0;         // and of the one converted
    bool asked = false;                                    // there is one
    bool starts = true, starts_next = true, starts_ahead = true;   // first tile of its unit, as far as this CTA sees
    auto look_up = [&]() {
      id_ahead = -1;
      const int key = tile * kTile + lane * 16;
      if (more && lane < 8 && key < ahead.q.limit(p, ahead.row_tile))
        id_ahead = p.table[ahead.r * p.table_row + (key >> p.log_block)];
    };
    // the tile asked for becomes the one converted, the one looked up the one asked for
    auto next = [&]() {
      id_now = id_next;
      ks_now = ks_next;
      vs_now = vs_next;
      starts = starts_next;
      id_next = (unsigned)id_ahead < (unsigned)p.blocks ? id_ahead : -1;
      starts_next = starts_ahead;
      starts_ahead = false;
      asked = more;
      key0_now = key0;
      limit_now = limit;
      head_now = head;
      key0 = tile * kTile;
      limit = more ? ahead.q.limit(p, ahead.row_tile) : 0;
      head = ahead.head;
      if (more && ++tile == ahead.to) {
        ahead.close(p);
        more = ahead.open();
        tile = ahead.from;
        starts_ahead = true;
      }
      look_up();
      ks_next = id_next >= 0 ? p.ks[id_next * p.ks_block + head] : 0.0f;
      vs_next = id_next >= 0 ? p.vs[id_next * p.vs_block + head] : 0.0f;
    };
    // a warp's keys lie in every other 16-key group: block of its u-th one (shuffles share a queue with the stores below)
    constexpr int kOwn = 4, kEach = kPieces / kOwn;
    auto group_of = [&](int u) { return 2 * u + (w >> 1); };
    const int first_key = (pair8 & 7) * 2 + in_key;         // of a group
    // this thread's first key of each in an operand of a tile (blocks `id`, keys from `key0` to `limit` of a head): its codes, and how
    // many keys of the group are there
    auto find = [&](const uint8_t* codes, int64_t block, int id, int key0, int limit, int head, const uint8_t* (&from)[kOwn], int (&count)[kOwn]) {
#pragma unroll
      for (int u = 0; u < kOwn; ++u) {
        const int b = __shfl_sync(0xffffffffu, id, group_of(u)), key = key0 + group_of(u) * 16;
        from[u] = codes + b * block + (((int64_t)head << p.log_block) + (key & ((1 << p.log_block) - 1)) + first_key) * D + in_chunk * 16;
        count[u] = b >= 0 ? limit - key : 0;
      }
    };
    auto find_next = [&](bool k, const uint8_t* (&from)[kOwn], int (&count)[kOwn]) {       // of the tile asked for
      find(k ? p.k : p.v, k ? p.k_block : p.v_block, id_next, key0, limit, head, from, count);
    };
    const uint8_t* from[kOwn];
    int count[kOwn];
    auto ask = [&](const uint8_t* const (&from)[kOwn], const int (&count)[kOwn], int i) -> uint4 {
      return load_or_zero(from[i / kEach] + i % kEach * 64, first_key < count[i / kEach]);
    };
    // pieces to halves times `factor` (lane h: of keys 16 h ..), into a tile in shared memory; behind them the next tile's are asked for
    auto convert = [&](uint4 (&r)[kPieces], float factor, int id, uint32_t dst, const uint8_t* const (&from)[kOwn], const int (&count)[kOwn]) {
      // Factors of 1 are tested for at D = 256 alone, whose warps spill without the test (mixed batch 55 us instead of 45.7); at D = 128 they
      // have no registers to spare for it (32 requests of 36 rows 118 us instead of 112).
      const bool plain = C::kConvert == 2 && __all_sync(0xffffffffu, lane >= 8 || id < 0 || factor == 1.0f);
      __half2 own[kOwn];
#pragma unroll
      for (int u = 0; u < kOwn; ++u) own[u] = __float2half2_rn(__shfl_sync(0xffffffffu, factor, group_of(u)));
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const int key = key_of(i), chunk = chunk_of(i);
        const uint32_t words[4] = {r[i].x, r[i].y, r[i].z, r[i].w};
        uint32_t h[8];
#pragma unroll
        for (int k = 0; k < 4; ++k) half4_of_e4m3x4(words[k], h[2 * k], h[2 * k + 1]);
        if (!plain) {
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const __half2 v = __hmul2(*reinterpret_cast<const __half2*>(&h[k]), own[i / kEach]);
            h[k] = *reinterpret_cast<const uint32_t*>(&v);
          }
        }
        const uint32_t row = dst + (chunk >> 2) * kSub + key * 128;
        const int c = (chunk & 3) * 2;
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(row + ((c ^ (key & 7)) << 4)), "r"(h[0]), "r"(h[1]), "r"(h[2]),
                     "r"(h[3])
                     : "memory");
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(row + (((c + 1) ^ (key & 7)) << 4)), "r"(h[4]), "r"(h[5]),
                     "r"(h[6]), "r"(h[7])
                     : "memory");
      }
#pragma unroll
      for (int i = 0; i < kPieces; ++i) r[i] = ask(from, count, i);
      fence_proxy_async_smem();
      __syncwarp();
    };
    int v_run = -200;                                      // largest exponent of the unit's value scales so far
    // exponents of the tile converted now: what its keys and values are relative to, and (lane h) those of keys 16 h .. where apart
    int ke, ve, ke_own, ve_own;
    bool apart;
    auto factors = [&]() {
      if (starts) v_run = -200;
      ke_own = id_now >= 0 ? scale_exp(ks_now) : -112;
      ve_own = id_now >= 0 ? scale_exp(vs_now) : -112;
      ke = __reduce_max_sync(0xffffffffu, ke_own);
      ve = __reduce_max_sync(0xffffffffu, ve_own);
      v_run = max(v_run, ve);
      ve = max(ve, v_run - 60);                            // the sum of weights relative to the reference stays within fp32
      apart = __any_sync(0xffffffffu, id_now >= 0 && (ke_own < ke - kNear || ve_own < ve - kNear));
      if (!apart) {
        ke_own = ke;
        ve_own = ve;
      }
    };
    auto do_k = [&](uint32_t n) {
      const int st = n % C::kStages;
      const uint32_t there = __ballot_sync(0xffffffffu, id_now >= 0);
      mbar_wait_warp(&k_free[st], (n / C::kStages & 1) ^ 1, err, 60);
      TileInfo& info = info_s[n % kInfo];
      if (t == 0) {
        info.k_factor = exp2_int(ke);
        info.v_log2 = (float)ve;
        info.there = apart ? 0 : there;
        info.apart = apart ? there : 0;
      }
      if (apart && t < 8) {
        info.k_exp[t] = (int8_t)ke_own;
        info.v_exp[t] = (int8_t)ve_own;
      }
      convert(kr, ks_now * exp2_int(-ke_own), id_now, smem_u32(smem + C::kK + st * C::kOperand), from, count);
      if (lane == 0) mbar_arrive(&k_full[st]);
    };
    auto do_v = [&](uint32_t n, uint4 (&r)[kPieces], float factor, int id) {
      const int st = n % C::kStages;
      mbar_wait_warp(&v_free[st], (n / C::kStages & 1) ^ 1, err, 61);
      convert(r, factor, id, smem_u32(smem + C::kV + st * C::kOperand), from, count);
      if (lane == 0) mbar_arrive(&v_full[st]);
    };
    if (more) {
      look_up();
      next();
      find_next(does_k, from, count);
#pragma unroll
      for (int i = 0; i < kPieces; ++i) kr[i] = ask(from, count, i);
    }
    uint32_t n = 0;
    if constexpr (C::kConvert == 1) {
      // K of a tile in front of V of the tile before it: V waits until a product two tiles back is complete, and S of the next
      // tile must not wait with it (units of 32 rows, 32 requests: 133 us the other way round)
      if (asked) {
        find_next(false, from, count);
#pragma unroll
        for (int i = 0; i < kPieces; ++i) vr[i] = ask(from, count, i);
      }
      bool v_left = false;                                 // V of tile n - 1 is to be done
      float v_factor = 0.0f;
      int v_id = -1;
      while (asked || v_left) {
        const bool tile_there = asked;
        if (tile_there) {
          next();
          factors();
          find_next(true, from, count);
          do_k(n);
        }
        if (v_left) {                                      // behind it, the values of this tile are asked for
          find(p.v, p.v_block, tile_there ? id_now : -1, key0_now, limit_now, head_now, from, count);
          do_v(n - 1, vr, v_factor, v_id);
        }
        v_left = tile_there;
        if (tile_there) {
          v_factor = vs_now * exp2_int(-ve_own);
          v_id = id_now;
          ++n;
        }
      }
    } else {
      for (; asked; ++n) {
        next();
        factors();
        find_next(does_k, from, count);
        if (does_k) do_k(n);
        else do_v(n, kr, vs_now * exp2_int(-ve_own), id_now);
      }
    }
  } else if (warp >= C::kIssue) {
    fewer_registers<C::kRegsIssue>();
    if (warp > C::kIssue) {
    // ------------------------------------------------------------------ query rows
    // L lanes a row, eight 16-byte pieces a lane: copied as they are, all rows of a warp at once, as soon as the last S of the
    // segment before is complete (its softmax and its result are still to come), then halves in their place.  A row of bf16 is
    // scaled by the power of two that brings its largest element to [2^12, 2^13): exact, but for elements below 2^-26 of
    // that one.  fp16 rows are taken as they are.  A scaling below zero turns q.
    constexpr int L = D / 64, kPass = 32 / L, kPasses = C::kRows / kPass;
    const int piece = lane % L, sub = lane >> 3, in8 = (lane & 7) / L;
    // eight lanes in a row of them touch every bank once
    const int row_in = L == 4 ? sub + 4 * in8 : 2 * in8 + (sub & 1) + 8 * (sub >> 1);
    Place at = sh.place;
    uint32_t seg = 0;
    for (; at.open(); at.close(p), ++seg) {
      const int rows = at.q.rows(p, at.row_tile), passes = rows > 128 ? kPasses : 128 / kPass;
      mbar_wait_warp(&q_free, (seg & 1) ^ 1, err, 70);
      auto place_of = [&](int row, int j) {                // of piece L j + piece
        const int c = L * j + piece;
        return smem_u32(smem + C::kQ) + (row >> 7) * C::kOperand + (c >> 3) * kSub + (row & 127) * 128 + (((c & 7) ^ (row & 7)) << 4);
      };
#pragma unroll 1
      for (int x = warp - C::kIssue - 1; x < passes; x += kLoaders) {
        const int row = x * kPass + row_in;
        const T* src = query_row<T>(p, at.q.t0, at.row_tile * C::kRows + min(row, rows - 1), at.head) + piece * 8;
        const uint32_t bytes = row < rows ? 16 : 0;
#pragma unroll
        for (int j = 0; j < 8; ++j)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(place_of(row, j)), "l"(src + j * L * 8), "r"(bytes) : "memory");
      }
      cp_async_commit();
      cp_async_wait<0>();
      const bool as_is = std::is_same<T, __half>::value && p.scale_log2 >= 0.0f;
#pragma unroll 1
      for (int x = warp - C::kIssue - 1; x < passes; x += kLoaders) {
        const int row = x * kPass + row_in;
        if (as_is) {
          if (piece == 0) c_s[row] = p.scale_log2;
          continue;
        }
        uint4 raw[8];
#pragma unroll
        for (int j = 0; j < 8; ++j)
          asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(raw[j].x), "=r"(raw[j].y), "=r"(raw[j].z), "=r"(raw[j].w)
                       : "r"(place_of(row, j)) : "memory");
        float up = -1.0f, c = fabsf(p.scale_log2);
        if constexpr (!std::is_same<T, __half>::value) {
          auto two = [](uint32_t w) { return *reinterpret_cast<const __nv_bfloat162*>(&w); };
          __nv_bfloat162 top = two(0u);
#pragma unroll
          for (int j = 0; j < 8; ++j)
            top = __hmax2(top, __hmax2(__hmax2(__habs2(two(raw[j].x)), __habs2(two(raw[j].y))),
                                       __hmax2(__habs2(two(raw[j].z)), __habs2(two(raw[j].w)))));
#pragma unroll
          for (int o = L / 2; o > 0; o >>= 1) {
            const uint32_t other = __shfl_xor_sync(0xffffffffu, *reinterpret_cast<const uint32_t*>(&top), o);
            top = __hmax2(top, two(other));
          }
          const float big = fmaxf(__low2float(top), __high2float(top));
          const int ex = min(max((int)(__float_as_uint(big) >> 23) - 127, -110), 127);
          up = copysignf(exp2_int(12 - ex), p.scale_log2);
          c = big == 0.0f ? 0.0f : c * exp2_int(ex - 12);
        }
        if (piece == 0) c_s[row] = c;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t words[4] = {raw[j].x, raw[j].y, raw[j].z, raw[j].w};
          uint32_t h[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            using T2 = typename std::conditional<std::is_same<T, __nv_bfloat16>::value, __nv_bfloat162, __half2>::type;
            const T2 t = *reinterpret_cast<const T2*>(&words[k]);
            h[k] = pack_16x2<__half>(to_f32<T>(t.x) * up, to_f32<T>(t.y) * up);
          }
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(place_of(row, j)), "r"(h[0]), "r"(h[1]), "r"(h[2]), "r"(h[3]) : "memory");
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_full);
    }
    } else {
    // ------------------------------------------------------------------ issue of the products
    Place at = sh.place;
    const bool leader = elect_one();
    const uint32_t id_s = make_idesc_bf16(128, C::kN, false, true), id_o = make_idesc_bf16(128, 128, true, true);
    const uint64_t b_q = desc_sw128(smem + C::kQ, 0), b_k = desc_sw128(smem + C::kK, 0);
    const uint64_t b_v = desc_sw128_mn(smem + C::kV, 0, kSub);
    uint32_t n = 0, seg = 0;                               // tiles and segments so far
    uint32_t p_phase = 0;                                  // of p_full, a bit a group and place
    uint32_t used = 0, o_phase = 0;                        // groups that have had a result, and how many, a bit a group
    for (; at.open(); at.close(p)) {
      const int tiles = at.to - at.from;
      const bool both = C::kGroups == 2 && at.q.rows(p, at.row_tile) > 128;
      const int turn = both || C::kGroups == 1 ? 1 : 2;    // a group takes every turn-th tile
      auto jobs_of = [&](int g) { return (turn == 1 ? tiles : (tiles + 1 - g) / 2) * C::kJobs; };
      auto tile_of = [&](int g, int j) { return j / C::kJobs * turn + (turn == 2 ? g : 0); };
      mbar_wait_warp(&q_full, seg & 1, err, 62);
      int s_left = jobs_of(0) + (C::kGroups == 2 ? jobs_of(1) : 0);
      auto issue_s = [&](int g, int j) {
        const bool last = --s_left == 0;
        const uint32_t tile = n + tile_of(g, j), st = tile % C::kStages;
        const int sub = j % C::kJobs;
        if (sub == 0 && (!both || g == 0)) mbar_wait(&k_full[st], (tile / C::kStages) & 1, err, 63);
        __syncwarp();
        tc_fence_after();
        if (leader) {
          const uint64_t x_q = b_q + (both && g ? C::kOperand >> 4 : 0);
          const uint64_t x_k = b_k + (uint64_t)(st * (C::kOperand >> 4) + sub * (C::kN * 128 >> 4));
#pragma unroll C::kIssueUnroll
          for (int c = 0; c < D / 64; ++c)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              umma_bf16(tmem + C::s_at(g, j & 1), x_q + c * (kSub >> 4) + k * 2, x_k + c * (kSub >> 4) + k * 2, id_s, (c > 0 || k > 0) ? 1u : 0u);
          umma_commit(&s_full[g][j & 1]);
          if (sub == C::kJobs - 1 && (!both || g == 1)) umma_commit(&k_free[st]);
          if (last) umma_commit(&q_free);
        }
        __syncwarp();
      };
      auto issue_pv = [&](int g, int j) {
        const uint32_t tile = n + tile_of(g, j), st = tile % C::kStages;
        const int sub = j % C::kJobs;
        if (j == 0 && (used >> g & 1)) mbar_wait(&o_free[g], (o_phase >> g & 1) ^ 1, err, 64);
        if (sub == 0 && (!both || g == 0)) mbar_wait(&v_full[st], (tile / C::kStages) & 1, err, 65);
        mbar_wait_warp(&p_full[g][j & 1], p_phase >> (2 * g + (j & 1)) & 1, err, 66);
        p_phase ^= 1u << (2 * g + (j & 1));
        tc_fence_after();
        if (leader) {
          const uint64_t x_v = b_v + (uint64_t)(st * (C::kOperand >> 4) + sub * (C::kN * 128 >> 4));
          const uint32_t x_p = tmem + C::s_at(g, j & 1) + C::kN / 2;
#pragma unroll C::kIssueUnroll
          for (int c = 0; c < D / 128; ++c)
#pragma unroll
            for (int k = 0; k < C::kN / 16; ++k)
              umma_bf16_ta(tmem + C::kO + g * 128 + c * 128, x_p + k * 8, x_v + c * (2 * kSub >> 4) + k * 128, id_o,
                           (k > 0 || j > 0) ? 1u : 0u);
          if (sub == C::kJobs - 1 && (!both || g == 1)) umma_commit(&v_free[st]);
          umma_commit(&pv_done[g]);
          if (j + 1 == jobs_of(g)) umma_commit(&o_full[g]);
        }
        __syncwarp();
        if (j == 0) {
          used |= 1u << g;
          o_phase ^= 1u << g;
        }
      };
      // Where the groups take turns, S of a tile must not stand in front of PV of the tile four before: its K is converted behind
      // V of the tile two before it, which waits for that place.  So there group 1 is a job behind group 0, and a step has both
      // groups' PV first.  With more than 128 rows both groups are at the same tile, and that PV is some steps old.
      const bool turns = C::kGroups == 2 && !both;
      const int steps = jobs_of(0) + (turns ? 1 : 0);
#pragma unroll 1
      for (int j = -2; j < steps; ++j) {                   // PV of job j behind S of job j + 1, S of job j + 2 behind that
        if (turns) {
#pragma unroll 1
          for (int x = 0; x < 4; ++x) {
            const int g = x & 1, at_j = j - g;
            if (x < 2 && at_j >= 0 && at_j < jobs_of(g)) issue_pv(g, at_j);
            if (x >= 2 && at_j >= -2 && at_j + 2 < jobs_of(g)) issue_s(g, at_j + 2);
          }
        } else {
#pragma unroll C::kIssueUnroll
          for (int g = 0; g < C::kGroups; ++g) {
            if (j >= 0 && j < jobs_of(g)) issue_pv(g, j);
            if (j + 2 < jobs_of(g)) issue_s(g, j + 2);
          }
        }
      }
      n += tiles;
      ++seg;
    }
    }
  } else {
    more_registers<C::kRegsSoft>();
    Place at = sh.place;
    // ------------------------------------------------------------------ softmax, a thread a row
    const int group = warp >> 2, wq = warp & 3, row_in = wq * 32 + lane;
    const uint32_t lane_addr = (uint32_t)(wq * 32) << 16;
    uint32_t n = 0;                                        // tiles so far
    uint32_t seg = 0;                                      // segments so far
    uint32_t s_phase = 0, results = 0, pv = 0;             // phases of s_full (a bit a place), o_full and pv_done so far
    bool first_segment = true;
    for (; at.open(); at.close(p)) {
      const int tiles = at.to - at.from;
      const int rows = at.q.rows(p, at.row_tile);
      const bool both = C::kGroups == 2 && rows > 128;
      const bool whole = at.whole();
      const int row = (both ? group * 128 : 0) + row_in;   // of the unit
      const bool live = row < rows;
      const int i_row = at.row_tile * C::kRows + row;      // of the request
      mbar_wait(&q_full, seg & 1, err, 71);
      ++seg;
      const float c_row = c_s[both ? row : row_in];
      // where both groups work on the same rows, they exchange results where q is
      const bool merge = C::kGroups == 2 && !both;
      __syncwarp();
      if (!merge && lane == 0) mbar_arrive(&q_free);
      const int limit = live || kTree ? at.q.seen(p, i_row) : 0;      // keys that this row sees, or (of a tree) that all rows see
      // the bits of a tree's row; rows of no query have those of the last one
      const uint32_t* const bits = kTree ? tree_row(p, at.q.t0 + token_of(p, min(i_row, at.row_tile * C::kRows + rows - 1))) : nullptr;
      float m = -INFINITY, ref = -INFINITY, l = 0.0f;

      const int turn = both || C::kGroups == 1 ? 1 : 2, my = turn == 2 ? group : 0;
      const int jobs = (turn == 1 ? tiles : (tiles + 1 - my) / 2) * C::kJobs;
#pragma unroll 1
      for (int j = 0; j < jobs; ++j) {
        constexpr int kChunks = C::kN / 32;
        const int place = j & 1, tile = j / C::kJobs * turn + my, sub = j % C::kJobs;
        const uint32_t s_at = tmem + lane_addr + C::s_at(group, place);
        const int key0 = (at.from + tile) * kTile + sub * C::kN;
        mbar_wait(&s_full[group][place], (s_phase >> place) & 1, err, 67);
        s_phase ^= 1u << place;
        tc_fence_after();
        __syncwarp();
        const TileInfo& info = info_s[(n + tile) % kInfo];
        const float k_factor = info.k_factor, v_log2 = info.v_log2;
        const uint32_t there = info.there >> (sub * (C::kN / 16));
        const bool masked = __any_sync(0xffffffffu, live && limit < key0 + C::kN) ||
                            (there & ((1u << (C::kN / 16)) - 1)) != (1u << (C::kN / 16)) - 1;
        const int visible = limit - key0;
        // columns x .. x + 31 of a tree's row, as far as there are keys
        auto tree_columns = [&](int x) -> uint32_t {
          const int left = at.q.len - key0 - x;
          return left <= 0 ? 0u : tree_bits(p, bits, x - visible) & (left >= 32 ? 0xFFFFFFFFu : (1u << left) - 1);
        };
        // columns 32 x .. of S: the next ones are on their way while the present ones are used, and the last two stay for
        // the exponentials, which therefore run from the end
        float top = -INFINITY;
        uint32_t s[2][32];
        if (masked) {                                      // a few tiles of a unit: S is edited where it is
          if (const uint32_t groups = info.apart; groups != 0) {
            // Scales far apart: scores in units of log2 with each group's K scale, the reference of the weights from scores with their
            // V scales, then two exponentials a score, for the sum and (times the V scale) for the product.
            constexpr int kOf = C::kN / 16;                // groups of a job
            float want = -INFINITY;
#pragma unroll 1
            for (int x = 0; x < kOf; ++x) {
              uint32_t now[16];
              tmem_ld16(s_at + x * 16, now);
              tmem_ld_wait();
              const int of = sub * kOf + x, left = groups >> of & 1 ? visible - x * 16 : 0;
              const uint32_t columns = kTree && (groups >> of & 1) ? tree_columns(x * 16) : 0u;
              const float f = scale_product(c_row, exp2_int(info.k_exp[of]));
              float t = -INFINITY;
#pragma unroll
              for (int e = 0; e < 16; ++e) {
                now[e] = (kTree ? (columns >> e & 1) != 0 : e < left) ? __float_as_uint(__uint_as_float(now[e]) * f) : 0xFF800000u;
                t = fmaxf(t, __uint_as_float(now[e]));
              }
              top = fmaxf(top, t);
              want = fmaxf(want, t + (float)info.v_exp[of]);
              tmem_st16(s_at + x * 16, now);
            }
            const float m_new = fmaxf(m, top), less = m_new == -INFINITY ? 0.0f : m_new;
            if (__any_sync(0xffffffffu, want > ref + kLag)) {
              const float ref_new = fmaxf(ref, want), f = want > ref ? ex2_approx(ref - ref_new) : 1.0f;
              ref = ref_new;
              if (j > 0) {
                mbar_wait(&pv_done[group], (pv - 1) & 1, err, 68);
                tc_fence_after();
                __syncwarp();
#pragma unroll 1
                for (int cc = 0; cc < D / 16; ++cc) {
                  const uint32_t o_at = tmem + lane_addr + C::kO + group * 128 + cc * 16;
                  uint32_t o[16];
                  tmem_ld16(o_at, o);
                  tmem_ld_wait();
#pragma unroll
                  for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                  tmem_st16(o_at, o);
                }
              }
            }
            tmem_st_wait();
            l *= m_new == -INFINITY ? 1.0f : ex2_approx(m - m_new);
            m = m_new;
#pragma unroll 1
            for (int x = kOf - 1; x >= 0; --x) {           // weights over scores that have been read
              uint32_t now[16], w[8];
              tmem_ld16(s_at + x * 16, now);
              tmem_ld_wait();
              const float plus = ref == -INFINITY ? 0.0f : (float)info.v_exp[sub * kOf + x] - ref + kLift;
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                const float y0 = __uint_as_float(now[2 * e]), y1 = __uint_as_float(now[2 * e + 1]);
                l += ex2_approx(y0 - less) + ex2_approx(y1 - less);
                w[e] = pack_16x2<__half>(ex2_approx(y0 + plus), ex2_approx(y1 + plus));
              }
              tmem_st8(s_at + C::kN / 2 + x * 8, w);
            }
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_full[group][place]);
            ++pv;
            continue;
          }
#pragma unroll 1
          for (int x = 0; x < kChunks; ++x) {
            tmem_ld32(s_at + x * 32, s[0]);
            tmem_ld_wait();
            const int left = visible - x * 32;
            uint32_t seen = kTree ? tree_columns(x * 32) : left >= 32 ? 0xFFFFFFFFu : left <= 0 ? 0u : (1u << left) - 1;
            seen &= ((there >> (2 * x) & 1) ? 0xFFFFu : 0u) | ((there >> (2 * x + 1) & 1) ? 0xFFFF0000u : 0u);
#pragma unroll
            for (int e = 0; e < 32; ++e) s[0][e] = (seen >> e & 1) ? s[0][e] : 0xFF800000u;
            tmem_st32(s_at + x * 32, s[0]);
          }
          tmem_st_wait();
        }
        tmem_ld32(s_at, s[0]);
        tmem_ld_wait();
#pragma unroll
        for (int x = 0; x < kChunks; ++x) {
          uint32_t (&now)[32] = s[x & 1];
          if (x < kChunks - 1) tmem_ld32(s_at + (x + 1) * 32, s[(x + 1) & 1]);
          float t0 = -INFINITY, t1 = -INFINITY;
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            t0 = max3(t0, now[e], now[e + 1]);
            t1 = max3(t1, now[e + 2], now[e + 3]);
          }
          top = fmaxf(top, fmaxf(t0, t1));
          if (x < kChunks - 1) tmem_ld_wait();
        }
        const float c = fmaxf(scale_product(c_row, k_factor), 0x1p-126f);   // never 0: hidden keys are -inf
        top = top == -INFINITY ? -INFINITY : top * c;
        // reference of the weights: moves only where the maximum has left it behind, and then for all rows of the warp, whose
        // results are all read and written anyway, so that the next move is a while away
        const float want = top + v_log2;
        bool moved = false;
        float f = 1.0f;
        if (__any_sync(0xffffffffu, want > ref + kLag)) {
          const float ref_new = fmaxf(ref, want);
          if (want > ref) f = ex2_approx(ref - ref_new);
          ref = ref_new;
          moved = j > 0;
        }
        const float minus = ref == -INFINITY ? 0.0f : v_log2 - ref + kLift;
        const uint64_t c2 = pair(__float_as_uint(c), __float_as_uint(c)), minus2 = pair(__float_as_uint(minus), __float_as_uint(minus));
        uint64_t sum_a = 0, sum_b = 0;
#pragma unroll
        for (int x = kChunks - 1; x >= 0; --x) {
          uint32_t (&now)[32] = s[x & 1];
          if (x <= kChunks - 3) tmem_ld_wait();
          uint32_t w[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const uint64_t y = fma_pair(pair(now[2 * e], now[2 * e + 1]), c2, minus2);
            now[2 * e] = (uint32_t)y;
            now[2 * e + 1] = (uint32_t)(y >> 32);
          }
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float x0 = ex2_approx(__uint_as_float(now[2 * e])), x1 = ex2_approx(__uint_as_float(now[2 * e + 1]));
            const uint64_t y = pair(__float_as_uint(x0), __float_as_uint(x1));
            if (e & 1) sum_b = add_pair(sum_b, y);
            else sum_a = add_pair(sum_a, y);
            w[e] = pack_16x2<__half>(x0, x1);
          }
          if (x >= 2) tmem_ld32(s_at + (x - 2) * 32, now);
          tmem_st16(s_at + C::kN / 2 + x * 16, w);         // over columns that have been read
        }
        if (moved) {                                       // the product before has to be complete: mostly it is by now
          mbar_wait(&pv_done[group], (pv - 1) & 1, err, 68);
          tc_fence_after();
          __syncwarp();
          const uint64_t f2 = pair(__float_as_uint(f), __float_as_uint(f));
#pragma unroll 1
          for (int cc = 0; cc < D / 64; ++cc) {
            const uint32_t o_at = tmem + lane_addr + C::kO + group * 128 + cc * 64;
            tmem_ld32(o_at, s[0]);
            tmem_ld32(o_at + 32, s[1]);
            tmem_ld_wait();
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
              for (int e = 0; e < 16; ++e) {
                const uint64_t y = mul_pair(pair(s[h][2 * e], s[h][2 * e + 1]), f2);
                s[h][2 * e] = (uint32_t)y;
                s[h][2 * e + 1] = (uint32_t)(y >> 32);
              }
              tmem_st32(o_at + h * 32, s[h]);
            }
          }
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[group][place]);
        ++pv;
        const float m_new = fmaxf(m, top);
        l *= m_new == -INFINITY ? 1.0f : ex2_approx(m - m_new);
        m = m_new;
        // the sum is of weights times 2^(v_log2 - ref + lift)
        sum_a = add_pair(sum_a, sum_b);
        const float sum = __uint_as_float((uint32_t)sum_a) + __uint_as_float((uint32_t)(sum_a >> 32));
        l += m == -INFINITY ? sum : sum * ex2_approx(ref - v_log2 - kLift - m);
      }

      // ---- result of the segment
      const int slot = 2 * (int)blockIdx.x + (first_segment ? 0 : 1);
      const bool has = jobs > 0;
      float f = ref == -INFINITY ? 1.0f : ex2_approx(ref - kLift - m);      // brings O to 2^-m (no key: zeros, or NaN)
      if (has) {
        mbar_wait(&o_full[group], results & 1, err, 69);
        ++results;
        tc_fence_after();
        __syncwarp();
      }
      const uint32_t o_at = tmem + lane_addr + C::kO + group * 128;
      bool writes = true;
      if (merge) {
        // the groups' results of the same rows: the second one's goes through shared memory, where q was
        sh.m[group][row_in] = m;
        if (group == 1) sh.l()[row_in] = l;
        named_bar_sync(1, 32 * C::kSoft);
        const float m_all = fmaxf(sh.m[0][row_in], sh.m[1][row_in]);
        f *= m_all == -INFINITY ? 1.0f : ex2_approx(m - m_all);
        const uint32_t buf = smem_u32(smem + C::kQ) + row_in * 512;
        if (group == 1 && has) {
#pragma unroll 1
          for (int cc = 0; cc < 4; ++cc) {
            uint32_t o[32];
            tmem_ld32(o_at + cc * 32, o);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 8; ++e)
              asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(buf + (((cc * 8 + e) ^ lane) << 4)),
                           "f"(__uint_as_float(o[4 * e]) * f), "f"(__uint_as_float(o[4 * e + 1]) * f),
                           "f"(__uint_as_float(o[4 * e + 2]) * f), "f"(__uint_as_float(o[4 * e + 3]) * f)
                           : "memory");
          }
        }
        named_bar_sync(1, 32 * C::kSoft);
        writes = group == 0;
        if (writes && tiles > 1) {
          const float m1 = sh.m[1][row_in], l1 = sh.l()[row_in];
          l = m_all == -INFINITY ? l + l1 : l * ex2_approx(m - m_all) + l1 * ex2_approx(m1 - m_all);
        }
        m = m_all;
      }
      const bool add = merge && tiles > 1;
      const int rows_warp = min(max(rows - (both ? group * 128 : 0) - wq * 32, 0), 32);    // of this warp that exist
      if (writes && rows_warp > 0) {
        const float inv = !whole ? 1.0f : l != 0.0f ? __frcp_rn(l) : 0.0f;
        if (whole) {
          if (live && p.lse != nullptr) p.lse[out_row(p, at.q.t0 * p.g + i_row, at.head)] = lse_of(m, l);
        } else if (live) {
          p.ws_m[(int64_t)slot * C::kRows + row] = m;
          p.ws_l[(int64_t)slot * C::kRows + row] = l;
        }
        // a lane a row: of a result a sector at a time, of a partial one four columns, which lie row by row
        T* to = static_cast<T*>(p.out) + out_row(p, at.q.t0 * p.g + min(i_row, at.row_tile * C::kRows + rows - 1), at.head) * D;
        float4* part = reinterpret_cast<float4*>(p.ws_acc + (int64_t)slot * C::kRows * D) + row;
#pragma unroll 1
        for (int cc = 0; cc < D / 32; ++cc) {
          uint32_t o[32];
          tmem_ld32(o_at + cc * 32, o);
          tmem_ld_wait();
          if (add) {
            const uint32_t buf = smem_u32(smem + C::kQ) + row_in * 512;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              float x[4];
              asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3]) : "r"(
                               buf + (((cc * 8 + e) ^ lane) << 4))
                           : "memory");
#pragma unroll
              for (int k = 0; k < 4; ++k) o[4 * e + k] = __float_as_uint((__uint_as_float(o[4 * e + k]) * f + x[k]) * inv);
            }
          } else {
            const float f_inv = f * inv;
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f_inv);
          }
          if (live && whole) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              uint32_t w[8];
#pragma unroll
              for (int k = 0; k < 8; ++k) w[k] = pack_16x2<T>(__uint_as_float(o[16 * e + 2 * k]), __uint_as_float(o[16 * e + 2 * k + 1]));
              store_sector(to + cc * 32 + e * 16, w);
            }
          } else if (live) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              *reinterpret_cast<uint4*>(part + (cc * 8 + e) * C::kRows) = make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
          }
          __syncwarp();
        }
      }
      tc_fence_before();
      __syncwarp();
      if (has && lane == 0) mbar_arrive(&o_free[group]);
      if (merge && lane == 0) mbar_arrive(&q_free);
      if (!whole && at.from == 0 && tid == 0) p.cut[blockIdx.x] = cut_unit(p, at, sh.share, first_segment);
      n += tiles;
      first_segment = false;
    }
  }
  clear_untouched<T, D, C::kRows, kTile, kTree>(p);
  tc_fence_before();
  __syncthreads();
  report_error(&expired, p.status);
  if (warp == C::kIssue) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <typename T, int D, bool kTree>
int run_kernel(const PagedParams& p, int ctas, cudaStream_t st) {
  using C = Cfg<D>;
  const void* kern = reinterpret_cast<const void*>(paged_chunk_kernel<T, D, kTree>);
  constexpr int kBytes = smem_bytes<D, kTree>();
  if (int rc = allow_smem("nvfp4_kv8_attention", kern, kBytes)) return rc;
  prefer_l1(kern, kSmemPercent);
  if (int rc = launch("nvfp4_kv8_attention", paged_chunk_kernel<T, D, kTree>, dim3(ctas), C::kThreads, kBytes, st, p)) return rc;
  return launch_combine<T, D, C::kRows, true>(p, ctas, st);
}
template <typename T, int D>
int run_chunk(const PagedParams& p, int ctas, cudaStream_t st) {
  return p.tree != nullptr ? run_kernel<T, D, true>(p, ctas, st) : run_kernel<T, D, false>(p, ctas, st);
}

}  // namespace

int launch_paged_chunk(const PagedParams& p, int q_dtype, int d, int ctas, cudaStream_t st) {
  if (q_dtype == NVFP4_DT_BF16) return d == 128 ? run_chunk<__nv_bfloat16, 128>(p, ctas, st) : run_chunk<__nv_bfloat16, 256>(p, ctas, st);
  return d == 128 ? run_chunk<__half, 128>(p, ctas, st) : run_chunk<__half, 256>(p, ctas, st);
}

}  // namespace nvfp4
