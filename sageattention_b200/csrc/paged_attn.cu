// Attention over the paged 8-bit KV cache for few query rows a request: decode and short drafts.
//
//   s_j = scaling * (q . k_j),  out = sum_j softmax(s)_j v_j,  k_j = ks_b * code, v_j = vs_b * code (b the block of key j)
//
// A unit's rows are 8 NT at most; every warp of a CTA streams keys of its own (kSub of each tile) through a ring of its own,
// filled by cp.async, so nothing in the stream waits for another warp.  Codes become halves (exact) on their way from shared
// memory into mma.sync m16n8k16 with the keys on its 16 rows: S^T = K Q^T and O^T = V^T P^T.  Eight query rows then cost
// half of what they would on the 16-row side, in products, exponentials and registers.
//
// What bounds it: HBM.  At 6.5 TB/s an SM gets 23 bytes a clock; the 8 KB that a warp takes at once (D = 128: 32 keys) are
// 32 NT products and some 400 instructions of four schedulers, a quarter of the issue slots at NT = 1; tcgen05 would need
// its 128 rows filled, and what it saves is not what bounds.
//
// Measured with the merge: one query row of 839 MB of cache 142 to 152 us (the kernel alone 131 to 135, 0.95 of the copy
// rate); 160 requests of 1 to 4100 keys, 51.7 MB, 22.5 us and D = 256, 87.7 MB, 28.7 us, of which 3 are the deal, 3 to 5 the
// merge, and the rest units of few tiles each; 20 rows a request, 169 MB, 68.2 us: 1290 instructions a warp and 32 keys at two
// warps a scheduler, which registers allow no more of.
//
// Precision: q enters as halves scaled by a power of two per row, so that a bf16 or fp16 q is exact unless 2^-26 of its row's
// maximum (an fp32 q is two halves); scores, sums and outputs are fp32, relative to a reference that lags behind the running
// maximum by 2^kLag at most, so that in most tiles no lane has to know another's maximum.  A weight p_j vs_b is a half (two
// for fp32), relative to a reference of its own and times 2^kLift: its rounding is 2^-11 of itself, and of weights below
// 2^-(14 + kLift) of the largest 2^-(25 + kLift) of that.
#include <limits.h>
#include "common/abi.cuh"
#include "common/fp4.cuh"
#include "common/kv8.cuh"
#include "common/launch.cuh"
#include "common/paged.cuh"
#include "common/sm100.cuh"

namespace nvfp4 {
namespace {

constexpr int kWarps = 4, kThreads = 32 * kWarps, kStages = 2;
constexpr int kCtas = 3;                      // of an SM
constexpr int kStageBytes = 8192;             // K and V of a warp's keys of a tile
constexpr float kLag = 9.0f, kLift = 5.0f;

template <int D>
struct Cfg {
  static constexpr int kSub = kStageBytes / (2 * D);       // keys of a warp in a tile: 32, or 16 at D = 256
  static constexpr int kTile = kSub * kWarps;
};

__device__ __forceinline__ void cp_async_16(uint32_t saddr, const void* gptr, uint32_t src_bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(saddr), "l"(gptr), "r"(src_bytes) : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ float2 lds_f2(uint32_t a) {
  float2 v;
  asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void ldmatrix_x4_t(uint32_t a, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a)
               : "memory");
}
// 8 x 8 matrix of halves, a row in four lanes: transposed
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Key of row i of eight: 0 4 1 5 2 6 3 7.  The rows that one phase of a 16-byte load touches then differ in bit 2, and with
// the swizzle (chunk ^ row) in their banks.
__device__ __forceinline__ int key_of_row(int i) { return (i >> 1) | ((i & 1) << 2); }
// Exponent of a scale, as log2 of what weights are kept relative to.
__device__ __forceinline__ float scale_exponent(float s) {
  return fmaxf((float)((int)(__float_as_uint(s) >> 23 & 0xFF) - 127), -112.0f);
}

template <typename T, int D, int NT>
struct Smem {
  static constexpr bool kTwo = sizeof(T) == 4;             // fp32: q and weights as two halves each
  static constexpr int kQ = 8 * NT * D * 2;                // one set of halves
  static constexpr int kMerge = kWarps * 8 * 64 * 4;       // eight rows of 64 columns of each warp
  static constexpr int kShared = kQ * (kTwo ? 2 : 1) > kMerge ? kQ * (kTwo ? 2 : 1) : kMerge;
  static constexpr int kRing = kWarps * kStages * kStageBytes;
  static constexpr int kBytes = kRing + kShared;
};

template <typename T, int D, int NT>
__global__ void __launch_bounds__(kThreads, NT == 1 ? kCtas : 2) paged_attn_kernel(PagedParams p) {
  using S = Smem<T, D, NT>;
  constexpr int kSub = Cfg<D>::kSub, kTile = Cfg<D>::kTile, kRows = 8 * NT;
  constexpr int kHalves = kSub / 16;                       // 16 keys are the rows of a product
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ int64_t list_s[kWarps + 2];
  __shared__ float q_inv[kRows];                           // undoes the power of two that a query row was scaled by
  __shared__ float m_s[kWarps][kRows], l_s[kWarps][kRows];
  __shared__ float scale_s[kWarps][kStages][4];            // K and V scales of the stage's two halves
  __shared__ int keys_s[kWarps][kStages][2];               // keys of each half that are there
  const int tid = threadIdx.x, lane = tid & 31, warp = warp_index();
  const int cta = blockIdx.x;
  griddep_wait();
  griddep_launch();

  using Place = Walk<kRows, kTile>;
  Place use;
  const int64_t share = deal_tiles<kThreads>(p, list_s, use);
  if (tid == 0) p.cut[cta] = make_int4(0, 0, 0, 0);
  if (use.left > 0) {
    // ---- the ring of this warp: copies of tile `ahead_tile` of `ahead` go into stage `fill`
    const uint32_t ring = smem_u32(smem) + warp * kStages * kStageBytes;
    const uint32_t shared = smem_u32(smem) + S::kRing;
    Place ahead = use;
    bool more = ahead.open();
    int ahead_tile = ahead.from, ahead_limit = ahead.q.limit(p, ahead.row_tile);
    int id[kHalves];
    auto look_up = [&]() {                                 // blocks of the keys of `ahead`, a tile before they are needed
      const int key = ahead_tile * kTile + warp * kSub;
#pragma unroll
      for (int h = 0; h < kHalves; ++h)
        id[h] = more && key + h * 16 < ahead_limit ? p.table[ahead.r * p.table_row + ((key + h * 16) >> p.log_block)] : -1;
    };
    auto warm = [&](const Place& u) {                      // query rows of a unit to come, into L2
      constexpr int kLines = D * sizeof(T) / 128;
      if (warp != 0) return;
      for (int i = lane; i < u.q.rows(p, u.row_tile) * kLines; i += 32)
        prefetch_l2(reinterpret_cast<const uint8_t*>(query_row<T>(p, u.q.t0, u.row_tile * kRows + i / kLines, u.head)) + i % kLines * 128);
    };
    // where a lane's 16-byte pieces of 16 keys go: piece i is key (32 i + lane) / (D / 16), and the swizzle has a period of eight keys
    auto piece = [&](int i) -> uint32_t {
      const int at = i * 32 + lane, key_in = at / (D / 16), chunk = at % (D / 16);
      return (uint32_t)(chunk >> 3) * (kSub * 128) + (uint32_t)key_in * 128 + (uint32_t)(((chunk & 7) ^ (key_in & 7)) << 4);
    };
    auto ask = [&](int stage) {
      if (more) {
        const int key = ahead_tile * kTile + warp * kSub;
        const uint32_t base_s = ring + stage * kStageBytes;
#pragma unroll
        for (int h = 0; h < kHalves; ++h) {
          const bool there = (unsigned)id[h] < (unsigned)p.blocks;
          const int keys = there ? min(max(ahead_limit - key - h * 16, 0), 16) : 0;
          if (keys > 0) {
            const int64_t row = ((int64_t)ahead.head << p.log_block) + ((key + h * 16) & ((1 << p.log_block) - 1));
            const uint8_t* pk = p.k + id[h] * p.k_block + row * D + lane * 16;
            const uint8_t* pv = p.v + id[h] * p.v_block + row * D + lane * 16;
            const uint32_t dst = base_s + h * 16 * 128;
            auto copy = [&](auto bytes) {                  // codes behind the last key: zeros
#pragma unroll
              for (int i = 0; i < D / 32; ++i) {
                cp_async_16(dst + piece(i), pk + i * 512, bytes(i));
                cp_async_16(dst + kStageBytes / 2 + piece(i), pv + i * 512, bytes(i));
              }
            };
            if (keys == 16) copy([](int) { return 16u; });
            else copy([&](int i) { return (i * 32 + lane) / (D / 16) < keys ? 16u : 0u; });
            if (lane < 2)
              cp_async_4(smem_u32(&scale_s[warp][stage][lane * 2 + h]),
                         (lane == 0 ? p.ks + id[h] * p.ks_block : p.vs + id[h] * p.vs_block) + ahead.head, 4);
          }
          if (lane == 0) keys_s[warp][stage][h] = keys;
        }
        if (++ahead_tile == ahead.to) {
          ahead.close(p);
          more = ahead.open();
          if (more) {
            ahead_tile = ahead.from;
            ahead_limit = ahead.q.limit(p, ahead.row_tile);
            warm(ahead);
          }
        }
        look_up();
      }
      cp_async_commit();
    };
    look_up();
    if (more) warm(ahead);
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) ask(s);
    int stage = 0;

    // ---- segments: the tiles of one unit in this share
    const int g8 = lane >> 2, c4 = lane & 3;               // row (key, or pair of the head dim) and pair of query rows of a product
    const int krow = key_of_row(g8);
    bool first = true;
    for (; use.open(); use.close(p)) {
      const int rows = use.q.rows(p, use.row_tile);
      const bool whole = use.whole();

      // query rows as fragments of the products: eight threads a row, elements 16 e .. 16 e + 15 for e = tid % 8 (+ 8)
#pragma unroll 1
      for (int row = tid >> 3; row < kRows; row += kThreads / 8) {
        const int e0 = tid & 7;
        const T* pq = query_row<T>(p, use.q.t0, use.row_tile * kRows + min(row, rows - 1), use.head);
        float x[D / 128][16];
        float big = 0.0f;
#pragma unroll
        for (int u = 0; u < D / 128; ++u) {
          constexpr int kPer = 16 / (int)sizeof(T);
          uint4 raw[16 / kPer];
#pragma unroll
          for (int w = 0; w < 16 / kPer; ++w) raw[w] = reinterpret_cast<const uint4*>(pq + (u * 8 + e0) * 16)[w];
          const T* t = reinterpret_cast<const T*>(raw);
#pragma unroll
          for (int k = 0; k < 16; ++k) x[u][k] = row < rows ? to_f32<T>(t[k]) : 0.0f;
        }
#pragma unroll
        for (int u = 0; u < D / 128; ++u)
#pragma unroll
          for (int k = 0; k < 16; ++k) big = fmaxf(big, fabsf(x[u][k]));
        const uint32_t eight = 0xFFu << (lane & 24);
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) big = fmaxf(big, __shfl_xor_sync(eight, big, o));
        // largest element in [2^12, 2^13); scaling below zero turns q
        const int ex = min(max((int)(__float_as_uint(big) >> 23) - 127, -110), 127);
        const float up = copysignf(__uint_as_float((uint32_t)(127 + 12 - ex) << 23), p.scale_log2);
        if (e0 == 0) q_inv[row] = big == 0.0f ? 0.0f : ldexpf(fabsf(p.scale_log2), ex - 12);
        // products of 16 elements: lane (row % 8) * 4 + e % 4 has elements 4 k .. 4 k + 3 of its 16; two products' words together
        const uint32_t dst = shared + (row >> 3) * 512;
#pragma unroll
        for (int u = 0; u < D / 128; ++u) {
          const int e = u * 8 + e0;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t a = dst + (((e >> 2) * 2 + (k >> 1)) * NT) * 512 + ((row & 7) * 4 + (e & 3)) * 16 + (k & 1) * 8;
            float lo[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) lo[j] = x[u][4 * k + j] * up;
            const uint32_t w0 = pack_16x2<__half>(lo[0], lo[1]), w1 = pack_16x2<__half>(lo[2], lo[3]);
            sts_v2(a, w0, w1);
            if constexpr (S::kTwo) {
              const float2 f0 = __half22float2(*reinterpret_cast<const __half2*>(&w0));
              const float2 f1 = __half22float2(*reinterpret_cast<const __half2*>(&w1));
              sts_v2(a + S::kQ, pack_16x2<__half>(lo[0] - f0.x, lo[1] - f0.y), pack_16x2<__half>(lo[2] - f1.x, lo[3] - f1.y));
            }
          }
        }
      }
      __syncthreads();
      // this thread's query rows: 8 nt + 2 c4, + 1.  Rows of no query see all keys (they are not stored).
      float inv[NT][2];
      int lim[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int row = nt * 8 + 2 * c4 + k;
          inv[nt][k] = q_inv[row];
          lim[nt][k] = row < rows ? use.q.seen(p, use.row_tile * kRows + row) : INT_MAX;
        }
      const int lim_first = use.q.seen(p, use.row_tile * kRows);       // the smallest of all rows

      float o[D / 16][NT][4];
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int k = 0; k < 4; ++k) o[i][nt][k] = 0.0f;
      // references of the scores and of the weights, 2^(their difference + kLift), sum
      float ref[NT][2], ref_w[NT][2], lift[NT][2], l[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          ref[nt][k] = ref_w[nt][k] = -INFINITY;
          lift[nt][k] = l[nt][k] = 0.0f;
        }

      for (int tile = use.from; tile < use.to; ++tile) {
        ask(stage == 0 ? kStages - 1 : stage - 1);
        cp_async_wait<kStages - 1>();
        __syncwarp();
        const uint32_t base_s = ring + stage * kStageBytes;
        const int key = tile * kTile + warp * kSub;
        int keys[kHalves];
        bool all = true;
        int any = 0;
#pragma unroll
        for (int h = 0; h < kHalves; ++h) {
          keys[h] = keys_s[warp][stage][h];
          all = all && keys[h] == 16;
          any |= keys[h];
        }
        if (any != 0) {
          float kscale[kHalves], vscale[kHalves], vexp[kHalves];
#pragma unroll
          for (int h = 0; h < kHalves; ++h) {
            kscale[h] = keys[h] ? scale_s[warp][stage][h] : 0.0f;
            vscale[h] = keys[h] ? scale_s[warp][stage][2 + h] : 0.0f;
            vexp[h] = scale_exponent(vscale[h]);
          }
          float s[kHalves][NT][4];
#pragma unroll
          for (int h = 0; h < kHalves; ++h)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int k = 0; k < 4; ++k) s[h][nt][k] = 0.0f;
#pragma unroll
          for (int e = 0; e < D / 64; ++e) {
            // rows of a missing half may be stale codes: masked below
            uint4 lo[kHalves], hi[kHalves];                // keys g8 and g8 + 8 of a half, 16 elements of each
#pragma unroll
            for (int h = 0; h < kHalves; ++h) {
              const uint32_t a = base_s + (e >> 1) * (kSub * 128) + (h * 16 + krow) * 128 + ((((e & 1) * 4 + c4) ^ krow) << 4);
              lo[h] = lds128(a);
              hi[h] = lds128(a + 8 * 128);
            }
#pragma unroll
            for (int k2 = 0; k2 < 2; ++k2) {
              uint4 b[NT], b2[NT];
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                b[nt] = lds128(shared + ((e * 2 + k2) * NT + nt) * 512 + lane * 16);
                if constexpr (S::kTwo) b2[nt] = lds128(shared + S::kQ + ((e * 2 + k2) * NT + nt) * 512 + lane * 16);
              }
#pragma unroll
              for (int h = 0; h < kHalves; ++h) {
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                  uint32_t a[4];
                  half4_of_e4m3x4(k2 == 0 ? (k == 0 ? lo[h].x : lo[h].y) : (k == 0 ? lo[h].z : lo[h].w), a[0], a[2]);
                  half4_of_e4m3x4(k2 == 0 ? (k == 0 ? hi[h].x : hi[h].y) : (k == 0 ? hi[h].z : hi[h].w), a[1], a[3]);
#pragma unroll
                  for (int nt = 0; nt < NT; ++nt) {
                    mma_16816(s[h][nt], a, k == 0 ? b[nt].x : b[nt].z, k == 0 ? b[nt].y : b[nt].w);
                    if constexpr (S::kTwo) mma_16816(s[h][nt], a, k == 0 ? b2[nt].x : b2[nt].z, k == 0 ? b2[nt].y : b2[nt].w);
                  }
                }
              }
            }
          }
          // scores in units of log2; element k of a product: key g8 + 8 (k / 2), row 2 c4 + k % 2
          const bool masks = !all || key + kSub > lim_first;
          float top[NT][2], top_w[NT][2];                  // largest of this thread's keys, and of them with their V scale
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int k = 0; k < 2; ++k) top[nt][k] = top_w[nt][k] = -INFINITY;
#pragma unroll
          for (int h = 0; h < kHalves; ++h)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                const float f = scale_product(inv[nt][k], kscale[h]);
                s[h][nt][k] *= f;
                s[h][nt][2 + k] *= f;
                if (masks) {
                  if (krow >= keys[h] || key + h * 16 + krow >= lim[nt][k]) s[h][nt][k] = -INFINITY;
                  if (krow + 8 >= keys[h] || key + h * 16 + krow + 8 >= lim[nt][k]) s[h][nt][2 + k] = -INFINITY;
                }
                const float t = fmaxf(s[h][nt][k], s[h][nt][2 + k]);
                top[nt][k] = fmaxf(top[nt][k], t);
                top_w[nt][k] = fmaxf(top_w[nt][k], t + vexp[h]);
              }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            bool move = false;
#pragma unroll
            for (int k = 0; k < 2; ++k) move = move || top[nt][k] > ref[nt][k] + kLag || top_w[nt][k] > ref_w[nt][k] + kLag;
            if (__any_sync(0xffffffffu, move)) {
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                float m = top[nt][k], w = top_w[nt][k];
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) {
                  m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
                  w = fmaxf(w, __shfl_xor_sync(0xffffffffu, w, x));
                }
                m = fmaxf(m, ref[nt][k]);
                w = fmaxf(w, ref_w[nt][k]);
                if (m != -INFINITY) {
                  l[nt][k] *= ex2_approx(ref[nt][k] - m);
                  const float f = ex2_approx(ref_w[nt][k] - w);
#pragma unroll
                  for (int i = 0; i < D / 16; ++i) {
                    o[i][nt][k] *= f;
                    o[i][nt][2 + k] *= f;
                  }
                  lift[nt][k] = ex2_approx(fminf(m - w + kLift, 126.0f));
                }
                ref[nt][k] = m;
                ref_w[nt][k] = w;
              }
            }
          }
#pragma unroll
          for (int h = 0; h < kHalves; ++h) {
            uint32_t pb[NT][2], pb2[NT][2];                // weights as the other operand: eight keys a word
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              float w[4];
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                const float r = ref[nt][k] == -INFINITY ? 0.0f : ref[nt][k], c = lift[nt][k] * vscale[h];
                const float p0 = ex2_approx(s[h][nt][k] - r), p1 = ex2_approx(s[h][nt][2 + k] - r);
                l[nt][k] += p0 + p1;
                w[k] = p0 * c;
                w[2 + k] = p1 * c;
              }
#pragma unroll
              for (int y = 0; y < 2; ++y) {
                const uint32_t v = pack_16x2<__half>(w[2 * y], w[2 * y + 1]);
                pb[nt][y] = transposed(v);
                if constexpr (S::kTwo) {
                  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&v));
                  pb2[nt][y] = transposed(pack_16x2<__half>(w[2 * y] - f.x, w[2 * y + 1] - f.y));
                }
              }
            }
            if (keys[h] == 0) continue;                    // nothing was copied: stale codes may be NaN
            const int vrow = h * 16 + ((lane >> 3) & 1) * 8 + key_of_row(lane & 7);
#pragma unroll
            for (int dg = 0; dg < D / 32; ++dg) {
              const int chunk = dg * 2 + (lane >> 4);
              uint32_t r[4];
              ldmatrix_x4_t(base_s + kStageBytes / 2 + (chunk >> 3) * (kSub * 128) + vrow * 128 +
                                (((chunk & 7) ^ (vrow & 7)) << 4),
                            r);
#pragma unroll
              for (int ch = 0; ch < 2; ++ch) {
                // bytes (d, d + 1) of two keys -> the keys of d (row g8 of the product), the keys of d + 1 (row g8 + 8)
                uint32_t a[4];
                half4_of_e4m3x4(__byte_perm(r[2 * ch], 0, 0x3120), a[0], a[1]);
                half4_of_e4m3x4(__byte_perm(r[2 * ch + 1], 0, 0x3120), a[2], a[3]);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                  mma_16816(o[dg * 2 + ch][nt], a, pb[nt][0], pb[nt][1]);
                  if constexpr (S::kTwo) mma_16816(o[dg * 2 + ch][nt], a, pb2[nt][0], pb2[nt][1]);
                }
              }
            }
          }
        }
        __syncwarp();                                      // the stage may be filled again
        stage = stage + 1 == kStages ? 0 : stage + 1;
      }

      // ---- merge of the four warps, in warp order: final rows, or a partial result of the unit
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) l[nt][k] += __shfl_xor_sync(0xffffffffu, l[nt][k], x);
          if (g8 == 0) {
            m_s[warp][nt * 8 + 2 * c4 + k] = ref[nt][k];
            l_s[warp][nt * 8 + 2 * c4 + k] = l[nt][k];
          }
        }
      __syncthreads();                                     // and nobody needs the query fragments any more
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          float top = m_s[0][nt * 8 + 2 * c4 + k];
#pragma unroll
          for (int w = 1; w < kWarps; ++w) top = fmaxf(top, m_s[w][nt * 8 + 2 * c4 + k]);
          // weights carry 2^(kLift - ref_w); brought to 2^-top
          const float f = ref_w[nt][k] == -INFINITY ? 0.0f : ex2_approx(ref_w[nt][k] - top - kLift);
#pragma unroll
          for (int i = 0; i < D / 16; ++i) {
            o[i][nt][k] *= f;
            o[i][nt][2 + k] *= f;
          }
        }
      const int slot = first ? 2 * cta : 2 * cta + 1;
#pragma unroll 1
      for (int pass = 0; pass < NT * (D / 64); ++pass) {
        const int nt = pass % NT, cols = pass / NT;        // rows 8 nt .., columns 64 cols ..
        if (nt * 8 >= rows) continue;
#pragma unroll
        for (int x = 0; x < NT * (D / 64); ++x)
          if (x == pass) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                const float* v = o[x / NT * 4 + i][x % NT];
                const uint32_t dst = shared + ((warp * 8 + 2 * c4 + k) * 64 + ((i ^ c4) * 16) + 2 * g8) * 4;
                asm volatile("st.shared.v2.f32 [%0], {%1, %2};" ::"r"(dst), "f"(v[k]), "f"(v[2 + k]) : "memory");
              }
          }
        __syncthreads();
#pragma unroll 1
        for (int in = warp * 2; in < warp * 2 + 2; ++in) {
          const int row = nt * 8 + in;
          if (row >= rows) break;
          float2 sum = make_float2(0.0f, 0.0f);
          float top = m_s[0][row], total_l = 0.0f;
#pragma unroll
          for (int w = 1; w < kWarps; ++w) top = fmaxf(top, m_s[w][row]);
#pragma unroll
          for (int w = 0; w < kWarps; ++w) {
            const float2 v = lds_f2(shared + ((w * 8 + in) * 64 + (((lane >> 3) ^ (in >> 1)) * 16) + 2 * (lane & 7)) * 4);
            sum.x += v.x;
            sum.y += v.y;
            total_l += top == -INFINITY ? l_s[w][row] : l_s[w][row] * ex2_approx(m_s[w][row] - top);   // no key: 0, or NaN
          }
          if (whole) {
            const float f = total_l == 0.0f ? 0.0f : __frcp_rn(total_l);
            const int64_t to = out_row(p, use.q.t0 * p.g + use.row_tile * kRows + row, use.head);
            T* dst = static_cast<T*>(p.out) + to * D + cols * 64 + lane * 2;
            if constexpr (S::kTwo) *reinterpret_cast<float2*>(dst) = make_float2(sum.x * f, sum.y * f);
            else *reinterpret_cast<uint32_t*>(dst) = pack_16x2<T>(sum.x * f, sum.y * f);
            if (cols == 0 && lane == 0 && p.lse != nullptr) p.lse[to] = lse_of(top, total_l);
          } else {
            *reinterpret_cast<float2*>(p.ws_acc + ((int64_t)slot * kRows + row) * D + cols * 64 + lane * 2) = sum;
            if (cols == 0 && lane == 0) {
              p.ws_m[slot * kRows + row] = top;
              p.ws_l[slot * kRows + row] = total_l;
            }
          }
        }
        __syncthreads();
      }
      // begun here, finished by the CTAs behind this one
      if (!whole && use.from == 0 && tid == 0) p.cut[cta] = cut_unit(p, use, share, first);
      first = false;
    }
  }
  clear_untouched<T, D, kRows, kTile>(p);
}

template <typename T, int D, int NT>
int run_attention(const PagedParams& p, int sms, cudaStream_t st) {
  using S = Smem<T, D, NT>;
  const int grid = (NT == 1 ? kCtas : 2) * sms;
  if (int rc = allow_smem("nvfp4_kv8_attention", reinterpret_cast<const void*>(paged_attn_kernel<T, D, NT>), S::kBytes)) return rc;
  if (int rc = launch("nvfp4_kv8_attention", paged_attn_kernel<T, D, NT>, dim3(grid), kThreads, S::kBytes, st, p)) return rc;
  return launch_combine<T, D, 8 * NT, false>(p, grid, st);
}

// Which kernel, by query rows a request on average (their numbers are on the device): eight, sixteen or (D = 128) 24 rows of
// this file's, rounded up, or (D = 128) two row tiles of sixteen; above them the one whose tensor-memory products take 128 or
// 256 rows at a time.  fp32 queries, whose products need two halves, stay here, sixteen rows at a time.  Measured, 32 requests
// of 300 to 8190 keys, Hk 8 G 4, the other kernel in brackets: D 128, 24 rows 73.7 (131) us, 32 rows 96 (133), 40 rows 121 (133) but
// of 256 requests 233 (207); Hk 4 D 256, 16 rows 59.4 (73.8), 20 rows (73.8).  The average is over all rows of the table and all
// query tokens, padded ones too, as the host knows no others: a chunk of 2048 tokens over 12288 keys takes 0.39 ms in a table of 32 rows and,
// in tiles of sixteen rows, 2.4 in one of 256 whose other rows are idle.
struct Choice {
  bool chunk;
  int nt, ctas;
  int64_t rows;
};
Choice choose(int q_dtype, int64_t tokens, int64_t requests, int64_t g, int d, int sms) {
  const int64_t rows = (tokens * g + requests - 1) / requests, most = d == 128 ? 32 : 16;
  if (q_dtype != NVFP4_DT_FP32 && rows > most) return {true, 0, sms, paged_chunk_rows(d)};
  const int nt = rows <= 8 ? 1 : rows <= 16 || rows > 24 || q_dtype == NVFP4_DT_FP32 ? 2 : 3;
  return {false, nt, (nt == 1 ? kCtas : 2) * sms, 8 * nt};
}
template <typename T, int D>
int run_rows(const PagedParams& p, int nt, int sms, cudaStream_t st) {
  if (nt == 1) return run_attention<T, D, 1>(p, sms, st);
  if constexpr (D == 128 && sizeof(T) == 2)
    if (nt == 3) return run_attention<T, D, 3>(p, sms, st);
  return run_attention<T, D, 2>(p, sms, st);
}

}  // namespace
}  // namespace nvfp4

using namespace nvfp4;

extern "C" int nvfp4_kv8_attention_plan(int q_dtype, int64_t tokens, int64_t requests, int g, int d, int sm_count,
                                        size_t* workspace_bytes) {
  NVFP4_REQUIRE(d == 128 || d == 256, "nvfp4_kv8_attention_plan: D must be 128 or 256");
  NVFP4_REQUIRE(tokens >= 0 && requests >= 1 && g >= 1 && sm_count >= 1 && workspace_bytes != nullptr,
                "nvfp4_kv8_attention_plan: bad argument");
  const Choice c = choose(q_dtype, tokens, requests, g, d, sm_count);
  *workspace_bytes = (size_t)(c.ctas * paged_slot_bytes(c.rows, d));
  return 0;
}

extern "C" int nvfp4_kv8_attention(const void* q, int q_dtype, int64_t s_qt, int64_t s_qh, const int32_t* cu_seqlens,
                                   int64_t tokens, const uint8_t* k_cache, int64_t k_block, const uint8_t* v_cache,
                                   int64_t v_block, const float* k_scale, int64_t ks_block, const float* v_scale,
                                   int64_t vs_block, int64_t blocks, int block_size, const int32_t* table, int64_t table_row,
                                   int64_t width, const int32_t* lengths, int64_t requests, int64_t hk, int g, int d,
                                   float scaling, void* out, float* lse, void* workspace, size_t workspace_bytes,
                                   int* status, nvfp4_stream_t stream) {
  NVFP4_REQUIRE(d == 128 || d == 256, "nvfp4_kv8_attention: D must be 128 or 256");
  int lb = 4;
  while (lb < 7 && (1 << lb) != block_size) ++lb;
  NVFP4_REQUIRE((1 << lb) == block_size, "nvfp4_kv8_attention: block_size must be 16, 32, 64 or 128");
  NVFP4_REQUIRE(requests >= 1 && requests < (1 << 30) && tokens >= 0 && hk >= 1 && g >= 1 && tokens * g < INT32_MAX &&
                    hk * g < (1 << 20) && blocks >= 0 && blocks < INT32_MAX && width >= 0 && width * block_size < INT32_MAX - 256,
                "nvfp4_kv8_attention: sizes out of range");
  NVFP4_REQUIRE(cu_seqlens != nullptr || tokens == requests, "nvfp4_kv8_attention: one token a request without cu_seqlens");
  NVFP4_REQUIRE((((uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)workspace) & 15) == 0 && ((uintptr_t)out & 31) == 0 &&
                    ((k_block | v_block) & 15) == 0,
                "nvfp4_kv8_attention: cache blocks and workspace must be 16-byte aligned, out 32-byte aligned");
  NVFP4_REQUIRE(((uintptr_t)q & 15) == 0 && ((s_qt | s_qh) * (q_dtype == NVFP4_DT_FP32 ? 4 : 2) & 15) == 0,
                "nvfp4_kv8_attention: query rows must be 16-byte aligned");
  NVFP4_REQUIRE(isfinite(scaling), "nvfp4_kv8_attention: scaling must be finite");
  if (tokens == 0) return 0;
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  const Choice c = choose(q_dtype, tokens, requests, g, d, sms);
  const int grid = c.ctas;
  const int64_t rows = c.rows;
  NVFP4_REQUIRE(workspace_bytes >= (size_t)(grid * paged_slot_bytes(rows, d)), "nvfp4_kv8_attention: workspace too small");
  NVFP4_REQUIRE(q_dtype >= NVFP4_DT_BF16 && q_dtype <= NVFP4_DT_FP32, "nvfp4_kv8_attention: unknown dtype %d", q_dtype);
  PagedParams p{q, s_qt, s_qh, cu_seqlens, tokens, k_cache, v_cache, k_block, v_block, k_scale, v_scale, ks_block, vs_block, table,
                table_row, lengths, (int)requests, (int)width, (int)blocks, lb, (int)hk, g, 0, 0, scaling * kLog2e, out, lse,
                nullptr, nullptr, nullptr, nullptr, status};
  set_group(p, g);
  p.ws_acc = static_cast<float*>(workspace);
  p.cut = reinterpret_cast<int4*>(p.ws_acc + 2 * grid * rows * d);
  p.ws_m = reinterpret_cast<float*>(p.cut + grid);
  p.ws_l = p.ws_m + 2 * grid * rows;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (c.chunk) return launch_paged_chunk(p, q_dtype, d, grid, st);
  switch (q_dtype) {
    case NVFP4_DT_BF16: return d == 128 ? run_rows<__nv_bfloat16, 128>(p, c.nt, sms, st) : run_rows<__nv_bfloat16, 256>(p, c.nt, sms, st);
    case NVFP4_DT_FP16: return d == 128 ? run_rows<__half, 128>(p, c.nt, sms, st) : run_rows<__half, 256>(p, c.nt, sms, st);
    default: return d == 128 ? run_rows<float, 128>(p, c.nt, sms, st) : run_rows<float, 256>(p, c.nt, sms, st);
  }
}
