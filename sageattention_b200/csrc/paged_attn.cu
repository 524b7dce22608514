// Attention over the paged 8-bit KV cache for few query rows a request: decode and short drafts.
//
//   s_j = scaling * (q . k_j),  out = sum_j softmax(s)_j v_j,  k_j = ks_b * code, v_j = vs_b * code (b the block of key j)
//
// A unit is (request, KV head, 16 query rows): the heads of a group, for each of the request's query tokens.  Its keys are
// cut into tiles, all tiles of all units are one list (request by request), and every CTA streams an equal share of it, so
// ragged lengths need no plan on the host.  HBM bounds it: each code is read once by cp.async into a ring of its warp's own
// (no barrier in the stream), turned into halves (exact) and multiplied by mma.sync m16n8k16, whose 16 rows are the unit's.
// At 6.5 TB/s an SM gets 23 bytes a clock; the products of those bytes are 370 of the 1024 multiplications a clock of the
// legacy tensor path, so tcgen05 would have nothing to give here.
//
// Precision: q enters as halves scaled by a power of two per row, so that a bf16 or fp16 q is exact unless 2^-26 of its row's
// maximum (an fp32 q is two halves); scores, maxima, sums and outputs are fp32.  A weight p_j vs_b is a half (two for
// fp32), relative to the largest weight so far and times 2^14: its rounding is 2^-11 of itself, and of weights below 2^-28 of
// the largest 2^-39 of that.
#include <limits.h>
#include "common/abi.cuh"
#include "common/fp4.cuh"
#include "common/kv8.cuh"
#include "common/launch.cuh"
#include "common/paged.cuh"
#include "common/sm100.cuh"

namespace nvfp4 {
namespace {

constexpr int kWarps = 4, kThreads = 32 * kWarps, kStages = 3;
constexpr int kRowTile = 16;
constexpr int kStageBytes = 8192;             // K and V of a warp's keys of a tile

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
__device__ __forceinline__ void ldmatrix_x4_t(uint32_t a, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a)
               : "memory");
}
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint4& a, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ex2(float x) { return ex2_approx(x); }
// Key of column i of a product of eight: 0 4 1 5 2 6 3 7.  The rows that one phase of a 16-byte load touches then differ in
// bit 2, and with the swizzle (chunk ^ row) in their banks.
__device__ __forceinline__ int key_of_column(int i) { return (i >> 1) | ((i & 1) << 2); }

// Exponent of a scale, as log2 of what weights are kept relative to.
__device__ __forceinline__ float scale_exponent(float s) {
  return fmaxf((float)((int)(__float_as_uint(s) >> 23 & 0xFF) - 127), -112.0f);
}

template <typename T, int D>
struct Smem {
  static constexpr bool kTwo = sizeof(T) == 4;             // fp32: q and weights as two halves each
  static constexpr int kQ = 16 * D * 2 * (kTwo ? 2 : 1);
  static constexpr int kMerge = kWarps * 8 * 128 * 4;      // eight rows of 128 columns of each warp
  static constexpr int kShared = kQ > kMerge ? kQ : kMerge;
  static constexpr int kRing = kWarps * kStages * kStageBytes;
  static constexpr int kBytes = kRing + kShared;
};

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 2) paged_attn_kernel(PagedParams p) {
  using S = Smem<T, D>;
  constexpr int kSub = Cfg<D>::kSub, kTile = Cfg<D>::kTile;
  constexpr int kNt = kSub / 8, kHalves = kSub / 16;
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ int64_t list_s[kWarps + 2];
  __shared__ float q_inv[kRowTile];                        // undoes the power of two that a query row was scaled by
  __shared__ float m_s[kWarps][kRowTile], l_s[kWarps][kRowTile];
  __shared__ float scale_s[kWarps][kStages][4];            // K and V scales of the stage's two halves
  __shared__ int keys_s[kWarps][kStages][2];               // keys of each half that are there
  const int tid = threadIdx.x, lane = tid & 31, warp = warp_index();
  const int cta = blockIdx.x;
  griddep_wait();
  griddep_launch();

  using Place = Cursor<kRowTile, kTile>;
  Place use;
  const auto [begin, end, share] = deal_tiles<kThreads>(p, list_s, use);
  if (tid == 0) p.cut[cta] = make_int4(0, 0, 0, 0);
  if (begin < end) {
    // ---- the ring of this warp: copies of tile `ahead` go into stage `fill`
    const uint32_t ring = smem_u32(smem) + warp * kStages * kStageBytes;
    const uint32_t shared = smem_u32(smem) + S::kRing;
    Place ahead = use;
    int64_t left = end - begin;                            // tiles still to be asked for
    int id[kHalves];
    auto look_up = [&]() {                                 // blocks of the keys of `ahead`, a tile before they are needed
      const int key = ahead.tile * kTile + warp * kSub;
#pragma unroll
      for (int h = 0; h < kHalves; ++h) {
        const int j = (key + h * 16) >> p.log_block;
        id[h] = left > 0 && key + h * 16 < ahead.q.len ? p.table[ahead.r * p.table_row + j] : -1;
      }
    };
    auto ask = [&](int stage) {
      if (left > 0) {
        const int key = ahead.tile * kTile + warp * kSub, limit = ahead.q.limit(p, ahead.row_tile);
        const uint32_t base_s = ring + stage * kStageBytes;
#pragma unroll
        for (int h = 0; h < kHalves; ++h) {
          const bool there = (unsigned)id[h] < (unsigned)p.blocks;
          const int keys = there ? min(max(limit - key - h * 16, 0), 16) : 0;
          const int64_t b = there ? id[h] : 0;
          const int64_t row = ((int64_t)ahead.head << p.log_block) + ((key + h * 16) & ((1 << p.log_block) - 1));
          const uint8_t* pk = p.k + b * p.k_block + row * D;
          const uint8_t* pv = p.v + b * p.v_block + row * D;
          if (keys > 0) {
#pragma unroll
            for (int i = 0; i < D / 32; ++i) {
              const int at = i * 32 + lane, key_in = at / (D / 16), chunk = at % (D / 16);
              const uint32_t dst = (uint32_t)(chunk >> 3) * (kSub * 128) + (uint32_t)(h * 16 + key_in) * 128 +
                                   (uint32_t)(((chunk & 7) ^ (key_in & 7)) << 4);
              const uint32_t bytes = key_in < keys ? 16 : 0;           // codes behind the last key: zeros
              cp_async_16(base_s + dst, pk + at * 16, bytes);
              cp_async_16(base_s + kStageBytes / 2 + dst, pv + at * 16, bytes);
            }
            if (lane < 2)
              cp_async_4(smem_u32(&scale_s[warp][stage][lane * 2 + h]),
                         lane == 0 ? p.ks + b * p.ks_block + ahead.head : p.vs + b * p.vs_block + ahead.head, 4);
          }
          if (lane == 0) keys_s[warp][stage][h] = keys;
        }
        if (--left > 0 && ++ahead.tile == ahead.tiles) ahead.next_unit(p);
        look_up();
      }
      cp_async_commit();
    };
    look_up();
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) ask(s);
    int stage = 0;

    // ---- segments: the tiles of one unit in this share
    const int g8 = lane >> 2, c4 = lane & 3;
    int64_t at = begin;
    bool first = true;
    while (at < end) {
      const int rows = use.q.rows(p, use.row_tile);
      const int tiles = (int)min((int64_t)(use.tiles - use.tile), end - at);
      const bool whole = use.tile == 0 && tiles == use.tiles;

      // query rows as fragments of the products: row tid / 8, elements 16 e .. 16 e + 15 for e = tid % 8 (+ 8)
      {
        const int row = tid >> 3, e0 = tid & 7;
        const int i = use.row_tile * kRowTile + row;
        const T* pq = static_cast<const T*>(p.q) + (int64_t)(use.q.t0 + i / p.g) * p.sqt +
                      (int64_t)(use.head * p.g + i % p.g) * p.sqh;
        float x[D / 128][16];
        float big = 0.0f;
#pragma unroll
        for (int u = 0; u < D / 128; ++u) {
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            x[u][k] = row < rows ? to_f32<T>(pq[(u * 8 + e0) * 16 + k]) : 0.0f;
            big = fmaxf(big, fabsf(x[u][k]));
          }
        }
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
        // largest element in [2^12, 2^13)
        const int ex = min(max((int)(__float_as_uint(big) >> 23) - 127, -110), 127);
        const float up = __uint_as_float((uint32_t)(127 + 12 - ex) << 23);
        if (e0 == 0) q_inv[row] = big == 0.0f ? 0.0f : ldexpf(1.0f, ex - 12);
        const uint32_t dst = shared + ((row & 7) * 4) * 16 + (row >> 3) * 4;
#pragma unroll
        for (int u = 0; u < D / 128; ++u) {
          const int e = u * 8 + e0;                        // 64 elements are four products; e % 4 is the lane of a group
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t a = dst + (((e >> 2) * 4 + k) * 32 + (e & 3)) * 16;
            float lo[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) lo[j] = x[u][4 * k + j] * up;
            const uint32_t w0 = pack_16x2<__half>(lo[0], lo[1]), w1 = pack_16x2<__half>(lo[2], lo[3]);
            sts_b32(a, w0);
            sts_b32(a + 8, w1);
            if constexpr (S::kTwo) {
              const float2 f0 = __half22float2(*reinterpret_cast<const __half2*>(&w0));
              const float2 f1 = __half22float2(*reinterpret_cast<const __half2*>(&w1));
              sts_b32(a + 16 * D * 2, pack_16x2<__half>(lo[0] - f0.x, lo[1] - f0.y));
              sts_b32(a + 16 * D * 2 + 8, pack_16x2<__half>(lo[2] - f1.x, lo[3] - f1.y));
            }
          }
        }
      }
      __syncthreads();
      const float inv0 = q_inv[g8] * p.scale_log2, inv1 = q_inv[g8 + 8] * p.scale_log2;
      // keys that this thread's two rows see; rows of no query see all (they are not stored)
      auto limit_of = [&](int row) {
        return row < rows ? use.q.seen(p, use.row_tile * kRowTile + row) : INT_MAX;
      };
      const int lim0 = limit_of(g8), lim1 = limit_of(g8 + 8);
      const int lim_first = use.q.seen(p, use.row_tile * kRowTile);    // the smallest of all rows

      float o[D / 16][2][4];
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int k = 0; k < 4; ++k) o[i][j][k] = 0.0f;
      float m[2] = {-INFINITY, -INFINITY}, mw[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};

      for (int tile = use.tile; tile < use.tile + tiles; ++tile) {
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
          float kscale[kHalves], vscale[kHalves];
#pragma unroll
          for (int h = 0; h < kHalves; ++h) {
            kscale[h] = keys[h] ? scale_s[warp][stage][h] : 0.0f;
            vscale[h] = keys[h] ? scale_s[warp][stage][2 + h] : 0.0f;
          }
          float s[kNt][4];
#pragma unroll
          for (int nt = 0; nt < kNt; ++nt)
#pragma unroll
            for (int k = 0; k < 4; ++k) s[nt][k] = 0.0f;
          const int krow = key_of_column(g8);
#pragma unroll
          for (int e = 0; e < D / 64; ++e) {
            uint4 a[4], a2[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              a[k] = lds128(shared + ((e * 4 + k) * 32 + lane) * 16);
              if constexpr (S::kTwo) a2[k] = lds128(shared + 16 * D * 2 + ((e * 4 + k) * 32 + lane) * 16);
            }
#pragma unroll
            for (int nt = 0; nt < kNt; ++nt) {
              // half a stage's keys may be stale where a block is missing: they are masked below
              const uint4 b = lds128(base_s + (e >> 1) * (kSub * 128) + (nt * 8 + krow) * 128 +
                                     ((((e & 1) * 4 + c4) ^ krow) << 4));
              const uint32_t w[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                uint32_t b0, b1;
                half4_of_e4m3x4(w[k], b0, b1);
                mma_16816(s[nt], a[k], b0, b1);
                if constexpr (S::kTwo) mma_16816(s[nt], a2[k], b0, b1);
              }
            }
          }
          float big[2] = {-INFINITY, -INFINITY};
          const bool masks = !all || key + kSub > lim_first;
#pragma unroll
          for (int nt = 0; nt < kNt; ++nt) {
            const int h = nt >> 1;
            s[nt][0] *= inv0 * kscale[h];
            s[nt][1] *= inv0 * kscale[h];
            s[nt][2] *= inv1 * kscale[h];
            s[nt][3] *= inv1 * kscale[h];
            if (masks) {
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const int in = (nt & 1) * 8 + c4 + (k & 1) * 4;          // key within its half
                if (in >= keys[h] || key + h * 16 + in >= (k < 2 ? lim0 : lim1)) s[nt][k] = -INFINITY;
              }
            }
            big[0] = fmaxf(big[0], fmaxf(s[nt][0], s[nt][1]));
            big[1] = fmaxf(big[1], fmaxf(s[nt][2], s[nt][3]));
          }
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            big[i] = fmaxf(big[i], __shfl_xor_sync(0xffffffffu, big[i], 1));
            big[i] = fmaxf(big[i], __shfl_xor_sync(0xffffffffu, big[i], 2));
          }
          float vexp = -112.0f;
#pragma unroll
          for (int h = 0; h < kHalves; ++h) vexp = keys[h] ? fmaxf(vexp, scale_exponent(vscale[h])) : vexp;
          float m_new[2], shrink_o[2], c[2][kHalves];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            m_new[i] = fmaxf(m[i], big[i]);
            const float w_new = fmaxf(mw[i], big[i] + vexp);
            const bool none = m_new[i] == -INFINITY;
            const float ref = none ? 0.0f : m_new[i];
            l[i] *= ex2(m[i] - ref);
            shrink_o[i] = none ? 1.0f : ex2(mw[i] - w_new);
            const float f = none ? 0.0f : ex2(fminf(ref - w_new + 14.0f, 126.0f));
#pragma unroll
            for (int h = 0; h < kHalves; ++h) c[i][h] = f * vscale[h];
            m[i] = m_new[i];
            mw[i] = w_new;
            m_new[i] = ref;
          }
          if (__any_sync(0xffffffffu, shrink_o[0] != 1.0f || shrink_o[1] != 1.0f)) {
#pragma unroll
            for (int i = 0; i < D / 16; ++i)
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                o[i][j][0] *= shrink_o[0];
                o[i][j][1] *= shrink_o[0];
                o[i][j][2] *= shrink_o[1];
                o[i][j][3] *= shrink_o[1];
              }
          }
          uint4 pw[kHalves], pw2[kHalves];
#pragma unroll
          for (int h = 0; h < kHalves; ++h) {
            uint32_t w[4], w2[4];
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
              for (int n = 0; n < 2; ++n) {
                const float p0 = ex2(s[2 * h + n][2 * i] - m_new[i]), p1 = ex2(s[2 * h + n][2 * i + 1] - m_new[i]);
                l[i] += p0 + p1;
                const float x0 = p0 * c[i][h], x1 = p1 * c[i][h];
                w[n * 2 + i] = pack_16x2<__half>(x0, x1);
                if constexpr (S::kTwo) {
                  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[n * 2 + i]));
                  w2[n * 2 + i] = pack_16x2<__half>(x0 - f.x, x1 - f.y);
                }
              }
            pw[h] = make_uint4(w[0], w[1], w[2], w[3]);
            if constexpr (S::kTwo) pw2[h] = make_uint4(w2[0], w2[1], w2[2], w2[3]);
          }
#pragma unroll
          for (int h = 0; h < kHalves; ++h) {
            if (keys[h] == 0) continue;                    // nothing was copied: stale codes may be NaN
            const int vrow = h * 16 + ((lane >> 3) & 1) * 8 + key_of_column(lane & 7);
#pragma unroll
            for (int dg = 0; dg < D / 32; ++dg) {
              const int chunk = dg * 2 + (lane >> 4);
              uint32_t r[4];
              ldmatrix_x4_t(base_s + kStageBytes / 2 + (chunk >> 3) * (kSub * 128) + vrow * 128 +
                                (((chunk & 7) ^ (vrow & 7)) << 4),
                            r);
#pragma unroll
              for (int ch = 0; ch < 2; ++ch) {
                // bytes (d, d + 1) of two keys -> the keys of d, the keys of d + 1
                uint32_t e0, o0, e1, o1;
                half4_of_e4m3x4(__byte_perm(r[2 * ch], 0, 0x3120), e0, o0);
                half4_of_e4m3x4(__byte_perm(r[2 * ch + 1], 0, 0x3120), e1, o1);
                mma_16816(o[dg * 2 + ch][0], pw[h], e0, e1);
                mma_16816(o[dg * 2 + ch][1], pw[h], o0, o1);
                if constexpr (S::kTwo) {
                  mma_16816(o[dg * 2 + ch][0], pw2[h], e0, e1);
                  mma_16816(o[dg * 2 + ch][1], pw2[h], o0, o1);
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
      for (int i = 0; i < 2; ++i) {
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
        if (c4 == 0) {
          m_s[warp][g8 + 8 * i] = m[i];
          l_s[warp][g8 + 8 * i] = l[i];
        }
      }
      __syncthreads();                                     // and nobody needs the query fragments any more
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int row = g8 + 8 * i;
        float top = m_s[0][row];
#pragma unroll
        for (int w = 1; w < kWarps; ++w) top = fmaxf(top, m_s[w][row]);
        // weights carry 2^(14 - mw); brought to 2^-top
        const float f = mw[i] == -INFINITY ? 0.0f : ex2(mw[i] - top) * 0x1p-14f;
#pragma unroll
        for (int a = 0; a < D / 16; ++a)
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            o[a][b][2 * i] *= f;
            o[a][b][2 * i + 1] *= f;
          }
      }
      const int slot = first ? 2 * cta : 2 * cta + 1;
#pragma unroll
      for (int pass = 0; pass < 2 * (D / 128); ++pass) {
        const int half = pass % 2, cols = pass / 2;        // rows 8 half .., columns 128 cols ..
        if (half * 8 < rows) {
#pragma unroll
          for (int a = 0; a < 8; ++a) {
            const float* x0 = o[cols * 8 + a][0] + 2 * half;
            const float* x1 = o[cols * 8 + a][1] + 2 * half;
            const uint32_t dst = shared + ((warp * 8 + g8) * 128 + ((a ^ (g8 & 1)) * 16) + 4 * c4) * 4;
            asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "f"(x0[0]), "f"(x1[0]), "f"(x0[1]), "f"(x1[1])
                         : "memory");
          }
          __syncthreads();
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const int in = warp * 2 + y, row = half * 8 + in;
            if (row < rows) {
              float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f}, top = m_s[0][row], total_l = 0.0f;
#pragma unroll
              for (int w = 1; w < kWarps; ++w) top = fmaxf(top, m_s[w][row]);
#pragma unroll
              for (int w = 0; w < kWarps; ++w) {
                const uint4 v = lds128(shared + ((w * 8 + in) * 128 + (((lane >> 2) ^ (in & 1)) * 16) + 4 * (lane & 3)) * 4);
                sum[0] += __uint_as_float(v.x);
                sum[1] += __uint_as_float(v.y);
                sum[2] += __uint_as_float(v.z);
                sum[3] += __uint_as_float(v.w);
                total_l += top == -INFINITY ? l_s[w][row] : l_s[w][row] * ex2(m_s[w][row] - top);   // no key: 0, or NaN
              }
              if (whole) {
                const float inv = total_l == 0.0f ? 0.0f : 1.0f / total_l;
                const int64_t to = out_row(p, (int64_t)use.q.t0 * p.g + use.row_tile * kRowTile + row, use.head);
#pragma unroll
                for (int k = 0; k < 4; ++k) sum[k] *= inv;
                store4<T>(static_cast<T*>(p.out) + to * D + cols * 128 + lane * 4, sum);
                if (cols == 0 && lane == 0 && p.lse != nullptr)
                  p.lse[to] = lse_of(top, total_l);
              } else {
                store4<float>(p.ws_acc + ((int64_t)slot * kRowTile + row) * D + cols * 128 + lane * 4, sum);
                if (cols == 0 && lane == 0) {
                  p.ws_m[slot * kRowTile + row] = top;
                  p.ws_l[slot * kRowTile + row] = total_l;
                }
              }
            }
          }
          __syncthreads();
        }
      }
      if (!whole && use.tile == 0 && tid == 0) {
        // begun here, finished by the CTAs behind this one
        p.cut[cta] = cut_unit(p, use, tiles, share, first);
      }
      at += tiles;
      first = false;
      if (at < end) use.next_unit(p);
    }
  }
  clear_untouched<T, D, kRowTile, kTile>(p);
}

template <typename T, int D>
int run_attention(const PagedParams& p, int grid, cudaStream_t st) {
  using S = Smem<T, D>;
  if (int rc = allow_smem("nvfp4_kv8_attention", reinterpret_cast<const void*>(paged_attn_kernel<T, D>), S::kBytes)) return rc;
  if (int rc = launch("nvfp4_kv8_attention", paged_attn_kernel<T, D>, dim3(grid), kThreads, S::kBytes, st, p)) return rc;
  return launch_combine<T, D, kRowTile>(p, grid, st);
}

// Which kernel: tensor-memory products take 128 or 256 rows at a time and are worth it from kChunkRows query rows a request
// on, on average (the lengths themselves are on the device); fp32 queries, whose products need two halves, stay here.
constexpr int kChunkRows = 32;
bool takes_chunk_kernel(int q_dtype, int64_t tokens, int64_t requests, int64_t g) {
  return q_dtype != NVFP4_DT_FP32 && tokens * g > kChunkRows * requests;
}

}  // namespace
}  // namespace nvfp4

using namespace nvfp4;

extern "C" int nvfp4_kv8_attention_plan(int q_dtype, int64_t tokens, int64_t requests, int g, int d, int sm_count,
                                        size_t* workspace_bytes) {
  NVFP4_REQUIRE(d == 128 || d == 256, "nvfp4_kv8_attention_plan: D must be 128 or 256");
  NVFP4_REQUIRE(tokens >= 0 && requests >= 1 && g >= 1 && sm_count >= 1 && workspace_bytes != nullptr,
                "nvfp4_kv8_attention_plan: bad argument");
  *workspace_bytes = (size_t)(takes_chunk_kernel(q_dtype, tokens, requests, g) ? sm_count * paged_slot_bytes(paged_chunk_rows(d), d)
                                                                               : 2 * sm_count * paged_slot_bytes(kRowTile, d));
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
  NVFP4_REQUIRE((((uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)out | (uintptr_t)workspace) & 15) == 0 &&
                    ((k_block | v_block) & 15) == 0,
                "nvfp4_kv8_attention: cache blocks, out and workspace must be 16-byte aligned");
  if (tokens == 0) return 0;
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  const bool chunk = takes_chunk_kernel(q_dtype, tokens, requests, g);
  const int grid = chunk ? sms : 2 * sms;
  const int64_t rows = chunk ? paged_chunk_rows(d) : kRowTile;
  NVFP4_REQUIRE(workspace_bytes >= (size_t)(grid * paged_slot_bytes(rows, d)), "nvfp4_kv8_attention: workspace too small");
  NVFP4_REQUIRE(q_dtype >= NVFP4_DT_BF16 && q_dtype <= NVFP4_DT_FP32, "nvfp4_kv8_attention: unknown dtype %d", q_dtype);
  PagedParams p{q, s_qt, s_qh, cu_seqlens, tokens, k_cache, v_cache, k_block, v_block, k_scale, v_scale, ks_block, vs_block, table,
                table_row, lengths, (int)requests, (int)width, (int)blocks, lb, (int)hk, g, scaling * kLog2e, out, lse,
                nullptr, nullptr, nullptr, nullptr, status};
  p.ws_acc = static_cast<float*>(workspace);
  p.cut = reinterpret_cast<int4*>(p.ws_acc + 2 * grid * rows * d);
  p.ws_m = reinterpret_cast<float*>(p.cut + grid);
  p.ws_l = p.ws_m + 2 * grid * rows;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (chunk) return launch_paged_chunk(p, q_dtype, d, grid, st);
  switch (q_dtype) {
    case NVFP4_DT_BF16: return d == 128 ? run_attention<__nv_bfloat16, 128>(p, grid, st) : run_attention<__nv_bfloat16, 256>(p, grid, st);
    case NVFP4_DT_FP16: return d == 128 ? run_attention<__half, 128>(p, grid, st) : run_attention<__half, 256>(p, grid, st);
    default: return d == 128 ? run_attention<float, 128>(p, grid, st) : run_attention<float, 256>(p, grid, st);
  }
}
