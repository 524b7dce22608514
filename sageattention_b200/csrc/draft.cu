// Trees of drafted tokens: what every node sees and where it stands, and which of them the target's probabilities keep.
//
// A request's tokens cu[r] .. cu[r + 1] are a tree: its node 0 is the token that the step before ended with, node i hangs on the
// earlier node that parents[] names.  Nodes from max_tokens (1024 at most) on are not part of it: they see none of it, and none is kept.
#include <limits.h>
#include "common/abi.cuh"
#include "common/fp4.cuh"
#include "common/launch.cuh"
#include "common/sm100.cuh"

namespace nvfp4 {
namespace {

constexpr int kTree = 1024;                    // nodes of a tree
constexpr int kPasses = 1 << 30;               // flag of a node that passes its test

// Tokens [t0, t0 + n) of request r, whatever cu holds within the call's tokens.
struct Span {
  int64_t t0;
  int64_t n;
  __device__ __forceinline__ Span(const int32_t* cu, int r, int64_t tokens) {
    t0 = min(max((int64_t)cu[r], (int64_t)0), tokens);
    n = max(min((int64_t)cu[r + 1], tokens) - t0, (int64_t)0);
  }
};
// Tokens in front of the first request and behind the last one, over all blocks of the grid.
template <typename F>
__device__ __forceinline__ void outside(const int32_t* cu, int requests, int64_t tokens, F clear) {
  const int64_t front = min(max((int64_t)cu[0], (int64_t)0), tokens), behind = min(max((int64_t)cu[requests], (int64_t)0), tokens);
  const int64_t at = ((int64_t)blockIdx.z * gridDim.x + blockIdx.x) * blockDim.x + threadIdx.x;
  const int64_t step = (int64_t)gridDim.x * gridDim.z * blockDim.x;
  for (int64_t t = at; t < front; t += step) clear(t);
  for (int64_t t = behind + at; t < tokens; t += step) clear(t);
}

// ------------------------------------------------------------------------------------------ tables
struct TreeParams {
  const int32_t *parents, *cu, *lengths;
  int64_t tokens;
  int requests, most, words;
  uint64_t* mask;
  int32_t* positions;
};

// A block of threads a request, a thread a node: up the tree through shared memory, in whose order the bits' words come.
// Bound by its trips to memory, one behind the other (cu, parents, results).
constexpr int kTreeThreads = 128;
__global__ void __launch_bounds__(kTreeThreads) draft_tree_kernel(TreeParams p) {
  __shared__ int16_t up[kTree];
  griddep_wait();
  griddep_launch();
  const int r = blockIdx.x;
  const Span s(p.cu, r, p.tokens);
  const int m = (int)min(s.n, (int64_t)p.most);
  const int64_t context = (int64_t)p.lengths[r] - s.n;
  for (int i = threadIdx.x; i < m; i += kTreeThreads) {
    const int a = p.parents[s.t0 + i];
    up[i] = (int16_t)(a >= 0 && a < i ? a : -1);
  }
  __syncthreads();
  for (int64_t i = threadIdx.x; i < s.n; i += kTreeThreads) {
    uint64_t* row = p.mask + (s.t0 + i) * p.words;
    int depth = 0;
    if (i < m) {
      int word = (int)i >> 6;
      for (int w = p.words - 1; w > word; --w) row[w] = 0;
      uint64_t bits = 0;
      for (int node = (int)i;;) {
        bits |= 1ull << (node & 63);
        node = up[node];
        if (node < 0) break;
        ++depth;
        while (word > node >> 6) {
          row[word--] = bits;
          bits = 0;
        }
      }
      for (; word >= 0; --word, bits = 0) row[word] = bits;
    } else {
      for (int w = 0; w < p.words; ++w) row[w] = 0;
    }
    p.positions[s.t0 + i] = (int32_t)max(context + depth, (int64_t)0);
  }
  outside(p.cu, p.requests, p.tokens, [&](int64_t t) {
    for (int w = 0; w < p.words; ++w) p.mask[t * p.words + w] = 0;
    p.positions[t] = 0;
  });
}

// ------------------------------------------------------------------------------------------ verification
struct VerifyParams {
  const void *p, *q;                           // rows of the target and (or null) of the draft
  int64_t sp, sq;                              // element strides of their rows
  const void* ids;
  int ids64;
  const int32_t *parents, *cu;
  const float* u;
  int64_t tokens;
  int requests, vocab, most;                   // most: nodes of a tree that may be kept
  int32_t *accepted, *count;
  int64_t* next;
};

// Threads of a block, two of which share an SM: with draft rows 128 registers a thread, in 64 of which (512 threads) they do not
// fit; without them more warps.  Chains of 32000 tokens 8.5 (13.4) us, the likeliest of 131072 tokens 18.6 (21.2).  Chosen drafts of 16-bit
// rows, eight elements a load, spill 84 bytes in 64 registers: 131072 tokens in bf16 17.4 us where fp32 takes 18.0.
__host__ __device__ constexpr int verify_threads(bool drawn) { return drawn ? 256 : 512; }

__device__ __forceinline__ double ld_cluster_f64(uint32_t saddr, uint32_t rank) {
  uint32_t a;
  double v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(saddr), "r"(rank));
  asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(a) : "memory");
  return v;
}

// A probability as it counts: what is no finite number above zero is none.
template <typename T>
__device__ __forceinline__ float mass_of(T v) {
  const float f = to_f32<T>(v);
  return f > 0.0f && f < INFINITY ? f : 0.0f;
}

// The walk down a request's tree.  At node x with the target's row p and children c_1, c_2, ... in order, R_0 = p, M_0 = 1:
//   with draft rows q:  c_j passes where u q(c_j) M < R(c_j); else R <- max(R / M - q, 0), M <- sum R
//   without:            c_j passes where u M < R(c_j); else M <- M - R(c_j), R(c_j) <- 0
// The first that passes is the next node; where none does, the next token is drawn from R: the first v with R(0) + .. + R(v) above
// w sum R, w the number of node 0.  All of it in 64 bits: a vocabulary's sums in 32 would move the draw by whole tokens.
//
// A cluster a request; every block walks for itself over values that all have fetched (a node's p and q at its token, one
// trip for all nodes).  Without draft rows all nodes are tested at once, as a test depends on a node's siblings alone, and the
// walk follows the first that pass; with them a rejection needs the sum of a row.  The blocks of the cluster share a row, a
// warp a piece of it.  What bounds it: the rows (one a rejection, one for the draw) where there are many requests, else the trips
// to memory and between the blocks, one behind the other.
template <typename T, bool kDrawn>
__global__ void __launch_bounds__(verify_threads(kDrawn), 2) verify_drafts_kernel(VerifyParams p) {
  constexpr int kThreads = verify_threads(kDrawn), kWarps = kThreads / 32;
  constexpr int kPer = 16 / sizeof(T);
  constexpr int kStep = 32 * kPer;             // elements of a warp's load
  constexpr int kAhead = 4;                    // loads of a lane under way together, of the draft's row as many again
  __shared__ int16_t up_s[kTree], path_s[kTree];
  __shared__ int32_t id_s[kTree];
  __shared__ float px_s[kTree], u_s[kTree];
  __shared__ float qx_s[kDrawn ? kTree : 1];
  // drawn: first child of a node, next one of its parent; else first child that passes, rejected ones of the path's last node
  __shared__ int first_s[kTree];
  __shared__ int16_t next_s[kTree];
  __shared__ double over_s[kDrawn ? kTree : 1];            // one over what was left behind j rejections
  __shared__ double block_s[2], warp_s[kWarps];
  __shared__ int node_s, k_s, len_s;
  __shared__ bool done_s;
  const int tid = threadIdx.x, lane = tid & 31, warp = warp_index();
  const int rank = blockIdx.z, ranks = gridDim.z, r = blockIdx.x;
  griddep_wait();
  griddep_launch();
  const Span span(p.cu, r, p.tokens);
  const int n = (int)min(span.n, (int64_t)p.most);
  const T* const target = static_cast<const T*>(p.p);
  const T* const draft = static_cast<const T*>(p.q);
  for (int i = tid; i < n; i += kThreads) {
    const int64_t t = span.t0 + i;
    const int a = p.parents[t];
    const int64_t id = p.ids64 ? static_cast<const int64_t*>(p.ids)[t] : (int64_t) static_cast<const int32_t*>(p.ids)[t];
    const bool child = a >= 0 && a < i, known = id >= 0 && id < p.vocab;
    float x = 0.0f, y = 0.0f;
    if (child && known) {
      x = mass_of<T>(target[(span.t0 + a) * p.sp + id]);
      if (kDrawn) y = mass_of<T>(draft[(span.t0 + a) * p.sq + id]);
    }
    up_s[i] = (int16_t)(child ? a : -1);
    id_s[i] = known ? (int32_t)id : -1;
    u_s[i] = p.u[t];
    px_s[i] = x;
    if (kDrawn) qx_s[i] = y;
    first_s[i] = kTree;
    next_s[i] = kTree;
  }
  if (tid == 0) {
    k_s = 0;
    path_s[0] = 0;
  }
  __syncthreads();
  // Where a node stands among its siblings.  A token again among them is worth nothing.
  // Of up to 32 nodes a warp knows it by itself.  Chosen, instead of the search below: 64 requests of 26 nodes over 131072 tokens 18.0 us (18.9), over
  // 32000 10.0 (11.2), 256 of 32 16.4 (17.8), one of 16 9.2 (10.0), a chain of eight 7.0 (7.1); drawn, whose search does less, it is as
  // fast: 64 of 20 30.6 (30.8), 16 of 32 23.5 (23.7), chains of six 10.5 (10.4).
  if (n <= 32) {
    if (warp == 0) {
      const int up = lane < n ? up_s[lane] : -1;
      const uint32_t in_front = (1u << lane) - 1, siblings = __match_any_sync(0xffffffffu, up >= 0 ? up : kTree + lane);
      if (kDrawn) {
        const uint32_t before = siblings & in_front;
        if (up >= 0) {
          if (before == 0) first_s[up] = (double)u_s[lane] * (double)qx_s[lane] < (double)px_s[lane] ? lane | kPasses : lane;
          else next_s[31 - __clz(before)] = (int16_t)lane;
        }
      } else {
        const int id = lane < n ? id_s[lane] : -1;
        const bool again = (__match_any_sync(0xffffffffu, id) & siblings & in_front) != 0;
        const float x = up >= 0 && !again ? px_s[lane] : 0.0f;
        double mass = 1.0;
        for (uint32_t m = siblings & in_front; __any_sync(0xffffffffu, m != 0); m &= m - 1) {
          const float other = __shfl_sync(0xffffffffu, x, m != 0 ? __ffs(m) - 1 : lane);
          if (m != 0) mass = fmax(mass - (double)other, 0.0);
        }
        const bool passes = up >= 0 && (double)u_s[lane] * mass < (double)x;
        const uint32_t all = __ballot_sync(0xffffffffu, passes) & siblings;
        if (passes && __ffs(all) - 1 == lane) first_s[up] = lane;
      }
    }
    __syncthreads();
  } else {
    if (!kDrawn) {
      uint32_t again = 0;                      // of this thread's nodes, a bit each
      for (int i = tid, bit = 0; i < n; i += kThreads, ++bit)
        if (up_s[i] >= 0)
#pragma unroll 4
          for (int j = up_s[i] + 1; j < i; ++j)
            if (up_s[j] == up_s[i] && id_s[j] == id_s[i]) again |= 1u << bit;
      __syncthreads();
      for (int i = tid, bit = 0; i < n; i += kThreads, ++bit)
        if (again >> bit & 1) px_s[i] = 0.0f;
      __syncthreads();
    }
    for (int i = tid; i < n; i += kThreads) {
      const int up = up_s[i];
      if (up < 0) continue;
      int before = -1;
      double mass = 1.0;
#pragma unroll 4
      for (int j = up + 1; j < i; ++j)
        if (up_s[j] == up) {
          before = j;
          if (!kDrawn) mass = fmax(mass - (double)px_s[j], 0.0);
        }
      if (kDrawn) {
        // the first child of a node that has lost none yet: at once known, and marked where it passes
        if (before < 0) first_s[up] = (double)u_s[i] * (double)qx_s[i] < (double)px_s[i] ? i | kPasses : i;
        else next_s[before] = (int16_t)i;
      } else if ((double)u_s[i] * mass < (double)px_s[i]) {
        atomicMin(&first_s[up], i);
      }
    }
    __syncthreads();
  }

  // what is left of a probability behind k rejections, one at least
  auto left_of = [&](float x, float q, int k) -> double {
    double r = x > q ? (double)x - (double)q : 0.0;        // mass 0 is 1
    for (int j = 1; j < k; ++j) {
      r = r * over_s[j] - q;
      if (!(r > 0.0)) r = 0.0;
    }
    return r;
  };

  // ---- a row: places are elements behind the 16 bytes that it begins in
  const T *row = nullptr, *row_q = nullptr;
  int head = 0, end_row = 0;                   // its places
  bool same = true;                            // the draft's row begins as the target's does, else it is read one by one
  int struck = -1;                             // chosen: place of this lane's rejected token, of the first 32
  auto open_row = [&](int node, int k) {
    row = target + (span.t0 + node) * p.sp;
    head = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
    end_row = head + p.vocab;
    row -= head;                               // at 16 bytes; places in front of `head` are never read
    if (kDrawn) {
      const T* q = draft + (span.t0 + node) * p.sq;
      same = (int)((reinterpret_cast<uintptr_t>(q) & 15) / sizeof(T)) == head;
      row_q = q - head;
    } else {
      struck = lane < k && id_s[next_s[lane]] >= 0 ? id_s[next_s[lane]] + head : -1;
    }
  };
  // Chosen: whether rejected tokens lie in places begin .. end; all lanes of the warp.
  auto touched = [&](int begin, int end, int k) {
    bool hit = struck >= begin && struck < end;
    for (int j = 32 + lane; j < k; j += 32) {
      const int id = id_s[next_s[j]];
      hit |= id >= 0 && id + head >= begin && id + head < end;
    }
    return __any_sync(0xffffffffu, hit);
  };
  // what is left of a lane's elements x (and y) of the step at `base` behind k rejections; all lanes of the warp
  auto rest = [&](int base, const uint4& raw, const uint4& raw_q, int k, bool hit, double (&left)[kPer]) {
    const T *x = reinterpret_cast<const T*>(&raw), *y = reinterpret_cast<const T*>(&raw_q);
    if (!kDrawn || k == 0) {
#pragma unroll
      for (int e = 0; e < kPer; ++e) left[e] = mass_of<T>(x[e]);
    } else {
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        const float a = mass_of<T>(x[e]), b = mass_of<T>(y[e]);
        left[e] = a > b ? (double)a - (double)b : 0.0;
      }
#pragma unroll 1
      for (int j = 1; j < k; ++j) {
        const double over = over_s[j];
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
          const double t = left[e] * over - (double)mass_of<T>(y[e]);
          left[e] = t > 0.0 ? t : 0.0;
        }
      }
    }
    if (!kDrawn && hit) {
      const int at = base + lane * kPer;
      auto strike = [&](int place) {
        for (uint32_t m = __ballot_sync(0xffffffffu, place >= base && place < base + kStep); m != 0; m &= m - 1) {
          const int one = __shfl_sync(0xffffffffu, place, __ffs(m) - 1) - at;
#pragma unroll
          for (int e = 0; e < kPer; ++e)
            if (one == e) left[e] = 0.0;
        }
      };
      strike(struck);
#pragma unroll 1
      for (int j = 32 + lane; j - lane < k; j += 32) strike(j < k && id_s[next_s[j]] >= 0 ? id_s[next_s[j]] + head : -1);
    }
  };
  // a lane's elements at place `at` .. (of the row, or of the draft's in its place) where 16 bytes are not all the row's: one by one
  auto edge = [&](const T* from, int at, uint4& x) {
    T* one = reinterpret_cast<T*>(&x);
#pragma unroll
    for (int e = 0; e < kPer; ++e) one[e] = at + e >= head && at + e < end_row ? from[at + e] : from_f32<T>(0.0f);
  };
  // sum of places begin .. end by a warp, in all its lanes; begin is a multiple of kStep
  auto piece_sum = [&](int begin, int end, int k) {
    const bool both = kDrawn && k > 0, hit = !kDrawn && touched(begin, end, k);
    double sum = 0.0;
#pragma unroll 1
    for (int base = begin; base < end; base += kAhead * kStep) {
      uint4 x[kAhead], y[kAhead];
      const int at = base + lane * kPer;
      auto full = [&](int at) { return at >= head && at + kPer <= end_row; };
#pragma unroll
      for (int a = 0; a < kAhead; ++a) x[a] = load_or_zero(row + at + a * kStep, full(at + a * kStep) && at + a * kStep < end);
      if (both) {
#pragma unroll
        for (int a = 0; a < kAhead; ++a) y[a] = load_or_zero(row_q + at + a * kStep, same && full(at + a * kStep) && at + a * kStep < end);
      }
      const bool inside = base >= head && base + kAhead * kStep <= end_row;
#pragma unroll
      for (int a = 0; a < kAhead; ++a) {
        const int to = at + a * kStep;
        if (base + a * kStep >= end) break;
        if (!inside && !full(to)) edge(row, to, x[a]);
        if (both && (!same || (!inside && !full(to)))) edge(row_q, to, y[a]);
        double left[kPer];
        rest(base + a * kStep, x[a], y[a], k, hit, left);
#pragma unroll
        for (int w = 1; w < kPer; w *= 2)
#pragma unroll
          for (int e = 0; e < kPer; e += 2 * w) left[e] += left[e + w];
        sum += left[0];
      }
    }
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
    return sum;
  };
  // sums over the lanes up to this one
  auto running = [&](double x) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    return x;
  };
  // first of the lanes' values whose running sum exceeds `at`, or the last above zero, or -1; `at` becomes relative to it
  auto pick = [&](double x, double& at) -> int {
    const double upto = running(x);
    const uint32_t some = __ballot_sync(0xffffffffu, x > 0.0), above = __ballot_sync(0xffffffffu, x > 0.0 && upto > at);
    const int who = above ? __ffs(above) - 1 : 31 - __clz(some);
    if (who >= 0) at -= __shfl_sync(0xffffffffu, upto - x, who);
    return who;
  };
  auto of_warps = [&]() { return lane < kWarps ? warp_s[lane] : 0.0; };
  double of_blocks = 0.0;                      // this lane's block of the cluster: its sum of the row
  int turn = 0;
  if (n > 0) {
    // thread 0 (drawn): on from node, behind `child`, which was rejected, until a row's sum is wanted or no child is left
    int node = 0, len = 1, child = kTree;
    int k = 0;                                 // rejections at the path's last node
    double sum = 0.0;
    int summed = -1, summed_k = 0;             // whose sum it is
    enum { kWalk, kWhole, kDraw } stage = kWalk;
    // the draw: its place within what is left, and the places begin .. end that it has been narrowed down to, `whole` of them
    double at = 0.0;
    int begin = 0, end = 0, whole = 0;
    bool mine = true;                          // this block has them
    // One loop, so that what goes through a row is there once: a kernel that runs its code a few times is as fast as that comes
    // from memory (three copies of it, the last one's four steps unrolled: chains 23.7 us).
#pragma unroll 1
    for (;;) {
      if (stage == kWalk) {
        if (tid == 0) {
          if (!kDrawn) {
            for (int c; (c = first_s[node]) < kTree; node = c) path_s[len++] = (int16_t)c;
          } else {
            // `child` has been rejected k - 1 times over: its next one is tested against what is left
            bool passes = false;
            if (k > 0) {
              child = next_s[child];
              passes = child < kTree && (double)u_s[child] * (double)qx_s[child] * sum < left_of(px_s[child], qx_s[child], k);
            }
            if (k == 0 || passes) {
              if (passes) {
                path_s[len++] = (int16_t)child;
                node = child;
                k = 0;
              }
              while ((child = first_s[node]) & kPasses) path_s[len++] = (int16_t)(node = child & ~kPasses);
            }
            done_s = child >= kTree;
            if (child < kTree) {
              if (k > 0) over_s[k] = sum > 0.0 ? 1.0 / sum : 0.0;
              ++k;
            }
            k_s = k;
          }
          node_s = node;
          len_s = len;
        }
        __syncthreads();
        const int last = node_s;
        if (!kDrawn) {
          for (int i = tid; i < n; i += kThreads)
            if (up_s[i] == last) next_s[atomicAdd(&k_s, 1)] = (int16_t)i;      // in any order
          __syncthreads();
        }
        k = k_s;
        if (!kDrawn || done_s) {
          const bool known = summed == last && summed_k == k;
          stage = known && sum > 0.0 ? kDraw : kWhole;
          if (known && stage == kWhole) k = 0;             // nothing is left: from the row itself
        }
        if (stage != kDraw) open_row(last, k);
        summed = last;
        summed_k = k;
      }
      const bool parts = stage == kDraw && whole != 0;     // of a piece, else pieces of the row
      if (stage != kDraw || parts) {
        const int size = parts ? (whole / kWarps + kStep - 1) / kStep * kStep
                               : ((end_row + kWarps * ranks - 1) / (kWarps * ranks) + kStep - 1) / kStep * kStep;
        const int b = parts ? begin + warp * size : (rank * kWarps + warp) * size;
        const double x = piece_sum(b, min(b + size, parts ? end : end_row), k);
        if (parts) __syncthreads();                        // the sums before have been read
        if (lane == 0) warp_s[warp] = x;
        __syncthreads();
        if (!parts) {
          turn ^= 1;
          double t = of_warps();
#pragma unroll
          for (int m = 16; m > 0; m >>= 1) t += __shfl_xor_sync(0xffffffffu, t, m);
          of_blocks = lane == 0 ? t : 0.0;
          if (ranks > 1) {
            if (tid == 0) block_s[turn] = t;
            cluster_sync_all();
            of_blocks = lane < ranks ? ld_cluster_f64(smem_u32(&block_s[turn]), lane) : 0.0;
            t = of_blocks;
#pragma unroll
            for (int m = 4; m > 0; m >>= 1) t += __shfl_xor_sync(0xffffffffu, t, m);
            t = __shfl_sync(0xffffffffu, t, 0);
          }
          sum = t;
          if (stage == kWalk) continue;
          if (!(sum > 0.0) && k > 0) {                     // nothing is left: from the row itself
            k = 0;
            struck = -1;
            __syncthreads();
            continue;
          }
          stage = kDraw;
        } else {
          begin += max(pick(of_warps(), at), 0) * size;
          end = min(begin + size, end);
          whole = size;
        }
      }
      if (whole == 0) {                                    // the cluster's block, its warp's piece
        at = (double)u_s[0] * sum;
        const int owner = pick(of_blocks, at);
        if (owner < 0 && rank == 0 && tid == 0) p.next[r] = 0;                 // a row of zeros
        mine = owner == rank;
        if (!mine) break;
        whole = ((end_row + kWarps * ranks - 1) / (kWarps * ranks) + kStep - 1) / kStep * kStep;
        begin = (rank * kWarps + max(pick(of_warps(), at), 0)) * whole;
        end = min(begin + whole, end_row);
      }
      if (whole == kStep) break;
    }
    if (mine && warp == 0) {                               // a warp's load of places: which one
      const bool both = kDrawn && k > 0;
      const int to = begin + lane * kPer;
      const bool full = to >= head && to + kPer <= end_row;
      uint4 x = load_or_zero(row + to, full && to < end), y = load_or_zero(row_q + to, both && same && full && to < end);
      if (!full && to < end) edge(row, to, x);
      if (both && to < end && (!same || !full)) edge(row_q, to, y);
      double left[kPer], own = 0.0;
      rest(begin, x, y, k, !kDrawn, left);
#pragma unroll
      for (int e = 0; e < kPer; ++e) own += left[e];
      double run = running(own) - own;
      int first = INT_MAX, last = 0;
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        run += left[e];
        if (left[e] > 0.0) {
          if (run > at) first = min(first, to + e);
          last = max(last, to + e);
        }
      }
      first = __reduce_min_sync(0xffffffffu, first);
      last = __reduce_max_sync(0xffffffffu, last);
      if (lane == 0) p.next[r] = max((first < INT_MAX ? first : last) - head, 0);
    }
    if (rank == 0) {
      const int kept = len_s;
      for (int64_t i = tid; i < span.n; i += kThreads) p.accepted[span.t0 + i] = i < kept ? path_s[i] : -1;
      if (tid == 0) p.count[r] = kept;
    }
  } else if (rank == 0 && tid == 0) {
    p.count[r] = 0;
    p.next[r] = -1;
  }
  outside(p.cu, p.requests, p.tokens, [&](int64_t t) { p.accepted[t] = -1; });
  if (ranks > 1) cluster_sync_all();           // another block may still read this one's sum
}

template <typename T>
int run_verify(const VerifyParams& p, int ranks, cudaStream_t st) {
  const auto kern = p.q != nullptr ? verify_drafts_kernel<T, true> : verify_drafts_kernel<T, false>;
  return launch_cluster("nvfp4_verify_drafts", kern, dim3((unsigned)p.requests, 1, (unsigned)ranks), (unsigned)ranks,
                        verify_threads(p.q != nullptr), 0, st, p);
}

}  // namespace
}  // namespace nvfp4

using namespace nvfp4;

extern "C" int nvfp4_draft_tree(const int32_t* parents, const int32_t* cu_seqlens, const int32_t* lengths, int64_t tokens, int64_t requests,
                                int64_t max_tokens, uint64_t* mask, int32_t* positions, nvfp4_stream_t stream) {
  NVFP4_REQUIRE(max_tokens >= 1 && max_tokens <= kTree, "nvfp4_draft_tree: max_tokens must be 1 to 1024");
  NVFP4_REQUIRE(requests >= 1 && requests < (1 << 30) && tokens >= 0 && tokens < (1ll << 31), "nvfp4_draft_tree: sizes out of range");
  if (tokens == 0) return 0;
  const TreeParams p{parents, cu_seqlens, lengths, tokens, (int)requests, (int)max_tokens, (int)((max_tokens + 63) / 64), mask, positions};
  return launch("nvfp4_draft_tree", draft_tree_kernel, dim3((unsigned)requests), kTreeThreads, 0, static_cast<cudaStream_t>(stream), p);
}

extern "C" int nvfp4_verify_drafts_within(const void* target_probs, int64_t target_row, const void* draft_probs, int64_t draft_row,
                                          int dtype, int64_t vocab, const void* tokens, int tokens_int64, const int32_t* parents,
                                          const int32_t* cu_seqlens, const float* uniforms, int64_t num_tokens, int64_t requests,
                                          int64_t max_tokens, int32_t* accepted, int32_t* num_accepted, int64_t* next_tokens,
                                          nvfp4_stream_t stream) {
  NVFP4_REQUIRE(max_tokens >= 1 && max_tokens <= kTree, "nvfp4_verify_drafts: max_tokens must be 1 to 1024");
  NVFP4_REQUIRE(vocab >= 1 && vocab < (1 << 30), "nvfp4_verify_drafts: vocabulary out of range");
  NVFP4_REQUIRE(requests >= 1 && requests < (1 << 30) && num_tokens >= 0 && num_tokens < (1ll << 31), "nvfp4_verify_drafts: sizes out of range");
  const int64_t size = dtype == NVFP4_DT_FP32 ? 4 : 2;
  NVFP4_REQUIRE((((uintptr_t)target_probs | (uintptr_t)draft_probs) & (uintptr_t)(size - 1)) == 0, "nvfp4_verify_drafts: unaligned rows");
  const VerifyParams p{target_probs, draft_probs, target_row, draft_row, tokens, tokens_int64, parents, cu_seqlens, uniforms, num_tokens,
                       (int)requests, (int)vocab, (int)max_tokens, accepted, num_accepted, next_tokens};
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  int ranks = 8;                               // as many blocks as are resident at once
  while (ranks > 1 && requests * ranks > 2 * sms) ranks >>= 1;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case NVFP4_DT_BF16: return run_verify<__nv_bfloat16>(p, ranks, st);
    case NVFP4_DT_FP16: return run_verify<__half>(p, ranks, st);
    case NVFP4_DT_FP32: return run_verify<float>(p, ranks, st);
  }
  return fail(-1, "nvfp4_verify_drafts: unknown dtype %d", dtype);
}

extern "C" int nvfp4_verify_drafts(const void* target_probs, int64_t target_row, const void* draft_probs, int64_t draft_row, int dtype,
                                   int64_t vocab, const void* tokens, int tokens_int64, const int32_t* parents, const int32_t* cu_seqlens,
                                   const float* uniforms, int64_t num_tokens, int64_t requests, int32_t* accepted, int32_t* num_accepted,
                                   int64_t* next_tokens, nvfp4_stream_t stream) {
  return nvfp4_verify_drafts_within(target_probs, target_row, draft_probs, draft_row, dtype, vocab, tokens, tokens_int64, parents, cu_seqlens,
                                    uniforms, num_tokens, requests, kTree, accepted, num_accepted, next_tokens, stream);
}
