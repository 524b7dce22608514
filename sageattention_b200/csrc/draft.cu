// Trees of drafted tokens: what every node sees and where it stands, and which of them the target's probabilities keep.
//
// A request's tokens cu[r] .. cu[r + 1] are a tree: its node 0 is the token that the step before ended with, node i hangs on the
// earlier node that parents[] names.  Nodes behind the 1024th are not part of it.
#include <limits.h>
#include "common/abi.cuh"
#include "common/fp4.cuh"
#include "common/launch.cuh"
#include "common/sm100.cuh"

namespace nvfp4 {
namespace {

constexpr int kTree = 1024;                    // nodes of a tree

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
  int requests, vocab;
  int32_t *accepted, *count;
  int64_t* next;
};

constexpr int kVerifyThreads = 512, kVerifyWarps = kVerifyThreads / 32;

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
// trip for all nodes), and where a sum over a row is needed the blocks of the cluster share it: a warp has a piece of the
// row.  What bounds it: the rows (one a rejection, one for the draw) where there are many requests, else the trips to memory and between
// the blocks, one behind the other.
template <typename T, bool kDrawn>
__global__ void __launch_bounds__(kVerifyThreads) verify_drafts_kernel(VerifyParams p) {
  constexpr int kPer = 16 / sizeof(T);
  constexpr int kStep = 32 * kPer;             // elements of a warp's load
  __shared__ int16_t up_s[kTree], path_s[kTree], rejected_s[kTree];
  __shared__ int32_t id_s[kTree];
  __shared__ float px_s[kTree], qx_s[kTree], u_s[kTree];
  __shared__ double mass_s[kTree];             // of what is left behind j rejections, and one over it
  __shared__ double block_s[2], warp_s[kVerifyWarps];
  __shared__ int node_s, k_s, len_s;
  __shared__ bool done_s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = blockIdx.z, ranks = gridDim.z, r = blockIdx.x;
  griddep_wait();
  griddep_launch();
  const Span span(p.cu, r, p.tokens);
  const int n = (int)min(span.n, (int64_t)kTree);
  const T* const target = static_cast<const T*>(p.p);
  const T* const draft = static_cast<const T*>(p.q);
  for (int i = tid; i < n; i += kVerifyThreads) {
    const int64_t t = span.t0 + i;
    const int a = p.parents[t];
    const int64_t id = p.ids64 ? static_cast<const int64_t*>(p.ids)[t] : (int64_t) static_cast<const int32_t*>(p.ids)[t];
    const bool child = a >= 0 && a < i, known = id >= 0 && id < p.vocab;
    up_s[i] = (int16_t)(child ? a : -1);
    id_s[i] = known ? (int32_t)id : -1;
    u_s[i] = p.u[t];
    float x = 0.0f, y = 0.0f;
    if (child && known) {
      x = mass_of<T>(target[(span.t0 + a) * p.sp + id]);
      if (kDrawn) y = mass_of<T>(draft[(span.t0 + a) * p.sq + id]);
    }
    px_s[i] = x;
    if (kDrawn) qx_s[i] = y;
  }
  __syncthreads();

  // what is left of a probability behind k rejections
  auto left_of = [&](double x, double q, int k) {
    for (int j = 0; j < k; ++j) x = fmax(x * mass_s[j] - q, 0.0);
    return x;
  };
  // ---- warp 0: on from node_s, behind child `from`, until a row's sum is wanted or no child is left
  int from = 1, len = 1, node = 0, k = 0;
  double mass = 1.0;                           // of what is left
  auto advance = [&]() -> bool {               // true: done
    for (;;) {
      int child = -1;
      for (int i0 = from & ~31; i0 < n && child < 0; i0 += 32) {
        const int i = i0 + lane;
        const uint32_t m = __ballot_sync(0xffffffffu, i >= from && i < n && up_s[i] == node);
        if (m) child = i0 + __ffs(m) - 1;
      }
      if (child < 0) return true;
      from = child + 1;
      bool passes;
      if (kDrawn) {
        passes = (double)u_s[child] * (double)qx_s[child] * mass < left_of(px_s[child], qx_s[child], k);
      } else {
        bool again = false;
        for (int j = lane; j < k; j += 32) again |= id_s[rejected_s[j]] == id_s[child];
        again = __any_sync(0xffffffffu, again);
        const double x = again ? 0.0 : (double)px_s[child];
        passes = (double)u_s[child] * mass < x;
        if (!passes) mass = fmax(mass - x, 0.0);
      }
      if (passes) {
        if (lane == 0) path_s[len] = (int16_t)child;
        ++len;
        node = child;
        k = 0;
        mass = 1.0;
      } else {
        if (!kDrawn && lane == 0) rejected_s[k] = (int16_t)child;
        __syncwarp();
        ++k;
        if (kDrawn) return false;
      }
    }
  };

  // ---- elements of the row of `node`: warp's piece [begin, end) of places, a place being an element behind the 16 bytes that
  // the row begins in
  const T *row = nullptr, *row_q = nullptr;
  int head = 0;
  bool same = false;
  auto open_row = [&](int node) {
    row = target + (span.t0 + node) * p.sp;
    head = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
    row -= head;                               // at 16 bytes; places in front of `head` are never read
    if (kDrawn) {
      const T* q = draft + (span.t0 + node) * p.sq;
      same = (int)((reinterpret_cast<uintptr_t>(q) & 15) / sizeof(T)) == head;
      row_q = q - head;
    }
  };
  auto load = [&](const T* base, int at, bool wide, T (&x)[kPer]) {
    if (wide && at >= head && at + kPer <= head + p.vocab) {
      *reinterpret_cast<uint4*>(x) = *reinterpret_cast<const uint4*>(base + at);
    } else {
#pragma unroll
      for (int e = 0; e < kPer; ++e) x[e] = at + e >= head && at + e < head + p.vocab ? base[at + e] : from_f32<T>(0.0f);
    }
  };
  // what is left of elements at .. at + kPer of the row, k rejections behind it; hit: some rejected token may be among them
  auto rest = [&](int at, int k, bool hit, double (&x)[kPer]) {
    alignas(16) T a[kPer], b[kPer];
    load(row, at, true, a);
    if (kDrawn && k > 0) load(row_q, at, same, b);
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      x[e] = mass_of<T>(a[e]);
      if (kDrawn && k > 0) x[e] = left_of(x[e], mass_of<T>(b[e]), k);
    }
    if (!kDrawn && hit) {
      for (int j = 0; j < k; ++j) {
        const int id = id_s[rejected_s[j]];
#pragma unroll
        for (int e = 0; e < kPer; ++e)
          if (id >= 0 && id + head == at + e) x[e] = 0.0;
      }
    }
  };
  auto touched = [&](int begin, int end, int k) {          // by a rejected token; all lanes of the warp
    bool hit = false;
    if (!kDrawn)
      for (int j = lane; j < k; j += 32) {
        const int id = id_s[rejected_s[j]];
        hit |= id >= 0 && id + head >= begin && id + head < end;
      }
    return __any_sync(0xffffffffu, hit);
  };
  // sum of places begin .. end by a warp, in all its lanes
  auto piece_sum = [&](int begin, int end, int k) {
    const bool hit = touched(begin, end, k);
    double sum = 0.0;
    constexpr int kAhead = 4;
#pragma unroll 1
    for (int at = begin + lane * kPer; at < end; at += kAhead * kStep) {
#pragma unroll
      for (int a = 0; a < kAhead; ++a) {
        if (at + a * kStep >= end) break;
        double x[kPer];
        rest(at + a * kStep, k, hit, x);
#pragma unroll
        for (int w = 1; w < kPer; w *= 2)
#pragma unroll
          for (int e = 0; e < kPer; e += 2 * w) x[e] += x[e + w];
        sum += x[0];
      }
    }
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
    return sum;
  };
  const int pieces = kVerifyWarps * ranks;
  auto piece = [&]() { return ((head + p.vocab + pieces - 1) / pieces + kStep - 1) / kStep * kStep; };
  // first of `n` pieces whose running sum exceeds `at`, or the last with any; `at` becomes relative to it
  auto pick = [](const auto& of, int n, double& at) {
    double before = 0.0, start = 0.0;
    int last = -1;
    for (int i = 0; i < n; ++i) {
      const double x = of(i);
      if (x > 0.0) {
        last = i;
        start = before;
        if (before + x > at) break;
      }
      before += x;
    }
    at -= start;
    return last;
  };
  int turn = 0;
  auto row_sum = [&](int node, int k) {        // all threads of the cluster; the same in all
    open_row(node);
    const int size = piece(), begin = (rank * kVerifyWarps + warp) * size;
    const double mine = piece_sum(begin, min(begin + size, head + p.vocab), k);
    if (lane == 0) warp_s[warp] = mine;
    __syncthreads();
    if (tid == 0) {
      double t = 0.0;
      for (int w = 0; w < kVerifyWarps; ++w) t += warp_s[w];
      block_s[turn] = t;
    }
    if (ranks > 1) cluster_sync_all();
    else __syncthreads();
    double t = 0.0;
    for (int c = 0; c < ranks; ++c) t += ranks > 1 ? ld_cluster_f64(smem_u32(&block_s[turn]), c) : block_s[turn];
    return t;
  };

  if (n > 0) {
    if (tid == 0) path_s[0] = 0;
    double sum = 0.0;
    int summed = -1, summed_k = 0;             // whose sum it is
    int at_node = 0, at_k = 0;
    for (;;) {
      if (warp == 0) {
        const bool done = advance();
        if (lane == 0) {
          node_s = node;
          k_s = k;
          len_s = len;
          done_s = done;
        }
      }
      __syncthreads();
      at_node = node_s;
      at_k = k_s;
      const bool done = done_s;
      if (done && summed == at_node && summed_k == at_k) break;
      turn ^= 1;
      if (kDrawn && !done) {                   // R_k is made of masses 0 .. k - 1
        if (tid == 0) mass_s[at_k - 1] = at_k == 1 ? 1.0 : sum > 0.0 ? 1.0 / sum : 0.0;
        __syncthreads();
      }
      sum = row_sum(at_node, at_k);
      summed = at_node;
      summed_k = at_k;
      if (done) break;
      mass = sum;
    }
    if (!(sum > 0.0)) {                        // nothing is left: from the row itself
      turn ^= 1;
      at_k = 0;
      sum = row_sum(at_node, 0);
    }
    // ---- the draw: block of the cluster, warp's piece, its part, element
    double at = (double)u_s[0] * sum;
    const int owner = pick([&](int c) { return ranks > 1 ? ld_cluster_f64(smem_u32(&block_s[turn]), c) : block_s[turn]; }, ranks, at);
    if (owner < 0) {
      if (rank == 0 && tid == 0) p.next[r] = 0;            // a row of zeros
    } else if (owner == rank) {
      const int size = piece();
      const int w = max(pick([&](int i) { return warp_s[i]; }, kVerifyWarps, at), 0);
      int begin = (rank * kVerifyWarps + w) * size, end = min(begin + size, head + p.vocab);
      if (size > 4 * kStep) {                  // a part a warp
        const int part = (size / kVerifyWarps + kStep - 1) / kStep * kStep, b = begin + warp * part;
        const double mine = piece_sum(b, min(b + part, end), at_k);
        __syncthreads();
        if (lane == 0) warp_s[warp] = mine;
        __syncthreads();
        const int x = max(pick([&](int i) { return warp_s[i]; }, kVerifyWarps, at), 0);
        begin += x * part;
        end = min(begin + part, end);
      }
      if (warp == 0) {
        const bool hit = touched(begin, end, at_k);
        double before = 0.0;
        int found = -1, last = -1;
        for (int i = begin; i < end && found < 0; i += kStep) {
          const int e0 = i + lane * kPer;
          double x[kPer], sums = 0.0;
          rest(e0, at_k, hit, x);
#pragma unroll
          for (int e = 0; e < kPer; ++e) sums += x[e];
          double upto = sums;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const double y = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += y;
          }
          double run = before + (upto - sums);
          int mine = INT_MAX, top = -1;
#pragma unroll
          for (int e = 0; e < kPer; ++e) {
            run += x[e];
            if (x[e] > 0.0 && e0 + e < end) {
              if (run > at && mine == INT_MAX) mine = e0 + e;
              top = e0 + e;
            }
          }
          before += __shfl_sync(0xffffffffu, upto, 31);
          const int first = __reduce_min_sync(0xffffffffu, mine);
          last = max(last, __reduce_max_sync(0xffffffffu, top));
          if (first != INT_MAX) found = first;
        }
        if (lane == 0) p.next[r] = max((found >= 0 ? found : last) - head, 0);
      }
    }
    if (rank == 0) {
      const int kept = len_s;
      for (int64_t i = tid; i < span.n; i += kVerifyThreads) p.accepted[span.t0 + i] = i < kept ? path_s[i] : -1;
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
  return launch_cluster("nvfp4_verify_drafts", kern, dim3((unsigned)p.requests, 1, (unsigned)ranks), (unsigned)ranks, kVerifyThreads, 0, st, p);
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

extern "C" int nvfp4_verify_drafts(const void* target_probs, int64_t target_row, const void* draft_probs, int64_t draft_row, int dtype,
                                   int64_t vocab, const void* tokens, int tokens_int64, const int32_t* parents, const int32_t* cu_seqlens,
                                   const float* uniforms, int64_t num_tokens, int64_t requests, int32_t* accepted, int32_t* num_accepted,
                                   int64_t* next_tokens, nvfp4_stream_t stream) {
  NVFP4_REQUIRE(vocab >= 1 && vocab < (1 << 30), "nvfp4_verify_drafts: vocabulary out of range");
  NVFP4_REQUIRE(requests >= 1 && requests < (1 << 30) && num_tokens >= 0 && num_tokens < (1ll << 31), "nvfp4_verify_drafts: sizes out of range");
  const int64_t size = dtype == NVFP4_DT_FP32 ? 4 : 2;
  NVFP4_REQUIRE((((uintptr_t)target_probs | (uintptr_t)draft_probs) & (uintptr_t)(size - 1)) == 0, "nvfp4_verify_drafts: unaligned rows");
  const VerifyParams p{target_probs, draft_probs, target_row, draft_row, tokens, tokens_int64, parents, cu_seqlens, uniforms, num_tokens,
                       (int)requests, (int)vocab, accepted, num_accepted, next_tokens};
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  int ranks = 8;                               // as many blocks as are resident twice over
  while (ranks > 1 && requests * ranks > 2 * sms) ranks >>= 1;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case NVFP4_DT_BF16: return run_verify<__nv_bfloat16>(p, ranks, st);
    case NVFP4_DT_FP16: return run_verify<__half>(p, ranks, st);
    case NVFP4_DT_FP32: return run_verify<float>(p, ranks, st);
  }
  return fail(-1, "nvfp4_verify_drafts: unknown dtype %d", dtype);
}
