// Routed experts around their matrix products: the choice of experts and the order of the rows, the gated activation
// with its 8-bit checkpoint, and the sum of the experts' rows back into tokens. All of it is bound by memory traffic (the
// routing of a large batch by instruction issue); values are read once (the routing reads the chosen logits again) and nothing
// is kept between calls.
#include "fs_experts.cuh"
#include "fs_tc.cuh"

#include <algorithm>
#include <cstring>

namespace fs {
namespace ex {
namespace {

constexpr unsigned kAll = 0xffffffffu;

// ---------------------------------------------------------------------------------------------------------------
// Routing
// ---------------------------------------------------------------------------------------------------------------
// Token t goes to the k experts with the largest score = logit + bias (fp32; ties to the lower expert), among those that
// are on: logit and bias above -inf, token not masked. Its gates are the soft-max of the LOGITS over the chosen experts or
// over all that are on. The (token, slot) pairs of an expert keep their order, so the result is the same in every run.
//
// One warp per token, lane l with experts [l PER, (l + 1) PER): the k-fold choice is a maximum over each lane's own experts and
// one over the lanes (redux), and the lowest of several lanes with the same score has the lowest expert. Two kernels of at
// most kMaxBlocks CTAs, CTA b with tokens [b c, (b + 1) c): the first selects and counts the CTA's pairs per expert, the
// second adds up the counts of the CTAs before it (every CTA for itself: E x kMaxBlocks words from L2, cheaper than a third
// launch or CTAs that wait for one another) and numbers its own pairs. Batches of one CTA do both in one launch.

constexpr int kMaxBlocks = 148;    // one for each SM: what the second kernel reads of the counts grows with the square of it
constexpr int kOrderWarps = 32, kGradWarps = 16;
constexpr int kMaxExperts = 1024;  // 32 per lane
constexpr int kMaxK = 32;          // one slot per lane

struct RouteArgs {
  const void* logits;
  long long ld;
  int T, E, k, chunk, blocks;
  const float* bias;
  const uint8_t* mask;
  int over_all;
  bool vec;
  float* gates;
  int *experts, *offsets, *pairs, *rows, *position;
  int* counts;  // [E, blocks]
  // gradient
  const float *gates_in, *grad;
  const int* experts_in;
  void* out;
};

// Unsigned keys in the order of the scores: 0 for an expert that is off, NaN above everything (it then shows in the gates).
__device__ __forceinline__ unsigned score_key(float s) {
  if (s != s) return 0xffffffffu;
  const unsigned b = __float_as_uint(s + 0.f);  // -0 becomes +0: they tie
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {
  float m;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(v));
  return m;
}

// Experts of a lane: chunks of C neighbours, those of the lanes side by side. The choice has one chunk (C = PER), so that the
// lowest lane with a score has the lowest expert.
template <int C>
__device__ __forceinline__ int expert_of(int lane, int i) {
  return i / C * (32 * C) + lane * C + i % C;
}
// The lane's part of a row of E; `fill` past its end. vec: its chunks are aligned and lie within the row or past it.
template <typename T, int PER, int C>
__device__ __forceinline__ void load_part(const T* row, int lane, int E, bool vec, float fill, float (&v)[PER]) {
#pragma unroll
  for (int q = 0; q < PER; q += C) {
    const int e = expert_of<C>(lane, q);
    float part[C];
#pragma unroll
    for (int i = 0; i < C; ++i) part[i] = fill;
    if (vec) {
      if (e < E) load_f32<T, C>(row + e, part);
    } else {
#pragma unroll
      for (int i = 0; i < C; ++i)
        if (e + i < E) part[i] = to_f32(row[e + i]);
    }
#pragma unroll
    for (int i = 0; i < C; ++i) v[q + i] = part[i];
  }
}
// Logits of a token, -inf for the experts that are off.
template <typename T, int PER, int C = PER>
__device__ __forceinline__ void load_logits(const RouteArgs& a, int t, int lane, const float (&bias)[PER], float (&l)[PER]) {
  load_part<T, PER, C>(static_cast<const T*>(a.logits) + (long long)t * a.ld, lane, a.E, a.vec, -INFINITY, l);
  const bool on = !a.mask || a.mask[t];
#pragma unroll
  for (int i = 0; i < PER; ++i) l[i] = on && bias[i] != -INFINITY ? l[i] : -INFINITY;
}
template <int PER, int C = PER>
__device__ __forceinline__ void load_bias(const RouteArgs& a, int lane, float (&bias)[PER]) {
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = expert_of<C>(lane, i);
    bias[i] = a.bias && e < a.E ? a.bias[e] : 0.f;
  }
}
// Largest of the logits (-inf: none is on), and 1 / the sum of exp(logit - largest).
template <int PER>
__device__ __forceinline__ void soft_max_over(const float (&l)[PER], float& top, float& inv) {
  top = l[0];
#pragma unroll
  for (int i = 1; i < PER; ++i) top = fmaxf(top, l[i]);
  top = warp_max(top);
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < PER; ++i) sum += expf(l[i] - top);
  inv = 1.f / warp_sum(sum);
}

// The experts of a lane that are still to be had, best first on demand. Up to 8 are sorted once (Batcher's odd-even merge
// network; equal keys by number), and taking the best is a shift; more are looked through anew after each one taken. 65536
// tokens, 8 experts a lane: 8 slots 78 us sorted and 108 us looked through, 2 slots 51 and 48; 16 a lane: 8 slots 163 us
// sorted, with half the warps for its registers, and 149 looked through, 2 slots 121 and 88.
template <int PER>
struct Candidates {
  static constexpr bool kSorted = PER <= 8;
  unsigned key[PER];
  int number[PER];  // sorted: expert of each key within the lane; else number[0] is that of the best
  unsigned best;
  __device__ __forceinline__ void look() {
    best = 0u;
    number[0] = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (key[i] > best) {
        best = key[i];
        number[0] = i;
      }
  }
  __device__ __forceinline__ void prepare() {
    if constexpr (!kSorted) {
      look();
    } else {
      sort();
    }
  }
  __device__ __forceinline__ void sort() {
#pragma unroll
    for (int i = 0; i < PER; ++i) number[i] = i;
#pragma unroll
    for (int p = 1; p < PER; p *= 2)
#pragma unroll
      for (int k = p; k >= 1; k /= 2)
#pragma unroll
        for (int j = k % p; j + k < PER; j += 2 * k)
#pragma unroll
          for (int i = j; i < j + k && i + k < PER; ++i)
            if (i / (2 * p) == (i + k) / (2 * p)) {
              const unsigned x = key[i], y = key[i + k];
              const int nx = number[i], ny = number[i + k];
              const bool swap = y > x || (y == x && ny < nx);
              key[i] = swap ? y : x;
              key[i + k] = swap ? x : y;
              number[i] = swap ? ny : nx;
              number[i + k] = swap ? nx : ny;
            }
    best = key[0];
  }
  __device__ __forceinline__ void take(bool mine) {
    if constexpr (kSorted) {
#pragma unroll
      for (int i = 0; i + 1 < PER; ++i) {
        key[i] = mine ? key[i + 1] : key[i];
        number[i] = mine ? number[i + 1] : number[i];
      }
      key[PER - 1] = mine ? 0u : key[PER - 1];
      best = key[0];
    } else {
      if (mine) {
#pragma unroll
        for (int i = 0; i < PER; ++i) key[i] = i == number[0] ? 0u : key[i];
        look();
      }
      __syncwarp();
    }
  }
};

template <typename T, int PER, int WARPS>
__device__ __forceinline__ void select_tokens(const RouteArgs& a, int* count) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int t0 = blockIdx.x * a.chunk, tokens = min(a.chunk, a.T - t0);
  float bias[PER], next[PER];
  load_bias<PER>(a, lane, bias);
  constexpr bool kEarly = PER <= 8;  // the next token's logits are on their way while this one's experts are chosen
  if (kEarly && warp < tokens) load_logits<T, PER>(a, t0 + warp, lane, bias, next);
  for (int i = warp; i < tokens; i += WARPS) {
    const int t = t0 + i;
    float l[PER], top, inv;
    if (kEarly) {
#pragma unroll
      for (int i = 0; i < PER; ++i) l[i] = next[i];
      if (i + WARPS < tokens) load_logits<T, PER>(a, t + WARPS, lane, bias, next);
    } else {
      load_logits<T, PER>(a, t, lane, bias, l);
    }
    Candidates<PER> left;
#pragma unroll
    for (int i = 0; i < PER; ++i) left.key[i] = l[i] != -INFINITY ? score_key(l[i] + bias[i]) : 0u;
    left.prepare();
    if (a.over_all) soft_max_over<PER>(l, top, inv);
    int expert = -1;  // of slot `lane`
    for (int s = 0; s < a.k; ++s) {
      const unsigned best = __reduce_max_sync(kAll, left.best);
      if (best == 0u) break;
      const int owner = __ffs(__ballot_sync(kAll, left.best == best)) - 1, j = owner * PER + __shfl_sync(kAll, left.number[0], owner);
      expert = lane == s ? j : expert;
      left.take(lane == owner);
    }
    const float chosen = expert >= 0 ? to_f32(static_cast<const T*>(a.logits)[(long long)t * a.ld + expert]) : -INFINITY;
    if (!a.over_all) {
      const float one[1] = {chosen};
      soft_max_over<1>(one, top, inv);
    }
    if (lane < a.k) {
      const long long p = (long long)t * a.k + lane;
      a.gates[p] = expert >= 0 ? expf(chosen - top) * inv : 0.f;
      a.experts[p] = expert;
      if (expert >= 0) atomicAdd(count + expert, 1);
    }
  }
}

// Exclusive prefix over v[0 .. n) in shared memory, by all threads of the CTA; the total comes back.
template <int WARPS>
__device__ __forceinline__ int scan_in_place(int* v, int n, int* scratch) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int base = 0;
  for (int c = 0; c < n; c += WARPS * 32) {
    const int j = c + threadIdx.x, x = j < n ? v[j] : 0;
    int inc = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(kAll, inc, o);
      inc += lane >= o ? y : 0;
    }
    if (lane == 31) scratch[warp] = inc;
    __syncthreads();
    int before = 0, total = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      before += w < warp ? scratch[w] : 0;
      total += scratch[w];
    }
    if (j < n) v[j] = base + before + inc - x;
    base += total;
    __syncthreads();
  }
  return base;
}

// The pairs of a warp, in order; the experts of the first kEarlyPairs x 32 of them are read ahead.
constexpr int kEarlyPairs = 4;
template <int WARPS>
struct WarpPairs {
  long long begin, end;
  int early[kEarlyPairs];
  __device__ __forceinline__ WarpPairs(const RouteArgs& a) {
    const int warp = threadIdx.x >> 5;
    const long long p0 = (long long)blockIdx.x * a.chunk * a.k, p1 = min((long long)a.T, (long long)(blockIdx.x + 1) * a.chunk) * a.k;
    const long long share = ((p1 - p0 + WARPS - 1) / WARPS + 31) / 32 * 32;
    begin = p0 + warp * share;
    end = min(p1, begin + share);
  }
  __device__ __forceinline__ void read(const RouteArgs& a, long long from) {
#pragma unroll
    for (int i = 0; i < kEarlyPairs; ++i) {
      const long long p = from + i * 32 + (threadIdx.x & 31);
      early[i] = p < end ? a.experts[p] : -1;
    }
  }
};

// Rows of this CTA's pairs. first[e]: row of its first pair of expert e. hist: [WARPS, E].
template <int WARPS>
__device__ __forceinline__ void number_pairs(const RouteArgs& a, WarpPairs<WARPS>& w, int* first, int* hist, int total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int j = threadIdx.x; j < WARPS * a.E; j += WARPS * 32) hist[j] = 0;
  __syncthreads();
  int* mine = hist + warp * a.E;
  constexpr int kRound = kEarlyPairs * 32;
  unsigned same[kEarlyPairs];  // lanes with the same expert
  for (long long from = w.begin; from < w.end; from += kRound) {
    if (from > w.begin) w.read(a, from);
#pragma unroll
    for (int i = 0; i < kEarlyPairs; ++i) same[i] = __match_any_sync(kAll, w.early[i]);
#pragma unroll
    for (int i = 0; i < kEarlyPairs; ++i) {
      const int e = w.early[i];
      if (e >= 0 && lane == __ffs(same[i]) - 1) mine[e] += __popc(same[i]);
      __syncwarp();
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < a.E; e += WARPS * 32) {
    int at = first[e], c[16];
#pragma unroll
    for (int j0 = 0; j0 < WARPS; j0 += 16) {
#pragma unroll
      for (int j = 0; j < 16; ++j) c[j] = hist[(j0 + j) * a.E + e];
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        hist[(j0 + j) * a.E + e] = at;
        at += c[j];
      }
    }
  }
  __syncthreads();
  const bool again = w.end - w.begin > kRound;
  for (long long from = w.begin; from < w.end; from += kRound) {
    if (again) {
      w.read(a, from);
#pragma unroll
      for (int i = 0; i < kEarlyPairs; ++i) same[i] = __match_any_sync(kAll, w.early[i]);
    }
#pragma unroll
    for (int i = 0; i < kEarlyPairs; ++i) {
      const int e = w.early[i];
      const long long p = from + i * 32 + lane;
      const int rank = __popc(same[i] & ((1u << lane) - 1u));
      const int at = e >= 0 ? mine[e] + rank : -1;
      __syncwarp();
      if (e >= 0 && rank == 0) mine[e] += __popc(same[i]);
      __syncwarp();
      if (p < w.end) {
        a.position[p] = at;
        if (at >= 0) {
          a.pairs[at] = (int)p;
          a.rows[at] = (int)((unsigned)p / (unsigned)a.k);
        }
        if (p >= total) a.pairs[p] = a.rows[p] = -1;  // rows after the last one that is routed
      }
    }
  }
}

// Warps of a CTA that chooses: as many as the registers allow (64 a thread, 128 with 32 experts a lane).
template <int PER>
constexpr int kSelectWarps = PER <= 16 ? 32 : 16;

template <typename T, int PER>
__global__ void __launch_bounds__(kSelectWarps<PER> * 32) route_select_kernel(const RouteArgs a) {
  constexpr int WARPS = kSelectWarps<PER>;
  extern __shared__ int sm[];
  __shared__ int scratch[WARPS];
  int* count = sm;  // [E], then the histograms of the warps
  for (int e = threadIdx.x; e < a.E; e += WARPS * 32) count[e] = 0;
  __syncthreads();
  select_tokens<T, PER, WARPS>(a, count);
  __syncthreads();
  if (a.blocks > 1) {
    for (int e = threadIdx.x; e < a.E; e += WARPS * 32) a.counts[e * a.blocks + blockIdx.x] = count[e];
    return;
  }
  const int total = scan_in_place<WARPS>(count, a.E, scratch);
  __syncthreads();
  for (int e = threadIdx.x; e < a.E; e += WARPS * 32) a.offsets[e] = count[e];
  if (threadIdx.x == 0) a.offsets[a.E] = total;
  WarpPairs<WARPS> pairs(a);
  pairs.read(a, pairs.begin);
  number_pairs(a, pairs, count, sm + a.E, total);
}

__global__ void __launch_bounds__(kOrderWarps * 32) route_order_kernel(const RouteArgs a) {
  extern __shared__ int sm[];
  __shared__ int scratch[kOrderWarps];
  int *all = sm, *before = sm + a.E;  // pairs of expert e in all CTAs, in the CTAs before this one
  WarpPairs<kOrderWarps> pairs(a);
  pairs.read(a, pairs.begin);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  constexpr int kSide = 4;  // experts that a warp adds up side by side, so that its loads are in flight together
  for (int e0 = warp * kSide; e0 < a.E; e0 += kOrderWarps * kSide) {
    int n[kSide] = {}, b[kSide] = {};
#pragma unroll 5
    for (int c = lane; c < a.blocks; c += 32)
#pragma unroll
      for (int i = 0; i < kSide; ++i) {
        const int v = e0 + i < a.E ? a.counts[(e0 + i) * a.blocks + c] : 0;
        n[i] += v;
        b[i] += c < (int)blockIdx.x ? v : 0;
      }
#pragma unroll
    for (int i = 0; i < kSide; ++i) {
      n[i] = __reduce_add_sync(kAll, n[i]);
      b[i] = __reduce_add_sync(kAll, b[i]);
      if (lane == 0 && e0 + i < a.E) {
        all[e0 + i] = n[i];
        before[e0 + i] = b[i];
      }
    }
  }
  __syncthreads();
  const int total = scan_in_place<kOrderWarps>(all, a.E, scratch);
  for (int e = threadIdx.x; e < a.E; e += kOrderWarps * 32) {
    if (blockIdx.x == 0) a.offsets[e] = all[e];
    before[e] += all[e];
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) a.offsets[a.E] = total;
  __syncthreads();
  number_pairs(a, pairs, before, sm + 2 * a.E, total);
}

// d logit_j = [j chosen as slot s] g_s dg_s - p_j sum_s g_s dg_s, p = the soft-max that the gates were taken from. The chosen
// experts' terms are added in a row of shared memory (E floats of every warp).
// Lanes hold 16 bytes of neighbours at a time, so that the warp's loads and its row are contiguous: 65536 tokens of 128 fp32
// logits take 19.6 us, of 1024 121 us (465 us with all of a lane's experts side by side).
template <typename T, int PER>
constexpr int kGradChunk = PER * sizeof(T) <= 16 ? PER : 16 / sizeof(T);
template <int PER>
constexpr int kGradCtas = PER <= 1 ? 4 : PER <= 4 ? 3 : PER <= 16 ? 2 : 1;  // on an SM, by their registers; a fourth, alone, added 3 us

template <typename T, int PER>
__global__ void __launch_bounds__(kGradWarps * 32, kGradCtas<PER>) route_grad_kernel(const RouteArgs a) {
  constexpr int C = kGradChunk<T, PER>;
  extern __shared__ float rows[];
  const int lane = threadIdx.x & 31;
  float* row = rows + (threadIdx.x >> 5) * (32 * PER);
  float bias[PER];
  load_bias<PER, C>(a, lane, bias);
  for (long long t = (long long)blockIdx.x * kGradWarps + (threadIdx.x >> 5); t < a.T; t += (long long)gridDim.x * kGradWarps) {
    const long long p = t * a.k + lane;
    const int expert = lane < a.k ? a.experts_in[p] : -1;
    const float gate = expert >= 0 ? a.gates_in[p] : 0.f;
    const float own = expert >= 0 ? gate * a.grad[p] : 0.f, inner = warp_sum(own);
    float v[PER];
    if (a.over_all) {
      float l[PER], top, inv;
      load_logits<T, PER, C>(a, (int)t, lane, bias, l);
      soft_max_over<PER>(l, top, inv);
#pragma unroll
      for (int i = 0; i < PER; ++i) v[i] = l[i] != -INFINITY ? -inner * (expf(l[i] - top) * inv) : 0.f;
    } else {
#pragma unroll
      for (int i = 0; i < PER; ++i) v[i] = 0.f;
    }
    __syncwarp();
#pragma unroll
    for (int q = 0; q < PER; q += C) {
      float part[C];
#pragma unroll
      for (int i = 0; i < C; ++i) part[i] = v[q + i];
      store_f32<float, C>(row + expert_of<C>(lane, q), part);
    }
    __syncwarp();
    if (expert >= 0 && expert < a.E) row[expert] += a.over_all ? own : own - gate * inner;
    __syncwarp();
    T* out = static_cast<T*>(a.out) + t * a.E;
#pragma unroll
    for (int q = 0; q < PER; q += C) {
      const int e = expert_of<C>(lane, q);
      float part[C];
      load_f32<float, C>(row + e, part);
      if (a.vec) {
        if (e < a.E) store_f32<T, C>(out + e, part);
      } else {
#pragma unroll
        for (int i = 0; i < C; ++i)
          if (e + i < a.E) out[e + i] = from_f32<T>(part[i]);
      }
    }
  }
}

// Tokens per CTA: whole rounds of 32 warps, at most kMaxBlocks CTAs. Batches of up to 64 tokens stay in one CTA and one launch:
// 64 tokens of 16 experts take 6.8 us there and 7.5 us in two launches (of 64 experts 8.1 and 10.5), 128 tokens 9.0 and
// 7.8 us (11.3 and 10.4).
void plan_route(int T, int& chunk, int& blocks) {
  chunk = (int)(((long long)T + kMaxBlocks - 1) / kMaxBlocks);
  chunk = (chunk + 31) / 32 * 32;
  if (T <= 64) chunk = 64;
  blocks = T > 0 ? (T - 1) / chunk + 1 : 1;
}

// Lets `kernel` take `most` bytes of dynamic shared memory, once for each device. The limit belongs to the kernel and all host
// threads, so it is the most that any call takes and never the size of the present one. `allowed`: the kernel's own, devices
// on which it is set.
template <typename K>
int allow_smem(K kernel, size_t most, std::atomic<uint64_t>& allowed) {
  if (most <= 48 * 1024) return FS_OK;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (e == cudaSuccess && !(allowed.load(std::memory_order_relaxed) & bit)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most);
    if (e == cudaSuccess) allowed.fetch_or(bit, std::memory_order_relaxed);
  }
  return e == cudaSuccess ? FS_OK : report_error(FS_ERR_CUDA, cudaGetErrorString(e));
}

std::atomic<uint64_t> g_order_allowed{0};  // of route_order_kernel, which all instances of launch_route share

template <typename T, int PER>
int launch_route(RouteArgs a, bool grad, cudaStream_t st) {
  const int C = grad ? kGradChunk<T, PER> : PER;
  const size_t part = sizeof(T) * C < 16 ? sizeof(T) * C : 16;
  a.vec = a.E % C == 0 && a.ld % C == 0 && aligned(a.logits, part) && aligned(a.out, part);
  if (grad) {
    const long long want = ((long long)a.T + kGradWarps - 1) / kGradWarps;
    const size_t bytes = (size_t)kGradWarps * 32 * PER * 4;
    static std::atomic<uint64_t> grad_allowed{0};
    const int s = allow_smem(route_grad_kernel<T, PER>, bytes, grad_allowed);
    if (s != FS_OK) return s;
    const long long most = 148 * kGradCtas<PER>;
    route_grad_kernel<T, PER><<<(int)(want < most ? want : most), kGradWarps * 32, bytes, st>>>(a);
    return launched(1);
  }
  constexpr int kWarps = kSelectWarps<PER>;
  const size_t one = (size_t)(a.blocks > 1 ? 1 : 1 + kWarps) * a.E * 4, two = (size_t)(2 + kOrderWarps) * a.E * 4;
  static std::atomic<uint64_t> select_allowed{0};
  int s = allow_smem(route_select_kernel<T, PER>, (size_t)(1 + kWarps) * 32 * PER * 4, select_allowed);
  if (s != FS_OK) return s;
  if (a.blocks > 1 && (s = allow_smem(route_order_kernel, (size_t)(2 + kOrderWarps) * kMaxExperts * 4, g_order_allowed)) != FS_OK) return s;
  route_select_kernel<T, PER><<<a.blocks, kWarps * 32, one, st>>>(a);
  if (a.blocks > 1) route_order_kernel<<<a.blocks, kOrderWarps * 32, two, st>>>(a);
  return launched(a.blocks > 1 ? 2 : 1);
}
template <typename T>
int launch_route(const RouteArgs& a, bool grad, cudaStream_t st) {
  const int per = (a.E + 31) / 32;
  if (per <= 1) return launch_route<T, 1>(a, grad, st);
  if (per <= 2) return launch_route<T, 2>(a, grad, st);
  if (per <= 4) return launch_route<T, 4>(a, grad, st);
  if (per <= 8) return launch_route<T, 8>(a, grad, st);
  if (per <= 16) return launch_route<T, 16>(a, grad, st);
  return launch_route<T, 32>(a, grad, st);
}
int launch_route(const RouteArgs& a, int type, bool grad, cudaStream_t st) {
  if (type == FS_TYPE_F32) return launch_route<float>(a, grad, st);
  if (type == FS_TYPE_F16) return launch_route<__half>(a, grad, st);
  return launch_route<__nv_bfloat16>(a, grad, st);
}

int check_route(const void* logits, int type, long long ld, int T, int E, int k) {
  if (type < 0 || type > 2) return report_error(FS_ERR_BAD_ARG, "type must be FS_TYPE_F32, FS_TYPE_F16 or FS_TYPE_BF16");
  if (T < 0 || E < 1 || E > kMaxExperts) return report_error(FS_ERR_BAD_ARG, "T must be >= 0 and E in [1, 1024]");
  if (k < 1 || k > kMaxK || k > E) return report_error(FS_ERR_BAD_ARG, "k must be in [1, min(E, 32)]");
  if ((long long)T * k > 0x7fffffffll) return report_error(FS_ERR_BAD_ARG, "T * k must be below 2^31");
  if (ld < E || (T > 0 && !logits)) return report_error(FS_ERR_BAD_ARG, "logits must have rows of at least E values");
  return check_device();
}

// ---------------------------------------------------------------------------------------------------------------
// Gated activation and its checkpoint
// ---------------------------------------------------------------------------------------------------------------
// h = p silu(g) v of rows u = [g | v], p = the gate of the row's pair (1 without a routing). The backward pass needs g and
// v; the checkpoint holds them in blocks of 32 along the row as integers in [-127, 127] times 2^e, e the smallest exponent
// at which the block's largest magnitude rounds to 127 at most: 8.25 bits instead of 16, an error of at most half a step. The
// maximum is 63.75 to 127.5 steps, so that is 1/127.5 of it at most (an eighth of the error of an 8-bit float with 3 bits of
// fraction at 64 to 128 steps, whose own steps are 8 there), and since
// scaling by a power of two is exact the codes do not depend on how the quotient is rounded. A block with an infinity or
// a NaN has exponent code 255 and stands for NaN throughout.
//
// VEC values of each half per lane: 16-byte loads for 16-bit types. 32 / VEC neighbouring lanes share a block.

constexpr int kActWarps = 8;

struct ActArgs {
  const void* u;
  long long ldu;
  int R, F, parts;
  const float* gates;
  const int* pairs;
  void* h;  // forward: the result; backward (may be null): the result recomputed from the checkpoint
  int8_t* codes;
  uint8_t* scales;
  // backward
  const int* position;
  const void* dh;
  long long lddh;
  void* du;
  float* dgates;
};

__device__ __forceinline__ unsigned block_exponent(unsigned amax_bits) {
  if (amax_bits >= 0x7f800000u) return 255u;
  const int e = (int)(amax_bits >> 23), m = (int)(amax_bits & 0x7fffffu);
  const int code = e - (m < 0x7f0000 ? 6 : 5);  // magnitude * 2^(127 - code) is in [64, 127.5)
  return (unsigned)(code < 1 ? 1 : code);
}
__device__ __forceinline__ float block_scale(unsigned code) {
  return code == 255u ? __uint_as_float(0x7fc00000u) : __uint_as_float(code << 23);
}
// Integers of at most 2^22 in magnitude and floats by way of an addition: 1.5 * 2^23 + x holds the nearest integer (ties to
// even) in its low bits, and a byte under the exponent of 2^23 is 2^23 plus its value. The conversion instructions have a
// sixteenth of the rate, which exp and the reciprocal of the sigmoid already take up.
constexpr float kToInt = 12582912.f;       // 1.5 * 2^23
constexpr float kFromByte = 8388608.f;     // 2^23
__device__ __forceinline__ uint32_t four_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {  // the lowest byte of each
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}
// fp32 bits of the largest magnitude of the lane's values and those of its neighbours in the block (whole warps; 32 / VEC
// lanes hold a block). 16-bit types compare pairs of bit patterns.
template <typename T, int VEC>
__device__ __forceinline__ unsigned block_maximum(const Pack<T, VEC>& q) {
  unsigned top = 0u;
  if constexpr (sizeof(T) == 2 && VEC % 2 == 0) {
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) top = __vmaxu2(top, q.w[i] & 0x7fff7fffu);
#pragma unroll
    for (int o = 16 / VEC; o; o >>= 1) top = __vmaxu2(top, __shfl_xor_sync(kAll, top, o));
    const unsigned short bits = (unsigned short)max(top & 0xffffu, top >> 16);
    T value;
    memcpy(&value, &bits, 2);
    return __float_as_uint(to_f32(value));
  } else {
    float x[VEC];
    unpack<T, VEC>(q, x);
#pragma unroll
    for (int i = 0; i < VEC; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
#pragma unroll
    for (int o = 16 / VEC; o; o >>= 1) top = max(top, __shfl_xor_sync(kAll, top, o));
    return top;
  }
}
// Codes of VEC values under an exponent code, as bytes.
template <int VEC>
struct alignas(VEC) Codes {
  uint8_t b[VEC];
};
template <int VEC>
__device__ __forceinline__ Codes<VEC> encode(const float (&x)[VEC], unsigned code) {
  const float inv = code == 255u ? 0.f : __uint_as_float((254u - code) << 23);  // infinities and NaN times 0: not looked at
  uint32_t n[VEC], w[(VEC + 3) / 4];
#pragma unroll
  for (int i = 0; i < VEC; ++i) n[i] = __float_as_uint(fmaf(x[i], inv, kToInt));
  if constexpr (VEC % 4 == 0) {
#pragma unroll
    for (int i = 0; i < VEC; i += 4) w[i / 4] = four_bytes(n[i], n[i + 1], n[i + 2], n[i + 3]);
  } else {
    w[0] = n[0];
  }
  Codes<VEC> q;
  memcpy(&q, w, VEC);
  return q;
}
// The values that codes stand for: ((2^23 + 128 + code) - (2^23 + 128)) * scale, exact in both steps. (2^23 times the scale is beyond
// fp32 for blocks from 2^111 on, so the difference comes first. A block's largest of 1.992 * 2^127 or more is held as 64 * 2^122 =
// 2^128: rounded towards zero, the product is the largest finite value, off by a quarter of a step at most.)
template <int VEC>
__device__ __forceinline__ void decode(const Codes<VEC>& codes, float scale, float (&x)[VEC]) {
  uint32_t w[(VEC + 3) / 4] = {};
  memcpy(w, &codes, VEC);
#pragma unroll
  for (int i = 0; i < VEC; ++i)
    x[i] = __fmul_rz(__uint_as_float(__byte_perm(w[i / 4] ^ 0x80808080u, 0x4b000000u, 0x7440u + (unsigned)(i % 4))) - (kFromByte + 128.f), scale);
}

__device__ __forceinline__ float row_gate(const ActArgs& a, int r, bool& routed) {
  routed = true;
  if (!a.pairs) return 1.f;
  const int p = a.pairs[r];
  routed = p >= 0 && p < a.R;  // as many pairs as rows
  return routed ? a.gates[p] : 0.f;
}
// 1 / (1 + 2^(-x log2 e)), to a relative 2^-21 and, below 0, |x| 2^-23 more: the power's argument is rounded to fp32, at -80 to
// 2^-18. 0 from about -87.3 down, where the sigmoid leaves the normal range of fp32. The instructions by themselves, with results
// below the normal range flushed: the intrinsics spend as much again on those.
__device__ __forceinline__ float sigmoid(float x) {
  float e, s;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(x * -1.4426950408889634f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s) : "f"(1.f + e));
  return s;
}
template <typename T, int VEC>
__device__ __forceinline__ Pack<T, VEC> read_pack(const T* p, bool in) {
  if (in) return read_only<T, VEC>(p);
  Pack<T, VEC> q;
  memset(&q, 0, sizeof(q));
  return q;
}
// A warp per row, or per part of a row where there are few.
template <typename T, int VEC>
__global__ void __launch_bounds__(kActWarps * 32, 4) act_kernel(const ActArgs a) {
  const int lane = threadIdx.x & 31;
  constexpr int kLanes = 32 / VEC;  // of a block of the checkpoint
  const int steps = (a.F + 32 * VEC - 1) / (32 * VEC), share = (steps + a.parts - 1) / a.parts, nb = (a.F + 31) / 32;
  const long long it = (long long)blockIdx.x * kActWarps + (threadIdx.x >> 5), r = a.parts == 1 ? it : it / a.parts;
  if (r >= a.R) return;
  const int s0 = a.parts == 1 ? 0 : (int)(it - r * a.parts) * share, end = min(a.F, (s0 + share) * 32 * VEC);
  bool routed;
  const float p = row_gate(a, (int)r, routed);
  const T* row = static_cast<const T*>(a.u) + r * a.ldu;
  T* out = static_cast<T*>(a.h) + r * a.F;
  uint8_t* codes = a.codes && routed ? reinterpret_cast<uint8_t*>(a.codes) + r * 2 * a.F : nullptr;
  uint8_t* scales = a.scales + r * 2 * nb;
  for (int c = (s0 * 32 + lane) * VEC; c - lane * VEC < end; c += 32 * VEC) {
    const bool in = c < a.F;
    const Pack<T, VEC> qg = read_pack<T, VEC>(row + c, in), qv = read_pack<T, VEC>(row + a.F + c, in);
    float g[VEC], v[VEC], h[VEC];
    unpack<T, VEC>(qg, g);
    unpack<T, VEC>(qv, v);
#pragma unroll
    for (int i = 0; i < VEC; ++i) h[i] = routed ? p * (g[i] * sigmoid(g[i])) * v[i] : 0.f;
    if (in) store_f32<T, VEC>(out + c, h);
    if (codes) {
      const unsigned eg = block_exponent(block_maximum<T, VEC>(qg)), ev = block_exponent(block_maximum<T, VEC>(qv));
      if (in) {
        *reinterpret_cast<Codes<VEC>*>(codes + c) = encode<VEC>(g, eg);
        *reinterpret_cast<Codes<VEC>*>(codes + a.F + c) = encode<VEC>(v, ev);
        if (lane % kLanes == 0) {
          scales[c / 32] = (uint8_t)eg;
          scales[nb + c / 32] = (uint8_t)ev;
        }
      }
    }
  }
}

// du = [p dh v s (1 + g (1 - s)) | p dh g s] with s = sigmoid(g), and d p = sum dh g s v, from the checkpoint (CODES) or
// from u as it was. One warp per row: the sum over the row stays in the warp.
template <typename T, int VEC, bool CODES>
__global__ void __launch_bounds__(kActWarps * 32, 4) act_grad_kernel(const ActArgs a) {
  const int lane = threadIdx.x & 31, nb = (a.F + 31) / 32;
  const long long r = (long long)blockIdx.x * kActWarps + (threadIdx.x >> 5);
  if (r >= a.R) return;
  bool routed;
  const float p = row_gate(a, (int)r, routed);
  const uint8_t *codes = reinterpret_cast<const uint8_t*>(a.codes) + r * 2 * a.F, *scales = a.scales + r * 2 * nb;
  const T *row = static_cast<const T*>(a.u) + r * a.ldu, *dh = static_cast<const T*>(a.dh) + r * a.lddh;
  T *du = static_cast<T*>(a.du) + r * 2 * a.F, *hr = a.h ? static_cast<T*>(a.h) + r * a.F : nullptr;
  float dp = 0.f;
  for (int c = lane * VEC; c < a.F; c += 32 * VEC) {
    float g[VEC], v[VEC], d[VEC], dg[VEC], dv[VEC], h[VEC];
    unpack<T, VEC>(read_only<T, VEC>(dh + c), d);
    if (CODES) {
      const Codes<VEC> cg = *reinterpret_cast<const Codes<VEC>*>(codes + c), cv = *reinterpret_cast<const Codes<VEC>*>(codes + a.F + c);
      const unsigned eg = scales[c / 32], ev = scales[nb + c / 32];
      decode<VEC>(cg, block_scale(eg), g);
      decode<VEC>(cv, block_scale(ev), v);
    } else {
      unpack<T, VEC>(read_only<T, VEC>(row + c), g);
      unpack<T, VEC>(read_only<T, VEC>(row + a.F + c), v);
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const float s = sigmoid(g[i]), gs = g[i] * s, dgs = d[i] * gs;
      dv[i] = routed ? p * dgs : 0.f;
      dg[i] = routed ? p * d[i] * v[i] * fmaf(gs, 1.f - s, s) : 0.f;
      h[i] = routed ? p * gs * v[i] : 0.f;
      dp = fmaf(dgs, v[i], dp);
    }
    store_f32<T, VEC>(du + c, dg);
    store_f32<T, VEC>(du + a.F + c, dv);
    if (hr) store_f32<T, VEC>(hr + c, h);
  }
  if (a.dgates) {
    dp = warp_sum(dp);
    if (lane == 0) {
      if (routed) a.dgates[a.pairs[r]] = dp;
      if (a.position[r] < 0) a.dgates[r] = 0.f;  // r as a pair: one that has no row
    }
  }
}

// Values a lane takes at a time: the most (8, 4 or 1; at most `most`) that divides the widths and that all pointers are aligned
// to.
template <typename... P>
int lane_values(int most, int F, int bytes, long long ld0, long long ld1, P... ptrs) {
  for (int v : {8, 4}) {
    const size_t a = (size_t)v * bytes < 16 ? (size_t)v * bytes : 16;
    if (v <= most && F % v == 0 && ld0 % v == 0 && ld1 % v == 0 && (aligned(ptrs, a) && ...)) return v;
  }
  return 1;
}

// Parts of a row, where the rows alone do not give every SM 16 warps (more of those that take few values at a time): a token of
// 8 slots and 2048 columns takes 3.6 us back from its rows in parts and 17.7 us by one warp.
int row_parts(long long rows, int width, int vec) {
  const int steps = (width + 32 * vec - 1) / (32 * vec);
  const long long want = rows > 0 ? (148 * 16 * (8 / vec) + rows - 1) / rows : 1;
  return (int)(want < 1 ? 1 : want > steps ? steps : want);
}
int row_blocks(long long items) {
  const long long b = (items + kActWarps - 1) / kActWarps;
  return (int)(b < 1 ? 1 : b > 148 * 64 ? 148 * 64 : b);
}

template <typename T, int VEC>
int launch_act(ActArgs a, bool grad, cudaStream_t st) {
  a.parts = grad ? 1 : row_parts(a.R, a.F, VEC);
  const long long warps = (long long)a.R * a.parts;
  const int blocks = (int)((warps + kActWarps - 1) / kActWarps);
  if (!grad) act_kernel<T, VEC><<<blocks, kActWarps * 32, 0, st>>>(a);
  else if (a.codes) act_grad_kernel<T, VEC, true><<<blocks, kActWarps * 32, 0, st>>>(a);
  else act_grad_kernel<T, VEC, false><<<blocks, kActWarps * 32, 0, st>>>(a);
  return launched(1);
}
template <typename T>
int launch_act(const ActArgs& a, bool grad, int vec, cudaStream_t st) {
  if (vec == 8) return launch_act<T, 8>(a, grad, st);
  if (vec == 4) return launch_act<T, 4>(a, grad, st);
  return launch_act<T, 1>(a, grad, st);
}
int launch_act(const ActArgs& a, int type, bool grad, int vec, cudaStream_t st) {
  if (type == FS_TYPE_F32) return launch_act<float>(a, grad, vec, st);
  if (type == FS_TYPE_F16) return launch_act<__half>(a, grad, vec, st);
  return launch_act<__nv_bfloat16>(a, grad, vec, st);
}

// ---------------------------------------------------------------------------------------------------------------
// Rows back into tokens
// ---------------------------------------------------------------------------------------------------------------
// y_t = sum_s w_ts o[position_ts] over the slots that are routed, w = the gates or 1, summed in fp32 in slot order and
// rounded once. A warp per token (or part of one), all its rows' loads in flight together.

struct CombineArgs {
  const void* o;
  long long ldo;
  int M, T, k, D, parts;
  const float* gates;  // null: weights of 1
  const int *position, *pairs;
  void* y;
  long long ldy;
  const void* dy;
  long long lddy;
  void* d_o;
  float* dgates;
};

template <typename T, typename Y, int VEC>
__global__ void __launch_bounds__(kActWarps * 32) combine_kernel(const CombineArgs a) {
  const int lane = threadIdx.x & 31;
  const int steps = (a.D + 32 * VEC - 1) / (32 * VEC), share = (steps + a.parts - 1) / a.parts;
  const long long items = (long long)a.T * a.parts;
  for (long long it = (long long)blockIdx.x * kActWarps + (threadIdx.x >> 5); it < items; it += (long long)gridDim.x * kActWarps) {
    const int t = (int)(it / a.parts), s0 = (int)(it - (long long)t * a.parts) * share, s1 = min(s0 + share, steps);
    const long long pair = (long long)t * a.k + lane;
    const int at = lane < a.k ? (a.position ? a.position[pair] : t) : -1;
    const float w = lane < a.k && a.gates ? a.gates[pair] : 1.f;
    for (int s = s0; s < s1; ++s) {
      const int c = (s * 32 + lane) * VEC;
      float y[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) y[i] = 0.f;
#pragma unroll 4
      for (int j = 0; j < a.k; ++j) {
        const int row = __shfl_sync(kAll, at, j);
        const float wj = __shfl_sync(kAll, w, j);
        if (row >= 0 && row < a.M && c < a.D) {
          float o[VEC];
          load_f32<T, VEC>(static_cast<const T*>(a.o) + (long long)row * a.ldo + c, o);
#pragma unroll
          for (int i = 0; i < VEC; ++i) y[i] += wj * o[i];
        }
      }
      if (c < a.D) store_f32<Y, VEC>(static_cast<Y*>(a.y) + (long long)t * a.ldy + c, y);
    }
  }
}

// do_i = w dy_t and d w = <dy_t, o_i> for the row i of a pair, zeros for a pair of no row and a row of no pair. A warp takes four
// slots of a token, so that dy is read once for them: by rows it comes back from DRAM for every slot, 45 % more bytes at
// four slots (112 us against 93 us for 65536 rows of 2048).
template <typename T, int VEC>
__global__ void __launch_bounds__(kActWarps * 32) combine_grad_kernel(const CombineArgs a) {
  constexpr int kSlots = 4;
  const int lane = threadIdx.x & 31, n = a.T * a.k, groups = (a.k + kSlots - 1) / kSlots;
  const long long it = (long long)blockIdx.x * kActWarps + (threadIdx.x >> 5);
  const int t = (int)(it / groups), s0 = (int)(it - (long long)t * groups) * kSlots, slots = min(kSlots, a.k - s0);
  if (t >= a.T) return;
  const int first = t * a.k + s0;
  const int at = lane < slots ? a.position[first + lane] : -1, other = lane < slots ? a.pairs[first + lane] : 0;
  const float weight = lane < slots && a.gates ? a.gates[first + lane] : 1.f;
  const T* dy = static_cast<const T*>(a.dy) + (long long)t * a.lddy;
  int row[kSlots];
  float w[kSlots], dw[kSlots] = {};
  bool any = false, empty[kSlots];  // empty: row first + j belongs to no pair
#pragma unroll
  for (int j = 0; j < kSlots; ++j) {
    const int r = __shfl_sync(kAll, at, j), p = __shfl_sync(kAll, other, j);
    w[j] = __shfl_sync(kAll, weight, j);
    row[j] = r < n ? r : -1;
    empty[j] = j < slots && (p < 0 || p >= n);
    any = any || row[j] >= 0;
  }
  if (any) {
    for (int c = lane * VEC; c < a.D; c += 32 * VEC) {
      const Pack<T, VEC> qg = read_only<T, VEC>(dy + c);
      Pack<T, VEC> qo[kSlots];
#pragma unroll
      for (int j = 0; j < kSlots; ++j)
        if (row[j] >= 0 && a.dgates) qo[j] = read_only<T, VEC>(static_cast<const T*>(a.o) + (long long)row[j] * a.ldo + c);
      float g[VEC], x[VEC];
      unpack<T, VEC>(qg, g);
#pragma unroll
      for (int j = 0; j < kSlots; ++j) {
        if (row[j] < 0) continue;
        if (a.dgates) {
          unpack<T, VEC>(qo[j], x);
#pragma unroll
          for (int i = 0; i < VEC; ++i) dw[j] = fmaf(g[i], x[i], dw[j]);
        }
#pragma unroll
        for (int i = 0; i < VEC; ++i) x[i] = g[i] * w[j];
        store_f32<T, VEC>(static_cast<T*>(a.d_o) + (long long)row[j] * a.D + c, x);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < kSlots; ++j) {
    if (empty[j]) {
      const float zero[VEC] = {};
      for (int c = lane * VEC; c < a.D; c += 32 * VEC) store_f32<T, VEC>(static_cast<T*>(a.d_o) + (long long)(first + j) * a.D + c, zero);
    }
    if (a.dgates && j < slots) {
      const float d = warp_sum(dw[j]);
      if (lane == 0) a.dgates[first + j] = d;
    }
  }
}

template <typename T, typename Y, int VEC>
int launch_combine(CombineArgs a, bool grad, cudaStream_t st) {
  a.parts = row_parts(a.T, a.D, VEC);
  if (!grad) combine_kernel<T, Y, VEC><<<row_blocks((long long)a.T * a.parts), kActWarps * 32, 0, st>>>(a);
  else combine_grad_kernel<T, VEC><<<(int)(((long long)a.T * ((a.k + 3) / 4) + kActWarps - 1) / kActWarps), kActWarps * 32, 0, st>>>(a);
  return launched(1);
}
// 16 bytes of a row at a time: 8 fp32 values, two loads, took 38.9 us for 29500 rows of 1024 into tokens where 4 take 34.2.
int sum_values(int type) { return type == FS_TYPE_F32 ? 4 : 8; }

template <typename T, typename Y>
int launch_combine(const CombineArgs& a, bool grad, int vec, cudaStream_t st) {
  if constexpr (sizeof(T) == 2)
    if (vec == 8) return launch_combine<T, Y, 8>(a, grad, st);
  if (vec == 4) return launch_combine<T, Y, 4>(a, grad, st);
  return launch_combine<T, Y, 1>(a, grad, st);
}
int launch_combine(const CombineArgs& a, int type, int y_type, bool grad, int vec, cudaStream_t st) {
  if (type == FS_TYPE_F16) return launch_combine<__half, __half>(a, grad, vec, st);
  if (type == FS_TYPE_BF16) return launch_combine<__nv_bfloat16, __nv_bfloat16>(a, grad, vec, st);
  if (y_type == FS_TYPE_F16) return launch_combine<float, __half>(a, grad, vec, st);
  if (y_type == FS_TYPE_BF16) return launch_combine<float, __nv_bfloat16>(a, grad, vec, st);
  return launch_combine<float, float>(a, grad, vec, st);
}

int check_rows(int type, int rows, int width) {
  if (type < 0 || type > 2) return report_error(FS_ERR_BAD_ARG, "type must be FS_TYPE_F32, FS_TYPE_F16 or FS_TYPE_BF16");
  if (rows < 0 || width < 1 || width > (1 << 28)) return report_error(FS_ERR_BAD_ARG, "rows must be >= 0 and the width in [1, 2^28]");
  return check_device();
}

}  // namespace
}  // namespace ex
}  // namespace fs

using namespace fs;
using namespace fs::ex;

extern "C" {

size_t fs_route_bytes(int T, int E, int k) {
  (void)k;
  if (T < 0 || E < 1 || E > kMaxExperts) return 0;
  int chunk, blocks;
  plan_route(T, chunk, blocks);
  return blocks > 1 ? (size_t)E * blocks * sizeof(int) : 0;
}

int fs_route(const void* logits, int type, long long ld, int T, int E, int k, const float* bias, const uint8_t* mask,
             int over_all, float* gates, int* experts, int* offsets, int* pairs, int* rows, int* position, void* ws,
             size_t ws_bytes, void* stream) {
  int s = check_route(logits, type, ld, T, E, k);
  if (s != FS_OK) return s;
  if (!offsets || (T > 0 && (!gates || !experts || !pairs || !rows || !position)))
    return report_error(FS_ERR_BAD_ARG, "null argument");
  if (ws_bytes < fs_route_bytes(T, E, k) || (fs_route_bytes(T, E, k) > 0 && !ws))
    return report_error(FS_ERR_WORKSPACE, "workspace smaller than fs_route_bytes()");
  RouteArgs a{};
  a.logits = logits; a.ld = ld; a.T = T; a.E = E; a.k = k; a.bias = bias; a.mask = mask; a.over_all = over_all;
  a.gates = gates; a.experts = experts; a.offsets = offsets; a.pairs = pairs; a.rows = rows; a.position = position;
  a.counts = static_cast<int*>(ws);
  plan_route(T, a.chunk, a.blocks);
  return launch_route(a, type, false, static_cast<cudaStream_t>(stream));
}

int fs_route_grad(const void* logits, int type, long long ld, int T, int E, int k, const float* bias, const uint8_t* mask,
                  int over_all, const float* gates, const int* experts, const float* grad, void* out, void* stream) {
  int s = check_route(logits, type, ld, T, E, k);
  if (s != FS_OK || T == 0) return s;
  if (!gates || !experts || !grad || !out) return report_error(FS_ERR_BAD_ARG, "null argument");
  RouteArgs a{};
  a.logits = logits; a.ld = ld; a.T = T; a.E = E; a.k = k; a.bias = bias; a.mask = mask; a.over_all = over_all;
  a.gates_in = gates; a.experts_in = experts; a.grad = grad; a.out = out;
  return launch_route(a, type, true, static_cast<cudaStream_t>(stream));
}

int fs_gated_act(const void* u, int type, long long ldu, int R, int F, const float* gates, const int* pairs, void* h,
                 int8_t* codes, uint8_t* scales, void* stream) {
  int s = check_rows(type, R, F);
  if (s != FS_OK || R == 0) return s;
  if (!u || !h || ldu < 2 * (long long)F || (pairs && !gates) || (codes && !scales))
    return report_error(FS_ERR_BAD_ARG, "null argument, or rows of u shorter than 2 F");
  ActArgs a{};
  a.u = u; a.ldu = ldu; a.R = R; a.F = F; a.gates = gates; a.pairs = pairs; a.h = h;
  a.codes = codes; a.scales = scales;
  // the codes' alignment is that of their first byte and the width: 8 values of a lane are one store
  int vec = lane_values(8, F, type_bytes(type), ldu, 0, u, h);
  while (codes && vec > 1 && !aligned(codes, vec)) vec = vec == 8 ? 4 : 1;
  return launch_act(a, type, false, vec, static_cast<cudaStream_t>(stream));
}

int fs_gated_act_grad(const void* u, long long ldu, const int8_t* codes, const uint8_t* scales, int type, int R, int F,
                      const float* gates, const int* pairs, const int* position, const void* dh, long long lddh, void* du,
                      float* dgates, void* h, void* stream) {
  int s = check_rows(type, R, F);
  if (s != FS_OK || R == 0) return s;
  if ((!u && !codes) || (codes && !scales) || !dh || !du || lddh < F || (u && !codes && ldu < 2 * (long long)F) ||
      (pairs && !gates) || (dgates && (!pairs || !position)))
    return report_error(FS_ERR_BAD_ARG, "null argument, or rows shorter than their width");
  ActArgs a{};
  a.u = u; a.ldu = ldu; a.R = R; a.F = F; a.gates = gates; a.pairs = pairs; a.position = position; a.h = h;
  a.codes = const_cast<int8_t*>(codes); a.scales = const_cast<uint8_t*>(scales);
  a.dh = dh; a.lddh = lddh; a.du = du; a.dgates = dgates;
  int vec = lane_values(8, F, type_bytes(type), codes ? 0 : ldu, lddh, codes ? nullptr : u, dh, du, static_cast<const void*>(h));
  while (codes && vec > 1 && !aligned(codes, vec)) vec = vec == 8 ? 4 : 1;
  return launch_act(a, type, true, vec, static_cast<cudaStream_t>(stream));
}

int fs_combine(const void* o, int type, long long ldo, int M, int T, int k, int D, const float* gates, const int* position,
               void* y, int y_type, long long ldy, void* stream) {
  int s = check_rows(type, T, D);
  if (s != FS_OK || T == 0) return s;
  if (k < 1 || k > kMaxK || (long long)T * k > 0x7fffffffll) return report_error(FS_ERR_BAD_ARG, "k must be in [1, 32], T * k below 2^31");
  if (!o || M < 0 || (!position && k != 1) || !y || ldo < D || ldy < D || y_type < 0 || y_type > 2 || (y_type != type && type != FS_TYPE_F32))
    return report_error(FS_ERR_BAD_ARG, "null argument, rows shorter than D, or a wrong type of the result");
  CombineArgs a{};
  a.o = o; a.ldo = ldo; a.M = M; a.T = T; a.k = k; a.D = D; a.gates = gates; a.position = position; a.y = y; a.ldy = ldy;
  return launch_combine(a, type, y_type, false, lane_values(sum_values(type), D, type_bytes(type), ldo, ldy, o, y), static_cast<cudaStream_t>(stream));
}

int fs_combine_grad(const void* o, int type, long long ldo, int T, int k, int D, const float* gates, const int* position,
                    const int* pairs, const void* dy, long long lddy, void* d_o, float* dgates, void* stream) {
  int s = check_rows(type, T, D);
  if (s != FS_OK || T == 0) return s;
  if (k < 1 || k > kMaxK || (long long)T * k > 0x7fffffffll) return report_error(FS_ERR_BAD_ARG, "k must be in [1, 32], T * k below 2^31");
  if (!position || !pairs || !dy || !d_o || lddy < D || (dgates && (!o || !gates || ldo < D)))
    return report_error(FS_ERR_BAD_ARG, "null argument, or rows shorter than D");
  CombineArgs a{};
  a.o = o; a.ldo = ldo; a.T = T; a.k = k; a.D = D; a.gates = gates; a.position = position; a.pairs = pairs;
  a.dy = dy; a.lddy = lddy; a.d_o = d_o; a.dgates = dgates;
  return launch_combine(a, type, type, true, lane_values(sum_values(type), D, type_bytes(type), o ? ldo : 0, lddy, o, dy, d_o), static_cast<cudaStream_t>(stream));
}

}  // extern "C"
