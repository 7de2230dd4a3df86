// Layer norm of rows of F values and its gradients:
//
//   m = sum x / F,  v = sum (x - m)^2 / F,  r = 1 / sqrt(v + eps),  n = (x - m) r,  y = n w + b
//   dx = r (u - mean(u) - n mean(u n)),  u = w dy;   dw = sum over rows of dy n,  db = sum over rows of dy
//
// A row lies in the registers of a group of warps (the mean first, then the squares of the differences from it: one read, and no
// cancellation), groups walk over the rows with several rows' loads under way (cp.async, each thread what it reads itself), and in the
// backward pass each thread adds what its columns contribute to dw and db over all its rows. A CTA leaves one row of sums, which a
// second launch adds in a fixed order, so every run gives the same bits. Rows whose columns are too many for that go without, and a third kernel
// reads them again. Sums are fp32; y, dx, dw and db are rounded once.
//
// Memory is the floor and latency of a row's two or three sums across warps what is seen: 16384 rows of 2048 in bf16 take 30.6 us forward (a copy: 22.7)
// and 47 + 6 backward (201 MB: 31 at 6.5 TB/s). Measured on the way: a whole row per warp reads w and b from L1 for every row, which takes as long as the
// row (36 to 40 us); eight warps to a row 36; 84 registers of 512 threads leave one CTA an SM (71 us backward); w, dy and n kept in
// registers instead of read and unpacked twice 62 -> 47.
#include "fs_experts.cuh"
#include "fs_ptx.cuh"

namespace fs {
namespace ex {
namespace {

using tc::add2;
using tc::fma2;
using tc::mul2;
using tc::pk;
using tc::u64;
using tc::upk;

constexpr int kMaxNormThreads = 512;
constexpr int kLongThreads = 512;  // of rows that registers do not hold

struct NormArgs {
  const void *x, *dy, *w, *b;
  long long ldx, lddy;
  void* out;  // y or dx, densely packed
  float *mean, *rstd;
  float* sums;  // [CTAs][2][F] (null: no dw, db)
  int rows, F;
  float eps;
  int group;  // threads of a row
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ void group_barrier(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }

// The sum over a group's warps of one or two values, the same bits in every thread; slot: N x 16 floats of this group, zeros where there
// is no warp, that the call before this one did not use.
template <int N>
__device__ __forceinline__ void group_sum(float (&v)[N], float* slot, int warps, int barrier) {
  const int lane = threadIdx.x & 31, warp = (threadIdx.x >> 5) % warps;
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = warp_sum(v[i]);
  if (warps == 1) return;
  if (lane == 0)
#pragma unroll
    for (int i = 0; i < N; ++i) slot[16 * i + warp] = v[i];
  group_barrier(barrier, warps * 32);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float4 p = *reinterpret_cast<const float4*>(slot + 16 * i);
    v[i] = (p.x + p.y) + (p.z + p.w);
    if (warps > 4) {
      const float4 q = *reinterpret_cast<const float4*>(slot + 16 * i + 4);
      v[i] += (q.x + q.y) + (q.z + q.w);
    }
    if (warps > 8) {
      const float4 q = *reinterpret_cast<const float4*>(slot + 16 * i + 8), u = *reinterpret_cast<const float4*>(slot + 16 * i + 12);
      v[i] += ((q.x + q.y) + (q.z + q.w)) + ((u.x + u.y) + (u.z + u.w));
    }
  }
}
// Pairs of a pack's values (V = 1: the value and 0).
template <typename T, int V>
__device__ __forceinline__ void pairs(const Pack<T, V>& q, u64 (&p)[(V + 1) / 2]) {
  if constexpr (V == 1) {
    p[0] = pk(to_f32(*reinterpret_cast<const T*>(&q.w[0])), 0.f);
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) p[i] = pk(__uint_as_float(q.w[2 * i]), __uint_as_float(q.w[2 * i + 1]));
  } else {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      float lo, hi;
      two_f32(q.w[i], lo, hi, T());
      p[i] = pk(lo, hi);
    }
  }
}
template <typename T, int V>
__device__ __forceinline__ void store_pairs(T* to, const u64 (&p)[(V + 1) / 2]) {
  float v[V + 1];
#pragma unroll
  for (int i = 0; i < (V + 1) / 2; ++i) upk(p[i], v[2 * i], v[2 * i + 1]);
  float out[V];
#pragma unroll
  for (int i = 0; i < V; ++i) out[i] = v[i];
  store_f32<T, V>(to, out);
}
__device__ __forceinline__ float both(u64 v) {
  float lo, hi;
  upk(v, lo, hi);
  return lo + hi;
}

// V values of w or b (null: `other`) from column c on, inside of F.
template <typename W, int V>
__device__ __forceinline__ void columns(const void* p, int c, float other, u64 (&v)[(V + 1) / 2]) {
  if (!p) {
#pragma unroll
    for (int i = 0; i < (V + 1) / 2; ++i) v[i] = pk(other, other);
  } else {
    pairs<W, V>(read_only<W, V>(static_cast<const W*>(p) + c), v);
  }
}

// Values of rows to come, in shared memory that only the thread itself reads: S - 1 rows are under way without a register, and
// no thread waits for another one. Loads of V values; those of two bytes are not to be had asynchronously and are waited for.
template <typename T, int V>
__device__ __forceinline__ void fetch(Pack<T, V>* to, const T* from) {
  constexpr int kBytes = V * sizeof(T);
  const uint32_t at = (uint32_t)__cvta_generic_to_shared(to);
  if constexpr (kBytes == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at), "l"(from) : "memory");
  else if constexpr (kBytes == 4) asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(at), "l"(from) : "memory");
  else *to = read_only<T, V>(from);
}
__device__ __forceinline__ void fetch_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>  // all but the last LEFT rows
__device__ __forceinline__ void fetch_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory"); }

constexpr int kForwardStages = 6;  // rows under way of the forward pass, with the one that is worked on

// One row per group of a.group threads, V values to a load, NV loads a thread. V > 1: rows, weights and F are aligned to it. Up to 16 values
// of a thread, w and b stay in registers (from L1 for every row of 2048, they took as long as the row itself) and several rows are under way;
// above that a row's loads are under way all at once.
template <typename T, typename W, int V, int NV>
__global__ void __launch_bounds__(V * NV <= (V > 1 ? 16 : 8) ? 256 : kMaxNormThreads, V * NV <= (V > 1 ? 16 : 8) ? 3 : 1) norm_kernel(const NormArgs a) {
  constexpr bool kHold = V * NV <= (V > 1 ? 16 : 8);
  constexpr int P = (V + 1) / 2, S = kHold ? kForwardStages : 1;
  __shared__ __align__(16) float slots[2][16][16];
  extern __shared__ __align__(16) uint8_t raw[];
  Pack<T, V>* ring = reinterpret_cast<Pack<T, V>*>(raw) + threadIdx.x;  // kHold: [S][NV][threads]
  const int group = a.group, groups = blockDim.x / group, g = threadIdx.x / group, t = threadIdx.x % group, warps = group / 32;
  u64 w[kHold ? NV : 1][P], b[kHold ? NV : 1][P];
  if (kHold)
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if ((i * group + t) * V < a.F) {
        columns<W, V>(a.w, (i * group + t) * V, 1.f, w[i]);
        columns<W, V>(a.b, (i * group + t) * V, 0.f, b[i]);
      }
  if (warps > 1) {
    for (int i = threadIdx.x; i < 512; i += blockDim.x) (&slots[0][0][0])[i] = 0.f;
    __syncthreads();
  }
  bool in[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) in[i] = (i * group + t) * V < a.F;
  const float per = 1.f / a.F;
  const long long stride = (long long)gridDim.x * groups;
  long long row = (long long)blockIdx.x * groups + g;
  long long left = row < a.rows ? (a.rows - row + stride - 1) / stride : 0, coming = left;  // rows of this group, and those not yet asked for
  const T* x = static_cast<const T*>(a.x) + row * a.ldx + t * V;
  T* out = static_cast<T*>(a.out) + row * a.F + t * V;
  const long long x_step = stride * a.ldx, out_step = stride * a.F;
  auto ask = [&](int s) {
    if (coming > 0) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (in[i]) fetch<T, V>(ring + (s * NV + i) * blockDim.x, x + i * group * V);
      x += x_step;
      --coming;
    }
    fetch_commit();
  };
  if (kHold)
    for (int s = 0; s < S - 1; ++s) ask(s);
  for (int stage = 0; left > 0; --left, row += stride, out += out_step, stage = stage + 1 == S ? 0 : stage + 1) {
    Pack<T, V> q[NV];
    if (kHold) {
      ask(stage ? stage - 1 : S - 1);
      fetch_wait<S - 1>();
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (in[i]) q[i] = ring[(stage * NV + i) * blockDim.x];
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (in[i]) q[i] = read_only<T, V>(x + i * group * V);
      x += x_step;
    }
    // unpacked once where registers hold that, else in each of the three passes
    u64 v[kHold ? NV : 1][P], sum = 0ull;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int k = kHold ? i : 0;
      pairs<T, V>(q[i], v[k]);
      if (in[i])
#pragma unroll
        for (int j = 0; j < P; ++j) sum = add2(sum, v[k][j]);
    }
    float s[1] = {both(sum)};
    group_sum(s, slots[0][g], warps, 1 + g);
    const float mean = s[0] * per;
    const u64 less = pk(-mean, V == 1 ? 0.f : -mean);
    sum = 0ull;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int k = kHold ? i : 0;
      if (!kHold) pairs<T, V>(q[i], v[0]);
      if (in[i])
#pragma unroll
        for (int j = 0; j < P; ++j) {
          v[k][j] = add2(v[k][j], less);
          sum = fma2(v[k][j], v[k][j], sum);
        }
    }
    s[0] = both(sum);
    group_sum(s, slots[1][g], warps, 1 + g);
    const float r = __frsqrt_rn(fmaf(s[0], per, a.eps));
    if (a.mean && t == 0) {
      a.mean[row] = mean;
      a.rstd[row] = r;
    }
    const u64 r2 = pk(r, r);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int k = kHold ? i : 0;
      if (!in[i]) continue;
      if (!kHold) {
        pairs<T, V>(q[i], v[0]);
#pragma unroll
        for (int j = 0; j < P; ++j) v[0][j] = add2(v[0][j], less);
        columns<W, V>(a.w, (i * group + t) * V, 1.f, w[0]);
        columns<W, V>(a.b, (i * group + t) * V, 0.f, b[0]);
      }
#pragma unroll
      for (int j = 0; j < P; ++j) v[k][j] = fma2(mul2(v[k][j], r2), w[k][j], b[k][j]);
      store_pairs<T, V>(out + i * group * V, v[k]);
    }
  }
}

// Rows under way, with the one that is worked on, by a thread's bytes of a row and its gradient: two CTAs of 96 KB to an SM, or one of 192 KB.
__host__ __device__ constexpr int norm_stages(int bytes) { return bytes <= 64 ? 6 : bytes <= 128 ? 3 : bytes <= 256 ? 3 : 1; }

// The gradients, from mean and rstd as the forward pass left them, as r u - r mean(u) - n r mean(u n). SUMS: those to w and b as well; up to 16 values of a thread, of which w and what
// both passes over them need stay in registers (read and unpacked again, they took a third of all instructions).
template <typename T, typename W, int V, int NV, bool SUMS>
__global__ void __launch_bounds__(256, SUMS ? 2 : 1) norm_grad_kernel(const NormArgs a) {
  constexpr int P = (V + 1) / 2, S = norm_stages(2 * NV * (int)sizeof(Pack<T, V>));
  __shared__ __align__(16) float slots[2][8][32];
  extern __shared__ __align__(16) uint8_t raw[];
  Pack<T, V>* ring = reinterpret_cast<Pack<T, V>*>(raw) + threadIdx.x;  // [S][2][NV][threads]; in the end the groups' sums
  const int groups = blockDim.x / a.group, g = threadIdx.x / a.group, t = threadIdx.x % a.group, warps = a.group / 32;
  u64 dw[SUMS ? NV : 1][P], db[SUMS ? NV : 1][P];
#pragma unroll
  for (int i = 0; i < (SUMS ? NV : 1); ++i)
#pragma unroll
    for (int j = 0; j < P; ++j) dw[i][j] = db[i][j] = 0ull;
  u64 w[SUMS ? NV : 1][P];
  if (SUMS)
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if ((i * a.group + t) * V < a.F) columns<W, V>(a.w, (i * a.group + t) * V, 1.f, w[i]);
  if (warps > 1) {
    for (int i = threadIdx.x; i < 512; i += blockDim.x) (&slots[0][0][0])[i] = 0.f;
    __syncthreads();
  }
  bool in[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) in[i] = (i * a.group + t) * V < a.F;
  const float per = 1.f / a.F;
  const long long stride = (long long)gridDim.x * groups, row = (long long)blockIdx.x * groups + g;
  long long left = row < a.rows ? (a.rows - row + stride - 1) / stride : 0, coming = left;  // rows of this group, and those not yet asked for
  const T *x = static_cast<const T*>(a.x) + row * a.ldx + t * V, *dy = static_cast<const T*>(a.dy) + row * a.lddy + t * V;
  T* out = a.out ? static_cast<T*>(a.out) + row * a.F + t * V : nullptr;
  const float *mean = a.mean + row, *rstd = a.rstd + row;
  const long long x_step = stride * a.ldx, dy_step = stride * a.lddy, out_step = stride * a.F;
  auto ask = [&](int s) {
    if (coming > 0) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (in[i]) {
          fetch<T, V>(ring + (s * 2 * NV + i) * blockDim.x, x + i * a.group * V);
          fetch<T, V>(ring + ((s * 2 + 1) * NV + i) * blockDim.x, dy + i * a.group * V);
        }
      x += x_step;
      dy += dy_step;
      --coming;
    }
    fetch_commit();
  };
  for (int s = 0; s < S - 1; ++s) ask(s);
  float next_mean = 0.f, next_r = 0.f;
  if (left > 0) {
    next_mean = __ldg(mean);
    next_r = __ldg(rstd);
  }
  for (int s = 0, turn = 0; left > 0; --left, s = s + 1 == S ? 0 : s + 1, turn ^= 1) {
    ask(s ? s - 1 : S - 1);
    const float r = next_r;
    const u64 r2 = pk(r, r), less = pk(-next_mean, V == 1 ? 0.f : -next_mean);
    if (left > 1) {
      mean += stride;
      rstd += stride;
      next_mean = __ldg(mean);
      next_r = __ldg(rstd);
    }
    fetch_wait<S - 1>();
    const Pack<T, V>*px = ring + s * 2 * NV * blockDim.x, *pg = px + NV * blockDim.x;
    u64 su = 0ull, sn = 0ull, n[SUMS ? NV : 1][P], u[SUMS ? NV : 1][P];
    auto read = [&](int i, int k) {  // n, and dy into u
      pairs<T, V>(px[i * blockDim.x], n[k]);
      pairs<T, V>(pg[i * blockDim.x], u[k]);
      if (!SUMS) columns<W, V>(a.w, (i * a.group + t) * V, 1.f, w[0]);
#pragma unroll
      for (int j = 0; j < P; ++j) n[k][j] = mul2(add2(n[k][j], less), r2);  // as the forward pass: x r - mean r would round a large mean twice
    };
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      constexpr int kOne = SUMS ? 1 : 0;
      const int k = i * kOne;
      if (!in[i]) continue;
      read(i, k);
#pragma unroll
      for (int j = 0; j < P; ++j) {
        if (SUMS) {
          dw[k][j] = fma2(u[k][j], n[k][j], dw[k][j]);
          db[k][j] = add2(db[k][j], u[k][j]);
        }
        u[k][j] = mul2(u[k][j], w[k][j]);
        su = add2(su, u[k][j]);
        sn = fma2(u[k][j], n[k][j], sn);
      }
    }
    if (!out) continue;
    float sum[2] = {both(su), both(sn)};
    group_sum(sum, slots[turn][g], warps, 1 + g);
    const float r1 = -sum[0] * per * r, rn = -sum[1] * per * r;
    const u64 m1 = pk(r1, r1), m2 = pk(rn, rn);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      constexpr int kOne = SUMS ? 1 : 0;
      const int k = i * kOne;
      if (!in[i]) continue;
      if (!SUMS) read(i, 0);
#pragma unroll
      for (int j = 0; j < P; ++j) n[k][j] = fma2(m2, n[k][j], fma2(SUMS ? u[k][j] : mul2(u[k][j], w[k][j]), r2, m1));
      store_pairs<T, V>(out + i * a.group * V, n[k]);
    }
    out += out_step;
  }
  if (!SUMS) return;
  fetch_wait<0>();
  float* merge = reinterpret_cast<float*>(raw);  // [groups - 1][2][F]
  __syncthreads();
  auto each = [&](auto&& f) {  // f(column, its dw, its db)
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < P; ++j) {
        const int c = (i * a.group + t) * V + 2 * j;
        float w0, w1, b0, b1;
        upk(dw[i][j], w0, w1);
        upk(db[i][j], b0, b1);
        if (c < a.F) f(c, w0, b0);
        if (V > 1 && c < a.F) f(c + 1, w1, b1);
      }
  };
  each([&](int c, float w, float b) {
    if (g > 0) {
      merge[(size_t)(g - 1) * 2 * a.F + c] = w;
      merge[(size_t)(g - 1) * 2 * a.F + a.F + c] = b;
    }
  });
  __syncthreads();
  if (g > 0) return;
  float* sums = a.sums + (size_t)blockIdx.x * 2 * a.F;
  each([&](int c, float w, float b) {
    for (int k = 0; k < groups - 1; ++k) {
      w += merge[(size_t)k * 2 * a.F + c];
      b += merge[(size_t)k * 2 * a.F + a.F + c];
    }
    sums[c] = w;
    sums[a.F + c] = b;
  });
}

// dw and db from the CTAs' sums: 32 columns of [2][F] to a block, its eight warps an eighth of the CTAs each.
template <typename W>
__global__ void __launch_bounds__(256) norm_sums_kernel(const float* sums, int ctas, int F, W* dw, W* db) {
  __shared__ float part[8][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long c = (long long)blockIdx.x * 32 + lane, width = 2ll * F;
  float s = 0.f;
  if (c < width) {
    const int per = (ctas + 7) / 8, end = min(ctas, (warp + 1) * per);
#pragma unroll 8
    for (int i = warp * per; i < end; ++i) s += __ldg(sums + i * width + c);
  }
  part[warp][lane] = s;
  __syncthreads();
  if (warp != 0 || c >= width) return;
#pragma unroll
  for (int k = 1; k < 8; ++k) s += part[k][lane];
  W* out = c < F ? dw : db;
  if (out) out[c < F ? c : c - F] = from_f32<W>(s);
}

// Rows too long for registers: a CTA per row, which reads it three times (the second and third time from L2).
template <typename T, typename W>
__global__ void __launch_bounds__(kLongThreads) norm_long_kernel(const NormArgs a) {
  __shared__ __align__(16) float slots[2][32];
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    float s[1] = {0.f};
    for (int c = threadIdx.x; c < a.F; c += kLongThreads) s[0] += to_f32(x[c]);
    group_sum(s, slots[0], kLongThreads / 32, 1);
    const float mean = s[0] / a.F;
    s[0] = 0.f;
    for (int c = threadIdx.x; c < a.F; c += kLongThreads) {
      const float d = to_f32(x[c]) - mean;
      s[0] = fmaf(d, d, s[0]);
    }
    group_sum(s, slots[1], kLongThreads / 32, 1);
    const float r = __frsqrt_rn(s[0] / a.F + a.eps);
    if (a.mean && threadIdx.x == 0) {
      a.mean[row] = mean;
      a.rstd[row] = r;
    }
    for (int c = threadIdx.x; c < a.F; c += kLongThreads) {
      const float w = a.w ? to_f32(static_cast<const W*>(a.w)[c]) : 1.f, b = a.b ? to_f32(static_cast<const W*>(a.b)[c]) : 0.f;
      static_cast<T*>(a.out)[row * a.F + c] = from_f32<T>(fmaf((to_f32(x[c]) - mean) * r, w, b));
    }
  }
}
template <typename T, typename W>
__global__ void __launch_bounds__(kLongThreads) norm_long_grad_kernel(const NormArgs a) {
  __shared__ __align__(16) float slots[2][32];
  int turn = 0;
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x, turn ^= 1) {
    const T *x = static_cast<const T*>(a.x) + row * a.ldx, *dy = static_cast<const T*>(a.dy) + row * a.lddy;
    const float mean = a.mean[row], r = a.rstd[row];
    float s[2] = {0.f, 0.f};
    for (int c = threadIdx.x; c < a.F; c += kLongThreads) {
      const float u = to_f32(dy[c]) * (a.w ? to_f32(static_cast<const W*>(a.w)[c]) : 1.f);
      s[0] += u;
      s[1] = fmaf(u, (to_f32(x[c]) - mean) * r, s[1]);
    }
    group_sum(s, slots[turn], kLongThreads / 32, 1);
    for (int c = threadIdx.x; c < a.F; c += kLongThreads) {
      const float u = to_f32(dy[c]) * (a.w ? to_f32(static_cast<const W*>(a.w)[c]) : 1.f);
      static_cast<T*>(a.out)[row * a.F + c] = from_f32<T>(r * (u - s[0] / a.F - (to_f32(x[c]) - mean) * r * (s[1] / a.F)));
    }
  }
}
// Column sums by themselves, where a row is too long for its threads to keep them: a warp takes 32 V columns, a CTA's eight warps every
// 8 gridDim.y-th row each.
template <typename T, int V>
__global__ void __launch_bounds__(256) norm_columns_kernel(const NormArgs a) {
  __shared__ float part[8][2][32 * V];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = (blockIdx.x * 32 + lane) * V;
  float dw[V], db[V];
#pragma unroll
  for (int j = 0; j < V; ++j) dw[j] = db[j] = 0.f;
  if (c < a.F) {
    constexpr int kDeep = 4;
    const long long stride = 8ll * gridDim.y;
    for (long long row = blockIdx.y * 8 + warp; row < a.rows; row += stride * kDeep) {
      Pack<T, V> px[kDeep], pg[kDeep];
      float r[kDeep], mean[kDeep];
#pragma unroll
      for (int d = 0; d < kDeep; ++d) {
        const long long at = row + d * stride;
        if (at >= a.rows) continue;
        px[d] = read_only<T, V>(static_cast<const T*>(a.x) + at * a.ldx + c);
        pg[d] = read_only<T, V>(static_cast<const T*>(a.dy) + at * a.lddy + c);
        r[d] = __ldg(a.rstd + at);
        mean[d] = __ldg(a.mean + at);
      }
#pragma unroll
      for (int d = 0; d < kDeep; ++d) {
        if (row + d * stride >= a.rows) continue;
        float x[V], dy[V];
        unpack<T, V>(px[d], x);
        unpack<T, V>(pg[d], dy);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          dw[j] = fmaf(dy[j], (x[j] - mean[d]) * r[d], dw[j]);
          db[j] += dy[j];
        }
      }
    }
  }
#pragma unroll
  for (int j = 0; j < V; ++j) {
    part[warp][0][lane * V + j] = dw[j];
    part[warp][1][lane * V + j] = db[j];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 64 * V; i += 256) {
    const int which = i / (32 * V), k = i - which * 32 * V, column = blockIdx.x * 32 * V + k;
    if (column >= a.F) continue;
    float s = part[0][which][k];
#pragma unroll
    for (int j = 1; j < 8; ++j) s += part[j][which][k];
    a.sums[(size_t)blockIdx.y * 2 * a.F + (size_t)which * a.F + column] = s;
  }
}

// ------------------------------------------------------------------ host side
struct NormPlan {
  int vec, values;  // values to a load and of a thread; 0 values: rows too long
  int group, block;  // threads of a row and of a CTA
  int ctas;          // of the backward pass's sums
};

constexpr int kMostSums = 592;  // rows of sums

// 16-byte loads where all rows and the weights allow it, else single values. Forward: 16 values of a thread, 8 for short or few rows, 64
// (single values: 16) where a row is too long for 256 threads.
NormPlan plan_forward(int rows, int F, int type, bool aligned16) {
  NormPlan p{};
  p.vec = aligned16 && F % (type == FS_TYPE_F32 ? 4 : 8) == 0 ? (type == FS_TYPE_F32 ? 4 : 8) : 1;
  const int few = p.vec > 1 ? 8 : 4;
  int values = 2 * few;
  if (F <= few * 32 || (rows < 148 * 4 && F <= few * 256)) values = few;
  else if (values * 256 < F) values = p.vec > 1 ? 64 : 16;
  if ((long long)values * kMaxNormThreads < F) {
    p.group = p.block = kLongThreads;
    return p;
  }
  p.values = values;
  p.group = (F + values * 32 - 1) / (values * 32) * 32;
  p.block = p.group < 256 ? 256 / p.group * p.group : p.group;
  return p;
}
// Backward: 16 values of a thread with the sums of their columns, or 8 for short rows; from 4096 values (single values: 2048) on 32 without sums.
NormPlan plan_backward(int rows, int F, int type, bool aligned16) {
  NormPlan p{};
  p.vec = aligned16 && F % (type == FS_TYPE_F32 ? 4 : 8) == 0 ? (type == FS_TYPE_F32 ? 4 : 8) : 1;
  const int most = p.vec > 1 ? 16 : 8;
  int values = p.vec > 1 ? 8 : 4;
  while (values < most && values * 32 < F) values *= 2;
  const bool keeps = values * 256 >= F;
  if (keeps) {
    p.values = values;
    p.group = (F + values * 32 - 1) / (values * 32) * 32;
    p.block = 256 / p.group * p.group;
    const long long want = ((long long)rows + p.block / p.group - 1) / (p.block / p.group), most_ctas = 2 * 148;
    p.ctas = (int)(want < most_ctas ? want : most_ctas);
    return p;
  }
  values = p.vec > 1 ? 64 : 16;
  if (values * 256 >= F) {
    p.values = values;
    p.group = p.block = (F + values * 32 - 1) / (values * 32) * 32;
  } else {
    p.group = p.block = kLongThreads;
  }
  const int across = (F + 32 * p.vec - 1) / (32 * p.vec);
  int down = (4 * 148 + across - 1) / across;
  if (down > (rows + 7) / 8) down = (rows + 7) / 8;
  p.ctas = down;
  return p;
}

template <typename K>
int allow_smem(K kernel, size_t bytes, std::atomic<uint64_t>& allowed) {
  if (bytes <= 40 * 1024) return FS_OK;  // with the static part below what needs no leave
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (e == cudaSuccess && !(allowed.load(std::memory_order_relaxed) & bit)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 220 * 1024);
    if (e == cudaSuccess) allowed.fetch_or(bit, std::memory_order_relaxed);
  }
  return e == cudaSuccess ? FS_OK : report_error(FS_ERR_CUDA, cudaGetErrorString(e));
}
template <typename T, typename W, int V, int NV, bool SUMS>
int launch_norm_grad(const NormPlan& p, const NormArgs& a, cudaStream_t st) {
  static std::atomic<uint64_t> allowed{0};
  const auto kernel = norm_grad_kernel<T, W, V, NV, SUMS>;
  const int groups = p.block / p.group, most = 148 * 2;
  const long long rows = ((long long)a.rows + groups - 1) / groups;
  size_t smem = (size_t)norm_stages(2 * NV * (int)sizeof(Pack<T, V>)) * 2 * NV * p.block * sizeof(Pack<T, V>);
  const size_t merge = (size_t)(groups - 1) * 2 * a.F * sizeof(float);
  if (SUMS && merge > smem) smem = merge;
  const int s = allow_smem(kernel, smem, allowed);
  if (s != FS_OK) return s;
  kernel<<<(unsigned)(SUMS ? p.ctas : rows < most ? rows : most), p.block, smem, st>>>(a);
  return launched(1);
}
template <typename T, typename W, int V, int NV>
int launch_forward(const NormPlan& p, const NormArgs& a, cudaStream_t st) {
  static std::atomic<uint64_t> allowed{0};
  constexpr bool kHold = V * NV <= (V > 1 ? 16 : 8);
  const int groups = p.block / p.group, most = kHold ? 3 * 148 : 8 * 148;
  const long long grid = ((long long)a.rows + groups - 1) / groups;
  const size_t smem = kHold ? (size_t)kForwardStages * NV * sizeof(Pack<T, V>) * p.block : 0;
  const int s = allow_smem(norm_kernel<T, W, V, NV>, smem, allowed);
  if (s != FS_OK) return s;
  norm_kernel<T, W, V, NV><<<(unsigned)(grid < most ? grid : most), p.block, smem, st>>>(a);
  return launched(1);
}
template <typename T, typename W, int V>
int launch_backward(const NormPlan& p, const NormArgs& a, cudaStream_t st) {
  constexpr int kShort = V > 1 ? 8 : 4, kLong = V > 1 ? 64 : 16;
  if (p.values == kLong) return a.out ? launch_norm_grad<T, W, V, kLong / V, false>(p, a, st) : FS_OK;
  if (p.values == kShort) return a.sums ? launch_norm_grad<T, W, V, kShort / V, true>(p, a, st) : launch_norm_grad<T, W, V, kShort / V, false>(p, a, st);
  return a.sums ? launch_norm_grad<T, W, V, 2 * kShort / V, true>(p, a, st) : launch_norm_grad<T, W, V, 2 * kShort / V, false>(p, a, st);
}
template <typename T, typename W>
int launch_typed(const NormPlan& p, const NormArgs& a, bool grad, cudaStream_t st) {
  constexpr int kWide = sizeof(T) == 4 ? 4 : 8;
  if (p.values == 0) {
    const int grid = a.rows < 148 * 4 ? a.rows : 148 * 4;
    if (!grad) norm_long_kernel<T, W><<<grid, kLongThreads, 0, st>>>(a);
    else if (a.out) norm_long_grad_kernel<T, W><<<grid, kLongThreads, 0, st>>>(a);
    const int s = launched(!grad || a.out ? 1 : 0);
    if (s != FS_OK || !grad) return s;
  } else if (!grad) {
    if (p.vec == 1)
      return p.values == 4 ? launch_forward<T, W, 1, 4>(p, a, st) : p.values == 8 ? launch_forward<T, W, 1, 8>(p, a, st) : launch_forward<T, W, 1, 16>(p, a, st);
    return p.values == 8    ? launch_forward<T, W, kWide, 8 / kWide>(p, a, st)
           : p.values == 16 ? launch_forward<T, W, kWide, 16 / kWide>(p, a, st)
                            : launch_forward<T, W, kWide, 64 / kWide>(p, a, st);
  } else {
    const int s = p.vec > 1 ? launch_backward<T, W, kWide>(p, a, st) : launch_backward<T, W, 1>(p, a, st);
    if (s != FS_OK || p.values < (p.vec > 1 ? 64 : 16)) return s;
  }
  if (!a.sums) return FS_OK;
  const dim3 grid((a.F + 32 * p.vec - 1) / (32 * p.vec), p.ctas);
  if (p.vec > 1) norm_columns_kernel<T, kWide><<<grid, 256, 0, st>>>(a);
  else norm_columns_kernel<T, 1><<<grid, 256, 0, st>>>(a);
  return launched(1);
}
int launch_any(const NormPlan& p, const NormArgs& a, int type, int w_type, bool grad, cudaStream_t st) {
  if (type == FS_TYPE_F32) return launch_typed<float, float>(p, a, grad, st);
  if (type == FS_TYPE_F16)
    return w_type == FS_TYPE_F32 ? launch_typed<__half, float>(p, a, grad, st) : launch_typed<__half, __half>(p, a, grad, st);
  return w_type == FS_TYPE_F32 ? launch_typed<__nv_bfloat16, float>(p, a, grad, st)
                               : launch_typed<__nv_bfloat16, __nv_bfloat16>(p, a, grad, st);
}

int check_norm(const void* x, int type, long long ldx, int rows, int F, int w_type, float eps) {
  if (type < FS_TYPE_F32 || type > FS_TYPE_BF16 || (w_type != type && w_type != FS_TYPE_F32))
    return report_error(FS_ERR_BAD_ARG, "type must be one of FS_TYPE_*, that of the weights the same or FS_TYPE_F32");
  if (rows < 0 || F < 1 || F > (1 << 24) || ldx < F || !(eps >= 0.f))
    return report_error(FS_ERR_BAD_ARG, "rows must not be negative, F in [1, 2^24], ldx at least F and eps not negative");
  if (rows > 0 && !x) return report_error(FS_ERR_BAD_ARG, "null argument");
  return check_device();
}
bool wide_rows(const void* p, long long ld, int bytes) { return aligned(p, 16) && ld * bytes % 16 == 0; }
bool wide_weights(const void* p) { return aligned(p, 16); }

}  // namespace
}  // namespace ex
}  // namespace fs

using namespace fs;
using namespace fs::ex;

extern "C" {

size_t fs_layer_norm_grad_bytes(int rows, int F) {
  if (rows < 1 || F < 1) return 0;
  return (size_t)(rows < kMostSums ? rows : kMostSums) * 2 * F * sizeof(float);
}

int fs_layer_norm(const void* x, int type, long long ldx, int rows, int F, const void* w, const void* b, int w_type, float eps,
                  void* y, float* mean, float* rstd, void* stream) {
  const int s = check_norm(x, type, ldx, rows, F, w_type, eps);
  if (s != FS_OK || rows == 0) return s;
  if (!y || !mean != !rstd) return report_error(FS_ERR_BAD_ARG, "null argument");
  const int bytes = type_bytes(type);
  NormArgs a{};
  a.x = x; a.ldx = ldx; a.w = w; a.b = b; a.out = y; a.mean = mean; a.rstd = rstd; a.rows = rows; a.F = F; a.eps = eps;
  const NormPlan p = plan_forward(rows, F, type, wide_rows(x, ldx, bytes) && aligned(y, 16) && wide_weights(w) && wide_weights(b));
  a.group = p.group;
  return launch_any(p, a, type, w_type, false, static_cast<cudaStream_t>(stream));
}

int fs_layer_norm_grad(const void* x, int type, long long ldx, int rows, int F, const void* w, int w_type, const float* mean,
                       const float* rstd, const void* dy, long long lddy, void* dx, void* dw, void* db, void* ws, size_t ws_bytes,
                       void* stream) {
  const int s = check_norm(x, type, ldx, rows, F, w_type, 0.f);
  if (s != FS_OK) return s;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (rows == 0) {
    for (void* p : {dw, db})
      if (p) {
        const cudaError_t e = cudaMemsetAsync(p, 0, (size_t)F * type_bytes(w_type), st);
        if (e != cudaSuccess) return report_error(FS_ERR_CUDA, cudaGetErrorString(e));
      }
    return FS_OK;
  }
  if (!mean || !rstd || !dy || lddy < F) return report_error(FS_ERR_BAD_ARG, "null argument, or too few columns");
  const bool sums = dw || db;
  if (!dx && !sums) return FS_OK;
  if (sums && (!ws || ws_bytes < fs_layer_norm_grad_bytes(rows, F))) return report_error(FS_ERR_WORKSPACE, "workspace too small");
  const int bytes = type_bytes(type);
  NormArgs a{};
  a.x = x; a.ldx = ldx; a.w = w; a.dy = dy; a.lddy = lddy; a.out = dx; a.rows = rows; a.F = F;
  a.mean = const_cast<float*>(mean); a.rstd = const_cast<float*>(rstd); a.sums = sums ? static_cast<float*>(ws) : nullptr;
  const NormPlan p = plan_backward(rows, F, type, wide_rows(x, ldx, bytes) && wide_rows(dy, lddy, bytes) && aligned(dx, 16) && wide_weights(w));
  a.group = p.group;
  const int r = launch_any(p, a, type, w_type, true, st);
  if (r != FS_OK || !sums) return r;
  const unsigned grid = (unsigned)((2ll * F + 31) / 32);
  if (w_type == FS_TYPE_F32) norm_sums_kernel<float><<<grid, 256, 0, st>>>(a.sums, p.ctas, F, static_cast<float*>(dw), static_cast<float*>(db));
  else if (w_type == FS_TYPE_F16) norm_sums_kernel<__half><<<grid, 256, 0, st>>>(a.sums, p.ctas, F, static_cast<__half*>(dw), static_cast<__half*>(db));
  else norm_sums_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(a.sums, p.ctas, F, static_cast<__nv_bfloat16*>(dw), static_cast<__nv_bfloat16*>(db));
  return launched(1);
}

}  // extern "C"
