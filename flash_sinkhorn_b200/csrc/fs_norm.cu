// Layer norm of rows of F values and its gradients:
//
//   m = sum x / F,  v = sum (x - m)^2 / F,  r = 1 / sqrt(v + eps),  n = (x - m) r,  y = n w + b
//   dx = r (u - mean(u) - n mean(u n)),  u = w dy;   dw = sum over rows of dy n,  db = sum over rows of dy
//
// Both passes are bound by memory: x is read and y written, then x and dy read and dx written. A row lies in the registers of
// a group of warps (the mean first, then the squares of the differences from it: one read, and no cancellation), groups walk
// over the rows with the next row's loads under way, and in the backward pass each thread adds what its columns contribute
// to dw and db over all its rows. A CTA leaves one row of sums, which a second launch adds in a fixed order, so every run gives
// the same bits. Sums are fp32; y, dx, dw and db are rounded once.
#include "fs_experts.cuh"

namespace fs {
namespace ex {
namespace {

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

// The sum over a group's warps of one or two values, the same bits in every thread; slot: 2 x 16 floats of this group that the
// call before this one did not use.
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
  for (int i = 0; i < N; ++i) v[i] = warp_sum(lane < warps ? slot[16 * i + lane] : 0.f);
}

// N values of w or b (null: `other`) from column c on, of which those past F count as 0.
template <typename W, int V>
__device__ __forceinline__ void columns(const void* p, int c, int F, float other, float (&v)[V]) {
  if (c >= F) {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = 0.f;
  } else if (!p) {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = other;
  } else {
    unpack<W, V>(read_only<W, V>(static_cast<const W*>(p) + c), v);
  }
}

// One row per group of a.group threads, V values to a load, NV loads a thread. V > 1: rows, weights and F are aligned to it.
template <typename T, typename W, int V, int NV>
__global__ void __launch_bounds__(kMaxNormThreads) norm_kernel(const NormArgs a) {
  constexpr bool kHold = V * NV <= 16;  // w and b stay in registers
  __shared__ float slots[2][16][32];
  const int groups = blockDim.x / a.group, g = threadIdx.x / a.group, t = threadIdx.x % a.group, warps = a.group / 32;
  float w[kHold ? NV : 1][V], b[kHold ? NV : 1][V];
  if (kHold)
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      columns<W, V>(a.w, (i * a.group + t) * V, a.F, 1.f, w[i]);
      columns<W, V>(a.b, (i * a.group + t) * V, a.F, 0.f, b[i]);
    }
  const float per = 1.f / a.F;
  Pack<T, V> next[NV];
  auto load = [&](long long row) {
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * a.group + t) * V;
      if (c < a.F) next[i] = read_only<T, V>(x + c);
    }
  };
  const long long stride = (long long)gridDim.x * groups;
  long long row = (long long)blockIdx.x * groups + g;
  if (row < a.rows) load(row);
  for (; row < a.rows; row += stride) {
    float x[NV][V], s[1] = {0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      unpack<T, V>(next[i], x[i]);
      const bool in = (i * a.group + t) * V < a.F;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        x[i][j] = in ? x[i][j] : 0.f;
        s[0] += x[i][j];
      }
    }
    if (row + stride < a.rows) load(row + stride);
    group_sum(s, slots[0][g], warps, 1 + g);
    const float mean = s[0] * per;
    s[0] = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const bool in = (i * a.group + t) * V < a.F;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        x[i][j] -= mean;
        s[0] = in ? fmaf(x[i][j], x[i][j], s[0]) : s[0];
      }
    }
    group_sum(s, slots[1][g], warps, 1 + g);
    const float r = 1.f / sqrtf(fmaf(s[0], per, a.eps));
    if (a.mean && t == 0) {
      a.mean[row] = mean;
      a.rstd[row] = r;
    }
    T* out = static_cast<T*>(a.out) + row * a.F;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * a.group + t) * V;
      if (!kHold) {
        columns<W, V>(a.w, c, a.F, 1.f, w[0]);
        columns<W, V>(a.b, c, a.F, 0.f, b[0]);
      }
#pragma unroll
      for (int j = 0; j < V; ++j) x[i][j] = fmaf(x[i][j] * r, w[kHold ? i : 0][j], b[kHold ? i : 0][j]);
      if (c < a.F) store_f32<T, V>(out + c, x[i]);
    }
  }
}

// The gradients, from mean and rstd as the forward pass left them.
template <typename T, typename W, int V, int NV>
__global__ void __launch_bounds__(kMaxNormThreads) norm_grad_kernel(const NormArgs a) {
  constexpr bool kHold = V * NV <= 16;
  __shared__ float slots[2][16][32];
  extern __shared__ float merge[];  // [groups - 1][2][F]
  const int groups = blockDim.x / a.group, g = threadIdx.x / a.group, t = threadIdx.x % a.group, warps = a.group / 32;
  float w[kHold ? NV : 1][V], dw[NV][V], db[NV][V];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (kHold) columns<W, V>(a.w, (i * a.group + t) * V, a.F, 1.f, w[i]);
#pragma unroll
    for (int j = 0; j < V; ++j) dw[i][j] = db[i][j] = 0.f;
  }
  const float per = 1.f / a.F;
  Pack<T, V> nx[NV], ng[NV];
  float nmean = 0.f, nr = 0.f;
  auto load = [&](long long row) {
    const T *x = static_cast<const T*>(a.x) + row * a.ldx, *dy = static_cast<const T*>(a.dy) + row * a.lddy;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * a.group + t) * V;
      if (c < a.F) {
        nx[i] = read_only<T, V>(x + c);
        ng[i] = read_only<T, V>(dy + c);
      }
    }
    nmean = __ldg(a.mean + row);
    nr = __ldg(a.rstd + row);
  };
  const long long stride = (long long)gridDim.x * groups;
  long long row = (long long)blockIdx.x * groups + g;
  if (row < a.rows) load(row);
  for (int turn = 0; row < a.rows; row += stride, turn ^= 1) {
    Pack<T, V> qx[NV], qg[NV];
    const float mean = nmean, r = nr;
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      qx[i] = nx[i];
      qg[i] = ng[i];
    }
    if (row + stride < a.rows) load(row + stride);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * a.group + t) * V;
      float x[V], dy[V];
      unpack<T, V>(qx[i], x);
      unpack<T, V>(qg[i], dy);
      if (!kHold) columns<W, V>(a.w, c, a.F, 1.f, w[0]);
      if (c < a.F)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float n = (x[j] - mean) * r, u = dy[j] * w[kHold ? i : 0][j];
          s[0] += u;
          s[1] = fmaf(u, n, s[1]);
          dw[i][j] = fmaf(dy[j], n, dw[i][j]);
          db[i][j] += dy[j];
        }
    }
    group_sum(s, slots[turn][g], warps, 1 + g);
    const float m1 = s[0] * per, m2 = s[1] * per;
    T* out = static_cast<T*>(a.out) + row * a.F;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * a.group + t) * V;
      float x[V], dy[V];
      unpack<T, V>(qx[i], x);
      unpack<T, V>(qg[i], dy);
      if (!kHold) columns<W, V>(a.w, c, a.F, 1.f, w[0]);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float n = (x[j] - mean) * r;
        x[j] = r * (fmaf(dy[j], w[kHold ? i : 0][j], -m1) - n * m2);
      }
      if (c < a.F && a.out) store_f32<T, V>(out + c, x);
    }
  }
  if (!a.sums) return;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = (i * a.group + t) * V + j;
      if (g > 0 && c < a.F) {
        merge[(size_t)(g - 1) * 2 * a.F + c] = dw[i][j];
        merge[(size_t)(g - 1) * 2 * a.F + a.F + c] = db[i][j];
      }
    }
  __syncthreads();
  if (g > 0) return;
  float* sums = a.sums + (size_t)blockIdx.x * 2 * a.F;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = (i * a.group + t) * V + j;
      if (c < a.F) {
        for (int k = 0; k < groups - 1; ++k) {
          dw[i][j] += merge[(size_t)k * 2 * a.F + c];
          db[i][j] += merge[(size_t)k * 2 * a.F + a.F + c];
        }
        sums[c] = dw[i][j];
        sums[a.F + c] = db[i][j];
      }
    }
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
  __shared__ float slots[2][32];
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
    const float r = 1.f / sqrtf(s[0] / a.F + a.eps);
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
  __shared__ float slots[2][32];
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
// Column sums of long rows: a CTA takes 256 columns and every gridDim.y-th row.
template <typename T>
__global__ void __launch_bounds__(256) norm_columns_kernel(const NormArgs a) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= a.F) return;
  float dw = 0.f, db = 0.f;
#pragma unroll 4
  for (long long row = blockIdx.y; row < a.rows; row += gridDim.y) {
    const float dy = to_f32(static_cast<const T*>(a.dy)[row * a.lddy + c]);
    dw = fmaf(dy, (to_f32(static_cast<const T*>(a.x)[row * a.ldx + c]) - a.mean[row]) * a.rstd[row], dw);
    db += dy;
  }
  float* sums = a.sums + (size_t)blockIdx.y * 2 * a.F;
  sums[c] = dw;
  sums[a.F + c] = db;
}

// ------------------------------------------------------------------ host side
struct NormPlan {
  int vec, loads;    // values to a load, loads of a thread; 0: rows too long
  int group, block;  // threads of a row and of a CTA
  int ctas;          // of the backward pass, each leaving sums
};

constexpr int kCtasOfSums = 296;

// 16-byte loads where all rows and the weights allow it, else single values.
NormPlan plan_norm(int rows, int F, int type, int w_type, bool aligned16) {
  NormPlan p{};
  const int wide = type == FS_TYPE_F32 ? 4 : 8;
  p.vec = aligned16 && F % wide == 0 ? wide : 1;
  const int per = p.vec > 1 ? 8 / p.vec * p.vec : 4;  // values of a thread, as few as one row in 512 threads allows
  int values = per;
  while (values <= (p.vec > 1 ? 32 : 16) && (long long)values * kMaxNormThreads < F) values *= 2;
  if (values > (p.vec > 1 ? 32 : 16)) {
    p.loads = 0;
    p.vec = 1;
    p.group = p.block = kLongThreads;
    p.ctas = rows < kCtasOfSums ? rows : kCtasOfSums;
    return p;
  }
  p.loads = values / p.vec;
  p.group = (F + values * 32 - 1) / (values * 32) * 32;
  const int groups = kMaxNormThreads / p.group;
  p.block = p.group * (groups > 8 ? 8 : groups);
  const long long want = ((long long)rows + p.block / p.group - 1) / (p.block / p.group);
  p.ctas = want < kCtasOfSums ? (int)want : kCtasOfSums;
  (void)w_type;
  return p;
}

template <typename T, typename W, int V, int NV>
int launch_norm(const NormPlan& p, const NormArgs& a, bool grad, cudaStream_t st) {
  const int groups = p.block / p.group;
  if (!grad) {
    long long grid = ((long long)a.rows + groups - 1) / groups;
    if (grid > 148 * 4) grid = 148 * 4;
    norm_kernel<T, W, V, NV><<<(unsigned)grid, p.block, 0, st>>>(a);
  } else {
    const size_t smem = a.sums ? (size_t)(groups - 1) * 2 * a.F * 4 : 0;
    norm_grad_kernel<T, W, V, NV><<<p.ctas, p.block, smem, st>>>(a);
  }
  return launched(1);
}
template <typename T, typename W>
int launch_typed(const NormPlan& p, const NormArgs& a, bool grad, cudaStream_t st) {
  constexpr int kWide = sizeof(T) == 4 ? 4 : 8;
  if (p.loads == 0) {
    const int grid = a.rows < 148 * 4 ? a.rows : 148 * 4;
    if (!grad) {
      norm_long_kernel<T, W><<<grid, kLongThreads, 0, st>>>(a);
      return launched(1);
    }
    if (a.out) norm_long_grad_kernel<T, W><<<grid, kLongThreads, 0, st>>>(a);
    int s = a.out ? launched(1) : FS_OK;
    if (s == FS_OK && a.sums) {
      norm_columns_kernel<T><<<dim3((a.F + 255) / 256, p.ctas), 256, 0, st>>>(a);
      s = launched(1);
    }
    return s;
  }
  const int values = p.vec * p.loads;
  if (p.vec == 1) {
    if (values == 4) return launch_norm<T, W, 1, 4>(p, a, grad, st);
    if (values == 8) return launch_norm<T, W, 1, 8>(p, a, grad, st);
    return launch_norm<T, W, 1, 16>(p, a, grad, st);
  }
  if (values == 8) return launch_norm<T, W, kWide, 8 / kWide>(p, a, grad, st);
  if (values == 16) return launch_norm<T, W, kWide, 16 / kWide>(p, a, grad, st);
  return launch_norm<T, W, kWide, 32 / kWide>(p, a, grad, st);
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
  return (size_t)(rows < kCtasOfSums ? rows : kCtasOfSums) * 2 * F * sizeof(float);
}

int fs_layer_norm(const void* x, int type, long long ldx, int rows, int F, const void* w, const void* b, int w_type, float eps,
                  void* y, float* mean, float* rstd, void* stream) {
  const int s = check_norm(x, type, ldx, rows, F, w_type, eps);
  if (s != FS_OK || rows == 0) return s;
  if (!y || !mean != !rstd) return report_error(FS_ERR_BAD_ARG, "null argument");
  const int bytes = type_bytes(type);
  NormArgs a{};
  a.x = x; a.ldx = ldx; a.w = w; a.b = b; a.out = y; a.mean = mean; a.rstd = rstd; a.rows = rows; a.F = F; a.eps = eps;
  const NormPlan p = plan_norm(rows, F, type, w_type, wide_rows(x, ldx, bytes) && aligned(y, 16) && wide_weights(w) && wide_weights(b));
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
  const NormPlan p = plan_norm(rows, F, type, w_type, wide_rows(x, ldx, bytes) && wide_rows(dy, lddy, bytes) && aligned(dx, 16) && wide_weights(w));
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
