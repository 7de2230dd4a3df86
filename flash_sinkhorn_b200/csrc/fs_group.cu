// Matrix products grouped by expert, with groups of any size.
#include "fs_experts.cuh"

namespace fs {
namespace ex {
namespace {

constexpr int kTile = 64, kDepth = 16;

struct GroupArgs {
  const void* x;  // forward: the rows; gradient to the weights: the rows that give the columns of dw
  long long ldx;
  int M;
  const int* rows;
  const void* y;  // gradient to the weights: the rows that give the rows of dw
  long long ldy;
  int My;
  const int* yrows;
  const void* w;
  long long w_expert, w_row, w_col;
  void* out;
  long long ldo;
  int R, E, N, K;
  const int* offsets;
};

// Group and first row of row tile `tile`; rows of no expert come last, as group E.
__device__ bool find_tile(const GroupArgs& a, int tile, int& e, int& lo, int& hi) {
  int end = 0;
  for (e = 0; e <= a.E; ++e) {
    const int begin = end;
    end = e < a.E ? max(begin, min(a.offsets[e + 1], a.R)) : a.R;
    const int tiles = (end - begin + kTile - 1) / kTile;
    if (tile < tiles) {
      lo = begin + tile * kTile;
      hi = end;
      return true;
    }
    tile -= tiles;
  }
  return false;
}

template <typename T>
__device__ __forceinline__ float row_value(const void* base, long long ld, int M, const int* rows, int i, int c, int width) {
  const int r = rows ? rows[i] : i;
  return r >= 0 && r < M && c < width ? to_f32(static_cast<const T*>(base)[(long long)r * ld + c]) : 0.f;
}

// 64 x 64 outputs per CTA, 4 x 4 per thread, fp32 throughout.
template <typename T>
__global__ void __launch_bounds__(256) group_rows_kernel(const GroupArgs a) {
  __shared__ float xs[kDepth][kTile + 1], ws[kDepth][kTile + 1];
  int e, lo, hi;
  if (!find_tile(a, blockIdx.y, e, lo, hi)) return;
  const int n0 = blockIdx.x * kTile, tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  float acc[4][4] = {};
  if (e < a.E) {
    const T* w = static_cast<const T*>(a.w) + e * a.w_expert;
    for (int k0 = 0; k0 < a.K; k0 += kDepth) {
      for (int i = threadIdx.x; i < kTile * kDepth; i += 256) {
        const int r = i / kDepth, c = i % kDepth, k = k0 + c;
        xs[c][r] = lo + r < hi ? row_value<T>(a.x, a.ldx, a.M, a.rows, lo + r, k, a.K) : 0.f;
        ws[c][r] = n0 + r < a.N && k < a.K ? to_f32(w[(n0 + r) * a.w_row + k * a.w_col]) : 0.f;
      }
      __syncthreads();
      for (int c = 0; c < kDepth; ++c)
        for (int i = 0; i < 4; ++i)
          for (int j = 0; j < 4; ++j) acc[i][j] += xs[c][ty * 4 + i] * ws[c][tx * 4 + j];
      __syncthreads();
    }
  }
  T* out = static_cast<T*>(a.out);
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j)
      if (lo + ty * 4 + i < hi && n0 + tx * 4 + j < a.N)
        out[(long long)(lo + ty * 4 + i) * a.ldo + n0 + tx * 4 + j] = from_f32<T>(acc[i][j]);
}

template <typename T>
__global__ void __launch_bounds__(256) group_weights_kernel(const GroupArgs a) {
  __shared__ float ys[kDepth][kTile + 1], xs[kDepth][kTile + 1];
  const int e = blockIdx.z, n0 = blockIdx.y * kTile, c0 = blockIdx.x * kTile, tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  int lo = 0, hi = 0;
  for (int g = 0; g <= e; ++g) {
    lo = hi;
    hi = max(lo, min(a.offsets[g + 1], a.R));
  }
  float acc[4][4] = {};
  for (int r0 = lo; r0 < hi; r0 += kDepth) {
    for (int i = threadIdx.x; i < kTile * kDepth; i += 256) {
      const int r = i / kTile, c = i % kTile;
      ys[r][c] = r0 + r < hi ? row_value<T>(a.y, a.ldy, a.My, a.yrows, r0 + r, n0 + c, a.N) : 0.f;
      xs[r][c] = r0 + r < hi ? row_value<T>(a.x, a.ldx, a.M, a.rows, r0 + r, c0 + c, a.K) : 0.f;
    }
    __syncthreads();
    for (int r = 0; r < kDepth; ++r)
      for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) acc[i][j] += ys[r][ty * 4 + i] * xs[r][tx * 4 + j];
    __syncthreads();
  }
  T* out = static_cast<T*>(a.out) + (long long)e * a.N * a.K;
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j)
      if (n0 + ty * 4 + i < a.N && c0 + tx * 4 + j < a.K)
        out[(long long)(n0 + ty * 4 + i) * a.K + c0 + tx * 4 + j] = from_f32<T>(acc[i][j]);
}

int check_group(int type, int R, int E, int N, int K, const int* offsets) {
  if (type != FS_TYPE_F16 && type != FS_TYPE_BF16) return report_error(FS_ERR_BAD_ARG, "type must be FS_TYPE_F16 or FS_TYPE_BF16");
  if (R < 0 || E < 1 || E > 1024 || N < 1 || K < 1 || N > (1 << 22) || K > (1 << 22))
    return report_error(FS_ERR_BAD_ARG, "R must be >= 0, E in [1, 1024], N and K in [1, 2^22]");
  if (!offsets) return report_error(FS_ERR_BAD_ARG, "null argument");
  return check_device();
}

}  // namespace
}  // namespace ex
}  // namespace fs

using namespace fs;
using namespace fs::ex;

extern "C" {

int fs_grouped_mm(const void* x, long long ldx, int M, const int* rows, int R, const void* w, long long w_expert,
                  long long w_row, long long w_col, int E, int N, int K, const int* offsets, void* out, long long ldo,
                  int type, void* stream) {
  int s = check_group(type, R, E, N, K, offsets);
  if (s != FS_OK || R == 0) return s;
  if (!x || !w || !out || ldx < K || ldo < N || M < 0 || (!rows && M < R)) return report_error(FS_ERR_BAD_ARG, "null argument, or too few rows or columns");
  GroupArgs a{};
  a.x = x; a.ldx = ldx; a.M = M; a.rows = rows; a.R = R; a.w = w; a.w_expert = w_expert; a.w_row = w_row; a.w_col = w_col;
  a.E = E; a.N = N; a.K = K; a.offsets = offsets; a.out = out; a.ldo = ldo;
  const dim3 grid((N + kTile - 1) / kTile, (R + kTile - 1) / kTile + E + 1);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (type == FS_TYPE_F16) group_rows_kernel<__half><<<grid, 256, 0, st>>>(a);
  else group_rows_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(a);
  return launched(1);
}

int fs_grouped_mm_wgrad(const void* dy, long long lddy, int M_dy, const int* dy_rows, const void* x, long long ldx, int M_x,
                        const int* x_rows, int R, int E, int N, int K, const int* offsets, void* dw, int type,
                        void* stream) {
  int s = check_group(type, R, E, N, K, offsets);
  if (s != FS_OK) return s;
  if (!dw || (R > 0 && (!dy || !x)) || lddy < N || ldx < K || M_dy < 0 || M_x < 0 || (!dy_rows && M_dy < R) || (!x_rows && M_x < R))
    return report_error(FS_ERR_BAD_ARG, "null argument, or too few rows or columns");
  GroupArgs a{};
  a.y = dy; a.ldy = lddy; a.My = M_dy; a.yrows = dy_rows; a.x = x; a.ldx = ldx; a.M = M_x; a.rows = x_rows;
  a.R = R; a.E = E; a.N = N; a.K = K; a.offsets = offsets; a.out = dw;
  const dim3 grid((K + kTile - 1) / kTile, (N + kTile - 1) / kTile, E);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (type == FS_TYPE_F16) group_weights_kernel<__half><<<grid, 256, 0, st>>>(a);
  else group_weights_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(a);
  return launched(1);
}

}  // extern "C"
