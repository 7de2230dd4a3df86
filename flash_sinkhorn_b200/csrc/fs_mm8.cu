// Matrix products grouped by expert in 8-bit floating point (4 bits of exponent, 3 of mantissa), with a scale for each block of 128:
//
//   x[i, k] = sx[i, k / 128] qx[i, k],   w_e[n, k] = sw_e[n / 128, k / 128] qw_e[n, k]
//   out[i, n] = sum over blocks c of sx[i, c] sw_e[n / 128, c] (sum over k in c of qx[i, k] qw_e[n, k])
//
// and the same with w_e transposed, the gradient to x. Scales are the smallest powers of two with which a block's largest magnitude
// is at most 448, so a division by one is exact, the codes are the same wherever they are computed, and the type's exponent makes up for
// the half of its range that a power of two may leave (a value is off by half a step of its own either way).
//
// Rows go into 8 bits and into the order of the experts in one pass. In the product the ROWS of a group are the M side of the
// tensor-core instruction, so that a thread's accumulators share the row's scale. The tensor core sums one block of 128 in
// TMEM (fp32); eight warps read that while the next block is summed beside it, and add it, scaled, to sums in registers.
// Per block and 128 x 256 tile the products take 512 clocks of the tensor core, reading 256 of TMEM and adding 256 of the fp32 units, but
// each of the two accumulators goes from the tensor core to the warps of both CTAs and back, which takes some 1200 clocks by itself: a
// block takes 550 ns, where loads and products alone take 373 (from HBM 550). 65536 rows of 64 equal groups, 2048 x 2048: 300 us, 1830 TFLOP/s, against
// 390 us of the 16-bit product (groups as a routing gives them: 326; under the power cap, after half a second of calls, 15 % more); with 1024 or 4096
// contraction values 1530 and 2040 TFLOP/s (a tile costs 2 us besides its blocks). The thread that issues waits for sums for 58 % of its clocks, for loads 9.
// What decided it: registers that spill in the loop of sums (a factor 1.5), loads of 16 columns a step ahead of the additions, results by TMA, and
// in the wait for a block no more than a look: with its limit handled there in 64 bits, before the first look, the same product took 334 us.
// Accumulators and barriers of their own for the two halves of a tile cost more than they saved (695 ns a block): products of 128 columns read as much
// shared memory as it gives. So did factors read four blocks ahead.
#include "fs_experts.cuh"
#include "fs_pair.cuh"
#include "fs_tc.cuh"

#include <cuda_fp8.h>

#include <atomic>

namespace fs {
namespace ex {
long long product_limit();  // fs_group.cu: of the calling thread

namespace {

constexpr int kBlock8 = 128;  // values that share a scale
constexpr float kTop8 = 448.f;

// ------------------------------------------------------------------ into 8 bits
// Bits of the scale for a largest magnitude (float bits), and of its reciprocal; NaN and 0 for an infinity or a NaN.
__device__ __forceinline__ void scale_of(uint32_t top, float& scale, float& inverse) {
  // 448 = 1.75 * 2^8: 1.f * 2^e needs 2^(e - 8), or one more where 1.f is above 1.75
  int j = (int)(top >> 23) - 135 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
  j = max(j, -126);
  const bool finite = top < 0x7f800000u;
  scale = __uint_as_float(finite ? (uint32_t)(j + 127) << 23 : 0x7fc00000u);
  inverse = __uint_as_float(finite ? (uint32_t)(127 - j) << 23 : 0u);
}
__device__ __forceinline__ uint32_t four_codes(float a, float b, float c, float d) {
  const __nv_fp8x2_storage_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const __nv_fp8x2_storage_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return (uint32_t)lo | (uint32_t)hi << 16;
}
// Eight values from column c on of a row of K, zeros past its end; vec: aligned to 16 bytes and K a multiple of 8.
template <typename T>
__device__ __forceinline__ void eight(const T* row, int c, int K, bool vec, float (&v)[8]) {
  if (vec && c < K) {
    unpack<T, 8>(read_only<T, 8>(row + c), v);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = c + j < K ? to_f32(row[c + j]) : 0.f;
  }
}
__device__ __forceinline__ uint32_t top_of(const float (&v)[8]) {
  uint32_t m = 0u;
#pragma unroll
  for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(v[j]) & 0x7fffffffu);
  return m;
}
// `finite` false: zeros (the scale is NaN).
__device__ __forceinline__ uint2 codes_of(const float (&v)[8], float inverse) {
  if (inverse == 0.f) return make_uint2(0u, 0u);
  return make_uint2(four_codes(v[0] * inverse, v[1] * inverse, v[2] * inverse, v[3] * inverse),
                    four_codes(v[4] * inverse, v[5] * inverse, v[6] * inverse, v[7] * inverse));
}

// Sixteen values from column c on of a row of K as they are in memory, zeros past its end. VEC: rows aligned to 16 bytes, K a multiple of 8.
template <bool VEC, typename T>
__device__ __forceinline__ void sixteen(const T* row, int c, int K, uint32_t (&w)[8]) {
  if (VEC) {
    const uint4 none = make_uint4(0u, 0u, 0u, 0u);
    const uint4 p = c < K ? __ldg(reinterpret_cast<const uint4*>(row + c)) : none, q = c + 8 < K ? __ldg(reinterpret_cast<const uint4*>(row + c) + 1) : none;
    w[0] = p.x; w[1] = p.y; w[2] = p.z; w[3] = p.w;
    w[4] = q.x; w[5] = q.y; w[6] = q.z; w[7] = q.w;
  } else {
    const uint16_t* v = reinterpret_cast<const uint16_t*>(row);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t lo = c + 2 * j < K ? __ldg(v + c + 2 * j) : 0u, hi = c + 2 * j + 1 < K ? __ldg(v + c + 2 * j + 1) : 0u;
      w[j] = lo | hi << 16;
    }
  }
}
// Magnitudes of 16-bit floating-point values are ordered as whole numbers: largest ones of both halves.
__device__ __forceinline__ uint32_t top_pair(const uint32_t (&w)[8]) {
  uint32_t m = 0u;
#pragma unroll
  for (int j = 0; j < 8; j += 2) m = __vimax3_u16x2(m, w[j] & 0x7fff7fffu, w[j + 1] & 0x7fff7fffu);
  return m;
}
// The larger half of a pair as float bits.
__device__ __forceinline__ uint32_t top_bits(uint32_t m, __nv_bfloat16) { return max(m << 16, m & 0xffff0000u); }
__device__ __forceinline__ uint32_t top_bits(uint32_t m, __half) {
  return __float_as_uint(__half2float(__ushort_as_half((unsigned short)max(m & 0xffffu, m >> 16))));
}
template <typename T>
__device__ __forceinline__ uint4 sixteen_codes(const uint32_t (&w)[8], float inverse) {
  uint32_t q[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float a, b, c, d;
    two_f32(w[2 * j], a, b, T());
    two_f32(w[2 * j + 1], c, d, T());
    q[j] = four_codes(a * inverse, b * inverse, c * inverse, d * inverse);
  }
  return inverse == 0.f ? make_uint4(0u, 0u, 0u, 0u) : make_uint4(q[0], q[1], q[2], q[3]);
}

// Rows x[rows[i]] of M rows of K values (zeros for numbers outside; rows null: row i) to codes [R, ldc] and scales [ceil(K / 128)][R]. Eight lanes
// take a row, sixteen values of a block each, a CTA 32 rows of `span` blocks, so that 32 rows' scales are written side by side. ldc is a
// multiple of 16; codes past K are zeros. Instructions count as much as bytes: magnitudes are compared in pairs, as whole
// numbers (65536 gathered rows of 2048: 104 us with 8 values a lane, compared one by one, 47 us so).
constexpr int kRows8 = 32, kSpan8 = 64;
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) rows8_kernel(const T* x, long long ldx, int M, const int* rows, int R, int K, int span, uint8_t* codes, long long ldc,
                                                    float* scales) {
  __shared__ float found[kSpan8][kRows8];
  constexpr int kDeep = 4;
  const int lane = threadIdx.x & 7, r = threadIdx.x >> 3, b0 = blockIdx.y * span;
  const int blocks = min(span, (K + kBlock8 - 1) / kBlock8 - b0);
  const long long i0 = (long long)blockIdx.x * kRows8, i = i0 + r;
  const int t = i >= R ? -1 : rows ? __ldg(rows + i) : (int)i;
  const T* row = x + (long long)t * ldx;
  const int end = (unsigned)t < (unsigned)M ? K : 0;
  uint8_t* out = codes + i * ldc;
  for (int j = 0; j < blocks; j += kDeep) {
    uint32_t w[kDeep][8];
#pragma unroll
    for (int d = 0; d < kDeep; ++d) sixteen<VEC>(row, (b0 + j + d) * kBlock8 + lane * 16, j + d < blocks ? end : 0, w[d]);
#pragma unroll
    for (int d = 0; d < kDeep; ++d) {
      uint32_t m = top_pair(w[d]);
#pragma unroll
      for (int o = 4; o; o >>= 1) m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, o));
      float scale, inverse;
      scale_of(top_bits(m, T()), scale, inverse);
      const int c = (b0 + j + d) * kBlock8 + lane * 16;
      if (j + d < blocks && i < R && c < ldc) *reinterpret_cast<uint4*>(out + c) = sixteen_codes<T>(w[d], inverse);
      if (j + d < blocks && lane == 0) found[j + d][r] = scale;
    }
  }
  __syncthreads();
  for (int u = threadIdx.x; u < blocks * kRows8; u += 256) {
    const int k = u & (kRows8 - 1);
    if (i0 + k < R) scales[(long long)(b0 + u / kRows8) * R + i0 + k] = found[u / kRows8][k];
  }
}

// Weights w [E, N, K] to codes (rows c_row, matrices c_expert apart) and scales [E][ceil(N / 128)][ceil(K / 128)]: a CTA to a block of
// 128 x 128, which it holds in registers between the search for the largest magnitude and the codes. Bound by memory: 64 Mi values 30 us, 6.7 TB/s.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) weights8_kernel(const T* w, long long w_expert, long long w_row, int N, int K, uint8_t* codes, long long c_expert,
                                                       long long c_row, float* scales) {
  __shared__ uint32_t part[8];
  const int kb = (K + kBlock8 - 1) / kBlock8, nb = (N + kBlock8 - 1) / kBlock8;
  const int e = blockIdx.x / (kb * nb), rest = blockIdx.x - e * kb * nb, n0 = rest / kb * kBlock8, k0 = rest % kb * kBlock8;
  const int c = k0 + (threadIdx.x & 7) * 16, r = n0 + (threadIdx.x >> 3);
  uint32_t held[4][8], m = 0u;
#pragma unroll
  for (int i = 0; i < 4; ++i) sixteen<VEC>(w + e * w_expert + (long long)(r + 32 * i) * w_row, c, r + 32 * i < N ? K : 0, held[i]);
#pragma unroll
  for (int i = 0; i < 4; ++i) m = __vmaxu2(m, top_pair(held[i]));
  const uint32_t top = __reduce_max_sync(0xffffffffu, top_bits(m, T()));
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = top;
  __syncthreads();
  uint32_t all = part[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) all = max(all, part[i]);
  float scale, inverse;
  scale_of(all, scale, inverse);
  if (threadIdx.x == 0) scales[blockIdx.x] = scale;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (r + 32 * i < N && c < (K + 15) / 16 * 16)
      *reinterpret_cast<uint4*>(codes + e * c_expert + (long long)(r + 32 * i) * c_row + c) = sixteen_codes<T>(held[i], inverse);
}

// ------------------------------------------------------------------ products
// Warps: a warpgroup for loads and products (two of its warps idle), then two that sum. With 256 columns the sums take
// more than the 168 registers that 384 threads have each: 40 for the first group, 232 for the others (128 x 40 + 256 x 232 = 384 x 168).
constexpr int kSumWarps = 8, kFetchWarp = 0, kIssueWarp = 1, kGroupWarp = 2, kFirstSum = 4, kThreads8 = 32 * (kFirstSum + kSumWarps);
constexpr uint32_t kTileA = 128 * 128;
constexpr int kStage8 = 2 * 4096 * kSumWarps;  // staging of results, two tiles of 32 x 128 bytes for each warp

struct Mm8Args {
  const int* offsets;
  int R, E, N, K;  // K: contraction
  const float* sx;  // [ceil(K / 128)][R]
  const float* sw;
  long long sw_expert;
  int sw_n, sw_k;  // distances of scales along N and K
  void* out;
  long long ldo;
  int out_type, out_bytes;  // bytes of a store: 16, 4 or 2
  bool boxes;               // whole blocks of 32 rows are written by TMA
  int nstage;
  unsigned limit;  // clocks that the warps which sum wait for a block of products; 0: none at all
  int* health;     // non-zero once a bounded wait gave up (read by fs_device_error)
};

template <int CG>
__device__ __forceinline__ void mma_f8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if (CG == 2)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}

// Sixteen columns of the accumulators; the values are there after the wait.
__device__ __forceinline__ void read16(uint32_t at, uint32_t (&r)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
                 "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
               : "r"(at));
}
__device__ __forceinline__ void wait16(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]),
                 "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}

struct Tile8 {
  int e, n0, lo, hi, blocks;  // expert, first feature, rows of the tile, blocks of 128 contraction values (0: rows of no expert)
};
template <int BM, int BN>  // rows and features of a tile
struct Tiles8 {
  const Mm8Args& a;
  const int *gs, *ts;
  int nt, e = 0;
  __device__ Tiles8(const Mm8Args& args, const int* rows, const int* tiles) : a(args), gs(rows), ts(tiles) { nt = (a.N + BN - 1) / BN; }
  __device__ int total() const { return ts[a.E + 1]; }
  __device__ Tile8 at(int tile) {  // in increasing order
    for (int end = a.E; e < end;) {
      const int mid = (e + end) / 2;
      if (tile >= ts[mid + 1]) e = mid + 1;
      else end = mid;
    }
    const int rest = tile - ts[e], m = rest / nt;
    Tile8 t;
    t.e = e;
    t.n0 = (rest - m * nt) * BN;
    t.lo = gs[e] + m * BM;
    t.hi = min(t.lo + BM, gs[e + 1]);
    t.blocks = e < a.E ? (a.K + kBlock8 - 1) / kBlock8 : 0;
    return t;
  }
};

__device__ __forceinline__ uint32_t two16(u64 v, int type) {
  float lo, hi;
  upk(v, lo, hi);
  return type == FS_TYPE_BF16 ? from_two(lo, hi, __nv_bfloat16()) : from_two(lo, hi, __half());
}

// MN: w contiguous along N (the transposed product). Single CTAs fetch rows in boxes of 32, as many as the tile has.
template <bool MN, int CG, int BN>
__global__ void __launch_bounds__(kThreads8, 1)
mm8_kernel(const Mm8Args a, const __grid_constant__ CUtensorMap mapA, const __grid_constant__ CUtensorMap mapB, const __grid_constant__ CUtensorMap mapC) {
  constexpr int BNC = BN / CG, kBufs = BN == 256 ? 2 : 4;
  constexpr uint32_t kTileB = BNC * 128, kStage = kTileA + kTileB, kColumns = BN * kBufs;
  constexpr int kBoxA = CG == 2 ? 128 : 32;
  static_assert(kColumns <= 512 && kStage % 1024 == 0 && !(MN && BNC < 128), "tile");
  extern __shared__ uint8_t raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  uint8_t* staging = ring + (size_t)a.nstage * kStage;
  uint64_t* bars = reinterpret_cast<uint64_t*>(staging + kStage8);
  const int FULL = 0, EMPTY = a.nstage, ACC_FULL = 2 * a.nstage, ACC_EMPTY = ACC_FULL + kBufs, DRAIN = ACC_EMPTY + kBufs;
  uint32_t* slot = reinterpret_cast<uint32_t*>(bars + DRAIN + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(slot + 1);
  int *words = reinterpret_cast<int*>(slot + 2), *gs = words + 4, *ts = gs + a.E + 2;
  auto bar = [&](int i) { return smem_u32(bars + i); };

  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int rank = CG == 2 ? (int)cta_rank() : 0;
  const int first = blockIdx.x / CG, stride = gridDim.x / CG;

  if (warp == kGroupWarp) {
    read_groups<true>(a.offsets, a.E, a.R, gs, ts, (a.N + BN - 1) / BN, 128 * CG);
  } else if (warp == kFetchWarp && lane == 0) {
    for (int s = 0; s < a.nstage; ++s) {
      mbar_init(bar(FULL + s), CG);  // in CTA 0: both CTAs' loads
      mbar_init(bar(EMPTY + s), 1);
    }
    for (int i = 0; i < kBufs; ++i) {
      mbar_init(bar(ACC_FULL + i), 1);
      mbar_init(bar(ACC_EMPTY + i), kSumWarps * CG);  // in CTA 0: all warps of the pair that sum
    }
    mbar_init(bar(DRAIN), 1);
    *abort_flag = 0;
    words[0] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  } else if (warp == kIssueWarp) {
    alloc_columns<CG>(smem_u32(slot), kColumns);
  }
  tc_fence_before();
  __syncthreads();
  if (CG == 2) cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem = *slot;
  Tiles8<128 * CG, BN> tiles(a, gs, ts);
  const int total = tiles.total();
  if (warp < kFirstSum) {
    if (BN == 256) asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    // ===================== loads =====================
    if (warp == kFetchWarp && elect_one()) {
      int s = 0, issued = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int it = first; ok && it < total; it += stride) {
        const Tile8 t = tiles.at(it);
        const int boxes = CG == 2 ? 1 : (t.hi - t.lo + kBoxA - 1) / kBoxA;
        for (int kb = 0; kb < t.blocks; ++kb) {
          if (!mbar_wait(bar(EMPTY + s), ph ^ 1, abort_flag)) {
            ok = false;
            break;
          }
          const uint32_t full = CG == 2 ? in_leader(bar(FULL + s)) : bar(FULL + s), dst = smem_u32(ring + (size_t)s * kStage);
          expect_at<CG>(full, boxes * kBoxA * 128 + kTileB);
          for (int i = 0; i < boxes; ++i) load_2d<CG>(dst + i * kBoxA * 128, &mapA, kb * 128, t.lo + rank * 128 + i * kBoxA, full);
          if (MN) {
#pragma unroll
            for (int c = 0; c < BNC / 128; ++c)
              load_3d<CG>(dst + kTileA + c * kTileA, &mapB, t.n0 + rank * BNC + c * 128, kb * 128, t.e, full);
          } else {
            load_3d<CG>(dst + kTileA, &mapB, kb * 128, t.n0 + rank * BNC, t.e, full);
          }
          ++issued;
          if (++s == a.nstage) {
            s = 0;
            ph ^= 1;
          }
        }
      }
      words[0] = issued;
    }
    // ===================== products =====================
    if (warp == kIssueWarp && rank == 0 && elect_one()) {
      // fp32 sums, both operands e4m3 (0)
      constexpr uint32_t idesc = (1u << 4) | ((MN ? 1u : 0u) << 16) | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(128 * CG >> 4) << 24);
      // a step of 32 contraction values: 32 bytes on, or 32 rows of 128 bytes; MN: the next 128 features one tile on
      constexpr uint32_t kStepB = (MN ? 32u * 128u : 32u) >> 4, kLeadB = MN ? kTileA >> 4 : 1u;
      int s = 0, buf = 0;
      uint32_t ph = 0, acc_ph = 0;
      bool ok = true;
      for (int it = first; ok && it < total; it += stride) {
        const Tile8 t = tiles.at(it);
        for (int kb = 0; kb < t.blocks; ++kb) {
          if (!mbar_wait(bar(ACC_EMPTY + buf), acc_ph ^ 1, abort_flag) || !mbar_wait(bar(FULL + s), ph, abort_flag)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t base = smem_u32(ring + (size_t)s * kStage);
          const uint32_t al = desc_lo(base), bl = (((base + kTileA) & 0x3FFFFu) >> 4) | (kLeadB << 16);
          const int left = a.K - kb * kBlock8;
#pragma unroll
          for (int ks = 0; ks < 4; ++ks)
            if (ks * 32 < left)
              mma_f8<CG>(tmem + buf * BN, pack_desc(al + ks * 2, kDescHi128), pack_desc(bl + ks * kStepB, kDescHi128), idesc, ks);
          commit<CG>(bar(EMPTY + s));
          commit<CG>(bar(ACC_FULL + buf));
          if (++s == a.nstage) {
            s = 0;
            ph ^= 1;
          }
          if (++buf == kBufs) {
            buf = 0;
            acc_ph ^= 1;
          }
        }
      }
    }
  } else {
    // ===================== sums and results =====================
    if (BN == 256) asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
    // Two warps to a quarter of the TMEM lanes (rows), with one half of the features each.
    constexpr int kMine = BN / 2;
    const int q = warp & 3, side = (warp - kFirstSum) >> 2;
    const uint32_t stages = smem_u32(staging + 8192 * (warp - kFirstSum));
    int buf = 0;
    uint32_t acc_ph = 0;
    bool lost = a.limit == 0;  // a wait of this CTA gave up: NaN from here on
    if (lost) *abort_flag = 1;
    uint32_t stage = stages;
    auto release = [&](bool whole) {  // the next staging tile: by the copy before last, or by all if no copy follows from this one
      if (a.boxes) {
        stage = stages + (stage == stages ? 4096 : 0);
        if (lane == 0) {
          if (whole) bulk_read<1>();
          else bulk_read<0>();
        }
        __syncwarp();
      }
    };
    auto send = [&](int n, int row) {
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) store_box(&mapC, n, row, stage);
    };
    // The tile after this one and its first factors are looked up before this one's results are written.
    const float *sx = a.sx, *sw = a.sw;
    float x_next = 0.f, w_next = 0.f;
    Tile8 next = {};
    auto look = [&](int it) {
      if (it >= total) return;
      next = tiles.at(it);
      sx = a.sx + min(next.lo + rank * 128 + q * 32 + lane, a.R - 1);
      sw = a.sw + next.e * a.sw_expert + (long long)min(next.n0 + side * kMine, a.N - 1) / kBlock8 * a.sw_n;
      if (next.blocks) {
        x_next = __ldg(sx);
        w_next = __ldg(sw);
      }
    };
    look(first);
    for (int it = first; it < total; it += stride) {
      const Tile8 t = next;
      const int row0 = t.lo + rank * 128 + q * 32, n0 = t.n0 + side * kMine;
      u64 sum[kMine / 2];
#pragma unroll
      for (int i = 0; i < kMine / 2; ++i) sum[i] = 0ull;
      for (int kb = 0; kb < t.blocks && !lost; ++kb) {
        const float f = x_next * w_next;
        if (kb + 1 < t.blocks) {
          x_next = __ldg(sx + (long long)(kb + 1) * a.R);
          w_next = __ldg(sw + (long long)(kb + 1) * a.sw_k);
        }
        lost = !__all_sync(0xffffffffu, wait_close(bar(ACC_FULL + buf), acc_ph, abort_flag, a.limit));
        if (lost) break;
        tc_fence_after();
        const u64 f2 = pk(f, f);
        const uint32_t acc = tmem + buf * BN + side * kMine + ((uint32_t)(q * 32) << 16);
        uint32_t r[2][16];  // 16 columns are on their way while the ones before them are added
        read16(acc, r[0]);
#pragma unroll
        for (int j = 0; j < kMine / 16; ++j) {
          wait16(r[j & 1]);
          if (j + 1 < kMine / 16) {
            read16(acc + 16 * (j + 1), r[(j + 1) & 1]);
          } else {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
              if (CG == 2) arrive_cluster(in_leader(bar(ACC_EMPTY + buf)));
              else mbar_arrive(bar(ACC_EMPTY + buf));
            }
          }
#pragma unroll
          for (int i = 0; i < 8; ++i)
            sum[8 * j + i] = fma2(pk(__uint_as_float(r[j & 1][2 * i]), __uint_as_float(r[j & 1][2 * i + 1])), f2, sum[8 * j + i]);
        }
        if (++buf == kBufs) {
          buf = 0;
          acc_ph ^= 1;
        }
      }
      look(it + stride);
      if (lost && t.blocks) {
        const float nan = __uint_as_float(0x7fc00000u);
#pragma unroll
        for (int i = 0; i < kMine / 2; ++i) sum[i] = pk(nan, nan);
      }
      const int rows = t.hi - row0;
      if (rows <= 0) continue;
      const int width = a.out_type == FS_TYPE_F32 ? 4 : 2;
      char* out = static_cast<char*>(a.out) + (long long)row0 * a.ldo * width;
      const bool whole = a.boxes && rows >= 32;  // the rows behind the last one are another tile's
      // 128 bytes of each row at a time
      const int at16 = kMine < 64 ? kMine : 64;
      if (a.out_type != FS_TYPE_F32) {
#pragma unroll
        for (int j = 0; j < kMine; j += at16) {
          if (n0 + j >= a.N) break;
          release(whole);
#pragma unroll
          for (int c = 0; c < at16 / 8; ++c)
            stage16(staged_row(stage, lane, c), two16(sum[j / 2 + 4 * c], a.out_type), two16(sum[j / 2 + 4 * c + 1], a.out_type),
                    two16(sum[j / 2 + 4 * c + 2], a.out_type), two16(sum[j / 2 + 4 * c + 3], a.out_type));
          if (whole) {
            send(n0 + j, row0);
          } else {
            __syncwarp();
            write_rows(out + 2ll * (n0 + j), a.ldo * 2, rows, 2 * min(a.N - n0 - j, at16), a.out_bytes, stage, lane);
            __syncwarp();
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < kMine; j += 32) {
          if (n0 + j >= a.N) break;
          release(whole);
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            float v[4];
            upk(sum[j / 2 + 2 * c], v[0], v[1]);
            upk(sum[j / 2 + 2 * c + 1], v[2], v[3]);
            stage16(staged_row(stage, lane, c), __float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
          }
          if (whole) {
            send(n0 + j, row0);
          } else {
            __syncwarp();
            write_rows(out + 4ll * (n0 + j), a.ldo * 4, rows, 4 * min(a.N - n0 - j, 32), a.out_bytes, stage, lane);
            __syncwarp();
          }
        }
      }
    }
    if (a.boxes && lane == 0) bulk_done();
  }
  settle<CG, 1>(abort_flag, words, bar(FULL), bar(DRAIN), a.nstage, warp == kIssueWarp, warp == kFetchWarp);
  if (warp == kIssueWarp) free_columns<CG>(tmem, kColumns);
  if (threadIdx.x == 0 && *abort_flag) atomicExch(a.health, 1);
}

// ------------------------------------------------------------------ short groups
// Groups of up to a few dozen rows are bound by reading their weights. Here the FEATURES are the M side and the rows N, as in the
// 16-bit products: a stage is 16 KB of weights and 4 KB of rows, an accumulator kShortRows columns, of which 256 / kShortRows are in use in turn, so that the
// tensor core does not wait for the sums. Two CTAs to an SM: one's first loads of a tile hide behind the other one's products. 64 experts of 2048 x 1024
// with two rows each: 28 us, 4.8 TB/s, some 8 of them launch, first loads and the last, partly filled round; twice the features 49 us, 5.4 TB/s.
constexpr int kShortRows = 32;                                       // of a tile: a lane's factor is that of one
constexpr int kShortThreads = 192, kShortFetch = 4, kShortIssue = 5;  // four warps that sum
constexpr size_t kShortSmem = 112 * 1024;                            // two fit an SM, and no kernel of this library beside one: they take 120 KB

__global__ void __launch_bounds__(kShortThreads, 2)
mm8_short_kernel(const Mm8Args a, const __grid_constant__ CUtensorMap mapW, const __grid_constant__ CUtensorMap mapX) {
  constexpr uint32_t kStage = kTileA + kShortRows * 128, kColumns = 256;
  constexpr int kBufs = kColumns / kShortRows, kAhead = 4;
  static_assert(kBufs % 2 == 0, "buffers of factors");
  extern __shared__ uint8_t raw[];
  __shared__ __align__(16) float factors[4][2][kShortRows];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(ring + (size_t)a.nstage * kStage);
  const int FULL = 0, EMPTY = a.nstage, ACC_FULL = 2 * a.nstage, ACC_EMPTY = ACC_FULL + kBufs, DRAIN = ACC_EMPTY + kBufs;
  uint32_t* slot = reinterpret_cast<uint32_t*>(bars + DRAIN + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(slot + 1);
  int *words = reinterpret_cast<int*>(slot + 2), *gs = words + 4, *ts = gs + a.E + 2;
  auto bar = [&](int i) { return smem_u32(bars + i); };
  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int first = blockIdx.x, stride = gridDim.x;

  if (warp == 0) {
    read_groups<true>(a.offsets, a.E, a.R, gs, ts, (a.N + 127) / 128, kShortRows);
  } else if (warp == kShortFetch && lane == 0) {
    for (int s = 0; s < 2 * a.nstage + 2 * kBufs + 1; ++s) mbar_init(bar(s), s >= ACC_EMPTY && s < DRAIN ? 4 : 1);
    *abort_flag = 0;
    words[0] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  } else if (warp == kShortIssue) {
    alloc_columns<1>(smem_u32(slot), kColumns);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *slot;
  Tiles8<kShortRows, 128> tiles(a, gs, ts);
  const int total = tiles.total();

  if (warp == kShortFetch) {
    // ===================== loads =====================
    if (elect_one()) {
      int s = 0, issued = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int it = first; ok && it < total; it += stride) {
        const Tile8 t = tiles.at(it);
        for (int kb = 0; kb < t.blocks; ++kb) {
          if (!mbar_wait(bar(EMPTY + s), ph ^ 1, abort_flag)) {
            ok = false;
            break;
          }
          const uint32_t full = bar(FULL + s), dst = smem_u32(ring + (size_t)s * kStage);
          mbar_expect_tx(full, kStage);
          load_3d<1>(dst, &mapW, kb * 128, t.n0, t.e, full);
          tma_load_2d(dst + kTileA, &mapX, kb * 128, t.lo, full);
          ++issued;
          if (++s == a.nstage) {
            s = 0;
            ph ^= 1;
          }
        }
      }
      words[0] = issued;
    }
  } else if (warp == kShortIssue) {
    // ===================== products =====================
    if (elect_one()) {
      int s = 0, buf = 0;
      uint32_t ph = 0, acc_ph = 0;
      bool ok = true;
      for (int it = first; ok && it < total; it += stride) {
        const Tile8 t = tiles.at(it);
        const uint32_t idesc = (1u << 4) | ((uint32_t)((t.hi - t.lo + 15) / 16 * 2) << 17) | ((uint32_t)(128 >> 4) << 24);
        for (int kb = 0; kb < t.blocks; ++kb) {
          if (!mbar_wait(bar(ACC_EMPTY + buf), acc_ph ^ 1, abort_flag) || !mbar_wait(bar(FULL + s), ph, abort_flag)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t base = smem_u32(ring + (size_t)s * kStage), al = desc_lo(base), bl = desc_lo(base + kTileA);
          const int left = a.K - kb * kBlock8;
#pragma unroll
          for (int ks = 0; ks < 4; ++ks)
            if (ks * 32 < left) mma_f8<1>(tmem + buf * kShortRows, pack_desc(al + ks * 2, kDescHi128), pack_desc(bl + ks * 2, kDescHi128), idesc, ks);
          commit<1>(bar(EMPTY + s));
          commit<1>(bar(ACC_FULL + buf));
          if (++s == a.nstage) {
            s = 0;
            ph ^= 1;
          }
          if (++buf == kBufs) {
            buf = 0;
            acc_ph ^= 1;
          }
        }
      }
    }
  } else {
    // ===================== sums and results =====================
    // A lane has a feature; the rows' factors, a lane's for its row, are read four blocks ahead and handed round in shared memory.
    int buf = 0;
    uint32_t acc_ph = 0;
    bool lost = a.limit == 0;  // a wait of this CTA gave up: NaN from here on
    if (lost) *abort_flag = 1;
    float xs[kAhead], ws[kAhead];
    const float *sx = a.sx, *sw = a.sw;
    Tile8 next = {};
    auto ask = [&](int kb, int d) {
      if (kb >= next.blocks) return;
      xs[d] = next.lo + lane < next.hi ? __ldg(sx + (long long)kb * a.R) : 0.f;
      ws[d] = __ldg(sw + (long long)kb * a.sw_k);
    };
    auto look = [&](int it) {
      if (it >= total) return;
      next = tiles.at(it);
      sx = a.sx + next.lo + lane;
      sw = a.sw + next.e * a.sw_expert + (long long)(next.n0 / kBlock8) * a.sw_n;
#pragma unroll
      for (int d = 0; d < kAhead; ++d) ask(d, d);
    };
    look(first);
    for (int it = first; it < total; it += stride) {
      const Tile8 t = next;
      u64 sum[kShortRows / 2];
#pragma unroll
      for (int i = 0; i < kShortRows / 2; ++i) sum[i] = 0ull;
      for (int k0 = 0; k0 < t.blocks; k0 += kAhead)
#pragma unroll
        for (int d = 0; d < kAhead; ++d) {
          if (k0 + d >= t.blocks || lost) continue;
          // Two buffers in turn, from tile to tile too (kBufs is even): every lane has passed the other buffer's barrier, behind its last read of
          // this one, before any writes here again.
          float* mine = factors[warp][buf & 1];
          mine[lane] = xs[d] * ws[d];
          ask(k0 + d + kAhead, d);
          __syncwarp();
          lost = !__all_sync(0xffffffffu, wait_close(bar(ACC_FULL + buf), acc_ph, abort_flag, a.limit));
          if (lost) continue;
          tc_fence_after();
#pragma unroll
          for (int j = 0; j < kShortRows / 16; ++j) {
            uint32_t r[16];
            read16(tmem + buf * kShortRows + 16 * j + ((uint32_t)(warp * 32) << 16), r);
            wait16(r);
            if (j + 1 == kShortRows / 16) {
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(bar(ACC_EMPTY + buf));
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float4 f = *reinterpret_cast<const float4*>(mine + 16 * j + 4 * i);
              sum[8 * j + 2 * i] = fma2(pk(__uint_as_float(r[4 * i]), __uint_as_float(r[4 * i + 1])), pk(f.x, f.y), sum[8 * j + 2 * i]);
              sum[8 * j + 2 * i + 1] = fma2(pk(__uint_as_float(r[4 * i + 2]), __uint_as_float(r[4 * i + 3])), pk(f.z, f.w), sum[8 * j + 2 * i + 1]);
            }
          }
          if (++buf == kBufs) {
            buf = 0;
            acc_ph ^= 1;
          }
        }
      look(it + stride);
      const int f = t.n0 + warp * 32 + lane, rows = t.hi - t.lo;
      if (f >= a.N) continue;
#pragma unroll
      for (int j = 0; j < kShortRows; ++j) {
        float lo, hi;
        upk(sum[j / 2], lo, hi);
        const float v = lost && t.blocks ? __uint_as_float(0x7fc00000u) : j & 1 ? hi : lo;
        if (j < rows) {
          const long long at = (long long)(t.lo + j) * a.ldo + f;
          if (a.out_type == FS_TYPE_F32) static_cast<float*>(a.out)[at] = v;
          else if (a.out_type == FS_TYPE_BF16) static_cast<__nv_bfloat16*>(a.out)[at] = from_f32<__nv_bfloat16>(v);
          else static_cast<__half*>(a.out)[at] = from_f32<__half>(v);
        }
      }
    }
  }
  settle<1, 1>(abort_flag, words, bar(FULL), bar(DRAIN), a.nstage, warp == kShortIssue, warp == kShortFetch);
  if (warp == kShortIssue) free_columns<1>(tmem, kColumns);
  if (threadIdx.x == 0 && *abort_flag) atomicExch(a.health, 1);
}

// ------------------------------------------------------------------ few rows
// A single token: bound by launch and latency beside its experts' weights, so a warp takes one feature of one expert, 16 codes a lane and load, as the
// 16-bit products do. Each CTA puts the rows into 8 bits itself, which takes less than a launch that does it once. Two rows of two experts, 2048 x 2048: 6.7 us.
constexpr int kFewRows8 = 2, kFewWarps8 = 8, kFewMost8 = 8192;  // rows; contraction values that shared memory takes

// Shared memory of a row: what its codes stand for as fp16 (exact), padded to 128, and their scales.
__host__ __device__ constexpr size_t few8_row_bytes(int blocks) { return ((size_t)blocks * (2 * kBlock8 + 4) + 15) / 16 * 16; }
__device__ __forceinline__ uint32_t two_of_codes(uint32_t pair) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(pair & 0xffffu), __NV_E4M3);
  return (uint32_t)h.x | (uint32_t)h.y << 16;
}
template <typename T, int ROWS>
__global__ void __launch_bounds__(32 * kFewWarps8, 4)
few8_kernel(const Mm8Args a, const T* x0, long long ldx, int M, const int* rows, const uint8_t* w, long long w_expert, long long w_row, bool vec) {
  __shared__ int first_after[2];
  extern __shared__ __align__(16) uint8_t held[];
  const int lane = threadIdx.x & 31, i = blockIdx.y, blocks = (a.K + kBlock8 - 1) / kBlock8;
  // The rows' first blocks are on their way while the expert is looked for, its weights while the rows are put into 8 bits.
  constexpr int kEarly = 2;
  const size_t row_bytes = few8_row_bytes(blocks);
  float early[kEarly][8];
  int from[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) from[r] = i + r < a.R ? (rows ? __ldg(rows + i + r) : i + r) : -1;
  auto fetch = [&](int u, float (&v)[8]) {
    const int r = u / blocks, b = u - r * blocks, n = ROWS > 1 && r ? from[ROWS - 1] : from[0];
    const bool in = u < ROWS * blocks && (unsigned)n < (unsigned)M;
    eight(x0 + (in ? n : 0) * ldx, in ? b * kBlock8 + (threadIdx.x & 15) * 8 : a.K, a.K, vec, v);
  };
#pragma unroll
  for (int k = 0; k < kEarly; ++k) fetch((threadIdx.x >> 4) + 2 * kFewWarps8 * k, early[k]);
  // The expert of row i is the one before the first offset above i (offsets as their running maximum); a row whose
  // predecessor has the same one is left to the CTA of the expert's first row.
  if (threadIdx.x < 2) first_after[threadIdx.x] = a.E + 1;
  __syncthreads();
  int above = a.E + 1, reached = a.E + 1;  // first offset above row i, above row i - 1
  for (int j = 1 + threadIdx.x; j <= a.E; j += 32 * kFewWarps8) {
    const int v = a.offsets[j];
    if (v > i) above = min(above, j);
    if (v >= i) reached = min(reached, j);
  }
  above = __reduce_min_sync(0xffffffffu, above);
  reached = __reduce_min_sync(0xffffffffu, reached);
  if (lane == 0) {
    atomicMin(&first_after[0], above);
    atomicMin(&first_after[1], reached);
  }
  __syncthreads();
  const int e = first_after[0] - 1, f = blockIdx.x * kFewWarps8 + (threadIdx.x >> 5);
  auto store = [&](int row, float v) {
    const long long at = (long long)row * a.ldo + f;
    if (a.out_type == FS_TYPE_F32) static_cast<float*>(a.out)[at] = v;
    else static_cast<T*>(a.out)[at] = from_f32<T>(v);
  };
  if (e == a.E) {  // a row of no expert
    if (lane == 0 && f < a.N) store(i, 0.f);
    return;
  }
  if (i > 0 && first_after[1] == first_after[0]) return;
  const int end = min(a.offsets[e + 1], a.R);
  const uint8_t* wf = w + e * w_expert + min(f, a.N - 1) * w_row;
  const float* sw = a.sw + e * a.sw_expert + (long long)(min(f, a.N - 1) / kBlock8) * a.sw_n;
  constexpr int kDeep = 4;
  const int chunks = (a.K + 15) / 16;
  uint4 q[kDeep];
  float s[kDeep];
  auto ask = [&](int c0) {
#pragma unroll
    for (int d = 0; d < kDeep; ++d) {
      const int c = c0 + 32 * d;
      if (c >= chunks) continue;
      if (16 * c + 16 <= a.K) {
        q[d] = __ldg(reinterpret_cast<const uint4*>(wf + 16 * c));
      } else {  // what lies past the row's end is not read
        uint32_t part[4] = {};
        for (int k = 16 * c; k < a.K; ++k) part[(k >> 2) & 3] |= (uint32_t)wf[k] << (8 * (k & 3));
        q[d] = make_uint4(part[0], part[1], part[2], part[3]);
      }
      s[d] = __ldg(sw + (long long)(c >> 3) * a.sw_k);
    }
  };
  ask(lane);
  const int units = min(ROWS, end - i) * blocks;  // of rows of this expert
  auto hold = [&](int u, const float (&v)[8]) {
    const int r = u / blocks, b = u - r * blocks, l = threadIdx.x & 15;
    uint32_t top = top_of(v);
#pragma unroll
    for (int o = 8; o; o >>= 1) top = max(top, __shfl_xor_sync(0xffffu << (threadIdx.x & 16), top, o));
    float scale, inverse;
    scale_of(top, scale, inverse);
    if (u >= units) return;
    const uint2 c = codes_of(v, inverse);
    *reinterpret_cast<uint4*>(held + r * row_bytes + 2 * (b * kBlock8 + l * 8)) =
        make_uint4(two_of_codes(c.x), two_of_codes(c.x >> 16), two_of_codes(c.y), two_of_codes(c.y >> 16));
    if (l == 0) *reinterpret_cast<float*>(held + r * row_bytes + 2 * blocks * kBlock8 + 4 * b) = scale;
  };
#pragma unroll
  for (int k = 0; k < kEarly; ++k)
    if ((threadIdx.x >> 4 & ~1) + 2 * kFewWarps8 * k < units) hold((threadIdx.x >> 4) + 2 * kFewWarps8 * k, early[k]);
  for (int u = (threadIdx.x >> 4) + 2 * kFewWarps8 * kEarly; u < units; u += 2 * kFewWarps8) {
    float v[8];
    fetch(u, v);
    hold(u, v);
  }
  __syncthreads();
  if (f >= a.N) return;
  float sums[ROWS] = {};
#pragma unroll 1
  for (int c0 = lane; c0 < chunks; c0 += 32 * kDeep) {
    if (c0 != lane) ask(c0);
#pragma unroll
    for (int d = 0; d < kDeep; ++d) {
      const int c = c0 + 32 * d;
      if (c >= chunks) continue;
      const uint32_t wq[4] = {q[d].x, q[d].y, q[d].z, q[d].w};
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        if (r > 0 && i + r >= end) continue;
        const uint4 p0 = *reinterpret_cast<const uint4*>(held + r * row_bytes + 32 * c), p1 = *reinterpret_cast<const uint4*>(held + r * row_bytes + 32 * c + 16);
        const uint32_t xh[8] = {p0.x, p0.y, p0.z, p0.w, p1.x, p1.y, p1.z, p1.w};
        float t = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          float w0, w1, x0, x1;
          two_f32(two_of_codes(wq[j / 2] >> (16 * (j & 1))), w0, w1, __half());
          two_f32(xh[j], x0, x1, __half());
          t = fmaf(w1, x1, fmaf(w0, x0, t));
        }
        sums[r] = fmaf(t, s[d] * *reinterpret_cast<const float*>(held + r * row_bytes + 2 * blocks * kBlock8 + 4 * (c >> 3)), sums[r]);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
#pragma unroll
    for (int o = 16; o; o >>= 1) sums[r] += __shfl_xor_sync(0xffffffffu, sums[r], o);
    if (lane == r && i + r < end) store(i + r, sums[r]);
  }
}

// ------------------------------------------------------------------ host side
// 8-bit tensor of 2 or 3 dimensions, contiguous along the first; boxes of 128 x box_rows.
bool encode8(CUtensorMap* map, const void* base, int dims, const long long (&size)[3], const long long (&stride)[2], int box_rows) {
  const cuuint64_t sizes[3] = {(cuuint64_t)size[0], (cuuint64_t)size[1], (cuuint64_t)size[2]};
  const cuuint64_t strides[2] = {(cuuint64_t)stride[0], (cuuint64_t)stride[1]};
  const cuuint32_t box[3] = {128, (cuuint32_t)box_rows, 1}, ones[3] = {1, 1, 1};
  const auto fn = encoder();
  return fn && fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, dims, const_cast<void*>(base), sizes, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Results of R rows; boxes of 32 rows of 128 bytes.
bool encode_out(CUtensorMap* map, int type, void* base, long long cols, long long rows, long long ld) {
  const int width = type_bytes(type);
  const cuuint64_t sizes[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)(ld * width)};
  const cuuint32_t box[2] = {(cuuint32_t)(128 / width), 32}, ones[2] = {1, 1};
  const auto fn = encoder();
  return fn && fn(map, type == FS_TYPE_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : type == FS_TYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                  2, base, sizes, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <bool MN, int CG, int BN>
int launch_mm8(Mm8Args a, const uint8_t* x, long long ldx, const uint8_t* w, long long w_expert, long long w_row, cudaStream_t st) {
  CUtensorMap mapA = {}, mapB = {}, mapC = {};
  const int width = type_bytes(a.out_type);
  a.boxes = BN >= 128 && aligned(a.out, 16) && a.ldo * width % 16 == 0;  // a warp has 128 bytes of a row
  // w's own rows and columns: K and N change places in the transposed product
  const long long w_cols = MN ? a.N : a.K, w_rows = MN ? a.K : a.N;
  if (!encode8(&mapA, x, 2, {a.K, a.R, 1}, {ldx, 0}, CG == 2 ? 128 : 32) ||
      !encode8(&mapB, w, 3, {w_cols, w_rows, a.E}, {w_row, w_expert ? w_expert : w_row}, MN ? 128 : BN / CG) ||
      (a.boxes && !encode_out(&mapC, a.out_type, a.out, a.N, a.R, a.ldo)))
    return report_error(FS_ERR_CUDA, "cuTensorMapEncodeTiled failed");
  constexpr size_t kStage = kTileA + BN / CG * 128;
  const size_t fixed = 1024 + kStage8 + 8 * (2 * 12 + 9) + 24 + 8 * ((size_t)a.E + 2);
  a.nstage = (int)((kSmemMax - fixed) / kStage);
  if (a.nstage > 12) a.nstage = 12;
  size_t smem = fixed + a.nstage * kStage;
  if (smem < (size_t)kSmemMin) smem = kSmemMin;
  const auto kernel = mm8_kernel<MN, CG, BN>;
  static std::atomic<uint64_t> allowed{0};  // devices on which the kernel may take all shared memory
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (e == cudaSuccess && !(allowed.load(std::memory_order_relaxed) & bit)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMax);
    if (e == cudaSuccess) allowed.fetch_or(bit, std::memory_order_relaxed);
  }
  if (e != cudaSuccess) return report_error(FS_ERR_CUDA, cudaGetErrorString(e));
  const long long most = ((a.R + 128ll * CG - 1) / (128 * CG) + a.E + 1) * ((a.N + BN - 1) / BN);
  if (most > 0x3fffffffll) return report_error(FS_ERR_UNSUPPORTED, "more than 2^30 tiles");
  long long grid = detail::free_ctas() / CG;
  if (grid > most) grid = most;
  if (grid < 1) grid = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)grid * CG);
  cfg.blockDim = dim3(kThreads8);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = CG;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  a.health = products_health();
  if (!a.health) return report_error(FS_ERR_CUDA, "cannot find the health word of the current CUDA device");
  e = cudaLaunchKernelEx(&cfg, kernel, a, mapA, mapB, mapC);
  if (e != cudaSuccess) return report_error(FS_ERR_CUDA, cudaGetErrorString(e));
  count_launches(1);
  return FS_OK;
}

int launch_short8(Mm8Args a, const uint8_t* x, long long ldx, const uint8_t* w, long long w_expert, long long w_row, cudaStream_t st) {
  CUtensorMap mapW = {}, mapX = {};
  if (!encode8(&mapW, w, 3, {a.K, a.N, a.E}, {w_row, w_expert ? w_expert : w_row}, 128) || !encode8(&mapX, x, 2, {a.K, a.R, 1}, {ldx, 0}, kShortRows))
    return report_error(FS_ERR_CUDA, "cuTensorMapEncodeTiled failed");
  constexpr size_t kStage = kTileA + kShortRows * 128, kStatic = 4 * 2 * kShortRows * sizeof(float);
  const size_t fixed = 1024 + 8 * (2 * 8 + 2 * (256 / kShortRows) + 1) + 24 + 8 * ((size_t)a.E + 2);
  a.nstage = (int)((kShortSmem - kStatic - fixed) / kStage);
  static_assert((kShortSmem - kStatic - 1024 - 8 * 33 - 24 - 8 * 1026) / kStage >= 4 && (kShortSmem / kStage) <= 8, "stages");
  const auto kernel = mm8_short_kernel;
  static std::atomic<uint64_t> allowed{0};  // devices on which the kernel may take that much shared memory
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (e == cudaSuccess && !(allowed.load(std::memory_order_relaxed) & bit)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(kShortSmem - kStatic));
    if (e == cudaSuccess) allowed.fetch_or(bit, std::memory_order_relaxed);
  }
  if (e != cudaSuccess) return report_error(FS_ERR_CUDA, cudaGetErrorString(e));
  const long long most = ((a.R + kShortRows - 1ll) / kShortRows + a.E + 1) * ((a.N + 127) / 128);
  if (most > 0x3fffffffll) return report_error(FS_ERR_UNSUPPORTED, "more than 2^30 tiles");
  // two to an SM; one, where SMs are to stay free: the second ones would go to those
  long long grid = detail::free_ctas() * (detail::free_ctas() == detail::sm_count() ? 2ll : 1ll);
  if (grid > most) grid = most;
  if (grid < 1) grid = 1;
  a.health = products_health();
  if (!a.health) return report_error(FS_ERR_CUDA, "cannot find the health word of the current CUDA device");
  kernel<<<(unsigned)grid, kShortThreads, kShortSmem - kStatic, st>>>(a, mapW, mapX);
  return launched(1);
}

template <typename T>
int launch_rows8(const void* x, long long ldx, int M, const int* rows, int R, int K, uint8_t* codes, long long ldc, float* scales, cudaStream_t st) {
  const int blocks = (K + kBlock8 - 1) / kBlock8, over = (R + kRows8 - 1) / kRows8;
  int span = kSpan8;
  while (span > 1 && (long long)over * ((blocks + span - 1) / span) < 4 * 148) span /= 2;
  const bool vec = aligned(x, 16) && ldx % 8 == 0 && K % 8 == 0;
  const dim3 grid(over, (blocks + span - 1) / span);
  const T* xt = static_cast<const T*>(x);
  if (vec) rows8_kernel<T, true><<<grid, 256, 0, st>>>(xt, ldx, M, rows, R, K, span, codes, ldc, scales);
  else rows8_kernel<T, false><<<grid, 256, 0, st>>>(xt, ldx, M, rows, R, K, span, codes, ldc, scales);
  return launched(1);
}
template <typename T>
int launch_few8(const Mm8Args& a, const void* x, long long ldx, int M, const int* rows, const uint8_t* w, long long w_expert, long long w_row, cudaStream_t st) {
  const dim3 grid((a.N + kFewWarps8 - 1) / kFewWarps8, a.R);
  const size_t smem = a.R * few8_row_bytes((a.K + kBlock8 - 1) / kBlock8);
  const bool vec = aligned(x, 16) && ldx % 8 == 0 && a.K % 8 == 0;
  const T* xt = static_cast<const T*>(x);
  if (a.R == 1) few8_kernel<T, 1><<<grid, 32 * kFewWarps8, smem, st>>>(a, xt, ldx, M, rows, w, w_expert, w_row, vec);
  else few8_kernel<T, 2><<<grid, 32 * kFewWarps8, smem, st>>>(a, xt, ldx, M, rows, w, w_expert, w_row, vec);
  return launched(1);
}

bool few8(int R, int K, bool transposed) { return R <= kFewRows8 && K <= kFewMost8 && !transposed; }
long long ldc_of(int K) { return ((long long)K + 15) / 16 * 16; }
size_t codes_bytes(int R, int K) { return ((size_t)R * ldc_of(K) + 255) / 256 * 256; }

int check8(int R, int E, int N, int K) {
  if (R < 0 || R > 0x7fffffff - 511 || E < 1 || E > 1024 || N < 1 || K < 1 || N > (1 << 22) || K > (1 << 22))
    return report_error(FS_ERR_BAD_ARG, "R must be in [0, 2^31 - 512], E in [1, 1024], N and K in [1, 2^22]");
  // A thread that has launched nothing yet (autograd's) has no current context, which the encoding of tensor maps needs;
  // setting the device that is current binds it.
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaSetDevice(dev) != cudaSuccess)
    return report_error(FS_ERR_CUDA, "cannot make the current CUDA device's context current");
  return check_device();
}
bool is16(int type) { return type == FS_TYPE_F16 || type == FS_TYPE_BF16; }

}  // namespace
}  // namespace ex
}  // namespace fs

using namespace fs;
using namespace fs::ex;

extern "C" {

int fs_weights8(const void* w, int type, long long w_expert, long long w_row, int E, int N, int K, uint8_t* codes, long long c_expert, long long c_row,
                float* scales, void* stream) {
  const int s = check8(0, E, N, K);
  if (s != FS_OK) return s;
  if (!is16(type)) return report_error(FS_ERR_BAD_ARG, "type must be FS_TYPE_F16 or FS_TYPE_BF16");
  if (!w || !codes || !scales || w_row < K || w_expert < 0 || c_row < K || c_row % 16 || c_expert % 16 || c_expert < 0 || (E > 1 && c_expert < c_row * N) || !aligned(codes, 16))
    return report_error(FS_ERR_BAD_ARG, "null argument, or rows or experts that overlap or are not a multiple of 16 codes apart");
  const long long grid = (long long)E * ((N + kBlock8 - 1) / kBlock8) * ((K + kBlock8 - 1) / kBlock8);
  if (grid > 0x7fffffffll) return report_error(FS_ERR_UNSUPPORTED, "too many blocks of 128 x 128 values");
  const bool vec = aligned(w, 16) && w_row % 8 == 0 && w_expert % 8 == 0 && K % 8 == 0;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto go = [&](auto* p) {
    if (vec) weights8_kernel<std::remove_const_t<std::remove_pointer_t<decltype(p)>>, true><<<(unsigned)grid, 256, 0, st>>>(p, w_expert, w_row, N, K, codes, c_expert, c_row, scales);
    else weights8_kernel<std::remove_const_t<std::remove_pointer_t<decltype(p)>>, false><<<(unsigned)grid, 256, 0, st>>>(p, w_expert, w_row, N, K, codes, c_expert, c_row, scales);
  };
  if (type == FS_TYPE_F16) go(static_cast<const __half*>(w));
  else go(static_cast<const __nv_bfloat16*>(w));
  return launched(1);
}

size_t fs_grouped_mm8_bytes(int R, int K, int transposed) {
  if (R < 1 || K < 1 || few8(R, K, transposed != 0)) return 0;
  return codes_bytes(R, K) + (size_t)R * ((K + kBlock8 - 1) / kBlock8) * sizeof(float);
}

int fs_grouped_mm8(const void* x, int type, long long ldx, int M, const int* rows, int R, const uint8_t* w, long long w_expert,
                   long long w_row, const float* scales, int E, int N, int K, int transposed, const int* offsets, void* out,
                   int out_type, long long ldo, void* ws, size_t ws_bytes, void* stream) {
  int s = check8(R, E, N, K);
  if (s != FS_OK || R == 0) return s;
  if (!is16(type) || (out_type != type && out_type != FS_TYPE_F32))
    return report_error(FS_ERR_BAD_ARG, "type must be FS_TYPE_F16 or FS_TYPE_BF16, the result's the same or FS_TYPE_F32");
  if (!x || !w || !scales || !offsets || !out || ldx < K || ldo < N || M < 1 || M > 0x7fffffff - 511 || (!rows && M < R))
    return report_error(FS_ERR_BAD_ARG, "null argument, or too few or too many rows or columns");
  const int w_cols = transposed ? N : K, w_rows = transposed ? K : N;
  if (w_row < w_cols || w_row % 16 || w_expert % 16 || w_expert < 0 || (E > 1 && w_expert == 0) || !aligned(w, 16))
    return report_error(FS_ERR_BAD_ARG, "rows and experts of w must be a multiple of 16 codes apart and not overlap, the first one aligned to 16 bytes");
  Mm8Args a{};
  a.offsets = offsets; a.R = R; a.E = E; a.N = N; a.K = K; a.out = out; a.ldo = ldo; a.out_type = out_type;
  a.sw = scales;
  const long long across = (w_cols + kBlock8 - 1) / kBlock8, down = (w_rows + kBlock8 - 1) / kBlock8;
  if (across * down > 0x7fffffffll) return report_error(FS_ERR_UNSUPPORTED, "too many blocks of 128 x 128 values");
  a.sw_expert = across * down; a.sw_n = transposed ? 1 : (int)across; a.sw_k = transposed ? (int)across : 1;
  a.limit = close_limit(product_limit());
  const int width = type_bytes(out_type);
  a.out_bytes = aligned(out, 16) && ldo * width % 16 == 0 && (long long)N * width % 16 == 0 ? 16
                : aligned(out, 4) && ldo * width % 4 == 0 && (long long)N * width % 4 == 0  ? 4 : 2;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (few8(R, K, transposed != 0))
    return type == FS_TYPE_F16 ? launch_few8<__half>(a, x, ldx, M, rows, w, w_expert, w_row, st)
                               : launch_few8<__nv_bfloat16>(a, x, ldx, M, rows, w, w_expert, w_row, st);
  if (!ws || ws_bytes < fs_grouped_mm8_bytes(R, K, transposed)) return report_error(FS_ERR_WORKSPACE, "workspace too small");
  if (!aligned(ws, 256)) return report_error(FS_ERR_BAD_ARG, "workspace must be aligned to 256 bytes");
  uint8_t* codes = static_cast<uint8_t*>(ws);
  float* sx = reinterpret_cast<float*>(codes + codes_bytes(R, K));
  a.sx = sx;
  const long long ldc = ldc_of(K);
  s = type == FS_TYPE_F16 ? launch_rows8<__half>(x, ldx, M, rows, R, K, codes, ldc, sx, st)
                          : launch_rows8<__nv_bfloat16>(x, ldx, M, rows, R, K, codes, ldc, sx, st);
  if (s != FS_OK) return s;
  // Up to 40 rows in a mean group its weights' bytes decide, and tiles of 32 rows with the features as M read them fastest; pairs of CTAs pay where
  // there are tiles of 256 x 256 for all of them, half of every group's last one empty, and a mean group fills one. us with short tiles, 128 x 128 and
  // 256 x 256: 64 experts 2048 -> 1024, 2 rows each 29, 34, -; 32 experts of 48 rows 24, 22, 31; 64 of 64 rows 44, 40, -; of 128 rows -, 44, 55; 32 of 160 rows,
  // 1024 -> 2048 -, 35, 34; 32 of 200 rows, 2048 x 2048 -, 64, 54; one of 1024 rows, 1024 x 1024 -, 8.1, 11.6.
  const long long tiles = ((R + 255ll) / 256 + (E < R ? E : R) / 2) * ((N + 255) / 256);
  const bool pairs = tiles * 2 > detail::free_ctas() && N > 128;
  // The transposed product has no short tiles; its pairs pay from 144 rows on. us with 128 x 128 and 256 x 256, sizes of groups as a skewed routing gives them
  // (equal ones up to 48): 64 experts, 1024 -> 2048, 2 rows 45, 59; 48 rows 47, 64; 80 rows 54, 67; 130 rows 68, 73; 160 rows 75, 74; 200 rows 88, 80;
  // 128 experts, 2048 -> 1024, 16 rows 76, 92; 100 rows 108, 110; 145 rows 132, 123; 200 rows 168, 143.
  if (transposed) {
    if (pairs && R / E >= 144) return launch_mm8<true, 2, 256>(a, codes, ldc, w, w_expert, w_row, st);
    return launch_mm8<true, 1, 128>(a, codes, ldc, w, w_expert, w_row, st);
  }
  if (R / E <= 40) return launch_short8(a, codes, ldc, w, w_expert, w_row, st);
  if (pairs && R / E >= 160) return launch_mm8<false, 2, 256>(a, codes, ldc, w, w_expert, w_row, st);
  return launch_mm8<false, 1, 128>(a, codes, ldc, w, w_expert, w_row, st);
}

}  // extern "C"
