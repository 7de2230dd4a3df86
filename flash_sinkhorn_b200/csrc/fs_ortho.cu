// Orthogonal updates: for each matrix G of a stack, with n = its smaller dimension as rows (a tall matrix is worked on transposed),
//
//   X = G / (|G| + eps)  (|.|: Frobenius),   then in every step   A = X X^T,  P = b A + c A A,  X <- a X + P X
//
// which maps each singular value s to a s + b s^3 + c s^5 and leaves the singular vectors: a chain of matrix products.
//
// Operands are fp16, sums fp32 (TMEM). A step multiplies the parts along small singular values by a = 3.4 or so, 485 over five steps, and
// with them whatever roundings left there: with bf16 operands a matrix with decaying singular values comes out 7 % off,
// with fp16 ones 1 %. So X is held as a sum of two fp16 values: the products take the upper one, and a X, which is what
// carries the small parts on, is of both (22 bits); the roundings of the products come in with b s^2 and c s^4 only, 0.02 to
// 0.2 % for those matrices, below the rounding of a bf16 result. X is held times 2^8, A and P times 2^10, so that small entries
// keep their bits: entries of X up to 255 and of P up to 63 in magnitude fit.
//
// A and P are symmetric: only tiles on and below the diagonal are computed, and written twice, unless there is a CTA for every tile: writing
// twice takes 0.5 us then, the other tiles nothing (one matrix of 512 x 512: 106.5 -> 100.5 us). The products are batched over the
// stack; tiles of 256 x 256 by pairs of CTAs, or 128 x 128 or 128 x 64 by single ones where there are too few. Small matrices go through all
// products in one launch.
//
// 32 matrices of 2048 x 1024, five steps: 1410 us on the device, of which squares and X take 115, a step's A 75, P 46 and P X 139 (the last one, without X's
// lower part, 124); the products' floors are 52, 26 and 83 at the burst rate of the tensor cores. A call takes 1480 us, and 1690 after half a second of them,
// under the power cap (1.3 GHz). Without the cap the tensor pipe is busy for 48 (A), 34 (P), 48 (P X) and 56 % (without the lower part) of the time;
// the thread that issues waits for loads for 46, 38, 36 and 25 % of its clocks and for the writers of results for 1, 6, 18 and 17 %: a partly filled
// round of tiles (4.3 rounds of A and P count as 5) and X's lower part, 540 MB through HBM in each P X but the last. One matrix of 512 x 512: a call
// 82 us, 72 in 15 products of 4.8 each, of which 2.2 are loads (a CTA's 192 KB, at most 60 bytes a clock), 0.8 the results and 1.5 the CTAs' meeting.
#include "fs_experts.cuh"
#include "fs_pair.cuh"
#include "fs_tc.cuh"

#include <atomic>

namespace fs {
namespace ex {
long long product_limit();  // fs_group.cu: of the calling thread

namespace {

constexpr float kXScale = 256.f, kAScale = 1024.f;  // X and A are held times these
// X goes without its lower part once what is left of the steps multiplies a rounding along small singular values by no more than this: with the default
// coefficients before the last step, which leaves 3.4 roundings of 2e-4 in the mean, 0.07 %. At 16, before the last two, matrices that have
// such directions came out 0.15 to 0.28 % off, as much as a bf16 result's own rounding.
constexpr float kFewTimes = 4.f;
constexpr int kNormParts = 64;                      // CTAs that sum the squares of a matrix

// ------------------------------------------------------------------ X = G / |G|
// Sums of squares in 64 bits: those of 32-bit values would overflow from 2^64 on. V values to a load.
template <typename T, int V>
__global__ void __launch_bounds__(256) squares_kernel(const T* g, long long g_matrix, long long g_row, int rows, int cols, double* parts) {
  __shared__ double warp_sums[8];
  const T* m = g + blockIdx.y * g_matrix;
  const int lane = threadIdx.x & 31;
  double s = 0.0;
  for (int r = blockIdx.x * 8 + (threadIdx.x >> 5); r < rows; r += gridDim.x * 8) {  // a warp to a row
    const T* row = m + (long long)r * g_row;
    constexpr int kDeep = 4;
    for (int c0 = lane * V; c0 < cols; c0 += 32 * V * kDeep) {
      Pack<T, V> p[kDeep];
#pragma unroll
      for (int d = 0; d < kDeep; ++d)
        if (c0 + 32 * V * d < cols) p[d] = read_only<T, V>(row + c0 + 32 * V * d);
#pragma unroll
      for (int d = 0; d < kDeep; ++d) {
        float v[V];
        unpack<T, V>(p[d], v);
        if (c0 + 32 * V * d < cols)
#pragma unroll
          for (int j = 0; j < V; ++j) s = fma((double)v[j], (double)v[j], s);
      }
    }
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (lane == 0) warp_sums[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 8; ++w) s += warp_sums[w];
    parts[blockIdx.y * gridDim.x + blockIdx.x] = s;
  }
}
// Tiles of 64 x 64 of G to both parts of X, transposed for a tall G; X [n, k], rows ldx apart. V values to a load of G.
template <typename T, int V>
__global__ void __launch_bounds__(256) begin_kernel(const T* g, long long g_matrix, long long g_row, int rows, int cols, const double* parts, int count,
                                                    float eps, bool tall, __half* hi, __half* lo, long long ldx, unsigned* meeting) {
  __shared__ float tile[64][65], factor;
  if (blockIdx.x + blockIdx.y + blockIdx.z + threadIdx.x == 0) *meeting = 0u;
  const int b = blockIdx.z, r0 = blockIdx.y * 64, c0 = blockIdx.x * 64;
  constexpr int kLanes = 64 / V;  // to a row of the tile
#pragma unroll
  for (int y = threadIdx.x / kLanes; y < 64; y += 256 / kLanes) {
    const int r = r0 + y, x = threadIdx.x % kLanes * V;
    float v[V];
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = 0.f;
    if (r < rows && c0 + x < cols) unpack<T, V>(read_only<T, V>(g + b * g_matrix + (long long)r * g_row + c0 + x), v);
#pragma unroll
    for (int j = 0; j < V; ++j) tile[y][x + j] = v[j];
  }
  if (threadIdx.x < 32) {  // one warp: square roots of 64 bits are dear
    double s = 0.0;
    for (int i = threadIdx.x; i < count; i += 32) s += parts[b * count + i];
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (threadIdx.x == 0) factor = (float)((double)kXScale / (sqrt(s) + (double)eps));
  }
  __syncthreads();
  const float f = factor;
  const int n = tall ? cols : rows, k = tall ? rows : cols, n0 = tall ? c0 : r0, k0 = tall ? r0 : c0;
#pragma unroll
  for (int y = threadIdx.x >> 3; y < 64; y += 32) {
    const int row = n0 + y, x = (threadIdx.x & 7) * 8, col = k0 + x;
    if (row >= n || col >= k) continue;
    uint32_t h[4], l[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float v0 = (tall ? tile[x + 2 * j][y] : tile[y][x + 2 * j]) * f, v1 = (tall ? tile[x + 2 * j + 1][y] : tile[y][x + 2 * j + 1]) * f;
      float u0, u1;
      h[j] = from_two(v0, v1, __half());
      two_f32(h[j], u0, u1, __half());
      l[j] = from_two(v0 - u0, v1 - u1, __half());
    }
    const long long at = ((long long)b * n + row) * ldx + col;  // rows are padded to 16 bytes
    *reinterpret_cast<uint4*>(hi + at) = make_uint4(h[0], h[1], h[2], h[3]);
    *reinterpret_cast<uint4*>(lo + at) = make_uint4(l[0], l[1], l[2], l[3]);
  }
}

// ------------------------------------------------------------------ products
enum Product { GRAM, SQUARE, APPLY, LAST };  // LAST: APPLY to the result

constexpr int kWriteWarps = 8, kGetWarp = 8, kMulWarp = 9, kGetWarpB = 10, kThreadsO = 32 * 11;
// Shared memory for results: two tiles of 32 rows of 64 columns, or 32 of narrow tiles, for each warp that writes.
__host__ __device__ constexpr int ortho_part(int bn) { return bn >= 128 ? 4096 : 2048; }
__host__ __device__ constexpr int ortho_staging(int bn) { return 2 * ortho_part(bn) * kWriteWarps; }

struct OrthoArgs {
  int batch, n, k;          // X is n x k, A and P are n x n
  long long ldx, lda;
  const __half *hi, *lo;    // X as it is (APPLY, LAST); lo null: zeros
  __half *hi_out, *lo_out;  // lo_out may be lo, or null: not wanted
  const __half* a;          // A (SQUARE)
  __half* sym;              // A (GRAM) or P (SQUARE)
  float ca, cb, cc;
  void* out;  // LAST: [n, k] or, tall, [k, n]
  int out_type, out_bytes;
  bool tall;
  bool whole;      // tiles of 64 columns: all of A and P are computed, none mirrored
  bool backwards;  // the last matrix first: it is what the product before left in L2
  int nstage;
  long long limit;
  int* health;  // non-zero once a bounded wait gave up (read by fs_device_error)
};

template <int FORM, int CG, int BN>
struct TilesO {
  const OrthoArgs& a;
  int mt, nt, per;
  __device__ explicit TilesO(const OrthoArgs& args) : a(args) {
    constexpr int BM = 128 * CG, R = BM / BN > 0 ? BM / BN : 1;
    mt = (a.n + BM - 1) / BM;
    nt = ((FORM >= APPLY ? a.k : a.n) + BN - 1) / BN;
    if (all()) {
      per = mt * nt;
    } else {  // tiles (i, j) with j < (i + 1) R, as far as there are columns
      per = R * mt * (mt - 1) / 2 + nt;
      if (per < 0) per = 0;
    }
  }
  __device__ bool all() const { return FORM >= APPLY || (CG == 1 && BN == 64 && a.whole); }
  __device__ long long total() const { return (long long)per * a.batch; }
  __device__ void at(long long tile, int& b, int& m0, int& n0) const {
    constexpr int BM = 128 * CG, R = BM / BN > 0 ? BM / BN : 1;
    b = BN == 64 ? (int)((unsigned)tile / (unsigned)per) : (int)(tile / per);  // narrow ones are few, and a division of 64 bits takes 100 clocks
    int rest = (int)(tile - (long long)b * per);
    if (a.backwards) b = a.batch - 1 - b;
    if (all()) {
      const int j = rest / mt;
      m0 = (rest - j * mt) * BM;
      n0 = j * BN;
    } else {
      int i = 0;
      while (i + 1 < mt && rest >= (i + 1) * R) rest -= (++i) * R;
      m0 = i * BM;
      n0 = rest * BN;
    }
  }
};

__device__ __forceinline__ uint4 load_chunk(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}

// What the threads of a CTA share over the products of a launch, and how far they are: the same in every lane of a warp.
struct OrthoPipe {
  uint8_t *ring, *staging;
  uint64_t* bars;
  volatile int* abort_flag;
  int* words;  // of settle()
  uint32_t tmem;
  int nstage, warp, lane, rank;
  int s;        // next stage
  uint32_t ph;  // its phase
  int tiles;    // that this CTA has done
  __device__ uint32_t bar(int i) const { return smem_u32(bars + i); }
  __device__ int full() const { return 0; }
  __device__ int empty() const { return nstage; }
  __device__ int acc_full() const { return 2 * nstage; }
  __device__ int acc_empty() const { return 2 * nstage + 2; }
  __device__ int drain() const { return 2 * nstage + 4; }
};

template <int CG, int BN>
__device__ __forceinline__ OrthoPipe ortho_begin(uint8_t* raw, int nstage) {
  constexpr uint32_t kStage = 128 * 128 + BN / CG * 128, kColumns = 2 * BN;
  static_assert(kColumns <= 512 && kStage % 1024 == 0 && BN / CG >= 64, "tile");
  OrthoPipe p;
  p.ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  p.staging = p.ring + (size_t)nstage * kStage;
  p.bars = reinterpret_cast<uint64_t*>(p.staging + ortho_staging(BN));
  p.nstage = nstage;
  uint32_t* slot = reinterpret_cast<uint32_t*>(p.bars + p.drain() + 1);
  p.abort_flag = reinterpret_cast<volatile int*>(slot + 1);
  p.words = reinterpret_cast<int*>(slot + 2);
  p.warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0);
  p.lane = threadIdx.x & 31;
  p.rank = CG == 2 ? (int)cta_rank() : 0;
  p.s = p.tiles = 0;
  p.ph = 0;
  if (p.warp == kGetWarp && p.lane == 0) {
    for (int s = 0; s < nstage; ++s) {
      mbar_init(p.bar(p.full() + s), 2 * CG);  // in CTA 0: both CTAs' loads of either operand
      mbar_init(p.bar(p.empty() + s), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(p.bar(p.acc_full() + i), 1);
      mbar_init(p.bar(p.acc_empty() + i), kWriteWarps * CG);  // in CTA 0: all warps of the pair that write
    }
    mbar_init(p.bar(p.drain()), 1);
    *p.abort_flag = p.words[0] = p.words[1] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  } else if (p.warp == kMulWarp) {
    alloc_columns<CG>(smem_u32(slot), kColumns);
  }
  tc_fence_before();
  __syncthreads();
  if (CG == 2) cluster_sync_all();
  tc_fence_after();
  p.tmem = *slot;
  return p;
}

// This CTA's tiles of one product.
template <int FORM, int CG, int BN>
__device__ __forceinline__ void ortho_product(const OrthoArgs& a, const CUtensorMap* mapA, const CUtensorMap* mapB, OrthoPipe& p) {
  constexpr bool B_MN = FORM >= APPLY;
  constexpr int BNC = BN / CG;  // columns whose operand this CTA fetches
  constexpr uint32_t kA = 128 * 128, kB = BNC * 128, kStage = kA + kB, kHalf = 64 * 128;
  uint8_t *const ring = p.ring, *const staging = p.staging;
  volatile int* const abort_flag = p.abort_flag;
  const uint32_t tmem = p.tmem;
  const int warp = p.warp, lane = p.lane, rank = p.rank, FULL = p.full(), EMPTY = p.empty(), ACC_FULL = p.acc_full(), ACC_EMPTY = p.acc_empty();
  auto bar = [&](int i) { return p.bar(i); };
  const int first = blockIdx.x / CG, stride = gridDim.x / CG;
  const int contraction = FORM == GRAM ? a.k : a.n, blocks = (contraction + 63) / 64;
  const TilesO<FORM, CG, BN> tiles(a);
  const long long total = tiles.total();

  if (warp == kGetWarp || warp == kGetWarpB) {
    // ===================== loads =====================
    // A warp for each operand: one thread takes 150 to 200 clocks for a tensor load, and a stage of P X has three of them for products of 512
    // (32 matrices of 2048 x 1024: 1405 -> 1346 us when it was measured, with X's lower part in three steps).
    if (elect_one()) {
      int s = p.s, issued = 0;
      uint32_t ph = p.ph;
      bool ok = *abort_flag == 0;  // a CTA that has given up starts nothing more
      for (long long it = first; ok && it < total; it += stride) {
        int b, m0, n0;
        tiles.at(it, b, m0, n0);
        for (int kb = 0; kb < blocks; ++kb) {
          if (!mbar_wait(bar(EMPTY + s), ph ^ 1, abort_flag)) {
            ok = false;
            break;
          }
          const uint32_t full = CG == 2 ? in_leader(bar(FULL + s)) : bar(FULL + s), dst = smem_u32(ring + (size_t)s * kStage);
          if (warp == kGetWarp) {
            expect_at<CG>(full, kA);
            load_3d<CG>(dst, mapA, kb * 64, m0 + rank * 128, b, full);
          } else {
            expect_at<CG>(full, kB);
            if (B_MN) {
#pragma unroll
              for (int c = 0; c < BNC / 64; ++c) load_3d<CG>(dst + kA + c * kHalf, mapB, n0 + rank * BNC + c * 64, kb * 64, b, full);
            } else {
              load_3d<CG>(dst + kA, mapB, kb * 64, n0 + rank * BNC, b, full);
            }
          }
          ++issued;
          if (++s == p.nstage) {
            s = 0;
            ph ^= 1;
          }
        }
      }
      p.words[warp == kGetWarp ? 0 : 1] += issued;
    }
  } else if (warp == kMulWarp) {
    // ===================== products =====================
    if (rank == 0 && elect_one()) {
      // fp32 sums of fp16 operands
      constexpr uint32_t idesc = (1u << 4) | ((B_MN ? 1u : 0u) << 16) | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(128 * CG >> 4) << 24);
      // a step of 16 contraction values: 32 bytes on, or 16 rows of 128 bytes; MN: the next 64 columns one half tile on
      constexpr uint32_t kStepB = (B_MN ? 16u * 128u : 32u) >> 4, kLeadB = B_MN ? kHalf >> 4 : 1u;
      int s = p.s, n = p.tiles;
      uint32_t ph = p.ph;
      bool ok = *abort_flag == 0;  // a CTA that has given up starts nothing more
      for (long long it = first; ok && it < total; it += stride, ++n) {
        const int buf = n & 1;
        if (!mbar_wait(bar(ACC_EMPTY + buf), ((n >> 1) & 1) ^ 1, abort_flag)) break;
        tc_fence_after();
        for (int kb = 0; kb < blocks; ++kb) {
          if (!mbar_wait(bar(FULL + s), ph, abort_flag)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t base = smem_u32(ring + (size_t)s * kStage);
          const uint32_t al = desc_lo(base), bl = (((base + kA) & 0x3FFFFu) >> 4) | (kLeadB << 16);
          const int left = contraction - kb * 64;
#pragma unroll
          for (int ks = 0; ks < 4; ++ks)
            if (ks * 16 < left)
              mma_f16<CG>(tmem + buf * BN, pack_desc(al + ks * 2, kDescHi128), pack_desc(bl + ks * kStepB, kDescHi128), idesc, kb | ks);
          commit<CG>(bar(EMPTY + s));
          if (++s == p.nstage) {
            s = 0;
            ph ^= 1;
          }
        }
        if (!ok) break;
        commit<CG>(bar(ACC_FULL + buf));
      }
    }
  } else {
    // ===================== results =====================
    // Two warps to a quarter of the TMEM lanes (rows), with every other block of kCols columns each. What a block adds to its
    // product (A, or both parts of X) comes by whole rows of 16-byte loads, is under way in registers while the block before it is
    // worked on, and goes through shared memory to the lanes that have its rows; results go back the same way.
    constexpr int kCols = BN >= 128 ? 64 : 32, kPart = ortho_part(BN), kPitch = 2 * kCols, kPer = kCols / 8, kFrom = FORM == GRAM ? 0 : FORM == SQUARE ? 1 : 2;
    const int q = warp & 3, side = warp >> 2;
    const uint32_t stage = smem_u32(staging + 2 * kPart * warp);
    const int width = FORM >= APPLY ? a.k : a.n;  // columns of the product
    const long long ld = FORM >= APPLY ? a.ldx : a.lda;
    uint4 ahead[kFrom ? kFrom : 1][kPer];
    auto ask = [&](int b, int row0, int col) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int r = row0 + i * (32 / kPer) + lane / kPer, c = col + 8 * (lane % kPer);
        const long long at = ((long long)b * a.n + r) * ld + c;
        const bool in = r < a.n && c < width;  // rows are padded to 16 bytes
#pragma unroll
        for (int k = 0; k < kFrom; ++k)
          if (in && (k == 0 || a.lo)) {  // in a chain of products, what other SMs have written in the same launch: past L1
            const uint4* from = reinterpret_cast<const uint4*>((FORM == SQUARE ? a.a : k ? a.lo : a.hi) + at);
            ahead[k][i] = CG == 2 ? *from : __ldcg(from);
          } else {
            ahead[k][i] = make_uint4(0u, 0u, 0u, 0u);
          }
      }
    };
    int t = p.tiles, b = 0, m0 = 0, n0 = 0;
    if (a.limit == 0) *abort_flag = 1;
    bool lost = a.limit == 0 || *abort_flag != 0;  // a wait of this CTA gave up: NaN from here on
    if (first < total) {
      tiles.at(first, b, m0, n0);
      if (kFrom) ask(b, m0 + rank * 128 + q * 32, n0 + kCols * side);
    }
    for (long long it = first; it < total; it += stride, ++t) {
      const int buf = t & 1, row0 = m0 + rank * 128 + q * 32, row = row0 + lane;
      int next_b = 0, next_m = 0, next_n = 0;
      if (it + stride < total) tiles.at(it + stride, next_b, next_m, next_n);
#pragma unroll 1
      for (int c = kCols * side; c < BN; c += 2 * kCols) {
        const int col = n0 + c;
        if (kFrom) {
#pragma unroll
          for (int i = 0; i < kPer; ++i)
#pragma unroll
            for (int k = 0; k < kFrom; ++k)
              stage16(staged_row<kPitch>(stage + kPart * k, i * (32 / kPer) + lane / kPer, lane % kPer), ahead[k][i].x, ahead[k][i].y, ahead[k][i].z, ahead[k][i].w);
          __syncwarp();
          if (c + 2 * kCols < BN) ask(b, row0, col + 2 * kCols);
          else if (it + stride < total) ask(next_b, next_m + rank * 128 + q * 32, next_n + kCols * side);
        }
        if (c == kCols * side && !lost) {
          lost = !__all_sync(0xffffffffu, CG == 2 ? wait_blocks(bar(ACC_FULL + buf), (t >> 1) & 1, abort_flag, blocks, a.limit)
                                                  : wait_close(bar(ACC_FULL + buf), (t >> 1) & 1, abort_flag, close_limit(a.limit + 4096ll * blocks)));
          tc_fence_after();
        }
        if (col < width && row0 < a.n) {
          const bool across = FORM == LAST ? a.tall : FORM <= SQUARE && !tiles.all() && n0 + BN <= m0;  // also, or only, written transposed
          uint32_t w[kCols / 2];
#pragma unroll
          for (int h = 0; h < kCols; h += 32) {
            float v[32];
            if (lost) {
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(0x7fc00000u);
            } else {
              tmem_ld32(tmem + buf * BN + c + h + ((uint32_t)(q * 32) << 16), v);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t at = staged_row<kPitch>(stage, lane, h / 8 + i);
              float* x = v + 8 * i;
              if (FORM == GRAM) {
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] *= kAScale / (kXScale * kXScale);
              } else {
                const uint4 p = load_chunk(at), l = kFrom == 2 ? load_chunk(at + kPart) : make_uint4(0u, 0u, 0u, 0u);
                const uint32_t pw[4] = {p.x, p.y, p.z, p.w}, lw[4] = {l.x, l.y, l.z, l.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                  float p0, p1, l0 = 0.f, l1 = 0.f;
                  two_f32(pw[j], p0, p1, __half());
                  if (kFrom == 2) two_f32(lw[j], l0, l1, __half());
                  const float own = FORM == SQUARE ? a.cb : FORM == LAST ? a.ca / kXScale : a.ca;
                  const float product = FORM == SQUARE ? a.cc / kAScale : FORM == LAST ? 1.f / (kAScale * kXScale) : 1.f / kAScale;
                  x[2 * j] = fmaf(x[2 * j], product, own * (p0 + l0));
                  x[2 * j + 1] = fmaf(x[2 * j + 1], product, own * (p1 + l1));
                }
              }
              uint32_t* u = w + h / 2 + 4 * i;
              uint32_t lower[4];
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                u[j] = FORM == LAST && a.out_type == FS_TYPE_BF16 ? from_two(x[2 * j], x[2 * j + 1], __nv_bfloat16()) : from_two(x[2 * j], x[2 * j + 1], __half());
                if (FORM == APPLY) {
                  float u0, u1;
                  two_f32(u[j], u0, u1, __half());
                  lower[j] = from_two(x[2 * j] - u0, x[2 * j + 1] - u1, __half());
                }
              }
              if (FORM != LAST || !across) stage16(at, u[0], u[1], u[2], u[3]);
              if (FORM == APPLY) stage16(at + kPart, lower[0], lower[1], lower[2], lower[3]);
            }
          }
          if (FORM != APPLY && across) {
            // Pairs of lanes exchange halves, so that each has two rows of a column; a column's 32 rows are 64 bytes side by side.
            __syncwarp();
#pragma unroll
            for (int j = 0; j < kCols / 2; ++j) {
              const uint32_t other = __shfl_xor_sync(0xffffffffu, w[j], 1);
              const uint32_t two = lane & 1 ? __byte_perm(other, w[j], 0x7632) : __byte_perm(w[j], other, 0x5410);
              asm volatile("st.shared.u32 [%0], %1;" ::"r"(stage + kPart + (2 * j + (lane & 1)) * 64 + (lane >> 1) * 4), "r"(two) : "memory");
            }
            __syncwarp();
            const long long pitch = FORM == LAST ? a.n : ld;
            uint16_t* out = FORM == LAST ? static_cast<uint16_t*>(a.out) + ((long long)b * a.k + col) * a.n + row0
                                         : reinterpret_cast<uint16_t*>(a.sym) + ((long long)b * a.n + col) * ld + row0;
            if (FORM != LAST || a.out_bytes == 16) {
#pragma unroll
              for (int i = 0; i < kCols / 8; ++i) {
                const int r = 8 * i + (lane >> 2), ch = lane & 3;
                const uint4 x = load_chunk(stage + kPart + r * 64 + ch * 16);
                if (col + r < width && row0 + 8 * ch < a.n) *reinterpret_cast<uint4*>(out + r * pitch + 8 * ch) = x;
              }
            } else {
#pragma unroll 4
              for (int r = 0; r < kCols; ++r) {
                uint16_t x;
                asm volatile("ld.shared.u16 %0, [%1];" : "=h"(x) : "r"(stage + kPart + r * 64 + lane * 2) : "memory");
                if (col + r < width && row < a.n) out[r * pitch + lane] = x;
              }
            }
          }
          __syncwarp();
          const int rows = a.n - row0, bytes = min(2 * (width - col), 2 * kCols);
          const long long at = ((long long)b * a.n + row0) * ld + col;
          if (FORM == LAST) {
            if (!across)
              write_rows<kPitch>(reinterpret_cast<char*>(static_cast<uint16_t*>(a.out) + ((long long)b * a.n + row0) * a.k + col), 2ll * a.k, rows, bytes, a.out_bytes,
                         stage, lane);
          } else {
            write_rows<kPitch>(reinterpret_cast<char*>((FORM == APPLY ? a.hi_out : a.sym) + at), 2 * ld, rows, bytes, 16, stage, lane);
            if (FORM == APPLY && a.lo_out) write_rows<kPitch>(reinterpret_cast<char*>(a.lo_out + at), 2 * ld, rows, bytes, 16, stage + kPart, lane);
          }
        }
        __syncwarp();
      }
      if (!lost) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (CG == 2) arrive_cluster(in_leader(bar(ACC_EMPTY + buf)));
          else mbar_arrive(bar(ACC_EMPTY + buf));
        }
      }
      b = next_b;
      m0 = next_m;
      n0 = next_n;
    }
  }
  // every lane goes on from here, whichever one did the work (in a chain of products, whose CTAs have few tiles)
  for (long long it = first; it < total; it += stride) {
    const unsigned past = p.s + blocks;
    p.ph ^= past / p.nstage & 1u;
    p.s = past % p.nstage;
    ++p.tiles;
  }
}

template <int CG, int BN>
__device__ __forceinline__ void ortho_end(const OrthoPipe& p, int* health) {
  settle<CG, 2>(p.abort_flag, p.words, p.bar(p.full()), p.bar(p.drain()), p.nstage, p.warp == kMulWarp, p.warp == kGetWarp);
  if (p.warp == kMulWarp) free_columns<CG>(p.tmem, 2 * BN);
  if (threadIdx.x == 0 && *p.abort_flag) atomicExch(health, 1);
}

template <int FORM, int CG, int BN>
__global__ void __launch_bounds__(kThreadsO, 1)
ortho_kernel(const OrthoArgs a, const __grid_constant__ CUtensorMap mapA, const __grid_constant__ CUtensorMap mapB) {
  extern __shared__ uint8_t raw[];
  OrthoPipe p = ortho_begin<CG, BN>(raw, a.nstage);
  ortho_product<FORM, CG, BN>(a, &mapA, &mapB, p);
  ortho_end<CG, BN>(p, a.health);
}

// All products of all steps in one launch, for small matrices, whose products take less than a launch: every CTA does its tiles of
// one, then waits for the others (bounded; a cooperative launch, so that they are all there).
struct OrthoChain {
  int steps, lower_until;
  __half *x[2], *lo, *sym, *poly;
  unsigned* meeting;  // zero at the start
};
struct OrthoMaps {
  CUtensorMap x128[2], x64[2], a128, a64, p128;  // boxes of 128 or 64 rows
};
constexpr int kChainBN = 64, kChainTiles = 2, kChainStages = 8;  // columns of a tile, tiles of a CTA

// What this CTA has written is there for the loads of all others behind it: the CTA's barrier and one thread's release order all of its
// writes, and a fence of the thread that releases and of the one that loads orders them before tensor loads (which go another way to
// memory). The same fences by all threads took 3 us.
__device__ __forceinline__ void ortho_meet(const OrthoPipe& p, unsigned* meeting, unsigned target, long long limit) {
  __syncthreads();
  if (threadIdx.x == 0 && !*p.abort_flag) {
    unsigned seen;
    asm volatile("fence.proxy.async.global;" ::: "memory");
    asm volatile("red.release.gpu.global.add.u32 [%0], 1;" ::"l"(meeting) : "memory");
    const long long t0 = clock64();
    do {
      asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(seen) : "l"(meeting) : "memory");
      if (seen < target && clock64() - t0 > limit) *p.abort_flag = 1;
    } while (seen < target && !*p.abort_flag);
  }
  __syncthreads();
  if (p.warp == kGetWarp || p.warp == kGetWarpB) asm volatile("fence.proxy.async.global;" ::: "memory");
}

__global__ void __launch_bounds__(kThreadsO, 1) ortho_chain_kernel(OrthoArgs a, const OrthoChain c, const __grid_constant__ OrthoMaps maps) {
  extern __shared__ uint8_t raw[];
  if (threadIdx.x < sizeof(OrthoMaps) / sizeof(CUtensorMap))
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<const CUtensorMap*>(&maps) + threadIdx.x) : "memory");
  OrthoPipe p = ortho_begin<1, kChainBN>(raw, kChainStages);
  unsigned target = 0;
#pragma unroll 1
  for (int i = 0; i < c.steps; ++i) {
    const bool from = i & 1;
    a.hi = from ? c.x[1] : c.x[0];
    a.lo = i < c.lower_until ? c.lo : nullptr;
    a.hi_out = from ? c.x[0] : c.x[1];
    a.lo_out = i + 1 < c.lower_until ? c.lo : nullptr;
    a.sym = c.sym;
    ortho_product<GRAM, 1, kChainBN>(a, &maps.x128[from], &maps.x64[from], p);
    ortho_meet(p, c.meeting, target += gridDim.x, a.limit);
    a.a = c.sym;
    a.sym = c.poly;
    ortho_product<SQUARE, 1, kChainBN>(a, &maps.a128, &maps.a64, p);
    ortho_meet(p, c.meeting, target += gridDim.x, a.limit);
    if (i + 1 < c.steps) {
      ortho_product<APPLY, 1, kChainBN>(a, &maps.p128, &maps.x64[from], p);
      ortho_meet(p, c.meeting, target += gridDim.x, a.limit);
    } else {
      ortho_product<LAST, 1, kChainBN>(a, &maps.p128, &maps.x64[from], p);
    }
  }
  ortho_end<1, kChainBN>(p, a.health);
}

// ------------------------------------------------------------------ host side
// fp16 stack [batch][rows][cols], rows ld apart; boxes of 64 x box_rows.
bool encode_stack(CUtensorMap* map, const __half* base, long long cols, long long rows, long long batch, long long ld, int box_rows) {
  const cuuint64_t sizes[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)batch};
  const cuuint64_t strides[2] = {(cuuint64_t)ld * 2, (cuuint64_t)(ld * rows) * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)box_rows, 1}, ones[3] = {1, 1, 1};
  const auto fn = encoder();
  return fn && fn(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<__half*>(base), sizes, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int FORM, int CG, int BN>
int launch_ortho(OrthoArgs a, cudaStream_t st) {
  CUtensorMap mapA = {}, mapB = {};
  const __half* left = FORM == GRAM ? a.hi : FORM == SQUARE ? a.a : a.sym;
  const bool good =
      FORM == GRAM ? encode_stack(&mapA, left, a.k, a.n, a.batch, a.ldx, 128) && encode_stack(&mapB, left, a.k, a.n, a.batch, a.ldx, BN / CG)
      : FORM == SQUARE ? encode_stack(&mapA, left, a.n, a.n, a.batch, a.lda, 128) && encode_stack(&mapB, left, a.n, a.n, a.batch, a.lda, BN / CG)
                       : encode_stack(&mapA, left, a.n, a.n, a.batch, a.lda, 128) && encode_stack(&mapB, a.hi, a.k, a.n, a.batch, a.ldx, 64);
  if (!good) return report_error(FS_ERR_CUDA, "cuTensorMapEncodeTiled failed");
  constexpr size_t kStage = 128 * 128 + BN / CG * 128;
  constexpr size_t fixed = 1024 + ortho_staging(BN) + 8 * (2 * 12 + 5) + 32;
  a.nstage = (int)((kSmemMax - fixed) / kStage);
  if (a.nstage > 12) a.nstage = 12;
  size_t smem = fixed + a.nstage * kStage;
  if (smem < (size_t)kSmemMin) smem = kSmemMin;
  const auto kernel = ortho_kernel<FORM, CG, BN>;
  static std::atomic<uint64_t> allowed{0};  // devices on which the kernel may take all shared memory
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (e == cudaSuccess && !(allowed.load(std::memory_order_relaxed) & bit)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMax);
    if (e == cudaSuccess) allowed.fetch_or(bit, std::memory_order_relaxed);
  }
  if (e != cudaSuccess) return report_error(FS_ERR_CUDA, cudaGetErrorString(e));
  const long long mt = (a.n + 128 * CG - 1) / (128 * CG), most = mt * (((FORM >= APPLY ? a.k : a.n) + BN - 1) / BN) * a.batch;
  long long grid = detail::free_ctas() / CG;
  a.whole = most <= grid;
  if (grid > most) grid = most;
  if (grid < 1) grid = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)grid * CG);
  cfg.blockDim = dim3(kThreadsO);
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
  e = cudaLaunchKernelEx(&cfg, kernel, a, mapA, mapB);
  if (e != cudaSuccess) return report_error(FS_ERR_CUDA, cudaGetErrorString(e));
  count_launches(1);
  return FS_OK;
}
// Whether all of it is one launch: tiles of 128 x 64, of which a CTA has few.
bool chained(const OrthoArgs& a) {
  const long long m = (a.n + 127) / 128, n = (a.k + kChainBN - 1) / kChainBN;
  return m * n * a.batch <= kChainTiles * (long long)detail::free_ctas();
}
int launch_chain(OrthoArgs a, const OrthoChain& c, cudaStream_t st) {
  OrthoMaps maps = {};
  for (int i = 0; i < 2; ++i)
    if (!encode_stack(&maps.x128[i], c.x[i], a.k, a.n, a.batch, a.ldx, 128) || !encode_stack(&maps.x64[i], c.x[i], a.k, a.n, a.batch, a.ldx, 64))
      return report_error(FS_ERR_CUDA, "cuTensorMapEncodeTiled failed");
  if (!encode_stack(&maps.a128, c.sym, a.n, a.n, a.batch, a.lda, 128) || !encode_stack(&maps.a64, c.sym, a.n, a.n, a.batch, a.lda, 64) ||
      !encode_stack(&maps.p128, c.poly, a.n, a.n, a.batch, a.lda, 128))
    return report_error(FS_ERR_CUDA, "cuTensorMapEncodeTiled failed");
  constexpr size_t kStage = 128 * 128 + kChainBN * 128, fixed = 1024 + ortho_staging(kChainBN) + 8 * (2 * 12 + 5) + 32;
  constexpr size_t smem = fixed + kChainStages * kStage;
  static_assert(smem >= (size_t)kSmemMin && smem <= kSmemMax, "shared memory");
  static std::atomic<uint64_t> allowed{0};  // devices on which the kernel may take all shared memory
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (e == cudaSuccess && !(allowed.load(std::memory_order_relaxed) & bit)) {
    e = cudaFuncSetAttribute(ortho_chain_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMax);
    if (e == cudaSuccess) allowed.fetch_or(bit, std::memory_order_relaxed);
  }
  if (e != cudaSuccess) return report_error(FS_ERR_CUDA, cudaGetErrorString(e));
  const long long high = (a.n + 127) / 128 * a.batch, most = high * ((a.k + kChainBN - 1) / kChainBN);
  a.whole = high * ((a.n + kChainBN - 1) / kChainBN) <= detail::free_ctas();
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(most < detail::free_ctas() ? most : detail::free_ctas()));
  cfg.blockDim = dim3(kThreadsO);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeCooperative;
  attr.val.cooperative = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  a.health = products_health();
  if (!a.health) return report_error(FS_ERR_CUDA, "cannot find the health word of the current CUDA device");
  e = cudaLaunchKernelEx(&cfg, ortho_chain_kernel, a, c, maps);
  if (e != cudaSuccess) return report_error(FS_ERR_CUDA, cudaGetErrorString(e));
  count_launches(1);
  return FS_OK;
}

template <int FORM>
int launch_form(const OrthoArgs& a, cudaStream_t st) {
  const int ctas = detail::free_ctas();
  auto tiles = [&](int bm, int bn) {
    const long long m = (a.n + bm - 1) / bm, n = ((FORM >= APPLY ? a.k : a.n) + bn - 1) / bn;
    return (FORM >= APPLY ? m * n : m * n / 2 + 1) * a.batch;
  };
  // Pairs where there are tiles of 256 x 256 for all of them, and rows for both CTAs; then the largest tile with which there is one for every CTA. us of five
  // steps with tiles of 128 x 64, 128 x 128 and 256 x 256 throughout (as chosen they differ from product to product): 32 matrices of 128 x 2048 198,
  // 202, 290; 300 of 64 x 72 155, 157, 262; 64 of 128 x 512 147, 145, 196; 32 of 256 x 2048 344, 303, 335; 16 of 300 x 700 180, 165, 233; 32 of 512 x 512 303,
  // 282, 294; 32 of 1024 x 2048 2362, 1732, 1581; one of 4096 x 4096 2651, 1575, 1230.
  if (a.n > 128 && tiles(256, 256) * 2 > ctas) return launch_ortho<FORM, 2, 256>(a, st);
  if (tiles(128, 128) > ctas) return launch_ortho<FORM, 1, 128>(a, st);
  return launch_ortho<FORM, 1, 64>(a, st);
}

template <typename T>
int begin(const void* g, long long g_matrix, long long g_row, int batch, int rows, int cols, double* parts, float eps, bool tall, __half* hi, __half* lo,
          long long ldx, unsigned* meeting, cudaStream_t st) {
  constexpr int kWide = 16 / sizeof(T);
  const bool wide = aligned(g, 16) && g_matrix % kWide == 0 && g_row % kWide == 0 && cols % kWide == 0;
  const int want = (rows + 7) / 8, count = want < kNormParts ? want : kNormParts;
  for (int b0 = 0; b0 < batch; b0 += 65535) {  // the limit of a grid's second and third dimension
    const int nb = batch - b0 < 65535 ? batch - b0 : 65535;
    const T* from = static_cast<const T*>(g) + b0 * g_matrix;
    double* sums = parts + (size_t)b0 * count;
    const long long at = (long long)b0 * (tall ? cols : rows) * ldx;
    const dim3 over(count, nb), tiles((cols + 63) / 64, (rows + 63) / 64, nb);
    if (wide) {
      squares_kernel<T, kWide><<<over, 256, 0, st>>>(from, g_matrix, g_row, rows, cols, sums);
      begin_kernel<T, kWide><<<tiles, 256, 0, st>>>(from, g_matrix, g_row, rows, cols, sums, count, eps, tall, hi + at, lo + at, ldx, meeting);
    } else {
      squares_kernel<T, 1><<<over, 256, 0, st>>>(from, g_matrix, g_row, rows, cols, sums);
      begin_kernel<T, 1><<<tiles, 256, 0, st>>>(from, g_matrix, g_row, rows, cols, sums, count, eps, tall, hi + at, lo + at, ldx, meeting);
    }
  }
  return launched(2);
}

struct OrthoSpace {
  size_t x, a, parts, all;  // bytes of one part of X, of A, of the sums of squares
};
OrthoSpace ortho_space(int batch, int rows, int cols) {
  const size_t n = rows < cols ? rows : cols, k = rows < cols ? cols : rows;
  auto round = [](size_t v, size_t to) { return (v + to - 1) / to * to; };
  OrthoSpace s;
  s.x = round((size_t)batch * n * round(k, 8) * 2, 256);
  s.a = round((size_t)batch * n * round(n, 8) * 2, 256);
  s.parts = round((size_t)batch * kNormParts * sizeof(double), 256);
  s.all = 3 * s.x + 2 * s.a + s.parts + 256;  // and the word of meetings
  return s;
}

}  // namespace
}  // namespace ex
}  // namespace fs

using namespace fs;
using namespace fs::ex;

extern "C" {

size_t fs_orthogonalize_bytes(int batch, int rows, int cols) {
  if (batch < 1 || rows < 1 || cols < 1) return 0;
  return ortho_space(batch, rows, cols).all;
}

int fs_orthogonalize(const void* g, int type, long long g_matrix, long long g_row, int batch, int rows, int cols, int steps, float a, float b,
                     float c, float eps, void* out, int out_type, void* ws, size_t ws_bytes, void* stream) {
  if (type < FS_TYPE_F32 || type > FS_TYPE_BF16 || (out_type != FS_TYPE_F16 && out_type != FS_TYPE_BF16))
    return report_error(FS_ERR_BAD_ARG, "type must be one of FS_TYPE_*, that of the result FS_TYPE_F16 or FS_TYPE_BF16");
  if (batch < 0 || rows < 1 || cols < 1 || rows > 65536 || cols > 65536 || g_row < cols || steps < 1 || steps > 64 || !(eps > 0.f))
    return report_error(FS_ERR_BAD_ARG, "batch must not be negative, rows and cols in [1, 65536], rows not overlap, steps in [1, 64] and eps be positive");
  const int s = check_device();
  if (s != FS_OK || batch == 0) return s;
  if (!g || !out || g_matrix < 0) return report_error(FS_ERR_BAD_ARG, "null argument");
  const OrthoSpace space = ortho_space(batch, rows, cols);
  if (!ws || ws_bytes < space.all) return report_error(FS_ERR_WORKSPACE, "workspace too small");
  if (!aligned(ws, 256)) return report_error(FS_ERR_BAD_ARG, "workspace must be aligned to 256 bytes");
  int dev = 0;  // binds the device's context to a thread that has launched nothing yet: the encoding of tensor maps needs one
  if (cudaGetDevice(&dev) != cudaSuccess || cudaSetDevice(dev) != cudaSuccess)
    return report_error(FS_ERR_CUDA, "cannot make the current CUDA device's context current");
  const bool tall = rows > cols;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  uint8_t* p = static_cast<uint8_t*>(ws);
  __half *hi = reinterpret_cast<__half*>(p), *other = reinterpret_cast<__half*>(p + space.x), *lo = reinterpret_cast<__half*>(p + 2 * space.x);
  __half *sym = reinterpret_cast<__half*>(p + 3 * space.x), *poly = reinterpret_cast<__half*>(p + 3 * space.x + space.a);
  double* parts = reinterpret_cast<double*>(p + 3 * space.x + 2 * space.a);
  unsigned* meeting = reinterpret_cast<unsigned*>(p + 3 * space.x + 2 * space.a + space.parts);
  OrthoArgs o{};
  o.batch = batch;
  o.n = tall ? cols : rows;
  o.k = tall ? rows : cols;
  o.ldx = (o.k + 7) / 8 * 8;
  o.lda = (o.n + 7) / 8 * 8;
  o.ca = a; o.cb = b; o.cc = c;
  o.lo = o.lo_out = lo;
  o.out = out; o.out_type = out_type; o.tall = tall;
  const int inner = tall ? o.n : o.k;  // values of a row of the result
  o.out_bytes = aligned(out, 16) && inner % 8 == 0 ? 16 : aligned(out, 4) && inner % 2 == 0 ? 4 : 2;
  o.limit = product_limit();
  int r = type == FS_TYPE_F32  ? begin<float>(g, g_matrix, g_row, batch, rows, cols, parts, eps, tall, hi, lo, o.ldx, meeting, st)
          : type == FS_TYPE_F16 ? begin<__half>(g, g_matrix, g_row, batch, rows, cols, parts, eps, tall, hi, lo, o.ldx, meeting, st)
                                : begin<__nv_bfloat16>(g, g_matrix, g_row, batch, rows, cols, parts, eps, tall, hi, lo, o.ldx, meeting, st);
  float grown = 1.f;  // what the steps from the last one on make of a rounding along small singular values
  int lower_until = steps;
  while (lower_until > 1 && grown * fabsf(a) <= kFewTimes) {
    grown *= fabsf(a);
    --lower_until;
  }
  if (r == FS_OK && chained(o)) {
    const OrthoChain chain{steps, lower_until, {hi, other}, lo, sym, poly, meeting};
    return launch_chain(o, chain, st);
  }
  for (int i = 0; i < steps && r == FS_OK; ++i) {
    o.hi = hi;
    o.lo = i < lower_until ? lo : nullptr;
    o.hi_out = other;
    o.lo_out = i + 1 < lower_until ? lo : nullptr;
    o.sym = sym;
    o.backwards = !o.backwards;
    r = launch_form<GRAM>(o, st);
    if (r != FS_OK) return r;
    o.a = sym;
    o.sym = poly;
    o.backwards = !o.backwards;
    r = launch_form<SQUARE>(o, st);
    if (r != FS_OK) return r;
    o.backwards = !o.backwards;
    r = i + 1 < steps ? launch_form<APPLY>(o, st) : launch_form<LAST>(o, st);
    __half* t = hi;
    hi = other;
    other = t;
  }
  return r;
}

}  // extern "C"
