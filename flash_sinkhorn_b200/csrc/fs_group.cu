// Matrix products grouped by expert on the 5th-generation tensor cores, with groups of any size.
//
//   rows     out[i, n] = sum_k W_e[n, k] x[row(i), k]           (forward, and the gradient to x with W transposed)
//   weights  dw_e[n, k] = sum_i dy[i, n] x[i, k]                 (i over the rows of expert e)
//
// In the rows form the FEATURES are the M side of the tensor-core instruction (128 lanes of TMEM per CTA) and the rows of a
// group its N side: N goes in steps of 16 at run time, so the last, partial tile of a group costs what it holds, and a
// group of one row costs 16 columns rather than 128. The rows of the next group that a tile load may bring along are other
// columns of the accumulator; they are not written. In the weights form the rows are the contraction, so those of
// another group must not be read: a group ends at a step of 16 of the contraction, and where its rows end inside of one,
// the rest of that step is overwritten with zeros in shared memory, in both operands, so that no infinity of a neighbour
// meets a zero.
//
// One persistent CTA per SM, or a pair of CTAs on neighbouring SMs that share a 256 x 256 tile (each holds 128 features and
// fetches half of the rows: two thirds of the bytes per product of 128 x 256 tiles). One warp fetches whole tiles (TMA into a
// ring of stages of 64 contraction values), one issues the products into one of two TMEM accumulators (either by one
// thread from beginning to end: choosing it anew for every instruction cost 500 clocks a stage, as much as the products of a
// 256 x 256 tile), and eight write the other one out, through shared memory in pieces of 64 bytes. Rows in another order are
// fetched by eight more, 16 bytes a lane (cp.async): TMA's loads of four rows each took 75 clocks apiece, 2.6 times the time
// of the whole product. That is for single CTAs: in a pair, rows that one CTA has written have to reach the thread of the other
// one that issues the products by a release and an acquire at the cluster's scope, about a microsecond for each stage of 0.27
// (541 -> 941 us for 65536 rows of 64 groups, 2048 x 2048; 582 with a copy first), so products that want pairs take their rows
// in order, and whoever has them in another one copies them first (fs_grouped_mm_in_order). Group boundaries are read by the
// kernel itself; every CTA takes every n-th tile, features fastest, so that the CTAs working at one time share a group's weights
// and rows in L2.
#include "fs_experts.cuh"
#include "fs_pair.cuh"
#include "fs_ptx.cuh"
#include "fs_tc.cuh"

#include <atomic>

namespace fs {
namespace ex {
namespace {

using namespace fs::tc;

thread_local long long t_product_limit = kSpinLimit;  // clocks, fs_set_product_limit

enum Form { ROWS_K, ROWS_MN, WEIGHTS };  // rows with W contiguous along the contraction; along the features

// Warps: 0 to kOutWarps - 1 write results, then one each for whole tiles, products and reports, then the copying ones.
constexpr int kOutWarps = 8, kLoadWarp = kOutWarps, kMmaWarp = kOutWarps + 1, kReportWarp = kOutWarps + 2;
constexpr int kThreads = 32 * (kOutWarps + 3);
constexpr int kStaging = 2048 * kOutWarps;
// Eight warps fetch single rows, four of them every other stage each: one iteration of a warp (a wait, up to eight copies) takes
// about as long as the products of a stage.
constexpr int kCopyWarps = 8, kCopyGroup = 128;  // threads that fetch a stage
constexpr int kCopyRows = kCopyGroup / 8;        // rows that they fetch 128 bytes of at a time
constexpr uint32_t kHalfTile = 64 * 128;  // 64 rows of 128 bytes
constexpr int kMaxGroups = 1024;
constexpr int kMaxRows = 0x7fffffff - 511;  // no tile reaches past 2^31 rows: neither the indices nor the boxes of tensor loads overflow

struct GroupArgs {
  const int* offsets;
  const int* rows;  // rows form: row numbers (null: in order)
  int M;            // and the rows that there are
  int R, E, N, K;
  void* out;
  long long ldo;
  int type, out_type;  // FS_TYPE_*
  int out_vec;         // values of a store: 8, 2 or 1
  int nstage;
  const void* x;  // the rows as plain memory, for fetching them one by one
  long long ldx;
  long long limit;  // clocks that the warps which write results wait, besides what the products take; 0: none at all
  int* health;      // non-zero once a bounded wait gave up (read by fs_device_error)
};

// ------------------------------------------------------------------ PTX of gathered loads
// 16 bytes, of which those past the first `valid` become zeros (the source is not read for them).
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, int valid) {
  asm volatile("cp.async.cg.shared.global.L2::256B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid) : "memory");
}
// Arrives at a barrier of this CTA when all copies that the thread has started so far are there.
__device__ __forceinline__ void copy_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void copy_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }
// Shared-memory operands, 128-byte swizzle. K-major: rows of 64 contraction values, groups of 8 rows 1024 bytes apart; a step
// of 16 values is 32 bytes on. MN-major: 64 rows (contraction) of 64 features, the next 64 features one half tile on (the
// leading offset), groups of 8 contraction rows 1024 bytes apart; a step of 16 contraction rows is 2048 bytes on.
template <bool MN>
__device__ __forceinline__ uint32_t operand_lo(uint32_t addr) {
  return ((addr & 0x3FFFFu) >> 4) | ((MN ? kHalfTile >> 4 : 1u) << 16);
}
__host__ __device__ constexpr uint32_t step_of(bool mn) { return mn ? 2048u >> 4 : 32u >> 4; }

// ------------------------------------------------------------------ tiles
struct Tile {
  int e, m0;     // expert, first feature
  int lo, hi;    // rows form: rows of the tile; weights form: rows of the expert
  int n0, cols;  // weights form: first column and columns; rows form: columns = rows
  int blocks;    // of 64 contraction values
};

template <int FORM, int CG, int BN>
struct Tiles {
  const GroupArgs& a;
  const int *gs, *ts;  // first row and first tile of every group
  int mt, nt, e = 0;
  __device__ Tiles(const GroupArgs& args, const int* rows, const int* tiles) : a(args), gs(rows), ts(tiles) {
    mt = (a.N + 128 * CG - 1) / (128 * CG);
    nt = (a.K + BN - 1) / BN;
  }
  __device__ int total() const { return FORM == WEIGHTS ? a.E * mt * nt : ts[a.E + 1]; }
  __device__ Tile at(int tile) {  // in increasing order
    Tile t;
    if (FORM == WEIGHTS) {
      t.e = tile / (mt * nt);
      const int rest = tile - t.e * mt * nt, n = rest / mt;
      t.m0 = (rest - n * mt) * 128 * CG;
      t.n0 = n * BN;
      t.cols = min(BN, a.K - t.n0);
      t.lo = gs[t.e];
      t.hi = gs[t.e + 1];
      t.blocks = (t.hi - t.lo + 63) / 64;
    } else {
      for (int end = a.E; e < end;) {  // the first group from e on that ends behind the tile
        const int mid = (e + end) / 2;
        if (tile >= ts[mid + 1]) e = mid + 1;
        else end = mid;
      }
      const int rest = tile - ts[e], n = rest / mt;
      t.e = e;
      t.m0 = (rest - n * mt) * 128 * CG;
      t.lo = gs[e] + n * BN;
      t.hi = min(t.lo + BN, gs[e + 1]);
      t.n0 = 0;
      t.cols = t.hi - t.lo;
      t.blocks = e < a.E ? (a.K + 63) / 64 : 0;  // group E: the rows of no expert
    }
    return t;
  }
};

__device__ __forceinline__ uint32_t pack_two(float lo, float hi, int type) {
  return type == FS_TYPE_BF16 ? from_two(lo, hi, __nv_bfloat16()) : from_two(lo, hi, __half());
}

// 32 lanes x 32 columns of an accumulator as 16-bit values into a warp's staging tile of 32 rows of 64 bytes, whose 16-byte
// chunks are exchanged so that neither side meets bank conflicts. FLIP: rows are columns of the accumulator.
__device__ __forceinline__ uint32_t staged(uint32_t base, int row, int chunk) {
  return base + row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4);
}
// The accumulator's values as the tensor core's fragments: of 16 TMEM lanes (h) and 8 columns (i), a lane holds columns
// 2 (lane % 4) and the next one of rows lane / 4 (g = 0) and lane / 4 + 8 (g = 1), in r[16 h + 4 i + 2 g].
__device__ __forceinline__ void read_block(uint32_t tmem, uint32_t (&r)[32]) {
#pragma unroll
  for (int h = 0; h < 2; ++h)
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[16 * h]), "=r"(r[16 * h + 1]), "=r"(r[16 * h + 2]), "=r"(r[16 * h + 3]), "=r"(r[16 * h + 4]), "=r"(r[16 * h + 5]),
          "=r"(r[16 * h + 6]), "=r"(r[16 * h + 7]), "=r"(r[16 * h + 8]), "=r"(r[16 * h + 9]), "=r"(r[16 * h + 10]),
          "=r"(r[16 * h + 11]), "=r"(r[16 * h + 12]), "=r"(r[16 * h + 13]), "=r"(r[16 * h + 14]), "=r"(r[16 * h + 15])
        : "r"(tmem + ((uint32_t)(16 * h) << 16))
        : "memory");
}
template <bool FLIP>
__device__ __forceinline__ void stage_block(const uint32_t (&r)[32], uint32_t base, int lane, int type) {
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      uint32_t m[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        m[i] = pack_two(__uint_as_float(r[16 * h + 4 * i + 2 * g]), __uint_as_float(r[16 * h + 4 * i + 2 * g + 1]), type);
      if (FLIP)
        asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(staged(base, lane, 2 * h + g)),
                     "r"(m[0]), "r"(m[1]), "r"(m[2]), "r"(m[3])
                     : "memory");
      else
        asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1, %2, %3, %4};"
                     ::"r"(staged(base, 16 * h + 8 * g + (lane & 7), lane >> 3)), "r"(m[0]), "r"(m[1]), "r"(m[2]), "r"(m[3])
                     : "memory");
    }
}
// rows x cols values (at most 32 x 32) of the staging tile, or `fill` (two values) throughout, to out, rows ld values apart.
__device__ __forceinline__ void write_block(uint16_t* out, long long ld, int rows, int cols, int vec, bool filled, uint32_t fill, uint32_t base,
                                            int lane) {
  if (vec == 8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 8 * i + (lane >> 2), c = lane & 3;
      uint4 v = make_uint4(fill, fill, fill, fill);
      if (!filled) asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(staged(base, r, c)));
      if (r < rows && 8 * c < cols) *reinterpret_cast<uint4*>(out + r * ld + 8 * c) = v;
    }
  } else if (vec == 2) {
#pragma unroll 4
    for (int i = 0; i < 16; ++i) {
      const int r = 2 * i + (lane >> 4), c = 2 * (lane & 15);
      uint32_t v = fill;
      if (!filled) asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(staged(base, r, c >> 3) + (c & 7) * 2));
      if (r < rows && c < cols) *reinterpret_cast<uint32_t*>(out + r * ld + c) = v;
    }
  } else {
#pragma unroll 4
    for (int r = 0; r < 32; ++r) {
      uint16_t v = (uint16_t)fill;
      if (!filled) asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(staged(base, r, lane >> 3) + (lane & 7) * 2));
      if (r < rows && lane < cols) out[r * ld + lane] = v;
    }
  }
}

// A row number that nothing waits for before it is used.
__device__ __forceinline__ int load_early(const int* p) {
  int v;
  asm volatile("ld.global.nc.b32 %0, [%1];" : "=r"(v) : "l"(p));
  return v;
}

// COPY (rows form, single CTAs): the rows come one by one.
template <int FORM, int CG, int BN, bool COPY>
__global__ void __launch_bounds__(kThreads + (COPY ? 32 * kCopyWarps : 0), 1)
group_kernel(const GroupArgs a, const __grid_constant__ CUtensorMap mapA, const __grid_constant__ CUtensorMap mapB) {
  constexpr int BNC = BN / CG;                         // columns whose operand this CTA fetches
  constexpr uint32_t kA = 2 * kHalfTile, kB = BNC * 128, kStage = kA + kB;
  constexpr bool A_MN = FORM != ROWS_K, B_MN = FORM == WEIGHTS;
  constexpr uint32_t kColumns = 2 * BN;
  static_assert(kColumns >= 32 && kColumns <= 512 && kStage % 1024 == 0 && !(COPY && (FORM == WEIGHTS || CG == 2)), "tile");
  extern __shared__ uint8_t raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  uint8_t* staging = ring + (size_t)a.nstage * kStage;  // 2 KB for each warp that writes results
  uint64_t* bars = reinterpret_cast<uint64_t*>(staging + kStaging);
  const int FULL = 0, EMPTY = a.nstage, PARTS = 2 * a.nstage, ACC_FULL = 3 * a.nstage, ACC_EMPTY = ACC_FULL + 2, DRAIN = ACC_EMPTY + 2;
  uint32_t* slot = reinterpret_cast<uint32_t*>(bars + DRAIN + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(slot + 1);
  int *gs = reinterpret_cast<int*>(slot + 2), *ts = gs + a.E + 2;
  auto bar = [&](int i) { return smem_u32(bars + i); };

  // from a shuffle, so that the compiler knows the roles' branches to be uniform and keeps operands in uniform registers
  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int rank = CG == 2 ? (int)cta_rank() : 0;
  const int first = blockIdx.x / CG, stride = gridDim.x / CG;

  if (warp == 0) {
    read_groups<FORM != WEIGHTS>(a.offsets, a.E, a.R, gs, ts, (a.N + 128 * CG - 1) / (128 * CG), BN);
  } else if (warp == kLoadWarp && lane == 0) {
    for (int s = 0; s < a.nstage; ++s) {
      mbar_init(bar(FULL + s), CG + (COPY ? 1 : 0));  // in CTA 0: both CTAs' loads; with COPY, the load and the report
      mbar_init(bar(EMPTY + s), 1);
      mbar_init(bar(PARTS + s), COPY ? kCopyGroup : 1);  // what the reporting warp waits for
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar(ACC_FULL + i), 1);
      mbar_init(bar(ACC_EMPTY + i), kOutWarps * CG);  // in CTA 0: every warp of the pair that writes results
    }
    mbar_init(bar(DRAIN), 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  } else if (warp == kMmaWarp) {
    alloc_columns<CG>(smem_u32(slot), kColumns);
  }
  tc_fence_before();
  __syncthreads();
  if (CG == 2) cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem = *slot;
  Tiles<FORM, CG, BN> tiles(a, gs, ts);
  const int total = tiles.total();
  int issued = 0;  // stages that this CTA's loading thread has started
  auto full_bar = [&](int s) { return CG == 2 ? in_leader(bar(FULL + s)) : bar(FULL + s); };

  if (warp == kLoadWarp) {
    // ===================== whole tiles =====================
    int s = 0;
    uint32_t ph = 0;
    bool ok = true;
    if (elect_one()) {
      for (int it = first; ok && it < total; it += stride) {
        const Tile t = tiles.at(it);
        const int npc = (t.cols + 16 * CG - 1) / (16 * CG) * 16;  // columns of the product that this CTA fetches
        const int m0 = t.m0 + rank * 128;
        for (int kb = 0; kb < t.blocks; ++kb) {
          if (!mbar_wait(bar(EMPTY + s), ph ^ 1, abort_flag)) {
            ok = false;
            break;
          }
          const uint32_t full = full_bar(s), dst = smem_u32(ring + (size_t)s * kStage);
          if (FORM == WEIGHTS) {  // a block that ends inside of a step goes by way of warp kReportWarp
            const int i0 = t.lo + kb * 64;
            const bool open = kb == t.blocks - 1 && (t.hi - t.lo) % 16 != 0;
            const uint32_t to = open ? bar(PARTS + s) : full;
            if (open) mbar_expect_tx(to, kStage);
            else expect_at<CG>(to, kStage);
#pragma unroll
            for (int c = 0; c < 2; ++c) load_2d<CG>(dst + c * kHalfTile, &mapA, m0 + c * 64, i0, to);
#pragma unroll
            for (int c = 0; c < BNC / 64; ++c) load_2d<CG>(dst + kA + c * kHalfTile, &mapB, t.n0 + rank * npc + c * 64, i0, to);
          } else {
            expect_at<CG>(full, kA + (COPY ? 0u : kB));
            if (FORM == ROWS_K) {
              load_3d<CG>(dst, &mapA, kb * 64, m0, t.e, full);
            } else {
              load_3d<CG>(dst, &mapA, m0, kb * 64, t.e, full);
              load_3d<CG>(dst + kHalfTile, &mapA, m0 + 64, kb * 64, t.e, full);
            }
            if (!COPY) load_2d<CG>(dst + kA, &mapB, kb * 64, t.lo + rank * npc, full);
          }
          ++issued;
          if (++s == a.nstage) {
            s = 0;
            ph ^= 1;
          }
        }
      }
    }
  } else if (warp == kMmaWarp) {
    // ===================== products =====================
    if (rank == 0 && elect_one()) {
      const uint32_t type = a.type == FS_TYPE_BF16 ? 1u : 0u;
      const uint32_t idesc0 = (1u << 4) | (type << 7) | (type << 10) | ((A_MN ? 1u : 0u) << 15) | ((B_MN ? 1u : 0u) << 16) |
                              ((uint32_t)(128 * CG >> 4) << 24);
      int s = 0, n = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int it = first; ok && it < total; it += stride) {
        const Tile t = tiles.at(it);
        if (t.blocks == 0) continue;
        const int np = (t.cols + 16 * CG - 1) / (16 * CG) * (16 * CG);
        const uint32_t idesc = idesc0 | ((uint32_t)(np >> 3) << 17);
        const int buf = n & 1;
        if (!mbar_wait(bar(ACC_EMPTY + buf), ((n >> 1) & 1) ^ 1, abort_flag)) break;
        ++n;
        tc_fence_after();
        const uint32_t d = tmem + buf * BN;
        for (int kb = 0; kb < t.blocks; ++kb) {
          const bool end = CG == 2 && FORM == WEIGHTS && kb == t.blocks - 1 && (t.hi - t.lo) % 16 != 0;  // by way of warp kReportWarp
          if (!(end ? wait_acquire_cluster(bar(FULL + s), ph, abort_flag) : mbar_wait(bar(FULL + s), ph, abort_flag))) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t base = smem_u32(ring + (size_t)s * kStage);
          const uint32_t al = operand_lo<A_MN>(base), bl = operand_lo<B_MN>(base + kA);
          const int left = FORM == WEIGHTS ? t.hi - t.lo - kb * 64 : a.K - kb * 64;  // contraction values from here on
#pragma unroll
          for (int ks = 0; ks < 4; ++ks)
            if (ks * 16 < left)
              mma_f16<CG>(d, pack_desc(al + ks * step_of(A_MN), kDescHi128), pack_desc(bl + ks * step_of(B_MN), kDescHi128), idesc, kb | ks);
          commit<CG>(bar(EMPTY + s));
          if (++s == a.nstage) {
            s = 0;
            ph ^= 1;
          }
        }
        if (!ok) break;
        commit<CG>(bar(ACC_FULL + buf));
      }
    }
  } else if (warp < kOutWarps) {
    // ===================== results =====================
    // Two warps to a quarter of the TMEM lanes, with every other 32 columns each.
    const int q = warp & 3, side = warp >> 2;
    const uint32_t stage = smem_u32(staging + 2048 * warp);
    constexpr int kStep = 32 * kOutWarps / 4;
    int n = 0;
    bool lost = false;  // a wait of this CTA gave up: NaN from here on
    for (int it = first; it < total; it += stride) {
      const Tile t = tiles.at(it);
      const int f = t.m0 + rank * 128 + q * 32;  // first of this warp's features
      const int buf = n & 1;
      const bool none = t.blocks == 0;  // no products: zeros
      if (!none && !lost) {
        lost = !__all_sync(0xffffffffu, wait_blocks(bar(ACC_FULL + buf), (n >> 1) & 1, abort_flag, t.blocks, a.limit));
        ++n;
        tc_fence_after();
      }
      const bool filled = none || lost;
      const uint32_t fill = none ? 0u : 0x7fff7fffu;  // NaN in any of the types
      const uint32_t acc = tmem + buf * BN + ((uint32_t)(q * 32) << 16);
      if (f < a.N) {
        if (FORM != WEIGHTS && a.out_type == FS_TYPE_F32) {
          for (int c = 32 * side; c < t.cols; c += kStep) {
            float v[32];
            if (!filled) tmem_ld32(acc + c, v);
            float* p = static_cast<float*>(a.out) + (long long)(t.lo + c) * a.ldo + f + lane;
            if (f + lane < a.N) {
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if (c + j < t.cols) p[j * a.ldo] = filled ? __uint_as_float(fill) : v[j];
            }
          }
        } else {
          uint32_t r[32];
          if (!filled && 32 * side < t.cols) read_block(acc + 32 * side, r);
          for (int c = 32 * side; c < t.cols; c += kStep) {
            if (!filled) {
              tmem_ld_wait(r);
              stage_block<FORM != WEIGHTS>(r, stage, lane, a.out_type);
              if (c + kStep < t.cols) read_block(acc + c + kStep, r);  // on its way while this one is written
              __syncwarp();
            }
            uint16_t* out = static_cast<uint16_t*>(a.out);
            if (FORM == WEIGHTS)
              write_block(out + ((long long)t.e * a.N + f) * a.K + t.n0 + c, a.K, a.N - f, t.cols - c, a.out_vec, filled, fill, stage, lane);
            else
              write_block(out + (long long)(t.lo + c) * a.ldo + f, a.ldo, t.cols - c, a.N - f, a.out_vec, filled, fill, stage, lane);
            __syncwarp();
          }
        }
      }
      if (!filled) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (CG == 2) arrive_cluster(in_leader(bar(ACC_EMPTY + buf)));
          else mbar_arrive(bar(ACC_EMPTY + buf));
        }
      }
    }
  } else if (COPY && warp > kReportWarp) {
    // ===================== single rows =====================
    // Chunk ch of rows r, r + kCopyRows, ... of a stage, the chunk exchanged with its row as the 128-byte swizzle has it.
    // These warps only start copies; that a stage's copies are there is seen by warp kReportWarp. Row numbers are read a tile ahead:
    // what is read behind the copies comes back after them.
    constexpr int kSteps = (BNC + kCopyRows - 1) / kCopyRows;
    const int side = (threadIdx.x - kThreads) / kCopyGroup, id = (threadIdx.x - kThreads) % kCopyGroup, r = id >> 3, ch = id & 7;
    const uint32_t at = kA + r * 128 + ((ch ^ (r & 7)) << 4);
    int s = side, ahead[kSteps], turn = 0;
    uint32_t ph = 0;
    bool ok = true;
    Tiles<FORM, CG, BN> ahead_tiles = tiles;
    auto read_ahead = [&](int it) {
      if (it >= total) return;
      const Tile t = ahead_tiles.at(it);
      const int npc = (t.cols + 16 * CG - 1) / (16 * CG) * 16;
#pragma unroll
      for (int j = 0; j < kSteps; ++j) {
        const int i = t.lo + rank * npc + r + kCopyRows * j;
        ahead[j] = t.blocks && r + kCopyRows * j < npc && i < t.hi ? load_early(a.rows + i) : -1;
      }
    };
    read_ahead(first);
    for (int it = first; ok && it < total; it += stride) {
      const Tile t = tiles.at(it);
      const uint16_t* src[kSteps];
#pragma unroll
      for (int j = 0; j < kSteps; ++j)
        src[j] = (unsigned)ahead[j] < (unsigned)a.M ? static_cast<const uint16_t*>(a.x) + ahead[j] * a.ldx + ch * 8 : nullptr;
      read_ahead(it + stride);
      for (int kb = 0; kb < t.blocks; ++kb, turn ^= 1) {
        if (turn != side) continue;
        if (!__all_sync(0xffffffffu, mbar_wait(bar(EMPTY + s), ph ^ 1, abort_flag, 2000))) {
          ok = false;
          break;
        }
        const uint32_t dst = smem_u32(ring + (size_t)s * kStage) + at;
        const int valid = min(max((a.K - kb * 64 - ch * 8) * 2, 0), 16);
#pragma unroll
        for (int j = 0; j < kSteps; ++j)
          copy16(dst + j * kCopyRows * 128, src[j] && valid ? src[j] + kb * 64 : a.x, src[j] ? valid : 0);
        copy_arrive(bar(PARTS + s));
        s += 2;
        if (s >= a.nstage) {
          s -= a.nstage;
          ph ^= 1;
        }
      }
    }
    copy_wait_all();
  } else if (COPY) {
    // ===================== reports of copied stages =====================
    // Copies are ordinary writes: their completion, seen here, is made visible to the tensor core, which reads by the
    // asynchronous proxy, and reported by a thread that has no copies of its own to wait for.
    int s = 0;
    uint32_t ph = 0;
    bool ok = lane == 0;
    for (int it = first; ok && it < total; it += stride) {
      const Tile t = tiles.at(it);
      for (int kb = 0; kb < t.blocks; ++kb) {
        if (!mbar_wait(bar(PARTS + s), ph, abort_flag)) {
          ok = false;
          break;
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        mbar_arrive(bar(FULL + s));
        if (++s == a.nstage) {
          s = 0;
          ph ^= 1;
        }
      }
    }
  } else if (FORM == WEIGHTS) {
    // ===================== ends of groups =====================
    int s = 0;             // first stage of the tile
    uint32_t uses = 0;     // bit s: parity of the uses of stage s here
    long long blocks = 0;  // since the last wait, which may be tiles ago
    for (int it = first; it < total; it += stride) {
      const Tile t = tiles.at(it);
      const int rows = t.hi - t.lo, stage = (s + t.blocks - 1) % a.nstage;
      s = (s + t.blocks) % a.nstage;
      blocks += t.blocks;
      if (rows % 16 == 0) continue;
      if (!__all_sync(0xffffffffu, wait_blocks(bar(PARTS + stage), uses >> stage & 1, abort_flag, blocks, kSpinLimit))) break;
      blocks = 0;
      uses ^= 1u << stage;
      uint8_t* block = ring + (size_t)stage * kStage;
      const int from = rows & 63, chunks = ((rows + 15) / 16 * 16 - rows) * 8;  // 16-byte chunks of a half tile
      for (int c = lane; c < chunks; c += 32)
#pragma unroll
        for (int h = 0; h < 2 + BNC / 64; ++h)
          *reinterpret_cast<uint4*>(block + h * kHalfTile + from * 128 + c * 16) = make_uint4(0u, 0u, 0u, 0u);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) {
        if (CG == 2) arrive_release_cluster(full_bar(stage));
        else mbar_arrive(bar(FULL + stage));
      }
      __syncwarp();
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {  // nobody waits any more, and the flag does not change
    if (warp == kMmaWarp && rank == 0) {  // every product issued here ends before TMEM is freed
      if (elect_one()) {
        commit<CG>(bar(DRAIN));
        mbar_wait_quiet(bar(DRAIN), 0);
      }
      __syncwarp();
    } else if (warp == kLoadWarp) {
      // The copies in flight land before the CTA ends. Those of the second CTA of a pair are counted in the first one, which
      // does not know of stages that it has not started itself: the second one stays for a millisecond, hundreds of times what
      // a copy takes.
      if (elect_one()) {
        const long long t0 = clock64();
        if (rank == 0)
          for (int j = issued > a.nstage ? issued - a.nstage : 0; j < issued; ++j) wait_landed(bar(FULL + j % a.nstage), (j / a.nstage) & 1, t0);
        else
          while (clock64() - t0 < (1ll << 21)) {}
      }
      __syncwarp();
    }
  }
  if (CG == 2) cluster_sync_all();
  tc_fence_after();
  if (warp == kMmaWarp) free_columns<CG>(tmem, kColumns);
  if (threadIdx.x == 0 && *abort_flag) atomicExch(a.health, 1);
}

// ------------------------------------------------------------------ few rows
// A single token: the products of one or two rows are bound by reading their experts' weights, and tiles of 128 features put
// a token's two experts of 2048 features on 32 of 148 SMs. Here a warp takes one feature of one expert, its lanes 16 bytes of
// it at a time and four of these at once; the sums are fp32 in a fixed order. Two rows of two experts, 2048 x 2048: 4.7 us
// against 10.4 us with tiles (1.2 us of either are the launch); four rows of four experts 14.8 us against 11.3 us, so
// these go the other way.
constexpr int kFewRows = 2;  // rows of a call that go this way
constexpr int kFewWarps = 8;

// sums[r] of the rows x[r] (null: none) with the feature w.
template <typename T, int ROWS>
__device__ __forceinline__ void few_rows_dot(const T* w, const T* const (&x)[ROWS], int K, int lane, float (&sums)[ROWS]) {
  constexpr int kDeep = 4;
  const int chunks = K / 8;
#pragma unroll 1
  for (int c0 = lane; c0 < chunks; c0 += 32 * kDeep) {
    Pack<T, 8> q[kDeep], p[kDeep][ROWS];
#pragma unroll
    for (int d = 0; d < kDeep; ++d) {
      const int c = c0 + 32 * d;
      if (c < chunks) q[d] = *reinterpret_cast<const Pack<T, 8>*>(w + c * 8);
#pragma unroll
      for (int r = 0; r < ROWS; ++r)
        if (c < chunks && x[r]) p[d][r] = *reinterpret_cast<const Pack<T, 8>*>(x[r] + c * 8);
    }
#pragma unroll
    for (int d = 0; d < kDeep; ++d) {
      float a[8], b[8];
      unpack<T, 8>(q[d], a);
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        unpack<T, 8>(p[d][r], b);
        if (c0 + 32 * d < chunks && x[r])
#pragma unroll
          for (int j = 0; j < 8; ++j) sums[r] = fmaf(a[j], b[j], sums[r]);
      }
    }
  }
  if (lane < K % 8)  // values after the last 16 bytes
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
      if (x[r]) sums[r] = fmaf(to_f32(w[chunks * 8 + lane]), to_f32(x[r][chunks * 8 + lane]), sums[r]);
}

template <typename T, int ROWS>  // rows of the call, 1 or 2
__global__ void __launch_bounds__(32 * kFewWarps, 4) few_rows_kernel(const GroupArgs a, const T* w, long long w_expert, long long w_row) {
  __shared__ int first_after[2];
  const int lane = threadIdx.x & 31, i = blockIdx.y;
  // The expert of row i is the one before the first offset above i (offsets as their running maximum); a row whose
  // predecessor has the same one is left to the CTA of the expert's first row.
  if (threadIdx.x < 2) first_after[threadIdx.x] = a.E + 1;
  __syncthreads();
  int above = a.E + 1, reached = a.E + 1;  // first offset above row i, above row i - 1
  for (int j = 1 + threadIdx.x; j <= a.E; j += 32 * kFewWarps) {
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
  const int e = first_after[0] - 1;
  const int f = blockIdx.x * kFewWarps + (threadIdx.x >> 5);
  if (f >= a.N) return;
  auto store = [&](int row, float v) {
    const long long at = (long long)row * a.ldo + f;
    if (a.out_type == FS_TYPE_F32) static_cast<float*>(a.out)[at] = v;
    else static_cast<T*>(a.out)[at] = from_f32<T>(v);
  };
  if (e == a.E) {  // a row of no expert
    if (lane == 0) store(i, 0.f);
    return;
  }
  if (i > 0 && first_after[1] == first_after[0]) return;
  const int end = min(a.offsets[e + 1], a.R);
  const T* x[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const int n = i + r < end ? (a.rows ? a.rows[i + r] : i + r) : -1;
    x[r] = (unsigned)n < (unsigned)a.M ? static_cast<const T*>(a.x) + n * a.ldx : nullptr;
  }
  float sums[ROWS] = {};
  few_rows_dot<T, ROWS>(w + e * w_expert + f * w_row, x, a.K, lane, sums);
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
#pragma unroll
    for (int o = 16; o; o >>= 1) sums[r] += __shfl_xor_sync(0xffffffffu, sums[r], o);
    if (lane == r && i + r < end) store(i + r, sums[r]);
  }
}
template <typename T>
int launch_few(const GroupArgs& a, const void* w, long long w_expert, long long w_row, cudaStream_t st) {
  const dim3 grid((a.N + kFewWarps - 1) / kFewWarps, a.R);
  const T* wt = static_cast<const T*>(w);
  if (a.R == 1) few_rows_kernel<T, 1><<<grid, 32 * kFewWarps, 0, st>>>(a, wt, w_expert, w_row);
  else few_rows_kernel<T, 2><<<grid, 32 * kFewWarps, 0, st>>>(a, wt, w_expert, w_row);
  return launched(1);
}

// ------------------------------------------------------------------ host side
// 16-bit tensor of 2 or 3 dimensions, contiguous along the first; boxes of 64 x box_rows.
bool encode(CUtensorMap* map, int type, const void* base, int dims, const long long (&size)[3], const long long (&stride)[2],
            int box_rows) {
  const cuuint64_t sizes[3] = {(cuuint64_t)size[0], (cuuint64_t)size[1], (cuuint64_t)size[2]};
  const cuuint64_t strides[2] = {(cuuint64_t)stride[0] * 2, (cuuint64_t)stride[1] * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)box_rows, 1}, ones[3] = {1, 1, 1};
  const auto fn = encoder();
  return fn && fn(map, type == FS_TYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, dims,
                  const_cast<void*>(base), sizes, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
bool encode_rows(CUtensorMap* map, int type, const void* base, long long cols, long long rows, long long ld, int box_rows) {
  return encode(map, type, base, 2, {cols, rows, 1}, {ld, 0}, box_rows);
}

int no_map() { return report_error(FS_ERR_CUDA, "cuTensorMapEncodeTiled failed"); }

template <int FORM, int CG, int BN, bool COPY>
int launch_group(GroupArgs a, const CUtensorMap& mapA, const CUtensorMap& mapB, long long most_tiles, cudaStream_t st) {
  constexpr size_t kStage = 2 * kHalfTile + BN / CG * 128;
  const size_t fixed = 1024 + kStaging + 8 * (3 * 12 + 5) + 8 + 8 * ((size_t)a.E + 2);
  a.nstage = (int)((kSmemMax - fixed) / kStage);
  static_assert((kSmemMax - 1024 - kStaging - 344 - 8 * (kMaxGroups + 2)) / kStage >= 4, "stages");
  if (a.nstage > 12) a.nstage = 12;
  size_t smem = fixed + a.nstage * kStage;
  if (smem < (size_t)kSmemMin) smem = kSmemMin;
  const auto kernel = group_kernel<FORM, CG, BN, COPY>;
  static std::atomic<uint64_t> allowed{0};  // devices on which the kernel may take all shared memory
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (e == cudaSuccess && !(allowed.load(std::memory_order_relaxed) & bit)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMax);
    if (e == cudaSuccess) allowed.fetch_or(bit, std::memory_order_relaxed);
  }
  if (e != cudaSuccess) return report_error(FS_ERR_CUDA, cudaGetErrorString(e));
  if (most_tiles > 0x3fffffffll) return report_error(FS_ERR_UNSUPPORTED, "more than 2^30 tiles");
  long long grid = detail::free_ctas() / CG;
  if (grid > most_tiles) grid = most_tiles;
  if (grid < 1) grid = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)grid * CG);
  cfg.blockDim = dim3(kThreads + (COPY ? 32 * kCopyWarps : 0));
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

template <int CG, int BN>
int launch_rows(const GroupArgs& a, bool k_major, const CUtensorMap& mapA, cudaStream_t st) {
  CUtensorMap mapB = {};
  const long long tiles = ((a.R + BN - 1ll) / BN + a.E + 1) * ((a.N + 128 * CG - 1) / (128 * CG));
  if constexpr (CG == 1)
    if (a.rows)
      return k_major ? launch_group<ROWS_K, CG, BN, true>(a, mapA, mapB, tiles, st) : launch_group<ROWS_MN, CG, BN, true>(a, mapA, mapB, tiles, st);
  if (!encode_rows(&mapB, a.type, a.x, a.K, a.M, a.ldx, BN / CG)) return no_map();
  return k_major ? launch_group<ROWS_K, CG, BN, false>(a, mapA, mapB, tiles, st) : launch_group<ROWS_MN, CG, BN, false>(a, mapA, mapB, tiles, st);
}

// Tile of the rows form: 32, 64 or 128 rows for one CTA (0, 1, 2), 128 or 256 for a pair (3, 4). The smallest with which all
// tiles are under way at once (half a tile of every group partly filled): 1024 rows of 8 groups, 512 x 512, take 6.2 us with
// 32 rows a tile and 10.0 us with 256. Where none does, by the rows of a mean group: a group of 40 rows or less is read with
// its weights anyhow, and larger tiles read the weights less often from L2. 64 groups, 2048 -> 1024, us with tiles 0 to 4:
// mean 24: 53 49 53 50 53, mean 64: 70 59 54 51 56, mean 192: 182 111 93 77 75, mean 512: 454 266 219 191 149.
// Rows that come one by one go to single CTAs, unless a copy into order and pairs take less: us one by one and by copy and
// product, 4 slots a token; 64 experts, 2048 -> 2048: 4096 rows 92 and 101, 8192: 130 and 123, 65536: 676 and 487; 64 experts,
// 512 -> 1024: 2048 rows 19.1 and 18.5, 65536: 121 and 93; 8 experts, 512 -> 512: 8192 rows 12.6 and 14.7, 16384: 20.2 and 20.1;
// 16 experts, 1024 -> 256: 16384 rows 17.7 and 23.4, 65536: 53 and 81, so up to 256 features they stay one by one.
constexpr int kOneByOneFeatures = 256;
int pick_rows(int R, int E, int N, bool one_by_one) {
  const int kRows[5] = {32, 64, 128, 128, 256}, ctas = detail::free_ctas();
  const int most = N > 128 && !one_by_one ? 5 : 3;  // a pair takes 256 features
  for (int i = 0; i < most; ++i) {
    const int pair = i < 3 ? 1 : 2;
    const double tiles = ((double)R / kRows[i] + 0.5 * (E < R ? E : R)) * ((N + 128 * pair - 1) / (128 * pair));
    if (tiles * pair <= ctas) return i;
  }
  const int mean = R / E, by_mean = mean < 24 ? 0 : mean < 40 ? 1 : mean < 160 ? 3 : 4;
  return by_mean < most ? by_mean : most - 1;
}

// Values of a 16-bit store: all rows start at multiples of it, and it divides the width.
int store_values(const void* out, long long ld, int width) {
  if (ld % 8 == 0 && width % 8 == 0 && aligned(out, 16)) return 8;
  return ld % 2 == 0 && width % 2 == 0 && aligned(out, 4) ? 2 : 1;
}

int check_group(int type, int R, int E, int N, int K, const int* offsets) {
  if (type != FS_TYPE_F16 && type != FS_TYPE_BF16) return report_error(FS_ERR_BAD_ARG, "type must be FS_TYPE_F16 or FS_TYPE_BF16");
  if (R < 0 || R > kMaxRows || E < 1 || E > kMaxGroups || N < 1 || K < 1 || N > (1 << 22) || K > (1 << 22))
    return report_error(FS_ERR_BAD_ARG, "R must be in [0, 2^31 - 512], E in [1, 1024], N and K in [1, 2^22]");
  if (!offsets) return report_error(FS_ERR_BAD_ARG, "null argument");
  // A thread that has launched nothing yet (autograd's) has no current context, which the encoding of tensor maps needs;
  // setting the device that is current binds it.
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaSetDevice(dev) != cudaSuccess)
    return report_error(FS_ERR_CUDA, "cannot make the current CUDA device's context current");
  return check_device();
}
// What tensor loads ask of an operand.
bool loadable(const void* p, long long ld) { return aligned(p, 16) && ld % 8 == 0; }
int not_loadable() {
  return report_error(FS_ERR_BAD_ARG, "operands must be aligned to 16 bytes, their rows and experts multiples of 8 values apart");
}

}  // namespace

long long product_limit() { return t_product_limit; }

}  // namespace ex
}  // namespace fs

using namespace fs;
using namespace fs::ex;

extern "C" {

long long fs_set_product_limit(long long clocks) {
  const long long before = t_product_limit;
  t_product_limit = clocks < 0 ? kSpinLimit : clocks;
  return before;
}

int fs_grouped_mm_in_order(int R, int E, int N) {
  if (R < 1 || E < 1 || N < 1) return 0;
  return R > kFewRows && N > kOneByOneFeatures && pick_rows(R, E, N, false) >= 3;
}

int fs_grouped_mm(const void* x, long long ldx, int M, const int* rows, int R, const void* w, long long w_expert,
                  long long w_row, long long w_col, int E, int N, int K, const int* offsets, void* out, int out_type,
                  long long ldo, int type, void* stream) {
  int s = check_group(type, R, E, N, K, offsets);
  if (s != FS_OK || R == 0) return s;
  if (!x || !w || !out || ldx < K || ldo < N || M < 1 || M > kMaxRows || (!rows && M < R) || (out_type != type && out_type != FS_TYPE_F32))
    return report_error(FS_ERR_BAD_ARG, "null argument, too few or too many rows or columns, or a wrong type of the result");
  const bool k_major = w_col == 1;
  const long long w_ld = k_major ? w_row : w_col;
  if (!k_major && w_row != 1) return report_error(FS_ERR_BAD_ARG, "w_row or w_col must be 1");
  if (w_ld < (k_major ? K : N) || w_expert < 0 || (w_expert == 0 && E > 1))
    return report_error(FS_ERR_BAD_ARG, "rows or experts of w overlap");
  if (!loadable(x, ldx) || !loadable(w, w_ld) || w_expert % 8) return not_loadable();
  GroupArgs a{};
  a.offsets = offsets; a.rows = rows; a.M = M; a.R = R; a.E = E; a.N = N; a.K = K;
  a.out = out; a.ldo = ldo; a.type = type; a.out_type = out_type; a.x = x; a.ldx = ldx;
  a.out_vec = store_values(out, ldo, N);
  a.limit = t_product_limit;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (R <= kFewRows && k_major) {
    return type == FS_TYPE_F16 ? launch_few<__half>(a, w, w_expert, w_row, st) : launch_few<__nv_bfloat16>(a, w, w_expert, w_row, st);
  }
  CUtensorMap mapA = {};
  if (!encode(&mapA, type, w, 3, {k_major ? K : N, k_major ? N : K, E}, {w_ld, w_expert ? w_expert : w_ld}, k_major ? 128 : 64))
    return no_map();
  switch (pick_rows(R, E, N, rows != nullptr)) {
    case 0: return launch_rows<1, 32>(a, k_major, mapA, st);
    case 1: return launch_rows<1, 64>(a, k_major, mapA, st);
    case 2: return launch_rows<1, 128>(a, k_major, mapA, st);
    case 3: return launch_rows<2, 128>(a, k_major, mapA, st);
    default: return launch_rows<2, 256>(a, k_major, mapA, st);
  }
}

int fs_grouped_mm_wgrad(const void* dy, long long lddy, const void* x, long long ldx, int R, int E, int N, int K,
                        const int* offsets, void* dw, int type, void* stream) {
  int s = check_group(type, R, E, N, K, offsets);
  if (s != FS_OK) return s;
  if (!dw || (R > 0 && (!dy || !x)) || lddy < N || ldx < K) return report_error(FS_ERR_BAD_ARG, "null argument, or too few columns");
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (R == 0) {
    const cudaError_t e = cudaMemsetAsync(dw, 0, (size_t)E * N * K * 2, st);
    return e == cudaSuccess ? FS_OK : report_error(FS_ERR_CUDA, cudaGetErrorString(e));
  }
  if (!loadable(dy, lddy) || !loadable(x, ldx)) return not_loadable();
  GroupArgs a{};
  a.offsets = offsets; a.R = R; a.E = E; a.N = N; a.K = K;
  a.out = dw; a.type = a.out_type = type; a.out_vec = store_values(dw, K, K);
  a.limit = t_product_limit;
  CUtensorMap mapA = {}, mapB = {};
  if (!encode_rows(&mapA, type, dy, N, R, lddy, 64) || !encode_rows(&mapB, type, x, K, R, ldx, 64)) return no_map();
  // The largest tile, unless smaller ones are all under way at once: 7 x 501 x 300 outputs of 6000 rows take 20.4 us with
  // 128 x 64, 24.2 us with 256 x 256.
  auto tiles = [&](int m, int n) { return (long long)E * ((N + m - 1) / m) * ((K + n - 1) / n); };
  const int ctas = detail::free_ctas();
  if (tiles(128, 64) <= ctas) return launch_group<WEIGHTS, 1, 64, false>(a, mapA, mapB, tiles(128, 64), st);
  if (tiles(128, 128) <= ctas || N <= 128 || K <= 128) return launch_group<WEIGHTS, 1, 128, false>(a, mapA, mapB, tiles(128, 128), st);
  return launch_group<WEIGHTS, 2, 256, false>(a, mapA, mapB, tiles(256, 256), st);
}

}  // extern "C"
