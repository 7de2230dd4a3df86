// What the kernels share whose tiles one CTA works on or a pair of CTAs on neighbouring SMs (fs_group.cu, fs_mm8.cu, fs_ortho.cu):
// PTX of pairs, and the encoding of tensor maps. Internal to the including file.
#pragma once
#include <cudaTypedefs.h>

#include <mutex>

#include "fs_ptx.cuh"

namespace fs {
namespace ex {
namespace {

using namespace fs::tc;

__device__ __forceinline__ uint32_t cta_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t in_leader(uint32_t addr) {  // the same shared-memory address in CTA 0 of the cluster
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr));
  return r;
}
__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Frees something of the leader's: only execution is ordered, for which the default scope will do.
__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// Shared memory that this CTA has written goes to the thread of the leader that issues the products reading it: released and
// acquired at the cluster's scope. For the end of a group only, once in a tile.
__device__ __forceinline__ void arrive_release_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool wait_acquire_cluster(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
  const long long t0 = clock64();
  for (;;) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    if (ok) return true;
    if (*abort_flag) return false;
    if (clock64() - t0 > kSpinLimit) {
      *abort_flag = 1;
      return false;
    }
  }
}
// For a barrier behind the products of many blocks of 64 contraction values, which take some 540 clocks each and are given
// 4096: the limit of a single wait would run out within a group of 32 million rows, whose products are one tile.
__device__ __forceinline__ bool wait_blocks(uint32_t bar, uint32_t parity, volatile int* abort_flag, long long blocks, long long limit) {
  if (limit == 0) *abort_flag = 1;  // without a look, for tests
  if (limit == 0) return false;
  if (mbar_try_wait(bar, parity)) return true;
  const long long t0 = clock64();
  limit += 4096 * blocks;
  while (!mbar_try_wait_hint(bar, parity, 2000)) {
    if (*abort_flag) return false;
    if (clock64() - t0 > limit) {
      *abort_flag = 1;
      return false;
    }
  }
  return true;
}
// For a wait that ends within a microsecond, many times in a tile: `limit` clocks at most, which only the slow way looks at.
__device__ __forceinline__ bool wait_close(uint32_t bar, uint32_t parity, volatile int* abort_flag, unsigned limit) {
  if (mbar_try_wait(bar, parity)) return true;
  const unsigned t0 = (unsigned)clock();
  while (!mbar_try_wait(bar, parity)) {
    if (*abort_flag) return false;
    if ((unsigned)clock() - t0 > limit) {
      *abort_flag = 1;
      return false;
    }
  }
  return true;
}
// A limit for it; 0: a CTA gives up at its first wait, without a look (for tests).
__host__ __device__ __forceinline__ unsigned close_limit(long long clocks) { return clocks > (1ll << 30) ? 1u << 30 : (unsigned)clocks; }
template <int CG>
__device__ __forceinline__ void load_2d(uint32_t dst, const CUtensorMap* map, int c0, int c1, uint32_t bar) {
  if (CG == 2)
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%3, %4}], [%2];"
        ::"r"(dst), "l"(map), "r"(bar), "r"(c0), "r"(c1) : "memory");
  else
    tma_load_2d(dst, map, c0, c1, bar);
}
template <int CG>
__device__ __forceinline__ void load_3d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, uint32_t bar) {
  if (CG == 2)
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%3, %4, %5}], [%2];"
        ::"r"(dst), "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(c2) : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
        ::"r"(dst), "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(c2) : "memory");
}
template <int CG>
__device__ __forceinline__ void expect_at(uint32_t bar, uint32_t bytes) {  // bar: in CTA 0 of the pair
  if (CG == 2) asm volatile("mbarrier.arrive.expect_tx.relaxed.cluster.shared::cluster.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
  else mbar_expect_tx(bar, bytes);
}
// After a wait that gave up: for the copies in flight to land, until about 0.14 s after `t0` at most.
__device__ __forceinline__ void wait_landed(uint32_t bar, uint32_t parity, long long t0) {
  while (!mbar_try_wait(bar, parity))
    if (clock64() - t0 > kSpinLimit) return;
}
template <int CG>
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if (CG == 2)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
template <int CG>
__device__ __forceinline__ void commit(uint32_t bar) {  // arrives at this barrier of every CTA of the pair
  if (CG == 2)
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
        ::"r"(bar), "h"((uint16_t)3) : "memory");
  else
    umma_commit(bar);
}
template <int CG>
__device__ __forceinline__ void alloc_columns(uint32_t slot, uint32_t n) {
  if (CG == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(n) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  } else {
    tmem_alloc(slot, n);
    tmem_relinquish();
  }
}
template <int CG>
__device__ __forceinline__ void free_columns(uint32_t addr, uint32_t n) {
  if (CG == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(n) : "memory");
  else tmem_dealloc(addr, n);
}

// The end of a kernel whose waits are bounded, for all threads, behind their roles: if one of them gave up (in either CTA of a pair), the products
// and tensor loads in flight end before TMEM and shared memory are given back. `words`, in shared memory: the stages that each of LOADERS warps has
// started, counted over the launch, and with pairs LOADERS + 1 words for what the other CTA says. A stage's full barrier (the leader's, `full` the first)
// takes one arrival of each loader of each CTA and the bytes of its loads. A loader is at most nstage stages ahead of another one, so those that
// only some of them have started are all in their barriers' present phases: the leader arrives there for the others and then waits
// for the bytes. Without anything given up this costs a pair two stores.
template <int CG, int LOADERS>
__device__ __forceinline__ void settle(volatile int* abort_flag, int* words, uint32_t full, uint32_t drain, int nstage, bool multiplies, bool loads) {
  __syncwarp();
  tc_fence_before();
  __syncthreads();  // nobody waits any more, and the flag does not change
  bool gave_up = *abort_flag != 0;
  if (CG == 2) {
    if (threadIdx.x == 0) {  // while the other CTA is there for certain
      uint32_t to;
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(smem_u32(words + LOADERS)), "r"(cta_rank() ^ 1u));
      asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(to), "r"((uint32_t)gave_up) : "memory");
#pragma unroll
      for (int i = 0; i < LOADERS; ++i) asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(to + 4 + 4 * i), "r"(words[i]) : "memory");
    }
    __syncwarp();
    cluster_sync_all();
    gave_up |= words[LOADERS] != 0;
  }
  if (gave_up) {
    if (CG == 1 || cta_rank() == 0) {
      if (multiplies) {
        if (elect_one()) {
          commit<CG>(drain);
          mbar_wait_quiet(drain, 0);
        }
      } else if (loads) {
        if (elect_one()) {
          int last = 0;
          for (int i = 0; i < CG * LOADERS; ++i) last = max(last, words[i < LOADERS ? i : i + 1]);
          for (int i = 0; i < CG * LOADERS; ++i)
            for (int j = words[i < LOADERS ? i : i + 1]; j < last; ++j) mbar_arrive(full + 8 * (j % nstage));
          const long long t0 = clock64();
          for (int j = max(last - nstage, 0); j < last; ++j) wait_landed(full + 8 * (j % nstage), (j / nstage) & 1, t0);
        }
      }
      __syncwarp();
    }
    if (CG == 2) cluster_sync_all();
  }
  tc_fence_after();
}

// First rows of the groups (running maximum of the offsets within [0, R]), of the rows of no expert (gs[E]) and the end
// (gs[E + 1]); with TILES the number of tiles before each of them. One warp.
template <bool TILES>
__device__ void read_groups(const int* offsets, int E, int R, int* gs, int* ts, int per_column, int bn) {
  const int lane = threadIdx.x & 31;
  int top = 0, sum = 0;
  if (lane == 0) gs[0] = 0;
  for (int c = 0; c <= E; c += 32) {
    const int j = c + lane;
    int end = j < E ? min(max(offsets[j + 1], 0), R) : R;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, end, o);
      end = lane >= o ? max(end, v) : end;
    }
    end = max(end, top);
    const int before = __shfl_up_sync(0xffffffffu, end, 1), begin = lane ? before : top;
    if (j <= E) gs[j + 1] = end;
    top = __shfl_sync(0xffffffffu, end, 31);
    if (TILES) {
      int n = j <= E ? (end - begin + bn - 1) / bn * per_column : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, n, o);
        n += lane >= o ? v : 0;
      }
      if (j <= E) ts[j + 1] = sum + n;
      sum += __shfl_sync(0xffffffffu, n, 31);
    }
  }
  if (TILES && lane == 0) ts[0] = 0;
}

// 16-byte chunk `chunk` of row `row` of a warp's staging tile of 32 rows of PITCH bytes (128 or 64): neither side meets bank conflicts.
template <int PITCH = 128>
__device__ __forceinline__ uint32_t staged_row(uint32_t base, int row, int chunk) {
  return base + row * PITCH + ((chunk ^ (PITCH == 128 ? row & 7 : (row >> 1) & 3)) << 4);
}
// rows x bytes (at most 32 x PITCH) of the staging tile to out, rows ld bytes apart, by stores of `vec` bytes.
template <int PITCH = 128>
__device__ __forceinline__ void write_rows(char* out, long long ld, int rows, int bytes, int vec, uint32_t base, int lane) {
  if (vec == 16) {
    constexpr int kLanes = PITCH / 16;  // to a row
#pragma unroll
    for (int i = 0; i < kLanes; ++i) {
      const int r = 32 / kLanes * i + lane / kLanes, c = lane % kLanes;
      uint4 v;
      asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(staged_row<PITCH>(base, r, c)));
      if (r < rows && 16 * c < bytes) *reinterpret_cast<uint4*>(out + r * ld + 16 * c) = v;
    }
  } else if (vec == 4) {
    constexpr int kLanes = PITCH / 4;
#pragma unroll 4
    for (int i = 0; i < kLanes; ++i) {
      const int r = 32 / kLanes * i + lane / kLanes, c = 4 * (lane % kLanes);
      uint32_t v;
      asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(staged_row<PITCH>(base, r, c >> 4) + (c & 15)));
      if (r < rows && c < bytes) *reinterpret_cast<uint32_t*>(out + r * ld + c) = v;
    }
  } else {
    constexpr int kParts = PITCH / 64;
#pragma unroll 4
    for (int i = 0; i < 32 * kParts; ++i) {
      const int r = i / kParts, c = 2 * lane + 64 * (i % kParts);
      uint16_t v;
      asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(staged_row<PITCH>(base, r, c >> 4) + (c & 15)));
      if (r < rows && c < bytes) *reinterpret_cast<uint16_t*>(out + r * ld + c) = v;
    }
  }
}
__device__ __forceinline__ void stage16(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// A warp's staging tile to the box of an output at (c0, c1), by TMA (the tile is laid out as its 128-byte swizzle has it). One lane; the tile
// is free again after bulk_read(), everything is written after bulk_done().
__device__ __forceinline__ void store_box(const CUtensorMap* map, int c0, int c1, uint32_t tile) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(map), "r"(tile), "r"(c0), "r"(c1) : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
template <int LEFT>  // but the last LEFT ones
__device__ __forceinline__ void bulk_read() { asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(LEFT) : "memory"); }
__device__ __forceinline__ void bulk_done() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

PFN_cuTensorMapEncodeTiled_v12000 encoder() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* sym = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &sym, cudaEnableDefault, &found) == cudaSuccess &&
        found == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(sym);
  });
  return fn;
}

}  // namespace
}  // namespace ex
}  // namespace fs
