// Matrix products grouped by row blocks on the 5th-generation tensor cores (tcgen05)
// of sm_100a: half and bfloat16 operands, float sums in tensor memory.
//
//   forward         C[r,:] = X[r,:] W[g]        A = X  (K-major),  B = W[g]   (MN-major)
//   input gradient  C[r,:] = dY[r,:] W[g]^T     A = dY (K-major),  B = W[g]   (K-major)
//   weight gradient C[g]   = X_g^T dY_g         A = X_g (MN-major), B = dY_g  (MN-major)
//
// No operand is transposed in memory: the tensor cores read either order from
// swizzled shared memory, and TMA brings 64 x 64 boxes of any of the three matrices
// there as they lie (64 x 128 where the rows are the result axis).
//
// The grid is persistent.  Every block works out from the group ends which unit (a
// tile of a group's result; for the weight gradient: of a chunk of its rows) is whose
// and takes units in stride.  Warp 0 issues the TMA loads of a ring of stages, warp 1
// the MMAs, warps 4 to 7 read the finished sums from tensor memory and write them
// while the MMAs of the next unit run into the other half of tensor memory.
//
// CTAS = 2: two blocks of a cluster share a tile of 256 x 256 (cta_group::2): each
// loads its 128 rows of A and its 128 columns of B, 32 KB a stage for 256 x 256 x 64
// multiply-adds instead of 48 KB for half of them, which is what the L2-to-SM path
// can deliver at the tensor cores' rate.  CTAS = 1 with narrower tiles serves small
// groups, where 256 rows would be mostly padding, and few groups, where the tiles
// would leave SMs without work.
//
// Ragged ends.  Forward and input gradient: a tile's rows behind its group belong to
// the next one; they are computed and not written.  Weight gradient: rows are the
// contracted axis, so the last box of a group must end with the group.  A small kernel
// writes a copy of both tensor maps for each group whose row count is the group's end;
// TMA fills what lies behind with zeros.
//
// Every wait is bounded; a waiter that gives up records an error in the handle's
// sticky word and takes its block to the common exit.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstdlib>

#include "core/convert.cuh"
#include "core/launch.cuh"
#include "core/trace.h"
#include "kernels/grouped_matmul/grouped_matmul_device.cuh"
#include "kernels/grouped_matmul/grouped_matmul_kernels.h"
#include "kernels/sparse_conv/tcgen05_primitives.cuh"

namespace mluop {
namespace grouped_matmul {

namespace {

using namespace sparse_conv::tc;

constexpr int kThreads = 256;
constexpr int kBlockRows = 128;  // rows of A and of the sums in one block
constexpr int kBlockK = 64;      // contracted axis of a stage: one 128-byte swizzle row
constexpr int kBox = 64;         // TMA boxes are kBox x kBox
constexpr int kBoxBytes = kBox * 128;
constexpr int kStagingBytes = 32 * 128;  // one epilogue warp: 32 rows of 128 bytes
constexpr long long kWaitCycles = 2000000000ll;  // a wait gives up after about one second
constexpr int kErrProducer = 0x20, kErrIssuer = 0x40, kErrAccumulator = 0x80;
constexpr int kMapBytes = 128;

template <int CTAS, int BN>
struct Config {
  static constexpr int kABytes = kBlockRows * 128;
  static constexpr int kBColumns = BN / CTAS;  // columns of B this block loads
  static constexpr int kBBytes = kBColumns * 128;
  static constexpr int kStageBytes = kABytes + kBBytes;
  static constexpr int kStages = 196608 / kStageBytes;  // 6 of 32 KB, 8 of 24 KB
  static constexpr int kTmemColumns = 2 * BN;           // two accumulators
  static constexpr size_t kSmemBytes = 1024 + (size_t)kStages * kStageBytes + 4 * kStagingBytes;
};

struct Params {
  const int32_t *ends;
  const CUtensorMap *group_maps;  // weight gradient: per group the maps of A and of B
  void *c;
  float *partial;
  int64_t rows, chunk_rows;
  int groups, ci, co;
  int bf16, float_out;
  int32_t *sticky;
  long long wait_limit;
  int test_drop_release;
};

__device__ __forceinline__ unsigned clusterRank() {
  unsigned r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;\n" : "=r"(r));
  return r;
}
__device__ __forceinline__ void clusterSync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
// Address, in the cluster's window, of what lies at `smem` in block `rank`.
__device__ __forceinline__ unsigned mapToRank(unsigned smem, unsigned rank) {
  unsigned a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(a) : "r"(smem), "r"(rank));
  return a;
}
__device__ __forceinline__ void arriveRemote(unsigned cluster_addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];\n" ::"r"(cluster_addr) : "memory");
}

// True in one lane of the (converged) warp.
__device__ __forceinline__ bool electOne() {
  unsigned r;
  asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}\n" : "=r"(r));
  return r != 0;
}

// TMA loads of one box; `bar` is an address in the cluster's window (CTAS = 2: the leading block's barrier).
template <int CTAS>
__device__ __forceinline__ void loadBox2(unsigned dst, const CUtensorMap *map, int x, int y, unsigned bar) {
  if (CTAS == 2) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], [%4];\n" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(bar)
        : "memory");
  } else {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];\n" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(bar)
        : "memory");
  }
}
template <int CTAS>
__device__ __forceinline__ void loadBox3(unsigned dst, const CUtensorMap *map, int x, int y, int z, unsigned bar) {
  if (CTAS == 2) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3, %4}], [%5];\n" ::"r"(
            dst),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
  } else {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];\n" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
  }
}
template <int CTAS>
__device__ __forceinline__ void mma(unsigned d, unsigned long long a, unsigned long long b, unsigned idesc, unsigned accumulate) {
  if (CTAS == 2) {
    asm volatile(
        "{\n.reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
  } else {
    umma(d, a, b, idesc, accumulate);
  }
}
// One arrival on the barrier (CTAS = 2: on both blocks') once every MMA issued so far has finished.
template <int CTAS>
__device__ __forceinline__ void commit(unsigned long long *bar) {
  if (CTAS == 2) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n" ::"r"(smemAddr(bar)),
        "h"((unsigned short)3)
        : "memory");
  } else {
    ummaCommit(bar);
  }
}
template <int CTAS>
__device__ __forceinline__ void allocate(unsigned *dst, unsigned columns) {
  if (CTAS == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smemAddr(dst)), "r"(columns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n" ::: "memory");
  } else {
    tmemAlloc(dst, columns);
  }
}
template <int CTAS>
__device__ __forceinline__ void deallocate(unsigned addr, unsigned columns) {
  if (CTAS == 2) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;\n" ::"r"(addr), "r"(columns));
  } else {
    tmemDealloc(addr, columns);
  }
}
// 32 lanes x 32 consecutive columns of tensor memory.
__device__ __forceinline__ void tmemLoad32(unsigned addr, unsigned (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr)
      : "memory");
}

// Operand in shared memory, 128-byte swizzle.  K-major: rows of 64 contracted values, groups of 8 rows 1024 bytes
// apart.  MN-major: 64 values of the result axis to a row, one row for each step of the contracted axis, groups of 8
// rows 1024 bytes apart, the next 64 values of the result axis kBoxBytes further.
__device__ __forceinline__ unsigned long long operandDesc(unsigned smem, bool mn_major) {
  unsigned long long d = (unsigned long long)((smem & 0x3FFFFu) >> 4);
  if (mn_major) d |= (unsigned long long)(kBoxBytes >> 4) << 16;
  d |= (unsigned long long)(1024u >> 4) << 32;
  d |= 1ull << 46;
  d |= 2ull << 61;
  return d;
}

// What a unit is.
struct Unit {
  int group, chunk;
  int row0;      // A's first row of the contracted axis (weight gradient) or of the result (otherwise)
  int m0, n0;    // the tile inside the group's result
  int m_n;       // rows of the group's result
  int k_blocks;
};
template <int MODE, int CTAS, int BN>
__device__ __forceinline__ Unit unitAt(const GroupMap &map, const Params &p, int m_tiles, int n_tiles, int unit) {
  Unit u;
  u.group = groupOfUnit(map, p.groups, unit);
  const int local = unit - map.first[u.group];
  const int lo = map.end[u.group], hi = map.end[u.group + 1];
  if (MODE == kBackwardWeight) {
    u.chunk = local / (m_tiles * n_tiles);
    const int tile = local % (m_tiles * n_tiles);
    u.row0 = lo + (int)(u.chunk * p.chunk_rows);
    const int64_t left = (int64_t)hi - u.row0;
    u.k_blocks = (int)(((left < p.chunk_rows ? left : p.chunk_rows) + kBlockK - 1) / kBlockK);
    u.m0 = tile / n_tiles * (kBlockRows * CTAS);
    u.n0 = tile % n_tiles * BN;
    u.m_n = p.ci;
  } else {
    u.chunk = 0;
    u.m0 = local / n_tiles * (kBlockRows * CTAS);
    u.n0 = local % n_tiles * BN;
    u.row0 = lo + u.m0;
    u.m_n = hi - lo;
    const int k = MODE == kForward ? p.ci : p.co;
    u.k_blocks = u.group < p.groups ? (k + kBlockK - 1) / kBlockK : 0;
  }
  return u;
}

template <typename T>
__device__ __forceinline__ unsigned pack2(float a, float b);
template <>
__device__ __forceinline__ unsigned pack2<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const unsigned *>(&h);
}
template <>
__device__ __forceinline__ unsigned pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const unsigned *>(&h);
}

// Writes a warp's 32 rows x BN columns of sums.  Each row of 128 bytes (64 16-bit columns or 32 floats) goes
// through shared memory, chunks of 16 bytes swizzled by the row, so that eight lanes write one row's 128
// consecutive bytes: a lane that wrote its own row would touch 32 rows with every store.
template <int BN>
__device__ __forceinline__ void writeSums(bool have, unsigned tmem, unsigned char *staging, void *dst, int64_t pitch,
                                          int rows, int columns, bool as_float, bool bf16) {
  const int lane = threadIdx.x & 31;
  const int width = as_float ? 32 : 64;
  const int size = as_float ? 4 : 2;
#pragma unroll 1
  for (int c0 = 0; c0 < BN && c0 < columns; c0 += width) {
    unsigned packed[32];
    if (!have) {
#pragma unroll
      for (int i = 0; i < 32; ++i) packed[i] = 0u;
    } else if (as_float) {
      tmemLoad32(tmem + c0, packed);
      tmemLoadWait();
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        unsigned v[32];
        tmemLoad32(tmem + c0 + 32 * h, v);
        tmemLoadWait();
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float a = __uint_as_float(v[2 * i]), b = __uint_as_float(v[2 * i + 1]);
          packed[16 * h + i] = bf16 ? pack2<__nv_bfloat16>(a, b) : pack2<__half>(a, b);
        }
      }
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 8; ++i)
      *reinterpret_cast<uint4 *>(staging + lane * 128 + ((i ^ (lane & 7)) << 4)) =
          make_uint4(packed[4 * i], packed[4 * i + 1], packed[4 * i + 2], packed[4 * i + 3]);
    __syncwarp();
    const int chunk = lane & 7, per = 16 / size;
    if (c0 + chunk * per < columns) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int row = i * 4 + (lane >> 3);
        if (row < rows) {
          const uint4 v = *reinterpret_cast<const uint4 *>(staging + row * 128 + ((chunk ^ (row & 7)) << 4));
          *reinterpret_cast<uint4 *>(static_cast<char *>(dst) + (row * pitch + c0 + chunk * per) * size) = v;
        }
      }
    }
  }
}

template <int MODE, int CTAS, int BN>
__global__ void __launch_bounds__(kThreads, 1)
groupedTcgen05Kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const Params p) {
  if (MODE == kBackwardWeight) letNextKernelStart();
  using Cfg = Config<CTAS, BN>;
  constexpr int S = Cfg::kStages;
  constexpr bool kWeight = MODE == kBackwardWeight;
  constexpr bool kAMn = kWeight, kBMn = MODE != kBackwardInput;
  extern __shared__ unsigned char smem_raw[];
  unsigned char *ring = reinterpret_cast<unsigned char *>((reinterpret_cast<size_t>(smem_raw) + 1023) & ~(size_t)1023);
  unsigned char *staging = ring + (size_t)S * Cfg::kStageBytes;
  __shared__ GroupMap map;
  __shared__ unsigned long long full[S], empty[S], sums_full[2], sums_empty[2], drain_bar;
  __shared__ unsigned tmem_base_s;
  __shared__ int abort_s;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const unsigned rank = CTAS == 2 ? clusterRank() : 0u;
  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbarInit(&full[s], 1);
      mbarInit(&empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbarInit(&sums_full[i], 1);
      mbarInit(&sums_empty[i], 4 * CTAS);
    }
    mbarInit(&drain_bar, 1);
    abort_s = 0;
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  // meanwhile: tensor memory and the tensor maps
  if (CTAS == 1 && warp == 2) allocate<CTAS>(&tmem_base_s, Cfg::kTmemColumns);
  if (!kWeight && threadIdx.x == 32) {
    asm volatile("prefetch.tensormap [%0];\n" ::"l"(&map_a) : "memory");
    asm volatile("prefetch.tensormap [%0];\n" ::"l"(&map_b) : "memory");
  }
  const int n_total = MODE == kBackwardInput ? p.ci : p.co;
  const int m_tiles = kWeight ? (p.ci + kBlockRows * CTAS - 1) / (kBlockRows * CTAS) : 1;
  const int n_tiles = (n_total + BN - 1) / BN;
  buildGroupMap<kWeight>(map, p.ends, p.groups, p.rows, kWeight ? p.chunk_rows : kBlockRows * CTAS, m_tiles * n_tiles);
  if (CTAS == 2) clusterSync();
  if (CTAS == 2 && warp == 2) allocate<CTAS>(&tmem_base_s, Cfg::kTmemColumns);
  tcFenceBefore();
  __syncthreads();
  if (CTAS == 2) clusterSync();  // both blocks' tensor memory is there before the first MMA writes to it
  tcFenceAfter();
  const unsigned tmem_base = tmem_base_s;
  if (kWeight) waitForKernelBefore();  // the one that writes the groups' tensor maps
  const int units = map.first[p.groups + 1];
  const int first_unit = blockIdx.x / CTAS, stride = gridDim.x / CTAS;
  volatile int *abort_flag = &abort_s;
  const ErrorSink sink{nullptr, p.sticky};
  const unsigned ring_addr = smemAddr(ring);

  if (warp == 0) {
    // ------------------------------------------------------------ loads (one elected lane issues)
    unsigned s = 0, parity = 0, issued = 0;
    bool ok = true;
    int known_group = -1;
    for (int unit = first_unit; unit < units && ok; unit += stride) {
      const Unit u = unitAt<MODE, CTAS, BN>(map, p, m_tiles, n_tiles, unit);
      if (kWeight && u.k_blocks > 0 && u.group != known_group) {
        // the group's maps were written by the kernel before this one
        known_group = u.group;
#pragma unroll
        for (int i = 0; i < 2; ++i)
          asm volatile("fence.proxy.tensormap::generic.acquire.gpu [%0], 128;\n" ::"l"(p.group_maps + 2 * u.group + i) : "memory");
      }
      const CUtensorMap *a_map = kWeight ? p.group_maps + 2 * u.group : &map_a;
      const CUtensorMap *b_map = kWeight ? p.group_maps + 2 * u.group + 1 : &map_b;
      const int b0 = u.n0 + (int)rank * Cfg::kBColumns;
      for (int kb = 0; kb < u.k_blocks; ++kb, ++issued) {
        if (issued >= S && !mbarWaitWarp(&empty[s], parity ^ 1u, abort_flag, sink, kErrProducer, p.wait_limit)) {
          ok = false;
          break;
        }
        if (electOne()) {
          if (rank == 0) mbarArriveExpectTx(&full[s], CTAS * Cfg::kStageBytes);
          const unsigned bar = CTAS == 2 ? mapToRank(smemAddr(&full[s]), 0) : smemAddr(&full[s]);
          const unsigned a_dst = ring_addr + s * Cfg::kStageBytes, b_dst = a_dst + Cfg::kABytes;
          const int k0 = kb * kBlockK;
          if (kAMn) {
#pragma unroll
            for (int i = 0; i < kBlockRows / kBox; ++i)
              loadBox2<CTAS>(a_dst + i * kBoxBytes, a_map, u.m0 + (int)rank * kBlockRows + i * kBox, u.row0 + k0, bar);
          } else {
            loadBox2<CTAS>(a_dst, a_map, k0, u.row0 + (int)rank * kBlockRows, bar);
          }
          if (kBMn) {
#pragma unroll
            for (int i = 0; i < Cfg::kBColumns / kBox; ++i) {
              if (kWeight) loadBox2<CTAS>(b_dst + i * kBoxBytes, b_map, b0 + i * kBox, u.row0 + k0, bar);
              else loadBox3<CTAS>(b_dst + i * kBoxBytes, b_map, b0 + i * kBox, k0, u.group, bar);
            }
          } else {
            loadBox3<CTAS>(b_dst, b_map, k0, b0, u.group, bar);
          }
        }
        __syncwarp();
        if (++s == S) {
          s = 0;
          parity ^= 1u;
        }
      }
    }
    if (*abort_flag) {
      // leaving early: see the copies in flight out (bounded); the other block's count on the leader's barriers
      const long long t0 = clock64();
      if (rank == 0) {
        for (unsigned i = issued > S ? issued - S : 0; i < issued; ++i) {
          while (!mbarTryWait(&full[i % S], (i / S) & 1u) && clock64() - t0 <= 1000000) {
          }
        }
      }
      while (clock64() - t0 <= 1000000) {
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (rank == 0) {
      // ---------------------------------------------------------- products
      // The whole warp walks the units, so that addresses and descriptors are the same in all lanes and live in uniform
      // registers; one elected lane issues.
      const unsigned idesc = (1u << 4) | ((unsigned)p.bf16 << 7) | ((unsigned)p.bf16 << 10) | ((kAMn ? 1u : 0u) << 15) |
                             ((kBMn ? 1u : 0u) << 16) | ((unsigned)(BN >> 3) << 17) |
                             ((unsigned)((kBlockRows * CTAS) >> 4) << 24);
      constexpr unsigned kAStep = (kAMn ? 16 * 128 : 32) >> 4, kBStep = (kBMn ? 16 * 128 : 32) >> 4;
      const unsigned long long a_desc = operandDesc(ring_addr, kAMn), b_desc = operandDesc(ring_addr + Cfg::kABytes, kBMn);
      unsigned s = 0, parity = 0, done = 0;
      bool ok = true, first = true;
      for (int unit = first_unit; unit < units && ok; unit += stride) {
        const Unit u = unitAt<MODE, CTAS, BN>(map, p, m_tiles, n_tiles, unit);
        if (u.k_blocks == 0) continue;
        const unsigned acc = done & 1u;
        if (done >= 2 && !mbarWaitWarp(&sums_empty[acc], ((done >> 1) - 1u) & 1u, abort_flag, sink, kErrIssuer, p.wait_limit)) {
          ok = false;
          break;
        }
        tcFenceAfter();
        const unsigned d = tmem_base + acc * BN;
        for (int kb = 0; kb < u.k_blocks; ++kb) {
          if (!mbarWaitWarp(&full[s], parity, abort_flag, sink, kErrIssuer, p.wait_limit)) {
            ok = false;
            break;
          }
          tcFenceAfter();
          if (electOne()) {
            // only the start-address field (16-byte units) differs between stages and steps
            const unsigned long long a = a_desc + (unsigned long long)(s * (Cfg::kStageBytes >> 4));
            const unsigned long long b = b_desc + (unsigned long long)(s * (Cfg::kStageBytes >> 4));
#pragma unroll
            for (int j = 0; j < kBlockK / 16; ++j)
              mma<CTAS>(d, a + (unsigned long long)(j * kAStep), b + (unsigned long long)(j * kBStep), idesc, kb > 0 || j > 0 ? 1u : 0u);
            // (test hook: the first release of a block is withheld, so that the loads' wait for that stage runs out)
            if (!(p.test_drop_release && first)) commit<CTAS>(&empty[s]);
            if (kb + 1 == u.k_blocks) commit<CTAS>(&sums_full[acc]);
          }
          __syncwarp();
          first = false;
          if (++s == S) {
            s = 0;
            parity ^= 1u;
          }
        }
        ++done;
      }
      if (*abort_flag && electOne()) {
        // leaving early: MMAs may still be running; tensor memory must not be freed under them
        commit<CTAS>(&drain_bar);
        const long long t0 = clock64();
        while (!mbarTryWait(&drain_bar, 0) && clock64() - t0 <= 1000000) {
        }
      }
    }
    __syncwarp();
  } else if (warp >= 4) {
    // ------------------------------------------------------------ results
    const int quarter = warp - 4;
    unsigned char *mine = staging + quarter * kStagingBytes;
    unsigned done = 0;
    for (int unit = first_unit; unit < units; unit += stride) {
      const Unit u = unitAt<MODE, CTAS, BN>(map, p, m_tiles, n_tiles, unit);
      const bool have = u.k_blocks > 0;
      const unsigned acc = done & 1u;
      if (have && !mbarWaitWarp(&sums_full[acc], (done >> 1) & 1u, abort_flag, sink, kErrAccumulator, p.wait_limit)) break;
      tcFenceAfter();
      const int m = u.m0 + (int)rank * kBlockRows + quarter * 32;  // the warp's first row in the group's result
      const int rows = u.m_n - m < 32 ? u.m_n - m : 32;
      const int columns = n_total - u.n0;
      bool as_float = false;
      char *dst = static_cast<char *>(p.c);
      if (kWeight) {
        const int chunks = map.slot[u.group + 1] - map.slot[u.group];
        as_float = p.float_out || chunks > 1;
        if (chunks > 1) {
          dst = reinterpret_cast<char *>(p.partial + ((int64_t)(map.slot[u.group] + u.chunk) * p.ci + m) * n_total + u.n0);
        } else {
          dst += (((int64_t)u.group * p.ci + m) * n_total + u.n0) * (as_float ? 4 : 2);
        }
      } else {
        dst += ((int64_t)(map.end[u.group] + m) * n_total + u.n0) * 2;
      }
      const unsigned tmem = tmem_base + acc * BN + ((unsigned)(quarter * 32) << 16);
      if (rows > 0) writeSums<BN>(have, tmem, mine, dst, n_total, rows, columns, as_float, p.bf16 != 0);
      if (have) {
        tcFenceBefore();
        __syncwarp();
        if (lane == 0) {
          if (CTAS == 2) arriveRemote(mapToRank(smemAddr(&sums_empty[acc]), 0));
          else arriveRemote(smemAddr(&sums_empty[acc]));
        }
        ++done;
      }
    }
    tcFenceBefore();
  }
  __syncthreads();
  if (CTAS == 2) clusterSync();
  if (warp == 2) {
    tcFenceAfter();
    deallocate<CTAS>(tmem_base, Cfg::kTmemColumns);
  }
}

// Weight gradient: for each group a copy of the two maps whose row count is the group's end.
__global__ void __launch_bounds__(kThreads)
groupMapsKernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const int32_t *ends,
                int groups, int64_t rows, CUtensorMap *out) {
  letNextKernelStart();
  __shared__ GroupMap map;
  buildGroupMap<true>(map, ends, groups, rows, rows, 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = blockIdx.x * (kThreads / 32) + warp; i < 2 * groups; i += gridDim.x * (kThreads / 32)) {
    const CUtensorMap *from = i & 1 ? &map_b : &map_a;
    if (lane < kMapBytes / 4)
      reinterpret_cast<unsigned *>(out + i)[lane] = reinterpret_cast<const unsigned *>(from)[lane];
    __threadfence();
    __syncwarp();
    if (lane == 0) {
      const int end = map.end[i / 2 + 1];
      asm volatile("tensormap.replace.tile.global_dim.global.b1024.b32 [%0], 1, %1;\n" ::"l"(out + i), "r"(end > 0 ? end : 1)
                   : "memory");
      asm volatile("fence.proxy.tensormap::generic.release.gpu;\n" ::: "memory");
    }
  }
}

using EncodeTiled = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                 const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encodeTiled() {
  static const EncodeTiled fn = [] {
    void *f = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess)
      f = nullptr;
    return reinterpret_cast<EncodeTiled>(f);
  }();
  return fn;
}

// Tensor map of a dense matrix or stack of matrices with `columns` contiguous 16-bit values.
bool encode(CUtensorMap *map, const void *base, bool bf16, int64_t columns, int64_t rows, int64_t depth, int box_rows) {
  const EncodeTiled fn = encodeTiled();
  if (!fn) return false;
  const cuuint64_t dims[3] = {(cuuint64_t)columns, (cuuint64_t)rows, (cuuint64_t)depth};
  const cuuint64_t strides[2] = {(cuuint64_t)columns * 2, (cuuint64_t)columns * rows * 2};
  const cuuint32_t box[3] = {kBox, (cuuint32_t)box_rows, 1}, steps[3] = {1, 1, 1};
  return fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, depth > 0 ? 3 : 2,
            const_cast<void *>(base), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int MODE, int CTAS, int BN>
cudaError_t launch(const Problem &p, const CUtensorMap &a, const CUtensorMap &b, const Params &params, int64_t most_units,
                   cudaStream_t stream) {
  using Cfg = Config<CTAS, BN>;
  auto kernel = groupedTcgen05Kernel<MODE, CTAS, BN>;
  static std::atomic<int> known_clusters{0};  // clusters of this kernel that run at a time (all devices are alike)
  cudaLaunchConfig_t config{};
  cudaLaunchAttribute attributes[2];
  attributes[0].id = cudaLaunchAttributeClusterDimension;
  attributes[0].val.clusterDim.x = CTAS;
  attributes[0].val.clusterDim.y = attributes[0].val.clusterDim.z = 1;
  attributes[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attributes[1].val.programmaticStreamSerializationAllowed = 1;
  config.blockDim = dim3(kThreads);
  config.dynamicSmemBytes = Cfg::kSmemBytes;
  config.stream = stream;
  config.attrs = attributes;
  config.numAttrs = 1;
  cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Cfg::kSmemBytes);
  if (err != cudaSuccess) return err;
  int clusters = known_clusters.load(std::memory_order_relaxed);
  if (clusters == 0) {
    clusters = p.sm_count / CTAS;
    if (CTAS > 1) {
      config.gridDim = dim3(clusters * CTAS);
      int active = 0;
      err = cudaOccupancyMaxActiveClusters(&active, kernel, &config);
      if (err != cudaSuccess) return err;
      if (active > 0 && active < clusters) clusters = active;
    }
    known_clusters.store(clusters, std::memory_order_relaxed);
  }
  config.gridDim = dim3((unsigned)std::min<int64_t>(clusters, most_units) * CTAS);
  const double rows = (double)p.rows;
  trace::Scope scope(MODE == kForward         ? "groupedTcgen05Kernel:forward"
                     : MODE == kBackwardInput ? "groupedTcgen05Kernel:input_grad"
                                              : "groupedTcgen05Kernel:weight_grad",
                     stream, 2.0 * (rows * (p.ci + p.co) + (double)p.groups * p.ci * p.co), 2.0 * rows * p.ci * p.co);
  if (MODE == kBackwardWeight) config.numAttrs = 2;  // it follows the kernel that writes the groups' tensor maps
  return cudaLaunchKernelEx(&config, kernel, a, b, params);
}

struct Tile {
  int ctas, columns;
};

// The tile for a result of `m_n` rows (on average, over the groups) and `n_n` columns.
Tile chooseTile(const Problem &p, int64_t m_n, int64_t groups, int64_t n_n) {
  auto units = [&](int64_t tm, int64_t tn) { return groups * ((m_n + tm - 1) / tm) * ((n_n + tn - 1) / tn); };
  if (m_n > 128 && n_n > 128 && units(256, 256) >= p.sm_count / 2) return {2, 256};
  if (units(128, 128) >= p.sm_count) return {1, 128};
  if (p.mode == kBackwardWeight) return {1, 64};
  // Rounds of tiles, times the rows and columns that a step brings in: steps take as long as their operands need from L2.
  // (Input gradient of 13 groups, 4,999 rows, 328 -> 200: 8.9 us with 104 tiles of 128 columns, 10.5 with 208 of 64.)
  auto cost = [&](int64_t tn) { return (units(128, tn) + p.sm_count - 1) / p.sm_count * (128 + tn); };
  return cost(128) < cost(64) ? Tile{1, 128} : Tile{1, 64};
}

Tile tileOf(const Problem &p) {
  if (p.mode == kBackwardWeight) return chooseTile(p, p.ci, p.groups, p.co);
  return chooseTile(p, (p.rows + p.groups - 1) / p.groups, p.groups, p.mode == kForward ? p.co : p.ci);
}

template <int MODE>
cudaError_t launchMode(const Problem &p, const Tile &t, const CUtensorMap &a, const CUtensorMap &b, const Params &params,
                       cudaStream_t stream) {
  const int64_t n_n = MODE == kBackwardInput ? p.ci : p.co;
  const int64_t n_tiles = (n_n + t.columns - 1) / t.columns, tm = kBlockRows * t.ctas;
  const int64_t m_units = MODE == kBackwardWeight
                              ? (p.rows / params.chunk_rows + p.groups) * ((p.ci + tm - 1) / tm)
                              : p.rows / tm + p.groups + 1;
  const int64_t most = std::max<int64_t>(1, m_units * n_tiles);
  if (t.ctas == 2) return launch<MODE, 2, 256>(p, a, b, params, most, stream);
  if (t.columns == 128) return launch<MODE, 1, 128>(p, a, b, params, most, stream);
  return launch<MODE, 1, 64>(p, a, b, params, most, stream);
}

}  // namespace

bool tensorCoresEligible(const Problem &p, const void *a, const void *b, const void *c) {
  auto ok = [](const void *q) { return reinterpret_cast<size_t>(q) % 16 == 0; };
  return p.dtype != MLUOP_DTYPE_FLOAT && p.ci % 8 == 0 && p.co % 8 == 0 && ok(a) && ok(b) && ok(c);
}

void weightGradTile(const Problem &p, int *tile_m, int *tile_n) {
  const Tile t = chooseTile(p, p.ci, p.groups, p.co);
  *tile_m = kBlockRows * t.ctas;
  *tile_n = t.columns;
}

cudaError_t launchTensorCores(const Problem &p, const void *a, const void *b, const int32_t *ends, void *c,
                              void *workspace, cudaStream_t stream) {
  const bool bf16 = p.dtype == MLUOP_DTYPE_BFLOAT16;
  const Tile tile = tileOf(p);
  Params params{};
  params.ends = ends;
  params.c = c;
  params.rows = p.rows;
  params.chunk_rows = 1;
  params.groups = p.groups;
  params.ci = p.ci;
  params.co = p.co;
  params.bf16 = bf16;
  params.float_out = p.float_weight_grad;
  params.sticky = p.sticky;
  params.wait_limit = kWaitCycles;
  // Test hook: MLUOP_B200_TEST_GROUPED_WAIT=<cycles> gives every wait that limit and withholds the first stage
  // release of every block, so that the bounded waits run out: the kernel must record the error, leave through its
  // common exit and return.  Nothing faults or spins on.
  if (const char *hook = std::getenv("MLUOP_B200_TEST_GROUPED_WAIT")) {
    const long long cycles = std::atoll(hook);
    if (cycles > 0) {
      params.wait_limit = cycles;
      params.test_drop_release = 1;
    }
  }
  CUtensorMap map_a, map_b;
  if (p.mode != kBackwardWeight) {
    if (!encode(&map_a, a, bf16, p.mode == kForward ? p.ci : p.co, p.rows, 0, kBlockRows) ||
        !encode(&map_b, b, bf16, p.co, p.ci, p.groups, p.mode == kForward ? kBox : tile.columns / tile.ctas))
      return cudaErrorInvalidValue;
    return p.mode == kForward ? launchMode<kForward>(p, tile, map_a, map_b, params, stream)
                              : launchMode<kBackwardInput>(p, tile, map_a, map_b, params, stream);
  }
  if (!encode(&map_a, a, bf16, p.ci, p.rows, 0, kBox) || !encode(&map_b, b, bf16, p.co, p.rows, 0, kBox)) return cudaErrorInvalidValue;
  const WeightGradPlan plan = planWeightGrad(p, true);
  char *base = reinterpret_cast<char *>((reinterpret_cast<size_t>(workspace) + 255) / 256 * 256);
  CUtensorMap *maps = reinterpret_cast<CUtensorMap *>(base + plan.maps);
  params.group_maps = maps;
  params.partial = reinterpret_cast<float *>(base + plan.partial);
  params.chunk_rows = plan.chunk_rows;
  {
    trace::Scope scope("groupedMapsKernel", stream);
    const int blocks = std::min((2 * p.groups + kThreads / 32 - 1) / (kThreads / 32), 32);
    groupMapsKernel<<<blocks, kThreads, 0, stream>>>(map_a, map_b, ends, p.groups, p.rows, maps);
  }
  cudaError_t err = cudaGetLastError();
  if (err == cudaSuccess) err = launchMode<kBackwardWeight>(p, tile, map_a, map_b, params, stream);
  return err != cudaSuccess ? err : launchAddChunks(p, plan, ends, params.partial, c, stream);
}

}  // namespace grouped_matmul
}  // namespace mluop
