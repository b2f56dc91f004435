// Matrix products grouped by row blocks, general kernel: float, and 16-bit types
// whose sizes or addresses the tensor-core kernel cannot take.  Products and sums in
// float on the FMA units.
//
// A block computes a 128 x 64 tile of a group's result; the contracted axis is walked
// 16 at a time through shared memory, the next 16 in flight in registers meanwhile.
// A thread owns 8 x 4 sums: 12 values read from shared memory for 32 multiply-adds.
// All three products are the same kernel; they differ in which axis of an operand is
// contiguous.
#include <cuda_runtime.h>

#include <algorithm>

#include "core/convert.cuh"
#include "core/trace.h"
#include "core/type.h"
#include "kernels/grouped_matmul/grouped_matmul_device.cuh"
#include "kernels/grouped_matmul/grouped_matmul_kernels.h"

namespace mluop {
namespace grouped_matmul {

namespace {

constexpr int kThreads = 256;
constexpr int kM = 128, kN = 64, kK = 16;
constexpr int kPad = 4;

// Up to VEC values from p on, `left` of them inside the tensor; zeros for the others.
template <int VEC, typename T>
__device__ __forceinline__ void fetch(const T *p, int left, float (&v)[VEC]) {
  if (VEC > 1 && left >= VEC) {
    const Pack<VEC, T> q = loadPack<VEC>(p);
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[j] = toFloat(q.v[j]);
  } else {
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[j] = j < left ? toFloat(p[j]) : 0.0f;
  }
}

// A tile of an operand: `kOuter` entries of its result axis by kK of the contracted axis, kept in registers
// between the load and the store to shared memory ([contracted][result axis]).
// kAlongK: the contracted axis is contiguous in memory.
template <int OUTER, int VEC, bool ALONG_K, typename T>
struct TileLoad {
  static constexpr int kPerThread = OUTER * kK / kThreads;
  static constexpr int kVectors = kPerThread / VEC;
  float v[kVectors][VEC];
  __device__ __forceinline__ void load(const T *base, int64_t pitch, int outer0, int outer_n, int64_t k0, int64_t k_n) {
#pragma unroll
    for (int i = 0; i < kVectors; ++i) {
      const int e = (i * kThreads + (int)threadIdx.x) * VEC;
      const int outer = ALONG_K ? e / kK : e % OUTER, k = ALONG_K ? e % kK : e / OUTER;
      const int64_t kk = k0 + k;
      const int oo = outer0 + outer;
      int left = 0;
      const T *p = base;
      if (ALONG_K) {
        if (oo < outer_n && kk < k_n) {
          left = k_n - kk < VEC ? (int)(k_n - kk) : VEC;
          p = base + (int64_t)oo * pitch + kk;
        }
      } else if (oo < outer_n && kk < k_n) {
        left = outer_n - oo < VEC ? outer_n - oo : VEC;
        p = base + kk * pitch + oo;
      }
      fetch<VEC>(p, left, v[i]);
    }
  }
  __device__ __forceinline__ void store(float (*smem)[OUTER + kPad]) const {
#pragma unroll
    for (int i = 0; i < kVectors; ++i) {
      const int e = (i * kThreads + (int)threadIdx.x) * VEC;
      const int outer = ALONG_K ? e / kK : e % OUTER, k = ALONG_K ? e % kK : e / OUTER;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        if (ALONG_K) smem[k + j][outer] = v[i][j];
        else smem[k][outer + j] = v[i][j];
      }
    }
  }
};

// c_n: columns of the result; contracted: length of the contracted axis (forward, input gradient).
template <typename T, typename OutT, int MODE, int VEC>
__global__ void __launch_bounds__(kThreads)
generalKernel(const T *a, const T *b, const int32_t *ends, OutT *c, float *partial, int64_t rows, int groups, int ci,
              int co, int64_t chunk_rows) {
  __shared__ GroupMap map;
  // read as 16-byte vectors: rows are multiples of 16 bytes
  __shared__ alignas(16) float as[kK][kM + kPad], bs[kK][kN + kPad];
  constexpr bool kWeight = MODE == kBackwardWeight;
  const int n_total = MODE == kBackwardInput ? ci : co;
  const int m_tiles = kWeight ? (ci + kM - 1) / kM : 1, n_tiles = (n_total + kN - 1) / kN;
  buildGroupMap<kWeight>(map, ends, groups, rows, kWeight ? chunk_rows : kM, m_tiles * n_tiles);
  const int units = map.first[groups + 1];
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  for (int unit = blockIdx.x; unit < units; unit += gridDim.x) {
    const int g = groupOfUnit(map, groups, unit);
    const int local = unit - map.first[g];
    const int lo = map.end[g], hi = map.end[g + 1];
    const int chunk = local / (m_tiles * n_tiles), tile = local % (m_tiles * n_tiles);
    const int n0 = tile % n_tiles * kN;
    int m0, m_n;       // first row of the tile and rows of the result
    int64_t k_n;       // length of the contracted axis
    const T *pa, *pb;
    if (kWeight) {
      const int64_t r0 = lo + chunk * chunk_rows;
      k_n = hi - r0 < chunk_rows ? hi - r0 : chunk_rows;
      m0 = tile / n_tiles * kM;
      m_n = ci;
      pa = a + r0 * ci;
      pb = b + r0 * co;
    } else {
      m0 = chunk * kM;
      m_n = hi - lo;
      k_n = g < groups ? (MODE == kForward ? ci : co) : 0;
      pa = a + (int64_t)lo * (MODE == kForward ? ci : co);
      pb = b + (int64_t)(g < groups ? g : 0) * ci * co;
    }
    constexpr bool kAAlongK = !kWeight, kBAlongK = MODE == kBackwardInput;
    TileLoad<kM, VEC, kAAlongK, T> ta;
    TileLoad<kN, VEC, kBAlongK, T> tb;
    const int64_t a_pitch = kWeight ? ci : (MODE == kForward ? ci : co), b_pitch = co;
    float sum[8][4];
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) sum[i][j] = 0.0f;
    if (k_n > 0) {
      ta.load(pa, a_pitch, m0, m_n, 0, k_n);
      tb.load(pb, b_pitch, n0, n_total, 0, k_n);
    }
    for (int64_t k0 = 0; k0 < k_n; k0 += kK) {
      __syncthreads();
      ta.store(as);
      tb.store(bs);
      __syncthreads();
      if (k0 + kK < k_n) {
        ta.load(pa, a_pitch, m0, m_n, k0 + kK, k_n);
        tb.load(pb, b_pitch, n0, n_total, k0 + kK, k_n);
      }
#pragma unroll
      for (int k = 0; k < kK; ++k) {
        alignas(16) float x[8], y[4];
        *reinterpret_cast<float4 *>(&x[0]) = *reinterpret_cast<const float4 *>(&as[k][ty * 4]);
        *reinterpret_cast<float4 *>(&x[4]) = *reinterpret_cast<const float4 *>(&as[k][64 + ty * 4]);
        *reinterpret_cast<float4 *>(&y[0]) = *reinterpret_cast<const float4 *>(&bs[k][tx * 4]);
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) sum[i][j] = fmaf(x[i], y[j], sum[i][j]);
      }
    }
    const bool split = kWeight && map.slot[g + 1] - map.slot[g] > 1;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int m = m0 + (i < 4 ? ty * 4 + i : 64 + ty * 4 + i - 4);
      if (m >= m_n) continue;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int n = n0 + tx * 4 + j;
        if (n >= n_total) continue;
        if (split) {
          partial[((int64_t)(map.slot[g] + chunk) * ci + m) * co + n] = sum[i][j];
        } else {
          const int64_t row = kWeight ? (int64_t)g * ci + m : (int64_t)lo + m;
          c[row * n_total + n] = fromFloat<OutT>(sum[i][j]);
        }
      }
    }
  }
}

// Weight gradient: c[g] = the chunks of a split group added in ascending order.
template <typename OutT>
__global__ void __launch_bounds__(kThreads)
addChunksKernel(const float *partial, const int32_t *ends, OutT *c, int64_t rows, int groups, int64_t elements,
                int64_t chunk_rows) {
  __shared__ GroupMap map;
  buildGroupMap<true>(map, ends, groups, rows, chunk_rows, 1);
  for (int g = 0; g < groups; ++g) {
    const int first = map.slot[g], chunks = map.slot[g + 1] - first;
    if (chunks < 2) continue;
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < elements; i += (int64_t)gridDim.x * kThreads) {
      float v = 0.0f;
      for (int k = 0; k < chunks; ++k) v += partial[(int64_t)(first + k) * elements + i];
      c[g * elements + i] = fromFloat<OutT>(v);
    }
  }
}

template <typename T, typename OutT, int MODE>
cudaError_t launchMode(const Problem &p, const void *a, const void *b, const int32_t *ends, void *c, float *partial,
                       int64_t chunk_rows, cudaStream_t stream) {
  const size_t align = 4 * sizeof(T);
  auto ok = [&](const void *q) { return reinterpret_cast<size_t>(q) % align == 0; };
  const bool vectors = p.ci % 4 == 0 && p.co % 4 == 0 && ok(a) && ok(b);
  auto kernel = vectors ? generalKernel<T, OutT, MODE, 4> : generalKernel<T, OutT, MODE, 1>;
  const double size = mluop::getSizeOfDataType(p.dtype);
  trace::Scope scope("groupedMatMulGeneralKernel", stream,
                     size * ((double)p.rows * (p.ci + p.co) + (double)p.groups * p.ci * p.co),
                     2.0 * p.rows * p.ci * p.co);
  kernel<<<4 * p.sm_count, kThreads, 0, stream>>>(static_cast<const T *>(a), static_cast<const T *>(b), ends,
                                                  static_cast<OutT *>(c), partial, p.rows, p.groups, p.ci, p.co,
                                                  chunk_rows);
  return cudaGetLastError();
}

template <typename T>
cudaError_t launchType(const Problem &p, const void *a, const void *b, const int32_t *ends, void *c, void *workspace,
                       cudaStream_t stream) {
  if (p.mode == kForward) return launchMode<T, T, kForward>(p, a, b, ends, c, nullptr, kM, stream);
  if (p.mode == kBackwardInput) return launchMode<T, T, kBackwardInput>(p, a, b, ends, c, nullptr, kM, stream);
  const WeightGradPlan plan = planWeightGrad(p, false);
  char *base = reinterpret_cast<char *>((reinterpret_cast<size_t>(workspace) + 255) / 256 * 256);
  float *partial = reinterpret_cast<float *>(base + plan.partial);
  const cudaError_t err =
      p.float_weight_grad
          ? launchMode<T, float, kBackwardWeight>(p, a, b, ends, c, partial, plan.chunk_rows, stream)
          : launchMode<T, T, kBackwardWeight>(p, a, b, ends, c, partial, plan.chunk_rows, stream);
  return err != cudaSuccess ? err : launchAddChunks(p, plan, ends, partial, c, stream);
}

}  // namespace

WeightGradPlan planWeightGrad(const Problem &p, bool tensor_cores) {
  WeightGradPlan plan{};
  plan.tensor_cores = tensor_cores;
  plan.tile_m = kM;
  plan.tile_n = kN;
  if (tensor_cores) weightGradTile(p, &plan.tile_m, &plan.tile_n);
  // About four units for each block that runs at a time: a group of many rows is then spread over several blocks
  // while the others are busy with the small groups.  A chunk has 512 rows at least, so that its products outweigh
  // the tile of float sums that it writes.
  const int64_t tiles = (int64_t)((p.ci + plan.tile_m - 1) / plan.tile_m) * ((p.co + plan.tile_n - 1) / plan.tile_n);
  const int64_t blocks = (tensor_cores ? 1 : 4) * (int64_t)p.sm_count * kM / plan.tile_m;
  int64_t chunk = (p.rows * tiles + 4 * blocks - 1) / (4 * blocks);
  chunk = (std::max<int64_t>(chunk, 512) + 63) / 64 * 64;
  plan.chunk_rows = chunk;
  plan.slots = p.rows > chunk ? 2 * p.rows / chunk : 0;  // ceil(r / chunk) <= 2 r / chunk for the groups that are split
  plan.maps = 0;
  plan.partial = tensor_cores ? (size_t)p.groups * 256 : 0;
  plan.total = plan.partial + (size_t)plan.slots * p.ci * p.co * sizeof(float) + 256;
  return plan;
}

size_t weightGradWorkspaceBytes(const Problem &p) {
  return std::max(planWeightGrad(p, false).total, planWeightGrad(p, true).total);
}

cudaError_t launchAddChunks(const Problem &p, const WeightGradPlan &plan, const int32_t *ends, const float *partial,
                            void *c, cudaStream_t stream) {
  if (plan.slots == 0) return cudaSuccess;
  const int64_t elements = (int64_t)p.ci * p.co;
  const unsigned blocks = (unsigned)std::min<int64_t>(8 * p.sm_count, (elements + kThreads - 1) / kThreads);
  trace::Scope scope("groupedMatMulAddChunksKernel", stream);
  if (p.float_weight_grad || p.dtype == MLUOP_DTYPE_FLOAT) {
    addChunksKernel<float><<<blocks, kThreads, 0, stream>>>(partial, ends, static_cast<float *>(c), p.rows, p.groups,
                                                            elements, plan.chunk_rows);
  } else if (p.dtype == MLUOP_DTYPE_HALF) {
    addChunksKernel<__half><<<blocks, kThreads, 0, stream>>>(partial, ends, static_cast<__half *>(c), p.rows, p.groups,
                                                             elements, plan.chunk_rows);
  } else {
    addChunksKernel<__nv_bfloat16><<<blocks, kThreads, 0, stream>>>(partial, ends, static_cast<__nv_bfloat16 *>(c),
                                                                    p.rows, p.groups, elements, plan.chunk_rows);
  }
  return cudaGetLastError();
}

cudaError_t launchGeneral(const Problem &p, const void *a, const void *b, const int32_t *ends, void *c, void *workspace,
                          cudaStream_t stream) {
  switch (p.dtype) {
    case MLUOP_DTYPE_FLOAT: return launchType<float>(p, a, b, ends, c, workspace, stream);
    case MLUOP_DTYPE_HALF: return launchType<__half>(p, a, b, ends, c, workspace, stream);
    default: return launchType<__nv_bfloat16>(p, a, b, ends, c, workspace, stream);
  }
}

}  // namespace grouped_matmul
}  // namespace mluop
