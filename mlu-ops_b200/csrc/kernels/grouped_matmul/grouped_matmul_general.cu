// Matrix products grouped by row blocks, general kernel: float, and 16-bit types
// whose sizes or addresses the tensor-core kernel cannot take.  Products and sums in
// float on the FMA units.
//
// A block computes a 128 x 64 tile of a group's result; the contracted axis is walked
// 16 at a time through shared memory, the next 16 (or the next tile's first 16) in
// flight in registers meanwhile.  A thread owns 8 x 4 sums: 12 values read from shared
// memory for 32 multiply-adds, which are issued two at a time on pairs of floats.
// All three products are the same kernel; they differ in which axis of an operand is
// contiguous.
#include <cuda_runtime.h>

#include <algorithm>
#include <type_traits>

#include "core/convert.cuh"
#include "core/launch.cuh"
#include "core/pair.cuh"
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

// A block's tile: where its operands begin, and what is left of each axis.
template <typename T>
struct Work {
  const T *a, *b;
  int64_t k_n;  // length of the contracted axis
  int group, chunk, m0, n0, m_n;  // m_n: rows of the group's result
};

// VEC: 4, all sizes are multiples of 4 and the operands are aligned to 4 values, or 1.
template <typename T, typename OutT, int MODE, int VEC>
__global__ void __launch_bounds__(kThreads)
generalKernel(const T *a, const T *b, const int32_t *ends, OutT *c, float *partial, int64_t rows, int groups, int ci,
              int co, int64_t chunk_rows, bool vector_out) {
  if (MODE == kBackwardWeight) letNextKernelStart();
  __shared__ GroupMap map;
  // read as 16-byte vectors: rows are multiples of 16 bytes
  __shared__ alignas(16) float as[kK][kM + kPad], bs[kK][kN + kPad];
  constexpr bool kWeight = MODE == kBackwardWeight;
  const int n_total = MODE == kBackwardInput ? ci : co;
  const int m_tiles = kWeight ? (ci + kM - 1) / kM : 1, n_tiles = (n_total + kN - 1) / kN, tiles = m_tiles * n_tiles;
  buildGroupMap<kWeight>(map, ends, groups, rows, kWeight ? chunk_rows : kM, tiles);
  const int units = map.first[groups + 1];
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  constexpr bool kAAlongK = !kWeight, kBAlongK = MODE == kBackwardInput;
  TileLoad<kM, VEC, kAAlongK, T> ta;
  TileLoad<kN, VEC, kBAlongK, T> tb;
  const int64_t a_pitch = MODE == kBackwardInput ? co : ci, b_pitch = co;
  auto workAt = [&](int unit) {
    Work<T> w;
    w.group = groupOfUnit(map, groups, unit);
    const int local = unit - map.first[w.group];
    const int lo = map.end[w.group], hi = map.end[w.group + 1];
    w.chunk = local / tiles;
    const int tile = local - w.chunk * tiles;
    w.n0 = tile % n_tiles * kN;
    if (kWeight) {
      const int64_t r0 = lo + w.chunk * chunk_rows;
      w.k_n = hi - r0 < chunk_rows ? hi - r0 : chunk_rows;
      w.m0 = tile / n_tiles * kM;
      w.m_n = ci;
      w.a = a + r0 * ci;
      w.b = b + r0 * co;
    } else {
      w.m0 = w.chunk * kM;
      w.m_n = hi - lo;
      w.k_n = w.group < groups ? (MODE == kForward ? ci : co) : 0;
      w.a = a + (int64_t)lo * a_pitch;
      w.b = b + (int64_t)(w.group < groups ? w.group : 0) * ci * co;
    }
    return w;
  };
  auto load = [&](const Work<T> &w, int64_t k0) {
    ta.load(w.a, a_pitch, w.m0, w.m_n, k0, w.k_n);
    tb.load(w.b, b_pitch, w.n0, n_total, k0, w.k_n);
  };
  if ((int)blockIdx.x >= units) return;
  Work<T> next = workAt(blockIdx.x);
  if (next.k_n > 0) load(next, 0);
  for (int unit = blockIdx.x; unit < units; unit += gridDim.x) {
    const Work<T> w = next;
    const bool more = unit + (int)gridDim.x < units;
    if (more) next = workAt(unit + gridDim.x);
    Two sum[8][2];
#pragma unroll
    for (int i = 0; i < 8; ++i) sum[i][0] = sum[i][1] = two(0.0f, 0.0f);
    if (w.k_n <= 0 && more && next.k_n > 0) load(next, 0);
    for (int64_t k0 = 0; k0 < w.k_n; k0 += kK) {
      __syncthreads();
      ta.store(as);
      tb.store(bs);
      __syncthreads();
      // in flight meanwhile: the next step's values, after the last step those of the next tile
      if (k0 + kK < w.k_n) load(w, k0 + kK);
      else if (more && next.k_n > 0) load(next, 0);
#pragma unroll
      for (int k = 0; k < kK; ++k) {
        const float4 x0 = *reinterpret_cast<const float4 *>(&as[k][ty * 4]);
        const float4 x1 = *reinterpret_cast<const float4 *>(&as[k][64 + ty * 4]);
        const float4 y = *reinterpret_cast<const float4 *>(&bs[k][tx * 4]);
        const Two y0 = two(y.x, y.y), y1 = two(y.z, y.w);
        const float x[8] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const Two xx = two(x[i], x[i]);
          sum[i][0] = fma(xx, y0, sum[i][0]);
          sum[i][1] = fma(xx, y1, sum[i][1]);
        }
      }
    }
    const bool split = kWeight && map.slot[w.group + 1] - map.slot[w.group] > 1;
    const int n = w.n0 + tx * 4;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int m = w.m0 + (i < 4 ? ty * 4 + i : 64 + ty * 4 + i - 4);
      if (m >= w.m_n || n >= n_total) continue;
      const float2 lo2 = mluop::split(sum[i][0]), hi2 = mluop::split(sum[i][1]);
      const float v[4] = {lo2.x, lo2.y, hi2.x, hi2.y};
      float *to_partial = split ? partial + ((int64_t)(map.slot[w.group] + w.chunk) * ci + m) * co + n : nullptr;
      const int64_t row = kWeight ? (int64_t)w.group * ci + m : (int64_t)map.end[w.group] + m;
      OutT *to = c + row * n_total + n;
      if (split) {
        if (VEC == 4) {
          *reinterpret_cast<float4 *>(to_partial) = make_float4(v[0], v[1], v[2], v[3]);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (n + j < n_total) to_partial[j] = v[j];
        }
      } else if (VEC == 4 && vector_out) {
        Pack<4, OutT> o;
#pragma unroll
        for (int j = 0; j < 4; ++j) o.v[j] = fromFloat<OutT>(v[j]);
        storePack<4>(to, o);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (n + j < n_total) to[j] = fromFloat<OutT>(v[j]);
      }
    }
  }
}

// Weight gradient: c[g] = the chunks of a split group added in ascending order.
template <typename OutT, int VEC>
__global__ void __launch_bounds__(kThreads)
addChunksKernel(const float *partial, const int32_t *ends, OutT *c, int64_t rows, int groups, int64_t elements,
                int64_t chunk_rows) {
  __shared__ GroupMap map;
  buildGroupMap<true>(map, ends, groups, rows, chunk_rows, 1);
  waitForKernelBefore();
  for (int g = 0; g < groups; ++g) {
    const int first = map.slot[g], chunks = map.slot[g + 1] - first;
    if (chunks < 2) continue;
    for (int64_t i = ((int64_t)blockIdx.x * kThreads + threadIdx.x) * VEC; i < elements; i += (int64_t)gridDim.x * kThreads * VEC) {
      const float *from = partial + (int64_t)first * elements + i;
      float v[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[j] = 0.0f;
#pragma unroll 4
      for (int k = 0; k < chunks; ++k) {
        const Pack<VEC, float> q = loadPack<VEC>(from + k * elements);
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[j] += q.v[j];
      }
      Pack<VEC, OutT> o;
#pragma unroll
      for (int j = 0; j < VEC; ++j) o.v[j] = fromFloat<OutT>(v[j]);
      storePack<VEC>(c + g * elements + i, o);
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
                                                  chunk_rows, reinterpret_cast<size_t>(c) % (4 * sizeof(OutT)) == 0);
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
  // Tensor cores, eight groups or more of a thousand rows or less on average: one unit each, which saves the second kernel.
  // 8,192 rows in half, unsplit and split, groups of one size | sizes from a log-normal of 1.2 | all rows in one group, us:
  // 13 groups of 200 x 328 15 and 31 | 16 and 24 | 46 and 25; 16 of 64 x 64 10 and 12 | 14 and 16 | 45 and 14; 4 of 64 x 64,
  // which are split, 18 and 15 | 25 and 15 | 45 and 15.  The general kernel's step is ten times as long: in float, 13 of
  // 64 x 64 42 and 43 | 104 and 41 | 482 and 39.
  if (tensor_cores && p.groups >= 8 && p.rows <= 8192) chunk = (std::max<int64_t>(p.rows, 1) + 63) / 64 * 64;
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
  trace::Scope scope("groupedMatMulAddChunksKernel", stream);
  auto launch = [&](auto *out) {
    using OutT = std::remove_pointer_t<decltype(out)>;
    const bool vectors = elements % 4 == 0 && reinterpret_cast<size_t>(c) % (4 * sizeof(OutT)) == 0;
    const int64_t threads = vectors ? elements / 4 : elements;
    const unsigned grid = (unsigned)std::min<int64_t>(8 * p.sm_count, (threads + kThreads - 1) / kThreads);
    auto kernel = vectors ? addChunksKernel<OutT, 4> : addChunksKernel<OutT, 1>;
    return launchAfterKernel(kernel, dim3(grid), dim3(kThreads), 0, stream, partial, ends, out, p.rows, p.groups, elements,
                             plan.chunk_rows);
  };
  if (p.float_weight_grad || p.dtype == MLUOP_DTYPE_FLOAT) return launch(static_cast<float *>(c));
  if (p.dtype == MLUOP_DTYPE_HALF) return launch(static_cast<__half *>(c));
  return launch(static_cast<__nv_bfloat16 *>(c));
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
