// AdamW step over many tensors, states in float or in 8 bits.
//
//   g = grad * grad_scale
//   m = beta1 m + (1 - beta1) g          v = beta2 v + (1 - beta2) g^2
//   p = p (1 - lr wd) - lr / bc1 * m / (sqrt(v) / sqrt(bc2) + eps),  bc = 1 - beta^t
//
// The step touches every byte once and computes about 15 operations an element, so
// it is bound by memory: 28 bytes an element for float parameters and states, 10
// for bfloat16 parameters with 8-bit states.  One launch serves up to kMaxTensors
// tensors: their pointers travel as a kernel argument (29 KB of the 32 KB that an
// argument list may have), so nothing is copied to the device and a captured graph
// carries them.  Tensors are cut into chunks of 4096 elements, a block each; a block
// finds its tensor by bisection of the chunk counts.
//
// The order of the roundings is fixed (no contraction into fused multiply-adds): the
// values before quantisation are then the same on any path through this file, and
// two elements that tie in 8 bits tie everywhere.
//
// 8-bit states: blocks of 256 consecutive elements share a float scale, one warp
// takes one block (8 elements a lane), its largest magnitude by one warp reduction.
// m is stored as e4m3 of m / scale.  v is stored as e4m3 of sqrt(v) / scale: the
// square root halves the range of exponents that the type has to cover, and it is
// what the update divides by.  A root that is not zero is raised to the smallest
// code, 2^-9: stored as zero it would leave the next step dividing by epsilon.  The
// update itself uses m and v of this step before they are rounded to 8 bits (off by
// 2^-4 of the value at most).
#include "kernels/multi_tensor_adamw/multi_tensor_adamw_kernels.h"

#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <cmath>

#include "core/convert.cuh"
#include "core/trace.h"
#include "core/type.h"

namespace mluop {
namespace multi_tensor_adamw {

namespace {

constexpr int kThreads = 256;
constexpr int kChunk = 4096;       // elements of one block; a multiple of kScaleBlock
constexpr int kMaxTensors = 480;   // tensors of one launch
constexpr float kCodeMax = 448.0f;  // largest e4m3 value
constexpr float kSmallest = 1e-30f;  // below it a block is stored as zeros: 448 / x would leave the float range
constexpr float kCodeTiny = 0.001953125f;  // 2^-9, the smallest e4m3 value above zero

struct Constants {
  float beta1, one_minus_beta1, beta2, one_minus_beta2, epsilon;
  float decay;       // 1 - lr * weight_decay
  float root_scale;  // 1 / sqrt(1 - beta2^t)
  float step_size;   // lr / (1 - beta1^t)
};

struct TensorTable {
  const float *grad_scale;
  const float *schedule;
  double weight_decay;
  Constants c;
  int tensors;
  int first_chunk[kMaxTensors + 1];
  int64_t n[kMaxTensors];
  void *param[kMaxTensors];
  const void *grad[kMaxTensors];
  void *exp_avg[kMaxTensors];
  void *exp_avg_sq[kMaxTensors];
  float *exp_avg_scale[kMaxTensors];
  float *exp_avg_sq_scale[kMaxTensors];
};
static_assert(sizeof(TensorTable) <= 32764, "kernel arguments");

// One element: m and v are updated in place, `root` receives sqrt(v).  Returns the new parameter.
__device__ __forceinline__ float updateOne(float p, float g, float &m, float &v, float &root, const Constants &c) {
  m = __fadd_rn(__fmul_rn(m, c.beta1), __fmul_rn(g, c.one_minus_beta1));
  v = __fadd_rn(__fmul_rn(v, c.beta2), __fmul_rn(__fmul_rn(g, g), c.one_minus_beta2));
  root = __fsqrt_rn(v);
  const float change = __fdiv_rn(m, __fadd_rn(__fmul_rn(root, c.root_scale), c.epsilon));
  return __fsub_rn(__fmul_rn(p, c.decay), __fmul_rn(change, c.step_size));
}

// The step's constants: from the launch, or (schedule) from three floats on the device, in double as the host does.
__device__ __forceinline__ Constants stepConstants(const TensorTable &t) {
  Constants c = t.c;
  if (t.schedule) {
    const double lr = t.schedule[0];
    c.decay = (float)(1.0 - lr * t.weight_decay);
    c.step_size = (float)(lr / (double)t.schedule[1]);
    c.root_scale = (float)(1.0 / sqrt((double)t.schedule[2]));
  }
  return c;
}

// The tensor that chunk `chunk` belongs to (the same for all threads of a block).
__device__ __forceinline__ int findTensor(const TensorTable &t, int chunk) {
  int lo = 0, hi = t.tensors;  // first_chunk[lo] <= chunk < first_chunk[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (t.first_chunk[mid] <= chunk) lo = mid;
    else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ bool aligned16(const void *p) { return (reinterpret_cast<size_t>(p) & 15) == 0; }

template <typename P, typename G>
__global__ void __launch_bounds__(kThreads) adamWKernel(const __grid_constant__ TensorTable t) {
  const int which = findTensor(t, blockIdx.x);
  const int64_t begin = (int64_t)((int)blockIdx.x - t.first_chunk[which]) * kChunk;
  const int64_t left = t.n[which] - begin;
  const int count = left < kChunk ? (int)left : kChunk;
  P *param = static_cast<P *>(t.param[which]) + begin;
  const G *grad = static_cast<const G *>(t.grad[which]) + begin;
  float *exp_avg = static_cast<float *>(t.exp_avg[which]) + begin;
  float *exp_avg_sq = static_cast<float *>(t.exp_avg_sq[which]) + begin;
  const Constants c = stepConstants(t);
  const bool scaled = t.grad_scale != nullptr;
  const float gs = scaled ? *t.grad_scale : 1.0f;
  const bool vectors = aligned16(param) && aligned16(grad) && aligned16(exp_avg) && aligned16(exp_avg_sq);
  if (count == kChunk && vectors) {
    // 4 elements a thread and turn, all loads of the four turns in flight before the first use
    constexpr int kTurns = kChunk / (4 * kThreads);
    Pack<4, P> p[kTurns];
    Pack<4, G> g[kTurns];
    Pack<4, float> m[kTurns], v[kTurns];
#pragma unroll
    for (int i = 0; i < kTurns; ++i) {
      const int at = (i * kThreads + threadIdx.x) * 4;
      p[i] = loadPack<4>(param + at);
      g[i] = loadPack<4>(grad + at);
      m[i] = loadPack<4>(exp_avg + at);
      v[i] = loadPack<4>(exp_avg_sq + at);
    }
#pragma unroll
    for (int i = 0; i < kTurns; ++i) {
      const int at = (i * kThreads + threadIdx.x) * 4;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float gj = toFloat(g[i].v[j]), root;
        if (scaled) gj = __fmul_rn(gj, gs);
        p[i].v[j] = fromFloat<P>(updateOne(toFloat(p[i].v[j]), gj, m[i].v[j], v[i].v[j], root, c));
      }
      storePack<4>(param + at, p[i]);
      storePack<4>(exp_avg + at, m[i]);
      storePack<4>(exp_avg_sq + at, v[i]);
    }
    return;
  }
  for (int at = threadIdx.x; at < count; at += kThreads) {
    float gj = toFloat(grad[at]), root, m = exp_avg[at], v = exp_avg_sq[at];
    if (scaled) gj = __fmul_rn(gj, gs);
    param[at] = fromFloat<P>(updateOne(toFloat(param[at]), gj, m, v, root, c));
    exp_avg[at] = m;
    exp_avg_sq[at] = v;
  }
}

struct BlockScale {
  float scale, inverse;
};
// Scale of a block of 256 whose lanes hold `largest` as the bits of magnitudes (unsigned order; NaN is the
// largest, so that a NaN reaches its whole block).
__device__ __forceinline__ BlockScale blockScale(unsigned largest_bits) {
  const float largest = __uint_as_float(__reduce_max_sync(0xffffffffu, largest_bits));
  BlockScale s{0.0f, 0.0f};
  if (!(largest < kSmallest)) {
    s.inverse = __fdiv_rn(kCodeMax, largest);
    s.scale = __fmul_rn(largest, 1.0f / kCodeMax);
  }
  return s;
}
__device__ __forceinline__ unsigned magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }
__device__ __forceinline__ float rootCode(float root, float inverse) {
  const float code = __fmul_rn(root, inverse);
  return (root > 0.0f && inverse > 0.0f && code < kCodeTiny) ? kCodeTiny : code;
}
__device__ __forceinline__ float fromCode(unsigned char code) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(code, __NV_E4M3)));
}
__device__ __forceinline__ unsigned char toCode(float v) { return __nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3); }

template <typename P, typename G>
__global__ void __launch_bounds__(kThreads) adamW8BitKernel(const __grid_constant__ TensorTable t) {
  const int which = findTensor(t, blockIdx.x);
  const int64_t begin = (int64_t)((int)blockIdx.x - t.first_chunk[which]) * kChunk;
  const int64_t left = t.n[which] - begin;
  const int count = left < kChunk ? (int)left : kChunk;
  P *param = static_cast<P *>(t.param[which]) + begin;
  const G *grad = static_cast<const G *>(t.grad[which]) + begin;
  unsigned char *exp_avg = static_cast<unsigned char *>(t.exp_avg[which]) + begin;
  unsigned char *exp_avg_sq = static_cast<unsigned char *>(t.exp_avg_sq[which]) + begin;
  float *m_scales = t.exp_avg_scale[which] + begin / kScaleBlock;
  float *v_scales = t.exp_avg_sq_scale[which] + begin / kScaleBlock;
  const Constants c = stepConstants(t);
  const bool scaled = t.grad_scale != nullptr;
  const float gs = scaled ? *t.grad_scale : 1.0f;
  const bool vectors = aligned16(param) && aligned16(grad) && aligned16(exp_avg) && aligned16(exp_avg_sq);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  constexpr int kWarps = kThreads / 32;
  constexpr int kBlocks = kChunk / (int)kScaleBlock / kWarps;  // blocks of 256 a warp takes: 2
  if (count == kChunk && vectors) {
    Pack<8, P> p[kBlocks];
    Pack<8, G> g[kBlocks];
    Pack<8, unsigned char> mc[kBlocks], vc[kBlocks];
    float ms[kBlocks], vs[kBlocks];
#pragma unroll
    for (int i = 0; i < kBlocks; ++i) {
      const int block = i * kWarps + warp, at = block * (int)kScaleBlock + lane * 8;
      p[i] = loadPack<8>(param + at);
      g[i] = loadPack<8>(grad + at);
      mc[i] = loadPack<8>(exp_avg + at);
      vc[i] = loadPack<8>(exp_avg_sq + at);
      ms[i] = m_scales[block];
      vs[i] = v_scales[block];
    }
#pragma unroll
    for (int i = 0; i < kBlocks; ++i) {
      const int block = i * kWarps + warp, at = block * (int)kScaleBlock + lane * 8;
      float m[8], root[8];
      unsigned m_max = 0u, v_max = 0u;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float gj = toFloat(g[i].v[j]);
        if (scaled) gj = __fmul_rn(gj, gs);
        m[j] = __fmul_rn(fromCode(mc[i].v[j]), ms[i]);
        const float old_root = __fmul_rn(fromCode(vc[i].v[j]), vs[i]);
        float v = __fmul_rn(old_root, old_root);
        p[i].v[j] = fromFloat<P>(updateOne(toFloat(p[i].v[j]), gj, m[j], v, root[j], c));
        m_max = max(m_max, magnitude(m[j]));
        v_max = max(v_max, magnitude(root[j]));
      }
      const BlockScale m_scale = blockScale(m_max), v_scale = blockScale(v_max);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        mc[i].v[j] = toCode(__fmul_rn(m[j], m_scale.inverse));
        vc[i].v[j] = toCode(rootCode(root[j], v_scale.inverse));
      }
      storePack<8>(param + at, p[i]);
      storePack<8>(exp_avg + at, mc[i]);
      storePack<8>(exp_avg_sq + at, vc[i]);
      if (lane == 0) {
        m_scales[block] = m_scale.scale;
        v_scales[block] = v_scale.scale;
      }
    }
    return;
  }
  // a tensor's last chunk, or pointers that are not 16-byte aligned: element by element, lanes side by side
  const int blocks = (count + (int)kScaleBlock - 1) / (int)kScaleBlock;
  for (int block = warp; block < blocks; block += kWarps) {
    const float ms = m_scales[block], vs = v_scales[block];
    float m[8], root[8];
    unsigned m_max = 0u, v_max = 0u;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int at = block * (int)kScaleBlock + j * 32 + lane;
      m[j] = root[j] = 0.0f;
      if (at < count) {
        float gj = toFloat(grad[at]);
        if (scaled) gj = __fmul_rn(gj, gs);
        m[j] = __fmul_rn(fromCode(exp_avg[at]), ms);
        const float old_root = __fmul_rn(fromCode(exp_avg_sq[at]), vs);
        float v = __fmul_rn(old_root, old_root);
        param[at] = fromFloat<P>(updateOne(toFloat(param[at]), gj, m[j], v, root[j], c));
        m_max = max(m_max, magnitude(m[j]));
        v_max = max(v_max, magnitude(root[j]));
      }
    }
    const BlockScale m_scale = blockScale(m_max), v_scale = blockScale(v_max);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int at = block * (int)kScaleBlock + j * 32 + lane;
      if (at < count) {
        exp_avg[at] = toCode(__fmul_rn(m[j], m_scale.inverse));
        exp_avg_sq[at] = toCode(rootCode(root[j], v_scale.inverse));
      }
    }
    if (lane == 0) {
      m_scales[block] = m_scale.scale;
      v_scales[block] = v_scale.scale;
    }
  }
}

template <typename P, typename G>
cudaError_t launchTable(const TensorTable &t, bool state_8bit, int chunks, double bytes, cudaStream_t stream) {
  if (state_8bit) {
    trace::Scope scope("adamW8BitKernel", stream, bytes);
    adamW8BitKernel<P, G><<<chunks, kThreads, 0, stream>>>(t);
  } else {
    trace::Scope scope("adamWKernel", stream, bytes);
    adamWKernel<P, G><<<chunks, kThreads, 0, stream>>>(t);
  }
  return cudaGetLastError();
}

cudaError_t dispatch(const AdamWProblem &p, const TensorTable &t, int chunks, double bytes, cudaStream_t stream) {
  const bool float_grad = p.grad_dtype == MLUOP_DTYPE_FLOAT;
  switch (p.param_dtype) {
    case MLUOP_DTYPE_FLOAT: return launchTable<float, float>(t, p.state_8bit, chunks, bytes, stream);
    case MLUOP_DTYPE_HALF:
      return float_grad ? launchTable<__half, float>(t, p.state_8bit, chunks, bytes, stream)
                        : launchTable<__half, __half>(t, p.state_8bit, chunks, bytes, stream);
    default:
      return float_grad ? launchTable<__nv_bfloat16, float>(t, p.state_8bit, chunks, bytes, stream)
                        : launchTable<__nv_bfloat16, __nv_bfloat16>(t, p.state_8bit, chunks, bytes, stream);
  }
}

}  // namespace

cudaError_t launchMultiTensorAdamW(const AdamWProblem &p, cudaStream_t stream) {
  TensorTable t;
  t.grad_scale = p.grad_scale;
  t.schedule = p.schedule;
  t.weight_decay = p.weight_decay;
  t.c.beta1 = (float)p.beta1;
  t.c.one_minus_beta1 = (float)(1.0 - p.beta1);
  t.c.beta2 = (float)p.beta2;
  t.c.one_minus_beta2 = (float)(1.0 - p.beta2);
  t.c.epsilon = (float)p.epsilon;
  t.c.decay = (float)(1.0 - p.lr * p.weight_decay);
  t.c.step_size = (float)(p.lr / (1.0 - std::pow(p.beta1, (double)p.step)));
  t.c.root_scale = (float)(1.0 / std::sqrt(1.0 - std::pow(p.beta2, (double)p.step)));
  const double element_bytes = 2.0 * mluop::getSizeOfDataType(p.param_dtype) +
                               (double)mluop::getSizeOfDataType(p.grad_dtype) + (p.state_8bit ? 4.0 : 16.0);
  int64_t i = 0;
  while (i < p.tensor_num) {
    int64_t chunks = 0, elements = 0;
    int k = 0;
    for (; i < p.tensor_num && k < kMaxTensors; ++i) {
      const int64_t n = p.element_num[i];
      if (n == 0) continue;
      const int64_t more = (n + kChunk - 1) / kChunk;
      if (k > 0 && chunks + more > INT32_MAX) break;  // (one tensor of 2^40 elements has 2^28 chunks)
      t.first_chunk[k] = (int)chunks;
      t.n[k] = n;
      t.param[k] = p.param[i];
      t.grad[k] = p.grad[i];
      t.exp_avg[k] = p.exp_avg[i];
      t.exp_avg_sq[k] = p.exp_avg_sq[i];
      t.exp_avg_scale[k] = p.state_8bit ? p.exp_avg_scale[i] : nullptr;
      t.exp_avg_sq_scale[k] = p.state_8bit ? p.exp_avg_sq_scale[i] : nullptr;
      chunks += more;
      elements += n;
      ++k;
    }
    if (k == 0) break;
    t.first_chunk[k] = (int)chunks;
    t.tensors = k;
    const cudaError_t err = dispatch(p, t, (int)chunks, element_bytes * elements, stream);
    if (err != cudaSuccess) return err;
  }
  return cudaSuccess;
}

}  // namespace multi_tensor_adamw
}  // namespace mluop
