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
// argument list may have; 2 KB for up to kFewTensors), so nothing is copied to the device and a captured graph
// carries them.  Tensors are cut into chunks of 1024 to 4096 elements, a block each; a
// block finds its tensor by bisection of the chunk counts.
//
// The moments and the root are rounded as the formula evaluated step by step is, on
// every path: a last bit that differs can tip an 8-bit code, which is 2^-4 of the
// element at the next step.
// 8-bit states: with 10 bytes an element the arithmetic is what has to be short.  It
// runs on pairs of floats, and the change of the parameter, which no code depends on,
// takes the approximate reciprocal (2^-22 of it).  Single operations and a correctly
// rounded quotient took 296 us for 10^8 bfloat16 elements, this form 210 us (1.0 GB).
// One block of 256 a warp and five blocks of threads an SM; two or four blocks a warp,
// their loads ahead of their use, were slower by 4 and 35 %.
//
// 8-bit states: blocks of 256 consecutive elements share a float scale, one warp
// takes one block (8 elements a lane), its largest magnitude by one warp reduction.
// m is stored as e4m3 of m / scale.  v is stored as e4m3 of sqrt(v) / scale: the
// square root halves the range of exponents that the type has to cover, and it is
// what the update divides by.  A root that is not zero is raised to the smallest
// code, 2^-9: stored as zero it would leave the next step dividing by epsilon.  The
// update itself uses m and v of this step before they are rounded to 8 bits (off by
// 2^-4 of the value at most).
//
// Rounding to codes.  To the nearest one, a moment that moves by less than half a code's step
// in one step stays where it is, and one that moves by 0.05 % (the root, beta2 =
// 0.999) against 3 to 6 % does so for good: 3,000 steps after the gradients of half
// the elements of a block grew fourfold, the others' roots were 3.2 times too large.
// Rounded up or down with the probability of its distance (STOCHASTIC), the stored
// value is right on average and follows: 0.99 to 1.00 of the float states' there.
// The random bits come from the step and the element alone (unitBits): no state,
// the same in a repeated call.  It takes 367 us where the nearest codes take 210: some 30
// more instructions an element in a kernel that waits for instructions.
#include "kernels/multi_tensor_adamw/multi_tensor_adamw_kernels.h"

#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cfloat>
#include <cmath>

#include "core/convert.cuh"
#include "core/pair.cuh"
#include "core/trace.h"
#include "core/type.h"

namespace mluop {
namespace multi_tensor_adamw {

namespace {

constexpr int kThreads = 256;
constexpr int kChunk = 4096;       // elements of one block, float states
constexpr int kSmallChunk = 1024;  // the same where chunks of 4096 would not fill the SMs
constexpr int kChunk8Bit = 2048;   // 8-bit states: a block of 256 for each warp
constexpr int kMaxTensors = 480;   // tensors of one launch
constexpr int kFewTensors = 32;    // so few: a shorter argument list
constexpr float kCodeMax = 448.0f;  // largest e4m3 value
constexpr float kSmallest = 1e-30f;  // below it a block is stored as zeros: 1 / x * 448 would leave the float range
constexpr float kCodeTiny = 0.001953125f;  // 2^-9, the smallest e4m3 value above zero

struct Constants {
  float beta1, one_minus_beta1, beta2, one_minus_beta2, epsilon;
  float decay;       // 1 - lr * weight_decay
  float root_scale;  // 1 / sqrt(1 - beta2^t)
  float step_size;   // lr / (1 - beta1^t)
  float one;         // 1 (see addRounded)
};

template <int MOST>
struct TensorTable {
  static constexpr int kMost = MOST;
  const float *grad_scale;
  const float *schedule;
  double weight_decay;
  int64_t step;
  const int64_t *step_count;
  Constants c;
  int tensors;
  int first_chunk[MOST + 1];
  int64_t n[MOST];
  void *param[MOST];
  const void *grad[MOST];
  void *exp_avg[MOST];
  void *exp_avg_sq[MOST];
  float *exp_avg_scale[MOST];
  float *exp_avg_sq_scale[MOST];
};
static_assert(sizeof(TensorTable<kMaxTensors>) <= 32764, "kernel arguments");

// One element: m and v are updated in place, `root` receives sqrt(v).  Returns the new parameter.
__device__ __forceinline__ float updateOne(float p, float g, float &m, float &v, float &root, const Constants &c) {
  m = __fadd_rn(__fmul_rn(m, c.beta1), __fmul_rn(g, c.one_minus_beta1));
  v = __fadd_rn(__fmul_rn(v, c.beta2), __fmul_rn(__fmul_rn(g, g), c.one_minus_beta2));
  root = __fsqrt_rn(v);
  const float change = __fdiv_rn(m, __fadd_rn(__fmul_rn(root, c.root_scale), c.epsilon));
  return __fsub_rn(__fmul_rn(p, c.decay), __fmul_rn(change, c.step_size));
}

// The step's constants: from the launch, or (schedule) from three floats on the device, in double as the host does.
template <typename Table>
__device__ __forceinline__ Constants stepConstants(const Table &t) {
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
template <typename Table>
__device__ __forceinline__ int findTensor(const Table &t, int chunk) {
  int lo = 0, hi = t.tensors;  // first_chunk[lo] <= chunk < first_chunk[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (t.first_chunk[mid] <= chunk) lo = mid;
    else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ bool aligned16(const void *p) { return (reinterpret_cast<size_t>(p) & 15) == 0; }

template <typename P, typename G, int CHUNK, typename Table>
__global__ void __launch_bounds__(kThreads) adamWKernel(const __grid_constant__ Table t) {
  const int which = findTensor(t, blockIdx.x);
  const int64_t begin = (int64_t)((int)blockIdx.x - t.first_chunk[which]) * CHUNK;
  const int64_t left = t.n[which] - begin;
  const int count = left < CHUNK ? (int)left : CHUNK;
  P *param = static_cast<P *>(t.param[which]) + begin;
  const G *grad = static_cast<const G *>(t.grad[which]) + begin;
  float *exp_avg = static_cast<float *>(t.exp_avg[which]) + begin;
  float *exp_avg_sq = static_cast<float *>(t.exp_avg_sq[which]) + begin;
  const Constants c = stepConstants(t);
  const bool scaled = t.grad_scale != nullptr;
  const float gs = scaled ? *t.grad_scale : 1.0f;
  const bool vectors = aligned16(param) && aligned16(grad) && aligned16(exp_avg) && aligned16(exp_avg_sq);
  if (count == CHUNK && vectors) {
    // 4 elements a thread and turn, all loads of the four turns in flight before the first use
    constexpr int kTurns = CHUNK / (4 * kThreads);
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

// 8-bit states.  A pair of codes as floats, and back.
__device__ __forceinline__ Two fromCodes(unsigned short codes) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(codes, __NV_E4M3);
  const float2 f = __half22float2(__half2(h));
  return two(f.x, f.y);
}
__device__ __forceinline__ unsigned short toCodes(Two t) { return __nv_cvt_float2_to_fp8x2(split(t), __NV_SATFINITE, __NV_E4M3); }

// Eight consecutive values as pairs.
template <typename T>
struct Eight {
  static constexpr int kEach = 16 / sizeof(T), kVectors = 8 / kEach;
  Values<T, kEach> v[kVectors];
  __device__ __forceinline__ void load(const T *p) {
#pragma unroll
    for (int i = 0; i < kVectors; ++i) v[i].load(p + i * kEach);
  }
  __device__ __forceinline__ Two pair(int j) const { return v[j / (kEach / 2)].pair(j % (kEach / 2)); }
  static __device__ __forceinline__ void store(T *p, const Two (&t)[4]) {
    if constexpr (kVectors == 1) {
      Values<T, kEach>::store(p, t);
    } else {
      Values<T, kEach>::store(p, {t[0], t[1]});
      Values<T, kEach>::store(p + kEach, {t[2], t[3]});
    }
  }
};

// The larger of a and |b|; NaN if either is one.
__device__ __forceinline__ float largest(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(fabsf(b)));
  return r;
}

struct Pairs {
  float one;
  Two beta1, one_minus_beta1, beta2, one_minus_beta2, epsilon, decay, root_scale, minus_step;
  __device__ __forceinline__ explicit Pairs(const Constants &c)
      : one(c.one),
        beta1(two(c.beta1, c.beta1)),
        one_minus_beta1(two(c.one_minus_beta1, c.one_minus_beta1)),
        beta2(two(c.beta2, c.beta2)),
        one_minus_beta2(two(c.one_minus_beta2, c.one_minus_beta2)),
        epsilon(two(c.epsilon, c.epsilon)),
        decay(two(c.decay, c.decay)),
        root_scale(two(c.root_scale, c.root_scale)),
        minus_step(two(-c.step_size, -c.step_size)) {}
};
// Two elements: m and root (sqrt(v)) are updated in place.  Returns the new parameters.
__device__ __forceinline__ Two updatePair(Two p, Two g, Two &m, Two &root, const Pairs &c) {
  m = addRounded(m * c.beta1, g * c.one_minus_beta1, c.one);
  const float2 r = split(addRounded((root * root) * c.beta2, (g * g) * c.one_minus_beta2, c.one));
  root = two(__fsqrt_rn(r.x), __fsqrt_rn(r.y));
  float2 d = split(fma(root, c.root_scale, c.epsilon));
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(d.x));
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(d.y));
  return fma(m * two(d.x, d.y), c.minus_step, p * c.decay);
}

struct BlockScale {
  float scale, inverse;
};
// Scale of a block of 256 from the largest magnitude that each lane holds (a NaN, larger than any other by its bits,
// reaches its whole block).
__device__ __forceinline__ BlockScale blockScale(float lane_largest) {
  const float most = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(lane_largest)));
  BlockScale s{0.0f, 0.0f};
  if (!(most < kSmallest)) {
    s.inverse = __fmul_rn(__frcp_rn(most), kCodeMax);
    s.scale = __fmul_rn(most, 1.0f / kCodeMax);
  }
  return s;
}
__device__ __forceinline__ Two rootCodes(Two root, float inverse) {
  const float2 r = split(root);
  float2 code = split(root * two(inverse, inverse));
  const float least = inverse > 0.0f ? kCodeTiny : 0.0f;
  code.x = r.x > 0.0f ? fmaxf(code.x, least) : code.x;
  code.y = r.y > 0.0f ? fmaxf(code.y, least) : code.y;
  return two(code.x, code.y);
}

// Random bits for an element of a step: products with shifts between them for each unit of 8 elements, the unit's bits
// times powers of one odd number for the elements inside it (the constants are bits of the golden ratio and of the roots of 2, 3
// and 5, made odd).  The upper half serves the first moment, the lower half the root.
__device__ __forceinline__ unsigned mixBits(unsigned h) {
  h ^= h >> 15;
  h *= 0x6A09E667u;
  h ^= h >> 13;
  h *= 0xBB67AE85u;
  return h ^ h >> 16;
}
constexpr unsigned kGolden = 0x9E3779BDu, kSpread = 0x3C6EF373u;
__device__ __forceinline__ unsigned stepBits(int64_t step) {
  const uint64_t s = (uint64_t)step;
  return mixBits(mixBits((unsigned)s * kGolden) + (unsigned)(s >> 32) * kSpread);
}
__device__ __forceinline__ unsigned unitBits(unsigned step_bits, int64_t element) {
  const uint64_t unit = (uint64_t)element >> 3;
  return mixBits((unsigned)unit * kSpread ^ (step_bits + (unsigned)(unit >> 32) * kGolden));
}
// kGolden to the power of k + 1, k < 8
__host__ __device__ constexpr unsigned elementFactor(int k) { return k == 0 ? kGolden : kGolden * elementFactor(k - 1); }
__device__ __forceinline__ unsigned elementFactorOf(int k) {
  unsigned f = kGolden;
#pragma unroll
  for (int i = 1; i < 8; ++i) f = i <= k ? f * kGolden : f;
  return f;
}

// x, in units of the scale, to one of the two e4m3 values next to it, up with the probability of its distance from the
// lower one.  Above 2^-6 a code is the upper 3 bits of the fraction, so that random bits below them carry with just that
// probability; below, the codes are 2^-9 apart, as they are behind 2^-6, to which the value is moved and back.  The largest
// of a block may be a rounding above 448 and is cut off there by the conversion.  What is not finite may come out as any code: its
// block's scale is infinite or NaN, and so is every product with it.
__device__ __forceinline__ float dither(float x, unsigned random16) {
  const float a = fabsf(x), base = a < 0.015625f ? 0.015625f : 0.0f;
  const unsigned bits = __float_as_uint(a + base) + (random16 << 4) + 8u;
  return copysignf(__uint_as_float(bits & 0xfff00000u) - base, x);
}
__device__ __forceinline__ Two dither(Two x, unsigned r0, unsigned r1) {
  const float2 f = split(x);
  return two(dither(f.x, r0), dither(f.y, r1));
}

template <typename P, typename G, bool STOCHASTIC, typename Table>
__global__ void __launch_bounds__(kThreads, STOCHASTIC ? 4 : 5) adamW8BitKernel(const __grid_constant__ Table t) {
  const int which = findTensor(t, blockIdx.x);
  const int64_t begin = (int64_t)((int)blockIdx.x - t.first_chunk[which]) * kChunk8Bit;
  const int64_t left = t.n[which] - begin;
  const int count = left < kChunk8Bit ? (int)left : kChunk8Bit;
  P *param = static_cast<P *>(t.param[which]) + begin;
  const G *grad = static_cast<const G *>(t.grad[which]) + begin;
  unsigned char *exp_avg = static_cast<unsigned char *>(t.exp_avg[which]) + begin;
  unsigned char *exp_avg_sq = static_cast<unsigned char *>(t.exp_avg_sq[which]) + begin;
  float *m_scales = t.exp_avg_scale[which] + begin / kScaleBlock;
  float *v_scales = t.exp_avg_sq_scale[which] + begin / kScaleBlock;
  const Pairs c(stepConstants(t));
  const float gs = t.grad_scale ? *t.grad_scale : 1.0f;
  const Two scale_grad = two(gs, gs);
  const unsigned step_bits = STOCHASTIC ? stepBits(t.step_count ? *t.step_count : t.step) : 0u;
  const bool vectors = aligned16(param) && aligned16(grad) && aligned16(exp_avg) && aligned16(exp_avg_sq);
  constexpr int kWarps = kThreads / 32;
  static_assert(kChunk8Bit == kWarps * kScaleBlock, "one block a warp");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (count == kChunk8Bit && vectors) {
    const int block = warp, at = block * (int)kScaleBlock + lane * 8;
    Eight<P> p;
    Eight<G> g;
    p.load(param + at);
    g.load(grad + at);
    const uint2 mc = *reinterpret_cast<const uint2 *>(exp_avg + at), vc = *reinterpret_cast<const uint2 *>(exp_avg_sq + at);
    const float ms = m_scales[block], vs = v_scales[block];
    Two m[4], root[4], next[4];
    float m_max = 0.0f, v_max = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const unsigned mw = j < 2 ? mc.x : mc.y, vw = j < 2 ? vc.x : vc.y;
      m[j] = fromCodes((unsigned short)(mw >> (j & 1) * 16)) * two(ms, ms);
      root[j] = fromCodes((unsigned short)(vw >> (j & 1) * 16)) * two(vs, vs);
      next[j] = updatePair(p.pair(j), g.pair(j) * scale_grad, m[j], root[j], c);
      const float2 a = split(m[j]), b = split(root[j]);
      m_max = largest(largest(m_max, a.x), a.y);
      v_max = largest(largest(v_max, b.x), b.y);
    }
    Eight<P>::store(param + at, next);
    const BlockScale m_scale = blockScale(m_max), v_scale = blockScale(v_max);
    unsigned short mo[4], vo[4];
    const unsigned unit = STOCHASTIC ? unitBits(step_bits, begin + at) : 0u;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      Two mx = m[j] * two(m_scale.inverse, m_scale.inverse), vx = rootCodes(root[j], v_scale.inverse);
      if (STOCHASTIC) {
        const unsigned r0 = unit * elementFactor(2 * j), r1 = unit * elementFactor(2 * j + 1);
        mx = dither(mx, r0 >> 16, r1 >> 16);
        vx = dither(vx, r0 & 0xffffu, r1 & 0xffffu);
      }
      mo[j] = toCodes(mx);
      vo[j] = toCodes(vx);
    }
    *reinterpret_cast<uint2 *>(exp_avg + at) = make_uint2(mo[0] | (unsigned)mo[1] << 16, mo[2] | (unsigned)mo[3] << 16);
    *reinterpret_cast<uint2 *>(exp_avg_sq + at) = make_uint2(vo[0] | (unsigned)vo[1] << 16, vo[2] | (unsigned)vo[3] << 16);
    if (lane == 0) {
      m_scales[block] = m_scale.scale;
      v_scales[block] = v_scale.scale;
    }
    return;
  }
  // A tensor's last chunk, or pointers that are not 16-byte aligned: element by element, lanes side by side.  A pair is
  // elements 32 apart.
  const int blocks = (count + (int)kScaleBlock - 1) / (int)kScaleBlock;
  for (int block = warp; block < blocks; block += kWarps) {
    const float ms = m_scales[block], vs = v_scales[block];
    Two m[4], root[4];
    float m_max = 0.0f, v_max = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int at0 = block * (int)kScaleBlock + 2 * j * 32 + lane, at1 = at0 + 32;
      const bool in0 = at0 < count, in1 = at1 < count;
      unsigned short mc = 0, vc = 0;
      float p0 = 0.0f, p1 = 0.0f, g0 = 0.0f, g1 = 0.0f;
      if (in0) {
        mc = exp_avg[at0];
        vc = exp_avg_sq[at0];
        p0 = toFloat(param[at0]);
        g0 = toFloat(grad[at0]);
      }
      if (in1) {
        mc |= (unsigned short)(exp_avg[at1] << 8);
        vc |= (unsigned short)(exp_avg_sq[at1] << 8);
        p1 = toFloat(param[at1]);
        g1 = toFloat(grad[at1]);
      }
      m[j] = fromCodes(mc) * two(ms, ms);
      root[j] = fromCodes(vc) * two(vs, vs);
      const float2 next = split(updatePair(two(p0, p1), two(g0, g1) * scale_grad, m[j], root[j], c));
      float2 a = split(m[j]), b = split(root[j]);
      if (in0) param[at0] = fromFloat<P>(next.x);
      else a.x = b.x = 0.0f;
      if (in1) param[at1] = fromFloat<P>(next.y);
      else a.y = b.y = 0.0f;
      m_max = largest(largest(m_max, a.x), a.y);
      v_max = largest(largest(v_max, b.x), b.y);
    }
    const BlockScale m_scale = blockScale(m_max), v_scale = blockScale(v_max);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int at0 = block * (int)kScaleBlock + 2 * j * 32 + lane, at1 = at0 + 32;
      Two mx = m[j] * two(m_scale.inverse, m_scale.inverse), vx = rootCodes(root[j], v_scale.inverse);
      if (STOCHASTIC) {
        const unsigned factor = elementFactorOf(at0 & 7);  // (at1 is 32 elements on)
        const unsigned r0 = unitBits(step_bits, begin + at0) * factor, r1 = unitBits(step_bits, begin + at1) * factor;
        mx = dither(mx, r0 >> 16, r1 >> 16);
        vx = dither(vx, r0 & 0xffffu, r1 & 0xffffu);
      }
      const unsigned short mc = toCodes(mx), vc = toCodes(vx);
      if (at0 < count) {
        exp_avg[at0] = (unsigned char)mc;
        exp_avg_sq[at0] = (unsigned char)vc;
      }
      if (at1 < count) {
        exp_avg[at1] = (unsigned char)(mc >> 8);
        exp_avg_sq[at1] = (unsigned char)(vc >> 8);
      }
    }
    if (lane == 0) {
      m_scales[block] = m_scale.scale;
      v_scales[block] = v_scale.scale;
    }
  }
}

template <typename P, typename G, typename Table>
cudaError_t launchTable(const AdamWProblem &p, const Table &t, int chunk, int chunks, double bytes, cudaStream_t stream) {
  trace::Scope scope(p.state_8bit ? "adamW8BitKernel" : "adamWKernel", stream, bytes);
  auto kernel = p.state_8bit && p.stochastic ? adamW8BitKernel<P, G, true, Table>
                : p.state_8bit               ? adamW8BitKernel<P, G, false, Table>
                : chunk == kChunk            ? adamWKernel<P, G, kChunk, Table>
                                             : adamWKernel<P, G, kSmallChunk, Table>;
  kernel<<<chunks, kThreads, 0, stream>>>(t);
  return cudaGetLastError();
}

template <typename Table>
cudaError_t dispatch(const AdamWProblem &p, const Table &t, int chunk, int chunks, double bytes, cudaStream_t stream) {
  const bool float_grad = p.grad_dtype == MLUOP_DTYPE_FLOAT;
  switch (p.param_dtype) {
    case MLUOP_DTYPE_FLOAT: return launchTable<float, float>(p, t, chunk, chunks, bytes, stream);
    case MLUOP_DTYPE_HALF:
      return float_grad ? launchTable<__half, float>(p, t, chunk, chunks, bytes, stream)
                        : launchTable<__half, __half>(p, t, chunk, chunks, bytes, stream);
    default:
      return float_grad ? launchTable<__nv_bfloat16, float>(p, t, chunk, chunks, bytes, stream)
                        : launchTable<__nv_bfloat16, __nv_bfloat16>(p, t, chunk, chunks, bytes, stream);
  }
}

template <typename Table>
cudaError_t launchAll(const AdamWProblem &p, cudaStream_t stream) {
  Table t;
  t.grad_scale = p.grad_scale;
  t.schedule = p.schedule;
  t.weight_decay = p.weight_decay;
  t.step = p.step;
  t.step_count = p.step_count;
  t.c.beta1 = (float)p.beta1;
  t.c.one_minus_beta1 = (float)(1.0 - p.beta1);
  t.c.beta2 = (float)p.beta2;
  t.c.one_minus_beta2 = (float)(1.0 - p.beta2);
  t.c.epsilon = (float)p.epsilon;
  // The 8-bit step's reciprocal takes denormals for zero: an element without a gradient would become 0 * infinity.  A root
  // that is not zero is above 2^-75, so that nothing else can tell.
  if (p.state_8bit && p.epsilon > 0.0) t.c.epsilon = std::max(t.c.epsilon, FLT_MIN);
  t.c.one = 1.0f;
  t.c.decay = (float)(1.0 - p.lr * p.weight_decay);
  t.c.step_size = (float)(p.lr / (1.0 - std::pow(p.beta1, (double)p.step)));
  t.c.root_scale = (float)(1.0 / std::sqrt(1.0 - std::pow(p.beta2, (double)p.step)));
  const double element_bytes = 2.0 * mluop::getSizeOfDataType(p.param_dtype) +
                               (double)mluop::getSizeOfDataType(p.grad_dtype) + (p.state_8bit ? 4.0 : 16.0);
  // Float states, fewer chunks than four blocks an SM: smaller ones.  Measured on 24 tensors of 500,000 elements together:
  // 7.7 us against 14 us.
  int64_t all = 0;
  for (int64_t k = 0; k < p.tensor_num; ++k) all += (p.element_num[k] + kChunk - 1) / kChunk;
  const int chunk = p.state_8bit ? kChunk8Bit : all >= 4 * p.sm_count ? kChunk : kSmallChunk;
  int64_t i = 0;
  while (i < p.tensor_num) {
    int64_t chunks = 0, elements = 0;
    int k = 0;
    for (; i < p.tensor_num && k < Table::kMost; ++i) {
      const int64_t n = p.element_num[i];
      if (n == 0) continue;
      const int64_t more = (n + chunk - 1) / chunk;
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
    const cudaError_t err = dispatch(p, t, chunk, (int)chunks, element_bytes * elements, stream);
    if (err != cudaSuccess) return err;
  }
  return cudaSuccess;
}

}  // namespace

// A launch that carries 29 KB of arguments takes 4 us longer on the host than one that carries 2 KB.
cudaError_t launchMultiTensorAdamW(const AdamWProblem &p, cudaStream_t stream) {
  return p.tensor_num <= kFewTensors ? launchAll<TensorTable<kFewTensors>>(p, stream)
                                     : launchAll<TensorTable<kMaxTensors>>(p, stream);
}

}  // namespace multi_tensor_adamw
}  // namespace mluop
