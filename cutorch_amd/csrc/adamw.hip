// One AdamW step of many tensors.
//
//   g = f grad;  m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g g
//   p = p (1 - lr wd) - (m / (sqrt(v) / sqrt(1 - b2^t) + eps)) lr / (1 - b1^t)
//
// in float, one rounding an operation, in this order; half parameters are rounded once at the end, from their float copy where the
// caller keeps one. 8-bit states hold the moments as codes and one float per 256 consecutive elements, the largest magnitude there:
//
//   m = top (c / 127) |c / 127|     c = sign(m) round(127 sqrt(|m| / top))
//   v = top (c / 255)^4             c = round(255 (v / top)^(1/4)), at least 1 where v > 0
//
// A code step is 1.6 % of the value near the top and a value of a hundredth of it still has a tenth of the codes. No v that is
// not zero is held as zero: the next step would divide by the root of its own gradient's share alone. What scales all of a block
// (the growth of the moments in the first steps) is in the float and is not rounded to codes.
#include <algorithm>
#include <cmath>
#include <vector>

#include "training.hpp"

namespace thc {
namespace {

constexpr int kStateBlock = 256;        // elements that share a scale: 4 a lane of one wave
constexpr float kSmallestTop = 0x1p-120f;   // below it a block of states is held as zeros: the reciprocal stays finite

struct Hyper {
  float beta1, oneMinusBeta1, beta2, oneMinusBeta2, rootScale, eps, keep, rate, gradScale;
};

__device__ __forceinline__ float adamw_step(const Hyper& h, float p, float g, float& m, float& v) {
  g = g * h.gradScale;
  m = m * h.beta1 + g * h.oneMinusBeta1;
  v = v * h.beta2 + (g * g) * h.oneMinusBeta2;
  const float root = sqrtf(v) * h.rootScale + h.eps;
  return p * h.keep - (m / root) * h.rate;
}

// The tensors of one launch, as kernel arguments.
struct Item {
  void* param;
  float* master;
  const void* grad;
  void *mean, *square;
  float *meanScale, *squareScale;
  int64_t size;
};

template <typename T>
__global__ __launch_bounds__(kBlock) void step_kernel(Item t, Hyper h) {
  constexpr int V = 4;
  const int64_t i0 = ((int64_t)blockIdx.x * kBlock + threadIdx.x) * V;
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const int64_t i = i0 + e;
    if (i >= t.size) return;
    T* param = static_cast<T*>(t.param);
    float *mean = static_cast<float*>(t.mean), *square = static_cast<float*>(t.square);
    float m = mean[i], v = square[i];
    const float p = adamw_step(h, t.master ? t.master[i] : Cvt<T>::up(param[i]), Cvt<T>::up(static_cast<const T*>(t.grad)[i]), m, v);
    mean[i] = m;
    square[i] = v;
    if (t.master) t.master[i] = p;
    param[i] = rounded<T>(p);
  }
}

__device__ __forceinline__ float decode_mean(int8_t c, float top) {
  const float t = (float)c * (1.f / 127);
  return (t * fabsf(t)) * top;
}
__device__ __forceinline__ float decode_square(uint8_t c, float top) {
  float t = (float)c * (1.f / 255);
  t = t * t;
  return (t * t) * top;
}
// The largest of a wave's magnitudes as bits: NaN is above infinity, so it is not lost.
__device__ __forceinline__ float wave_top(uint32_t bits) {
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) bits = max(bits, (uint32_t)__shfl_xor((int)bits, d));
  return __uint_as_float(bits);
}
__device__ __forceinline__ float inverse_top(float& top) {
  if (top < kSmallestTop) top = 0.f;
  return top > 0.f ? 1.f / top : 0.f;
}

// A wave a block of states.
template <typename T>
__global__ __launch_bounds__(kBlock) void step8_kernel(Item t, Hyper h) {
  constexpr int V = 4;
  const int lane = threadIdx.x & 63;
  const int64_t block = (int64_t)blockIdx.x * (kBlock / 64) + (threadIdx.x >> 6);
  if (block * kStateBlock >= t.size) return;      // whole waves
  T* param = static_cast<T*>(t.param);
  int8_t* mean = static_cast<int8_t*>(t.mean);
  uint8_t* square = static_cast<uint8_t*>(t.square);
  const float oldMean = t.meanScale[block], oldSquare = t.squareScale[block];
  float m[V], v[V];
  uint32_t topMean = 0, topSquare = 0;
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const int64_t i = block * kStateBlock + lane * V + e;
    m[e] = v[e] = 0.f;
    if (i < t.size) {
      m[e] = decode_mean(mean[i], oldMean);
      v[e] = decode_square(square[i], oldSquare);
      const float p = adamw_step(h, t.master ? t.master[i] : Cvt<T>::up(param[i]), Cvt<T>::up(static_cast<const T*>(t.grad)[i]), m[e], v[e]);
      if (t.master) t.master[i] = p;
      param[i] = rounded<T>(p);
      topMean = max(topMean, __float_as_uint(fabsf(m[e])));
      topSquare = max(topSquare, __float_as_uint(v[e]));
    }
  }
  float newMean = wave_top(topMean), newSquare = wave_top(topSquare);
  const float inverseMean = inverse_top(newMean), inverseSquare = inverse_top(newSquare);
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const int64_t i = block * kStateBlock + lane * V + e;
    if (i < t.size) {
      const float c = rintf(sqrtf(fabsf(m[e]) * inverseMean) * 127.f);
      mean[i] = (int8_t)(int)(m[e] < 0.f ? -c : c);
      const float share = v[e] * inverseSquare;
      const float d = rintf(sqrtf(sqrtf(share)) * 255.f);
      square[i] = (uint8_t)(int)(share > 0.f ? fmaxf(d, 1.f) : d);
    }
  }
  if (lane == 0) {
    t.meanScale[block] = newMean;
    t.squareScale[block] = newSquare;
  }
}

// The moments that 8-bit states stand for.
__global__ __launch_bounds__(kBlock) void decode_kernel(const int8_t* mean, const float* meanScale, const uint8_t* square, const float* squareScale,
                                                        float* meanOut, float* squareOut, int64_t n) {
  const int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x;
  if (i >= n) return;
  meanOut[i] = decode_mean(mean[i], meanScale[i / kStateBlock]);
  squareOut[i] = decode_square(square[i], squareScale[i / kStateBlock]);
}

// ------------------------------------------------------------------------- host --
// Operands that are written where they are if they are dense, else through a copy.
struct Held {
  THCState* s;
  struct One {
    AnyTensor* tensor;     // the caller's
    AnyTensor* dense;
    DType dt;
    bool written;
  };
  std::vector<One> all;
  explicit Held(THCState* s_) : s(s_) {}
  Held(const Held&) = delete;
  Held& operator=(const Held&) = delete;
  ~Held() {
    for (One& o : all) tensor_free(s, o.dense);
  }
  void* add(AnyTensor* t, DType dt, bool written) {
    all.reserve(all.size() + 1);
    AnyTensor* dense = tensor_new_contiguous(s, t, dt);
    all.push_back(One{t, dense, dt, written});
    return tensor_data(dense, dt);
  }
  void write_back() {
    for (One& o : all)
      if (o.written && o.dense != o.tensor) copy_tensor(s, o.dt, o.tensor, o.dense, false);
  }
};

struct Lists {
  AnyTensor **param, **master, **grad, **mean, **square, **meanScale, **squareScale;   // master: or null; scales: null with 32-bit states
};

int64_t state_blocks(int64_t n) { return (n + kStateBlock - 1) / kStateBlock; }

void check_scales(const AnyTensor* scale, int64_t n, int arg, int index) {
  THC_ARG_CHECK(scale, arg, "no scales of tensor %d's states", index + 1);
  THC_ARG_CHECK(tensor_numel(scale) == state_blocks(n), arg, "%ld scales for the %ld blocks of tensor %d's states", (long)tensor_numel(scale),
                (long)state_blocks(n), index + 1);
}

void check_list(THCState* s, const AnyTensor* t, const AnyTensor* like, int arg, int index, bool written) {
  THC_ARG_CHECK(t, arg, "tensor %d is missing", index + 1);
  check_same_gpu(s, 1, &t);
  THC_ARG_CHECK(t->nDimension <= kMaxDims, arg, "%s", kDimWarning);
  THC_ARG_CHECK(same_sizes(t, like), arg, "tensor %d has other sizes than its parameter", index + 1);
  THC_ARG_CHECK(!written || !overlapping(tensor_layout(t)), arg, "elements of tensor %d overlap", index + 1);
}

void adamw(THCState* s, DType dt, int count, const Lists& l, double lr, double beta1, double beta2, double eps, double weightDecay, long step,
           double gradScale) {
  const bool eight = l.meanScale != nullptr, half = dt == DType::F16;
  const int base = half ? 5 : 4;     // argument numbers: state, count, param, [master], grad, ...
  THC_ARG_CHECK(count >= 0, 2, "a negative number of tensors");
  THC_ARG_CHECK(count == 0 || (l.param && l.grad && l.mean && l.square && (!eight || l.squareScale)), 3, "a list of tensors is missing");
  const int hyperArg = base + (eight ? 5 : 3);
  THC_ARG_CHECK(beta1 >= 0 && beta1 < 1, hyperArg + 1, "beta1 is not in [0, 1)");
  THC_ARG_CHECK(beta2 >= 0 && beta2 < 1, hyperArg + 2, "beta2 is not in [0, 1)");
  THC_ARG_CHECK(eps >= 0, hyperArg + 3, "eps is negative");
  THC_ARG_CHECK(step >= 1, hyperArg + 5, "steps are counted from 1");
  const DType meanType = eight ? DType::I8 : DType::F32, squareType = eight ? DType::U8 : DType::F32;
  for (int i = 0; i < count; ++i) {
    const AnyTensor* p = l.param[i];
    THC_ARG_CHECK(p, 3, "tensor %d is missing", i + 1);
    check_list(s, p, p, 3, i, true);
    if (l.master) check_list(s, l.master[i], p, 4, i, true);
    check_list(s, l.grad[i], p, base, i, false);
    check_list(s, l.mean[i], p, base + 1, i, true);
    if (eight) check_scales(l.meanScale[i], tensor_numel(p), base + 2, i);
    check_list(s, l.square[i], p, base + (eight ? 3 : 2), i, true);
    if (eight) check_scales(l.squareScale[i], tensor_numel(p), base + 4, i);
  }
  Hyper h;
  h.beta1 = (float)beta1;
  h.oneMinusBeta1 = (float)(1 - beta1);
  h.beta2 = (float)beta2;
  h.oneMinusBeta2 = (float)(1 - beta2);
  h.rootScale = (float)(1 / std::sqrt(1 - std::pow(beta2, (double)step)));
  h.eps = (float)eps;
  h.keep = (float)(1 - lr * weightDecay);
  h.rate = (float)(lr / (1 - std::pow(beta1, (double)step)));
  h.gradScale = (float)gradScale;
  hipStream_t st = current_stream(s);
  Held held(s);
  for (int i = 0; i < count; ++i) {
    if (!has_elements(l.param[i])) continue;
    note_stream_use(s, {l.param[i], l.master ? l.master[i] : nullptr, l.grad[i], l.mean[i], l.square[i], eight ? l.meanScale[i] : nullptr,
                        eight ? l.squareScale[i] : nullptr});
    Item t{};
    t.size = tensor_numel(l.param[i]);
    t.param = held.add(l.param[i], dt, true);
    if (l.master) t.master = (float*)held.add(l.master[i], DType::F32, true);
    t.grad = held.add(l.grad[i], dt, false);
    t.mean = held.add(l.mean[i], meanType, true);
    t.square = held.add(l.square[i], squareType, true);
    if (eight) {
      t.meanScale = (float*)held.add(l.meanScale[i], DType::F32, true);
      t.squareScale = (float*)held.add(l.squareScale[i], DType::F32, true);
    }
    const dim3 grid((unsigned)((t.size + 4 * kBlock - 1) / (4 * kBlock)));
    if (eight) {
      if (half) hipLaunchKernelGGL((step8_kernel<__half>), grid, dim3(kBlock), 0, st, t, h);
      else hipLaunchKernelGGL((step8_kernel<float>), grid, dim3(kBlock), 0, st, t, h);
    } else {
      if (half) hipLaunchKernelGGL((step_kernel<__half>), grid, dim3(kBlock), 0, st, t, h);
      else hipLaunchKernelGGL((step_kernel<float>), grid, dim3(kBlock), 0, st, t, h);
    }
  }
  THC_CHECK(hipGetLastError());
  note_kernel(eight ? "adamw8" : "adamw");
  held.write_back();
}

// Floats of 8-bit states.
void moments(THCState* s, int count, AnyTensor** meanOut, AnyTensor** squareOut, AnyTensor** mean, AnyTensor** meanScale, AnyTensor** square,
             AnyTensor** squareScale) {
  THC_ARG_CHECK(count >= 0, 2, "a negative number of tensors");
  THC_ARG_CHECK(count == 0 || (meanOut && squareOut && mean && meanScale && square && squareScale), 3, "a list of tensors is missing");
  for (int i = 0; i < count; ++i) {
    THC_ARG_CHECK(mean[i], 5, "tensor %d is missing", i + 1);
    check_list(s, square[i], mean[i], 7, i, false);
    check_scales(meanScale[i], tensor_numel(mean[i]), 6, i);
    check_scales(squareScale[i], tensor_numel(mean[i]), 8, i);
    THC_ARG_CHECK(meanOut[i], 3, "tensor %d is missing", i + 1);
    THC_ARG_CHECK(squareOut[i], 4, "tensor %d is missing", i + 1);
  }
  hipStream_t st = current_stream(s);
  Held held(s);
  for (int i = 0; i < count; ++i) {
    const int64_t n = tensor_numel(mean[i]);
    tensor_resize_as(s, meanOut[i], mean[i], DType::F32);
    tensor_resize_as(s, squareOut[i], mean[i], DType::F32);
    if (n == 0) continue;
    note_stream_use(s, {meanOut[i], squareOut[i], mean[i], meanScale[i], square[i], squareScale[i]});
    float* to = (float*)held.add(meanOut[i], DType::F32, true);
    float* toSquare = (float*)held.add(squareOut[i], DType::F32, true);
    const int8_t* from = (const int8_t*)held.add(mean[i], DType::I8, false);
    const uint8_t* fromSquare = (const uint8_t*)held.add(square[i], DType::U8, false);
    const float* scale = (const float*)held.add(meanScale[i], DType::F32, false);
    const float* scaleSquare = (const float*)held.add(squareScale[i], DType::F32, false);
    hipLaunchKernelGGL(decode_kernel, dim3((unsigned)((n + kBlock - 1) / kBlock)), dim3(kBlock), 0, st, from, scale, fromSquare, scaleSquare, to,
                       toSquare, n);
  }
  THC_CHECK(hipGetLastError());
  note_kernel("adamw8-moments");
  held.write_back();
}

}  // namespace
}  // namespace thc

#define TL(x) reinterpret_cast<thc::AnyTensor**>(x)
THC_API void THCudaTensor_adamW(THCState* s, int count, THCudaTensor** param, THCudaTensor** grad, THCudaTensor** mean, THCudaTensor** square,
                                double lr, double beta1, double beta2, double eps, double weightDecay, long step, double gradScale) {
  THC_GUARD_ALL(thc::adamw(s, thc::DType::F32, count, {TL(param), nullptr, TL(grad), TL(mean), TL(square), nullptr, nullptr}, lr, beta1, beta2,
                           eps, weightDecay, step, gradScale))
}
THC_API void THCudaHalfTensor_adamW(THCState* s, int count, THCudaHalfTensor** param, THCudaTensor** master, THCudaHalfTensor** grad,
                                    THCudaTensor** mean, THCudaTensor** square, double lr, double beta1, double beta2, double eps,
                                    double weightDecay, long step, double gradScale) {
  THC_GUARD_ALL(thc::adamw(s, thc::DType::F16, count, {TL(param), TL(master), TL(grad), TL(mean), TL(square), nullptr, nullptr}, lr, beta1,
                           beta2, eps, weightDecay, step, gradScale))
}
THC_API void THCudaTensor_adamW8(THCState* s, int count, THCudaTensor** param, THCudaTensor** grad, THCudaCharTensor** mean,
                                 THCudaTensor** meanScale, THCudaByteTensor** square, THCudaTensor** squareScale, double lr, double beta1,
                                 double beta2, double eps, double weightDecay, long step, double gradScale) {
  THC_GUARD_ALL({
    THC_ARG_CHECK(count <= 0 || meanScale, 6, "a list of tensors is missing");
    static thc::AnyTensor* none[1];
    thc::adamw(s, thc::DType::F32, count, {TL(param), nullptr, TL(grad), TL(mean), TL(square), meanScale ? TL(meanScale) : none, TL(squareScale)}, lr,
               beta1, beta2, eps, weightDecay, step, gradScale);
  })
}
THC_API void THCudaHalfTensor_adamW8(THCState* s, int count, THCudaHalfTensor** param, THCudaTensor** master, THCudaHalfTensor** grad,
                                     THCudaCharTensor** mean, THCudaTensor** meanScale, THCudaByteTensor** square, THCudaTensor** squareScale,
                                     double lr, double beta1, double beta2, double eps, double weightDecay, long step, double gradScale) {
  THC_GUARD_ALL({
    THC_ARG_CHECK(count <= 0 || meanScale, 7, "a list of tensors is missing");
    static thc::AnyTensor* none[1];
    thc::adamw(s, thc::DType::F16, count, {TL(param), TL(master), TL(grad), TL(mean), TL(square), meanScale ? TL(meanScale) : none, TL(squareScale)},
               lr, beta1, beta2, eps, weightDecay, step, gradScale);
  })
}
THC_API void THCudaTensor_adamW8Moments(THCState* s, int count, THCudaTensor** mean, THCudaTensor** square, THCudaCharTensor** meanCode,
                                        THCudaTensor** meanScale, THCudaByteTensor** squareCode, THCudaTensor** squareScale) {
  THC_GUARD_ALL(thc::moments(s, count, TL(mean), TL(square), TL(meanCode), TL(meanScale), TL(squareCode), TL(squareScale)))
}
