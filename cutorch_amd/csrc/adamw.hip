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
// not zero is held as zero: the next step would divide by the root of its own gradient's share alone. So that code 1 stands for a number even
// where a block's largest v is tiny, a top that is not zero is 2^-116 at least; means below 2^-120 are held as zeros. What scales all of a block
// (the growth of the moments in the first steps) is in the float and is not rounded to codes.
#include <algorithm>
#include <cmath>
#include <functional>
#include <type_traits>
#include <vector>

#include "training.hpp"

namespace thc {
namespace {

constexpr int kStateBlock = 256;        // elements that share a scale: 4 a lane of one wave
constexpr float kSmallestMean = 0x1p-120f;     // below it a block of means is held as zeros: the reciprocal stays finite
constexpr float kSmallestSquare = 0x1p-116f;   // a block of squares has this for its top at least, unless all are zero: (1 / 255)^4 of it is 2^-148

struct Hyper {
  float beta1, oneMinusBeta1, beta2, oneMinusBeta2, rootScale, eps, keep, rate, gradScale;
};

// The square root of a share (0 to 1), from the reciprocal root r: with y = x r, y + (x - y y) r / 2 is the root's nearest float
// for every float from 2^-97 on (compared with sqrtf for each of them) and 0 for 0. It is off by one place at most from there down to 2^-126 and
// too small below, where the correction is not a normal number and r is held back: shares that small have code 0 or 1 either way. sqrtf looks
// after every range of its argument and takes 16 instructions, this 6, of which a step makes four: 8-bit steps are bound by arithmetic.
constexpr float kRootFrom = 0x1p-97f;
__device__ __forceinline__ float share_root(float x) {
  const float r = __builtin_amdgcn_rsqf(fmaxf(x, 0x1p-126f)), y = x * r;
  return __builtin_fmaf(__builtin_fmaf(-y, y, x), 0.5f * r, y);
}
// The nearest floats to the roots of second moments, which may be infinite, or so small that a step without eps divides by very little.
// A wave takes the short root where all it has are zeros or in that one's range, and sqrtf else. As bits a NaN and what is negative are above
// infinity, and zero less one above all. us of 8-bit steps of 4.5 M floats, 4.4 M halves and 184 M floats: 14.7, 14.5, 463 so, 16.4, 15.8, 493 with
// sqrtf alone. Steps with 32-bit states wait for memory and take sqrtf (202 M halves with float copies 956, 960 with this).
__device__ __forceinline__ void moment_roots(float (&root)[4], const float (&v)[4]) {
  uint32_t low = ~0u, high = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    low = min(low, __float_as_uint(v[e]) - 1);
    high = max(high, __float_as_uint(v[e]));
  }
  if (__ballot(low < __float_as_uint(kRootFrom) - 1 || high >= __float_as_uint(__builtin_inff())) == 0) {
#pragma unroll
    for (int e = 0; e < 4; ++e) root[e] = share_root(v[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) root[e] = sqrtf(v[e]);
  }
}

__device__ __forceinline__ void take_gradient(const Hyper& h, float g, float& m, float& v) {
  g = g * h.gradScale;
  m = m * h.beta1 + g * h.oneMinusBeta1;
  v = v * h.beta2 + (g * g) * h.oneMinusBeta2;
}
__device__ __forceinline__ float stepped(const Hyper& h, float p, float m, float root) {
  return p * h.keep - (m / (root * h.rootScale + h.eps)) * h.rate;
}

// The tensors of one launch travel as kernel arguments, so that no table has to reach the device first: the parameter, the gradient, the
// moments, with 8-bit states their scales, and the float copies if there are any. A launch costs the host more the more arguments
// it has (2.4 us for few, about 4 for 4 KiB), so there is a form for few tensors and one for as many as 4 KiB hold (147 tensors of a few
// thousand floats in two launches 11.0 us, in three of 64 15.2). Large ones take 56 a launch, where one
// load finds a workgroup's tensor as among any up to 64: of 202 M halves with float copies, 147 tensors, two sets in turn take 961 us, with up to 77 a launch 978
// (one set again and again 934 and 938; 291 small tensors, 24 M halves, 127 and 122).
enum { kParam, kGrad, kMean, kSquare, kMeanScale, kSquareScale };
template <int POINTERS, int N>
struct Args {
  static constexpr int kPointers = POINTERS, kItems = N;
  Hyper h;
  int32_t count;
  uint32_t firstPart[N];                // the workgroup that each tensor begins with
  struct {
    void* p[POINTERS];
    int64_t size;
  } item[N];
};
constexpr int kFewItems = 32, kLargeItems = 56;
template <int POINTERS>
constexpr int kManyItems = (4096 - 48) / (8 * POINTERS + 12);

// What this workgroup has: a tensor, found by every lane looking at one or two, and the place in it. All that the arguments say of it is
// asked for at once.
template <typename A>
struct Part {
  void* p[A::kPointers];
  int64_t base, left;
  __device__ __forceinline__ Part(const A& a, int part) {
    constexpr int J = (A::kItems + 63) / 64;
    const int lane = threadIdx.x & 63;
    uint32_t first[J];
#pragma unroll
    for (int j = 0; j < J; ++j) first[j] = a.firstPart[min(j * 64 + lane, A::kItems - 1)];
    int n = 0;
#pragma unroll
    for (int j = 0; j < J; ++j) n += __popcll(__ballot(j * 64 + lane < a.count && first[j] <= blockIdx.x));
    const int i = __builtin_amdgcn_readfirstlane(n - 1);
#pragma unroll
    for (int k = 0; k < A::kPointers; ++k) p[k] = a.item[i].p[k];
    base = (int64_t)(blockIdx.x - a.firstPart[i]) * part;
    left = a.item[i].size - base;
  }
};

// Packs of 4 elements of every operand that a lane has in flight, by kernel, and so the elements of a workgroup. us with 1, 2, 4: 4.4 M floats
// 25.5, 22.5, 27.0, 202 M halves with float copies 959, 953, 962; 8-bit states: 0.9 M halves 12.2, 14.9, 13.7, 184 M floats with the
// moments as floats 805, 829, 840.
constexpr int kStepPacks = 2, kStep8Packs = 1, kDecodePacks = 1;
constexpr int part_size(int packs) { return kBlock * 4 * packs; }

// Four neighbours as floats, and back; `n` of them are the tensor's.
template <bool NT, typename T>
__device__ __forceinline__ void load4(float (&to)[4], const T* from, int n) {
  using P = Pack<T, 4>;
  if (n >= 4) {
    const P p = load_pack_unaligned<NT, P>(from);
#pragma unroll
    for (int e = 0; e < 4; ++e) to[e] = Cvt<T>::up(p.v[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) to[e] = e < n ? Cvt<T>::up(from[e]) : 0.f;
  }
}
template <bool NT, typename T>
__device__ __forceinline__ void store4(T* to, const float (&from)[4], int n) {
  using P = Pack<T, 4>;
  if (n >= 4) {
    P p;
#pragma unroll
    for (int e = 0; e < 4; ++e) p.v[e] = rounded<T>(from[e]);
    store_pack_unaligned<NT>(to, p);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < n) to[e] = rounded<T>(from[e]);
  }
}

// States in 32 bits, in place. FULL: the tensor does not end in this part. Bound by memory: 202 M halves with float copies 955 us, 5.9 TB/s;
// a model of 27 tensors and 120 thousand floats 4.4 us, the launch and the host's work for it.
template <typename T, bool MASTER, bool NT, bool FULL>
__device__ __forceinline__ void step_part(const Hyper& h, void* const* pointers, int64_t base, int left) {
  constexpr int U = kStepPacks;
  T* param = static_cast<T*>(pointers[kParam]) + base;
  const T* grad = static_cast<const T*>(pointers[kGrad]) + base;
  float *mean = static_cast<float*>(pointers[kMean]) + base, *square = static_cast<float*>(pointers[kSquare]) + base;
  float* master = MASTER ? static_cast<float*>(pointers[kSquare + 1]) + base : nullptr;
  float p[U][4], g[U][4], m[U][4], v[U][4];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int i = (u * kBlock + threadIdx.x) * 4;
    if (FULL || i < left) {
      const int n = FULL ? 4 : left - i;
      if constexpr (MASTER) load4<true>(p[u], master + i, n);
      else load4<true>(p[u], param + i, n);
      load4<true>(g[u], grad + i, n);
      load4<true>(m[u], mean + i, n);
      load4<true>(v[u], square + i, n);
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int i = (u * kBlock + threadIdx.x) * 4;
    if (FULL || i < left) {
      const int n = FULL ? 4 : left - i;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        take_gradient(h, g[u][e], m[u][e], v[u][e]);
        p[u][e] = stepped(h, p[u][e], m[u][e], sqrtf(v[u][e]));
      }
      store4<NT>(mean + i, m[u], n);
      store4<NT>(square + i, v[u], n);
      if constexpr (MASTER) store4<NT>(master + i, p[u], n);
      store4<NT>(param + i, p[u], n);
    }
  }
}
template <typename T, bool MASTER, bool NT, typename A>
__global__ __launch_bounds__(kBlock) void step_kernel(A a) {
  constexpr int kPart = part_size(kStepPacks);
  const Part<A> t(a, kPart);
  if (t.left >= kPart) step_part<T, MASTER, NT, true>(a.h, t.p, t.base, kPart);
  else step_part<T, MASTER, NT, false>(a.h, t.p, t.base, (int)t.left);
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
// The largest of a wave's magnitudes as bits: NaN is above infinity, so it is not lost. Each row of 16 lanes by shifts, then the rows.
__device__ __forceinline__ float wave_top(uint32_t bits) {
  int v = (int)bits;
  auto step = [&](auto control, auto rows) {
    const int o = __builtin_amdgcn_update_dpp(v, v, decltype(control)::value, decltype(rows)::value, 0xf, false);
    v = (int)max((uint32_t)v, (uint32_t)o);
  };
  using std::integral_constant;
  step(integral_constant<int, 0x111>{}, integral_constant<int, 0xf>{});   // row_shr 1, 2, 4, 8
  step(integral_constant<int, 0x112>{}, integral_constant<int, 0xf>{});
  step(integral_constant<int, 0x114>{}, integral_constant<int, 0xf>{});
  step(integral_constant<int, 0x118>{}, integral_constant<int, 0xf>{});
  step(integral_constant<int, 0x142>{}, integral_constant<int, 0xa>{});   // lane 15 of a row to the next one
  step(integral_constant<int, 0x143>{}, integral_constant<int, 0xc>{});   // lane 31 to the last two rows
  return __uint_as_float((uint32_t)__builtin_amdgcn_readlane(v, 63));
}
// 1 / top; 0 where a block has nothing to code (zeros, or a top that is not finite, which makes NaN of all of it).
__device__ __forceinline__ float inverse_of(float top) { return top > 0.f ? 1.f / top : 0.f; }
template <typename T>
__device__ __forceinline__ void load4_codes(T (&to)[4], const T* from, int n) {
  using P = Pack<T, 4>;
  if (n >= 4) {
    const P p = load_pack_unaligned<true, P>(from);
#pragma unroll
    for (int e = 0; e < 4; ++e) to[e] = p.v[e];
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) to[e] = e < n ? from[e] : T(0);
  }
}
template <bool NT, typename T>
__device__ __forceinline__ void store4_codes(T* to, const T (&from)[4], int n) {
  using P = Pack<T, 4>;
  if (n >= 4) {
    P p;
#pragma unroll
    for (int e = 0; e < 4; ++e) p.v[e] = from[e];
    store_pack_unaligned<NT>(to, p);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < n) to[e] = from[e];
  }
}

// States in 8 bits: a wave has a block of states per pack, 4 elements a lane. What is behind a tensor's end counts as zeros. Bound by
// arithmetic and memory alike in large calls (184 M floats 501 us, 5.9 TB/s, halves alone 489, 3.8; about 530 instructions for a block of 256), by
// arithmetic in those that the caches hold (4.5 M floats 17.4 us, halves 18.4).
// FULL: the tensor does not end in this part.
template <typename T, bool MASTER, bool NT, bool FULL>
__device__ __forceinline__ void step8_part(const Hyper& h, void* const* pointers, int64_t base, int left) {
  constexpr int U = kStep8Packs;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  T* param = static_cast<T*>(pointers[kParam]) + base;
  const T* grad = static_cast<const T*>(pointers[kGrad]) + base;
  int8_t* mean = static_cast<int8_t*>(pointers[kMean]) + base;
  uint8_t* square = static_cast<uint8_t*>(pointers[kSquare]) + base;
  float* meanScale = static_cast<float*>(pointers[kMeanScale]) + base / kStateBlock;
  float* squareScale = static_cast<float*>(pointers[kSquareScale]) + base / kStateBlock;
  float* master = MASTER ? static_cast<float*>(pointers[kSquareScale + 1]) + base : nullptr;
  float p[U][4], g[U][4], topMean[U], topSquare[U];
  int8_t codeMean[U][4];
  uint8_t codeSquare[U][4];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int block = u * (kBlock / 64) + wave, i = block * kStateBlock + lane * 4;
    if (FULL || block * kStateBlock < left) {      // whole waves
      const int n = FULL ? 4 : left - i;           // none for the lanes behind the end
      topMean[u] = meanScale[block];
      topSquare[u] = squareScale[block];
      if constexpr (MASTER) load4<true>(p[u], master + i, n);
      else load4<true>(p[u], param + i, n);
      load4<true>(g[u], grad + i, n);
      load4_codes(codeMean[u], mean + i, n);
      load4_codes(codeSquare[u], square + i, n);
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int block = u * (kBlock / 64) + wave, i = block * kStateBlock + lane * 4;
    if (FULL || block * kStateBlock < left) {
      const int n = FULL ? 4 : left - i;
      float m[4], v[4], root[4];
      uint32_t maxMean = 0, maxSquare = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        m[e] = decode_mean(codeMean[u][e], topMean[u]);
        v[e] = decode_square(codeSquare[u][e], topSquare[u]);
        take_gradient(h, g[u][e], m[e], v[e]);
      }
      moment_roots(root, v);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        p[u][e] = stepped(h, p[u][e], m[e], root[e]);
        if (FULL || e < n) {          // (zeros behind the end may meet a factor that is not finite)
          maxMean = max(maxMean, __float_as_uint(fabsf(m[e])));
          maxSquare = max(maxSquare, __float_as_uint(v[e]));
        }
      }
      if constexpr (MASTER) store4<NT>(master + i, p[u], n);
      store4<NT>(param + i, p[u], n);
      float newMean = wave_top(maxMean), newSquare = wave_top(maxSquare);
      if (newMean < kSmallestMean) newMean = 0.f;
      if (newSquare > 0.f) newSquare = fmaxf(newSquare, kSmallestSquare);
      const float inverseMean = inverse_of(newMean), inverseSquare = inverse_of(newSquare);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float c = rintf(share_root(fabsf(m[e]) * inverseMean) * 127.f);
        codeMean[u][e] = (int8_t)(int)(m[e] < 0.f ? -c : c);
        // (an infinite top has no inverse, and its codes are 0; the share of a v that is not zero may be, below a large top)
        const float d = rintf(share_root(share_root(v[e] * inverseSquare)) * 255.f);
        codeSquare[u][e] = (uint8_t)(int)(v[e] > 0.f && inverseSquare > 0.f ? fmaxf(d, 1.f) : d);
      }
      store4_codes<NT>(mean + i, codeMean[u], n);
      store4_codes<NT>(square + i, codeSquare[u], n);
      if (lane == 0) {
        meanScale[block] = newMean;
        squareScale[block] = newSquare;
      }
    }
  }
}
template <typename T, bool MASTER, bool NT, typename A>
__global__ __launch_bounds__(kBlock) void step8_kernel(A a) {
  constexpr int kPart = part_size(kStep8Packs);
  const Part<A> t(a, kPart);
  if (t.left >= kPart) step8_part<T, MASTER, NT, true>(a.h, t.p, t.base, kPart);
  else step8_part<T, MASTER, NT, false>(a.h, t.p, t.base, (int)t.left);
}

// The moments that 8-bit states stand for: from codes and scales, the mean into kParam and the square into kGrad. Bound by its stores: of 184 M
// 318 us, 5.8 TB/s.
template <bool FULL>
__device__ __forceinline__ void decode_part(void* const* pointers, int64_t base, int left) {
  constexpr int U = kDecodePacks;
  const int8_t* mean = static_cast<const int8_t*>(pointers[kMean]) + base;
  const uint8_t* square = static_cast<const uint8_t*>(pointers[kSquare]) + base;
  const float* meanScale = static_cast<const float*>(pointers[kMeanScale]) + base / kStateBlock;
  const float* squareScale = static_cast<const float*>(pointers[kSquareScale]) + base / kStateBlock;
  float *meanOut = static_cast<float*>(pointers[kParam]) + base, *squareOut = static_cast<float*>(pointers[kGrad]) + base;
  int8_t codeMean[U][4];
  uint8_t codeSquare[U][4];
  float topMean[U], topSquare[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int i = (u * kBlock + threadIdx.x) * 4;
    if (FULL || i < left) {
      const int n = FULL ? 4 : left - i;
      topMean[u] = meanScale[i / kStateBlock];
      topSquare[u] = squareScale[i / kStateBlock];
      load4_codes(codeMean[u], mean + i, n);
      load4_codes(codeSquare[u], square + i, n);
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int i = (u * kBlock + threadIdx.x) * 4;
    if (FULL || i < left) {
      const int n = FULL ? 4 : left - i;
      float m[4], v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        m[e] = decode_mean(codeMean[u][e], topMean[u]);
        v[e] = decode_square(codeSquare[u][e], topSquare[u]);
      }
      store4<true>(meanOut + i, m, n);
      store4<true>(squareOut + i, v, n);
    }
  }
}
template <typename A>
__global__ __launch_bounds__(kBlock) void decode_kernel(A a) {
  constexpr int kPart = part_size(kDecodePacks);
  const Part<A> t(a, kPart);
  if (t.left >= kPart) decode_part<true>(t.p, t.base, kPart);
  else decode_part<false>(t.p, t.base, (int)t.left);
}

// ------------------------------------------------------------------------- host --
template <int POINTERS>
struct Operands {
  void* p[POINTERS];
  int64_t size;
};

// Collects tensors of elements of these sizes and launches a kernel (by launch(args, grid)) for as many as its arguments hold.
template <typename A, typename Launch>
struct Batch {
  A a{};
  int part;
  const int* elementSize;      // of each pointer; 0: a scale for each block
  uint32_t parts = 0;
  Launch launch;
  Batch(const Hyper& h, int partSize, const int* sizes, Launch l) : part(partSize), elementSize(sizes), launch(l) { a.h = h; }
  void add(void* const* pointers, int64_t size) {
    // (a launch has less than 2^32 threads: a larger tensor goes in pieces)
    const int64_t most = (int64_t)part << 22;
    for (int64_t at = 0; at < size; at += most) {
      const int64_t n = std::min(most, size - at), count = (n + part - 1) / part;
      if (a.count == A::kItems || parts + count > (int64_t)1 << 23) flush();
      a.firstPart[a.count] = parts;
      a.item[a.count].size = n;
      for (int k = 0; k < A::kPointers; ++k)
        a.item[a.count].p[k] = static_cast<char*>(pointers[k]) + (elementSize[k] ? at * elementSize[k] : at / kStateBlock * 4);
      ++a.count;
      parts += (uint32_t)count;
    }
  }
  void flush() {
    if (a.count) launch(a, dim3(parts));
    a.count = 0;
    parts = 0;
  }
};

struct Lists {
  AnyTensor **param, **master, **grad, **mean, **square, **meanScale, **squareScale;   // master: or null; scales: null with 32-bit states
};

int64_t state_blocks(int64_t n) { return (n + kStateBlock - 1) / kStateBlock; }

void check_scales(THCState* s, const AnyTensor* scale, int64_t n, int arg, int index, bool written) {
  THC_ARG_CHECK(scale, arg, "no scales of tensor %d's states", index + 1);
  check_same_gpu(s, 1, &scale);
  THC_ARG_CHECK(tensor_numel(scale) == state_blocks(n), arg, "%ld scales for the %ld blocks of tensor %d's states", (long)tensor_numel(scale),
                (long)state_blocks(n), index + 1);
  THC_ARG_CHECK(!written || tensor_is_contiguous(scale) || !overlapping(tensor_layout(scale)), arg, "scales of tensor %d's states overlap", index + 1);
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
    if (eight) check_scales(s, l.meanScale[i], tensor_numel(p), base + 2, i, true);
    check_list(s, l.square[i], p, base + (eight ? 3 : 2), i, true);
    if (eight) check_scales(s, l.squareScale[i], tensor_numel(p), base + 4, i, true);
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
  int64_t elements = 0;
  for (int i = 0; i < count; ++i) elements += tensor_numel(l.param[i]);
  // Streaming stores where the whole call's operands do not stay in the 256 MiB memory-side cache until the next step. us, plain and
  // streaming: 4.4 M floats (70 MB) 25.4, 26.6; 17.7 M halves with float copies 100, 95, with 8-bit states (177 MB) 112, 118; 161 M floats
  // with 8-bit states 891, 868.
  const int64_t touched = elements * (2 * (int64_t)dtype_size(dt) + (l.master ? 4 : 0) + (eight ? 2 : 8));
  const bool nt = tuning("adamw.nt", touched >= (int64_t(256) << 20)) != 0;
  hipStream_t st = current_stream(s);
  Held held(s);
  auto run = [&](auto type, auto withMaster, auto withEight, auto streaming, auto items) {
    using T = decltype(type);
    constexpr bool M = decltype(withMaster)::value, E = decltype(withEight)::value, NT = decltype(streaming)::value;
    constexpr int P = (E ? 6 : 4) + M;
    constexpr int N = decltype(items)::value;
    using A = Args<P, N ? N : kManyItems<P>>;
    static_assert(sizeof(A) <= 4096, "kernel arguments");
    auto launch = [&](const A& a, dim3 grid) {
      if constexpr (E) hipLaunchKernelGGL((step8_kernel<T, M, NT, A>), grid, dim3(kBlock), 0, st, a);
      else hipLaunchKernelGGL((step_kernel<T, M, NT, A>), grid, dim3(kBlock), 0, st, a);
    };
    constexpr int kSize = sizeof(T), kState = E ? 1 : 4;
    const int sizes[7] = {kSize, kSize, kState, kState, E ? 0 : 4, 0, 4};
    // every copy is made before the first launch: a step that fails has changed nothing
    std::vector<Operands<P>> all;
    all.reserve(count);
    for (int i = 0; i < count; ++i) {
      if (!has_elements(l.param[i])) continue;
      note_stream_use(s, {l.param[i], M ? l.master[i] : nullptr, l.grad[i], l.mean[i], l.square[i], E ? l.meanScale[i] : nullptr,
                          E ? l.squareScale[i] : nullptr});
      Operands<P> o;
      void** p = o.p;
      p[kParam] = held.add(l.param[i], dt, true);
      p[kGrad] = held.add(l.grad[i], dt, false);
      p[kMean] = held.add(l.mean[i], meanType, true);
      p[kSquare] = held.add(l.square[i], squareType, true);
      if constexpr (E) {
        p[kMeanScale] = held.add(l.meanScale[i], DType::F32, true);
        p[kSquareScale] = held.add(l.squareScale[i], DType::F32, true);
      }
      if constexpr (M) p[P - 1] = held.add(l.master[i], DType::F32, true);
      o.size = tensor_numel(l.param[i]);
      all.push_back(o);
    }
    Batch<A, decltype(launch)> batch(h, part_size(E ? kStep8Packs : kStepPacks), sizes, launch);
    for (const Operands<P>& o : all) batch.add(o.p, o.size);
    batch.flush();
  };
  using std::false_type;
  using std::true_type;
  auto typed = [&](auto type, auto master, auto bits) {
    using std::integral_constant;
    if (nt) run(type, master, bits, true_type{}, integral_constant<int, kLargeItems>{});
    else if (count <= kFewItems) run(type, master, bits, false_type{}, integral_constant<int, kFewItems>{});
    else run(type, master, bits, false_type{}, integral_constant<int, 0>{});      // as many as fit
  };
  auto states = [&](auto bits) {
    if (!half) typed(float{}, false_type{}, bits);
    else if (!l.master) typed(__half{}, false_type{}, bits);
    else typed(__half{}, true_type{}, bits);
  };
  if (eight) states(true_type{});
  else states(false_type{});
  THC_CHECK(hipGetLastError());
  note_kernel(eight ? "adamw8" : "adamw");
  held.write_back();
}

// All tensors are decoded side by side: an output on another tensor's scales or output would be written before or after those are read or
// written. Looked for among the dense operands, which are used where they are, in the order of their addresses.
void refuse_meeting(int count, AnyTensor** meanOut, AnyTensor** squareOut, AnyTensor** mean, AnyTensor** meanScale, AnyTensor** squareScale) {
  struct Span {
    const void* storage;
    int64_t first, last;      // elements
    int arg, index;           // arg: of an output, 0 for scales
  };
  std::vector<Span> spans;
  spans.reserve(4 * (size_t)count);
  for (int i = 0; i < count; ++i) {
    if (!has_elements(mean[i])) continue;
    const AnyTensor* t[4] = {meanOut[i], squareOut[i], meanScale[i], squareScale[i]};
    const int args[4] = {3, 4, 0, 0};
    for (int k = 0; k < 4; ++k)
      if (tensor_is_contiguous(t[k])) spans.push_back(Span{t[k]->storage, t[k]->storageOffset, t[k]->storageOffset + tensor_numel(t[k]), args[k], i});
  }
  std::sort(spans.begin(), spans.end(), [](const Span& a, const Span& b) {
    if (a.storage != b.storage) return std::less<const void*>()(a.storage, b.storage);
    return a.first < b.first;
  });
  // those before it that reach farthest: of the outputs, and of the scales
  const Span *out = nullptr, *scale = nullptr;
  for (const Span& x : spans) {
    for (const Span* y : {out, scale}) {
      if (!y || y->storage != x.storage || y->last <= x.first || (!x.arg && !y->arg)) continue;
      const Span &one = x.arg ? x : *y, &other = x.arg ? *y : x;
      THC_ARG_CHECK(false, one.arg, "tensor %d lies on tensor %d's %s", one.index + 1, other.index + 1, other.arg ? "moments" : "scales");
    }
    const Span*& farthest = x.arg ? out : scale;
    if (!farthest || farthest->storage != x.storage || farthest->last < x.last) farthest = &x;
  }
}

// Floats of 8-bit states.
void moments(THCState* s, int count, AnyTensor** meanOut, AnyTensor** squareOut, AnyTensor** mean, AnyTensor** meanScale, AnyTensor** square,
             AnyTensor** squareScale) {
  THC_ARG_CHECK(count >= 0, 2, "a negative number of tensors");
  THC_ARG_CHECK(count == 0 || (meanOut && squareOut && mean && meanScale && square && squareScale), 3, "a list of tensors is missing");
  for (int i = 0; i < count; ++i) {
    THC_ARG_CHECK(mean[i], 5, "tensor %d is missing", i + 1);
    check_list(s, square[i], mean[i], 7, i, false);
    check_scales(s, meanScale[i], tensor_numel(mean[i]), 6, i, false);
    check_scales(s, squareScale[i], tensor_numel(mean[i]), 8, i, false);
    THC_ARG_CHECK(meanOut[i], 3, "tensor %d is missing", i + 1);
    THC_ARG_CHECK(squareOut[i], 4, "tensor %d is missing", i + 1);
  }
  hipStream_t st = current_stream(s);
  using A = Args<6, kManyItems<6>>;
  auto launch = [&](const A& a, dim3 grid) { hipLaunchKernelGGL((decode_kernel<A>), grid, dim3(kBlock), 0, st, a); };
  const int sizes[6] = {4, 4, 1, 1, 0, 0};
  Batch<A, decltype(launch)> batch(Hyper{}, part_size(kDecodePacks), sizes, launch);
  Held held(s);
  // Dense operands are used where they are; those with gaps are read and written by copies around the launches, and may lie in each other's.
  auto dense_meet = [](const AnyTensor* a, const AnyTensor* b) {
    return spans_meet(a, DType::F32, b, DType::F32) && tensor_is_contiguous(a) && tensor_is_contiguous(b);
  };
  // (all are resized before any pointer is taken: they may share a storage)
  for (int i = 0; i < count; ++i) {
    tensor_resize_as(s, meanOut[i], mean[i], DType::F32);
    tensor_resize_as(s, squareOut[i], mean[i], DType::F32);
  }
  for (int i = 0; i < count; ++i) {
    if (!has_elements(mean[i])) continue;
    const AnyTensor *out[2] = {meanOut[i], squareOut[i]}, *in[2] = {meanScale[i], squareScale[i]};
    for (int j = 0; j < 2; ++j) {
      THC_ARG_CHECK(tensor_is_contiguous(out[j]) || !overlapping(tensor_layout(out[j])), 3 + j, "elements of tensor %d overlap", i + 1);
      for (int k = 0; k < 2; ++k) THC_ARG_CHECK(!dense_meet(out[j], in[k]), 3 + j, "tensor %d lies on its scales", i + 1);
    }
    THC_ARG_CHECK(!dense_meet(out[0], out[1]), 4, "tensor %d's two moments share memory", i + 1);
  }
  refuse_meeting(count, meanOut, squareOut, mean, meanScale, squareScale);
  // every copy is made before the first launch: outputs may lie in the gaps of scales that are read through one
  std::vector<Operands<6>> all;
  all.reserve(count);
  for (int i = 0; i < count; ++i) {
    if (!has_elements(mean[i])) continue;
    note_stream_use(s, {meanOut[i], squareOut[i], mean[i], meanScale[i], square[i], squareScale[i]});
    Operands<6> o;
    o.p[kParam] = held.add(meanOut[i], DType::F32, true);
    o.p[kGrad] = held.add(squareOut[i], DType::F32, true);
    o.p[kMean] = held.add(mean[i], DType::I8, false);
    o.p[kSquare] = held.add(square[i], DType::U8, false);
    o.p[kMeanScale] = held.add(meanScale[i], DType::F32, false);
    o.p[kSquareScale] = held.add(squareScale[i], DType::F32, false);
    o.size = tensor_numel(mean[i]);
    all.push_back(o);
  }
  for (const Operands<6>& o : all) batch.add(o.p, o.size);
  batch.flush();
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
