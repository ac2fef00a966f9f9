// Rotary positions: each head's pairs of elements turned by their token's position.
//
//   (a, b) -> s (a cos t - b sin t, a sin t + b cos t)      t = position * frequency_j, backwards: -t
//
// Pairs lie side by side (interleaved) or half of the turned part apart; what lies behind the turned part stays as it is. The angle is a product in
// 64 bits, its distance to the nearest quarter of a turn goes on in float: far positions are as exact as near ones. (In 32 bits a position of
// 131072 would leave an angle 2^-7 off.) The turn itself is in float and rounds once to the type.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "training.hpp"

namespace thc {
namespace {

using std::integral_constant;

// cos and sin of a position's angle, by the series around the nearest quarter of a turn: at most pi / 4 away, where terms up to the 11th
// power leave (pi / 4)^13 / 13! = 7e-12 (sin) and up to the 10th (pi / 4)^12 / 12! = 1.2e-10 (cos), beside a float's rounding of 6e-8.
struct Turn {
  float c, s;
};
__device__ __forceinline__ Turn turn_of(double position, double frequency) {
  constexpr double kPerRadian = 0.15915494309189533577;
  const double turns = position * frequency * kPerRadian, part = turns - rint(turns), quarter = rint(part * 4.0);
  const float a = (float)(part - 0.25 * quarter) * 6.28318530717958647693f, q = a * a;
  const int k = (int)quarter;
  float s = -1.f / 39916800.f, c = -1.f / 3628800.f;
  s = __builtin_fmaf(s, q, 1.f / 362880.f);
  s = __builtin_fmaf(s, q, -1.f / 5040.f);
  s = __builtin_fmaf(s, q, 1.f / 120.f);
  s = __builtin_fmaf(s, q, -1.f / 6.f);
  s = __builtin_fmaf(s * q, a, a);
  c = __builtin_fmaf(c, q, 1.f / 40320.f);
  c = __builtin_fmaf(c, q, -1.f / 720.f);
  c = __builtin_fmaf(c, q, 1.f / 24.f);
  c = __builtin_fmaf(c, q, -0.5f);
  c = __builtin_fmaf(c, q, 1.f);
  const float sin = k & 1 ? c : s, cos = k & 1 ? s : c;
  return Turn{((k + 1) & 2) ? -cos : cos, (k & 2) ? -sin : sin};
}

template <typename T>
struct RotaryArgs {
  const T* x;
  T* y;
  const int64_t* positions;      // null: a token's place in its sequence
  const double* frequencies;
  RowOffsets xo, yo;             // of tokens
  int64_t xHead, yHead;          // between heads
  Divisor<uint32_t> slots, headLanes, sequence;
  uint32_t firstToken, items;
  int32_t heads, headStep, dim, turned, turnSlots;
  float scale, sinScale;         // sinScale: negative to turn back
};

// An item is a pack of V elements (and the pack of their partners, where those are half the turned part away) of every headStep-th head of a token,
// so that its angles serve several heads; the loads of two heads are in flight. The last pack of a part is moved back into it and repeats elements
// of the one before, which a call in place may not do: that takes packs that divide the part. Bound by memory.
template <typename T, int V, bool INTERLEAVED>
__global__ __launch_bounds__(kBlock) void rotary_kernel(RotaryArgs<T> a) {
  constexpr int U = 2, N = INTERLEAVED ? V / 2 : V, S = INTERLEAVED ? 1 : 2;
  using P = Pack<T, V>;
  const uint32_t i = blockIdx.x * kBlock + threadIdx.x;
  if (i >= a.items) return;
  uint32_t rest, slot, token, lane, sequence, place;
  a.slots.divmod(i, rest, slot);
  a.headLanes.divmod(rest, token, lane);
  token += a.firstToken;
  const T* x = a.x + a.xo.at(token);
  T* y = a.y + a.yo.at(token);
  if ((int32_t)slot >= a.turnSlots) {      // behind the turned part
    const int32_t first = a.turned + ((int32_t)slot - a.turnSlots) * V, at = min(first, a.dim - V);
    for (int32_t h = lane; h < a.heads; h += a.headStep) {
      if (at >= a.turned) {
        store_pack_unaligned<true>(y + h * a.yHead + at, load_pack_unaligned<true, P>(x + h * a.xHead + at));
      } else {
        for (int32_t e = a.turned; e < a.dim; ++e) y[h * a.yHead + e] = x[h * a.xHead + e];
      }
    }
    return;
  }
  const int32_t half = a.turned / 2, at = min((int32_t)slot * V, (INTERLEAVED ? a.turned : half) - V);
  P v[U][S];
  auto load = [&](int32_t h) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (h + u * a.headStep < a.heads) {
#pragma unroll
        for (int s = 0; s < S; ++s) v[u][s] = load_pack_unaligned<true, P>(x + (h + u * a.headStep) * a.xHead + at + s * half);
      }
    }
  };
  load(lane);
  a.sequence.divmod(token, sequence, place);
  const double position = (double)(a.positions ? a.positions[place] : (int64_t)place);
  float c[N], s[N];
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const Turn t = turn_of(position, a.frequencies[(INTERLEAVED ? at / 2 : at) + e]);
    c[e] = t.c * a.scale;
    s[e] = t.s * a.sinScale;
  }
  for (int32_t h = lane; h < a.heads; h += U * a.headStep) {
    if (h != (int32_t)lane) load(h);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (h + u * a.headStep < a.heads) {
        P o[S];
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const int e0 = INTERLEAVED ? 2 * e : e, e1 = INTERLEAVED ? 2 * e + 1 : e;
          const float p = Cvt<T>::up(v[u][0].v[e0]), q = Cvt<T>::up(v[u][S - 1].v[e1]);
          o[0].v[e0] = rounded<T>(__builtin_fmaf(p, c[e], -(q * s[e])));
          o[S - 1].v[e1] = rounded<T>(__builtin_fmaf(p, s[e], q * c[e]));
        }
        T* out = y + (h + u * a.headStep) * a.yHead + at;
#pragma unroll
        for (int k = 0; k < S; ++k) store_pack_unaligned<true>(out + k * half, o[k]);
      }
    }
  }
}

// Tokens of heads: the leading dims merge into two at most, a head has unit stride.
bool as_tokens(const AnyTensor* t, Rows* tokens, int64_t* headStride) {
  const int nd = t->nDimension;
  tokens->length = t->size[nd - 1];
  if (t->stride[nd - 1] != 1 && tokens->length > 1) return false;
  *headStride = t->stride[nd - 2];
  tokens->count = tokens->inner = 1;
  tokens->stride = tokens->outerStride = 0;
  if (nd == 2) return true;
  Layout l = make_layout(nd - 2, t->size, t->stride);
  tokens->count = l.numel();
  collapse(l);
  if (l.dims > 2) return false;
  tokens->inner = l.size[l.dims - 1];
  tokens->stride = l.stride[l.dims - 1];
  if (l.dims == 2) tokens->outerStride = l.stride[0];
  return true;
}

template <typename T>
void launch_rotary(THCState* s, RotaryArgs<T>& a, int64_t tokens, bool interleaved, bool inPlace) {
  constexpr int kPack = 16 / sizeof(T);
  hipStream_t st = current_stream(s);
  const int32_t part = interleaved ? a.turned : a.turned / 2;
  int V = kPack;
  while (V > part || (inPlace && part % V)) V /= 2;
  a.turnSlots = (part + V - 1) / V;
  const int32_t slots = a.turnSlots + (inPlace ? 0 : (a.dim - a.turned + V - 1) / V);
  // Heads side by side: at least what fills the chip, few enough that an item's angles serve four heads where there are many.
  const int64_t want = (int64_t)num_compute_units(s) * 2048;
  int64_t lanes = std::max<int64_t>(1, a.heads / 4);
  lanes = std::max(lanes, std::min<int64_t>(a.heads, want / std::max<int64_t>(1, tokens * slots)));
  a.headStep = (int32_t)lanes;
  a.slots.set((uint64_t)slots);
  a.headLanes.set((uint64_t)lanes);
  const int64_t each = slots * lanes, most = std::max<int64_t>(1, tuning("rotary.items", 1 << 30) / each);
  for (int64_t first = 0; first < tokens; first += most) {
    a.firstToken = (uint32_t)first;
    a.items = (uint32_t)(std::min(most, tokens - first) * each);
    const dim3 grid((a.items + kBlock - 1) / kBlock);
    auto go = [&](auto vec) {
      constexpr int VV = decltype(vec)::value;
      if constexpr (VV >= 2) {
        if (interleaved) {
          hipLaunchKernelGGL((rotary_kernel<T, VV, true>), grid, dim3(kBlock), 0, st, a);
          return;
        }
      }
      hipLaunchKernelGGL((rotary_kernel<T, VV, false>), grid, dim3(kBlock), 0, st, a);
    };
    if (V == 8) {
      if constexpr (kPack == 8) go(integral_constant<int, 8>{});
    } else if (V == 4) {
      go(integral_constant<int, 4>{});
    } else if (V == 2) {
      go(integral_constant<int, 2>{});
    } else {
      go(integral_constant<int, 1>{});
    }
  }
}

template <typename T>
void run_rotary(THCState* s, DType dt, AnyTensor* self, AnyTensor* input, AnyTensor* positions, AnyTensor* frequencies, int64_t sequence, float scale,
                bool interleaved, bool inverse) {
  Rows xt, yt;
  RotaryArgs<T> a{};
  TensorRef x(s, nullptr), y(s, nullptr);
  if (as_tokens(input, &xt, &a.xHead)) {
    tensor_retain(input);
    x.t = input;
  } else {
    refuse_capture(s, "a turn of heads that lie apart");
    x.t = tensor_new_contiguous(s, input, dt);
    as_tokens(x.t, &xt, &a.xHead);
  }
  if ((positions && !tensor_is_contiguous(positions)) || !tensor_is_contiguous(frequencies)) refuse_capture(s, "a turn by strided positions or frequencies");
  TensorRef at(s, positions ? tensor_new_contiguous(s, positions, DType::I64) : nullptr);
  Dense f(s, frequencies, DType::F64);
  bool direct = as_tokens(self, &yt, &a.yHead) && !overlapping(tensor_layout(self)), inPlace = false;
  if (direct && spans_meet(self, dt, x.t, dt)) {
    inPlace = self->storageOffset == x.t->storageOffset && xt.inner == yt.inner && xt.stride == yt.stride && xt.outerStride == yt.outerStride &&
              a.xHead == a.yHead;
    direct = inPlace;
  }
  direct = direct && !(at.t && spans_meet(self, dt, at.t, DType::I64)) && !spans_meet(self, dt, f.ref.t, DType::F64);
  if (direct) {
    tensor_retain(self);
    y.t = self;
  } else {
    refuse_capture(s, "a turn whose output lies apart or on what it reads");
    inPlace = false;
    y.t = tensor_new_with_size(s, self->nDimension, self->size, dt);
    as_tokens(y.t, &yt, &a.yHead);
  }
  a.x = static_cast<const T*>(tensor_data(x.t, dt));
  a.y = static_cast<T*>(tensor_data(y.t, dt));
  a.positions = at.t ? static_cast<const int64_t*>(tensor_data(at.t, DType::I64)) : nullptr;
  a.frequencies = f.data<double>();
  a.xo = offsets_of(xt);
  a.yo = offsets_of(yt);
  a.heads = (int32_t)input->size[input->nDimension - 2];
  a.dim = (int32_t)xt.length;
  a.turned = 2 * (int32_t)tensor_numel(frequencies);
  a.sequence.set((uint64_t)sequence);
  a.scale = scale;
  a.sinScale = inverse ? -scale : scale;
  launch_rotary<T>(s, a, xt.count, interleaved, inPlace);
  THC_CHECK(hipGetLastError());
  note_kernel("rotary");
  if (y.t != self) copy_tensor(s, dt, self, y.t, false);
}

void rotary(THCState* s, DType dt, AnyTensor* self, AnyTensor* input, AnyTensor* positions, AnyTensor* frequencies, double scale, int interleaved,
            int inverse) {
  const AnyTensor* all[4] = {self, input, positions, frequencies};
  check_same_gpu(s, 4, all);
  THC_ARG_CHECK(has_elements(frequencies), 5, "no frequencies");
  if (!has_elements(input)) {
    tensor_resize_as(s, self, input, dt);
    return;
  }
  const int nd = input->nDimension;
  THC_ARG_CHECK(nd >= 2, 3, "heads of tokens have two dims at least");
  THC_ARG_CHECK(nd <= kMaxDims, 3, "%s", kDimWarning);
  const int64_t dim = input->size[nd - 1], heads = input->size[nd - 2], tokens = tensor_numel(input) / dim / heads;
  THC_ARG_CHECK(dim < (int64_t(1) << 20) && heads < (int64_t(1) << 20) && dim * heads < (int64_t(1) << 28), 3, "heads are too long or too many");
  THC_ARG_CHECK(tokens < kIndex32Limit, 3, "too many tokens");
  THC_ARG_CHECK(tensor_numel(frequencies) <= dim / 2, 5, "%ld frequencies turn more than heads of %ld", (long)tensor_numel(frequencies), (long)dim);
  int64_t sequence = nd > 2 ? input->size[nd - 3] : 1;
  if (positions) {
    const int64_t n = tensor_numel(positions);
    THC_ARG_CHECK(n == tokens || n == sequence, 4, "%ld positions for %ld tokens in sequences of %ld", (long)n, (long)tokens, (long)sequence);
    sequence = n;
  }
  tensor_resize_as(s, self, input, dt);
  note_stream_use(s, {self, input, positions, frequencies});
  if (dt == DType::F32) run_rotary<float>(s, dt, self, input, positions, frequencies, sequence, (float)scale, interleaved != 0, inverse != 0);
  else run_rotary<__half>(s, dt, self, input, positions, frequencies, sequence, (float)scale, interleaved != 0, inverse != 0);
}

// frequency_j = base^(-2 j / dim), those that turn `fast` times or more within `length` positions as they are, `slow` times or less over `factor`, in between
// by their turns.
__global__ __launch_bounds__(kBlock) void frequencies_kernel(double* out, int64_t count, double dim, double base, double factor, double length, double slow,
                                                             double fast) {
  constexpr double kPerRadian = 0.15915494309189533577;
  const int64_t j = (int64_t)blockIdx.x * kBlock + threadIdx.x;
  if (j >= count) return;
  const double f = pow(base, -2.0 * (double)j / dim), turns = length * f * kPerRadian;
  const double kept = fast > slow ? fmin(1.0, fmax(0.0, (turns - slow) / (fast - slow))) : 0.0;
  out[j] = f * (kept + (1.0 - kept) / factor);
}

void frequencies(THCState* s, AnyTensor* self, long dim, double base, double factor, double length, double slow, double fast) {
  const AnyTensor* all[1] = {self};
  check_same_gpu(s, 1, all);
  THC_ARG_CHECK(dim >= 2 && dim % 2 == 0 && dim < (1L << 20), 3, "an even number of elements is turned");
  THC_ARG_CHECK(base > 0, 4, "the base is not positive");
  THC_ARG_CHECK(factor > 0, 5, "the factor is not positive");
  THC_ARG_CHECK(fast >= slow, 8, "fast frequencies turn more often than slow ones");
  const long n = dim / 2;
  if (tensor_numel(self) != n) tensor_resize_nd(s, self, 1, &n, nullptr, DType::F64);
  note_stream_use(s, {self});
  const bool direct = tensor_is_contiguous(self);
  TensorRef out(s, direct ? (tensor_retain(self), self) : tensor_new_with_size(s, self->nDimension, self->size, DType::F64));
  hipLaunchKernelGGL(frequencies_kernel, dim3((unsigned)((n + kBlock - 1) / kBlock)), dim3(kBlock), 0, current_stream(s),
                     static_cast<double*>(tensor_data(out.t, DType::F64)), (int64_t)n, (double)dim, base, factor, length, slow, fast);
  THC_CHECK(hipGetLastError());
  if (out.t != self) copy_tensor(s, DType::F64, self, out.t, false);
}

}  // namespace
}  // namespace thc

#define TN(x) reinterpret_cast<thc::AnyTensor*>(x)
#define THC_AMD_DEFINE_ROTARY(Tensor, DT)                                                                                                  \
  THC_API void Tensor##_rotary(THCState* s, Tensor* self, Tensor* input, THCudaLongTensor* positions, THCudaDoubleTensor* frequencies,     \
                               double scale, int interleaved, int inverse) {                                                               \
    THC_GUARD_ALL(thc::rotary(s, DT, TN(self), TN(input), TN(positions), TN(frequencies), scale, interleaved, inverse))                    \
  }
THC_AMD_DEFINE_ROTARY(THCudaTensor, thc::DType::F32)
THC_AMD_DEFINE_ROTARY(THCudaHalfTensor, thc::DType::F16)
THC_API void THCudaDoubleTensor_rotaryFrequencies(THCState* s, THCudaDoubleTensor* self, long dim, double base, double factor, double length, double slow,
                                                  double fast) {
  THC_GUARD_ALL(thc::frequencies(s, TN(self), dim, base, factor, length, slow, fast))
}
