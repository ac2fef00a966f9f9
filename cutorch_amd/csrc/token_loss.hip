// Log-probabilities of tokens under rows of logits, and the clipped policy loss on them with its gradient.
//
//   tokenLogProb   lp_i = x_i[t_i] - m_i - log s_i       m_i = max_j x_ij, s_i = sum_j exp(x_ij - m_i)
//   policyLoss     r = exp(lp - old), l = -min(r A, clip(r, 1 - low, 1 + high) A) + kl (exp(ref - lp) - (ref - lp) - 1)
//                  loss_i = w_i l_i,   dx_ij = f w_i (dl/dlp) ([j = t_i] - exp(x_ij - m_i) / s_i)
//                  dl/dlp = (r A where r A <= clip(r) A, negated, else 0) + kl (1 - exp(ref - lp))
//
// A row is read once. Maxima, sums and the loss are in float; the gradient is rounded once. A row of weight 0 is not read: its loss,
// log-probability and gradient are 0, whatever its logits, token and other inputs hold. A token outside 1..V makes its row NaN.
#include <algorithm>

#include "training.hpp"

namespace thc {
namespace {

constexpr float kLog2e = 1.44269504088896340736f;
__device__ __forceinline__ float minus_infinity() { return -__builtin_inff(); }

// A running maximum and the sum of exp(x - max) below it. The empty one has -inf and 0; a part all of whose values are -inf too.
struct Soft {
  float m, s;
};
__device__ __forceinline__ float exp_below(float x, float m) { return __builtin_amdgcn_exp2f((x - m) * kLog2e); }
__device__ __forceinline__ Soft join(Soft a, Soft b) {
  const float m = fmaxf(a.m, b.m);
  const float safe = m == minus_infinity() ? 0.f : m;
  return Soft{m, a.s * exp_below(a.m, safe) + b.s * exp_below(b.m, safe)};
}
__device__ __forceinline__ Soft wave_join(Soft a) {
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) a = join(a, Soft{__shfl_xor(a.m, d), __shfl_xor(a.s, d)});
  return a;
}
template <int W>
__device__ __forceinline__ Soft block_join(Soft a, Soft* lds) {
  a = wave_join(a);
  if constexpr (W == 1) return a;
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = a;
  __syncthreads();
  a = lds[0];
#pragma unroll
  for (int w = 1; w < W; ++w) a = join(a, lds[w]);
  return a;
}

// The row's aligned 16-byte packs: the first begins at or below the row's first element, so it and the last may hold neighbours'
// elements, which count as -inf. Every pack holds an element of the row, so no access leaves a 16-byte unit the row owns part of.
template <typename T>
struct RowPacks {
  static constexpr int V = 16 / sizeof(T);
  using P = Pack<T, V>;
  const P* first;
  int32_t before, length, packs;
  __device__ __forceinline__ RowPacks(const T* row, int32_t n) {
    before = (int32_t)((reinterpret_cast<uintptr_t>(row) / sizeof(T)) & (V - 1));
    first = reinterpret_cast<const P*>(row - before);
    length = n;
    packs = (before + n + V - 1) / V;
  }
  __device__ __forceinline__ bool whole(int32_t k) const { return k * V >= before && (k + 1) * V <= before + length; }
  // Pack k with -inf in the place of what is not the row's.
  __device__ __forceinline__ P load(int32_t k) const {
    P p = load_pack<true>(first + k);
    if (!whole(k)) {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const int32_t i = k * V + e - before;
        if (i < 0 || i >= length) p.v[e] = Cvt<T>::down(minus_infinity());
      }
    }
    return p;
  }
};

struct RowOffsets {
  int64_t stride, outerStride;
  Divisor<uint32_t> inner;
  __device__ __forceinline__ int64_t at(uint32_t row) const {
    uint32_t q, r;
    inner.divmod(row, q, r);
    return (int64_t)q * outerStride + (int64_t)r * stride;
  }
};

// What a position brings along and what it gets, besides its row.
struct PolicyArgs {
  const int64_t* token;
  const float *old, *advantage, *reference, *weight;   // reference, weight: or null
  float *loss, *logProb;                               // loss: or null (log-probabilities alone)
  float low, high, kl, gradScale, evenWeight;
};

__device__ __forceinline__ float weight_of(const PolicyArgs& a, uint32_t row) { return a.weight ? a.weight[row] : a.evenWeight; }

// Loss and log-probability of a row, by its first lane; returns the slope f w dl/dlp.
__device__ __forceinline__ float policy_row(const PolicyArgs& a, uint32_t row, float chosen, Soft soft, float w, bool write) {
  const float lp = (chosen - soft.m) - logf(soft.s);
  if (!a.loss) {
    if (write) a.logProb[row] = lp;
    return 0.f;
  }
  const float advantage = a.advantage[row];
  const float ratio = expf(lp - a.old[row]);
  const float free = ratio * advantage, held = fminf(fmaxf(ratio, a.low), a.high) * advantage;
  // (neither below nor above: a NaN, which fmin would drop)
  float loss = free <= held ? -free : free > held ? -held : free + held;
  float slope = free <= held ? -free : free > held ? 0.f : free + held;
  if (a.reference) {
    const float away = a.reference[row] - lp, e = expf(away);
    loss += a.kl * (e - away - 1.f);
    slope += a.kl * (1.f - e);
  }
  if (write) {
    a.loss[row] = w * loss;
    a.logProb[row] = lp;
  }
  return w * slope * a.gradScale;
}

// One workgroup a row; the row is read twice, the second time for the gradient.
template <typename T, int W, bool GRAD>
__global__ __launch_bounds__(W * 64) void row_kernel(PolicyArgs a, const T* logits, RowOffsets lo, T* grad, RowOffsets go,
                                                     int32_t vocab) {
  constexpr int V = RowPacks<T>::V;
  using P = Pack<T, V>;
  __shared__ Soft lds[W];
  const uint32_t row = blockIdx.x;
  const float w = weight_of(a, row);
  T* out = GRAD ? grad + go.at(row) : nullptr;
  if (w == 0.f) {
    if (threadIdx.x == 0) {
      if (a.loss) a.loss[row] = 0.f;
      a.logProb[row] = 0.f;
    }
    if constexpr (GRAD)
      for (int32_t i = threadIdx.x; i < vocab; i += W * 64) out[i] = Cvt<T>::down(0.f);
    return;
  }
  const T* x = logits + lo.at(row);
  const int64_t token = a.token[row] - 1;
  const float chosen = (uint64_t)token < (uint64_t)vocab ? Cvt<T>::up(x[token]) : __builtin_nanf("");
  const RowPacks<T> packs(x, vocab);
  Soft soft{minus_infinity(), 0.f};
  for (int32_t k = threadIdx.x; k < packs.packs; k += W * 64) {
    const P p = packs.load(k);
    float m = Cvt<T>::up(p.v[0]);
#pragma unroll
    for (int e = 1; e < V; ++e) m = fmaxf(m, Cvt<T>::up(p.v[e]));
    const float top = fmaxf(m, soft.m), safe = top == minus_infinity() ? 0.f : top;
    float s = soft.s * exp_below(soft.m, safe);
#pragma unroll
    for (int e = 0; e < V; ++e) s += exp_below(Cvt<T>::up(p.v[e]), safe);
    soft = Soft{top, s};
  }
  soft = block_join<W>(soft, lds);
  const float slope = policy_row(a, row, chosen, soft, w, threadIdx.x == 0);
  if constexpr (GRAD) {
    const float c = -slope / soft.s;
    const int32_t hit = (int32_t)token;
    for (int32_t k = threadIdx.x; k < packs.packs; k += W * 64) {
      const P p = packs.load(k);
      P g;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        float d = c * exp_below(Cvt<T>::up(p.v[e]), soft.m);
        if (k * V + e - packs.before == hit) d += slope;
        g.v[e] = rounded<T>(d);
      }
      const int32_t i0 = k * V - packs.before;
      if (packs.whole(k)) {
        store_pack_unaligned<false>(out + i0, g);
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (i0 + e >= 0 && i0 + e < vocab) out[i0 + e] = g.v[e];
      }
    }
  }
}

RowOffsets offsets_of(const Rows& r) {
  RowOffsets o;
  o.stride = r.stride;
  o.outerStride = r.outerStride;
  o.inner.set((uint64_t)r.inner);
  return o;
}

template <typename T>
void launch_rows(THCState* s, const PolicyArgs& a, const T* logits, const Rows& lr, T* grad, const Rows& gr) {
  hipStream_t st = current_stream(s);
  const dim3 grid((unsigned)lr.count);
  if (grad)
    hipLaunchKernelGGL((row_kernel<T, 4, true>), grid, dim3(256), 0, st, a, logits, offsets_of(lr), grad, offsets_of(gr), (int32_t)lr.length);
  else
    hipLaunchKernelGGL((row_kernel<T, 4, false>), grid, dim3(256), 0, st, a, logits, offsets_of(lr), grad, offsets_of(lr), (int32_t)lr.length);
}

// A per-position operand: float, as many elements as there are rows.
void check_positions(const AnyTensor* t, int64_t rows, int arg, const char* what) {
  THC_ARG_CHECK(tensor_numel(t) == rows, arg, "%ld %s for %ld rows of logits", (long)tensor_numel(t), what, (long)rows);
}

// Outputs take the tokens' sizes and are written densely; `meets`: one lies on what the call reads.
AnyTensor* position_output(THCState* s, AnyTensor* out, bool meets) {
  if (tensor_is_contiguous(out) && !meets) {
    tensor_retain(out);
    return out;
  }
  return tensor_new_with_size(s, out->nDimension, out->size, DType::F32);
}

struct PolicyCall {
  AnyTensor *loss, *logProb, *grad, *logits, *tokens, *old, *advantage, *reference, *weight;   // loss null: log-probabilities alone
  double low, high, kl, gradScale;
};

void token_loss(THCState* s, DType dt, const PolicyCall& c) {
  const AnyTensor* all[9] = {c.loss, c.logProb, c.grad, c.logits, c.tokens, c.old, c.advantage, c.reference, c.weight};
  check_same_gpu(s, 9, all);
  const bool policy = c.loss != nullptr;
  const int logitsArg = policy ? 5 : 3, tokensArg = policy ? 6 : 4;
  THC_ARG_CHECK(has_elements(c.logits), logitsArg, "the logits are empty");
  THC_ARG_CHECK(c.logits->nDimension <= kMaxDims, logitsArg, "%s", kDimWarning);
  const int64_t vocab = c.logits->size[c.logits->nDimension - 1], rows = tensor_numel(c.logits) / vocab;
  THC_ARG_CHECK(vocab < (int64_t(1) << 30), logitsArg, "rows of the logits are too long");
  THC_ARG_CHECK(rows < kIndex32Limit, logitsArg, "too many rows of logits");
  check_positions(c.tokens, rows, tokensArg, "tokens");
  if (policy) {
    check_positions(c.old, rows, 7, "old log-probabilities");
    check_positions(c.advantage, rows, 8, "advantages");
    if (c.reference) check_positions(c.reference, rows, 9, "reference log-probabilities");
    if (c.weight) check_positions(c.weight, rows, 10, "weights");
    THC_ARG_CHECK(c.low >= 0 && c.low <= 1 && c.high >= 0, 11, "the ratio is clipped to 1 - low and 1 + high, low from 0 to 1, high from 0");
  }
  note_stream_use(s, {c.loss, c.logProb, c.grad, c.logits, c.tokens, c.old, c.advantage, c.reference, c.weight});

  Rows lr{};
  const bool direct = as_rows(c.logits, &lr);
  TensorRef logits(s, direct ? (tensor_retain(c.logits), c.logits) : tensor_new_contiguous(s, c.logits, dt));
  as_rows(logits.t, &lr);
  Dense tokens(s, c.tokens, DType::I64);
  PolicyArgs a{};
  a.token = tokens.data<int64_t>();
  a.evenWeight = 1.f;
  TensorRef old(s, nullptr), advantage(s, nullptr), reference(s, nullptr), weight(s, nullptr);
  if (policy) {
    auto dense = [&](TensorRef& hold, AnyTensor* t) -> const float* {
      if (!t) return nullptr;
      hold.t = tensor_new_contiguous(s, t, DType::F32);
      return (const float*)tensor_data(hold.t, DType::F32);
    };
    a.old = dense(old, c.old);
    a.advantage = dense(advantage, c.advantage);
    a.reference = c.kl != 0 ? dense(reference, c.reference) : nullptr;
    a.weight = dense(weight, c.weight);
    a.evenWeight = (float)(1.0 / (double)rows);
    a.low = (float)(1.0 - c.low);
    a.high = (float)(1.0 + c.high);
    a.kl = (float)c.kl;
    a.gradScale = (float)c.gradScale;
  }
  const AnyTensor* read[5] = {logits.t, old.t, advantage.t, reference.t, weight.t};
  const DType readType[5] = {dt, DType::F32, DType::F32, DType::F32, DType::F32};
  auto meets = [&](const AnyTensor* out, DType t, int from) {
    for (int i = from; i < 5; ++i)
      if (spans_meet(out, t, read[i], readType[i])) return true;
    return false;
  };
  TensorRef loss(s, nullptr), logProb(s, nullptr), grad(s, nullptr);
  tensor_resize_as(s, c.logProb, c.tokens, DType::F32);
  logProb.t = position_output(s, c.logProb, meets(c.logProb, DType::F32, 0));
  a.logProb = (float*)tensor_data(logProb.t, DType::F32);
  if (policy) {
    tensor_resize_as(s, c.loss, c.tokens, DType::F32);
    loss.t = position_output(s, c.loss, meets(c.loss, DType::F32, 0));
    a.loss = (float*)tensor_data(loss.t, DType::F32);
  }
  Rows gr{};
  if (c.grad) {
    tensor_resize_as(s, c.grad, c.logits, dt);
    // in the place of the logits, or apart from everything that is read
    bool fits = as_rows(c.grad, &gr) && !overlapping(tensor_layout(c.grad)) && !meets(c.grad, dt, 1);
    if (fits && spans_meet(c.grad, dt, logits.t, dt))
      fits = c.grad->storageOffset == logits.t->storageOffset && gr.inner == lr.inner && gr.stride == lr.stride && gr.outerStride == lr.outerStride;
    grad.t = fits ? (tensor_retain(c.grad), c.grad) : tensor_new_with_size(s, c.grad->nDimension, c.grad->size, dt);
    as_rows(grad.t, &gr);
  }
  if (dt == DType::F32)
    launch_rows<float>(s, a, (const float*)tensor_data(logits.t, dt), lr, grad.t ? (float*)tensor_data(grad.t, dt) : nullptr, gr);
  else
    launch_rows<__half>(s, a, (const __half*)tensor_data(logits.t, dt), lr, grad.t ? (__half*)tensor_data(grad.t, dt) : nullptr, gr);
  THC_CHECK(hipGetLastError());
  note_kernel(policy ? "policy-loss" : "token-logprob");
  if (loss.t && loss.t != c.loss) copy_tensor(s, DType::F32, c.loss, loss.t, false);
  if (logProb.t != c.logProb) copy_tensor(s, DType::F32, c.logProb, logProb.t, false);
  if (grad.t && grad.t != c.grad) copy_tensor(s, dt, c.grad, grad.t, false);
}

}  // namespace
}  // namespace thc

#define TN(x) reinterpret_cast<thc::AnyTensor*>(x)
#define THC_AMD_DEFINE_TOKEN_LOSS(Tensor, DT)                                                                                              \
  THC_API void Tensor##_tokenLogProb(THCState* s, THCudaTensor* self, Tensor* logits, THCudaLongTensor* tokens) {                          \
    THC_GUARD_ALL(thc::token_loss(s, DT, {nullptr, TN(self), nullptr, TN(logits), TN(tokens), nullptr, nullptr, nullptr, nullptr, 0, 0, 0, 0})) \
  }                                                                                                                                        \
  THC_API void Tensor##_policyLoss(THCState* s, THCudaTensor* loss, THCudaTensor* logProb, Tensor* gradLogits, Tensor* logits,            \
                                   THCudaLongTensor* tokens, THCudaTensor* oldLogProb, THCudaTensor* advantage,                           \
                                   THCudaTensor* refLogProb, THCudaTensor* weight, double clipLow, double clipHigh, double klCoef,         \
                                   double gradScale) {                                                                                     \
    THC_GUARD_ALL({                                                                                                                        \
      THC_ARG_CHECK(loss != nullptr, 2, "no tensor for the losses");                                                                       \
      thc::token_loss(s, DT, {TN(loss), TN(logProb), TN(gradLogits), TN(logits), TN(tokens), TN(oldLogProb), TN(advantage),               \
                              TN(refLogProb), TN(weight), clipLow, clipHigh, klCoef, gradScale});                                          \
    })                                                                                                                                     \
  }
THC_AMD_DEFINE_TOKEN_LOSS(THCudaTensor, thc::DType::F32)
THC_AMD_DEFINE_TOKEN_LOSS(THCudaHalfTensor, thc::DType::F16)
