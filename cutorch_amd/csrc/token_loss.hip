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
#include <type_traits>

#include "training.hpp"

namespace thc {
namespace {

constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
__device__ __forceinline__ float minus_infinity() { return -__builtin_inff(); }

// A running maximum and the sum of 2^(distance below it), distances in powers of two. The empty part has -inf and 0; so has one all of
// whose values are -inf.
//   half   m is the maximum times log2(e), rounded; x log2(e) - m is one operation, which takes x as it is, and rounds once, near 0 for the
//          values that count. What m's rounding moved cancels: the chosen logit and the gradient are measured from the same m.
//   float  m is the maximum itself and (x - m) log2(e) two operations: the product with m overflows where a whole row holds the type's
//          lowest value.
struct Soft {
  float m, s;
};
template <typename T>
__device__ __forceinline__ float scaled(float x) {
  return sizeof(T) == 2 ? x * kLog2e : x;
}
template <typename T>
__device__ __forceinline__ float below(float x, float m) {
  if constexpr (sizeof(T) == 2) return __builtin_fmaf(x, kLog2e, -m);
  else return (x - m) * kLog2e;
}
template <typename T>
__device__ __forceinline__ float exp_below(float x, float m) {
  return __builtin_amdgcn_exp2f(below<T>(x, m));
}
// What a sum below m becomes below `top`.
template <typename T>
__device__ __forceinline__ float lowered(float m, float top) {
  return __builtin_amdgcn_exp2f(sizeof(T) == 2 ? m - top : (m - top) * kLog2e);
}
__device__ __forceinline__ float finite_or_zero(float m) { return m == minus_infinity() ? 0.f : m; }
template <typename T>
__device__ __forceinline__ Soft join(Soft a, Soft b) {
  const float m = fmaxf(a.m, b.m), safe = finite_or_zero(m);
  return Soft{m, a.s * lowered<T>(a.m, safe) + b.s * lowered<T>(b.m, safe)};
}
template <typename T>
__device__ __forceinline__ Soft wave_join(Soft a) {
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) a = join<T>(a, Soft{__shfl_xor(a.m, d), __shfl_xor(a.s, d)});
  return a;
}
template <typename T, int W>
__device__ __forceinline__ Soft block_join(Soft a, Soft* lds) {
  a = wave_join<T>(a);
  if constexpr (W > 1) {
    const int lane = threadIdx.x & 63;
    if (lane == 0) lds[threadIdx.x >> 6] = a;
    lds_barrier();
    a = lds[lane & (W - 1)];
#pragma unroll
    for (int d = W / 2; d >= 1; d >>= 1) a = join<T>(a, Soft{__shfl_xor(a.m, d), __shfl_xor(a.s, d)});
  }
  return a;
}
// log(2^(x's distance below m) / s)
template <typename T>
__device__ __forceinline__ float log_share(float x, Soft soft) {
  if constexpr (sizeof(T) == 2) return (below<T>(x, soft.m) - log2f(soft.s)) * kLn2;
  else return (x - soft.m) - log2f(soft.s) * kLn2;
}

// A row as its aligned 16-byte packs and the elements before and behind them, of which lanes 0 to 15 of the first wave hold one each.
template <typename T>
struct RowParts {
  static constexpr int V = 16 / sizeof(T);
  using P = Pack<T, V>;
  const T* row;
  const P* first;
  int32_t head, packs, tail;
  int32_t lane0;      // the pack that thread 0 has first: it lies where a 128-byte line begins, so that no two waves write into one line
  __device__ __forceinline__ RowParts(const T* x, int32_t n) {
    row = x;
    head = min(n, (int32_t)((-reinterpret_cast<uintptr_t>(x) / sizeof(T)) & (V - 1)));
    first = reinterpret_cast<const P*>(x + head);
    packs = (n - head) / V;
    tail = n - head - packs * V;
    lane0 = -(int32_t)((reinterpret_cast<uintptr_t>(first) / 16) & 7);
  }
  __device__ __forceinline__ bool has(int32_t k) const { return (uint32_t)k < (uint32_t)packs; }
  // The element that this lane holds besides its packs, or -1.
  __device__ __forceinline__ int32_t edge() const {
    const int32_t t = threadIdx.x;
    return t < V ? (t < head ? t : -1) : t < 2 * V && t - V < tail ? head + packs * V + t - V : -1;
  }
  __device__ __forceinline__ P load(int32_t k) const { return load_pack<true>(first + k); }
  __device__ __forceinline__ float load_edge(int32_t i) const { return i >= 0 ? Cvt<T>::up(row[i]) : minus_infinity(); }
};

// Rows go along the grid's x and, behind the first 2^21 of them, y (a launch has less than 2^32 threads in a dim).
constexpr int kRowsAcross = 21;
__device__ __forceinline__ uint32_t grid_row() { return blockIdx.x + (blockIdx.y << kRowsAcross); }

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

// A position's numbers, asked for before its row is.
struct Position {
  int64_t token;      // 0-based
  float weight, old, advantage, reference;
};
__device__ __forceinline__ Position position_of(const PolicyArgs& a, uint32_t row) {
  Position p{};
  p.token = a.token[row] - 1;
  p.weight = a.weight ? a.weight[row] : a.evenWeight;
  if (a.loss) {
    p.old = a.old[row];
    p.advantage = a.advantage[row];
    if (a.reference) p.reference = a.reference[row];
  }
  return p;
}

// Loss and log-probability of a row, by its first lane; returns the slope f w dl/dlp.
template <typename T>
__device__ __forceinline__ float policy_row(const PolicyArgs& a, uint32_t row, const Position& p, float chosen, Soft soft, bool write) {
  const float lp = log_share<T>(chosen, soft);
  if (!a.loss) {
    if (write) a.logProb[row] = lp;
    return 0.f;
  }
  const float ratio = expf(lp - p.old);
  const float free = ratio * p.advantage, held = fminf(fmaxf(ratio, a.low), a.high) * p.advantage;
  // (neither below nor above: a NaN, which fmin would drop)
  float loss = free <= held ? -free : free > held ? -held : free + held;
  float slope = free <= held ? -free : free > held ? 0.f : free + held;
  if (a.reference) {
    const float away = p.reference - lp, e = expf(away);
    loss += a.kl * (e - away - 1.f);
    slope += a.kl * (1.f - e);
  }
  if (write) {
    a.loss[row] = p.weight * loss;
    a.logProb[row] = lp;
  }
  return p.weight * slope * a.gradScale;
}

template <typename T>
__device__ __forceinline__ float top_of(const Pack<T, 16 / sizeof(T)>& p) {
  if constexpr (sizeof(T) == 2) {
    typedef _Float16 Two __attribute__((ext_vector_type(2)));
    Two h[4];
    __builtin_memcpy(h, &p, 16);
    const Two m = __builtin_elementwise_max(__builtin_elementwise_max(h[0], h[1]), __builtin_elementwise_max(h[2], h[3]));
    return fmaxf((float)m[0], (float)m[1]);
  } else {
    return fmaxf(fmaxf(p.v[0], p.v[1]), fmaxf(p.v[2], p.v[3]));
  }
}
template <typename T>
__device__ __forceinline__ float sum_below(const Pack<T, 16 / sizeof(T)>& p, float m) {
  constexpr int V = 16 / sizeof(T);
  float s[V];
#pragma unroll
  for (int e = 0; e < V; ++e) s[e] = exp_below<T>(Cvt<T>::up(p.v[e]), m);
#pragma unroll
  for (int w = V / 2; w >= 1; w /= 2) {
#pragma unroll
    for (int e = 0; e < w; ++e) s[e] += s[e + w];
  }
  return s[0];
}

// What a row's gradient is made from: c 2^(x log2(e) - m), and `slope` more at the token, element `hit` of the row.
struct RowSlope {
  float c, slope, m;
  int32_t hit;
};
// A pack of the gradient; its first element is element i0 of the row. The stores are streaming ones at every size: with plain ones 4096 x
// 100001 halves take 305 us instead of 285, 512 x 32000 16.5 instead of 13.9, 1000 x 8000 11.6 instead of 9.2.
template <typename T>
__device__ __forceinline__ void store_gradient(T* out, int32_t i0, const Pack<T, 16 / sizeof(T)>& p, const RowSlope& r) {
  constexpr int V = 16 / sizeof(T);
  float g[V];
#pragma unroll
  for (int e = 0; e < V; ++e) g[e] = r.c * exp_below<T>(Cvt<T>::up(p.v[e]), r.m);
  if ((uint32_t)(r.hit - i0) < (uint32_t)V) {
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (i0 + e == r.hit) g[e] += r.slope;
  }
  Pack<T, V> q;
  if constexpr (sizeof(T) == 2) {
    typedef _Float16 Half2 __attribute__((ext_vector_type(2)));
    typedef float Float2 __attribute__((ext_vector_type(2)));
    Half2 h[V / 2];
#pragma unroll
    for (int e = 0; e < V / 2; ++e) h[e] = __builtin_convertvector((Float2{g[2 * e], g[2 * e + 1]}), Half2);
    __builtin_memcpy(&q, h, 16);
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) q.v[e] = g[e];
  }
  store_pack_unaligned<true>(out + i0, q);
}
template <typename T>
__device__ __forceinline__ void store_edge(T* out, int32_t i, float x, const RowSlope& r) {
  if (i >= 0) out[i] = rounded<T>(r.c * exp_below<T>(x, r.m) + (i == r.hit ? r.slope : 0.f));
}
// Streaming stores for short rows, plain ones for long ones, whose workgroups are done when the caches have them (a tenth of the rows; us
// with plain and with streaming ones: 16384 x 1000 halves 19.5, 18.5, 8192 x 32000 169, 178, 4096 x 100001 288, 293).
template <typename T, int W>
__device__ __forceinline__ void store_zeros(T* out, int32_t n) {
  constexpr int V = 16 / sizeof(T);
  const RowParts<T> x(out, n);
  Pack<T, V> zero;
#pragma unroll
  for (int e = 0; e < V; ++e) zero.v[e] = Cvt<T>::down(0.f);
  if (x.edge() >= 0) out[x.edge()] = zero.v[0];
  for (int32_t k = x.lane0 + (int32_t)threadIdx.x; k < x.packs; k += W * 64)
    if (x.has(k)) store_pack_unaligned<W == 1>(out + x.head + k * V, zero);
}

// A row without a weight: its outputs are 0. (A NaN weight is one.)
template <typename T, int W, bool GRAD>
__device__ __forceinline__ void skip_row(const PolicyArgs& a, uint32_t row, T* out, int32_t vocab) {
  if (threadIdx.x == 0) {
    if (a.loss) a.loss[row] = 0.f;
    a.logProb[row] = 0.f;
  }
  if constexpr (GRAD) store_zeros<T, W>(out, vocab);
}
template <typename T>
__device__ __forceinline__ float chosen_of(const T* x, int64_t token, int32_t vocab) {
  return (uint64_t)token < (uint64_t)vocab ? Cvt<T>::up(x[token]) : __builtin_nanf("");
}

// Takes the packs at k, k + step, ... (U of them; those behind `end` are not there) into a running maximum and sum.
template <typename T, int U>
__device__ __forceinline__ Soft take(Soft soft, const Pack<T, 16 / sizeof(T)>* v, int32_t k, int32_t step, int32_t end) {
  float m = soft.m;
#pragma unroll
  for (int u = 0; u < U; ++u)
    if ((uint32_t)(k + u * step) < (uint32_t)end) m = fmaxf(m, scaled<T>(top_of<T>(v[u])));
  const float safe = finite_or_zero(m);
  float s = soft.s * lowered<T>(soft.m, safe);
#pragma unroll
  for (int u = 0; u < U; ++u)
    if ((uint32_t)(k + u * step) < (uint32_t)end) s += sum_below<T>(v[u], safe);
  return Soft{m, s};
}
template <typename T>
__device__ __forceinline__ Soft take_edge(float x) {
  const float m = scaled<T>(x);
  return Soft{m, m == minus_infinity() ? 0.f : exp_below<T>(x, m)};
}

// Direct load of one pack a lane into LDS: lane i's 16 bytes go to `to` + 16 i of the wave's part.
__device__ __forceinline__ void load_to_lds(const void* from, void* to) {
  typedef const __attribute__((address_space(1))) void* Global;
  typedef __attribute__((address_space(3))) void* Local;
  __builtin_amdgcn_global_load_lds((Global)from, (Local)to, 16, 0, /*nt*/ 2);
}

// A workgroup has a row, a lane R packs of it in registers and L in LDS from the first read to the gradient: the row crosses the memory
// once each way. What is longer than that is read again for the gradient (REST): the first time with plain loads, so that
// the caches may have it (2048 x 262144 halves 484 us with streaming ones, 437). E: waves a SIMD that the registers leave room for.
// Bound by memory, reads and writes in turn: 4096 x 100001 halves, a tenth of them without a weight, 285 us, 5.5 TB/s (a flat copy 6.1); 96 x 1000
// floats 4.1, a launch. (Workgroups that ask for their next row while this one's gradient is made: 334 to 378 us, 333 to 363 without, for
// the registers that it takes.)
template <typename T, int W, int R, int L, int E, bool REST>
__global__ __launch_bounds__(W * 64) __attribute__((amdgpu_waves_per_eu(E, E))) void held_row_kernel(PolicyArgs a, const T* logits, RowOffsets lo, T* grad,
                                                                                               RowOffsets go, int32_t vocab, uint32_t rows) {
  constexpr int U = R < 4 ? R : 4, kStep = W * 64, V = 16 / sizeof(T);
  static_assert(R % U == 0, "registers are taken U packs at a time");
  using P = Pack<T, V>;
  __shared__ Soft lds[W];
  extern __shared__ __attribute__((aligned(16))) char room[];      // L packs a lane
  P(*more)[W][64] = reinterpret_cast<P(*)[W][64]>(room);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t row = grid_row();
  if (row >= rows) return;
  const Position at = position_of(a, row);
  T* out = grad + go.at(row);
  if (at.weight == 0.f) {
    skip_row<T, W, true>(a, row, out, vocab);
    return;
  }
  const RowParts<T> x(logits + lo.at(row), vocab);
  P v[R];
#pragma unroll
  for (int u = 0; u < R; ++u) {
    const int32_t k = x.lane0 + (int32_t)threadIdx.x + u * kStep;
    if (x.has(k)) v[u] = x.load(k);
  }
#pragma unroll
  for (int u = 0; u < L; ++u) {
    const int32_t k = x.lane0 + (int32_t)threadIdx.x + (R + u) * kStep;
    if (x.has(k)) load_to_lds(x.first + k, &more[u][wave][0]);
  }
  float chosen = chosen_of(x.row, at.token, vocab);
  const float edge = x.load_edge(x.edge());
  Soft soft{minus_infinity(), 0.f};
#pragma unroll
  for (int u = 0; u < R; u += U) soft = take<T, U>(soft, v + u, x.lane0 + (int32_t)threadIdx.x + u * kStep, kStep, x.packs);
  if constexpr (L > 0) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
    for (int u = 0; u < L; ++u) {
      const int32_t k = x.lane0 + (int32_t)threadIdx.x + (R + u) * kStep;
      const P p = more[u][wave][lane];
      soft = take<T, 1>(soft, &p, k, kStep, x.packs);
    }
  }
  if constexpr (REST) {
    for (int32_t k = x.lane0 + (int32_t)threadIdx.x + (R + L) * kStep; k < x.packs; k += U * kStep) {
      P q[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (x.has(k + u * kStep)) q[u] = load_pack<false>(x.first + k + u * kStep);
      soft = take<T, U>(soft, q, k, kStep, x.packs);
    }
  }
  // (the barrier does not wait for loads, and behind it another wave may write where the chosen logit was)
  asm volatile("" : "+v"(chosen));
  soft = block_join<T, W>(join<T>(soft, take_edge<T>(edge)), lds);
  const float slope = policy_row<T>(a, row, at, chosen, soft, threadIdx.x == 0);
  const RowSlope r{-slope / soft.s, slope, soft.m, (int32_t)at.token};
  store_edge(out, x.edge(), edge, r);
#pragma unroll
  for (int u = 0; u < R; ++u) {
    const int32_t k = x.lane0 + (int32_t)threadIdx.x + u * kStep;
    if (x.has(k)) store_gradient<T>(out, x.head + k * V, v[u], r);
  }
#pragma unroll
  for (int u = 0; u < L; ++u) {
    const int32_t k = x.lane0 + (int32_t)threadIdx.x + (R + u) * kStep;
    if (x.has(k)) store_gradient<T>(out, x.head + k * V, more[u][wave][lane], r);
  }
  if constexpr (REST) {
    for (int32_t k = x.lane0 + (int32_t)threadIdx.x + (R + L) * kStep; k < x.packs; k += U * kStep) {
      P q[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (x.has(k + u * kStep)) q[u] = x.load(k + u * kStep);
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (x.has(k + u * kStep)) store_gradient<T>(out, x.head + (k + u * kStep) * V, q[u], r);
    }
  }
}

// Losses and log-probabilities alone: a workgroup has a row. Bound by reading: 4096 x 50001 floats 123 us, 6.7 TB/s.
template <typename T, int W>
__global__ __launch_bounds__(W * 64) void row_kernel(PolicyArgs a, const T* __restrict__ logits, RowOffsets lo, int32_t vocab, uint32_t rows) {
  constexpr int U = 4, kStep = W * 64, V = 16 / sizeof(T);
  using P = Pack<T, V>;
  __shared__ Soft lds[W];
  const uint32_t row = grid_row();
  if (row >= rows) return;
  const Position at = position_of(a, row);
  if (at.weight == 0.f) {
    skip_row<T, W, false>(a, row, (T*)nullptr, vocab);
    return;
  }
  const RowParts<T> x(logits + lo.at(row), vocab);
  const float chosen = chosen_of(x.row, at.token, vocab);
  Soft soft = take_edge<T>(x.load_edge(x.edge()));
  for (int32_t k = x.lane0 + (int32_t)threadIdx.x; k < x.packs; k += U * kStep) {
    P v[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (x.has(k + u * kStep)) v[u] = x.load(k + u * kStep);
    soft = take<T, U>(soft, v, k, kStep, x.packs);
  }
  soft = block_join<T, W>(soft, lds);
  policy_row<T>(a, row, at, chosen, soft, threadIdx.x == 0);
}

// Few long rows: each is cut into `parts` (at most 64) of `per` packs, a workgroup each, and a second launch joins their maxima and sums;
// with a gradient every part joins them for itself and reads its packs again, from the caches. Bound by the two launches: 24 x 128000 halves 7.4 us,
// 4.5 and 2.8 (in one launch, the row's last workgroup to arrive joining: 11.2, for a store, a count and a load past the caches in turn).
struct Parts {
  Soft* soft;       // of each row, side by side
  float* chosen;    // of each row: the second launch may write the gradient over it
  int32_t parts, per;
};
template <typename T, int W>
__global__ __launch_bounds__(W * 64) void part_kernel(PolicyArgs a, const T* __restrict__ logits, RowOffsets lo, int32_t vocab, Parts p) {
  constexpr int U = 4, kStep = W * 64, V = 16 / sizeof(T);
  using P = Pack<T, V>;
  __shared__ Soft lds[W];
  const uint32_t row = blockIdx.y, part = blockIdx.x;
  if (a.weight && a.weight[row] == 0.f) return;
  const RowParts<T> x(logits + lo.at(row), vocab);
  Soft soft = take_edge<T>(part == 0 ? x.load_edge(x.edge()) : minus_infinity());
  const int32_t begin = x.lane0 + (int32_t)part * p.per, end = min(x.packs, begin + p.per);
  for (int32_t k = begin + (int32_t)threadIdx.x; k < end; k += U * kStep) {
    P v[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (k + u * kStep < end && x.has(k + u * kStep)) v[u] = x.load(k + u * kStep);
    soft = take<T, U>(soft, v, k, kStep, end);
  }
  soft = block_join<T, W>(soft, lds);
  if (threadIdx.x == 0) {
    p.soft[(int64_t)row * p.parts + part] = soft;
    if (part == 0) p.chosen[row] = chosen_of(x.row, a.token[row] - 1, vocab);
  }
}
template <typename T, int W, bool GRAD>
__global__ __launch_bounds__(W * 64) void join_kernel(PolicyArgs a, const T* logits, RowOffsets lo, T* grad, RowOffsets go, int32_t vocab, Parts p) {
  constexpr int U = 4, kStep = W * 64, V = 16 / sizeof(T);
  using P = Pack<T, V>;
  const uint32_t row = blockIdx.y, part = blockIdx.x;
  const int lane = threadIdx.x & 63;
  const Position at = position_of(a, row);
  const RowParts<T> x(logits + lo.at(row), vocab);
  T* out = GRAD ? grad + go.at(row) : nullptr;
  const int32_t begin = x.lane0 + (int32_t)part * p.per, end = min(x.packs, begin + p.per);
  const bool first = part == 0 && threadIdx.x == 0;
  Soft soft{minus_infinity(), 0.f};
  RowSlope r{0.f, 0.f, 0.f, -1};
  if (at.weight != 0.f) {
    if (lane < p.parts) soft = p.soft[(int64_t)row * p.parts + lane];
    const float chosen = p.chosen[row];
    soft = wave_join<T>(soft);
    const float slope = policy_row<T>(a, row, at, chosen, soft, first);
    r = RowSlope{-slope / soft.s, slope, soft.m, (int32_t)at.token};
  } else if (first) {
    if (a.loss) a.loss[row] = 0.f;
    a.logProb[row] = 0.f;
  }
  if constexpr (GRAD) {
    const bool used = at.weight != 0.f;
    if (part == 0) {
      const int32_t i = x.edge();
      if (used) store_edge(out, i, x.load_edge(i), r);
      else if (i >= 0) out[i] = Cvt<T>::down(0.f);
    }
    for (int32_t k = begin + (int32_t)threadIdx.x; k < end; k += U * kStep) {
      P v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (k + u * kStep < end && x.has(k + u * kStep)) {
          if (used) {
            v[u] = x.load(k + u * kStep);
          } else {
#pragma unroll
            for (int e = 0; e < V; ++e) v[u].v[e] = Cvt<T>::down(0.f);
          }
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (k + u * kStep < end && x.has(k + u * kStep)) store_gradient<T>(out, x.head + (k + u * kStep) * V, v[u], r);
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
  const uint32_t rows = (uint32_t)lr.count;
  const dim3 grid(std::min(rows, 1u << kRowsAcross), (rows + (1u << kRowsAcross) - 1) >> kRowsAcross);
  const int32_t vocab = (int32_t)lr.length;
  constexpr int V = 16 / sizeof(T);
  const int32_t packs = vocab / V + 7;      // at most, with those that a line's begin is before the row
  const RowOffsets lo = offsets_of(lr), go = grad ? offsets_of(gr) : lo;
  // Few long rows are split. us with a workgroup a row and split: log-probabilities of 24 rows of 32000 halves 6.5, 6.4, of 128000 13.3, 7.6;
  // 128 x 128000 15.2, 13.0; 256 x 128000 16.5, 18.7; 1 x 262144 22, 6. Losses with gradients, whose rows are then read twice: 24 x 32000
  // 8.4, 8.7; 24 x 128000 18.5, 11.1; 64 x 128000 19.2, 16.7; 128 x 128000 20.4, 25.7.
  const int64_t perRow = tuning("loss.split", 100);
  if (lr.count <= 128 && packs >= (grad ? 10240 : 6144) && packs >= lr.count * perRow * (grad ? 2 : 1)) {
    constexpr int W = 4;
    Parts p;
    p.parts = (int32_t)std::max<int64_t>(1, std::min<int64_t>(64, 4096 / (lr.count * W)));
    p.per = ((packs + p.parts - 1) / p.parts + W * 64 - 1) / (W * 64) * (W * 64);
    p.parts = (packs + p.per - 1) / p.per;
    Workspace w(s, lr.count * (p.parts * (int64_t)sizeof(Soft) + 4));
    p.soft = reinterpret_cast<Soft*>(w.data());
    p.chosen = reinterpret_cast<float*>(p.soft + lr.count * p.parts);
    const dim3 cut((unsigned)p.parts, (unsigned)lr.count);
    hipLaunchKernelGGL((part_kernel<T, W>), cut, dim3(W * 64), 0, st, a, logits, lo, vocab, p);
    if (grad) hipLaunchKernelGGL((join_kernel<T, W, true>), cut, dim3(W * 64), 0, st, a, logits, lo, grad, go, vocab, p);
    else hipLaunchKernelGGL((join_kernel<T, 1, false>), dim3(1, (unsigned)lr.count), dim3(64), 0, st, a, logits, lo, grad, go, vocab, p);
    return;
  }
  using std::integral_constant;
  if (!grad) {
    // Waves a row: as many as leave about 16 to a CU, but two packs a lane. us with 1, 2, 4, 8, 16: 16384 rows of 4000 halves 23.5, 23.6, 34,
    // 56, 88; 1000 x 32000 22, 14.5, 16, 15, 18.5; 600 x 128000 72, 42, 45, 31, 35; 256 x 16000 fp32 with 4 and 16 11.4, 6.9.
    auto go = [&](auto wTag) {
      constexpr int W = decltype(wTag)::value;
      hipLaunchKernelGGL((row_kernel<T, W>), grid, dim3(W * 64), 0, st, a, logits, lo, vocab, rows);
    };
    const int64_t want = 4800;
    if (lr.count >= want || packs < 256) go(integral_constant<int, 1>{});
    else if (lr.count * 2 >= want || packs < 512) go(integral_constant<int, 2>{});
    else if (lr.count * 4 >= want || packs < 1024) go(integral_constant<int, 4>{});
    else if (lr.count * 8 >= want || packs < 2048) go(integral_constant<int, 8>{});
    else go(integral_constant<int, 16>{});
    return;
  }
  auto held = [&](auto waves, auto registers, auto shared, auto perSimd, auto rest) {
    constexpr int W = decltype(waves)::value, R = decltype(registers)::value, L = decltype(shared)::value;
    hipLaunchKernelGGL((held_row_kernel<T, W, R, L, decltype(perSimd)::value, decltype(rest)::value>), grid, dim3(W * 64), L * W * 64 * 16, st, a,
                       logits, lo, grad, go, vocab, rows);
  };
#define HELD(W, R, L, E, REST)                                                                                            \
  held(integral_constant<int, W>{}, integral_constant<int, R>{}, integral_constant<int, L>{}, integral_constant<int, E>{}, \
       integral_constant<bool, REST>{})
  // The least that hold a row, so that a CU has several: one loads while another computes and a third stores. us, halves with gradients:
  // 16384 x 8000 with 4 waves of 4, 8 and 16 packs 82, 84, 100; 8192 x 16000 with 8 waves of 4 and 8, 16 of 8 84, 88, 111; 8192 x 32000
  // with 8 of 8, 16 of 8 and 16 of 16 168, 170, 256; 4096 x 65000 with 16 of 8 and 16 of 16 173, 215; 4096 x 100001 with 8 waves of 16
  // and 9 more in LDS (two workgroups a CU) and 16 of 16 285, 312; 2048 x 190000 with 16 waves of 16 and 9 282, of 12 and 9 and the end read
  // again 292, 2048 x 262144 so 437, with 8 waves 457.
  if (packs <= 64) HELD(1, 1, 0, 8, false);
  else if (packs <= 256) HELD(1, 4, 0, 8, false);
  else if (packs <= 1024) HELD(4, 4, 0, 8, false);
  else if (packs <= 2048) HELD(8, 4, 0, 8, false);
  else if (packs <= 4096) HELD(8, 8, 0, 6, false);
  else if (packs <= 8192) HELD(16, 8, 0, 8, false);
  else if (packs <= 12800) HELD(8, 16, 9, 4, false);
  else if (packs <= 25600) HELD(16, 16, 9, 4, false);
  else HELD(16, 12, 9, 4, true);
#undef HELD
}

// A per-position operand: float, as many elements as there are rows.
void check_positions(const AnyTensor* t, int64_t rows, int arg, const char* what) {
  THC_ARG_CHECK(tensor_numel(t) == rows, arg, "%ld %s for %ld rows of logits", (long)tensor_numel(t), what, (long)rows);
}

// Outputs take the tokens' sizes and are written densely; `meets`: one lies on what the call reads or within the gradient.
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
  THC_ARG_CHECK(c.logProb != c.logits && c.logProb != c.grad, policy ? 3 : 2, "the log-probabilities may not be the logits or their gradient");
  if (policy)
    THC_ARG_CHECK(c.loss != c.logits && c.loss != c.grad && c.loss != c.logProb, 2, "the losses may not be the logits, their gradient or the log-probabilities");

  Rows lr{};
  const bool direct = as_rows(c.logits, &lr);
  TensorRef logits(s, direct ? (tensor_retain(c.logits), c.logits) : tensor_new_contiguous(s, c.logits, dt));
  as_rows(logits.t, &lr);
  Dense tokens(s, c.tokens, DType::I64);
  TensorRef old(s, nullptr), advantage(s, nullptr), reference(s, nullptr), weight(s, nullptr);
  if (policy) {
    auto dense = [&](TensorRef& hold, AnyTensor* t) {
      if (t) hold.t = tensor_new_contiguous(s, t, DType::F32);
    };
    dense(old, c.old);
    dense(advantage, c.advantage);
    if (c.kl != 0) dense(reference, c.reference);
    dense(weight, c.weight);
  }
  // outputs may share a storage with each other and with what is read: all are resized before any address is taken
  tensor_resize_as(s, c.logProb, c.tokens, DType::F32);
  if (policy) tensor_resize_as(s, c.loss, c.tokens, DType::F32);
  if (c.grad) tensor_resize_as(s, c.grad, c.logits, dt);
  // Outputs on one another would be written over by each other's workgroups: dense ones are refused. Those with gaps may lie in each other's:
  // losses and log-probabilities that do are copied there behind the launches.
  auto apart = [&](const AnyTensor* x, DType xt, const AnyTensor* y, DType yt, int arg, const char* what) {
    THC_ARG_CHECK(!spans_meet(x, xt, y, yt) || !tensor_is_contiguous(x) || !tensor_is_contiguous(y), arg, "%s share memory", what);
  };
  if (policy) {
    apart(c.loss, DType::F32, c.logProb, DType::F32, 2, "the losses and the log-probabilities");
    if (c.grad) {
      apart(c.loss, DType::F32, c.grad, dt, 2, "the losses and the gradient");
      apart(c.logProb, DType::F32, c.grad, dt, 3, "the log-probabilities and the gradient");
    }
  }
  note_stream_use(s, {c.loss, c.logProb, c.grad, c.logits, c.tokens, c.old, c.advantage, c.reference, c.weight});
  PolicyArgs a{};
  a.token = tokens.data<int64_t>();
  a.evenWeight = 1.f;
  if (policy) {
    auto data = [&](const TensorRef& t) { return t.t ? (const float*)tensor_data(t.t, DType::F32) : nullptr; };
    a.old = data(old);
    a.advantage = data(advantage);
    a.reference = data(reference);
    a.weight = data(weight);
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
  logProb.t = position_output(s, c.logProb, meets(c.logProb, DType::F32, 0) || spans_meet(c.logProb, DType::F32, c.grad, dt));
  a.logProb = (float*)tensor_data(logProb.t, DType::F32);
  if (policy) {
    loss.t = position_output(s, c.loss, meets(c.loss, DType::F32, 0) || spans_meet(c.loss, DType::F32, c.grad, dt));
    a.loss = (float*)tensor_data(loss.t, DType::F32);
  }
  Rows gr{};
  if (c.grad) {
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
