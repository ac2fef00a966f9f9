// Embedding lookup and its gradient.
//
//   embedding       y[i, :] = f W[t_i, :]
//   embeddingGrad   dW[v, :] = f sum over the i with t_i = v of dY[i, :]      (or dW += that)
//
// Tokens are 1-based as all indices of this library are. A token outside the table reads nothing: its output row is NaN and its
// gradient goes nowhere. Sums are in float, in the order of the positions, and are rounded once: the same call gives the same bits.
#include <algorithm>
#include <limits>

#include "training.hpp"

namespace thc {
namespace {

// ------------------------------------------------------------------ lookup --
// One 16-byte pack of the output per item, U items in flight per lane; items are counted over (row, pack), so that short rows share a
// workgroup. Packs lie at element-aligned addresses (rows of any length), a row's last one is moved back into the row and
// repeats elements of the one before it: the same values are written twice, nothing needs a tail.
template <typename T, int V, int U, bool NT, typename I>
__global__ __launch_bounds__(kBlock) void lookup_kernel(T* __restrict__ out, const T* __restrict__ table, const int64_t* __restrict__ tokens,
                                                        int64_t vocab, int64_t tableStride, int32_t dim, I items, Divisor<I> packs, float factor) {
  using P = Pack<T, V>;
  const I base = (I)blockIdx.x * (kBlock * U) + threadIdx.x;
  I row[U];
  int32_t at[U];
  int64_t token[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const I i = base + (I)u * kBlock;
    I r;
    packs.divmod(i < items ? i : 0, row[u], r);
    at[u] = min((int32_t)r * V, dim - V);
    token[u] = tokens[row[u]] - 1;
  }
  P v[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if ((uint64_t)token[u] < (uint64_t)vocab) {
      v[u] = load_pack_unaligned<false, P>(table + token[u] * tableStride + at[u]);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) v[u].v[e] = Cvt<T>::down(__builtin_nanf(""));
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (base + (I)u * kBlock < items) {
#pragma unroll
      for (int e = 0; e < V; ++e) v[u].v[e] = rounded<T>(Cvt<T>::up(v[u].v[e]) * factor);
      store_pack_unaligned<NT>(out + (int64_t)row[u] * dim + at[u], v[u]);
    }
  }
}

template <typename T>
void launch_lookup(THCState* s, T* out, const T* table, const int64_t* tokens, int64_t count, int64_t vocab, int64_t tableStride, int64_t dim,
                   float factor) {
  hipStream_t st = current_stream(s);
  auto go = [&](auto vTag, auto uTag, auto idxTag) {
    using I = decltype(idxTag);
    constexpr int V = decltype(vTag)::value, U = decltype(uTag)::value;
    const int64_t packs = (dim + V - 1) / V, items = count * packs;
    Divisor<I> d;
    d.set((uint64_t)packs);
    const dim3 grid((unsigned)((items + kBlock * U - 1) / (kBlock * U)));
    if (streaming_store("embedding.nt", count * dim * (int64_t)sizeof(T)))
      hipLaunchKernelGGL((lookup_kernel<T, V, U, true, I>), grid, dim3(kBlock), 0, st, out, table, tokens, vocab, tableStride, (int32_t)dim,
                         (I)items, d, factor);
    else
      hipLaunchKernelGGL((lookup_kernel<T, V, U, false, I>), grid, dim3(kBlock), 0, st, out, table, tokens, vocab, tableStride, (int32_t)dim,
                         (I)items, d, factor);
  };
  constexpr int kPack = 16 / sizeof(T);
  auto width = [&](auto uTag, auto idxTag) {
    if (dim >= kPack) go(std::integral_constant<int, kPack>{}, uTag, idxTag);
    else go(std::integral_constant<int, 1>{}, uTag, idxTag);
  };
  const int64_t items = count * (dim >= kPack ? (dim + kPack - 1) / kPack : dim);
  if (force_64bit_index() || items + 4 * kBlock >= kIndex32Limit) width(std::integral_constant<int, 4>{}, uint64_t{});
  else width(std::integral_constant<int, 4>{}, uint32_t{});
}

void check_table(const AnyTensor* table, int arg) {
  THC_ARG_CHECK(table->nDimension == 2, arg, "the table must have two dims, has %d", table->nDimension);
  THC_ARG_CHECK(table->size[1] < (int64_t(1) << 30), arg, "rows of the table are too long");
}

void embedding(THCState* s, DType dt, AnyTensor* self, AnyTensor* table, AnyTensor* tokens, float factor) {
  const AnyTensor* ts[3] = {self, table, tokens};
  check_same_gpu(s, 3, ts);
  check_table(table, 3);
  THC_ARG_CHECK(tokens->nDimension < kMaxDims, 4, "%s", kDimWarning);
  THC_ARG_CHECK(self != table, 2, "the output may not be the table");
  const int64_t count = tensor_numel(tokens), dim = table->size[1];
  long size[kMaxDims];
  for (int d = 0; d < tokens->nDimension; ++d) size[d] = tokens->size[d];
  size[tokens->nDimension] = dim;
  if (count == 0) {
    tensor_resize_nd(s, self, 0, nullptr, nullptr, dt);
    return;
  }
  bool same = self->nDimension == tokens->nDimension + 1;
  for (int d = 0; same && d < self->nDimension; ++d) same = self->size[d] == size[d];
  if (!same) tensor_resize_nd(s, self, tokens->nDimension + 1, size, nullptr, dt);
  if (dim == 0) return;
  note_stream_use(s, {self, table, tokens});
  Dense at(s, tokens, DType::I64);
  // rows of the table may lie apart (a window of a wider matrix); another order of its dims is copied once
  const bool rows = table->stride[1] == 1 || dim == 1;
  TensorRef copy(s, rows ? nullptr : tensor_new_contiguous(s, table, dt));
  AnyTensor* from = rows ? table : copy.t;
  const bool direct = tensor_is_contiguous(self) && !spans_meet(self, dt, from, dt);
  TensorRef out(s, direct ? (tensor_retain(self), self) : tensor_new_with_size(s, self->nDimension, self->size, dt));
  if (dt == DType::F32)
    launch_lookup<float>(s, (float*)tensor_data(out.t, dt), (const float*)tensor_data(from, dt), at.data<int64_t>(), count, from->size[0],
                         from->stride[0], dim, factor);
  else
    launch_lookup<__half>(s, (__half*)tensor_data(out.t, dt), (const __half*)tensor_data(from, dt), at.data<int64_t>(), count, from->size[0],
                          from->stride[0], dim, factor);
  THC_CHECK(hipGetLastError());
  note_kernel("embedding");
  if (!direct) copy_tensor(s, dt, self, out.t, false);
}

// ---------------------------------------------------------------- gradient --
// Three launches:
//   group   the positions of each token side by side, in their order: slot -> position and token
//   sum     chunks of slots are summed in registers; a token whose slots lie in one chunk is done, one that crosses a chunk's
//           edge leaves a partial sum. Rows of tokens that do not occur are zeroed by other workgroups of this launch.
//   fold    the partial sums of each token that crosses edges, in the chunks' order

// Grouping. Token k (0-based) belongs to owner k mod G; every owner reads all tokens and places its own. No owner waits for another:
// it counts the tokens of the owners before it on the way, which is where its slots begin. A token's slots are side by side and
// its positions in order; the order of the tokens does not matter to the sums.
struct Grouping {
  int32_t* position;   // of each slot
  int32_t* token;      // of each slot, 0-based
  int32_t* used;       // occurrences of each token
  int32_t* total;      // slots
};
constexpr int kGroupThreads = 512, kGroupWaves = kGroupThreads / 64;
constexpr int kOwnTokens = 1024;     // tokens that one owner takes at most: 32 KiB of counts

__device__ __forceinline__ int wave_sum(int v) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) v += __shfl_xor(v, m);
  return v;
}

__global__ __launch_bounds__(kGroupThreads) void group_kernel(Grouping g, const int64_t* __restrict__ tokens, int32_t n, int64_t vocab,
                                                              int64_t padding, int shift) {
  __shared__ int counts[kGroupWaves][kOwnTokens];
  __shared__ int waveTotal[kGroupWaves], before[kGroupWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint64_t mask = (uint64_t(1) << shift) - 1, me = blockIdx.x;
  const int owned = (int)((vocab - 1 - (int64_t)me) >> shift) + 1;   // me < vocab
  for (int i = threadIdx.x; i < kGroupWaves * kOwnTokens; i += kGroupThreads) (&counts[0][0])[i] = 0;
  __syncthreads();
  // a wave takes a run of positions, 64 at a time
  const int32_t run = ((n + kGroupWaves - 1) / kGroupWaves + 63) & ~63;
  const int32_t first = min(n, wave * run), last = min(n, first + run);
  int lower = 0;
  for (int32_t i = first + lane; i < last; i += 64) {
    const uint64_t k = (uint64_t)(tokens[i] - 1);
    if (k < (uint64_t)vocab && (int64_t)k != padding - 1) {
      const uint64_t owner = k & mask;
      lower += owner < me;
      if (owner == me) atomicAdd(&counts[wave][k >> shift], 1);      // whole numbers: any order gives the same
    }
  }
  lower = wave_sum(lower);
  if (lane == 0) before[wave] = lower;
  __syncthreads();
  int start = 0;
  for (int w = 0; w < kGroupWaves; ++w) start += before[w];
  // the slots of each wave's occurrences of each token: tokens in order, each wave after the ones before it
  constexpr int kPer = kOwnTokens / kGroupThreads;
  int mine[kPer], sum = 0;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int r = threadIdx.x * kPer + j;
    mine[j] = 0;
    for (int w = 0; w < kGroupWaves; ++w) mine[j] += counts[w][r];
    sum += mine[j];
    if (r < owned) g.used[me + ((int64_t)r << shift)] = mine[j];
  }
  int upto = sum;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int o = __shfl_up(upto, d);
    if (lane >= d) upto += o;
  }
  if (lane == 63) waveTotal[wave] = upto;
  __syncthreads();
  int at = start + upto - sum;
  for (int w = 0; w < wave; ++w) at += waveTotal[w];
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    int slot = at;
    for (int w = 0; w < kGroupWaves; ++w) {
      const int c = counts[w][threadIdx.x * kPer + j];
      counts[w][threadIdx.x * kPer + j] = slot;
      slot += c;
    }
    at += mine[j];
  }
  if (me == mask && threadIdx.x == kGroupThreads - 1) *g.total = at;
  __syncthreads();
  for (int32_t i0 = first; i0 < last; i0 += 64) {
    const int32_t i = i0 + lane;
    const uint64_t k = i < last ? (uint64_t)(tokens[i] - 1) : ~uint64_t(0);
    uint64_t left = __ballot(k < (uint64_t)vocab && (int64_t)k != padding - 1 && (k & mask) == me);
    const int r = (int)(k >> shift);
    while (left) {        // the lanes that hold one token take its next slots, in order
      const int leader = __ffsll((unsigned long long)left) - 1;
      const int which = __shfl(r, leader);
      const bool same = ((left >> lane) & 1) && r == which;
      const uint64_t peers = __ballot(same);
      const int slot = counts[wave][which];
      if (same) {
        const int to = slot + __popcll(peers & ((uint64_t(1) << lane) - 1));
        g.position[to] = i;
        g.token[to] = (int32_t)k;
      }
      __builtin_amdgcn_wave_barrier();
      if (lane == leader) counts[wave][which] = slot + __popcll(peers);
      __builtin_amdgcn_wave_barrier();
      left &= ~peers;
    }
  }
}

struct GradArgs {
  Grouping g;
  float* partial;        // per chunk: of the run that began before it, of the run that goes on behind it
  int64_t outRowStride;  // of the output's gradient (elements)
  int64_t gradStride;    // of the table's gradient
  int32_t dim, chunk;    // slots a chunk
  int32_t lanes;         // that share a row
  int32_t chunks;
  float factor;
  bool add;
};

template <typename T, int V>
__device__ __forceinline__ void finish_row(T* grad, const float (&acc)[V], float factor, bool add) {
  using P = Pack<T, V>;
  P r;
  if (add) {
    const P old = load_pack_unaligned<false, P>(grad);
#pragma unroll
    for (int e = 0; e < V; ++e) r.v[e] = rounded<T>(Cvt<T>::up(old.v[e]) + acc[e] * factor);
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) r.v[e] = rounded<T>(acc[e] * factor);
  }
  store_pack_unaligned<false>(grad, r);
}

// V columns a lane (a row's last lane may be moved back when the gradient is written whole; added to, each column has one owner, so the
// odd rest is left to lanes of one column: blockIdx.y counts slabs of packs, then of single columns).
template <typename T, int V, int U>
__global__ __launch_bounds__(kBlock) void sum_kernel(GradArgs a, const T* __restrict__ out, T* __restrict__ grad, int32_t firstColumn,
                                                     int32_t columns, int64_t vocab, int32_t chunkBlocks) {
  using P = Pack<T, V>;
  const int sub = threadIdx.x / a.lanes, lane = threadIdx.x % a.lanes, subs = blockDim.x / a.lanes;
  const int32_t c0 = firstColumn + ((int32_t)blockIdx.y * a.lanes + lane) * V;
  if (c0 >= firstColumn + columns) return;
  if ((int32_t)blockIdx.x >= chunkBlocks) {     // rows of tokens that do not occur
    P zero;
#pragma unroll
    for (int e = 0; e < V; ++e) zero.v[e] = Cvt<T>::down(0.f);
    const int64_t row0 = (int64_t)(blockIdx.x - chunkBlocks) * (subs * 16) + sub;
    for (int j = 0; j < 16; ++j) {
      const int64_t row = row0 + (int64_t)j * subs;
      if (row < vocab && a.g.used[row] == 0) store_pack_unaligned<false>(grad + row * a.gradStride + c0, zero);
    }
    return;
  }
  const int32_t c = (int32_t)blockIdx.x * subs + sub;
  const int32_t total = *a.g.total;
  const int32_t s0 = c * a.chunk, s1 = min(total, s0 + a.chunk);
  if (s0 >= s1) return;
  const int32_t previous = s0 > 0 ? a.g.token[s0 - 1] : -1, next = s1 < total ? a.g.token[s1] : -1;
  float acc[V];
#pragma unroll
  for (int e = 0; e < V; ++e) acc[e] = 0.f;
  int32_t token = a.g.token[s0];
  bool here = token != previous;       // the run began in this chunk
  float* part = a.partial + (int64_t)c * 2 * a.dim + c0;
  for (int32_t s = s0; s < s1; s += U) {
    int32_t at[U], tok[U];
    P v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int32_t q = min(s + u, s1 - 1);
      at[u] = a.g.position[q];
      tok[u] = a.g.token[q];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = load_pack_unaligned<true, P>(out + (int64_t)at[u] * a.outRowStride + c0);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (s + u < s1) {
        if (tok[u] != token) {
          if (here) {
            finish_row<T, V>(grad + (int64_t)token * a.gradStride + c0, acc, a.factor, a.add);
          } else {
#pragma unroll
            for (int e = 0; e < V; ++e) part[e] = acc[e];
          }
          token = tok[u];
          here = true;
#pragma unroll
          for (int e = 0; e < V; ++e) acc[e] = 0.f;
        }
#pragma unroll
        for (int e = 0; e < V; ++e) acc[e] += Cvt<T>::up(v[u].v[e]);
      }
    }
  }
  if (here && token != next) {
    finish_row<T, V>(grad + (int64_t)token * a.gradStride + c0, acc, a.factor, a.add);
  } else {
    if (here) part += a.dim;
#pragma unroll
    for (int e = 0; e < V; ++e) part[e] = acc[e];
  }
}

// The token whose run begins in chunk c and goes on behind it: its partial sums, chunk by chunk.
template <typename T>
__global__ __launch_bounds__(kBlock) void fold_kernel(GradArgs a, T* __restrict__ grad) {
  const int32_t c = blockIdx.x, total = *a.g.total;
  const int32_t s0 = c * a.chunk, s1 = s0 + a.chunk;
  if (s1 >= total) return;
  const int32_t token = a.g.token[s1];
  if (a.g.token[s1 - 1] != token) return;
  if (a.g.token[s0] == token && s0 > 0 && a.g.token[s0 - 1] == token) return;    // began before
  const int32_t column = (int32_t)blockIdx.y * kBlock + threadIdx.x;
  if (column >= a.dim) return;
  float acc[1] = {a.partial[((int64_t)c * 2 + 1) * a.dim + column]};
  for (int32_t d = c + 1;; ++d) {
    acc[0] += a.partial[(int64_t)d * 2 * a.dim + column];
    const int64_t behind = (int64_t)(d + 1) * a.chunk;
    if (behind >= total || a.g.token[behind] != token) break;
  }
  finish_row<T, 1>(grad + (int64_t)token * a.gradStride + column, acc, a.factor, a.add);
}

template <typename T>
void launch_grad(THCState* s, T* grad, int64_t vocab, int64_t gradStride, const int64_t* tokens, int32_t n, const T* out, int64_t outStride,
                 int32_t dim, float factor, int64_t padding, bool add) {
  hipStream_t st = current_stream(s);
  constexpr int kPack = 16 / sizeof(T);
  GradArgs a{};
  a.dim = dim;
  a.chunk = 16;
  a.outRowStride = outStride;
  a.gradStride = gradStride;
  a.factor = factor;
  a.add = add;
  a.chunks = (n + a.chunk - 1) / a.chunk;
  // owners: a power of two, none of which has more tokens than it has room to count
  int shift = 0;
  while ((int64_t(1) << shift) < std::min<int64_t>(vocab, 256) || ((vocab - 1) >> shift) + 1 > kOwnTokens) ++shift;
  while ((int64_t(1) << shift) > vocab) --shift;
  const int64_t slots = (n + 3) & ~3, words = (vocab + 3) & ~int64_t(3);
  Workspace w(s, (slots * 2 + words + 4) * 4 + (int64_t)a.chunks * 2 * dim * 4);
  a.g.position = reinterpret_cast<int32_t*>(w.data());
  a.g.token = a.g.position + slots;
  a.g.used = a.g.token + slots;
  a.g.total = a.g.used + words;
  a.partial = reinterpret_cast<float*>(a.g.total + 4);
  hipLaunchKernelGGL(group_kernel, dim3(1u << shift), dim3(kGroupThreads), 0, st, a.g, tokens, n, vocab, padding, shift);
  auto sum = [&](auto vTag, int32_t first, int32_t columns) {
    constexpr int V = decltype(vTag)::value;
    if (columns <= 0) return;
    const int32_t packs = columns / V;
    int lanes = 1;
    while (lanes < 64 && lanes < packs) lanes *= 2;
    if (packs > 64) lanes = std::min(kBlock, (packs + 63) / 64 * 64);
    a.lanes = lanes;
    const int subs = std::max(1, kBlock / lanes);
    const int32_t chunkBlocks = (a.chunks + subs - 1) / subs;
    const int64_t zeroBlocks = add ? 0 : (vocab + subs * 16 - 1) / (subs * 16);
    hipLaunchKernelGGL((sum_kernel<T, V, 8>), dim3((unsigned)(chunkBlocks + zeroBlocks), (packs + lanes - 1) / lanes), dim3(subs * lanes), 0, st,
                       a, out, grad, first, columns, vocab, chunkBlocks);
  };
  const int32_t whole = dim / kPack * kPack;
  sum(std::integral_constant<int, kPack>{}, 0, whole);
  sum(std::integral_constant<int, 1>{}, whole, dim - whole);
  hipLaunchKernelGGL((fold_kernel<T>), dim3(a.chunks, (dim + kBlock - 1) / kBlock), dim3(kBlock), 0, st, a, grad);
}

void embedding_grad(THCState* s, DType dt, AnyTensor* grad, AnyTensor* tokens, AnyTensor* out, float factor, long padding, int accumulate) {
  const AnyTensor* ts[3] = {grad, tokens, out};
  check_same_gpu(s, 3, ts);
  check_table(grad, 2);
  THC_ARG_CHECK(!overlapping(tensor_layout(grad)), 2, "elements of the gradient overlap");
  const int64_t count = tensor_numel(tokens), vocab = grad->size[0], dim = grad->size[1];
  THC_ARG_CHECK(tensor_numel(out) == count * dim, 4, "%ld elements of the output's gradient for %ld tokens of %ld",
                (long)tensor_numel(out), (long)count, (long)dim);
  THC_ARG_CHECK(count <= int64_t(1) << 30, 3, "too many tokens");
  THC_ARG_CHECK(vocab < kIndex32Limit, 2, "the table has too many rows");
  THC_ARG_CHECK(padding >= 0 && padding <= vocab, 6, "the padding token is outside the table");
  if (count == 0) {
    if (!accumulate && !pointwise_apply(s, dt, PointOp::Fill, 0.f, grad, nullptr, nullptr, nullptr)) raise_arg_error(2, "%s", kDimWarning);
    return;
  }
  note_stream_use(s, {grad, tokens, out});
  Dense at(s, tokens, DType::I64);
  // rows of the output's gradient one stride apart, and of the table's; anything else goes through a dense copy
  Rows r{};
  const bool rows = as_rows(out, &r) && r.length == dim && r.inner == r.count;
  TensorRef copy(s, rows ? nullptr : tensor_new_contiguous(s, out, dt));
  const bool direct = (grad->stride[1] == 1 || dim == 1) && !spans_meet(grad, dt, out, dt);
  TensorRef to(s, direct ? (tensor_retain(grad), grad) : accumulate ? tensor_new_clone(s, grad, dt) : tensor_new_with_size(s, 2, grad->size, dt));
  const void* from = tensor_data(rows ? out : copy.t, dt);
  const int64_t stride = rows ? r.stride : dim;
  if (dt == DType::F32)
    launch_grad<float>(s, (float*)tensor_data(to.t, dt), vocab, to.t->stride[0], at.data<int64_t>(), (int32_t)count, (const float*)from, stride,
                       (int32_t)dim, factor, padding, accumulate != 0);
  else
    launch_grad<__half>(s, (__half*)tensor_data(to.t, dt), vocab, to.t->stride[0], at.data<int64_t>(), (int32_t)count, (const __half*)from, stride,
                        (int32_t)dim, factor, padding, accumulate != 0);
  THC_CHECK(hipGetLastError());
  note_kernel("embedding-grad");
  if (!direct) copy_tensor(s, dt, grad, to.t, false);
}

}  // namespace
}  // namespace thc

#define TN(x) reinterpret_cast<thc::AnyTensor*>(x)
THC_API void THCudaTensor_embedding(THCState* s, THCudaTensor* self, THCudaTensor* weight, THCudaLongTensor* tokens, float scale) {
  THC_GUARD_ALL(thc::embedding(s, thc::DType::F32, TN(self), TN(weight), TN(tokens), scale))
}
THC_API void THCudaHalfTensor_embedding(THCState* s, THCudaHalfTensor* self, THCudaHalfTensor* weight, THCudaLongTensor* tokens, float scale) {
  THC_GUARD_ALL(thc::embedding(s, thc::DType::F16, TN(self), TN(weight), TN(tokens), scale))
}
THC_API void THCudaTensor_embeddingGrad(THCState* s, THCudaTensor* gradWeight, THCudaLongTensor* tokens, THCudaTensor* gradOutput, float scale,
                                        long padding, int accumulate) {
  THC_GUARD_ALL(thc::embedding_grad(s, thc::DType::F32, TN(gradWeight), TN(tokens), TN(gradOutput), scale, padding, accumulate))
}
THC_API void THCudaHalfTensor_embeddingGrad(THCState* s, THCudaHalfTensor* gradWeight, THCudaLongTensor* tokens, THCudaHalfTensor* gradOutput,
                                            float scale, long padding, int accumulate) {
  THC_GUARD_ALL(thc::embedding_grad(s, thc::DType::F16, TN(gradWeight), TN(tokens), TN(gradOutput), scale, padding, accumulate))
}
