// Embedding lookup and its gradient.
//
//   embedding       y[i, :] = f W[t_i, :]
//   embeddingGrad   dW[v, :] = f sum over the i with t_i = v of dY[i, :]      (or dW += that)
//
// Tokens are 1-based as all indices of this library are. A token outside the table reads nothing: its output row is NaN and its
// gradient goes nowhere. Sums are in float and in an order that the sizes and tokens alone decide; the product with f and what it is
// added to round in float, the result once more to its type.
#include <algorithm>

#include "training.hpp"

namespace thc {
namespace {

// ------------------------------------------------------------------ lookup --
// One 16-byte pack of the output per item, U items in flight per lane; items are counted over (row, pack), so that short rows share a
// workgroup. Packs lie at element-aligned addresses (rows of any length), a row's last one is moved back into the row and
// repeats elements of the one before it: the same values are written twice, nothing needs a tail. Stores are streaming ones at every
// size (us with plain ones and so: 2048 rows of 2048 halves 4.9, 4.8, 8192 x 1024 6.5, 5.5, 65536 x 1024 43.5, 29.0); table rows may
// come again and are read plainly. Bound by memory: 16392 x 2048 halves out of 32000 rows, as even as words in a text, 16.3 us, 5.5 TB/s of
// rows written and distinct rows read; 16 rows take 3.3 us, a launch.
template <typename T, int V, int U>
__global__ __launch_bounds__(kBlock) void lookup_kernel(T* __restrict__ out, const T* __restrict__ table, const int64_t* __restrict__ tokens,
                                                        int64_t vocab, int64_t tableStride, int32_t dim, uint32_t items,
                                                        Divisor<uint32_t> packs, float factor) {
  using P = Pack<T, V>;
  const uint32_t base = blockIdx.x * (kBlock * U) + threadIdx.x;
  uint32_t row[U];
  int32_t at[U];
  int64_t token[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t i = base + u * kBlock;
    uint32_t r;
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
    if (base + u * kBlock < items) {
#pragma unroll
      for (int e = 0; e < V; ++e) v[u].v[e] = rounded<T>(Cvt<T>::up(v[u].v[e]) * factor);
      store_pack_unaligned<true>(out + (int64_t)row[u] * dim + at[u], v[u]);
    }
  }
}

template <typename T>
void launch_lookup(THCState* s, T* out, const T* table, const int64_t* tokens, int64_t count, int64_t vocab, int64_t tableStride, int64_t dim,
                   float factor) {
  constexpr int kPack = 16 / sizeof(T), U = 4;
  const int V = dim >= kPack ? kPack : 1;
  const int64_t packs = (dim + V - 1) / V;
  Divisor<uint32_t> d;
  d.set((uint64_t)packs);
  // rows by the 2^30 items: a launch counts them in 32 bits
  const int64_t most = std::max<int64_t>(1, tuning("embedding.items", 1 << 30) / packs);
  for (int64_t first = 0; first < count; first += most) {
    const uint32_t items = (uint32_t)(std::min(most, count - first) * packs);
    const dim3 grid((items + kBlock * U - 1) / (kBlock * U));
    if (V == 1)
      hipLaunchKernelGGL((lookup_kernel<T, 1, U>), grid, dim3(kBlock), 0, current_stream(s), out + first * dim, table, tokens + first, vocab,
                         tableStride, (int32_t)dim, items, d, factor);
    else
      hipLaunchKernelGGL((lookup_kernel<T, kPack, U>), grid, dim3(kBlock), 0, current_stream(s), out + first * dim, table, tokens + first,
                         vocab, tableStride, (int32_t)dim, items, d, factor);
  }
}

void check_table(const AnyTensor* table, int arg) {
  THC_ARG_CHECK(table->nDimension == 2, arg, "the table must have two dims, has %d", table->nDimension);
  THC_ARG_CHECK(table->size[1] <= (int64_t(1) << 23), arg, "rows of the table are too long");      // (256 columns a workgroup along a grid's y)
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
//   fold    the partial sums of each token that crosses edges

// Grouping. Token k (0-based) belongs to owner k mod G. An owner sweeps the tokens twice, counts its own and places them; the tokens of
// the owners before it, which it counts on the way, say where its slots begin: no owner waits for another. A token's slots are side
// by side and its positions in order; the order of the tokens does not matter to the sums.
// Bound by latency, sweep by sweep, and by how often the commonest token is counted: 1500 positions 5.6 us, 32768 12.3, 131072 split 18 behind
// the splitting's 5.
// Few positions are swept as they are, by every owner. Of many, each owner would look at all: they are first split, tile by tile, into
// the owners' shares.
struct Grouping {
  int32_t* position;   // of each slot
  int32_t* token;      // of each slot, 0-based
  int32_t* used;       // occurrences of each token
  int32_t* total;      // slots
};
constexpr int kGroupThreads = 1024, kGroupWaves = kGroupThreads / 64;
constexpr int kOwnTokens = 512;      // tokens that one owner takes at most: 32 KiB of counts
constexpr int kFound = 896;          // positions that a wave remembers between its two sweeps: 112 KiB
constexpr int kTile = 1024;          // positions that are split together, one a lane
// Splitting costs a launch and saves every owner the sight of the others' positions. us of the whole gradient, swept and split (rows of 64 halves,
// added): 8192 positions 18.3, 21.6; 30000 26.4, 26.4; 40000 30.6, 29.3; 65536 36.6, 31.9; 131072 139, 51. Tiles of 4096 positions instead of
// 1024 took 4 us more at 65536.
constexpr int kSplitFrom = 40000;
constexpr int kMostSplit = 1024;     // owners that they are split between
constexpr int kAhead = 8;            // loads in flight

__device__ __forceinline__ int wave_sum(int v) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) v += __shfl_xor(v, m);
  return v;
}

// The lanes among those with `valid` that hold what this one holds, of `bits` bits: found bit by bit.
__device__ __forceinline__ uint64_t equal_lanes(uint32_t what, int bits, bool valid) {
  uint64_t peers = __ballot(valid);
  for (int b = 0; b < bits; ++b) {
    const bool one = (what >> b) & 1;
    const uint64_t set = __ballot(one);
    peers &= one ? set : ~set;
  }
  return peers;
}

// Calls f(position, token, whether it is one of the table's and not padding) for positions [first, last), 64 side by side and in order.
// Tokens are 0-based here and have 32 bits once their upper half has been looked at.
template <typename F>
__device__ __forceinline__ void each_token(const int64_t* __restrict__ tokens, int32_t first, int32_t last, uint32_t vocab, uint32_t padding,
                                           const F& f) {
  const int lane = threadIdx.x & 63;
  for (int32_t i0 = first; i0 < last; i0 += 64 * kAhead) {
    uint64_t k[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) k[u] = (uint64_t)tokens[min(i0 + u * 64 + lane, last - 1)];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int32_t i = i0 + u * 64 + lane;
      const uint32_t token = (uint32_t)k[u] - 1;
      f(i, token, (k[u] >> 32) == 0 && token < vocab && token != padding && i < last);
    }
  }
}

// A tile's positions by owner, in order within each: entries (position, token) and where each owner's begin; padding and tokens outside
// the table are left out.
struct Split {
  int2* entry;        // kTile per tile
  int32_t* begin;     // owners + 1 per tile
};
__global__ __launch_bounds__(kGroupThreads) void split_kernel(Split to, const int64_t* __restrict__ tokens, int32_t n, uint32_t vocab,
                                                              uint32_t padding, int shift) {
  constexpr int kPer = kTile / kGroupThreads;
  __shared__ int counts[kGroupWaves][kMostSplit];
  __shared__ int waveTotal[kGroupWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, owners = 1 << shift;
  const uint64_t below = (uint64_t(1) << lane) - 1;
  const uint32_t mask = (uint32_t)owners - 1;
  const int32_t first = (int32_t)blockIdx.x * kTile + wave * (64 * kPer) + lane;
  uint64_t k[kPer];
#pragma unroll
  for (int u = 0; u < kPer; ++u) k[u] = (uint64_t)tokens[min(first + u * 64, n - 1)];
  for (int b = lane; b < owners; b += 64) counts[wave][b] = 0;       // (each wave its own)
  int rank[kPer];
  bool valid[kPer];
#pragma unroll
  for (int u = 0; u < kPer; ++u) {
    const uint32_t token = (uint32_t)k[u] - 1, owner = token & mask;
    valid[u] = (k[u] >> 32) == 0 && token < vocab && token != padding && first + u * 64 < n;
    const uint64_t peers = equal_lanes(owner, shift, valid[u]);
    if (valid[u]) {
      const int at = counts[wave][owner];
      rank[u] = at + __popcll(peers & below);
      __builtin_amdgcn_wave_barrier();
      if ((peers & below) == 0) counts[wave][owner] = at + __popcll(peers);
    }
    __builtin_amdgcn_wave_barrier();
  }
  __syncthreads();
  // owners in order, a thread each; each wave's after those of the ones before it
  const int b = threadIdx.x;
  int count[kGroupWaves], sum = 0;
  if (b < owners) {
#pragma unroll
    for (int w = 0; w < kGroupWaves; ++w) {
      count[w] = counts[w][b];
      sum += count[w];
    }
  }
  int upto = sum;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int o = __shfl_up(upto, d);
    if (lane >= d) upto += o;
  }
  if (lane == 63) waveTotal[wave] = upto;
  __syncthreads();
  int at = upto - sum;
  for (int w = 0; w < wave; ++w) at += waveTotal[w];
  int32_t* begin = to.begin + (int64_t)blockIdx.x * (owners + 1);
  if (b < owners) {
    begin[b] = at;
#pragma unroll
    for (int w = 0; w < kGroupWaves; ++w) {
      counts[w][b] = at;
      at += count[w];
    }
    if (b == owners - 1) begin[owners] = at;
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < kPer; ++u) {
    const uint32_t token = (uint32_t)k[u] - 1;
    if (valid[u]) to.entry[(int64_t)blockIdx.x * kTile + counts[wave][token & mask] + rank[u]] = int2{first + u * 64, (int)token};
  }
}

template <bool SPLIT>
__global__ __launch_bounds__(kGroupThreads) void group_kernel(Grouping g, Split split, const int64_t* __restrict__ tokens, int32_t n, uint32_t vocab,
                                                              uint32_t padding, int shift) {
  __shared__ int counts[kGroupWaves][kOwnTokens];
  __shared__ int2 found[kGroupWaves][kFound];
  __shared__ int waveTotal[kGroupWaves], before[kGroupWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint64_t below = (uint64_t(1) << lane) - 1;
  const uint32_t mask = (1u << shift) - 1, me = blockIdx.x;
  const int owned = (int)((vocab - 1 - me) >> shift) + 1;            // me < vocab
  for (int r = lane; r < owned; r += 64) counts[wave][r] = 0;        // (each wave its own)
  int lower = 0, mine = 0;
  // The owner's positions, in order: f(position, token, whether it is the owner's). A wave takes a run of positions, or of tiles.
  auto sweep = [&](const auto& f) {
    if constexpr (SPLIT) {
      // its shares of a few tiles are asked for together: where they lie, then the first 128 entries of each
      constexpr int U = kAhead / 2;
      const int tiles = (n + kTile - 1) / kTile, run = (tiles + kGroupWaves - 1) / kGroupWaves;
      const int last = min(tiles, (wave + 1) * run);
      for (int t0 = wave * run; t0 < last; t0 += U) {
        const int32_t* begin = split.begin + (int64_t)min(t0 + (lane >> 1), last - 1) * (mask + 2) + me + (lane & 1);
        const int bound = lane < 2 * U ? *begin : 0;
        int from[U], to[U];
        int2 e[U], more[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          from[u] = __builtin_amdgcn_readlane(bound, 2 * u);
          to[u] = t0 + u < last ? __builtin_amdgcn_readlane(bound, 2 * u + 1) : from[u];
          const int2* entry = split.entry + (int64_t)(t0 + u) * kTile + from[u] + lane;
          if (from[u] + lane < to[u]) e[u] = entry[0];
          if (from[u] + 64 + lane < to[u]) more[u] = entry[64];
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (from[u] < to[u]) f(e[u].x, (uint32_t)e[u].y, from[u] + lane < to[u]);
          if (from[u] + 64 < to[u]) f(more[u].x, (uint32_t)more[u].y, from[u] + 64 + lane < to[u]);
          for (int j = from[u] + 128; j < to[u]; j += 64) {
            const int2 rest = split.entry[(int64_t)(t0 + u) * kTile + min(j + lane, to[u] - 1)];
            f(rest.x, (uint32_t)rest.y, j + lane < to[u]);
          }
        }
      }
    } else {
      const int32_t run = ((n + kGroupWaves - 1) / kGroupWaves + 63) & ~63;
      const int32_t first = min(n, wave * run), last = min(n, first + run);
      each_token(tokens, first, last, vocab, padding, [&](int32_t i, uint32_t token, bool valid) {
        const uint32_t owner = valid ? token & mask : ~0u;
        lower += owner < me;
        f(i, token, owner == me);
      });
    }
  };
  if constexpr (SPLIT) {       // a tile's share begins behind the owners before this one
    const int tiles = (n + kTile - 1) / kTile;
    for (int t = threadIdx.x; t < tiles; t += kGroupThreads) lower += split.begin[(int64_t)t * (mask + 2) + me];
  }
  sweep([&](int32_t i, uint32_t token, bool own) {
    const uint64_t all = __ballot(own);
    if (all) {
      if (own) {
        atomicAdd(&counts[wave][token >> shift], 1);      // whole numbers: any order gives the same
        const int to = mine + __popcll(all & below);
        if (to < kFound) found[wave][to] = int2{i, (int)(token >> shift)};
      }
      mine += __popcll(all);
    }
  });
  lower = wave_sum(lower);
  if (lane == 0) before[wave] = lower;
  __syncthreads();
  int start = 0;
#pragma unroll
  for (int w = 0; w < kGroupWaves; ++w) start += before[w];
  // the slots of each wave's occurrences of each token: tokens in order, a thread each, each wave's after those of the ones before it
  const int r = threadIdx.x;
  int count[kGroupWaves], sum = 0;
  if (r < owned) {
#pragma unroll
    for (int w = 0; w < kGroupWaves; ++w) {
      count[w] = counts[w][r];
      sum += count[w];
    }
    g.used[me + ((uint32_t)r << shift)] = sum;
  }
  int upto = sum;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int o = __shfl_up(upto, d);
    if (lane >= d) upto += o;
  }
  if (lane == 63) waveTotal[wave] = upto;
  __syncthreads();
  int slot = start + upto - sum;
  for (int w = 0; w < wave; ++w) slot += waveTotal[w];
  if (r < owned) {
#pragma unroll
    for (int w = 0; w < kGroupWaves; ++w) {
      counts[w][r] = slot;
      slot += count[w];
    }
  }
  if (me == mask && threadIdx.x == kGroupThreads - 1) *g.total = slot;
  __syncthreads();
  // up to 64 occurrences, in order: the lanes that hold one token take its next slots
  const int bits = owned > 1 ? 32 - __clz(owned - 1) : 0;
  auto place = [&](int32_t position, int which, bool own) {
    if (!__ballot(own)) return;
    const uint64_t peers = equal_lanes(which, bits, own);
    if (own) {
      const int at = counts[wave][which], to = at + __popcll(peers & below);
      g.position[to] = position;
      g.token[to] = (int32_t)(me + ((uint32_t)which << shift));
      __builtin_amdgcn_wave_barrier();
      if ((peers & below) == 0) counts[wave][which] = at + __popcll(peers);
    }
    __builtin_amdgcn_wave_barrier();
  };
  if (mine <= kFound) {
    for (int i = lane; i - lane < mine; i += 64) {
      const int2 f = found[wave][min(i, mine - 1)];
      place(f.x, f.y, i < mine);
    }
  } else {      // a common token's owner: its positions again
    sweep([&](int32_t i, uint32_t token, bool own) { place(i, (int)(token >> shift), own); });
  }
}

struct GradArgs {
  Grouping g;
  float* partial;        // two rows per chunk: of the run that began before it, of the run that goes on behind it
  int64_t outRowStride;  // of the output's gradient (elements)
  int64_t gradStride;    // of the table's gradient
  int32_t dim, partialStride, chunk;    // chunk: its slots
  int32_t lanes;         // that share a row
  int32_t chunks;
  uint32_t zeroShares;   // workgroups for 64 rows; 0: a team for a row
  float factor;
  bool add;
};

// The sums of V columns into the table's gradient, which held `old`, but for the first `skip` of them (another lane's) and those from `end` on.
template <typename T, int V>
__device__ __forceinline__ void finish_row(T* grad, const Pack<T, V>& old, const float (&acc)[V], float factor, bool add, int skip, int end = V) {
  Pack<T, V> r;
#pragma unroll
  for (int e = 0; e < V; ++e) r.v[e] = rounded<T>((add ? Cvt<T>::up(old.v[e]) : 0.f) + acc[e] * factor);
  if (skip == 0 && end >= V) {
    store_pack_unaligned<false>(grad, r);
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (e >= skip && e < end) grad[e] = r.v[e];
  }
}
template <typename T, int V>
__device__ __forceinline__ void finish_row(T* grad, const float (&acc)[V], float factor, bool add, int skip, int end = V) {
  Pack<T, V> old;
  if (add) {
    if (end >= V) {
      old = load_pack_unaligned<false, Pack<T, V>>(grad);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (e < end) old.v[e] = grad[e];
    }
  }
  finish_row<T, V>(grad, old, acc, factor, add, skip, end);
}
template <int V>
__device__ __forceinline__ void write_partial(float* to, const float (&acc)[V]) {
  if constexpr (V % 4 == 0) {
#pragma unroll
    for (int e = 0; e < V; e += 4) store_pack_unaligned<false>(to + e, Pack<float, 4>{{acc[e], acc[e + 1], acc[e + 2], acc[e + 3]}});
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) to[e] = acc[e];
  }
}

// Workgroups that share 64 rows: as many as leave each about 32 KiB. The workgroups above each other along a grid's y take shares, too.
template <typename T>
int32_t zero_shares(int64_t dim, int64_t slabs) {
  return (int32_t)std::max<int64_t>(1, std::min<int64_t>(64, 64 * dim * (int64_t)sizeof(T) >> 15) / slabs);
}
__device__ __forceinline__ uint64_t share_of_rows(uint32_t share, uint32_t shares) {
  const uint32_t i = share * gridDim.y + blockIdx.y, n = shares * gridDim.y, from = 64 * i / n, to = 64 * (i + 1) / n;
  return from < to ? ~uint64_t(0) >> (64 - (to - from)) << from : 0;
}

// Zeros to the rows row0 + (the bits of `rows`) by a workgroup: rows side by side are one piece of memory, whose 16-byte packs are
// counted from a 128-byte line's begin, so that a wave writes whole lines whatever the rows' length. us, pack by pack of each row and so: 1 x 7309 floats into 28416 rows 264, 164,
// 112 x 5055 into 22959 146, 95, 3000 x 3000 into 50000 157, 147 (at a copy's rate 136, 77, 104).
template <bool NT, typename T>
__device__ __forceinline__ void zero_rows(T* grad, int64_t stride, int32_t dim, int64_t row0, uint64_t rows) {
  constexpr int V = 16 / sizeof(T), kLine = 128 / 16;
  Pack<T, V> zero;
#pragma unroll
  for (int e = 0; e < V; ++e) zero.v[e] = Cvt<T>::down(0.f);
  while (rows) {
    const int first = __ffsll((unsigned long long)rows) - 1;
    const uint64_t from = rows >> first;
    const int count = stride != dim ? 1 : ~from ? __ffsll((unsigned long long)~from) - 1 : 64;
    rows &= count == 64 ? 0 : ~(((uint64_t(1) << count) - 1) << first);
    T* begin = grad + (row0 + first) * stride;
    const int64_t n = (int64_t)count * dim;
    const int head = (int)min(n, (int64_t)((16 - ((uintptr_t)begin & 15)) & 15) / (int64_t)sizeof(T));
    const int64_t packs = (n - head) / V;
    const int tail = (int)(n - head - packs * V), t = threadIdx.x;
    if (t < head) begin[t] = zero.v[0];
    if (t < tail) begin[head + packs * V + t] = zero.v[0];
    T* body = begin + head;
    for (int64_t k = t - (int)(((uintptr_t)body >> 4) & (kLine - 1)); k < packs; k += blockDim.x)
      if (k >= 0) store_pack_unaligned<NT>(body + k * V, zero);
  }
}

// V columns a lane; a row's last lane is moved back into the row and leaves the columns that it shares to the lane before it. Bound by
// memory: 32768 x 2048 halves into 50000 rows 60 us, 5.7 TB/s of rows read and written, besides the partial sums, which stay in the caches. (A run
// that crosses one edge summed to its end by the chunk that it begins in: 1.5 us less to fold, but 9 more here; the few chunks that go on
// are the launch's end. What sums are added to, asked for together with the rows: the same, for the registers.)
template <typename T, int V, int U, bool NT>
__global__ __launch_bounds__(kBlock) void sum_kernel(GradArgs a, const T* __restrict__ out, T* __restrict__ grad, int64_t vocab,
                                                     int32_t chunkBlocks) {
  using P = Pack<T, V>;
  const int sub = threadIdx.x / a.lanes, lane = threadIdx.x % a.lanes, subs = blockDim.x / a.lanes;
  const int32_t column = ((int32_t)blockIdx.y * a.lanes + lane) * V;
  if ((int32_t)blockIdx.x >= chunkBlocks) {
    const uint32_t block = blockIdx.x - chunkBlocks;
    if (a.zeroShares > 0) {
      const int64_t row0 = (int64_t)(block / a.zeroShares) * 64, row = row0 + (threadIdx.x & 63);
      const uint64_t unused = __ballot(row < vocab && a.g.used[row] == 0);
      zero_rows<NT>(grad, a.gradStride, a.dim, row0, unused & share_of_rows(block % a.zeroShares, a.zeroShares));
      return;
    }
    // short rows: a team each, 16 one after another, whose tokens' numbers are asked for together
    P zero;
#pragma unroll
    for (int e = 0; e < V; ++e) zero.v[e] = Cvt<T>::down(0.f);
    const int64_t row0 = (int64_t)block * (subs * 16) + sub;
    int32_t used[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) used[j] = a.g.used[min(row0 + (int64_t)j * subs, vocab - 1)];
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const int64_t row = row0 + (int64_t)j * subs;
      if (column < a.dim && row < vocab && used[j] == 0) store_pack_unaligned<false>(grad + row * a.gradStride + min(column, a.dim - V), zero);
    }
    return;
  }
  if (column >= a.dim) return;
  const int32_t c0 = min(column, a.dim - V);
  const int skip = column - c0;
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
  float* part = a.partial + (int64_t)c * 2 * a.partialStride + c0;
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
          if (here) finish_row<T, V>(grad + (int64_t)token * a.gradStride + c0, acc, a.factor, a.add, skip);
          else write_partial(part, acc);
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
  if (here && token != next) finish_row<T, V>(grad + (int64_t)token * a.gradStride + c0, acc, a.factor, a.add, skip);
  else write_partial(here ? part + a.partialStride : part, acc);
}

// The partial sums of the runs that cross edges, by the first edge that they cross. A workgroup looks at 64 edges, a lane each, and has a strip of
// columns, four a lane: a run of few partial sums is a team of lanes', of more a wave's, and of many all waves', whose sums meet in LDS.
// Bound by latency, load by load: 8192 x 1024 halves 5.0 us, 32768 x 2048 6.5 (a workgroup for every edge, most of which have none: 8.7, 6.9; where
// all tokens are the same, the whole gradient of 32768 x 256 219 us instead of 87).
constexpr int kFoldWaves = 8, kFoldGrid = 512;
constexpr int kTeamFold = 8, kWaveFold = 32;      // partial sums that a team, and that a wave's teams each, take
template <typename T>
__global__ __launch_bounds__(kFoldWaves * 64) void fold_kernel(GradArgs a, T* __restrict__ grad, int32_t n, int lanes) {
  constexpr int W = kFoldWaves, U = 8;
  using P = Pack<float, 4>;
  __shared__ float meet[W][4][64];
  __shared__ int32_t runFirst[64], runLast[64], runToken[64];
  __shared__ int number[3];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int subs = 64 / lanes, sub = lane / lanes, team = wave * subs + sub, teams = W * subs;
  if (wave == 0) {
    const int32_t total = *a.g.total;
    const int64_t edge = (int64_t)blockIdx.x * 64 + lane, at = (edge + 1) * a.chunk;
    // (slots behind the last one have room, but nothing in it)
    const auto token_at = [&](int64_t s) {
      const int32_t token = a.g.token[min(max(s, int64_t(0)), (int64_t)n - 1)];
      return s >= 0 && s < total ? token : -1;
    };
    const int32_t token = token_at(at), ahead = token_at(at - 1), begin = token_at(at - a.chunk), before = token_at(at - a.chunk - 1);
    const int32_t behind = token_at(at + a.chunk);
    const bool crosses = token >= 0 && ahead == token, starts = crosses && !(begin == token && before == token);
    const uint64_t goesOn = __ballot(crosses && behind == token), over = ~goesOn >> lane;
    int32_t last = (int32_t)edge + 1;
    if (over) last += __ffsll((unsigned long long)over) - 1;
    if (starts && !over) {
      // the run that crosses the last of them goes on: it begins in this chunk, so its length says where it ends but for one chunk
      last = (int32_t)edge + (a.g.used[token] - 1) / a.chunk;
      if (token_at(((int64_t)last + 1) * a.chunk) == token) ++last;
    }
    // those of teams, of waves and of all, one list behind the other
    const int parts = last - (int32_t)edge + 1, kind = parts <= kTeamFold ? 0 : parts <= kWaveFold * subs ? 1 : 2;
    int behindOthers = 0;
#pragma unroll
    for (int j = 0; j < 3; ++j) {
      const uint64_t all = __ballot(starts && kind == j);
      if (starts && kind == j) {
        const int i = behindOthers + __popcll(all & ((uint64_t(1) << lane) - 1));
        runFirst[i] = (int32_t)edge;
        runLast[i] = last;
        runToken[i] = token;
      }
      behindOthers += __popcll(all);
      if (lane == 0) number[j] = behindOthers;
    }
  }
  __syncthreads();
  const int ofTeams = number[0], ofWaves = number[1], runs = number[2];
  const int32_t column = ((int32_t)blockIdx.y * lanes + lane % lanes) * 4;
  const bool active = column < a.dim;
  // chunk `first` has its share in its second row, those behind it in their first; chunks j, j + step, ... to `last`
  auto add_parts = [&](float(&acc)[4], int32_t first, int32_t j, int32_t step, int32_t last) {
    for (; j <= last; j += U * step) {
      P v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int32_t q = j + u * step;
        if (q <= last) v[u] = *reinterpret_cast<const P*>(a.partial + ((int64_t)q * 2 + (q == first)) * a.partialStride + column);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (j + u * step <= last) {
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[e] += v[u].v[e];
        }
      }
    }
  };
  auto finish = [&](int i, const float(&acc)[4]) {
    finish_row<T, 4>(grad + (int64_t)runToken[i] * a.gradStride + column, acc, a.factor, a.add, 0, a.dim - column);
  };
  auto join_teams = [&](float(&acc)[4]) {
    for (int d = lanes; d < 64; d <<= 1) {
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] += __shfl_xor(acc[e], d);
    }
  };
  for (int i = ofWaves; i < runs; ++i) {
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    if (active) add_parts(acc, runFirst[i], runFirst[i] + team, teams, runLast[i]);
    join_teams(acc);
#pragma unroll
    for (int e = 0; e < 4; ++e) meet[wave][e][lane] = acc[e];
    __syncthreads();
    if (wave == 0 && sub == 0 && active) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
#pragma unroll
        for (int w = 1; w < W; ++w) acc[e] += meet[w][e][lane];
      }
      finish(i, acc);
    }
    __syncthreads();
  }
  for (int i = ofTeams + wave; i < ofWaves; i += W) {
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    if (active) add_parts(acc, runFirst[i], runFirst[i] + sub, subs, runLast[i]);
    join_teams(acc);
    if (sub == 0 && active) finish(i, acc);
  }
  for (int i = team; i < ofTeams; i += teams) {
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    if (active) {
      add_parts(acc, runFirst[i], runFirst[i], 1, runLast[i]);
      finish(i, acc);
    }
  }
}

// Few positions: one launch. A workgroup has one position and 64 lanes of columns; where its token has no earlier position, it lists the later
// ones and sums their rows, its waves in turn. Every workgroup looks at all tokens, which is what bounds the number of positions: 512 x 2048
// halves 7.5 us.
// Workgroups behind the positions zero the rows, kFewRows each, of tokens that do not occur.
constexpr int kFew = 2048, kFewRows = 64;
template <typename T, int V>
__global__ __launch_bounds__(kBlock) void few_kernel(T* __restrict__ grad, int64_t gradStride, const int64_t* __restrict__ tokens, int32_t n,
                                                     uint32_t vocab, uint32_t padding, const T* __restrict__ out, int64_t outStride, int32_t dim,
                                                     float factor, bool add, uint32_t zeroShares) {
  using P = Pack<T, V>;
  constexpr int W = kBlock / 64, U = 8;
  __shared__ uint64_t same[kFew / 64];
  __shared__ uint16_t list[kFew];
  __shared__ float meet[W][V][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int32_t column = ((int32_t)blockIdx.y * 64 + lane) * V, c0 = min(column, dim - V);
  const int skip = column - c0;
  auto token_at = [&](int32_t i) -> uint32_t {      // 0-based; ~0 for one that has no row
    const uint64_t k = (uint64_t)tokens[i];
    const uint32_t token = (uint32_t)k - 1;
    return (k >> 32) == 0 && token < vocab && token != padding ? token : ~0u;
  };
  if ((int32_t)blockIdx.x >= n) {
    const uint32_t row0 = (blockIdx.x - n) / zeroShares * kFewRows;
    if (threadIdx.x == 0) same[0] = 0;
    __syncthreads();
    for (int32_t i = threadIdx.x; i < n; i += kBlock) {
      const uint32_t token = token_at(i);
      if (token - row0 < (uint32_t)kFewRows) atomicOr((unsigned long long*)&same[0], 1ull << (token - row0));
    }
    __syncthreads();
    uint64_t rows = ~same[0] & share_of_rows((blockIdx.x - n) % zeroShares, zeroShares);
    if (vocab - row0 < (uint32_t)kFewRows) rows &= (uint64_t(1) << (vocab - row0)) - 1;
    zero_rows<false>(grad, gradStride, dim, row0, rows);
    return;
  }
  const uint32_t me = token_at(blockIdx.x);
  if (me == ~0u) return;
  // wave w looks at the words w, w + 4, ... of 64 positions, all loads in flight
  constexpr int kWords = kFew / 64 / W;
  const int64_t mine = (int64_t)me + 1;
  int64_t seen[kWords];
#pragma unroll
  for (int j = 0; j < kWords; ++j) {
    const int32_t i = (j * W + wave) * 64 + lane;
    seen[j] = i < n ? tokens[i] : 0;
  }
#pragma unroll
  for (int j = 0; j < kWords; ++j) {
    const uint64_t m = __ballot(seen[j] == mine);
    if (lane == 0) same[j * W + wave] = m;
  }
  __syncthreads();
  // a lane a word: how many positions lie before it, and whether an earlier position's workgroup has the token
  const uint64_t word = lane < kFew / 64 ? same[lane] : 0;
  int upto = __popcll(word);
#pragma unroll
  for (int d = 1; d < kFew / 64; d <<= 1) {
    const int o = __shfl_up(upto, d);
    if (lane >= d) upto += o;
  }
  const int count = __shfl(upto, kFew / 64 - 1), before = upto - __popcll(word);
  const int32_t here = blockIdx.x;
  const uint64_t earlier = lane * 64 + 64 <= here ? word : lane * 64 < here ? word & ((uint64_t(1) << (here & 63)) - 1) : 0;
  if (__ballot(earlier != 0)) return;      // the same for all
#pragma unroll
  for (int j = 0; j < kWords; ++j) {
    const int w = j * W + wave, base = __shfl(before, w);
    if (seen[j] == mine) list[base + __popcll(same[w] & ((uint64_t(1) << lane) - 1))] = (uint16_t)(w * 64 + lane);
  }
  __syncthreads();
  float acc[V];
#pragma unroll
  for (int e = 0; e < V; ++e) acc[e] = 0.f;
  if (column < dim) {
    for (int k = wave; k < count; k += W * U) {
      P v[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (k + u * W < count) v[u] = load_pack_unaligned<true, P>(out + (int64_t)list[k + u * W] * outStride + c0);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (k + u * W < count) {
#pragma unroll
          for (int e = 0; e < V; ++e) acc[e] += Cvt<T>::up(v[u].v[e]);
        }
      }
    }
  }
  if (count > 1) {
#pragma unroll
    for (int e = 0; e < V; ++e) meet[wave][e][lane] = acc[e];
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int e = 0; e < V; ++e) {
#pragma unroll
      for (int w = 1; w < W; ++w) acc[e] += meet[w][e][lane];
    }
  }
  if (wave == 0 && column < dim) finish_row<T, V>(grad + (int64_t)me * gradStride + c0, acc, factor, add, skip);
}

// Some thousand positions: one launch. A workgroup has an owner's tokens, grouped in LDS as above, and a strip of columns: short runs are summed
// by a team of lanes each, long ones by all teams, whose sums meet in LDS; rows of tokens that do not occur are zeroed. Bound by latency, step by
// step, and by the commonest token's workgroups: 1500 x 513 floats 8.1 us.
constexpr int kOwn = 4096, kOwnWaves = 8, kLongRun = 16, kOwnGrid = 512;
template <typename T, int V>
__global__ __launch_bounds__(kOwnWaves * 64) void own_kernel(T* __restrict__ grad, int64_t gradStride, const int64_t* __restrict__ tokens, int32_t n,
                                                             uint32_t vocab, uint32_t padding, const T* __restrict__ out, int64_t outStride,
                                                             int32_t dim, int lanes, float factor, bool add, int shift) {
  using P = Pack<T, V>;
  constexpr int W = kOwnWaves, kPer = kOwn / (W * 64), U = 8;
  static_assert(kOwnTokens == W * 64 && V * 64 <= kOwnTokens, "a thread for each token; the sums meet where the counts were");
  __shared__ int counts[W][kOwnTokens];
  __shared__ uint32_t found[W][kOwn / W];       // position and token, 16 bits each
  __shared__ uint16_t list[kOwn], runToken[kOwnTokens], runStart[kOwnTokens + 1], longRun[kOwn / kLongRun];
  __shared__ uint32_t waveTotal[W];
  __shared__ uint64_t occurs[W];
  float(*meet)[V][64] = reinterpret_cast<float(*)[V][64]>(counts);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint64_t below = (uint64_t(1) << lane) - 1;
  const uint32_t mask = (1u << shift) - 1, me = blockIdx.x;
  const int owned = (int)((vocab - 1 - me) >> shift) + 1;            // me < vocab
  const int32_t run = (n + W * 64 - 1) / (W * 64) * 64, first = wave * run + lane;
  uint64_t k[kPer];
#pragma unroll
  for (int u = 0; u < kPer; ++u)
    if (u * 64 < run) k[u] = (uint64_t)tokens[min(first + u * 64, n - 1)];
  for (int r = lane; r < owned; r += 64) counts[wave][r] = 0;        // (each wave its own)
  int mine = 0;
#pragma unroll
  for (int u = 0; u < kPer; ++u) {
    if (u * 64 < run) {
      const int32_t i = first + u * 64;
      const uint32_t token = (uint32_t)k[u] - 1;
      const bool own = i < n && (k[u] >> 32) == 0 && token < vocab && token != padding && (token & mask) == me;
      const uint64_t all = __ballot(own);
      if (own) {
        atomicAdd(&counts[wave][token >> shift], 1);      // whole numbers: any order gives the same
        found[wave][mine + __popcll(all & below)] = (uint32_t)i | (token >> shift) << 16;
      }
      mine += __popcll(all);
    }
  }
  __syncthreads();
  // tokens in order, a thread each; counted side by side: positions (13 bits), tokens that occur (10), long runs
  const int r = threadIdx.x;
  int count[W], sum = 0;
  if (r < owned) {
#pragma unroll
    for (int w = 0; w < W; ++w) {
      count[w] = counts[w][r];
      sum += count[w];
    }
  }
  const uint32_t one = (uint32_t)sum | (sum > 0 ? 1u << 13 : 0) | (sum > kLongRun ? 1u << 23 : 0);
  uint32_t upto = one;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t o = __shfl_up(upto, d);
    if (lane >= d) upto += o;
  }
  if (lane == 63) waveTotal[wave] = upto;
  const uint64_t some = __ballot(sum > 0);
  if (lane == 0) occurs[wave] = some;
  __syncthreads();
  uint32_t at = upto - one, total = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    if (w < wave) at += waveTotal[w];
    total += waveTotal[w];
  }
  const int runs = (total >> 13) & 1023, longs = total >> 23;
  if (sum > 0) {
    int slot = at & 8191;
    const int u = (at >> 13) & 1023;
    runToken[u] = (uint16_t)r;
    runStart[u] = (uint16_t)slot;
    if (sum > kLongRun) longRun[at >> 23] = (uint16_t)u;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      counts[w][r] = slot;
      slot += count[w];
    }
  }
  if (threadIdx.x == 0) runStart[runs] = (uint16_t)(total & 8191);
  __syncthreads();
  const int bits = owned > 1 ? 32 - __clz(owned - 1) : 0;
  for (int i = lane; i - lane < mine; i += 64) {
    const bool own = i < mine;
    const uint32_t f = found[wave][min(i, mine - 1)], which = f >> 16;
    const uint64_t peers = equal_lanes(which, bits, own);
    if (own) {
      const int to = counts[wave][which];
      list[to + __popcll(peers & below)] = (uint16_t)f;
      __builtin_amdgcn_wave_barrier();
      if ((peers & below) == 0) counts[wave][which] = to + __popcll(peers);
    }
    __builtin_amdgcn_wave_barrier();
  }
  __syncthreads();
  const int subs = 64 / lanes, sub = lane / lanes, team = wave * subs + sub, teams = W * subs;
  const int32_t column = ((int32_t)blockIdx.y * lanes + lane % lanes) * V, c0 = min(column, dim - V);
  const int skip = column - c0;
  const bool active = column < dim;
  // positions list[s], list[s + step], ... before `end`
  auto add_rows = [&](float(&acc)[V], int s, int step, int end) {
    for (; s < end; s += U * step) {
      P v[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (s + u * step < end) v[u] = load_pack_unaligned<true, P>(out + (int64_t)list[s + u * step] * outStride + c0);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (s + u * step < end) {
#pragma unroll
          for (int e = 0; e < V; ++e) acc[e] += Cvt<T>::up(v[u].v[e]);
        }
      }
    }
  };
  auto row_of = [&](int which) { return grad + (int64_t)(me + ((uint32_t)which << shift)) * gradStride + c0; };
  for (int j = 0; j < longs; ++j) {
    const int u = longRun[j];
    float acc[V];
#pragma unroll
    for (int e = 0; e < V; ++e) acc[e] = 0.f;
    P old;
    if (add && wave == 0 && sub == 0 && active) old = load_pack_unaligned<false, P>(row_of(runToken[u]));
    if (active) add_rows(acc, runStart[u] + team, teams, runStart[u + 1]);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      for (int d = lanes; d < 64; d <<= 1) acc[e] += __shfl_xor(acc[e], d);
      meet[wave][e][lane] = acc[e];
    }
    __syncthreads();
    if (wave == 0 && sub == 0 && active) {
#pragma unroll
      for (int e = 0; e < V; ++e) {
#pragma unroll
        for (int w = 1; w < W; ++w) acc[e] += meet[w][e][lane];
      }
      finish_row<T, V>(row_of(runToken[u]), old, acc, factor, add, skip);
    }
    __syncthreads();
  }
  if (!active) return;
  for (int u = team; u < runs; u += teams) {
    const int s = runStart[u], end = runStart[u + 1];
    if (end - s > kLongRun) continue;
    float acc[V];
#pragma unroll
    for (int e = 0; e < V; ++e) acc[e] = 0.f;
    P old;
    if (add) old = load_pack_unaligned<false, P>(row_of(runToken[u]));
    add_rows(acc, s, 1, end);
    finish_row<T, V>(row_of(runToken[u]), old, acc, factor, add, skip);
  }
  if (add) return;
  P zero;
#pragma unroll
  for (int e = 0; e < V; ++e) zero.v[e] = Cvt<T>::down(0.f);
  for (int q = team; q < owned; q += teams)
    if (!((occurs[q >> 6] >> (q & 63)) & 1)) store_pack_unaligned<false>(row_of(q), zero);
}

template <typename T>
void launch_grad(THCState* s, T* grad, int64_t vocab, int64_t gradStride, const int64_t* tokens, int32_t n, const T* out, int64_t outStride,
                 int32_t dim, float factor, int64_t padding, bool add) {
  hipStream_t st = current_stream(s);
  constexpr int kPack = 16 / sizeof(T);
  const int V = dim >= kPack ? kPack : 1;
  const int32_t packs = (dim + V - 1) / V, fewSlabs = (packs + 63) / 64;
  const uint32_t left = (uint32_t)(padding - 1);
  // A launch of owners: strips of columns so narrow, and owners so many, that there are up to 512 workgroups (two a CU; us with 256, 512 and
  // 1024 of them: 1500 x 513 fp32 7.8, 8.1, 9.6, 2000 x 1000 half 12.3, 11.1, 17.6). The commonest token's sum is a workgroup's for each strip,
  // which bounds the bytes that are summed; rows are zeroed less evenly than by the three launches, which bounds the table. us in three
  // launches and in this one, tokens as in text and all the same, added: 2000 x 64 half 15.2, 7.9 and 32.4, 15.0; 1500 x 513 fp32 13.5, 8.1 and
  // 29, 22; 2000 x 1000 half 15.7, 11.1 and 32, 44; 1500 x 2048 14.9, 11.9 and 27, 58. Tables written whole: 1500 x 513 fp32 into 10007
  // rows 16.9, 10.7, 2000 x 500 half into 32000 17.8, 19.0.
  int lanes = 8, shift = 0;
  while (((vocab - 1) >> shift) + 1 > kOwnTokens) ++shift;
  while (lanes < 64 && lanes < packs && ((int64_t)(packs + lanes - 1) / lanes << shift) > kOwnGrid) lanes *= 2;
  while (lanes > 1 && lanes / 2 >= packs) lanes /= 2;
  const int32_t strips = (packs + lanes - 1) / lanes;
  while (shift < 8 && (int64_t(2) << shift) <= vocab && ((int64_t)strips << (shift + 1)) <= kOwnGrid) ++shift;
  const bool own = n <= kOwn && ((int64_t)strips << shift) <= kOwnGrid && (int64_t)n * dim * (int64_t)sizeof(T) <= tuning("embedding.own", 4 << 20) &&
                   (add || vocab * dim * (int64_t)sizeof(T) <= 24 << 20);
  // A launch of positions: its time goes with the workgroups times what each looks at. us in that launch, of owners and in three (halves, added):
  // 16 x 2048 3.7, 5.2, 10.0; 600 x 2048 6.6, 7.7, 13.0; 1024 x 513 8.4, 8.8, 13.8; 1500 x 64 9.6, 7.5, 13.0; 1000 x 2048 13.7, 10.2, 13.7;
  // 512 x 8192 15.3, 18, 15.1.
  if (n <= kFew && vocab <= int64_t(1) << 28 && (int64_t)n * n * fewSlabs <= std::min<int64_t>(tuning("embedding.few", 3 << 20), own ? 3 << 19 : 3 << 20)) {
    const int32_t shares = zero_shares<T>(dim, fewSlabs);
    const dim3 grid((unsigned)(n + (add ? 0 : (vocab + kFewRows - 1) / kFewRows * shares)), fewSlabs);
    auto go = [&](auto v) {
      hipLaunchKernelGGL((few_kernel<T, decltype(v)::value>), grid, dim3(kBlock), 0, st, grad, gradStride, tokens, n, (uint32_t)vocab, left, out,
                         outStride, dim, factor, add, (uint32_t)shares);
    };
    if (V == 1) go(std::integral_constant<int, 1>{});
    else go(std::integral_constant<int, kPack>{});
    return;
  }
  if (own) {
    auto go = [&](auto v) {
      hipLaunchKernelGGL((own_kernel<T, decltype(v)::value>), dim3(1u << shift, strips), dim3(kOwnWaves * 64), 0, st, grad, gradStride, tokens, n,
                         (uint32_t)vocab, left, out, outStride, dim, lanes, factor, add, shift);
    };
    if (V == 1) go(std::integral_constant<int, 1>{});
    else go(std::integral_constant<int, kPack>{});
    return;
  }
  GradArgs a{};
  a.dim = dim;
  a.partialStride = (dim + 3) & ~3;
  a.outRowStride = outStride;
  a.gradStride = gradStride;
  a.factor = factor;
  a.add = add;
  // a power of two of lanes for a short row, several chunks to a workgroup; whole waves for a long one
  lanes = 1;
  while (lanes < 64 && lanes < packs) lanes *= 2;
  const int slabs = (packs + kBlock - 1) / kBlock;
  if (packs > 64) lanes = ((packs + slabs - 1) / slabs + 63) / 64 * 64;
  a.lanes = lanes;
  const int subs = std::max(1, kBlock / lanes);
  // Chunks that leave four workgroups to a CU, of 8 to 32 slots: each may leave partial sums. us with 4, 8, 16, 32, 64 (added): 8192 x 1024 half
  // 23.3, 20.9, 23.1, 31, 45; 32768 x 2048 half 85, 67, 62, 62, 71; 100000 x 64 half 48, 43, 45, 52, 71; 130000 x 1000 half 180, 133, 115,
  // 111, 116.
  const int64_t want = (int64_t)num_compute_units(s) * 4 * kBlock;
  a.chunk = (int32_t)std::min<int64_t>(32, std::max<int64_t>(8, (int64_t)n * lanes * slabs / want));
  a.chunks = (n + a.chunk - 1) / a.chunk;
  // owners: a power of two, none of which has more tokens than it has room to count
  shift = 0;
  while ((int64_t(1) << shift) < std::min<int64_t>(vocab, 256) || ((vocab - 1) >> shift) + 1 > kOwnTokens) ++shift;
  while ((int64_t(1) << shift) > vocab) --shift;
  const bool apart = n > tuning("embedding.split", kSplitFrom) && (1 << shift) <= kMostSplit;
  const int64_t tiles = apart ? (n + kTile - 1) / kTile : 0;
  const int64_t slots = (n + 3) & ~3, words = (vocab + 3) & ~int64_t(3), partials = (int64_t)a.chunks * 2 * a.partialStride;
  Workspace w(s, (slots * 2 + words + 4 + partials) * 4 + tiles * (kTile * 8 + ((1 << shift) + 1) * 4));
  a.g.position = reinterpret_cast<int32_t*>(w.data());
  a.g.token = a.g.position + slots;
  a.g.used = a.g.token + slots;
  a.g.total = a.g.used + words;
  a.partial = reinterpret_cast<float*>(a.g.total + 4);
  Split split;
  split.entry = reinterpret_cast<int2*>(a.partial + partials);
  split.begin = reinterpret_cast<int32_t*>(split.entry + tiles * kTile);
  if (apart) {
    hipLaunchKernelGGL(split_kernel, dim3((unsigned)tiles), dim3(kGroupThreads), 0, st, split, tokens, n, (uint32_t)vocab, left, shift);
    hipLaunchKernelGGL(group_kernel<true>, dim3(1u << shift), dim3(kGroupThreads), 0, st, a.g, split, tokens, n, (uint32_t)vocab, left, shift);
  } else {
    hipLaunchKernelGGL(group_kernel<false>, dim3(1u << shift), dim3(kGroupThreads), 0, st, a.g, split, tokens, n, (uint32_t)vocab, left, shift);
  }
  const int32_t chunkBlocks = (a.chunks + subs - 1) / subs;
  const bool shortRows = dim * (int64_t)sizeof(T) <= 128;
  a.zeroShares = shortRows ? 0 : zero_shares<T>(dim, slabs);
  const int64_t zeroBlocks = add ? 0 : shortRows ? (vocab + subs * 16 - 1) / (subs * 16) : (vocab + 63) / 64 * a.zeroShares;
  const dim3 grid((unsigned)(chunkBlocks + zeroBlocks), slabs), block(subs * lanes);
  // Zeros are streaming stores in large tables whose rows are whole lines: us, plain and streaming, of 32768 x 2048 halves into 50000 rows (205 MB)
  // 84, 78 (68, 77 where the caches still hold the table from the call before), 6000 x 8192 floats into 30000 219, 205; of 8192 x 1024 halves into
  // 32000 (66 MB) 29.3, 30.8; with lines that rows share, 3000 x 3000 floats into 50000 150, 159, 5000 x 1000 halves into 200000 98, 117.
  const bool lines = ((uintptr_t)grad | (uintptr_t)(gradStride * sizeof(T)) | (uintptr_t)(dim * sizeof(T))) % 128 == 0;
  const bool streaming = lines && vocab * dim * (int64_t)sizeof(T) >= int64_t(128) << 20;
  if (V == 1) hipLaunchKernelGGL((sum_kernel<T, 1, 8, false>), grid, block, 0, st, a, out, grad, vocab, chunkBlocks);
  else if (!streaming) hipLaunchKernelGGL((sum_kernel<T, kPack, 8, false>), grid, block, 0, st, a, out, grad, vocab, chunkBlocks);
  else hipLaunchKernelGGL((sum_kernel<T, kPack, 8, true>), grid, block, 0, st, a, out, grad, vocab, chunkBlocks);
  // strips of columns as narrow as leave two workgroups a CU
  const int32_t edges = (a.chunks + 63) / 64, quads = (dim + 3) / 4;
  lanes = 8;
  while (lanes < 64 && lanes < quads && (int64_t)((quads + lanes - 1) / lanes) * edges > kFoldGrid) lanes *= 2;
  while (lanes > 1 && lanes / 2 >= quads) lanes /= 2;
  hipLaunchKernelGGL((fold_kernel<T>), dim3(edges, (quads + lanes - 1) / lanes), dim3(kFoldWaves * 64), 0, st, a, grad, n, lanes);
}

void embedding_grad(THCState* s, DType dt, AnyTensor* grad, AnyTensor* tokens, AnyTensor* out, float factor, long padding, int accumulate) {
  const AnyTensor* ts[3] = {grad, tokens, out};
  check_same_gpu(s, 3, ts);
  check_table(grad, 2);
  THC_ARG_CHECK(!overlapping(tensor_layout(grad)), 2, "elements of the gradient overlap");
  const int64_t count = tensor_numel(tokens), vocab = grad->size[0], dim = grad->size[1];
  THC_ARG_CHECK(tensor_numel(out) == count * dim, 4, "%ld elements of the output's gradient for %ld tokens of %ld",
                (long)tensor_numel(out), (long)count, (long)dim);
  THC_ARG_CHECK(count <= int64_t(1) << 29, 3, "too many tokens");
  THC_ARG_CHECK(vocab <= int64_t(1) << 30, 2, "the table has too many rows");
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
