// Layer norm along the last dim, and its gradients.
//
//   layerNorm       y = (x - m) r w + b      m = mean(x), r = 1 / sqrt(mean((x - m)^2) + eps), of each row
//   layerNormGrad   h = (x - m) r;  dx = r (g w - mean(g w) - h mean(g w h)),  dw = sum over rows of g h,  db = sum over rows of g
//
// Statistics and sums are in float, outputs round once to their type. The mean is taken in two steps: m' = x0 + mean(x - x0), x0 the row's first element,
// then what is left, c = mean(x - m'), beside the squares; m = m' + c and the variance mean((x - m')^2) - c^2 lose nothing to a large offset of the
// row (m' as a float is off by 2^-24 of the offset, which may be much of the deviation). With x0 = 0, which takes an operation less an element, m' would
// be off by many times that in long rows, and the variance of a row of equal elements not 0 but what its two terms round to, below 0 among others: 1 % of
// the time in floats. Up to 8192 halves take 0 (2 to 3 %): as many equal ones sum exactly. The gradient's pass takes the statistics anew: the row is there
// anyway, the sums of its second step travel with those of g w and g w (x - m'), and nothing is kept between the passes.
#include <algorithm>
#include <type_traits>

#include "training.hpp"

namespace thc {
namespace {

using std::integral_constant;

// The sum over L neighbouring lanes, the same bits in each.
template <int CONTROL>
__device__ __forceinline__ float dpp(float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CONTROL, 0xf, 0xf, true));
}
template <int L>
__device__ __forceinline__ float lane_sum(float x) {
  if constexpr (L >= 2) x += dpp<0xb1>(x);       // the neighbour's
  if constexpr (L >= 4) x += dpp<0x4e>(x);       // the other pair's of four
  if constexpr (L >= 8) x += dpp<0x141>(x);      // mirrored in eight
  if constexpr (L >= 16) x += dpp<0x140>(x);     // mirrored in sixteen
  if constexpr (L >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  if constexpr (L >= 64) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  return x;
}

// N sums at once over the L lanes of each team of a workgroup of TEAMS teams; teams of more than a wave meet in LDS, of which two sums in turn use
// two parts, so that one barrier each is enough.
template <int N, int L, int TEAMS>
__device__ __forceinline__ void team_sum(float (&v)[N], float* lds) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = lane_sum<(L < 64 ? L : 64)>(v[i]);
  if constexpr (L > 64) {
    constexpr int W = L / 64;
    const int lane = threadIdx.x & 63, wave = (threadIdx.x >> 6) % W, team = threadIdx.x / L;
    float* mine = lds + team * N * W;
    if (lane == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) mine[i * W + wave] = v[i];
    }
    lds_barrier();
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = lane_sum<W>(mine[i * W + (lane & (W - 1))]);
  }
}

// 1 / sqrt(v), a unit in the last place off at most: the instruction, which takes numbers below the normal ones for zero.
__device__ __forceinline__ float inverse_root(float v) {
  return v < 0x1p-96f ? __builtin_amdgcn_rsqf(v * 0x1p96f) * 0x1p48f : __builtin_amdgcn_rsqf(v);
}

// What sums leave of a variance, which is not below 0. (NaN stays.)
__device__ __forceinline__ float variance(float squares, float c) {
  const float v = __builtin_fmaf(-c, c, squares);
  return v < 0.f ? 0.f : v;
}

// The packs of a row that a lane of a team of L has: pack p begins at element at[p], the first skip[p] of its V elements belong to the pack before
// it (a row's last pack is moved back into the row, so that reads need no tail; V where there is no pack at all). `whole`: none is moved.
template <int V, int L, int P>
struct Packs {
  int32_t at[P], skip[P];
  bool whole;
  __device__ __forceinline__ Packs(int32_t lane, int32_t dim) : whole(dim == V * L * P) {
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const int32_t first = (lane + p * L) * V;
      at[p] = min(first, dim - V);
      skip[p] = min(first - at[p], V);
    }
  }
  __device__ __forceinline__ bool has(int p) const { return skip[p] < V; }
};
// Elements that count elsewhere become 0.
template <int V, int L, int P>
__device__ __forceinline__ void clear_skipped(const Packs<V, L, P>& packs, float (&x)[P][V]) {
  if (packs.whole) return;
#pragma unroll
  for (int p = 0; p < P; ++p) {
    if (packs.skip[p]) {
#pragma unroll
      for (int e = 0; e < V; ++e) x[p][e] = e < packs.skip[p] ? 0.f : x[p][e];
    }
  }
}

// A row's first element as what distances are taken from, or 0.
template <typename T, bool WANTED>
struct First {
  T value;
  __device__ __forceinline__ void load(const T* row) {
    if constexpr (WANTED) value = *row;
  }
  __device__ __forceinline__ float get() const { return WANTED ? Cvt<T>::up(value) : 0.f; }
};
template <typename T>
constexpr bool from_first(int most) { return sizeof(T) == 4 || most > 8192; }
// What a lane adds to the sum of the row's distances to `from`.
template <bool FROM, int V, int L, int P>
__device__ __forceinline__ float distances(const Packs<V, L, P>& packs, const float (&x)[P][V], float from) {
  float d[P][V], sum = 0.f;
#pragma unroll
  for (int p = 0; p < P; ++p)
#pragma unroll
    for (int e = 0; e < V; ++e) d[p][e] = FROM ? x[p][e] - from : x[p][e];
  clear_skipped<V, L, P>(packs, d);
#pragma unroll
  for (int p = 0; p < P; ++p)
#pragma unroll
    for (int e = 0; e < V; ++e) sum += d[p][e];
  return sum;
}

template <typename T>
struct NormArgs {
  const T *x, *weight, *bias;      // weight, bias: or null
  T* y;
  RowOffsets xo, yo;
  uint32_t rows;
  int32_t dim;
  float eps;
};

template <typename T, int V, int P, int L>
__device__ __forceinline__ void store_row(T* row, const Packs<V, L, P>& packs, int p, const Pack<T, V>& v) {
  if (packs.whole || packs.skip[p] == 0) {
    store_pack_unaligned<true>(row + packs.at[p], v);
  } else if (packs.has(p)) {
#pragma unroll
    for (int e = 1; e < V; ++e)
      if (e >= packs.skip[p]) row[packs.at[p] + e] = v.v[e];
  }
}
template <typename T, int V, int P, int L>
__device__ __forceinline__ void load_row(const T* row, const Packs<V, L, P>& packs, Pack<T, V> (&v)[P]) {
#pragma unroll
  for (int p = 0; p < P; ++p) v[p] = load_pack_unaligned<true, Pack<T, V>>(row + packs.at[p]);
}
template <typename T, int V, int P>
__device__ __forceinline__ void to_floats(const Pack<T, V> (&v)[P], float (&x)[P][V]) {
#pragma unroll
  for (int p = 0; p < P; ++p)
#pragma unroll
    for (int e = 0; e < V; ++e) x[p][e] = Cvt<T>::up(v[p].v[e]);
}
template <typename T, int V, int P, int L>
__device__ __forceinline__ void load_columns(const T* from, const Packs<V, L, P>& packs, float (&v)[P][V], float otherwise) {
#pragma unroll
  for (int p = 0; p < P; ++p) {
    Pack<T, V> t{};
    if (from) t = load_pack_unaligned<false, Pack<T, V>>(from + packs.at[p]);
#pragma unroll
    for (int e = 0; e < V; ++e) v[p][e] = from ? Cvt<T>::up(t.v[e]) : otherwise;
  }
}

// A team of L lanes has a row in registers from its read to its write; teams go on to other rows with the weights that they hold, the next of which is
// asked for before the one at hand is computed. Bound by memory: 16392 rows of 2048 halves 24.6 us, 5.5 TB/s.
template <typename T, int V, int L, int TEAMS, int P>
__global__ __launch_bounds__(L * TEAMS) void norm_kernel(NormArgs<T> a) {
  __shared__ float lds[L > 64 ? 3 * TEAMS * (L / 64) : 1];
  const int32_t lane = threadIdx.x % L;
  const uint32_t team = threadIdx.x / L;
  const Packs<V, L, P> packs(lane, a.dim);
  const float n = (float)a.dim, share = 1.f / n;
  float w[P][V], b[P][V];
  load_columns<T, V, P, L>(a.weight, packs, w, 1.f);
  load_columns<T, V, P, L>(a.bias, packs, b, 0.f);
  Pack<T, V> raw[P];
  constexpr bool kFrom = from_first<T>(V * L * P);
  First<T, kFrom> start;
  auto load = [&](uint32_t first) {
    const T* in = a.x + a.xo.at(min(first + team, a.rows - 1));
    load_row<T, V, P, L>(in, packs, raw);
    start.load(in);
  };
  load(blockIdx.x * TEAMS);
  for (uint32_t first = blockIdx.x * TEAMS; first < a.rows; first += gridDim.x * TEAMS) {
    const uint32_t row = min(first + team, a.rows - 1);
    float x[P][V];
    to_floats(raw, x);
    const float x0 = start.get();
    // the next row is asked for before this one is computed
    if (first + gridDim.x * TEAMS < a.rows) load(first + gridDim.x * TEAMS);
    float one[1] = {distances<kFrom>(packs, x, x0)};
    team_sum<1, L, TEAMS>(one, lds);
    const float m = kFrom ? x0 + one[0] / n : one[0] / n;
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
      for (int e = 0; e < V; ++e) x[p][e] -= m;
    clear_skipped<V, L, P>(packs, x);
    float two[2] = {0.f, 0.f};
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        two[0] += x[p][e];
        two[1] = __builtin_fmaf(x[p][e], x[p][e], two[1]);
      }
    team_sum<2, L, TEAMS>(two, lds + TEAMS * (L / 64));
    const float c = two[0] * share, r = inverse_root(variance(two[1] * share, c) + a.eps), cr = -c * r;
    if (first + team < a.rows) {
      T* out = a.y + a.yo.at(row);
#pragma unroll
      for (int p = 0; p < P; ++p) {
        Pack<T, V> v;
#pragma unroll
        for (int e = 0; e < V; ++e) v.v[e] = rounded<T>(__builtin_fmaf(__builtin_fmaf(x[p][e], r, cr), w[p][e], b[p][e]));
        store_row(out, packs, p, v);
      }
    }
  }
}

template <typename T>
struct GradArgs {
  const T *x, *g, *weight;         // weight: or null
  T* dx;
  RowOffsets xo, go, dxo;
  float *weightPart, *biasPart;    // a row of sums for each workgroup; null: not wanted
  T *weightGrad, *biasGrad;        // where the only workgroup's sums go, with those null; or null
  int accumulate;
  uint32_t rows;
  int32_t dim;
  float eps;
};

// The same with the sums over rows of what a lane's columns add to the weights' gradients, which stay in its registers; the workgroup's teams join
// theirs at the end. Bound by memory and, in halves, by arithmetic nearly as much: 16392 rows of 4096 halves 78 us with the joining launch, 5.2 TB/s.
template <typename T, int V, int L, int TEAMS, int P, bool WEIGHTS, bool AHEAD>
__global__ __launch_bounds__(L * TEAMS, 2) void norm_grad_kernel(GradArgs<T> a) {
  __shared__ float lds[L > 64 ? 5 * TEAMS * (L / 64) : 1];
  constexpr int kCols = L * P * V;                                       // (teams that share a wave join by lanes first)
  constexpr int kJoin = L < 64 ? L * TEAMS / 64 : TEAMS;
  __shared__ float join[WEIGHTS && kJoin > 1 ? 2 * kCols : 1];
  const int32_t lane = threadIdx.x % L;
  const uint32_t team = threadIdx.x / L;
  const Packs<V, L, P> packs(lane, a.dim);
  const float n = (float)a.dim, share = 1.f / n;
  float w[P][V], dw[P][V], db[P][V];
  load_columns<T, V, P, L>(a.weight, packs, w, 1.f);
  clear_skipped<V, L, P>(packs, w);
#pragma unroll
  for (int p = 0; p < P; ++p)
#pragma unroll
    for (int e = 0; e < V; ++e) dw[p][e] = db[p][e] = 0.f;
  Pack<T, V> raw[P], graw[P];
  constexpr bool kFrom = from_first<T>(V * L * P);
  First<T, kFrom> start;
  auto load = [&](uint32_t first) {
    const uint32_t row = min(first + team, a.rows - 1);
    const T* in = a.x + a.xo.at(row);
    load_row<T, V, P, L>(in, packs, raw);
    load_row<T, V, P, L>(a.g + a.go.at(row), packs, graw);
    start.load(in);
  };
  if (AHEAD) load(blockIdx.x * TEAMS);
  for (uint32_t first = blockIdx.x * TEAMS; first < a.rows; first += gridDim.x * TEAMS) {
    if (!AHEAD) load(first);
    float d[P][V], g[P][V];
    to_floats(raw, d);
    to_floats(graw, g);
    const float x0 = start.get();
    // the next row is asked for before this one is computed
    if (AHEAD && first + gridDim.x * TEAMS < a.rows) load(first + gridDim.x * TEAMS);
    float one[1] = {distances<kFrom>(packs, d, x0)};
    team_sum<1, L, TEAMS>(one, lds);
    const float m = kFrom ? x0 + one[0] / n : one[0] / n;
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
      for (int e = 0; e < V; ++e) d[p][e] -= m;
    clear_skipped<V, L, P>(packs, d);
    float four[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float gw = g[p][e] * w[p][e];             // (w is 0 where d is)
        four[0] += d[p][e];
        four[1] = __builtin_fmaf(d[p][e], d[p][e], four[1]);
        four[2] += gw;
        four[3] = __builtin_fmaf(gw, d[p][e], four[3]);
      }
    team_sum<4, L, TEAMS>(four, lds + TEAMS * (L / 64));
    const float c = four[0] * share, r = inverse_root(variance(four[1] * share, c) + a.eps), cr = -c * r;
    // mean(g w h) and mean(g w), times r
    const float meanH = (four[3] - c * four[2]) * r * share * r, meanG = four[2] * share * r;
    if (TEAMS > 1 && first + team >= a.rows) continue;      // (all of a wave's lanes that still sum are back together at its next row)
    T* out = a.dx + a.dxo.at(first + team);
#pragma unroll
    for (int p = 0; p < P; ++p) {
      Pack<T, V> v;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float h = __builtin_fmaf(d[p][e], r, cr);
        v.v[e] = rounded<T>(__builtin_fmaf(-h, meanH, __builtin_fmaf(g[p][e] * w[p][e], r, -meanG)));
        if constexpr (WEIGHTS) {
          dw[p][e] = __builtin_fmaf(g[p][e], h, dw[p][e]);
          db[p][e] += g[p][e];
        }
      }
      store_row(out, packs, p, v);
    }
  }
  if constexpr (WEIGHTS) {
#pragma unroll
    for (int p = 0; p < P; ++p) {
#pragma unroll
      for (int e = 0; e < V; ++e) {
#pragma unroll
        for (int s = L; s < 64; s <<= 1) {
          dw[p][e] += __shfl_xor(dw[p][e], s);
          db[p][e] += __shfl_xor(db[p][e], s);
        }
      }
    }
    if constexpr (kJoin > 1) {
      // the part with the highest number writes, those below it add theirs one after another: the first one's registers get the sum
      const int part = L < 64 ? threadIdx.x / 64 : team;
      const bool writes = L >= 64 || threadIdx.x % 64 < L;
      for (int k = kJoin - 1; k >= 0; --k) {
        if (part == k && writes) {
#pragma unroll
          for (int p = 0; p < P; ++p) {
#pragma unroll
            for (int e = 0; e < V; ++e) {
              float *jw = join + (p * V + e) * L + lane, *jb = jw + kCols;
              if (k < kJoin - 1) {
                dw[p][e] += *jw;
                db[p][e] += *jb;
              }
              if (k > 0) {
                *jw = dw[p][e];
                *jb = db[p][e];
              }
            }
          }
        }
        lds_barrier();
      }
    }
    if (threadIdx.x < L && gridDim.x == 1) {
      auto write = [&](T* to, const float (&sum)[P][V]) {
        if (!to) return;
#pragma unroll
        for (int p = 0; p < P; ++p) {
          T* at = to + packs.at[p];
          auto value = [&](int e, T was) { return rounded<T>(a.accumulate ? Cvt<T>::up(was) + sum[p][e] : sum[p][e]); };
          if (packs.skip[p] == 0) {
            Pack<T, V> v{};
            if (a.accumulate) v = load_pack_unaligned<false, Pack<T, V>>(at);
#pragma unroll
            for (int e = 0; e < V; ++e) v.v[e] = value(e, v.v[e]);
            store_pack_unaligned<false>(at, v);
          } else {
#pragma unroll
            for (int e = 1; e < V; ++e)
              if (e >= packs.skip[p]) at[e] = value(e, at[e]);
          }
        }
      };
      write(a.weightGrad, dw);
      write(a.biasGrad, db);
    } else if (threadIdx.x < L) {
      auto leave = [&](float* part, const float (&sum)[P][V]) {
        if (!part) return;
#pragma unroll
        for (int p = 0; p < P; ++p) {
          float* at = part + (int64_t)blockIdx.x * a.dim + packs.at[p];
          constexpr int N = V < 4 ? V : 4;
          if (packs.skip[p] == 0) {
#pragma unroll
            for (int q = 0; q < V / N; ++q) {
              Pack<float, N> v;
#pragma unroll
              for (int e = 0; e < N; ++e) v.v[e] = sum[p][q * N + e];
              store_pack_unaligned<false>(at + q * N, v);
            }
          } else {
#pragma unroll
            for (int e = 1; e < V; ++e)
              if (e >= packs.skip[p]) at[e] = sum[p][e];
          }
        }
      };
      leave(a.weightPart, dw);
      leave(a.biasPart, db);
    }
  }
}

// The workgroups' rows of sums, added up for 32 columns a workgroup (blockIdx.y: weight or bias), 32 shares of the rows side by side.
template <typename T>
__global__ __launch_bounds__(1024) void join_kernel(const float* weightPart, const float* biasPart, T* weight, T* bias, int32_t parts,
                                                    int32_t dim, int accumulate) {
  __shared__ float lds[32][33];
  const float* from = blockIdx.y ? biasPart : weightPart;
  T* to = blockIdx.y ? bias : weight;
  if (!from) return;
  const int32_t x = threadIdx.x & 31, y = threadIdx.x >> 5, column = blockIdx.x * 32 + x;
  float sum = 0.f;
  if (column < dim) {
    constexpr int U = 8;
    for (int32_t i = y; i < parts; i += 32 * U) {
      float v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) v[u] = i + u * 32 < parts ? from[(int64_t)(i + u * 32) * dim + column] : 0.f;
#pragma unroll
      for (int u = 0; u < U; ++u) sum += v[u];
    }
  }
  lds[y][x] = sum;
  __syncthreads();
  sum = lane_sum<32>(lds[x][y]);           // column y of this workgroup, by the 32 lanes that have its shares
  const int32_t mine = blockIdx.x * 32 + y;
  if (x == 0 && mine < dim) {
    T* p = to + mine;
    *p = rounded<T>(accumulate ? Cvt<T>::up(*p) + sum : sum);
  }
}

// ------------------------------------------------------------------ long rows --
// Rows that registers do not hold are read again for each step: a workgroup's lanes go over a row's packs and, one by one, the elements behind them.
template <typename T, typename F>
__device__ __forceinline__ void over_row(int32_t dim, F f) {
  constexpr int V = 16 / sizeof(T);
  const int32_t packs = dim / V;
  for (int32_t k = threadIdx.x; k < packs; k += blockDim.x) f(k * V, integral_constant<int, V>{});
  const int32_t i = packs * V + threadIdx.x;
  if (i < dim) f(i, integral_constant<int, 1>{});
}
template <typename T, int N>
__device__ __forceinline__ void load_some(const T* p, float (&v)[N], float otherwise = 0.f) {
  Pack<T, N> t{};
  if (p) t = load_pack_unaligned<false, Pack<T, N>>(p);
#pragma unroll
  for (int e = 0; e < N; ++e) v[e] = p ? Cvt<T>::up(t.v[e]) : otherwise;
}
constexpr int kLong = 1024;

// The mean's two parts and one over the deviation.
struct RowStats {
  float m, c, r, meanG, meanH;      // meanG, meanH: of the gradient, times r
};
template <typename T>
__device__ __forceinline__ RowStats stats_of(const T* row, const T* g, const T* weight, int32_t dim, float eps, float* lds) {
  RowStats s{};
  const float n = (float)dim, x0 = Cvt<T>::up(*row);
  float one[1] = {0.f};
  over_row<T>(dim, [&](int32_t i, auto count) {
    float x[decltype(count)::value];
    load_some(row + i, x);
    for (float v : x) one[0] += v - x0;
  });
  team_sum<1, kLong, 1>(one, lds);
  s.m = x0 + one[0] / n;
  float four[4] = {0.f, 0.f, 0.f, 0.f};
  over_row<T>(dim, [&](int32_t i, auto count) {
    constexpr int N = decltype(count)::value;
    float x[N], gr[N], w[N];
    load_some(row + i, x);
    if (g) {
      load_some(g + i, gr);
      load_some(weight ? weight + i : nullptr, w, 1.f);
    }
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float d = x[e] - s.m;
      four[0] += d;
      four[1] = __builtin_fmaf(d, d, four[1]);
      if (g) {
        const float gw = gr[e] * w[e];
        four[2] += gw;
        four[3] = __builtin_fmaf(gw, d, four[3]);
      }
    }
  });
  team_sum<4, kLong, 1>(four, lds + kLong / 64);
  s.c = four[0] / n;
  s.r = 1.f / sqrtf(variance(four[1] / n, s.c) + eps);
  s.meanH = (four[3] - s.c * four[2]) * s.r / n * s.r;
  s.meanG = four[2] / n * s.r;
  return s;
}

template <typename T>
__global__ __launch_bounds__(kLong) void long_norm_kernel(NormArgs<T> a) {
  __shared__ float lds[5 * (kLong / 64)];
  for (uint32_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* in = a.x + a.xo.at(row);
    T* out = a.y + a.yo.at(row);
    const RowStats s = stats_of<T>(in, (const T*)nullptr, (const T*)nullptr, a.dim, a.eps, lds);
    over_row<T>(a.dim, [&](int32_t i, auto count) {
      constexpr int N = decltype(count)::value;
      float x[N], w[N], b[N];
      load_some(in + i, x);
      load_some(a.weight ? a.weight + i : nullptr, w, 1.f);
      load_some(a.bias ? a.bias + i : nullptr, b);
      Pack<T, N> v;
#pragma unroll
      for (int e = 0; e < N; ++e) v.v[e] = rounded<T>(__builtin_fmaf((x[e] - s.m - s.c) * s.r, w[e], b[e]));
      store_pack_unaligned<true>(out + i, v);
    });
  }
}
template <typename T>
__global__ __launch_bounds__(kLong) void long_stats_kernel(GradArgs<T> a, RowStats* stats) {
  __shared__ float lds[5 * (kLong / 64)];
  for (uint32_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const RowStats s = stats_of<T>(a.x + a.xo.at(row), a.g + a.go.at(row), a.weight, a.dim, a.eps, lds);
    if (threadIdx.x == 0) stats[row] = s;
  }
}
// Sums over a share of the rows for 256 columns a workgroup; before the gradient of the input, which may lie on what is read.
template <typename T>
__global__ __launch_bounds__(kBlock) void long_columns_kernel(GradArgs<T> a, const RowStats* stats, uint32_t rowsEach) {
  const int32_t column = blockIdx.x * kBlock + threadIdx.x;
  if (column >= a.dim) return;
  const uint32_t begin = blockIdx.y * rowsEach, end = min(a.rows, begin + rowsEach);
  float dw = 0.f, db = 0.f;
  for (uint32_t row = begin; row < end; ++row) {
    const RowStats s = stats[row];
    const float g = Cvt<T>::up(a.g[a.go.at(row) + column]), h = (Cvt<T>::up(a.x[a.xo.at(row) + column]) - s.m - s.c) * s.r;
    dw = __builtin_fmaf(g, h, dw);
    db += g;
  }
  if (a.weightPart) a.weightPart[(int64_t)blockIdx.y * a.dim + column] = dw;
  if (a.biasPart) a.biasPart[(int64_t)blockIdx.y * a.dim + column] = db;
}
template <typename T>
__global__ __launch_bounds__(kLong) void long_grad_kernel(GradArgs<T> a, const RowStats* stats) {
  for (uint32_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const RowStats s = stats[row];
    const T *in = a.x + a.xo.at(row), *grad = a.g + a.go.at(row);
    T* out = a.dx + a.dxo.at(row);
    over_row<T>(a.dim, [&](int32_t i, auto count) {
      constexpr int N = decltype(count)::value;
      float x[N], g[N], w[N];
      load_some(in + i, x);
      load_some(grad + i, g);
      load_some(a.weight ? a.weight + i : nullptr, w, 1.f);
      Pack<T, N> v;
#pragma unroll
      for (int e = 0; e < N; ++e)
        v.v[e] = rounded<T>(__builtin_fmaf(-((x[e] - s.m - s.c) * s.r), s.meanH, __builtin_fmaf(g[e] * w[e], s.r, -s.meanG)));
      store_pack_unaligned<true>(out + i, v);
    });
  }
}

// ------------------------------------------------------------------- launches --
template <typename T>
void launch_norm(THCState* s, const NormArgs<T>& a) {
  constexpr int V = 16 / sizeof(T);
  hipStream_t st = current_stream(s);
  const int64_t cus = num_compute_units(s), packs = (a.dim + V - 1) / V;
  auto go = [&](auto vec, auto lanes, auto teams, auto each) {
    constexpr int VV = decltype(vec)::value, L = decltype(lanes)::value, TEAMS = decltype(teams)::value, P = decltype(each)::value;
    const int64_t groups = ((int64_t)a.rows + TEAMS - 1) / TEAMS, most = cus * std::max(1, (P == 1 ? 2048 : packs <= 256 ? 1024 : 512) / (L * TEAMS));
    hipLaunchKernelGGL((norm_kernel<T, VV, L, TEAMS, P>), dim3((unsigned)std::min(groups, most)), dim3(L * TEAMS), 0, st, a);
  };
#define GO(VV, L, TEAMS, P) go(integral_constant<int, VV>{}, integral_constant<int, L>{}, integral_constant<int, TEAMS>{}, integral_constant<int, P>{})
  // Two packs a lane where rows have them: half of the lanes that meet at a sum. us for 16392 rows of 2048 halves with 64 lanes of 4 packs, 128 of 2 and 256 of
  // 1: 29.2, 25.3, 26.4. Threads a CU: with 512, 1024 and 2048 16384 rows of 2048 halves 26.1, 25.1, 27.7, 65536 of 500 38.6, 30.5, 32.8; 8192 of 8192
  // 46.4, 51.1, 48.3, 16384 of 2000 floats 44.9, 47.9, 48.6; 65536 of 64 floats 8.9, 7.9, 7.3.
  if (a.dim < V) GO(1, 8, 32, 1);
  else if (packs <= 8) GO(V, 8, 32, 1);
  else if (packs <= 16) GO(V, 16, 16, 1);
  else if (packs <= 32) GO(V, 32, 8, 1);
  else if (packs <= 64) GO(V, 32, 8, 2);
  else if (packs <= 128) GO(V, 64, 4, 2);
  else if (packs <= 256) GO(V, 128, 2, 2);
  else if (packs <= 512) GO(V, 256, 1, 2);
  else if (packs <= 1024) GO(V, 256, 1, 4);
  else if (packs <= 2048) GO(V, 512, 1, 4);
  else if (V == 4 && packs <= 4096) GO(V, (V == 4 ? 1024 : 512), 1, 4);      // (a length that halves have already)
  else hipLaunchKernelGGL((long_norm_kernel<T>), dim3((unsigned)std::min<int64_t>(a.rows, cus * 2)), dim3(kLong), 0, st, a);
#undef GO
}

template <typename T>
struct WeightGrads {
  T *weight, *bias;      // null: not wanted
  bool accumulate;
};
template <typename T>
void launch_grad(THCState* s, GradArgs<T>& a, const WeightGrads<T>& to) {
  constexpr int V = 16 / sizeof(T);
  hipStream_t st = current_stream(s);
  const int64_t cus = num_compute_units(s), packs = (a.dim + V - 1) / V;
  const bool sums = to.weight || to.bias;
  if (sums || packs > (V == 4 ? 4096 : 2048)) refuse_capture(s, "the gradient of a norm's weights, or of long rows,");
  auto parts = [&](int64_t count, Workspace& w) {
    float* p = reinterpret_cast<float*>(w.data());
    a.weightPart = to.weight ? p : nullptr;
    a.biasPart = to.bias ? p + (to.weight ? count * a.dim : 0) : nullptr;
  };
  auto bytes = [&](int64_t count) { return count * a.dim * 4 * ((to.weight != nullptr) + (to.bias != nullptr)); };
  auto join = [&](int64_t count) {
    hipLaunchKernelGGL((join_kernel<T>), dim3((a.dim + 31) / 32, 2), dim3(1024), 0, st, a.weightPart, a.biasPart, to.weight, to.bias, (int32_t)count, a.dim, (int)to.accumulate);
  };
  auto go = [&](auto vec, auto lanes, auto teams, auto each, auto ahead, int64_t threads) {
    constexpr int VV = decltype(vec)::value, L = decltype(lanes)::value, TEAMS = decltype(teams)::value, P = decltype(each)::value;
    constexpr bool A = decltype(ahead)::value;
    const int64_t groups = ((int64_t)a.rows + TEAMS - 1) / TEAMS, most = cus * std::max<int64_t>(1, threads / (L * TEAMS));
    if (!sums) {
      hipLaunchKernelGGL((norm_grad_kernel<T, VV, L, TEAMS, P, false, A>), dim3((unsigned)std::min(groups, 2 * most)), dim3(L * TEAMS), 0, st, a);
      return;
    }
    // Few rows: one workgroup has the sums, and no launch joins them. us with a join and so: 4 rows of 2048 halves 6.9, 6.0, 8 of them 7.5, 7.7; 8 of 500 6.7,
    // 5.7, 16 7.0, 6.9; 2 of 4096 6.7, 5.1, 4 of them 7.4, 7.6; 1 of 16384 11.7, 7.4, 4 of them 14.1, 14.9.
    // Else a workgroup's sums cross memory twice: each has two rows at least, or three. us with two, three and four: 300 rows of 4096 halves 10.5, 10.7, 11.4,
    // 1024 19.3, 17.7, 15.3; 1500 of 513 floats 9.7, 9.3, 10.3; 600 of 8192 23.2, 20.8, 20.4; 100 of 2048 halves 8.0, 10.2, 11.1.
    const int64_t count = groups <= 3 ? 1 : std::max<int64_t>(2, std::min(groups / (groups < 512 ? 2 : 3), most));
    if (count == 1) {
      a.weightGrad = to.weight;
      a.biasGrad = to.bias;
      a.accumulate = to.accumulate;
      hipLaunchKernelGGL((norm_grad_kernel<T, VV, L, TEAMS, P, true, A>), dim3(1), dim3(L * TEAMS), 0, st, a);
      return;
    }
    Workspace w(s, bytes(count));
    parts(count, w);
    hipLaunchKernelGGL((norm_grad_kernel<T, VV, L, TEAMS, P, true, A>), dim3((unsigned)count), dim3(L * TEAMS), 0, st, a);
    join(count);
  };
#define GO(VV, L, TEAMS, P, A, THREADS) \
  go(integral_constant<int, VV>{}, integral_constant<int, L>{}, integral_constant<int, TEAMS>{}, integral_constant<int, P>{}, integral_constant<bool, A>{}, THREADS)
  // The last number: threads a CU. More hide the two sums of a row better, and make more rows of sums that cross memory. us with 512, 768 and 1024 of
  // them: 16384 rows of 4096 halves 78, 80, 90, of 2048 42, 45, 51, 16384 of 2000 floats 74, 78, 81; 65536 of 500 halves 53, 50, 50. The next row is
  // asked for early where registers allow it (4096 halves 148 without, 88 with, at that time in 768; two rows early 2 to 6 % slower).
  if (a.dim < V) GO(1, 8, 32, 1, true, 1024);
  else if (packs <= 8) GO(V, 8, 32, 1, true, 1024);
  else if (packs <= 16) GO(V, 16, 16, 1, true, 1024);
  else if (packs <= 32) GO(V, 32, 8, 1, true, 1024);
  else if (packs <= 64) GO(V, 64, 4, 1, true, 1024);
  else if (packs <= 128) GO(V, 64, 4, 2, true, 512);
  else if (packs <= 256) GO(V, 128, 2, 2, true, 512);
  else if (packs <= 512) GO(V, 256, 1, 2, true, 512);
  else if (packs <= 1024) GO(V, 256, 1, 4, true, 512);
  else if (packs <= 2048) GO(V, 512, 1, 4, true, 512);
  else if (V == 4 && packs <= 4096) GO(V, (V == 4 ? 1024 : 512), 1, 4, (V == 8), 1024);
  else {
    const dim3 grid((unsigned)std::min<int64_t>(a.rows, cus * 2));
    Workspace stats(s, (int64_t)a.rows * sizeof(RowStats));
    RowStats* p = reinterpret_cast<RowStats*>(stats.data());
    hipLaunchKernelGGL((long_stats_kernel<T>), grid, dim3(kLong), 0, st, a, p);
    if (sums) {
      const int64_t across = (a.dim + kBlock - 1) / kBlock, want = std::max<int64_t>(1, cus * 8 / across);
      const int64_t each = std::max<int64_t>(16, (a.rows + want - 1) / want), count = (a.rows + each - 1) / each;
      Workspace w(s, bytes(count));
      parts(count, w);
      hipLaunchKernelGGL((long_columns_kernel<T>), dim3((unsigned)across, (unsigned)count), dim3(kBlock), 0, st, a, p, (uint32_t)each);
      join(count);
    }
    hipLaunchKernelGGL((long_grad_kernel<T>), grid, dim3(kLong), 0, st, a, p);
  }
#undef GO
}

// A row of weights, one for each column: dense for the kernels.
void check_columns(const AnyTensor* t, int64_t dim, int arg, const char* what) {
  THC_ARG_CHECK(tensor_numel(t) == dim, arg, "%ld %s for rows of %ld", (long)tensor_numel(t), what, (long)dim);
}
void check_rows(const AnyTensor* x, int arg) {
  THC_ARG_CHECK(x->nDimension <= kMaxDims, arg, "%s", kDimWarning);
  const int64_t dim = x->size[x->nDimension - 1];
  THC_ARG_CHECK(dim < (int64_t(1) << 24), arg, "rows are too long");       // (their lengths are exact floats)
  THC_ARG_CHECK(tensor_numel(x) / dim < kIndex32Limit, arg, "too many rows");
}

// Rows to be read: the tensor's own, or a dense copy's.
struct RowInput {
  TensorRef ref;
  Rows rows;
  RowInput(THCState* s, AnyTensor* t, DType dt) : ref(s, nullptr) {
    if (as_rows(t, &rows)) {
      tensor_retain(t);
      ref.t = t;
    } else {
      refuse_capture(s, "a norm of rows that lie apart");
      ref.t = tensor_new_contiguous(s, t, dt);
      as_rows(ref.t, &rows);
    }
  }
  bool same_place(const AnyTensor* t, const Rows& r) const {
    return ref.t->storage == t->storage && ref.t->storageOffset == t->storageOffset && r.count == rows.count && r.length == rows.length &&
           r.inner == rows.inner && r.stride == rows.stride && r.outerStride == rows.outerStride;
  }
};
// Rows to be written: the tensor's own where they do not overlap and lie on nothing that is read but the same rows of an input.
struct RowOutput {
  THCState* s;
  AnyTensor* to;
  DType dt;
  TensorRef ref;
  Rows rows;
  RowOutput(THCState* s_, AnyTensor* t, DType d, std::initializer_list<const RowInput*> inputs, std::initializer_list<const AnyTensor*> others)
      : s(s_), to(t), dt(d), ref(s_, nullptr) {
    bool direct = as_rows(t, &rows) && !overlapping(tensor_layout(t));
    for (const RowInput* i : inputs) direct = direct && (!spans_meet(t, d, i->ref.t, d) || i->same_place(t, rows));
    for (const AnyTensor* o : others) direct = direct && !spans_meet(t, d, o, d);
    if (direct) {
      tensor_retain(t);
      ref.t = t;
    } else {
      refuse_capture(s, "a norm whose output lies apart or on what it reads");
      ref.t = tensor_new_with_size(s, t->nDimension, t->size, d);
      as_rows(ref.t, &rows);
    }
  }
  void write_back() {
    if (ref.t != to) copy_tensor(s, dt, to, ref.t, false);
  }
};

// A row of numbers for the columns, dense.
AnyTensor* columns(THCState* s, AnyTensor* t, DType dt) {
  if (t && !tensor_is_contiguous(t)) refuse_capture(s, "a norm with strided weights");
  return t ? tensor_new_contiguous(s, t, dt) : nullptr;
}

template <typename T>
const T* data_of(const TensorRef& r, DType dt) {
  return r.t ? static_cast<const T*>(tensor_data(r.t, dt)) : nullptr;
}

template <typename T>
void run_norm(THCState* s, DType dt, AnyTensor* self, AnyTensor* input, AnyTensor* weight, AnyTensor* bias, float eps) {
  RowInput x(s, input, dt);
  TensorRef w(s, columns(s, weight, dt)), b(s, columns(s, bias, dt));
  RowOutput y(s, self, dt, {&x}, {w.t, b.t});
  NormArgs<T> a;
  a.x = data_of<T>(x.ref, dt);
  a.weight = data_of<T>(w, dt);
  a.bias = data_of<T>(b, dt);
  a.y = static_cast<T*>(tensor_data(y.ref.t, dt));
  a.xo = offsets_of(x.rows);
  a.yo = offsets_of(y.rows);
  a.rows = (uint32_t)x.rows.count;
  a.dim = (int32_t)x.rows.length;
  a.eps = eps;
  launch_norm<T>(s, a);
  THC_CHECK(hipGetLastError());
  note_kernel("layer-norm");
  y.write_back();
}

void layer_norm(THCState* s, DType dt, AnyTensor* self, AnyTensor* input, AnyTensor* weight, AnyTensor* bias, double eps) {
  const AnyTensor* all[4] = {self, input, weight, bias};
  check_same_gpu(s, 4, all);
  THC_ARG_CHECK(eps >= 0, 6, "eps is negative");
  if (!has_elements(input)) {
    tensor_resize_as(s, self, input, dt);
    return;
  }
  check_rows(input, 3);
  const int64_t dim = input->size[input->nDimension - 1];
  if (weight) check_columns(weight, dim, 4, "weights");
  if (bias) check_columns(bias, dim, 5, "biases");
  THC_ARG_CHECK(self != weight && self != bias, 2, "the output may not be the weight or the bias");
  tensor_resize_as(s, self, input, dt);
  note_stream_use(s, {self, input, weight, bias});
  if (dt == DType::F32) run_norm<float>(s, dt, self, input, weight, bias, (float)eps);
  else run_norm<__half>(s, dt, self, input, weight, bias, (float)eps);
}

// A gradient of columns: the tensor itself where it is dense and lies on nothing that is read or written, or one that is copied there.
struct ColumnOutput {
  THCState* s;
  AnyTensor* to;
  DType dt;
  TensorRef ref;
  ColumnOutput(THCState* s_, AnyTensor* t, DType d, bool accumulate, std::initializer_list<const AnyTensor*> touched) : s(s_), to(t), dt(d), ref(s_, nullptr) {
    if (!t) return;
    bool direct = tensor_is_contiguous(t);
    for (const AnyTensor* o : touched) direct = direct && !spans_meet(t, d, o, d);
    if (direct) {
      tensor_retain(t);
      ref.t = t;
    } else {
      ref.t = accumulate ? tensor_new_clone(s, t, d) : tensor_new_with_size(s, t->nDimension, t->size, d);
    }
  }
  void write_back() {
    if (to && ref.t != to) copy_tensor(s, dt, to, ref.t, false);
  }
};

template <typename T>
void run_grad(THCState* s, DType dt, AnyTensor* gradInput, AnyTensor* gradWeight, AnyTensor* gradBias, AnyTensor* input, AnyTensor* gradOutput,
              AnyTensor* weight, float eps, bool accumulate) {
  RowInput x(s, input, dt), g(s, gradOutput, dt);
  TensorRef w(s, columns(s, weight, dt));
  ColumnOutput dw(s, gradWeight, dt, accumulate, {x.ref.t, g.ref.t, w.t}), db(s, gradBias, dt, accumulate, {x.ref.t, g.ref.t, w.t});
  RowOutput dx(s, gradInput, dt, {&x, &g}, {w.t, gradWeight, gradBias});
  GradArgs<T> a{};
  a.x = data_of<T>(x.ref, dt);
  a.g = data_of<T>(g.ref, dt);
  a.weight = data_of<T>(w, dt);
  a.dx = static_cast<T*>(tensor_data(dx.ref.t, dt));
  a.xo = offsets_of(x.rows);
  a.go = offsets_of(g.rows);
  a.dxo = offsets_of(dx.rows);
  a.rows = (uint32_t)x.rows.count;
  a.dim = (int32_t)x.rows.length;
  a.eps = eps;
  WeightGrads<T> to{};
  to.weight = const_cast<T*>(data_of<T>(dw.ref, dt));
  to.bias = const_cast<T*>(data_of<T>(db.ref, dt));
  to.accumulate = accumulate;
  launch_grad<T>(s, a, to);
  THC_CHECK(hipGetLastError());
  note_kernel("layer-norm-grad");
  dx.write_back();
  dw.write_back();
  db.write_back();
}

// Two outputs on one another would be written over by each other's workgroups.
void check_apart(const AnyTensor* a, const AnyTensor* b, DType dt, int arg, const char* what) {
  if (!a || !b) return;
  THC_ARG_CHECK(a != b && (!spans_meet(a, dt, b, dt) || !tensor_is_contiguous(a) || !tensor_is_contiguous(b)), arg, "%s share memory", what);
}

void layer_norm_grad(THCState* s, DType dt, AnyTensor* gradInput, AnyTensor* gradWeight, AnyTensor* gradBias, AnyTensor* input, AnyTensor* gradOutput,
                     AnyTensor* weight, double eps, int accumulate) {
  const AnyTensor* all[6] = {gradInput, gradWeight, gradBias, input, gradOutput, weight};
  check_same_gpu(s, 6, all);
  THC_ARG_CHECK(gradInput, 2, "no tensor for the input's gradient");
  THC_ARG_CHECK(has_elements(input), 5, "the input is empty");
  check_rows(input, 5);
  THC_ARG_CHECK(same_sizes(input, gradOutput), 6, "the output's gradient has other sizes than the input");
  THC_ARG_CHECK(eps >= 0, 8, "eps is negative");
  const int64_t dim = input->size[input->nDimension - 1];
  if (weight) check_columns(weight, dim, 7, "weights");
  THC_ARG_CHECK(gradInput != weight, 2, "the input's gradient may not be the weight");
  AnyTensor* sums[2] = {gradWeight, gradBias};
  for (int k = 0; k < 2; ++k) {
    AnyTensor* t = sums[k];
    if (!t) continue;
    THC_ARG_CHECK(t != gradInput && t != input && t != gradOutput && t != weight, 3 + k, "a gradient of columns may not be another operand");
    THC_ARG_CHECK(t->nDimension <= kMaxDims, 3 + k, "%s", kDimWarning);
    if (accumulate) check_columns(t, dim, 3 + k, "sums to be added to");
  }
  THC_ARG_CHECK(!gradWeight || gradWeight != gradBias, 4, "the gradients of weight and bias are one tensor");
  // all are resized before any address is taken: they may share a storage that grows
  tensor_resize_as(s, gradInput, input, dt);
  const long size = (long)dim;
  for (int k = 0; k < 2; ++k) {
    AnyTensor* t = sums[k];
    if (t && tensor_numel(t) != dim) tensor_resize_nd(s, t, 1, &size, nullptr, dt);
    if (t) THC_ARG_CHECK(!overlapping(tensor_layout(t)), 3 + k, "elements of the gradient overlap");
  }
  check_apart(gradWeight, gradBias, dt, 4, "the gradients of weight and bias");
  check_apart(gradWeight, gradInput, dt, 3, "the gradients of weight and input");
  check_apart(gradBias, gradInput, dt, 4, "the gradients of bias and input");
  note_stream_use(s, {gradInput, gradWeight, gradBias, input, gradOutput, weight});
  if (dt == DType::F32) run_grad<float>(s, dt, gradInput, gradWeight, gradBias, input, gradOutput, weight, (float)eps, accumulate != 0);
  else run_grad<__half>(s, dt, gradInput, gradWeight, gradBias, input, gradOutput, weight, (float)eps, accumulate != 0);
}

}  // namespace
}  // namespace thc

#define TN(x) reinterpret_cast<thc::AnyTensor*>(x)
#define THC_AMD_DEFINE_LAYER_NORM(Tensor, DT)                                                                                              \
  THC_API void Tensor##_layerNorm(THCState* s, Tensor* self, Tensor* input, Tensor* weight, Tensor* bias, double eps) {                    \
    THC_GUARD_ALL(thc::layer_norm(s, DT, TN(self), TN(input), TN(weight), TN(bias), eps))                                                  \
  }                                                                                                                                        \
  THC_API void Tensor##_layerNormGrad(THCState* s, Tensor* gradInput, Tensor* gradWeight, Tensor* gradBias, Tensor* input,                \
                                      Tensor* gradOutput, Tensor* weight, double eps, int accumulate) {                                    \
    THC_GUARD_ALL(thc::layer_norm_grad(s, DT, TN(gradInput), TN(gradWeight), TN(gradBias), TN(input), TN(gradOutput), TN(weight), eps, accumulate)) \
  }
THC_AMD_DEFINE_LAYER_NORM(THCudaTensor, thc::DType::F32)
THC_AMD_DEFINE_LAYER_NORM(THCudaHalfTensor, thc::DType::F16)
