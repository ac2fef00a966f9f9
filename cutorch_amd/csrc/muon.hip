// Newton-Schulz orthogonalisation of matrices, and the optimizer whose step it is.
//
//   orthogonalize   X = G / (|G| + eps);  A = X X', B = b A + c A A, X = a X + B X, `steps` times, the shorter side first
//   muon            m = beta m + g;  u = g + beta m (or m);  p = p (1 - lr decay) - rate orthogonalize(u)
//
// The products run on the matrix cores in half precision, every factor as a sum of two halves (x = h + l, 22 bits where a float has 24): h h' + h l' + l h'
// is about as exact as a product of floats (against 64 bits after five steps 0.4 to 2.5 times as far, figures at chain_of), at a third of the
// halves' rate, where float products have a ninth of it (1190 and 126 TFLOP/s in products of that size). One half alone would leave 1e-3 to 5e-3. Sums are in float throughout, the norm's in 64 bits.
// Singular values of X stay below 1.21 once they are at most 1 (a s + b s^3 + c s^5 on 0 ... 1.21), so no element of X, A and B leaves
// +-1.21, +-1.46, +-2.81, nor P = a + B, P P' and P P' P'' +-a, +-a^2 and +-a^3, and each is held times a power of two that brings its usual size to
// where halves are exact, and its largest below their largest: S for X, 2^14 for A and P A, 2^13 for B and P, 2^12 and 2^10 for P P' and P P' P''.
#include <algorithm>
#include <cmath>
#include <type_traits>
#include <vector>

#include "training.hpp"

namespace thc {
namespace {

using std::integral_constant;

constexpr float kA = 3.4445f, kB = -4.7750f, kC = 2.0315f;
constexpr float kScaleA = 16384.f, kScaleB = 8192.f;

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef float acc16 __attribute__((ext_vector_type(16)));
typedef unsigned uint4v __attribute__((ext_vector_type(4)));

// A matrix of R rows and K columns as the products read it: rows of blocks of 32 columns, each block the 32 upper halves and the 32 lower ones,
// 128 bytes. Columns up to the next multiple of 32 hold zeros.
constexpr int kBlockK = 32, kBlockBytes = 128, kLower = 64;
__host__ __device__ constexpr int64_t blocks_of(int64_t k) { return (k + kBlockK - 1) / kBlockK; }
__host__ __device__ constexpr int64_t row_bytes(int64_t k) { return blocks_of(k) * kBlockBytes; }
__device__ __forceinline__ int64_t split_at(int64_t row, int32_t column, int64_t rowBytes) {
  return row * rowBytes + (column >> 5) * kBlockBytes + (column & 31) * 2;      // of the upper half; the lower one kLower bytes on
}

// `batch` matrices of m x n, m <= n, X short side first; `tall`: their tensors have n rows and m columns.
struct Matrix {
  char* work;                  // X, X', the next X, the next X', and two planes of m x m, or four, of each one
  const void* in;              // what is orthogonalised, or the gradient
  void* out;                   // what the result goes to, or the parameter
  float *momentum, *master;    // of the optimizer
  int32_t m, n, batch;
  uint32_t tall, norms;        // norms: the first of its parts of sums of squares
  float scale, rate;
};
__host__ __device__ inline int64_t plane_x(const Matrix& a) { return a.m * row_bytes(a.n); }
__host__ __device__ inline int64_t plane_t(const Matrix& a) { return a.n * row_bytes(a.m); }
__host__ __device__ inline int64_t plane_a(const Matrix& a) { return a.m * row_bytes(a.m); }
// Where n = r m is long, several steps read X once: P = a + B takes A on to the next step's, P A P, as well as X, and what X is multiplied by is those
// steps' P P' P''. In units of m^3, five steps cost 7.5 r + 2.5 one by one, 4.5 r + 5.5 as 2 + 2 + 1 and 3 r + 7 as 3 + 2. us, one by one and in these
// two ways: 8192 x 2048 2023, 1612, 1407; 1024 x 4096 489, 431, 407; eight of these 2455, 1923, 1680; 2048 x 4096 1187, 1119, 1085; 1024 x 2048 343, 345, 348 (more
// launches); 256 x 512 141, 145, 152; 1024 x 1536 298, 314, 325; 4096 x 4096 4046, 4124, 4160.
// (A rule on each matrix alone: its bits do not depend on what else a call has.)
__host__ __device__ inline bool is_long(const Matrix& a) { return a.n / 2 >= a.m; }
__host__ __device__ inline int64_t work_bytes(const Matrix& a) { return 2 * (plane_x(a) + plane_t(a)) + (is_long(a) ? 4 : 2) * plane_a(a); }

constexpr int kMatrices = 48;
struct Group {
  Matrix matrix[kMatrices];
  uint32_t first[kMatrices + 1];      // the first workgroup of each
  int32_t count;
};
static_assert(sizeof(Group) + 64 <= 4096, "kernel arguments");
struct Place {
  Matrix a;
  uint32_t index;      // of the workgroup within one matrix
  int32_t batch;
};
// Workgroups go to the eight dies in turn: of every 512 (what the chip has at a time), and of what is left, those of one die get neighbouring numbers, so
// that what they read in common comes from its own cache. (All of a launch in eight runs would leave dies idle whose matrices have shorter sums.)
constexpr uint32_t kDies = 8, kRound = 512;
__device__ __forceinline__ uint32_t by_die(uint32_t block, uint32_t blocks) {
  const uint32_t first = block / kRound * kRound, count = min(kRound, blocks - first), at = block - first;
  const uint32_t each = count / kDies, more = count % kDies, die = at % kDies;
  return first + die * each + min(die, more) + at / kDies;
}
// The matrix of this workgroup, `each` workgroups (by the matrix) for one of a batch.
template <typename F>
__device__ __forceinline__ Place place_of(const Group& g, uint32_t block, F each) {
  // (a lane looks at a matrix: one after another they would wait for the arguments a time each)
  static_assert(kMatrices <= 64, "a lane each");
  const int lane = threadIdx.x & 63;
  const uint32_t next = g.first[min(lane, kMatrices - 1) + 1];
  const int k = __popcll(__ballot(lane + 1 < g.count && block >= next));
  Place p{g.matrix[k], block - g.first[k], 0};
  const uint32_t n = each(p.a);
  p.batch = (int32_t)(p.index / n);
  p.index -= p.batch * n;
  return p;
}

// ------------------------------------------------------------ norms, planes --
constexpr int kNormPart = 16384;      // elements a workgroup
__host__ __device__ inline uint32_t norm_parts(const Matrix& a) { return (uint32_t)(((int64_t)a.m * a.n + kNormPart - 1) / kNormPart); }

struct Update {
  float beta, gradScale, keep, eps;
  int32_t nesterov;
};

// Eight neighbouring elements of a tensor, or as many as there are and zeros.
template <typename T>
__device__ __forceinline__ void load_values(const T* at, int64_t count, float (&v)[8]) {
  if (count >= 8) {
    constexpr int N = 16 / sizeof(T);
#pragma unroll
    for (int k = 0; k < 8 / N; ++k) {
      const Pack<T, N> t = load_pack_unaligned<false, Pack<T, N>>(at + k * N);
#pragma unroll
      for (int e = 0; e < N; ++e) v[k * N + e] = Cvt<T>::up(t.v[e]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < count ? Cvt<T>::up(at[e]) : 0.f;
  }
}
__device__ __forceinline__ void store_values(float* at, int64_t count, const float (&v)[8]) {
  if (count >= 8) {
#pragma unroll
    for (int k = 0; k < 2; ++k) store_pack_unaligned<false>(at + k * 4, Pack<float, 4>{v[k * 4], v[k * 4 + 1], v[k * 4 + 2], v[k * 4 + 3]});
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < count) at[e] = v[e];
  }
}

__device__ __forceinline__ void store_values(__half* at, int64_t count, const float (&v)[8]) {
  Pack<__half, 8> t;
#pragma unroll
  for (int e = 0; e < 8; ++e) t.v[e] = rounded<__half>(v[e]);
  if (count >= 8) {
    store_pack_unaligned<false>(at, t);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < count) at[e] = t.v[e];
  }
}

// The sum of squares of a part of a matrix, in 64 bits; the optimizer's momentum on the way.
template <typename T, bool MUON>
__global__ __launch_bounds__(kBlock) void norm_kernel(Group g, Update h, double* parts) {
  __shared__ double lds[kBlock / 64];
  const Place p = place_of(g, blockIdx.x, [](const Matrix& a) { return norm_parts(a); });
  const int64_t size = (int64_t)p.a.m * p.a.n, from = (int64_t)p.index * kNormPart, to = min(size, from + kNormPart);
  const T* in = static_cast<const T*>(p.a.in) + p.batch * size;
  float* momentum = MUON ? p.a.momentum + p.batch * size : nullptr;
  double sum = 0;
  constexpr int U = 2;
  for (int64_t i = from + threadIdx.x * 8; i < to; i += U * kBlock * 8) {
    float u[U][8], m[U][8];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int64_t at = i + k * kBlock * 8;
      if (at < to) load_values(in + at, to - at, u[k]);
      if (MUON && at < to) load_values(momentum + at, to - at, m[k]);
    }
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int64_t at = i + k * kBlock * 8;
      if (at >= to) continue;
      if constexpr (MUON) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float grad = u[k][e] * h.gradScale;
          m[k][e] = __builtin_fmaf(m[k][e], h.beta, grad);
          u[k][e] = h.nesterov ? __builtin_fmaf(m[k][e], h.beta, grad) : m[k][e];
        }
        store_values(momentum + at, to - at, m[k]);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) sum += (double)u[k][e] * u[k][e];      // (zeros behind the end)
    }
  }
  for (int d = 32; d >= 1; d >>= 1) sum += __shfl_xor(sum, d);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kBlock / 64; ++w) sum += lds[w];
    parts[blockIdx.x] = sum;
  }
}

// What elements are multiplied by: their scale over the norm, which may lie beyond the floats where elements are near their ends. (Powers of two round
// nothing.)
struct Factor {
  float first, second;
  __device__ __forceinline__ Factor(float scale, double sum, float eps) : Factor((double)scale / (sqrt(sum) + (double)eps)) {}
  __device__ __forceinline__ explicit Factor(double f) {
    first = f > 0x1p100 ? 0x1p64f : f < 0x1p-100 ? 0x1p-64f : 1.f;
    second = (float)(f / (double)first);
  }
  __device__ __forceinline__ float operator()(float x) const { return x * first * second; }
};

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef float float2v __attribute__((ext_vector_type(2)));
// Two elements as upper and lower halves. What is left of one is exact. (The operation before must not become one with the rounding to half: it would round
// once there and twice for the lower half, which now and then then goes with another upper one.)
__device__ __forceinline__ void split(float x, float y, half2v& h, half2v& l) {
  asm("" : "+v"(x), "+v"(y));
  h = __builtin_convertvector(float2v{x, y}, half2v);
  float2v left;
  asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(left[0]) : "v"(h), "v"(x));
  asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(left[1]) : "v"(h), "v"(y));
  l = __builtin_convertvector(left, half2v);
}
template <typename V, int N>
__device__ __forceinline__ void split(const float (&x)[N], V& h, V& l) {
#pragma unroll
  for (int e = 0; e < N; e += 2) {
    half2v a, b;
    split(x[e], x[e + 1], a, b);
    h[e] = a[0];
    h[e + 1] = a[1];
    l[e] = b[0];
    l[e + 1] = b[1];
  }
}
// Eight neighbouring elements of a plane.
struct Eight {
  half8 h, l;
};
__device__ __forceinline__ Eight load_eight(const char* at) { return Eight{*reinterpret_cast<const half8*>(at), *reinterpret_cast<const half8*>(at + kLower)}; }
__device__ __forceinline__ void store_eight(char* at, const float (&v)[8]) {
  half8 h, l;
  split(v, h, l);
  *reinterpret_cast<half8*>(at) = h;
  *reinterpret_cast<half8*>(at + kLower) = l;
}

// A tile of 64 x 64 elements of the tensor into both planes, over the norm.
__host__ __device__ inline uint32_t tiles64(const Matrix& a) { return (uint32_t)(((a.m + 63) / 64) * (int64_t)((a.n + 63) / 64)); }
template <typename T, bool MUON>
__global__ __launch_bounds__(kBlock) void split_kernel(Group g, Update h, const double* parts) {
  __shared__ float tile[64][65];
  __shared__ double lds[kBlock / 64];
  const Place p = place_of(g, blockIdx.x, [](const Matrix& a) { return tiles64(a); });
  const Matrix& a = p.a;
  const int64_t size = (int64_t)a.m * a.n;
  // the norm, from its parts
  const uint32_t count = norm_parts(a);
  const double* mine = parts + a.norms + (int64_t)p.batch * count;
  double sum = 0;
  for (uint32_t i = threadIdx.x; i < count; i += kBlock) sum += mine[i];
  for (int d = 32; d >= 1; d >>= 1) sum += __shfl_xor(sum, d);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = sum;
  __syncthreads();
  sum = 0;
  for (int w = 0; w < kBlock / 64; ++w) sum += lds[w];
  const Factor factor(a.scale, sum, h.eps);
  const int32_t rows = a.tall ? a.n : a.m, cols = a.tall ? a.m : a.n, across = (cols + 63) / 64;
  const int32_t r0 = (int32_t)(p.index / across) * 64, c0 = (int32_t)(p.index % across) * 64;
  const T* in = static_cast<const T*>(a.in) + p.batch * size;
  const float* momentum = MUON ? a.momentum + p.batch * size : nullptr;
  char *work = a.work + p.batch * work_bytes(a), *byRow = a.tall ? work + plane_x(a) : work, *byColumn = a.tall ? work : work + plane_x(a);
  const int64_t rowBytes = row_bytes(cols), columnBytes = row_bytes(rows);
  const int32_t colEnd = (int32_t)blocks_of(cols) * kBlockK, rowEnd = (int32_t)blocks_of(rows) * kBlockK;
  // thread t has eight columns of rows t / 8 and t / 8 + 32, then eight rows of such columns
  const int32_t eighth = (threadIdx.x & 7) * 8, line = threadIdx.x >> 3;
#pragma unroll
  for (int k = 0; k < 64; k += 32) {
    const int32_t r = r0 + line + k, c = c0 + eighth;
    float u[8] = {};
    if (r < rows && c < cols) {
      const int64_t at = (int64_t)r * cols + c;
      load_values(in + at, cols - c, u);
      if constexpr (MUON) {
        float m[8];
        load_values(momentum + at, cols - c, m);
#pragma unroll
        for (int e = 0; e < 8; ++e) u[e] = h.nesterov ? __builtin_fmaf(m[e], h.beta, u[e] * h.gradScale) : m[e];
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      u[e] = factor(u[e]);
      if (c + e >= cols) u[e] = 0.f;
      tile[line + k][eighth + e] = u[e];
    }
    if (r < rows && c < colEnd) store_eight(byRow + split_at(r, c, rowBytes), u);
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 64; k += 32) {
    const int32_t c = c0 + line + k, r = r0 + eighth;
    float u[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) u[e] = r + e < rows ? tile[eighth + e][line + k] : 0.f;
    if (c < cols && r < rowEnd) store_eight(byColumn + split_at(c, r, columnBytes), u);
  }
}

// ----------------------------------------------------------------- products --
// C = P Q', P and Q in the split layout: a workgroup has a tile of 128 x 128, each of its four waves 64 x 64 of that as 2 x 2 products of
// 32 x 32. A block of 32 columns of both operands, upper and lower halves, is 32 KiB of LDS; the next one is on its way there while one is
// multiplied, and there is room for two workgroups a CU. Bound by the matrix cores' power: 1024 tiles of 4096 columns 354 to 364 us
// with what becomes of them, 1150 TFLOP/s of halves,
// with the cores busy in 60 % of the cycles at 1.9 GHz; a library's product of halves of that size reaches 1190. A row's eight 16-byte pieces lie in the order of their number xor half the row's, so that
// sixteen lanes that read the same piece of neighbouring rows meet all banks. (Blocks of 16 columns, four of which are on their way: 5 % slower, as
// waves meet at twice as many barriers.)
// Few matrices of some hundred rows would leave most CUs idle with that: they take tiles of 64 x 64, a wave's part 32 x 32, four blocks in LDS. The
// sums of an element are the same ones.
constexpr int kTile = 128, kSmallTile = 64;
__host__ __device__ inline int32_t tiles_of(int32_t n, int32_t tile) { return (n + tile - 1) / tile; }

__device__ __forceinline__ uint4v resource(const void* p, uint32_t bytes) {
  const uint64_t a = reinterpret_cast<uint64_t>(p);
  uint4v r;
  r[0] = __builtin_amdgcn_readfirstlane((uint32_t)a);
  r[1] = __builtin_amdgcn_readfirstlane((uint32_t)(a >> 32) & 0xffff);
  r[2] = __builtin_amdgcn_readfirstlane(bytes);
  r[3] = 0x00020000;
  return r;
}
// 16 bytes for each lane from resource + lane's offset + offset into LDS, a lane after another from `lds` on. Not waited for.
__device__ __forceinline__ void load_to_lds(uint4v from, uint32_t laneOffset, uint32_t offset, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(lds), "v"(laneOffset), "s"(from), "s"(offset) : "memory");
}
// Until at most N of this wave's loads are on their way, then until all waves are there.
template <int N>
__device__ __forceinline__ void wait_loads_and_barrier() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

struct Operand {
  const char* rows;      // of the tile's first row
  int64_t rowBytes;
  int32_t count;         // rows from there on
};
// The sum over blocks of 32 columns is one of up to eight sums of equal parts, added up in their order: parts that several workgroups make come to the
// same bits as those that one makes, so that a matrix's result does not depend on what else a call has. As many as give each CU two workgroups
// where a matrix has few tiles.
__host__ __device__ inline int32_t sum_parts(int32_t blocks, uint32_t tiles) {
  const int32_t most = tiles <= 256 ? 512 / (int32_t)tiles : 8;
  return max(1, min(blocks / 16, min(most, 8)));
}
__host__ __device__ inline int32_t part_begin(int32_t blocks, int32_t parts, int32_t k) { return (int32_t)((int64_t)blocks * k / parts); }

template <int TILE>
struct Stages {
  static constexpr int kCount = TILE == kTile ? 2 : 4, kOperand = TILE * kBlockBytes, kBytes = 2 * kOperand;
};
// Adds the parts first ... last - 1 of `parts` to `total`, products of 32 x 32 of which a wave has W x W.
template <int TILE, int W = TILE / 64>
__device__ __forceinline__ void product(const Operand& P, const Operand& Q, int32_t blocks, int32_t parts, int32_t first, int32_t last, char* lds,
                                        acc16 (&total)[W][W]) {
  constexpr int kStages = Stages<TILE>::kCount, kStageBytes = Stages<TILE>::kBytes, kOperandBytes = Stages<TILE>::kOperand;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
  const uint4v fromP = resource(P.rows, (uint32_t)min(P.count, TILE) * (uint32_t)P.rowBytes), fromQ = resource(Q.rows, (uint32_t)min(Q.count, TILE) * (uint32_t)Q.rowBytes);
  // an operand's block is loads of a wave of 8 rows each; wave w has those with numbers w, w + 4, ...
  constexpr int U = TILE / 32;
  uint32_t offP[U], offQ[U];
#pragma unroll
  for (int q = 0; q < U; ++q) {
    const int32_t row = (q * 4 + wave) * 8 + (lane >> 3), piece = (lane & 7) ^ ((row >> 1) & 7);
    offP[q] = (uint32_t)min(row, P.count - 1) * (uint32_t)P.rowBytes + piece * 16;
    offQ[q] = (uint32_t)min(row, Q.count - 1) * (uint32_t)Q.rowBytes + piece * 16;
  }
  auto load = [&](int32_t k, uint32_t stage) {
#pragma unroll
    for (int q = 0; q < U; ++q) {
      const uint32_t to = __builtin_amdgcn_readfirstlane(base + stage * kStageBytes + (q * 4 + wave) * 1024);
      load_to_lds(fromP, offP[q], k * kBlockBytes, to);
      load_to_lds(fromQ, offQ[q], k * kBlockBytes, to + kOperandBytes);
    }
  };
  const int rowP = ((wave >> 1) * (TILE / 2) + (lane & 31)) * kBlockBytes, rowQ = ((wave & 1) * (TILE / 2) + (lane & 31)) * kBlockBytes + kOperandBytes;
  acc16 acc[W][W] = {};
  int32_t part = first, until = part_begin(blocks, parts, first + 1);
  const int32_t begin = part_begin(blocks, parts, first), end = part_begin(blocks, parts, last);
  // products into the same sums lie W x W apart
  auto products = [&](const half8 (&p)[W], const half8 (&q)[W]) {
#pragma unroll
    for (int i = 0; i < W; ++i)
#pragma unroll
      for (int j = 0; j < W; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(p[i], q[j], acc[i][j], 0, 0, 0);
  };
  // 16 of a block's columns
  struct Half {
    half8 ph[W], pl[W], qh[W], ql[W];
  };
  auto read = [&](uint32_t stage, int s, Half& b) {
    const char *fp = lds + stage * kStageBytes + rowP, *fq = lds + stage * kStageBytes + rowQ;
    const int swizzle = (lane >> 1) & 7, high = ((2 * s + (lane >> 5)) ^ swizzle) * 16, low = ((4 + 2 * s + (lane >> 5)) ^ swizzle) * 16;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      b.ph[i] = *reinterpret_cast<const half8*>(fp + i * 32 * kBlockBytes + high);
      b.qh[i] = *reinterpret_cast<const half8*>(fq + i * 32 * kBlockBytes + high);
      b.ql[i] = *reinterpret_cast<const half8*>(fq + i * 32 * kBlockBytes + low);
      b.pl[i] = *reinterpret_cast<const half8*>(fp + i * 32 * kBlockBytes + low);
    }
  };
  auto multiply = [&](const Half& b) {
    products(b.ph, b.qh);
    products(b.ph, b.ql);
    products(b.pl, b.qh);
  };
  auto next_part = [&](int32_t k) {
    if (k != until) return;
    until = part_begin(blocks, parts, ++part + 1);
#pragma unroll
    for (int q = 0; q < W * W; ++q) {
      total[q / W][q % W] += acc[q / W][q % W];
      acc[q / W][q % W] = acc16{};
    }
  };
  auto after = [](uint32_t stage) { return stage == kStages - 1 ? 0 : stage + 1; };
  uint32_t stage = 0;
  if constexpr (TILE == kTile) {
    if (begin < end) load(begin, 0);
    for (int32_t k = begin; k < end; ++k) {
      next_part(k);
      // this block is there; the one that is asked for now takes the room that was read last before the barrier
      wait_loads_and_barrier<0>();
      if (k + 1 < end) load(k + 1, after(stage));
      // all of the block's operands are asked for before the first product (2 % quicker than by halves)
      Half one, two;
      read(stage, 0, one);
      read(stage, 1, two);
      stage = after(stage);
      __builtin_amdgcn_sched_barrier(0);
      multiply(one);
      multiply(two);
    }
  } else {
    // Half a block is read while the one before it is multiplied: a CU often has no other workgroup that would do so (one matrix of 1024 x 1024 267 -> 252 us; in
    // large tiles 1 to 4 % slower, a whole block ahead 3 % slower). A block's room is free when all waves have its second half.
    auto lds_is_here = [] {      // (known to the compiler, which otherwise waits for the reads behind those as well)
      __builtin_amdgcn_s_waitcnt(0xc07f);
      __builtin_amdgcn_sched_barrier(0);
    };
#pragma unroll
    for (int k = 0; k < kStages; ++k)
      if (begin + k < end) load(begin + k, k);
    if (begin + kStages <= end) wait_loads_and_barrier<2 * U * (kStages - 1)>();
    else wait_loads_and_barrier<0>();
    Half one, two;
    read(0, 0, one);
    for (int32_t k = begin; k < end; ++k) {
      next_part(k);
      lds_is_here();
      read(stage, 1, two);
      __builtin_amdgcn_sched_barrier(0);
      multiply(one);
      __builtin_amdgcn_sched_barrier(0);
      lds_is_here();
      if (k + 1 < end) {
        // (of the next block's loads and those behind it, the latter may be on their way)
        if (k + kStages <= end) wait_loads_and_barrier<2 * U * (kStages - 2)>();
        else wait_loads_and_barrier<0>();
        if (k + kStages < end) load(k + kStages, stage);
        stage = after(stage);
        read(stage, 0, one);
        __builtin_amdgcn_sched_barrier(0);
      }
      multiply(two);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
#pragma unroll
  for (int q = 0; q < W * W; ++q) total[q / W][q % W] += acc[q / W][q % W];
}

// What becomes of the products' sums, with the planes of m x m by number:
//   kGram         to = X X'
//   kPolynomial   to = b from + c from from + own (on the diagonal)
//   kProduct      to = from with
//   kStep, kLast  the next X = own X + from X
enum Op { kGram, kPolynomial, kProduct, kStep, kLast };
struct Way {
  int turn;               // which of the two pairs of planes X is in
  int from, with, to;
  float own, factor;      // factor: of the sums, from the factors' scales to the result's (kProduct, kStep, kLast)
};

__host__ __device__ inline uint32_t symmetric_tiles(int32_t t) { return (uint32_t)(t * (int64_t)(t + 1) / 2); }
__host__ __device__ inline uint32_t product_tiles(const Matrix& a, bool symmetric, int32_t tile = kTile) {
  return symmetric ? symmetric_tiles(tiles_of(a.m, tile)) : (uint32_t)(tiles_of(a.m, tile) * (int64_t)tiles_of(a.n, tile));
}

// Tiles in an order in which neighbours share operands: bands of eight rows of them, column by column.
constexpr int kBand = 8;
__device__ __forceinline__ void tile_at(uint32_t index, int32_t down, int32_t across, int32_t& ti, int32_t& tj) {
  const uint32_t band = index / (uint32_t)(kBand * across), rest = index - band * (kBand * across), rows = min(kBand, down - (int32_t)band * kBand);
  ti = (int32_t)(band * kBand + rest % rows);
  tj = (int32_t)(rest / rows);
}
// The same for tiles on and above the diagonal: a band begins with its triangle.
__device__ __forceinline__ void symmetric_tile_at(uint32_t index, int32_t tiles, int32_t& ti, int32_t& tj) {
  int32_t first = 0;
  for (;; first += kBand) {
    const int32_t rows = min(kBand, tiles - first);
    const uint32_t triangle = symmetric_tiles(rows), count = triangle + (uint32_t)rows * (uint32_t)(tiles - first - rows);
    if (index < count) {
      if (index < triangle) {
        int32_t column = 0;
        while (index > (uint32_t)column) index -= ++column;
        ti = first + (int32_t)index;
        tj = first + column;
      } else {
        index -= triangle;
        ti = first + (int32_t)(index % rows);
        tj = first + rows + (int32_t)(index / rows);
      }
      return;
    }
    index -= count;
  }
}

// One of a step's products and what is made of it. Those of m x m are symmetric (their factors are polynomials of one A): tiles above the diagonal go to
// both places. The last step's result goes to the tensor, or into the parameter. The sums pass through LDS, so that memory sees whole packs of
// neighbouring elements in both directions.
// The last tiles, which would leave much of the chip idle, are cut into the parts of their sums: a workgroup for each leaves its sums in memory, and a
// launch behind this one (JOIN) adds them up and goes on from there.
struct Tail {
  uint32_t whole;      // tiles before them
  int32_t parts;       // 1: none are cut
  acc16* sums;         // of each part: the products of each of 256 lanes
};
template <int OP, typename T, bool MUON, bool JOIN, int TILE>
__global__ __launch_bounds__(256, 2) void product_kernel(Group g, Update h, Way way, Tail tail) {
  // (the joining launch has a workgroup for each wave's quarter of a large tile: one CU alone would wait long for what all parts left)
  constexpr int W = TILE / 64, kQuarters = JOIN ? W * W : 1, kSpan = JOIN ? 64 : TILE;
  constexpr int kStride = kSpan + 4;      // floats: columns of sums, four rows at once, meet all banks
  constexpr int kSums = kSpan * kStride * 4, kBlocks = JOIN ? 0 : Stages<TILE>::kCount * Stages<TILE>::kBytes;
  __shared__ __attribute__((aligned(128))) char lds[kSums > kBlocks ? kSums : kBlocks];
  constexpr bool kSymmetric = OP != kStep && OP != kLast;
  const uint32_t unit = JOIN ? blockIdx.x / kQuarters : by_die(blockIdx.x, gridDim.x), quarter = blockIdx.x % kQuarters;
  const bool cut = !JOIN && unit >= tail.whole;
  // (of the tiles that are cut, the first parts of all, then the second ones, ...: a die's workgroups read less that way, 1024 x 4096 halves 395 -> 386 us)
  const uint32_t rest = (gridDim.x - tail.whole) / (uint32_t)tail.parts;
  const uint32_t tile = JOIN ? tail.whole + unit : cut ? tail.whole + (unit - tail.whole) % rest : unit;
  const Place p = place_of(g, tile, [](const Matrix& a) { return product_tiles(a, kSymmetric, TILE); });
  const Matrix& a = p.a;
  char* work = a.work + p.batch * work_bytes(a);
  const int64_t px = plane_x(a), pt = plane_t(a);
  char *x = work + way.turn * (px + pt), *t = x + px, *xn = work + (way.turn ^ 1) * (px + pt), *tn = xn + px, *square = work + 2 * (px + pt);
  const char *left = square + way.from * plane_a(a), *right = square + way.with * plane_a(a);
  char* to = square + way.to * plane_a(a);
  const int64_t bytesM = row_bytes(a.m), bytesN = row_bytes(a.n);
  const bool flipped = OP == kLast && a.tall;      // the tensor's rows are the longer side: its tile is the product's transpose
  const int32_t rows = flipped ? a.n : a.m, cols = kSymmetric || flipped ? a.m : a.n;
  int32_t ti, tj;
  if constexpr (kSymmetric) symmetric_tile_at(p.index, tiles_of(a.m, TILE), ti, tj);
  else tile_at(p.index, tiles_of(rows, TILE), tiles_of(cols, TILE), ti, tj);
  const int32_t i0 = ti * TILE + (int32_t)(quarter >> 1) * kSpan, j0 = tj * TILE + (int32_t)(quarter & 1) * kSpan;
  if (JOIN && (i0 >= rows || j0 >= cols || (kSymmetric && i0 > j0))) return;
  // Symmetric products hold each of their elements once: above the diagonal. (Element (j, i) sums its lower halves' products the other way round.)
  const bool diagonal = kSymmetric && i0 == j0;
  const char *from, *with;
  int64_t bytesK;
  if constexpr (OP == kGram) {
    from = with = x;
    bytesK = bytesN;
  } else {
    bytesK = bytesM;
    from = flipped ? t : left;
    with = kSymmetric ? right : flipped ? left : t;
  }
  const Operand P{from + i0 * bytesK, bytesK, rows - i0}, Q{with + j0 * bytesK, bytesK, cols - j0};
  // The sums as columns: a lane has column `lane % 32` of each 32 x 32 product, four rows in a row of each eight.
  float* sums = reinterpret_cast<float*>(lds);
  // (four rows of a column stay side by side; eight columns on they have changed places, so that sixteen lanes that have eight columns each meet all banks)
  auto spot = [&](int i, int j) { return sums + j * kStride + (i ^ ((j >> 3 & 15) << 2)); };
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  auto keep = [&](int down, int over, const acc16& acc) {      // 32 x 32 at these times 32
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = down * 32 + r * 8 + (lane >> 5) * 4, j = over * 32 + (lane & 31);
      *reinterpret_cast<Pack<float, 4>*>(spot(i, j)) = Pack<float, 4>{acc[r * 4], acc[r * 4 + 1], acc[r * 4 + 2], acc[r * 4 + 3]};
    }
  };
  // Rows: a thread has eight columns of every kRows-th row. What goes into the result beside the products is asked for as early as there are registers for it:
  // before the products of small tiles, behind those of large ones.
  constexpr int kAcross = kSpan / 8, kRows = 256 / kAcross, kSteps = kSpan / kRows;
  constexpr bool kBased = OP == kPolynomial || OP == kStep || OP == kLast;
  const int32_t jt = (threadIdx.x % kAcross) * 8, it = threadIdx.x / kAcross, j = j0 + jt;
  const int32_t colEnd = (int32_t)blocks_of(cols) * kBlockK;
  Eight beside[kBased ? kSteps : 1] = {};
  float was[OP == kLast && MUON ? kSteps : 1][8];      // of the parameter
  const int64_t result = p.batch * ((int64_t)a.m * a.n) + j;
  auto ask = [&] {
    if constexpr (OP == kLast && MUON) {
#pragma unroll
      for (int u = 0; u < kSteps; ++u) {
        const int64_t at = result + (int64_t)min(i0 + it + u * kRows, rows - 1) * cols;
        if (a.master) load_values(a.master + at, cols - j, was[u]);
        else load_values(static_cast<const T*>(a.out) + at, cols - j, was[u]);
      }
    }
    if (!kBased || (OP != kPolynomial && way.own == 0)) return;
    const char* base = kSymmetric ? right : flipped ? t : x;
#pragma unroll
    for (int u = 0; u < kSteps; ++u)
      beside[kBased ? u : 0] = load_eight(base + split_at(min(i0 + it + u * kRows, rows - 1), min(j, colEnd - 8), kSymmetric || flipped ? bytesM : bytesN));
  };
  if constexpr (JOIN) {
    ask();
    // each of the four waves has one of the 2 x 2 products of 64 x 64
    constexpr int kEach = W * W * 256;
    const acc16* from16 = tail.sums + (int64_t)unit * tail.parts * kEach + (W == 2 ? wave * 256 + quarter * 64 : wave * 64) + lane;
    acc16 acc = {};
#pragma unroll 8
    for (int k = 0; k < tail.parts; ++k) acc += from16[k * kEach];
    keep(wave >> 1, wave & 1, acc);
  } else {
    const int32_t blocks = (int32_t)(bytesK / kBlockBytes), parts = sum_parts(blocks, product_tiles(a, kSymmetric)), part = cut ? (int32_t)((unit - tail.whole) / rest) : 0;
    acc16 acc[W][W] = {};
    if (TILE == kSmallTile && !cut) ask();
    product<TILE>(P, Q, blocks, parts, part, cut ? part + 1 : parts, lds, acc);
    if (cut) {
      acc16* to16 = tail.sums + ((int64_t)(tile - tail.whole) * tail.parts + part) * (W * W * 256) + threadIdx.x;
#pragma unroll
      for (int q = 0; q < W * W; ++q) to16[q * 256] = acc[q / W][q % W];
      return;
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < W * W; ++q) keep((wave >> 1) * W + q / W, (wave & 1) * W + q % W, acc[q / W][q % W]);
    if (TILE != kSmallTile) ask();
  }
  __syncthreads();
  // (few of these steps at a time where registers do not ask for them all: each of their instructions runs but a few times, and has to come from memory first)
#pragma unroll(kBased ? kSteps : 2)
  for (int u = 0; u < kSpan; u += kRows) {
    const int32_t i = i0 + it + u;
    const Eight& one = beside[kBased ? u / kRows : 0];
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float sum = *spot(it + u, jt + e);
      if (kSymmetric && diagonal && it + u > jt + e) sum = *spot(jt + e, it + u);
      if constexpr (OP == kGram) {
        v[e] = sum * (kScaleA / (a.scale * a.scale));
      } else if constexpr (OP == kProduct) {
        v[e] = sum * way.factor;
      } else {
        const float o = (float)one.h[e] + (float)one.l[e];
        if constexpr (OP == kPolynomial) v[e] = __builtin_fmaf(o, kB * (kScaleB / kScaleA), sum * (kC * kScaleB / (kScaleA * kScaleA))) + (i == j + e ? way.own * kScaleB : 0.f);
        else v[e] = __builtin_fmaf(o, way.own, sum * way.factor);
      }
      if (i >= rows || j + e >= cols) v[e] = 0.f;
    }
    if constexpr (OP == kLast) {
      if (i >= rows || j >= cols) continue;
      const int64_t at = result + (int64_t)i * cols;
      const float down = 1.f / a.scale;      // (a power of two)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if constexpr (MUON) v[e] = __builtin_fmaf(v[e] * down, -a.rate, was[u / kRows][e] * h.keep);
        else v[e] *= down;
      }
      if constexpr (MUON) {
        if (a.master) store_values(a.master + at, cols - j, v);
      }
      store_values(static_cast<T*>(a.out) + at, cols - j, v);
    } else {
      if (i < rows && j < colEnd) store_eight((OP == kStep ? xn : to) + split_at(i, j, OP == kStep ? bytesN : bytesM), v);
      if (!diagonal) {
#pragma unroll
        for (int e = 0; e < 8; ++e) *spot(it + u, jt + e) = v[e];
      }
    }
  }
  if constexpr (OP != kLast) {
    if (diagonal) return;
    __syncthreads();
    // and columns, in the same way
    char* mirrored = OP == kStep ? tn : to;
    const int32_t rowEnd = (int32_t)blocks_of(rows) * kBlockK, i = i0 + jt;
#pragma unroll 2
    for (int u = 0; u < kSpan; u += kRows) {
      const int32_t c = it + u;
      if (j0 + c >= cols || i >= rowEnd) continue;
      const Pack<float, 4> low = *reinterpret_cast<const Pack<float, 4>*>(spot(jt, c)), high = *reinterpret_cast<const Pack<float, 4>*>(spot(jt + 4, c));
      const float v[8] = {low.v[0], low.v[1], low.v[2], low.v[3], high.v[0], high.v[1], high.v[2], high.v[3]};
      store_eight(mirrored + split_at(j0 + c, i, bytesM), v);
    }
  }
}

// ---------------------------------------------------------- short matrices --
// Up to 128 rows: A and B are one tile each, and what bounds a step is how long its launches wait for memory one after another (12 matrices of 65 x 513: 17
// launches of 9 to 17 us each). A workgroup has a strip of 128 columns of X. It adds up the strips' shares of A, makes B of it by itself,
// takes its strip through the step and leaves the strip's share of the next A. Two steps
// a launch (three where results are only written as halves) where it takes A along, P A P: 12 of 65 x 513 floats took 98 us with a launch for each step and 82 so; 67 since strips
// begin without a launch for the norm and the kernels have 0.6 of the instructions. Of a launch's 49 thousand cycles for two steps a CU's four SIMDs have
// vector instructions for 21 thousand, matrix ones for 10, and LDS is read or written in 13: nine waves that wait for one another at barriers.
// One launch for all steps where X is a single strip, which makes each A from X.
// LDS: one plane for A, then B, then the new X, a second one for the strip's transpose, both split, rows of 16-byte pieces in the order of their
// number xor what brings sixteen rows to different banks.
// No launch makes the norm first: a strip begins over its own norm, by a power of two, and the step that adds up the shares knows all strips' norms.
constexpr int kShortThreads = 1024, kShort = 128, kStrip = 128;
__host__ __device__ inline bool is_short(const Matrix& a) { return a.m <= kShort; }
__host__ __device__ inline bool is_thin(const Matrix& a) { return a.m <= 32; }
__host__ __device__ inline bool is_alone(const Matrix& a) { return is_short(a) && a.n <= kStrip; }
__host__ __device__ inline int32_t strips_of(const Matrix& a) { return (a.n + kStrip - 1) / kStrip; }
__host__ __device__ inline int32_t bands_of(const Matrix& a) { return (a.m + 31) / 32; }
__host__ __device__ inline int64_t gram_bytes(const Matrix& a) { return (int64_t)bands_of(a) * bands_of(a) * 4096; }
// X', the strips' shares of A for this step and the next, their sum; the strips' sums of squares and the sum of those.
__host__ __device__ inline int64_t shares_end(const Matrix& a) { return plane_t(a) + (2 * (int64_t)strips_of(a) + 1) * gram_bytes(a); }
__host__ __device__ inline int64_t short_bytes(const Matrix& a) { return shares_end(a) + ((int64_t)strips_of(a) + 1 + 31) / 32 * 256; }
__host__ __device__ inline int short_lds(int bands) { return bands * 32 * 512 + kStrip * bands * 128; }

struct Plane {
  char* at;
  int rowBytes;      // a multiple of 128
  __device__ __forceinline__ int swizzle(int row) const { return (rowBytes & 128) ? row >> 1 & 7 : row & 15; }
  __device__ __forceinline__ char* piece(int row, int k) const { return at + row * rowBytes + ((k ^ swizzle(row)) << 4); }
};
// Four neighbouring elements of a plane: the lower halves' piece is the upper ones' with another bit of its number.
struct Fours {
  char* row;
  int piece;      // its place in the row, without that of the four in it
  __device__ __forceinline__ half4* upper(int at) const { return reinterpret_cast<half4*>(row + (piece ^ at)); }
  __device__ __forceinline__ half4* lower(int at) const { return upper(at ^ 64); }
  __device__ __forceinline__ void store(int at, const float (&x)[4]) const {
    half4 h, l;
    split(x, h, l);
    *upper(at) = h;
    *lower(at) = l;
  }
};
// 32 x 32 of P Q' over `blocks` blocks of 32 columns. Two sums side by side, and none in two products in a row (three: 3 % slower).
// `fine`: the lower halves' product too.
__device__ __forceinline__ acc16 small_product(const Plane& P, int i0, const Plane& Q, int j0, int blocks, bool fine) {
  int lane = threadIdx.x & 63;
  asm volatile("" : "+v"(lane));      // (addresses are made where they are used: kept through the steps they would be registers' spills)
  const int rowP = i0 + (lane & 31), rowQ = j0 + (lane & 31), pieceP = ((lane >> 5) ^ P.swizzle(rowP)) << 4, pieceQ = ((lane >> 5) ^ Q.swizzle(rowQ)) << 4;
  const char *atP = P.at + rowP * P.rowBytes, *atQ = Q.at + rowQ * Q.rowBytes;
  acc16 high, rest;
  // (the first products take their sums' zeros as a constant)
  auto add = [&](int at, const acc16& h, const acc16& r) {
    const half8 ph = *reinterpret_cast<const half8*>(atP + (pieceP ^ at)), pl = *reinterpret_cast<const half8*>(atP + (pieceP ^ at ^ 64));
    const half8 qh = *reinterpret_cast<const half8*>(atQ + (pieceQ ^ at)), ql = *reinterpret_cast<const half8*>(atQ + (pieceQ ^ at ^ 64));
    rest = __builtin_amdgcn_mfma_f32_32x32x16_f16(ph, ql, r, 0, 0, 0);
    high = __builtin_amdgcn_mfma_f32_32x32x16_f16(ph, qh, h, 0, 0, 0);
    rest = __builtin_amdgcn_mfma_f32_32x32x16_f16(pl, qh, rest, 0, 0, 0);
    if (fine) rest = __builtin_amdgcn_mfma_f32_32x32x16_f16(pl, ql, rest, 0, 0, 0);
  };
  add(0, acc16{}, acc16{});
  add(32, high, rest);
#pragma unroll 1
  for (int k = 1; k < blocks; ++k) {
    add(k * 128, high, rest);
    add(k * 128 + 32, high, rest);
  }
  return high + rest;
}
// Four lanes side by side that have a column of 4 x 4 each get a row each.
template <int CONTROL>
__device__ __forceinline__ float from_neighbour(float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CONTROL, 0xf, 0xf, true));
}
__device__ __forceinline__ void transpose4(float (&v)[4]) {
  const bool odd = threadIdx.x & 1, second = threadIdx.x & 2;
#pragma unroll
  for (int k = 0; k < 4; k += 2) {      // 2 x 2 blocks within themselves
    const float mine = odd ? v[k] : v[k + 1], theirs = from_neighbour<0xb1>(mine);
    (odd ? v[k] : v[k + 1]) = theirs;
  }
#pragma unroll
  for (int k = 0; k < 2; ++k) {         // and the two off the diagonal against each other
    const float mine = second ? v[k] : v[k + 2], theirs = from_neighbour<0x4e>(mine);
    (second ? v[k] : v[k + 2]) = theirs;
  }
}

// A workgroup's strip. Its sixteen waves have one of the 32 x 32 products each, of which there are 4 x 4 at most.
struct Strip {
  const Matrix& a;
  int bands, blocks, j0, lane, wave;      // blocks: of 32 columns in the strip
  Plane square, fresh, across;            // A or B; the new X in the same place; the strip's transpose
  __device__ __forceinline__ Strip(const Matrix& m, int strip, char* lds) : a(m) {
    bands = bands_of(m);
    j0 = strip * kStrip;
    blocks = (min(kStrip, m.n - j0) + 31) / 32;
    lane = threadIdx.x & 63;
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    square = Plane{lds, bands * 128};
    fresh = Plane{lds, 512};
    across = Plane{lds + bands * 32 * 512, bands * 128};
  }
  // f(its place) for this wave's product, of `down` x `over`, up to 4 each
  template <typename F>
  __device__ __forceinline__ void each(int down, int over, F f) const {
    const int ti = (wave * (over == 1 ? 256 : over == 2 ? 128 : over == 3 ? 86 : 64)) >> 8;
    if (ti < down) f(ti, wave - ti * over);
  }
  __device__ __forceinline__ int this_lane() const {
    int l = lane;
    asm volatile("" : "+v"(l));
    return l;
  }
  // f(e0, row, column) for the first of each four rows that a lane has of a product
  template <typename F>
  __device__ __forceinline__ void fours(int ti, int tj, F f) const {
    const int lane = this_lane();
#pragma unroll
    for (int q = 0; q < 4; ++q) f(q * 4, ti * 32 + q * 8 + (lane >> 5) * 4, tj * 32 + (lane & 31));
  }
  // The same as the transpose's row of that column holds them, the fours 16 bytes apart, and into it.
  __device__ __forceinline__ Fours turned(const Plane& plane, int ti, int tj) const {
    const int lane = this_lane(), row = tj * 32 + (lane & 31);
    return Fours{plane.at + row * plane.rowBytes + (lane >> 5) * 8, ((ti * 8) ^ plane.swizzle(row)) << 4};
  }
  __device__ __forceinline__ void store(const Plane& plane, int ti, int tj, const acc16& x) const {
    const Fours at = turned(plane, ti, tj);
#pragma unroll
    for (int q = 0; q < 4; ++q) at.store(q * 16, {x[q * 4], x[q * 4 + 1], x[q * 4 + 2], x[q * 4 + 3]});
  }
  // Sums as the products leave them to A.
  __device__ __forceinline__ void scaled(acc16& sums) const { sums *= kScaleA / (a.scale * a.scale); }
  // From A to B in the square.
  __device__ __forceinline__ void polynomial(acc16 sums) const {
    each(bands, bands, [&](int ti, int tj) { store(square, ti, tj, sums); });
    __syncthreads();
    each(bands, bands, [&](int ti, int tj) {
      const acc16 twice = small_product(square, ti * 32, square, tj * 32, bands, bands == 1);
#pragma unroll
      for (int e = 0; e < 16; ++e) sums[e] = __builtin_fmaf(sums[e], kB * (kScaleB / kScaleA), twice[e] * (kC * kScaleB / (kScaleA * kScaleA)));
    });
    __syncthreads();
    each(bands, bands, [&](int ti, int tj) { store(square, ti, tj, sums); });
    __syncthreads();
  }
  // The next X, times its scale and `factor`.
  __device__ __forceinline__ void step(acc16& x, float factor) const {
    each(bands, blocks, [&](int ti, int tj) {
      x = small_product(square, ti * 32, across, tj * 32, bands, bands == 1);
      const Fours at = turned(across, ti, tj);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const half4 h = *at.upper(q * 16), l = *at.lower(q * 16);
#pragma unroll
        for (int k = 0; k < 4; ++k) x[q * 4 + k] = __builtin_fmaf((float)h[k] + (float)l[k], kA, x[q * 4 + k] * (1.f / kScaleB)) * factor;
      }
    });
    __syncthreads();
  }
  // After a step, from its A and B to the next A, (a + B) A (a + B), and X to its place. (A and P A pass through the transpose's room.)
  __device__ __forceinline__ void turn(const acc16& x, acc16& sums) const {
    const Plane other{across.at, bands * 128};
#pragma unroll 1
    for (int k = 0; k < 2; ++k) {
      each(bands, bands, [&](int ti, int tj) { store(other, ti, tj, sums); });
      __syncthreads();
      each(bands, bands, [&](int ti, int tj) {
        const acc16 rest = small_product(square, ti * 32, other, tj * 32, bands, bands == 1);
#pragma unroll
        for (int e = 0; e < 16; ++e) sums[e] = __builtin_fmaf(sums[e], kA, rest[e] * (1.f / kScaleB));
      });
      __syncthreads();
    }
    each(bands, blocks, [&](int ti, int tj) { store(across, ti, tj, x); });
  }
  // X into both planes, then the strip's share of A.
  __device__ __forceinline__ void gram(const acc16& x, acc16& sums) const {
    each(bands, blocks, [&](int ti, int tj) {
      store(across, ti, tj, x);
      // rows, of which a lane has every eighth
      const int lane = this_lane(), row = ti * 32 + (lane >> 5) * 4 + (lane & 3);
      const Fours at{fresh.at + row * 512 + (lane & 4) * 2, ((tj * 8 + (lane >> 3 & 3)) ^ (row & 15)) << 4};
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        float four[4] = {x[q * 4], x[q * 4 + 1], x[q * 4 + 2], x[q * 4 + 3]};
        transpose4(four);
        Fours{at.row + q * 8 * 512, at.piece}.store((q & 1) * 128, four);      // (eight rows on, the swizzle has another bit)
      }
    });
    __syncthreads();
    each(bands, bands, [&](int ti, int tj) { sums = small_product(fresh, ti * 32, fresh, tj * 32, blocks, bands == 1); });
    __syncthreads();
  }
  // Element (row, column of the strip) of a matrix that begins at element `at` of its tensor; -1: there is none.
  __device__ __forceinline__ int64_t place(int64_t at, int i, int j) const {
    const int32_t column = j0 + j;
    if (i >= a.m || column >= a.n) return -1;
    return at + (a.tall ? (int64_t)column * a.m + i : (int64_t)i * a.n + column);
  }
  // The result to the tensor or into the parameter; `at`: of this matrix.
  template <typename T, bool MUON>
  __device__ __forceinline__ void emit(const acc16& x, const Update& h, int64_t at) const {
    const float down = 1.f / a.scale;
    each(bands, blocks, [&](int ti, int tj) {
      fours(ti, tj, [&](int e, int i, int j) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int64_t to = place(at, i + k, j);
          if (to < 0) continue;
          T* out = static_cast<T*>(a.out) + to;
          const float o = x[e + k] * down;
          if constexpr (MUON) {
            const float was = a.master ? a.master[to] : Cvt<T>::up(*out), is = __builtin_fmaf(o, -a.rate, was * h.keep);
            if (a.master) a.master[to] = is;
            *out = rounded<T>(is);
          } else {
            *out = rounded<T>(o);
          }
        }
      });
    });
  }
};

// The strip's transpose and its share of A into memory. Of each row 32 lanes have a piece, of which there are 32 at most.
constexpr int kStripLoads = kStrip * 32 / kShortThreads;
__device__ __forceinline__ void leave(const Strip& strip, const acc16& sums, char* work, uint32_t index, int turn) {
  const Matrix& a = strip.a;
  const int pieces = strip.bands * 8, rows = min(kStrip, a.n - strip.j0), piece = threadIdx.x & 31;
  uint4v* to = reinterpret_cast<uint4v*>(work + (int64_t)strip.j0 * strip.bands * 128);
#pragma unroll
  for (int q = 0; q < kStripLoads; ++q) {
    const int row = (threadIdx.x >> 5) + q * (kShortThreads / 32);
    if (row < rows && piece < pieces) to[row * pieces + piece] = *reinterpret_cast<const uint4v*>(strip.across.piece(row, piece));
  }
  acc16* share = reinterpret_cast<acc16*>(work + plane_t(a) + ((int64_t)turn * strips_of(a) + index) * gram_bytes(a));
  strip.each(strip.bands, strip.bands, [&](int ti, int tj) { share[(ti * strip.bands + tj) * 64 + strip.lane] = sums; });
}

// A strip's elements are at first multiplied by 2^this: S over their norm, or up to twice as much.
__device__ __forceinline__ int strip_exponent(double squares, float scale) {
  const int e = (int)(__double_as_longlong(squares) >> 52) - 1023;      // of the greatest power of two up to it
  return ilogbf(scale) - (squares > 0 ? e >> 1 : -150);
}
// What a strip's X then lacks to be over the whole norm, at most 1.
__device__ __forceinline__ float strip_factor(double norm, double squares, const Matrix& a) {
  return (float)ldexp((double)a.scale / norm, -strip_exponent(squares, a.scale));
}
constexpr int kFewStrips = 8;

// The strip's elements into both planes (and the momentum). WHOLE: all of the launch's strips are whole matrices, and go through all steps in it.
template <typename T, bool MUON, bool WHOLE>
__global__ __launch_bounds__(kShortThreads) void short_begin_kernel(Group g, Update h, int steps) {
  extern __shared__ __attribute__((aligned(256))) char lds[];
  __shared__ double norms[kShortThreads / 64];
  const Place p = place_of(g, blockIdx.x, [](const Matrix& a) { return (uint32_t)strips_of(a); });
  const Matrix& a = p.a;
  const int64_t at = p.batch * ((int64_t)a.m * a.n);
  const Strip strip(a, (int)p.index, lds);
  const T* in = static_cast<const T*>(a.in);
  acc16 x = {}, was = {}, sums = {};
  strip.each(strip.bands, strip.blocks, [&](int ti, int tj) {
    strip.fours(ti, tj, [&](int e, int i, int j) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int64_t from = strip.place(at, i + k, j);
        if (from < 0) continue;
        x[e + k] = Cvt<T>::up(in[from]);
        if constexpr (MUON) was[e + k] = a.momentum[from];
      }
    });
  });
  double sum = 0;
  strip.each(strip.bands, strip.blocks, [&](int ti, int tj) {
    strip.fours(ti, tj, [&](int e, int i, int j) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float u = x[e + k];
        if constexpr (MUON) {
          const float grad = u * h.gradScale, m = __builtin_fmaf(was[e + k], h.beta, grad);
          const int64_t to = strip.place(at, i + k, j);
          if (to >= 0) a.momentum[to] = m;
          u = h.nesterov ? __builtin_fmaf(m, h.beta, grad) : m;
        }
        x[e + k] = u;
        sum += (double)u * u;
      }
    });
  });
  for (int d = 32; d >= 1; d >>= 1) sum += __shfl_xor(sum, d);
  if (strip.lane == 0) norms[strip.wave] = sum;
  __syncthreads();
  sum = 0;
  for (int w = 0; w < kShortThreads / 64; ++w) sum += norms[w];
  const bool alone = WHOLE || is_alone(a);
  const Factor factor = alone ? Factor(a.scale, sum, h.eps) : Factor(ldexp(1.0, strip_exponent(sum, a.scale)));
#pragma unroll
  for (int e = 0; e < 16; ++e) x[e] = factor(x[e]);
  strip.gram(x, sums);
  if constexpr (WHOLE) {
    for (int k = 0; k < steps; ++k) {
      strip.scaled(sums);
      strip.polynomial(sums);
      strip.step(x, 1.f);
      if (k + 1 < steps) strip.gram(x, sums);
    }
    strip.emit<T, MUON>(x, h, at);
  } else {
    char* work = a.work + p.batch * short_bytes(a);
    leave(strip, sums, work, p.index, 0);
    if (threadIdx.x == 0) reinterpret_cast<double*>(work + shares_end(a))[p.index] = sum;
  }
}

// The sum of the strips' shares of A, before the step that takes it: where each strip's workgroup would read many of them. (The order is the same.)
constexpr int kShareThreads = 64;
__host__ __device__ inline uint32_t share_parts(const Matrix& a) { return (uint32_t)(gram_bytes(a) / 16 / kShareThreads); }
__global__ __launch_bounds__(kShareThreads) void shares_kernel(Group g, Update h, int turn, bool first) {
  const Place p = place_of(g, blockIdx.x, [](const Matrix& a) { return share_parts(a); });
  const Matrix& a = p.a;
  const int strips = strips_of(a);
  const int64_t bytes = gram_bytes(a), step = bytes / 16;
  char* shares = a.work + p.batch * short_bytes(a) + plane_t(a);
  typedef float float4v __attribute__((ext_vector_type(4)));
  const int64_t k = (int64_t)p.index * kShareThreads + threadIdx.x;
  const float4v* from = reinterpret_cast<const float4v*>(shares + turn * strips * bytes) + k;
  float4v sum = {};
  if (first && !is_alone(a)) {
    double* norms = reinterpret_cast<double*>(a.work + p.batch * short_bytes(a) + shares_end(a));
    double squares = 0;
    if (strips <= kFewStrips) {
      for (int s = 0; s < strips; ++s) squares += norms[s];
    } else {
      for (int s = threadIdx.x; s < strips; s += kShareThreads) squares += norms[s];
      for (int d = 32; d >= 1; d >>= 1) squares += __shfl_xor(squares, d);
    }
    if (p.index == 0 && threadIdx.x == 0) norms[strips] = squares;
    const double norm = sqrt(squares) + (double)h.eps;
#pragma unroll 4
    for (int s = 0; s < strips; ++s) {
      const float f = strip_factor(norm, norms[s], a);
      sum += from[s * step] * (f * f);
    }
  } else {
#pragma unroll 8
    for (int s = 0; s < strips; ++s) sum += from[s * step];
  }
  reinterpret_cast<float4v*>(shares + 2 * strips * bytes)[k] = sum;
}

template <typename T, bool MUON, bool LAST>
__global__ __launch_bounds__(kShortThreads) void short_step_kernel(Group g, Update h, int turn, bool summed, bool first, int steps) {
  extern __shared__ __attribute__((aligned(256))) char lds[];
  const Place p = place_of(g, blockIdx.x, [](const Matrix& a) { return (uint32_t)strips_of(a); });
  const Matrix& a = p.a;
  const Strip strip(a, (int)p.index, lds);
  char* work = a.work + p.batch * short_bytes(a);
  // the strip's transpose is on its way while A is made
  const int pieces = strip.bands * 8, rows = min(kStrip, a.n - strip.j0), piece = threadIdx.x & 31;
  const uint4v* from = reinterpret_cast<const uint4v*>(work + (int64_t)strip.j0 * strip.bands * 128);
  uint4v held[kStripLoads];
#pragma unroll
  for (int q = 0; q < kStripLoads; ++q) {
    const int row = (threadIdx.x >> 5) + q * (kShortThreads / 32);
    held[q] = row < rows && piece < pieces ? from[row * pieces + piece] : uint4v{0, 0, 0, 0};
  }
  const int strips = strips_of(a);
  const int64_t bytes = gram_bytes(a);
  const char* shares = work + plane_t(a) + (summed ? 2 * strips : turn * strips) * bytes;
  acc16 sums = {}, x = {};
  const bool weighed = first && !is_alone(a);
  const double* norms = reinterpret_cast<const double*>(work + shares_end(a));
  double norm = 0;
  if (weighed) {
    if (summed) norm = norms[strips];
    else for (int k = 0; k < strips; ++k) norm += norms[k];
    norm = sqrt(norm) + (double)h.eps;
  }
  float factor = weighed ? strip_factor(norm, norms[p.index], a) : 1.f;
  const float factors = weighed && !summed ? strip_factor(norm, norms[min(strip.lane, strips - 1)], a) : 1.f;      // of as many strips as lanes
  strip.each(strip.bands, strip.bands, [&](int ti, int tj) {
    const acc16* mine = reinterpret_cast<const acc16*>(shares) + (ti * strip.bands + tj) * 64 + strip.lane;
    for (int k = 0; k < (summed ? 1 : strips); ++k) {
      const float f = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(factors), k));
      sums += mine[k * (bytes / 64)] * (f * f);
    }
  });
#pragma unroll
  for (int q = 0; q < kStripLoads; ++q)
    if (piece < pieces) *reinterpret_cast<uint4v*>(strip.across.piece((threadIdx.x >> 5) + q * (kShortThreads / 32), piece)) = held[q];
  strip.scaled(sums);
#pragma unroll 1
  for (int k = 0;;) {
    strip.polynomial(sums);
    strip.step(x, factor);
    if (++k == steps) break;
    factor = 1.f;
    if (is_alone(a)) {
      strip.gram(x, sums);
      strip.scaled(sums);
    } else {
      strip.turn(x, sums);
    }
  }
  if constexpr (LAST) {
    strip.emit<T, MUON>(x, h, p.batch * ((int64_t)a.m * a.n));
  } else {
    strip.gram(x, sums);
    leave(strip, sums, work, p.index, turn ^ 1);
  }
}

// ----------------------------------------------------------------- launches --
template <typename Count>
uint32_t number(Group& g, Count count) {
  uint32_t n = 0;
  for (int k = 0; k < g.count; ++k) {
    g.first[k] = n;
    n += count(g.matrix[k]) * (uint32_t)g.matrix[k].batch;
  }
  g.first[g.count] = n;
  return n;
}

float scale_of(int64_t m, int64_t n) {
  int e = 0;
  while (e < 15 && (int64_t(1) << (2 * (e + 1))) <= m * n) ++e;
  return (float)(1 << e);
}

// Workspace that the matrices of one pass share, which are equal shares of all: enough of them to fill the chip many times over. ms in passes of up to 0.5, 1
// and 2 GiB, medians of four runs in turn, each within 0.3 %: 72 matrices of 150 M halves with copies 10.11, 9.12, 9.08; 36 of 75 M floats 5.28, 4.56, 4.55; 78 of 100 M halves
// 6.68, 6.24, 6.02; 64 of 1000 x 1000 halves 5.57, 5.51, 5.15; 40 of 1024 x 4096 7.92, 6.56, 6.32; 2000 of 100 x 1000 floats 6.68, 6.74, 6.36; 300 of 600 x 600 7.15, 6.90, 7.03.
constexpr int64_t kPassBytes = int64_t(2) << 30;

struct Bytes {
  int64_t work, norms;
};
enum Kind { kThinOnes, kShortOnes, kLongOnes, kOthers };      // whose launches are others
int kind_of(const Matrix& a) { return is_thin(a) ? kThinOnes : is_short(a) ? kShortOnes : is_long(a) ? kLongOnes : kOthers; }
int64_t each_bytes(const Matrix& a) { return is_short(a) ? short_bytes(a) : work_bytes(a); }
Bytes bytes_of(const Matrix& a) { return Bytes{each_bytes(a) * a.batch, is_short(a) ? 0 : (int64_t)norm_parts(a) * a.batch * 8}; }

// What workgroups that each multiply `blocks` blocks take, us, as measured with one matrix of 256 to 4096 rows: up to one to a CU, or rounds of two to each.
double product_time(int32_t tile, double blocks, int64_t units, int64_t cus, bool cut) {
  const double fixed = tile == kTile ? (cut ? 5 : 11) : (cut ? 3 : 6);      // (parts have no results to write)
  if (units <= cus) return (tile == kTile ? 0.74 : 0.325) * blocks + fixed;
  return (double)((units + 2 * cus - 1) / (2 * cus)) * ((tile == kTile ? 1.08 : 0.43) * blocks + fixed);
}

// One of a step's products over a group: its tiles, numbered, and which of them are cut: those of the last round of workgroups, if that saves more than
// the joining launch costs. Large or small tiles by what they take. us with large, large and cut, small, small and cut ones, before the latter read ahead: A of 256 x 256
// 17, -, 8, -; of 512 x 2048 55, 23, 26, 17; of 1024 x 1024 33, 24, 16, 20; of 2048 x 8192 198, 111, 181, 133; of 4096 x 4096 235, 161, 243, 215.
struct Launch {
  Group g;
  int32_t tile;
  Tail tail;
  Launch(const Group& from, int op, int64_t cus) : g(from) {
    const bool symmetric = op != kStep;
    auto blocks = [&](int k) { return (int32_t)blocks_of(op == kGram ? g.matrix[k].n : g.matrix[k].m); };
    auto parts_of = [&](int k) { return sum_parts(blocks(k), product_tiles(g.matrix[k], symmetric)); };
    const int32_t parts = parts_of(g.count - 1);
    int same = g.count - 1;      // the first of the matrices at the end whose sums have as many parts
    while (same > 0 && parts_of(same - 1) == parts) --same;
    auto plan = [&](int32_t t, Tail& to) {
      const uint32_t tiles = number(g, [&](const Matrix& a) { return product_tiles(a, symmetric, t); });
      double length = 0;
      for (int k = 0; k < g.count; ++k) length += (double)blocks(k) * (g.first[k + 1] - g.first[k]) / tiles;
      const uint32_t last = tiles % (uint32_t)(2 * cus), rest = std::min(last, tiles - g.first[same]);
      const double rounds = product_time(t, length, tiles - last, cus, false);
      to = Tail{tiles, 1, nullptr};
      if (last == 0) return rounds;
      const double tail = (double)blocks(g.count - 1), whole = product_time(t, tail, last, cus, false);
      const int64_t units = (int64_t)rest * parts;
      const double cut = product_time(t, tail / parts, units, cus, true) + 7 + (t == kTile ? 0.014 : 0.002) * (double)units;
      const bool cuts = parts > 1 && rest == last && cut < whole;
      if (cuts) {
        to.whole = tiles - rest;
        to.parts = parts;
      }
      return (tiles > last ? rounds : 0) + (cuts ? cut : whole);
    };
    const double large = plan(kTile, tail), small = plan(kSmallTile, tail);
    tile = large <= small ? kTile : kSmallTile;
    plan(tile, tail);      // (which numbers the tiles)
  }
  uint32_t rest() const { return g.first[g.count] - tail.whole; }
  int64_t bytes() const { return (int64_t)rest() * tail.parts * tile * tile * 4; }
  template <int OP, typename T, bool MUON>
  void go(THCState* s, const Update& h, const Way& way) const {
    if (tile == kTile) go_tiles<OP, T, MUON, kTile>(s, h, way);
    else go_tiles<OP, T, MUON, kSmallTile>(s, h, way);
  }
  template <int OP, typename T, bool MUON, int TILE>
  void go_tiles(THCState* s, const Update& h, const Way& way) const {
    hipStream_t st = current_stream(s);
    const dim3 grid(tail.whole + rest() * tail.parts), joins(rest() * (TILE / 64) * (TILE / 64));
    hipLaunchKernelGGL((product_kernel<OP, T, MUON, false, TILE>), grid, dim3(256), 0, st, g, h, way, tail);
    if (rest()) hipLaunchKernelGGL((product_kernel<OP, T, MUON, true, TILE>), joins, dim3(256), 0, st, g, h, way, tail);
  }
};
struct Plan {
  Launch gram, polynomial, step;
  Plan(const Group& g, int64_t cus) : gram(g, kGram, cus), polynomial(g, kPolynomial, cus), step(g, kStep, cus) {}
  int64_t bytes() const { return std::max({gram.bytes(), polynomial.bytes(), step.bytes()}); }
};

// How many steps go with one A from X. An error of A grows with what it belongs to, up to 12 times a step where singular values are small. Two steps
// leave what single ones do. Against 64 bits after five steps, in 1e-6 of the result's norm, by products of floats, singly, as 2 + 2 + 1 (medians of
// four; elements alike / few directions with most of the norm / singular values from 1 to 1e-3): 65 x 513 1.7 1.9 1.9 / 1.2 1.0 1.1 / 3.5 2.8 3.0,
// 33 x 500 2.4 2.3 3.7 / 1.5 1.3 1.3 / 3.6 3.3 3.4, 300 x 700 2.2 1.9 1.9 / 1.9 1.7 2.4 / 3.4 5.4 5.2, 1024 x 4096 3.7 1.4 1.6 / 2.7 1.5 1.4 / 4.7 5.4 4.7.
// Three steps do not where few directions share the norm (11 of 33 x 500): they are for results that are only written as halves (`rough`), which come with
// 200 of their own, not for float copies of half parameters. (4 + 1 leaves 20 to 60.)
// Up to 32 rows sums of floats round least, and the later pairs would show (23 x 1024 2.4 in place of 1.8 singly): two first, then singly, and all four
// products of halves, 1.7 (49 us instead of 39).
int chain_of(int done, int steps, bool rough, bool thin) {
  if (rough) return done == 0 && steps % 2 && steps >= 3 ? 3 : std::min(2, steps - done);
  return std::min(thin && done ? 1 : 2, steps - done);
}
// (all parameters of a call have copies, or none)
template <typename T, bool MUON>
bool is_rough(const Group& g) { return std::is_same_v<T, __half> && !(MUON && g.matrix[0].master); }

// One launch for all steps, and no workspace.
bool is_whole(const Group& g) {
  for (int k = 0; k < g.count; ++k)
    if (!is_alone(g.matrix[k])) return false;
  return true;
}
template <typename T, bool MUON>
void run_short(THCState* s, Group& g, const Update& h, int steps) {
  hipStream_t st = current_stream(s);
  int bands = 0, most = 0;
  int64_t read = 0;
  for (int k = 0; k < g.count; ++k) {
    const Matrix& a = g.matrix[k];
    bands = std::max(bands, bands_of(a));
    most = std::max(most, strips_of(a));
    read += (int64_t)a.batch * strips_of(a) * strips_of(a) * gram_bytes(a);
  }
  // (40 matrices of 100 x 1000, 8 strips and 168 MB of shares: 329 us without the sums' launches, 255 with; a launch that few bytes would not pay takes 5)
  const bool many = most > kFewStrips || read > (int64_t(24) << 20);
  const int lds = short_lds(bands);
  const dim3 threads(kShortThreads);
  Group shares = g;
  const uint32_t parts = many ? number(shares, share_parts) : 0;
  const dim3 strips(number(g, [](const Matrix& a) { return (uint32_t)strips_of(a); }));
  auto roomy = [&](auto kernel) {
    if (lds > 65536) THC_CHECK(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, lds));
    return kernel;
  };
  if (is_whole(g)) {
    hipLaunchKernelGGL(roomy(short_begin_kernel<T, MUON, true>), strips, threads, lds, st, g, h, steps);
    return;
  }
  hipLaunchKernelGGL(roomy(short_begin_kernel<T, MUON, false>), strips, threads, lds, st, g, h, steps);
  for (int done = 0, turn = 0; done < steps; turn ^= 1) {
    const int chain = chain_of(done, steps, is_rough<T, MUON>(g), is_thin(g.matrix[0]));
    const bool first = done == 0;
    done += chain;
    if (many) hipLaunchKernelGGL(shares_kernel, dim3(parts), dim3(kShareThreads), 0, st, shares, h, turn, first);
    if (done < steps) hipLaunchKernelGGL(roomy(short_step_kernel<float, false, false>), strips, threads, lds, st, g, h, turn, many, first, chain);
    else hipLaunchKernelGGL(roomy(short_step_kernel<T, MUON, true>), strips, threads, lds, st, g, h, turn, many, first, chain);
  }
}

template <typename T, bool MUON>
void run_group(THCState* s, Group& g, const Update& h, int steps, char* work, double* norms, acc16* sums) {
  hipStream_t st = current_stream(s);
  for (int k = 0; k < g.count; ++k) {
    g.matrix[k].work = work;
    work += bytes_of(g.matrix[k]).work;
  }
  if (is_short(g.matrix[0])) {
    run_short<T, MUON>(s, g, h, steps);
    return;
  }
  const uint32_t parts = number(g, norm_parts);
  for (int k = 0; k < g.count; ++k) g.matrix[k].norms = g.first[k];
  hipLaunchKernelGGL((norm_kernel<T, MUON>), dim3(parts), dim3(kBlock), 0, st, g, h, norms);
  const uint32_t tiles = number(g, tiles64);
  hipLaunchKernelGGL((split_kernel<T, MUON>), dim3(tiles), dim3(kBlock), 0, st, g, h, norms);
  Plan plan(g, num_compute_units(s));
  plan.gram.tail.sums = plan.polynomial.tail.sums = plan.step.tail.sums = sums;
  const bool chained = is_long(g.matrix[0]);
  for (int done = 0, turn = 0; done < steps; turn ^= 1) {
    plan.gram.go<kGram, float, false>(s, h, Way{turn, 0, 0, 0, 0, 0});
    Way way{turn, 1, 0, 0, kA, 1 / kScaleB};
    if (chained) {
      const int last = done + chain_of(done, steps, is_rough<T, MUON>(g), false);
      int a = 0, p = 1, c = 2, q = 1;
      float scale = kScaleB;      // of Q
      plan.polynomial.go<kPolynomial, float, false>(s, h, Way{turn, a, a, p, kA, 0});
      while (++done < last) {
        plan.polynomial.go<kProduct, float, false>(s, h, Way{turn, p, a, c, 0, 1 / kScaleB});
        plan.polynomial.go<kProduct, float, false>(s, h, Way{turn, c, p, a, 0, 1 / kScaleB});
        plan.polynomial.go<kPolynomial, float, false>(s, h, Way{turn, a, a, c, kA, 0});
        const int free = q == p ? 3 : p, next = scale == kScaleB ? 2 : 4;      // (Q's elements stay below a^2, a^3)
        plan.polynomial.go<kProduct, float, false>(s, h, Way{turn, c, q, free, 0, 1 / (kScaleB * next)});
        scale /= next;
        p = c;
        c = q;
        q = free;
      }
      way = Way{turn, q, 0, 0, 0, 1 / scale};
    } else {
      plan.polynomial.go<kPolynomial, float, false>(s, h, Way{turn, 0, 0, 1, 0, 0});
      ++done;
    }
    if (done < steps) plan.step.go<kStep, float, false>(s, h, way);
    else plan.step.go<kLast, T, MUON>(s, h, way);
  }
}

// Matrices, short and others, by as many as a launch's arguments hold and a pass's workspace has room for; that is taken before the first launch.
template <typename T, bool MUON>
void run(THCState* s, std::vector<Matrix>& all, const Update& h, int steps) {
  // (equal ones side by side, long sums first: what is left of a launch at its end is short)
  std::stable_sort(all.begin(), all.end(), [](const Matrix& a, const Matrix& b) { return a.n != b.n ? a.n > b.n : a.m > b.m; });
  std::vector<Group> groups;
  for (int kind : {kThinOnes, kShortOnes, kLongOnes, kOthers}) {
    // passes of equal shares
    int64_t total = 0, largest = 0;
    for (const Matrix& a : all) {
      if (kind_of(a) != kind) continue;
      total += each_bytes(a) * a.batch;
      largest = std::max(largest, each_bytes(a));
    }
    const int64_t share = total / (total / kPassBytes + 1) + largest;
    int64_t sum = 0;
    bool open = false;
    auto add = [&](const Matrix& a) {
      const int64_t bytes = bytes_of(a).work;
      if (!open || groups.back().count == kMatrices || sum + bytes > share) {
        groups.emplace_back();
        groups.back().count = 0;
        sum = 0;
        open = true;
      }
      Group& g = groups.back();
      g.matrix[g.count++] = a;
      sum += bytes;
    };
    for (const Matrix& a : all) {
      if (kind_of(a) != kind) continue;
      // a batch in pieces: by the workspace, and by what the workgroups of a launch are counted in
      const int64_t size = (int64_t)a.m * a.n;
      const int64_t each = std::max<int64_t>(1, std::min<int64_t>(share / each_bytes(a), 1 << 20));
      for (int64_t first = 0; first < a.batch; first += each) {
        Matrix piece = a;
        piece.batch = (int32_t)std::min<int64_t>(each, a.batch - first);
        piece.in = static_cast<const T*>(a.in) + first * size;
        piece.out = static_cast<T*>(a.out) + first * size;
        if (a.momentum) piece.momentum = a.momentum + first * size;
        if (a.master) piece.master = a.master + first * size;
        add(piece);
      }
    }
  }
  Bytes most{8, 8};
  int64_t tails = 8;
  for (const Group& g : groups) {
    if (is_whole(g)) continue;
    Bytes sum{0, 0};
    for (int k = 0; k < g.count; ++k) {
      const Bytes b = bytes_of(g.matrix[k]);
      sum.work += b.work;
      sum.norms += b.norms;
    }
    most = Bytes{std::max(most.work, sum.work), std::max(most.norms, sum.norms)};
    if (!is_short(g.matrix[0])) tails = std::max(tails, Plan(g, num_compute_units(s)).bytes());
  }
  Workspace work(s, most.work), norms(s, most.norms), sums(s, tails);
  for (Group& g : groups)
    run_group<T, MUON>(s, g, h, steps, work.data(), reinterpret_cast<double*>(norms.data()), reinterpret_cast<acc16*>(sums.data()));
}

void check_matrices(const AnyTensor* t, int arg) {
  const int nd = t->nDimension;
  THC_ARG_CHECK(nd >= 2, arg, "matrices have two dims at least");
  THC_ARG_CHECK(nd <= kMaxDims, arg, "%s", kDimWarning);
  const int64_t rows = t->size[nd - 2], cols = t->size[nd - 1];
  THC_ARG_CHECK(rows <= (int64_t(1) << 20) && cols <= (int64_t(1) << 20) && rows * cols < (int64_t(1) << 34), arg, "matrices are too large");
  THC_ARG_CHECK(tensor_numel(t) / rows / cols < kIndex32Limit, arg, "too many matrices");
}
Matrix matrix_of(const AnyTensor* t) {
  const int64_t rows = t->size[t->nDimension - 2], cols = t->size[t->nDimension - 1];
  Matrix a{};
  a.m = (int32_t)std::min(rows, cols);
  a.n = (int32_t)std::max(rows, cols);
  a.batch = (int32_t)(tensor_numel(t) / rows / cols);
  a.tall = rows > cols;
  a.scale = scale_of(a.m, a.n);
  return a;
}
void check_steps(int steps, int arg) { THC_ARG_CHECK(steps >= 1 && steps <= 1000, arg, "%d steps", steps); }

void orthogonalize(THCState* s, DType dt, AnyTensor* self, AnyTensor* input, int steps, double eps) {
  const AnyTensor* both[2] = {self, input};
  check_same_gpu(s, 2, both);
  check_steps(steps, 4);
  THC_ARG_CHECK(eps >= 0, 5, "eps is negative");
  if (!has_elements(input)) {
    tensor_resize_as(s, self, input, dt);
    return;
  }
  check_matrices(input, 3);
  refuse_capture(s, "orthogonalising");
  tensor_resize_as(s, self, input, dt);
  note_stream_use(s, {self, input});
  Dense in(s, input, dt);
  // every matrix is read before its place is written
  const bool same = self->storage == in.ref.t->storage && self->storageOffset == in.ref.t->storageOffset;
  const bool direct = tensor_is_contiguous(self) && (same || !spans_meet(self, dt, in.ref.t, dt));
  TensorRef out(s, direct ? (tensor_retain(self), self) : tensor_new_with_size(s, self->nDimension, self->size, dt));
  Update h{};
  h.eps = (float)eps;
  Matrix a = matrix_of(input);
  a.in = tensor_data(in.ref.t, dt);
  a.out = tensor_data(out.t, dt);
  std::vector<Matrix> all{a};
  if (dt == DType::F32) run<float, false>(s, all, h, steps);
  else run<__half, false>(s, all, h, steps);
  THC_CHECK(hipGetLastError());
  note_kernel("orthogonalize");
  if (out.t != self) copy_tensor(s, dt, self, out.t, false);
}

struct Lists {
  AnyTensor **param, **master, **grad, **momentum;      // master: or null
};
void muon(THCState* s, DType dt, int count, const Lists& l, double lr, double beta, double weightDecay, int nesterov, int steps, double eps,
          double matchRms, double gradScale) {
  const int base = dt == DType::F16 ? 5 : 4;      // argument numbers: state, count, param, [master], grad, ...
  THC_ARG_CHECK(count >= 0, 2, "a negative number of tensors");
  THC_ARG_CHECK(count == 0 || (l.param && l.grad && l.momentum), 3, "a list of tensors is missing");
  THC_ARG_CHECK(beta >= 0 && beta < 1, base + 3, "beta is not in [0, 1)");
  check_steps(steps, base + 6);
  THC_ARG_CHECK(eps >= 0, base + 7, "eps is negative");
  THC_ARG_CHECK(matchRms >= 0, base + 8, "the update's size is negative");
  for (int i = 0; i < count; ++i) {
    const AnyTensor* p = l.param[i];
    THC_ARG_CHECK(p, 3, "tensor %d is missing", i + 1);
    check_list(s, p, p, 3, i, true);
    if (l.master) check_list(s, l.master[i], p, 4, i, true);
    check_list(s, l.grad[i], p, base, i, false);
    check_list(s, l.momentum[i], p, base + 1, i, true);
    if (has_elements(p)) check_matrices(p, 3);
  }
  refuse_capture(s, "a step of the optimizer of matrices");
  Update h;
  h.beta = (float)beta;
  h.gradScale = (float)gradScale;
  h.keep = (float)(1 - lr * weightDecay);
  h.eps = (float)eps;
  h.nesterov = nesterov;
  // every copy is made before the first launch: a step that fails has changed nothing
  Held held(s);
  std::vector<Matrix> all;
  all.reserve(count);
  for (int i = 0; i < count; ++i) {
    AnyTensor* p = l.param[i];
    if (!has_elements(p)) continue;
    note_stream_use(s, {p, l.master ? l.master[i] : nullptr, l.grad[i], l.momentum[i]});
    Matrix a = matrix_of(p);
    const double rows = a.tall ? a.n : a.m, cols = a.tall ? a.m : a.n;
    a.rate = (float)(lr * (matchRms > 0 ? matchRms * std::sqrt((double)a.n) : std::sqrt(std::max(1.0, rows / cols))));
    a.out = held.add(p, dt, true);
    a.in = held.add(l.grad[i], dt, false);
    a.momentum = static_cast<float*>(held.add(l.momentum[i], DType::F32, true));
    a.master = l.master ? static_cast<float*>(held.add(l.master[i], DType::F32, true)) : nullptr;
    all.push_back(a);
  }
  if (dt == DType::F32) run<float, true>(s, all, h, steps);
  else run<__half, true>(s, all, h, steps);
  THC_CHECK(hipGetLastError());
  note_kernel("muon");
  held.write_back();
}

}  // namespace
}  // namespace thc

#define TN(x) reinterpret_cast<thc::AnyTensor*>(x)
#define TL(x) reinterpret_cast<thc::AnyTensor**>(x)
THC_API void THCudaTensor_orthogonalize(THCState* s, THCudaTensor* self, THCudaTensor* input, int steps, double eps) {
  THC_GUARD_ALL(thc::orthogonalize(s, thc::DType::F32, TN(self), TN(input), steps, eps))
}
THC_API void THCudaHalfTensor_orthogonalize(THCState* s, THCudaHalfTensor* self, THCudaHalfTensor* input, int steps, double eps) {
  THC_GUARD_ALL(thc::orthogonalize(s, thc::DType::F16, TN(self), TN(input), steps, eps))
}
THC_API void THCudaTensor_muon(THCState* s, int count, THCudaTensor** param, THCudaTensor** grad, THCudaTensor** momentum, double lr, double beta,
                               double weightDecay, int nesterov, int steps, double eps, double matchRms, double gradScale) {
  THC_GUARD_ALL(thc::muon(s, thc::DType::F32, count, {TL(param), nullptr, TL(grad), TL(momentum)}, lr, beta, weightDecay, nesterov, steps, eps, matchRms,
                          gradScale))
}
THC_API void THCudaHalfTensor_muon(THCState* s, int count, THCudaHalfTensor** param, THCudaTensor** master, THCudaHalfTensor** grad,
                                   THCudaTensor** momentum, double lr, double beta, double weightDecay, int nesterov, int steps, double eps,
                                   double matchRms, double gradScale) {
  THC_GUARD_ALL(thc::muon(s, thc::DType::F16, count, {TL(param), TL(master), TL(grad), TL(momentum)}, lr, beta, weightDecay, nesterov, steps, eps,
                          matchRms, gradScale))
}
