// Newton-Schulz orthogonalisation of matrices, and the optimizer whose step it is.
//
//   orthogonalize   X = G / (|G| + eps);  A = X X', B = b A + c A A, X = a X + B X, `steps` times, the shorter side first
//   muon            m = beta m + g;  u = g + beta m (or m);  p = p (1 - lr decay) - rate orthogonalize(u)
//
// The products run on the matrix cores in half precision, every factor as a sum of two halves (x = h + l, 22 bits): h h' + h l' + l h' is as exact
// as a product of floats (measured against 64 bits after five steps: 2e-6 of the result's norm, as float products have), at a third of the
// halves' rate, where float products have a sixteenth of it. One half alone would leave 1e-3 to 5e-3. Sums are in float throughout, the norm's in 64 bits.
// Singular values of X stay below 1.21 once they are at most 1 (a s + b s^3 + c s^5 on 0 ... 1.21), so no element of X, A and B leaves
// +-1.21, +-1.46, +-2.81, and each is held times a power of two that brings its usual size to where halves are exact, and its
// largest below their largest: S for X, 2^14 for A, 2^13 for B.
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
constexpr int kBlockK = 32;
__host__ __device__ constexpr int64_t blocks_of(int64_t k) { return (k + kBlockK - 1) / kBlockK; }
__host__ __device__ constexpr int64_t row_bytes(int64_t k) { return blocks_of(k) * 128; }
__device__ __forceinline__ int64_t split_at(int64_t row, int32_t column, int64_t rowBytes) {
  return row * rowBytes + (column >> 5) * 128 + (column & 31) * 2;      // of the upper half; the lower one 64 bytes on
}

// `batch` matrices of m x n, m <= n, X short side first; `tall`: their tensors have n rows and m columns.
struct Matrix {
  char* work;                  // X, X', the next X, the next X', A, B of each one
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
__host__ __device__ inline int64_t work_bytes(const Matrix& a) { return 2 * (plane_x(a) + plane_t(a) + plane_a(a)); }

constexpr int kMatrices = 48;
struct Group {
  Matrix matrix[kMatrices];
  uint32_t first[kMatrices + 1];      // the first workgroup of each
  int32_t count;
};
struct Place {
  Matrix a;
  uint32_t index;      // of the workgroup within one matrix
  int32_t batch;
  uint32_t begin;      // of the descriptor's workgroups
};
// The matrix of this workgroup, `each` workgroups (by the matrix) for one of a batch.
template <typename F>
__device__ __forceinline__ Place place_of(const Group& g, uint32_t block, F each) {
  int k = 0;
  while (k + 1 < g.count && block >= g.first[k + 1]) ++k;
  Place p{g.matrix[k], block - g.first[k], 0, g.first[k]};
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

// The sum of squares of a part of a matrix, in 64 bits; the optimizer's momentum on the way.
template <typename T, bool MUON>
__global__ __launch_bounds__(kBlock) void norm_kernel(Group g, Update h, double* parts) {
  __shared__ double lds[kBlock / 64];
  const Place p = place_of(g, blockIdx.x, [](const Matrix& a) { return norm_parts(a); });
  const int64_t size = (int64_t)p.a.m * p.a.n, from = (int64_t)p.index * kNormPart, to = min(size, from + kNormPart);
  const T* in = static_cast<const T*>(p.a.in) + p.batch * size;
  float* momentum = MUON ? p.a.momentum + p.batch * size : nullptr;
  double sum = 0;
  for (int64_t i = from + threadIdx.x; i < to; i += kBlock) {
    float u = Cvt<T>::up(in[i]);
    if constexpr (MUON) {
      u *= h.gradScale;
      const float m = __builtin_fmaf(momentum[i], h.beta, u);
      momentum[i] = m;
      u = h.nesterov ? __builtin_fmaf(m, h.beta, u) : m;
    }
    sum += (double)u * u;
  }
  for (int d = 32; d >= 1; d >>= 1) sum += __shfl_xor(sum, d);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kBlock / 64; ++w) sum += lds[w];
    parts[blockIdx.x] = sum;
  }
}

struct Split {
  _Float16 h, l;
};
__device__ __forceinline__ Split split(float x) {
  Split s;
  s.h = (_Float16)x;
  s.l = (_Float16)(x - (float)s.h);
  return s;
}
__device__ __forceinline__ void store_split(char* plane, int64_t at, float x) {
  const Split s = split(x);
  *reinterpret_cast<_Float16*>(plane + at) = s.h;
  *reinterpret_cast<_Float16*>(plane + at + 64) = s.l;
}
__device__ __forceinline__ float load_split(const char* plane, int64_t at) {
  return (float)*reinterpret_cast<const _Float16*>(plane + at) + (float)*reinterpret_cast<const _Float16*>(plane + at + 64);
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
  const float factor = (float)((double)a.scale / (sqrt(sum) + (double)h.eps));
  const int32_t rows = a.tall ? a.n : a.m, cols = a.tall ? a.m : a.n, across = (cols + 63) / 64;
  const int32_t r0 = (int32_t)(p.index / across) * 64, c0 = (int32_t)(p.index % across) * 64;
  const T* in = static_cast<const T*>(a.in) + p.batch * size;
  const float* momentum = MUON ? a.momentum + p.batch * size : nullptr;
  for (int i = threadIdx.x; i < 64 * 64; i += kBlock) {
    const int32_t r = r0 + i / 64, c = c0 + i % 64;
    float u = 0.f;
    if (r < rows && c < cols) {
      const int64_t at = (int64_t)r * cols + c;
      u = Cvt<T>::up(in[at]);
      if constexpr (MUON) u = h.nesterov ? __builtin_fmaf(momentum[at], h.beta, u * h.gradScale) : momentum[at];
      u *= factor;
    }
    tile[i / 64][i % 64] = u;
  }
  __syncthreads();
  char *work = a.work + p.batch * work_bytes(a), *byRow = a.tall ? work + plane_x(a) : work, *byColumn = a.tall ? work : work + plane_x(a);
  const int64_t rowBytes = row_bytes(cols), columnBytes = row_bytes(rows);
  const int32_t colEnd = (int32_t)blocks_of(cols) * kBlockK, rowEnd = (int32_t)blocks_of(rows) * kBlockK;
  for (int i = threadIdx.x; i < 64 * 64; i += kBlock) {
    const int32_t x = i / 64, y = i % 64;
    if (r0 + x < rows && c0 + y < colEnd) store_split(byRow, split_at(r0 + x, c0 + y, rowBytes), tile[x][y]);
    if (c0 + x < cols && r0 + y < rowEnd) store_split(byColumn, split_at(c0 + x, r0 + y, columnBytes), tile[y][x]);
  }
}

// ----------------------------------------------------------------- products --
// C = P Q', P and Q in the split layout: a workgroup has a tile of 128 x 128, each of its four waves 64 x 64 of that as 2 x 2 products of
// 32 x 32. A block of 32 columns of both operands, upper and lower halves, is 32 KiB of LDS; the next one is on its way there while one is
// multiplied. A row's eight 16-byte pieces lie in the order of their number xor the row's, so that lanes that read the same piece of
// neighbouring rows meet all banks.
constexpr int kTile = 128;
__host__ __device__ inline int32_t tiles_of(int32_t n) { return (n + kTile - 1) / kTile; }

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
__device__ __forceinline__ void wait_loads_and_barrier() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

struct Operand {
  const char* rows;      // of the tile's first row
  int64_t rowBytes;
  int32_t count;         // rows from there on
};
__device__ __forceinline__ void product(const Operand& P, const Operand& Q, int32_t blocks, char* lds, acc16 (&acc)[2][2]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
  const uint4v fromP = resource(P.rows, (uint32_t)min(P.count, kTile) * (uint32_t)P.rowBytes), fromQ = resource(Q.rows, (uint32_t)min(Q.count, kTile) * (uint32_t)Q.rowBytes);
  // 16 KiB of an operand are 16 loads of a wave, 8 rows each; wave w has those with numbers w, w + 4, ...
  uint32_t offP[4], offQ[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int32_t row = (q * 4 + wave) * 8 + (lane >> 3), piece = (lane & 7) ^ (lane >> 3);
    offP[q] = (uint32_t)min(row, P.count - 1) * (uint32_t)P.rowBytes + piece * 16;
    offQ[q] = (uint32_t)min(row, Q.count - 1) * (uint32_t)Q.rowBytes + piece * 16;
  }
  auto load = [&](int32_t k, uint32_t stage) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const uint32_t to = __builtin_amdgcn_readfirstlane(base + stage * 32768 + (q * 4 + wave) * 1024);
      load_to_lds(fromP, offP[q], k * 128, to);
      load_to_lds(fromQ, offQ[q], k * 128, to + 16384);
    }
  };
  const int rowP = (wave >> 1) * 64 + (lane & 31), rowQ = (wave & 1) * 64 + (lane & 31);
  load(0, 0);
  for (int32_t k = 0; k < blocks; ++k) {
    wait_loads_and_barrier();
    if (k + 1 < blocks) load(k + 1, (k + 1) & 1);
    const char *fp = lds + (k & 1) * 32768 + rowP * 128, *fq = lds + (k & 1) * 32768 + 16384 + rowQ * 128;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int high = ((2 * s + (lane >> 5)) ^ (lane & 7)) * 16, low = ((4 + 2 * s + (lane >> 5)) ^ (lane & 7)) * 16;
      half8 ph[2], pl[2], qh[2], ql[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        ph[i] = *reinterpret_cast<const half8*>(fp + i * 4096 + high);
        pl[i] = *reinterpret_cast<const half8*>(fp + i * 4096 + low);
        qh[i] = *reinterpret_cast<const half8*>(fq + i * 4096 + high);
        ql[i] = *reinterpret_cast<const half8*>(fq + i * 4096 + low);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ph[i], qh[j], acc[i][j], 0, 0, 0);
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ph[i], ql[j], acc[i][j], 0, 0, 0);
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(pl[i], qh[j], acc[i][j], 0, 0, 0);
        }
    }
  }
}

enum Op { kGram, kPolynomial, kStep, kLast };

__host__ __device__ inline uint32_t symmetric_tiles(int32_t t) { return (uint32_t)(t * (int64_t)(t + 1) / 2); }
__host__ __device__ inline uint32_t product_tiles(const Matrix& a, bool symmetric) {
  return symmetric ? symmetric_tiles(tiles_of(a.m)) : (uint32_t)(tiles_of(a.m) * (int64_t)tiles_of(a.n));
}

// One of a step's three products and what is made of it. The first two are symmetric: tiles above the diagonal go to both places. `turn`: which of the
// two pairs of planes X is in. The last step's result goes to the tensor, or into the parameter.
template <int OP, typename T, bool MUON>
__global__ __launch_bounds__(256) void product_kernel(Group g, Update h, int turn) {
  __shared__ __attribute__((aligned(128))) char lds[65536];
  constexpr bool kSymmetric = OP == kGram || OP == kPolynomial;
  const Place p = place_of(g, blockIdx.x, [](const Matrix& a) { return product_tiles(a, kSymmetric); });
  const Matrix& a = p.a;
  char* work = a.work + p.batch * work_bytes(a);
  const int64_t px = plane_x(a), pt = plane_t(a);
  char *x = work + turn * (px + pt), *t = x + px, *xn = work + (turn ^ 1) * (px + pt), *tn = xn + px, *am = work + 2 * (px + pt), *bm = am + plane_a(a);
  const int64_t bytesM = row_bytes(a.m), bytesN = row_bytes(a.n);
  const bool flipped = OP == kLast && a.tall;      // the tensor's rows are the longer side: its tile is the product's transpose
  int32_t ti, tj;
  if constexpr (kSymmetric) {
    // row by row of the upper triangle
    const int32_t n = tiles_of(a.m);
    ti = 0;
    uint32_t rest = p.index;
    while (rest >= (uint32_t)(n - ti)) {
      rest -= n - ti;
      ++ti;
    }
    tj = ti + (int32_t)rest;
  } else {
    const int32_t n = tiles_of(flipped ? a.m : a.n);
    ti = (int32_t)(p.index / n);
    tj = (int32_t)(p.index % n);
  }
  const int32_t rows = flipped ? a.n : a.m, cols = kSymmetric || flipped ? a.m : a.n, i0 = ti * kTile, j0 = tj * kTile;
  const char *from, *with;
  int64_t bytesK;
  if constexpr (OP == kGram) {
    from = with = x;
    bytesK = bytesN;
  } else {
    bytesK = bytesM;
    from = OP == kPolynomial ? am : flipped ? t : bm;
    with = OP == kPolynomial ? am : flipped ? bm : t;
  }
  const Operand P{from + i0 * bytesK, bytesK, rows - i0}, Q{with + j0 * bytesK, bytesK, cols - j0};
  acc16 acc[2][2] = {};
  product(P, Q, (int32_t)(bytesK / 128), lds, acc);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t size = (int64_t)a.m * a.n;
  // a lane has column `lane % 32` of each 32 x 32 product, four rows in a row of each eight
#pragma unroll
  for (int bi = 0; bi < 2; ++bi) {
#pragma unroll
    for (int bj = 0; bj < 2; ++bj) {
      const int32_t j = j0 + (wave & 1) * 64 + bj * 32 + (lane & 31);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int32_t i = i0 + (wave >> 1) * 64 + bi * 32 + q * 8 + (lane >> 5) * 4;
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const bool inside = i + e < rows && j < cols;
          const float sum = acc[bi][bj][q * 4 + e];
          if constexpr (OP == kGram) {
            v[e] = sum * (kScaleA / (a.scale * a.scale));
          } else if constexpr (OP == kPolynomial) {
            const float one = inside ? load_split(am, split_at(i + e, j, bytesM)) : 0.f;
            v[e] = __builtin_fmaf(one, kB * (kScaleB / kScaleA), sum * (kC * kScaleB / (kScaleA * kScaleA)));
          } else {
            const float one = inside ? (flipped ? load_split(t, split_at(i + e, j, bytesM)) : load_split(x, split_at(i + e, j, bytesN))) : 0.f;
            v[e] = __builtin_fmaf(one, kA, sum * (1.f / kScaleB));
          }
          if (!inside) v[e] = 0.f;
        }
        if constexpr (OP == kLast) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (i + e >= rows || j >= cols) continue;
            const int64_t at = p.batch * size + (int64_t)(i + e) * cols + j;
            const float o = v[e] / a.scale;
            T* out = static_cast<T*>(a.out);
            if constexpr (MUON) {
              const float was = a.master ? a.master[at] : Cvt<T>::up(out[at]), is = __builtin_fmaf(o, -a.rate, was * h.keep);
              if (a.master) a.master[at] = is;
              out[at] = rounded<T>(is);
            } else {
              out[at] = rounded<T>(o);
            }
          }
        } else {
          char* direct = OP == kGram ? am : OP == kPolynomial ? bm : xn;
          char* mirrored = OP == kStep ? tn : direct;
          const int64_t bytesDirect = OP == kStep ? bytesN : bytesM;
          const int32_t colEnd = (int32_t)blocks_of(cols) * kBlockK, rowEnd = (int32_t)blocks_of(rows) * kBlockK;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (i + e < rows && j < colEnd) store_split(direct, split_at(i + e, j, bytesDirect), v[e]);
          if ((OP == kStep || ti != tj) && j < cols && i < rowEnd) {
            half4 hi, lo;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const Split s = split(v[e]);
              hi[e] = s.h;
              lo[e] = s.l;
            }
            char* to = mirrored + split_at(j, i, bytesM);
            *reinterpret_cast<half4*>(to) = hi;
            *reinterpret_cast<half4*>(to + 64) = lo;
          }
        }
      }
    }
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

// Workspace that the matrices of one pass share: enough of them to fill the chip many times over.
constexpr int64_t kPassBytes = int64_t(1) << 30;

struct Bytes {
  int64_t work, norms;
};
Bytes bytes_of(const Matrix& a) { return Bytes{work_bytes(a) * a.batch, (int64_t)norm_parts(a) * a.batch * 8}; }

template <typename T, bool MUON>
void run_group(THCState* s, Group& g, const Update& h, int steps, char* work, double* norms) {
  hipStream_t st = current_stream(s);
  for (int k = 0; k < g.count; ++k) {
    g.matrix[k].work = work;
    work += bytes_of(g.matrix[k]).work;
  }
  const uint32_t parts = number(g, norm_parts);
  for (int k = 0; k < g.count; ++k) g.matrix[k].norms = g.first[k];
  hipLaunchKernelGGL((norm_kernel<T, MUON>), dim3(parts), dim3(kBlock), 0, st, g, h, norms);
  const uint32_t tiles = number(g, tiles64);
  hipLaunchKernelGGL((split_kernel<T, MUON>), dim3(tiles), dim3(kBlock), 0, st, g, h, norms);
  Group symmetric = g;
  const uint32_t half = number(symmetric, [](const Matrix& a) { return product_tiles(a, true); });
  const uint32_t whole = number(g, [](const Matrix& a) { return product_tiles(a, false); });
  for (int k = 0; k < steps; ++k) {
    const int turn = k & 1;
    hipLaunchKernelGGL((product_kernel<kGram, T, MUON>), dim3(half), dim3(256), 0, st, symmetric, h, turn);
    hipLaunchKernelGGL((product_kernel<kPolynomial, T, MUON>), dim3(half), dim3(256), 0, st, symmetric, h, turn);
    if (k + 1 < steps) hipLaunchKernelGGL((product_kernel<kStep, T, MUON>), dim3(whole), dim3(256), 0, st, g, h, turn);
    else hipLaunchKernelGGL((product_kernel<kLast, T, MUON>), dim3(whole), dim3(256), 0, st, g, h, turn);
  }
}

// Matrices by as many as a launch's arguments hold and a pass's workspace has room for; that is taken before the first launch.
template <typename T, bool MUON>
void run(THCState* s, const std::vector<Matrix>& all, const Update& h, int steps) {
  std::vector<Group> groups;
  Bytes most{0, 0}, sum{0, 0};
  auto add = [&](const Matrix& a) {
    const Bytes b = bytes_of(a);
    if (groups.empty() || groups.back().count == kMatrices || sum.work + b.work > kPassBytes) {
      groups.emplace_back();
      groups.back().count = 0;
      sum = Bytes{0, 0};
    }
    Group& g = groups.back();
    g.matrix[g.count++] = a;
    sum.work += b.work;
    sum.norms += b.norms;
    most.work = std::max(most.work, sum.work);
    most.norms = std::max(most.norms, sum.norms);
  };
  for (const Matrix& a : all) {
    // a batch in pieces
    const int64_t each = std::max<int64_t>(1, kPassBytes / work_bytes(a)), size = (int64_t)a.m * a.n;
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
  Workspace work(s, most.work), norms(s, most.norms);
  for (Group& g : groups) run_group<T, MUON>(s, g, h, steps, work.data(), reinterpret_cast<double*>(norms.data()));
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
  if (dt == DType::F32) run<float, false>(s, {a}, h, steps);
  else run<__half, false>(s, {a}, h, steps);
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
