// What the operators of a language model's training step share on the host: rows of tensors of any rank, dense operands,
// workspaces, and the guard of their entry points.
#pragma once
#include <new>

#include "common.hpp"
#include "device_util.hpp"
#include "stream_guard.hpp"

namespace thc {

// The float x in a tensor's type. A float operation right before the rounding to half would otherwise become one instruction with it
// (v_fma_mixlo_f16), which rounds once where the two round twice: results would differ by how the compiler arranged a kernel.
template <typename T>
__device__ __forceinline__ T rounded(float x) {
  if constexpr (sizeof(T) == 2) asm("" : "+v"(x));
  return Cvt<T>::down(x);
}

// Body of a void entry point that uses the C++ library's containers: nothing but an error leaves it.
#define THC_GUARD_ALL(...)                                             \
  try {                                                                \
    __VA_ARGS__;                                                       \
  } catch (const ::thc::Error& e_) {                                   \
    ::thc::deliver_error(e_);                                          \
  } catch (const std::bad_alloc&) {                                    \
    ::thc::deliver_error(::thc::Error("out of host memory", 0));       \
  } catch (const std::exception& e_) {                                 \
    ::thc::deliver_error(::thc::Error(e_.what(), 0));                  \
  }

// Row i of a tensor seen as rows along its last dim (unit stride) begins (i / inner) * outerStride + (i % inner) * stride elements
// into it: the leading dims merge into two at most (a matrix, a batch of sequences, a window of either).
struct Rows {
  int64_t count, length, inner, stride, outerStride;
};

// false: the last dim is strided or the leading dims do not merge.
inline bool as_rows(const AnyTensor* t, Rows* r) {
  const int nd = t->nDimension;
  if (nd == 0 || nd > kMaxDims) return false;
  r->length = t->size[nd - 1];
  if (t->stride[nd - 1] != 1 && r->length > 1) return false;
  r->count = r->inner = 1;
  r->stride = r->outerStride = 0;
  if (nd == 1) return true;
  Layout l = make_layout(nd - 1, t->size, t->stride);
  r->count = l.numel();
  collapse(l);
  if (l.dims > 2) return false;
  r->inner = l.size[l.dims - 1];
  r->stride = l.stride[l.dims - 1];
  if (l.dims == 2) r->outerStride = l.stride[0];
  return true;
}

// A tensor as an operand that kernels read: itself if it is contiguous, else a dense copy that lives as long as this.
struct Dense {
  TensorRef ref;
  DType dt;
  Dense(THCState* s, AnyTensor* t, DType d) : ref(s, tensor_new_contiguous(s, t, d)), dt(d) {}
  template <typename T>
  T* data() const {
    return static_cast<T*>(tensor_data(ref.t, dt));
  }
};

// `bytes` of device memory from the state's allocator, given back when this goes (on the stream's order with the caching allocator).
struct Workspace {
  TensorRef ref;
  Workspace(THCState* s, int64_t bytes) : ref(s, nullptr) {
    const long n = (long)((bytes + 7) / 8);
    ref.t = tensor_new_with_size(s, 1, &n, DType::I64);
  }
  char* data() const { return static_cast<char*>(tensor_data(ref.t, DType::I64)); }
};

inline bool same_sizes(const AnyTensor* a, const AnyTensor* b) {
  if (a->nDimension != b->nDimension) return false;
  for (int d = 0; d < a->nDimension; ++d)
    if (a->size[d] != b->size[d]) return false;
  return true;
}

// Whether the memory spans of two tensors meet (elements between strided ones count). What is written directly must not meet what
// is read; an output that does goes through a temporary.
inline bool spans_meet(const AnyTensor* a, DType da, const AnyTensor* b, DType db) {
  if (!a || !b || !a->storage || a->storage != b->storage || a->nDimension == 0 || b->nDimension == 0) return false;
  auto span = [](const AnyTensor* t, DType dt, int64_t* first, int64_t* last) {
    const int64_t e = (int64_t)dtype_size(dt);
    *first = t->storageOffset * e;
    *last = *first + e;
    for (int d = 0; d < t->nDimension; ++d) *last += (t->size[d] - 1) * t->stride[d] * e;
  };
  int64_t a0, a1, b0, b1;
  span(a, da, &a0, &a1);
  span(b, db, &b0, &b1);
  return a0 < b1 && b0 < a1;
}

inline bool has_elements(const AnyTensor* t) { return t->nDimension > 0 && tensor_numel(t) > 0; }

}  // namespace thc
