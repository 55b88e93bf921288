// Rows of logits at any alignment, for the kernels that read whole rows.
#pragma once

#include "common.h"

namespace shard {
namespace {

typedef __bf16 bf16_t;

// A row seen as 16-byte granules from the aligned address at or before it.
template <class T>
struct Row {
  static constexpr int VEC = 16 / sizeof(T);
  typedef T vec __attribute__((ext_vector_type(VEC)));
  const T* p;
  int64_t n;
  int mis;       // elements of the first granule that lie before the row
  int64_t count; // granules
  __device__ Row(const T* row, int64_t vocab) : p(row), n(vocab) {
    mis = (int)(((uintptr_t)row & 15) / sizeof(T));
    count = (n + mis + VEC - 1) / VEC;
  }
  // Granules lo .. hi - 1 lie wholly within the row.
  __device__ __forceinline__ int64_t lo() const { return mis ? 1 : 0; }
  __device__ __forceinline__ int64_t hi() const { return (n + mis) / VEC; }
  __device__ __forceinline__ vec raw(int64_t j) const { return *(const vec*)(p + (j * VEC - mis)); }
  // Elements outside the row are -inf.  Returns the index of x[0].
  __device__ __forceinline__ int64_t load(int64_t j, float (&x)[VEC]) const {
    const int64_t e0 = j * VEC - mis;
    if (e0 >= 0 && e0 + VEC <= n) {
      const vec v = *(const vec*)(p + e0);
#pragma unroll
      for (int i = 0; i < VEC; ++i) x[i] = (float)v[i];
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) x[i] = e0 + i >= 0 && e0 + i < n ? (float)p[e0 + i] : -INFINITY;
    }
    return e0;
  }
};

}  // namespace
}  // namespace shard
