// Rows at any element address as runs of 16-byte vectors, and packed f32 arithmetic: shared by the kernels that read rows of logits.
#pragma once
#include "common.cuh"
#include <type_traits>

namespace cb {

// ---- layout of a row in 16-byte vectors ---------------------------------------------------------------------------
// A row may start at any element address.  Its vectors are those of memory: vector v covers the 16 bytes at (address rounded
// down) + 16 v, its element e is row element v VEC + e - head.  The first and the last vector may hold elements of the
// neighbouring rows ("foreign"); they are never the first bytes before, or the last after, the whole tensor: there the vector is
// fetched element by element.
template <typename T> struct RowVecs {
  const unsigned char* base;     // address of vector 0
  int head;                      // foreign elements at the start of vector 0
  int nvec;
  __device__ __forceinline__ RowVecs(const T* row, int V) {
    const uint64_t a = reinterpret_cast<uint64_t>(row);
    base = reinterpret_cast<const unsigned char*>(a & ~15ull);
    head = (int)(a & 15) / (int)sizeof(T);
    nvec = (head + V + Elem<T>::VEC - 1) / Elem<T>::VEC;
  }
};

// two f32 operations an instruction
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, z, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
      "fma.rn.f32x2 w, x, y, z;\n\tmov.b64 {%0, %1}, w;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 w, x, y;\n\tmov.b64 {%0, %1}, w;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 w, x, y;\n\tmov.b64 {%0, %1}, w;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

}  // namespace cb
