// Shared by the text-decoding kernels (rope.cu, paged_kv.cu, paged_attention.cu):
// element types, the rotation, and the address of a cache row.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "../../include/pi05_b200.h"
#include "host_util.h"
#include "ptx.cuh"

namespace pi05 {

constexpr int kMaxRotary = 512;
constexpr int kSMs = 148;

// ---- element types ---------------------------------------------------------
template <class T>
__device__ __forceinline__ float to_f32(T x);
template <>
__device__ __forceinline__ float to_f32(float x) { return x; }
template <>
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <>
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }

template <class T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32(float x) { return __float2bfloat16(x); }
template <>
__device__ __forceinline__ __half from_f32(float x) { return __float2half_rn(x); }

// Two values as one 32-bit word of 16-bit elements (lower half first).
template <class T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// V consecutive elements, moved by 16-byte words (V = 8, aligned) or one by one.
template <class T, int V>
struct Chunk {
  __align__(16) T e[V];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (V * sizeof(T) % 16 == 0) {
#pragma unroll
      for (int i = 0; i < (int)(V * sizeof(T) / 16); ++i)
        reinterpret_cast<uint4*>(e)[i] = reinterpret_cast<const uint4*>(p)[i];
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) e[i] = p[i];
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (V * sizeof(T) % 16 == 0) {
#pragma unroll
      for (int i = 0; i < (int)(V * sizeof(T) / 16); ++i)
        reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(e)[i];
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) p[i] = e[i];
    }
  }
};

// ---- rotation --------------------------------------------------------------
// The angle of a position is position * turns / 2^64 turns.  The product wraps at
// one turn by itself, for any sign, so its top 32 bits (rounded) are the angle to
// 2^-33 turn however far the position; a 32-bit float angle would be off by
// 2^-24 of its size, 0.06 rad at position 10^6.
__device__ __forceinline__ float2 rotation(long long position, uint64_t turns, float magnitude, bool back) {
  const uint64_t phase = (uint64_t)position * turns + 0x80000000ull;
  const float half_turns = (float)(int32_t)(phase >> 32) * 0x1p-31f;
  float s, c;
  sincospif(half_turns, &s, &c);
  return make_float2(c * magnitude, (back ? -s : s) * magnitude);
}

// What one thread does at a time: V pairs of the half layout (two chunks of V), or
// V / 2 pairs (one chunk; V = 1: one pair) of the interleaved one, or a chunk of
// the values that pass through.
template <int V>
__host__ __device__ __forceinline__ int rotary_units(int rotary, bool interleaved) {
  return interleaved ? (V == 1 ? rotary / 2 : rotary / V) : rotary / (2 * V);
}

// cs: cos, sin of each pair.
template <class T, int V>
__device__ __forceinline__ void rotate_unit(const T* src, T* dst, int unit, int rotary, bool interleaved,
                                            const float2* cs) {
  if (!interleaved) {
    Chunk<T, V> a, b;
    const int i = unit * V;
    a.load(src + i);
    b.load(src + rotary / 2 + i);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float2 r = cs[i + j];
      const float x = to_f32(a.e[j]), y = to_f32(b.e[j]);
      a.e[j] = from_f32<T>(x * r.x - y * r.y);
      b.e[j] = from_f32<T>(y * r.x + x * r.y);
    }
    a.store(dst + i);
    b.store(dst + rotary / 2 + i);
  } else {
    constexpr int W = V == 1 ? 2 : V;
    Chunk<T, W> a;
    const int i = unit * W;
    a.load(src + i);
#pragma unroll
    for (int j = 0; j < W; j += 2) {
      const float2 r = cs[(i + j) / 2];
      const float x = to_f32(a.e[j]), y = to_f32(a.e[j + 1]);
      a.e[j] = from_f32<T>(x * r.x - y * r.y);
      a.e[j + 1] = from_f32<T>(y * r.x + x * r.y);
    }
    a.store(dst + i);
  }
}

// ---- division by a number known at launch (n < 2^31) ------------------------
struct FastDiv {
  uint32_t mul, shift, d;
  FastDiv() = default;
  __host__ explicit FastDiv(uint32_t div) : d(div) {
    shift = 0;
    while ((1ull << shift) < div) ++shift;
    mul = (uint32_t)((((1ull << shift) - div) << 32) / div + 1);
  }
  __device__ __forceinline__ uint32_t div(uint32_t n) const { return (__umulhi(n, mul) + n) >> shift; }
};

// ---- the cache as the kernels take it ---------------------------------------
struct Pages {
  char* k;
  char* v;
  long long page_stride, head_stride, row_stride;  // bytes
  float* weight;
  int32_t* pos;
  const int32_t* table;
  int32_t* counts;
  int* status;
  int* ticket;
  int32_t* moves;  // eviction: per (sequence, head) two counts and a list of `capacity`
  FastDiv page_div;
  int num_pages, page_size, heads, dim, batch, pitch, capacity;

  __device__ __forceinline__ int rows(int b) const { return min(max(counts[b], 0), capacity); }
  // Page of row r (r < capacity) as the table has it, and its line.
  __device__ __forceinline__ int page_of(int b, int r, int* line) const {
    const int p = (int)page_div.div((uint32_t)r);
    *line = r - p * page_size;
    return table[(size_t)b * pitch + p];
  }
  __device__ __forceinline__ bool real(int page) const { return (unsigned)page < (unsigned)num_pages; }
  __device__ __forceinline__ size_t row_at(int page, int head, int line) const {
    return (size_t)(page * page_stride + head * head_stride + line * row_stride);
  }
  __device__ __forceinline__ size_t slot_at(int page, int head, int line) const {
    return ((size_t)page * heads + head) * page_size + line;
  }
};

// Checks the struct and lays out its workspace.
int paged_check(const Pi05PagedCache* c, const char* op, Pages* out);

// Workspace of a cache: status word and ticket in the first 16640 bytes (as in the
// engine's workspace, so that the same status call reads it), then the eviction's
// move lists.
inline size_t paged_moves_bytes(const Pi05PagedCache* c) {
  return (size_t)c->batch * c->n_kv_heads * ((size_t)c->pages_per_seq * c->page_size + 2) * sizeof(int32_t);
}

}  // namespace pi05
