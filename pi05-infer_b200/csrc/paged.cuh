// Shared by the text-decoding kernels (rope.cu, paged_kv.cu, paged_attention.cu):
// element types, the rotation, and the address of a cache row.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include <atomic>

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

// Two 16-bit elements of a 32-bit word (lower half first).
template <class T>
__device__ __forceinline__ float2 unpack2(uint32_t u);
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t u) {
  return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t u) {
  return __half22float2(*reinterpret_cast<const __half2*>(&u));
}

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

// What one thread does at a time: V pairs of the half layout (two words of V elements),
// or V / 2 pairs of the interleaved one, or a word of the values that pass through.  V = 1
// takes single elements, a pair at a time.
template <int V>
__host__ __device__ __forceinline__ int rotary_units(int rotary, bool interleaved) {
  return rotary / (interleaved && V > 1 ? V : 2 * V);
}

// (a, b) -> (a c - b s, b c + a s)
__device__ __forceinline__ void turn(float& a, float& b, float2 r) {
  const float x = a;
  a = x * r.x - b * r.y;
  b = b * r.x + x * r.y;
}

// A unit in registers between its load and its store, so that a thread has several
// loads on their way before it needs the first.  cs: cos and sin of the pairs, pair i at
// place(i): two pairs to 16 bytes, and these of neighbouring units side by side, so that
// the units of a warp read them without bank conflicts.
template <class T, int V>
struct Unit;

template <class T>
struct Unit<T, 1> {
  T a, b;
  static __device__ __forceinline__ int place(int i, int, bool) { return i; }
  __device__ __forceinline__ void load_row(const T* src, int u) { a = src[u]; }
  __device__ __forceinline__ void store_row(T* dst, int u) const { dst[u] = a; }
  __device__ __forceinline__ void load(const T* src, int u, int turned, int rotary, bool interleaved) {
    if (u >= turned) {
      a = src[rotary + u - turned];
    } else {
      a = src[interleaved ? 2 * u : u];
      b = src[interleaved ? 2 * u + 1 : rotary / 2 + u];
    }
  }
  __device__ __forceinline__ void store(T* dst, int u, int turned, int rotary, bool interleaved,
                                        const float2* cs) const {
    if (u >= turned) {
      dst[rotary + u - turned] = a;
    } else {
      float x = to_f32(a), y = to_f32(b);
      turn(x, y, cs[u]);
      dst[interleaved ? 2 * u : u] = from_f32<T>(x);
      dst[interleaved ? 2 * u + 1 : rotary / 2 + u] = from_f32<T>(y);
    }
  }
};

__device__ __forceinline__ uint4 ld16(const void* p) { return *static_cast<const uint4*>(p); }
__device__ __forceinline__ void st16(void* p, const uint4& v) { *static_cast<uint4*>(p) = v; }

// 16-byte words: V = 8 of the 16-bit types, 4 of fp32.
template <class T, int V>
struct Unit {
  static_assert(V * sizeof(T) == 16, "a word");
  uint4 a, b;
  static __device__ __forceinline__ int place(int i, int turned, bool interleaved) {
    const int per = interleaved ? V / 2 : V;
    return (i % per / 2 * turned + i / per) * 2 + (i & 1);
  }
  __device__ __forceinline__ void load_row(const T* src, int u) { a = ld16(src + u * V); }
  __device__ __forceinline__ void store_row(T* dst, int u) const { st16(dst + u * V, a); }
  __device__ __forceinline__ void load(const T* src, int u, int turned, int rotary, bool interleaved) {
    a = ld16(src + (u < turned ? u * V : rotary + (u - turned) * V));
    if (u < turned && !interleaved) b = ld16(src + rotary / 2 + u * V);
  }
  // r: cos and sin of two pairs.  Interleaved: each word a pair (16 bit), or each two (fp32).
  static __device__ __forceinline__ void turn_pairs(uint32_t& x, uint32_t& y, float4 r) {
    float2 v = unpack2<T>(x), w = unpack2<T>(y);
    turn(v.x, v.y, make_float2(r.x, r.y));
    turn(w.x, w.y, make_float2(r.z, r.w));
    x = pack2<T>(v.x, v.y);
    y = pack2<T>(w.x, w.y);
  }
  // Half layout: two values of one half and their partners.
  static __device__ __forceinline__ void turn_halves(uint32_t& x, uint32_t& y, float4 r) {
    float2 v = unpack2<T>(x), w = unpack2<T>(y);
    turn(v.x, w.x, make_float2(r.x, r.y));
    turn(v.y, w.y, make_float2(r.z, r.w));
    x = pack2<T>(v.x, v.y);
    y = pack2<T>(w.x, w.y);
  }
  static __device__ __forceinline__ void turn_f32(uint32_t& x, uint32_t& y, float c, float s) {
    float v = __uint_as_float(x), w = __uint_as_float(y);
    turn(v, w, make_float2(c, s));
    x = __float_as_uint(v);
    y = __float_as_uint(w);
  }
  __device__ __forceinline__ void store(T* dst, int u, int turned, int rotary, bool interleaved, const float2* cs) {
    if (u >= turned) {
      st16(dst + rotary + (u - turned) * V, a);
      return;
    }
    const float4* r = reinterpret_cast<const float4*>(cs) + u;
    if (interleaved) {
      if constexpr (V == 8) {
        turn_pairs(a.x, a.y, r[0]);
        turn_pairs(a.z, a.w, r[turned]);
      } else {
        turn_f32(a.x, a.y, r[0].x, r[0].y);
        turn_f32(a.z, a.w, r[0].z, r[0].w);
      }
      st16(dst + u * V, a);
    } else {
      if constexpr (V == 8) {
        turn_halves(a.x, b.x, r[0]);
        turn_halves(a.y, b.y, r[turned]);
        turn_halves(a.z, b.z, r[2 * turned]);
        turn_halves(a.w, b.w, r[3 * turned]);
      } else {
        turn_f32(a.x, b.x, r[0].x, r[0].y);
        turn_f32(a.y, b.y, r[0].z, r[0].w);
        turn_f32(a.z, b.z, r[turned].x, r[turned].y);
        turn_f32(a.w, b.w, r[turned].z, r[turned].w);
      }
      st16(dst + u * V, a);
      st16(dst + rotary / 2 + u * V, b);
    }
  }
};

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
  int* ticket;     // of an append
  int* tickets;    // of an eviction's sequences
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

// Whether every pointer (or none) starts on a multiple of n bytes.
template <class... P>
bool aligned_to(size_t n, P... p) {
  return (((reinterpret_cast<uintptr_t>(p) % n) == 0) && ...);
}

// Lets a kernel have `bytes` of dynamic shared memory, once for each device (the call
// costs a microsecond).  `done`: a static of the kernel's own.
template <class K>
int allow_smem(K kernel, int bytes, std::atomic<uint64_t>* done, const char* op) {
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  const uint64_t bit = 1ull << (device & 63);
  if (e == cudaSuccess && device < 64 && (done->load(std::memory_order_relaxed) & bit)) return PI05_OK;
  if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) {
    set_last_error("%s: %s", op, cudaGetErrorString(e));
    return PI05_ERR_LAUNCH;
  }
  done->fetch_or(bit, std::memory_order_relaxed);
  return PI05_OK;
}

// Checks the struct and lays out its workspace.
int paged_check(const Pi05PagedCache* c, const char* op, Pages* out);

// Workspace of a cache: status word and ticket in the first 16640 bytes (as in the
// engine's workspace, so that the same status call reads it), then the eviction's tickets
// and move lists.
inline size_t paged_moves_bytes(const Pi05PagedCache* c) {
  return (size_t)c->batch * (1 + c->n_kv_heads * ((size_t)c->pages_per_seq * c->page_size + 2)) * sizeof(int32_t);
}

}  // namespace pi05
