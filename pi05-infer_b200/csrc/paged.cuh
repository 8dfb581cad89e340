// Shared by the text-decoding kernels (rope.cu, paged_kv.cu, paged_attention.cu):
// element types, the rotation, and the address of a cache row.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include <atomic>
#include <initializer_list>

#include "../../include/pi05_b200.h"
#include "host_util.h"
#include "ptx.cuh"

namespace pi05 {

constexpr int kMaxRotary = 512;
constexpr int kSMs = 148;

// Whether every pointer (or none) starts on a multiple of n bytes.
template <class... P>
bool aligned_to(size_t n, P... p) {
  return (((reinterpret_cast<uintptr_t>(p) % n) == 0) && ...);
}

// The stride of a dimension of one element means nothing.
inline long long stride_of(int elements, long long stride) { return elements == 1 ? 0 : stride; }

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
// The angle of a position is position * turns / 2^64 turns.  The product wraps at one turn by
// itself, for any sign, so it is off by the table's 2^-65 turn for each position and no more; a
// 32-bit float angle would be off by 2^-24 of its size, 0.06 rad at position 10^6.  Of its top 32
// bits (rounded: 2^-33 turn) what lies beyond the nearest quarter turn, 1/8 turn at most, becomes a
// float, 2^-28 turn at most; the whole angle as a float would lose 2^-26.
__device__ __forceinline__ float2 rotation(long long position, uint64_t turns, float magnitude, bool back) {
  const uint32_t phase = (uint32_t)(((uint64_t)position * turns + 0x80000000ull) >> 32);
  const uint32_t quarter = (phase + (1u << 29)) >> 30;
  float s, c;
  sincospif((float)(int32_t)(phase - (quarter << 30)) * 0x1p-31f, &s, &c);
  const float across = quarter & 1 ? s : c, up = quarter & 1 ? c : s;
  c = (quarter ^ (quarter >> 1)) & 1 ? -across : across;
  s = (quarter >> 1 & 1) != back ? -up : up;
  return make_float2(c * magnitude, s * magnitude);
}

// What one thread does at a time: V pairs of the half layout (two words of V elements),
// or V / 2 pairs of the interleaved one, or a word of the values that pass through.  V = 1
// takes single elements, a pair at a time (half layout with an odd number of pairs, or
// rows at odd elements).
template <int V>
__host__ __device__ __forceinline__ int rotary_units(int rotary, bool interleaved) {
  return rotary / (interleaved && V > 1 ? V : 2 * V);
}

// (a, b) -> (a c - b s, b c + a s); which product is fused stands here, so that every word
// width gives the same bits.
__device__ __forceinline__ void turn(float& a, float& b, float2 r) {
  const float x = a;
  a = fmaf(-b, r.y, x * r.x);
  b = fmaf(x, r.y, b * r.x);
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

// 4 * NW bytes that are loaded and stored at once, and the 32-bit words in them.
template <int NW>
struct WordOf;
template <>
struct WordOf<4> {
  using type = uint4;
  static __device__ __forceinline__ void split(uint32_t (&x)[4], uint4 v) {
    x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
  }
  static __device__ __forceinline__ uint4 join(const uint32_t (&x)[4]) { return make_uint4(x[0], x[1], x[2], x[3]); }
};
template <>
struct WordOf<2> {
  using type = uint2;
  static __device__ __forceinline__ void split(uint32_t (&x)[2], uint2 v) { x[0] = v.x, x[1] = v.y; }
  static __device__ __forceinline__ uint2 join(const uint32_t (&x)[2]) { return make_uint2(x[0], x[1]); }
};
template <>
struct WordOf<1> {
  using type = uint32_t;
  static __device__ __forceinline__ void split(uint32_t (&x)[1], uint32_t v) { x[0] = v; }
  static __device__ __forceinline__ uint32_t join(const uint32_t (&x)[1]) { return x[0]; }
};

// Words of 4, 8 or 16 bytes: V = 2, 4 or 8 of the 16-bit types, 2 or 4 of fp32.
template <class T, int V>
struct Unit {
  static constexpr int NW = V * sizeof(T) / 4;
  using Words = WordOf<NW>;
  using Word = typename Words::type;
  Word a, b;
  static __device__ __forceinline__ int place(int i, int turned, bool interleaved) {
    const int per = interleaved ? V / 2 : V;
    if (V == 2 && interleaved) return i;  // a pair to a unit
    return (i % per / 2 * turned + i / per) * 2 + (i & 1);
  }
  static __device__ __forceinline__ Word get(const T* p) { return *reinterpret_cast<const Word*>(p); }
  static __device__ __forceinline__ void put(T* p, const Word& v) { *reinterpret_cast<Word*>(p) = v; }
  __device__ __forceinline__ void load_row(const T* src, int u) { a = get(src + u * V); }
  __device__ __forceinline__ void store_row(T* dst, int u) const { put(dst + u * V, a); }
  __device__ __forceinline__ void load(const T* src, int u, int turned, int rotary, bool interleaved) {
    a = get(src + (u < turned ? u * V : rotary + (u - turned) * V));
    if (u < turned && !interleaved) b = get(src + rotary / 2 + u * V);
  }
  // One pair in a word of two 16-bit values, or in two words of fp32.
  static __device__ __forceinline__ void turn_word(uint32_t& x, float c, float s) {
    float2 v = unpack2<T>(x);
    turn(v.x, v.y, make_float2(c, s));
    x = pack2<T>(v.x, v.y);
  }
  static __device__ __forceinline__ void turn_f32(uint32_t& x, uint32_t& y, float c, float s) {
    float v = __uint_as_float(x), w = __uint_as_float(y);
    turn(v, w, make_float2(c, s));
    x = __float_as_uint(v);
    y = __float_as_uint(w);
  }
  // Half layout: two 16-bit values of one half and their partners.
  static __device__ __forceinline__ void turn_halves(uint32_t& x, uint32_t& y, float4 r) {
    float2 v = unpack2<T>(x), w = unpack2<T>(y);
    turn(v.x, w.x, make_float2(r.x, r.y));
    turn(v.y, w.y, make_float2(r.z, r.w));
    x = pack2<T>(v.x, v.y);
    y = pack2<T>(w.x, w.y);
  }
  __device__ __forceinline__ void store(T* dst, int u, int turned, int rotary, bool interleaved, const float2* cs) {
    if (u >= turned) {
      put(dst + rotary + (u - turned) * V, a);
      return;
    }
    const float4* r = reinterpret_cast<const float4*>(cs) + u;  // two pairs
    uint32_t x[NW], y[NW];
    Words::split(x, a);
    if (interleaved) {
      if constexpr (V == 2) {
        if constexpr (sizeof(T) == 2) turn_word(x[0], cs[u].x, cs[u].y);
        else turn_f32(x[0], x[1], cs[u].x, cs[u].y);
      } else {
#pragma unroll
        for (int g = 0; g < V / 4; ++g) {
          const float4 v = r[g * turned];
          if constexpr (sizeof(T) == 2) {
            turn_word(x[2 * g], v.x, v.y);
            turn_word(x[2 * g + 1], v.z, v.w);
          } else {
            turn_f32(x[4 * g], x[4 * g + 1], v.x, v.y);
            turn_f32(x[4 * g + 2], x[4 * g + 3], v.z, v.w);
          }
        }
      }
    } else {
      Words::split(y, b);
#pragma unroll
      for (int g = 0; g < V / 2; ++g) {
        const float4 v = r[g * turned];
        if constexpr (sizeof(T) == 2) {
          turn_halves(x[g], y[g], v);
        } else {
          turn_f32(x[2 * g], y[2 * g], v.x, v.y);
          turn_f32(x[2 * g + 1], y[2 * g + 1], v.z, v.w);
        }
      }
      put(dst + rotary / 2 + u * V, Words::join(y));
    }
    put(dst + u * V, Words::join(x));
  }
};

// Values to a unit: as many as a word of 16, 8 or 4 bytes holds (or one) that divide the pairs' halves,
// the head, every stride and every pointer.  `bytes`: of a value.  Single values cost an
// instruction each: 32768 tokens of 32 heads of 72 (36 pairs, no multiple of the 8
// values of 16 bytes) turn in 51 us with 8-byte words and took 160 with single values; the append of 16384
// tokens of 8 + 8 heads of 72 takes 30 instead of 93.
template <class... P>
int unit_values(int bytes, int rotary, bool interleaved, int dim, std::initializer_list<long long> strides,
                P... pointers) {
  for (int v = 16 / bytes; v > 1; v /= 2) {
    bool fits = (interleaved ? rotary : rotary / 2) % v == 0 && dim % v == 0 && aligned_to(v * bytes, pointers...);
    for (long long s : strides) fits = fits && s % v == 0;
    if (fits) return v;
  }
  return 1;
}

// ---- division by a number known at launch (n < 2^31) ------------------------
// By a multiplication, after Granlund and Montgomery, "Division by invariant integers using
// multiplication" (1994).
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
  // Eviction: tickets of the sequences; of each (sequence, head) the number of its moves (-1: the
  // sequence stays as it is) and the rows left; and a list.
  int* tickets;
  int2* moves;
  int32_t* move_list;
  FastDiv page_div;
  int num_pages, page_size, heads, dim, batch, pitch, capacity;
  bool list_by_slot;

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
// engine's workspace, so that the same status call reads it); then, for a cache that keeps
// weights and positions, the eviction's tickets, counts and lists.
inline size_t paged_pairs(const Pi05PagedCache* c) { return (size_t)c->batch * c->n_kv_heads; }

// A list has an entry for each row that the table can reach, or, where that takes more than 16 MB
// and more than the pool's rows, stands at the rows' own slots: 4 bytes a slot of the pool, however
// long the table, for a look into the table with each entry.
inline bool paged_list_by_slot(const Pi05PagedCache* c) {
  const size_t reach = paged_pairs(c) * c->pages_per_seq * c->page_size;
  return reach * sizeof(int32_t) > (16u << 20) && (size_t)c->num_pages * c->n_kv_heads * c->page_size < reach;
}

inline size_t paged_moves_bytes(const Pi05PagedCache* c) {
  if (c->weight == nullptr || c->pos == nullptr) return 0;
  const size_t rows = paged_list_by_slot(c) ? (size_t)c->num_pages * c->n_kv_heads * c->page_size
                                            : paged_pairs(c) * c->pages_per_seq * c->page_size;
  return ((size_t)c->batch + (c->batch & 1) + 2 * paged_pairs(c) + rows) * sizeof(int32_t);
}

}  // namespace pi05
