// Rotary positions for any position, layout, rotated part and scaling: pi05_rope.
//
//   (a, b) of a pair -> (a c - b s, b c + a s),  c + i s = magnitude * exp(i angle)
//
// Memory bound: x read once, out written once.  A token's cos and sin are worked out
// once per CTA into shared memory and used for all its heads.
#include "paged.cuh"

namespace pi05 {
namespace {

constexpr int kThreads = 256;

struct RopeParams {
  long long xt, xh, ot, oh;  // strides, elements
  const void* positions;
  const uint64_t* turns;
  int pos64, tokens, heads, dim, rotary, interleaved, back, per_cta;
  float magnitude;
};

template <class T, int V>
__global__ void __launch_bounds__(kThreads) rope_kernel(const T* x, T* out, RopeParams p) {
  extern __shared__ float2 cs[];  // [per_cta][rotary / 2]
  pdl_wait();
  pdl_launch_dependents();
  const int pairs = p.rotary / 2;
  const int turned = rotary_units<V>(p.rotary, p.interleaved);
  const int units = turned + (x == out ? 0 : (p.dim - p.rotary) / V);  // in place, the rest is there already
  for (long long t0 = (long long)blockIdx.x * p.per_cta; t0 < p.tokens; t0 += (long long)gridDim.x * p.per_cta) {
    const int n = min((long long)p.per_cta, p.tokens - t0);
    for (int i = threadIdx.x; i < n * pairs; i += kThreads) {
      const int t = i / pairs, f = i - t * pairs;
      const long long pos = p.pos64 ? static_cast<const long long*>(p.positions)[t0 + t]
                                    : static_cast<const int32_t*>(p.positions)[t0 + t];
      cs[i] = rotation(pos, p.turns[f], p.magnitude, p.back);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n * p.heads * units; i += kThreads) {
      const int row = i / units, u = i - row * units, t = row / p.heads, h = row - t * p.heads;
      const T* src = x + (t0 + t) * p.xt + h * p.xh;
      T* dst = out + (t0 + t) * p.ot + h * p.oh;
      if (u < turned) {
        rotate_unit<T, V>(src, dst, u, p.rotary, p.interleaved, cs + t * pairs);
      } else {
        Chunk<T, V> c;
        const int at = p.rotary + (u - turned) * V;
        c.load(src + at);
        c.store(dst + at);
      }
    }
    __syncthreads();
  }
}

template <class T>
int rope_run(const void* x, void* out, RopeParams p, cudaStream_t stream) {
  constexpr int kVec = 8;
  const long long step = 16 / (long long)sizeof(T);
  // 16-byte chunks need every row, and the partner half of a row, on a 16-byte boundary.
  const bool vec = aligned16(x) && aligned16(out) && p.xt % step == 0 && p.xh % step == 0 && p.ot % step == 0 &&
                   p.oh % step == 0 && p.dim % kVec == 0 && p.rotary % (p.interleaved ? kVec : 2 * kVec) == 0;
  p.per_cta = 1;
  const size_t smem = (size_t)p.per_cta * (p.rotary / 2) * sizeof(float2);
  const int grid = (int)std::min<long long>((p.tokens + p.per_cta - 1) / p.per_cta, kSMs * 8);
  return launch_pdl(vec ? rope_kernel<T, kVec> : rope_kernel<T, 1>, dim3(grid), dim3(kThreads), smem, stream,
                    pdl_enabled(), static_cast<const T*>(x), static_cast<T*>(out), p);
}

}  // namespace
}  // namespace pi05

using namespace pi05;

extern "C" int pi05_rope(const void* x, void* out, int dtype, int tokens, int heads, int head_dim,
                         long long x_token_stride, long long x_head_stride, long long out_token_stride,
                         long long out_head_stride, const void* positions, int positions_i64, const Pi05Rotary* rotary,
                         int transpose, void* stream) {
  if (rotary == nullptr || (tokens > 0 && (x == nullptr || out == nullptr || positions == nullptr)) ||
      rotary->turns == nullptr) {
    set_last_error("rope: null pointer");
    return PI05_ERR_INVALID_ARG;
  }
  if (dtype != PI05_BF16 && dtype != PI05_FP16 && dtype != PI05_FP32) {
    set_last_error("rope: dtype %d is not bf16, fp16 or fp32", dtype);
    return PI05_ERR_INVALID_ARG;
  }
  const int r = rotary->rotary_dim;
  if (tokens < 0 || heads <= 0 || head_dim <= 0 || r <= 0 || r % 2 || r > head_dim || r > kMaxRotary ||
      (long long)heads * head_dim > (1 << 24)) {
    set_last_error("rope: bad shape tokens=%d heads=%d head_dim=%d rotary_dim=%d", tokens, heads, head_dim, r);
    return PI05_ERR_SHAPE;
  }
  if (x == out && (x_token_stride != out_token_stride || x_head_stride != out_head_stride)) {
    set_last_error("rope: in place needs the same strides");
    return PI05_ERR_INVALID_ARG;
  }
  if (tokens == 0) return PI05_OK;
  RopeParams p;
  p.xt = x_token_stride;
  p.xh = x_head_stride;
  p.ot = out_token_stride;
  p.oh = out_head_stride;
  p.positions = positions;
  p.turns = rotary->turns;
  p.pos64 = positions_i64;
  p.tokens = tokens;
  p.heads = heads;
  p.dim = head_dim;
  p.rotary = r;
  p.interleaved = rotary->interleaved;
  p.back = transpose;
  p.magnitude = rotary->magnitude;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == PI05_BF16) return rope_run<__nv_bfloat16>(x, out, p, st);
  if (dtype == PI05_FP16) return rope_run<__half>(x, out, p, st);
  return rope_run<float>(x, out, p, st);
}
