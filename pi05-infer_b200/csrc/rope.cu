// Rotary positions for any position, layout, rotated part and scaling: pi05_rope.
//
//   (a, b) of a pair -> (a c - b s, b c + a s),  c + i s = magnitude * exp(i angle)
//
// Memory bound: x read once, out written once.  A CTA takes a few tokens: it asks for its
// first values, works out the tokens' cos and sin into shared memory while they are on
// their way (once for all heads), then streams.  A thread keeps its place within a head
// and goes from head to head; values that pass through go by themselves, so that no warp
// does both.  32768 tokens of 32 heads of 128, half of each rotated (537 MB): 86 us;
// with a word's place worked out for every word 99 (integer arithmetic in 76% of the issue
// slots), with turned and passed words in the same warps 90.
#include <algorithm>

#include "paged.cuh"

namespace pi05 {
namespace {

constexpr int kThreads = 128;

struct RopeParams {
  int xt, xh, ot, oh;  // strides, elements
  const void* positions;
  const uint64_t* turns;
  FastDiv by_heads, by_pairs;
  int pos64, tokens, heads, dim, rotary, interleaved, back, per_cta;
  int turned, turned_lanes;  // units of a head that turn; threads to a head
  int passed, passed_lanes;  // units that pass through
  float magnitude;
};

template <class T, int V, int J>
__global__ void __launch_bounds__(kThreads) rope_kernel(const T* x, T* out, const __grid_constant__ RopeParams p) {
  extern __shared__ __align__(16) float2 cs[];  // [per_cta][rotary / 2]
  pdl_wait();
  pdl_launch_dependents();
  const int pairs = p.rotary / 2, tid = threadIdx.x;
  const long long t0 = (long long)blockIdx.x * p.per_cta;
  const int n = (int)min((long long)p.per_cta, p.tokens - t0), rows = n * p.heads;
  x += t0 * p.xt;
  out += t0 * p.ot;
  // `lanes` threads to a head's units, kThreads / lanes heads at a time, J of them at once.
  // `first`: what is done between the first loads and the first stores.
  auto stream = [&](int units, int lanes, auto load, auto store, auto first) {
    const int row0 = tid / lanes, u0 = tid - row0 * lanes, step = kThreads / lanes;
    bool begun = false;
    for (int u = u0; u < units || !begun; u += lanes) {
      const bool mine = u < units && row0 < step;
      for (int r = row0; r < rows || !begun; r += J * step) {
        Unit<T, V> unit[J];
        int token[J], head[J];
#pragma unroll
        for (int j = 0; j < J; ++j) {
          const int row = r + j * step;
          token[j] = p.by_heads.div(row);
          head[j] = row - token[j] * p.heads;
          if (mine && row < rows)
            load(unit[j], x + (long long)token[j] * p.xt + (long long)head[j] * p.xh, u);
        }
        if (!begun) first();
        begun = true;
#pragma unroll
        for (int j = 0; j < J; ++j)
          if (mine && r + j * step < rows)
            store(unit[j], out + (long long)token[j] * p.ot + (long long)head[j] * p.oh, u, token[j]);
      }
    }
  };
  stream(
      p.turned, p.turned_lanes,
      [&](Unit<T, V>& unit, const T* src, int u) { unit.load(src, u, p.turned, p.rotary, p.interleaved); },
      [&](Unit<T, V>& unit, T* dst, int u, int t) {
        unit.store(dst, u, p.turned, p.rotary, p.interleaved, cs + t * pairs);
      },
      [&]() {
        for (int i = tid; i < n * pairs; i += kThreads) {
          const int t = p.by_pairs.div(i), f = i - t * pairs;
          const long long pos = p.pos64 ? static_cast<const long long*>(p.positions)[t0 + t]
                                        : static_cast<const int32_t*>(p.positions)[t0 + t];
          cs[t * pairs + Unit<T, V>::place(f, p.turned, p.interleaved)] =
              rotation(pos, p.turns[f], p.magnitude, p.back);
        }
        __syncthreads();
      });
  if (p.passed > 0)
    stream(
        p.passed, p.passed_lanes, [&](Unit<T, V>& unit, const T* src, int u) { unit.load_row(src + p.rotary, u); },
        [&](Unit<T, V>& unit, T* dst, int u, int) { unit.store_row(dst + p.rotary, u); }, [] {});
}

template <class T, int V>
int rope_run(const void* x, void* out, RopeParams p, cudaStream_t stream) {
  constexpr int J = 4;
  p.turned = rotary_units<V>(p.rotary, p.interleaved);
  p.passed = x == out ? 0 : (p.dim - p.rotary) / V;  // in place, the rest is there already
  p.turned_lanes = std::min(p.turned, kThreads);
  p.passed_lanes = std::min(p.passed, kThreads);
  p.by_heads = FastDiv(p.heads);
  p.by_pairs = FastDiv(p.rotary / 2);
  // A few batches of loads for a CTA, but for tokens enough to fill the SMs.  The longer of
  // the two passes counts: with many tokens to a CTA, L2 has lost the sectors and lines that
  // both touch before the second comes (32768 tokens of 32 heads of 80, 40 of them turned: 81
  // us; by the turned part alone 137).
  const int fill = std::max(1, 4 * J * (kThreads / std::max(p.turned_lanes, p.passed_lanes)) / p.heads);
  p.per_cta = std::max(1, std::min({fill, p.tokens / (4 * kSMs), 48 * 1024 / (p.rotary / 2 * (int)sizeof(float2))}));
  return launch_pdl(rope_kernel<T, V, J>, dim3((p.tokens + p.per_cta - 1) / p.per_cta), dim3(kThreads),
                    (size_t)p.per_cta * (p.rotary / 2) * sizeof(float2), stream, pdl_enabled(),
                    static_cast<const T*>(x), static_cast<T*>(out), p);
}

template <class T>
int rope_type(const void* x, void* out, const RopeParams& p, cudaStream_t stream) {
  switch (unit_values(sizeof(T), p.rotary, p.interleaved, p.dim, {p.xt, p.xh, p.ot, p.oh}, x, out)) {
    case 8:
      if constexpr (sizeof(T) == 2) return rope_run<T, 8>(x, out, p, stream);
    case 4: return rope_run<T, 4>(x, out, p, stream);
    case 2: return rope_run<T, 2>(x, out, p, stream);
    default: return rope_run<T, 1>(x, out, p, stream);
  }
}

}  // namespace
}  // namespace pi05

using namespace pi05;

extern "C" int pi05_rope(const Pi05RopeArgs* a, const Pi05Rotary* rotary, void* stream) {
  if (a == nullptr || rotary == nullptr || rotary->turns == nullptr ||
      (a->tokens > 0 && (a->x == nullptr || a->out == nullptr || a->positions == nullptr))) {
    set_last_error("rope: null pointer");
    return PI05_ERR_INVALID_ARG;
  }
  if (a->dtype != PI05_BF16 && a->dtype != PI05_FP16 && a->dtype != PI05_FP32) {
    set_last_error("rope: dtype %d is not bf16, fp16 or fp32", a->dtype);
    return PI05_ERR_INVALID_ARG;
  }
  const int r = rotary->rotary_dim;
  if (a->tokens < 0 || a->heads <= 0 || a->head_dim <= 0 || r <= 0 || r % 2 || r > a->head_dim || r > kMaxRotary ||
      (long long)a->heads * a->head_dim > (1 << 24)) {
    set_last_error("rope: bad shape tokens=%d heads=%d head_dim=%d rotary_dim=%d", a->tokens, a->heads, a->head_dim, r);
    return PI05_ERR_SHAPE;
  }
  const long long xt = stride_of(a->tokens, a->x_token_stride), xh = stride_of(a->heads, a->x_head_stride);
  const long long ot = stride_of(a->tokens, a->out_token_stride), oh = stride_of(a->heads, a->out_head_stride);
  if (a->x == a->out && (xt != ot || xh != oh)) {
    set_last_error("rope: in place needs the same strides");
    return PI05_ERR_INVALID_ARG;
  }
  for (long long stride : {xt, xh, ot, oh})
    if (stride < 0 || stride >= 1ll << 31) {
      set_last_error("rope: stride of %lld elements", stride);
      return PI05_ERR_SHAPE;
    }
  if (!aligned_to(a->dtype == PI05_FP32 ? 4 : 2, a->x, a->out) || !aligned_to(a->positions_i64 ? 8 : 4, a->positions) ||
      !aligned_to(8, rotary->turns)) {
    set_last_error("rope: pointer not aligned to its elements");
    return PI05_ERR_ALIGN;
  }
  if (a->tokens == 0) return PI05_OK;
  RopeParams p;
  p.xt = (int)xt;
  p.xh = (int)xh;
  p.ot = (int)ot;
  p.oh = (int)oh;
  p.positions = a->positions;
  p.turns = rotary->turns;
  p.pos64 = a->positions_i64;
  p.tokens = a->tokens;
  p.heads = a->heads;
  p.dim = a->head_dim;
  p.rotary = r;
  p.interleaved = rotary->interleaved;
  p.back = a->transpose;
  p.magnitude = rotary->magnitude;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (a->dtype == PI05_BF16) return rope_type<__nv_bfloat16>(a->x, a->out, p, st);
  if (a->dtype == PI05_FP16) return rope_type<__half>(a->x, a->out, p, st);
  return rope_type<float>(a->x, a->out, p, st);
}
