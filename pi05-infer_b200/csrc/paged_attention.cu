// Attention of one new token of each sequence over its pages, split over the cache's
// rows and joined: pi05_paged_attention.
//
//   s_r = scale q . k_r,   m = max s,   l = sum 2^(s_r - m),   o = sum 2^(s_r - m) v_r / l
//
// (s in units of log2, so that one exp2 serves).  Bound: HBM, every k and v row read
// once for all query heads of its key-value head.
//
// Work: a sequence's rows are cut into blocks of 64; the blocks of all (sequence, head)
// pairs, laid end to end, are dealt out in equal contiguous shares to a fixed grid, so
// lengths may differ at will and the host need not know them.  A share that covers a
// whole pair writes its result; pairs cut between CTAs leave fp32 partials (o, m, l)
// that the finish kernel adds up in order.
//
// A warp takes 16 rows at a time, in a cp.async ring of its own (no block barrier in
// the loop).  The products run on the tensor cores with the rows as M:  S^T = K q^T
// (16 rows x 8 heads), then O^T += V^T P^T, where the probabilities pass from one
// fragment layout to the other by a matrix transpose in registers; with the heads as
// N = 8, half as many products and accumulators as with 16 padded query rows.  The
// probabilities enter the second product in the cache's 16-bit type (2^-9 relative for
// bf16, the size of the output's own rounding); m, l and o stay fp32, l sums the
// unrounded ones.
#include <algorithm>

#include "paged.cuh"

namespace pi05 {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kWarpRows = 16;
constexpr int kBlockRows = kWarps * kWarpRows;
constexpr int kStages = 3;
constexpr float kLn2 = 0.69314718055994530942f;

struct AttnParams {
  Pages c;
  const void* q;
  void* out;
  float* lse;
  const uint8_t* valid;
  long long qt, qh, valid_pitch;
  int valid_rows;
  int q_heads, group, parts;  // query heads per key-value head, cut into `parts` of at most 8 NT heads
  float scale_log2;
  int track, n_ctas;
  // scratch
  float* part_o;    // [2 n_ctas][8 NT][dim]
  float2* part_ml;  // [2 n_ctas][8 NT]
  int2* row_info;   // [rows]: first partial slot (-1: done), last CTA
  float* row_lse;   // [rows][8 NT] log2 units, of the rows done in one piece
  float* scores;    // [rows][capacity][8 NT], log2 units (track)
};

template <class T>
__device__ __forceinline__ void mma16816(float* c, const uint32_t* a, const uint32_t* b);
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float* c, const uint32_t* a, const uint32_t* b) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
template <>
__device__ __forceinline__ void mma16816<__half>(float* c, const uint32_t* a, const uint32_t* b) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}

__device__ __forceinline__ void ldsm4(uint32_t* r, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldsm4_trans(uint32_t* r, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// 16 bytes through L2, or 16 zero bytes (nothing is read then).
__device__ __forceinline__ void cp_async_16_or_zero(uint32_t dst, const void* src, bool read) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(read ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

template <int DP>
struct Tile {
  static constexpr int kPitch = DP * 2 + 16;  // bytes; an odd number of 16-byte chunks: ldmatrix without conflicts
  static constexpr int kBytes = kWarpRows * kPitch;
  static constexpr int kChunks = DP / 8;                    // 16-byte chunks of a row
  static constexpr int kRowsAtOnce = 32 / kChunks;          // rows one copy instruction of a warp covers
  static constexpr int kSmem = kWarps * kStages * 2 * kBytes;
};

// Where a warp's lane r (< 16) finds row r of a 16-row tile (line -1: the row does not
// count), asked for ahead of time, so that the latency is not waited for.
struct RowRef {
  int page, line;
};

template <class T, int DP, int NT, bool FULL>
struct Segment {
  using L = Tile<DP>;
  const AttnParams& p;
  int b, kvh, heads;  // heads of this part
  const char *k, *v;
  int len, lane, w;
  int d;
  uint32_t ring;  // this warp's shared memory

  __device__ __forceinline__ RowRef look_up(int row0) const {
    RowRef r{0, -1};
    const int row = row0 + lane;
    if (lane < kWarpRows && row < len) {
      r.page = p.c.page_of(b, row, &r.line);
      if (row < p.valid_rows && p.valid[b * p.valid_pitch + row] == 0) r.line = -1;
    }
    return r;
  }

  // Copies a tile's K and V, zeros in the place of rows that do not count; returns a
  // bit for each row that does.
  __device__ __forceinline__ uint32_t fetch(const RowRef& ref, int stage) const {
    long long off = -1;
    if (ref.line >= 0) {
      if (p.c.real(ref.page)) off = (long long)p.c.row_at(ref.page, kvh, ref.line);
      else report_status(p.c.status, PI05_DEV_BAD_INDEX);
    }
    const int chunk = lane % L::kChunks;
    const int have = FULL ? DP / 8 : d / 8, used = FULL ? DP / 8 : ((d + 15) / 16) * 2;
    const uint32_t dst = ring + stage * 2 * L::kBytes + chunk * 16;
#pragma unroll
    for (int i = 0; i < kWarpRows / L::kRowsAtOnce; ++i) {
      const int row = i * L::kRowsAtOnce + lane / L::kChunks;
      const long long o = __shfl_sync(~0u, off, row);
      if (FULL || chunk < used) {
        const bool read = o >= 0 && (FULL || chunk < have);
        const long long at = read ? o + chunk * 16 : 0;
        cp_async_16_or_zero(dst + row * L::kPitch, k + at, read);
        cp_async_16_or_zero(dst + L::kBytes + row * L::kPitch, v + at, read);
      }
    }
    return __ballot_sync(~0u, off >= 0);
  }
};

// One contiguous run [tile0, tile1) of the blocks of one (sequence, head, part).
template <class T, int DP, int NT, bool FULL>
__device__ void run_segment(const AttnParams& p, char* smem, int b, int row, int kvh, int part, int len, int tile0,
                            int tile1, int slot, bool whole) {
  using L = Tile<DP>;
  constexpr int H = 8 * NT;
  constexpr int KS = DP / 16;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int d = FULL ? DP : p.c.dim, steps = FULL ? KS : (d + 15) / 16;
  const int heads = min(H, p.group - part * H), head0 = kvh * p.group + part * H;
  Segment<T, DP, NT, FULL> s{p, b, kvh, heads, p.c.k, p.c.v, len, lane, w, d,
                             smem_u32(smem) + w * kStages * 2 * L::kBytes};
  // This warp's tiles: row0 = (tile0 * 4 + w + 4 j) * 16.
  const int n_tiles = tile1 - tile0;
  auto row0_of = [&](int j) { return ((tile0 + j) * kWarps + w) * kWarpRows; };

  uint32_t live[kStages];  // of the tiles in flight, the oldest first
  RowRef ref = s.look_up(n_tiles > 0 ? row0_of(0) : len);
#pragma unroll
  for (int j = 0; j < kStages - 1; ++j) {
    const RowRef now = ref;
    ref = s.look_up(j + 1 < n_tiles ? row0_of(j + 1) : len);
    live[j] = j < n_tiles ? s.fetch(now, j) : 0u;
    cp_async_commit();
  }

  // q^T fragments: lane holds head lane / 4, values 2 (lane % 4) + {0, 1, 8, 9} of each step.
  uint32_t qf[KS][NT][2];
  {
    const int n = lane >> 2, c = 2 * (lane & 3);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int h = nt * 8 + n;
        const T* q = static_cast<const T*>(p.q) + b * p.qt + (long long)(head0 + h) * p.qh;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int at = ks * 16 + c + 8 * i;
          qf[ks][nt][i] = h < heads && at < d ? *reinterpret_cast<const uint32_t*>(q + at) : 0u;
        }
      }
  }

  float o[KS][NT][4], m[NT][2], l[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[ks][nt][i] = 0.f;
    m[nt][0] = m[nt][1] = -INFINITY;
    l[nt][0] = l[nt][1] = 0.f;
  }

  const uint32_t k_lane = (lane & 15) * L::kPitch + (lane >> 4) * 16;
  const uint32_t v_lane = ((lane & 7) + ((lane >> 4) << 3)) * L::kPitch + ((lane >> 3) & 1) * 16;
  for (int j = 0; j < n_tiles; ++j) {
    const int row0 = row0_of(j);
    cp_async_wait<kStages - 2>();
    __syncwarp();
    {  // refill the slot read in the last turn
      const RowRef now = ref;
      const int next = j + kStages - 1;
      ref = s.look_up(next + 1 < n_tiles ? row0_of(next + 1) : len);
      live[kStages - 1] = next < n_tiles ? s.fetch(now, next % kStages) : 0u;
      cp_async_commit();
    }
    // Which of this lane's two rows count (row lane / 4 and that plus 8).
    const bool live0 = live[0] >> (lane >> 2) & 1, live1 = live[0] >> (lane >> 2) >> 8 & 1;
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) live[i] = live[i + 1];
    const uint32_t k_at = s.ring + (j % kStages) * 2 * L::kBytes + k_lane;
    const uint32_t v_at = s.ring + (j % kStages) * 2 * L::kBytes + L::kBytes + v_lane;
    float x[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) x[nt][0] = x[nt][1] = x[nt][2] = x[nt][3] = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      if (FULL || ks < steps) {
        uint32_t a[4];
        ldsm4(a, k_at + ks * 32);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma16816<T>(x[nt], a, qf[ks][nt]);
      }
    }
    const int r0 = row0 + (lane >> 2), r1 = r0 + 8;
    uint32_t pf[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float* xs = x[nt];
      xs[0] = live0 ? xs[0] * p.scale_log2 : -INFINITY;
      xs[1] = live0 ? xs[1] * p.scale_log2 : -INFINITY;
      xs[2] = live1 ? xs[2] * p.scale_log2 : -INFINITY;
      xs[3] = live1 ? xs[3] * p.scale_log2 : -INFINITY;
      if (p.track) {
        const int h = nt * 8 + 2 * (lane & 3);
        float* dst = p.scores + ((size_t)row * p.c.capacity) * H + h;
        if (r0 < len) *reinterpret_cast<float2*>(dst + (size_t)r0 * H) = make_float2(xs[0], xs[1]);
        if (r1 < len) *reinterpret_cast<float2*>(dst + (size_t)r1 * H) = make_float2(xs[2], xs[3]);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float top = fmaxf(xs[i], xs[i + 2]);
#pragma unroll
        for (int sft = 4; sft < 32; sft <<= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, sft));
        top = fmaxf(top, m[nt][i]);
        const float base = top == -INFINITY ? 0.f : top;
        const float keep = ex2_approx(m[nt][i] - base);
        m[nt][i] = top;
        xs[i] = ex2_approx(xs[i] - base);
        xs[i + 2] = ex2_approx(xs[i + 2] - base);
        l[nt][i] = l[nt][i] * keep + xs[i] + xs[i + 2];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          o[ks][nt][i] *= keep;
          o[ks][nt][i + 2] *= keep;
        }
      }
      pf[nt][0] = transpose8x8(pack2<T>(xs[0], xs[1]));
      pf[nt][1] = transpose8x8(pack2<T>(xs[2], xs[3]));
    }
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      if (FULL || ks < steps) {
        uint32_t a[4];
        ldsm4_trans(a, v_at + ks * 32);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma16816<T>(o[ks][nt], a, pf[nt]);
      }
    }
  }
  cp_async_wait<0>();
  __syncthreads();  // the rings are free: the warps' results meet there

  float* so = reinterpret_cast<float*>(smem);                      // [kWarps][H][DP]
  float2* sml = reinterpret_cast<float2*>(so + kWarps * H * DP);   // [kWarps][H]
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float sum = l[nt][i];
#pragma unroll
      for (int sft = 4; sft < 32; sft <<= 1) sum += __shfl_xor_sync(~0u, sum, sft);
      const int h = nt * 8 + 2 * (lane & 3) + i;
      if (lane < 4) sml[w * H + h] = make_float2(m[nt][i], sum);
      float* dst = so + (w * H + h) * DP + (lane >> 2);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        dst[ks * 16] = o[ks][nt][i];
        dst[ks * 16 + 8] = o[ks][nt][i + 2];
      }
    }
  __syncthreads();
  for (int i = threadIdx.x; i < heads * DP; i += kThreads) {
    const int h = i / DP, x = i - h * DP;
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < kWarps; ++j) top = fmaxf(top, sml[j * H + h].x);
    const float base = top == -INFINITY ? 0.f : top;
    float sum = 0.f, acc = 0.f;
#pragma unroll
    for (int j = 0; j < kWarps; ++j) {
      const float f = ex2_approx(sml[j * H + h].x - base);
      sum += sml[j * H + h].y * f;
      acc += so[(j * H + h) * DP + x] * f;
    }
    if (whole) {
      // A sum of 0 has no row that counts; NaN stays NaN.
      if (x < d)
        static_cast<T*>(p.out)[((size_t)b * p.q_heads + head0 + h) * d + x] =
            from_f32<T>(sum == 0.f ? 0.f : acc / sum);
      if (x == 0) {
        const float lse2 = sum == 0.f ? -INFINITY : top + log2f(sum);
        if (p.lse != nullptr) p.lse[(size_t)b * p.q_heads + head0 + h] = lse2 * kLn2;
        if (p.track) p.row_lse[(size_t)row * H + h] = lse2;
      }
    } else {
      if (x < d) p.part_o[((size_t)slot * H + h) * d + x] = acc;
      if (x == 0) p.part_ml[(size_t)slot * H + h] = make_float2(top, sum);
    }
  }
  __syncthreads();  // before the rings fill again
}

template <class T, int DP, int NT, bool FULL>
__global__ void __launch_bounds__(kThreads) paged_attention_kernel(const AttnParams p) {
  extern __shared__ __align__(16) char smem[];
  __shared__ long long sh_sum[kThreads / 32];
  __shared__ long long sh_base;
  __shared__ int sh_b;
  pdl_wait();
  pdl_launch_dependents();
  const int per_block = p.c.heads * p.parts, tid = threadIdx.x;
  // All blocks there are, then the sequence that this CTA's share begins in.
  long long mine = 0;
  for (int b = tid; b < p.c.batch; b += kThreads) {
    mine += (p.c.rows(b) + kBlockRows - 1) / kBlockRows;
    if (blockIdx.x == 0 && p.c.rows(b) != p.c.counts[b]) report_status(p.c.status, PI05_DEV_BAD_INDEX);
  }
  for (int sft = 16; sft > 0; sft >>= 1) mine += __shfl_xor_sync(~0u, mine, sft);
  if ((tid & 31) == 0) sh_sum[tid >> 5] = mine;
  __syncthreads();
  long long total = 0;
  for (int i = 0; i < kThreads / 32; ++i) total += sh_sum[i];
  total *= per_block;
  const long long n = min((long long)gridDim.x, total), cta = blockIdx.x;
  if (cta >= n) return;
  const long long lo = cta * total / n, hi = (cta + 1) * total / n;
  long long before = 0;
  for (int b0 = 0; b0 < p.c.batch; b0 += kThreads) {
    const int b = b0 + tid;
    const long long own = b < p.c.batch ? (long long)((p.c.rows(b) + kBlockRows - 1) / kBlockRows) * per_block : 0;
    long long incl = own;
    for (int sft = 1; sft < 32; sft <<= 1) {
      const long long u = __shfl_up_sync(~0u, incl, sft);
      if ((tid & 31) >= sft) incl += u;
    }
    __syncthreads();
    if ((tid & 31) == 31) sh_sum[tid >> 5] = incl;
    __syncthreads();
    for (int i = 0; i < (tid >> 5); ++i) incl += sh_sum[i];
    incl += before;
    for (int i = 0; i < kThreads / 32; ++i) before += sh_sum[i];
    if (incl - own <= lo && lo < incl) {
      sh_b = b;
      sh_base = incl - own;
    }
    if (before > lo) break;
  }
  __syncthreads();
  int b = sh_b;
  long long base = sh_base, at = lo;
  while (at < hi) {
    const int len = p.c.rows(b), blocks = (len + kBlockRows - 1) / kBlockRows;
    if (at >= base + (long long)blocks * per_block) {
      base += (long long)blocks * per_block;
      ++b;
      continue;
    }
    const int pair = (int)((at - base) / blocks);  // head, part
    const int tile0 = (int)((at - base) - (long long)pair * blocks);
    const int tile1 = (int)min((long long)blocks, tile0 + (hi - at));
    const int row = b * per_block + pair;
    const bool whole = tile0 == 0 && tile1 == blocks;
    const int slot = 2 * (int)cta + (at == lo ? 0 : 1);
    if (tile0 == 0 && tid == 0) {
      const long long end = base + (long long)pair * blocks + blocks;  // the CTA that has the row's last block
      p.row_info[row] = whole ? make_int2(-1, -1) : make_int2(slot, (int)((end * n - 1) / total));
    }
    run_segment<T, DP, NT, FULL>(p, smem, b, row, pair / p.parts, pair % p.parts, len, tile0, tile1, slot, whole);
    at += tile1 - tile0;
  }
}

// Joins the partials of a row (blockIdx.y == 0), and adds its probabilities to the
// cache's weights (blockIdx.y > 0).
constexpr int kFinishThreads = 256;
constexpr int kTrackRows = 1024;  // of the longest sequence there can be, for each CTA

// log2 of the row's sum over everything, from its partials.
template <int H>
__device__ __forceinline__ float joined(const AttnParams& p, int2 info, int h, float* top_out, float* sum_out) {
  float top = -INFINITY, sum = 0.f;
  for (int slot = info.x; slot <= 2 * info.y; slot = (slot | 1) + 1) {
    const float2 ml = p.part_ml[(size_t)slot * H + h];
    const float t = fmaxf(top, ml.x), base = t == -INFINITY ? 0.f : t;
    sum = sum * ex2_approx(top - base) + ml.y * ex2_approx(ml.x - base);
    top = t;
  }
  *top_out = top;
  *sum_out = sum;
  return sum == 0.f ? -INFINITY : top + log2f(sum);
}

template <class T, int H>
__global__ void __launch_bounds__(kFinishThreads) paged_finish_kernel(const AttnParams p) {
  __shared__ float sh_lse[H];
  pdl_wait();
  pdl_launch_dependents();
  const int row = blockIdx.x, per = p.c.heads * p.parts, b = row / per, pair = row - b * per;
  const int kvh = pair / p.parts, part = pair - kvh * p.parts;
  const int heads = min(H, p.group - part * H), head0 = kvh * p.group + part * H, d = p.c.dim;
  const int len = p.c.rows(b);
  if (blockIdx.y == 0) {
    if (len > 0 && p.row_info[row].x < 0) return;
    const int2 info = len > 0 ? p.row_info[row] : make_int2(1, 0);  // no partial at all
    for (int i = threadIdx.x; i < heads * d; i += kFinishThreads) {
      const int h = i / d, x = i - h * d;
      float top, sum, acc = 0.f;
      const float lse2 = joined<H>(p, info, h, &top, &sum);
      const float base = top == -INFINITY ? 0.f : top;
      for (int slot = info.x; slot <= 2 * info.y; slot = (slot | 1) + 1)
        acc += p.part_o[((size_t)slot * H + h) * d + x] * ex2_approx(p.part_ml[(size_t)slot * H + h].x - base);
      static_cast<T*>(p.out)[((size_t)b * p.q_heads + head0) * d + i] = from_f32<T>(sum == 0.f ? 0.f : acc / sum);
      if (x == 0 && p.lse != nullptr) p.lse[(size_t)b * p.q_heads + head0 + h] = lse2 * kLn2;
    }
    return;
  }
  // The first part's CTAs add up all parts, so that a weight has one writer.
  if (part != 0) return;
  float* weight = p.c.weight;
  const int first = (blockIdx.y - 1) * kFinishThreads, step = (gridDim.y - 1) * kFinishThreads;
  for (int r0 = first; r0 < len; r0 += step) {
    const int r = r0 + threadIdx.x;
    float add = 0.f;
    for (int q = 0; q < p.parts; ++q) {
      const int2 info = p.row_info[row + q];
      const int here = min(H, p.group - q * H);
      __syncthreads();
      if (threadIdx.x < here) {
        float top, sum;
        sh_lse[threadIdx.x] = info.x < 0 ? p.row_lse[(size_t)(row + q) * H + threadIdx.x]
                                         : joined<H>(p, info, threadIdx.x, &top, &sum);
      }
      __syncthreads();
      if (r < len) {
        const float* s = p.scores + ((size_t)(row + q) * p.c.capacity + r) * H;
        for (int h = 0; h < here; ++h) add += s[h] == -INFINITY ? 0.f : ex2_approx(s[h] - sh_lse[h]);
      }
    }
    if (r < len) {
      int line;
      const int page = p.c.page_of(b, r, &line);
      if (p.c.real(page)) weight[p.c.slot_at(page, kvh, line)] += add;
    }
  }
}

// ---- host ----------------------------------------------------------------------
struct Plan {
  int nt, parts, dp, ctas, rows;
  size_t part_o, part_ml, row_info, row_lse, scores, bytes;
};

Plan make_plan(const Pi05PagedCache* c, int q_heads, int track) {
  Plan s;
  const int group = q_heads / c->n_kv_heads;
  s.nt = group <= 8 ? 1 : 2;
  s.parts = (group + 8 * s.nt - 1) / (8 * s.nt);
  s.dp = c->head_dim <= 64 ? 64 : c->head_dim <= 128 ? 128 : 256;
  s.rows = c->batch * c->n_kv_heads * s.parts;
  const long long capacity = (long long)c->pages_per_seq * c->page_size;
  const long long blocks = (capacity + kBlockRows - 1) / kBlockRows * s.rows;
  const int per_sm = s.dp == 64 ? 4 : s.dp == 128 ? 2 : 1;
  s.ctas = (int)std::min<long long>(blocks, (long long)kSMs * per_sm);
  const size_t h = 8 * s.nt;
  size_t at = 0;
  auto take = [&](size_t n) {
    const size_t here = at;
    at = (at + n + 255) & ~size_t(255);
    return here;
  };
  s.part_o = take(2 * (size_t)s.ctas * h * c->head_dim * 4);
  s.part_ml = take(2 * (size_t)s.ctas * h * 8);
  s.row_info = take((size_t)s.rows * 8);
  s.row_lse = take((size_t)s.rows * h * 4);
  s.scores = take(track ? (size_t)s.rows * capacity * h * 4 : 0);
  s.bytes = at;
  return s;
}

template <class T, int DP, int NT, bool FULL>
int launch(const AttnParams& p, const Plan& s, cudaStream_t st) {
  constexpr int kJoin = kWarps * 8 * NT * (DP * 4 + 8);
  constexpr int kSmem = Tile<DP>::kSmem > kJoin ? Tile<DP>::kSmem : kJoin;
  static_assert(kSmem <= 227 * 1024, "shared memory");
  auto kernel = paged_attention_kernel<T, DP, NT, FULL>;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
  if (e != cudaSuccess) {
    set_last_error("paged_attention: %s", cudaGetErrorString(e));
    return PI05_ERR_LAUNCH;
  }
  int rc = launch_pdl(kernel, dim3(s.ctas), dim3(kThreads), kSmem, st, pdl_enabled(), p);
  if (rc) return rc;
  const int chunks = p.track ? std::min((p.c.capacity + kTrackRows - 1) / kTrackRows, 1024) : 0;
  return launch_pdl(paged_finish_kernel<T, 8 * NT>, dim3(s.rows, 1 + chunks), dim3(kFinishThreads), 0, st,
                    pdl_enabled(), p);
}

template <class T, int DP, bool FULL>
int launch_nt(const AttnParams& p, const Plan& s, cudaStream_t st) {
  return s.nt == 1 ? launch<T, DP, 1, FULL>(p, s, st) : launch<T, DP, 2, FULL>(p, s, st);
}

template <class T>
int launch_type(const AttnParams& p, const Plan& s, cudaStream_t st) {
  const int d = p.c.dim;
  if (s.dp == 64) return d == 64 ? launch_nt<T, 64, true>(p, s, st) : launch_nt<T, 64, false>(p, s, st);
  if (s.dp == 128) return d == 128 ? launch_nt<T, 128, true>(p, s, st) : launch_nt<T, 128, false>(p, s, st);
  return d == 256 ? launch_nt<T, 256, true>(p, s, st) : launch_nt<T, 256, false>(p, s, st);
}

bool plain_shape(const Pi05PagedCache* c, int q_heads) {
  return c != nullptr && c->batch > 0 && c->n_kv_heads > 0 && c->page_size > 0 && c->pages_per_seq > 0 &&
         c->head_dim > 0 && c->head_dim <= 256 && q_heads > 0 && q_heads % c->n_kv_heads == 0;
}

}  // namespace
}  // namespace pi05

using namespace pi05;

extern "C" {

size_t pi05_paged_attention_scratch_bytes(const Pi05PagedCache* cache, int n_q_heads, int track) {
  return plain_shape(cache, n_q_heads) ? make_plan(cache, n_q_heads, track).bytes : 0;
}

int pi05_paged_attention(const Pi05PagedCache* cache, const Pi05PagedAttention* a, void* stream) {
  AttnParams p;
  int rc = paged_check(cache, "paged_attention", &p.c);
  if (rc) return rc;
  if (a == nullptr || a->q == nullptr || a->out == nullptr) {
    set_last_error("paged_attention: null pointer");
    return PI05_ERR_INVALID_ARG;
  }
  if (!plain_shape(cache, a->n_q_heads) || (long long)cache->batch * a->n_q_heads >= (1 << 24)) {
    set_last_error("paged_attention: %d query heads do not share %d key-value heads", a->n_q_heads,
                   cache->n_kv_heads);
    return PI05_ERR_SHAPE;
  }
  if (a->track && p.c.weight == nullptr) {
    set_last_error("paged_attention: the cache keeps no weights");
    return PI05_ERR_INVALID_ARG;
  }
  if ((reinterpret_cast<uintptr_t>(a->q) & 3) || a->q_token_stride % 2 || a->q_head_stride % 2) {
    set_last_error("paged_attention: q rows must start on 4-byte boundaries");
    return PI05_ERR_ALIGN;
  }
  const Plan s = make_plan(cache, a->n_q_heads, a->track);
  if (a->scratch == nullptr || a->scratch_bytes < s.bytes) {
    set_last_error("paged_attention: scratch missing or too small (%zu bytes needed)", s.bytes);
    return PI05_ERR_WORKSPACE;
  }
  if (!aligned16(a->scratch)) {
    set_last_error("paged_attention: scratch not 16-byte aligned");
    return PI05_ERR_ALIGN;
  }
  char* sc = static_cast<char*>(a->scratch);
  p.q = a->q;
  p.out = a->out;
  p.lse = a->lse;
  p.valid = a->key_valid;
  p.qt = a->q_token_stride;
  p.qh = a->q_head_stride;
  p.valid_pitch = a->valid_pitch;
  p.valid_rows = a->key_valid != nullptr ? a->valid_rows : 0;
  p.q_heads = a->n_q_heads;
  p.group = a->n_q_heads / cache->n_kv_heads;
  p.parts = s.parts;
  p.scale_log2 = a->scale * 1.44269504088896340736f;
  p.track = a->track;
  p.n_ctas = s.ctas;
  p.part_o = reinterpret_cast<float*>(sc + s.part_o);
  p.part_ml = reinterpret_cast<float2*>(sc + s.part_ml);
  p.row_info = reinterpret_cast<int2*>(sc + s.row_info);
  p.row_lse = reinterpret_cast<float*>(sc + s.row_lse);
  p.scores = reinterpret_cast<float*>(sc + s.scores);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return cache->dtype == PI05_BF16 ? launch_type<__nv_bfloat16>(p, s, st) : launch_type<__half>(p, s, st);
}

}  // extern "C"
