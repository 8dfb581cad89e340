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
// that the join kernel adds up in order.  Few short sequences take a cluster of CTAs for
// each pair instead, and no other kernel (SHORT, and make_plan).
//
// A warp takes 16 rows at a time, brought by TMA into a ring of its own (no block barrier
// in the loop), and its copies run ahead of its products across the borders of pairs.  The
// products run on the tensor cores with the rows as M:  S^T = K q^T (16 rows x 8 heads),
// then O^T += V^T P^T, where the probabilities pass from one fragment layout to the other
// by a matrix transpose in registers; with the heads as N = 8, half as many products and
// accumulators as with 16 padded query rows.  The probabilities enter the second product as
// a sum of two numbers of the cache's 16-bit type (see halves()); m, l and o stay fp32.
//
// Measured: 2 x 131072 rows, 32 / 8 heads of 128: 167 us with the join's 5 = 6.6 TB/s (with
// one 16-bit number for a probability 166).  An earlier form with 16-byte cp.async copies
// through registers' addresses took 190 us where TMA took 157 (430 instructions a tile, and 8
// warps an SM are too few to hide them); with a bulk copy for each row, issued one by one, 174
// with 12 warps, 206 with 8.  More than 8 query heads to a key-value head are the weak side:
// with 256 columns one CTA of four warps has an SM, and its accumulators leave the registers (430
// bytes): 54 x 16 pairs of 104 rows, 16 query heads each, 143 us for 92 MB; above 16 each part
// reads the rows again (33 heads over 131072 rows of 128: 54 us for 67 MB).
#include <algorithm>
#include <type_traits>

#include "paged.cuh"

namespace pi05 {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kWarpRows = 16;
constexpr int kBlockRows = kWarps * kWarpRows;
constexpr float kLn2 = 0.69314718055994530942f;
// The running maximum is -inf while no row has counted and at least this from then on, so that
// rows whose scores are all -inf (0 / 0, NaN) are told from no rows (0) at the end.  A row that
// counts leaves this score for -inf, and a masked one -inf, to the tracking.
constexpr float kLowest = -3.402823466e38f;

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
  int track, box_rows;
  int ctas;  // of a pair (SHORT)
  // scratch
  float* part_o;    // [2 n_ctas][8 NT][dim]
  float2* part_ml;  // [2 n_ctas][8 NT]
  int2* row_info;   // [rows]: first partial slot (-1: done), last CTA
  float* row_lse;   // [rows][8 NT] log2 units, of the rows done in one piece
  // track: scores in log2 units, [score_units][kBlockRows][score_pitch], where a row's begin with
  // its unit (see Walk)
  float* scores;
  int* row_unit;  // [rows]: or -1, when there are more units than scores
  int score_units;
  int score_pitch;  // heads of a part, up to a power of two from 2 on
};

template <class T>
__device__ __forceinline__ void mma16816(float* c, const uint32_t* a, const uint32_t* b);
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float* c, const uint32_t* a, const uint32_t* b) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
template <>
__device__ __forceinline__ void mma16816<__half>(float* c, const uint32_t* a, const uint32_t* b) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}

// A probability x <= 1 as hi + lo for the matrix unit, which takes 16-bit numbers: one alone
// would be off by as much as the output's own rounding (2^-9 of it in bf16), and in fp16 lose
// what lies below 2^-25.  hi has x's leading bits (8 in bf16, 11 in fp16) and lo rounds the rest,
// to 2^-16 of x in bf16 and 2^-21 in fp16, where both hold 2^15 x, so that nothing above 2^-39
// of the largest is lost either.  hi lies below x, so that lo is not 0: hi * inf + 0 * inf would be
// NaN where x * inf is infinite.
template <class T>
struct Prob;
template <>
struct Prob<__nv_bfloat16> {
  static constexpr float kOne = 1.f;
  static constexpr uint32_t kLeading = 0xffff0000u;
};
template <>
struct Prob<__half> {
  static constexpr float kOne = 0x1p15f;
  static constexpr uint32_t kLeading = 0xffffe000u;
};
template <class T>
__device__ __forceinline__ float2 halves(float x) {
  const float v = x * Prob<T>::kOne, hi = __uint_as_float((max(__float_as_uint(v), 1u) - 1) & Prob<T>::kLeading);
  return make_float2(hi, v - hi);
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
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* tm, uint32_t bar, int x, int y, int z,
                                            int w, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, "
      "{%2, %3, %4, %5}], [%6], %7;" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(tm)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar), "l"(policy)
      : "memory");
}

// A tile of 16 rows: boxes of 64 columns, 16 rows of 128 bytes each, whose 16-byte chunk
// c of row r lies at chunk c ^ (r & 7) (the 128-byte swizzle): ldmatrix without conflicts.
// KS: steps of 16 columns that the products take; what lies beyond a head is zeros.
// SHORT (see the kernel) leaves shared memory to the scores.
template <int KS, int NT, bool SHORT>
struct Tile {
  static constexpr int kBoxes = (KS + 3) / 4;
  static constexpr int kBox = kWarpRows * 128;
  static constexpr int kBytes = kBoxes * kBox;
  static constexpr int kStages = kBoxes == 4 && NT == 1 && !SHORT ? 3 : 2;
  static constexpr int kRing = kWarps * kStages * 2 * kBytes;
  static constexpr int kSlot = (KS * NT * 4 + NT * 4) * 32 * 4;  // a warp's o, m and l, at a segment's end
  static constexpr int kSmem = 1024 + kRing + 2 * kSlot;
  // CTAs on an SM: as many as shared memory and the accumulators' registers leave room for.
  static constexpr int kPerSM = kBoxes == 1 ? (NT == 1 ? 4 : 3) : kBoxes == 2 ? (NT == 1 ? 3 : 2) : kBoxes == 3 && NT == 1 ? 2 : 1;
  static_assert(kPerSM * (kSmem + 1024) <= 228 * 1024, "shared memory of an SM");
};

// One contiguous run of blocks of one (sequence, key-value head, part of its query heads).
struct Segment {
  int b, row, kvh, part, len, tile0, n;
  bool whole;
};

// a / b; 32-bit division, a tenth of the 64-bit one's instructions, where it will do.
__device__ __forceinline__ long long divide(long long a, long long b) {
  return ((a | b) >> 32) == 0 ? (long long)((uint32_t)a / (uint32_t)b) : a / b;
}

// Starting and joining a pair costs a CTA about as much as kBorder blocks, so each pair
// counts for so many more than it has: shares of equal numbers of blocks left the CTAs with
// the shortest sequences, a border at every block, behind: 38 us where the others took 24 (24
// sequences of 1 to 1500 rows, 16 heads of 80).
constexpr int kBorder = 2;

// Walks through a CTA's share, segment by segment, in units of a block; the first kBorder
// units of a pair stand for its border.
struct Walk {
  int b;
  long long base, at, end;  // first unit of sequence b; the next unit; the share's end
  long long pair_end;       // of the pair of the last segment

  __device__ __forceinline__ bool next(const AttnParams& p, Segment& s) {
    const int per = p.c.heads * p.parts;
    while (at < end) {
      s.len = p.c.rows(b);
      const int blocks = (s.len + kBlockRows - 1) / kBlockRows, units = blocks > 0 ? blocks + kBorder : 0;
      if (at >= base + (long long)units * per) {
        base += (long long)units * per;
        ++b;
        continue;
      }
      const int pair = (int)divide(at - base, units);
      const long long first_block = base + (long long)pair * units + kBorder;
      pair_end = first_block + blocks;
      s.tile0 = (int)max(at - first_block, 0ll);
      at = min(end, pair_end);
      s.n = (int)(at - first_block) - s.tile0;
      if (s.n <= 0) continue;  // nothing but the border
      s.b = b;
      s.row = b * per + pair;
      s.kvh = pair / p.parts;
      s.part = pair - s.kvh * p.parts;
      s.whole = s.n == blocks;
      return true;
    }
    return false;
  }
};

// A row of the cache as lane r < 16 of a warp knows row r of a tile; asked for one tile
// ahead of its copy, so that the table's latency is not waited for.
struct Ref {
  int page, line, kvh;
  bool tile, counts;  // there is a tile; this row counts
};

__device__ __forceinline__ Ref look_up(const AttnParams& p, const Segment& s, int row0, int lane) {
  Ref r{0, 0, s.kvh, true, false};
  const int row = row0 + (lane & 15);
  if (row < s.len) {
    r.page = p.c.page_of(s.b, row, &r.line);
    r.counts = row >= p.valid_rows || p.valid[s.b * p.valid_pitch + row] != 0;
  }
  return r;
}

// Starts the copies of a tile's K and V by TMA, `p.box_rows` rows of 64 columns at a time
// (the largest power of two that divides the page size, so that a box lies in one page);
// a lane for each group of rows.  Returns a bit for each row that counts.
template <int KS, int NT, bool SHORT>
__device__ __forceinline__ uint32_t fetch(const AttnParams& p, const CUtensorMap* tm_k, const CUtensorMap* tm_v,
                                          const Ref& ref, uint64_t* bar, uint32_t dst, int lane,
                                          uint64_t policy) {
  using L = Tile<KS, NT, SHORT>;
  const bool real = p.c.real(ref.page);
  if (ref.counts && !real) report_status(p.c.status, PI05_DEV_BAD_INDEX);
  const uint32_t mask = __ballot_sync(~0u, ref.counts && real) & 0xffff;
  constexpr uint32_t kRowBytes = 128 * L::kBoxes * 2;  // of a box row, over all boxes of K and V
  bool mine;
  if (p.box_rows == kWarpRows) {
    mine = lane == 0 && mask != 0;
    if (lane == 0) mbar_arrive_expect_tx(bar, mask != 0 ? kWarpRows * kRowBytes : 0);
  } else {
    mine = lane < kWarpRows && (lane & (p.box_rows - 1)) == 0 && (mask >> lane & ((1u << p.box_rows) - 1)) != 0;
    const int groups = __popc(__ballot_sync(~0u, mine));
    if (lane == 0) mbar_arrive_expect_tx(bar, groups * p.box_rows * kRowBytes);
    __syncwarp();
  }
  if (mine) {
    const uint32_t to = dst + lane * 128, at = smem_u32(bar);
#pragma unroll
    for (int i = 0; i < L::kBoxes; ++i) {
      tma_load_4d(to + i * L::kBox, tm_k, at, i * 64, ref.line, ref.kvh, ref.page, policy);
      tma_load_4d(to + L::kBytes + i * L::kBox, tm_v, at, i * 64, ref.line, ref.kvh, ref.page, policy);
    }
  }
  return mask;
}

// What a row adds to its weight, by its score and the logarithm of its head's sum (log2 units);
// a sum of 0 gives NaN to the rows that count.
__device__ __forceinline__ float track_lse(float lse2) { return lse2 == -INFINITY ? NAN : lse2; }
__device__ __forceinline__ float probability(float score, float lse2) {
  return score == -INFINITY ? 0.f : ex2_approx(score - lse2);
}

__device__ __forceinline__ float ld_peer(const float* x, int rank, int ctas) {
  if (ctas == 1) return *x;
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(mapa_shared(smem_u32(x), rank)) : "memory");
  return v;
}

// SHORT: a cluster of p.ctas CTAs for each pair instead of equal shares, which joins its
// parts through distributed shared memory and keeps its scores there: no other kernel.
template <class T, int KS, int NT, bool SHORT>
__global__ void __launch_bounds__(kThreads, Tile<KS, NT, SHORT>::kPerSM)
    paged_attention_kernel(const __grid_constant__ AttnParams p, const __grid_constant__ CUtensorMap tm_k,
                           const __grid_constant__ CUtensorMap tm_v) {
  using L = Tile<KS, NT, SHORT>;
  constexpr int H = 8 * NT, S = L::kStages;
  extern __shared__ char smem_raw[];
  __shared__ long long sh_sum[kWarps];
  __shared__ long long sh_base;
  __shared__ int sh_b;
  __shared__ uint64_t all_bars[kWarps * S];
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  if (tid == 0) {
    prefetch_tmap(&tm_k);
    prefetch_tmap(&tm_v);
  }
  if (tid < kWarps * S) mbar_init(&all_bars[tid], 1);
  fence_mbar_init();
  pdl_wait();
  pdl_launch_dependents();

  const int d = p.c.dim;
  long long total = 0, n = 0;  // all units, and the CTAs that share them
  const long long cta = blockIdx.x;
  int rank = 0;
  Segment fs;             // of the copies, which run ahead of the products
  Walk ahead{0, 0, 0, 0, 0};
  bool more;
  if constexpr (SHORT) {
    const int pair = blockIdx.x / p.ctas;  // the grid is a line of clusters
    rank = blockIdx.x - pair * p.ctas;
    const int b = pair / p.c.heads, len = p.c.rows(b), blocks = (len + kBlockRows - 1) / kBlockRows;
    if (rank == 0 && tid == 0 && len != p.c.counts[b]) report_status(p.c.status, PI05_DEV_BAD_INDEX);
    fs = Segment{b, pair, pair - b * p.c.heads, 0, len, rank * blocks / p.ctas, 0, false};
    fs.n = (rank + 1) * blocks / p.ctas - fs.tile0;
    if (len == 0) {  // the whole cluster alike: nothing to attend to
      const int head = fs.kvh * p.group;
      if (rank == 0)
        for (int i = tid; i < p.group * d; i += kThreads)
          static_cast<T*>(p.out)[((size_t)b * p.q_heads + head) * d + i] = from_f32<T>(0.f);
      if (rank == 0 && p.lse != nullptr)
        for (int i = tid; i < p.group; i += kThreads) p.lse[(size_t)b * p.q_heads + head + i] = -INFINITY;
      return;
    }
    more = fs.n > 0;
    __syncthreads();  // the barriers are there
  } else {
    // All units there are, then the sequence that this CTA's share begins in: one scan for
    // up to kThreads sequences, else a sum and a scan of one part after the other.
    const int per_block = p.c.heads * p.parts;
    const bool few = p.c.batch <= kThreads;
    auto scan = [&](long long own) {  // of the CTA's threads; inclusive
      for (int sft = 1; sft < 32; sft <<= 1) {
        const long long u = __shfl_up_sync(~0u, own, sft);
        if (lane >= sft) own += u;
      }
      __syncthreads();
      if (lane == 31) sh_sum[w] = own;
      __syncthreads();
      for (int i = 0; i < w; ++i) own += sh_sum[i];
      return own;
    };
    auto units_of = [&](int b) {
      const int len = p.c.rows(b);
      if (blockIdx.x == 0 && len != p.c.counts[b]) report_status(p.c.status, PI05_DEV_BAD_INDEX);
      return len > 0 ? (long long)((len + kBlockRows - 1) / kBlockRows + kBorder) * per_block : 0ll;
    };
    long long own = 0;
    for (int b = tid; b < p.c.batch; b += kThreads) own += units_of(b);
    long long incl = scan(own);
    for (int i = 0; i < kWarps; ++i) total += sh_sum[i];
    n = min((long long)gridDim.x, total);
    // More rows than the pool has: pages that stand twice in the table, or none.
    if (p.track && total > p.score_units && cta == 0 && tid == 0) report_status(p.c.status, PI05_DEV_BAD_INDEX);
    if (cta >= n) return;
    const long long lo = divide(cta * total, n), hi = divide((cta + 1) * total, n);
    long long before = 0;
    for (int b0 = 0; b0 < p.c.batch; b0 += kThreads) {
      const int b = b0 + tid;
      if (!few) {
        own = b < p.c.batch ? units_of(b) : 0;
        incl = before + scan(own);
        for (int i = 0; i < kWarps; ++i) before += sh_sum[i];
      }
      if (incl - own <= lo && lo < incl) {
        sh_b = b;
        sh_base = incl - own;
      }
      if (before > lo) break;
    }
    __syncthreads();

    ahead = Walk{sh_b, sh_base, lo, hi, 0};
    more = ahead.next(p, fs);
  }

  const uint32_t base_addr = (smem_u32(smem_raw) + 1023) & ~1023u;  // swizzled boxes start at multiples of 1024
  const uint32_t ring = base_addr + w * S * 2 * L::kBytes;
  float* slots = reinterpret_cast<float*>(smem_raw + (base_addr - smem_u32(smem_raw)) + L::kRing);
  uint64_t* bars = all_bars + w * S;
  float* my_scores = slots + 2 * (L::kSlot / 4);  // SHORT: [rows of this CTA][score_pitch]

  // K and V pass through L2 once, unless other parts of the query heads read them too; what
  // is written for the kernels behind this one (scores: 34 of 1110 MB) should stay there.
  const uint64_t policy = p.parts == 1 ? l2_policy_evict_first() : l2_policy_evict_normal();

  // The warp's copies run ahead of its products, across the segments' borders.
  Segment next = fs;
  Walk walk = ahead;
  bool have = SHORT || more;  // a segment to work on, `next`: now, since `more` runs ahead
  int fj = 0;
  auto next_ref = [&]() {
    if (more && fj == fs.n) {
      more = !SHORT && ahead.next(p, fs);
      fj = 0;
    }
    if (!more) return Ref{0, 0, 0, false, false};
    return look_up(p, fs, ((fs.tile0 + fj++) * kWarps + w) * kWarpRows, lane);
  };
  int flying = 0;    // tiles asked for and not read yet
  uint32_t live[S];  // rows that count of these, the oldest first
  Ref ref = next_ref();
#pragma unroll
  for (int j = 0; j < S - 1; ++j) {
    const Ref now = ref;
    ref = next_ref();
    live[j] = now.tile ? fetch<KS, NT, SHORT>(p, &tm_k, &tm_v, now, bars + j, ring + j * 2 * L::kBytes, lane, policy) : 0u;
    flying += now.tile;
  }
  int stage = 0;
  uint32_t phase = 0;
  bool broken = false;  // a wait ran out: this warp reads no more

  // Chunk 2 ks + c of row r lies at 128 r + 16 ((2 ks + c) ^ (r & 7)) of its box.
  const uint32_t k_lane = (lane & 15) * 128 + (((lane >> 4) ^ (lane & 7)) << 4);
  const uint32_t v_lane = ((lane & 7) + ((lane >> 4) << 3)) * 128 + ((((lane >> 3) & 1) ^ (lane & 7)) << 4) + L::kBytes;
  auto step_at = [](uint32_t at, int ks) { return (at ^ ((ks & 3) << 5)) + (ks >> 2) * L::kBox; };

  // q^T fragments: lane holds head lane / 4, values 2 (lane % 4) + {0, 1, 8, 9} of each step.
  uint32_t qf[KS][NT][2];
  auto load_q = [&](const Segment& s) {
    const int heads = min(H, p.group - s.part * H), head0 = s.kvh * p.group + s.part * H;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int h = nt * 8 + (lane >> 2);
        const T* q = static_cast<const T*>(p.q) + s.b * p.qt + (long long)(head0 + h) * p.qh;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int at = ks * 16 + 2 * (lane & 3) + 8 * i;
          qf[ks][nt][i] = h < heads && at < d ? *reinterpret_cast<const uint32_t*>(q + at) : 0u;
        }
      }
  };
  if (have) load_q(next);
  for (int slot = 2 * (int)cta; have; slot |= 1) {
    const Segment s = next;
    const int heads = min(H, p.group - s.part * H), head0 = s.kvh * p.group + s.part * H;
    int unit = 0;  // the pair's first, where its scores go; all into the first, unread, if they have no room
    if constexpr (!SHORT) {
      const bool room = total <= p.score_units;
      if (p.track && room) unit = (int)(walk.pair_end - (s.len + kBlockRows - 1) / kBlockRows - kBorder);
      if (s.tile0 == 0 && tid == 0) {
        // the CTA that has the pair's last block
        p.row_info[s.row] = s.whole ? make_int2(-1, -1) : make_int2(slot, (int)divide(walk.pair_end * n - 1, total));
        if (p.track) p.row_unit[s.row] = room ? unit : -1;
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

    for (int j = 0; j < s.n && !broken; ++j) {
      if (__any_sync(~0u, !mbar_wait(bars + stage, phase))) {
        report_status(p.c.status, PI05_DEV_TIMEOUT_PRODUCER);
        broken = true;
        break;
      }
      {  // refill the stage read in the last turn
        const Ref now = ref;
        ref = next_ref();
        const int to = stage == 0 ? S - 1 : stage - 1;
        live[S - 1] = now.tile ? fetch<KS, NT, SHORT>(p, &tm_k, &tm_v, now, bars + to, ring + to * 2 * L::kBytes, lane, policy) : 0u;
        flying += now.tile ? 0 : -1;
      }
      const uint32_t tile = ring + stage * 2 * L::kBytes, rows = live[0];
      if (++stage == S) {
        stage = 0;
        phase ^= 1;
      }
#pragma unroll
      for (int i = 0; i < S - 1; ++i) live[i] = live[i + 1];
      // Which of this lane's two rows count (row lane / 4 and that plus 8).
      const bool live0 = rows >> (lane >> 2) & 1, live1 = rows >> (lane >> 2) >> 8 & 1;

      // Fragments by the batch, ahead of the products that take them; two chains of sums.
      // What a row that does not count holds may be anything, and 0 times that has to be 0:
      // its values are cut out of the V fragments (two rows to a register).
      const uint32_t r2 = rows >> (2 * (lane & 3));
      const uint32_t cut0 = (r2 & 1 ? 0xffffu : 0u) | (r2 & 2 ? 0xffff0000u : 0u);
      const uint32_t cut1 = (r2 & 0x100 ? 0xffffu : 0u) | (r2 & 0x200 ? 0xffff0000u : 0u);
      auto load_v = [&](uint32_t* a, int ks) {
        ldsm4_trans(a, step_at(tile + v_lane, ks));
        if (rows != 0xffff) {
          a[0] &= cut0;
          a[1] &= cut0;
          a[2] &= cut1;
          a[3] &= cut1;
        }
      };
      constexpr int B = KS < 8 ? KS : NT == 1 ? 8 : 4;
      float x[NT][4], x2[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) x[nt][i] = x2[nt][i] = 0.f;
#pragma unroll
      for (int k0 = 0; k0 < KS; k0 += B) {
        uint32_t a[B][4];
#pragma unroll
        for (int ks = 0; ks < B; ++ks)
          if (k0 + ks < KS) ldsm4(a[ks], step_at(tile + k_lane, k0 + ks));
#pragma unroll
        for (int ks = 0; ks < B; ++ks)
          if (k0 + ks < KS) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma16816<T>(ks & 1 ? x2[nt] : x[nt], a[ks], qf[k0 + ks][nt]);
          }
      }
      uint32_t va[B][4];
#pragma unroll
      for (int ks = 0; ks < B; ++ks)
        load_v(va[ks], ks);
      uint32_t pf[NT][2], pl[NT][2];  // the probabilities' hi and lo
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float* xs = x[nt];
#pragma unroll
        for (int i = 0; i < 4; ++i) xs[i] = (i < 2 ? live0 : live1) ? (xs[i] + x2[nt][i]) * p.scale_log2 : -INFINITY;
        if (p.track) {
          const int h = nt * 8 + 2 * (lane & 3), r0 = ((s.tile0 + j) * kWarps + w) * kWarpRows + (lane >> 2);
          float* dst = SHORT ? my_scores + (r0 - s.tile0 * kBlockRows) * p.score_pitch + h
                             : p.scores + ((size_t)unit * kBlockRows + r0) * p.score_pitch + h;
          auto score = [](bool counts, float x) { return counts && x == -INFINITY ? kLowest : x; };
          if (r0 < s.len && h < heads)
            *reinterpret_cast<float2*>(dst) = make_float2(score(live0, xs[0]), score(live0, xs[1]));
          if (r0 + 8 < s.len && h < heads)
            *reinterpret_cast<float2*>(dst + 8 * (size_t)p.score_pitch) =
                make_float2(score(live1, xs[2]), score(live1, xs[3]));
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float top = fmaxf(xs[i], xs[i + 2]);
#pragma unroll
          for (int sft = 4; sft < 32; sft <<= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, sft));
          top = fmaxf(top, fmaxf(m[nt][i], rows != 0 ? kLowest : -INFINITY));
          const float base = top == -INFINITY ? 0.f : top;
          const float keep = ex2_approx(m[nt][i] - base);
          m[nt][i] = top;
          xs[i] = ex2_approx(xs[i] - base);
          xs[i + 2] = ex2_approx(xs[i + 2] - base);
          l[nt][i] = l[nt][i] * keep + xs[i] + xs[i + 2];
          if (__any_sync(~0u, keep != 1.f)) {
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
              o[ks][nt][i] *= keep;
              o[ks][nt][i + 2] *= keep;
            }
          }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float2 a = halves<T>(xs[2 * i]), b = halves<T>(xs[2 * i + 1]);
          pf[nt][i] = transpose8x8(pack2<T>(a.x, b.x));
          pl[nt][i] = transpose8x8(pack2<T>(a.y, b.y));
        }
      }
#pragma unroll
      for (int k0 = 0; k0 < KS; k0 += B) {
        if (k0 > 0) {
#pragma unroll
          for (int ks = 0; ks < B; ++ks)
            if (k0 + ks < KS) load_v(va[ks], k0 + ks);
        }
#pragma unroll
        for (int ks = 0; ks < B; ++ks)
          if (k0 + ks < KS) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              mma16816<T>(o[k0 + ks][nt], va[ks], pl[nt]);
              mma16816<T>(o[k0 + ks][nt], va[ks], pf[nt]);
            }
          }
      }
    }

    have = !SHORT && walk.next(p, next);
    if (have) load_q(next);  // on its way while this segment is joined

    // The four warps' results, joined two by two in a fixed order: warps 2 and 3 hand theirs
    // to 0 and 1, then 1 to 0, fragment by fragment.
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int sft = 4; sft < 32; sft <<= 1) l[nt][i] += __shfl_xor_sync(~0u, l[nt][i], sft);
    auto give = [&](int i_slot) {
      float* to = slots + i_slot * (L::kSlot / 4) + lane;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          to[(nt * 4 + i) * 32] = m[nt][i];
          to[(nt * 4 + 2 + i) * 32] = l[nt][i];
        }
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int i = 0; i < 4; ++i) to[(NT * 4 + (ks * NT + nt) * 4 + i) * 32] = o[ks][nt][i];
      }
    };
    auto take = [&](int i_slot) {
      const float* from = slots + i_slot * (L::kSlot / 4) + lane;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float m2 = from[(nt * 4 + i) * 32], top = fmaxf(m[nt][i], m2), base = top == -INFINITY ? 0.f : top;
          const float f = ex2_approx(m[nt][i] - base), f2 = ex2_approx(m2 - base);
          m[nt][i] = top;
          l[nt][i] = l[nt][i] * f + from[(nt * 4 + 2 + i) * 32] * f2;
#pragma unroll
          for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int k = i; k < 4; k += 2)
              o[ks][nt][k] = o[ks][nt][k] * f + from[(NT * 4 + (ks * NT + nt) * 4 + k) * 32] * f2;
        }
    };
    __syncthreads();  // warp 0 is done with the last segment's
    if (w >= 2) give(w - 2);
    __syncthreads();
    if (w < 2) take(w);
    if (w == 1) give(1);
    __syncthreads();
    if (SHORT) {
      if (w == 0) {
        take(1);
        give(0);
      }
      break;
    }
    if (w == 0) {
      take(1);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int h = nt * 8 + 2 * (lane & 3) + i;
          if (h >= heads) continue;
          const float sum = l[nt][i];
          const bool none = m[nt][i] == -INFINITY;
          const float lse2 = m[nt][i] + log2f(sum), scale = 1.f / (sum * Prob<T>::kOne);
          T* out = static_cast<T*>(p.out) + ((size_t)s.b * p.q_heads + head0 + h) * d;
          float* part = p.part_o + ((size_t)slot * H + h) * d;
#pragma unroll
          for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const int x = ks * 16 + k * 8 + (lane >> 2);
              if (x >= d) continue;
              const float v = o[ks][nt][i + 2 * k];
              if (s.whole) out[x] = from_f32<T>(none ? 0.f : v * scale);
              else part[x] = v * (1.f / Prob<T>::kOne);
            }
          if (lane < 4) {
            if (!s.whole) {
              p.part_ml[(size_t)slot * H + h] = make_float2(m[nt][i], sum);
            } else {
              if (p.lse != nullptr) p.lse[(size_t)s.b * p.q_heads + head0 + h] = lse2 * kLn2;
              if (p.track) p.row_lse[(size_t)s.row * H + h] = track_lse(lse2);
            }
          }
        }
    }
  }

  if (broken) {  // no copy may land in the shared memory of a CTA that has ended
    for (; flying > 0; --flying) {
      mbar_wait(bars + stage, phase);
      if (++stage == S) {
        stage = 0;
        phase ^= 1;
      }
    }
  }
  if constexpr (SHORT) {
    __shared__ float sh_lse[H];
    const int ctas = p.ctas, heads = p.group, head0 = fs.kvh * p.group;
    auto sync_all = [&]() {
      if (ctas > 1) cluster_sync_all();
      else __syncthreads();
    };
    sync_all();
    // Value e of a slot: fragment e / 32 of lane e % 32, as give() lays them out.  The
    // cluster's CTAs take every ctas-th run of values and add the parts up in rank order.
    auto total_of = [&](int nt, int i, int of_lane, float* scale) {  // scale[r]: what rank r's part counts
      const float* ml = slots + (nt * 4 + i) * 32 + of_lane;
      float m[8], l[8], top = -INFINITY, sum = 0.f;
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        m[r] = r < ctas ? ld_peer(ml, r, ctas) : -INFINITY;
        l[r] = r < ctas ? ld_peer(ml + 64, r, ctas) : 0.f;
      }
#pragma unroll
      for (int r = 0; r < 8; ++r) top = fmaxf(top, m[r]);
      const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        scale[r] = ex2_approx(m[r] - base);
        sum += l[r] * scale[r];
      }
      const float inv = top == -INFINITY ? 0.f : 1.f / (sum * Prob<T>::kOne);
#pragma unroll
      for (int r = 0; r < 8; ++r) scale[r] *= inv;
      return top + log2f(sum);
    };
    float scale[8];
    for (int e = rank * kThreads + tid; e < KS * NT * 4 * 32; e += ctas * kThreads) {
      const int at = e >> 5, l = e & 31, i = at & 3, nt = (at >> 2) % NT, ks = (at >> 2) / NT;
      const int h = nt * 8 + 2 * (l & 3) + (i & 1), x = ks * 16 + (i >> 1) * 8 + (l >> 2);
      if (h >= heads || x >= d) continue;
      const float lse2 = total_of(nt, i & 1, l, scale);
      const float* o = slots + NT * 4 * 32 + e;
      float part[8], v = 0.f;
#pragma unroll
      for (int r = 0; r < 8; ++r) part[r] = r < ctas ? ld_peer(o, r, ctas) : 0.f;
#pragma unroll
      for (int r = 0; r < 8; ++r)
        if (r < ctas) v += part[r] * scale[r];
      const size_t head = (size_t)fs.b * p.q_heads + head0 + h;
      static_cast<T*>(p.out)[head * d + x] = from_f32<T>(v);
      if (x == 0 && p.lse != nullptr) p.lse[head] = lse2 * kLn2;
    }
    if (p.track) {
      if (tid < heads) {
        sh_lse[tid] = track_lse(total_of(tid >> 3, tid & 1, (tid & 7) >> 1, scale));
      }
      __syncthreads();
      const int r_first = fs.tile0 * kBlockRows, r_end = min(fs.len, r_first + fs.n * kBlockRows);
      for (int r = r_first + tid; r < r_end; r += kThreads) {
        int line;
        const int page = p.c.page_of(fs.b, r, &line);
        const float* sc = my_scores + (r - r_first) * p.score_pitch;
        float add = 0.f;
        for (int h = 0; h < heads; ++h) add += probability(sc[h], sh_lse[h]);
        if (p.c.real(page)) p.c.weight[p.c.slot_at(page, fs.kvh, line)] += add;
      }
    }
    if (ctas > 1) cluster_sync_all();  // nobody leaves while others look at its shared memory
  }
}

// Joins what was cut, a CTA for each (sequence, query head).  Every warp works out the
// head's maximum and sum from the partials' (m, l), a lane for each; the partial outputs
// are added by groups of dim / 4 threads, each taking every n-th, and then in group order.
// (One thread per value, walking all partials one after the other, took 40 us for 19
// partials: two loads from L2 at a time.)
constexpr int kFinishThreads = 128;

struct Total {
  float top, sum;  // log2 units
  __device__ __forceinline__ float lse2() const { return top + log2f(sum); }
};

// A row's partials are the first's slot and the even ones after it, up to the last CTA's.
__device__ __forceinline__ int partials(int2 info) { return info.y - (info.x >> 1) + 1; }
__device__ __forceinline__ int slot_of(int2 info, int i) { return i == 0 ? info.x : ((info.x >> 1) + i) * 2; }

// All lanes of a warp together.
template <int H>
__device__ __forceinline__ Total total_of(const AttnParams& p, int2 info, int h) {
  const int n = partials(info), lane = threadIdx.x & 31;
  float top = -INFINITY, sum = 0.f;
  for (int i = lane; i < n; i += 32) top = fmaxf(top, p.part_ml[(size_t)slot_of(info, i) * H + h].x);
  for (int sft = 16; sft > 0; sft >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, sft));
  const float base = top == -INFINITY ? 0.f : top;
  for (int i = lane; i < n; i += 32) {
    const float2 ml = p.part_ml[(size_t)slot_of(info, i) * H + h];
    sum += ml.y * ex2_approx(ml.x - base);
  }
  for (int sft = 16; sft > 0; sft >>= 1) sum += __shfl_xor_sync(~0u, sum, sft);
  return {top, sum};
}

template <class T, int H>
__global__ void __launch_bounds__(kFinishThreads) paged_join_kernel(const __grid_constant__ AttnParams p) {
  __shared__ float4 acc_of[kFinishThreads];
  pdl_wait();
  pdl_launch_dependents();
  const int b = blockIdx.x / p.q_heads, head = blockIdx.x - b * p.q_heads;
  const int kvh = head / p.group, in_group = head - kvh * p.group, part = in_group / H, h = in_group - part * H;
  const int row = (b * p.c.heads + kvh) * p.parts + part, d = p.c.dim, quads = d / 4;
  T* out = static_cast<T*>(p.out) + ((size_t)b * p.q_heads + head) * d;
  if (p.c.rows(b) == 0) {  // nothing to attend to
    for (int i = threadIdx.x; i < d; i += kFinishThreads) out[i] = from_f32<T>(0.f);
    if (threadIdx.x == 0 && p.lse != nullptr) p.lse[(size_t)b * p.q_heads + head] = -INFINITY;
    return;
  }
  const int2 info = p.row_info[row];
  if (info.x < 0) return;  // done in one piece
  const Total t = total_of<H>(p, info, h);
  const float base = t.top == -INFINITY ? 0.f : t.top;
  const int n = partials(info), groups = kFinishThreads / quads, g = threadIdx.x / quads, at = threadIdx.x - g * quads;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  if (g < groups) {
#pragma unroll 4
    for (int i = g; i < n; i += groups) {
      const size_t slot = (size_t)slot_of(info, i) * H + h;
      const float f = ex2_approx(p.part_ml[slot].x - base);
      const float4 o = *reinterpret_cast<const float4*>(p.part_o + slot * d + at * 4);
      acc.x += o.x * f;
      acc.y += o.y * f;
      acc.z += o.z * f;
      acc.w += o.w * f;
    }
  }
  acc_of[threadIdx.x] = acc;
  __syncthreads();
  for (int i = threadIdx.x; i < d; i += kFinishThreads) {
    const float* v = reinterpret_cast<const float*>(acc_of) + i;
    float x = 0.f;
    for (int j = 0; j < groups; ++j) x += v[j * d];
    out[i] = from_f32<T>(t.top == -INFINITY ? 0.f : x / t.sum);
  }
  if (threadIdx.x == 0) {
    if (p.lse != nullptr) p.lse[(size_t)b * p.q_heads + head] = t.lse2() * kLn2;
    if (p.track) p.row_lse[(size_t)row * H + h] = track_lse(t.lse2());
  }
}

// Adds the probabilities to the cache's weights: R rows a thread of one (sequence,
// key-value head), a power of two P of scores for each, all loads before the first use.
// A kernel of its own, behind the join: where its CTAs worked the sums out for themselves,
// that was most of their instructions (33 us with 1024 rows a CTA, 52 us with the loads in
// front but fewer CTAs on an SM; 64 sequences of 17 to 8192 rows, 8 key-value heads, 4
// query heads each).
template <int P, int H>
__global__ void __launch_bounds__(kFinishThreads) paged_track_kernel(const __grid_constant__ AttnParams p) {
  constexpr int R = P == 16 ? 2 : 4;
  pdl_wait();
  pdl_launch_dependents();
  const int b = blockIdx.x / p.c.heads, kvh = blockIdx.x - b * p.c.heads, len = p.c.rows(b);
  const long long step = R * kFinishThreads;
  for (long long r0 = blockIdx.y * step; r0 < len; r0 += gridDim.y * step) {
    float* weight[R];
    float was[R], add[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const long long r = r0 + i * kFinishThreads + threadIdx.x;
      int line = 0;
      const int page = r < len ? p.c.page_of(b, (int)r, &line) : -1;
      weight[i] = p.c.real(page) ? p.c.weight + p.c.slot_at(page, kvh, line) : nullptr;
      was[i] = weight[i] != nullptr ? *weight[i] : 0.f;
      add[i] = 0.f;
    }
    for (int part = 0; part < p.parts; ++part) {
      const int row = (int)blockIdx.x * p.parts + part, heads = min(H, p.group - part * H);
      const int unit = p.row_unit[row];
      if (unit < 0) return;
      const float* from = p.scores + ((size_t)unit * kBlockRows + r0 + threadIdx.x) * P;
      __align__(16) float s[R][P];
      float lse[P];
#pragma unroll
      for (int h = 0; h < P; ++h) lse[h] = h < heads ? p.row_lse[(size_t)row * H + h] : 0.f;
#pragma unroll
      for (int i = 0; i < R; ++i)
        if (weight[i] != nullptr) {
          if constexpr (P == 2) {
            *reinterpret_cast<float2*>(s[i]) = *reinterpret_cast<const float2*>(from + i * kFinishThreads * P);
          } else {
#pragma unroll
            for (int h = 0; h < P; h += 4)
              *reinterpret_cast<float4*>(s[i] + h) = *reinterpret_cast<const float4*>(from + i * kFinishThreads * P + h);
          }
        }
#pragma unroll
      for (int h = 0; h < P; ++h) {
#pragma unroll
        for (int i = 0; i < R; ++i)
          if (h < heads) add[i] += probability(s[i][h], lse[h]);
      }
    }
#pragma unroll
    for (int i = 0; i < R; ++i)
      if (weight[i] != nullptr) *weight[i] = was[i] + add[i];
  }
}

// ---- host ----------------------------------------------------------------------
struct Plan {
  int nt, parts, ks, ctas, rows, score_pitch;
  int short_ctas;       // CTAs of a pair in the form without further kernels, or 0
  size_t short_scores;  // its shared memory for scores
  int score_units;
  size_t part_o, part_ml, row_info, row_lse, row_unit, scores, bytes;
};

// Steps of 16 columns that there are kernels for: every even size up to 12 and 5, which
// heads of 72 and 80 need, then 16.
int steps_for(int dim) {
  const int need = (dim + 15) / 16;
  return need <= 4 ? 4 : need <= 6 ? need : need <= 8 ? 8 : need <= 10 ? 10 : need <= 12 ? 12 : 16;
}

template <class F>
auto with_steps(int ks, F f) {
  switch (ks) {
    case 4: return f(std::integral_constant<int, 4>());
    case 5: return f(std::integral_constant<int, 5>());
    case 6: return f(std::integral_constant<int, 6>());
    case 8: return f(std::integral_constant<int, 8>());
    case 10: return f(std::integral_constant<int, 10>());
    case 12: return f(std::integral_constant<int, 12>());
    default: return f(std::integral_constant<int, 16>());
  }
}

constexpr size_t kMaxSmem = 227 * 1024 - 2048;  // dynamic; the kernels have some static

size_t short_smem(int ks, int nt) {
  return with_steps(ks, [&](auto k) { return nt == 1 ? Tile<k(), 1, true>::kSmem : Tile<k(), 2, true>::kSmem; });
}

int per_sm(int ks, int nt) {
  return with_steps(ks, [&](auto k) { return nt == 1 ? Tile<k(), 1, false>::kPerSM : Tile<k(), 2, false>::kPerSM; });
}

Plan make_plan(const Pi05PagedCache* c, int q_heads, int track) {
  Plan s{};
  const int group = q_heads / c->n_kv_heads;
  s.nt = group <= 8 ? 1 : 2;
  s.parts = (group + 8 * s.nt - 1) / (8 * s.nt);
  s.ks = steps_for(c->head_dim);
  s.rows = c->batch * c->n_kv_heads * s.parts;
  const long long capacity = (long long)c->pages_per_seq * c->page_size;
  auto blocks_of = [](long long rows) { return (rows + kBlockRows - 1) / kBlockRows; };
  const long long blocks = blocks_of(capacity) * s.rows;
  s.ctas = (int)std::min<long long>(blocks, (long long)kSMs * per_sm(s.ks, s.nt));
  s.score_pitch = 2;
  while (s.score_pitch < std::min(8 * s.nt, group)) s.score_pitch *= 2;
  // The form without further kernels: up to 8 CTAs for each pair while two of them (one,
  // for heads over 128) have an SM to themselves, with 1024 rows each at most (512).  us a
  // call there / with equal shares (32 / 8 heads of 128, uniform lengths): 32 pairs of 1000
  // rows 7.8 / 13.5, of 8000 26 / 31; 128 of 512 13 / 16, of 2000 28 / 30, of 1 to 2000 24 /
  // 22; 120 of 512 rows of 256 columns 22 / 28.  Beyond, the longest sequence or the scores'
  // share of an SM decides: 320 pairs of 512 rows, tracked, 36 / 28; 384 of 1 to 1500 rows
  // of 80 columns 30 / 26; 150 of 512 rows of 256 columns 40 / 29; 1600 of 512 rows of 64
  // columns 44 / 43.  All with tables of the longest sequence's length: the host knows the table's
  // reach and not the lengths, so short sequences behind a long table go by the second figures.
  const bool narrow = s.ks <= 8;
  const long long pairs = (long long)c->batch * c->n_kv_heads, at_once = narrow ? 2 * kSMs : kSMs;
  int ctas = 8;
  while (ctas > 1 && (pairs * ctas > at_once || ctas > blocks_of(capacity))) ctas /= 2;
  const size_t scores = (size_t)((blocks_of(capacity) + ctas - 1) / ctas) * kBlockRows * s.score_pitch * 4;
  if (s.parts == 1 && capacity <= (narrow ? 1024 : 512) * ctas && pairs * ctas <= at_once &&
      short_smem(s.ks, s.nt) + scores <= kMaxSmem) {  // with or without tracking, so that it changes no result
    s.short_ctas = ctas;
    s.short_scores = track ? scores : 0;
    return s;  // no scratch
  }
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
  // Scores for every row that the table reaches, or, beyond 64 MB, that the pool has (in blocks: a
  // block begun and the border for each pair): whoever tracks has each row in one sequence alone.
  // No less than for one pair that the table's reach fills.
  const size_t unit_bytes = (size_t)kBlockRows * s.score_pitch * 4;
  const long long pool = ((long long)c->num_pages * c->page_size / kBlockRows + (1ll + kBorder) * c->batch) *
                         c->n_kv_heads * s.parts;
  const long long longest = blocks_of(capacity) + kBorder;
  s.score_units = (int)std::min<long long>(
      {longest * s.rows, std::max<long long>({pool, longest, (long long)((64 << 20) / unit_bytes)}), 0x7fffffff});
  s.row_unit = take(track ? (size_t)s.rows * 4 : 0);
  s.scores = take(track ? s.score_units * unit_bytes : 0);
  s.bytes = at;
  return s;
}

template <class T, int KS, int NT>
int launch(const AttnParams& p, const Plan& s, const CUtensorMap* tm, cudaStream_t st) {
  using L = Tile<KS, NT, false>;
  using LS = Tile<KS, NT, true>;
  static_assert(L::kSmem <= 227 * 1024 && LS::kSmem <= kMaxSmem, "shared memory");
  if (s.short_ctas > 0) {
    static std::atomic<uint64_t> allowed{0};
    auto kernel = paged_attention_kernel<T, KS, NT, true>;
    int rc = allow_smem(kernel, kMaxSmem, &allowed, "paged_attention");
    if (rc) return rc;
    return launch_pdl_cluster(kernel, dim3(p.c.batch * p.c.heads * s.short_ctas), dim3(kThreads),
                              LS::kSmem + s.short_scores, st, pdl_enabled(), dim3(s.short_ctas), p, tm[0], tm[1]);
  }
  static std::atomic<uint64_t> allowed{0};
  auto kernel = paged_attention_kernel<T, KS, NT, false>;
  int rc = allow_smem(kernel, L::kSmem, &allowed, "paged_attention");
  if (rc) return rc;
  // Not ahead of the kernel before it: on an SM where that still runs, with less shared
  // memory set apart, fewer of the CTAs fit than the shares are made for, and the rest come
  // after the first (24 x 32 pairs of 2000 rows back to back: 164 us, and 122 in order).
  rc = launch_pdl(kernel, dim3(s.ctas), dim3(kThreads), L::kSmem, st, false, p, tm[0], tm[1]);
  if (rc) return rc;
  rc = launch_pdl(paged_join_kernel<T, 8 * NT>, dim3(p.c.batch * p.q_heads), dim3(kFinishThreads), 0, st,
                  pdl_enabled(), p);
  if (rc || !p.track) return rc;
  const int per_cta = (p.score_pitch == 16 ? 2 : 4) * kFinishThreads;
  const int pairs = p.c.batch * p.c.heads;  // CTAs for the longest there can be, but not many more than can run
  const dim3 grid(pairs, std::min((p.c.capacity + per_cta - 1) / per_cta, std::max(16, 4096 / pairs)));
  if constexpr (NT == 2)
    return launch_pdl(paged_track_kernel<16, 16>, grid, dim3(kFinishThreads), 0, st, pdl_enabled(), p);
  else
    return launch_pdl(p.score_pitch == 2   ? paged_track_kernel<2, 8>
                      : p.score_pitch == 4 ? paged_track_kernel<4, 8>
                                           : paged_track_kernel<8, 8>,
                      grid, dim3(kFinishThreads), 0, st, pdl_enabled(), p);
}

template <class T>
int launch_type(const AttnParams& p, const Plan& s, const CUtensorMap* tm, cudaStream_t st) {
  return with_steps(s.ks, [&](auto k) {
    return s.nt == 1 ? launch<T, k(), 1>(p, s, tm, st) : launch<T, k(), 2>(p, s, tm, st);
  });
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
  const long long q_token = stride_of(cache->batch, a->q_token_stride);
  const long long q_head = stride_of(a->n_q_heads, a->q_head_stride);
  if (!aligned_to(4, a->q, a->lse) || !aligned_to(2, a->out) || q_token % 2 || q_head % 2) {
    set_last_error("paged_attention: q rows and lse must start on 4-byte boundaries, out on 2-byte ones");
    return PI05_ERR_ALIGN;
  }
  const Plan s = make_plan(cache, a->n_q_heads, a->track);
  if (s.bytes > 0 && (a->scratch == nullptr || a->scratch_bytes < s.bytes)) {
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
  p.qt = q_token;
  p.qh = q_head;
  p.valid_pitch = a->valid_pitch;
  p.valid_rows = a->key_valid != nullptr ? a->valid_rows : 0;
  p.q_heads = a->n_q_heads;
  p.group = a->n_q_heads / cache->n_kv_heads;
  p.parts = s.parts;
  p.scale_log2 = a->scale * 1.44269504088896340736f;
  p.track = a->track;
  p.part_o = reinterpret_cast<float*>(sc + s.part_o);
  p.part_ml = reinterpret_cast<float2*>(sc + s.part_ml);
  p.row_info = reinterpret_cast<int2*>(sc + s.row_info);
  p.row_lse = reinterpret_cast<float*>(sc + s.row_lse);
  p.scores = reinterpret_cast<float*>(sc + s.scores);
  p.row_unit = reinterpret_cast<int*>(sc + s.row_unit);
  p.score_units = s.score_units;
  p.score_pitch = s.score_pitch;
  p.ctas = s.short_ctas;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  p.box_rows = std::min(kWarpRows, cache->page_size & -cache->page_size);
  const uint64_t dims[4] = {(uint64_t)cache->head_dim, (uint64_t)cache->page_size, (uint64_t)cache->n_kv_heads,
                            (uint64_t)cache->num_pages};
  const uint64_t strides[3] = {(uint64_t)p.c.row_stride, (uint64_t)p.c.head_stride, (uint64_t)p.c.page_stride};
  CUtensorMap tm[2];
  for (int i = 0; i < 2; ++i) {
    rc = make_tmap_16bit_4d(&tm[i], i == 0 ? cache->k_pages : cache->v_pages, dims, strides, p.box_rows);
    if (rc) return rc;
  }
  return cache->dtype == PI05_BF16 ? launch_type<__nv_bfloat16>(p, s, tm, st) : launch_type<__half>(p, s, tm, st);
}

}  // extern "C"
