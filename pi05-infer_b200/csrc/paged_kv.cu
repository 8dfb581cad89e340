// The paged key-value cache: append (with the rotation of q and k) and eviction by
// accumulated attention weight.
#include <algorithm>

#include "paged.cuh"

namespace pi05 {

int paged_check(const Pi05PagedCache* c, const char* op, Pages* out) {
  if (c == nullptr || c->k_pages == nullptr || c->v_pages == nullptr || c->page_table == nullptr ||
      c->counts == nullptr) {
    set_last_error("%s: null pointer", op);
    return PI05_ERR_INVALID_ARG;
  }
  if (c->dtype != PI05_BF16 && c->dtype != PI05_FP16) {
    set_last_error("%s: dtype %d is not bf16 or fp16", op, c->dtype);
    return PI05_ERR_INVALID_ARG;
  }
  const long long capacity = (long long)c->pages_per_seq * c->page_size;
  if (c->num_pages <= 0 || c->page_size <= 0 || c->n_kv_heads <= 0 || c->batch <= 0 || c->pages_per_seq <= 0 ||
      c->table_pitch < c->pages_per_seq || c->head_dim <= 0 || c->head_dim % 8 || c->head_dim > 256 ||
      capacity >= (1ll << 31) - (1 << 20) || (long long)c->batch * c->n_kv_heads >= (1 << 24)) {
    set_last_error("%s: bad cache shape pages=%d x %d kv_heads=%d head_dim=%d batch=%d pages_per_seq=%d pitch=%d", op,
                   c->num_pages, c->page_size, c->n_kv_heads, c->head_dim, c->batch, c->pages_per_seq, c->table_pitch);
    return PI05_ERR_SHAPE;
  }
  if (!aligned16(c->k_pages) || !aligned16(c->v_pages) || c->page_stride % 8 || c->head_stride % 8 ||
      c->row_stride % 8) {
    set_last_error("%s: cache rows must start on 16-byte boundaries", op);
    return PI05_ERR_ALIGN;
  }
  if (!aligned_to(4, c->weight, c->pos, c->page_table, c->counts)) {
    set_last_error("%s: weight, pos, page_table and counts must be 4-byte aligned", op);
    return PI05_ERR_ALIGN;
  }
  if (c->workspace == nullptr || c->workspace_bytes < kWsAccumOffset + paged_moves_bytes(c)) {
    set_last_error("%s: workspace missing or too small", op);
    return PI05_ERR_WORKSPACE;
  }
  if ((reinterpret_cast<uintptr_t>(c->workspace) & 255) != 0) {
    set_last_error("%s: workspace not 256-byte aligned", op);
    return PI05_ERR_ALIGN;
  }
  char* ws = static_cast<char*>(c->workspace);
  out->k = static_cast<char*>(c->k_pages);
  out->v = static_cast<char*>(c->v_pages);
  out->page_stride = c->page_stride * 2;
  out->head_stride = c->head_stride * 2;
  out->row_stride = c->row_stride * 2;
  out->weight = c->weight;
  out->pos = c->pos;
  out->table = c->page_table;
  out->counts = c->counts;
  out->status = reinterpret_cast<int*>(ws + kWsStatusOffset);
  out->ticket = reinterpret_cast<int*>(ws + kWsCounterOffset);
  out->tickets = reinterpret_cast<int*>(ws + kWsAccumOffset);
  out->moves = reinterpret_cast<int2*>(out->tickets + c->batch + (c->batch & 1));
  out->move_list = reinterpret_cast<int32_t*>(out->moves + paged_pairs(c));
  out->list_by_slot = paged_list_by_slot(c);
  out->page_div = FastDiv((uint32_t)c->page_size);
  out->num_pages = c->num_pages;
  out->page_size = c->page_size;
  out->heads = c->n_kv_heads;
  out->dim = c->head_dim;
  out->batch = c->batch;
  out->pitch = c->table_pitch;
  out->capacity = (int)capacity;
  return PI05_OK;
}

namespace {

// ---- append ------------------------------------------------------------------
// Memory bound: q, k and v read once; rotated q, and k and v at their rows, written
// once.  A CTA takes a few tokens: it asks for their values, finds their rows (sequence,
// count, page: three loads one after the other) and cos and sin while those are on their
// way, rotates and stores.
constexpr int kAppendThreads = 128;

struct AppendParams {
  const void *k, *v, *q;
  void* q_out;
  int kt, kh, vt, vh, qt, qh;  // strides, elements
  const int32_t* cu;
  const float* new_weight;
  const uint64_t* turns;
  FastDiv by_qk, by_heads, by_pairs;
  int tokens, q_heads, rotary, interleaved, per_cta;
  int turned, units, lanes;    // of a head of q or k
  int row_units, row_lanes;    // of a head of v
  float magnitude;
};

struct __align__(16) TokenRow {
  long long at;    // byte offset of the row in its head's lines, or -1
  long long slot;  // the same of weight and pos
  int position;
};

// ROT: with rotation.  Two kernels, since the registers of the one cost the other its
// occupancy: with v's first batch held over the row search as well, the append of 16384
// rotated tokens took 44 us instead of 37 (38 with the angles' quarter turns); without, that of
// 65536 plain ones 105 instead of 93.
template <class T, int V, int VC, bool ROT>
__global__ void __launch_bounds__(kAppendThreads) append_kernel(const __grid_constant__ Pages c,
                                                                const __grid_constant__ AppendParams p) {
  extern __shared__ __align__(16) char smem[];
  TokenRow* row_of = reinterpret_cast<TokenRow*>(smem);        // [per_cta]
  float2* cs = reinterpret_cast<float2*>(row_of + p.per_cta);  // [per_cta][rotary / 2]
  __shared__ int last, cu_of[kAppendThreads], held_of[kAppendThreads], seen_of[kAppendThreads];
  pdl_wait();
  pdl_launch_dependents();
  const int tid = threadIdx.x, pairs = p.rotary / 2;
  const int t0 = blockIdx.x * p.per_cta;
  const int used = p.cu != nullptr ? min(max(p.cu[c.batch], 0), p.tokens) : p.tokens;
  const int n = max(0, min(p.per_cta, used - t0));  // 0: padding alone

  const T* q = static_cast<const T*>(p.q) + (long long)t0 * p.qt;
  const T* k = static_cast<const T*>(p.k) + (long long)t0 * p.kt;
  const T* v = static_cast<const T*>(p.v) + (long long)t0 * p.vt;
  T* q_out = static_cast<T*>(p.q_out) + (long long)t0 * p.q_heads * c.dim;

  // Where the CTA's tokens go, and their cos and sin.
  const bool few = p.cu != nullptr && c.batch <= kAppendThreads;
  auto find_rows = [&]() {
    if (few) {  // one load's latency instead of a search's
      if (tid < c.batch) {
        cu_of[tid] = p.cu[tid];
        held_of[tid] = c.counts[tid];
        seen_of[tid] = c.counts[c.batch + tid];
      }
      __syncthreads();
    }
    for (int i = tid; i < n; i += kAppendThreads) {
      const int t = t0 + i;
      int b = t, off = 0;
      if (p.cu != nullptr) {  // the sequence with cu[b] <= t < cu[b + 1]
        int lo = 0, hi = c.batch;
        while (hi - lo > 1) {
          const int mid = (lo + hi) >> 1;
          ((few ? cu_of[mid] : p.cu[mid]) <= t ? lo : hi) = mid;
        }
        b = lo;
        off = t - (few ? cu_of[b] : p.cu[b]);
      }
      const int held = few ? held_of[b] : c.counts[b], seen = few ? seen_of[b] : c.counts[c.batch + b];
      const long long r = (long long)held + off;
      int line = 0, page = -1;
      if (r >= 0 && r < c.capacity) page = c.page_of(b, (int)r, &line);
      TokenRow row{-1, -1, seen + off};
      if (c.real(page)) {
        row.at = (long long)c.row_at(page, 0, line);
        row.slot = (long long)c.slot_at(page, 0, line);
      } else {
        report_status(c.status, PI05_DEV_BAD_INDEX);
      }
      row_of[i] = row;
      if (p.cu == nullptr) {  // nobody else has the sequence
        c.counts[b] = max(held, min(held + 1, c.capacity));
        c.counts[c.batch + b] = seen + 1;
      }
    }
    __syncthreads();
    for (int i = tid; i < n * pairs; i += kAppendThreads) {
      const int t = p.by_pairs.div(i);
      const int f = i - t * pairs;
      cs[t * pairs + Unit<T, V>::place(f, p.turned, p.interleaved)] =
          rotation(row_of[t].position, p.turns[f], p.magnitude, false);
    }
    for (int i = tid; i < n * c.heads; i += kAppendThreads) {
      const int t = p.by_heads.div(i), h = i - t * c.heads;
      if (row_of[t].at < 0) continue;
      const size_t s = row_of[t].slot + (size_t)h * c.page_size;
      if (c.pos != nullptr) c.pos[s] = row_of[t].position;
      if (c.weight != nullptr)
        c.weight[s] = p.new_weight != nullptr ? p.new_weight[(size_t)(t0 + t) * c.heads + h] : 0.f;
    }
    __syncthreads();
  };

  // Rows that are stored as they are (v, and k without rotation): `row_lanes` threads to a
  // row, C rows of a thread at once.  The first batches are asked for before the rows are
  // looked for.
  constexpr int C = ROT ? 2 : 4;
  const int copy_rows = n * c.heads, copy0 = tid / p.row_lanes, copy_step = kAppendThreads / p.row_lanes;
  const int copy_u = tid - copy0 * p.row_lanes;
  auto copy_load = [&](Unit<T, VC>* unit, const T* src, int tt, int hh, int r, int u) {
#pragma unroll
    for (int j = 0; j < C; ++j) {
      const int row = r + j * copy_step, t = p.by_heads.div(row), h = row - t * c.heads;
      if (copy0 < copy_step && row < copy_rows && u < p.row_units)
        unit[j].load_row(src + (long long)t * tt + (long long)h * hh, u);
    }
  };
  auto copy_store = [&](const Unit<T, VC>* unit, char* pages, int r, int u) {
#pragma unroll
    for (int j = 0; j < C; ++j) {
      const int row = r + j * copy_step, t = p.by_heads.div(row), h = row - t * c.heads;
      if (copy0 < copy_step && row < copy_rows && u < p.row_units && row_of[t].at >= 0)
        unit[j].store_row(reinterpret_cast<T*>(pages + row_of[t].at + h * c.head_stride), u);
    }
  };
  auto copy_rest = [&](const T* src, int tt, int hh, char* pages, bool all) {
    for (int u = copy_u; u < p.row_units; u += p.row_lanes)
      for (int r = copy0 + (u == copy_u && !all ? C * copy_step : 0); r < copy_rows; r += C * copy_step) {
        Unit<T, VC> unit[C];
        copy_load(unit, src, tt, hh, r, u);
        copy_store(unit, pages, r, u);
      }
  };

  if constexpr (!ROT) {
    Unit<T, VC> k_first[C], v_first[C];
    copy_load(k_first, k, p.kt, p.kh, copy0, copy_u);
    copy_load(v_first, v, p.vt, p.vh, copy0, copy_u);
    find_rows();
    copy_store(k_first, c.k, copy0, copy_u);
    copy_store(v_first, c.v, copy0, copy_u);
    copy_rest(k, p.kt, p.kh, c.k, false);
  } else {  // q and k: `lanes` threads to a head's units, kAppendThreads / lanes heads at a time
    constexpr int J = 2;
    bool ready = false;
    const int heads = p.q_heads + c.heads, rows = n * heads;
    const int row0 = tid / p.lanes, u0 = tid - row0 * p.lanes, step = kAppendThreads / p.lanes;
    for (int u = u0; u < p.units || u == u0; u += p.lanes) {
      const bool mine = u < p.units && row0 < step;
      for (int r = row0; r < rows || !ready; r += J * step) {
        Unit<T, V> unit[J];
        int token[J], head[J];
#pragma unroll
        for (int j = 0; j < J; ++j) {
          const int row = r + j * step;
          token[j] = p.by_qk.div(row);
          head[j] = row - token[j] * heads;
          if (mine && row < rows)
            unit[j].load(head[j] < p.q_heads ? q + (long long)token[j] * p.qt + (long long)head[j] * p.qh
                                             : k + (long long)token[j] * p.kt + (long long)(head[j] - p.q_heads) * p.kh,
                         u, p.turned, p.rotary, p.interleaved);
        }
        if (!ready) find_rows();
        ready = true;
#pragma unroll
        for (int j = 0; j < J; ++j) {
          if (!mine || r + j * step >= rows) continue;
          T* dst;
          if (head[j] < p.q_heads) {
            dst = q_out + (long long)(token[j] * p.q_heads + head[j]) * c.dim;
          } else {
            const long long at = row_of[token[j]].at;
            if (at < 0) continue;
            dst = reinterpret_cast<T*>(c.k + at + (head[j] - p.q_heads) * c.head_stride);
          }
          unit[j].store(dst, u, p.turned, p.rotary, p.interleaved, cs + token[j] * pairs);
        }
      }
    }
  }
  copy_rest(v, p.vt, p.vh, c.v, ROT);
  if (p.cu == nullptr) return;
  // Ragged: the CTA that finishes last moves the counts on, when all have read them.
  __syncthreads();
  if (tid == 0) last = atom_add_acq_rel_gpu(c.ticket, 1) == (int)gridDim.x - 1;
  __syncthreads();
  if (!last) return;
  for (int b = tid; b < c.batch; b += kAppendThreads) {
    const int m = max(min(p.cu[b + 1], p.tokens) - max(p.cu[b], 0), 0), held = c.counts[b];
    c.counts[b] = max(held, (int)min((long long)held + m, (long long)c.capacity));
    c.counts[c.batch + b] += m;
  }
  if (tid == 0) *c.ticket = 0;
}

// ---- eviction ------------------------------------------------------------------
// A cluster of CTAs for each (sequence, head): each holds a run of the rows as 32-bit keys
// that sort like the weight in shared memory, so that weights and positions are read from
// memory once.  Radix selection, 11 bits a pass over all the cluster's histograms, gives
// the key of the last row to go and how many rows of just that key go with it; then the
// holes below the budget and the rows that fill them are counted, and listed in order.
// Bound: latency (three passes and a count, each a cluster barrier).  One CTA that read
// the weights from L2 in every pass took 100 us for 512 pairs of 2049 rows and 409 us for
// 8 pairs of 65536.  With 8 bits a pass, 26 and 57 us: a weight's top 8 bits are its
// sign and exponent but one bit, so that most rows of a pass add to the same few counters,
// one after the other.  This form: 10 us (one row to go) and 31 us.
constexpr int kFew = 4;  // rows to go that are looked for one by one
constexpr int kBuckets = 2048;
constexpr int kMaxKeys = 48 * 1024;  // that a CTA holds; later ones are worked out again
constexpr int kMoveThreads = 256;

__device__ __forceinline__ uint32_t evict_key(float w, int pos, long long recent_from, int sinks) {
  if (pos >= recent_from || pos < sinks) return 0xffffffffu;
  if (w != w) return 0u;
  if (w == 0.f) return 0x80000000u;
  const uint32_t u = __float_as_uint(w);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ int4 ld_cluster4(const int4* p, uint32_t rank) {
  int4 v;
  asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(mapa_shared(smem_u32(p), rank))
               : "memory");
  return v;
}
__device__ __forceinline__ int ld_cluster(const void* p, uint32_t rank) {
  int v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(mapa_shared(smem_u32(p), rank)) : "memory");
  return v;
}

// Copies a row's key and value, weight and position; one warp.  Rows of no page can only come
// from a list at slots that another sequence has, too (which the table may not say); elsewhere the
// copy does not wait to know.
__device__ __forceinline__ void move_row(const Pages& c, bool check, int b, int h, int from_row, int to_row,
                                         int lane) {
  int from_line, to_line;
  const int from = c.page_of(b, from_row, &from_line), to = c.page_of(b, to_row, &to_line);
  if (check && (!c.real(from) || !c.real(to))) {
    if (lane == 0) report_status(c.status, PI05_DEV_BAD_INDEX);
    return;
  }
  const size_t src = c.row_at(from, h, from_line), dst = c.row_at(to, h, to_line);
  if (lane < c.dim / 8) {
    const uint4 k = ld16(c.k + src + lane * 16), v = ld16(c.v + src + lane * 16);
    st16(c.k + dst + lane * 16, k);
    st16(c.v + dst + lane * 16, v);
  }
  if (lane == 0) {
    const size_t s = c.slot_at(from, h, from_line), t = c.slot_at(to, h, to_line);
    c.weight[t] = c.weight[s];
    c.pos[t] = c.pos[s];
  }
}

// Sum of the first `n` (at most 32) of a warp's `x`.
__device__ __forceinline__ int sum_before(const int* x, int n, int lane) {
  return __reduce_add_sync(~0u, lane < n ? x[lane] : 0);
}

struct Victim {
  uint32_t key;
  int row;
  __device__ __forceinline__ bool before(uint32_t k, int r) const { return key < k || (key == k && row < r); }
};
// The warp's least: lowest key, then lowest row.
__device__ __forceinline__ Victim warp_least(Victim v) {
  const uint32_t k = __reduce_min_sync(~0u, v.key);
  return {k, (int)__reduce_min_sync(~0u, v.key == k ? (unsigned)v.row : 0x7fffffffu)};
}

// The list of a (sequence, head); entry i is below the rows it holds, all in real pages.
struct MoveList {
  const Pages& c;
  const bool by_slot;
  int b, h;
  int32_t* dense;
  __device__ __forceinline__ MoveList(const Pages& pages, bool slots, int seq, int head)
      : c(pages), by_slot(slots), b(seq), h(head),
        dense(pages.move_list + (size_t)(seq * pages.heads + head) * pages.capacity) {}
  __device__ __forceinline__ int32_t* at(int i) const {
    if (!by_slot) return dense + i;
    int line;
    const int page = c.page_of(b, i, &line);
    return c.move_list + c.slot_at(page, h, line);
  }
};

// The list: the holes, ascending, and from entry `left` on the rows that fill them.
// `move_here`: few enough, however long the sequence, to do them on the spot.  FIT: a CTA holds all its keys.
template <int NT, bool FIT>
__global__ void __launch_bounds__(NT) evict_select_kernel(const __grid_constant__ Pages c, int budget, int recent,
                                                          int sinks, int ctas, int held, int move_here) {
  constexpr int NW = NT / 32;
  extern __shared__ uint32_t keys[];  // [held]
  __shared__ __align__(16) int hist[2][kBuckets];
  __shared__ int warp_a[NW], warp_b[NW];
  __shared__ int sh_bad, sh_counts[2];
  __shared__ uint32_t sh_prefix;
  __shared__ int sh_want, sh_same;
  __shared__ Victim warp_best[2][NW], cta_best[2];
  pdl_wait();
  pdl_launch_dependents();
  const int pair = blockIdx.x / ctas, rank = blockIdx.x - pair * ctas;  // the grid is a line of clusters
  const int b = pair / c.heads, h = pair - b * c.heads, tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  const int len = c.rows(b);
  const long long recent_from = (long long)c.counts[c.batch + b] - recent;
  if (len <= budget) {  // the whole cluster alike
    if (tid == 0 && rank == 0) c.moves[pair].x = -1;
    return;
  }
  auto sync_all = [&]() {
    if (ctas > 1) cluster_sync_all();
    else __syncthreads();
  };
  auto peer = [&](const int* p, int r) { return ctas > 1 ? ld_cluster(p, r) : *p; };

  // This CTA's rows, and a warp's among them: whole groups of 32 in order.
  const int share = ((len + ctas - 1) / ctas + 31) & ~31, first = min(len, rank * share);
  const int n = min(len - first, share);
  bool bad = false;
  auto key_of = [&](int i) {
    int line;
    const int page = c.page_of(b, first + i, &line);
    if (!c.real(page)) {
      bad = true;
      return 0u;
    }
    const size_t s = c.slot_at(page, h, line);
    return evict_key(c.weight[s], c.pos[s], recent_from, sinks);
  };
  const int kept = FIT ? n : min(n, held);
  constexpr int U = 8;  // rows of a thread whose table entries, then weights, are on their way at once
  for (int i0 = tid; i0 < kept; i0 += U * NT) {
    int page[U], line[U], pos[U];
    float weight[U];
#pragma unroll
    for (int j = 0; j < U; ++j) page[j] = i0 + j * NT < kept ? c.page_of(b, first + i0 + j * NT, &line[j]) : -1;
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const bool real = c.real(page[j]);
      const size_t s = real ? c.slot_at(page[j], h, line[j]) : 0;
      weight[j] = real ? c.weight[s] : 0.f;
      pos[j] = real ? c.pos[s] : 0;
      bad = bad || (!real && i0 + j * NT < kept);
    }
#pragma unroll
    for (int j = 0; j < U; ++j)
      if (i0 + j * NT < kept) keys[i0 + j * NT] = evict_key(weight[j], pos[j], recent_from, sinks);
  }
  for (int i = kept + tid; i < n; i += NT) key_of(i);  // for a bad page
  auto key = [&](int i) { return FIT || i < held ? keys[i] : key_of(i); };
  if (tid == 0) sh_bad = 0;
  __syncthreads();
  if (bad) sh_bad = 1;
  sync_all();
  // Others' values: a lane for each CTA, all on their way at once (one after the other, the
  // eight of a cluster took 2 us each time).
  auto of_all = [&](const int* x) { return lane < ctas ? peer(x, lane) : 0; };
  if (__any_sync(~0u, of_all(&sh_bad) != 0)) {
    if (tid == 0 && rank == 0) {
      c.moves[pair].x = -1;
      report_status(c.status, PI05_DEV_BAD_INDEX);
    }
    sync_all();  // nobody leaves while others look at its shared memory
    return;
  }
  auto cut_count = [&]() {  // the head that is done last cuts the count, when all have read it
    if (tid == 0 && rank == 0 && atom_add_acq_rel_gpu(&c.tickets[b], 1) == c.heads - 1) {
      c.tickets[b] = 0;
      c.counts[b] = budget;
    }
  };

  // A few rows to go (one, in a program that evicts after every token): one by one, the
  // least that comes after the last.
  if (len - budget <= kFew) {
    if (tid == 0 && rank == 0) c.moves[pair].x = -1;  // done here
    Victim gone[kFew];
    const int few = len - budget;
#pragma unroll
    for (int v = 0; v < kFew; ++v) {
      if (v >= few) break;
      Victim best{0xffffffffu, 0x7fffffff};
      for (int i = tid; i < n; i += NT) {
        const uint32_t k = key(i);
        if ((v == 0 || gone[v > 0 ? v - 1 : 0].before(k, first + i)) && !best.before(k, first + i)) best = {k, first + i};
      }
      best = warp_least(best);
      if (lane == 0) warp_best[v & 1][w] = best;
      __syncthreads();
      best = warp_least(lane < NW ? warp_best[v & 1][lane] : Victim{0xffffffffu, 0x7fffffff});
      if (ctas > 1) {
        if (tid == 0) cta_best[v & 1] = best;
        sync_all();
        const int r = min(lane, ctas - 1);
        best.key = (uint32_t)ld_cluster(&cta_best[v & 1].key, r);
        best.row = ld_cluster(&cta_best[v & 1].row, r);
        best = warp_least(best);
      }
      gone[v] = best;
    }
    if (w == 0 && rank == 0) {
      // Holes in order, and the rows from the budget on that stay, in order: lane v has the
      // v-th victim and row budget + v.
      int mine = 0x7fffffff;
#pragma unroll
      for (int v = 0; v < kFew; ++v)
        if (v < few && lane == v) mine = gone[v].row;
      bool stays = lane < few;
      int at = 0;
#pragma unroll
      for (int v = 0; v < kFew; ++v) {
        if (v < few && gone[v].row == budget + lane) stays = false;
        if (v < few && gone[v].row < mine) ++at;
      }
      const uint32_t tails = __ballot_sync(~0u, stays);
      for (int v = 0; v < __popc(tails); ++v) {
        const int to = __shfl_sync(~0u, mine, __ffs(__ballot_sync(~0u, lane < few && at == v)) - 1);
        move_row(c, false, b, h, budget + __fns(tails, 0, v + 1), to, lane);
      }
    }
    if (ctas > 1) sync_all();  // nobody leaves while others look at its shared memory
    cut_count();
    return;
  }

  for (int i = tid; i < 2 * kBuckets; i += NT) (&hist[0][0])[i] = 0;
  __syncthreads();
  uint32_t prefix = 0;
  int want = len - budget, same = 0;  // the want-th smallest of the keys that begin with `prefix`
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
    int* mine = hist[pass & 1];
    for (int g = w * 32; g < n; g += NT) {
      const int i = g + lane;
      const uint32_t k = i < n ? key(i) : 0u;
      const bool in = i < n && (pass == 0 || (k >> (shift + bits)) == (prefix >> (shift + bits)));
      // Rows of the same bucket as the warp's first (all protected, say, or all 0) in one go.
      const uint32_t bucket = in ? (k >> shift) & ((1u << bits) - 1) : ~0u, lead = __shfl_sync(~0u, bucket, 0);
      const uint32_t alike = __ballot_sync(~0u, in && bucket == lead);
      if (lane == 0 && in) atomicAdd(&mine[bucket], __popc(alike));
      else if (in && bucket != lead) atomicAdd(&mine[bucket], 1);
    }
    sync_all();
    if (pass > 0)  // the buffer of the pass before: everybody has read it
      for (int i = tid; i < kBuckets; i += NT) hist[1 - (pass & 1)][i] = 0;
    // Four or eight buckets a thread, over all the cluster.
    constexpr int Q = kBuckets / NT / 4;
    int4 of[Q];
    int sum = 0;
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const int4* own = reinterpret_cast<const int4*>(mine) + tid * Q + q;
      of[q] = make_int4(0, 0, 0, 0);
#pragma unroll 8
      for (int r = 0; r < ctas; ++r) {
        const int4 v = ctas > 1 ? ld_cluster4(own, r) : *own;
        of[q].x += v.x;
        of[q].y += v.y;
        of[q].z += v.z;
        of[q].w += v.w;
      }
      sum += of[q].x + of[q].y + of[q].z + of[q].w;
    }
    int incl = sum;
    for (int sft = 1; sft < 32; sft <<= 1) {
      const int u = __shfl_up_sync(~0u, incl, sft);
      if (lane >= sft) incl += u;
    }
    if (lane == 31) warp_a[w] = incl;
    __syncthreads();
    incl += sum_before(warp_a, w, lane);
    if (incl >= want && incl - sum < want) {
      int before = incl - sum, bucket = tid * Q * 4;
      bool found = false;
      auto look = [&](int count) {
        if (found) return;
        if (before + count >= want) {
          sh_prefix = prefix | ((uint32_t)bucket << shift);
          sh_want = want - before;
          sh_same = count;
          found = true;
        }
        before += count;
        ++bucket;
      };
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        look(of[q].x);
        look(of[q].y);
        look(of[q].z);
        look(of[q].w);
      }
    }
    __syncthreads();
    prefix = sh_prefix;
    want = sh_want;
    same = sh_same;
  }

  // Keys below `prefix` go, and the first `want` of those that equal it.  Warp w has the
  // groups of 32 from w * per on.
  const uint32_t below = (1u << lane) - 1;
  const int per = (share / 32 + NW - 1) / NW, g0 = w * per;
  int ties = 0;  // before this warp's rows
  if (same > want) {
    int count = 0;
    for (int g = g0; g < g0 + per; ++g) {
      const int i = g * 32 + lane;
      count += __popc(__ballot_sync(~0u, i < n && key(i) == prefix));
    }
    if (lane == 0) warp_a[w] = count;
    __syncthreads();
    if (w == 0) {
      const int sum = sum_before(warp_a, NW, lane);
      if (lane == 0) sh_counts[0] = sum;
    }
    sync_all();
    const int others = of_all(&sh_counts[0]);
    ties = __reduce_add_sync(~0u, lane < rank ? others : 0) + sum_before(warp_a, w, lane);
    sync_all();  // before the counts are written anew
  }
  auto classify = [&](int g, int& seen, bool& hole, bool& tail) {
    const int i = g * 32 + lane, r = first + i;
    const uint32_t k = i < n ? key(i) : ~0u;
    bool gone = i < n && k < prefix;
    const bool tie = i < n && k == prefix;
    if (same > want) {
      const uint32_t m = __ballot_sync(~0u, tie);
      gone = gone || (tie && seen + __popc(m & below) < want);
      seen += __popc(m);
    } else {
      gone = gone || tie;
    }
    hole = gone && r < budget;
    tail = i < n && !gone && r >= budget;
  };
  int holes = 0, tails = 0, seen = ties;
  for (int g = g0; g < g0 + per; ++g) {
    bool hole, tail;
    classify(g, seen, hole, tail);
    holes += __popc(__ballot_sync(~0u, hole));
    tails += __popc(__ballot_sync(~0u, tail));
  }
  if (lane == 0) {
    warp_a[w] = holes;
    warp_b[w] = tails;
  }
  __syncthreads();
  if (w == 0) {
    const int x = sum_before(warp_a, NW, lane), y = sum_before(warp_b, NW, lane);
    if (lane == 0) sh_counts[0] = x, sh_counts[1] = y;
  }
  sync_all();
  const int their_holes = of_all(&sh_counts[0]), their_tails = of_all(&sh_counts[1]);
  const int all = __reduce_add_sync(~0u, their_holes);
  int at_hole = __reduce_add_sync(~0u, lane < rank ? their_holes : 0) + sum_before(warp_a, w, lane);
  int at_tail = __reduce_add_sync(~0u, lane < rank ? their_tails : 0) + sum_before(warp_b, w, lane);
  seen = ties;
  const MoveList list(c, c.list_by_slot, b, h);
  for (int g = g0; g < g0 + per; ++g) {
    bool hole, tail;
    classify(g, seen, hole, tail);
    const uint32_t m = __ballot_sync(~0u, hole), m2 = __ballot_sync(~0u, tail);
    if (hole) *list.at(at_hole + __popc(m & below)) = first + g * 32 + lane;
    if (tail) *list.at(budget + at_tail + __popc(m2 & below)) = first + g * 32 + lane;
    at_hole += __popc(m);
    at_tail += __popc(m2);
  }
  if (tid == 0 && rank == 0) c.moves[pair] = make_int2(all, budget);
  sync_all();  // the lists are written; and nobody leaves while others look at its shared memory
  if (!move_here) return;
  for (int m = rank * NW + w; m < all; m += ctas * NW)
    move_row(c, c.list_by_slot, b, h, *list.at(budget + m), *list.at(m), lane);
  cut_count();
}

// (At most 32 registers: with 40 the moves of 8 pairs of 65536 rows cut to 8192 take 18 us, not 15.)
// One warp per move.  Sources lie at or above the budget and targets below it, so no
// move reads what another writes.
template <bool BY_SLOT>
__global__ void __launch_bounds__(kMoveThreads, 8) evict_move_kernel(const __grid_constant__ Pages c) {
  pdl_wait();
  pdl_launch_dependents();
  const int b = blockIdx.x / c.heads, h = blockIdx.x - b * c.heads;
  const int n = c.moves[blockIdx.x].x;
  if (n < 0) return;
  const int left = c.moves[blockIdx.x].y;
  const MoveList list(c, BY_SLOT, b, h);
  for (int m = blockIdx.y * (kMoveThreads / 32) + (threadIdx.x >> 5); m < n; m += gridDim.y * (kMoveThreads / 32))
    move_row(c, BY_SLOT, b, h, *list.at(left + m), *list.at(m), threadIdx.x & 31);
  if (h == 0 && blockIdx.y == 0 && threadIdx.x == 0) c.counts[b] = left;
}

template <class T, int V, int VC, bool ROT>
int append_run(const Pages& c, AppendParams p, cudaStream_t stream) {
  p.turned = ROT ? rotary_units<V>(p.rotary, p.interleaved) : 0;
  p.units = p.turned + (c.dim - p.rotary) / V;
  p.lanes = std::min(p.units, kAppendThreads);
  p.row_units = c.dim / VC;
  p.row_lanes = std::min(p.row_units, kAppendThreads);
  p.by_qk = FastDiv(p.q_heads + c.heads);
  p.by_heads = FastDiv(c.heads);
  p.by_pairs = FastDiv(std::max(1, p.rotary / 2));
  // A few batches of loads for a CTA, but for tokens enough to fill the SMs.
  const int fill = 16 * (kAppendThreads / p.lanes) / (p.q_heads + c.heads);
  p.per_cta = std::max(1, std::min({fill, p.tokens / (4 * kSMs), 40}));  // 40 x (1 KB + 32) of shared memory at most
  return launch_pdl(append_kernel<T, V, VC, ROT>, dim3((p.tokens + p.per_cta - 1) / p.per_cta), dim3(kAppendThreads),
                    p.per_cta * (sizeof(TokenRow) + (size_t)(p.rotary / 2) * sizeof(float2)), stream, pdl_enabled(), c,
                    p);
}

// The turned rows take the widest word that fits them; the copied ones (v, and k without rotation)
// 16 bytes, or single values where that does not fit.
template <class T, int V>
int append_rotated(const Pages& c, const AppendParams& p, bool rows, cudaStream_t stream) {
  return rows ? append_run<T, V, 8, true>(c, p, stream) : append_run<T, V, 1, true>(c, p, stream);
}

template <class T>
int append_type(const Pages& c, const AppendParams& p, cudaStream_t stream) {
  if (p.rotary == 0) {
    const bool rows = unit_values(2, 0, false, c.dim, {p.vt, p.vh, p.kt, p.kh}, p.v, p.k) == 8;
    return rows ? append_run<T, 8, 8, false>(c, p, stream) : append_run<T, 1, 1, false>(c, p, stream);
  }
  const bool rows = unit_values(2, 0, false, c.dim, {p.vt, p.vh}, p.v) == 8;
  switch (unit_values(2, p.rotary, p.interleaved, c.dim, {p.kt, p.kh, p.qt, p.qh}, p.k, p.q, p.q_out)) {
    case 8: return append_rotated<T, 8>(c, p, rows, stream);
    case 4: return append_rotated<T, 4>(c, p, rows, stream);
    case 2: return append_rotated<T, 2>(c, p, rows, stream);
    default: return append_rotated<T, 1>(c, p, rows, stream);
  }
}

}  // namespace
}  // namespace pi05

using namespace pi05;

extern "C" {

size_t pi05_paged_workspace_bytes(const Pi05PagedCache* cache) {
  if (cache == nullptr || cache->batch <= 0 || cache->n_kv_heads <= 0 || cache->pages_per_seq <= 0 ||
      cache->page_size <= 0)
    return 0;
  return (kWsAccumOffset + paged_moves_bytes(cache) + 255) & ~size_t(255);
}

int pi05_paged_append(const Pi05PagedCache* cache, const Pi05PagedAppend* a, void* stream) {
  Pages c;
  int rc = paged_check(cache, "paged_append", &c);
  if (rc) return rc;
  if (a == nullptr || (a->tokens > 0 && (a->k == nullptr || a->v == nullptr)) ||
      (a->q != nullptr && a->q_out == nullptr)) {
    set_last_error("paged_append: null pointer");
    return PI05_ERR_INVALID_ARG;
  }
  const Pi05Rotary* rot = a->rotary;
  if (rot == nullptr && a->q != nullptr) {
    set_last_error("paged_append: q without rotary has nothing to do");
    return PI05_ERR_INVALID_ARG;
  }
  if (rot != nullptr && (rot->turns == nullptr || rot->rotary_dim <= 0 || rot->rotary_dim % 2 ||
                         rot->rotary_dim > c.dim)) {
    set_last_error("paged_append: bad rotary_dim %d for head_dim %d", rot->rotary_dim, c.dim);
    return PI05_ERR_SHAPE;
  }
  if (a->tokens < 0 || (a->q != nullptr && (a->n_q_heads <= 0 || (long long)a->n_q_heads * c.dim > (1 << 24))) ||
      (a->cu_tokens == nullptr && a->tokens != c.batch)) {
    set_last_error("paged_append: bad shape tokens=%d n_q_heads=%d batch=%d", a->tokens, a->n_q_heads, c.batch);
    return PI05_ERR_SHAPE;
  }
  if (a->new_weight != nullptr && c.weight == nullptr) {
    set_last_error("paged_append: the cache keeps no weights");
    return PI05_ERR_INVALID_ARG;
  }
  if (!aligned_to(2, a->k, a->v, a->q, a->q_out) || !aligned_to(4, a->cu_tokens, a->new_weight) ||
      (rot != nullptr && !aligned_to(8, rot->turns))) {
    set_last_error("paged_append: pointer not aligned to its elements");
    return PI05_ERR_ALIGN;
  }
  const long long kt = stride_of(a->tokens, a->k_token_stride), kh = stride_of(c.heads, a->k_head_stride);
  const long long vt = stride_of(a->tokens, a->v_token_stride), vh = stride_of(c.heads, a->v_head_stride);
  const bool q = a->q != nullptr;
  const long long qt = q ? stride_of(a->tokens, a->q_token_stride) : 0;
  const long long qh = q ? stride_of(a->n_q_heads, a->q_head_stride) : 0;
  for (long long stride : {kt, kh, vt, vh, qt, qh})
    if (stride < 0 || stride >= 1ll << 31) {
      set_last_error("paged_append: stride of %lld elements", stride);
      return PI05_ERR_SHAPE;
    }
  if (a->tokens == 0) return PI05_OK;
  AppendParams p;
  p.k = a->k;
  p.v = a->v;
  p.q = a->q;
  p.q_out = a->q_out;
  p.kt = (int)kt;
  p.kh = (int)kh;
  p.vt = (int)vt;
  p.vh = (int)vh;
  p.qt = (int)qt;
  p.qh = (int)qh;
  p.cu = a->cu_tokens;
  p.new_weight = a->new_weight;
  p.turns = rot ? rot->turns : nullptr;
  p.tokens = a->tokens;
  p.q_heads = q ? a->n_q_heads : 0;
  p.rotary = rot ? rot->rotary_dim : 0;
  p.interleaved = rot ? rot->interleaved : 0;
  p.magnitude = rot ? rot->magnitude : 1.f;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return cache->dtype == PI05_BF16 ? append_type<__nv_bfloat16>(c, p, st) : append_type<__half>(c, p, st);
}

int pi05_paged_evict(const Pi05PagedCache* cache, int budget, int recent, int sinks, void* stream) {
  Pages c;
  int rc = paged_check(cache, "paged_evict", &c);
  if (rc) return rc;
  if (c.weight == nullptr || c.pos == nullptr) {
    set_last_error("paged_evict: the cache keeps no weights or positions");
    return PI05_ERR_INVALID_ARG;
  }
  if (budget < 1 || recent < 0 || sinks < 0 || (long long)recent + sinks > budget) {
    set_last_error("paged_evict: need budget >= 1 and 0 <= recent + sinks <= budget (budget=%d recent=%d sinks=%d)",
                   budget, recent, sinks);
    return PI05_ERR_SHAPE;
  }
  if (budget >= c.capacity) return PI05_OK;  // no sequence can hold more
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int pairs = c.batch * c.heads;
  // CTAs of a pair: up to 8 while they hold 4096 rows each and find an SM of their own.  A
  // cluster's barriers cost more than they share out for fewer: 8 pairs of 3712 rows take
  // 11 us in one CTA each and 13 in four; 8 pairs of 65536 take 42 in four and 33 in eight.
  int ctas = 1;
  while (ctas < 8 && pairs * ctas * 2 <= kSMs && c.capacity / (ctas * 2) >= 4096) ctas *= 2;
  const int share = ((c.capacity + ctas - 1) / ctas + 31) & ~31, held = std::min(share, kMaxKeys);
  const int most = std::min(budget, c.capacity - budget);  // moves of a pair
  const int move_here = most <= 64 * ctas;
  const size_t smem = (size_t)held * sizeof(uint32_t);
  // A pass over the buckets costs every thread the same: 512 pairs of 2080 rows take 10 us
  // with 256 threads each and 14 with 512; where the CTAs have an SM each, 8 pairs of 3712
  // rows take 16 and 11.
  const int threads = share <= 4096 && pairs * ctas > kSMs ? 256 : 512;
  const int which = held < share ? 2 : threads == 256 ? 0 : 1;
  auto kernel = which == 2   ? evict_select_kernel<512, false>
                : which == 0 ? evict_select_kernel<256, true>
                             : evict_select_kernel<512, true>;
  static std::atomic<uint64_t> allowed[3];
  if (smem > 24 * 1024 && (rc = allow_smem(kernel, kMaxKeys * 4, &allowed[which], "paged_evict"))) return rc;
  rc = launch_pdl_cluster(kernel, dim3(pairs * ctas), dim3(threads), smem, st, pdl_enabled(), dim3(ctas), c, budget,
                          recent, sinks, ctas, held, move_here);
  if (rc || move_here) return rc;
  const int chunks = std::min((most + kMoveThreads / 32 - 1) / (kMoveThreads / 32), std::max(1, kSMs * 16 / pairs));
  return launch_pdl(c.list_by_slot ? evict_move_kernel<true> : evict_move_kernel<false>, dim3(pairs, chunks),
                    dim3(kMoveThreads), 0, st, pdl_enabled(), c);
}

}  // extern "C"
