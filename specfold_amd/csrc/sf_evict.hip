// Eviction from the prefix cache by accumulated attention weight (sf_kv_evict).  No
// counterpart in the reference, whose cache only grows.
//
// Of the P keys of a (layer, kv head): the first `sinks`, the last `recent` and the
// k = keep - sinks - recent others with the largest mass, equal ones by the lower index.
//  * select: one workgroup per (layer, kv head).  The masses are mapped to unsigned
//    integers of the same order and stay in registers; the k-th largest value is built
//    eight bits at a time from the top: a histogram in LDS of the digit of the keys that
//    agree so far (integer counts, whatever their order; one copy: four, a lane in its
//    own, gained nothing), which every wave sums from the top for itself, so a step has
//    one barrier.  It ends as soon as just the keys that are needed are left.  Two ballot
//    scans number the ties and the kept keys in index order.  (Two bits a step by counting
//    with ballots, no histogram: 56 lists of 1056 keys with their copy 33 us, 25 so; 320
//    of 16384 542 and 524.)  Bound by its latencies: 7.5 us for 56 lists of 1056 or 112 of
//    4095 keys, 41 for 320 of 16384.
//  * move: the kept rows to slots 0 .. keep - 1, ascending, bound by reading and writing
//    them once (2.7 GB at 5.7 TB/s, 115 MB at 5.2).  Into another cache every 128 rows are
//    a workgroup's.  In place slot j takes a row from a slot >= j, so a workgroup goes up
//    the slots of its (layer, kv head) alone: a tile is written when all of its rows have
//    been read, and the rows of the tile behind it, which no write of this one reaches,
//    are on their way.
#include "sf_common.h"

namespace {

constexpr int kHD = 128;
constexpr int kMaxKeys = 32768;
constexpr int kSelThreads = 1024;
constexpr int kSelWaves = kSelThreads / 64;
constexpr int kSteps = 4;    // of 8 bits

// The order of a float as an unsigned integer: NaN above all, -0 as 0.
SF_DEV uint32_t order_of(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t u = __float_as_uint(x + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

template <int PER>   // keys of a thread: t = i * 1024 + tid
__global__ __launch_bounds__(kSelThreads) void sf_evict_select_kernel(
    const float* mass, long long mass_layer, long long mass_head, int Hkv, int P, int sinks,
    int recent, int keep, int32_t* __restrict__ kept, float* mass_out, long long out_layer,
    long long out_head, int zero_to, int32_t* length_dev, int32_t* position_dev, int position) {
  __shared__ sf_u32x4 s_hist[kSteps * 64];
  __shared__ int s_cnt[PER * kSelWaves];
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  const int l = blockIdx.x / Hkv, h = blockIdx.x - l * Hkv;
  if (blockIdx.x == 0 && tid == 0) {   // (two launches fewer for who keeps them)
    if (length_dev) *length_dev = keep;
    if (position_dev) *position_dev = position;
  }
  const float* in = mass + l * mass_layer + h * mass_head;
  const int last = P - recent;
  uint32_t key[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int t = i * kSelThreads + tid;
    // only the keys in between compete
    key[i] = t >= sinks && t < last ? order_of(in[t]) : 0u;
  }
  const int need = keep - sinks - recent;   // <= last - sinks
  // thr: the need-th largest, or (exact) a bound that just the `need` largest reach
  uint32_t thr = 0;
  int ties = need;   // of the keys that agree with thr in the digits found: how many stay
  bool exact = false;
  if (need > 0) {
    for (int i = tid; i < kSteps * 64; i += kSelThreads)
      s_hist[i] = sf_u32x4{0u, 0u, 0u, 0u};
    __syncthreads();
#pragma unroll 1
    for (int sh = 24; sh >= 0 && !exact; sh -= 8) {   // workgroup-uniform
      int* hist = reinterpret_cast<int*>(s_hist) + (sh >> 3) * 256;
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (key[i] != 0u && ((key[i] ^ thr) >> sh) < 256u)
          atomicAdd(&hist[key[i] >> sh & 255u], 1);
      __syncthreads();
      // every wave: lane x has the digits 4x .. 4x + 3, at[d] counts them and those above
      const sf_u32x4 w = reinterpret_cast<const sf_u32x4*>(hist)[lane];
      int n[4], at[4], sum = 0;
#pragma unroll
      for (int d = 3; d >= 0; --d) {
        n[d] = (int)w[d];
        sum += n[d];
        at[d] = sum;
      }
      int up = sum;
#pragma unroll
      for (int o = 1; o <= 32; o <<= 1) {
        const int t = __shfl(up, lane + o < 64 ? lane + o : lane, 64);
        up += lane + o < 64 ? t : 0;
      }
      up -= sum;
      // the digit: the largest with `ties` keys at or above it
      int mine = -1, over = 0, in_it = 0;
#pragma unroll
      for (int d = 0; d < 4; ++d)
        if (at[d] + up >= ties) mine = d, over = at[d] + up - n[d], in_it = n[d];
      const int top = __popcll(__ballot(mine >= 0)) - 1;   // (lanes 0 .. top)
      thr |= (uint32_t)(4 * top + __shfl(mine, top, 64)) << sh;
      ties -= __shfl(over, top, 64);
      exact = __shfl(in_it, top, 64) == ties;
    }
  }
  uint32_t keeps = 0, equal = 0;   // bit i: key i of this thread
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int t = i * kSelThreads + tid;
    const bool mid = t >= sinks && t < last;
    const bool in_it = mid & (need > 0);
    const bool over = in_it & (exact ? key[i] >= thr : key[i] > thr);
    if (t < P && (!mid || over)) keeps |= 1u << i;
    if (in_it && !exact && key[i] == thr) equal |= 1u << i;
  }
  // index-order numbering of the flagged keys: s_cnt holds, for each 64 of them, how
  // many are flagged in front
  auto scan = [&](uint32_t bits) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const unsigned long long b = __ballot(bits >> i & 1u);
      if (lane == 0) s_cnt[i * kSelWaves + wv] = __popcll(b);
    }
    __syncthreads();
    if (wv == 0) {   // lane x: entries x PER / 4 ..
      constexpr int kE = PER / 4;
      int e[kE], sum = 0;
#pragma unroll
      for (int i = 0; i < kE; ++i) {
        e[i] = sum;
        sum += s_cnt[lane * kE + i];
      }
      int at = sum;
#pragma unroll
      for (int o = 1; o <= 32; o <<= 1) {
        const int up = __shfl(at, lane >= o ? lane - o : lane, 64);
        at += lane >= o ? up : 0;
      }
      at -= sum;
#pragma unroll
      for (int i = 0; i < kE; ++i) s_cnt[lane * kE + i] = at + e[i];
    }
    __syncthreads();
  };
  const unsigned long long below = (1ull << lane) - 1;
  if (need > 0 && !exact) {   // of the equal ones the first
    scan(equal);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const unsigned long long b = __ballot(equal >> i & 1u);
      const int rank = s_cnt[i * kSelWaves + wv] + __popcll(b & below);
      if ((equal >> i & 1u) && rank < ties) keeps |= 1u << i;
    }
  }
  scan(keeps);
  int32_t* kp = kept + (size_t)blockIdx.x * keep;
  float* mo = mass_out ? mass_out + l * out_layer + h * out_head : nullptr;
  // the masses again (in place they are all read before the first is written)
  float val[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) val[i] = mo && (keeps >> i & 1u) ? in[i * kSelThreads + tid] : 0.f;
#pragma unroll
  for (int i = 0; i < PER; ++i) sf_pin(val[i]);
  sf_wait_vm_loads();
  __syncthreads();
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int t = i * kSelThreads + tid;
    const unsigned long long b = __ballot(keeps >> i & 1u);
    if (keeps >> i & 1u) {
      const int rank = s_cnt[i * kSelWaves + wv] + __popcll(b & below);
      kp[rank] = t;
      if (mo) mo[rank] = val[i];
    }
    if (mo && t >= keep && t < zero_to) mo[t] = 0.f;
  }
}

struct Pages {
  uint16_t* base;
  const int32_t* table;
  long long layer_stride, page_stride, head_stride;
  int page_size, pages;
};
SF_DEV long long slot_off(const Pages& p, int l, int h, int t, bool& ok) {
  const int lp = t / p.page_size;
  const int id = p.table[lp];
  ok = id >= 0 && id < p.pages;
  return l * p.layer_stride + (ok ? id : 0) * p.page_stride + h * p.head_stride +
         (long long)(t - lp * p.page_size) * kHD;
}

constexpr int kMoveThreads = 256;
constexpr int kMoveRows = 8;   // 16-byte units of a thread in a tile

// Into another cache: 16 threads a row, 128 rows a workgroup.
__global__ __launch_bounds__(kMoveThreads) void sf_evict_copy_kernel(
    Pages fk, Pages fv, Pages tk, Pages tv, const int32_t* __restrict__ kept, int Hkv, int keep) {
  const int tiles = (keep + 16 * kMoveRows - 1) / (16 * kMoveRows);
  const int lh = blockIdx.x / tiles, j0 = (blockIdx.x - lh * tiles) * 16 * kMoveRows;
  const int l = lh / Hkv, h = lh - l * Hkv;
  const Pages from = blockIdx.y ? fv : fk, to = blockIdx.y ? tv : tk;
  const int32_t* kp = kept + (size_t)lh * keep;
  const int unit = threadIdx.x & 15, r = j0 + (threadIdx.x >> 4);
  sf_u32x4 w[kMoveRows];
#pragma unroll
  for (int i = 0; i < kMoveRows; ++i) {
    bool ok;
    const long long at = slot_off(from, l, h, kp[min(r + 16 * i, keep - 1)], ok);
    w[i] = sf_stream_load16(from.base + at + unit * 8);
  }
#pragma unroll
  for (int i = 0; i < kMoveRows; ++i) {
    bool ok;
    const long long at = slot_off(to, l, h, min(r + 16 * i, keep - 1), ok);
    if (r + 16 * i < keep && ok)
      sf_handoff_store(reinterpret_cast<sf_u32x4*>(to.base + at + unit * 8), w[i]);
  }
}

// In place: 8 threads a half row (64 dims), 256 rows a tile; blockIdx.y: K or V, its half.
__global__ __launch_bounds__(kMoveThreads) void sf_evict_move_kernel(
    Pages pk, Pages pv, const int32_t* __restrict__ kept, int Hkv, int keep) {
  constexpr int kTile = 32 * kMoveRows;
  const int l = blockIdx.x / Hkv, h = blockIdx.x - l * Hkv;
  const Pages pg = blockIdx.y >> 1 ? pv : pk;
  const int32_t* kp = kept + (size_t)blockIdx.x * keep;
  const int dim = 64 * (blockIdx.y & 1) + 8 * (threadIdx.x & 7), r = threadIdx.x >> 3;
  sf_u32x4 cur[kMoveRows], next[kMoveRows];
  auto load = [&](int j0, sf_u32x4 (&w)[kMoveRows]) {
#pragma unroll
    for (int i = 0; i < kMoveRows; ++i) {
      bool ok;
      const long long at = slot_off(pg, l, h, kp[min(j0 + 32 * i + r, keep - 1)], ok);
      w[i] = *reinterpret_cast<const sf_u32x4*>(pg.base + at + dim);
    }
  };
  auto store = [&](int j0, sf_u32x4 (&w)[kMoveRows]) {
#pragma unroll
    for (int i = 0; i < kMoveRows; ++i) sf_pin(w[i]);   // (this thread's rows of the tile are here)
    __syncthreads();                                    // and everyone's
#pragma unroll
    for (int i = 0; i < kMoveRows; ++i) {
      const int j = j0 + 32 * i + r;
      bool ok;
      const long long at = slot_off(pg, l, h, min(j, keep - 1), ok);
      if (j < keep && ok) *reinterpret_cast<sf_u32x4*>(pg.base + at + dim) = w[i];
    }
  };
  load(0, cur);
  for (int j0 = 0; j0 < keep; j0 += 2 * kTile) {   // (tiles past the end: nothing is written)
    load(j0 + kTile, next);
    store(j0, cur);
    load(j0 + 2 * kTile, cur);
    store(j0 + kTile, next);
  }
}

int check_pages(const sf_kv_pages* p, int keys) {
  if (!p || !p->k || !p->v || !p->page_table) return SF_ERR_ARG;
  if (reinterpret_cast<uintptr_t>(p->k) % 16 || reinterpret_cast<uintptr_t>(p->v) % 16)
    return SF_ERR_ARG;
  if (p->page_size != 16 && p->page_size != 32 && p->page_size != 64 && p->page_size != 128)
    return SF_ERR_SHAPE;
  if (p->pages < 1 || (long long)p->pages * p->page_size < keys) return SF_ERR_SHAPE;
  if (p->layer_stride % 8 || p->page_stride % 8 || p->head_stride % 8) return SF_ERR_SHAPE;
  return SF_OK;
}

}  // namespace

extern "C" int sf_kv_evict(const float* mass, long long mass_layer, long long mass_head,
                           int layers, int Hkv, int hd, int P, int sinks, int recent, int keep,
                           const sf_kv_pages* from, const sf_kv_pages* to, int32_t* kept,
                           float* mass_out, long long mass_out_layer, long long mass_out_head,
                           int32_t* length_dev, int32_t* position_dev, int position,
                           void* stream) {
  if (!mass || !kept) return SF_ERR_ARG;
  if (hd != kHD || layers < 1 || Hkv < 1 || P < 1 || P > kMaxKeys) return SF_ERR_SHAPE;
  if (keep < 1 || keep > P || sinks < 0 || recent < 0 || sinks > keep || recent > keep - sinks)
    return SF_ERR_SHAPE;
  int st = check_pages(from, P);
  if (st == SF_OK) st = check_pages(to, keep);
  if (st != SF_OK) return st;
  if (mass_out == mass && (mass_out_layer != mass_layer || mass_out_head != mass_head))
    return SF_ERR_ARG;
  if (mass_out) {   // its rows must not overlap
    const long long n = mass_out == mass ? P : keep;
    const bool heads_inside = Hkv == 1 || layers == 1 || mass_out_head <= mass_out_layer;
    const long long head_span = Hkv > 1 ? mass_out_head * (Hkv - 1) : 0;
    const long long layer_span = layers > 1 ? mass_out_layer * (layers - 1) : 0;
    if (Hkv > 1 && mass_out_head < n + (heads_inside ? 0 : layer_span)) return SF_ERR_SHAPE;
    if (layers > 1 && mass_out_layer < n + (heads_inside ? head_span : 0)) return SF_ERR_SHAPE;
  }
  // the same pool through the same table: the same mapping, in place
  const bool in_place = from->k == to->k && from->page_table == to->page_table;
  if (in_place && (from->v != to->v || from->layer_stride != to->layer_stride ||
                   from->page_stride != to->page_stride || from->head_stride != to->head_stride ||
                   from->page_size != to->page_size))
    return SF_ERR_ARG;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
#define SF_EVICT_SELECT(PER)                                                                    \
  hipLaunchKernelGGL((sf_evict_select_kernel<PER>), dim3(layers * Hkv), dim3(kSelThreads), 0, s, \
                     mass, mass_layer, mass_head, Hkv, P, sinks, recent, keep, kept, mass_out,   \
                     mass_out_layer, mass_out_head, mass_out == mass ? P : 0, length_dev,        \
                     position_dev, position)
  if (P <= 4 * kSelThreads) SF_EVICT_SELECT(4);
  else if (P <= 16 * kSelThreads) SF_EVICT_SELECT(16);
  else SF_EVICT_SELECT(32);
#undef SF_EVICT_SELECT
  auto pages = [](const sf_kv_pages* p, uint16_t* base) {
    return Pages{base, p->page_table, p->layer_stride, p->page_stride, p->head_stride,
                 p->page_size, p->pages};
  };
  if (in_place) {
    hipLaunchKernelGGL(sf_evict_move_kernel, dim3(layers * Hkv, 4), dim3(kMoveThreads), 0, s,
                       pages(to, to->k), pages(to, to->v), kept, Hkv, keep);
  } else {
    const int tiles = (keep + 16 * kMoveRows - 1) / (16 * kMoveRows);
    hipLaunchKernelGGL(sf_evict_copy_kernel, dim3(layers * Hkv * tiles, 2), dim3(kMoveThreads), 0,
                       s, pages(from, from->k), pages(from, from->v), pages(to, to->k),
                       pages(to, to->v), kept, Hkv, keep);
  }
  return sf_launch_status();
}
