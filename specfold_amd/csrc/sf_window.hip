// Attention of new rows over paged caches with a sliding window and sinks, several
// sequences in one call (sf_attn_window), and the weight each cached key got from those
// rows (sf_attn_key_mass).  No counterpart in the reference.
//
// Row m of a sequence (n rows, P cached keys, its own the last n of them) is at position
// p = P - n + m and sees the keys t < end(m) = P - n + min(n, (m / block + 1) * block)
// with t < sinks or t > p - window (window 0: all).  o = softmax(scaling q.k) v,
// lse = ln sum exp(scaling q.k); mass[t] += exp(scaling q.k - lse).
//
// Attention.  The queries of a (sequence, kv head) are its rows x the G q-heads, qi =
// m * G + g, cut into tiles; a tile walks the 32-key stages that its rows see, running
// maximum and sum per query, and skips the stages between the sinks and the window.
// Scores are formed transposed, S^T = K Q^T (v_mfma_f32_32x32x16_bf16, K the A operand),
// so a lane holds 16 of a stage's keys for ONE query (lane % 32) and the softmax is in
// the lane; registers 8kk .. 8kk + 7 of S^T are the B operand of O^T += V^T P^T for the
// keys 16kk + {8 (e / 4) + 4 (lane / 32) + e % 4} without a shuffle, and V^T comes in
// the same key order from row-major V by transposing LDS reads.
#include <math.h>

#include "sf_common.h"
#include "sf_index.h"

namespace {

using namespace sfw;

constexpr int kHD = 128;
constexpr int kMaxSeqs = 32;
constexpr int kMaxKeys = 32768;
constexpr int kMaxG = 16;
constexpr int kMaxH = 256;   // (a sequence's rows of q: 32-bit byte offsets)
constexpr int kThreads = 256;
constexpr int kCUs = 256;
constexpr int kTileQ = 128;   // queries of a tile
// Few queries: tiles of 9 to 36 stages go to eight waves and one range, if there are no more
// of them than CUs (a workgroup's LDS fills one).
constexpr int kWideLeast = 9, kWideMost = 36;
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;
constexpr float kLazy = 8.f;   // base-2 headroom of the softmax reference

typedef float sf_f32x16 __attribute__((ext_vector_type(16)));

SF_DEV sf_f32x16 mfma32(const sf_bf16x8 a, const sf_bf16x8 b, const sf_f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

template <int N>
struct Int {
  static constexpr int value = N;
};

// Lane i's value of v (i wave-uniform), and a wait for all but the N youngest vector
// memory operations of this wave without a workgroup barrier (the wave's lanes are
// through with what they did before).  Elsewhere than on the GPU the wave's lanes are
// only kept in step.
#if defined(__HIPCC__)
SF_DEV int lane_value(int v, int i) { return __builtin_amdgcn_readlane(v, i); }
template <int N>
SF_DEV void wait_vm_wave() {
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4));   // lgkmcnt(0) too
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
}
#else
inline int lane_value(int v, int i) { return __shfl(v, i, 64); }
template <int N>
inline void wait_vm_wave() { (void)__builtin_amdgcn_readfirstlane(0); }
#endif

struct Seq {
  const uint16_t* k;
  const uint16_t* v;
  const int32_t* table;
  long long page_stride, head_stride;
  int length, rows, row0, pages;
  int tile0, tiles;        // of the launch this sequence belongs to (0 tiles: of another)
};
struct Call {
  Seq s[kMaxSeqs];
  int n_seqs, page_shift, block, window, sinks, H, Hkv, rows;
  int tiles, nr, spr;      // tiles of all sequences, ranges of a tile, stages of a range
  int longest;             // stages of the longest tile
};

SF_DEV int page_in(const Seq& s, int id) { return id >= 0 && id < s.pages ? id : 0; }
SF_DEV int page_of(const Seq& s, int page_shift, int key) {
  return page_in(s, s.table[key >> page_shift]);
}

// ---- LDS stages ------------------------------------------------------------------------
// 32 keys: K rows of 256 bytes, then V rows; 16-byte unit u of row r at unit u ^ (r & 15)
// (K: the 16-row operand reads hit 16 different units) and u ^ 2 (r & 7) (V: the
// transposing reads take four consecutive rows x 64 bytes).
constexpr int kRowBytes = 2 * kHD;
constexpr int kHalf = kStage * kRowBytes;    // K rows of a stage
constexpr int kSlot = 2 * kHalf;             // 16 KB

// This lane's byte offsets in a slot: K operand (key lane % 32, dims 16ks + 8 (lane / 32)
// .. + 8) and V^T operand of dim tile dt (32 dims, keys 4 (lane / 32) + {0..3}; the next
// 8 keys 8 rows on).
SF_DEV uint32_t k_off(int lane, int ks) {
  const int r = lane & 31, u = 2 * ks + (lane >> 5);
  return (uint32_t)(r * kRowBytes + (u ^ (r & 15)) * 16);
}
SF_DEV uint32_t v_off(int lane, int dt) {
  const int r = 4 * (lane >> 5) + ((lane & 15) >> 2);
  const int u = 4 * dt + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
  return (uint32_t)(kHalf + r * kRowBytes + (u ^ (2 * (r & 7))) * 16 + (lane & 1) * 8);
}

// Element offset of the 16-key group that starts at key g0 from its kv head's first row; id:
// the page table's entry of the group.
SF_DEV long long group_off(const Seq& s, int page_shift, int id, int g0) {
  if (!s.table) return (long long)g0 * kHD;
  return page_in(s, id) * s.page_stride + (long long)(g0 & ((1 << page_shift) - 1)) * kHD;
}
// The offsets of 64 groups, one a lane; lane i's as a wave-uniform value.
struct Groups {
  int lo, hi;
  SF_DEV void set(long long off) {
    lo = (int)(uint32_t)off;
    hi = (int)(off >> 32);
  }
  SF_DEV long long at(int i) const {
    return (long long)((unsigned long long)(uint32_t)lane_value(hi, i) << 32 |
                       (uint32_t)lane_value(lo, i));
  }
};
// Copies 4 N rows of a group to a stage: off: copy i's element offset of this lane, its row
// (4i + lane / 16 of them) * kHD + copy_unit.
template <int N>
SF_DEV void copy_rows(const uint16_t* src, const uint32_t (&off)[N], uint8_t* dst) {
#pragma unroll
  for (int i = 0; i < N; ++i) sf_lds_dma16(src + off[i], dst + 4 * i * kRowBytes);
}
// the logical unit (in elements) that this lane's copy of rows r0 .. + 4 brings
SF_DEV int copy_unit(int lane, int r0, bool is_v) {
  const int r = r0 + (lane >> 4), p = lane & 15;
  return (is_v ? p ^ (2 * (r & 7)) : p ^ (r & 15)) * 8;
}

// copy_rows' offset of this lane for rows r0 .. + 4, rows behind `last` repeating it
SF_DEV uint32_t copy_off(int lane, int r0, bool is_v, int last) {
  return (uint32_t)(min(r0 + (lane >> 4), last) * kHD + copy_unit(lane, r0, is_v));
}

SF_DEV int last_group(int P) { return (P - 1) & ~15; }

// p[.] of one query of a stage (16 keys a lane) -> the two B operands
SF_DEV void pack_p(const float (&p)[16], sf_u32x4 (&pb)[2]) {
#pragma unroll
  for (int kk = 0; kk < 2; ++kk)
#pragma unroll
    for (int w = 0; w < 4; ++w) pb[kk][w] = sf_pack2(p[8 * kk + 2 * w], p[8 * kk + 2 * w + 1]);
}

SF_DEV bool seen_key(int key, int end, int lo, int sinks) {   // (lo <= end)
  return ((unsigned)(key - lo) < (unsigned)(end - lo)) | ((key < sinks) & (key < end));
}
// The mask of a stage's scores for one query: keys at or behind `end`, and keys of
// [sinks, lo).
SF_DEV void mask_scores(sf_f32x16& s, int key0, int hf, int end, int lo, int sinks) {
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int key = key0 + 8 * (i >> 2) + 4 * hf + (i & 3);
    s[i] = seen_key(key, end, lo, sinks) ? s[i] : -INFINITY;
  }
}

// Queries q0 .. q0 + nw of an item a key at a time, for a wave whose masked stages held a
// value that is not finite: the weight of a hidden key is 0, but 0 * inf is not.  Lane: a
// key of 64 for the scores, two dims for the values.  One range is written to o and lse,
// of several the partial.
struct Out {
  uint16_t* o;
  float* lse;
  float* ws_o;
  float* ws_ml;
  float scale_log2;
};
SF_DEV void slow_queries(const uint16_t* q, const Call& c,
                                                       const Seq& s, int h, int r, int q0, int nw,
                                                       Keys keys, int c0, int nst, const Out& out) {
  const int lane = threadIdx.x & 63, G = c.H / c.Hkv;
  const long long head = (long long)h * s.head_stride;
  auto key_at = [&](int t) {
    return head + (s.table ? page_of(s, c.page_shift, t) * s.page_stride +
                                 (long long)(t & ((1 << c.page_shift) - 1)) * kHD
                           : (long long)t * kHD);
  };
  for (int qi = q0; qi < min(q0 + nw, s.rows * G); ++qi) {
    const int m = qi / G;
    const int end = row_end(m, s.rows, s.length, c.block);
    const int lo = row_lo(m, s.rows, s.length, c.window);
    const size_t rh = (size_t)(s.row0 + m) * c.H + h * G + (qi - m * G);
    float mx = -INFINITY, l = 0.f, a0 = 0.f, a1 = 0.f;
    for (int k = 0; k < nst; k += 2) {   // two stages: 64 keys
      const int kk = k + (lane >> 5);
      const int t = keys.key0(c0 + min(kk, nst - 1)) + (lane & 31);
      const bool see = kk < nst && t < end && (t < c.sinks || t >= lo);
      float x = -INFINITY;
      if (see) {
        const uint16_t* kr = s.k + key_at(t);
        x = 0.f;
        for (int d = 0; d < kHD; d += 8) {
          float a[8], b[8];
          sf_unpack8(*reinterpret_cast<const sf_u32x4*>(kr + d), a);
          sf_unpack8(*reinterpret_cast<const sf_u32x4*>(q + rh * kHD + d), b);
          for (int i = 0; i < 8; ++i) x = fmaf(a[i], b[i], x);
        }
        x *= out.scale_log2;
      }
      const float nm = fmaxf(mx, sf_wave_max(x));
      const float mu = nm == -INFINITY ? 0.f : nm;
      const float alpha = __builtin_amdgcn_exp2f(mx - mu);
      const float p = see ? __builtin_amdgcn_exp2f(x - mu) : 0.f;
      l = l * alpha + sf_wave_sum(p);
      a0 *= alpha;
      a1 *= alpha;
      mx = nm;
      for (unsigned long long bits = __ballot(see); bits; bits &= bits - 1) {
        const int j = __builtin_ctzll(bits);
        const float pj = __shfl(p, j, 64);
        const uint32_t w = *reinterpret_cast<const uint32_t*>(
            s.v + key_at(keys.key0(c0 + k + (j >> 5)) + (j & 31)) + 2 * lane);
        a0 = fmaf(pj, __uint_as_float(w << 16), a0);
        a1 = fmaf(pj, __uint_as_float(w & 0xffff0000u), a1);
      }
    }
    if (keys.nst <= c.spr) {
      *reinterpret_cast<uint32_t*>(out.o + rh * kHD + 2 * lane) = sf_pack2(a0 / l, a1 / l);
      if (out.lse && lane == 0) out.lse[rh] = mx * kLn2 + logf(l);
    } else {
      const size_t slot = (size_t)r * c.rows * c.H + rh;
      out.ws_o[slot * kHD + 2 * lane] = a0;
      out.ws_o[slot * kHD + 2 * lane + 1] = a1;
      if (lane == 0) out.ws_ml[2 * slot] = mx, out.ws_ml[2 * slot + 1] = l;
    }
  }
}

// Whether any of the wave's V^T operands has an exponent of all ones.
SF_DEV bool any_not_finite(const sf_u32x2 (&vf)[16]) {
  uint32_t t = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i)
    t |= ((vf[i][0] & 0x7f807f80u) + 0x00800080u) | ((vf[i][1] & 0x7f807f80u) + 0x00800080u);
  return __ballot((t & 0x80008000u) != 0) != 0;
}

// The V^T operands of a stage (dim tile dt, 16 keys kk, 8-key halves): vf[8kk + 2dt + r].
template <int OFF>
SF_DEV void read_v(const sf_lds_off (&va)[4], sf_u32x2 (&vf)[16]) {
#pragma unroll
  for (int dt = 0; dt < 4; ++dt) {
    vf[2 * dt] = sf_lds_read8_tr<OFF>(va[dt]);
    vf[2 * dt + 1] = sf_lds_read8_tr<OFF + 8 * kRowBytes>(va[dt]);
    vf[8 + 2 * dt] = sf_lds_read8_tr<OFF + 16 * kRowBytes>(va[dt]);
    vf[8 + 2 * dt + 1] = sf_lds_read8_tr<OFF + 24 * kRowBytes>(va[dt]);
  }
}
template <int OFF>
SF_DEV void read_k(const sf_lds_off (&ka)[8], sf_u32x4 (&kf)[8]) {
#pragma unroll
  for (int ks = 0; ks < 8; ++ks) kf[ks] = sf_lds_read16<OFF>(ka[ks]);
}
SF_DEV sf_bf16x8 v_operand(const sf_u32x2 (&vf)[16], int kk, int dt) {
  const sf_u32x2 a = vf[8 * kk + 2 * dt], b = vf[8 * kk + 2 * dt + 1];
  return sf_as_bf16x8(sf_u32x4{a[0], a[1], b[0], b[1]});
}

// One query's result: unnormalised o (registers 16dt' ..), reference m (base 2) and sum l.
SF_DEV void write_direct(const sf_f32x16 (&acc)[4], float m, float l, int hf, uint16_t* o,
                         float* lse) {
  const float inv = 1.0f / l;
#pragma unroll
  for (int dt = 0; dt < 4; ++dt)
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      sf_u32x2 w;
      w[0] = sf_pack2(acc[dt][4 * b] * inv, acc[dt][4 * b + 1] * inv);
      w[1] = sf_pack2(acc[dt][4 * b + 2] * inv, acc[dt][4 * b + 3] * inv);
      *reinterpret_cast<sf_u32x2*>(o + 32 * dt + 8 * b + 4 * hf) = w;
    }
  if (lse && hf == 0) *lse = m * kLn2 + logf(l);
}
SF_DEV void write_partial(const sf_f32x16 (&acc)[4], float m, float l, int hf, float* po,
                          float* pml) {
#pragma unroll
  for (int dt = 0; dt < 4; ++dt)
#pragma unroll
    for (int b = 0; b < 4; ++b)
      sf_handoff_store(reinterpret_cast<sf_f32x4*>(po + 32 * dt + 8 * b + 4 * hf),
                       sf_f32x4{acc[dt][4 * b], acc[dt][4 * b + 1], acc[dt][4 * b + 2],
                                acc[dt][4 * b + 3]});
  if (hf == 0) sf_handoff_store(reinterpret_cast<sf_f32x2*>(pml), sf_f32x2{m, l});
}

// Work item of block b: the kv head fastest (blocks go round robin over the 8 XCDs, so
// with 1, 2, 4 or 8 kv heads a head stays on its XCDs and their L2).  Then the sequences'
// tiles, the last tile of a sequence (the most keys) first, then the range: blocks of
// ranges that a tile does not have end at once, and stand behind those that work
// (INNER = false; 1494 causal rows of 12 / 2 heads: 67 us with the ranges inside, 53).
// Range r starts r tiles on, or with 4 kv heads and 16 tiles the even tiles, which have
// more ranges, would all be on the same XCDs and be more than these hold at once.
// INNER: the ranges of a tile side by side, for the few-query kernel (8 tokens over 8
// sequences of unlike lengths: 31 us, 38 with the ranges outside).
struct Item {
  int si, tile, r, h;
};
template <bool INNER>
SF_DEV Item find_item(const Call& c) {
  Item it;
  it.h = blockIdx.x % c.Hkv;
  const int rest = blockIdx.x / c.Hkv;
  it.r = INNER ? rest % c.nr : rest / c.tiles;
  const int tt = INNER ? rest / c.nr : (rest - it.r * c.tiles + it.r) % c.tiles;
  it.si = 0;
  while (tt >= c.s[it.si].tile0 + c.s[it.si].tiles) ++it.si;
  it.tile = c.s[it.si].tiles - 1 - (tt - c.s[it.si].tile0);
  return it;
}

// ---- tiles of 128 queries ------------------------------------------------------------------
// Four waves, wave w the queries 32 w .. + 32 of the tile, all walking the same stages
// through an LDS ring that direct copies fill three stages ahead (wave w: the 16-key group
// w & 1 of K or V).  The step of stage k runs three independent things side by side within
// the wave, the matrix core's and the vector ALU's: the softmax of stage k, O^T += V^T P^T
// of stage k - 1 and S^T of stage k + 1.  Two workgroups share a CU and drift apart, so
// that one's matrix products meet the other's loads; one workgroup of eight waves and 256
// queries, which copies half as much, measured 506 against 499 us on 8192 rows of 28 / 4
// heads and 175 against 150 on four shorter runs of rows.
// Bound by the matrix core and the vector ALU, 40 % of the cycles each and mostly in turn,
// and by the waits between them: 8192 rows of 28 / 4 heads over themselves 495 us (0.97
// PFLOP/s; a large library product 1.5), under a window of 2048 (40 / 8 heads) 350 us
// (0.87).  Copies issued between the parts of a step instead of together: 531 -> 507 us;
// exponentials pinned beside the products (the compiler sank them behind): 560 -> 505.
constexpr int kRing = 4;
constexpr int kAhead = kRing - 1;
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(2, 2))) void
sf_window_tile_kernel(const uint16_t* __restrict__ q, Call c, float scale_log2,
                      uint16_t* __restrict__ o, float* __restrict__ lse, float* __restrict__ ws_o,
                      float* __restrict__ ws_ml) {
  __shared__ __attribute__((aligned(16))) uint8_t ring[kRing * kSlot];
  const Item it = find_item<false>(c);
  const Seq& s = c.s[it.si];
  const int lane = threadIdx.x & 63, hf = lane >> 5;
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);   // wave-uniform
  const int G = c.H / c.Hkv, nq = s.rows * G, P = s.length;
  const Keys keys = query_tile_keys(it.tile, kTileQ, G, s.rows, P, c.block, c.window, c.sinks);
  const int c0 = it.r * c.spr;
  if (c0 >= keys.nst) return;
  const int nst = min(c.spr, keys.nst - c0);
  const int lastg = last_group(P);

  // lane i: 16-key group i & 1 of stage 32u + i / 2 of the range (past it: its last stage)
  auto lane_group = [&](int u) {
    return min(keys.key0(c0 + min(32 * u + (lane >> 1), nst - 1)) + 16 * (lane & 1), lastg);
  };
  // ... and the page table's entry of it
  auto load_pages = [&](int u) { return s.table ? s.table[lane_group(u) >> c.page_shift] : 0; };
  int pg_next = load_pages(0);
  const int q0 = it.tile * kTileQ + wv * 32;   // the wave's first query
  const int qi = min(q0 + (lane & 31), nq - 1);   // padding: the last query again
  const int m = qi / G;
  const int end = row_end(m, s.rows, P, c.block), lo = row_lo(m, s.rows, P, c.window);
  const size_t rh = (size_t)(s.row0 + m) * c.H + it.h * G + (qi - m * G);
  sf_u32x4 qf[8];
#pragma unroll
  for (int ks = 0; ks < 8; ++ks)
    qf[ks] = *reinterpret_cast<const sf_u32x4*>(q + rh * kHD + 8 * hf + 16 * ks);
  // stages whose keys every query of the wave sees need no mask
  const int end_min = row_end(min(q0, nq - 1) / G, s.rows, P, c.block);
  const int lo_max = row_lo(min(q0 + 31, nq - 1) / G, s.rows, P, c.window);
  sf_wait_vm_loads();
#pragma unroll
  for (int ks = 0; ks < 8; ++ks) sf_pin(qf[ks]);

  // copies: group wv & 1 of K (wv < 2) or V
  const int grp = wv & 1;
  const bool is_v = wv >= 2;
  const uint16_t* const base = (is_v ? s.v : s.k) + (long long)it.h * s.head_stride;
  // (off_last: of the last group of the cache, which may hold fewer than 16 keys)
  uint32_t off[4], off_last[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    off[i] = 2 * copy_off(lane, 4 * i, is_v, 15);   // (bytes)
    off_last[i] = 2 * copy_off(lane, 4 * i, is_v, P - 1 - lastg);
  }
  uint8_t* const dst = ring + (is_v ? kHalf : 0) + 16 * grp * kRowBytes;
  const int k_last = keys.stage_of(lastg - 16 * grp) - c0;   // from this stage on
  Groups groups;   // of the 32 stages being copied
  // The copies of a stage go out one at a time between the parts of a step: right behind
  // the barrier the sixteen of a workgroup queue up and hold their waves.
  const char* from = nullptr;   // the stage being copied
  uint8_t* to = dst;
  bool last = false;
  auto aim = [&](int k) {   // past the range: its last stage again
    if ((k & 31) == 0) {
      groups.set(group_off(s, c.page_shift, pg_next, lane_group(k >> 5)));
      pg_next = load_pages((k >> 5) + 1);
    }
    last = k >= k_last;   // wave-uniform
    from = reinterpret_cast<const char*>(base + groups.at(2 * (k & 31) + grp));
    to = dst + (k % kRing) * kSlot;
  };
  auto copy = [&](int i) {
    sf_lds_dma16(from + (last ? off_last[i] : off[i]), to + 4 * i * kRowBytes);
    __builtin_amdgcn_sched_barrier(0);
  };
#pragma unroll 1
  for (int k = 0; k < kAhead; ++k) {
    aim(k);
#pragma unroll
    for (int i = 0; i < 4; ++i) copy(i);
  }

  uint32_t koff[8], voff[4];
#pragma unroll
  for (int ks = 0; ks < 8; ++ks) koff[ks] = k_off(lane, ks);
#pragma unroll
  for (int dt = 0; dt < 4; ++dt) voff[dt] = v_off(lane, dt);

  // online softmax per query: acc and l_run are kept against the reference m_ref (-inf:
  // nothing yet; mu: m_ref, or 0), which moves up to a stage's maximum only when that
  // passes it by more than kLazy, so every exponential is at most 2^kLazy; l_run is per
  // lane (its own keys).
  float m_ref = -INFINITY, m_lim = -INFINITY, mu = 0.f, l_run = 0.f, alpha = 1.f;
  sf_f32x16 acc[4], sa, sb;
  sf_u32x2 vf[16];
  sf_u32x4 pa[2], pb[2];
  bool resc = false, bad = false;
#pragma unroll
  for (int dt = 0; dt < 4; ++dt)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[dt][i] = 0.f;
  pb[0] = pb[1] = sf_u32x4{0u, 0u, 0u, 0u};
#pragma unroll
  for (int i = 0; i < 16; ++i) vf[i] = sf_u32x2{0u, 0u};

  auto qk = [&](const sf_u32x4 (&kf)[8], sf_f32x16& out) {
#pragma unroll
    for (int i = 0; i < 16; ++i) out[i] = 0.f;
#pragma unroll
    for (int ks = 0; ks < 8; ++ks) out = mfma32(sf_as_bf16x8(kf[ks]), sf_as_bf16x8(qf[ks]), out);
  };

  // S^T of stage 0
  sf_wait_vm_barrier<(kAhead - 1) * 4>();
  {
    sf_lds_off ka[8];
#pragma unroll
    for (int ks = 0; ks < 8; ++ks) ka[ks] = sf_lds_addr(ring) + koff[ks];
    sf_u32x4 kf[8];
    read_k<0>(ka, kf);
    sf_lds_reads_done(kf);
    qk(kf, sa);
  }

  // stage k: its scores in sc, its P^T to pc; stage k - 1's V^T in vf and P^T in pp; stage
  // k + 1's scores to sn.  ka / va: LDS addresses of stage k + 1's K and of stage k's V but
  // for the constants OK / OV.
  auto step = [&](int k, sf_f32x16& sc, sf_f32x16& sn, const sf_u32x4 (&pp)[2],
                  sf_u32x4 (&pc)[2], const sf_lds_off (&ka)[8], auto OK, const sf_lds_off (&va)[4],
                  auto OV) {
    sf_u32x4 kf[8];
    read_k<decltype(OK)::value>(ka, kf);
    __builtin_amdgcn_sched_barrier(0);
    if (resc) {   // what the step before decided: acc to the reference of its P
#pragma unroll
      for (int dt = 0; dt < 4; ++dt) acc[dt] = acc[dt] * alpha;
    }
    const int key0 = keys.key0(c0 + k);
    const bool masked = key0 + kStage > end_min || (key0 < lo_max && key0 + kStage > c.sinks);
    if (masked) mask_scores(sc, key0, hf, end, lo, c.sinks);
    // O^T += V^T P^T of stage k - 1: dim tiles d0 .. d1 of the keys 16kk
    auto pv = [&](int kk, int d0, int d1) {
#pragma unroll
      for (int dt = 0; dt < 4; ++dt)
        if (dt >= d0 && dt < d1)
          acc[dt] = mfma32(v_operand(vf, kk, dt), sf_as_bf16x8(pp[kk]), acc[dt]);
    };
    copy(0);
    pv(0, 0, 2);
    float mx = sc[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) mx = fmaxf(mx, sc[i]);
    mx *= scale_log2;
    resc = __ballot(mx > m_lim) != 0;   // wave-uniform
    if (resc) {
      const float m_new = fmaxf(m_ref, fmaxf(mx, __shfl_xor(mx, 32, 64)));
      mu = m_new == -INFINITY ? 0.f : m_new;
      alpha = __builtin_amdgcn_exp2f(m_ref - mu);
      m_ref = m_new;
      m_lim = m_new + kLazy;
      l_run *= alpha;
    }
    float p[16];
    copy(1);
    pv(0, 2, 4);
    pv(1, 0, 4);
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = __builtin_amdgcn_exp2f(fmaf(sc[i], scale_log2, -mu));
    // (pinned: the compiler would take them to their use, behind all the MFMAs)
#pragma unroll
    for (int i = 0; i < 8; ++i) sf_pin(p[i]);
#pragma unroll
    for (int i = 0; i < 6; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x402, 3, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
    copy(2);
    sf_lds_reads_done(kf);
    read_v<decltype(OV)::value>(va, vf);
    __builtin_amdgcn_sched_barrier(0);
    qk(kf, sn);
#pragma unroll
    for (int i = 8; i < 16; ++i) p[i] = __builtin_amdgcn_exp2f(fmaf(sc[i], scale_log2, -mu));
    float s0 = 0.f, s1 = 0.f;
#pragma unroll
    for (int i = 0; i < 16; i += 2) s0 += p[i], s1 += p[i + 1];
    l_run += s0 + s1;
    pack_p(p, pc);
    sf_pin(l_run);
    sf_pin(pc[0]);
    sf_pin(pc[1]);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x402, 6, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
    copy(3);
    sf_lds_reads_done(vf);
    if (masked) bad = bad || any_not_finite(vf);
  };

  // Two stages a turn: slots 2i, 2i + 1 of the ring.  At the start of step k the stages to
  // k + 1 have landed and every wave is through with stage k - 1's slot, which takes
  // stage k + kAhead.
#pragma unroll 1
  for (int k = 0; k < nst; k += 2) {
    const sf_lds_off b0 = sf_lds_addr(ring) + (k % kRing) * kSlot;
    sf_lds_off ka[8], va[4];
#pragma unroll
    for (int ks = 0; ks < 8; ++ks) ka[ks] = b0 + koff[ks];
#pragma unroll
    for (int dt = 0; dt < 4; ++dt) va[dt] = b0 + voff[dt];
    aim(k + kAhead);
    sf_wait_vm_barrier<(kAhead - 2) * 4>();
    step(k, sa, sb, pb, pa, ka, Int<kSlot>{}, va, Int<0>{});
    if (k + 1 == nst) {   // (workgroup-uniform) the last: its P.V follows from the b side
      pb[0] = pa[0];
      pb[1] = pa[1];
      break;
    }
    const sf_lds_off b1 = sf_lds_addr(ring) + ((k + 2) % kRing) * kSlot;
#pragma unroll
    for (int ks = 0; ks < 8; ++ks) ka[ks] = b1 + koff[ks];
    aim(k + 1 + kAhead);
    sf_wait_vm_barrier<(kAhead - 2) * 4>();
    step(k + 1, sb, sa, pa, pb, ka, Int<0>{}, va, Int<kSlot>{});
  }
  sf_wait_vm_barrier<0>();   // drain the copies past the range's end
  if (bad) {   // wave-uniform
    slow_queries(q, c, s, it.h, it.r, q0, 32, keys, c0, nst, Out{o, lse, ws_o, ws_ml, scale_log2});
    return;
  }
  if (resc) {
#pragma unroll
    for (int dt = 0; dt < 4; ++dt) acc[dt] = acc[dt] * alpha;
  }
#pragma unroll
  for (int kk = 0; kk < 2; ++kk)
#pragma unroll
    for (int dt = 0; dt < 4; ++dt)
      acc[dt] = mfma32(v_operand(vf, kk, dt), sf_as_bf16x8(pb[kk]), acc[dt]);

  const float l = l_run + __shfl_xor(l_run, 32, 64);
  if (q0 + (lane & 31) >= nq) return;
  if (keys.nst <= c.spr) {
    write_direct(acc, m_ref, l, hf, o + rh * kHD, lse ? lse + rh : nullptr);
  } else {
    const size_t slot = (size_t)it.r * c.rows * c.H + rh;
    write_partial(acc, m_ref, l, hf, ws_o + slot * kHD, ws_ml + slot * 2);
  }
}

// ---- up to 32 queries of a kv head (a token, or a few) ---------------------------------------
// Bound by reading the cache once: each of the W waves takes every W-th stage of the
// range with all the queries, through an LDS slot of its own (no workgroup barrier): a
// stage's operands go to registers as soon as it has landed, and the slot takes the next
// one.  Four waves, two workgroups a CU, or eight waves and one: 128 KB on their way.  The
// waves' states are joined at the end.  Eight waves take a tile's stages without ranges, so
// without their join: one token of a cache (32 / 8 heads), ranges and join against eight
// waves: 7 stages 7.3 / 7.3 us, 13 9.8 / 8.6, 19 10.5 / 9.2, 26 10.5 / 10.5, 33 10.6 / 11.9
// (eight sequences: 12.9 / 12.0; a launch less, 4 us of the host, on this side), 41 10.7 /
// 13.4.
// 8 tokens over caches of up to 8192 keys (32 / 8 heads): 23.5 us, 5.4 TB/s, and 7 us to
// join the ranges; one token that sees 1028 of 16384 keys (40 / 8): 12 us of eight waves,
// latency: page id, then five rounds of keys.
template <int W>   // waves
__global__ __launch_bounds__(64 * W) __attribute__((amdgpu_waves_per_eu(2, 2))) void
sf_window_few_kernel(const uint16_t* __restrict__ q, Call c, float scale_log2,
                     uint16_t* __restrict__ o, float* __restrict__ lse, float* __restrict__ ws_o,
                     float* __restrict__ ws_ml) {
  __shared__ __attribute__((aligned(16))) uint8_t ring[W * kSlot];
  __shared__ int s_bad[W];
  __shared__ sf_f32x2 s_ml[W][32];
  const Item it = find_item<true>(c);
  const Seq& s = c.s[it.si];
  const int lane = threadIdx.x & 63, hf = lane >> 5;
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);   // wave-uniform
  const int G = c.H / c.Hkv, nq = s.rows * G, P = s.length;
  const Keys keys = query_tile_keys(0, 32, G, s.rows, P, c.block, c.window, c.sinks);
  const int c0 = it.r * c.spr;
  if (c0 >= keys.nst) return;
  const int nst = min(c.spr, keys.nst - c0);
  const int lastg = last_group(P);
  // lane i: 16-key group i & 1 of this wave's stage 32u + i / 2 (past the range: the last)
  auto lane_group = [&](int u) {
    return min(keys.key0(c0 + min(wv + W * (32 * u + (lane >> 1)), nst - 1)) + 16 * (lane & 1),
               lastg);
  };
  auto load_pages = [&](int u) { return s.table ? s.table[lane_group(u) >> c.page_shift] : 0; };
  const int pg = load_pages(0);
  const int qi = min(lane & 31, nq - 1);
  const int m = qi / G;
  const int end = row_end(m, s.rows, P, c.block), lo = row_lo(m, s.rows, P, c.window);
  const int end_min = row_end(0, s.rows, P, c.block);
  const int lo_max = row_lo(s.rows - 1, s.rows, P, c.window);
  const size_t rh = (size_t)(s.row0 + m) * c.H + it.h * G + (qi - m * G);
  sf_u32x4 qf[8];
#pragma unroll
  for (int ks = 0; ks < 8; ++ks)
    qf[ks] = *reinterpret_cast<const sf_u32x4*>(q + rh * kHD + 16 * ks + 8 * hf);

  uint8_t* mine = ring + wv * kSlot;
  const uint16_t* const kb = s.k + (long long)it.h * s.head_stride;
  const uint16_t* const vb = s.v + (long long)it.h * s.head_stride;
  Groups groups;
  groups.set(group_off(s, c.page_shift, pg, lane_group(0)));
  auto issue = [&](int j) {   // this wave's stage j
    if (j > 0 && (j & 31) == 0)
      groups.set(group_off(s, c.page_shift, load_pages(j >> 5), lane_group(j >> 5)));
    const int key0 = keys.key0(c0 + wv + W * j);
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const int last = min(15, P - 1 - min(key0 + 16 * g, lastg));   // of the group's rows
      uint32_t ok[4], ov[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        ok[i] = copy_off(lane, 4 * i, false, last);
        ov[i] = copy_off(lane, 4 * i, true, last);
      }
      const long long at = groups.at(2 * (j & 31) + g);
      copy_rows<4>(kb + at, ok, mine + 16 * g * kRowBytes);
      copy_rows<4>(vb + at, ov, mine + kHalf + 16 * g * kRowBytes);
    }
  };
  if (wv < nst) issue(0);
  sf_lds_off ka[8], va[4];
#pragma unroll
  for (int ks = 0; ks < 8; ++ks) ka[ks] = sf_lds_addr(mine) + k_off(lane, ks);
#pragma unroll
  for (int dt = 0; dt < 4; ++dt) va[dt] = sf_lds_addr(mine) + v_off(lane, dt);

  float m_ref = -INFINITY, l_run = 0.f;   // the query's reference: its running maximum
  bool bad = false;
  sf_f32x16 acc[4];
#pragma unroll
  for (int dt = 0; dt < 4; ++dt)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[dt][i] = 0.f;

#pragma unroll 1
  for (int j = 0; wv + W * j < nst; ++j) {
    wait_vm_wave<0>();   // the stage (and the queries) have landed
    sf_u32x4 kf[8];
    sf_u32x2 vf[16];
    read_k<0>(ka, kf);
    read_v<0>(va, vf);
    sf_lds_reads_done(kf);
    sf_lds_reads_done(vf);
    wait_vm_wave<63>();   // (every lane has read)
    if (wv + W * (j + 1) < nst) issue(j + 1);
    sf_f32x16 sc;
#pragma unroll
    for (int i = 0; i < 16; ++i) sc[i] = 0.f;
#pragma unroll
    for (int ks = 0; ks < 8; ++ks)
      sc = mfma32(sf_as_bf16x8(kf[ks]), sf_as_bf16x8(qf[ks]), sc);
    const int key0 = keys.key0(c0 + wv + W * j);
    const bool masked = key0 + kStage > end_min || (key0 < lo_max && key0 + kStage > c.sinks);
    if (masked) mask_scores(sc, key0, hf, end, lo, c.sinks);
    float mx = sc[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) mx = fmaxf(mx, sc[i]);
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64)) * scale_log2;
    const float nm = fmaxf(m_ref, mx);
    const float mu = nm == -INFINITY ? 0.f : nm;
    const float alpha = __builtin_amdgcn_exp2f(m_ref - mu);
    m_ref = nm;
    float p[16], s0 = 0.f, s1 = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) p[i] = __builtin_amdgcn_exp2f(fmaf(sc[i], scale_log2, -mu));
#pragma unroll
    for (int i = 0; i < 16; i += 2) s0 += p[i], s1 += p[i + 1];
    l_run = l_run * alpha + (s0 + s1);
    sf_u32x4 pb[2];
    pack_p(p, pb);
#pragma unroll
    for (int dt = 0; dt < 4; ++dt) acc[dt] = acc[dt] * alpha;
    if (masked) bad = bad || any_not_finite(vf);
#pragma unroll
    for (int kk = 0; kk < 2; ++kk)
#pragma unroll
      for (int dt = 0; dt < 4; ++dt)
        acc[dt] = mfma32(v_operand(vf, kk, dt), sf_as_bf16x8(pb[kk]), acc[dt]);
  }
  l_run += __shfl_xor(l_run, 32, 64);
  sf_wait_vm_barrier<0>();   // the ring is free: every copy landed, every wave done

  // a hidden value that was not finite: the item again, a key at a time
  if (lane == 0) s_bad[wv] = bad;
  __syncthreads();
  int any = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) any |= s_bad[w];
  if (any) {   // workgroup-uniform
    slow_queries(q, c, s, it.h, it.r, 32 / W * wv, 32 / W, keys, c0, nst,
                 Out{o, lse, ws_o, ws_ml, scale_log2});
    return;
  }

  // join the waves' states through LDS, each wave 16 / W of the 16 pieces of the dims
  float* const xo = reinterpret_cast<float*>(ring);   // [wave][dt][4][lane] x 4
#pragma unroll
  for (int dt = 0; dt < 4; ++dt)
#pragma unroll
    for (int b = 0; b < 4; ++b)
      *reinterpret_cast<sf_f32x4*>(xo + (((wv * 4 + dt) * 4 + b) * 64 + lane) * 4) =
          sf_f32x4{acc[dt][4 * b], acc[dt][4 * b + 1], acc[dt][4 * b + 2], acc[dt][4 * b + 3]};
  if (hf == 0) s_ml[wv][lane] = sf_f32x2{m_ref, l_run};
  __syncthreads();
  float f[W], mm = -INFINITY, l = 0.f;
  sf_f32x2 ml[W];
#pragma unroll
  for (int w = 0; w < W; ++w) {
    ml[w] = s_ml[w][lane & 31];
    mm = fmaxf(mm, ml[w].x);
  }
  const float mu = mm == -INFINITY ? 0.f : mm;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    f[w] = __builtin_amdgcn_exp2f(ml[w].x - mu);
    l = fmaf(ml[w].y, f[w], l);
  }
  if ((lane & 31) >= nq) return;
  const bool direct = keys.nst <= c.spr;
  const size_t slot_at = direct ? 0 : (size_t)it.r * c.rows * c.H + rh;
  const float inv = 1.0f / l;
#pragma unroll
  for (int u = 0; u < 16 / W; ++u) {
    const int piece = 16 / W * wv + u, dim = 8 * piece + 4 * hf;
    sf_f32x4 x{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const sf_f32x4 y =
          *reinterpret_cast<const sf_f32x4*>(xo + ((w * 16 + piece) * 64 + lane) * 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = fmaf(y[i], f[w], x[i]);
    }
    if (direct)
      *reinterpret_cast<sf_u32x2*>(o + rh * kHD + dim) =
          sf_u32x2{sf_pack2(x[0] * inv, x[1] * inv), sf_pack2(x[2] * inv, x[3] * inv)};
    else
      sf_handoff_store(reinterpret_cast<sf_f32x4*>(ws_o + slot_at * kHD + dim), x);
  }
  if (wv > 0 || hf > 0) return;
  if (!direct)
    sf_handoff_store(reinterpret_cast<sf_f32x2*>(ws_ml + slot_at * 2), sf_f32x2{mm, l});
  else if (lse)
    lse[rh] = mm * kLn2 + logf(l);
}

// ---- join the ranges: one wave per (row, q-head), two dims a lane, NB ranges on their way ------
// (bound by the latency of a launch and two dependent loads: 5.5 to 8 us for 1 to 90 rows)
template <int NB>
__global__ __launch_bounds__(kThreads) void sf_window_merge_kernel(Call c, int bq,
                                                                   uint16_t* __restrict__ o,
                                                                   float* __restrict__ lse,
                                                                   const float* __restrict__ ws_o,
                                                                   const float* __restrict__ ws_ml) {
  const int lane = threadIdx.x & 63;
  const int e = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (e >= c.rows * c.H) return;
  const int row = e / c.H, hq = e - row * c.H;
  int si = 0;
  while (row >= c.s[si].row0 + c.s[si].rows) ++si;
  const Seq& s = c.s[si];
  if (s.tiles == 0) return;   // of the other launch
  const int G = c.H / c.Hkv;
  const int qi = (row - s.row0) * G + hq % G;
  const Keys keys =
      query_tile_keys(qi / bq, bq, G, s.rows, s.length, c.block, c.window, c.sinks);
  const int nm = (keys.nst + c.spr - 1) / c.spr;   // <= nr <= 64
  if (nm == 1) return;   // written by its only range
  const size_t step = (size_t)c.rows * c.H;
  sf_f32x2 a[NB];
  auto load = [&](int r0) {
#pragma unroll
    for (int u = 0; u < NB; ++u)
      a[u] = sf_handoff_load(reinterpret_cast<const sf_f32x2*>(
          ws_o + (e + min(r0 + u, nm - 1) * step) * kHD + 2 * lane));
  };
  load(0);
  const sf_f32x2 ml = sf_handoff_load(
      reinterpret_cast<const sf_f32x2*>(ws_ml + (e + min(lane, nm - 1) * step) * 2));
  const float mr = lane < nm ? ml.x : -INFINITY;
  const float mm = sf_wave_max(mr);
  const float mu = mm == -INFINITY ? 0.f : mm;
  const float w = lane < nm ? __builtin_amdgcn_exp2f(mr - mu) : 0.f;
  // (a range in which the row sees nothing: m -inf, l 0, acc 0)
  const float l = sf_wave_sum(lane < nm ? ml.y * w : 0.f);
  const float inv = 1.0f / l;
  float ax = 0.f, ay = 0.f;
  for (int r0 = 0; r0 < nm; r0 += NB) {
    if (r0 > 0) load(r0);
#pragma unroll
    for (int u = 0; u < NB; ++u) {
      if (r0 + u < nm) {   // wave-uniform
        const float wr = __shfl(w, r0 + u, 64);
        ax = fmaf(wr, a[u].x, ax);
        ay = fmaf(wr, a[u].y, ay);
      }
    }
  }
  *reinterpret_cast<uint32_t*>(o + (size_t)e * kHD + 2 * lane) = sf_pack2(ax * inv, ay * inv);
  if (lse && lane == 0) lse[e] = mm * kLn2 + logf(l);
}

// ---- key mass --------------------------------------------------------------------------------
// A workgroup sums the weights of 256 keys (wave w: 64 of them, K operands in registers)
// over a range of the queries that see them, 32 at a time through an LDS ring: S^T = K Q^T
// as above, so a lane adds up the weights one of every 32 queries gives to 32 keys, and the
// lanes are joined every 32 stages, in a fixed order: the error of one fp32 chain over all
// of them would grow with the queries (3e-6 relative for 4096 rows, 1.7e-7 so).  The step
// of stage i runs the weights of stage i beside S^T of stage i + 1.
// Many rows: bound by matrix products, weights (an fma, an exponential and an addition per
// score) and copies in turn on every SIMD: 4096 rows of 28 / 4 heads over themselves 90 us
// and 4.7 to join the ranges (0.65 PFLOP/s), of which the weights, half the products, the
// masks or the copies taken away give 8 to 11 us each.  Few rows: latency (page id, K rows,
// K operands, stages, the lanes' join): 32 rows of 40 / 8 heads over 16416 keys 17 us, 8
// tokens over 12600 keys in all (32 / 8) 8.5 us.
struct MassSeq {
  const float* in;
  float* out;
  long long in_stride, out_stride;
  int key0;   // its first key's place in a row of partial sums
};
struct MassCall : Call {
  MassSeq mass[kMaxSeqs];
  Div div_g, div_block;
  int keys;   // of all sequences
  int last_first;
};
// 4 bytes per lane of a direct copy, and an LDS read of 4 bytes without a wait.
#if defined(__HIPCC__)
SF_DEV void lds_dma4(const void* src, void* lds_base) {
  __builtin_amdgcn_global_load_lds(const_cast<void*>(src), (sf_lds_void*)lds_base, 4, 0, 0);
}
SF_DEV uint32_t lds_read4(sf_lds_off addr) {
  uint32_t v;
  asm volatile("ds_read_b32 %0, %1" : "=v"(v) : "v"(addr));
  return v;
}
#else
inline void lds_dma4(const void* src, void* lds_base) {
  __builtin_memcpy(static_cast<char*>(lds_base) + 4 * sim_lane(), src, 4);
}
inline uint32_t lds_read4(sf_lds_off addr) { return sf_lds_read4_now(addr); }
#endif

constexpr int kQSlot = 32 * kRowBytes;   // 32 queries: 8 KB
constexpr int kMassRing = 4;             // slot 0 of its own, the others over the K rows
constexpr int kFlush = 32;               // stages summed lane by lane

__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(2, 2))) void
sf_window_mass_kernel(const uint16_t* __restrict__ q, const float* __restrict__ lse, MassCall c,
                      float scale_log2, float decay, float* __restrict__ ws) {
  // K rows of the four waves (16 KB each), slot 0, the stages' lse (256 bytes a slot)
  __shared__ __attribute__((aligned(16))) uint8_t lds[4 * 2 * kHalf + kQSlot + kMassRing * 256];
  const Item it = find_item<false>(c);
  const Seq& s = c.s[it.si];
  const MassSeq& ms = c.mass[it.si];
  // the first keys (the most rows) first; where every tile has as many, the last ones, which
  // may be few and then make room for another tile early
  const int tile = c.last_first ? it.tile : s.tiles - 1 - it.tile;
  const int lane = threadIdx.x & 63, hf = lane >> 5;
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);   // wave-uniform
  const int G = c.H / c.Hkv, P = s.length, n = s.rows;
  const int k0 = tile * kMassKeys;
  const Rows rows = seen_rows(k0, min(k0 + kMassKeys, P) - 1, n, P, c.block, c.window, c.sinks);
  const int all = mass_stages(rows, G);
  const int i0 = it.r * c.spr;
  if (i0 >= all && it.r > 0) return;
  const int nst = max(0, min(c.spr, all - i0));
  const int qb = rows.m0 * G + 32 * i0, q_end = rows.m1 * G;
  const int kw0 = k0 + 64 * wv;   // the wave's first key
  // this lane's query qi as a byte offset into its sequence's rows of q (of lse: / 64)
  const uint32_t row_gap = (uint32_t)(c.H - G) * kRowBytes;
  auto q_off = [&](int qi) {
    return (uint32_t)qi * kRowBytes + (uint32_t)c.div_g.of(qi) * row_gap;
  };
  const char* const qh = reinterpret_cast<const char*>(q + ((size_t)s.row0 * c.H + it.h * G) * kHD);
  const char* const lseh = reinterpret_cast<const char*>(lse + (size_t)s.row0 * c.H + it.h * G);

  uint8_t* const kmine = lds + wv * 2 * kHalf;
  uint8_t* const lse_at = lds + 4 * 2 * kHalf + kQSlot;
  auto slot = [&](int i) {
    return i % kMassRing == 0 ? lds + 4 * 2 * kHalf : lds + (i % kMassRing - 1) * kQSlot;
  };
  uint32_t unit[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) unit[u] = (uint32_t)copy_unit(lane, 8 * wv + 4 * u, false) * 2;
  // stage i's queries (wave w: 8 rows) and their lse: past the range its last stage again,
  // past the queries the last query
  auto issue = [&](int i) {
    const int q0 = qb + 32 * min(i, nst - 1);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int r0 = 8 * wv + 4 * u;
      sf_lds_dma16(qh + (q_off(min(q0 + r0 + (lane >> 4), q_end - 1)) + unit[u]),
                   slot(i) + r0 * kRowBytes);
    }
    // (all four waves write the same values: the copies a wave counts stay alike)
    lds_dma4(lseh + q_off(min(q0 + (lane & 31), q_end - 1)) / 64, lse_at + 256 * (i % kMassRing));
  };

  float acc[2][16], total = 0.f;
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[t][i] = 0.f;
  // the key this lane ends with, and what that had (on its way beside the K rows)
  const int x = lane & 31;
  const int key = kw0 + 32 * (x >> 4) + 8 * ((x & 15) >> 2) + 4 * hf + (x & 3);
  float had = 0.f;
  if (c.nr == 1 && ms.in && key < P) had = decay * ms.in[it.h * ms.in_stride + key];
  // acc joined over the lanes and added to the total of this lane's key: lane x of a half
  // ends with value x of the 32 (key tile x / 16)
  auto flush = [&]() {
    float v[32];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int j = 0; j < 16; ++j) v[16 * t + j] = acc[t][j], acc[t][j] = 0.f;
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) {
      const bool up = lane & o;
#pragma unroll
      for (int x = 0; x < o; ++x) {
        const float give = up ? v[x] : v[x + o], keep = up ? v[x + o] : v[x];
        v[x] = keep + __shfl_xor(give, o, 64);
      }
    }
    total += v[0];
  };

  if (nst > 0) {   // workgroup-uniform
    // ---- the wave's 64 keys, stage 0, then the K operands to registers --------------------
    {
      const int lastg = last_group(P);
      const uint16_t* const kb = s.k + (long long)it.h * s.head_stride;
      const int g0 = min(kw0 + 16 * (lane & 3), lastg);   // lane g: the wave's group g
      Groups groups;
      groups.set(group_off(s, c.page_shift, s.table ? s.table[g0 >> c.page_shift] : 0, g0));
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        uint32_t off[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          off[i] = copy_off(lane, 4 * i, false, min(15, P - 1 - min(kw0 + 16 * g, lastg)));
        copy_rows<4>(kb + groups.at(g), off, kmine + 16 * g * kRowBytes);
      }
    }
    issue(0);
    sf_wait_vm_barrier<0>();
    uint32_t koff[8];
#pragma unroll
    for (int ks = 0; ks < 8; ++ks) koff[ks] = k_off(lane, ks);
    sf_u32x4 kf[2][8];
    {
      sf_lds_off ka[8];
#pragma unroll
      for (int ks = 0; ks < 8; ++ks) ka[ks] = sf_lds_addr(kmine) + koff[ks];
      read_k<0>(ka, kf[0]);
      read_k<kHalf>(ka, kf[1]);
      sf_lds_reads_done(kf[0]);
      sf_lds_reads_done(kf[1]);
    }
    sf_lds_barrier();   // the K rows make room for slots 1 ..
#pragma unroll
    for (int i = 1; i < kMassRing - 1; ++i) issue(i);

    const sf_lds_off lse_addr = sf_lds_addr(lse_at) + 4 * lane;
    // In stages [full0, full1) every query sees all of the wave's keys: rows from the first
    // that sees the last key to the last whose window reaches the first.
    const int kw1 = min(kw0 + 64, P) - 1;   // (a wave behind the last key: none)
    const Rows some = seen_rows(kw0, kw1, n, P, c.block, c.window, c.sinks);
    const int full_m0 = seen_rows(kw1, kw1, n, P, c.block, 0, 0).m0;
    const int full_m1 = kw1 < c.sinks ? n : seen_rows(kw0, kw0, n, P, c.block, c.window, 0).m1;
    const bool none = kw0 >= P || some.m1 <= some.m0;
    const int full0 = (full_m0 * G - qb + 31) >> 5, full1 = (min(full_m1 * G, q_end) - qb) >> 5;

    auto read_q = [&](int i, sf_u32x4 (&qf)[8], uint32_t& w) {
      sf_lds_off ka[8];
      const sf_lds_off b = sf_lds_addr(slot(i));
#pragma unroll
      for (int ks = 0; ks < 8; ++ks) ka[ks] = b + koff[ks];
      read_k<0>(ka, qf);
      w = lds_read4(lse_addr + 256 * (i % kMassRing));
    };
    // S^T of a stage (both key tiles)
    auto scores = [&](const sf_u32x4 (&qf)[8], sf_f32x16 (&out)[2]) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int j = 0; j < 16; ++j) out[t][j] = 0.f;
#pragma unroll
      for (int ks = 0; ks < 8; ++ks)
#pragma unroll
        for (int t = 0; t < 2; ++t)
          out[t] = mfma32(sf_as_bf16x8(kf[t][ks]), sf_as_bf16x8(qf[ks]), out[t]);
    };
    // stage i: its scores in sc, its queries' -lse (base 2) in nl; stage i + 1's to sn, nn
    auto step = [&](int i, sf_f32x16 (&sc)[2], const float& nl, sf_f32x16 (&sn)[2], float& nn) {
      // stage i + 1 has landed, and every wave is through with stage i - 1's slot
      sf_wait_vm_barrier<(kMassRing - 3) * 3>();
      issue(i + kMassRing - 1);
      sf_u32x4 qf[8];
      uint32_t w;
      read_q(i + 1, qf, w);
      __builtin_amdgcn_sched_barrier(0);
      auto weights = [&](int t) {
#pragma unroll
        for (int j = 0; j < 16; ++j)
          sc[t][j] = __builtin_amdgcn_exp2f(fmaf(sc[t][j], scale_log2, nl));
      };
      weights(0);
      sf_pin(sc[0]);   // (here, not at its use)
      __builtin_amdgcn_sched_barrier(0);
      sf_lds_reads_done(qf);
      sf_pin(w);
      nn = -kLog2e * __uint_as_float(w);
      scores(qf, sn);
      weights(1);
      sf_pin(sc[1]);
#pragma unroll
      for (int u = 0; u < 16; ++u) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x402, 2, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
      if (i < full0 || i >= full1) {   // wave-uniform
        const int qi = qb + 32 * i + (lane & 31);
        const int m = c.div_g.of(min(qi, q_end - 1));
        const bool any = qi < q_end && !none;
        const int end = any ? P - n + min(n, (c.div_block.of(m) + 1) * (int)c.div_block.d) : 0;
        const int lo = any ? row_lo(m, n, P, c.window) : 0;
        const int sinks = any ? c.sinks : 0;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const int key = kw0 + 32 * t + 8 * (j >> 2) + 4 * hf + (j & 3);
            sc[t][j] = seen_key(key, end, lo, sinks) ? sc[t][j] : 0.f;
          }
        sf_pin(sc[0]);
        sf_pin(sc[1]);
      }
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int j = 0; j < 16; ++j) acc[t][j] += sc[t][j];
    };
    sf_f32x16 sa[2], sb[2];
    float na, nb;
    {
      sf_u32x4 qf[8];
      uint32_t w;
      read_q(0, qf, w);
      sf_lds_reads_done(qf);
      sf_pin(w);
      na = -kLog2e * __uint_as_float(w);
      scores(qf, sa);
    }
#pragma unroll 1
    for (int i = 0; i < nst; i += 2) {
      step(i, sa, na, sb, nb);
      if (i + 1 < nst) step(i + 1, sb, nb, sa, na);
      if ((i & (kFlush - 1)) == kFlush - 2) flush();
    }
    sf_wait_vm_barrier<0>();   // drain the copies past the range's end
  }

  flush();
  if (key >= P) return;
  if (c.nr == 1) {
    ms.out[it.h * ms.out_stride + key] = had + total;
  } else {
    sf_handoff_store(ws + ((size_t)it.r * c.Hkv + it.h) * c.keys + ms.key0 + key, total);
  }
}

// the ranges' sums in order, and what the key had
__global__ __launch_bounds__(kMassKeys) void sf_window_mass_merge_kernel(
    MassCall c, float decay, const float* __restrict__ ws) {
  const int h = blockIdx.x % c.Hkv, tt = blockIdx.x / c.Hkv;
  int si = 0;
  while (tt >= c.s[si].tile0 + c.s[si].tiles) ++si;
  const Seq& s = c.s[si];
  const MassSeq& ms = c.mass[si];
  const int k0 = (tt - s.tile0) * kMassKeys, key = k0 + threadIdx.x;
  if (key >= s.length) return;
  const Rows rows = seen_rows(k0, min(k0 + kMassKeys, s.length) - 1, s.rows, s.length, c.block,
                              c.window, c.sinks);
  const int nm = (mass_stages(rows, c.H / c.Hkv) + c.spr - 1) / c.spr;
  const float had = ms.in ? decay * ms.in[h * ms.in_stride + key] : 0.f;
  float sum = 0.f;
  for (int r0 = 0; r0 < nm; r0 += 8) {   // (8 loads on their way together)
    float v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u)
      v[u] = sf_handoff_load(ws + ((size_t)min(r0 + u, nm - 1) * c.Hkv + h) * c.keys + ms.key0 +
                             key);
#pragma unroll
    for (int u = 0; u < 8; ++u) sum += r0 + u < nm ? v[u] : 0.f;
  }
  ms.out[h * ms.out_stride + key] = had + sum;
}

bool aligned(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

int make_call(const sf_kv_seq* seqs, int n_seqs, int page_size, int block, int window, int sinks,
              int H, int Hkv, int hd, float scaling, bool mass, Call& c) {
  if (!seqs) return SF_ERR_ARG;
  if (hd != kHD || H < 1 || Hkv < 1 || H % Hkv != 0 || H / Hkv > kMaxG || H > kMaxH)
    return SF_ERR_SHAPE;
  if (n_seqs < 1 || n_seqs > kMaxSeqs) return SF_ERR_SHAPE;
  if (block < 1 || window < 0 || sinks < 0) return SF_ERR_SHAPE;
  // (the running maximum is the scores' before scaling)
  if (!(scaling > 0.f && scaling < INFINITY)) return SF_ERR_ARG;
  c = Call{};
  c.n_seqs = n_seqs;
  c.page_shift = page_size > 0 ? __builtin_ctz(page_size) : 0;
  c.block = block;
  c.window = window;
  c.sinks = sinks;
  c.H = H;
  c.Hkv = Hkv;
  for (int i = 0; i < n_seqs; ++i) {
    const sf_kv_seq& x = seqs[i];
    if (x.length < 0 || x.length > kMaxKeys || x.rows < 0 || x.rows > x.length) return SF_ERR_SHAPE;
    if (x.reserved != 0) return SF_ERR_ARG;
    if (x.length > 0) {
      if (x.rows > 0 && (!x.k || (!mass && !x.v))) return SF_ERR_ARG;
      if (!aligned(x.k) || !aligned(x.v)) return SF_ERR_ARG;
      if (x.page_stride % 8 || x.head_stride % 8) return SF_ERR_SHAPE;
      if (x.page_table) {
        if (page_size != 16 && page_size != 32 && page_size != 64 && page_size != 128)
          return SF_ERR_SHAPE;
        if (x.pages < 1) return SF_ERR_SHAPE;
      } else if (x.head_stride < (long long)x.length * kHD && Hkv > 1) {
        return SF_ERR_SHAPE;
      }
      if (mass) {
        if (!x.mass_out) return SF_ERR_ARG;
        if (Hkv > 1 && (x.mass_out_stride < x.length || (x.mass_in && x.mass_in_stride < x.length)))
          return SF_ERR_SHAPE;
        if (x.mass_in == x.mass_out && x.mass_in_stride != x.mass_out_stride) return SF_ERR_ARG;
        // sequences that share what one of them writes
        for (int j = 0; j < i; ++j)
          if (x.length > 0 && seqs[j].length > 0 &&
              (x.mass_out == seqs[j].mass_out || x.mass_out == seqs[j].mass_in ||
               x.mass_in == seqs[j].mass_out))
            return SF_ERR_ARG;
      }
    }
    c.s[i] = Seq{x.k, x.v, x.page_table, x.page_stride, x.head_stride, x.length, x.rows, c.rows,
                 x.pages, 0, 0};
    c.rows += x.rows;
  }
  return SF_OK;
}

// Ranges of the tiles for `slots` workgroups at once, in stages: an item costs its stages
// and a fixed part (set-up, and with several ranges its partial sums and their join).  The
// longest item, or the work spread evenly and half an item of imbalance.
struct Cost {
  int one, many;   // stages' worth of an item's fixed part, in one range / several
};
void plan_spread(Call& c, long long work, int longest, int cap, int slots, Cost fix, int unit) {
  double best = 0;
  for (int nr = 1; nr <= cap && nr <= longest; ++nr) {
    const int spr = ((longest + nr - 1) / nr + unit - 1) / unit * unit;
    const double items = c.Hkv * (nr == 1 ? (double)c.tiles : (double)work / spr + 0.5 * c.tiles);
    const double one = spr + (nr == 1 ? fix.one : fix.many + fix.many * (nr / 16) / 4);
    const double all = (c.Hkv * (double)work + items * (one - spr)) / slots;
    // (an XCD may get a few more than its share: one item too many doubles the time)
    const double cost = items <= slots - slots / 32 ? one : all + 0.5 * one;
    if (nr == 1 || cost < best) {
      best = cost;
      c.nr = (longest + spr - 1) / spr;
      c.spr = spr;
    }
  }
}

// The tiles of the sequences with least to most queries a kv head, and their ranges.
int plan_ranges(Call& c, int bq, int least, int most, int slots, Cost fix, int unit) {
  const int G = c.H / c.Hkv;
  long long work = 0;
  int longest = 0;
  c.tiles = 0;
  for (int i = 0; i < c.n_seqs; ++i) {
    Seq& s = c.s[i];
    const int nq = s.rows * G;
    s.tile0 = c.tiles;
    s.tiles = nq >= least && nq <= most ? tiles_of(s.rows, G, bq) : 0;
    c.tiles += s.tiles;
    for (int t = 0; t < s.tiles; ++t) {
      const int n =
          query_tile_keys(t, bq, G, s.rows, s.length, c.block, c.window, c.sinks).nst;
      work += n;
      longest = n > longest ? n : longest;
    }
  }
  if (c.tiles == 0) return 0;
  c.longest = longest;
  plan_spread(c, work, longest, ranges_cap(c.rows), slots, fix, unit);
  return c.tiles * c.nr * c.Hkv;
}

}  // namespace

extern "C" size_t sf_attn_window_workspace_bytes(int rows, int H) {
  if (rows < 0 || H < 1) return 0;
  if (rows == 0) return 16;
  return (size_t)ranges_cap(rows) * rows * H * (kHD + 2) * sizeof(float);
}

extern "C" int sf_attn_window(const uint16_t* q, const sf_kv_seq* seqs, int n_seqs, int page_size,
                              int block, int window, int sinks, int H, int Hkv, int hd,
                              float scaling, uint16_t* o, float* lse, void* workspace,
                              size_t workspace_bytes, void* stream) {
  Call c;
  const int st =
      make_call(seqs, n_seqs, page_size, block, window, sinks, H, Hkv, hd, scaling, false, c);
  if (st != SF_OK) return st;
  if (c.rows == 0) return SF_OK;
  if (!q || !o || !workspace || !aligned(q) || !aligned(o) || !aligned(workspace))
    return SF_ERR_ARG;
  if (workspace_bytes < sf_attn_window_workspace_bytes(c.rows, H)) return SF_ERR_WORKSPACE;
  hipStream_t hs = reinterpret_cast<hipStream_t>(stream);
  const float scale_log2 = scaling * kLog2e;
  float* ws_o = reinterpret_cast<float*>(workspace);
  float* ws_ml = ws_o + (size_t)ranges_cap(c.rows) * c.rows * H * kHD;
  // Sequences of up to 32 queries a kv head, then the others.  Beside others, short ones go
  // along in tiles that they leave mostly empty: a launch of their own takes about 8 us,
  // in which the CUs walk some 3500 stages of such tiles (a call of 2, 26, 30 and 32 rows
  // over 2000 keys, 28 / 4 heads: 33 us in two launches, 22 in one).
  const int G = H / Hkv;
  long long few_stages = 0;
  bool others = false;
  for (int i = 0; i < n_seqs; ++i) {
    const Seq& x = c.s[i];
    if (x.rows * G > 32)
      others = true;
    else if (x.rows > 0)
      few_stages += tile_keys(0, x.rows - 1, x.rows, x.length, block, window, sinks).nst;
  }
  const int few_most = others && few_stages * Hkv < 3500 ? 0 : 32;
  for (int few = 1; few >= 0; --few) {
    const int bq = few ? 32 : kTileQ;
    int items =
        few ? plan_ranges(c, bq, 1, few_most, 2 * kCUs, Cost{12, 20}, 4)
            : plan_ranges(c, bq, few_most + 1, 1 << 30, 2 * kCUs, Cost{6, 24}, 1);
    if (items == 0) continue;
    const int longest = c.longest;
    const bool wide = few && c.tiles * Hkv <= kCUs && longest >= kWideLeast && longest <= kWideMost;
    if (wide) {   // all of a tile's stages
      c.nr = 1;
      c.spr = longest;
      items = c.tiles * Hkv;
    }
    if (few && wide)
      hipLaunchKernelGGL(sf_window_few_kernel<8>, dim3(items), dim3(512), 0, hs, q, c, scale_log2,
                         o, lse, ws_o, ws_ml);
    else if (few)
      hipLaunchKernelGGL(sf_window_few_kernel<4>, dim3(items), dim3(256), 0, hs, q, c, scale_log2,
                         o, lse, ws_o, ws_ml);
    else
      hipLaunchKernelGGL(sf_window_tile_kernel, dim3(items), dim3(kThreads), 0, hs, q, c,
                         scale_log2, o, lse, ws_o, ws_ml);
    if (c.nr > 4)
      hipLaunchKernelGGL((sf_window_merge_kernel<16>), dim3((c.rows * H + 3) / 4), dim3(kThreads),
                         0, hs, c, bq, o, lse, ws_o, ws_ml);
    else if (c.nr > 1)
      hipLaunchKernelGGL((sf_window_merge_kernel<4>), dim3((c.rows * H + 3) / 4), dim3(kThreads),
                         0, hs, c, bq, o, lse, ws_o, ws_ml);
  }
  return sf_launch_status();
}

extern "C" size_t sf_attn_key_mass_workspace_bytes(int keys, int Hkv) {
  if (keys < 0 || Hkv < 1) return 0;
  return keys == 0 ? 16 : (size_t)kMassRanges * Hkv * keys * sizeof(float);
}

extern "C" int sf_attn_key_mass(const uint16_t* q, const float* lse, const sf_kv_seq* seqs,
                                int n_seqs, int page_size, int block, int window, int sinks, int H,
                                int Hkv, int hd, float scaling, float decay, void* workspace,
                                size_t workspace_bytes, void* stream) {
  MassCall c;
  const int st =
      make_call(seqs, n_seqs, page_size, block, window, sinks, H, Hkv, hd, scaling, true, c);
  if (st != SF_OK) return st;
  if (!(decay >= 0.f && decay <= 1.f)) return SF_ERR_ARG;
  if (c.rows > 0 && (!q || !lse || !aligned(q))) return SF_ERR_ARG;
  c.div_g = make_div(H / Hkv);
  c.div_block = make_div(block < kMaxKeys ? block : kMaxKeys);
  // tiles and their stages; ranges as plan_ranges: the longest item, or the work spread
  long long work = 0;
  int longest = 1;
  c.keys = c.tiles = 0;
  for (int i = 0; i < n_seqs; ++i) {
    Seq& s = c.s[i];
    c.mass[i] = MassSeq{seqs[i].mass_in, seqs[i].mass_out, seqs[i].mass_in_stride,
                        seqs[i].mass_out_stride, c.keys};
    c.keys += s.length;
    s.tile0 = c.tiles;
    s.tiles = (s.length + kMassKeys - 1) / kMassKeys;
    c.tiles += s.tiles;
    for (int t = 0; t < s.tiles; ++t) {
      const int k1 = (t + 1) * kMassKeys < s.length ? (t + 1) * kMassKeys : s.length;
      const int n = mass_stages(
          seen_rows(t * kMassKeys, k1 - 1, s.rows, s.length, block, window, sinks), H / Hkv);
      work += n;
      longest = n > longest ? n : longest;
    }
  }
  if (c.keys == 0) return SF_OK;
  if (!workspace || !aligned(workspace)) return SF_ERR_ARG;
  if (workspace_bytes < sf_attn_key_mass_workspace_bytes(c.keys, Hkv)) return SF_ERR_WORKSPACE;
  c.last_first = work == (long long)longest * c.tiles;
  plan_spread(c, work, longest, kMassRanges, 2 * kCUs, Cost{6, 10}, 1);
  hipStream_t hs = reinterpret_cast<hipStream_t>(stream);
  float* ws = reinterpret_cast<float*>(workspace);
  hipLaunchKernelGGL(sf_window_mass_kernel, dim3(c.tiles * c.nr * Hkv), dim3(kThreads), 0, hs, q,
                     lse, c, scaling * kLog2e, decay, ws);
  if (c.nr > 1)
    hipLaunchKernelGGL(sf_window_mass_merge_kernel, dim3(c.tiles * Hkv), dim3(kMassKeys), 0, hs, c,
                       decay, ws);
  return sf_launch_status();
}
