// Attention of new rows over paged caches with a sliding window and sinks, several
// sequences in one call (sf_attn_window), and the weight each cached key got from those
// rows (sf_attn_key_mass).  No counterpart in the reference.
//
// Row m of a sequence (n rows, P cached keys, its own the last n of them) is at position
// p = P - n + m and sees the keys t < end(m) = P - n + min(n, (m / block + 1) * block)
// with t < sinks or t > p - window (window 0: all).  o = softmax(scaling q.k) v,
// lse = ln sum exp(scaling q.k); mass[t] += exp(scaling q.k - lse).
#include <math.h>

#include "sf_common.h"

namespace {

constexpr int kHD = 128;
constexpr int kMaxSeqs = 32;
constexpr int kMaxKeys = 32768;
constexpr int kMaxG = 16;

struct Seq {
  const uint16_t* k;
  const uint16_t* v;
  const int32_t* table;
  const float* mass_in;
  float* mass_out;
  long long page_stride, head_stride, mass_in_stride, mass_out_stride;
  int length, rows, row0, pages;
};
struct Call {
  Seq s[kMaxSeqs];
  int n_seqs, page_size, block, window, sinks, H, Hkv, rows;
};

SF_DEV long long key_off(const Seq& s, int page_size, int h, int t) {
  long long off = (long long)h * s.head_stride;
  if (!s.table) return off + (long long)t * kHD;
  const int lp = t / page_size;
  const int id = s.table[lp];
  return off + (id >= 0 && id < s.pages ? id : 0) * s.page_stride +
         (long long)(t - lp * page_size) * kHD;
}
SF_DEV int row_end(const Call& c, const Seq& s, int m) {
  const long long e = ((long long)(m / c.block) + 1) * c.block;
  return s.length - s.rows + (int)(e < s.rows ? e : s.rows);
}
SF_DEV int row_lo(const Call& c, const Seq& s, int m) {
  const int p = s.length - s.rows + m;
  return c.window && p >= c.window ? p - c.window + 1 : 0;
}

// One wave per (row, q-head), 64 keys at a time: a key per lane for the scores, two dims
// per lane for the values.
__global__ __launch_bounds__(256) void sf_window_attn_kernel(const uint16_t* __restrict__ q,
                                                             Call c, float scaling,
                                                             uint16_t* __restrict__ o,
                                                             float* __restrict__ lse) {
  const int lane = threadIdx.x & 63;
  const int e = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (e >= c.rows * c.H) return;
  const int row = e / c.H, hq = e - row * c.H;
  const int h = hq / (c.H / c.Hkv);
  int si = 0;
  while (row >= c.s[si].row0 + c.s[si].rows) ++si;
  const Seq& s = c.s[si];
  const int m = row - s.row0;
  const int end = row_end(c, s, m), lo = row_lo(c, s, m);
  const uint16_t* qr = q + (size_t)row * c.H * kHD + hq * kHD;
  float mx = -INFINITY, l = 0.f, a0 = 0.f, a1 = 0.f;
  for (int t0 = 0; t0 < end; t0 += 64) {
    if (t0 >= c.sinks && t0 + 64 <= lo) continue;
    const int t = t0 + lane;
    const bool see = t < end && (t < c.sinks || t >= lo);
    float x = -INFINITY;
    if (see) {
      const uint16_t* kr = s.k + key_off(s, c.page_size, h, t);
      x = 0.f;
      for (int d = 0; d < kHD; d += 8) {
        float a[8], b[8];
        sf_unpack8(*reinterpret_cast<const sf_u32x4*>(kr + d), a);
        sf_unpack8(*reinterpret_cast<const sf_u32x4*>(qr + d), b);
        for (int i = 0; i < 8; ++i) x = fmaf(a[i], b[i], x);
      }
      x *= scaling;
    }
    const float nm = fmaxf(mx, sf_wave_max(x));
    const float ref = nm == -INFINITY ? 0.f : nm;
    const float alpha = expf(mx - ref);
    const float p = see ? expf(x - ref) : 0.f;
    l = l * alpha + sf_wave_sum(p);
    a0 *= alpha;
    a1 *= alpha;
    mx = nm;
    unsigned long long bits = __ballot(see);
    while (bits) {
      const int j = __builtin_ctzll(bits);
      bits &= bits - 1;
      const float pj = __shfl(p, j, 64);
      const uint32_t w = *reinterpret_cast<const uint32_t*>(
          s.v + key_off(s, c.page_size, h, t0 + j) + 2 * lane);
      a0 = fmaf(pj, __uint_as_float(w << 16), a0);
      a1 = fmaf(pj, __uint_as_float(w & 0xffff0000u), a1);
    }
  }
  *reinterpret_cast<uint32_t*>(o + (size_t)row * c.H * kHD + hq * kHD + 2 * lane) =
      sf_pack2(a0 / l, a1 / l);
  if (lse && lane == 0) lse[(size_t)row * c.H + hq] = mx + logf(l);
}

// One thread per (sequence, kv head, key).
__global__ __launch_bounds__(256) void sf_window_mass_kernel(const uint16_t* __restrict__ q,
                                                             const float* __restrict__ lse,
                                                             Call c, float scaling, float decay) {
  int tile = blockIdx.x, si = 0;
  for (; si < c.n_seqs; ++si) {
    const int nt = (c.s[si].length + 255) / 256;
    if (tile < nt) break;
    tile -= nt;
  }
  if (si == c.n_seqs) return;
  const Seq& s = c.s[si];
  const int h = blockIdx.y, G = c.H / c.Hkv;
  const int t = tile * 256 + threadIdx.x;
  if (t >= s.length) return;
  sf_u32x4 kv[16];
  const uint16_t* kr = s.k + key_off(s, c.page_size, h, t);
  for (int i = 0; i < 16; ++i) kv[i] = *reinterpret_cast<const sf_u32x4*>(kr + 8 * i);
  float sum = 0.f;
  for (int m = 0; m < s.rows; ++m) {
    if (t >= row_end(c, s, m) || (t >= c.sinks && t < row_lo(c, s, m))) continue;
    for (int g = 0; g < G; ++g) {
      const size_t r = (size_t)(s.row0 + m) * c.H + h * G + g;
      float x = 0.f;
      for (int i = 0; i < 16; ++i) {
        float a[8], b[8];
        sf_unpack8(kv[i], a);
        sf_unpack8(*reinterpret_cast<const sf_u32x4*>(q + r * kHD + 8 * i), b);
        for (int j = 0; j < 8; ++j) x = fmaf(a[j], b[j], x);
      }
      sum += expf(x * scaling - lse[r]);
    }
  }
  const float had = s.mass_in ? decay * s.mass_in[h * s.mass_in_stride + t] : 0.f;
  s.mass_out[h * s.mass_out_stride + t] = had + sum;
}

bool aligned(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

int make_call(const sf_kv_seq* seqs, int n_seqs, int page_size, int block, int window, int sinks,
              int H, int Hkv, int hd, bool mass, Call& c) {
  if (!seqs) return SF_ERR_ARG;
  if (hd != kHD || H < 1 || Hkv < 1 || H % Hkv != 0 || H / Hkv > kMaxG) return SF_ERR_SHAPE;
  if (n_seqs < 1 || n_seqs > kMaxSeqs) return SF_ERR_SHAPE;
  if (block < 1 || window < 0 || sinks < 0) return SF_ERR_SHAPE;
  c = Call{};
  c.n_seqs = n_seqs;
  c.page_size = page_size;
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
      }
    }
    c.s[i] = Seq{x.k, x.v, x.page_table, x.mass_in, x.mass_out, x.page_stride, x.head_stride,
                 x.mass_in_stride, x.mass_out_stride, x.length, x.rows, c.rows, x.pages};
    c.rows += x.rows;
  }
  return SF_OK;
}

}  // namespace

extern "C" size_t sf_attn_window_workspace_bytes(int rows, int H) {
  if (rows < 0 || H < 1) return 0;
  return 16;
}

extern "C" int sf_attn_window(const uint16_t* q, const sf_kv_seq* seqs, int n_seqs, int page_size,
                              int block, int window, int sinks, int H, int Hkv, int hd,
                              float scaling, uint16_t* o, float* lse, void* workspace,
                              size_t workspace_bytes, void* stream) {
  Call c;
  const int st = make_call(seqs, n_seqs, page_size, block, window, sinks, H, Hkv, hd, false, c);
  if (st != SF_OK) return st;
  if (c.rows == 0) return SF_OK;
  if (!q || !o || !workspace || !aligned(q) || !aligned(o) || !aligned(workspace))
    return SF_ERR_ARG;
  if (workspace_bytes < sf_attn_window_workspace_bytes(c.rows, H)) return SF_ERR_WORKSPACE;
  hipLaunchKernelGGL(sf_window_attn_kernel, dim3((c.rows * H + 3) / 4), dim3(256), 0,
                     reinterpret_cast<hipStream_t>(stream), q, c, scaling, o, lse);
  return sf_launch_status();
}

extern "C" size_t sf_attn_key_mass_workspace_bytes(int keys, int Hkv) {
  if (keys < 0 || Hkv < 1) return 0;
  return 16;
}

extern "C" int sf_attn_key_mass(const uint16_t* q, const float* lse, const sf_kv_seq* seqs,
                                int n_seqs, int page_size, int block, int window, int sinks, int H,
                                int Hkv, int hd, float scaling, float decay, void* workspace,
                                size_t workspace_bytes, void* stream) {
  Call c;
  const int st = make_call(seqs, n_seqs, page_size, block, window, sinks, H, Hkv, hd, true, c);
  if (st != SF_OK) return st;
  if (!(decay >= 0.f && decay <= 1.f)) return SF_ERR_ARG;
  if (c.rows > 0 && (!q || !lse || !aligned(q))) return SF_ERR_ARG;
  int keys = 0, tiles = 0;
  for (int i = 0; i < n_seqs; ++i) {
    keys += c.s[i].length;
    tiles += (c.s[i].length + 255) / 256;
  }
  if (keys == 0) return SF_OK;
  if (!workspace || !aligned(workspace)) return SF_ERR_ARG;
  if (workspace_bytes < sf_attn_key_mass_workspace_bytes(keys, Hkv)) return SF_ERR_WORKSPACE;
  hipLaunchKernelGGL(sf_window_mass_kernel, dim3(tiles, Hkv), dim3(256), 0,
                     reinterpret_cast<hipStream_t>(stream), q, lse, c, scaling, decay);
  return sf_launch_status();
}
