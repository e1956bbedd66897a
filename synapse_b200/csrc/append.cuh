// append.cuh -- the batched append of new rows to the KV cache.
#pragma once

#include "internal.cuh"

namespace syn {

// ---------------------------------------------------------------------------
// Batched append: rows of new tokens of several sequences, row t of sequence s
// at position len[s] + t. Per head row: x' = x * w / sqrt(mean(x^2) + eps)
// (q and k, where a norm weight is given), then the rotation of the pairs
// (i, i + hd/2) by the position's angle; q goes to q_out, k and the raw v to
// the position's cache row.
// LP lanes (a power of two) take one head row, VEC pairs each; ONE: a head row
// is one step of its lanes, kept in registers between the sum and the rotation.
// Bound by HBM for prompts, by its launch for single tokens.
// ---------------------------------------------------------------------------
constexpr int AP_MAX = 256;  // sequences per launch (by value)
constexpr int AP_THREADS = 256;

struct AppendArgs {
  const float *q, *k, *v;
  long long ld;
  float* q_out;
  long long ldq;
  int n_heads, n_kv, hd;
  const float *qn, *kn;
  float eps;
  const float *cos_t, *sin_t;
  float *kc, *vc;  // this layer
  const int* ptab;
  int page, maxp, max_seq;
  const int* len;
  const int* seq_of;  // device: one row of each sequence seq_of[row] (replaces the lists below)
  int rows;
  int n;
  int seq[AP_MAX];
  int row0[AP_MAX + 1];  // first row of each sequence; [n] = rows
};

template <int VEC> struct ApVec;
template <> struct ApVec<4> { using T = float4; };
template <> struct ApVec<1> { using T = float; };

template <int VEC, int LP, bool ONE>
__device__ __forceinline__ void append_rows(const AppendArgs& a) {
  using T = typename ApVec<VEC>::T;
  const int heads = a.n_heads + 2 * a.n_kv, half = a.hd >> 1, nv = half / VEC;
  const long long unit = (long long)blockIdx.x * (AP_THREADS / LP) + threadIdx.x / LP;
  const int lane = threadIdx.x % LP;
  const int row = (int)(unit / heads), h = (int)(unit - (long long)row * heads);
  const bool live = row < a.rows;
  int s = 0;
  if (live && !a.seq_of)
    for (int step = AP_MAX / 2; step; step >>= 1)  // the last sequence that starts at or before row
      if (s + step < a.n && a.row0[s + step] <= row) s += step;
  const bool is_q = h < a.n_heads, is_v = h >= a.n_heads + a.n_kv;
  const float* src = nullptr;
  if (live)
    src = (is_q ? a.q + (long long)h * a.hd
                : is_v ? a.v + (long long)(h - a.n_heads - a.n_kv) * a.hd
                       : a.k + (long long)(h - a.n_heads) * a.hd) +
          (long long)row * a.ld;
  const float* w = is_q ? a.qn : is_v ? nullptr : a.kn;
  griddep_wait();
  griddep_launch();
  T x1[1], x2[1];
  float scale = 1.0f;
  if (ONE && live && lane < nv) {
    x1[0] = reinterpret_cast<const T*>(src)[lane];
    x2[0] = reinterpret_cast<const T*>(src + half)[lane];
  }
  if (a.qn || a.kn) {  // (uniform: the shuffles need every lane)
    float acc = 0.0f;
    if (live && w)
      for (int i = lane; i < nv; i += LP) {
        T b1, b2;
        if (ONE) {
          b1 = x1[0];
          b2 = x2[0];
        } else {
          b1 = reinterpret_cast<const T*>(src)[i];
          b2 = reinterpret_cast<const T*>(src + half)[i];
        }
        const float* f1 = reinterpret_cast<const float*>(&b1);
        const float* f2 = reinterpret_cast<const float*>(&b2);
#pragma unroll
        for (int e = 0; e < VEC; e++) acc = fmaf(f1[e], f1[e], fmaf(f2[e], f2[e], acc));
      }
#pragma unroll
    for (int o = LP / 2; o; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
    scale = 1.0f / sqrtf(acc / (float)a.hd + a.eps);
  }
  if (!live) return;
  const int sq = a.seq_of ? a.seq_of[row] : a.seq[s];
  const int pos = a.len[sq] + (a.seq_of ? 0 : row - a.row0[s]);
  if (pos >= a.max_seq) return;  // (a replayed graph that has run past the cache)
  float* dst;
  if (is_q) {
    dst = a.q_out + (long long)row * a.ldq + (long long)h * a.hd;
  } else {
    size_t slot = (size_t)sq * a.max_seq + pos;
    if (a.ptab) {
      const int pg = a.ptab[(size_t)sq * a.maxp + pos / a.page];
      if (pg < 0) return;
      slot = (size_t)pg * a.page + pos % a.page;
    }
    dst = (is_v ? a.vc + (size_t)(h - a.n_heads - a.n_kv) * a.hd
                : a.kc + (size_t)(h - a.n_heads) * a.hd) +
          slot * a.n_kv * a.hd;
  }
  const float* ct = a.cos_t + (size_t)pos * half;
  const float* st = a.sin_t + (size_t)pos * half;
  for (int i = lane; i < nv; i += LP) {
    T b1, b2;
    if (ONE) {
      b1 = x1[0];
      b2 = x2[0];
    } else {
      b1 = reinterpret_cast<const T*>(src)[i];
      b2 = reinterpret_cast<const T*>(src + half)[i];
    }
    if (!is_v) {
      float* f1 = reinterpret_cast<float*>(&b1);
      float* f2 = reinterpret_cast<float*>(&b2);
#pragma unroll
      for (int e = 0; e < VEC; e++) {
        const int d = i * VEC + e;
        float y1 = f1[e], y2 = f2[e];
        if (w) {
          y1 *= w[d] * scale;
          y2 *= w[half + d] * scale;
        }
        const float c = ct[d], sn = st[d];
        f1[e] = y1 * c - y2 * sn;
        f2[e] = y2 * c + y1 * sn;
      }
    }
    reinterpret_cast<T*>(dst)[i] = b1;
    reinterpret_cast<T*>(dst + half)[i] = b2;
  }
}

// Lanes a head row, and whether 16-byte accesses may be used (every head row's
// halves start on 16 bytes).
struct AppendShape {
  int lp;
  bool vec, one;
};
inline AppendShape append_shape(const AppendArgs& a) {
  const uintptr_t low = reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.k) |
                        reinterpret_cast<uintptr_t>(a.v) | reinterpret_cast<uintptr_t>(a.q_out);
  const bool vec = a.hd % 8 == 0 && low % 16 == 0 && a.ld % 4 == 0 && a.ldq % 4 == 0;
  const int lanes = a.hd / 2 / 4;
  if (!vec || lanes > 32) return {32, vec, false};
  return {lanes <= 4 ? 4 : lanes <= 8 ? 8 : lanes <= 16 ? 16 : 32, true, true};
}
// What an append to a layer of cache c takes from its attention arguments; rows, seq, row0
// and seq_of are the caller's.
inline AppendArgs append_args(const AttnArgs& at, float* q_out, size_t ldq, size_t row) {
  const syn_cuda_kvcache_t* c = at.cache;
  const size_t kvd = c->n_kv * c->hd;
  const size_t rows_per_layer = c->page ? c->n_pages * c->page : c->batch * c->max_seq;
  AppendArgs a;
  a.q = at.q + row * at.ld;
  a.k = at.k + row * at.ld;
  a.v = at.v + row * at.ld;
  a.ld = (long long)at.ld;
  a.q_out = q_out + row * ldq;
  a.ldq = (long long)ldq;
  a.n_heads = (int)at.n_heads;
  a.n_kv = (int)c->n_kv;
  a.hd = (int)c->hd;
  a.qn = at.qn;
  a.kn = at.kn;
  a.eps = at.eps;
  a.cos_t = at.cos_t;
  a.sin_t = at.sin_t;
  a.kc = c->k + at.layer * rows_per_layer * kvd;
  a.vc = c->v + at.layer * rows_per_layer * kvd;
  a.ptab = c->page ? c->d_ptab : nullptr;
  a.page = (int)c->page;
  a.maxp = (int)c->maxp;
  a.max_seq = (int)c->max_seq;
  a.len = c->d_len;
  a.seq_of = nullptr;
  a.n = 0;
  return a;
}

}  // namespace syn
