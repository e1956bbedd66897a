// append.cuh -- the batched append of new rows to the KV cache.
#pragma once

#include <initializer_list>

#include "internal.cuh"

namespace syn {

// ---------------------------------------------------------------------------
// Batched append: rows of new tokens of several sequences, row t of sequence s
// at position len[s] + t. Per head row: x' = x * w / sqrt(mean(x^2) + eps)
// (q and k, where a norm weight is given), then the rotation of the pairs
// (i, i + hd/2) by the position's angle; q goes to q_out, k and the raw v to
// the position's cache row.
// LP lanes (a power of two) take one head row, VEC pairs each; ONE: a head row
// is one step of its lanes, kept in registers between the sum and the rotation,
// and HC heads of a row are under way at once, with the position found and its
// angles read once for all of them. Single tokens of 32 sequences (48 head rows of
// 128) take 2.5 us, the launch's own time; 7 ragged prompts (189 MB read and
// written) 42.7 us, 69 % of what a copy of them takes.
// ---------------------------------------------------------------------------
constexpr int AP_MAX = 256;  // sequences per launch (by value)
constexpr int AP_THREADS = 256;
// Blocks from which a launch fills the device: from there on HC is 2. 32 head rows of 128 a token, one
// and two heads a lane group: 8 tokens 2.8 and 3.4 us, 89 tokens 3.2 and 3.6, 281 tokens 4.4 and 4.0, 920
// tokens 10.0 and 8.3, 5736 tokens 53.4 and 43.1.
constexpr size_t AP_FILL = 600;

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
  const int* seq_of;  // device: one row of each sequence seq_of[row] (replaces the lists below) ...
  const int* set_rows;  // ... if *set_rows is `rows`; else nothing
  int* err;  // where a position without a page is reported; may be nullptr
  int rows;
  int n;
  int seq[AP_MAX];
  int row0[AP_MAX + 1];  // first row of each sequence; [n] = rows
};

template <int VEC> struct ApVec;
template <> struct ApVec<4> { using T = float4; };
template <> struct ApVec<1> { using T = float; };

// What else becomes of a rotated q row: find(row, head) before the wait for the kernels before,
// take(...) with its lanes' elements j, j + LP, ... of each half.
struct NoTaker {
  __device__ void find(int, int) {}
  template <int VEC, int LP, typename T> __device__ void take(int, int, const T (&)[2], const T (&)[2]) {}
};

template <int VEC, int LP, bool ONE, int HC, typename Taker = NoTaker>
__device__ __forceinline__ void append_rows(const AppendArgs& a, Taker taker = Taker()) {
  static_assert(ONE || HC == 1, "several heads are held in registers");
  using T = typename ApVec<VEC>::T;
  const int heads = a.n_heads + 2 * a.n_kv, half = a.hd >> 1, nv = half / VEC;
  const int groups = (heads + HC - 1) / HC;
  const long long unit = (long long)blockIdx.x * (AP_THREADS / LP) + threadIdx.x / LP;
  const int lane = threadIdx.x % LP;
  const int row = (int)(unit / groups), h0 = (int)(unit - (long long)row * groups) * HC;
  const bool live = row < a.rows;
  int s = 0;
  if (live && !a.seq_of)
    for (int step = AP_MAX / 2; step; step >>= 1)  // the last sequence that starts at or before row
      if (s + step < a.n && a.row0[s + step] <= row) s += step;
  auto source = [&](int h) {
    return (h < a.n_heads             ? a.q + (long long)h * a.hd
            : h < a.n_heads + a.n_kv ? a.k + (long long)(h - a.n_heads) * a.hd
                                     : a.v + (long long)(h - a.n_heads - a.n_kv) * a.hd) +
           (long long)row * a.ld;
  };
  if (live && HC == 1 && h0 < a.n_heads) taker.find(row, h0);
  griddep_wait();
  griddep_launch();
  T x1[HC], x2[HC];
  const bool mine = live && lane < nv;
  if (ONE)
#pragma unroll
    for (int i = 0; i < HC; i++)
      if (mine && h0 + i < heads) {
        x1[i] = reinterpret_cast<const T*>(source(h0 + i))[lane];
        x2[i] = reinterpret_cast<const T*>(source(h0 + i) + half)[lane];
      }
  int sq = 0, pos = 0;
  if (live) {
    sq = a.seq_of ? a.seq_of[row] : a.seq[s];
    pos = a.len[sq] + (a.seq_of ? 0 : row - a.row0[s]);
  }
  // (a replayed graph may have run past the cache, or its plan may have been set for other rows)
  const bool in = live && pos < a.max_seq && (!a.seq_of || *a.set_rows == a.rows);
  const float* ct = a.cos_t + (size_t)pos * half;
  const float* st = a.sin_t + (size_t)pos * half;
  T c1, s1;
  if (ONE && mine && in) {
    c1 = reinterpret_cast<const T*>(ct)[lane];
    s1 = reinterpret_cast<const T*>(st)[lane];
  }
  long long slot = -1;  // the position's cache row
  if (in) {
    slot = (long long)sq * a.max_seq + pos;
    if (a.ptab) {
      const int pg = a.ptab[(size_t)sq * a.maxp + pos / a.page];
      slot = pg < 0 ? -1 : (long long)pg * a.page + pos % a.page;
      if (pg < 0 && a.err) atomicExch(a.err, SYN_ERR_INVALID_ARG);
    }
  }
#pragma unroll
  for (int i = 0; i < HC; i++) {
    const int h = h0 + i;
    const bool is_q = h < a.n_heads, is_v = h >= a.n_heads + a.n_kv;
    const float* src = live && h < heads ? source(h) : nullptr;
    const float* w = is_q ? a.qn : is_v ? nullptr : a.kn;
    float scale = 1.0f;
    if (a.qn || a.kn) {  // (uniform: the shuffles need every lane)
      float acc = 0.0f;
      if (src && w)
        for (int j = lane; j < nv; j += LP) {
          T b1, b2;
          if (ONE) {
            b1 = x1[i];
            b2 = x2[i];
          } else {
            b1 = reinterpret_cast<const T*>(src)[j];
            b2 = reinterpret_cast<const T*>(src + half)[j];
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
    if (!src || !in || (!is_q && slot < 0)) continue;
    float* dst = is_q ? a.q_out + (long long)row * a.ldq + (long long)h * a.hd
                      : (is_v ? a.vc + (size_t)(h - a.n_heads - a.n_kv) * a.hd
                              : a.kc + (size_t)(h - a.n_heads) * a.hd) +
                            (size_t)slot * a.n_kv * a.hd;
    T r1[2] = {}, r2[2] = {};  // (half a head row of up to 128 elements is two steps of 32 lanes)
    for (int j = lane, step = 0; j < nv; j += LP, step ^= 1) {
      T b1, b2, c, sn;
      if (ONE) {
        b1 = x1[i];
        b2 = x2[i];
        c = c1;
        sn = s1;
      } else {
        b1 = reinterpret_cast<const T*>(src)[j];
        b2 = reinterpret_cast<const T*>(src + half)[j];
        c = reinterpret_cast<const T*>(ct)[j];
        sn = reinterpret_cast<const T*>(st)[j];
      }
      if (!is_v) {
        float* f1 = reinterpret_cast<float*>(&b1);
        float* f2 = reinterpret_cast<float*>(&b2);
        const float* fc = reinterpret_cast<const float*>(&c);
        const float* fs = reinterpret_cast<const float*>(&sn);
        if (w) {
          const T w1 = reinterpret_cast<const T*>(w)[j], w2 = reinterpret_cast<const T*>(w + half)[j];
          const float* g1 = reinterpret_cast<const float*>(&w1);
          const float* g2 = reinterpret_cast<const float*>(&w2);
#pragma unroll
          for (int e = 0; e < VEC; e++) {
            f1[e] *= g1[e] * scale;
            f2[e] *= g2[e] * scale;
          }
        }
#pragma unroll
        for (int e = 0; e < VEC; e++) {
          const float y1 = f1[e], y2 = f2[e];
          // (written out, so that every variant rounds alike)
          f1[e] = __fmaf_rn(y1, fc[e], -__fmul_rn(y2, fs[e]));
          f2[e] = __fmaf_rn(y2, fc[e], __fmul_rn(y1, fs[e]));
        }
      }
      reinterpret_cast<T*>(dst)[j] = b1;
      reinterpret_cast<T*>(dst + half)[j] = b2;
      r1[ONE ? 0 : step] = b1;
      r2[ONE ? 0 : step] = b2;
    }
    if (is_q) taker.template take<VEC, LP>(lane, nv, r1, r2);
  }
}

// Lanes a head row, and whether 16-byte accesses may be used (every head row's
// halves start on 16 bytes).
struct AppendShape {
  int lp;
  bool vec, one;
};
inline AppendShape append_shape(const AppendArgs& a) {
  uintptr_t low = 0;
  for (const float* p : {a.q, a.k, a.v, (const float*)a.q_out, a.cos_t, a.sin_t, a.qn, a.kn})
    low |= reinterpret_cast<uintptr_t>(p);
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
  a.seq_of = a.set_rows = nullptr;
  a.err = nullptr;
  a.n = 0;
  return a;
}

}  // namespace syn
