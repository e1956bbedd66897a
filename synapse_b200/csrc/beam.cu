// beam.cu -- beam search around the paged KV cache: sequences that share
// their leading pages (fork), the batched append of new tokens, the choice of
// the best continuations over beams x vocabulary, and the reordering of the
// beams' caches after it. The reference decodes one greedy sequence
// (generation/pipeline.rs:197-280) and has no counterpart.
#include <math.h>

#include <algorithm>
#include <map>
#include <mutex>
#include <new>
#include <vector>

#include "append.cuh"
#include "internal.cuh"

namespace syn {
namespace {

syn_status_t launched(cudaError_t e, const char* where) {
  if (e == cudaSuccess) return SYN_OK;
  set_last_cuda_error(e, where);
  return SYN_ERR_CUDA;
}

bool capturing(cudaStream_t st) {
  cudaStreamCaptureStatus cs = cudaStreamCaptureStatusNone;
  cudaStreamIsCapturing(st, &cs);
  return cs != cudaStreamCaptureStatusNone;
}

// ---------------------------------------------------------------------------
// One page's first rows to another page: grid (chunks, layers, K / V)
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(256) k_kv_copy_page(float4* k, float4* v, size_t layer4,
                                                      size_t src4, size_t dst4, size_t n4) {
  float4* p = (blockIdx.z ? v : k) + blockIdx.y * layer4;
  for (size_t i = blockIdx.x * 256 + threadIdx.x; i < n4; i += gridDim.x * 256)
    p[dst4 + i] = p[src4 + i];
}

// ---------------------------------------------------------------------------
// Reordering of beams. Group members are numbered 0..B-1; member i takes the
// context of member par(i). Full pages move by their table entries alone. The
// last, partly filled page of every member stays private, since it is written
// next: of a parent's children one (the parent itself if it is among them,
// else the lowest) takes the page over, and each other child copies it into
// the page of a member that has no child, matched in ascending order. No page
// is both read and written, so the copies need no second buffer. The last block
// to finish writes the tail entries, so one launch does it all (two took 48 us where
// this takes 39.3: 4 x 8 beams, 28 layers, 257 MB of copies, the copy rate; 6.1 us for
// 4 beams of 16 layers, latency).
// ---------------------------------------------------------------------------
constexpr int RO_MAX = 256;  // sequences per call (by value in the launch)

struct ReorderArgs {
  float4 *k, *v;
  size_t layer4;   // float4s between layers
  int* ptab;
  int* done;  // finished blocks; zero between launches
  int maxp, page, row4;  // row4: float4s of one position
  int max_seq;
  const int32_t* parents;
  const int* len;  // the sequences' lengths on the device, where a replay finds the current ones
  int n, beams;
  int seq[RO_MAX];
};

__device__ __forceinline__ int ro_parent(const int32_t* par, int i, int beams) {
  const int p = par[i];
  return p >= 0 && p < beams ? p : i;  // out of range: the member keeps its own
}

// The parents of the group from member g0 on, and its length; 0, so that nothing moves, where the
// lengths differ (a replay finds them so; a call refuses them). Whole block.
__device__ __forceinline__ int ro_group(const ReorderArgs& a, int g0, int* par) {
  const int len = min(a.len[a.seq[g0]], a.max_seq);
  bool same = true;
  if (threadIdx.x < a.beams) {
    par[threadIdx.x] = ro_parent(a.parents + g0, threadIdx.x, a.beams);
    same = a.len[a.seq[g0 + threadIdx.x]] == len;
  }
  return __syncthreads_and(same) ? len : 0;
}

// Where member i's last page comes from: {member whose page it takes, 1 if
// the parent's rows have to be copied into it}.
__device__ __forceinline__ int2 ro_tail(const int* par, int i, int beams) {
  const int p = par[i];
  int keeper = -1;
  if (par[p] == p) {
    keeper = p;
  } else {
    for (int j = 0; j < beams && keeper < 0; j++)
      if (par[j] == p) keeper = j;
  }
  if (keeper == i) return make_int2(p, 0);
  // rank of i among the children that keep no page, then the childless member of that rank
  int rank = 0;
  for (int j = 0; j < i; j++) {
    const int pj = par[j];
    bool keeps = pj == j;
    if (!keeps && par[pj] != pj) {
      keeps = true;
      for (int u = 0; u < j; u++)
        if (par[u] == pj) keeps = false;
    }
    rank += !keeps;
  }
  for (int j = 0; j < beams; j++) {
    bool child = false;
    for (int u = 0; u < beams; u++) child |= par[u] == j;
    if (!child && rank-- == 0) return make_int2(j, 1);
  }
  return make_int2(i, 0);  // not reached: as many childless members as copies
}

// grid (chunks, n, layers + 1): the copies of each layer; then, column chunks by group, the
// table entries of full pages. Those of the last pages, which the copies go by, are
// written by the block that finishes last. (The lengths from the device, for the replays, cost 4 x 8
// beams 0.7 us of 39.3.)
__global__ void __launch_bounds__(256) k_reorder(const __grid_constant__ ReorderArgs a) {
  __shared__ int par[RO_MAX], old[RO_MAX][9];
  __shared__ int2 t;
  __shared__ int last;
  const int tid = threadIdx.x;
  griddep_wait();
  griddep_launch();
  if (blockIdx.z < gridDim.z - 1) {
    const int i = blockIdx.y, g0 = i / a.beams * a.beams;
    const int len = ro_group(a, g0, par), tail = len % a.page;
    if (tid == 0) t = ro_tail(par, i - g0, a.beams);
    __syncthreads();
    if (t.y && tail) {
      const int col = len / a.page;
      const int src = a.ptab[(size_t)a.seq[g0 + par[i - g0]] * a.maxp + col];
      const int dst = a.ptab[(size_t)a.seq[g0 + t.x] * a.maxp + col];
      if (src >= 0 && dst >= 0) {
        const size_t n4 = (size_t)tail * a.row4;
        const size_t s4 = (size_t)src * a.page * a.row4, d4 = (size_t)dst * a.page * a.row4;
        float4* k = a.k + blockIdx.z * a.layer4;
        float4* v = a.v + blockIdx.z * a.layer4;
        for (size_t j = blockIdx.x * 256 + tid; j < n4; j += gridDim.x * 256) {
          const float4 x = k[s4 + j], y = v[s4 + j];
          k[d4 + j] = x;
          v[d4 + j] = y;
        }
      }
    }
  } else if (blockIdx.y < a.n / a.beams) {
    const int g0 = blockIdx.y * a.beams, full = ro_group(a, g0, par) / a.page;
    for (int c0 = blockIdx.x * 8; c0 < full; c0 += gridDim.x * 8) {
      for (int u = tid; u < a.beams * 8; u += 256) {
        const int b = u >> 3, c = c0 + (u & 7);
        if (c < full) old[b][u & 7] = a.ptab[(size_t)a.seq[g0 + b] * a.maxp + c];
      }
      __syncthreads();
      for (int u = tid; u < a.beams * 8; u += 256) {
        const int b = u >> 3, c = c0 + (u & 7);
        if (c < full) a.ptab[(size_t)a.seq[g0 + b] * a.maxp + c] = old[par[b]][u & 7];
      }
      __syncthreads();
    }
  }
  __syncthreads();  // (the block has read what it needs of the last pages' entries)
  if (tid == 0) last = atomicAdd(a.done, 1) == (int)(gridDim.x * gridDim.y * gridDim.z) - 1;
  __syncthreads();
  if (!last) return;
  __shared__ int lens[RO_MAX];
  const int g0 = tid / a.beams * a.beams;
  if (tid < a.n) {
    par[tid] = ro_parent(a.parents + g0, tid - g0, a.beams);
    lens[tid] = a.len[a.seq[tid]];
  }
  __syncthreads();
  int entry = -1, len = 0;
  if (tid < a.n) {
    len = min(lens[g0], a.max_seq);
    for (int j = g0; j < g0 + a.beams; j++)
      if (lens[j] != len) len = 0;  // (as ro_group)
  }
  const size_t col = len / a.page;
  const bool mine = len % a.page;
  if (mine) entry = a.ptab[(size_t)a.seq[g0 + ro_tail(par + g0, tid - g0, a.beams).x] * a.maxp + col];
  __syncthreads();
  if (mine) a.ptab[(size_t)a.seq[tid] * a.maxp + col] = entry;
  if (tid == 0) *a.done = 0;
}

template <int VEC, int LP, bool ONE, int HC>
__global__ void __launch_bounds__(AP_THREADS) k_append_batch(const __grid_constant__ AppendArgs a) {
  append_rows<VEC, LP, ONE, HC>(a);
}
template <int HC>
void (*append_kernel(int lp))(const AppendArgs) {
  return lp == 4 ? k_append_batch<4, 4, true, HC> : lp == 8 ? k_append_batch<4, 8, true, HC>
         : lp == 16 ? k_append_batch<4, 16, true, HC> : k_append_batch<4, 32, true, HC>;
}

// ---------------------------------------------------------------------------
// Beam selection. Candidate (b, t) of a group has the value
//   score_b + (x_bt - logsumexp(x_b)),
// compared in 64 bits; equal values go to the lower beam, then to the larger
// logit, then to the lower token. NaN logits count as -inf and +inf as the
// largest float. A finished beam has one candidate, (eos, score_b); its others
// are -inf.
//
// One kernel, CTA = (segment of a row). Within a row the value is monotone in x, so
// a segment's k best logits are all that can be chosen from it. They are found
// in one pass with 64-bit keys (ordered bits of x, then the lower index): of the
// threads' maxima of the first tile, the smallest of the 8 warps' ceil(k / 8)-th
// largest bounds the k-th best from below, and what reaches it is listed; the
// same bound of the whole segment cuts the list before it is ranked. Data that
// defeat the bound (equal or sorted logits) overflow the list and are taken
// once more with an exact bound after each tile. The pass also sums exp(x - m),
// with m the thread's first maximum unless a later one is more than 20 above.
// The group's last CTA to finish joins the segments: logsumexp of each row from
// their (max, sum), a bound on the lists' heads as above (an exact one where that
// lets too many through), one on the elements that are left, and what reaches it
// ranked by counting. Which CTA is last changes no result.
// Bound by HBM for many rows (4 bytes a logit): 160 rows of 128256 take 34.6 us, a third of
// the copy rate, in 2.2 waves of segments (1280 CTAs, four on an SM). By latency for few: 8.4 us for
// 4 rows of 32000, 12.3 for 8 of 151936, a chain of pass, bound, list and join.
// ---------------------------------------------------------------------------
constexpr int BS_THREADS = 256, BS_KMAX = (int)BEAMS_MAX, BS_BMAX = (int)BEAMS_MAX;

__device__ __forceinline__ uint32_t ord32(float x) {  // order-preserving, > 0 for every float
  const uint32_t u = __float_as_uint(x + 0.0f);       // (-0 becomes 0)
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float unord32(uint32_t o) {
  return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ uint64_t ord64(double x) {
  const uint64_t u = (uint64_t)__double_as_longlong(x);
  return u >> 63 ? ~u : u | (1ull << 63);
}
__device__ __forceinline__ double unord64(uint64_t o) {
  return __longlong_as_double((long long)(o >> 63 ? o & ~(1ull << 63) : ~o));
}
__device__ __forceinline__ float ex2f(float x) {  // 2^x, 2 ulp; below 2^-126: 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float tame(float x) {
  return fminf(fmaxf(x, -INFINITY), 3.402823466e+38f);  // (the maximum drops a NaN)
}

struct BeamArgs {
  const float* x;
  long long ld;
  int beams, vocab, k, nseg, tiles, vec;  // tiles of a segment
  int cap;                                // elements that beam_pick has room for
  const float* scores;
  const uint8_t* fin;
  int eos;
  int* cnt;        // [groups] finished segments; zero between launches
  uint64_t* cand;  // [rows][nseg][k], best first, 0 = none
  float2* part;    // [rows][nseg] (max, sum of exp(x - max))
  float* out_s;
  int32_t *out_p, *out_t;
  uint8_t* out_f;
};

constexpr int BS_TILE = BS_THREADS * 8;    // elements of a tile
constexpr int BS_LIST = 1024;              // a longer list is cut ...
constexpr int BS_CAP = BS_LIST + BS_TILE;  // ... before another tile can overflow it
constexpr int BS_WARPS = BS_THREADS / 32;

// The k-th largest of the threads' keys (0 where fewer are not 0). Whole block.
__device__ __forceinline__ uint64_t kth_key(uint64_t key, int k, uint64_t* keys, uint64_t* kth) {
  const int tid = threadIdx.x;
  keys[tid] = key;
  if (tid == 0) *kth = 0;
  __syncthreads();
  int above = 0;
  const ulonglong2* p = reinterpret_cast<const ulonglong2*>(keys);
#pragma unroll 8
  for (int j = 0; j < BS_THREADS / 2; j++) {
    const ulonglong2 u = p[j];
    above += (u.x > key) + (u.y > key);
  }
  if (key && above == k - 1) *kth = key;
  __syncthreads();
  return *kth;
}

// A value that at least k of the threads' values reach (0 where a warp has too few that
// are not 0): the smallest of the warps' ceil(k / 8)-th largest. Whole block.
__device__ __forceinline__ uint32_t low_bound(uint32_t x, int k, uint32_t* warps) {
  const int lane = threadIdx.x & 31;
  uint32_t top = 0;
  for (int r = (k + BS_WARPS - 1) / BS_WARPS; r > 0; r--) {
    top = __reduce_max_sync(0xffffffffu, x);
    const uint32_t has = __ballot_sync(0xffffffffu, x == top);
    if (lane == __ffs(has) - 1) x = 0;
  }
  if (lane == 0) warps[threadIdx.x >> 5] = top;
  __syncthreads();
  uint32_t low = warps[0];
#pragma unroll
  for (int w = 1; w < BS_WARPS; w++) low = min(low, warps[w]);
  return low;
}

// A candidate is ord64 of its value (0 = none) and, for equal values, beam,
// logit and token in 6, 32 and 25 bits, the larger the earlier.
constexpr int BS_TBITS = 25;
__device__ __forceinline__ bool over(uint64_t v, uint64_t i, uint64_t w, uint64_t j) {
  return v > w || (v == w && i > j);
}

// The group's selection from its rows' segments. Whole block; raw: as k_beam_select's.
__device__ __forceinline__ void beam_pick(const BeamArgs& a, int g, uint8_t* raw, uint64_t* tv, uint64_t* ti) {
  const int lists = a.beams * a.nseg, cap = a.cap;
  ulonglong2* best = reinterpret_cast<ulonglong2*>(raw);  // (v, i) of heads, then of finalists
  __shared__ double lse[BS_BMAX];
  __shared__ float sc[BS_BMAX];
  __shared__ uint8_t fin[BS_BMAX];
  __shared__ uint64_t bv, bi;
  __shared__ uint32_t lows[BS_WARPS], lows2[BS_WARPS];
  __shared__ int cnt, nsel, sel[BS_THREADS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int r0 = g * a.beams;
  const uint64_t* cand = a.cand + (size_t)r0 * a.nseg * a.k;
  // (a row's lists on all warps: lists w, w + 8, ... are warp w's)
  const int l0 = lane * BS_WARPS + warp;
  const uint64_t head = l0 < lists ? __ldcg(cand + (size_t)l0 * a.k) : 0;
  for (int b = warp; b < a.beams; b += BS_WARPS) {
    const float2* p = a.part + (size_t)(r0 + b) * a.nseg;
    const float2 first = lane < a.nseg ? __ldcg(p + lane) : make_float2(-INFINITY, 0.0f);
    float M = first.x;
    for (int i = 32 + lane; i < a.nseg; i += 32) M = fmaxf(M, __ldcg(p + i).x);
    M = warp_max(M);
    double s = first.x > -INFINITY ? (double)(first.y * ex2f((first.x - M) * 1.4426950408889634f)) : 0.0;
    for (int i = 32 + lane; i < a.nseg; i += 32) {
      const float2 x = __ldcg(p + i);
      if (x.x > -INFINITY) s += (double)(x.y * ex2f((x.x - M) * 1.4426950408889634f));
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) {
      lse[b] = M > -INFINITY ? (double)M + log(s) : 0.0;
      sc[b] = tame(a.scores[r0 + b]);
      fin[b] = a.fin ? a.fin[r0 + b] : 0;
    }
  }
  if (tid == 0) {
    bv = 0;
    bi = 0;
    cnt = 0;
    nsel = 0;
  }
  __syncthreads();
  auto value = [&](int b, uint64_t key, uint64_t& v, uint64_t& i) {
    v = 0;
    i = 0;
    if (!key) return;
    v = ord64((double)sc[b] + ((double)unord32((uint32_t)(key >> 32)) - lse[b]));
    i = (uint64_t)(BS_BMAX - 1 - b) << (32 + BS_TBITS) | key >> 32 << BS_TBITS |
        ((uint32_t)key & ((1u << BS_TBITS) - 1));
  };
  // a bound on the k-th best of the threads' best list heads, and the lists that reach it
  uint64_t mv, mi;
  value(l0 / a.nseg, head, mv, mi);
  for (int l = l0 + BS_THREADS; l < lists; l += BS_THREADS) {
    uint64_t v, i;
    value(l / a.nseg, __ldcg(cand + (size_t)l * a.k), v, i);
    if (over(v, i, mv, mi)) {
      mv = v;
      mi = i;
    }
  }
  uint64_t Tv = (uint64_t)low_bound((uint32_t)(mv >> 32), a.k, lows) << 32, Ti = 0;
  for (int l = l0; l < lists; l += BS_THREADS) {
    uint64_t v, i;
    value(l / a.nseg, l == l0 ? head : __ldcg(cand + (size_t)l * a.k), v, i);
    if (v && v >= Tv) {
      const int c = atomicAdd(&nsel, 1);
      if (c < BS_THREADS) sel[c] = l;
    }
  }
  __syncthreads();
  // the elements of ns lists that reach the bound; whether there was room for them
  auto gather = [&](int ns) {
    bool fits = true;
    for (int e = tid; e < ns * a.k; e += BS_THREADS) {
      const int l = sel[e / a.k];
      uint64_t v, i;
      value(l / a.nseg, __ldcg(cand + (size_t)l * a.k + e % a.k), v, i);
      if (v && !over(Tv, Ti, v, i)) {
        const int c = atomicAdd(&cnt, 1);
        fits &= c < cap;
        if (c < cap) best[c] = make_ulonglong2(v, i);
      }
    }
    return !__syncthreads_or(!fits);
  };
  const int ns = nsel;
  if (ns > BS_THREADS || !gather(ns)) {  // too many: the exact k-th best of the threads' best ...
    tv[tid] = mv;
    ti[tid] = mi;
    __syncthreads();
    if (tid == 0) nsel = cnt = 0;
    int above = 0;
    for (int j = 0; j < BS_THREADS; j++) above += over(tv[j], ti[j], mv, mi);
    if (mv && above == a.k - 1) {
      bv = mv;
      bi = mi;
    }
    __syncthreads();
    Tv = bv;
    Ti = bi;
    // ... and, where a thread has several lists, of the heads that reach it
    if (lists > BS_THREADS) {
      for (int l = tid; l < lists; l += BS_THREADS) {
        uint64_t v, i;
        value(l / a.nseg, __ldcg(cand + (size_t)l * a.k), v, i);
        if (v && !over(Tv, Ti, v, i)) {
          best[atomicAdd(&cnt, 1)] = make_ulonglong2(v, i);
        }
      }
      __syncthreads();
      const int n = cnt;
      for (int c = tid; c < n; c += BS_THREADS) {
        const ulonglong2 x = best[c];
        int r = 0;
        for (int j = 0; j < n; j++) r += over(best[j].x, best[j].y, x.x, x.y);
        if (r == a.k - 1) {
          bv = x.x;
          bi = x.y;
        }
      }
      __syncthreads();
      Tv = bv;
      Ti = bi;
      if (tid == 0) cnt = 0;
    }
    for (int l = tid; l < lists; l += BS_THREADS) {
      uint64_t v, i;
      value(l / a.nseg, __ldcg(cand + (size_t)l * a.k), v, i);
      if (v && !over(Tv, Ti, v, i)) sel[atomicAdd(&nsel, 1)] = l;
    }
    __syncthreads();
    gather(nsel);  // at most k lists, k * k elements
  }
  int n = cnt;
  if (n > 2 * a.k && n <= BS_THREADS) {  // a bound from all of them, and what reaches it, to the front
    const ulonglong2 x = tid < n ? best[tid] : make_ulonglong2(0, 0);
    const uint64_t low = (uint64_t)low_bound((uint32_t)(x.x >> 32), a.k, lows2) << 32;
    if (tid == 0) cnt = 0;  // (the bound's barrier is past every read)
    __syncthreads();
    if (x.x && x.x >= low) best[atomicAdd(&cnt, 1)] = x;
    __syncthreads();
    n = cnt;
  }
  for (int c = tid; c < n; c += BS_THREADS) {
    const uint64_t v = best[c].x, i = best[c].y;
    int r = 0;
#pragma unroll 4
    for (int j = 0; j < n; j++) {
      const ulonglong2 x = best[j];
      r += over(x.x, x.y, v, i);
    }
    if (r < a.k) {
      const int b = BS_BMAX - 1 - (int)(i >> (32 + BS_TBITS));
      const int t = (int)((1u << BS_TBITS) - 1 - ((uint32_t)i & ((1u << BS_TBITS) - 1)));
      const size_t o = (size_t)g * a.k + r;
      a.out_s[o] = (float)unord64(v);
      a.out_p[o] = b;
      a.out_t[o] = t;
      if (a.out_f) a.out_f[o] = fin[b] || t == a.eos;
    }
  }
}

// PER: elements a thread takes at a time, 8 or 16.
template <int PER>
__global__ void __launch_bounds__(BS_THREADS, 4) k_beam_select(const BeamArgs a) {
  constexpr float LOG2E = 1.4426950408889634f;
  constexpr int TILE = BS_THREADS * PER;
  extern __shared__ __align__(16) uint8_t raw[];
  uint64_t* list = reinterpret_cast<uint64_t*>(raw);  // [BS_CAP], then beam_pick's
  __shared__ __align__(16) uint64_t keys[BS_THREADS], keys2[BS_THREADS];
  __shared__ uint64_t kth;
  __shared__ uint32_t lows[2][BS_WARPS];
  __shared__ int cnt, kept;
  __shared__ float2 red[BS_WARPS];
  const int row = blockIdx.y, seg = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int base = seg * a.tiles * BS_TILE, end = min(a.vocab, base + a.tiles * BS_TILE);
  if (tid == 0) cnt = 0;
  griddep_wait();
  const bool fin = a.fin && a.fin[row];
  const float* xr = a.x + (long long)row * a.ld;
  // element e of a thread's tile is at place(t, e): float4s
  auto place = [&](int t, int e) { return base + t * TILE + ((e >> 2) * BS_THREADS + tid) * 4 + (e & 3); };
  auto load = [&](int t, float (&v)[PER]) {
#pragma unroll
    for (int h = 0; h < PER; h += 4) {
      const int i = place(t, h);
      if (a.vec && i + 4 <= end) {
        const float4 f = __ldg(reinterpret_cast<const float4*>(xr + i));
        v[h] = f.x;
        v[h + 1] = f.y;
        v[h + 2] = f.z;
        v[h + 3] = f.w;
      } else {
#pragma unroll
        for (int e = 0; e < 4; e++) v[h + e] = i + e < end ? __ldg(xr + i + e) : -INFINITY;
      }
    }
  };
  // a finished beam's logits are not read: eos first, where it is in the segment, then the
  // lowest tokens
  const int nt = fin ? 0 : (end - base + TILE - 1) / TILE;
  float m = -INFINITY, s = 0.0f;
  uint64_t T = 1;        // (no key is 0)
  float Tf = -INFINITY;  // the least value whose keys reach T
  uint32_t top = 0;      // ordered bits of the thread's largest element
  bool overflow = false;
  float v[PER], w[PER];
  if (nt) load(0, v);
  for (int t = 0; t < nt; t++) {
    if (t + 1 < nt) load(t + 1, w);
    float mt = -INFINITY;
#pragma unroll
    for (int e = 0; e < PER; e++) {
      v[e] = tame(v[e]);
      mt = fmaxf(mt, v[e]);
    }
    if (mt > m + 20.0f) {  // (also from -inf)
      s *= m > -INFINITY ? ex2f((m - mt) * LOG2E) : 0.0f;
      m = mt;
    }
    if (m > -INFINITY) {
      float p[PER];
#pragma unroll
      for (int e = 0; e < PER; e++) p[e] = ex2f((v[e] - m) * LOG2E);
#pragma unroll
      for (int o = 1; o < PER; o <<= 1)
#pragma unroll
        for (int e = 0; e < PER; e += 2 * o) p[e] += p[e + o];
      s += p[0];
    }
    const uint32_t here = place(t, 0) < end ? ord32(mt) : 0;
    top = max(top, here);
    if (t == 0) T = max(T, (uint64_t)low_bound(here, a.k, lows[0]) << 32);
    if (t == 0) Tf = T > 1 ? unord32((uint32_t)(T >> 32)) : -INFINITY;
    if (mt >= Tf) {
#pragma unroll
      for (int e = 0; e < PER; e++)
        if (v[e] >= Tf) {
          const int i = place(t, e);
          if (i < end) {
            const int c = atomicAdd(&cnt, 1);
            if (c < BS_CAP) list[c] = (uint64_t)ord32(v[e]) << 32 | (uint32_t)~i;
            else overflow = true;
          }
        }
    }
#pragma unroll
    for (int e = 0; e < PER; e++) v[e] = w[e];
  }
  if (__syncthreads_or(overflow)) {  // once more, in tiles of 2048 with an exact bound after each
    T = 1;
    if (tid == 0) cnt = 0;
    __syncthreads();
    for (int t = 0; t < a.tiles; t++) {
      uint64_t x[12], best = 0;
      for (int e = 0; e < 8; e++) {
        const int i = base + t * BS_TILE + e * BS_THREADS + tid;
        x[e] = 0;
        if (i < end) {
          const float f = tame(__ldg(xr + i));
          x[e] = (uint64_t)ord32(f) << 32 | (uint32_t)~i;
        }
        best = max(best, x[e]);
      }
      if (t == 0) T = max(T, kth_key(best, a.k, keys, &kth));
      for (int e = 0; e < 8; e++)
        if (x[e] >= T) list[atomicAdd(&cnt, 1)] = x[e];
      __syncthreads();
      const int n = cnt;
      __syncthreads();
      if (n > BS_LIST) {  // what reaches the k-th largest of the threads' maxima: at most 12 k
        best = 0;
        for (int e = 0; e < 12; e++) {
          x[e] = e * BS_THREADS + tid < n ? list[e * BS_THREADS + tid] : 0;
          best = max(best, x[e]);
        }
        T = max(T, kth_key(best, a.k, keys, &kth));
        if (tid == 0) cnt = 0;
        __syncthreads();
        for (int e = 0; e < 12; e++)
          if (x[e] >= T) list[atomicAdd(&cnt, 1)] = x[e];
        __syncthreads();
      }
    }
  }
  // (max, sum) of the segment
  const float wm = warp_max(m);
  const float ws = warp_sum(m > -INFINITY ? s * ex2f((m - wm) * LOG2E) : 0.0f);
  if (lane == 0) red[warp] = make_float2(wm, ws);
  // the list, less what the whole segment's bound excludes, ranked
  T = max(T, (uint64_t)low_bound(top, a.k, lows[1]) << 32);
  int n = cnt;
  uint64_t* out = a.cand + ((size_t)row * a.nseg + seg) * a.k;
  const uint64_t* final = list;
  if (n > 32) {
    if (tid == 0) kept = 0;
    __syncthreads();
    for (int i = tid; i < n; i += BS_THREADS) {
      const uint64_t x = list[i];
      if (x >= T) {
        const int c = atomicAdd(&kept, 1);
        if (c < BS_THREADS) keys[c] = x;
      }
    }
    __syncthreads();
    if (kept <= BS_THREADS) {
      n = kept;
      final = keys;
    }
  }
  for (int i = tid; i < n; i += BS_THREADS) {
    const uint64_t x = final[i];
    int r = 0;
#pragma unroll 8
    for (int j = 0; j < n; j++) r += final[j] > x;
    if (r < a.k) out[r] = x;
  }
  // (fewer than k elements are listed only where the segment has no more)
  for (int i = n + tid; i < a.k && !fin; i += BS_THREADS) out[i] = 0;
  const bool has = fin && a.eos >= base && a.eos < end;
  if (fin && tid < a.k) {
    int i = base + tid - has;
    i += has && i >= a.eos;
    out[tid] = has && tid == 0 ? (uint64_t)ord32(0.0f) << 32 | (uint32_t)~a.eos
               : i < end       ? (uint64_t)ord32(-INFINITY) << 32 | (uint32_t)~i
                               : 0;
  }
  if (fin && tid == 0) {
    a.part[(size_t)row * a.nseg + seg] = has ? make_float2(0.0f, 1.0f) : make_float2(-INFINITY, 0.0f);
  } else if (tid == 0) {
    float M = red[0].x, t = 0.0f;
#pragma unroll
    for (int i = 1; i < BS_WARPS; i++) M = fmaxf(M, red[i].x);
#pragma unroll
    for (int i = 0; i < BS_WARPS; i++)
      if (red[i].x > -INFINITY) t += red[i].y * ex2f((red[i].x - M) * LOG2E);
    a.part[(size_t)row * a.nseg + seg] = make_float2(M, t);
  }
  __syncthreads();
  const int g = row / a.beams;
  if (tid == 0) {
    __threadfence();
    cnt = atomicAdd(&a.cnt[g], 1);
    __threadfence();
  }
  __syncthreads();
  griddep_launch();
  if (cnt != a.beams * a.nseg - 1) return;
  if (tid == 0) a.cnt[g] = 0;
  beam_pick(a, g, raw, keys, keys2);
}

// Elements that beam_pick needs room for, with segments of t tiles: k lists of k, or the heads that
// reach the threads' k-th best.
size_t beam_cap(size_t beams, size_t vocab, size_t k, int t) {
  const size_t seg = (size_t)BS_TILE * t, lists = beams * ((vocab + seg - 1) / seg);
  return std::max({k * k, k * ((lists + BS_THREADS - 1) / BS_THREADS), (size_t)BS_CAP / 2});
}
constexpr size_t BS_SMEM = 200 * 1024;

// Tiles of a segment: as few as give at most two CTAs on every SM (which has room for four),
// at most 8 (uneven waves then cost less than longer segments save) unless a group's
// lists would not fit (64 beams and continuations of 13 million tokens or more).
int beam_tiles(size_t rows, size_t beams, size_t vocab, size_t k, int sms) {
  const size_t tiles = (vocab + BS_TILE - 1) / BS_TILE;
  int t = 1;
  while (t < 8 && rows * ((tiles + t - 1) / t) > 2 * (size_t)sms) t++;
  while (beam_cap(beams, vocab, k, t) * 2 * sizeof(uint64_t) > BS_SMEM) t++;
  return t;
}
constexpr size_t BS_GROUPS = 65536;  // arrival counters, at the front of the scratch

// A few numbers a step; in the step's graph, so that nothing of it changes with the position.
__global__ void k_beam_note(int* len, const int* slots, int n, int advance, const int32_t* tok,
                            const int32_t* par, int32_t* hist, int32_t* hist_parent, int ld) {
  griddep_wait();
  griddep_launch();
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const int s = slots[i], at = len[s] + advance;
    if (at < ld) {
      hist[(size_t)s * ld + at] = tok[i];
      hist_parent[(size_t)s * ld + at] = par[i];
      len[s] = at;
    }
  }
}

}  // namespace

syn_status_t launch_beam_note(syn_cuda_kvcache_t* c, const int* slots, size_t n, int advance,
                              const int32_t* tok, const int32_t* par, int32_t* hist,
                              int32_t* hist_parent, int ld, cudaStream_t st) {
  return launched(launch_pdl(k_beam_note, dim3(1), dim3(64), 0, st, c->d_len, slots, (int)n, advance,
                             tok, par, hist, hist_parent, ld),
                  "k_beam_note");
}

syn_status_t more_smem(const void* fn, size_t bytes) {
  static std::mutex mu;
  static std::map<std::pair<const void*, int>, size_t> granted;
  int dev = 0;
  SYN_CUDA_TRY(cudaGetDevice(&dev));
  std::lock_guard<std::mutex> g(mu);
  size_t& has = granted[{fn, dev}];
  if (bytes <= has) return SYN_OK;
  SYN_CUDA_TRY(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
  has = bytes;
  return SYN_OK;
}

syn_status_t kv_copy_page(syn_cuda_kvcache_t* c, int src, int dst, size_t rows, cudaStream_t st) {
  const size_t row4 = c->n_kv * c->hd / 4, page4 = c->page * row4;
  const size_t n4 = rows * row4;
  if (!n4) return SYN_OK;
  for (size_t l0 = 0; l0 < c->layers; l0 += 32768) {
    const unsigned nl = (unsigned)std::min<size_t>(c->layers - l0, 32768);
    const size_t layer4 = c->n_pages * page4;
    k_kv_copy_page<<<dim3((unsigned)std::min<size_t>(8, (n4 + 255) / 256), nl, 2), 256, 0, st>>>(
        reinterpret_cast<float4*>(c->k) + l0 * layer4, reinterpret_cast<float4*>(c->v) + l0 * layer4,
        layer4, src * page4, dst * page4, n4);
  }
  SYN_LAUNCH_CHECK("k_kv_copy_page");
  return SYN_OK;
}

syn_status_t no_free_page() {
  set_last_cuda_error(cudaErrorMemoryAllocation, "paged KV cache: no free page");
  return SYN_ERR_OUT_OF_MEMORY;
}

syn_status_t kv_own_page(syn_cuda_kvcache_t* c, size_t seq, cudaStream_t st) {
  // (a reorder leaves private last pages, and kv_release sees to it that one by a graph finds them so)
  return c->page && c->stale[seq] ? SYN_OK : kv_copy_shared(c, seq, st);
}

syn_status_t kv_cut(syn_cuda_kvcache_t* c, size_t seq, size_t new_len, cudaStream_t st) {
  if (!c->page || c->stale[seq] != 2 || new_len % c->page == 0) return SYN_OK;
  syn_status_t s = kv_sync(c, st);
  if (s) return s;
  const int* row = c->ptab_h + seq * c->maxp;
  const size_t col = new_len / c->page;
  if (row[col] < 0 || c->refs[row[col]] <= 1) return SYN_OK;
  size_t free = c->n_free;
  for (size_t i = col + 1; i < c->maxp; i++) free += row[i] >= 0 && c->refs[row[i]] == 1;
  return free ? SYN_OK : no_free_page();
}

syn_status_t kv_copy_shared(syn_cuda_kvcache_t* c, size_t seq, cudaStream_t st) {
  if (!c->page) return SYN_OK;
  const size_t col = c->len[seq] / c->page;
  if (col >= c->maxp) return SYN_OK;
  int* e = c->ptab_h + seq * c->maxp + col;
  if (*e < 0 || c->refs[*e] <= 1) return SYN_OK;
  if (capturing(st)) return SYN_ERR_UNSUPPORTED;  // a replay would copy again
  if (!c->n_free) {  // (those of dropped beams are counted only when a table is read back)
    syn_status_t s = kv_sync(c, st);
    if (s) return s;
    if (c->refs[*e] <= 1) return SYN_OK;
    if (!c->n_free) return no_free_page();
  }
  const int old = *e, own = c->free_pages[c->n_free - 1];
  syn_status_t s = kv_copy_page(c, old, own, c->len[seq] % c->page, st);
  if (s) return s;
  c->n_free--;
  c->refs[old]--;
  c->refs[own] = 1;
  *e = own;
  kv_changed(c, seq, st);
  SYN_CUDA_TRY(cudaMemcpyAsync(c->d_ptab + seq * c->maxp + col, e, sizeof(int),
                               cudaMemcpyHostToDevice, st));
  return SYN_OK;
}

void kv_changed(syn_cuda_kvcache_t* c, size_t seq, cudaStream_t st) {
  c->shrunk[seq]++;
  plans_changed(c, seq, st);
}

syn_status_t kv_sync(syn_cuda_kvcache_t* c, cudaStream_t st) {
  if (!c->page || !c->n_stale) return SYN_OK;
  if (capturing(st)) return SYN_ERR_UNSUPPORTED;
  SYN_CUDA_TRY(cudaDeviceSynchronize());
  const size_t entries = c->batch * c->maxp;
  SYN_CUDA_TRY(cudaMemcpy(c->ptab_h, c->d_ptab, entries * sizeof(int), cudaMemcpyDeviceToHost));
  std::fill(c->refs, c->refs + c->n_pages, 0);
  for (size_t i = 0; i < entries; i++)
    if (c->ptab_h[i] >= 0) c->refs[c->ptab_h[i]]++;
  c->n_free = 0;
  for (size_t p = c->n_pages; p-- > 0;)
    if (!c->refs[p]) c->free_pages[c->n_free++] = (int)p;
  c->n_stale = 0;
  for (size_t b = 0; b < c->batch; b++) {
    if (c->stale[b] == 1) c->stale[b] = 0;
    c->n_stale += c->stale[b] != 0;  // (2: permuted by a captured graph, at any time)
  }
  return SYN_OK;
}

syn_status_t launch_kv_reorder(syn_cuda_kvcache_t* c, size_t n, const int32_t* seqs,
                               const int32_t* parents, size_t beams, const size_t* lens,
                               cudaStream_t st) {
  ReorderArgs a;
  a.k = reinterpret_cast<float4*>(c->k);
  a.v = reinterpret_cast<float4*>(c->v);
  a.row4 = (int)(c->n_kv * c->hd / 4);
  a.layer4 = c->n_pages * c->page * a.row4;
  a.ptab = c->d_ptab;
  a.done = c->d_ptab + c->batch * c->maxp;
  a.maxp = (int)c->maxp;
  a.page = (int)c->page;
  a.max_seq = (int)c->max_seq;
  a.parents = parents;
  a.len = c->d_len;
  a.n = (int)n;
  a.beams = (int)beams;
  size_t cols = 0, tail = 0;
  for (size_t i = 0; i < n; i++) a.seq[i] = seqs[i];
  for (size_t g = 0; g < n / beams; g++) {
    cols = std::max(cols, (lens[g] + c->page - 1) / c->page);
    tail = std::max(tail, lens[g] % c->page);
  }
  if (capturing(st)) tail = c->page - 1;  // (a replay's may be any)
  else if (!cols) return SYN_OK;
  if (c->layers > 65534) return SYN_ERR_UNSUPPORTED;
  // about four 16-byte copies a thread, K and V: 28 layers x 20 beams x 28 rows of 4 KB (257 MB
  // read and written) take 39 us; one copy a thread takes 64
  const unsigned ch = (unsigned)std::max<size_t>(1, std::min<size_t>(16, (tail * a.row4 + 1023) / 1024));
  return launched(launch_pdl(k_reorder, dim3(ch, (unsigned)n, (unsigned)c->layers + 1), dim3(256), 0, st, a),
                  "k_reorder");
}

syn_status_t launch_append_batch(const AttnArgs& at, float* q_out, size_t ldq, size_t n,
                                 const int32_t* seqs, const size_t* counts, cudaStream_t st) {
  size_t done = 0;
  for (size_t i0 = 0; i0 < n; i0 += AP_MAX) {
    AppendArgs a = append_args(at, q_out, ldq, done);
    a.n = (int)std::min<size_t>(AP_MAX, n - i0);
    size_t rows = 0;
    for (int i = 0; i < a.n; i++) {
      a.seq[i] = seqs[i0 + i];
      a.row0[i] = (int)rows;
      rows += counts[i0 + i];
    }
    a.row0[a.n] = (int)rows;
    a.rows = (int)rows;
    if (rows) {
      const AppendShape sh = append_shape(a);
      // two heads a lane group once that still fills the device
      const size_t heads = a.n_heads + 2 * a.n_kv, per = AP_THREADS / sh.lp;
      const bool many = sh.one && rows * heads >= 2 * per * AP_FILL;
      void (*kern)(const AppendArgs) = !sh.vec   ? k_append_batch<1, 32, false, 1>
                                       : !sh.one ? k_append_batch<4, 32, false, 1>
                                       : many    ? append_kernel<2>(sh.lp)
                                                 : append_kernel<1>(sh.lp);
      const size_t units = rows * (many ? (heads + 1) / 2 : heads), blocks = (units + per - 1) / per;
      if (blocks > 0x7FFFFFFF) return SYN_ERR_UNSUPPORTED;
      syn_status_t s = launched(launch_pdl(kern, dim3((unsigned)blocks), dim3(AP_THREADS), 0, st, a),
                                "k_append_batch");
      if (s) return s;
    }
    done += rows;
  }
  return SYN_OK;
}

size_t beam_scratch_bytes(size_t rows, size_t beams, size_t vocab, size_t k, int sms) {
  const size_t seg = (size_t)BS_TILE * beam_tiles(rows, beams, vocab, k, sms), nseg = (vocab + seg - 1) / seg;
  return BS_GROUPS * sizeof(int) + rows * nseg * (k * sizeof(uint64_t) + sizeof(float2));
}

syn_status_t launch_beam_select(const float* x, size_t ld, size_t groups, size_t beams,
                                size_t vocab, const float* scores, const uint8_t* fin, int eos,
                                size_t k, float* out_s, int32_t* out_p, int32_t* out_t,
                                uint8_t* out_f, void* scratch, int sms, cudaStream_t st) {
  const size_t rows = groups * beams;
  BeamArgs a;
  a.x = x;
  a.ld = (long long)ld;
  a.beams = (int)beams;
  a.vocab = (int)vocab;
  a.k = (int)k;
  a.tiles = beam_tiles(rows, beams, vocab, k, sms);
  a.nseg = (int)((vocab + (size_t)BS_TILE * a.tiles - 1) / ((size_t)BS_TILE * a.tiles));
  a.vec = ld % 4 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0;
  a.scores = scores;
  a.fin = fin;
  a.eos = eos;
  a.cnt = static_cast<int*>(scratch);
  a.cand = reinterpret_cast<uint64_t*>(a.cnt + BS_GROUPS);
  a.part = reinterpret_cast<float2*>(a.cand + rows * a.nseg * k);
  a.out_s = out_s;
  a.out_p = out_p;
  a.out_t = out_t;
  a.out_f = out_f;
  const size_t cap = beam_cap(beams, vocab, k, a.tiles), smem = cap * 2 * sizeof(uint64_t);
  a.cap = (int)cap;
  void (*kern)(const BeamArgs) = a.tiles > 2 ? k_beam_select<16> : k_beam_select<8>;
  if (smem > 40 * 1024) {
    syn_status_t s = more_smem((const void*)kern, BS_SMEM);
    if (s) return s;
  }
  return launched(launch_pdl(kern, dim3((unsigned)a.nseg, (unsigned)rows), dim3(BS_THREADS), smem, st, a),
                  "k_beam_select");
}

}  // namespace syn

using namespace syn;

extern "C" {

syn_status_t syn_cuda_kvcache_pool(const syn_cuda_kvcache_t* c, size_t layer, float** k, float** v) {
  if (!c) return SYN_ERR_NULL_PTR;
  if (layer >= c->layers) return SYN_ERR_INVALID_ARG;
  if (!c->page) return SYN_ERR_UNSUPPORTED;
  const size_t off = layer * c->n_pages * c->page * c->n_kv * c->hd;
  if (k) *k = c->k + off;
  if (v) *v = c->v + off;
  return SYN_OK;
}

syn_status_t syn_cuda_kvcache_page_table(const syn_cuda_kvcache_t* c, const int32_t** table,
                                         size_t* pages_per_seq) {
  if (!c) return SYN_ERR_NULL_PTR;
  if (!c->page) return SYN_ERR_UNSUPPORTED;
  if (table) *table = c->d_ptab;
  if (pages_per_seq) *pages_per_seq = c->maxp;
  return SYN_OK;
}

syn_status_t syn_cuda_kvcache_fork(syn_cuda_kvcache_t* c, size_t src, size_t dst, size_t len,
                                   void* stream) {
  if (!c) return SYN_ERR_NULL_PTR;
  if (!c->page) return SYN_ERR_UNSUPPORTED;
  if (src >= c->batch || dst >= c->batch || src == dst || len > c->len[src] || c->len[dst])
    return SYN_ERR_INVALID_ARG;
  DeviceGuard g(c->device);
  if (!g.ok) return SYN_ERR_CUDA;
  cudaStream_t st = (cudaStream_t)stream;
  if (capturing(st)) return SYN_ERR_UNSUPPORTED;  // the tables are kept on the host
  syn_status_t s = kv_sync(c, st);
  if (s) return s;
  int *from = c->ptab_h + src * c->maxp, *to = c->ptab_h + dst * c->maxp;
  if (to[0] >= 0 && (s = kv_release(c, dst, 0, st))) return s;  // pages taken for a call, never committed
  const size_t full = len / c->page, tail = len % c->page;
  if (tail && !c->n_free) return no_free_page();
  for (size_t i = 0; i < full; i++) {
    to[i] = from[i];
    c->refs[to[i]]++;
  }
  if (tail) {
    to[full] = c->free_pages[--c->n_free];
    c->refs[to[full]] = 1;
    if ((s = kv_copy_page(c, from[full], to[full], tail, st))) return s;
  }
  kv_changed(c, dst, st);
  if (len)
    SYN_CUDA_TRY(cudaMemcpyAsync(c->d_ptab + dst * c->maxp, to, (full + (tail != 0)) * sizeof(int),
                                 cudaMemcpyHostToDevice, st));
  if ((s = launch_kv_set(c, dst, (int)len, 0, st))) return s;
  c->len[dst] = len;
  return SYN_OK;
}

syn_status_t syn_cuda_kvcache_reorder(syn_cuda_kvcache_t* c, size_t n, const int32_t* seqs,
                                      const int32_t* parents, size_t beams, void* stream) try {
  if (!c || !seqs || !parents) return SYN_ERR_NULL_PTR;
  if (!c->page) return SYN_ERR_UNSUPPORTED;
  if (!n) return SYN_OK;
  if (!beams || n % beams) return SYN_ERR_SHAPE_MISMATCH;
  std::vector<uint8_t> seen(c->batch, 0);
  for (size_t i = 0; i < n; i++) {
    if (seqs[i] < 0 || (size_t)seqs[i] >= c->batch || seen[seqs[i]]) return SYN_ERR_INVALID_ARG;
    seen[seqs[i]] = 1;
    if (c->len[seqs[i]] != c->len[seqs[i - i % beams]]) return SYN_ERR_INVALID_ARG;
  }
  if (beams > RO_MAX) return SYN_ERR_UNSUPPORTED;
  if (beams == 1) return SYN_OK;
  DeviceGuard g(c->device);
  if (!g.ok) return SYN_ERR_CUDA;
  cudaStream_t st = (cudaStream_t)stream;
  syn_status_t s;
  for (size_t i = 0; i < n; i++)
    if ((s = kv_own_page(c, seqs[i], st))) return s;
  const bool captured = capturing(st);
  for (size_t i = 0; i < n; i += beams) {
    plans_reordered(c, seqs + i, beams, st);
    std::vector<int32_t> mix(seqs + i, seqs + i + beams);
    std::sort(mix.begin(), mix.end());
    if (captured && std::find(c->mixes.begin(), c->mixes.end(), mix) == c->mixes.end())
      c->mixes.push_back(std::move(mix));
  }
  if (captured) plans_mixed(c, st);
  const size_t per = RO_MAX / beams * beams;
  for (size_t i0 = 0; i0 < n; i0 += per) {
    const size_t m = std::min(per, n - i0);
    size_t lens[RO_MAX];
    for (size_t i = 0; i < m; i += beams) lens[i / beams] = c->len[seqs[i0 + i]];
    if ((s = launch_kv_reorder(c, m, seqs + i0, parents + i0, beams, lens, st))) return s;
  }
  const uint8_t mark = captured ? 2 : 1;
  for (size_t i = 0; i < n; i++) {
    c->n_stale += !c->stale[seqs[i]];
    c->stale[seqs[i]] = std::max(c->stale[seqs[i]], mark);
  }
  return SYN_OK;
} catch (const std::bad_alloc&) {
  return SYN_ERR_OUT_OF_MEMORY;
}

syn_status_t syn_cuda_qk_norm_rope_kv_append_batch(
    syn_cuda_kvcache_t* c, size_t layer, size_t n_seqs, const int32_t* seqs, const size_t* n_tokens,
    const float* q, const float* k, const float* v, size_t ld, size_t n_heads, const float* q_norm,
    const float* k_norm, float eps, const float* rope_cos, const float* rope_sin, float* q_out,
    size_t ldq, void* stream) try {
  if (!c || !seqs || !n_tokens || !q || !k || !v || !rope_cos || !rope_sin || !q_out)
    return SYN_ERR_NULL_PTR;
  if (layer >= c->layers) return SYN_ERR_INVALID_ARG;
  if (!n_heads || n_heads % c->n_kv) return SYN_ERR_SHAPE_MISMATCH;
  std::vector<uint8_t> seen(c->batch, 0);
  size_t rows = 0;
  for (size_t i = 0; i < n_seqs; i++) {
    if (seqs[i] < 0 || (size_t)seqs[i] >= c->batch || seen[seqs[i]]) return SYN_ERR_INVALID_ARG;
    seen[seqs[i]] = 1;
    if (n_tokens[i] > c->max_seq || c->len[seqs[i]] + n_tokens[i] > c->max_seq)
      return SYN_ERR_INVALID_ARG;  // CacheFull
    rows += n_tokens[i];
  }
  if (!rows) return SYN_OK;
  if (rows > 0x7FFFFFFF) return SYN_ERR_UNSUPPORTED;
  if (ld < c->hd || ldq < n_heads * c->hd) return SYN_ERR_SHAPE_MISMATCH;
  DeviceGuard g(c->device);
  if (!g.ok) return SYN_ERR_CUDA;
  cudaStream_t st = (cudaStream_t)stream;
  syn_status_t s;
  for (size_t i = 0; i < n_seqs; i++)
    if (n_tokens[i] && (s = kv_reserve(c, seqs[i], c->len[seqs[i]] + n_tokens[i], st))) return s;
  AttnArgs a{const_cast<float*>(q), k, v, ld, n_heads, q_norm, k_norm, eps, rope_cos, rope_sin, 0, c,
             layer, nullptr, 0};
  return launch_append_batch(a, q_out, ldq, n_seqs, seqs, n_tokens, st);
} catch (const std::bad_alloc&) {
  return SYN_ERR_OUT_OF_MEMORY;
}

syn_status_t syn_cuda_beam_select(syn_cuda_ctx_t* ctx, const float* logits, size_t ld,
                                  size_t groups, size_t beams, size_t vocab, const float* scores,
                                  const uint8_t* finished, int32_t eos, size_t k, float* out_scores,
                                  int32_t* out_parents, int32_t* out_tokens, uint8_t* out_finished,
                                  void* stream) try {
  if (!ctx || !logits || !scores || !out_scores || !out_parents || !out_tokens)
    return SYN_ERR_NULL_PTR;
  if (!groups) return SYN_OK;
  if (!beams || !vocab || !k) return SYN_ERR_INVALID_DIMENSIONS;
  if (ld < vocab) return SYN_ERR_SHAPE_MISMATCH;
  if (beams > BS_BMAX || k > BS_KMAX || vocab > 1u << BS_TBITS || groups > 0x7FFFFFFF ||
      groups * beams > 65535)
    return SYN_ERR_UNSUPPORTED;
  if (k > beams * vocab) return SYN_ERR_INVALID_ARG;
  if (finished && (eos < 0 || (size_t)eos >= vocab)) return SYN_ERR_INVALID_ARG;
  DeviceGuard g(ctx->device);
  if (!g.ok) return SYN_ERR_CUDA;
  cudaStream_t st = (cudaStream_t)stream;
  const size_t bytes = beam_scratch_bytes(groups * beams, beams, vocab, k, ctx->sms);
  const bool captured = capturing(st);
  if (bytes > ctx->beam_bytes && ctx->beam_captured && !captured) {
    ctx->beam_kept.push_back(ctx->beam);
    ctx->beam = nullptr;
    ctx->beam_bytes = 0;
    ctx->beam_captured = false;
  }
  syn_status_t s = grow_scratch(&ctx->beam, &ctx->beam_bytes, bytes, st);
  if (s) return s;
  ctx->beam_captured |= captured;
  return launch_beam_select(logits, ld, groups, beams, vocab, scores, finished, eos, k, out_scores,
                            out_parents, out_tokens, out_finished, ctx->beam, ctx->sms, st);
} catch (const std::bad_alloc&) {
  return SYN_ERR_OUT_OF_MEMORY;
}

}  // extern "C"
