// shared_attn.cu -- decode attention for a batch whose sequences share their
// leading cache pages (syn_cuda_kvcache_fork): beams of a prompt, samples of a
// document, users behind one system prompt. For one query row with scores
// s_j = q.k_j / sqrt(hd) over its positions,
//   o = sum_j e^{s_j} v_j / sum_j e^{s_j},
// and any partition of the positions into parts with (m_i, l_i, o_i) = (max,
// sum of e^{s-m_i}, sum of e^{s-m_i} v) joins as M = max m_i,
//   o = sum_i e^{m_i-M} o_i / sum_i e^{m_i-M} l_i.
// The shared prefix of a group is one part set, computed once for all its
// rows, so its K and V cross HBM once per step instead of once per row; each
// row's own positions are the other. Kernels of one call:
//   k_begin   the new rows normalised, rotated and appended; k_span's shares
//   k_prefix  the shared prefixes of many query rows, on the tensor cores and a
//             schedule made on the host
//   k_span    each row's own positions, and the shared prefixes of few query
//             rows
//   k_join    the parts of each query row
#include <math.h>

#include <algorithm>
#include <map>
#include <new>
#include <type_traits>
#include <vector>

#include "append.cuh"
#include "internal.cuh"
#include "tcgen05.cuh"

// A group's rows share their leading positions: who holds those pages. A reorder among holders
// leaves every row with them; one that brings in another sequence's context does not.
struct PlanFamily {
  size_t len;                  // shared positions
  std::vector<uint8_t> holds;  // [batch]: 1, and 2 for those that the group depends on (its rows, and
};                             // whatever a captured reorder may exchange with them)

// A batch of decode rows in groups. Built on the host by _set: which leading
// pages each group shares, and the schedule of its prefix work.
struct syn_cuda_decode_plan_s {
  syn_cuda_kvcache_t* cache;
  int device, sms;
  size_t n_heads;
  size_t rows = 0, groups = 0;
  std::vector<int32_t> seqs;
  std::vector<PlanFamily> families;    // of the groups that share
  bool parted = false;                 // a reorder since _set has taken what a group shared from it
  int* err = nullptr;                  // device: where the public calls' kernels record what failed
  std::vector<size_t> prefix, shrunk;  // per row: shared positions; the sequence's state at _set
  // device
  float* q = nullptr;        // rotated queries [batch][n_heads * hd]
  uint8_t* qparts = nullptr; // k_prefix's: as fp16 parts, job by job (QParts)
  float* qup = nullptr;      // their rows' scales
  int* meta = nullptr;       // MetaView, copied from meta_h
  int* meta_h = nullptr;     // pinned
  cudaEvent_t copied = nullptr;
  size_t meta_ints = 0;
  float* po = nullptr;       // partial o, prefix then suffix
  float2* pml = nullptr;     // partial (m, l)
  size_t part_rows = 0;      // records of po / pml
  void* shares = nullptr;    // k_span's shares and jobs (Share, SpanJob), written by k_begin
  int units = 0, span_jobs = 0, jobs = 0;  // k_span's units and jobs; k_prefix's jobs
  int prefix_ctas = 0, span_sms = 0;       // of their launches
  // How the captured calls of so many rows were laid out. A replay launches the same kernels and grids
  // and reads the rest from the plan, so later sets of as many rows give k_prefix nothing to do where
  // a graph has been made without it.
  struct Captured {
    bool without = false;  // k_prefix
    int ctas = 0;          // of k_prefix, the last capture's
  };
  std::map<size_t, Captured> captured;
};

namespace syn {
namespace {

constexpr int PT = 64;         // keys of a prefix tile
constexpr int PM = 128;        // query rows of a prefix job
constexpr int SP_WARPS = 4, SP_T = 32, SP_SLOTS = 3;  // k_span: computing warps of a CTA, keys of a tile
constexpr int SP_THREADS = 64 * SP_WARPS;
constexpr int SP_V = 8;        // most query vectors of a k_span job
// A group of at most so many query rows per KV head goes to k_span, which reads its prefix once for 8
// of them. 8 query rows of 128 behind 512, 2048, 8192 positions take 12.7, 17.2, 26.8 us there and
// 14.1, 17.3, 28.1 in k_prefix; 16 (two readings) 13.4, 19.7, 36.2 and 14.8, 18.4, 29.0. (8 rows of 64
// behind 512: 12.9 and 12.2.)
constexpr int SP_FEW = 8;
constexpr int ROWS_MAX = 512;  // rows of a plan
constexpr int UNITS_MAX = ROWS_MAX + ROWS_MAX / 2;

struct Job {      // prefix work of one (group, tile of query rows, KV head)
  int row0;       // first row of the group
  int m0, m;      // query rows m0 .. m0+m of the group: row0 + i / G, head i % G
  int kvh;
  int len;        // shared positions
  int part0;      // first partial record; split i is at part0 + i * m
  int splits;
  int q0;         // query rows of the jobs before
};
struct Item {     // a CTA's share of a job: key tiles t0 .. t1, partial records from part
  int row0, m0, m, kvh;
  int len, t0, t1, part;
  int seq, lowest, q0, pad;  // lowest: no row of the job sees a position below (set on the device)
};

// k_span's work: the positions of one row behind its prefix (n = 0), or the
// prefix of a group of n rows from row0 on. A job is one KV head's part of it for
// up to 8 query vectors: n_kv * nch jobs, the first job0.
struct Unit {
  int row0, n, pre, job0, nch;
};

// A k_span warp's share: n tiles from tile k0 of a job on.
struct Share {
  int job, k0, n, pad;
};
// A k_span job: query vectors (row, g), (row, g + 1), ..., where g counts the heads of
// KV head kvh, over the positions r0 .. r1 of a sequence; its tiles; the warps that
// take part.
struct SpanJob {
  int seq, kvh, nq, row;
  int g, r0, r1, nt;
  int prefix, w0, nw, pad;
};

// What a plan's set has laid out, at the front of its metadata: rows, k_span's units (the last
// `rows` are theirs) and jobs, and the CTAs that k_prefix's items are divided among. A replayed graph
// goes by these, not by the set that it was captured under; only the number of rows has to be the same.
struct Head {
  int rows, units, span_jobs, ctas;
};
// Offsets (ints) of the arrays in the plan's metadata block, behind the Head.
struct Meta {
  int rows, max_jobs, max_items, ctas;
  __host__ __device__ int seq() const { return 4; }
  __host__ __device__ int pre() const { return seq() + rows; }       // shared positions of each row
  __host__ __device__ int job_of() const { return seq() + 2 * rows; }  // first job of the row's group, -1
  __host__ __device__ int local() const { return seq() + 3 * rows; }   // row - first row of its group
  __host__ __device__ int start() const { return seq() + 4 * rows; }   // [ctas + 1] items of each CTA
  __host__ __device__ int items() const { return (start() + ctas + 1 + 3) / 4 * 4; }
  __host__ __device__ int jobs() const { return items() + 12 * max_items; }
  __host__ __device__ int unit_of() const { return jobs() + 8 * max_jobs; }  // k_span's prefix unit of the row, -1
  __host__ __device__ int units() const { return unit_of() + rows; }          // prefixes first, then the rows
  __host__ __device__ int total() const { return units() + 5 * (rows + rows / 2); }
};

struct SharedArgs {
  const float* q;  // rotated
  uint8_t* qparts;
  float* qup;
  int n_heads, n_kv, hd, G;
  const float *kc, *vc;  // this layer
  const int* ptab;       // nullptr: contiguous
  int page, maxp, max_seq;
  const int* len;
  int window;
  const int* meta;
  Meta mv;
  float* po;
  float2* pml;
  int rows, span0;   // rows; k_span's first record
  int warps;         // of k_span
  int after_prefix;  // k_prefix runs before it
  struct Share* shares;
  struct SpanJob* sjobs;
  float* out;
  long long ldo;
  float scale;
  int* err;
};

// ---------------------------------------------------------------------------
// Shared prefixes on the tensor cores. A job is 128 query rows (tensor-memory
// lanes) of one group and KV head; a CTA runs through its items' tiles of 64
// keys:
//   16 warps load K and V rows (8 lanes a row) straight into registers, a tile
//     ahead, and write them as fp16 hi + lo parts, x' = x 2^-e = hi + lo with
//     lo = fp16(x' - hi) and e from the row's largest element: 22 bits,
//     whatever the rows' magnitudes. (k_begin has left Q in this form.)
//   one thread issues tcgen05.mma: S = Qh Kl + Ql Kh + Qh Kh and, with the
//     softmax's P split the same way, O += Ph Vh and O2 += Ph Vl + Pl Vh. Each
//     product cuts its sum off below the accumulator's last bit, towards zero, and
//     over thousands of keys that adds up: so the small products come first in S
//     and have a sum of their own beside O (64 rows, 3500 keys an item: 1.3e-5 off
//     with one sum, 5e-6 with two). Q and P are A operands in tensor memory, P in
//     the place of its S. K and V lie alike, [key][hd] in swizzled
//     128-byte rows: K-major for S, MN-major for O, so nothing is transposed;
//   8 warps turn S into P, two threads per query row, 32 keys each.
// Issuing blocks while the tensor pipe is busy (a product of 64 columns takes
// 45 cycles, one of 128 takes 65), so its warp does nothing else. Registers go
// where they are needed (setmaxnreg): what spills goes to L2, since shared
// memory leaves next to no L1.
// V's row scales go into the softmax: with V_j = V'_j 2^{e_j}, the weight of V'_j
// is 2^{x_j}, x_j = s_j log2(e) + e_j, so the running maximum is taken over x_j,
// P_j = 2^{x_j - M} is the size of the whole contribution, and l = sum P_j 2^{-e_j}.
// O stays in tensor memory; it is rescaled only when the maximum grows by more
// than 2^8 (P keeps 2^7 as its nominal top, so it stays below fp16's 2^16).
// Waits are bounded (SYN_ERR_TIMEOUT). The two warps of the same query rows also wait for each other at
// a barrier that is not, so a warp whose wait has run out does not leave by itself: it says so at
// their next barrier, and both leave behind it.
// 64 rows x 32 heads behind 32768 positions (8 KV heads of 128) take 153 us in all, 140
// of them here: 2.4 us a tile, of which the products are 0.9; conversions and
// softmax fill 69 % of the issue slots and wait for each other the rest. (When it was built: 8
// converting warps in place of 16, 176 us; a warp that issues among them, 303.) A CTA's first tile
// takes 7 us, latencies of the page table, the rows, and 64 KB of O per item.
// ---------------------------------------------------------------------------
constexpr int PX_SOFT = 8, PX_CONV = 16;  // warps; then four of which one issues the products
constexpr int PX_MMA_WARP = PX_SOFT + PX_CONV;
constexpr int PX_THREADS = 32 * (PX_SOFT + PX_CONV + 4);
// Registers a thread: 72 at launch (28 warps); what the converters and the last four warps
// give up is the softmax's.
constexpr int PX_REGS = 72, PX_REGS_SOFT = 88, PX_REGS_CONV = 64, PX_REGS_MMA = 64;
static_assert(2 * PX_REGS_SOFT + 4 * PX_REGS_CONV + PX_REGS_MMA <= 7 * PX_REGS, "register split");
constexpr float P_TOP = 7.0f, P_GROW = 8.0f;

template <int HDP>
struct PxSmem {
  static constexpr int PART = PT * HDP * 2;   // one fp16 part of K or V
  static constexpr int STAGE = 4 * PART;      // K hi, K lo, V hi, V lo
  static constexpr int O = 2 * STAGE;         // O on its way out: [8 warps][32 rows][HDP / 2]
  static constexpr int BYTES = O + PM * HDP * 4 + 1024;
};

__device__ __forceinline__ Head head_of(const SharedArgs& a) {
  const int4 h = __ldg(reinterpret_cast<const int4*>(a.meta));
  return Head{h.x, h.y, h.z, h.w};
}

// Item it, less the tiles that no row sees. Whole warps.
__device__ __forceinline__ Item px_item(const SharedArgs& a, int it) {
  union {
    int4 v[3];
    Item r;
  };
#pragma unroll
  for (int i = 0; i < 3; i++) v[i] = __ldg(reinterpret_cast<const int4*>(a.meta + a.mv.items()) + 3 * it + i);
  r.lowest = 0;
  if (a.window) {
    const int first = r.row0 + r.m0 / a.G, last = r.row0 + (r.m0 + r.m - 1) / a.G;
    int low = r.len;
    for (int row = first + (threadIdx.x & 31); row <= last; row += 32)
      low = min(low, a.len[a.meta[a.mv.seq() + row]] + 1 - a.window);
    r.lowest = max(0, __reduce_min_sync(0xffffffffu, low));
    r.t0 = min(r.t1, max(r.t0, r.lowest / PT));
  }
  return r;
}

// Pairs of f32 in one register pair: one instruction for both.
using f32x2 = unsigned long long;
__device__ __forceinline__ f32x2 pk(float a, float b) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpk(f32x2 v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ void acc2(f32x2& acc, f32x2 a, f32x2 b) {  // acc += a b
  asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(acc) : "l"(a), "l"(b));
}
// A pair -> packed fp16 hi and lo
__device__ __forceinline__ void split2(f32x2 v, uint32_t& hi, uint32_t& lo) {
  float a, b;
  unpk(v, a, b);
  const __half2 h = __floats2half2_rn(a, b);
  const float2 f = __half22float2(h);
  unpk(fma2(pk(f.x, f.y), pk(-1.0f, -1.0f), v), a, b);
  const __half2 r = __floats2half2_rn(a, b);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = *reinterpret_cast<const uint32_t*>(&r);
}

// Biased exponent that scales a row with largest magnitude m to [2^13, 2^14):
// x' = x * px_down(eb), x = x' * px_up(eb). Clamped so that both are normal.
__device__ __forceinline__ int px_exp(float m) {
  return min(max((int)(__float_as_uint(m) >> 23), 67), 254);
}
__device__ __forceinline__ float px_down(int eb) { return __uint_as_float((uint32_t)(267 - eb) << 23); }
__device__ __forceinline__ float px_up(int eb) { return __uint_as_float((uint32_t)(eb - 13) << 23); }

__device__ __forceinline__ float ex2(float x) {  // 2^x, 2 ulp; below 2^-126: 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void prefetch_l2(const float* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }

__device__ __forceinline__ float max_nan(float a, float b) {  // NaN if one of them is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

template <int N>
__device__ __forceinline__ void more_regs() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void less_regs() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
__device__ __forceinline__ void pair_sync(int id) {  // the two warps of the same query rows
  asm volatile("bar.sync %0, 64;" ::"r"(id) : "memory");
}

// Row k of an operand of PT rows, 8 lanes a row (lane l has the float4s l, l + 8, ...): the
// fp16 parts into `part` and psize bytes behind it; the row's exponent.
template <int NV>
__device__ __forceinline__ int px_row(const float4 (&v)[NV], uint8_t* part, int psize, int k) {
  const int l8 = threadIdx.x & 7;
  float m = 0.0f;
#pragma unroll
  for (int u = 0; u < NV; u++)
    m = fmaxf(fmaxf(fmaxf(m, fabsf(v[u].x)), fabsf(v[u].y)), fmaxf(fabsf(v[u].z), fabsf(v[u].w)));
#pragma unroll
  for (int o = 4; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  const int eb = px_exp(m);
  const f32x2 down = pk(px_down(eb), px_down(eb));
  uint8_t* row = part + (k >> 3) * 1024 + (k & 7) * 128 + (l8 & 1) * 8;
#pragma unroll
  for (int u = 0; u < NV; u++) {
    uint2 hi, lo;
    split2(mul2(pk(v[u].x, v[u].y), down), hi.x, lo.x);
    split2(mul2(pk(v[u].z, v[u].w), down), hi.y, lo.y);
    uint8_t* p = row + (u >> 1) * PT * 128 + ((((u & 1) * 4 + (l8 >> 1)) ^ (k & 7)) << 4);
    *reinterpret_cast<uint2*>(p) = hi;
    *reinterpret_cast<uint2*>(p + psize) = lo;
  }
  return eb;
}

template <int HDP>
__global__ void __launch_bounds__(PX_THREADS, 1) k_prefix(const SharedArgs a) {
  using L = PxSmem<HDP>;
  constexpr int QC = HDP / 2;   // tensor-memory columns of one part of Q
  constexpr int NV = HDP / 32;  // float4s of a row per lane
  constexpr uint32_t C_Q = 0, C_S = 2 * QC, C_O = C_S + 2 * PT, C_O2 = C_O + HDP, COLS = 512;
  static_assert(C_O2 + HDP <= COLS, "tensor memory");
  extern __shared__ uint8_t raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  __shared__ __align__(8) uint64_t kfull[2], vfull[2], pfull[2], qk_done[2], pv_done[2], qfull;
  __shared__ __align__(16) float kup[2][PT], vexp[2][PT], vdown[2][PT];
  __shared__ float pmax[2][2][PM];  // [tile parity][half of the keys][row]
  __shared__ int gone[PX_SOFT];     // a softmax warp's wait has run out, told with an item's record
  __shared__ uint32_t tbase_sh;
  __shared__ int fail;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int s = 0; s < 2; s++) {
      mbar_init(&kfull[s], PX_CONV);
      mbar_init(&vfull[s], PX_CONV);
      mbar_init(&pfull[s], PX_SOFT);
      mbar_init(&qk_done[s], 1);
      mbar_init(&pv_done[s], 1);
    }
    mbar_init(&qfull, PX_SOFT);
    fail = 0;
    mbar_fence_init();
  }
  if (warp == PX_MMA_WARP) tc_alloc(&tbase_sh, COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tb = tbase_sh;
  volatile int* failed = &fail;
  auto wait = [&](uint64_t* bar, int use) {  // a whole warp, until the use-th completion
    bool done = mbar_try_wait(bar, use & 1);
    if (!done && !*failed) {
      done = mbar_wait_bounded(bar, use & 1);
      if (!done) *failed = 1;
    }
    return __all_sync(0xffffffffu, done) != 0;
  };
  // The plan, the lengths, the page table and the shared pages are from before k_begin, which
  // let this kernel begin when they were in place: only the queries have to be waited for (and
  // k_span, which reads what k_begin wrote and does not wait itself, begins after that).
  const Head head = head_of(a);
  const int* start = a.meta + a.mv.start();
  int i0 = start[blockIdx.x], i1 = start[blockIdx.x + 1];
  if (head.ctas != (int)gridDim.x) {  // a set made for other grids: its CTAs' items, a few of them each
    i0 = start[(int)blockIdx.x * head.ctas / (int)gridDim.x];
    i1 = start[((int)blockIdx.x + 1) * head.ctas / (int)gridDim.x];
  }
  if (head.rows != a.rows) i1 = i0;
  int n = 0;    // tiles so far; tile n uses stage n & 1 for the (n >> 1)-th time
  int ord = 0;  // items with tiles so far

  if (warp < PX_SOFT) {
    // ---- two threads per query row: half h has keys 32h .. 32h+31 of a tile ----
    more_regs<PX_REGS_SOFT>();
    const int h = warp >> 2, r = tid & 127, pair = 1 + (warp & 3);
    const uint32_t tl = tb + ((uint32_t)((warp & 3) * 32) << 16);  // this warp's lanes
    bool ok = true;
    griddep_wait();
    griddep_launch();
    for (int it = i0; it < i1 && ok; it++) {
      const Item item = px_item(a, it);
      const bool busy = (warp & 3) * 32 < item.m;  // else no row of this warp is one
      const size_t rec = item.part + r;
      if (item.t0 == item.t1) {  // nothing of it is in any window
        if (r < item.m && h == 0) {
          a.pml[rec] = make_float2(-INFINITY, 0.0f);
          for (int d = 0; d < a.hd; d += 4)
            *reinterpret_cast<float4*>(a.po + rec * a.hd + d) = make_float4(0, 0, 0, 0);
        }
        continue;
      }
      float cq = 0.0f;
      int low = 0;
      if (busy) {  // half h brings Q's part h (the last item's products are done: its O was read)
        const bool is = r < item.m;
        if (is) cq = a.qup[item.q0 + r] * a.scale * 1.4426950408889634f;
        if (a.window && is)
          low = max(0, a.len[a.meta[a.mv.seq() + item.row0 + (item.m0 + r) / a.G]] + 1 - a.window);
        tc_fence_after();
        const uint4* q = reinterpret_cast<const uint4*>(a.qparts + (size_t)item.q0 * (HDP * 4)) + h * (HDP / 8) * item.m + r;
#pragma unroll
        for (int c = 0; c < HDP / 8; c += 8) {  // 16-byte chunks
          uint4 u[8];
#pragma unroll
          for (int e = 0; e < 8; e++) u[e] = is && (c + e) * 8 < a.hd ? q[(c + e) * item.m] : make_uint4(0, 0, 0, 0);
          tc_st16(tl + C_Q + h * QC + c * 4, reinterpret_cast<const uint32_t*>(u));
          tc_st16(tl + C_Q + h * QC + c * 4 + 16, reinterpret_cast<const uint32_t*>(u + 4));
        }
        tc_wait_st();
        tc_fence_before();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&qfull);
      ord++;
      float M = -INFINITY;
      f32x2 l = 0;
      const f32x2 cq2 = pk(cq, cq);
      for (int t = item.t0; t < item.t1; t++, n++) {
        const int s = n & 1, use = n >> 1;
        // (the scales of the tile's rows come with V)
        ok = wait(&vfull[s], use) && wait(&qk_done[s], use);
        if (!busy && !ok) break;
        if (busy) {  // (!ok: it goes on with what is there, as far as the barrier)
          tc_fence_after();
          f32x2 y[16];
          {
            float x[32];
            tc_ld32(tl + C_S + s * PT + h * 32, x);
            tc_wait_ld();
#pragma unroll
            for (int j = 0; j < 32; j += 4) {
              const ulonglong2 ku = *reinterpret_cast<const ulonglong2*>(&kup[s][h * 32 + j]);
              const ulonglong2 ve = *reinterpret_cast<const ulonglong2*>(&vexp[s][h * 32 + j]);
              y[j / 2] = fma2(mul2(pk(x[j], x[j + 1]), ku.x), cq2, ve.x);
              y[j / 2 + 1] = fma2(mul2(pk(x[j + 2], x[j + 3]), ku.y), cq2, ve.y);
            }
          }
          const int vlo = low - t * PT - h * 32, vhi = item.len - t * PT - h * 32;
          if (__any_sync(0xffffffffu, vlo > 0 || vhi < 32)) {
#pragma unroll
            for (int j = 0; j < 32; j += 2) {
              float p, q;
              unpk(y[j / 2], p, q);
              if (j < vlo || j >= vhi) p = -INFINITY;
              if (j + 1 < vlo || j + 1 >= vhi) q = -INFINITY;
              y[j / 2] = pk(p, q);
            }
          }
          float mx = -INFINITY, mx2 = -INFINITY;
#pragma unroll
          for (int j = 0; j < 16; j += 2) {
            float p, q;
            unpk(y[j], p, q);
            mx = fmaxf(fmaxf(mx, p), q);
            unpk(y[j + 1], p, q);
            mx2 = fmaxf(fmaxf(mx2, p), q);
          }
          mx = fmaxf(mx, mx2);
          if (!ok) mx = NAN;  // (otherwise it never is: this warp gives up)
          pmax[n & 1][h][r] = mx;
          pair_sync(pair);
          mx = max_nan(mx, pmax[n & 1][h ^ 1][r]);
          // a new reference only when the old one is too far below (the same in both halves)
          const bool grow = !(mx <= M + P_GROW);  // (also from -inf)
          const float ref = grow ? mx : M;
          if (__any_sync(0xffffffffu, mx != mx)) {
            ok = false;
            break;
          }
          if (t == item.t0) {
            M = ref;
          } else if (__any_sync(0xffffffffu, grow)) {
            const float f = !grow ? 1.0f : M == -INFINITY ? 0.0f : ex2(M - ref);
            M = ref;
            l = mul2(l, pk(f, f));
            wait(&pv_done[(n - 1) & 1], (n - 1) >> 1);  // (if it runs out, `fail` is set and the result void)
            tc_fence_after();
#pragma unroll 1
            for (int c = h * HDP; c < (h + 1) * HDP; c += 8) {  // (of both sums)
              float o[8];
              tc_ld8(tl + C_O + c, o);
              tc_wait_ld();
              uint32_t u[8];
#pragma unroll
              for (int j = 0; j < 8; j++) u[j] = __float_as_uint(o[j] * f);
              tc_st8(tl + C_O + c, u);
            }
            tc_wait_st();
          }
          tc_fence_after();  // (both halves have read S; P takes its place)
          const float shift = M == -INFINITY ? 0.0f : P_TOP - M;
          const f32x2 shift2 = pk(shift, shift);
#pragma unroll
          for (int c = 0; c < 32; c += 16) {
            uint32_t hi[8], lo[8];
#pragma unroll
            for (int j = 0; j < 16; j += 4) {
              const ulonglong2 vd = *reinterpret_cast<const ulonglong2*>(&vdown[s][h * 32 + c + j]);
              float p, q;
              unpk(add2(y[(c + j) / 2], shift2), p, q);
              f32x2 e = pk(ex2(p), ex2(q));
              l = fma2(e, vd.x, l);
              split2(e, hi[j / 2], lo[j / 2]);
              unpk(add2(y[(c + j) / 2 + 1], shift2), p, q);
              e = pk(ex2(p), ex2(q));
              l = fma2(e, vd.y, l);
              split2(e, hi[j / 2 + 1], lo[j / 2 + 1]);
            }
            tc_st8(tl + C_S + s * PT + h * 16 + c / 2, hi);
            tc_st8(tl + C_S + s * PT + 32 + h * 16 + c / 2, lo);
          }
          tc_wait_st();
          tc_fence_before();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&pfull[s]);
      }
      if (!ok) break;
      // the item's record: O and l are both relative to 2^(M - P_TOP)
      ok = wait(&pv_done[(n - 1) & 1], (n - 1) >> 1);
      if (!busy && !ok) break;
      if (busy) {
        tc_fence_after();
        float la, lb;
        unpk(l, la, lb);
        la += lb;
        if (h == 1) pmax[n & 1][1][r] = la;
        if (lane == 0) gone[warp] = !ok;
        pair_sync(pair);
        if (!ok || gone[warp ^ 4]) {
          ok = false;
          break;
        }
        // (M = -inf: nothing seen, or nothing that weighs; the sum is NaN where a score was)
        if (h == 0 && r < item.m) a.pml[rec] = make_float2(M - P_TOP, la + pmax[n & 1][1][r]);
        pair_sync(pair);  // (the slot is the next item's)
        // O: from rows to whole lines
        constexpr int CH = HDP / 8;  // 16-byte chunks of a row's half
        uint8_t* stage = sm + L::O + warp * (32 * CH * 16);
        for (int c = 0; c < HDP / 2; c += 32) {
          float o[32];
          tc_ld32(tl + C_O + h * (HDP / 2) + c, o);
          tc_wait_ld();
#pragma unroll
          for (int j = 0; j < 32; j += 8) {
            float o2[8];
            tc_ld8(tl + C_O2 + h * (HDP / 2) + c + j, o2);
            tc_wait_ld();
#pragma unroll
            for (int e = 0; e < 8; e++) o[j + e] += o2[e];
          }
#pragma unroll
          for (int j = 0; j < 32; j += 4)
            *reinterpret_cast<float4*>(stage + (lane * CH + (((c + j) / 4) ^ (lane % CH))) * 16) =
                make_float4(o[j], o[j + 1], o[j + 2], o[j + 3]);
        }
        const int c = lane % CH, col = h * (HDP / 2) + c * 4, r0 = (warp & 3) * 32;
#pragma unroll 4
        for (int q = lane / CH; q < 32; q += 32 / CH) {
          float4 o = *reinterpret_cast<const float4*>(stage + (q * CH + (c ^ (q % CH))) * 16);
          if (r0 + q < item.m && col < a.hd)
            *reinterpret_cast<float4*>(a.po + (size_t)(item.part + r0 + q) * a.hd + col) = o;
        }
        __syncwarp();
        tc_fence_before();
      }
    }
  } else if (warp < PX_MMA_WARP) {
    // ---- K and V rows to fp16 parts: 8 lanes a row, 4 rows of each a warp and tile. (Of 8 rows, a
    // warp has 0, 4, 1, 5 or 2, 6, 3, 7: their stores meet all banks.)
    less_regs<PX_REGS_CONV>();
    const int cw = warp - PX_SOFT, l8 = lane & 7, q4 = lane >> 3;
    const int jj = (cw >> 1) * 8 + (((q4 & 1) << 2) | (q4 >> 1)) + (cw & 1) * 2;  // this lane's key
    const int dcol = PT / a.page, doff = PT - dcol * a.page;
    // Three tiles are under way: x holds one's rows, `at` has the next one's places, `pg` the
    // page numbers of the one after as they come.
    int it = i0, left = 0;  // the item of the last tile asked for, and its tiles still to ask for
    int len = 0, lowest = 0, pos = 0, kvh = 0, col = 0, off = 0;
    const int* tab = nullptr;
    struct Pages { int kvh, pg, off; };  // kvh < 0: no tile
    struct Rows { bool any; long long at; };  // at < 0: no row
    auto ask = [&]() {
      Pages r;
      if (left == 0) {
        it -= (tab == nullptr);
        while (left == 0 && ++it < i1) {
          const Item item = px_item(a, it);
          left = item.t1 - item.t0;
          len = item.len;
          lowest = item.lowest;
          kvh = item.kvh;
          tab = a.ptab + (size_t)item.seq * a.maxp;
          pos = item.t0 * PT + jj;
          col = pos / a.page;
          off = pos - col * a.page;
        }
      }
      r.kvh = left ? kvh : -1;
      r.pg = left && pos < len && pos >= lowest ? __ldg(tab + col) : -1;
      r.off = off;
      col += dcol;
      off += doff;
      if (off >= a.page) {
        off -= a.page;
        col++;
      }
      pos += PT;
      if (left) left--;
      return r;
    };
    auto place = [&](const Pages& p) {
      Rows r;
      r.any = p.kvh >= 0;
      r.at = p.pg < 0 ? -1 : (((long long)p.pg * a.page + p.off) * a.n_kv + p.kvh) * a.hd + l8 * 4;
      return r;
    };
    auto load = [&](float4 (&v)[NV], const float* cache, const Rows& r) {
#pragma unroll
      for (int u = 0; u < NV; u++) {
        v[u] = make_float4(0, 0, 0, 0);
        if (r.at >= 0 && u * 32 + l8 * 4 < a.hd)
          v[u] = __ldg(reinterpret_cast<const float4*>(cache + r.at + u * 32));
      }
    };
    float4 xk[NV], xv[NV];
    Pages pages = ask();
    Rows next = place(pages);
    pages = ask();
    load(xk, a.kc, next);
    load(xv, a.vc, next);
    bool cur = next.any;
    next = place(pages);
    pages = ask();
    bool ok = true;
    for (; cur && ok; n++) {
      const int s = n & 1, use = n >> 1;
      uint8_t* st = sm + s * L::STAGE;
      if (use && !(ok = wait(&qk_done[s], use - 1))) break;
      const int ek = px_row<NV>(xk, st, L::PART, jj);
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&kfull[s]);
      load(xk, a.kc, next);
      if (use && !(ok = wait(&pv_done[s], use - 1))) break;
      const int ev = px_row<NV>(xv, st + 2 * L::PART, L::PART, jj);
      if (l8 == 0) {  // (the softmax is done with the stage's last scales: P was used)
        kup[s][jj] = px_up(ek);
        vexp[s][jj] = (float)(ev - 140);
        vdown[s][jj] = px_down(ev);
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&vfull[s]);
      load(xv, a.vc, next);
      cur = next.any;
      next = place(pages);
      // (the tile after next on its way to L2: 64 rows behind 32768 positions take 161 us with it, 171
      // without)
      if (next.at >= 0) prefetch_l2((l8 < 4 ? a.kc : a.vc) + next.at - l8 * 4 + (l8 & 3) * (a.hd / 4));
      pages = ask();
    }
  } else {
    less_regs<PX_REGS_MMA>();
    if (warp == PX_MMA_WARP) {
      // ---- one thread issues the products ----
      constexpr uint32_t id_s = (1u << 4) | ((uint32_t)(PT >> 3) << 17) | ((uint32_t)(PM >> 4) << 24);
      constexpr uint32_t id_o = (1u << 4) | (1u << 16) | ((uint32_t)(HDP >> 3) << 17) | ((uint32_t)(PM >> 4) << 24);
      const uint64_t kd = tc_desc_k(smem_u32(sm)), vd = tc_desc_mn(smem_u32(sm) + 2 * L::PART, PT * 128);
      const uint32_t k_lo = (uint32_t)kd, k_hi = (uint32_t)(kd >> 32), v_lo = (uint32_t)vd, v_hi = (uint32_t)(vd >> 32);
      bool ok = true;
      auto scores = [&](int k) {  // S of tile k
        const int s = k & 1, use = k >> 1;
        if (!(ok = wait(&kfull[s], use))) return;
        if (use && !(ok = wait(&pv_done[s], use - 1))) return;  // P of the tile before last is there
        tc_fence_after();
        if (tc_elect()) {
          const uint32_t kb = k_lo + s * (L::STAGE >> 4), d = tb + C_S + s * PT, q = tb + C_Q;
          auto at = [](int ks) { return (uint32_t)((ks >> 2) * PT * 128 + (ks & 3) * 32) >> 4; };
#pragma unroll
          for (int ks = 0; ks < HDP / 16; ks++) {
            if (ks == 0) tc_mma_ts<false>(d, q, kb + (L::PART >> 4), k_hi, id_s);
            else tc_mma_ts<true>(d, q + ks * 8, kb + (L::PART >> 4) + at(ks), k_hi, id_s);
            tc_mma_ts<true>(d, q + QC + ks * 8, kb + at(ks), k_hi, id_s);
          }
#pragma unroll
          for (int ks = 0; ks < HDP / 16; ks++) tc_mma_ts<true>(d, q + ks * 8, kb + at(ks), k_hi, id_s);
          tc_commit(&qk_done[s]);
        }
        __syncwarp();
      };
      for (int it = i0; it < i1 && ok; it++) {
        const Item item = px_item(a, it);
        const int nt = item.t1 - item.t0;
        if (!nt) continue;
        if (!(ok = wait(&qfull, ord++))) break;
        scores(n);
        for (int t = 0; t < nt && ok; t++, n++) {
          if (t + 1 < nt) scores(n + 1);
          const int s = n & 1, use = n >> 1;
          if (!ok || !(ok = wait(&pfull[s], use))) break;  // (after V: the softmax waits for its scales)
          tc_fence_after();
          if (tc_elect()) {
            const uint32_t vb = v_lo + s * (L::STAGE >> 4), p = tb + C_S + s * PT, d = tb + C_O, d2 = tb + C_O2;
#pragma unroll
            for (int ks = 0; ks < PT / 16; ks++) {
              const uint32_t o = ks * 2048 >> 4;
              if (ks == 0 && t == 0) {
                tc_mma_ts<false>(d, p, vb, v_hi, id_o);
                tc_mma_ts<false>(d2, p, vb + (L::PART >> 4), v_hi, id_o);
              } else {
                tc_mma_ts<true>(d, p + ks * 8, vb + o, v_hi, id_o);
                tc_mma_ts<true>(d2, p + ks * 8, vb + (L::PART >> 4) + o, v_hi, id_o);
              }
              tc_mma_ts<true>(d2, p + 32 + ks * 8, vb + o, v_hi, id_o);
            }
            tc_commit(&pv_done[s]);
          }
          __syncwarp();
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (*failed && tid == 0 && a.err) atomicExch(a.err, SYN_ERR_TIMEOUT);
  if (warp == PX_MMA_WARP) {
    tc_fence_after();
    if (*failed && lane == 0) {  // products may be in flight: they end before the memory goes
      mbar_init(&qfull, 1);
      tc_commit(&qfull);
      mbar_wait_bounded(&qfull, 0);
    }
    __syncwarp();
    tc_dealloc(tb, COLS);
  }
}

// ---------------------------------------------------------------------------
// Few query vectors over a range of positions: each row's own positions, and
// prefixes of few query rows. All jobs' tiles of 32 keys, one after another, are
// dealt to all computing warps in equal, contiguous shares (the lengths are read on
// the device), so uneven rows cost nothing. Beside each computing warp a copying one
// brings the K and V rows, a bulk copy a row, into the ring of three half tiles (16
// bytes of padding a row keep a lane per row free of bank conflicts); lane = key for
// the scores, with q broadcast from shared memory, so no sum crosses lanes; lane =
// four columns for the weighted sum, with the weights broadcast. For four query
// vectors a tile of 128 columns takes 1500 cycles for the scores, 270 for the weights and
// 1300 for the sum, against 1400 of an SM's share of HBM for four warps' tiles. A warp
// that copies for itself spends 2000 more on that: 32 rows behind 2048 shared
// positions took 45 us instead of 38.
// ---------------------------------------------------------------------------
__device__ __forceinline__ float redux_max(float x) {
  float y;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
  return y;
}

// Positions of unit u: [lo, hi)
__device__ __forceinline__ int2 unit_range(const SharedArgs& a, const Unit& u) {
  const int* seq = a.meta + a.mv.seq();
  if (u.n) {
    int lo = 0;
    if (a.window) {
      lo = u.pre;
      for (int r = u.row0; r < u.row0 + u.n; r++) lo = min(lo, max(0, a.len[seq[r]] + 1 - a.window));
    }
    return make_int2(lo, u.pre);
  }
  const int L = a.len[seq[u.row0]] + 1;
  if (L > a.max_seq) {  // a replayed graph that has run past the cache
    if (a.err) atomicExch(a.err, SYN_ERR_INVALID_ARG);
    return make_int2(0, 0);
  }
  return make_int2(max(u.pre, a.window ? L - a.window : 0), L);
}

// Deals the tiles of all units to k_span's warps: tile t of T is warp w's where
// floor(w T / W) <= t < floor((w + 1) T / W), so of tile t the warp is
// ceil((t + 1) W / T) - 1. Every block finds the units' first tiles; the shares and
// jobs are divided among the blocks' threads.
__device__ __forceinline__ void deal_shares(const SharedArgs& a, int block, int blocks) {
  __shared__ int starts[UNITS_MAX + 1], lows[UNITS_MAX], highs[UNITS_MAX], sums[AP_THREADS / 32];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const Unit* units = reinterpret_cast<const Unit*>(a.meta + a.mv.units());
  // (loaded beside the number of units: there is room for as many as rows, and for half as many more)
  const Unit mine = units[min(tid, a.mv.rows - 1)];
  const Head head = head_of(a);
  if (head.rows != a.rows) {  // a replay after a set of another number of rows
    if (block == 0 && tid == 0 && a.err) atomicExch(a.err, SYN_ERR_INVALID_ARG);
    return;
  }
  const int nu = head.units, per = (nu + AP_THREADS - 1) / AP_THREADS;
  const int u0 = min(nu, tid * per), u1 = min(nu, u0 + per);
  int sum = 0;
  for (int u = u0; u < u1; u++) {
    const Unit x = u == tid && u < a.mv.rows ? mine : units[u];
    const int2 r = unit_range(a, x);
    const int t = (max(0, r.y - r.x) + SP_T - 1) / SP_T * a.n_kv * x.nch;
    starts[u] = t;
    lows[u] = r.x;
    highs[u] = r.y;
    sum += t;
  }
  int inc = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += y;
  }
  if (lane == 31) sums[warp] = inc;
  __syncthreads();
  int base = inc - sum;
  for (int w = 0; w < warp; w++) base += sums[w];
  for (int u = u0; u < u1; u++) {
    const int t = starts[u];
    starts[u] = base;
    base += t;
  }
  if (u1 == nu) starts[nu] = base;
  __syncthreads();
  const int total = starts[nu], warps = min(a.warps, total);
  // the last unit whose first tile (or job) is at or before x; an empty one starts where the next does
  auto find = [&](int x, auto&& at) {
    int lo = 0, hi = nu;
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (at(mid) <= x) lo = mid;
      else hi = mid;
    }
    return lo;
  };
  for (int w = block * AP_THREADS + tid; w < a.warps; w += blocks * AP_THREADS) {
    Share s{0, 0, 0, 0};
    if (w < warps) {
      const int t0 = (int)((long long)w * total / warps), t1 = (int)((long long)(w + 1) * total / warps);
      const int u = find(t0, [&](int i) { return starts[i]; });
      const Unit x = units[u];
      const int nt = (starts[u + 1] - starts[u]) / (a.n_kv * x.nch), r = t0 - starts[u];
      s = Share{x.job0 + r / nt, r % nt, t1 - t0, 0};
    }
    a.shares[w] = s;
  }
  for (int j = block * AP_THREADS + tid; j < head.span_jobs; j += blocks * AP_THREADS) {
    const int u = find(j, [&](int i) { return units[i].job0; });
    const Unit x = units[u];
    const int jl = j - x.job0, kvh = jl / x.nch, v0 = (jl - kvh * x.nch) * SP_V;
    SpanJob s;
    s.seq = a.meta[a.mv.seq() + x.row0];
    s.kvh = kvh;
    s.nq = min(SP_V, (x.n ? x.n * a.G : a.G) - v0);
    s.row = x.row0 + (x.n ? v0 / a.G : 0);
    s.g = x.n ? v0 % a.G : v0;
    s.r0 = lows[u];
    s.r1 = highs[u];
    s.nt = (starts[u + 1] - starts[u]) / (a.n_kv * x.nch);
    s.prefix = x.n > 0;
    s.w0 = s.nw = s.pad = 0;
    if (s.nt) {
      const long long t0 = starts[u] + (long long)jl * s.nt, t1 = t0 + s.nt;
      s.w0 = (int)(((t0 + 1) * warps - 1) / total);
      s.nw = (int)((t1 * warps - 1) / total) - s.w0 + 1;
    }
    a.sjobs[j] = s;
  }
}

// A rotated query row as k_prefix wants it, x' = x 2^-e = hi + lo: of a job's m rows the hi parts
// and then the lo parts, each [HDP / 8][m] chunks of 16 bytes (a thread per row reads whole lines).
struct QParts {
  const SharedArgs& a;
  uint8_t* at = nullptr;  // the row's first chunk; nullptr: no job
  float* up = nullptr;
  int m = 0;
  __device__ QParts(const SharedArgs& a) : a(a) {}
  __device__ __forceinline__ void find(int row, int head) {  // (the plan: from before this kernel)
    const int job0 = a.meta[a.mv.job_of() + row];
    if (job0 < 0) return;
    const int kvh = head / a.G, i = a.meta[a.mv.local() + row] * a.G + head - kvh * a.G;
    const Job job = reinterpret_cast<const Job*>(a.meta + a.mv.jobs())[job0 + i / PM * a.n_kv + kvh];
    m = job.m;
    up = a.qup + job.q0 + i - job.m0;
    at = a.qparts + (size_t)job.q0 * (a.hd > 64 ? 512 : 256) + (i - job.m0) * 16;
  }
  template <int VEC, int LP, typename T>
  __device__ __forceinline__ void take(int lane, int nv, const T (&r1)[2], const T (&r2)[2]) {
    if (!at) return;  // (the same for the LP lanes of the row)
    constexpr int STEPS = VEC == 4 ? 1 : 2;
    float mx = 0.0f;
#pragma unroll
    for (int i = 0; i < STEPS; i++)
#pragma unroll
      for (int e = 0; e < VEC; e++)
        mx = fmaxf(mx, fmaxf(fabsf(reinterpret_cast<const float*>(&r1[i])[e]), fabsf(reinterpret_cast<const float*>(&r2[i])[e])));
    const uint32_t mask = (LP == 32 ? 0xffffffffu : (1u << (LP & 31)) - 1) << (threadIdx.x & 31 & ~(LP - 1));
#pragma unroll
    for (int o = LP / 2; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(mask, mx, o));
    const int eb = px_exp(mx), lo = (a.hd > 64 ? 16 : 8) * m * 16;
    if (lane == 0) *up = px_up(eb);
    const float down = px_down(eb);
#pragma unroll
    for (int i = 0; i < STEPS; i++)
      if (lane + i * LP < nv)
#pragma unroll
        for (int h = 0; h < 2; h++) {
          const float* f = reinterpret_cast<const float*>(h ? &r2[i] : &r1[i]);
          const int d = h * (a.hd >> 1) + (lane + i * LP) * VEC;  // 8 elements a chunk
          uint8_t* p = at + (d >> 3) * m * 16 + (d & 7) * 2;
          if constexpr (VEC == 4) {
            uint2 x, y;
            split2(mul2(pk(f[0], f[1]), pk(down, down)), x.x, y.x);
            split2(mul2(pk(f[2], f[3]), pk(down, down)), x.y, y.y);
            *reinterpret_cast<uint2*>(p) = x;
            *reinterpret_cast<uint2*>(p + lo) = y;
          } else {
            uint32_t x, y;
            split2(mul2(pk(f[0], 0.0f), pk(down, down)), x, y);
            *reinterpret_cast<uint16_t*>(p) = (uint16_t)x;
            *reinterpret_cast<uint16_t*>(p + lo) = (uint16_t)y;
          }
        }
    const int over = a.hd + lane;  // the rest of the last chunk
    if ((a.hd & 7) && over < (a.hd | 7) + 1) {
      uint8_t* p = at + (over >> 3) * m * 16 + (over & 7) * 2;
      *reinterpret_cast<uint16_t*>(p) = 0;
      *reinterpret_cast<uint16_t*>(p + lo) = 0;
    }
  }
};

// The append, and in the last `deal` blocks the shares. PARTS: with k_prefix behind it.
template <int VEC, int LP, bool ONE, bool PARTS>
__global__ void __launch_bounds__(AP_THREADS) k_begin(const __grid_constant__ AppendArgs p,
                                                      const __grid_constant__ SharedArgs a, int deal) {
  const int block = (int)blockIdx.x - ((int)gridDim.x - deal);
  if (block < 0) {
    if constexpr (PARTS) append_rows<VEC, LP, ONE, 1>(p, QParts(a));
    else append_rows<VEC, LP, ONE, 1>(p);
  } else {
    griddep_wait();
    griddep_launch();
    deal_shares(a, block, deal);
  }
}

// N floats, to or from shared memory
template <int N>
__device__ __forceinline__ void weights(float* to, const float* from) {
  if constexpr (N >= 4) {
#pragma unroll
    for (int v = 0; v < N; v += 4) *reinterpret_cast<float4*>(to + v) = *reinterpret_cast<const float4*>(from + v);
  } else {
#pragma unroll
    for (int v = 0; v < N; v++) to[v] = from[v];
  }
}

// A warp's ring of half tiles (K and V of a tile in turn): `used` counts those that this side, the
// copying or the computing warp, is past.
struct SpanRing {
  uint8_t* at;
  int slot_bytes;
  uint64_t *full, *empty;
  uint32_t slot = 0, turn = 0;
  __device__ __forceinline__ void next() {
    if (++slot == SP_SLOTS) {
      slot = 0;
      turn++;
    }
  }
  __device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity) {
    bool ok = mbar_try_wait(bar + slot, parity);
    if (!ok) ok = mbar_wait_bounded(bar + slot, parity);
    return __all_sync(0xffffffffu, ok) != 0;
  }
};

// Tiles [k0, k1) of a job into the ring, lane = key.
__device__ __forceinline__ bool span_fill(const SharedArgs& a, const SpanJob& job, int k0, int k1, int hd,
                                          SpanRing& ring) {
  const int lane = threadIdx.x & 31, stride = hd * 4 + 16;
  // the place of this lane's key in the tile that is asked for next
  int pos = job.r0 + k0 * SP_T + lane, col = a.ptab ? pos / a.page : 0, off = pos - col * a.page;
  const int dcol = a.ptab ? SP_T / a.page : 0, doff = SP_T - dcol * a.page;
  auto ask = [&]() {  // offset of its row in the cache, -1 = none
    long long row = -1;
    if (pos < job.r1) {
      if (a.ptab) {
        const int pg = __ldg(a.ptab + (size_t)job.seq * a.maxp + col);
        if (pg >= 0) row = (long long)pg * a.page + off;
      } else {
        row = (long long)job.seq * a.max_seq + pos;
      }
    }
    pos += SP_T;
    col += dcol;
    off += doff;
    if (a.ptab && off >= a.page) {
      off -= a.page;
      col++;
    }
    return row < 0 ? -1 : (row * a.n_kv + job.kvh) * hd;
  };
  auto fill = [&](const float* cache, long long at) {
    if (ring.turn && !ring.wait(ring.empty, (ring.turn - 1) & 1)) return false;
    uint64_t* bar = ring.full + ring.slot;
    const uint32_t rows = __popc(__ballot_sync(0xffffffffu, at >= 0));
    if (lane == 0) mbar_expect_tx(bar, rows * hd * 4);
    __syncwarp();
    if (at >= 0) bulk_g2s(ring.at + ring.slot * ring.slot_bytes + lane * stride, cache + at, hd * 4, bar);
    ring.next();
    return true;
  };
  long long next = ask();
  for (int k = k0; k < k1; k++) {
    const long long at = next;
    if (k + 1 < k1) next = ask();
    if (!fill(a.kc, at) || !fill(a.vc, at)) return false;
  }
  return true;
}

// Tiles [k0, k1) of a job, by one warp; the record of each query vector. HD: the
// head dim where it is 64 or 128, else 0.
template <int LPR, int HD, int NQ>
__device__ __forceinline__ bool span_job(const SharedArgs& a, const SpanJob& job, int k0, int k1, size_t rec,
                                         SpanRing& ring, float* qs, float* ps) {
  constexpr int SUBS = 32 / LPR;
  const int lane = threadIdx.x & 31, hd = HD ? HD : a.hd, stride = hd * 4 + 16;
  const int sub = lane / LPR, l4 = (lane % LPR) * 4;
  const int nt = k1 - k0;
  const uint8_t* tile = nullptr;
  auto ready = [&]() {  // the next half tile is in `tile`
    tile = ring.at + ring.slot * ring.slot_bytes;
    return ring.wait(ring.full, ring.turn & 1);
  };
  auto past = [&]() {
    fence_async_smem();  // (this warp's reads before the copies that follow)
    __syncwarp();
    if (lane == 0) mbar_arrive(ring.empty + ring.slot);
    ring.next();
  };
  float m[NQ], l[NQ];
  f32x2 o[NQ][2];
#pragma unroll
  for (int v = 0; v < NQ; v++) {
    m[v] = -INFINITY;
    l[v] = 0.0f;
    o[v][0] = o[v][1] = 0;
  }
  // queries, times scale * log2(e)
  const float qscale = a.scale * 1.4426950408889634f;
  int low[NQ];
  {
    int row = job.row, g = job.g;
#pragma unroll
    for (int v = 0; v < NQ; v++) {
      low[v] = 0;
      const bool live = v < job.nq;
      if (live && job.prefix && a.window) low[v] = a.len[a.meta[a.mv.seq() + row]] + 1 - a.window;
      const float* q = a.q + ((size_t)row * a.n_heads + job.kvh * a.G + g) * hd;
      for (int d = lane * 4; d < hd; d += 128) {
        float4 f = make_float4(0, 0, 0, 0);
        if (live) f = *reinterpret_cast<const float4*>(q + d);
        *reinterpret_cast<float4*>(qs + v * hd + d) =
            make_float4(f.x * qscale, f.y * qscale, f.z * qscale, f.w * qscale);
      }
      if (++g == a.G) {
        g = 0;
        row++;
      }
    }
  }
  __syncwarp();
  for (int k = 0; k < nt; k++) {
    const int key = job.r0 + (k0 + k) * SP_T + lane;
    const int nk = min(SP_T, job.r1 - job.r0 - (k0 + k) * SP_T);
    if (!ready()) return false;
    f32x2 acc[NQ][2];
#pragma unroll
    for (int v = 0; v < NQ; v++) acc[v][0] = acc[v][1] = 0;
    const uint8_t* kr = tile + lane * stride;
#pragma unroll 4
    for (int d = 0; d < hd; d += 4) {
      const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(kr + d * 4);
#pragma unroll
      for (int v = 0; v < NQ; v++) {
        const ulonglong2 q = *reinterpret_cast<const ulonglong2*>(qs + v * hd + d);
        acc2(acc[v][0], x.x, q.x);
        acc2(acc[v][1], x.y, q.y);
      }
    }
    past();
    // softmax weights
    float corr[NQ];
    float w[NQ];
    bool grown = false;
#pragma unroll
    for (int v = 0; v < NQ; v++) {
      float x, y;
      unpk(add2(acc[v][0], acc[v][1]), x, y);
      const bool seen = lane < nk && key >= low[v];
      x = seen ? x + y : -INFINITY;
      const float mx = fmaxf(m[v], redux_max(x));
      corr[v] = m[v] == -INFINITY ? 0.0f : ex2(m[v] - mx);
      grown |= mx != m[v];
      const float p = mx == -INFINITY && !seen ? 0.0f : ex2(x - mx);  // (NaN where only NaN and -inf are seen)
      l[v] = fmaf(l[v], corr[v], p);
      m[v] = mx;
      w[v] = p;
    }
    if (grown) {
#pragma unroll
      for (int v = 0; v < NQ; v++) {
        o[v][0] = mul2(o[v][0], pk(corr[v], corr[v]));
        o[v][1] = mul2(o[v][1], pk(corr[v], corr[v]));
      }
    }
    weights<NQ>(ps + lane * NQ, w);
    __syncwarp();
    if (!ready()) return false;
    if (l4 < hd) {
#pragma unroll 4
      for (int j = sub; j < nk; j += SUBS) {
        const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(tile + j * stride + l4 * 4);
        float p[NQ];
        weights<NQ>(p, ps + j * NQ);
#pragma unroll
        for (int v = 0; v < NQ; v++) {
          const f32x2 pp = pk(p[v], p[v]);
          acc2(o[v][0], pp, x.x);
          acc2(o[v][1], pp, x.y);
        }
      }
    }
    past();
  }
#pragma unroll
  for (int v = 0; v < NQ; v++) {
    float x[4];
    unpk(o[v][0], x[0], x[1]);
    unpk(o[v][1], x[2], x[3]);
#pragma unroll
    for (int s = LPR; s < 32; s <<= 1)
#pragma unroll
      for (int e = 0; e < 4; e++) x[e] += __shfl_xor_sync(0xffffffffu, x[e], s);
    const float sum = warp_sum(l[v]);
    if (v < job.nq) {
      if (lane == 0) a.pml[rec + v] = make_float2(m[v], sum);
      if (sub == 0 && l4 < hd)
        *reinterpret_cast<float4*>(a.po + (rec + v) * hd + l4) = make_float4(x[0], x[1], x[2], x[3]);
    }
  }
  __syncwarp();
  return true;
}

// Warps 0 .. 3 compute, 4 .. 7 copy for them.
template <int LPR, int HD>
__global__ void __launch_bounds__(SP_THREADS, 1) k_span(const SharedArgs a) {
  extern __shared__ __align__(16) uint8_t sraw[];
  __shared__ __align__(8) uint64_t full[SP_WARPS][SP_SLOTS], empty[SP_WARPS][SP_SLOTS];
  const int warp = (threadIdx.x >> 5) % SP_WARPS, lane = threadIdx.x & 31, hd = HD ? HD : a.hd;
  const bool copies = threadIdx.x >= SP_WARPS * 32;
  const int slot_bytes = SP_T * (hd * 4 + 16), per_warp = SP_SLOTS * slot_bytes + SP_V * hd * 4 + SP_T * SP_V * 4;
  SpanRing ring{sraw + warp * per_warp, slot_bytes, full[warp], empty[warp]};
  float* qs = reinterpret_cast<float*>(ring.at + SP_SLOTS * slot_bytes);
  float* ps = qs + SP_V * hd;
  if (!copies && lane < SP_SLOTS) {
    mbar_init(&full[warp][lane], 1);
    mbar_init(&empty[warp][lane], 1);
    mbar_fence_init();
  }
  __syncthreads();
  // Behind k_prefix this kernel needs nothing of it: k_begin is complete where k_prefix has
  // let it begin, and so it runs on every SM that k_prefix has left.
  if (!a.after_prefix) griddep_wait();
  griddep_launch();
  const int gw = warp * gridDim.x + blockIdx.x;  // (neighbouring shares on different SMs)
  const int4 sh = __ldcg(reinterpret_cast<const int4*>(a.shares) + gw);
  int j = sh.x, k0 = sh.y, left = head_of(a).rows == a.rows ? sh.z : 0;
  bool ok = true;
  while (left > 0 && ok) {
    union {
      int4 v[3];
      SpanJob job;
    };
#pragma unroll
    for (int i = 0; i < 3; i++) v[i] = __ldcg(reinterpret_cast<const int4*>(a.sjobs + j) + i);
    const int k1 = min(job.nt, k0 + left);
    const size_t rec = a.span0 + (size_t)(gw + j) * SP_V;
    if (k1 > k0)
      ok = copies        ? span_fill(a, job, k0, k1, hd, ring)
           : job.nq > 4 ? span_job<LPR, HD, 8>(a, job, k0, k1, rec, ring, qs, ps)
           : job.nq > 2 ? span_job<LPR, HD, 4>(a, job, k0, k1, rec, ring, qs, ps)
           : job.nq > 1 ? span_job<LPR, HD, 2>(a, job, k0, k1, rec, ring, qs, ps)
                        : span_job<LPR, HD, 1>(a, job, k0, k1, rec, ring, qs, ps);
    left -= k1 - k0;
    k0 = 0;
    j++;
  }
  if (!ok && lane == 0 && a.err) atomicExch(a.err, SYN_ERR_TIMEOUT);
  if (!ok && copies)  // nothing may land in a CTA that has gone: each slot's last copies
    for (int i = 0; i < SP_SLOTS; i++) {
      const int turn = (int)ring.turn - (i >= (int)ring.slot);
      if (turn >= 0) mbar_wait_bounded(ring.full + i, turn & 1);
    }
  if (a.after_prefix) griddep_wait();  // (k_join waits for this kernel's end, and so for k_prefix's)
}

// ---------------------------------------------------------------------------
// The parts of a query row: k_span's of its own positions, and of its prefix
// k_span's or k_prefix's. A CTA per (row, head): warp w takes records w, w + 4, ...,
// up to eight of them in flight before their weights are known, since what bounds
// this is the latency of its two loads. (Maxima are in units of log2.)
// ---------------------------------------------------------------------------
constexpr int JN_WARPS = 4, JN_BLOCK = 32;  // records at a time

// A query row from its definition, over the positions that it sees: exp(s - M) without a guard, so that NaN
// and infinities go where the formula takes them. The other kernels cannot do that (a running maximum
// drops NaN, a tile's other rows multiply what they do not see by 0, fp16 parts of an infinity are
// NaN): they leave a sum or a value that is not finite, and the row comes here. A query or a score that
// is NaN decides it, in no more time than a finite row; otherwise it is slow (each key's row by one warp,
// twice): 64 rows x 4 heads that see an infinite V element among 32768 positions take 11.4 ms.
// Never taken by finite operands whose products stay finite.
__device__ __noinline__ float join_plain(const SharedArgs& a, int b, int head, float (*red)[128]) {
  __shared__ double sums[JN_WARPS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, hd = a.hd, kvh = head / a.G;
  const int seq = a.meta[a.mv.seq() + b], L = a.len[seq] + 1;
  if (L > a.max_seq) return 0.0f;  // (reported where the shares are dealt)
  const bool act = lane * 4 < hd;
  const float4 zero = make_float4(0, 0, 0, 0);
  float4 q = zero;
  if (act) q = *(reinterpret_cast<const float4*>(a.q + ((size_t)b * a.n_heads + head) * hd) + lane);
  if (__any_sync(0xffffffffu, q.x != q.x || q.y != q.y || q.z != q.z || q.w != q.w)) return NAN;
  constexpr int U = 2;  // rows under way in a warp
  auto each = [&](auto with_v, auto&& take) {  // (score, the lane's columns of V)
    for (int p0 = (a.window ? max(0, L - a.window) : 0) + warp; p0 < L; p0 += U * JN_WARPS) {
      float4 k[U], v[U];
      bool is[U];
#pragma unroll
      for (int i = 0; i < U; i++) {
        const int pos = p0 + i * JN_WARPS;
        long long row = -1;
        if (pos < L) {
          row = (long long)seq * a.max_seq + pos;
          if (a.ptab) {
            const int pg = a.ptab[(size_t)seq * a.maxp + pos / a.page];
            row = pg < 0 ? -1 : (long long)pg * a.page + pos % a.page;
          }
        }
        is[i] = row >= 0;
        const size_t at = ((size_t)row * a.n_kv + kvh) * hd + lane * 4;
        k[i] = v[i] = zero;
        if (is[i] && act) {
          k[i] = *reinterpret_cast<const float4*>(a.kc + at);
          if (with_v) v[i] = *reinterpret_cast<const float4*>(a.vc + at);
        }
      }
#pragma unroll
      for (int i = 0; i < U; i++) {
        const float s = warp_sum(fmaf(q.x, k[i].x, fmaf(q.y, k[i].y, fmaf(q.z, k[i].z, q.w * k[i].w)))) * a.scale;
        if (is[i]) take(s, v[i]);
      }
    }
  };
  float M = -INFINITY;
  bool none = false;
  each(std::false_type(), [&](float s, const float4&) {
    M = fmaxf(M, s);
    none |= s != s;
  });
  if (lane == 0) red[warp][0] = M;
  if (__syncthreads_or(none)) return NAN;
  M = fmaxf(fmaxf(red[0][0], red[1][0]), fmaxf(red[2][0], red[3][0]));
  double l = 0.0, o[4] = {0.0, 0.0, 0.0, 0.0};
  each(std::true_type(), [&](float s, const float4& v) {
    const double p = expf(s - M);
    l += p;
    o[0] += p * v.x;
    o[1] += p * v.y;
    o[2] += p * v.z;
    o[3] += p * v.w;
  });
  if (lane == 0) sums[warp] = l;
  __syncthreads();
  l = sums[0] + sums[1] + sums[2] + sums[3];
  *reinterpret_cast<float4*>(&red[warp][lane * 4]) =
      make_float4((float)(o[0] / l), (float)(o[1] / l), (float)(o[2] / l), (float)(o[3] / l));
  __syncthreads();
  const int d = threadIdx.x;
  return (red[0][d] + red[1][d]) + (red[2][d] + red[3][d]);
}

__global__ void __launch_bounds__(JN_WARPS * 32, 7) k_join(const __grid_constant__ SharedArgs a) {
  __shared__ __align__(16) float red[JN_WARPS][128];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, hd = a.hd;
  const int b = blockIdx.x / a.n_heads, head = blockIdx.x - b * a.n_heads;
  const int kvh = head / a.G, g = head - kvh * a.G;
  const Unit* units = reinterpret_cast<const Unit*>(a.meta + a.mv.units());
  const Head plan = head_of(a);
  if (plan.rows != a.rows) {  // (as in deal_shares: nothing was computed)
    griddep_wait();
    if (threadIdx.x < hd) a.out[(long long)b * a.ldo + (long long)head * hd + threadIdx.x] = NAN;
    return;
  }
  // Records first + c * step, c < n. (The plan and k_begin's jobs may be read before the
  // wait: k_span begins, and lets this kernel begin, after them.)
  struct Parts { size_t first; int n, step; };
  auto span_parts = [&](int u, int idx) {
    const Unit x = units[u];
    const int j = x.job0 + kvh * x.nch + idx / SP_V;
    const int4 s = __ldcg(reinterpret_cast<const int4*>(a.sjobs + j) + 2);  // prefix, w0, nw
    return Parts{a.span0 + (size_t)(s.y + j) * SP_V + idx % SP_V, s.z, SP_V};
  };
  const int pu = a.meta[a.mv.unit_of() + b], job0 = a.meta[a.mv.job_of() + b];
  const int local = a.meta[a.mv.local() + b] * a.G + g;
  const Parts own = span_parts(plan.units - a.rows + b, g);
  Parts pre{0, 0, 0};
  if (pu >= 0) {
    pre = span_parts(pu, local);
  } else if (job0 >= 0) {
    const Job job = reinterpret_cast<const Job*>(a.meta + a.mv.jobs())[job0 + local / PM * a.n_kv + kvh];
    pre = Parts{(size_t)(job.part0 + local - job.m0), job.splits, job.m};
  }
  const int n = own.n + pre.n;
  auto rec = [&](int c) {
    return c < own.n ? own.first + (size_t)c * own.step : pre.first + (size_t)(c - own.n) * pre.step;
  };
  const bool act = lane * 4 < hd;
  float4 x[JN_BLOCK / JN_WARPS];
  auto fetch = [&](int c0) {
#pragma unroll
    for (int e = 0; e < JN_BLOCK / JN_WARPS; e++) {
      const int c = c0 + warp + e * JN_WARPS;
      x[e] = make_float4(0, 0, 0, 0);
      if (act && c < n) x[e] = __ldcg(reinterpret_cast<const float4*>(a.po + rec(c) * hd) + lane);
    }
  };
  griddep_wait();
  const float2 none = make_float2(-INFINITY, 0.0f);
  const float2 mine = lane < n ? __ldcg(&a.pml[rec(lane)]) : none;
  fetch(0);
  float M = mine.x;
  for (int c = 32 + lane; c < n; c += 32) M = fmaxf(M, __ldcg(&a.pml[rec(c)]).x);
  M = warp_max(M);
  float4 o = make_float4(0, 0, 0, 0);
  float sum = 0.0f;
  for (int c0 = 0; c0 < n; c0 += JN_BLOCK) {
    const float2 ml = c0 == 0 ? mine : c0 + lane < n ? __ldcg(&a.pml[rec(c0 + lane)]) : none;
    if (c0) fetch(c0);
    const float f = ml.x == -INFINITY ? 0.0f : ex2(ml.x - M);
    sum = fmaf(f, ml.y, sum);
#pragma unroll
    for (int e = 0; e < JN_BLOCK / JN_WARPS; e++) {
      const float fc = __shfl_sync(0xffffffffu, f, warp + e * JN_WARPS);
      o.x = fmaf(x[e].x, fc, o.x);  // (0 times what is not finite too: the row is taken again)
      o.y = fmaf(x[e].y, fc, o.y);
      o.z = fmaf(x[e].z, fc, o.z);
      o.w = fmaf(x[e].w, fc, o.w);
    }
  }
  griddep_launch();
  *reinterpret_cast<float4*>(&red[warp][lane * 4]) = o;
  sum = warp_sum(sum);
  const float inv = sum > 0.0f ? 1.0f / sum : 0.0f * sum;  // (NaN stays)
  __syncthreads();
  const int d = threadIdx.x;
  float y = 0.0f;
  if (d < hd) y = ((red[0][d] + red[1][d]) + (red[2][d] + red[3][d])) * inv;
  if (__syncthreads_or(!(fabsf(y) < INFINITY) || M == -INFINITY)) y = join_plain(a, b, head, red);
  if (d < hd) a.out[(long long)b * a.ldo + (long long)head * hd + d] = y;
}

syn_status_t launched(cudaError_t e, const char* where) {
  if (e == cudaSuccess) return SYN_OK;
  set_last_cuda_error(e, where);
  return SYN_ERR_CUDA;
}

template <bool PARTS>
void (*begin_kernel(const AppendShape& sh))(const AppendArgs, const SharedArgs, int) {
  return !sh.vec       ? k_begin<1, 32, false, PARTS>
         : sh.lp == 4 ? k_begin<4, 4, true, PARTS>
         : sh.lp == 8 ? k_begin<4, 8, true, PARTS>
                      : k_begin<4, 16, true, PARTS>;
}

// Most jobs and items of a batch of `batch` rows (groups of two or more share).
size_t max_jobs(size_t batch, size_t n_kv, size_t G) {
  return n_kv * (batch * G / PM + batch / 2 + 1);
}

Meta meta_of(const syn_cuda_decode_plan_t* p) {
  const syn_cuda_kvcache_t* c = p->cache;
  const size_t jobs = max_jobs(c->batch, c->n_kv, p->n_heads / c->n_kv);
  return Meta{(int)c->batch, (int)jobs, (int)(jobs + p->sms), p->sms};
}

// k_span's shared memory. (One CTA on an SM, whatever it leaves free: 256 threads of up to 254 registers.
// Twice the grid for heads of up to 60, where the memory would allow it, ran in two waves: 32 rows behind
// 2048 positions, 600 of their own, took 37.3 us at head dim 32 and take 33.6; 34.6 and 30.4 at 48.)
size_t span_smem(size_t hd) {
  return SP_WARPS * (SP_SLOTS * SP_T * (hd * 4 + 16) + SP_V * hd * 4 + SP_T * SP_V * 4);
}
// Most k_span jobs of a batch
size_t span_jobs(size_t batch, size_t n_kv, size_t G) {
  return n_kv * (batch * ((G + SP_V - 1) / SP_V) + batch / 2 * (SP_FEW / SP_V));
}

}  // namespace

namespace {

// A sequence holds a family's pages no longer.
void family_loses(syn_cuda_decode_plan_t* p, PlanFamily& f, size_t seq, cudaStream_t st) {
  if (f.holds[seq] == 2 && !p->parted) {
    p->parted = true;
    // No number of rows is this one, so what was captured computes nothing until the next set. (A
    // captured reorder moves nothing yet, and must not do this whenever it is replayed.)
    cudaStreamCaptureStatus cs = cudaStreamCaptureStatusNone;
    cudaStreamIsCapturing(st, &cs);
    if (cs == cudaStreamCaptureStatusNone) cudaMemsetAsync(p->meta, 0xff, sizeof(int), st);
  }
  f.holds[seq] = 0;
}

// Whoever a captured reorder may exchange with a sequence that the group depends on is depended on too; and
// a holder that one may exchange with a sequence that is none is no holder for long.
void family_close(syn_cuda_decode_plan_t* p, PlanFamily& f, cudaStream_t st) {
  for (bool more = true; more;) {
    more = false;
    for (const auto& mix : p->cache->mixes) {
      const bool all = std::all_of(mix.begin(), mix.end(), [&](int32_t s) { return f.holds[s] != 0; });
      const bool core = std::any_of(mix.begin(), mix.end(), [&](int32_t s) { return f.holds[s] == 2; });
      for (int32_t s : mix) {
        const uint8_t was = f.holds[s];
        if (!all) family_loses(p, f, s, st);
        else if (core) f.holds[s] = 2;
        more |= f.holds[s] != was;
      }
    }
  }
}

}  // namespace

void plans_mixed(syn_cuda_kvcache_t* c, cudaStream_t st) {
  for (auto* p : c->plans)
    for (auto& f : p->families) family_close(p, f, st);
}

void plans_changed(syn_cuda_kvcache_t* c, size_t seq, cudaStream_t st) {
  for (auto* p : c->plans)
    for (auto& f : p->families)
      if (c->len[seq] < f.len) family_loses(p, f, seq, st);
}

void plans_reordered(syn_cuda_kvcache_t* c, const int32_t* seqs, size_t n, cudaStream_t st) {
  for (auto* p : c->plans)
    for (auto& f : p->families)
      if (!std::all_of(seqs, seqs + n, [&](int32_t s) { return f.holds[s] != 0; }))
        for (size_t i = 0; i < n; i++) family_loses(p, f, seqs[i], st);
}

void plans_orphaned(syn_cuda_kvcache_t* c) {
  for (auto* p : c->plans) p->cache = nullptr;
}

int decode_plan_layout(const syn_cuda_decode_plan_t* p) {
  return p->jobs ? p->prefix_ctas : 0;
}

syn_status_t launch_attn_shared(syn_cuda_decode_plan_t* p, const AttnArgs& at, int* err,
                                cudaStream_t st) {
  syn_cuda_kvcache_t* c = p->cache;
  const size_t kvd = c->n_kv * c->hd, qd = p->n_heads * c->hd;
  syn_status_t s;
  const size_t rows_per_layer = c->page ? c->n_pages * c->page : c->batch * c->max_seq;
  SharedArgs a;
  a.q = p->q;
  a.qparts = p->qparts;
  a.qup = p->qup;
  a.n_heads = (int)p->n_heads;
  a.n_kv = (int)c->n_kv;
  a.hd = (int)c->hd;
  a.G = (int)(p->n_heads / c->n_kv);
  a.kc = c->k + at.layer * rows_per_layer * kvd;
  a.vc = c->v + at.layer * rows_per_layer * kvd;
  a.ptab = c->page ? c->d_ptab : nullptr;
  a.page = (int)c->page;
  a.maxp = (int)c->maxp;
  a.max_seq = (int)c->max_seq;
  a.len = c->d_len;
  a.window = (int)std::min<size_t>(at.window, c->max_seq + 1);
  a.meta = p->meta;
  a.mv = meta_of(p);
  a.po = p->po;
  a.pml = p->pml;
  a.rows = (int)p->rows;
  a.warps = p->span_sms * SP_WARPS;
  a.span0 = (int)(p->part_rows - (p->sms * SP_WARPS + span_jobs(c->batch, c->n_kv, a.G)) * SP_V);
  a.after_prefix = p->jobs > 0;
  a.shares = static_cast<Share*>(p->shares);
  a.sjobs = reinterpret_cast<SpanJob*>(a.shares + a.warps);
  a.out = at.out;
  a.ldo = (long long)at.ldo;
  a.scale = 1.0f / sqrtf((float)c->hd);
  a.err = err;
  {
    AppendArgs ap = append_args(at, p->q, qd, 0);
    ap.seq_of = p->meta + a.mv.seq();
    ap.set_rows = p->meta;
    ap.err = err;
    ap.rows = a.rows;
    const AppendShape sh = append_shape(ap);
    void (*kern)(const AppendArgs, const SharedArgs, int) = p->jobs ? begin_kernel<true>(sh) : begin_kernel<false>(sh);
    const size_t per = AP_THREADS / sh.lp, blocks = (p->rows * (p->n_heads + 2 * c->n_kv) + per - 1) / per;
    const int deal = (std::max(a.warps, p->span_jobs) + AP_THREADS - 1) / AP_THREADS;
    s = launched(launch_pdl(kern, dim3((unsigned)(blocks + deal)), dim3(AP_THREADS), 0, st, ap, a, deal), "k_begin");
    if (s) return s;
  }
  if (p->jobs) {
    const bool w = c->hd > 64;
    void (*kern)(const SharedArgs) = w ? k_prefix<128> : k_prefix<64>;
    const size_t smem = w ? PxSmem<128>::BYTES : PxSmem<64>::BYTES;
    if ((s = more_smem((const void*)kern, smem))) return s;
    s = launched(launch_pdl(kern, dim3(p->prefix_ctas), dim3(PX_THREADS), smem, st, a), "k_prefix");
    if (s) return s;
  }
  void (*span)(const SharedArgs) = c->hd == 128  ? k_span<32, 128>
                                   : c->hd == 64 ? k_span<16, 64>
                                   : c->hd <= 32 ? k_span<8, 0>
                                   : c->hd < 64  ? k_span<16, 0>
                                                 : k_span<32, 0>;
  if ((s = more_smem((const void*)span, span_smem(c->hd)))) return s;
  s = launched(launch_pdl(span, dim3(p->span_sms), dim3(SP_THREADS), span_smem(c->hd), st, a),
               "k_span");
  if (s) return s;
  return launched(launch_pdl(k_join, dim3((unsigned)(p->rows * p->n_heads)), dim3(JN_WARPS * 32), 0, st, a),
                  "k_join");
}

}  // namespace syn

using namespace syn;

extern "C" {

syn_status_t syn_cuda_decode_plan_create(syn_cuda_kvcache_t* c, size_t n_heads,
                                         syn_cuda_decode_plan_t** out) {
  if (!c || !out) return SYN_ERR_NULL_PTR;
  *out = nullptr;
  if (!n_heads || n_heads % c->n_kv) return SYN_ERR_SHAPE_MISMATCH;
  if (c->hd > 128 || c->batch > 32768 || n_heads > 65535) return SYN_ERR_UNSUPPORTED;
  DeviceGuard g(c->device);
  if (!g.ok) return SYN_ERR_CUDA;
  auto* p = new (std::nothrow) syn_cuda_decode_plan_s();
  if (!p) return SYN_ERR_OUT_OF_MEMORY;
  p->cache = c;
  p->device = c->device;
  p->sms = num_sms();
  p->n_heads = n_heads;
  const Meta mv = meta_of(p);
  p->meta_ints = mv.total();
  // prefix records: a job's rows for each CTA that shares in it, at most one job's rows more
  const size_t G = n_heads / c->n_kv;
  // per CTA than the batch's query rows; k_span records: 8 of each (warp, job) that meet
  const size_t prefix = c->batch * n_heads + (size_t)p->sms * std::min<size_t>(PM, c->batch * G);
  const size_t span = (p->sms * SP_WARPS + span_jobs(c->batch, c->n_kv, G)) * SP_V;
  p->part_rows = prefix + span;
  if (p->part_rows > 0x7FFFFFFF) {
    delete p;
    return SYN_ERR_UNSUPPORTED;
  }
  cudaError_t e = cudaMalloc(&p->q, c->batch * n_heads * c->hd * sizeof(float));
  const size_t qbytes = c->batch * n_heads * (c->hd > 64 ? 512 : 256);
  if (e == cudaSuccess) e = cudaMalloc(&p->qparts, qbytes);
  if (e == cudaSuccess) e = cudaMalloc(&p->qup, c->batch * n_heads * sizeof(float));
  if (e == cudaSuccess) e = cudaMalloc(&p->meta, p->meta_ints * sizeof(int));
  if (e == cudaSuccess) e = cudaMallocHost(&p->meta_h, p->meta_ints * sizeof(int));
  if (e == cudaSuccess) std::fill(p->meta_h, p->meta_h + p->meta_ints, 0);  // (all of it is copied)
  if (e == cudaSuccess) e = cudaMalloc(&p->po, p->part_rows * c->hd * sizeof(float));
  if (e == cudaSuccess) e = cudaMalloc(&p->pml, p->part_rows * sizeof(float2));
  if (e == cudaSuccess)
    e = cudaMalloc(&p->shares, p->sms * SP_WARPS * sizeof(Share) +
                                   span_jobs(c->batch, c->n_kv, G) * sizeof(SpanJob));
  if (e == cudaSuccess) e = cudaMalloc(&p->err, sizeof(int));
  if (e == cudaSuccess) e = cudaMemset(p->err, 0, sizeof(int));
  if (e == cudaSuccess) e = cudaMemset(p->meta, 0, p->meta_ints * sizeof(int));
  if (e == cudaSuccess) e = cudaEventCreateWithFlags(&p->copied, cudaEventDisableTiming);
  if (e == cudaSuccess) e = cudaDeviceSynchronize();
  if (e != cudaSuccess) {
    set_last_cuda_error(e, "syn_cuda_decode_plan_create");
    syn_cuda_decode_plan_destroy(p);
    return SYN_ERR_OUT_OF_MEMORY;
  }
  try {
    c->plans.push_back(p);
  } catch (const std::bad_alloc&) {
    syn_cuda_decode_plan_destroy(p);
    return SYN_ERR_OUT_OF_MEMORY;
  }
  *out = p;
  return SYN_OK;
}

syn_status_t syn_cuda_decode_plan_destroy(syn_cuda_decode_plan_t* p) {
  if (!p) return SYN_ERR_NULL_PTR;
  DeviceGuard g(p->device);
  if (p->cache) {
    auto& plans = p->cache->plans;
    plans.erase(std::remove(plans.begin(), plans.end(), p), plans.end());
  }
  cudaDeviceSynchronize();
  cudaFree(p->q);
  cudaFree(p->qparts);
  cudaFree(p->qup);
  cudaFree(p->meta);
  if (p->meta_h) cudaFreeHost(p->meta_h);
  cudaFree(p->po);
  cudaFree(p->pml);
  cudaFree(p->shares);
  cudaFree(p->err);
  if (p->copied) cudaEventDestroy(p->copied);
  delete p;
  return SYN_OK;
}

syn_status_t syn_cuda_decode_plan_set(syn_cuda_decode_plan_t* p, size_t n_groups,
                                      const size_t* group_rows, const int32_t* seqs,
                                      void* stream) try {
  if (!p || (n_groups && (!group_rows || !seqs))) return SYN_ERR_NULL_PTR;
  syn_cuda_kvcache_t* c = p->cache;
  if (!c) return SYN_ERR_INVALID_ARG;
  DeviceGuard g(p->device);
  if (!g.ok) return SYN_ERR_CUDA;
  cudaStream_t st = (cudaStream_t)stream;
  cudaStreamCaptureStatus cs = cudaStreamCaptureStatusNone;
  SYN_CUDA_TRY(cudaStreamIsCapturing(st, &cs));
  if (cs != cudaStreamCaptureStatusNone) return SYN_ERR_UNSUPPORTED;
  size_t rows = 0;
  std::vector<uint8_t> seen(c->batch, 0);
  for (size_t i = 0; i < n_groups; i++) {
    if (!group_rows[i] || group_rows[i] > c->batch - rows) return SYN_ERR_INVALID_ARG;
    for (size_t j = rows; j < rows + group_rows[i]; j++) {
      if (seqs[j] < 0 || (size_t)seqs[j] >= c->batch || seen[seqs[j]]) return SYN_ERR_INVALID_ARG;
      seen[seqs[j]] = 1;
    }
    rows += group_rows[i];
  }
  if (rows > ROWS_MAX) return SYN_ERR_UNSUPPORTED;
  syn_status_t s = kv_sync(c, st);
  // (a row cut back into a shared page gets its own copy now, not in a later call)
  for (size_t i = 0; i < rows && s == SYN_OK; i++) s = kv_own_page(c, seqs[i], st);
  if (s) return s;
  SYN_CUDA_TRY(cudaEventSynchronize(p->copied));  // the last copy has left meta_h
  const Meta mv = meta_of(p);
  const int G = (int)(p->n_heads / c->n_kv);
  int* h = p->meta_h;
  Job* jobs = reinterpret_cast<Job*>(h + mv.jobs());
  Item* items = reinterpret_cast<Item*>(h + mv.items());
  p->parted = true;  // (until all of it is in place)
  p->seqs.assign(seqs, seqs + rows);
  p->prefix.assign(rows, 0);
  p->shrunk.assign(rows, 0);
  p->families.clear();
  // the sequences of a group, and those that a captured reorder may exchange with them at any time
  auto related = [&](size_t r0, size_t n) {
    std::vector<uint8_t> in(c->batch, 0);
    for (size_t j = r0; j < r0 + n; j++) in[seqs[j]] = 2;
    for (bool more = true; more;) {
      more = false;
      for (const auto& mix : c->mixes)
        if (std::any_of(mix.begin(), mix.end(), [&](int32_t s) { return in[s]; }))
          for (int32_t s : mix) {
            more |= !in[s];
            in[s] = 2;
          }
    }
    return in;
  };
  auto pages = [&](size_t s) { return c->ptab_h + s * c->maxp; };
  size_t r0 = 0;
  for (size_t i = 0; i < n_groups; r0 += group_rows[i++]) {
    const size_t n = group_rows[i];
    size_t shared = 0;  // leading positions in pages that all rows hold
    if (n > 1 && c->page) {
      size_t most = c->len[seqs[r0]];
      for (size_t j = r0; j < r0 + n; j++) most = std::min(most, c->len[seqs[j]]);
      PlanFamily f{0, related(r0, n)};
      const int* first = pages(seqs[r0]);
      size_t col = most / c->page;
      for (size_t s = 0; s < c->batch; s++)
        if (f.holds[s]) col = std::mismatch(first, first + col, pages(s)).first - first;
      f.len = shared = col * c->page;
      for (size_t s = 0; s < c->batch && shared; s++)
        if (std::equal(first, first + col, pages(s))) f.holds[s] = std::max<uint8_t>(f.holds[s], 1);
      if (shared) {
        family_close(p, f, st);
        p->families.push_back(std::move(f));
      }
    }
    for (size_t j = r0; j < r0 + n; j++) {
      p->prefix[j] = shared;
      if (c->page) p->shrunk[j] = c->shrunk[seqs[j]];
    }
  }
  Unit* units = reinterpret_cast<Unit*>(h + mv.units());
  const int row_ch = (G + SP_V - 1) / SP_V;  // k_span jobs of a row and KV head
  int nj = 0, nu = 0, uj = 0, widest = 0;
  size_t tiles = 0, own = 0, longest = 0;  // k_prefix's; k_span's, of a row and in all, with 128 positions more
  auto tiles_of = [&](int j) { return ((size_t)jobs[j].len + PT - 1) / PT; };
  // few, many: whether groups of few query rows share their prefix (in k_span), and those of many
  // (in k_prefix)
  auto lay_out = [&](bool share_few, bool share_many) {
    int q0 = 0;
    nj = nu = uj = widest = 0;
    tiles = own = longest = 0;
    r0 = 0;
    for (size_t i = 0; i < n_groups; r0 += group_rows[i++]) {
      const size_t n = group_rows[i];
      const bool small = n * G <= SP_FEW;
      const size_t shared = (small ? share_few : share_many) ? p->prefix[r0] : 0;
      const bool few = shared && small;
      for (size_t j = r0; j < r0 + n; j++) {
        h[mv.seq() + j] = seqs[j];
        h[mv.pre() + j] = (int)shared;
        h[mv.job_of() + j] = shared && !few ? nj : -1;
        h[mv.unit_of() + j] = few ? nu : -1;
        h[mv.local() + j] = (int)(j - r0);
        const size_t t = (c->len[seqs[j]] - shared + 128) / SP_T + 1;
        own += c->n_kv * row_ch * t;
        longest = std::max(longest, t);
      }
      if (few) {
        const int nch = ((int)n * G + SP_V - 1) / SP_V;
        units[nu++] = Unit{(int)r0, (int)n, (int)shared, uj, nch};
        uj += (int)c->n_kv * nch;
        own += c->n_kv * nch * ((shared + SP_T - 1) / SP_T);
      } else if (shared)
        for (int m0 = 0; m0 < (int)n * G; m0 += PM)
          for (int kvh = 0; kvh < (int)c->n_kv; kvh++) {
            const int m = std::min(PM, (int)n * G - m0);
            jobs[nj] = Job{(int)r0, m0, m, kvh, (int)shared, 0, 0, q0};
            widest = std::max(widest, m);
            q0 += m;
            tiles += tiles_of(nj++);
          }
    }
    for (size_t j = 0; j < rows; j++) {  // each row's own positions
      units[nu++] = Unit{(int)j, 0, h[mv.pre() + j], uj, row_ch};
      uj += (int)c->n_kv * row_ch;
    }
  };
  auto most_of = [&](size_t n) {  // tiles of a CTA of k_prefix, with n of them
    size_t most = (tiles + n - 1) / n;
    auto items_at = [&](size_t q) {
      size_t k = 0;
      for (int j = 0; j < nj; j++) k += (tiles_of(j) + q - 1) / q;
      return k;
    };
    while ((size_t)nj <= n && items_at(most) > n) most++;
    return most;
  };
  // What the kernels take (us, measured at head dim 128 and used for all): k_prefix 4 + 0.05 m for m query rows (at
  // least 7) and 1.2 + 0.0165 m (at most 2.6) a tile; k_span 4, 2.5 a tile of each warp, and k_join 1 for 32 records
  // of a row. The rows are taken 128 positions on, as they grow before the plan is next set.
  auto prefix_us = [&](int n) { return std::max(7.0, 4 + 0.05 * widest) + std::min(2.6, 1.2 + 0.0165 * widest) * most_of(n); };
  auto span_us = [&](int n) {
    const size_t per = std::max<size_t>(1, (own + SP_WARPS * n - 1) / (SP_WARPS * n));
    return 4 + 2.5 * per + longest / per / 32;
  };
  // SYN_PLAN_LAYOUT=1, 2 or 3 keeps to: every row for itself, k_span behind k_prefix, beside it.
  const char* env = getenv("SYN_PLAN_LAYOUT");
  const int only = env ? atoi(env) : 0;
  const auto kept = p->captured.find(rows);
  const bool many = kept == p->captured.end() || !kept->second.without;
  const int ctas_kept = kept == p->captured.end() ? 0 : kept->second.ctas;
  lay_out(true, many);
  p->prefix_ctas = p->span_sms = p->sms;
  double best = span_us(p->sms) + (nj ? prefix_us(p->sms) : 0);
  if (nj && ctas_kept) {
    p->prefix_ctas = ctas_kept;
    if (ctas_kept < p->sms) p->span_sms = p->sms - ctas_kept;
  } else if (nj && only != 2) {
    // k_span behind k_prefix, each on all SMs, or side by side, each on its own: 8 rows behind 2048
    // positions take 19.1 us behind and 15.6 side by side, 64 rows behind 32768 are 7 % slower so
    double least = only == 3 ? 1e30 : 0.85 * best;
    for (int n = 12; n < p->sms; n += 12) {
      const double us = std::max(prefix_us(n), span_us(p->sms - n));
      if (us < least) {
        best = least = us;
        p->prefix_ctas = n;
        p->span_sms = p->sms - n;
      }
    }
  }
  // A short prefix is read by each row for itself: 56 rows behind 42 positions take 11.2 us so, and
  // 20.3 with k_prefix.
  const bool has_jobs = nj > 0;
  lay_out(false, false);
  if (has_jobs && ctas_kept ? false : only ? only == 1 : span_us(p->sms) < 0.85 * best)
    p->prefix_ctas = p->span_sms = p->sms;
  else
    lay_out(true, many);
  if (own > 1u << 30) return SYN_ERR_UNSUPPORTED;  // (the device counts k_span's tiles in 32 bits)
  size_t ni = 0, part = 0, done = 0, jt = 0;
  auto item_of = [&](const Job& job, size_t t0, size_t t1) {
    return Item{job.row0, job.m0, job.m,     job.kvh, job.len, (int)t0, (int)t1, (int)part,
                seqs[job.row0], 0, job.q0, 0};
  };
  // With no more jobs than CTAs, an item per CTA: the shortest items of which there are enough
  // CTAs for (a CTA that goes from one job to another drains its pipeline in between). Else
  // the tiles of all jobs, one after another, in equal shares.
  const int ctas = p->prefix_ctas;
  int cta = 0;
  if (nj && nj <= ctas) {
    const size_t most = most_of(ctas);
    for (int j = 0; j < nj; j++) {
      Job& job = jobs[j];
      const size_t nt = tiles_of(j);
      job.splits = (int)((nt + most - 1) / most);
      job.part0 = (int)part;
      for (int i = 0; i < job.splits; i++) {
        h[mv.start() + cta++] = (int)ni;
        items[ni++] = item_of(job, nt * i / job.splits, nt * (i + 1) / job.splits);
        part += job.m;
      }
    }
  }
  for (int j = 0; cta < ctas; cta++) {
    h[mv.start() + cta] = (int)ni;
    size_t share = nj > ctas ? tiles * (cta + 1) / ctas - done : 0;
    done += share;
    while (share) {
      Job& job = jobs[j];
      const size_t nt = tiles_of(j), take = std::min(share, nt - jt);
      if (!jt) job.part0 = (int)part;
      items[ni++] = item_of(job, jt, jt + take);
      part += job.m;
      job.splits++;
      share -= take;
      if ((jt += take) == nt) {
        j++;
        jt = 0;
      }
    }
  }
  h[mv.start() + ctas] = (int)ni;
  *reinterpret_cast<Head*>(h) = Head{(int)rows, nu, uj, ctas};
  p->units = nu;
  p->span_jobs = uj;
  p->jobs = nj;
  p->rows = rows;
  p->groups = n_groups;
  SYN_CUDA_TRY(cudaMemcpyAsync(p->meta, h, p->meta_ints * sizeof(int), cudaMemcpyHostToDevice, st));
  SYN_CUDA_TRY(cudaEventRecord(p->copied, st));
  p->parted = false;
  return SYN_OK;
} catch (const std::bad_alloc&) {
  return SYN_ERR_OUT_OF_MEMORY;
}

syn_status_t syn_cuda_decode_plan_prefix(const syn_cuda_decode_plan_t* p, size_t row, size_t* len) {
  if (!p || !len) return SYN_ERR_NULL_PTR;
  if (row >= p->rows || p->parted) return SYN_ERR_INVALID_ARG;
  *len = p->prefix[row];
  return SYN_OK;
}

syn_status_t syn_cuda_decode_plan_get_error(syn_cuda_decode_plan_t* p, int32_t* status) {
  if (!p || !status) return SYN_ERR_NULL_PTR;
  DeviceGuard g(p->device);
  if (!g.ok) return SYN_ERR_CUDA;
  int v = 0;
  SYN_CUDA_TRY(cudaDeviceSynchronize());
  SYN_CUDA_TRY(cudaMemcpy(&v, p->err, sizeof(int), cudaMemcpyDeviceToHost));
  SYN_CUDA_TRY(cudaMemset(p->err, 0, sizeof(int)));
  *status = v;
  return SYN_OK;
}

syn_status_t syn_cuda_attention_decode_shared(syn_cuda_decode_plan_t* p, size_t layer,
                                              const float* q, const float* k, const float* v,
                                              size_t ld, const float* q_norm, const float* k_norm,
                                              float eps, const float* rope_cos,
                                              const float* rope_sin, size_t window, float* out,
                                              size_t ldo, void* stream) try {
  if (!p || !q || !k || !v || !rope_cos || !rope_sin || !out) return SYN_ERR_NULL_PTR;
  syn_cuda_kvcache_t* c = p->cache;
  if (!c || layer >= c->layers) return SYN_ERR_INVALID_ARG;
  if (p->parted) return SYN_ERR_INVALID_ARG;
  if (!p->rows) return SYN_OK;
  if (ld < c->hd || ldo < p->n_heads * c->hd) return SYN_ERR_SHAPE_MISMATCH;
  for (size_t i = 0; i < p->rows; i++) {
    const int sq = p->seqs[i];
    if (c->len[sq] + 1 > c->max_seq) return SYN_ERR_INVALID_ARG;  // CacheFull
    // what the rows shared when the plan was set, they must share still
    if (c->len[sq] < p->prefix[i] || (c->page && c->shrunk[sq] != p->shrunk[i]))
      return SYN_ERR_INVALID_ARG;
  }
  DeviceGuard g(p->device);
  if (!g.ok) return SYN_ERR_CUDA;
  cudaStream_t st = (cudaStream_t)stream;
  syn_status_t s;
  for (size_t i = 0; i < p->rows; i++)
    if ((s = kv_reserve(c, p->seqs[i], c->len[p->seqs[i]] + 1, st))) return s;
  cudaStreamCaptureStatus cs = cudaStreamCaptureStatusNone;
  SYN_CUDA_TRY(cudaStreamIsCapturing(st, &cs));
  if (cs != cudaStreamCaptureStatusNone) {
    auto& k = p->captured[p->rows];
    if (p->jobs) k.ctas = p->prefix_ctas;
    else k.without = true;
  }
  AttnArgs a{const_cast<float*>(q), k, v, ld, p->n_heads, q_norm, k_norm, eps, rope_cos, rope_sin,
             window, c, layer, out, ldo};
  return launch_attn_shared(p, a, p->err, st);
} catch (const std::bad_alloc&) {
  return SYN_ERR_OUT_OF_MEMORY;
}

}  // extern "C"
