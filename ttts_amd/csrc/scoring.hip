// Scoring of given tokens and distillation on a teacher's alternatives: row operators over logits [R, ldl], C classes a row.
//   token_logprobs : y = x / T, log p of the given token, entropy, the k best classes with their log p; and the gradient
//   distill        : KL(teacher's listed classes || student), optionally with the mass that the list leaves out; and the gradient
// All sums, maxima and statistics are fp32 whatever the logits' type; a row's maximum m and log Z = log sum e^((x - m) / T) are
// handed to the gradient APART: one log-sum-exp would round log Z to the maximum's step.  Bound by HBM: the logits once (twice and a
// write with the gradient).
#include <math.h>

#include "common.hpp"

namespace ttts {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f, FMAX = 3.402823466e38f;

// ---- one wave = up to 2048 columns of a row, held in registers as fp32 -------------------------------------------------
// A row is read ONCE: maximum, sums, and the alternatives all come from the registers.  Rows up to 2048 columns take one wave, up to 32768
// one workgroup of up to 16 waves that meet in LDS, longer ones several workgroups (segments) and a second kernel that joins
// their results.  A lane holds 8 neighbouring columns per load (16 or 32 bytes, at whatever alignment the row has; only the row's last
// columns are read one by one), 64 lanes 512 neighbouring ones: x[i][j] is column c0 + 512 i + 8 lane + j.
constexpr int NV = 4, WAVE_COLS = NV * 512, MAX_WAVES = 16, SEG_COLS = WAVE_COLS * MAX_WAVES;

struct Split {   // columns of a row -> segments (workgroups) -> waves, in whole 512s: the fewest steps over all waves
  int seg, nseg, waves, wave_cols;
};
static Split split_row(int C) {
  Split s;
  s.nseg = (int)cdiv(C, SEG_COLS);
  s.seg = (int)cdiv(cdiv(C, 512), s.nseg) * 512;
  s.nseg = (int)cdiv(C, s.seg);
  s.waves = (int)cdiv(s.seg, WAVE_COLS);
  s.wave_cols = (int)cdiv(s.seg / 512, s.waves) * 512;
  return s;
}

template <typename T> struct Eight { typedef T type __attribute__((ext_vector_type(8), aligned(sizeof(T)))); };   // 8 columns, aligned to T only
template <typename T>
__device__ __forceinline__ void load8(const T* p, int n, float (&v)[8]) {   // the first n (>= 1) of 8 columns
  if (n >= 8) {
    const typename Eight<T>::type r = *reinterpret_cast<const typename Eight<T>::type*>(p);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = (float)r[j];
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < n ? (float)p[j] : -INFINITY;
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, int n, const float (&v)[8]) {
  if (n >= 8) {
    typename Eight<T>::type r;
#pragma unroll
    for (int j = 0; j < 8; ++j) r[j] = (T)v[j];
    *reinterpret_cast<typename Eight<T>::type*>(p) = r;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < n) p[j] = (T)v[j];
  }
}
// columns c0 .. cend - 1 of a row; columns outside are -inf
template <typename T>
__device__ __forceinline__ void load_wave(const T* row, int c0, int cend, int lane, float (&x)[NV][8]) {
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = c0 + i * 512 + lane * 8;
    if (c0 + i * 512 + 512 <= cend) {
      load8<T>(row + c, 8, x[i]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[i][j] = -INFINITY;
      if (c < cend) load8<T>(row + c, cend - c, x[i]);
    }
  }
}

// e = 2^((x - m) c); t = (x - m) c kept finite (a class at -inf, or at the type's lowest value, has e = 0: e t must be 0, not NaN).
// m is never -inf here (>= -FMAX), so -inf - m = -inf; NaN passes through e.  The difference comes first: lowest - lowest is 0.
__device__ __forceinline__ float expo(float x, float m, float c, float& t) {
  t = (x - m) * c;
  const float e = __builtin_amdgcn_exp2f(t);
  t = fmaxf(t, -200.f);
  return e;
}
__device__ __forceinline__ void wave_fence() {   // LDS written by this wave's lanes is read by its other lanes
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// ---- the k best columns --------------------------------------------------------------------------------------------------
// Order: larger value first, lower class first among equals.  A 64-bit key holds both: the value's bits in the order of the numbers
// (zeros of both signs the same), and the class, inverted; key 0 is none.
typedef unsigned long long u64;
__device__ __forceinline__ uint32_t ord(float v) {
  const uint32_t b = __builtin_bit_cast(uint32_t, v + 0.f);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float unord(uint32_t u) { return __builtin_bit_cast(float, (u & 0x80000000u) ? u ^ 0x80000000u : ~u); }
__device__ __forceinline__ u64 top_key(float v, int c) { return ((u64)ord(v) << 32) | (uint32_t)~c; }
__device__ __forceinline__ int key_class(u64 k) { return (int)~(uint32_t)k; }
constexpr uint32_t ORD_NONE = 0x007fffffu;   // ord(-inf)
__device__ __forceinline__ int lanes_below(u64 mask) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
}

// A threshold first: the k-th largest of the maxima of groups of columns is at most the k-th largest column, and few columns reach it
// (k + 10 .. 30 % of ordinary rows).  It is found bit by bit with ballots over n group maxima a lane, and any value that exactly k
// groups reach will do (early).  What reaches it lies in at most k groups, unless values repeat at the threshold: then (exact) fewer
// than k groups go above it, and of the columns AT it the lowest classes are taken, as many as are needed.
template <int N>
__device__ __forceinline__ float group_threshold(const uint32_t (&g)[N], int n, int k, bool early) {
  uint32_t t = 0;
  for (uint32_t bit = 0x80000000u; bit; bit >>= 1) {
    const uint32_t c = t | bit;
    int cnt = 0;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < n) cnt += __builtin_popcountll(__ballot(g[i] >= c));
    if (cnt >= k) {
      t = c;
      if (early && cnt == k) break;
    }
  }
  return t <= ORD_NONE ? -FMAX : unord(t);   // (a class at -inf is no alternative)
}
// bit 31 - (8 i + j): x[i][j] reaches the threshold / is above it
template <bool ABOVE>
__device__ __forceinline__ uint32_t reached(const float (&x)[NV][8], float thr, int c0, int cend) {
  uint32_t bits = 0;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (c0 + i * 512 < cend) {
#pragma unroll
      for (int j = 0; j < 8; ++j) bits = bits + bits + (ABOVE ? x[i][j] > thr : x[i][j] >= thr);
    } else {
      bits <<= 8;
    }
  }
  return bits;
}
// the columns marked in `bits` become keys from place n on (those before `cap`); their values are read again (a register cannot be
// indexed by a lane).  Returns the place behind the last.
template <typename T, typename Place>
__device__ __forceinline__ void collect(uint32_t bits, const T* row, int c0, int lane, u64* cand, int cap, Place place) {
  for (u64 mask = __ballot(bits != 0); mask; mask = __ballot(bits != 0)) {
    const int at = place(mask);
    if (bits) {
      const int e = __builtin_clz(bits), c = c0 + (e >> 3) * 512 + lane * 8 + (e & 7);
      bits &= ~(0x80000000u >> e);
      if (at < cap) cand[at] = top_key((float)row[c], c);
    }
  }
}
// columns equal to thr, lowest classes first, become keys from place n on, up to `end`; first: ties of earlier waves.  Returns n + ties.
__device__ __forceinline__ int collect_ties(const float (&x)[NV][8], float thr, int c0, int lane, u64* cand, int n, int end) {
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    int mine = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) mine += x[i][j] == thr;
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int v = __shfl_up(upto, o, 64);
      if (lane >= o) upto += v;
    }
    int at = n + upto - mine;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (x[i][j] == thr) {
        if (at < end) cand[at] = top_key(x[i][j], c0 + i * 512 + lane * 8 + j);
        ++at;
      }
    n += __shfl(upto, 63, 64);
  }
  return n;
}
// f(rank, key) for the keys of rank < k among n distinct ones (cand[n] and cand[n + 1] writable): ranked by counting
template <typename F>
__device__ __forceinline__ void rank_keys(u64* cand, int n, int k, int thread, int threads, F f) {
  for (int s = thread; s < n; s += threads) {
    const u64 key = cand[s];
    int r = 0;
    for (int j = 0; j < n; j += 2) r += (cand[j] > key) + (cand[j + 1] > key);
    if (r < k) f(r, key);
  }
}
constexpr int WAVE_CAND = 64 * 8 + 64, WAVE_TOP_LDS = WAVE_CAND + 2;      // one wave: groups of 8 columns (exact)
constexpr int GROUP_CAND = 64 * 32 + 64;                                  // a workgroup: a lane's 32 columns are a group
// one wave: f(rank, key) of its k best; returns how many there are (<= k)
template <typename T, typename F>
__device__ __forceinline__ int wave_top(const float (&x)[NV][8], const float (&vmax)[NV], const T* row, int c0, int cend, int k, int lane, u64* cand,
                                        F f) {
  uint32_t g[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) g[i] = ord(vmax[i]);
  float thr;
  if (k <= 32) {          // groups of a lane's 32 columns: one ballot a bit
    const uint32_t one[1] = {max(max(g[0], g[1]), max(g[2], g[3]))};
    thr = group_threshold<1>(one, 1, k, true);
  } else {                // of 8 columns: with 64 groups the least of them would have to do
    thr = group_threshold<NV>(g, NV, k, true);
  }
  int n = 0;
  auto next = [&](u64 mask) { const int at = n + lanes_below(mask); n += __builtin_popcountll(mask); return at; };
  collect<T>(reached<false>(x, thr, c0, cend), row, c0, lane, cand, WAVE_CAND, next);
  if (n > WAVE_CAND) {
    thr = group_threshold<NV>(g, NV, k, false);
    n = 0;
    collect<T>(reached<true>(x, thr, c0, cend), row, c0, lane, cand, WAVE_CAND, next);
    const int end = max(n, k);
    n = min(end, collect_ties(x, thr, c0, lane, cand, n, end));
  }
  if (lane < 2) cand[n + lane] = 0;
  wave_fence();
  rank_keys(cand, n, k, lane, 64, f);
  return min(n, k);
}
// place of list w's entry r among `lists` sorted lists of k (stride in u64): its own, and in each other one those above it
__device__ __forceinline__ int merged_rank(const u64* base, int stride, int lists, int w, int r, int k, u64 key) {
  int rank = r;
  for (int o = 0; o < lists; ++o) {
    if (o == w) continue;
    const u64* l = base + o * stride;
    int lo = 0, hi = k;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (l[mid] > key) lo = mid + 1; else hi = mid;
    }
    rank += lo;
    if (rank >= k) break;
  }
  return rank;
}

struct RowSums { float m, z, s; };   // maximum, sum e, sum e t (t in bits, from the maximum)
__device__ __forceinline__ void add_sums(RowSums& a, float m, float z, float s, float M, float c) {   // a's maximum is M already
  const float d = fmaxf((m - M) * c, -200.f), f = __builtin_amdgcn_exp2f(d);
  a.z += z * f;
  a.s += f * (s + z * d);
}

struct ScoreParams {
  const void* logits; int64_t ldl;
  const int64_t* tokens;
  float *logp, *entropy, *stats, *top_logp;
  int64_t* top_idx;
  float4* part;      // [R, nseg] (m, z, s, -) of the segments of a long row, and their sorted keys [R, nseg, k]
  u64* part_key;
  int R, C, k;
  float inv_t;
  Split sp;
};

__device__ __forceinline__ void write_row(const ScoreParams& p, int64_t row, const RowSums& a, bool given, float xt) {
  const bool none = a.z == 0.f;   // every class at -inf
  const float log2z = __builtin_amdgcn_logf(a.z);
  p.stats[2 * row] = none ? -INFINITY : a.m;
  p.stats[2 * row + 1] = none ? -INFINITY : log2z * LN2;
  p.entropy[row] = none ? 0.f : (log2z - a.s / a.z) * LN2;
  p.logp[row] = !given ? 0.f : none ? -INFINITY : (xt - a.m) * p.inv_t - log2z * LN2;
}
__device__ __forceinline__ void write_top(const ScoreParams& p, int64_t row, int r, u64 key, const RowSums& a) {
  const bool nan = a.z != a.z, have = key != 0 && !nan;
  p.top_idx[row * p.k + r] = have ? key_class(key) : -1;
  p.top_logp[row * p.k + r] = have ? (unord((uint32_t)(key >> 32)) - a.m) * p.inv_t - __builtin_amdgcn_logf(a.z) * LN2 : nan ? a.z : -INFINITY;
}

// MULTI false: a wave per row, four rows a workgroup, no barrier.  MULTI: a workgroup per segment of a row; its alternatives come from one
// threshold over all its lanes (with a list per wave, 64 alternatives of 100003 classes took 570 us instead of TOPTIME).
template <typename T, bool MULTI>
__global__ __launch_bounds__(MULTI ? 1024 : 256) void token_logprobs_fwd_kernel(ScoreParams p) {
  extern __shared__ __attribute__((aligned(16))) u64 score_lds[];
  __shared__ RowSums sm[MULTI ? MAX_WAVES : 1];
  __shared__ int sm_n[MAX_WAVES + 2];    // ties of each wave; [MAX_WAVES]: keys so far; [MAX_WAVES + 1]: the threshold's bits
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t unit = MULTI ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * 4 + wave;
  const int64_t row = MULTI ? blockIdx.x / (unsigned)p.sp.nseg : unit;
  if (row >= p.R) return;
  const int seg = MULTI ? (int)(blockIdx.x % (unsigned)p.sp.nseg) : 0;
  const T* lr = (const T*)p.logits + row * p.ldl;
  const int64_t tok = p.tokens[row];
  const bool given = tok >= 0 && tok < p.C;
  const float xt = given ? (float)lr[tok] : 0.f;      // (its latency runs beside the row's)
  const int send = MULTI ? min(p.C, (seg + 1) * p.sp.seg) : p.C;
  const int c0 = MULTI ? seg * p.sp.seg + wave * p.sp.wave_cols : 0, cend = MULTI ? min(send, c0 + p.sp.wave_cols) : p.C;
  const float c = p.inv_t * LOG2E;
  float x[NV][8], vmax[NV];
  load_wave<T>(lr, c0, cend, lane, x);
  float m = -FMAX, lmax = -INFINITY;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    vmax[i] = -INFINITY;
#pragma unroll
    for (int j = 0; j < 8; ++j) vmax[i] = fmaxf(vmax[i], x[i][j]);
    lmax = fmaxf(lmax, vmax[i]);
  }
  RowSums a;
  a.m = wave_max(fmaxf(m, lmax));
  a.z = a.s = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (c0 + i * 512 < cend)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float t;
        const float e = expo(x[i][j], a.m, c, t);
        a.z += e;
        a.s = fmaf(e, t, a.s);
      }
  a.z = wave_sum(a.z);
  a.s = wave_sum(a.s);
  if (!MULTI) {
    if (lane == 0) write_row(p, row, a, given, xt);
    if (p.k) {
      const int have = wave_top<T>(x, vmax, lr, c0, cend, p.k, lane, score_lds + wave * WAVE_TOP_LDS, [&](int r, u64 key) { write_top(p, row, r, key, a); });
      if (lane >= have && lane < p.k) write_top(p, row, lane, 0, a);
    }
    return;
  }
  const int nw = p.sp.waves;
  u64* cand = score_lds;                                                       // [GROUP_CAND + 2]
  uint32_t* gmax = reinterpret_cast<uint32_t*>(score_lds + GROUP_CAND + 2);    // [nw][64]
  if (lane == 0) sm[wave] = a;
  if (p.k) gmax[threadIdx.x] = ord(lmax);
  if (threadIdx.x == 0) sm_n[MAX_WAVES] = 0;
  __syncthreads();
  RowSums b = {sm[0].m, 0.f, 0.f};
  for (int w = 1; w < nw; ++w) b.m = fmaxf(b.m, sm[w].m);
  for (int w = 0; w < nw; ++w) add_sums(b, sm[w].m, sm[w].z, sm[w].s, b.m, c);
  const bool whole = p.sp.nseg == 1;
  if (threadIdx.x == 0) {
    if (whole) write_row(p, row, b, given, xt);
    else p.part[unit] = make_float4(b.m, b.z, b.s, 0.f);
  }
  if (!p.k) return;
  if (wave == 0) {
    uint32_t g[MAX_WAVES];
#pragma unroll
    for (int w = 0; w < MAX_WAVES; ++w) g[w] = w < nw ? gmax[w * 64 + lane] : 0;
    const float thr = group_threshold<MAX_WAVES>(g, nw, p.k, true);
    if (lane == 0) sm_n[MAX_WAVES + 1] = __builtin_bit_cast(int, thr);
  }
  __syncthreads();
  const float thr = __builtin_bit_cast(float, sm_n[MAX_WAVES + 1]);
  auto next = [&](u64 mask) {
    int base = 0;
    if (lane == 0) base = atomicAdd(&sm_n[MAX_WAVES], __builtin_popcountll(mask));
    return __builtin_amdgcn_readfirstlane(base) + lanes_below(mask);
  };
  if (__any(lmax >= thr)) collect<T>(reached<false>(x, thr, c0, cend), lr, c0, lane, cand, GROUP_CAND, next);
  __syncthreads();
  int n = sm_n[MAX_WAVES];
  if (n > GROUP_CAND) {   // values repeat at the threshold (the k-th group's own then: exactly k groups hold no more than GROUP_CAND)
    int ties = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) ties += __builtin_popcountll(__ballot(x[i][j] == thr));
    __syncthreads();
    if (threadIdx.x == 0) sm_n[MAX_WAVES] = 0;
    if (lane == 0) sm_n[wave] = ties;
    __syncthreads();
    collect<T>(reached<true>(x, thr, c0, cend), lr, c0, lane, cand, GROUP_CAND, next);
    __syncthreads();
    n = sm_n[MAX_WAVES];
    const int end = max(n, p.k);
    int all = n, mine = n;
    for (int w = 0; w < nw; ++w) {
      if (w < wave) mine += sm_n[w];
      all += sm_n[w];
    }
    if (mine < end) collect_ties(x, thr, c0, lane, cand, mine, end);
    n = min(all, end);
  }
  if (threadIdx.x < 2) cand[n + threadIdx.x] = 0;
  __syncthreads();
  rank_keys(cand, n, p.k, threadIdx.x, 64 * nw, [&](int r, u64 key) {
    if (whole) write_top(p, row, r, key, b);
    else p.part_key[unit * p.k + r] = key;
  });
  for (int r = n + threadIdx.x; r < p.k; r += 64 * nw) {
    if (whole) write_top(p, row, r, 0, b);
    else p.part_key[unit * p.k + r] = 0;
  }
}

// the segments of a long row: at most 32 of them, their sums in one wave, their lists as the waves' above
template <typename T>
__global__ __launch_bounds__(256) void token_logprobs_join_kernel(ScoreParams p) {
  extern __shared__ __attribute__((aligned(16))) u64 score_lds[];   // [nseg][k]
  const int64_t row = blockIdx.x;
  const int lane = threadIdx.x & 63, nseg = p.sp.nseg, total = nseg * p.k;
  for (int i = threadIdx.x; i < total; i += 256) score_lds[i] = p.part_key[row * total + i];
  float4 s = make_float4(-FMAX, 0.f, 0.f, 0.f);
  if (lane < nseg) s = p.part[row * nseg + lane];
  RowSums a = {wave_max(s.x), 0.f, 0.f};
  add_sums(a, s.x, s.y, s.z, a.m, p.inv_t * LOG2E);
  a.z = wave_sum(a.z);
  a.s = wave_sum(a.s);
  if (threadIdx.x == 0) {
    const int64_t tok = p.tokens[row];
    const bool given = tok >= 0 && tok < p.C;
    write_row(p, row, a, given, given ? (float)((const T*)p.logits)[row * p.ldl + tok] : 0.f);
  }
  if (!p.k) return;
  __syncthreads();
  int have = 0;
  for (int i = lane; i < total; i += 64) have += score_lds[i] != 0;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) have += __shfl_xor(have, o, 64);
  for (int i = threadIdx.x; i < total; i += 256) {
    const u64 key = score_lds[i];
    if (!key) continue;
    const int r = merged_rank(score_lds, p.k, nseg, i / p.k, i % p.k, p.k, key);
    if (r < p.k) write_top(p, row, r, key, a);
  }
  for (int r = threadIdx.x; r < p.k; r += 256)
    if (r >= have) write_top(p, row, r, 0, a);
}

// (n / d, n % d) of a piece's number: in 32 bits where it fits (a 64-bit division costs as much as the piece's work)
__device__ __forceinline__ void split_id(int64_t n, int d, int64_t& q, int& r) {
  if ((uint64_t)n >> 32) { q = n / d; r = (int)(n % d); }
  else { q = (uint32_t)n / (uint32_t)d; r = (int)((uint32_t)n % (uint32_t)d); }
}

// ---- gradient of the log-probabilities: one thread per 8 columns, everything of the row is known -------------------------
struct ScoreGradParams {
  const void* logits; int64_t ldl;
  const int64_t* tokens;
  const float *stats, *entropy, *g_logp, *g_entropy;
  void* dlogits; int64_t ldd;
  int C, Cd, per_row;   // per_row: 8-column pieces of a row
  int64_t pieces;
  float inv_t;
};
template <typename T>
__global__ __launch_bounds__(256) void token_logprobs_bwd_kernel(ScoreGradParams p) {
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (id >= p.pieces) return;
  int64_t row;
  int piece;
  split_id(id, p.per_row, row, piece);
  const int first = piece * 8;
  float v[8];
  if (first < p.C) load8<T>((const T*)p.logits + row * p.ldl + first, p.C - first, v);
  const float m = p.stats[2 * row], logz = p.stats[2 * row + 1], H = p.entropy[row];
  const int64_t tok = p.tokens[row];
  const bool given = tok >= 0 && tok < p.C;
  const float gl = given ? p.g_logp[row] : 0.f, gh = p.g_entropy ? p.g_entropy[row] : 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    float g = 0.f;
    if (first + j < p.C && m != -INFINITY) {
      const float y = (v[j] - m) * p.inv_t - logz;
      const float q = __builtin_amdgcn_exp2f(y * LOG2E);
      g = q == 0.f ? 0.f : -q * (gl + gh * (y + H));
      if (given && first + j == (int)tok) g += gl;
      g *= p.inv_t;
    }
    v[j] = g;
  }
  store8<T>((T*)p.dlogits + row * p.ldd + first, p.Cd - first, v);
}

// ---- distillation ---------------------------------------------------------------------------------------------------------
// A row's list, two entries a lane: class (or -1), p and log p, and the list's mass.
struct Listed { int id[2]; float p[2], logp[2], mass; };
__device__ __forceinline__ Listed load_listed(const int64_t* idx, const float* tl, int K, int C, float inv_t, int tail, int lane) {
  Listed L;
  float t[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int j = lane + 64 * h;
    L.id[h] = -1;
    t[h] = -INFINITY;
    if (j < K) {
      const int64_t i = idx[j];
      const float v = tl[j];
      if (i >= 0 && i < C) { L.id[h] = (int)i; t[h] = v; }
    }
  }
  if (tail) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      L.logp[h] = t[h];
      L.p[h] = L.id[h] >= 0 ? __expf(t[h]) : 0.f;
    }
  } else {
    const float m = fmaxf(wave_max(fmaxf(t[0], t[1])), -FMAX);
    float e[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      L.logp[h] = (t[h] - m) * inv_t;
      e[h] = L.id[h] >= 0 ? __expf(L.logp[h]) : 0.f;
    }
    const float z = wave_sum(e[0] + e[1]);
    const float logz = __logf(z);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      L.p[h] = z == 0.f ? 0.f : e[h] / z;
      L.logp[h] -= logz;
    }
  }
  L.mass = wave_sum(L.p[0] + L.p[1]);
  return L;
}

struct DistillParams {
  const void* logits; int64_t ldl;
  const int64_t* idx;
  const float* tlogp;
  float *row_loss, *stats;
  float4* part;        // [R, nseg] (m, z of the listed classes, z of the others, -)
  int R, C, K, tail;
  float inv_t;
  Split sp;
};
// by one wave: the row's loss from its sums (listed and other classes apart with tail, else all in zr) and the listed classes' logits
__device__ __forceinline__ void finish_distill(const DistillParams& p, int64_t row, const Listed& L, const float (&xl)[2], float m, float zl, float zr,
                                               int lane) {
  const float z = zl + zr, logz = __logf(z);
  float loss = 0.f;
#pragma unroll
  for (int h = 0; h < 2; ++h)
    if (L.p[h] != 0.f) loss += L.p[h] * (L.logp[h] - ((xl[h] - m) * p.inv_t - logz));
  loss = wave_sum(loss);
  if (lane == 0) {
    const float left = 1.f - L.mass;
    // log of the student's rest = -log(1 + listed / others): the difference of two log-sums would lose it where little is listed
    if (p.tail && left > 0.f && zr > 0.f) loss += left * (log1pf(-L.mass) + log1pf(zl / zr));
    const bool none = z == 0.f;
    p.row_loss[row] = none ? 0.f : loss;
    p.stats[3 * row] = none ? -INFINITY : m;
    p.stats[3 * row + 1] = none ? -INFINITY : logz;
    p.stats[3 * row + 2] = none || !p.tail ? 0.f : zl / zr;
  }
}
template <typename T>
__device__ __forceinline__ void listed_logits(const T* row, const Listed& L, float (&xl)[2]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) xl[h] = L.id[h] >= 0 ? (float)row[L.id[h]] : 0.f;
}

// as token_logprobs_fwd_kernel; with tail each wave marks the listed classes of its columns in a bit map of its own
template <typename T, bool MULTI>
__global__ __launch_bounds__(MULTI ? 1024 : 256) void distill_fwd_kernel(DistillParams p) {
  __shared__ uint32_t marks[MULTI ? MAX_WAVES : 4][WAVE_COLS / 32];
  __shared__ RowSums sm[MAX_WAVES];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t unit = MULTI ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * 4 + wave;
  const int64_t row = MULTI ? blockIdx.x / (unsigned)p.sp.nseg : unit;
  if (row >= p.R) return;
  const int seg = MULTI ? (int)(blockIdx.x % (unsigned)p.sp.nseg) : 0;
  const T* lr = (const T*)p.logits + row * p.ldl;
  const int send = MULTI ? min(p.C, (seg + 1) * p.sp.seg) : p.C;
  const int c0 = MULTI ? seg * p.sp.seg + wave * p.sp.wave_cols : 0, cend = MULTI ? min(send, c0 + p.sp.wave_cols) : p.C;
  const float c = p.inv_t * LOG2E;
  float x[NV][8];
  load_wave<T>(lr, c0, cend, lane, x);
  const bool first = wave == 0 || !MULTI, whole = !MULTI || p.sp.nseg == 1;
  Listed L;
  float xl[2] = {0.f, 0.f};
  if (p.tail || (first && whole)) L = load_listed(p.idx + row * p.K, p.tlogp + row * p.K, p.K, p.C, p.inv_t, p.tail, lane);
  if (first && whole) listed_logits(lr, L, xl);
  uint32_t* mark = marks[wave];
  if (p.tail) {
    mark[lane] = 0;
    wave_fence();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int at = L.id[h] - c0;
      if (L.id[h] >= c0 && L.id[h] < cend) atomicOr(&mark[at >> 5], 1u << (at & 31));
    }
    wave_fence();
  }
  float m = -FMAX;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) m = fmaxf(m, x[i][j]);
  m = wave_max(m);
  float zl = 0.f, zr = 0.f;
  if (p.tail) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (c0 + i * 512 >= cend) break;
      const uint32_t bits = reinterpret_cast<const uint8_t*>(mark)[i * 64 + lane];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float e = __builtin_amdgcn_exp2f((x[i][j] - m) * c);
        const bool hit = (bits >> j) & 1u;
        zl += hit ? e : 0.f;
        zr += hit ? 0.f : e;
      }
    }
    zl = wave_sum(zl);
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (c0 + i * 512 >= cend) break;
#pragma unroll
      for (int j = 0; j < 8; ++j) zr += __builtin_amdgcn_exp2f((x[i][j] - m) * c);
    }
  }
  zr = wave_sum(zr);
  if (!MULTI) {
    finish_distill(p, row, L, xl, m, zl, zr, lane);
    return;
  }
  if (lane == 0) sm[wave] = RowSums{m, zl, zr};
  __syncthreads();
  if (wave) return;
  float M = sm[0].m, Zl = 0.f, Zr = 0.f;
  for (int w = 1; w < p.sp.waves; ++w) M = fmaxf(M, sm[w].m);
  for (int w = 0; w < p.sp.waves; ++w) {
    const float f = __builtin_amdgcn_exp2f((sm[w].m - M) * c);
    Zl += sm[w].z * f;
    Zr += sm[w].s * f;
  }
  if (whole) finish_distill(p, row, L, xl, M, Zl, Zr, lane);
  else if (lane == 0) p.part[unit] = make_float4(M, Zl, Zr, 0.f);
}
template <typename T>
__global__ __launch_bounds__(256) void distill_join_kernel(DistillParams p) {   // a wave per row; at most 32 segments
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= p.R) return;
  float4 s = make_float4(-FMAX, 0.f, 0.f, 0.f);
  if (lane < p.sp.nseg) s = p.part[row * p.sp.nseg + lane];
  const Listed L = load_listed(p.idx + row * p.K, p.tlogp + row * p.K, p.K, p.C, p.inv_t, p.tail, lane);
  float xl[2];
  listed_logits((const T*)p.logits + row * p.ldl, L, xl);
  const float m = wave_max(s.x), f = __builtin_amdgcn_exp2f((s.x - m) * p.inv_t * LOG2E);
  const float zl = wave_sum(s.y * f), zr = wave_sum(s.z * f);
  finish_distill(p, row, L, xl, m, zl, zr, lane);
}

struct DistillGradParams {
  const void* logits; int64_t ldl;
  const int64_t* idx;
  const float *tlogp, *stats, *g_loss;
  void* dlogits; int64_t ldd;
  int C, Cd, K, tail, accumulate, per_row, wave_cols;
  int64_t units;
  float inv_t;
};
// A wave on its own takes up to 2048 columns of a row.  With q = softmax(y) and w = (listed / other mass of the student),
//   d / dy = q (mass - left w) on the classes that the list does not name (left: the mass it leaves out; 0 without tail)
//          = q (mass + left) - p on those it names:
// one exponential a class by the first form, then the few named ones again by the second, each by the lane that holds its entry (whose
// logit, and what is accumulated to, is fetched beside the row; a wave's own stores to one address stay in order).  Entries that
// name one class find out by leaving their number at its place in LDS: each then writes the sum of their p, in the list's order.
template <typename T>
__global__ __launch_bounds__(256) void distill_bwd_kernel(DistillGradParams p) {
  __shared__ uint8_t tags[4][WAVE_COLS];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t unit = (int64_t)blockIdx.x * 4 + wave;
  if (unit >= p.units) return;
  int64_t row;
  int piece;
  split_id(unit, p.per_row, row, piece);
  const int c0 = piece * p.wave_cols, dend = min(p.Cd, c0 + p.wave_cols), cend = min(p.C, dend);
  const T* lr = (const T*)p.logits + row * p.ldl;
  T* dr = (T*)p.dlogits + row * p.ldd;
  float x[NV][8];
  load_wave<T>(lr, c0, cend, lane, x);
  Listed L = load_listed(p.idx + row * p.K, p.tlogp + row * p.K, p.K, p.C, p.inv_t, p.tail, lane);
  const float m = p.stats[3 * row], logz = p.stats[3 * row + 1], w = p.stats[3 * row + 2], g = p.g_loss[row] * p.inv_t;
  uint8_t* tag = tags[wave];
  bool here[2];
  float xl[2] = {0.f, 0.f}, old[2] = {0.f, 0.f};
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    here[h] = L.id[h] >= c0 && L.id[h] < cend;
    if (here[h]) {
      tag[L.id[h] - c0] = (uint8_t)(lane + 64 * h);
      xl[h] = (float)lr[L.id[h]];
      if (p.accumulate) old[h] = (float)dr[L.id[h]];
    }
  }
  wave_fence();
  bool twice = false;
#pragma unroll
  for (int h = 0; h < 2; ++h) twice |= here[h] && tag[L.id[h] - c0] != (uint8_t)(lane + 64 * h);
  if (__any(twice)) {
    float sum[2] = {0.f, 0.f};
    for (int j = 0; j < p.K; ++j) {
      const int idj = __shfl(j < 64 ? L.id[0] : L.id[1], j & 63, 64);
      const float pj = __shfl(j < 64 ? L.p[0] : L.p[1], j & 63, 64);
#pragma unroll
      for (int h = 0; h < 2; ++h) sum[h] += idj == L.id[h] ? pj : 0.f;
    }
    L.p[0] = sum[0];
    L.p[1] = sum[1];
  }
  const bool held = p.tail && w < INFINITY;          // other classes than the listed ones hold something
  const float left = held ? fmaxf(1.f - L.mass, 0.f) : 0.f;
  const bool none = m == -INFINITY;                  // every class at -inf: no gradient
  const float on = L.mass + left, off = (left > 0.f ? L.mass - left * w : L.mass) * g;
  const float c = p.inv_t * LOG2E, log2z = logz * LOG2E;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int first = c0 + i * 512 + lane * 8;
    if (c0 + i * 512 >= dend) break;
    float d[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) d[j] = __builtin_amdgcn_exp2f((x[i][j] - m) * c - log2z) * off;
    if (none || c0 + i * 512 + 512 > p.C) {
#pragma unroll
      for (int j = 0; j < 8; ++j) d[j] = first + j < p.C && !none ? d[j] : 0.f;
    }
    const int n = (p.accumulate ? cend : dend) - first;
    if (n <= 0) continue;
    if (p.accumulate) {
      float o[8];
      load8<T>(dr + first, n, o);
#pragma unroll
      for (int j = 0; j < 8; ++j) d[j] += o[j];
    }
    store8<T>(dr + first, n, d);
  }
  wave_fence();
  if (none) return;
#pragma unroll
  for (int h = 0; h < 2; ++h)
    if (here[h]) {
      const float q = __builtin_amdgcn_exp2f((xl[h] - m) * c - log2z);
      dr[L.id[h]] = (T)(old[h] + fmaf(q, on, -L.p[h]) * g);
    }
}

// run F<T> for the logits' type
#define TTTS_BY_TYPE(dtype, what, CALL)                                             \
  switch (dtype) {                                                                  \
    case TTTS_DTYPE_F32: { using T = float; CALL; break; }                          \
    case TTTS_DTYPE_BF16: { using T = bf16; CALL; break; }                          \
    case TTTS_DTYPE_F16: { using T = _Float16; CALL; break; }                       \
    default: return fail(TTTS_EINVAL, what ": unknown type code %d", (int)(dtype)); \
  }

}  // namespace ttts

using namespace ttts;

static int check_logits(const char* what, const void* logits, int32_t dtype, int64_t ldl, int32_t R, int32_t C, float temperature) {
  TTTS_REQUIRE(dtype == TTTS_DTYPE_F32 || dtype == TTTS_DTYPE_BF16 || dtype == TTTS_DTYPE_F16, "%s: unknown type code %d", what, (int)dtype);
  TTTS_REQUIRE(R >= 0 && C > 0 && C <= TTTS_SCORE_MAX_CLASSES && ldl >= C, "%s: need R >= 0, 0 < C <= %d, ldl >= C (R %d, C %d, ldl %lld)", what,
               TTTS_SCORE_MAX_CLASSES, R, C, (long long)ldl);
  TTTS_REQUIRE(temperature > 0.f && temperature <= 3.0e38f && 1.0f / temperature <= 3.0e38f, "%s: the temperature must be positive and finite", what);
  TTTS_REQUIRE(R == 0 || logits, "%s: null pointer", what);
  const uintptr_t es = dtype == TTTS_DTYPE_F32 ? 4 : 2;
  TTTS_REQUIRE(reinterpret_cast<uintptr_t>(logits) % es == 0, "%s: logits are not aligned to their type", what);
  return TTTS_OK;
}

static int need_workspace(const char* what, int64_t need, const void* ws, int64_t have) {
  TTTS_REQUIRE(need == 0 || (ws && have >= need && aligned16(ws)), "%s: needs a 16-byte aligned workspace of %lld bytes", what, (long long)need);
  return TTTS_OK;
}
static int need_grid(const char* what, int64_t grid) {
  TTTS_REQUIRE(grid <= 0x7fffffff, "%s: more work than one launch holds", what);
  return TTTS_OK;
}

extern "C" int64_t ttts_token_logprobs_workspace_bytes(int32_t R, int32_t C, int32_t top_k) {
  if (R <= 0 || C <= 0 || top_k < 0) return 0;
  const Split sp = split_row(C);
  return sp.nseg > 1 ? cdiv((int64_t)R * sp.nseg * (16 + 8 * (int64_t)top_k), 16) * 16 : 0;
}

template <typename T>
static int launch_score(const ScoreParams& p, hipStream_t st) {
  const char* what = "token_logprobs_fwd";
  if (p.sp.nseg == 1 && p.sp.waves == 1) {
    token_logprobs_fwd_kernel<T, false><<<(unsigned)cdiv(p.R, 4), 256, p.k ? 4 * WAVE_TOP_LDS * 8 : 0, st>>>(p);
    return check_launch(what);
  }
  const int64_t grid = (int64_t)p.R * p.sp.nseg;
  int rc = need_grid(what, grid);
  if (rc) return rc;
  token_logprobs_fwd_kernel<T, true><<<(unsigned)grid, 64 * p.sp.waves, p.k ? (GROUP_CAND + 2) * 8 + p.sp.waves * 64 * 4 : 0, st>>>(p);
  rc = check_launch(what);
  if (rc || p.sp.nseg == 1) return rc;
  token_logprobs_join_kernel<T><<<p.R, 256, p.sp.nseg * p.k * 8, st>>>(p);
  return check_launch("token_logprobs_fwd join");
}

extern "C" int ttts_token_logprobs_fwd(const void* logits, int32_t dtype, int64_t ldl, const int64_t* tokens, float* logp, float* entropy,
                                       float* stats, float* top_logp, int64_t* top_idx, int32_t R, int32_t C, int32_t top_k,
                                       float temperature, void* workspace, int64_t workspace_bytes, void* stream) {
  int rc = check_logits("token_logprobs_fwd", logits, dtype, ldl, R, C, temperature);
  if (rc) return rc;
  TTTS_REQUIRE(top_k >= 0 && top_k <= TTTS_SCORE_MAX_TOP, "token_logprobs_fwd: need 0 <= top_k <= %d", TTTS_SCORE_MAX_TOP);
  if (R == 0) return TTTS_OK;
  TTTS_REQUIRE(tokens && logp && entropy && stats && (top_k == 0 || (top_logp && top_idx)), "token_logprobs_fwd: null pointer");
  rc = need_workspace("token_logprobs_fwd", ttts_token_logprobs_workspace_bytes(R, C, top_k), workspace, workspace_bytes);
  if (rc) return rc;
  ScoreParams p{logits, ldl, tokens, logp, entropy, stats, top_logp, top_idx, (float4*)workspace, nullptr, R, C, top_k, 1.0f / temperature, split_row(C)};
  p.part_key = (u64*)(p.part + (int64_t)R * p.sp.nseg);
  TTTS_BY_TYPE(dtype, "token_logprobs_fwd", rc = launch_score<T>(p, as_stream(stream)));
  return rc;
}

extern "C" int ttts_token_logprobs_bwd(const void* logits, int32_t dtype, int64_t ldl, const int64_t* tokens, const float* stats,
                                       const float* entropy, const float* g_logp, const float* g_entropy, void* dlogits, int64_t ldd,
                                       int32_t R, int32_t C, int32_t Cd, float temperature, void* stream) {
  int rc = check_logits("token_logprobs_bwd", logits, dtype, ldl, R, C, temperature);
  if (rc) return rc;
  TTTS_REQUIRE(Cd >= C && ldd >= Cd, "token_logprobs_bwd: need C <= Cd <= ldd");
  if (R == 0) return TTTS_OK;
  TTTS_REQUIRE(tokens && stats && entropy && g_logp && dlogits, "token_logprobs_bwd: null pointer");
  const int per_row = (int)cdiv(Cd, 8);
  const ScoreGradParams p{logits, ldl, tokens, stats, entropy, g_logp, g_entropy, dlogits, ldd, C, Cd, per_row, (int64_t)R * per_row, 1.0f / temperature};
  const int64_t grid = cdiv(p.pieces, 256);
  rc = need_grid("token_logprobs_bwd", grid);
  if (rc) return rc;
  TTTS_BY_TYPE(dtype, "token_logprobs_bwd", (token_logprobs_bwd_kernel<T><<<(unsigned)grid, 256, 0, as_stream(stream)>>>(p)));
  return check_launch("token_logprobs_bwd");
}

extern "C" int64_t ttts_distill_workspace_bytes(int32_t R, int32_t C) {
  if (R <= 0 || C <= 0) return 0;
  const Split sp = split_row(C);
  return sp.nseg > 1 ? (int64_t)R * sp.nseg * 16 : 0;
}

template <typename T>
static int launch_distill(const DistillParams& p, hipStream_t st) {
  const char* what = "distill_fwd";
  if (p.sp.nseg == 1 && p.sp.waves == 1) {
    distill_fwd_kernel<T, false><<<(unsigned)cdiv(p.R, 4), 256, 0, st>>>(p);
    return check_launch(what);
  }
  const int64_t grid = (int64_t)p.R * p.sp.nseg;
  int rc = need_grid(what, grid);
  if (rc) return rc;
  distill_fwd_kernel<T, true><<<(unsigned)grid, 64 * p.sp.waves, 0, st>>>(p);
  rc = check_launch(what);
  if (rc || p.sp.nseg == 1) return rc;
  distill_join_kernel<T><<<(unsigned)cdiv(p.R, 4), 256, 0, st>>>(p);
  return check_launch("distill_fwd join");
}

extern "C" int ttts_distill_fwd(const void* logits, int32_t dtype, int64_t ldl, const int64_t* teacher_idx, const float* teacher_logp,
                                float* row_loss, float* stats, int32_t R, int32_t C, int32_t K, float temperature, int32_t tail,
                                void* workspace, int64_t workspace_bytes, void* stream) {
  int rc = check_logits("distill_fwd", logits, dtype, ldl, R, C, temperature);
  if (rc) return rc;
  TTTS_REQUIRE(K > 0 && K <= TTTS_DISTILL_MAX_K, "distill_fwd: need 0 < K <= %d", TTTS_DISTILL_MAX_K);
  if (R == 0) return TTTS_OK;
  TTTS_REQUIRE(teacher_idx && teacher_logp && row_loss && stats, "distill_fwd: null pointer");
  rc = need_workspace("distill_fwd", ttts_distill_workspace_bytes(R, C), workspace, workspace_bytes);
  if (rc) return rc;
  const DistillParams p{logits, ldl, teacher_idx, teacher_logp, row_loss, stats, (float4*)workspace, R, C, K, tail != 0, 1.0f / temperature, split_row(C)};
  TTTS_BY_TYPE(dtype, "distill_fwd", rc = launch_distill<T>(p, as_stream(stream)));
  return rc;
}

extern "C" int ttts_distill_bwd(const void* logits, int32_t dtype, int64_t ldl, const int64_t* teacher_idx, const float* teacher_logp,
                                const float* stats, const float* g_loss, void* dlogits, int64_t ldd, int32_t R, int32_t C, int32_t Cd,
                                int32_t K, float temperature, int32_t tail, int32_t accumulate, void* stream) {
  int rc = check_logits("distill_bwd", logits, dtype, ldl, R, C, temperature);
  if (rc) return rc;
  TTTS_REQUIRE(K > 0 && K <= TTTS_DISTILL_MAX_K, "distill_bwd: need 0 < K <= %d", TTTS_DISTILL_MAX_K);
  TTTS_REQUIRE(Cd >= C && ldd >= Cd, "distill_bwd: need C <= Cd <= ldd");
  if (R == 0) return TTTS_OK;
  TTTS_REQUIRE(teacher_idx && teacher_logp && stats && g_loss && dlogits, "distill_bwd: null pointer");
  DistillGradParams p{logits, ldl, teacher_idx, teacher_logp, stats, g_loss, dlogits, ldd, C, Cd, K, tail != 0, accumulate != 0, 0, 0, 0, 1.0f / temperature};
  p.per_row = (int)cdiv(Cd, WAVE_COLS);
  p.wave_cols = (int)cdiv(cdiv(Cd, 512), p.per_row) * 512;
  p.per_row = (int)cdiv(Cd, p.wave_cols);
  p.units = (int64_t)R * p.per_row;
  const int64_t grid = cdiv(p.units, 4);
  rc = need_grid("distill_bwd", grid);
  if (rc) return rc;
  TTTS_BY_TYPE(dtype, "distill_bwd", (distill_bwd_kernel<T><<<(unsigned)grid, 256, 0, as_stream(stream)>>>(p)));
  return check_launch("distill_bwd");
}
