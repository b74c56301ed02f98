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
// A row is read ONCE: maximum, sums, and the alternatives' threshold all come from the registers.  Rows up to 2048 columns take one wave;
// longer ones a wave per 2048 columns, each on its own (a workgroup per row whose waves meet at barriers read 2.1 - 2.5 TB/s where
// these read 5.4), and a second kernel that joins a row's parts.  A lane holds 8 neighbouring columns per load (16 or 32 bytes,
// at whatever alignment the row has; only the row's last columns are read one by one), 64 lanes 512 neighbouring ones: x[i][j] is
// column c0 + 512 i + 8 lane + j.  A rest of up to 64 columns behind the last whole 512 -- a codebook and its few special classes --
// is one more column a lane (`narrow`) instead of a step of eight.  NV: the steps of 512 that a kernel is compiled for; rows up to 1088
// columns have one of two (the instructions of two empty steps were a fifth of all).
constexpr int STEPS = 4, WAVE_COLS = STEPS * 512, NARROW = 64;
struct Cols {   // a wave's columns: c0 .. wide - 1 in `steps` of 512, wide .. end - 1 one a lane
  int c0, wide, end, steps;
  __device__ __forceinline__ Cols(int first, int last) : c0(first), wide(last), end(last), steps((last - first + 511) >> 9) {
    const int rest = (last - first) & 511;
    if (rest && rest <= NARROW) { --steps; wide -= rest; }
  }
  __device__ __forceinline__ bool narrow() const { return wide < end; }
  // its load, of some column of the row where the lane has none (no branch, so that nothing waits for it there), and its value
  template <typename T> __device__ __forceinline__ T load_narrow(const T* row, int last, int lane) const { return row[min(wide + lane, last)]; }
  template <typename T> __device__ __forceinline__ float narrow_value(T v, int cend, int lane) const {
    return wide + lane < min(end, cend) ? (float)v : -INFINITY;
  }
};
__device__ __forceinline__ float sum_wave(float v) { return over_wave(v, add_op); }
__device__ __forceinline__ float max_wave(float v) { return over_wave(v, max_op); }

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
// Columns c0 .. cend - 1 of a row, as they lie in memory (all loads on their way before the first is waited for); as fp32, columns outside
// are -inf.
template <typename T, int NV> struct Raw { typename Eight<T>::type v[NV]; };
template <typename T, int NV>
__device__ __forceinline__ void load_raw(Raw<T, NV>& r, const T* row, int c0, int cend, int lane) {
  if (c0 + NV * 512 <= cend) {   // (all of them: one address for the wave)
#pragma unroll
    for (int i = 0; i < NV; ++i) r.v[i] = *reinterpret_cast<const typename Eight<T>::type*>(row + c0 + (unsigned)(i * 512 + lane * 8));
    return;
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = c0 + i * 512 + lane * 8;
    if (c0 + i * 512 + 512 <= cend || c + 8 <= cend) r.v[i] = *reinterpret_cast<const typename Eight<T>::type*>(row + c);
  }
}
template <typename T, int NV>
__device__ __forceinline__ void expand(const Raw<T, NV>& r, const T* row, int c0, int cend, int lane, float (&x)[NV][8]) {
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = c0 + i * 512 + lane * 8;
    if (c0 + i * 512 + 512 <= cend) {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[i][j] = (float)r.v[i][j];
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[i][j] = c + 8 <= cend ? (float)r.v[i][j] : -INFINITY;
      if (c < cend && c + 8 > cend) load8<T>(row + c, cend - c, x[i]);
    }
  }
}

// The exponent of a class from its row's (or wave's) maximum m >= -FMAX:  t = (x - m) c, in bits.  As fma(x, c, -m c) it is one
// instruction and off by the one rounding of m c for the whole row, delta, which comes off the sums again; where m c is so large that
// delta would matter (or not finite: a row of the type's lowest value) the difference is taken first.
struct Exponent {
  float m, c, mc, delta;
  bool plain;   // uniform over the wave
  __device__ __forceinline__ Exponent(float m_, float c_) : m(m_), c(c_) {
    mc = m * c;
    plain = __builtin_amdgcn_readfirstlane(fabsf(mc) <= 1048576.f);
    delta = plain ? fmaf(m, c, -mc) : 0.f;
  }
};
// (n / d, n % d) of the number of a launch's wave or thread, which fits 32 bits
__device__ __forceinline__ void split_id(int64_t n, int d, int64_t& q, int& r) {
  const uint32_t whole = (uint32_t)n / (uint32_t)d;
  q = whole;
  r = (int)((uint32_t)n - whole * (uint32_t)d);
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

// bits of ord() that values of the type leave alike (below a 16-bit type's mantissa): nothing to search there
template <typename T> struct LowBits { static constexpr int n = 0; };
template <> struct LowBits<bf16> { static constexpr int n = 16; };
template <> struct LowBits<_Float16> { static constexpr int n = 13; };

// A threshold first: the k-th largest of the maxima of groups of columns is at most the k-th largest column, and few columns reach it
// (k + 10 .. 30 % of ordinary rows).  It is found bit by bit with ballots over n group maxima a lane, and any value that exactly k
// groups reach will do (early).  What reaches it lies in at most k groups, unless values repeat at the threshold: then (exact) fewer
// than k groups go above it, and of the columns AT it the lowest classes are taken, as many as are needed.
template <typename T>
__device__ __forceinline__ float threshold_of(uint32_t t) {   // (a class at -inf is no alternative)
  if (LowBits<T>::n && !(t >> 31)) t |= (1u << LowBits<T>::n) - 1;   // below zero ord() has ones there
  return t <= ORD_NONE ? -FMAX : unord(t);
}
template <typename T, int N>
__device__ __forceinline__ float group_threshold(const uint32_t (&g)[N], int k, bool early, uint32_t lo = 0, uint32_t hi = 0xffffffffu) {
  if (lo == hi) return threshold_of<T>(lo);
  uint32_t bit = 0x80000000u >> __builtin_clz(lo ^ hi), t = lo & ~(bit + bit - 1);   // lo <= it <= hi: it begins as both do
  for (; bit >> LowBits<T>::n; bit >>= 1) {
    const uint32_t c = t | bit;
    int cnt = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) cnt += __builtin_popcountll(__ballot(g[i] >= c));
    if (cnt >= k) {
      t = c;
      if (early && cnt == k) break;
    }
  }
  return threshold_of<T>(t);
}
// bounds of the k-th largest (k <= 64) of a wave's groups, from the largest of each lane's
__device__ __forceinline__ void lane_bounds(float most, uint32_t& lo, uint32_t& hi) {
  lo = __builtin_amdgcn_readfirstlane(ord(-max_wave(-most)));
  hi = __builtin_amdgcn_readfirstlane(ord(max_wave(most)));
}
// bit 31 - (8 i + j): x[i][j] reaches the threshold / is above it
template <bool ABOVE, int NV>
__device__ __forceinline__ uint32_t reached(const float (&x)[NV][8], float thr, int steps) {
  uint32_t bits = 0;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (i < steps) {
#pragma unroll
      for (int j = 0; j < 8; ++j) bits = bits + bits + (ABOVE ? x[i][j] > thr : x[i][j] >= thr);
    } else {
      bits <<= 8;
    }
  }
  return bits << (32 - 8 * NV);
}
// A wave's own keys of a 16-bit type fit 32 bits: the ord() that the type has, and the column among the wave's, inverted.
template <typename T> struct WaveKey {
  typedef u64 type;
  static __device__ __forceinline__ type make(float v, int at, int c0) { return top_key(v, c0 + at); }
  static __device__ __forceinline__ u64 full(type k, int) { return k; }
};
template <typename T> struct WaveKey16 {
  typedef uint32_t type;
  static __device__ __forceinline__ type make(float v, int at, int) { return (ord(v) >> LowBits<T>::n << 12) | (uint32_t)(4095 - at); }
  static __device__ __forceinline__ u64 full(type k, int c0) {
    uint32_t o = k >> 12 << LowBits<T>::n;
    if (!(o >> 31)) o |= (1u << LowBits<T>::n) - 1;   // below zero ord() has ones there
    return ((u64)o << 32) | (uint32_t)~(c0 + 4095 - (int)(k & 4095));
  }
};
template <> struct WaveKey<bf16> : WaveKey16<bf16> {};
template <> struct WaveKey<_Float16> : WaveKey16<_Float16> {};
static_assert(WAVE_COLS + NARROW <= 4096, "12 bits of a wave's key are a column");

// The marked columns (bits, narrow) are listed, n of them with what was there, those before `cap` stored: the loop goes by the most marks that a
// lane has, so it does no more than that (reading each column again in it cost a wait a round: 200000 rows of 1026 classes, 20 alternatives: 151 us, 139 now).
template <typename K>
__device__ __forceinline__ int list_marked(uint32_t bits, bool narrow, const Cols& cols, int lane, K* cand, int cap) {
  int n = 0;
  if (const u64 mask = __ballot(narrow)) {
    const int at = lanes_below(mask);
    if (narrow && at < cap) cand[at] = (K)(cols.wide - cols.c0 + lane);
    n = __builtin_popcountll(mask);
  }
  for (u64 mask = __ballot(bits != 0); mask; mask = __ballot(bits != 0)) {
    const int at = n + lanes_below(mask);
    n += __builtin_popcountll(mask);
    if (bits) {
      const int e = __builtin_clz(bits);
      bits &= ~(0x80000000u >> e);
      if (at < cap) cand[at] = (K)((e >> 3) * 512 + lane * 8 + (e & 7));
    }
  }
  return n;
}
// columns equal to thr, lowest classes first, become keys from place n on, up to `end`; returns n + ties
template <typename T, int NV>
__device__ __forceinline__ int collect_ties(const float (&x)[NV][8], float xn, float thr, const Cols& cols, int lane,
                                            typename WaveKey<T>::type* cand, int n, int end) {
  const int c0 = cols.c0;
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
        if (at < end) cand[at] = WaveKey<T>::make(x[i][j], i * 512 + lane * 8 + j, c0);
        ++at;
      }
    n += __shfl(upto, 63, 64);
  }
  const u64 mask = __ballot(xn == thr);
  const int at = n + lanes_below(mask);
  if (xn == thr && at < end) cand[at] = WaveKey<T>::make(xn, cols.wide - c0 + lane, c0);
  return n + __builtin_popcountll(mask);
}
// f(rank, key) for the keys of rank < k among n distinct ones (four places behind them writable): ranked by counting
template <typename K, typename F>
__device__ __forceinline__ void rank_keys(const K* cand, int n, int k, int thread, int threads, F f) {
  for (int s = thread; s < n; s += threads) {
    const K key = cand[s];
    int r = 0;
    for (int j = 0; j < n; j += 4) r += (cand[j] > key) + (cand[j + 1] > key) + (cand[j + 2] > key) + (cand[j + 3] > key);
    if (r < k) f(r, key);
  }
}
constexpr int WAVE_CAND = 64 * 9, WAVE_TOP_LDS = WAVE_CAND + 4;           // one wave: groups of 8 or 9 columns (exact)
constexpr int GROUP_CAND = 64 * 33;                                       // a workgroup: a lane's 32 or 33 columns are a group
// one wave: f(rank, key) of its k best; returns how many there are (<= k)
template <typename T, int NV, typename F>
__device__ __forceinline__ int wave_top(const float (&x)[NV][8], float xn, const float (&vmax)[NV], const T* row, const Cols& cols, int k, int lane,
                                        typename WaveKey<T>::type* cand, F f) {
  uint32_t g[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) g[i] = ord(vmax[i]);
  float thr;
  if (k <= 32) {          // groups of a lane's 32 columns: one ballot a bit
    uint32_t one[1] = {g[0]};
#pragma unroll
    for (int i = 1; i < NV; ++i) one[0] = max(one[0], g[i]);
    thr = group_threshold<T, 1>(one, k, true);
  } else {                // of 8 columns: with 64 groups the least of them would have to do
    thr = group_threshold<T, NV>(g, k, true);
  }
  int n = list_marked(reached<false, NV>(x, thr, cols.steps), xn >= thr, cols, lane, cand, WAVE_CAND);
  const bool exact = n > WAVE_CAND;
  if (exact) {
    thr = group_threshold<T, NV>(g, k, false);
    n = list_marked(reached<true, NV>(x, thr, cols.steps), xn > thr, cols, lane, cand, WAVE_CAND);
  }
  wave_fence();
  for (int s = lane; s < n; s += 64) {      // (a register cannot be indexed by a lane: their values are read again)
    const int at = (int)cand[s];
    cand[s] = WaveKey<T>::make((float)row[cols.c0 + at], at, cols.c0);
  }
  if (exact) {
    const int end = max(n, k);
    n = min(end, collect_ties<T, NV>(x, xn, thr, cols, lane, cand, n, end));
  }
  if (lane < 4) cand[n + lane] = 0;
  wave_fence();
  rank_keys(cand, n, k, lane, 64, [&](int r, typename WaveKey<T>::type key) { f(r, WaveKey<T>::full(key, cols.c0)); });
  return min(n, k);
}

// Maximum, excess = sum e - 1, sum e t (t in bits, from the maximum).  The 1 is the maximum's own, which is never added: the log-probability of a
// class that is nearly certain, -log(1 + excess), and the row's entropy keep the bits that beside a 1 would be lost (an excess of 0.006 was off by
// 2e-5 of itself; leaving the 1 out takes 46 of the 507 vector instructions a wave of two steps: 12816 rows of 1026 classes, 20
// alternatives: 13.2 -> 14.2 us).  Without a class above -inf the excess is -1.
struct RowSums {
  float m, excess, s;
  __device__ __forceinline__ float z() const { return 1.f + excess; }
  __device__ __forceinline__ bool none() const { return excess < 0.f; }
  __device__ __forceinline__ float log_z() const {   // log(1 + excess): by its series up to 1 / 16 (the rest 2^-27 of it)
    const float x = excess;
    const float series = x * fmaf(x, fmaf(x, fmaf(x, fmaf(x, fmaf(x, -1.f / 6, 1.f / 5), -1.f / 4), 1.f / 3), -1.f / 2), 1.f);
    return x < 0.0625f ? series : __builtin_amdgcn_logf(z()) * LN2;
  }
};
// of one wave's columns.  A class at -inf, or at the type's lowest value, has e = 0: e t must be 0, not NaN, so t is kept finite
// there (a NaN passes through e).  vmax: the lanes' maxima of their 8 columns a step (vmax[0] may know the narrow one too).
template <int NV>
__device__ __forceinline__ RowSums wave_sums(const float (&x)[NV][8], float xn, const float (&vmax)[NV], const Cols& cols, float lmax, float c) {
  const int steps = cols.steps;
  RowSums a;
  a.m = max_wave(fmaxf(lmax, -FMAX));
  a.excess = a.s = 0.f;
  const Exponent ex(a.m, c);
  int most = 0;           // classes at the maximum: counted, not added (as 64 less those of a column that are not)
  auto add = [&](float t) {
    const float e = __builtin_amdgcn_exp2f(t);
    a.excess += e;
    a.s = fmaf(e, fmaxf(t, -200.f), a.s);
  };
  auto leave_out = [&](float& t, float v) {
    const bool below = v != a.m;
    most += 64 - __builtin_popcountll(__ballot(below));
    t = below ? t : -INFINITY;
  };
  auto add_up = [&](auto exponent) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (i >= steps) break;
      float t[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) t[j] = exponent(x[i][j]);
      if (__any(vmax[i] == a.m)) {        // (one step of the row's, as a rule)
#pragma unroll
        for (int j = 0; j < 8; ++j) leave_out(t[j], x[i][j]);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) add(t[j]);
    }
    if (cols.narrow()) {
      float t = exponent(xn);
      leave_out(t, xn);
      add(t);
    }
  };
  if (ex.plain) add_up([&](float v) { return fmaf(v, c, -ex.mc); });
  else add_up([&](float v) { return (v - a.m) * c; });
  const float f = __builtin_amdgcn_exp2f(-ex.delta), below = sum_wave(a.excess) * f;
  a.s = sum_wave(a.s) * f - ex.delta * below;
  a.excess = below + (float)(most - 1) + (a.m - a.m);   // (NaN of an infinite maximum)
  return a;
}

// Groups of a long row's unit, 64 of 32 neighbouring columns each: from the maxima of a lane's 8 columns a step (and its narrow column) lane
// l gets that of step l & 3 of the four lanes around it, columns 512 (l & 3) + 32 (l / 4) ..+31 of the unit (and narrow column l).
// (A lane's own 4 x 8 columns as a group lay in four places when they were read again.)
__device__ __forceinline__ float group_max(const float (&v)[STEPS], float xn, int lane) {
  static_assert(STEPS == 4, "four lanes, four steps");
  const bool odd = lane & 1, high = lane & 2;
  const float a = max_op(odd ? v[1] : v[0], dpp_mov<0xb1>(odd ? v[0] : v[1]));   // quad_perm 1, 0, 3, 2
  const float b = max_op(odd ? v[3] : v[2], dpp_mov<0xb1>(odd ? v[2] : v[3]));
  const float m = max_op(high ? b : a, dpp_mov<0x4e>(high ? a : b));             // quad_perm 2, 3, 0, 1
  return max_op(max_op(m, xn), -INFINITY);
}
struct ScoreParams {
  const void* logits; int64_t ldl;
  const int64_t* tokens;
  float *logp, *entropy, *stats, *top_logp;
  int64_t* top_idx;
  float4* part;          // long rows: [R, units] RowSums of each wave's columns,
  void* part_max;        // and with alternatives [R, units, 64] of the logits' type: the maximum of each group of columns (group_max)
  int R, C, k, units, unit_cols, narrow_at;   // the row's columns from narrow_at on are its last unit's narrow ones
  float inv_t;
};

__device__ __forceinline__ void write_row(const ScoreParams& p, int64_t row, const RowSums& a, float logz, bool given, float xt) {
  const bool none = a.none();   // every class at -inf
  p.stats[2 * row] = none ? -INFINITY : a.m;
  p.stats[2 * row + 1] = none ? -INFINITY : logz;
  p.entropy[row] = none ? 0.f : logz - a.s / a.z() * LN2;
  p.logp[row] = !given ? 0.f : none ? -INFINITY : (xt - a.m) * p.inv_t - logz;
}
__device__ __forceinline__ void write_top(const ScoreParams& p, int64_t row, int r, u64 key, const RowSums& a, float logz) {
  const bool nan = a.excess != a.excess, have = key != 0 && !nan;
  p.top_idx[row * p.k + r] = have ? key_class(key) : -1;
  p.top_logp[row * p.k + r] = have ? (unord((uint32_t)(key >> 32)) - a.m) * p.inv_t - logz : nan ? a.excess : -INFINITY;
}

// A long row's sums, by one wave, from its units' parts; every lane gets them.  What it takes from memory is asked for first, and by every
// lane, so that its way is short when it is needed.
struct LongRow { float4 first; int tok; float xt; };   // tok: -1 if none is given
template <typename T>
__device__ __forceinline__ LongRow load_long_row(const ScoreParams& p, int64_t row, int lane) {
  LongRow r;
  const int64_t tok = p.tokens[row];
  r.first = p.part[row * p.units + min(lane, p.units - 1)];
  r.tok = tok >= 0 && tok < p.C ? (int)tok : -1;
  r.xt = (float)((const T*)p.logits)[row * p.ldl + max(r.tok, 0)];
  return r;
}
__device__ __forceinline__ RowSums join_sums(const ScoreParams& p, const float4* part, const LongRow& r, int lane) {
  const float c = p.inv_t * LOG2E;
  float m = r.first.x;
  for (int u = lane + 64; u < p.units; u += 64) m = fmaxf(m, part[u].x);
  RowSums a = {max_wave(m), 0.f, 0.f};
  float most = 0.f;       // parts at the maximum: their 1 is counted, not added
  auto add = [&](const float4& u) {
    const bool top = u.x == a.m;
    const float d = fmaxf((u.x - a.m) * c, -200.f), f = __builtin_amdgcn_exp2f(d), z = 1.f + u.y;
    most += top ? 1.f : 0.f;
    a.excess += top ? u.y : z * f;
    a.s += top ? u.z : f * (u.z + z * d);
  };
  if (lane < p.units) add(r.first);
  for (int u = lane + 64; u < p.units; u += 64) add(part[u]);
  a.excess = sum_wave(a.excess) + (sum_wave(most) - 1.f);
  a.s = sum_wave(a.s);
  return a;
}
// Alternatives of a row of up to UNITS units by one wave: v are the maxima of all its groups, so the threshold is exact at once.  Where the
// candidates do not fit (values that repeat, or a row whose largest ones crowd into few groups): the k-th largest column itself,
// searched by counting over the row, the fewer than k columns above it, and the lowest classes at it.
constexpr int ROW_CAND = 320, ROW_LIST = 128;
template <typename T, int UNITS>
__device__ __forceinline__ void row_top(const ScoreParams& p, int64_t row, const T* lr, const float (&v)[UNITS], const RowSums& a, u64* cand, int* list,
                                        int lane) {
  const int k = p.k;
  uint32_t g[UNITS], lo, hi;
  float most = -INFINITY;
#pragma unroll
  for (int i = 0; i < UNITS; ++i) {
    g[i] = ord(v[i]);
    most = max_op(most, v[i]);
  }
  lane_bounds(most, lo, hi);
  float thr = group_threshold<T, UNITS>(g, k, true, lo, hi);
  int n = 0, listed = 0;
  {
    const uint32_t tb = ord(thr);
#pragma unroll
    for (int i = 0; i < UNITS; ++i) {
      const u64 mask = __ballot(g[i] >= tb);
      if (mask) {
        const int at = listed + lanes_below(mask);
        if (g[i] >= tb && at < ROW_LIST) list[at] = i * 64 + lane;
        listed += __builtin_popcountll(mask);
      }
    }
  }
  wave_fence();
  // v: the lane's 8 columns from c on; test(v) of them become keys
  auto push = [&](const float (&v)[8], int c, auto test) {
    uint32_t bits = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) bits |= test(v[j]) ? 1u << j : 0u;
    for (u64 mask = __ballot(bits != 0); mask; mask = __ballot(bits != 0)) {
      const int at = n + lanes_below(mask);
      n += __builtin_popcountll(mask);
      if (bits) {
        const int e = __builtin_ctz(bits);
        bits &= bits - 1;
        float x = v[0];
#pragma unroll
        for (int j = 1; j < 8; ++j) x = e == j ? v[j] : x;
        if (at < ROW_CAND) cand[at] = top_key(x, c + e);
      }
    }
  };
  auto eight = [&](int c, int end, float (&v)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = -INFINITY;
    if (c < end) load8<T>(lr + c, end - c, v);
  };
  bool full = listed > ROW_LIST;
  if (!full) {
    for (int s = 0; s < listed * (STEPS + 1); s += 64) {
      const int task = s + lane, i = task % (STEPS + 1), id = task < listed * (STEPS + 1) ? list[task / (STEPS + 1)] : 0;
      int c = (id >> 6) * p.unit_cols + (id & 3) * 512 + (id & 60) * 8 + i * 8, end = (id & 3) * 512 < p.unit_cols ? p.narrow_at : 0;
      if (i == STEPS) {                              // the unit's narrow columns
        c = p.narrow_at + (id & 63);
        end = (id >> 6) == p.units - 1 ? min(p.C, c + 1) : 0;
      }
      float v[8];
      eight(c, task < listed * (STEPS + 1) ? end : 0, v);
      push(v, c, [&](float x) { return x >= thr; });
    }
    full = n > ROW_CAND;
  }
  if (full) {
    float v[8];
    uint32_t t = 0;
    for (uint32_t bit = 0x80000000u; bit >> LowBits<T>::n; bit >>= 1) {
      float cnt = 0.f;                        // (whole numbers up to 32832)
      for (int c0 = 0; c0 < p.C; c0 += 512) {
        eight(c0 + lane * 8, p.C, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) cnt += ord(v[j]) >= (t | bit) && v[j] == v[j] ? 1.f : 0.f;
      }
      if (sum_wave(cnt) >= (float)k) t |= bit;
    }
    thr = threshold_of<T>(t);
    n = 0;
    for (int c0 = 0; c0 < p.C; c0 += 512) {
      eight(c0 + lane * 8, p.C, v);
      push(v, c0 + lane * 8, [&](float x) { return x > thr; });
    }
    for (int c0 = 0; c0 < p.C && n < k; c0 += 512) {
      eight(c0 + lane * 8, p.C, v);
      int mine = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) mine += v[j] == thr;
      int upto = mine;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int u = __shfl_up(upto, o, 64);
        if (lane >= o) upto += u;
      }
      int at = n + upto - mine;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (v[j] == thr) {
          if (at < k) cand[at] = top_key(v[j], c0 + lane * 8 + j);
          ++at;
        }
      n = min(k, n + __shfl(upto, 63, 64));
    }
    n = min(n, k);
  }
  if (lane < 4) cand[n + lane] = 0;
  wave_fence();
  const float logz = a.log_z();
  rank_keys(cand, n, k, lane, 64, [&](int r, u64 key) { write_top(p, row, r, key, a, logz); });
  if (lane >= n && lane < k) write_top(p, row, lane, 0, a, logz);
}

// One wave per row (ONE), or per unit of up to 2048 columns of a row: with a workgroup for a row (ROW), whose waves meet once and the first ends
// the row, or on their own (PART), with a second kernel that does.  A workgroup a row saves the parts' way through memory and a launch:
// 25000 fp32 rows of 4096 classes, 20 alternatives: 78 us, 105 in two kernels; 3125 of 32768: 80, 89.  Of 16-bit types, half the bytes for
// the same arithmetic, only up to four waves: 25000 rows of 8194: 87, 107; but 10240 of 20000: 112, 96 (ten waves start where
// ten have ended).  (Waves that went through several units, the next one's loads under this one's arithmetic, were slower at every grid:
// 118 - 125 us instead of 109 for logits of 2048 x 100003 with 64 alternatives.)
enum Kind { ONE, ROW, PART };
template <typename T> struct RowUnits { static constexpr int n = sizeof(T) == 4 ? 16 : 4; };
template <typename T, Kind KIND, int NV, int UNITS = 1>
__global__ __launch_bounds__(KIND == ROW ? UNITS * 64 : 256, 8) void token_logprobs_fwd_kernel(ScoreParams p) {
  extern __shared__ __attribute__((aligned(16))) unsigned char score_lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t id = (int64_t)blockIdx.x * 4 + wave;
  int64_t row = KIND == ROW ? blockIdx.x : id;
  int unit = KIND == ROW ? wave : 0;
  if (KIND == PART) split_id(id, p.units, row, unit);
  if (row >= p.R) return;
  const T* lr = (const T*)p.logits + row * p.ldl;
  const Cols cols(unit * p.unit_cols, unit == p.units - 1 ? p.C : (unit + 1) * p.unit_cols);
  float x[NV][8], vmax[NV];
  int64_t tok = -1;
  float xt = 0.f, xn;
  {
    Raw<T, NV> raw;
    if (KIND != PART && unit == 0) tok = p.tokens[row];
    load_raw(raw, lr, cols.c0, cols.wide, lane);
    const T narrow = cols.load_narrow(lr, p.C - 1, lane);
    const bool given = tok >= 0 && tok < p.C;
    const T at_tok = KIND == PART ? T(0.f) : lr[given ? tok : 0];   // (its latency runs beside the row's)
    expand(raw, lr, cols.c0, cols.wide, lane, x);
    xn = cols.narrow_value(narrow, p.C, lane);
    xt = given ? (float)at_tok : 0.f;
  }
  float lmax = xn;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    vmax[i] = -INFINITY;
#pragma unroll
    for (int j = 0; j < 8; ++j) vmax[i] = max_op(vmax[i], x[i][j]);
    lmax = max_op(lmax, vmax[i]);
  }
  if (KIND == ONE) vmax[0] = max_op(vmax[0], xn);
  lmax = max_op(lmax, -INFINITY);                         // (xn may be NaN)
  const RowSums a = wave_sums(x, xn, vmax, cols, lmax, p.inv_t * LOG2E);
  if constexpr (KIND == PART) {
    if (lane == 0) p.part[id] = make_float4(a.m, a.excess, a.s, 0.f);
    if (p.k) ((T*)p.part_max)[id * 64 + lane] = (T)group_max(vmax, xn, lane);
  } else if constexpr (KIND == ROW) {
    __shared__ float4 sm_part[UNITS];
    __shared__ float sm_max[UNITS][64];
    __shared__ __attribute__((aligned(16))) u64 sm_cand[ROW_CAND + 4];
    __shared__ int sm_list[ROW_LIST];
    if (lane == 0) sm_part[unit] = make_float4(a.m, a.excess, a.s, 0.f);
    if (p.k) sm_max[unit][lane] = group_max(vmax, xn, lane);
    __syncthreads();
    if (unit) return;
    const LongRow r = {sm_part[min(lane, p.units - 1)], tok >= 0 && tok < p.C ? (int)tok : -1, xt};
    const RowSums all = join_sums(p, sm_part, r, lane);
    if (lane == 0) write_row(p, row, all, all.log_z(), r.tok >= 0, r.xt);
    if (p.k) {
      float v[UNITS];
#pragma unroll
      for (int i = 0; i < UNITS; ++i) v[i] = i < p.units ? sm_max[i][lane] : -INFINITY;
      row_top<T, UNITS>(p, row, lr, v, all, sm_cand, sm_list, lane);
    }
  } else {
    const float logz = a.log_z();
    if (lane == 0) write_row(p, row, a, logz, tok >= 0 && tok < p.C, xt);
    if (p.k) {
      const int have = wave_top<T, NV>(x, xn, vmax, lr, cols, p.k, lane, reinterpret_cast<typename WaveKey<T>::type*>(score_lds) + wave * WAVE_TOP_LDS, [&](int r, u64 key) { write_top(p, row, r, key, a, logz); });
      if (lane >= have && lane < p.k) write_top(p, row, lane, 0, a, logz);
    }
  }
}

template <typename T>
__global__ __launch_bounds__(256) void token_logprobs_join_kernel(ScoreParams p) {   // no alternatives: a wave per row
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= p.R) return;
  const int lane = threadIdx.x & 63;
  const LongRow r = load_long_row<T>(p, row, lane);
  const RowSums a = join_sums(p, p.part + row * p.units, r, lane);
  if (lane == 0) write_row(p, row, a, a.log_z(), r.tok >= 0, r.xt);
}

// Alternatives of a long row: W waves, up to W * N * 64 groups of 32 columns.  A bound that k groups reach: the least of the waves' own
// (k / W)-th largest of the maxima of 2 or 4 sets of their groups a lane; a third more than k groups reach it where the row's largest
// are spread over the waves' units (a wave has every W-th).  Where they are not, and more reach it than are listed: the largest of the waves' own
// k-th largest.  The columns of the listed groups are read again, and those that reach the bound ranked.
// Where values repeat at the bound, so that more reach it than there is room for: the exact threshold over all groups, the
// fewer than k groups above it, and then the row's columns AT it in the order of the classes until there are k.
template <typename T, int W, int N>
__global__ __launch_bounds__(W * 64, 8) void token_logprobs_top_kernel(ScoreParams p) {
  constexpr int LIST = 96 * W, SETS = N > 16 ? 2 : 4;   // (with 32 groups a lane four sets would not fit 64 registers)
  __shared__ __attribute__((aligned(16))) u64 cand[GROUP_CAND + 4];
  __shared__ int list_id[LIST];
  __shared__ float sm_thr[W];
  __shared__ RowSums sm_row;
  __shared__ int sm_n, sm_list[2], sm_cnt[W];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t row = blockIdx.x;
  const T* lr = (const T*)p.logits + row * p.ldl;
  const int k = p.k, groups = p.units * 64;
  const T* gm = (const T*)p.part_max + row * groups;
  if (tid == 0) sm_n = sm_list[0] = sm_list[1] = 0;
  float bound;
  int listed;
  LongRow r;
  if (wave == W - 1) r = load_long_row<T>(p, row, lane);
  {
    float v[N];                               // wave w has the units w, w + W, ..; group id = unit * 64 + lane
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (float)(gm + min(i * W + wave, p.units - 1) * 64)[lane];
    uint32_t q[SETS], lo, hi;
    float most = -INFINITY;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = i * W + wave < p.units ? v[i] : -INFINITY;
#pragma unroll
    for (int i = 0; i < SETS; ++i) {
      float set = v[i];
#pragma unroll
      for (int j = i + SETS; j < N; j += SETS) set = max_op(set, v[j]);
      most = max_op(most, set);
      q[i] = ord(set);
    }
    lane_bounds(most, lo, hi);
    for (int round = 0; round < 2; ++round) {
      const float mine = group_threshold<T, SETS>(q, round ? k : (k + W - 1) / W, true, lo, hi);
      if (lane == 0) sm_thr[wave] = mine;
      __syncthreads();
      bound = sm_thr[0];
      for (int w = 1; w < W; ++w) bound = round ? fmaxf(bound, sm_thr[w]) : fminf(bound, sm_thr[w]);
      int at = 0;
#pragma unroll
      for (int i = 0; i < N; ++i) at += v[i] >= bound;
      if (at) at = atomicAdd(&sm_list[round], at);
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (v[i] >= bound) {
          if (at < LIST) list_id[at] = (i * W + wave) * 64 + lane;
          ++at;
        }
      if (wave == W - 1 && round == 0) {
        const RowSums a = join_sums(p, p.part + row * p.units, r, lane);
        if (lane == 0) sm_row = a;
      }
      __syncthreads();
      listed = sm_list[round];
      if (listed <= LIST) break;              // (uniform over the workgroup)
    }
  }
  auto push = [&](const float (&v)[8], int c, float t, bool above) {   // columns that reach t (or lie above it) become keys
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (above ? v[j] > t : v[j] >= t) {
        const int at = atomicAdd(&sm_n, 1);
        if (at < GROUP_CAND) cand[at] = top_key(v[j], c + j);
      }
  };
  // where piece i of a group lies: `end - c` columns, none if that is not positive; its narrow column goes with piece 0
  auto piece = [&](int id, int i, int& c, int& end, int& cn) {
    c = (id >> 6) * p.unit_cols + (id & 3) * 512 + (id & 60) * 8 + i * 8;
    end = (id & 3) * 512 < p.unit_cols ? p.narrow_at : 0;
    cn = i == 0 && (id >> 6) == p.units - 1 ? p.narrow_at + (id & 63) : p.C;
  };
  auto push_narrow = [&](T x, int cn, float t, bool above) {
    const float v = (float)x;
    if (cn < p.C && (above ? v > t : v >= t)) {
      const int at = atomicAdd(&sm_n, 1);
      if (at < GROUP_CAND) cand[at] = top_key(v, cn);
    }
  };
  bool full = listed > LIST;
  if (!full) {
    const int tasks = listed * STEPS;
    for (int s = tid; s < tasks; s += 2 * W * 64) {   // two pieces a thread, their loads together
      typename Eight<T>::type r[2];
      T rn[2];
      int c[2], end[2], cn[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int task = s + h * W * 64;
        piece(list_id[min(task, tasks - 1) / STEPS], task % STEPS, c[h], end[h], cn[h]);
        if (task >= tasks) { end[h] = 0; cn[h] = p.C; }
        if (c[h] + 8 <= end[h]) r[h] = *reinterpret_cast<const typename Eight<T>::type*>(lr + c[h]);
        rn[h] = lr[min(cn[h], p.C - 1)];
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (c[h] < end[h]) {
          float v[8];
          if (c[h] + 8 <= end[h]) {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = (float)r[h][j];
          } else {
            load8<T>(lr + c[h], end[h] - c[h], v);
          }
          push(v, c[h], bound, false);
        }
        push_narrow(rn[h], cn[h], bound, false);
      }
    }
    __syncthreads();
    full = sm_n > GROUP_CAND;
  }
  if (full) {
    uint32_t t = 0;                           // the exact threshold over all groups of the row
    for (uint32_t bit = 0x80000000u; bit >> LowBits<T>::n; bit >>= 1) {
      int cnt = 0;
      for (int u = wave; u < p.units; u += W) cnt += __builtin_popcountll(__ballot(ord((float)gm[u * 64 + lane]) >= (t | bit)));
      __syncthreads();
      if (lane == 0) sm_cnt[wave] = cnt;
      __syncthreads();
      cnt = 0;
      for (int w = 0; w < W; ++w) cnt += sm_cnt[w];
      if (cnt >= k) t |= bit;
    }
    const float thr = threshold_of<T>(t);
    const uint32_t tb = ord(thr);
    __syncthreads();
    if (tid == 0) sm_n = 0;
    __syncthreads();
    for (int u = wave; u < p.units; u += W)
      if (ord((float)gm[u * 64 + lane]) > tb)
#pragma unroll 1
        for (int e = 0; e < STEPS; ++e) {
          int c, end, cn;
          piece(u * 64 + lane, e, c, end, cn);
          if (c < end) {
            float v[8];
            load8<T>(lr + c, end - c, v);
            push(v, c, thr, true);
          }
          if (cn < p.C) push_narrow(lr[cn], cn, thr, true);
        }
    __syncthreads();
    int n = sm_n;
    const int end = max(n, k);
    for (int c0 = 0; c0 < p.C && n < end; c0 += W * 512) {
      const int c = c0 + tid * 8;
      float v[8];
      int mine = 0;
      if (c < p.C) {
        load8<T>(lr + c, p.C - c, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) mine += v[j] == thr;
      }
      int upto = mine;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int s = __shfl_up(upto, o, 64);
        if (lane >= o) upto += s;
      }
      __syncthreads();
      if (lane == 63) sm_cnt[wave] = upto;
      __syncthreads();
      int at = n + upto - mine;
      for (int w = 0; w < W; ++w) {
        if (w < wave) at += sm_cnt[w];
        n += sm_cnt[w];
      }
      if (mine)
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (v[j] == thr) {
            if (at < end) cand[at] = top_key(v[j], c + j);
            ++at;
          }
    }
    __syncthreads();
    if (tid == 0) sm_n = min(n, end);
    __syncthreads();
  }
  const int n = sm_n;
  const RowSums a = sm_row;
  if (tid < 4) cand[n + tid] = 0;
  __syncthreads();
  const float logz = a.log_z();
  rank_keys(cand, n, k, tid, W * 64, [&](int r, u64 key) { write_top(p, row, r, key, a, logz); });
  for (int e = n + tid; e < k; e += W * 64) write_top(p, row, e, 0, a, logz);
  if (wave == W - 1 && lane == 0) write_row(p, row, a, a.log_z(), r.tok >= 0, r.xt);
}

// A wave per row of up to UNITS units, four rows a workgroup and no barrier (6250 rows of 32768 classes, 20 alternatives: 92 us, 104 with a
// workgroup each; 8 units with the registers of 16 cost a tenth more).
template <typename T, int UNITS>
__global__ __launch_bounds__(256) void token_logprobs_top_wave_kernel(ScoreParams p) {
  __shared__ __attribute__((aligned(16))) u64 sm_cand[4][ROW_CAND + 4];
  __shared__ int sm_list[4][ROW_LIST];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t row = (int64_t)blockIdx.x * 4 + wave;
  if (row >= p.R) return;
  const T* gm = (const T*)p.part_max + row * p.units * 64;
  T raw[UNITS];
#pragma unroll
  for (int i = 0; i < UNITS; ++i) raw[i] = gm[min(i, p.units - 1) * 64 + lane];
  const LongRow r = load_long_row<T>(p, row, lane);
  float v[UNITS];
#pragma unroll
  for (int i = 0; i < UNITS; ++i) v[i] = i < p.units ? (float)raw[i] : -INFINITY;
  const RowSums a = join_sums(p, p.part + row * p.units, r, lane);
  if (lane == 0) write_row(p, row, a, a.log_z(), r.tok >= 0, r.xt);
  row_top<T, UNITS>(p, row, (const T*)p.logits + row * p.ldl, v, a, sm_cand[wave], sm_list[wave], lane);
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
// A row's list, two entries a lane (one, and no work for the other, up to 64 entries): class (or -1), p and log p, and the list's mass.
// Its loads go first and without branches: everything behind them in the wave then has one wait for them, not one each.
struct ListLoads { int64_t id[2]; float t[2]; };
__device__ __forceinline__ ListLoads load_list(const int64_t* idx, const float* tl, int K, int lane) {
  ListLoads r;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    r.id[h] = -1;
    r.t[h] = 0.f;
    if (h * 64 < K) {
      const int j = min(lane + 64 * h, K - 1);
      r.id[h] = idx[j];
      r.t[h] = tl[j];
    }
  }
  return r;
}
struct Listed { int id[2]; float p[2], logp[2], mass; };
__device__ __forceinline__ void list_classes(Listed& L, const ListLoads& r, int K, int C, int lane) {
#pragma unroll
  for (int h = 0; h < 2; ++h) L.id[h] = lane + 64 * h < K && r.id[h] >= 0 && r.id[h] < C ? (int)r.id[h] : -1;
}
__device__ __forceinline__ void list_weights(Listed& L, const ListLoads& r, int K, float inv_t, int tail) {
  float t[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    t[h] = L.id[h] >= 0 ? r.t[h] : -INFINITY;
    L.p[h] = 0.f;
    L.logp[h] = -INFINITY;
  }
  if (tail) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (h * 64 < K) {
        L.logp[h] = t[h];
        L.p[h] = L.id[h] >= 0 ? __expf(t[h]) : 0.f;
      }
    L.mass = sum_wave(L.p[0] + L.p[1]);
    return;
  }
  const float m = fmaxf(max_wave(K > 64 ? fmaxf(t[0], t[1]) : t[0]), -FMAX);
#pragma unroll
  for (int h = 0; h < 2; ++h)
    if (h * 64 < K) {
      L.logp[h] = (t[h] - m) * inv_t;
      L.p[h] = L.id[h] >= 0 ? __expf(L.logp[h]) : 0.f;
    }
  const float z = sum_wave(L.p[0] + L.p[1]), over = __builtin_amdgcn_rcpf(z), logz = __builtin_amdgcn_logf(z) * LN2;   // (one step each; z is at least 1)
#pragma unroll
  for (int h = 0; h < 2; ++h)
    if (h * 64 < K) {
      L.p[h] = z == 0.f ? 0.f : L.p[h] * over;
      L.logp[h] -= logz;
    }
  L.mass = z == 0.f ? 0.f : z * over;   // 1; 0 of a row without entries; NaN of one with
}

struct DistillParams {
  const void* logits; int64_t ldl;
  const int64_t* idx;
  const float* tlogp;
  float *row_loss, *stats;
  float4* part;        // long rows: [R, units] DistillSums of each wave's columns
  int R, C, K, tail, units, unit_cols;
  float inv_t;
};
// Maximum and sum of e^((x - maximum) / T) of the classes that the list names and of the others (without tail: all are others), each of its own: with
// the row's maximum for both, others 87 nats below a named class had the sum 0 and were as good as not there.
// None: -FMAX and 0; whatever there is has a sum of at least about 1.
struct DistillSums { float ml, zl, mr, zr; };
// Statistics of the tail form, [m, n, w] a row: (max, log Z, Z of the named classes over Z of the others), infinite w where there are no others.
// Where the named classes lie more than FAR bits above the others, every class but them would be lost in the first two: then (max of the
// others, FAR_MARK - log of their Z, log-sum-exp of the named classes in the logits' unit), known by n < -1 (log Z is at least 0).
constexpr float FAR = 32.f, FAR_MARK = -2.f;
// by one wave: the row's loss from its sums and the listed classes' logits
__device__ __forceinline__ void finish_distill(const DistillParams& p, int64_t row, const Listed& L, float x0, float x1, const DistillSums& a,
                                               int lane) {
  const float c = p.inv_t * LOG2E, m = fmaxf(a.ml, a.mr);
  float z = a.zr;
  if (p.tail) z = fmaf(a.zl, __builtin_amdgcn_exp2f((a.ml - m) * c), a.zr * __builtin_amdgcn_exp2f((a.mr - m) * c));
  const float logz = __builtin_amdgcn_logf(z) * LN2;
  float loss = 0.f;
#pragma unroll
  for (int h = 0; h < 2; ++h)
    if (h * 64 < p.K && L.p[h] != 0.f) loss += L.p[h] * (L.logp[h] - (((h ? x1 : x0) - m) * p.inv_t - logz));
  loss = sum_wave(loss);
  if (lane == 0) {
    const bool none = z == 0.f;
    float s0 = m, s1 = logz, s2 = 0.f;
    if (p.tail) {
      const float left = 1.f - L.mass, gap = (a.ml - a.mr) * c;
      const bool far = gap > FAR && a.zr != 0.f;
      const float ratio = a.zl / a.zr * __builtin_amdgcn_exp2f(fminf(gap, FAR));
      // log of the student's rest = -log(1 + listed / others): the difference of two log-sums would lose it where little is listed
      if (left > 0.f && a.zr != 0.f)
        loss += left * (log1pf(-L.mass) + (far ? (a.ml - a.mr) * p.inv_t + __builtin_amdgcn_logf(a.zl / a.zr) * LN2 : log1pf(ratio)));
      s2 = a.zr == 0.f ? INFINITY : ratio;
      if (far && z == z) {
        s0 = a.mr;
        s1 = FAR_MARK - __builtin_amdgcn_logf(a.zr) * LN2;
        s2 = a.ml + __builtin_amdgcn_logf(a.zl) * LN2 / p.inv_t;
      }
    }
    p.row_loss[row] = none ? 0.f : loss;
    p.stats[3 * row] = none ? -INFINITY : s0;
    p.stats[3 * row + 1] = none ? -INFINITY : s1;
    p.stats[3 * row + 2] = none ? 0.f : s2;
  }
}
// A column's value as it was loaded: nothing is done to it, and so not waited for, before it is used.
template <typename T> struct Later {
  uint32_t bits = 0;
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (sizeof(T) == 4) bits = *reinterpret_cast<const uint32_t*>(p);
    else bits = *reinterpret_cast<const uint16_t*>(p);
  }
  __device__ __forceinline__ float value() const {
    if constexpr (sizeof(T) == 4) return __builtin_bit_cast(T, bits);
    else return (float)__builtin_bit_cast(T, (uint16_t)bits);
  }
};
template <typename T>
__device__ __forceinline__ void listed_logits(const T* row, const Listed& L, int K, Later<T> (&xl)[2]) {   // (some column's for an empty entry)
#pragma unroll
  for (int h = 0; h < 2; ++h)
    if (h * 64 < K) xl[h].load(row + max(L.id[h], 0));
}

__device__ __forceinline__ float4 as_part(const DistillSums& a) { return make_float4(a.ml, a.zl, a.mr, a.zr); }
// a row's sums, by one wave, from its units' parts; first: that of unit `lane`, or the last
__device__ __forceinline__ DistillSums join_parts(const DistillParams& p, const float4* part, float4 first, int lane) {
  if (lane >= p.units) first = make_float4(-FMAX, 0.f, -FMAX, 0.f);
  DistillSums a = {first.x, 0.f, first.z, 0.f};
  for (int u = lane + 64; u < p.units; u += 64) {
    a.ml = fmaxf(a.ml, part[u].x);
    a.mr = fmaxf(a.mr, part[u].z);
  }
  a.mr = max_wave(a.mr);
  if (p.tail) a.ml = max_wave(a.ml);
  const float c = p.inv_t * LOG2E;
  for (int u = lane; u < p.units; u += 64) {
    const float4 s = u < 64 ? first : part[u];
    if (p.tail) a.zl = fmaf(s.y, __builtin_amdgcn_exp2f((s.x - a.ml) * c), a.zl);
    a.zr = fmaf(s.w, __builtin_amdgcn_exp2f((s.z - a.mr) * c), a.zr);
  }
  if (p.tail) a.zl = sum_wave(a.zl);
  a.zr = sum_wave(a.zr);
  return a;
}
template <bool TAIL> struct Form { static constexpr bool value = TAIL; };
// as token_logprobs_fwd_kernel; with tail each wave marks the listed classes of its columns in a bit map of its own
template <typename T, Kind KIND, int NV, int UNITS = 4>
__global__ __launch_bounds__(KIND == ROW ? UNITS * 64 : 256, 8) void distill_fwd_kernel(DistillParams p) {
  __builtin_assume(p.K > 0);   // (no branch around a list's loads, and so no wait behind each)
  __shared__ uint32_t marks[UNITS][(WAVE_COLS + NARROW) / 32];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t id = (int64_t)blockIdx.x * 4 + wave;
  int64_t row = KIND == ROW ? blockIdx.x : id;
  int unit = KIND == ROW ? wave : 0;
  if (KIND == PART) split_id(id, p.units, row, unit);
  if (row >= p.R) return;
  const T* lr = (const T*)p.logits + row * p.ldl;
  const Cols cols(unit * p.unit_cols, unit == p.units - 1 ? p.C : (unit + 1) * p.unit_cols);
  const bool ends = KIND != PART && unit == 0;   // this wave has the row's last word
  ListLoads list;
  if (ends || p.tail) list = load_list(p.idx + row * p.K, p.tlogp + row * p.K, p.K, lane);
  Raw<T, NV> raw;
  load_raw(raw, lr, cols.c0, cols.wide, lane);
  const T narrow = cols.load_narrow(lr, p.C - 1, lane);
  Listed L;
  Later<T> xl[2];
  if (ends || p.tail) list_classes(L, list, p.K, p.C, lane);
  if (ends) listed_logits(lr, L, p.K, xl);
  uint32_t* mark = marks[wave];
  if (p.tail) {
    mark[lane] = 0;
    if (lane < NARROW / 32) mark[64 + lane] = 0;
    wave_fence();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int c = L.id[h];
      if (c >= cols.c0 && c < cols.end) atomicOr(&mark[(c - cols.c0) >> 5], 1u << ((c - cols.c0) & 31));
    }
    wave_fence();
  }
  if (ends) list_weights(L, list, p.K, p.inv_t, p.tail);
  const float xn = cols.narrow_value(narrow, p.C, lane);
  float x[NV][8];
  expand(raw, lr, cols.c0, cols.wide, lane, x);
  DistillSums a = {-FMAX, 0.f, -FMAX, 0.f};
  const float c = p.inv_t * LOG2E;
  auto sums = [&](auto form) {
    constexpr bool TAIL = decltype(form)::value;
    uint32_t hits[NV];     // the listed ones of a lane's columns, a bit each
    bool hit_n = false;
    if constexpr (TAIL) {
#pragma unroll
      for (int i = 0; i < NV; ++i) hits[i] = i < cols.steps ? reinterpret_cast<const uint8_t*>(mark)[i * 64 + lane] : 0u;
      const int at = cols.steps * 512 + lane;
      hit_n = cols.narrow() && (mark[at >> 5] >> (at & 31)) & 1u;
      if (hit_n) a.ml = fmaxf(xn, -FMAX);
    }
    if (!hit_n) a.mr = fmaxf(xn, -FMAX);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (TAIL && __any(hits[i] != 0)) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const bool hit = (hits[i] >> j) & 1u;
          a.ml = max_op(a.ml, hit ? x[i][j] : -FMAX);
          a.mr = max_op(a.mr, hit ? -FMAX : x[i][j]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) a.mr = max_op(a.mr, x[i][j]);
      }
    }
    a.mr = max_wave(a.mr);
    if (TAIL) a.ml = max_wave(a.ml);
    const Exponent er(a.mr, c), el(a.ml == -FMAX ? a.mr : a.ml, c);   // (without a listed class: nothing is taken from it)
    const bool plain = er.plain && (!TAIL || el.plain);
    auto add_up = [&](auto exponent) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (i >= cols.steps) break;
        if (TAIL && __any(hits[i] != 0)) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const bool hit = (hits[i] >> j) & 1u;
            const float e = __builtin_amdgcn_exp2f(exponent(x[i][j], hit));
            a.zl += hit ? e : 0.f;
            a.zr += hit ? 0.f : e;
          }
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) a.zr += __builtin_amdgcn_exp2f(exponent(x[i][j], false));
        }
      }
      if (cols.narrow()) {
        const float e = __builtin_amdgcn_exp2f(exponent(xn, hit_n));
        a.zl += hit_n ? e : 0.f;
        a.zr += hit_n ? 0.f : e;
      }
    };
    if (plain) add_up([&](float v, bool hit) { return fmaf(v, c, hit ? -el.mc : -er.mc); });
    else add_up([&](float v, bool hit) { return (v - (hit ? el.m : er.m)) * c; });
    a.zr = sum_wave(a.zr) * (plain ? __builtin_amdgcn_exp2f(-er.delta) : 1.f);
    if (TAIL) {
      a.zl = sum_wave(a.zl) * (plain ? __builtin_amdgcn_exp2f(-el.delta) : 1.f);
      if (a.zl != 0.f) a.ml = el.m;
    }
  };
  if (p.tail) sums(Form<true>{});
  else sums(Form<false>{});
  if constexpr (KIND == PART) {
    if (lane == 0) p.part[id] = as_part(a);
  } else {
    if constexpr (KIND == ROW) {
      __shared__ float4 sm_part[UNITS];
      if (lane == 0) sm_part[unit] = as_part(a);
      __syncthreads();
      if (unit) return;
      a = join_parts(p, sm_part, sm_part[min(lane, p.units - 1)], lane);
    }
    finish_distill(p, row, L, xl[0].value(), xl[1].value(), a, lane);
  }
}
template <typename T>
__global__ __launch_bounds__(256) void distill_join_kernel(DistillParams p) {   // a wave per row
  __builtin_assume(p.K > 0);
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= p.R) return;
  const float4* part = p.part + row * p.units;
  const ListLoads list = load_list(p.idx + row * p.K, p.tlogp + row * p.K, p.K, lane);
  const float4 first = part[min(lane, p.units - 1)];
  Listed L;
  list_classes(L, list, p.K, p.C, lane);
  Later<T> xl[2];
  listed_logits((const T*)p.logits + row * p.ldl, L, p.K, xl);
  list_weights(L, list, p.K, p.inv_t, p.tail);
  finish_distill(p, row, L, xl[0].value(), xl[1].value(), join_parts(p, part, first, lane), lane);
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
//          = q (mass + left) - p on those it names;
// where the named classes lie far above the others (finish_distill), with r = softmax of the others alone and s their share of the student's
// mass, q = s r of the former, and so d / dy = r ((mass + left) s - left):
// one exponential a class by the first form, then the few named ones again by the second, each by the lane that holds its entry (whose
// logit, and what is accumulated to, is fetched beside the row; a wave's own stores to one address stay in order).  Entries that
// name one class find out by leaving their number at its place in LDS: each then writes the sum of their p, in the list's order.
template <typename T, int NV>
__global__ __launch_bounds__(256) void distill_bwd_kernel(DistillGradParams p) {
  __builtin_assume(p.K > 0);
  __shared__ uint8_t tags[4][WAVE_COLS + NARROW];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t unit = (int64_t)blockIdx.x * 4 + wave;
  if (unit >= p.units) return;
  int64_t row;
  int piece;
  split_id(unit, p.per_row, row, piece);
  const int c0 = piece * p.wave_cols;
  const Cols cols(c0, piece == p.per_row - 1 ? p.Cd : c0 + p.wave_cols);   // of what is written; the classes end at cend
  const int dend = cols.wide, cend = min(p.C, cols.end);
  const T* lr = (const T*)p.logits + row * p.ldl;
  T* dr = (T*)p.dlogits + row * p.ldd;
  const ListLoads list = load_list(p.idx + row * p.K, p.tlogp + row * p.K, p.K, lane);
  Raw<T, NV> raw;
  load_raw(raw, lr, c0, min(p.C, cols.wide), lane);
  const T narrow = cols.load_narrow(lr, p.C - 1, lane);
  Listed L;
  list_classes(L, list, p.K, p.C, lane);
  bool here[2];
  Later<T> xl[2], old[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    here[h] = L.id[h] >= c0 && L.id[h] < cend;
    if (h * 64 < p.K) {
      xl[h].load(lr + (here[h] ? L.id[h] : 0));
      if (p.accumulate) old[h].load(dr + (here[h] ? L.id[h] : 0));
    }
  }
  const float m = p.stats[3 * row], logz = p.stats[3 * row + 1], w = p.stats[3 * row + 2], g = p.g_loss[row] * p.inv_t;
  uint8_t* tag = tags[wave];
#pragma unroll
  for (int h = 0; h < 2; ++h)
    if (here[h]) tag[L.id[h] - c0] = (uint8_t)(lane + 64 * h);
  list_weights(L, list, p.K, p.inv_t, p.tail);
  float x[NV][8];
  expand(raw, lr, c0, min(p.C, cols.wide), lane, x);
  const float xn = cols.narrow_value(narrow, p.C, lane);
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
  const bool far = p.tail && !none && logz < -1.f;   // (uniform)
  const float on = L.mass + left, c = p.inv_t * LOG2E, log2z = (far ? FAR_MARK - logz : logz) * LOG2E;
  const float named_m = far ? w : m, named_log2z = far ? 0.f : log2z;
  const float off = (far ? on * __builtin_amdgcn_exp2f((m - w) * c + log2z) - left : left > 0.f ? L.mass - left * w : L.mass) * g;
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
    const int n = (p.accumulate ? min(cend, dend) : dend) - first;
    if (n <= 0) continue;
    if (p.accumulate) {
      float o[8];
      load8<T>(dr + first, n, o);
#pragma unroll
      for (int j = 0; j < 8; ++j) d[j] += o[j];
    }
    store8<T>(dr + first, n, d);
  }
  {
    const int col = cols.wide + lane;
    float d = col < p.C && !none ? __builtin_amdgcn_exp2f((xn - m) * c - log2z) * off : 0.f;
    if (col < (p.accumulate ? cend : cols.end)) {
      if (p.accumulate) d += (float)dr[col];
      dr[col] = (T)d;
    }
  }
  wave_fence();
  if (none) return;
#pragma unroll
  for (int h = 0; h < 2; ++h)
    if (here[h]) {
      const float q = __builtin_amdgcn_exp2f((xl[h].value() - named_m) * c - named_log2z);
      dr[L.id[h]] = (T)(old[h].value() + fmaf(q, on, -L.p[h]) * g);
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
  TTTS_REQUIRE(temperature >= TTTS_SCORE_MIN_TEMPERATURE && temperature <= TTTS_SCORE_MAX_TEMPERATURE,
               "%s: the temperature must be positive and finite, and log2 e over it finite in fp32", what);
  TTTS_REQUIRE(R == 0 || logits, "%s: null pointer", what);
  const uintptr_t es = dtype == TTTS_DTYPE_F32 ? 4 : 2;
  TTTS_REQUIRE(reinterpret_cast<uintptr_t>(logits) % es == 0, "%s: logits are not aligned to their type", what);
  return TTTS_OK;
}

static int need_workspace(const char* what, int64_t need, const void* ws, int64_t have) {
  TTTS_REQUIRE(need == 0 || (ws && have >= need && aligned16(ws)), "%s: needs a 16-byte aligned workspace of %lld bytes", what, (long long)need);
  return TTTS_OK;
}
static int need_grid(const char* what, int64_t grid, int threads = 256) {
  TTTS_REQUIRE(one_launch(grid, threads), "%s: more work than one launch holds", what);
  return TTTS_OK;
}

// n columns -> waves (1: one wave's) and the columns of each but the last, which takes the rest: whole 512s, as few steps as there can
// be, and no small rest but a narrow one
struct Units { int units, cols, narrow_at; };
static Units split_columns(int n) {
  const int rest = n % 512, narrow = rest <= NARROW ? rest : 0, steps = (int)cdiv(n - narrow, 512);
  Units u;
  u.units = steps > STEPS ? (int)cdiv(steps, STEPS) : 1;
  u.cols = steps > 0 ? (int)cdiv(steps, u.units) * 512 : 512;
  u.units = steps > 0 ? (int)cdiv(steps * 512, u.cols) : 1;
  u.narrow_at = n - narrow;
  return u;
}

// rows of the type whose units are the waves of one workgroup need no scratch (the queries do not know the type: 16 bits)
static_assert(RowUnits<float>::n * WAVE_COLS + NARROW == TTTS_SCORE_F32_NO_WORKSPACE, "its meaning");
static bool no_scratch(int32_t dtype, int32_t C) { return dtype == TTTS_DTYPE_F32 && C <= TTTS_SCORE_F32_NO_WORKSPACE; }

extern "C" int64_t ttts_token_logprobs_workspace_bytes(int32_t R, int32_t C, int32_t top_k) {
  const int units = C > 0 ? split_columns(C).units : 1;
  return R > 0 && units > RowUnits<bf16>::n ? (int64_t)R * units * (16 + (top_k > 0 ? 256 : 0)) : 0;
}

template <typename T>
static int launch_score(const ScoreParams& p, hipStream_t st) {
  const char* what = "token_logprobs_fwd";
  const int64_t grid = cdiv((int64_t)p.R * p.units, 4);
  int rc = need_grid(what, grid);
  if (!rc && p.k && p.units > 16) rc = need_grid(what, p.R, p.units <= 64 ? 256 : 1024);
  if (rc) return rc;
  if (p.units == 1) {
    const size_t lds = p.k ? 4 * WAVE_TOP_LDS * sizeof(typename WaveKey<T>::type) : 0;
    if (p.narrow_at <= 1024) token_logprobs_fwd_kernel<T, ONE, 2><<<(unsigned)grid, 256, lds, st>>>(p);
    else token_logprobs_fwd_kernel<T, ONE, STEPS><<<(unsigned)grid, 256, lds, st>>>(p);
    return check_launch(what);
  }
  if (p.units <= RowUnits<T>::n) {
    if (p.units <= 4) token_logprobs_fwd_kernel<T, ROW, STEPS, 4><<<(unsigned)p.R, p.units * 64, 0, st>>>(p);              // up to 8256 classes
    else if constexpr (RowUnits<T>::n > 4) {
      if (p.units <= 8) token_logprobs_fwd_kernel<T, ROW, STEPS, 8><<<(unsigned)p.R, p.units * 64, 0, st>>>(p);            // up to 16448
      else token_logprobs_fwd_kernel<T, ROW, STEPS, RowUnits<T>::n><<<(unsigned)p.R, p.units * 64, 0, st>>>(p);            // up to 32832
    }
    return check_launch(what);
  }
  token_logprobs_fwd_kernel<T, PART, STEPS><<<(unsigned)grid, 256, 0, st>>>(p);
  rc = check_launch(what);
  if (rc) return rc;
  if (p.k == 0) token_logprobs_join_kernel<T><<<(unsigned)cdiv(p.R, 4), 256, 0, st>>>(p);
  else if (p.units <= 16) {
    if constexpr (RowUnits<T>::n < 16) {
      if (p.units <= 8) token_logprobs_top_wave_kernel<T, 8><<<(unsigned)cdiv(p.R, 4), 256, 0, st>>>(p);
      else token_logprobs_top_wave_kernel<T, 16><<<(unsigned)cdiv(p.R, 4), 256, 0, st>>>(p);
    }
  }
  else if (p.units <= 64) token_logprobs_top_kernel<T, 4, 16><<<p.R, 256, 0, st>>>(p);     // up to 131136
  else token_logprobs_top_kernel<T, 16, 32><<<p.R, 1024, 0, st>>>(p);                      // up to TTTS_SCORE_MAX_CLASSES
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
  rc = need_workspace("token_logprobs_fwd", no_scratch(dtype, C) ? 0 : ttts_token_logprobs_workspace_bytes(R, C, top_k), workspace, workspace_bytes);
  if (rc) return rc;
  const Units u = split_columns(C);
  ScoreParams p{logits, ldl, tokens, logp, entropy, stats, top_logp, top_idx, (float4*)workspace, nullptr, R, C, top_k, u.units, u.cols, u.narrow_at, 1.0f / temperature};
  p.part_max = p.part + (int64_t)R * p.units;
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
  const int units = C > 0 ? split_columns(C).units : 1;
  return R > 0 && units > RowUnits<bf16>::n ? (int64_t)R * units * 16 : 0;
}

template <typename T>
static int launch_distill(const DistillParams& p, hipStream_t st) {
  const char* what = "distill_fwd";
  const int64_t grid = cdiv((int64_t)p.R * p.units, 4);
  int rc = need_grid(what, grid);
  if (rc) return rc;
  if (p.units == 1) {
    if (split_columns(p.C).narrow_at <= 1024) distill_fwd_kernel<T, ONE, 2><<<(unsigned)grid, 256, 0, st>>>(p);
    else distill_fwd_kernel<T, ONE, STEPS><<<(unsigned)grid, 256, 0, st>>>(p);
    return check_launch(what);
  }
  if (p.units <= RowUnits<T>::n) {
    if (p.units <= 4) distill_fwd_kernel<T, ROW, STEPS, 4><<<(unsigned)p.R, p.units * 64, 0, st>>>(p);
    else if constexpr (RowUnits<T>::n > 4) distill_fwd_kernel<T, ROW, STEPS, RowUnits<T>::n><<<(unsigned)p.R, p.units * 64, 0, st>>>(p);
    return check_launch(what);
  }
  distill_fwd_kernel<T, PART, STEPS><<<(unsigned)grid, 256, 0, st>>>(p);
  rc = check_launch(what);
  if (rc) return rc;
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
  rc = need_workspace("distill_fwd", no_scratch(dtype, C) ? 0 : ttts_distill_workspace_bytes(R, C), workspace, workspace_bytes);
  if (rc) return rc;
  const Units u = split_columns(C);
  const DistillParams p{logits, ldl, teacher_idx, teacher_logp, row_loss, stats, (float4*)workspace, R, C, K, tail != 0, u.units, u.cols, 1.0f / temperature};
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
  const Units u = split_columns(Cd);
  p.per_row = u.units;
  p.wave_cols = u.cols;
  p.units = (int64_t)R * p.per_row;
  const int64_t grid = cdiv(p.units, 4);
  rc = need_grid("distill_bwd", grid);
  if (rc) return rc;
  if (u.units == 1 && u.narrow_at <= 1024) TTTS_BY_TYPE(dtype, "distill_bwd", (distill_bwd_kernel<T, 2><<<(unsigned)grid, 256, 0, as_stream(stream)>>>(p)))
  else TTTS_BY_TYPE(dtype, "distill_bwd", (distill_bwd_kernel<T, STEPS><<<(unsigned)grid, 256, 0, as_stream(stream)>>>(p)))
  return check_launch("distill_bwd");
}
