// Paged key / value cache: pages [P, H, page, dh] shared by all sequences, a block table [M, pages] per sequence.
//   kv_page_write     : rows of new tokens -> their slots
//   attn_paged_decode : softmax(scale q K^T) V of one new token per sequence over the keys its table lists
// Everything that comes from device memory (slots, table entries, lengths) is checked there: a slot outside the cache writes
// nothing, keys of a page outside the cache are left out, a length beyond the table ends with it.
#include <float.h>
#include <math.h>

#include "common.hpp"

namespace ttts {

// One 16-byte piece of a row's keys and of its values per thread; pieces of a row run over (head, column).  Bound by HBM: 30011 rows of 8
// heads of 128, 232 MB read and written, take 46.5 us = 5.0 TB/s, what a large copy reaches.
__global__ __launch_bounds__(256) void kv_page_write_kernel(const uint4* __restrict__ k, const uint4* __restrict__ v, int64_t ks_n, int64_t ks_h,
                                                            int64_t vs_n, int64_t vs_h, uint4* __restrict__ kp, uint4* __restrict__ vp,
                                                            const int64_t* __restrict__ slots, int N, unsigned pieces, unsigned chunks,
                                                            int page_shift, int64_t n_slots) {
  const unsigned rows = 256 / pieces;                 // of a workgroup (at least one; longer rows: several rounds)
  const unsigned r = rows ? threadIdx.x / pieces : 0;
  const int64_t n = (int64_t)blockIdx.x * (rows ? rows : 1) + r;
  if (n >= N || (rows && r >= rows)) return;
  const int64_t slot = slots[n];
  if (slot < 0 || slot >= n_slots) return;
  const int64_t page = slot >> page_shift, at = slot & ((1 << page_shift) - 1);
  const unsigned heads = pieces / chunks;
  for (unsigned i = rows ? threadIdx.x % pieces : threadIdx.x; i < pieces; i += rows ? pieces : 256) {
    const unsigned h = i / chunks, c = i % chunks;
    const int64_t dst = (((page * heads + h) << page_shift) + at) * chunks + c;
    const uint4 x = k[n * ks_n + h * ks_h + c], y = v[n * vs_n + h * vs_h + c];
    kp[dst] = x;
    vp[dst] = y;
  }
}

struct PagedParams {
  const void *q, *kp, *vp;
  void* out;
  float *lse, *part_o, *part_ml;          // partial results of split sequences: [M, H, chunks, DH] and [M, H, chunks][2]
  const int32_t *table, *lens;
  int64_t qs_m, qs_h, os_m, os_h, ts_m;   // strides in elements
  int M, H, Hkv, group, tiles, page_shift, P, width, chunk, chunks, ordered;   // tiles: 16-row tiles of a head group; width: pages of a table row
  float scale_log2;
};

// The i-th sequence of a batch by length, longest first, in 16 steps of length, for up to PAGED_ORDERED sequences: a batch that fills the card
// several times over then ends with its short sequences (96 ragged ones up to 4096 keys, 8 heads of 128: 147 -> 139 us a call; 64 up to 2404,
// 8 heads of 64: 40.5 -> 39.2).
// Every workgroup works it out for itself, from one load a lane and 64 sequences.
constexpr int PAGED_ORDERED = 512;
__device__ __forceinline__ int ordered_sequence(const int32_t* lens, int M, int i, int longest, int lane) {
  constexpr int N = PAGED_ORDERED / 64;
  const float per = 16.f / (float)longest;
  int level[N];
#pragma unroll
  for (int j = 0; j < N; ++j) level[j] = j * 64 + lane < M ? max(0, min(15, (int)((float)lens[j * 64 + lane] * per))) : -1;
  for (int l = 15; l >= 0; --l) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if (j * 64 >= M) break;
      const unsigned long long mask = __ballot(level[j] == l);
      const int n = __builtin_popcountll(mask);
      if (i < n) {
        const int below = __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
        return j * 64 + __builtin_ctzll(__ballot(level[j] == l && below == i));
      }
      i -= n;
    }
  }
  return 0;   // (not reached: every sequence has a level)
}

// A weight e in [0, 1] enters the product with V as two numbers of the cache's type, hi + lo = weight e: with hi alone, rounded, the outputs' error
// was 17 % larger in bf16 (0.0019 of their size against 0.0016) than their own rounding makes it.  hi lies half a step to one and a
// half below the weight, so lo is above zero wherever hi is: an infinite value stays infinite.
template <typename T> struct Frag;
template <> struct Frag<bf16> {
  static constexpr float weight = 1.f;
  static __device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
  static __device__ __forceinline__ void split(float e, bf16& hi, bf16& lo) {
    const uint32_t h = __builtin_elementwise_sub_sat(__builtin_bit_cast(uint32_t, e), 0x8000u) & 0xffff0000u;
    hi = __builtin_bit_cast(bf16, (uint16_t)(h >> 16));
    lo = (bf16)(e - __builtin_bit_cast(float, h));
  }
};
template <> struct Frag<_Float16> {
  static constexpr float weight = 32768.f;   // a weight of one enters the product as this: fp16 then holds them down to 2^-39 of the
                                             // largest (thousands of keys 2^-25 below it are part of the result)
  static __device__ __forceinline__ f32x4 mfma(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
  static __device__ __forceinline__ void split(float e, _Float16& hi, _Float16& lo) {
    e *= weight;
    const float below = __builtin_bit_cast(float, __builtin_elementwise_sub_sat(__builtin_bit_cast(uint32_t, e), 0x1000u));
    hi = (_Float16)__builtin_amdgcn_cvt_pkrtz(below, below)[0];   // (towards zero)
    lo = (_Float16)(e - (float)hi);
  }
};
// One workgroup = one chunk of keys of one (sequence, key / value head, 16 query rows); its waves take the chunk's 32-key tiles in turn,
// each with a running maximum, sum and accumulator of its own, joined through LDS at the end.
// A tile never touches LDS: both products are 16x16x32 MFMAs with the operand layout row = lane & 15, k = 8 (lane >> 4) ..+7,
//   S[key][q]   = K Q^T   two products of 16 keys: lane (g = lane >> 4) gets the scores of keys 16 t + 4 g + r of query lane & 15;
//   O^T[d][q]  += V^T P   the k index is a key in ANY order that both operands share: with k = 8 g + 4 t + r <-> key 16 t + 4 g + r the
//                         weights are the B operand where they are, and a lane loads V rows 16 t + 4 g + r, DH / 16 neighbouring
//                         columns each, which it re-pairs across rows in registers (product r of DH / 16 has rows d = (DH / 16) m + r).
// The next tile's keys are loaded as soon as this one's have been multiplied, its values after the second product (held twice over,
// 64 registers more at 128 columns, they were no faster), the table entries another tile ahead.  Both parts of the weights (Frag) cost
// nothing that shows beside the loads: 175 us with them and without for 4 sequences of 130000 keys, 32 heads over 4 of 128.  The queries of a shared
// head fill rows of the products that are there anyway, so a cached key is read once for up to 16 of them.
template <typename T, int DH, int NW>
__global__ __launch_bounds__(NW * 64) void attn_paged_decode_kernel(PagedParams p) {
  constexpr int W = DH / 16, KC = DH / 32;
  typedef T T8 __attribute__((ext_vector_type(8)));
  typedef T TW __attribute__((ext_vector_type(W)));
  extern __shared__ __attribute__((aligned(16))) float paged_lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, g = lane >> 4;
  int id = blockIdx.x;
  const int hk = id % p.Hkv; id /= p.Hkv;
  const int tile = id % p.tiles; id /= p.tiles;
  const int chunk = id % p.chunks;
  const int64_t m = p.ordered ? ordered_sequence(p.lens, p.M, id / p.chunks, p.width << p.page_shift, lane) : id / p.chunks;
  const int len = min(p.lens[m], p.width << p.page_shift);
  const int c0 = chunk * p.chunk, c1 = min(len, c0 + p.chunk);
  if (c0 >= len && !(chunk == 0 && p.chunks == 1)) return;   // (the join looks at no chunk behind the sequence's end)
  const int rows = min(16, p.group - tile * 16);
  const int h0 = hk * p.group + tile * 16;
  T8 qf[KC];
#pragma unroll
  for (int c = 0; c < KC; ++c) {
    qf[c] = T8{};
    if (col < rows) qf[c] = *reinterpret_cast<const T8*>((const T*)p.q + m * p.qs_m + (int64_t)(h0 + col) * p.qs_h + 32 * c + 8 * g);
  }
  float mx = -FLT_MAX, l = 0.f;
  f32x4 acc[W];
#pragma unroll
  for (int r = 0; r < W; ++r) acc[r] = f32x4{0.f, 0.f, 0.f, 0.f};

  const int32_t* tab = p.table + m * p.ts_m;
  const int last = max((c1 - 1) >> p.page_shift, 0);
  auto entry = [&](int key) { return tab[min(key >> p.page_shift, last)]; };   // (never past the chunk's own pages)
  T8 kf[2][KC];
  TW vf[8];
  struct Place { int64_t base[2]; int ok[2]; };   // where a tile's two 16-key halves lie (a page holds whole halves), and whether they count
  auto place = [&](int key0, int e0, int e1) {
    Place w;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int e = h ? e1 : e0, key = key0 + 16 * h;
      w.ok[h] = key < c1 && e >= 0 && e < p.P;
      w.base[h] = ((((int64_t)(w.ok[h] ? e : 0) * p.Hkv + hk) << p.page_shift) + (key & ((1 << p.page_shift) - 1))) * DH;
    }
    return w;
  };
  auto load_k = [&](const Place& w) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int c = 0; c < KC; ++c) kf[h][c] = *reinterpret_cast<const T8*>((const T*)p.kp + w.base[h] + col * DH + 8 * g + 32 * c);
  };
  auto load_v = [&](const Place& w) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      vf[j] = *reinterpret_cast<const TW*>((const T*)p.vp + w.base[j >> 2] + (4 * g + (j & 3)) * DH + col * W);
  };
  constexpr int STEP = 32 * NW;
  int key = c0 + 32 * wave;
  if (key < c1) {
    Place cur = place(key, entry(key), entry(key + 16));
    load_k(cur);
    load_v(cur);
    int e0 = entry(key + STEP), e1 = entry(key + STEP + 16);
    for (; key < c1; key += STEP) {
      const bool more = key + STEP < c1;
      float s[8];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        f32x4 d = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < KC; ++c) d = Frag<T>::mfma(kf[h][c], qf[c], d);
#pragma unroll
        for (int r = 0; r < 4; ++r) s[4 * h + r] = d[r] * p.scale_log2;
      }
      Place next = cur;
      if (more) {
        next = place(key + STEP, e0, e1);
        load_k(next);
        e0 = entry(key + 2 * STEP); e1 = entry(key + 2 * STEP + 16);
      }
      if (!(cur.ok[0] && cur.ok[1] && key + 32 <= c1)) {   // keys behind the end, or of no page: whatever the memory holds there
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const bool in = cur.ok[j >> 2] && key + 16 * (j >> 2) + 4 * g + (j & 3) < c1;
          s[j] = in ? s[j] : -INFINITY;
          vf[j] = in ? vf[j] : TW{};
        }
      }
      float mt = fmaxf(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])), fmaxf(fmaxf(s[4], s[5]), fmaxf(s[6], s[7])));
      mt = over_rows(mt, max_op);
      if (__any(mt > mx)) {
        const float mn = fmaxf(mx, mt), a = __builtin_amdgcn_exp2f(mx - mn);
        l *= a;
#pragma unroll
        for (int r = 0; r < W; ++r) acc[r] *= a;
        mx = mn;
      }
      T8 hi, lo;                   // the weights in two parts of the cache's type; their sum is of the weights themselves
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float e = __builtin_amdgcn_exp2f(s[j] - mx);
        l += e;
        T a, b;
        Frag<T>::split(e, a, b);
        hi[j] = a;
        lo[j] = b;
      }
#pragma unroll
      for (int r = 0; r < W; ++r) {
        T8 a;
#pragma unroll
        for (int j = 0; j < 8; ++j) a[j] = vf[j][r];
        acc[r] = Frag<T>::mfma(a, lo, acc[r]);
        acc[r] = Frag<T>::mfma(a, hi, acc[r]);
      }
      if (more) load_v(next);
      cur = next;
    }
  }
  l = over_rows(l, add_op);
  // ---- join the waves
  float* sm_o = paged_lds;                       // [NW][rows][DH]
  float* sm_ml = paged_lds + NW * rows * DH;     // [NW][rows][2]
  if (col < rows) {
    float* o = sm_o + (wave * rows + col) * DH + 4 * g * W;   // acc[r][i] is d = (4 g + i) W + r
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int r = 0; r < W; ++r) o[i * W + r] = acc[r][i] * (1.f / Frag<T>::weight);
    if (g == 0) { sm_ml[(wave * rows + col) * 2] = mx; sm_ml[(wave * rows + col) * 2 + 1] = l; }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < rows * DH; e += NW * 64) {
    const int r = e / DH, d = e % DH;
    float M = sm_ml[r * 2];
#pragma unroll
    for (int w = 1; w < NW; ++w) M = fmaxf(M, sm_ml[(w * rows + r) * 2]);
    float L = 0.f, o = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float a = __builtin_amdgcn_exp2f(sm_ml[(w * rows + r) * 2] - M);
      L += sm_ml[(w * rows + r) * 2 + 1] * a;
      o += sm_o[(w * rows + r) * DH + d] * a;
    }
    const int64_t mh = m * p.H + h0 + r;
    if (p.chunks == 1) {
      ((T*)p.out)[m * p.os_m + (int64_t)(h0 + r) * p.os_h + d] = (T)(L == 0.f ? 0.f : o / L);
      if (d == 0) p.lse[mh] = L == 0.f ? -INFINITY : (M + __log2f(L)) * 0.6931471805599453f;
    } else {
      p.part_o[(mh * p.chunks + chunk) * DH + d] = o;
      if (d == 0) { p.part_ml[(mh * p.chunks + chunk) * 2] = M; p.part_ml[(mh * p.chunks + chunk) * 2 + 1] = L; }
    }
  }
}

// The chunks of a split sequence: one workgroup per (sequence, query head).  Every chunk's weight 2^(m - M), a chunk per thread, and DH / 4
// lanes per chunk that add up the weighted parts; the first 8 parts of a thread are on their way before the weights (and the
// length) are known, so it takes one round of loads up to 8 * 1024 / DH chunks.
constexpr int PAGED_MAX_CHUNKS = 2048;   // whose weights a workgroup holds; paged_split makes no more
template <typename T, int DH>
__global__ __launch_bounds__(256) void attn_paged_join_kernel(PagedParams p) {
  constexpr int LPC = DH / 4, G = 256 / LPC, AHEAD = 8;
  __shared__ float sm_w[PAGED_MAX_CHUNKS];
  __shared__ float4 sm_o[G][LPC];
  __shared__ float sm_r[2][4];
  const int64_t mh = blockIdx.x, m = mh / p.H;
  const int tid = threadIdx.x, sub = tid % LPC, grp = tid / LPC;
  const float2* ml = reinterpret_cast<const float2*>(p.part_ml) + mh * p.chunks;
  const float4* po = reinterpret_cast<const float4*>(p.part_o) + mh * p.chunks * LPC + sub;
  const int len = min(p.lens[m], p.width << p.page_shift);
  float4 ahead[AHEAD];                       // (parts behind the sequence's end were not written: whatever the memory holds, not used)
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) ahead[i] = po[(int64_t)min(grp + i * G, p.chunks - 1) * LPC];
  const float2 s0 = ml[min(tid, p.chunks - 1)];
  const int n = len > 0 ? (len + p.chunk - 1) / p.chunk : 0;
  float M = tid < n ? s0.x : -FLT_MAX;
  for (int c = tid + 256; c < n; c += 256) M = fmaxf(M, ml[c].x);
  M = over_wave(M, max_op);
  if ((tid & 63) == 0) sm_r[0][tid >> 6] = M;
  __syncthreads();
  M = fmaxf(fmaxf(sm_r[0][0], sm_r[0][1]), fmaxf(sm_r[0][2], sm_r[0][3]));
  float L = 0.f;
  for (int c = tid; c < n; c += 256) {
    const float2 s = c < 256 ? s0 : ml[c];
    const float w = __builtin_amdgcn_exp2f(s.x - M);
    sm_w[c] = w;
    L += s.y * w;
  }
  L = over_wave(L, add_op);
  if ((tid & 63) == 0) sm_r[1][tid >> 6] = L;
  __syncthreads();
  L = (sm_r[1][0] + sm_r[1][1]) + (sm_r[1][2] + sm_r[1][3]);
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add = [&](const float4& v, float w) {
    o.x = fmaf(v.x, w, o.x); o.y = fmaf(v.y, w, o.y); o.z = fmaf(v.z, w, o.z); o.w = fmaf(v.w, w, o.w);
  };
#pragma unroll
  for (int i = 0; i < AHEAD; ++i)
    if (grp + i * G < n) add(ahead[i], sm_w[grp + i * G]);
#pragma unroll 8
  for (int c = grp + AHEAD * G; c < n; c += G) add(po[(int64_t)c * LPC], sm_w[c]);
  sm_o[grp][sub] = o;
  __syncthreads();
  if (tid < DH) {
    float x = 0.f;
#pragma unroll
    for (int i = 0; i < G; ++i) x += reinterpret_cast<const float*>(sm_o[i])[tid];
    ((T*)p.out)[m * p.os_m + (mh % p.H) * p.os_h + tid] = (T)(L == 0.f ? 0.f : x / L);
    if (tid == 0) p.lse[mh] = L == 0.f ? -INFINITY : (M + __log2f(L)) * 0.6931471805599453f;
  }
}

// How sequences of up to `longest` keys (what the table holds; their lengths stay on the device) are split into chunks, one workgroup each;
// units = workgroups of an unsplit call:
//  * not at all up to 768 keys (three tiles for each of 8 waves): 613 keys of one sequence, 8 heads of 64: 6.0 us; split 6.4 - 7.0.
//    Nor up to 4096 keys where the units alone give every CU two workgroups (of 4 waves then): 64 sequences up to 2404, 8 heads:
//    40.5 us, 42.9 split; 96 up to 4096, 8 heads of 128: 147 us, 153 split (39.2 and 139 unsplit and longest first).
//  * into 256 keys, one tile a wave, while that gives the card's 256 CUs one workgroup each at most: 2404 keys of one sequence
//    6.9 us, against 10.8 in chunks of 1024; more workgroups than CUs cost more than they give (20000 keys: 12.2 us, 14.2 with 512).
//  * beyond that into 1024 keys or more, about 1024 workgroups (4 sequences of 130000 keys: 178 us, 188 with 2048), or about 2048
//    where a sequence gets few chunks, and chunks of at most 4096 keys while there are under 16384 of them: the lengths may be
//    anything up to the longest, and a workgroup's chunk is what the others wait for.
// No sequence gets more than PAGED_MAX_CHUNKS, the join's room (fewer than 8 units with tables of more than 8388608 keys would).
struct PagedSplit { int chunk, chunks, waves; };
static PagedSplit paged_split(int64_t units, int64_t longest) {
  auto least = [](int64_t a, int64_t b) { return a < b ? a : b; };
  auto most = [](int64_t a, int64_t b) { return a > b ? a : b; };
  PagedSplit s;
  int64_t n = 1;
  const bool many = units >= 512;
  if (longest > (many ? 4096 : 768)) {
    int64_t wide = cdiv(1024, units);
    if (wide < 8) wide = cdiv(2048, units);
    n = most(least(cdiv(longest, 1024), wide), least(cdiv(longest, 256), 256 / units));
    n = least(most(n, least(cdiv(longest, 4096), 16384 / units)), PAGED_MAX_CHUNKS);
  }
  s.waves = many && n == 1 ? 4 : 8;
  const int64_t c = cdiv(cdiv(longest, n), 32 * s.waves) * 32 * s.waves;
  s.chunk = (int)c;
  s.chunks = (int)cdiv(longest, c);
  return s;
}

}  // namespace ttts

using namespace ttts;

static int check_pages(const char* what, int32_t dtype, int32_t H, int32_t dh, int32_t page, int32_t P) {
  TTTS_REQUIRE(dtype == TTTS_DTYPE_BF16 || dtype == TTTS_DTYPE_F16, "%s: the cache is bf16 or fp16 (type code %d)", what, (int)dtype);
  TTTS_REQUIRE(dh == 32 || dh == 64 || dh == 128, "%s: head_dim must be 32, 64 or 128 (got %d)", what, dh);
  TTTS_REQUIRE(page >= 16 && page <= 1024 && (page & (page - 1)) == 0, "%s: the page size must be a power of two, 16 .. 1024 (got %d)", what, page);
  TTTS_REQUIRE(H > 0 && P > 0, "%s: need heads and pages (heads %d, pages %d)", what, H, P);
  return TTTS_OK;
}

extern "C" int ttts_kv_page_write(const void* k, const void* v, int64_t k_stride_n, int64_t k_stride_h, int64_t v_stride_n, int64_t v_stride_h,
                                  void* k_pages, void* v_pages, const int64_t* slots, int32_t dtype, int32_t N, int32_t H, int32_t head_dim,
                                  int32_t page, int32_t P, void* stream) {
  const int rc = check_pages("kv_page_write", dtype, H, head_dim, page, P);
  if (rc) return rc;
  TTTS_REQUIRE(N >= 0, "kv_page_write: negative number of rows");
  if (N == 0) return TTTS_OK;
  TTTS_REQUIRE(k && v && k_pages && v_pages && slots, "kv_page_write: null pointer");
  TTTS_REQUIRE(aligned16(k) && aligned16(v) && aligned16(k_pages) && aligned16(v_pages), "kv_page_write: 16-byte aligned bases are needed");
  TTTS_REQUIRE(((k_stride_n | k_stride_h | v_stride_n | v_stride_h) & 7) == 0, "kv_page_write: strides must be multiples of 8 elements");
  const unsigned chunks = head_dim / 8, pieces = H * chunks, rows = pieces < 256 ? 256 / pieces : 1;
  TTTS_REQUIRE(H <= 65536, "kv_page_write: %d heads", H);
  TTTS_REQUIRE(one_launch(cdiv(N, rows), 256), "kv_page_write: more work than one launch holds (%d rows)", N);
  kv_page_write_kernel<<<(unsigned)cdiv(N, rows), 256, 0, as_stream(stream)>>>((const uint4*)k, (const uint4*)v, k_stride_n / 8, k_stride_h / 8,
                                                                               v_stride_n / 8, v_stride_h / 8, (uint4*)k_pages, (uint4*)v_pages,
                                                                               slots, N, pieces, chunks, __builtin_ctz(page), (int64_t)P * page);
  return check_launch("kv_page_write");
}

static int64_t paged_tiles(int32_t H, int32_t Hkv) { return cdiv(H / Hkv, 16); }
// bytes of the partial results; 0 where no sequence is split
static int64_t paged_bytes(int64_t M, int64_t H, int dh, int chunks) { return chunks > 1 ? cdiv(M * H * chunks * (dh + 2) * 4, 16) * 16 : 0; }

extern "C" int64_t ttts_attn_paged_decode_workspace_bytes(int32_t M, int32_t H, int32_t Hkv, int32_t head_dim, int32_t page, int32_t width) {
  if (M <= 0 || Hkv <= 0 || H < Hkv || head_dim <= 0 || page <= 0 || width <= 0) return 0;
  return paged_bytes(M, H, head_dim, paged_split(M * (int64_t)Hkv * paged_tiles(H, Hkv), (int64_t)width * page).chunks);
}

template <typename T, int DH, int NW>
static int launch_paged_waves(const PagedParams& p, int64_t grid, hipStream_t st) {
  static OnceFlag once;
  const int lds = NW * (p.group < 16 ? p.group : 16) * (DH + 2) * 4;
  if (lds > 64 * 1024 && lds_opt_in(once, (const void*)attn_paged_decode_kernel<T, DH, NW>, NW * 16 * (DH + 2) * 4) != hipSuccess)
    return fail(TTTS_EHIP, "attn_paged_decode: LDS opt-in failed");
  attn_paged_decode_kernel<T, DH, NW><<<(unsigned)grid, NW * 64, lds, st>>>(p);
  return check_launch("attn_paged_decode");
}
template <typename T, int DH>
static int launch_paged(const PagedParams& p, int waves, int64_t grid, int64_t rows, hipStream_t st) {
  const int rc = waves == 4 ? launch_paged_waves<T, DH, 4>(p, grid, st) : launch_paged_waves<T, DH, 8>(p, grid, st);
  if (rc || p.chunks == 1) return rc;
  attn_paged_join_kernel<T, DH><<<(unsigned)rows, 256, 0, st>>>(p);
  return check_launch("attn_paged_decode join");
}

extern "C" int ttts_attn_paged_decode(const void* q, int64_t q_stride_m, int64_t q_stride_h, const void* k_pages, const void* v_pages,
                                      const int32_t* block_table, int64_t table_stride, const int32_t* seq_lens, void* out,
                                      int64_t o_stride_m, int64_t o_stride_h, float* lse, int32_t dtype, int32_t M, int32_t H, int32_t Hkv,
                                      int32_t head_dim, int32_t page, int32_t P, int32_t width, float scale, void* workspace,
                                      int64_t workspace_bytes, void* stream) {
  int rc = check_pages("attn_paged_decode", dtype, Hkv, head_dim, page, P);
  if (rc) return rc;
  TTTS_REQUIRE(M >= 0 && H > 0 && H % Hkv == 0, "attn_paged_decode: need M >= 0 and H %% Hkv == 0 (M %d, H %d, Hkv %d)", M, H, Hkv);
  TTTS_REQUIRE(width > 0 && table_stride >= width && (int64_t)width * page <= 0x40000000,
               "attn_paged_decode: bad block table (width %d, row pitch %lld, at most 2^30 keys)", width, (long long)table_stride);
  const float scale_log2 = scale * 1.4426950408889634f;
  TTTS_REQUIRE(scale_log2 - scale_log2 == 0.f, "attn_paged_decode: the scale must be finite, times log2 e too");
  if (M == 0) return TTTS_OK;
  TTTS_REQUIRE(q && k_pages && v_pages && block_table && seq_lens && out && lse, "attn_paged_decode: null pointer");
  TTTS_REQUIRE(aligned16(q) && aligned16(k_pages) && aligned16(v_pages) && aligned16(out), "attn_paged_decode: 16-byte aligned bases are needed");
  TTTS_REQUIRE(((q_stride_m | q_stride_h | o_stride_m | o_stride_h) & 7) == 0, "attn_paged_decode: strides must be multiples of 8 elements");
  PagedParams p{};
  p.q = q; p.kp = k_pages; p.vp = v_pages; p.out = out; p.lse = lse; p.table = block_table; p.lens = seq_lens;
  p.qs_m = q_stride_m; p.qs_h = q_stride_h; p.os_m = o_stride_m; p.os_h = o_stride_h; p.ts_m = table_stride;
  p.M = M; p.H = H; p.Hkv = Hkv; p.group = H / Hkv; p.tiles = (int)paged_tiles(H, Hkv); p.page_shift = __builtin_ctz(page); p.P = P; p.width = width;
  p.scale_log2 = scale_log2;
  const int64_t units = M * (int64_t)Hkv * p.tiles;
  const PagedSplit sp = paged_split(units, (int64_t)width * page);
  p.chunk = sp.chunk; p.chunks = sp.chunks;
  TTTS_REQUIRE(p.chunks <= PAGED_MAX_CHUNKS, "attn_paged_decode: %d parts of a sequence, more than the join holds", p.chunks);
  p.ordered = units >= 512 && M <= PAGED_ORDERED;
  const int64_t grid = units * p.chunks, rows = (int64_t)M * H, need = paged_bytes(M, H, head_dim, p.chunks);
  TTTS_REQUIRE(one_launch(grid, sp.waves * 64) && one_launch(rows, 256), "attn_paged_decode: more work than one launch holds (M %d, H %d)", M, H);
  TTTS_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && aligned16(workspace)),
               "attn_paged_decode: needs a 16-byte aligned workspace of %lld bytes", (long long)need);
  p.part_o = (float*)workspace;
  p.part_ml = p.part_o + rows * p.chunks * head_dim;
  hipStream_t st = as_stream(stream);
  if (dtype == TTTS_DTYPE_BF16)
    return head_dim == 32 ? launch_paged<bf16, 32>(p, sp.waves, grid, rows, st) : head_dim == 64 ? launch_paged<bf16, 64>(p, sp.waves, grid, rows, st)
                                                                                       : launch_paged<bf16, 128>(p, sp.waves, grid, rows, st);
  return head_dim == 32 ? launch_paged<_Float16, 32>(p, sp.waves, grid, rows, st) : head_dim == 64 ? launch_paged<_Float16, 64>(p, sp.waves, grid, rows, st)
                                                                                         : launch_paged<_Float16, 128>(p, sp.waves, grid, rows, st);
}
