// Paged key / value cache: pages [P, H, page, dh] shared by all sequences, a block table [M, pages] per sequence.
//   kv_page_write     : rows of new tokens -> their slots
//   attn_paged_decode : softmax(scale q K^T) V of one new token per sequence over the keys its table lists
// Everything that comes from device memory (slots, table entries, lengths) is checked there: a slot outside the cache writes
// nothing, keys of a page outside the cache are left out, a length beyond the table ends with it.
#include <math.h>

#include "common.hpp"

namespace ttts {

// one 16-byte piece per thread: piece (n, which, h, c) of row n
__global__ __launch_bounds__(256) void kv_page_write_kernel(const uint4* __restrict__ k, const uint4* __restrict__ v, int64_t ks_n, int64_t ks_h,
                                                            int64_t vs_n, int64_t vs_h, uint4* __restrict__ kp, uint4* __restrict__ vp,
                                                            const int64_t* __restrict__ slots, int64_t total, int H, int chunks, int page,
                                                            int64_t n_slots) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int c = (int)(i % chunks);
    const int h = (int)(i / chunks % H);
    const int64_t n = i / chunks / H;
    const int64_t slot = slots[n];
    if (slot < 0 || slot >= n_slots) continue;
    const int64_t dst = (((slot / page) * H + h) * page + slot % page) * chunks + c;
    kp[dst] = k[n * ks_n + h * ks_h + c];
    vp[dst] = v[n * vs_n + h * vs_h + c];
  }
}

struct PagedParams {
  const void *q, *kp, *vp;
  void* out;
  float* lse;
  const int32_t *table, *lens;
  int64_t qs_m, qs_h, os_m, os_h, ts_m;   // strides in elements
  int M, H, Hkv, page, P, width;          // width: pages of a table row
  float scale_log2;
};

template <typename T, int DH>
__global__ __launch_bounds__(256) void attn_paged_decode_kernel(PagedParams p) {
  constexpr int LPK = DH / 8, KPW = 64 / LPK;
  typedef T T8 __attribute__((ext_vector_type(8)));
  __shared__ float sm_acc[4][DH];
  __shared__ float sm_ml[4][2];
  const int h = blockIdx.x, m = blockIdx.y, hk = h / (p.H / p.Hkv);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, sub = lane % LPK, grp = lane / LPK;
  const int len = min(p.lens[m], (int)min((int64_t)p.width * p.page, (int64_t)0x7fffffff));
  const T8 qv = *reinterpret_cast<const T8*>((const T*)p.q + m * p.qs_m + h * p.qs_h + sub * 8);
  float mx = -3.0e38f, l = 0.f, acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  for (int k0 = wave * KPW; k0 < len; k0 += 4 * KPW) {
    const int key = k0 + grp;
    if (key >= len) continue;
    const int pg = p.table[m * p.ts_m + key / p.page];
    if (pg < 0 || pg >= p.P) continue;
    const int64_t at = (((int64_t)pg * p.Hkv + hk) * p.page + key % p.page) * DH + sub * 8;
    const T8 kv = *reinterpret_cast<const T8*>((const T*)p.kp + at), vv = *reinterpret_cast<const T8*>((const T*)p.vp + at);
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) s = fmaf((float)qv[e], (float)kv[e], s);
#pragma unroll
    for (int o = 1; o < LPK; o <<= 1) s += __shfl_xor(s, o, 64);
    s *= p.scale_log2;
    const float mn = fmaxf(mx, s), a = __builtin_amdgcn_exp2f(mx - mn), e = __builtin_amdgcn_exp2f(s - mn);
    l = l * a + e;
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] = acc[j] * a + e * (float)vv[j];
    mx = mn;
  }
#pragma unroll
  for (int o = LPK; o < 64; o <<= 1) {
    const float m2 = __shfl_xor(mx, o, 64), l2 = __shfl_xor(l, o, 64), mn = fmaxf(mx, m2);
    const float a = __builtin_amdgcn_exp2f(mx - mn), b = __builtin_amdgcn_exp2f(m2 - mn);
    l = l * a + l2 * b;
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] = acc[j] * a + __shfl_xor(acc[j], o, 64) * b;
    mx = mn;
  }
  if (grp == 0) {
#pragma unroll
    for (int j = 0; j < 8; ++j) sm_acc[wave][sub * 8 + j] = acc[j];
    if (sub == 0) { sm_ml[wave][0] = mx; sm_ml[wave][1] = l; }
  }
  __syncthreads();
  if (threadIdx.x < DH) {
    const float M = fmaxf(fmaxf(sm_ml[0][0], sm_ml[1][0]), fmaxf(sm_ml[2][0], sm_ml[3][0]));
    float L = 0.f, o = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float a = __builtin_amdgcn_exp2f(sm_ml[w][0] - M);
      L += sm_ml[w][1] * a;
      o += sm_acc[w][threadIdx.x] * a;
    }
    ((T*)p.out)[m * p.os_m + h * p.os_h + threadIdx.x] = (T)(L == 0.f ? 0.f : o / L);
    if (threadIdx.x == 0) p.lse[(int64_t)m * p.H + h] = L == 0.f ? -INFINITY : (M + __log2f(L)) * 0.6931471805599453f;
  }
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
  const int chunks = head_dim / 8;
  const int64_t total = (int64_t)N * H * chunks;
  const int grid = (int)(cdiv(total, 256) < 1048576 ? cdiv(total, 256) : 1048576);
  kv_page_write_kernel<<<grid, 256, 0, as_stream(stream)>>>((const uint4*)k, (const uint4*)v, k_stride_n / 8, k_stride_h / 8, v_stride_n / 8,
                                                             v_stride_h / 8, (uint4*)k_pages, (uint4*)v_pages, slots, total, H, chunks, page,
                                                             (int64_t)P * page);
  return check_launch("kv_page_write");
}

extern "C" int64_t ttts_attn_paged_decode_workspace_bytes(int32_t M, int32_t H, int32_t Hkv, int32_t head_dim, int32_t page, int32_t width) {
  return 0;
}

template <typename T>
static void launch_paged(const PagedParams& p, int dh, hipStream_t st) {
  const dim3 grid(p.H, p.M);
  if (dh == 32) attn_paged_decode_kernel<T, 32><<<grid, 256, 0, st>>>(p);
  else if (dh == 64) attn_paged_decode_kernel<T, 64><<<grid, 256, 0, st>>>(p);
  else attn_paged_decode_kernel<T, 128><<<grid, 256, 0, st>>>(p);
}

extern "C" int ttts_attn_paged_decode(const void* q, int64_t q_stride_m, int64_t q_stride_h, const void* k_pages, const void* v_pages,
                                      const int32_t* block_table, int64_t table_stride, const int32_t* seq_lens, void* out,
                                      int64_t o_stride_m, int64_t o_stride_h, float* lse, int32_t dtype, int32_t M, int32_t H, int32_t Hkv,
                                      int32_t head_dim, int32_t page, int32_t P, int32_t width, float scale, void* workspace,
                                      int64_t workspace_bytes, void* stream) {
  const int rc = check_pages("attn_paged_decode", dtype, Hkv, head_dim, page, P);
  if (rc) return rc;
  TTTS_REQUIRE(M >= 0 && M <= 65535 && H > 0 && H % Hkv == 0, "attn_paged_decode: need 0 <= M <= 65535 and H %% Hkv == 0 (M %d, H %d, Hkv %d)", M, H, Hkv);
  TTTS_REQUIRE(width > 0 && table_stride >= width && (int64_t)width * page <= 0x7fffffff, "attn_paged_decode: bad block table");
  TTTS_REQUIRE(scale == scale && scale - scale == 0.f, "attn_paged_decode: the scale must be finite");
  if (M == 0) return TTTS_OK;
  TTTS_REQUIRE(q && k_pages && v_pages && block_table && seq_lens && out && lse, "attn_paged_decode: null pointer");
  TTTS_REQUIRE(aligned16(q) && aligned16(k_pages) && aligned16(v_pages) && aligned16(out), "attn_paged_decode: 16-byte aligned bases are needed");
  TTTS_REQUIRE(((q_stride_m | q_stride_h | o_stride_m | o_stride_h) & 7) == 0, "attn_paged_decode: strides must be multiples of 8 elements");
  PagedParams p{q, k_pages, v_pages, out, lse, block_table, seq_lens, q_stride_m, q_stride_h, o_stride_m, o_stride_h, table_stride,
                M, H, Hkv, page, P, width, scale * 1.4426950408889634f};
  if (dtype == TTTS_DTYPE_BF16) launch_paged<bf16>(p, head_dim, as_stream(stream));
  else launch_paged<_Float16>(p, head_dim, as_stream(stream));
  return check_launch("attn_paged_decode");
}
