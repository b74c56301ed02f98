// Scoring of given tokens and distillation on a teacher's alternatives: row operators over logits [R, ldl], C classes a row.
//   token_logprobs : y = x / T, log p of the given token, entropy, the k best classes with their log p; and the gradient
//   distill        : KL(teacher's listed classes || student), optionally with the mass that the list leaves out; and the gradient
// All sums, maxima and statistics are fp32 whatever the logits' type; a row's maximum m and log Z = log sum e^((x - m) / T) are
// handed to the gradient APART: one log-sum-exp would round log Z to the maximum's step.
#include <math.h>

#include "common.hpp"

namespace ttts {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

template <typename T>
struct Row {   // one row of logits as fp32
  const T* p;
  __device__ __forceinline__ float operator[](int64_t c) const { return (float)p[c]; }
};

constexpr int ROW_T = 256;
template <typename F>
__device__ __forceinline__ float block_reduce(float v, F op, float* sh) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = op(v, __shfl_xor(v, o, 64));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  return op(op(sh[0], sh[1]), op(sh[2], sh[3]));
}
__device__ __forceinline__ float add_f(float a, float b) { return a + b; }
__device__ __forceinline__ float max_f(float a, float b) { return fmaxf(a, b); }

// (value, class) order of the alternatives: larger value first, lower class first among equals
__device__ __forceinline__ bool before(float va, int ia, float vb, int ib) { return va > vb || (va == vb && ia < ib); }

// e = 2^((x - m) c), t = (x - m) c kept finite (a class at -inf, or at the type's lowest value, has e = 0: e t must be 0, not NaN).
// m is never -inf here (>= -FLT_MAX), so -inf - m = -inf; NaN passes through e.
__device__ __forceinline__ float expo(float x, float m, float c, float& t) {
  t = (x - m) * c;
  const float e = __builtin_amdgcn_exp2f(t);
  t = fmaxf(t, -200.f);
  return e;
}

template <typename T>
__global__ __launch_bounds__(ROW_T) void token_logprobs_fwd_kernel(const T* __restrict__ logits, int64_t ldl,
                                                                   const int64_t* __restrict__ tokens, float* __restrict__ logp,
                                                                   float* __restrict__ entropy, float* __restrict__ stats,
                                                                   float* __restrict__ top_logp, int64_t* __restrict__ top_idx, int C,
                                                                   int top_k, float inv_t) {
  __shared__ float sh[4];
  __shared__ float shv[4];
  __shared__ int shi[4];
  const int64_t row = blockIdx.x;
  const Row<T> x{logits + row * ldl};
  const float c = inv_t * LOG2E;
  float mx = -3.402823466e38f;
  for (int i = threadIdx.x; i < C; i += ROW_T) mx = fmaxf(mx, x[i]);
  mx = block_reduce(mx, max_f, sh);
  float z = 0.f, s = 0.f;
  for (int i = threadIdx.x; i < C; i += ROW_T) {
    float t;
    const float e = expo(x[i], mx, c, t);
    z += e;
    s = fmaf(e, t, s);
  }
  z = block_reduce(z, add_f, sh);
  s = block_reduce(s, add_f, sh);
  const bool none = z == 0.f;          // every class at -inf
  const float log2z = __log2f(z);
  if (threadIdx.x == 0) {
    const int64_t tok = tokens[row];
    stats[2 * row] = none ? -INFINITY : mx;
    stats[2 * row + 1] = none ? -INFINITY : log2z * LN2;
    entropy[row] = none ? 0.f : (log2z - s / z) * LN2;
    float lp = 0.f;
    if (tok >= 0 && tok < C) lp = none ? -INFINITY : (x[tok] - mx) * inv_t - log2z * LN2;
    logp[row] = lp;
  }
  float pv = INFINITY;
  int pi = -1;
  for (int k = 0; k < top_k; ++k) {
    float bv = -INFINITY;
    int bi = 0x7fffffff;
    if (z == z)
      for (int i = threadIdx.x; i < C; i += ROW_T) {
        const float v = x[i];
        if (v > -INFINITY && before(pv, pi, v, i) && before(v, i, bv, bi)) { bv = v; bi = i; }
      }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const float v2 = __shfl_xor(bv, o, 64);
      const int i2 = __shfl_xor(bi, o, 64);
      if (before(v2, i2, bv, bi)) { bv = v2; bi = i2; }
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) { shv[threadIdx.x >> 6] = bv; shi[threadIdx.x >> 6] = bi; }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 4; ++w)
      if (before(shv[w], shi[w], bv, bi)) { bv = shv[w]; bi = shi[w]; }
    const bool have = bi != 0x7fffffff;
    if (threadIdx.x == 0) {
      top_idx[row * top_k + k] = have ? bi : -1;
      top_logp[row * top_k + k] = z != z ? z : (have ? (bv - mx) * inv_t - log2z * LN2 : -INFINITY);
    }
    pv = have ? bv : -INFINITY;
    pi = bi;
  }
}

template <typename T>
__global__ __launch_bounds__(ROW_T) void token_logprobs_bwd_kernel(const T* __restrict__ logits, int64_t ldl,
                                                                   const int64_t* __restrict__ tokens, const float* __restrict__ stats,
                                                                   const float* __restrict__ entropy, const float* __restrict__ g_logp,
                                                                   const float* __restrict__ g_entropy, T* __restrict__ dlogits,
                                                                   int64_t ldd, int C, int Cd, float inv_t) {
  const int64_t row = blockIdx.x;
  const Row<T> x{logits + row * ldl};
  const float mx = stats[2 * row], logz = stats[2 * row + 1], H = entropy[row];
  const int64_t tok = tokens[row];
  const bool given = tok >= 0 && tok < C;
  const float gl = given ? g_logp[row] : 0.f, gh = g_entropy ? g_entropy[row] : 0.f;
  for (int i = threadIdx.x; i < Cd; i += ROW_T) {
    float d = 0.f;
    if (i < C && mx != -INFINITY) {
      const float y = (x[i] - mx) * inv_t - logz;
      const float p = __builtin_amdgcn_exp2f(y * LOG2E);
      d = -gl * p - (p == 0.f ? 0.f : gh * p * (y + H));
      if (given && i == tok) d += gl;
      d *= inv_t;
    }
    dlogits[row * ldd + i] = (T)d;
  }
}

// the teacher's list of one row in LDS: class (or -1), p and log p
struct Listed {
  int idx[TTTS_DISTILL_MAX_K];
  float p[TTTS_DISTILL_MAX_K], logp[TTTS_DISTILL_MAX_K];
};
__device__ __forceinline__ void load_listed(Listed& L, const int64_t* idx, const float* tl, int K, int C, float inv_t, int tail, float& mass,
                                            float* sh) {
  const int j = threadIdx.x;
  int id = -1;
  float t = -INFINITY;
  if (j < K) {
    const int64_t i = idx[j];
    if (i >= 0 && i < C) { id = (int)i; t = tl[j]; }
  }
  float p, lp;
  if (tail) {
    lp = t;
    p = id >= 0 ? __expf(t) : 0.f;
  } else {
    const float m = fmaxf(block_reduce(t, max_f, sh), -3.402823466e38f);
    const float u = (t - m) * inv_t;
    const float e = id >= 0 ? __expf(u) : 0.f;
    const float z = block_reduce(e, add_f, sh);
    p = z > 0.f ? e / z : (z == 0.f ? 0.f : z);
    lp = u - __logf(z);
  }
  if (j < K) { L.idx[j] = id; L.p[j] = p; L.logp[j] = lp; }
  mass = block_reduce(p, add_f, sh);
  __syncthreads();
}

template <typename T>
__global__ __launch_bounds__(ROW_T) void distill_fwd_kernel(const T* __restrict__ logits, int64_t ldl, const int64_t* __restrict__ tidx,
                                                            const float* __restrict__ tlogp, float* __restrict__ row_loss,
                                                            float* __restrict__ stats, int C, int K, float inv_t, int tail) {
  __shared__ float sh[4];
  __shared__ Listed L;
  const int64_t row = blockIdx.x;
  const Row<T> x{logits + row * ldl};
  const float c = inv_t * LOG2E;
  float mass;
  load_listed(L, tidx + row * K, tlogp + row * K, K, C, inv_t, tail, mass, sh);
  float mx = -3.402823466e38f;
  for (int i = threadIdx.x; i < C; i += ROW_T) mx = fmaxf(mx, x[i]);
  mx = block_reduce(mx, max_f, sh);
  float zl = 0.f, zr = 0.f;
  for (int i = threadIdx.x; i < C; i += ROW_T) {
    float t;
    const float e = expo(x[i], mx, c, t);
    bool hit = false;
    for (int j = 0; j < K; ++j) hit |= L.idx[j] == i;
    if (hit) zl += e; else zr += e;
  }
  zl = block_reduce(zl, add_f, sh);
  zr = block_reduce(zr, add_f, sh);
  const float z = zl + zr;
  const bool none = z == 0.f;
  const float logz = __logf(z);
  float loss = 0.f;
  if ((int)threadIdx.x < K && L.idx[threadIdx.x] >= 0) {
    const float p = L.p[threadIdx.x];
    const float logq = (x[L.idx[threadIdx.x]] - mx) * inv_t - logz;
    loss = p == 0.f ? 0.f : p * (L.logp[threadIdx.x] - logq);
  }
  loss = block_reduce(loss, add_f, sh);
  if (threadIdx.x == 0) {
    const float left = 1.f - mass;
    if (tail && left > 0.f && zr > 0.f) loss += left * (log1pf(-mass) + log1pf(zl / zr));
    row_loss[row] = none ? 0.f : loss;
    stats[3 * row] = none ? -INFINITY : mx;
    stats[3 * row + 1] = none ? -INFINITY : logz;
    stats[3 * row + 2] = none ? -INFINITY : __logf(zr);
  }
}

template <typename T>
__global__ __launch_bounds__(ROW_T) void distill_bwd_kernel(const T* __restrict__ logits, int64_t ldl, const int64_t* __restrict__ tidx,
                                                            const float* __restrict__ tlogp, const float* __restrict__ stats,
                                                            const float* __restrict__ g_loss, T* __restrict__ dlogits, int64_t ldd, int C,
                                                            int Cd, int K, float inv_t, int tail, int accumulate) {
  __shared__ float sh[4];
  __shared__ Listed L;
  const int64_t row = blockIdx.x;
  const Row<T> x{logits + row * ldl};
  float mass;
  load_listed(L, tidx + row * K, tlogp + row * K, K, C, inv_t, tail, mass, sh);
  const float mx = stats[3 * row], logz = stats[3 * row + 1], logzr = stats[3 * row + 2];
  const float left = tail && logzr > -INFINITY ? fmaxf(1.f - mass, 0.f) : 0.f;
  const float g = g_loss[row] * inv_t;
  for (int i = threadIdx.x; i < Cd; i += ROW_T) {
    float d = 0.f;
    if (i < C && mx != -INFINITY) {
      const float u = (x[i] - mx) * inv_t;
      const float q = __expf(u - logz);
      float p = 0.f;
      bool hit = false;
      for (int j = 0; j < K; ++j)
        if (L.idx[j] == i) { p += L.p[j]; hit = true; }
      d = q * (mass + left) - p;
      if (left > 0.f && !hit) d -= left * __expf(u - logzr);
      d *= g;
    }
    T* o = dlogits + row * ldd + i;
    if (accumulate) { if (i < C) *o = (T)((float)*o + d); }
    else *o = (T)d;
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

extern "C" int64_t ttts_token_logprobs_workspace_bytes(int32_t R, int32_t C, int32_t top_k) { return 0; }

extern "C" int ttts_token_logprobs_fwd(const void* logits, int32_t dtype, int64_t ldl, const int64_t* tokens, float* logp, float* entropy,
                                       float* stats, float* top_logp, int64_t* top_idx, int32_t R, int32_t C, int32_t top_k,
                                       float temperature, void* workspace, int64_t workspace_bytes, void* stream) {
  int rc = check_logits("token_logprobs_fwd", logits, dtype, ldl, R, C, temperature);
  if (rc) return rc;
  TTTS_REQUIRE(top_k >= 0 && top_k <= TTTS_SCORE_MAX_TOP, "token_logprobs_fwd: need 0 <= top_k <= %d", TTTS_SCORE_MAX_TOP);
  if (R == 0) return TTTS_OK;
  TTTS_REQUIRE(tokens && logp && entropy && stats && (top_k == 0 || (top_logp && top_idx)), "token_logprobs_fwd: null pointer");
  TTTS_BY_TYPE(dtype, "token_logprobs_fwd",
               (token_logprobs_fwd_kernel<T><<<R, ROW_T, 0, as_stream(stream)>>>((const T*)logits, ldl, tokens, logp, entropy, stats, top_logp,
                                                                                top_idx, C, top_k, 1.0f / temperature)));
  return check_launch("token_logprobs_fwd");
}

extern "C" int ttts_token_logprobs_bwd(const void* logits, int32_t dtype, int64_t ldl, const int64_t* tokens, const float* stats,
                                       const float* entropy, const float* g_logp, const float* g_entropy, void* dlogits, int64_t ldd,
                                       int32_t R, int32_t C, int32_t Cd, float temperature, void* stream) {
  int rc = check_logits("token_logprobs_bwd", logits, dtype, ldl, R, C, temperature);
  if (rc) return rc;
  TTTS_REQUIRE(Cd >= C && ldd >= Cd, "token_logprobs_bwd: need C <= Cd <= ldd");
  if (R == 0) return TTTS_OK;
  TTTS_REQUIRE(tokens && stats && entropy && g_logp && dlogits, "token_logprobs_bwd: null pointer");
  TTTS_BY_TYPE(dtype, "token_logprobs_bwd",
               (token_logprobs_bwd_kernel<T><<<R, ROW_T, 0, as_stream(stream)>>>((const T*)logits, ldl, tokens, stats, entropy, g_logp, g_entropy,
                                                                                (T*)dlogits, ldd, C, Cd, 1.0f / temperature)));
  return check_launch("token_logprobs_bwd");
}

extern "C" int64_t ttts_distill_workspace_bytes(int32_t R, int32_t C) { return 0; }

extern "C" int ttts_distill_fwd(const void* logits, int32_t dtype, int64_t ldl, const int64_t* teacher_idx, const float* teacher_logp,
                                float* row_loss, float* stats, int32_t R, int32_t C, int32_t K, float temperature, int32_t tail,
                                void* workspace, int64_t workspace_bytes, void* stream) {
  int rc = check_logits("distill_fwd", logits, dtype, ldl, R, C, temperature);
  if (rc) return rc;
  TTTS_REQUIRE(K > 0 && K <= TTTS_DISTILL_MAX_K, "distill_fwd: need 0 < K <= %d", TTTS_DISTILL_MAX_K);
  if (R == 0) return TTTS_OK;
  TTTS_REQUIRE(teacher_idx && teacher_logp && row_loss && stats, "distill_fwd: null pointer");
  TTTS_BY_TYPE(dtype, "distill_fwd",
               (distill_fwd_kernel<T><<<R, ROW_T, 0, as_stream(stream)>>>((const T*)logits, ldl, teacher_idx, teacher_logp, row_loss, stats, C, K,
                                                                         1.0f / temperature, tail)));
  return check_launch("distill_fwd");
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
  TTTS_BY_TYPE(dtype, "distill_bwd",
               (distill_bwd_kernel<T><<<R, ROW_T, 0, as_stream(stream)>>>((const T*)logits, ldl, teacher_idx, teacher_logp, stats, g_loss,
                                                                         (T*)dlogits, ldd, C, Cd, K, 1.0f / temperature, tail, accumulate)));
  return check_launch("distill_bwd");
}
