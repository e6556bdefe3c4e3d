// Log-probabilities of given tokens, entropy and the top alternatives from materialised logits, with the gradient.
//
//   log p_rj = (x_rj - m_r) - log sum_j exp(x_rj - m_r),  m_r = max_j x_rj
//   lp[r] = log p_r,tgt  (0 where tgt < 0)      ent[r] = -sum_j p_rj log p_rj
//   the k largest x_rj in falling order, the lowest index first among equals, as log-probs and ids
// and, with incoming gradients g (log-prob), e (entropy) and u_i (alternatives with ids id_i),
//   dx_j = g [j = tgt] + sum_i u_i [j = id_i] - (g + sum_i u_i) p_j - e p_j (log p_j + ent).
// Everything is relative to the row's maximum, also what the backward pass gets (m and log s, with s the sum): a
// large common offset of the logits, up to rows of the type's lowest value, then cancels exactly.  With
// t = sum exp(x - m) (x - m) the entropy is log s - t / s.  Entries of -inf
// (masked vocabulary) have p = 0 and add nothing; a row of nothing else has log-probs -inf, entropy 0 and no gradient.
// A row with NaN or +inf gives NaN.
#include <cuda_fp16.h>

#include "common.cuh"

namespace rlb {

constexpr int kTopMost = 64;  // alternatives per row

RLB_DEVICE float to_f(float x) { return x; }
RLB_DEVICE float to_f(__half x) { return __half2float(x); }
RLB_DEVICE float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> RLB_DEVICE T from_f(float x);
template <> RLB_DEVICE float from_f<float>(float x) { return x; }
template <> RLB_DEVICE __half from_f<__half>(float x) { return __float2half(x); }
template <> RLB_DEVICE __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16(x); }

// A logit and its index as one number: larger for larger logits, for the lower index among equals; NaN on top.
RLB_DEVICE unsigned long long rank_key(float x, int j) {
  const uint32_t u = __float_as_uint(x + 0.f);
  const uint32_t k = x != x ? 0xffffffffu : (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return ((unsigned long long)k << 32) | (uint32_t)~j;
}

RLB_DEVICE unsigned long long max64(unsigned long long a, unsigned long long b) { return a > b ? a : b; }

struct RowStats {
  float m, s, t;  // maximum, sum exp(x - m), sum exp(x - m) (x - m)
};

RLB_DEVICE RowStats merge(RowStats a, RowStats b) {
  const float m = fmaxf(a.m, b.m);
  if (m == -INFINITY) return RowStats{m, a.s + b.s, a.t + b.t};  // nothing yet (or NaN in the sums)
  const float da = a.m - m, db = b.m - m;
  const float fa = expf(da), fb = expf(db);
  return RowStats{m, a.s * fa + b.s * fb,
                  (fa == 0.f ? 0.f : fa * (a.t + da * a.s)) + (fb == 0.f ? 0.f : fb * (b.t + db * b.s))};
}

RLB_DEVICE RowStats single(float x) {
  return x == -INFINITY ? RowStats{-INFINITY, 0.f, 0.f} : RowStats{x, x - x + 1.f, 0.f};  // NaN and +inf: NaN
}

template <typename T>
__global__ void __launch_bounds__(512) token_logprob_kernel(const T* __restrict__ logits, long long ld, int V,
                                                            const long long* __restrict__ tgt, int k,
                                                            float* __restrict__ m_out, float* __restrict__ ls_out,
                                                            float* __restrict__ lp_out,
                                                            float* __restrict__ ent_out, float* __restrict__ top_lp,
                                                            long long* __restrict__ top_ids, int* status) {
  __shared__ RowStats red[16];
  __shared__ unsigned long long best[16];
  const long long r = blockIdx.x;
  const T* row = logits + r * ld;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  RowStats st{-INFINITY, 0.f, 0.f};
  for (int j = threadIdx.x; j < V; j += 512) st = merge(st, single(to_f(row[j])));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    st = merge(st, RowStats{__shfl_xor_sync(0xffffffffu, st.m, o), __shfl_xor_sync(0xffffffffu, st.s, o),
                            __shfl_xor_sync(0xffffffffu, st.t, o)});
  if (lane == 0) red[warp] = st;
  __syncthreads();
  st = red[0];
  for (int w = 1; w < 16; ++w) st = merge(st, red[w]);
  const bool none = st.m == -INFINITY && st.s == 0.f;
  const float ls = logf(st.s);
  if (threadIdx.x == 0) {
    const long long tg = tgt[r];
    float lp = 0.f;
    if (tg >= V) report(status, kBadIndex);
    else if (tg >= 0) lp = none ? -INFINITY : to_f(row[tg]) - st.m - ls;
    m_out[r] = st.m;
    ls_out[r] = ls;
    lp_out[r] = lp;
    ent_out[r] = none ? 0.f : ls - st.t / st.s;
  }
  unsigned long long below = ~0ull;  // the last one found; the next is the largest key under it
  for (int i = 0; i < k; ++i) {
    unsigned long long b = 0;
    for (int j = threadIdx.x; j < V; j += 512) {
      const unsigned long long key = rank_key(to_f(row[j]), j);
      if (key < below) b = max64(b, key);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) b = max64(b, __shfl_xor_sync(0xffffffffu, b, o));
    __syncthreads();
    if (lane == 0) best[warp] = b;
    __syncthreads();
    b = best[0];
    for (int w = 1; w < 16; ++w) b = max64(b, best[w]);
    below = b;
    if (threadIdx.x == 0) {
      const int j = (int)~(uint32_t)b;
      top_ids[r * k + i] = j;
      top_lp[r * k + i] = none ? -INFINITY : to_f(row[j]) - st.m - ls;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(512) token_logprob_bwd_kernel(
    const T* __restrict__ logits, long long ld, int V, const long long* __restrict__ tgt,
    const float* __restrict__ row_m, const float* __restrict__ row_ls, const float* __restrict__ ent, const long long* __restrict__ top_ids, int k,
    const float* __restrict__ g_lp, const float* __restrict__ g_ent, const float* __restrict__ g_top,
    T* __restrict__ dx) {
  const long long r = blockIdx.x;
  const T* row = logits + r * ld;
  T* out = dx + r * V;
  const float m = row_m[r], ls = row_ls[r];
  const long long tg = tgt[r];
  const bool has = tg >= 0 && tg < V;
  const float g = g_lp && has ? g_lp[r] : 0.f, e = g_ent ? g_ent[r] : 0.f, H = ent[r];
  float a = g;
  if (g_top)
    for (int i = 0; i < k; ++i) a += g_top[r * k + i];
  auto grad = [&](float x) {
    const float logp = (x - m) - ls;
    const float p = expf(logp);
    return p == 0.f || m == -INFINITY ? 0.f : -p * (a + e * (logp + H));
  };
  for (int j = threadIdx.x; j < V; j += 512) out[j] = from_f<T>(grad(to_f(row[j])));
  __syncthreads();
  if (m == -INFINITY) return;
  // the target's and the alternatives' entries again, with their own terms, rounded once
  const int i = threadIdx.x - 1;
  if (i >= (g_top ? k : 0) || (i < 0 && !has)) return;
  const long long j = i < 0 ? tg : top_ids[r * k + i];
  float d = grad(to_f(row[j])) + (has && j == tg ? g : 0.f);
  if (g_top)
    for (int u = 0; u < k; ++u) d += top_ids[r * k + u] == j ? g_top[r * k + u] : 0.f;
  out[j] = from_f<T>(d);
}

}  // namespace rlb

using namespace rlb;

#define RLB_LOGIT_TYPE(call)                                       \
  do {                                                             \
    if (dtype == 0) { using T = float; call; }                     \
    else if (dtype == 1) { using T = __nv_bfloat16; call; }        \
    else if (dtype == 2) { using T = __half; call; }               \
    else return cudaErrorNotSupported;                             \
  } while (0)

cudaError_t rlb_token_logprob(const void* logits, int dtype, long long ld, long long rows, int V, const long long* tgt,
                              int k, float* m, float* ls, float* lp, float* ent, float* top_lp, long long* top_ids, int* status,
                              cudaStream_t s) {
  if (rows == 0) return cudaSuccess;
  if (k > kTopMost) return cudaErrorInvalidValue;
  RLB_LOGIT_TYPE((token_logprob_kernel<T><<<(unsigned)rows, 512, 0, s>>>((const T*)logits, ld, V, tgt, k, m, ls, lp, ent,
                                                                         top_lp, top_ids, status)));
  return cudaGetLastError();
}

cudaError_t rlb_token_logprob_bwd(const void* logits, int dtype, long long ld, long long rows, int V,
                                  const long long* tgt, const float* m, const float* ls, const float* ent,
                                  const long long* top_ids,
                                  int k, const float* g_lp, const float* g_ent, const float* g_top, void* dx,
                                  cudaStream_t s) {
  if (rows == 0) return cudaSuccess;
  RLB_LOGIT_TYPE((token_logprob_bwd_kernel<T><<<(unsigned)rows, 512, 0, s>>>(
      (const T*)logits, ld, V, tgt, m, ls, ent, top_ids, k, g_lp, g_ent, g_top, (T*)dx)));
  return cudaGetLastError();
}
