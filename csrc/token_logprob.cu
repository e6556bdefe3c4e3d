// Log-probabilities of given tokens, entropy and the top alternatives from materialised logits, with the gradient.
//
//   log p_rj = (x_rj - m_r) - log sum_j exp(x_rj - m_r),  m_r about max_j x_rj
//   lp[r] = log p_r,tgt  (0 where tgt < 0)      ent[r] = -sum_j p_rj log p_rj
//   the k largest x_rj in falling order, the lowest index first among equals, as log-probs and ids
// and, with incoming gradients g (log-prob), e (entropy) and u_i (alternatives with ids id_i),
//   dx_j = g [j = tgt] + sum_i u_i [j = id_i] - (g + sum_i u_i) p_j - e p_j (log p_j + ent).
// Everything is relative to about the row's maximum, also what the backward pass gets (m and log s, s the sum): a
// large common offset of the logits, up to rows of the type's lowest value, then cancels exactly.  With
// t = sum exp(x - m) (x - m) the entropy is log s - t / s.  Entries of -inf
// (masked vocabulary) have p = 0 and add nothing; a row of nothing else has log-probs -inf, entropy 0 and no gradient.
// A row with NaN or +inf gives NaN.
#include <cooperative_groups.h>
#include <cuda_fp16.h>
#include <type_traits>

#include "common.cuh"
#include "sm100.cuh"

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
RLB_DEVICE float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
RLB_DEVICE float fast_exp(float d) { return sm100::ex2_approx(d * 1.4426950408889634f); }

struct RowStats {
  float m, s, t;  // a reference no more than kSlack below the maximum, sum exp(x - m), sum exp(x - m) (x - m)
};
constexpr float kSlack = 8.f;

// Statistics relative to a new, not smaller maximum.
RLB_DEVICE void raise_to(RowStats& a, float m) {
  const float d = a.m - m, f = a.m == m ? 1.f : a.m == -INFINITY ? 0.f : fast_exp(d);
  a.t = f == 0.f ? 0.f : f * (a.t + d * a.s);
  if (a.m == m) return;
  a.s = f == 0.f && a.s == a.s ? 0.f : f * a.s;  // (NaN stays)
  a.m = m;
}

// Statistics of a warp's lanes as one, in every lane: one common reference, then plain sums.
RLB_DEVICE RowStats warp_stats(RowStats a) {
  const float m = warp_max(a.m);
  if (m != -INFINITY) raise_to(a, m);
  return RowStats{m, warp_sum(a.s), warp_sum(a.t)};
}

// VEC logits into the statistics; vm: their maximum, NaN if one is.
template <int VEC>
RLB_DEVICE void add_logits(RowStats& a, const float (&x)[VEC], float vm) {
  if (vm > a.m + kSlack) raise_to(a, vm);  // (rarely after the first logits: no new maximum costs a rescaling)
  const float m = a.m == -INFINITY ? 0.f : a.m;
  if constexpr (VEC % 2 == 0) {
    float2 s = make_float2(0.f, 0.f), t = s;
    const float2 mm = make_float2(-m, -m), l2e = make_float2(1.4426950408889634f, 1.4426950408889634f);
#pragma unroll
    for (int i = 0; i < VEC; i += 2) {
      float2 d = add2(make_float2(x[i], x[i + 1]), mm);
      const float2 y = mul2(d, l2e), e = make_float2(sm100::ex2_approx(y.x), sm100::ex2_approx(y.y));
      d.x = fmaxf(d.x, -1e30f);  // -inf: e is 0 and adds nothing
      d.y = fmaxf(d.y, -1e30f);
      s = add2(s, e);
      t = fma2(e, d, t);
    }
    a.s += s.x + s.y;
    a.t += t.x + t.y;
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const float d = x[i] - m, e = fast_exp(d);
      a.s += e;
      a.t = fmaf(e, fmaxf(d, -1e30f), a.t);
    }
  }
}

template <typename T>
RLB_DEVICE uint4 load16(const T* p) { return __ldcs(reinterpret_cast<const uint4*>(p)); }  // read once

template <typename T>
RLB_DEVICE void unpack16(const uint4& v, float* x) {
  const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
  for (int i = 0; i < (int)(16 / sizeof(T)); ++i) x[i] = to_f(e[i]);
}

template <typename T>
RLB_DEVICE void store16(T* p, const float (&x)[16 / sizeof(T)]) {
  uint4 v;
  T* e = reinterpret_cast<T*>(&v);
#pragma unroll
  for (int i = 0; i < (int)(16 / sizeof(T)); ++i) e[i] = from_f<T>(x[i]);
  __stcs(reinterpret_cast<uint4*>(p), v);
}

constexpr int kThreads = 256;
constexpr int kCtas = 1024 / kThreads;    // on an SM at a time
constexpr int kGroup = kThreads / 64;     // threads of each of 64 groups
constexpr int kHold = 160;                // candidates that may wait before the buffer is cut down, at most
constexpr int kEach = 16;                 // logits of a thread in a round
constexpr int kRound = kThreads * kEach;  // logits of a round, at most

// The k largest keys of buf[0, c), largest first, into out (zeros behind).  The whole block calls it; keys differ.
// Few candidates are ranked against each other, many are picked off one by one.
RLB_DEVICE void pick_top(const unsigned long long* buf, int c, int k, unsigned long long* out,
                         unsigned long long* scratch) {
  __syncthreads();
  for (int i = threadIdx.x; i < k; i += kThreads) out[i] = 0;
  __syncthreads();
  if (c <= 2 * kThreads) {
    // P neighbouring threads share a candidate's comparisons
    const int P = c <= 64 ? 8 : c <= 128 ? 4 : c <= 256 ? 2 : 1, part = threadIdx.x % P;
    for (int i0 = 0; i0 < c; i0 += kThreads / P) {
      const int i = i0 + threadIdx.x / P;
      const unsigned long long key = i < c ? buf[i] : ~0ull;
      int rank = 0;
#pragma unroll 8
      for (int j = part; j < c; j += P) rank += buf[j] > key;
      for (int o = 1; o < P; o <<= 1) rank += __shfl_xor_sync(0xffffffffu, rank, o);
      if (i < c && part == 0 && rank < k) out[rank] = key;
    }
  } else {
    unsigned long long below = ~0ull;
    for (int n = 0; n < k; ++n) {
      unsigned long long b = 0;
      for (int i = threadIdx.x; i < c; i += kThreads)
        if (buf[i] < below) b = max64(b, buf[i]);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) b = max64(b, __shfl_xor_sync(0xffffffffu, b, o));
      __syncthreads();
      if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = b;
      __syncthreads();
      b = scratch[0];
      for (int w = 1; w < kThreads / 32; ++w) b = max64(b, scratch[w]);
      below = b;
      if (threadIdx.x == 0) out[n] = b;
    }
  }
  __syncthreads();
}

struct TopShared {
  unsigned long long buf[kRound + kHold], out[kTopMost], scratch[kTopMost];
  int count;
};

// A cluster of CTAs takes a row, each a slice (one CTA where there are rows enough to fill the GPU).  One pass: online
// statistics per thread, and of the alternatives only those logits leave their registers that reach a bar known to
// have k logits at or above it: at first the k-th largest of the maxima of 64 groups of 4 threads, later the k-th
// largest candidate whenever more than 2 k + 32 of them wait (checked once a round of 4096 logits, by the barrier
// itself).  Rank 0 joins the slices over distributed shared memory.  Bound by the read of the logits and, close behind, by
// issue (exponential, sums and the bar's comparison of each): 2048 rows of 128256 in bf16 without alternatives 106 us,
// 5.0 TB/s; 1000 rows of 65536 in fp32 with 20 alternatives 70 us, 3.7 TB/s; 48 rows of 128256 with 5 in 16 us, mostly
// latency (a cluster's launch and barriers, the selection and its join).  A CTA has a whole row once rows fill the GPU, so
// a number of rows just above the 592 CTAs that fit at a time leaves the second wave half empty: 592 rows of 128256 in
// bf16 take 50 us, 700 take 63 and 1000 take 67 (each with the call's launch, which is 10 of them).
template <typename T, bool TOP>
__global__ void __launch_bounds__(kThreads, kCtas) token_logprob_kernel(
    const T* __restrict__ logits, long long ld, int V, const long long* __restrict__ tgt, int k,
    float* __restrict__ m_out, float* __restrict__ ls_out, float* __restrict__ lp_out, float* __restrict__ ent_out,
    float* __restrict__ top_lp, long long* __restrict__ top_ids, int* status) {
  constexpr int VEC = 16 / sizeof(T), U = kEach / VEC;
  extern __shared__ __align__(16) uint8_t dyn[];
  TopShared& top = *reinterpret_cast<TopShared*>(dyn);
  __shared__ RowStats red[kThreads / 32], mine;
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int slices = cluster.num_blocks(), slice = cluster.block_rank();
  const long long r = blockIdx.x / slices;
  const T* row = logits + r * ld;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int head = min(V, (int)((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / (int)sizeof(T));
  const int nvec = (V - head) / VEC;
  const int v0 = (int)((long long)nvec * slice / slices), v1 = (int)((long long)nvec * (slice + 1) / slices);
  RowStats st{-INFINITY, 0.f, 0.f};
  unsigned long long bar = 0;  // keys from here on are candidates
  float bar_x = -INFINITY;     // the bar's logit
  bool full = false;           // this thread saw more than `hold` candidates wait
  const int hold = 2 * k + 32;
  if (TOP) {
    if (tid == 0) top.count = 0;
    __syncthreads();
  }
  auto offer = [&](float x, int j) {
    const unsigned long long key = rank_key(x, j);
    if (key >= bar) {
      const int at = atomicAdd(&top.count, 1);
      top.buf[at] = key;
      full |= at >= hold;
    }
  };
  auto set_bar = [&](unsigned long long key) {
    bar = key;
    const uint32_t u = (uint32_t)(key >> 32);
    bar_x = key == 0 ? -INFINITY : __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
  };
  // the row's unaligned ends, by single threads of the first and the last slice
  auto ends = [&](int j) {
    const float x[1] = {to_f(row[j])};
    add_logits<1>(st, x, x[0]);
    if (TOP) offer(x[0], j);
  };
  const uint4 absent = sizeof(T) == 4 ? make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u)  // -inf
                       : std::is_same<T, __half>::value ? make_uint4(0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u)
                                                        : make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u);
  const T* data = row + head;
  uint4 next[U];
  auto fetch = [&](int base) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int v = base + u * kThreads + tid;
      next[u] = v < v1 ? load16(data + (long long)v * VEC) : absent;
    }
  };
  fetch(v0);
  for (int base = v0; base < v1; base += U * kThreads) {
    float x[U * VEC];
#pragma unroll
    for (int u = 0; u < U; ++u) unpack16<T>(next[u], x + u * VEC);
    if (base + U * kThreads < v1) fetch(base + U * kThreads);
    float vec_max[U], vm;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      vec_max[u] = x[u * VEC];
#pragma unroll
      for (int i = 1; i < VEC; ++i) vec_max[u] = max_nan(vec_max[u], x[u * VEC + i]);
      vm = u == 0 ? vec_max[0] : max_nan(vm, vec_max[u]);
    }
    add_logits<U * VEC>(st, x, vm);
    if (TOP) {
      const int j0 = head + (base + tid) * VEC;  // vector u begins u * kThreads * VEC behind
      if (base == v0) {
        // (a key no larger than the maximum's: the last place that this thread could have it at)
        const bool has = base + tid < v1;
        unsigned long long best = has ? rank_key(vm, V - 1) : 0;
#pragma unroll
        for (int o = 1; o < kGroup; o <<= 1) best = max64(best, __shfl_xor_sync(0xffffffffu, best, o));
        if (tid % kGroup == 0) top.scratch[tid / kGroup] = best;
        __syncthreads();
        // the k-th largest of the 64 (absent groups: 0, so that fewer than k groups leave no bar)
        const int at = tid / kGroup;
        const unsigned long long key = top.scratch[at];
        int rank = 0;
#pragma unroll
        for (int i = tid % kGroup; i < 64; i += kGroup) rank += top.scratch[i] > key || (top.scratch[i] == key && i < at);
#pragma unroll
        for (int o = 1; o < kGroup; o <<= 1) rank += __shfl_xor_sync(0xffffffffu, rank, o);
        if (rank == k - 1 && tid % kGroup == 0) top.out[0] = key;
        __syncthreads();
        set_bar(top.out[0]);
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (!(vec_max[u] < bar_x) && base + u * kThreads + tid < v1)
#pragma unroll
          for (int i = 0; i < VEC; ++i)
            if (!(x[u * VEC + i] < bar_x)) offer(x[u * VEC + i], j0 + u * kThreads * VEC + i);
      if (__syncthreads_or(full)) {
        const int c = top.count;
        pick_top(top.buf, c, k, top.out, top.scratch);
        if (tid < k) top.buf[tid] = top.out[tid];
        if (tid == 0) top.count = k;  // (more than k candidates waited)
        set_bar(top.out[k - 1]);
        full = false;
        __syncthreads();
      }
    }
  }
  if (slice == 0 && tid < head) ends(tid);
  if (slice == slices - 1 && tid < V - head - nvec * VEC) ends(head + nvec * VEC + tid);
  st = warp_stats(st);
  if (lane == 0) red[warp] = st;
  __syncthreads();
  if (warp == 0) {
    st = warp_stats(lane < kThreads / 32 ? red[lane] : RowStats{-INFINITY, 0.f, 0.f});
    if (lane == 0) mine = st;
  }
  if (TOP) pick_top(top.buf, top.count, k, top.out, top.scratch);
  if (slices > 1) {
    cluster.sync();
    if (slice == 0) {
      if (TOP) {
        for (int i = tid; i < slices * k; i += kThreads) top.buf[i] = cluster.map_shared_rank(&top, i / k)->out[i % k];
        pick_top(top.buf, slices * k, k, top.out, top.scratch);  // (zeros stand for nothing and rank last)
      }
      if (warp == 0) {
        st = warp_stats(lane < slices ? *cluster.map_shared_rank(&mine, lane) : RowStats{-INFINITY, 0.f, 0.f});
        __syncwarp();
        if (lane == 0) mine = st;
      }
    }
    cluster.sync();  // the others' shared memory is still read until here
    if (slice != 0) return;
  }
  __syncthreads();
  st = mine;
  const bool none = st.m == -INFINITY && st.s == 0.f;
  const float ls = logf(st.s);
  if (tid == 0) {
    const long long tg = tgt[r];
    float lp = 0.f;
    if (tg >= V) report(status, kBadIndex);
    else if (tg >= 0) lp = none ? -INFINITY : to_f(row[tg]) - st.m - ls;
    if (m_out != nullptr) {
      m_out[r] = st.m;
      ls_out[r] = ls;
    }
    lp_out[r] = lp;
    ent_out[r] = none ? 0.f : ls - st.t / st.s;
  }
  if (TOP && tid < k) {
    const int j = (int)~(uint32_t)top.out[tid];
    top_ids[r * k + tid] = j;
    top_lp[r * k + tid] = none ? -INFINITY : to_f(row[j]) - st.m - ls;
  }
}

// One CTA per stretch of a row.  Bound by the read of the logits and the write of their gradient: 2048 rows of 128256 in
// bf16 (1.05 GB) in 166 us, 6.3 TB/s.  Where a row and its gradient are not aligned alike (a slice of a padded vocabulary),
// entry by entry: 4096 rows of 50257 in bf16 in 418 us, against 188 as rows of their own; in fp32 455 against 321.
constexpr int kBwdThreads = 256;
constexpr int kBwdStretch = kBwdThreads * 8 * 8;  // logits

template <typename T>
__global__ void __launch_bounds__(kBwdThreads) token_logprob_bwd_kernel(
    const T* __restrict__ logits, long long ld, int V, int stretches, const long long* __restrict__ tgt,
    const float* __restrict__ row_m, const float* __restrict__ row_ls, const float* __restrict__ ent,
    const long long* __restrict__ top_ids, int k, const float* __restrict__ g_lp, const float* __restrict__ g_ent,
    const float* __restrict__ g_top, T* __restrict__ dx) {
  constexpr int VEC = 16 / sizeof(T);
  const long long r = blockIdx.x / stretches;
  const int j0 = (int)(blockIdx.x % stretches) * kBwdStretch, j1 = (int)min((long long)V, (long long)j0 + kBwdStretch);
  const T* row = logits + r * ld;
  T* out = dx + r * V;
  const float m = row_m[r], ls = row_ls[r], H = ent[r];
  const long long tg = tgt[r];
  const bool has = tg >= 0 && tg < V;
  const float g = g_lp && has ? g_lp[r] : 0.f, e = g_ent ? g_ent[r] : 0.f;
  float a = g;
  if (g_top)
    for (int i = 0; i < k; ++i) a += g_top[r * k + i];
  const float c0 = -(a + e * H), c1 = -e;
  auto grad = [&](float x) {
    // p is 0 from log p < -104 on: the bound keeps 0 times -inf out (a row of NaN stays NaN by its entropy)
    const float logp = fmaxf((x - m) - ls, -200.f);
    return fast_exp(logp) * fmaf(c1, logp, c0);
  };
  // whole vectors where the row and its gradient are aligned alike, single entries at the ends (or everywhere)
  const bool alike = ((reinterpret_cast<uintptr_t>(row) ^ reinterpret_cast<uintptr_t>(out)) & 15) == 0;
  const int lead = (int)((16 - (reinterpret_cast<uintptr_t>(row + j0) & 15)) & 15) / (int)sizeof(T);
  const int w0 = alike ? min(j1, j0 + lead) : j1, nvec = (j1 - w0) / VEC;
#pragma unroll 2
  for (int v = threadIdx.x; v < nvec; v += kBwdThreads) {
    float x[VEC];
    unpack16<T>(load16(row + w0 + v * VEC), x);
#pragma unroll
    for (int i = 0; i < VEC; i += 2) {  // grad(), for two
      float2 d = add2(add2(make_float2(x[i], x[i + 1]), make_float2(-m, -m)), make_float2(-ls, -ls));
      d = make_float2(fmaxf(d.x, -200.f), fmaxf(d.y, -200.f));
      const float2 y = mul2(d, make_float2(1.4426950408889634f, 1.4426950408889634f));
      const float2 g2 = mul2(make_float2(sm100::ex2_approx(y.x), sm100::ex2_approx(y.y)),
                             fma2(make_float2(c1, c1), d, make_float2(c0, c0)));
      x[i] = g2.x;
      x[i + 1] = g2.y;
    }
    store16(out + w0 + v * VEC, x);
  }
  for (int j = j0 + threadIdx.x; j < w0; j += kBwdThreads) out[j] = from_f<T>(grad(to_f(row[j])));
  for (int j = w0 + nvec * VEC + threadIdx.x; j < j1; j += kBwdThreads) out[j] = from_f<T>(grad(to_f(row[j])));
  __syncthreads();
  if (m == -INFINITY) return;
  // the target's and the alternatives' entries of this stretch again, with their own terms, rounded once
  for (int i = (int)threadIdx.x - 1; i < (g_top ? k : 0); i += kBwdThreads) {
    if (i < 0 && !has) continue;
    const long long j = i < 0 ? tg : top_ids[r * k + i];
    if (j < j0 || j >= j1) continue;
    float d = grad(to_f(row[j])) + (has && j == tg ? g : 0.f);
    if (g_top)
      for (int u = 0; u < k; ++u) d += top_ids[r * k + u] == j ? g_top[r * k + u] : 0.f;
    out[j] = from_f<T>(d);
  }
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

template <typename T, bool TOP>
static cudaError_t token_logprob_launch(const void* logits, long long ld, long long rows, int V, const long long* tgt,
                                        int k, float* m, float* ls, float* lp, float* ent, float* top_lp,
                                        long long* top_ids, int sms, int* status, cudaStream_t s) {
  // Slices: two as long as the CTAs fit on the GPU at a time, four and eight while three CTAs an SM hold them, and a slice
  // keeps a round of logits.  (Rows of 128256 in bf16 with 5 alternatives, in us, by 1, 2, 4 and 8 slices: 1 row
  // 33, 25, 18, 16; 48 rows 35, 27, 23, 21; 74 rows 37, 27, 25, 29; 148 rows 37, 29, 37, 39; 296 rows 41, 37, 53, 64;
  // 400 rows 45, 53, 62, 82.)
  int slices = 1;
  while (slices < 8 && rows * slices * 2 <= (slices == 1 ? kCtas : 3LL) * sms && V / (slices * 2) >= kRound) slices *= 2;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = slices;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows * slices));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = TOP ? sizeof(TopShared) : 0;
  cfg.stream = s;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  if (TOP) {
    const cudaError_t e = cudaFuncSetAttribute(token_logprob_kernel<T, TOP>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               (int)sizeof(TopShared));
    if (e != cudaSuccess) return e;
  }
  return cudaLaunchKernelEx(&cfg, token_logprob_kernel<T, TOP>, (const T*)logits, ld, V, tgt, k, m, ls, lp, ent, top_lp,
                            top_ids, status);
}

cudaError_t rlb_token_logprob(const void* logits, int dtype, long long ld, long long rows, int V, const long long* tgt,
                              int k, float* m, float* ls, float* lp, float* ent, float* top_lp, long long* top_ids,
                              int sms, int* status, cudaStream_t s) {
  if (rows == 0) return cudaSuccess;
  if (k > kTopMost || rows > (1LL << 31) - 1) return cudaErrorInvalidValue;
  cudaError_t e = cudaSuccess;
  RLB_LOGIT_TYPE((e = k > 0 ? token_logprob_launch<T, true>(logits, ld, rows, V, tgt, k, m, ls, lp, ent, top_lp, top_ids,
                                                            sms, status, s)
                            : token_logprob_launch<T, false>(logits, ld, rows, V, tgt, k, m, ls, lp, ent, top_lp,
                                                             top_ids, sms, status, s)));
  return e;
}

cudaError_t rlb_token_logprob_bwd(const void* logits, int dtype, long long ld, long long rows, int V,
                                  const long long* tgt, const float* m, const float* ls, const float* ent,
                                  const long long* top_ids, int k, const float* g_lp, const float* g_ent,
                                  const float* g_top, void* dx, cudaStream_t s) {
  if (rows == 0) return cudaSuccess;
  const long long stretches = ((long long)V + kBwdStretch - 1) / kBwdStretch;
  if (rows * stretches > (1LL << 31) - 1) return cudaErrorInvalidValue;
  RLB_LOGIT_TYPE((token_logprob_bwd_kernel<T><<<(unsigned)(rows * stretches), kBwdThreads, 0, s>>>(
      (const T*)logits, ld, V, (int)stretches, tgt, m, ls, ent, top_ids, k, g_lp, g_ent, g_top, (T*)dx)));
  return cudaGetLastError();
}
