// Paged KV cache held in 4 bits: storing and reading rows, decode attention over it, eviction.
//
// Pool layout (k_pool and v_pool alike): uint8 [num_blocks][Hkv][block bytes], a block being 16 tokens of one KV
// head.  With groups of g = min(D, 64) dimensions a block holds, for each group, the codes [16][g / 2] (element 2i
// in the low half of byte i) and behind all codes, for each group, [16] pairs (scale, minimum) in bf16.  An element
// stands for minimum + scale * code, with
//   minimum = min x,  scale = bf16((max x - min x) / 15),  code = clamp(rint((x - minimum) / scale), 0, 15)
// over the group: the inputs are bf16, so the minimum is exact, and the codes are chosen against the rounded scale.
// Group-major codes keep the 16 tokens x 64 dimensions that a matrix instruction works on contiguous (512 bytes).
#include "common.cuh"

namespace rlb {

constexpr int kTok = 16;  // tokens per block

template <int D>
struct Q4 {
  static constexpr int kGroup = D < 64 ? D : 64;
  static constexpr int kGroups = D / kGroup;
  static constexpr int kRow = kGroup / 2;                     // code bytes of one token in one group
  static constexpr int kCodes = kTok * D / 2;                 // code bytes of a block
  static constexpr int kBytes = kCodes + kTok * kGroups * 4;  // bytes of a block
  static constexpr int kLanes = kGroup / 8;                   // threads that share a group, 8 elements each
};

RLB_DEVICE float bf16_lo_f(uint32_t v) { return __uint_as_float(v << 16); }
RLB_DEVICE float bf16_hi_f(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }

// ---------------------------------------------------------------- storing rows
// A group's threads reduce its minimum and maximum by shuffles (NaN-propagating), then each quantises its 8
// elements to one 32-bit word.  Bound by memory: 2 bytes read and about 0.56 written per element.
template <int D>
__global__ void __launch_bounds__(256) q4_write_kernel(
    const __nv_bfloat16* __restrict__ k_new, const __nv_bfloat16* __restrict__ v_new, long long k_sn, long long k_sh,
    long long v_sn, long long v_sh, uint8_t* __restrict__ k_pool, uint8_t* __restrict__ v_pool,
    const int* __restrict__ slot_block, const int* __restrict__ slot_off, long long N, int Hkv, int num_blocks,
    int* status) {
  using L = Q4<D>;
  const bool is_v = blockIdx.y != 0;
  const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  const int lane = (int)(i % L::kLanes);
  const long long team = i / L::kLanes;
  const int grp = (int)(team % L::kGroups);
  const int h = (int)(team / L::kGroups % Hkv);
  const long long n = team / L::kGroups / Hkv;
  if (n >= N) return;  // whole teams leave together: kLanes divides the block
  const int blk = slot_block[n], off = slot_off[n];
  if (blk < 0 || blk >= num_blocks || off < 0 || off >= kTok) {
    if (lane == 0) report(status, kBadIndex);
    return;
  }
  const __nv_bfloat16* src = is_v ? v_new + n * v_sn + h * v_sh : k_new + n * k_sn + h * k_sh;
  const bf16x8 x = ldg8(src + grp * L::kGroup + lane * 8);
  __nv_bfloat162 mn = __hmin2_nan(__hmin2_nan(x.h[0], x.h[1]), __hmin2_nan(x.h[2], x.h[3]));
  __nv_bfloat162 mx = __hmax2_nan(__hmax2_nan(x.h[0], x.h[1]), __hmax2_nan(x.h[2], x.h[3]));
  const unsigned mask = (L::kLanes == 32 ? 0xffffffffu : ((1u << L::kLanes) - 1)) << (threadIdx.x & 31 & ~(L::kLanes - 1));
#pragma unroll
  for (int o = 1; o < L::kLanes; o <<= 1) {
    mn = __hmin2_nan(mn, __shfl_xor_sync(mask, mn, o));
    mx = __hmax2_nan(mx, __shfl_xor_sync(mask, mx, o));
  }
  const __nv_bfloat16 lo = __hmin_nan(mn.x, mn.y);
  const float lof = __bfloat162float(lo);
  const __nv_bfloat16 scale = __float2bfloat16(__fdiv_rn(__bfloat162float(__hmax_nan(mx.x, mx.y)) - lof, 15.f));
  const float sf = __bfloat162float(scale);
  float f[8];
  unpack8(x, f);
  uint32_t word = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float c = rintf(__fdiv_rn(f[e] - lof, sf));
    const float cl = fminf(fmaxf(c, 0.f), 15.f);  // NaN (a group without spread, or not finite) becomes 0
    word |= (uint32_t)cl << (4 * e);
  }
  uint8_t* dst = (is_v ? v_pool : k_pool) + ((long long)blk * Hkv + h) * L::kBytes;
  *reinterpret_cast<uint32_t*>(dst + (grp * kTok + off) * L::kRow + lane * 4) = word;
  if (lane == 0)
    *reinterpret_cast<uint32_t*>(dst + L::kCodes + (grp * kTok + off) * 4) =
        (uint32_t)__bfloat16_as_ushort(scale) | ((uint32_t)__bfloat16_as_ushort(lo) << 16);
}

// ---------------------------------------------------------------- reading rows
// One thread per 8 elements.  Row r is slot (slot_block[r], slot_off[r]), or, with a block table, position
// r % max_len of sequence r / max_len.  Rows without a place in the pool read as zeros.
template <int D>
__global__ void __launch_bounds__(256) q4_read_kernel(const uint8_t* __restrict__ k_pool,
                                                      const uint8_t* __restrict__ v_pool,
                                                      const int* __restrict__ slot_block,
                                                      const int* __restrict__ slot_off, const int* __restrict__ tables,
                                                      const int* __restrict__ lens, int max_blocks, int max_len,
                                                      long long N, int Hkv, int num_blocks,
                                                      __nv_bfloat16* __restrict__ k_out,
                                                      __nv_bfloat16* __restrict__ v_out, int* status) {
  using L = Q4<D>;
  const bool is_v = blockIdx.y != 0;
  const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  const int d8 = (int)(i % (D / 8));
  const int h = (int)(i / (D / 8) % Hkv);
  const long long n = i / (D / 8) / Hkv;
  if (n >= N) return;
  int blk = -1, off = 0;
  bool absent = false;
  if (tables == nullptr) {
    blk = slot_block[n];
    off = slot_off[n];
  } else {
    const long long b = n / max_len;
    const int pos = (int)(n % max_len);
    off = pos % kTok;
    absent = pos >= lens[b];
    if (!absent && pos / kTok < max_blocks) blk = tables[b * max_blocks + pos / kTok];
  }
  float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (!absent) {
    if (blk < 0 || blk >= num_blocks || off < 0 || off >= kTok) {
      if (d8 == 0 && h == 0) report(status, kBadIndex);
    } else {
      const uint8_t* src = (is_v ? v_pool : k_pool) + ((long long)blk * Hkv + h) * L::kBytes;
      const int grp = d8 * 8 / L::kGroup, lane = d8 % L::kLanes;
      const uint32_t word = *reinterpret_cast<const uint32_t*>(src + (grp * kTok + off) * L::kRow + lane * 4);
      const uint32_t meta = *reinterpret_cast<const uint32_t*>(src + L::kCodes + (grp * kTok + off) * 4);
      const float s = bf16_lo_f(meta), lo = bf16_hi_f(meta);
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = fmaf((float)((word >> (4 * e)) & 15u), s, lo);
    }
  }
  stg8((is_v ? v_out : k_out) + (n * Hkv + h) * D + d8 * 8, pack8(f));
}

// ---------------------------------------------------------------- decode attention
struct Q4Cache {
  const uint8_t *k_pool, *v_pool;
  const int *tables, *lens;
  int Hkv, G, max_blocks, num_blocks, window;
  float scale, softcap;
};

// A lane's D / 32 dimensions of a stored row; false where the token's block is not in the pool.
template <int D>
RLB_DEVICE bool q4_row(const Q4Cache& c, const uint8_t* pool, int b, int h, int t, float* f) {
  using L = Q4<D>;
  constexpr int E = D / 32;
  const int lane = threadIdx.x & 31, grp = lane * E / L::kGroup, in_grp = lane * E % L::kGroup;
  const int blk = c.tables[(long long)b * c.max_blocks + t / kTok], off = t % kTok;
  if (blk < 0 || blk >= c.num_blocks) return false;
  const uint8_t* src = pool + ((long long)blk * c.Hkv + h) * L::kBytes;
  const uint32_t meta = *reinterpret_cast<const uint32_t*>(src + L::kCodes + (grp * kTok + off) * 4);
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int byte = src[(grp * kTok + off) * L::kRow + (in_grp + e) / 2];
    f[e] = fmaf((float)(((in_grp + e) & 1) ? byte >> 4 : byte & 15), bf16_lo_f(meta), bf16_hi_f(meta));
  }
  return true;
}

template <int D>
RLB_DEVICE float q4_score(const Q4Cache& c, int b, int h, int t, const float* qf) {
  float f[D / 32], s = 0.f;
  if (!q4_row<D>(c, c.k_pool, b, h, t, f)) return -INFINITY;
#pragma unroll
  for (int e = 0; e < D / 32; ++e) s += qf[e] * f[e];
  s = warp_sum(s) * c.scale;
  return c.softcap > 0.f ? tanhf(s / c.softcap) * c.softcap : s;
}

// One CTA per (query head, sequence); each warp takes every fourth token, a lane D / 32 dimensions of it.  `ml`
// (optional, [B][Hq][2]) receives the softmax's maximum and sum.
template <int D>
__global__ void __launch_bounds__(128) q4_decode_kernel(const __nv_bfloat16* __restrict__ q, Q4Cache c,
                                                        __nv_bfloat16* __restrict__ out, float* __restrict__ ml,
                                                        int* status) {
  constexpr int E = D / 32;
  const int hq = blockIdx.x, b = blockIdx.y, h = hq / c.G;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long row = (long long)b * c.Hkv * c.G + hq;
  int len = c.lens[b];
  if (len > c.max_blocks * kTok) {
    report(status, kBadIndex);
    len = c.max_blocks * kTok;
  }
  const int t0 = c.window > 0 && len > c.window ? len - c.window : 0;
  float qf[E];
#pragma unroll
  for (int e = 0; e < E; ++e) qf[e] = __bfloat162float(q[row * D + lane * E + e]);
  float m = -INFINITY, l = 0.f, acc[E] = {};
  for (int t = t0 + warp; t < len; t += 4) {
    const float s = q4_score<D>(c, b, h, t, qf);
    float f[E];
    if (!q4_row<D>(c, c.v_pool, b, h, t, f)) {
      report(status, kBadIndex);
      continue;
    }
    const float mn = fmaxf(m, s), cr = expf(m - mn), p = expf(s - mn);
    l = l * cr + p;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = acc[e] * cr + p * f[e];
    m = mn;
  }
  __shared__ float sm[4], sl[4], sa[4][D];
  if (lane == 0) {
    sm[warp] = m;
    sl[warp] = l;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) sa[warp][lane * E + e] = acc[e];
  __syncthreads();
  const float M = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
  float Lsum = 0.f, cr[4];
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    cr[w] = sm[w] == -INFINITY ? 0.f : expf(sm[w] - M);
    Lsum += sl[w] * cr[w];
  }
  for (int d = threadIdx.x; d < D; d += 128) {
    float a = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) a += sa[w][d] * cr[w];
    out[row * D + d] = __float2bfloat16(Lsum != 0.f ? a / Lsum : 0.f);
  }
  if (ml != nullptr && threadIdx.x == 0) {
    ml[row * 2] = M;
    ml[row * 2 + 1] = Lsum;
  }
}

// Adds each token's attention weight, summed over its KV head's query heads, to its accumulator.
template <int D>
__global__ void __launch_bounds__(128) q4_weights_kernel(const __nv_bfloat16* __restrict__ q, Q4Cache c,
                                                         const float* __restrict__ ml, float* __restrict__ weights,
                                                         const int* __restrict__ weight_rows, long long w_rows,
                                                         int w_len, int* status) {
  constexpr int E = D / 32;
  const int h = blockIdx.x, b = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r = weight_rows[b], len = min(c.lens[b], c.max_blocks * kTok);
  if (len <= 0 || r < 0) return;
  if (r >= w_rows || len > w_len) report(status, kBadIndex);
  if (r >= w_rows) return;
  const int t0 = c.window > 0 && len > c.window ? len - c.window : 0;
  for (int t = t0 + warp; t < min(len, w_len); t += 4) {
    float p = 0.f;
    for (int g = 0; g < c.G; ++g) {
      const long long row = ((long long)b * c.Hkv + h) * c.G + g;
      float qf[E];
#pragma unroll
      for (int e = 0; e < E; ++e) qf[e] = __bfloat162float(q[row * D + lane * E + e]);
      p += expf(q4_score<D>(c, b, h, t, qf) - ml[row * 2]) / ml[row * 2 + 1];
    }
    if (lane == 0 && p > 0.f) atomicAdd(weights + ((long long)r * c.Hkv + h) * w_len + t, p);
  }
}

// ---------------------------------------------------------------- eviction
// Order-preserving key of a weight: larger keys for larger weights, -0 like +0, NaN below everything.
RLB_DEVICE uint32_t weight_key(float w) {
  if (w != w) return 0u;
  const uint32_t u = __float_as_uint(w + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// Exclusive prefix sum of one flag per thread over a 1024-thread block (`scratch`: 33 ints), and the total.
RLB_DEVICE int block_rank(bool flag, int* scratch, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const unsigned vote = __ballot_sync(0xffffffffu, flag);
  __syncthreads();
  if (lane == 0) scratch[warp] = __popc(vote);
  __syncthreads();
  if (warp == 0) {
    const int c = scratch[lane];
    int s = c;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += y;
    }
    scratch[lane] = s - c;
    if (lane == 31) scratch[32] = s;
  }
  __syncthreads();
  total = scratch[32];
  return scratch[warp] + __popc(vote & ((1u << lane) - 1));
}

// One CTA per (KV head, sequence): finds the weight of the last kept token by a radix selection over 8-bit digits,
// then walks the tokens in order, writing the kept ones' positions and moving their weights to the front.  Moving
// in place is safe because a token never moves backwards past one that is still to be read: a tile's weights are
// all read before any of it is written.
__global__ void __launch_bounds__(1024) q4_select_kernel(const int* __restrict__ lens, float* __restrict__ weights,
                                                         const int* __restrict__ weight_rows, int* __restrict__ kept,
                                                         int* __restrict__ new_lens, int Hkv, long long w_rows,
                                                         int w_len, int keep, int recent, int sink, int* status) {
  __shared__ int hist[256], scratch[33], pick[2];
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  int n = lens[b];
  const int r = weight_rows[b];
  if (n > w_len || (n > 0 && (r < 0 || r >= w_rows))) {
    if (tid == 0) report(status, kBadIndex);
    n = 0;
  }
  n = max(n, 0);
  int* out = kept + ((long long)b * Hkv + h) * keep;
  if (h == 0 && tid == 0) new_lens[b] = min(n, keep);
  if (n <= keep) {
    for (int j = tid; j < keep; j += 1024) out[j] = j < n ? j : -1;
    return;
  }
  float* w = weights + ((long long)r * Hkv + h) * w_len;
  const int first = sink, last = n - recent;  // tokens [first, last) compete for `need` places
  int need = keep - sink - recent;
  uint32_t prefix = 0, known = 0;
  for (int shift = 24; need > 0 && shift >= 0; shift -= 8) {
    if (tid < 256) hist[tid] = 0;
    __syncthreads();
    for (int t = first + tid; t < last; t += 1024) {
      const uint32_t key = weight_key(w[t]);
      if ((key & known) == prefix) atomicAdd(&hist[(key >> shift) & 255], 1);
    }
    __syncthreads();
    if (tid == 0) {
      int left = need, d = 255;
      while (hist[d] < left) left -= hist[d--];  // the digits above hold fewer than `need`: ends at d >= 0
      pick[0] = d;
      pick[1] = left;
    }
    __syncthreads();
    prefix |= (uint32_t)pick[0] << shift;
    known |= 255u << shift;
    need = pick[1];
    __syncthreads();
  }
  // every competitor above `prefix` is kept, and the first `need` of those equal to it
  const bool any = keep - sink - recent > 0;
  int done = 0, ties = 0;
  for (int base = 0; base < n; base += 1024) {
    const int t = base + tid;
    const float x = t < n ? w[t] : 0.f;
    const bool competes = t >= first && t < last;
    const uint32_t key = weight_key(x);
    int total;
    const bool tie = any && competes && key == prefix;
    const int rank = block_rank(tie, scratch, total);
    const bool keep_it = t < n && (!competes || (any && (key > prefix || (tie && ties + rank < need))));
    ties += total;
    const int at = done + block_rank(keep_it, scratch, total);
    if (keep_it) {  // every thread has read its weight: block_rank() synchronised
      w[at] = x;
      out[at] = t;
    }
    done += total;
    __syncthreads();
  }
  for (int t = keep + tid; t < n; t += 1024) w[t] = 0.f;
}

// Moves the kept tokens' stored rows (codes and scales) to the new blocks, 16 bytes a thread.
template <int D>
__global__ void __launch_bounds__(256) q4_move_kernel(uint8_t* k_pool, uint8_t* v_pool, const int* __restrict__ tables,
                                                      const int* __restrict__ new_tables, const int* __restrict__ kept,
                                                      const int* __restrict__ new_lens, int B, int Hkv, int max_blocks,
                                                      int new_blocks, int num_blocks, int keep, int* status) {
  using L = Q4<D>;
  constexpr int UNITS = L::kRow / 16;  // 16-byte units of a token in a group
  uint8_t* pool = blockIdx.y ? v_pool : k_pool;
  const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  const int unit = (int)(i % UNITS);
  const long long tok = i / UNITS;
  const int slot = (int)(tok % kTok);
  const int grp = (int)(tok / kTok % L::kGroups);
  const int nb = (int)(tok / kTok / L::kGroups % new_blocks);
  const long long bh = tok / kTok / L::kGroups / new_blocks;
  if (bh >= (long long)B * Hkv) return;
  const int b = (int)(bh / Hkv), h = (int)(bh % Hkv), j = nb * kTok + slot;
  if (j >= new_lens[b]) return;
  const int t = kept[bh * keep + j];
  const int from = t / kTok < max_blocks ? tables[(long long)b * max_blocks + t / kTok] : -1;
  const int to = new_tables[(long long)b * new_blocks + nb];
  if (from < 0 || from >= num_blocks || to < 0 || to >= num_blocks) {
    report(status, kBadIndex);
    return;
  }
  const uint8_t* src = pool + ((long long)from * Hkv + h) * L::kBytes;
  uint8_t* dst = pool + ((long long)to * Hkv + h) * L::kBytes;
  const int off = t % kTok;
  *reinterpret_cast<uint4*>(dst + (grp * kTok + slot) * L::kRow + unit * 16) =
      *reinterpret_cast<const uint4*>(src + (grp * kTok + off) * L::kRow + unit * 16);
  if (unit == 0)
    *reinterpret_cast<uint32_t*>(dst + L::kCodes + (grp * kTok + slot) * 4) =
        *reinterpret_cast<const uint32_t*>(src + L::kCodes + (grp * kTok + off) * 4);
}

}  // namespace rlb

using namespace rlb;

#define RLB_Q4_D(call)                                  \
  do {                                                  \
    if (D == 32) { constexpr int DD = 32; call; }       \
    else if (D == 64) { constexpr int DD = 64; call; }  \
    else if (D == 128) { constexpr int DD = 128; call; }\
    else return cudaErrorNotSupported;                  \
  } while (0)

cudaError_t rlb_q4_write(const void* k_new, const void* v_new, long long k_sn, long long k_sh, long long v_sn,
                         long long v_sh, void* k_pool, void* v_pool, const int* slot_block, const int* slot_off,
                         long long N, int Hkv, int D, int num_blocks, int* status, cudaStream_t s) {
  if (N == 0) return cudaSuccess;
  const long long threads = N * Hkv * (D / 8);
  const dim3 grid((unsigned)((threads + 255) / 256), 2);
  RLB_Q4_D((q4_write_kernel<DD><<<grid, 256, 0, s>>>(
      (const __nv_bfloat16*)k_new, (const __nv_bfloat16*)v_new, k_sn, k_sh, v_sn, v_sh, (uint8_t*)k_pool,
      (uint8_t*)v_pool, slot_block, slot_off, N, Hkv, num_blocks, status)));
  return cudaGetLastError();
}

cudaError_t rlb_q4_read(const void* k_pool, const void* v_pool, const int* slot_block, const int* slot_off,
                        const int* tables, const int* lens, int max_blocks, int max_len, long long N, int Hkv, int D,
                        int num_blocks, void* k_out, void* v_out, int* status, cudaStream_t s) {
  if (N == 0) return cudaSuccess;
  const long long threads = N * Hkv * (D / 8);
  const dim3 grid((unsigned)((threads + 255) / 256), 2);
  RLB_Q4_D((q4_read_kernel<DD><<<grid, 256, 0, s>>>((const uint8_t*)k_pool, (const uint8_t*)v_pool, slot_block,
                                                    slot_off, tables, lens, max_blocks, max_len, N, Hkv, num_blocks,
                                                    (__nv_bfloat16*)k_out, (__nv_bfloat16*)v_out, status)));
  return cudaGetLastError();
}

cudaError_t rlb_q4_decode(const void* q, const void* k_pool, const void* v_pool, const int* tables, const int* lens,
                          void* out, int B, int Hkv, int G, int D, int max_blocks, int num_blocks, float scale,
                          float softcap, int window, float* ml, float* weights, const int* weight_rows,
                          long long w_rows, int w_len, int* status, cudaStream_t s) {
  if (B == 0) return cudaSuccess;
  const Q4Cache c{(const uint8_t*)k_pool, (const uint8_t*)v_pool, tables, lens, Hkv, G, max_blocks, num_blocks,
                  window, scale, softcap};
  RLB_Q4_D((q4_decode_kernel<DD><<<dim3(Hkv * G, B), 128, 0, s>>>((const __nv_bfloat16*)q, c, (__nv_bfloat16*)out, ml,
                                                                  status)));
  if (weights != nullptr)
    RLB_Q4_D((q4_weights_kernel<DD><<<dim3(Hkv, B), 128, 0, s>>>((const __nv_bfloat16*)q, c, ml, weights, weight_rows,
                                                                 w_rows, w_len, status)));
  return cudaGetLastError();
}

cudaError_t rlb_q4_evict(void* k_pool, void* v_pool, const int* tables, const int* lens, const int* new_tables,
                         float* weights, const int* weight_rows, int* kept, int* new_lens, int B, int Hkv, int D,
                         int max_blocks, int new_blocks, int num_blocks, long long w_rows, int w_len, int keep,
                         int recent, int sink, int* status, cudaStream_t s) {
  if (B == 0) return cudaSuccess;
  q4_select_kernel<<<dim3(Hkv, B), 1024, 0, s>>>(lens, weights, weight_rows, kept, new_lens, Hkv, w_rows, w_len, keep,
                                                 recent, sink, status);
  const long long rows = (long long)B * Hkv * new_blocks * kTok;
  RLB_Q4_D((q4_move_kernel<DD><<<dim3((unsigned)((rows * Q4<DD>::kGroups * (Q4<DD>::kRow / 16) + 255) / 256), 2), 256, 0, s>>>(
      (uint8_t*)k_pool, (uint8_t*)v_pool, tables, new_tables, kept, new_lens, B, Hkv, max_blocks, new_blocks,
      num_blocks, keep, status)));
  return cudaGetLastError();
}
