// Paged KV cache held in 4 bits: storing and reading rows, decode attention over it, eviction.
//
// Pool layout (k_pool and v_pool alike): uint8 [num_blocks][Hkv][block bytes], a block being 16 tokens of one KV
// head.  With groups of g = min(D, 64) dimensions a block holds, for each group, the codes [16][g / 2] (element 2i
// in the low half of byte i) and behind all codes, for each group, [16] pairs (scale, minimum) in bf16.  An element
// stands for minimum + scale * code, with
//   minimum = min x,  scale = bf16((max x - min x) / 15),  code = clamp(rint((x - minimum) / scale), 0, 15)
// over the group: the inputs are bf16, so the minimum is exact, and the codes are chosen against the rounded scale.
// Group-major codes keep the 16 tokens x 64 dimensions that a matrix instruction works on contiguous (512 bytes).
#include <cooperative_groups.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "sm100.cuh"

namespace rlb {

constexpr int kTok = 16;  // tokens per block

template <int D>
struct Q4 {
  static constexpr int kGroup = D < 64 ? D : 64;
  static constexpr int kGroups = D / kGroup;
  static constexpr int kRow = kGroup / 2;                     // code bytes of one token in one group
  static constexpr int kCodes = kTok * D / 2;                 // code bytes of a block
  static constexpr int kBytes = kCodes + kTok * kGroups * 4;  // bytes of a block
  static constexpr int kLanes = kGroup / 16;                  // threads that share a group, 16 elements each
  static constexpr int kRows = 4096 / D;                      // rows of 256 threads with 16 elements each
};

RLB_DEVICE float bf16_lo_f(uint32_t v) { return __uint_as_float(v << 16); }
RLB_DEVICE float bf16_hi_f(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }

// Two nibbles of a word in one instruction: (w & mask) | 0x64006400.  (Written out because the compiler takes two
// where both constants are immediates; `magic` comes from a register.)
template <uint32_t MASK>
RLB_DEVICE uint32_t nibbles(uint32_t w, uint32_t magic) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(w), "n"(MASK), "r"(magic));
  return r;
}

RLB_DEVICE uint32_t half2_add(uint32_t x, uint32_t both) {
  const __half2 y = __hadd2(*reinterpret_cast<const __half2*>(&x), *reinterpret_cast<const __half2*>(&both));
  return *reinterpret_cast<const uint32_t*>(&y);
}

// Nibbles j and j + 4 of a word as two fp16 numbers: code - 8 for j = 0 and 2, 1024 + 16 code for j = 1 and 3.
RLB_DEVICE void codes_f16(uint32_t w, uint32_t (&r)[4], uint32_t magic) {
  constexpr uint32_t off = 0xe408e408u;  // -1032
  const uint32_t x = w >> 8;
  r[0] = half2_add(nibbles<0x000f000fu>(w, magic), off);
  r[1] = nibbles<0x00f000f0u>(w, magic);
  r[2] = half2_add(nibbles<0x000f000fu>(x, magic), off);
  r[3] = nibbles<0x00f000f0u>(x, magic);
}

// The same nibbles as two bf16 numbers, code - 8 (bits 0x4300 | code are 128 + code; bf16 has too few bits for the
// second nibble's 16 code).
RLB_DEVICE void codes_bf16(uint32_t w, uint32_t (&r)[4], uint32_t magic) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t x = nibbles<0x000f000fu>(w >> (4 * j), magic);
    const __nv_bfloat162 y = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&x), __float2bfloat162_rn(136.f));
    r[j] = *reinterpret_cast<const uint32_t*>(&y);
  }
}

// ---------------------------------------------------------------- storing rows
// A group's four threads (two at D 32) reduce its minimum and maximum by shuffles (NaN-propagating), then each
// quantises its 16 elements to two 32-bit words.  Bound by memory latency and pattern (rows of 256 bytes in, 32-byte
// pieces of a block out): 32768 rows of 8 heads x 128 in 48 us, 3.6 TB/s; 8 elements a thread took 4 us more, and 40
// registers for half as many warps again 59, a grid of one wave that fetches the next row ahead 56.
//
// code = clamp(rint((x - lo) / s)) without a division per element: q = (x - lo) (1 / s) and its remainder's share
// q + (x - lo - q s) (1 / s) is the correctly rounded quotient (a quotient corrected by its remainder, after P. Markstein,
// 1990), and adding 1.5 2^23 rounds that to a whole number.
RLB_DEVICE uint32_t q4_codes(const bf16x8& x, float lo, float s) {
  float f[8];
  unpack8(x, f);
  uint32_t word = 0;
  if (!(s >= 1e-36f && s < INFINITY)) {  // no spread, one too small for 1 / s, or not finite (all codes are 0)
#pragma unroll
    for (int e = 0; e < 8; ++e)
      word |= (uint32_t)fminf(fmaxf(rintf(__fdiv_rn(f[e] - lo, s)), 0.f), 15.f) << (4 * e);  // NaN becomes 0
    return word;
  }
  const float inv = __fdividef(1.f, s);  // (the remainder makes up for its last bit)
  const float2 inv2 = make_float2(inv, inv), minus_s = make_float2(-s, -s), minus_lo = make_float2(-lo, -lo);
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    const float2 d = add2(make_float2(f[e], f[e + 1]), minus_lo), q = mul2(d, inv2);
    const float2 y = add2(fma2(fma2(q, minus_s, d), inv2, q), make_float2(12582912.f, 12582912.f));
    word += __float_as_uint(y.x) << (4 * e);
    word += __float_as_uint(y.y) << (4 * e + 4);
  }
  // y's bits are 0x4b400000 + code; no code is above 15, s being within 2^-9 of a 15th of the spread
  return word - 0x4b400000u * 0x11111111u;
}

RLB_DEVICE __nv_bfloat162 min8(const bf16x8& a, const bf16x8& b) {
  return __hmin2_nan(__hmin2_nan(__hmin2_nan(a.h[0], a.h[1]), __hmin2_nan(a.h[2], a.h[3])),
                     __hmin2_nan(__hmin2_nan(b.h[0], b.h[1]), __hmin2_nan(b.h[2], b.h[3])));
}
RLB_DEVICE __nv_bfloat162 max8(const bf16x8& a, const bf16x8& b) {
  return __hmax2_nan(__hmax2_nan(__hmax2_nan(a.h[0], a.h[1]), __hmax2_nan(a.h[2], a.h[3])),
                     __hmax2_nan(__hmax2_nan(b.h[0], b.h[1]), __hmax2_nan(b.h[2], b.h[3])));
}

// Blocks of threads take 4096 / D rows of one KV head, keys and values alike; the heads (x) of the same rows (y) are
// neighbours in the grid, as they are in memory.
template <int D>
__global__ void __launch_bounds__(256) q4_write_kernel(
    const __nv_bfloat16* __restrict__ k_new, const __nv_bfloat16* __restrict__ v_new, long long k_sn, long long k_sh,
    long long v_sn, long long v_sh, uint8_t* __restrict__ k_pool, uint8_t* __restrict__ v_pool,
    const int* __restrict__ slot_block, const int* __restrict__ slot_off, long long N, int num_blocks, int* status) {
  using L = Q4<D>;
  const int h = blockIdx.x, Hkv = gridDim.x, part = threadIdx.x % (D / 16);
  const int grp = part / L::kLanes, lane = part % L::kLanes;
  const unsigned mask = ((1u << L::kLanes) - 1) << (threadIdx.x & 31 & ~(L::kLanes - 1));
  for (long long n = (long long)blockIdx.y * L::kRows + threadIdx.x / (D / 16); n < N; n += (long long)gridDim.y * L::kRows) {
    const __nv_bfloat16* kp = k_new + n * k_sn + h * k_sh + part * 16;
    const __nv_bfloat16* vp = v_new + n * v_sn + h * v_sh + part * 16;
    const bf16x8 x[2][2] = {{ldg8(kp), ldg8(kp + 8)}, {ldg8(vp), ldg8(vp + 8)}};
    const int blk = slot_block[n], off = slot_off[n];
    if (blk < 0 || blk >= num_blocks || off < 0 || off >= kTok) {  // (whole groups: they share a row)
      if (lane == 0) report(status, kBadIndex);
      continue;
    }
    const long long at = ((long long)blk * Hkv + h) * L::kBytes;
    const int code = (grp * kTok + off) * L::kRow + lane * 8, meta = L::kCodes + (grp * kTok + off) * 4;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint8_t* pool = (i ? v_pool : k_pool) + at;
      const __nv_bfloat162 mn = min8(x[i][0], x[i][1]), mx = max8(x[i][0], x[i][1]);
      // minimum and negated maximum side by side: one shuffle and one minimum a step
      __nv_bfloat162 ends = __halves2bfloat162(__hmin_nan(mn.x, mn.y), __hneg(__hmax_nan(mx.x, mx.y)));
#pragma unroll
      for (int o = 1; o < L::kLanes; o <<= 1) ends = __hmin2_nan(ends, __shfl_xor_sync(mask, ends, o));
      const __nv_bfloat16 lo = ends.x;
      const float lof = __bfloat162float(lo);
      // the range over 15, correctly rounded (a quotient and its remainder's)
      const float range = -__bfloat162float(ends.y) - lof, q0 = range * (1.f / 15.f);
      const __nv_bfloat16 scale = __float2bfloat16(fmaf(fmaf(-15.f, q0, range), 1.f / 15.f, q0));
      const float sf = __bfloat162float(scale);
      *reinterpret_cast<uint2*>(pool + code) = make_uint2(q4_codes(x[i][0], lof, sf), q4_codes(x[i][1], lof, sf));
      if (lane == 0)
        *reinterpret_cast<uint32_t*>(pool + meta) =
            (uint32_t)__bfloat16_as_ushort(scale) | ((uint32_t)__bfloat16_as_ushort(lo) << 16);
    }
  }
}

// ---------------------------------------------------------------- reading rows
// The 8 elements of a word: codes become bf16 numbers by their bits (128 + code), and minimum + scale code is rounded once.
RLB_DEVICE uint4 q4_elements(uint32_t word, uint32_t scale_min) {
  const uint32_t ss = __byte_perm(scale_min, 0, 0x1010), ll = __byte_perm(scale_min, 0, 0x3232);
  const __nv_bfloat162 s = *reinterpret_cast<const __nv_bfloat162*>(&ss), lo = *reinterpret_cast<const __nv_bfloat162*>(&ll);
  uint32_t x[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {  // elements j and j + 4
    const uint32_t m = nibbles<0x000f000fu>(word >> (4 * j), 0x43004300u);
    const __nv_bfloat162 n = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&m), __float2bfloat162_rn(128.f));
    const __nv_bfloat162 y = __hfma2(n, s, lo);
    x[j] = *reinterpret_cast<const uint32_t*>(&y);
  }
  return make_uint4(__byte_perm(x[0], x[1], 0x5410), __byte_perm(x[2], x[3], 0x5410), __byte_perm(x[0], x[1], 0x7632),
                    __byte_perm(x[2], x[3], 0x7632));
}

// One thread per 8 elements of a key and of a value (16 of each would write every sector in two halves: 119 us where
// this takes 39 for 32768 rows of 8 x 128).  Row n is slot (slot_block[n], slot_off[n]), or, with a block table, position
// n % max_len of sequence n / max_len.  Rows without a place in the pool read as zeros.  Bound by the write of the rows:
// 32768 rows of 8 x 128 in 37 us (4.7 TB/s, reads and writes); 16 sequences of 1024 by table in 18.
template <int D>
__global__ void __launch_bounds__(256) q4_read_kernel(const uint8_t* __restrict__ k_pool,
                                                      const uint8_t* __restrict__ v_pool,
                                                      const int* __restrict__ slot_block,
                                                      const int* __restrict__ slot_off, const int* __restrict__ tables,
                                                      const int* __restrict__ lens, int max_blocks, int max_len,
                                                      long long N, int num_blocks,
                                                      __nv_bfloat16* __restrict__ k_out,
                                                      __nv_bfloat16* __restrict__ v_out, int* status) {
  using L = Q4<D>;
  constexpr int ROWS = L::kRows / 2;
  const int h = blockIdx.x, Hkv = gridDim.x, part = threadIdx.x % (D / 8);
  const int grp = part * 8 / L::kGroup, lane = part % (L::kGroup / 8);
  for (long long n = (long long)blockIdx.y * ROWS + threadIdx.x / (D / 8); n < N; n += (long long)gridDim.y * ROWS) {
    int blk = -1, off = 0;
    bool absent = false;
    if (tables == nullptr) {
      blk = slot_block[n];
      off = slot_off[n];
    } else {
      const long long b = n >> 31 == 0 ? (long long)((unsigned)n / (unsigned)max_len) : n / max_len;
      const int pos = (int)(n - b * max_len);
      off = pos % kTok;
      absent = pos >= lens[b];
      if (!absent && pos / kTok < max_blocks) blk = tables[b * max_blocks + pos / kTok];
    }
    uint4 k = make_uint4(0, 0, 0, 0), v = k;
    if (!absent && (blk < 0 || blk >= num_blocks || off < 0 || off >= kTok)) {
      if (part == 0 && h == 0) report(status, kBadIndex);
      absent = true;
    }
    if (!absent) {
      const long long at = ((long long)blk * Hkv + h) * L::kBytes;
      const int code = (grp * kTok + off) * L::kRow + lane * 4, meta = L::kCodes + (grp * kTok + off) * 4;
      const uint32_t kw = *reinterpret_cast<const uint32_t*>(k_pool + at + code), km = *reinterpret_cast<const uint32_t*>(k_pool + at + meta);
      const uint32_t vw = *reinterpret_cast<const uint32_t*>(v_pool + at + code), vm = *reinterpret_cast<const uint32_t*>(v_pool + at + meta);
      k = q4_elements(kw, km);
      v = q4_elements(vw, vm);
    }
    const long long to = (n * Hkv + h) * D + part * 8;
    *reinterpret_cast<uint4*>(k_out + to) = k;
    *reinterpret_cast<uint4*>(v_out + to) = v;
  }
}

// ---------------------------------------------------------------- decode attention
// The work is the turns (2 or 4 blocks of 16 tokens) of all (sequence, KV head) rows in a line, cut into equal
// stretches, one for each warp that fits on the GPU: lengths are ragged and known on the device only, and a grid of
// whole rows or of fixed parts leaves SMs idle at the end.  A warp works alone, with no barrier: it brings blocks (codes,
// scales and minima of K and V, one contiguous piece each) into its own ring of shared memory with bulk copies, which
// run ahead across the rows' borders, and computes on matrix instructions
// (mma.sync m16n8k16, two fp16 or two bf16 operands -> fp32) with the 16 tokens, then the dimensions, as the 16 rows and up to 8
// query heads of the KV head as the 8 columns.  The kernel is bound by the latency of the dependent instructions that
// unpack the codes, not by bytes or tensor throughput: at 1/8 of the rows a tcgen05 tile (64 or 128 rows at least,
// operands in shared memory) would need the unpacked values written back to shared memory first.  32 ragged sequences of
// up to 8192 tokens (8 KV heads x 128, 4 queries each, 189 MB): 66 us with the join (kernel 61, 3.1 TB/s); one of 100001:
// 45 us, 2.6 TB/s; 64 of up to 4096 with heads of 64 (90 MB): 39 us.  (With one fp16 weight 59, 41 and 37 us.)  406
// instructions per block of 16 tokens and 128 dimensions, issued at 2.2 of the 4 a cycle that an SM has slots for: 2.8
// warps a scheduler (167 registers a thread) do not cover the fixed latencies, no pipe is above 51 %, and memory is
// waited for least.
//
// K's codes become fp16 numbers exactly, by the format alone: bits 0x6400 | code are 1024 + code and 0x6400 | code << 4
// are 1024 + 16 code, so half of the nibbles need no shift, and a packed add makes code - 8 of the others.
// S^T = K Q^T.  With a token's scale s and minimum m:  k . q = s (code . q) + m sum(q), per group of dimensions.  Q
// is fp16 after division by a power of two per head (its largest element then lies in [2^13, 2^14)): bf16's 8 bits
// fit, and what falls below 2^-24 is 2^-38 of the largest.  K's odd nibbles stay 1024 + 16 code: their q are divided by 16,
// and the sums start at 8 sum(q even) - 64 sum(q odd) instead of zero, which leaves code . q.  The order of the
// dimensions inside the product is free as long as Q's registers use the same: a lane reads 16 consecutive dimensions of a token as two
// words and takes nibbles j and j + 4 of a word as one operand register.
// O^T = V^T P^T in bf16.  The token's scale goes into the weight and its minimum into a separate fp32 sum of
// p (m + 8 s).  A weight p s is held in two bf16 parts, its upper 8 bits and what is left of it rounded to 8 bits
// (2^-16 of each weight, below a hundredth of the output's own rounding to bf16), and both go through the matrix
// instruction.  bf16 has fp32's exponents, so that values of any size keep these bits beside each other: p is kept times
// 2^-32, with which 2^20 tokens of the type's largest values stay in range and values from 2^-58 on keep all their bits.
// (One fp16 weight, 2^-11 of each, needed the weights scaled by V's largest scale, from which values far below it
// lost bits even where that token's weight was nothing.)
// The tokens' order is free too: row g of S^T (of each half of the block) is token g / 2 for even g and
// 4 + (g / 2 ^ 2) for odd g.  After the 8 x 8 transposition (movmatrix) that turns S^T's registers into P^T's, lane
// t of a quad has the tokens t and 4 + (t ^ 2) of both halves; neither its four V words nor the K words that a half
// warp reads at a time then share a bank.
//
// Softmax statistics are fp32 in base 2.  The running maximum is only raised (and the sums rescaled) when a score
// exceeds it by 8, so weights stay below 2^8 relative to it.  It is a whole number (rounded up), so that it and the
// factors between the maxima of parts are exact.  A turn of several blocks shares the waits, votes and bookkeeping
// among 32 (D = 128) or 64 tokens.
struct Q4Cache {
  const uint8_t *k_pool, *v_pool;
  const int *tables, *lens;
  int Hkv, G, max_blocks, num_blocks, window;
  int turn;  // blocks a warp takes at a time (q4_turn)
  float scale, softcap;
};

constexpr int kDecodeWarps = 4;
constexpr float kDown = 32.f;  // weights, their sums and the outputs are kept times 2^-kDown
constexpr uint32_t kWaitLimit = 1u << 22;  // polls; a copy takes microseconds

RLB_DEVICE void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, float c0, float c1, float c2,
                        float c3) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}

RLB_DEVICE void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

RLB_DEVICE uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

RLB_DEVICE void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

// Two fp32 numbers as two bf16 parts of each: the upper bits, and what they leave, rounded.
RLB_DEVICE void split_bf16(float x, float y, uint32_t& upper, uint32_t& rest) {
  const uint32_t a = __float_as_uint(x), b = __float_as_uint(y);
  upper = __byte_perm(a, b, 0x7632);
  const __nv_bfloat162 r = __floats2bfloat162_rn(x - __uint_as_float(a & 0xffff0000u), y - __uint_as_float(b & 0xffff0000u));
  rest = *reinterpret_cast<const uint32_t*>(&r);
}

RLB_DEVICE uint32_t pack_f16(float lo, float hi) {
  const __half2 r = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&r);
}

RLB_DEVICE int q4_token(int g) { return g & 1 ? 4 + (g >> 1 ^ 2) : g >> 1; }

RLB_DEVICE float pow2(int e) { return __int_as_float((e + 127) << 23); }  // -126 <= e <= 127

RLB_DEVICE int q4_len(const Q4Cache& c, int b, int* status) {
  const int len = c.lens[b], most = c.max_blocks * kTok;
  if (len > most) report(status, kBadIndex);
  return min(max(len, 0), most);
}

// First token that a sequence of `len` tokens attends to, and its turns from there on.
RLB_DEVICE int q4_first(const Q4Cache& c, int len) { return c.window > 0 && len > c.window ? len - c.window : 0; }
RLB_DEVICE int q4_turns(const Q4Cache& c, int len) {
  if (len == 0) return 0;
  const int blocks = (len - 1) / kTok - q4_first(c, len) / kTok + 1;
  return (blocks + c.turn - 1) / c.turn;
}

// The turns of all rows lie in a line: row (b, h) holds [base(b) + h n(b), + n(b)), and warp k of C the stretch
// [cut(k), cut(k + 1)).  A part (k, row) gets scratch slot k + row: along the line each next part raises one of the two.
RLB_DEVICE int q4_cut(int k, int total, int C) { return k * (total / C) + k * (total % C) / C; }  // C^2 < 2^31
RLB_DEVICE int q4_owner(int x, int total, int C) {  // ((x + 1) C - 1) / total: exact, the numbers have fewer than 53 bits
  return (int)(((double)(x + 1) * C - 1) / total);
}

// Turns of all sequences (all KV heads), the warps that share them (each gets one at least, so that a row's slots follow
// each other without a gap), and the sequence that holds turn x = cut(k), with the turns before it.
struct Q4Line {
  int total, warps, x, seq, base;
};
RLB_DEVICE Q4Line q4_line(const Q4Cache& c, int B, int k, int C, int* status) {
  const int lane = threadIdx.x & 31;
  Q4Line r{0, 0, 0, B, 0};
  int n = 0;
  for (int b0 = 0; b0 < B; b0 += 32) {
    n = b0 + lane < B ? q4_turns(c, q4_len(c, b0 + lane, status)) * c.Hkv : 0;
    r.total += __reduce_add_sync(0xffffffffu, n);
  }
  r.warps = min(C, r.total);
  if (k >= r.warps) return r;
  r.x = q4_cut(k, r.total, r.warps);
  for (int b0 = 0; b0 < B; b0 += 32) {
    if (B > 32) n = b0 + lane < B ? q4_turns(c, q4_len(c, b0 + lane, nullptr)) * c.Hkv : 0;
    int incl = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += y;
    }
    const unsigned behind = __ballot_sync(0xffffffffu, r.x < r.base + incl);
    if (behind) {
      const int at = __ffs(behind) - 1;
      r.seq = b0 + at;
      r.base += __shfl_sync(0xffffffffu, incl - n, at);
      break;
    }
    r.base += __shfl_sync(0xffffffffu, incl, 31);
  }
  return r;
}

constexpr float kLog2e = 1.4426950408889634f;

constexpr int q4_ctas(int D, int NT) { return NT == 2 ? 2 : D == 128 ? 3 : 4; }  // CTAs on an SM at a time
template <int D>
constexpr int q4_turn() { return D == 128 ? 2 : 4; }   // blocks a turn
template <int D>
constexpr int q4_stages() { return 2; }                // turns in a warp's ring

// One turn's work of a warp: the blocks at `ks` (each K then V).  MASKED: some of the tokens are not seen.
template <int D, int NT>
struct Q4Warp {
  using L = Q4<D>;
  static constexpr int NG = L::kGroups, WPL = L::kGroup / 32, MT = L::kGroup / 16, BT = q4_turn<D>();
  uint32_t qb[NT][NG][WPL][4];                   // Q^T's registers (column n = head g of each tile)
  float qs[NT][NG][2], qc[NT][NG][2], qf[NT][2]; // heads 2t, 2t + 1: sums of q, where S starts, the scores' factor
  float m[NT][2], lim[NT][2];                    // maximum when it was last raised, the s that lies 8 above it
  float mref[NT][2], l[NT][2];                   // what exponents are taken against, sum of p
  float z[NT][NG][2], o[NT][NG][MT][4];          // sums of p (m + 8 s) and of p s (code - 8)
  uint32_t magic, magic_bf16;                    // 0x64006400, 0x43004300

  RLB_DEVICE void load_q(const __nv_bfloat16* q, int G, float scale) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int head = n * 8 + g;
      float f[NG][WPL][8], big = 0.f;
#pragma unroll
      for (int r = 0; r < NG; ++r)
#pragma unroll
        for (int w = 0; w < WPL; ++w) {
          if (head < G) unpack8(ldg8(q + head * D + r * L::kGroup + (t * WPL + w) * 8), f[r][w]);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            if (head >= G) f[r][w][j] = 0.f;
            big = fmaxf(big, fabsf(f[r][w][j]));
          }
        }
      big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
      big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
      // q 2^e has its largest element in [2^13, 2^14)
      const int e = min(max(140 - (int)(__float_as_uint(big) >> 23), -126), 126);
      const float up = scale < 0.f ? -pow2(e) : pow2(e);  // a negative scale's sign goes into q
      float factor = fmaxf(fabsf(scale) * pow2(-e), 1e-37f);  // not 0, which -inf of unseen tokens could not take
#pragma unroll
      for (int r = 0; r < NG; ++r) {
        float sum = 0.f, odd = 0.f;
#pragma unroll
        for (int w = 0; w < WPL; ++w)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float x = f[r][w][j] * up, y = f[r][w][j + 4] * up, part = j & 1 ? 0.0625f : 1.f;
            qb[n][r][w][j] = pack_f16(x * part, y * part);
            sum += x + y;
            if (j & 1) odd += x + y;
          }
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
          sum += __shfl_xor_sync(0xffffffffu, sum, o);
          odd += __shfl_xor_sync(0xffffffffu, odd, o);
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          qs[n][r][e] = __shfl_sync(0xffffffffu, sum, t * 8 + 4 * e);
          qc[n][r][e] = 8.f * qs[n][r][e] - 72.f * __shfl_sync(0xffffffffu, odd, t * 8 + 4 * e);
        }
      }
      qf[n][0] = __shfl_sync(0xffffffffu, factor, t * 8);
      qf[n][1] = __shfl_sync(0xffffffffu, factor, t * 8 + 4);
    }
  }

  RLB_DEVICE void reset() {
    asm volatile("mov.b32 %0, 0x64006400;" : "=r"(magic));  // kept in registers
    asm volatile("mov.b32 %0, 0x43004300;" : "=r"(magic_bf16));
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        m[n][e] = lim[n][e] = -INFINITY;
        mref[n][e] = l[n][e] = 0.f;
#pragma unroll
        for (int r = 0; r < NG; ++r) {
          z[n][r][e] = 0.f;
#pragma unroll
          for (int i = 0; i < MT; ++i) o[n][r][i][e] = o[n][r][i][e + 2] = 0.f;
        }
      }
  }

  static RLB_DEVICE float largest(const float (&s)[BT][4], int e) {
    float x = fmaxf(s[0][e], s[0][e + 2]);
#pragma unroll
    for (int k = 1; k < BT; ++k) x = fmaxf(x, fmaxf(s[k][e], s[k][e + 2]));
    return x;
  }

  // seen: bit 2k + i: this lane's token i of block k is attended to, bit 8 + 2k + i: it has a place in `scores`.  `scores`: this lane's token 0 of block 0, or null.
  template <bool MASKED>
  RLB_DEVICE void turn(const uint8_t* ks, unsigned seen, float softcap, float* scores, int Gs) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int tok = q4_token(g);  // this lane's tokens of a block in S^T: tok and tok + 8
    float s[NT][BT][4];
#pragma unroll
    for (int k = 0; k < BT; ++k)
#pragma unroll
      for (int r = 0; r < NG; ++r) {
        const uint8_t* blk = ks + k * 2 * L::kBytes;
        float acc[NT][4];
        uint32_t u0[WPL], u1[WPL];
        const uint8_t* row = blk + (r * kTok + tok) * L::kRow + t * WPL * 4;
        if constexpr (WPL == 2) {
          *reinterpret_cast<uint2*>(u0) = *reinterpret_cast<const uint2*>(row);
          *reinterpret_cast<uint2*>(u1) = *reinterpret_cast<const uint2*>(row + 8 * L::kRow);
        } else {
          u0[0] = *reinterpret_cast<const uint32_t*>(row);
          u1[0] = *reinterpret_cast<const uint32_t*>(row + 8 * L::kRow);
        }
#pragma unroll
        for (int w = 0; w < WPL; ++w) {
          uint32_t c0[4], c1[4];
          codes_f16(u0[w], c0, magic);
          codes_f16(u1[w], c1, magic);
#pragma unroll
          for (int j = 0; j < 4; j += 2) {
            const uint32_t a[4] = {c0[j], c1[j], c0[j + 1], c1[j + 1]};
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              const bool first = w == 0 && j == 0;
              mma_f16(acc[n], a, qb[n][r][w][j], qb[n][r][w][j + 1], first ? qc[n][r][0] : acc[n][0],
                      first ? qc[n][r][1] : acc[n][1], first ? qc[n][r][0] : acc[n][2], first ? qc[n][r][1] : acc[n][3]);
            }
          }
        }
        const uint32_t me0 = *reinterpret_cast<const uint32_t*>(blk + L::kCodes + (r * kTok + tok) * 4);
        const uint32_t me1 = *reinterpret_cast<const uint32_t*>(blk + L::kCodes + (r * kTok + tok + 8) * 4);
        const float s0 = bf16_lo_f(me0), s1 = bf16_lo_f(me1), z0 = bf16_hi_f(me0), z1 = bf16_hi_f(me1);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float x = r == 0 ? z0 * qs[n][r][e] : fmaf(z0, qs[n][r][e], s[n][k][e]);
            const float y = r == 0 ? z1 * qs[n][r][e] : fmaf(z1, qs[n][r][e], s[n][k][e + 2]);
            s[n][k][e] = fmaf(s0, acc[n][e], x);
            s[n][k][e + 2] = fmaf(s1, acc[n][e + 2], y);
          }
      }
    // from here on a score in base 2 is s qf
    if (softcap > 0.f) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int k = 0; k < BT; ++k)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float x = s[n][k][e] * qf[n][e & 1] * (1.f / kLog2e);
            s[n][k][e] = tanhf(x / softcap) * (softcap * kLog2e) / qf[n][e & 1];
          }
    }
    bool raise = false;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int k = 0; k < BT; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (MASKED && !((seen >> (2 * k + (e >> 1))) & 1)) s[n][k][e] = -INFINITY;
#pragma unroll
      for (int e = 0; e < 2; ++e) raise |= largest(s[n], e) > lim[n][e];
      if (scores != nullptr && n * 8 + 2 * t < Gs) {
#pragma unroll
        for (int k = 0; k < BT; ++k)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            if (!MASKED || ((seen >> (8 + 2 * k + i)) & 1))
              *reinterpret_cast<float2*>(scores + (k * kTok + 8 * i) * Gs + n * 8 + 2 * t) =
                  make_float2(s[n][k][2 * i] * qf[n][0], s[n][k][2 * i + 1] * qf[n][1]);
      }
    }
    if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float x = largest(s[n], e) * qf[n][e];
#pragma unroll
          for (int k = 4; k < 32; k <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, k));
          const float was = m[n][e];
          x = fmaxf(ceilf(x), was);
          const float up = was == -INFINITY ? 0.f : sm100::ex2_approx(was - x);
          m[n][e] = x;
          lim[n][e] = (x + 8.f) / qf[n][e];
          mref[n][e] = (x == -INFINITY ? 0.f : x) + kDown;
          l[n][e] *= up;
#pragma unroll
          for (int r = 0; r < NG; ++r) {
            z[n][r][e] *= up;
#pragma unroll
            for (int k = 0; k < MT; ++k) {
              o[n][r][k][e] *= up;
              o[n][r][k][e + 2] *= up;
            }
          }
        }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int k = 0; k < BT; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[n][k][e] = sm100::ex2_approx(fmaf(s[n][k][e], qf[n][e & 1], -mref[n][e & 1]));
          l[n][e & 1] += s[n][k][e];
        }
#pragma unroll
    for (int k = 0; k < BT; ++k)
#pragma unroll
      for (int r = 0; r < NG; ++r) {
        const uint8_t* blk = ks + (2 * k + 1) * L::kBytes;
        uint32_t vm[2];  // (scale, minimum) of this lane's tokens
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          vm[i] = *reinterpret_cast<const uint32_t*>(blk + L::kCodes + (r * kTok + tok + 8 * i) * 4);
          if (MASKED && !((seen >> (2 * k + i)) & 1)) vm[i] = 0;  // unseen slots may hold anything, NaN too
        }
        const float s0 = bf16_lo_f(vm[0]), s1 = bf16_lo_f(vm[1]);
        const float z0 = fmaf(8.f, s0, bf16_hi_f(vm[0])), z1 = fmaf(8.f, s1, bf16_hi_f(vm[1]));
        uint32_t b[NT][2][2];  // [upper part, rest]
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          split_bf16(s[n][k][0] * s0, s[n][k][1] * s0, b[n][0][0], b[n][1][0]);
          split_bf16(s[n][k][2] * s1, s[n][k][3] * s1, b[n][0][1], b[n][1][1]);
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 0; e < 2; ++e) b[n][i][e] = transpose8x8(b[n][i][e]);
          z[n][r][0] = fmaf(s[n][k][0], z0, fmaf(s[n][k][2], z1, z[n][r][0]));
          z[n][r][1] = fmaf(s[n][k][1], z0, fmaf(s[n][k][3], z1, z[n][r][1]));
        }
        // the group's codes for this lane: dimensions 8 g .. 8 g + 7 (4 g .. 4 g + 3), tokens t and u of both halves
        const int u = 4 + (t ^ 2);
        uint32_t c[2][WPL][4];  // [half of the block][dimensions 0-3 or 4-7], a token in each half of the registers
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint8_t* row = blk + (r * kTok + 8 * i) * L::kRow + g * WPL * 2;
          if constexpr (WPL == 2) {
            const uint32_t x = *reinterpret_cast<const uint32_t*>(row + t * L::kRow);
            const uint32_t y = *reinterpret_cast<const uint32_t*>(row + u * L::kRow);
            codes_bf16(__byte_perm(x, y, 0x5410), c[i][0], magic_bf16);
            codes_bf16(__byte_perm(x, y, 0x7632), c[i][1], magic_bf16);
          } else {
            codes_bf16(*reinterpret_cast<const uint16_t*>(row + t * L::kRow) |
                           ((uint32_t)*reinterpret_cast<const uint16_t*>(row + u * L::kRow) << 16),
                       c[i][0], magic_bf16);
          }
        }
#pragma unroll
        for (int i = 0; i < MT; ++i) {  // rows g and g + 8 of tile i are dimensions 2i and 2i + 1 of the lane's
          const int w = i >> 1, j = 2 * (i & 1);
          const uint32_t a[4] = {c[0][w][j], c[0][w][j + 1], c[1][w][j], c[1][w][j + 1]};
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            mma_bf16(o[n][r][i], a, b[n][1][0], b[n][1][1]);
            mma_bf16(o[n][r][i], a, b[n][0][0], b[n][0][1]);
          }
        }
      }
  }
};

// NT: tiles of 8 query heads.  Rows that lie in one warp's stretch are finished here, the others' parts go to `part`
// [slots][G][D] (unnormalised outputs) and `ml` [slots][G][2] (statistics); `plan` [row] = its first slot and its parts.
// `scores` [B][Hkv][tokens][Gs] receives the base-2 scores for q4_finish_kernel, which then needs every row's statistics.
template <int D, int NT>
__global__ void __launch_bounds__(kDecodeWarps * 32, q4_ctas(D, NT)) q4_decode_kernel(
    const __nv_bfloat16* __restrict__ q, Q4Cache c, int B, __nv_bfloat16* __restrict__ out, float* __restrict__ part,
    float* __restrict__ ml, int2* __restrict__ plan, float* __restrict__ scores, int Gs, int* status) {
  using L = Q4<D>;
  using W = Q4Warp<D, NT>;
  constexpr int S = q4_stages<D>(), BT = q4_turn<D>(), PER = 32 / BT;  // PER: turns whose blocks a warp has looked up
  constexpr int kStage = BT * 2 * L::kBytes;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(8) uint64_t bars[kDecodeWarps][S];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int G = c.G, me = blockIdx.x * kDecodeWarps + warp;
  uint8_t* ring = smem + warp * S * kStage;
  if (lane == 0) {
    for (int s = 0; s < S; ++s) sm100::mbar_init(&bars[warp][s], BT);
    sm100::fence_barrier_init();
    sm100::fence_async_shared();
  }
  __syncwarp();
  const Q4Line line = q4_line(c, B, me, gridDim.x * kDecodeWarps, me == 0 ? status : nullptr);
  if (me >= line.warps) return;
  const int turns = q4_cut(me + 1, line.total, line.warps) - line.x;

  // Where the warp's turns lie: lane BT i + k looks up block k of turn i of the next PER turns, one group ahead.
  int lb = line.seq, lbase = line.base, llen = q4_len(c, lb, nullptr);
  auto look = [&](int i0) {
    const int i = i0 + lane / BT, x = line.x + i;
    if (i >= turns) return -1;
    int n = q4_turns(c, llen);
    while (x >= lbase + n * c.Hkv) {  // ends: the last turn of the line is behind x
      lbase += n * c.Hkv;
      llen = q4_len(c, ++lb, nullptr);
      n = q4_turns(c, llen);
    }
    const int h = (x - lbase) / n, p = x - lbase - h * n;
    const int at = q4_first(c, llen) / kTok + p * BT + lane % BT;
    if (at > (llen - 1) / kTok) return -1;
    const int id = c.tables[(long long)lb * c.max_blocks + at];
    if (id >= 0 && id < c.num_blocks) return id * c.Hkv + h;
    report(status, kBadIndex);
    return -1;
  };
  int unit = -1, next = look(0);  // block * Hkv + head, or -1
  unsigned good = 0;              // bit BT i + k: that block is there
  const uint32_t ring_at = sm100::smem_u32(ring) + lane % BT * 2 * L::kBytes, bar_at = sm100::smem_u32(&bars[warp][0]);
  auto issue = [&](int i) {
    if (i >= turns) return;
    if (i % PER == 0) {
      unit = next;
      good = __ballot_sync(0xffffffffu, unit >= 0);
      next = look(i + PER);
    }
    if (lane / BT == i % PER) {  // the lanes that looked the turn's blocks up
      const uint32_t dst = ring_at + i % S * kStage, bar = bar_at + i % S * 8;
      asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(unit >= 0 ? 2 * L::kBytes : 0) : "memory");
      if (unit >= 0) {
        const long long at = (long long)unit * L::kBytes;
        bulk_load(dst, c.k_pool + at, L::kBytes, bar);
        bulk_load(dst + L::kBytes, c.v_pool + at, L::kBytes, bar);
      }
    }
  };
#pragma unroll
  for (int i = 0; i < S; ++i) issue(i);

  const int tok = q4_token(g);
  int b = line.seq, base = line.base, len = q4_len(c, b, nullptr), n = q4_turns(c, len);
  while (n == 0) {  // (sequences without tokens hold nothing)
    len = q4_len(c, ++b, nullptr);
    n = q4_turns(c, len);
  }
  int h = (line.x - base) / n, p = line.x - base - h * n;
  W w;
  unsigned here_now = 0;  // `good` of the PER turns that are being worked on
  for (int i = 0; i < turns;) {
    // one part: turns p .. p1 of row (b, h)
    const int p0 = p, p1 = min(n, p + turns - i), t0 = q4_first(c, len), jfirst = t0 / kTok;
    const long long row = (long long)b * c.Hkv + h;
    w.load_q(q + row * G * D, G, c.scale * kLog2e);
    w.reset();
    float* srow = scores != nullptr ? scores + (row * c.max_blocks * kTok + tok) * Gs : nullptr;
    for (; p < p1; ++p, ++i) {
      const int stage = i % S;
      const bool here = sm100::mbar_wait_bounded(&bars[warp][stage], (i / S) & 1, kWaitLimit);
      if (!__all_sync(0xffffffffu, here)) {  // wait, bounded, for the copies still under way, then stop
        if (lane == 0) report(status, kTimeout);
        for (int k = i + 1; k < min(turns, i + S); ++k)
          sm100::mbar_wait_bounded(&bars[warp][k % S], (k / S) & 1, kWaitLimit);
        return;
      }
      const uint8_t* ks = ring + stage * kStage;
      const int jb = jfirst + p * BT, at = jb * kTok;
      if (i % PER == 0) here_now = good;  // (copies run S - 1 < PER turns ahead: `good` is still this turn's)
      const unsigned ok = here_now >> (i % PER * BT) & ((1u << BT) - 1);
      float* sc = srow != nullptr ? srow + (long long)at * Gs : nullptr;
      if (ok == (1u << BT) - 1 && at >= t0 && at + BT * kTok <= len) {
        w.template turn<false>(ks, 0u, c.softcap, sc, Gs);
      } else {
        unsigned seen = 0;
#pragma unroll
        for (int k = 0; k < 2 * BT; ++k) {
          const int y = at + (k >> 1) * kTok + tok + 8 * (k & 1);
          seen |= (unsigned)((ok >> (k >> 1) & 1) && y >= t0 && y < len) << k;
          seen |= (unsigned)(y < len) << (8 + k);
        }
        w.template turn<true>(ks, seen, c.softcap, sc, Gs);
      }
      __syncwarp();  // every lane has read the stage
      issue(i + S);
    }
    // the part's sums: over the quads for l and z, the outputs are whole in each lane (8 or 4 dimensions of two heads)
    const long long slot = me + row;
    const bool whole = p0 == 0 && p1 == n;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int head = nt * 8 + 2 * t + e;
        float l = w.l[nt][e];
#pragma unroll
        for (int k = 4; k < 32; k <<= 1) l += __shfl_xor_sync(0xffffffffu, l, k);
        const float inv = l != 0.f ? 1.f / l : 0.f;
#pragma unroll
        for (int r = 0; r < W::NG; ++r) {
          float z = w.z[nt][r][e];
#pragma unroll
          for (int k = 4; k < 32; k <<= 1) z += __shfl_xor_sync(0xffffffffu, z, k);
          if (head >= G) continue;
          const int d = r * L::kGroup + g * W::MT * 2;
          float x[W::MT * 2];
#pragma unroll
          for (int k = 0; k < W::MT; ++k) {
            x[2 * k] = w.o[nt][r][k][e] + z;
            x[2 * k + 1] = w.o[nt][r][k][e + 2] + z;
          }
          if (whole) {
            __nv_bfloat16* dst = out + (row * G + head) * D + d;
#pragma unroll
            for (int k = 0; k < W::MT * 2; k += 2)
              *reinterpret_cast<__nv_bfloat162*>(dst + k) = __floats2bfloat162_rn(x[k] * inv, x[k + 1] * inv);
          } else {
            float* dst = part + (slot * G + head) * D + d;
#pragma unroll
            for (int k = 0; k < W::MT * 2; k += 4)
              *reinterpret_cast<float4*>(dst + k) = make_float4(x[k], x[k + 1], x[k + 2], x[k + 3]);
          }
        }
        if (g == 0 && head < G && (!whole || scores != nullptr))
          *reinterpret_cast<float2*>(ml + (slot * G + head) * 2) = make_float2(w.m[nt][e] + kDown, l);
      }
    if (p0 == 0 && lane == 0) {  // the row's first slot and its parts, for q4_finish_kernel
      const int last = base + h * n + n - 1;
      plan[row] = make_int2((int)slot, q4_owner(last, line.total, line.warps) - me + 1);
    }
    if (p == n) {  // the next row
      p = 0;
      if (++h == c.Hkv && i < turns) {
        h = 0;
        base += n * c.Hkv;
        do {
          len = q4_len(c, ++b, nullptr);
          n = q4_turns(c, len);
        } while (n == 0);
      }
    }
  }
}

// Maximum and 1 / sum of one query head over a row's parts; a whole warp calls it.  Where no block of the row was there
// to be read, its scores are all -inf: the maximum then is 0, and the weights 0.
RLB_DEVICE float2 q4_join(const float* ml, int G, int parts) {
  const int lane = threadIdx.x & 31;
  float M = -INFINITY, sum = 0.f;
#pragma unroll 4
  for (int s = lane; s < parts; s += 32) M = fmaxf(M, ml[2LL * s * G]);
  M = warp_max(M);
#pragma unroll 4
  for (int s = lane; s < parts; s += 32) {
    const float ms = ml[2LL * s * G], ls = ml[2LL * s * G + 1];
    sum += ms == -INFINITY ? ls : ls * sm100::ex2_approx(ms - M);
  }
  sum = warp_sum(sum);
  return make_float2(M == -INFINITY ? 0.f : M, sum != 0.f ? 1.f / sum : 0.f);
}

// Unnormalised output (dimensions lane + 32 e) and statistics of parts first, first + step, ... of one query head, by a
// whole warp, 8 parts at a time, relative to the largest maximum so far.  (A part that saw nothing has none: its
// sums are 0, or NaN.)
template <int D>
RLB_DEVICE float2 q4_add_parts(const float* part, const float* stats, int G, int first, int step, int parts,
                               float (&acc)[D / 32]) {
  constexpr int E = D / 32;
  const int lane = threadIdx.x & 31;
  float M = -INFINITY, sum = 0.f;
  for (int s0 = first; s0 < parts; s0 += 8 * step) {
    const int mine = s0 + step * (lane & 7);
    const float2 x = mine < parts ? *reinterpret_cast<const float2*>(stats + 2LL * mine * G) : make_float2(-INFINITY, 0.f);
    float a[8][E];
#pragma unroll
    for (int k = 0; k < 8; ++k)
#pragma unroll
      for (int e = 0; e < E; ++e)
        a[k][e] = s0 + step * k < parts ? part[(long long)(s0 + step * k) * G * D + lane + 32 * e] : 0.f;
    float m = x.x;
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    m = fmaxf(m, M);
    const float was = M == -INFINITY ? 1.f : sm100::ex2_approx(M - m);
    M = m;
    sum *= was;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] *= was;
    const float f = x.x == -INFINITY ? 1.f : sm100::ex2_approx(x.x - m), l = x.y * f;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      sum += __shfl_sync(0xffffffffu, l, k);
      const float fk = __shfl_sync(0xffffffffu, f, k);
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] += a[k][e] * fk;
    }
  }
  return make_float2(M, sum);
}

// Joins the parts of the rows that several warps of q4_decode_kernel shared, and writes zeros for empty sequences.
// WIDE: CTA z of a row does query head z, its eight warps taking the parts in turn (few rows, long contexts);
// otherwise a warp does a query head.  With `weights` the CTAs behind add a stretch each of the tokens' attention
// weights, summed over the heads, to their accumulators.  Bound by latency (plan, statistics, parts, output: 4 to 8 us
// alone, 2 to 5 behind the decode kernel's end).
template <int D, bool WIDE>
__global__ void __launch_bounds__(256) q4_finish_kernel(Q4Cache c, const float* __restrict__ part,
                                                        const float* __restrict__ ml, const int2* __restrict__ plan,
                                                        int slots, __nv_bfloat16* __restrict__ out,
                                                        const float* __restrict__ scores, int Gs,
                                                        float* __restrict__ weights,
                                                        const int* __restrict__ weight_rows, long long w_rows,
                                                        int w_len, int* status) {
  constexpr int E = D / 32;
  __shared__ float2 stat[16];
  cudaGridDependencySynchronize();  // (every CTA: what follows this kernel must not overtake the one before)
  const int h = blockIdx.x, b = blockIdx.y, z = blockIdx.z, G = c.G, joins = WIDE ? G : (G + 7) / 8;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long row = (long long)b * c.Hkv + h;
  const int len = q4_len(c, b, nullptr);
  const int2 at = len > 0 ? plan[row] : make_int2(0, 0);  // first slot, parts
  // (a decode kernel that gave up on a copy, and reported it, has left rows without a plan)
  if (at.x < 0 || at.y < (len > 0) || at.x >= slots || at.y > slots - at.x) return;
  const float* stats = ml + (long long)at.x * G * 2;
  if (z < joins) {
    const int head = WIDE ? z : z * 8 + warp;
    if (head >= G || at.y == 1) return;  // (one part: written already)
    __nv_bfloat16* dst = out + (row * G + head) * D;
    float acc[E] = {};
    const float* from = part + ((long long)at.x * G + head) * D;
    float2 s = q4_add_parts<D>(from, stats + 2 * head, G, WIDE ? warp : 0, WIDE ? 8 : 1, at.y, acc);
    if constexpr (!WIDE) {
      const float inv = s.y != 0.f ? 1.f / s.y : 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) dst[lane + 32 * e] = __float2bfloat16(acc[e] * inv);
    } else {
      __shared__ float sums[8][D];
#pragma unroll
      for (int e = 0; e < E; ++e) sums[warp][lane + 32 * e] = acc[e];
      if (lane == 0) stat[warp] = s;
      __syncthreads();
      float most = -INFINITY, total = 0.f, f[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) most = fmaxf(most, stat[i].x);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        f[i] = stat[i].x == -INFINITY ? 1.f : sm100::ex2_approx(stat[i].x - most);
        total += stat[i].y * f[i];
      }
      for (int d = threadIdx.x; d < D; d += 256) {
        float a = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) a += sums[i][d] * f[i];
        dst[d] = __float2bfloat16(total != 0.f ? a / total : 0.f);
      }
    }
    return;
  }
  if (len == 0) return;
  const int r = weight_rows[b];
  if (r < 0) return;
  if (threadIdx.x == 0 && z == joins && h == 0 && (r >= w_rows || len > w_len)) report(status, kBadIndex);
  if (r >= w_rows) return;
  for (int head = warp; head < G; head += 8) {
    const float2 x = q4_join(stats + 2 * head, G, at.y);
    if (lane == 0) stat[head] = x;
  }
  __syncthreads();
  float* w = weights + ((long long)r * c.Hkv + h) * w_len;
  const float* sc = scores + row * c.max_blocks * kTok * Gs;
  const int end = min(len, w_len);
  constexpr int U = 4;  // tokens a thread takes at a time
  for (long long t0 = q4_first(c, len) + (z - joins) * 256LL * U + threadIdx.x; t0 < end; t0 += (gridDim.z - joins) * 256LL * U) {
    float p[U] = {};
    for (int head = 0; head < G; head += 2) {
      float2 x[U];
#pragma unroll
      for (int i = 0; i < U; ++i)
        x[i] = t0 + 256 * i < end ? *reinterpret_cast<const float2*>(sc + (t0 + 256 * i) * Gs + head) : make_float2(0.f, 0.f);
      const float2 s0 = stat[head], s1 = stat[head + 1];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        p[i] += sm100::ex2_approx(x[i].x - s0.x) * s0.y;
        if (head + 1 < G) p[i] += sm100::ex2_approx(x[i].y - s1.x) * s1.y;
      }
    }
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (t0 + 256 * i < end && p[i] != 0.f) atomicAdd(w + t0 + 256 * i, p[i]);
  }
}

// ---------------------------------------------------------------- eviction
// Order-preserving key of a weight: larger keys for larger weights, -0 like +0, NaN below everything.
RLB_DEVICE uint32_t weight_key(float w) {
  if (w != w) return 0u;
  const uint32_t u = __float_as_uint(w + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// Choosing what stays has three forms.  This one, a CTA per (KV head, sequence), takes sequences whose weights do not fit
// into a CTA's registers, where they do not fit into a cluster's either or are too many rows for clusters.  The weight of the last kept token is found by a radix selection (11, 11 and 10 bits:
// a histogram in shared memory, whose bins a scan then walks from the top).  Each warp then takes a stretch of the
// tokens: it counts the tokens above that weight and those equal to it, a scan over the warps gives it its place, and
// it writes its kept positions in order.  The weights move to the front last, tile by tile: a token never moves to a
// higher place, so a tile is read before anything that a later one reads is written.
constexpr int kSelect = 1024, kTile = 8;  // threads; weights a thread moves at a time

__global__ void __launch_bounds__(kSelect) q4_select_kernel(const int* __restrict__ lens, float* __restrict__ weights,
                                                            const int* __restrict__ weight_rows,
                                                            int* __restrict__ kept, int* __restrict__ new_lens,
                                                            int Hkv, long long w_rows, int w_len, int keep, int recent,
                                                            int sink, int* status) {
  __shared__ int hist[2048], part[33], part2[33], pick[2];
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
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
    for (int j = tid; j < keep; j += kSelect) out[j] = j < n ? j : -1;
    return;
  }
  float* w = weights + ((long long)r * Hkv + h) * w_len;
  const int first = sink, last = n - recent;  // tokens [first, last) compete for `need` places
  int need = keep - sink - recent;
  const bool any = need > 0;
  uint32_t prefix = 0, known = 0;
  for (int step = 0; any && step < 3; ++step) {
    const int shift = step == 0 ? 21 : step == 1 ? 10 : 0, bins = step == 2 ? 1024 : 2048;
    hist[tid] = hist[tid + kSelect] = 0;
    __syncthreads();
#pragma unroll 8
    for (int t = first + tid; t < last; t += kSelect) {
      const uint32_t key = weight_key(w[t]);
      if ((key & known) == prefix) atomicAdd(&hist[(key >> shift) & (bins - 1)], 1);
    }
    __syncthreads();
    // this thread's two bins, counted from the top; how many lie in higher bins
    const int d = bins - 1 - 2 * tid;
    const int c0 = d > 0 ? hist[d] : 0, c1 = d > 0 ? hist[d - 1] : 0;
    int incl = c0 + c1;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += y;
    }
    if (lane == 31) part[warp] = incl;
    __syncthreads();
    int above = incl - c0 - c1;
    for (int i = 0; i < warp; ++i) above += part[i];
    if (above < need && need <= above + c0) {
      pick[0] = d;
      pick[1] = need - above;
    } else if (above + c0 < need && need <= above + c0 + c1) {
      pick[0] = d - 1;
      pick[1] = need - above - c0;
    }
    __syncthreads();
    prefix |= (uint32_t)pick[0] << shift;
    known |= (uint32_t)(bins - 1) << shift;
    need = pick[1];
  }
  // every competitor above `prefix` is kept, and the first `need` of those equal to it
  auto state = [&](int t, bool& tie) {  // whether token t is kept whatever the ties, and whether it is one
    tie = false;
    if (t >= n) return false;
    if (t < first || t >= last) return true;
    const uint32_t key = weight_key(w[t]);
    tie = any && key == prefix;
    return any && key > prefix;
  };
  const int per = (n + 32 * 32 - 1) / (32 * 32) * 32, s0 = min(n, warp * per), s1 = min(n, s0 + per);
  int sure = 0, ties = 0;
#pragma unroll 8
  for (int t = s0 + lane; t < s0 + per; t += 32) {
    bool tie;
    sure += state(t < s1 ? t : n, tie);
    ties += tie;
  }
  sure = __reduce_add_sync(0xffffffffu, sure);
  ties = __reduce_add_sync(0xffffffffu, ties);
  if (lane == 0) {
    part[warp] = sure;
    part2[warp] = ties;
  }
  __syncthreads();
  int done = 0, ties_before = 0;
  for (int i = 0; i < warp; ++i) {
    done += part[i];
    ties_before += part2[i];
  }
  done += min(need, ties_before);
  const unsigned below = (1u << lane) - 1;
#pragma unroll 4
  for (int t0 = s0; t0 < s1; t0 += 32) {
    bool tie;
    const bool keep_it = state(t0 + lane < s1 ? t0 + lane : n, tie);
    const unsigned tied = __ballot_sync(0xffffffffu, tie);
    const bool in = keep_it || (tie && ties_before + __popc(tied & below) < need);
    const unsigned all = __ballot_sync(0xffffffffu, in);
    if (in) out[done + __popc(all & below)] = t0 + lane;
    done += __popc(all);
    ties_before += __popc(tied);
  }
  __syncthreads();
  for (int j0 = 0; j0 < keep; j0 += kSelect * kTile) {
    float x[kTile];
#pragma unroll
    for (int i = 0; i < kTile; ++i) {
      const int j = j0 + i * kSelect + tid;
      x[i] = j < keep ? w[out[j]] : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kTile; ++i)
      if (j0 + i * kSelect + tid < keep) w[j0 + i * kSelect + tid] = x[i];
  }
  __syncthreads();  // (the last tile may have read from behind `keep`)
  for (int t = keep + tid; t < n; t += kSelect) w[t] = 0.f;
}

// The same with K keys a thread in registers: the weights are read once.  A bar that exactly `keep` keys reach is
// searched by halving the interval of keys and counting: 10 to 20 times K compares and a barrier (32 where many weights
// are equal), where histograms pay for colliding atomics, weights crowding in few exponents.  Warp w holds tokens
// [32 K w, 32 K (w + 1)), 32 neighbours at a time.  Bound by the chain of barriers (K 4: 128 rows of 4096 tokens in
// 10 us) and by the compares (K 40: 8 rows of 40000 in 41 us, up to 148 such rows in no more).
template <int K>
__global__ void __launch_bounds__(kSelect) q4_select_regs_kernel(const int* __restrict__ lens, float* __restrict__ weights,
                                                                 const int* __restrict__ weight_rows,
                                                                 int* __restrict__ kept, int* __restrict__ new_lens,
                                                                 int Hkv, long long w_rows, int w_len, int keep,
                                                                 int recent, int sink, int* status) {
  __shared__ int part[2][32], place[2][32];
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int n = lens[b];
  const int r = weight_rows[b];
  if (n > min(w_len, K * kSelect) || (n > 0 && (r < 0 || r >= w_rows))) {
    if (tid == 0) report(status, kBadIndex);
    n = 0;
  }
  n = max(n, 0);
  int* out = kept + ((long long)b * Hkv + h) * keep;
  if (h == 0 && tid == 0) new_lens[b] = min(n, keep);
  if (n <= keep) {
    for (int j = tid; j < keep; j += kSelect) out[j] = j < n ? j : -1;
    return;
  }
  float* w = weights + ((long long)r * Hkv + h) * w_len;
  const int t0 = warp * 32 * K + lane;
  uint32_t key[K];  // above all for protected tokens, 0 for absent ones (a NaN's is 1)
#pragma unroll
  for (int i = 0; i < K; ++i) key[i] = t0 + 32 * i < n ? __float_as_uint(w[t0 + 32 * i]) : 0u;
#pragma unroll
  for (int i = 0; i < K; ++i) {
    const int t = t0 + 32 * i;
    key[i] = t >= n ? 0u : t < sink || t >= n - recent ? 0xffffffffu : max(weight_key(__uint_as_float(key[i])), 1u);
  }
  int turn = 0;
  auto count = [&](uint32_t least) {  // keys of at least `least`, in the block
    int c = 0;
#pragma unroll
    for (int i = 0; i < K; ++i) c += key[i] >= least;
    c = __reduce_add_sync(0xffffffffu, c);
    if (lane == 0) part[turn & 1][warp] = c;
    __syncthreads();
    c = __reduce_add_sync(0xffffffffu, part[turn & 1][lane]);
    ++turn;
    return c;
  };
  // at_bar >= keep keys are at least `bar`, fewer at least `over`
  uint32_t bar = 1, over = 0xffffffffu;
  int at_bar = n;
  if (sink + recent == keep) {
    bar = over;
    at_bar = keep;
  }
  while (over - bar > 1 && at_bar > keep) {
    const uint32_t least = bar + (over - bar) / 2;
    const int c = count(least);
    if (c >= keep) {
      bar = least;
      at_bar = c;
    } else {
      over = least;
    }
  }
  const unsigned below = (1u << lane) - 1;
  if (at_bar > keep) {  // of the keys equal to the bar only the first find a place: the others fall below it
    const int taken = keep - count(bar + 1);
    int ties = 0;
#pragma unroll
    for (int i = 0; i < K; ++i) ties += key[i] == bar;
    ties = __reduce_add_sync(0xffffffffu, ties);
    if (lane == 0) place[1][warp] = ties;
    __syncthreads();
    int before = __reduce_add_sync(0xffffffffu, lane < warp ? place[1][lane] : 0);
#pragma unroll
    for (int i = 0; i < K; ++i) {
      const unsigned tied = __ballot_sync(0xffffffffu, key[i] == bar);
      if (key[i] == bar && before + __popc(tied & below) >= taken) key[i] = 0;
      before += __popc(tied);
    }
  }
  int mine = 0;
#pragma unroll
  for (int i = 0; i < K; ++i) mine += key[i] >= bar;
  mine = __reduce_add_sync(0xffffffffu, mine);
  if (lane == 0) place[0][warp] = mine;
  float x[K];  // the kept tokens' weights
  unsigned in[(K + 31) / 32] = {};
#pragma unroll
  for (int i = 0; i < K; ++i) {
    in[i / 32] |= (unsigned)(key[i] >= bar) << (i % 32);
    x[i] = key[i] >= bar ? w[t0 + 32 * i] : 0.f;
  }
  __syncthreads();  // every weight has been read
  int done = __reduce_add_sync(0xffffffffu, lane < warp ? place[0][lane] : 0);
#pragma unroll
  for (int i = 0; i < K; ++i) {
    const bool keep_it = in[i / 32] >> (i % 32) & 1;
    const unsigned all = __ballot_sync(0xffffffffu, keep_it);
    const int to = done + __popc(all & below);
    if (keep_it) {
      out[to] = t0 + 32 * i;
      w[to] = x[i];
    }
    done += __popc(all);
  }
  for (int t = keep + tid; t < n; t += kSelect) w[t] = 0.f;
}

// For few long sequences a cluster of 8 CTAs per (KV head, sequence), 16 keys a thread: there one CTA's loads and
// compares leave most SMs idle.  A barrier of the cluster costs above 1 us, so the bar is found in three turns (two where
// the second leaves no bin in part): each CTA counts its keys' digits (11, 11 and 10 bits) in a histogram of its own, and
// every CTA adds the eight up over distributed shared memory.  8 rows of 40000 tokens take 18 us (41 by one CTA each,
// 35 by clusters that halve the interval), 13 us more for each further 18 rows, as one cluster fills 8 SMs.
constexpr int kCtas = 8;
__global__ void __launch_bounds__(kSelect) q4_select_cluster_kernel(const int* __restrict__ lens,
                                                                    float* __restrict__ weights,
                                                                    const int* __restrict__ weight_rows,
                                                                    int* __restrict__ kept, int* __restrict__ new_lens,
                                                                    int Hkv, long long w_rows, int w_len, int keep,
                                                                    int recent, int sink, int* status) {
  constexpr int K = 16, threads = kCtas * kSelect;
  __shared__ __align__(8) int hist[3][2048];
  __shared__ int part[32], place[32], pick[2], sums[2];
  cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
  const int h = blockIdx.x / kCtas, rank = blockIdx.x % kCtas, b = blockIdx.y;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, me = rank * kSelect + tid;
  int n = lens[b];
  const int r = weight_rows[b];
  if (n > min(w_len, K * threads) || (n > 0 && (r < 0 || r >= w_rows))) {
    if (me == 0) report(status, kBadIndex);
    n = 0;
  }
  n = max(n, 0);
  int* out = kept + ((long long)b * Hkv + h) * keep;
  if (h == 0 && me == 0) new_lens[b] = min(n, keep);
  if (n <= keep) {
    for (int j = me; j < keep; j += threads) out[j] = j < n ? j : -1;
    return;  // (the whole cluster)
  }
  float* w = weights + ((long long)r * Hkv + h) * w_len;
  const int used = (n + threads - 1) / threads;  // keys that a thread holds
  const int t0 = (rank * 32 + warp) * 32 * used + lane;
  float x[K];
#pragma unroll
  for (int i = 0; i < K; ++i) x[i] = i < used && t0 + 32 * i < n ? w[t0 + 32 * i] : 0.f;
#pragma unroll
  for (int i = 0; i < 6; ++i) (&hist[0][0])[tid + i * kSelect] = 0;
  auto key_of = [&](int i) {  // above all for protected tokens, 0 for absent ones (a NaN's is 1)
    const int t = t0 + 32 * i;
    return i >= used || t >= n ? 0u : t < sink || t >= n - recent ? 0xffffffffu : max(weight_key(x[i]), 1u);
  };
  __syncthreads();
  // Of the keys that agree with `bar` in the bits `known` (none at first), `need` are kept, and all above them.
  uint32_t bar = 0, known = 0;
  int need = keep;
  bool whole = false;
  for (int step = 0; step < 3 && !whole; ++step) {
    const int shift = step == 0 ? 21 : step == 1 ? 10 : 0, bins = step == 2 ? 1024 : 2048;
#pragma unroll
    for (int i = 0; i < K; ++i) {
      if (i >= used) break;
      const uint32_t key = key_of(i);
      if (key != 0 && (key & known) == bar) atomicAdd(&hist[step][(key >> shift) & (bins - 1)], 1);
    }
    cluster.sync();
    // this thread's two bins, counted from the top; how many lie in higher bins
    const int d = bins - 1 - 2 * tid;
    int c0 = 0, c1 = 0;
    if (d > 0)
#pragma unroll
      for (int i = 0; i < kCtas; ++i) {
        const int2 two = *reinterpret_cast<const int2*>(cluster.map_shared_rank(&hist[step][d - 1], i));
        c1 += two.x;
        c0 += two.y;
      }
    int incl = c0 + c1;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += y;
    }
    if (lane == 31) part[warp] = incl;
    __syncthreads();
    const int above = incl - c0 - c1 + __reduce_add_sync(0xffffffffu, lane < warp ? part[lane] : 0);
    if (above < need && need <= above + c0) {
      pick[0] = d;
      pick[1] = need - above;
      sums[0] = c0;
    } else if (above + c0 < need && need <= above + c0 + c1) {
      pick[0] = d - 1;
      pick[1] = need - above - c0;
      sums[0] = c1;
    }
    __syncthreads();
    bar |= (uint32_t)pick[0] << shift;
    known |= (uint32_t)(bins - 1) << shift;
    need = pick[1];
    whole = need == sums[0];
  }
  const unsigned below = (1u << lane) - 1;
  // Sums over the warps before this one: in the cluster for the tied keys (only if some of them go), then for the kept.
  auto before_me = [&](int mine, int& slot) {
    mine = __reduce_add_sync(0xffffffffu, mine);
    if (lane == 0) place[warp] = mine;
    __syncthreads();
    const int all = __reduce_add_sync(0xffffffffu, place[lane]);
    int ahead = __reduce_add_sync(0xffffffffu, lane < warp ? place[lane] : 0);
    if (tid == 0) slot = all;
    cluster.sync();
    return ahead + __reduce_add_sync(0xffffffffu, lane < rank ? *cluster.map_shared_rank(&slot, lane) : 0);
  };
  unsigned in = 0;
  if (whole) {
#pragma unroll
    for (int i = 0; i < K; ++i) in |= (unsigned)(key_of(i) >= bar) << i;
  } else {
    int ties = 0;
#pragma unroll
    for (int i = 0; i < K; ++i) ties += key_of(i) == bar;
    int before = before_me(ties, sums[1]);
#pragma unroll
    for (int i = 0; i < K; ++i) {
      if (i >= used) break;
      const uint32_t key = key_of(i);
      const unsigned tied = __ballot_sync(0xffffffffu, key == bar);
      in |= (unsigned)(key > bar || (key == bar && before + __popc(tied & below) < need)) << i;
      before += __popc(tied);
    }
  }
  int done = before_me(__popc(in), pick[0]);  // every weight has been read by then
#pragma unroll
  for (int i = 0; i < K; ++i) {
    if (i >= used) break;
    const unsigned all = __ballot_sync(0xffffffffu, in >> i & 1);
    const int to = done + __popc(all & below);
    if (in >> i & 1) {
      out[to] = t0 + 32 * i;
      w[to] = x[i];
    }
    done += __popc(all);
  }
  for (int t = keep + me; t < n; t += threads) w[t] = 0.f;
  cluster.sync();  // the others' shared memory is still read until here
}

// Moves the kept tokens' stored rows (codes and scales) to the new blocks: 16 bytes of a key and of a value a thread, and
// nothing shared, so that all reads are in flight at once.  Kept rows lie 32 bytes here and there: 16 x 1024 rows of
// 8 x 128 in 12 us (38 MB read and written, 3.2 TB/s), of which about 4 are the chain of tables, positions and rows.
template <int D>
__global__ void __launch_bounds__(256) q4_move_kernel(uint8_t* k_pool, uint8_t* v_pool, const int* __restrict__ tables,
                                                      const int* __restrict__ new_tables, const int* __restrict__ kept,
                                                      const int* __restrict__ new_lens, int Hkv, int max_blocks,
                                                      int new_blocks, int num_blocks, int keep, int* status) {
  using L = Q4<D>;
  constexpr int UNITS = L::kRow / 16;                  // 16-byte units of a token in a group
  constexpr int PER = kTok * UNITS * L::kGroups;       // threads for a block
  const int h = blockIdx.y, b = blockIdx.z, len = new_lens[b];
  const int nb = blockIdx.x * (256 / PER) + threadIdx.x / PER, x = threadIdx.x % PER;
  const int unit = x % UNITS, slot = x / UNITS % kTok, grp = x / UNITS / kTok, j = nb * kTok + slot;
  if (j >= len) return;
  const int t = kept[((long long)b * Hkv + h) * keep + j];
  const int to = new_tables[(long long)b * new_blocks + nb];
  const int from = t >= 0 && t / kTok < max_blocks ? tables[(long long)b * max_blocks + t / kTok] : -1;
  if (from < 0 || from >= num_blocks || to < 0 || to >= num_blocks) {
    report(status, kBadIndex);
    return;
  }
  const int off = t % kTok;
  const long long src = ((long long)from * Hkv + h) * L::kBytes, dst = ((long long)to * Hkv + h) * L::kBytes;
  const int code_from = (grp * kTok + off) * L::kRow + unit * 16, code_to = (grp * kTok + slot) * L::kRow + unit * 16;
  const uint4 k = *reinterpret_cast<const uint4*>(k_pool + src + code_from);
  const uint4 v = *reinterpret_cast<const uint4*>(v_pool + src + code_from);
  *reinterpret_cast<uint4*>(k_pool + dst + code_to) = k;
  *reinterpret_cast<uint4*>(v_pool + dst + code_to) = v;
  if (unit == 0) {
    const int meta_from = L::kCodes + (grp * kTok + off) * 4, meta_to = L::kCodes + (grp * kTok + slot) * 4;
    const uint32_t km = *reinterpret_cast<const uint32_t*>(k_pool + src + meta_from);
    const uint32_t vm = *reinterpret_cast<const uint32_t*>(v_pool + src + meta_from);
    *reinterpret_cast<uint32_t*>(k_pool + dst + meta_to) = km;
    *reinterpret_cast<uint32_t*>(v_pool + dst + meta_to) = vm;
  }
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
  const long long chunks = (N + 4096 / D - 1) / (4096 / D);
  const dim3 grid(Hkv, (unsigned)(chunks < 65535 ? chunks : 65535));
  RLB_Q4_D((q4_write_kernel<DD><<<grid, 256, 0, s>>>(
      (const __nv_bfloat16*)k_new, (const __nv_bfloat16*)v_new, k_sn, k_sh, v_sn, v_sh, (uint8_t*)k_pool,
      (uint8_t*)v_pool, slot_block, slot_off, N, num_blocks, status)));
  return cudaGetLastError();
}

cudaError_t rlb_q4_read(const void* k_pool, const void* v_pool, const int* slot_block, const int* slot_off,
                        const int* tables, const int* lens, int max_blocks, int max_len, long long N, int Hkv, int D,
                        int num_blocks, void* k_out, void* v_out, int* status, cudaStream_t s) {
  if (N == 0) return cudaSuccess;
  const long long chunks = (N + 2048 / D - 1) / (2048 / D);
  const dim3 grid(Hkv, (unsigned)(chunks < 65535 ? chunks : 65535));
  RLB_Q4_D((q4_read_kernel<DD><<<grid, 256, 0, s>>>((const uint8_t*)k_pool, (const uint8_t*)v_pool, slot_block,
                                                    slot_off, tables, lens, max_blocks, max_len, N, num_blocks,
                                                    (__nv_bfloat16*)k_out, (__nv_bfloat16*)v_out, status)));
  return cudaGetLastError();
}

template <int D, int NT>
static cudaError_t q4_decode_launch(const void* q, const Q4Cache& c, void* out, int B, int C, float* part, float* ml,
                                    int2* plan, float* scores, int Gs, int* status, cudaStream_t s) {
  constexpr int smem = kDecodeWarps * q4_stages<D>() * q4_turn<D>() * 2 * Q4<D>::kBytes;
  static_assert(smem <= 47 * 1024, "above 48 KB a kernel has to ask for its shared memory");
  q4_decode_kernel<D, NT><<<C, kDecodeWarps * 32, smem, s>>>((const __nv_bfloat16*)q, c, B, (__nv_bfloat16*)out, part,
                                                              ml, plan, scores, Gs, status);
  return cudaGetLastError();
}

static int q4_turn_of(int D) { return D == 128 ? q4_turn<128>() : q4_turn<64>(); }

int rlb_q4_decode_ctas(int B, int Hkv, int G, int D, int max_blocks, int sms) {
  // As many CTAs as fit at a time, but a turn for each warp if the tables are full.
  const long long fit = (long long)sms * q4_ctas(D, G <= 8 ? 1 : 2);
  const long long turns = (long long)B * Hkv * ((max_blocks + q4_turn_of(D) - 1) / q4_turn_of(D));
  const long long want = (turns + kDecodeWarps - 1) / kDecodeWarps;
  return (int)(want < 1 ? 1 : want < fit ? want : fit);
}

cudaError_t rlb_q4_decode(const void* q, const void* k_pool, const void* v_pool, const int* tables, const int* lens,
                          void* out, int B, int Hkv, int G, int D, int max_blocks, int num_blocks, float scale,
                          float softcap, int window, int ctas, float* scratch, bool weighted, float* weights,
                          const int* weight_rows, long long w_rows, int w_len, int sms, int* status, cudaStream_t s) {
  if (B == 0) return cudaSuccess;
  // the kernel counts turns and blocks of all heads in 32 bits
  if ((long long)B * Hkv * ((max_blocks + q4_turn_of(D) - 1) / q4_turn_of(D)) >= (1LL << 31) - (1 << 20) ||
      (long long)num_blocks * Hkv >= 1LL << 31 ||
      (long long)ctas * kDecodeWarps + (long long)B * Hkv >= 1LL << 31)
    return cudaErrorInvalidValue;
  const Q4Cache c{(const uint8_t*)k_pool, (const uint8_t*)v_pool, tables, lens, Hkv, G, max_blocks, num_blocks,
                  window, q4_turn_of(D), scale, softcap};
  const int Gs = (G + 1) & ~1;
  const long long slots = (long long)ctas * kDecodeWarps + (long long)B * Hkv;
  float* scores = weighted ? scratch : nullptr;  // first: written in pairs
  if (weighted) scratch += (long long)B * Hkv * max_blocks * kTok * Gs;
  float* part = scratch;  // 16-byte pieces
  float* ml = part + slots * G * D;
  int2* plan = (int2*)(ml + slots * G * 2);
  cudaError_t e = cudaSuccess;
  RLB_Q4_D(e = G <= 8 ? (q4_decode_launch<DD, 1>(q, c, out, B, ctas, part, ml, plan, scores, Gs, status, s))
                      : (q4_decode_launch<DD, 2>(q, c, out, B, ctas, part, ml, plan, scores, Gs, status, s)));
  if (e != cudaSuccess) return e;
  // CTAs per row that add weights: one wave of the GPU, 1024 tokens each at least (192 rows of 5000 tokens and 4 heads:
  // 11 us with the join; four waves of 256 tokens at a time, each reading the statistics again, took 19)
  int chunks = 0;
  if (weighted) {
    const long long rows = (long long)B * Hkv, want = (8LL * sms + rows - 1) / rows;
    const long long most = ((long long)max_blocks * kTok + 1023) / 1024;
    chunks = (int)(want < most ? want : most);
    if (chunks < 1) chunks = 1;
  }
  // launched while the decode kernel still runs; it waits for that one's end itself
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  // wide where more than about 6 parts fall on a row (at 7, 32 x 8192 tokens of 128: 8.6 us wide, 10.4 narrow; at 4.6,
  // 64 x 4096 of 64: 9.7 wide, 7.2 narrow)
  const bool wide = (long long)ctas * kDecodeWarps > 6LL * B * Hkv;
  cfg.gridDim = dim3(Hkv, B, (wide ? G : (G + 7) / 8) + chunks);
  cfg.blockDim = dim3(256);
  cfg.stream = s;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  RLB_Q4_D(e = cudaLaunchKernelEx(&cfg, wide ? q4_finish_kernel<DD, true> : q4_finish_kernel<DD, false>, c, (const float*)part, (const float*)ml, (const int2*)plan, (int)slots,
                                  (__nv_bfloat16*)out, (const float*)scores, Gs, weights, weight_rows, w_rows, w_len,
                                  status));
  return e;
}

long long rlb_q4_decode_scratch(int B, int Hkv, int G, int D, int max_blocks, int ctas, bool weighted) {
  const long long rows = (long long)B * Hkv;
  return (weighted ? rows * max_blocks * kTok * ((G + 1) & ~1) : 0) + 2 * rows + (ctas * (long long)kDecodeWarps + rows) * G * (D + 2);
}

cudaError_t rlb_q4_evict(void* k_pool, void* v_pool, const int* tables, const int* lens, const int* new_tables,
                         float* weights, const int* weight_rows, int* kept, int* new_lens, int B, int Hkv, int D,
                         int max_blocks, int new_blocks, int num_blocks, long long w_rows, int w_len, int keep,
                         int recent, int sink, int* status, cudaStream_t s) {
  if (B == 0) return cudaSuccess;
  const long long most = (long long)max_blocks * kTok < w_len ? (long long)max_blocks * kTok : w_len;  // tokens
  // Clusters while their rows take less than one CTA each does: up to 40960 tokens, keys in registers, rows x 0.9 us and
  // up against 41; beyond, in us of the whole call by clusters and by one CTA a row: 8 rows of 60000 tokens 35 and 80, 64
  // rows 94 and 85, 256 rows 297 and 145, 64 rows of 100000 110 and 122.  (Above 131072 tokens one CTA a row is all there
  // is: 8 or 64 rows of 140000 take 160, 8 rows of 400000 405.)
  const bool few = (long long)B * Hkv <= (most > 40 * kSelect ? 64 : 32);
  if (few && most > 16 * kSelect && most <= 16 * kSelect * kCtas) {
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = kCtas;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(Hkv * kCtas, B);
    cfg.blockDim = dim3(kSelect);
    cfg.stream = s;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, q4_select_cluster_kernel, lens, weights, weight_rows, kept, new_lens,
                                             Hkv, w_rows, w_len, keep, recent, sink, status);
    if (e != cudaSuccess) return e;
  } else {
    auto select = most <= 4 * kSelect    ? q4_select_regs_kernel<4>
                  : most <= 16 * kSelect ? q4_select_regs_kernel<16>
                  : most <= 40 * kSelect ? q4_select_regs_kernel<40>  // (64 registers a thread hold no more)
                                         : q4_select_kernel;
    select<<<dim3(Hkv, B), kSelect, 0, s>>>(lens, weights, weight_rows, kept, new_lens, Hkv, w_rows, w_len, keep,
                                            recent, sink, status);
  }
  const int rows = (keep + kTok - 1) / kTok * kTok;  // the new blocks that can hold a token
  RLB_Q4_D((q4_move_kernel<DD><<<dim3((unsigned)(((long long)rows * Q4<DD>::kGroups * (Q4<DD>::kRow / 16) + 255) / 256), Hkv, B),
                                 256, 0, s>>>((uint8_t*)k_pool, (uint8_t*)v_pool, tables, new_tables, kept, new_lens,
                                              Hkv, max_blocks, new_blocks, num_blocks, keep, status)));
  return cudaGetLastError();
}
