// Attention of one new token per sequence over the paged MX key-value cache (kv_rows.cuh).
//
//   s_j = scale * sum_d q_d k_jd,  j < length;   o = sum_j exp(s_j) v_j / sum_j exp(s_j);
//   lse = log sum_j exp(s_j);  length 0: o = 0, lse = -inf.
//
// Every key-value head is read once for all the query heads that share it (up to 8 * NT of them
// to a block), so the kernel is bound by the cache's bytes: 2 * D * (8 or 4) / 8 + D / 16 per key.
// One pass: running maximum and sum of the softmax in fp32, sums of o in fp32.
//
// A warp works on tiles of 16 keys and holds everything in registers; the codes come by plain
// loads straight into the lanes that need them as MMA operands, so there is no shared memory and
// no wait in the loop.  With lane = 4 g + t:
//   scores  S^T[key][head] = K Q^T, K as the 16-row operand (m16n8k16, f16).  Lane (g, t) holds,
//           of keys g and g + 8, the 8 values 32 b + 8 t .. + 7 of each 32-value group b.  The
//           codes convert exactly to f16; q is scaled per head by a power of two so that f16
//           holds every bf16 bit of it, and each group's fp32 partial is multiplied by the key's
//           scale.
//   output  O^T[d][head] = V^T P^T, V as the 16-row operand (m16n8k16, bf16).  Lane (g, t) holds,
//           of keys 2t, 2t+1, 2t+8, 2t+9, the D / 8 values from g D / 8 on: all in one 32-value
//           group, so one scale byte per key.  The codes become bf16 by moving their fields into
//           place, which is the value times 2^-120 (E4M3) or 2^-126 (E2M1), and one exact multiply by
//           scale * 2^64, which leaves v * 2^-kCarry (kCarry = 56 or 62); p carries 2^kCarry.
//           bf16 has the range for any scale below 2^64 whatever the other keys' scales are;
//           larger ones count as 2^63.
//           The transposition between S^T's accumulators and P^T's operand is one
//           movmatrix per 8 keys.
//
// The sequences are cut into units of 4 warps * KT tiles; every block takes an equal, contiguous
// share of all units in (sequence, kv head, head chunk) order, whatever the lengths are (they are
// read on the device).  A head whose units lie in one block is written at once; the parts of the
// others go to the workspace and attn_join_kernel adds them in the blocks' order.
#pragma once

#include "common.cuh"
#include "gemm_small.cuh"
#include "kv_rows.cuh"

namespace mxb {

constexpr int kAttnWarps = 4;
constexpr int kAttnThreads = 32 * kAttnWarps;

// Tiles of 16 keys a warp takes per step: about 32 registers each of K and V codes in flight.
__host__ __device__ constexpr int attn_tiles(int dim, int fmt, int nt) {
  const int t = (fmt == kFmtE4M3 ? 256 : 512) / dim / nt;
  return t < 1 ? 1 : (t > 4 ? 4 : t);
}
__host__ __device__ constexpr int attn_unit_keys(int dim, int fmt, int nt) {
  return 16 * kAttnWarps * attn_tiles(dim, fmt, nt);
}

// Blocks resident per SM (the kernel's launch bound).
__host__ __device__ constexpr int attn_resident(int dim, int nt) { return dim == 256 || nt == 2 ? 2 : 3; }

struct AttnArgs {
  const __nv_bfloat16* q;  // [seqs][q_heads][dim], rows q_stride apart
  long long q_stride;
  KvCacheView cache;
  const int* table;        // [seqs][max_pages], rows table_stride apart
  long long table_stride;
  int max_pages;
  const int* lengths;
  int seqs, q_heads, group, chunks;  // group = q heads per kv head, in chunks of 8 * NT
  float scale;
  __nv_bfloat16* out;      // [seqs][q_heads][dim]
  float* lse;              // [seqs][q_heads] or null
  float* parts;            // [blocks][2][8 * NT heads][dim + 2]
  int blocks;              // of the main kernel
};

__device__ __forceinline__ void mma_bf16_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                               uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ float exp2_approx(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Length of a sequence in keys, within what its page table can hold.
__device__ __forceinline__ int attn_length(const AttnArgs& a, int b) {
  const int len = __ldg(a.lengths + b);
  const long long most = static_cast<long long>(a.max_pages) << a.cache.page_shift;
  if (len > most) {
    record_error(kErrBadLength);
    return static_cast<int>(most);
  }
  return len < 0 ? 0 : len;
}

// Units of all sequences, and of those before sequence `before` (block-wide; red: 2 * warps words).
__device__ __forceinline__ void attn_count_units(const AttnArgs& a, int unit_keys, int before, long long& total,
                                                 long long& ahead, long long* red) {
  long long s = 0, p = 0;
  for (int b = threadIdx.x; b < a.seqs; b += blockDim.x) {
    const long long u = (attn_length(a, b) + unit_keys - 1) / unit_keys;
    s += u;
    if (b < before) p += u;
  }
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, m);
    p += __shfl_xor_sync(0xffffffffu, p, m);
  }
  const int w = threadIdx.x >> 5, n = blockDim.x >> 5;
  if ((threadIdx.x & 31) == 0) red[w] = s, red[n + w] = p;
  __syncthreads();
  total = ahead = 0;
  for (int i = 0; i < n; ++i) total += red[i], ahead += red[n + i];
  __syncthreads();
  const long long per = static_cast<long long>(a.cache.heads) * a.chunks;
  total *= per;
  ahead *= per;
}

__device__ __forceinline__ long long attn_share(long long total, int blocks) { return (total + blocks - 1) / blocks; }

// Finds the sequence that unit u of all units lies in, and the unit index at which it begins.
// One warp; u < total.
__device__ __forceinline__ void attn_find(const AttnArgs& a, int unit_keys, long long u, int& seq, long long& begin) {
  const long long per = static_cast<long long>(a.cache.heads) * a.chunks;
  const int lane = threadIdx.x & 31;
  long long base = 0;
  for (int b0 = 0; b0 < a.seqs; b0 += 32) {
    long long n = b0 + lane < a.seqs ? (attn_length(a, b0 + lane) + unit_keys - 1) / unit_keys * per : 0;
    long long run = n;
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
      const long long o = __shfl_up_sync(0xffffffffu, run, m);
      if (lane >= m) run += o;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, base + run > u);
    if (hit) {
      const int f = __ffs(hit) - 1;
      seq = b0 + f;
      begin = base + __shfl_sync(0xffffffffu, run - n, f);
      return;
    }
    base += __shfl_sync(0xffffffffu, run, 31);
  }
  seq = a.seqs;
  begin = base;
}

template <int D, int kFmt>
struct AttnTile {
  static constexpr int kGroups = D / 32;
  static constexpr int kKWords = kFmt == kFmtE4M3 ? D / 8 : D / 16;  // words of K codes a lane holds, 2 keys
  static constexpr int kVWords = kFmt == kFmtE4M3 ? D / 8 : D / 16;  // words of V codes a lane holds, 4 keys
  uint32_t k[kKWords];        // [key g / g+8][group][words]
  uint32_t ks[2][(kGroups + 3) / 4];
  uint32_t v[kVWords];        // [key 2t, 2t+1, 2t+8, 2t+9][words]
  uint32_t vs[4];
};

template <int kWords>
__device__ __forceinline__ void load_words(const uint8_t* p, uint32_t* w) {
  if constexpr (kWords % 4 == 0) {
#pragma unroll
    for (int i = 0; i < kWords; i += 4) {
      const uint4 u = __ldg(reinterpret_cast<const uint4*>(p + 4 * i));
      w[i] = u.x, w[i + 1] = u.y, w[i + 2] = u.z, w[i + 3] = u.w;
    }
  } else if constexpr (kWords == 2) {
    const uint2 u = __ldg(reinterpret_cast<const uint2*>(p));
    w[0] = u.x, w[1] = u.y;
  } else {
    static_assert(kWords == 1, "");
    w[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
  }
}

// K codes and scales of the 16 keys whose first cache row is `row`.
template <int D, int kFmt>
__device__ __forceinline__ void load_k(const KvCacheView& c, size_t row, AttnTile<D, kFmt>& x) {
  using T = AttnTile<D, kFmt>;
  constexpr int kRowBytes = kFmt == kFmtE4M3 ? D : D / 2, kGroupBytes = kRowBytes / T::kGroups;
  constexpr int kW = kGroupBytes / 16;  // words per lane and group: 2 (E4M3) or 1
  const int g = (threadIdx.x & 31) >> 2, t = threadIdx.x & 3;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const size_t r = row + g + 8 * h;
#pragma unroll
    for (int b = 0; b < T::kGroups; ++b)
      load_words<kW>(c.k_codes + r * kRowBytes + b * kGroupBytes + 4 * kW * t, x.k + (h * T::kGroups + b) * kW);
    const uint8_t* s = c.k_scales + r * T::kGroups;
    if constexpr (T::kGroups == 2) x.ks[h][0] = __ldg(reinterpret_cast<const uint16_t*>(s));
    else load_words<T::kGroups / 4>(s, x.ks[h]);
  }
}

template <int D, int kFmt>
__device__ __forceinline__ void load_v(const KvCacheView& c, size_t row, AttnTile<D, kFmt>& x) {
  using T = AttnTile<D, kFmt>;
  constexpr int kRowBytes = kFmt == kFmtE4M3 ? D : D / 2, kW = kRowBytes / 32;  // words per lane and key
  const int g = (threadIdx.x & 31) >> 2, t = threadIdx.x & 3;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const size_t r = row + 2 * t + (j & 1) + 8 * (j >> 1);
    load_words<kW>(c.v_codes + r * kRowBytes + 4 * kW * g, x.v + j * kW);
    x.vs[j] = __ldg(c.v_scales + r * T::kGroups + (g * D / 8) / 32);
  }
}

// bf16x2 multiplier of two keys' scale bytes (see kCarry at the top): 2^(b - 63), 255 is NaN.
__device__ __forceinline__ uint32_t v_factor(uint32_t b) {
  return b == 255u ? 0x7FC0u : (min(b + 64u, 254u) << 7);
}

// V operand words of one pair of keys: for each of the lane's D / 8 values, (key a, key b) as
// bf16x2 times the keys' factors.
template <int D, int kFmt>
__device__ __forceinline__ void v_pairs(const uint32_t* a, const uint32_t* b, uint32_t factor, uint32_t (&o)[D / 8]) {
  if constexpr (kFmt == kFmtE4M3) {
#pragma unroll
    for (int i = 0; i < D / 8; ++i) {
      // the two codes in the high bytes of the halves; low bytes are masked away
      const uint32_t x = prmt(a[i / 4], b[i / 4], ((4 + (i & 3)) << 12) | ((i & 3) << 4));
      o[i] = mul_bf16x2(((x >> 4) & 0x07F007F0u) | (x & 0x80008000u), factor);
    }
  } else {
#pragma unroll
    for (int i = 0; i < D / 8; i += 4) {
      // four nibbles of key a in the low half, of key b in the high half
      const uint32_t z = prmt(a[i / 8], b[i / 8], (i & 4) ? 0x7632 : 0x5410);
      o[i] = mul_bf16x2(((z << 6) & 0x01C001C0u) | ((z << 12) & 0x80008000u), factor);
      o[i + 1] = mul_bf16x2(((z << 2) & 0x01C001C0u) | ((z << 8) & 0x80008000u), factor);
      o[i + 2] = mul_bf16x2(((z >> 2) & 0x01C001C0u) | ((z << 4) & 0x80008000u), factor);
      o[i + 3] = mul_bf16x2(((z >> 6) & 0x01C001C0u) | (z & 0x80008000u), factor);
    }
  }
}

template <int D, int kFmt, int NT>
__global__ void __launch_bounds__(kAttnThreads, attn_resident(D, NT)) attn_kernel(const __grid_constant__ AttnArgs a) {
  using T = AttnTile<D, kFmt>;
  constexpr int KT = attn_tiles(D, kFmt, NT);
  constexpr int kUnitTiles = kAttnWarps * KT, kUnitKeys = 16 * kUnitTiles;
  constexpr int kGroups = D / 32, kHeads = 8 * NT;
  constexpr float kCarry = kFmt == kFmtE4M3 ? 56.0f : 62.0f;  // p carries 2^kCarry, v 2^-kCarry
  constexpr int kStride = D + 4;                              // floats per head of a warp's part in shared memory
  constexpr float kInf = __builtin_huge_valf();
  extern __shared__ float sm[];                               // [warps][kHeads][kStride], then m, l [warps][kHeads]
  float* sm_m = sm + kAttnWarps * kHeads * kStride;
  float* sm_l = sm_m + kAttnWarps * kHeads;
  __shared__ long long red[2 * kAttnWarps];

  griddep_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;

  long long total, none;
  attn_count_units(a, kUnitKeys, 0, total, none, red);
  const long long share = attn_share(total, a.blocks);
  long long u = share * blockIdx.x;
  const long long u_end = min(u + share, total);
  if (u >= u_end) return;
  int seq;
  long long begin;
  attn_find(a, kUnitKeys, u, seq, begin);

  while (u < u_end) {
    // the segment: units [first, last) of head (seq, head, chunk)
    const int len = attn_length(a, seq);
    const int units = (len + kUnitKeys - 1) / kUnitKeys;
    if (units == 0) {
      ++seq;
      continue;
    }
    const int hc = static_cast<int>((u - begin) / units);
    const int first = static_cast<int>((u - begin) - static_cast<long long>(hc) * units);
    const int last = static_cast<int>(min(static_cast<long long>(units), first + (u_end - u)));
    const int head = hc / a.chunks, chunk = hc - head * a.chunks;
    const int h0 = head * a.group + chunk * kHeads;                  // first q head
    const int nh = min(kHeads, a.group - chunk * kHeads);            // q heads here
    const int* table = a.table + a.table_stride * seq;
    const int tiles = (len + 15) >> 4;

    // the cache row of a tile's first key, or -1 if there is none
    const int tile_shift = a.cache.page_shift - 4;
    auto tile_row = [&](int tile) -> long long {
      if (tile >= tiles) return -1;
      const int page = __ldg(table + (tile >> tile_shift));
      if (page < 0 || page >= a.cache.num_pages) {
        record_error(kErrBadPage);
        return -1;
      }
      return (((static_cast<long long>(page) * a.cache.heads + head) << a.cache.page_shift) +
              ((tile & ((1 << tile_shift) - 1)) << 4));
    };

    // Q operand: head g of n-tile n, values 32 b + 8 t .. + 7, scaled into f16
    uint32_t q[NT][kGroups][4];
    float mult[NT][2];  // of heads 2t, 2t+1: scale * log2(e) / the power of two
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const bool real = 8 * n + g < nh;
      const __nv_bfloat16* src = a.q + a.q_stride * seq + static_cast<size_t>(h0 + 8 * n + g) * D + 8 * t;
      uint32_t amax = 0;
#pragma unroll
      for (int b = 0; b < kGroups; ++b) {
        uint4 x = make_uint4(0, 0, 0, 0);
        if (real) x = *reinterpret_cast<const uint4*>(src + 32 * b);
        q[n][b][0] = x.x, q[n][b][1] = x.y, q[n][b][2] = x.z, q[n][b][3] = x.w;
#pragma unroll
        for (int i = 0; i < 4; ++i) amax = max(amax, max(q[n][b][i] & 0x7FFFu, (q[n][b][i] >> 16) & 0x7FFFu));
      }
      amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      // largest |q| into [2^14, 2^15): shift = 14 - floor(log2), at most 114
      const int shift = 14 + 127 - max(static_cast<int>(amax >> 7), 27);
      const float two = __uint_as_float(static_cast<uint32_t>(shift + 127) << 23);
#pragma unroll
      for (int b = 0; b < kGroups; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const __half2 h = __floats2half2_rn(__uint_as_float(q[n][b][i] << 16) * two,
                                              __uint_as_float(q[n][b][i] & 0xFFFF0000u) * two);
          q[n][b][i] = *reinterpret_cast<const uint32_t*>(&h);
        }
      const float back = a.scale * 1.4426950408889634f * __uint_as_float(static_cast<uint32_t>(127 - shift) << 23);
#pragma unroll
      for (int j = 0; j < 2; ++j) mult[n][j] = __shfl_sync(0xffffffffu, back, 4 * (2 * t + j));
    }

    float acc[D / 16][NT][4];
    float m[NT][2], lsum[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][n][j] = 0.0f;
      m[n][0] = m[n][1] = -kInf;
      lsum[n][0] = lsum[n][1] = 0.0f;
    }

    T x[KT];
    bool some[KT];
    const int tile_first = first * kUnitTiles + warp * KT, tile_last = min(last * kUnitTiles, tiles);
    long long row[KT];
#pragma unroll
    for (int i = 0; i < KT; ++i) {
      row[i] = tile_row(tile_first + i);
      some[i] = row[i] >= 0;
      if (some[i]) {
        load_k<D, kFmt>(a.cache, row[i], x[i]);
        load_v<D, kFmt>(a.cache, row[i], x[i]);
      }
    }
    for (int tile = tile_first; tile < tile_last; tile += kUnitTiles) {
      const int next = tile + kUnitTiles;
      bool more[KT];
#pragma unroll
      for (int i = 0; i < KT; ++i) {
        row[i] = next < tile_last ? tile_row(next + i) : -1;
        more[i] = row[i] >= 0;
      }
      // scores
      float s[KT][NT][4];
#pragma unroll
      for (int i = 0; i < KT; ++i) {
#pragma unroll
        for (int n = 0; n < NT; ++n) s[i][n][0] = s[i][n][1] = s[i][n][2] = s[i][n][3] = 0.0f;
#pragma unroll
        for (int b = 0; b < kGroups; ++b) {
          uint32_t f[2][4];  // [key g / g+8][value pairs 8t + 2j]
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if constexpr (kFmt == kFmtE4M3) {
              const uint32_t w0 = x[i].k[(h * kGroups + b) * 2], w1 = x[i].k[(h * kGroups + b) * 2 + 1];
              const uint32_t p[4] = {w0 & 0xFFFFu, w0 >> 16, w1 & 0xFFFFu, w1 >> 16};
#pragma unroll
              for (int j = 0; j < 4; ++j)
                asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(f[h][j]) : "h"(static_cast<uint16_t>(p[j])));
            } else {
              e2m1x8_to_f16x2(x[i].k[h * kGroups + b], f[h]);
            }
          }
          const float s0 = e8m0_value((x[i].ks[0][b / 4] >> (8 * (b & 3))) & 255u);
          const float s1 = e8m0_value((x[i].ks[1][b / 4] >> (8 * (b & 3))) & 255u);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            mma_f16_16816(d, f[0][0], f[1][0], f[0][1], f[1][1], q[n][b][0], q[n][b][1]);
            mma_f16_16816(d, f[0][2], f[1][2], f[0][3], f[1][3], q[n][b][2], q[n][b][3]);
            s[i][n][0] = fmaf(d[0], s0, s[i][n][0]);
            s[i][n][1] = fmaf(d[1], s0, s[i][n][1]);
            s[i][n][2] = fmaf(d[2], s1, s[i][n][2]);
            s[i][n][3] = fmaf(d[3], s1, s[i][n][3]);
          }
        }
      }
      // K registers are free: the next step's keys
#pragma unroll
      for (int i = 0; i < KT; ++i)
        if (more[i]) load_k<D, kFmt>(a.cache, row[i], x[i]);

      // masked scores, running maximum, p = 2^(s - m + kCarry)
      uint32_t p[KT][NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float top[2] = {m[n][0], m[n][1]};
#pragma unroll
        for (int i = 0; i < KT; ++i) {
          const int key = (tile + i) * 16 + g;
          const bool in0 = some[i] && key < len, in1 = some[i] && key + 8 < len;
          s[i][n][0] = in0 ? s[i][n][0] * mult[n][0] : -kInf;
          s[i][n][1] = in0 ? s[i][n][1] * mult[n][1] : -kInf;
          s[i][n][2] = in1 ? s[i][n][2] * mult[n][0] : -kInf;
          s[i][n][3] = in1 ? s[i][n][3] * mult[n][1] : -kInf;
          top[0] = fmaxf(top[0], fmaxf(s[i][n][0], s[i][n][2]));
          top[1] = fmaxf(top[1], fmaxf(s[i][n][1], s[i][n][3]));
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          top[j] = fmaxf(top[j], __shfl_xor_sync(0xffffffffu, top[j], 4));
          top[j] = fmaxf(top[j], __shfl_xor_sync(0xffffffffu, top[j], 8));
          top[j] = fmaxf(top[j], __shfl_xor_sync(0xffffffffu, top[j], 16));
          const float base = top[j] == -kInf ? 0.0f : top[j];  // nothing seen yet
          const float fade = exp2_approx(m[n][j] - base);
          m[n][j] = top[j];
          lsum[n][j] *= fade;
#pragma unroll
          for (int i = 0; i < D / 16; ++i) acc[i][n][j] *= fade, acc[i][n][j + 2] *= fade;
          top[j] = base - kCarry;
        }
#pragma unroll
        for (int i = 0; i < KT; ++i) {
          const float p0 = exp2_approx(s[i][n][0] - top[0]), p1 = exp2_approx(s[i][n][1] - top[1]);
          const float p2 = exp2_approx(s[i][n][2] - top[0]), p3 = exp2_approx(s[i][n][3] - top[1]);
          lsum[n][0] += p0 + p2;
          lsum[n][1] += p1 + p3;
          // p is rounded to bf16 for the product (relative 2^-9 each, of either sign); the sum is not
          p[i][n][0] = transpose8x8(pack_bf16x2(p0, p1));
          p[i][n][1] = transpose8x8(pack_bf16x2(p2, p3));
        }
      }
      // output
#pragma unroll
      for (int i = 0; i < KT; ++i) {
        if (!some[i]) continue;
        constexpr int kW = T::kVWords / 4;
        const int key = (tile + i) * 16;
        if (key + 16 > len) {  // rows behind the sequence may hold anything
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (key + 2 * t + (j & 1) + 8 * (j >> 1) >= len) {
              x[i].vs[j] = 0;
#pragma unroll
              for (int w = 0; w < kW; ++w) x[i].v[j * kW + w] = 0;
            }
        }
        uint32_t va[D / 8], vb[D / 8];
        v_pairs<D, kFmt>(x[i].v, x[i].v + kW, v_factor(x[i].vs[0]) | (v_factor(x[i].vs[1]) << 16), va);
        v_pairs<D, kFmt>(x[i].v + 2 * kW, x[i].v + 3 * kW, v_factor(x[i].vs[2]) | (v_factor(x[i].vs[3]) << 16), vb);
#pragma unroll
        for (int c = 0; c < D / 16; ++c)
#pragma unroll
          for (int n = 0; n < NT; ++n)
            mma_bf16_16816(acc[c][n], va[2 * c], va[2 * c + 1], vb[2 * c], vb[2 * c + 1], p[i][n][0], p[i][n][1]);
      }
#pragma unroll
      for (int i = 0; i < KT; ++i) {
        some[i] = more[i];
        if (more[i]) load_v<D, kFmt>(a.cache, row[i], x[i]);
      }
    }

    // join the warps
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float l = lsum[n][j];
        l += __shfl_xor_sync(0xffffffffu, l, 4);
        l += __shfl_xor_sync(0xffffffffu, l, 8);
        l += __shfl_xor_sync(0xffffffffu, l, 16);
        const int h = 8 * n + 2 * t + j;
        if (g == 0) sm_m[warp * kHeads + h] = m[n][j], sm_l[warp * kHeads + h] = l;
        float* dst = sm + (warp * kHeads + h) * kStride + g * (D / 8);
#pragma unroll
        for (int c = 0; c < D / 16; ++c)
          *reinterpret_cast<float2*>(dst + 2 * c) = make_float2(acc[c][n][j], acc[c][n][j + 2]);
      }
    __syncthreads();
    const bool whole = first == 0 && last == units;
    float* part = a.parts + (2 * static_cast<size_t>(blockIdx.x) + (first == 0 ? 1 : 0)) * kHeads * (D + 2);
    for (int i = threadIdx.x; i < nh * (D / 4); i += kAttnThreads) {
      const int h = i / (D / 4), d = 4 * (i - h * (D / 4));
      float top = -kInf;
#pragma unroll
      for (int w = 0; w < kAttnWarps; ++w) top = fmaxf(top, sm_m[w * kHeads + h]);
      const float base = top == -kInf ? 0.0f : top;
      float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      float l = 0.0f;
#pragma unroll
      for (int w = 0; w < kAttnWarps; ++w) {
        const float f = exp2_approx(sm_m[w * kHeads + h] - base);
        const float4 x4 = *reinterpret_cast<const float4*>(sm + (w * kHeads + h) * kStride + d);
        l = fmaf(sm_l[w * kHeads + h], f, l);
        o.x = fmaf(x4.x, f, o.x), o.y = fmaf(x4.y, f, o.y), o.z = fmaf(x4.z, f, o.z), o.w = fmaf(x4.w, f, o.w);
      }
      l *= exp2f(-kCarry);
      if (whole) {
        const float r = l == 0.0f ? 0.0f : 1.0f / l;  // no key in reach (bad pages): zeros
        const size_t at = static_cast<size_t>(seq) * a.q_heads + h0 + h;
        uint2 o2;
        o2.x = pack_bf16x2(o.x * r, o.y * r), o2.y = pack_bf16x2(o.z * r, o.w * r);
        *reinterpret_cast<uint2*>(a.out + at * D + d) = o2;
        if (a.lse && d == 0) a.lse[at] = l == 0.0f ? -kInf : (top + log2f(l)) * 0.6931471805599453f;
      } else {
        *reinterpret_cast<float4*>(part + h * D + d) = o;
        if (d == 0) part[kHeads * D + 2 * h] = top, part[kHeads * D + 2 * h + 1] = l;
      }
    }
    __syncthreads();
    u += last - first;
    if (last == units && hc + 1 == a.cache.heads * a.chunks) {
      begin += static_cast<long long>(units) * a.cache.heads * a.chunks;
      ++seq;
    }
  }
}

// Joins the parts of the heads that lie in several blocks' shares, in the blocks' order, and
// writes the rows of empty sequences.  One block per (sequence, kv head, chunk).
template <int D, int NT>
__global__ void __launch_bounds__(128) attn_join_kernel(const __grid_constant__ AttnArgs a, int unit_keys) {
  constexpr int kHeads = 8 * NT;
  constexpr float kInf = __builtin_huge_valf();
  __shared__ long long red[8];
  __shared__ float top_s[kHeads], sum_s[kHeads];
  const int per = a.cache.heads * a.chunks;
  const int seq = blockIdx.x / per, hc = blockIdx.x - seq * per;
  const int head = hc / a.chunks, chunk = hc - head * a.chunks;
  const int h0 = head * a.group + chunk * kHeads, nh = min(kHeads, a.group - chunk * kHeads);
  long long total, ahead;
  attn_count_units(a, unit_keys, seq, total, ahead, red);
  const int units = (attn_length(a, seq) + unit_keys - 1) / unit_keys;
  const size_t at0 = static_cast<size_t>(seq) * a.q_heads + h0;
  griddep_wait();
  if (units == 0) {
    for (int i = threadIdx.x; i < nh * (D / 4); i += 128)
      *reinterpret_cast<uint2*>(a.out + at0 * D + 4 * static_cast<size_t>(i)) = make_uint2(0, 0);
    if (a.lse && threadIdx.x < nh) a.lse[at0 + threadIdx.x] = -kInf;
    return;
  }
  const long long share = attn_share(total, a.blocks), u0 = ahead + static_cast<long long>(hc) * units;
  const int c0 = static_cast<int>(u0 / share), c1 = static_cast<int>((u0 + units - 1) / share);
  if (c0 == c1) return;
  // the head begins in block c0 (its slot 1) and covers the start of the others (their slot 0)
  auto part_of = [&](int c) { return a.parts + (2 * static_cast<size_t>(c) + (c == c0 ? 1 : 0)) * kHeads * (D + 2); };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int h = warp; h < nh; h += 4) {
    float top = -kInf;
    for (int c = c0 + lane; c <= c1; c += 32) top = fmaxf(top, part_of(c)[kHeads * D + 2 * h]);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
    const float base = top == -kInf ? 0.0f : top;
    float l = 0.0f;
    for (int c = c0 + lane; c <= c1; c += 32) {
      const float2 ml = *reinterpret_cast<const float2*>(part_of(c) + kHeads * D + 2 * h);
      l = fmaf(ml.y, exp2_approx(ml.x - base), l);
    }
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
    if (lane == 0) {
      top_s[h] = base, sum_s[h] = l;
      if (a.lse) a.lse[at0 + h] = l == 0.0f ? -kInf : (top + log2f(l)) * 0.6931471805599453f;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < nh * (D / 4); i += 128) {
    const int h = i / (D / 4), d = 4 * (i - h * (D / 4));
    const float base = top_s[h], l = sum_s[h];
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
    for (int c = c0; c <= c1; ++c) {
      const float* part = part_of(c);
      const float f = exp2_approx(part[kHeads * D + 2 * h] - base);
      const float4 x4 = *reinterpret_cast<const float4*>(part + h * D + d);
      o.x = fmaf(x4.x, f, o.x), o.y = fmaf(x4.y, f, o.y), o.z = fmaf(x4.z, f, o.z), o.w = fmaf(x4.w, f, o.w);
    }
    const float r = l == 0.0f ? 0.0f : 1.0f / l;
    uint2 o2;
    o2.x = pack_bf16x2(o.x * r, o.y * r), o2.y = pack_bf16x2(o.z * r, o.w * r);
    *reinterpret_cast<uint2*>(a.out + (at0 + h) * D + d) = o2;
  }
}

}  // namespace mxb
