// Attention of one new token per sequence over the paged MX key-value cache (kv_rows.cuh).
//
//   s_j = scale * sum_d q_d k_jd,  j < length;   o = sum_j exp(s_j) v_j / sum_j exp(s_j);
//   lse = log sum_j exp(s_j);  length 0: o = 0, lse = -inf.
//
// Every key-value head is read once for all the query heads that share it (up to 8 * NT of them
// to a block), so the kernel is bound by the cache's bytes: 2 * D * (8 or 4) / 8 + D / 16 per key.
// One pass: running maximum and sum of the softmax in fp32, sums of o in fp32.
//
// A warp takes steps of attn_tiles tiles of 16 keys through a ring of asynchronous copies of its own
// (16-byte copies that each lane sends for and waits for itself, then one __syncwarp: no barrier, no
// mbarrier, nothing that could hang).  With lane = 4 g + t:
//   scores  S^T[key][head] = K Q^T, K as the 16-row operand (m16n8k16, f16): row g is key
//           pi(g) = g / 2 + 4 (g % 2), row g + 8 key pi(g) + 8.  Lane (g, t) holds their values 32 b + 8 t
//           .. + 7 of each 32-value group b (any order of the values serves, if q has the same).  The
//           codes convert exactly to f16; q is scaled per head by a power of two, with which f16
//           holds every bf16 bit of values down to 2^-31 of the head's largest, and each group's
//           fp32 partial is multiplied by the key's scale.  Where q has smaller ones, or a scale byte is outside
//           64 .. 191, q goes through in levels of 31 binades each (see walk).
//   output  O^T[d][head] = V^T P^T, V as the 16-row operand (m16n8k16, bf16).  With pi, lane (g, t) needs
//           keys t, t + 4, t + 8, t + 12, which lie in different banks, and holds the D / 8 values from
//           g D / 8 on: all in one 32-value group, so one scale byte per key.  The codes become bf16 by
//           moving their fields into place, which is the value times 2^-120 (E4M3) or 2^-126
//           (E2M1), and one exact multiply by scale * 2^63, which leaves v * 2^-kCarry (kCarry = 57 or
//           63); p carries 2^kCarry.  bf16 has the range for the scale bytes 64 .. 191, whatever the other
//           keys' are.  A warp that meets another one takes its keys again, in up to three parts of
//           their own power of two each (see walk).  (f16 here, with the hardware's conversion and a scale
//           relative to a running one, measured 5 to 8 % faster and would lose weights below
//           2^-36 and values 2^-20 below the largest: not taken.)
//           P^T is two bf16 operands whose sum holds 16 bits of each weight, so the output is rounded once.
//           The transposition between S^T's accumulators and P^T's operands is one movmatrix each per 8 keys.
// What bounds it, measured: E4M3 D = 128, 8 heads to a kv head, 2 x 131072 keys: 102 us for 554 MB, 82 % of the
// HBM copy rate; E2M1 88 us, 50 %.  452 and 460 instructions per tile (2 x 65536 keys, starts and ends
// included), 54 and 63 % of the issue slots, ALU pipe 57 and 54 %, tensor pipe 23 and 26 %: the issue slots, and bursts
// of products that wait for the tensor pipe.  D = 64: 57 % (E4M3), D = 256: 70 % (E4M3) and 48 % (E2M1, 4 heads to
// a kv head).  Of that the second product of the weights is 5 % (E2M1 10 %, 16 heads to a kv head 16 to 18 %), the
// look for NaN codes 6 % (E4M3), for scales out of the usual range 1 to 3 %.
// One tile to a step against two, E2M1: 94 us, and 92 against 87 on 256 x 1000 keys; four resident blocks
// of 127 registers against three of 168, E4M3: 109 us against 92 on 2 x ~115k keys.
// Measured with one product of the weights and without those looks, as are the comparisons of forms below and at
// attn_plan: three and four tiles to a step 76 and 75 us against 78 for E2M1 there but 82 and 90 against 76 on 256 x
// 1000 keys; five blocks of 96 registers 89; the left shifts of its decode as multiplications by a number the
// compiler does not know 77, and as much slower elsewhere; E4M3 loads straight into registers (no ring) 111
// against 87 us on 2 x ~115k keys, 12 warps cannot both hold the bytes and compute.
//
// A head's keys are cut into units of kAttnWarps steps, and the heads into pieces of at most `share`
// units, share so that there are about as many pieces as blocks are resident: one block to a piece,
// found from the lengths on the device, so that long and short sequences share the GPU evenly and a
// block's first loads run beside the other blocks' work (64 ragged sequences, E2M1: 42 us; 46 with one
// equal share of all units to a block, which then went through several heads one after another).  A
// head of one piece is written at once; the parts of the others go to the workspace and
// attn_join_kernel adds them in order.
// Where even the longest sequence that the page table can hold is a few units, a cluster of 1 to 8
// blocks takes a head instead and joins its parts through distributed shared memory: one launch, no
// workspace, and each block looks at the length of its own sequence only (200 of up to 500 keys: 31 us
// against 67, which also paid for the joining kernel's blocks).  Its blocks take units in turn, so that the
// first pages are known before the length is, and all remote parts are loaded before the first is
// used: one sequence of 700 keys 5.3 us, 7.1 without the two.
#pragma once

#include <type_traits>

#include "common.cuh"
#include "gemm_small.cuh"
#include "kv_rows.cuh"

namespace mxb {

constexpr int kAttnWarps = 4;
constexpr int kAttnThreads = 32 * kAttnWarps;
// Pieces per resident block, where the heads are many: 1, 2, 3, 4 measured 65, 61, 65, 69 us on 32 x 4096 keys
// (E4M3, 8 kv heads), 49, 48, 49, 51 us on 64 ragged sequences (E2M1).
constexpr int kAttnPieces = 2;
// Units to a block of a cluster, at most: 4, 8, 16, 32 measured 89, 57, 57, 57 us on 256 sequences of up to
// 1000 keys, 30, 30, 30, 49 us on 16 of up to 8192 (E4M3).
constexpr int kAttnClusterSteps = 16;

// Tiles of 16 keys a warp takes in one step; steps in its ring; blocks resident per SM (the kernel's
// launch bound).
__host__ __device__ constexpr int attn_tiles(int dim, int fmt) { return dim == 256 && fmt == kFmtE4M3 ? 1 : 2; }
__host__ __device__ constexpr int attn_ring(int dim, int fmt) { return (dim == 256 && fmt == kFmtE4M3) || dim == 64 ? 3 : 2; }
__host__ __device__ constexpr int attn_resident(int dim, int fmt, int nt) {
  // 16 heads to a kv head, D = 128, two blocks against three: E2M1 116 and 127 us on 2 x 131072 keys, 82 and 81 on 32 x
  // 4096, 46 and 42 on 64 ragged, 10.5 and 13.3 on 8 x 1000 (three spill); E4M3 129 us with two on 2 x 131072, 104 and
  // 118 with one product of the weights
  if (nt == 2) return dim == 128 ? 2 : 3;
  return dim == 256 ? 2 : (dim == 128 && fmt == kFmtE4M3 ? 3 : 4);
}
__host__ __device__ constexpr int attn_unit_keys(int dim, int fmt) { return 16 * kAttnWarps * attn_tiles(dim, fmt); }
__host__ __device__ constexpr int attn_row_bytes(int dim, int fmt) { return fmt == kFmtE4M3 ? dim : dim / 2; }
constexpr int kAttnMinUnit = 16 * kAttnWarps;
// K codes, V codes, K scales, V scales of 16 keys
__host__ __device__ constexpr int attn_tile_bytes(int dim, int fmt) {
  return 16 * 2 * (attn_row_bytes(dim, fmt) + dim / 32);
}
__host__ __device__ constexpr int attn_smem_bytes(int dim, int fmt, int nt) {
  const int ring = kAttnWarps * attn_ring(dim, fmt) * attn_tiles(dim, fmt) * attn_tile_bytes(dim, fmt);
  const int join = 8 * nt * (kAttnWarps * (dim + 4 + 2) + 2) * 4;  // the warps' parts, after the ring
  return ring > join ? ring : join;
}

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
  int2* heads;             // [seqs][kv heads][chunks]: pieces of each head that has any, and its first part
  float* parts;            // [2 * target][8 * NT heads][dim + 2]
  int target;              // pieces to cut the work into
  int fit;                 // heads are few: no more pieces than that
  int unit_keys;
  int cluster;             // blocks to a head, joining among themselves; 0: pieces
  int stride;              // tiles from one step of a warp to its next: of one unit, times the cluster's blocks
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

__device__ __forceinline__ float4 ld_dsmem_f32x4(const float* local, uint32_t rank) {
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_u32(local)), "r"(rank));
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(remote) : "memory");
  return v;
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

__device__ __forceinline__ int attn_units(const AttnArgs& a, int b, int unit_keys) {
  return static_cast<int>((static_cast<unsigned>(attn_length(a, b)) + unit_keys - 1) / unit_keys);
}

// Sum of f(sequence) over sequences 0 .. n - 1 (below 2^31: so is the number of all units).  Every
// warp on its own.
template <typename F>
__device__ __forceinline__ int attn_sum(int n, F f) {
  int s = 0;
#pragma unroll 4
  for (int b = threadIdx.x & 31; b < n; b += 32) s += f(b);
  return __reduce_add_sync(0xffffffffu, s);
}
__device__ __forceinline__ int ceil_ratio(long long a, int b) {
  if (a < 0x7FFFFFFFll - b) return (static_cast<int>(a) + b - 1) / b;
  return static_cast<int>(min((a + b - 1) / b, 0x3FFFFFFFll));  // no head has more units
}

// Pieces of each head of a sequence.
__device__ __forceinline__ int attn_pieces(int units, int share) {
  return static_cast<int>((static_cast<unsigned>(units) + share - 1) / share);
}

// Most units of a piece.  All units over the pieces wanted; where the heads are few, the least with
// which the pieces are no more than wanted, so that they all run at once (rounding up leaves up to one
// short piece per head, and a second round of blocks for them would double the time).
__device__ __forceinline__ int attn_share(const AttnArgs& a, int unit_keys) {
  const long long per = static_cast<long long>(a.cache.heads) * a.chunks, heads = per * a.seqs;
  const long long total = per * attn_sum(a.seqs, [&](int b) { return attn_units(a, b, unit_keys); });
  int lo = max(1, ceil_ratio(total, a.target));
  if (a.fit) {
    // with total / share + heads <= target there are enough
    int hi = max(lo, ceil_ratio(total, a.target - static_cast<int>(heads)));
    while (lo < hi) {
      const int mid = lo + (hi - lo) / 2;
      if (per * attn_sum(a.seqs, [&](int b) { return attn_pieces(attn_units(a, b, unit_keys), mid); }) <= a.target) hi = mid;
      else lo = mid + 1;
    }
  }
  return lo;
}

struct AttnPiece {
  int seq, head_chunk, index, of;  // the index-th of `of` pieces of a head
  int slot;                        // its place in the workspace, where of > 1
};
// The piece-th piece of all; false if there are fewer.  Every warp on its own.
__device__ __forceinline__ bool attn_find(const AttnArgs& a, int unit_keys, int share, int piece, AttnPiece& found) {
  const int per = a.cache.heads * a.chunks, lane = threadIdx.x & 31;
  int pieces = 0, slots = 0;  // of the sequences before
  for (int b0 = 0; b0 < a.seqs; b0 += 32) {
    const int n = b0 + lane < a.seqs ? attn_pieces(attn_units(a, b0 + lane, unit_keys), share) : 0;
    const int all = __reduce_add_sync(0xffffffffu, n) * per, held = __reduce_add_sync(0xffffffffu, n > 1 ? n : 0) * per;
    if (pieces + all > piece) {
      int run = n, kept = n > 1 ? n : 0;
#pragma unroll
      for (int m = 1; m < 32; m <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, run, m), y = __shfl_up_sync(0xffffffffu, kept, m);
        if (lane >= m) run += x, kept += y;
      }
      const int f = __ffs(__ballot_sync(0xffffffffu, pieces + run * per > piece)) - 1;
      found.seq = b0 + f;
      found.of = __shfl_sync(0xffffffffu, n, f);
      const int r = piece - pieces - (__shfl_sync(0xffffffffu, run, f) - found.of) * per;
      found.head_chunk = r / found.of;
      found.index = r - found.head_chunk * found.of;
      found.slot = slots + (__shfl_sync(0xffffffffu, kept, f) - found.of) * per + r;
      return true;
    }
    pieces += all;
    slots += held;
  }
  return false;
}

// Placement of the 16-byte units of key row r (0..15) of a tile in shared memory: unit u of the row
// goes to u ^ attn_swizzle.  The rows a load instruction touches in one phase (K: rows pi(g), see
// below; V: rows t + 4 i) then lie in different banks.
template <int D, int kFmt, bool kV>
__device__ __forceinline__ constexpr int attn_swizzle(int r) {
  constexpr int kRowBytes = attn_row_bytes(D, kFmt);
  if constexpr (kFmt == kFmtE4M3) {
    if constexpr (kV) return kRowBytes == 64 ? r & 2 : (kRowBytes == 128 ? 2 * (r & 3) : (r & 1) | ((r & 2) << 1));
    return kRowBytes == 64 ? (r >> 1) & 2 : ((r >> 1) & 2) | ((r & 1) << 2);
  } else {
    if constexpr (kV) return kRowBytes == 32 ? 0 : (kRowBytes == 64 ? r & 2 : 2 * (r & 3));
    return kRowBytes == 32 ? (r >> 2) & 1 : (kRowBytes == 64 ? (r >> 1) & 3 : r & 7);
  }
}

// Copies the 16 keys of a tile into shared memory at dst (one warp): codes from k and v, scales
// from sc, each with the lane's own offset already in it.  base_k and base_v: the lane's first
// place in the tile; a later one differs by whole rows and, as the swizzle is linear over xor in
// the row's bits, by an xor with a constant.
template <int D, int kFmt, bool kV>
__device__ __forceinline__ uint32_t attn_copy_base() {
  constexpr int kRowBytes = attn_row_bytes(D, kFmt), kUnits = kRowBytes / 16;
  const int lane = threadIdx.x & 31, r = lane / kUnits, u = lane % kUnits;
  return r * kRowBytes + 16 * (u ^ attn_swizzle<D, kFmt, kV>(r));
}
template <int D, int kFmt>
__device__ __forceinline__ void attn_copy_tile(const uint8_t* k, const uint8_t* v, const uint8_t* sc, uint32_t dst,
                                               uint32_t base_k, uint32_t base_v) {
  constexpr int kRowBytes = attn_row_bytes(D, kFmt), kUnits = kRowBytes / 16, kRows = 32 / kUnits;
#pragma unroll
  for (int j = 0; j < kUnits / 2; ++j) {
    cp_async16(dst + (base_k ^ (16 * attn_swizzle<D, kFmt, false>(kRows * j))) + 512 * j, k + 512 * j);
    cp_async16(dst + (base_v ^ (16 * attn_swizzle<D, kFmt, true>(kRows * j))) + 512 * j + 16 * kRowBytes, v + 512 * j);
  }
  const int lane = threadIdx.x & 31;
  if (lane < D / 16) cp_async16(dst + 32 * kRowBytes + 16 * lane, sc);
}

template <int kWords>
__device__ __forceinline__ void lds_words(uint32_t a, uint32_t* w) {
  if constexpr (kWords % 4 == 0) {
    const uint4 u = lds128(a);
    w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
  } else if constexpr (kWords == 2) {
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(a));
  } else {
    w[0] = lds32(a);
  }
}

// Four E4M3 codes as f16x2 words, exact.
__device__ __forceinline__ void e4m3x4_to_f16x2(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 l, h;\n\t"
      "mov.b32 {l, h}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, l;\n\t"
      "cvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(w));
}
// Two E8M0 bytes as bf16x2: 2^(b - 127), 255 is NaN.
__device__ __forceinline__ uint32_t e8m0x2_bf16x2(uint32_t b) {
  uint32_t r;
  asm("cvt.rn.bf16x2.ue8m0x2 %0, %1;" : "=r"(r) : "h"(static_cast<uint16_t>(b)));
  return r;
}
// Four of them (the low two, the high two).
__device__ __forceinline__ void e8m0x4_bf16x2(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 l, h;\n\t"
      "mov.b32 {l, h}, %2;\n\t"
      "cvt.rn.bf16x2.ue8m0x2 %0, l;\n\t"
      "cvt.rn.bf16x2.ue8m0x2 %1, h;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(w));
}
__device__ __forceinline__ float bf16_lo(uint32_t x) { return __uint_as_float(x << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t x) { return __uint_as_float(x & 0xFFFF0000u); }

// bf16x2 multiplier of two keys' scale bytes (see kCarry at the top): 2^(byte - 64), for bytes of 64 .. 191.
__device__ __forceinline__ uint32_t v_factor(uint32_t b0, uint32_t b1) { return prmt(b0, b1, 0x5410) * 128u + 0x1F801F80u; }
// All scale bytes come in three classes, 0 .. 63, 64 .. 191 and 192 .. 255; the multiplier 2^(byte - 64 + 64 (1 - cls)) of
// one of class `cls` as bf16, zero for another class's, NaN for 255.
__device__ __forceinline__ uint32_t v_class_factor(uint32_t byte, int cls) {
  if (static_cast<int>(byte + 64) >> 7 != cls) return 0;
  return byte == 255 ? 0x7FC0u : (byte + 63 + 64 * (1 - cls)) << 7;
}
// Whether one of the lane's scale bytes w (as many as mask has 0x80s) is outside 64 .. 191.
__device__ __forceinline__ bool odd_scales(uint32_t both, uint32_t mask) { return (both & mask) != mask; }

// V operand words of one pair of keys: for each of the lane's D / 8 values, (key a, key b) as
// bf16x2 times the keys' factors.  E4M3: `most` follows the largest magnitudes, each half of it, and with
// kNan the NaN codes become NaN.
template <int D, int kFmt, bool kNan>
__device__ __forceinline__ void v_pairs(const uint32_t* a, const uint32_t* b, uint32_t factor, uint32_t (&o)[D / 8], uint32_t& most) {
  if constexpr (kFmt == kFmtE4M3) {
#pragma unroll
    for (int i = 0; i < D / 8; i += 2) {
      uint32_t m[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        // the two codes in the high bytes of the halves; low bytes are masked away
        const uint32_t x = prmt(a[i / 4], b[i / 4], ((4 + ((i + j) & 3)) << 12) | (((i + j) & 3) << 4));
        m[j] = (x >> 4) & 0x07F007F0u;
        uint32_t v = m[j] | (x & 0x80008000u);
        if constexpr (kNan) {
          if ((v & 0x7FFFu) == 0x07F0u) v |= 0x7FC0u;
          if ((v & 0x7FFF0000u) == 0x07F00000u) v |= 0x7FC00000u;
        }
        o[i + j] = mul_bf16x2(v, factor);
      }
      most = __vimax3_u16x2(most, m[0], m[1]);
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
// Whether v_pairs met a NaN code, all ones: moved into bf16 it would be 480, 0x07F0, the most there can be.
__device__ __forceinline__ bool has_nan_code(uint32_t most) { return ((most + 0x00100010u) & 0x08000800u) != 0; }

// A part of a head (a warp's, a block's) is a reference m, the sum l of p and the sums o of p v.  Where values of 2^56
// and more are among them, o is kept in units of 1 / kHugeUnit, so that it stays in the range of fp32, and l
// negative to say so.  Parts are joined in small units if one of them is (`any`).
constexpr float kHugeUnit = 0x1p-40f;
__device__ __forceinline__ float part_factor(float f, float l, bool any) { return any && !(l < 0.0f) ? f * kHugeUnit : f; }
__device__ __forceinline__ uint2 attn_output(const float4& o, float r, bool any) {
  const float up = any ? 1.0f / kHugeUnit : 1.0f;
  return make_uint2(pack_bf16x2(o.x * r * up, o.y * r * up), pack_bf16x2(o.z * r * up, o.w * r * up));
}

// Exponent of a finite bf16 that is not zero: |x| is in [2^e, 2^(e + 1)).
__device__ __forceinline__ int bf16_exponent(uint32_t mag) { return mag >= 0x80u ? static_cast<int>(mag >> 7) - 127 : -102 - __clz(mag); }
// The level of a query value, scaled by 2^shift so that the head's largest is in [2^14, 2^15).
__device__ __forceinline__ int q_level(uint32_t mag, int shift) { return (14 - (bf16_exponent(mag) + shift)) / 31; }
// x * 2^(shift + 31 * level) in f16 if x is of that level (exact: 8 bits of at least 2^-16), else zero.
__device__ __forceinline__ uint32_t q_of_level(uint32_t x, int shift, int level) {
  const uint32_t mag = x & 0x7FFFu;
  if (mag >= 0x7F80u) return level ? 0u : (mag > 0x7F80u ? 0x7FFFu : 0x7C00u | (x & 0x8000u));
  if (mag == 0 || q_level(mag, shift) != level) return 0;
  return __half_as_ushort(__float2half_rn(ldexpf(__uint_as_float(x << 16), shift + 31 * level)));
}

template <int D, int kFmt, int NT>
__global__ void __launch_bounds__(kAttnThreads, attn_resident(D, kFmt, NT)) attn_kernel(const __grid_constant__ AttnArgs a) {
  constexpr int kGroups = D / 32, kHeads = 8 * NT, kRing = attn_ring(D, kFmt);
  constexpr int kRowBytes = attn_row_bytes(D, kFmt), kTile = attn_tile_bytes(D, kFmt);
  constexpr int KT = attn_tiles(D, kFmt), kUnitKeys = attn_unit_keys(D, kFmt);
  constexpr int kKw = kRowBytes / kGroups / 16;  // words of K codes per lane, key and group: 2 or 1
  constexpr int kVw = kRowBytes / 32;            // words of V codes per lane and key
  constexpr float kRaise = kFmt == kFmtE4M3 ? 0x1p57f : 0x1p63f;  // 2^kCarry: what p carries, and v its inverse
  constexpr float kRise = 8.0f;                               // see below
  constexpr int kStride = D + 4;                              // floats per head of a warp's part in shared memory
  constexpr float kInf = __builtin_huge_valf();
  extern __shared__ __align__(128) float sm[];                // the warps' rings; then [warps][kHeads][kStride]
  float* sm_m = sm + kAttnWarps * kHeads * kStride;           // and m, l [warps][kHeads]
  float* sm_l = sm_m + kAttnWarps * kHeads;
  float* sm_joined = sm_l + kAttnWarps * kHeads;              // of the block: m, l [kHeads]

  griddep_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int key_g = (g >> 1) + 4 * (g & 1);  // pi(g): the key of operand row g (and key_g + 8 of row g + 8)
  const uint32_t ring = smem_u32(sm) + warp * kRing * KT * kTile;
  const uint32_t base_k = attn_copy_base<D, kFmt, false>(), base_v = attn_copy_base<D, kFmt, true>();

  AttnPiece me;
  if (a.cluster) {
    const int per = a.cache.heads * a.chunks, all = blockIdx.x / a.cluster;
    me.of = a.cluster, me.index = blockIdx.x - all * a.cluster;
    me.seq = all / per, me.head_chunk = all - me.seq * per;
    me.slot = 0;
  } else if (!attn_find(a, kUnitKeys, attn_share(a, kUnitKeys), blockIdx.x, me)) {
    return;
  }
  {
    const int seq = me.seq;
    const int* table = a.table + a.table_stride * seq;
    const int tile_shift = a.cache.page_shift - 4;
    // The blocks of a cluster take units in turn, so that the first is known, and its pages are on their
    // way, before the length is.
    int first = me.index, page[KT];
    if (a.cluster) {
#pragma unroll
      for (int i = 0; i < KT; ++i) {
        const int at = ((first * kAttnWarps + warp) * KT + i) >> tile_shift;
        page[i] = at < a.max_pages ? __ldg(table + at) : 0;
      }
    }
    const int len = attn_length(a, seq);
    int tile_last = (len + 15) >> 4;
    if (!a.cluster) {  // units first .. of a piece
      const int units = attn_units(a, seq, kUnitKeys);
      first = static_cast<int>(static_cast<long long>(units) * me.index / me.of);
      tile_last = min(static_cast<int>(static_cast<long long>(units) * (me.index + 1) / me.of) * kAttnWarps * KT, tile_last);
    }
    const int tile_first = (first * kAttnWarps + warp) * KT;
    auto first_pages = [&]() {
#pragma unroll
      for (int i = 0; i < KT; ++i) page[i] = tile_first + i < tile_last ? __ldg(table + ((tile_first + i) >> tile_shift)) : 0;
    };
    if (!a.cluster) first_pages();
    const int head = me.head_chunk / a.chunks, chunk = me.head_chunk - head * a.chunks;
    const int h0 = head * a.group + chunk * kHeads;                  // first q head
    const int nh = min(kHeads, a.group - chunk * kHeads);            // q heads here

    // Copies into the ring, one commit group per step; the pages of the step after are on their way.
    // `good` has KT bits for each of the last copies: whether the tile's page is one of the cache's.
    uint32_t good = 0;
    int copy_tile = tile_first, copy_slot = 0;
    const uint32_t page_rows = static_cast<uint32_t>(a.cache.heads) << a.cache.page_shift;
    const size_t head_rows = static_cast<size_t>(head) << a.cache.page_shift;
    const uint8_t* k_lane = a.cache.k_codes + head_rows * kRowBytes + 16 * lane;
    const uint8_t* v_lane = a.cache.v_codes + head_rows * kRowBytes + 16 * lane;
    const uint8_t* s_lane = (lane < kGroups ? a.cache.k_scales + 16 * lane : a.cache.v_scales + 16 * (lane - kGroups)) +
                            head_rows * kGroups;
    auto copy_next = [&]() {
      good <<= KT;
#pragma unroll
      for (int i = 0; i < KT; ++i)
        if (copy_tile + i < tile_last) {
          if (page[i] >= 0 && page[i] < a.cache.num_pages) {
            const size_t row = static_cast<size_t>(page[i]) * page_rows + (((copy_tile + i) & ((1 << tile_shift) - 1)) << 4);
            attn_copy_tile<D, kFmt>(k_lane + row * kRowBytes, v_lane + row * kRowBytes, s_lane + row * kGroups,
                                    ring + (copy_slot * KT + i) * kTile, base_k, base_v);
            good |= 1u << i;
          } else {
            record_error(kErrBadPage);
          }
        }
      copy_tile += a.stride;
#pragma unroll
      for (int i = 0; i < KT; ++i)
        if (copy_tile + i < tile_last) page[i] = __ldg(table + ((copy_tile + i) >> tile_shift));
      copy_slot = copy_slot + 1 == kRing ? 0 : copy_slot + 1;
      cp_async_commit();
    };
#pragma unroll
    for (int i = 0; i < kRing - 1; ++i) copy_next();

    // Q operand: head g of n-tile n, values 32 b + 8 t .. + 7, scaled into f16
    uint32_t q[NT][kGroups][4];
    float mult[NT][2];  // of heads 2t, 2t+1: scale * log2(e) / the power of two
    bool held = true;   // f16 and fp32 hold all of that
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const bool real = 8 * n + g < nh;
      const __nv_bfloat16* src = a.q + a.q_stride * seq + static_cast<size_t>(h0 + 8 * n + g) * D + 8 * t;
      uint32_t large = 0, least = 0x7FFF7FFFu;  // least: magnitudes - 0x8001 in signed 16 bits, of zero the most
#pragma unroll
      for (int b = 0; b < kGroups; ++b) {
        uint4 x = make_uint4(0, 0, 0, 0);
        if (real) x = *reinterpret_cast<const uint4*>(src + 32 * b);
        q[n][b][0] = x.x, q[n][b][1] = x.y, q[n][b][2] = x.z, q[n][b][3] = x.w;
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
          large = __vimax3_u16x2(large, q[n][b][i] & 0x7FFF7FFFu, q[n][b][i + 1] & 0x7FFF7FFFu);
          least = __vimin3_s16x2(least, (q[n][b][i] | 0x80008000u) - 0x00010001u, (q[n][b][i + 1] | 0x80008000u) - 0x00010001u);
        }
      }
      uint32_t amax = max(large & 0xFFFFu, large >> 16);
      amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      // largest |q| into [2^14, 2^15): shift = 14 - floor(log2), at most 114
      const int shift = 14 + 127 - max(static_cast<int>(amax >> 7), 27);
      const float two = __uint_as_float(static_cast<uint32_t>(shift + 127) << 23);
#pragma unroll
      for (int b = 0; b < kGroups; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const __half2 h = __floats2half2_rn(bf16_lo(q[n][b][i]) * two, bf16_hi(q[n][b][i]) * two);
          q[n][b][i] = *reinterpret_cast<const uint32_t*>(&h);
        }
      // values of 2^-16 and more there keep all their bits
      const int low = min(static_cast<int>(least << 16) >> 16, static_cast<int>(least) >> 16) + 0x8001;
      const float back = a.scale * 1.4426950408889634f * __uint_as_float(static_cast<uint32_t>(127 - shift) << 23);
      held &= !real || ((low >> 7) + shift >= 127 - 16 && (a.scale == 0.0f || (fabsf(back) >= 0x1p-126f && fabsf(back) < kInf)));
#pragma unroll
      for (int j = 0; j < 2; ++j) mult[n][j] = __shfl_sync(0xffffffffu, back, 4 * (2 * t + j));
    }

    float acc[D / 16][NT][4];
    float m[NT][2], sub[NT][2], lsum[NT][2];  // reference maximum, the same or 0 before any score, sum of p
    auto clear = [&]() {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[i][n][j] = 0.0f;
        m[n][0] = m[n][1] = -kInf;
        sub[n][0] = sub[n][1] = 0.0f;
        lsum[n][0] = lsum[n][1] = 0.0f;
      }
    };
    clear();

    // Largest of V's codes, see has_nan_code; or why else the keys have to be taken again with care (kHuge: values
    // of 2^56 and more may be among them, whose sum could leave the range of fp32).
    constexpr uint32_t kCare = 0x07F007F0u, kHuge = 0x0EF00EF0u;
    uint32_t most = held ? 0 : kCare;
    float raise = kRaise;
    bool huge = false;
    // For a walk with care: the power of two of the lane's own head in the q operand, of heads 2t and 2t + 1, and the levels.
    int own_shift[NT], shift_of[NT][2], levels = 1;
    auto q_at = [&](int n) { return a.q + a.q_stride * seq + static_cast<size_t>(h0 + 8 * n + g) * D + 8 * t; };
    // Looks closer at a step that has scales out of the usual range: groups of zeros (byte 0) are none of
    // those, nor are rows of no key.  A lane has one key's scales of K or of V.
    auto look_at_scales = [&](int tile, uint32_t have, uint32_t at) {
      const int key = lane & 15, of_v = lane >> 4;
#pragma unroll 1
      for (int i = 0; i < KT; ++i) {
        if (!((have >> i) & 1) || (tile + i) * 16 + key >= len) continue;
        const uint32_t codes = at + i * kTile + lane * kRowBytes, scales = at + i * kTile + 32 * kRowBytes + lane * kGroups;
        const uint32_t swizzle = 16 * (of_v ? attn_swizzle<D, kFmt, true>(key) : attn_swizzle<D, kFmt, false>(key));
#pragma unroll 1
        for (int b = 0; b < kGroups; ++b) {
          const uint32_t byte = lds_u8(scales + b);
          if (byte - 64u < 128u) continue;
          uint32_t any = byte;
          if (byte == 0) {
#pragma unroll
            for (int u = 0; u < kRowBytes / kGroups; u += 16) {
              const uint4 x = lds128(codes + ((b * (kRowBytes / kGroups) + u) ^ swizzle));
              any |= (x.x | x.y | x.z | x.w) & (kFmt == kFmtE4M3 ? 0x7F7F7F7Fu : 0x77777777u);
            }
          }
          if (any) most = max(most, of_v && byte >= 192 && byte != 255 ? kHuge : kCare);
        }
      }
    };
    // Scores of a tile's keys key_g (the first two of a head pair's) and key_g + 8, without mult.
    auto scores = [&](uint32_t at, float (&s)[NT][4]) {
      uint32_t two[2][kGroups / 2];  // the two keys' scales, a bf16x2 per pair of groups
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t sa = at + 32 * kRowBytes + (key_g + 8 * h) * kGroups;
        uint32_t w[(kGroups + 3) / 4];
        if constexpr (kGroups == 2) {
          asm volatile("ld.shared.u16 %0, [%1];" : "=r"(w[0]) : "r"(sa));
          two[h][0] = e8m0x2_bf16x2(w[0]);
        } else {
          lds_words<kGroups / 4>(sa, w);
#pragma unroll
          for (int b = 0; b < kGroups; b += 4) e8m0x4_bf16x2(w[b / 4], two[h][b / 2], two[h][b / 2 + 1]);
        }
      }
#pragma unroll
      for (int b = 0; b < kGroups; ++b) {
        uint32_t f[2][4];  // [key][value pairs 8t + 2j]
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int key = key_g + 8 * h;
          const int byte = b * (kRowBytes / kGroups) + 4 * kKw * t;
          uint32_t w[kKw];
          lds_words<kKw>(at + key * kRowBytes + (byte ^ (16 * attn_swizzle<D, kFmt, false>(key))), w);
          if constexpr (kFmt == kFmtE4M3) {
            e4m3x4_to_f16x2(w[0], f[h][0], f[h][1]);
            e4m3x4_to_f16x2(w[1], f[h][2], f[h][3]);
          } else {
            e2m1x8_to_f16x2(w[0], f[h]);
          }
        }
        const float s0 = b & 1 ? bf16_hi(two[0][b / 2]) : bf16_lo(two[0][b / 2]);
        const float s1 = b & 1 ? bf16_hi(two[1][b / 2]) : bf16_lo(two[1][b / 2]);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
          mma_f16_16816(d, f[0][0], f[1][0], f[0][1], f[1][1], q[n][b][0], q[n][b][1]);
          mma_f16_16816(d, f[0][2], f[1][2], f[0][3], f[1][3], q[n][b][2], q[n][b][3]);
          s[n][0] = fmaf(d[0], s0, s[n][0]);
          s[n][1] = fmaf(d[1], s0, s[n][1]);
          s[n][2] = fmaf(d[2], s1, s[n][2]);
          s[n][3] = fmaf(d[3], s1, s[n][3]);
        }
      }
    };
    // The same in powers of two, for any scale byte and query: levels of the query one after another, and the factors
    // of each group's sum put together as exponents.
    auto scores_with_care = [&](uint32_t at, float (&s)[NT][4]) {
      int of_scale;
      const float base = frexpf(a.scale, &of_scale) * 1.4426950408889634f;
#pragma unroll 1
      for (int level = 0; level < levels; ++level)
#pragma unroll 1
        for (int b = 0; b < kGroups; ++b) {
          uint32_t f[2][4], byte[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int key = key_g + 8 * h;
            byte[h] = lds_u8(at + 32 * kRowBytes + key * kGroups + b);
            uint32_t w[kKw];
            lds_words<kKw>(at + key * kRowBytes + ((b * (kRowBytes / kGroups) + 4 * kKw * t) ^ (16 * attn_swizzle<D, kFmt, false>(key))), w);
            if constexpr (kFmt == kFmtE4M3) {
              e4m3x4_to_f16x2(w[0], f[h][0], f[h][1]);
              e4m3x4_to_f16x2(w[1], f[h][2], f[h][3]);
            } else {
              e2m1x8_to_f16x2(w[0], f[h]);
            }
          }
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            uint4 x4 = make_uint4(0, 0, 0, 0);
            if (8 * n + g < nh) x4 = *reinterpret_cast<const uint4*>(q_at(n) + 32 * b);
            uint32_t x[4] = {x4.x, x4.y, x4.z, x4.w};
#pragma unroll
            for (int i = 0; i < 4; ++i)
              x[i] = q_of_level(x[i] & 0xFFFFu, own_shift[n], level) | q_of_level(x[i] >> 16, own_shift[n], level) << 16;
            float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            mma_f16_16816(d, f[0][0], f[1][0], f[0][1], f[1][1], x[0], x[1]);
            mma_f16_16816(d, f[0][2], f[1][2], f[0][3], f[1][3], x[2], x[3]);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int by = static_cast<int>(byte[j >> 1]) - 127 + of_scale - shift_of[n][j & 1] - 31 * level;
              s[n][j] += byte[j >> 1] == 255 ? __uint_as_float(0x7FC00000u) : ldexpf(d[j] * base, by);
            }
          }
        }
    };
    // One step; `ragged`: the sequence ends inside it, or a page of it is missing; `careful`: see below.
    auto do_step = [&](int tile, uint32_t have, uint32_t at, auto ragged, auto careful) {
      uint32_t usual = 0xFFFFFFFFu;  // see odd_scales; a key's scales of K or V to each lane
      constexpr uint32_t kUsual = kGroups == 2 ? 0x8080u : 0x80808080u;
      if constexpr (!decltype(careful)::value) {
#pragma unroll
        for (int i = 0; i < KT; ++i) {
          const uint32_t sa = at + i * kTile + 32 * kRowBytes + lane * kGroups;
          uint32_t w[2];
          if constexpr (kGroups == 2) asm volatile("ld.shared.u16 %0, [%1];" : "=r"(w[0]) : "r"(sa));
          else lds_words<kGroups / 4>(sa, w);
          usual &= w[0] ^ (w[0] << 1);
          if constexpr (kGroups == 8) usual &= w[1] ^ (w[1] << 1);
        }
      }
      // scores
      float s[KT][NT][4];
#pragma unroll
      for (int i = 0; i < KT; ++i) {
#pragma unroll
        for (int n = 0; n < NT; ++n) s[i][n][0] = s[i][n][1] = s[i][n][2] = s[i][n][3] = 0.0f;
        if constexpr (decltype(careful)::value) scores_with_care(at + i * kTile, s[i]);
        else scores(at + i * kTile, s[i]);
        // in powers of two, those of no key at -inf
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if constexpr (!decltype(careful)::value) s[i][n][j] *= mult[n][j & 1];
            if constexpr (decltype(ragged)::value)
              if (!((have >> i) & 1) || (tile + i) * 16 + key_g + 8 * (j >> 1) >= len) s[i][n][j] = -kInf;
          }
      }
      // The reference m follows the running maximum only when a score passes it by kRise: p stays
      // below 2^(kCarry + kRise), and most steps need no exchange between lanes and no rescaling.  (With care it
      // follows at once: large values have no room for 2^kRise.)
      float top[NT][2];
      bool rise = false;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          top[n][j] = fmaxf(s[0][n][j], s[0][n][j + 2]);
#pragma unroll
          for (int i = 1; i < KT; ++i) top[n][j] = fmaxf(top[n][j], fmaxf(s[i][n][j], s[i][n][j + 2]));
          rise |= top[n][j] > m[n][j] + (decltype(careful)::value ? 0.0f : kRise);
        }
      const bool odd = odd_scales(usual, kUsual);
      // One vote for both; scales may be odd in rows of no key, which must not move the reference.
      if (__any_sync(0xffffffffu, rise || odd)) {
        if (odd) look_at_scales(tile, have, at);
        if (__any_sync(0xffffffffu, rise)) {
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              float u = fmaxf(m[n][j], top[n][j]);
              u = fmaxf(u, __shfl_xor_sync(0xffffffffu, u, 4));
              u = fmaxf(u, __shfl_xor_sync(0xffffffffu, u, 8));
              u = fmaxf(u, __shfl_xor_sync(0xffffffffu, u, 16));
              const float base = u == -kInf ? 0.0f : u;  // no score yet
              const float fade = exp2_approx(m[n][j] - base);
              m[n][j] = u;
              sub[n][j] = base;
              lsum[n][j] *= fade;
#pragma unroll
              for (int c = 0; c < D / 16; ++c) acc[c][n][j] *= fade, acc[c][n][j + 2] *= fade;
            }
        }
      }
      // p as the sum of two bf16 values, the rounded weight and what that rounding left: relative 2^-16 at
      // most (each rounds by 2^-8), where the rounded weight alone is off by as much as the output's own rounding.
      uint32_t p[KT][NT][2], rest[KT][NT][2];
      const float up = decltype(careful)::value ? raise : kRaise;
#pragma unroll
      for (int i = 0; i < KT; ++i)
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          // times 2^kCarry, not the exponent plus kCarry: that sum would be rounded to 2^-19
          const float p0 = exp2_approx(s[i][n][0] - sub[n][0]) * up, p1 = exp2_approx(s[i][n][1] - sub[n][1]) * up;
          const float p2 = exp2_approx(s[i][n][2] - sub[n][0]) * up, p3 = exp2_approx(s[i][n][3] - sub[n][1]) * up;
          lsum[n][0] += p0 + p2;
          lsum[n][1] += p1 + p3;
          const uint32_t p01 = pack_bf16x2(p0, p1), p23 = pack_bf16x2(p2, p3);
          p[i][n][0] = transpose8x8(p01);
          p[i][n][1] = transpose8x8(p23);
          rest[i][n][0] = transpose8x8(pack_bf16x2(p0 - bf16_lo(p01), p1 - bf16_hi(p01)));
          rest[i][n][1] = transpose8x8(pack_bf16x2(p2 - bf16_lo(p23), p3 - bf16_hi(p23)));
        }
      // output
#pragma unroll
      for (int i = 0; i < KT; ++i) {
        uint32_t w[4][kVw], vs[4];  // keys t, t + 4, t + 8, t + 12
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int key = t + 4 * j;
          const uint32_t row = at + i * kTile + 16 * kRowBytes + key * kRowBytes;
#pragma unroll
          for (int c = 0; c < kVw; c += 4)
            lds_words<(kVw < 4 ? kVw : 4)>(row + ((4 * kVw * g + 4 * c) ^ (16 * attn_swizzle<D, kFmt, true>(key))), w[j] + c);
          vs[j] = lds_u8(at + i * kTile + 32 * kRowBytes + 16 * kGroups + key * kGroups + (g * D / 8) / 32);
          if constexpr (decltype(ragged)::value)
            if (!((have >> i) & 1) || (tile + i) * 16 + key >= len) {  // the bytes of no key may be anything
              vs[j] = 0;
#pragma unroll
              for (int c = 0; c < kVw; ++c) w[j][c] = 0;
            }
        }
        uint32_t va[D / 8], vb[D / 8];
        if constexpr (decltype(careful)::value) {
#pragma unroll 1
          for (int cls = 0; cls < 3; ++cls) {
            uint32_t f[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) f[j] = v_class_factor(vs[j], cls);
            if (!__any_sync(0xffffffffu, (f[0] | f[1] | f[2] | f[3]) != 0)) continue;
            v_pairs<D, kFmt, true>(w[0], w[1], f[0] | f[1] << 16, va, most);
            v_pairs<D, kFmt, true>(w[2], w[3], f[2] | f[3] << 16, vb, most);
            const float unit = cls == 0 ? 0x1p-64f : (cls == 1 ? 1.0f : 0x1p64f);
#pragma unroll
            for (int c = 0; c < D / 16; ++c)
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                float o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                mma_bf16_16816(o, va[2 * c], va[2 * c + 1], vb[2 * c], vb[2 * c + 1], p[i][n][0], p[i][n][1]);
                mma_bf16_16816(o, va[2 * c], va[2 * c + 1], vb[2 * c], vb[2 * c + 1], rest[i][n][0], rest[i][n][1]);
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[c][n][j] = fmaf(o[j], unit, acc[c][n][j]);
              }
          }
        } else {
          v_pairs<D, kFmt, false>(w[0], w[1], v_factor(vs[0], vs[1]), va, most);
          v_pairs<D, kFmt, false>(w[2], w[3], v_factor(vs[2], vs[3]), vb, most);
#pragma unroll
          for (int c = 0; c < D / 16; ++c)
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              mma_bf16_16816(acc[c][n], va[2 * c], va[2 * c + 1], vb[2 * c], vb[2 * c + 1], p[i][n][0], p[i][n][1]);
              mma_bf16_16816(acc[c][n], va[2 * c], va[2 * c + 1], vb[2 * c], vb[2 * c + 1], rest[i][n][0], rest[i][n][1]);
            }
        }
      }
    };
    auto walk = [&](auto careful) {
      int slot = 0;
#pragma unroll 1
      for (int tile = tile_first; tile < tile_last; tile += a.stride) {
        cp_async_wait<kRing - 2>();
        __syncwarp();  // every lane's copies have landed, and all lanes have left the slot copied into next
        copy_next();
        const uint32_t at = ring + slot * KT * kTile, have = (good >> (KT * (kRing - 1))) & ((1u << KT) - 1);
        slot = slot + 1 == kRing ? 0 : slot + 1;
        if constexpr (decltype(careful)::value) {
          if (have) do_step(tile, have, at, std::true_type{}, careful);
        } else if (have == (1u << KT) - 1 && (tile + KT) * 16 <= len) {
          do_step(tile, have, at, std::false_type{}, careful);
        } else if (have) {
          do_step(tile, have, at, std::true_type{}, careful);
        }
      }
      cp_async_wait<0>();
    };
    walk(std::false_type{});
    // A NaN code among the values, a scale out of the usual range, or a query that the operand does not hold:
    // this warp's steps once more, with care for them.  The first walk only follows whether there was one (a branch
    // for NaN codes in its loop cost 14 %, the largest code 6 %).
    if (__any_sync(0xffffffffu, has_nan_code(most))) {
      __syncwarp();  // all lanes have left the ring
      huge = __any_sync(0xffffffffu, most >= kHuge);
      if (huge) raise = kRaise * kHugeUnit;
      int deepest = 0;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        uint32_t amax = 0, least = 0x7F80u;  // magnitudes other than zero
        if (8 * n + g < nh)
#pragma unroll 1
          for (int d = 0; d < D; d += 32)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const uint32_t mag = reinterpret_cast<const uint16_t*>(q_at(n))[d + i] & 0x7FFFu;
              amax = max(amax, mag);
              if (mag) least = min(least, mag);
            }
#pragma unroll
        for (int x = 1; x < 4; x <<= 1) {
          amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, x));
          least = min(least, __shfl_xor_sync(0xffffffffu, least, x));
        }
        own_shift[n] = 14 + 127 - max(static_cast<int>(amax >> 7), 27);
        if (least < 0x7F80u) deepest = max(deepest, q_level(least, own_shift[n]));
#pragma unroll
        for (int j = 0; j < 2; ++j) shift_of[n][j] = __shfl_sync(0xffffffffu, own_shift[n], 4 * (2 * t + j));
      }
      levels = 1 + __reduce_max_sync(0xffffffffu, deepest);
      clear();
      copy_tile = tile_first, copy_slot = 0;
      first_pages();
#pragma unroll 1
      for (int i = 0; i < kRing - 1; ++i) copy_next();
      walk(std::true_type{});
    }
    // Not earlier: the blocks of a call after this one would fill up the SMs that are busy already.
    griddep_launch_dependents();
    __syncthreads();  // the rings become the buffer of the parts

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
        if (g == 0) sm_m[warp * kHeads + h] = m[n][j], sm_l[warp * kHeads + h] = huge ? l * (-1.0f / kHugeUnit) : l;
        float* dst = sm + (warp * kHeads + h) * kStride + g * (D / 8);
#pragma unroll
        for (int c = 0; c < D / 16; ++c)
          *reinterpret_cast<float2*>(dst + 2 * c) = make_float2(acc[c][n][j], acc[c][n][j + 2]);
      }
    __syncthreads();
    const bool whole = me.of == 1;
    if (!a.cluster && me.index == 0 && threadIdx.x == 0)
      a.heads[static_cast<size_t>(seq) * a.cache.heads * a.chunks + me.head_chunk] = make_int2(me.of, me.slot);
    float* part = a.cluster ? nullptr : a.parts + static_cast<size_t>(me.slot) * kHeads * (D + 2);
    for (int i = threadIdx.x; i < nh * (D / 4); i += kAttnThreads) {
      const int h = i / (D / 4), d = 4 * (i - h * (D / 4));
      float top = -kInf;
#pragma unroll
      for (int w = 0; w < kAttnWarps; ++w) top = fmaxf(top, sm_m[w * kHeads + h]);
      const float base = top == -kInf ? 0.0f : top;
      bool any = false;  // a part of small unit
#pragma unroll
      for (int w = 0; w < kAttnWarps; ++w) any |= sm_l[w * kHeads + h] < 0.0f;
      float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      float l = 0.0f;
#pragma unroll
      for (int w = 0; w < kAttnWarps; ++w) {
        const float f = exp2_approx(sm_m[w * kHeads + h] - base);
        const float4 x4 = *reinterpret_cast<const float4*>(sm + (w * kHeads + h) * kStride + d);
        const float lw = sm_l[w * kHeads + h], fo = part_factor(f, lw, any);
        l = fmaf(fabsf(lw), f, l);
        o.x = fmaf(x4.x, fo, o.x), o.y = fmaf(x4.y, fo, o.y), o.z = fmaf(x4.z, fo, o.z), o.w = fmaf(x4.w, fo, o.w);
      }
      l *= 1.0f / kRaise;
      if (whole) {
        const float r = l == 0.0f ? 0.0f : 1.0f / l;  // no key in reach (bad pages): zeros
        const size_t at = static_cast<size_t>(seq) * a.q_heads + h0 + h;
        *reinterpret_cast<uint2*>(a.out + at * D + d) = attn_output(o, r, any);
        if (a.lse && d == 0) a.lse[at] = l == 0.0f ? -kInf : (top + log2f(l)) * 0.6931471805599453f;
      } else if (a.cluster) {
        // over the first warp's part, which no other thread reads here
        *reinterpret_cast<float4*>(sm + h * kStride + d) = o;
        if (d == 0) sm_joined[h] = top, sm_joined[kHeads + h] = any ? -l : l;
      } else {
        *reinterpret_cast<float4*>(part + h * D + d) = o;
        if (d == 0) part[kHeads * D + 2 * h] = top, part[kHeads * D + 2 * h + 1] = any ? -l : l;
      }
    }
    if (a.cluster > 1) {  // every block of the cluster gets here: none returns before
      cluster_sync_all();
      for (int i = me.index * kAttnThreads + threadIdx.x; i < nh * (D / 4); i += a.cluster * kAttnThreads) {
        const int h = i / (D / 4), d = 4 * (i - h * (D / 4));
        float top = -kInf, m_of[8], l_of[8];  // all loads before the first use: each is a trip to another SM
        float4 o_of[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          m_of[c] = -kInf, l_of[c] = 0.0f, o_of[c] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          if (c < a.cluster) {
            m_of[c] = ld_dsmem_f32(sm_joined + h, c);
            l_of[c] = ld_dsmem_f32(sm_joined + kHeads + h, c);
            o_of[c] = ld_dsmem_f32x4(sm + h * kStride + d, c);
          }
        }
#pragma unroll
        for (int c = 0; c < 8; ++c) top = fmaxf(top, m_of[c]);
        const float base = top == -kInf ? 0.0f : top;
        bool any = false;
#pragma unroll
        for (int c = 0; c < 8; ++c) any |= l_of[c] < 0.0f;
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float l = 0.0f;
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          const float f = exp2_approx(m_of[c] - base), fo = part_factor(f, l_of[c], any);
          l = fmaf(fabsf(l_of[c]), f, l);
          o.x = fmaf(o_of[c].x, fo, o.x), o.y = fmaf(o_of[c].y, fo, o.y);
          o.z = fmaf(o_of[c].z, fo, o.z), o.w = fmaf(o_of[c].w, fo, o.w);
        }
        const float r = l == 0.0f ? 0.0f : 1.0f / l;
        const size_t at = static_cast<size_t>(seq) * a.q_heads + h0 + h;
        *reinterpret_cast<uint2*>(a.out + at * D + d) = attn_output(o, r, any);
        if (a.lse && d == 0) a.lse[at] = l == 0.0f ? -kInf : (top + log2f(l)) * 0.6931471805599453f;
      }
      cluster_sync_all();  // the others may still read this block's part
    }
  }
}

// Joins the parts of the heads of several pieces, in a fixed order, and writes the rows of empty
// sequences.  One block per (sequence, kv head, chunk) and query head; the parts are
// dealt to its lanes, D / 4 of them to a part.
template <int D, int NT>
__global__ void __launch_bounds__(kAttnThreads) attn_join_kernel(const __grid_constant__ AttnArgs a) {
  constexpr int kHeads = 8 * NT, kLanes = D / 4, kTeams = kAttnThreads / kLanes;
  constexpr float kInf = __builtin_huge_valf();
  __shared__ float4 sums[kTeams][kLanes];
  __shared__ float ls[kTeams];
  const int per = a.cache.heads * a.chunks;
  const int seq = blockIdx.x / per, hc = blockIdx.x - seq * per;
  const int head = hc / a.chunks, chunk = hc - head * a.chunks, h = blockIdx.y;
  if (h >= a.group - chunk * kHeads) return;
  const size_t at = static_cast<size_t>(seq) * a.q_heads + head * a.group + chunk * kHeads + h;
  const int team = threadIdx.x / kLanes, d = 4 * (threadIdx.x - team * kLanes);
  const bool empty = attn_length(a, seq) == 0;  // before the wait: attn_kernel's blocks have waited themselves
  griddep_wait();
  griddep_launch_dependents();
  if (empty) {
    if (team == 0) *reinterpret_cast<uint2*>(a.out + at * D + d) = make_uint2(0, 0);
    if (a.lse && threadIdx.x == 0) a.lse[at] = -kInf;
    return;
  }
  const int2 mine = a.heads[blockIdx.x];
  const int pieces = mine.x, slot = mine.y;
  if (pieces == 1) return;
  auto part_of = [&](int c) { return a.parts + static_cast<size_t>(slot + c) * kHeads * (D + 2); };
  float top = -kInf;
  bool any = false;  // a part of small unit
  for (int c = threadIdx.x & 31; c < pieces; c += 32) {
    const float2 ml = *reinterpret_cast<const float2*>(part_of(c) + kHeads * D + 2 * h);
    top = fmaxf(top, ml.x);
    any |= ml.y < 0.0f;
  }
  any = __any_sync(0xffffffffu, any);
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
  const float base = top == -kInf ? 0.0f : top;
  float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  float l = 0.0f;
#pragma unroll 4
  for (int c = team; c < pieces; c += kTeams) {
    const float* part = part_of(c);
    const float2 ml = *reinterpret_cast<const float2*>(part + kHeads * D + 2 * h);
    const float4 x4 = *reinterpret_cast<const float4*>(part + h * D + d);
    const float f = exp2_approx(ml.x - base), fo = part_factor(f, ml.y, any);
    l = fmaf(fabsf(ml.y), f, l);
    o.x = fmaf(x4.x, fo, o.x), o.y = fmaf(x4.y, fo, o.y), o.z = fmaf(x4.z, fo, o.z), o.w = fmaf(x4.w, fo, o.w);
  }
  sums[team][threadIdx.x - team * kLanes] = o;
  if (d == 0) ls[team] = l;
  __syncthreads();
  if (team != 0) return;
#pragma unroll
  for (int i = 1; i < kTeams; ++i) {
    const float4 x4 = sums[i][threadIdx.x];
    o.x += x4.x, o.y += x4.y, o.z += x4.z, o.w += x4.w;
    l += ls[i];
  }
  const float r = l == 0.0f ? 0.0f : 1.0f / l;
  *reinterpret_cast<uint2*>(a.out + at * D + d) = attn_output(o, r, any);
  if (a.lse && threadIdx.x == 0) a.lse[at] = l == 0.0f ? -kInf : (top + log2f(l)) * 0.6931471805599453f;
}

}  // namespace mxb
