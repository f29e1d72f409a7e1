// Head rows between the QKV GEMM and the attention: per-head RMS norm, rotation, and the MX
// key-value cache those rows are coded into and read back from.
//
// A row is one head of one token, D bf16 values (D % 32 == 0, D <= 256).  A lane holds 8
// neighbouring values (one 16-byte load), so a row takes LPR = 4, 8, 16 or 32 lanes and a warp
// works on 32 / LPR rows of one kind (q, k or v) at a time.
//
//   norm      y_i = x_i * w_i / sqrt(mean(x^2) + eps)
//   rotation  of the first R values with c = cos[p][i], s = sin[p][i], i < R/2:
//             halves       (y_i, y_{i+R/2})   -> (y_i c - y_{i+R/2} s, y_{i+R/2} c + y_i s)
//             interleaved  (y_{2i}, y_{2i+1}) -> the same of the neighbouring pair
//   coding    per group of 32 values: e = floor(log2(amax)) - top clipped to [-127, 127]
//             (top = 8 for E4M3, 2 for E2M1; -127 for an all-zero group), codes = the values
//             * 2^-e rounded to nearest even and saturated at 448 / 6, scale byte e + 127.  A
//             group that holds a NaN gets the scale byte 255, which reads back as NaN.
//
// Cache layout, per (page, kv head): page_size rows of D codes (E4M3) or D/2 bytes (E2M1, even
// element in the low nibble) and, in an array of its own, D/32 scale bytes per row.
#pragma once

#include "common.cuh"
#include "gemm_mx.cuh"
#include "quant.cuh"

namespace mxb {

constexpr int kFmtNone = 0, kFmtE4M3 = 1, kFmtE2M1 = 2;

struct KvCacheView {
  uint8_t *k_codes, *v_codes, *k_scales, *v_scales;
  int num_pages, heads, page_shift, dim;
  __device__ __forceinline__ long long slots() const { return static_cast<long long>(num_pages) << page_shift; }
  // index of the row of (slot, head) in units of rows
  __device__ __forceinline__ size_t row(int slot, int head) const {
    const size_t page = static_cast<size_t>(slot >> page_shift);
    return ((page * heads + head) << page_shift) + (slot & ((1 << page_shift) - 1));
  }
};

struct RowArgs {
  const __nv_bfloat16 *q, *k, *v;            // first head of the first token of each kind
  long long q_stride, k_stride, v_stride;    // elements from one token to the next
  int tokens, q_heads, kv_heads, dim;
  const float *cos, *sin;                    // [table_rows][rot / 2]; rot == 0: no rotation
  int table_rows, rot, interleaved;
  const int* positions;                      // table row of each token; null: the token's index
  const void *q_weight, *k_weight;           // [dim]; null: no norm
  int weight_f32;
  double eps;
  __nv_bfloat16 *q_out, *k_out;              // [tokens][heads][dim]
  KvCacheView cache;
  const int* slots;                          // cache row of each token; negative: not stored
};

// Eight values of a 16-byte load of bf16.
template <typename Real>
__device__ __forceinline__ void unpack_bf16x8(const uint4& u, Real (&v)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}

template <typename Real>
__device__ __forceinline__ void load_weight8(const void* w, int f32, int at, Real (&v)[8]) {
  if (f32) {
    const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(w) + at);
    const float4 a = __ldg(p), b = __ldg(p + 1);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  } else {
    unpack_bf16x8(__ldg(reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(w) + at)), v);
  }
}

__device__ __forceinline__ float inv_sqrt(float x) { return rsqrtf(x); }
__device__ __forceinline__ double inv_sqrt(double x) { return rsqrt(x); }

// Norm and rotation of one row in the precision of Real: x are the lane's 8 values, c and s its
// cos / sin (8 of them for the halves form, the first 4 for the interleaved one).  Every lane of
// the warp takes part (shuffles); lanes past the row hold zeros.
template <int LPR, typename Real>
__device__ __forceinline__ void norm_rotate(const RowArgs& a, const uint4& x, const void* weight, const float (&c)[8],
                                            const float (&s)[8], Real (&y)[8]) {
  const int l = threadIdx.x & (LPR - 1), at = 8 * l;
  const bool live = at < a.dim;
  unpack_bf16x8(x, y);
  Real r = 1;
  if (weight) {
    Real ss = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss += y[i] * y[i];
#pragma unroll
    for (int m = LPR / 2; m > 0; m >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, m);
    r = inv_sqrt(ss / static_cast<Real>(a.dim) + static_cast<Real>(a.eps));
    if (live) {
      Real w[8];
      load_weight8(weight, a.weight_f32, at, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = y[i] * r * w[i];
    }
  }
  if (a.rot == 0) return;
  if (a.interleaved) {
    if (at < a.rot) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const Real u = y[2 * i], v = y[2 * i + 1];
        y[2 * i] = u * static_cast<Real>(c[i]) - v * static_cast<Real>(s[i]);
        y[2 * i + 1] = v * static_cast<Real>(c[i]) + u * static_cast<Real>(s[i]);
      }
    }
    return;
  }
  // halves: the partner's values come as the packed input (4 shuffles) and are normed here too
  const int half = a.rot >> 1, lane = threadIdx.x & 31;
  const bool rotated = at < a.rot, low = at < half;
  const int src = rotated ? (low ? lane + (half >> 3) : lane - (half >> 3)) : lane;
  uint4 px;
  px.x = __shfl_sync(0xffffffffu, x.x, src);
  px.y = __shfl_sync(0xffffffffu, x.y, src);
  px.z = __shfl_sync(0xffffffffu, x.z, src);
  px.w = __shfl_sync(0xffffffffu, x.w, src);
  if (!rotated) return;
  Real z[8];
  unpack_bf16x8(px, z);
  if (weight) {
    Real w[8];
    load_weight8(weight, a.weight_f32, low ? at + half : at - half, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) z[i] = z[i] * r * w[i];
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const Real sn = low ? -static_cast<Real>(s[i]) : static_cast<Real>(s[i]);
    y[i] = y[i] * static_cast<Real>(c[i]) + z[i] * sn;
  }
}

// A double as a float rounded to odd: truncated, the last bit set when anything was cut off.  A
// later rounding to fewer bits then equals the rounding of the double itself.
__device__ __forceinline__ float round_odd(double d) {
  const float f = __double2float_rz(d);
  return static_cast<double>(f) == d ? f : __uint_as_float(__float_as_uint(f) | 1u);
}
__device__ __forceinline__ float round_odd(float f) { return f; }

__device__ __forceinline__ uint32_t e2m1x2(float lo, float hi) {
  uint32_t r;
  asm("{\n\t.reg .b8 t;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 t, %1, %2;\n\t"
      "cvt.u32.u8 %0, t;\n\t}"
      : "=r"(r)
      : "f"(hi), "f"(lo));
  return r;
}

// Codes the lane's 8 values as part of their 32-value group (4 lanes) and writes codes and scale.
template <int kFmt, typename Real>
__device__ __forceinline__ void code_and_store(const Real (&y)[8], bool live, size_t row, int dim, int at,
                                               uint8_t* codes, uint8_t* scales) {
  float f[8];
  uint32_t amax = 0;  // of the magnitudes' bits: a NaN sorts above infinity
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    f[i] = round_odd(y[i]);
    amax = max(amax, __float_as_uint(f[i]) & 0x7FFFFFFFu);
  }
  amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
  amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
  const bool nan = amax > 0x7F800000u;
  // biased exponent field = floor(log2(amax)) + 127 (0 for zero and subnormals, which clip anyway)
  const int byte = max(static_cast<int>(amax >> 23) - (kFmt == kFmtE4M3 ? 8 : 2), 0);
  const float inv = nan ? 0.0f : exp2_neg(byte - 127);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = nan ? 0.0f : f[i] * inv;
  if (!live) return;
  if (kFmt == kFmtE4M3) {
    uint2 o;
    o.x = e4m3x2(f[0], f[1]) | (e4m3x2(f[2], f[3]) << 16);
    o.y = e4m3x2(f[4], f[5]) | (e4m3x2(f[6], f[7]) << 16);
    *reinterpret_cast<uint2*>(codes + row * dim + at) = o;
  } else {
    // + 0.0f: a negative zero is coded as zero, as mxfp4_quantize does
    uint32_t o = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) o |= e2m1x2(f[2 * i] + 0.0f, f[2 * i + 1] + 0.0f) << (8 * i);
    *reinterpret_cast<uint32_t*>(codes + row * (dim / 2) + at / 2) = o;
  }
  if ((at & 31) == 0) scales[row * (dim / 32) + at / 32] = static_cast<uint8_t>(nan ? 255 : byte);
}

constexpr int kRowThreads = 128;

// One token per blockIdx.x, a share of its head rows per blockIdx.y.
//
// Bound by HBM: each row is read once and written once.  q is computed in 32 bits and rounded to
// bf16 once.  A key on its way into the cache is computed in 64 bits: next to a rounding border
// an error in the 24th bit would pick the neighbouring code, and with it the stored byte would
// depend on how the norm's sum was ordered.  Its few rows (kv_heads of q_heads + 2 kv_heads) hide
// behind the loads.
//
// Two tokens of one launch that name the same slot: the later one is stored (every block looks
// through the slots behind its own; the caller keeps a launch to 4096 tokens).
template <int LPR, int kFmt>
__global__ void __launch_bounds__(kRowThreads) head_rows_kernel(const __grid_constant__ RowArgs a, int first) {
  constexpr int kRows = 32 / LPR;  // rows a warp works on at a time
  const int t = first + blockIdx.x;
  const int warp = (blockIdx.y * kRowThreads + threadIdx.x) >> 5, warps = gridDim.y * (kRowThreads / 32);
  const int lane = threadIdx.x & 31, l = lane & (LPR - 1), sub = lane / LPR, at = 8 * l;
  const bool live = at < a.dim;

  bool good = true;
  float c[8], s[8];
  if (a.rot) {
    const int p = a.positions ? __ldg(a.positions + t) : t;
    good = p >= 0 && p < a.table_rows;
    if (!good && threadIdx.x == 0) record_error(kErrBadPosition);
    if (good && at < a.rot) {
      const int half = a.rot >> 1;
      const int i0 = a.interleaved ? at >> 1 : (at < half ? at : at - half);
      const float4* pc = reinterpret_cast<const float4*>(a.cos + static_cast<size_t>(p) * half + i0);
      const float4* ps = reinterpret_cast<const float4*>(a.sin + static_cast<size_t>(p) * half + i0);
      const float4 c0 = __ldg(pc), s0 = __ldg(ps);
      c[0] = c0.x, c[1] = c0.y, c[2] = c0.z, c[3] = c0.w, s[0] = s0.x, s[1] = s0.y, s[2] = s0.z, s[3] = s0.w;
      if (!a.interleaved) {
        const float4 c1 = __ldg(pc + 1), s1 = __ldg(ps + 1);
        c[4] = c1.x, c[5] = c1.y, c[6] = c1.z, c[7] = c1.w, s[4] = s1.x, s[5] = s1.y, s[6] = s1.z, s[7] = s1.w;
      }
    }
  }
  int slot = -1;
  if (kFmt != kFmtNone) {
    slot = __ldg(a.slots + t);
    if (slot >= a.cache.slots()) {
      if (threadIdx.x == 0) record_error(kErrBadSlot);
      slot = -1;
    }
    if (!good) slot = -1;
    bool later = false;
    if (slot >= 0)
      for (int u = blockIdx.x + 1 + threadIdx.x; u < gridDim.x; u += kRowThreads) later |= __ldg(a.slots + first + u) == slot;
    if (__syncthreads_or(later)) slot = -1;
  }

  const int q_groups = ceil_div(a.q_heads, kRows), kv_groups = ceil_div(a.kv_heads, kRows);
  const int groups = q_groups + kv_groups * (kFmt != kFmtNone ? 2 : 1);
  for (int g = warp; g < groups; g += warps) {
    const int kind = g < q_groups ? 0 : (g < q_groups + kv_groups ? 1 : 2);
    const int h = (kind == 0 ? g : kind == 1 ? g - q_groups : g - q_groups - kv_groups) * kRows + sub;
    const int heads = kind == 0 ? a.q_heads : a.kv_heads;
    const bool here = live && h < heads;
    if (kFmt != kFmtNone && kind != 0 && slot < 0) continue;
    uint4 x = make_uint4(0, 0, 0, 0);
    if (here) {
      const __nv_bfloat16* src = kind == 0 ? a.q + a.q_stride * t : kind == 1 ? a.k + a.k_stride * t : a.v + a.v_stride * t;
      x = *reinterpret_cast<const uint4*>(src + static_cast<size_t>(h) * a.dim + at);
    }
    if (kind == 0 || (kind == 1 && kFmt == kFmtNone)) {
      float y[8];
      norm_rotate<LPR, float>(a, x, kind == 0 ? a.q_weight : a.k_weight, c, s, y);
      if (here) {
        uint4 o = make_uint4(0, 0, 0, 0);
        if (good)
          o = make_uint4(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]), pack_bf16x2(y[4], y[5]),
                         pack_bf16x2(y[6], y[7]));
        __nv_bfloat16* dst = kind == 0 ? a.q_out : a.k_out;
        *reinterpret_cast<uint4*>(dst + (static_cast<size_t>(t) * heads + h) * a.dim + at) = o;
      }
    } else if (kFmt != kFmtNone) {
      const size_t row = here ? a.cache.row(slot, h) : 0;
      if (kind == 1) {
        double y[8];
        norm_rotate<LPR, double>(a, x, a.k_weight, c, s, y);
        code_and_store<kFmt>(y, here, row, a.dim, at, a.cache.k_codes, a.cache.k_scales);
      } else {
        float y[8];
        unpack_bf16x8(x, y);
        code_and_store<kFmt>(y, here, row, a.dim, at, a.cache.v_codes, a.cache.v_scales);
      }
    }
  }
}

// E8M0 byte as fp32: 2^(b-127), 255 is NaN.
__device__ __forceinline__ float e8m0_value(uint32_t b) {
  return b == 255u ? __uint_as_float(0x7FC00000u) : e8m0_to_f32(b);
}

// Eight codes (8 bytes of E4M3, 4 of E2M1) times their scale, as bf16.
template <int kFmt>
__device__ __forceinline__ uint4 decode8(const uint2& w, float scale) {
  uint32_t h[4];
  if (kFmt == kFmtE4M3) {
    const uint32_t p[4] = {w.x & 0xFFFFu, w.x >> 16, w.y & 0xFFFFu, w.y >> 16};
#pragma unroll
    for (int i = 0; i < 4; ++i) asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h[i]) : "h"(static_cast<uint16_t>(p[i])));
  } else {
    e2m1x8_to_f16x2(w.x, h);
  }
  uint32_t o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
    o[i] = pack_bf16x2(f.x * scale, f.y * scale);
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}

constexpr int kReadThreads = 128;
constexpr int kReadRows = 4;  // rows per block, their loads in flight together

// k and v of the cache rows that `slots` names, [rows][heads][dim] bf16; a negative slot reads zeros.
template <int kFmt>
__global__ void __launch_bounds__(kReadThreads)
    kv_read_kernel(const __grid_constant__ KvCacheView cache, const int* __restrict__ slots, int rows,
                   __nv_bfloat16* __restrict__ k, __nv_bfloat16* __restrict__ v) {
  const int per_head = cache.dim / 8, units = cache.heads * per_head;
  const int r0 = blockIdx.x * kReadRows;
  int slot[kReadRows];
#pragma unroll
  for (int r = 0; r < kReadRows; ++r) {
    slot[r] = r0 + r < rows ? __ldg(slots + r0 + r) : -1;
    if (slot[r] >= cache.slots()) {
      if (threadIdx.x == 0) record_error(kErrBadSlot);
      slot[r] = -1;
    }
  }
  for (int u = threadIdx.x; u < units; u += kReadThreads) {
    const int h = u / per_head, at = 8 * (u - h * per_head);
    uint2 wk[kReadRows], wv[kReadRows];
    uint32_t sk[kReadRows], sv[kReadRows];
#pragma unroll
    for (int r = 0; r < kReadRows; ++r) {
      wk[r] = wv[r] = make_uint2(0, 0);
      sk[r] = sv[r] = 127;
      if (slot[r] >= 0) {
        const size_t row = cache.row(slot[r], h);
        if (kFmt == kFmtE4M3) {
          wk[r] = *reinterpret_cast<const uint2*>(cache.k_codes + row * cache.dim + at);
          wv[r] = *reinterpret_cast<const uint2*>(cache.v_codes + row * cache.dim + at);
        } else {
          wk[r].x = *reinterpret_cast<const uint32_t*>(cache.k_codes + row * (cache.dim / 2) + at / 2);
          wv[r].x = *reinterpret_cast<const uint32_t*>(cache.v_codes + row * (cache.dim / 2) + at / 2);
        }
        sk[r] = cache.k_scales[row * (cache.dim / 32) + at / 32];
        sv[r] = cache.v_scales[row * (cache.dim / 32) + at / 32];
      }
    }
#pragma unroll
    for (int r = 0; r < kReadRows; ++r) {
      if (r0 + r >= rows) break;
      const size_t dst = static_cast<size_t>(r0 + r) * units * 8 + static_cast<size_t>(u) * 8;
      *reinterpret_cast<uint4*>(k + dst) = decode8<kFmt>(wk[r], e8m0_value(sk[r]));
      *reinterpret_cast<uint4*>(v + dst) = decode8<kFmt>(wv[r], e8m0_value(sv[r]));
    }
  }
}

}  // namespace mxb
