// The residual's addition with the RMSNorm behind it, and the norm's 8-bit form, in one pass for gfx950 (a decoder layer of the
// reference adds first, in a tensor expression, and launches its norm on the sum: src/loquetier_src/models/mixed_llama.py:53-66).
//
//   h = round16(x + residual),  y = h w / sqrt(mean h^2 + eps),  out = round16(y),  out8 = e4m3(y / scale),  scale = max |y| / 448
//
// by row or by 128 columns.  The norm is of h as it is stored, as a norm launched on the stored sum would have it, so the residual
// stream and the backward see the same h.  y is rounded once for each of its forms: y / scale is the correctly rounded quotient (a product
// with 1 / scale is not, and of 8.65 million codes 248 were the neighbour of the quotient's).  448 is the largest e4m3, so the largest of a
// group becomes it; a group whose scale is below the normal floats is zeros with a scale of 0.  An infinite y makes the scale infinite, NaN makes it NaN.
//
// Bound by HBM: 4 bytes read and 4 written an element, 5 with the 8-bit form.  A row stays in registers from its sum to its last
// output.  The backward is rms_norm.hpp's, to which the gradient that reaches h through the residual is added.  (4096 columns: 4096
// rows bf16 23.2 us, 5.8 TB/s, backward 26.4, 5.1, and its fold 3.9; 2112 rows with e4m3 by 128 columns 17.3, 4.5 (16.6 with
// products for quotients); 256 rows with e4m3 by row 4.4.)
#pragma once
#include "rms_norm.hpp"

namespace smlm {

struct AddRmsArgs {
  uint16_t* out;             // [rows, cols] or NULL
  float* rms;                // [rows] or NULL
  uint16_t* h;               // [rows, cols] or NULL (without a residual)
  const uint16_t* x;         // [rows, cols]
  const uint16_t* residual;  // [rows, cols] or NULL
  const uint16_t* w;         // [cols]
  uint8_t* out8;             // [rows, cols] or NULL
  float* scale;              // [rows], or [rows, cols / 128]
  int rows, cols, grouped;
  float eps;
};

constexpr float kMostE4m3 = 448.0f;

// The larger, NaN if either is.
__device__ __forceinline__ float max_or_nan(float a, float b) { return __builtin_elementwise_maximum(a, b); }
// Over the sixteen lanes of a row of lanes, in every lane of it.
__device__ __forceinline__ float row_max16(float x) {
#define SMLM_ROW_MAX(n) \
  x = max_or_nan(x, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x120 + n, 0xf, 0xf, false)))
  SMLM_ROW_MAX(8);  // row_ror
  SMLM_ROW_MAX(4);
  SMLM_ROW_MAX(2);
  SMLM_ROW_MAX(1);
#undef SMLM_ROW_MAX
  return x;
}
__device__ __forceinline__ float wave_max(float x) {
  x = row_max16(x);
  auto lane = [&](int l) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), l)); };
  return max_or_nan(max_or_nan(lane(0), lane(16)), max_or_nan(lane(32), lane(48)));
}
// A group's scale from its largest value, and what its values are divided by: that, and one over it (0 and 0 of an infinite scale: finite
// values become 0).
__device__ __forceinline__ float scale8(float most, float& by, float& inv) {
  float s = most * (1.0f / kMostE4m3);
  if (s < 0x1p-126f) s = 0.0f;
  inv = s == 0.0f ? 0.0f : 1.0f / s;
  by = s < INFINITY ? s : 0.0f;
  return s;
}
// x / s, correctly rounded, from the correctly rounded inv = 1 / s: the remainder of the first guess corrects it (Markstein's
// theorem; x / s is at most 448 and s is normal).  s 0 with inv 0: 0, and NaN of an infinity or NaN.
__device__ __forceinline__ float divide8(float x, float s, float inv) {
  const float q = x * inv;
  return __builtin_fmaf(__builtin_fmaf(-q, s, x), inv, q);
}
__device__ __forceinline__ uint32_t pack8(float a, float b, float c, float d) {
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false), true);
}

// WPR waves share a row (1 or 4), CH pieces of 512 columns a wave, eight columns a lane; a workgroup takes 4 / WPR rows.
template <int DT, int WPR, int CH>
__global__ __launch_bounds__(256) void add_rms_kernel(AddRmsArgs a) {
  __shared__ float part[2][4];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, sub = wave % WPR;
  const int row = (int)blockIdx.x * (4 / WPR) + wave / WPR;
  if (row >= a.rows) return;  // (WPR 4: the whole workgroup)
  const int64_t at = (int64_t)row * a.cols;
  bool ok[CH];
  int col[CH];
  u32x4 hv[CH], rv[CH], wv[CH];
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    col[i] = ((i * WPR + sub) * 64 + lane) * 8;
    ok[i] = col[i] < a.cols;
    if (!ok[i]) col[i] = 0;
    hv[i] = ldg16_nt(a.x + at + col[i]);
  }
  if (a.residual) {
#pragma unroll
    for (int i = 0; i < CH; ++i) rv[i] = ldg16_nt(a.residual + at + col[i]);
  }
#pragma unroll
  for (int i = 0; i < CH; ++i) wv[i] = ldg16(a.w + col[i]);
  if (a.residual) {
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      float f[8], g[8];
      unpack8<DT>(hv[i], f);
      unpack8<DT>(rv[i], g);
#pragma unroll
      for (int e = 0; e < 4; ++e) hv[i][e] = pack2<DT>(f[2 * e] + g[2 * e], f[2 * e + 1] + g[2 * e + 1]);
      if (ok[i] && a.h) stg16_nt(a.h + at + col[i], hv[i]);
    }
  }
  float ss = 0.0f;
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    float f[8], s = 0.0f;
    unpack8<DT>(hv[i], f);
#pragma unroll
    for (int e = 0; e < 8; ++e) s += f[e] * f[e];
    ss += ok[i] ? s : 0.0f;
  }
  ss = wave_sum_f32(ss);
  if (WPR > 1) {
    if (lane == 0) part[0][wave] = ss;
    __syncthreads();
    ss = (part[0][0] + part[0][1]) + (part[0][2] + part[0][3]);
  }
  const float rms = 1.0f / sqrtf(ss / (float)a.cols + a.eps);
  if (a.rms && lane == 0 && sub == 0) a.rms[row] = rms;
  float by = 0.0f, inv = 0.0f;
  if (a.out8 && !a.grouped) {
    float most = 0.0f;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      float f[8], g[8], m = 0.0f;
      unpack8<DT>(hv[i], f);
      unpack8<DT>(wv[i], g);
#pragma unroll
      for (int e = 0; e < 8; ++e) m = max_or_nan(m, fabsf(f[e] * rms * g[e]));
      if (ok[i]) most = max_or_nan(most, m);
    }
    most = wave_max(most);
    if (WPR > 1) {
      if (lane == 0) part[1][wave] = most;
      __syncthreads();
      most = max_or_nan(max_or_nan(part[1][0], part[1][1]), max_or_nan(part[1][2], part[1][3]));
    }
    const float s = scale8(most, by, inv);
    if (lane == 0 && sub == 0) a.scale[row] = s;
  }
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    float f[8], g[8];
    unpack8<DT>(hv[i], f);
    unpack8<DT>(wv[i], g);
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = f[e] * rms * g[e];
    if (a.out && ok[i]) {
      u32x4 o;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = pack2<DT>(f[2 * e], f[2 * e + 1]);
      stg16_nt(a.out + at + col[i], o);
    }
    if (a.out8) {
      if (a.grouped) {  // sixteen lanes hold a group (columns are a multiple of 128: all of them or none)
        float m = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) m = max_or_nan(m, fabsf(f[e]));
        const float s = scale8(row_max16(m), by, inv);
        if (ok[i] && (lane & 15) == 0) a.scale[(int64_t)row * (a.cols >> 7) + (col[i] >> 7)] = s;
      }
      if (ok[i]) {
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = divide8(f[e], by, inv);
        const u32x2 o = {pack8(f[0], f[1], f[2], f[3]), pack8(f[4], f[5], f[6], f[7])};
        __builtin_nontemporal_store(o, (SMLM_GLOBAL u32x2*)(a.out8 + at + col[i]));
      }
    }
  }
}

// Rows of more than kRmsMaxCols columns: a workgroup a row, which reads the sum again for each of the sweeps (from the caches).
template <int DT>
__global__ __launch_bounds__(256) void add_rms_wide_kernel(AddRmsArgs a) {
  __shared__ float red4[4];
  for (int row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const int64_t at = (int64_t)row * a.cols;
    auto sum = [&](int col, float (&f)[8]) {
      unpack8<DT>(ldg16(a.x + at + col), f);
      if (!a.residual) return;
      float g[8];
      unpack8<DT>(ldg16(a.residual + at + col), g);
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const uint32_t two = pack2<DT>(f[e] + g[e], f[e + 1] + g[e + 1]);
        f[e] = Num<DT>::lo(two), f[e + 1] = Num<DT>::hi(two);
      }
    };
    // (h and out may lie where x or the residual does: what the later sweeps read is h, or not written before they are done)
    const bool kept = a.residual && a.h;
    auto again = [&](int col, float (&f)[8]) {
      if (kept) unpack8<DT>(ldg16(a.h + at + col), f);
      else sum(col, f);
    };
    float ss = 0.0f;
    for (int col = threadIdx.x * 8; col < a.cols; col += 256 * 8) {
      float f[8];
      sum(col, f);
#pragma unroll
      for (int e = 0; e < 8; ++e) ss += f[e] * f[e];
      if (kept) {
        u32x4 o;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = pack2<DT>(f[2 * e], f[2 * e + 1]);
        stg16(a.h + at + col, o);
      }
    }
    ss = block_sum_f32(ss, red4);
    const float rms = 1.0f / sqrtf(ss / (float)a.cols + a.eps);
    if (a.rms && threadIdx.x == 0) a.rms[row] = rms;
    float by = 0.0f, inv = 0.0f;
    if (a.out8 && !a.grouped) {
      float most = 0.0f;
      for (int col = threadIdx.x * 8; col < a.cols; col += 256 * 8) {
        float f[8], g[8];
        again(col, f);
        unpack8<DT>(ldg16(a.w + col), g);
#pragma unroll
        for (int e = 0; e < 8; ++e) most = max_or_nan(most, fabsf(f[e] * rms * g[e]));
      }
      most = wave_max(most);
      __syncthreads();
      if ((threadIdx.x & 63) == 0) red4[threadIdx.x >> 6] = most;
      __syncthreads();
      const float s = scale8(max_or_nan(max_or_nan(red4[0], red4[1]), max_or_nan(red4[2], red4[3])), by, inv);
      if (threadIdx.x == 0) a.scale[row] = s;
    }
    for (int c0 = 0; c0 < a.cols; c0 += 256 * 8) {  // (all lanes stay: groups of sixteen of them meet)
      const int mine = c0 + (int)threadIdx.x * 8, col = mine < a.cols ? mine : 0;
      const bool ok = mine < a.cols;
      float f[8], g[8];
      again(col, f);
      unpack8<DT>(ldg16(a.w + col), g);
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = f[e] * rms * g[e];
      if (a.out && ok) {
        u32x4 o;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = pack2<DT>(f[2 * e], f[2 * e + 1]);
        stg16(a.out + at + col, o);
      }
      if (a.out8) {
        if (a.grouped) {
          float m = 0.0f;
#pragma unroll
          for (int e = 0; e < 8; ++e) m = max_or_nan(m, fabsf(f[e]));
          const float s = scale8(row_max16(m), by, inv);
          if (ok && (threadIdx.x & 15) == 0) a.scale[(int64_t)row * (a.cols >> 7) + (col >> 7)] = s;
        }
        if (ok) {
#pragma unroll
          for (int e = 0; e < 8; ++e) f[e] = divide8(f[e], by, inv);
          *(SMLM_GLOBAL u32x2*)(a.out8 + at + col) = u32x2{pack8(f[0], f[1], f[2], f[3]), pack8(f[4], f[5], f[6], f[7])};
        }
      }
    }
  }
}

}  // namespace smlm
