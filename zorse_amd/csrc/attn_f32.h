// What the fp32 attention kernels share (attn_f32.hip, attn_packed_f32.hip): 16
// rows of one side per wave, the other side in LDS tiles of 32 rows.
#pragma once
#include <initializer_list>

#include "attn_common.h"
#include "vec.h"

namespace zk {

namespace {

constexpr int kTile = 32;  // rows per LDS tile

// Rows r0 .. r0 + ROWS - 1 (of `rows`) of a [.., d] tensor, spread over THREADS:
// load() issues the global loads, store() writes the LDS tile.
template <int D, bool kVec, int ROWS = kTile, int THREADS = 256>
struct TileReg {
  static constexpr int NC = ROWS * D / 4 / THREADS;  // 4-float chunks per thread
  float4 v[NC];
  __device__ __forceinline__ void load(const float* base, int64_t ld, int64_t r0, int64_t rows, int d) {
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int id = i * THREADS + static_cast<int>(threadIdx.x);
      const int r = id / (D / 4), c = 4 * (id % (D / 4));
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
      if (r0 + r < rows && c < d) {
        const float* p = base + (r0 + r) * ld + c;
        if (kVec) {
          x = *reinterpret_cast<const float4*>(p);
        } else {
          x.x = p[0];
          if (c + 1 < d) x.y = p[1];
          if (c + 2 < d) x.z = p[2];
          if (c + 3 < d) x.w = p[3];
        }
      }
      v[i] = x;
    }
  }
  // returns whether one of this thread's values is an infinity or NaN
  __device__ __forceinline__ int store(float* tile) const {
    float z = 0.f;  // stays 0 for finite values, else NaN
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int id = i * THREADS + static_cast<int>(threadIdx.x);
      *reinterpret_cast<float4*>(&tile[(id / (D / 4)) * (D + 4) + 4 * (id % (D / 4))]) = v[i];
      z += 0.f * v[i].x + 0.f * v[i].y + 0.f * v[i].z + 0.f * v[i].w;
    }
    return z != 0.f;
  }
};

// This lane's operand of row `row` (null: zeros): elements 16 c + 4 q4 .. + 3.
template <int D, bool kVec>
__device__ __forceinline__ void load_row(float4 (&x)[D / 16], const float* row, int d) {
  const int q4 = (threadIdx.x & 63) >> 4;
#pragma unroll
  for (int c = 0; c < D / 16; ++c) {
    const int e = 16 * c + 4 * q4;
    x[c] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (row == nullptr || e >= d) continue;
    if (kVec) {
      x[c] = *reinterpret_cast<const float4*>(row + e);
    } else {
      x[c].x = row[e];
      if (e + 1 < d) x[c].y = row[e + 1];
      if (e + 2 < d) x[c].z = row[e + 2];
      if (e + 3 < d) x[c].w = row[e + 3];
    }
  }
}

__device__ __forceinline__ f32x4 mma4(float a, float b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

// X Y^T over d of the LDS rows row0 .. + 15 (X) and this lane's operand y.
template <int D>
__device__ __forceinline__ f32x4 dot_rows(const float* tile, int row0, const float4 (&y)[D / 16]) {
  const int l16 = threadIdx.x & 15, q4 = (threadIdx.x & 63) >> 4;
  const float* p = tile + (row0 + l16) * (D + 4) + 4 * q4;
  f32x4 s{};
#pragma unroll
  for (int c = 0; c < D / 16; ++c) {
    const float4 x = *reinterpret_cast<const float4*>(p + 16 * c);
    s = mma4(x.x, y[c].x, s);
    s = mma4(x.y, y[c].y, s);
    s = mma4(x.z, y[c].z, s);
    s = mma4(x.w, y[c].w, s);
  }
  return s;
}

// acc^T += X^T w over the 16 LDS rows row0 ..: w[e] belongs to row 4 q4 + e.
template <int D>
__device__ __forceinline__ void add_rows(f32x4 (&acc)[D / 16], const float* tile, int row0,
                                         const f32x4& w) {
  const int l16 = threadIdx.x & 15, q4 = (threadIdx.x & 63) >> 4;
  const float* p = tile + (row0 + 4 * q4) * (D + 4) + l16;
#pragma unroll
  for (int e = 0; e < 4; ++e)
#pragma unroll
    for (int nt = 0; nt < D / 16; ++nt)
      acc[nt] = mma4(p[e * (D + 4) + 16 * nt], w[e], acc[nt]);
}

// The same for a tile that holds an infinity or NaN, where a product with the
// zero weight of a masked row would be NaN: row by row, masked rows left out.
template <int D, typename Vis>
__device__ __forceinline__ void add_rows_visible(f32x4 (&acc)[D / 16], const float* tile, int row0,
                                              const f32x4& w, Vis visible) {
  const int l16 = threadIdx.x & 15, q4 = (threadIdx.x & 63) >> 4;
  for (int r = 0; r < 16; ++r) {
    float wr = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) wr = (r & 3) == e ? w[e] : wr;
    wr = __shfl(wr, (r >> 2) * 16 + l16, 64);
    if (!visible(row0 + r)) continue;
#pragma unroll
    for (int nt = 0; nt < D / 16; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        acc[nt][e] = fmaf(wr, tile[(row0 + r) * (D + 4) + 16 * nt + 4 * q4 + e], acc[nt][e]);
  }
}

// sum / max over the four lane groups that share a column
__device__ __forceinline__ float group_sum(float x) {
  x += __shfl_xor(x, 16, 64);
  return x + __shfl_xor(x, 32, 64);
}
__device__ __forceinline__ float group_max(float x) {
  x = fmaxf(x, __shfl_xor(x, 16, 64));
  return fmaxf(x, __shfl_xor(x, 32, 64));
}

// This lane's accumulators (elements 16 (nt0 + nt) + 4 q4 + e of its row), scaled,
// to the row at dst.
template <int D, bool kVec, int N = D / 16>
__device__ __forceinline__ void store_row(float* dst, const f32x4 (&x)[N], float scale, int d,
                                          int nt0 = 0) {
  const int q4 = (threadIdx.x & 63) >> 4;
#pragma unroll
  for (int nt = 0; nt < N; ++nt) {
    const int e0 = 16 * (nt0 + nt) + 4 * q4;
    if (kVec) {
      if (e0 < d)
        *reinterpret_cast<float4*>(dst + e0) = make_float4(x[nt][0] * scale, x[nt][1] * scale,
                                                           x[nt][2] * scale, x[nt][3] * scale);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e0 + e < d) dst[e0 + e] = x[nt][e] * scale;
    }
  }
}

// float4 accesses: head dim and strides multiples of 4, pointers of 16 bytes
bool vec4_ok(int64_t d, std::initializer_list<int64_t> strides,
             std::initializer_list<const void*> ptrs) {
  if (d % 4 != 0) return false;
  for (int64_t s : strides)
    if (s % 4 != 0) return false;
  for (const void* p : ptrs)
    if (!aligned(p, 16)) return false;
  return true;
}

}  // namespace

}  // namespace zk
