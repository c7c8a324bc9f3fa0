// RMS norm of every query and key head and the position rotation, in one pass.
//
// For a head's row x of d elements at position pos, with the weights w [d]:
//   r = 1 / sqrt(mean(x^2) + eps)      n = w x r       y = R(pos) n
// and backward, from dy:
//   dn = R(pos)^T dy    dw = sum over rows of dn x r
//   g = dn w            dx = r (g - x r mean(g x r))
// all in fp32 with one rounding of y, dx and dw.  The backward takes r from x
// again (x is read for dw and dx anyway), so nothing but the inputs is kept.
//
// A lane holds 8 pairs of a row (16 elements: two 16-byte accesses of 2-byte
// types), 2^log_g lanes a row, so a row's sums take log_g shuffles and a wave
// holds 64 >> log_g rows of one or more positions at a time.  A wave stays
// with its positions and goes through their heads: cos, sin and w are read
// once for all of them.  HBM bounds both directions: x and y, or x, dy and dx.
#include "part8.h"

namespace zk {

struct QkSide {  // the query or the key heads
  const void* x;
  const void* dy;  // backward
  void* out;       // y, or dx
  const void* w;
  int64_t x_sb, x_ss, x_sh, dy_sb, dy_ss, dy_sh, o_sb, o_ss, o_sh;
  int heads;
  int log_hpw;     // heads a wave holds at a time
  int splits;      // waves that share a position's heads
  int64_t wgs;     // workgroups of 4 waves
};

struct QkArgs {
  QkSide q, k;
  const float* cosT;
  const float* sinT;
  const int64_t* positions;
  int64_t pos_sb;  // positions' batch stride (0: shared)
  int64_t n_pos, S, rows;  // rows: B * S
  float* part;     // backward: [wgs of q, then of k][d]
  int d, w_dt;
  float eps;
};

// One lane's 8 pairs of a row: elements i and i + half of the half-split
// pairing, 2i and 2i + 1 of the interleaved one; n of them exist.
template <typename T, int kPairing>
struct Pairs {
  Part8<T> a, b;
  __device__ __forceinline__ void load(const T* row, int i0, int half, int n) {
    if (kPairing == ZK_ROPE_HALF) {
      a.load(row + i0, n);
      b.load(row + half + i0, n);
    } else {
      a.load(row + 2 * i0, 2 * n);
      b.load(row + 2 * i0 + 8, 2 * n - 8);
    }
  }
  // the pairs' first and second elements
  __device__ __forceinline__ float first(int i) const {
    return kPairing == ZK_ROPE_HALF ? a[i] : i < 4 ? a[2 * i] : b[2 * i - 8];
  }
  __device__ __forceinline__ float second(int i) const {
    return kPairing == ZK_ROPE_HALF ? b[i] : i < 4 ? a[2 * i + 1] : b[2 * i - 7];
  }
  static __device__ __forceinline__ void store(T* row, const float (&u)[8], const float (&v)[8],
                                               int i0, int half, int n) {
    if (kPairing == ZK_ROPE_HALF) {
      Part8<T>::store(row + i0, u, n);
      Part8<T>::store(row + half + i0, v, n);
    } else {
      const float lo[8] = {u[0], v[0], u[1], v[1], u[2], v[2], u[3], v[3]};
      const float hi[8] = {u[4], v[4], u[5], v[5], u[6], v[6], u[7], v[7]};
      Part8<T>::store(row + 2 * i0, lo, 2 * n);
      Part8<T>::store(row + 2 * i0 + 8, hi, 2 * n - 8);
    }
  }
};

template <int kPairing>
__device__ __forceinline__ int first_of(int i, int half) {
  return kPairing == ZK_ROPE_HALF ? i : 2 * i;
}
template <int kPairing>
__device__ __forceinline__ int second_of(int i, int half) {
  return kPairing == ZK_ROPE_HALF ? i + half : 2 * i + 1;
}

__device__ __forceinline__ float group_sum(float v, int lanes) {
  for (int off = lanes >> 1; off >= 1; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}

template <typename T, int kPairing, bool kBwd>
__global__ __launch_bounds__(256) void qk_kernel(QkArgs A, int log_g) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const bool is_q = blockIdx.x < A.q.wgs;
  const QkSide& X = is_q ? A.q : A.k;
  const int64_t wg = is_q ? blockIdx.x : blockIdx.x - A.q.wgs;
  const int half = A.d / 2, lanes = 1 << log_g;
  const int i0 = (lane & (lanes - 1)) * 8;
  const int n = half - i0 < 0 ? 0 : half - i0 < 8 ? half - i0 : 8;
  const int slot = lane >> log_g;                      // row slot of this lane
  const int log_ppw = 6 - log_g - X.log_hpw;           // positions a wave holds
  const int h0 = slot & ((1 << X.log_hpw) - 1), p_in = slot >> X.log_hpw;
  float wa[8], wb[8], da[8], db[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    wa[i] = i < n ? load_dt(X.w, first_of<kPairing>(i0 + i, half), A.w_dt) : 0.f;
    wb[i] = i < n ? load_dt(X.w, second_of<kPairing>(i0 + i, half), A.w_dt) : 0.f;
    da[i] = db[i] = 0.f;
  }
  const int64_t groups = (A.rows + (1 << log_ppw) - 1) >> log_ppw;
  const int64_t items = groups * X.splits;
  const float inv_d = 1.f / static_cast<float>(A.d);
  for (int64_t item = wg * 4 + wave; item < items; item += X.wgs * 4) {
    const int64_t group = X.splits == 1 ? item : item / X.splits;
    const int split = X.splits == 1 ? 0 : static_cast<int>(item - group * X.splits);
    const int64_t p = (group << log_ppw) + p_in;
    const bool in = p < A.rows && n > 0;
    const int64_t b = in ? p / A.S : 0, s = in ? p - b * A.S : 0;
    int64_t pos = s;
    if (A.positions != nullptr && in) pos = A.positions[b * A.pos_sb + s];
    const bool known = pos >= 0 && pos < A.n_pos;  // rows off the table are NaN
    Part8<float> cs, sn;
    cs.load(A.cosT + (known ? pos : 0) * half + i0, in ? n : 0);
    sn.load(A.sinT + (known ? pos : 0) * half + i0, in ? n : 0);
    float c[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = known ? cs[i] : __builtin_nanf("");
    const T* xr = static_cast<const T*>(X.x) + b * X.x_sb + s * X.x_ss;
    const T* gr = static_cast<const T*>(X.dy) + (kBwd ? b * X.dy_sb + s * X.dy_ss : 0);
    T* yr = static_cast<T*>(X.out) + b * X.o_sb + s * X.o_ss;
    for (int hb = split << X.log_hpw; hb < X.heads; hb += X.splits << X.log_hpw) {
      const int h = hb + h0;
      const bool on = in && h < X.heads;
      Pairs<T, kPairing> x, g;
      x.load(xr + h * X.x_sh, i0, half, on ? n : 0);
      if (kBwd) g.load(gr + h * X.dy_sh, i0, half, on ? n : 0);
      float ss = 0.f, t = 0.f, ga[8], gb[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float u = x.first(i), v = x.second(i);
        ss = fmaf(u, u, fmaf(v, v, ss));
        if (kBwd) {  // dn = R^T dy
          const float e = g.first(i), f = g.second(i);
          ga[i] = fmaf(e, c[i], f * sn[i]);
          gb[i] = fmaf(f, c[i], -(e * sn[i]));
          t = fmaf(ga[i] * wa[i], u, fmaf(gb[i] * wb[i], v, t));
        }
      }
      ss = group_sum(ss, lanes);
      const float r = 1.f / sqrtf(ss * inv_d + A.eps);
      float oa[8], ob[8];
      if (!kBwd) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float u = x.first(i) * r * wa[i], v = x.second(i) * r * wb[i];
          oa[i] = fmaf(u, c[i], -(v * sn[i]));
          ob[i] = fmaf(v, c[i], u * sn[i]);
        }
      } else {
        t = group_sum(t, lanes) * r * r * inv_d;  // r mean(g x r)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float u = x.first(i), v = x.second(i);
          if (on) {
            da[i] = fmaf(ga[i], u * r, da[i]);
            db[i] = fmaf(gb[i], v * r, db[i]);
          }
          oa[i] = r * fmaf(-t, u, ga[i] * wa[i]);
          ob[i] = r * fmaf(-t, v, gb[i] * wb[i]);
        }
      }
      if (on) Pairs<T, kPairing>::store(yr + h * X.o_sh, oa, ob, i0, half, n);
    }
  }
  if (!kBwd) return;
  // dw: this workgroup's row of partial sums
  __shared__ float sums[4][1024];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    for (int off = lanes; off < 64; off <<= 1) {
      da[i] += __shfl_xor(da[i], off, 64);
      db[i] += __shfl_xor(db[i], off, 64);
    }
    if (slot == 0 && i < n) {
      sums[wave][first_of<kPairing>(i0 + i, half)] = da[i];
      sums[wave][second_of<kPairing>(i0 + i, half)] = db[i];
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < A.d; i += 256)
    A.part[static_cast<int64_t>(blockIdx.x) * A.d + i] =
        (sums[0][i] + sums[1][i]) + (sums[2][i] + sums[3][i]);
}

// dw [d] from the partial rows: 64 columns a workgroup, 16 waves a share of
// the rows each, in order.
__global__ __launch_bounds__(1024) void qk_dw(const float* __restrict__ part, int64_t q_rows,
                                              int64_t k_rows, int d, void* dwq, void* dwk,
                                              int w_dt) {
  __shared__ float sums[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int col = blockIdx.x * 64 + lane;
  const int64_t first = blockIdx.y == 0 ? 0 : q_rows;
  const int64_t rows = blockIdx.y == 0 ? q_rows : k_rows;
  const int64_t a = rows * wave / 16, b = rows * (wave + 1) / 16;
  float v = 0.f;
  if (col < d) {
#pragma unroll 8
    for (int64_t i = a; i < b; ++i) v += part[(first + i) * d + col];
  }
  sums[wave][lane] = v;
  __syncthreads();
  if (wave != 0 || col >= d) return;
#pragma unroll
  for (int i = 1; i < 16; ++i) v += sums[i][lane];
  store_dt(blockIdx.y == 0 ? dwq : dwk, col, w_dt, v);
}

static int log_lanes(int64_t d) {
  int lg = 0;
  while ((int64_t(16) << lg) < d) ++lg;
  return lg;
}

static constexpr int64_t kMaxWgs = int64_t(1) << 22;  // below 2^32 threads a launch
static constexpr int64_t kBwdWgs = 1024;              // partial rows of dw for each side

static void plan(QkSide& s, int64_t rows, int64_t heads, int log_g, bool bwd) {
  s.heads = static_cast<int>(heads);
  s.log_hpw = 0;
  while (s.log_hpw < 6 - log_g && (int64_t(1) << s.log_hpw) < heads) ++s.log_hpw;
  const int log_ppw = 6 - log_g - s.log_hpw;
  const int64_t groups = (rows + (int64_t(1) << log_ppw) - 1) >> log_ppw;
  const int64_t passes = (heads + (int64_t(1) << s.log_hpw) - 1) >> s.log_hpw;
  // few positions: a wave for every pass over the heads
  s.splits = groups < 2048 ? static_cast<int>(passes) : 1;
  const int64_t wgs = (groups * s.splits + 3) / 4, cap = bwd ? kBwdWgs : kMaxWgs;
  s.wgs = heads == 0 ? 0 : wgs < cap ? wgs : cap;
}

template <bool kBwd>
static void launch_qk(const QkArgs& A, int dtype, int pairing, int log_g, hipStream_t st) {
  const dim3 grid(static_cast<unsigned>(A.q.wgs + A.k.wgs));
#define ZK_QK(T, P) hipLaunchKernelGGL((qk_kernel<T, P, kBwd>), grid, dim3(256), 0, st, A, log_g)
#define ZK_QKP(T)                                  \
  do {                                             \
    if (pairing == ZK_ROPE_HALF) ZK_QK(T, ZK_ROPE_HALF); \
    else ZK_QK(T, ZK_ROPE_INTERLEAVED);            \
  } while (0)
  if (dtype == ZK_F32) ZK_QKP(float);
  else if (dtype == ZK_BF16) ZK_QKP(bf16);
  else ZK_QKP(f16);
#undef ZK_QKP
#undef ZK_QK
}

// The checks that both directions share, and the arguments' common part.
static int qk_args(const char* who, const zk_qk_desc* D, const void* q, const void* k,
                   const void* wq, const void* wk, const float* cos, const float* sin,
                   const int64_t* positions, bool bwd, QkArgs& A) {
  ZK_REQUIRE(D != nullptr, ZK_EINVAL, "%s: null descriptor", who);
  ZK_REQUIRE(valid_dtype(D->dtype) && valid_dtype(D->w_dtype), ZK_EDTYPE, "%s: bad dtype (%d, %d)",
             who, D->dtype, D->w_dtype);
  ZK_REQUIRE(D->pairing == ZK_ROPE_HALF || D->pairing == ZK_ROPE_INTERLEAVED, ZK_EINVAL,
             "%s: bad pairing %d", who, D->pairing);
  ZK_REQUIRE(D->B >= 0 && D->S >= 0 && D->Hq > 0 && D->Hkv >= 0 && D->d > 0 && D->d % 2 == 0,
             ZK_EINVAL, "%s: bad shape (d must be even, got %lld)", who, (long long)D->d);
  ZK_REQUIRE(D->d <= 1024, ZK_EUNSUPPORTED, "%s: head dims up to 1024 (got %lld)", who,
             (long long)D->d);
  ZK_REQUIRE(D->Hq < (1 << 24) && D->Hkv < (1 << 24) && D->B < (int64_t(1) << 31) &&
                 D->S < (int64_t(1) << 31),
             ZK_EINVAL, "%s: too many heads or positions", who);
  ZK_REQUIRE(D->eps >= 0, ZK_EINVAL, "%s: negative eps", who);
  const bool none = D->B == 0 || D->S == 0;  // empty tensors have no address
  ZK_REQUIRE((q || none) && wq && cos && sin && (D->Hkv == 0 || ((k || none) && wk)), ZK_EINVAL,
             "%s: null pointer", who);
  ZK_REQUIRE(D->n_pos > 0 && (positions != nullptr || D->n_pos >= D->S), ZK_EINVAL,
             "%s: table has %lld positions for S=%lld", who, (long long)D->n_pos, (long long)D->S);
  const int e = dtype_bytes(D->dtype), we = dtype_bytes(D->w_dtype);
  ZK_REQUIRE(aligned(q, e) && aligned(k, e) && aligned(wq, we) && aligned(wk, we) &&
                 aligned(cos, 4) && aligned(sin, 4) && aligned(positions, 8),
             ZK_EALIGN, "%s: tensors must be aligned to their element size", who);
  A = QkArgs{};
  A.q.x = q; A.q.w = wq;
  A.q.x_sb = D->q_sb; A.q.x_ss = D->q_ss; A.q.x_sh = D->q_sh;
  A.q.dy_sb = D->dyq_sb; A.q.dy_ss = D->dyq_ss; A.q.dy_sh = D->dyq_sh;
  A.q.o_sb = D->oq_sb; A.q.o_ss = D->oq_ss; A.q.o_sh = D->oq_sh;
  A.k.x = k; A.k.w = wk;
  A.k.x_sb = D->k_sb; A.k.x_ss = D->k_ss; A.k.x_sh = D->k_sh;
  A.k.dy_sb = D->dyk_sb; A.k.dy_ss = D->dyk_ss; A.k.dy_sh = D->dyk_sh;
  A.k.o_sb = D->ok_sb; A.k.o_ss = D->ok_ss; A.k.o_sh = D->ok_sh;
  A.cosT = cos; A.sinT = sin; A.positions = positions; A.pos_sb = D->pos_sb;
  A.n_pos = D->n_pos; A.S = D->S; A.rows = D->B * D->S;
  A.d = static_cast<int>(D->d); A.w_dt = D->w_dtype; A.eps = D->eps;
  const int lg = log_lanes(D->d);
  plan(A.q, A.rows, D->Hq, lg, bwd);
  plan(A.k, A.rows, D->Hkv, lg, bwd);
  return ZK_OK;
}

}  // namespace zk

using namespace zk;

extern "C" int zk_qk_norm_rope_fwd(const zk_qk_desc* desc, const void* q, const void* k,
                                   const void* wq, const void* wk, void* q_out, void* k_out,
                                   const float* cos, const float* sin, const int64_t* positions,
                                   zk_stream_t stream) {
  QkArgs A;
  const int rc = qk_args("zk_qk_norm_rope_fwd", desc, q, k, wq, wk, cos, sin, positions, false, A);
  if (rc != ZK_OK) return rc;
  if (A.rows == 0) return ZK_OK;
  ZK_REQUIRE(q_out && (desc->Hkv == 0 || k_out), ZK_EINVAL, "zk_qk_norm_rope_fwd: null output");
  ZK_REQUIRE(aligned(q_out, dtype_bytes(desc->dtype)) && aligned(k_out, dtype_bytes(desc->dtype)),
             ZK_EALIGN, "zk_qk_norm_rope_fwd: tensors must be aligned to their element size");
  A.q.out = q_out;
  A.k.out = k_out;
  launch_qk<false>(A, desc->dtype, desc->pairing, log_lanes(desc->d), as_stream(stream));
  return launch_status("zk_qk_norm_rope_fwd");
}

extern "C" int64_t zk_qk_norm_rope_bwd_workspace(int64_t d) {
  return d > 0 && d <= 1024 ? 2 * kBwdWgs * d * 4 : -1;
}

extern "C" int zk_qk_norm_rope_bwd(const zk_qk_desc* desc, const void* q, const void* k,
                                   const void* wq, const void* wk, const void* dq_out,
                                   const void* dk_out, void* dq, void* dk, void* dwq, void* dwk,
                                   const float* cos, const float* sin, const int64_t* positions,
                                   void* workspace, int64_t workspace_bytes, zk_stream_t stream) {
  QkArgs A;
  const int rc = qk_args("zk_qk_norm_rope_bwd", desc, q, k, wq, wk, cos, sin, positions, true, A);
  if (rc != ZK_OK) return rc;
  const bool none = A.rows == 0;
  ZK_REQUIRE((none || (dq_out && dq)) && dwq && workspace &&
                 (desc->Hkv == 0 || ((none || (dk_out && dk)) && dwk)),
             ZK_EINVAL, "zk_qk_norm_rope_bwd: null pointer");
  const int e = dtype_bytes(desc->dtype), we = dtype_bytes(desc->w_dtype);
  ZK_REQUIRE(aligned(dq_out, e) && aligned(dk_out, e) && aligned(dq, e) && aligned(dk, e) &&
                 aligned(dwq, we) && aligned(dwk, we) && aligned(workspace, 4),
             ZK_EALIGN, "zk_qk_norm_rope_bwd: tensors must be aligned to their element size");
  ZK_REQUIRE(workspace_bytes >= zk_qk_norm_rope_bwd_workspace(desc->d), ZK_EWORKSPACE,
             "zk_qk_norm_rope_bwd: workspace of %lld bytes, %lld needed", (long long)workspace_bytes,
             (long long)zk_qk_norm_rope_bwd_workspace(desc->d));
  A.q.dy = dq_out; A.q.out = dq;
  A.k.dy = dk_out; A.k.out = dk;
  A.part = static_cast<float*>(workspace);
  hipStream_t st = as_stream(stream);
  if (A.rows > 0) launch_qk<true>(A, desc->dtype, desc->pairing, log_lanes(desc->d), st);
  // without rows there are no partial rows: dw is zero
  hipLaunchKernelGGL(qk_dw, dim3(static_cast<unsigned>((A.d + 63) / 64), desc->Hkv > 0 ? 2 : 1),
                     dim3(1024), 0, st, A.part, A.q.wgs, A.k.wgs, A.d, dwq, dwk, A.w_dt);
  return launch_status("zk_qk_norm_rope_bwd");
}
