// Orthogonal factors of matrices by Newton-Schulz products, and the step that
// takes them (momentum, factor, weights), over lists of matrices.
//
// With s <= t the sides of a matrix U, X0 = U / (|U| + eps) as [s, t] (tall ones
// transposed), each of the steps makes
//   G = X X^T,   P = b G + c G G,   X <- a X + P X,
// a polynomial a z + b z^3 + c z^5 of every singular value.  G and P are
// symmetric: their tiles on and below the diagonal are computed, and stored
// twice.  s^2 t + s^3 + 2 s^2 t multiply-adds' operations a step, on the fp16
// matrix cores.
//
// Numbers.  The products' operands are fp16, with sums in fp32: singular values
// lie below 1.3, so scaled by powers of two that the host takes from the
// polynomial's bounds (X by Sx, G by S^2, P by R) they use fp16's whole
// range, and its step is an eighth of bf16's at the same rate.  X itself is held
// in two fp16 numbers (22 bits), and a X is added in fp32: small singular values
// grow by a = 3.4 a step, and a rounding of X relative to the largest ones would
// grow with them (a matrix of 8 strong directions over noise a hundredth as
// large: 3.6e-2 off with X in one fp16 number, 0.3 in bf16, 3e-4 like this; other
// spectra 0.3 - 1.7e-3).  The second number has its bits only where the first is
// above 2^-3 (below that it is subnormal): X's elements, about 1 / sqrt(t), need
// the largest scale there is, 2^15 for singular values up to 1.23 (2048 x 2048 of
// that spectrum in two numbers throughout: 4.0e-5 off with Sx = 2^7, S's, and
// 7e-6 with 2^15).  Matrices with s <= kExactSide, whose products cost no
// time, and results in fp32 have G and P in two numbers as well, and products of
// three terms.
//
// What bounds it.  Large lists: the products, at 1.11 - 1.13 PF/s (four matrices of
// 4096 x 4096 and three of 4096 x 11008: 13.2 of 14.7 ms; 3 passes over momenta and
// weights 1.5, 4.4 TB/s).  Small ones: launches of 6 us, two and one for the passes
// and three for each step (four of 256 x 256: 111 us), which all matrices of a list
// share for that reason.
#include <algorithm>
#include <cmath>

#include "muon.h"

namespace zk {

namespace {

constexpr int kPartials = 256;       // partial sums of squares of a matrix
constexpr int64_t kExactSide = 128;  // matrices up to here are computed with 22 bits throughout
constexpr int kTile = 64;

// One matrix of a launch of the element-wise kernels.
struct Matrix {
  const void* grad;
  float* momentum;   // step: else NULL
  float* param;
  void* out;         // factors, or the step's rounded copy
  f16* hi;           // X, [sp, tp]
  f16* lo;
  double* partial;   // [kPartials]
  int64_t rows, cols, ld_grad, ld_momentum, ld_param, ld_out;
  int64_t sp, tp;    // padded sides
  float lr_scale;
  int grad_dtype, out_dtype, tall;
  int vec;           // columns, rows and addresses are multiples of four elements
};
struct MatrixGroup {
  Matrix p[gemm::kPolyMost];
  int first[gemm::kPolyMost + 1];
  int n;
  float mu, nu, keep, lr, scale, eps;  // nu = 1 - mu, keep = 1 - lr weight_decay; scale: Sx
  int nesterov;
};

__device__ __forceinline__ const Matrix& matrix_of(const MatrixGroup& g, int64_t& at) {
  int i = 0;
  while (i + 1 < g.n && at >= g.first[i + 1]) ++i;
  at -= g.first[i];
  return g.p[i];
}

// What is orthogonalised, from the gradient and the momentum after this step's.
__device__ __forceinline__ float update_of(const MatrixGroup& g, float grad, float m) {
  return g.nesterov ? fmaf(g.mu, m, g.nu * grad) : m;
}

// Four elements of a row from column c on (those below `cols`, else zeros); vec:
// rows and columns are multiples of four elements and aligned.
__device__ __forceinline__ float4 load4(const void* p, int64_t at, int dt, bool vec, int64_t left) {
  if (vec) {
    if (dt == ZK_F32) return *reinterpret_cast<const float4*>(static_cast<const float*>(p) + at);
    const u32x2 w = *reinterpret_cast<const u32x2*>(static_cast<const uint16_t*>(p) + at);
    if (dt == ZK_BF16) {
      const bf16x4 v = __builtin_bit_cast(bf16x4, w);
      return make_float4(v[0], v[1], v[2], v[3]);
    }
    const f16x4 v = __builtin_bit_cast(f16x4, w);
    return make_float4(v[0], v[1], v[2], v[3]);
  }
  float v[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = e < left ? load_dt(p, at + e, dt) : 0.f;
  return make_float4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ void store4(void* p, int64_t at, int dt, bool vec, int64_t left, float4 x) {
  const float v[4] = {x.x, x.y, x.z, x.w};
  if (vec) {
    if (dt == ZK_F32) {
      *reinterpret_cast<float4*>(static_cast<float*>(p) + at) = x;
    } else if (dt == ZK_BF16) {
      *reinterpret_cast<bf16x4*>(static_cast<bf16*>(p) + at) =
          bf16x4{static_cast<bf16>(v[0]), static_cast<bf16>(v[1]), static_cast<bf16>(v[2]), static_cast<bf16>(v[3])};
    } else {
      *reinterpret_cast<f16x4*>(static_cast<f16*>(p) + at) =
          f16x4{static_cast<f16>(v[0]), static_cast<f16>(v[1]), static_cast<f16>(v[2]), static_cast<f16>(v[3])};
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (e < left) store_dt(p, at + e, dt, v[e]);
}
__device__ __forceinline__ float4 update4(const MatrixGroup& g, const float4& v, const float4& m) {
  return make_float4(update_of(g, v.x, m.x), update_of(g, v.y, m.y), update_of(g, v.z, m.z),
                     update_of(g, v.w, m.w));
}

// The momentum's step, and kPartials sums of squares (64 bits: squares of small
// gradients leave fp32's range): runs of 4096 columns of a row, workgroup w of
// the matrix taking runs w, w + kPartials, ..; a run's loads are issued together.
__global__ __launch_bounds__(256) void muon_begin_kernel(MatrixGroup g) {
  int64_t w = blockIdx.x;
  const Matrix& x = matrix_of(g, w);
  const int64_t per_row = (x.cols + 4095) / 4096, runs = x.rows * per_row;
  const bool step = x.momentum != nullptr;
  double sum = 0;
  for (int64_t u = w; u < runs; u += kPartials) {
    const int64_t row = u / per_row, c0 = (u - row * per_row) * 4096 + 4 * threadIdx.x;
    float4 v[4], m[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int64_t c = c0 + k * 1024;
      v[k] = m[k] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (c >= x.cols) continue;
      v[k] = load4(x.grad, row * x.ld_grad + c, x.grad_dtype, x.vec, x.cols - c);
      if (step) m[k] = load4(x.momentum, row * x.ld_momentum + c, ZK_F32, x.vec, x.cols - c);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int64_t c = c0 + k * 1024;
      if (c >= x.cols) continue;
      float4 t = v[k];
      if (step) {
        const float h = g.nu;
        const float4 n = make_float4(fmaf(g.mu, m[k].x, h * t.x), fmaf(g.mu, m[k].y, h * t.y),
                                     fmaf(g.mu, m[k].z, h * t.z), fmaf(g.mu, m[k].w, h * t.w));
        store4(x.momentum, row * x.ld_momentum + c, ZK_F32, x.vec, x.cols - c, n);
        t = update4(g, t, n);
      }
      sum += static_cast<double>(t.x) * t.x + static_cast<double>(t.y) * t.y +
             (static_cast<double>(t.z) * t.z + static_cast<double>(t.w) * t.w);
    }
  }
  __shared__ double part[256];
  part[threadIdx.x] = sum;
  __syncthreads();
  for (int n = 128; n > 0; n /= 2) {
    if (static_cast<int>(threadIdx.x) < n) part[threadIdx.x] += part[threadIdx.x + n];
    __syncthreads();
  }
  if (threadIdx.x == 0) x.partial[w] = part[0];
}

// X0, padded with zeros: 64 x 64 tiles of X, through LDS where U is tall.
__global__ __launch_bounds__(256) void muon_scale_kernel(MatrixGroup g) {
  int64_t at = blockIdx.x;
  const Matrix& x = matrix_of(g, at);
  __shared__ double total;
  __shared__ float tile[kTile][kTile + 1];
  if (threadIdx.x < 64) {
    double v = 0;
    for (int i = threadIdx.x; i < kPartials; i += 64) v += x.partial[i];
    for (int n = 32; n > 0; n /= 2) v += __shfl_xor(v, n, 64);
    if (threadIdx.x == 0) total = v;
  }
  const int64_t per_row = x.tp / kTile;
  const int64_t s0 = at / per_row * kTile, t0 = at % per_row * kTile;
  // U's rows and columns of this tile
  const int64_t r0 = x.tall ? t0 : s0, c0 = x.tall ? s0 : t0;
  const int col = threadIdx.x % 16 * 4, row0 = threadIdx.x / 16;
  float4 v[4], m[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int64_t r = r0 + row0 + 16 * k, c = c0 + col;
    v[k] = m[k] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (r >= x.rows || c >= x.cols) continue;
    v[k] = load4(x.grad, r * x.ld_grad + c, x.grad_dtype, x.vec, x.cols - c);
    if (x.momentum != nullptr) m[k] = load4(x.momentum, r * x.ld_momentum + c, ZK_F32, x.vec, x.cols - c);
  }
  if (x.momentum != nullptr) {
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = update4(g, v[k], m[k]);
  }
  if (x.tall) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float* row = &tile[row0 + 16 * k][col];
      row[0] = v[k].x; row[1] = v[k].y; row[2] = v[k].z; row[3] = v[k].w;
    }
  }
  __syncthreads();
  // in 64 bits: Sx / |u| may leave fp32's range where u Sx / |u| does not
  const double f = g.scale / (sqrt(total) + static_cast<double>(g.eps));
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int r = row0 + 16 * k;
    if (x.tall) v[k] = make_float4(tile[col][r], tile[col + 1][r], tile[col + 2][r], tile[col + 3][r]);
    float y[4] = {static_cast<float>(v[k].x * f), static_cast<float>(v[k].y * f),
                  static_cast<float>(v[k].z * f), static_cast<float>(v[k].w * f)};
    f16x4 hi, lo;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      asm("" : "+v"(y[e]));  // see poly_store
      hi[e] = static_cast<f16>(y[e]);
      lo[e] = static_cast<f16>(y[e] - static_cast<float>(hi[e]));
    }
    const int64_t i = (s0 + r) * x.tp + t0 + col;
    *reinterpret_cast<f16x4*>(x.hi + i) = hi;
    *reinterpret_cast<f16x4*>(x.lo + i) = lo;
  }
}

// The factor to its place, or the weights' step with it: 64 x 64 tiles of U.
__global__ __launch_bounds__(256) void muon_finish_kernel(MatrixGroup g) {
  int64_t at = blockIdx.x;
  const Matrix& x = matrix_of(g, at);
  __shared__ float tile[kTile][kTile + 1];
  const int64_t per_row = x.tp / kTile;
  const int64_t s0 = at / per_row * kTile, t0 = at % per_row * kTile;
  const int64_t r0 = x.tall ? t0 : s0, c0 = x.tall ? s0 : t0;
  const int col = threadIdx.x % 16 * 4, row0 = threadIdx.x / 16;
  f16x4 hi[4], lo[4];
  float4 p[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int64_t i = (s0 + row0 + 16 * k) * x.tp + t0 + col;
    hi[k] = *reinterpret_cast<const f16x4*>(x.hi + i);
    lo[k] = *reinterpret_cast<const f16x4*>(x.lo + i);
    const int64_t r = r0 + row0 + 16 * k, c = c0 + col;
    p[k] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (x.param != nullptr && r < x.rows && c < x.cols)
      p[k] = load4(x.param, r * x.ld_param + c, ZK_F32, x.vec, x.cols - c);
  }
  float4 v[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    float y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e)
      y[e] = (static_cast<float>(hi[k][e]) + static_cast<float>(lo[k][e])) / g.scale;
    v[k] = make_float4(y[0], y[1], y[2], y[3]);
    if (x.tall) {
      float* row = &tile[row0 + 16 * k][col];
      row[0] = y[0]; row[1] = y[1]; row[2] = y[2]; row[3] = y[3];
    }
  }
  __syncthreads();
  const float f = -g.lr * x.lr_scale, keep = g.keep;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int rr = row0 + 16 * k;
    const int64_t r = r0 + rr, c = c0 + col;
    if (r >= x.rows || c >= x.cols) continue;
    if (x.tall) v[k] = make_float4(tile[col][rr], tile[col + 1][rr], tile[col + 2][rr], tile[col + 3][rr]);
    if (x.param != nullptr) {
      v[k] = make_float4(fmaf(f, v[k].x, p[k].x * keep), fmaf(f, v[k].y, p[k].y * keep),
                         fmaf(f, v[k].z, p[k].z * keep), fmaf(f, v[k].w, p[k].w * keep));
      store4(x.param, r * x.ld_param + c, ZK_F32, x.vec, x.cols - c, v[k]);
    }
    if (x.out != nullptr) store4(x.out, r * x.ld_out + c, x.out_dtype, x.vec, x.cols - c, v[k]);
  }
}

// ---------------------------------------------------------------------- host --
struct Sides {
  int64_t s, t, sp, tp;
  bool exact;
};
int64_t up(int64_t n, int64_t m) { return (n + m - 1) / m * m; }

// Tiles of one product of a run of matrices (`square`: of its two symmetric ones,
// whose tiles above the diagonal alone are computed).
//  * 256 x 256 where the 128 x 128 tiles would not fit on the CUs at once, two to
//    each: 2048 x 5632 772 us a matrix against 818, but two of 2048 x 2048 684
//    against 639, whose X has 512 of the smaller tiles.  Not where sides far from
//    multiples of 256 make padding of a twentieth of it (five odd matrices of 546 to
//    2748 485 us against 416).
//  * else 128 x 128 where that ends sooner than 64 x 64.  Steps along K: a tile of
//    128 rows takes one step's time alone on its CU, one of 64 half a step's when
//    several share a CU.  So few tiles, or some with a far longer K than the others',
//    are cut small: 1024 x 4096 293 us against 427, two 414 against 496; but one of
//    2048 x 2048 459 against 496, four of 512 x 2048 217 against 232 (X).
gemm::Tile tile_of(const Sides* x, int n, bool square) {
  if (x[0].exact) return gemm::k64;
  int64_t tiles256 = 0, tiles128 = 0, steps128 = 0, steps64 = 0, longest = 0;
  for (int i = 0; i < n; ++i) {
    const auto count = [&](gemm::Tile t) {
      const int64_t rows = (x[i].s + gemm::tile_rows(t) - 1) / gemm::tile_rows(t);
      return square ? rows * (rows + 1) / 2 : gemm::tile_count(t, x[i].s, x[i].t);
    };
    const int64_t k = square ? x[i].t : x[i].s;
    tiles256 += count(gemm::k256);
    tiles128 += count(gemm::k128);
    steps128 += count(gemm::k128) * k;
    steps64 += count(gemm::k64) * k;
    longest = std::max(longest, k);
  }
  const int64_t cus = device_cus();
  if (tiles128 > 2 * cus && 80 * tiles256 <= 21 * tiles128) return gemm::k256;
  return std::max(longest * cus, steps128) < steps64 / 2 ? gemm::k128 : gemm::k64;
}

Sides sides_of(const zk_muon_matrix& x) {
  Sides d;
  d.s = x.rows < x.cols ? x.rows : x.cols;
  d.t = x.rows < x.cols ? x.cols : x.rows;
  d.exact = d.s <= kExactSide || (x.param == nullptr && x.out_dtype == ZK_F32);
  d.sp = d.tp = 0;
  return d;
}

// A run of matrices that share launches: of one precision, at most kPolyMost.
int run_length(const zk_muon_matrix* list, int64_t n) {
  int len = 0;
  while (len < n && len < gemm::kPolyMost && sides_of(list[len]).exact == sides_of(list[0]).exact) ++len;
  return len;
}

int64_t bytes_of(const Sides& d) {
  const int64_t square = d.sp * d.sp * 2, x = d.sp * d.tp * 2;
  return up(4 * x + (d.exact ? 4 : 2) * square + kPartials * 8, 256);
}

void plan_run(const zk_muon_matrix* list, int n, Sides* d) {
  for (int i = 0; i < n; ++i) d[i] = sides_of(list[i]);
  const bool wide = tile_of(d, n, true) == gemm::k256 || tile_of(d, n, false) == gemm::k256;
  for (int i = 0; i < n; ++i) {
    d[i].sp = up(d[i].s, wide ? 256 : 64);
    d[i].tp = up(d[i].t, wide ? 256 : 64);
  }
}

// Bounds of the polynomial's iterates on [0, 1]: the powers of two that Sx X, S^2 G
// and R P stay in fp16's range with.  False: the iterates leave it.
bool scales_of(int steps, double a, double b, double c, float* Sx, float* S, float* R) {
  if (!(std::isfinite(a) && std::isfinite(b) && std::isfinite(c))) return false;
  double most = 1.0, most_p = 0, most_l = 1.0;
  // where a z + b z^3 + c z^5 and b l + c l^2, l = z^2, may be largest: at the range's end
  // and where their derivatives are zero
  double roots[3] = {c != 0 ? -b / (2 * c) : -1};
  if (c != 0) {
    const double half = 0.3 * b / c, q = half * half - 0.2 * a / c;
    if (q >= 0) roots[1] = -half + sqrt(q), roots[2] = -half - sqrt(q);
  } else if (b != 0) {
    roots[1] = -a / (3 * b);
  }
  for (int k = 0; k < steps; ++k) {
    double next = 0;
    const auto at = [&](double l) {
      if (!(l > 0 && l <= most * most)) return;
      const double p = b * l + c * l * l;
      next = fmax(next, fabs(sqrt(l) * (a + p)));
      most_p = fmax(most_p, fabs(p));
    };
    at(most * most);
    for (const double l : roots) at(l);
    if (!(next < 16.0)) return false;
    most = next * 1.02;  // roundings
    most_l = fmax(most_l, most * most);
  }
  // Sx = 2^h, Sx^2 most_l < 2^31; S = 2^i, S^2 most_l < 2^15.5; R = 2^j
  *Sx = static_cast<float>(exp2(floor(log2(46000.0 / sqrt(most_l)))));
  *S = static_cast<float>(exp2(floor(0.5 * log2(46000.0 / most_l))));
  *R = most_p > 0 ? static_cast<float>(exp2(fmin(13.0, floor(log2(46000.0 / most_p))))) : 1.f;
  return true;
}

int check_list(const char* who, const zk_muon_matrix* list, int64_t n, bool step) {
  ZK_REQUIRE(n >= 0 && (n == 0 || list != nullptr), ZK_EINVAL, "%s: no list", who);
  for (int64_t i = 0; i < n; ++i) {
    const zk_muon_matrix& x = list[i];
    ZK_REQUIRE(x.rows > 0 && x.cols > 0 && x.rows < (int64_t(1) << 20) && x.cols < (int64_t(1) << 20),
               ZK_EINVAL, "%s: matrix %lld is %lld x %lld (1 .. 2^20 - 1)", who, (long long)i,
               (long long)x.rows, (long long)x.cols);
    ZK_REQUIRE(x.rows * x.cols <= int64_t(1) << 32, ZK_EINVAL, "%s: matrix %lld has more than 2^32 elements",
               who, (long long)i);
    ZK_REQUIRE(valid_dtype(static_cast<int>(x.grad_dtype)) && (x.out == nullptr || valid_dtype(static_cast<int>(x.out_dtype))), ZK_EDTYPE,
               "%s: matrix %lld has a bad dtype", who, (long long)i);
    ZK_REQUIRE(x.grad != nullptr && (step ? x.param != nullptr && x.momentum != nullptr
                                          : x.out != nullptr && x.param == nullptr && x.momentum == nullptr),
               ZK_EINVAL, "%s: matrix %lld lacks a pointer, or has one too many", who, (long long)i);
    ZK_REQUIRE(x.ld_grad >= x.cols && (!step || (x.ld_param >= x.cols && x.ld_momentum >= x.cols)) &&
                   (x.out == nullptr || x.ld_out >= x.cols),
               ZK_EINVAL, "%s: rows of matrix %lld overlap", who, (long long)i);
    ZK_REQUIRE(aligned(x.grad, dtype_bytes(static_cast<int>(x.grad_dtype))) && aligned(x.param, 4) && aligned(x.momentum, 4) &&
                   (x.out == nullptr || aligned(x.out, dtype_bytes(static_cast<int>(x.out_dtype)))),
               ZK_EALIGN, "%s: matrix %lld is not aligned to its elements", who, (long long)i);
  }
  return ZK_OK;
}

struct Hyper {
  int steps;
  double a, b, c, eps, lr, mu, decay;
  int nesterov, adjust;
};

int run_list(const char* who, const zk_muon_matrix* list, int64_t n, bool step, const Hyper& h,
             void* workspace, int64_t workspace_bytes, hipStream_t s) {
  const int rc = check_list(who, list, n, step);
  if (rc != ZK_OK) return rc;
  ZK_REQUIRE(h.steps >= 1 && h.steps <= 100, ZK_EINVAL, "%s: %d steps (1 .. 100)", who, h.steps);
  ZK_REQUIRE(h.eps >= 0, ZK_EINVAL, "%s: eps must not be negative", who);
  float Sx, S, R;
  ZK_REQUIRE(scales_of(h.steps, h.a, h.b, h.c, &Sx, &S, &R), ZK_EINVAL,
             "%s: the polynomial (%g, %g, %g) grows beyond 16 within %d steps", who, h.a, h.b, h.c, h.steps);
  if (n == 0) return ZK_OK;
  const int64_t need = zk_muon_workspace(list, n);
  ZK_REQUIRE((workspace != nullptr && workspace_bytes >= need), ZK_EWORKSPACE,
             "%s: workspace %lld < %lld bytes", who, (long long)workspace_bytes, (long long)need);
  for (int64_t at = 0; at < n;) {
    Sides d[gemm::kPolyMost];
    const int len = run_length(list + at, n - at);
    plan_run(list + at, len, d);
    const gemm::Tile tile_square = tile_of(d, len, true), tile_x = tile_of(d, len, false);
    char* ws = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(workspace) + 255) & ~uintptr_t(255));
    MatrixGroup m = {};
    f16 *hi[2][gemm::kPolyMost], *lo[2][gemm::kPolyMost], *G[2][gemm::kPolyMost], *P[2][gemm::kPolyMost];
    m.n = len;
    m.mu = static_cast<float>(h.mu); m.nu = static_cast<float>(1 - h.mu);
    m.keep = static_cast<float>(1 - h.lr * h.decay);
    m.lr = static_cast<float>(h.lr); m.scale = Sx; m.eps = static_cast<float>(h.eps);
    m.nesterov = h.nesterov;
    for (int i = 0; i < len; ++i) {
      const zk_muon_matrix& x = list[at + i];
      const int64_t big = d[i].sp * d[i].tp, square = d[i].sp * d[i].sp;
      f16* p = reinterpret_cast<f16*>(ws);
      for (int k = 0; k < 2; ++k) {
        hi[k][i] = p; p += big;
        lo[k][i] = p; p += big;
      }
      for (int k = 0; k < (d[i].exact ? 2 : 1); ++k) {
        G[k][i] = p; p += square;
        P[k][i] = p; p += square;
      }
      if (!d[i].exact) G[1][i] = P[1][i] = nullptr;
      Matrix& y = m.p[i];
      y.partial = reinterpret_cast<double*>(p);
      ws += bytes_of(d[i]);
      y.grad = x.grad; y.momentum = x.momentum; y.param = x.param; y.out = x.out;
      y.hi = hi[0][i]; y.lo = lo[0][i];
      y.rows = x.rows; y.cols = x.cols;
      y.ld_grad = x.ld_grad; y.ld_momentum = x.ld_momentum; y.ld_param = x.ld_param; y.ld_out = x.ld_out;
      y.sp = d[i].sp; y.tp = d[i].tp;
      y.grad_dtype = static_cast<int>(x.grad_dtype); y.out_dtype = static_cast<int>(x.out_dtype);
      y.tall = x.rows > x.cols;
      y.vec = x.cols % 4 == 0 && x.ld_grad % 4 == 0 && aligned(x.grad, 4 * dtype_bytes(y.grad_dtype)) &&
              (!step || (x.ld_momentum % 4 == 0 && x.ld_param % 4 == 0 && aligned(x.momentum, 16) &&
                         aligned(x.param, 16))) &&
              (x.out == nullptr || (x.ld_out % 4 == 0 && aligned(x.out, 4 * dtype_bytes(y.out_dtype))));
      y.lr_scale = static_cast<float>(
          h.adjust == ZK_MUON_MATCH_RMS ? 0.2 * sqrt(static_cast<double>(d[i].t))
                                        : sqrt(fmax(1.0, static_cast<double>(x.rows) / x.cols)));
    }
    auto spread = [&](auto&& count) {
      for (int i = 0; i < len; ++i) m.first[i + 1] = m.first[i] + static_cast<int>(count(i));
      return dim3(static_cast<unsigned>(m.first[len]));
    };
    const dim3 begin = spread([](int) { return kPartials; });
    hipLaunchKernelGGL(muon_begin_kernel, begin, dim3(256), 0, s, m);
    const dim3 tiles = spread([&](int i) { return d[i].sp / kTile * (d[i].tp / kTile); });
    hipLaunchKernelGGL(muon_scale_kernel, tiles, dim3(256), 0, s, m);

    // tiles with the longest reduction start first
    int by_length[gemm::kPolyMost];
    for (int i = 0; i < len; ++i) by_length[i] = i;
    std::stable_sort(by_length, by_length + len, [&](int a, int b) { return d[a].tp > d[b].tp; });
    // product `which` of step k: 0 G, 1 P, 2 X
    auto product = [&](int k, int which) {
      const gemm::Tile tile = which == 2 ? tile_x : tile_square;
      gemm::PolyGroup g = {};
      g.n = len;
      for (int n = 0; n < len; ++n) {
        const int i = which == 0 ? by_length[n] : n;
        gemm::GemmArgs& q = g.p[n];
        const Sides& e = d[i];
        f16 *const xh = hi[k & 1][i], *const xl = lo[k & 1][i];
        q.thrice = e.exact;
        q.M = e.sp;
        if (which == 0) {
          q.a = q.b = xh; q.a2 = q.b2 = xl;
          q.lda = q.ldb = e.tp; q.K = e.tp; q.N = e.sp;
          q.c = G[0][i]; q.c2 = G[1][i]; q.ldc = e.sp;
          q.alpha = S * S / (Sx * Sx); q.tri = 1;
        } else if (which == 1) {
          q.a = q.b = q.r = G[0][i]; q.a2 = q.b2 = q.z = G[1][i];
          q.lda = q.ldb = e.sp; q.K = e.sp; q.N = e.sp;
          q.c = P[0][i]; q.c2 = P[1][i]; q.ldc = e.sp;
          q.alpha = static_cast<float>(h.c * R / (static_cast<double>(S) * S * S * S));
          q.beta = static_cast<float>(h.b * R / (static_cast<double>(S) * S));
          q.tri = 1;
        } else {
          q.a = P[0][i]; q.a2 = P[1][i]; q.lda = e.sp;
          q.b = xh; q.b2 = xl; q.ldb = e.tp;
          q.K = e.sp; q.N = e.tp;
          q.r = xh; q.z = xl;
          q.c = hi[1 - (k & 1)][i]; q.c2 = lo[1 - (k & 1)][i]; q.ldc = e.tp;
          q.alpha = 1.f / R; q.beta = static_cast<float>(h.a);
        }
        const int64_t rows = (q.M + gemm::tile_rows(tile) - 1) / gemm::tile_rows(tile);
        g.first[n + 1] = g.first[n] + static_cast<int>(q.tri ? rows * (rows + 1) / 2
                                                             : gemm::tile_count(tile, q.M, q.N));
      }
      if (which == 2)
        gemm::launch_poly_kmajor(tile, g, s);
      else
        gemm::launch_poly(tile, g, s);
    };
    for (int k = 0; k < h.steps; ++k)
      for (int which = 0; which < 3; ++which) product(k, which);
    for (int i = 0; i < len; ++i) {
      m.p[i].hi = hi[h.steps & 1][i];
      m.p[i].lo = lo[h.steps & 1][i];
    }
    hipLaunchKernelGGL(muon_finish_kernel, tiles, dim3(256), 0, s, m);
    at += len;
  }
  return launch_status(who);
}

}  // namespace

}  // namespace zk

using namespace zk;

extern "C" int64_t zk_muon_workspace(const zk_muon_matrix* list, int64_t n) {
  if (list == nullptr || n <= 0) return 0;
  int64_t most = 0;
  for (int64_t at = 0; at < n;) {
    Sides d[gemm::kPolyMost];
    const int len = run_length(list + at, n - at);
    plan_run(list + at, len, d);
    int64_t sum = 256;
    for (int i = 0; i < len; ++i) sum += bytes_of(d[i]);
    most = sum > most ? sum : most;
    at += len;
  }
  return most;
}

extern "C" int zk_orthogonalize(const zk_muon_matrix* list, int64_t n, int steps, double a, double b,
                                double c, double eps, void* workspace, int64_t workspace_bytes,
                                zk_stream_t stream) {
  const Hyper h = {steps, a, b, c, eps, 0, 0, 0, 0, 0};
  return run_list("zk_orthogonalize", list, n, false, h, workspace, workspace_bytes, as_stream(stream));
}

extern "C" int zk_muon_multi(const zk_muon_matrix* list, int64_t n, int steps, double a, double b, double c,
                             double eps, double lr, double momentum, double weight_decay, int nesterov,
                             int adjust, void* workspace, int64_t workspace_bytes, zk_stream_t stream) {
  const char* who = "zk_muon_multi";
  ZK_REQUIRE(lr >= 0 && weight_decay >= 0 && momentum >= 0 && momentum < 1, ZK_EINVAL,
             "%s: lr %g, momentum %g, weight decay %g", who, lr, momentum, weight_decay);
  ZK_REQUIRE(adjust == ZK_MUON_ORIGINAL || adjust == ZK_MUON_MATCH_RMS, ZK_EINVAL, "%s: bad adjustment %d",
             who, adjust);
  const Hyper h = {steps, a, b, c, eps, lr, momentum, weight_decay, nesterov, adjust};
  return run_list(who, list, n, true, h, workspace, workspace_bytes, as_stream(stream));
}
