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
// types), 2^log_g lanes a row, so a row's sums take log_g steps among lanes and
// a wave holds 64 >> log_g rows at a time: those of one position, or of several
// where heads are few.  A wave goes through the heads of its positions, query
// and key heads being different waves' work, so that cos, sin and the weight
// are read once for all of them.  HBM bounds both directions: x and y, or x, dy
// and dx.  bf16 heads of 128, forward / backward: 32 and 32 of 4096 positions
// (134 / 201 MB) 24.5 us, 5.5 TB/s / 36.7 us, 5.5 TB/s; 32 and 8 of 30035
// positions (615 / 923 MB) 120 us, 5.1 TB/s / 184 us, 5.0 TB/s.  fp32 heads of
// 100, interleaved, 32 and 32 of 2048 (105 / 157 MB): 24.8 / 32.0 us.  One token
// of three sequences, 40 heads: 4.0 us, a launch.
#include <type_traits>

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

// One lane's 8 pairs of a row from pair i0 on: elements i and i + half of the
// half-split pairing, 2i and 2i + 1 of the interleaved one.  Every lane loads 8
// pairs that exist (n of them where a row has fewer, in all lanes): a row's last
// lane takes its last 8 and leaves the first `skip` of them, which are another
// lane's, out of the sums and the stores; a lane behind it leaves all out.
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
  __device__ __forceinline__ void drop(int skip) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const bool out = i < skip;
      if (kPairing == ZK_ROPE_HALF) {
        a.u[i] = out ? static_cast<T>(0.f) : a.u[i];
        b.u[i] = out ? static_cast<T>(0.f) : b.u[i];
      } else if (i < 4) {
        a.u[2 * i] = out ? static_cast<T>(0.f) : a.u[2 * i];
        a.u[2 * i + 1] = out ? static_cast<T>(0.f) : a.u[2 * i + 1];
      } else {
        b.u[2 * i - 8] = out ? static_cast<T>(0.f) : b.u[2 * i - 8];
        b.u[2 * i - 7] = out ? static_cast<T>(0.f) : b.u[2 * i - 7];
      }
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
                                               int i0, int half, int skip, int n) {
    if (skip == 0 && n == 8) {
      if (kPairing == ZK_ROPE_HALF) {
        Part8<T>::store(row + i0, u, 8);
        Part8<T>::store(row + half + i0, v, 8);
      } else {
        const float lo[8] = {u[0], v[0], u[1], v[1], u[2], v[2], u[3], v[3]};
        const float hi[8] = {u[4], v[4], u[5], v[5], u[6], v[6], u[7], v[7]};
        Part8<T>::store(row + 2 * i0, lo, 8);
        Part8<T>::store(row + 2 * i0 + 8, hi, 8);
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i >= skip && i < n) {
        row[kPairing == ZK_ROPE_HALF ? i0 + i : 2 * (i0 + i)] = static_cast<T>(u[i]);
        row[kPairing == ZK_ROPE_HALF ? half + i0 + i : 2 * (i0 + i) + 1] = static_cast<T>(v[i]);
      }
  }
};

// The sums of two values over a row's lanes, in every lane of the row: among
// 16 lanes by permutations within them, then across.
template <int kCtrl>
__device__ __forceinline__ float lanes_add(float v) {
  return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(
                                           0, __builtin_bit_cast(int, v), kCtrl, 0xf, 0xf, true));
}
template <bool kBoth>
__device__ __forceinline__ void row_sums(float& a, float& b, int lanes) {
  if (lanes > 1) {
    a = lanes_add<0xb1>(a);  // quad_perm: 1 0 3 2
    if (kBoth) b = lanes_add<0xb1>(b);
  }
  if (lanes > 2) {
    a = lanes_add<0x4e>(a);  // quad_perm: 2 3 0 1
    if (kBoth) b = lanes_add<0x4e>(b);
  }
  if (lanes > 4) {
    a = lanes_add<0x141>(a);  // row_half_mirror: the other four of 8
    if (kBoth) b = lanes_add<0x141>(b);
  }
  if (lanes > 8) {
    a = lanes_add<0x140>(a);  // row_mirror: the other 8 of 16
    if (kBoth) b = lanes_add<0x140>(b);
  }
  if (lanes > 16) {
    a += __shfl_xor(a, 16, 64);
    if (kBoth) b += __shfl_xor(b, 16, 64);
  }
  if (lanes > 32) {
    a += __shfl_xor(a, 32, 64);
    if (kBoth) b += __shfl_xor(b, 32, 64);
  }
}

template <int kPairing>
__device__ __forceinline__ void load_weight(const void* w, int dt, int i0, int half, int n,
                                            float (&a)[8], float (&b)[8]) {
  auto take = [&](auto* p) {
    typedef typename std::remove_const<typename std::remove_pointer<decltype(p)>::type>::type W;
    Pairs<W, kPairing> x;
    x.load(p, i0, half, n);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      a[i] = x.first(i);
      b[i] = x.second(i);
    }
  };
  if (dt == ZK_F32) take(static_cast<const float*>(w));
  else if (dt == ZK_BF16) take(static_cast<const bf16*>(w));
  else take(static_cast<const f16*>(w));
}

template <typename T, int kPairing, bool kBwd>
__global__ __launch_bounds__(256, 3) void qk_kernel(QkArgs A, int log_g) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const bool is_q = blockIdx.x < A.q.wgs;
  const QkSide& X = is_q ? A.q : A.k;
  const int64_t wg = is_q ? blockIdx.x : blockIdx.x - A.q.wgs;
  const int half = A.d / 2, lanes = 1 << log_g;
  const int my0 = (lane & (lanes - 1)) * 8;            // this lane's first pair, if all were there
  const int n = half < 8 ? half : 8;
  const int i0 = half < 8 ? 0 : my0 < half - 8 ? my0 : half - 8;
  const int skip = my0 - i0 < 8 ? my0 - i0 : 8;
  const bool ragged = (half & 7) != 0 || lanes * 8 != half;
  const int slot = lane >> log_g;                      // row slot of this lane
  const int log_ppw = 6 - log_g - X.log_hpw;           // positions a wave holds
  const int h0 = slot & ((1 << X.log_hpw) - 1), p_in = slot >> X.log_hpw;
  float wa[8], wb[8], da[8], db[8];
  load_weight<kPairing>(X.w, A.w_dt, i0, half, n, wa, wb);
#pragma unroll
  for (int i = 0; i < 8; ++i) da[i] = db[i] = 0.f;
  const int64_t groups = (A.rows + (1 << log_ppw) - 1) >> log_ppw;
  const int64_t items = groups * X.splits;
  const int step = X.splits << X.log_hpw;              // heads from one step to the next
  const float inv_d = 1.f / static_cast<float>(A.d);
  for (int64_t item = wg * 4 + wave; item < items; item += X.wgs * 4) {
    const int64_t group = X.splits == 1 ? item : item / X.splits;
    const int split = X.splits == 1 ? 0 : static_cast<int>(item - group * X.splits);
    const int64_t p = (group << log_ppw) + p_in;
    const bool in = p < A.rows;
    const int64_t b = in ? p / A.S : 0, s = in ? p - b * A.S : 0;
    // a slot without a position reads the first one's rows; every slot has a
    // head (2^log_hpw divides their number)
    const int h = (split << X.log_hpw) + h0;
    const T* xr = static_cast<const T*>(X.x) + b * X.x_sb + s * X.x_ss + h * X.x_sh;
    const T* gr = static_cast<const T*>(X.dy) + (kBwd ? b * X.dy_sb + s * X.dy_ss + h * X.dy_sh : 0);
    T* yr = static_cast<T*>(X.out) + b * X.o_sb + s * X.o_ss + h * X.o_sh;
    Pairs<T, kPairing> x, g;
    x.load(xr, i0, half, n);
    if (kBwd) g.load(gr, i0, half, n);
    int64_t pos = s;
    if (A.positions != nullptr && in) pos = A.positions[b * A.pos_sb + s];
    const bool known = pos >= 0 && pos < A.n_pos;  // rows off the table are NaN
    Part8<float> cs, sn;
    cs.load(A.cosT + (known ? pos : 0) * half + i0, n);
    sn.load(A.sinT + (known ? pos : 0) * half + i0, n);
    float c[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = known ? cs[i] : __builtin_nanf("");
    for (int hb = split << X.log_hpw; hb < X.heads; hb += step) {
      Pairs<T, kPairing> x1 = x, g1 = g;
      if (hb + step < X.heads) {  // the next step's rows, ahead of this one's work
        xr += step * X.x_sh;
        x.load(xr, i0, half, n);
        if (kBwd) {
          gr += step * X.dy_sh;
          g.load(gr, i0, half, n);
        }
      }
      if (ragged) {
        x1.drop(skip);
        if (kBwd) g1.drop(skip);
      }
      float ss = 0.f, t = 0.f, ga[8], gb[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float u = x1.first(i), v = x1.second(i);
        ss = fmaf(u, u, fmaf(v, v, ss));
        if (kBwd) {  // dn = R^T dy
          const float e = g1.first(i), f = g1.second(i);
          ga[i] = fmaf(e, c[i], f * sn[i]);
          gb[i] = fmaf(f, c[i], -(e * sn[i]));
          t = fmaf(ga[i] * wa[i], u, fmaf(gb[i] * wb[i], v, t));
        }
      }
      row_sums<kBwd>(ss, t, lanes);
      const float r = 1.f / sqrtf(ss * inv_d + A.eps);
      float oa[8], ob[8];
      if (!kBwd) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float u = x1.first(i) * r * wa[i], v = x1.second(i) * r * wb[i];
          oa[i] = fmaf(u, c[i], -(v * sn[i]));
          ob[i] = fmaf(v, c[i], u * sn[i]);
        }
      } else {
        t *= r * r * inv_d;  // r mean(g x r)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float u = x1.first(i), v = x1.second(i);
          if (in) {
            da[i] = fmaf(ga[i], u * r, da[i]);
            db[i] = fmaf(gb[i], v * r, db[i]);
          }
          oa[i] = r * fmaf(-t, u, ga[i] * wa[i]);
          ob[i] = r * fmaf(-t, v, gb[i] * wb[i]);
        }
      }
      if (in) Pairs<T, kPairing>::store(yr, oa, ob, i0, half, skip, n);
      yr += step * X.o_sh;
    }
  }
  if (!kBwd) return;
  // dw: this workgroup's row of partial sums, of 4 waves' row slots in order.
  // A slot's 16 * lanes values in LDS: the pairs' first elements, the second.
  __shared__ float sums[4][1024];
  float* mine = sums[wave] + slot * 16 * lanes;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i >= skip) {  // pair i0 + i < 8 lanes
      mine[i0 + i] = da[i];
      mine[8 * lanes + i0 + i] = db[i];
    }
  __syncthreads();
  for (int i = threadIdx.x; i < A.d; i += 256) {
    int at;
    if (kPairing == ZK_ROPE_HALF) at = i < half ? i : i - half + 8 * lanes;
    else at = (i & 1) * 8 * lanes + (i >> 1);
    float v = 0.f;
    for (int w = 0; w < 4; ++w)
      for (int k = 0; k < 64 / lanes; ++k) v += sums[w][k * 16 * lanes + at];
    A.part[static_cast<int64_t>(blockIdx.x) * A.d + i] = v;
  }
}

// dw [d] from the partial rows: 16 columns a workgroup, of whose 64 times 16
// threads each 16 take a share of the rows, in order.  The latency of 12 rows one
// after another bounds it: 4 us for 770 rows of 128.
__global__ __launch_bounds__(1024) void qk_dw(const float* __restrict__ part, int64_t q_rows,
                                              int64_t k_rows, int d, void* dwq, void* dwk,
                                              int w_dt) {
  __shared__ float sums[64][16];
  const int c = threadIdx.x & 15, share = threadIdx.x >> 4;
  const int col = blockIdx.x * 16 + c;
  const int64_t first = blockIdx.y == 0 ? 0 : q_rows;
  const int64_t rows = blockIdx.y == 0 ? q_rows : k_rows;
  const int64_t a = rows * share / 64, b = rows * (share + 1) / 64;
  float v = 0.f;
  if (col < d) {
#pragma unroll 8
    for (int64_t i = a; i < b; ++i) v += part[(first + i) * d + col];
  }
  sums[share][c] = v;
  __syncthreads();
  if (share != 0 || col >= d) return;
  for (int i = 1; i < 64; ++i) v += sums[i][c];
  store_dt(blockIdx.y == 0 ? dwq : dwk, col, w_dt, v);
}

static int log_lanes(int64_t d) {
  int lg = 0;
  while ((int64_t(16) << lg) < d) ++lg;
  return lg;
}

static constexpr int64_t kMaxWgs = int64_t(1) << 22;  // below 2^32 threads a launch
// The backward's workgroups, which are dw's partial rows: what three a CU hold
// at once.  us at 768 / 1024 / 2048: 32 and 32 heads of 128, 4096 positions
// 42.5 / 50.2 / 48.3, 32 and 8 heads, 30035 positions 181 / 219 / 200.
static constexpr int64_t kBwdWgs = 768;
// What a group's positions, cos and sin cost a wave, in steps through heads.
static constexpr int64_t kStart = 2;

// A wave's row slots hold 2^log_hpw heads of a position at a time: the largest
// power of two that divides the heads (32 and 8 heads in 8 slots: 8; 12: 4, of
// two positions; 5: 1, of eight), so that no slot is without a row.
static int heads_a_wave(int64_t heads, int slots_log) {
  int lh = 0;
  while (lh < slots_log && heads % (int64_t(2) << lh) == 0) ++lh;
  return lh;
}

// Steps of a wave through one group of positions, and the groups.
static int64_t steps_of(const QkSide& s) { return s.heads >> s.log_hpw; }

static void plan(QkArgs& A, int64_t Hq, int64_t Hkv, int log_g, bool bwd) {
  int64_t work[2] = {0, 0};
  QkSide* sides[2] = {&A.q, &A.k};
  const int64_t heads[2] = {Hq, Hkv};
  for (int i = 0; i < 2; ++i) {
    QkSide& s = *sides[i];
    s.heads = static_cast<int>(heads[i]);
    s.log_hpw = heads_a_wave(heads[i], 6 - log_g);
    s.splits = 1;
    s.wgs = 0;
    if (heads[i] == 0) continue;
    const int log_ppw = 6 - log_g - s.log_hpw;
    const int64_t groups = (A.rows + (int64_t(1) << log_ppw) - 1) >> log_ppw;
    // few positions: a wave for every step
    if (groups < 2048) s.splits = static_cast<int>(steps_of(s));
    s.wgs = (groups * s.splits + 3) / 4;
    // a group's positions, cos and sin cost a wave as much as kStart steps
    work[i] = groups * (steps_of(s) + kStart * s.splits);
  }
  // few enough workgroups for the partial rows of dw, shared by the work
  const int64_t cap = bwd ? kBwdWgs : 2 * kMaxWgs;
  for (int i = 0; i < 2; ++i) {
    const double share = work[i] > 0 ? static_cast<double>(work[i]) / (work[0] + work[1]) : 0.0;
    const int64_t most = static_cast<int64_t>(share * cap) > 1 ? static_cast<int64_t>(share * cap) : 1;
    if (sides[i]->wgs > most) sides[i]->wgs = most;
  }
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
  plan(A, D->Hq, D->Hkv, lg, bwd);
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
  return d > 0 && d <= 1024 ? (kBwdWgs + 2) * d * 4 : -1;
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
  // without rows, or of keys without a head, there are no partial rows: dw is zero
  hipLaunchKernelGGL(qk_dw, dim3(static_cast<unsigned>((A.d + 15) / 16), dwk ? 2 : 1),
                     dim3(1024), 0, st, A.part, A.q.wgs, A.k.wgs, A.d, dwq, dwk, A.w_dt);
  return launch_status("zk_qk_norm_rope_bwd");
}
