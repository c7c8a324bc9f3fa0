// AdamW steps over lists of tensors, with the moments in 32 or in 8 bits.
//
// One launch steps as many tensors as their table fits into a kernel's
// arguments (no table in device memory to fill, nothing to keep for a captured
// launch).  A workgroup steps kTile elements of one tensor, which it finds by
// comparing its number with the tensors' first ones, a lane for each.
//
// HBM bounds all of it: 28 bytes an element with 32-bit moments and gradients,
// 16 with 8-bit moments, 16-bit gradients and a 16-bit copy.  605 M elements with
// 8-bit moments, bf16 gradients and copies (9.7 GB) take 1540 us, 6.3 TB/s; their
// moments read as bf16 (3.6 GB) 600 us, 6.0 TB/s; 65 tensors of 4096 with 32-bit
// moments two launches of 5 us.  Small lists are bound by their launches: 150
// tensors of up to 300000 elements, 5 M in all, are four launches of 6 to 10 us.
//
// 8-bit moments (the format is stated in zorse_amd.h): r(x), the top 12 bits
// below the sign of a float, is an integer that grows with |x|, 8 steps an
// octave.  256 neighbouring elements share the integer that their codes are
// counted from.  Since it is an integer, moving it with the block's largest
// value rounds nothing again: a code that does not change its value stays what
// it is.  The second moment changes by 1 - beta2 of its distance from g^2 a
// step, far less than the eighth of an octave between codes, so rounding it to
// nearest would hold it where it is for ever; rounded up with the probability
// of the fraction cut off, it moves rarely and by whole steps, and its mean is
// right.  The first moment moves by a tenth and is rounded to nearest.
#include "adamw_math.h"

namespace zk {

static constexpr int kTile = 1024;        // elements a workgroup steps
static constexpr int kMax32 = 56, kMax8 = 44;  // tensors a launch: 4 KB of arguments
static constexpr int64_t kPiece = int64_t(1) << 31;       // elements of a tensor a launch
static constexpr int64_t kMaxGrid = int64_t(1) << 23;     // workgroups a launch
// Larger tensors with 32-bit moments are launched alone (adamw.hip's kernel, an
// element a thread): it streams 6.5 TB/s where a workgroup that first looks its
// tensor up reaches 6.0, and a launch costs 3 us.  us for equal tensors, alone
// / in one launch: 48 of 2^20 elements 317 / 238, 24 of 2^22 507 / 504, 12 of
// 2^23 460 / 498, 4 of 2^25 567 / 612.
static constexpr int64_t kAlone = 6 << 20;

struct AdamCommon {
  float decay, one_minus_b1, b2, one_minus_b2, eps;
};

struct Tensor32 {
  float* p;
  const void* g;
  float* m;
  float* v;
  void* low;
  int64_t n;
  float step_size, bc2_sqrt;
  int g_dt, low_dt;  // low_dt -1: no copy
};
struct Tensor8 {
  float* p;
  const void* g;
  uint8_t* m;
  uint8_t* v;
  int16_t* base;
  void* low;
  int64_t n, index0;  // index0: of the piece's first element in its tensor
  float step_size, bc2_sqrt, inv_bc2;
  uint32_t seed;
  short g_dt, low_dt;
};
struct View8 {
  const uint8_t* m;
  const uint8_t* v;
  const int16_t* base;
  void* mo;
  void* vo;
  int64_t n;
};

template <typename E, int N>
struct Table {
  E e[N];
  int first[N];  // first workgroup of each
  AdamCommon c;
  int count;
};
static_assert(sizeof(Table<Tensor32, kMax32>) <= 4096 && sizeof(Table<Tensor8, kMax8>) <= 4096 &&
                  kMax32 <= 64 && kMax8 <= 64,
              "a table is a kernel's arguments, a lane looks at each tensor");

// The tensor that a workgroup belongs to.
template <typename E, int N>
__device__ __forceinline__ int find_tensor(const Table<E, N>& t) {
  const int lane = threadIdx.x & 63;
  const bool at_or_before = lane < t.count && t.first[lane < N ? lane : 0] <= static_cast<int>(blockIdx.x);
  return __builtin_amdgcn_readfirstlane(__popcll(__ballot(at_or_before)) - 1);
}

__device__ __forceinline__ AdamScalars scalars(const AdamCommon& c, float step_size, float bc2_sqrt) {
  return AdamScalars{c.decay, c.one_minus_b1, c.b2, c.one_minus_b2, step_size, bc2_sqrt, c.eps};
}

// One element a lane and access (see adamw.hip), four of them in flight.
template <typename G, typename L, bool kCopy>
__device__ __forceinline__ void step32(const Tensor32& t, const AdamScalars& s, int64_t i0) {
  const G* g = static_cast<const G*>(t.g);
  constexpr int K = kTile / 256;
  float p[K], m[K], v[K], gv[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int64_t i = i0 + k * 256;
    if (i < t.n) {
      p[k] = __builtin_nontemporal_load(t.p + i);
      m[k] = __builtin_nontemporal_load(t.m + i);
      v[k] = __builtin_nontemporal_load(t.v + i);
      gv[k] = static_cast<float>(__builtin_nontemporal_load(g + i));
    }
  }
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int64_t i = i0 + k * 256;
    if (i < t.n) {
      adam_one(p[k], gv[k], m[k], v[k], s);
      __builtin_nontemporal_store(p[k], t.p + i);
      __builtin_nontemporal_store(m[k], t.m + i);
      __builtin_nontemporal_store(v[k], t.v + i);
      if (kCopy) {
        asm volatile("" : "+v"(p[k]));  // round the stored fp32 value (see adamw.hip)
        __builtin_nontemporal_store(static_cast<L>(p[k]), static_cast<L*>(t.low) + i);
      }
    }
  }
}

template <typename G>
__device__ __forceinline__ void step32_low(const Tensor32& t, const AdamScalars& s, int64_t i0) {
  if (t.low_dt < 0) step32<G, float, false>(t, s, i0);
  else if (t.low_dt == ZK_BF16) step32<G, bf16, true>(t, s, i0);
  else if (t.low_dt == ZK_F16) step32<G, f16, true>(t, s, i0);
  else step32<G, float, true>(t, s, i0);
}

__global__ __launch_bounds__(256) void adamw_list(const Table<Tensor32, kMax32> tab) {
  const int k = find_tensor(tab);
  const Tensor32 t = tab.e[k];
  const AdamScalars s = scalars(tab.c, t.step_size, t.bc2_sqrt);
  const int64_t i0 = static_cast<int64_t>(static_cast<int>(blockIdx.x) - tab.first[k]) * kTile +
                     threadIdx.x;
  if (t.g_dt == ZK_BF16) step32_low<bf16>(t, s, i0);
  else if (t.g_dt == ZK_F16) step32_low<f16>(t, s, i0);
  else step32_low<float>(t, s, i0);
}

// ------------------------------------------------------------ 8-bit moments --
// N neighbouring elements, the first n of them, at any alignment.
template <typename T, int N>
struct PartN {
  typedef T VN __attribute__((ext_vector_type(N)));
  typedef VN VNu __attribute__((aligned(sizeof(T))));
  VN u;
  __device__ __forceinline__ void load(const T* p, int n) {
    if (n >= N) {
      u = __builtin_nontemporal_load(reinterpret_cast<const VNu*>(p));
      return;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) u[i] = i < n ? p[i] : static_cast<T>(0);
  }
  __device__ __forceinline__ void store(T* p, int n) const {
    if (n >= N) {
      __builtin_nontemporal_store(u, reinterpret_cast<VNu*>(p));
      return;
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < n) p[i] = u[i];
  }
};

static constexpr int kLane = 4;    // neighbouring elements a lane: a block a wave
static constexpr int kTile8 = 256 * kLane;
static constexpr int kLaneR = 8, kTileR = 256 * kLaneR;  // of the reading kernel
static constexpr int kTopM = 127, kTopV = 255;     // largest codes
static constexpr uint32_t kMaxR = 0x7f7;           // r of the largest finite float
static constexpr uint32_t kInf = 0x7f800000u;

__device__ __forceinline__ float code_value(uint32_t c, int base) {
  return c != 0 ? __uint_as_float((c + base) << 20) : 0.f;
}
__device__ __forceinline__ float code_value_m(uint32_t c, int base) {
  const float v = code_value(c & 127, base);
  return c & 128 ? -v : v;
}

// 20 random bits of element i + k: index and seed through two products with
// odd constants (the fractions of the roots of 2 and 3 times 2^32) and shifts.
// `mixed` is mix_index(seed, i), whose products (quarter rate) a lane takes
// once; i is a multiple of kLane, so i + k carries nothing over.
static constexpr uint32_t kIndexMul = 0x9E3779B1u;
__device__ __forceinline__ uint32_t mix_index(uint32_t seed, int64_t i) {
  return static_cast<uint32_t>(i) * kIndexMul +
         static_cast<uint32_t>(static_cast<uint64_t>(i) >> 32) * 0x85157AF5u + seed;
}
__device__ __forceinline__ uint32_t random20(uint32_t mixed, int k) {
  uint32_t x = mixed + static_cast<uint32_t>(k) * kIndexMul;
  x = (x ^ (x >> 16)) * 0x6A09E667u;
  x = (x ^ (x >> 15)) * 0xBB67AE85u;
  return (x ^ (x >> 16)) >> 12;
}

// r of a float (its bits below the sign), rounded to nearest, ties to even.
__device__ __forceinline__ uint32_t r_nearest(uint32_t b) {
  return (b + 0x7ffff + ((b >> 20) & 1)) >> 20;
}

// The update with the hardware's reciprocal and root (1 ulp each) in place of
// the IEEE sequences, for moments whose roots and squares neither overflow nor
// reach the numbers that those flush; 30 operations fewer an element, without
// which the vector units and not HBM would bound the step.
__device__ __forceinline__ void adam_one_fast(float& p, float g, float& m, float& v,
                                              const AdamScalars& s, float inv_bc2) {
  m = fmaf(s.one_minus_b1, g - m, m);
  v = fmaf(s.one_minus_b2, g * g, v * s.b2);
  const float denom = fmaf(__builtin_amdgcn_sqrtf(v), inv_bc2, s.eps);
  p = fmaf(-s.step_size, m * __builtin_amdgcn_rcpf(denom), p * s.decay);
}

// One lane's elements after the update.
struct Rounded {
  uint32_t bm[kLane];            // the first moment's bits
  uint32_t rm[kLane], rv[kLane];
  bool zero[kLane], odd[kLane];  // second moment 0; not finite
};

template <bool kFast, typename G>
__device__ __forceinline__ bool update8(PartN<float, kLane>& p, const PartN<G, kLane>& g,
                                        const PartN<uint8_t, kLane>& mc,
                                        const PartN<uint8_t, kLane>& vc, int mb, int vb,
                                        const AdamScalars& s, float inv_bc2, uint32_t mixed,
                                        Rounded& R) {
  bool fast = true;
#pragma unroll
  for (int k = 0; k < kLane; ++k) {
    float m = code_value_m(mc.u[k], mb), v = code_value(vc.u[k], vb), q = p.u[k];
    if (kFast) adam_one_fast(q, static_cast<float>(g.u[k]), m, v, s, inv_bc2);
    else adam_one(q, static_cast<float>(g.u[k]), m, v, s);
    p.u[k] = q;
    const uint32_t bm = __float_as_uint(m), bv = __float_as_uint(v);
    R.bm[k] = bm;
    R.zero[k] = bv == 0;
    R.rm[k] = r_nearest(bm & 0x7fffffffu);
    R.rv[k] = (bv + random20(mixed, k)) >> 20;
    R.odd[k] = false;
    if (kFast) {
      // 2^-96 .. 2^120, or 0: finite, and so is m
      fast = fast && (R.zero[k] || bv - (31u << 23) <= (216u << 23));
    } else {
      R.odd[k] = (bm & 0x7fffffffu) >= kInf || (bv & 0x7fffffffu) >= kInf;
      R.rm[k] = R.odd[k] ? 0 : R.rm[k] < kMaxR ? R.rm[k] : kMaxR;
      R.rv[k] = R.odd[k] ? 0 : R.rv[k] < kMaxR ? R.rv[k] : kMaxR;
    }
  }
  return fast;
}

// The largest r of both moments in a wave's block, 16 bits each: the lanes of
// 16 by rotations among them, the four sixteens by the two broadcasts, and the
// last lane's for all (elements behind the tensor's last have only zeros for
// inputs, and r = 0).
typedef uint16_t Largest __attribute__((ext_vector_type(2)));
template <int kCtrl, int kRows>
__device__ __forceinline__ Largest max_with(Largest x) {
  const int y = __builtin_bit_cast(int, x);
  return __builtin_elementwise_max(
      x, __builtin_bit_cast(Largest, __builtin_amdgcn_update_dpp(y, y, kCtrl, kRows, 0xf, false)));
}
__device__ __forceinline__ Largest block_largest(const Rounded& R) {
  uint32_t a = R.rm[0], b = R.rv[0];
#pragma unroll
  for (int k = 1; k < kLane; ++k) {
    a = R.rm[k] > a ? R.rm[k] : a;
    b = R.rv[k] > b ? R.rv[k] : b;
  }
  Largest most = __builtin_bit_cast(Largest, b << 16 | a);
  most = max_with<0x121, 0xf>(most);  // row_ror:1, 2, 4, 8
  most = max_with<0x122, 0xf>(most);
  most = max_with<0x124, 0xf>(most);
  most = max_with<0x128, 0xf>(most);
  most = max_with<0x142, 0xa>(most);  // row_bcast:15 into rows 1 and 3
  most = max_with<0x143, 0xc>(most);  // row_bcast:31 into rows 2 and 3
  return __builtin_bit_cast(Largest, __builtin_amdgcn_readlane(__builtin_bit_cast(int, most), 63));
}

__device__ __forceinline__ uint32_t four_bytes(const uint32_t (&b)[4]) {
  return (b[3] << 8 | b[2]) << 16 | (b[1] << 8 | b[0]);
}

// One block of 256 elements a wave, from element i of this lane on; kFull: all
// of them are there.
template <typename G, typename L, bool kCopy, bool kFull>
__device__ __forceinline__ void step8(const Tensor8& t, const AdamScalars& s, int64_t i) {
  const int n = kFull ? kLane : i < t.n ? (t.n - i < kLane ? static_cast<int>(t.n - i) : kLane) : 0;
  PartN<float, kLane> p;
  PartN<G, kLane> g;
  PartN<uint8_t, kLane> mc, vc;
  p.load(t.p + i, n);
  g.load(static_cast<const G*>(t.g) + i, n);
  mc.load(t.m + i, n);
  vc.load(t.v + i, n);
  const int64_t block = __builtin_amdgcn_readfirstlane(static_cast<int>(i >> 8));
  int16_t* bp = t.base + block * 2;
  const int mb = bp[0], vb = bp[1];
  Rounded R;
  const uint32_t mixed = mix_index(t.seed, t.index0 + i);
  bool fast = s.eps == 0.f || s.eps >= 1e-30f;
  fast = update8<true>(p, g, mc, vc, mb, vb, s, t.inv_bc2, mixed, R) && fast;
  const bool slow = __ballot(!fast) != 0;
  if (slow) {  // the IEEE sequences, and codes of what is not finite
    p.load(t.p + i, n);
    update8<false>(p, g, mc, vc, mb, vb, s, 0.f, mixed, R);
  }
  p.store(t.p + i, n);
  if (kCopy) {
    PartN<L, kLane> low;
#pragma unroll
    for (int k = 0; k < kLane; ++k) {
      float q = p.u[k];
      asm volatile("" : "+v"(q));  // round the stored fp32 value (see adamw.hip)
      low.u[k] = static_cast<L>(q);
    }
    low.store(static_cast<L*>(t.low) + i, n);
  }
  const Largest most = block_largest(R);
  const uint32_t nm = most[0] > kTopM ? most[0] - kTopM : 0, nv = most[1] > kTopV ? most[1] - kTopV : 0;
  uint32_t cm[kLane], cv[kLane];
#pragma unroll
  for (int k = 0; k < kLane; ++k) {
    const uint32_t a = __builtin_elementwise_sub_sat(R.rm[k], nm);
    const uint32_t b = __builtin_elementwise_sub_sat(R.rv[k], nv);
    cm[k] = a != 0 ? a | (R.bm[k] >> 24 & 128) : 0;
    cv[k] = R.zero[k] ? 0 : b > 1 ? b : 1;
    if (slow && R.odd[k]) {
      cm[k] = kTopM | (R.bm[k] >> 24 & 128);
      cv[k] = kTopV;
    }
  }
  mc.u = __builtin_bit_cast(decltype(mc.u), four_bytes(cm));
  vc.u = __builtin_bit_cast(decltype(vc.u), four_bytes(cv));
  mc.store(t.m + i, n);
  vc.store(t.v + i, n);
  if ((threadIdx.x & 63) == 0) {
    bp[0] = static_cast<int16_t>(nm);
    bp[1] = static_cast<int16_t>(nv);
  }
}

template <typename G, typename L, bool kCopy>
__device__ __forceinline__ void block8(const Tensor8& t, const AdamScalars& s, int64_t i) {
  const int64_t first = i - (threadIdx.x & 63) * kLane;
  if (first >= t.n) return;
  if (first + 256 <= t.n) step8<G, L, kCopy, true>(t, s, i);
  else step8<G, L, kCopy, false>(t, s, i);
}

template <typename G>
__device__ __forceinline__ void block8_low(const Tensor8& t, const AdamScalars& s, int64_t i) {
  if (t.low_dt < 0) block8<G, float, false>(t, s, i);
  else if (t.low_dt == ZK_BF16) block8<G, bf16, true>(t, s, i);
  else if (t.low_dt == ZK_F16) block8<G, f16, true>(t, s, i);
  else block8<G, float, true>(t, s, i);
}

__global__ __launch_bounds__(256) void adamw8_list(const Table<Tensor8, kMax8> tab) {
  const int k = find_tensor(tab);
  const Tensor8 t = tab.e[k];
  const AdamScalars s = scalars(tab.c, t.step_size, t.bc2_sqrt);
  const int64_t i = static_cast<int64_t>(static_cast<int>(blockIdx.x) - tab.first[k]) * kTile8 +
                    threadIdx.x * kLane;
  if (t.g_dt == ZK_BF16) block8_low<bf16>(t, s, i);
  else if (t.g_dt == ZK_F16) block8_low<f16>(t, s, i);
  else block8_low<float>(t, s, i);
}

template <typename T>
__global__ __launch_bounds__(256) void adamw8_read(const Table<View8, kMax32> tab) {
  const int k = find_tensor(tab);
  const View8 t = tab.e[k];
  const int64_t i = static_cast<int64_t>(static_cast<int>(blockIdx.x) - tab.first[k]) * kTileR +
                    threadIdx.x * kLaneR;
  if (i >= t.n) return;
  const int n = t.n - i < kLaneR ? static_cast<int>(t.n - i) : kLaneR;
  const int mb = t.base[i / 256 * 2], vb = t.base[i / 256 * 2 + 1];
  PartN<uint8_t, kLaneR> mc, vc;
  mc.load(t.m + i, n);
  vc.load(t.v + i, n);
  PartN<T, kLaneR> mo, vo;
#pragma unroll
  for (int q = 0; q < kLaneR; ++q) {
    mo.u[q] = static_cast<T>(code_value_m(mc.u[q], mb));
    vo.u[q] = static_cast<T>(code_value(vc.u[q], vb));
  }
  mo.store(static_cast<T*>(t.mo) + i, n);
  vo.store(static_cast<T*>(t.vo) + i, n);
}

// ------------------------------------------------------------------- host ---
// Fills tables and launches them as they fill up.
template <typename E, int N, int kTileOf, typename F>
struct Launcher {
  Table<E, N> t;
  int64_t grid = 0;
  bool any = false;
  F launch;
  explicit Launcher(F f) : launch(f) { t.count = 0; }
  void add(const E& e) {
    const int64_t wgs = (e.n + kTileOf - 1) / kTileOf;
    if (wgs == 0) return;
    if (t.count == N || grid + wgs > kMaxGrid) flush();
    t.e[t.count] = e;
    t.first[t.count++] = static_cast<int>(grid);
    grid += wgs;
  }
  void flush() {
    if (t.count == 0) return;
    launch(t, dim3(static_cast<unsigned>(grid)));
    any = true;
    t.count = 0;
    grid = 0;
  }
  int status(const char* who) {
    flush();
    return any ? launch_status(who) : ZK_OK;
  }
};

static AdamCommon common(double lr, double beta1, double beta2, double eps, double wd) {
  const AdamScalars s = adam_scalars(lr, beta1, beta2, eps, wd, 1);
  return AdamCommon{s.decay, s.one_minus_b1, s.b2, s.one_minus_b2, s.eps};
}

static int check_hyper(const char* who, int64_t count, const void* table, double lr, double beta1,
                       double beta2, double eps, double wd) {
  ZK_REQUIRE(count >= 0 && (count == 0 || table), ZK_EINVAL, "%s: null table", who);
  ZK_REQUIRE(lr >= 0 && beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1 && eps >= 0 && wd >= 0,
             ZK_EINVAL, "%s: hyper-parameter out of range", who);
  return ZK_OK;
}

// What both tables' rows share.
template <typename R>
static int check_row(const char* who, int64_t i, const R& r) {
  ZK_REQUIRE(r.grad_dtype >= 0 && r.grad_dtype <= 2 && (!r.lowp || (r.lowp_dtype >= 0 && r.lowp_dtype <= 2)),
             ZK_EDTYPE, "%s: tensor %lld: bad dtype (%lld, %lld)", who, (long long)i,
             (long long)r.grad_dtype, (long long)r.lowp_dtype);
  ZK_REQUIRE(r.n >= 0 && r.step >= 1, ZK_EINVAL,
             "%s: tensor %lld: n %lld must not be negative, step %lld at least 1", who, (long long)i,
             (long long)r.n, (long long)r.step);
  ZK_REQUIRE(r.n == 0 || (r.param && r.grad && r.exp_avg && r.exp_avg_sq), ZK_EINVAL,
             "%s: tensor %lld: null pointer", who, (long long)i);
  ZK_REQUIRE(aligned(r.param, 4) && aligned(r.grad, dtype_bytes(static_cast<int>(r.grad_dtype))) &&
                 (!r.lowp || aligned(r.lowp, dtype_bytes(static_cast<int>(r.lowp_dtype)))),
             ZK_EALIGN, "%s: tensor %lld: operands must be aligned to their element size", who,
             (long long)i);
  return ZK_OK;
}

template <typename T>
static T* ahead(T* p, int64_t n) { return p ? p + n : nullptr; }
static const void* ahead_dt(const void* p, int64_t n, int dt) {
  return p ? static_cast<const char*>(p) + n * dtype_bytes(dt) : nullptr;
}

}  // namespace zk

using namespace zk;

extern "C" int zk_adamw_multi(const zk_adamw_tensor* tensors, int64_t count, double lr,
                              double beta1, double beta2, double eps, double weight_decay,
                              zk_stream_t stream) {
  const char* who = "zk_adamw_multi";
  int rc = check_hyper(who, count, tensors, lr, beta1, beta2, eps, weight_decay);
  for (int64_t i = 0; rc == ZK_OK && i < count; ++i) {
    rc = check_row(who, i, tensors[i]);
    if (rc == ZK_OK)
      ZK_REQUIRE(aligned(tensors[i].exp_avg, 4) && aligned(tensors[i].exp_avg_sq, 4), ZK_EALIGN,
                 "%s: tensor %lld: operands must be aligned to their element size", who, (long long)i);
  }
  if (rc != ZK_OK) return rc;
  hipStream_t st = as_stream(stream);
  auto launch = [st](const Table<Tensor32, kMax32>& t, dim3 grid) {
    hipLaunchKernelGGL(adamw_list, grid, dim3(256), 0, st, t);
  };
  Launcher<Tensor32, kMax32, kTile, decltype(launch)> L(launch);
  L.t.c = common(lr, beta1, beta2, eps, weight_decay);
  for (int64_t i = 0; i < count; ++i) {
    const zk_adamw_tensor& r = tensors[i];
    const AdamScalars s = adam_scalars(lr, beta1, beta2, eps, weight_decay, r.step);
    const int gdt = static_cast<int>(r.grad_dtype), ldt = static_cast<int>(r.lowp_dtype);
    if (r.n > kAlone) {
      for (int64_t at = 0; at < r.n; at += kPiece) {
        rc = zk_adamw_step(r.param + at, ahead_dt(r.grad, at, gdt), gdt, r.exp_avg + at,
                           r.exp_avg_sq + at, const_cast<void*>(ahead_dt(r.lowp, at, ldt)), ldt,
                           r.n - at < kPiece ? r.n - at : kPiece, lr, beta1, beta2, eps, weight_decay,
                           r.step, stream);
        if (rc != ZK_OK) return rc;
      }
      continue;
    }
    L.add(Tensor32{r.param, r.grad, r.exp_avg, r.exp_avg_sq, r.lowp, r.n, s.step_size, s.bc2_sqrt,
                   gdt, r.lowp ? ldt : -1});
  }
  return L.status(who);
}

extern "C" int zk_adamw8_multi(const zk_adamw8_tensor* tensors, int64_t count, double lr,
                               double beta1, double beta2, double eps, double weight_decay,
                               zk_stream_t stream) {
  const char* who = "zk_adamw8_multi";
  int rc = check_hyper(who, count, tensors, lr, beta1, beta2, eps, weight_decay);
  for (int64_t i = 0; rc == ZK_OK && i < count; ++i) {
    rc = check_row(who, i, tensors[i]);
    if (rc == ZK_OK) {
      ZK_REQUIRE(tensors[i].n == 0 || tensors[i].base, ZK_EINVAL, "%s: tensor %lld: null pointer", who,
                 (long long)i);
      ZK_REQUIRE(aligned(tensors[i].base, 2), ZK_EALIGN,
                 "%s: tensor %lld: operands must be aligned to their element size", who, (long long)i);
    }
  }
  if (rc != ZK_OK) return rc;
  hipStream_t st = as_stream(stream);
  auto launch = [st](const Table<Tensor8, kMax8>& t, dim3 grid) {
    hipLaunchKernelGGL(adamw8_list, grid, dim3(256), 0, st, t);
  };
  Launcher<Tensor8, kMax8, kTile8, decltype(launch)> L(launch);
  L.t.c = common(lr, beta1, beta2, eps, weight_decay);
  for (int64_t i = 0; i < count; ++i) {
    const zk_adamw8_tensor& r = tensors[i];
    const AdamScalars s = adam_scalars(lr, beta1, beta2, eps, weight_decay, r.step);
    const int gdt = static_cast<int>(r.grad_dtype), ldt = static_cast<int>(r.lowp_dtype);
    for (int64_t at = 0; at < r.n; at += kPiece)
      L.add(Tensor8{r.param + at, ahead_dt(r.grad, at, gdt), r.exp_avg + at, r.exp_avg_sq + at,
                    r.base + at / 256 * 2, const_cast<void*>(ahead_dt(r.lowp, at, ldt)),
                    r.n - at < kPiece ? r.n - at : kPiece, at, s.step_size, s.bc2_sqrt,
                    1.f / s.bc2_sqrt, static_cast<uint32_t>(r.seed), static_cast<short>(gdt),
                    static_cast<short>(r.lowp ? ldt : -1)});
  }
  return L.status(who);
}

extern "C" int zk_adamw8_values(const zk_adamw8_view* tensors, int64_t count, int out_dtype,
                                zk_stream_t stream) {
  const char* who = "zk_adamw8_values";
  ZK_REQUIRE(count >= 0 && (count == 0 || tensors), ZK_EINVAL, "%s: null table", who);
  ZK_REQUIRE(out_dtype == ZK_F32 || out_dtype == ZK_BF16, ZK_EDTYPE,
             "%s: fp32 or bf16, which hold every code's value (got %d)", who, out_dtype);
  const int e = dtype_bytes(out_dtype);
  for (int64_t i = 0; i < count; ++i) {
    const zk_adamw8_view& r = tensors[i];
    ZK_REQUIRE(r.n >= 0 && (r.n == 0 || (r.exp_avg && r.exp_avg_sq && r.base && r.m_out && r.v_out)),
               ZK_EINVAL, "%s: tensor %lld: null pointer or negative n", who, (long long)i);
    ZK_REQUIRE(aligned(r.base, 2) && aligned(r.m_out, e) && aligned(r.v_out, e), ZK_EALIGN,
               "%s: tensor %lld: operands must be aligned to their element size", who, (long long)i);
  }
  hipStream_t st = as_stream(stream);
  auto launch = [st, out_dtype](const Table<View8, kMax32>& t, dim3 grid) {
    if (out_dtype == ZK_F32) hipLaunchKernelGGL(adamw8_read<float>, grid, dim3(256), 0, st, t);
    else hipLaunchKernelGGL(adamw8_read<bf16>, grid, dim3(256), 0, st, t);
  };
  Launcher<View8, kMax32, kTileR, decltype(launch)> L(launch);
  L.t.c = AdamCommon{};
  for (int64_t i = 0; i < count; ++i) {
    const zk_adamw8_view& r = tensors[i];
    for (int64_t at = 0; at < r.n; at += kPiece)
      L.add(View8{r.exp_avg + at, r.exp_avg_sq + at, r.base + at / 256 * 2,
                  static_cast<char*>(r.m_out) + at * e, static_cast<char*>(r.v_out) + at * e,
                  r.n - at < kPiece ? r.n - at : kPiece});
  }
  return L.status(who);
}
