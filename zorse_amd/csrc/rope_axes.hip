// Rotation of query and key heads by positions of several axes (time, height,
// width of images and video): pair i of a head is turned by the angle that the
// tables hold for its own axis' position,
//   (x, y) -> (x c - y s, x s + y c),  c, s = cos / sin[positions[axis(i)][token]][i]
// in fp32 with one rounding; the transpose (the backward) with -s.
//
// Bound by the bytes of q and k, read and written once.  A thread owns V
// neighbouring pairs (16 bytes of each half where alignment allows) and turns
// them in up to kHeads heads of one token, all loads of which are issued before
// any is used; its cosines and sines are read once and serve them all.  16384
// tokens of 40 heads of 128 in bf16: 66 us a direction, 5.1 TB/s, the rate of a
// large copy; with one, two and eight heads in flight 112, 86 and 67.  Nontemporal
// loads and stores take such a pass to 61 us but a layer's rotation with the
// attention that reads it (4096 tokens, 64 heads) from 70 us to 75.
#include "zk_common.h"

namespace zk {

constexpr int kMaxPairs = 256;
constexpr int kHeads = 4;  // heads of a thread in flight

struct PairAxes {
  uint8_t axis[kMaxPairs];
};

struct AxesArgs {
  const void* q;
  const void* k;
  void* qo;
  void* ko;
  int64_t q_sb, q_ss, q_sh, k_sb, k_ss, k_sh;
  int64_t qo_sb, qo_ss, qo_sh, ko_sb, ko_ss, ko_sh;
  const float* cos;
  const float* sin;
  const int64_t* positions;  // [axes, tokens]
  int64_t tokens, S, n_pos;
  int Hq, H, half, n_chunks;
  int at_once, lanes, per_group;  // heads at once and threads of a token, tokens of a workgroup
  float sign;
};

template <typename T, int V, bool kInterleaved>
__global__ __launch_bounds__(256) void rope_axes_kernel(AxesArgs a, PairAxes axes) {
  typedef T TV __attribute__((ext_vector_type(V)));
  const int slot = threadIdx.x / a.lanes;
  const int64_t token = group_id() * a.per_group + slot;
  if (slot >= a.per_group || token >= a.tokens) return;
  const int r = threadIdx.x - slot * a.lanes;
  const int h0 = r / a.n_chunks, i0 = (r - h0 * a.n_chunks) * V;
  const int64_t b = token / a.S, s = token - b * a.S;

  float c[V], sn[V];
  {
    int64_t at[V];
    bool in[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int64_t pos = a.positions[axes.axis[i0 + j] * a.tokens + token];
      in[j] = pos >= 0 && pos < a.n_pos;
      at[j] = (in[j] ? pos : 0) * a.half + i0 + j;
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
      c[j] = a.cos[at[j]];
      sn[j] = a.sin[at[j]] * a.sign;
    }
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (!in[j]) c[j] = sn[j] = NAN;  // outside the tables
  }
  const T* qi = static_cast<const T*>(a.q) + b * a.q_sb + s * a.q_ss;
  T* qo = static_cast<T*>(a.qo) + b * a.qo_sb + s * a.qo_ss;
  const T* ki = static_cast<const T*>(a.k) + b * a.k_sb + s * a.k_ss;
  T* ko = static_cast<T*>(a.ko) + b * a.ko_sb + s * a.ko_ss;
  const int e0 = kInterleaved ? 2 * i0 : i0, e1 = kInterleaved ? 2 * i0 + V : i0 + a.half;
  for (int hb = h0; hb < a.H; hb += kHeads * a.at_once) {
    TV x[kHeads], y[kHeads];
#pragma unroll
    for (int n = 0; n < kHeads; ++n) {
      const int h = hb + n * a.at_once;
      if (h >= a.H) break;
      const T* row = h < a.Hq ? qi + h * a.q_sh : ki + (h - a.Hq) * a.k_sh;
      x[n] = *reinterpret_cast<const TV*>(row + e0);
      y[n] = *reinterpret_cast<const TV*>(row + e1);
    }
#pragma unroll
    for (int n = 0; n < kHeads; ++n) {
      const int h = hb + n * a.at_once;
      if (h >= a.H) break;
      TV u, w;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        float p, q;
        if constexpr (kInterleaved) {
          p = to_f32(2 * j < V ? x[n][2 * j % V] : y[n][2 * j % V]);
          q = to_f32(2 * j + 1 < V ? x[n][(2 * j + 1) % V] : y[n][(2 * j + 1) % V]);
        } else {
          p = to_f32(x[n][j]);
          q = to_f32(y[n][j]);
        }
        const T pr = from_f32<T>(fmaf(p, c[j], -(q * sn[j])));
        const T qr = from_f32<T>(fmaf(q, c[j], p * sn[j]));
        if constexpr (kInterleaved) {
          if (2 * j < V) u[2 * j % V] = pr; else w[2 * j % V] = pr;
          if (2 * j + 1 < V) u[(2 * j + 1) % V] = qr; else w[(2 * j + 1) % V] = qr;
        } else {
          u[j] = pr;
          w[j] = qr;
        }
      }
      T* row = h < a.Hq ? qo + h * a.qo_sh : ko + (h - a.Hq) * a.ko_sh;
      *reinterpret_cast<TV*>(row + e0) = u;
      *reinterpret_cast<TV*>(row + e1) = w;
    }
  }
}

template <typename T, int V>
static void launch_rope_axes(AxesArgs& a, const PairAxes& axes, bool interleaved, hipStream_t s) {
  a.n_chunks = a.half / V;
  a.at_once = (a.H + kHeads - 1) / kHeads;
  const int most = a.n_chunks < 256 ? 256 / a.n_chunks : 1;
  if (a.at_once > most) a.at_once = most;
  a.lanes = a.at_once * a.n_chunks;
  a.per_group = 256 / a.lanes;
  const dim3 grid = group_grid((a.tokens + a.per_group - 1) / a.per_group);
  if (interleaved)
    hipLaunchKernelGGL((rope_axes_kernel<T, V, true>), grid, dim3(256), 0, s, a, axes);
  else
    hipLaunchKernelGGL((rope_axes_kernel<T, V, false>), grid, dim3(256), 0, s, a, axes);
}

}  // namespace zk

using namespace zk;

extern "C" int zk_rope_axes(const zk_axes_desc* D, const void* q, const void* k, void* q_out,
                            void* k_out, const float* cos, const float* sin,
                            const int64_t* positions, const unsigned char* pair_axes,
                            zk_stream_t stream) {
  const char* who = "zk_rope_axes";
  ZK_REQUIRE(D != nullptr, ZK_EINVAL, "%s: null descriptor", who);
  ZK_REQUIRE(valid_dtype(D->dtype), ZK_EDTYPE, "%s: bad dtype %d", who, D->dtype);
  ZK_REQUIRE(D->pairing == ZK_ROPE_HALF || D->pairing == ZK_ROPE_INTERLEAVED, ZK_EINVAL,
             "%s: bad pairing %d", who, D->pairing);
  ZK_REQUIRE(D->B >= 0 && D->S >= 0 && D->Hq > 0 && D->Hkv >= 0 && D->Hq + D->Hkv < 65536, ZK_EINVAL,
             "%s: bad shape", who);
  ZK_REQUIRE(D->S == 0 || D->B < (int64_t(1) << 31) / D->S, ZK_EINVAL, "%s: 2^31 tokens and more", who);
  ZK_REQUIRE(D->d > 0 && D->d % 2 == 0 && D->d <= 2 * kMaxPairs, ZK_EUNSUPPORTED,
             "%s: head dims are even and up to %d (got %lld)", who, 2 * kMaxPairs, (long long)D->d);
  ZK_REQUIRE(D->n_axes > 0 && D->n_axes <= 256 && D->n_pos > 0, ZK_EINVAL,
             "%s: %lld axes (1 .. 256), tables of %lld positions", who, (long long)D->n_axes,
             (long long)D->n_pos);
  ZK_REQUIRE(pair_axes != nullptr, ZK_EINVAL, "%s: null pointer", who);
  PairAxes axes = {};
  for (int64_t i = 0; i < D->d / 2; ++i) {
    ZK_REQUIRE(pair_axes[i] < D->n_axes, ZK_EINVAL, "%s: pair %lld has axis %d of %lld", who,
               (long long)i, pair_axes[i], (long long)D->n_axes);
    axes.axis[i] = pair_axes[i];
  }
  if (D->B == 0 || D->S == 0) return ZK_OK;
  ZK_REQUIRE(q && q_out && cos && sin && positions && (D->Hkv == 0 || (k && k_out)), ZK_EINVAL,
             "%s: null pointer", who);
  const int e = dtype_bytes(D->dtype);
  ZK_REQUIRE(aligned(q, e) && aligned(q_out, e) && aligned(k, e) && aligned(k_out, e) && aligned(cos, 4) &&
                 aligned(sin, 4) && aligned(positions, 8),
             ZK_EALIGN, "%s: tensors must be aligned to their elements", who);
  AxesArgs a = {};
  a.q = q; a.k = k; a.qo = q_out; a.ko = k_out;
  a.q_sb = D->q_sb; a.q_ss = D->q_ss; a.q_sh = D->q_sh;
  a.k_sb = D->k_sb; a.k_ss = D->k_ss; a.k_sh = D->k_sh;
  a.qo_sb = D->oq_sb; a.qo_ss = D->oq_ss; a.qo_sh = D->oq_sh;
  a.ko_sb = D->ok_sb; a.ko_ss = D->ok_ss; a.ko_sh = D->ok_sh;
  a.cos = cos; a.sin = sin; a.positions = positions;
  a.tokens = D->B * D->S; a.S = D->S; a.n_pos = D->n_pos;
  a.Hq = static_cast<int>(D->Hq); a.H = static_cast<int>(D->Hq + D->Hkv);
  a.half = static_cast<int>(D->d / 2);
  a.sign = D->inverse ? -1.f : 1.f;
  // pairs of a thread: as many as 16 bytes hold, fewer where a row's address or
  // the number of pairs is no multiple of that
  int v = 16 / e;
  const int64_t strides[] = {a.q_sb, a.q_ss, a.q_sh, a.qo_sb, a.qo_ss, a.qo_sh};
  const int64_t kstrides[] = {a.k_sb, a.k_ss, a.k_sh, a.ko_sb, a.ko_ss, a.ko_sh};
  auto fits = [&](int n) {
    bool ok = a.half % n == 0 && aligned(q, n * e) && aligned(q_out, n * e);
    for (int64_t s : strides) ok = ok && s % n == 0;
    if (D->Hkv > 0) {
      ok = ok && aligned(k, n * e) && aligned(k_out, n * e);
      for (int64_t s : kstrides) ok = ok && s % n == 0;
    }
    return ok;
  };
  while (v > 1 && !fits(v)) v /= 2;
  hipStream_t s = as_stream(stream);
  const bool inter = D->pairing == ZK_ROPE_INTERLEAVED;
#define ZK_AXES(T)                                        \
  do {                                                    \
    if (v == 4) launch_rope_axes<T, 4>(a, axes, inter, s); \
    else if (v == 2) launch_rope_axes<T, 2>(a, axes, inter, s); \
    else launch_rope_axes<T, 1>(a, axes, inter, s);       \
  } while (0)
  if (D->dtype == ZK_F32) {
    ZK_AXES(float);
  } else if (D->dtype == ZK_BF16) {
    if (v == 8) launch_rope_axes<bf16, 8>(a, axes, inter, s); else ZK_AXES(bf16);
  } else {
    if (v == 8) launch_rope_axes<f16, 8>(a, axes, inter, s); else ZK_AXES(f16);
  }
#undef ZK_AXES
  return launch_status(who);
}
