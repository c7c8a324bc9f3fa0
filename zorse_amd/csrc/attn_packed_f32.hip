// Attention over packed sequences for fp32 layers, on the fp32 matrix cores; the
// arrangement is that of attn_f32.hip with the ranges of attn_packed.h.  4 waves of
// 16 rows, 32-row tiles of the other side.  Products and sums are fp32; a tile that
// holds an infinity or a NaN is added row by row, masked rows left out.
#include "attn_f32.h"
#include "attn_packed.h"

namespace zk {

namespace {

constexpr int kRows = 64;  // rows per workgroup

// The workgroup's block and head; whether there is such a block.
template <bool kKeys>
__device__ __forceinline__ bool block_of(const PackedArgs& a, const PackedPlan& plan, int& r0, int& h) {
  const int64_t bid = group_id();
  const int H = kKeys ? a.Hkv : a.Hq;
  if (bid >= packed_blocks(a.T, kRows) * H) return false;
  h = static_cast<int>(bid % H);
  r0 = plan.first_row<kRows, kKeys>(a, static_cast<int>(bid / H));
  return r0 < a.T;
}

// Tokens [lo, hi) that rows r0 .. r0 + kRows - 1 meet.
template <bool kKeys>
__device__ __forceinline__ void tokens_of(const PackedArgs& a, const PackedPlan& plan, int r0, int& lo,
                                          int& hi) {
  const int past = r0 + kRows < a.T ? r0 + kRows : static_cast<int>(a.T);
  lo = kKeys ? plan.query_lo(a, r0) : plan.key_lo(a, r0);
  hi = (kKeys ? plan.query_hi(a, past - 1) : plan.key_hi(a, past - 1)) + 1;
  if (hi > plan.n) hi = plan.n;
}

template <int D, bool kVec>
__global__ __launch_bounds__(256) void packed_fwd_f32(PackedArgs a) {
  __shared__ __attribute__((aligned(16))) float Ks[kTile * (D + 4)], Vs[kTile * (D + 4)];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l16 = lane & 15, q4 = lane >> 4;
  const PackedPlan plan(a);
  int q0, hq;
  if (!block_of<false>(a, plan, q0, hq)) return;
  const int hk = hq / (a.Hq / a.Hkv), my_q = q0 + 16 * wave + l16, d = a.d;
  const bool in = my_q < a.T;
  const float* K = static_cast<const float*>(a.k) + hk * a.k_h;
  const float* V = static_cast<const float*>(a.v) + hk * a.v_h;
  const int my_lo = in ? plan.key_lo(a, my_q) : 1, my_hi = in ? plan.key_hi(a, my_q) : 0;
  float4 q[D / 16];
  load_row<D, kVec>(q, in ? static_cast<const float*>(a.q) + hq * a.q_h + my_q * a.q_s : nullptr, d);
  f32x4 o[D / 16];
#pragma unroll
  for (int nt = 0; nt < D / 16; ++nt) o[nt] = f32x4{};
  float m = -INFINITY, l = 0.f;
  int lo, hi;
  tokens_of<false>(a, plan, q0, lo, hi);
  TileReg<D, kVec> kr, vr;
  if (lo < hi) {
    kr.load(K, a.k_s, lo, plan.n, d);
    vr.load(V, a.v_s, lo, plan.n, d);
  }
  for (int k0 = lo; k0 < hi; k0 += kTile) {
    __syncthreads();  // the previous tile's reads are done
    kr.store(Ks);
    const bool odd = __syncthreads_or(vr.store(Vs));
    auto visible = [&](int r) __attribute__((always_inline)) {
      return k0 + r >= my_lo && k0 + r <= my_hi;
    };
    if (k0 + kTile < hi) {
      kr.load(K, a.k_s, k0 + kTile, plan.n, d);
      vr.load(V, a.v_s, k0 + kTile, plan.n, d);
    }
    f32x4 s[2];
    float mloc = -INFINITY;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      s[h] = dot_rows<D>(Ks, 16 * h, q);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[h][e] = visible(16 * h + 4 * q4 + e) ? s[h][e] * a.scale : -INFINITY;
        mloc = fmaxf(mloc, s[h][e]);
      }
    }
    const float m_new = fmaxf(m, group_max(mloc));
    const float ref = m_new == -INFINITY ? 0.f : m_new;  // nothing visible yet
    const float alpha = expf(m - ref);
    m = m_new;
    l *= alpha;
#pragma unroll
    for (int nt = 0; nt < D / 16; ++nt) o[nt] *= alpha;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[h][e] = expf(s[h][e] - ref);
        l += s[h][e];
      }
      if (odd)
        add_rows_visible<D>(o, Vs, 16 * h, s[h], visible);
      else
        add_rows<D>(o, Vs, 16 * h, s[h]);
    }
  }
  l = group_sum(l);
  if (!in || (my_q >= plan.n && a.keep_tail)) return;
  const bool any_key = my_hi >= my_lo;
  // no weight although keys are visible: every score is -inf or NaN, and so is O
  store_row<D, kVec>(static_cast<float*>(a.out) + hq * a.o_h + my_q * a.o_s, o,
                     l > 0.f ? 1.0f / l : any_key ? NAN : 0.f, d);
  if (q4 == 0)
    a.lse_out[static_cast<int64_t>(hq) * a.T + my_q] = l > 0.f ? m + logf(l) : any_key ? NAN : -INFINITY;
}

// dQ, and delta = rowsum(dO o O) and the LSE for the dK / dV kernel that follows.
template <int D, bool kVec>
__global__ __launch_bounds__(256) void packed_dq_f32(PackedArgs a) {
  __shared__ __attribute__((aligned(16))) float Ks[kTile * (D + 4)], Vs[kTile * (D + 4)];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l16 = lane & 15, q4 = lane >> 4;
  const PackedPlan plan(a);
  int q0, hq;
  if (!block_of<false>(a, plan, q0, hq)) return;
  const int hk = hq / (a.Hq / a.Hkv), my_q = q0 + 16 * wave + l16, d = a.d;
  const bool in = my_q < a.T;
  const float* K = static_cast<const float*>(a.k) + hk * a.k_h;
  const float* V = static_cast<const float*>(a.v) + hk * a.v_h;
  const int my_lo = in ? plan.key_lo(a, my_q) : 1, my_hi = in ? plan.key_hi(a, my_q) : 0;
  float4 q[D / 16], g[D / 16];
  load_row<D, kVec>(q, in ? static_cast<const float*>(a.q) + hq * a.q_h + my_q * a.q_s : nullptr, d);
  load_row<D, kVec>(g, in ? static_cast<const float*>(a.dout) + hq * a.do_h + my_q * a.do_s : nullptr, d);
  float lse = INFINITY, del = 0.f;
  {
    float4 ov[D / 16];
    load_row<D, kVec>(ov, in ? static_cast<const float*>(a.o) + hq * a.o_h + my_q * a.o_s : nullptr, d);
#pragma unroll
    for (int c = 0; c < D / 16; ++c) {
      del = fmaf(ov[c].x, g[c].x, del);
      del = fmaf(ov[c].y, g[c].y, del);
      del = fmaf(ov[c].z, g[c].z, del);
      del = fmaf(ov[c].w, g[c].w, del);
    }
    del = group_sum(del);
    if (in) {
      const int64_t i = static_cast<int64_t>(hq) * a.T + my_q;
      lse = my_q < plan.n ? a.lse[i] : -INFINITY;
      if (q4 == 0) {
        a.delta[i] = del;
        a.lse2[i] = lse;
      }
    }
  }
  f32x4 dq[D / 16];
#pragma unroll
  for (int nt = 0; nt < D / 16; ++nt) dq[nt] = f32x4{};
  int lo, hi;
  tokens_of<false>(a, plan, q0, lo, hi);
  TileReg<D, kVec> kr, vr;
  if (lo < hi) {
    kr.load(K, a.k_s, lo, plan.n, d);
    vr.load(V, a.v_s, lo, plan.n, d);
  }
  for (int k0 = lo; k0 < hi; k0 += kTile) {
    __syncthreads();
    vr.store(Vs);
    const bool odd = __syncthreads_or(kr.store(Ks));
    auto visible = [&](int r) __attribute__((always_inline)) {
      return k0 + r >= my_lo && k0 + r <= my_hi;
    };
    if (k0 + kTile < hi) {
      kr.load(K, a.k_s, k0 + kTile, plan.n, d);
      vr.load(V, a.v_s, k0 + kTile, plan.n, d);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      f32x4 s = dot_rows<D>(Ks, 16 * h, q);
      const f32x4 dp = dot_rows<D>(Vs, 16 * h, g);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        s[e] = visible(16 * h + 4 * q4 + e) ? expf(s[e] * a.scale - lse) * (dp[e] - del) : 0.f;
      if (odd)
        add_rows_visible<D>(dq, Ks, 16 * h, s, visible);
      else
        add_rows<D>(dq, Ks, 16 * h, s);
    }
  }
  if (in && (my_q < plan.n || !a.keep_tail))
    store_row<D, kVec>(static_cast<float*>(a.dq) + hq * a.dq_h + my_q * a.dq_s, dq, a.scale, d);
}

// dK and dV of 64 keys, summed over the query heads of the group.
template <int D, bool kVec>
__global__ __launch_bounds__(256) void packed_dkdv_f32(PackedArgs a) {
  __shared__ __attribute__((aligned(16))) float Qs[kTile * (D + 4)], Gs[kTile * (D + 4)];
  __shared__ __attribute__((aligned(16))) float ls[kTile], ds[kTile];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l16 = lane & 15, q4 = lane >> 4;
  const PackedPlan plan(a);
  int k0, hk;
  if (!block_of<true>(a, plan, k0, hk)) return;
  const int n_rep = a.Hq / a.Hkv, my_k = k0 + 16 * wave + l16, d = a.d;
  const bool in = my_k < a.T;
  const int my_lo = in ? plan.query_lo(a, my_k) : 1, my_hi = in ? plan.query_hi(a, my_k) : 0;
  float4 k[D / 16], v[D / 16];
  load_row<D, kVec>(k, in ? static_cast<const float*>(a.k) + hk * a.k_h + my_k * a.k_s : nullptr, d);
  load_row<D, kVec>(v, in ? static_cast<const float*>(a.v) + hk * a.v_h + my_k * a.v_s : nullptr, d);
  f32x4 dk[D / 16], dv[D / 16];
#pragma unroll
  for (int nt = 0; nt < D / 16; ++nt) {
    dk[nt] = f32x4{};
    dv[nt] = f32x4{};
  }
  int lo, hi;
  tokens_of<true>(a, plan, k0, lo, hi);
  const int nt = hi > lo ? (hi - lo + kTile - 1) / kTile : 0, n_it = nt * n_rep;
  TileReg<D, kVec> qr, gr;
  float lr = 0.f, dr = 0.f;
  auto load = [&](int it) __attribute__((always_inline)) {
    const int hq = hk * n_rep + it / nt, r0 = lo + it % nt * kTile;
    qr.load(static_cast<const float*>(a.q) + hq * a.q_h, a.q_s, r0, plan.n, d);
    gr.load(static_cast<const float*>(a.dout) + hq * a.do_h, a.do_s, r0, plan.n, d);
    if (threadIdx.x < kTile) {
      const int qi = r0 + static_cast<int>(threadIdx.x);
      const int64_t i = static_cast<int64_t>(hq) * a.T + qi;
      lr = qi < plan.n ? a.lse2[i] : INFINITY;
      dr = qi < plan.n ? a.delta[i] : 0.f;
    }
  };
  if (n_it > 0) load(0);
  for (int it = 0; it < n_it; ++it) {
    __syncthreads();
    const int odd_q = qr.store(Qs), odd_g = gr.store(Gs);
    if (threadIdx.x < kTile) {
      ls[threadIdx.x] = lr;
      ds[threadIdx.x] = dr;
    }
    const bool odd = __syncthreads_or(odd_q | odd_g);
    if (it + 1 < n_it) load(it + 1);
    const int r0 = lo + it % nt * kTile;
    auto visible = [&](int r) __attribute__((always_inline)) {
      return r0 + r >= my_lo && r0 + r <= my_hi;
    };
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const f32x4 s = dot_rows<D>(Qs, 16 * h, k);
      const f32x4 dp = dot_rows<D>(Gs, 16 * h, v);
      f32x4 p, w;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = 16 * h + 4 * q4 + e;
        const bool vis = visible(r);
        p[e] = vis ? expf(s[e] * a.scale - ls[r]) : 0.f;
        w[e] = vis ? p[e] * (dp[e] - ds[r]) : 0.f;
      }
      if (odd) {
        add_rows_visible<D>(dv, Gs, 16 * h, p, visible);
        add_rows_visible<D>(dk, Qs, 16 * h, w, visible);
      } else {
        add_rows<D>(dv, Gs, 16 * h, p);
        add_rows<D>(dk, Qs, 16 * h, w);
      }
    }
  }
  if (!in || (my_k >= plan.n && a.keep_tail)) return;
  store_row<D, kVec>(static_cast<float*>(a.dk) + hk * a.dk_h + my_k * a.dk_s, dk, a.scale, d);
  store_row<D, kVec>(static_cast<float*>(a.dv) + hk * a.dv_h + my_k * a.dv_s, dv, 1.f, d);
}

#define ZK_PACKED_F32(KERNEL, GRID)                                              \
  do {                                                                           \
    if (a.d <= 64 && vec)                                                        \
      hipLaunchKernelGGL((KERNEL<64, true>), GRID, dim3(256), 0, s, a);          \
    else if (a.d <= 64)                                                          \
      hipLaunchKernelGGL((KERNEL<64, false>), GRID, dim3(256), 0, s, a);         \
    else if (vec)                                                                \
      hipLaunchKernelGGL((KERNEL<128, true>), GRID, dim3(256), 0, s, a);         \
    else                                                                         \
      hipLaunchKernelGGL((KERNEL<128, false>), GRID, dim3(256), 0, s, a);        \
  } while (0)

}  // namespace

void launch_packed_fwd_f32(const PackedArgs& a, hipStream_t s) {
  const bool vec = vec4_ok(a.d, {a.q_s, a.q_h, a.k_s, a.k_h, a.v_s, a.v_h, a.o_s, a.o_h},
                           {a.q, a.k, a.v, a.out});
  const dim3 grid = group_grid(packed_blocks(a.T, kRows) * a.Hq);
  ZK_PACKED_F32(packed_fwd_f32, grid);
}

void launch_packed_bwd_f32(const PackedArgs& a, hipStream_t s) {
  const bool vec = vec4_ok(a.d, {a.q_s, a.q_h, a.k_s, a.k_h, a.v_s, a.v_h, a.o_s, a.o_h, a.do_s, a.do_h,
                                 a.dq_s, a.dq_h, a.dk_s, a.dk_h, a.dv_s, a.dv_h},
                           {a.q, a.k, a.v, a.o, a.dout, a.dq, a.dk, a.dv});
  const dim3 qgrid = group_grid(packed_blocks(a.T, kRows) * a.Hq);
  const dim3 kgrid = group_grid(packed_blocks(a.T, kRows) * a.Hkv);
  ZK_PACKED_F32(packed_dq_f32, qgrid);
  ZK_PACKED_F32(packed_dkdv_f32, kgrid);
}

}  // namespace zk
