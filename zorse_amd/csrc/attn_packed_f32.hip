// Attention over packed sequences for fp32 layers, on the fp32 matrix cores (the
// operands' lanes are those of attn_f32.hip), with the ranges of attn_packed.h.  A wave
// owns 16 rows and meets the other side in LDS tiles.  Two shapes:
//  * Whole: 64 rows a workgroup, 4 waves, each meets whole tiles of 32 rows.
//  * Split: 32 rows, 8 waves; the four waves of 16 rows take 16 rows each of tiles of
//    64, and their partial sums are joined through LDS at the end.
//   Bound by the matrix instructions (a 16 x 16 x 4 product takes its SIMD 32 cycles)
// in launches that fill the chip; where a launch has few workgroups, by the chain of each
// tile (loads, LDS, two barriers, products, exponentials) in the one with the most tiles,
// of which Split does a quarter at a time (1111 tokens in texts of up to 385, 8 heads of
// 64: the matrix units are busy 8 - 13 % of the time).  So Split up to two of Whole's workgroups a CU
// (head dim 64, causal, forward and backward in us, Whole against Split: 1024 tokens,
// 8 heads 78 + 357 against 42 + 153 (one sum a key head); 2048, 16 heads 180 + 526 against 135 + 414, but in
// sequences of 200 31 + 86 against 31 + 104), Whole past it (4096 tokens, 16 heads of
// 128: 811 + 2570, 67 - 85 TFLOP/s of the 157 that the matrix cores have in fp32;
// Split 991 + 2970).  A key head's query heads go to several workgroups as for the
// 2-byte types (1024 tokens, 8 heads of 4: 153 us backward, 110 with two sums).
//   Products and sums are fp32; a tile that holds an infinity or a NaN is added row by
// row, masked rows left out.
#include "attn_f32.h"
#include "attn_packed.h"

namespace zk {

namespace {

// SETS sets of 16 rows, SLICES waves to each, PIECES times 16 rows of a tile a wave.
template <int SETS, int SLICES, int PIECES>
struct Shape {
  static constexpr int sets = SETS, slices = SLICES, pieces = PIECES;
  static constexpr int rows = 16 * SETS, tile = 16 * SLICES * PIECES, threads = 64 * SETS * SLICES;
};
typedef Shape<4, 1, 2> Whole;
typedef Shape<2, 4, 1> Split;

// Sums acc over the waves of a row set; a wave is left with its share of the columns,
// N times 16 from N times its slice on.
// `lds`: two tiles of rows of D + 4 floats that no wave reads any more.
template <typename G, int D, int N = D / 16 / G::slices>
__device__ __forceinline__ void join(f32x4 (&sum)[N], const f32x4 (&acc)[D / 16], float* lds, int set,
                                     int slice) {
  constexpr int SLICE = G::sets * (D / 16) * 64;
  static_assert(G::slices == 1 || G::threads * (D / 4) <= 2 * G::tile * (D + 4),
                "the sums do not fit in the tiles");
  if constexpr (G::slices == 1) {
#pragma unroll
    for (int nt = 0; nt < N; ++nt) sum[nt] = acc[nt];
  } else {
    f32x4* const all = reinterpret_cast<f32x4*>(lds) + set * (D / 16) * 64 + (threadIdx.x & 63);
#pragma unroll
    for (int nt = 0; nt < D / 16; ++nt) all[slice * SLICE + nt * 64] = acc[nt];
    __syncthreads();
#pragma unroll
    for (int j = 0; j < N; ++j) {
      f32x4 x = all[(slice * N + j) * 64];
#pragma unroll
      for (int i = 1; i < G::slices; ++i) x += all[i * SLICE + (slice * N + j) * 64];
      sum[j] = x;
    }
  }
}

// The workgroup's block and head; whether there is such a block.
template <typename G, bool kKeys>
__device__ __forceinline__ bool block_of(const PackedArgs& a, const PackedPlan& plan, int& r0, int& h) {
  const int64_t bid = group_id();
  const int H = kKeys ? a.Hkv * a.parts : a.Hq;  // h of a key block: part Hkv + head
  if (bid >= packed_blocks(a.T, G::rows) * H) return false;
  h = static_cast<int>(bid % H);
  r0 = plan.first_row<G::rows, kKeys>(a, static_cast<int>(bid / H));
  return r0 < a.T;
}

// Tokens [lo, hi) that rows r0 .. r0 + G::rows - 1 meet.
template <typename G, bool kKeys>
__device__ __forceinline__ void tokens_of(const PackedArgs& a, const PackedPlan& plan, int r0, int& lo,
                                          int& hi) {
  const int past = r0 + G::rows < a.T ? r0 + G::rows : static_cast<int>(a.T);
  lo = kKeys ? plan.query_lo(a, r0) : plan.key_lo(a, r0);
  hi = (kKeys ? plan.query_hi(a, past - 1) : plan.key_hi(a, past - 1)) + 1;
  if (hi > plan.n) hi = plan.n;
}

template <typename G, int D, bool kVec>
__global__ __launch_bounds__(G::threads, D > 64 ? 2 : G::slices > 1 ? 4 : 3) void packed_fwd_f32(PackedArgs a) {
  __shared__ __attribute__((aligned(16))) float tiles[2 * G::tile * (D + 4)];
  float *const Ks = tiles, *const Vs = tiles + G::tile * (D + 4);
  __shared__ float ms[G::slices][G::rows], ls[G::slices][G::rows];
  const int lane = threadIdx.x & 63, set = (threadIdx.x >> 6) % G::sets, l16 = lane & 15, q4 = lane >> 4;
  const int slice = threadIdx.x / (64 * G::sets), at = 16 * G::pieces * slice;
  const PackedPlan plan(a);
  int q0, hq;
  if (!block_of<G, false>(a, plan, q0, hq)) return;
  const int hk = hq / (a.Hq / a.Hkv), my_q = q0 + 16 * set + l16, d = a.d;
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
  tokens_of<G, false>(a, plan, q0, lo, hi);
  TileReg<D, kVec, G::tile, G::threads> kr, vr;
  if (lo < hi) {
    kr.load(K, a.k_s, lo, plan.n, d);
    vr.load(V, a.v_s, lo, plan.n, d);
  }
  for (int k0 = lo; k0 < hi; k0 += G::tile) {
    __syncthreads();  // the previous tile's reads are done
    kr.store(Ks);
    const bool odd = __syncthreads_or(vr.store(Vs));
    auto visible = [&](int r) __attribute__((always_inline)) {
      return k0 + r >= my_lo && k0 + r <= my_hi;
    };
    if (k0 + G::tile < hi) {
      kr.load(K, a.k_s, k0 + G::tile, plan.n, d);
      vr.load(V, a.v_s, k0 + G::tile, plan.n, d);
    }
    if (!__any(my_lo < k0 + at + 16 * G::pieces && my_hi >= k0 + at)) continue;
    f32x4 s[G::pieces];
    float mloc = -INFINITY;
#pragma unroll
    for (int h = 0; h < G::pieces; ++h) {
      s[h] = dot_rows<D>(Ks, at + 16 * h, q);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[h][e] = visible(at + 16 * h + 4 * q4 + e) ? s[h][e] * a.scale : -INFINITY;
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
    for (int h = 0; h < G::pieces; ++h) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[h][e] = expf(s[h][e] - ref);
        l += s[h][e];
      }
      if (odd)
        add_rows_visible<D>(o, Vs, at + 16 * h, s[h], visible);
      else
        add_rows<D>(o, Vs, at + 16 * h, s[h]);
    }
  }
  l = group_sum(l);
  if constexpr (G::slices > 1) {  // the row's maximum and sum over the slices
    if (q4 == 0) {
      ms[slice][16 * set + l16] = m;
      ls[slice][16 * set + l16] = l;
    }
    __syncthreads();
    const float mine = m;
#pragma unroll
    for (int i = 0; i < G::slices; ++i) m = fmaxf(m, ms[i][16 * set + l16]);
    const float ref = m == -INFINITY ? 0.f : m, alpha = expf(mine - ref);
    l = 0.f;
#pragma unroll
    for (int i = 0; i < G::slices; ++i) l += ls[i][16 * set + l16] * expf(ms[i][16 * set + l16] - ref);
#pragma unroll
    for (int nt = 0; nt < D / 16; ++nt) o[nt] *= alpha;
  }
  f32x4 out[D / 16 / G::slices];
  join<G, D>(out, o, tiles, set, slice);
  if (!in || (my_q >= plan.n && a.keep_tail)) return;
  const bool any_key = my_hi >= my_lo;
  // no weight although keys are visible: every score is -inf or NaN, and so is O
  store_row<D, kVec>(static_cast<float*>(a.out) + hq * a.o_h + my_q * a.o_s, out,
                     l > 0.f ? 1.0f / l : any_key ? NAN : 0.f, d, slice * (D / 16 / G::slices));
  if (slice == 0 && q4 == 0)
    a.lse_out[static_cast<int64_t>(hq) * a.T + my_q] = l > 0.f ? m + logf(l) : any_key ? NAN : -INFINITY;
}

// dQ, and delta = rowsum(dO o O) and the LSE for the dK / dV kernel that follows.
template <typename G, int D, bool kVec>
__global__ __launch_bounds__(G::threads, D > 64 || G::slices > 1 ? 2 : 3) void packed_dq_f32(PackedArgs a) {
  __shared__ __attribute__((aligned(16))) float tiles[2 * G::tile * (D + 4)];
  float *const Ks = tiles, *const Vs = tiles + G::tile * (D + 4);
  const int lane = threadIdx.x & 63, set = (threadIdx.x >> 6) % G::sets, l16 = lane & 15, q4 = lane >> 4;
  const int slice = threadIdx.x / (64 * G::sets), at = 16 * G::pieces * slice;
  const PackedPlan plan(a);
  int q0, hq;
  if (!block_of<G, false>(a, plan, q0, hq)) return;
  const int hk = hq / (a.Hq / a.Hkv), my_q = q0 + 16 * set + l16, d = a.d;
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
      if (slice == 0 && q4 == 0) {
        a.delta[i] = del;
        a.lse2[i] = lse;
      }
    }
  }
  f32x4 dq[D / 16];
#pragma unroll
  for (int nt = 0; nt < D / 16; ++nt) dq[nt] = f32x4{};
  int lo, hi;
  tokens_of<G, false>(a, plan, q0, lo, hi);
  TileReg<D, kVec, G::tile, G::threads> kr, vr;
  if (lo < hi) {
    kr.load(K, a.k_s, lo, plan.n, d);
    vr.load(V, a.v_s, lo, plan.n, d);
  }
  for (int k0 = lo; k0 < hi; k0 += G::tile) {
    __syncthreads();
    vr.store(Vs);
    const bool odd = __syncthreads_or(kr.store(Ks));
    auto visible = [&](int r) __attribute__((always_inline)) {
      return k0 + r >= my_lo && k0 + r <= my_hi;
    };
    if (k0 + G::tile < hi) {
      kr.load(K, a.k_s, k0 + G::tile, plan.n, d);
      vr.load(V, a.v_s, k0 + G::tile, plan.n, d);
    }
    if (!__any(my_lo < k0 + at + 16 * G::pieces && my_hi >= k0 + at)) continue;
#pragma unroll
    for (int r = at; r < at + 16 * G::pieces; r += 16) {
      f32x4 s = dot_rows<D>(Ks, r, q);
      const f32x4 dp = dot_rows<D>(Vs, r, g);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        s[e] = visible(r + 4 * q4 + e) ? expf(s[e] * a.scale - lse) * (dp[e] - del) : 0.f;
      if (odd)
        add_rows_visible<D>(dq, Ks, r, s, visible);
      else
        add_rows<D>(dq, Ks, r, s);
    }
  }
  f32x4 out[D / 16 / G::slices];
  if (G::slices > 1) __syncthreads();
  join<G, D>(out, dq, tiles, set, slice);
  if (in && (my_q < plan.n || !a.keep_tail))
    store_row<D, kVec>(static_cast<float*>(a.dq) + hq * a.dq_h + my_q * a.dq_s, out, a.scale, d,
                       slice * (D / 16 / G::slices));
}

// dK and dV of a block of keys, summed over the query heads of the group.
template <typename G, int D, bool kVec>
__global__ __launch_bounds__(G::threads, D > 64 || G::slices > 1 ? 2 : 3) void packed_dkdv_f32(PackedArgs a) {
  __shared__ __attribute__((aligned(16))) float tiles[2 * G::tile * (D + 4)];
  float *const Qs = tiles, *const Gs = tiles + G::tile * (D + 4);
  __shared__ __attribute__((aligned(16))) float ls[G::tile], ds[G::tile];
  const int lane = threadIdx.x & 63, set = (threadIdx.x >> 6) % G::sets, l16 = lane & 15, q4 = lane >> 4;
  const int slice = threadIdx.x / (64 * G::sets), at = 16 * G::pieces * slice;
  const PackedPlan plan(a);
  int k0, in_block;
  if (!block_of<G, true>(a, plan, k0, in_block)) return;
  const int hk = in_block % a.Hkv, part = in_block / a.Hkv;
  // this part's query heads
  const int n_rep = a.Hq / a.Hkv / a.parts, h_first = (hk * a.parts + part) * n_rep;
  const int my_k = k0 + 16 * set + l16, d = a.d;
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
  tokens_of<G, true>(a, plan, k0, lo, hi);
  const int nt = hi > lo ? (hi - lo + G::tile - 1) / G::tile : 0, n_it = nt * n_rep;
  TileReg<D, kVec, G::tile, G::threads> qr, gr;
  float lr = 0.f, dr = 0.f;
  auto load = [&](int it) __attribute__((always_inline)) {
    const int hq = h_first + it / nt, r0 = lo + it % nt * G::tile;
    qr.load(static_cast<const float*>(a.q) + hq * a.q_h, a.q_s, r0, plan.n, d);
    gr.load(static_cast<const float*>(a.dout) + hq * a.do_h, a.do_s, r0, plan.n, d);
    if (threadIdx.x < G::tile) {
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
    if (threadIdx.x < G::tile) {
      ls[threadIdx.x] = lr;
      ds[threadIdx.x] = dr;
    }
    const bool odd = __syncthreads_or(odd_q | odd_g);
    if (it + 1 < n_it) load(it + 1);
    const int r0 = lo + it % nt * G::tile;
    auto visible = [&](int r) __attribute__((always_inline)) {
      return r0 + r >= my_lo && r0 + r <= my_hi;
    };
    if (!__any(my_lo < r0 + at + 16 * G::pieces && my_hi >= r0 + at)) continue;
#pragma unroll
    for (int row = at; row < at + 16 * G::pieces; row += 16) {
      const f32x4 s = dot_rows<D>(Qs, row, k);
      const f32x4 dp = dot_rows<D>(Gs, row, v);
      f32x4 p, w;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = row + 4 * q4 + e;
        const bool vis = visible(r);
        p[e] = vis ? expf(s[e] * a.scale - ls[r]) : 0.f;
        w[e] = vis ? p[e] * (dp[e] - ds[r]) : 0.f;
      }
      if (odd) {
        add_rows_visible<D>(dv, Gs, row, p, visible);
        add_rows_visible<D>(dk, Qs, row, w, visible);
      } else {
        add_rows<D>(dv, Gs, row, p);
        add_rows<D>(dk, Qs, row, w);
      }
    }
  }
  f32x4 dk_sum[D / 16 / G::slices], dv_sum[D / 16 / G::slices];
  if (G::slices > 1) __syncthreads();
  join<G, D>(dk_sum, dk, tiles, set, slice);
  if (G::slices > 1) __syncthreads();
  join<G, D>(dv_sum, dv, tiles, set, slice);
  const bool whole = a.parts == 1;
  if (!in || (my_k >= plan.n && (a.keep_tail || !whole))) return;
  const int64_t at_part = ((static_cast<int64_t>(part) * a.T + my_k) * a.Hkv + hk) * d;
  float* dkp = whole ? static_cast<float*>(a.dk) + hk * a.dk_h + my_k * a.dk_s : a.dk_part + at_part;
  float* dvp = whole ? static_cast<float*>(a.dv) + hk * a.dv_h + my_k * a.dv_s : a.dv_part + at_part;
  store_row<D, kVec>(dkp, dk_sum, a.scale, d, slice * (D / 16 / G::slices));
  store_row<D, kVec>(dvp, dv_sum, 1.f, d, slice * (D / 16 / G::slices));
}

#define ZK_PACKED_F32_OF(KERNEL, G, HEADS)                                                \
  do {                                                                                    \
    const dim3 grid = group_grid(packed_blocks(a.T, G::rows) * (HEADS)), block(G::threads); \
    if (a.d <= 64 && vec)                                                                 \
      hipLaunchKernelGGL((KERNEL<G, 64, true>), grid, block, 0, s, a);                    \
    else if (a.d <= 64)                                                                   \
      hipLaunchKernelGGL((KERNEL<G, 64, false>), grid, block, 0, s, a);                   \
    else if (vec)                                                                         \
      hipLaunchKernelGGL((KERNEL<G, 128, true>), grid, block, 0, s, a);                   \
    else                                                                                  \
      hipLaunchKernelGGL((KERNEL<G, 128, false>), grid, block, 0, s, a);                  \
  } while (0)
#define ZK_PACKED_F32(KERNEL, HEADS)                                                      \
  do {                                                                                    \
    if (packed_blocks(a.T, Whole::rows) * (HEADS) <= 2 * device_cus())                    \
      ZK_PACKED_F32_OF(KERNEL, Split, HEADS);                                             \
    else                                                                                  \
      ZK_PACKED_F32_OF(KERNEL, Whole, HEADS);                                             \
  } while (0)

}  // namespace

void launch_packed_fwd_f32(const PackedArgs& a, hipStream_t s) {
  const bool vec = vec4_ok(a.d, {a.q_s, a.q_h, a.k_s, a.k_h, a.v_s, a.v_h, a.o_s, a.o_h},
                           {a.q, a.k, a.v, a.out});
  ZK_PACKED_F32(packed_fwd_f32, a.Hq);
}

void launch_packed_bwd_f32(const PackedArgs& a, hipStream_t s) {
  const bool vec = vec4_ok(a.d, {a.q_s, a.q_h, a.k_s, a.k_h, a.v_s, a.v_h, a.o_s, a.o_h, a.do_s, a.do_h,
                                 a.dq_s, a.dq_h, a.dk_s, a.dk_h, a.dv_s, a.dv_h},
                           {a.q, a.k, a.v, a.o, a.dout, a.dq, a.dk, a.dv});
  ZK_PACKED_F32(packed_dq_f32, a.Hq);
  ZK_PACKED_F32(packed_dkdv_f32, a.Hkv * a.parts);
}

}  // namespace zk
