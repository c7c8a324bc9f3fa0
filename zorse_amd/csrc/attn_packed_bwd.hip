// Attention over packed sequences, backward (bf16 / fp16 storage), without
// atomics: two kernels on the caller's stream.  With P = exp(S - LSE), dP = dO V^T
// and dS = P (dP - rowsum(dO O)):  dV = P^T dO, dQ = scale dS K, dK = scale dS^T Q.
//   Bound by the matrix instructions: seven products where five are needed, because
// each kernel forms S and dP for itself (one kernel for all three would add dQ in
// fp32 with atomics, in no fixed order).  32 causal heads of 128, 8 key heads, 8192
// tokens: dQ 755 us (3 products, 1090 TFLOP/s), dK / dV 1045 (4, 1052), their sums
// 29; documents of 30 to 1209 of 4096 tokens, 32 heads: 74 and 97, where a quarter of the
// tiles' area is masked, blocks of few tiles wait for their first loads, and those of the
// longest document end last (matrix units busy 27 % of the time).  P and dS are rounded to the storage type as
// operands of the products that follow, with fp32 sums; in fp16 scaled first (kScaled).
#include <type_traits>

#include "attn_packed.h"

namespace zk {

int check_packed(const zk_packed_desc* D, const char* who, bool bwd, bool* ragged,
                 std::initializer_list<const void*> tensors);
void packed_args(PackedArgs& a, const zk_packed_desc* D, const void* plan);

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

// Stores this lane's accumulators in fp32 (rows of an even number of elements).
template <int NB, int KR>
__device__ __forceinline__ void store_partial(float* row, const f32x16 (&x)[NB], float scale, int g, int d) {
#pragma unroll
  for (int nt = 0; nt < NB; ++nt)
#pragma unroll
    for (int a2 = 0; a2 < 8; ++a2) {
      const int d0 = 32 * nt + 8 * (a2 >> 1) + 4 * g + 2 * (a2 & 1);
      if (!ragged_step<KR>(2 * nt + a2 / 4) || d0 < d)
        *reinterpret_cast<float2*>(row + d0) = make_float2(x[nt][2 * a2] * scale, x[nt][2 * a2 + 1] * scale);
    }
}

// Transposed operand of tile X for its 16-row step kk, from the lane's byte offset.
template <typename T, int D>
__device__ __forceinline__ typename Mfma<T>::vec8 tr_operand(const T* X, int off, int kk) {
  const char* base = reinterpret_cast<const char*>(X) + kk * 16 * D * 2;
  const s16x4 x0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(base + off));
  const s16x4 x1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(base + 8 * D * 2 + (off ^ 32)));
  const s16x8 w = {x0[0], x0[1], x0[2], x0[3], x1[0], x1[1], x1[2], x1[3]};
  return __builtin_bit_cast(typename Mfma<T>::vec8, w);
}

// fp16's range.  P (dP - delta) may leave it: dO may be small or large, and P is about
// 1 / T.  So fp16 operands are scaled by powers of two, which the results take out
// again (in bf16, with fp32's range, nothing is scaled):
//  * P by 2^kPShift where dK / dV round it (P is at most 1), with the LSE that dQ
//    leaves for them;
//  * dS by 2^e, where e is the row's own and follows the largest of its dS so far, as
//    the reference maximum of a softmax does: above 2^15 it moves so that this one lies
//    in [2^7, 2^8).  A dS is then off by half a step of itself, or by 2^-31 of its row's
//    largest so far.
// dO of size 1e-4, 1500 tokens: dQ off by 6e-4 of itself, 1.4e-2 without; the forward and
// both kernels at 8000 tokens, window 1024, 32 heads of 64: 378 us, 367 without.
template <typename T>
constexpr bool kScaled = std::is_same<T, f16>::value;
template <typename T>
constexpr float kPShift = kScaled<T> ? 15.f : 0.f;
constexpr float kFirstE = 60.f;  // any row's first dS moves it but for one below 2^-45

// For 16 scaled dS of a lane's row: what e moves by, 0 or less (both halves of a row
// alike; the common case, no row of the wave moves, is false).
__device__ __forceinline__ bool moved_e(const f32x16& w, float& by) {
  float m = 0.f;
#pragma unroll
  for (int j = 0; j < 16; j += 2) m = fmaxf(fmaxf(m, fabsf(w[j])), fabsf(w[j + 1]));
  if (!__any(m > 32768.f)) return false;
  m = 0.f;  // of those that are finite
#pragma unroll
  for (int j = 0; j < 16; ++j) m = fmaxf(m, fabsf(w[j]) < INFINITY ? fabsf(w[j]) : 0.f);
  m = fmaxf(m, other_half(m));
  by = m > 32768.f ? 134.f - static_cast<float>(__float_as_uint(m) >> 23) : 0.f;
  return true;
}

// Adds the second group's accumulators (waves 4 .. 7) to the first's, through four
// tiles of BYTES that no wave reads any more; whether this wave is of the first.
// (Tiles of their own, not parts of one array: for parts the compiler makes every read
// wait for all loads in flight, 10 % of the forward's time.)
template <int BYTES, int NB>
__device__ __forceinline__ bool join_groups(f32x16 (&x)[NB], void* t0, void* t1, void* t2, void* t3) {
  constexpr int EACH = BYTES / (4 * 8 * 256);  // pieces of 8 accumulators in a tile
  static_assert(4 * EACH >= 2 * NB, "the sums do not fit in the tiles");
  void* const tile[4] = {t0, t1, t2, t3};
  auto at = [&](int nt, int j) __attribute__((always_inline)) {
    const int n = 2 * nt + j / 8;
    return static_cast<float*>(tile[n / EACH]) + (n % EACH * 8 + j % 8) * 256 + (threadIdx.x & 255);
  };
  const bool first = threadIdx.x < 256;
  if (!first) {
#pragma unroll
    for (int nt = 0; nt < NB; ++nt)
#pragma unroll
      for (int j = 0; j < 16; ++j) *at(nt, j) = x[nt][j];
  }
  __syncthreads();
  if (first) {
#pragma unroll
    for (int nt = 0; nt < NB; ++nt)
#pragma unroll
      for (int j = 0; j < 16; ++j) x[nt][j] += *at(nt, j);
  }
  return first;
}

// --------------------------------------------------------------------- dQ --
// 4 waves of 32 queries, whose Q and dO rows stay in registers; 64-key tiles of
// K and V.  Also delta = rowsum(dO o O) and the log2-domain LSE for the other kernel.
// kSplit, here and below: two groups of four waves take every other tile of the same
// rows and join their sums at the end, for launches of so few blocks that they wait for
// the one with the most tiles (head dim 128, causal, both kernels: 8 heads of 4096 tokens
// 300 us, split 216; 2 of 8192 573 and 390; but 2048 tokens in sequences of 200 46 and 48).
template <typename T, int D, int KR, bool kSplit>
__global__ __launch_bounds__(kSplit ? 512 : 256, 2) void packed_dq_kernel(PackedArgs a) {
  typedef Mfma<T> M;
  typedef typename M::vec8 V8;
  constexpr int BM = 128, BN = 64, PF = 2;  // PF: operand reads in flight
  constexpr int NT = kSplit ? 512 : 256, TN = kSplit ? 2 * BN : BN;  // TN: keys of a step
  constexpr int KS = KR ? KR : D / 16, NB = (KS + 1) / 2;
  const int hd = KR ? a.d : D;
  __shared__ __attribute__((aligned(16))) T K0[TN * D], K1[TN * D], V0[TN * D], V1[TN * D];

  const int lane = threadIdx.x & 63;
  int l32 = lane & 31, g = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
  const PackedPlan plan(a);
  int block, hq;
  packed_block(a, block, hq);
  const int q0 = plan.first_row<BM, false>(a, block);
  const int rows = static_cast<int>(a.T);
  if (q0 >= rows) return;
  const int hk = hq / (a.Hq / a.Hkv);
  const int qw0 = q0 + 32 * (wave & 3);
  const int k_off = kSplit ? wave / 4 * BN : 0;  // this wave's keys in a step
  int my_q = qw0 + l32;
  bool in = my_q < rows;
  const float c2 = a.scale_log2;

  const int last = rows - 1;
  auto clip = [&](int r) __attribute__((always_inline)) { return r < last ? r : last; };
  auto below = [&](int j) __attribute__((always_inline)) { return j < plan.n ? j : plan.n - 1; };
  const int b_last = clip(q0 + BM - 1);
  const int w_first = clip(qw0), w_last = clip(qw0 + 31);
  const int kv_lo = plan.key_lo(a, q0), kv_hi = below(plan.key_hi(a, b_last)) + 1;
  const int w_lo = plan.key_lo(a, w_first), w_hi = below(plan.key_hi(a, w_last));
  const int f_lo = plan.key_lo(a, w_last), f_hi = plan.key_hi(a, w_first);
  const bool idle = qw0 >= rows;
  int vis_lo = 0x40000000, vis_span = 0;
  if (in) {
    const int lo = plan.key_lo(a, my_q), hi = plan.key_hi(a, my_q);
    if (hi >= lo) {
      vis_lo = lo;
      vis_span = hi - lo;
    }
  }

  const T* Qp = static_cast<const T*>(a.q) + hq * a.q_h;
  const T* Dp = static_cast<const T*>(a.dout) + hq * a.do_h;
  const T* Kp = static_cast<const T*>(a.k) + hk * a.k_h;
  const T* Vp = static_cast<const T*>(a.v) + hk * a.v_h;
  V8 qreg[KS], dreg[KS];
  load_operand<T, KS, KR>(qreg, in ? Qp + my_q * a.q_s : nullptr, g, hd);
  load_operand<T, KS, KR>(dreg, in ? Dp + my_q * a.do_s : nullptr, g, hd);
  float lse2 = INFINITY, del = 0.f;
  {
    const T* Op = static_cast<const T*>(a.o) + hq * a.o_h;
    V8 oreg[KS];
    load_operand<T, KS, KR>(oreg, in ? Op + my_q * a.o_s : nullptr, g, hd);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int e = 0; e < 8; ++e) del = fmaf(to_f32(oreg[ks][e]), to_f32(dreg[ks][e]), del);
    del += other_half(del);
    if (in) {
      const int64_t i = static_cast<int64_t>(hq) * a.T + my_q;
      const float l = my_q < plan.n ? a.lse[i] : -INFINITY;
      lse2 = l == -INFINITY ? INFINITY : l * kLog2e;
      if (g == 0 && k_off == 0) {
        a.delta[i] = del;
        a.lse2[i] = lse2 - kPShift<T>;
      }
    }
  }
  float e_q = kScaled<T> ? kFirstE : 0.f, lse2_e = lse2 - e_q;

  const int n_t = kv_hi > kv_lo ? (kv_hi - kv_lo + TN - 1) / TN : 0;
  PackedLoader<T, D, TN, NT> kload, vload;
  kload.init(a.k_s, hd);
  vload.init(a.v_s, hd);
  auto issue = [&](int t, int st) {
    const int k0 = kv_lo + t * TN;
    kload.issue(st ? K1 : K0, Kp, a.k_s, k0, plan.n);
    vload.issue(st ? V1 : V0, Vp, a.v_s, k0, plan.n);
  };
  const int rbase = 2 * (tile_off<D>(l32, 8 * g) + k_off * D);
  const int tbase =
      2 * (tile_off<D>(4 * g + ((lane & 15) >> 2), 16 * ((lane >> 4) & 1) + 4 * (lane & 3)) + k_off * D);

  f32x16 dq[NB];
#pragma unroll
  for (int nt = 0; nt < NB; ++nt) dq[nt] = f32x16{};

  auto step = [&](auto stage_tag, int t) {
    constexpr int st = decltype(stage_tag)::value;
    const int k0 = kv_lo + t * TN + k_off;
    wait_vmcnt<0>();
    __syncthreads();
    if (t + 1 < n_t) issue(t + 1, st ^ 1);
    if (idle || k0 > w_hi || k0 + BN <= w_lo) return;
    const bool need_mask = k0 < f_lo || k0 + BN - 1 > f_hi;
    const T* Kt = st ? K1 : K0;
    const T* Vt = st ? V1 : V0;
    int rb = rbase, tb = tbase;
    asm volatile("" : "+v"(rb), "+v"(tb));
#pragma unroll
    for (int tt = 0; tt < BN / 32; ++tt) {
      f32x16 s = f32x16{}, dp = f32x16{};
      // operands read PF steps ahead; the fences keep the reads where they are
      auto rowread = [&](const T* X, int ks) __attribute__((always_inline)) {
        const int ro = (rb ^ (ks << 5)) + tt * 32 * D * 2;
        return *reinterpret_cast<const V8*>(reinterpret_cast<const char*>(X) + ro);
      };
      V8 kq[PF], vq[PF];
#pragma unroll
      for (int i = 0; i < PF; ++i) {
        kq[i] = rowread(Kt, i);
        vq[i] = rowread(Vt, i);
      }
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        __builtin_amdgcn_sched_barrier(0);
        V8 kA = kq[ks % PF], vA = vq[ks % PF];
        if (ragged_step<KR>(ks)) {
          kA = mask_cols<T>(kA, 16 * ks + 8 * g, hd);
          vA = mask_cols<T>(vA, 16 * ks + 8 * g, hd);
        }
        if (ks + PF < KS) {
          kq[ks % PF] = rowread(Kt, ks + PF);
          vq[ks % PF] = rowread(Vt, ks + PF);
        }
        s = M::mma(kA, qreg[ks], s);
        dp = M::mma(vA, dreg[ks], dp);
      }
      __builtin_amdgcn_sched_barrier(0);
      V8 sb[2];
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const float p = __builtin_amdgcn_exp2f(fmaf(s[j], c2, -lse2_e));
        float w = p * (dp[j] - del);
        if (need_mask) {
          const int rel = k0 - vis_lo + 32 * tt + 8 * (j >> 2) + 4 * g + (j & 3);
          if (static_cast<unsigned>(rel) > static_cast<unsigned>(vis_span)) w = 0.f;
        }
        if constexpr (kScaled<T>)
          dp[j] = w;
        else
          sb[j >> 3][j & 7] = static_cast<T>(w);
      }
      if constexpr (kScaled<T>) {
        float by;
        if (moved_e(dp, by)) {
          const float f = __builtin_amdgcn_exp2f(by);
          e_q += by;
          lse2_e = lse2 - e_q;
          dp *= f;
#pragma unroll
          for (int nt = 0; nt < NB; ++nt) dq[nt] *= f;
        }
#pragma unroll
        for (int j = 0; j < 16; ++j) sb[j >> 3][j & 7] = static_cast<T>(dp[j]);
      }
      constexpr int NM = 2 * NB;
      auto trread = [&](int m) __attribute__((always_inline)) {
        return tr_operand<T, D>(Kt, tb ^ ((m % NB) << 6), 2 * tt + m / NB);
      };
      V8 tq[PF];
#pragma unroll
      for (int i = 0; i < PF; ++i) tq[i] = trread(i);
#pragma unroll
      for (int m = 0; m < NM; ++m) {
        __builtin_amdgcn_sched_barrier(0);
        const V8 w = tq[m % PF];
        if (m + PF < NM) tq[m % PF] = trread(m + PF);
        dq[m % NB] = M::mma(w, sb[m / NB], dq[m % NB]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  if (n_t > 0) issue(0, 0);
  for (int t = 0; t < n_t; t += 2) {
    step(std::integral_constant<int, 0>{}, t);
    if (t + 1 < n_t) step(std::integral_constant<int, 1>{}, t + 1);
  }

  if constexpr (kScaled<T>) {
    const float f = __builtin_amdgcn_exp2f(-e_q);
#pragma unroll
    for (int nt = 0; nt < NB; ++nt) dq[nt] *= f;
  }
  if constexpr (kSplit) {
    __syncthreads();  // every wave is past its last product
    if (!join_groups<TN * D * 2>(dq, K0, K1, V0, V1)) return;
  }
  relane(l32, g);
  my_q = qw0 + l32;
  in = my_q < rows;
  const bool put = in && (my_q < plan.n || !a.keep_tail);
  T* out = static_cast<T*>(a.dq) + hq * a.dq_h + my_q * a.dq_s;
  const bool bad = put && row_has_nan<NB, KR>(dq, g, hd);
  if (put) store_accumulators<T, NB, KR>(out, dq, a.scale, g, hd);
  if (__builtin_expect(!__any(bad), 1)) return;

  // see row_has_nan.  A masked dS is zero whatever V and K hold, so only K's own odd
  // elements are a cause.
  auto seen = [&](int j) __attribute__((always_inline)) {
    return static_cast<unsigned>(j - vis_lo) <= static_cast<unsigned>(vis_span);
  };
  auto by_all = [&](int k0) __attribute__((always_inline)) { return k0 >= f_lo && k0 + 31 <= f_hi; };
  auto sees_all = [&](int k0) __attribute__((always_inline)) { return seen(k0) && seen(k0 + 31); };
  // whether every row sees all of a tile or nothing of it
  auto whole_rows = [&](int k0) __attribute__((always_inline)) {
    return !__any(!sees_all(k0) && k0 + 31 >= vis_lo && k0 <= vis_lo + vis_span);
  };
  bool found = false;
  {
    const int t_lo = w_lo > kv_lo ? kv_lo + ((w_lo - kv_lo) & ~(BN - 1)) : kv_lo;
    int past = kv_lo + ((w_hi - kv_lo) & ~(BN - 1)) + BN;
    past = past < plan.n ? past : plan.n;
#pragma unroll 1
    for (int k0 = t_lo; k0 < past && !found; k0 += 32)
      if (!by_all(k0)) found = odd_rows<T, KS, KR>(Kp, a.k_s, k0, past, f_lo, f_hi, g, hd) != 0;
  }
  if (__builtin_expect(!found, 1)) return;
#pragma unroll 1
  for (int c0 = 0; c0 < hd; c0 += 32) {  // as in the forward
    float e = kScaled<T> ? kFirstE : 0.f;
    f32x16 acc[1] = {f32x16{}};
#pragma unroll 1
    for (int k0 = w_lo; k0 <= w_hi; k0 += 32) {
      const T* kr = k0 + l32 <= w_hi ? Kp + (k0 + l32) * a.k_s : nullptr;
      const T* vr = k0 + l32 <= w_hi ? Vp + (k0 + l32) * a.v_s : nullptr;
      f32x16 s = f32x16{}, dp = f32x16{};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        s = M::mma(operand_step<T, KR>(kr, ks, g, hd), qreg[ks], s);
        dp = M::mma(operand_step<T, KR>(vr, ks, g, hd), dreg[ks], dp);
      }
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const float w = __builtin_amdgcn_exp2f(fmaf(s[j], c2, e - lse2)) * (dp[j] - del);
        dp[j] = seen(k0 + 8 * (j >> 2) + 4 * g + (j & 3)) ? w : 0.f;
      }
      if constexpr (kScaled<T>) {
        float by;
        if (moved_e(dp, by)) {
          const float f = __builtin_amdgcn_exp2f(by);
          e += by;
          dp *= f;
          acc[0] *= f;
        }
      }
      V8 w[2];
#pragma unroll
      for (int j = 0; j < 16; ++j) w[j >> 3][j & 7] = static_cast<T>(dp[j]);
      const bool kept = whole_rows(k0);
      add_columns<T, 1>(acc, Kp, a.k_s, k0, w_hi + 1, c0, w, kept, sees_all(k0), g, hd);
      if (!kept)
        add_odd<T, 1>(acc, Kp, a.k_s, k0, odd_rows<T, KS, KR>(Kp, a.k_s, k0, w_hi + 1, 1, 0, g, hd), c0, dp,
                      seen, g, hd);
      if (!__any(bad && !all_nan<1, KR>(acc, c0, g, hd))) break;
    }
    if (bad) store_block<T>(out, acc[0], a.scale * __builtin_amdgcn_exp2f(-e), c0, g, hd);
  }
}

// ------------------------------------------------------------------ dK / dV --
// 4 waves of 32 keys (K rows in registers, V rows in LDS); 32-query blocks of
// every query head of the group, whose sums stay in the accumulators.  At a head dim
// of 64, whose blocks take half as long, two of them between barriers: the loads of the
// next ones have that time (8000 tokens, window 1024, 32 heads of 8: both kernels 345 us
// with one, 314 with two; three waves a SIMD or 128 keys a step in dQ: slower).
template <typename T, int D, int KR, bool kSplit>
__global__ __launch_bounds__(kSplit ? 512 : 256, 2) void packed_dkdv_kernel(PackedArgs a) {
  typedef Mfma<T> M;
  typedef typename M::vec8 V8;
  constexpr int BK = 128, MQ = 32;
  constexpr int NT = kSplit ? 512 : 256;
  constexpr int SUB = D == 64 ? 2 : 1, TQ = (kSplit ? 2 : 1) * SUB * MQ;  // blocks of a wave in a step; queries
  constexpr int KS = KR ? KR : D / 16, NB = (KS + 1) / 2;
  const int hd = KR ? a.d : D;
  __shared__ __attribute__((aligned(16))) T Q0[TQ * D], Q1[TQ * D], dO0[TQ * D], dO1[TQ * D];
  __shared__ __attribute__((aligned(16))) float lse2s[2][NT / 64][64];  // 64 lanes load, SUB MQ used
  __shared__ __attribute__((aligned(16))) float dels[2][NT / 64][64];
  __shared__ __attribute__((aligned(16))) T Vw[4][32 * D];

  const int lane = threadIdx.x & 63;
  int l32 = lane & 31, g = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
  const PackedPlan plan(a);
  const int block = blockIdx.x / (a.Hkv * a.parts), in_block = blockIdx.x % (a.Hkv * a.parts);
  const int hk = in_block % a.Hkv, part = in_block / a.Hkv;
  // this part's query heads
  const int n_rep = a.Hq / a.Hkv / a.parts, h_first = (hk * a.parts + part) * n_rep;
  const int k0 = plan.first_row<BK, true>(a, block);
  const int rows = static_cast<int>(a.T);
  if (k0 >= rows) return;
  const int kw0 = k0 + 32 * (wave & 3);
  const int q_off = kSplit ? wave / 4 * (SUB * MQ) : 0;  // this wave's queries in a step
  int my_key = kw0 + l32;
  bool in = my_key < rows;
  const float c2 = a.scale_log2;

  const int last = rows - 1;
  auto clip = [&](int r) __attribute__((always_inline)) { return r < last ? r : last; };
  auto below = [&](int j) __attribute__((always_inline)) { return j < plan.n ? j : plan.n - 1; };
  const int b_last = clip(k0 + BK - 1);
  const int w_first = clip(kw0), w_last = clip(kw0 + 31);
  const int q_lo = plan.query_lo(a, k0), q_hi = below(plan.query_hi(a, b_last)) + 1;
  const int w_lo = plan.query_lo(a, w_first), w_hi = below(plan.query_hi(a, w_last));
  const int f_lo = plan.query_lo(a, w_last), f_hi = plan.query_hi(a, w_first);
  const bool idle = kw0 >= rows;
  int vis_lo = 0x40000000, vis_span = 0;
  if (in) {
    const int lo = plan.query_lo(a, my_key), hi = plan.query_hi(a, my_key);
    if (hi >= lo) {
      vis_lo = lo;
      vis_span = hi - lo;
    }
  }

  const T* Kp = static_cast<const T*>(a.k) + hk * a.k_h;
  const T* Vp = static_cast<const T*>(a.v) + hk * a.v_h;
  V8 kreg[KS];
  T* Vme = Vw[wave & 3];
  load_operand<T, KS, KR>(kreg, in ? Kp + my_key * a.k_s : nullptr, g, hd);
  if (wave < 4) {  // a barrier stands before the first read
    V8 vv[KS];
    load_operand<T, KS, KR>(vv, in ? Vp + my_key * a.v_s : nullptr, g, hd);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
      *reinterpret_cast<V8*>(&Vme[tile_off<D>(l32, 16 * ks + 8 * g)]) = vv[ks];
  }

  f32x16 dk[NB], dv[NB];
#pragma unroll
  for (int nt = 0; nt < NB; ++nt) {
    dk[nt] = f32x16{};
    dv[nt] = f32x16{};
  }
  float e_k = kFirstE, f_k = __builtin_amdgcn_exp2f(kFirstE - kPShift<T>);  // e and 2^(e - kPShift)
  const int rbase = 2 * (tile_off<D>(l32, 8 * g) + q_off * D);
  const int tbase =
      2 * (tile_off<D>(4 * g + ((lane & 15) >> 2), 16 * ((lane >> 4) & 1) + 4 * (lane & 3)) + q_off * D);

  const int n_qb = q_hi > q_lo ? (q_hi - q_lo + TQ - 1) / TQ : 0;
  const int n_it = n_qb * n_rep;
  PackedLoader<T, D, TQ, NT> qload, dload;
  qload.init(a.q_s, hd);
  dload.init(a.do_s, hd);
  auto issue = [&](int qb, int hr, int st) {
    const int hq = h_first + hr;
    const int qb0 = q_lo + qb * TQ;
    qload.issue(st ? Q1 : Q0, static_cast<const T*>(a.q) + hq * a.q_h, a.q_s, qb0, plan.n);
    dload.issue(st ? dO1 : dO0, static_cast<const T*>(a.dout) + hq * a.do_h, a.do_s, qb0, plan.n);
    const int first = below(qb0 + q_off), qi = below(first + lane);
    const int64_t r0 = static_cast<int64_t>(hq) * a.T + first;
    const uint32_t off = static_cast<uint32_t>((qi - first) * 4);
    dma_lds<4>(raw_rsrc(a.lse2 + r0), off, 0, &lse2s[st][wave][0]);
    dma_lds<4>(raw_rsrc(a.delta + r0), off, 0, &dels[st][wave][0]);
  };

  auto step = [&](auto stage_tag, int qb, int nxt_qb, int nxt_hr, bool has_next) {
    constexpr int st = decltype(stage_tag)::value;
    const int qb_first = q_lo + qb * TQ + q_off;
    wait_vmcnt<0>();
    __syncthreads();
    if (has_next) issue(nxt_qb, nxt_hr, st ^ 1);
#pragma unroll
    for (int sub = 0; sub < SUB; ++sub) {
      const int qb0 = qb_first + sub * MQ;
      if (idle || qb0 > w_hi || qb0 + MQ <= w_lo) continue;
      const bool need_mask = qb0 < f_lo || qb0 + MQ - 1 > f_hi;
      const T* Qt = (st ? Q1 : Q0) + sub * MQ * D;
      const T* dOt = (st ? dO1 : dO0) + sub * MQ * D;
      const float* l2v = lse2s[st][wave] + sub * MQ;
      const float* dlv = dels[st][wave] + sub * MQ;
      int rb = rbase, tb = tbase;  // opaque: addresses derived in the step
      asm volatile("" : "+v"(rb), "+v"(tb));
      const int vb0 = kSplit ? rb - 2 * q_off * D : rb;
      f32x16 s = f32x16{}, dp = f32x16{};
      // each step's Q operand is read one step ahead
      V8 qa = *reinterpret_cast<const V8*>(reinterpret_cast<const char*>(Qt) + rb);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const int ro = rb ^ (ks << 5);
        V8 da = *reinterpret_cast<const V8*>(reinterpret_cast<const char*>(dOt) + ro);
        const V8 vb = *reinterpret_cast<const V8*>(reinterpret_cast<const char*>(Vme) + (vb0 ^ (ks << 5)));
        V8 qn = qa;
        if (ks + 1 < KS)
          qn = *reinterpret_cast<const V8*>(reinterpret_cast<const char*>(Qt) + (rb ^ ((ks + 1) << 5)));
        if (ragged_step<KR>(ks)) {
          qa = mask_cols<T>(qa, 16 * ks + 8 * g, hd);
          da = mask_cols<T>(da, 16 * ks + 8 * g, hd);
        }
        __builtin_amdgcn_sched_barrier(0);
        s = M::mma(qa, kreg[ks], s);
        dp = M::mma(da, vb, dp);
        qa = qn;
      }
      // one body with the mask in a branch of its own: two bodies, as in the
      // forward, take more registers than there are here
      if (need_mask) {
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const int rel = qb0 - vis_lo + 8 * (j >> 2) + 4 * g + (j & 3);
          s[j] = static_cast<unsigned>(rel) <= static_cast<unsigned>(vis_span) ? s[j] : -INFINITY;
        }
      }
      V8 pb[2], sb[2];
#pragma unroll
      for (int a4 = 0; a4 < 4; ++a4) {
        const int r0 = 8 * a4 + 4 * g;
        const float4 l4 = *reinterpret_cast<const float4*>(&l2v[r0]);
        const float4 d4 = *reinterpret_cast<const float4*>(&dlv[r0]);
        const float lv[4] = {l4.x, l4.y, l4.z, l4.w};
        const float dl[4] = {d4.x, d4.y, d4.z, d4.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int j = 4 * a4 + e;
          const float p = __builtin_amdgcn_exp2f(fmaf(s[j], c2, -lv[e]));
          pb[j >> 3][j & 7] = static_cast<T>(p);
          if constexpr (kScaled<T>)
            dp[j] = p * ((dp[j] - dl[e]) * f_k);
          else
            sb[j >> 3][j & 7] = static_cast<T>(p * (dp[j] - dl[e]));
        }
      }
      if constexpr (kScaled<T>) {
        float by;
        if (moved_e(dp, by)) {
          const float f = __builtin_amdgcn_exp2f(by);
          e_k += by;
          f_k *= f;
          dp *= f;
#pragma unroll
          for (int nt = 0; nt < NB; ++nt) dk[nt] *= f;
        }
#pragma unroll
        for (int j = 0; j < 16; ++j) sb[j >> 3][j & 7] = static_cast<T>(dp[j]);
      }
#pragma unroll
      for (int kk = 0; kk < 2; ++kk)
#pragma unroll
        for (int nt = 0; nt < NB; ++nt) {
          dv[nt] = M::mma(tr_operand<T, D>(dOt, tb ^ (nt << 6), kk), pb[kk], dv[nt]);
          dk[nt] = M::mma(tr_operand<T, D>(Qt, tb ^ (nt << 6), kk), sb[kk], dk[nt]);
        }
    }
  };

  int qb = 0, hr = 0;
  auto advance = [&](int& q, int& h) {
    if (++q == n_qb) {
      q = 0;
      ++h;
    }
  };
  if (n_it > 0) issue(0, 0, 0);
  for (int it = 0; it < n_it; it += 2) {
    int nq = qb, nh = hr;
    advance(nq, nh);
    step(std::integral_constant<int, 0>{}, qb, nq, nh, it + 1 < n_it);
    qb = nq;
    hr = nh;
    if (it + 1 < n_it) {
      advance(nq, nh);
      step(std::integral_constant<int, 1>{}, qb, nq, nh, it + 2 < n_it);
      qb = nq;
      hr = nh;
    }
  }

  if constexpr (kScaled<T>) {
    const float f = __builtin_amdgcn_exp2f(-e_k);
#pragma unroll
    for (int nt = 0; nt < NB; ++nt) {
      dk[nt] *= f;
      dv[nt] *= 1.f / 32768.f;  // 2^-kPShift
    }
  }
  if constexpr (kSplit) {
    __syncthreads();
    const bool first = join_groups<TQ * D * 2>(dk, Q0, Q1, dO0, dO1);
    __syncthreads();
    join_groups<TQ * D * 2>(dv, Q0, Q1, dO0, dO1);
    if (!first) return;
  }
  relane(l32, g);
  my_key = kw0 + l32;
  in = my_key < rows;
  const bool whole = a.parts == 1;
  const bool put = in && (my_key < plan.n || (whole && !a.keep_tail));
  T* dkp = static_cast<T*>(a.dk) + hk * a.dk_h + my_key * a.dk_s;
  T* dvp = static_cast<T*>(a.dv) + hk * a.dv_h + my_key * a.dv_s;
  const int64_t at_part = ((static_cast<int64_t>(part) * a.T + my_key) * a.Hkv + hk) * hd;
  const bool bad_k = put && row_has_nan<NB, KR>(dk, g, hd), bad_v = put && row_has_nan<NB, KR>(dv, g, hd);
  if (put && whole) {
    store_accumulators<T, NB, KR>(dkp, dk, a.scale, g, hd);
    store_accumulators<T, NB, KR>(dvp, dv, 1.f, g, hd);
  } else if (put) {
    store_partial<NB, KR>(a.dk_part + at_part, dk, a.scale, g, hd);
    store_partial<NB, KR>(a.dv_part + at_part, dv, 1.f, g, hd);
  }
  if (__builtin_expect(!__any(bad_k | bad_v), 1)) return;

  // see row_has_nan
  auto seen = [&](int i) __attribute__((always_inline)) {
    return static_cast<unsigned>(i - vis_lo) <= static_cast<unsigned>(vis_span);
  };
  auto by_all = [&](int i0) __attribute__((always_inline)) { return i0 >= f_lo && i0 + 31 <= f_hi; };
  auto sees_all = [&](int i0) __attribute__((always_inline)) { return seen(i0) && seen(i0 + 31); };
  // whether every row sees all of a tile or nothing of it
  auto whole_rows = [&](int i0) __attribute__((always_inline)) {
    return !__any(!sees_all(i0) && i0 + 31 >= vis_lo && i0 <= vis_lo + vis_span);
  };
  // products of 32 rows of X (those up to `top`) with an operand of the keys
  auto products = [&](f32x16& c, const T* X, int64_t ld, int i0, int top, auto&& other) __attribute__((always_inline)) {
    const T* row = i0 + l32 <= top ? X + (i0 + l32) * ld : nullptr;
    c = f32x16{};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      c = M::mma(operand_step<T, KR>(row, ks, g, hd), other(ks), c);
    }
  };
  auto k_operand = [&](int ks) __attribute__((always_inline)) { return kreg[ks]; };
  auto v_operand = [&](int ks) __attribute__((always_inline)) {
    return *reinterpret_cast<const V8*>(&Vme[tile_off<D>(l32, 16 * ks + 8 * g)]);
  };
  bool found = false;
  const int t_lo = w_lo > q_lo ? q_lo + ((w_lo - q_lo) & ~(MQ - 1)) : q_lo;
  const int t_top = below(q_lo + ((w_hi - q_lo) & ~(MQ - 1)) + MQ - 1);
#pragma unroll 1
  for (int h = h_first; h < h_first + n_rep && !found; ++h) {
    const T* Qp = static_cast<const T*>(a.q) + h * a.q_h;
    const T* Dp = static_cast<const T*>(a.dout) + h * a.do_h;
    const int64_t at = static_cast<int64_t>(h) * a.T;
#pragma unroll 1
    for (int i0 = t_lo; i0 <= t_top && !found; i0 += 32) {
      if (by_all(i0)) continue;
      f32x16 dp;
      products(dp, Dp, a.do_s, i0, t_top, v_operand);
      bool odd = false;  // a masked P or dS that is not zero
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const int i = i0 + 8 * (j >> 2) + 4 * g + (j & 3), r = i < t_top ? i : t_top;
        const float p = __builtin_amdgcn_exp2f(-INFINITY - a.lse2[at + r]);
        odd |= !seen(i) && (p != 0.f || p * (dp[j] - a.delta[at + r]) != 0.f);
      }
      found = __any(odd) || (odd_rows<T, KS, KR>(Qp, a.q_s, i0, t_top + 1, f_lo, f_hi, g, hd) |
                             odd_rows<T, KS, KR>(Dp, a.do_s, i0, t_top + 1, f_lo, f_hi, g, hd)) != 0;
    }
  }
  if (__builtin_expect(!found, 1)) return;
#pragma unroll 1
  for (int pass = 0; pass < 2; ++pass) {  // dK, then dV
    const bool second = pass == 1, bad = second ? bad_v : bad_k;
    if (!__any(bad)) continue;
    const int64_t ld = second ? a.do_s : a.q_s;
    float e = kFirstE, f_e = __builtin_amdgcn_exp2f(kFirstE - kPShift<T>);
#pragma unroll
    for (int nt = 0; nt < NB; ++nt) dk[nt] = f32x16{};
    bool open = true;
#pragma unroll 1
    for (int h = h_first; h < h_first + n_rep && open; ++h) {
      const T* Qp = static_cast<const T*>(a.q) + h * a.q_h;
      const T* Dp = static_cast<const T*>(a.dout) + h * a.do_h;
      const T* X = second ? Dp : Qp;
      const int64_t at = static_cast<int64_t>(h) * a.T;
#pragma unroll 1
      for (int i0 = w_lo; i0 <= w_hi && open; i0 += 32) {
        f32x16 s, dp;
        products(s, Qp, a.q_s, i0, w_hi, k_operand);
        products(dp, Dp, a.do_s, i0, w_hi, v_operand);
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const int i = i0 + 8 * (j >> 2) + 4 * g + (j & 3), r = i < w_hi ? i : w_hi;
          float p = __builtin_amdgcn_exp2f(fmaf(s[j], c2, -a.lse2[at + r]));
          if (!second) p *= kScaled<T> ? (dp[j] - a.delta[at + r]) * f_e : dp[j] - a.delta[at + r];
          s[j] = seen(i) ? p : 0.f;
        }
        if constexpr (kScaled<T>) {
          float by;
          if (!second && moved_e(s, by)) {
            const float f = __builtin_amdgcn_exp2f(by);
            e += by;
            f_e *= f;
            s *= f;
#pragma unroll
            for (int nt = 0; nt < NB; ++nt) dk[nt] *= f;
          }
        }
        V8 w[2];
#pragma unroll
        for (int j = 0; j < 16; ++j) w[j >> 3][j & 7] = static_cast<T>(s[j]);
        const bool kept = whole_rows(i0);
        add_columns<T, NB>(dk, X, ld, i0, w_hi + 1, 0, w, kept, sees_all(i0), g, hd);
        if (!kept)
          add_odd<T, NB>(dk, X, ld, i0, odd_rows<T, KS, KR>(X, ld, i0, w_hi + 1, 1, 0, g, hd), 0, s,
                      seen, g, hd);
        open = __any(bad && !all_nan<NB, KR>(dk, 0, g, hd));
      }
    }
    const float f = second ? __builtin_amdgcn_exp2f(-kPShift<T>)
                           : a.scale * (kScaled<T> ? __builtin_amdgcn_exp2f(-e) : 1.f);
    if (bad && whole) store_accumulators<T, NB, KR>(second ? dvp : dkp, dk, f, g, hd);
    if (bad && !whole) store_partial<NB, KR>((second ? a.dv_part : a.dk_part) + at_part, dk, f, g, hd);
  }
}

// The parts' sum, first to last, in the storage type; zeros behind the last
// sequence.  V elements a thread (2-byte heads have an even number).
template <typename T, int V>
__global__ __launch_bounds__(256) void packed_sum_kernel(PackedArgs a) {
  typedef T TV __attribute__((ext_vector_type(V)));
  typedef float FV __attribute__((ext_vector_type(V)));
  const int64_t n = a.T * a.Hkv * a.d, i = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * V;
  if (i >= n) return;
  const int e = static_cast<int>(i % a.d);
  const int64_t r = i / a.d;
  const int h = static_cast<int>(r % a.Hkv);
  const int64_t t = r / a.Hkv;
  const bool tail = t >= a.plan[0];
  if (tail && a.keep_tail) return;
  float k[V] = {}, v[V] = {};
  if (!tail)
    for (int p = 0; p < a.parts; ++p) {
      const FV x = *reinterpret_cast<const FV*>(a.dk_part + p * n + i);
      const FV y = *reinterpret_cast<const FV*>(a.dv_part + p * n + i);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        k[j] += x[j];
        v[j] += y[j];
      }
    }
  TV ks, vs;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    ks[j] = static_cast<T>(k[j]);
    vs[j] = static_cast<T>(v[j]);
  }
  *reinterpret_cast<TV*>(static_cast<T*>(a.dk) + t * a.dk_s + h * a.dk_h + e) = ks;
  *reinterpret_cast<TV*>(static_cast<T*>(a.dv) + t * a.dv_s + h * a.dv_h + e) = vs;
}
template <typename T, int V>
static void launch_packed_sum(const PackedArgs& a, hipStream_t s) {
  if (a.parts == 1) return;
  const int64_t threads = a.T * a.Hkv * a.d / V;
  hipLaunchKernelGGL((packed_sum_kernel<T, V>), dim3(static_cast<unsigned>((threads + 255) / 256)), dim3(256), 0,
                     s, a);
}

// Sums of a key head's query heads: one where its key blocks are enough to fill the
// chip and to even out their different work (a causal block's is from nothing to the
// whole sequence), else as many as make them so.  8192 causal tokens, 32 query heads
// of 8 key heads: one sum 1640 us, two 1160 us with their addition.  A window far
// below T evens blocks out itself.
static int packed_parts(int64_t T, int64_t Hq, int64_t Hkv, int64_t window) {
  const bool even = window > 0 && window < T / 4;
  const int64_t rep = Hq / Hkv, n = packed_blocks(T, 128) * Hkv, want = device_cus() * (even ? 3 : 7) / 2;
  for (int64_t p = 1; p < rep; ++p)
    if (rep % p == 0 && n * p >= want) return static_cast<int>(p);
  return static_cast<int>(rep);
}

template <typename T, int D, int KR>
static void launch_packed_bwd(const PackedArgs& a, hipStream_t s) {
  const int64_t blocks = packed_blocks(a.T, 128), nq = blocks * a.Hq, nk = blocks * a.Hkv * a.parts;
  const dim3 gq(static_cast<unsigned>(nq)), gk(static_cast<unsigned>(nk));
  if (packed_split(a, nq))
    hipLaunchKernelGGL((packed_dq_kernel<T, D, KR, true>), gq, dim3(512), 0, s, a);
  else
    hipLaunchKernelGGL((packed_dq_kernel<T, D, KR, false>), gq, dim3(256), 0, s, a);
  if (packed_split(a, nk))
    hipLaunchKernelGGL((packed_dkdv_kernel<T, D, KR, true>), gk, dim3(512), 0, s, a);
  else
    hipLaunchKernelGGL((packed_dkdv_kernel<T, D, KR, false>), gk, dim3(256), 0, s, a);
  launch_packed_sum<T, 2>(a, s);
}
template <typename T>
static void launch_packed_bwd_t(const PackedArgs& a, bool ragged, hipStream_t s) {
  if (!ragged) {
    if (a.d == 128) launch_packed_bwd<T, 128, 0>(a, s);
    else launch_packed_bwd<T, 64, 0>(a, s);
    return;
  }
  switch ((a.d + 15) / 16) {
    case 1:
    case 2: launch_packed_bwd<T, 64, 2>(a, s); break;
    case 3: launch_packed_bwd<T, 64, 3>(a, s); break;
    case 4: launch_packed_bwd<T, 64, 4>(a, s); break;
    case 5: launch_packed_bwd<T, 128, 5>(a, s); break;
    case 6: launch_packed_bwd<T, 128, 6>(a, s); break;
    case 7: launch_packed_bwd<T, 128, 7>(a, s); break;
    default: launch_packed_bwd<T, 128, 8>(a, s); break;
  }
}

}  // namespace zk

using namespace zk;

extern "C" int64_t zk_attn_packed_bwd_workspace(const zk_packed_desc* desc) {
  if (desc == nullptr || desc->T < 0 || desc->Hq <= 0 || desc->Hkv <= 0 || desc->Hq % desc->Hkv != 0)
    return 0;
  const int parts = packed_parts(desc->T, desc->Hq, desc->Hkv, desc->window);
  const int64_t sums = parts > 1 ? 2 * parts * desc->T * desc->Hkv * desc->d : 0;
  return (2 * ((desc->Hq * desc->T + 63) / 64 * 64) + sums) * 4 + 256;
}

extern "C" int zk_attn_packed_bwd(const zk_packed_desc* desc, const void* q, const void* k,
                                  const void* v, const void* plan, const void* o,
                                  const void* dout, const float* lse, void* dq, void* dk, void* dv,
                                  void* workspace, int64_t workspace_bytes, zk_stream_t stream) {
  const char* who = "zk_attn_packed_bwd";
  bool ragged;
  const int rc = check_packed(desc, who, true, &ragged, {q, k, v, o, dout, dq, dk, dv});
  if (rc != ZK_OK) return rc;
  if (desc->T == 0) return ZK_OK;
  ZK_REQUIRE(plan && lse, ZK_EINVAL, "%s: null pointer", who);
  ZK_REQUIRE(aligned(plan, 4) && aligned(lse, 4), ZK_EALIGN, "%s: plan and lse must be 4-byte aligned", who);
  const int64_t need = zk_attn_packed_bwd_workspace(desc);
  ZK_REQUIRE(workspace != nullptr && workspace_bytes >= need, ZK_EWORKSPACE,
             "%s: workspace %lld < %lld bytes", who, (long long)workspace_bytes, (long long)need);
  PackedArgs a = {};
  packed_args(a, desc, plan);
  a.q = q; a.k = k; a.v = v; a.o = o; a.dout = dout; a.lse = lse;
  a.dq = dq; a.dk = dk; a.dv = dv;
  a.delta = reinterpret_cast<float*>((reinterpret_cast<uintptr_t>(workspace) + 255) & ~uintptr_t(255));
  a.lse2 = a.delta + (desc->Hq * desc->T + 63) / 64 * 64;
  a.parts = packed_parts(desc->T, desc->Hq, desc->Hkv, desc->window);
  a.dk_part = a.lse2 + (desc->Hq * desc->T + 63) / 64 * 64;
  a.dv_part = a.dk_part + a.parts * desc->T * desc->Hkv * desc->d;
  hipStream_t s = as_stream(stream);
  if (desc->dtype == ZK_F32) {
    launch_packed_bwd_f32(a, s);
    launch_packed_sum<float, 1>(a, s);
  } else if (desc->dtype == ZK_BF16) {
    launch_packed_bwd_t<bf16>(a, ragged, s);
  } else {
    launch_packed_bwd_t<f16>(a, ragged, s);
  }
  return launch_status(who);
}
