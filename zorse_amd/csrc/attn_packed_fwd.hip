// Attention over packed sequences, forward (bf16 / fp16 storage): the plan, the
// kernel and the entry.
#include <type_traits>

#include "attn_packed.h"

namespace zk {

// ------------------------------------------------------------------- plan --
// Each token's sequence by a search among the offsets.  What the offsets hold
// is not trusted: whatever they are, start <= token < end <= n <= T.
template <typename I>
__global__ __launch_bounds__(256) void packed_rows_kernel(const I* __restrict__ offsets, int64_t n_seq,
                                                          int64_t T, int32_t* __restrict__ plan,
                                                          int64_t* __restrict__ positions) {
  const int64_t last = n_seq > 0 ? static_cast<int64_t>(offsets[n_seq]) : 0;
  const int n = static_cast<int>(last < 0 ? 0 : last > T ? T : last);
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i == 0) plan[0] = n;
  if (i >= T) return;
  int lo = static_cast<int>(i), hi = lo;
  if (i < n) {
    int64_t a = 0, b = n_seq;  // offsets[a] <= i < offsets[b], as if offsets[0] were 0
    while (b - a > 1) {
      const int64_t m = (a + b) / 2;
      if (static_cast<int64_t>(offsets[m]) <= i) a = m; else b = m;
    }
    const int64_t s = static_cast<int64_t>(offsets[a]), e = static_cast<int64_t>(offsets[b]);
    lo = static_cast<int>(s < 0 || s > i ? 0 : s);
    hi = static_cast<int>(e <= i ? i + 1 : e > n ? n : e);
  }
  plan[kPlanHeader + i] = lo;
  plan[kPlanHeader + T + i] = hi;
  if (positions != nullptr) positions[i] = i - lo;
}

// Blocks by their work, most first: a counting sort on the tokens that the
// block's last query (first key) sees under the causal mask, one workgroup.  The
// largest blocks start first, so that the launch's end is short whatever the
// lengths are.
__global__ __launch_bounds__(1024) void packed_order_kernel(int64_t T, int32_t* __restrict__ plan) {
  const int32_t* start = plan + kPlanHeader;
  const int32_t* end = start + T;
  __shared__ int hist[1024];
  int shift = 5;
  while ((T >> shift) >= 1024) ++shift;
  for (int which = 0; which < 2; ++which) {
    const int rows = kPlanRows, nb = static_cast<int>((T + rows - 1) / rows);
    int32_t* order = plan + plan_order_at(T, which);
    auto key = [&](int b) {
      const int64_t first = static_cast<int64_t>(b) * rows;
      const int64_t past = first + rows < T ? first + rows : T;
      const int64_t work = which == 0 ? past - start[first] : end[past - 1] - first;
      const int bin = static_cast<int>((work < 0 ? 0 : work) >> shift);
      return 1023 - (bin < 1024 ? bin : 1023);  // the largest in bin 0
    };
    hist[threadIdx.x] = 0;
    __syncthreads();
    for (int b = threadIdx.x; b < nb; b += 1024) atomicAdd(&hist[key(b)], 1);
    __syncthreads();
    for (int step = 1; step < 1024; step *= 2) {  // inclusive sums
      const int add = static_cast<int>(threadIdx.x) >= step ? hist[threadIdx.x - step] : 0;
      __syncthreads();
      hist[threadIdx.x] += add;
      __syncthreads();
    }
    // a bin's blocks from its end down; their order within it changes no result
    for (int b = threadIdx.x; b < nb; b += 1024) order[atomicSub(&hist[key(b)], 1) - 1] = b;
    __syncthreads();
  }
}

// ---------------------------------------------------------------- forward --
// 128 queries of one head, 32 a wave, whose Q rows stay in registers; 64-key tiles of
// K and V in LDS, row-major with swizzled 16-byte chunks.  Scores are computed
// transposed (S^T = K Q^T): a lane holds one query's scores of 32 keys, so the softmax
// is per lane with one exchange between the wave's halves, and the probabilities are
// the next product's operand as they are (O^T += V^T P^T, V^T by transposed reads).
// The reference maximum moves when a score exceeds it by 2^8 only.
//
// Four waves, so that two workgroups share a CU (four at d 64): the one's loads of Q,
// first tiles and stores lie beside the other's products.  Eight waves and 256 queries
// are 3 % faster for one sequence of 8192 tokens (505 us against 520, 32 heads of
// 128: 1060 TFLOP/s) and 37 % slower for documents of 128 tokens (41 us for 4096
// tokens against 30, where the tensors' own bytes take 27).
static constexpr float kGrowth = 8.0f;  // in the exp2 domain

// Orders the compiler's memory accesses and waits for the other waves, but not for
// this wave's loads in flight.
__device__ __forceinline__ void phase_barrier() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

// kSplit: two groups of four waves take every other tile of the same queries and join
// their sums at the end, for launches of so few blocks that they wait for the one with
// the most tiles (8 heads of 4096 causal tokens 60 us against 80).
// The groups alternate: the softmax of a tile takes a wave about as long on the vector
// units as its two products take on the matrix units, and waves that run in step do the
// same thing at the same time; so while one group multiplies (P V of its last tile and
// the scores of the next one) the other one is at its softmax, with a barrier between
// the phases.
// KR: 0 for a head dim of D and 16-byte aligned heads, else ceil(d / 16), at least 2.
template <typename T, int D, int KR, bool kSplit>
__global__ __launch_bounds__(kSplit ? 512 : 256) __attribute__((amdgpu_waves_per_eu(2)))
void packed_fwd_kernel(PackedArgs a) {
  typedef Mfma<T> M;
  typedef typename M::vec8 V8;
  constexpr int QW = 4, NW = kSplit ? 2 * QW : QW;
  constexpr int BM = 32 * QW, BN = 64, NT = 64 * NW;
  constexpr int TN = kSplit ? 2 * BN : BN;  // keys of a step
  constexpr int PF = 4;                     // operand reads in flight
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
  const int qw0 = q0 + 32 * (wave % QW);
  const int k_off = kSplit ? wave / QW * BN : 0;  // this wave's keys in a step
  int my_q = qw0 + l32;
  bool in = my_q < rows;

  // the wave's and the block's ranges of keys (scalar: their rows are uniform)
  const int last = rows - 1;
  auto clip = [&](int r) __attribute__((always_inline)) { return r < last ? r : last; };
  const int b_last = clip(q0 + BM - 1);
  const int w_first = clip(qw0), w_last = clip(qw0 + 31);
  auto below = [&](int j) __attribute__((always_inline)) { return j < plan.n ? j : plan.n - 1; };
  const int kv_lo = plan.key_lo(a, q0), kv_hi = below(plan.key_hi(a, b_last)) + 1;
  const int w_lo = plan.key_lo(a, w_first), w_hi = below(plan.key_hi(a, w_last));  // seen by any
  const int f_lo = plan.key_lo(a, w_last), f_hi = plan.key_hi(a, w_first);         // seen by all
  const bool idle = qw0 >= rows;
  int vis_lo = 0x40000000, vis_span = 0;
  bool any_key = false;
  if (in) {
    const int lo = plan.key_lo(a, my_q), hi = plan.key_hi(a, my_q);
    if (hi >= lo) {
      vis_lo = lo;
      vis_span = hi - lo;
      any_key = true;
    }
  }

  const T* Qp = static_cast<const T*>(a.q) + hq * a.q_h;
  const T* Kp = static_cast<const T*>(a.k) + hk * a.k_h;
  const T* Vp = static_cast<const T*>(a.v) + hk * a.v_h;
  V8 qreg[KS];
  load_operand<T, KS, KR>(qreg, in ? Qp + my_q * a.q_s : nullptr, g, hd);

  const int n_t = kv_hi > kv_lo ? (kv_hi - kv_lo + TN - 1) / TN : 0;
  PackedLoader<T, D, TN, NT> kload, vload;
  kload.init(a.k_s, hd);
  vload.init(a.v_s, hd);
  auto issue_k = [&](int t, int st) {
    kload.issue(st ? K1 : K0, Kp, a.k_s, kv_lo + t * TN, plan.n);
  };
  auto issue_v = [&](int t, int st) {
    vload.issue(st ? V1 : V0, Vp, a.v_s, kv_lo + t * TN, plan.n);
  };
  // LDS byte offsets from two per-lane bases (the swizzle XORs chunk indices)
  const int rbase = 2 * (tile_off<D>(l32, 8 * g) + k_off * D);
  const int tbase = 2 * (tile_off<D>(4 * g + ((lane & 15) >> 2), 16 * ((lane >> 4) & 1) + 4 * (lane & 3)) + k_off * D);

  f32x16 o[NB], s[BN / 32];
  V8 pb[BN / 16];
#pragma unroll
  for (int nt = 0; nt < NB; ++nt) o[nt] = f32x16{};
  float m_ref = -INFINITY, l_i = 0.f;
  const float c2 = a.scale_log2;

  auto skipped = [&](int t) __attribute__((always_inline)) {
    const int k0 = kv_lo + t * TN + k_off;
    return idle || t < 0 || t >= n_t || k0 > w_hi || k0 + BN <= w_lo;
  };
  // S^T = K Q^T of tile t, which starts from -inf where a key is not seen
  auto scores = [&](const T* Kt, int t) __attribute__((always_inline)) {
    int rb = rbase;  // opaque: addresses derived here
    asm volatile("" : "+v"(rb));
    const int k0 = kv_lo + t * TN + k_off;
    const bool need_mask = k0 < f_lo || k0 + BN - 1 > f_hi;
    // operands are read PF products ahead; the fences keep the reads there (left
    // alone, the compiler reads all of them first and has no registers left)
    auto rowread = [&](int i) __attribute__((always_inline)) {
      const int ks = i / (BN / 32), tt = i % (BN / 32);
      return *reinterpret_cast<const V8*>(reinterpret_cast<const char*>(Kt) + (rb ^ (ks << 5)) +
                                          tt * 32 * D * 2);
    };
    constexpr int NM = KS * (BN / 32);
    V8 kq[PF];
#pragma unroll
    for (int i = 0; i < PF; ++i) kq[i] = rowread(i);
#pragma unroll
    for (int tt = 0; tt < BN / 32; ++tt) {
      if (ragged_step<KR>(0)) kq[tt] = mask_cols<T>(kq[tt], 8 * g, hd);
    }
    // each branch with its own first products: what they leave needs no copies
    if (need_mask) {
      const int kb = k0 + 4 * g - vis_lo;
#pragma unroll
      for (int tt = 0; tt < BN / 32; ++tt) {
        f32x16 c;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const int rel = kb + 32 * tt + 8 * (j >> 2) + (j & 3);
          c[j] = static_cast<unsigned>(rel) <= static_cast<unsigned>(vis_span) ? 0.f : -INFINITY;
        }
        s[tt] = M::mma(kq[tt], qreg[0], c);
      }
    } else {
#pragma unroll
      for (int tt = 0; tt < BN / 32; ++tt) s[tt] = M::mma(kq[tt], qreg[0], f32x16{});
    }
#pragma unroll
    for (int i = 0; i < BN / 32; ++i)
      if (i + PF < NM) kq[i % PF] = rowread(i + PF);
#pragma unroll
    for (int i = BN / 32; i < NM; ++i) {
      __builtin_amdgcn_sched_barrier(0);
      const int ks = i / (BN / 32), tt = i % (BN / 32);
      V8 kv = kq[i % PF];
      if (ragged_step<KR>(ks)) kv = mask_cols<T>(kv, 16 * ks + 8 * g, hd);
      if (i + PF < NM) kq[i % PF] = rowread(i + PF);
      s[tt] = M::mma(kv, qreg[ks], s[tt]);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  // P^T from S^T, and the running maximum and sum
  auto softmax = [&]() __attribute__((always_inline)) {
    // opaque here and at the end: the vector work stays between the barriers
#pragma unroll
    for (int tt = 0; tt < BN / 32; ++tt) asm volatile("" : "+v"(s[tt]));
    float mloc = -INFINITY;
#pragma unroll
    for (int tt = 0; tt < BN / 32; ++tt)
#pragma unroll
      for (int j = 0; j < 16; j += 2) mloc = fmaxf(fmaxf(mloc, s[tt][j]), s[tt][j + 1]);
    mloc = fmaxf(mloc, other_half(mloc));
    const bool grow = (mloc - m_ref) * c2 > kGrowth;
    if (__any(grow)) {
      const float m_new = fmaxf(m_ref, mloc);
      const float alpha = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m_ref - m_new) * c2);
      m_ref = m_new;
      l_i *= alpha;
#pragma unroll
      for (int nt = 0; nt < NB; ++nt) o[nt] *= alpha;
    }
    const float mc = m_ref == -INFINITY ? 0.f : m_ref * c2;
    float lsum[4] = {};
#pragma unroll
    for (int tt = 0; tt < BN / 32; ++tt)
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const float p = __builtin_amdgcn_exp2f(fmaf(s[tt][j], c2, -mc));
        lsum[j & 3] += p;
        pb[2 * tt + (j >> 3)][j & 7] = static_cast<T>(p);
      }
    l_i += (lsum[0] + lsum[1]) + (lsum[2] + lsum[3]);
#pragma unroll
    for (int kk = 0; kk < BN / 16; ++kk) asm volatile("" : "+v"(pb[kk]));
    asm volatile("" : "+v"(l_i));
  };
  // O^T += V^T P^T (V^T read transposed from the row-major tile)
  auto weighted = [&](const T* Vt) __attribute__((always_inline)) {
    int tb = tbase;
    asm volatile("" : "+v"(tb));
    auto trread = [&](int i) __attribute__((always_inline)) {
      typedef short s16x4 __attribute__((ext_vector_type(4)));
      typedef short s16x8 __attribute__((ext_vector_type(8)));
      typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
      const char* vb = reinterpret_cast<const char*>(Vt) + i / NB * 16 * D * 2;
      const int off = tb ^ ((i % NB) << 6);
      const s16x4 x0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(vb + off));
      const s16x4 x1 =
          __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(vb + 8 * D * 2 + (off ^ 32)));
      const s16x8 w = {x0[0], x0[1], x0[2], x0[3], x1[0], x1[1], x1[2], x1[3]};
      return __builtin_bit_cast(V8, w);
    };
    constexpr int NM = BN / 16 * NB;
    V8 tq[PF];
#pragma unroll
    for (int i = 0; i < PF; ++i) tq[i] = trread(i);
#pragma unroll
    for (int i = 0; i < NM; ++i) {
      __builtin_amdgcn_sched_barrier(0);
      const V8 w = tq[i % PF];
      if (i + PF < NM) tq[i % PF] = trread(i + PF);
      o[i % NB] = M::mma(w, pb[i / NB], o[i % NB]);
    }
    __builtin_amdgcn_sched_barrier(0);
  };

  if constexpr (kSplit) {
    // Tiles outside a wave's range are not left out here: it would wait for the
    // others at the next barrier all the same, and branches around what lives from
    // one phase to the next cost registers.  par: t % 2.
    auto begin = [&](auto par, int t) __attribute__((always_inline)) {
      constexpr int p = decltype(par)::value;
      wait_vmcnt<0>();  // K of tile t and V of tile t - 1
      phase_barrier();  // ... and every wave's; all are done with what they replaced
      if (t < n_t) issue_v(t, p);
      if (t + 1 < n_t) issue_k(t + 1, p ^ 1);
    };
    auto step = [&](auto par, auto second, int t) __attribute__((always_inline)) {
      constexpr int p = decltype(par)::value;
      begin(par, t);
      if constexpr (decltype(second)::value) {
        softmax();
      } else {
        weighted(p ? V0 : V1);
        scores(p ? K1 : K0, t);
      }
      phase_barrier();
      if constexpr (decltype(second)::value) {
        weighted(p ? V0 : V1);
        scores(p ? K1 : K0, t);
      } else {
        softmax();
      }
    };
    auto end = [&](auto par, auto second) __attribute__((always_inline)) {
      constexpr int p = decltype(par)::value;
      begin(par, n_t);
      if constexpr (decltype(second)::value) softmax(); else weighted(p ? V0 : V1);
      phase_barrier();
      if constexpr (decltype(second)::value) weighted(p ? V0 : V1);
    };
    auto run = [&](auto second) __attribute__((always_inline)) {
      constexpr std::integral_constant<int, 0> even{};
      constexpr std::integral_constant<int, 1> odd{};
      begin(even, 0);
      if constexpr (!decltype(second)::value) scores(K0, 0);
      phase_barrier();
      if constexpr (decltype(second)::value) scores(K0, 0); else softmax();
      int t = 1;
      for (; t + 1 < n_t; t += 2) {
        step(odd, second, t);
        step(even, second, t + 1);
      }
      if (t < n_t) {
        step(odd, second, t);
        end(even, second);
      } else {
        end(odd, second);
      }
    };
    if (n_t > 0) {
      issue_k(0, 0);
      if (wave < QW)
        run(std::false_type{});
      else
        run(std::true_type{});
    }
  } else {
    auto step = [&](auto par, int t) __attribute__((always_inline)) {
      constexpr int p = decltype(par)::value;
      wait_vmcnt<0>();  // this wave's loads of tile t have landed
      __syncthreads();  // ... and every other wave's; all are done with the other stage
      if (t + 1 < n_t) {
        issue_k(t + 1, p ^ 1);
        issue_v(t + 1, p ^ 1);
      }
      if (skipped(t)) return;
      scores(p ? K1 : K0, t);
      softmax();
      weighted(p ? V1 : V0);
    };
    if (n_t > 0) {
      issue_k(0, 0);
      issue_v(0, 0);
    }
    for (int t = 0; t < n_t; t += 2) {
      step(std::integral_constant<int, 0>{}, t);
      if (t + 1 < n_t) step(std::integral_constant<int, 1>{}, t + 1);
    }
  }

  if constexpr (kSplit) {
    // the second group's maximum, sum and O to the first, through the tiles' memory
    const int slot = threadIdx.x & (64 * QW - 1);
    float* ml = reinterpret_cast<float*>(V0);
    auto at = [&](int nt, int j) __attribute__((always_inline)) {
      constexpr int EACH = TN * D / 2 / (16 * 64 * QW);  // accumulators that a tile has room for
      static_assert(2 * EACH >= NB, "the sums do not fit in the tiles");
      return reinterpret_cast<float*>(nt < EACH ? K0 : K1) + (nt % EACH * 16 + j) * (64 * QW) + slot;
    };
    __syncthreads();  // every wave is past its last product
    if (wave >= QW) {
      ml[slot] = m_ref;
      ml[64 * QW + slot] = l_i;
#pragma unroll
      for (int nt = 0; nt < NB; ++nt)
#pragma unroll
        for (int j = 0; j < 16; ++j) *at(nt, j) = o[nt][j];
    }
    __syncthreads();
    if (wave >= QW) return;
    const float m2 = ml[slot], m_new = fmaxf(m_ref, m2);
    const float f1 = m_ref == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m_ref - m_new) * c2);
    const float f2 = m2 == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m2 - m_new) * c2);
    m_ref = m_new;
    l_i = l_i * f1 + ml[64 * QW + slot] * f2;
#pragma unroll
    for (int nt = 0; nt < NB; ++nt)
#pragma unroll
      for (int j = 0; j < 16; ++j) o[nt][j] = o[nt][j] * f1 + *at(nt, j) * f2;
  }
  relane(l32, g);
  my_q = qw0 + l32;
  in = my_q < rows;
  const float l_tot = l_i + other_half(l_i);
  // no weight although keys are visible: every score is -inf or NaN, and so is O
  const float inv = l_tot > 0.f ? 1.0f / l_tot : any_key ? NAN : 0.f;
  const bool put = in && (my_q < plan.n || !a.keep_tail);
  T* Op = static_cast<T*>(a.out) + hq * a.o_h + my_q * a.o_s;
  float* lp = a.lse_out + static_cast<int64_t>(hq) * a.T + my_q;
  const bool bad = put && row_has_nan<NB, KR>(o, g, hd);
  if (put) {
    store_accumulators<T, NB, KR>(Op, o, inv, g, hd);
    if (g == 0) *lp = l_tot > 0.f ? m_ref * a.scale + logf(l_tot) : any_key ? NAN : -INFINITY;
  }
  if (__builtin_expect(!__any(bad), 1)) return;

  // see row_has_nan; the products of one 32-key tile
  auto raw_scores = [&](f32x16& c, int k0, int past) __attribute__((always_inline)) {
    const T* row = k0 + l32 < past ? Kp + (k0 + l32) * a.k_s : nullptr;
    c = f32x16{};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      c = M::mma(operand_step<T, KR>(row, ks, g, hd), qreg[ks], c);
    }
  };
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
    // what the wave met: whole 64-key tiles, of its own range or (kSplit) the block's
    const int t_lo = !kSplit && w_lo > kv_lo ? kv_lo + ((w_lo - kv_lo) & ~(BN - 1)) : kv_lo;
    int past = kSplit ? kv_lo + n_t * TN : kv_lo + ((w_hi - kv_lo) & ~(BN - 1)) + BN;
    past = past < plan.n ? past : plan.n;
#pragma unroll 1
    for (int k0 = t_lo; k0 < past && !found; k0 += 32) {
      if (by_all(k0)) continue;
      f32x16 c;
      raw_scores(c, k0, past);
      bool odd = false;  // a masked score that -inf does not hide
#pragma unroll
      for (int j = 0; j < 16; ++j) odd |= !seen(k0 + 8 * (j >> 2) + 4 * g + (j & 3)) && is_odd(c[j]);
      found = __any(odd) || odd_rows<T, KS, KR>(Vp, a.v_s, k0, past, f_lo, f_hi, g, hd) != 0;
    }
  }
  if (__builtin_expect(!found, 1)) return;
  const bool l_stands = l_tot == l_tot;
  // 32 columns of the result at a time: few registers, so that the loops before keep theirs
#pragma unroll 1
  for (int c0 = 0; c0 < hd; c0 += 32) {
    float m = -INFINITY, l = 0.f;
    f32x16 acc[1] = {f32x16{}};
#pragma unroll 1
    for (int k0 = w_lo; k0 <= w_hi; k0 += 32) {
      f32x16 c;
      raw_scores(c, k0, w_hi + 1);
      float mloc = -INFINITY;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        c[j] = seen(k0 + 8 * (j >> 2) + 4 * g + (j & 3)) ? c[j] : -INFINITY;
        mloc = fmaxf(mloc, c[j]);
      }
      const float m_new = fmaxf(m, fmaxf(mloc, other_half(mloc)));
      const float alpha = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m - m_new) * c2);
      const float mc = m_new == -INFINITY ? 0.f : m_new * c2;
      m = m_new;
      l *= alpha;
      acc[0] *= alpha;
      V8 w[2];
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        c[j] = __builtin_amdgcn_exp2f(fmaf(c[j], c2, -mc));
        l += c[j];
        w[j >> 3][j & 7] = static_cast<T>(c[j]);
      }
      const bool kept = whole_rows(k0);
      add_columns<T, 1>(acc, Vp, a.v_s, k0, w_hi + 1, c0, w, kept, sees_all(k0), g, hd);
      if (!kept)
        add_odd<T, 1>(acc, Vp, a.v_s, k0, odd_rows<T, KS, KR>(Vp, a.v_s, k0, w_hi + 1, 1, 0, g, hd), c0, c,
                      seen, g, hd);
      if (!__any(bad && !(all_nan<1, KR>(acc, c0, g, hd) && (l_stands || l != l)))) break;
    }
    l += other_half(l);
    if (bad) {
      store_block<T>(Op, acc[0], l > 0.f ? 1.0f / l : any_key ? NAN : 0.f, c0, g, hd);
      if (c0 == 0 && g == 0 && !l_stands) *lp = l > 0.f ? m * a.scale + logf(l) : any_key ? NAN : -INFINITY;
    }
  }
}

int check_packed(const zk_packed_desc* D, const char* who, bool bwd, bool* ragged,
                 std::initializer_list<const void*> tensors) {
  ZK_REQUIRE(D != nullptr, ZK_EINVAL, "%s: null descriptor", who);
  ZK_REQUIRE(valid_dtype(D->dtype), ZK_EDTYPE, "%s: bad dtype %d", who, D->dtype);
  ZK_REQUIRE(D->T >= 0 && D->T < (int64_t(1) << 30), ZK_EINVAL, "%s: T=%lld tokens, 0 .. 2^30 - 1",
             who, (long long)D->T);
  ZK_REQUIRE(D->Hq > 0 && D->Hkv > 0 && D->Hq < 65536 && D->Hq % D->Hkv == 0, ZK_EINVAL,
             "%s: Hq=%lld not a multiple of Hkv=%lld", who, (long long)D->Hq, (long long)D->Hkv);
  ZK_REQUIRE(D->window >= 0 && (D->causal || D->window == 0), ZK_EINVAL,
             "%s: a window (%lld) needs causal attention", who, (long long)D->window);
  ZK_REQUIRE(D->scale > 0.f && D->scale < INFINITY, ZK_EINVAL, "%s: scale must be positive", who);
  ZK_REQUIRE(D->d > 0 && D->d <= 128 && (D->dtype == ZK_F32 || D->d % 2 == 0), ZK_EUNSUPPORTED,
             "%s: head dims up to 128, even ones for 2-byte types (got %lld)", who, (long long)D->d);
  const int64_t strides[] = {D->q_s, D->q_h, D->k_s, D->k_h, D->v_s, D->v_h, D->o_s, D->o_h,
                             D->do_s, D->do_h, D->dq_s, D->dq_h, D->dk_s, D->dk_h, D->dv_s, D->dv_h};
  bool vec16 = D->d == 64 || D->d == 128, vec4 = true;
  for (int i = 0; i < (bwd ? 16 : 8); ++i) {
    vec16 = vec16 && strides[i] % 8 == 0;
    vec4 = vec4 && strides[i] % 2 == 0;
    // the tile loaders keep a tile's rows in a 32-bit byte offset
    ZK_REQUIRE(i % 2 != 0 || (strides[i] >= 0 && strides[i] < (int64_t(1) << 23)), ZK_EUNSUPPORTED,
               "%s: row stride %lld out of range", who, (long long)strides[i]);
  }
  for (const void* p : tensors) {
    ZK_REQUIRE(p != nullptr || D->T == 0, ZK_EINVAL, "%s: null pointer", who);
    vec16 = vec16 && aligned(p, 16);
    vec4 = vec4 && aligned(p, 4);
  }
  bool at4 = true;
  for (const void* p : tensors) at4 = at4 && aligned(p, 4);
  ZK_REQUIRE(D->dtype == ZK_F32 ? at4 : vec4, ZK_EALIGN, "%s: heads start at multiples of 4 bytes",
             who);
  // a launch holds fewer than 2^32 threads
  ZK_REQUIRE(D->Hq * ((D->T + 127) / 128) < int64_t(1) << 23, ZK_EUNSUPPORTED,
             "%s: %lld heads of %lld tokens: 2^30 rows or more", who, (long long)D->Hq, (long long)D->T);
  *ragged = !vec16;
  return ZK_OK;
}

void packed_args(PackedArgs& a, const zk_packed_desc* D, const void* plan) {
  a.plan = static_cast<const int32_t*>(plan);
  a.T = D->T; a.Hq = static_cast<int>(D->Hq); a.Hkv = static_cast<int>(D->Hkv); a.d = static_cast<int>(D->d);
  a.q_s = D->q_s; a.q_h = D->q_h; a.k_s = D->k_s; a.k_h = D->k_h; a.v_s = D->v_s; a.v_h = D->v_h;
  a.o_s = D->o_s; a.o_h = D->o_h; a.do_s = D->do_s; a.do_h = D->do_h;
  a.dq_s = D->dq_s; a.dq_h = D->dq_h; a.dk_s = D->dk_s; a.dk_h = D->dk_h; a.dv_s = D->dv_s; a.dv_h = D->dv_h;
  a.scale = D->scale;
  a.scale_log2 = D->scale * kLog2e;
  a.causal = D->causal != 0;
  // a window of all tokens is none
  a.window = D->window >= D->T ? 0 : static_cast<int>(D->window);
  a.keep_tail = D->keep_tail != 0;
}

}  // namespace zk

using namespace zk;

extern "C" int64_t zk_packed_plan_bytes(int64_t T) {
  if (T < 0 || T >= (int64_t(1) << 30)) {
    set_error("zk_packed_plan_bytes: T=%lld tokens, 0 .. 2^30 - 1", (long long)T);
    return ZK_EINVAL;
  }
  return 4 * plan_order_at(T, 2);
}

extern "C" int zk_packed_plan(const void* offsets, int offsets_64, int64_t n_seq, int64_t T, void* plan,
                              int64_t plan_bytes, int64_t* positions, zk_stream_t stream) {
  const char* who = "zk_packed_plan";
  ZK_REQUIRE(T >= 0 && T < (int64_t(1) << 30) && n_seq >= 0 && n_seq < (int64_t(1) << 31), ZK_EINVAL,
             "%s: T=%lld tokens (0 .. 2^30 - 1), %lld sequences", who, (long long)T, (long long)n_seq);
  ZK_REQUIRE(offsets != nullptr && plan != nullptr, ZK_EINVAL, "%s: null pointer", who);
  ZK_REQUIRE(aligned(plan, 16) && aligned(offsets, offsets_64 ? 8 : 4) && aligned(positions, 8), ZK_EALIGN,
             "%s: the plan must be 16-byte aligned, offsets and positions as their types", who);
  ZK_REQUIRE(plan_bytes >= zk_packed_plan_bytes(T), ZK_EWORKSPACE, "%s: plan %lld < %lld bytes", who,
             (long long)plan_bytes, (long long)zk_packed_plan_bytes(T));
  hipStream_t s = as_stream(stream);
  int32_t* p = static_cast<int32_t*>(plan);
  const dim3 grid(static_cast<unsigned>(T > 0 ? (T + 255) / 256 : 1));
  if (offsets_64)
    hipLaunchKernelGGL(packed_rows_kernel<int64_t>, grid, dim3(256), 0, s,
                       static_cast<const int64_t*>(offsets), n_seq, T, p, positions);
  else
    hipLaunchKernelGGL(packed_rows_kernel<int32_t>, grid, dim3(256), 0, s,
                       static_cast<const int32_t*>(offsets), n_seq, T, p, positions);
  if (T > 0) hipLaunchKernelGGL(packed_order_kernel, dim3(1), dim3(1024), 0, s, T, p);
  return launch_status(who);
}

namespace zk {
template <typename T, int D, int KR>
static void launch_packed_fwd(const PackedArgs& a, hipStream_t s) {
  const int64_t n = packed_blocks(a.T, 128) * a.Hq;
  if (packed_split(a, n))
    hipLaunchKernelGGL((packed_fwd_kernel<T, D, KR, true>), dim3(static_cast<unsigned>(n)), dim3(512), 0, s, a);
  else
    hipLaunchKernelGGL((packed_fwd_kernel<T, D, KR, false>), dim3(static_cast<unsigned>(n)), dim3(256), 0, s, a);
}
template <typename T>
static void launch_packed_fwd_t(const PackedArgs& a, bool ragged, hipStream_t s) {
  if (!ragged) {
    if (a.d == 128) launch_packed_fwd<T, 128, 0>(a, s);
    else launch_packed_fwd<T, 64, 0>(a, s);
    return;
  }
  switch ((a.d + 15) / 16) {
    case 1:
    case 2: launch_packed_fwd<T, 64, 2>(a, s); break;
    case 3: launch_packed_fwd<T, 64, 3>(a, s); break;
    case 4: launch_packed_fwd<T, 64, 4>(a, s); break;
    case 5: launch_packed_fwd<T, 128, 5>(a, s); break;
    case 6: launch_packed_fwd<T, 128, 6>(a, s); break;
    case 7: launch_packed_fwd<T, 128, 7>(a, s); break;
    default: launch_packed_fwd<T, 128, 8>(a, s); break;
  }
}
}  // namespace zk

extern "C" int zk_attn_packed_fwd(const zk_packed_desc* desc, const void* q, const void* k,
                                  const void* v, const void* plan, void* o, float* lse,
                                  zk_stream_t stream) {
  const char* who = "zk_attn_packed_fwd";
  bool ragged;
  const int rc = check_packed(desc, who, false, &ragged, {q, k, v, o});
  if (rc != ZK_OK) return rc;
  if (desc->T == 0) return ZK_OK;
  ZK_REQUIRE(plan && lse, ZK_EINVAL, "%s: null pointer", who);
  ZK_REQUIRE(aligned(plan, 4) && aligned(lse, 4), ZK_EALIGN, "%s: plan and lse must be 4-byte aligned", who);
  PackedArgs a = {};
  packed_args(a, desc, plan);
  a.q = q; a.k = k; a.v = v; a.out = o; a.lse_out = lse;
  hipStream_t s = as_stream(stream);
  if (desc->dtype == ZK_F32)
    launch_packed_fwd_f32(a, s);
  else if (desc->dtype == ZK_BF16)
    launch_packed_fwd_t<bf16>(a, ragged, s);
  else
    launch_packed_fwd_t<f16>(a, ragged, s);
  return launch_status(who);
}
