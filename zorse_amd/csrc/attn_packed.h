// Packed sequences: T tokens in a row, sequence s the tokens [offsets[s],
// offsets[s + 1]); shared by the plan, the forward and the backward kernels.
//
// The keys that a query sees form one range [key_lo, key_hi] of tokens (its
// sequence, cut by the causal mask and by the window), and so do the queries
// that see a key.  Both ends grow with the row, so a block of rows needs the
// tokens from its first row's lower end to its last row's upper one, whatever
// number of sequences it holds: blocks are cut from the run of tokens as it
// stands, and short sequences share them.
//
// The plan (zk_packed_plan), int32 words on the device:
//   [0]            n, the tokens that belong to a sequence (offsets' last)
//   [16 ..]        start[T], end[T]: a token's sequence; tokens from n on have
//                  start = end = their own index, so they see and are seen by
//                  nothing
//   then           two orders of the blocks of 128 rows, most work first: for
//                  kernels that own queries, and for those that own keys
#pragma once
#include "attn_common.h"

namespace zk {

constexpr int kPlanHeader = 16;

constexpr int kPlanRows = 128;  // rows of a listed block

// Words before order `which` (0: of queries, 1: of keys; 2: of the whole plan).
__host__ __device__ inline int64_t plan_order_at(int64_t T, int which) {
  return kPlanHeader + 2 * T + which * ((T + kPlanRows - 1) / kPlanRows);
}

struct PackedArgs {
  const void* q;
  const void* k;
  const void* v;
  const void* o;
  const void* dout;
  const float* lse;
  void* out;
  float* lse_out;
  void* dq;
  void* dk;
  void* dv;
  float* delta;  // backward workspace, fp32 [Hq, T] each
  float* lse2;
  // dK / dV of the query heads of a key head in `parts` sums: parts > 1 are stored
  // in fp32, [parts, T, Hkv, d] each, and added by a launch of their own
  float* dk_part;
  float* dv_part;
  int parts;
  const int32_t* plan;
  int64_t T;
  int Hq, Hkv, d;
  int64_t q_s, q_h, k_s, k_h, v_s, v_h, o_s, o_h, do_s, do_h;
  int64_t dq_s, dq_h, dk_s, dk_h, dv_s, dv_h;
  float scale, scale_log2;
  int causal, window;  // window: 0 or the keys that a query sees at most
  int keep_tail;       // rows behind the last sequence are left as they are
};

struct PackedPlan {
  const int32_t* start;
  const int32_t* end;
  int n;
  __device__ __forceinline__ PackedPlan(const PackedArgs& a) {
    n = a.plan[0];
    start = a.plan + kPlanHeader;
    end = start + a.T;
  }
  // first row of a block of ROWS, a divisor of the listed blocks' rows, in the order
  // of launch
  template <int ROWS, bool kKeys>
  __device__ __forceinline__ int first_row(const PackedArgs& a, int block) const {
    constexpr int PER = kPlanRows / ROWS;
    const int32_t* order = a.plan + plan_order_at(a.T, kKeys);
    return order[block / PER] * kPlanRows + (block % PER) * ROWS;
  }
  // keys that query i sees: [key_lo, key_hi]
  __device__ __forceinline__ int key_lo(const PackedArgs& a, int i) const {
    const int s = start[i], w = i - a.window + 1;
    return a.window > 0 && w > s ? w : s;
  }
  __device__ __forceinline__ int key_hi(const PackedArgs& a, int i) const {
    const int e = end[i] - 1;
    return a.causal && e > i ? i : e;
  }
  // queries that see key j: [query_lo, query_hi]
  __device__ __forceinline__ int query_lo(const PackedArgs& a, int j) const {
    return a.causal ? j : start[j];
  }
  __device__ __forceinline__ int query_hi(const PackedArgs& a, int j) const {
    const int e = end[j] - 1;
    // the sum of two positions fits 32 bits: T and the window are below 2^30
    return a.window > 0 && j + a.window - 1 < e ? j + a.window - 1 : e;
  }
};

// fp32 (attn_packed_f32.hip)
void launch_packed_fwd_f32(const PackedArgs& a, hipStream_t s);
void launch_packed_bwd_f32(const PackedArgs& a, hipStream_t s);

// Workgroups for blocks of `rows` rows of T: whole listed blocks.
__host__ __device__ inline int64_t packed_blocks(int64_t T, int rows) {
  return (T + kPlanRows - 1) / kPlanRows * (kPlanRows / rows);
}

// Whether the 2-byte kernels take a block in two groups of waves (their kSplit) in a
// launch of n workgroups: one a CU at most, and rows that may meet more than 256
// tokens.  64 tokens in two groups: forward 8 us, backward 20, else 6 and 17.  At two
// a CU long sequences gain by it (16 heads of 4096 causal tokens forward 105 and 90 us)
// what sequences of 500 tokens lose (24 and 33).
inline bool packed_split(const PackedArgs& a, int64_t n) {
  return n <= device_cus() && a.T > 256 && (a.window == 0 || a.window > 128);
}

// Head of a block in the order of launch: the workgroups of one XCD (dispatch
// goes round the eight of them) take the query heads of as few key heads as
// possible, so that a key head's tiles are fetched into one L2.
__device__ __forceinline__ void packed_block(const PackedArgs& a, int& block, int& hq) {
  const unsigned H = a.Hq, rep = a.Hq / a.Hkv, bid = blockIdx.x;
  block = bid / H;
  const unsigned r = bid % H;
  hq = (a.Hkv & 7) == 0 ? static_cast<int>(((r & 7) + 8 * (r / (8 * rep))) * rep + (r >> 3) % rep)
                        : static_cast<int>(r);
}

// The lane's row and half of the wave once more: loops before that are short of registers
// then need not keep what is made of them.
__device__ __forceinline__ void relane(int& l32, int& g) {
  int n = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u));
  asm volatile("" : "+v"(n));
  l32 = n & 31;
  g = n >> 5;
}

// Tile loads (asynchronous, global memory to LDS) of ROWS tokens from token g0
// on: rows at or past `nrows` and, for a head dim d < D (KR != 0), chunks past
// the head arrive as zeros, the offsets of a chunk that straddles its end as
// what follows it (mask_cols takes that out).  16-byte loads need 4-byte
// aligned rows only.
template <typename T, int D, int ROWS, int NT>
struct PackedLoader {
  static constexpr int NI = ROWS * D / 8 / NT;
  static constexpr int RSTEP = NT / (D / 8);
  static_assert(NI >= 1 && RSTEP % 16 == 0, "unsupported tile shape");
  uint32_t lane_off;
  int64_t row_bytes;

  __device__ __forceinline__ void init(int64_t ld, int d) {
    const int tid = threadIdx.x;
    const int row = tid / (D / 8);
    const int c = (tid % (D / 8)) ^ tile_sw<D>(row);
    lane_off = c * 8 < d ? static_cast<uint32_t>(row * ld * static_cast<int64_t>(sizeof(T)) + c * 16)
                         : 0x80000000u;
    row_bytes = d * static_cast<int64_t>(sizeof(T));
  }
  __device__ __forceinline__ void issue(T* tile, const T* gbase, int64_t ld, int64_t g0,
                                        int64_t nrows) const {
    const int wave_chunk0 = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) & ~63);
    int64_t left = (nrows - 1 - g0) * ld * static_cast<int64_t>(sizeof(T)) + row_bytes;
    left = left < 0 ? 0 : left > 0x7fffffff ? 0x7fffffff : left;
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<T*>(gbase + g0 * ld), 0, static_cast<int>(left), 0x00020000);
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const uint32_t soff =
          static_cast<uint32_t>(static_cast<int64_t>(i) * RSTEP * ld * static_cast<int64_t>(sizeof(T)));
      dma_lds<16>(r, lane_off, soff, tile + (i * NT + wave_chunk0) * 8);
    }
  }
};

// Whether step ks of a ragged head (its columns 16 ks .. 16 ks + 15) may hold elements
// from d on (d above 16 KR - 16, or any for the smallest KR, 2).
template <int KR>
__host__ __device__ constexpr bool ragged_step(int ks) {
  return KR != 0 && (ks >= KR - 1 || KR == 2);
}

// This lane's 8 elements 16 ks + 8 g .. of a row of d (null: zeros), and those of each
// step.
template <typename T, int KR>
__device__ __forceinline__ typename Mfma<T>::vec8 operand_step(const T* row, int ks, int g, int d) {
  typedef typename Mfma<T>::vec8 V8;
  if (row == nullptr) return V8{};
  typedef uint32_t u32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));
  if (ragged_step<KR>(ks)) return load_cols8<T>(row, 16 * ks + 8 * g, d);
  if constexpr (KR != 0)
    return __builtin_bit_cast(V8, static_cast<u32x4>(*reinterpret_cast<const u32x4_a4*>(row + 16 * ks + 8 * g)));
  return *reinterpret_cast<const V8*>(row + 16 * ks + 8 * g);
}
template <typename T, int KS, int KR>
__device__ __forceinline__ void load_operand(typename Mfma<T>::vec8 (&x)[KS], const T* row, int g,
                                             int d) {
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) x[ks] = operand_step<T, KR>(row, ks, g, d);
}

// Stores this lane's accumulators (elements 32 nt + 8 (j / 4) + 4 g + j % 4 of a
// row), scaled.
template <typename T, int NB, int KR>
__device__ __forceinline__ void store_accumulators(T* row, const f32x16 (&x)[NB], float scale, int g,
                                                   int d) {
#pragma unroll
  for (int nt = 0; nt < NB; ++nt)
#pragma unroll
    for (int a4 = 0; a4 < 4; ++a4) {
      const int d0 = 32 * nt + 8 * a4 + 4 * g;
      typedef T T4 __attribute__((ext_vector_type(4)));
      T4 w;
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = static_cast<T>(x[nt][4 * a4 + e] * scale);
      typedef uint32_t u32x2_a4 __attribute__((ext_vector_type(2), aligned(4)));
      if (ragged_step<KR>(2 * nt + a4 / 2))
        store_cols4(row, d0, d, w);
      else if constexpr (KR != 0)
        *reinterpret_cast<u32x2_a4*>(row + d0) = __builtin_bit_cast(u32x2, w);
      else
        *reinterpret_cast<T4*>(row + d0) = w;
    }
}

// ---- Rows with a NaN ("odd": an infinity or a NaN).
// A masked probability is an exact zero, and the matrix product adds its product with
// the masked row as well: NaN where that row holds an odd element.  So a wave that finds
// a NaN among its rows' results (row_has_nan) asks whether a masked row can be the
// cause: whether among the tokens that it met and some row does not see any is odd.
// These are few (the tiles on the diagonal and at sequences' ends), so a pass whose
// results are NaN by right, as those of a step that overflows under a loss scale are,
// takes no longer.  Where one is, the wave takes its rows once more, in tiles of 32
// tokens from global memory: in tiles that some row does not see, the product takes
// zeros for the odd elements (add_columns), and those that are seen are added one by one
// (add_odd); but a row that sees all of a tile takes its product, and one that sees
// nothing of it leaves it out.  It ends early when every element is NaN.
//   32 heads of 128 over 8 key heads, 8192 causal tokens, forward and backward 2.3 - 2.6
// ms: with a NaN in the last row of dO 2.5, an infinity in one of its middle 6.0 and a
// NaN in its first (which all keys of the first tile but one do not see) 9.8, NaN in all
// of q, k, v or dO 2.3 - 2.7, infinities in all of v 8.4.

// Whether a lane's row (both halves of it) holds a NaN in its first d elements.
template <int NB, int KR>
__device__ __forceinline__ bool row_has_nan(const f32x16 (&x)[NB], int g, int d) {
  bool bad = false;
#pragma unroll
  for (int nt = 0; nt < NB; ++nt)
#pragma unroll
    for (int j = 0; j < 16; ++j)
      bad |= (!ragged_step<KR>(2 * nt + j / 8) || 32 * nt + 8 * (j >> 2) + 4 * g + (j & 3) < d) &&
             x[nt][j] != x[nt][j];
  const uint64_t b = __ballot(bad);
  return ((b >> (threadIdx.x & 31)) | (b >> ((threadIdx.x & 31) + 32))) & 1;
}

// Whether all of this lane's elements below d are NaN, of the columns from c0 on (not 0
// for one block of 32 only).
template <int NB, int KR>
__device__ __forceinline__ bool all_nan(const f32x16 (&x)[NB], int c0, int g, int d) {
  bool all = true;
#pragma unroll
  for (int nt = 0; nt < NB; ++nt)
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const bool may_end = KR != 0 && (NB == 1 || ragged_step<KR>(2 * nt + j / 8));
      all &= (may_end && c0 + 32 * nt + 8 * (j >> 2) + 4 * g + (j & 3) >= d) || x[nt][j] != x[nt][j];
    }
  return all;
}

// Stores one block of accumulators, the columns from c0 on, scaled.
template <typename T>
__device__ __forceinline__ void store_block(T* row, const f32x16& x, float scale, int c0, int g, int d) {
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    const int c = c0 + 8 * (j >> 2) + 4 * g + (j & 3);
    if (c < d) row[c] = static_cast<T>(x[j] * scale);
  }
}

template <typename T>
__device__ __forceinline__ bool is_odd(T x) {
  return !(fabsf(to_f32(x)) < INFINITY);
}
template <typename T>
__device__ __forceinline__ bool any_odd(typename Mfma<T>::vec8 x) {
  bool odd = false;
#pragma unroll
  for (int e = 0; e < 8; ++e) odd |= is_odd<T>(x[e]);
  return odd;
}

// Bit r: row r0 + r of X (below past) holds an odd element and lies outside
// [in_lo, in_hi].
template <typename T, int KS, int KR>
__device__ __forceinline__ uint32_t odd_rows(const T* X, int64_t ld, int r0, int past, int in_lo, int in_hi,
                                             int g, int d) {
  const int r = r0 + static_cast<int>(threadIdx.x & 31);
  const T* row = r < past && (r < in_lo || r > in_hi) ? X + r * ld : nullptr;
  bool odd = false;
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) odd |= any_odd<T>(operand_step<T, KR>(row, ks, g, d));
  const uint64_t b = __ballot(odd);
  return static_cast<uint32_t>(b | b >> 32);
}

// A column, which the compiler does not know: nothing made of it is kept outside the
// loops around.
__device__ __forceinline__ int column(int c) {
  asm volatile("" : "+s"(c));
  return c;
}

// acc += X^T w of the columns from c0 on of 32 rows of X from r0 on, as tr_operand's
// products; kept: with odd
// elements, for the lanes that see all of the rows (the others see none of them), else
// with zeros in their place.  Rows from past on, which are not kept and whose weights are
// zero, are read as the last one; columns from d on, which nothing stores, as the last one.
template <typename T, int NB>
__device__ __forceinline__ void add_columns(f32x16 (&acc)[NB], const T* X, int64_t ld, int r0, int past,
                                            int c0, const typename Mfma<T>::vec8 (&w)[2], bool kept,
                                            bool sees_all, int g, int d) {
#pragma unroll
  for (int kk = 0; kk < 2; ++kk)
#pragma unroll
    for (int nt = 0; nt < NB; ++nt) {
      __builtin_amdgcn_sched_barrier(0);  // one block's loads at a time: few registers
      const int c = column(c0 + 32 * nt) + static_cast<int>(threadIdx.x & 31), at = c < d ? c : d - 1;
      typename Mfma<T>::vec8 x;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int r = r0 + 16 * kk + 8 * (e >> 2) + 4 * g + (e & 3);
        x[e] = X[(r < past ? r : past - 1) * ld + at];
        if (!kept && is_odd<T>(x[e])) x[e] = static_cast<T>(0.f);
      }
      const f32x16 sum = Mfma<T>::mma(x, w[kk], acc[nt]);
      const bool mine = !kept || sees_all;
#pragma unroll
      for (int j = 0; j < 16; ++j) acc[nt][j] = mine ? sum[j] : acc[nt][j];
    }
}

// acc += weight X[r] of the odd elements of these columns of the rows r0 + (bits of rows)
// that the lane's row sees.  weights: of the tile's 32 rows, where the products leave
// them (row 8 (j / 4) + 4 g + j % 4).
template <typename T, int NB, typename S>
__device__ __forceinline__ void add_odd(f32x16 (&acc)[NB], const T* X, int64_t ld, int r0, uint32_t rows,
                                        int c0, const f32x16& weights, S&& seen, int g, int d) {
#pragma unroll 1
  while (rows != 0) {
    const int at = __builtin_ctz(rows), r = r0 + at;
    rows &= rows - 1;
    float w = weights[0];
#pragma unroll
    for (int j = 1; j < 16; ++j) w = (at >> 3) * 4 + (at & 3) == j ? weights[j] : w;
    const float other = other_half(w);
    if ((at >> 2 & 1) != g) w = other;
    const bool mine = seen(r);
    const T* row = X + r * ld;
#pragma unroll
    for (int nt = 0; nt < NB; ++nt) {
      const int c_nt = column(c0 + 32 * nt) + 4 * g;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const int c = c_nt + 8 * (j >> 2) + (j & 3);
        const T x = row[c < d ? c : d - 1];
        if (mine && is_odd<T>(x)) acc[nt][j] = fmaf(w, to_f32(x), acc[nt][j]);
      }
    }
  }
}

}  // namespace zk
