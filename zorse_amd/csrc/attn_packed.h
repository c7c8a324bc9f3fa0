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

// This lane's 8 elements 16 ks + 8 g .. of each step of a row of d (null: zeros).
template <typename T, int KS, int KR>
__device__ __forceinline__ void load_operand(typename Mfma<T>::vec8 (&x)[KS], const T* row, int g,
                                             int d) {
  typedef typename Mfma<T>::vec8 V8;
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    if (row == nullptr)
      x[ks] = V8{};
    else if constexpr (KR != 0)
      x[ks] = load_cols8<T>(row, 16 * ks + 8 * g, d);
    else
      x[ks] = *reinterpret_cast<const V8*>(row + 16 * ks + 8 * g);
  }
}

// Whether step ks of a ragged head may hold elements from d on (d above 16 KR -
// 16, or any for the smallest KR, 2).
template <int KR>
__host__ __device__ constexpr bool ragged_step(int ks) {
  return KR != 0 && (ks == KR - 1 || KR == 2);
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
      if constexpr (KR != 0)
        store_cols4(row, d0, d, w);
      else
        *reinterpret_cast<T4*>(row + d0) = w;
    }
}

// Whether a lane's row (both halves of it) holds a NaN in its first d elements.
// A masked probability is an exact zero, and the matrix product adds its
// product with the masked row as well: NaN where that row holds an infinity or
// a NaN.  Such rows are computed again from what they see alone, 16 columns at a
// time (few registers, so that the loops before keep theirs; no one waits for it).
template <int NB>
__device__ __forceinline__ bool row_has_nan(const f32x16 (&x)[NB], int g, int d) {
  bool bad = false;
#pragma unroll
  for (int nt = 0; nt < NB; ++nt)
#pragma unroll
    for (int j = 0; j < 16; ++j)
      bad |= 32 * nt + 8 * (j >> 2) + 4 * g + (j & 3) < d && x[nt][j] != x[nt][j];
  const uint64_t b = __ballot(bad);
  return ((b >> (threadIdx.x & 31)) | (b >> ((threadIdx.x & 31) + 32))) & 1;
}

// x . y of two rows of d elements, each half of the wave taking half of them.
template <typename T>
__device__ __forceinline__ float dot_two_rows(const T* x, const T* y, int g, int d) {
  float s = 0.f;
#pragma unroll 1
  for (int c = 8 * g; c < d; c += 16)
    for (int e = 0; e < 8; ++e)
      if (c + e < d) s = fmaf(to_f32(x[c + e]), to_f32(y[c + e]), s);
  return s + other_half(s);
}

}  // namespace zk
