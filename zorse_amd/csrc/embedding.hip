// Token embedding: y[t] = round(s W[id_t]), and its gradient
// dW[r] = round(s sum_{t: id_t = r} dy[t]) (+ dW[r]).
//
// Both move rows and hardly compute: HBM bounds them.  The gradient's sums
// are taken in the order of the tokens, in fp32, without atomics, so that a
// repeated pass gives the same bits.  Three launches:
//   1. embed_sort: the tokens grouped by id (stable), and each id's count.
//      Workgroup g of G (a power of two) owns the ids with id mod G = g, so
//      that the frequent low ids of a text spread over all of them.  Every
//      workgroup reads all ids, to count its own and the tokens of the groups
//      before it -- its offset, so none waits for another.  For the stable
//      order each of 16 waves owns a sixteenth of the tokens, a row of counters
//      and a list of the tokens it found; what a full list does not hold (a
//      token that fills much of a batch) is looked for again.
//   2. embed_grad: the grouped tokens in blocks, one wave for each block and
//      512 columns, whatever the ids: a token that fills half the batch costs
//      no more than many single ones.  An id whose tokens lie in one block is
//      finished there; of one that crosses blocks, each block leaves a partial
//      sum (at most two a block: the id it begins with and the id it ends in).
//      Waves after those write the rows of unused ids.
//   3. embed_join: the partial sums of ids that cross blocks.
// Up to kFew tokens take one launch instead, embed_few: every wave holds all
// ids, two a lane, and finds a row's tokens by comparing.
#include "part8.h"

namespace zk {

static constexpr int kSortWaves = 16;
static constexpr int kMaxSlots = 512;   // ids a sort workgroup owns: 32 KB of counters
static constexpr int kList = 448;       // found tokens a wave remembers: 28 KB

struct Token {
  int t, id;
};
struct Fill {  // the rows that a workgroup looks at, 2^log_tpr threads each
  int rows, log_tpr;
};
struct Span {  // the id that crosses out of the block where it begins (-1: none)
  int id, parts;
};

// ---------------------------------------------------------------- forward ---
// tpr (a power of two up to 256) threads a row, 8 elements each at a time: a
// workgroup holds a long row or several short ones.  HBM bounds it: 16312 tokens
// of 2048 in fp16 (134 MB at most, repeated rows come from the caches) take 16
// us, 4096 of 4096 in bf16 (67 MB) 10.  A ragged row's end goes element by element
// (see part8.h), which costs little beside the rows of other waves: 16384 tokens
// of 2047 in bf16 22.4 us, of 2048 20.5; 8192 of 1001 6.5, of 1000 5.7.
template <typename I, typename W, typename Y>
__global__ __launch_bounds__(256) void embed_fwd(const I* __restrict__ ids, int64_t T,
                                                 const W* __restrict__ w, int64_t V, int h,
                                                 Y* __restrict__ y, float scale, int log_tpr) {
  const int tpr = 1 << log_tpr;
  const int64_t step = static_cast<int64_t>(gridDim.x) << (8 - log_tpr);
  for (int64_t t = (static_cast<int64_t>(blockIdx.x) << (8 - log_tpr)) + (threadIdx.x >> log_tpr);
       t < T; t += step) {
    const int64_t id = ids[t];
    const bool known = id >= 0 && id < V;
    for (int c = (threadIdx.x & (tpr - 1)) * 8; c < h; c += tpr * 8) {
      float o[8];
      if (known) {
        Part8<W> x;
        x.load(w + id * h + c, h - c);
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = scale * x[i];
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = __builtin_nanf("");
      }
      Part8<Y>::store(y + t * h + c, o, h - c);
    }
  }
}

// ------------------------------------------------------------------- sort ---
// Every workgroup reads all ids, from its die's L2: T 8 bytes each.  Vector
// instructions (two ballots a chunk of 64 tokens) and the latency of those reads
// bound it: 4096 tokens 8 us, 16312 9, 65536 31.
// A token's id in 32 bits, or all ones for one that has no row of the table
// (vocab < 2^28).
__device__ __forceinline__ uint32_t id32(const int32_t* ids, int64_t t) {
  return static_cast<uint32_t>(ids[t]);
}
__device__ __forceinline__ uint32_t id32(const int64_t* ids, int64_t t) {
  const uint2 u = reinterpret_cast<const uint2*>(ids)[t];
  return u.y == 0 ? u.x : ~0u;
}

// The keys of N chunks of 64 tokens from t on, one a lane and chunk: the id
// turned right by log_g bits, so that the group stands above the slot and keys
// order the groups; all ones where there is no token with a gradient (no key:
// an id is below 2^28, its slot below 2^20).
template <int N, typename I>
__device__ __forceinline__ void load_keys(const I* ids, int64_t t, int64_t end, uint32_t V,
                                          uint32_t pad, int log_g, uint32_t (&key)[N]) {
  const int lane = threadIdx.x & 63;
  if (t + N * 64 <= end) {
#pragma unroll
    for (int k = 0; k < N; ++k) key[k] = id32(ids, t + k * 64 + lane);
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k) key[k] = t + k * 64 + lane < end ? id32(ids, t + k * 64 + lane) : ~0u;
  }
#pragma unroll
  for (int k = 0; k < N; ++k)
    key[k] = key[k] < V && key[k] != pad ? __builtin_rotateright32(key[k], log_g) : ~0u;
}

template <typename I>
__global__ __launch_bounds__(64 * kSortWaves) void embed_sort(
    const I* __restrict__ ids, int T, uint32_t V, int log_g, int slots, uint32_t pad,
    Token* __restrict__ out, int* __restrict__ count, int* __restrict__ total) {
  extern __shared__ int cnt[];  // [kSortWaves][slots]
  __shared__ uint32_t list[kSortWaves][kList];
  __shared__ int red[kSortWaves], run[kSortWaves];
  const uint32_t g = blockIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  for (int i = threadIdx.x; i < kSortWaves * slots; i += 64 * kSortWaves) cnt[i] = 0;
  __syncthreads();
  // this wave's tokens: chunks of 64 from t0 on
  const int chunks = (T + 64 * kSortWaves - 1) / (64 * kSortWaves);
  const int64_t t0 = static_cast<int64_t>(wave) * chunks * 64;
  const int64_t end = t0 + chunks * 64 < T ? t0 + chunks * 64 : T;
  const uint32_t first = g << (32 - log_g), own = slots;  // this group's keys: first + slot
  int* mine = cnt + wave * slots;
  const uint64_t below = (1ull << lane) - 1;
  int before = 0, found = 0, again = -1;  // again: the first chunk that the list does not hold
  constexpr int kAhead = 8;
  for (int c0 = 0; c0 < chunks; c0 += kAhead) {
    uint32_t key[kAhead];
    load_keys(ids, t0 + c0 * 64, end, V, pad, log_g, key);
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      before += __popcll(__ballot(key[k] < first));
      const uint32_t slot = key[k] - first;
      const bool is = slot < own;
      const uint64_t m = __ballot(is);
      if (m == 0) continue;
      const int n = __popcll(m);
      if (n <= 8) {
        if (is) atomicAdd(mine + slot, 1);
      } else {  // mostly one id: one lane adds for all of an id's
        for (uint64_t left = m; left != 0;) {
          const int lead = __builtin_ctzll(left);
          const uint64_t same = left & __ballot(slot == __builtin_amdgcn_readlane(slot, lead));
          if (lane == lead) atomicAdd(mine + slot, __popcll(same));
          left &= ~same;
        }
      }
      if (again < 0) {
        // an entry: 17 bits of chunk, 6 of lane, 9 of slot
        if (found + n <= kList && c0 + k < 1 << 17) {
          if (is) list[wave][found + __popcll(m & below)] =
              static_cast<uint32_t>(c0 + k) << 15 | lane << 9 | slot;
          found += n;
        } else {
          again = c0 + k;
        }
      }
    }
  }
  if (again < 0) again = chunks;
  if (lane == 0) red[wave] = before;
  __syncthreads();
  int base = 0;
#pragma unroll
  for (int i = 0; i < kSortWaves; ++i) base += red[i];
  // thread i: the tokens of the workgroup's i-th id, and those of the ids before
  const int i = threadIdx.x;
  int n = 0;
  if (i < slots)
    for (int k = 0; k < kSortWaves; ++k) n += cnt[k * slots + i];
  int incl = n;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int up = __shfl_up(incl, off, 64);
    if (lane >= off) incl += up;
  }
  if (lane == 63) run[wave] = incl;
  __syncthreads();
  int all = 0, prior = 0;
#pragma unroll
  for (int k = 0; k < kSortWaves; ++k) {
    if (k < wave) prior += run[k];
    all += run[k];
  }
  if (g == gridDim.x - 1 && i == 0) *total = base + all;
  if (i < slots) {
    int at = base + prior + incl - n;
    for (int k = 0; k < kSortWaves; ++k) {
      const int c = cnt[k * slots + i];
      cnt[k * slots + i] = at;
      at += c;
    }
    const uint32_t id = (static_cast<uint32_t>(i) << log_g) + g;
    if (id < V) count[id] = n;
  }
  __syncthreads();
  // place: up to 64 tokens at a time, the lanes of one id after another; a
  // wave's counters are its own, and its LDS accesses (volatile) are in order
  volatile int* next = mine;
  auto place = [&](int slot, int t, uint64_t left) {
    while (left != 0) {
      const int lead = __builtin_ctzll(left);
      const int key = __builtin_amdgcn_readlane(slot, lead);
      const bool same = ((left >> lane) & 1) != 0 && slot == key;
      const uint64_t m = __ballot(same);
      const int at = next[key];
      if (same) out[at + __popcll(m & below)] = Token{t, static_cast<int>((key << log_g) + g)};
      if (lane == lead) next[key] = at + __popcll(m);
      left &= ~m;
    }
  };
  for (int i0 = 0; i0 < found; i0 += 64) {
    const bool is = i0 + lane < found;
    const uint32_t e = is ? list[wave][i0 + lane] : 0;
    place(e & 511, static_cast<int>(t0 + (e >> 15) * 64 + (e >> 9 & 63)), __ballot(is));
  }
  for (int c0 = again; c0 < chunks; c0 += kAhead) {
    uint32_t key[kAhead];
    load_keys(ids, t0 + c0 * 64, end, V, pad, log_g, key);
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      place(static_cast<int>(key[k] - first), static_cast<int>(t0 + (c0 + k) * 64 + lane),
            __ballot(key[k] - first < own));
  }
}

// --------------------------------------------------------------- gradient ---
// A wave's columns of a row: `lanes` chunks of 8 a slice.  The row's last chunk
// ends with the row and may overlap the one before it, lanes behind it repeat
// it: they read, compute and store the same values in the same instructions (why
// not element by element: part8.h).
// Rows of less than 8 columns are one chunk of h.
struct Columns {
  int lanes, slices;  // chosen so that a slice has more than an overlapping chunk:
                      // two waves may not add to the same column
};
__device__ __forceinline__ int my_column(const Columns& cols, int slice, int h) {
  const int lane = threadIdx.x & 63;
  const int c = (slice * cols.lanes + (lane < cols.lanes ? lane : cols.lanes - 1)) * 8;
  return h < 8 ? 0 : c < h - 8 ? c : h - 8;
}

// Zeros for the rows r0 + i of the set bits i of `empty`, by a workgroup: each of
// its accesses writes neighbouring 16 bytes a thread, 4 KB, of one row or of
// several.  Lines are written whole: nontemporal stores of half lines (8 fp32 a
// lane) took 2.4 times as long.
template <typename W>
__device__ __forceinline__ void fill_rows(W* dw, int64_t r0, uint64_t empty, int h, const Fill& fill) {
  constexpr int E = 16 / sizeof(W);
  typedef W V __attribute__((ext_vector_type(E)));
  typedef V Vu __attribute__((aligned(sizeof(W))));
  const int tpr = 1 << fill.log_tpr;
  for (int i = threadIdx.x >> fill.log_tpr; i < fill.rows; i += 256 >> fill.log_tpr) {
    if (!(empty >> i & 1)) continue;
    W* p = dw + (r0 + i) * h;
    int c = (threadIdx.x & (tpr - 1)) * E;
    for (; c + E <= h; c += tpr * E) __builtin_nontemporal_store(V{}, reinterpret_cast<Vu*>(p + c));
    for (int j = c; j < h && j < c + E; ++j) __builtin_nontemporal_store(static_cast<W>(0.f), p + j);
  }
}

// part: [blocks][2][hp] fp32 (hp: part_row(h)): the sum of the id that
// a block begins with and of the one that it ends in, where they reach over
// its border (an id that does both: the first).  blk: tokens a block, up to 64
// (a lane holds one).  kStream: dy is larger than the last-level cache, and its
// rows take no place there.
//
// HBM bounds it: a table of 49152 x 4096 in bf16, 4096 tokens (403 MB written,
// most of it zeros, 34 read) 68 us, 6.4 TB/s; 65536 tokens of 5120 in bf16 added
// to an fp32 table (671 MB of dy, the named rows read and written: 1.29 GB) 267
// us, 4.8 TB/s; 16312 tokens of 2048 in fp16, half of them padding, 28 us.
template <typename D, typename W, bool kAdd, bool kStream>
__global__ __launch_bounds__(256) void embed_grad(
    const D* __restrict__ dy, W* __restrict__ dw, const Token* __restrict__ tok,
    const int* __restrict__ count, const int* __restrict__ total, float* __restrict__ part,
    Span* __restrict__ span, int64_t V, int h, int hp, Columns cols, int blk, int64_t sum_items,
    Fill fill, float scale) {
  const int lane = threadIdx.x & 63;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * 4 +
                       __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (item >= sum_items) {
    const int64_t wg = blockIdx.x - (sum_items + 3) / 4;
    if (kAdd || wg < 0) return;  // a wave that rounds the sums' last workgroup up
    const int64_t r0 = wg * fill.rows, r = r0 + lane;
    fill_rows(dw, r0, __ballot(lane < fill.rows && r < V && count[r < V ? r : 0] == 0), h, fill);
    return;
  }
  const int64_t j = item / cols.slices;
  const int c = my_column(cols, static_cast<int>(item - j * cols.slices), h), nc = h < 8 ? h : 8;
  const int n_all = *total;
  const int64_t p0 = j * blk;
  if (p0 >= n_all) {
    if (c == 0) span[j] = Span{-1, 0};
    return;
  }
  const int n = n_all - p0 < blk ? static_cast<int>(n_all - p0) : blk;
  const Token e = lane < n ? tok[p0 + lane] : Token{0, -1};
  const int prev = p0 > 0 ? tok[p0 - 1].id : -1;
  const int next = p0 + n < n_all ? tok[p0 + n].id : -1;
  // bit i: token i is the last of its id here; the first of them ends an id
  // that began before this block, the last one may reach into the next
  const int after = __shfl_down(e.id, 1, 64);
  const uint64_t ends = __ballot(lane < n && (lane == n - 1 || after != e.id));
  const bool head = __builtin_amdgcn_readfirstlane(e.id) == prev;
  const int first_end = __builtin_ctzll(ends);
  const int last_id = __builtin_amdgcn_readlane(e.id, n - 1);
  if (c == 0) {  // one lane: what embed_join has to add up from this block on
    Span sp = {-1, 0};
    const uint64_t before = ends & ~(1ull << (n - 1));  // where the last id begins
    const int first = before != 0 ? 64 - __builtin_clzll(before) : 0;
    if (last_id == next && !(head && first == 0))
      sp = Span{last_id, static_cast<int>((p0 + first + count[last_id] - 1) / blk - j) + 1};
    span[j] = sp;
  }
  float* pj = part + j * 2 * hp + c;
  float acc[8] = {};
  // rows in flight; with kAdd also the old rows of the ids that end among them
  constexpr int kAhead = 8, kSame = 16;
  for (int i0 = 0; i0 < n;) {
    if (i0 + kSame <= n && (ends >> i0 & ((1u << kSame) - 1)) == 0) {
      Part8<D> x[kSame];  // rows of one id that goes on after them
#pragma unroll
      for (int k = 0; k < kSame; ++k)
        x[k].template get<kStream>(
            dy + static_cast<int64_t>(__builtin_amdgcn_readlane(e.t, i0 + k)) * h + c, nc);
#pragma unroll
      for (int k = 0; k < kSame; ++k) {
#pragma unroll
        for (int q = 0; q < 8; ++q) acc[q] += x[k][q];
      }
      i0 += kSame;
      continue;
    }
    Part8<D> x[kAhead];
    Part8<W> old[kAdd ? kAhead : 1];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int i = i0 + k;
      if (i >= n) break;
      const int64_t t = __builtin_amdgcn_readlane(e.t, i);
      x[k].template get<kStream>(dy + t * h + c, nc);
      if (kAdd && (ends >> i & 1)) {
        const int64_t id = __builtin_amdgcn_readlane(e.id, i);
        old[kAdd ? k : 0].load(dw + id * h + c, nc);
      }
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int i = i0 + k;
      if (i >= n) break;
#pragma unroll
      for (int q = 0; q < 8; ++q) acc[q] += x[k][q];
      if (!(ends >> i & 1)) continue;
      const bool begun = head && i == first_end;
      if (begun || (i == n - 1 && last_id == next)) {
        Part8<float>::store(begun ? pj : pj + hp, acc, nc);
      } else {
        float o[8];
#pragma unroll
        for (int q = 0; q < 8; ++q)
          o[q] = kAdd ? old[kAdd ? k : 0][q] + scale * acc[q] : scale * acc[q];
        const int64_t id = __builtin_amdgcn_readlane(e.id, i);
        Part8<W>::store(dw + id * h + c, o, nc);
      }
#pragma unroll
      for (int q = 0; q < 8; ++q) acc[q] = 0.f;
    }
    i0 += kAhead;
  }
}

// The partial sums of each id that crosses blocks, in order, 256 columns a
// workgroup.  Each of 8 waves looks at a block and adds a few parts alone; the
// parts of an id that spans many blocks are shared by the eight.  Latency
// bounds it, not bytes: 7 us for the parts of 4096 tokens of 4096 columns, 22 for
// 65536 of 5120.  16 parts are in flight at a time, and 65536 tokens of 5120,
// nine tenths of them one id, take 282 us in all where four waves a workgroup
// took 320.
static constexpr int kJoinWaves = 8, kAloneParts = 16;

__device__ __forceinline__ float4 add_parts(const float* part, int64_t j, int64_t a, int64_t b,
                                            int h, int hp, int c) {
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  if (c >= h) return acc;
  // part 0 at block j's end, the others at their blocks' beginnings
  const float* base = part + j * 2 * hp + c;
  constexpr int kAhead = 16;
  for (int64_t k = a; k < b; k += kAhead) {
    float4 x[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int64_t q = k + u < b ? k + u : b - 1;
      x[u] = *reinterpret_cast<const float4*>(base + (q == 0 ? hp : q * 2 * hp));
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const bool on = k + u < b;
      acc.x += on ? x[u].x : 0.f;
      acc.y += on ? x[u].y : 0.f;
      acc.z += on ? x[u].z : 0.f;
      acc.w += on ? x[u].w : 0.f;
    }
  }
  return acc;
}

// The old elements of a row's 4 columns, fetched before the parts they add to.
template <typename W, bool kAdd>
__device__ __forceinline__ void get_old(const W* p, int n, float (&old)[4]) {
  typedef W W4 __attribute__((ext_vector_type(4)));
  typedef W4 W4u __attribute__((aligned(sizeof(W))));
#pragma unroll
  for (int q = 0; q < 4; ++q) old[q] = 0.f;
  if (!kAdd) return;
  if (n >= 4) {
    const W4 u = *reinterpret_cast<const W4u*>(p);
#pragma unroll
    for (int q = 0; q < 4; ++q) old[q] = to_f32(static_cast<W>(u[q]));
  } else {
#pragma unroll
    for (int q = 0; q < 3; ++q)
      if (q < n) old[q] = to_f32(p[q]);
  }
}

template <typename W, bool kAdd>
__device__ __forceinline__ void put_sum(W* p, const float4& acc, const float (&old)[4], int n,
                                        float scale) {
  typedef W W4 __attribute__((ext_vector_type(4)));
  typedef W4 W4u __attribute__((aligned(sizeof(W))));
  const float a[4] = {acc.x, acc.y, acc.z, acc.w};
  W4 u;
#pragma unroll
  for (int q = 0; q < 4; ++q) u[q] = static_cast<W>(kAdd ? old[q] + scale * a[q] : scale * a[q]);
  if (n >= 4) {
    *reinterpret_cast<W4u*>(p) = u;
    return;
  }
#pragma unroll
  for (int q = 0; q < 3; ++q)
    if (q < n) p[q] = u[q];
}

template <typename W, bool kAdd>
__global__ __launch_bounds__(64 * kJoinWaves) void embed_join(
    W* __restrict__ dw, const Span* __restrict__ span, const float* __restrict__ part, int64_t blocks,
    int h, int hp, float scale) {
  __shared__ int many[kJoinWaves], many_id[kJoinWaves];
  __shared__ float4 sums[kJoinWaves][64];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t j = static_cast<int64_t>(blockIdx.x) * kJoinWaves + wave;
  const int c = blockIdx.y * 256 + lane * 4;
  const Span sp = j < blocks ? span[j] : Span{-1, 0};
  const int parts = sp.parts, id = sp.id;
  if (lane == 0) {
    many[wave] = parts > kAloneParts ? parts : 0;
    many_id[wave] = id;
  }
  if (parts > 0 && parts <= kAloneParts) {
    W* p = dw + static_cast<int64_t>(id) * h + c;
    float old[4];
    get_old<W, kAdd>(p, h - c, old);
    put_sum<W, kAdd>(p, add_parts(part, j, 0, parts, h, hp, c), old, h - c, scale);
  }
  __syncthreads();
  for (int w = 0; w < kJoinWaves; ++w) {
    const int64_t all = many[w];
    if (all == 0) continue;  // the same for every wave
    sums[wave][lane] = add_parts(part, static_cast<int64_t>(blockIdx.x) * kJoinWaves + w,
                                 all * wave / kJoinWaves, all * (wave + 1) / kJoinWaves, h, hp, c);
    __syncthreads();
    if (wave == 0 && c < h) {
      float4 acc = sums[0][lane];
#pragma unroll
      for (int k = 1; k < kJoinWaves; ++k) {
        const float4 x = sums[k][lane];
        acc.x += x.x; acc.y += x.y; acc.z += x.z; acc.w += x.w;
      }
      W* p = dw + static_cast<int64_t>(many_id[w]) * h + c;
      float old[4];
      get_old<W, kAdd>(p, h - c, old);
      put_sum<W, kAdd>(p, acc, old, h - c, scale);
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------- few tokens ---
// Tokens that a wave holds, two a lane.  us in one launch / in three: 128 tokens
// of 256 columns, 320 rows 5.1 / 12.5, added 5.6 / 13.5; one token 128 times 15.4
// / 11.5 (a wave adds all rows in order, 16 at a time); 4096 columns and 49152
// rows, mostly zeros, 61 / 69.  The host does not know which ids are equal, and
// takes the one launch that all but batches of one token gain by.
static constexpr int kFew = 128;

// A wave's 512 columns of the row that a token names first; waves after those
// fill the rows that no token names.
template <typename I, typename D, typename W, bool kAdd>
__global__ __launch_bounds__(256) void embed_few(
    const I* __restrict__ ids, int T, const D* __restrict__ dy, W* __restrict__ dw, uint32_t V, int h,
    Columns cols, Fill fill, float scale, uint32_t pad) {
  const int lane = threadIdx.x & 63;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * 4 +
                       __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  uint32_t key[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int t = k * 64 + lane;
    key[k] = t < T ? id32(ids, t) : ~0u;
    key[k] = key[k] < V && key[k] != pad ? key[k] : ~0u;
  }
  const int64_t sums = static_cast<int64_t>(T) * cols.slices;
  if (item >= sums) {
    const int64_t wg = blockIdx.x - (sums + 3) / 4;
    if (kAdd || wg < 0) return;  // a wave that rounds the sums' last workgroup up
    const int64_t r0 = wg * fill.rows;
    uint64_t empty = 0;
    for (int i = 0; i < fill.rows && r0 + i < V; ++i) {
      const uint32_t r = static_cast<uint32_t>(r0) + i;
      if ((__ballot(key[0] == r) | __ballot(key[1] == r)) == 0) empty |= 1ull << i;
    }
    fill_rows(dw, r0, empty, h, fill);
    return;
  }
  const int t = static_cast<int>(item / cols.slices);
  const uint32_t r = __builtin_amdgcn_readlane(t < 64 ? key[0] : key[1], t & 63);
  uint64_t m0 = __ballot(key[0] == r), m1 = __ballot(key[1] == r);
  const int first = m0 != 0 ? __builtin_ctzll(m0) : 64 + __builtin_ctzll(m1);
  if (r == ~0u || first != t) return;
  const int c = my_column(cols, static_cast<int>(item - t * static_cast<int64_t>(cols.slices)), h);
  const int nc = h < 8 ? h : 8;
  W* p = dw + static_cast<int64_t>(r) * h + c;
  Part8<W> old;
  if (kAdd) old.load(p, nc);
  float acc[8] = {};
  constexpr int kAhead = sizeof(D) == 2 ? 16 : 8;
  // the tokens in order: those that fill rounds, then the others
  for (int left = __popcll(m0) + __popcll(m1); left >= kAhead; left -= kAhead) {
    Part8<D> x[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int next = m0 != 0 ? __builtin_ctzll(m0) : 64 + __builtin_ctzll(m1);
      if (m0 != 0) m0 &= m0 - 1;
      else m1 &= m1 - 1;
      x[k].load(dy + static_cast<int64_t>(next) * h + c, nc);
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
#pragma unroll
      for (int q = 0; q < 8; ++q) acc[q] += x[k][q];
    }
  }
  if ((m0 | m1) != 0) {
    Part8<D> x[kAhead];
    bool on[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      on[k] = (m0 | m1) != 0;
      const int next = m0 != 0 ? __builtin_ctzll(m0) : 64 + (m1 != 0 ? __builtin_ctzll(m1) : 0);
      if (m0 != 0) m0 &= m0 - 1;
      else m1 &= m1 - 1;
      x[k].load(dy + static_cast<int64_t>(on[k] ? next : 0) * h + c, nc);
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
#pragma unroll
      for (int q = 0; q < 8; ++q) acc[q] += on[k] ? x[k][q] : 0.f;
    }
  }
  float o[8];
#pragma unroll
  for (int q = 0; q < 8; ++q) o[q] = kAdd ? old[q] + scale * acc[q] : scale * acc[q];
  Part8<W>::store(p, o, nc);
}

// The groups of embed_sort: at least 256 workgroups, at most kMaxSlots ids each.
static int sort_log_groups(int64_t V) {
  int lg = 8;
  while (((V + (int64_t(1) << lg) - 1) >> lg) > kMaxSlots) ++lg;
  return lg;
}

// Tokens a block of embed_grad: 64, or fewer while there would be less than 4096
// waves of 512 columns (16 a CU).
static int embed_block(int64_t T, int64_t h) {
  int blk = 64;
  while (blk > 8 && (T + blk - 1) / blk * ((h + 511) / 512) < 4096) blk >>= 1;
  return blk;
}
static int64_t embed_blocks(int64_t T, int64_t h) {
  const int blk = embed_block(T, h);
  return (T + blk - 1) / blk;
}
static Columns columns(int64_t h) {
  const int64_t chunks = (h + 7) / 8;
  int lanes = 64;
  if (h % 8 != 0)
    while (chunks > lanes && chunks % lanes == 1) --lanes;
  return Columns{lanes, static_cast<int>((chunks + lanes - 1) / lanes)};
}
static int64_t pad_to(int64_t n, int64_t m) { return (n + m - 1) / m * m; }
// Floats of a partial row: two of them are an odd number of 256-byte units, so
// that the parts of one column, which embed_join reads together, lie in all of
// the memory's channels.
static int64_t part_row(int64_t h) { return ((h + 31) / 32 | 1) * 32; }

// Workspace: the partial sums, the spans, the grouped tokens, the counts, the total.
static int64_t embed_ws_bytes(int64_t T, int64_t V, int64_t h) {
  if (T <= kFew) return 0;
  return embed_blocks(T, h) * (2 * part_row(h) * 4 + 16) + pad_to(T * 8, 16) +
         pad_to(V * 4, 16) + 16;
}

// Every launch stays below 2^32 threads, 2^24 workgroups of the gradient: its
// blocks of 64 tokens are less than 2^23, the waves of its sums less than 2^25.3
// (a slice is 488 columns or more), 2^23.3 workgroups of four, and those that
// fill 2^22 and one.
static constexpr int64_t kMaxFills = int64_t(1) << 22;
static bool embed_sizes_ok(int64_t T, int64_t V, int64_t h) {
  return T >= 0 && T < (int64_t(1) << 29) && V > 0 && V < (int64_t(1) << 28) && h > 0 &&
         h < (int64_t(1) << 23) && T * h < (int64_t(1) << 40);
}

// Rows that a filling workgroup looks at, up to a wave's lanes: 8 KB of rows
// above 4 KB, 16 KB of shorter ones, less while there would be less than 1024
// workgroups, more while there would be more than kMaxFills (64 rows always do:
// vocab < 2^28).  us of the whole gradient at 8 / 16 / 64 KB: 4096 tokens, 49152 rows
// of 8 KB 83 / 91 / 98, 16312 tokens, 32000 rows of 4 KB 60.5 / 58.3 / 60.7, 8192
// tokens, 32000 rows of 2 KB 32.1 / 30.7 / 30.9.
static Fill rows_to_fill(int64_t V, int64_t row_bytes) {
  const int64_t most = row_bytes > 4096 ? 8192 : 16384;
  Fill f{64, 0};
  while (f.rows > 1 && (f.rows * row_bytes > most || V / f.rows < 1024)) f.rows >>= 1;
  while (V / f.rows > kMaxFills) f.rows <<= 1;
  while (f.log_tpr < 8 && (int64_t(16) << f.log_tpr) < row_bytes) ++f.log_tpr;
  return f;
}

template <typename I, typename W>
static void launch_fwd(const void* ids, int64_t T, const void* w, int64_t V, int64_t h, void* y,
                       int ydt, float scale, hipStream_t st) {
  int lt = 0;
  while (lt < 8 && (int64_t(8) << lt) < h) ++lt;
  const int64_t wgs = (T + (256 >> lt) - 1) >> (8 - lt);
  const dim3 grid(static_cast<unsigned>(wgs < (1 << 22) ? wgs : 1 << 22));
#define ZK_E(Y)                                                                              \
  hipLaunchKernelGGL((embed_fwd<I, W, Y>), grid, dim3(256), 0, st, (const I*)ids, T,         \
                     (const W*)w, V, static_cast<int>(h), (Y*)y, scale, lt)
  if (ydt == ZK_F32) ZK_E(float);
  else if (ydt == ZK_BF16) ZK_E(bf16);
  else ZK_E(f16);
#undef ZK_E
}

template <typename I>
static void launch_fwd_w(const void* ids, int64_t T, const void* w, int wdt, int64_t V, int64_t h,
                         void* y, int ydt, float scale, hipStream_t st) {
  if (wdt == ZK_F32) launch_fwd<I, float>(ids, T, w, V, h, y, ydt, scale, st);
  else if (wdt == ZK_BF16) launch_fwd<I, bf16>(ids, T, w, V, h, y, ydt, scale, st);
  else launch_fwd<I, f16>(ids, T, w, V, h, y, ydt, scale, st);
}

template <typename D, typename W, bool kAdd>
static void launch_few(const void* ids, int ids_64, int64_t T, const void* dy, void* dw, int64_t V,
                       int64_t h, float scale, uint32_t pad, hipStream_t st) {
  const Columns cols = columns(h);
  const Fill fill = rows_to_fill(V, h * static_cast<int64_t>(sizeof(W)));
  const dim3 grid(static_cast<unsigned>((T * cols.slices + 3) / 4 +
                                        (kAdd ? 0 : (V + fill.rows - 1) / fill.rows)));
#define ZK_FEW(I)                                                                                \
  hipLaunchKernelGGL((embed_few<I, D, W, kAdd>), grid, dim3(256), 0, st, (const I*)ids,          \
                     static_cast<int>(T), (const D*)dy, (W*)dw, static_cast<uint32_t>(V),        \
                     static_cast<int>(h), cols, fill, scale, pad)
  if (ids_64) ZK_FEW(int64_t); else ZK_FEW(int32_t);
#undef ZK_FEW
}

template <typename D, typename W, bool kAdd>
static void launch_grad(const void* dy, void* dw, const Token* tok, const int* count,
                        const int* total, float* part, Span* span, int64_t T, int64_t V,
                        int64_t h, float scale, hipStream_t st) {
  const int hp = static_cast<int>(part_row(h));
  const Columns cols = columns(h);
  const int blk = embed_block(T, h);
  const int64_t blocks = embed_blocks(T, h), sums = blocks * cols.slices;
  const Fill fill = rows_to_fill(V, h * static_cast<int64_t>(sizeof(W)));
  const dim3 grid(static_cast<unsigned>((sums + 3) / 4 + (kAdd ? 0 : (V + fill.rows - 1) / fill.rows)));
#define ZK_GRAD(S)                                                                            \
  hipLaunchKernelGGL((embed_grad<D, W, kAdd, S>), grid, dim3(256), 0, st, (const D*)dy, (W*)dw, \
                     tok, count, total, part, span, V, static_cast<int>(h), hp, cols, blk, sums, fill, \
                     scale)
  // dy within the 256 MB of last-level cache may still be there from the kernel
  // that wrote it.  us with streaming loads / ordinary ones: 65536 tokens of
  // 5120 (671 MB), a text's ids 337 / 348, nine tenths one id 361 / 427; 8192 of
  // 1000 (16 MB, fresh) 35 / 31, 4096 of 4096 (34 MB) 94 / 92
  const bool stream = T * h * static_cast<int64_t>(sizeof(D)) > (int64_t(1) << 28);
  if (grid.x > 0) {
    if (stream) ZK_GRAD(true); else ZK_GRAD(false);
  }
#undef ZK_GRAD
  if (blocks > 1)
    hipLaunchKernelGGL((embed_join<W, kAdd>),
                       dim3(static_cast<unsigned>((blocks - 1 + kJoinWaves - 1) / kJoinWaves),
                            static_cast<unsigned>((h + 255) / 256)),
                       dim3(64 * kJoinWaves), 0, st, (W*)dw, span, part, blocks - 1,
                       static_cast<int>(h), hp, scale);
}

}  // namespace zk

using namespace zk;

extern "C" int zk_embedding_fwd(const void* ids, int ids_64, int64_t tokens, const void* w,
                                int64_t vocab, int64_t hidden, void* y, float scale, int w_dtype,
                                int y_dtype, zk_stream_t stream) {
  ZK_REQUIRE(valid_dtype(w_dtype) && valid_dtype(y_dtype), ZK_EDTYPE,
             "zk_embedding_fwd: bad dtype (%d, %d)", w_dtype, y_dtype);
  ZK_REQUIRE(embed_sizes_ok(tokens, vocab, hidden), ZK_EINVAL,
             "zk_embedding_fwd: bad size (%lld tokens, table %lld x %lld)", (long long)tokens,
             (long long)vocab, (long long)hidden);
  if (tokens == 0) return ZK_OK;
  ZK_REQUIRE(ids && w && y, ZK_EINVAL, "zk_embedding_fwd: null pointer");
  ZK_REQUIRE(aligned(ids, ids_64 ? 8 : 4) && aligned(w, dtype_bytes(w_dtype)) &&
                 aligned(y, dtype_bytes(y_dtype)),
             ZK_EALIGN, "zk_embedding_fwd: tensors must be aligned to their element size");
  hipStream_t st = as_stream(stream);
  if (ids_64) launch_fwd_w<int64_t>(ids, tokens, w, w_dtype, vocab, hidden, y, y_dtype, scale, st);
  else launch_fwd_w<int32_t>(ids, tokens, w, w_dtype, vocab, hidden, y, y_dtype, scale, st);
  return launch_status("zk_embedding_fwd");
}

extern "C" int64_t zk_embedding_bwd_workspace(int64_t tokens, int64_t vocab, int64_t hidden) {
  if (!embed_sizes_ok(tokens, vocab, hidden)) return -1;
  return embed_ws_bytes(tokens, vocab, hidden);
}

extern "C" int zk_embedding_bwd(const void* ids, int ids_64, int64_t tokens, const void* dy,
                                int dy_dtype, void* dw, int dw_dtype, int64_t vocab,
                                int64_t hidden, float scale, int64_t padding_idx, int accumulate,
                                void* workspace, int64_t workspace_bytes, zk_stream_t stream) {
  ZK_REQUIRE(valid_dtype(dy_dtype) && valid_dtype(dw_dtype), ZK_EDTYPE,
             "zk_embedding_bwd: bad dtype (%d, %d)", dy_dtype, dw_dtype);
  ZK_REQUIRE(embed_sizes_ok(tokens, vocab, hidden), ZK_EINVAL,
             "zk_embedding_bwd: bad size (%lld tokens, table %lld x %lld)", (long long)tokens,
             (long long)vocab, (long long)hidden);
  if (tokens == 0 && accumulate) return ZK_OK;
  const int64_t needed = embed_ws_bytes(tokens, vocab, hidden);
  ZK_REQUIRE((tokens == 0 || (ids && dy)) && dw && (needed == 0 || workspace), ZK_EINVAL,
             "zk_embedding_bwd: null pointer");
  ZK_REQUIRE(aligned(ids, ids_64 ? 8 : 4) && aligned(dy, dtype_bytes(dy_dtype)) &&
                 aligned(dw, dtype_bytes(dw_dtype)) && aligned(workspace, 16),
             ZK_EALIGN, "zk_embedding_bwd: tensors must be aligned to their element size, the "
             "workspace to 16 bytes");
  ZK_REQUIRE(workspace_bytes >= needed, ZK_EWORKSPACE,
             "zk_embedding_bwd: workspace of %lld bytes, %lld needed", (long long)workspace_bytes,
             (long long)needed);
  hipStream_t st = as_stream(stream);
  const uint32_t pad = padding_idx >= 0 && padding_idx < vocab ? static_cast<uint32_t>(padding_idx) : ~0u;
#define ZK_DTYPES(ZK_G)                            \
  do {                                             \
    if (dy_dtype == ZK_F32) ZK_DW(ZK_G, float);    \
    else if (dy_dtype == ZK_BF16) ZK_DW(ZK_G, bf16); \
    else ZK_DW(ZK_G, f16);                         \
  } while (0)
#define ZK_DW(ZK_G, D)                             \
  do {                                             \
    if (dw_dtype == ZK_F32) ZK_G(D, float);        \
    else if (dw_dtype == ZK_BF16) ZK_G(D, bf16);   \
    else ZK_G(D, f16);                             \
  } while (0)
  if (tokens <= kFew) {
#define ZK_G(D, W)                                                                               \
  do {                                                                                           \
    if (accumulate) launch_few<D, W, true>(ids, ids_64, tokens, dy, dw, vocab, hidden, scale, pad, st); \
    else launch_few<D, W, false>(ids, ids_64, tokens, dy, dw, vocab, hidden, scale, pad, st);    \
  } while (0)
    ZK_DTYPES(ZK_G);
#undef ZK_G
    return launch_status("zk_embedding_bwd");
  }
  char* ws = static_cast<char*>(workspace);
  float* part = reinterpret_cast<float*>(ws);
  ws += embed_blocks(tokens, hidden) * 2 * part_row(hidden) * 4;
  Span* span = reinterpret_cast<Span*>(ws);
  ws += embed_blocks(tokens, hidden) * 16;
  Token* tok = reinterpret_cast<Token*>(ws);
  ws += pad_to(tokens * 8, 16);
  int* count = reinterpret_cast<int*>(ws);
  ws += pad_to(vocab * 4, 16);
  int* total = reinterpret_cast<int*>(ws);
  const int lg = sort_log_groups(vocab);
  const int slots = static_cast<int>((vocab + (int64_t(1) << lg) - 1) >> lg);
  const dim3 grid(1u << lg), block(64 * kSortWaves);
  const size_t lds = sizeof(int) * kSortWaves * slots;
  if (ids_64)
    hipLaunchKernelGGL((embed_sort<int64_t>), grid, block, lds, st, (const int64_t*)ids,
                       static_cast<int>(tokens), static_cast<uint32_t>(vocab), lg, slots, pad, tok,
                       count, total);
  else
    hipLaunchKernelGGL((embed_sort<int32_t>), grid, block, lds, st, (const int32_t*)ids,
                       static_cast<int>(tokens), static_cast<uint32_t>(vocab), lg, slots, pad, tok,
                       count, total);
#define ZK_G(D, W)                                                                               \
  do {                                                                                           \
    if (accumulate) launch_grad<D, W, true>(dy, dw, tok, count, total, part, span, tokens, vocab, hidden, scale, st); \
    else launch_grad<D, W, false>(dy, dw, tok, count, total, part, span, tokens, vocab, hidden, scale, st); \
  } while (0)
  ZK_DTYPES(ZK_G);
#undef ZK_G
#undef ZK_DW
#undef ZK_DTYPES
  return launch_status("zk_embedding_bwd");
}
