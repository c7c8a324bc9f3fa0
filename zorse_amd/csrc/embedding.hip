// Token embedding: y[t] = round(s W[id_t]), and its gradient
// dW[r] = round(s sum_{t: id_t = r} dy[t]) (+ dW[r]).
//
// Both move rows and hardly compute: HBM bounds them.  The gradient's sums
// are taken in the order of the tokens, in fp32, without atomics, so that a
// repeated pass gives the same bits.  Three launches:
//   1. embed_sort: the tokens grouped by id (stable), and each id's count.
//      Workgroup g of G (a power of two) owns the ids with id mod G = g, so
//      that the frequent low ids of a text spread over all of them.  It reads
//      every id twice: once to count its own ids and the tokens of the groups
//      before it -- its offset, so no workgroup waits for another -- and once
//      to place its tokens.  For the stable order each of 16 waves owns a
//      sixteenth of the tokens and a row of counters in LDS.
//   2. embed_grad: the grouped tokens in blocks of kBlock, one wave for each
//      block and 512 columns, whatever the ids: a token that fills half the
//      batch costs no more than many single ones.  An id whose tokens lie in
//      one block is finished there; of one that crosses blocks, each block
//      leaves a partial sum (at most two a block: the id it begins with and
//      the id it ends in).  Waves after those write the rows of unused ids.
//   3. embed_join: the partial sums of ids that cross blocks.
#include "part8.h"

namespace zk {

static constexpr int kSortWaves = 16;
static constexpr int kMaxSlots = 512;   // ids a sort workgroup owns: 32 KB of counters
static constexpr int kBlock = 64;       // grouped tokens a gradient wave sums (one a lane)
static constexpr int kFillRows = 8;     // table rows a filling wave looks at

struct Token {
  int t, id;
};

// ---------------------------------------------------------------- forward ---
// tpr (a power of two up to 256) threads a row, 8 elements each at a time.
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
template <typename I>
__global__ __launch_bounds__(64 * kSortWaves) void embed_sort(
    const I* __restrict__ ids, int T, int64_t V, int log_g, int slots, int64_t pad,
    Token* __restrict__ out, int* __restrict__ count, int* __restrict__ total) {
  extern __shared__ int cnt[];  // [kSortWaves][slots]
  __shared__ int red[kSortWaves], run[kSortWaves];
  const int g = blockIdx.x, groups = 1 << log_g;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  for (int i = threadIdx.x; i < kSortWaves * slots; i += 64 * kSortWaves) cnt[i] = 0;
  __syncthreads();
  const int per = (T + 64 * kSortWaves - 1) / (64 * kSortWaves) * 64;
  const int64_t t0 = static_cast<int64_t>(wave) * per;
  const int t1 = static_cast<int>(t0 + per < T ? t0 + per : T);
  int* mine = cnt + wave * slots;
  // the group of a token, or `groups` for one that has no gradient
  auto group = [&](int64_t id) {
    return id >= 0 && id < V && id != pad ? static_cast<int>(id & (groups - 1)) : groups;
  };
  int before = 0;
#pragma unroll 4
  for (int64_t t = t0 + lane; t < t1; t += 64) {
    const int64_t id = ids[t];
    const int gi = group(id);
    before += gi < g;
    if (gi == g) atomicAdd(mine + static_cast<int>(id >> log_g), 1);
  }
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) before += __shfl_xor(before, off, 64);
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
  if (g == groups - 1 && i == 0) *total = base + all;
  if (i < slots) {
    int at = base + prior + incl - n;
    for (int k = 0; k < kSortWaves; ++k) {
      const int c = cnt[k * slots + i];
      cnt[k * slots + i] = at;
      at += c;
    }
    const int64_t id = (static_cast<int64_t>(i) << log_g) + g;
    if (id < V) count[id] = n;
  }
  __syncthreads();
  // place: 64 tokens at a time, the lanes of one id after another; a wave's
  // counters are its own, and its LDS accesses (volatile) are in order
  volatile int* next = mine;
  for (int64_t tb = t0; tb < t1; tb += 64) {
    const int64_t t = tb + lane;
    const int64_t id = t < t1 ? static_cast<int64_t>(ids[t]) : -1;
    unsigned long long left = __ballot(group(id) == g);
    while (left != 0) {
      const int lead = __builtin_ctzll(left);
      const int key = __builtin_amdgcn_readlane(static_cast<int>(id), lead);
      const bool same = ((left >> lane) & 1) != 0 && static_cast<int>(id) == key;
      const unsigned long long m = __ballot(same);
      const int slot = key >> log_g;
      const int at = next[slot];
      if (same) out[at + __popcll(m & ((1ull << lane) - 1))] = Token{static_cast<int>(t), key};
      if (lane == lead) next[slot] = at + __popcll(m);
      left &= ~m;
    }
  }
}

// --------------------------------------------------------------- gradient ---
template <typename W>
__device__ __forceinline__ void put_row(W* p, const float (&acc)[8], int n, float scale,
                                        bool accumulate) {
  float o[8];
  if (accumulate) {
    Part8<W> old;
    old.load(p, n);
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = old[i] + scale * acc[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = scale * acc[i];
  }
  Part8<W>::store(p, o, n);
}

__device__ __forceinline__ void put_part(float* p, const float (&acc)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(acc[0], acc[1], acc[2], acc[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
}

// part: [blocks][2][hp] fp32 (hp = h rounded up to 8): the sum of the id that
// a block begins with and of the one that it ends in, where they reach over
// its border (an id that does both: the first).
template <typename D, typename W>
__global__ __launch_bounds__(256) void embed_grad(
    const D* __restrict__ dy, W* __restrict__ dw, const Token* __restrict__ tok,
    const int* __restrict__ count, const int* __restrict__ total, float* __restrict__ part,
    int64_t V, int h, int hp, int slices, int64_t sum_items, float scale, bool accumulate) {
  const int lane = threadIdx.x & 63;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * 4 +
                       __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (item >= sum_items) {  // rows of ids without tokens
    if (accumulate) return;  // (a wave that rounds the last workgroup up)
    const int64_t r0 = (item - sum_items) * kFillRows;
    const float zero[8] = {};
    for (int64_t r = r0; r < r0 + kFillRows && r < V; ++r) {
      if (count[r] != 0) continue;
      for (int c = lane * 8; c < h; c += 512) Part8<W>::store(dw + r * h + c, zero, h - c);
    }
    return;
  }
  const int64_t j = item / slices;
  const int c = static_cast<int>(item - j * slices) * 512 + lane * 8;
  const int n_all = *total;
  const int64_t p0 = j * kBlock;
  if (p0 >= n_all) return;
  const int n = n_all - p0 < kBlock ? static_cast<int>(n_all - p0) : kBlock;
  const Token e = lane < n ? tok[p0 + lane] : Token{0, -1};
  const int prev = p0 > 0 ? tok[p0 - 1].id : -1;
  const int next = p0 + n < n_all ? tok[p0 + n].id : -1;
  const int nc = h - c;  // columns from here on
  float acc[8] = {};
  int cur = __builtin_amdgcn_readlane(e.id, 0);
  bool head = cur == prev;
  float* pj = part + j * 2 * hp + c;
  constexpr int kAhead = 8;
  for (int i0 = 0; i0 < n; i0 += kAhead) {
    Part8<D> x[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int64_t t = __builtin_amdgcn_readlane(e.t, (i0 + k) & 63);
      if (i0 + k < n && nc > 0) x[k].load(dy + t * h + c, nc);
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      if (i0 + k >= n) break;
      const int id = __builtin_amdgcn_readlane(e.id, (i0 + k) & 63);
      if (id != cur) {
        if (nc > 0) {
          if (head) put_part(pj, acc);
          else put_row(dw + static_cast<int64_t>(cur) * h + c, acc, nc, scale, accumulate);
        }
        head = false;
        cur = id;
#pragma unroll
        for (int q = 0; q < 8; ++q) acc[q] = 0.f;
      }
      if (nc > 0) {
#pragma unroll
        for (int q = 0; q < 8; ++q) acc[q] += x[k][q];
      }
    }
  }
  if (nc <= 0) return;
  if (head) put_part(pj, acc);
  else if (cur == next) put_part(pj + hp, acc);
  else put_row(dw + static_cast<int64_t>(cur) * h + c, acc, nc, scale, accumulate);
}

// Block j's last id, if it begins there and crosses into the next block: its
// partial sums of all blocks, in order, 256 columns a workgroup.  Four waves
// take a quarter of the blocks each.
template <typename W>
__global__ __launch_bounds__(256) void embed_join(
    W* __restrict__ dw, const Token* __restrict__ tok, const int* __restrict__ count,
    const int* __restrict__ total, const float* __restrict__ part, int h, int hp, float scale,
    bool accumulate) {
  const int64_t j = blockIdx.x, p1 = (j + 1) * kBlock;
  if (p1 >= *total) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int id = tok[p1].id;
  const int mine = tok[p1 - kBlock + lane].id;
  const unsigned long long same = __ballot(mine == id);
  if (same == 0) return;  // no id crosses this border
  const int64_t start = p1 - __popcll(same);  // grouped: the lanes of an id are the last ones
  if (start == p1 - kBlock && start > 0 && tok[start - 1].id == id) return;  // began earlier
  const int64_t last = (start + count[id] - 1) / kBlock;
  const int64_t parts = last - j + 1;  // the first from block j's end, the others' beginnings
  const int c = blockIdx.y * 256 + lane * 4;
  const int64_t a = parts * wave / 4, b = parts * (wave + 1) / 4;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  if (c < hp) {
#pragma unroll 8
    for (int64_t k = a; k < b; ++k) {
      const float* p = part + (j + k) * 2 * hp + (k == 0 ? hp : 0) + c;
      const float4 x = *reinterpret_cast<const float4*>(p);
      acc.x += x.x; acc.y += x.y; acc.z += x.z; acc.w += x.w;
    }
  }
  __shared__ float4 sums[4][64];
  sums[wave][lane] = acc;
  __syncthreads();
  if (wave != 0 || c >= h) return;
#pragma unroll
  for (int k = 1; k < 4; ++k) {
    const float4 x = sums[k][lane];
    acc.x += x.x; acc.y += x.y; acc.z += x.z; acc.w += x.w;
  }
  const float v[8] = {acc.x, acc.y, acc.z, acc.w, 0.f, 0.f, 0.f, 0.f};
  put_row(dw + static_cast<int64_t>(id) * h + c, v, h - c < 4 ? h - c : 4, scale, accumulate);
}

// The groups of embed_sort: at least 256 workgroups, at most kMaxSlots ids each.
static int sort_log_groups(int64_t V) {
  int lg = 8;
  while (((V + (int64_t(1) << lg) - 1) >> lg) > kMaxSlots) ++lg;
  return lg;
}

static int64_t embed_blocks(int64_t T) { return (T + kBlock - 1) / kBlock; }
static int64_t pad_to(int64_t n, int64_t m) { return (n + m - 1) / m * m; }

// Workspace: the partial sums, the grouped tokens, the counts, the total.
static int64_t embed_ws_bytes(int64_t T, int64_t V, int64_t h) {
  return embed_blocks(T) * 2 * pad_to(h, 8) * 4 + pad_to(T * 8, 16) + pad_to(V * 4, 16) + 16;
}

static bool embed_sizes_ok(int64_t T, int64_t V, int64_t h) {
  // every launch stays below 2^32 threads
  return T >= 0 && T < (int64_t(1) << 29) && V > 0 && V < (int64_t(1) << 28) && h > 0 &&
         h < (int64_t(1) << 23);
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

template <typename D, typename W>
static void launch_grad(const void* dy, void* dw, const Token* tok, const int* count,
                        const int* total, float* part, int64_t T, int64_t V, int64_t h,
                        float scale, bool accumulate, hipStream_t st) {
  const int hp = static_cast<int>(pad_to(h, 8)), slices = static_cast<int>((h + 511) / 512);
  const int64_t blocks = embed_blocks(T), sums = blocks * slices;
  const int64_t items = sums + (accumulate ? 0 : (V + kFillRows - 1) / kFillRows);
  if (items > 0)
    hipLaunchKernelGGL((embed_grad<D, W>), dim3(static_cast<unsigned>((items + 3) / 4)), dim3(256),
                       0, st, (const D*)dy, (W*)dw, tok, count, total, part, V,
                       static_cast<int>(h), hp, slices, sums, scale, accumulate);
  if (blocks > 1)
    hipLaunchKernelGGL((embed_join<W>),
                       dim3(static_cast<unsigned>(blocks - 1), static_cast<unsigned>((h + 255) / 256)),
                       dim3(256), 0, st, (W*)dw, tok, count, total, part, static_cast<int>(h), hp,
                       scale, accumulate);
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
  ZK_REQUIRE((tokens == 0 || (ids && dy)) && dw && workspace, ZK_EINVAL,
             "zk_embedding_bwd: null pointer");
  ZK_REQUIRE(aligned(ids, ids_64 ? 8 : 4) && aligned(dy, dtype_bytes(dy_dtype)) &&
                 aligned(dw, dtype_bytes(dw_dtype)) && aligned(workspace, 16),
             ZK_EALIGN, "zk_embedding_bwd: tensors must be aligned to their element size, the "
             "workspace to 16 bytes");
  ZK_REQUIRE(workspace_bytes >= embed_ws_bytes(tokens, vocab, hidden), ZK_EWORKSPACE,
             "zk_embedding_bwd: workspace of %lld bytes, %lld needed", (long long)workspace_bytes,
             (long long)embed_ws_bytes(tokens, vocab, hidden));
  char* ws = static_cast<char*>(workspace);
  float* part = reinterpret_cast<float*>(ws);
  ws += embed_blocks(tokens) * 2 * pad_to(hidden, 8) * 4;
  Token* tok = reinterpret_cast<Token*>(ws);
  ws += pad_to(tokens * 8, 16);
  int* count = reinterpret_cast<int*>(ws);
  ws += pad_to(vocab * 4, 16);
  int* total = reinterpret_cast<int*>(ws);
  const int lg = sort_log_groups(vocab);
  const int slots = static_cast<int>((vocab + (int64_t(1) << lg) - 1) >> lg);
  hipStream_t st = as_stream(stream);
  const dim3 grid(1u << lg), block(64 * kSortWaves);
  const size_t lds = sizeof(int) * kSortWaves * slots;
  if (ids_64)
    hipLaunchKernelGGL((embed_sort<int64_t>), grid, block, lds, st, (const int64_t*)ids,
                       static_cast<int>(tokens), vocab, lg, slots, padding_idx, tok, count, total);
  else
    hipLaunchKernelGGL((embed_sort<int32_t>), grid, block, lds, st, (const int32_t*)ids,
                       static_cast<int>(tokens), vocab, lg, slots, padding_idx, tok, count, total);
#define ZK_G(D, W) \
  launch_grad<D, W>(dy, dw, tok, count, total, part, tokens, vocab, hidden, scale, accumulate != 0, st)
#define ZK_GW(D)                             \
  do {                                       \
    if (dw_dtype == ZK_F32) ZK_G(D, float);  \
    else if (dw_dtype == ZK_BF16) ZK_G(D, bf16); \
    else ZK_G(D, f16);                       \
  } while (0)
  if (dy_dtype == ZK_F32) ZK_GW(float);
  else if (dy_dtype == ZK_BF16) ZK_GW(bf16);
  else ZK_GW(f16);
#undef ZK_GW
#undef ZK_G
  return launch_status("zk_embedding_bwd");
}
