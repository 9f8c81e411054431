// Token lookup with a scale, and its gradient by sorted tokens.
//
//   out[t, :]  = s W[id_t, :]                                  (ids outside [0, V): a zero row)
//   dW[r, :]   = s sum_{t : id_t = r, r != padding_idx} dout[t, :]     (every row written)
//
// Both move bytes and add: the forward reads each token's row (repeated rows from L2) and writes
// n E elements, the backward reads n E elements once and writes V E.  8192 x 64 text-like tokens, half of them
// padding, 200k x 256 fp32: forward 152 us (537 MB written, 128 MB read from memory; 86 us without the reads, 44
// without the writes, and 152-161 for 1 to 16 tokens in flight, stores past the caches or not), sort 40 us, tiles
// 70 us (344 MB, 4.9 TB/s), joins and empty rows 42 us (148 MB); a 4 GiB copy runs at 4.8 TB/s.  The backward needs each
// row's tokens together: a long call sorts them (the bags' stable counting sort, token_plan_build), a short one
// lets every workgroup pick the tokens of its own rows from the ids.
#include "common.hpp"

namespace tt {
namespace {

constexpr int kBlock = 256;
constexpr int kWavesPerBlock = kBlock / kWave;

__device__ __forceinline__ int64_t id_at(const void* ids, bool wide, int64_t i) {
  return wide ? static_cast<const int64_t*>(ids)[i] : (int64_t)static_cast<const int32_t*>(ids)[i];
}

// log2 of the lanes that hold one row: the smallest power of two covering its E / VEC accesses.
inline int row_lanes_log2(int E, int vec) {
  int l = 0;
  while (l < 6 && (vec << l) < E) ++l;
  return l;
}

// ---- forward: a group of 2^lg lanes per token, U tokens in flight per group.  A long call deals its
// workgroups to the XCDs (workgroup b runs on XCD b mod 8) in runs of kXcdRun consecutive ones, 1 MB of output
// at 16 KB a workgroup: 152 us instead of 162 at 8192 x 64 rows of 1 KB (runs of 8: 155, an eighth of the
// output to each: 157).
constexpr int kXcdRun = 64;
template <typename TW, typename TO, int VEC, int U>
__global__ __launch_bounds__(kBlock) void lookup_fwd_kernel(const TW* __restrict__ table, int64_t V, int E, int64_t ld,
                                                            const void* __restrict__ ids, bool wide, int64_t n,
                                                            float scale, TO* __restrict__ out, int lg, bool runs) {
  const int lane = lane_id(), groups = kWave >> lg, sub = lane >> lg, c = lane & ((1 << lg) - 1);
  int64_t block = block_index();
  if (runs) {  // (the grid is whole spans of 8 kXcdRun workgroups)
    const int in = (int)(block % (8 * kXcdRun));
    block += (in & 7) * kXcdRun + (in >> 3) - in;
  }
  const int64_t wave = block * kWavesPerBlock + (threadIdx.x >> 6);
  const int64_t t0 = wave * groups * U + sub;
  int64_t id[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t t = t0 + (int64_t)u * groups;
    id[u] = t < n ? id_at(ids, wide, t) : -1;
  }
  for (int e = c * VEC; e < E; e += VEC << lg) {
    float x[U][VEC];
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) x[u][i] = 0.f;
      if (id[u] >= 0 && id[u] < V) load_elems<VEC>(table + id[u] * ld + e, x[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t t = t0 + (int64_t)u * groups;
      if (t < n) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) x[u][i] = (id[u] >= 0 && id[u] < V) ? scale * x[u][i] : 0.f;
        store_elems_nt<VEC>(out + t * E + e, x[u]);
      }
    }
  }
}

// ---- gradient of a short call (n <= kDirectN): one launch, no workspace.  A workgroup owns R
// consecutive rows; it reads all ids, keeps its own tokens in LDS in token order, and a wave per
// row adds that row's tokens.  A row with more than kCoop tokens is shared by the workgroup's waves,
// each adding the tokens of its part of the list, folded in wave order.  Its time grows with n V (every
// workgroup reads all ids), the sorted form's hardly at all, and about kDirectN they meet (us, n = 1000 / 4000 /
// 8000): 34 x 64 9 / 19 / 32 against 25 / 29 / 32; 2000 x 256 10 / 17 / 26 against 40 / 45 / 45; 50k x 128 21 / 40 /
// 80 against 41 / 47 / 49; 200k x 256 47 / 80 / 150 against 71 / 79 / 80 (30 us of it the bytes of the gradient).
constexpr int kDirectN = TT_LOOKUP_DIRECT_TOKENS;
constexpr int kDirectThreads = 512;
constexpr int kDirectWaves = kDirectThreads / kWave;
constexpr int kDirectRows = 64;
constexpr int kCoop = 64;

// acc += the rows of dout named by list[beg, end) whose local row is r, in list order
template <typename TO, int VEC>
__device__ __forceinline__ void direct_add(const TO* __restrict__ dout, int E, int e, bool on,
                                           const uint32_t* list, int beg, int end, int r, float (&acc)[VEC]) {
  constexpr int U = 8;
  const int lane = lane_id();
  for (int b = beg; b < end; b += kWave) {
    const uint32_t v = b + lane < end ? list[b + lane] : 0xffffffffu;
    uint64_t m = __ballot((int)(v & 255u) == r);
    while (m) {
      int64_t tok[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        tok[u] = m ? (int64_t)(__builtin_amdgcn_readlane((int)v, __builtin_ctzll(m)) >> 8) : -1;
        m &= m - 1;  // (0 stays 0)
      }
      float x[U][VEC];  // (filled before the first is used: loaded and added under one condition they ran one by one)
#pragma unroll
      for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) x[u][i] = 0.f;
        if (on && tok[u] >= 0) load_elems<VEC>(dout + tok[u] * E + e, x[u]);
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (tok[u] >= 0) {
#pragma unroll
          for (int i = 0; i < VEC; ++i) acc[i] += x[u][i];
        }
    }
  }
}

template <typename TO, typename TW, int VEC>
__global__ __launch_bounds__(kDirectThreads) void lookup_grad_direct_kernel(
    const TO* __restrict__ dout, const void* __restrict__ ids, bool wide, int n, int64_t V, int E, int R, int64_t pad,
    float scale, TW* __restrict__ grad) {
  __shared__ uint32_t list[kDirectN];  // token << 8 | local row
  __shared__ int cnt[kDirectRows];
  __shared__ int wcnt[kDirectWaves];
  __shared__ float part[kDirectWaves][kWave * VEC];
  const int lane = lane_id(), w = threadIdx.x >> 6;
  const int64_t r0 = block_index() * R;
  if (r0 >= V) return;
  const int rows = (int)(V - r0 < R ? V - r0 : R);
  if (threadIdx.x < kDirectRows) cnt[threadIdx.x] = 0;
  int m = 0;  // tokens kept so far (the same in every thread)
  __syncthreads();
  for (int base = 0; base < n; base += kDirectThreads) {
    const int i = base + threadIdx.x;
    const int64_t id = i < n ? id_at(ids, wide, i) : -1;
    const bool mine = id >= r0 && id < r0 + rows && id != pad;
    const uint64_t b = __ballot(mine);
    if (lane == 0) wcnt[w] = __popcll(b);
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int k = 0; k < kDirectWaves; ++k) {
      before += k < w ? wcnt[k] : 0;
      all += wcnt[k];
    }
    if (mine) {
      const int local = (int)(id - r0);
      list[m + before + __popcll(b & ((uint64_t(1) << lane) - 1))] = (uint32_t)i << 8 | (uint32_t)local;
      atomicAdd(&cnt[local], 1);
    }
    m += all;
    __syncthreads();
  }
  for (int r = w; r < rows; r += kDirectWaves) {
    const int c = cnt[r];
    if (c > kCoop) continue;
    for (int e0 = 0; e0 < E; e0 += kWave * VEC) {
      const int e = e0 + lane * VEC;
      float acc[VEC] = {};
      if (c) direct_add<TO, VEC>(dout, E, e, e < E, list, 0, m, r, acc);
#pragma unroll
      for (int i = 0; i < VEC; ++i) acc[i] *= scale;
      if (e < E) store_elems<VEC>(grad + (r0 + r) * E + e, acc);
    }
  }
  const int share = (m + kDirectWaves - 1) / kDirectWaves;
  for (int r = 0; r < rows; ++r) {
    if (cnt[r] <= kCoop) continue;
    for (int e0 = 0; e0 < E; e0 += kWave * VEC) {
      const int e = e0 + lane * VEC;
      float acc[VEC] = {};
      direct_add<TO, VEC>(dout, E, e, e < E, list, min(w * share, m), min((w + 1) * share, m), r, acc);
#pragma unroll
      for (int i = 0; i < VEC; ++i) part[w][lane * VEC + i] = acc[i];
      __syncthreads();
      if (w == 0) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          float a = part[0][lane * VEC + i];
#pragma unroll
          for (int k = 1; k < kDirectWaves; ++k) a += part[k][lane * VEC + i];
          acc[i] = a * scale;
        }
        if (e < E) store_elems<VEC>(grad + (r0 + r) * E + e, acc);
      }
      __syncthreads();
    }
  }
}

// ---- gradient of a long call, from the sorted tokens.  The sorted order is cut into tiles of kTile tokens
// and a group of 2^lg lanes runs through each: every group has the same work and eight rows of dout in
// flight, whatever the rows' lengths.  A row whose tokens lie in one tile is finished there.  A row that
// crosses tiles leaves its sum in the first as that tile's `tail` and in each later one as its `head`, and
// the row pass adds them (runs of kSuper tiles of one row through their own sums); it also writes the
// rows without tokens.  (A group per row, its first tokens fetched at once, kept 1.4 rows of dout in flight:
// 1.7 TB/s, 132 us with the frequent rows' tiles at 8192 x 64 text-like tokens, 200k rows of 256 floats.)
constexpr int kTile = 32;
constexpr int kSuper = 32;

template <typename TO, typename TW, int VEC>
__global__ __launch_bounds__(kBlock) void lookup_tile_sum_kernel(TokenPlan p, const TO* __restrict__ dout, int E,
                                                                 float scale, TW* __restrict__ grad, int lg,
                                                                 float* __restrict__ head, float* __restrict__ tail) {
  constexpr int U = 8;
  const int64_t tile = ((int64_t)blockIdx.x * kBlock + threadIdx.x) >> lg;
  const int c = threadIdx.x & ((1 << lg) - 1);
  const int n = *p.count;
  if (tile * kTile >= n) return;
  const int lo = (int)(tile * kTile), hi = min(lo + kTile, n);
  const uint32_t first = p.keys[lo], last = p.keys[hi - 1];
  const bool before = lo > 0 && p.keys[lo - 1] == first, after = hi < n && p.keys[hi] == last;
  for (int e = c * VEC; e < E; e += VEC << lg) {
    float acc[VEC] = {};
    uint32_t cur = first;
    auto flush = [&](bool end) {
      if (cur == first && before) {
        store_elems<VEC>(head + tile * E + e, acc);
      } else if (end && after) {
        store_elems<VEC>(tail + tile * E + e, acc);
      } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[i] *= scale;
        store_elems_nt<VEC>(grad + (int64_t)cur * E + e, acc);
      }
#pragma unroll
      for (int i = 0; i < VEC; ++i) acc[i] = 0.f;
    };
    uint32_t key[U];
    int tok[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = min(lo + u, hi - 1);
      key[u] = p.keys[k];
      tok[u] = p.vals[k];
    }
    for (int k0 = lo; k0 < hi; k0 += U) {
      Elems<TO, VEC> x[U];
#pragma unroll
      for (int u = 0; u < U; ++u) x[u] = *reinterpret_cast<const Elems<TO, VEC>*>(dout + (int64_t)tok[u] * E + e);
      uint32_t now[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        now[u] = key[u];
        const int k = min(k0 + U + u, hi - 1);  // the next ones' names, while these are on their way
        key[u] = p.keys[k];
        tok[u] = p.vals[k];
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (k0 + u < hi) {
          if (now[u] != cur) {
            flush(false);
            cur = now[u];
          }
#pragma unroll
          for (int i = 0; i < VEC; ++i) acc[i] += (float)x[u].v[i];
        }
      }
    }
    flush(true);
  }
}

// sum of rows [beg, end) of part: U sums (row k to sum k % U), folded in order
template <int VEC>
__device__ __forceinline__ void part_add(const float* __restrict__ part, int E, int e, int64_t beg, int64_t end,
                                         float (&acc)[VEC]) {
  constexpr int U = 4;
  float s[U][VEC];
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int i = 0; i < VEC; ++i) s[u][i] = 0.f;
  for (int64_t k = beg; k < end; k += U) {
    float x[U][VEC];
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) x[u][i] = 0.f;
      if (k + u < end) load_elems<VEC>(part + (k + u) * E + e, x[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < VEC; ++i) s[u][i] += x[u][i];
  }
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int i = 0; i < VEC; ++i) acc[i] += s[u][i];
}

// sup[j] = the heads of tiles [kSuper j, kSuper (j + 1)) added, where one row runs through them all
template <int VEC>
__global__ __launch_bounds__(kBlock) void lookup_super_sum_kernel(TokenPlan p, const float* __restrict__ head, int E,
                                                                  int lg, float* __restrict__ sup) {
  const int64_t j = ((int64_t)blockIdx.x * kBlock + threadIdx.x) >> lg;
  const int c = threadIdx.x & ((1 << lg) - 1);
  const int64_t lo = j * kSuper * kTile, hi = lo + kSuper * kTile;
  if (lo == 0 || hi > *p.count || p.keys[lo - 1] != p.keys[hi - 1]) return;
  for (int e = c * VEC; e < E; e += VEC << lg) {
    float acc[VEC] = {};
    part_add<VEC>(head, E, e, j * kSuper, (j + 1) * kSuper, acc);
    store_elems<VEC>(sup + j * E + e, acc);
  }
}

// the first position in [lo, hi) of the ascending keys with keys[i] >= r, hi if there is none
__device__ __forceinline__ int first_at_least(const uint32_t* __restrict__ keys, int lo, int hi, uint32_t r) {
  while (lo < hi) {
    const int mid = lo + ((hi - lo) >> 1);
    if (keys[mid] < r) lo = mid + 1;
    else hi = mid;
  }
  return lo;
}

// What the tiles left to do: the first `join_blocks` workgroups add up the rows that cross tiles (a group per
// tile, for a row that leaves its first tile there; first, because the most frequent row is the longest
// chain), the others write the rows without tokens: a wave finds where kZeroRows rows would lie in the
// sorted order and stores those that do not (a group of lanes per row at a time), the stores following
// each other without a load between them.  (A table of the rows' starts, written from the keys, took one
// thread through every gap between two of them: 135 us for 8192 tokens in 200k rows.)
constexpr int kZeroRows = 32;
template <typename TW, int VEC>
__global__ __launch_bounds__(kBlock) void lookup_row_join_kernel(TokenPlan p, int64_t V, int E, float scale,
                                                                 TW* __restrict__ grad, int lg, unsigned join_blocks,
                                                                 const float* __restrict__ head,
                                                                 const float* __restrict__ tail,
                                                                 const float* __restrict__ sup) {
  const int c = threadIdx.x & ((1 << lg) - 1);
  const int n = *p.count;
  if (block_index() >= join_blocks) {
    const int64_t r0 = ((block_index() - join_blocks) * kWavesPerBlock + (threadIdx.x >> 6)) * kZeroRows;
    const int lane = lane_id(), groups = kWave >> lg;
    const int64_t r = r0 + (lane < kZeroRows ? lane : kZeroRows);
    const int at = first_at_least(p.keys, 0, n, (uint32_t)(r < V ? r : V));
    const int next = __shfl(at, lane < kZeroRows ? lane + 1 : kZeroRows);
    const uint64_t empty = __ballot(lane < kZeroRows && r < V && next == at);
    const float zero[VEC] = {};
    for (int i = lane >> lg; i < kZeroRows; i += groups)
      if (empty >> i & 1)
        for (int e = c * VEC; e < E; e += VEC << lg) store_elems_nt<VEC>(grad + (r0 + i) * E + e, zero);
    return;
  }
  const int64_t t0 = (block_index() * kBlock + threadIdx.x) >> lg;
  const int64_t next_tile = (t0 + 1) * kTile;
  if (next_tile >= n) return;  // no tile after it
  const uint32_t r = p.keys[next_tile];
  if (p.keys[next_tile - 1] != r) return;                                  // no row crosses here,
  if (t0 > 0 && p.keys[t0 * kTile - 1] == r) return;                       // or it began before this tile
  const int end = first_at_least(p.keys, (int)next_tile, n, r + 1);
  const int64_t t1 = (end - 1) / kTile;
  // its heads t0 + 1 .. t1.  Super-tile j is the row's if the row began before it and holds its last token.
  const int64_t s0 = (t0 + kSuper) / kSuper, s1 = max((int64_t)end / (kSuper * kTile), s0);
  const bool whole = s1 > s0;
  for (int e = c * VEC; e < E; e += VEC << lg) {
    float acc[VEC];
    load_elems<VEC>(tail + t0 * E + e, acc);
    for (int k = 0; k < 3; ++k) {  // heads, super-tiles, heads
      const int64_t from = k == 0 ? t0 + 1 : k == 1 ? s0 : whole ? s1 * kSuper : t1 + 1;
      const int64_t to = k == 0 ? (whole ? s0 * kSuper : t1 + 1) : k == 1 ? s1 : t1 + 1;
      part_add<VEC>(k == 1 ? sup : head, E, e, from, to, acc);
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) acc[i] *= scale;
    store_elems_nt<VEC>(grad + (int64_t)r * E + e, acc);
  }
}

template <typename TW, typename TO>
int launch_fwd(const void* table, int64_t V, int E, int64_t ld, const void* ids, bool wide, int64_t n, float scale,
               void* out, hipStream_t s) {
  const int64_t counts[] = {E, ld};
  const void* ptrs[] = {table, out};
  const int bytes[] = {(int)sizeof(TW), (int)sizeof(TO)};
  int vec = vec_for(counts, 2, ptrs, bytes, 2);
  if (sizeof(TW) == 4 && sizeof(TO) == 4 && vec > 4) vec = 4;
  const int lg = row_lanes_log2(E, vec);
  constexpr int U = 4;
  const int64_t per_block = (int64_t)kWavesPerBlock * (kWave >> lg) * U;
  int64_t blocks = (n + per_block - 1) / per_block;
  const bool runs = blocks >= 8 * 8 * kXcdRun;
  if (runs) blocks = (blocks + 8 * kXcdRun - 1) / (8 * kXcdRun) * (8 * kXcdRun);
  const dim3 grid = wide_grid(blocks), block(kBlock);
  const TW* t = static_cast<const TW*>(table);
  TO* o = static_cast<TO*>(out);
#define TT_LF(VV) \
  case VV: lookup_fwd_kernel<TW, TO, VV, U><<<grid, block, 0, s>>>(t, V, E, ld, ids, wide, n, scale, o, lg, runs); break;
  switch (vec) { TT_LF(8) TT_LF(4) TT_LF(2) default: TT_LF(1) }
#undef TT_LF
  TT_LAUNCH_CHECK("lookup_fwd");
  return TT_OK;
}

template <typename TW, typename TO>
int launch_bwd(const void* dout, const void* ids, int ids_dtype, int64_t n, int64_t V, int E, int64_t pad, float scale,
               void* grad, const void* plan, float* ws, hipStream_t s) {
  const int64_t counts[] = {E};
  const void* ptrs[] = {n > 0 ? dout : grad, grad};
  const int bytes[] = {(int)sizeof(TO), (int)sizeof(TW)};
  int vec = vec_for(counts, 1, ptrs, bytes, 2);
  if (sizeof(TW) == 4 && sizeof(TO) == 4 && vec > 4) vec = 4;
  const TO* d = static_cast<const TO*>(dout);
  TW* g = static_cast<TW*>(grad);
  if (n <= kDirectN) {
    // few rows each spread the frequent (low) ids over workgroups and give a wave one or two rows; at most
    // kDirectRows, so that the ids are read V / 64 times at most (30k x 100, 1073 text-like tokens: 15 us, V / 1024
    // rows each 30 us; 200k x 256, 4096 tokens: 38 and 39 us)
    int64_t R = V / 4096;
    R = R < 1 ? 1 : R > kDirectRows ? kDirectRows : R;
    const dim3 grid = wide_grid((V + R - 1) / R), block(kDirectThreads);
#define TT_LD(VV) \
  case VV: lookup_grad_direct_kernel<TO, TW, VV><<<grid, block, 0, s>>>(d, ids, ids_dtype == TT_IDS_I64, (int)n, V, E, (int)R, pad, scale, g); break;
    switch (vec) { TT_LD(8) TT_LD(4) TT_LD(2) default: TT_LD(1) }
#undef TT_LD
    TT_LAUNCH_CHECK("lookup_grad_direct");
    return TT_OK;
  }
  const TokenPlan p = token_plan_view(const_cast<void*>(plan), n, V);
  const int lg = row_lanes_log2(E, vec);
  const int64_t tiles = (n + kTile - 1) / kTile, supers = tiles / kSuper, per = kBlock >> lg;
  float *head = ws, *tail = head + tiles * E, *sup = tail + tiles * E;
  auto grid = [&](int64_t groups) { return dim3((unsigned)((groups + per - 1) / per)); };
  const int64_t zero_rows = (int64_t)kWavesPerBlock * kZeroRows;
  const dim3 block(kBlock), join = wide_grid(grid(tiles).x + (V + zero_rows - 1) / zero_rows);
#define TT_LS(VV)                                                                                                  \
  case VV:                                                                                                         \
    lookup_tile_sum_kernel<TO, TW, VV><<<grid(tiles), block, 0, s>>>(p, d, E, scale, g, lg, head, tail);           \
    TT_LAUNCH_CHECK("lookup_tile_sum");                                                                            \
    if (supers > 0) lookup_super_sum_kernel<VV><<<grid(supers), block, 0, s>>>(p, head, E, lg, sup);               \
    TT_LAUNCH_CHECK("lookup_super_sum");                                                                           \
    lookup_row_join_kernel<TW, VV><<<join, block, 0, s>>>(p, V, E, scale, g, lg, grid(tiles).x, head, tail, sup);  \
    break;
  switch (vec) { TT_LS(8) TT_LS(4) TT_LS(2) default: TT_LS(1) }
#undef TT_LS
  TT_LAUNCH_CHECK("lookup_row_join");
  return TT_OK;
}

int check_lookup(int64_t n, int64_t V, int E, const void* ids, int ids_dtype, int table_dtype, int out_dtype) {
  TT_REQUIRE(V > 0 && V < TT_LOOKUP_MAX, "V=%lld out of range", (long long)V);
  TT_REQUIRE(E > 0, "E=%d must be positive", E);
  TT_REQUIRE(n >= 0 && n < TT_LOOKUP_MAX, "n=%lld tokens out of range", (long long)n);
  TT_REQUIRE(ids_dtype == TT_IDS_I32 || ids_dtype == TT_IDS_I64, "ids_dtype=%d", ids_dtype);
  TT_REQUIRE(ids != nullptr || n == 0, "ids is NULL");
  TT_REQUIRE(elem_ok(table_dtype) && elem_ok(out_dtype) && (out_dtype == table_dtype || table_dtype == TT_E_F32),
             "lookup: rows of type %d from a table of type %d", out_dtype, table_dtype);
  return TT_OK;
}

}  // namespace
}  // namespace tt

using namespace tt;

// (table, row) types: equal, or fp32 -> 16 bit
#define TT_LOOKUP_TYPES(TABLE, ROW, CALL)                                                     \
  do {                                                                                       \
    if ((TABLE) == TT_E_BF16) return CALL(__bf16, __bf16);                                   \
    if ((TABLE) == TT_E_F16) return CALL(_Float16, _Float16);                                \
    if ((ROW) == TT_E_BF16) return CALL(float, __bf16);                                      \
    if ((ROW) == TT_E_F16) return CALL(float, _Float16);                                     \
    return CALL(float, float);                                                               \
  } while (0)

extern "C" int tt_lookup_fwd(const void* table, int table_dtype, int64_t V, int E, int64_t ld_table, const void* ids,
                             int ids_dtype, int64_t n, float scale, void* out, int out_dtype, tt_stream_t stream) {
  if (int rc = check_lookup(n, V, E, ids, ids_dtype, table_dtype, out_dtype)) return rc;
  TT_REQUIRE(ld_table >= E, "ld_table=%lld < E=%d", (long long)ld_table, E);
  if (n == 0) return TT_OK;
  TT_REQUIRE(table && out, "null pointer");
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
#define TT_CALL(TW, TO) (launch_fwd<TW, TO>(table, V, E, ld_table, ids, ids_dtype == TT_IDS_I64, n, scale, out, s))
  TT_LOOKUP_TYPES(table_dtype, out_dtype, TT_CALL);
#undef TT_CALL
}

extern "C" size_t tt_lookup_plan_size(int64_t n, int64_t V) {
  return n <= kDirectN || V <= 0 ? 0 : token_plan_bytes(n, V);
}

extern "C" int tt_lookup_plan(const void* ids, int ids_dtype, int64_t n, int64_t V, int64_t padding_idx, void* plan,
                              size_t plan_bytes, tt_stream_t stream) {
  if (int rc = check_lookup(n, V, 1, ids, ids_dtype, TT_E_F32, TT_E_F32)) return rc;
  if (n <= kDirectN) return TT_OK;
  return token_plan_build(ids, ids_dtype, n, V, padding_idx, plan, plan_bytes, reinterpret_cast<hipStream_t>(stream));
}

extern "C" size_t tt_lookup_bwd_ws_size(int64_t n, int E) {
  if (n <= kDirectN || E <= 0) return 0;
  const size_t tiles = (size_t)(n + kTile - 1) / kTile;
  return (2 * tiles + tiles / kSuper) * (size_t)E * sizeof(float);
}

extern "C" int tt_lookup_bwd(const void* dout, int dout_dtype, const void* ids, int ids_dtype, int64_t n, int64_t V,
                             int E, int64_t padding_idx, float scale, void* grad, int grad_dtype, const void* plan,
                             size_t plan_bytes, void* ws, size_t ws_bytes, tt_stream_t stream) {
  if (int rc = check_lookup(n, V, E, ids, ids_dtype, grad_dtype, dout_dtype)) return rc;
  TT_REQUIRE(grad && (dout || n == 0), "null pointer");
  if (n > kDirectN) {
    TT_REQUIRE(plan && plan_bytes >= token_plan_bytes(n, V), "plan too small: need %zu have %zu",
               token_plan_bytes(n, V), plan_bytes);
    TT_REQUIRE(ws && ws_bytes >= tt_lookup_bwd_ws_size(n, E) && reinterpret_cast<size_t>(ws) % 16 == 0,
               "workspace too small: need %zu have %zu", tt_lookup_bwd_ws_size(n, E), ws_bytes);
  }
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
#define TT_CALL(TW, TO) \
  (launch_bwd<TW, TO>(dout, ids, ids_dtype, n, V, E, padding_idx, scale, grad, plan, static_cast<float*>(ws), s))
  TT_LOOKUP_TYPES(grad_dtype, dout_dtype, TT_CALL);
#undef TT_CALL
}
