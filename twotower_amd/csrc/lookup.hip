// Token lookup with a scale, and its gradient by sorted tokens.
//
//   out[t, :]  = s W[id_t, :]                                  (ids outside [0, V): a zero row, or NaN)
//   dW[r, :]   = s sum_{t : id_t = r, r != padding_idx} dout[t, :]     (every row written)
//
// Both move bytes and add: the forward reads each token's row (repeated rows from L2) and writes
// n E elements, the backward reads n E elements once and writes V E.  8192 x 64 text-like tokens, half of them
// padding, 200k x 256 fp32: forward 150 us (537 MB written, 128 MB read from memory; 86 us without the reads, 44
// without the writes; eight tokens in flight instead of four 164), sort 40 us, tiles 70 us (344 MB, 4.9 TB/s), joins and
// empty rows 42 us (148 MB); a 4 GiB copy runs at 4.8 TB/s.  The backward needs each row's tokens together: a long
// call sorts them (the bags' stable counting sort, token_plan_build), a short one finds them among the ids in LDS.
#include "common.hpp"

#include <algorithm>

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
                                                            float scale, float outside, TO* __restrict__ out, int lg,
                                                            bool runs) {
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
    Elems<TW, VEC> x[U];  // (row 0 for an id outside: no load waits for a condition)
#pragma unroll
    for (int u = 0; u < U; ++u)
      x[u] = *reinterpret_cast<const Elems<TW, VEC>*>(table + (id[u] >= 0 && id[u] < V ? id[u] : 0) * ld + e);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t t = t0 + (int64_t)u * groups;
      if (t < n) {
        float y[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) y[i] = (id[u] >= 0 && id[u] < V) ? scale * (float)x[u].v[i] : outside;
        store_elems_nt<VEC>(out + t * E + e, y);
      }
    }
  }
}

// ---- gradient of a short call, in one launch: some workgroups write the rows without tokens, in the others a wave
// per token writes the row of its id if it is the first of them.  A token workgroup holds the n ids in LDS; a wave
// walks them in order, leaves at an earlier token of its id, and lists the later ones.  A short list is
// added up by the wave, a long one by the whole workgroup (a wide row in chunks of columns, one after the other), the
// parts folded in a fixed order.  Bound by the fill of the table where that is large (200k x 256, 1000 tokens: 29 us for
// 205 MB), else by a chain of latencies: ids, walk, rows.
// (Every workgroup owning rows, and reading all ids to find their tokens: 38 us there; at 4000 tokens 34 x 64 18, 30k x
// 100 fp16 39, 200k x 256 79 us instead of the 15, 14 and 33 below.)
//
// Short is up to kDirectN tokens, fewer of rows wider than 1 KB or 192 accesses, whose long lists take as many
// chunks: about there the sort is as fast (us, text-like ids, n = 4000 / 8000 / 12000; then sorted, 8000 / 12000):
// 34 x 64 15 / 25 / 34, 31 / 34; 30k x 100 fp16 14 / 29 / 48, 48 / 49; 50k x 128 16 / 31 / 51, 48 / 49; 200k x 256 33 /
// 50 / 70, 80 / 80; half the ids one row, 2000 x 256: 29 / 59 / 85, 51 / 53; 500 x 512 48 / 96, 51; 116 x 339 fp16 95 / 214, 78.
constexpr int kDirectN = TT_LOOKUP_DIRECT_TOKENS;
bool short_call(int64_t n, int E, int row_dtype) {
  const int bytes = elem_bytes(row_dtype);
  int vec = 16 / bytes;
  while (E % vec) vec >>= 1;
  return n * std::max(((int64_t)E * bytes + 1023) / 1024, ((int64_t)E / vec + 191) / 192) <= kDirectN;
}
constexpr int kDirectThreads = 512;
constexpr int kDirectWaves = kDirectThreads / kWave;
constexpr int kStrip = 4 * kWave;  // tokens that a wave looks at together
constexpr int kZeroSpan = 1 << 16;  // rows of a workgroup that writes empty ones, at most
constexpr int kLight = 32;  // tokens that a wave lists for itself
static_assert(kDirectN <= 1 << 16, "a list names its tokens in 16 bits");

// acc += the rows of dout named by list[first], list[first + step], ... below `count`, column e on: U in
// flight, past the end the last one again (loads under a condition of their own ran one by one)
template <int U, typename TO, int VEC>
__device__ __forceinline__ void list_add(const TO* __restrict__ dout, int E, int e, const uint16_t* list, int first,
                                         int step, int count, float (&acc)[VEC]) {
  for (int j = first; j < count; j += U * step) {
    Elems<TO, VEC> x[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      x[u] = *reinterpret_cast<const Elems<TO, VEC>*>(dout + (int64_t)list[min(j + u * step, count - 1)] * E + e);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < VEC; ++i) acc[i] += j + u * step < count ? (float)x[u].v[i] : 0.f;
  }
}

// Which of 256 tokens (from `row` on, 4 a lane) have id r: any, and per lane the number of them before the
// lane's own and a bit per own token.
struct Matches {
  uint32_t own;
  int before, all;
  __device__ __forceinline__ Matches(const int32_t* row, int r, int lane) {
    const int4 v = *reinterpret_cast<const int4*>(row + 4 * lane);
    own = (v.x == r) | (v.y == r) << 1 | (v.z == r) << 2 | (v.w == r) << 3;
    before = all = 0;
    if (!__ballot(own != 0)) return;
    const uint64_t below = (uint64_t(1) << lane) - 1;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint64_t m = __ballot(own >> j & 1);
      before += __popcll(m & below);
      all += __popcll(m);
    }
  }
};

// the sums of a wave's groups of 2^lg lanes, in every group
template <int VEC>
__device__ __forceinline__ void fold_groups(float (&acc)[VEC], int lg) {
  for (int o = 1 << lg; o < kWave; o <<= 1) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) acc[i] += __shfl_xor(acc[i], o);
  }
}

// f(i, ids[i]) for every i < limit (-1 for i >= n), eight loads in flight
template <typename F>
__device__ __forceinline__ void each_id(const void* ids, bool wide, int n, int limit, F f) {
  for (int i0 = threadIdx.x; i0 < limit; i0 += 8 * kDirectThreads) {
    int64_t id[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) id[u] = i0 + u * kDirectThreads < n ? id_at(ids, wide, i0 + u * kDirectThreads) : -1;
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (i0 + u * kDirectThreads < limit) f(i0 + u * kDirectThreads, id[u]);
  }
}

// Zeros in those of a workgroup's rows [lo, hi) that no token has (a bit per row in `mark`): EPU elements
// of consecutive memory at a time, one by one where rows with and without tokens meet.
template <int EPU, typename TW>
__device__ __forceinline__ void zero_rows(const void* ids, bool wide, int n, int64_t lo, int64_t hi, int E, int64_t pad,
                                          uint32_t* mark, TW* __restrict__ grad) {
  const int rows = (int)(hi - lo);
  for (int i = threadIdx.x; i < (rows + 31) / 32; i += kDirectThreads) mark[i] = 0;
  __syncthreads();
  each_id(ids, wide, n, n, [&](int, int64_t id) {
    if (id >= lo && id < hi && id != pad) atomicOr(&mark[(id - lo) >> 5], 1u << ((id - lo) & 31));
  });
  __syncthreads();
  auto marked = [&](int r) { return (mark[r >> 5] >> (r & 31) & 1) != 0; };
  TW* base = grad + lo * E;
  const int64_t total = (int64_t)rows * E, at0 = (int64_t)threadIdx.x * EPU;
  const int rows_on = kDirectThreads * EPU / E, cols_on = kDirectThreads * EPU % E;
  int r = (int)(at0 / E), c = (int)(at0 % E);
  for (int64_t at = at0; at < total; at += kDirectThreads * EPU) {
    const int over = c + EPU - E;  // elements of the next row (E >= EPU, or EPU = 1)
    const bool m0 = marked(r), m1 = over > 0 && r + 1 < rows ? marked(r + 1) : m0;
    if (!m0 && !m1 && at + EPU <= total) {
      const float zero[EPU] = {};
      store_elems<EPU>(base + at, zero);
    } else if (!m0 || !m1) {
#pragma unroll
      for (int j = 0; j < EPU; ++j)
        if (at + j < total && !(c + j < E ? m0 : m1)) base[at + j] = (TW)0.f;
    }
    r += rows_on;
    c += cols_on;
    if (c >= E) {
      c -= E;
      ++r;
    }
  }
}

// workgroups [0, token_blocks): the tokens; the others: the rows without any, zero_span rows each
template <typename TO, typename TW, int VEC>
__global__ __launch_bounds__(kDirectThreads) void lookup_grad_direct_kernel(
    const TO* __restrict__ dout, const void* __restrict__ ids, bool wide, int n, int64_t V, int E, int lg, int64_t pad,
    float scale, TW* __restrict__ grad, int token_blocks, int zero_span) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  if ((int)blockIdx.x >= token_blocks) {
    constexpr int kEpu = 16 / sizeof(TW);
    const int64_t lo = (int64_t)((int)blockIdx.x - token_blocks) * zero_span, hi = min(lo + zero_span, V);
    uint32_t* mark = reinterpret_cast<uint32_t*>(smem);
    if (E >= kEpu && (reinterpret_cast<size_t>(grad) & 15) == 0) zero_rows<kEpu>(ids, wide, n, lo, hi, E, pad, mark, grad);
    else zero_rows<1>(ids, wide, n, lo, hi, E, pad, mark, grad);
    return;
  }
  __shared__ uint16_t own[kDirectWaves][kLight];
  __shared__ int heavy[kDirectWaves], wcnt[kDirectWaves];
  const int np = (n + kStrip - 1) / kStrip * kStrip, strips = np / kStrip;
  float(*part)[kWave * VEC] = reinterpret_cast<float(*)[kWave * VEC]>(smem);          // [kDirectWaves - 1]
  int32_t* row = reinterpret_cast<int32_t*>(smem + (kDirectWaves - 1) * kWave * VEC * 4);  // [np], -1: no token
  uint16_t* list = reinterpret_cast<uint16_t*>(row + np);                              // [np]
  const int lane = lane_id(), w = threadIdx.x >> 6, c = lane & ((1 << lg) - 1), g = lane >> lg, groups = kWave >> lg;
  const int chunk = VEC << lg, chunks = (E + chunk - 1) / chunk;
  each_id(ids, wide, n, np, [&](int i, int64_t id) { row[i] = id >= 0 && id < V && id != pad ? (int32_t)id : -1; });
  __syncthreads();
  // consecutive tokens go to different workgroups: the frequent ids' first ones, all near the start, do too
  const int t = w * token_blocks + (int)blockIdx.x;
  const int r = t < n ? __builtin_amdgcn_readfirstlane(row[t]) : -1;
  int count = 0;
  if (r >= 0)
    for (int b = 0; b < np; b += kStrip) {
      const Matches m(row + b, r, lane);
      if (!m.all) continue;
      int at = count + m.before;
      for (uint32_t o = m.own; o; o &= o - 1, ++at)
        if (at < kLight) own[w][at] = (uint16_t)(b + 4 * lane + __builtin_ctz(o));
      if (count == 0 && __ballot(m.before == 0 && m.own && b + 4 * lane + __builtin_ctz(m.own) < t)) break;
      count += m.all;
    }
  const bool light = count <= kLight && count * chunks <= 2 * kLight;
  if (lane == 0) heavy[w] = light ? -1 : r;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // (own[w] is the wave's alone)
  if (count > 0 && light)
    for (int e = c * VEC; e < chunks * chunk; e += chunk) {
      float acc[VEC] = {};
      if (e < E) list_add<4>(dout, E, e, own[w], g, groups, count, acc);
      fold_groups<VEC>(acc, lg);
#pragma unroll
      for (int i = 0; i < VEC; ++i) acc[i] *= scale;
      if (g == 0 && e < E) store_elems<VEC>(grad + (int64_t)r * E + e, acc);
    }
  __syncthreads();
  // the workgroup's long lists: `parts` waves to a column chunk
  const int parts = chunks >= kDirectWaves ? 1 : kDirectWaves / chunks, step = kDirectWaves / parts;
  const int per = (strips + kDirectWaves - 1) / kDirectWaves;
  const int b0 = w * per, b1 = min(b0 + per, strips);
  for (int k = 0; k < kDirectWaves; ++k) {
    const int hr = heavy[k];
    if (hr < 0) continue;
    int mine = 0;
    for (int b = b0; b < b1; ++b) mine += Matches(row + b * kStrip, hr, lane).all;
    if (lane == 0) wcnt[w] = mine;
    __syncthreads();
    int at = 0, all = 0;
#pragma unroll
    for (int i = 0; i < kDirectWaves; ++i) {
      at += i < w ? wcnt[i] : 0;
      all += wcnt[i];
    }
    for (int b = b0; b < b1; ++b) {
      const Matches m(row + b * kStrip, hr, lane);
      int to = at + m.before;
      for (uint32_t o = m.own; o; o &= o - 1, ++to) list[to] = (uint16_t)(b * kStrip + 4 * lane + __builtin_ctz(o));
      at += m.all;
    }
    __syncthreads();
    const int p = w % parts;
    for (int k0 = 0; k0 < chunks; k0 += step) {
      const int e = (k0 + w / parts) * chunk + c * VEC;
      const bool on = w < parts * step && e < E;
      float acc[VEC] = {};
      if (on) list_add<8>(dout, E, e, list, p * groups + g, parts * groups, all, acc);
      fold_groups<VEC>(acc, lg);
      if (on && p > 0) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) part[w - 1][lane * VEC + i] = acc[i];
      }
      __syncthreads();
      if (on && p == 0 && g == 0) {
        for (int q = 1; q < parts; ++q) {
#pragma unroll
          for (int i = 0; i < VEC; ++i) acc[i] += part[w + q - 1][lane * VEC + i];
        }
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[i] *= scale;
        store_elems<VEC>(grad + (int64_t)hr * E + e, acc);
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
// a group's columns of a row: the grid's z chunks of them run side by side.  The tiles' and the joins' do where there are
// few (kFewWaves): 1051 x 306 bf16, 38,318 tokens: tiles and joins 10 and 10 us, chunk after chunk 18 and 21;
// 200k x 306, 524,288 tokens: 153 and 73, 142 and 51, as every chunk reads the tokens' names again.
constexpr int64_t kFewWaves = 4096;
#define TT_COLUMNS(e) for (int64_t e = (((int64_t)blockIdx.z << lg) + c) * VEC; e < E; e += (int64_t)(VEC << lg) * gridDim.z)

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
  TT_COLUMNS(e) {
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
__device__ __forceinline__ void part_add(const float* __restrict__ part, int E, int64_t e, int64_t beg, int64_t end,
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
  TT_COLUMNS(e) {
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
    if (blockIdx.z > 0) return;
    const int64_t r0 = ((block_index() - join_blocks) * kWavesPerBlock + (threadIdx.x >> 6)) * kZeroRows;
    const int lane = lane_id(), groups = kWave >> lg;
    const int64_t r = r0 + (lane < kZeroRows ? lane : kZeroRows);
    const int at = first_at_least(p.keys, 0, n, (uint32_t)(r < V ? r : V));
    const int next = __shfl(at, lane < kZeroRows ? lane + 1 : kZeroRows);
    const uint64_t empty = __ballot(lane < kZeroRows && r < V && next == at);
    const float zero[VEC] = {};
    for (int i = lane >> lg; i < kZeroRows; i += groups)
      if (empty >> i & 1)
        for (int64_t e = c * VEC; e < E; e += VEC << lg) store_elems_nt<VEC>(grad + (r0 + i) * E + e, zero);
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
  TT_COLUMNS(e) {
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

#undef TT_COLUMNS

template <typename TW, typename TO>
int launch_fwd(const void* table, int64_t V, int E, int64_t ld, const void* ids, bool wide, int64_t n, float scale,
               float outside, void* out, hipStream_t s) {
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
  case VV: lookup_fwd_kernel<TW, TO, VV, U><<<grid, block, 0, s>>>(t, V, E, ld, ids, wide, n, scale, outside, o, lg, runs); break;
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
  const int lg = row_lanes_log2(E, vec);
  if (plan == nullptr) {
    const int64_t np = (n + kStrip - 1) / kStrip * kStrip, bytes = V * E * (int64_t)sizeof(TW);
    const size_t need = (size_t)(kDirectWaves - 1) * kWave * vec * 4 + (size_t)np * 6;
    const size_t lds = std::max<size_t>(need, kZeroSpan / 8);
    // the empty rows' workgroups: 64 KB each or more (up to two to a CU), and a bit a row in LDS
    int64_t zero = std::min<int64_t>((bytes + (1 << 16) - 1) >> 16, 2048);
    const int64_t span = std::min<int64_t>(((V + zero - 1) / zero + 7) & ~7, kZeroSpan);  // (whole 16 bytes)
    zero = (V + span - 1) / span;
    const int tokens = (int)((n + kDirectWaves - 1) / kDirectWaves);
    const dim3 grid((unsigned)(tokens + zero)), block(kDirectThreads);
#define TT_LD(VV)                                                                                                     \
  case VV: {                                                                                                          \
    auto kernel = lookup_grad_direct_kernel<TO, TW, VV>;                                                              \
    if (lds > 60 * 1024)                                                                                              \
      TT_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,    \
                                 (int)lds), "lookup_grad_direct LDS");                                                \
    kernel<<<grid, block, lds, s>>>(d, ids, ids_dtype == TT_IDS_I64, (int)n, V, E, lg, pad, scale, g, tokens, (int)span); \
    break;                                                                                                            \
  }
    switch (vec) { TT_LD(8) TT_LD(4) TT_LD(2) default: TT_LD(1) }
#undef TT_LD
    TT_LAUNCH_CHECK("lookup_grad_direct");
    return TT_OK;
  }
  const TokenPlan p = token_plan_view(const_cast<void*>(plan), n, V);
  const int64_t tiles = (n + kTile - 1) / kTile, supers = tiles / kSuper, per = kBlock >> lg;
  float *head = ws, *tail = head + tiles * E, *sup = tail + tiles * E;
  const unsigned chunks = (unsigned)std::min<int64_t>(((int64_t)E + (vec << lg) - 1) / (vec << lg), 65535);
  auto grid = [&](int64_t groups) { return dim3((unsigned)((groups + per - 1) / per), 1, chunks); };
  dim3 tile_grid = grid(tiles);
  const int64_t waves = (tiles << lg) / kWave + 1;
  tile_grid.z = (unsigned)std::min<int64_t>(chunks, (kFewWaves + waves - 1) / waves);
  const int64_t zero_rows = (int64_t)kWavesPerBlock * kZeroRows;
  const dim3 block(kBlock);
  dim3 join = wide_grid(grid(tiles).x + (V + zero_rows - 1) / zero_rows);
  join.z = tile_grid.z;
#define TT_LS(VV)                                                                                                  \
  case VV:                                                                                                         \
    lookup_tile_sum_kernel<TO, TW, VV><<<tile_grid, block, 0, s>>>(p, d, E, scale, g, lg, head, tail);             \
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
  const float outside = ids_dtype & TT_LOOKUP_NAN_OUTSIDE ? __builtin_nanf("") : 0.f;
  ids_dtype &= ~TT_LOOKUP_NAN_OUTSIDE;
  if (int rc = check_lookup(n, V, E, ids, ids_dtype, table_dtype, out_dtype)) return rc;
  TT_REQUIRE(ld_table >= E, "ld_table=%lld < E=%d", (long long)ld_table, E);
  if (n == 0) return TT_OK;
  TT_REQUIRE(table && out, "null pointer");
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
#define TT_CALL(TW, TO) (launch_fwd<TW, TO>(table, V, E, ld_table, ids, ids_dtype == TT_IDS_I64, n, scale, outside, out, s))
  TT_LOOKUP_TYPES(table_dtype, out_dtype, TT_CALL);
#undef TT_CALL
}

extern "C" size_t tt_lookup_plan_size(int64_t n, int64_t V, int E, int dout_dtype) {
  return n < 0 || V <= 0 || short_call(n, E, dout_dtype) ? 0 : token_plan_bytes(n, V);
}

extern "C" int tt_lookup_plan(const void* ids, int ids_dtype, int64_t n, int64_t V, int64_t padding_idx, void* plan,
                              size_t plan_bytes, tt_stream_t stream) {
  if (int rc = check_lookup(n, V, 1, ids, ids_dtype, TT_E_F32, TT_E_F32)) return rc;
  if (plan_bytes == 0) return TT_OK;  // a short call's
  return token_plan_build(ids, ids_dtype, n, V, padding_idx, plan, plan_bytes, reinterpret_cast<hipStream_t>(stream));
}

extern "C" size_t tt_lookup_bwd_ws_size(int64_t n, int E, int dout_dtype) {
  if (n < 0 || E <= 0 || short_call(n, E, dout_dtype)) return 0;
  const size_t tiles = (size_t)(n + kTile - 1) / kTile;
  return (2 * tiles + tiles / kSuper) * (size_t)E * sizeof(float);
}

extern "C" int tt_lookup_bwd(const void* dout, int dout_dtype, const void* ids, int ids_dtype, int64_t n, int64_t V,
                             int E, int64_t padding_idx, float scale, void* grad, int grad_dtype, const void* plan,
                             size_t plan_bytes, void* ws, size_t ws_bytes, tt_stream_t stream) {
  if (int rc = check_lookup(n, V, E, ids, ids_dtype, grad_dtype, dout_dtype)) return rc;
  TT_REQUIRE(grad && (dout || n == 0), "null pointer");
  const bool direct = short_call(n, E, dout_dtype);
  if (!direct) {
    TT_REQUIRE(plan && plan_bytes >= token_plan_bytes(n, V), "plan too small: need %zu have %zu",
               token_plan_bytes(n, V), plan_bytes);
    TT_REQUIRE(ws && ws_bytes >= tt_lookup_bwd_ws_size(n, E, dout_dtype) && reinterpret_cast<size_t>(ws) % 16 == 0,
               "workspace too small: need %zu have %zu", tt_lookup_bwd_ws_size(n, E, dout_dtype), ws_bytes);
  }
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
#define TT_CALL(TW, TO) \
  (launch_bwd<TW, TO>(dout, ids, ids_dtype, n, V, E, padding_idx, scale, grad, direct ? nullptr : plan,              \
                      static_cast<float*>(ws), s))
  TT_LOOKUP_TYPES(grad_dtype, dout_dtype, TT_CALL);
#undef TT_CALL
}
