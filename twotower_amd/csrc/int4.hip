// 4-bit rows with group scales, and their products with a few fp32 vectors: the document index of the
// search at 4.5 bits a value (group 32) instead of 32.
//
//   score[i, j] = sum_g s_jg sum_{k in g} (c_jk - 8) q_ik
//
// One or a few queries are bound by the index bytes (n (H / 2 + 2 H / group)); 256 codes a row leave no
// time to widen each code to a float in vector instructions, so the inner sums run on the
// matrix cores: codes are small integers, exact in fp16, and q is cut into three fp16 terms
// (query_exponent says what they hold), so v_mfma_f32_16x16x32_f16 forms the sum of 32 exact products in fp32; the group's
// scale multiplies that sum.  32 columns are the instruction's K and the smallest group.
//
// 1M x 256, group 32 (us for 1 / 16 / 64 queries): 31-36 / 46-50 / 118-123, for 148 MB of index and 4 MB of scores a
// query (fp32 cosine scores of the same rows: 188 / 234 / 437); group 128: 30 / 45 / 117.  One query is bound by the
// index's reads, 4.2-5.0 TB/s (workgroups of 256: 32-38; with these 1, 2 or 4 tiles a wave, half as many waves, loads
// past the caches: no faster).  Short indexes are bound by the launch and the queries' layout: 200k x 128, 8 queries
// 10.3 us, 28,834 x 100, 33 queries 8.7.
//
// Layout (written once per index): tiles of 16 rows; a tile is a run of quads of 128 columns, a quad
// of 64 lanes x 16 bytes in the order the kernel loads it: lane (row j = l % 16, h = l / 16), dword d
// holds row j's columns 128 quad + 32 d + 8 h .. + 7.  A wave's load is 1 KB of consecutive bytes and
// dword d is the B operand of column block d without any exchange.  A short last quad has as many
// dwords a lane as column blocks.  Nibble s of a dword is column 2 s, nibble s + 4 column 2 s + 1, so
// (u >> 4 s) & 0x000f000f is an fp16 pair in operand order.  Scales: per tile and quad, 16 rows x 128 / group.
#include "common.hpp"

namespace tt {
namespace {

constexpr int kBlock = 256;
constexpr int kRows = 16;   // documents per tile
constexpr int kBlk = 32;    // columns per matrix instruction
constexpr int kQuad = 128;  // columns per lane load
constexpr int kTPW = 2;     // tiles a wave scores together (they share the query operands' LDS reads)
constexpr uint32_t kZeroCodes = 0x88888888u;

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

inline int blocks_of(int H) { return (H + kBlk - 1) / kBlk; }
inline int quads_of(int H) { return (H + kQuad - 1) / kQuad; }
inline int64_t tiles_of(int64_t n) { return (n + kRows - 1) / kRows; }

__device__ __forceinline__ float bf16_value(uint16_t b) { return __uint_as_float((uint32_t)b << 16); }

// where the codes of row `row`, column block b, columns 8 h .. 8 h + 7 of it are
__device__ __forceinline__ int64_t code_word(int64_t row, int b, int h, int nblk) {
  const int quad = b >> 2, dpl = nblk - 4 * quad < 4 ? nblk - 4 * quad : 4;  // dwords per lane of the quad
  return (row / kRows) * nblk * 64 + quad * 256 + (h * kRows + row % kRows) * dpl + (b & 3);
}
__device__ __forceinline__ int64_t scale_at(int64_t row, int b, int nquad, int group) {
  const int spq = kQuad / group, quad = b >> 2;
  return (((row / kRows) * nquad + quad) * kRows + row % kRows) * spq + (b & 3) * kBlk / group;
}

// 8 codes (0..15) of columns 8 h .. 8 h + 7 -> their dword
__device__ __forceinline__ uint32_t pack8(const int* c) {
  uint32_t u = 0;
#pragma unroll
  for (int s = 0; s < 4; ++s) u |= (uint32_t)c[2 * s] << (4 * s) | (uint32_t)c[2 * s + 1] << (4 * s + 16);
  return u;
}

// max / 7 rounded to bf16, to nearest even of the exact quotient: the fp32 quotient is on the right side
// of every bf16 midpoint unless it equals one, and 7 x a midpoint (9 bits) is exact in fp32.
__device__ __forceinline__ uint16_t group_scale(float mx) {
  const uint32_t u = __float_as_uint(mx / 7.f);
  uint32_t r = u >> 16;
  const uint32_t low = u & 0xffffu;
  bool up = low > 0x8000u;
  if (low == 0x8000u) {
    const float d = __builtin_fmaf(-7.f, __uint_as_float(u), mx);  // sign of the exact difference
    up = d > 0.f || (d == 0.f && (r & 1));
  }
  return (uint16_t)(r + (up ? 1 : 0));
}

// the integer nearest to x / s (ties to even), |x / s| <= 7.5: x - r s is exact in fp32 for the small
// integers r next to the quotient, so the comparison with s / 2 decides the rounding exactly.
__device__ __forceinline__ int group_code(float x, float s) {
  float r = rintf(x / s);
  const float d = __builtin_fmaf(-r, s, x);
  const float twice = 2.f * d;
  const bool odd = ((int)r) & 1;
  if (twice > s || (twice == s && odd)) r += 1.f;
  else if (twice < -s || (twice == -s && odd)) r -= 1.f;
  return (int)fminf(fmaxf(r, -7.f), 7.f);
}

// elements k0 .. k0 + 7 of a row of H, zeros past H (wide: 4 at a time are aligned and H % 4 == 0)
template <typename T>
__device__ __forceinline__ void load8(const T* __restrict__ row, int k0, int H, bool wide, float (&x)[8]) {
#pragma unroll
  for (int g = 0; g < 8; g += 4) {
    float y[4] = {0.f, 0.f, 0.f, 0.f};
    if (wide) {
      if (k0 + g < H) load_elems<4>(row + k0 + g, y);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (k0 + g + e < H) y[e] = (float)row[k0 + g + e];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) x[g + e] = y[e];
  }
}

// The layout kernels take a thread per (row, 8 columns), the threads of a row's columns side by side: the
// rows are read and written in consecutive runs, and the threads of a group join their maxima.  1M x 256, group 32:
// packed in 191 us, quantized from fp32 in 303 (1.2 GB moved).
struct Place {
  int64_t row;
  int b, h;
};
__device__ __forceinline__ Place place_of(int64_t id, int nquad) {
  const int64_t row = id / (16 * nquad);
  const int w = (int)(id - row * (16 * nquad));
  return Place{row, w >> 2, w & 3};
}

template <typename T>
__global__ __launch_bounds__(kBlock) void int4_quantize_kernel(const T* __restrict__ x, int64_t n, int H, int64_t ld,
                                                               int group, int nblk, int nquad, bool wide,
                                                               uint32_t* __restrict__ codes,
                                                               uint16_t* __restrict__ scales) {
  const Place p = place_of(block_index() * kBlock + threadIdx.x, nquad);
  if (p.row >= (n + kRows - 1) / kRows * kRows) return;  // (whole groups of lanes leave together)
  float v[8] = {};
  if (p.row < n) load8(x + p.row * ld, p.b * kBlk + 8 * p.h, H, wide, v);
  float mx = 0.f;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    bad = bad || !(fabsf(v[i]) <= 3.402823466e38f);
    mx = fmaxf(mx, fabsf(v[i]));
  }
  for (int o = 1; o < group / 8; o <<= 1) {
    mx = fmaxf(mx, __shfl_xor(mx, o));
    bad = __shfl_xor((int)bad, o) || bad;
  }
  uint16_t sb = group_scale(mx);
  if (bad) sb = 0x7fc0u;
  if (p.h == 0 && (p.b & (group / kBlk - 1)) == 0) scales[scale_at(p.row, p.b, nquad, group)] = sb;
  if (p.b >= nblk) return;
  const float s = bf16_value(sb);
  int c[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) c[i] = 8 + ((bad || s == 0.f) ? 0 : group_code(v[i], s));
  codes[code_word(p.row, p.b, p.h, nblk)] = pack8(c);
}

__global__ __launch_bounds__(kBlock) void int4_pack_kernel(const int8_t* __restrict__ src,
                                                           const uint16_t* __restrict__ sc, int64_t n, int H,
                                                           int group, int nblk, int nquad, bool wide,
                                                           uint32_t* __restrict__ codes,
                                                           uint16_t* __restrict__ scales) {
  const Place p = place_of(block_index() * kBlock + threadIdx.x, nquad);
  if (p.row >= (n + kRows - 1) / kRows * kRows) return;
  const int ng = (H + group - 1) / group, g = p.b * kBlk / group;
  if (p.h == 0 && (p.b & (group / kBlk - 1)) == 0)
    scales[scale_at(p.row, p.b, nquad, group)] = p.row < n && g < ng ? sc[p.row * ng + g] : (uint16_t)0;
  if (p.b >= nblk) return;
  const int k0 = p.b * kBlk + 8 * p.h;
  const int8_t* at = src + p.row * H + k0;
  Elems<int8_t, 8> v = {};
  if (wide) {  // (8 at a time are aligned and H % 8 == 0)
    if (p.row < n && k0 < H) v = *reinterpret_cast<const Elems<int8_t, 8>*>(at);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (p.row < n && k0 + i < H) v.v[i] = at[i];
  }
  int c[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) c[i] = 8 + (v.v[i] < -8 ? -8 : v.v[i] > 7 ? 7 : (int)v.v[i]);
  codes[code_word(p.row, p.b, p.h, nblk)] = pack8(c);
}

__global__ __launch_bounds__(kBlock) void int4_unpack_kernel(const uint32_t* __restrict__ codes,
                                                             const uint16_t* __restrict__ scales, int64_t n, int H,
                                                             int group, int nblk, int nquad, float* __restrict__ out) {
  const Place p = place_of(block_index() * kBlock + threadIdx.x, nquad);
  const int k0 = p.b * kBlk + 8 * p.h;
  if (p.row >= n || k0 >= H) return;
  const float s = bf16_value(scales[scale_at(p.row, p.b, nquad, group)]);
  const uint32_t u = codes[code_word(p.row, p.b, p.h, nblk)];
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = (float)((int)(u >> (4 * (i >> 1) + 16 * (i & 1)) & 15) - 8) * s;
  float* o = out + p.row * H + k0;
  if (H % 4 == 0) {  // (H is then a multiple of every access: k0 + 4 <= H)
#pragma unroll
    for (int g = 0; g < 8; g += 4) {
      const float y[4] = {v[g], v[g + 1], v[g + 2], v[g + 3]};
      if (k0 + g < H) store_elems<4>(o + g, y);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (k0 + i < H) o[i] = v[i];
  }
}

// ---- scores.  Query rows are the A operand (16 rows), documents the B operand, so a lane of the
// result holds one document (column l % 16) and the four A rows 4 h .. 4 h + 3 of its quarter h = l / 16.
//   NQT = 0: up to 4 queries; A rows 4 i, 4 i + 1, 4 i + 2 are query i's three terms, so one instruction
//            does all of them and the lane adds its own rows;
//   NQT > 0: 16 queries per A operand, NQT operands; three instructions chain the terms.
template <int NQT>
struct QueryTiles {
  static constexpr int kOps = NQT == 0 ? 1 : 3 * NQT;   // A operands per column block
  static constexpr int kQ = NQT == 0 ? 4 : 16 * NQT;    // queries per pass
  static constexpr int kAcc = NQT == 0 ? 1 : 4 * NQT;   // results per lane and document tile
};

__device__ __forceinline__ f16x8 widen(uint32_t u) {
  // nibble pairs under the exponent of 1024 are the fp16 numbers 1024 + c; minus 1032: c - 8, exact
  union { f16x8 v; f16x2 p[4]; uint32_t w[4]; } r;
  const f16x2 bias = {(_Float16)(-1032.f), (_Float16)(-1032.f)};
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    r.w[s] = ((u >> (4 * s)) & 0x000f000fu) | 0x64006400u;
    r.p[s] += bias;
  }
  return r.v;
}

// 2^14 <= max |q| 2^e < 2^15 over a query's finite elements, as far up as fp16 goes.  The three terms take 11 bits each
// of a scaled element, but none below fp16's least step 2^-24: fp32's 24 bits are whole from 2^-1 up, that is down to
// 2^-15 of the query's largest element, and a smaller one is off by at most 2^-25, 2^-39 of the largest.  (Under 2^4 that was 2^-28: with zero codes at
// a dominant column and the other elements 2^-15 of it scores were off by 1.7e-5 of their mass, in fp32 by 5e-8.
// Terms with factors of their own, 1, 2^-11 and 2^-22, reach further, but the codes under each factor take vector
// instructions: 64 queries, 1M x 256, 172 us instead of 118.)
__device__ __forceinline__ int query_exponent(float mx) {
  return mx > 0.f ? 14 - ilogbf(mx) : 0;
}

// What a wave loads for one quad of its tiles.
template <int SPQ>
struct QuadLoad {
  uint32_t c[kTPW][4];
  Elems<uint16_t, SPQ> s[kTPW];
};
template <int SPQ>
__device__ __forceinline__ void load_quad(QuadLoad<SPQ>& x, const uint32_t* __restrict__ codes,
                                          const uint16_t* __restrict__ scales, int64_t t0, int64_t ntile, int b,
                                          int nblk, int nquad, int lane) {
  const int dpl = nblk - 4 * b < 4 ? nblk - 4 * b : 4;
#pragma unroll
  for (int u = 0; u < kTPW; ++u) {
    const int64_t t = t0 + u < ntile ? t0 + u : ntile - 1;  // (a clamped tile is never stored)
    const uint32_t* p = codes + t * nblk * 64 + b * 256 + lane * dpl;
    if (dpl == 4) {
      const tt_u32x4 v = *reinterpret_cast<const tt_u32x4*>(p);
#pragma unroll
      for (int d = 0; d < 4; ++d) x.c[u][d] = v[d];
    } else {
#pragma unroll
      for (int d = 0; d < 4; ++d) x.c[u][d] = d < dpl ? p[d] : kZeroCodes;
    }
    x.s[u] = *reinterpret_cast<const Elems<uint16_t, SPQ>*>(scales + ((t * nquad + b) * kRows + (lane & 15)) * SPQ);
  }
}

constexpr uint32_t kInf = 0x7f800000u;

// f(query, column block, column in it, value) for a workgroup's queries, element by element
template <typename T, typename F>
__device__ __forceinline__ void each_element(const T* __restrict__ q, int nq, int64_t ldq, int H, int items, int nrow,
                                             int nthread, F f) {
#pragma unroll 1
  for (int it = threadIdx.x; it < 8 * items; it += nthread) {
    const int k = it % kBlk, i = it / kBlk % nrow, b = it / kBlk / nrow;
    if (i < nq && b * kBlk + k < H) f(i, b, k, (float)q[i * ldq + b * kBlk + k]);
  }
}

template <typename T, int NQT, int SPQ, int BLOCK>
__global__ __launch_bounds__(BLOCK) void int4_scores_kernel(const T* __restrict__ q, int nq, int64_t ldq,
                                                            const uint32_t* __restrict__ codes,
                                                            const uint16_t* __restrict__ scales, int64_t n, int H,
                                                            int nblk, int nquad, bool wide,
                                                            float* __restrict__ scores, int64_t ld_scores) {
  using Q = QueryTiles<NQT>;
  constexpr int kWaves = BLOCK / kWave;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  f16x8* A = reinterpret_cast<f16x8*>(smem);  // [4 nquad][kOps][64]
  __shared__ int qe[Q::kQ];
  const int lane = lane_id(), w = threadIdx.x >> 6, j = lane & 15, h = lane >> 4;
  const int64_t ntile = (n + kRows - 1) / kRows;
  const int64_t step = (int64_t)gridDim.x * kWaves * kTPW;
  int64_t t0 = ((int64_t)blockIdx.x * kWaves + w) * kTPW;
  QuadLoad<SPQ> cur;  // the first documents are on their way while the queries are laid out
  if (t0 < ntile) load_quad<SPQ>(cur, codes, scales, t0, ntile, 0, nblk, nquad, lane);

  // A thread takes runs of 8 elements of a query, kRuns of them in flight: their maxima join the query's (an
  // integer maximum of the bits, whatever the order), then their terms go to the operands.  (us, 1 and 4 runs in
  // flight: 3994 x 327, 31 queries 12.9 and 11.3; 1M x 256, one query, which has one run a thread, 30.0 and 32.9.)
  constexpr int kRuns = NQT >= 2 ? 4 : 1;
  if (threadIdx.x < Q::kQ) qe[threadIdx.x] = 0;
  __syncthreads();
  const int items = nblk * Q::kQ * 4;
  float x[kRuns][8];
  auto load_runs = [&](int it0) {
#pragma unroll
    for (int u = 0; u < kRuns; ++u) {
      const int it = it0 + u * BLOCK, i = (it >> 2) % Q::kQ;
      load8(q + i * ldq, ((it >> 2) / Q::kQ) * kBlk + 8 * (it & 3), it < items && i < nq ? H : 0, wide, x[u]);
    }
  };
  for (int it0 = threadIdx.x; it0 < items; it0 += kRuns * BLOCK) {
    load_runs(it0);
#pragma unroll
    for (int u = 0; u < kRuns; ++u) {
      uint32_t mx = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) mx = max(mx, __float_as_uint(fabsf(x[u][e])));
      if (mx) atomicMax(reinterpret_cast<uint32_t*>(&qe[((it0 + u * BLOCK) >> 2) % Q::kQ]), mx);
    }
  }
  __syncthreads();
  uint32_t own = (uint32_t)qe[lane % Q::kQ];
  // an infinity or a NaN among the queries: their exponents from the finite elements, and an infinity's terms mended
  // below, apart from the loop that does them all: within it that took a register too many (1M x 256, one query: 32.3
  // instead of 31.5 us).
  const bool wild = __any(own >= kInf);  // (every wave reads every query's)
  __syncthreads();
  if (wild) {
    if (threadIdx.x < Q::kQ) qe[threadIdx.x] = 0;
    __syncthreads();
    each_element(q, nq, ldq, H, items, Q::kQ, BLOCK, [&](int i, int, int, float v) {
      const uint32_t a = __float_as_uint(fabsf(v));
      if (a < kInf) atomicMax(reinterpret_cast<uint32_t*>(&qe[i]), a);
    });
    __syncthreads();
    own = (uint32_t)qe[lane % Q::kQ];
    __syncthreads();
  }
  if (threadIdx.x < Q::kQ) qe[threadIdx.x] = query_exponent(__uint_as_float(own));
  __syncthreads();
  for (int it0 = threadIdx.x; it0 < items; it0 += kRuns * BLOCK) {
    if (items > kRuns * BLOCK) load_runs(it0);
#pragma unroll
    for (int u = 0; u < kRuns; ++u) {
      const int it = it0 + u * BLOCK, hh = it & 3, i = (it >> 2) % Q::kQ, b = (it >> 2) / Q::kQ;
      if (it >= items) break;
      f16x8 t0v, t1v, t2v;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float y = ldexpf(x[u][e], qe[i]);
        t0v[e] = (_Float16)y;
        const float r1 = y - (float)t0v[e];
        t1v[e] = (_Float16)r1;
        t2v[e] = (_Float16)(r1 - (float)t1v[e]);
      }
      if constexpr (NQT == 0) {
        f16x8* at = A + b * kWave + hh * 16 + 4 * i;
        at[0] = t0v;
        at[1] = t1v;
        at[2] = t2v;
        at[3] = f16x8{};
      } else {
        f16x8* at = A + ((size_t)b * Q::kOps + 3 * (i >> 4)) * kWave + hh * 16 + (i & 15);
        at[0] = t0v;
        at[kWave] = t1v;
        at[2 * kWave] = t2v;
      }
    }
  }
  __syncthreads();
  if (wild) {  // an infinity less its first term is NaN: it is that term alone
    each_element(q, nq, ldq, H, items, Q::kQ, BLOCK, [&](int i, int b, int k, float v) {
      if (!__builtin_isinf(v)) return;
      const int hh = k >> 3, step = NQT == 0 ? 1 : kWave;
      f16x8* at = NQT == 0 ? A + b * kWave + hh * 16 + 4 * i
                           : A + ((size_t)b * Q::kOps + 3 * (i >> 4)) * kWave + hh * 16 + (i & 15);
      for (int t = 1; t < 3; ++t) reinterpret_cast<_Float16*>(at + t * step)[k & 7] = (_Float16)0.f;
    });
    __syncthreads();
  }

  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  for (; t0 < ntile; t0 += step) {
    float acc[kTPW][Q::kAcc] = {};
    for (int b = 0; b < nquad; ++b) {
      const int dpl = nblk - 4 * b < 4 ? nblk - 4 * b : 4;
      QuadLoad<SPQ> next;  // the quad after this one, loaded before this one is used
      const bool last = b + 1 == nquad;
      if (!last || t0 + step < ntile)
        load_quad<SPQ>(next, codes, scales, last ? t0 + step : t0, ntile, last ? 0 : b + 1, nblk, nquad, lane);
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        if (d >= dpl) break;
        f16x8 B[kTPW];
        float s[kTPW];
#pragma unroll
        for (int u = 0; u < kTPW; ++u) {
          B[u] = widen(cur.c[u][d]);
          s[u] = bf16_value(cur.s[u].v[d * SPQ / 4]);
        }
        const f16x8* Ab = A + (size_t)(4 * b + d) * Q::kOps * kWave + lane;
        if constexpr (NQT == 0) {
          const f16x8 a = Ab[0];
#pragma unroll
          for (int u = 0; u < kTPW; ++u) {
            const f32x4 r = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, B[u], zero, 0, 0, 0);
            acc[u][0] = __builtin_fmaf(s[u], (r[2] + r[1]) + r[0], acc[u][0]);
          }
        } else {
#pragma unroll
          for (int qt = 0; qt < NQT; ++qt) {
            const f16x8 a0 = Ab[(3 * qt) * kWave], a1 = Ab[(3 * qt + 1) * kWave], a2 = Ab[(3 * qt + 2) * kWave];
#pragma unroll
            for (int u = 0; u < kTPW; ++u) {
              f32x4 r = __builtin_amdgcn_mfma_f32_16x16x32_f16(a2, B[u], zero, 0, 0, 0);
              r = __builtin_amdgcn_mfma_f32_16x16x32_f16(a1, B[u], r, 0, 0, 0);
              r = __builtin_amdgcn_mfma_f32_16x16x32_f16(a0, B[u], r, 0, 0, 0);
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[u][4 * qt + e] = __builtin_fmaf(s[u], r[e], acc[u][4 * qt + e]);
            }
          }
        }
      }
      cur = next;
    }
#pragma unroll
    for (int u = 0; u < kTPW; ++u) {
      const int64_t doc = (t0 + u) * kRows + j;
      if (doc >= n) continue;
#pragma unroll
      for (int r = 0; r < Q::kAcc; ++r) {
        const int i = NQT == 0 ? h : 16 * (r >> 2) + 4 * h + (r & 3);
        if (i < nq) scores[i * ld_scores + doc] = ldexpf(acc[u][r], -qe[i]);
      }
    }
  }
}

// Query operands per workgroup.  Rows wider than 1024 values take the form of up to 4 queries whatever their number,
// and read the index for every four (100k x 2048, 4 / 16 / 64 queries: 34 / 133 / 528 us).
constexpr size_t kMaxLds = 96 * 1024;

template <typename T, int NQT, int SPQ, int BLOCK>
int launch_scores_block(const T* q, int nq, int64_t ldq, const uint32_t* codes, const uint16_t* scales, int64_t n,
                        int H, float* scores, int64_t ld_scores, hipStream_t s) {
  const int nquad = quads_of(H);
  const size_t lds = (size_t)4 * nquad * QueryTiles<NQT>::kOps * kWave * 16;
  const int64_t per = (int64_t)kTPW * (BLOCK / kWave), groups = (tiles_of(n) + per - 1) / per;
  // (for up to 4 queries every wave that fits; more leave the time to fewer, longer workgroups)
  int64_t per_cu = (int64_t)(160 * 1024) / (int64_t)(lds + 1024);  // workgroups a CU's LDS and 32 waves hold
  const int64_t waves = NQT == 0 ? 32 : 16;
  if (per_cu > waves * kWave / BLOCK) per_cu = waves * kWave / BLOCK;
  const int64_t most = 256 * (per_cu < 1 ? 1 : per_cu);
  const int64_t rounds = (groups + most - 1) / most;  // every workgroup the same number of passes, nearly
  const bool wide = H % 4 == 0 && ldq % 4 == 0 && reinterpret_cast<size_t>(q) % (4 * sizeof(T)) == 0;
  auto kernel = int4_scores_kernel<T, NQT, SPQ, BLOCK>;
  if (lds > 64 * 1024)
    TT_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                               (int)lds), "int4_scores LDS");
  kernel<<<dim3((unsigned)((groups + rounds - 1) / rounds)), dim3(BLOCK), lds, s>>>(
      q, nq, ldq, codes, scales, n, H, blocks_of(H), nquad, wide, scores, ld_scores);
  TT_LAUNCH_CHECK("int4_scores");
  return TT_OK;
}

// The workgroups of a CU share its LDS, each with the query operands: workgroups of 512, or of 1024 where the
// operands are large and the index gives each of their waves its tiles (us, 256 / 512 / 1024 threads: 1M x 256, one query
// 32.0 / 30.1 / 30.0; 200k x 256, 42 queries 47 / 33 / 28; 9729 x 384, 32 queries 11.3 / 10.1 / 12.9).
template <typename T, int NQT, int SPQ>
int launch_scores(const T* q, int nq, int64_t ldq, const uint32_t* codes, const uint16_t* scales, int64_t n, int H,
                  float* scores, int64_t ld_scores, hipStream_t s) {
  const size_t lds = (size_t)4 * quads_of(H) * QueryTiles<NQT>::kOps * kWave * 16;
  if (lds > 78 * 1024 && tiles_of(n) > 256 * 8 * kTPW)
    return launch_scores_block<T, NQT, SPQ, 1024>(q, nq, ldq, codes, scales, n, H, scores, ld_scores, s);
  return launch_scores_block<T, NQT, SPQ, 512>(q, nq, ldq, codes, scales, n, H, scores, ld_scores, s);
}

template <typename T, int SPQ>
int scores_passes(const T* q, int64_t nq, int64_t ldq, const uint32_t* codes, const uint16_t* scales, int64_t n, int H,
                  float* scores, hipStream_t s) {
  const size_t lds16 = (size_t)4 * quads_of(H) * 3 * kWave * 16;  // one 16-query operand set
  for (int64_t i = 0; i < nq;) {
    const int64_t left = nq - i;
    const T* qi = q + i * ldq;
    float* si = scores + i * n;
    int rc, m;
    if (left <= 4 || lds16 > kMaxLds) {
      m = (int)(left < 4 ? left : 4);
      rc = launch_scores<T, 0, SPQ>(qi, m, ldq, codes, scales, n, H, si, n, s);
    } else if (left <= 16 || 2 * lds16 > kMaxLds) {
      m = (int)(left < 16 ? left : 16);
      rc = launch_scores<T, 1, SPQ>(qi, m, ldq, codes, scales, n, H, si, n, s);
    } else if (left <= 32 || 4 * lds16 > kMaxLds) {
      m = (int)(left < 32 ? left : 32);
      rc = launch_scores<T, 2, SPQ>(qi, m, ldq, codes, scales, n, H, si, n, s);
    } else {
      m = (int)(left < 64 ? left : 64);
      rc = launch_scores<T, 4, SPQ>(qi, m, ldq, codes, scales, n, H, si, n, s);
    }
    if (rc) return rc;
    i += m;
  }
  return TT_OK;
}

template <typename T>
int scores_groups(const void* q, int64_t nq, int64_t ldq, const void* codes, const void* scales, int64_t n, int H,
                  int group, float* out, hipStream_t s) {
  const T* tq = static_cast<const T*>(q);
  const uint32_t* c = static_cast<const uint32_t*>(codes);
  const uint16_t* sc = static_cast<const uint16_t*>(scales);
  if (group == 32) return scores_passes<T, 4>(tq, nq, ldq, c, sc, n, H, out, s);
  if (group == 64) return scores_passes<T, 2>(tq, nq, ldq, c, sc, n, H, out, s);
  return scores_passes<T, 1>(tq, nq, ldq, c, sc, n, H, out, s);
}

int check_int4(int64_t n, int H, int group, const void* codes, const void* scales) {
  TT_REQUIRE(n >= 0 && n < (int64_t(1) << 40) / TT_INT4_MAX_H, "int4: n=%lld rows out of range", (long long)n);
  TT_REQUIRE(H >= 1 && H <= TT_INT4_MAX_H, "int4: H=%d must be in [1, %d]", H, TT_INT4_MAX_H);
  TT_REQUIRE(group == 32 || group == 64 || group == 128, "int4: group=%d must be 32, 64 or 128", group);
  TT_REQUIRE(n == 0 || (codes && scales), "null pointer");
  TT_REQUIRE(reinterpret_cast<size_t>(codes) % 16 == 0 && reinterpret_cast<size_t>(scales) % 16 == 0,
             "int4: codes and scales must be 16-byte aligned");
  return TT_OK;
}

// workgroups of the layout kernels: a thread per (row of a whole tile, 8 columns of a whole quad)
inline int64_t layout_blocks(int64_t n, int H) {
  return (tiles_of(n) * kRows * 16 * quads_of(H) + kBlock - 1) / kBlock;
}

}  // namespace
}  // namespace tt

using namespace tt;

extern "C" size_t tt_int4_codes_bytes(int64_t n, int H) {
  return n < 0 || H < 1 ? 0 : (size_t)tiles_of(n) * blocks_of(H) * 256;
}

extern "C" size_t tt_int4_scales_bytes(int64_t n, int H, int group) {
  return n < 0 || H < 1 || group < 1 ? 0 : (size_t)tiles_of(n) * quads_of(H) * kRows * (kQuad / group) * 2;
}

extern "C" int tt_int4_quantize(const void* x, int dtype, int64_t n, int H, int64_t ld, int group, void* codes,
                                void* scales, tt_stream_t stream) {
  if (int rc = check_int4(n, H, group, codes, scales)) return rc;
  TT_REQUIRE(elem_ok(dtype) && ld >= H && (x || n == 0), "int4: element type %d, ld=%lld", dtype, (long long)ld);
  if (n == 0) return TT_OK;
  TT_REQUIRE(layout_blocks(n, H) < (int64_t(1) << 31), "int4: too many values");
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const dim3 grid = wide_grid(layout_blocks(n, H)), block(kBlock);
  const bool wide = H % 4 == 0 && ld % 4 == 0 && reinterpret_cast<size_t>(x) % (4 * elem_bytes(dtype)) == 0;
#define TT_QZ(T)                                                                                              \
  int4_quantize_kernel<T><<<grid, block, 0, s>>>(static_cast<const T*>(x), n, H, ld, group, blocks_of(H),     \
                                                 quads_of(H), wide, static_cast<uint32_t*>(codes),                  \
                                                 static_cast<uint16_t*>(scales))
  if (dtype == TT_E_F32) TT_QZ(float);
  else if (dtype == TT_E_BF16) TT_QZ(__bf16);
  else TT_QZ(_Float16);
#undef TT_QZ
  TT_LAUNCH_CHECK("int4_quantize");
  return TT_OK;
}

extern "C" int tt_int4_pack(const int8_t* c, const void* sc, int64_t n, int H, int group, void* codes, void* scales,
                            tt_stream_t stream) {
  if (int rc = check_int4(n, H, group, codes, scales)) return rc;
  TT_REQUIRE(n == 0 || (c && sc), "null pointer");
  if (n == 0) return TT_OK;
  TT_REQUIRE(layout_blocks(n, H) < (int64_t(1) << 31), "int4: too many values");
  int4_pack_kernel<<<wide_grid(layout_blocks(n, H)), dim3(kBlock), 0, reinterpret_cast<hipStream_t>(stream)>>>(
      c, static_cast<const uint16_t*>(sc), n, H, group, blocks_of(H), quads_of(H),
      H % 8 == 0 && reinterpret_cast<size_t>(c) % 8 == 0, static_cast<uint32_t*>(codes), static_cast<uint16_t*>(scales));
  TT_LAUNCH_CHECK("int4_pack");
  return TT_OK;
}

extern "C" int tt_int4_unpack(const void* codes, const void* scales, int64_t n, int H, int group, float* out,
                              tt_stream_t stream) {
  if (int rc = check_int4(n, H, group, codes, scales)) return rc;
  TT_REQUIRE(n == 0 || out, "null pointer");
  TT_REQUIRE(reinterpret_cast<size_t>(out) % 16 == 0, "int4: out must be 16-byte aligned");
  if (n == 0) return TT_OK;
  const int64_t blocks = layout_blocks(n, H);
  TT_REQUIRE(blocks < (int64_t(1) << 31), "int4: too many values");
  int4_unpack_kernel<<<wide_grid(blocks), dim3(kBlock), 0, reinterpret_cast<hipStream_t>(stream)>>>(
      static_cast<const uint32_t*>(codes), static_cast<const uint16_t*>(scales), n, H, group, blocks_of(H),
      quads_of(H), out);
  TT_LAUNCH_CHECK("int4_unpack");
  return TT_OK;
}

extern "C" int tt_int4_scores(const void* q, int dtype, int64_t nq, int64_t ldq, const void* codes, const void* scales,
                              int64_t n, int H, int group, float* scores, tt_stream_t stream) {
  if (int rc = check_int4(n, H, group, codes, scales)) return rc;
  TT_REQUIRE(nq >= 0 && elem_ok(dtype) && ldq >= H, "int4: nq=%lld, query type %d, ldq=%lld", (long long)nq, dtype,
             (long long)ldq);
  if (nq == 0 || n == 0) return TT_OK;
  TT_REQUIRE(q && scores, "null pointer");
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (dtype == TT_E_F32) return scores_groups<float>(q, nq, ldq, codes, scales, n, H, group, scores, s);
  if (dtype == TT_E_BF16) return scores_groups<__bf16>(q, nq, ldq, codes, scales, n, H, group, scores, s);
  return scores_groups<_Float16>(q, nq, ldq, codes, scales, n, H, group, scores, s);
}
