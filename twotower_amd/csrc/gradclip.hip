// The global norm of many gradient tensors, and clipping by it.
//
//   norm = (sum over all tensors of g^2)^(1/2)   or   max |g|
//   dst  = src * min(1, max_norm / (norm + 1e-6))
//
// Bound by bytes: every gradient is read once for the norm and once more to be scaled (from the
// Infinity Cache where the tensors fit), and written once.  Tensors are cut into chunks; a
// launch takes up to TT_CLIP_MAX_TENSORS of them by value, so nothing is staged through memory and
// a captured call keeps its own list.  Squares are added in 64 bits: the norm neither overflows
// nor underflows before its own rounding to 32 bits, and the vector units have room for it beside
// the loads (added in 32 bits the pass took 54 instead of 57 us).  All sums run in a fixed order (no atomics).
//
// 51.3M fp32 elements into another buffer: norm 36 us (205 MB, 5.7 TB/s), scaling 64 us (410 MB, 6.4 TB/s, its
// reads partly cached; a 4 GiB copy runs at 4.8 TB/s).  16,384-element chunks on 1024 workgroups took 57 and
// 70 us, and results kept in the caches 50 (the next norm's reads then wait for their write-back) and 72.  Few
// elements: 131,584 in 4 tensors 3.9 + 4.2 us (chunks of 8192 4.7 + 4.9), 1.7M of three types 4.5 + 7.8 (5.3 + 12.6).
// Loads that a condition guards wait for each other in some of these loops and not in others (measured one by one:
// the norm's aligned one 36 us without and 40 with, the scaling's unaligned one, 12M elements, 16.6 and 19.8).
#include "common.hpp"

namespace tt {
namespace {

constexpr int kBlock = 256;
constexpr int kChunk = 8192, kMinChunk = 2048;  // elements per chunk
constexpr int kMaxParts = 2048;     // partial norms of all launches together
constexpr int kNormBlocks = 2048;   // workgroups (= partials) of one norm launch
constexpr int kScaleBlocks = 2048;

struct ClipList {
  const void* src[TT_CLIP_MAX_TENSORS];
  void* dst[TT_CLIP_MAX_TENSORS];
  int32_t first[TT_CLIP_MAX_TENSORS + 1];  // first chunk of each tensor
  // elements of its last chunk, src type | dst type << 2: 16 and 8 bits each, read as words (kernel arguments come
  // by scalar loads, which have no narrower ones)
  uint32_t last2[TT_CLIP_MAX_TENSORS / 2], type4[TT_CLIP_MAX_TENSORS / 4];
  int count, chunk;                        // tensors; elements per chunk
};

__device__ __forceinline__ int last_of(const ClipList& l, int t) { return l.last2[t >> 1] >> (t & 1) * 16 & 0xffff; }
__device__ __forceinline__ int type_of(const ClipList& l, int t) { return l.type4[t >> 2] >> (t & 3) * 8 & 0xff; }

__device__ __forceinline__ int tensor_of(const ClipList& l, int chunk) {
  int lo = 0, hi = l.count - 1;  // the last tensor with first[] <= chunk
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (l.first[mid] <= chunk) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ bool aligned16(const void* p) { return ((size_t)p & 15) == 0; }

template <bool INF>
__device__ __forceinline__ void norm_add(double& a, float g) {
  if constexpr (INF) {
    const double m = (double)fabsf(g);
    a = (m > a || m != m) ? m : a;  // a NaN stays
  } else {
    a = __builtin_fma((double)g, (double)g, a);
  }
}
template <bool INF>
__device__ __forceinline__ double norm_join(double a, double b) {
  if constexpr (INF) return (b > a || b != b) ? b : a;
  else return a + b;
}

// this thread's part of a chunk: 16-byte accesses where the tensor is aligned, four in flight
template <typename T, bool INF>
__device__ __forceinline__ double norm_chunk(const T* __restrict__ p, int n) {
  constexpr int VEC = 16 / sizeof(T), U = 4;
  double acc[U] = {};
  if (aligned16(p)) {
    const int nv = n / VEC;
    for (int i = threadIdx.x; i < nv; i += U * kBlock) {
      Elems<T, VEC> x[U];  // (past the end the last one again: no load waits for a condition)
#pragma unroll
      for (int u = 0; u < U; ++u)
        x[u] = *reinterpret_cast<const Elems<T, VEC>*>(p + (size_t)min(i + u * kBlock, nv - 1) * VEC);
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i + u * kBlock < nv) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) norm_add<INF>(acc[u], (float)x[u].v[j]);
        }
    }
    for (int i = nv * VEC + threadIdx.x; i < n; i += kBlock) norm_add<INF>(acc[0], (float)p[i]);
  } else {
    for (int i = threadIdx.x; i < n; i += 4 * U * kBlock) {
      float x[4 * U];
#pragma unroll
      for (int u = 0; u < 4 * U; ++u) x[u] = i + u * kBlock < n ? (float)p[i + u * kBlock] : 0.f;
#pragma unroll
      for (int u = 0; u < 4 * U; ++u) norm_add<INF>(acc[u % U], x[u]);
    }
  }
  return norm_join<INF>(norm_join<INF>(acc[0], acc[1]), norm_join<INF>(acc[2], acc[3]));
}

template <bool INF>
__device__ __forceinline__ double block_join(double a) {
  __shared__ double ws[kBlock / kWave];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) a = norm_join<INF>(a, __shfl_xor(a, o));
  if (lane_id() == 0) ws[threadIdx.x >> 6] = a;
  __syncthreads();
  double r = ws[0];
#pragma unroll
  for (int k = 1; k < kBlock / kWave; ++k) r = norm_join<INF>(r, ws[k]);
  __syncthreads();
  return r;
}

template <bool INF>
__global__ __launch_bounds__(kBlock) void clip_norm_kernel(ClipList l, double* __restrict__ parts) {
  double acc = 0.0;
  const int chunks = l.first[l.count];
  for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
    const int t = tensor_of(l, c);
    const int64_t at = (int64_t)(c - l.first[t]) * l.chunk;
    const int n = c + 1 < l.first[t + 1] ? l.chunk : last_of(l, t);
    const int ty = type_of(l, t) & 3;
    double a;
    if (ty == TT_E_F32) a = norm_chunk<float, INF>(static_cast<const float*>(l.src[t]) + at, n);
    else if (ty == TT_E_BF16) a = norm_chunk<__bf16, INF>(static_cast<const __bf16*>(l.src[t]) + at, n);
    else a = norm_chunk<_Float16, INF>(static_cast<const _Float16*>(l.src[t]) + at, n);
    acc = norm_join<INF>(acc, a);
  }
  acc = block_join<INF>(acc);
  if (threadIdx.x == 0) parts[blockIdx.x] = acc;
}

template <bool INF>
__device__ __forceinline__ double joined_norm(const double* __restrict__ parts, int np) {
  constexpr int U = kMaxParts / kBlock;  // loads in flight: all of them, where kMaxParts is not exceeded
  double a = 0.0;
  for (int i = threadIdx.x; i < np; i += U * kBlock) {
    double x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) x[u] = parts[min(i + u * kBlock, np - 1)];
#pragma unroll
    for (int u = 0; u < U; ++u) a = i + u * kBlock < np ? norm_join<INF>(a, x[u]) : a;
  }
  a = block_join<INF>(a);
  return INF ? a : __builtin_sqrt(a);
}

// The factor as a * b: b = 1 but for factors so small (gradients near 1e38) that fp32 would hold them as
// subnormals of few bits; then b = 2^-64 takes the power and a keeps the 24 bits.
struct Coef {
  float a, b;
  __device__ __forceinline__ float operator()(float x) const { return (x * a) * b; }
};
__device__ __forceinline__ Coef clip_coef(double norm, double max_norm) {
  const double c = max_norm / (norm + 1e-6);
  if (c > 0.0 && c < 0x1p-100) return Coef{(float)(c * 0x1p64), 0x1p-64f};
  return Coef{c < 1.0 || c != c ? (float)c : 1.f, 1.f};
}

template <bool INF>
__global__ __launch_bounds__(kBlock) void clip_finish_kernel(const double* __restrict__ parts, int np,
                                                             float* __restrict__ norm) {
  const double v = joined_norm<INF>(parts, np);
  if (threadIdx.x == 0) *norm = (float)v;
}

template <typename TS, typename TD>
__device__ __forceinline__ void scale_chunk(const TS* src, TD* dst, int n, Coef coef) {
  constexpr int VEC = 16 / sizeof(TS), U = 4;  // (src may be dst: every element is read by the thread that writes it)
  if (aligned16(src) && aligned16(dst)) {
    const int nv = n / VEC;
    for (int i = threadIdx.x; i < nv; i += U * kBlock) {
      float x[U][VEC];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i + u * kBlock < nv) load_elems<VEC>(src + (size_t)(i + u * kBlock) * VEC, x[u]);
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i + u * kBlock < nv) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) x[u][j] = coef(x[u][j]);
          store_elems_nt<VEC>(dst + (size_t)(i + u * kBlock) * VEC, x[u]);
        }
    }
    for (int i = nv * VEC + threadIdx.x; i < n; i += kBlock) dst[i] = (TD)coef((float)src[i]);
  } else {
    for (int i = threadIdx.x; i < n; i += 4 * U * kBlock) {
      float x[4 * U];
#pragma unroll
      for (int u = 0; u < 4 * U; ++u) x[u] = (float)src[min(i + u * kBlock, n - 1)];
#pragma unroll
      for (int u = 0; u < 4 * U; ++u)
        if (i + u * kBlock < n) dst[i + u * kBlock] = (TD)coef(x[u]);
    }
  }
}

// Chunks in descending order: the norm pass read the last ones last, so they are still cached.
template <bool INF>
__global__ __launch_bounds__(kBlock) void clip_scale_kernel(ClipList l, const double* __restrict__ parts, int np,
                                                            double max_norm, float* __restrict__ norm) {
  const double v = joined_norm<INF>(parts, np);
  const Coef coef = clip_coef(v, max_norm);
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)v;
  const int chunks = l.first[l.count];
  for (int c = chunks - 1 - (int)blockIdx.x; c >= 0; c -= gridDim.x) {
    const int t = tensor_of(l, c);
    const int64_t at = (int64_t)(c - l.first[t]) * l.chunk;
    const int n = c + 1 < l.first[t + 1] ? l.chunk : last_of(l, t);
    const int ty = type_of(l, t);
    if (coef.a == 1.f && coef.b == 1.f && l.src[t] == l.dst[t]) continue;  // in place and not clipped: nothing changes
#define TT_SC(TS, TD) scale_chunk<TS, TD>(static_cast<const TS*>(l.src[t]) + at, static_cast<TD*>(l.dst[t]) + at, n, coef)
    if (ty == (TT_E_F32 | TT_E_F32 << 2)) TT_SC(float, float);
    else if (ty == (TT_E_BF16 | TT_E_BF16 << 2)) TT_SC(__bf16, __bf16);
    else if (ty == (TT_E_F16 | TT_E_F16 << 2)) TT_SC(_Float16, _Float16);
    else if (ty == (TT_E_BF16 | TT_E_F32 << 2)) TT_SC(__bf16, float);
    else TT_SC(_Float16, float);
#undef TT_SC
  }
}

// the call's tensors, as the caller's host arrays
struct ClipCall {
  const void* const* src;
  void* const* dst;
  const int64_t* n;
  const uint8_t* src_dtype;
  const uint8_t* dst_dtype;
  int count;
};

// tensors [at, at + TT_CLIP_MAX_TENSORS) of the call as one launch's list
void fill_list(ClipList& l, const ClipCall& t, int at) {
  const int m = t.count - at < TT_CLIP_MAX_TENSORS ? t.count - at : TT_CLIP_MAX_TENSORS;
  // smaller chunks where there are few: a workgroup's time is then its latencies
  int64_t total = 0, chunk = 0;
  for (int i = 0; i < m; ++i) total += t.n[at + i];
  l.chunk = kChunk;
  while (l.chunk > kMinChunk && total < (int64_t)l.chunk * 1024) l.chunk >>= 1;
  for (int i = 0; i < m; ++i) {
    l.src[i] = t.src[at + i];
    l.dst[i] = t.dst[at + i];
    if (i % 2 == 0) l.last2[i / 2] = 0;
    if (i % 4 == 0) l.type4[i / 4] = 0;
    l.type4[i / 4] |= (uint32_t)(t.src_dtype[at + i] | t.dst_dtype[at + i] << 2) << i % 4 * 8;
    l.first[i] = (int32_t)chunk;
    const int64_t chunks = (t.n[at + i] + l.chunk - 1) / l.chunk;
    l.last2[i / 2] |= (uint32_t)(t.n[at + i] - (chunks - 1) * l.chunk) << i % 2 * 16;
    chunk += chunks;
  }
  l.first[m] = (int32_t)chunk;
  l.count = m;
}

template <bool INF>
int run_clip(const ClipCall& t, bool scale, double max_norm, float* norm, double* parts,
             hipStream_t s) {
  const int count = t.count, launches = (count + TT_CLIP_MAX_TENSORS - 1) / TT_CLIP_MAX_TENSORS;
  int cap = launches > 0 ? kMaxParts / launches : 1;
  cap = cap < 1 ? 1 : cap > kNormBlocks ? kNormBlocks : cap;
  static_assert(sizeof(ClipList) <= 4096 - 64, "kernel arguments");  // (4 KB, with the others)
  ClipList l;
  int np = 0;
  for (int at = 0; at < count; at += TT_CLIP_MAX_TENSORS) {
    fill_list(l, t, at);
    const int chunks = l.first[l.count];
    if (chunks == 0) continue;
    const int g = chunks < cap ? chunks : cap;
    clip_norm_kernel<INF><<<dim3(g), dim3(kBlock), 0, s>>>(l, parts + np);
    TT_LAUNCH_CHECK("clip_norm");
    np += g;
  }
  bool wrote = false;
  if (scale)
    for (int at = 0; at < count; at += TT_CLIP_MAX_TENSORS) {
      if (launches > 1) fill_list(l, t, at);
      const int chunks = l.first[l.count];
      if (chunks == 0) continue;
      const int g = chunks < kScaleBlocks ? chunks : kScaleBlocks;
      clip_scale_kernel<INF><<<dim3(g), dim3(kBlock), 0, s>>>(l, parts, np, max_norm, wrote ? nullptr : norm);
      TT_LAUNCH_CHECK("clip_scale");
      wrote = true;
    }
  if (!wrote) {
    clip_finish_kernel<INF><<<dim3(1), dim3(kBlock), 0, s>>>(parts, np, norm);
    TT_LAUNCH_CHECK("clip_finish");
  }
  return TT_OK;
}

}  // namespace
}  // namespace tt

using namespace tt;

extern "C" size_t tt_clip_ws_size(int count) {
  const int64_t launches = ((int64_t)(count > 0 ? count : 1) + TT_CLIP_MAX_TENSORS - 1) / TT_CLIP_MAX_TENSORS;
  return sizeof(double) * (size_t)(launches > kMaxParts ? launches : kMaxParts);
}

extern "C" int tt_clip_grads(const void* const* src, void* const* dst, const int64_t* n, const uint8_t* src_dtype,
                             const uint8_t* dst_dtype, int count, int inf_norm, double max_norm, int scale,
                             float* norm, void* ws, size_t ws_bytes, tt_stream_t stream) {
  TT_REQUIRE(count >= 0 && ((src && dst && n && src_dtype && dst_dtype) || count == 0) && norm,
             "clip: null pointer or count=%d", count);
  TT_REQUIRE(!scale || max_norm >= 0.0, "clip: max_norm must not be negative");
  TT_REQUIRE(ws && ws_bytes >= tt_clip_ws_size(count) && reinterpret_cast<size_t>(ws) % 8 == 0,
             "workspace too small: need %zu have %zu", tt_clip_ws_size(count), ws_bytes);
  int64_t chunks = 0;  // of one launch, counted in 32 bits
  for (int i = 0; i < count; ++i) {
    TT_REQUIRE(n[i] >= 0 && n[i] < (int64_t(1) << 44), "clip: tensor %d has %lld elements", i, (long long)n[i]);
    TT_REQUIRE(n[i] == 0 || (src[i] && (!scale || dst[i])), "clip: tensor %d is NULL", i);
    TT_REQUIRE(elem_ok(src_dtype[i]) && elem_ok(dst_dtype[i]) &&
                   (dst_dtype[i] == src_dtype[i] || dst_dtype[i] == TT_E_F32),
               "clip: tensor %d of type %d into type %d", i, src_dtype[i], dst_dtype[i]);
    chunks = (i % TT_CLIP_MAX_TENSORS ? chunks : 0) + (n[i] + kChunk - 1) / kChunk;
    TT_REQUIRE(chunks < (int64_t(1) << 31) - kScaleBlocks, "clip: too many elements");
  }
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  double* parts = static_cast<double*>(ws);
  const ClipCall t{src, dst, n, src_dtype, dst_dtype, count};
  return inf_norm ? run_clip<true>(t, scale != 0, max_norm, norm, parts, s)
                  : run_clip<false>(t, scale != 0, max_norm, norm, parts, s);
}
