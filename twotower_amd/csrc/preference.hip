// Paired preference loss on tower outputs.
//
// Under the softmax the towers are trained with (logits q . d / tau) the normaliser cancels in a log
// ratio of two documents of one query, log P(p|q) - log P(n|q) = (q.p - q.n) / tau.  With r the same
// ratio under a frozen reference model, pair (i, k) has the margin
//   h = q_i . (p_i - n_ik) / tau - r_ik
// and the loss is the mean over the valid pairs of
//   sigmoid:  (1 - e) softplus(-b h) + e softplus(b h)      l'(h) = b (e - sigma(-b h))
//   squared:  (h - 1 / (2 b))^2                             l'(h) = 2 (h - 1 / (2 b))
// With c_ik = l'(h_ik) and G = upstream / (pairs tau):
//   dq_i = G sum_k c_ik (p_i - n_ik),   dp_i = G (sum_k c_ik) q_i,   dn_ik = -G c_ik q_i.
// A masked pair is not read, counts nothing and gets a zero gradient; no valid pair: loss 0.
// Row passes, bound by their bytes (forward: q, p, n once; backward: again, and the gradients): 8192 x 256 fp32,
// one negative: forward 7.9 us + 3.0 for the mean (25 MB), backward 8.8 (50 MB, 5.7 TB/s); bf16, four
// negatives: 7.5 + 3.0 and 8.9 us.  A group of lanes takes a query and up to kKT of its pairs at once: q and p are
// then read once however many pairs there are up to that, and a row's loads are all in flight together (a masked
// pair's from p again: behind a condition the backward's waited, 9.3 instead of 8.9 us).
// The differences p - n are formed before the products, so two close documents lose nothing to
// cancellation.  One workgroup does all of a small batch, the mean included (64 x 128: 5.0 us, one launch).
#include "common.hpp"

#include <algorithm>

namespace tt {
namespace {

constexpr int kBlock = 256;
constexpr int kFinish = 1024;  // the one workgroup that joins the rows
constexpr int kKT = 4;         // pairs of a query in flight (a query with one has a form of its own)

constexpr int64_t kFewWaves = 4096;  // what the card runs at half its residence

enum { kSigmoid = 0, kSquared = 1 };

struct PrefArgs {
  int64_t B;
  int K, H;
  int64_t ldq, ldp, ldnb, ldnk;
  const float* ref;
  const uint8_t* mask;
  int kind;
  float beta, inv_tau, smooth;
};

__device__ __forceinline__ bool pair_valid(const PrefArgs& a, int64_t i, int k) {
  return !a.mask || a.mask[i * a.K + k] != 0;
}

__device__ __forceinline__ void pair_loss(const PrefArgs& a, float h, float& loss, float& dl) {
  if (a.kind == kSigmoid) {
    const float x = a.beta * h, t = expf(-fabsf(x)), tail = log1pf(t);
    const float neg = (x >= 0.f ? t : 1.f) / (1.f + t);  // sigma(-x)
    loss = (1.f - a.smooth) * (fmaxf(-x, 0.f) + tail);
    if (a.smooth != 0.f) loss += a.smooth * (fmaxf(x, 0.f) + tail);  // (0 * inf would be NaN)
    dl = a.beta * (a.smooth - neg);
  } else {
    const float d = h - 0.5f / a.beta;
    loss = d * d;
    dl = 2.f * d;
  }
}

// One group of 2^lg lanes: query i's pairs.  Returns (in every lane) the row's loss sum and count.
template <typename T, int VEC, int KT>
__device__ __forceinline__ void pref_row(const PrefArgs& a, const T* __restrict__ q, const T* __restrict__ p,
                                         const T* __restrict__ n, int64_t i, int c, int lg, float* __restrict__ coef,
                                         float* __restrict__ margins, float& sum, int& count) {
  sum = 0.f;
  count = 0;
  const T *qi = q + i * a.ldq, *pi = p + i * a.ldp, *ni = n + i * a.ldnb;
  for (int k0 = 0; k0 < a.K; k0 += KT) {
    bool on[KT], any = false;
#pragma unroll
    for (int k = 0; k < KT; ++k) {
      on[k] = k0 + k < a.K && pair_valid(a, i, k0 + k);
      any = any || on[k];
    }
    float dot[KT] = {};
    if (any) {
      for (int e = c * VEC; e < a.H; e += VEC << lg) {
        float x[VEC], y[VEC], z[KT][VEC];
        load_elems<VEC>(qi + e, x);
        load_elems<VEC>(pi + e, y);
#pragma unroll
        for (int k = 0; k < KT; ++k)
          load_elems<VEC>((on[k] ? ni + (k0 + k) * a.ldnk : pi) + e, z[k]);
#pragma unroll
        for (int k = 0; k < KT; ++k)
          if (on[k]) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) dot[k] = __builtin_fmaf(x[j], y[j] - z[k][j], dot[k]);
          }
      }
    }
    for (int o = 1; o < 1 << lg; o <<= 1) {
#pragma unroll
      for (int k = 0; k < KT; ++k) dot[k] += __shfl_xor(dot[k], o);
    }
    // every lane has the products: lanes c, c + 4, ... take pair c's loss, or each lane all of them where a group
    // has fewer lanes (one after the other in every lane, 16 x 256 with 8 pairs took 11 us instead of 7)
    float part = 0.f;
    auto pair = [&](int m, float s, bool valid, bool writes) {
      const int64_t at = i * a.K + k0 + m;
      float h = 0.f, loss = 0.f, dl = 0.f;
      if (valid) {
        h = s * a.inv_tau - (a.ref ? a.ref[at] : 0.f);
        pair_loss(a, h, loss, dl);
      }
      part += loss;
      if (writes && k0 + m < a.K) {
        if (coef) coef[at] = dl;
        if (margins) margins[at] = h;
      }
    };
    if (KT == 4 && lg >= 2) {
      const int m = c & 3;
      float s = dot[0];
      bool valid = on[0];
#pragma unroll
      for (int k = 1; k < KT; ++k) {
        s = m == k ? dot[k] : s;
        valid = m == k ? on[k] : valid;
      }
      pair(m, s, valid, c < 4);
      part += __shfl_xor(part, 1);
      part += __shfl_xor(part, 2);
    } else {
#pragma unroll
      for (int k = 0; k < KT; ++k) pair(k, dot[k], on[k], c == 0);
    }
    sum += part;
#pragma unroll
    for (int k = 0; k < KT; ++k) count += on[k];
  }
}

// loss = sum / max(count, 1) and 1 / max(count, 1), the sums folded in a fixed order.
__device__ __forceinline__ void pref_finish(double sum, double count, float* loss, float* inv_pairs) {
  __shared__ double ss[kFinish / kWave], sc[kFinish / kWave];
  const int t = threadIdx.x;
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    sum += __shfl_xor(sum, o);
    count += __shfl_xor(count, o);
  }
  if (lane_id() == 0) {
    ss[t >> 6] = sum;
    sc[t >> 6] = count;
  }
  __syncthreads();
  if (t == 0) {
    for (int w = 1; w < kFinish / kWave; ++w) {
      sum += ss[w];
      count += sc[w];
    }
    const double inv = 1.0 / (count > 1.0 ? count : 1.0);
    *loss = (float)(sum * inv);
    *inv_pairs = (float)inv;
  }
}

template <typename T, int VEC, int KT>
__global__ __launch_bounds__(kBlock) void pref_fwd_kernel(PrefArgs a, const T* __restrict__ q, const T* __restrict__ p,
                                                          const T* __restrict__ n, int lg, float* __restrict__ coef,
                                                          float* __restrict__ margins, float* __restrict__ rows,
                                                          int32_t* __restrict__ counts) {
  const int lane = lane_id(), sub = lane >> lg, c = lane & ((1 << lg) - 1);
  const int64_t i = ((block_index() * kBlock + threadIdx.x) >> 6) * (kWave >> lg) + sub;
  if (i >= a.B) return;
  float sum;
  int count;
  pref_row<T, VEC, KT>(a, q, p, n, i, c, lg, coef, margins, sum, count);
  if (c == 0 && rows) {
    rows[i] = sum;
    counts[i] = count;
  }
}

// the same and the mean in one launch, for a batch that one workgroup passes in a few rounds
template <typename T, int VEC, int KT>
__global__ __launch_bounds__(kFinish) void pref_fwd_small_kernel(PrefArgs a, const T* __restrict__ q,
                                                                 const T* __restrict__ p, const T* __restrict__ n,
                                                                 int lg, float* __restrict__ coef,
                                                                 float* __restrict__ margins, float* __restrict__ loss,
                                                                 float* __restrict__ inv_pairs) {
  const int lane = lane_id(), sub = lane >> lg, c = lane & ((1 << lg) - 1);
  double ds = 0.0, dc = 0.0;
  for (int64_t i = (int64_t)(threadIdx.x >> 6) * (kWave >> lg) + sub; i < a.B; i += kFinish >> lg) {
    float sum;
    int count;
    pref_row<T, VEC, KT>(a, q, p, n, i, c, lg, coef, margins, sum, count);
    if (c == 0) {
      ds += (double)sum;
      dc += (double)count;
    }
  }
  pref_finish(ds, dc, loss, inv_pairs);
}

__global__ __launch_bounds__(kFinish) void pref_mean_kernel(const float* __restrict__ rows,
                                                            const int32_t* __restrict__ counts, int64_t B,
                                                            float* __restrict__ loss, float* __restrict__ inv_pairs) {
  double s = 0.0, c = 0.0;
  constexpr int U = 8;  // loads in flight (one at a time: 4.1 us instead of 3.0 for 8192 rows)
  for (int64_t i = threadIdx.x; i < B; i += U * kFinish) {
    float x[U];
    int32_t n[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t k = min(i + u * kFinish, B - 1);
      x[u] = rows[k];
      n[u] = counts[k];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      s += i + u * kFinish < B ? (double)x[u] : 0.0;
      c += i + u * kFinish < B ? (double)n[u] : 0.0;
    }
  }
  pref_finish(s, c, loss, inv_pairs);
}

template <typename T, int VEC>
__global__ __launch_bounds__(kBlock) void pref_bwd_kernel(PrefArgs a, const T* __restrict__ q, const T* __restrict__ p,
                                                          const T* __restrict__ n, int lg,
                                                          const float* __restrict__ coef,
                                                          const float* __restrict__ inv_pairs,
                                                          const float* __restrict__ grad_loss, T* __restrict__ dq,
                                                          T* __restrict__ dp, T* __restrict__ dn) {
  const int lane = lane_id(), sub = lane >> lg, c = lane & ((1 << lg) - 1);
  const int64_t i = ((block_index() * kBlock + threadIdx.x) >> 6) * (kWave >> lg) + sub;
  if (i >= a.B) return;
  const float G = grad_loss[0] * (inv_pairs[0] * a.inv_tau);
  const T *qi = q + i * a.ldq, *pi = p + i * a.ldp, *ni = n + i * a.ldnb;
  const float* ci = coef + i * a.K;
  float csum = 0.f;  // (a masked pair's coefficient is 0)
  int any = 0;
  if (a.K <= kKT) {
#pragma unroll
    for (int k = 0; k < kKT; ++k)
      if (k < a.K) {
        csum += ci[k];
        any |= pair_valid(a, i, k);
      }
  } else {
    for (int k = c; k < a.K; k += 1 << lg) {
      csum += ci[k];
      any |= pair_valid(a, i, k);
    }
    for (int o = 1; o < 1 << lg; o <<= 1) {
      csum += __shfl_xor(csum, o);
      any |= __shfl_xor(any, o);
    }
  }
  csum *= G;
  // (the grid's z chunks of a row's columns run side by side)
  for (int64_t e = (((int64_t)blockIdx.z << lg) + c) * VEC; e < a.H; e += (int64_t)(VEC << lg) * gridDim.z) {
    float x[VEC] = {}, y[VEC] = {}, gq[VEC] = {}, gp[VEC] = {};
    if (any) {
      load_elems<VEC>(qi + e, x);
      load_elems<VEC>(pi + e, y);
    }
    for (int k0 = 0; k0 < a.K; k0 += kKT) {
      bool on[kKT];
      float z[kKT][VEC];
#pragma unroll
      for (int k = 0; k < kKT; ++k) {
        on[k] = k0 + k < a.K && pair_valid(a, i, k0 + k);
        load_elems<VEC>((on[k] ? ni + (k0 + k) * a.ldnk : pi) + e, z[k]);
      }
#pragma unroll
      for (int k = 0; k < kKT; ++k) {
        if (k0 + k >= a.K) break;
        float g[VEC] = {};
        if (on[k]) {
          const float ck = ci[k0 + k] * G;
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            gq[j] = __builtin_fmaf(ck, y[j] - z[k][j], gq[j]);
            g[j] = -ck * x[j];
          }
        }
        store_elems<VEC>(dn + (i * a.K + k0 + k) * a.H + e, g);
      }
    }
    if (any) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) gp[j] = csum * x[j];
    }
    store_elems<VEC>(dq + i * a.H + e, gq);
    store_elems<VEC>(dp + i * a.H + e, gp);
  }
}

template <typename T>
int pref_vec(const PrefArgs& a, const void* const* ptrs, int np) {
  const int64_t counts[] = {a.H, a.ldq, a.ldp, a.ldnb, a.ldnk};
  int bytes[6];
  for (int i = 0; i < np; ++i) bytes[i] = sizeof(T);
  const int v = vec_for(counts, 5, ptrs, bytes, np);
  return sizeof(T) == 4 && v > 4 ? 4 : v;
}

inline int lanes_log2(int H, int vec) {
  int l = 0;
  while (l < 6 && (vec << l) < H) ++l;
  return l;
}

#define TT_PREF_VEC(vec, CALL)        \
  switch (vec) {                      \
    case 8: CALL(8); break;           \
    case 4: CALL(4); break;           \
    case 2: CALL(2); break;           \
    default: CALL(1); break;          \
  }

template <typename T>
int launch_pref_fwd(const PrefArgs& a, const void* q, const void* p, const void* n, float* coef, float* margins,
                    float* rows, int32_t* counts, float* loss, float* inv_pairs, hipStream_t s) {
  const void* ptrs[] = {q, p, n};
  const int vec = pref_vec<T>(a, ptrs, 3), lg = lanes_log2(a.H, vec);
  const T *tq = static_cast<const T*>(q), *tp = static_cast<const T*>(p), *tn = static_cast<const T*>(n);
  // one workgroup, and no launch for the mean, while it has its rows, pairs and columns in two steps (us, it and the
  // two launches: one step, 16 x 256 4.0 and 5.4; two, 64 x 128 5.2 and 5.3; four, 64 x 256 8.0 and 5.4)
  const int64_t rounds = ((a.B << lg) + kFinish - 1) / kFinish, chunks = (a.H + (vec << lg) - 1) / (vec << lg);
  if (loss && rounds * chunks * ((a.K + kKT - 1) / kKT) <= 2) {
#define TT_CALL(V) (a.K == 1 ? pref_fwd_small_kernel<T, V, 1> : pref_fwd_small_kernel<T, V, kKT>)<<<dim3(1), dim3(kFinish), 0, s>>>(a, tq, tp, tn, lg, coef, margins, loss, inv_pairs)
    TT_PREF_VEC(vec, TT_CALL)
#undef TT_CALL
    TT_LAUNCH_CHECK("preference_fwd_small");
    return TT_OK;
  }
  const int64_t per = (kBlock / kWave) * (kWave >> lg);
  if (a.B > 0) {
    const dim3 grid = wide_grid((a.B + per - 1) / per), block(kBlock);
#define TT_CALL(V) (a.K == 1 ? pref_fwd_kernel<T, V, 1> : pref_fwd_kernel<T, V, kKT>)<<<grid, block, 0, s>>>(a, tq, tp, tn, lg, coef, margins, loss ? rows : nullptr, counts)
    TT_PREF_VEC(vec, TT_CALL)
#undef TT_CALL
    TT_LAUNCH_CHECK("preference_fwd");
  }
  if (loss) {
    pref_mean_kernel<<<dim3(1), dim3(kFinish), 0, s>>>(rows, counts, a.B, loss, inv_pairs);
    TT_LAUNCH_CHECK("preference_mean");
  }
  return TT_OK;
}

template <typename T>
int launch_pref_bwd(const PrefArgs& a, const void* q, const void* p, const void* n, const float* coef,
                    const float* inv_pairs, const float* grad_loss, void* dq, void* dp, void* dn, hipStream_t s) {
  const void* ptrs[] = {q, p, n, dq, dp, dn};
  const int vec = pref_vec<T>(a, ptrs, 6), lg = lanes_log2(a.H, vec);
  const int64_t per = (kBlock / kWave) * (kWave >> lg);
  const dim3 block(kBlock);
  dim3 grid = wide_grid((a.B + per - 1) / per);
  // a wide row's column chunks side by side where there are few rows (33 x 382 fp16, 8 pairs: 11 us one after the
  // other, 6 side by side; 5236 x 181 bf16, 3 pairs: 10 and 12)
  const int64_t chunks = (a.H + (vec << lg) - 1) / (vec << lg), waves = (a.B << lg) / kWave + 1;
  grid.z = (unsigned)std::min(chunks, (kFewWaves + waves - 1) / waves);
#define TT_CALL(V)                                                                                              \
  pref_bwd_kernel<T, V><<<grid, block, 0, s>>>(a, static_cast<const T*>(q), static_cast<const T*>(p),           \
                                               static_cast<const T*>(n), lg, coef, inv_pairs, grad_loss,          \
                                               static_cast<T*>(dq), static_cast<T*>(dp), static_cast<T*>(dn))
  TT_PREF_VEC(vec, TT_CALL)
#undef TT_CALL
  TT_LAUNCH_CHECK("preference_bwd");
  return TT_OK;
}

int check_pref(const PrefArgs& a, const void* q, const void* p, const void* n, int dtype) {
  TT_REQUIRE(elem_ok(dtype), "preference: element type %d", dtype);
  TT_REQUIRE(a.B >= 0 && a.K >= 1 && a.H >= 1, "preference: bad shape B=%lld K=%d H=%d", (long long)a.B, a.K, a.H);
  TT_REQUIRE(a.B < (int64_t(1) << 31) && a.B * (int64_t)a.K < (int64_t(1) << 31), "preference: too many pairs");
  TT_REQUIRE(a.B == 0 || (q && p && n), "null pointer");
  TT_REQUIRE(a.kind == kSigmoid || a.kind == kSquared, "preference: loss kind %d", a.kind);
  TT_REQUIRE(a.beta > 0.f && a.inv_tau > 0.f && a.smooth >= 0.f && a.smooth < 1.f,
             "preference: beta and temperature must be positive and smoothing in [0, 1)");
  return TT_OK;
}

}  // namespace
}  // namespace tt

using namespace tt;

extern "C" int tt_preference_fwd(const void* q, int64_t ldq, const void* p, int64_t ldp, const void* n, int64_t ldn_b,
                                 int64_t ldn_k, int dtype, int64_t B, int K, int H, const float* ref,
                                 const uint8_t* mask, int kind, float beta, float inv_tau, float smoothing,
                                 float* coef, float* margins, float* loss, float* inv_pairs, void* ws, size_t ws_bytes,
                                 tt_stream_t stream) {
  const PrefArgs a{B, K, H, ldq, ldp, ldn_b, ldn_k, ref, mask, kind, beta, inv_tau, smoothing};
  if (int rc = check_pref(a, q, p, n, dtype)) return rc;
  TT_REQUIRE(!loss || inv_pairs, "null pointer");
  TT_REQUIRE(!loss || B == 0 || (ws && ws_bytes >= (size_t)B * 8), "workspace too small: need %lld bytes",
             (long long)B * 8);
  float* rows = static_cast<float*>(ws);
  int32_t* counts = reinterpret_cast<int32_t*>(rows + B);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (dtype == TT_E_F32) return launch_pref_fwd<float>(a, q, p, n, coef, margins, rows, counts, loss, inv_pairs, s);
  if (dtype == TT_E_BF16) return launch_pref_fwd<__bf16>(a, q, p, n, coef, margins, rows, counts, loss, inv_pairs, s);
  return launch_pref_fwd<_Float16>(a, q, p, n, coef, margins, rows, counts, loss, inv_pairs, s);
}

extern "C" int tt_preference_bwd(const void* q, int64_t ldq, const void* p, int64_t ldp, const void* n, int64_t ldn_b,
                                 int64_t ldn_k, int dtype, int64_t B, int K, int H, const uint8_t* mask,
                                 float inv_tau, const float* coef, const float* inv_pairs, const float* grad_loss,
                                 void* dq, void* dp, void* dn, tt_stream_t stream) {
  const PrefArgs a{B, K, H, ldq, ldp, ldn_b, ldn_k, nullptr, mask, kSigmoid, 1.f, inv_tau, 0.f};
  if (int rc = check_pref(a, q, p, n, dtype)) return rc;
  if (B == 0) return TT_OK;
  TT_REQUIRE(coef && inv_pairs && grad_loss && dq && dp && dn, "null pointer");
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (dtype == TT_E_F32) return launch_pref_bwd<float>(a, q, p, n, coef, inv_pairs, grad_loss, dq, dp, dn, s);
  if (dtype == TT_E_BF16) return launch_pref_bwd<__bf16>(a, q, p, n, coef, inv_pairs, grad_loss, dq, dp, dn, s);
  return launch_pref_bwd<_Float16>(a, q, p, n, coef, inv_pairs, grad_loss, dq, dp, dn, s);
}
