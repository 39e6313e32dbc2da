// Preference loss over pairs of answers, from logits, and its gradient.
//
// The logits are all that counts: (tokens, vocab) read once forward (a running maximum and sum of exponentials),
// read again and answered with the gradient backward; ignored tokens' logits are not read at all. Both passes are bound
// by memory: for 8200 of 16384 rows of 50280 bf16 values 151 us (5.5 TB/s) and 383 us (6.4 TB/s, with the zeros of the
// ignored rows), for 1865 of 3108 rows of 50277 float32 values 77 us (4.9 TB/s) and 158 us (6.3 TB/s). Sums over the
// tokens of an answer and over the pairs are taken in 64 bits and in a fixed order: an answer's log-probability
// is a sum of a thousand values near -10 of which the loss sees small differences.
#include "mm_common.cuh"

namespace mm {
namespace pref {

constexpr int kThreads = 512;
// Forward with the loss, repeated on the same rows: 8200 rows of 50280 bf16 values in blocks of 64, 128, 256 and 512
// threads 151, 149, 163 and 190 us (without loading ahead 152, 149, 157, 189), 1865 rows of 50277 float32 values in
// 128, 256 and 512 81, 77 and 81.
template <typename T> constexpr int kStatsThreads = sizeof(T) == 4 ? 256 : 128;

struct Params {
  const void* logits;
  const int64_t* labels;
  const float* ref;
  float *loss, *chosen, *rejected, *stats, *slope;
  const float* grad_loss;
  void* dlogits;
  double* gain;  // beta (logp - ref) of every answer
  unsigned* done;  // answers whose gain is there
  float4* part;  // of every (token, split): maximum, sum of exp(x - maximum), the label's logit
  long long ls[2], ds[2];
  long long tokens;
  long long ignore;
  int pairs, length, vocab, splits;
  double beta, smoothing;
};

// Scalar elements before the first 16-byte boundary of p, at most n
template <typename T> MM_DEV int head_of(const T* p, int n) {
  const int h = (int)((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / (int)sizeof(T);
  return min(h, n);
}
template <typename T> constexpr int kVec = 16 / (int)sizeof(T);

struct MaxSum {
  float m, s;  // the sum is relative to base(m)
};
// A maximum of -inf (no finite value so far) leaves sums relative to 0, which are 0; its own factor on the way
// to another maximum is exp(-inf) = 0
MM_DEV float base(float m) { return m == -INFINITY ? 0.f : m; }
MM_DEV MaxSum join(MaxSum a, MaxSum b) {
  MaxSum r;
  r.m = fmaxf(a.m, b.m);
  const float z = base(r.m);
  r.s = a.s * ex2((a.m - z) * kLog2e) + b.s * ex2((b.m - z) * kLog2e);
  return r;
}

template <typename T>
__global__ void __launch_bounds__(kStatsThreads<T>) stats_kernel(const Params p) {
  if (blockIdx.x == 0 && threadIdx.x == 0) *p.done = 0;  // for loss_kernel, which follows
  const long long token = blockIdx.x / p.splits;
  const int split = (int)(blockIdx.x % p.splits);
  const long long label = p.labels[token];
  if (label == p.ignore) return;
  const T* x = static_cast<const T*>(p.logits) + token / p.length * p.ls[0] + token % p.length * p.ls[1];
  const int head = head_of(x, p.vocab);
  const int nv = (p.vocab - head) / kVec<T>;
  const int v0 = (int)((long long)nv * split / p.splits), v1 = (int)((long long)nv * (split + 1) / p.splits);
  MaxSum a = {-INFINITY, 0.f};
  auto add1 = [&](float v) {
    const float m = fmaxf(a.m, v), z = base(m);
    a.s = a.s * ex2((a.m - z) * kLog2e) + ex2((v - z) * kLog2e);
    a.m = m;
  };
  const uint4* xv = reinterpret_cast<const uint4*>(x + head);
  constexpr int kU = 4;  // vectors that are on their way while as many are worked on
  uint4 q[kU], next[kU];
  auto load = [&](uint4 (&r)[kU], int i) {
#pragma unroll
    for (int u = 0; u < kU; ++u)
      if (i + u * kStatsThreads<T> < v1) r[u] = xv[i + u * kStatsThreads<T>];
  };
  load(q, v0 + threadIdx.x);
  for (int i = v0 + threadIdx.x; i < v1; i += kU * kStatsThreads<T>) {
    load(next, i + kU * kStatsThreads<T>);
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      if (i + u * kStatsThreads<T> >= v1) break;
      float m = a.m;
#pragma unroll
      for (int k = 0; k < kVec<T>; ++k) m = fmaxf(m, vec_elem<T>(q[u], k));
      const float z = base(m);  // subtracted before the scaling: exact near the maximum, finite for rows at -3.4e38
      float s = 0.f;
#pragma unroll
      for (int k = 0; k < kVec<T>; ++k) s += ex2((vec_elem<T>(q[u], k) - z) * kLog2e);
      a.s = fmaf(a.s, ex2((a.m - z) * kLog2e), s);
      a.m = m;
    }
#pragma unroll
    for (int u = 0; u < kU; ++u) q[u] = next[u];
  }
  if (split == 0)
    for (int i = threadIdx.x; i < head; i += kStatsThreads<T>) add1(ld_f32(x + i));
  if (split == p.splits - 1)
    for (int i = head + nv * kVec<T> + threadIdx.x; i < p.vocab; i += kStatsThreads<T>) add1(ld_f32(x + i));
#pragma unroll
  for (int h = 16; h > 0; h >>= 1) {
    MaxSum b;
    b.m = __shfl_xor_sync(0xffffffffu, a.m, h);
    b.s = __shfl_xor_sync(0xffffffffu, a.s, h);
    a = join(a, b);
  }
  __shared__ MaxSum warp[kStatsThreads<T> / 32];
  if ((threadIdx.x & 31) == 0) warp[threadIdx.x >> 5] = a;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kStatsThreads<T> / 32; ++w) a = join(a, warp[w]);
    const bool valid = label >= 0 && label < p.vocab;
    p.part[token * p.splits + split] = make_float4(a.m, a.s, valid ? ld_f32(x + label) : __uint_as_float(0x7fffffffu), 0.f);
  }
}

MM_DEV double softplus64(double v) { return fmax(v, 0.0) + log1p(exp(-fabs(v))); }
MM_DEV double sigmoid64(double v) { return 1.0 / (1.0 + exp(-v)); }

// A CTA per answer joins the splits and sums the answer's tokens; the last one to finish takes the pairs' losses. One
// launch in place of two; 5 us for answers of two tokens, 9 for 1024, the latency of the 64-bit logarithms and sums.
constexpr int kLossThreads = 256;
MM_DEV double block_sum(double v, double* warps) {  // in a fixed order; the result is thread 0's
#pragma unroll
  for (int h = 16; h > 0; h >>= 1) v += __shfl_xor_sync(0xffffffffu, v, h);
  if ((threadIdx.x & 31) == 0) warps[threadIdx.x >> 5] = v;
  __syncthreads();
  if (threadIdx.x == 0)
    for (int w = 1; w < kLossThreads / 32; ++w) v += warps[w];
  return v;
}
__global__ void __launch_bounds__(kLossThreads) loss_kernel(const Params p) {
  __shared__ double warps[kLossThreads / 32];
  __shared__ bool last;
  const int r = blockIdx.x;
  double sum = 0;
  for (int t = threadIdx.x; t < p.length; t += kLossThreads) {
    const long long token = (long long)r * p.length + t;
    if (p.labels[token] == p.ignore) continue;
    float4 a = p.part[token * p.splits];
    MaxSum ms = {a.x, a.y};
    for (int i = 1; i < p.splits; ++i) {
      const float4 b = p.part[token * p.splits + i];
      ms = join(ms, MaxSum{b.x, b.y});
    }
    p.stats[2 * token] = ms.m;
    p.stats[2 * token + 1] = ms.s;
    sum += (double)a.z - (double)ms.m - log((double)ms.s);
  }
  sum = block_sum(sum, warps);
  if (threadIdx.x == 0) {
    const double gain = p.beta * (sum - (double)p.ref[r]);
    p.gain[r] = gain;
    if (r < p.pairs)
      p.chosen[r] = (float)gain;
    else
      p.rejected[r - p.pairs] = (float)gain;
    __threadfence();  // the gain is there before the count says so
    last = atomicAdd(p.done, 1u) == 2u * p.pairs - 1u;
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  double loss = 0;
  for (int i = threadIdx.x; i < p.pairs; i += kLossThreads) {
    const double m = __ldcg(p.gain + i) - __ldcg(p.gain + p.pairs + i);
    loss += (1.0 - p.smoothing) * softplus64(-m) + p.smoothing * softplus64(m);
    const double dm = (p.smoothing * sigmoid64(m) - (1.0 - p.smoothing) * sigmoid64(-m)) * p.beta / p.pairs;
    p.slope[i] = (float)dm;
    p.slope[p.pairs + i] = (float)-dm;
  }
  loss = block_sum(loss, warps);
  if (threadIdx.x == 0) *p.loss = (float)(loss / p.pairs);
}

// dlogits of one (token, split of the vocabulary). Tokens run from the last to the first: the forward pass read
// them in order, so the last ones' logits are what L2 (126 MB) still holds.
template <typename T>
__global__ void __launch_bounds__(kThreads) grad_kernel(const Params p) {
  const long long block = (long long)gridDim.x - 1 - blockIdx.x;
  const long long token = block / p.splits;
  const int split = (int)(block % p.splits);
  const long long label = p.labels[token];
  T* dx = static_cast<T*>(p.dlogits) + token / p.length * p.ds[0] + token % p.length * p.ds[1];
  const int head = head_of(dx, p.vocab);
  const int nv = (p.vocab - head) / kVec<T>;
  const int v0 = (int)((long long)nv * split / p.splits), v1 = (int)((long long)nv * (split + 1) / p.splits);
  uint4* dv = reinterpret_cast<uint4*>(dx + head);
  const int tail = head + nv * kVec<T>;
  if (label == p.ignore) {
    for (int i = v0 + threadIdx.x; i < v1; i += kThreads) __stcs(dv + i, make_uint4(0, 0, 0, 0));
    if (split == 0)
      for (int i = threadIdx.x; i < head; i += kThreads) st_f32(dx + i, 0.f);
    if (split == p.splits - 1)
      for (int i = tail + threadIdx.x; i < p.vocab; i += kThreads) st_f32(dx + i, 0.f);
    return;
  }
  const T* x = static_cast<const T*>(p.logits) + token / p.length * p.ls[0] + token % p.length * p.ls[1];
  const float slope = *p.grad_loss * p.slope[token / p.length];
  const float z = base(p.stats[2 * token]), scale = -slope / p.stats[2 * token + 1];
  auto grad = [&](float v, int i) {
    const float g = scale * ex2((v - z) * kLog2e);
    return i == label ? g + slope : g;
  };
  const bool same = (reinterpret_cast<uintptr_t>(x + head) & 15) == 0;
  const uint4* xv = reinterpret_cast<const uint4*>(x + head);
  constexpr int kU = 4;
  for (int i = v0 + threadIdx.x; i < v1; i += kU * kThreads) {
    uint4 q[kU];
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int k = i + u * kThreads;
      if (k >= v1) continue;
      if (same) {
        q[u] = __ldcs(xv + k);
      } else {
#pragma unroll
        for (int e = 0; e < kVec<T>; ++e) vec_set<T>(q[u], e, ld_f32(x + head + k * kVec<T> + e));
      }
    }
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int k = i + u * kThreads;
      if (k >= v1) continue;
      const int at = head + k * kVec<T>;
      uint4 o;
#pragma unroll
      for (int e = 0; e < kVec<T>; e += 2)
        vec_set_pair<T>(o, e / 2, grad(vec_elem<T>(q[u], e), at + e), grad(vec_elem<T>(q[u], e + 1), at + e + 1));
      __stcs(dv + k, o);
    }
  }
  if (split == 0)
    for (int i = threadIdx.x; i < head; i += kThreads) st_f32(dx + i, grad(ld_f32(x + i), i));
  if (split == p.splits - 1)
    for (int i = tail + threadIdx.x; i < p.vocab; i += kThreads) st_f32(dx + i, grad(ld_f32(x + i), i));
}

// Few tokens: the vocabulary is split so that about four CTAs come to every SM, each with at least 512 vectors.
inline int splits_of(const MMPreferenceArgs* a) {
  const long long tokens = 2 * a->pairs * a->length, vecs = a->vocab * dtype_size(a->dtype) / 16;
  long long s = (4 * 148 + tokens - 1) / tokens;
  const long long most = vecs / kThreads > 1 ? vecs / kThreads : 1;
  return (int)(s < most ? s : most);
}

inline int check(const MMPreferenceArgs* a) {
  if (!a) return MM_ERR_ARG;
  if (!dtype_size(a->dtype)) return MM_ERR_DTYPE;
  if (a->pairs < 1 || a->length < 0 || a->vocab < 1 || a->pairs > (1 << 20) || a->length > 0x7fffffffLL ||
      a->vocab > 0x7fffffffLL - 4096)
    return MM_ERR_SHAPE;
  if (a->length > 0 && 2 * a->pairs > 0x7fffffffLL / a->length) return MM_ERR_SHAPE;
  return MM_OK;
}

inline Params params_of(const MMPreferenceArgs* a) {
  Params p = {};
  p.logits = a->logits;
  p.labels = a->labels;
  p.ref = a->ref;
  p.loss = a->loss;
  p.chosen = a->chosen;
  p.rejected = a->rejected;
  p.stats = a->stats;
  p.slope = a->slope;
  p.grad_loss = a->grad_loss;
  p.dlogits = a->dlogits;
  for (int i = 0; i < 2; ++i) {
    p.ls[i] = a->logits_stride[i];
    p.ds[i] = a->dlogits_stride[i];
  }
  p.tokens = 2 * a->pairs * a->length;
  p.ignore = a->ignore_index;
  p.pairs = (int)a->pairs;
  p.length = (int)a->length;
  p.vocab = (int)a->vocab;
  p.splits = p.tokens ? splits_of(a) : 1;
  p.beta = a->beta;
  p.smoothing = a->smoothing;
  return p;
}

}  // namespace pref
}  // namespace mm

using namespace mm;
using namespace mm::pref;

extern "C" int mm_preference_loss_workspace_size(const MMPreferenceArgs* a, size_t* bytes) {
  const int rc = check(a);
  if (rc != MM_OK) return rc;
  if (!bytes) return MM_ERR_ARG;
  const long long tokens = 2 * a->pairs * a->length;
  *bytes = 16 + (size_t)(2 * a->pairs) * 16 + (tokens ? (size_t)tokens * splits_of(a) * sizeof(float4) : 0);
  return MM_OK;
}

extern "C" int mm_preference_loss_fwd(const MMPreferenceArgs* a, void* workspace, size_t workspace_bytes,
                                      mm_stream_t stream) {
  size_t need = 0;
  const int rc = mm_preference_loss_workspace_size(a, &need);
  if (rc != MM_OK) return rc;
  Params p = params_of(a);
  if (!a->ref || !a->loss || !a->chosen || !a->rejected || !a->slope) return MM_ERR_ARG;
  if (p.tokens && (!a->logits || !a->labels || !a->stats)) return MM_ERR_ARG;
  if (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 256) return MM_ERR_WORKSPACE;
  p.done = static_cast<unsigned*>(workspace);
  p.gain = reinterpret_cast<double*>(static_cast<char*>(workspace) + 16);
  p.part = reinterpret_cast<float4*>(static_cast<char*>(workspace) + 16 + (size_t)(2 * a->pairs) * 16);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const long long grid = p.tokens * p.splits;
  if (grid > 0x7fffffffLL) return MM_ERR_SHAPE;
  if (grid) {
    switch (a->dtype) {
      case MM_F32: stats_kernel<float><<<(unsigned)grid, kStatsThreads<float>, 0, s>>>(p); break;
      case MM_F16: stats_kernel<__half><<<(unsigned)grid, kStatsThreads<__half>, 0, s>>>(p); break;
      default: stats_kernel<__nv_bfloat16><<<(unsigned)grid, kStatsThreads<__nv_bfloat16>, 0, s>>>(p);
    }
    if (cudaGetLastError() != cudaSuccess) return MM_ERR_LAUNCH;
  } else if (cudaMemsetAsync(p.done, 0, sizeof(unsigned), s) != cudaSuccess) {
    return MM_ERR_LAUNCH;
  }
  loss_kernel<<<(unsigned)(2 * a->pairs), kLossThreads, 0, s>>>(p);
  return cudaGetLastError() == cudaSuccess ? MM_OK : MM_ERR_LAUNCH;
}

extern "C" int mm_preference_loss_bwd(const MMPreferenceArgs* a, mm_stream_t stream) {
  const int rc = check(a);
  if (rc != MM_OK) return rc;
  const Params p = params_of(a);
  const long long grid = p.tokens * p.splits;
  if (grid == 0) return MM_OK;
  if (grid > 0x7fffffffLL) return MM_ERR_SHAPE;
  if (!a->logits || !a->labels || !a->stats || !a->slope || !a->grad_loss || !a->dlogits) return MM_ERR_ARG;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (a->dtype) {
    case MM_F32: grad_kernel<float><<<(unsigned)grid, kThreads, 0, s>>>(p); break;
    case MM_F16: grad_kernel<__half><<<(unsigned)grid, kThreads, 0, s>>>(p); break;
    default: grad_kernel<__nv_bfloat16><<<(unsigned)grid, kThreads, 0, s>>>(p);
  }
  return cudaGetLastError() == cudaSuccess ? MM_OK : MM_ERR_LAUNCH;
}
