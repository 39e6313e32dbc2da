// Causal depthwise conv1d (width 4) for training: the forward pass that leaves an 8-bit checkpoint of its input,
// and the gradient, taken at the input or at the values the checkpoint stands for.
//
// Both are memory-bound stencils. Forward: x is read once and gives out, codes and exponents. Backward, with
// dpre[t] = dout[t] silu'(pre[t]) recomputed from x:  dx[t] = sum_k w[k] dpre[t+3-k]  (a window that looks three
// steps ahead), dw[k] = sum dpre[t] x[t-3+k], db = sum dpre. Sums over time are kept in registers by one warp
// (time contiguous) or thread (channels contiguous), leave as one partial per stretch of time, and a second
// kernel adds the partials in a fixed order.
#include "mm_checkpoint8.cuh"

#include <type_traits>

namespace mm {
namespace convt {

constexpr int kW = 4;
constexpr int kE = 8;    // values per lane and step (time contiguous)
constexpr int kSums = 5; // dw[0..3], db

struct Params {
  const void* x;
  const int8_t* codes;
  const uint8_t* exps;
  int8_t* codes_out;
  uint8_t* exps_out;
  const float* w;
  const float* bias;
  const void* dout;
  void* out;  // forward: out, backward: dx
  float* part;
  long long xs[3], cs[3], es[3], gs[3], os[3];
  int batch, dim, seqlen;
  int silu;
};

// A channel's four weights, in one word where they lie on 16 bytes; a parameter may also be a view into a flat buffer
// (bf16 4x5120x5601, channels last, forward and backward: 483 us; always one by one 494)
MM_DEV float4 weights_of(const Params& p, int d) {
  const float* w = p.w + (long long)d * kW;
  if ((reinterpret_cast<uintptr_t>(p.w) & 15) == 0) return *reinterpret_cast<const float4*>(w);
  return make_float4(w[0], w[1], w[2], w[3]);
}

MM_DEV float act(float v, int silu_on) { return silu_on ? silu(v) : v; }
// d silu(v) / dv = s (1 + v (1 - s)), s = sigmoid(v). Below -88, s is 0 and so is the product.
MM_DEV float dact(float v, int silu_on) {
  const float s = rcp(1.f + ex2(-v * kLog2e));
  return silu_on ? s * fmaf(v, 1.f - s, 1.f) : 1.f;
}

// The same on pairs
MM_DEV f2_t both(float x) { return f2_pack(x, x); }
MM_DEV f2_t sigmoid2(f2_t v) {
  const float2 x = f2_unpack(f2_mul(v, both(-kLog2e)));
  const float2 y = f2_unpack(f2_add(f2_pack(ex2(x.x), ex2(x.y)), both(1.f)));
  return f2_pack(rcp(y.x), rcp(y.y));
}
MM_DEV f2_t act2(f2_t v, int silu_on) { return silu_on ? f2_mul(v, sigmoid2(v)) : v; }
MM_DEV f2_t dact2(f2_t v, int silu_on) {
  if (!silu_on) return both(1.f);
  const f2_t s = sigmoid2(v);
  return f2_mul(s, f2_fma(v, f2_sub(both(1.f), s), both(1.f)));
}
MM_DEV f2_t taps(const f2_t (&w)[kW], f2_t bias, f2_t a, f2_t b, f2_t c, f2_t d) {
  return f2_fma(w[3], d, f2_fma(w[2], c, f2_fma(w[1], b, f2_fma(w[0], a, bias))));
}

// ---- time contiguous --------------------------------------------------------------------------------
// A warp covers CPT * 256 consecutive steps of one row: chunk j of lane l are the 8 steps from 256 j + 8 l. All
// its loads are in flight before the first is used: at CPT 4 2 KB a warp forward in a 16-bit type, 3 KB backward from a
// checkpoint, 4 KB from x; twice that in float32, from a checkpoint 5 KB (f16 8x1536x4096, CPT 1 and 4: forward 84
// and 62 us; 58 now, 4.4 TB/s). Halos come from the neighbouring lanes, and for the warp's first and last lane
// from memory. Rows of up to 512 steps take CPT 1, or half their warps had nothing to do. Rows off a 16-byte boundary
// (bf16 4x5120x5601: forward 264 us, backward 398) pay for the shifting of words, two thirds more than aligned ones.

template <typename T, int ACCESS, int CPT>
__global__ void __launch_bounds__(256) fwd_rows_kernel(const Params p, int warps_per_row) {
  const int lane = threadIdx.x & 31;
  const long long gw = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const long long rows = (long long)p.batch * p.dim;
  if (gw >= rows * warps_per_row) return;
  const long long row = gw / warps_per_row;
  const int begin = (int)(gw % warps_per_row) * CPT * 256;
  const int b = (int)(row / p.dim), d = (int)(row % p.dim);
  const T* xr = static_cast<const T*>(p.x) + b * p.xs[0] + d * p.xs[1];
  Raw8<T> x[CPT];
#pragma unroll
  for (int j = 0; j < CPT; ++j) {
    const int t = begin + j * 256 + lane * kE;
    x[j] = raw_load(xr + (long long)t * p.xs[2], p.xs[2], ACCESS, min(kE, p.seqlen - t));
  }
  float before[3];  // the three steps before the warp's chunk
#pragma unroll
  for (int k = 0; k < 3; ++k) before[k] = begin > 0 ? ld_f32(xr + (long long)(begin - 3 + k) * p.xs[2]) : 0.f;
  const float4 w = weights_of(p, d);
  const float bb = p.bias ? p.bias[d] : 0.f;
  T* orow = static_cast<T*>(p.out) + b * p.os[0] + d * p.os[1];
  int8_t* crow = p.codes_out + b * p.cs[0] + d * p.cs[1];
#pragma unroll
  for (int j = 0; j < CPT; ++j) {
    const int t0 = begin + j * 256 + lane * kE, n = min(kE, p.seqlen - t0);
    float win[kE + 3];
    unsigned m = ck_max_bits(x[j]);
#pragma unroll
    for (int k = 0; k < kE; ++k) win[k + 3] = raw_at(x[j], k);
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      const float v = __shfl_sync(0xffffffffu, win[kE + k], (lane + 31) & 31);  // lane 0 takes lane 31's for the next chunk
      win[k] = lane == 0 ? before[k] : v;
      before[k] = v;
    }
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
    float o[kE];
#pragma unroll
    for (int k = 0; k < kE; ++k)
      o[k] = act(fmaf(w.w, win[k + 3], fmaf(w.z, win[k + 2], fmaf(w.y, win[k + 1], fmaf(w.x, win[k], bb)))), p.silu);
    const unsigned byte = ck_exponent(m);
    const float inv = ck_inverse_scale(byte);
    if ((lane & 3) == 0 && n > 0) p.exps_out[b * p.es[0] + d * p.es[1] + (long long)(t0 / kCkBlock) * p.es[2]] = (uint8_t)byte;
    row_store(orow + (long long)t0 * p.os[2], p.os[2], ACCESS, n, o);
    if (ACCESS != kAnyStride && n == kE) {
      uint2 c;
      c.x = ck_pack4(ck_code(win[3], inv), ck_code(win[4], inv), ck_code(win[5], inv), ck_code(win[6], inv));
      c.y = ck_pack4(ck_code(win[7], inv), ck_code(win[8], inv), ck_code(win[9], inv), ck_code(win[10], inv));
      __stcs(reinterpret_cast<uint2*>(crow + t0), c);
    } else {
#pragma unroll
      for (int k = 0; k < kE; ++k)
        if (k < n) crow[(long long)(t0 + k) * p.cs[2]] = (int8_t)ck_code(win[k + 3], inv);
    }
  }
}

// x of row (b, d) at step t, from the input or its checkpoint
template <typename T, bool CK> struct Source {
  const T* x;
  const int8_t* codes;
  const uint8_t* exps;
  long long xs, cs, es;
  MM_DEV Source(const Params& p, int b, int d) {
    if (CK) {
      codes = p.codes + b * p.cs[0] + d * p.cs[1];
      exps = p.exps + b * p.es[0] + d * p.es[1];
      cs = p.cs[2];
      es = p.es[2];
    } else {
      x = static_cast<const T*>(p.x) + b * p.xs[0] + d * p.xs[1];
      xs = p.xs[2];
    }
  }
  MM_DEV float at(int t) const {
    return CK ? ck_restore<T>((float)codes[t * cs], ck_scale(exps[(long long)(t / kCkBlock) * es])) : ld_f32(x + t * xs);
  }
  // eight steps as they lie in memory, their scale, and a value of them
  struct Eight {
    Raw8<T> x;
    uint2 c;
    float scale;
    MM_DEV float at(int k) const { return CK ? ck_restore<T>(ck_converted(k < 4 ? c.x : c.y, k & 3), scale) : raw_at(x, k); }
  };
  MM_DEV Eight load(int t0, int access, int n) const {
    Eight r = {};
    if (!CK) {
      r.x = raw_load(x + (long long)t0 * xs, xs, access, n);
    } else if (n > 0) {
      if (access != kAnyStride && n == kE) {
        r.c = __ldcs(reinterpret_cast<const uint2*>(codes + t0));
      } else {
        int v[kE];
#pragma unroll
        for (int k = 0; k < kE; ++k) v[k] = k < n ? codes[(t0 + k) * cs] : 0;
        r.c = make_uint2(ck_pack4(v[0], v[1], v[2], v[3]), ck_pack4(v[4], v[5], v[6], v[7]));
      }
      r.scale = ck_scale(exps[(long long)(t0 / kCkBlock) * es]);
    }
    return r;
  }
};

// The chunks from the last to the first, so that the three dpre after a chunk are known. Bound by instructions rather
// than memory: an element takes its pre-activation again, silu', four taps for dx and five sums (f16 8x1536x4096 from
// the checkpoint 105 us, 2.4 TB/s; from x itself 83, 3.6; without SiLU 79 and 62).
// Past the row's end dpre is 0, but its window may hold a last value that is no number, and 0 times that is not 0. With SiLU
// such a value has made the last dpre, and with it every sum, NaN already; without, those steps are left out.
template <typename T, bool CK, int ACCESS, int CPT, bool SILU>
__global__ void __launch_bounds__(256) bwd_rows_kernel(const Params p, int warps_per_row) {
  const int lane = threadIdx.x & 31;
  const long long gw = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const long long rows = (long long)p.batch * p.dim;
  if (gw >= rows * warps_per_row) return;
  const long long row = gw / warps_per_row;
  const int part = (int)(gw % warps_per_row), begin = part * CPT * 256, end = begin + CPT * 256;
  const int b = (int)(row / p.dim), d = (int)(row % p.dim);
  const Source<T, CK> src(p, b, d);
  const T* grow = static_cast<const T*>(p.dout) + b * p.gs[0] + d * p.gs[1];
  typename Source<T, CK>::Eight x[CPT];
  Raw8<T> g[CPT];
#pragma unroll
  for (int j = 0; j < CPT; ++j) {
    const int t = begin + j * 256 + lane * kE, n = min(kE, p.seqlen - t);
    x[j] = src.load(t, ACCESS, n);
    g[j] = raw_load(grow + (long long)t * p.gs[2], p.gs[2], ACCESS, n);
  }
  float before[3], after[3];  // x before the warp's steps; dpre of the three steps that follow the chunk at hand
  const float* wp = p.w + (long long)d * kW;  // one by one: with weights_of's branch f32 8x1536x4096 from x 114 us for 109
  const float4 w = make_float4(wp[0], wp[1], wp[2], wp[3]);
  const float bb = p.bias ? p.bias[d] : 0.f;
  auto pre = [&](float a, float c, float e, float f) { return fmaf(w.w, f, fmaf(w.z, e, fmaf(w.y, c, fmaf(w.x, a, bb)))); };
#pragma unroll
  for (int k = 0; k < 3; ++k) before[k] = begin > 0 ? src.at(begin - 3 + k) : 0.f;
  {
    float v[6];
#pragma unroll
    for (int k = 0; k < 6; ++k) v[k] = end - 3 + k < p.seqlen ? src.at(end - 3 + k) : 0.f;
#pragma unroll
    for (int k = 0; k < 3; ++k)
      after[k] = end + k < p.seqlen ? ld_f32(grow + (long long)(end + k) * p.gs[2]) *
                                          dact(pre(v[k], v[k + 1], v[k + 2], v[k + 3]), SILU)
                                    : 0.f;
  }
  T* orow = static_cast<T*>(p.out) + b * p.os[0] + d * p.os[1];
  float sum[kSums] = {0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int j = CPT - 1; j >= 0; --j) {
    const int t0 = begin + j * 256 + lane * kE, n = min(kE, p.seqlen - t0);
    float win[kE + 3], dp[kE + 3];
#pragma unroll
    for (int k = 0; k < kE; ++k) win[k + 3] = x[j].at(k);
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      win[k] = __shfl_up_sync(0xffffffffu, win[kE + k], 1);
      const float last = j > 0 ? __shfl_sync(0xffffffffu, x[j > 0 ? j - 1 : 0].at(kE - 3 + k), 31) : before[k];
      if (lane == 0) win[k] = last;
    }
#pragma unroll
    for (int k = 0; k < kE; ++k) {
      dp[k] = raw_at(g[j], k) * dact(pre(win[k], win[k + 1], win[k + 2], win[k + 3]), SILU);
      if (SILU || k < n) {
#pragma unroll
        for (int i = 0; i < kW; ++i) sum[i] = fmaf(dp[k], win[k + i], sum[i]);
        sum[4] += dp[k];
      }
    }
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      dp[kE + k] = __shfl_down_sync(0xffffffffu, dp[k], 1);
      if (lane == 31) dp[kE + k] = after[k];
      after[k] = __shfl_sync(0xffffffffu, dp[k], 0);
    }
    float o[kE];
#pragma unroll
    for (int k = 0; k < kE; ++k)
      o[k] = fmaf(w.w, dp[k], fmaf(w.z, dp[k + 1], fmaf(w.y, dp[k + 2], w.x * dp[k + 3])));
    row_store(orow + (long long)t0 * p.os[2], p.os[2], ACCESS, n, o);
  }
#pragma unroll
  for (int j = 0; j < kSums; ++j)
#pragma unroll
    for (int h = 16; h > 0; h >>= 1) sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], h);
  if (lane == 0) {
    float* out = p.part + (((long long)b * warps_per_row + part) * p.dim + d) * kSums;
#pragma unroll
    for (int j = 0; j < kSums; ++j) out[j] = sum[j];
  }
}

// ---- channels contiguous ------------------------------------------------------------------------------
// A thread walks `run` steps (a multiple of the checkpoint block) of C neighbouring channels (8 bytes of them), so a
// warp's accesses run along 128 channels of a 16-bit type, 64 of float32.
template <typename T> constexpr int kC = 8 / (int)sizeof(T);

template <typename T, bool VEC> MM_DEV void load_few(const T* p, long long s, int n, f2_t (&v)[kC<T> / 2]) {
  if (VEC) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    uint4 q;
    q.x = u.x;
    q.y = u.y;
#pragma unroll
    for (int c = 0; c < kC<T> / 2; ++c) {
      const float2 f = vec_pair<T>(q, c);
      v[c] = f2_pack(f.x, f.y);
    }
  } else {
#pragma unroll
    for (int c = 0; c < kC<T> / 2; ++c)
      v[c] = f2_pack(2 * c < n ? ld_f32(p + 2 * c * s) : 0.f, 2 * c + 1 < n ? ld_f32(p + (2 * c + 1) * s) : 0.f);
  }
}
// The same as they lie in memory, to be unpacked later
template <typename T, bool VEC> MM_DEV uint2 fetch_few(const T* p, long long s, int n) {
  if (VEC) return __ldcs(reinterpret_cast<const uint2*>(p));
  uint4 q = make_uint4(0, 0, 0, 0);
#pragma unroll
  for (int c = 0; c < kC<T>; ++c)
    if (c < n) vec_set<T>(q, c, ld_f32(p + c * s));
  return make_uint2(q.x, q.y);
}
template <typename T> MM_DEV f2_t unpack_few(uint2 u, int c) {
  uint4 q;
  q.x = u.x;
  q.y = u.y;
  const float2 f = vec_pair<T>(q, c);
  return f2_pack(f.x, f.y);
}
template <typename T, bool VEC> MM_DEV void store_few(T* p, long long s, int n, const f2_t (&v)[kC<T> / 2]) {
  if (VEC) {
    uint4 q = make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int c = 0; c < kC<T> / 2; ++c) vec_set_pair<T>(q, c, f2_unpack(v[c]).x, f2_unpack(v[c]).y);
    __stcs(reinterpret_cast<uint2*>(p), make_uint2(q.x, q.y));
  } else {
#pragma unroll
    for (int c = 0; c < kC<T> / 2; ++c) {
      if (2 * c < n) st_f32(p + 2 * c * s, f2_unpack(v[c]).x);
      if (2 * c + 1 < n) st_f32(p + (2 * c + 1) * s, f2_unpack(v[c]).y);
    }
  }
}
// C bytes (codes or exponents)
template <int C, bool VEC> MM_DEV unsigned load_bytes(const void* q, long long s, int n) {
  const uint8_t* p = static_cast<const uint8_t*>(q);
  if (VEC) return C == 4 ? *reinterpret_cast<const unsigned*>(p) : *reinterpret_cast<const unsigned short*>(p);
  unsigned r = 0;
#pragma unroll
  for (int c = 0; c < C; ++c)
    if (c < n) r |= (unsigned)p[c * s] << (8 * c);
  return r;
}
template <int C, bool VEC> MM_DEV void store_bytes(void* q, long long s, int n, unsigned v) {
  uint8_t* p = static_cast<uint8_t*>(q);
  if (VEC) {
    if (C == 4)
      *reinterpret_cast<unsigned*>(p) = v;
    else
      *reinterpret_cast<unsigned short*>(p) = (unsigned short)v;
  } else {
#pragma unroll
    for (int c = 0; c < C; ++c)
      if (c < n) p[c * s] = (uint8_t)(v >> (8 * c));
  }
}

// Channels of a thread: d, d + step, ..; neighbours by words of 8 bytes, or, where those do not fit the rows, 32 apart so
// that a warp's elements are side by side (bf16 4x5119x5601, forward and backward: by fours 1156 us).
struct Walk {
  int b, d, step, t0, t1, run, n;  // n: channels of this thread that exist
};
template <int C, bool VEC> __host__ __device__ inline int walkers(int dim) { return VEC ? (dim + C - 1) / C : (dim + 32 * C - 1) / (32 * C) * 32; }
template <int C, bool VEC> MM_DEV bool walk_of(const Params& p, int run, int runs, Walk& k) {
  const int cg = walkers<C, VEC>(p.dim);
  const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= (long long)p.batch * runs * cg) return false;
  const int j = (int)(i % cg);
  k.step = VEC ? 1 : 32;
  k.d = VEC ? j * C : j / 32 * 32 * C + j % 32;
  k.run = (int)(i / cg % runs);
  k.b = (int)(i / cg / runs);
  k.t0 = k.run * run;
  k.t1 = min(p.seqlen, k.t0 + run);
  k.n = VEC ? min(C, p.dim - k.d) : min(C, (p.dim - k.d + 31) / 32);
  return k.n > 0;
}
template <int C> MM_DEV void load_weights(const Params& p, const Walk& k, f2_t (&w)[C / 2][kW], f2_t (&bb)[C / 2]) {
#pragma unroll
  for (int c = 0; c < C / 2; ++c) {
    const int d = min(k.d + 2 * c * k.step, p.dim - 1), e = min(k.d + (2 * c + 1) * k.step, p.dim - 1);
    const float4 v = weights_of(p, d), u = weights_of(p, e);
    w[c][0] = f2_pack(v.x, u.x), w[c][1] = f2_pack(v.y, u.y), w[c][2] = f2_pack(v.z, u.z), w[c][3] = f2_pack(v.w, u.w);
    bb[c] = f2_pack(p.bias ? p.bias[d] : 0.f, p.bias ? p.bias[e] : 0.f);
  }
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(256) fwd_columns_kernel(const Params p, int run, int runs) {
  constexpr int C = kC<T>, H = C / 2;
  Walk k;
  if (!walk_of<C, VEC>(p, run, runs, k)) return;
  const T* x = static_cast<const T*>(p.x) + k.b * p.xs[0] + k.d * p.xs[1];
  T* out = static_cast<T*>(p.out) + k.b * p.os[0] + k.d * p.os[1];
  int8_t* codes = p.codes_out + k.b * p.cs[0] + k.d * p.cs[1];
  uint8_t* exps = p.exps_out + k.b * p.es[0] + k.d * p.es[1];
  f2_t w[H][kW], bb[H], win[3][H];
  load_weights<C>(p, k, w, bb);
#pragma unroll
  for (int j = 0; j < 3; ++j) {
#pragma unroll
    for (int c = 0; c < H; ++c) win[j][c] = both(0.f);
    if (k.t0 > 0) load_few<T, VEC>(x + (long long)(k.t0 - 3 + j) * p.xs[2], k.step * p.xs[1], k.n, win[j]);
  }
  // Twice over each block: for its maxima, then, out of L1, for everything else (bf16 4x5120x5601 187 us, 3.1 TB/s;
  // the block held in registers instead leaves 8 warps an SM, 255 us).
  for (int tb = k.t0; tb < k.t1; tb += kCkBlock) {
    const int n = min(kCkBlock, k.t1 - tb);
    const T* xb = x + (long long)tb * p.xs[2];
    unsigned m[C];
#pragma unroll
    for (int c = 0; c < C; ++c) m[c] = 0;
#pragma unroll 8
    for (int i = 0; i < n; ++i) {
      f2_t v[H];
      load_few<T, VEC>(xb + i * p.xs[2], k.step * p.xs[1], k.n, v);
#pragma unroll
      for (int c = 0; c < H; ++c) {
        const float2 q = f2_unpack(v[c]);
        m[2 * c] = max(m[2 * c], ck_abs_bits(q.x));
        m[2 * c + 1] = max(m[2 * c + 1], ck_abs_bits(q.y));
      }
    }
    float inv[C];
    unsigned bytes = 0;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const unsigned byte = ck_exponent(m[c]);
      inv[c] = ck_inverse_scale(byte);
      bytes |= byte << (8 * c);
    }
    store_bytes<C, false>(exps + (long long)(tb / kCkBlock) * p.es[2], k.step * p.es[1], k.n, bytes);
#pragma unroll 4
    for (int i = 0; i < n; ++i) {
      f2_t v[H], o[H];
      load_few<T, VEC>(xb + i * p.xs[2], k.step * p.xs[1], k.n, v);
      unsigned code = 0;
#pragma unroll
      for (int c = 0; c < H; ++c) {
        const float2 q = f2_unpack(v[c]);
        o[c] = act2(taps(w[c], bb[c], win[0][c], win[1][c], win[2][c], v[c]), p.silu);
        code |= (unsigned)(ck_code(q.x, inv[2 * c]) & 0xff) << (16 * c) |
                (unsigned)(ck_code(q.y, inv[2 * c + 1]) & 0xff) << (16 * c + 8);
        win[0][c] = win[1][c];
        win[1][c] = win[2][c];
        win[2][c] = v[c];
      }
      store_few<T, VEC>(out + (long long)(tb + i) * p.os[2], k.step * p.os[1], k.n, o);
      store_bytes<C, VEC>(codes + (long long)(tb + i) * p.cs[2], k.step * p.cs[1], k.n, code);
    }
  }
}

// Backward: step t completes dx[t-3] from the last four dpre; three steps past the run finish its end. Only the
// run's own steps enter the sums. The loads of the next eight steps are in flight while eight are worked on; two
// CTAs of an SM (128 registers) hide them best (bf16 4x5120x5601 from the checkpoint 246 us, 2.4 TB/s, with the sums of the
// partials). Neither a pipe nor memory bounds it: with 3.7 warps a scheduler it issues 0.51 a clock, waiting for results
// of its own (2.3 warps an issue) and for loads (1.3). 92 bytes a thread are spilled: 3 % of the instructions, and as
// many loads as from global memory.
template <typename T, bool CK, bool VEC>
__global__ void __launch_bounds__(256, 2) bwd_columns_kernel(const Params p, int run, int runs) {
  constexpr int C = kC<T>, H = C / 2, kU = 8;
  static_assert(kU > 3 && kCkBlock % kU == 0, "from the second group on, step t - 3 is the run's own");
  Walk k;
  if (!walk_of<C, VEC>(p, run, runs, k)) return;
  const T* x = CK ? nullptr : static_cast<const T*>(p.x) + k.b * p.xs[0] + k.d * p.xs[1];
  const int8_t* codes = CK ? p.codes + k.b * p.cs[0] + k.d * p.cs[1] : nullptr;
  const uint8_t* exps = CK ? p.exps + k.b * p.es[0] + k.d * p.es[1] : nullptr;
  const T* dout = static_cast<const T*>(p.dout) + k.b * p.gs[0] + k.d * p.gs[1];
  T* dx = static_cast<T*>(p.out) + k.b * p.os[0] + k.d * p.os[1];
  f2_t w[H][kW], bb[H], win[3][H], dp[3][H], sum[kSums][H], scale[H];
  load_weights<C>(p, k, w, bb);
  auto scales = [&](int t) {  // of the block that holds step t
    const unsigned e = load_bytes<C, false>(exps + (long long)(t / kCkBlock) * p.es[2], k.step * p.es[1], k.n);
#pragma unroll
    for (int c = 0; c < H; ++c)
      scale[c] = f2_pack(ck_scale((e >> (16 * c)) & 0xff), ck_scale((e >> (16 * c + 8)) & 0xff));
  };
  auto code_row = [&](int t) { return load_bytes<C, VEC>(codes + (long long)t * p.cs[2], k.step * p.cs[1], k.n); };
  auto value = [&](unsigned v, int c) {
    const float2 x = f2_unpack(f2_mul(f2_pack(ck_converted(v, 2 * c), ck_converted(v, 2 * c + 1)), scale[c]));
    return f2_pack(ck_limited<T>(x.x), ck_limited<T>(x.y));
  };
  if (CK && k.t0 > 0) scales(k.t0 - 1);
#pragma unroll
  for (int j = 0; j < 3; ++j) {
#pragma unroll
    for (int c = 0; c < H; ++c) win[j][c] = dp[j][c] = both(0.f);
    if (k.t0 > 0) {
      if (CK) {
        const unsigned v = code_row(k.t0 - 3 + j);
#pragma unroll
        for (int c = 0; c < H; ++c) win[j][c] = value(v, c);
      } else {
        load_few<T, VEC>(x + (long long)(k.t0 - 3 + j) * p.xs[2], k.step * p.xs[1], k.n, win[j]);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < kSums; ++j)
#pragma unroll
    for (int c = 0; c < H; ++c) sum[j][c] = both(0.f);
  // of the next kU steps, while these are worked on
  uint2 v[kU], g[kU];
  unsigned code[kU];
  const int end = min(k.t1 + 3, p.seqlen);
  auto fetch = [&](int i, int t) {
    if (CK)
      code[i] = code_row(t);
    else
      v[i] = fetch_few<T, VEC>(x + (long long)t * p.xs[2], k.step * p.xs[1], k.n);
    g[i] = fetch_few<T, VEC>(dout + (long long)t * p.gs[2], k.step * p.gs[1], k.n);
  };
  auto fetch_some = [&](int i, int t) {
    code[i] = 0;
    v[i] = g[i] = make_uint2(0, 0);
    if (t < end) fetch(i, t);
  };
  auto step = [&](int i, int t, bool inside, bool next) {
    f2_t o[H], xv[H], gv[H];
#pragma unroll
    for (int c = 0; c < H; ++c) {
      xv[c] = CK ? value(code[i], c) : unpack_few<T>(v[i], c);
      gv[c] = unpack_few<T>(g[i], c);
    }
    if (next)
      fetch(i, t + kU);
    else
      fetch_some(i, t + kU);
#pragma unroll
    for (int c = 0; c < H; ++c) {
      // past the end dout is 0, past the run's own steps the sums are left alone
      const f2_t q = f2_mul(gv[c], dact2(taps(w[c], bb[c], win[0][c], win[1][c], win[2][c], xv[c]), p.silu));
      if (inside || t < k.t1) {
        sum[0][c] = f2_fma(q, win[0][c], sum[0][c]);
        sum[1][c] = f2_fma(q, win[1][c], sum[1][c]);
        sum[2][c] = f2_fma(q, win[2][c], sum[2][c]);
        sum[3][c] = f2_fma(q, xv[c], sum[3][c]);
        sum[4][c] = f2_add(sum[4][c], q);
      }
      o[c] = f2_fma(w[c][3], dp[0][c], f2_fma(w[c][2], dp[1][c], f2_fma(w[c][1], dp[2][c], f2_mul(w[c][0], q))));
      win[0][c] = win[1][c];
      win[1][c] = win[2][c];
      win[2][c] = xv[c];
      dp[0][c] = dp[1][c];
      dp[1][c] = dp[2][c];
      dp[2][c] = q;
    }
    if (inside || (t - 3 >= k.t0 && t < k.t1 + 3)) store_few<T, VEC>(dx + (long long)(t - 3) * p.os[2], k.step * p.os[1], k.n, o);
  };
#pragma unroll
  for (int i = 0; i < kU; ++i) fetch_some(i, k.t0 + i);
  for (int tb = k.t0; tb < k.t1 + 3; tb += kU) {
    if (CK && tb % kCkBlock == 0 && tb < p.seqlen) scales(tb);
    if (tb > k.t0 && tb + 2 * kU <= k.t1) {  // nothing to check: without branches the steps overlap
#pragma unroll
      for (int i = 0; i < kU; ++i) step(i, tb + i, true, true);
    } else {
#pragma unroll
      for (int i = 0; i < kU; ++i) step(i, tb + i, false, false);
    }
  }
  float* out = p.part + (((long long)k.b * runs + k.run) * p.dim + k.d) * kSums;
#pragma unroll
  for (int c = 0; c < H; ++c)
#pragma unroll
    for (int j = 0; j < kSums; ++j) {
      const float2 v = f2_unpack(sum[j][c]);
      if (2 * c < k.n) out[2 * c * k.step * kSums + j] = v.x;
      if (2 * c + 1 < k.n) out[(2 * c + 1) * k.step * kSums + j] = v.y;
    }
}

// Sums the partials of every channel in a fixed order, in 64 bits: eight threads share a value (4 us for 32 partials of
// 1536 channels, 22 for 352 of 5120).
__global__ void __launch_bounds__(256) sum_kernel(const float* part, long long parts, int dim, float* dw, float* db) {
  __shared__ double sum[8][32];
  const int lane = threadIdx.x & 31, row = threadIdx.x >> 5, i = blockIdx.x * 32 + lane;
  const long long pitch = (long long)dim * kSums;
  double s = 0;
  if (i < pitch) {
#pragma unroll 4
    for (long long k = row; k < parts; k += 8) s += part[k * pitch + i];
  }
  sum[row][lane] = s;
  __syncthreads();
  if (row != 0 || i >= pitch) return;
  for (int k = 1; k < 8; ++k) s += sum[k][lane];
  const int d = i / kSums, j = i % kSums;
  if (j < kW)
    dw[d * kW + j] = (float)s;
  else if (db)
    db[d] = (float)s;
}

struct Plan {
  bool columns;
  int run, parts;  // steps per part of a row, parts per row
};

// Channels contiguous: runs long enough to be worth their three extra steps, short enough that the runs of all
// rows fill the GPU twice over (148 SMs x 2048 threads).
inline Plan make_plan(int64_t dtype, int64_t batch, int64_t dim, int64_t seqlen, bool columns) {
  Plan pl;
  const int C = 8 / dtype_size(dtype);
  pl.columns = columns;
  if (columns) {
    const int64_t want = 2 * 148 * 2048 / (batch * dim / C + 1) + 1;
    int64_t run = (seqlen / (want > 0 ? want : 1) + kCkBlock - 1) / kCkBlock * kCkBlock;
    run = run < kCkBlock ? kCkBlock : run > 256 ? 256 : run;
    pl.run = (int)run;
  } else {
    pl.run = seqlen <= 512 ? 256 : 1024;  // CPT 1 or 4: a warp per row where a row is short
  }
  pl.parts = (int)((seqlen + pl.run - 1) / pl.run);
  return pl;
}

inline Access least(Access a, Access b) { return a < b ? a : b; }
// run(std::integral_constant<int, access>)
template <typename F> void with_access(Access access, F run) {
  switch (access) {
    case kAligned: return run(std::integral_constant<int, kAligned>{});
    case kContiguous: return run(std::integral_constant<int, kContiguous>{});
    default: return run(std::integral_constant<int, kAnyStride>{});
  }
}
inline bool unit(const int64_t* st, int64_t n, int i) { return n <= 1 || st[i] == 1; }

inline int check(int64_t dtype, int64_t batch, int64_t dim, int64_t seqlen, int64_t width) {
  if (width != kW) return MM_ERR_SHAPE;
  if (!dtype_size(dtype)) return MM_ERR_DTYPE;
  if (batch < 0 || dim < 0 || seqlen < 0 || batch > 0x7fffffffLL || dim > 0x7fffffffLL / 8 || seqlen > 0x7fffffffLL - 2048)
    return MM_ERR_SHAPE;
  return MM_OK;
}
inline void copy3(long long (&to)[3], const int64_t* from) {
  for (int i = 0; i < 3; ++i) to[i] = from[i];
}

// Every tensor contiguous along channels and none of them along time
inline bool all_columns(int64_t dim, int64_t seqlen, const int64_t* const* st, int n) {
  if (dim < 2 || seqlen < 2) return false;
  for (int i = 0; i < n; ++i)
    if (st[i][1] != 1 || st[i][2] == 1) return false;
  return true;
}
inline bool columns_aligned(const void* p, const int64_t* st, int64_t dim, int elem, int count) {
  const int a = count * elem;
  return dim % count == 0 && reinterpret_cast<uintptr_t>(p) % a == 0 && (st[0] * elem) % a == 0 && (st[2] * elem) % a == 0;
}

template <typename T> int launch_fwd(const MMConvCheckpointArgs* a, cudaStream_t s) {
  Params p = {};
  p.x = a->x;
  p.w = a->weight;
  p.bias = a->bias;
  p.out = a->out;
  p.codes_out = a->codes;
  p.exps_out = a->exponents;
  copy3(p.xs, a->x_stride);
  copy3(p.os, a->out_stride);
  copy3(p.cs, a->codes_stride);
  copy3(p.es, a->exponents_stride);
  p.batch = (int)a->batch;
  p.dim = (int)a->dim;
  p.seqlen = (int)a->seqlen;
  p.silu = a->silu != 0;
  const int64_t* st[3] = {a->x_stride, a->out_stride, a->codes_stride};
  const Plan pl = make_plan(a->dtype, a->batch, a->dim, a->seqlen, all_columns(a->dim, a->seqlen, st, 3));
  const int es = (int)sizeof(T);
  if (pl.columns) {
    const bool vec = columns_aligned(a->x, a->x_stride, a->dim, es, kC<T>) &&
                     columns_aligned(a->out, a->out_stride, a->dim, es, kC<T>) &&
                     columns_aligned(a->codes, a->codes_stride, a->dim, 1, kC<T>);
    const long long per = vec ? walkers<kC<T>, true>((int)a->dim) : walkers<kC<T>, false>((int)a->dim);
    const long long grid = (a->batch * pl.parts * per + 255) / 256;
    if (grid > 0x7fffffffLL) return MM_ERR_SHAPE;
    vec ? fwd_columns_kernel<T, true><<<(unsigned)grid, 256, 0, s>>>(p, pl.run, pl.parts)
        : fwd_columns_kernel<T, false><<<(unsigned)grid, 256, 0, s>>>(p, pl.run, pl.parts);
  } else {
    const long long grid = (a->batch * a->dim * pl.parts + 7) / 8;
    if (grid > 0x7fffffffLL) return MM_ERR_SHAPE;
    Access access = least(ck_access(a->x, a->x_stride, a->batch, a->dim, a->seqlen, es),
                          ck_access(a->out, a->out_stride, a->batch, a->dim, a->seqlen, es));
    if (!unit(a->codes_stride, a->seqlen, 2) || !ck_rows_aligned(a->codes, a->codes_stride, a->batch, a->dim, 1, 8))
      access = kAnyStride;
    auto run = [&](auto level) {
      constexpr int A = decltype(level)::value;
      pl.run == 256 ? fwd_rows_kernel<T, A, 1><<<(unsigned)grid, 256, 0, s>>>(p, pl.parts)
                    : fwd_rows_kernel<T, A, 4><<<(unsigned)grid, 256, 0, s>>>(p, pl.parts);
    };
    with_access(access, run);
  }
  return cudaGetLastError() == cudaSuccess ? MM_OK : MM_ERR_LAUNCH;
}

inline Plan bwd_plan(const MMConvBwdArgs* a) {
  const int64_t* st[3] = {a->x ? a->x_stride : a->codes_stride, a->dout_stride, a->dx_stride};
  return make_plan(a->dtype, a->batch, a->dim, a->seqlen, all_columns(a->dim, a->seqlen, st, 3));
}

template <typename T, bool CK> int launch_bwd(const MMConvBwdArgs* a, float* part, cudaStream_t s) {
  Params p = {};
  p.x = a->x;
  p.codes = a->codes;
  p.exps = a->exponents;
  p.w = a->weight;
  p.bias = a->bias;
  p.dout = a->dout;
  p.out = a->dx;
  p.part = part;
  copy3(p.xs, a->x_stride);
  copy3(p.cs, a->codes_stride);
  copy3(p.es, a->exponents_stride);
  copy3(p.gs, a->dout_stride);
  copy3(p.os, a->dx_stride);
  p.batch = (int)a->batch;
  p.dim = (int)a->dim;
  p.seqlen = (int)a->seqlen;
  p.silu = a->silu != 0;
  const Plan pl = bwd_plan(a);
  const int es = (int)sizeof(T);
  if (pl.columns) {
    const bool src = CK ? columns_aligned(a->codes, a->codes_stride, a->dim, 1, kC<T>)
                        : columns_aligned(a->x, a->x_stride, a->dim, es, kC<T>);
    const bool vec = src && columns_aligned(a->dout, a->dout_stride, a->dim, es, kC<T>) &&
                     columns_aligned(a->dx, a->dx_stride, a->dim, es, kC<T>);
    const long long per = vec ? walkers<kC<T>, true>((int)a->dim) : walkers<kC<T>, false>((int)a->dim);
    const long long grid = (a->batch * pl.parts * per + 255) / 256;
    if (grid > 0x7fffffffLL) return MM_ERR_SHAPE;
    vec ? bwd_columns_kernel<T, CK, true><<<(unsigned)grid, 256, 0, s>>>(p, pl.run, pl.parts)
        : bwd_columns_kernel<T, CK, false><<<(unsigned)grid, 256, 0, s>>>(p, pl.run, pl.parts);
  } else {
    const long long grid = (a->batch * a->dim * pl.parts + 7) / 8;
    if (grid > 0x7fffffffLL) return MM_ERR_SHAPE;
    Access access = least(ck_access(a->dout, a->dout_stride, a->batch, a->dim, a->seqlen, es),
                          ck_access(a->dx, a->dx_stride, a->batch, a->dim, a->seqlen, es));
    if (!CK) access = least(access, ck_access(a->x, a->x_stride, a->batch, a->dim, a->seqlen, es));
    if (CK && (!unit(a->codes_stride, a->seqlen, 2) || !ck_rows_aligned(a->codes, a->codes_stride, a->batch, a->dim, 1, 8)))
      access = kAnyStride;
    auto run = [&](auto level) {
      constexpr int A = decltype(level)::value;
      auto launch = [&](auto kernel) { kernel<<<(unsigned)grid, 256, 0, s>>>(p, pl.parts); };
      if (p.silu)
        pl.run == 256 ? launch(bwd_rows_kernel<T, CK, A, 1, true>) : launch(bwd_rows_kernel<T, CK, A, 4, true>);
      else
        pl.run == 256 ? launch(bwd_rows_kernel<T, CK, A, 1, false>) : launch(bwd_rows_kernel<T, CK, A, 4, false>);
    };
    with_access(access, run);
  }
  if (cudaGetLastError() != cudaSuccess) return MM_ERR_LAUNCH;
  sum_kernel<<<(unsigned)((a->dim * kSums + 31) / 32), 256, 0, s>>>(part, a->batch * pl.parts, (int)a->dim, a->dweight,
                                                                     a->dbias);
  return cudaGetLastError() == cudaSuccess ? MM_OK : MM_ERR_LAUNCH;
}

}  // namespace convt
}  // namespace mm

using namespace mm;
using namespace mm::convt;

extern "C" int mm_causal_conv1d_fwd_checkpoint8(const MMConvCheckpointArgs* a, mm_stream_t stream) {
  if (!a) return MM_ERR_ARG;
  const int rc = check(a->dtype, a->batch, a->dim, a->seqlen, a->width);
  if (rc != MM_OK) return rc;
  if (a->batch == 0 || a->dim == 0 || a->seqlen == 0) return MM_OK;
  if (!a->x || !a->weight || !a->out || !a->codes || !a->exponents) return MM_ERR_ARG;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (a->dtype) {
    case MM_F32: return launch_fwd<float>(a, s);
    case MM_F16: return launch_fwd<__half>(a, s);
    default: return launch_fwd<__nv_bfloat16>(a, s);
  }
}

extern "C" int mm_causal_conv1d_bwd_workspace_size(const MMConvBwdArgs* a, size_t* bytes) {
  if (!a || !bytes) return MM_ERR_ARG;
  const int rc = check(a->dtype, a->batch, a->dim, a->seqlen, a->width);
  if (rc != MM_OK) return rc;
  *bytes = 256;
  if (a->batch > 0 && a->dim > 0 && a->seqlen > 0)
    *bytes += (size_t)(a->batch * bwd_plan(a).parts * a->dim * kSums) * sizeof(float);
  return MM_OK;
}

extern "C" int mm_causal_conv1d_bwd(const MMConvBwdArgs* a, void* workspace, size_t workspace_bytes, mm_stream_t stream) {
  size_t need = 0;
  const int rc = mm_causal_conv1d_bwd_workspace_size(a, &need);
  if (rc != MM_OK) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (a->dim == 0) return MM_OK;
  if (!a->dweight) return MM_ERR_ARG;
  if (a->batch == 0 || a->seqlen == 0) {  // sums over nothing
    if (cudaMemsetAsync(a->dweight, 0, sizeof(float) * kW * a->dim, s) != cudaSuccess) return MM_ERR_LAUNCH;
    if (a->dbias && cudaMemsetAsync(a->dbias, 0, sizeof(float) * a->dim, s) != cudaSuccess) return MM_ERR_LAUNCH;
    return MM_OK;
  }
  if ((!a->x && (!a->codes || !a->exponents)) || !a->weight || !a->dout || !a->dx) return MM_ERR_ARG;
  if (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 256) return MM_ERR_WORKSPACE;
  float* part = static_cast<float*>(workspace);
  if (a->x) {
    switch (a->dtype) {
      case MM_F32: return launch_bwd<float, false>(a, part, s);
      case MM_F16: return launch_bwd<__half, false>(a, part, s);
      default: return launch_bwd<__nv_bfloat16, false>(a, part, s);
    }
  }
  switch (a->dtype) {
    case MM_F32: return launch_bwd<float, true>(a, part, s);
    case MM_F16: return launch_bwd<__half, true>(a, part, s);
    default: return launch_bwd<__nv_bfloat16, true>(a, part, s);
  }
}
