// Causal depthwise conv1d (width 4) for training: the forward pass that leaves an 8-bit checkpoint of its input,
// and the gradient, taken at the input or at the values the checkpoint stands for.
//
// Both are memory-bound stencils. Forward: x is read once and gives out, codes and exponents. Backward, with
// dpre[t] = dout[t] silu'(pre[t]) recomputed from x:  dx[t] = sum_k w[k] dpre[t+3-k]  (a window that looks three
// steps ahead), dw[k] = sum dpre[t] x[t-3+k], db = sum dpre. Sums over time are kept in registers by one warp
// (time contiguous) or thread (channels contiguous), leave as one partial per stretch of time, and a second
// kernel adds the partials in a fixed order.
#include "mm_checkpoint8.cuh"

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

MM_DEV float act(float v, int silu_on) { return silu_on ? silu(v) : v; }
// d silu(v) / dv = s (1 + v (1 - s)), s = sigmoid(v). Below -88, s is 0 and so is the product.
MM_DEV float dact(float v, int silu_on) {
  const float s = rcp(1.f + ex2(-v * kLog2e));
  return silu_on ? s * fmaf(v, 1.f - s, 1.f) : 1.f;
}

// ---- time contiguous --------------------------------------------------------------------------------
// A warp covers 256 consecutive steps of one row, 8 per lane; halos come from the neighbouring lanes, and for
// the warp's first and last lane from memory.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) fwd_rows_kernel(const Params p, int warps_per_row) {
  const int lane = threadIdx.x & 31;
  const long long gw = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const long long rows = (long long)p.batch * p.dim;
  if (gw >= rows * warps_per_row) return;
  const long long row = gw / warps_per_row;
  const int t0 = ((int)(gw % warps_per_row) * 32 + lane) * kE;
  const int b = (int)(row / p.dim), d = (int)(row % p.dim);
  const T* xr = static_cast<const T*>(p.x) + b * p.xs[0] + d * p.xs[1];
  const int n = min(kE, p.seqlen - t0);
  float win[kE + 3];
  float v[kE];
  if (VEC && n == kE) {
    ck_load8<T>(xr + t0, v);
  } else {
#pragma unroll
    for (int k = 0; k < kE; ++k) v[k] = k < n ? ld_f32(xr + (long long)(t0 + k) * p.xs[2]) : 0.f;
  }
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    win[k] = __shfl_up_sync(0xffffffffu, v[kE - 3 + k], 1);
    if (lane == 0) win[k] = t0 > 0 ? ld_f32(xr + (long long)(t0 - 3 + k) * p.xs[2]) : 0.f;
  }
  unsigned m = 0;
#pragma unroll
  for (int k = 0; k < kE; ++k) {
    win[k + 3] = v[k];
    m = max(m, ck_abs_bits(v[k]));
  }
  m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
  m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
  if (n <= 0) return;
  const float4 w = *reinterpret_cast<const float4*>(p.w + (long long)d * kW);
  const float bb = p.bias ? p.bias[d] : 0.f;
  float o[kE];
#pragma unroll
  for (int k = 0; k < kE; ++k)
    o[k] = act(fmaf(w.w, win[k + 3], fmaf(w.z, win[k + 2], fmaf(w.y, win[k + 1], fmaf(w.x, win[k], bb)))), p.silu);
  const unsigned byte = ck_exponent(m);
  const float inv = ck_inverse_scale(byte);
  T* orow = static_cast<T*>(p.out) + b * p.os[0] + d * p.os[1];
  int8_t* crow = p.codes_out + b * p.cs[0] + d * p.cs[1];
  if ((lane & 3) == 0) p.exps_out[b * p.es[0] + d * p.es[1] + (long long)(t0 / kCkBlock) * p.es[2]] = (uint8_t)byte;
  if (VEC && n == kE) {
    ck_store8<T>(orow + t0, o);
    uint2 c;
    c.x = ck_pack4(ck_code(v[0], inv), ck_code(v[1], inv), ck_code(v[2], inv), ck_code(v[3], inv));
    c.y = ck_pack4(ck_code(v[4], inv), ck_code(v[5], inv), ck_code(v[6], inv), ck_code(v[7], inv));
    __stcs(reinterpret_cast<uint2*>(crow + t0), c);
  } else {
#pragma unroll
    for (int k = 0; k < kE; ++k)
      if (k < n) {
        st_f32(orow + (long long)(t0 + k) * p.os[2], o[k]);
        crow[(long long)(t0 + k) * p.cs[2]] = (int8_t)ck_code(v[k], inv);
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
    return CK ? (float)codes[t * cs] * ck_scale(exps[(long long)(t / kCkBlock) * es]) : ld_f32(x + t * xs);
  }
  MM_DEV void load8(int t0, float (&v)[kE]) const {
    if (CK) {
      const uint2 c = __ldcs(reinterpret_cast<const uint2*>(codes + t0));
      const float scale = ck_scale(exps[(long long)(t0 / kCkBlock) * es]);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        v[k] = (float)ck_byte(c.x, k) * scale;
        v[k + 4] = (float)ck_byte(c.y, k) * scale;
      }
    } else {
      ck_load8<T>(x + t0, v);
    }
  }
};

template <typename T, bool CK, bool VEC>
__global__ void __launch_bounds__(256) bwd_rows_kernel(const Params p, int warps_per_row) {
  const int lane = threadIdx.x & 31;
  const long long gw = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const long long rows = (long long)p.batch * p.dim;
  if (gw >= rows * warps_per_row) return;
  const long long row = gw / warps_per_row;
  const int part = (int)(gw % warps_per_row);
  const int t0 = (part * 32 + lane) * kE;
  const int b = (int)(row / p.dim), d = (int)(row % p.dim);
  const Source<T, CK> src(p, b, d);
  const T* grow = static_cast<const T*>(p.dout) + b * p.gs[0] + d * p.gs[1];
  const int n = min(kE, p.seqlen - t0);
  float v[kE], dp[kE + 3], win[kE + 3];
  if (VEC && n == kE) {
    src.load8(t0, v);
    float g[kE];
    ck_load8<T>(grow + t0, g);
#pragma unroll
    for (int k = 0; k < kE; ++k) dp[k] = g[k];
  } else {
#pragma unroll
    for (int k = 0; k < kE; ++k) {
      v[k] = k < n ? src.at(t0 + k) : 0.f;
      dp[k] = k < n ? ld_f32(grow + (long long)(t0 + k) * p.gs[2]) : 0.f;
    }
  }
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    win[k] = __shfl_up_sync(0xffffffffu, v[kE - 3 + k], 1);
    if (lane == 0) win[k] = t0 > 0 ? src.at(t0 - 3 + k) : 0.f;
  }
#pragma unroll
  for (int k = 0; k < kE; ++k) win[k + 3] = v[k];
  const float4 w = *reinterpret_cast<const float4*>(p.w + (long long)d * kW);
  const float bb = p.bias ? p.bias[d] : 0.f;
  auto pre = [&](float a, float c, float e, float f) { return fmaf(w.w, f, fmaf(w.z, e, fmaf(w.y, c, fmaf(w.x, a, bb)))); };
  float sum[kSums] = {0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int k = 0; k < kE; ++k) {
    dp[k] *= dact(pre(win[k], win[k + 1], win[k + 2], win[k + 3]), p.silu);
#pragma unroll
    for (int j = 0; j < kW; ++j) sum[j] = fmaf(dp[k], win[k + j], sum[j]);
    sum[4] += dp[k];
  }
#pragma unroll
  for (int k = 0; k < 3; ++k) dp[kE + k] = __shfl_down_sync(0xffffffffu, dp[k], 1);
  if (lane == 31) {  // the three steps that the next warp owns
    float a = win[kE], c = win[kE + 1], e = win[kE + 2];
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      const int t = t0 + kE + k;
      float f = 0.f, g = 0.f;
      if (t < p.seqlen) {
        f = src.at(t);
        g = ld_f32(grow + (long long)t * p.gs[2]);
      }
      dp[kE + k] = t < p.seqlen ? g * dact(pre(a, c, e, f), p.silu) : 0.f;
      a = c;
      c = e;
      e = f;
    }
  }
  float o[kE];
#pragma unroll
  for (int k = 0; k < kE; ++k)
    o[k] = fmaf(w.w, dp[k], fmaf(w.z, dp[k + 1], fmaf(w.y, dp[k + 2], w.x * dp[k + 3])));
  T* orow = static_cast<T*>(p.out) + b * p.os[0] + d * p.os[1];
  if (VEC && n == kE) {
    ck_store8<T>(orow + t0, o);
  } else {
#pragma unroll
    for (int k = 0; k < kE; ++k)
      if (k < n) st_f32(orow + (long long)(t0 + k) * p.os[2], o[k]);
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
// A thread walks `run` steps (a multiple of the checkpoint block) of two neighbouring channels, so a warp's
// accesses run along 64 channels.
constexpr int kC = 2;

template <typename T, bool VEC> MM_DEV void load_pair(const T* p, long long s, bool two, float (&v)[kC]) {
  if (VEC && sizeof(T) == 2) {
    const unsigned u = *reinterpret_cast<const unsigned*>(p);
    uint4 q;
    q.x = u;
    const float2 f = vec_pair<T>(q, 0);
    v[0] = f.x;
    v[1] = f.y;
  } else if (VEC) {
    const float2 f = *reinterpret_cast<const float2*>(p);
    v[0] = f.x;
    v[1] = f.y;
  } else {
    v[0] = ld_f32(p);
    v[1] = two ? ld_f32(p + s) : 0.f;
  }
}
template <typename T, bool VEC> MM_DEV void store_pair(T* p, long long s, bool two, const float (&v)[kC]) {
  if (VEC && sizeof(T) == 2) {
    uint4 q;
    vec_set_pair<T>(q, 0, v[0], v[1]);
    *reinterpret_cast<unsigned*>(p) = q.x;
  } else if (VEC) {
    *reinterpret_cast<float2*>(p) = make_float2(v[0], v[1]);
  } else {
    st_f32(p, v[0]);
    if (two) st_f32(p + s, v[1]);
  }
}
template <bool VEC> MM_DEV void load_codes(const int8_t* p, long long s, bool two, int (&c)[kC]) {
  if (VEC) {
    const int u = *reinterpret_cast<const short*>(p);
    c[0] = (int)(int8_t)u;
    c[1] = u >> 8;
  } else {
    c[0] = *p;
    c[1] = two ? p[s] : 0;
  }
}

struct Walk {
  int b, d, t0, t1, run;
  bool two;
};
MM_DEV bool walk_of(const Params& p, int run, int runs, Walk& k) {
  const int cg = (p.dim + kC - 1) / kC;
  const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= (long long)p.batch * runs * cg) return false;
  k.d = (int)(i % cg) * kC;
  k.run = (int)(i / cg % runs);
  k.b = (int)(i / cg / runs);
  k.t0 = k.run * run;
  k.t1 = min(p.seqlen, k.t0 + run);
  k.two = k.d + 1 < p.dim;
  return true;
}
MM_DEV void load_weights(const Params& p, const Walk& k, float (&w)[kC][kW], float (&bb)[kC]) {
#pragma unroll
  for (int c = 0; c < kC; ++c) {
    const int d = min(k.d + c, p.dim - 1);
#pragma unroll
    for (int j = 0; j < kW; ++j) w[c][j] = p.w[(long long)d * kW + j];
    bb[c] = p.bias ? p.bias[d] : 0.f;
  }
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(256) fwd_columns_kernel(const Params p, int run, int runs) {
  Walk k;
  if (!walk_of(p, run, runs, k)) return;
  const T* x = static_cast<const T*>(p.x) + k.b * p.xs[0] + k.d * p.xs[1];
  T* out = static_cast<T*>(p.out) + k.b * p.os[0] + k.d * p.os[1];
  int8_t* codes = p.codes_out + k.b * p.cs[0] + k.d * p.cs[1];
  uint8_t* exps = p.exps_out + k.b * p.es[0] + k.d * p.es[1];
  float w[kC][kW], bb[kC], win[kC][3];
  load_weights(p, k, w, bb);
#pragma unroll
  for (int j = 0; j < 3; ++j) {
    float v[kC] = {0.f, 0.f};
    if (k.t0 > 0) load_pair<T, VEC>(x + (long long)(k.t0 - 3 + j) * p.xs[2], p.xs[1], k.two, v);
    win[0][j] = v[0];
    win[1][j] = v[1];
  }
  for (int tb = k.t0; tb < k.t1; tb += kCkBlock) {
    T raw[kC][kCkBlock];
    unsigned m[kC] = {0, 0};
#pragma unroll
    for (int i = 0; i < kCkBlock; ++i) {
      float v[kC] = {0.f, 0.f};
      if (tb + i < k.t1) load_pair<T, VEC>(x + (long long)(tb + i) * p.xs[2], p.xs[1], k.two, v);
#pragma unroll
      for (int c = 0; c < kC; ++c) {
        raw[c][i] = ElemTraits<T>::from_f32(v[c]);
        m[c] = max(m[c], ck_abs_bits(v[c]));
      }
    }
    float inv[kC];
#pragma unroll
    for (int c = 0; c < kC; ++c) {
      const unsigned byte = ck_exponent(m[c]);
      inv[c] = ck_inverse_scale(byte);
      if (c == 0 || k.two) exps[(long long)(tb / kCkBlock) * p.es[2] + c * p.es[1]] = (uint8_t)byte;
    }
#pragma unroll
    for (int i = 0; i < kCkBlock; ++i) {
      if (tb + i < k.t1) {
        float o[kC];
        int code[kC];
#pragma unroll
        for (int c = 0; c < kC; ++c) {
          const float v = ElemTraits<T>::to_f32(raw[c][i]);
          o[c] = act(fmaf(w[c][3], v, fmaf(w[c][2], win[c][2], fmaf(w[c][1], win[c][1], fmaf(w[c][0], win[c][0], bb[c])))),
                     p.silu);
          code[c] = ck_code(v, inv[c]);
          win[c][0] = win[c][1];
          win[c][1] = win[c][2];
          win[c][2] = v;
        }
        store_pair<T, VEC>(out + (long long)(tb + i) * p.os[2], p.os[1], k.two, o);
        int8_t* cp = codes + (long long)(tb + i) * p.cs[2];
        if (VEC) {
          *reinterpret_cast<short*>(cp) = (short)((code[0] & 0xff) | (code[1] << 8));
        } else {
          cp[0] = (int8_t)code[0];
          if (k.two) cp[p.cs[1]] = (int8_t)code[1];
        }
      }
    }
  }
}

// Backward: step t completes dx[t-3] from the last four dpre; three steps past the run finish its end. Only the
// run's own steps enter the sums.
template <typename T, bool CK, bool VEC>
__global__ void __launch_bounds__(256) bwd_columns_kernel(const Params p, int run, int runs) {
  Walk k;
  if (!walk_of(p, run, runs, k)) return;
  const T* x = CK ? nullptr : static_cast<const T*>(p.x) + k.b * p.xs[0] + k.d * p.xs[1];
  const int8_t* codes = CK ? p.codes + k.b * p.cs[0] + k.d * p.cs[1] : nullptr;
  const uint8_t* exps = CK ? p.exps + k.b * p.es[0] + k.d * p.es[1] : nullptr;
  const T* dout = static_cast<const T*>(p.dout) + k.b * p.gs[0] + k.d * p.gs[1];
  T* dx = static_cast<T*>(p.out) + k.b * p.os[0] + k.d * p.os[1];
  float w[kC][kW], bb[kC], win[kC][3], dp[kC][3], sum[kC][kSums];
  load_weights(p, k, w, bb);
  auto load_x = [&](int t, float (&v)[kC]) {
    if (CK) {
      int c[kC];
      load_codes<VEC>(codes + (long long)t * p.cs[2], p.cs[1], k.two, c);
      const uint8_t* e = exps + (long long)(t / kCkBlock) * p.es[2];
      v[0] = (float)c[0] * ck_scale(e[0]);
      v[1] = k.two ? (float)c[1] * ck_scale(e[p.es[1]]) : 0.f;
    } else {
      load_pair<T, VEC>(x + (long long)t * p.xs[2], p.xs[1], k.two, v);
    }
  };
#pragma unroll
  for (int j = 0; j < 3; ++j) {
    float v[kC] = {0.f, 0.f};
    if (k.t0 > 0) load_x(k.t0 - 3 + j, v);
#pragma unroll
    for (int c = 0; c < kC; ++c) {
      win[c][j] = v[c];
      dp[c][j] = 0.f;
    }
  }
#pragma unroll
  for (int c = 0; c < kC; ++c)
#pragma unroll
    for (int j = 0; j < kSums; ++j) sum[c][j] = 0.f;
#pragma unroll 8
  for (int t = k.t0; t < k.t1 + 3; ++t) {
    float v[kC] = {0.f, 0.f}, g[kC] = {0.f, 0.f}, o[kC];
    if (t < p.seqlen) {
      load_x(t, v);
      load_pair<T, VEC>(dout + (long long)t * p.gs[2], p.gs[1], k.two, g);
    }
    const bool mine = t < k.t1;
#pragma unroll
    for (int c = 0; c < kC; ++c) {
      const float pre = fmaf(w[c][3], v[c], fmaf(w[c][2], win[c][2], fmaf(w[c][1], win[c][1], fmaf(w[c][0], win[c][0], bb[c]))));
      const float q = t < p.seqlen ? g[c] * dact(pre, p.silu) : 0.f;
      const float own = mine ? q : 0.f;
      sum[c][0] = fmaf(own, win[c][0], sum[c][0]);
      sum[c][1] = fmaf(own, win[c][1], sum[c][1]);
      sum[c][2] = fmaf(own, win[c][2], sum[c][2]);
      sum[c][3] = fmaf(own, v[c], sum[c][3]);
      sum[c][4] += own;
      o[c] = fmaf(w[c][3], dp[c][0], fmaf(w[c][2], dp[c][1], fmaf(w[c][1], dp[c][2], w[c][0] * q)));
      win[c][0] = win[c][1];
      win[c][1] = win[c][2];
      win[c][2] = v[c];
      dp[c][0] = dp[c][1];
      dp[c][1] = dp[c][2];
      dp[c][2] = q;
    }
    if (t - 3 >= k.t0) store_pair<T, VEC>(dx + (long long)(t - 3) * p.os[2], p.os[1], k.two, o);
  }
  float* out = p.part + (((long long)k.b * runs + k.run) * p.dim + k.d) * kSums;
#pragma unroll
  for (int j = 0; j < kSums; ++j) {
    out[j] = sum[0][j];
    if (k.two) out[kSums + j] = sum[1][j];
  }
}

// Sums the partials of every channel in order, in 64 bits (a channel has up to a few thousand).
__global__ void __launch_bounds__(256) sum_kernel(const float* part, long long parts, int dim, float* dw, float* db) {
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= dim * kSums) return;
  double s = 0;
  for (long long k = 0; k < parts; ++k) s += part[k * dim * kSums + i];
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
inline Plan make_plan(int64_t batch, int64_t dim, int64_t seqlen, bool columns) {
  Plan pl;
  pl.columns = columns;
  if (columns) {
    const int64_t want = (2 * 148 * 2048 + batch * dim / kC) / (batch * dim / kC + 1);
    int64_t run = (seqlen / (want > 0 ? want : 1) + kCkBlock - 1) / kCkBlock * kCkBlock;
    run = run < kCkBlock ? kCkBlock : run > 256 ? 256 : run;
    pl.run = (int)run;
  } else {
    pl.run = 32 * kE;
  }
  pl.parts = (int)((seqlen + pl.run - 1) / pl.run);
  return pl;
}

inline bool unit(const int64_t* st, int64_t n, int i) { return n <= 1 || st[i] == 1; }

inline int check(int64_t dtype, int64_t batch, int64_t dim, int64_t seqlen, int64_t width) {
  if (width != kW) return MM_ERR_SHAPE;
  if (!dtype_size(dtype)) return MM_ERR_DTYPE;
  if (batch < 0 || dim < 0 || seqlen < 0 || batch > 0x7fffffffLL || dim > 0x7fffffffLL / 8 || seqlen > 0x7fffffffLL - 512)
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
inline bool columns_aligned(const void* p, const int64_t* st, int64_t dim, int elem) {
  const int a = kC * elem;
  return dim % kC == 0 && reinterpret_cast<uintptr_t>(p) % a == 0 && (st[0] * elem) % a == 0 && (st[2] * elem) % a == 0;
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
  const Plan pl = make_plan(a->batch, a->dim, a->seqlen, all_columns(a->dim, a->seqlen, st, 3));
  const int es = (int)sizeof(T);
  if (pl.columns) {
    const long long threads = a->batch * pl.parts * ((a->dim + kC - 1) / kC), grid = (threads + 255) / 256;
    if (grid > 0x7fffffffLL) return MM_ERR_SHAPE;
    if (columns_aligned(a->x, a->x_stride, a->dim, es) && columns_aligned(a->out, a->out_stride, a->dim, es) &&
        columns_aligned(a->codes, a->codes_stride, a->dim, 1))
      fwd_columns_kernel<T, true><<<(unsigned)grid, 256, 0, s>>>(p, pl.run, pl.parts);
    else
      fwd_columns_kernel<T, false><<<(unsigned)grid, 256, 0, s>>>(p, pl.run, pl.parts);
  } else {
    const long long grid = (a->batch * a->dim * pl.parts + 7) / 8;
    if (grid > 0x7fffffffLL) return MM_ERR_SHAPE;
    if (unit(a->x_stride, a->seqlen, 2) && unit(a->out_stride, a->seqlen, 2) && unit(a->codes_stride, a->seqlen, 2) &&
        ck_rows_aligned(a->x, a->x_stride, a->batch, a->dim, es, 16) &&
        ck_rows_aligned(a->out, a->out_stride, a->batch, a->dim, es, 16) &&
        ck_rows_aligned(a->codes, a->codes_stride, a->batch, a->dim, 1, 8))
      fwd_rows_kernel<T, true><<<(unsigned)grid, 256, 0, s>>>(p, pl.parts);
    else
      fwd_rows_kernel<T, false><<<(unsigned)grid, 256, 0, s>>>(p, pl.parts);
  }
  return cudaGetLastError() == cudaSuccess ? MM_OK : MM_ERR_LAUNCH;
}

inline Plan bwd_plan(const MMConvBwdArgs* a) {
  const int64_t* st[3] = {a->x ? a->x_stride : a->codes_stride, a->dout_stride, a->dx_stride};
  return make_plan(a->batch, a->dim, a->seqlen, all_columns(a->dim, a->seqlen, st, 3));
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
    const long long threads = a->batch * pl.parts * ((a->dim + kC - 1) / kC), grid = (threads + 255) / 256;
    if (grid > 0x7fffffffLL) return MM_ERR_SHAPE;
    const bool src = CK ? columns_aligned(a->codes, a->codes_stride, a->dim, 1) : columns_aligned(a->x, a->x_stride, a->dim, es);
    if (src && columns_aligned(a->dout, a->dout_stride, a->dim, es) && columns_aligned(a->dx, a->dx_stride, a->dim, es))
      bwd_columns_kernel<T, CK, true><<<(unsigned)grid, 256, 0, s>>>(p, pl.run, pl.parts);
    else
      bwd_columns_kernel<T, CK, false><<<(unsigned)grid, 256, 0, s>>>(p, pl.run, pl.parts);
  } else {
    const long long grid = (a->batch * a->dim * pl.parts + 7) / 8;
    if (grid > 0x7fffffffLL) return MM_ERR_SHAPE;
    const int64_t* ss = CK ? a->codes_stride : a->x_stride;
    const bool src = CK ? ck_rows_aligned(a->codes, a->codes_stride, a->batch, a->dim, 1, 8)
                        : ck_rows_aligned(a->x, a->x_stride, a->batch, a->dim, es, 16);
    if (src && unit(ss, a->seqlen, 2) && unit(a->dout_stride, a->seqlen, 2) && unit(a->dx_stride, a->seqlen, 2) &&
        ck_rows_aligned(a->dout, a->dout_stride, a->batch, a->dim, es, 16) &&
        ck_rows_aligned(a->dx, a->dx_stride, a->batch, a->dim, es, 16))
      bwd_rows_kernel<T, CK, true><<<(unsigned)grid, 256, 0, s>>>(p, pl.parts);
    else
      bwd_rows_kernel<T, CK, false><<<(unsigned)grid, 256, 0, s>>>(p, pl.parts);
  }
  if (cudaGetLastError() != cudaSuccess) return MM_ERR_LAUNCH;
  sum_kernel<<<(unsigned)((a->dim * kSums + 255) / 256), 256, 0, s>>>(part, a->batch * pl.parts, (int)a->dim, a->dweight,
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
  if (!a->x || !a->weight || !a->out || !a->codes || !a->exponents || !aligned16(a->weight)) return MM_ERR_ARG;
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
  if ((!a->x && (!a->codes || !a->exponents)) || !a->weight || !a->dout || !a->dx || !aligned16(a->weight)) return MM_ERR_ARG;
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
