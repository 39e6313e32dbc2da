// What the selective scan's training kernels share: sizes, parameters, elementwise parts, and access to
// (batch, channels, time) tensors in any layout.
#pragma once

#include "mm_common.cuh"

namespace mm {
namespace train {

constexpr int kT = 32;     // steps of a chunk
constexpr int kK = 8;      // steps of a unit
constexpr int kSegs = kT / kK;

struct Params {
  const void *u, *delta, *z, *B, *C, *dy;
  const float *A, *D, *bias, *dstate;
  void *y, *du, *ddelta, *dz, *dB, *dC;
  float *state_out, *dA, *dD, *dbias;
  long long us[3], ds[3], zs[3], Bs[3], Cs[3], ys[3], As[2];  // ys: y forward, dy backward
  long long dus[3], dds[3], dzs[3], dBs[3], dCs[3];
  int batch, dim, dstate_n, seqlen;
  int softplus;
  int access;      // of the activations' rows along time: the least that any of them allows
  int by_channel;  // u is contiguous along channels
  int ahead;       // grad_kernel copies its raw inputs ahead: all contiguous along one axis, rows 16-byte aligned
  int np;          // states, rounded up to a multiple of four: rows of the buffers below
  int chunks, longs, per_long;  // chunks, long chunks, chunks of a long one
  int whole;                    // a single long chunk, walked by the kernels of mm_scan_rows.cu
  // (batch, chunks, dim, np): the state every chunk starts from; the k it gets from the later chunks of its long one
  float *hst, *kst;
  float* later;  // (batch, chunks, dim): the sum of d over those
  // (batch, longs, dim, np) and (batch, longs, dim): what a long chunk starts from, its sum of d
  float *hlong, *klong, *slong;
  float *pB, *pC;          // (batch, groups, chunks, passes, 16, 32)
  float *pA, *pD, *pbias;  // (batch, chunks, dim, np), (batch, chunks, dim)
  int passes, groups, tiles, width;  // a CTA of grad_kernel works off `tiles` tiles of `width` channels
};

MM_DEV float4 f4(float a, float b, float c, float d) { return make_float4(a, b, c, d); }

// ---- elementwise parts, on pairs of steps -------------------------------------------------------------
MM_DEV f2_t dup(float x) { return f2_pack(x, x); }
MM_DEV f2_t ex2_pair(f2_t x) {
  const float2 v = f2_unpack(x);
  return f2_pack(ex2(v.x), ex2(v.y));
}
MM_DEV f2_t rcp_pair(f2_t x) {
  const float2 v = f2_unpack(x);
  return f2_pack(rcp(v.x), rcp(v.y));
}
MM_DEV f2_t sigmoid(f2_t z) { return rcp_pair(f2_add(ex2_pair(f2_mul(z, dup(-kLog2e))), dup(1.f))); }
MM_DEV f2_t silu_of(f2_t z) { return f2_mul(z, sigmoid(z)); }
// silu'(z) = s (1 + z (1 - s))
MM_DEV f2_t silu_slope(f2_t z) {
  const f2_t s = sigmoid(z);
  return f2_mul(s, f2_fma(z, f2_sub(dup(1.f), s), dup(1.f)));
}
// exp(x) for x <= 20: 2^(x log2 e), log2 e in two words after Cody and Waite, with the product's rounding error carried
// along
MM_DEV f2_t exp_of(f2_t x) {
  const f2_t y = f2_mul(x, dup(kLog2e));
  const f2_t rest = f2_fma(x, dup(1.925963033e-8f), f2_fma(x, dup(kLog2e), f2_mul(y, dup(-1.f))));  // log2 e's second word
  const f2_t e = ex2_pair(y);
  return f2_fma(e, f2_mul(rest, dup(kLn2)), e);
}
// Arguments of exp_of: above 20 softplus does not need it, below -120 it is 0 (and finite arithmetic)
MM_DEV f2_t clamped(f2_t x) {
  const float2 v = f2_unpack(x);
  return f2_pack(fminf(fmaxf(v.x, -120.f), 20.f), fminf(fmaxf(v.y, -120.f), 20.f));
}
// softplus with the forward's cutoff at 20, without a branch (several run side by side). log(1 + e): below
// e = 0.4 as 2 artanh(e / (2 + e)), whose Taylor series keeps the relative accuracy of small steps (truncated below
// 1e-7); above, where the result is no longer small against 1, as lg2(1 + e).
MM_DEV f2_t step_of(f2_t raw, int softplus) {
  const f2_t e = exp_of(clamped(raw));
  const f2_t s = f2_mul(e, rcp_pair(f2_add(e, dup(2.f)))), z = f2_mul(s, s);
  const f2_t small =
      f2_mul(s, f2_fma(z, f2_fma(z, f2_fma(z, dup(0.285714286f), dup(0.4f)), dup(0.666666667f)), dup(2.f)));
  const float2 w = f2_unpack(f2_add(e, dup(1.f)));
  const float2 large = f2_unpack(f2_mul(f2_pack(lg2(w.x), lg2(w.y)), dup(kLn2)));
  const float2 ev = f2_unpack(e), sv = f2_unpack(small), rv = f2_unpack(raw);
  return f2_pack(softplus && rv.x <= 20.f ? (ev.x < 0.4f ? sv.x : large.x) : rv.x,
                 softplus && rv.y <= 20.f ? (ev.y < 0.4f ? sv.y : large.y) : rv.y);
}
MM_DEV f2_t step_slope(f2_t raw, int softplus) {
  const f2_t e = exp_of(clamped(raw));
  const float2 v = f2_unpack(f2_mul(e, rcp_pair(f2_add(e, dup(1.f))))), rv = f2_unpack(raw);
  return f2_pack(softplus && rv.x <= 20.f ? v.x : 1.f, softplus && rv.y <= 20.f ? v.y : 1.f);
}

// Eight consecutive steps of one channel; n of them exist
template <typename T> MM_DEV void load_steps(const T* p, long long s, int access, int n, float (&v)[kK]) {
  if (access == kAligned && n == kK) {
#pragma unroll
    for (int h = 0; h < (int)sizeof(T) / 2; ++h) {
      const uint4 a = *(reinterpret_cast<const uint4*>(p) + h);
      constexpr int pairs = 8 / (int)sizeof(T);
#pragma unroll
      for (int k = 0; k < pairs; ++k) {
        const float2 q = vec_pair<T>(a, k);
        v[2 * (h * pairs + k)] = q.x;
        v[2 * (h * pairs + k) + 1] = q.y;
      }
    }
  } else if (access == kContiguous && n == kK) {
    const Raw8<T> r = raw_load_shifted(p);
#pragma unroll
    for (int k = 0; k < kK; ++k) v[k] = raw_at(r, k);
  } else {
#pragma unroll
    for (int k = 0; k < kK; ++k) v[k] = k < n ? ld_f32(p + k * s) : 0.f;
  }
}
template <typename T> MM_DEV void store_steps(T* p, long long s, int access, int n, const float (&v)[kK]) {
  if (access == kAligned && n == kK) {
    const Raw8<T> r = raw_pack<T>(v);
#pragma unroll
    for (int h = 0; h < (int)sizeof(T) / 2; ++h) __stcs(reinterpret_cast<uint4*>(p) + h, r.v[h]);
  } else if (sizeof(T) == 2 && access == kContiguous && n == kK) {
    // by words of 4 bytes; from an odd element on, one element, three words, one element
    const Raw8<T> r = raw_pack<T>(v);
    unsigned* q = reinterpret_cast<unsigned*>(p);
    if (reinterpret_cast<uintptr_t>(p) & 2) {
      q = reinterpret_cast<unsigned*>(p + 1);
      st_f32(p, v[0]);
#pragma unroll
      for (int k = 0; k < 3; ++k) q[k] = __funnelshift_r(u4_word(r.v[0], k), u4_word(r.v[0], k + 1), 16);
      st_f32(p + kK - 1, v[kK - 1]);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) q[k] = u4_word(r.v[0], k);
    }
  } else {
#pragma unroll
    for (int k = 0; k < kK; ++k)
      if (k < n) st_f32(p + k * s, v[k]);
  }
}

// Where a thread's unit (eight steps of a channel) of a staged tile lies. Lanes run along whichever of time and
// channels is contiguous in memory.
template <int CH, int SEGS = kSegs> MM_DEV void unit_of(int i, int by_channel, int& ch, int& seg) {
  if (by_channel) {
    ch = i % CH;
    seg = i / CH;
  } else {
    seg = i % SEGS;
    ch = i / SEGS;
  }
}

MM_DEV f2_t mul1(f2_t a, float x) { return f2_mul(a, dup(x)); }
MM_DEV f2_t fma1(f2_t a, float x, f2_t c) { return f2_fma(a, dup(x), c); }

// Four consecutive states' entries of a (dim, dstate)-shaped row; zeros past the last state
MM_DEV float4 load_A(const Params& p, int d, int n0) {
  const float* a = p.A + d * p.As[0] + n0 * p.As[1];
  const int n = p.dstate_n - n0;
  return f4(n > 0 ? a[0] : 0.f, n > 1 ? a[p.As[1]] : 0.f, n > 2 ? a[2 * p.As[1]] : 0.f, n > 3 ? a[3 * p.As[1]] : 0.f);
}
template <typename T>
MM_DEV float4 load_BC(const T* base, const long long (&st)[3], int b, int n0, int t, const Params& p) {
  const T* q = base + b * st[0] + n0 * st[1] + t * st[2];
  const int n = t < p.seqlen ? p.dstate_n - n0 : 0;
  return f4(n > 0 ? ld_f32(q) : 0.f, n > 1 ? ld_f32(q + st[1]) : 0.f, n > 2 ? ld_f32(q + 2 * st[1]) : 0.f,
            n > 3 ? ld_f32(q + 3 * st[1]) : 0.f);
}

// ---- host ---------------------------------------------------------------------------------------------
inline void copy3(long long (&to)[3], const int64_t* from) {
  for (int i = 0; i < 3; ++i) to[i] = from[i];
}
inline Access access_of(const void* q, const int64_t* st, const MMScanArgs& f) {
  const int es = dtype_size(f.dtype);
  if (f.seqlen > 1 && st[2] != 1) return kAnyStride;
  return aligned16(q) && (f.batch <= 1 || st[0] * es % 16 == 0) && (f.dim <= 1 || st[1] * es % 16 == 0) ? kAligned : kContiguous;
}
inline Access least(Access a, Access b) { return a < b ? a : b; }
// float32's contiguous rows off a 16-byte boundary go element by element: the shifted words' registers cost
// grad_kernel more (f32 8x1536x2047: 1.26 ms, by elements 0.99)
inline void set_access(Params& p, Access access, const MMScanArgs& f) {
  p.access = access == kContiguous && f.dtype == MM_F32 ? kAnyStride : access;
  p.by_channel = access == kAnyStride && f.u_stride[1] == 1;
}
inline int chunks_of(const MMScanArgs& f) { return (int)((f.seqlen + kT - 1) / kT); }
// Up to 256 steps of up to 16 states are walked whole, by the kernels of mm_scan_rows.cu: one launch, and nothing to join
// (bf16 1x1536 forward: 128 steps 12 us, cut 29; 256 21 and 29; 512 40 and 35).
inline bool walked_whole(const MMScanArgs& f) { return f.dstate <= 16 && f.seqlen <= 256; }
// Chunks of a long one: four; fewer where that leaves an SM less than twelve warps of 32 channels to walk them. Two chunks
// are one long chunk, which needs no joining.
inline int per_long_of(const MMScanArgs& f) {
  if (walked_whole(f)) return f.seqlen > 0 ? chunks_of(f) : 1;
  int n = 4;
  while (chunks_of(f) > 2 && n > 1 && f.batch * ((f.dim + 31) / 32) * ((chunks_of(f) + n - 1) / n) < 12 * 148) n /= 2;
  return n;
}
inline int longs_of(const MMScanArgs& f) { return (chunks_of(f) + per_long_of(f) - 1) / per_long_of(f); }
inline int check_sizes(const MMScanArgs& f) {
  if (!dtype_size(f.dtype)) return MM_ERR_DTYPE;
  if (f.batch < 0 || f.dim < 0 || f.seqlen < 0 || f.dstate < 1 || f.dstate > MM_MAX_DSTATE || f.batch > 0x7fffffffLL ||
      f.dim > 0x7fffffffLL / (2 * MM_MAX_DSTATE) || f.seqlen > 0x7fffffffLL - 256)
    return MM_ERR_SHAPE;
  return MM_OK;
}
// Offsets of consecutive float arrays in a buffer, each on 256 bytes
struct Offsets {
  size_t at = 0;
  size_t take(size_t n) {
    const size_t r = at;
    at += (n * sizeof(float) + 255) / 256 * 256;
    return r;
  }
};
// The forward's inputs
inline void set_inputs(Params& p, const MMScanArgs& f) {
  p.u = f.u;
  p.delta = f.delta;
  p.z = f.z;
  p.B = f.B;
  p.C = f.C;
  p.A = f.A;
  p.D = f.D;
  p.bias = f.delta_bias;
  copy3(p.us, f.u_stride);
  copy3(p.ds, f.delta_stride);
  copy3(p.zs, f.z_stride);
  copy3(p.Bs, f.B_stride);
  copy3(p.Cs, f.C_stride);
  p.As[0] = f.A_stride[0];
  p.As[1] = f.A_stride[1];
  p.batch = (int)f.batch;
  p.dim = (int)f.dim;
  p.dstate_n = (int)f.dstate;
  p.seqlen = (int)f.seqlen;
  p.softplus = f.delta_softplus != 0;
  p.np = (int)(f.dstate + 3) / 4 * 4;
  p.chunks = chunks_of(f);
  p.longs = longs_of(f);
  p.per_long = per_long_of(f);
  p.whole = walked_whole(f);
}

// Fills kst, later, klong and slong (mm_scan_walk.cu): the part of the gradient that runs through time
int walk_back(const Params& p, int64_t dtype, cudaStream_t s);
// Over whole sequences of up to 16 states (mm_scan_rows.cu): y, state_out and hst, or kst and later
template <bool BACK> int walk_rows(const Params& p, int64_t dtype, cudaStream_t s);

}  // namespace train
}  // namespace mm
