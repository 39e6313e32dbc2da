// Gradient of the selective scan.
//
// With d = softplus(delta + bias), a_t = exp(d_t A), h_t = a_t h_{t-1} + d_t u_t B_t, p_t = sum_n C_t h_t + D u_t,
// y = p silu(z), and e = dy silu(z), the gradient runs the same kind of recurrence backwards in time:
//   g_t = C_t e_t + k_t,  k_t = a_{t+1} g_{t+1}  (k at the end: the last state's gradient)
//   dC_t = sum_d h e     dB_t = sum_d g d u     du = d sum_n g B + D e     w = g a h_{t-1}
//   dd = u sum_n g B + sum_n A w     dA = sum_{b,t} d w     dz = dy p silu'(z)     dD = sum e u
// Nothing is kept from the forward pass: time is cut into chunks of 64 steps, and three kernels make the chunks
// independent of one another:
//   1. carry_kernel: of every chunk, the state it ends with from zero, the k it hands to the chunk before from
//      zero, and the sum of d (the chunk's decay is exp(A sum d), so no products are kept);
//   2. join_kernel: those in order, forwards for the states and backwards for k;
//   3. grad_kernel: every chunk from its true incoming state and k.
// Sums over channels and over chunks leave as partials that reduce_kernel adds in a fixed order, so the results
// do not depend on timing. All state and all sums are float32 (the last sums over partials float64).
#include "mm_common.cuh"

namespace mm {
namespace bwd {

constexpr int kT = 64;        // steps of a chunk
constexpr int kK = 8;         // steps of a lane
constexpr int kCh = 64;       // channels staged at a time
constexpr int kPitch = kT + 4;  // floats of a staged row; rows stay 16-byte aligned, neighbours in other banks
constexpr int kNB = 16;       // states of a pass

struct Params {
  const void *u, *delta, *z, *B, *C, *dy;
  const float *A, *D, *bias, *dstate;
  void *du, *ddelta, *dz, *dB, *dC;
  float *dA, *dD, *dbias;
  long long us[3], ds[3], zs[3], Bs[3], Cs[3], ys[3], As[2];
  long long dus[3], dds[3], dzs[3], dBs[3], dCs[3];
  int batch, dim, dstate_n, seqlen;
  int softplus;
  int vec;        // every activation's rows are contiguous in time and 16-byte aligned
  int by_channel; // u is contiguous along channels
  int ahead;      // grad_kernel copies its raw inputs ahead: all contiguous along one axis, rows 16-byte aligned
  // workspace
  float *hst, *kst, *sum_d;  // (batch, chunks, dim, np): states and k; (batch, chunks, dim)
  float *pB, *pC;            // (batch, groups, chunks, passes, 16, 64)
  float *pA, *pD, *pbias;    // (batch, chunks, dim, np), (batch, chunks, dim)
  int chunks, np, passes, groups, tiles;  // tiles of `width` channels that one CTA works off
  int width;
};

MM_DEV float4 f4(float a, float b, float c, float d) { return make_float4(a, b, c, d); }

// ---- elementwise parts -----------------------------------------------------------------------------
struct Gate {
  float silu, slope;  // silu(z), silu'(z)
};
MM_DEV Gate gate_of(float z) {
  const float s = rcp(1.f + ex2(-z * kLog2e));
  return Gate{z * s, s * fmaf(z, 1.f - s, 1.f)};
}
// exp(x) for x <= 20: 2^(x log2 e) with the product's rounding error carried along
MM_DEV float exp_of(float x) {
  const float y = x * kLog2e;
  const float rest = fmaf(x, 1.925963033e-8f, fmaf(x, kLog2e, -y));  // the second word of log2 e
  const float e = ex2(y);
  return fmaf(e, rest * kLn2, e);
}
// softplus with the forward's cutoff at 20, without a branch (eight of them run side by side). log(1 + e): below
// e = 0.4 as 2 artanh(e / (2 + e)), whose series keeps the relative accuracy of small steps (truncated below
// 1e-7); above, where the result is no longer small against 1, as lg2(1 + e).
MM_DEV float step_of(float raw, int softplus) {
  const float e = exp_of(fminf(raw, 20.f));
  const float s = e * rcp(2.f + e), z = s * s;
  const float small = s * fmaf(z, fmaf(z, fmaf(z, 0.285714286f, 0.4f), 0.666666667f), 2.f);
  const float r = e < 0.4f ? small : lg2(1.f + e) * kLn2;
  return softplus && raw <= 20.f ? r : raw;
}
MM_DEV float step_slope(float raw, int softplus) {
  const float e = exp_of(fminf(raw, 20.f));
  return softplus && raw <= 20.f ? e * rcp(1.f + e) : 1.f;
}

// Eight consecutive steps of one channel; n of them exist
template <typename T> MM_DEV void load_steps(const T* p, long long s, bool vec, int n, float (&v)[kK]) {
  if (vec && n == kK) {
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
  } else {
#pragma unroll
    for (int k = 0; k < kK; ++k) v[k] = k < n ? ld_f32(p + k * s) : 0.f;
  }
}
template <typename T> MM_DEV void store_steps(T* p, long long s, bool vec, int n, const float (&v)[kK]) {
  if (vec && n == kK) {
#pragma unroll
    for (int h = 0; h < (int)sizeof(T) / 2; ++h) {
      uint4 a;
      constexpr int pairs = 8 / (int)sizeof(T);
#pragma unroll
      for (int k = 0; k < pairs; ++k) vec_set_pair<T>(a, k, v[2 * (h * pairs + k)], v[2 * (h * pairs + k) + 1]);
      __stcs(reinterpret_cast<uint4*>(p) + h, a);
    }
  } else {
#pragma unroll
    for (int k = 0; k < kK; ++k)
      if (k < n) st_f32(p + k * s, v[k]);
  }
}

// Where a thread's unit (eight steps of a channel) of a staged tile lies. Lanes run along whichever of time and
// channels is contiguous in memory.
template <int CH> MM_DEV void unit_of(int i, int by_channel, int& ch, int& seg) {
  if (by_channel) {
    ch = i % CH;
    seg = i / CH;
  } else {
    seg = i % (kT / kK);
    ch = i / (kT / kK);
  }
}

// The raw values of a unit, so that several units' loads can be in flight before the first is worked on
struct Raw {
  float dt[kK], u[kK], e[kK], g[kK];
};
template <typename T, bool HAS_Z> MM_DEV void load_unit(const Params& p, int b, int d, int t, Raw& r) {
  const int n = min(kK, p.seqlen - t);
  load_steps(static_cast<const T*>(p.delta) + b * p.ds[0] + d * p.ds[1] + t * p.ds[2], p.ds[2], p.vec, n, r.dt);
  load_steps(static_cast<const T*>(p.u) + b * p.us[0] + d * p.us[1] + t * p.us[2], p.us[2], p.vec, n, r.u);
  load_steps(static_cast<const T*>(p.dy) + b * p.ys[0] + d * p.ys[1] + t * p.ys[2], p.ys[2], p.vec, n, r.e);
  if (HAS_Z) load_steps(static_cast<const T*>(p.z) + b * p.zs[0] + d * p.zs[1] + t * p.zs[2], p.zs[2], p.vec, n, r.g);
}

// d, d u and e (zeros where there are no steps: a = 1 there, so states and k pass through)
template <bool HAS_Z>
MM_DEV void stage_unit(const Params& p, int d, int t, const Raw& r, float (&dt)[kK], float (&dtu)[kK], float (&e)[kK]) {
  const int n = min(kK, p.seqlen - t);
  const float bias = p.bias ? p.bias[d] : 0.f;
#pragma unroll
  for (int k = 0; k < kK; ++k) {
    dt[k] = k < n ? step_of(r.dt[k] + bias, p.softplus) : 0.f;
    dtu[k] = dt[k] * r.u[k];
    e[k] = HAS_Z ? r.e[k] * gate_of(r.g[k]).silu : r.e[k];
  }
}

MM_DEV f2_t ex2_pair(f2_t x) {
  const float2 v = f2_unpack(x);
  return f2_pack(ex2(v.x), ex2(v.y));
}
MM_DEV f2_t dup(float x) { return f2_pack(x, x); }
#ifdef V_DUP
MM_DEV f2_t mul1(f2_t a, float x) { return f2_mul(a, dup(x)); }
MM_DEV f2_t fma1(f2_t a, float x, f2_t c) { return f2_fma(a, dup(x), c); }
#else
MM_DEV f2_t mul1(f2_t a, float x) {
  const float2 v = f2_unpack(a);
  return f2_pack(v.x * x, v.y * x);
}
MM_DEV f2_t fma1(f2_t a, float x, f2_t c) {
  const float2 v = f2_unpack(a), w = f2_unpack(c);
  return f2_pack(fmaf(v.x, x, w.x), fmaf(v.y, x, w.y));
}
#endif

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

// ---- 1. what every chunk contributes -----------------------------------------------------------------
// A CTA takes 64 channels of one chunk. Lanes are channels, warps pairs of a channel half and four states; each
// thread walks the chunk's 64 steps: h = a h + d u B,  P = a P,  k += P C e.
constexpr int kCarryThreads = 256;
constexpr int kCarryPitch = kCh + 1;

template <typename T, bool HAS_Z>
__global__ void __launch_bounds__(kCarryThreads) carry_kernel(const Params p) {
  extern __shared__ float4 smem4[];
  float* sd = reinterpret_cast<float*>(smem4);  // [t][channel] each
  float* sdu = sd + kT * kCarryPitch;
  float* se = sdu + kT * kCarryPitch;
  __shared__ float4 sB[kT][kNB / 4], sC[kT][kNB / 4];
  const int dtiles = (p.dim + kCh - 1) / kCh;
  const int d0 = (int)(blockIdx.x % dtiles) * kCh;
  const long long bc = blockIdx.x / dtiles;
  const int c = (int)(bc % p.chunks), b = (int)(bc / p.chunks), t0 = c * kT;
  for (int i = threadIdx.x; i < kCh * kT / kK; i += kCarryThreads) {
    int ch, seg;
    unit_of<kCh>(i, p.by_channel, ch, seg);
    float dt[kK], dtu[kK], e[kK];
    if (d0 + ch < p.dim) {
      Raw r;
      load_unit<T, HAS_Z>(p, b, d0 + ch, t0 + seg * kK, r);
      stage_unit<HAS_Z>(p, d0 + ch, t0 + seg * kK, r, dt, dtu, e);
    } else {
#pragma unroll
      for (int k = 0; k < kK; ++k) dt[k] = dtu[k] = e[k] = 0.f;
    }
#pragma unroll
    for (int k = 0; k < kK; ++k) {
      const int at = (seg * kK + k) * kCarryPitch + ch;
      sd[at] = dt[k];
      sdu[at] = dtu[k];
      se[at] = e[k];
    }
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int ch = (warp & 1) * 32 + lane, q = warp >> 1, d = d0 + ch;
  for (int pass = 0; pass < p.passes; ++pass) {
    const int n0 = pass * kNB;
    __syncthreads();
    for (int i = threadIdx.x; i < kT * kNB / 4; i += kCarryThreads) {
      const int t = i % kT, j = i / kT;
      sB[t][j] = load_BC(static_cast<const T*>(p.B), p.Bs, b, n0 + 4 * j, t0 + t, p);
      sC[t][j] = load_BC(static_cast<const T*>(p.C), p.Cs, b, n0 + 4 * j, t0 + t, p);
    }
    __syncthreads();
    if (n0 + 4 * q >= p.np || d >= p.dim) continue;
    const float4 A = load_A(p, d, n0 + 4 * q);
    const f2_t A0 = f2_mul(f2_pack(A.x, A.y), dup(kLog2e)), A1 = f2_mul(f2_pack(A.z, A.w), dup(kLog2e));
    f2_t h0 = dup(0.f), h1 = h0, k0 = h0, k1 = h0, P0 = dup(1.f), P1 = P0;
    float sum = 0.f;
#pragma unroll 4
    for (int t = 0; t < kT; ++t) {
      const float dt = sd[t * kCarryPitch + ch];
      const f2_t dd = dup(dt), du = dup(sdu[t * kCarryPitch + ch]), e = dup(se[t * kCarryPitch + ch]);
      const float4 Bv = sB[t][q], Cv = sC[t][q];
      const f2_t a0 = ex2_pair(f2_mul(dd, A0)), a1 = ex2_pair(f2_mul(dd, A1));
      h0 = f2_fma(a0, h0, f2_mul(du, f2_pack(Bv.x, Bv.y)));
      h1 = f2_fma(a1, h1, f2_mul(du, f2_pack(Bv.z, Bv.w)));
      P0 = f2_mul(P0, a0);
      P1 = f2_mul(P1, a1);
      k0 = f2_fma(P0, f2_mul(e, f2_pack(Cv.x, Cv.y)), k0);
      k1 = f2_fma(P1, f2_mul(e, f2_pack(Cv.z, Cv.w)), k1);
      sum += dt;
    }
    const long long at = (bc * p.dim + d) * p.np + n0 + 4 * q;
    const float2 x = f2_unpack(h0), y = f2_unpack(h1), v = f2_unpack(k0), w = f2_unpack(k1);
    *reinterpret_cast<float4*>(p.hst + at) = f4(x.x, x.y, y.x, y.y);
    *reinterpret_cast<float4*>(p.kst + at) = f4(v.x, v.y, w.x, w.y);
    if (n0 + 4 * q == 0) p.sum_d[bc * p.dim + d] = sum;
  }
}

// ---- 2. the chunks in order ---------------------------------------------------------------------------
// A thread per state and direction replaces, chunk by chunk, what the chunk contributes by what comes into it.
__global__ void __launch_bounds__(256) join_kernel(const Params p) {
  const long long per = (long long)p.dim * p.np;
  const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= p.batch * per) return;
  const long long b = i / per, dn = i % per;
  const int d = (int)(dn / p.np), n = (int)(dn % p.np);
  const bool back = blockIdx.y != 0;
  const float A = n < p.dstate_n ? p.A[d * p.As[0] + n * p.As[1]] * kLog2e : 0.f;
  float* st = (back ? p.kst : p.hst) + b * p.chunks * per + dn;
  const float* sum = p.sum_d + b * p.chunks * p.dim + d;
  float v = back && p.dstate && n < p.dstate_n ? p.dstate[(b * p.dim + d) * p.dstate_n + n] : 0.f;
  constexpr int kU = 8;
  for (int c0 = 0; c0 < p.chunks; c0 += kU) {
    float own[kU], s[kU];
#pragma unroll
    for (int j = 0; j < kU; ++j) {
      if (c0 + j >= p.chunks) break;
      const long long c = back ? p.chunks - 1 - (c0 + j) : c0 + j;
      own[j] = st[c * per];
      s[j] = sum[c * p.dim];
    }
#pragma unroll
    for (int j = 0; j < kU; ++j) {
      if (c0 + j >= p.chunks) break;
      const long long c = back ? p.chunks - 1 - (c0 + j) : c0 + j;
      st[c * per] = v;
      v = fmaf(ex2(s[j] * A), v, own[j]);
    }
  }
}

// ---- 3. the gradient of every chunk -----------------------------------------------------------------
// A warp works off channels one by one: lane = 4 * segment + quad holds eight steps of four states. Each segment
// runs its steps from zero, a scan over the eight segments gives its true start, and a second run the values;
// the same backwards. B, C and the sums for dB and dC stay in registers over all channels, so the sum over
// channels costs nothing but the final one over warps; sums over states go across the four quads.
#ifndef V_GCH
#define V_GCH 32
#endif
#ifndef V_OCC
#define V_OCC 2
#endif
constexpr int kGCh = V_GCH;      // channels staged at a time
constexpr int kGradWarps = 4;
constexpr int kGradThreads = kGradWarps * 32;
constexpr int kGradSmem = 5 * kGCh * kPitch * (int)sizeof(float);  // and the raw buffers
static_assert(kGradThreads == kGCh * kNB / 4, "a thread per channel and four states");

// The raw tile of one array in shared memory, [channel][step] or, contiguous along channels, [step][channel]
constexpr int kRawOne = kGCh * kT;
constexpr int kRaw = 4 * kRawOne;

MM_DEV void cp_async16_part(void* dst, const void* src, int bytes) {  // zeros after the first `bytes`
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes) : "memory");
}
// Starts copying a tile's raw inputs; one commit group. Channels and steps that do not exist arrive as zeros.
template <typename T>
MM_DEV void copy_one(const void* base, const long long (&st)[3], const Params& p, int b, int t0, int d0, T* raw) {
  const T* x = static_cast<const T*>(base) + b * st[0] + d0 * st[1] + t0 * st[2];
  constexpr int per = 16 / (int)sizeof(T);
  const int width = min(p.width, p.dim - d0), steps = min(kT, p.seqlen - t0);
#pragma unroll
  for (int i = threadIdx.x; i < kRawOne / per; i += kGradThreads) {
    const int row = p.by_channel ? i / (kGCh / per) : i / (kT / per);
    const int col = (p.by_channel ? i % (kGCh / per) : i % (kT / per)) * per;
    const int n = p.by_channel ? (row < steps ? width - col : 0) : (row < width ? steps - col : 0);
    const T* src = n > 0 ? x + row * (p.by_channel ? st[2] : st[1]) + col : x;
    cp_async16_part(raw + i * per, src, min(max(n, 0), per) * (int)sizeof(T));
  }
}
template <typename T, bool HAS_Z> MM_DEV void copy_ahead(const Params& p, int b, int t0, int d0, T* raw) {
  if (d0 < p.dim) {
    copy_one(p.delta, p.ds, p, b, t0, d0, raw);
    copy_one(p.u, p.us, p, b, t0, d0, raw + kRawOne);
    copy_one(p.dy, p.ys, p, b, t0, d0, raw + 2 * kRawOne);
    if (HAS_Z) copy_one(p.z, p.zs, p, b, t0, d0, raw + 3 * kRawOne);
  }
  cp_async_commit();
}
template <typename T, bool HAS_Z>
MM_DEV void load_unit(const Params& p, int b, int d, int t, Raw& r, const T* raw, int ch, int seg) {
  if (!p.ahead) {
    load_unit<T, HAS_Z>(p, b, d, t, r);
    return;
  }
  const T* x = raw + (p.by_channel ? seg * kK * kGCh + ch : ch * kT + seg * kK);
  const int st = p.by_channel ? kGCh : 1;
  load_steps(x, st, !p.by_channel, kK, r.dt);
  load_steps(x + kRawOne, st, !p.by_channel, kK, r.u);
  load_steps(x + 2 * kRawOne, st, !p.by_channel, kK, r.e);
  if (HAS_Z) load_steps(x + 3 * kRawOne, st, !p.by_channel, kK, r.g);
}

// Position of step t in a staged row: quarter rows of every segment lie side by side, so that the eight
// segments' 16-byte reads fall into different banks.
MM_DEV int at_step(int seg, int half) { return (half * (kT / kK) + seg) * 4; }

MM_DEV f2_t shfl_up2(f2_t v, int by) {
  const float2 x = f2_unpack(v);
  return f2_pack(__shfl_up_sync(0xffffffffu, x.x, by), __shfl_up_sync(0xffffffffu, x.y, by));
}
MM_DEV f2_t shfl_down2(f2_t v, int by) {
  const float2 x = f2_unpack(v);
  return f2_pack(__shfl_down_sync(0xffffffffu, x.x, by), __shfl_down_sync(0xffffffffu, x.y, by));
}

// Sums v[0..7] over the four quads; quad q is left with the sums of steps 4 (q & 1) + 2 (q >> 1) + {0, 1}
MM_DEV float2 sum_quads(const float (&v)[kK], int q) {
  float w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float keep = (q & 1) ? v[4 + i] : v[i], give = (q & 1) ? v[i] : v[4 + i];
    w[i] = keep + __shfl_xor_sync(0xffffffffu, give, 1);
  }
  float2 r;
  {
    const float keep = (q & 2) ? w[2] : w[0], give = (q & 2) ? w[0] : w[2];
    r.x = keep + __shfl_xor_sync(0xffffffffu, give, 2);
  }
  {
    const float keep = (q & 2) ? w[3] : w[1], give = (q & 2) ? w[1] : w[3];
    r.y = keep + __shfl_xor_sync(0xffffffffu, give, 2);
  }
  return r;
}

template <typename T, bool HAS_Z>
__global__ void __launch_bounds__(kGradThreads, V_OCC) grad_kernel(const Params p) {
  extern __shared__ float4 smem4[];
  float* sd = reinterpret_cast<float*>(smem4);  // [channel][step] each
  float* sdu = sd + kGCh * kPitch;
  float* se = sdu + kGCh * kPitch;
  float* s2 = se + kGCh * kPitch;  // sum_n A w
  float* s3 = s2 + kGCh * kPitch;  // sum_n C h
  T* raw = reinterpret_cast<T*>(s3 + kGCh * kPitch);  // two buffers of the raw delta, u, dy, z
  float* more = reinterpret_cast<float*>(raw + 2 * kRaw);
  // sum_n g B, and rows of [A, state, k][16 states]: where one pass takes all states, in the place of the d u
  // that the same lanes have read, and of the sums that the same warp has yet to write
  const bool once = p.passes == 1;
  float* s1 = once ? sdu : more;
  float* in = once ? s2 : more + kGCh * kPitch;
  __shared__ float sums[2][kGCh][kT / kK];  // of dD and ddelta, per segment
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, q = lane & 3, s = lane >> 2;
  const int group = (int)(blockIdx.x % p.groups);
  const long long bc = blockIdx.x / p.groups;
  const int c = (int)(bc % p.chunks), b = (int)(bc / p.chunks), t0 = c * kT;

  for (int pass = 0; pass < p.passes; ++pass) {
    const int n0 = pass * kNB + 4 * q;
    f2_t Bv[kK][2], Cv[kK][2], accB[kK][2], accC[kK][2];
#pragma unroll
    for (int i = 0; i < kK; ++i) {
      const float4 x = load_BC(static_cast<const T*>(p.B), p.Bs, b, n0, t0 + s * kK + i, p);
      const float4 y = load_BC(static_cast<const T*>(p.C), p.Cs, b, n0, t0 + s * kK + i, p);
      Bv[i][0] = f2_pack(x.x, x.y);
      Bv[i][1] = f2_pack(x.z, x.w);
      Cv[i][0] = f2_pack(y.x, y.y);
      Cv[i][1] = f2_pack(y.z, y.w);
      accB[i][0] = accB[i][1] = accC[i][0] = accC[i][1] = dup(0.f);
    }
    if (pass == 0 && p.ahead) copy_ahead<T, HAS_Z>(p, b, t0, group * p.tiles * p.width, raw);
    for (int tile = 0; tile < p.tiles; ++tile) {
      const int d0 = (group * p.tiles + tile) * p.width;
      const int width = min(p.width, p.dim - d0);  // channels of this tile; none past the last
      if (width <= 0) break;
      T* now = raw + (tile & 1) * kRaw;
      __syncthreads();  // the tile before has been read
      // of this pass's states, for every channel: A, the incoming state and k (one of each per thread)
      const int jc = threadIdx.x / 4, jn = pass * kNB + 4 * (threadIdx.x % 4);
      float4 jA = f4(0.f, 0.f, 0.f, 0.f), jh = jA, jk = jA;
      if (jc < width) {
        jA = load_A(p, d0 + jc, jn);
        if (p.chunks > 1) {
          const long long at = (bc * p.dim + d0 + jc) * p.np + jn;
          if (jn < p.np) {
            jh = *reinterpret_cast<const float4*>(p.hst + at);
            jk = *reinterpret_cast<const float4*>(p.kst + at);
          }
        } else if (p.dstate) {
          const float* x = p.dstate + ((long long)b * p.dim + d0 + jc) * p.dstate_n + jn;
          const int m = p.dstate_n - jn;
          jk = f4(m > 0 ? x[0] : 0.f, m > 1 ? x[1] : 0.f, m > 2 ? x[2] : 0.f, m > 3 ? x[3] : 0.f);
        }
      }
      if (pass == 0) {
        if (p.ahead) {
          if (tile + 1 < p.tiles) copy_ahead<T, HAS_Z>(p, b, t0, d0 + p.width, raw + ((tile + 1) & 1) * kRaw);
          else cp_async_commit();
          cp_async_wait<1>();
          __syncthreads();
        }
#pragma unroll
        for (int i = threadIdx.x; i < kGCh * kT / kK; i += kGradThreads) {
          int ch, seg;
          unit_of<kGCh>(i, p.by_channel, ch, seg);
          if (ch >= width) continue;
          float dt[kK], dtu[kK], e[kK];
          Raw r;
          load_unit<T, HAS_Z>(p, b, d0 + ch, t0 + seg * kK, r, now, ch, seg);
          stage_unit<HAS_Z>(p, d0 + ch, t0 + seg * kK, r, dt, dtu, e);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int at = ch * kPitch + at_step(seg, h);
            *reinterpret_cast<float4*>(sd + at) = f4(dt[4 * h], dt[4 * h + 1], dt[4 * h + 2], dt[4 * h + 3]);
            *reinterpret_cast<float4*>(sdu + at) = f4(dtu[4 * h], dtu[4 * h + 1], dtu[4 * h + 2], dtu[4 * h + 3]);
            *reinterpret_cast<float4*>(se + at) = f4(e[4 * h], e[4 * h + 1], e[4 * h + 2], e[4 * h + 3]);
          }
        }
      }
      float* j = in + jc * kPitch + 4 * (threadIdx.x % 4);
      *reinterpret_cast<float4*>(j) = jA;
      *reinterpret_cast<float4*>(j + kNB) = jh;
      *reinterpret_cast<float4*>(j + 2 * kNB) = jk;
      __syncthreads();
      for (int ch = warp; ch < width; ch += kGradWarps) {
        const int d = d0 + ch;
        const float4* row = reinterpret_cast<const float4*>(in + ch * kPitch);
        const float4 xA = row[q], xh = row[kNB / 4 + q], xk = row[2 * kNB / 4 + q];
        const f2_t A2[2] = {f2_mul(f2_pack(xA.x, xA.y), dup(kLog2e)), f2_mul(f2_pack(xA.z, xA.w), dup(kLog2e))};
        const f2_t first[2] = {f2_pack(xh.x, xh.y), f2_pack(xh.z, xh.w)}, last[2] = {f2_pack(xk.x, xk.y), f2_pack(xk.z, xk.w)};
        float dt[kK], dtu[kK], e[kK];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int at = ch * kPitch + at_step(s, h);
          const float4 x = *reinterpret_cast<const float4*>(sd + at);
          const float4 y = *reinterpret_cast<const float4*>(sdu + at);
          const float4 w = *reinterpret_cast<const float4*>(se + at);
          dt[4 * h] = x.x, dt[4 * h + 1] = x.y, dt[4 * h + 2] = x.z, dt[4 * h + 3] = x.w;
          dtu[4 * h] = y.x, dtu[4 * h + 1] = y.y, dtu[4 * h + 2] = y.z, dtu[4 * h + 3] = y.w;
          e[4 * h] = w.x, e[4 * h + 1] = w.y, e[4 * h + 2] = w.z, e[4 * h + 3] = w.w;
        }
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < kK; ++i) sum += dt[i];
        f2_t a[kK][2], ah[kK][2], P[2], Q[2], h[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          Q[j] = P[j] = ex2_pair(mul1(A2[j], sum));
          h[j] = s == 0 ? first[j] : dup(0.f);
        }
        // both directions from zero (neither needs the other), then across segments
        f2_t k[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) k[j] = s == 7 ? last[j] : dup(0.f);
#pragma unroll
        for (int i = 0; i < kK; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j) a[i][j] = ex2_pair(mul1(A2[j], dt[i]));
#pragma unroll
        for (int i = 0; i < kK; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            h[j] = f2_fma(a[i][j], h[j], mul1(Bv[i][j], dtu[i]));
            k[j] = f2_mul(a[kK - 1 - i][j], fma1(Cv[kK - 1 - i][j], e[kK - 1 - i], k[j]));
          }
#pragma unroll
        for (int by = 1; by < 8; by *= 2)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const f2_t hb = shfl_up2(h[j], 4 * by), kb = shfl_down2(k[j], 4 * by);
            const f2_t Pb = shfl_up2(P[j], 4 * by), Qb = shfl_down2(Q[j], 4 * by);
            if (s >= by) {
              h[j] = f2_fma(P[j], hb, h[j]);
              P[j] = f2_mul(P[j], Pb);
            }
            if (s + by < 8) {
              k[j] = f2_fma(Q[j], kb, k[j]);
              Q[j] = f2_mul(Q[j], Qb);
            }
          }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const f2_t hb = shfl_up2(h[j], 4), kb = shfl_down2(k[j], 4);
          h[j] = s == 0 ? first[j] : hb;
          k[j] = s == 7 ? last[j] : kb;
        }
        float v3[kK];
#pragma unroll
        for (int i = 0; i < kK; ++i) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            ah[i][j] = f2_mul(a[i][j], h[j]);
            h[j] = fma1(Bv[i][j], dtu[i], ah[i][j]);
            accC[i][j] = fma1(h[j], e[i], accC[i][j]);
          }
          if (HAS_Z) {
            const float2 x = f2_unpack(f2_fma(h[0], Cv[i][0], f2_mul(h[1], Cv[i][1])));
            v3[i] = x.x + x.y;
          }
        }
        float v1[kK], v2[kK];
        f2_t dA[2] = {dup(0.f), dup(0.f)};
#pragma unroll
        for (int i = kK - 1; i >= 0; --i) {
          f2_t gB = dup(0.f), wA = dup(0.f);
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const f2_t g = fma1(Cv[i][j], e[i], k[j]);
            k[j] = f2_mul(a[i][j], g);
            accB[i][j] = fma1(g, dtu[i], accB[i][j]);
            gB = f2_fma(g, Bv[i][j], gB);
            const f2_t w = f2_mul(g, ah[i][j]);
            wA = f2_fma(w, A2[j], wA);
            dA[j] = fma1(w, dt[i], dA[j]);
          }
          const float2 x = f2_unpack(gB), y = f2_unpack(wA);
          v1[i] = x.x + x.y;
          v2[i] = y.x + y.y;
        }
        // sums over states, for the two steps that this quad keeps
        const int at = ch * kPitch + at_step(s, q & 1) + 2 * (q >> 1);
        float2 r1 = sum_quads(v1, q), r2 = sum_quads(v2, q), r3 = make_float2(0.f, 0.f);
        if (HAS_Z) r3 = sum_quads(v3, q);
        if (pass > 0) {
          const float2 x = *reinterpret_cast<float2*>(s1 + at), y = *reinterpret_cast<float2*>(s2 + at);
          r1 = make_float2(r1.x + x.x, r1.y + x.y);
          r2 = make_float2(r2.x + y.x, r2.y + y.y);
          if (HAS_Z) {
            const float2 w = *reinterpret_cast<float2*>(s3 + at);
            r3 = make_float2(r3.x + w.x, r3.y + w.y);
          }
        }
        *reinterpret_cast<float2*>(s1 + at) = r1;
        *reinterpret_cast<float2*>(s2 + at) = r2;
        if (HAS_Z) *reinterpret_cast<float2*>(s3 + at) = r3;
        // dA over the segments: lanes are left with one state each (twice)
        {
          const float2 x = f2_unpack(dA[0]), y = f2_unpack(dA[1]);
          const bool hi = s & 4, mid = s & 2;
          const float k0 = hi ? y.x : x.x, k1 = hi ? y.y : x.y, g0 = hi ? x.x : y.x, g1 = hi ? x.y : y.y;
          const float m0 = k0 + __shfl_xor_sync(0xffffffffu, g0, 16), m1 = k1 + __shfl_xor_sync(0xffffffffu, g1, 16);
          float v = (mid ? m1 : m0) + __shfl_xor_sync(0xffffffffu, mid ? m0 : m1, 8);
          v += __shfl_xor_sync(0xffffffffu, v, 4);
          const int n = n0 + (hi ? 2 : 0) + (mid ? 1 : 0);
          if (!(s & 1) && n < p.np) p.pA[(bc * p.dim + d) * p.np + n] = v;
        }
      }
      if (pass == p.passes - 1) {
        __syncthreads();
#pragma unroll
        for (int i = threadIdx.x; i < kGCh * kT / kK; i += kGradThreads) {
          int ch, seg;
          unit_of<kGCh>(i, p.by_channel, ch, seg);
          if (ch >= width) continue;
          const int d = d0 + ch, t = t0 + seg * kK, n = min(kK, p.seqlen - t);
          Raw r;
          load_unit<T, HAS_Z>(p, b, d, t, r, now, ch, seg);
          const float bias = p.bias ? p.bias[d] : 0.f, D = p.D ? p.D[d] : 0.f;
          float du[kK], dd[kK], sumD = 0.f, sumb = 0.f;
#pragma unroll
          for (int k = 0; k < kK; ++k) {
            const int at = ch * kPitch + at_step(seg, k >> 2) + (k & 3);
            const float e = se[at], gB = s1[at];
            du[k] = fmaf(sd[at], gB, D * e);
            dd[k] = fmaf(r.u[k], gB, s2[at] * kLn2) * step_slope(r.dt[k] + bias, p.softplus);
            sumD = fmaf(e, r.u[k], sumD);
            sumb += k < n ? dd[k] : 0.f;
            if (HAS_Z) r.g[k] = r.e[k] * fmaf(D, r.u[k], s3[at]) * gate_of(r.g[k]).slope;
          }
          store_steps(static_cast<T*>(p.du) + b * p.dus[0] + d * p.dus[1] + t * p.dus[2], p.dus[2], p.vec, n, du);
          store_steps(static_cast<T*>(p.ddelta) + b * p.dds[0] + d * p.dds[1] + t * p.dds[2], p.dds[2], p.vec, n, dd);
          if (HAS_Z)
            store_steps(static_cast<T*>(p.dz) + b * p.dzs[0] + d * p.dzs[1] + t * p.dzs[2], p.dzs[2], p.vec, n, r.g);
          sums[0][ch][seg] = sumD;
          sums[1][ch][seg] = sumb;
        }
        __syncthreads();
        for (int ch = threadIdx.x; ch < width; ch += kGradThreads) {
          float x = 0.f, y = 0.f;
#pragma unroll
          for (int seg = 0; seg < kT / kK; ++seg) {
            x += sums[0][ch][seg];
            y += sums[1][ch][seg];
          }
          p.pD[bc * p.dim + d0 + ch] = x;
          p.pbias[bc * p.dim + d0 + ch] = y;
        }
      }
    }
    // dB and dC of this group's channels: the warps' sums, in order, as [state][step]
    __syncthreads();
    float* all = sd;  // [warp][B or C][state][step]; the staged rows that a later pass reads are restored below
    static_assert(kGradWarps * 2 * kNB * kT <= (5 * kGCh * kPitch), "the warps' sums fit the free rows");
    all = once ? sd : more + 2 * kGCh * kPitch;
    float* mine = all + warp * 2 * kNB * kT;
#pragma unroll
    for (int i = 0; i < kK; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float2 x = f2_unpack(accB[i][j]), y = f2_unpack(accC[i][j]);
        const int at = (4 * q + 2 * j) * kT + s * kK + i;
        mine[at] = x.x;
        mine[at + kT] = x.y;
        mine[kNB * kT + at] = y.x;
        mine[kNB * kT + at + kT] = y.y;
      }
    __syncthreads();
    const long long out = ((((long long)b * p.groups + group) * p.chunks + c) * p.passes + pass) * kNB * kT;
    for (int i = threadIdx.x; i < kNB * kT; i += kGradThreads) {
      float x = 0.f, y = 0.f;
#pragma unroll
      for (int w = 0; w < kGradWarps; ++w) {
        x += all[w * 2 * kNB * kT + i];
        y += all[w * 2 * kNB * kT + kNB * kT + i];
      }
      p.pB[out + i] = x;
      p.pC[out + i] = y;
    }
  }
}

// ---- sums over groups and chunks -------------------------------------------------------------------
template <typename T> __global__ void __launch_bounds__(256) reduce_kernel(const Params p, long long bc_blocks) {
  if (blockIdx.x < bc_blocks) {  // dB and dC: over the groups of channels
    const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    const long long per = (long long)p.chunks * p.passes * kNB * kT;
    if (i >= p.batch * per) return;
    const long long b = i / per, r = i % per;
    const int step = (int)(r % kT), n = (int)(r / kT % (p.passes * kNB)), t = (int)(r / kT / (p.passes * kNB)) * kT + step;
    if (n >= p.dstate_n || t >= p.seqlen) return;
    double x = 0, y = 0;
    for (int g = 0; g < p.groups; ++g) {
      x += p.pB[(b * p.groups + g) * per + r];
      y += p.pC[(b * p.groups + g) * per + r];
    }
    st_f32(static_cast<T*>(p.dB) + b * p.dBs[0] + n * p.dBs[1] + t * p.dBs[2], (float)x);
    st_f32(static_cast<T*>(p.dC) + b * p.dCs[0] + n * p.dCs[1] + t * p.dCs[2], (float)y);
    return;
  }
  // dA, dD, dbias: over batch and chunks. Eight threads share a value, every eighth chunk each
  const int dn = p.dim * p.np;
  const long long v = ((long long)(blockIdx.x - bc_blocks) * 32) + threadIdx.x % 32;
  const int part = threadIdx.x / 32;
  const long long rows = (long long)p.batch * p.chunks;
  const float* src = nullptr;
  long long pitch = 0;
  if (v < dn) {
    src = p.pA + v;
    pitch = dn;
  } else if (v < dn + p.dim) {
    src = p.pD + (v - dn);
    pitch = p.dim;
  } else if (v < dn + 2LL * p.dim) {
    src = p.pbias + (v - dn - p.dim);
    pitch = p.dim;
  }
  double x = 0;
  if (src)
    for (long long r = part; r < rows; r += 8) x += src[r * pitch];
  __shared__ double sum[8][32];
  sum[part][threadIdx.x % 32] = x;
  __syncthreads();
  if (part != 0 || !src) return;
  for (int k = 1; k < 8; ++k) x += sum[k][threadIdx.x];
  if (v < dn) {
    const int d = (int)(v / p.np), n = (int)(v % p.np);
    if (n < p.dstate_n) p.dA[(long long)d * p.dstate_n + n] = (float)x;
  } else if (v < dn + p.dim) {
    if (p.dD) p.dD[v - dn] = (float)x;
  } else if (p.dbias) {
    p.dbias[v - dn - p.dim] = (float)x;
  }
}

// ---- host ---------------------------------------------------------------------------------------------
struct Layout {
  int chunks, np, passes, groups, tiles, width;
  size_t hst, kst, sum_d, pB, pC, pA, pD, pbias, bytes;
};

int make_layout(const MMScanBwdArgs* a, Layout* l) {
  const MMScanArgs& f = a->fwd;
  if (!dtype_size(f.dtype)) return MM_ERR_DTYPE;
  if (f.batch < 0 || f.dim < 0 || f.seqlen < 0 || f.dstate < 1 || f.dstate > MM_MAX_DSTATE || f.batch > 0x7fffffffLL ||
      f.dim > 0x7fffffffLL / (2 * MM_MAX_DSTATE) || f.seqlen > 0x7fffffffLL - kT)
    return MM_ERR_SHAPE;
  l->chunks = (int)((f.seqlen + kT - 1) / kT);
  l->np = (int)(f.dstate + 3) / 4 * 4;
  l->passes = (int)((f.dstate + kNB - 1) / kNB);
  // Channels of a CTA: as many as leave four CTAs to every one of the 2 x 148 places (fewer partial sums of dB
  // and dC), in tiles of 64; down to 16 channels where there are few chunks. States above 16 keep their staged
  // tile over the passes, so there one tile is the most.
  const long long rows = f.batch * (l->chunks > 0 ? l->chunks : 1);
  long long want = f.dim * rows / (4 * 2 * 148);
  l->width = want >= kGCh ? kGCh : 16;
  long long tiles = want / kGCh;
  l->tiles = (int)(l->passes > 1 || tiles < 1 ? 1 : tiles > 512 / kGCh ? 512 / kGCh : tiles);
  const long long per = (long long)l->width * l->tiles;
  l->groups = (int)((f.dim + per - 1) / per);
  size_t at = 0;
  auto take = [&](size_t n) {
    const size_t r = at;
    at += (n * sizeof(float) + 255) / 256 * 256;
    return r;
  };
  const size_t rowd = (size_t)rows * f.dim, st = rowd * l->np;
  const size_t bc = (size_t)rows * l->groups * l->passes * kNB * kT;
  l->hst = take(l->chunks > 1 ? st : 0);
  l->kst = take(l->chunks > 1 ? st : 0);
  l->sum_d = take(l->chunks > 1 ? rowd : 0);
  l->pB = take(bc);
  l->pC = take(bc);
  l->pA = take(st);
  l->pD = take(rowd);
  l->pbias = take(rowd);
  l->bytes = at + 256;
  return MM_OK;
}

inline void copy3(long long (&to)[3], const int64_t* from) {
  for (int i = 0; i < 3; ++i) to[i] = from[i];
}

template <typename T, bool HAS_Z> int launch(const Params& p, cudaStream_t s) {
  const long long rows = (long long)p.batch * p.chunks;
  const int carry_smem = 3 * kT * kCarryPitch * (int)sizeof(float);
  const int grad_smem = kGradSmem + 2 * kRaw * (int)sizeof(T) +
                        (p.passes > 1 ? (2 * kGCh * kPitch + kGradWarps * 2 * kNB * kT) * (int)sizeof(float) : 0);
  const long long dtiles = (p.dim + kCh - 1) / kCh;
  if (rows * dtiles > 0x7fffffffLL || rows * p.groups > 0x7fffffffLL) return MM_ERR_SHAPE;
  if (p.chunks > 1) {
    if (cudaFuncSetAttribute(carry_kernel<T, HAS_Z>, cudaFuncAttributeMaxDynamicSharedMemorySize, carry_smem) != cudaSuccess)
      return MM_ERR_LAUNCH;
    carry_kernel<T, HAS_Z><<<(unsigned)(rows * dtiles), kCarryThreads, carry_smem, s>>>(p);
    if (cudaGetLastError() != cudaSuccess) return MM_ERR_LAUNCH;
    const long long states = (long long)p.batch * p.dim * p.np;
    if ((states + 255) / 256 > 0x7fffffffLL) return MM_ERR_SHAPE;
    join_kernel<<<dim3((unsigned)((states + 255) / 256), 2), 256, 0, s>>>(p);
    if (cudaGetLastError() != cudaSuccess) return MM_ERR_LAUNCH;
  }
  if (cudaFuncSetAttribute(grad_kernel<T, HAS_Z>, cudaFuncAttributeMaxDynamicSharedMemorySize, grad_smem) != cudaSuccess)
    return MM_ERR_LAUNCH;
  grad_kernel<T, HAS_Z><<<(unsigned)(rows * p.groups), kGradThreads, grad_smem, s>>>(p);
  if (cudaGetLastError() != cudaSuccess) return MM_ERR_LAUNCH;
  const long long bc = (rows * p.passes * kNB * kT + 255) / 256;
  const long long rest = ((long long)p.dim * (p.np + 2) + 31) / 32;
  if (bc + rest > 0x7fffffffLL) return MM_ERR_SHAPE;
  reduce_kernel<T><<<(unsigned)(bc + rest), 256, 0, s>>>(p, bc);
  return cudaGetLastError() == cudaSuccess ? MM_OK : MM_ERR_LAUNCH;
}

template <typename T> int launch_z(const Params& p, cudaStream_t s) {
  return p.z ? launch<T, true>(p, s) : launch<T, false>(p, s);
}

bool rows_aligned(const void* q, const int64_t* st, const MMScanArgs& f) {
  const int es = dtype_size(f.dtype);
  return aligned16(q) && st[2] == 1 && (f.batch <= 1 || st[0] * es % 16 == 0) && (f.dim <= 1 || st[1] * es % 16 == 0);
}

bool columns_aligned(const void* q, const int64_t* st, const MMScanArgs& f) {
  const int es = dtype_size(f.dtype);
  return aligned16(q) && st[1] == 1 && (f.batch <= 1 || st[0] * es % 16 == 0) && st[2] * es % 16 == 0;
}

}  // namespace bwd
}  // namespace mm

using namespace mm;
using namespace mm::bwd;

extern "C" int mm_selective_scan_bwd_workspace_size(const MMScanBwdArgs* a, size_t* bytes) {
  if (!a || !bytes) return MM_ERR_ARG;
  Layout l;
  const int rc = make_layout(a, &l);
  if (rc == MM_OK) *bytes = l.bytes;
  return rc;
}

extern "C" int mm_selective_scan_bwd(const MMScanBwdArgs* a, void* workspace, size_t workspace_bytes, mm_stream_t stream) {
  if (!a) return MM_ERR_ARG;
  Layout l;
  const int rc = make_layout(a, &l);
  if (rc != MM_OK) return rc;
  const MMScanArgs& f = a->fwd;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (f.dim == 0) return MM_OK;
  if (!a->dA) return MM_ERR_ARG;
  if (f.batch == 0 || f.seqlen == 0) {  // sums over nothing
    if (cudaMemsetAsync(a->dA, 0, sizeof(float) * f.dim * f.dstate, s) != cudaSuccess) return MM_ERR_LAUNCH;
    if (a->dD && cudaMemsetAsync(a->dD, 0, sizeof(float) * f.dim, s) != cudaSuccess) return MM_ERR_LAUNCH;
    if (a->ddelta_bias && cudaMemsetAsync(a->ddelta_bias, 0, sizeof(float) * f.dim, s) != cudaSuccess) return MM_ERR_LAUNCH;
    return MM_OK;
  }
  if (!f.u || !f.delta || !f.A || !f.B || !f.C || !a->dy || !a->du || !a->ddelta || !a->dB || !a->dC || (f.z && !a->dz))
    return MM_ERR_ARG;
  if (!workspace || workspace_bytes < l.bytes || reinterpret_cast<uintptr_t>(workspace) % 256) return MM_ERR_WORKSPACE;
  Params p = {};
  p.u = f.u;
  p.delta = f.delta;
  p.z = f.z;
  p.B = f.B;
  p.C = f.C;
  p.dy = a->dy;
  p.A = f.A;
  p.D = f.D;
  p.bias = f.delta_bias;
  p.dstate = a->dstate;
  p.du = a->du;
  p.ddelta = a->ddelta;
  p.dz = a->dz;
  p.dB = a->dB;
  p.dC = a->dC;
  p.dA = a->dA;
  p.dD = a->dD;
  p.dbias = a->ddelta_bias;
  copy3(p.us, f.u_stride);
  copy3(p.ds, f.delta_stride);
  copy3(p.zs, f.z_stride);
  copy3(p.Bs, f.B_stride);
  copy3(p.Cs, f.C_stride);
  copy3(p.ys, a->dy_stride);
  copy3(p.dus, a->du_stride);
  copy3(p.dds, a->ddelta_stride);
  copy3(p.dzs, a->dz_stride);
  copy3(p.dBs, a->dB_stride);
  copy3(p.dCs, a->dC_stride);
  p.As[0] = f.A_stride[0];
  p.As[1] = f.A_stride[1];
  p.batch = (int)f.batch;
  p.dim = (int)f.dim;
  p.dstate_n = (int)f.dstate;
  p.seqlen = (int)f.seqlen;
  p.softplus = f.delta_softplus != 0;
  p.vec = rows_aligned(f.u, f.u_stride, f) && rows_aligned(f.delta, f.delta_stride, f) &&
          rows_aligned(a->dy, a->dy_stride, f) && rows_aligned(a->du, a->du_stride, f) &&
          rows_aligned(a->ddelta, a->ddelta_stride, f) &&
          (!f.z || (rows_aligned(f.z, f.z_stride, f) && rows_aligned(a->dz, a->dz_stride, f)));
  p.by_channel = !p.vec && f.u_stride[1] == 1 && f.u_stride[2] != 1;
  const void* act[4] = {f.u, f.delta, a->dy, f.z};
  const int64_t* act_stride[4] = {f.u_stride, f.delta_stride, a->dy_stride, f.z_stride};
  p.ahead = 1;
  for (int i = 0; i < (f.z ? 4 : 3); ++i)
    if (!(p.by_channel ? columns_aligned(act[i], act_stride[i], f) : rows_aligned(act[i], act_stride[i], f))) p.ahead = 0;
  p.chunks = l.chunks;
  p.np = l.np;
  p.passes = l.passes;
  p.groups = l.groups;
  p.tiles = l.tiles;
  p.width = l.width;
  char* w = static_cast<char*>(workspace);
  p.hst = reinterpret_cast<float*>(w + l.hst);
  p.kst = reinterpret_cast<float*>(w + l.kst);
  p.sum_d = reinterpret_cast<float*>(w + l.sum_d);
  p.pB = reinterpret_cast<float*>(w + l.pB);
  p.pC = reinterpret_cast<float*>(w + l.pC);
  p.pA = reinterpret_cast<float*>(w + l.pA);
  p.pD = reinterpret_cast<float*>(w + l.pD);
  p.pbias = reinterpret_cast<float*>(w + l.pbias);
  switch (f.dtype) {
    case MM_F32: return launch_z<float>(p, s);
    case MM_F16: return launch_z<__half>(p, s);
    default: return launch_z<__nv_bfloat16>(p, s);
  }
}
