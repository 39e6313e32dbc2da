// Gradient of the selective scan.
//
// With d = softplus(delta + bias), a_t = exp(d_t A), h_t = a_t h_{t-1} + d_t u_t B_t, p_t = sum_n C_t h_t + D u_t,
// y = p silu(z), and e = dy silu(z), the gradient runs the same kind of recurrence backwards in time:
//   g_t = C_t e_t + k_t,  k_t = a_{t+1} g_{t+1}  (k at the end: the last state's gradient)
//   dC_t = sum_d h e     dB_t = sum_d g d u     du = d sum_n g B + D e     w = g a h_{t-1}
//   dd = u sum_n g B + sum_n A w     dA = sum_{b,t} d w     dz = dy p silu'(z)     dD = sum e u
// Time is cut into chunks of 32 steps. The forward pass leaves the state that every chunk starts from; walk_back
// (mm_scan_walk.cu) finds the k that comes into every chunk; then grad_kernel takes all chunks side by side.
// Sums over channels and over chunks leave as partials that reduce_kernel adds in a fixed order, so the results
// do not depend on timing. All state and all sums are float32 (the last sums over partials float64).
#include "mm_scan_train.cuh"

namespace mm {
namespace train {

constexpr int kPitch = kT + 4;  // floats of a staged row; rows stay 16-byte aligned, neighbours in other banks
constexpr int kNB = 16;         // states of a pass

// The raw values of a unit, so that several units' loads can be in flight before the first is worked on
struct Raw {
  float dt[kK], u[kK], e[kK], g[kK];
};
template <typename T, bool HAS_Z> MM_DEV void load_unit(const Params& p, int b, int d, int t, Raw& r) {
  const int n = min(kK, p.seqlen - t);
  load_steps(static_cast<const T*>(p.delta) + b * p.ds[0] + d * p.ds[1] + t * p.ds[2], p.ds[2], p.access, n, r.dt);
  load_steps(static_cast<const T*>(p.u) + b * p.us[0] + d * p.us[1] + t * p.us[2], p.us[2], p.access, n, r.u);
  load_steps(static_cast<const T*>(p.dy) + b * p.ys[0] + d * p.ys[1] + t * p.ys[2], p.ys[2], p.access, n, r.e);
  if (HAS_Z) load_steps(static_cast<const T*>(p.z) + b * p.zs[0] + d * p.zs[1] + t * p.zs[2], p.zs[2], p.access, n, r.g);
}

// d, d u and e (zeros where there are no steps: a = 1 there, so states and k pass through)
template <bool HAS_Z>
MM_DEV void stage_unit(const Params& p, int d, int t, const Raw& r, float (&dt)[kK], float (&dtu)[kK], float (&e)[kK]) {
  const int n = min(kK, p.seqlen - t);
  const f2_t bias = dup(p.bias ? p.bias[d] : 0.f);
#pragma unroll
  for (int k = 0; k < kK; k += 2) {
    const float2 x = f2_unpack(step_of(f2_add(f2_pack(r.dt[k], r.dt[k + 1]), bias), p.softplus));
    dt[k] = k < n ? x.x : 0.f;
    dt[k + 1] = k + 1 < n ? x.y : 0.f;
    const float2 y = f2_unpack(f2_mul(f2_pack(dt[k], dt[k + 1]), f2_pack(r.u[k], r.u[k + 1])));
    dtu[k] = y.x;
    dtu[k + 1] = y.y;
    f2_t g = f2_pack(r.e[k], r.e[k + 1]);
    if (HAS_Z) g = f2_mul(g, silu_of(f2_pack(r.g[k], r.g[k + 1])));
    const float2 w = f2_unpack(g);
    e[k] = w.x;
    e[k + 1] = w.y;
  }
}

// ---- the gradient of every chunk ------------------------------------------------------------------------
// A warp works off channels one by one: lane = 8 * segment + pair holds eight steps of two states. Each segment
// runs its steps from zero, a scan over the four segments gives its true start, and a second run the values;
// the same backwards. B, C and the sums for dB and dC stay in registers over all channels, so the sum over
// channels costs nothing but the final one over warps; sums over states go across the eight lanes of a segment.

// Position of a segment's half in a staged row: the first halves of the segments lie side by side, so that their
// 16-byte reads fall into different banks.
MM_DEV int at_step(int seg, int half) { return (half * kSegs + seg) * 4; }
MM_DEV void fetch_steps(const float* row, int seg, float (&v)[kK]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const float4 x = *reinterpret_cast<const float4*>(row + at_step(seg, h));
    v[4 * h] = x.x, v[4 * h + 1] = x.y, v[4 * h + 2] = x.z, v[4 * h + 3] = x.w;
  }
}

MM_DEV f2_t shfl_up2(f2_t v, int by) {
  const float2 x = f2_unpack(v);
  return f2_pack(__shfl_up_sync(0xffffffffu, x.x, by), __shfl_up_sync(0xffffffffu, x.y, by));
}
MM_DEV f2_t shfl_down2(f2_t v, int by) {
  const float2 x = f2_unpack(v);
  return f2_pack(__shfl_down_sync(0xffffffffu, x.x, by), __shfl_down_sync(0xffffffffu, x.y, by));
}

// A staged channel's record: rows of d, d u, e; A, the incoming state and k of 16 states; rows of the sums over
// states sum_n g B, A w, C h. The pitch puts neighbouring channels' 16-byte words into different banks.
struct Once {  // all states in one pass: sums replace what the same warp has read
  static constexpr int d = 0, du = kPitch, e = 2 * kPitch, s1 = du, s2 = 3 * kPitch, s3 = 4 * kPitch, in = s2, size = 5 * kPitch;
};
struct Passes {
  static constexpr int d = 0, du = kPitch, e = 2 * kPitch, s1 = 3 * kPitch, s2 = 4 * kPitch, s3 = 5 * kPitch, in = 6 * kPitch,
                       size = 6 * kPitch + 3 * kNB + 4;
};
static_assert(2 * kPitch >= 3 * kNB && Once::size / 4 % 2 == 1 && Passes::size / 4 % 2 == 1, "the records' layout");

// One channel of a chunk, by one warp: lane = 8 * segment + pair. The sums go to the channel's record (added to
// what is there if `more`), dA's partial sum to pA. temp: this warp's.
constexpr int kTempRow = 7;  // 16-byte words of a lane: six, and one for the banks' sake
constexpr int kTemp = 32 * kTempRow;

template <typename R, bool HAS_Z>
MM_DEV void work_channel(int lane, float* rec, bool more, float4* temp, const f2_t (&Bv)[kK], const f2_t (&Cv)[kK],
                         f2_t (&accB)[kK], f2_t (&accC)[kK], float* pA, int np) {
  const int q = lane & 7, s = lane >> 3;
  const float *sd = rec + R::d, *sdu = rec + R::du, *se = rec + R::e;
  const f2_t* in2 = reinterpret_cast<const f2_t*>(rec + R::in);
  const f2_t A2 = f2_mul(in2[q], dup(kLog2e)), first = in2[kNB / 2 + q], last = in2[kNB + q];
  float4* mine = temp + lane * kTempRow;
  f2_t a[kK], ah[kK], P, Q, h, k;
  float dt[kK], dtu[kK], e[kK];
  {
    fetch_steps(sd, s, dt);
    fetch_steps(sdu, s, dtu);
    fetch_steps(se, s, e);
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < kK; ++i) sum += dt[i];
    const f2_t span = ex2_pair(mul1(A2, sum));
    // The first segment has its true start, and nothing comes into it: its span counts as 0, which also makes
    // what the shuffles give lanes that have no partner count for nothing
    P = s == 0 ? dup(0.f) : span;
    Q = s == kSegs - 1 ? dup(0.f) : span;
    h = s == 0 ? first : dup(0.f);
    k = s == kSegs - 1 ? last : dup(0.f);
    // both directions from zero (neither needs the other), then across segments
#pragma unroll
    for (int i = 0; i < kK; ++i) a[i] = ex2_pair(mul1(A2, dt[i]));
#pragma unroll
    for (int i = 0; i < kK; ++i) {
      h = f2_fma(a[i], h, mul1(Bv[i], dtu[i]));
      k = f2_mul(a[kK - 1 - i], fma1(Cv[kK - 1 - i], e[kK - 1 - i], k));
    }
  }
#pragma unroll
  for (int by = 1; by < kSegs; by *= 2) {
    h = f2_fma(P, shfl_up2(h, 8 * by), h);
    k = f2_fma(Q, shfl_down2(k, 8 * by), k);
    if (by < kSegs / 2) {
      P = f2_mul(P, shfl_up2(P, 8 * by));
      Q = f2_mul(Q, shfl_down2(Q, 8 * by));
    }
  }
  {
    const f2_t hb = shfl_up2(h, 8), kb = shfl_down2(k, 8);
    h = s == 0 ? first : hb;
    k = s == kSegs - 1 ? last : kb;
  }
  {
    float v[kK];
#pragma unroll
    for (int i = 0; i < kK; ++i) {
      ah[i] = f2_mul(a[i], h);
      h = fma1(Bv[i], dtu[i], ah[i]);
      accC[i] = fma1(h, e[i], accC[i]);
      const float2 x = f2_unpack(f2_mul(h, Cv[i]));
      v[i] = x.x + x.y;
    }
    if (HAS_Z) {
      mine[4] = f4(v[0], v[1], v[2], v[3]);
      mine[5] = f4(v[4], v[5], v[6], v[7]);
    }
  }
  f2_t dA = dup(0.f);
#pragma unroll
  for (int half = 1; half >= 0; --half) {
    float v1[4], v2[4];
#pragma unroll
    for (int j = 3; j >= 0; --j) {
      const int i = 4 * half + j;
      const f2_t g = fma1(Cv[i], e[i], k);
      k = f2_mul(a[i], g);
      accB[i] = fma1(g, dtu[i], accB[i]);
      const f2_t w = f2_mul(g, ah[i]);
      dA = fma1(w, dt[i], dA);
      const float2 x = f2_unpack(f2_mul(g, Bv[i])), y = f2_unpack(f2_mul(w, A2));
      v1[j] = x.x + x.y;
      v2[j] = y.x + y.y;
    }
    mine[half] = f4(v1[0], v1[1], v1[2], v1[3]);
    mine[2 + half] = f4(v2[0], v2[1], v2[2], v2[3]);
  }
  __syncwarp();
  // sums over states: of a segment's eight lanes two each add sum_n g B, A w, C h, four steps each
  if (q < (HAS_Z ? 6 : 4)) {
    float* out = rec + (q < 2 ? R::s1 : q < 4 ? R::s2 : R::s3) + at_step(s, q & 1);
    float4 sum = more ? *reinterpret_cast<float4*>(out) : f4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float4 x = temp[(8 * s + i) * kTempRow + q];
      sum = f4(sum.x + x.x, sum.y + x.y, sum.z + x.z, sum.w + x.w);
    }
    *reinterpret_cast<float4*>(out) = sum;
  }
  __syncwarp();
  // dA over the segments: lanes are left with one state each (twice)
  {
    const float2 x = f2_unpack(dA);
    const bool hi = s & 2;
    float v = (hi ? x.y : x.x) + __shfl_xor_sync(0xffffffffu, hi ? x.x : x.y, 16);
    v += __shfl_xor_sync(0xffffffffu, v, 8);
    const int n = 2 * q + (hi ? 1 : 0);
    if (!(s & 1) && n < np) pA[n] = v;
  }
}

// B and C of a lane's steps and its two states
template <typename T>
MM_DEV void load_BC_lane(const Params& p, int b, int n, int t, f2_t (&Bv)[kK], f2_t (&Cv)[kK]) {
  const T* x = static_cast<const T*>(p.B) + b * p.Bs[0] + n * p.Bs[1] + t * p.Bs[2];
  const T* y = static_cast<const T*>(p.C) + b * p.Cs[0] + n * p.Cs[1] + t * p.Cs[2];
#pragma unroll
  for (int i = 0; i < kK; ++i) {
    const bool one = t + i < p.seqlen && n < p.dstate_n, two = t + i < p.seqlen && n + 1 < p.dstate_n;
    Bv[i] = f2_pack(one ? ld_f32(x + i * p.Bs[2]) : 0.f, two ? ld_f32(x + i * p.Bs[2] + p.Bs[1]) : 0.f);
    Cv[i] = f2_pack(one ? ld_f32(y + i * p.Cs[2]) : 0.f, two ? ld_f32(y + i * p.Cs[2] + p.Cs[1]) : 0.f);
  }
}

// What work_channel wants of a channel besides its row: A, the incoming state and the incoming k of four states
struct Incoming {
  float4 A, h, k;
};
MM_DEV Incoming load_incoming(const Params& p, long long bc, int b, int d, int n0) {
  Incoming r;
  r.A = load_A(p, d, n0);
  r.h = r.k = f4(0.f, 0.f, 0.f, 0.f);
  const long long at = (bc * p.dim + d) * p.np + n0;
  if (p.longs > 1) {
    if (n0 < p.np) {
      const long long bl = (long long)b * p.longs + (int)(bc % p.chunks) / p.per_long;
      r.k = *reinterpret_cast<const float4*>(p.klong + (bl * p.dim + d) * p.np + n0);
    }
  } else if (p.dstate) {
    const float* x = p.dstate + ((long long)b * p.dim + d) * p.dstate_n + n0;
    const int m = p.dstate_n - n0;
    r.k = f4(m > 0 ? x[0] : 0.f, m > 1 ? x[1] : 0.f, m > 2 ? x[2] : 0.f, m > 3 ? x[3] : 0.f);
  }
  if (p.chunks > 1 && n0 < p.np) {
    r.h = *reinterpret_cast<const float4*>(p.hst + at);
    const float4 x = *reinterpret_cast<const float4*>(p.kst + at);
    const float span = p.later[bc * p.dim + d] * kLog2e;
    r.k = f4(fmaf(ex2(span * r.A.x), r.k.x, x.x), fmaf(ex2(span * r.A.y), r.k.y, x.y), fmaf(ex2(span * r.A.z), r.k.z, x.z),
             fmaf(ex2(span * r.A.w), r.k.w, x.w));
  }
  return r;
}
MM_DEV void store_incoming(float* row, int quad, const Incoming& v) {
  float4* x = reinterpret_cast<float4*>(row);
  x[quad] = v.A;
  x[kNB / 4 + quad] = v.h;
  x[2 * kNB / 4 + quad] = v.k;
}

MM_DEV void store_unit(float* row, int seg, const float (&v)[kK]) {
#pragma unroll
  for (int h = 0; h < 2; ++h)
    *reinterpret_cast<float4*>(row + at_step(seg, h)) = f4(v[4 * h], v[4 * h + 1], v[4 * h + 2], v[4 * h + 3]);
}
MM_DEV void fetch_unit(const float* row, int seg, f2_t (&v)[kK / 2]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(row + at_step(seg, h));
    v[2 * h] = x.x;
    v[2 * h + 1] = x.y;
  }
}

// From the sums over states to the gradients of a unit's steps, and the unit's sums for dD and of ddelta
template <typename T, typename R, bool HAS_Z>
MM_DEV void finish_unit(const Params& p, int b, int d, int t, int seg, const Raw& r, const float* rec, float& sumD,
                        float& sumb) {
  const int n = min(kK, p.seqlen - t);
  const f2_t bias = dup(p.bias ? p.bias[d] : 0.f), D = dup(p.D ? p.D[d] : 0.f);
  f2_t e[kK / 2], gB[kK / 2], x[kK / 2], sum = dup(0.f);
  float out[kK];
  auto put = [&](int k, f2_t v) {
    const float2 w = f2_unpack(v);
    out[2 * k] = w.x;
    out[2 * k + 1] = w.y;
  };
  fetch_unit(rec + R::e, seg, e);
  fetch_unit(rec + R::s1, seg, gB);
  fetch_unit(rec + R::d, seg, x);
#pragma unroll
  for (int k = 0; k < kK / 2; ++k) {
    put(k, f2_fma(x[k], gB[k], f2_mul(D, e[k])));
    sum = f2_fma(e[k], f2_pack(r.u[2 * k], r.u[2 * k + 1]), sum);
  }
  sumD = f2_unpack(sum).x + f2_unpack(sum).y;
  store_steps(static_cast<T*>(p.du) + b * p.dus[0] + d * p.dus[1] + t * p.dus[2], p.dus[2], p.access, n, out);
  fetch_unit(rec + R::s2, seg, x);
#pragma unroll
  for (int k = 0; k < kK / 2; ++k)
    put(k, f2_mul(f2_fma(f2_pack(r.u[2 * k], r.u[2 * k + 1]), gB[k], f2_mul(x[k], dup(kLn2))),
                  step_slope(f2_add(f2_pack(r.dt[2 * k], r.dt[2 * k + 1]), bias), p.softplus)));
  sumb = 0.f;
#pragma unroll
  for (int k = 0; k < kK; ++k) sumb += k < n ? out[k] : 0.f;
  store_steps(static_cast<T*>(p.ddelta) + b * p.dds[0] + d * p.dds[1] + t * p.dds[2], p.dds[2], p.access, n, out);
  if (HAS_Z) {
    fetch_unit(rec + R::s3, seg, x);
#pragma unroll
    for (int k = 0; k < kK / 2; ++k)
      put(k, f2_mul(f2_mul(f2_pack(r.e[2 * k], r.e[2 * k + 1]), f2_fma(D, f2_pack(r.u[2 * k], r.u[2 * k + 1]), x[k])),
                    silu_slope(f2_pack(r.g[2 * k], r.g[2 * k + 1]))));
    store_steps(static_cast<T*>(p.dz) + b * p.dzs[0] + d * p.dzs[1] + t * p.dzs[2], p.dzs[2], p.access, n, out);
  }
}

// Offset of a chunk's [state][step] block in the partial sums of dB and dC
MM_DEV long long block_of(const Params& p, int b, int group, int c, int pass) {
  return ((((long long)b * p.groups + group) * p.chunks + c) * p.passes + pass) * kNB * kT;
}
// Register pair i of a lane holds, of accB or accC, its two states at its step i
MM_DEV int lane_place(int state, int step) { return ((step % kK) * 2 + state % 2) * 32 + (step / kK) * 8 + state / 2; }
template <bool ADD> MM_DEV void put_sums(float* at, int lane, const f2_t (&acc)[kK]) {
#pragma unroll
  for (int i = 0; i < kK; ++i) {
    float2 x = f2_unpack(acc[i]);
    float* q = at + i * 2 * 32 + lane;
    if (ADD) {
      x.x += q[0];
      x.y += q[32];
    }
    q[0] = x.x;
    q[32] = x.y;
  }
}

// ---- up to 16 states ----
// Three CTAs of four warps per SM (the registers' limit) take (chunk, group of channels) items tile by tile: some are
// in their elementwise parts while others work. The raw inputs of the next tile arrive by cp.async meanwhile.
//
// f16 8x1536x4096, 16 states: 1.25 ms. 478 instructions for 32 steps of a channel, 0.51 of them a clock and scheduler
// with three warps on each; the way in from shared memory is 59 % taken, the FMA pipe 46 %, memory (0.7 TB/s) hardly.
// What did not pay: tiles of 64 steps with four states a lane, which halve the shuffles but leave two CTAs an SM; warps
// for the elementwise parts beside warps for the states, whose registers then spill.
constexpr int kGradThreads = 128;
// float32's raw inputs take twice the room, and a tile of half the channels keeps three CTAs on an SM
template <typename T> constexpr int kTile = sizeof(T) == 4 ? 16 : 32;
template <typename T> constexpr int kRawOne = kTile<T> * kT;  // [channel][step] or, contiguous along channels, [step][channel]
template <typename T> constexpr int kRaw = 4 * kRawOne<T>;
template <typename T> constexpr int kGradSmem = kTile<T> * Once::size * 4 + 2 * kRaw<T> * (int)sizeof(T) + 4 * kTemp * 16;

MM_DEV void cp_async16_part(void* dst, const void* src, int bytes) {  // zeros after the first `bytes`
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes) : "memory");
}
// Starts copying a tile's raw inputs; one commit group. Channels and steps that do not exist arrive as zeros.
template <typename T>
MM_DEV void copy_one(const void* base, const long long (&st)[3], const Params& p, int b, int t0, int d0, T* raw) {
  const T* x = static_cast<const T*>(base) + b * st[0] + d0 * st[1] + t0 * st[2];
  constexpr int per = 16 / (int)sizeof(T), CH = kTile<T>;
  const int width = min(CH, p.dim - d0), steps = min(kT, p.seqlen - t0);
#pragma unroll
  for (int j = 0; j < kRawOne<T> / per / kGradThreads; ++j) {
    const int i = threadIdx.x + j * kGradThreads;
    const int row = p.by_channel ? i / (CH / per) : i / (kT / per);
    const int col = (p.by_channel ? i % (CH / per) : i % (kT / per)) * per;
    const int n = p.by_channel ? (row < steps ? width - col : 0) : (row < width ? steps - col : 0);
    const T* src = n > 0 ? x + row * (p.by_channel ? st[2] : st[1]) + col : x;
    cp_async16_part(raw + i * per, src, min(max(n, 0), per) * (int)sizeof(T));
  }
}
template <typename T, bool HAS_Z> MM_DEV void copy_tile(const Params& p, int b, int t0, int d0, T* raw) {
  if (d0 < p.dim) {
    copy_one(p.delta, p.ds, p, b, t0, d0, raw);
    copy_one(p.u, p.us, p, b, t0, d0, raw + kRawOne<T>);
    copy_one(p.dy, p.ys, p, b, t0, d0, raw + 2 * kRawOne<T>);
    if (HAS_Z) copy_one(p.z, p.zs, p, b, t0, d0, raw + 3 * kRawOne<T>);
  }
  cp_async_commit();
}
template <typename T, bool HAS_Z>
MM_DEV void load_unit(const Params& p, int b, int d, int t, Raw& r, const T* raw, int ch, int seg) {
  if (!p.ahead) {
    load_unit<T, HAS_Z>(p, b, d, t, r);
    return;
  }
  const T* x = raw + (p.by_channel ? seg * kK * kTile<T> + ch : ch * kT + seg * kK);
  const int st = p.by_channel ? kTile<T> : 1, access = p.by_channel ? kAnyStride : kAligned;
  load_steps(x, st, access, kK, r.dt);
  load_steps(x + kRawOne<T>, st, access, kK, r.u);
  load_steps(x + 2 * kRawOne<T>, st, access, kK, r.e);
  if (HAS_Z) load_steps(x + 3 * kRawOne<T>, st, access, kK, r.g);
}

template <typename T, bool HAS_Z>
__global__ void __launch_bounds__(kGradThreads, 3) grad_kernel(const Params p) {
  constexpr int CH = kTile<T>, units = (CH * kSegs + kGradThreads - 1) / kGradThreads;
  extern __shared__ float4 smem4[];
  float* recs = reinterpret_cast<float*>(smem4);
  T* raw = reinterpret_cast<T*>(recs + CH * Once::size);  // two buffers of the raw delta, u, dy, z
  float4* temp = reinterpret_cast<float4*>(raw + 2 * kRaw<T>);
  __shared__ float sums[2][CH][kSegs];  // of dD and ddelta, per segment
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int group = (int)(blockIdx.x % p.groups);
  const long long bc = blockIdx.x / p.groups;
  const int c = (int)(bc % p.chunks), b = (int)(bc / p.chunks), t0 = c * kT;
  const int begin = group * p.tiles * p.width, end = min(p.dim, begin + p.tiles * p.width);

  if (p.ahead) copy_tile<T, HAS_Z>(p, b, t0, begin, raw);
  f2_t Bv[kK], Cv[kK], accB[kK], accC[kK];
  load_BC_lane<T>(p, b, 2 * (lane & 7), t0 + (lane >> 3) * kK, Bv, Cv);
#pragma unroll
  for (int k = 0; k < kK; ++k) accB[k] = accC[k] = dup(0.f);

  for (int d0 = begin, i = 0; d0 < end; d0 += p.width, ++i) {
    const int width = min(p.width, end - d0);
    T* now = raw + (i & 1) * kRaw<T>;
    Incoming x = {};
    if (tid / 4 < width) x = load_incoming(p, bc, b, d0 + tid / 4, 4 * (tid % 4));
    __syncthreads();  // the tile before has been read
    if (p.ahead) {
      copy_tile<T, HAS_Z>(p, b, t0, d0 + p.width < end ? d0 + p.width : p.dim, raw + (~i & 1) * kRaw<T>);
      cp_async_wait<1>();
      __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < units; ++j) {
      int ch, seg;
      unit_of<CH>(tid + j * kGradThreads, p.by_channel, ch, seg);
      if (ch >= width || seg >= kSegs) continue;
      Raw r;
      float dt[kK], dtu[kK], e[kK];
      load_unit<T, HAS_Z>(p, b, d0 + ch, t0 + seg * kK, r, now, ch, seg);
      stage_unit<HAS_Z>(p, d0 + ch, t0 + seg * kK, r, dt, dtu, e);
      float* rec = recs + ch * Once::size;
      store_unit(rec + Once::d, seg, dt);
      store_unit(rec + Once::du, seg, dtu);
      store_unit(rec + Once::e, seg, e);
    }
    if (tid / 4 < CH) store_incoming(recs + tid / 4 * Once::size + Once::in, tid % 4, x);
    __syncthreads();
    for (int ch = warp; ch < width; ch += kGradThreads / 32)
      work_channel<Once, HAS_Z>(lane, recs + ch * Once::size, false, temp + warp * kTemp, Bv, Cv, accB, accC,
                                p.pA + (bc * p.dim + d0 + ch) * p.np, p.np);
    __syncthreads();
#pragma unroll
    for (int j = 0; j < units; ++j) {
      int ch, seg;
      unit_of<CH>(tid + j * kGradThreads, p.by_channel, ch, seg);
      if (ch >= width || seg >= kSegs) continue;
      Raw r;
      load_unit<T, HAS_Z>(p, b, d0 + ch, t0 + seg * kK, r, now, ch, seg);
      finish_unit<T, Once, HAS_Z>(p, b, d0 + ch, t0 + seg * kK, seg, r, recs + ch * Once::size, sums[0][ch][seg],
                                  sums[1][ch][seg]);
    }
    __syncthreads();
    if (tid < 2 * width) {
      float v = 0.f;
#pragma unroll
      for (int seg = 0; seg < kSegs; ++seg) v += sums[tid & 1][tid >> 1][seg];
      ((tid & 1) ? p.pbias : p.pD)[bc * p.dim + d0 + (tid >> 1)] = v;
    }
  }
  // dB and dC of this group's channels: the warps' sums, in order
  float* all = reinterpret_cast<float*>(temp);  // [B or C][lane place]
  static_assert(2 * kNB * kT * 4 <= 4 * kTemp * 16, "the sums fit");
  for (int k = 0; k < kGradThreads / 32; ++k) {
    if (k == warp) {
      if (k == 0) {
        put_sums<false>(all, lane, accB);
        put_sums<false>(all + kNB * kT, lane, accC);
      } else {
        put_sums<true>(all, lane, accB);
        put_sums<true>(all + kNB * kT, lane, accC);
      }
    }
    __syncthreads();
  }
  const long long out = block_of(p, b, group, c, 0);
  for (int k = tid; k < kNB * kT; k += kGradThreads) {
    const int place = lane_place(k / kT, k % kT);
    p.pB[out + k] = all[place];
    p.pC[out + k] = all[kNB * kT + place];
  }
}

// ---- more than 16 states ----
// The same in passes of 16 states over one staged tile of channels per CTA; every warp does all of it (bf16 8x1536x512
// with 64 states 0.86 ms; a state and step takes 1.4 times what it takes with 16, for the staging of every pass).
constexpr int kWideThreads = 128;
constexpr int kWideCh = 32;
constexpr int kWideSmem = kWideCh * Passes::size * 4 + 4 * kTemp * 16 + 4 * 2 * kNB * kT * 4;

template <typename T, bool HAS_Z>
__global__ void __launch_bounds__(kWideThreads, 1) grad_wide_kernel(const Params p) {
  extern __shared__ float4 smem4[];
  float* recs = reinterpret_cast<float*>(smem4);
  float4* temp = reinterpret_cast<float4*>(recs + kWideCh * Passes::size);
  float* all = reinterpret_cast<float*>(temp + 4 * kTemp);  // [warp][B or C][lane place]
  __shared__ float sums[2][kWideCh][kSegs];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int group = (int)(blockIdx.x % p.groups);
  const long long bc = blockIdx.x / p.groups;
  const int c = (int)(bc % p.chunks), b = (int)(bc / p.chunks), t0 = c * kT;
  const int d0 = group * p.width, width = min(p.width, p.dim - d0);
  for (int k = tid; k < kWideCh * kSegs; k += kWideThreads) {
    int ch, seg;
    unit_of<kWideCh>(k, p.by_channel, ch, seg);
    if (ch >= width) continue;
    Raw r;
    float dt[kK], dtu[kK], e[kK];
    load_unit<T, HAS_Z>(p, b, d0 + ch, t0 + seg * kK, r);
    stage_unit<HAS_Z>(p, d0 + ch, t0 + seg * kK, r, dt, dtu, e);
    float* rec = recs + ch * Passes::size;
    store_unit(rec + Passes::d, seg, dt);
    store_unit(rec + Passes::du, seg, dtu);
    store_unit(rec + Passes::e, seg, e);
  }
  for (int pass = 0; pass < p.passes; ++pass) {
    const int n0 = pass * kNB;
    f2_t Bv[kK], Cv[kK], accB[kK], accC[kK];
    load_BC_lane<T>(p, b, n0 + 2 * (lane & 7), t0 + (lane >> 3) * kK, Bv, Cv);
#pragma unroll
    for (int k = 0; k < kK; ++k) accB[k] = accC[k] = dup(0.f);
    if (tid / 4 < width)
      store_incoming(recs + tid / 4 * Passes::size + Passes::in, tid % 4, load_incoming(p, bc, b, d0 + tid / 4, n0 + 4 * (tid % 4)));
    __syncthreads();
    for (int ch = warp; ch < width; ch += 4)
      work_channel<Passes, HAS_Z>(lane, recs + ch * Passes::size, pass > 0, temp + warp * kTemp, Bv, Cv, accB, accC,
                                  p.pA + (bc * p.dim + d0 + ch) * p.np + n0, p.np - n0);
    float* mine = all + warp * 2 * kNB * kT;
    put_sums<false>(mine, lane, accB);
    put_sums<false>(mine + kNB * kT, lane, accC);
    __syncthreads();
    const long long out = block_of(p, b, group, c, pass);
    for (int k = tid; k < kNB * kT; k += kWideThreads) {
      const int place = lane_place(k / kT, k % kT);
      float x = 0.f, y = 0.f;
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        x += all[v * 2 * kNB * kT + place];
        y += all[v * 2 * kNB * kT + kNB * kT + place];
      }
      p.pB[out + k] = x;
      p.pC[out + k] = y;
    }
  }
  for (int k = tid; k < kWideCh * kSegs; k += kWideThreads) {
    int ch, seg;
    unit_of<kWideCh>(k, p.by_channel, ch, seg);
    if (ch >= width) continue;
    Raw r;
    load_unit<T, HAS_Z>(p, b, d0 + ch, t0 + seg * kK, r);
    finish_unit<T, Passes, HAS_Z>(p, b, d0 + ch, t0 + seg * kK, seg, r, recs + ch * Passes::size, sums[0][ch][seg],
                                  sums[1][ch][seg]);
  }
  __syncthreads();
  if (tid < width) {
    float x = 0.f, y = 0.f;
#pragma unroll
    for (int seg = 0; seg < kSegs; ++seg) {
      x += sums[0][tid][seg];
      y += sums[1][tid][seg];
    }
    p.pD[bc * p.dim + d0 + tid] = x;
    p.pbias[bc * p.dim + d0 + tid] = y;
  }
}

// ---- sums over groups and chunks -------------------------------------------------------------------
// With more than 16 partials eight threads share a value (every eighth partial each): 5120 or 24 channels in groups of
// 16 would otherwise be one chain of up to 320 loads. With fewer a thread has its own (f16 8x1536x4096 37 us).
template <typename T> __global__ void __launch_bounds__(256) reduce_kernel(const Params p, long long bc_blocks) {
  __shared__ double sum[2][8][32];
  const int lane = threadIdx.x % 32, part = threadIdx.x / 32;
  if (blockIdx.x < bc_blocks) {  // dB and dC: over the groups of channels; a warp is 32 steps of a state
    const int of = p.groups > 16 ? 8 : 1;
    const long long per = (long long)p.chunks * p.passes * kNB;  // rows of 32 steps
    const long long row = (long long)blockIdx.x * (8 / of) + part / of, b = row / per, r = row % per;
    const int n = (int)(r % (p.passes * kNB)), t = (int)(r / (p.passes * kNB)) * kT + lane;
    double x = 0, y = 0;
    if (b < p.batch && n < p.dstate_n) {
#pragma unroll 4
      for (int g = part % of; g < p.groups; g += of) {
        x += p.pB[((b * p.groups + g) * per + r) * kT + lane];
        y += p.pC[((b * p.groups + g) * per + r) * kT + lane];
      }
    }
    if (of > 1) {
      sum[0][part][lane] = x;
      sum[1][part][lane] = y;
      __syncthreads();
      if (part > 0) return;
      for (int k = 1; k < 8; ++k) {
        x += sum[0][k][lane];
        y += sum[1][k][lane];
      }
    }
    if (b >= p.batch || n >= p.dstate_n || t >= p.seqlen) return;
    st_f32(static_cast<T*>(p.dB) + b * p.dBs[0] + n * p.dBs[1] + t * p.dBs[2], (float)x);
    st_f32(static_cast<T*>(p.dC) + b * p.dCs[0] + n * p.dCs[1] + t * p.dCs[2], (float)y);
    return;
  }
  // dA, dD, dbias: over batch and chunks
  const int dn = p.dim * p.np;
  const long long v = ((long long)(blockIdx.x - bc_blocks) * 32) + lane;
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
  if (src) {
#pragma unroll 16
    for (long long r = part; r < rows; r += 8) x += src[r * pitch];
  }
  sum[0][part][lane] = x;
  __syncthreads();
  if (part != 0 || !src) return;
  for (int k = 1; k < 8; ++k) x += sum[0][k][lane];
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
  int passes, groups, tiles, width;
  size_t kst, later, klong, slong, pB, pC, pA, pD, pbias, bytes;
};

int make_layout(const MMScanBwdArgs* a, Layout* l) {
  const MMScanArgs& f = a->fwd;
  const int rc = check_sizes(f);
  if (rc != MM_OK) return rc;
  const int chunks = chunks_of(f), longs = longs_of(f), np = (int)(f.dstate + 3) / 4 * 4;
  l->passes = (int)((f.dstate + kNB - 1) / kNB);
  // Channels of a CTA: as many (fewer partial sums of dB and dC) as leave every one of the 3 x 148 places four CTAs,
  // at most 512, in tiles of 32 (16 for float32, and where 32 would leave places empty).
  const long long rows = f.batch * (chunks > 0 ? chunks : 1), lrows = f.batch * (longs > 0 ? longs : 1);
  const long long want = f.dim * rows / (4 * 3 * 148);
  l->width = (f.dtype == MM_F32 && l->passes == 1) || f.dim * rows < 3 * 148 * 32 ? 16 : 32;
  const long long tiles = want / l->width;
  l->tiles = (int)(l->passes > 1 || tiles < 1 ? 1 : tiles > 512 / l->width ? 512 / l->width : tiles);
  const long long per = (long long)l->width * l->tiles;
  l->groups = (int)((f.dim + per - 1) / per);
  const size_t rowd = (size_t)rows * f.dim, st = rowd * np, lrowd = (size_t)lrows * f.dim;
  const size_t bc = (size_t)rows * l->groups * l->passes * kNB * kT;
  Offsets o;
  l->kst = o.take(chunks > 1 ? st : 0);
  l->later = o.take(chunks > 1 ? rowd : 0);
  l->klong = o.take(chunks > 1 ? lrowd * np : 0);
  l->slong = o.take(chunks > 1 ? lrowd : 0);
  l->pB = o.take(bc);
  l->pC = o.take(bc);
  l->pA = o.take(st);
  l->pD = o.take(rowd);
  l->pbias = o.take(rowd);
  l->bytes = o.at + 256;
  return MM_OK;
}

template <typename T> int reduce(const Params& p, cudaStream_t s) {
  static_assert(kT == 32, "a warp of reduce_kernel is a chunk of a state");
  const long long rows = (long long)p.batch * p.chunks;
  const long long bc = (rows * p.passes * kNB * (p.groups > 16 ? 8 : 1) + 7) / 8;
  const long long rest = ((long long)p.dim * (p.np + 2) + 31) / 32;
  if (bc + rest > 0x7fffffffLL) return MM_ERR_SHAPE;
  reduce_kernel<T><<<(unsigned)(bc + rest), 256, 0, s>>>(p, bc);
  return cudaGetLastError() == cudaSuccess ? MM_OK : MM_ERR_LAUNCH;
}

template <typename T, bool HAS_Z> int launch(const Params& p, int64_t dtype, cudaStream_t s) {
  const long long rows = (long long)p.batch * p.chunks;
  if (rows * p.groups > 0x7fffffffLL) return MM_ERR_SHAPE;
  if (p.chunks > 1) {
    const int rc = walk_back(p, dtype, s);
    if (rc != MM_OK) return rc;
  }
  if (p.passes > 1) {
    if (cudaFuncSetAttribute(grad_wide_kernel<T, HAS_Z>, cudaFuncAttributeMaxDynamicSharedMemorySize, kWideSmem) != cudaSuccess)
      return MM_ERR_LAUNCH;
    grad_wide_kernel<T, HAS_Z><<<(unsigned)(rows * p.groups), kWideThreads, kWideSmem, s>>>(p);
  } else {
    if (cudaFuncSetAttribute(grad_kernel<T, HAS_Z>, cudaFuncAttributeMaxDynamicSharedMemorySize, kGradSmem<T>) != cudaSuccess)
      return MM_ERR_LAUNCH;
    grad_kernel<T, HAS_Z><<<(unsigned)(rows * p.groups), kGradThreads, kGradSmem<T>, s>>>(p);
  }
  return cudaGetLastError() == cudaSuccess ? reduce<T>(p, s) : MM_ERR_LAUNCH;
}

template <typename T> int launch_z(const Params& p, int64_t dtype, cudaStream_t s) {
  if (p.dim == 0) return reduce<T>(p, s);  // dB and dC are sums over no channels
  return p.z ? launch<T, true>(p, dtype, s) : launch<T, false>(p, dtype, s);
}

bool columns_aligned(const void* q, const int64_t* st, const MMScanArgs& f) {
  const int es = dtype_size(f.dtype);
  return aligned16(q) && st[1] == 1 && (f.batch <= 1 || st[0] * es % 16 == 0) && st[2] * es % 16 == 0;
}

}  // namespace train
}  // namespace mm

using namespace mm;
using namespace mm::train;

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
  if (f.dim > 0 && !a->dA) return MM_ERR_ARG;
  if (f.batch == 0 || f.seqlen == 0) {  // sums over nothing
    if (f.dim == 0) return MM_OK;
    if (cudaMemsetAsync(a->dA, 0, sizeof(float) * f.dim * f.dstate, s) != cudaSuccess) return MM_ERR_LAUNCH;
    if (a->dD && cudaMemsetAsync(a->dD, 0, sizeof(float) * f.dim, s) != cudaSuccess) return MM_ERR_LAUNCH;
    if (a->ddelta_bias && cudaMemsetAsync(a->ddelta_bias, 0, sizeof(float) * f.dim, s) != cudaSuccess) return MM_ERR_LAUNCH;
    return MM_OK;
  }
  if (!a->dB || !a->dC) return MM_ERR_ARG;
  if (f.dim > 0 && (!f.u || !f.delta || !f.A || !f.B || !f.C || !a->dy || !a->du || !a->ddelta || (f.z && !a->dz)))
    return MM_ERR_ARG;
  if (!workspace || workspace_bytes < l.bytes || reinterpret_cast<uintptr_t>(workspace) % 256) return MM_ERR_WORKSPACE;
  if (f.dim > 0 && chunks_of(f) > 1 && (!a->states || reinterpret_cast<uintptr_t>(a->states) % 16)) return MM_ERR_ARG;
  Params p = {};
  set_inputs(p, f);
  p.dy = a->dy;
  p.dstate = a->dstate;
  p.du = a->du;
  p.ddelta = a->ddelta;
  p.dz = a->dz;
  p.dB = a->dB;
  p.dC = a->dC;
  p.dA = a->dA;
  p.dD = a->dD;
  p.dbias = a->ddelta_bias;
  copy3(p.ys, a->dy_stride);
  copy3(p.dus, a->du_stride);
  copy3(p.dds, a->ddelta_stride);
  copy3(p.dzs, a->dz_stride);
  copy3(p.dBs, a->dB_stride);
  copy3(p.dCs, a->dC_stride);
  Access access = least(access_of(f.u, f.u_stride, f), access_of(f.delta, f.delta_stride, f));
  access = least(access, least(access_of(a->dy, a->dy_stride, f), access_of(a->du, a->du_stride, f)));
  access = least(access, access_of(a->ddelta, a->ddelta_stride, f));
  if (f.z) access = least(access, least(access_of(f.z, f.z_stride, f), access_of(a->dz, a->dz_stride, f)));
  set_access(p, access, f);
  const void* act[4] = {f.u, f.delta, a->dy, f.z};
  const int64_t* act_stride[4] = {f.u_stride, f.delta_stride, a->dy_stride, f.z_stride};
  p.ahead = 1;
  for (int i = 0; i < (f.z ? 4 : 3); ++i)
    if (!(p.by_channel ? columns_aligned(act[i], act_stride[i], f) : access_of(act[i], act_stride[i], f) == kAligned)) p.ahead = 0;
  p.passes = l.passes;
  p.groups = l.groups;
  p.tiles = l.tiles;
  p.width = l.width;
  char* w = static_cast<char*>(workspace);
  p.hst = const_cast<float*>(a->states);
  p.kst = reinterpret_cast<float*>(w + l.kst);
  p.later = reinterpret_cast<float*>(w + l.later);
  p.klong = reinterpret_cast<float*>(w + l.klong);
  p.slong = reinterpret_cast<float*>(w + l.slong);
  p.pB = reinterpret_cast<float*>(w + l.pB);
  p.pC = reinterpret_cast<float*>(w + l.pC);
  p.pA = reinterpret_cast<float*>(w + l.pA);
  p.pD = reinterpret_cast<float*>(w + l.pD);
  p.pbias = reinterpret_cast<float*>(w + l.pbias);
  switch (f.dtype) {
    case MM_F32: return launch_z<float>(p, f.dtype, s);
    case MM_F16: return launch_z<__half>(p, f.dtype, s);
    default: return launch_z<__nv_bfloat16>(p, f.dtype, s);
  }
}
