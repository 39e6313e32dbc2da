// The walks of mm_scan_walk.cu over whole sequences: time is not cut, so no step is walked twice and nothing is joined.
// Forward y and h at the start of every 32 steps, back (from zero) k at the end of them.
//
// Four lanes share a channel, a quarter of the states each, so a block of four warps takes 32 channels. A tile is a
// chunk of 32 steps: d, d u or e, B and C go through shared memory, one buffer being filled while the other is worked
// on, and the next tile's raw values arrive in registers meanwhile; one barrier a tile.
//
// With one block on an SM a step takes 75 ns, some 40 instructions of which few are independent; two blocks take 97,
// three 119 (f16 8x1536x4096: 0.49 ms, the three launches over cut time 0.76). Taken where that is the shorter way.
#include "mm_scan_train.cuh"

namespace mm {
namespace train {

namespace {
constexpr int kCh = 32, kThreads = 128;
constexpr int kPairs = kT * kCh + 4 * kSegs;  // (d, d u or e) of a tile
constexpr int kPitchY = kCh + 8, kOuts = kT * kPitchY + 8 * kSegs;
// Segments of eight steps are shifted against each other so that units' accesses fall into different banks
MM_DEV int pair_at(int t, int ch) { return t * kCh + t / kK * 4 + ch; }
MM_DEV int out_at(int t, int ch) { return t * kPitchY + t / kK * 8 + ch; }
template <bool BACK, int S> constexpr int kSmem =
    2 * (kPairs * 8 + (BACK ? 1 : 2) * kT * 4 * S * 4 + (BACK ? 0 : kOuts * 4));

template <int N> MM_DEV void read_states(const float* x, f2_t (&v)[N]) {
  if constexpr (N == 1) {
    v[0] = *reinterpret_cast<const f2_t*>(x);
  } else {
#pragma unroll
    for (int m = 0; m < N; m += 2) {
      const ulonglong2 w = *reinterpret_cast<const ulonglong2*>(x + 2 * m);
      v[m] = w.x;
      v[m + 1] = w.y;
    }
  }
}

template <typename T> MM_DEV T zero_of() { return T(); }
template <> MM_DEV __half zero_of<__half>() { return __ushort_as_half(0); }
template <> MM_DEV __nv_bfloat16 zero_of<__nv_bfloat16>() { return __ushort_as_bfloat16(0); }
// Four states' B or C of a step as they lie in memory
template <typename T> struct Quad {
  T v[4];
};
template <typename T> MM_DEV Quad<T> load_quad(const void* base, const long long (&st)[3], int b, int n0, int t, const Params& p) {
  const T* q = static_cast<const T*>(base) + b * st[0] + n0 * st[1] + t * st[2];
  const int n = t < p.seqlen ? p.dstate_n - n0 : 0;
  Quad<T> r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r.v[i] = n > i ? q[i * st[1]] : zero_of<T>();
  return r;
}
template <typename T> MM_DEV float4 floats_of(const Quad<T>& r) {
  return f4(ld_f32(&r.v[0]), ld_f32(&r.v[1]), ld_f32(&r.v[2]), ld_f32(&r.v[3]));
}
}  // namespace

// S: states of a lane
template <bool BACK, typename T, int S> __global__ void __launch_bounds__(kThreads, 3) rows_kernel(const Params p) {
  constexpr int NM = 4 * S;
  extern __shared__ float4 smem4[];
  float* sB = reinterpret_cast<float*>(smem4);  // [2][step][state]: B, or C back
  float* sC = sB + 2 * kT * NM;
  float2* sx = reinterpret_cast<float2*>(sC + (BACK ? 0 : 2 * kT * NM));
  float* sy = reinterpret_cast<float*>(sx + 2 * kPairs);
  const int tid = threadIdx.x, q = tid & 3, c = tid >> 2;  // the thread's states, from q S on, of channel c
  const int groups = (p.dim + kCh - 1) / kCh;
  const int d0 = (int)(blockIdx.x % groups) * kCh, b = (int)(blockIdx.x / groups), d = d0 + c;
  const bool mine = d < p.dim;
  int uch, useg;  // the thread's unit of a tile
  unit_of<kCh>(tid, p.by_channel, uch, useg);
  const bool unit = d0 + uch < p.dim;
  const f2_t bias = dup(p.bias && unit ? p.bias[d0 + uch] : 0.f), D = dup(!BACK && p.D && unit ? p.D[d0 + uch] : 0.f);
  // and its part of B and C: four states of a step; threads run along whichever of time and states is contiguous
  // (f16 8x1536x4096, channels contiguous: along time 0.89 ms, along states 0.86)
  constexpr int Q = NM / 4;
  const bool across = p.Cs[1] == 1, brings = tid < kT * Q;
  const int tq = across ? tid / Q : tid % kT, n0 = 4 * (across ? tid % Q : tid / kT);

  f2_t A[S / 2], h[S / 2];
#pragma unroll
  for (int j = 0; j < S / 2; ++j) {
    float v[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int n = q * S + 2 * j + i;
      v[i] = mine && n < p.dstate_n ? p.A[d * p.As[0] + n * p.As[1]] * kLog2e : 0.f;
    }
    A[j] = f2_pack(v[0], v[1]);
    h[j] = dup(0.f);
  }

  float sum = 0.f;      // back: of d
  Raw8<T> raw, xs, zs;  // of the tile to come: delta, u or dy, z
  Quad<T> Bq, Cq;
  auto fetch = [&](const void* base, const long long (&st)[3], int t0) {
    const int t = t0 + useg * kK, n = unit ? min(kK, p.seqlen - t) : 0;
    return raw_load(static_cast<const T*>(base) + b * st[0] + (d0 + uch) * st[1] + t * st[2], st[2], p.access, n);
  };
  auto load = [&](int t0) {
    raw = fetch(p.delta, p.ds, t0);
    xs = BACK ? fetch(p.dy, p.ys, t0) : fetch(p.u, p.us, t0);
    if (p.z && (BACK || p.y)) zs = fetch(p.z, p.zs, t0);
    if (brings) {
      Bq = BACK ? load_quad<T>(p.C, p.Cs, b, n0, t0 + tq, p) : load_quad<T>(p.B, p.Bs, b, n0, t0 + tq, p);
      if (!BACK) Cq = load_quad<T>(p.C, p.Cs, b, n0, t0 + tq, p);
    }
  };
  // zeros where there are no steps or channels: a = 1 there, and nothing is added
  auto stage = [&](int t0, int buf) {
    const int n = unit ? min(kK, p.seqlen - (t0 + useg * kK)) : 0;
    float2* to = sx + buf * kPairs + pair_at(useg * kK, uch);
#pragma unroll
    for (int k = 0; k < kK; k += 2) {
      float2 dt = f2_unpack(step_of(f2_add(f2_pack(raw_at(raw, k), raw_at(raw, k + 1)), bias), p.softplus));
      dt.x = k < n ? dt.x : 0.f;
      dt.y = k + 1 < n ? dt.y : 0.f;
      f2_t v = f2_pack(raw_at(xs, k), raw_at(xs, k + 1));
      if (!BACK)
        v = f2_mul(v, f2_pack(dt.x, dt.y));
      else if (p.z)
        v = f2_mul(v, silu_of(f2_pack(raw_at(zs, k), raw_at(zs, k + 1))));
      const float2 w = f2_unpack(v);
      to[k * kCh] = make_float2(dt.x, w.x);
      to[(k + 1) * kCh] = make_float2(dt.y, w.y);
    }
    if (brings) {
      *reinterpret_cast<float4*>(sB + (buf * kT + tq) * NM + n0) = floats_of(Bq);
      if (!BACK) *reinterpret_cast<float4*>(sC + (buf * kT + tq) * NM + n0) = floats_of(Cq);
    }
  };

  auto start = [&](int i) { return (BACK ? p.chunks - 1 - i : i) * kT; };
  load(start(0));
  stage(start(0), 0);
  __syncthreads();
  for (int i = 0; i < p.chunks; ++i) {
    const int t0 = start(i), buf = i & 1;
    const Raw8<T> u = xs, z = zs;
    if (i + 1 < p.chunks) load(start(i + 1));
    const long long row = ((long long)b * p.chunks + t0 / kT) * p.dim + d;
    if (BACK && mine && q == 0) p.later[row] = sum;
    if (mine && (BACK || p.hst)) {
      float* to = (BACK ? p.kst : p.hst) + row * p.np + q * S;
#pragma unroll
      for (int j = 0; j < S / 2; ++j)
        if (q * S + 2 * j < p.np) *reinterpret_cast<float2*>(to + 2 * j) = f2_unpack(h[j]);
    }
    float* out = sy + buf * kOuts;
#pragma unroll 1
    for (int g = 0; g < kSegs; ++g) {
      const int t8 = (BACK ? kSegs - 1 - g : g) * kK;
      const float2* x = sx + buf * kPairs + pair_at(t8, c);
      const float *Bt = sB + (buf * kT + t8) * NM + q * S, *Ct = sC + (buf * kT + t8) * NM + q * S;
#pragma unroll
      for (int j = 0; j < kK; j += 4) {
        float y[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int t = BACK ? kK - 1 - (j + k) : j + k;
          const float2 v = x[t * kCh];
          const f2_t dt2 = dup(v.x), x2 = dup(v.y);
          f2_t Bv[S / 2], Cv[S / 2], acc = dup(0.f);
          read_states(Bt + t * NM, Bv);
          if (BACK)
            sum += v.x;
          else
            read_states(Ct + t * NM, Cv);
#pragma unroll
          for (int m = 0; m < S / 2; ++m) {
            const f2_t a = ex2_pair(f2_mul(A[m], dt2));
            if (BACK) {
              h[m] = f2_mul(a, f2_fma(Bv[m], x2, h[m]));
            } else {
              h[m] = f2_fma(a, h[m], f2_mul(Bv[m], x2));
              acc = f2_fma(h[m], Cv[m], acc);
            }
          }
          const float2 w = f2_unpack(acc);
          y[k] = w.x + w.y;
        }
        if (!BACK) {  // over the channel's four lanes, which are left with one step each
          const bool one = q & 1, two = q & 2;
          const float r0 = (one ? y[2] : y[0]) + __shfl_xor_sync(0xffffffffu, one ? y[0] : y[2], 1);
          const float r1 = (one ? y[3] : y[1]) + __shfl_xor_sync(0xffffffffu, one ? y[1] : y[3], 1);
          out[out_at(t8, c) + (j + 2 * one + two) * kPitchY] =
              (two ? r1 : r0) + __shfl_xor_sync(0xffffffffu, two ? r0 : r1, 2);
        }
      }
    }
    if (i + 1 < p.chunks) stage(start(i + 1), buf ^ 1);
    __syncthreads();
    if (!BACK && p.y && unit) {
      const int t = t0 + useg * kK, n = min(kK, p.seqlen - t), dc = d0 + uch;
      const float* from = out + out_at(useg * kK, uch);
      float v[kK];
#pragma unroll
      for (int k = 0; k < kK; k += 2) {
        f2_t w = f2_fma(D, f2_pack(raw_at(u, k), raw_at(u, k + 1)), f2_pack(from[k * kPitchY], from[(k + 1) * kPitchY]));
        if (p.z) w = f2_mul(w, silu_of(f2_pack(raw_at(z, k), raw_at(z, k + 1))));
        const float2 r = f2_unpack(w);
        v[k] = r.x;
        v[k + 1] = r.y;
      }
      store_steps(static_cast<T*>(p.y) + b * p.ys[0] + dc * p.ys[1] + t * p.ys[2], p.ys[2], p.access, n, v);
    }
  }
  if (!BACK && p.state_out && mine) {
    float* to = p.state_out + ((long long)b * p.dim + d) * p.dstate_n;
#pragma unroll
    for (int j = 0; j < S / 2; ++j) {
      const float2 v = f2_unpack(h[j]);
      const int n = q * S + 2 * j;
      if (n < p.dstate_n) to[n] = v.x;
      if (n + 1 < p.dstate_n) to[n + 1] = v.y;
    }
  }
}

template <bool BACK, typename T, int S> int launch_rows(const Params& p, cudaStream_t s) {
  const long long grid = (long long)p.batch * ((p.dim + kCh - 1) / kCh);
  if (grid > 0x7fffffffLL) return MM_ERR_SHAPE;
  constexpr int smem = kSmem<BACK, S>;
  if (smem > 48 * 1024 &&
      cudaFuncSetAttribute(rows_kernel<BACK, T, S>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
    return MM_ERR_LAUNCH;
  rows_kernel<BACK, T, S><<<(unsigned)grid, kThreads, smem, s>>>(p);
  return cudaGetLastError() == cudaSuccess ? MM_OK : MM_ERR_LAUNCH;
}
template <bool BACK, typename T> int rows_of(const Params& p, cudaStream_t s) {
  return p.dstate_n <= 8 ? launch_rows<BACK, T, 2>(p, s) : launch_rows<BACK, T, 4>(p, s);
}
template <bool BACK> int walk_rows(const Params& p, int64_t dtype, cudaStream_t s) {
  switch (dtype) {
    case MM_F32: return rows_of<BACK, float>(p, s);
    case MM_F16: return rows_of<BACK, __half>(p, s);
    default: return rows_of<BACK, __nv_bfloat16>(p, s);
  }
}
template int walk_rows<false>(const Params&, int64_t, cudaStream_t);
template int walk_rows<true>(const Params&, int64_t, cudaStream_t);

}  // namespace train
}  // namespace mm
