// The parts of the selective scan's training kernels that run through time: the forward pass, and the gradient's
// reverse recurrence.
//
// Time is cut into long chunks of up to 128 steps. A warp takes 32 channels (a lane each, all its states in registers)
// of one long chunk and walks its steps:
//   kState: from zero, what the chunk adds to the state that comes into it;
//   kOut:   from the state that comes into it, y, and h at the start of every 32 steps (what the gradient needs);
//   kBack:  in reverse from zero, k_{t-1} = a_t (C_t e_t + k_t), and k at the end of every 32 steps.
// Between kState and kOut, and after kBack, join_kernel runs over the long chunks in order: exp(A sum d) is a
// chunk's decay. d, d u and e are computed once per element by the lane that loads it and pass through shared
// memory as [step][channel]; warps share nothing, so no block barriers.
//
// Bound by the MUFU (one ex2 for each state and step, 16 per clock and SM: 805 M, 0.18 ms at 1.9 GHz for a walk of
// 8x1536x4096 with 16 states) and close behind by the registers' way in from shared memory, 128 bytes per clock: a
// step's B and C arrive as 32 lanes x 128 bytes. Measured there, f16: kState 0.28 ms, kOut 0.45, kBack 0.31, with
// four blocks of four warps on an SM (five and six spill: kOut 0.50 and 0.58); tiles of 32 steps 0.32, 0.55, 0.39;
// two channels a lane, which share B and C but leave 12 warps, 0.30, 0.53, 0.48. The forward pass now walks that size
// whole (mm_scan_rows.cu); f32 1x1536x5601 (31 us of MUFU): 63, 92 and 71 us.
#include "mm_scan_train.cuh"

namespace mm {
namespace train {

enum Walk { kState, kOut, kBack };
constexpr int kWarps = 4;
constexpr int kSub = 16;  // steps staged at a time

constexpr int kTile = kSub * 33;
template <int MODE, int NM> constexpr int kWarpFloats = 2 * kTile + (MODE == kOut ? 2 : 1) * kSub * NM;

// B or C of a tile's steps as [step][state]; lanes l and l + 16 share a step
template <typename T, int NM>
MM_DEV void stage_states(const void* base, const long long (&st)[3], const Params& p, int b, int t0, int lane, float* out) {
#pragma unroll 4
  for (int j = lane / kSub; j < NM / 4; j += 2)
    *reinterpret_cast<float4*>(out + lane % kSub * NM + 4 * j) =
        load_BC(static_cast<const T*>(base), st, b, 4 * j, t0 + lane % kSub, p);
}

template <int MODE, typename T, int NM>
__global__ void __launch_bounds__(kWarps * 32, NM <= 16 ? 4 : NM <= 32 ? 3 : 2) walk_kernel(const Params p) {
  constexpr int PITCH = 33, UNITS = kSub / kK;
  extern __shared__ float4 smem4[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float* sB = reinterpret_cast<float*>(smem4) + warp * ((kWarpFloats<MODE, NM> + 3) / 4 * 4);  // B, or C
  float* sC = sB + kSub * NM;
  float* sd = sC + (MODE == kOut ? kSub * NM : 0);
  float* sx = sd + kTile;  // d u (then y without D u and the gate), or e
  const int groups = (p.dim + 31) / 32;
  const long long item = (long long)blockIdx.x * kWarps + warp;
  if (item >= (long long)p.batch * p.longs * groups) return;
  const int d0 = (int)(item % groups) * 32, d = d0 + lane;
  const long long bl = item / groups;
  const int l = (int)(bl % p.longs), b = (int)(bl / p.longs);
  const int begin = l * p.per_long * kT, end = min(p.seqlen, begin + p.per_long * kT);

  const bool mine = d < p.dim;

  f2_t A[NM / 2], h[NM / 2];
  float sum = 0.f;
#pragma unroll
  for (int j = 0; j < NM / 4; ++j) {
    const float4 a = mine ? load_A(p, d, 4 * j) : f4(0.f, 0.f, 0.f, 0.f);
    A[2 * j] = mul1(f2_pack(a.x, a.y), kLog2e);
    A[2 * j + 1] = mul1(f2_pack(a.z, a.w), kLog2e);
    float4 x = f4(0.f, 0.f, 0.f, 0.f);
    if (MODE == kOut && p.longs > 1 && mine && 4 * j < p.np)
      x = *reinterpret_cast<const float4*>(p.hlong + (bl * p.dim + d) * p.np + 4 * j);
    h[2 * j] = f2_pack(x.x, x.y);
    h[2 * j + 1] = f2_pack(x.z, x.w);
  }
  // the lane's states to their row of `to`, (.., dim, np)
  auto put = [&](float* to, long long row) {
    if (!mine) return;
#pragma unroll
    for (int j = 0; j < NM / 4; ++j)
      if (4 * j < p.np) {
        const float2 x = f2_unpack(h[2 * j]), y = f2_unpack(h[2 * j + 1]);
        *reinterpret_cast<float4*>(to + (row * p.dim + d) * p.np + 4 * j) = f4(x.x, x.y, y.x, y.y);
      }
  };

  const int tiles = (end - begin + kSub - 1) / kSub;
  for (int i = 0; i < tiles; ++i) {
    const int t0 = begin + (MODE == kBack ? tiles - 1 - i : i) * kSub;
    __syncwarp();
    Raw8<T> raw[UNITS], x[UNITS], z[UNITS];  // delta; u or dy; z: all loads in flight together
    auto fetch = [&](const void* base, const long long (&st)[3], Raw8<T>(&r)[UNITS]) {
#pragma unroll
      for (int j = 0; j < UNITS; ++j) {
        int ch, seg;
        unit_of<32, kSub / kK>(lane + 32 * j, p.by_channel, ch, seg);
        const int t = t0 + seg * kK, n = d0 + ch < p.dim ? min(kK, p.seqlen - t) : 0;
        r[j] = raw_load(static_cast<const T*>(base) + b * st[0] + (d0 + ch) * st[1] + t * st[2], st[2], p.access, n);
      }
    };
    fetch(p.delta, p.ds, raw);
    if (MODE == kBack) {
      fetch(p.dy, p.ys, x);
      if (p.z) fetch(p.z, p.zs, z);
    } else {
      fetch(p.u, p.us, x);
    }
    if (MODE != kBack) stage_states<T, NM>(p.B, p.Bs, p, b, t0, lane, sB);
    if (MODE == kOut) stage_states<T, NM>(p.C, p.Cs, p, b, t0, lane, sC);
    if (MODE == kBack) stage_states<T, NM>(p.C, p.Cs, p, b, t0, lane, sB);
    // d and d u or e; zeros where there are no steps or channels: a = 1 there, and nothing is added
#pragma unroll
    for (int j = 0; j < UNITS; ++j) {
      int ch, seg;
      unit_of<32, kSub / kK>(lane + 32 * j, p.by_channel, ch, seg);
      const int t = t0 + seg * kK, n = d0 + ch < p.dim ? min(kK, p.seqlen - t) : 0;
      const f2_t bias = dup(p.bias && d0 + ch < p.dim ? p.bias[d0 + ch] : 0.f);
#pragma unroll
      for (int k = 0; k < kK; k += 2) {
        float2 dt = f2_unpack(step_of(f2_add(f2_pack(raw_at(raw[j], k), raw_at(raw[j], k + 1)), bias), p.softplus));
        dt.x = k < n ? dt.x : 0.f;
        dt.y = k + 1 < n ? dt.y : 0.f;
        f2_t v = f2_pack(raw_at(x[j], k), raw_at(x[j], k + 1));
        if (MODE != kBack)
          v = f2_mul(v, f2_pack(dt.x, dt.y));
        else if (p.z)
          v = f2_mul(v, silu_of(f2_pack(raw_at(z[j], k), raw_at(z[j], k + 1))));
        const float2 w = f2_unpack(v);
        const int at = (seg * kK + k) * PITCH + ch;
        sd[at] = dt.x;
        sd[at + PITCH] = dt.y;
        sx[at] = w.x;
        sx[at + PITCH] = w.y;
      }
    }
    const long long bc = (long long)b * p.chunks + t0 / kT;
    if (MODE == kOut && p.hst && t0 % kT == 0) put(p.hst, bc);
    if (MODE == kBack && (t0 % kT == kT - kSub || i == 0)) {  // the chunk's last tile that has steps
      put(p.kst, bc);
      if (mine) p.later[bc * p.dim + d] = sum;
    }
    __syncwarp();
#pragma unroll 2
    for (int j = 0; j < kSub; ++j) {
      const int t = MODE == kBack ? kSub - 1 - j : j;
      const ulonglong2* Bt = reinterpret_cast<const ulonglong2*>(sB + t * NM);
      const ulonglong2* Ct = reinterpret_cast<const ulonglong2*>(sC + t * NM);
      const float dt = sd[t * PITCH + lane];
      sum += dt;
      const f2_t dt2 = dup(dt), x2 = dup(sx[t * PITCH + lane]);
      f2_t y0 = dup(0.f), y1 = y0;
#pragma unroll
      for (int k = 0; k < NM / 4; ++k) {
        const ulonglong2 Bv = Bt[k];
        f2_t &h0 = h[2 * k], &h1 = h[2 * k + 1];
        const f2_t a0 = ex2_pair(f2_mul(A[2 * k], dt2)), a1 = ex2_pair(f2_mul(A[2 * k + 1], dt2));
        if (MODE == kBack) {
          h0 = f2_mul(a0, f2_fma(Bv.x, x2, h0));
          h1 = f2_mul(a1, f2_fma(Bv.y, x2, h1));
        } else {
          h0 = f2_fma(a0, h0, f2_mul(Bv.x, x2));
          h1 = f2_fma(a1, h1, f2_mul(Bv.y, x2));
        }
        if (MODE == kOut) {
          const ulonglong2 Cv = Ct[k];
          y0 = f2_fma(h0, Cv.x, y0);
          y1 = f2_fma(h1, Cv.y, y1);
        }
      }
      if (MODE == kOut) {
        const float2 w = f2_unpack(f2_add(y0, y1));
        sx[t * PITCH + lane] = w.x + w.y;
      }
    }
    if (MODE == kOut && p.y) {
      fetch(p.u, p.us, x);
      if (p.z) fetch(p.z, p.zs, z);
      __syncwarp();
#pragma unroll
      for (int j = 0; j < UNITS; ++j) {
        int ch, seg;
        unit_of<32, kSub / kK>(lane + 32 * j, p.by_channel, ch, seg);
        if (d0 + ch >= p.dim) continue;
        const int t = t0 + seg * kK, n = min(kK, p.seqlen - t), dc = d0 + ch;
        float out[kK];
        const f2_t D = dup(p.D ? p.D[dc] : 0.f);
#pragma unroll
        for (int k = 0; k < kK; k += 2) {
          const int at = (seg * kK + k) * PITCH + ch;
          f2_t v = f2_fma(D, f2_pack(raw_at(x[j], k), raw_at(x[j], k + 1)), f2_pack(sx[at], sx[at + PITCH]));
          if (p.z) v = f2_mul(v, silu_of(f2_pack(raw_at(z[j], k), raw_at(z[j], k + 1))));
          const float2 w = f2_unpack(v);
          out[k] = w.x;
          out[k + 1] = w.y;
        }
        store_steps(static_cast<T*>(p.y) + b * p.ys[0] + dc * p.ys[1] + t * p.ys[2], p.ys[2], p.access, n, out);
      }
    }
  }
  if (MODE == kState) put(p.hlong, bl);
  if (MODE == kBack) put(p.klong, bl);
  if (!mine) return;
  if (MODE != kOut) p.slong[bl * p.dim + d] = sum;
  if (MODE == kOut && p.state_out && l == p.longs - 1) {
    float* out = p.state_out + ((long long)b * p.dim + d) * p.dstate_n;
#pragma unroll
    for (int j = 0; j < NM / 2; ++j) {
      const float2 x = f2_unpack(h[j]);
      if (2 * j < p.dstate_n) out[2 * j] = x.x;
      if (2 * j + 1 < p.dstate_n) out[2 * j + 1] = x.y;
    }
  }
}

// A thread per state replaces, long chunk by long chunk, what it adds by what comes into it.
template <bool BACK> __global__ void __launch_bounds__(128) join_kernel(const Params p) {
  const long long per = (long long)p.dim * p.np;
  const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= p.batch * per) return;
  const long long b = i / per, dn = i % per;
  const int d = (int)(dn / p.np), n = (int)(dn % p.np);
  const float A = n < p.dstate_n ? p.A[d * p.As[0] + n * p.As[1]] * kLog2e : 0.f;
  float* st = (BACK ? p.klong : p.hlong) + b * p.longs * per + dn;
  const float* sum = p.slong + b * p.longs * p.dim + d;
  float v = BACK && p.dstate && n < p.dstate_n ? p.dstate[(b * p.dim + d) * p.dstate_n + n] : 0.f;
  constexpr int kU = 8;  // long chunks whose values are loaded before the first is needed
  for (int c0 = 0; c0 < p.longs; c0 += kU) {
    float own[kU], s[kU];
#pragma unroll
    for (int j = 0; j < kU; ++j) {
      if (c0 + j >= p.longs) break;
      const long long c = BACK ? p.longs - 1 - (c0 + j) : c0 + j;
      own[j] = st[c * per];
      s[j] = sum[c * p.dim];
    }
#pragma unroll
    for (int j = 0; j < kU; ++j) {
      if (c0 + j >= p.longs) break;
      const long long c = BACK ? p.longs - 1 - (c0 + j) : c0 + j;
      st[c * per] = v;
      v = fmaf(ex2(s[j] * A), v, own[j]);
    }
  }
}

// ---- host ---------------------------------------------------------------------------------------------
template <int MODE, typename T, int NM> int launch_walk(const Params& p, cudaStream_t s) {
  const long long items = (long long)p.batch * p.longs * ((p.dim + 31) / 32), grid = (items + kWarps - 1) / kWarps;
  if (grid > 0x7fffffffLL) return MM_ERR_SHAPE;
  constexpr int smem = kWarps * ((kWarpFloats<MODE, NM> + 3) / 4 * 4) * (int)sizeof(float);
  if (smem > 48 * 1024 &&
      cudaFuncSetAttribute(walk_kernel<MODE, T, NM>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
    return MM_ERR_LAUNCH;
  walk_kernel<MODE, T, NM><<<(unsigned)grid, kWarps * 32, smem, s>>>(p);
  return cudaGetLastError() == cudaSuccess ? MM_OK : MM_ERR_LAUNCH;
}
template <int MODE, typename T> int launch_states(const Params& p, cudaStream_t s) {
  if (p.dstate_n <= 8) return launch_walk<MODE, T, 8>(p, s);
  if (p.dstate_n <= 16) return launch_walk<MODE, T, 16>(p, s);
  if (p.dstate_n <= 32) return launch_walk<MODE, T, 32>(p, s);
  return launch_walk<MODE, T, 64>(p, s);
}
template <int MODE> int walk(const Params& p, int64_t dtype, cudaStream_t s) {
  switch (dtype) {
    case MM_F32: return launch_states<MODE, float>(p, s);
    case MM_F16: return launch_states<MODE, __half>(p, s);
    default: return launch_states<MODE, __nv_bfloat16>(p, s);
  }
}
template <bool BACK> int join(const Params& p, cudaStream_t s) {
  const long long states = (long long)p.batch * p.dim * p.np, grid = (states + 127) / 128;
  if (grid > 0x7fffffffLL) return MM_ERR_SHAPE;
  join_kernel<BACK><<<(unsigned)grid, 128, 0, s>>>(p);
  return cudaGetLastError() == cudaSuccess ? MM_OK : MM_ERR_LAUNCH;
}

int walk_back(const Params& p, int64_t dtype, cudaStream_t s) {
  if (p.whole) return walk_rows<true>(p, dtype, s);
  const int rc = walk<kBack>(p, dtype, s);
  return rc == MM_OK && p.longs > 1 ? join<true>(p, s) : rc;
}

namespace {
// Longer sequences are walked whole where that leaves an SM two blocks of 32 channels or nearly: f16 8x1536x4096 0.49
// ms, cut 0.76; 1x8192x4096 0.38 and 0.50; 1x5120x4096 0.38 and 0.33.
bool forward_whole(const MMScanArgs& f) {
  return walked_whole(f) || (f.dstate <= 16 && f.batch * f.dim >= 8192);
}
struct Layout {
  size_t hlong, slong, bytes;
};
int make_layout(const MMScanArgs* a, Layout* l) {
  if (!a) return MM_ERR_ARG;
  const int rc = check_sizes(*a);
  if (rc != MM_OK) return rc;
  const size_t n = longs_of(*a) > 1 && !forward_whole(*a) ? (size_t)a->batch * longs_of(*a) * a->dim : 0;
  Offsets o;
  l->hlong = o.take(n * ((a->dstate + 3) / 4 * 4));
  l->slong = o.take(n);
  l->bytes = o.at;
  return MM_OK;
}
}  // namespace

}  // namespace train
}  // namespace mm

using namespace mm;
using namespace mm::train;

extern "C" int mm_selective_scan_states_size(const MMScanArgs* a, size_t* bytes) {
  if (!a || !bytes) return MM_ERR_ARG;
  const int rc = check_sizes(*a);
  if (rc != MM_OK) return rc;
  *bytes = chunks_of(*a) > 1 ? (size_t)a->batch * chunks_of(*a) * a->dim * ((a->dstate + 3) / 4 * 4) * sizeof(float) : 0;
  return MM_OK;
}

extern "C" int mm_selective_scan_train_workspace_size(const MMScanArgs* a, size_t* bytes) {
  Layout l;
  const int rc = make_layout(a, &l);
  if (rc != MM_OK) return rc;
  if (!bytes) return MM_ERR_ARG;
  *bytes = l.bytes;
  return MM_OK;
}

extern "C" int mm_selective_scan_train_fwd(const MMScanArgs* a, float* states, void* workspace, size_t workspace_bytes,
                                           mm_stream_t stream) {
  Layout l;
  int rc = make_layout(a, &l);
  if (rc != MM_OK) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (a->batch == 0 || a->dim == 0) return MM_OK;
  if (a->seqlen == 0) {  // no steps leave the state at zero
    if (a->state_out && cudaMemsetAsync(a->state_out, 0, sizeof(float) * a->batch * a->dim * a->dstate, s) != cudaSuccess)
      return MM_ERR_LAUNCH;
    return MM_OK;
  }
  if (!a->u || !a->delta || !a->A || !a->B || !a->C) return MM_ERR_ARG;
  if (chunks_of(*a) > 1 && (!states || reinterpret_cast<uintptr_t>(states) % 16)) return MM_ERR_ARG;
  if (l.bytes && (!workspace || workspace_bytes < l.bytes || reinterpret_cast<uintptr_t>(workspace) % 256))
    return MM_ERR_WORKSPACE;
  Params p = {};
  set_inputs(p, *a);
  p.y = a->y;
  p.state_out = a->state_out;
  copy3(p.ys, a->y_stride);
  Access access = least(access_of(a->u, a->u_stride, *a), access_of(a->delta, a->delta_stride, *a));
  if (a->y) access = least(access, access_of(a->y, a->y_stride, *a));
  if (a->z) access = least(access, access_of(a->z, a->z_stride, *a));
  set_access(p, access, *a);
  p.hst = p.chunks > 1 ? states : nullptr;
  p.hlong = reinterpret_cast<float*>(static_cast<char*>(workspace) + l.hlong);
  p.slong = reinterpret_cast<float*>(static_cast<char*>(workspace) + l.slong);
  if (forward_whole(*a)) return walk_rows<false>(p, a->dtype, s);
  if (p.longs > 1) {
    rc = walk<kState>(p, a->dtype, s);
    if (rc == MM_OK) rc = join<false>(p, s);
    if (rc != MM_OK) return rc;
  }
  return walk<kOut>(p, a->dtype, s);
}
