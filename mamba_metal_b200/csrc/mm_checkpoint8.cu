// Packing and unpacking of 8-bit activation checkpoints. Memory-bound: a packed value moves its own bytes
// once, one byte of code and 1/32 byte of exponent.
#include "mm_checkpoint8.cuh"

namespace mm {
namespace ck {

struct Params {
  void* x;
  int8_t* codes;
  uint8_t* exps;
  long long xs[3], cs[3], es[3];
  long long rows;
  int dim, length;
};

// Time contiguous: a lane takes 8 consecutive values, so four lanes share a block and agree on its maximum by
// two shuffles. A warp covers CPT * 256 values of one row, with all its loads in flight before the first is used:
// memory is the bound, and bytes in flight decide (bf16 10240 x 32768: packed in 170 us and restored in 163, 1.02 GB
// each way, 6.0 and 6.2 TB/s. Before the codes were made and read without conversion instructions, together: CPT 4
// 370, 2 450, 1 625; blocks of 512 threads 390). Short rows take CPT 1, or half their warps had nothing to do.
// ACCESS: that of x; codes are taken by 8-byte words but for kAnyStride.
template <typename T, bool PACK, int ACCESS, int CPT>
__global__ void __launch_bounds__(256) rows_kernel(const Params p, int warps_per_row) {
  const int lane = threadIdx.x & 31;
  const long long gw = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (gw >= p.rows * warps_per_row) return;
  const long long row = gw / warps_per_row;
  const int begin = (int)(gw % warps_per_row) * CPT * 256 + lane * 8;
  const long long b = row / p.dim, d = row % p.dim;
  T* x = static_cast<T*>(p.x) + b * p.xs[0] + d * p.xs[1];
  int8_t* codes = p.codes + b * p.cs[0] + d * p.cs[1];
  uint8_t* exps = p.exps + b * p.es[0] + d * p.es[1];
  if (PACK) {
    Raw8<T> raw[CPT];
#pragma unroll
    for (int j = 0; j < CPT; ++j) {
      const int t = begin + j * 256;
      raw[j] = raw_load(x + t * p.xs[2], p.xs[2], ACCESS, min(8, p.length - t));
    }
#pragma unroll
    for (int j = 0; j < CPT; ++j) {
      const int t = begin + j * 256, n = min(8, p.length - t);  // values of this lane; none past the row's end
      unsigned m = ck_max_bits(raw[j]);
      m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
      m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
      if (n <= 0) continue;
      const unsigned byte = ck_exponent(m);
      const float inv = ck_inverse_scale(byte);
      if ((lane & 3) == 0) exps[(long long)(t / kCkBlock) * p.es[2]] = (uint8_t)byte;
      unsigned c[8];
#pragma unroll
      for (int k = 0; k < 8; k += 2) {
        const uint2 w = ck_code_pair(f2_pack(raw_at(raw[j], k), raw_at(raw[j], k + 1)), f2_pack(inv, inv));
        c[k] = w.x;
        c[k + 1] = w.y;
      }
      if (ACCESS != kAnyStride && n == 8) {
        __stcs(reinterpret_cast<uint2*>(codes + t), make_uint2(ck_pack4(c[0], c[1], c[2], c[3]), ck_pack4(c[4], c[5], c[6], c[7])));
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (k < n) codes[(t + k) * p.cs[2]] = (int8_t)c[k];
      }
    }
  } else {
    uint2 raw[CPT];
    // one load for the scales of the warp's blocks: the four lanes of a block hold those of its four chunks
    const int first = begin + (lane & 3) * 256;
    unsigned mine = 0;
    if ((lane & 3) < CPT && first - (lane & 3) * 8 < p.length) mine = exps[(long long)(first / kCkBlock) * p.es[2]];
#pragma unroll
    for (int j = 0; j < CPT; ++j) {
      const int t = begin + j * 256;
      if (t >= p.length) continue;
      if (ACCESS != kAnyStride && t + 8 <= p.length) raw[j] = __ldcs(reinterpret_cast<const uint2*>(codes + t));
    }
#pragma unroll
    for (int j = 0; j < CPT; ++j) {
      const int t = begin + j * 256, n = min(8, p.length - t);
      float v[8];
      const unsigned byte = __shfl_sync(0xffffffffu, mine, (lane & ~3) | j);
      const float scale = ck_scale(byte);
      if (ACCESS != kAnyStride && n == 8) {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = ck_value(k < 4 ? raw[j].x : raw[j].y, k & 3) * scale;
        if (!ck_in_range<T>(byte)) {
#pragma unroll
          for (int k = 0; k < 8; ++k) v[k] = ck_restore<T>(v[k], 1.f);
        }
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = k < n ? ck_restore<T>(codes[(t + k) * p.cs[2]], scale) : 0.f;
      }
      if (ACCESS == kAligned && n == 8)
        row_store(x + t, 1, ACCESS, 8, v);
      else
        row_store(x + t * p.xs[2], p.xs[2], ACCESS, n, v);
    }
  }
}

// Channels contiguous: a thread takes one block of one channel, so a warp's accesses run along channels. It keeps
// the block in registers from the maximum to the codes. (bf16 4x5120x5601, 0.35 GB each way: packed in 203 us and restored
// in 289, 1.7 and 1.2 TB/s. Values are loaded one by one, 64 bytes a warp and step in a 16-bit type.)
template <typename T, bool PACK>
__global__ void __launch_bounds__(256) columns_kernel(const Params p, int blocks) {
  const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  const long long batch = p.rows / p.dim;
  if (i >= batch * blocks * p.dim) return;
  const long long d = i % p.dim, k = i / p.dim % blocks, b = i / p.dim / blocks;
  const int t0 = (int)k * kCkBlock, n = min(kCkBlock, p.length - t0);
  T* x = static_cast<T*>(p.x) + b * p.xs[0] + d * p.xs[1] + (long long)t0 * p.xs[2];
  int8_t* codes = p.codes + b * p.cs[0] + d * p.cs[1] + (long long)t0 * p.cs[2];
  uint8_t* exps = p.exps + b * p.es[0] + d * p.es[1] + k * p.es[2];
  if (PACK) {
    T v[kCkBlock];
    unsigned m = 0;
#pragma unroll
    for (int t = 0; t < kCkBlock; ++t) {
      v[t] = t < n ? x[t * p.xs[2]] : ElemTraits<T>::from_f32(0.f);
      m = max(m, ck_abs_bits(ElemTraits<T>::to_f32(v[t])));
    }
    const unsigned byte = ck_exponent(m);
    const float inv = ck_inverse_scale(byte);
    *exps = (uint8_t)byte;
#pragma unroll
    for (int t = 0; t < kCkBlock; ++t)
      if (t < n) codes[t * p.cs[2]] = (int8_t)ck_code(ElemTraits<T>::to_f32(v[t]), inv);
  } else {
    const float scale = ck_scale(*exps);
#pragma unroll 8
    for (int t = 0; t < n; ++t) st_f32(x + t * p.xs[2], ck_restore<T>(codes[t * p.cs[2]], scale));
  }
}

template <typename T, bool PACK> int launch(const MMCheckpoint8Args* a, cudaStream_t s) {
  Params p;
  p.x = a->x;
  p.codes = a->codes;
  p.exps = a->exponents;
  for (int i = 0; i < 3; ++i) {
    p.xs[i] = a->x_stride[i];
    p.cs[i] = a->codes_stride[i];
    p.es[i] = a->exponents_stride[i];
  }
  p.rows = a->batch * a->dim;
  p.dim = (int)a->dim;
  p.length = (int)a->length;
  const bool columns = a->dim > 1 && a->length > 1 && p.xs[1] == 1 && p.cs[1] == 1 && p.xs[2] != 1;
  if (columns) {
    const int blocks = (int)((a->length + kCkBlock - 1) / kCkBlock);
    const long long grid = (p.rows * blocks + 255) / 256;
    if (grid > 0x7fffffffLL) return MM_ERR_SHAPE;
    columns_kernel<T, PACK><<<(unsigned)grid, 256, 0, s>>>(p, blocks);
  } else {
    const bool few = a->length <= 512;  // a warp per row, or half of one, where rows are short
    const int wpr = (int)((a->length + (few ? 255 : 1023)) / (few ? 256 : 1024));
    const long long grid = (p.rows * wpr + 7) / 8;
    if (grid > 0x7fffffffLL) return MM_ERR_SHAPE;
    Access access = ck_access(a->x, a->x_stride, a->batch, a->dim, a->length, (int)sizeof(T));
    if ((a->length > 1 && p.cs[2] != 1) || !ck_rows_aligned(a->codes, a->codes_stride, a->batch, a->dim, 1, 8)) access = kAnyStride;
    switch (access) {
      case kAligned:
        few ? rows_kernel<T, PACK, kAligned, 1><<<(unsigned)grid, 256, 0, s>>>(p, wpr)
            : rows_kernel<T, PACK, kAligned, 4><<<(unsigned)grid, 256, 0, s>>>(p, wpr);
        break;
      case kContiguous:
        few ? rows_kernel<T, PACK, kContiguous, 1><<<(unsigned)grid, 256, 0, s>>>(p, wpr)
            : rows_kernel<T, PACK, kContiguous, 4><<<(unsigned)grid, 256, 0, s>>>(p, wpr);
        break;
      default:
        few ? rows_kernel<T, PACK, kAnyStride, 1><<<(unsigned)grid, 256, 0, s>>>(p, wpr)
            : rows_kernel<T, PACK, kAnyStride, 4><<<(unsigned)grid, 256, 0, s>>>(p, wpr);
    }
  }
  return cudaGetLastError() == cudaSuccess ? MM_OK : MM_ERR_LAUNCH;
}

template <bool PACK> int dispatch(const MMCheckpoint8Args* a, mm_stream_t stream) {
  if (!a) return MM_ERR_ARG;
  if (!dtype_size(a->dtype)) return MM_ERR_DTYPE;
  if (a->batch < 0 || a->dim < 0 || a->length < 0 || a->dim > 0x7fffffffLL || a->length > 0x7fffffffLL - 2048)
    return MM_ERR_SHAPE;
  if (a->batch == 0 || a->dim == 0 || a->length == 0) return MM_OK;
  if (!a->x || !a->codes || !a->exponents) return MM_ERR_ARG;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (a->dtype) {
    case MM_F32: return launch<float, PACK>(a, s);
    case MM_F16: return launch<__half, PACK>(a, s);
    default: return launch<__nv_bfloat16, PACK>(a, s);
  }
}

}  // namespace ck
}  // namespace mm

extern "C" int mm_checkpoint8_pack(const MMCheckpoint8Args* a, mm_stream_t stream) {
  return mm::ck::dispatch<true>(a, stream);
}
extern "C" int mm_checkpoint8_unpack(const MMCheckpoint8Args* a, mm_stream_t stream) {
  return mm::ck::dispatch<false>(a, stream);
}
