// Shared by the two attention kernels: arguments, the list of work, dequantised operands, and the kernel that joins the pieces of
// units that several CTAs have worked on.
#pragma once
#include "kernels.cuh"
#include "kv_cache.cuh"
#include "tensor_memory.cuh"

namespace padra {
namespace attention {

constexpr float kNever = -1e30f; // the running maximum before any token
constexpr float kTop = 8.f, kRaise = 15.f; // log2 of the largest weight after a raise / before the next
constexpr float kLeastFactor = 0x1p-126f, kLargestFactor = 0x1p64f; // of scores: see FactorOf
constexpr float kLargestTop = 0x1p24f; // the largest magnitude of a running maximum, in log2: beyond it weights next to each other are
                                       // more than a factor of two apart, and soon none is finite
constexpr int kMaxGrid = 512, kMaxWideGrid = 160; // CTAs that the workspace provides for, of either kernel

// Two codes as FP16 numbers: nibbles 0 and 4 of a word become 1024 + n, nibbles 1 and 5 become 64 + n, one logic operation each.
// The masks come from the kernel's arguments: as literals the compiler spends two operations (AND, OR) on every one.
struct CodeMasks {
  unsigned low, high, low_base, high_base;
};
constexpr CodeMasks kCodeMasks{0x000f000fu, 0x00f000f0u, 0x64006400u, 0x54005400u};

// The unit that begins in a CTA's run and goes on in others': how many pieces there are (0: no such unit), in which slot this
// CTA left the first one (the others are in their CTAs' slot 0), and where the output goes.
struct Split {
  int pieces, first_slot, row_begin, block, head, columns;
};

struct AttentionArgs {
  KvView cache;
  SequenceView seq;
  const void *q;
  void *out;
  long long q_stride, out_stride;
  int q_heads, group; // heads that share a KV head
  float scale;        // |scale| * log2(e), or 1 where scale is 0
  float sign;         // of scale: the queries are multiplied by it
  int window;
  struct Split *split; // [grid]
  float *partial;      // [grid][2]: outputs [columns][head_dim], then maximum and sum [columns][2]
  CodeMasks masks;
  int *bad;
};

__device__ __forceinline__ unsigned MaskOr(unsigned w, unsigned mask, unsigned base) {
  unsigned r;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(w), "r"(mask), "r"(base)); // (w & mask) | base
  return r;
}
__device__ __forceinline__ unsigned Low(unsigned w, const CodeMasks &m) { return MaskOr(w, m.low, m.low_base); }
__device__ __forceinline__ unsigned High(unsigned w, const CodeMasks &m) { return MaskOr(w, m.high, m.high_base); }
__device__ __forceinline__ unsigned Scaled(unsigned x, unsigned offset, __half2 scale) {
  const __half2 v = __hmul2(__hsub2(*reinterpret_cast<__half2 *>(&x), *reinterpret_cast<__half2 *>(&offset)), scale);
  return *reinterpret_cast<const unsigned *>(&v);
}
__device__ __forceinline__ unsigned Pack(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const unsigned *>(&h);
}
__device__ __forceinline__ float Exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// What a column's scores are multiplied by.  It does not become zero, which would make a NaN of a masked token's -infinity; at the least
// factor every score (below 2^25 before the factor) is as good as zero.  At the largest they stay above kNever; a score that is not zero is
// beyond kLargestTop there, or lost in 32 bits.
__device__ __forceinline__ float FactorOf(float scale, float power) {
  return fminf(fmaxf(scale * power, kLeastFactor), kLargestFactor);
}
__device__ __forceinline__ void Widen(uint4 u, const __nv_bfloat16 *, float (&x)[8]) {
  const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    x[2 * i] = __uint_as_float(w[i] << 16), x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
}
__device__ __forceinline__ void Widen(uint4 u, const __half *, float (&x)[8]) {
  const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
    x[2 * i] = f.x, x[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ void Store4(__nv_bfloat16 *p, float4 v) {
  const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
  *reinterpret_cast<uint2 *>(p) = make_uint2(*reinterpret_cast<const unsigned *>(&a), *reinterpret_cast<const unsigned *>(&b));
}
__device__ __forceinline__ void Store4(__half *p, float4 v) {
  *reinterpret_cast<uint2 *>(p) = make_uint2(Pack(v.x, v.y), Pack(v.z, v.w));
}

// Shared memory by 32-bit address: through pointers the compiler used 64-bit generic addresses, several operations for each access.
__device__ __forceinline__ void StoreShared(unsigned address, uint4 v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(address), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ uint4 LoadShared16(unsigned address) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(address) : "memory");
  return v;
}
__device__ __forceinline__ uint2 LoadShared8(unsigned address) {
  uint2 v;
  asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(address) : "memory");
  return v;
}
__device__ __forceinline__ unsigned LoadShared4(unsigned address) {
  unsigned v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(address) : "memory");
  return v;
}
__device__ __forceinline__ unsigned short LoadShared2(unsigned address) {
  unsigned short v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(address) : "memory");
  return v;
}

// a / b of numbers that are nearly always below 2^32, where the division is much cheaper
__device__ __forceinline__ long long Quotient(long long a, long long b) {
  return (a | b) >> 32 ? a / b : static_cast<unsigned>(a) / static_cast<unsigned>(b);
}

// Exclusive prefix sum of one value per thread over the CTA; *total gets the sum.
template <int Warps> __device__ __forceinline__ long long BlockPrefix(long long value, long long *scan, long long *total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long inclusive = value;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const long long other = __shfl_up_sync(0xffffffffu, inclusive, d);
    if (lane >= d)
      inclusive += other;
  }
  if (lane == 31)
    scan[warp] = inclusive;
  __syncthreads();
  long long before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < Warps; ++w) {
    before += w < warp ? scan[w] : 0;
    all += scan[w];
  }
  __syncthreads();
  *total = all;
  return before + inclusive - value;
}

// Where a CTA leaves a piece of a unit: which = 0 for the first unit of its run, 1 for the last.
template <int D, int Columns> __device__ __forceinline__ float *PartialOf(const AttentionArgs &a, long long cta, int which) {
  return a.partial + (cta * 2 + which) * (Columns * (D + 2));
}
template <typename T, int D, int Columns>
__device__ __forceinline__ void StoreOutput(const AttentionArgs &a, int row_begin, int block, int head, int column, int dim, float4 v, float sum) {
  const int place = block * Columns + column, row = place / a.group, h = head * a.group + place % a.group;
  const float inverse = sum > 0 ? 1.f / sum : 0.f;
  Store4(static_cast<T *>(a.out) + static_cast<long long>(row_begin + row) * a.out_stride + h * D + dim,
         make_float4(v.x * inverse, v.y * inverse, v.z * inverse, v.w * inverse));
}

// Joins the pieces of the unit that begins in run blockIdx.x.  Few pieces: a warp per column.  Many: all warps read a column's
// pieces, each some of them, for columns y, y + gridDim.y, ...
constexpr int kJoinWarps = 8, kFewPieces = 16;
template <typename T, int D, int Columns> __global__ void __launch_bounds__(kJoinWarps * 32) JoinKernel(const __grid_constant__ AttentionArgs a) {
  constexpr int kLanes = D / 4, kSide = 32 / kLanes, kAtOnce = kJoinWarps * kSide, kFlight = 4; // pieces read at a time; loads in flight
  __shared__ float s_sum[kAtOnce];
  __shared__ float4 s_out[kAtOnce][kLanes];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const Split split = a.split[blockIdx.x];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, dim = threadIdx.x % kLanes * 4;
  if (!split.pieces)
    return;
  const bool few = split.pieces <= kFewPieces;
  const int side = few ? lane / kLanes : threadIdx.x / kLanes, step = few ? kSide : kAtOnce;
  for (int column = few ? blockIdx.y * kJoinWarps + warp : blockIdx.y; column < split.columns; column += few ? gridDim.y * kJoinWarps : gridDim.y) {
    auto piece = [&](int p) { return PartialOf<D, Columns>(a, blockIdx.x + p, p ? 0 : split.first_slot); };
    float top = kNever, sum = 0;
    for (int p = lane; p < split.pieces; p += 32)
      top = fmaxf(top, __ldcg(piece(p) + Columns * D + 2 * column));
#pragma unroll
    for (int m = 1; m < 32; m *= 2)
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, m));
    float4 v = make_float4(0, 0, 0, 0);
    for (int p0 = side; p0 < split.pieces; p0 += step * kFlight) {
      float4 x[kFlight];
      float2 ml[kFlight];
#pragma unroll
      for (int j = 0; j < kFlight; ++j)
        if (p0 + j * step < split.pieces) {
          const float *const from = piece(p0 + j * step);
          x[j] = __ldcg(reinterpret_cast<const float4 *>(from + column * D + dim));
          ml[j] = __ldcg(reinterpret_cast<const float2 *>(from + Columns * D + 2 * column));
        }
#pragma unroll
      for (int j = 0; j < kFlight; ++j)
        if (p0 + j * step < split.pieces) {
          const float f = Exp2(ml[j].x - top);
          sum += f * ml[j].y;
          v.x += f * x[j].x, v.y += f * x[j].y, v.z += f * x[j].z, v.w += f * x[j].w;
        }
    }
    if (few) {
#pragma unroll
      for (int m = kLanes; m < 32; m *= 2) {
        sum += __shfl_xor_sync(0xffffffffu, sum, m);
        v.x += __shfl_xor_sync(0xffffffffu, v.x, m), v.y += __shfl_xor_sync(0xffffffffu, v.y, m);
        v.z += __shfl_xor_sync(0xffffffffu, v.z, m), v.w += __shfl_xor_sync(0xffffffffu, v.w, m);
      }
      if (side == 0)
        StoreOutput<T, D, Columns>(a, split.row_begin, split.block, split.head, column, dim, v, sum);
      continue;
    }
    s_out[side][dim / 4] = v;
    if (dim == 0)
      s_sum[side] = sum;
    __syncthreads();
    if (threadIdx.x < kLanes) {
      for (int i = 1; i < kAtOnce; ++i) {
        const float4 x = s_out[i][threadIdx.x];
        v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
      }
      sum = 0;
      for (int i = 0; i < kAtOnce; ++i)
        sum += s_sum[i];
      StoreOutput<T, D, Columns>(a, split.row_begin, split.block, split.head, column, dim, v, sum);
    }
    __syncthreads();
  }
}

template <typename T, int D, int Columns> int LaunchJoin(const AttentionArgs &a, int grid, cudaStream_t stream) {
  cudaLaunchConfig_t config{};
  cudaLaunchAttribute attribute{};
  attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute.val.programmaticStreamSerializationAllowed = 1;
  // Columns of a unit side by side: a CTA per column where few units share the GPU, so that each has many pieces (one sequence of 131072
  // tokens: 31 us with 8, 34 us with 4); otherwise most CTAs find nothing to join and cost time (32 short sequences: 15.4 us with 4, 16.5 us with 8).
  const bool few_units = static_cast<long long>(a.seq.count) * a.cache.kv_heads <= 16;
  config.gridDim = dim3(grid, Columns == 256 ? 16 : few_units ? 8 : 4), config.blockDim = dim3(kJoinWarps * 32), config.stream = stream;
  config.attrs = &attribute, config.numAttrs = 1;
  return CudaStatus(cudaLaunchKernelEx(&config, JoinKernel<T, D, Columns>, a));
}

// attention_wide.cu: blocks of 256 columns on tcgen05
template <typename T, int D> int LaunchWide(const AttentionArgs &a, int sms, cudaStream_t stream);
size_t WidePartialBytes(int head_dim);

} // namespace attention
} // namespace padra
