// Attention over the paged 4-bit cache: out = softmax(scale * q k^T + mask) v.
//
// One warp per (row, query head): 32 tokens at a time, one per lane for the scores, running maximum and sum, then every lane
// gathers its share of the output over the 32 tokens.
#include "kernels.cuh"
#include "kv_cache.cuh"

namespace padra {
namespace {

constexpr int kWarps = 4;

template <typename T> __device__ __forceinline__ float ToFloat(T x) { return static_cast<float>(x); }
__device__ __forceinline__ void FromFloat(float x, __nv_bfloat16 *to) { *to = __float2bfloat16_rn(x); }
__device__ __forceinline__ void FromFloat(float x, __half *to) { *to = __float2half_rn(x); }

template <typename T, int D>
__global__ void __launch_bounds__(kWarps * 32) AttentionKernel(KvView cache, SequenceView seq, const T *q, T *out, long long q_stride,
                                                               long long out_stride, int q_heads, float scale, int window, int *bad) {
  constexpr int kGroups = D / kKvGroup, kOwn = D / 32;
  __shared__ float s_q[kWarps][D];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int row = blockIdx.x, head = blockIdx.y * kWarps + warp, group = q_heads / cache.kv_heads;
  if (head >= q_heads)
    return;
  int position = -1;
  const int s = LocateRow(seq, cache, row, &position, bad);
  if (s < 0)
    return;
  T *const mine = out + row * out_stride + head * D;
  bool finite = true;
  for (int d = lane; d < D; d += 32) {
    const float x = position >= 0 ? ToFloat(q[row * q_stride + head * D + d]) : 0.f;
    finite &= isfinite(x) != 0;
    s_q[warp][d] = x * scale;
  }
  if (__any_sync(0xffffffffu, !finite)) {
    Raise(bad);
    position = -1;
  }
  __syncwarp();
  float m = -INFINITY, l = 0, o[kOwn] = {};
  const int first = window > 0 && position >= window ? position - window + 1 : 0;
  for (int t0 = first; t0 <= position; t0 += 32) {
    const int t = t0 + lane;
    float score = -INFINITY;
    int page = -1;
    if (t <= position)
      page = PageOf(seq, cache, s, t, bad);
    const int slot = t & (cache.page_size - 1);
    const unsigned char *block = cache.block(page < 0 ? 0 : page, head / group);
    if (page >= 0) {
      score = 0;
      for (int w = 0; w < D / 8; ++w) {
        const int g = w % kGroups, c = w / kGroups;
        const unsigned word = reinterpret_cast<const unsigned *>(block + slot * (D / 2))[w];
        const float f = HalfBitsToFloat(reinterpret_cast<const unsigned short *>(block + cache.code_bytes() + slot * (D / 16))[g]);
        float sum = 0;
        for (int n = 0; n < 8; ++n)
          sum += static_cast<float>(static_cast<int>(word >> (4 * n) & 15u) - 8) * s_q[warp][32 * g + 8 * c + n];
        score += sum * f;
      }
    }
    float most = score;
    for (int d = 1; d < 32; d *= 2)
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
    if (most == -INFINITY)
      continue;
    const float next = fmaxf(m, most), shrink = expf(m - next), p = expf(score - next);
    m = next, l = l * shrink;
    for (int j = 0; j < kOwn; ++j)
      o[j] *= shrink;
    for (int n = 0; n < 32; ++n) {
      const float pn = __shfl_sync(0xffffffffu, p, n);
      const unsigned long long b = __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(block), n);
      const int sn = __shfl_sync(0xffffffffu, slot, n);
      if (pn == 0.f)
        continue;
      l += pn;
      const unsigned char *values = reinterpret_cast<const unsigned char *>(b) + cache.code_bytes() + cache.scale_bytes();
      for (int j = 0; j < kOwn; ++j) {
        const int d = j * 32 + lane, place = (d / 8 & 3) * kGroups + j;
        const unsigned word = reinterpret_cast<const unsigned *>(values + sn * (D / 2))[place];
        const float f = HalfBitsToFloat(reinterpret_cast<const unsigned short *>(values + cache.code_bytes() + sn * (D / 16))[j]);
        o[j] += pn * f * static_cast<float>(static_cast<int>(word >> (4 * (d & 7)) & 15u) - 8);
      }
    }
  }
  for (int j = 0; j < kOwn; ++j)
    FromFloat(l > 0 ? o[j] / l : 0.f, mine + j * 32 + lane);
}

template <typename T, int D>
int Launch(const KvView &c, const SequenceView &s, const void *q, void *out, long long q_stride, long long out_stride, int q_heads, float scale,
           int window, int *bad, cudaStream_t stream) {
  AttentionKernel<T, D><<<dim3(s.rows, (q_heads + kWarps - 1) / kWarps), kWarps * 32, 0, stream>>>(
      c, s, static_cast<const T *>(q), static_cast<T *>(out), q_stride, out_stride, q_heads, scale, window, bad);
  return CudaStatus(cudaGetLastError());
}

} // namespace

int LaunchAttention(const padra_kv_cache *cache, const padra_sequences *sequences, const void *q, void *out, long long q_stride,
                    long long out_stride, int q_heads, int type, float scale, int window, int *bad, cudaStream_t stream) {
  KvView c;
  SequenceView s;
  if (!ViewOf(cache, &c) || !ViewOf(sequences, c, &s) || !bad || q_heads < 1 || q_heads > 4096 || q_heads % c.kv_heads || window < 0)
    return PADRA_INVALID_ARGUMENT;
  if ((c.head_dim != 64 && c.head_dim != 128) || (type != PADRA_ROWS_BF16 && type != PADRA_ROWS_F16))
    return PADRA_UNSUPPORTED;
  if (!RowsOk(q, q_stride, q_heads, c.head_dim) || !RowsOk(out, out_stride, q_heads, c.head_dim))
    return PADRA_INVALID_ARGUMENT;
  if (!s.rows || !s.count)
    return PADRA_OK;
  if (type == PADRA_ROWS_BF16)
    return c.head_dim == 64 ? Launch<__nv_bfloat16, 64>(c, s, q, out, q_stride, out_stride, q_heads, scale, window, bad, stream)
                            : Launch<__nv_bfloat16, 128>(c, s, q, out, q_stride, out_stride, q_heads, scale, window, bad, stream);
  return c.head_dim == 64 ? Launch<__half, 64>(c, s, q, out, q_stride, out_stride, q_heads, scale, window, bad, stream)
                          : Launch<__half, 128>(c, s, q, out, q_stride, out_stride, q_heads, scale, window, bad, stream);
}

} // namespace padra
