// Per-head norm and rotation of queries and keys, appending keys and values to the paged 4-bit cache, reading it back.
//
// Norm + rotation: y = x * w / sqrt(mean(x^2) + eps), then pair (a, b) -> amplitude * (a cos t - b sin t, a sin t + b cos t)
// with t = position * inv_freq.  One pass: a head of a row sits in the registers of head_dim / 8 lanes (16 bytes of 16-bit
// values each), the sum of squares is one value per lane and a few shuffles, and the partner of a rotated value is in the same lane
// (interleaved) or dims / 16 lanes on (half layout).  cos and sin of a row are computed once per CTA for all of its heads:
// the angle is reduced to a fraction of a turn in 64 bits, so a far position costs no precision and no slow path.
// Bound by bandwidth for many rows and by launch latency for few.
#include "kernels.cuh"
#include "kv_cache.cuh"

namespace padra {
namespace {

constexpr int kRowThreads = 256, kRowWarps = kRowThreads / 32;
constexpr int kMaxCtaRows = 4;

template <typename T> struct Rows;
template <> struct Rows<__nv_bfloat16> {
  static __device__ __forceinline__ void Load(const __nv_bfloat16 *p, float (&x)[8]) {
    const uint4 u = *reinterpret_cast<const uint4 *>(p);
    const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      x[2 * i] = __uint_as_float(w[i] << 16), x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
  // false where a rounded value is not finite
  template <typename Real> static __device__ __forceinline__ bool Store(__nv_bfloat16 *p, const Real (&x)[8]) {
    unsigned w[4], wrong = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 pair = __floats2bfloat162_rn(static_cast<float>(x[2 * i]), static_cast<float>(x[2 * i + 1]));
      w[i] = *reinterpret_cast<const unsigned *>(&pair);
      wrong |= ((w[i] & 0x7f80u) == 0x7f80u) | ((w[i] & 0x7f800000u) == 0x7f800000u);
    }
    *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    return !wrong;
  }
};
template <> struct Rows<__half> {
  static __device__ __forceinline__ void Load(const __half *p, float (&x)[8]) {
    const uint4 u = *reinterpret_cast<const uint4 *>(p);
    const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
      x[2 * i] = f.x, x[2 * i + 1] = f.y;
    }
  }
  template <typename Real> static __device__ __forceinline__ bool Store(__half *p, const Real (&x)[8]) {
    unsigned w[4], wrong = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 pair = __floats2half2_rn(static_cast<float>(x[2 * i]), static_cast<float>(x[2 * i + 1]));
      w[i] = *reinterpret_cast<const unsigned *>(&pair);
      wrong |= ((w[i] & 0x7c00u) == 0x7c00u) | ((w[i] & 0x7c000000u) == 0x7c000000u);
    }
    *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    return !wrong;
  }
};
template <> struct Rows<float> {
  static __device__ __forceinline__ void Load(const float *p, float (&x)[8]) {
    const float4 a = *reinterpret_cast<const float4 *>(p), b = *reinterpret_cast<const float4 *>(p + 4);
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  }
  template <typename Real> static __device__ __forceinline__ bool Store(float *p, const Real (&x)[8]) {
    bool fine = true;
    float f[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      f[i] = static_cast<float>(x[i]);
      fine &= isfinite(f[i]) != 0;
    }
    *reinterpret_cast<float4 *>(p) = make_float4(f[0], f[1], f[2], f[3]);
    *reinterpret_cast<float4 *>(p + 4) = make_float4(f[4], f[5], f[6], f[7]);
    return fine;
  }
};

template <typename Real> struct Turn { // cos and sin of one pair, times the amplitude
  Real cos, sin;
};
__device__ __forceinline__ double Turns(int position, double inv_freq) {
  const double t = static_cast<double>(position) * inv_freq * 0.15915494309189533577; // 1 / (2 pi)
  return t - rint(t);
}
__device__ __forceinline__ void MakeTurn(double turns, double amplitude, Turn<float> *to) {
  float s, c;
  sincospif(static_cast<float>(2.0 * turns), &s, &c);
  to->cos = c * static_cast<float>(amplitude), to->sin = s * static_cast<float>(amplitude);
}
__device__ __forceinline__ void MakeTurn(double turns, double amplitude, Turn<double> *to) {
  double s, c;
  sincospi(2.0 * turns, &s, &c);
  to->cos = c * amplitude, to->sin = s * amplitude;
}
__device__ __forceinline__ float InverseRoot(float x) { return rsqrtf(x); }
__device__ __forceinline__ double InverseRoot(double x) { return 1.0 / sqrt(x); }

// Norm and rotation of one head held by D / 8 neighbouring lanes, eight values each.  `at` = the lane's place in the head.
// Every lane of the warp takes part in the exchanges.
template <int D, typename Real, typename TableReal>
__device__ __forceinline__ void NormRotate(Real (&x)[8], int at, const unsigned short *weight, double eps, const Turn<TableReal> *turns, int dims,
                                           bool interleaved) {
  constexpr int kLanes = D / 8;
  if (weight) {
    Real sum = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      sum += x[i] * x[i];
#pragma unroll
    for (int d = 1; d < kLanes; d *= 2)
      sum += __shfl_xor_sync(0xffffffffu, sum, d);
    const Real inverse = InverseRoot(sum * static_cast<Real>(1.0 / D) + static_cast<Real>(eps));
    const uint4 u = __ldg(reinterpret_cast<const uint4 *>(weight) + at);
    const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = x[2 * i] * inverse * static_cast<Real>(__uint_as_float(w[i] << 16));
      x[2 * i + 1] = x[2 * i + 1] * inverse * static_cast<Real>(__uint_as_float(w[i] & 0xffff0000u));
    }
  }
  if (interleaved) {
    if (8 * at < dims) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const Turn<TableReal> t = turns[4 * at + i];
        const Real a = x[2 * i], b = x[2 * i + 1], c = static_cast<Real>(t.cos), s = static_cast<Real>(t.sin);
        x[2 * i] = a * c - b * s;
        x[2 * i + 1] = a * s + b * c;
      }
    }
  } else if (dims) {
    const int half = dims / 16; // lanes between the two values of a pair
    const bool second = at >= half;
    const int lane = threadIdx.x & 31, from = at >= 2 * half ? lane : second ? lane - half : lane + half;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const Real other = __shfl_sync(0xffffffffu, x[i], from);
      if (at < 2 * half) {
        const Turn<TableReal> t = turns[8 * (second ? at - half : at) + i];
        const Real c = static_cast<Real>(t.cos), s = static_cast<Real>(t.sin);
        x[i] = second ? other * s + x[i] * c : x[i] * c - other * s;
      }
    }
  }
}

struct HeadRows { // one of q, k, v: rows of `heads` heads
  const void *in;
  void *out;
  long long stride, out_stride;
  const unsigned short *weight;
  int heads;
};
struct RotaryArgs {
  const double *inv_freq;
  double amplitude;
  int dims, interleaved;
};

// ---- norm + rotation without a cache ----
// A CTA takes `cta_rows` rows and the heads [y * share, ...) of them; a warp takes 32 / (D / 8) heads of a row at a time.
template <typename T, int D>
__global__ void __launch_bounds__(kRowThreads) NormRopeKernel(HeadRows q, HeadRows k, double eps, const int *positions, RotaryArgs rotary, int rows,
                                                              int cta_rows, int share, int *bad) {
  constexpr int kLanes = D / 8, kSide = 32 / kLanes;
  __shared__ Turn<float> turns[kMaxCtaRows][D / 2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, pairs = rotary.dims / 2;
  const int first = blockIdx.x * cta_rows, count = min(cta_rows, rows - first);
  for (int i = threadIdx.x; i < count * pairs; i += kRowThreads) {
    const int r = i / pairs, p = i - r * pairs;
    MakeTurn(Turns(positions[first + r], rotary.inv_freq[p]), rotary.amplitude, &turns[r][p]);
  }
  __syncthreads();
  const int q_units = (q.heads + kSide - 1) / kSide, units = q_units + (k.heads + kSide - 1) / kSide;
  const int from = blockIdx.y * share, to = min(units, from + share), mine = to - from;
  const int at = lane % kLanes;
  for (int i = warp; i < count * mine; i += kRowWarps) {
    const int r = i / mine, unit = from + i - r * mine;
    const bool is_q = unit < q_units;
    const HeadRows &a = is_q ? q : k;
    const int head = (is_q ? unit : unit - q_units) * kSide + lane / kLanes;
    const bool there = head < a.heads;
    float x[8] = {};
    if (there)
      Rows<T>::Load(static_cast<const T *>(a.in) + static_cast<long long>(first + r) * a.stride + head * D + 8 * at, x);
    NormRotate<D, float>(x, at, a.weight, eps, turns[r], rotary.dims, rotary.interleaved);
    if (there && !Rows<T>::Store(static_cast<T *>(a.out) + static_cast<long long>(first + r) * a.out_stride + head * D + 8 * at, x))
      Raise(bad);
  }
}

// ---- append ----
// Eight values of a lane as eight codes, four lanes to a group.  Everything here is 64-bit: the border between two codes is
// met by values that a 32-bit rotation could put on either side, and equal inputs have to give equal bytes.  The FP64
// pipe has the room: 2048 rows of four heads are a million values, some 15 operations each.
__device__ __forceinline__ unsigned QuantiseWord(const double (&x)[8], unsigned short *scale_bits, bool *fine) {
  double most = 0;
  bool finite = true;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    most = fmax(most, fabs(x[i]));
    finite &= isfinite(x[i]) != 0;
  }
#pragma unroll
  for (int d = 1; d < 4; d *= 2)
    most = fmax(most, __shfl_xor_sync(0xffffffffu, most, d));
  *fine = finite && most <= static_cast<double>(kKvLargest);
  const __half h = __double2half(most / 7.0);
  const double scale = static_cast<double>(__half2float(h));
  unsigned word = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const double code = scale > 0 ? fmin(fmax(rint(x[i] / scale), -7.0), 7.0) : 0.0;
    word |= static_cast<unsigned>(static_cast<int>(code) + 8) << (4 * i);
  }
  *scale_bits = __half_as_ushort(h);
  return word;
}

template <typename T, int D>
__global__ void __launch_bounds__(kRowThreads) AppendKernel(KvView cache, SequenceView seq, HeadRows q, HeadRows k, HeadRows v, double eps,
                                                            RotaryArgs rotary, int cta_rows, int share, int *bad) {
  constexpr int kLanes = D / 8, kSide = 32 / kLanes, kGroups = D / kKvGroup;
  __shared__ Turn<double> turns[kMaxCtaRows][D / 2];
  __shared__ int s_page[kMaxCtaRows], s_position[kMaxCtaRows];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, pairs = rotary.dims / 2;
  const int first = blockIdx.x * cta_rows, count = min(cta_rows, seq.rows - first);
  if (warp < count) {
    int position = -1, page = -1;
    const int s = LocateRow(seq, cache, first + warp, &position, bad);
    if (s >= 0 && position >= 0)
      page = PageOf(seq, cache, s, position, bad);
    if (!lane)
      s_page[warp] = page, s_position[warp] = position; // page -1: nothing is done for the row
  }
  __syncthreads();
  for (int i = threadIdx.x; i < count * pairs; i += kRowThreads) {
    const int r = i / pairs, p = i - r * pairs;
    if (s_page[r] >= 0)
      MakeTurn(Turns(s_position[r], rotary.inv_freq[p]), rotary.amplitude, &turns[r][p]);
  }
  __syncthreads();
  const int q_units = (q.heads + kSide - 1) / kSide, kv_units = (k.heads + kSide - 1) / kSide, units = q_units + 2 * kv_units;
  const int from = blockIdx.y * share, to = min(units, from + share), mine = to - from;
  const int at = lane % kLanes;
  for (int i = warp; i < count * mine; i += kRowWarps) { // warp-uniform up to the head
    const int r = i / mine, unit = from + i - r * mine;
    if (s_page[r] < 0)
      continue;
    const int kind = unit < q_units ? 0 : unit < q_units + kv_units ? 1 : 2;
    const HeadRows &a = kind == 0 ? q : kind == 1 ? k : v;
    const int head = (kind == 0 ? unit : unit - q_units - (kind - 1) * kv_units) * kSide + lane / kLanes;
    const bool there = head < a.heads;
    float x[8] = {};
    if (there)
      Rows<T>::Load(static_cast<const T *>(a.in) + static_cast<long long>(first + r) * a.stride + head * D + 8 * at, x);
    if (kind == 0) {
      NormRotate<D, float>(x, at, a.weight, eps, turns[r], rotary.dims, rotary.interleaved);
      if (there && !Rows<T>::Store(static_cast<T *>(a.out) + static_cast<long long>(first + r) * a.out_stride + head * D + 8 * at, x))
        Raise(bad);
      continue;
    }
    double y[8];
#pragma unroll
    for (int j = 0; j < 8; ++j)
      y[j] = static_cast<double>(x[j]);
    if (kind == 1)
      NormRotate<D, double>(y, at, a.weight, eps, turns[r], rotary.dims, rotary.interleaved);
    unsigned short scale;
    bool fine;
    const unsigned word = QuantiseWord(y, &scale, &fine);
    // one decision for the whole head: it is written or left as it was
    const unsigned lanes = (kLanes == 32 ? 0xffffffffu : (1u << kLanes) - 1) << (lane / kLanes * kLanes);
    const bool whole = (__ballot_sync(0xffffffffu, !fine) & lanes) == 0;
    if (!there)
      continue;
    if (!whole) {
      Raise(bad);
      continue;
    }
    const int slot = s_position[r] & (cache.page_size - 1), group = at / 4, quarter = at & 3;
    unsigned char *codes = cache.block(s_page[r], head) + (kind == 2 ? cache.code_bytes() + cache.scale_bytes() : 0);
    reinterpret_cast<unsigned *>(codes + slot * (D / 2))[quarter * kGroups + group] = word;
    if (!quarter)
      reinterpret_cast<unsigned short *>(codes + cache.code_bytes() + slot * (D / 16))[group] = scale;
  }
}

// ---- read ----
// A thread takes one word (eight codes) of K and of V of one head.
constexpr int kReadRows = 16;
template <typename T, int D>
__global__ void __launch_bounds__(kRowThreads) ReadKernel(KvView cache, SequenceView seq, T *k_out, T *v_out, long long k_stride, long long v_stride,
                                                          int *bad) {
  constexpr int kWords = D / 8, kGroups = D / kKvGroup;
  __shared__ int s_page[kReadRows], s_slot[kReadRows];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int first = blockIdx.x * kReadRows, count = min(kReadRows, seq.rows - first);
  for (int r = warp; r < count; r += kRowWarps) {
    int position = -1, page = -1;
    const int s = LocateRow(seq, cache, first + r, &position, bad);
    if (s >= 0 && position >= 0)
      page = PageOf(seq, cache, s, position, bad);
    if (!lane)
      s_page[r] = page, s_slot[r] = position & (cache.page_size - 1);
  }
  __syncthreads();
  const int per_row = cache.kv_heads * kWords;
  for (int i = threadIdx.x; i < count * per_row; i += kRowThreads) {
    const int r = i / per_row, j = i - r * per_row, head = j / kWords, at = j % kWords; // values 8 at .. 8 at + 7 of the head
    if (s_page[r] < 0)
      continue;
    const unsigned char *codes = cache.block(s_page[r], head);
    const int group = at / 4, place = (at & 3) * kGroups + group;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      const unsigned word = reinterpret_cast<const unsigned *>(codes + s_slot[r] * (D / 2))[place];
      const float scale = HalfBitsToFloat(reinterpret_cast<const unsigned short *>(codes + cache.code_bytes() + s_slot[r] * (D / 16))[group]);
      float x[8];
#pragma unroll
      for (int n = 0; n < 8; ++n)
        x[n] = static_cast<float>(static_cast<int>(word >> (4 * n) & 15u) - 8) * scale;
      T *out = which ? v_out + (first + r) * v_stride : k_out + (first + r) * k_stride;
      if (!Rows<T>::Store(out + head * D + 8 * at, x))
        Raise(bad);
      codes += cache.code_bytes() + cache.scale_bytes();
    }
  }
}

// Rows per CTA and heads per CTA: four rows share a CTA's cos and sin where there are rows for every SM anyway; few rows are
// spread over the SMs by splitting their heads, one warp's share each at the least.
void Shape(int rows, int units, int *cta_rows, dim3 *grid, int *share) {
  *cta_rows = rows >= 4 * 148 ? 4 : 1;
  const int x = (rows + *cta_rows - 1) / *cta_rows;
  int parts = *cta_rows > 1 ? 1 : (2 * 148 + x - 1) / x;
  const int most = (units + kRowWarps - 1) / kRowWarps;
  parts = parts < 1 ? 1 : parts > most ? most : parts;
  *share = (units + parts - 1) / parts;
  *grid = dim3(x, (units + *share - 1) / *share);
}

template <template <typename, int> class Op, typename T, typename... A> int ByDim(int head_dim, const A &...a) {
  if (head_dim == 64)
    return Op<T, 64>::Run(a...);
  if (head_dim == 128)
    return Op<T, 128>::Run(a...);
  if constexpr (Op<T, 64>::kWidest == 256)
    if (head_dim == 256)
      return Op<T, 256>::Run(a...);
  return PADRA_UNSUPPORTED;
}
template <template <typename, int> class Op, typename... A> int ByTypeAndDim(int type, int head_dim, const A &...a) {
  switch (type) {
  case PADRA_ROWS_BF16:
    return ByDim<Op, __nv_bfloat16>(head_dim, a...);
  case PADRA_ROWS_F16:
    return ByDim<Op, __half>(head_dim, a...);
  case PADRA_ROWS_F32:
    return ByDim<Op, float>(head_dim, a...);
  default:
    return PADRA_UNSUPPORTED;
  }
}

template <typename T, int D> struct NormRope {
  static constexpr int kWidest = 256;
  static int Run(const HeadRows &q, const HeadRows &k, double eps, const int *positions, const RotaryArgs &rotary, int rows, int *bad,
                 cudaStream_t stream) {
    constexpr int kSide = 32 / (D / 8);
    int cta_rows, share;
    dim3 grid;
    Shape(rows, (q.heads + kSide - 1) / kSide + (k.heads + kSide - 1) / kSide, &cta_rows, &grid, &share);
    NormRopeKernel<T, D><<<grid, kRowThreads, 0, stream>>>(q, k, eps, positions, rotary, rows, cta_rows, share, bad);
    return CudaStatus(cudaGetLastError());
  }
};
template <typename T, int D> struct Append {
  static constexpr int kWidest = 128;
  static int Run(const KvView &cache, const SequenceView &seq, const HeadRows &q, const HeadRows &k, const HeadRows &v, double eps,
                 const RotaryArgs &rotary, int *bad, cudaStream_t stream) {
    constexpr int kSide = 32 / (D / 8);
    int cta_rows, share;
    dim3 grid;
    Shape(seq.rows, (q.heads + kSide - 1) / kSide + 2 * ((k.heads + kSide - 1) / kSide), &cta_rows, &grid, &share);
    AppendKernel<T, D><<<grid, kRowThreads, 0, stream>>>(cache, seq, q, k, v, eps, rotary, cta_rows, share, bad);
    return CudaStatus(cudaGetLastError());
  }
};
template <typename T, int D> struct Read {
  static constexpr int kWidest = 128;
  static int Run(const KvView &cache, const SequenceView &seq, void *k_out, void *v_out, long long k_stride, long long v_stride, int *bad,
                 cudaStream_t stream) {
    ReadKernel<T, D><<<(seq.rows + kReadRows - 1) / kReadRows, kRowThreads, 0, stream>>>(cache, seq, static_cast<T *>(k_out), static_cast<T *>(v_out),
                                                                                       k_stride, v_stride, bad);
    return CudaStatus(cudaGetLastError());
  }
};

bool RotaryOk(const padra_rotary *r, int head_dim, RotaryArgs *to) {
  *to = RotaryArgs{nullptr, 1.0, 0, 0};
  if (!r || !r->dims)
    return true;
  if (!r->inv_freq || r->dims < 0 || r->dims > head_dim || r->dims % 16)
    return false;
  *to = RotaryArgs{r->inv_freq, r->amplitude, r->dims, r->interleaved != 0};
  return true;
}
bool WeightOk(const unsigned short *w) {
  return reinterpret_cast<uintptr_t>(w) % 16 == 0;
}

} // namespace

int LaunchNormRope(const void *q, void *q_out, long long q_stride, long long q_out_stride, int q_heads, const void *k, void *k_out,
                   long long k_stride, long long k_out_stride, int k_heads, const unsigned short *q_weight, const unsigned short *k_weight,
                   double eps, const int *positions, const padra_rotary *rotary, int rows, int head_dim, int type, int *bad,
                   cudaStream_t stream) {
  RotaryArgs r;
  if (rows < 0 || rows > (1 << 24) || q_heads < 1 || q_heads > 4096 || k_heads < 0 || k_heads > 4096 || !bad || !(eps >= 0) ||
      !RotaryOk(rotary, head_dim, &r) || (r.dims && !positions) || !WeightOk(q_weight) || !WeightOk(k_weight))
    return PADRA_INVALID_ARGUMENT;
  if (head_dim != 64 && head_dim != 128 && head_dim != 256)
    return PADRA_UNSUPPORTED;
  if (!RowsOk(q, q_stride, q_heads, head_dim) || !RowsOk(q_out, q_out_stride, q_heads, head_dim) ||
      (k_heads && (!RowsOk(k, k_stride, k_heads, head_dim) || !RowsOk(k_out, k_out_stride, k_heads, head_dim))))
    return PADRA_INVALID_ARGUMENT;
  if (!rows)
    return PADRA_OK;
  const HeadRows qr{q, q_out, q_stride, q_out_stride, q_weight, q_heads}, kr{k, k_out, k_stride, k_out_stride, k_weight, k_heads};
  return ByTypeAndDim<NormRope>(type, head_dim, qr, kr, eps, positions, r, rows, bad, stream);
}

int LaunchKvAppend(const padra_kv_cache *cache, const padra_sequences *sequences, const void *k, const void *v, long long k_stride,
                   long long v_stride, const unsigned short *k_weight, double eps, const padra_rotary *rotary, const void *q, void *q_out,
                   long long q_stride, long long q_out_stride, int q_heads, const unsigned short *q_weight, int type, int *bad,
                   cudaStream_t stream) {
  KvView c;
  SequenceView s;
  RotaryArgs r;
  if (!ViewOf(cache, &c) || !ViewOf(sequences, c, &s) || !bad || !(eps >= 0) || !RotaryOk(rotary, c.head_dim, &r) || !WeightOk(q_weight) ||
      !WeightOk(k_weight))
    return PADRA_INVALID_ARGUMENT;
  if (c.head_dim != 64 && c.head_dim != 128)
    return PADRA_UNSUPPORTED;
  if (!RowsOk(k, k_stride, c.kv_heads, c.head_dim) || !RowsOk(v, v_stride, c.kv_heads, c.head_dim))
    return PADRA_INVALID_ARGUMENT;
  if (q && (q_heads < 1 || q_heads > 4096 || !RowsOk(q, q_stride, q_heads, c.head_dim) || !RowsOk(q_out, q_out_stride, q_heads, c.head_dim)))
    return PADRA_INVALID_ARGUMENT;
  if (!s.rows || !s.count)
    return PADRA_OK;
  const HeadRows qr{q, q_out, q_stride, q_out_stride, q_weight, q ? q_heads : 0}, kr{k, nullptr, k_stride, 0, k_weight, c.kv_heads},
      vr{v, nullptr, v_stride, 0, nullptr, c.kv_heads};
  return ByTypeAndDim<Append>(type, c.head_dim, c, s, qr, kr, vr, eps, r, bad, stream);
}

int LaunchKvRead(const padra_kv_cache *cache, const padra_sequences *sequences, void *k_out, void *v_out, long long k_stride, long long v_stride,
                 int type, int *bad, cudaStream_t stream) {
  KvView c;
  SequenceView s;
  if (!ViewOf(cache, &c) || !ViewOf(sequences, c, &s) || !bad)
    return PADRA_INVALID_ARGUMENT;
  if (c.head_dim != 64 && c.head_dim != 128)
    return PADRA_UNSUPPORTED;
  if (!RowsOk(k_out, k_stride, c.kv_heads, c.head_dim) || !RowsOk(v_out, v_stride, c.kv_heads, c.head_dim))
    return PADRA_INVALID_ARGUMENT;
  if (!s.rows || !s.count)
    return PADRA_OK;
  return ByTypeAndDim<Read>(type, c.head_dim, c, s, k_out, v_out, k_stride, v_stride, bad, stream);
}

} // namespace padra
