// Per-head norm and rotation of queries and keys, appending keys and values to the paged 4-bit cache, reading it back.
//
// Norm + rotation: y = x * w / sqrt(mean(x^2) + eps), then pair (a, b) -> amplitude * (a cos t - b sin t, a sin t + b cos t)
// with t = position * inv_freq.  One pass: a head of a row sits in the registers of head_dim / 8 lanes.  A warp stays with one row, so
// that weights and the row's cos and sin stay in registers, and it has the loads of its next heads under way meanwhile, the first of them
// from before the table is made.  cos and sin of a row are computed once per CTA for all of its heads: the angle is reduced to a
// fraction of a turn in 64 bits, so a far position costs no precision and no slow path.
// Many rows (16384 of 32 + 4 heads of 128 in FP16: 64 us, 4.7 TB/s) take 73% of the copy rate at 67% of the issue slots, few (one row: 3 us)
// are all latency.
#include "kernels.cuh"
#include "kv_cache.cuh"

namespace padra {
namespace {

constexpr int kRowThreads = 256, kRowWarps = kRowThreads / 32;
constexpr int kMaxCtaRows = kRowWarps;

// Four neighbouring values of a row as they lie in memory.
template <typename T> struct Rows;
template <> struct Rows<__nv_bfloat16> {
  using Raw = uint2;
  static __device__ __forceinline__ void Unpack(const Raw &u, float *x) {
    x[0] = __uint_as_float(u.x << 16), x[1] = __uint_as_float(u.x & 0xffff0000u);
    x[2] = __uint_as_float(u.y << 16), x[3] = __uint_as_float(u.y & 0xffff0000u);
  }
  // Largest magnitude of the rounded values so far, two at a time; an infinity or a NaN stays.
  struct Most {
    __nv_bfloat162 m = __floats2bfloat162_rn(0.f, 0.f);
    __device__ __forceinline__ bool Finite() const {
      const unsigned u = *reinterpret_cast<const unsigned *>(&m);
      return (u & 0x7fffu) < 0x7f80u && (u & 0x7fffffffu) < 0x7f800000u;
    }
  };
  static __device__ __forceinline__ void Pack(const float (&x)[8], Raw *lo, Raw *hi, Most *most) {
    __nv_bfloat162 p[4];
    unsigned w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      p[i] = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
      w[i] = *reinterpret_cast<const unsigned *>(&p[i]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      most->m = __hmax2_nan(most->m, __habs2(p[i]));
    *lo = make_uint2(w[0], w[1]), *hi = make_uint2(w[2], w[3]);
  }
};
template <> struct Rows<__half> {
  using Raw = uint2;
  static __device__ __forceinline__ void Unpack(const Raw &u, float *x) {
    const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&u.x)), b = __half22float2(*reinterpret_cast<const __half2 *>(&u.y));
    x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
  }
  struct Most {
    __half2 m = __floats2half2_rn(0.f, 0.f);
    __device__ __forceinline__ bool Finite() const {
      const unsigned u = *reinterpret_cast<const unsigned *>(&m);
      return (u & 0x7fffu) < 0x7c00u && (u & 0x7fffffffu) < 0x7c000000u;
    }
  };
  static __device__ __forceinline__ void Pack(const float (&x)[8], Raw *lo, Raw *hi, Most *most) {
    __half2 p[4];
    unsigned w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      p[i] = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
      w[i] = *reinterpret_cast<const unsigned *>(&p[i]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      most->m = __hmax2_nan(most->m, __habs2(p[i]));
    *lo = make_uint2(w[0], w[1]), *hi = make_uint2(w[2], w[3]);
  }
};
template <> struct Rows<float> {
  using Raw = float4;
  static __device__ __forceinline__ void Unpack(const Raw &u, float *x) { x[0] = u.x, x[1] = u.y, x[2] = u.z, x[3] = u.w; }
  struct Most {
    float m = 0; // zero times each value: NaN once one was not finite
    __device__ __forceinline__ bool Finite() const { return m == 0.f; }
  };
  static __device__ __forceinline__ void Pack(const float (&x)[8], Raw *lo, Raw *hi, Most *most) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      most->m = fmaf(x[i], 0.f, most->m);
    *lo = make_float4(x[0], x[1], x[2], x[3]), *hi = make_float4(x[4], x[5], x[6], x[7]);
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

// ---- norm + rotation in 32 bits ----
// A lane holds values lo .. lo+3 and hi .. hi+3 of its head, chosen so that both values of a pair are its own: no exchange but the sum's.
struct Lane {
  int at, lo, hi, pair; // pair: the first of its four pairs, -1 where its values are not rotated
};
template <int D> __device__ __forceinline__ Lane LaneOf(const RotaryArgs &rotary) {
  Lane l;
  l.at = (threadIdx.x & 31) % (D / 8);
  const bool rotated = 8 * l.at < rotary.dims, apart = rotated && !rotary.interleaved;
  l.lo = apart ? 4 * l.at : 8 * l.at, l.hi = apart ? rotary.dims / 2 + 4 * l.at : 8 * l.at + 4;
  l.pair = rotated ? 4 * l.at : -1;
  return l;
}
template <typename T> struct Eight { // a lane's values as they lie in memory
  typename Rows<T>::Raw lo, hi;
  __device__ __forceinline__ void Load(const T *head, const Lane &lane) {
    lo = *reinterpret_cast<const typename Rows<T>::Raw *>(head + lane.lo), hi = *reinterpret_cast<const typename Rows<T>::Raw *>(head + lane.hi);
  }
};
struct Weights {
  float w[8];
  __device__ __forceinline__ void Load(const unsigned short *weight, const Lane &lane) {
    Rows<__nv_bfloat16>::Unpack(__ldg(reinterpret_cast<const uint2 *>(weight + lane.lo)), w);
    Rows<__nv_bfloat16>::Unpack(__ldg(reinterpret_cast<const uint2 *>(weight + lane.hi)), w + 4);
  }
};
// Sum over the D / 8 lanes of a head.
template <int D> __device__ __forceinline__ float HeadSum(float x) {
#pragma unroll
  for (int d = 1; d < D / 8; d *= 2)
    x += __shfl_xor_sync(0xffffffffu, x, d);
  return x;
}
template <int D, bool Interleaved>
__device__ __forceinline__ void NormRotate(float (&x)[8], const Lane &lane, bool normed, const Weights &weights, double eps, const Turn<float> (&turns)[4]) {
  if (normed) {
    float sum = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      sum += x[i] * x[i];
    const float mean = HeadSum<D>(sum) * (1.f / D) + static_cast<float>(eps);
    float inverse = rsqrtf(mean);
    // Squares of values beyond 2^64 are infinite in 32 bits, those of small ones lose bits or vanish beside a small eps.  Such a head is
    // multiplied by a power of two first; the whole warp goes there, with a factor of one for its other heads.
    const bool narrow = mean >= 0x1p-100f && mean <= 0x1p100f;
    if (__any_sync(0xffffffffu, !narrow)) {
      float most = sqrtf(static_cast<float>(eps));
#pragma unroll
      for (int i = 0; i < 8; ++i)
        most = fmaxf(most, fabsf(x[i]));
#pragma unroll
      for (int d = 1; d < D / 8; d *= 2)
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
      // 2^-k for most in [2^k, 2^(k + 1)), within 2^-126 .. 2^126: the exponent's bits from those of 2^254
      const float power = narrow ? 1.f : __uint_as_float((254u << 23) - min(max(__float_as_uint(most) & 0x7f800000u, 1u << 23), 253u << 23));
      sum = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        x[i] *= power, sum += x[i] * x[i];
      sum = HeadSum<D>(sum);
      if (!narrow)
        inverse = rsqrtf(sum * (1.f / D) + static_cast<float>(eps * power * power));
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
      x[i] = x[i] * inverse * weights.w[i];
  }
  if (lane.pair < 0)
    return;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (Interleaved) {
      const float a = x[2 * i], b = x[2 * i + 1];
      x[2 * i] = a * turns[i].cos - b * turns[i].sin, x[2 * i + 1] = a * turns[i].sin + b * turns[i].cos;
    } else {
      const float a = x[i], b = x[4 + i];
      x[i] = a * turns[i].cos - b * turns[i].sin, x[4 + i] = a * turns[i].sin + b * turns[i].cos;
    }
  }
}

// Units (32 / (D / 8) heads each) first, first + step, ... of one row of q or k, by one warp; Ahead loads are under way.
template <typename T, int D, int Ahead> struct UnitLoop {
  static constexpr int kSide = 32 / (D / 8);
  Eight<T> raw[Ahead];
  const T *in;                  // this lane's values of the next unit to be loaded
  int head, heads, stride, left; // the unit being worked on: this lane's head; units to do
  __device__ __forceinline__ UnitLoop(const HeadRows &a, long long row, int first, int step, const Lane &lane)
      : head(first * kSide + (threadIdx.x & 31) / (D / 8)), heads(a.heads), stride(step * kSide) {
    const int units = (heads + kSide - 1) / kSide;
    left = first < units ? (units - first + step - 1) / step : 0;
    in = static_cast<const T *>(a.in) + row * a.stride + head * D;
#pragma unroll
    for (int j = 0; j < Ahead; ++j) {
      raw[j] = Eight<T>{};
      Fetch(j, head + j * stride, lane);
    }
  }
  __device__ __forceinline__ void Fetch(int j, int at, const Lane &lane) {
    if (at < heads)
      raw[j].Load(in, lane);
    in += stride * D;
  }
  template <bool Interleaved, typename Turns>
  __device__ __forceinline__ void Run(const HeadRows &a, long long row, const Lane &lane, double eps, const Turns &turns_of_row, int *bad) {
    Weights weights{};
    Turn<float> turns[4] = {};
    const bool normed = a.weight != nullptr;
    if (normed)
      weights.Load(a.weight, lane);
    if (lane.pair >= 0) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        turns[i] = turns_of_row[lane.pair + i];
    }
    T *out = static_cast<T *>(a.out) + row * a.out_stride + head * D;
    typename Rows<T>::Most most;
    for (; left > 0; left -= Ahead) {
#pragma unroll
      for (int j = 0; j < Ahead; ++j) {
        if (j >= left)
          break;
        float x[8];
        Rows<T>::Unpack(raw[j].lo, x), Rows<T>::Unpack(raw[j].hi, x + 4);
        Fetch(j, head + Ahead * stride, lane);
        NormRotate<D, Interleaved>(x, lane, normed, weights, eps, turns);
        if (head < heads) {
          Eight<T> y;
          Rows<T>::Pack(x, &y.lo, &y.hi, &most);
          *reinterpret_cast<typename Rows<T>::Raw *>(out + lane.lo) = y.lo;
          *reinterpret_cast<typename Rows<T>::Raw *>(out + lane.hi) = y.hi;
        }
        head += stride, out += stride * D;
      }
    }
    if (!most.Finite())
      Raise(bad);
  }
};

// The units of a row are dealt to its `row_warps` warps in each of gridDim.y CTAs.
struct Share {
  int row, first, step; // row within the CTA
  __device__ __forceinline__ explicit Share(int row_warps) {
    const int warp = threadIdx.x >> 5;
    row = warp / row_warps, first = blockIdx.y * row_warps + warp % row_warps, step = row_warps * gridDim.y;
  }
};
__device__ __forceinline__ int After(int first, int units, int step) { // the first of first, first + step, ... behind `units`, counted from there
  return first >= units ? first - units : (first - units) % step + (((first - units) % step) ? step : 0);
}

// Three CTAs an SM at 80 registers with 20 bytes spilled; left to itself the compiler takes 89, for two (16384 rows: a call of 74 us instead of 68).
template <typename T, int D>
__global__ void __launch_bounds__(kRowThreads, sizeof(T) == 2 ? 3 : 2) NormRopeKernel(HeadRows q, HeadRows k, double eps, const int *positions, RotaryArgs rotary, int rows,
                                                              int row_warps, int *bad) {
  constexpr int kSide = 32 / (D / 8);
  __shared__ __align__(16) Turn<float> turns[kMaxCtaRows][D / 2];
  const int pairs = rotary.dims / 2, cta_rows = kRowWarps / row_warps;
  const int first = blockIdx.x * cta_rows, count = min(cta_rows, rows - first);
  const Lane lane = LaneOf<D>(rotary);
  const Share share(row_warps);
  const long long row = min(first + share.row, rows - 1); // a warp without a row reads the last one and stops
  UnitLoop<T, D, 4> q_loop(q, row, share.first, share.step, lane);
  for (int i = threadIdx.x; i < count * pairs; i += kRowThreads) {
    const int r = i / pairs, p = i - r * pairs;
    MakeTurn(Turns(positions[first + r], rotary.inv_freq[p]), rotary.amplitude, &turns[r][p]);
  }
  __syncthreads();
  if (share.row >= count)
    return;
  UnitLoop<T, D, 2> k_loop(k, row, After(share.first, (q.heads + kSide - 1) / kSide, share.step), share.step, lane);
  if (rotary.interleaved) {
    q_loop.template Run<true>(q, row, lane, eps, turns[share.row], bad);
    k_loop.template Run<true>(k, row, lane, eps, turns[share.row], bad);
  } else {
    q_loop.template Run<false>(q, row, lane, eps, turns[share.row], bad);
    k_loop.template Run<false>(k, row, lane, eps, turns[share.row], bad);
  }
}

// ---- append ----
// Measured: 64 rows of 32 + 4 + 4 heads of 128 in BF16 some 6 us, all latency (row -> sequence -> page, the table of cos and sin in 64 bits, the
// rows' loads under both); 6240 FP32 rows of 16 + 8 + 8 heads of 64 25 us.
// Norm and rotation of a key in 64 bits: the border between two codes is met by values that a 32-bit rotation could put on either side,
// and equal inputs have to give equal bytes.  `at` = the lane's place in the head; it holds eight neighbouring values, the partner of
// a rotated value is in the same lane (interleaved) or dims / 16 lanes on (half layout).  Every lane of the warp takes part.
template <int D>
__device__ __forceinline__ void NormRotateKey(double (&x)[8], int at, const unsigned short *weight, double eps, const Turn<double> *turns, int dims,
                                              bool interleaved) {
  if (weight) {
    double sum = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      sum += x[i] * x[i];
#pragma unroll
    for (int d = 1; d < D / 8; d *= 2)
      sum += __shfl_xor_sync(0xffffffffu, sum, d);
    const double inverse = 1.0 / sqrt(sum * (1.0 / D) + eps);
    const uint4 u = __ldg(reinterpret_cast<const uint4 *>(weight) + at);
    const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = x[2 * i] * inverse * static_cast<double>(__uint_as_float(w[i] << 16));
      x[2 * i + 1] = x[2 * i + 1] * inverse * static_cast<double>(__uint_as_float(w[i] & 0xffff0000u));
    }
  }
  if (interleaved) {
    if (8 * at < dims) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const Turn<double> t = turns[4 * at + i];
        const double a = x[2 * i], b = x[2 * i + 1];
        x[2 * i] = a * t.cos - b * t.sin;
        x[2 * i + 1] = a * t.sin + b * t.cos;
      }
    }
  } else if (dims) {
    const int half = dims / 16; // lanes between the two values of a pair
    const bool second = at >= half;
    const int lane = threadIdx.x & 31, from = at >= 2 * half ? lane : second ? lane - half : lane + half;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const double other = __shfl_sync(0xffffffffu, x[i], from);
      if (at < 2 * half) {
        const Turn<double> t = turns[8 * (second ? at - half : at) + i];
        x[i] = second ? other * t.sin + x[i] * t.cos : x[i] * t.cos - other * t.sin;
      }
    }
  }
}

// Adding and subtracting kInteger rounds to an integer, which is then in the sum's low bits.
template <typename Real> struct Rounding;
template <> struct Rounding<float> {
  static constexpr float kInteger = 12582912.f; // 1.5 * 2^23
  static __device__ __forceinline__ unsigned LowBits(float x) { return __float_as_uint(x) - 0x4b400000u; }
};
template <> struct Rounding<double> {
  static constexpr double kInteger = 6755399441055744.0; // 1.5 * 2^52
  static __device__ __forceinline__ unsigned LowBits(double x) { return static_cast<unsigned>(__double2loint(x)); }
};

// Eight values of a lane as eight codes, four lanes to a group.  The code is the nearest of x / scale, ties to even, as a division in 64
// bits would give it, without the division: a product with 1 / scale in 32 bits (its error is far below one half) gives an integer, and
// what is left of x, exact or rounded far below the difference between two inputs, tells whether that is the nearest one.
template <typename Real> __device__ __forceinline__ unsigned QuantiseWord(const Real (&x)[8], unsigned short *scale_bits, bool *fine) {
  Real most = 0;
  bool finite = true;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    most = max(most, abs(x[i]));
    finite &= isfinite(x[i]) != 0;
  }
#pragma unroll
  for (int d = 1; d < 4; d *= 2)
    most = max(most, __shfl_xor_sync(0xffffffffu, most, d));
  *fine = finite && most <= static_cast<Real>(kKvLargest);
  const __half h = __double2half(static_cast<double>(most) / 7.0);
  const float scale = __half2float(h), inverse = scale > 0 ? 1.f / scale : 0.f;
  const Real step = static_cast<Real>(scale), half = static_cast<Real>(0.5f * scale), factor = static_cast<Real>(inverse);
  Real worst = 0;
  unsigned word = 0x88888888u;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const Real sum = fma(x[i], factor, Rounding<Real>::kInteger), guess = sum - Rounding<Real>::kInteger;
    worst = max(worst, abs(fma(-guess, step, x[i])));
    word += Rounding<Real>::LowBits(sum) << (4 * i);
  }
  // a tie, a guess that is off by one, or a scale below FP16's normal range, of which there may be more than seven steps
  if (scale > 0 && (worst >= half || static_cast<float>(most) * inverse >= 7.5f)) {
    word = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float guess = fminf(fmaxf(rintf(static_cast<float>(x[i]) * inverse), -8.f), 8.f);
      const Real rest = fma(-static_cast<Real>(guess), step, x[i]);
      int code = static_cast<int>(guess);
      const bool odd = code & 1;
      code += (rest > half || (rest == half && odd)) - (rest < -half || (rest == -half && odd));
      word |= static_cast<unsigned>(min(max(code, -7), 7) + 8) << (4 * i);
    }
  }
  *scale_bits = __half_as_ushort(h);
  return word;
}

template <typename T, int D>
__global__ void __launch_bounds__(kRowThreads) AppendKernel(KvView cache, SequenceView seq, HeadRows q, HeadRows k, HeadRows v, double eps,
                                                            RotaryArgs rotary, int row_warps, int *bad) {
  constexpr int kLanes = D / 8, kSide = 32 / kLanes, kGroups = D / kKvGroup;
  __shared__ __align__(16) Turn<double> turns[kMaxCtaRows][D / 2];
  __shared__ __align__(16) Turn<float> q_turns[kMaxCtaRows][D / 2];
  __shared__ int s_page[kMaxCtaRows], s_position[kMaxCtaRows];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, pairs = rotary.dims / 2, cta_rows = kRowWarps / row_warps;
  const int first = blockIdx.x * cta_rows, count = min(cta_rows, seq.rows - first);
  const Share share(row_warps);
  const long long row = min(first + share.row, seq.rows - 1);
  const Lane q_lane = LaneOf<D>(rotary);
  UnitLoop<T, D, 2> q_loop(q, row, share.first, share.step, q_lane);
  const int kv_units = (k.heads + kSide - 1) / kSide, at = lane % kLanes;
  typename Rows<T>::Raw lo{}, hi{};
  auto fetch = [&](int unit) { // K and V as they come
    const HeadRows &a = unit < kv_units ? k : v;
    const int head = (unit < kv_units ? unit : unit - kv_units) * kSide + lane / kLanes;
    if (unit < 2 * kv_units && head < k.heads) {
      const T *const from = static_cast<const T *>(a.in) + row * a.stride + head * D + 8 * at;
      lo = *reinterpret_cast<const typename Rows<T>::Raw *>(from), hi = *reinterpret_cast<const typename Rows<T>::Raw *>(from + 4);
    }
  };
  int unit = After(share.first, (q.heads + kSide - 1) / kSide, share.step);
  fetch(unit);
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
    if (s_page[r] >= 0) {
      Turn<double> turn;
      MakeTurn(Turns(s_position[r], rotary.inv_freq[p]), rotary.amplitude, &turn);
      turns[r][p] = turn, q_turns[r][p] = Turn<float>{static_cast<float>(turn.cos), static_cast<float>(turn.sin)};
    }
  }
  __syncthreads();
  if (share.row >= count || s_page[share.row] < 0)
    return;
  if (rotary.interleaved)
    q_loop.template Run<true>(q, row, q_lane, eps, q_turns[share.row], bad);
  else
    q_loop.template Run<false>(q, row, q_lane, eps, q_turns[share.row], bad);
  const int slot = s_position[share.row] & (cache.page_size - 1), group = at / 4, quarter = at & 3;
  for (; unit < 2 * kv_units; unit += share.step) { // warp-uniform up to the head
    const bool is_v = unit >= kv_units;
    const int head = (is_v ? unit - kv_units : unit) * kSide + lane / kLanes;
    const bool there = head < k.heads;
    float x[8] = {};
    if (there)
      Rows<T>::Unpack(lo, x), Rows<T>::Unpack(hi, x + 4);
    fetch(unit + share.step);
    unsigned short scale;
    bool fine;
    unsigned word;
    if (is_v) { // 24 bits at most: a multiple of half a scale is exact in 32
      word = QuantiseWord(x, &scale, &fine);
    } else {
      double y[8];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        y[j] = static_cast<double>(x[j]);
      NormRotateKey<D>(y, at, k.weight, eps, turns[share.row], rotary.dims, rotary.interleaved);
      word = QuantiseWord(y, &scale, &fine);
    }
    // one decision for the whole head: it is written or left as it was
    const unsigned lanes = (kLanes == 32 ? 0xffffffffu : (1u << kLanes) - 1) << (lane / kLanes * kLanes);
    const bool whole = (__ballot_sync(0xffffffffu, !fine) & lanes) == 0;
    if (!there)
      continue;
    if (!whole) {
      Raise(bad);
      continue;
    }
    unsigned char *codes = cache.block(s_page[share.row], head) + (is_v ? cache.code_bytes() + cache.scale_bytes() : 0);
    reinterpret_cast<unsigned *>(codes + slot * (D / 2))[quarter * kGroups + group] = word;
    if (!quarter)
      reinterpret_cast<unsigned short *>(codes + cache.code_bytes() + slot * (D / 16))[group] = scale;
  }
}

// ---- read ----
// Bound by latency (each row is looked up by itself) and by what the rows take to write: 12872 rows of 8 heads of 64 as FP32 in 11 us.  A warp takes one row; a lane one word (eight codes) of K and of V of one head at a time, two of each with all loads first.
template <typename T, int D>
__global__ void __launch_bounds__(kRowThreads) ReadKernel(KvView cache, SequenceView seq, T *k_out, T *v_out, long long k_stride, long long v_stride,
                                                          int *bad) {
  constexpr int kWords = D / 8, kGroups = D / kKvGroup, kFlight = 4;
  const int lane = threadIdx.x & 31, row = blockIdx.x * kRowWarps + (threadIdx.x >> 5);
  if (row >= seq.rows)
    return;
  int position = -1;
  const int s = LocateRow(seq, cache, row, &position, bad);
  const int page = s >= 0 && position >= 0 ? PageOf(seq, cache, s, position, bad) : -1;
  if (page < 0)
    return;
  const int words = cache.kv_heads * kWords, block_bytes = cache.block_bytes(), second = cache.code_bytes() + cache.scale_bytes();
  const int slot = position & (cache.page_size - 1), at = lane % kWords, group = at / 4, place = (at & 3) * kGroups + group;
  const unsigned char *const codes = cache.block(page, 0) + slot * (D / 2) + 4 * place;
  const unsigned char *const scales = cache.block(page, 0) + cache.code_bytes() + slot * (D / 16) + 2 * group;
  typename Rows<T>::Most most;
  for (int j0 = lane; j0 < words; j0 += 16 * kFlight) {
    unsigned word[kFlight];
    unsigned short scale[kFlight];
#pragma unroll
    for (int i = 0; i < kFlight; ++i) { // K and V in turn; word j of the row is word `at` of head j / kWords
      const int j = j0 + i / 2 * 32;
      if (j < words) {
        const long long offset = static_cast<long long>(j / kWords) * block_bytes + i % 2 * second;
        word[i] = *reinterpret_cast<const unsigned *>(codes + offset);
        scale[i] = *reinterpret_cast<const unsigned short *>(scales + offset);
      }
    }
#pragma unroll
    for (int i = 0; i < kFlight; ++i) {
      const int j = j0 + i / 2 * 32;
      if (j < words) {
        const float step = HalfBitsToFloat(scale[i]);
        float x[8];
#pragma unroll
        for (int n = 0; n < 8; ++n) // 2^23 + code as a float's bits, less 2^23 + 8
          x[n] = (__uint_as_float(0x4b000000u | (word[i] >> (4 * n) & 15u)) - 8388616.f) * step;
        T *const out = (i % 2 ? v_out + row * v_stride : k_out + row * k_stride) + 8 * j;
        Eight<T> y;
        Rows<T>::Pack(x, &y.lo, &y.hi, &most);
        if constexpr (sizeof(T) == 2) {
          *reinterpret_cast<uint4 *>(out) = make_uint4(y.lo.x, y.lo.y, y.hi.x, y.hi.y);
        } else {
          *reinterpret_cast<float4 *>(out) = y.lo, *reinterpret_cast<float4 *>(out + 4) = y.hi;
        }
      }
    }
  }
  if (!most.Finite())
    Raise(bad);
}

// Warps per row and CTAs per row: a warp takes a row whole where that fills the SMs twice over (16384 rows of 36 heads: 64 us, against
// 72 us with two warps to a row, since fewer warps wait for tables); few rows are spread over the SMs by splitting their
// heads, one unit per warp at the least.
void Shape(int rows, int units, int *row_warps, dim3 *grid) {
  const int cta_rows = rows >= 2 * 148 * kMaxCtaRows ? kMaxCtaRows : rows >= 4 * 148 ? 4 : 1;
  *row_warps = kRowWarps / cta_rows;
  const int x = (rows + cta_rows - 1) / cta_rows, most = (units + *row_warps - 1) / *row_warps;
  int parts = cta_rows > 1 ? 1 : (2 * 148 + x - 1) / x;
  *grid = dim3(x, parts < 1 ? 1 : parts > most ? most : parts);
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
    int row_warps;
    dim3 grid;
    Shape(rows, (q.heads + kSide - 1) / kSide + (k.heads + kSide - 1) / kSide, &row_warps, &grid);
    NormRopeKernel<T, D><<<grid, kRowThreads, 0, stream>>>(q, k, eps, positions, rotary, rows, row_warps, bad);
    return CudaStatus(cudaGetLastError());
  }
};
template <typename T, int D> struct Append {
  static constexpr int kWidest = 128;
  static int Run(const KvView &cache, const SequenceView &seq, const HeadRows &q, const HeadRows &k, const HeadRows &v, double eps,
                 const RotaryArgs &rotary, int *bad, cudaStream_t stream) {
    constexpr int kSide = 32 / (D / 8);
    int row_warps;
    dim3 grid;
    Shape(seq.rows, (q.heads + kSide - 1) / kSide + 2 * ((k.heads + kSide - 1) / kSide), &row_warps, &grid);
    AppendKernel<T, D><<<grid, kRowThreads, 0, stream>>>(cache, seq, q, k, v, eps, rotary, row_warps, bad);
    return CudaStatus(cudaGetLastError());
  }
};
template <typename T, int D> struct Read {
  static constexpr int kWidest = 128;
  static int Run(const KvView &cache, const SequenceView &seq, void *k_out, void *v_out, long long k_stride, long long v_stride, int *bad,
                 cudaStream_t stream) {
    ReadKernel<T, D><<<(seq.rows + kRowWarps - 1) / kRowWarps, kRowThreads, 0, stream>>>(cache, seq, static_cast<T *>(k_out), static_cast<T *>(v_out),
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
      !RotaryOk(rotary, head_dim, &r) || (r.dims && rows && !positions) || !WeightOk(q_weight) || !WeightOk(k_weight))
    return PADRA_INVALID_ARGUMENT;
  if (head_dim != 64 && head_dim != 128 && head_dim != 256)
    return PADRA_UNSUPPORTED;
  if (!RowsOk(q, q_stride, rows, q_heads, head_dim) || !RowsOk(q_out, q_out_stride, rows, q_heads, head_dim) ||
      (k_heads && (!RowsOk(k, k_stride, rows, k_heads, head_dim) || !RowsOk(k_out, k_out_stride, rows, k_heads, head_dim))))
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
  if (!RowsOk(k, k_stride, s.rows, c.kv_heads, c.head_dim) || !RowsOk(v, v_stride, s.rows, c.kv_heads, c.head_dim))
    return PADRA_INVALID_ARGUMENT;
  if (q && (q_heads < 1 || q_heads > 4096 || !RowsOk(q, q_stride, s.rows, q_heads, c.head_dim) || !RowsOk(q_out, q_out_stride, s.rows, q_heads, c.head_dim)))
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
  if (!RowsOk(k_out, k_stride, s.rows, c.kv_heads, c.head_dim) || !RowsOk(v_out, v_stride, s.rows, c.kv_heads, c.head_dim))
    return PADRA_INVALID_ARGUMENT;
  if (!s.rows || !s.count)
    return PADRA_OK;
  return ByTypeAndDim<Read>(type, c.head_dim, c, s, k_out, v_out, k_stride, v_stride, bad, stream);
}

} // namespace padra
