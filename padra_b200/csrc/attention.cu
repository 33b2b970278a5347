// Attention over the paged 4-bit cache for few query rows per sequence: out = softmax(scale * q k^T + mask) v.
//
// With one row and G heads to a KV head there are G dot products per cached value: bound by the cache's bytes, if the codes
// become tensor-core operands cheaply enough.
//   * Work is (sequence, KV head, block of 8 * NT query columns) x 32-token tiles.  All tiles of a call form one list, and
//     every CTA takes an equal run of it (ends may lie inside a sequence), so neither one long context nor ragged ones
//     leave SMs idle.  A run's piece of a unit that is not the whole unit leaves maximum, sum and unnormalised output in the
//     workspace, and a second kernel, launched as a programmatic dependent, joins the pieces in list order (as the last
//     CTA's task inside the first kernel that cost fences, tickets, and up to 25 us where one CTA read a hundred pieces).
//   * A warp owns tiles w, w + 4, ... of the CTA's run, with a private ring of tiles filled by cp.async: no barrier between
//     warps until the piece ends.
//   * Scores: K is the MMA's A operand (16 tokens x 16 values), queries the B columns.  A lane's word holds eight codes of one
//     group, and two MMAs cover a group of 32 values, so the FP16 scale of (token, group) is applied to the group's
//     FP32 sum.  A code becomes an FP16 number by inserting it into the mantissa of 1024 (low nibble) or 64 (high nibble), one
//     logic operation for two codes; the offsets (1032, 72) times the query are subtracted through the accumulator's
//     initial value, which costs some eight of its 24 bits: scores are off by about 2^-16 of sum |q k|, 2^-14 at the most.
//   * Output: V^T is the A operand (16 values x 16 tokens).  ldmatrix.trans on 16-bit pieces hands a lane four codes of two
//     neighbouring tokens in one register, which is where the MMA wants a pair; offset and scale are applied as FP16 (codes
//     and offsets exact, the product rounded once, 2^-11).  Weights go from the score layout to the B operand with one 8x8
//     transpose (movmatrix) per eight tokens.
//   * The running maximum is only raised when a weight would pass 2^15 (weights are FP16, at least 2^8 for the largest
//     after a raise): a warp vote per tile instead of a reduction.
// Measured: 64 sequences of 1 to 16384 tokens, 32 heads over 4, head size 128: 81 us, 3.8 TB/s of codes and scales (58% of a copy): 168
// registers allow 11 warps an SM, whose chains of dependent instructions fill 59% of the issue slots.  One sequence of 131072 tokens: 24 us and
// 7 us for the join; of 4097: 13 us, all latency.
#include <cmath>
#include <mutex>
#include <type_traits>

#include "attention.cuh"

namespace padra {
namespace {

using namespace attention;

// Small CTAs, as many to an SM as the registers of a column block leave room for: what a CTA does between two pieces
// (queries, joining its warps) runs under the others' tiles.
constexpr int kWarps = 4, kThreads = kWarps * 32;
template <int NT> struct Cta {
  static constexpr int kPerSm = NT == 1 ? 3 : 2;
};
constexpr int kTile = 32;   // tokens of a tile
constexpr int kStages = 4;  // tiles of a warp's ring

__device__ __forceinline__ void CopyAsync16(unsigned to, const void *from, int bytes) { // the rest of the 16 bytes becomes zero
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ void MmaF16(float (&d)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// What one sequence asks for: `blocks` column blocks of each KV head, `tiles` tiles for each of them, the first being tile
// `first` of the sequence.  A sequence without rows, or one whose numbers contradict the call, has no work; rows that see
// nothing still get one (empty) tile, so that their zeros are written.
struct Demand {
  int begin, rows, context, first, tiles, blocks;
};
template <int Columns> __device__ __forceinline__ Demand DemandOf(const AttentionArgs &a, int s) {
  Demand d{};
  if (!SequenceRows(a.seq, a.cache, s, &d.begin, &d.rows, &d.context, a.bad) || !d.rows)
    return d;
  const int low = a.window ? max(0, d.context - d.rows + 1 - a.window) : 0;
  d.first = low / kTile;
  d.tiles = max(1, (d.context + kTile - 1) / kTile - d.first);
  d.blocks = (d.rows * a.group + Columns - 1) / Columns;
  return d;
}
__device__ __forceinline__ long long CostOf(const AttentionArgs &a, const Demand &d) {
  return static_cast<long long>(d.tiles) * d.blocks * a.cache.kv_heads;
}

template <int D> struct TileBytes {
  static constexpr int kCodes = kTile * D / 2, kScales = kTile * D / 16, kAll = 2 * (kCodes + kScales);
};

// One piece: tiles [from, from + count) of a unit, `base` tiles into the sequence.
template <typename T, int D, int NT> struct Piece {
  static constexpr int kGroups = D / kKvGroup, kChunks = D / 32, kColumns = 8 * NT;
  static constexpr int kRow = D + 4; // floats of a column's row in shared memory while warps are joined
  // FP16 rows are rounded by 2^-11 themselves, so that the weights' own rounding shows beside it: what it leaves off goes through a second
  // MMA (error against 64 bits 0.00028 instead of 0.00033, the output's rounding alone 0.00021).  BF16 rows hide it.
  static constexpr bool kRests = std::is_same<T, __half>::value;

  // column -> row of the sequence and head of the group
  static __device__ __forceinline__ void Run(const AttentionArgs &a, const Demand &d, int s, int head, int block, int first_tile, int count,
                                             unsigned char *ring, float *join, float *join_ml, int2 (*cta_limits)[kColumns]) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
    int2 *const limits = cta_limits[warp]; // first and last token that a column sees
    const int columns = min(kColumns, d.rows * a.group - block * kColumns);
    const int start = d.context - d.rows; // position of the sequence's first row

    uint4 raw[NT][kGroups]; // on their way while the first tiles are asked for
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int column = 8 * n + g, place = block * kColumns + column, row = place / a.group, h = head * a.group + place % a.group;
#pragma unroll
      for (int i = 0; i < kGroups; ++i)
        raw[n][i] = column < columns && start + row >= 0
                        ? *reinterpret_cast<const uint4 *>(static_cast<const T *>(a.q) + static_cast<long long>(d.begin + row) * a.q_stride + h * D + 32 * i + 8 * c)
                        : make_uint4(0, 0, 0, 0);
    }

    // ---- the ring ----
    const int mine = count > warp ? (count - warp + kWarps - 1) / kWarps : 0; // tiles of this warp: warp, warp + kWarps, ...
    const int visible_low = a.window ? max(0, start + 1 - a.window) : 0;
    unsigned char *const own_ring = ring + warp * kStages * TileBytes<D>::kAll;
    const unsigned ring_address = SmemAddress(own_ring);
    // a warp-wide copy takes 512 bytes of codes: 16 per lane, V's swizzled inside the token's row
    const int code_scale_bytes = a.cache.code_bytes() + a.cache.scale_bytes(), copy_token = lane / kChunks, copy_chunk = lane % kChunks;
    const unsigned copy_offset = 16 * lane,
                   swizzled_offset = TileBytes<D>::kCodes + TileBytes<D>::kScales + copy_token * (D / 2) +
                                     16 * (kChunks == 4 ? copy_chunk ^ ((copy_token >> 1) & 3) : copy_chunk ^ ((copy_token >> 2) & 1));
    constexpr int kScaleTokens = 256 / D, kScaleLanes = kTile / kScaleTokens; // tokens whose scales fill 16 bytes; lanes for K, as many for V
    const int scale_of_v = lane / kScaleLanes, scale_from = a.cache.code_bytes() + scale_of_v * code_scale_bytes;
    const unsigned scale_offset = TileBytes<D>::kCodes + scale_of_v * (TileBytes<D>::kCodes + TileBytes<D>::kScales) + 16 * (lane % kScaleLanes);
    int page_low = -1, page_high = -1; // of this lane's tile among the next 32: first and second 16 tokens
    auto fetch = [&](int i) {
      if (i < mine) {
        if ((i & 31) == 0) {
          const int t = (first_tile + warp + (i + lane) * kWarps) * kTile;
          page_low = page_high = -1;
          if (i + lane < mine && t < d.context) {
            if (a.cache.page_size > 16) {
              page_low = page_high = PageOf(a.seq, a.cache, s, t, a.bad);
            } else {
              if (t + 16 > visible_low)
                page_low = PageOf(a.seq, a.cache, s, t, a.bad);
              if (t + 16 < d.context)
                page_high = PageOf(a.seq, a.cache, s, t + 16, a.bad);
            }
          }
        }
        const int lo = __shfl_sync(0xffffffffu, page_low, i & 31), hi = __shfl_sync(0xffffffffu, page_high, i & 31);
        const int t0 = (first_tile + warp + i * kWarps) * kTile;
        // first token of either half of the tile; a half without a page reads page 0's and gets scales of zero
        const int slot = t0 & (a.cache.page_size - 1), slot_high = (t0 + 16) & (a.cache.page_size - 1);
        const unsigned char *const from_low = a.cache.block(max(lo, 0), head), *const from_high = a.cache.block(max(hi, 0), head);
        const unsigned to = ring_address + (i & (kStages - 1)) * TileBytes<D>::kAll;
        constexpr int kRowsPerCopy = 32 / kChunks, kCopies = kTile / kRowsPerCopy; // tokens per warp-wide copy
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const unsigned char *const from = (h ? from_high + slot_high * (D / 2) : from_low + slot * (D / 2)) + 16 * lane;
          const unsigned char *const from_v = from + code_scale_bytes;
#pragma unroll
          for (int k = h * kCopies / 2; k < (h + 1) * kCopies / 2; ++k) {
            CopyAsync16(to + copy_offset + k * 512, from + (k - h * kCopies / 2) * 512, 16);
            CopyAsync16(to + swizzled_offset + k * 512, from_v + (k - h * kCopies / 2) * 512, 16);
          }
        }
        if (lane < 2 * kScaleLanes) {
          const int t = lane % kScaleLanes * kScaleTokens;
          const int valid = (t >= 16 ? hi : lo) < 0 ? 0 : max(0, min(kScaleTokens, d.context - t0 - t));
          const unsigned char *const from = t >= 16 ? from_high + (slot_high + t - 16) * (D / 16) : from_low + (slot + t) * (D / 16);
          CopyAsync16(to + scale_offset, from + scale_from, valid * (D / 16));
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i)
      fetch(i);

    // ---- queries: FP16 after division by a power of two that brings the row's largest value below 2 ----
    unsigned q[NT][kGroups][4];
    float factor[NT][2], correction[NT][kGroups][2];
    int least = 0x7fffffff, latest_low = 0;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int column = 8 * n + g, place = block * kColumns + column, row = place / a.group;
      float x[kGroups][8], most = 0;
      bool finite = true;
#pragma unroll
      for (int i = 0; i < kGroups; ++i) {
        Widen(raw[n][i], static_cast<const T *>(nullptr), x[i]);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          finite &= isfinite(x[i][j]) != 0;
          most = fmaxf(most, fabsf(x[i][j]));
        }
      }
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
      const bool fine = (__ballot_sync(0xffffffffu, !finite) & (0xfu << (lane & 28))) == 0;
      if (!fine)
        Raise(a.bad);
      const int exponent = most > 0 && fine ? min(126, max(-126, ilogbf(most))) : 0;
      const float shrink = fine ? ldexpf(1.f, -exponent) : 0.f;
      float sums[kGroups];
#pragma unroll
      for (int i = 0; i < kGroups; ++i) {
        float y[8], sum = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          y[j] = fine ? __half2float(__float2half_rn(x[i][j] * shrink)) * a.sign : 0.f;
          sum += y[j] * (j & 1 ? -72.f : -1032.f);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
          q[n][i][j] = Pack(y[j], y[j + 4]);
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sums[i] = sum + __shfl_xor_sync(0xffffffffu, sum, 2);
      }
      const float mine = FactorOf(a.scale, ldexpf(1.f, exponent));
      // a row at a negative position sees nothing, nor does one that is not finite, nor a column beyond the last
      const int to = column < columns && fine ? start + row : -1, from = a.window ? max(0, to - a.window + 1) : 0;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int owner = 4 * (2 * c + e);
        factor[n][e] = __shfl_sync(0xffffffffu, mine, owner);
#pragma unroll
        for (int i = 0; i < kGroups; ++i)
          correction[n][i][e] = __shfl_sync(0xffffffffu, sums[i], owner);
      }
      if (column < columns)
        least = min(least, to), latest_low = max(latest_low, from);
      if (c == 0)
        limits[column] = make_int2(from, to);
    }
#pragma unroll
    for (int m = 4; m < 32; m *= 2) {
      least = min(least, __shfl_xor_sync(0xffffffffu, least, m));
      latest_low = max(latest_low, __shfl_xor_sync(0xffffffffu, latest_low, m));
    }

    __syncwarp();

    float top[NT][2], sum[NT][2], o[NT][2 * kChunks][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      top[n][0] = top[n][1] = kNever, sum[n][0] = sum[n][1] = 0;
#pragma unroll
      for (int t = 0; t < 2 * kChunks; ++t)
        o[n][t][0] = o[n][t][1] = o[n][t][2] = o[n][t][3] = 0;
    }

    for (int i = 0; i < mine; ++i) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
      __syncwarp(); // the tile is here for every lane, and nobody reads the slot that is filled next
      fetch(i + kStages - 1);
      const unsigned tile = ring_address + (i & (kStages - 1)) * TileBytes<D>::kAll;
      const int t0 = (first_tile + warp + i * kWarps) * kTile;
      const bool edge = t0 + kTile - 1 > least || t0 < latest_low;
      if (t0 < visible_low) { // tokens before every row's window may hold anything: a weight of zero does not make a NaN vanish
        if (t0 + lane < visible_low)
          for (int which = 0; which < 2; ++which)
            for (int x = 0; x < D / 16; x += 4)
              asm volatile("st.shared.b32 [%0], %1;" ::"r"(tile + which * (TileBytes<D>::kCodes + TileBytes<D>::kScales) + TileBytes<D>::kCodes + lane * (D / 16) + x), "r"(0) : "memory");
        __syncwarp();
      }

      float score[2][NT][4];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        unsigned w[2][kGroups];
        float f[2][kGroups];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int token = 16 * half + 8 * r + g;
          if constexpr (kGroups == 4) {
            const uint4 u = LoadShared16(tile + token * (D / 2) + 16 * c);
            w[r][0] = u.x, w[r][1] = u.y, w[r][2] = u.z, w[r][3] = u.w;
            const uint2 v = LoadShared8(tile + TileBytes<D>::kCodes + token * (D / 16));
            const float2 f0 = __half22float2(*reinterpret_cast<const __half2 *>(&v.x)), f1 = __half22float2(*reinterpret_cast<const __half2 *>(&v.y));
            f[r][0] = f0.x, f[r][1] = f0.y, f[r][2] = f1.x, f[r][3] = f1.y;
          } else {
            const uint2 u = LoadShared8(tile + token * (D / 2) + 8 * c);
            w[r][0] = u.x, w[r][1] = u.y;
            const unsigned v = LoadShared4(tile + TileBytes<D>::kCodes + token * (D / 16));
            const float2 f0 = __half22float2(*reinterpret_cast<const __half2 *>(&v));
            f[r][0] = f0.x, f[r][1] = f0.y;
          }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
          score[half][n][0] = score[half][n][1] = score[half][n][2] = score[half][n][3] = 0;
#pragma unroll
        for (int k = 0; k < kGroups; ++k) {
          const unsigned u0 = w[0][k], u1 = w[1][k], v0 = u0 >> 8, v1 = u1 >> 8;
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            float acc[4] = {correction[n][k][0], correction[n][k][1], correction[n][k][0], correction[n][k][1]};
            MmaF16(acc, Low(u0, a.masks), Low(u1, a.masks), High(u0, a.masks), High(u1, a.masks), q[n][k][0], q[n][k][1]);
            MmaF16(acc, Low(v0, a.masks), Low(v1, a.masks), High(v0, a.masks), High(v1, a.masks), q[n][k][2], q[n][k][3]);
            score[half][n][0] += acc[0] * f[0][k], score[half][n][1] += acc[1] * f[0][k];
            score[half][n][2] += acc[2] * f[1][k], score[half][n][3] += acc[3] * f[1][k];
          }
        }
      }
      if (edge) { // tokens that some column does not see
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int t = t0 + 16 * half + 8 * (e >> 1) + g;
              const int2 seen = limits[8 * n + 2 * c + (e & 1)];
              if (t < seen.x || t > seen.y)
                score[half][n][e] = -INFINITY;
            }
      }
      float most[NT][2], over = kNever; // largest score of a column, and by how much log2 of a weight is largest
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          most[n][e] = fmaxf(fmaxf(score[0][n][e], score[0][n][e + 2]), fmaxf(score[1][n][e], score[1][n][e + 2]));
          over = fmaxf(over, fmaf(most[n][e], factor[n][e], -top[n][e]));
        }
      if (__any_sync(0xffffffffu, over > kRaise)) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float x = most[n][e];
#pragma unroll
            for (int m = 4; m < 32; m *= 2)
              x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, m));
            const float next = fmaxf(top[n][e], fmaf(x, factor[n][e], -kTop)), shrink = Exp2(top[n][e] - next);
            if (next > kNever && fabsf(next) > kLargestTop)
              Raise(a.bad);
            top[n][e] = next, sum[n][e] *= shrink;
#pragma unroll
            for (int t = 0; t < 2 * kChunks; ++t)
              o[n][t][e] *= shrink, o[n][t][e + 2] *= shrink;
          }
      }
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        // weights, transposed from (token, column) to (column, token)
        unsigned p[NT][2], rest[kRests ? NT : 1][2];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const float p0 = Exp2(fmaf(score[half][n][2 * r], factor[n][0], -top[n][0])),
                        p1 = Exp2(fmaf(score[half][n][2 * r + 1], factor[n][1], -top[n][1]));
            sum[n][0] += p0, sum[n][1] += p1;
            const unsigned weights = Pack(p0, p1);
            asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(p[n][r]) : "r"(weights));
            if constexpr (kRests) {
              const float2 rounded = __half22float2(*reinterpret_cast<const __half2 *>(&weights));
              asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(rest[n][r]) : "r"(Pack(p0 - rounded.x, p1 - rounded.y)));
            }
          }
        // V's scales of tokens 2c, 2c + 1 and 2c + 8, 2c + 9 in this lane's group
        const unsigned values = tile + TileBytes<D>::kCodes + TileBytes<D>::kScales;
        const unsigned f = values + TileBytes<D>::kCodes + 2 * ((16 * half + 2 * c) * kGroups + (g >> 1) % kGroups);
        __half2 scale[2];
#pragma unroll
        for (int r = 0; r < 2; ++r)
          scale[r] = __halves2half2(__ushort_as_half(LoadShared2(f + 16 * r * kGroups)), __ushort_as_half(LoadShared2(f + (16 * r + 2) * kGroups)));
#pragma unroll
        for (int j = 0; j < kChunks; j += 2) {
          // four 8x8 matrices of 16-bit pieces: tokens 0..7 and 8..15 of chunk j, then of chunk j + 1
          unsigned v[4];
          const int token = lane & 15, chunk = j + (lane >> 4);
          const int swizzled = kChunks == 4 ? chunk ^ ((token >> 1) & 3) : chunk ^ ((token >> 2) & 1);
          asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                       : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
                       : "r"(values + (16 * half + token) * (D / 2) + 16 * swizzled)
                       : "memory");
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const unsigned u0 = v[2 * k], u1 = v[2 * k + 1], w0 = u0 >> 8, w1 = u1 >> 8;
            const unsigned a0 = Scaled(Low(u0, a.masks), 0x64086408u, scale[0]), a1 = Scaled(High(u0, a.masks), 0x54805480u, scale[0]);
            const unsigned a2 = Scaled(Low(u1, a.masks), 0x64086408u, scale[1]), a3 = Scaled(High(u1, a.masks), 0x54805480u, scale[1]);
            const unsigned b0 = Scaled(Low(w0, a.masks), 0x64086408u, scale[0]), b1 = Scaled(High(w0, a.masks), 0x54805480u, scale[0]);
            const unsigned b2 = Scaled(Low(w1, a.masks), 0x64086408u, scale[1]), b3 = Scaled(High(w1, a.masks), 0x54805480u, scale[1]);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              MmaF16(o[n][2 * (j + k)], a0, a1, a2, a3, p[n][0], p[n][1]);
              MmaF16(o[n][2 * (j + k) + 1], b0, b1, b2, b3, p[n][0], p[n][1]);
              if constexpr (kRests) {
                MmaF16(o[n][2 * (j + k)], a0, a1, a2, a3, rest[n][0], rest[n][1]);
                MmaF16(o[n][2 * (j + k) + 1], b0, b1, b2, b3, rest[n][0], rest[n][1]);
              }
            }
          }
        }
      }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");

    // ---- the warps' maxima, sums and outputs to shared memory (over the rings: every warp is done with its own) ----
    __syncthreads();
    if (mine || warp == 0) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float x = sum[n][e];
#pragma unroll
          for (int m = 4; m < 32; m *= 2)
            x += __shfl_xor_sync(0xffffffffu, x, m);
          const int column = 8 * n + 2 * c + e;
          if (g == 0)
            join_ml[(warp * kColumns + column) * 2] = top[n][e], join_ml[(warp * kColumns + column) * 2 + 1] = x;
          float *const to = join + (warp * kColumns + column) * kRow;
#pragma unroll
          for (int t = 0; t < 2 * kChunks; ++t)
#pragma unroll
            for (int r = 0; r < 2; ++r) { // chunk t / 2, nibble 2 (t % 2) + r of piece g
              const int word = 4 * (t / 2) + (g >> 1), dim = 32 * (word % kGroups) + 8 * (word / kGroups) + 4 * (g & 1) + 2 * (t & 1) + r;
              to[dim] = o[n][t][e + 2 * r];
            }
        }
    }
    __syncthreads();
  }

  // Joins the CTA's warps: join_ml becomes the weight of every (warp, column), ml the column's maximum and sum.
  static __device__ __forceinline__ void Weigh(float *join_ml, float2 *ml, int warps, int columns) {
    const int column = threadIdx.x;
    if (column < columns) {
      float m = kNever, l = 0, f[kWarps];
#pragma unroll
      for (int w = 0; w < kWarps; ++w)
        m = fmaxf(m, w < warps ? join_ml[(w * kColumns + column) * 2] : kNever);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        f[w] = w < warps ? Exp2(join_ml[(w * kColumns + column) * 2] - m) : 0.f;
        l += w < warps ? f[w] * join_ml[(w * kColumns + column) * 2 + 1] : 0.f;
      }
#pragma unroll
      for (int w = 0; w < kWarps; ++w)
        join_ml[(w * kColumns + column) * 2] = f[w];
      ml[column] = make_float2(m, l);
    }
    __syncthreads();
  }
  static __device__ __forceinline__ float4 Joined(const float *join, const float *join_ml, int warps, int column, int dim) {
    float4 v = make_float4(0, 0, 0, 0);
#pragma unroll
    for (int w = 0; w < kWarps; ++w)
      if (w < warps) {
        const float f = join_ml[(w * kColumns + column) * 2];
        const float4 x = *reinterpret_cast<const float4 *>(join + (w * kColumns + column) * kRow + dim);
        v.x += f * x.x, v.y += f * x.y, v.z += f * x.z, v.w += f * x.w;
      }
    return v;
  }
};

template <typename T, int D, int NT> __global__ void __launch_bounds__(kThreads, Cta<NT>::kPerSm) SplitAttentionKernel(const __grid_constant__ AttentionArgs a) {
  using P = Piece<T, D, NT>;
  constexpr int kColumns = P::kColumns;
  extern __shared__ __align__(128) unsigned char ring[];
  __shared__ float join_ml[kWarps * kColumns * 2];
  __shared__ int2 limits[kWarps][kColumns];
  __shared__ long long scan[kWarps], s_offset;
  __shared__ float2 s_ml[kColumns];
  __shared__ Demand s_demand;
  __shared__ int s_sequence;
  float *const join = reinterpret_cast<float *>(ring);
  const int tid = threadIdx.x;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); // the joining kernel fills SMs as CTAs leave

  // ---- this CTA's run of the list: every CTA adds up the same demands, one sequence per thread at a time ----
  Demand mine{};
  long long total = 0, at_mine = 0, cost_mine = 0;
  for (int s0 = 0; s0 < a.seq.count; s0 += kThreads) {
    long long part;
    mine = s0 + tid < a.seq.count ? DemandOf<kColumns>(a, s0 + tid) : Demand{};
    cost_mine = CostOf(a, mine);
    at_mine = total + BlockPrefix<kWarps>(cost_mine, scan, &part);
    total += part;
  }
  // at least one tile for every warp: shorter runs only make more pieces to join
  const long long share = max(static_cast<long long>(kWarps), Quotient(total + gridDim.x - 1, gridDim.x));
  const long long begin = blockIdx.x * share, end = min(total, begin + share);
  if (tid == 0)
    a.split[blockIdx.x].pieces = 0;
  if (begin >= end)
    return;
  if (a.seq.count <= kThreads) { // the demands are still in the threads' registers
    if (begin >= at_mine && begin < at_mine + cost_mine)
      s_sequence = tid, s_offset = begin - at_mine, s_demand = mine;
  } else {
    long long before = 0;
    for (int s0 = 0; s0 < a.seq.count && before <= begin; s0 += kThreads) {
      long long part;
      mine = s0 + tid < a.seq.count ? DemandOf<kColumns>(a, s0 + tid) : Demand{};
      cost_mine = CostOf(a, mine);
      at_mine = before + BlockPrefix<kWarps>(cost_mine, scan, &part);
      if (begin >= at_mine && begin < at_mine + cost_mine)
        s_sequence = s0 + tid, s_offset = begin - at_mine, s_demand = mine;
      before += part;
    }
  }
  __syncthreads();
  int s = s_sequence;
  long long offset = s_offset; // tiles into sequence s
  Demand d = s_demand;
  for (long long at = begin; at < end;) {
    while (offset >= CostOf(a, d)) { // next sequence with work
      offset -= CostOf(a, d);
      d = DemandOf<kColumns>(a, ++s);
    }
    const long long unit = Quotient(offset, d.tiles);
    const int skip = static_cast<int>(offset - unit * d.tiles), head = static_cast<int>(Quotient(unit, d.blocks)), block = static_cast<int>(unit - static_cast<long long>(head) * d.blocks);
    const int count = static_cast<int>(min(static_cast<long long>(d.tiles - skip), end - at));
    P::Run(a, d, s, head, block, d.first + skip, count, ring, join, join_ml, limits);
    const int warps = min(count, kWarps), columns = min(kColumns, d.rows * a.group - block * kColumns);
    P::Weigh(join_ml, s_ml, warps, columns);
    const bool whole = count == d.tiles;
    const int slot = at == begin ? 0 : 1;
    for (int i = tid; i < columns * (D / 4); i += kThreads) {
      const int column = i / (D / 4), dim = i % (D / 4) * 4;
      const float4 v = P::Joined(join, join_ml, warps, column, dim);
      if (whole) {
        StoreOutput<T, D, kColumns>(a, d.begin, block, head, column, dim, v, s_ml[column].y);
      } else {
        float *const to = PartialOf<D, kColumns>(a, blockIdx.x, slot);
        *reinterpret_cast<float4 *>(to + column * D + dim) = v;
        if (dim == 0)
          *reinterpret_cast<float2 *>(to + kColumns * D + 2 * column) = s_ml[column];
      }
    }
    if (!whole && !skip && tid == 0) { // only the last unit of a run can go on in the next
      const long long last = Quotient(at + d.tiles - 1, share);
      a.split[blockIdx.x] = Split{static_cast<int>(last - blockIdx.x) + 1, slot, d.begin, block, head, columns};
    }
    __syncthreads(); // the rings are free again
    at += count, offset += count;
  }
}

template <typename T, int D, int NT> int LaunchSplit(AttentionArgs a, int sms, cudaStream_t stream) {
  using P = Piece<T, D, NT>;
  constexpr size_t kRing = static_cast<size_t>(kWarps) * kStages * TileBytes<D>::kAll, kJoin = sizeof(float) * kWarps * P::kColumns * P::kRow;
  constexpr size_t kSmem = kRing > kJoin ? kRing : kJoin;
  if (cudaFuncSetAttribute(SplitAttentionKernel<T, D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kSmem)) != cudaSuccess)
    return PADRA_RESOURCE_EXHAUSTED;
  const int grid = min(sms * Cta<NT>::kPerSm, kMaxGrid);
  SplitAttentionKernel<T, D, NT><<<grid, kThreads, kSmem, stream>>>(a);
  if (cudaGetLastError() != cudaSuccess)
    return PADRA_INTERNAL;
  return LaunchJoin<T, D, P::kColumns>(a, grid, stream);
}

// Columns of a block: 8 where a sequence's rows have no more; else 16 as long as converting the codes once per block is cheaper than
// the other kernel's blocks of 256, most of which would be empty.  Measured with 8 sequences of up to 32000 tokens and 4 KV heads, here and there:
// heads of 128 with 32 columns 69 and 98 us, with 48 99 and 98 us (64 sequences of up to 2000: 32 columns 78 and 77 us, 48 107 and
// 78 us); heads of 64 with 48 columns 67 and 81 us.  One long chunk decides for the whole call: 63 decode rows beside a chunk of 512 take 414 us, in a
// call of their own and the chunk's 162 us together.
template <typename T, int D> int LaunchColumns(const AttentionArgs &a, int sms, cudaStream_t stream) {
  constexpr int kFewColumns = D == 64 ? 48 : 32;
  const long long columns = static_cast<long long>(a.seq.max_rows) * a.group;
  return columns <= 8 ? LaunchSplit<T, D, 1>(a, sms, stream) : columns <= kFewColumns ? LaunchSplit<T, D, 2>(a, sms, stream) : LaunchWide<T, D>(a, sms, stream);
}

constexpr size_t kSplitBytes = kMaxGrid * sizeof(Split);
static_assert(kSplitBytes % 16 == 0, "the pieces behind are read 16 bytes at a time");
constexpr int kMaxColumns = 16;
constexpr float kLog2e = 1.4426950408889634f;

// A call is two launches, and the second reads what the first has left in the workspace.  Host threads that share a workspace on one
// stream take turns here: a call's first launch may not come between the two of another.
std::mutex &OrderOf(const void *workspace) {
  static std::mutex order[64];
  return order[reinterpret_cast<uintptr_t>(workspace) / 256 % 64];
}

} // namespace

size_t AttentionWorkspaceBytes(int head_dim) {
  if (head_dim != 64 && head_dim != 128)
    return 0;
  const size_t narrow = static_cast<size_t>(kMaxGrid) * 2 * kMaxColumns * (head_dim + 2) * sizeof(float), wide = WidePartialBytes(head_dim);
  return kSplitBytes + (narrow > wide ? narrow : wide);
}
int LaunchAttention(const padra_kv_cache *cache, const padra_sequences *sequences, const void *q, void *out, long long q_stride,
                    long long out_stride, int q_heads, int type, float scale, int window, void *workspace, size_t workspace_bytes, int *bad,
                    cudaStream_t stream) {
  KvView c;
  SequenceView s;
  if (!ViewOf(cache, &c) || !ViewOf(sequences, c, &s) || !bad || q_heads < 1 || q_heads > 4096 || q_heads % c.kv_heads || window < 0 ||
      !std::isfinite(scale * kLog2e))
    return PADRA_INVALID_ARGUMENT;
  if ((c.head_dim != 64 && c.head_dim != 128) || (type != PADRA_ROWS_BF16 && type != PADRA_ROWS_F16))
    return PADRA_UNSUPPORTED;
  if (!RowsOk(q, q_stride, s.rows, q_heads, c.head_dim) || !RowsOk(out, out_stride, s.rows, q_heads, c.head_dim))
    return PADRA_INVALID_ARGUMENT;
  if (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16 || workspace_bytes < AttentionWorkspaceBytes(c.head_dim))
    return PADRA_INVALID_ARGUMENT;
  if (!s.rows || !s.count)
    return PADRA_OK;
  int device = 0, sms = 0;
  if (cudaGetDevice(&device) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess || sms < 1)
    return PADRA_INTERNAL;
  AttentionArgs a{c, s, q, out, q_stride, out_stride, q_heads, q_heads / c.kv_heads, scale ? fabsf(scale) * kLog2e : 1.f,
                  scale > 0 ? 1.f : scale < 0 ? -1.f : 0.f,
                  window >> 30 ? 0 : window, // positions are below 2^30: nothing is outside, and position - window stays in 32 bits
                  static_cast<Split *>(workspace), reinterpret_cast<float *>(static_cast<unsigned char *>(workspace) + kSplitBytes), kCodeMasks, bad};
  const std::lock_guard<std::mutex> turn(OrderOf(workspace));
  if (type == PADRA_ROWS_BF16)
    return c.head_dim == 64 ? LaunchColumns<__nv_bfloat16, 64>(a, sms, stream) : LaunchColumns<__nv_bfloat16, 128>(a, sms, stream);
  return c.head_dim == 64 ? LaunchColumns<__half, 64>(a, sms, stream) : LaunchColumns<__half, 128>(a, sms, stream);
}

} // namespace padra
