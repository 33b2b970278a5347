// Attention over the paged 4-bit cache for many query rows per sequence (prefill chunks, verifier rows): S = Q K^T and O += P V on
// the 5th-generation tensor cores, accumulators in tensor memory, K and V turned from codes into FP16 operands on the way.
//
// A unit is (sequence, KV head, block of 256 query columns); a column is a row of the sequence with one of the heads that
// share the KV head, so heads of a group share every K and V tile.  A tile is 128 tokens.  As in attention.cu all tiles of a call form
// one list and every CTA (one per SM) takes an equal run of it; pieces of units are joined by JoinKernel.
//   * Eight producer warps load codes and scales one tile ahead into registers and store FP16 rows (value = (code - 8) * scale, one
//     rounding of 2^-12) in the 128-byte-swizzled layout, the same for K (K-major: contraction over the head's values) and V
//     (MN-major: contraction over tokens), so that V needs no transposition.  Values inside a block of eight lie in the order
//     0 4 1 5 2 6 3 7 in which a code word yields pairs; Q is stored in that order and the output put back.
//   * A thread for each half issues its MMAs: S (128 columns x 128 tokens) of each half of the block in its own tensor memory, so that one
//     half's MMAs run under the other half's softmax.  P replaces S in tensor memory as the A operand of O += P V.
//   * Two softmax warpgroups, one per half, one thread per column: no shuffles.  The maximum is raised lazily (by a factor of up to
//     2^15 in FP16 weights), and only then is O rescaled.
//   * A block with at most 128 columns would leave one half idle: then the halves take even and odd tiles of the SAME columns,
//     each with its own maximum, sum and O, and are joined through tensor memory at the end of the piece.
// Tensor memory: S/P of the halves in columns 0 and 128, O in 256 and 384.  Every wait is bounded in time; on expiry the CTA raises the
// error flag and leaves.
#include "attention.cuh"

namespace padra {
namespace attention {
namespace {

constexpr int kTile = 128, kSub = 64, kColumns = 256; // scores and weights go by sub-tiles of 64 tokens
constexpr int kSoftmaxWarps = 8, kProducerWarps = 8, kMmaWarp = kSoftmaxWarps + kProducerWarps;
constexpr int kWarps = kMmaWarp + 2, kThreads = kWarps * 32;
constexpr int kStages = 2;

// place / group and its remainder inside a unit: `reciprocal` = ceil(2^32 / group) gives the quotient exactly while
// place * group < 2^32, which places counted from the block's first row (below group + 256, group at most 4096) keep to.
struct Places {
  int row0, rest0; // row and head of the block's first column
  unsigned reciprocal;
  int group;
  __device__ __forceinline__ void Split(int column, int *row, int *head) const {
    const unsigned x = static_cast<unsigned>(rest0 + column);
    const int quotient = group == 1 ? static_cast<int>(x) : static_cast<int>(__umulhi(x, reciprocal));
    *row = row0 + quotient, *head = static_cast<int>(x) - quotient * group;
  }
};
__device__ __forceinline__ Places PlacesOf(const AttentionArgs &a, int block) {
  Places p;
  p.row0 = block * kColumns / a.group, p.rest0 = block * kColumns - p.row0 * a.group, p.group = a.group;
  p.reciprocal = static_cast<unsigned>((0x100000000ull + a.group - 1) / static_cast<unsigned>(a.group));
  return p;
}

// Blocks of a sequence, and what one of them asks for.
struct Rows {
  int begin, rows, context, blocks;
};
struct Unit {
  int first, tiles, columns; // first tile and number of tiles of the whole unit
};
__device__ __forceinline__ Rows RowsOf(const AttentionArgs &a, int s) {
  Rows r{};
  if (SequenceRows(a.seq, a.cache, s, &r.begin, &r.rows, &r.context, a.bad) && r.rows)
    r.blocks = static_cast<int>((static_cast<long long>(r.rows) * a.group + kColumns - 1) / kColumns);
  return r;
}
__device__ __forceinline__ Unit UnitOf(const AttentionArgs &a, const Rows &r, int block) {
  const int from = block * kColumns, to = min(from + kColumns, r.rows * a.group), start = r.context - r.rows;
  const int first_row = from / a.group, last_row = (to - 1) / a.group;
  const int low = a.window ? max(0, start + first_row + 1 - a.window) : 0, high = max(0, start + last_row + 1);
  Unit u;
  u.columns = to - from, u.first = low / kTile, u.tiles = max(1, (high + kTile - 1) / kTile - u.first);
  return u;
}

// A CTA's run, piece by piece; every role walks it by itself.
struct Walk {
  long long at, end;
  int s, block, head, skip; // the piece begins `skip` tiles into its unit
  Rows rows;
  Unit unit;
  int count;
  __device__ __noinline__ void Begin(const AttentionArgs &a, long long from, long long to, int sequence, int first_block, long long offset) {
    at = from, end = to, s = sequence, block = first_block;
    rows = RowsOf(a, s), unit = UnitOf(a, rows, block);
    head = static_cast<int>(Quotient(offset, unit.tiles)), skip = static_cast<int>(offset - static_cast<long long>(head) * unit.tiles);
    count = static_cast<int>(min(static_cast<long long>(unit.tiles - skip), end - at));
  }
  __device__ __forceinline__ bool More() const { return at < end; }
  __device__ __noinline__ void Next(const AttentionArgs &a) {
    at += count, skip = 0;
    if (at >= end)
      return;
    if (++head == a.cache.kv_heads) {
      head = 0;
      if (++block == rows.blocks) {
        block = 0;
        do
          rows = RowsOf(a, ++s);
        while (!rows.blocks);
      }
      unit = UnitOf(a, rows, block);
    }
    count = static_cast<int>(min(static_cast<long long>(unit.tiles), end - at));
  }
  __device__ __forceinline__ bool Paired() const { return unit.columns <= 128; }
};

template <int D> struct Smem {
  static constexpr int kHalves = D / 64;
  alignas(1024) unsigned char q[2][kHalves][128 * 128]; // rows of 64 values (128 bytes), 16-byte pieces swizzled by row
  alignas(1024) unsigned char k[kStages][kHalves][kTile * 128];
  alignas(1024) unsigned char v[kStages][kHalves][kTile * 128];
  alignas(8) unsigned long long q_full[2], k_full[kStages], k_empty[kStages], v_full[kStages], v_empty[kStages], s_full[2][2], p_full[2][2], o_full[2], o_last[2]; // [half][sub-tile]; O after every sub-tile, after a piece's last
  unsigned long long q_empty;
  unsigned long long shared_ready, shared_done; // the second half's maximum and sum are there / have been used
  struct {
    float factor; // what a column's scores are multiplied by
    int last;     // its position: the last token it sees (-1: none)
  } column[2][kColumns]; // of this piece and of the next
  alignas(16) unsigned char out[kSoftmaxWarps][32 * 64]; // a warp's rows on their way out, 32 values at a time
  float2 other[128];
  int item_begin[kThreads];
  long long scan[kWarps], start_offset;
  int start_sequence, start_block;
  Walk walk[kMmaWarp + 2]; // every working warp's place in the run: in registers it crowded out what the loops need
  unsigned tmem;
  int abort;
};

// Bounded wait (see BarrierWait).  Code size is what this kernel's three roles compete for: with every wait written out they did not fit the
// instruction cache together and fetched their loops anew for every tile.  So a wait is one poll in place (which the hardware may
// suspend) and a call for the rest.
__device__ __forceinline__ bool Passed(unsigned address, unsigned parity) {
  unsigned done;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(done)
               : "r"(address), "r"(parity), "r"(2000u)
               : "memory");
  return done != 0;
}
__device__ __noinline__ bool WaitOn(unsigned address, unsigned parity, const volatile int *abort) {
  unsigned long long started = 0;
  while (!Passed(address, parity)) {
    if (*abort)
      return false;
    unsigned long long now;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
    if (!started)
      started = now;
    else if (now - started > kWaitLimitNs)
      return false;
  }
  return true;
}
__device__ __forceinline__ bool SuspendedWait(unsigned long long *bar, unsigned parity, const volatile int *abort) {
  const unsigned address = SmemAddress(bar);
  return Passed(address, parity) || WaitOn(address, parity, abort);
}
// One lane waits for its warp: true for all lanes or for none.
__device__ __forceinline__ bool WarpWait(unsigned long long *bar, unsigned parity, const volatile int *abort) {
  int done = 0;
  if ((threadIdx.x & 31) == 0)
    done = SuspendedWait(bar, parity, abort);
  return __shfl_sync(0xffffffffu, done, 0) != 0;
}
__device__ __forceinline__ void FenceToTensorCores() { // this thread's shared-memory writes before the tensor cores' reads
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}
__device__ __forceinline__ void BeforeSync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void AfterSync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// Operand descriptors (see SwizzledOperandDescriptor for the fields), low and high word apart: the steps of a tile differ in the low
// word's address only, and one thread builds two descriptors per MMA.
// K-major (Q, K): the leading offset is unused.  MN-major (V: rows of 64 values, one per token; the contraction runs over rows): blocks of 64
// output values are 16 KB apart, groups of eight tokens 1024 bytes.
constexpr unsigned kDescriptorHigh = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ unsigned DescriptorLow(unsigned smem_address, unsigned leading) {
  return ((smem_address & 0x3ffffu) >> 4) | (leading >> 4) << 16;
}
__device__ __forceinline__ void MmaStepSS(unsigned tmem_d, unsigned a_low, unsigned b_low, unsigned idesc, bool accumulate) {
  asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tsetp.ne.b32 p, %5, 0;\n\tmov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\t"
               "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, p;\n\t}" ::"r"(tmem_d),
               "r"(a_low), "r"(b_low), "r"(kDescriptorHigh), "r"(idesc), "r"(accumulate ? 1u : 0u)
               : "memory");
}
constexpr unsigned kSecondOperandRowMajor = 1u << 16; // instruction descriptor: B is MN-major
__device__ __forceinline__ void MmaStepTS(unsigned tmem_d, unsigned tmem_a, unsigned b_low, unsigned idesc, bool accumulate) {
  asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 b;\n\tsetp.ne.b32 p, %5, 0;\n\tmov.b64 b, {%2, %3};\n\t"
               "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n\t}" ::"r"(tmem_d),
               "r"(tmem_a), "r"(b_low), "r"(kDescriptorHigh), "r"(idesc), "r"(accumulate ? 1u : 0u)
               : "memory");
}
__device__ __forceinline__ void TmemStore16(unsigned taddr, const unsigned (&v)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
               "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
               "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
               : "memory");
}
// Columns of the thread's lane, in pairs for the packed FP32 operations.  One statement with the wait: nothing that uses a value can
// move before it, and the pairs are the registers that the load fills.
using Pair = unsigned long long;
__device__ __forceinline__ void TmemLoadPairs(unsigned taddr, Pair (&v)[8]) {
  asm volatile("{\n\t.reg .b32 r0, r1, r2, r3, r4, r5, r6, r7, r8, r9, r10, r11, r12, r13, r14, r15;\n\t"
               "tcgen05.ld.sync.aligned.32x32b.x16.b32 {r0, r1, r2, r3, r4, r5, r6, r7, r8, r9, r10, r11, r12, r13, r14, r15}, [%8];\n\t"
               "tcgen05.wait::ld.sync.aligned;\n\t"
               "mov.b64 %0, {r0, r1}; mov.b64 %1, {r2, r3}; mov.b64 %2, {r4, r5}; mov.b64 %3, {r6, r7};\n\t"
               "mov.b64 %4, {r8, r9}; mov.b64 %5, {r10, r11}; mov.b64 %6, {r12, r13}; mov.b64 %7, {r14, r15};\n\t"
               "}"
               : "=l"(v[0]), "=l"(v[1]), "=l"(v[2]), "=l"(v[3]), "=l"(v[4]), "=l"(v[5]), "=l"(v[6]), "=l"(v[7])
               : "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void TmemLoadPairs(unsigned taddr, Pair (&v)[16]) {
  asm volatile("{\n\t.reg .b32 r0, r1, r2, r3, r4, r5, r6, r7, r8, r9, r10, r11, r12, r13, r14, r15, r16, r17, r18, r19, r20, r21, r22, r23, r24, r25, r26, r27, r28, r29, r30, r31;\n\t"
               "tcgen05.ld.sync.aligned.32x32b.x32.b32 {r0, r1, r2, r3, r4, r5, r6, r7, r8, r9, r10, r11, r12, r13, r14, r15, r16, r17, r18, r19, r20, r21, r22, r23, r24, r25, r26, r27, r28, r29, r30, r31}, [%16];\n\t"
               "tcgen05.wait::ld.sync.aligned;\n\t"
               "mov.b64 %0, {r0, r1}; mov.b64 %1, {r2, r3}; mov.b64 %2, {r4, r5}; mov.b64 %3, {r6, r7};\n\t"
               "mov.b64 %4, {r8, r9}; mov.b64 %5, {r10, r11}; mov.b64 %6, {r12, r13}; mov.b64 %7, {r14, r15};\n\t"
               "mov.b64 %8, {r16, r17}; mov.b64 %9, {r18, r19}; mov.b64 %10, {r20, r21}; mov.b64 %11, {r22, r23};\n\t"
               "mov.b64 %12, {r24, r25}; mov.b64 %13, {r26, r27}; mov.b64 %14, {r28, r29}; mov.b64 %15, {r30, r31};\n\t"
               "}"
               : "=l"(v[0]), "=l"(v[1]), "=l"(v[2]), "=l"(v[3]), "=l"(v[4]), "=l"(v[5]), "=l"(v[6]), "=l"(v[7]),
                 "=l"(v[8]), "=l"(v[9]), "=l"(v[10]), "=l"(v[11]), "=l"(v[12]), "=l"(v[13]), "=l"(v[14]), "=l"(v[15])
               : "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void TmemStoreWait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Byte offset of 16-byte piece `piece` (0 .. D / 8 - 1) of row `row` inside a tile of [D / 64][128 rows][128 bytes].
__device__ __forceinline__ unsigned PieceOffset(int row, int piece) {
  return (piece >> 3) * (128 * 128) + row * 128 + (((piece & 7) ^ (row & 7)) << 4);
}

// ---- producers: tiles of codes to FP16 rows ----
template <int D> struct Producer {
  static constexpr int kGroups = D / kKvGroup, kChunks = D / 32; // 16-byte chunks of a token's codes
  static constexpr int kTokens = 16 * kChunks / 32;              // tokens per lane: its warp's 16 tokens, one chunk each
  uint4 codes[kTokens];
  uint2 scales[kTokens]; // of the token's groups (head size 64: in .x)

  // Lanes of a quarter warp (whose stores go out together) take rows whose swizzle leaves no bank twice: rows t and t + 4 with
  // four chunks, rows {0, 1, 4, 5} or {2, 3, 6, 7} with two.
  static __device__ __forceinline__ int TokenOf(int lane, int i) {
    if constexpr (kChunks == 4)
      return 8 * i + ((lane >> 3) & 3) + ((lane >> 2) & 1) * 4;
    else
      return (lane >> 4) * 8 + ((lane >> 3) & 1) * 2 + ((lane >> 1) & 1) + ((lane >> 2) & 1) * 4;
  }
  // Codes and scales of this warp's 16 tokens, of which `there` exist (their codes begin at `codes_from`, their scales at `scales_from`): lanes
  // beyond them read the last one that exists and take scales of zero.
  __device__ __forceinline__ void Load(const unsigned char *codes_from, const unsigned char *scales_from, int there) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < kTokens; ++i) {
      const int token = TokenOf(lane, i), row = max(0, min(token, there - 1));
      codes[i] = __ldg(reinterpret_cast<const uint4 *>(codes_from + row * (D / 2) + 16 * (lane % kChunks)));
      if constexpr (kGroups == 4)
        scales[i] = __ldg(reinterpret_cast<const uint2 *>(scales_from + row * (D / 16)));
      else
        scales[i] = make_uint2(__ldg(reinterpret_cast<const unsigned *>(scales_from + row * (D / 16))), 0);
      if (token >= there)
        scales[i] = make_uint2(0, 0);
    }
  }
  // Byte offset of the first word's piece of (row, chunk) in a tile: word c * groups + g of a row holds piece 4 g + c of eight values.
  static __device__ __forceinline__ unsigned OffsetOf(int row, int chunk) { return PieceOffset(row, 4 * chunk / kGroups); }
  // Word w of the chunk lies 4 (w % groups) + w / groups pieces on; pieces 0 .. 7 of a half change places with the row (XOR), so
  // neighbours are found by XOR too: bit 2 of the piece is bit 6 of the offset.
  static __device__ __forceinline__ void Store(unsigned tile, unsigned offset, const uint4 &codes, const uint2 &scales, const CodeMasks &masks) {
    const unsigned word[4] = {codes.x, codes.y, codes.z, codes.w};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const int g = w % kGroups, c = w / kGroups;
      const unsigned pair = g & 2 ? scales.y : scales.x;
      const __half2 both = *reinterpret_cast<const __half2 *>(&pair), scale = w & 1 ? __high2half2(both) : __low2half2(both);
      const unsigned u = word[w], x = u >> 8;
      StoreShared(tile + (offset ^ ((g & 1) << 6 | c << 4)) + (g >> 1) * (128 * 128),
                  make_uint4(Scaled(Low(u, masks), 0x64086408u, scale), Scaled(High(u, masks), 0x54805480u, scale),
                             Scaled(Low(x, masks), 0x64086408u, scale), Scaled(High(x, masks), 0x54805480u, scale)));
    }
  }
};

// ---- softmax ----
__device__ __forceinline__ Pair MakePair(float x, float y) {
  Pair p;
  asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(x), "f"(y));
  return p;
}
__device__ __forceinline__ void SplitPair(Pair p, float *x, float *y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(*x), "=f"(*y) : "l"(p)); }
__device__ __forceinline__ Pair Fma2(Pair x, Pair y, Pair z) {
  Pair r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(x), "l"(y), "l"(z));
  return r;
}
__device__ __forceinline__ Pair Mul2(Pair x, Pair y) {
  Pair r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
  return r;
}
__device__ __forceinline__ Pair Add2(Pair x, Pair y) {
  Pair r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
  return r;
}
__device__ __forceinline__ float Max3(float x, float y, float z) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
  return r;
}

// ---- queries ----
// 2^exponent of a float's leading bit, and the reciprocal (finite, in the normal range of both)
__device__ __forceinline__ float PowerOf(float x) {
  return __uint_as_float(min(max(__float_as_uint(x) & 0x7f800000u, 1u << 23), 253u << 23));
}
__device__ __forceinline__ float ReciprocalPower(float power) {
  return __uint_as_float((254u << 23) - __float_as_uint(power));
}

// Stages the query rows of 32 columns of a block (column0 ..., those below `columns`) as FP16, divided by a power of two and times the
// sign of scale, into a half's Q tile (rows column0 % 128 ...), and notes their factors and positions.  D / 8 lanes read a row together.
template <typename T, int D>
__device__ __forceinline__ void StageQueries(const AttentionArgs &a, const Rows &r, int head, const Places &places, int column0, int columns, Smem<D> &sm,
                                             int parity) {
  constexpr int kLanes = D / 8, kSide = 32 / kLanes, kFlight = 4;
  const int lane = threadIdx.x & 31, side = lane / kLanes, piece = lane % kLanes;
  const int start = r.context - r.rows;
  unsigned char *const tile = sm.q[column0 >> 7][0];
#pragma unroll 1
  for (int c0 = column0; c0 < column0 + 32; c0 += kSide * kFlight) {
    uint4 raw[kFlight];
    int position[kFlight];
#pragma unroll
    for (int f = 0; f < kFlight; ++f) {
      const int c = c0 + f * kSide + side;
      int row, h;
      places.Split(c, &row, &h);
      position[f] = start + row;
      raw[f] = c < columns && position[f] >= 0
                   ? __ldg(reinterpret_cast<const uint4 *>(static_cast<const T *>(a.q) + static_cast<long long>(r.begin + row) * a.q_stride +
                                                           (head * a.group + h) * D + 8 * piece))
                   : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int f = 0; f < kFlight; ++f) {
      const int c = c0 + f * kSide + side;
      float x[8], most = 0;
      Widen(raw[f], static_cast<const T *>(nullptr), x);
#pragma unroll
      for (int j = 0; j < 8; ++j) // as integers: an exponent of all ones (infinity, NaN) is larger than everything else
        most = __uint_as_float(max(__float_as_uint(most), __float_as_uint(x[j]) & 0x7fffffffu));
      unsigned bits = __float_as_uint(most);
#pragma unroll
      for (int m = 1; m < kLanes; m *= 2)
        bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, m));
      const bool finite = bits < 0x7f800000u;
      const float power = PowerOf(__uint_as_float(bits)), shrink = finite ? ReciprocalPower(power) * a.sign : 0.f;
      if (finite) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          x[j] *= shrink;
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          x[j] = 0;
      }
      *reinterpret_cast<uint4 *>(tile + PieceOffset(c & 127, piece)) = make_uint4(Pack(x[0], x[4]), Pack(x[1], x[5]), Pack(x[2], x[6]), Pack(x[3], x[7]));
      if (piece == 0) {
        if (!finite)
          Raise(a.bad);
        sm.column[parity][c].factor = a.scale * (finite ? power : 1.f);
        sm.column[parity][c].last = c < columns && finite ? position[f] : -1;
      }
    }
  }
}

// The MMAs of one half, issued by one thread: S of a tile's two sub-tiles, then O of a sub-tile and S of the same sub-tile of the next tile.  So S is
// ready a sub-tile before its softmax begins, and softmax and tensor cores do not wait for each other in turn.  In blocks with
// columns for both halves every tile is the half's, otherwise every other one.  Each half has a thread of its own, on another scheduler:
// between the many warps an MMA's ten instructions take longer to come by than its 64 cycles on the tensor cores.  Half and sub-tile
// are compile-time and tensor memory begins at column 0 (the CTA has all of it): with addresses in registers an MMA took up to a
// hundred instructions.
template <int D, int Half, int Sub> __device__ __forceinline__ void IssueScores(unsigned q_low, unsigned k_low) {
#pragma unroll
  for (int s = 0; s < D / 16; ++s) {
    const unsigned offset = ((s >> 2) * (128 * 128) + (s & 3) * 32) >> 4;
    MmaStepSS(128 * Half + kSub * Sub, q_low + offset, k_low + offset + ((Sub * kSub * 128) >> 4), InstructionDescriptor(kSub), s > 0);
  }
}
template <int D, int Half, int Sub> __device__ __forceinline__ void IssueOutput(unsigned v_low, bool accumulate) {
#pragma unroll
  for (int s = 0; s < kSub / 16; ++s)
    MmaStepTS(256 + 128 * Half, 128 * Half + kSub * Sub + 8 * s, v_low + (((Sub * kSub + 16 * s) * 128) >> 4),
              InstructionDescriptor(D) | kSecondOperandRowMajor, accumulate || s > 0);
}
template <int D, int Half> __device__ __forceinline__ bool IssueMmas(const AttentionArgs &a, Smem<D> &sm, Walk &walk) {
  const volatile int *const abort = &sm.abort;
  unsigned tiles = 0, jobs = 0, pieces = 0, staged = 0; // so far: tiles, this half's jobs, pieces, pieces with queries of its own
  bool alive = true;
  for (; alive && walk.More(); walk.Next(a), ++pieces) {
    const bool paired = walk.Paired();
    const int count = walk.count, step = paired ? 2 : 1, first = paired ? Half : 0;
    auto wait = [&](unsigned long long *full, int tile) { return SuspendedWait(full + ((tiles + tile) & (kStages - 1)), ((tiles + tile) / kStages) & 1, abort); };
    // A tile that is the other half's is released here too, once it is there (an arrival must not count for an earlier tile).
    auto pass = [&](unsigned long long *full, unsigned long long *empty, int tile) {
      if (tile < 0 || tile >= count || !paired)
        return true;
      const bool there = wait(full, tile);
      BarrierArrive(empty + ((tiles + tile) & (kStages - 1)));
      return there;
    };
    auto q_low = [&] { return DescriptorLow(SmemAddress(sm.q[Half && !paired][0]), 16); };
    auto stage_of = [&](int tile) { return (tiles + tile) & (kStages - 1); };
    auto first_scores = [&](int tile) {
      if (!pass(sm.k_full, sm.k_empty, tile - 1) || !wait(sm.k_full, tile))
        return false;
      AfterSync();
      IssueScores<D, Half, 0>(q_low(), DescriptorLow(SmemAddress(sm.k[stage_of(tile)][0]), 16));
      MmaCommit(&sm.s_full[Half][0]);
      return true;
    };
    auto second_scores = [&](int tile) {
      IssueScores<D, Half, 1>(q_low(), DescriptorLow(SmemAddress(sm.k[stage_of(tile)][0]), 16));
      MmaCommit(&sm.s_full[Half][1]);
      MmaCommit(&sm.k_empty[stage_of(tile)]);
      if (tile + step >= count)
        MmaCommit(&sm.q_empty);
    };
    alive = Half && !paired ? SuspendedWait(&sm.q_full[1], staged++ & 1, abort) : SuspendedWait(&sm.q_full[0], pieces & 1, abort);
    if (!alive)
      break;
    if (first >= count) // a single tile, the other half's
      BarrierArrive(&sm.q_empty);
    int tile = first - step; // the first turn of the loop has scores only
    for (; alive && tile < count; tile += step) {
      const int next = tile + step;
      const unsigned v_low = DescriptorLow(SmemAddress(sm.v[stage_of(tile)][0]), 128 * 128);
      if (tile >= first) {
        if (!(alive = pass(sm.v_full, sm.v_empty, tile - 1) && wait(sm.v_full, tile) && SuspendedWait(&sm.p_full[Half][0], jobs & 1, abort)))
          break;
        AfterSync();
        IssueOutput<D, Half, 0>(v_low, tile > first);
        MmaCommit(&sm.o_full[Half]);
      }
      if (next < count && !(alive = first_scores(next)))
        break;
      if (tile >= first) {
        if (!(alive = SuspendedWait(&sm.p_full[Half][1], jobs & 1, abort)))
          break;
        AfterSync();
        IssueOutput<D, Half, 1>(v_low, true);
        MmaCommit(&sm.o_full[Half]);
        MmaCommit(&sm.v_empty[stage_of(tile)]);
        ++jobs;
      }
      if (next < count)
        second_scores(next);
      else if (tile >= first)
        MmaCommit(&sm.o_last[Half]);
    }
    if (alive) // what follows this half's last tile
      alive = pass(sm.k_full, sm.k_empty, tile - 1) && pass(sm.v_full, sm.v_empty, tile - 1);
    tiles += count;
  }
  return alive;
}

template <typename T, int D> __global__ void __launch_bounds__(kThreads, 1) WideAttentionKernel(const __grid_constant__ AttentionArgs a) {
  using S = Smem<D>;
  extern __shared__ __align__(16) unsigned char raw_smem[];
  S &sm = *reinterpret_cast<S *>(raw_smem + ((1024u - (SmemAddress(raw_smem) & 1023u)) & 1023u));
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // ---- this CTA's run: items are (sequence, block), each worth its tiles for every KV head ----
  long long total = 0, at_mine = 0, cost_mine = 0;
  int item_sequence = 0, item_block = 0, rounds = 0;
  auto scan = [&](long long begin) { // adds up all items; the thread whose item holds tile `begin` of the list publishes it
    total = 0, rounds = 0;
    for (int s0 = 0; s0 < a.seq.count; s0 += kThreads) {
      long long items;
      const long long blocks = s0 + tid < a.seq.count ? RowsOf(a, s0 + tid).blocks : 0;
      const int before = static_cast<int>(BlockPrefix<kWarps>(blocks, sm.scan, &items));
      sm.item_begin[tid] = before;
      __syncthreads();
      for (int i0 = 0; i0 < items; i0 += kThreads, ++rounds) {
        const int i = i0 + tid;
        cost_mine = 0;
        if (i < items) {
          int low = 0, high = kThreads - 1; // the last sequence that begins at or before item i has it
          while (low < high) {
            const int middle = (low + high + 1) / 2;
            if (sm.item_begin[middle] <= i)
              low = middle;
            else
              high = middle - 1;
          }
          item_sequence = s0 + low, item_block = i - sm.item_begin[low];
          cost_mine = static_cast<long long>(UnitOf(a, RowsOf(a, item_sequence), item_block).tiles) * a.cache.kv_heads;
        }
        long long part;
        at_mine = total + BlockPrefix<kWarps>(cost_mine, sm.scan, &part);
        total += part;
        if (begin >= at_mine && begin < at_mine + cost_mine)
          sm.start_sequence = item_sequence, sm.start_block = item_block, sm.start_offset = begin - at_mine;
      }
      __syncthreads();
    }
  };
  scan(-1);
  const long long share = max(2ll, Quotient(total + gridDim.x - 1, gridDim.x)), begin = blockIdx.x * share, end = min(total, begin + share);
  if (tid == 0) {
    a.split[blockIdx.x].pieces = 0;
    sm.abort = 0;
    for (int i = 0; i < 2; ++i) {
      BarrierInit(&sm.q_full[i], kProducerWarps / 2), BarrierInit(&sm.o_full[i], 1), BarrierInit(&sm.o_last[i], 1);
      for (int sub = 0; sub < 2; ++sub)
        BarrierInit(&sm.s_full[i][sub], 1), BarrierInit(&sm.p_full[i][sub], kSoftmaxWarps / 2);
    }
    for (int i = 0; i < kStages; ++i) {
      BarrierInit(&sm.k_full[i], kProducerWarps), BarrierInit(&sm.v_full[i], kProducerWarps);
      BarrierInit(&sm.k_empty[i], 2), BarrierInit(&sm.v_empty[i], 2); // both halves let go of a tile
    }
    BarrierInit(&sm.q_empty, 2);
    BarrierInit(&sm.shared_ready, kSoftmaxWarps / 2), BarrierInit(&sm.shared_done, kSoftmaxWarps / 2);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (begin >= end)
    return;
  if (rounds == 1) { // the items are still in the threads' registers
    if (begin >= at_mine && begin < at_mine + cost_mine)
      sm.start_sequence = item_sequence, sm.start_block = item_block, sm.start_offset = begin - at_mine;
  } else {
    scan(begin);
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(SmemAddress(&sm.tmem)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  BeforeSync();
  __syncthreads();
  AfterSync();
  constexpr unsigned tmem = 0; // all 512 columns are this CTA's
  const volatile int *const abort = &sm.abort;
  Walk &walk = sm.walk[min(warp, kMmaWarp + 1)];
  if (lane == 0 && warp <= kMmaWarp + 1)
    walk.Begin(a, begin, end, sm.start_sequence, sm.start_block, sm.start_offset);
  __syncwarp();
  auto next_piece = [&]() { // by the whole warp
    __syncwarp();
    if (lane == 0)
      walk.Next(a);
    __syncwarp();
  };
  bool alive = sm.tmem == 0;

  if (warp >= kSoftmaxWarps && warp < kMmaWarp) {
    // =============================== producers ===============================
    using P = Producer<D>;
    const int mine = 16 * (warp - kSoftmaxWarps); // this warp's tokens of a tile
    unsigned offset[P::kTokens];
#pragma unroll
    for (int j = 0; j < P::kTokens; ++j)
      offset[j] = P::OffsetOf(mine + P::TokenOf(lane, j), lane % P::kChunks);
    int tile = 0; // of the piece: the tile that is loaded next
    const unsigned char *codes_from = a.cache.pool, *scales_from = a.cache.pool; // K's codes and scales of the warp's tokens in it
    int there = 0;                                                             // how many of them the columns may see
    const int v_behind = a.cache.code_bytes() + a.cache.scale_bytes();
    auto find = [&]() {
      there = 0;
      if (walk.More()) {
        const int t = (walk.unit.first + walk.skip + tile) * kTile + mine, context = walk.rows.context;
        // first token that some column of the unit sees
        const int low = a.window ? max(0, context - walk.rows.rows + walk.block * kColumns / a.group + 1 - a.window) : 0;
        if (t < context && t + 16 > low) {
          const int page = PageOf(a.seq, a.cache, walk.s, t, a.bad), slot = t & (a.cache.page_size - 1);
          if (page >= 0) {
            const unsigned char *const block = a.cache.block(page, walk.head);
            codes_from = block + slot * (D / 2), scales_from = block + a.cache.code_bytes() + slot * (D / 16);
            there = min(16, context - t);
          }
        }
      }
    };
    auto advance = [&]() {
      if (++tile == walk.count)
        next_piece(), tile = 0;
      find();
    };
    auto load = [&](P &to, bool is_v) {
      const int behind = is_v ? v_behind : 0;
      to.Load(codes_from + behind, scales_from + behind, there);
    };
    // A piece's queries come before its first tile: this warp's 32 columns, once the MMAs of the piece before are done with Q.
    unsigned pieces = 0;
    auto stage_queries = [&]() {
      const int column0 = 32 * (warp - kSoftmaxWarps);
      if (pieces && !(alive = WarpWait(&sm.q_empty, (pieces - 1) & 1, abort)))
        return;
      if (column0 < 128 || !walk.Paired()) {
        StageQueries<T, D>(a, walk.rows, walk.head, PlacesOf(a, walk.block), column0, walk.unit.columns, sm, pieces & 1);
        FenceToTensorCores();
        __syncwarp();
        if (lane == 0)
          BarrierArrive(&sm.q_full[column0 >> 7]);
      }
      ++pieces;
    };
    // K and V of a tile are two steps of the same code; what is stored next has been loaded two steps before.
    P front, back;
    find();
    const int steps = 2 * static_cast<int>(end - begin);
#pragma unroll 1
    for (int n = -2; n < steps && alive; ++n) {
      const bool is_v = n & 1;
      if (n >= 0) {
        const int stage = (n >> 1) & (kStages - 1);
        alive = WarpWait(is_v ? &sm.v_empty[stage] : &sm.k_empty[stage], ((n / (2 * kStages)) & 1) ^ 1, abort);
        if (!alive)
          break;
        const unsigned to = SmemAddress(sm.k[0][0]) + (is_v ? kStages + stage : stage) * static_cast<unsigned>(sizeof(sm.k[0])); // V lies behind K
#pragma unroll
        for (int j = 0; j < P::kTokens; ++j)
          P::Store(to, offset[j], front.codes[j], front.scales[j], a.masks);
        FenceToTensorCores();
        __syncwarp();
        if (lane == 0)
          BarrierArrive(is_v ? &sm.v_full[stage] : &sm.k_full[stage]);
      }
      front = back;
      if (n + 2 < steps) {
        load(back, is_v); // the same of the next tile
        if (is_v) {
          if (tile == 0) // that tile begins a piece
            stage_queries();
          advance();
        }
      }
    }
  } else if (warp >= kMmaWarp) {
    // =============================== MMA issue ===============================
    if (lane == 0 && warp <= kMmaWarp + 1) {
      alive = alive && (warp == kMmaWarp ? IssueMmas<D, 0>(a, sm, walk) : IssueMmas<D, 1>(a, sm, walk));
      if (!alive) {
        sm.abort = 1;
        Raise(a.bad);
      }
    }
    __syncwarp();
  } else {
    // =============================== softmax ===============================
    const int half = warp / 4, row = tid & 127; // the thread's column of its half, and its lane in tensor memory
    const unsigned lanes = static_cast<unsigned>((warp & 3) * 32) << 16, s_address = tmem + lanes + 128 * half, o_address = tmem + lanes + 256 + 128 * half;
    // phases gone by: this half's tiles, pieces with queries of either half, O after either half's sub-tiles, joins
    unsigned jobs = 0, staged_first = 0, staged_second = 0, outputs = 0, finished = 0, other_finished = 0, shared = 0, pieces = 0;
    for (; alive && walk.More(); next_piece(), ++pieces) {
      const bool paired = walk.Paired();
      const int own = paired ? row : 128 * half + row; // column of the block
      const bool there = own < walk.unit.columns;
      // the block's columns are staged by the producers, those that both halves work on once
      if (paired || !half) {
        alive = WarpWait(&sm.q_full[0], staged_first & 1, abort);
      } else {
        alive = WarpWait(&sm.q_full[1], staged_second & 1, abort);
      }
      ++staged_first, staged_second += !paired;
      if (!alive)
        break;
      const float factor = sm.column[pieces & 1][own].factor;
      const int last = sm.column[pieces & 1][own].last, first = a.window ? max(0, last - a.window + 1) : 0;
      float top = kNever, total = 0;
      const int least = __reduce_min_sync(0xffffffffu, there ? last : 0x7fffffff), latest = __reduce_max_sync(0xffffffffu, there ? first : 0);
      const int first_tile = walk.unit.first + walk.skip, count = walk.count;
      const int begin_tile = paired ? half : 0, end_sub = 2 * count;
      // sub-tiles of this half: both of every tile, or of every other one
      for (int i = 2 * begin_tile; i < end_sub; i += i & 1 && paired ? 3 : 1) {
        const int sub = i & 1, t0 = first_tile * kTile + i * kSub;
        const unsigned score_address = s_address + kSub * sub;
        alive = WarpWait(&sm.s_full[half][sub], jobs & 1, abort);
        if (!alive)
          break;
        AfterSync();
        if (t0 + kSub - 1 > least || t0 < latest) { // some column does not see all of the sub-tile: masked in place
#pragma unroll 1
          for (int piece = 0; piece < kSub / 16; ++piece) {
            Pair x[8];
            unsigned y[16];
            TmemLoadPairs(score_address + 16 * piece, x);
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              const int t = t0 + 16 * piece + j;
              y[j] = t < first || t > last ? 0xff800000u : static_cast<unsigned>(x[j / 2] >> 32 * (j & 1));
            }
            TmemStore16(score_address + 16 * piece, y);
          }
          TmemStoreWait();
        }
        float most = -INFINITY;
#pragma unroll 1
        for (int piece = 0; piece < 2; ++piece) {
          Pair x[16];
          TmemLoadPairs(score_address + 32 * piece, x);
          float part[2] = {most, most};
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            float front, back;
            SplitPair(x[j], &front, &back);
            part[j & 1] = Max3(part[j & 1], front, back);
          }
          most = fmaxf(part[0], part[1]);
        }
        const bool raise = fmaf(most, factor, -top) > kRaise;
        if (__any_sync(0xffffffffu, raise)) {
          const float next = raise ? fmaf(most, factor, -kTop) : top, shrink = Exp2(top - next);
          top = next, total *= shrink;
          if (i != 2 * begin_tile) {
            // O as the sub-tile before left it (the one before that is done: this sub-tile's S was asked for after it)
            alive = WarpWait(&sm.o_full[half], (outputs - 1) & 1, abort);
            if (!alive)
              break;
            AfterSync();
#pragma unroll 1
            for (int piece = 0; piece < D / 16; ++piece) {
              Pair y[8];
              TmemLoadPairs(o_address + 16 * piece, y);
              unsigned z[16];
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                const Pair scaled = Mul2(y[j], MakePair(shrink, shrink));
                z[2 * j] = static_cast<unsigned>(scaled), z[2 * j + 1] = static_cast<unsigned>(scaled >> 32);
              }
              TmemStore16(o_address + 16 * piece, z);
            }
          }
        }
        const Pair factors = MakePair(factor, factor), minus_top = MakePair(-top, -top);
        Pair sum[2] = {MakePair(total, 0), MakePair(0, 0)};
#pragma unroll 1
        for (int piece = 0; piece < 2; ++piece) {
          Pair x[16];
          TmemLoadPairs(score_address + 32 * piece, x);
          unsigned packed[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            float p0, p1;
            SplitPair(Fma2(x[j], factors, minus_top), &p0, &p1);
            p0 = Exp2(p0), p1 = Exp2(p1);
            sum[j & 1] = Add2(sum[j & 1], MakePair(p0, p1));
            packed[j] = Pack(p0, p1);
          }
          TmemStore16(score_address + 16 * piece, packed); // over scores that have been read
        }
        float sum0, sum1;
        SplitPair(Add2(sum[0], sum[1]), &sum0, &sum1);
        total = sum0 + sum1;
        TmemStoreWait();
        BeforeSync();
        __syncwarp();
        if (lane == 0)
          BarrierArrive(&sm.p_full[half][sub]);
        ++outputs, jobs += sub;
      }
      if (!alive)
        break;
      // ---- the piece's output ----
      const bool other_half = paired && walk.count > 1; // the second half has had tiles of these columns
      if (paired && half) {
        if (other_half) {
          sm.other[row] = make_float2(top, total);
          __syncwarp();
          if (lane == 0)
            BarrierArrive(&sm.shared_ready);
          // its O may be overwritten only when the first half has read it
          alive = WarpWait(&sm.shared_done, shared++ & 1, abort);
          ++finished;
        }
        continue;
      }
      float own_weight = 1.f, other_weight = 0.f;
      if (other_half) {
        alive = WarpWait(&sm.shared_ready, shared++ & 1, abort) && WarpWait(&sm.o_last[1], other_finished & 1, abort);
        if (!alive)
          break;
        const float2 other = sm.other[row];
        const float larger = fmaxf(top, other.x);
        own_weight = Exp2(top - larger), other_weight = Exp2(other.x - larger);
        top = larger, total = own_weight * total + other_weight * other.y;
      }
      other_finished += !paired || other_half;
      alive = WarpWait(&sm.o_last[half], finished++ & 1, abort);
      if (!alive)
        break;
      AfterSync();
      const bool whole = walk.count == walk.unit.tiles;
      const int slot = walk.at == begin ? 0 : 1;
      float *const partial = PartialOf<D, kColumns>(a, blockIdx.x, slot);
      const float inverse = whole ? (total > 0 ? 1.f / total : 0.f) : 1.f;
      own_weight *= inverse, other_weight *= inverse;
      // Rows of a whole unit go out 32 values at a time through shared memory, four lanes to a row.  Blocks of eight values lie in
      // the order 0 4 1 5 2 6 3 7.
      const Places places = PlacesOf(a, walk.block);
      unsigned char *const out = sm.out[warp];
      const int warp_there = walk.unit.columns - (own - lane); // columns of this warp that exist, if less than 32
#pragma unroll 1
      for (int piece = 0; piece < D / 32; ++piece) {
        float x[32];
        TmemLoad32(o_address + 32 * piece, x);
#pragma unroll
        for (int j = 0; j < 32; ++j)
          x[j] *= own_weight;
        if (other_half) {
          float y[32];
          TmemLoad32(o_address + 128 + 32 * piece, y);
#pragma unroll
          for (int j = 0; j < 32; ++j)
            x[j] = fmaf(y[j], other_weight, x[j]);
        }
#pragma unroll
        for (int b = 0; b < 32; b += 8) {
          const float4 front = make_float4(x[b], x[b + 2], x[b + 4], x[b + 6]), back = make_float4(x[b + 1], x[b + 3], x[b + 5], x[b + 7]);
          if (whole) {
            unsigned char *const to = out + 64 * lane + 16 * ((b / 8) ^ ((lane >> 1) & 3));
            Store4(reinterpret_cast<T *>(to), front), Store4(reinterpret_cast<T *>(to + 8), back);
          } else if (there) {
            *reinterpret_cast<float4 *>(partial + own * D + 32 * piece + b) = front;
            *reinterpret_cast<float4 *>(partial + own * D + 32 * piece + b + 4) = back;
          }
        }
        if (whole) {
          __syncwarp();
#pragma unroll
          for (int c = lane / 4; c < 32; c += 8)
            if (c < warp_there) {
              int sequence_row, h;
              places.Split(own - lane + c, &sequence_row, &h);
              *reinterpret_cast<uint4 *>(static_cast<T *>(a.out) + static_cast<long long>(walk.rows.begin + sequence_row) * a.out_stride +
                                         (walk.head * a.group + h) * D + 32 * piece + 8 * (lane & 3)) =
                  *reinterpret_cast<const uint4 *>(out + 64 * c + 16 * ((lane & 3) ^ ((c >> 1) & 3)));
            }
          __syncwarp();
        }
      }
      if (other_half) {
        BeforeSync();
        __syncwarp();
        if (lane == 0)
          BarrierArrive(&sm.shared_done);
      }
      if (!whole) {
        if (there)
          *reinterpret_cast<float2 *>(partial + kColumns * D + 2 * own) = make_float2(top, total);
        if (!walk.skip && tid == 0) { // the unit begins here and goes on in the next runs
          const long long last = Quotient(walk.at + walk.unit.tiles - 1, share);
          a.split[blockIdx.x] = Split{static_cast<int>(last - blockIdx.x) + 1, slot, walk.rows.begin, walk.block, walk.head, walk.unit.columns};
        }
      }
      BeforeSync(); // reads of O come before the MMAs that the next piece's weights release
    }
  }
  if (!alive) {
    sm.abort = 1;
    Raise(a.bad);
  }
  BeforeSync();
  __syncthreads();
  if (sm.abort) // MMAs that were issued before somebody gave up may still be running: far more time than they need
    for (int i = 0; i < 100; ++i)
      __nanosleep(1000);
  if (warp == kMmaWarp) {
    AfterSync();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(sm.tmem), "r"(512) : "memory");
  }
}

} // namespace

size_t WidePartialBytes(int head_dim) {
  return static_cast<size_t>(kMaxWideGrid) * 2 * kColumns * (head_dim + 2) * sizeof(float);
}

template <typename T, int D> int LaunchWide(const AttentionArgs &a, int sms, cudaStream_t stream) {
  const size_t smem = sizeof(Smem<D>) + 1024; // room to start the struct on a 1024-byte boundary
  if (cudaFuncSetAttribute(WideAttentionKernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)) != cudaSuccess)
    return PADRA_RESOURCE_EXHAUSTED;
  const int grid = min(sms, kMaxWideGrid);
  WideAttentionKernel<T, D><<<grid, kThreads, smem, stream>>>(a);
  if (cudaGetLastError() != cudaSuccess)
    return PADRA_INTERNAL;
  return LaunchJoin<T, D, kColumns>(a, grid, stream);
}
template int LaunchWide<__nv_bfloat16, 64>(const AttentionArgs &, int, cudaStream_t);
template int LaunchWide<__nv_bfloat16, 128>(const AttentionArgs &, int, cudaStream_t);
template int LaunchWide<__half, 64>(const AttentionArgs &, int, cudaStream_t);
template int LaunchWide<__half, 128>(const AttentionArgs &, int, cudaStream_t);

} // namespace attention
} // namespace padra
