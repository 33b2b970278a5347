// Attention over the paged 4-bit cache for many query rows per sequence (prefill chunks, verifier rows): S = Q K^T and O += P V on
// the 5th-generation tensor cores, accumulators in tensor memory, K and V turned from codes into FP16 operands on the way.
//
// A unit is (sequence, KV head, block of 256 query columns); a column is a row of the sequence with one of the heads that
// share the KV head, so heads of a group share every K and V tile.  A tile is 128 tokens.  As in attention.cu all tiles of a call form
// one list and every CTA (one per SM) takes an equal run of it; pieces of units are joined by JoinKernel.
//   * Eight producer warps load codes and scales one tile ahead into registers and store FP16 rows (value = (code - 8) * scale, one
//     rounding of 2^-11) in the 128-byte-swizzled layout, the same for K (K-major: contraction over the head's values) and V
//     (MN-major: contraction over tokens), so that V needs no transposition.  Values inside a block of eight lie in the order
//     0 4 1 5 2 6 3 7 in which a code word yields pairs; Q is stored in that order and the output put back.
//   * One thread issues the MMAs: S (128 columns x 128 tokens) of each half of the block in its own tensor memory, so that one
//     half's MMAs run under the other half's softmax.  P replaces S in tensor memory as the A operand of O += P V.
//   * Two softmax warpgroups, one per half, one thread per column: no shuffles.  The maximum is raised lazily (by a factor of up to
//     2^15 in FP16 weights), and only then are O and the weights that the tile already has rescaled (the latter rounded to FP16 a second time).
//   * A block with at most 128 columns would leave one half idle: then the halves take even and odd tiles of the SAME columns,
//     each with its own maximum, sum and O, and are joined through tensor memory at the end of the piece.
// Measured (32 heads over 4, head size 128, BF16): 2048 rows behind 32767 tokens 1370 us (828 TFLOP/s), the first 2048 rows of a prompt 100 us, 5
// rows of 8 sequences of up to 32000 tokens 100 us.  Per tile and half some 2900 cycles of softmax, 870 for S and 700 for P V; a producer warp
// takes 2000 to 3500 for its part of a tile.  S waits for the product that reads P, whose place it takes: 512 columns hold no second S beside
// O of two halves of heads of 128 (heads of 64 keep the same places), so the parts overlap between the halves only.
// Tensor memory: S/P of the halves in columns 0 and 128, O in 256 and 384.  Every wait is bounded in time; on expiry the CTA raises the
// error flag and leaves.
#include <type_traits>

#include "attention.cuh"

namespace padra {
namespace attention {
namespace {

constexpr int kTile = 128, kColumns = 256;
constexpr int kSoftmaxWarps = 8, kProducerWarps = 8, kMmaWarp = kSoftmaxWarps + kProducerWarps;
constexpr int kWarps = kMmaWarp + 4, kThreads = kWarps * 32; // whole warpgroups, for the register split; three warps idle
// Registers per thread: launched with 96 (640 threads), then split 2 * 120 + 2 * 88 + 64 = 5 * 96.
constexpr int kSoftmaxRegisters = 120, kProducerRegisters = 88, kMmaRegisters = 64;
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

// What a unit takes beyond its tiles (queries in, output out, the pipeline's filling), in tiles: the list of work counts it, or CTAs with
// many short units would take several times as long as those with a part of a long one.
constexpr int kSetup = 4;

// A CTA's run, piece by piece; every role walks it by itself.  A unit is kSetup + tiles long in the list.
struct Walk {
  long long at, end;
  int s, block, head;
  int from, span;  // the piece's place in its unit, in the list's measure
  int skip, count; // and in tiles: the piece begins `skip` tiles into its unit
  Rows rows;
  Unit unit;
  __device__ __forceinline__ void Place(int x) {
    from = x, span = static_cast<int>(min(static_cast<long long>(kSetup + unit.tiles - x), end - at));
    skip = max(0, x - kSetup), count = max(0, x + span - kSetup) - skip;
  }
  __device__ __forceinline__ void Begin(const AttentionArgs &a, long long first, long long last, int sequence, int first_block, long long offset) {
    at = first, end = last, s = sequence, block = first_block;
    rows = RowsOf(a, s), unit = UnitOf(a, rows, block);
    const int length = kSetup + unit.tiles;
    head = static_cast<int>(Quotient(offset, length));
    Place(static_cast<int>(offset - static_cast<long long>(head) * length));
    if (!count)
      Next(a);
  }
  __device__ __forceinline__ bool More() const { return at < end; }
  __device__ __forceinline__ void Next(const AttentionArgs &a) { // the next piece with tiles
    do {
      at += span;
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
      Place(0);
    } while (!count);
  }
  __device__ __forceinline__ bool Paired() const { return unit.columns <= 128; }
};

template <int D> struct Smem {
  static constexpr int kHalves = D / 64;
  alignas(1024) unsigned char q[2][kHalves][128 * 128]; // rows of 64 values (128 bytes), 16-byte pieces swizzled by row
  alignas(1024) unsigned char k[kStages][kHalves][kTile * 128];
  alignas(1024) unsigned char v[kStages][kHalves][kTile * 128];
  alignas(8) unsigned long long q_full[2], k_full[kStages], k_empty[kStages], v_full[kStages], v_empty[kStages], s_full[2], p_full[2], o_full[2];
  // A piece's queries may be replaced: its last S is done, and every softmax warp has seen them come and read its `column`.  Without the
  // softmax warps' share a run of short pieces could stage queries twice while a warp still wrote rows out, and its wait, which knows
  // one phase from the next only, would have taken the later staging for none.
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
  Walk walk[kMmaWarp + 1]; // every working warp's place in the run: in registers it crowded out what the loops need
  unsigned tmem;
  int abort;
};

// Bounded wait (see BarrierWait) that lets the hardware suspend the thread for up to two microseconds at a time: seventeen warps wait
// here most of the time, and plain polling took issue slots from the ones at work.
__device__ __forceinline__ bool SuspendedWait(unsigned long long *bar, unsigned parity, const volatile int *abort) {
  const unsigned address = SmemAddress(bar);
  unsigned long long started = 0;
  for (;;) {
    unsigned done;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(done)
                 : "r"(address), "r"(parity), "r"(2000u)
                 : "memory");
    if (done)
      return true;
    if (*abort)
      return false;
    unsigned long long now;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
    if (!started)
      started = now;
    else if (now - started > kWaitLimitNs)
      return false;
  }
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
__device__ __forceinline__ void TmemStore32(unsigned taddr, const unsigned (&v)[32]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
               "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
               "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]),
               "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]),
               "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
               : "memory");
}
// Columns of the thread's lane.
__device__ __forceinline__ void TmemLoad16(unsigned taddr, float (&v)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 "
               "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]),
                 "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
               : "r"(taddr)
               : "memory");
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 16; ++i)
    asm volatile("" : "+f"(v[i])); // no use of a value moves up across the wait
}
__device__ __forceinline__ void TmemLoad64(unsigned taddr, float (&v)[64]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x64.b32 "
               "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%64];"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]),
                 "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]),
                 "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]),
                 "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31]),
                 "=f"(v[32]), "=f"(v[33]), "=f"(v[34]), "=f"(v[35]), "=f"(v[36]), "=f"(v[37]), "=f"(v[38]), "=f"(v[39]),
                 "=f"(v[40]), "=f"(v[41]), "=f"(v[42]), "=f"(v[43]), "=f"(v[44]), "=f"(v[45]), "=f"(v[46]), "=f"(v[47]),
                 "=f"(v[48]), "=f"(v[49]), "=f"(v[50]), "=f"(v[51]), "=f"(v[52]), "=f"(v[53]), "=f"(v[54]), "=f"(v[55]),
                 "=f"(v[56]), "=f"(v[57]), "=f"(v[58]), "=f"(v[59]), "=f"(v[60]), "=f"(v[61]), "=f"(v[62]), "=f"(v[63])
               : "r"(taddr)
               : "memory");
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 64; ++i)
    asm volatile("" : "+f"(v[i])); // no use of a value moves up across the wait
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
  uint4 k[kTokens], v[kTokens];
  uint2 k_scale[kTokens], v_scale[kTokens]; // the groups' scales (head size 64: in .x)

  // Lanes of a quarter warp (whose stores go out together) take rows whose swizzle leaves no bank twice: rows t and t + 4 with
  // four chunks, rows {0, 1, 4, 5} or {2, 3, 6, 7} with two.
  static __device__ __forceinline__ int TokenOf(int lane, int i) {
    if constexpr (kChunks == 4)
      return 8 * i + ((lane >> 3) & 3) + ((lane >> 2) & 1) * 4;
    else
      return (lane >> 4) * 8 + ((lane >> 3) & 1) * 2 + ((lane >> 1) & 1) + ((lane >> 2) & 1) * 4;
  }
  // Codes and scales of this warp's 16 tokens from token t on; zeros (scale 0) for tokens outside [low, context) or without a page:
  // their slots may hold anything, and a weight of zero does not make a NaN vanish.
  static __device__ __forceinline__ void Load(const AttentionArgs &a, int page, int head, int t, int low, int context, int offset, uint4 (&words)[kTokens],
                                              uint2 (&scale)[kTokens]) { // offset: of K or V in the block
    const int lane = threadIdx.x & 31, chunk = lane % kChunks;
    const unsigned char *const block = a.cache.block(max(page, 0), head) + offset;
    const int slot = t & (a.cache.page_size - 1), code_bytes = a.cache.code_bytes();
#pragma unroll
    for (int i = 0; i < kTokens; ++i) {
      const int token = TokenOf(lane, i);
      words[i] = make_uint4(0, 0, 0, 0), scale[i] = make_uint2(0, 0);
      if (page >= 0 && t + token < context && t + token >= low) {
        const unsigned char *const codes = block + (slot + token) * (D / 2) + 16 * chunk, *const scales = block + code_bytes + (slot + token) * (D / 16);
        words[i] = __ldg(reinterpret_cast<const uint4 *>(codes));
        if constexpr (kGroups == 4)
          scale[i] = __ldg(reinterpret_cast<const uint2 *>(scales));
        else
          scale[i].x = __ldg(reinterpret_cast<const unsigned *>(scales));
      }
    }
  }
  static __device__ __forceinline__ void Store(unsigned tile, int row, int chunk, const uint4 &codes, const uint2 &scales, const CodeMasks &masks) {
    const unsigned word[4] = {codes.x, codes.y, codes.z, codes.w};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const int place = 4 * chunk + w, piece = 4 * (place % kGroups) + place / kGroups; // word c * groups + g holds piece 4 g + c
      const unsigned pair = (w % kGroups) & 2 ? scales.y : scales.x;                    // place % groups == w % groups
      const __half2 both = *reinterpret_cast<const __half2 *>(&pair), scale = w & 1 ? __high2half2(both) : __low2half2(both);
      const unsigned u = word[w], x = u >> 8;
      StoreShared(tile + PieceOffset(row, piece), make_uint4(Scaled(Low(u, masks), 0x64086408u, scale), Scaled(High(u, masks), 0x54805480u, scale),
                                                             Scaled(Low(x, masks), 0x64086408u, scale), Scaled(High(x, masks), 0x54805480u, scale)));
    }
  }
};

// ---- softmax ----
__device__ __forceinline__ float2 Fma2(float2 x, float2 y, float2 z) {
  float2 r;
  asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\tfma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(x.x), "f"(x.y), "f"(y.x), "f"(y.y), "f"(z.x), "f"(z.y));
  return r;
}
__device__ __forceinline__ float2 Add2(float2 x, float2 y) {
  float2 r;
  asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(x.x), "f"(x.y), "f"(y.x), "f"(y.y));
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
        sm.column[parity][c].factor = FactorOf(a.scale, finite ? power : 1.f);
        sm.column[parity][c].last = c < columns && finite ? position[f] : -1;
      }
    }
  }
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
          cost_mine = static_cast<long long>(kSetup + UnitOf(a, RowsOf(a, item_sequence), item_block).tiles) * a.cache.kv_heads;
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
  const long long share = max(2ll + kSetup, Quotient(total + gridDim.x - 1, gridDim.x)), begin = blockIdx.x * share, end = min(total, begin + share);
  if (tid == 0) {
    a.split[blockIdx.x].pieces = 0;
    sm.abort = 0;
    for (int i = 0; i < 2; ++i) {
      BarrierInit(&sm.q_full[i], kProducerWarps / 2), BarrierInit(&sm.s_full[i], 1);
      BarrierInit(&sm.p_full[i], kSoftmaxWarps / 2), BarrierInit(&sm.o_full[i], 1);
    }
    for (int i = 0; i < kStages; ++i) {
      BarrierInit(&sm.k_full[i], kProducerWarps), BarrierInit(&sm.v_full[i], kProducerWarps);
      BarrierInit(&sm.k_empty[i], 1), BarrierInit(&sm.v_empty[i], 1);
    }
    BarrierInit(&sm.q_empty, 1 + kSoftmaxWarps);
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
  constexpr unsigned tmem = 0; // all 512 columns are this CTA's; addresses known to the compiler make an MMA some 10 instructions instead of 100
  const volatile int *const abort = &sm.abort;
  Walk &walk = sm.walk[min(warp, kMmaWarp)];
  if (lane == 0 && warp <= kMmaWarp)
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
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kProducerRegisters));
    const int mine = 16 * (warp - kSoftmaxWarps), chunk = lane % P::kChunks; // this warp's tokens of a tile
    int tile = 0, page = -1, low = 0; // of the piece: the tile that is loaded next, the page of the warp's tokens in it, the first token seen
    P data;
    auto find = [&]() { // the page is checked only when it is used: its load takes as long as the codes'
      page = -1;
      if (walk.More()) {
        const int t = (walk.unit.first + walk.skip + tile) * kTile + mine;
        // first token that some column of the unit sees
        low = a.window ? max(0, walk.rows.context - walk.rows.rows + walk.block * kColumns / a.group + 1 - a.window) : 0;
        if (t < walk.rows.context && t + 16 > low)
          page = __ldg(a.seq.page_table + static_cast<long long>(walk.s) * a.seq.table_stride + (t >> a.cache.page_shift));
        else
          low = 0x7fffffff; // no token of the warp counts
      }
    };
    // A piece's queries come before its first tile: this warp's 32 columns, once nobody needs those of the piece before.
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
    auto load_k = [&]() {
      if (low != 0x7fffffff && (page < 0 || page >= a.cache.pages))
        Raise(a.bad), page = -1;
      P::Load(a, page, walk.head, (walk.unit.first + walk.skip + tile) * kTile + mine, low, walk.rows.context, 0, data.k, data.k_scale);
    };
    auto load_v = [&]() { // then the page of the tile after it
      P::Load(a, page, walk.head, (walk.unit.first + walk.skip + tile) * kTile + mine, low, walk.rows.context, a.cache.code_bytes() + a.cache.scale_bytes(),
              data.v, data.v_scale);
      if (++tile == walk.count)
        next_piece(), tile = 0;
      find();
    };
    bool have = walk.More(); // a tile has been loaded and not been stored
    if (have) {
      find();
      stage_queries();
      load_k();
      load_v();
    }
    for (unsigned n = 0; have && alive; ++n) {
      const int stage = n & (kStages - 1);
      const unsigned free_parity = ((n / kStages) & 1) ^ 1;
      alive = WarpWait(&sm.k_empty[stage], free_parity, abort);
      if (!alive)
        break;
#pragma unroll
      for (int j = 0; j < P::kTokens; ++j)
        P::Store(SmemAddress(sm.k[stage][0]), mine + P::TokenOf(lane, j), chunk, data.k[j], data.k_scale[j], a.masks);
      FenceToTensorCores();
      __syncwarp();
      if (lane == 0)
        BarrierArrive(&sm.k_full[stage]);
      have = walk.More();
      if (have)
        load_k(); // the next tile's keys come while this one's values are converted, its values while its keys are
      alive = WarpWait(&sm.v_empty[stage], free_parity, abort);
      if (!alive)
        break;
#pragma unroll
      for (int j = 0; j < P::kTokens; ++j)
        P::Store(SmemAddress(sm.v[stage][0]), mine + P::TokenOf(lane, j), chunk, data.v[j], data.v_scale[j], a.masks);
      FenceToTensorCores();
      __syncwarp();
      if (lane == 0)
        BarrierArrive(&sm.v_full[stage]);
      if (have) {
        if (tile == 0) // the next tile begins a piece
          stage_queries();
        load_v();
      }
    }
  } else if (warp >= kMmaWarp) {
    // =============================== MMA issue ===============================
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kMmaRegisters));
    // Job i of a piece: half i & 1 with tile i / 2, or with tile i where both halves work on the same columns.
    if (warp == kMmaWarp && lane == 0) {
      const unsigned s_desc = InstructionDescriptor(kTile), o_desc = InstructionDescriptor(D) | kSecondOperandRowMajor;
      unsigned tiles = 0, jobs_of[2] = {0, 0}, pieces_of[2] = {0, 0}; // all so far: tiles, jobs and staged Q tiles of the halves
      for (; alive && walk.More(); walk.Next(a)) {
        const bool paired = walk.Paired();
        const int jobs = paired ? walk.count : 2 * walk.count;
        auto scores = [&](int i, auto half) { // S of job i
          const int tile = paired ? i : i >> 1, stage = (tiles + tile) & (kStages - 1);
          if (paired || half == 0)
            if (!(alive = SuspendedWait(&sm.k_full[stage], ((tiles + tile) / kStages) & 1, abort)))
              return;
          AfterSync();
          const unsigned q_low = DescriptorLow(SmemAddress(sm.q[paired ? 0 : half][0]), 16), k_low = DescriptorLow(SmemAddress(sm.k[stage][0]), 16);
#pragma unroll
          for (int step = 0; step < D / 16; ++step) {
            const unsigned offset = ((step >> 2) * (128 * 128) + (step & 3) * 32) >> 4;
            MmaStepSS(tmem + 128 * half, q_low + offset, k_low + offset, s_desc, step > 0);
          }
          MmaCommit(&sm.s_full[half]);
          if (paired || half == 1)
            MmaCommit(&sm.k_empty[stage]);
          if (i == jobs - 1)
            MmaCommit(&sm.q_empty);
        };
        auto outputs = [&](int i, auto half) { // O += P V of job i, then S of the job after the next
          const int tile = paired ? i : i >> 1, stage = (tiles + tile) & (kStages - 1);
          if (paired || half == 0)
            if (!(alive = SuspendedWait(&sm.v_full[stage], ((tiles + tile) / kStages) & 1, abort)))
              return;
          if (!(alive = SuspendedWait(&sm.p_full[half], jobs_of[half]++ & 1, abort)))
            return;
          AfterSync();
          const unsigned v_low = DescriptorLow(SmemAddress(sm.v[stage][0]), 128 * 128);
#pragma unroll
          for (int step = 0; step < kTile / 16; ++step)
            MmaStepTS(tmem + 256 + 128 * half, tmem + 128 * half + 8 * step, v_low + step * (2048 >> 4), o_desc, i > 1 || step > 0);
          if (paired || half == 1)
            MmaCommit(&sm.v_empty[stage]);
          if (i + 2 >= jobs)
            MmaCommit(&sm.o_full[half]);
          else
            scores(i + 2, half);
        };
        constexpr std::integral_constant<int, 0> kFirst{};
        constexpr std::integral_constant<int, 1> kSecond{};
        // Q of this piece: the second half's tile is staged only where it has columns of its own
        alive = SuspendedWait(&sm.q_full[0], pieces_of[0]++ & 1, abort);
        if (alive)
          scores(0, kFirst);
        if (alive && !paired)
          alive = SuspendedWait(&sm.q_full[1], pieces_of[1]++ & 1, abort);
        if (alive && jobs > 1)
          scores(1, kSecond);
        for (int i = 0; i < jobs && alive; i += 2) {
          outputs(i, kFirst);
          if (alive && i + 1 < jobs)
            outputs(i + 1, kSecond);
        }
        tiles += walk.count;
      }
      if (!alive) {
        sm.abort = 1;
        Raise(a.bad);
      }
    }
    __syncwarp();
  } else {
    // =============================== softmax ===============================
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegisters));
    const int half = warp / 4, row = tid & 127; // the thread's column of its half, and its lane in tensor memory
    const unsigned lanes = static_cast<unsigned>((warp & 3) * 32) << 16, s_address = tmem + lanes + 128 * half, o_address = tmem + lanes + 256 + 128 * half;
    unsigned jobs = 0, staged[2] = {0, 0}, finished[2] = {0, 0}, shared = 0, pieces = 0; // phases gone by: S, Q, outputs of the halves, joins
    for (; alive && walk.More(); next_piece(), ++pieces) {
      const bool paired = walk.Paired();
      const int own = paired ? row : 128 * half + row; // column of the block
      const bool there = own < walk.unit.columns;
      // the block's columns are staged by the producers, those that both halves work on once
      if (paired || !half) {
        alive = WarpWait(&sm.q_full[0], staged[0]++ & 1, abort);
        staged[1] += !paired;
      } else {
        ++staged[0];
        alive = WarpWait(&sm.q_full[1], staged[1]++ & 1, abort);
      }
      if (!alive)
        break;
      const float factor = sm.column[pieces & 1][own].factor;
      const int last = sm.column[pieces & 1][own].last, first = a.window ? max(0, last - a.window + 1) : 0;
      __syncwarp();
      if (lane == 0)
        BarrierArrive(&sm.q_empty);
      float top = kNever, total = 0;
      const int least = __reduce_min_sync(0xffffffffu, there ? last : 0x7fffffff), latest = __reduce_max_sync(0xffffffffu, there ? first : 0);
      const int first_tile = walk.unit.first + walk.skip;
      const int step = paired ? 2 : 1, begin_tile = paired ? half : 0;
      for (int i = begin_tile; i < walk.count; i += step, ++jobs) {
        const int t0 = (first_tile + i) * kTile;
        alive = WarpWait(&sm.s_full[half], jobs & 1, abort);
        if (!alive)
          break;
        AfterSync();
        if (t0 + kTile - 1 > least || t0 < latest) { // some column does not see all of the tile: masked in place
#pragma unroll 1
          for (int piece = 0; piece < kTile / 16; ++piece) {
            float x[16];
            unsigned y[16];
            TmemLoad16(s_address + 16 * piece, x);
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              const int t = t0 + 16 * piece + j;
              y[j] = t < first || t > last ? 0xff800000u : __float_as_uint(x[j]);
            }
            TmemStore16(s_address + 16 * piece, y);
          }
          TmemStoreWait();
        }
        // 64 scores at a time, from tensor memory once: a maximum that is raised in the second half of the tile scales the first's weights too
        float2 sum[2] = {make_float2(total, 0), make_float2(0, 0)};
#pragma unroll 1
        for (int piece = 0; piece < 2; ++piece) {
          float x[64];
          TmemLoad64(s_address + 64 * piece, x);
          float part[2] = {x[0], x[1]};
#pragma unroll
          for (int j = 2; j < 64; j += 2)
            part[j >> 1 & 1] = Max3(part[j >> 1 & 1], x[j], x[j + 1]);
          const float most = fmaxf(part[0], part[1]);
          const bool raise = fmaf(most, factor, -top) > kRaise;
          if (__any_sync(0xffffffffu, raise)) {
            const float next = raise ? fmaf(most, factor, -kTop) : top, shrink = Exp2(top - next);
            if (raise && fabsf(next) > kLargestTop)
              Raise(a.bad);
            top = next;
#pragma unroll
            for (int k = 0; k < 2; ++k)
              sum[k].x *= shrink, sum[k].y *= shrink;
            if (piece) {
              TmemStoreWait();
#pragma unroll 1
              for (int k = 0; k < 32; k += 16) {
                float y[16];
                TmemLoad16(s_address + k, y);
                unsigned z[16];
#pragma unroll
                for (int j = 0; j < 16; ++j) { // in 32 bits: the factor may be below what FP16 holds, and the product not
                  const float2 p = __half22float2(*reinterpret_cast<const __half2 *>(&y[j]));
                  z[j] = Pack(p.x * shrink, p.y * shrink);
                }
                TmemStore16(s_address + k, z);
              }
            }
            if (i != begin_tile) { // the S that has just come says that the MMAs before it are done with O
#pragma unroll 1
              for (int k = 0; k < D / 16; ++k) {
                float y[16];
                TmemLoad16(o_address + 16 * k, y);
                unsigned z[16];
#pragma unroll
                for (int j = 0; j < 16; ++j)
                  z[j] = __float_as_uint(y[j] * shrink);
                TmemStore16(o_address + 16 * k, z);
              }
            }
            TmemLoad64(s_address + 64 * piece, x); // again: not held over all this
          }
          const float2 factors = make_float2(factor, factor), minus_top = make_float2(-top, -top);
          unsigned packed[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            const float2 e = Fma2(make_float2(x[2 * j], x[2 * j + 1]), factors, minus_top), p = make_float2(Exp2(e.x), Exp2(e.y));
            sum[j & 1] = Add2(sum[j & 1], p);
            packed[j] = Pack(p.x, p.y);
          }
          TmemStore32(s_address + 32 * piece, packed); // over scores that have been read
        }
        sum[0] = Add2(sum[0], sum[1]);
        total = sum[0].x + sum[0].y;
        TmemStoreWait();
        BeforeSync();
        __syncwarp();
        if (lane == 0)
          BarrierArrive(&sm.p_full[half]);
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
          ++finished[1];
        }
        continue;
      }
      float own_weight = 1.f, other_weight = 0.f;
      if (other_half) {
        alive = WarpWait(&sm.shared_ready, shared++ & 1, abort) && WarpWait(&sm.o_full[1], finished[1]++ & 1, abort);
        if (!alive)
          break;
        const float2 other = sm.other[row];
        const float larger = fmaxf(top, other.x);
        own_weight = Exp2(top - larger), other_weight = Exp2(other.x - larger);
        top = larger, total = own_weight * total + other_weight * other.y;
      }
      if (!paired && !half)
        ++finished[1]; // an output that is not this half's business
      alive = WarpWait(&sm.o_full[half], finished[half]++ & 1, abort);
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
          const long long last = Quotient(walk.at - walk.from + kSetup + walk.unit.tiles - 1, share);
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
