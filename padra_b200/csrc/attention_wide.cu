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
//   * One thread issues the MMAs: S (128 columns x 128 tokens) of each half of the block in its own tensor memory, so that one
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

constexpr int kTile = 128, kColumns = 256;
constexpr int kSoftmaxWarps = 8, kProducerWarps = 8, kMmaWarp = kSoftmaxWarps + kProducerWarps, kWarps = kMmaWarp + 1, kThreads = kWarps * 32;
constexpr int kStages = 2;

template <int D> struct Smem {
  static constexpr int kHalves = D / 64;
  alignas(1024) unsigned char q[2][kHalves][128 * 128]; // rows of 64 values (128 bytes), 16-byte pieces swizzled by row
  alignas(1024) unsigned char k[kStages][kHalves][kTile * 128];
  alignas(1024) unsigned char v[kStages][kHalves][kTile * 128];
  alignas(8) unsigned long long q_full[2], k_full[kStages], k_empty[kStages], v_full[kStages], v_empty[kStages], s_full[2], p_full[2], o_full[2];
  unsigned long long shared_ready, shared_done; // the second half's maximum and sum are there / have been used
  float2 other[128];
  int item_begin[kThreads];
  long long scan[kWarps], start_offset;
  int start_sequence, start_block;
  unsigned tmem;
  int abort;
};

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
  __device__ __forceinline__ void Begin(const AttentionArgs &a, long long from, long long to, int sequence, int first_block, long long offset) {
    at = from, end = to, s = sequence, block = first_block;
    rows = RowsOf(a, s), unit = UnitOf(a, rows, block);
    head = static_cast<int>(Quotient(offset, unit.tiles)), skip = static_cast<int>(offset - static_cast<long long>(head) * unit.tiles);
    count = static_cast<int>(min(static_cast<long long>(unit.tiles - skip), end - at));
  }
  __device__ __forceinline__ bool More() const { return at < end; }
  __device__ __forceinline__ void Next(const AttentionArgs &a) {
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

// One lane polls for its warp: true for all lanes or for none.
__device__ __forceinline__ bool WarpWait(unsigned long long *bar, unsigned parity, const volatile int *abort) {
  int done = 0;
  if ((threadIdx.x & 31) == 0)
    done = BarrierWait(bar, parity, abort, 0);
  return __shfl_sync(0xffffffffu, done, 0) != 0;
}
__device__ __forceinline__ void FenceToTensorCores() { // this thread's shared-memory writes before the tensor cores' reads
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}
__device__ __forceinline__ void BeforeSync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void AfterSync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// V: rows of 64 values, one per token; the contraction runs over rows.  Blocks of 64 output values are `leading` bytes apart,
// groups of eight tokens 1024.
__device__ __forceinline__ unsigned long long RowMajorOperandDescriptor(unsigned smem_address, unsigned leading) {
  return static_cast<unsigned long long>((smem_address & 0x3ffffu) >> 4) | (static_cast<unsigned long long>(leading >> 4) << 16) |
         (static_cast<unsigned long long>(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
constexpr unsigned kSecondOperandRowMajor = 1u << 16; // instruction descriptor: B is MN-major
__device__ __forceinline__ void MmaTS(unsigned tmem_d, unsigned tmem_a, unsigned long long b_desc, unsigned idesc, bool accumulate) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
               "r"(tmem_a), "l"(b_desc), "r"(idesc), "r"(accumulate ? 1u : 0u)
               : "memory");
}
__device__ __forceinline__ void TmemStore16(unsigned taddr, const unsigned (&v)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr), "r"(v[0]),
               "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]),
               "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
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
  // Codes and scales of this warp's 16 tokens from token t on; zeros (scale 0) for tokens at and beyond `context` or without a page.
  __device__ __forceinline__ void Load(const AttentionArgs &a, int page, int head, int t, int context) {
    const int lane = threadIdx.x & 31, chunk = lane % kChunks;
    const unsigned char *const block = a.cache.block(max(page, 0), head);
    const int slot = t & (a.cache.page_size - 1), code_bytes = a.cache.code_bytes(), both = code_bytes + a.cache.scale_bytes();
#pragma unroll
    for (int i = 0; i < kTokens; ++i) {
      const int token = TokenOf(lane, i);
      k[i] = v[i] = make_uint4(0, 0, 0, 0), k_scale[i] = v_scale[i] = make_uint2(0, 0);
      if (page >= 0 && t + token < context) {
        const unsigned char *const codes = block + (slot + token) * (D / 2) + 16 * chunk, *const scales = block + code_bytes + (slot + token) * (D / 16);
        k[i] = __ldg(reinterpret_cast<const uint4 *>(codes)), v[i] = __ldg(reinterpret_cast<const uint4 *>(codes + both));
        if constexpr (kGroups == 4) {
          k_scale[i] = __ldg(reinterpret_cast<const uint2 *>(scales)), v_scale[i] = __ldg(reinterpret_cast<const uint2 *>(scales + both));
        } else {
          k_scale[i].x = __ldg(reinterpret_cast<const unsigned *>(scales)), v_scale[i].x = __ldg(reinterpret_cast<const unsigned *>(scales + both));
        }
      }
    }
  }
  static __device__ __forceinline__ void Store(unsigned char *tile, int row, int chunk, const uint4 &codes, const uint2 &scales) {
    const unsigned word[4] = {codes.x, codes.y, codes.z, codes.w};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const int place = 4 * chunk + w, piece = 4 * (place % kGroups) + place / kGroups; // word c * groups + g holds piece 4 g + c
      const unsigned pair = (w % kGroups) & 2 ? scales.y : scales.x;                    // place % groups == w % groups
      const __half2 both = *reinterpret_cast<const __half2 *>(&pair), scale = w & 1 ? __high2half2(both) : __low2half2(both);
      const unsigned u = word[w], x = u >> 8;
      *reinterpret_cast<uint4 *>(tile + PieceOffset(row, piece)) = make_uint4(Scaled(Low(u), 0x64086408u, scale), Scaled(High(u), 0x54805480u, scale),
                                                                              Scaled(Low(x), 0x64086408u, scale), Scaled(High(x), 0x54805480u, scale));
    }
  }
};

// ---- softmax ----
template <typename T, int D> struct Column { // one query column of a block
  float factor, top, sum;
  int first, last; // tokens it sees
};

// Stages one query row as FP16 (divided by a power of two, times the sign of scale) into row `row` of a half's Q tile.
template <typename T, int D>
__device__ __forceinline__ void StageQuery(const AttentionArgs &a, const Rows &r, int head, int place, bool there, unsigned char *tile, int row,
                                           Column<T, D> *to) {
  const int sequence_row = place / a.group, h = head * a.group + place % a.group, position = r.context - r.rows + sequence_row;
  const bool load = there && position >= 0;
  const T *const from = static_cast<const T *>(a.q) + static_cast<long long>(r.begin + sequence_row) * a.q_stride + h * D;
  uint4 raw[D / 8];
#pragma unroll
  for (int i = 0; i < D / 8; ++i)
    raw[i] = load ? *reinterpret_cast<const uint4 *>(from + 8 * i) : make_uint4(0, 0, 0, 0);
  float most = 0;
  bool finite = true;
#pragma unroll
  for (int i = 0; i < D / 8; ++i) {
    float x[8];
    Widen(raw[i], from, x);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      finite &= isfinite(x[j]) != 0;
      most = fmaxf(most, fabsf(x[j]));
    }
  }
  if (!finite)
    Raise(a.bad);
  const int exponent = most > 0 && finite ? min(126, max(-126, ilogbf(most))) : 0;
  const float shrink = finite ? ldexpf(a.sign, -exponent) : 0.f;
#pragma unroll
  for (int i = 0; i < D / 8; ++i) {
    float x[8];
    Widen(raw[i], from, x);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      x[j] = finite ? x[j] * shrink : 0.f;
    *reinterpret_cast<uint4 *>(tile + PieceOffset(row, i)) = make_uint4(Pack(x[0], x[4]), Pack(x[1], x[5]), Pack(x[2], x[6]), Pack(x[3], x[7]));
  }
  to->factor = a.scale * ldexpf(1.f, exponent), to->top = kNever, to->sum = 0;
  to->last = there && finite ? position : -1;
  to->first = a.window ? max(0, to->last - a.window + 1) : 0;
}

// Smallest `last` and largest `first` over the warp's columns that exist: a tile inside them needs no mask.
__device__ __forceinline__ int WarpMin(int x) { return __reduce_min_sync(0xffffffffu, x); }
__device__ __forceinline__ int WarpMax(int x) { return __reduce_max_sync(0xffffffffu, x); }

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
      BarrierInit(&sm.q_full[i], kSoftmaxWarps / 2), BarrierInit(&sm.s_full[i], 1);
      BarrierInit(&sm.p_full[i], kSoftmaxWarps / 2), BarrierInit(&sm.o_full[i], 1);
    }
    for (int i = 0; i < kStages; ++i) {
      BarrierInit(&sm.k_full[i], kProducerWarps), BarrierInit(&sm.v_full[i], kProducerWarps);
      BarrierInit(&sm.k_empty[i], 1), BarrierInit(&sm.v_empty[i], 1);
    }
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
  const unsigned tmem = sm.tmem;
  const volatile int *const abort = &sm.abort;
  Walk walk;
  walk.Begin(a, begin, end, sm.start_sequence, sm.start_block, sm.start_offset);
  bool alive = true;

  if (warp >= kSoftmaxWarps && warp < kMmaWarp) {
    // =============================== producers ===============================
    using P = Producer<D>;
    const int mine = 16 * (warp - kSoftmaxWarps), chunk = lane % P::kChunks; // this warp's tokens of a tile
    Walk ahead = walk; // the piece of the tile that is loaded next
    int ahead_tile = 0;
    P next;
    int next_page = -1;
    auto low_of = [&](const Walk &w) { // first token that some column of the unit sees
      return a.window ? max(0, w.rows.context - w.rows.rows + w.block * kColumns / a.group + 1 - a.window) : 0;
    };
    auto find = [&]() { // the page of the warp's tokens in the tile at `ahead`
      next_page = -1;
      if (ahead.More()) {
        const int t = (ahead.unit.first + ahead.skip + ahead_tile) * kTile + mine;
        if (t < ahead.rows.context && t + 16 > low_of(ahead))
          next_page = PageOf(a.seq, a.cache, ahead.s, t, a.bad);
      }
    };
    auto load = [&]() { // that tile's codes, then the page of the one after it
      if (ahead.More()) {
        next.Load(a, next_page, ahead.head, (ahead.unit.first + ahead.skip + ahead_tile) * kTile + mine, ahead.rows.context);
        if (++ahead_tile == ahead.count)
          ahead.Next(a), ahead_tile = 0;
        find();
      }
    };
    find();
    load();
    for (unsigned n = 0; alive && walk.More(); walk.Next(a))
      for (int i = 0; i < walk.count; ++i, ++n) {
        const P now = next;
        load();
        const int stage = n & (kStages - 1);
        const unsigned free_parity = ((n / kStages) & 1) ^ 1;
        alive = WarpWait(&sm.k_empty[stage], free_parity, abort);
        if (!alive)
          break;
#pragma unroll
        for (int j = 0; j < P::kTokens; ++j)
          P::Store(sm.k[stage][0], mine + P::TokenOf(lane, j), chunk, now.k[j], now.k_scale[j]);
        FenceToTensorCores();
        __syncwarp();
        if (lane == 0)
          BarrierArrive(&sm.k_full[stage]);
        alive = WarpWait(&sm.v_empty[stage], free_parity, abort);
        if (!alive)
          break;
#pragma unroll
        for (int j = 0; j < P::kTokens; ++j)
          P::Store(sm.v[stage][0], mine + P::TokenOf(lane, j), chunk, now.v[j], now.v_scale[j]);
        FenceToTensorCores();
        __syncwarp();
        if (lane == 0)
          BarrierArrive(&sm.v_full[stage]);
      }
  } else if (warp == kMmaWarp) {
    // =============================== MMA issue ===============================
    // Job i of a piece: half i & 1 with tile i / 2, or with tile i where both halves work on the same columns.
    if (lane == 0) {
      const unsigned s_desc = InstructionDescriptor(kTile), o_desc = InstructionDescriptor(D) | kSecondOperandRowMajor;
      unsigned tiles = 0, jobs_of[2] = {0, 0}, pieces_of[2] = {0, 0}; // all so far: tiles, jobs and staged Q tiles of the halves
      for (; alive && walk.More(); walk.Next(a)) {
        const bool paired = walk.Paired();
        const int jobs = paired ? walk.count : 2 * walk.count;
        auto scores = [&](int i) { // S of job i
          const int half = i & 1, tile = paired ? i : i >> 1, stage = (tiles + tile) & (kStages - 1);
          if (paired || half == 0)
            if (!(alive = BarrierWait(&sm.k_full[stage], ((tiles + tile) / kStages) & 1, abort, 0)))
              return;
          AfterSync();
          const unsigned q_address = SmemAddress(sm.q[paired ? 0 : half][0]), k_address = SmemAddress(sm.k[stage][0]);
#pragma unroll
          for (int step = 0; step < D / 16; ++step) {
            const unsigned offset = (step >> 2) * (128 * 128) + (step & 3) * 32;
            MmaSS(tmem + 128 * half, SwizzledOperandDescriptor(q_address + offset), SwizzledOperandDescriptor(k_address + offset), s_desc, step > 0);
          }
          MmaCommit(&sm.s_full[half]);
          if (paired || half == 1)
            MmaCommit(&sm.k_empty[stage]);
        };
        // Q of this piece: the second half's tile is staged only where it has columns of its own
        alive = BarrierWait(&sm.q_full[0], pieces_of[0]++ & 1, abort, 0);
        if (alive)
          scores(0);
        if (alive && !paired)
          alive = BarrierWait(&sm.q_full[1], pieces_of[1]++ & 1, abort, 0);
        if (alive && jobs > 1)
          scores(1);
        for (int i = 0; i < jobs && alive; ++i) {
          const int half = i & 1, tile = paired ? i : i >> 1, stage = (tiles + tile) & (kStages - 1);
          if (paired || half == 0)
            if (!(alive = BarrierWait(&sm.v_full[stage], ((tiles + tile) / kStages) & 1, abort, 0)))
              break;
          if (!(alive = BarrierWait(&sm.p_full[half], jobs_of[half]++ & 1, abort, 0)))
            break;
          AfterSync();
          const unsigned v_address = SmemAddress(sm.v[stage][0]);
#pragma unroll
          for (int step = 0; step < kTile / 16; ++step)
            MmaTS(tmem + 256 + 128 * half, tmem + 128 * half + 8 * step, RowMajorOperandDescriptor(v_address + step * 2048, 128 * 128), o_desc,
                  i > 1 || step > 0);
          if (paired || half == 1)
            MmaCommit(&sm.v_empty[stage]);
          if (i + 2 >= jobs)
            MmaCommit(&sm.o_full[half]);
          else
            scores(i + 2);
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
    const int half = warp / 4, row = tid & 127; // the thread's column of its half, and its lane in tensor memory
    const unsigned lanes = static_cast<unsigned>((warp & 3) * 32) << 16, s_address = tmem + lanes + 128 * half, o_address = tmem + lanes + 256 + 128 * half;
    unsigned jobs = 0, finished[2] = {0, 0}, shared = 0; // phases gone by: S tiles, outputs of the halves, joined pieces
    for (; alive && walk.More(); walk.Next(a)) {
      const bool paired = walk.Paired();
      const int own = paired ? row : 128 * half + row, place = walk.block * kColumns + own;
      const bool there = own < walk.unit.columns;
      Column<T, D> column;
      // where both halves work on the same columns, the first one stages them; the second needs the numbers only
      StageQuery<T, D>(a, walk.rows, walk.head, place, there, sm.q[half][0], row, &column);
      FenceToTensorCores();
      __syncwarp();
      if (lane == 0 && !(paired && half))
        BarrierArrive(&sm.q_full[half]);
      const int least = WarpMin(there ? column.last : 0x7fffffff), latest = WarpMax(there ? column.first : 0);
      const int first_tile = walk.unit.first + walk.skip;
      const int step = paired ? 2 : 1, begin_tile = paired ? half : 0;
      for (int i = begin_tile; i < walk.count; i += step, ++jobs) {
        const int t0 = (first_tile + i) * kTile;
        const bool edge = t0 + kTile - 1 > least || t0 < latest; // some column does not see all of the tile
        alive = WarpWait(&sm.s_full[half], jobs & 1, abort);
        if (!alive)
          break;
        AfterSync();
        float most = -INFINITY;
#pragma unroll
        for (int piece = 0; piece < 4; ++piece) {
          float x[32];
          TmemLoad32(s_address + 32 * piece, x);
          if (edge) {
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              const int t = t0 + 32 * piece + j;
              x[j] = t < column.first || t > column.last ? -INFINITY : x[j];
            }
          }
#pragma unroll
          for (int j = 0; j < 32; ++j)
            most = fmaxf(most, x[j]);
        }
        const bool raise = fmaf(most, column.factor, -column.top) > kRaise;
        if (__any_sync(0xffffffffu, raise)) {
          const float next = raise ? fmaf(most, column.factor, -kTop) : column.top, shrink = Exp2(column.top - next);
          column.top = next, column.sum *= shrink;
          if (i != begin_tile) { // the S that has just come says that the MMAs before it are done with O
#pragma unroll 1
            for (int piece = 0; piece < D / 32; ++piece) {
              float x[32];
              TmemLoad32(o_address + 32 * piece, x);
#pragma unroll
              for (int j = 0; j < 32; ++j)
                x[j] *= shrink;
              TmemStore32(o_address + 32 * piece, x);
            }
          }
        }
        float sum = 0;
#pragma unroll
        for (int piece = 0; piece < 4; ++piece) {
          float x[32];
          TmemLoad32(s_address + 32 * piece, x);
#pragma unroll
          for (int j = 0; j < 32; ++j)
            x[j] = Exp2(fmaf(x[j], column.factor, -column.top));
          if (edge) {
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              const int t = t0 + 32 * piece + j;
              x[j] = t < column.first || t > column.last ? 0.f : x[j];
            }
          }
          unsigned packed[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            sum += x[2 * j] + x[2 * j + 1];
            packed[j] = Pack(x[2 * j], x[2 * j + 1]);
          }
          TmemStore16(s_address + 16 * piece, packed); // over scores that have been read
        }
        column.sum += sum;
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
      float own_weight = 1.f, other_weight = 0.f;
      if (paired && half) {
        if (other_half) {
          sm.other[row] = make_float2(column.top, column.sum);
          __syncwarp();
          if (lane == 0)
            BarrierArrive(&sm.shared_ready);
          // its O may be overwritten only when the first half has read it
          alive = WarpWait(&sm.shared_done, shared++ & 1, abort);
          ++finished[1];
        }
        continue;
      }
      if (other_half) {
        alive = WarpWait(&sm.shared_ready, shared++ & 1, abort) && WarpWait(&sm.o_full[1], finished[1]++ & 1, abort);
        if (!alive)
          break;
        const float2 other = sm.other[row];
        const float top = fmaxf(column.top, other.x);
        own_weight = Exp2(column.top - top), other_weight = Exp2(other.x - top);
        column.top = top, column.sum = own_weight * column.sum + other_weight * other.y;
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
      const float inverse = whole ? (column.sum > 0 ? 1.f / column.sum : 0.f) : 1.f;
      own_weight *= inverse, other_weight *= inverse;
      const int sequence_row = place / a.group, h = walk.head * a.group + place % a.group;
      T *const out = static_cast<T *>(a.out) + static_cast<long long>(walk.rows.begin + sequence_row) * a.out_stride + h * D;
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
        if (there) { // blocks of eight lie in the order 0 4 1 5 2 6 3 7
#pragma unroll
          for (int b = 0; b < 32; b += 8) {
            const float4 first = make_float4(x[b], x[b + 2], x[b + 4], x[b + 6]), second = make_float4(x[b + 1], x[b + 3], x[b + 5], x[b + 7]);
            if (whole) {
              Store4(out + 32 * piece + b, first), Store4(out + 32 * piece + b + 4, second);
            } else {
              *reinterpret_cast<float4 *>(partial + own * D + 32 * piece + b) = first;
              *reinterpret_cast<float4 *>(partial + own * D + 32 * piece + b + 4) = second;
            }
          }
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
          *reinterpret_cast<float2 *>(partial + kColumns * D + 2 * own) = make_float2(column.top, column.sum);
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
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
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
