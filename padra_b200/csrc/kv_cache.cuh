// The paged 4-bit cache and the description of a call's sequences, shared by the kernels that fill and read them.
#pragma once
#include "common.cuh"

namespace padra {

constexpr int kKvGroup = 32;             // values that share a scale
constexpr float kKvLargest = 57344.f;    // 7 * 8192: the largest magnitude whose codes stay finite as FP16 values
constexpr int kMinPage = 16, kMaxPage = 256;

// The cache as the kernels see it.  A block (one page of one KV head) holds K codes, K scales, V codes, V scales.
struct KvView {
  unsigned char *pool;
  long long pages;
  int page_size, page_shift, kv_heads, head_dim;
  __host__ __device__ int code_bytes() const { return page_size * head_dim / 2; }
  __host__ __device__ int scale_bytes() const { return page_size * head_dim / 16; }
  __host__ __device__ int block_bytes() const { return 2 * (code_bytes() + scale_bytes()); }
  __device__ unsigned char *block(int page, int head) const { // 64-bit offsets: a pool may pass 4 GB
    return pool + (static_cast<long long>(page) * kv_heads + head) * block_bytes();
  }
};

struct SequenceView {
  const int *page_table, *row_begin, *context;
  int count, table_stride, rows, max_rows;
};

inline bool ViewOf(const padra_kv_cache *c, KvView *v) {
  if (!c || !c->pool || reinterpret_cast<uintptr_t>(c->pool) % 16 || c->pages < 1 || c->pages > 0x7fffffffll || c->kv_heads < 1 ||
      c->kv_heads > 1024 || c->page_size < kMinPage || c->page_size > kMaxPage || (c->page_size & (c->page_size - 1)))
    return false;
  int shift = 0;
  while ((1 << shift) < c->page_size)
    ++shift;
  *v = KvView{static_cast<unsigned char *>(c->pool), c->pages, c->page_size, shift, c->kv_heads, c->head_dim};
  return true;
}
inline bool ViewOf(const padra_sequences *s, const KvView &cache, SequenceView *v) {
  // positions are 32-bit: a table may not describe more tokens than that
  if (!s || s->count < 0 || s->rows < 0 || s->max_rows < 0 || s->table_stride < 0 || s->count > (1 << 20) || s->rows > (1 << 24) ||
      (static_cast<long long>(s->table_stride) << cache.page_shift) > (1ll << 30))
    return false;
  if (s->count && (!s->row_begin || !s->context || (s->table_stride && !s->page_table)))
    return false;
  *v = SequenceView{s->page_table, s->row_begin, s->context, s->count, s->table_stride, s->rows, s->max_rows};
  return true;
}
inline bool RowsOk(const void *p, long long stride, int rows, int heads, int head_dim) { // no rows need no memory
  return (p || !rows) && reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride % 8 == 0 && stride >= static_cast<long long>(heads) * head_dim;
}

// Rows and context of sequence s, checked: false (and *bad raised) where they contradict the call.
__device__ __forceinline__ bool SequenceRows(const SequenceView &v, const KvView &cache, int s, int *begin, int *rows, int *context, int *bad) {
  const int b = v.row_begin[s], e = v.row_begin[s + 1], c = v.context[s];
  *begin = b, *rows = e - b, *context = c;
  if (b < 0 || e < b || e > v.rows || e - b > v.max_rows || c < 0 || c > (static_cast<long long>(v.table_stride) << cache.page_shift)) {
    Raise(bad);
    return false;
  }
  return true;
}

// The sequence that owns `row` and the row's position, found by one warp (all lanes get the answer).  Returns -1 for rows
// that belong to nobody, and where the sequence's numbers contradict the call (*bad raised).
__device__ __forceinline__ int LocateRow(const SequenceView &v, const KvView &cache, int row, int *position, int *bad) {
  const int lane = threadIdx.x & 31;
  int s = 0; // sequences that end at or before `row`
#pragma unroll 4
  for (int i = 0; i < v.count; i += 32) {
    const bool before = i + lane < v.count && v.row_begin[i + lane + 1] <= row;
    s += __popc(__ballot_sync(0xffffffffu, before));
  }
  if (s >= v.count)
    return -1;
  int begin, rows, context;
  if (!SequenceRows(v, cache, s, &begin, &rows, &context, bad))
    return -1;
  if (row < begin || row >= begin + rows) { // bounds that do not ascend
    Raise(bad);
    return -1;
  }
  *position = context - rows + (row - begin);
  return s;
}

// Page of a position of sequence s (position within the sequence's context); -1 and *bad raised outside the pool.
__device__ __forceinline__ int PageOf(const SequenceView &v, const KvView &cache, int s, int position, int *bad) {
  const int page = v.page_table[static_cast<long long>(s) * v.table_stride + (position >> cache.page_shift)];
  if (page < 0 || page >= cache.pages) {
    Raise(bad);
    return -1;
  }
  return page;
}

} // namespace padra
