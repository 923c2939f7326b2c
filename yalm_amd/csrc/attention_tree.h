// Attention of drafted tokens: the arguments of its kernels, and which keys a row sees.
#pragma once
#include "common.h"

struct TreeArgs {
  const void* q;               // [T, n_heads, head_dim]
  const void* k_pages;
  const void* v_pages;
  const int* block_table;
  int table_stride;
  int n_slots;
  int ring_pages;
  const int* seq_slot;         // [B]
  const int* seq_len;          // [B], the drafted tokens included
  const int* cu_nodes;         // [B + 1]
  const unsigned long long* mask;      // [T, mask_words]
  int mask_words;
  const int* positions;        // [T], or null
  void* out;
  float* partial;
  int T, B, n_heads, n_kv_heads, head_dim, window, n_splits, max_nodes, n_pages, page_layout;
  const int* step_max_len;     // [1], or null
  unsigned group_inverse;      // 2^32 / (n_heads / n_kv_heads) and a part more: exact for the columns of groups up to MAX_GROUP
  // the node of a sequence whose query a column is
  __device__ __forceinline__ int node_of(int column) const {
    return group_inverse == 0 ? column : (int)__umulhi((unsigned)column, group_inverse);
  }
};
constexpr int MAX_NODES = 256;                     // of a sequence
constexpr int MAX_GROUP = 4095;                    // column * (what the inverse is too great by) stays below 2^32

// A number of the step's tables, which no kernel writes while one reads them: where all lanes ask for the same one it comes by the
// scalar cache, and no load of a page in flight is waited for with it.
__device__ __forceinline__ int table_entry(const int* p) {
#if defined(__HIP_DEVICE_COMPILE__)
  return *(const __attribute__((address_space(4))) int*)p;
#else
  return *p;
#endif
}

// A sequence of the step: its slot's row of the block table, its rows, its length (0 where it has no slot) and how many tokens it
// held before the drafted ones.
struct TreeSeq {
  int slot, row0, nodes, len, base;
  __device__ __forceinline__ TreeSeq(const TreeArgs& a, int b) {
    slot = table_entry(a.seq_slot + b);
    row0 = table_entry(a.cu_nodes + b);
    nodes = min(table_entry(a.cu_nodes + b + 1), a.T) - row0;
    len = (unsigned)slot < (unsigned)a.n_slots ? table_entry(a.seq_len + b) : 0;
    base = max(len - nodes, 0);
  }
};

__device__ __forceinline__ int tree_page(const TreeArgs& a, const TreeSeq& s, int page) {
  return min(max(table_entry(a.block_table + (size_t)s.slot * a.table_stride + page % a.ring_pages), 0), a.n_pages - 1);
}

// The first of the sequence's own tokens that row r sees (base and more: none).  Without positions a row stands as many places behind
// the base as it has ancestors.
__device__ __forceinline__ int tree_first(const TreeArgs& a, const TreeSeq& s, int r) {
  if (a.window <= 0) return 0;
  int pos = s.base - 1;
  if (a.positions != nullptr) {
    pos = a.positions[r];
  } else {
    for (int w = 0; w < a.mask_words; ++w) pos += __popcll(a.mask[(size_t)r * a.mask_words + w]);
  }
  return max(0, pos - a.window + 1);
}

// Which of the 64 positions of a page row r sees: bit i is position 64 page + i.
__device__ __forceinline__ unsigned long long tree_seen(const TreeArgs& a, const TreeSeq& s, int r, int lo, int page) {
  const unsigned long long all = ~0ull;
  const int p0 = page * PAGE, before = s.base - p0;          // places of the page in front of the drafted tokens
  unsigned long long held = before >= PAGE ? all : before > 0 ? (1ull << before) - 1 : 0;
  const int hidden = lo - p0;
  held = hidden >= PAGE ? 0 : hidden > 0 ? held & (all << hidden) : held;
  unsigned long long drafted = 0;
  if (before < PAGE) {
    const unsigned long long* m = a.mask + (size_t)r * a.mask_words;
    if (before > 0) {
      drafted = m[0] << before;
    } else {
      const int at = -before, w = at >> 6, bit = at & 63;
      if (w < a.mask_words) drafted = m[w] >> bit;
      if (bit != 0 && w + 1 < a.mask_words) drafted |= m[w + 1] << (PAGE - bit);
    }
  }
  const int left = s.len - p0;                               // places of the page that hold a token at all
  if (left < PAGE) drafted = left > 0 ? drafted & ((1ull << left) - 1) : 0;
  return held | drafted;
}
