// Pages and lines of the cache that move: whole pages copied for a sequence that goes on from another one's tokens, and
// the drafted tokens that were taken moved together behind their sequence's tokens.
#include "common.h"
#include "yalm_hip.h"

namespace {

// ---------------------------------------------------------------------------
// copy: block src[i] of every line of a (and of b) to block dst[i].  Bound by memory: every byte is read once and written
// once.  The parts of a block run fastest in the launch order: workgroups that run together then write one run of memory, where
// the same part of several blocks, powers of two apart, would crowd into few memory channels (seven copies of one page, 32
// lines of 128 KB, from a warm cache 18.2 -> 12.3 us).  Nothing is read again soon, so loads and stores are non-temporal (96 pages of
// 28 lines 264 -> 248 us, 5.7 TB/s; with eight pieces a thread 255, with two 231, but 19.9 for the seven copies).
// ---------------------------------------------------------------------------
constexpr int COPY_THREADS = 256;
constexpr int COPY_PIECES = 4;                   // pieces a thread has in flight
typedef unsigned piece16 __attribute__((ext_vector_type(4)));

template <typename P>
__global__ __launch_bounds__(COPY_THREADS) void copy_blocks_kernel(P* a, P* b, int n_lines, int n_blocks, long block_pieces,
                                                                   const int* __restrict__ src, const int* __restrict__ dst, int n,
                                                                   int parts) {
  const int tid = threadIdx.x;
  const int part = (int)(blockIdx.x % (unsigned)parts);
  unsigned rest = blockIdx.x / (unsigned)parts;
  const int i = (int)(rest % (unsigned)n);
  rest /= (unsigned)n;
  const int line = (int)(rest % (unsigned)n_lines);
  P* base = rest / (unsigned)n_lines == 0 ? a : b;
  const int from = src[i], to = dst[i];
  // of several copies to one block the last one stands
  int again = 0;
  for (int j = i + 1 + tid; j < n; j += COPY_THREADS) again |= dst[j] == to && (unsigned)src[j] < (unsigned)n_blocks;
  const long p0 = (long)part * (COPY_THREADS * COPY_PIECES) + tid;
  const bool fine = (unsigned)from < (unsigned)n_blocks && (unsigned)to < (unsigned)n_blocks && from != to;
  P v[COPY_PIECES];
  const P* s = base + ((size_t)line * n_blocks + (fine ? from : 0)) * block_pieces;
#pragma unroll
  for (int u = 0; u < COPY_PIECES; ++u) v[u] = __builtin_nontemporal_load(s + min(p0 + (long)u * COPY_THREADS, block_pieces - 1));
  if (__syncthreads_or(again) || !fine) return;
  P* d = base + ((size_t)line * n_blocks + to) * block_pieces;
#pragma unroll
  for (int u = 0; u < COPY_PIECES; ++u) {
    const long p = p0 + (long)u * COPY_THREADS;
    if (p < block_pieces) __builtin_nontemporal_store(v[u], d + p);
  }
}

template <typename P>
int launch_copy(void* a, void* b, int n_lines, int n_blocks, long block_bytes, const int* src, const int* dst, int n, hipStream_t stream) {
  const long pieces = block_bytes / (long)sizeof(P);
  const long parts = (pieces + COPY_THREADS * COPY_PIECES - 1) / (COPY_THREADS * COPY_PIECES);
  const long groups = (long)n * parts * n_lines * (b != nullptr ? 2 : 1);
  if (parts > (1l << 30) || groups > 0x7FFFFFFFl) return YALM_ERR_ARG;
  copy_blocks_kernel<P><<<(unsigned)groups, COPY_THREADS, 0, stream>>>((P*)a, (P*)b, n_lines, n_blocks, pieces, src, dst, n, (int)parts);
  return launch_status();
}

// ---------------------------------------------------------------------------
// compaction: line start + keep[k] of a sequence to line start + k, k in turn, for keep ascending: place k is never the source
// of a later move, so that a thread that owns one element of a head's keys and values moves them all without waiting for
// anyone.  Grid (KV head, line, sequence).  What a move of 2-byte values costs is not their bytes but the memory
// they lie in: a value's elements stand 64 bytes apart (pages in blocks) or more, so that every line of a half page is read and written for
// one element of each.  64 sequences that keep up to 7 of 40 tokens, 32 lines of 8 heads of 128 in bfloat16, ask for 54 MB and take 95 us, with
// some 240 MB read and 78 written.  Half pages staged in LDS, read and written 16 bytes at a time, took 93 us with a workgroup for a head and
// 155 with a wave for 64 elements (fewer waves in flight), and were left.
// ---------------------------------------------------------------------------
constexpr int MOVES = 8;                         // moves a thread has in flight

template <typename T>
__global__ void compact_lines_kernel(T* k_pages, T* v_pages, const int* __restrict__ block_table, int table_stride, int n_slots,
                                     int ring_pages, const int* __restrict__ seq_slot, const int* __restrict__ seq_start,
                                     const int* __restrict__ cu_keep, const int* __restrict__ keep, int n_keep, int max_keep,
                                     int n_pages, int n_kv_heads, int hd, int page_layout) {
  const int g = blockIdx.x, line = blockIdx.y, b = blockIdx.z;
  const int slot = seq_slot[b], start = seq_start[b];
  if ((unsigned)slot >= (unsigned)n_slots || start < 0) return;
  const int first = max(cu_keep[b], 0), count = min(min(cu_keep[b + 1], n_keep) - first, max_keep);
  const int* table = block_table + (size_t)slot * table_stride;
  const size_t page_elems = (size_t)n_kv_heads * PAGE * hd;
  const size_t line0 = (size_t)line * n_pages * page_elems + (size_t)g * PAGE * hd;
  // a position's page, or -1
  auto page_of = [&](int pos) {
    const int p = table[pos / PAGE % ring_pages];
    return (unsigned)p < (unsigned)n_pages ? p : -1;
  };
  for (int e = threadIdx.x; e < hd; e += blockDim.x) {
    for (int k0 = 0; k0 < count; k0 += MOVES) {
      T kv[MOVES], vv[MOVES];
      size_t to_k[MOVES], to_v[MOVES];
      bool moves[MOVES];
#pragma unroll
      for (int u = 0; u < MOVES; ++u) {
        const int k = min(k0 + u, count - 1);
        const int from = start + keep[first + k], to = start + k;
        const int p0 = from > to ? page_of(from) : -1, p1 = page_of(to);
        moves[u] = k0 + u < count && p0 >= 0 && p1 >= 0;
        if (moves[u]) {
          const T* kp = k_pages + line0 + p0 * page_elems;
          const T* vp = v_pages + line0 + p0 * page_elems;
          kv[u] = kp[page_k_offset(page_layout, from & (PAGE - 1), e, hd)];
          vv[u] = vp[page_v_offset(page_layout, from & (PAGE - 1), e, hd)];
          to_k[u] = line0 + p1 * page_elems + page_k_offset(page_layout, to & (PAGE - 1), e, hd);
          to_v[u] = line0 + p1 * page_elems + page_v_offset(page_layout, to & (PAGE - 1), e, hd);
        }
      }
#pragma unroll
      for (int u = 0; u < MOVES; ++u)
        if (moves[u]) {
          k_pages[to_k[u]] = kv[u];
          v_pages[to_v[u]] = vv[u];
        }
    }
  }
}

}  // namespace

extern "C" int yalm_copy_blocks(void* a, void* b, int n_lines, int n_blocks, long block_bytes, const int* src, const int* dst, int n,
                                hipStream_t stream) {
  if (n <= 0 || n_lines <= 0) return YALM_OK;
  if (a == nullptr || n_blocks <= 0 || block_bytes <= 0) return YALM_ERR_ARG;
  const uintptr_t at = (uintptr_t)a | (uintptr_t)b | (uintptr_t)block_bytes;
  if ((at & 15) == 0) return launch_copy<piece16>(a, b, n_lines, n_blocks, block_bytes, src, dst, n, stream);
  if ((at & 3) == 0) return launch_copy<unsigned>(a, b, n_lines, n_blocks, block_bytes, src, dst, n, stream);
  if ((at & 1) == 0) return launch_copy<unsigned short>(a, b, n_lines, n_blocks, block_bytes, src, dst, n, stream);
  return launch_copy<unsigned char>(a, b, n_lines, n_blocks, block_bytes, src, dst, n, stream);
}

extern "C" int yalm_compact_lines(void* k_pages, void* v_pages, const int* block_table, int table_stride, int n_slots, int ring_pages,
                                  const int* seq_slot, const int* seq_start, const int* cu_keep, const int* keep, int B, int n_keep,
                                  int max_keep, int n_lines, int n_pages, int n_kv_heads, int head_dim, int page_layout, int dtype,
                                  hipStream_t stream) {
  if (B <= 0 || n_keep <= 0 || max_keep <= 0 || n_lines <= 0) return YALM_OK;
  if (n_pages <= 0 || n_kv_heads <= 0 || head_dim <= 0 || ring_pages <= 0 || ring_pages > table_stride || n_slots <= 0 || n_lines > 65535 ||
      B > 65535 || !page_layout_ok(page_layout, head_dim))
    return YALM_ERR_ARG;
  const dim3 grid(n_kv_heads, n_lines, B);
  const int threads = min(256, (head_dim + WAVE - 1) / WAVE * WAVE);
  if (dtype == YALM_F32)
    compact_lines_kernel<float><<<grid, threads, 0, stream>>>((float*)k_pages, (float*)v_pages, block_table, table_stride, n_slots, ring_pages,
                                                              seq_slot, seq_start, cu_keep, keep, n_keep, max_keep, n_pages, n_kv_heads,
                                                              head_dim, page_layout);
  else if (dtype == YALM_BF16)
    compact_lines_kernel<unsigned short><<<grid, threads, 0, stream>>>((unsigned short*)k_pages, (unsigned short*)v_pages, block_table,
                                                                       table_stride, n_slots, ring_pages, seq_slot, seq_start, cu_keep, keep,
                                                                       n_keep, max_keep, n_pages, n_kv_heads, head_dim, page_layout);
  else
    return YALM_ERR_DTYPE;
  return launch_status();
}
