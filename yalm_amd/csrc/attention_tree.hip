// Attention of drafted tokens over the paged cache.  A sequence brings n tokens at once, a tree: their keys and values lie at
// the cache positions base ... base + n - 1 behind the base tokens that it holds, and token r sees the base tokens (those its
// window covers, counted from its position) and of the drafted ones those whose bit its mask names - itself and its ancestors:
//
//   out[r] = sum_j p[r, j] v[j],  p[r, j] = exp(s[r, j]) / sum over the seen keys,  s = q[r] . k[j] / sqrt(head_dim)
//
// A key that a row does not see does not reach it, whatever it holds.  A row that sees nothing gives zeros.
#include <float.h>
#include "common.h"
#include "attention_tree.h"
#include "yalm_hip.h"

int yalm_attn_tree_bf16_mfma(const TreeArgs& a, hipStream_t stream);       // attention_tree_bf16.hip, attention_tree_f32.hip
int yalm_attn_tree_f32_mfma(const TreeArgs& a, hipStream_t stream);

namespace {

// the last sequence whose first row is not behind r
__device__ __forceinline__ int sequence_of(const int* cu, int B, int r) {
  int b = 0;
  for (int hi = B - 1; b < hi;) {
    const int mid = (b + hi + 1) >> 1;
    if (cu[mid] <= r) b = mid; else hi = mid - 1;
  }
  return b;
}

// ---------------------------------------------------------------------------
// Every head size and type, in float32 arithmetic: a wave a (row, head), 64 keys at a time, a lane a key for the scores and a
// lane an output element for the mix.  For the shapes that the matrix cores' kernel does not take; every row reads its sequence's keys
// by itself, which is what bounds it (16 nodes of 32 heads of 128 behind 3,056 tokens, bfloat16: 1,344 us, where that kernel takes 15).
// ---------------------------------------------------------------------------
constexpr int MAX_HD = 1024;

template <typename T>
__global__ __launch_bounds__(WAVE) void attn_tree_simple_kernel(TreeArgs a) {
  constexpr int ACC = MAX_HD / WAVE;
  __shared__ float qs[MAX_HD];
  __shared__ float ps[PAGE];
  const int r = blockIdx.x, h = blockIdx.y, lane = threadIdx.x, hd = a.head_dim;
  if (r >= a.cu_nodes[a.B]) return;
  const int b = sequence_of(a.cu_nodes, a.B, r);
  const TreeSeq s(a, b);
  T* out = (T*)a.out + ((size_t)r * a.n_heads + h) * hd;
  const T* q = (const T*)a.q + ((size_t)r * a.n_heads + h) * hd;
  for (int e = lane; e < hd; e += WAVE) qs[e] = to_f32(q[e]);
  __syncthreads();
  const int g = h / (a.n_heads / a.n_kv_heads);
  const size_t page_elems = (size_t)a.n_kv_heads * PAGE * hd;
  const int lo = tree_first(a, s, r);
  const float scale = 1.0f / sqrtf((float)hd);
  float m = -FLT_MAX, l = 0.f, o[ACC];
#pragma unroll
  for (int u = 0; u < ACC; ++u) o[u] = 0.f;
  for (int page = s.len > 0 ? max(0, min(lo, s.base)) / PAGE : 0; page * PAGE < s.len; ++page) {
    const int phys = tree_page(a, s, page);
    const T* kp = (const T*)a.k_pages + phys * page_elems + (size_t)g * PAGE * hd;
    const T* vp = (const T*)a.v_pages + phys * page_elems + (size_t)g * PAGE * hd;
    const unsigned long long seen = tree_seen(a, s, r, lo, page);
    if (seen == 0) continue;
    float score = -INFINITY;
    if ((seen >> lane) & 1) {
      score = 0.f;
      for (int e = 0; e < hd; ++e) score = fmaf(qs[e], to_f32(kp[page_k_offset(a.page_layout, lane, e, hd)]), score);
      score *= scale;
    }
    const float m_new = fmaxf(m, wave_max(score));
    const float corr = expf(m - m_new);
    const float p = (seen >> lane) & 1 ? expf(score - m_new) : 0.f;
    l = l * corr + wave_sum(p);
    m = m_new;
    __syncthreads();
    ps[lane] = p;
    __syncthreads();
#pragma unroll
    for (int u = 0; u < ACC; ++u) {
      const int e = lane + u * WAVE;
      if (e >= hd) break;
      float part = 0.f;
      for (int j = 0; j < PAGE; ++j)
        if ((seen >> j) & 1) part = fmaf(ps[j], to_f32(vp[page_v_offset(a.page_layout, j, e, hd)]), part);
      o[u] = o[u] * corr + part;
    }
  }
  const float inv = l > 0.f ? 1.0f / l : l == l ? 0.f : l;          // a sum that is no number stays one
#pragma unroll
  for (int u = 0; u < ACC; ++u) {
    const int e = lane + u * WAVE;
    if (e < hd) out[e] = from_f32<T>(o[u] * inv);
  }
}

// ---------------------------------------------------------------------------
// The splits' parts [T, n_heads, n_splits, hd + 2] = (sum[hd], maximum as an exponent of 2, denominator), merged in one order: a
// wave a (row, head).  12 splits of 16 rows of 32 heads of 128 4.0 us, 16 of 61 rows 5.4 (16 MB from the cache, 3 TB/s): a launch and two trips to memory.
// ---------------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(256) void attn_tree_merge_kernel(TreeArgs a) {
  const int lane = threadIdx.x % WAVE, hd = a.head_dim, n = a.n_splits, stride = hd + 2;
  const long head = (long)blockIdx.x * (256 / WAVE) + threadIdx.x / WAVE;
  const int r = (int)(head / a.n_heads);
  if (r >= min(a.cu_nodes[a.B], a.T)) return;
  if (r - a.cu_nodes[sequence_of(a.cu_nodes, a.B, r)] >= a.max_nodes) return;
  const float* part = a.partial + head * (long)n * stride;
  float m = -FLT_MAX;
  for (int s = lane; s < n; s += WAVE) m = fmaxf(m, part[(long)s * stride + hd]);
  m = wave_max(m);
  float l = 0.f;
  for (int s = lane; s < n; s += WAVE) l = fmaf(part[(long)s * stride + hd + 1], __builtin_amdgcn_exp2f(part[(long)s * stride + hd] - m), l);
  l = wave_sum(l);
  const float inv = l > 0.f ? 1.0f / l : l == l ? 0.f : l;
  T* out = (T*)a.out + head * hd;
  for (int e = 2 * lane; e < hd; e += 2 * WAVE) {
    float x = 0.f, y = 0.f;
#pragma unroll 4
    for (int s = 0; s < n; ++s) {
      const float* p = part + (long)s * stride;
      const float f = __builtin_amdgcn_exp2f(p[hd] - m);
      const float2 v = *reinterpret_cast<const float2*>(p + e);
      x = fmaf(v.x, f, x);
      y = fmaf(v.y, f, y);
    }
    out[e] = from_f32<T>(x * inv);
    out[e + 1] = from_f32<T>(y * inv);
  }
}

}  // namespace

extern "C" int yalm_attn_tree(const void* q, const void* k_pages, const void* v_pages, const int* block_table, int table_stride,
                              int n_slots, int ring_pages, const int* seq_slot, const int* seq_len, const int* cu_nodes,
                              const long long* mask, int mask_words, const int* positions, void* out, float* partial, int T, int B,
                              int n_heads, int n_kv_heads, int head_dim, int window, int n_splits, int max_nodes, int n_pages,
                              int page_layout, int dtype, int force_simple, const int* step_max_len, hipStream_t stream) {
  if (T <= 0 || B <= 0) return YALM_OK;
  if (n_heads <= 0 || n_kv_heads <= 0 || n_heads % n_kv_heads != 0 || head_dim <= 0 || head_dim > MAX_HD || ring_pages <= 0 ||
      ring_pages > table_stride || n_slots <= 0 || n_pages <= 0 || mask_words <= 0 || n_splits <= 0 || max_nodes <= 0 || max_nodes > MAX_NODES || n_heads > 65535 ||
      !page_layout_ok(page_layout, head_dim))
    return YALM_ERR_ARG;
  const int group = n_heads / n_kv_heads;
  const TreeArgs a = {q, k_pages, v_pages, block_table, table_stride, n_slots, ring_pages, seq_slot, seq_len, cu_nodes,
                      (const unsigned long long*)mask, mask_words, positions, out, partial, T, B, n_heads, n_kv_heads, head_dim, window,
                      n_splits, max_nodes, n_pages, page_layout, step_max_len, group == 1 ? 0u : (unsigned)((1ull << 32) / group + 1)};
  if (dtype != YALM_F32 && dtype != YALM_BF16) return YALM_ERR_DTYPE;
  // The matrix cores' kernels load and store 16 bytes a lane, from pages as the cache keeps them.
  const uintptr_t at = (uintptr_t)q | (uintptr_t)k_pages | (uintptr_t)v_pages | (uintptr_t)out | (n_splits > 1 ? (uintptr_t)partial : 0);
  const bool cores = !force_simple && group <= MAX_GROUP && head_dim % 16 == 0 && head_dim <= 128 && (at & 15) == 0 &&
                     (page_layout == YALM_PAGE_BLOCKS) == (head_dim % 32 == 0);
  if (!cores) {
    if (dtype == YALM_F32) attn_tree_simple_kernel<float><<<dim3(T, n_heads), WAVE, 0, stream>>>(a);
    else attn_tree_simple_kernel<bf16><<<dim3(T, n_heads), WAVE, 0, stream>>>(a);
    return launch_status();
  }
  if (n_splits > 1 && partial == nullptr) return YALM_ERR_ARG;
  const int rc = dtype == YALM_F32 ? yalm_attn_tree_f32_mfma(a, stream) : yalm_attn_tree_bf16_mfma(a, stream);
  if (rc != YALM_OK || n_splits == 1) return rc;
  const long groups = ((long)T * n_heads + 3) / 4;
  if (groups > 0x7FFFFFFFl) return YALM_ERR_ARG;
  if (dtype == YALM_F32) attn_tree_merge_kernel<float><<<(unsigned)groups, 256, 0, stream>>>(a);
  else attn_tree_merge_kernel<bf16><<<(unsigned)groups, 256, 0, stream>>>(a);
  return launch_status();
}
