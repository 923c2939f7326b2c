// Attention of drafted tokens in bfloat16 on the matrix cores: few columns (16 or 32 a workgroup) from registers, more from LDS.
#include "attention_tree_mfma.h"

namespace {

// ---------------------------------------------------------------------------
// More columns: a workgroup of two groups of four waves takes 64 NC columns, a wave 16 NC of them; the groups take every second
// page of a split, which goes from memory straight into LDS (pages in blocks lie there as they are read: a fragment is 1 KB of
// consecutive bytes), the next one in flight while this one is multiplied; the second group hands its results to the first at
// the end.
// ---------------------------------------------------------------------------
template <int HD, int NC>
__global__ __launch_bounds__(512, 1) void attn_tree_lds_kernel(TreeArgs a, int chunks) {
  typedef TreeColumns<bf16, HD, NC> C;
  static_assert(HD % 32 == 0, "pages in blocks");
  constexpr int DT = C::DT, TILE = PAGE * HD;      // elements of a page of a head
  constexpr int NLOAD = TILE / 8 / 256;            // 16-byte pieces a thread takes of it
  extern __shared__ __attribute__((aligned(16))) unsigned char smem_raw[];          // [2][group][keys, values]
  const TreeWork w(a, chunks);
  if (!w.any) return;
  const TreeSeq s(a, w.b);
  const int G = a.n_heads / a.n_kv_heads, cols = min(s.nodes, a.max_nodes) * G, x0 = w.chunk * NC * 64;
  if (x0 >= cols) return;
  const int half = __builtin_amdgcn_readfirstlane(threadIdx.x / 256), tid = threadIdx.x % 256;
  const int wave = __builtin_amdgcn_readfirstlane(tid / WAVE), lane = tid % WAVE, qd = lane / 16, j = lane % 16;
  C col;
  col.begin(a, s, w.g, x0 + wave * 16 * NC, cols, lane);
  __shared__ int least[4];
  if (half == 0 && lane == 0) least[wave] = col.lo_least;
  __syncthreads();
  const int lo = min(min(least[0], least[1]), min(least[2], least[3]));
  const TreePages pages(a, s, w.split, __builtin_amdgcn_readfirstlane(min(lo, s.base)) / PAGE);
  const float scale = 1.4426950408889634f / sqrtf((float)HD);
  const size_t page_elems = (size_t)a.n_kv_heads * PAGE * HD;
  const bf16* k0 = (const bf16*)a.k_pages + (size_t)w.g * PAGE * HD;
  const bf16* v0 = (const bf16*)a.v_pages + (size_t)w.g * PAGE * HD;
  auto fetch = [&](int page, int buf) {
#if defined(__HIP_DEVICE_COMPILE__)
    const size_t at = (size_t)__builtin_amdgcn_readfirstlane(tree_page(a, s, page)) * page_elems;
    unsigned char* to = smem_raw + (size_t)((buf * 2 + half) * 2) * TILE * sizeof(bf16);
#pragma unroll
    for (int p = 0; p < NLOAD; ++p) {
      __builtin_amdgcn_global_load_lds(k0 + at + (tid + p * 256) * 8, to + (wave + p * 4) * 1024, 16, 0, 0);
      __builtin_amdgcn_global_load_lds(v0 + at + (tid + p * 256) * 8, to + TILE * sizeof(bf16) + (wave + p * 4) * 1024, 16, 0, 0);
    }
#endif
  };
  const bool live = x0 + wave * 16 * NC < cols;    // a wave without columns only fetches
  if (pages.begin + half < pages.end) fetch(pages.begin + half, 0);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  int buf = 0;
  for (int first = pages.begin; first < pages.end; first += 2, buf ^= 1) {
    const int ap = first + half;
    if (ap + 2 < pages.end) fetch(ap + 2, buf ^ 1);          // read before the last barrier
    if (ap < pages.end && live) {
      const bf16* ks = reinterpret_cast<const bf16*>(smem_raw) + (size_t)((buf * 2 + half) * 2) * TILE;
      const bf16* vs = ks + TILE;
      auto values = [&](int dt, int t) { return ld8(vs + C::value_place(dt, t, qd, j)); };
      col.page(a, s, ap, qd, scale, [&](int t, int k) { return ld8(ks + C::key_place(t, k, qd, j)); }, values, values, []() {});
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");         // this wave's share of the next page has landed
    __syncthreads();
  }
  // the second group hands its maxima, sums and results to the first, which merges and writes
  f32x4* mo = reinterpret_cast<f32x4*>(smem_raw);            // [NC][DT][256]
  float* ml = reinterpret_cast<float*>(mo + NC * DT * 256);  // [NC][2][256]
  if (half == 1) {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) mo[(c * DT + dt) * 256 + tid] = col.o[c][dt];
      ml[(c * 2) * 256 + tid] = col.m[c];
      ml[(c * 2 + 1) * 256 + tid] = col.l[c];
    }
  }
  __syncthreads();
  if (half == 1) return;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const float m2 = ml[(c * 2) * 256 + tid], l2 = ml[(c * 2 + 1) * 256 + tid];
    const float m = fmaxf(col.m[c], m2);
    const float f1 = __builtin_amdgcn_exp2f(col.m[c] - m), f2 = __builtin_amdgcn_exp2f(m2 - m);
    const float lt = fold_column(col.l[c] * f1 + l2 * f2, [](float u, float v) { return u + v; });
    const int x = x0 + (wave * NC + c) * 16 + j;
    if (x >= cols) continue;
    const size_t head = (size_t)(s.row0 + x / G) * a.n_heads + w.g * G + x % G;
    const float inv = tree_inverse(lt);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
      tree_store<bf16, HD>(a, head, w.split, dt * 16 + 4 * qd, col.o[c][dt] * f1 + mo[(c * DT + dt) * 256 + tid] * f2, inv);
    if (a.n_splits > 1 && qd == 0)
      *reinterpret_cast<float2*>(a.partial + (head * a.n_splits + w.split) * (HD + 2) + HD) = make_float2(m, lt);
  }
}

template <int HD, int NC>
int launch_lds(const TreeArgs& a, hipStream_t stream) {
  constexpr int bytes = 8 * PAGE * HD * (int)sizeof(bf16), merge = NC * (HD / 16 * 16 + 8) * 256;
  constexpr int lds = bytes > merge ? bytes : merge;
  auto kernel = &attn_tree_lds_kernel<HD, NC>;
  if (lds > 60 * 1024) {
    static LdsAllowance allowed;
    if (int rc = allow_dynamic_lds(allowed, (const void*)kernel, lds); rc != YALM_OK) return rc;
  }
  const int chunks = ((long)a.max_nodes * (a.n_heads / a.n_kv_heads) + NC * 64 - 1) / (NC * 64);
  const long units = (long)a.n_splits * a.n_kv_heads * a.B, groups = (units + 7) / 8 * 8 * chunks;
  if (groups > 0x7FFFFFFFl) return YALM_ERR_ARG;
  kernel<<<(unsigned)groups, 512, lds, stream>>>(a, chunks);
  return launch_status();
}
template <int HD>
int launch_hd(const TreeArgs& a, hipStream_t stream) {
  const long cols = (long)a.max_nodes * (a.n_heads / a.n_kv_heads);
  if (cols <= 16) return launch_tree<bf16, HD, 1>(a, stream);
  if constexpr (HD % 32 == 0) {
    if (cols > 64) return launch_lds<HD, 2>(a, stream);
    if (cols > 32) return launch_lds<HD, 1>(a, stream);
  }
  return launch_tree<bf16, HD, 2>(a, stream);
}

}  // namespace

int yalm_attn_tree_bf16_mfma(const TreeArgs& a, hipStream_t stream) {
  switch (a.head_dim) {
    case 16: return launch_hd<16>(a, stream);
    case 32: return launch_hd<32>(a, stream);
    case 48: return launch_hd<48>(a, stream);
    case 64: return launch_hd<64>(a, stream);
    case 80: return launch_hd<80>(a, stream);
    case 96: return launch_hd<96>(a, stream);
    case 112: return launch_hd<112>(a, stream);
    case 128: return launch_hd<128>(a, stream);
  }
  return YALM_ERR_ARG;
}
