// Attention of drafted tokens in bfloat16 on the matrix cores: few columns (16 or 32 a workgroup) from registers, more from LDS.
#include "attention_tree_mfma.h"

namespace {

// The columns that a workgroup takes: no more tiles than the step fills.  More than 32 go over LDS, where a page is read once for all of
// them (61 nodes, 244 columns, behind 28,000 tokens: 47.5 us, in 32s from registers 65 with the splits that suit those; 64 sequences of 40 nodes 157, 225).  More than
// 128 go in one workgroup as soon as the halves would not all run at once (61 nodes behind 2,000 tokens, 8 KV heads, no splits: 18 sequences 74 us, in halves 92; 28
// 81 and 100), and in halves as long as they do (16 sequences 48 us, in one 74; one sequence of 28,000 in 16 splits 47.5, in one 71).
int tree_columns(int B, int max_nodes, int n_heads, int n_kv_heads, int head_dim) {
  const long cols = (long)max_nodes * (n_heads / n_kv_heads);
  if (cols <= 16) return 16;
  if (cols <= 32 || head_dim % 32 != 0) return 32;
  if (cols <= 64) return 64;
  return cols > 128 && 2l * B * n_kv_heads > compute_units() ? 256 : 128;
}

// ---------------------------------------------------------------------------
// More columns: eight waves share a run of pages, which go from memory straight into LDS two at a time (pages in blocks: a fragment is 1 KB
// of consecutive bytes), the next two in flight while these are multiplied.  A round of two pages against 128 columns of 128 elements takes 2.0 us, where
// the vector units want 1.07 (322 instructions a wave, two waves a unit), the matrix cores 0.85 and LDS 1.07: with 128 KB of pages a compute unit holds
// one workgroup, whose waves meet at a barrier a round and wait for the pages of the next.
// One sequence of 28,000 tokens and 61 nodes 46 us (2.5 TB/s, 600 TFLOP/s), 64 of up to 3,041 and 40 nodes 146 to 160 (3.6 to 3.9 TB/s).  With up to 64 NC columns
// two groups of four waves take a page each and the second hands its results to the first at the end; with more (`wide`, up
// to 128 NC) all eight waves split the columns and take both pages.  A wave has the tiles wave, wave + 4 (wide: + 8), ... of 16
// columns, and leaves out those that the sequence does not fill.
// ---------------------------------------------------------------------------
template <int HD, int NC>
constexpr int tree_merge_bytes() { return NC * (HD + 8) * 256; }

template <int HD, int NC>
__global__ __launch_bounds__(512, 1) void attn_tree_lds_kernel(TreeArgs a, int chunks, int wide_chunks) {
  typedef TreeColumns<bf16, HD, NC> C;
  static_assert(HD % 32 == 0, "pages in blocks");
  constexpr int DT = C::DT, TILE = PAGE * HD;      // elements of a page of a head
  constexpr int NLOAD = TILE / 8 / 256;            // 16-byte pieces a thread takes of it
  extern __shared__ __attribute__((aligned(16))) unsigned char smem_raw[];          // [2][group][keys, values]
  const TreeWork w(a, chunks);
  if (!w.any) return;
  const TreeSeq s(a, w.b);
  const int G = a.n_heads / a.n_kv_heads, x0 = w.chunk * (wide_chunks ? NC * 128 : NC * 64);
  const int cols = min(min(s.nodes, a.max_nodes) * G, x0 + (wide_chunks ? NC * 128 : NC * 64));
  if (x0 >= cols) return;
  const bool wide = cols - x0 > NC * 64;
  const int half = __builtin_amdgcn_readfirstlane(threadIdx.x / 256), tid = threadIdx.x % 256;
  const int wave = __builtin_amdgcn_readfirstlane(tid / WAVE), lane = tid % WAVE, qd = lane / 16, j = lane % 16;
  // the wave's first tile, and from tile to tile (columns)
  const int mine = x0 + (wide ? wave + 4 * half : wave) * 16, step = wide ? 128 : 64;
  const int tiles = __builtin_amdgcn_readfirstlane(min(NC, max(0, (cols - mine + step - 1) / step)));
  C col;
  col.begin(a, s, w.g, mine, step, cols, lane);
  __shared__ int least[8], most[8];
  if (lane == 0) {
    least[wave + 4 * half] = col.lo_least;
    most[wave + 4 * half] = col.lo_most;
  }
  __syncthreads();
  int lo = least[0], lo_most = most[0];
#pragma unroll
  for (int v = 1; v < 8; ++v) {
    lo = min(lo, least[v]);
    lo_most = max(lo_most, most[v]);
  }
  lo_most = col.lo_most = __builtin_amdgcn_readfirstlane(lo_most);       // which pages are at an edge is the workgroup's matter
  const TreePages pages(a, s, w.split, __builtin_amdgcn_readfirstlane(min(lo, s.base)) / PAGE);
  const float scale = 1.4426950408889634f / sqrtf((float)HD);
  const size_t page_elems = (size_t)a.n_kv_heads * PAGE * HD;
  const bf16* k0 = (const bf16*)a.k_pages + (size_t)w.g * PAGE * HD;
  const bf16* v0 = (const bf16*)a.v_pages + (size_t)w.g * PAGE * HD;
  auto fetch = [&](int phys, int buf) {          // phys: the page's place in the pool
#if defined(__HIP_DEVICE_COMPILE__)
    const size_t at = (size_t)__builtin_amdgcn_readfirstlane(phys) * page_elems;
    unsigned char* to = smem_raw + (size_t)((buf * 2 + half) * 2) * TILE * sizeof(bf16);
    // a fragment's 64 pieces of 16 bytes lie in the order of the lanes that read them (qd, j), not of their rows (j, qd): lanes that
    // follow each other then read from all banks
    const int here = from_here(lane), piece = wave * 64 + here % 16 * 4 + here / 16;
#pragma unroll
    for (int p = 0; p < NLOAD; ++p) {
      __builtin_amdgcn_global_load_lds(k0 + at + (piece + p * 256) * 8, to + (wave + p * 4) * 1024, 16, 0, 0);
      __builtin_amdgcn_global_load_lds(v0 + at + (piece + p * 256) * 8, to + TILE * sizeof(bf16) + (wave + p * 4) * 1024, 16, 0, 0);
    }
#endif
  };
  // places are looked up a round ahead of the page's way into LDS: the one trip to memory would else wait for the other
  auto place = [&](int page) { return page < pages.end ? tree_page(a, s, page) : 0; };
  int ahead = place(pages.begin + half + 2);
  if (pages.begin + half < pages.end) fetch(place(pages.begin + half), 0);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  // The walk over the pages two by two, for waves with N tiles: each number its own loops, with the registers that they need, and the
  // rounds between the first and the last ones whose pages every column sees whole in a loop of their own.
  const int rounds = (pages.end - pages.begin + 1) / 2;
  const int whole = min(rounds, max(0, ((lo_most + PAGE - 1) / PAGE - pages.begin + 1) / 2));
  const int behind = pages.end <= s.base / PAGE ? rounds : min(rounds, max(whole, (s.base / PAGE - pages.begin) / 2));
  bool odd = false;
  auto walk = [&](auto tiles_tag) {
    constexpr int N = decltype(tiles_tag)::value;
    auto go = [&](int from, int to, auto edge_tag) {
      constexpr bool EDGE = decltype(edge_tag)::value;
      for (int round = from; round < to; ++round) {
        const int first = pages.begin + 2 * round, buf = round & 1;
        if (first + half + 2 < pages.end) {
          fetch(ahead, buf ^ 1);                 // that buffer was read before the last barrier
          ahead = place(first + half + 4);
        }
        // Values at an edge of what is seen: those behind the sequence, and those that are no finite numbers, are 0 from here on (0 times
        // what they are is not always 0); the latter are read again behind the walk, for the columns that see them.
        if constexpr (EDGE) {
          bool mine_odd = false;
          const int here = from_here(threadIdx.x);
#pragma unroll 1
          for (int which = 0; which < 2; ++which) {
            if (first + which >= pages.end || !col.at_edge(s, first + which)) continue;
            bf16* vs = reinterpret_cast<bf16*>(smem_raw) + (size_t)((buf * 2 + which) * 2 + 1) * TILE;
            const int left = s.len - (first + which) * PAGE;
#pragma unroll
            for (int p = 0; p < (NLOAD + 1) / 2; ++p) {
              const int piece = here + p * 512, key = piece % 64 / 16 * 8 + piece / (4 * HD) * 32;      // eight keys of an element
              if (NLOAD % 2 != 0 && piece >= TILE / 8) continue;
              words4 v = *reinterpret_cast<const words4*>(vs + piece * 8);
              if (tidy_values(v, left - key, mine_odd)) *reinterpret_cast<words4*>(vs + piece * 8) = v;
            }
          }
          odd = __syncthreads_or(mine_odd) || odd;
        }
        if constexpr (N > 0) {
#pragma unroll 1
          for (int which = wide ? 0 : half; which <= (wide ? 1 : half) && first + which < pages.end; ++which) {
            const bf16* ks = reinterpret_cast<const bf16*>(smem_raw) + (size_t)((buf * 2 + which) * 2) * TILE;
            const bf16* vs = ks + TILE;
            col.template page<N, EDGE ? C::PART : C::WHOLE>(a, s, first + which, qd, scale,
                                                            [&](int t, int k) { return ld8(ks + (k * 4 + t) * 512 + lane * 8); },
                                                            [&](int dt, int t) { return ld8(vs + (t * DT + dt) * 512 + lane * 8); }, []() {});
          }
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");     // this wave's share of the next pages has landed
        __syncthreads();
      }
    };
    go(0, whole, std::true_type{});
    go(whole, behind, std::false_type{});
    go(behind, rounds, std::true_type{});
  };
  if (tiles == NC) walk(std::integral_constant<int, NC>{});
  else if (NC > 1 && tiles == 1) walk(std::integral_constant<int, 1>{});
  else walk(std::integral_constant<int, 0>{});
  if (odd)
    for (int ap = pages.begin + (wide ? 0 : half); ap < pages.end; ap += wide ? 1 : 2)
      if (col.at_edge(s, ap)) {
        const bf16* vp = v0 + tree_page(a, s, ap) * page_elems;
        col.add_odd(a, s, ap, qd, [&](int dt, int t) { return ld8(vp + C::value_place(dt, t, qd, j)); });
      }
  // the second group hands its maxima, sums and results to the first, which merges and writes
  f32x4* mo = reinterpret_cast<f32x4*>(smem_raw);            // [NC][DT][256]
  float* ml = reinterpret_cast<float*>(mo + NC * DT * 256);  // [NC][2][256]
  if (!wide && half == 1) {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) mo[(c * DT + dt) * 256 + tid] = col.o[c][dt];
      ml[(c * 2) * 256 + tid] = col.m[c];
      ml[(c * 2 + 1) * 256 + tid] = col.l[c];
    }
  }
  __syncthreads();
  if (!wide && half == 1) return;
  // one step for all tiles and then the next, each without branches: this code runs once, and what it waits for most is itself
  if (!wide) {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const float m2 = ml[(c * 2) * 256 + tid], l2 = ml[(c * 2 + 1) * 256 + tid], m = fmaxf(col.m[c], m2);
      const float f1 = __builtin_amdgcn_exp2f(col.m[c] - m), f2 = __builtin_amdgcn_exp2f(m2 - m);
      col.m[c] = m;
      col.l[c] = col.l[c] * f1 + l2 * f2;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) col.o[c][dt] = col.o[c][dt] * f1 + mo[(c * DT + dt) * 256 + tid] * f2;
    }
  }
  // behind what the second group left, which the other waves may still read
  unsigned char* own = smem_raw + (wide ? 0 : tree_merge_bytes<HD, NC>()) + (wide ? wave + 4 * half : wave) * tree_leave_bytes<bf16, HD>();
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const float lt = fold_column(col.l[c], [](float u, float v) { return u + v; });
    tree_leave<bf16, HD>(a, s, w, mine + c * step, cols, lane, col.m[c], lt, col.o[c], own);
  }
}

template <int HD, int NC>
int launch_lds(const TreeArgs& a, hipStream_t stream) {
  constexpr int lds = 8 * PAGE * HD * (int)sizeof(bf16);       // four pages of a head's keys and values
  static_assert(lds >= tree_merge_bytes<HD, NC>() + 4 * tree_leave_bytes<bf16, HD>() && lds >= 8 * tree_leave_bytes<bf16, HD>(), "the results' places");
  auto kernel = &attn_tree_lds_kernel<HD, NC>;
  if (lds > 60 * 1024) {
    static LdsAllowance allowed;
    if (int rc = allow_dynamic_lds(allowed, (const void*)kernel, lds); rc != YALM_OK) return rc;
  }
  const int columns = tree_columns(a.B, a.max_nodes, a.n_heads, a.n_kv_heads, HD);
  const int chunks = ((long)a.max_nodes * (a.n_heads / a.n_kv_heads) + columns - 1) / columns;
  const long units = (long)a.n_splits * a.n_kv_heads * a.B, groups = (units + 7) / 8 * 8 * chunks;
  if (groups > 0x7FFFFFFFl) return YALM_ERR_ARG;
  kernel<<<(unsigned)groups, 512, lds, stream>>>(a, chunks, columns > NC * 64);
  return launch_status();
}
template <int HD>
int launch_hd(const TreeArgs& a, hipStream_t stream) {
  const int columns = tree_columns(a.B, a.max_nodes, a.n_heads, a.n_kv_heads, HD);
  if (columns == 16) return launch_tree<bf16, HD, 1>(a, stream);
  if constexpr (HD % 32 == 0) {
    if (columns > 64) return launch_lds<HD, 2>(a, stream);
    if (columns > 32) return launch_lds<HD, 1>(a, stream);
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
