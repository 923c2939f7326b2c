// Attention of drafted tokens on the matrix cores (attention_tree.h: who sees what; attention_mfma.h: the products' layout).
//
//   scores^T[key, col] = K[key, :] . Q[col, :]      out^T[elem, col] += V^T[elem, key] P^T[key, col]
//
// A column is a (drafted token, query head of the group): the tree's rows and the heads that share a KV head go over its keys
// together.  In float32 (v_mfma_f32_16x16x4_f32) lane (qd, j) takes four consecutive elements of a row for four products, which go
// over k in the order 4 qd + c, and a page's part of the sum is formed from zero and joins the rest once.
#pragma once
#include <float.h>
#include <math.h>
#include <type_traits>
#include "attention_mfma.h"
#include "attention_tree.h"

namespace {

// A lane's number as nothing can be known of it before here: what is worked out from it for a rare branch is worked out there, and
// takes no registers from the loop around it.
__device__ __forceinline__ int from_here(int v) {
  asm volatile("" : "+v"(v));
  return v;
}

// the four lanes that share a column fold a value
template <class F>
__device__ __forceinline__ float fold_column(float v, F f) {
#if defined(__HIP_DEVICE_COMPILE__)
  typedef __attribute__((ext_vector_type(2))) unsigned both;
  both x = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = f(__uint_as_float(x[0]), __uint_as_float(x[1]));
  x = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = f(__uint_as_float(x[0]), __uint_as_float(x[1]));
#endif
  return v;
}

template <typename T>
struct TreeTypes;
template <>
struct TreeTypes<bf16> {
  typedef bf16x8 Frag;
  static constexpr int PER = 8;                    // elements a lane holds of a fragment
  static constexpr int KEYS = 2;                   // fragments of values over a page's keys
  static __device__ __forceinline__ f32x4 mma(Frag a, Frag b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <>
struct TreeTypes<float> {
  typedef f32x4 Frag;
  static constexpr int PER = 4;
  static constexpr int KEYS = 4;
  static __device__ __forceinline__ f32x4 mma(Frag a, Frag b, f32x4 c) {
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
    return c;
  }
};

// Which piece of the step's work a workgroup has.  Workgroups go to the chip's eight parts in turn: the chunks of columns of one run
// of pages follow each other on one part, whose second-level cache then serves all but the first; the splits of a sequence start
// at another one from unit to unit, for the first splits, which every sequence fills, would else stand on few parts.
struct TreeWork {
  int chunk, split, g, b;
  bool any;
  __device__ __forceinline__ TreeWork(const TreeArgs& a, int chunks) {
    const int unit = (int)(blockIdx.x / (8 * chunks)) * 8 + (int)(blockIdx.x % 8), rest = unit / a.n_splits;
    chunk = (int)(blockIdx.x / 8) % chunks;
    split = (unit + rest) % a.n_splits;
    g = rest % a.n_kv_heads;
    b = rest / a.n_kv_heads;
    any = unit < a.n_splits * a.n_kv_heads * a.B;
  }
};

// Eight values in bfloat16, of which the first `left` are the sequence's: the others and those that are no finite numbers become 0; `odd`
// where there are some of the latter.  Words of two values each, on whole registers: an exponent of ones and one more at its end reach the
// place of the sign.  True: something changed.
typedef __attribute__((ext_vector_type(4))) unsigned words4;
__device__ __forceinline__ bool tidy_values(words4& v, int left, bool& odd) {
  unsigned ends[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) ends[e] = (v[e] & 0x7F807F80u) + 0x00800080u;
  if (left >= 8 && ((ends[0] | ends[1] | ends[2] | ends[3]) & 0x80008000u) == 0) return false;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const unsigned held = 2 * e + 1 < left ? ~0u : 2 * e < left ? 0xFFFFu : 0u, at = ends[e] & held & 0x80008000u;
    odd = odd || at != 0;
    v[e] &= held & ~((at << 1) - (at >> 15));      // from a half's sign place to all of the half
  }
  return true;
}

// The columns of a wave: queries, running maxima (exponents of 2), sums and results.
template <typename T, int HD, int NC>
struct TreeColumns {
  typedef TreeTypes<T> X;
  typedef typename X::Frag Frag;
  static constexpr int PER = X::PER, KEYS = X::KEYS, STEP = 4 * PER;     // STEP: elements of a row that a product goes over
  static constexpr int KS = (HD + STEP - 1) / STEP, DT = HD / 16;
  static constexpr bool BLOCKS = HD % 32 == 0;

  Frag q[NC][KS];
  int row[NC], lo[NC];                             // a column's row of the step, and the first token that it sees
  int lo_least, lo_most;                           // over the wave's columns
  float m[NC], l[NC];
  f32x4 o[NC][DT];

  // tiles of 16 columns from x0, x0 + step, ... of `cols`
  __device__ __forceinline__ void begin(const TreeArgs& a, const TreeSeq& s, int g, int x0, int step, int cols, int lane) {
    const int qd = lane / 16, j = lane % 16, G = a.n_heads / a.n_kv_heads;
    lo_least = 0x7FFFFFFF;
    lo_most = 0;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int x = x0 + c * step + j;
      const bool live = x < cols;
      const int node = live ? a.node_of(x) : 0;
      row[c] = s.row0 + node;
      const T* qr = (const T*)a.q + ((size_t)row[c] * a.n_heads + g * G + (live ? x - node * G : 0)) * HD;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const int e = k * STEP + qd * PER;
        q[c][k] = *reinterpret_cast<const Frag*>(qr + min(e, HD - PER));
        if (!live || e >= HD) q[c][k] = (Frag){};
      }
      lo[c] = tree_first(a, s, row[c]);
      lo_least = live ? min(lo_least, lo[c]) : lo_least;
      lo_most = live ? max(lo_most, lo[c]) : lo_most;
      m[c] = -FLT_MAX;
      l[c] = 0.f;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) o[c][dt] = (f32x4){0.f, 0.f, 0.f, 0.f};
    }
#pragma unroll
    for (int x = 8; x > 0; x >>= 1) {
      lo_least = min(lo_least, __shfl_xor(lo_least, x, WAVE));
      lo_most = max(lo_most, __shfl_xor(lo_most, x, WAVE));
    }
  }

  // where lane (qd, j) finds its part of fragment (t, k) of a page's keys and of fragment (dt, t) of its values
  static __device__ __forceinline__ int key_place(int t, int k, int qd, int j) {
    return BLOCKS ? (k * STEP / 32 * PAGE + t * 16 + j) * 32 + k * STEP % 32 + qd * PER : key_row(t, j) * HD + min(k * STEP + qd * PER, HD - PER);
  }
  static __device__ __forceinline__ int value_key(int t, int qd) {       // the first key of a lane's fragment t of values
    return KEYS == 2 ? 32 * t + 8 * qd : 32 * (t >> 1) + 8 * qd + 4 * (t & 1);
  }
  static __device__ __forceinline__ int value_place(int dt, int t, int qd, int j) {
    const int half = KEYS == 2 ? t : t >> 1;
    return BLOCKS ? (half * HD + dt * 16 + j) * 32 + value_key(t, qd) - 32 * half : (dt * 16 + j) * PAGE + value_key(t, qd);
  }

  __device__ __forceinline__ bool at_edge(const TreeSeq& s, int at) const { return at * PAGE + PAGE > s.base || at * PAGE < lo_most; }

  // A page, for the first N tiles of columns.  keys(t, k) and values(dt, t) give a lane its fragments, between() stands behind the
  // last use of the keys.  EDGE: the page may be one at an edge of what the columns see (WHOLE: it is none; ANY: that is looked up here; PART:
  // it may be one, and its values come without what must not reach the sums).  True: values of an edge page are no finite numbers (of
  // a lane's); the sums went without them.
  enum Edge { WHOLE, ANY, PART };
  template <int N, Edge EDGE, class KF, class VF, class B>
  __device__ __forceinline__ bool page(const TreeArgs& a, const TreeSeq& s, int at, int qd, float scale, KF keys, VF values, B between) {
    f32x4 sc[N][4];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int c = 0; c < N; ++c) sc[c][t] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const Frag f = keys(t, k);
#pragma unroll
        for (int c = 0; c < N; ++c) sc[c][t] = X::mma(f, q[c][k], sc[c][t]);
      }
    between();
    const int p0 = at * PAGE;
    // The probabilities as the second product's operands: in bfloat16 rounded, as the values are (a weighted mean moves by 2^-8
    // of a value at most, what its own rounding may move it by).
    Frag pr[N][KEYS];
    float corr[N];
    unsigned seen[N][2];                          // an edge page's keys that the column sees: the lane's eight of each half
    auto softmax = [&](auto masked) {
#pragma unroll
      for (int c = 0; c < N; ++c) {
        float mx = -FLT_MAX;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            if constexpr (decltype(masked)::value)
              sc[c][t][r] = (seen[c][t >> 1] >> (4 * (t & 1) + r)) & 1 ? sc[c][t][r] : -INFINITY;
            mx = fmaxf(mx, sc[c][t][r]);
          }
        mx = fold_column(mx, [](float u, float v) { return fmaxf(u, v); });
        const float m_new = fmaxf(m[c], mx * scale);
        corr[c] = __builtin_amdgcn_exp2f(m[c] - m_new);
        float sum = 0.f;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float e = __builtin_amdgcn_exp2f(fmaf(sc[c][t][r], scale, -m_new));
            sum += e;
            if constexpr (KEYS == 2) pr[c][t >> 1][4 * (t & 1) + r] = static_cast<bf16>(e);
            else pr[c][t][r] = e;
          }
        l[c] = l[c] * corr[c] + sum;
        m[c] = m_new;
      }
      if constexpr (KEYS == 2) {                   // always: results in two places, one for a branch that leaves them, would cost their registers
#pragma unroll
        for (int c = 0; c < N; ++c)
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) o[c][dt] *= corr[c];
      }
    };
    auto mix = [&](auto careful, auto tidy) {
      if constexpr (KEYS == 2) {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int t = 0; t < KEYS; ++t) {
            if constexpr (decltype(careful)::value) __builtin_amdgcn_sched_barrier(0);       // a fragment at a time: registers are few
            const Frag f = tidy(values(dt, t), t);
#pragma unroll
            for (int c = 0; c < N; ++c) o[c][dt] = X::mma(f, pr[c][t], o[c][dt]);
          }
      } else {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          if constexpr (decltype(careful)::value) __builtin_amdgcn_sched_barrier(0);
          f32x4 part[N];
#pragma unroll
          for (int c = 0; c < N; ++c) part[c] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int t = 0; t < KEYS; ++t) {
            const Frag f = tidy(values(dt, t), t);
#pragma unroll
            for (int c = 0; c < N; ++c) part[c] = X::mma(f, pr[c][t], part[c]);
          }
#pragma unroll
          for (int c = 0; c < N; ++c)
#pragma unroll
            for (int r = 0; r < 4; ++r) o[c][dt][r] = fmaf(o[c][dt][r], corr[c], part[c][r]);
        }
      }
    };
    if (EDGE == WHOLE || (EDGE == ANY && !at_edge(s, at))) {
      softmax(std::false_type{});
      mix(std::false_type{}, [](Frag f, int) { return f; });
      return false;
    }
#pragma unroll
    for (int c = 0; c < N; ++c) {
      const unsigned long long all = tree_seen(a, s, from_here(row[c]), lo[c], at) >> (8 * qd);
      seen[c][0] = (unsigned)all & 0xFF;
      seen[c][1] = (unsigned)(all >> 32) & 0xFF;
    }
    softmax(std::true_type{});
    __builtin_amdgcn_sched_barrier(0);
    // Places behind the sequence may hold anything, and 0 times that is not always 0; nor is 0 times what is no finite number.
    bool odd = false;
    if constexpr (EDGE == PART) {
      mix(std::false_type{}, [](Frag f, int) { return f; });
    } else {
      mix(std::true_type{}, [&](Frag f, int t) {
        if constexpr (KEYS == 2) {
          words4 v = __builtin_bit_cast(words4, f);
          tidy_values(v, s.len - p0 - value_key(t, qd), odd);
          return __builtin_bit_cast(Frag, v);
        }
#pragma unroll
        for (int e = 0; e < PER; ++e) {
          const bool none = p0 + value_key(t, qd) + e >= s.len, finite = fabsf(to_f32((T)f[e])) <= FLT_MAX;
          odd = odd || (!finite && !none);
          if (none || !finite) f[e] = from_f32<T>(0.f);
        }
        return f;
      });
    }
    return odd;
  }

  // Values of an edge page that are no finite numbers, for the columns that see them: products of ones count them.  Behind all pages,
  // which went without them: what they add is the same in any order, and the loop over the pages keeps its registers.
  template <class AF>
  __device__ __forceinline__ void add_odd(const TreeArgs& a, const TreeSeq& s, int at, int qd, AF again) {
    const int p0 = at * PAGE;
    unsigned long long all[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) all[c] = tree_seen(a, s, row[c], lo[c], at);
#pragma unroll 1
    for (int kind = 0; kind < 3; ++kind) {         // no number, infinity, minus infinity
      const float what = kind == 0 ? NAN : kind == 1 ? INFINITY : -INFINITY;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        __builtin_amdgcn_sched_barrier(0);
        Frag ones[KEYS];
#pragma unroll
        for (int t = 0; t < KEYS; ++t) {
          const Frag f = again(dt, t);
#pragma unroll
          for (int e = 0; e < PER; ++e) {
            const float v = to_f32((T)f[e]);
            ones[t][e] = from_f32<T>((kind == 0 ? v != v : v == what) && p0 + value_key(t, qd) + e < s.len ? 1.f : 0.f);
          }
        }
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          f32x4 count = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int t = 0; t < KEYS; ++t) {
            Frag sees;
#pragma unroll
            for (int e = 0; e < PER; ++e) sees[e] = from_f32<T>((float)((unsigned)(all[c] >> (value_key(t, qd) + e)) & 1));
            count = X::mma(ones[t], sees, count);
          }
#pragma unroll
          for (int r = 0; r < 4; ++r) o[c][dt][r] += count[r] > 0.f ? what : 0.f;
        }
      }
    }
  }
};

// The pages p_begin ... p_end - 1 of a split, `first` being the first page that one of the columns sees.
struct TreePages {
  int begin, end;
  __device__ __forceinline__ TreePages(const TreeArgs& a, const TreeSeq& s, int split, int first) {
    begin = end = 0;
    if (s.len <= 0) return;
    const int last = (s.len - 1) / PAGE, total = last - first + 1;
    int per = (total + a.n_splits - 1) / a.n_splits;
    if (a.step_max_len != nullptr) {               // sequences of unequal lengths: pieces of the longest one's size, fewer of a short one
      const int most = max(table_entry(a.step_max_len), 1);
      const int pages = (most - 1) / PAGE - (a.window > 0 ? max(0, most - a.max_nodes - a.window + 1) / PAGE : 0) + 1;
      per = max(per, (pages + a.n_splits - 1) / a.n_splits);
    }
    begin = first + split * per;
    end = min(last + 1, begin + per);
  }
};

// Four consecutive elements of a column's result (or of its split's part), weighed; and its maximum and sum.
template <typename T, int HD>
__device__ __forceinline__ void tree_store(const TreeArgs& a, size_t head, int split, int e, f32x4 v, float inv) {
  if (a.n_splits == 1) {
    typedef __attribute__((ext_vector_type(4))) T out4;
    out4 r4;
#pragma unroll
    for (int r = 0; r < 4; ++r) r4[r] = from_f32<T>(v[r] * inv);
    *reinterpret_cast<out4*>((T*)a.out + head * HD + e) = r4;
  } else {
    float* to = a.partial + (head * a.n_splits + split) * (HD + 2) + e;
    *reinterpret_cast<float2*>(to) = make_float2(v[0], v[1]);
    *reinterpret_cast<float2*>(to + 2) = make_float2(v[2], v[3]);
  }
}
__device__ __forceinline__ float tree_inverse(float l) { return l > 0.f ? 1.0f / l : l == l ? 0.f : l; }       // a sum that is no number stays one

// What a wave leaves of a tile of 16 columns, the first of them x0, their sums folded.  Results that are none of a split go through LDS that is
// the wave's own (tree_leave_bytes), so that a store writes whole rows (45 prompts of 20 tokens and 25 nodes 20.6 -> 19.7 us).
template <typename T, int HD>
constexpr int tree_leave_bytes() { return 16 * (HD * (int)sizeof(T) + 16); }
template <typename T, int HD>
__device__ __forceinline__ void tree_leave(const TreeArgs& a, const TreeSeq& s, const TreeWork& w, int x0, int cols, int lane, float m, float l,
                                           const f32x4 (&o)[HD / 16], unsigned char* own) {
  const int G = a.n_heads / a.n_kv_heads, qd = lane / 16, j = lane % 16;
  auto head_of = [&](int x) {
    const int node = a.node_of(x);
    return (size_t)(s.row0 + node) * a.n_heads + w.g * G + x - node * G;
  };
  if (a.n_splits == 1) {
    typedef __attribute__((ext_vector_type(4))) T out4;
    constexpr int PER = 16 / (int)sizeof(T), PIECES = HD / PER, ROW = HD + PER;
    T* rows = reinterpret_cast<T*>(own);
    const float inv = tree_inverse(l);
#pragma unroll
    for (int dt = 0; dt < HD / 16; ++dt) {
      out4 r4;
#pragma unroll
      for (int r = 0; r < 4; ++r) r4[r] = from_f32<T>(o[dt][r] * inv);
      *reinterpret_cast<out4*>(rows + j * ROW + dt * 16 + 4 * qd) = r4;
    }
    wave_order();
#pragma unroll
    for (int i = lane; i < 16 * PIECES; i += WAVE)
      if (const int x = x0 + i / PIECES; x < cols)
        *reinterpret_cast<words4*>((T*)a.out + head_of(x) * HD + i % PIECES * PER) = *reinterpret_cast<const words4*>(rows + i / PIECES * ROW + i % PIECES * PER);
  } else {
    if (x0 + j < cols) {                           // 64 bytes of a row a store: rows of 520 bytes whole were no faster
      float* to = a.partial + (head_of(x0 + j) * a.n_splits + w.split) * (HD + 2);
#pragma unroll
      for (int dt = 0; dt < HD / 16; ++dt) {
        *reinterpret_cast<float2*>(to + dt * 16 + 4 * qd) = make_float2(o[dt][0], o[dt][1]);
        *reinterpret_cast<float2*>(to + dt * 16 + 4 * qd + 2) = make_float2(o[dt][2], o[dt][3]);
      }
      if (qd == 0) *reinterpret_cast<float2*>(to + HD) = make_float2(m, l);
    }
  }
  wave_order();                                    // the next tile takes the same place
}

// ---------------------------------------------------------------------------
// Few columns (16 NC of them a workgroup): four waves take the pages of a split in turn, straight from memory into registers - a page
// is one wave's, and its load instructions read 1 KB of consecutive bytes -, each with the keys of its next page in flight, and
// merge at the end.  With few columns a page's bytes outweigh its products: 8 sequences of 2,000 tokens and 8 nodes (32 columns) 23 us, 29 sequences of
// 1,423 and 3 nodes (16 columns) 31 at 4.2 TB/s.  In float32 a page's products bound it (a sixteenth of the rate): 8 sequences of 3,028 tokens and 6 nodes of
// 16 heads of 64 37 us.
// ---------------------------------------------------------------------------
constexpr int TREE_WAVES = 4;

template <typename T, int HD, int NC>
__global__ __launch_bounds__(TREE_WAVES * WAVE, NC == 1 && sizeof(T) == 2 ? 2 : 1) void attn_tree_mfma_kernel(TreeArgs a, int chunks) {
  typedef TreeColumns<T, HD, NC> C;
  typedef typename C::Frag Frag;
  constexpr int KEYS = C::KEYS, KS = C::KS, DT = C::DT, NW = TREE_WAVES;
  __shared__ float sm_m[NW][NC * 16];
  __shared__ float sm_l[NW][NC * 16];
  __shared__ f32x4 sm_o[NW][DT][WAVE];
  const TreeWork w(a, chunks);
  if (!w.any) return;
  const TreeSeq s(a, w.b);
  const int G = a.n_heads / a.n_kv_heads, cols = min(s.nodes, a.max_nodes) * G, x0 = w.chunk * NC * 16;
  if (x0 >= cols) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), lane = threadIdx.x % WAVE, qd = lane / 16, j = lane % 16;
  C col;
  col.begin(a, s, w.g, x0, 16, cols, lane);
  const TreePages pages(a, s, w.split, __builtin_amdgcn_readfirstlane(min(col.lo_least, s.base)) / PAGE);
  const float scale = 1.4426950408889634f / sqrtf((float)HD);          // scores in exponents of 2
  const size_t page_elems = (size_t)a.n_kv_heads * PAGE * HD;
  const T* k0 = (const T*)a.k_pages + (size_t)w.g * PAGE * HD;
  const T* v0 = (const T*)a.v_pages + (size_t)w.g * PAGE * HD;
  Frag kreg[4][KS];
  auto load_keys = [&](int phys) {
    const T* kp = k0 + phys * page_elems;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int k = 0; k < KS; ++k) kreg[t][k] = *reinterpret_cast<const Frag*>(kp + C::key_place(t, k, qd, j));
  };
  int ap = pages.begin + wave;
  int phys = ap < pages.end ? tree_page(a, s, ap) : 0;
  if (ap < pages.end) load_keys(phys);
  bool odd = false;
  auto one_page = [&](auto has_next) {
    const T* vp = v0 + phys * page_elems;
    Frag vreg[DT][KEYS];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int t = 0; t < KEYS; ++t) vreg[dt][t] = *reinterpret_cast<const Frag*>(vp + C::value_place(dt, t, qd, j));
    int physn = 0;
    if constexpr (decltype(has_next)::value) physn = tree_page(a, s, ap + NW);
    __builtin_amdgcn_sched_barrier(0);             // the values are asked for before the keys are waited for
    const bool found = col.template page<NC, C::ANY>(a, s, ap, qd, scale, [&](int t, int k) { return kreg[t][k]; }, [&](int dt, int t) { return vreg[dt][t]; },
                                                    [&]() {
      if constexpr (decltype(has_next)::value) {
        load_keys(physn);                          // they stay in flight while this page is mixed
        phys = physn;
        __builtin_amdgcn_sched_barrier(0);
      }
    });
    odd = odd || __any(found);
  };
  for (; ap + NW < pages.end; ap += NW) one_page(std::true_type{});
  if (ap < pages.end) one_page(std::false_type{});
  if (odd)
    for (ap = pages.begin + wave; ap < pages.end; ap += NW)
      if (col.at_edge(s, ap)) {
        const T* vp = v0 + tree_page(a, s, ap) * page_elems;
        col.add_odd(a, s, ap, qd, [&](int dt, int t) { return *reinterpret_cast<const Frag*>(vp + C::value_place(dt, t, qd, j)); });
      }

  // the four lanes of a column hold parts of its sum; then the waves merge, a tile of columns at a time
  float factor[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    col.l[c] = fold_column(col.l[c], [](float u, float v) { return u + v; });
    if (qd == 0) sm_m[wave][c * 16 + j] = col.m[c];
  }
  __syncthreads();
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    float all = sm_m[0][c * 16 + j];
#pragma unroll
    for (int v = 1; v < NW; ++v) all = fmaxf(all, sm_m[v][c * 16 + j]);
    factor[c] = __builtin_amdgcn_exp2f(col.m[c] - all);
    col.m[c] = all;
    if (qd == 0) sm_l[wave][c * 16 + j] = col.l[c] * factor[c];
  }
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    if (c > 0) __syncthreads();                    // the tile before has been read
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) sm_o[wave][dt][lane] = col.o[c][dt] * factor[c];
    __syncthreads();
    const int x = x0 + c * 16 + j;
    if (x >= cols) continue;
    float lt = sm_l[0][c * 16 + j];
#pragma unroll
    for (int v = 1; v < NW; ++v) lt += sm_l[v][c * 16 + j];
    const int node = a.node_of(x);
    const size_t head = (size_t)(s.row0 + node) * a.n_heads + w.g * G + x - node * G;
    const float inv = tree_inverse(lt);
    for (int dt = wave; dt < DT; dt += NW) {
      f32x4 v = sm_o[0][dt][lane];
#pragma unroll
      for (int u = 1; u < NW; ++u) v += sm_o[u][dt][lane];
      tree_store<T, HD>(a, head, w.split, dt * 16 + 4 * qd, v, inv);
    }
    if (a.n_splits > 1 && wave == 0 && qd == 0)
      *reinterpret_cast<float2*>(a.partial + (head * a.n_splits + w.split) * (HD + 2) + HD) = make_float2(col.m[c], lt);
  }
}

template <typename T, int HD, int NC>
int launch_tree(const TreeArgs& a, hipStream_t stream) {
  const int chunks = ((long)a.max_nodes * (a.n_heads / a.n_kv_heads) + NC * 16 - 1) / (NC * 16);
  const long units = (long)a.n_splits * a.n_kv_heads * a.B, groups = (units + 7) / 8 * 8 * chunks;
  if (groups > 0x7FFFFFFFl) return YALM_ERR_ARG;
  attn_tree_mfma_kernel<T, HD, NC><<<(unsigned)groups, TREE_WAVES * WAVE, 0, stream>>>(a, chunks);
  return launch_status();
}

}  // namespace
