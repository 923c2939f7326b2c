// Sampling under a temperature, top-k, top-p and min-p of each row's own, from a given uniform number a row.
//
// With w_i = exp((l_i - max) / T), in the order of falling logits and rising indices:
//   K  the first top_k tokens;  P  the shortest prefix of K whose weights reach top_p of K's;  M  those of P with w >= min_p
// and the draw is the first token of M, in the order of the indices, at which M's running sum reaches u times its total.
//
// Two tokens with neighbouring shares of the total are told apart by sums over the whole vocabulary, so weights are fixed-point
// numbers of 64 bits (2^SCALE for the greatest, formed in double precision, off by 2^-45 of it): sums of them are exact and the
// same in every order, atomics included.  Weights below 2^-SCALE of the greatest count as none.
//
// No row is sorted.  Tokens fall into BINS bins by (max - l) / T; the bin in which a filter's border lies comes from running
// sums over the bins, and only that bin's tokens are ranked against each other.
//
// A step of few rows spreads each over several workgroups, in four launches whose results pass through a workspace (a launch's
// end is what makes them visible): the maxima of 1,024 interleaved groups of a row; then a row with a rank collects the tokens that
// may have it (the k-th of the groups' maxima is no greater than the k-th of all tokens) and a row with a nucleus adds its weights
// up by bins; then the kept weights of each chunk of the row, and the tokens of the border's bin; then one workgroup a row ranks
// the collected tokens, finds the chunk in which the number falls and the token in it.  Ranks beyond MAX_RANK go the way of a nucleus: they
// become a limit on the weight.  What this does not take - more than LIST tokens to rank against each other - the last launch does as a call
// without a workspace does: one workgroup a row over the whole row, whose borders are narrowed by the bits of the logits where many share a bin.
//
// Bound by the launches and their chains of loads where rows are few, by passes over the logits where they are many.  Of 128,256 logits: one row
// with a rank of 50 15 us, 8 rows 16, with a nucleus 31, without a filter 16; 256 rows 50, 136 and 79 (131 MB a pass: 27 us at a copy's rate).
#include <float.h>
#include <math.h>
#include <type_traits>
#include "common.h"
#include "yalm_hip.h"

namespace {

typedef unsigned long long u64;

constexpr int NT = 1024, NW = NT / WAVE;         // a workgroup a row
constexpr int TILE = 4 * WAVE;                   // logits a wave takes with one load a lane
constexpr int BINS = 2048;
constexpr int ROOTS = 32;
constexpr int OCTAVES = 44;                      // the bins reach down to 2^-44 of the greatest weight
constexpr int SEG = 192;                         // tokens of the list that a wave's run of the row may hold
constexpr int BORDER = 768;                      // tokens of one bin that are ranked against each other
constexpr int MAX_RANK = 768;                    // of 1,024 groups of a row: some 1,400 tokens reach the 768th of their maxima
constexpr int GROUPS = BINS / NW;                // partial sums of the row that a wave leaves for the walk

// A value moved between the lanes of a wave in its registers; lanes that nothing reaches get 0.
template <int CTRL, int ROWS>
__device__ __forceinline__ unsigned moved(unsigned v) {
  return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ u64 moved(u64 v) {
  return (u64)moved<CTRL, ROWS>((unsigned)(v >> 32)) << 32 | moved<CTRL, ROWS>((unsigned)v);
}
// Inclusive running sums over a wave: within rows of 16 lanes 1, 2, 4 and 8 lanes on, then the last lanes of rows 0 and 2 to rows 1
// and 3, then lane 31 to rows 2 and 3.
template <typename V>
__device__ __forceinline__ V wave_scan(V v) {
  v += moved<0x111, 0xF>(v);
  v += moved<0x112, 0xF>(v);
  v += moved<0x114, 0xF>(v);
  v += moved<0x118, 0xF>(v);
  v += moved<0x142, 0xA>(v);
  v += moved<0x143, 0xC>(v);
  return v;
}
// The greatest of a wave, in its last lane.
template <int CTRL, int ROWS>
__device__ __forceinline__ float max_with(float v) {      // a lane that nothing reaches keeps its own
  const int own = (int)__float_as_uint(v);
  return fmaxf(v, __uint_as_float((unsigned)__builtin_amdgcn_update_dpp(own, own, CTRL, ROWS, 0xF, false)));
}
__device__ __forceinline__ float wave_greatest(float v) {
  v = max_with<0x111, 0xF>(v);
  v = max_with<0x112, 0xF>(v);
  v = max_with<0x114, 0xF>(v);
  v = max_with<0x118, 0xF>(v);
  v = max_with<0x142, 0xA>(v);
  return max_with<0x143, 0xC>(v);
}
__device__ __forceinline__ u64 last_lane(u64 v) {
  return (u64)(unsigned)__builtin_amdgcn_readlane((int)(v >> 32), WAVE - 1) << 32 | (unsigned)__builtin_amdgcn_readlane((int)v, WAVE - 1);
}
__device__ __forceinline__ u64 first_lane(u64 v) {       // lane 0's
  return (u64)(unsigned)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32 | (unsigned)__builtin_amdgcn_readfirstlane((int)v);
}
__device__ __forceinline__ u64 wave_sum64(u64 v) { return last_lane(wave_scan(v)); }

// order of floats as order of unsigned numbers; both zeros are one, no number (NaN) stands below all
__device__ __forceinline__ unsigned key_of(float l) {
  const unsigned b = __float_as_uint(l + 0.f);
  return l != l ? 0u : b ^ ((b >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}

struct Row {
  const float* l;
  int V;
  bool aligned;
  float m;                     // the greatest logit
  float to_bin;                // bins a unit of l
  double to_exponent;          // exponents of 2 a unit of l, in parts of ROOTS
  int scale;                   // the greatest weight is 2^scale
  const double* roots;         // fill_roots' table

  // not falling as l falls; BINS: the token weighs nothing
  __device__ __forceinline__ int bin(float v) const {
    const float t = (v == m ? 0.f : m - v) * to_bin;
    return t < (float)BINS ? (int)t : BINS;
  }
  // 2^(n / 32) from a table times the series of what is left (|z| <= ln 2 / 64: the first term left out is 2e-15); `up` whole
  // exponents more.  Of a token whose bin is below BINS.
  __device__ __forceinline__ double power(float v, int up) const {
    const double x = m < INFINITY ? ((double)v - (double)m) * to_exponent : v == m ? 0.0 : -1e6;
    const double n = rint(x), z = (x - n) * (0.69314718055994530942 / ROOTS);
    double p = fma(z, 1.0 / 120.0, 1.0 / 24.0);
    p = fma(p, z, 1.0 / 6.0);
    p = fma(p, z, 0.5);
    p = fma(p, z, 1.0);
    p = fma(p, z, 1.0);
    const int i = (int)n;
    return ldexp(roots[i & (ROOTS - 1)] * p, (i >> 5) + up);
  }
  // at most 2^44: adding 2^52 rounds to the nearest whole number
  __device__ __forceinline__ u64 weight(float v) const {
    return (u64)__double_as_longlong(power(v, scale) + 4503599627370496.0) & ((1ull << 52) - 1);
  }
};

// 2^(i / 32)
__device__ const double ROOT_TABLE[ROOTS] = {
    1.0, 1.0218971486541166, 1.0442737824274138, 1.0671404006768237,
    1.0905077326652577, 1.1143867425958924, 1.1387886347566916, 1.1637248587775775,
    1.189207115002721, 1.215247359980469, 1.241857812073484, 1.2690509571917332,
    1.2968395546510096, 1.3252366431597413, 1.3542555469368927, 1.383909881963832,
    1.4142135623730951, 1.4451808069770467, 1.4768261459394993, 1.5091644275934228,
    1.5422108254079407, 1.5759808451078865, 1.6104903319492543, 1.645755478153965,
    1.681792830507429, 1.718619298122478, 1.7562521603732995, 1.7947090750031072,
    1.8340080864093424, 1.8741676341103, 1.9152065613971474, 1.9571441241754002,
};
__device__ __forceinline__ void fill_roots(double* roots) {
  if (threadIdx.x < ROOTS) roots[threadIdx.x] = ROOT_TABLE[threadIdx.x];
}

struct Lds {
  u64 mass[BINS];              // weights by bin; then partial sums of the walk [NW][GROUPS]
  unsigned count[BINS];
  float list_l[NW * SEG];
  int list_i[NW * SEG];
  u64 border_a[BORDER];
  unsigned border_key[BORDER];
  int border_i[BORDER];
  u64 wave_a[NW];
  unsigned wave_c[NW];
  int list_n[NW];
  float red[NW];
  u64 found_above;
  int found_bin;
  unsigned found_in, found_through;
  unsigned thr_key;
  int thr_i;
  int n, best, full;
  unsigned key_lo, key_hi;
};

// The tokens of the row (list false) or of the list, f(logit, index): a wave takes a run of its own, a lane never an index in
// front of one that a lane before it takes in the same turn.
template <int U, typename F>
__device__ __forceinline__ void each(const Row& r, const Lds& s, bool list, int t0, int t1, int wave, int lane, F f) {
  if (list) {
    for (int i = lane; i < s.list_n[wave]; i += WAVE) f(s.list_l[wave * SEG + i], s.list_i[wave * SEG + i]);
    return;
  }
  for (int t = t0; t < t1; t += U) {
    float4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = min(t + u, t1 - 1) * TILE + 4 * lane;
      if (r.aligned && i + 4 <= r.V) {
        v[u] = *reinterpret_cast<const float4*>(r.l + i);
      } else {
        v[u].x = r.l[min(i, r.V - 1)];
        v[u].y = r.l[min(i + 1, r.V - 1)];
        v[u].z = r.l[min(i + 2, r.V - 1)];
        v[u].w = r.l[min(i + 3, r.V - 1)];
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (t + u >= t1) break;
      const int i = (t + u) * TILE + 4 * lane;
      if (i < r.V) f(v[u].x, i);
      if (i + 1 < r.V) f(v[u].y, i + 1);
      if (i + 2 < r.V) f(v[u].z, i + 2);
      if (i + 3 < r.V) f(v[u].w, i + 3);
    }
  }
}

struct Found {
  int bin;                     // BINS: the limit lies behind every bin
  u64 above;                   // the amount in front of the bin
  unsigned in, through;        // tokens in the bin, and up to its end
};

// The first bin at which the running amount (MASS: of weights, else of tokens) reaches limit(total).
template <bool MASS, typename F>
__device__ __forceinline__ Found find_bin(Lds& s, F limit_of) {
  const int t = threadIdx.x, wave = t / WAVE, lane = t % WAVE;
  const unsigned c0 = s.count[2 * t], c1 = s.count[2 * t + 1];
  const u64 a0 = MASS ? s.mass[2 * t] : c0, a1 = MASS ? s.mass[2 * t + 1] : c1;
  unsigned c = wave_scan(c0 + c1);
  u64 a = wave_scan(a0 + a1);
  if (lane == WAVE - 1) {
    s.wave_c[wave] = c;
    s.wave_a[wave] = a;
  }
  if (t == 0) s.found_bin = BINS;
  __syncthreads();
  u64 total = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    if (w < wave) {
      c += s.wave_c[w];
      a += s.wave_a[w];
    }
    total += s.wave_a[w];
  }
  const u64 limit = limit_of(total);
  const u64 before1 = a - a1, before0 = before1 - a0;
  if (before0 < limit && before1 >= limit) {
    s.found_bin = 2 * t;
    s.found_above = before0;
    s.found_in = c0;
    s.found_through = c - c1;
  } else if (before1 < limit && a >= limit) {
    s.found_bin = 2 * t + 1;
    s.found_above = before1;
    s.found_in = c1;
    s.found_through = c;
  }
  __syncthreads();
  return {s.found_bin, s.found_above, s.found_in, s.found_through};
}

__device__ __forceinline__ void clear_bins(Lds& s) {
  __syncthreads();
  for (int i = threadIdx.x; i < BINS; i += NT) {
    s.mass[i] = 0;
    s.count[i] = 0;
  }
  __syncthreads();
}

__device__ __forceinline__ bool kept(const Lds& s, unsigned key, int i, unsigned thr_key, int thr_i) {
  return key > thr_key || (key == thr_key && i <= thr_i);
}

struct Step {
  const float* logits;
  const float* us;
  const float* temperature;
  const int* top_k;
  const float* top_p;
  const float* min_p;
  int* out;
  float* prob;
  int V, scale;
  unsigned char* ws;           // of the rows one after the other, row_bytes each
  long row_bytes;
  int chunks;
};

// A row's settings.
struct Wish {
  float T, p, mp, u;
  int k;
  bool by_rank, by_mass;
  bool few, far;               // ranks whose tokens are collected, and ranks that lie behind more of them
  u64 least;                   // the weight of min_p
  __device__ __forceinline__ Wish(const Step& st, int row) {
    // asked for together: what is left out reads the row's number in its place
    const float t = *(st.temperature != nullptr ? st.temperature + row : st.us + row);
    const int n = *(st.top_k != nullptr ? st.top_k + row : reinterpret_cast<const int*>(st.us) + row);
    const float a = *(st.top_p != nullptr ? st.top_p + row : st.us + row), b = *(st.min_p != nullptr ? st.min_p + row : st.us + row);
    u = st.us[row];
    T = st.temperature != nullptr ? t : 1.f;
    k = st.top_k != nullptr ? n : 0;
    p = st.top_p != nullptr ? a : 1.f;
    mp = st.min_p != nullptr ? b : 0.f;
    by_rank = k > 0 && k < st.V;
    few = by_rank && k <= MAX_RANK;
    far = by_rank && k > MAX_RANK;
    by_mass = p < 1.f;
    const double f = mp > 0.f ? ceil(ldexp((double)fminf(mp, 1.f), st.scale)) : 0.0;
    least = f > 1.0 ? (u64)f : 1ull;
  }
  // the weight that the shortest prefix of `total` has to reach
  __device__ __forceinline__ u64 mass_limit(u64 total) const {
    const double x = ceil((double)p * (double)total);
    return x >= 1.0 ? (u64)x : 1ull;
  }
  __device__ __forceinline__ u64 target(u64 total) const {       // u of 0 or no number: the first; of 1 and more the last
    const double goal = ceil((double)u * (double)total);
    return goal >= 1.0 ? min((u64)goal, total) : 1ull;
  }
};

__device__ __forceinline__ Row row_of(const Step& st, int row, const double* roots) {
  Row r;
  r.roots = roots;
  r.l = st.logits + (size_t)row * st.V;
  r.V = st.V;
  r.aligned = ((uintptr_t)r.l & 15) == 0;
  r.scale = st.scale;
  return r;
}
__device__ __forceinline__ void set_scale(Row& r, float m, float T) {
  const double octaves = 1.4426950408889634074 / (double)T;
  r.m = m;
  r.to_exponent = octaves * ROOTS;
  r.to_bin = (float)fmin(octaves * ((double)BINS / OCTAVES), 1e30);
}
__device__ __forceinline__ void write_token(const Step& st, int row, int token, float prob) {
  st.out[row] = token;
  if (st.prob != nullptr) st.prob[row] = prob;
}

// A whole row by one workgroup.
__device__ __forceinline__ void row_alone(Lds& s, const double* roots, const Step& st, int row, const Wish& want) {
  const int tid = threadIdx.x, wave = tid / WAVE, lane = tid % WAVE;
  const int V = st.V, k = want.k;
  Row r = row_of(st, row, roots);
  const int n_tiles = (V + TILE - 1) / TILE, tpw = (n_tiles + NW - 1) / NW;
  const int t0 = min(n_tiles, wave * tpw), t1 = min(n_tiles, t0 + tpw);     // the tiles of this wave
  bool list = false;

  float mx = -INFINITY;                          // fmaxf passes over what is no number
  each<8>(r, s, false, t0, t1, wave, lane, [&](float l, int) { mx = fmaxf(mx, l); });
  r.m = block_max<NW>(mx, s.red);
  if (tid == 0) {
    s.best = V;
    s.full = 0;
    s.thr_key = 0;
    s.thr_i = 0x7FFFFFFF;
  }
  __syncthreads();
  if (!(r.m > -INFINITY)) {                      // nothing to draw from
    if (tid == 0) write_token(st, row, -1, 0.f);
    return;
  }
  if (!(want.T > 0.f)) {                              // the first of the greatest
    int first = V;
    each<4>(r, s, false, t0, t1, wave, lane, [&](float l, int i) { first = l == r.m ? min(first, i) : first; });
    if (first < V) atomicMin(&s.best, first);
    __syncthreads();
    if (tid == 0) write_token(st, row, s.best, 1.f);
    return;
  }
  set_scale(r, r.m, want.T);

  unsigned thr_key = 0;                          // a token is kept if it stands in front of (thr_key, thr_i) or there
  int thr_i = 0x7FFFFFFF;
  auto fill = [&](bool mass) {                   // the bins of the kept tokens
    clear_bins(s);
    each<4>(r, s, list, t0, t1, wave, lane, [&](float l, int i) {
      const int b = r.bin(l);
      if (b < BINS && kept(s, key_of(l), i, thr_key, thr_i)) {
        atomicAdd(&s.count[b], 1u);
        if (mass) atomicAdd(&s.mass[b], r.weight(l));
      }
    });
    __syncthreads();
  };
  // the tokens of the bins up to `last` into the list, in the order of their indices, if a wave's part holds its own
  auto collect = [&](int last) {
    int n = 0;
    for (int t = t0; t < t1; ++t) {
      const int i = t * TILE + 4 * lane;
      float v[4];
      u64 takes[4];
      bool mine[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = r.l[min(i + j, V - 1)];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        mine[j] = i + j < V && r.bin(v[j]) <= last;
        takes[j] = __ballot(mine[j]);
      }
      const int more = __popcll(takes[0]) + __popcll(takes[1]) + __popcll(takes[2]) + __popcll(takes[3]);
      if (more == 0) continue;
      if (n + more > SEG) {
        n = SEG + 1;
        break;
      }
      const u64 lower = (1ull << lane) - 1;
      int at = wave * SEG + n + __popcll(takes[0] & lower) + __popcll(takes[1] & lower) + __popcll(takes[2] & lower) + __popcll(takes[3] & lower);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (mine[j]) {
          s.list_l[at] = v[j];
          s.list_i[at] = i + j;
          ++at;
        }
      n += more;
    }
    if (lane == 0) {
      s.list_n[wave] = n;
      if (n > SEG) s.full = 1;
    }
    __syncthreads();
    list = s.full == 0;
  };
  // The last kept token of bin b in front of which less than `limit` stands (MASS: weights, else tokens), `above` of it in front of
  // the bin: the new threshold.
  auto narrow = [&](auto mass_tag, const Found& f, u64 limit) {
    constexpr bool MASS = decltype(mass_tag)::value;
    if (f.in <= (unsigned)BORDER) {
      if (tid == 0) {
        s.n = 0;
        s.best = -1;
      }
      __syncthreads();
      each<4>(r, s, list, t0, t1, wave, lane, [&](float l, int i) {
        const unsigned key = key_of(l);
        if (r.bin(l) == f.bin && kept(s, key, i, thr_key, thr_i)) {
          const int at = atomicAdd(&s.n, 1);
          if (at < BORDER) {
            s.border_key[at] = key;
            s.border_i[at] = i;
            s.border_a[at] = MASS ? r.weight(l) : 1ull;
          }
        }
      });
      __syncthreads();
      const int n = min(s.n, BORDER);
      int share = WAVE;                          // lanes a token
      while (share > 1 && n * share > NT) share >>= 1;
      const int e = tid / share, part = tid % share;
      u64 before = f.above;
      int rank = 0;
      const unsigned key = e < n ? s.border_key[e] : 0;
      const int index = e < n ? s.border_i[e] : 0;
      u64 mine = 0;
      for (int j = part; j < n; j += share) {
        const unsigned kj = s.border_key[j];
        if (kj > key || (kj == key && s.border_i[j] < index)) {
          mine += s.border_a[j];
          ++rank;
        }
      }
      for (int o = share / 2; o > 0; o >>= 1) {
        mine += __shfl_xor(mine, o, WAVE);
        rank += __shfl_xor(rank, o, WAVE);
      }
      before += mine;
      const bool in = e < n && part == 0 && before < limit;
      if (in) atomicMax(&s.best, rank);
      __syncthreads();
      if (in && rank == s.best) {
        s.thr_key = key;
        s.thr_i = index;
      }
      __syncthreads();
      thr_key = s.thr_key;
      thr_i = s.thr_i;
      return;
    }
    // Many tokens in one bin: between the least and the greatest of their keys, a part of 2,048 at a time, down to one key.
    if (tid == 0) {
      s.key_lo = 0xFFFFFFFFu;
      s.key_hi = 0;
    }
    __syncthreads();
    unsigned lo = 0xFFFFFFFFu, hi = 0;
    each<4>(r, s, list, t0, t1, wave, lane, [&](float l, int i) {
      const unsigned key = key_of(l);
      if (r.bin(l) == f.bin && kept(s, key, i, thr_key, thr_i)) {
        lo = min(lo, key);
        hi = max(hi, key);
      }
    });
    atomicMin(&s.key_lo, lo);
    atomicMax(&s.key_hi, hi);
    __syncthreads();
    lo = s.key_lo;
    hi = s.key_hi;
    u64 above = f.above;
    unsigned ties = f.in;
    while (lo < hi) {
      int shift = 0;
      while (((hi - lo) >> shift) >= (unsigned)BINS) ++shift;
      clear_bins(s);
      each<4>(r, s, list, t0, t1, wave, lane, [&](float l, int i) {
        const unsigned key = key_of(l);
        if (key >= lo && key <= hi && r.bin(l) < BINS && kept(s, key, i, thr_key, thr_i)) {
          const unsigned b = (hi - key) >> shift;
          atomicAdd(&s.count[b], 1u);
          if (MASS) atomicAdd(&s.mass[b], r.weight(l));
        }
      });
      __syncthreads();
      const u64 front = above;
      const Found g = find_bin<MASS>(s, [&](u64) { return limit - front; });
      if (g.bin == BINS) break;                  // the bin's own total reached the limit: not met
      above += g.above;
      ties = g.in;
      hi -= (unsigned)g.bin << shift;
      const unsigned width = (1u << shift) - 1;
      lo = hi - lo > width ? hi - width : lo;
      __syncthreads();
    }
    // `ties` tokens with the logit of key hi: the first `take` of them
    u64 take = ties;
    {
      const float l = __uint_as_float((hi >> 31) ? hi ^ 0x80000000u : ~hi);
      const u64 each_a = MASS ? r.weight(l) : 1ull;
      if (each_a > 0) take = min(take, (limit - above + each_a - 1) / each_a);
      if (take < 1) take = 1;
    }
    int mine = 0;                                // this wave's ties
    each<4>(r, s, list, t0, t1, wave, lane, [&](float l, int i) {
      const unsigned key = key_of(l);
      mine += key == hi && kept(s, key, i, thr_key, thr_i);
    });
#pragma unroll
    for (int o = WAVE / 2; o > 0; o >>= 1) mine += __shfl_xor(mine, o, WAVE);
    if (lane == 0) s.wave_a[wave] = (u64)mine;
    if (tid == 0) {
      s.thr_key = hi;
      s.thr_i = V;
    }
    __syncthreads();
    u64 front = 0;
    for (int w = 0; w < wave; ++w) front += s.wave_a[w];
    if (front < take && take <= front + (u64)mine) {          // the last one lies in this wave's run
      const int n = list ? s.list_n[wave] : (t1 - t0) * TILE;
      for (int x = 0; x < n; x += WAVE) {
        const int e = x + lane;
        const int i = list ? (e < n ? s.list_i[wave * SEG + e] : V) : t0 * TILE + e;
        const float l = e < n && i < V ? r.l[i] : 0.f;
        const unsigned key = key_of(l);
        u64 hit = __ballot(e < n && i < V && key == hi && kept(s, key, i, thr_key, thr_i));
        const u64 c = (u64)__popcll(hit);
        if (front + c >= take) {
          for (u64 q = take - front; q > 1; --q) hit &= hit - 1;
          const int at = __ffsll((long long)hit) - 1;
          if (lane == at) s.thr_i = i;
          break;
        }
        front += c;
      }
    }
    __syncthreads();
    thr_key = s.thr_key;
    thr_i = s.thr_i;
  };
  if (want.by_rank) {
    fill(false);
    const Found f = find_bin<false>(s, [&](u64) { return (u64)k; });
    if (f.bin < BINS) {
      if (f.through <= (unsigned)(NW * SEG)) collect(f.bin);
      narrow(std::false_type{}, f, (u64)k);
    }
  }
  if (want.by_mass) {
    fill(true);
    u64 limit = 1;
    const Found f = find_bin<true>(s, [&](u64 total) { return limit = want.mass_limit(total); });
    if (f.bin < BINS) {
      if (!list && f.through <= (unsigned)(NW * SEG)) collect(f.bin);
      narrow(std::true_type{}, f, limit);
    }
  }

  // the walk: partial sums, the part in which the target falls, the token in it
  auto amount = [&](float l, int i) -> u64 {
    if (r.bin(l) >= BINS || !kept(s, key_of(l), i, thr_key, thr_i)) return 0;
    const u64 w = r.weight(l);
    return w >= want.least ? w : 0;
  };
  const int n_mine = list ? s.list_n[wave] : max(0, min(V, t1 * TILE) - t0 * TILE);
  const int turns = list ? (n_mine + WAVE - 1) / WAVE : t1 - t0;              // a load a lane each
  const int turns_a_group = list ? 1 : max(4, (tpw + GROUPS - 1) / GROUPS);
  __syncthreads();
  u64 sum = 0;                                   // of this wave
  for (int turn = 0; turn < turns; turn += turns_a_group) {
    u64 part = 0;
    if (list) {
      const int e = turn * WAVE + lane;
      if (e < n_mine) part = amount(s.list_l[wave * SEG + e], s.list_i[wave * SEG + e]);
    } else {
      each<4>(r, s, false, t0 + turn, min(t1, t0 + turn + turns_a_group), wave, lane, [&](float l, int i) { part += amount(l, i); });
    }
    part = wave_sum64(part);
    if (lane == 0) s.mass[wave * GROUPS + turn / turns_a_group] = part;
    sum += part;
  }
  if (lane == 0) s.wave_a[wave] = sum;
  __syncthreads();
  u64 total = 0, front = 0;
  for (int w = 0; w < NW; ++w) {
    if (w < wave) front += s.wave_a[w];
    total += s.wave_a[w];
  }
  const u64 target = want.target(total);
  if (!(front < target && target <= front + sum)) return;
  for (int g = 0; g * turns_a_group < turns; ++g) {
    const u64 a = s.mass[wave * GROUPS + g];
    if (front + a < target) {
      front += a;
      continue;
    }
    for (int turn = g * turns_a_group; turn < turns; ++turn) {
      float l[4] = {0.f, 0.f, 0.f, 0.f};
      int i[4] = {V, V, V, V};
      u64 a4[4] = {0, 0, 0, 0};
      if (list) {
        const int e = turn * WAVE + lane;
        if (e < n_mine) {
          l[0] = s.list_l[wave * SEG + e];
          i[0] = s.list_i[wave * SEG + e];
          a4[0] = amount(l[0], i[0]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          i[j] = (t0 + turn) * TILE + 4 * lane + j;
          l[j] = r.l[min(i[j], V - 1)];
          a4[j] = i[j] < V ? amount(l[j], i[j]) : 0;
        }
      }
      const u64 mine = (a4[0] + a4[1]) + (a4[2] + a4[3]);
      const u64 incl = wave_scan(mine);
      const u64 reached = __ballot(front + incl >= target);
      if (reached == 0) {
        front += last_lane(incl);
        continue;
      }
      if (lane == __ffsll((long long)reached) - 1) {
        u64 c = front + (incl - mine);
        int j = 0;
        while (j < 3 && c + a4[j] < target) c += a4[j++];
        const float at_l = j == 0 ? l[0] : j == 1 ? l[1] : j == 2 ? l[2] : l[3];
        write_token(st, row, j == 0 ? i[0] : j == 1 ? i[1] : j == 2 ? i[2] : i[3], (float)(r.power(at_l, 0) / ldexp((double)total, -st.scale)));
      }
      return;
    }
  }
}

__global__ __launch_bounds__(NT) void sample_alone_kernel(Step st) {
  __shared__ Lds s;
  __shared__ double roots[ROOTS];
  fill_roots(roots);
  const Wish want(st, blockIdx.x);
  row_alone(s, roots, st, blockIdx.x, want);
}

// ---------------------------------------------------------------------------
// rows over several workgroups
// ---------------------------------------------------------------------------
constexpr int CHUNK = 4 * NT;                    // logits that a workgroup takes with one load a thread
constexpr int MAX_GROUPS_ROW = 64;               // workgroups a row: a power of two
constexpr int LIST = 2048;                       // collected tokens that the last launch ranks
constexpr int CHUNKS_EACH = 64;                  // chunks that a workgroup takes at most
constexpr int MAX_CHUNKS = BINS;

// What the launches leave for each other of a row.
struct Left {
  float* top;                  // [NT] maxima of the groups
  float* peak;                 // [chunks][NW] maxima of a chunk's parts, a wave's logits each
  u64* mass;                   // [BINS]
  u64* list;                   // [LIST] ~key << 32 | index: rising numbers are the tokens' order
  u64* sums;                   // [chunks] kept weights
  unsigned* counts;            // [BINS] tokens
  int* count;                  // collected tokens
  int* first;                  // the first of the greatest
  __device__ __forceinline__ Left(const Step& st, int row) {
    unsigned char* at = st.ws + (size_t)row * st.row_bytes;
    mass = reinterpret_cast<u64*>(at);
    list = mass + BINS;
    sums = list + LIST;
    counts = reinterpret_cast<unsigned*>(sums + st.chunks);
    top = reinterpret_cast<float*>(counts + BINS);
    peak = top + NT;
    count = reinterpret_cast<int*>(peak + (size_t)st.chunks * NW);
    first = count + 1;
  }
};
inline long left_bytes(int chunks) { return ((BINS + LIST + chunks) * 8l + (BINS + NT + (long)chunks * NW) * 4l + 8 + 15) / 16 * 16; }

// the thread's four logits of a chunk; behind the row's end no number
__device__ __forceinline__ float4 chunk4(const Row& r, int chunk) {
  const int i = chunk * CHUNK + 4 * (int)threadIdx.x;
  if (r.aligned && i + 4 <= r.V) return *reinterpret_cast<const float4*>(r.l + i);
  float4 v;
  v.x = i < r.V ? r.l[i] : NAN;
  v.y = i + 1 < r.V ? r.l[i + 1] : NAN;
  v.z = i + 2 < r.V ? r.l[i + 2] : NAN;
  v.w = i + 3 < r.V ? r.l[i + 3] : NAN;
  return v;
}
// f(chunk, its four logits) for the workgroup's chunks, U of them asked for at a time
template <int U, typename F>
__device__ __forceinline__ void chunks_of(const Row& r, int chunks, F f) {
  for (int c = blockIdx.x; c < chunks; c += U * gridDim.x) {
    float4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = chunk4(r, min(c + u * (int)gridDim.x, chunks - 1));
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (c + u * (int)gridDim.x < chunks) f(c + u * (int)gridDim.x, v[u]);
  }
}

// The same for the parts of chunks of which the caller's wave wants to see the logits, by their maximum: the others are not read.  For
// what is found in few parts: 256 rows of 128,256 logits, greedy 48 -> 35 us, ranks of 50 58 -> 49; where every part is wanted (a nucleus, no
// filter) looking first costs 4 of 75 us, and chunks_of serves.
template <int U, typename W, typename F>
__device__ __forceinline__ void parts_of(const Row& r, const Left& left, int chunks, W wants, F f) {
  const int lane = threadIdx.x % WAVE, wave = threadIdx.x / WAVE, step = gridDim.x;
  static_assert(CHUNKS_EACH <= WAVE, "a lane looks at a chunk");
  const int c = blockIdx.x + lane * step;
  u64 todo = __ballot(c < chunks && wants(left.peak[min(c, chunks - 1) * NW + wave]));
  while (todo != 0) {
    float4 v[U];
    int at[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      at[u] = -1;
      if (todo != 0) {
        at[u] = blockIdx.x + (__ffsll((long long)todo) - 1) * step;
        todo &= todo - 1;
        v[u] = chunk4(r, at[u]);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (at[u] >= 0) f(at[u], v[u]);
  }
}

// The maxima, and the workspace's start.  256 rows of 128,256: 31 us, 4.3 TB/s.
__global__ __launch_bounds__(NT) void sample_top_kernel(Step st) {
  const int row = blockIdx.y, n = gridDim.x, wave = threadIdx.x / WAVE, lane = threadIdx.x % WAVE;
  const Row r = row_of(st, row, nullptr);
  const Left left(st, row);
  float mx = -INFINITY;
  chunks_of<8>(r, st.chunks, [&](int chunk, float4 v) {
    const float here = fmaxf(fmaxf(fmaxf(-INFINITY, v.x), fmaxf(v.y, v.z)), v.w);
    mx = fmaxf(mx, here);
    const float peak = wave_greatest(here);
    if (lane == WAVE - 1) left.peak[chunk * NW + wave] = peak;
  });
  for (int o = 1; o < n; o <<= 1) mx = fmaxf(mx, __shfl_xor(mx, o, WAVE));
  if (threadIdx.x % n == 0) left.top[blockIdx.x * (NT / n) + threadIdx.x / n] = mx;
  for (int i = blockIdx.x * NT + threadIdx.x; i < BINS; i += n * NT) {
    left.mass[i] = 0;
    left.counts[i] = 0;
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    *left.count = 0;
    *left.first = 0x7FFFFFFF;
  }
}

// the threads of a wave that have something take places of the list
__device__ __forceinline__ void append(const Left& left, bool has, u64 what) {
  const u64 who = __ballot(has);
  if (who == 0) return;
  const int lane = threadIdx.x % WAVE, leader = __ffsll((long long)who) - 1;
  int at = 0;
  if (lane == leader) at = atomicAdd(left.count, __popcll(who));
  at = __shfl(at, leader, WAVE) + __popcll(who & ((1ull << lane) - 1));
  if (has && at < LIST) left.list[at] = what;
}
__device__ __forceinline__ u64 order_of(float l, int i) { return ((u64)~key_of(l) << 32) | (unsigned)i; }
__device__ __forceinline__ float logit_of(u64 order) {
  const unsigned key = ~(unsigned)(order >> 32);
  return __uint_as_float((key >> 31) ? key ^ 0x80000000u : ~key);
}

// Rows with a rank: the tokens up to the bin of the k-th of the groups' maxima.  Rows with a nucleus or a far rank: weights by bins, and for
// the rank the tokens by bins.  Rows with a rank read few parts (256 rows of 128,256 and a rank of 50: 9 us); by bins it is the additions in LDS, 64 bits each
// to places that collide, that take longest (256 rows: some 55 us, where the next pass with as many weights takes 35).
__global__ __launch_bounds__(NT, 8) void sample_sift_kernel(Step st) {
  __shared__ double roots[ROOTS];
  __shared__ u64 mass[BINS];
  __shared__ unsigned counts[BINS];
  __shared__ float red[NW];
  __shared__ unsigned waves[NW];
  __shared__ int border;
  const int row = blockIdx.y, tid = threadIdx.x, wave = tid / WAVE, lane = tid % WAVE;
  const Wish want(st, row);
  if (!(want.T > 0.f) || !(want.by_rank || want.by_mass)) return;
  fill_roots(roots);
  Row r = row_of(st, row, roots);
  const Left left(st, row);
  const float mine = left.top[tid];
  const float m = block_max<NW>(mine, red);
  if (!(m > -INFINITY)) return;
  set_scale(r, m, want.T);
  if (want.few) {
    counts[tid] = counts[tid + NT] = 0;
    if (tid == 0) border = BINS - 1;
    __syncthreads();
    const int b = r.bin(mine);
    if (b < BINS) atomicAdd(&counts[b], 1u);
    __syncthreads();
    const unsigned c0 = counts[2 * tid], c1 = counts[2 * tid + 1];
    unsigned c = wave_scan(c0 + c1);
    if (lane == WAVE - 1) waves[wave] = c;
    __syncthreads();
    for (int w = 0; w < wave; ++w) c += waves[w];
    const unsigned k = (unsigned)want.k;
    if (c >= k && c - c1 < k) border = 2 * tid + 1;
    if (c - c1 >= k && c - c1 - c0 < k) border = 2 * tid;
    __syncthreads();
    const int last = border;
    parts_of<4>(r, left, st.chunks, [&](float peak) { return r.bin(peak) <= last; }, [&](int chunk, float4 v) {
      const float l[4] = {v.x, v.y, v.z, v.w};
      bool in[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) in[j] = r.bin(l[j]) <= last;
      if (!__any(in[0] || in[1] || in[2] || in[3])) return;
#pragma unroll
      for (int j = 0; j < 4; ++j) append(left, in[j], order_of(l[j], chunk * CHUNK + 4 * tid + j));
    });
    return;
  }
  mass[tid] = mass[tid + NT] = 0;
  counts[tid] = counts[tid + NT] = 0;
  __syncthreads();
  chunks_of<4>(r, st.chunks, [&](int, float4 v) {
    const float l[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int b = r.bin(l[j]);
      if (b < BINS) {
        atomicAdd(&mass[b], r.weight(l[j]));
        if (want.far) atomicAdd(&counts[b], 1u);
      }
    }
  });
  __syncthreads();
  for (int i = tid; i < BINS; i += NT) {
    if (mass[i] != 0) atomicAdd(&left.mass[i], mass[i]);
    if (counts[i] != 0) atomicAdd(&left.counts[i], counts[i]);
  }
}

// The bin in which the running mass reaches the limit, the mass in front of it, and the limit.
constexpr int FOUND = 7;
struct Border {
  int bin;
  u64 above, limit;
};
__device__ __forceinline__ Border find_border(const Left& left, const Wish& want, u64* waves, u64* found) {
  const int tid = threadIdx.x, wave = tid / WAVE, lane = tid % WAVE;
  const ulonglong2 a = reinterpret_cast<const ulonglong2*>(left.mass)[tid];
  u64 c = wave_scan((u64)(a.x + a.y));
  if (lane == WAVE - 1) waves[wave] = c;
  if (tid == 0) found[0] = BINS;
  __syncthreads();
  u64 total = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    if (w < wave) c += waves[w];
    total += waves[w];
  }
  const u64 limit = want.mass_limit(total), before1 = c - a.y, before0 = before1 - a.x;
  if (before0 < limit && before1 >= limit) {
    found[0] = 2 * tid;
    found[1] = before0;
  } else if (before1 < limit && c >= limit) {
    found[0] = 2 * tid + 1;
    found[1] = before1;
  }
  __syncthreads();
  return {(int)found[0], found[1], limit};
}

// A far rank.  Its border's bin comes from the tokens by bins; the weight of the first k lies between that of the bins in front of it and that
// of those with it, and so does what top_p leaves of it: the bins from `lo` to `hi` can hold the end of the prefix, and all in front is kept.
// Without a nucleus that is the rank's bin.  A rank of 2,000 of 128,256: 29 us for a row, 33 for 8, 70 for 64 (one workgroup a row 101, 102 and
// 113); of 20,000 with 0.9 of the weight 42, 49 and 90 (242, 246, 257).
struct Far {
  int rank, lo, hi;
  int need;                    // tokens of the rank's bin that belong to the first k
  u64 above_rank, above_lo;    // the mass in front
};
__device__ __forceinline__ Far far_borders(const Left& left, const Wish& want, u64* waves, u64* found) {
  const int tid = threadIdx.x, wave = tid / WAVE, lane = tid % WAVE;
  const uint2 n = reinterpret_cast<const uint2*>(left.counts)[tid];
  const ulonglong2 a = reinterpret_cast<const ulonglong2*>(left.mass)[tid];
  u64 c = wave_scan((u64)(n.x + n.y));
  if (lane == WAVE - 1) waves[wave] = c;
  if (tid == 0) {
    found[0] = BINS;
    found[1] = 0;
  }
  __syncthreads();
  for (int w = 0; w < wave; ++w) c += waves[w];
  const u64 k = (u64)want.k, c1 = c - n.y, c0 = c1 - n.x;
  if (c0 < k && c >= k) {
    const bool second = c1 < k;
    found[0] = 2 * tid + (second ? 1 : 0);
    found[1] = k - (second ? c1 : c0);
  }
  __syncthreads();
  Far f;
  f.rank = (int)found[0];
  f.need = (int)found[1];
  u64 m = wave_scan((u64)(a.x + a.y));
  if (lane == WAVE - 1) waves[wave] = m;
  __syncthreads();
  u64 total = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    if (w < wave) m += waves[w];
    total += waves[w];
  }
  const u64 m1 = m - a.y, m0 = m1 - a.x;
  if (f.rank < BINS ? f.rank / 2 == tid : tid == 0) {
    found[2] = f.rank == BINS ? total : (f.rank & 1) ? m1 : m0;
    found[3] = f.rank == BINS ? total : (f.rank & 1) ? m : m1;
  }
  __syncthreads();
  f.above_rank = f.above_lo = found[2];
  f.lo = f.hi = f.rank;
  if (!want.by_mass) return f;
  const u64 least = want.mass_limit(f.above_rank), most = want.mass_limit(found[3]);
  if (m0 < least && m >= least) {
    found[4] = 2 * tid + (m1 < least ? 1 : 0);
    found[5] = m1 < least ? m1 : m0;
  }
  if (m0 < most && m >= most) found[6] = 2 * tid + (m1 < most ? 1 : 0);
  __syncthreads();
  f.lo = (int)found[4];
  f.above_lo = found[5];
  f.hi = (int)found[6];
  return f;
}

// Rows but for those with a collected rank: the kept weights of each chunk (in front of the border's bin), and the tokens of the bins in which
// a border may lie.  256 rows without a filter: 35 us, the logits' way and a weight's double precision.
__global__ __launch_bounds__(NT, 8) void sample_sum_kernel(Step st) {
  __shared__ double roots[ROOTS];
  __shared__ float red[NW];
  __shared__ u64 waves[NW], found[FOUND];
  __shared__ u64 parts[CHUNKS_EACH][NW];
  const int row = blockIdx.y, tid = threadIdx.x, wave = tid / WAVE, lane = tid % WAVE;
  const Wish want(st, row);
  if (want.T > 0.f && want.few) return;
  fill_roots(roots);
  Row r = row_of(st, row, roots);
  const Left left(st, row);
  const float m = block_max<NW>(left.top[tid], red);
  if (!(m > -INFINITY)) return;
  if (!(want.T > 0.f)) {
    int first = 0x7FFFFFFF;
    parts_of<4>(r, left, st.chunks, [&](float peak) { return peak == m; }, [&](int chunk, float4 v) {
      const int i = chunk * CHUNK + 4 * tid;
      first = min(first, v.x == m ? i : v.y == m ? i + 1 : v.z == m ? i + 2 : v.w == m ? i + 3 : 0x7FFFFFFF);
    });
    if (first < 0x7FFFFFFF) atomicMin(left.first, first);
    return;
  }
  set_scale(r, m, want.T);
  int bin = BINS, hi = BINS, rank = -1;
  if (want.far) {
    const Far f = far_borders(left, want, waves, found);
    bin = f.lo;
    hi = f.hi;
    if (f.rank < BINS) rank = f.rank;
  } else if (want.by_mass) {
    bin = hi = find_border(left, want, waves, found).bin;
  }
  auto border = [&](int b) { return (unsigned)(b - bin) <= (unsigned)(hi - bin) || b == rank; };       // with bin < BINS
  chunks_of<4>(r, st.chunks, [&](int chunk, float4 v) {
    const float l[4] = {v.x, v.y, v.z, v.w};
    int b[4];
    u64 sum = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      b[j] = r.bin(l[j]);
      if (b[j] < bin) {
        const u64 w = r.weight(l[j]);
        sum += w >= want.least ? w : 0;
      }
    }
    if (bin < BINS && __any(border(b[0]) || border(b[1]) || border(b[2]) || border(b[3]))) {
#pragma unroll
      for (int j = 0; j < 4; ++j) append(left, border(b[j]), order_of(l[j], chunk * CHUNK + 4 * tid + j));
    }
    sum = wave_sum64(sum);
    if (lane == 0) parts[chunk / (int)gridDim.x][wave] = sum;
  });
  __syncthreads();
  for (int c = tid; c * (int)gridDim.x + (int)blockIdx.x < st.chunks; c += NT) {
    u64 all = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) all += parts[c][w];
    left.sums[c * gridDim.x + blockIdx.x] = all;
  }
}

constexpr int FINE = 256;                        // parts of the border's bin
struct Last {                                    // LDS of the last launch beside row_alone's
  u64 a[LIST], b[LIST];
  u64 sums[MAX_CHUNKS];
  u64 fine[FINE];
  u64 waves[NW], found[FOUND], last;
  float red[NW];
  int best, n;
};

// x[0 ... n - 1] into rising order (n <= LIST); y holds as many.  Few are ranked by counting, more sorted by exchanges.
__device__ __forceinline__ void sort_rising(u64* x, u64* y, int n) {
  const int tid = threadIdx.x;
  if (n <= 512) {
    int share = WAVE;                            // lanes a number
    while (share > 1 && n * share > NT) share >>= 1;
    const int e = tid / share;
    const u64 mine = e < n ? x[e] : 0;
    int rank = 0;
    for (int j = tid % share; j < n; j += share) rank += x[j] < mine;
    for (int o = share / 2; o > 0; o >>= 1) rank += __shfl_xor(rank, o, WAVE);
    __syncthreads();
    if (e < n && tid % share == 0) y[rank] = mine;
    __syncthreads();
    for (int i = tid; i < n; i += NT) x[i] = y[i];
    __syncthreads();
    return;
  }
  int size = 1024;
  while (size < n) size <<= 1;
  for (int i = n + tid; i < size; i += NT) x[i] = ~0ull;
  __syncthreads();
  for (int run = 2; run <= size; run <<= 1)
    for (int step = run >> 1; step > 0; step >>= 1) {
      for (int i = tid; i < size / 2; i += NT) {
        const int lo = 2 * i - (i & (step - 1)), hi = lo + step;
        const u64 p = x[lo], q = x[hi];
        if ((p > q) == ((lo & run) == 0)) {
          x[lo] = q;
          x[hi] = p;
        }
      }
      __syncthreads();
    }
}

// Inclusive running sums of f(i), i < n <= LIST, in out; the total.
template <typename F>
__device__ __forceinline__ u64 running_sums(u64* out, int n, u64* waves, F f) {
  const int tid = threadIdx.x, wave = tid / WAVE, lane = tid % WAVE;
  const u64 a0 = 2 * tid < n ? f(2 * tid) : 0, a1 = 2 * tid + 1 < n ? f(2 * tid + 1) : 0;
  u64 c = wave_scan(a0 + a1);
  __syncthreads();
  if (lane == WAVE - 1) waves[wave] = c;
  __syncthreads();
  u64 total = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    if (w < wave) c += waves[w];
    total += waves[w];
  }
  if (2 * tid < n) out[2 * tid] = c - a1;
  if (2 * tid + 1 < n) out[2 * tid + 1] = c;
  __syncthreads();
  return total;
}

// A row with a rank whose candidates are few: one wave has one a lane, in the order of the ranks and then in that of the indices.
// `x` holds 2 WAVE numbers.
__device__ __forceinline__ void last_of_few(const Step& st, int row, const Wish& want, Row r, u64* x, u64 order, int n) {
  const int lane = threadIdx.x;
  u64* y = x + WAVE;
  x[lane] = lane < n ? order : ~0ull;
  wave_order();
  int rank = 0;
#pragma unroll 8
  for (int j = 0; j < (n + 7) / 8 * 8; ++j) rank += x[j] < order;
  if (lane < n) y[rank] = order;
  wave_order();
  order = y[lane];                               // the token of this rank (lanes from n on: anything)
  const float l = logit_of(order);
  set_scale(r, logit_of(first_lane(order)), want.T);
  const bool in_k = lane < min(n, want.k);
  const u64 w = in_k ? r.weight(l) : 0, c = wave_scan(w);
  const u64 limit = want.mass_limit(last_lane(c));         // with every lane at work: a lane that is left out has no sum to read
  const bool in = in_k && (!want.by_mass || c - w < limit) && w >= want.least;
  const int kept = __popcll(__ballot(in));       // the first ones
  const unsigned index = in ? (unsigned)order : 0xFFFFFFFFu;
  x[lane] = index;
  wave_order();
  int place = 0;
#pragma unroll 8
  for (int j = 0; j < (kept + 7) / 8 * 8; ++j) place += (unsigned)x[j] < index;
  if (in) y[place] = order;
  wave_order();
  const u64 mine = y[lane];
  const float ml = logit_of(mine);
  const u64 mw = lane < kept ? r.weight(ml) : 0, reach = wave_scan(mw), sum = last_lane(reach), target = want.target(sum);
  if (mw > 0 && reach >= target && reach - mw < target) write_token(st, row, (int)mine, (float)(r.power(ml, 0) / ldexp((double)sum, -st.scale)));
}

// One workgroup a row: what was collected ranked, the number placed.  8 rows with a nucleus 12 us, a chain of barriers and scans over LDS; a row with a
// rank 3.4, by one wave.
__global__ __launch_bounds__(NT) void sample_last_kernel(Step st) {
  __shared__ union {
    Lds alone;
    Last last;
  } lds;
  __shared__ double roots[ROOTS];
  Last& s = lds.last;
  const int row = blockIdx.x, tid = threadIdx.x, wave = tid / WAVE, lane = tid % WAVE;
  const Wish want(st, row);
  fill_roots(roots);
  Row r = row_of(st, row, roots);
  const Left left(st, row);
  const bool greedy = !(want.T > 0.f);
  const int n = *left.count;
  const float top = left.top[tid];
  const u64 first = left.list[tid];
  __syncthreads();
  if (!greedy && n > LIST) {
    row_alone(lds.alone, roots, st, row, want);
    return;
  }
  if (!greedy && want.few && n > 0 && n <= WAVE) {
    if (wave == 0) last_of_few(st, row, want, r, s.a, first, n);
    return;
  }
  const float m = block_max<NW>(top, s.red);
  if (!(m > -INFINITY)) {
    if (tid == 0) write_token(st, row, -1, 0.f);
    return;
  }
  if (greedy) {
    if (tid == 0) write_token(st, row, *left.first, 1.f);
    return;
  }
  set_scale(r, m, want.T);
  if (tid < n) s.a[tid] = first;
  if (tid + NT < n) s.a[tid + NT] = left.list[tid + NT];
  auto weight = [&](u64 order) { return r.weight(logit_of(order)); };
  if (tid == 0) s.best = 0;
  if (want.few) {
    // all that can be drawn is in the list: the first k of it, the shortest prefix of those, down to min_p, in the order of indices
    __syncthreads();
    sort_rising(s.a, s.b, n);
    const int k = min(n, want.k);
    const u64 total = running_sums(s.b, k, s.waves, [&](int i) { return weight(s.a[i]); });
    const u64 limit = want.by_mass ? want.mass_limit(total) : total;
    int kept = 0;
    for (int i = tid; i < k; i += NT) {
      const u64 before = i > 0 ? s.b[i - 1] : 0;
      if ((before < limit || !want.by_mass) && weight(s.a[i]) >= want.least) kept = i + 1;
    }
    atomicMax(&s.best, kept);
    __syncthreads();
    kept = s.best;
    __syncthreads();
    for (int i = tid; i < kept; i += NT) s.a[i] = s.a[i] << 32 | s.a[i] >> 32;
    __syncthreads();
    sort_rising(s.a, s.b, kept);
    auto turned = [&](int i) { return weight(s.a[i] << 32 | s.a[i] >> 32); };
    const u64 sum = running_sums(s.b, kept, s.waves, turned);
    const u64 target = want.target(sum);
    for (int i = tid; i < kept; i += NT)
      if (s.b[i] >= target && (i == 0 || s.b[i - 1] < target))
        write_token(st, row, (int)(s.a[i] >> 32), (float)(r.power(logit_of(s.a[i] << 32), 0) / ldexp((double)sum, -st.scale)));
    return;
  }
  // Kept tokens of the border's bin join their chunks' sums; the chunk in which the number falls; the token.  The bin's tokens by FINE
  // parts of it, and those of the part in which the border lies against each other.
  int bin = BINS;
  for (int i = tid; i < st.chunks; i += NT) s.sums[i] = left.sums[i];
  if (tid == 0) {
    s.last = 0;
    s.n = 0;
  }
  if (want.far) {
    // the collected tokens in their order: the rank's border gives the weight of the first k, that the limit, and the running sums the tokens
    const Far f = far_borders(left, want, s.waves, s.found);
    bin = f.lo;
    __syncthreads();
    sort_rising(s.a, s.b, n);
    running_sums(s.b, n, s.waves, [&](int i) { return weight(s.a[i]); });
    auto bin_at = [&](int i) { return r.bin(logit_of(s.a[i])); };
    for (int i = tid; i < n; i += NT)
      if (bin_at(i) == f.rank && (i == 0 || bin_at(i - 1) != f.rank)) s.n = i;
    __syncthreads();
    const int of_rank = s.n;
    u64 limit = f.above_rank;
    if (f.rank < BINS) limit += s.b[of_rank + f.need - 1] - (of_rank > 0 ? s.b[of_rank - 1] : 0);
    if (want.by_mass) limit = want.mass_limit(limit);
    for (int i = tid; i < n; i += NT)
      if (bin_at(i) <= f.hi && f.above_lo + (i > 0 ? s.b[i - 1] : 0) < limit) {
        const u64 w = weight(s.a[i]);
        if (w >= want.least) atomicAdd(&s.sums[(unsigned)s.a[i] / CHUNK], w);
        atomicMax(&s.last, s.a[i]);
      }
  } else if (want.by_mass) {
    for (int i = tid; i < FINE; i += NT) s.fine[i] = 0;
    const Border f = find_border(left, want, s.waves, s.found);
    bin = f.bin;
    auto part = [&](u64 order) {
      const float l = logit_of(order), t = (l == m ? 0.f : m - l) * r.to_bin - (float)bin;
      return min((int)(t * FINE), FINE - 1);
    };
    u64 mine[2], w[2];
    int at[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      mine[u] = tid + u * NT < n ? s.a[tid + u * NT] : ~0ull;
      at[u] = FINE;
      if (tid + u * NT < n) {
        w[u] = weight(mine[u]);
        at[u] = part(mine[u]);
        atomicAdd(&s.fine[at[u]], w[u]);
      }
    }
    __syncthreads();
    running_sums(s.b, FINE, s.waves, [&](int i) { return s.fine[i]; });
    // the part whose running sum reaches the limit; in front of it all are kept
    if (tid < FINE) {
      const u64 c = f.above + s.b[tid], before = c - s.fine[tid];
      if (before < f.limit && c >= f.limit) s.best = tid;
    }
    __syncthreads();
    const int border = s.best;
    const u64 above = f.above + (border > 0 ? s.b[border - 1] : 0);
    __syncthreads();
#pragma unroll
    for (int u = 0; u < 2; ++u)
      if (at[u] == border) {
        const int p = atomicAdd(&s.n, 1);
        s.b[p] = mine[u];
        s.a[p] = w[u];
      }
    __syncthreads();
    const int few = s.n;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      bool in = at[u] < border;
      if (at[u] == border) {
        u64 before = above;
        for (int j = 0; j < few; ++j)
          if (s.b[j] < mine[u]) before += s.a[j];
        in = before < f.limit;
      }
      if (in) {
        atomicMax(&s.last, mine[u]);
        if (w[u] >= want.least) atomicAdd(&s.sums[(unsigned)mine[u] / CHUNK], w[u]);
      }
    }
  }
  __syncthreads();
  const u64 border_last = s.last;                // of the border's bin the tokens up to this one are kept
  const u64 total = running_sums(s.b, st.chunks, s.waves, [&](int i) { return s.sums[i]; });
  const u64 target = want.target(total);
  for (int i = tid; i < st.chunks; i += NT)
    if (s.b[i] >= target && (i == 0 || s.b[i - 1] < target)) s.best = i;
  __syncthreads();
  const int chunk = s.best;
  const u64 front = chunk > 0 ? s.b[chunk - 1] : 0;
  const float4 v = chunk4(r, chunk);
  const float l[4] = {v.x, v.y, v.z, v.w};
  u64 a[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int b = r.bin(l[j]);
    const bool in = b < BINS && (b < bin || order_of(l[j], chunk * CHUNK + 4 * tid + j) <= border_last);
    const u64 w = in ? r.weight(l[j]) : 0;
    a[j] = w >= want.least ? w : 0;
  }
  const u64 mine = (a[0] + a[1]) + (a[2] + a[3]);
  u64 c = wave_scan(mine);
  __syncthreads();
  if (lane == WAVE - 1) s.waves[wave] = c;
  __syncthreads();
  for (int w = 0; w < wave; ++w) c += s.waves[w];
  c += front;
  if (c >= target && c - mine < target) {
    c -= mine;
    int j = 0;
    while (j < 3 && c + a[j] < target) c += a[j++];
    const float at_l = j == 0 ? l[0] : j == 1 ? l[1] : j == 2 ? l[2] : l[3];
    write_token(st, row, chunk * CHUNK + 4 * tid + j, (float)(r.power(at_l, 0) / ldexp((double)total, -st.scale)));
  }
}

}  // namespace

extern "C" long yalm_sample_filtered_workspace(int R, int V) {
  const long chunks = ((long)V + CHUNK - 1) / CHUNK;
  return R <= 0 || V <= 0 || chunks > MAX_CHUNKS ? 0 : R * left_bytes((int)chunks);
}

extern "C" int yalm_sample_filtered(const float* logits, const float* u, const float* temperature, const int* top_k, const float* top_p,
                                    const float* min_p, int* out, float* prob, void* workspace, int R, int V, hipStream_t stream) {
  if (R <= 0) return YALM_OK;
  if (V <= 0 || ((uintptr_t)workspace & 15)) return YALM_ERR_ARG;
  int bits = 0;                                  // the weights of V tokens add up to 2^62 at most
  while (bits < 31 && (1l << bits) < V) ++bits;
  const int scale = OCTAVES < 62 - bits ? OCTAVES : 62 - bits;
  const long chunks = ((long)V + CHUNK - 1) / CHUNK;
  Step st = {logits, u, temperature, top_k, top_p, min_p, out, prob, V, scale, (unsigned char*)workspace, 0, (int)chunks};
  if (workspace == nullptr || chunks > MAX_CHUNKS || R > 65535) {
    sample_alone_kernel<<<R, NT, 0, stream>>>(st);
    return launch_status();
  }
  st.row_bytes = left_bytes((int)chunks);
  // As many workgroups as run at once, twice over for rows of unequal settings, and no more a row than it has chunks: 8 rows of 128,256 with a nucleus
  // 31 us in 32 workgroups each, 191 in one each (as without a workspace); 256 rows in 4 each 100 to 104 (mixed settings), in one each 227.
  int n = 1;
  while (n < MAX_GROUPS_ROW && n < chunks && (n * R < 4 * compute_units() || n * CHUNKS_EACH < chunks)) n <<= 1;
  const dim3 grid(n, R);
  sample_top_kernel<<<grid, NT, 0, stream>>>(st);
  if (top_k != nullptr || top_p != nullptr) sample_sift_kernel<<<grid, NT, 0, stream>>>(st);
  sample_sum_kernel<<<grid, NT, 0, stream>>>(st);
  sample_last_kernel<<<R, NT, 0, stream>>>(st);
  return launch_status();
}
