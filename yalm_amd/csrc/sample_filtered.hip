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
// Nothing is sorted.  Tokens fall into BINS bins by (max - l) / T; the bin in which a filter's border lies comes from running
// sums over the bins, and only that bin's tokens are ranked against each other (or, where many share a bin, narrowed by the
// bits of their logits until all that are left are equal).  Up to LIST tokens in front of the border are copied to LDS and
// everything behind that is done there.
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
constexpr int OCTAVES = 44;                      // the bins reach down to 2^-44 of the greatest weight
constexpr int SEG = 192;                         // tokens of the list that a wave's run of the row may hold
constexpr int BORDER = 768;                      // tokens of one bin that are ranked against each other
constexpr int GROUPS = BINS / NW;                // partial sums of the row that a wave leaves for the walk

__device__ __forceinline__ u64 wave_sum64(u64 v) {
#pragma unroll
  for (int o = WAVE / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, WAVE);
  return v;
}
template <typename V>
__device__ __forceinline__ V wave_scan(V v, int lane) {       // inclusive
#pragma unroll
  for (int o = 1; o < WAVE; o <<= 1) {
    const V up = __shfl_up(v, o, WAVE);
    if (lane >= o) v += up;
  }
  return v;
}

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
  double to_exponent;          // exponents of 2 a unit of l
  int scale;                   // the greatest weight is 2^scale

  // not falling as l falls; BINS: the token weighs nothing
  __device__ __forceinline__ int bin(float v) const {
    const float t = (v == m ? 0.f : m - v) * to_bin;
    return t < (float)BINS ? (int)t : BINS;
  }
  // 2^y by its series around the nearest whole exponent (|z| <= ln 2 / 2: the first term left out is 6e-15 of it)
  __device__ __forceinline__ double power(float v) const {
    const double y = v == m ? 0.0 : fmax(((double)v - (double)m) * to_exponent, -1000.0);
    const double n = rint(y), z = (y - n) * 0.69314718055994530942;
    double p = 1.0 / 39916800.0;
    p = fma(p, z, 1.0 / 3628800.0);
    p = fma(p, z, 1.0 / 362880.0);
    p = fma(p, z, 1.0 / 40320.0);
    p = fma(p, z, 1.0 / 5040.0);
    p = fma(p, z, 1.0 / 720.0);
    p = fma(p, z, 1.0 / 120.0);
    p = fma(p, z, 1.0 / 24.0);
    p = fma(p, z, 1.0 / 6.0);
    p = fma(p, z, 0.5);
    p = fma(p, z, 1.0);
    p = fma(p, z, 1.0);
    return ldexp(p, (int)n);
  }
  // of a token whose bin is below BINS; at most 2^44: adding 2^52 rounds to the nearest whole number
  __device__ __forceinline__ u64 weight(float v) const {
    return (u64)__double_as_longlong(ldexp(power(v), scale) + 4503599627370496.0) & ((1ull << 52) - 1);
  }
};

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
  unsigned c = wave_scan(c0 + c1, lane);
  u64 a = wave_scan(a0 + a1, lane);
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

__global__ __launch_bounds__(NT) void sample_filtered_kernel(const float* __restrict__ logits, const float* __restrict__ us,
                                                             const float* __restrict__ temperature, const int* __restrict__ top_k,
                                                             const float* __restrict__ top_p, const float* __restrict__ min_p,
                                                             int* __restrict__ out, float* __restrict__ prob, int V, int scale) {
  __shared__ Lds s;
  const int tid = threadIdx.x, wave = tid / WAVE, lane = tid % WAVE;
  const int row = blockIdx.x;
  Row r;
  r.l = logits + (size_t)row * V;
  r.V = V;
  r.aligned = ((uintptr_t)r.l & 15) == 0;
  r.scale = scale;
  const int n_tiles = (V + TILE - 1) / TILE, tpw = (n_tiles + NW - 1) / NW;
  const int t0 = min(n_tiles, wave * tpw), t1 = min(n_tiles, t0 + tpw);     // the tiles of this wave
  const float T = temperature != nullptr ? temperature[row] : 1.f;
  const int k = top_k != nullptr ? top_k[row] : 0;
  const float p = top_p != nullptr ? top_p[row] : 1.f;
  const float mp = min_p != nullptr ? min_p[row] : 0.f;
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
    if (tid == 0) {
      out[row] = -1;
      if (prob != nullptr) prob[row] = 0.f;
    }
    return;
  }
  if (!(T > 0.f)) {                              // the first of the greatest
    int first = V;
    each<4>(r, s, false, t0, t1, wave, lane, [&](float l, int i) { first = l == r.m ? min(first, i) : first; });
    if (first < V) atomicMin(&s.best, first);
    __syncthreads();
    if (tid == 0) {
      out[row] = s.best;
      if (prob != nullptr) prob[row] = 1.f;
    }
    return;
  }
  r.to_exponent = 1.4426950408889634074 / (double)T;
  r.to_bin = (float)fmin(r.to_exponent * ((double)BINS / OCTAVES), 1e30);

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
  const bool by_rank = k > 0 && k < V, by_mass = p < 1.f;
  auto mass_limit = [&](u64 total) {
    const double x = ceil((double)p * (double)total);
    return x >= 1.0 ? (u64)x : 1ull;
  };
  if (by_rank) {
    fill(false);
    const Found f = find_bin<false>(s, [&](u64) { return (u64)k; });
    if (f.bin < BINS) {
      if (f.through <= (unsigned)(NW * SEG)) collect(f.bin);
      narrow(std::false_type{}, f, (u64)k);
    }
  }
  if (by_mass) {
    fill(true);
    u64 limit = 1;
    const Found f = find_bin<true>(s, [&](u64 total) { return limit = mass_limit(total); });
    if (f.bin < BINS) {
      if (!list && f.through <= (unsigned)(NW * SEG)) collect(f.bin);
      narrow(std::true_type{}, f, limit);
    }
  }

  // the walk: partial sums, the part in which the target falls, the token in it
  const double floor_w = mp > 0.f ? ceil(ldexp((double)fminf(mp, 1.f), scale)) : 0.0;
  const u64 least = floor_w > 1.0 ? (u64)floor_w : 1ull;
  auto amount = [&](float l, int i) -> u64 {
    if (r.bin(l) >= BINS || !kept(s, key_of(l), i, thr_key, thr_i)) return 0;
    const u64 w = r.weight(l);
    return w >= least ? w : 0;
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
  const double goal = ceil((double)us[row] * (double)total);
  const u64 target = goal >= 1.0 ? min((u64)goal, total) : 1ull;      // u of 0 or no number: the first; of 1 and more the last
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
      const u64 incl = wave_scan(mine, lane);
      const u64 reached = __ballot(front + incl >= target);
      if (reached == 0) {
        front += __shfl(incl, WAVE - 1, WAVE);
        continue;
      }
      if (lane == __ffsll((long long)reached) - 1) {
        u64 c = front + (incl - mine);
        int j = 0;
        while (j < 3 && c + a4[j] < target) c += a4[j++];
        const float at_l = j == 0 ? l[0] : j == 1 ? l[1] : j == 2 ? l[2] : l[3];
        out[row] = j == 0 ? i[0] : j == 1 ? i[1] : j == 2 ? i[2] : i[3];
        if (prob != nullptr) prob[row] = (float)(r.power(at_l) / ldexp((double)total, -scale));
      }
      return;
    }
  }
}

}  // namespace

extern "C" int yalm_sample_filtered(const float* logits, const float* u, const float* temperature, const int* top_k, const float* top_p,
                                    const float* min_p, int* out, float* prob, int R, int V, hipStream_t stream) {
  if (R <= 0) return YALM_OK;
  if (V <= 0) return YALM_ERR_ARG;
  int bits = 0;                                  // the weights of V tokens add up to 2^62 at most
  while (bits < 31 && (1l << bits) < V) ++bits;
  const int scale = OCTAVES < 62 - bits ? OCTAVES : 62 - bits;
  sample_filtered_kernel<<<R, NT, 0, stream>>>(logits, u, temperature, top_k, top_p, min_p, out, prob, V, scale);
  return launch_status();
}
